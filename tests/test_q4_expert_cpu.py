"""4-bit weights and expert routing without a GPU: the packed size, the layout's restatement, and every refusal of the
C entry points. The refusals come before any device work, so a zeroed block of memory stands in for a handle (it is
never used as one)."""
from __future__ import annotations

import ctypes

import numpy as np
import pytest
import torch

import emugemm
import q4ref

INVALID_HANDLE, INVALID_POINTER, INVALID_SIZE, INVALID_VALUE = 1, 3, 4, 11
P = 4096            # an aligned address that is never read


@pytest.fixture()
def h():
    return ctypes.create_string_buffer(1 << 16)


@pytest.mark.parametrize("E,N,K,group", [(1, 1, 1, 32), (1, 16, 64, 64), (3, 17, 65, 128), (2, 100, 1000, 32)])
def test_q4_bytes(E, N, K, group):
    nb, kb, G = -(-N // 16), -(-K // 64), -(-K // group)
    codes = E * nb * kb * 512
    assert emugemm.q4_bytes(E, N, K, group) == -(-codes // 256) * 256 + E * nb * G * 32


@pytest.mark.parametrize("E,N,K,group", [(0, 8, 8, 32), (1025, 8, 8, 32), (1, 0, 8, 32), (1, 8, 0, 32), (1, 8, 8, 16),
                                         (1, 8, 8, 256), (1, 8, 1 << 31, 32), (-1, 8, 8, 32)])
def test_q4_bytes_out_of_range(E, N, K, group):
    assert emugemm.q4_bytes(E, N, K, group) == 0


@pytest.mark.parametrize("E,N,K", [(1024, 1 << 30, 1 << 30), (1024, 1 << 20, (1 << 20) + 1), (1, 1 << 30, 1 << 30)])
def test_q4_bytes_of_more_than_memory(E, N, K):
    """More than 2^50 weights: the count of bytes would wrap, so they are refused."""
    assert emugemm.q4_bytes(E, N, K, 32) == 0
    assert emugemm.q4_bytes(1024, 1 << 20, 1 << 20, 32) == 2 ** 49 + 2 ** 46


def test_layout_restatement_round_trip():
    """q4ref.pack against the layout read back nibble by nibble."""
    E, N, K, group = 2, 19, 70, 32
    g = np.random.default_rng(0)
    q, s = q4ref.quantise(g.standard_normal((E * N, K)), group)
    raw = q4ref.pack(q, s, E, N, K, group)
    nb, kb, G = 2, 2, 3
    at = -(-E * nb * kb * 512 // 256) * 256
    for e, n, k in ((0, 0, 0), (1, 18, 69), (0, 9, 33), (1, 3, 64), (0, 15, 7)):
        r, kk = n % 16, k % 64
        word = ((e * nb + n // 16) * kb + k // 64) * 128 + (4 * (r % 8) + kk % 32 // 8) * 4 + (kk // 32) * 2 + r // 8
        nibble = [0, 4, 1, 5, 2, 6, 3, 7][kk % 8]
        assert (int(raw[:at].view(np.uint32)[word]) >> (4 * nibble)) & 15 == q[e * N + n, k] + 8
        bits = raw[at:].view(np.uint16)[((e * nb + n // 16) * G + k // group) * 16 + (r % 8) * 2 + r // 8]
        assert torch.tensor([int(bits)], dtype=torch.int32).to(torch.int16).view(torch.bfloat16).item() == s[e * N + n, k // group]


def test_q4_refusals(h):
    L = emugemm.lib()
    ok = dict(E=2, N=8, K=64, W=P, ldw=64, dt=0, group=32, packed=P)

    def pack(hd=h, **kw):
        a = {**ok, **kw}
        return L.emugemm_q4_pack(hd, a["E"], a["N"], a["K"], a["W"], a["ldw"], a["dt"], a["group"], a["packed"])

    def unpack(hd=h, **kw):
        a = {**ok, **kw}
        return L.emugemm_q4_unpack(hd, a["E"], a["N"], a["K"], a["group"], a["packed"], a["W"], a["ldw"])

    for f in (pack, unpack):
        assert f(hd=None) == INVALID_HANDLE
        assert f(group=48) == INVALID_VALUE
        for kw in (dict(E=0), dict(E=1025), dict(N=0), dict(K=0), dict(ldw=63), dict(N=-4)):
            assert f(**kw) == INVALID_SIZE, kw
        for kw in (dict(W=0), dict(W=P + 1), dict(packed=0), dict(packed=P + 8)):
            assert f(**kw) == INVALID_POINTER, kw
    assert pack(dt=3) == INVALID_VALUE and pack(dt=-1) == INVALID_VALUE
    assert pack(dt=2, W=P + 1) == INVALID_POINTER


def test_q4_gemm_refusals(h):
    L = emugemm.lib()
    ok = dict(M=4, E=2, N=8, K=64, A=P, lda=64, dt=0, off=P, packed=P, group=32, C=P, ldc=8)

    def gemm(hd=h, **kw):
        a = {**ok, **kw}
        return L.emugemm_q4_gemm(hd, a["M"], a["N"], a["K"], a["A"], a["lda"], a["dt"], a["packed"], a["group"], a["C"],
                                 a["ldc"])

    def experts(hd=h, **kw):
        a = {**ok, **kw}
        return L.emugemm_q4_gemm_experts(hd, a["M"], a["E"], a["N"], a["K"], a["A"], a["lda"], a["dt"], a["off"],
                                         a["packed"], a["group"], a["C"], a["ldc"])

    for f in (gemm, experts):
        assert f(hd=None) == INVALID_HANDLE
        for kw in (dict(group=0), dict(dt=7)):
            assert f(**kw) == INVALID_VALUE
        for kw in (dict(M=-1), dict(N=0), dict(K=0), dict(lda=63), dict(ldc=7), dict(K=1 << 31, lda=1 << 31)):
            assert f(**kw) == INVALID_SIZE, kw
        for kw in (dict(A=0), dict(A=P + 2), dict(C=0), dict(C=P + 1), dict(packed=0), dict(packed=P + 4),
                   dict(dt=1, A=P + 1)):
            assert f(**kw) == INVALID_POINTER, kw
        assert f(M=0, A=0, C=0) == 0          # nothing to do
    assert experts(E=0) == INVALID_SIZE and experts(E=1025) == INVALID_SIZE
    assert experts(off=0) == INVALID_POINTER and experts(off=P + 2) == INVALID_POINTER


def test_expert_refusals(h):
    L = emugemm.lib()

    def sort(hd=h, T=4, k=2, E=8, a=P, b=P, c=P, d=P):
        return L.emugemm_expert_sort(hd, T, k, E, a, b, c, d)

    assert sort(hd=None) == INVALID_HANDLE
    for kw in (dict(T=-1), dict(k=0), dict(E=0), dict(E=1025), dict(T=1 << 30, k=2)):
        assert sort(**kw) == INVALID_SIZE, kw
    for kw in (dict(a=0), dict(b=0), dict(c=0), dict(d=0), dict(a=P + 2), dict(T=0, d=0)):
        assert sort(**kw) == INVALID_POINTER, kw

    ok = dict(T=4, k=2, H=16, X=P, ldx=16, dt=0, place=P, w=P, Y=P, ldy=16, D=P, ldd=16, dw=P)

    def gather(hd=h, **kw):
        a = {**ok, **kw}
        return L.emugemm_expert_gather(hd, a["T"], a["k"], a["H"], a["X"], a["ldx"], a["dt"], a["place"], a["Y"], a["ldy"])

    def gather_backward(hd=h, **kw):
        a = {**ok, **kw}
        return L.emugemm_expert_gather_backward(hd, a["T"], a["k"], a["H"], a["X"], a["ldx"], a["dt"], a["place"], a["Y"],
                                                a["ldy"])

    def combine(hd=h, **kw):
        a = {**ok, **kw}
        return L.emugemm_expert_combine(hd, a["T"], a["k"], a["H"], a["X"], a["ldx"], a["dt"], a["place"], a["w"], a["Y"],
                                        a["ldy"])

    def combine_backward(hd=h, **kw):
        a = {**ok, **kw}
        return L.emugemm_expert_combine_backward(hd, a["T"], a["k"], a["H"], a["X"], a["ldx"], a["Y"], a["ldy"], a["dt"],
                                                 a["place"], a["w"], a["D"], a["ldd"], a["dw"])

    for f in (gather, gather_backward, combine, combine_backward):
        assert f(hd=None) == INVALID_HANDLE
        assert f(dt=3) == INVALID_VALUE
        for kw in (dict(T=-1), dict(k=0), dict(H=-1), dict(ldx=15), dict(ldy=15), dict(T=1 << 30, k=2)):
            assert f(**kw) == INVALID_SIZE, kw
        for kw in (dict(X=0), dict(Y=0), dict(place=0), dict(X=P + 2), dict(place=P + 1)):
            assert f(**kw) == INVALID_POINTER, kw
        assert f(T=0, X=0, Y=0, place=0) == 0
    assert combine(w=0) == INVALID_POINTER and combine_backward(w=0) == INVALID_POINTER
    assert combine_backward(dw=0) == INVALID_POINTER and combine_backward(D=0) == INVALID_POINTER
    assert combine_backward(ldd=15) == INVALID_SIZE
    assert gather(H=0, X=0, Y=0, place=0) == 0


def test_binding_checks_tensor_types():
    x, y = torch.zeros(4), torch.zeros(4, dtype=torch.bfloat16)
    assert emugemm._dtype(None, x) == emugemm.F32 and emugemm._dtype(None, y) == emugemm.BF16
    assert emugemm._dtype(emugemm.F16, 4096, 4096) == emugemm.F16
    with pytest.raises(ValueError):
        emugemm._dtype(None, x, y)
    with pytest.raises(ValueError):
        emugemm._dtype(emugemm.F16, x)
    with pytest.raises(ValueError):
        emugemm._dtype(None, 4096)
    h = emugemm.Handle.__new__(emugemm.Handle)      # the checks need no device
    h.h, h.device = None, -1                        # -1: the host, where these tensors are
    i = torch.zeros(4, dtype=torch.int32)
    assert h._at(i, "torch.int32") == i.data_ptr() and h._at(None) == 0 and h._at(4096, "torch.int32") == 4096
    with pytest.raises(ValueError):
        h._at(torch.zeros(4, dtype=torch.int64), "torch.int32")
    h.device = 0
    with pytest.raises(ValueError):
        h._at(i, "torch.int32")                     # a host tensor


def test_every_entry_point_is_bound():
    for n in emugemm.header_functions():
        if "q4" in n or "expert" in n:
            assert n in emugemm._SIGS, n
