"""Sizes beyond a C int are refused by the binding of the 4-bit and routing calls instead of arriving as their low 32 bits.
A stand-in for the library, which accepts everything, shows what would have been passed on."""
from __future__ import annotations

import pytest

import emugemm

INVALID_SIZE = 4
P = 4096
OK = {
    "q4_pack": (dict(E=1, N=16, K=64, W=P, ldw=64, group=32, packed=P, dtype=0), ("E", "N", "group")),
    "q4_unpack": (dict(E=1, N=16, K=64, group=32, packed=P, W=P, ldw=64), ("E", "N", "group")),
    "q4_gemm": (dict(M=4, N=16, K=64, A=P, lda=64, packed=P, group=32, C=P, ldc=16, dtype=0), ("M", "N", "group")),
    "q4_gemm_experts": (dict(R=4, E=2, N=16, K=64, A=P, lda=64, offsets=P, packed=P, group=32, C=P, ldc=16, dtype=0),
                        ("R", "E", "N", "group")),
    "expert_sort": (dict(T=4, topk=2, E=8, expert=P, order=P, place=P, offsets=P), ("T", "topk", "E")),
    "expert_gather": (dict(T=4, topk=2, H=16, X=P, ldx=16, place=P, XS=P, ldxs=16, dtype=0), ("T", "topk", "H")),
    "expert_gather_backward": (dict(T=4, topk=2, H=16, dXS=P, lddxs=16, place=P, dX=P, lddx=16, dtype=0), ("T", "topk", "H")),
    "expert_combine": (dict(T=4, topk=2, H=16, YS=P, ldys=16, place=P, weights=P, Y=P, ldy=16, dtype=0), ("T", "topk", "H")),
    "expert_combine_backward": (dict(T=4, topk=2, H=16, dY=P, lddy=16, YS=P, ldys=16, place=P, weights=P, dYS=P, lddys=16,
                                     dweights=P, dtype=0), ("T", "topk", "H")),
}


class StandIn:
    def __init__(self):
        self.calls = []

    def __getattr__(self, name):
        return lambda *args: self.calls.append((name, args)) or 0


@pytest.mark.parametrize("name", list(OK))
def test_calls_refuse_sizes_beyond_int(monkeypatch, name):
    lib = StandIn()
    monkeypatch.setattr(emugemm, "_lib", lib)
    h = emugemm.Handle.__new__(emugemm.Handle)
    h.h, h.device = None, 0
    kw, sizes = OK[name]
    getattr(h, name)(**kw)
    assert [c[0] for c in lib.calls] == ["emugemm_" + name]
    for s in sizes:
        for big in (kw[s] + 2 ** 32, 2 ** 31, -2 ** 31 - 1, kw[s] - 2 ** 32):
            with pytest.raises(emugemm.EmuGemmError) as e:
                getattr(h, name)(**{**kw, s: big})
            assert e.value.code == INVALID_SIZE
        getattr(h, name)(**{**kw, s: -1})        # left to the library, which refuses it
        assert lib.calls.pop()[1]
    assert len(lib.calls) == 1


@pytest.mark.parametrize("E,N,group", [(1, 2 ** 32 + 16, 32), (2 ** 32 + 1, 16, 32), (1, 16, 2 ** 32 + 32), (1, 2 ** 31, 32),
                                       (1 - 2 ** 32, 16, 32), (1, 16 - 2 ** 32, 32)])
def test_q4_bytes_beyond_int(E, N, group):
    assert emugemm.q4_bytes(E, N, 64, group) == 0
