"""4-bit weights on the GPU, through the C ABI, against plain 64-bit restatements (q4ref).

Bars: packing and unpacking bit for bit; products within q4ref.product_bound, which counts the output's rounding and
the FP32 accumulation; the same call twice bit for bit."""
from __future__ import annotations

import os
import subprocess
import sys

import numpy as np
import pytest

import emugemm
import q4ref
from q4ref import TYPES

pytestmark = pytest.mark.gpu


def packed_on_gpu(torch, h, w, E, N, K, group, ldw=None):
    out = torch.full((emugemm.q4_bytes(E, N, K, group),), 0xA5, dtype=torch.uint8, device="cuda")
    h.q4_pack(E, N, K, w, ldw or K, group, out)
    h.sync()
    return out.cpu().numpy()


def same_bytes(got, want, E, N, K):
    """Equal but for the bytes between the codes and the scales, which no one reads or writes."""
    codes = E * -(-N // 16) * -(-K // 64) * 512
    at = -(-codes // 256) * 256
    return np.array_equal(got[:codes], want[:codes]) and np.array_equal(got[at:], want[at:])


# --------------------------------------------------------------------------------------------------- pack and unpack
@pytest.mark.parametrize("kind", ["fp32", "fp16", "bf16"])
@pytest.mark.parametrize("E,N,K,group", [(1, 1, 1, 32), (1, 16, 64, 64), (1, 17, 65, 128), (3, 40, 200, 32),
                                         (2, 33, 129, 64), (1, 100, 1000, 128), (5, 16, 31, 32)])
def test_pack_bits(cuda, handle, kind, E, N, K, group):
    torch = cuda
    g = torch.Generator().manual_seed(N * K)
    w = (torch.randn(E * N, K, generator=g) * 0.02).to(TYPES[kind])
    q, s = q4ref.quantise(w.double().numpy(), group)
    assert same_bytes(packed_on_gpu(torch, handle, w.cuda(), E, N, K, group), q4ref.pack(q, s, E, N, K, group), E, N, K)


@pytest.mark.parametrize("group", [32, 64, 128])
def test_pack_special_values(cuda, handle, group):
    """Ties of the quotient and values one ulp beside them, groups of zeros, Inf, NaN, FP32 subnormals, the largest
    FP32 values, and scales that round to subnormal bf16 or to zero."""
    torch = cuda
    N, K = 20, 4 * group + 5
    g = np.random.default_rng(group)
    w = g.standard_normal((N, K)).astype(np.float32)
    for r in range(8):                       # scale 2^j exactly: the quotient's ties are representable
        w[r, :group] = ((g.integers(-14, 15, group) * 0.5).astype(np.float32) * np.float32(2.0 ** (r - 4)))
        w[r, 0] = 7 * 2.0 ** (r - 4)
        half = w[r, 1:group:3].copy()
        w[r, 1:group:3] = np.nextafter(half, np.float32(np.inf) if r % 2 else np.float32(-np.inf))
        w[r, 0] = 7 * 2.0 ** (r - 4)
    s = np.float32(0.171875)                 # ties of a scale with more bits: (j + 1/2) s
    w[8, :group] = (g.integers(-7, 7, group) + 0.5).astype(np.float32) * s
    w[8, 0] = 7 * s
    w[9, group:2 * group] = 0
    w[10, 3] = np.inf
    w[11, 3] = -np.inf
    w[12, 3] = np.nan
    w[13] = g.integers(-100, 100, K) * np.float32(2.0 ** -149)
    w[14] = g.standard_normal(K).astype(np.float32) * np.float32(2.0 ** -126)
    w[15] = g.standard_normal(K).astype(np.float32) * np.float32(3e-39)
    w[16] = g.uniform(-1, 1, K).astype(np.float32) * np.float32(3.4e38)
    w[17] = g.standard_normal(K).astype(np.float32) * np.float32(2.0 ** -100)
    q, sc = q4ref.quantise(w, group)
    got = packed_on_gpu(torch, handle, torch.from_numpy(w).cuda(), 1, N, K, group)
    assert same_bytes(got, q4ref.pack(q, sc, 1, N, K, group), 1, N, K)


@pytest.mark.parametrize("kind", ["fp32", "bf16"])
def test_pack_strided_and_misaligned(cuda, handle, kind):
    """Rows further apart than K (with NaN between them) and a base one element off the vector alignment."""
    torch = cuda
    N, K, ld, group = 37, 200, 211, 64
    g = torch.Generator().manual_seed(5)
    w = torch.randn(N, K, generator=g).to(TYPES[kind])
    q, s = q4ref.quantise(w.double().numpy(), group)
    want = q4ref.pack(q, s, 1, N, K, group)
    for off in (0, 1):
        buf = torch.full((N * ld + 1,), float("nan"), dtype=TYPES[kind], device="cuda")
        view = buf[off:off + N * ld].view(N, ld)
        view[:, :K] = w.cuda()
        assert same_bytes(packed_on_gpu(torch, handle, view, 1, N, K, group, ld), want, 1, N, K)


@pytest.mark.parametrize("E,N,K,group,ld", [(1, 1, 1, 32, 1), (2, 19, 70, 32, 70), (1, 33, 200, 128, 204), (1, 16, 64, 64, 67)])
def test_unpack_exact(cuda, handle, E, N, K, group, ld):
    torch = cuda
    packed, w = q4ref.weights(N + K, E, N, K, group)
    out = torch.full((E * N, ld), -7.5, device="cuda")
    handle.q4_unpack(E, N, K, group, packed, out, ld)
    handle.sync()
    o = out.cpu().numpy()
    assert np.array_equal(o[:, :K].astype(np.float64), w.reshape(E * N, K))
    assert (o[:, K:] == -7.5).all()


def test_pack_beyond_32_bit_offsets(cuda, handle):
    """More than 2^31 weights: the last rows of the last expert are read, packed and read back at 64-bit offsets."""
    torch = cuda
    E, N, K, group = 9, 16384, 16384, 128
    w = torch.zeros(E * N, K, dtype=torch.bfloat16, device="cuda")
    tail = torch.randn(48, K, generator=torch.Generator().manual_seed(1)).bfloat16()
    w[-48:] = tail.cuda()
    packed = torch.empty(emugemm.q4_bytes(E, N, K, group), dtype=torch.uint8, device="cuda")
    handle.q4_pack(E, N, K, w, K, group, packed)
    q, s = q4ref.quantise(tail.double().numpy(), group)
    x = torch.randn(2, K, generator=torch.Generator().manual_seed(2)).bfloat16()
    off = torch.zeros(E + 1, dtype=torch.int32)
    off[E] = 2
    y = torch.empty(2, N, dtype=torch.bfloat16, device="cuda")
    handle.q4_gemm_experts(2, E, N, K, x.cuda(), K, off.cuda(), packed, group, y, N)
    handle.sync()
    v, xd = q4ref.values(q, s, group), x.double().numpy()
    ref = xd @ v.T
    got = y[:, -48:].double().cpu().numpy()
    assert (np.abs(got - ref) <= q4ref.product_bound(xd, v, ref, group, "bf16")).all()
    assert (y[:, :-48] == 0).all().item()


# ----------------------------------------------------------------------------------------------------------- product
def check_product(torch, h, M, N, K, group, kind, seed=0, lda=None, ldc=None, packed=None, w=None, x=None):
    lda, ldc = lda or K, ldc or N
    if packed is None:
        packed, w = q4ref.weights(seed + N, 1, N, K, group)
        w = w[0]
    if x is None:
        x = torch.randn(M, K, generator=torch.Generator().manual_seed(seed + M)).to(TYPES[kind])
    a = torch.full((M, lda), float("nan"), dtype=TYPES[kind], device="cuda")
    a[:, :K] = x.cuda()
    c = torch.full((M + 1, ldc), -7.5, dtype=TYPES[kind], device="cuda")
    h.q4_gemm(M, N, K, a, lda, packed, group, c, ldc)
    h.sync()
    got = c.double().cpu().numpy()
    assert (got[M:] == -7.5).all() and (got[:, N:] == -7.5).all(), "written outside C"
    xd = x.double().numpy()
    ref = xd @ w.T
    bad = np.abs(got[:M, :N] - ref) > q4ref.product_bound(xd, w, ref, group, kind)
    assert not bad.any(), (int(bad.sum()), np.argwhere(bad)[:4], np.abs(got[:M, :N] - ref).max())
    return c


@pytest.mark.parametrize("kind", ["fp32", "fp16", "bf16"])
@pytest.mark.parametrize("M,N,K,group", [
    (1, 1, 1, 32), (1, 16, 64, 64), (1, 4096, 4096, 128), (2, 300, 1000, 32), (3, 17, 129, 128), (5, 130, 127, 64),
    (8, 256, 512, 32), (9, 257, 2048, 128), (16, 64, 8192, 64), (17, 2000, 640, 32), (24, 333, 1111, 32),
    (33, 1024, 1024, 128), (48, 100, 333, 64), (65, 96, 4100, 32), (128, 384, 512, 128), (131, 129, 200, 64),
    (257, 640, 1088, 32), (300, 77, 65, 128), (1, 20000, 96, 32), (4, 48, 16000, 128)])
def test_product(cuda, handle, kind, M, N, K, group):
    check_product(cuda, handle, M, N, K, group, kind)


@pytest.mark.parametrize("kind", ["fp32", "bf16"])
@pytest.mark.parametrize("M,N,K,group", [(100, 300, 2200, 64), (70, 600, 4100, 128), (128, 4096, 1100, 32), (90, 2500, 1024, 64),
                                         (60, 256, 6500, 32), (127, 4100, 2176, 128)])
def test_product_k_splits(cuda, handle, kind, M, N, K, group):
    """Few tiles: two or four CTA pairs share a tile and split its K, also into parts that are not equal."""
    check_product(cuda, handle, M, N, K, group, kind)


@pytest.mark.parametrize("kind", ["fp32", "fp16"])
@pytest.mark.parametrize("M,N,K,group", [(61, 4096, 1536, 128), (128, 4900, 1700, 64), (49, 5600, 2100, 32), (100, 3800, 2048, 64),
                                         (128, 5700, 1536, 128), (66, 8400, 1050, 64)])
def test_product_three_k_splits(cuda, handle, kind, M, N, K, group):
    """As many tiles as clusters of four, three or two pairs just fit, and one more."""
    check_product(cuda, handle, M, N, K, group, kind)


@pytest.mark.parametrize("kind", ["fp16", "bf16"])
@pytest.mark.parametrize("M,N,K,group", [(300, 8, 128, 32), (150, 104, 200, 64), (1000, 2008, 256, 128), (777, 1288, 65, 128)])
def test_product_wide_stores(cuda, handle, kind, M, N, K, group):
    """Columns in eights that end inside a warp's 32 and a CTA's 128, rows inside a tile."""
    check_product(cuda, handle, M, N, K, group, kind)
    check_product(cuda, handle, M, N, K, group, kind, ldc=N + 24)


@pytest.mark.parametrize("kind", ["fp32", "bf16"])
@pytest.mark.parametrize("counts", [[60, 70, 0, 90], [0, 130, 1], [55] * 6])
def test_experts_k_splits(cuda, handle, kind, counts):
    check_experts(cuda, handle, counts, 200, 2100, 32, kind, tail=5)


@pytest.mark.parametrize("kind", ["fp32", "fp16", "bf16"])
@pytest.mark.parametrize("M", [1, 6, 40, 150])
@pytest.mark.parametrize("lda,ldc", [(200, 96), (201, 97), (208, 104)])
def test_product_strides(cuda, handle, kind, M, lda, ldc):
    """Leading dimensions beyond the rows (NaN between the rows of A), K = 200, also not multiples of the vectors."""
    check_product(cuda, handle, M, 96, 200, 64, kind, lda=lda, ldc=ldc)


@pytest.mark.parametrize("kind", ["fp32", "bf16"])
@pytest.mark.parametrize("M", [2, 70])
def test_product_misaligned_base(cuda, handle, kind, M):
    """A and C one element off their vector alignment."""
    torch = cuda
    N, K, group = 50, 256, 128
    packed, w = q4ref.weights(3, 1, N, K, group)
    x = torch.randn(M, K, generator=torch.Generator().manual_seed(9)).to(TYPES[kind])
    a = torch.empty(M * K + 1, dtype=TYPES[kind], device="cuda")
    a[1:] = x.cuda().view(-1)
    c = torch.empty(M * N + 1, dtype=TYPES[kind], device="cuda")
    handle.q4_gemm(M, N, K, a[1:], K, packed, group, c[1:], N)
    handle.sync()
    xd = x.double().numpy()
    ref = xd @ w[0].T
    got = c[1:].view(M, N).double().cpu().numpy()
    assert (np.abs(got - ref) <= q4ref.product_bound(xd, w[0], ref, group, kind)).all()


@pytest.mark.parametrize("M", [1, 30, 200])
def test_product_fp32_keeps_24_bits(cuda, handle, M):
    """One value of K: C = scale * q * a. The three slices' products are exact, so only their two additions and the
    final rounding of the FP32 result are off: at most 3 * 2^-24 of the value; also for values near the ends of FP32."""
    torch = cuda
    N = 40
    packed, w = q4ref.weights(7, 1, N, 1, 32, scale=1.0)
    g = np.random.default_rng(M)
    for mag in (1.0, 1e30, 2.0 ** -90, 2.0 ** -100):
        x = (g.standard_normal((M, 1)) * mag).astype(np.float32)
        a = torch.from_numpy(x).cuda()
        c = torch.empty(M, N, device="cuda")
        handle.q4_gemm(M, N, 1, a, 1, packed, 32, c, N)
        handle.sync()
        ref = x.astype(np.float64) @ w[0].T
        assert (np.abs(c.double().cpu().numpy() - ref) <= 3 * 2.0 ** -24 * np.abs(ref)).all(), mag


@pytest.mark.parametrize("kind", ["fp32", "fp16", "bf16"])
@pytest.mark.parametrize("M", [3, 40, 150])
def test_product_nonfinite_rows(cuda, handle, kind, M):
    """Inf and NaN in a row of A stay in that row and come out as in the formula: NaN where a weight of the place is 0."""
    torch = cuda
    N, K, group = 64, 320, 64
    packed, w = q4ref.weights(11, 1, N, K, group)
    w = w[0]
    x = torch.randn(M, K, generator=torch.Generator().manual_seed(4)).to(TYPES[kind])
    x[0, 5] = float("inf")
    x[M - 1, 300] = float("nan")
    c = torch.empty(M, N, dtype=TYPES[kind], device="cuda")
    handle.q4_gemm(M, N, K, x.cuda(), K, packed, group, c, N)
    handle.sync()
    got = c.double().cpu().numpy()
    q = w[:, 5]
    assert np.array_equal(np.isnan(got[0]), q == 0)
    assert np.array_equal(got[0][q != 0], np.where(q > 0, np.inf, -np.inf)[q != 0])
    assert np.isnan(got[M - 1]).all()
    xd = x.double().numpy()
    ref = xd[1:M - 1] @ w.T
    assert (np.abs(got[1:M - 1] - ref) <= q4ref.product_bound(xd[1:M - 1], w, ref, group, kind)).all()


def test_product_nan_scale(cuda, handle):
    """A weight group that held NaN makes its output NaN and no other."""
    torch = cuda
    N, K = 40, 256
    w = torch.randn(N, K, generator=torch.Generator().manual_seed(4))
    w[13, 200] = float("nan")
    packed = torch.empty(emugemm.q4_bytes(1, N, K, 64), dtype=torch.uint8, device="cuda")
    handle.q4_pack(1, N, K, w.cuda(), K, 64, packed)
    for M in (2, 100):
        c = torch.empty(M, N, device="cuda")
        handle.q4_gemm(M, N, K, torch.ones(M, K, device="cuda"), K, packed, 64, c, N)
        handle.sync()
        nan = c.isnan().cpu()
        assert nan[:, 13].all() and nan.sum() == M


def test_product_minus_eight(cuda, handle):
    """Weights quantised elsewhere may use q = -8."""
    torch = cuda
    N, K, group = 16, 64, 32
    g = np.random.default_rng(1)
    q = g.integers(-8, 8, (N, K)).astype(np.float64)
    s = np.full((N, 2), 0.5)
    packed = torch.from_numpy(q4ref.pack(q, s, 1, N, K, group)).cuda()
    check_product(torch, handle, 4, N, K, group, "bf16", packed=packed, w=q4ref.values(q, s, group))
    check_product(torch, handle, 200, N, K, group, "fp16", packed=packed, w=q4ref.values(q, s, group))


@pytest.mark.parametrize("kind", ["fp32", "bf16"])
@pytest.mark.parametrize("M", [1, 20, 140])
def test_product_repeats(cuda, handle, kind, M):
    torch = cuda
    c = [check_product(torch, handle, M, 500, 3000, 128, kind).clone() for _ in range(2)]
    assert torch.equal(c[0], c[1])


def test_product_zero_rows(cuda, handle):
    torch = cuda
    c = torch.full((1, 16), -7.5, device="cuda")
    handle.q4_gemm(0, 16, 64, c, 64, c, 32, c, 16)
    handle.sync()
    assert (c == -7.5).all()


# ----------------------------------------------------------------------------------------------------------- experts
def check_experts(torch, h, counts, N, K, group, kind, tail=0, seed=0):
    E = len(counts)
    off = np.concatenate([[0], np.cumsum(counts)]).astype(np.int32)
    used, R = int(off[-1]), int(off[-1]) + tail
    packed, w = q4ref.weights(seed + E, E, N, K, group)
    x = torch.randn(R, K, generator=torch.Generator().manual_seed(seed)).to(TYPES[kind])
    c = torch.full((R + 1, N), -7.5, dtype=TYPES[kind], device="cuda")
    h.q4_gemm_experts(R, E, N, K, x.cuda(), K, torch.from_numpy(off).cuda(), packed, group, c, N)
    h.sync()
    got, xd = c.double().cpu().numpy(), x.double().numpy()
    assert (got[used:] == -7.5).all(), "rows behind the last expert's were written"
    for e in range(E):
        a, b = off[e], off[e + 1]
        if a == b:
            continue
        ref = xd[a:b] @ w[e].T
        bad = np.abs(got[a:b] - ref) > q4ref.product_bound(xd[a:b], w[e], ref, group, kind)
        assert not bad.any(), (e, int(bad.sum()))


@pytest.mark.parametrize("kind", ["fp32", "fp16", "bf16"])
@pytest.mark.parametrize("counts,N,K,group,tail", [
    ([1], 33, 70, 32, 0), ([0, 0, 5, 0], 64, 256, 64, 3), ([3, 0, 1, 9, 0, 2], 100, 333, 128, 1),
    ([0, 40, 1, 130, 0, 7], 160, 520, 32, 5), ([0] * 63 + [4], 48, 128, 64, 0), ([300, 0, 1], 129, 192, 128, 2),
    ([64, 128, 256], 256, 256, 64, 0), ([1] * 40, 80, 1000, 128, 8)])
def test_experts(cuda, handle, kind, counts, N, K, group, tail):
    check_experts(cuda, handle, counts, N, K, group, kind, tail)


def test_experts_many_and_none(cuda, handle):
    """1024 experts with a few rows among them; and no row at all: nothing is written."""
    counts = [0] * 1024
    for i in (0, 31, 32, 500, 1023):
        counts[i] = 2
    check_experts(cuda, handle, counts, 32, 64, 32, "bf16", tail=4)
    check_experts(cuda, handle, [0, 0, 0], 32, 64, 32, "fp32", tail=6)
    check_experts(cuda, handle, [0, 0, 0], 32, 64, 32, "bf16", tail=300)


@pytest.mark.parametrize("R", [10, 400])
def test_experts_bad_offsets_stay_inside(cuda, handle, R):
    """Offsets outside 0 .. R or decreasing: no row outside the R rows of A is read (they are NaN there) and none
    outside the R rows of C is written."""
    torch = cuda
    E, N, K, group = 3, 32, 128, 64
    packed, w = q4ref.weights(1, E, N, K, group)
    a = torch.full((3 * R, K), float("nan"), dtype=torch.bfloat16, device="cuda")
    a[R:2 * R] = 1
    c = torch.full((3 * R, N), -7.5, dtype=torch.bfloat16, device="cuda")
    for off in ([-5, 3, R + 7, R + 9], [4, 2, 6, 1], [R + 1, R + 2, R + 3, R + 4], [0, 5, 3, R]):
        handle.q4_gemm_experts(R, E, N, K, a[R:], K, torch.tensor(off, dtype=torch.int32, device="cuda"), packed, group,
                               c[R:], N)
        handle.sync()
        assert (c[:R] == -7.5).all() and (c[2 * R:] == -7.5).all()
        assert not c[R:2 * R].isnan().any()


@pytest.mark.parametrize("N,K", [(32, 128), (264, 2048)])
def test_experts_extreme_offsets_stay_inside(cuda, handle, N, K):
    """Offsets at the ends of int32, whose differences wrap, and all rows claimed by every expert: nothing outside of C is
    written, and the next call of the handle is right."""
    torch = cuda
    lo, hi = -2 ** 31, 2 ** 31 - 1
    E, R, group = 5, 400, 64
    packed, w = q4ref.weights(1, E, N, K, group)
    a = torch.full((3 * R, K), float("nan"), dtype=torch.bfloat16, device="cuda")
    a[R:2 * R] = 1
    c = torch.full((3 * R, N), -7.5, dtype=torch.bfloat16, device="cuda")
    for off in ([hi, lo, hi, lo, hi, lo], [lo, hi, lo, hi, lo, hi], [0, R, 0, R, 0, R], [hi] * 6, [lo] * 6):
        handle.q4_gemm_experts(R, E, N, K, a[R:], K, torch.tensor(off, dtype=torch.int32, device="cuda"), packed, group,
                               c[R:], N)
        handle.sync()
        assert (c[:R] == -7.5).all() and (c[2 * R:] == -7.5).all()
        assert not c[R:2 * R].isnan().any()
    check_experts(torch, handle, [80] * 5, N, K, group, "bf16")


# -------------------------------------------------------------------------------- streams, graphs, handles, workspace
@pytest.mark.parametrize("M,kind", [(1, "bf16"), (40, "fp32"), (200, "fp32"), (200, "bf16")])
def test_capture_and_replay_with_new_inputs(cuda, M, kind):
    """A call captured into a graph and replayed on other contents of the same buffers, beside an eager call of the
    same handle at another size, gives the bits of the eager call."""
    torch = cuda
    N, K, group = 200, 515, 32
    packed, w = q4ref.weights(2, 1, N, K, group)
    xs = [torch.randn(M, K, generator=torch.Generator().manual_seed(i)).to(TYPES[kind]).cuda() for i in range(3)]
    a, c = xs[0].clone(), torch.empty(M, N, dtype=TYPES[kind], device="cuda")
    st = torch.cuda.Stream()
    with emugemm.Handle(st) as h, torch.cuda.stream(st):
        eager = []
        for x in xs:
            a.copy_(x)
            h.q4_gemm(M, N, K, a, K, packed, group, c, N)
            eager.append(c.clone())
        graph = torch.cuda.CUDAGraph()
        torch.cuda.synchronize()
        with torch.cuda.graph(graph, stream=st):
            h.q4_gemm(M, N, K, a, K, packed, group, c, N)
        # a larger eager call between capture and replay: the buffers that the graph uses stay
        big, wb = q4ref.weights(3, 1, 300, 1500, group)
        xb, cb = torch.ones(700, 1500, dtype=TYPES[kind], device="cuda"), torch.empty(700, 300, dtype=TYPES[kind], device="cuda")
        h.q4_gemm(700, 300, 1500, xb, 1500, big, group, cb, 300)
        for x, want in zip(xs, eager):
            a.copy_(x)
            c.fill_(-1)
            graph.replay()
            torch.cuda.synchronize()
            assert torch.equal(c, want)
        h.sync()
        del graph


@pytest.mark.parametrize("M", [1, 20, 100])
def test_first_call_of_a_process_inside_a_capture(cuda, M):
    """Nothing that a call does once per process or device is closed to a capture."""
    code = f"""
import torch, emugemm, q4ref
M, N, K, group = {M}, 520, 2048, 64
s = torch.cuda.Stream()
h = emugemm.Handle(s)
packed, w = q4ref.weights(3, 1, N, K, group)
x = torch.ones(M, K, dtype=torch.bfloat16, device="cuda")
y = torch.full((M, N), -7.5, dtype=torch.bfloat16, device="cuda")
torch.cuda.synchronize()
g = torch.cuda.CUDAGraph()
with torch.cuda.graph(g, stream=s):
    h.q4_gemm(M, N, K, x, K, packed, group, y, N)
assert (y == -7.5).all()
g.replay()
torch.cuda.synchronize()
h.sync()
xd = x.double().cpu().numpy()
ref = xd @ w[0].T
assert (abs(y.double().cpu().numpy() - ref) <= q4ref.product_bound(xd, w[0], ref, group, "bf16")).all()
print("right")
"""
    here = os.path.dirname(os.path.abspath(__file__))
    path = os.pathsep.join([here, os.path.dirname(os.path.abspath(emugemm.__file__)), os.environ.get("PYTHONPATH", "")])
    r = subprocess.run([sys.executable, "-c", code], env={**os.environ, "PYTHONPATH": path}, capture_output=True, text=True,
                       timeout=120)
    assert r.returncode == 0 and "right" in r.stdout, r.stderr[-2000:]


def test_capture_needs_the_workspace_first(cuda):
    """Many FP32 rows are staged in the workspace: captured on a handle that never ran the size, the call is refused, the
    capture stays valid and the handle usable."""
    torch = cuda
    M, N, K, group = 300, 64, 256, 64
    packed, w = q4ref.weights(5, 1, N, K, group)
    a, c = torch.randn(M, K, generator=torch.Generator().manual_seed(1)).cuda(), torch.zeros(M, N, device="cuda")
    st = torch.cuda.Stream()
    with emugemm.Handle(st) as h, torch.cuda.stream(st):
        torch.cuda.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=st):
            with pytest.raises(emugemm.EmuGemmError) as e:
                h.q4_gemm(M, N, K, a, K, packed, group, c, N)
            assert e.value.code == 5        # MEMORY_ERROR
            c.add_(1)
        graph.replay()
        torch.cuda.synchronize()
        assert (c == 1).all()
        h.q4_gemm(M, N, K, a, K, packed, group, c, N)
        h.sync()
        xd = a.double().cpu().numpy()
        ref = xd @ w[0].T
        assert (np.abs(c.double().cpu().numpy() - ref) <= q4ref.product_bound(xd, w[0], ref, group, "fp32")).all()
        del graph


def test_workspace_limit(cuda):
    torch = cuda
    packed, _ = q4ref.weights(5, 1, 32, 64, 32)
    a, c = torch.ones(200, 64, device="cuda"), torch.empty(200, 32, device="cuda")
    with emugemm.Handle() as h:
        h.set_workspace_limit(1024)
        with pytest.raises(emugemm.EmuGemmError) as e:
            h.q4_gemm(200, 32, 64, a, 64, packed, 32, c, 32)
        assert e.value.code == 5
        h.q4_gemm(2, 32, 64, a, 64, packed, 32, c, 32)     # few rows need none
        h.set_workspace_limit(0)
        h.q4_gemm(200, 32, 64, a, 64, packed, 32, c, 32)
        h.sync()


def test_two_handles_on_two_streams(cuda):
    """Two handles working at the same time on streams of their own do not disturb each other."""
    torch = cuda
    M, N, K, group = 300, 700, 2000, 128
    st = [torch.cuda.Stream() for _ in range(2)]
    hs = [emugemm.Handle(s) for s in st]
    data = [q4ref.weights(20 + i, 1, N, K, group) for i in range(2)]
    x = [torch.randn(M, K, generator=torch.Generator().manual_seed(i)).cuda() for i in range(2)]
    c = [torch.empty(M, N, device="cuda") for _ in range(2)]
    torch.cuda.synchronize()
    for _ in range(5):
        for i in range(2):
            hs[i].q4_gemm(M, N, K, x[i], K, data[i][0], group, c[i], N)
    for i in range(2):
        hs[i].sync()
        xd = x[i].double().cpu().numpy()
        ref = xd @ data[i][1][0].T
        assert (np.abs(c[i].double().cpu().numpy() - ref) <= q4ref.product_bound(xd, data[i][1][0], ref, group, "fp32")).all()
        hs[i].close()
