"""4-bit products on the GPU, what the other files leave of their range: workspaces that captured graphs keep, row tiles of
both heights with more tiles than CTA pairs, the low bits of FP32 rows, rows that are not there, the choice between the
kernels, captures without an earlier run, and the calls after a failed one.

Bars: q4ref.product_bound, or derived at the test."""
from __future__ import annotations

import functools
import os
import subprocess
import sys

import numpy as np
import pytest

import emugemm
import q4ref
from q4ref import TYPES

pytestmark = pytest.mark.gpu


# --------------------------------------------------------------------------------------------------------- workspace
def test_refused_growth_keeps_what_a_graph_uses(cuda):
    """A larger call that the workspace limit refuses takes nothing from the handle: the size that a captured graph uses
    still runs, can be captured again and is replayed."""
    torch = cuda
    M, N, K, group = 300, 64, 256, 64
    packed, w = q4ref.weights(5, 1, N, K, group)
    a = torch.randn(M, K, generator=torch.Generator().manual_seed(1)).cuda()
    c, c2 = torch.empty(M, N, device="cuda"), torch.empty(M, N, device="cuda")
    big, cbig = torch.ones(400, K, device="cuda"), torch.empty(400, N, device="cuda")
    st = torch.cuda.Stream()
    with emugemm.Handle(st) as h, torch.cuda.stream(st):
        h.q4_gemm(M, N, K, a, K, packed, group, c, N)      # 6 bytes for each of 300 x 256 values: 460800
        want = c.clone()
        torch.cuda.synchronize()
        graphs = [torch.cuda.CUDAGraph() for _ in range(2)]
        with torch.cuda.graph(graphs[0], stream=st):
            h.q4_gemm(M, N, K, a, K, packed, group, c, N)
        h.set_workspace_limit(700000)
        for _ in range(2):
            with pytest.raises(emugemm.EmuGemmError) as e:
                h.q4_gemm(400, N, K, big, K, packed, group, cbig, N)     # 614400 more beside the kept 460800
            assert e.value.code == 5
            c2.zero_()
            h.q4_gemm(M, N, K, a, K, packed, group, c2, N)
            torch.cuda.synchronize()
            assert torch.equal(c2, want)
        with torch.cuda.graph(graphs[1], stream=st):
            h.q4_gemm(M, N, K, a, K, packed, group, c2, N)
        for g, out in zip(graphs, (c, c2)):
            out.zero_()
            g.replay()
            torch.cuda.synchronize()
            assert torch.equal(out, want)
        h.set_workspace_limit(0)
        h.q4_gemm(400, N, K, big, K, packed, group, cbig, N)
        c.zero_()
        graphs[0].replay()
        h.sync()
        assert torch.equal(c, want)
        del graphs, g


# ------------------------------------------------------------------------------------------- row tiles of both heights
def tile_rows(torch, R, N, experts=0):
    """(rows of A per tile, tiles) by the launch's rule for products of many rows whose K is not split: rounds of the CTA
    pairs, 1.3 times as long for 256 rows. With experts one tile more for each, which the host cannot rule out."""
    pairs = torch.cuda.get_device_properties(0).multi_processor_count // 2
    tiles = {h: (experts + -(-R // h)) * -(-N // 256) for h in (128, 256)}
    rounds = {h: -(-tiles[h] // pairs) for h in tiles}
    return (256, tiles[256]) if 1.3 * rounds[256] <= rounds[128] else (128, tiles[128])


@functools.lru_cache(maxsize=None)
def layer(E, N, K, group):
    return q4ref.weights(E * N + K, E, N, K, group)


def close(got, x, w, group, kind):
    ref = x @ w.T
    bad = ~(np.abs(got - ref) <= q4ref.product_bound(x, w, ref, group, kind))     # NaN is bad, too
    assert not bad.any(), (int(bad.sum()), np.argwhere(bad)[:4], np.nanmax(np.abs(got - ref)))


# One tile per pair and several; K of one panel, of odd counts, and of more panels than the shared memory has stages
MANY = [(2100, 1200, 200, 256, False), (2400, 1999, 1100, 256, True), (2560, 2048, 64, 256, True), (100, 19300, 330, 128, True),
        (5000, 4000, 70, 256, True)]


@pytest.mark.parametrize("kind", ["fp32", "fp16", "bf16"])
@pytest.mark.parametrize("group", [32, 64, 128])
@pytest.mark.parametrize("M,N,K,height,several", MANY)
def test_product_of_many_tiles(cuda, handle, kind, group, M, N, K, height, several):
    torch = cuda
    rows, tiles = tile_rows(torch, M, N)
    pairs = torch.cuda.get_device_properties(0).multi_processor_count // 2
    assert rows == height and (tiles > pairs) == several        # the case is what it stands for
    packed, w = layer(1, N, K, group)
    x = torch.randn(M, K, generator=torch.Generator().manual_seed(M)).to(TYPES[kind])
    c = torch.full((M + 1, N), -7.5, dtype=TYPES[kind], device="cuda")
    handle.q4_gemm(M, N, K, x.cuda(), K, packed, group, c, N)
    handle.sync()
    got = c.double().cpu().numpy()
    assert (got[M] == -7.5).all()
    close(got[:M], x.double().numpy(), w[0], group, kind)
    c2 = torch.empty_like(c)
    handle.q4_gemm(M, N, K, x.cuda(), K, packed, group, c2, N)
    handle.sync()
    assert torch.equal(c[:M], c2[:M])


EXPERTS = [([700, 0, 1300, 3, 256, 257, 0], 1500, 333, 5, 256), ([300, 1, 90, 0, 250, 130], 2600, 200, 0, 128),
           ([0, 2560, 0], 2048, 130, 40, 256)]


@pytest.mark.parametrize("kind", ["fp32", "fp16", "bf16"])
@pytest.mark.parametrize("group", [32, 64, 128])
@pytest.mark.parametrize("counts,N,K,tail,height", EXPERTS)
def test_experts_of_many_tiles(cuda, handle, kind, group, counts, N, K, tail, height):
    torch = cuda
    E, off = len(counts), np.concatenate([[0], np.cumsum(counts)]).astype(np.int32)
    used, R = int(off[-1]), int(off[-1]) + tail
    assert tile_rows(torch, R, N, E)[0] == height
    pairs = torch.cuda.get_device_properties(0).multi_processor_count // 2
    assert sum(-(-n // height) for n in counts) * -(-N // 256) > pairs      # a pair takes more than one tile
    packed, w = layer(E, N, K, group)
    x = torch.randn(R, K, generator=torch.Generator().manual_seed(R)).to(TYPES[kind])
    c = torch.full((R + 1, N), -7.5, dtype=TYPES[kind], device="cuda")
    handle.q4_gemm_experts(R, E, N, K, x.cuda(), K, torch.from_numpy(off).cuda(), packed, group, c, N)
    handle.sync()
    got, xd = c.double().cpu().numpy(), x.double().numpy()
    assert (got[used:] == -7.5).all()
    for e in range(E):
        if counts[e]:
            close(got[off[e]:off[e + 1]], xd[off[e]:off[e + 1]], w[e], group, kind)


# ------------------------------------------------------------------------------------------------ 24 bits of FP32 rows
def one_value_rows(rows, K, seed):
    """Rows of zeros with one value each, whose 24 significant bits end in a byte of 64 or more: without the lowest slice
    it is off by at least 2^-18 of itself. The places k run over all of K."""
    g = np.random.default_rng(seed)
    k = (g.permutation(rows) * K // rows + g.integers(0, max(1, K // rows), rows)).clip(max=K - 1)
    m = (g.integers(2 ** 15, 2 ** 16, rows) * 256 + g.integers(64, 256, rows)).astype(np.float64)
    x = np.zeros((rows, K), np.float32)
    x[np.arange(rows), k] = m * 2.0 ** (g.integers(-3, 4, rows) - 23) * g.choice([-1, 1], rows)
    return x


def check_low_bits(got, x, w):
    """C is scale * q * x of one place, the rest adds zeros: the sum of the three slices' products loses at most one step
    of 2^-23 in the tensor cores, which truncate, and each of the multiplication by the scale and the two additions of
    slices kept apart rounds by 2^-24 at most (a kernel does one or the other)."""
    ref = x.astype(np.float64) @ w.T
    bad = ~(np.abs(got - ref) <= 3 * 2.0 ** -24 * np.abs(ref))
    assert not bad.any(), (int(bad.sum()), np.argwhere(bad)[:4], np.nanmax(np.abs(got - ref) / np.abs(ref)))


# The column tiles of few rows, K splits over pairs, and row tiles of 128 and 256; K with a last group that is not whole
LOW = [(1, 40, 2052), (1, 700, 4096), (2, 300, 1300), (4, 130, 1028), (8, 260, 1500), (10, 100, 2052), (16, 300, 1100),
       (60, 130, 1036), (100, 300, 2200), (128, 520, 4100), (400, 640, 1088), (2100, 1200, 200), (2400, 1999, 260)]


@pytest.mark.parametrize("group", [32, 64, 128])
@pytest.mark.parametrize("M,N,K", LOW)
@pytest.mark.parametrize("gap", [0, 1])
def test_product_keeps_the_low_bits(cuda, handle, group, M, N, K, gap):
    """gap: a leading dimension that breaks the rows' alignment."""
    torch = cuda
    packed, w = layer(1, N, K, group)
    for seed in range(max(1, 24 // M)):
        x = one_value_rows(M, K, 100 * seed + M) if M > 1 else one_value_rows(24, K, M)[seed:seed + 1]
        a = torch.full((M, K + gap), float("nan"), device="cuda")
        a[:, :K] = torch.from_numpy(x).cuda()
        c = torch.empty(M, N, device="cuda")
        handle.q4_gemm(M, N, K, a, K + gap, packed, group, c, N)
        handle.sync()
        check_low_bits(c.double().cpu().numpy(), x, w[0])


@pytest.mark.parametrize("group", [32, 64, 128])
@pytest.mark.parametrize("counts,N,K", [([3, 0, 1, 9, 0, 2], 100, 332), ([40, 1, 0, 130], 160, 1052), ([60, 70, 0, 90], 200, 2100),
                                        ([700, 0, 1300, 3, 256, 257, 0], 1500, 332)])
def test_experts_keep_the_low_bits(cuda, handle, group, counts, N, K):
    torch = cuda
    E, off = len(counts), np.concatenate([[0], np.cumsum(counts)]).astype(np.int32)
    R = int(off[-1])
    packed, w = layer(E, N, K, group)
    x = one_value_rows(R, K, R)
    c = torch.empty(R, N, device="cuda")
    handle.q4_gemm_experts(R, E, N, K, torch.from_numpy(x).cuda(), K, torch.from_numpy(off).cuda(), packed, group, c, N)
    handle.sync()
    got = c.double().cpu().numpy()
    for e in range(E):
        if counts[e]:
            check_low_bits(got[off[e]:off[e + 1]], x[off[e]:off[e + 1]], w[e])


# ------------------------------------------------------------------------------------------------------ rows not there
def test_work_follows_the_rows_that_are_there(cuda):
    """FP32 rows are staged before the product: 64 rows that are there among 262144 are done in a small part of the time of
    all of them (staging all R takes more than half of it, so a quarter tells the two apart)."""
    torch = cuda
    E, R, N, K, group = 4, 1 << 18, 16, 1024, 64
    packed, w = layer(E, N, K, group)
    a = torch.randn(R, K, device="cuda")
    c = torch.full((R, N), -7.5, device="cuda")
    few, every = ([n * i for i in range(E + 1)] for n in (16, R // E))
    off = {n: torch.tensor(o, dtype=torch.int32, device="cuda") for n, o in (("few", few), ("all", every))}
    ms = {}
    with emugemm.Handle() as h:
        for name in ("few", "all"):
            for _ in range(4):
                h.profile_begin()
                h.q4_gemm_experts(R, E, N, K, a, K, off[name], packed, group, c, N)
                ms[name] = min(ms.get(name, 1e9), h.profile_end()["q4"][0])
            if name == "few":
                assert (c[64:] == -7.5).all()
                got, x = c[:64].double().cpu().numpy(), a[:64].double().cpu().numpy()
                for e in range(E):
                    close(got[16 * e:16 * e + 16], x[16 * e:16 * e + 16], w[e], group, "fp32")
    assert ms["few"] < ms["all"] / 4, ms


def test_backward_offsets_stage_what_is_claimed(cuda, handle):
    """Offsets that run backwards: the rows of the experts that do have rows are right, whatever the last offset says."""
    torch = cuda
    E, R, N, K, group = 4, 300, 40, 132, 32
    packed, w = layer(E, N, K, group)
    a = torch.randn(R, K, generator=torch.Generator().manual_seed(1)).cuda()
    c = torch.full((R, N), -7.5, device="cuda")
    off = torch.tensor([0, 120, 260, 250, 3], dtype=torch.int32, device="cuda")      # experts 0 and 1; 2 and 3 have none
    handle.q4_gemm_experts(R, E, N, K, a, K, off, packed, group, c, N)
    handle.sync()
    got, x = c.double().cpu().numpy(), a.double().cpu().numpy()
    close(got[:120], x[:120], w[0], group, "fp32")
    close(got[120:260], x[120:260], w[1], group, "fp32")
    assert (got[260:] == -7.5).all()


# ------------------------------------------------------------------------------------------------------ rows or tiles
@pytest.mark.parametrize("E,launches", [(4, 1), (16, 2)])
def test_many_experts_go_to_tiles(cuda, handle, E, launches):
    """Groups of 32 with a mean of 60 rows: of more than 8 experts, which are seldom even, on row tiles, where unaligned rows
    are staged first (two launches); of few experts in passes of 48 columns (one)."""
    torch = cuda
    N, K, group = (1 << 24) // (1024 * E) + 8, 1025, 32
    R = 60 * E
    w = torch.randn(E * N, K, generator=torch.Generator().manual_seed(E)).bfloat16().cuda()
    packed = torch.empty(emugemm.q4_bytes(E, N, K, group), dtype=torch.uint8, device="cuda")
    handle.q4_pack(E, N, K, w, K, group, packed)
    off = torch.arange(0, R + 1, 60, dtype=torch.int32, device="cuda")
    x = torch.randn(R, K, generator=torch.Generator().manual_seed(2)).bfloat16().cuda()
    c = torch.empty(R, N, dtype=torch.bfloat16, device="cuda")
    before = emugemm.lib().emugemm_kernel_launch_count()
    handle.q4_gemm_experts(R, E, N, K, x, K, off, packed, group, c, N)
    assert emugemm.lib().emugemm_kernel_launch_count() - before == launches
    out = torch.empty(E * N, K, device="cuda")
    handle.q4_unpack(E, N, K, group, packed, out, K)
    handle.sync()
    v, xd = out.view(E, N, K).double().cpu().numpy(), x.double().cpu().numpy()
    for e in (0, E - 1):
        close(c[60 * e:60 * e + 60].double().cpu().numpy(), xd[60 * e:60 * e + 60], v[e], group, "bf16")


# -------------------------------------------------------------------------------------------------- after a failed call
def test_a_failed_launch_is_reported_once(cuda):
    """A call into a capture that has become invalid fails; the calls after the capture has ended are not blamed for it.
    (A process of its own: torch does not get over a broken capture.)"""
    code = """
import os, torch, emugemm, q4ref
M, N, K, group = 4, 520, 2048, 64
s = torch.cuda.Stream()
h = emugemm.Handle(s)
packed, w = q4ref.weights(3, 1, N, K, group)
x = torch.ones(M, K, dtype=torch.bfloat16, device="cuda")
y = torch.zeros(M, N, dtype=torch.bfloat16, device="cuda")
def one():
    h.q4_gemm(M, N, K, x, K, packed, group, y, N)
one()
torch.cuda.synchronize()
g = torch.cuda.CUDAGraph()
failed = 0
with torch.cuda.stream(s):
    g.capture_begin()
    try:
        torch.cuda.synchronize()          # not allowed in a capture: it makes the capture invalid
    except RuntimeError:
        failed += 1
    try:
        one()
    except emugemm.EmuGemmError:
        failed += 1
    try:
        g.capture_end()
    except RuntimeError:
        failed += 1
assert failed == 3, failed
y.zero_()
torch.cuda.synchronize()
one()                                          # raised what the capture's call had already reported
h.sync()
xd = x.double().cpu().numpy()
ref = xd @ w[0].T
assert (abs(y.double().cpu().numpy() - ref) <= q4ref.product_bound(xd, w[0], ref, group, "bf16")).all()
print("right", flush=True)
os._exit(0)
"""
    here = os.path.dirname(os.path.abspath(__file__))
    path = os.pathsep.join([here, os.path.dirname(os.path.abspath(emugemm.__file__)), os.environ.get("PYTHONPATH", "")])
    r = subprocess.run([sys.executable, "-c", code], env={**os.environ, "PYTHONPATH": path}, capture_output=True, text=True,
                       timeout=120)
    assert r.returncode == 0 and "right" in r.stdout, r.stderr[-2000:]


# ------------------------------------------------------------------------------------------- what needs no earlier run
@pytest.mark.parametrize("group", [32, 64, 128])
@pytest.mark.parametrize("kind,rows,many", [("bf16", 32, 100), ("fp16", 32, 100), ("fp32", 16, 40)])
@pytest.mark.parametrize("E", [1, 3])
def test_captures_within_the_documented_limit(cuda, group, kind, rows, many, E):
    """Unaligned rows, a first call of the handle inside a capture: up to 32 rows (16 in FP32), of experts on the average, it
    is captured and replays to the bits of an eager call; more rows are refused and can be captured after one call of the size."""
    torch = cuda
    N, K = 4096 // E, 8195
    packed = torch.randint(0, 256, (emugemm.q4_bytes(E, N, K, group),), dtype=torch.uint8, device="cuda")
    codes = E * -(-N // 16) * -(-K // 64) * 512
    at = -(-codes // 256) * 256
    packed[at:] = torch.full(((packed.numel() - at) // 2,), 0.01, dtype=torch.bfloat16, device="cuda").view(torch.uint8)
    st = torch.cuda.Stream()
    with emugemm.Handle(st) as h, torch.cuda.stream(st):
        for per, fits in ((rows, True), (many, False)):
            R = per * E + (E - 1 if fits else 0)
            a = torch.randn(R, K, generator=torch.Generator().manual_seed(R)).to(TYPES[kind]).cuda()
            off = torch.arange(0, (per + 1) * E, per, dtype=torch.int32, device="cuda")
            off[E] = R
            c = torch.zeros(R, N, dtype=TYPES[kind], device="cuda")

            def call():
                if E == 1:
                    h.q4_gemm(R, N, K, a, K, packed, group, c, N)
                else:
                    h.q4_gemm_experts(R, E, N, K, a, K, off, packed, group, c, N)

            torch.cuda.synchronize()
            if not fits:
                graph = torch.cuda.CUDAGraph()
                with torch.cuda.graph(graph, stream=st):
                    with pytest.raises(emugemm.EmuGemmError) as e:
                        call()
                    assert e.value.code == 5        # MEMORY_ERROR
                    c.add_(1)
                call()
                torch.cuda.synchronize()
            graph = torch.cuda.CUDAGraph()
            with torch.cuda.graph(graph, stream=st):
                call()
            c.zero_()
            graph.replay()
            torch.cuda.synchronize()
            got = c.clone()
            c.zero_()
            call()
            h.sync()
            assert torch.equal(got, c) and c.abs().sum() > 0
            del graph
