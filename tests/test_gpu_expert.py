"""Expert routing on the GPU, through the C ABI, against plain restatements; and a run of the operators together.

Bars: the sort and the gathered rows exact; sums over the choices in FP32 and one rounding (bounds at each test)."""
from __future__ import annotations

import numpy as np
import pytest

import emugemm
import q4ref
from q4ref import HALF_STEP, TINY, TYPES

pytestmark = pytest.mark.gpu


def make_ids(seed, T, topk, E, dropped=0.1):
    g = np.random.default_rng(seed)
    ids = g.integers(0, E, (T, topk)).astype(np.int32)
    ids[g.random((T, topk)) < dropped] = -1
    return ids


def run_sort(torch, h, ids, E):
    T, topk = ids.shape
    d = torch.from_numpy(ids).cuda()
    order, place = (torch.full((T * topk,), -99, dtype=torch.int32, device="cuda") for _ in range(2))
    offsets = torch.full((E + 2,), -99, dtype=torch.int32, device="cuda")
    h.expert_sort(T, topk, E, d, order, place, offsets)
    h.sync()
    assert offsets[E + 1].item() == -99
    return order, place, offsets[:E + 1]


@pytest.mark.parametrize("T,topk,E", [(1, 1, 1), (1, 8, 8), (31, 1, 3), (16, 2, 8), (33, 3, 64), (100, 7, 256), (1024, 8, 13),
                                      (1025, 8, 1024), (4096, 2, 33), (8193, 1, 1000), (8192, 4, 64), (30011, 5, 129),
                                      (200000, 6, 1024)])
def test_sort(cuda, handle, T, topk, E):
    ids = make_ids(T, T, topk, E)
    ids[0, 0] = E          # outside, as -1
    got = run_sort(cuda, handle, ids, E)
    for g, want in zip(got, q4ref.sort(ids, E)):
        assert np.array_equal(g.cpu().numpy(), want)


@pytest.mark.parametrize("fill", [-1, 0, 5, 7, 2 ** 31 - 1, -2 ** 31])
@pytest.mark.parametrize("T", [9, 9000])
def test_sort_one_expert_or_none(cuda, handle, fill, T):
    ids = np.full((T, 2), fill, np.int32)
    for g, want in zip(run_sort(cuda, handle, ids, 8), q4ref.sort(ids, 8)):
        assert np.array_equal(g.cpu().numpy(), want)


def test_sort_no_tokens(cuda, handle):
    torch = cuda
    offsets = torch.full((6,), -99, dtype=torch.int32, device="cuda")
    handle.expert_sort(0, 2, 5, None, None, None, offsets)
    handle.sync()
    assert offsets.tolist() == [0] * 6


ROWS = [(1, 1, 1, 1, 1), (16, 2, 8, 64, 64), (33, 3, 5, 1001, 1003), (7, 8, 64, 130, 136), (500, 5, 12, 96, 100),
        (129, 4, 1, 2048, 2048), (40, 1, 8, 7, 7)]


def case(torch, seed, T, topk, E, H, ld, kind):
    """Routing arrays on the GPU (and place on the host) and a maker of (rows x H) inputs inside rows of ld with NaN
    between them."""
    ids = make_ids(seed, T, topk, E)
    _, place, offsets = q4ref.sort(ids, E)
    place = place.reshape(T, topk)
    g = torch.Generator().manual_seed(seed)

    def rows(n, fill=float("nan")):
        x = torch.randn(n, H, generator=g).to(TYPES[kind])
        d = torch.full((n, ld), fill, dtype=TYPES[kind], device="cuda")
        d[:, :H] = x.cuda()
        return d, x.double().numpy()

    w = torch.randn(T, topk, generator=g)
    return place, torch.from_numpy(place).int().cuda(), rows, w


@pytest.mark.parametrize("kind", ["fp32", "fp16", "bf16"])
@pytest.mark.parametrize("T,topk,E,H,ld", ROWS)
def test_gather_and_its_gradient(cuda, handle, kind, T, topk, E, H, ld):
    torch = cuda
    place, dplace, rows, _ = case(torch, T + H, T, topk, E, H, ld, kind)
    S = T * topk
    x, xd = rows(T)
    xs = torch.full((S + 1, ld), -7.5, dtype=TYPES[kind], device="cuda")
    handle.expert_gather(T, topk, H, x, ld, dplace, xs, ld)
    handle.sync()
    want = np.full((S + 1, ld), -7.5)
    for t, j in np.argwhere(place >= 0):
        want[place[t, j], :H] = xd[t]
    assert np.array_equal(xs.double().cpu().numpy(), want)

    dxs, dd = rows(S)
    dx = torch.full((T + 1, ld), -7.5, dtype=TYPES[kind], device="cuda")
    handle.expert_gather_backward(T, topk, H, dxs, ld, dplace, dx, ld)
    handle.sync()
    ref, mag = np.zeros((T, H)), np.zeros((T, H))
    for t, j in np.argwhere(place >= 0):
        ref[t] += dd[place[t, j]]
        mag[t] += np.abs(dd[place[t, j]])
    got = dx.double().cpu().numpy()
    assert (got[T:] == -7.5).all() and (got[:, H:] == -7.5).all()
    # topk FP32 additions of half a step each, one rounding to the type
    assert (np.abs(got[:T, :H] - ref) <= HALF_STEP[kind] * np.abs(ref) + (topk + 1) * 2.0 ** -24 * mag + TINY[kind]).all()


@pytest.mark.parametrize("kind", ["fp32", "fp16", "bf16"])
@pytest.mark.parametrize("T,topk,E,H,ld", ROWS)
def test_combine_and_its_gradients(cuda, handle, kind, T, topk, E, H, ld):
    torch = cuda
    place, dplace, rows, w = case(torch, T * 3 + H, T, topk, E, H, ld, kind)
    S, wd, dw_ = T * topk, w.double().numpy(), w.cuda()
    ys, yd = rows(S)
    y = torch.full((T + 1, ld), -7.5, dtype=TYPES[kind], device="cuda")
    handle.expert_combine(T, topk, H, ys, ld, dplace, dw_, y, ld)
    dy, dd = rows(T)
    dys = torch.full((S + 1, ld), -7.5, dtype=TYPES[kind], device="cuda")
    dw = torch.full((T + 1, topk), -7.5, device="cuda")
    handle.expert_combine_backward(T, topk, H, dy, ld, ys, ld, dplace, dw_, dys, ld, dw)
    handle.sync()
    ref, mag = np.zeros((T, H)), np.zeros((T, H))
    rdys, rdw, mdw = np.full((S + 1, ld), -7.5), np.zeros((T, topk)), np.zeros((T, topk))
    for t, j in np.argwhere(place >= 0):
        r = place[t, j]
        ref[t] += wd[t, j] * yd[r]
        mag[t] += np.abs(wd[t, j] * yd[r])
        rdys[r, :H] = wd[t, j] * dd[t]
        rdw[t, j] = dd[t] @ yd[r]
        mdw[t, j] = np.abs(dd[t]) @ np.abs(yd[r])
    got = y.double().cpu().numpy()
    assert (got[T:] == -7.5).all() and (got[:, H:] == -7.5).all()
    assert (np.abs(got[:T, :H] - ref) <= HALF_STEP[kind] * np.abs(ref) + (topk + 1) * 2.0 ** -24 * mag + TINY[kind]).all()
    got = dys.double().cpu().numpy()
    half = HALF_STEP[kind] + 2.0 ** -24      # the FP32 product, then its rounding to the type
    assert (np.abs(got - rdys) <= half * np.abs(rdys) + TINY[kind]).all()
    assert (got[rdys == -7.5] == -7.5).all()
    got = dw.double().cpu().numpy()
    assert (got[T] == -7.5).all()
    # a sum of H products: at most H / 32 + 40 FP32 additions on the way of any of them
    assert (np.abs(got[:T] - rdw) <= (H / 32 + 40) * 2.0 ** -24 * mdw + 2.0 ** -149).all()
    assert (got[:T][place < 0] == 0).all()


def test_gradients_against_differences(cuda, handle):
    """Both movements are linear in their rows and the combination in its weights, so a central difference with any step
    is the derivative: <dY, f(x + v) - f(x - v)> / 2 = <gradient, v>, within FP32 rounding."""
    torch = cuda
    T, topk, E, H = 60, 3, 7, 129
    place, dplace, rows, w = case(torch, 1, T, topk, E, H, H, "fp32")
    S, w = T * topk, w.cuda()
    (x, _), (v, _), (ys, _), (u, _), (dy, _), (dxs, _) = (rows(n) for n in (T, T, S, S, T, S))
    dW = torch.randn(T, topk, generator=torch.Generator().manual_seed(8)).cuda()
    real = torch.zeros(S, 1, device="cuda", dtype=torch.float64)
    real[dplace[dplace >= 0].long()] = 1

    def gather(a):
        o = torch.zeros(S, H, device="cuda")
        handle.expert_gather(T, topk, H, a, H, dplace, o, H)
        return o.double()

    def combine(a, b):
        o = torch.empty(T, H, device="cuda")
        handle.expert_combine(T, topk, H, a, H, dplace, b, o, H)
        return o.double()

    def close(a, b, mag):
        assert abs(a - b) <= 1e-6 * mag, (a, b)     # a few roundings of 2^-24 of terms that add up to mag

    dx = torch.empty(T, H, device="cuda")
    handle.expert_gather_backward(T, topk, H, dxs, H, dplace, dx, H)
    num = ((gather(x + v) - gather(x - v)) * dxs.double() * real).sum().item() / 2
    close(num, (dx.double() * v.double()).sum().item(), (gather(v.abs() + x.abs()) * dxs.double().abs() * real).sum().item())

    dys, dw = torch.zeros(S, H, device="cuda"), torch.empty(T, topk, device="cuda")
    handle.expert_combine_backward(T, topk, H, dy, H, ys, H, dplace, w, dys, H, dw)
    num = ((combine(ys + u, w) - combine(ys - u, w)) * dy.double()).sum().item() / 2
    close(num, (dys.double() * u.double()).sum().item(), (combine(ys.abs() + u.abs(), w.abs()) * dy.double().abs()).sum().item())
    num = ((combine(ys, w + dW) - combine(ys, w - dW)) * dy.double()).sum().item() / 2
    close(num, (dw.double() * dW.double()).sum().item(),
          (combine(ys.abs(), w.abs() + dW.abs()) * dy.double().abs()).sum().item())


def test_bad_places_stay_inside(cuda, handle):
    """Places outside 0 .. T * topk - 1 are taken as no row."""
    torch = cuda
    T, topk, H = 4, 2, 32
    S = T * topk
    place = torch.tensor([[0, S], [-1, 1], [2 ** 31 - 1, 2], [-2 ** 31, 3]], dtype=torch.int32, device="cuda")
    x = torch.ones(T, H, device="cuda")
    buf = torch.full((3 * S, H), -7.5, device="cuda")
    handle.expert_gather(T, topk, H, x, H, place, buf[S:], H)
    handle.sync()
    assert (buf[:S] == -7.5).all() and (buf[2 * S:] == -7.5).all()
    assert (buf[S:S + 4] == 1).all() and (buf[S + 4:2 * S] == -7.5).all()
    y = torch.empty(T, H, device="cuda")
    handle.expert_combine(T, topk, H, buf[S:], H, place, torch.ones(T, topk, device="cuda"), y, H)
    handle.sync()
    assert (y == 1).all()
    dw = torch.empty(T, topk, device="cuda")
    handle.expert_combine_backward(T, topk, H, x, H, x.repeat(2, 1), H, place, torch.ones(T, topk, device="cuda"), buf[S:], H, dw)
    handle.sync()
    assert (buf[:S] == -7.5).all() and (buf[2 * S:] == -7.5).all()
    assert dw.cpu().tolist() == [[H, 0], [0, H], [0, H], [0, H]]


def test_rows_beyond_32_bit_offsets(cuda, handle):
    """Sorted rows of more than 2^32 bytes: the last row is moved and read back at 64-bit offsets."""
    torch = cuda
    T, topk, H = 70000, 2, 16384                     # 140000 rows of 32 KB
    place = torch.arange(T * topk, dtype=torch.int32, device="cuda").view(T, topk)
    x = torch.zeros(T, H, dtype=torch.bfloat16, device="cuda")
    x[-1] = torch.arange(H, device="cuda") % 128
    xs = torch.full((T * topk, H), -1, dtype=torch.bfloat16, device="cuda")
    handle.expert_gather(T, topk, H, x, H, place, xs, H)
    y = torch.empty(T, H, dtype=torch.bfloat16, device="cuda")
    handle.expert_combine(T, topk, H, xs, H, place, torch.ones(T, topk, device="cuda"), y, H)
    handle.sync()
    assert torch.equal(xs[-1], x[-1]) and torch.equal(xs[-2], x[-1]) and (xs[:-2] == 0).all()
    assert torch.equal(y, 2 * x)


# ------------------------------------------------------------------------------------------------------- runs together
@pytest.mark.parametrize("T,kind", [(1, "bf16"), (5, "fp16"), (300, "fp32"), (1000, "bf16")])
def test_expert_layer(cuda, handle, T, kind):
    """A layer of 4-bit experts as a server runs it: pack, sort, gather, up, SiLU, down, combine; against FP64 with the
    same weights and the intermediate roundings of the type put in."""
    torch = cuda
    topk, E, H, F, group = 2, 6, 192, 264, 64
    g = torch.Generator().manual_seed(T)
    w1 = torch.randn(E, F, H, generator=g) * 0.05
    w2 = torch.randn(E, H, F, generator=g) * 0.05
    x = torch.randn(T, H, generator=g).to(TYPES[kind])
    ids = torch.rand(T, E, generator=g).topk(topk, 1).indices.int()
    if T > 10:
        ids[-3:] = -1
    wt = torch.rand(T, topk, generator=g)
    p1, p2 = (torch.empty(emugemm.q4_bytes(E, w.shape[1], w.shape[2], group), dtype=torch.uint8, device="cuda") for w in (w1, w2))
    handle.q4_pack(E, F, H, w1.cuda(), H, group, p1)
    handle.q4_pack(E, H, F, w2.cuda(), F, group, p2)
    S, t = T * topk, TYPES[kind]
    order, offsets = torch.empty(S, dtype=torch.int32, device="cuda"), torch.empty(E + 1, dtype=torch.int32, device="cuda")
    place = torch.empty(T, topk, dtype=torch.int32, device="cuda")
    xs, up, out = (torch.zeros(S, n, dtype=t, device="cuda") for n in (H, F, H))
    y = torch.empty(T, H, dtype=t, device="cuda")
    handle.expert_sort(T, topk, E, ids.cuda(), order, place, offsets)
    handle.expert_gather(T, topk, H, x.cuda(), H, place, xs, H)
    handle.q4_gemm_experts(S, E, F, H, xs, H, offsets, p1, group, up, F)
    act = torch.nn.functional.silu(up.float()).to(t)
    handle.q4_gemm_experts(S, E, H, F, act, F, offsets, p2, group, out, H)
    handle.expert_combine(T, topk, H, out, H, place, wt.cuda(), y, H)
    handle.sync()
    v1, v2 = (q4ref.values(*q4ref.quantise(w.reshape(-1, w.shape[2]).numpy(), group), group).reshape(w.shape) for w in (w1, w2))
    ref, mag = np.zeros((T, H)), np.zeros((T, H))
    step = 2 * HALF_STEP[kind] + 2.0 ** -18     # a product's rounding, and its FP32 sum over at most 264 values
    for i in range(T):
        for j in range(topk):
            e = int(ids[i, j])
            if e < 0:
                continue
            u = v1[e] @ x[i].double().numpy()
            a = u / (1 + np.exp(-u))
            du = step * (np.abs(v1[e]) @ np.abs(x[i].double().numpy()) * 2.0 ** -3 + np.abs(u))
            da = 1.1 * du + step * np.abs(a)    # |SiLU'| is at most 1.1
            o = v2[e] @ a
            ref[i] += float(wt[i, j]) * o
            mag[i] += float(wt[i, j]) * (np.abs(v2[e]) @ da + step * (np.abs(v2[e]) @ np.abs(a) * 2.0 ** -3 + np.abs(o)))
    assert (np.abs(y.double().cpu().numpy() - ref) <= mag + step * np.abs(ref) + 1e-7).all()


def test_training_step_with_fp32_experts(cuda, handle):
    """Sort, gather, emugemm_sgemm of every expert's rows (native FP32), combine, and the gradients back to the tokens
    and the combination weights, against torch's autograd in FP64 on the same routing."""
    torch = cuda
    T, topk, E, H, F = 90, 2, 4, 64, 48
    g = torch.Generator().manual_seed(3)
    x, w = torch.randn(T, H, generator=g).cuda(), torch.randn(E, H, F, generator=g).cuda()
    ids = torch.rand(T, E, generator=g).topk(topk, 1).indices.int()
    ids[-2:] = -1
    wt, dy = torch.rand(T, topk, generator=g).cuda(), torch.randn(T, F, generator=g).cuda()
    S = T * topk
    i32 = dict(dtype=torch.int32, device="cuda")
    order, place, offsets = torch.empty(S, **i32), torch.empty(T, topk, **i32), torch.empty(E + 1, **i32)
    xs, ys, dys, dxs = (torch.zeros(S, n, device="cuda") for n in (H, F, F, H))
    y, dw, dx = torch.empty(T, F, device="cuda"), torch.empty(T, topk, device="cuda"), torch.empty(T, H, device="cuda")
    h = handle
    h.expert_sort(T, topk, E, ids.cuda(), order, place, offsets)
    h.expert_gather(T, topk, H, x, H, place, xs, H)
    off = offsets.tolist()
    for e in range(E):
        a, b = off[e], off[e + 1]
        h.sgemm(b - a, F, H, xs[a:b], w[e], ys[a:b], force=emugemm.NATIVE_FP32)
    h.expert_combine(T, topk, F, ys, F, place, wt, y, F)
    h.expert_combine_backward(T, topk, F, dy, F, ys, F, place, wt, dys, F, dw)
    for e in range(E):
        a, b = off[e], off[e + 1]
        h.sgemm(b - a, H, F, dys[a:b], w[e].t().contiguous(), dxs[a:b], force=emugemm.NATIVE_FP32)
    h.expert_gather_backward(T, topk, H, dxs, H, place, dx, H)
    h.sync()
    xd, wd = x.double().requires_grad_(), wt.double().requires_grad_()
    each = torch.einsum("th,ehf->tef", xd, w.double())
    pick = ids.clamp(min=0).long().cuda()
    on = (ids >= 0).double().cuda()
    ref = (torch.gather(each, 1, pick[..., None].expand(-1, -1, F)) * (wd * on)[..., None]).sum(1)
    ref.backward(dy.double())
    # sums of at most 64 + 48 + 2 FP32 terms around 1: relative to the largest value, 200 roundings of 2^-24
    for got, want in ((y, ref.detach()), (dw, wd.grad), (dx, xd.grad)):
        assert (got.double() - want).abs().max() <= 200 * 2.0 ** -24 * want.abs().max()
    assert (y[-2:] == 0).all() and (dx[-2:] == 0).all() and (dw[-2:] == 0).all()


def test_routing_captured_and_replayed(cuda):
    """Sort, gather, experts' products and combine captured once and replayed for other ids and tokens."""
    torch = cuda
    T, topk, E, H, N, group = 50, 2, 9, 96, 80, 32
    packed, w = q4ref.weights(2, E, N, H, group)
    S = T * topk
    i32 = dict(dtype=torch.int32, device="cuda")
    ids, order, place, offsets = (torch.zeros(T, topk, **i32), torch.empty(S, **i32), torch.empty(T, topk, **i32),
                                  torch.empty(E + 1, **i32))
    x, xs, ys, y = (torch.zeros(n, m, device="cuda") for n, m in ((T, H), (S, H), (S, N), (T, N)))
    wt = torch.rand(T, topk, device="cuda")
    st = torch.cuda.Stream()
    with emugemm.Handle(st) as h, torch.cuda.stream(st):
        def step():
            h.expert_sort(T, topk, E, ids, order, place, offsets)
            h.expert_gather(T, topk, H, x, H, place, xs, H)
            h.q4_gemm_experts(S, E, N, H, xs, H, offsets, packed, group, ys, N)
            h.expert_combine(T, topk, N, ys, N, place, wt, y, N)

        step()
        torch.cuda.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=st):
            step()
        for seed in range(3):
            new = make_ids(seed, T, topk, E)
            ids.copy_(torch.from_numpy(new))
            x.copy_(torch.randn(T, H, generator=torch.Generator().manual_seed(seed)))
            step()
            want = y.clone()
            y.fill_(-1)
            graph.replay()
            torch.cuda.synchronize()
            assert torch.equal(y, want)
            _, p, _ = q4ref.sort(new, E)
            assert np.array_equal(place.cpu().numpy().reshape(-1), p)
        del graph


def test_profile_kinds(cuda, handle):
    torch = cuda
    handle.profile_begin()
    offsets = torch.empty(4, dtype=torch.int32, device="cuda")
    handle.expert_sort(0, 1, 3, None, None, None, offsets)
    packed, _ = q4ref.weights(1, 1, 16, 64, 32)
    a, c = torch.ones(2, 64, device="cuda"), torch.empty(2, 16, device="cuda")
    handle.q4_gemm(2, 16, 64, a, 64, packed, 32, c, 16)
    p = handle.profile_end()
    assert p["expert"][1] == 1 and p["q4"][1] == 1 and p["tc_gemm"][1] == 0
