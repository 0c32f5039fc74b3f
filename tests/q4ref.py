"""Plain 64-bit restatement of the packed 4-bit weights and of the expert routing, used by the tests."""
from __future__ import annotations

import numpy as np
import torch

TYPES = {"fp32": torch.float32, "fp16": torch.float16, "bf16": torch.bfloat16}
# half a step of a type relative to the value, and its smallest positive step
HALF_STEP = {"fp32": 2.0 ** -24, "fp16": 2.0 ** -11, "bf16": 2.0 ** -8}
TINY = {"fp32": 2.0 ** -149, "fp16": 2.0 ** -24, "bf16": 2.0 ** -133}


def quantise(w: np.ndarray, group: int):
    """(q, s) of w (rows x K): integer codes and float64 scales, one scale per group (the last may be short)."""
    w = np.asarray(w, np.float64)
    rows, K = w.shape
    G = -(-K // group)
    q, s = np.zeros((rows, K)), np.zeros((rows, G))
    for g in range(G):
        v = w[:, g * group:(g + 1) * group]
        m = np.abs(v).max(1)
        bad = ~np.isfinite(m)
        sg = torch.from_numpy(np.where(bad, 0, m) / 7.0).float().bfloat16().double().numpy()
        safe = np.where(sg > 0, sg, 1.0)[:, None]
        c = np.clip(np.rint(np.where(bad[:, None], 0, v) / safe), -7, 7)
        q[:, g * group:(g + 1) * group] = np.where((sg > 0)[:, None], c, 0)
        s[:, g] = np.where(bad, np.nan, sg)
    return q, s


def values(q, s, group):
    return q * np.repeat(s, group, 1)[:, :q.shape[1]]


def pack(q, s, E, N, K, group) -> np.ndarray:
    """The packed bytes, written value by value from the layout's description."""
    nb, kb, G = -(-N // 16), -(-K // 64), -(-K // group)
    codes = np.full((E, nb, kb, 8, 4, 4), 0x88888888, np.uint32)     # [g][t][word]
    scales = np.zeros((E, nb, G, 8, 2), np.uint16)
    nib = [0, 4, 1, 5, 2, 6, 3, 7]                                   # nibble of k % 8
    e, n, k = np.meshgrid(np.arange(E), np.arange(N), np.arange(K), indexing="ij")
    r, kk = n % 16, k % 64
    word = (kk // 32) * 2 + r // 8
    shift = 4 * np.array(nib)[kk % 8]
    idx = (e, n // 16, k // 64, r % 8, kk % 32 // 8, word)
    c = (q.reshape(E, N, K) + 8).astype(np.uint32)
    np.bitwise_xor.at(codes, idx, ((c ^ 8) << shift.astype(np.uint32)).astype(np.uint32))
    bits = torch.from_numpy(s).bfloat16().view(torch.int16).numpy().view(np.uint16).reshape(E, N, G)
    bits = np.where(np.isnan(s.reshape(E, N, G)), np.uint16(0x7FC0), bits)   # the library's NaN (torch's has any payload)
    ee, nn, gg = np.meshgrid(np.arange(E), np.arange(N), np.arange(G), indexing="ij")
    scales[ee, nn // 16, gg, nn % 8, nn % 16 // 8] = bits
    raw = codes.reshape(-1).view(np.uint8)
    at = -(-raw.size // 256) * 256
    out = np.zeros(at + scales.size * 2, np.uint8)
    out[:raw.size] = raw
    out[at:] = scales.reshape(-1).view(np.uint8)
    return out


def weights(seed, E, N, K, group, scale=0.02):
    """Random packed weights on the GPU and their float64 values (E, N, K)."""
    g = np.random.default_rng(seed)
    w = (g.standard_normal((E * N, K)) * scale).astype(np.float32)
    q, s = quantise(w, group)
    return torch.from_numpy(pack(q, s, E, N, K, group)).cuda(), values(q, s, group).reshape(E, N, K)


def product_bound(x, w, y, group, kind):
    """Largest |C - y| of C = x w^T (float64 y): the output's rounding; the products of a group of 16-value steps added
    by the tensor cores, each step losing at most 2^-21 of the magnitudes it adds; one FP32 rounding of 2^-24 for each
    group's scale and addition and up to 64 partial sums (24 of them for slices, warps and CTAs)."""
    K = x.shape[1]
    mag = np.abs(x) @ np.abs(w).T
    acc = (-(-min(group, K) // 16)) * 2.0 ** -21 + (2 * (-(-K // group)) + 64) * 2.0 ** -24
    return HALF_STEP[kind] * (1 + acc) * np.abs(y) + acc * mag + TINY[kind]


def sort(ids, E):
    """order, place, offsets of flat ids by a stable sort."""
    ids = np.asarray(ids).reshape(-1)
    ok = (ids >= 0) & (ids < E)
    slots = np.nonzero(ok)[0]
    by = slots[np.argsort(ids[slots], kind="stable")]
    order = np.full(ids.size, -1, np.int64)
    order[:by.size] = by
    place = np.full(ids.size, -1, np.int64)
    place[by] = np.arange(by.size)
    offsets = np.zeros(E + 1, np.int64)
    offsets[1:] = np.cumsum(np.bincount(ids[slots], minlength=E))
    return order, place, offsets
