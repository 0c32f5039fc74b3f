"""Arrays without a leading dimension (ids, places, offsets, weights of the choices) are refused when a tensor does not hold
its values one behind the other; host tensors stand in for device ones, and nothing is launched."""
from __future__ import annotations

import pytest
import torch

import emugemm

P, T, TOPK, E = 4096, 6, 2, 4


class StandIn:
    def __getattr__(self, name):
        return lambda *args: 0


def i32(*shape):
    return torch.zeros(*shape, dtype=torch.int32)


CALLS = {
    "expert_sort": (dict(T=T, topk=TOPK, E=E, expert=i32(T, TOPK), order=i32(T * TOPK), place=i32(T, TOPK), offsets=i32(E + 1)),
                    dict(expert=T * TOPK, order=T * TOPK, place=T * TOPK, offsets=E + 1)),
    "q4_gemm_experts": (dict(R=4, E=E, N=16, K=64, A=P, lda=64, offsets=i32(E + 1), packed=P, group=32, C=P, ldc=16, dtype=0),
                        dict(offsets=E + 1)),
    "expert_gather": (dict(T=T, topk=TOPK, H=16, X=P, ldx=16, place=i32(T, TOPK), XS=P, ldxs=16, dtype=0), dict(place=T * TOPK)),
    "expert_gather_backward": (dict(T=T, topk=TOPK, H=16, dXS=P, lddxs=16, place=i32(T, TOPK), dX=P, lddx=16, dtype=0),
                               dict(place=T * TOPK)),
    "expert_combine": (dict(T=T, topk=TOPK, H=16, YS=P, ldys=16, place=i32(T, TOPK), weights=torch.zeros(T, TOPK), Y=P, ldy=16,
                            dtype=0), dict(place=T * TOPK, weights=T * TOPK)),
    "expert_combine_backward": (dict(T=T, topk=TOPK, H=16, dY=P, lddy=16, YS=P, ldys=16, place=i32(T, TOPK),
                                     weights=torch.zeros(T, TOPK), dYS=P, lddys=16, dweights=torch.zeros(T, TOPK), dtype=0),
                                dict(place=T * TOPK, weights=T * TOPK, dweights=T * TOPK)),
}


@pytest.mark.parametrize("name,arg", [(n, a) for n, (_, args) in CALLS.items() for a in args])
def test_gaps_are_refused(monkeypatch, name, arg):
    monkeypatch.setattr(emugemm, "_lib", StandIn())
    h = emugemm.Handle.__new__(emugemm.Handle)
    h.h, h.device = None, -1                        # -1: the host, where these tensors are
    kw, sizes = CALLS[name]
    n, t = sizes[arg], kw[arg].dtype
    call = getattr(h, name)
    call(**kw)
    call(**{**kw, arg: P})                          # an address is taken as it is
    call(**{**kw, arg: torch.zeros(n + 3, dtype=t)[1:]})
    other = torch.float64 if t == torch.float32 else torch.int64
    for bad in (torch.zeros(2 * n, dtype=t)[::2], torch.zeros(TOPK, n, dtype=t).t(), torch.zeros(1, dtype=t).expand(n),
                torch.zeros(n, 3, dtype=t)[:, :2], torch.zeros(n, dtype=other)):
        with pytest.raises(ValueError):
            call(**{**kw, arg: bad})


def test_no_tokens_need_no_arrays(monkeypatch):
    monkeypatch.setattr(emugemm, "_lib", StandIn())
    h = emugemm.Handle.__new__(emugemm.Handle)
    h.h, h.device = None, -1
    h.expert_sort(0, 2, 5, None, None, None, i32(6))
    h.expert_gather(0, 2, 16, P, 16, i32(0, 2), P, 16, dtype=0)


def test_types_before_and_after_the_first_tensor(monkeypatch):
    """The names stand for torch's types until a call has seen a tensor."""
    for name, t in (("_i32", torch.int32), ("_f32", torch.float32)):
        monkeypatch.setattr(emugemm, name, str(t))
    monkeypatch.setattr(emugemm, "_lib", StandIn())
    h = emugemm.Handle.__new__(emugemm.Handle)
    h.h, h.device = None, -1
    kw, _ = CALLS["expert_combine"]
    with pytest.raises(ValueError):
        h.expert_combine(**{**kw, "weights": torch.zeros(T, TOPK, dtype=torch.int32)})
    h.expert_combine(**kw)
    assert emugemm._i32 is torch.int32 and emugemm._f32 is torch.float32
    h.expert_combine(**kw)
    with pytest.raises(ValueError):
        h.expert_combine(**{**kw, "weights": torch.zeros(T, TOPK, dtype=torch.int32)})
