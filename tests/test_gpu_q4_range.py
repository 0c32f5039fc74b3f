"""4-bit products on the GPU, what the other files leave of their range: workspaces that captured graphs keep."""
from __future__ import annotations

import pytest

import emugemm
import q4ref

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
