"""Calls of NINTM tensors and feed-forward blocks with quantised activations (act=) as a program that captures its steps makes them."""
import numpy as np
import pytest
import torch

from test_mx_scaled_gpu import hidden, mixed_moe, routes
import mx_scaled_ref as P

pytestmark = pytest.mark.gpu


def experts(rng, E, out, K, parts):
    """a NINTM tensor of MXFP4 cohorts alone"""
    from tyloquant_amd import formats as F
    from tyloquant_amd import runtime_moe as RM
    pools = []
    for ids in parts:
        v, s, _ = P.weight(rng, len(ids) * out, K)
        pools.append((ids.astype(np.int32), "MXFP4", F.write_mx("MXFP4", len(ids) * out, K, v, s)))
    return RM.NintMoeWeight.from_blob(F.nintm_blob(E, out, K, pools))


@pytest.mark.parametrize("T", [4, 40])
@pytest.mark.parametrize("cohorts", [1, 2, "mixed"])
def test_a_first_call_may_be_captured(cohorts, T):
    """With its scales laid out a tensor's first call with `act` can be part of a graph; replays follow new inputs and give the bits of
    eager calls."""
    from tyloquant_amd import runtime_moe as RM
    rng = np.random.default_rng(T)
    E, out, K, R = 12, 96, 384, 3
    if cohorts == "mixed":
        w = mixed_moe(rng, E, out, K)[0]
    else:
        w = experts(rng, E, out, K, np.array_split(rng.permutation(E), cohorts))
    x = hidden(rng, T, K).to(torch.bfloat16).cuda()
    route = RM.build_moe_route_plan(torch.from_numpy(routes(rng, T, R, E, "any")).cuda(), E)
    with pytest.raises(RuntimeError, match="before a graph is captured"):
        with torch.cuda.graph(torch.cuda.CUDAGraph()):
            w.forward(x, route, act="MXFP6")
    w.lay_scales()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        held = w.forward(x, route, act="MXFP6"), w.forward_glu(x, route, act="MXFP4")
    for k in range(3):
        x.copy_(hidden(rng, T, K))
        eager = w.forward(x, route, act="MXFP6"), w.forward_glu(x, route, act="MXFP4")
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(eager, held)), k
