"""FP8 products of routed experts in a decode step on the GPU: plans of a few tokens, which have no route map."""
import pytest
import torch

import mx8_ref as P
from mx8_ref import BF16, FP16, FP32
from test_mx8_gpu import check_pairs, routes, tensor

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("T", [1, 3, 8, 9])
@pytest.mark.parametrize("K", [20480, 20608])
def test_long_rows(T, K):
    """a block a pair up to 20480 columns, beyond them the tiles of a map that the call makes: the same from one token on"""
    from tyloquant_amd import runtime_moe as RM
    from tyloquant_amd import runtime_mx8 as R8
    E, R, out = 5, 2, 128
    w, wd = tensor(K, E * out, K, out=out)
    ids = routes(T, T, R, E, 0.2)
    route = RM.build_moe_route_plan(ids, E)
    assert (route.ids_dst is None) == (T <= 8)
    x = P.make_x(T, T, K, BF16)
    xd = P.rounded(x)
    check_pairs(R8.mx8_moe_matmul(w, x, route, out_dtype=FP32), xd, wd, ids, out, E, False, False)
    check_pairs(R8.mx8_moe_glu(w, R8.mx8_quantize(x), route), xd, wd, ids, out, E, False, True)
    x = P.make_x(T + 1, T * R, K, FP16)
    check_pairs(R8.mx8_moe_matmul(w, x, route, routed=True, out_dtype=BF16), P.rounded(x), wd, ids, out, E, True, False)
    assert (route.ids_dst is None) == (T <= 8)       # the plan is the caller's


def test_long_rows_in_a_graph():
    from tyloquant_amd import runtime_moe as RM
    from tyloquant_amd import runtime_mx8 as R8
    E, out, K = 4, 128, 20608
    w, _ = tensor(1, E * out, K, out=out)
    x, ids = P.make_x(2, 4, K, BF16), routes(3, 4, 2, E, 0.1)
    work = lambda: R8.mx8_moe_matmul(w, x, RM.build_moe_route_plan(ids, E))
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        work()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = work()
    for n in range(3):
        x.copy_(P.make_x(10 + n, 4, K, BF16))
        ids.copy_(routes(20 + n, 4, 2, E, 0.1))
        want = work()
        got.zero_()
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(got, want)
