"""Cohorts of a NINTM tensor and quantised activations (act=) without a GPU: tables, refusals."""
import types

import numpy as np
import pytest
import torch

from tyloquant_amd import _lib as L
from tyloquant_amd import runtime_moe as RM


def cohort(ids, linears=0, mx=None):
    """a cohort as its constructor leaves it, on the CPU"""
    c = RM.ForeignCohort.__new__(RM.ForeignCohort)
    c.dtype, c.expert_ids, c.out, c.neuron_len = "MXFP4" if mx else "NVQ2J", np.asarray(ids, np.int32), 16, 64
    c.nepq, c.mx = None, mx
    c.linears = [types.SimpleNamespace(weight=types.SimpleNamespace(data=torch.zeros(8, dtype=torch.uint8), desc=L.NvqDesc())) for _ in range(linears)]
    c._slot = c._wtab = None
    c.live = np.ones(len(ids), dtype=bool)
    return c


def test_slots_come_with_the_addresses_of_the_experts(monkeypatch):
    """A decode launch gets the table of weights whoever asked for the slots first."""
    got = {}
    monkeypatch.setattr(L, "lib", lambda: types.SimpleNamespace(mfq_hip_nvq_gemv_pairs=lambda desc, wtab, *a: got.update(wtab=wtab) or 0))
    monkeypatch.setattr(RM, "_stream", lambda: None)
    c = cohort([2, 0], linears=2)
    assert c.slots(4, "cpu").tolist() == [1, -1, 0, -1]
    x, ids, flat = torch.zeros(1, 64, dtype=torch.bfloat16), torch.zeros(1, 2, dtype=torch.int32), torch.zeros(2, 16)
    c.matmul_pairs(4, x, False, ids, 1, 2, flat)
    assert got["wtab"] is not None and c._wtab.tolist() == [q.weight.data.data_ptr() for q in c.linears]


def test_tables_of_cohorts_are_there_from_the_start():
    """A first call may be a captured one, in which nothing can be copied from the host."""
    parts = [cohort([3, 0], mx=types.SimpleNamespace(kind=4)), cohort([1], linears=1)]
    w = RM.NintMoeWeight(4, 16, 64, [], [], torch.device("cpu"), parts)
    assert [None if c._slot is None else c._slot.tolist() for c in w.foreign] == [[1, -1, -1, 0], [-1, 0, -1, -1]]
    assert w.foreign[1]._wtab is not None


def test_scales_of_every_capable_cohort_are_laid_out():
    laid = []
    parts = [cohort([i], mx=types.SimpleNamespace(kind=4, laid_scales=lambda i=i: laid.append(i))) for i in (0, 1)] + [cohort([2], linears=1)]
    RM.NintMoeWeight(3, 16, 64, [], [], torch.device("cpu"), parts).lay_scales()
    assert laid == [0, 1]


@pytest.mark.parametrize("decode", [True, False])
def test_feed_forward_block_refuses_unknown_activation_types(decode, monkeypatch):
    """Whichever launches would serve the call, and before any of them."""
    gate_up = RM.NintMoeWeight(2, 32, 64, [], [], torch.device("cpu"))
    down = RM.NintMoeWeight(2, 64, 16, [], [], torch.device("cpu"))
    ran = []
    monkeypatch.setattr(RM, "moe_topk", lambda *a: ran.append("topk") or (torch.zeros(1, 1, dtype=torch.int32), torch.ones(1, 1)))
    monkeypatch.setattr(RM, "build_moe_route_plan", lambda ids, n: RM.MoeRoutePlan(ids, n))
    for w in (gate_up, down):
        w.decode_capable = lambda *a: decode
        w.forward_decode = lambda *a, **k: ran.append("decode") or torch.zeros(1, 64)
        w.forward_shared = lambda *a, **k: torch.zeros(2, 64)
    monkeypatch.setattr(RM, "moe_weighted_reduce", lambda *a: a[0])
    with pytest.raises(ValueError, match="MXFP4 or MXFP6, not MXFP8"):
        RM.nint_moe_ffn_forward(gate_up, down, torch.zeros(1, 64), torch.zeros(1, 2), 1, act="MXFP8", shared=(None, None))
    assert not ran
