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
