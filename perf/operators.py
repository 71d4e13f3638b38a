"""Matrix products of microscaled (OCP MX) operands: activations quantised on the GPU against packed MXFP4 weights.

Three operators, each as an inference program calls it on activations that are already on the device:

  quantize   rows of bf16, fp16 or fp32 to MXFP4 (E2M1) or MXFP6 (E2M3), a power of two for every 32 columns, and back to
             the values they stand for
  linear     one projection: activations quantised to MXFP4 ("a4") or MXFP6 ("a6"), times an MXFP4 tensor; with `glu` the
             tensor holds gate and up and the product leaves as silu(gate) * up
  experts    the same product grouped by expert: every (token, route) pair against the tensor of its expert, groups of any
             size; with `routed` every pair has an activation row of its own (the down projection)

`rows` is the number of activation rows (tokens): 1 is a decode step of one sequence, up to a few dozen a batched decode or
speculative step, hundreds to thousands a prefill chunk.  Codes of weights are drawn uniformly -- every bit pattern is a valid
payload -- with block scales within a few octaves of one; activations are N(0, 1) with one channel in a thousand scaled by
20, as hidden states have them.
"""
from __future__ import annotations

import math

import numpy as np
import torch

own = False

DTYPE = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}
ACT = {"a4": "MXFP4", "a6": "MXFP6"}
MAX_FLOPS = 1.47e12


def listed():
    return [
        # the hidden state of one sequence before a projection: launch latency
        dict(name="quantize_a4_row1", kind="quantize", act="a4", rows=1, k=4096, dtype="bf16"),
        # the hidden rows of a prefill chunk in front of a down projection
        dict(name="quantize_a6_rows2048", kind="quantize", act="a6", rows=2048, k=12288, dtype="bf16"),
        # the fp32 rows that the packed matmuls return, for every (token, route) pair of a chunk
        dict(name="quantize_a4_fp32_rows16383", kind="quantize", act="a4", rows=16383, k=4096, dtype="fp32"),
        # one projection of a decode step: the weights are read once
        dict(name="linear_a4_row1", kind="linear", act="a4", out=12288, k=4096, rows=1, dtype="bf16", glu=False, result="fp32"),
        # a batched decode step through a down projection
        dict(name="linear_a6_rows13", kind="linear", act="a6", out=4096, k=12288, rows=13, dtype="bf16", glu=False, result="fp32"),
        # a prefill chunk of an odd length
        dict(name="linear_a4_rows601", kind="linear", act="a4", out=12288, k=4096, rows=601, dtype="bf16", glu=False, result="fp32"),
        # gate and up of a dense feed-forward block over a full prefill chunk
        dict(name="linear_a6_glu_rows2048", kind="linear", act="a6", out=24576, k=4096, rows=2048, dtype="fp16", glu=True, result="fp16"),
        # several prompts prefilled together: the most arithmetic
        dict(name="linear_a4_rows8192", kind="linear", act="a4", out=17408, k=5120, rows=8192, dtype="bf16", glu=False, result="bf16"),
        # gate and up of the routed experts of one token
        dict(name="experts_a6_glu_row1", kind="experts", act="a6", experts=64, top_k=8, out=4096, k=4096, rows=1, dtype="bf16",
             glu=True, routed=False, dropped=0.0, result="fp16"),
        # the down projection of a batched decode step that hits every expert, some routes dropped
        dict(name="experts_a4_rows61", kind="experts", act="a4", experts=64, top_k=8, out=4096, k=2048, rows=61, dtype="fp16",
             glu=False, routed=True, dropped=0.02, result="fp32"),
        # gate and up of a prefill chunk, many small experts
        dict(name="experts_a4_glu_rows2048", kind="experts", act="a4", experts=128, top_k=8, out=2048, k=2048, rows=2048, dtype="bf16",
             glu=True, routed=False, dropped=0.0, result="bf16"),
        # the down projection of a prefill chunk where rows end inside every tile
        dict(name="experts_a6_rows1501", kind="experts", act="a6", experts=32, top_k=4, out=2880, k=1440, rows=1501, dtype="bf16",
             glu=False, routed=True, dropped=0.0, result="fp32"),
    ]


def _log_int(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    while True:
        c = dict(kind=rng.choice(("quantize",) + ("linear",) * 3 + ("experts",) * 3), act=rng.choice(("a4", "a6")))
        if c["kind"] == "quantize":
            c.update(rows=_log_int(rng, 1, 16384), k=32 * _log_int(rng, 32, 544), dtype=rng.choice(tuple(DTYPE)))
            if c["rows"] * c["k"] > 6.72e7:
                continue
            return c
        c.update(dtype=rng.choice(("bf16", "bf16", "fp16")), glu=rng.random() < 0.4)
        c["result"] = rng.choice(("bf16", "fp16")) if c["glu"] else rng.choice(("fp32", "fp32", "bf16"))
        if c["kind"] == "linear":
            c.update(out=32 * _log_int(rng, 32, 544), k=32 * _log_int(rng, 32, 544), rows=_log_int(rng, 1, 8192))
        else:
            hidden, inter, experts = rng.choice(((4096, 2048, 64), (2048, 1024, 128), (2048, 768, 128), (2880, 1440, 32)))
            c.update(experts=experts, top_k=rng.choice((1, 2, 4, 8)), rows=_log_int(rng, 1, 4096), routed=not c["glu"],
                     out=2 * inter if c["glu"] else hidden, k=hidden if c["glu"] else inter, dropped=rng.choice((0.0, 0.0, 0.05)))
        if work(c)["flops"] <= MAX_FLOPS:
            return c


# ---- inputs --------------------------------------------------------------------------------------------------------
def _generator(seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    return g


def _activations(g, rows, k, dtype):
    x = torch.randn(rows, k, generator=g, device="cuda")
    x[:, torch.randperm(k, generator=g, device="cuda")[:max(1, k // 1000)]] *= 20.0
    return x.to(DTYPE[dtype])


def _weight(g, rows, k):
    """value and scale bytes of an MXFP4 tensor: scales 2^-9 .. 2^-2, so that products of a few thousand terms are of order one"""
    return (torch.randint(0, 256, (rows, k // 2), generator=g, device="cuda", dtype=torch.uint8),
            torch.randint(118, 126, (rows, k // 32), generator=g, device="cuda", dtype=torch.uint8))


def _routes(g, c):
    """expert ids [rows, top_k] of a router with a few favourites; a dropped route is -1"""
    liking = torch.randn(c["experts"], generator=g, device="cuda") * 0.5
    score = torch.randn(c["rows"], c["experts"], generator=g, device="cuda") + liking
    ids = score.topk(c["top_k"], dim=1).indices.to(torch.int32)
    gone = torch.rand(ids.shape, generator=g, device="cuda") < c["dropped"]
    return torch.where(gone, torch.full_like(ids, -1), ids).contiguous()


def prepare(case, seed):
    c, g = case, _generator(seed)
    s = dict(c)
    if c["kind"] == "quantize":
        s["x"] = _activations(g, c["rows"], c["k"], c["dtype"])
        return s
    experts = c.get("experts", 1)
    s["values"], s["scales"] = _weight(g, experts * c["out"], c["k"])
    s["x"] = _activations(g, c["rows"] * (c["top_k"] if c.get("routed") else 1), c["k"], c["dtype"])
    if c["kind"] == "experts":
        s["ids"] = _routes(g, c)
        s["most"] = int(torch.bincount(s["ids"].reshape(-1).clamp(min=0).long(), minlength=experts).max())
    if own:
        from tyloquant_amd.runtime_mx import MxWeight
        s["w"] = MxWeight.from_tensors("MXFP4", s["values"], s["scales"], out=c["out"])
    return s


# ---- the plain forms -------------------------------------------------------------------------------------------------
def _quantized(x, act):
    """fp32 values of the rows after quantisation: in each block of 32 the scale 2^(e - emax), e = the exponent of the largest
    magnitude and emax = 2; elements rounded to the nearest of E2M1 (up to 6) or E2M3 (up to 7.5), ties to even, the largest
    where they are beyond it.  The scale's exponent is at least -127."""
    mant, most = (1, 6.0) if act == "a4" else (3, 7.5)
    v = x.float().reshape(x.shape[0], -1, 32)
    e = torch.frexp(v.abs().amax(-1, keepdim=True))[1] - 1
    scale = torch.ldexp(torch.ones_like(v[..., :1]), (e - 2).clamp(min=-127))
    v = v / scale
    step = torch.ldexp(torch.ones_like(v), (torch.frexp(v)[1] - 1).clamp(min=0) - mant)
    return ((torch.round(v / step) * step).clamp(-most, most) * scale).reshape(x.shape[0], -1)


def _dequantized(values, scales):
    """fp32 values of an MXFP4 tensor: the low nibble is the even column; sign, two exponent bits (bias 1), one mantissa bit"""
    code = torch.stack((values & 15, values >> 4), -1).reshape(values.shape[0], -1)
    mag = (code & 7).float()
    mag = torch.where(mag < 4, mag * 0.5, torch.where(mag < 6, mag - 2.0, 2.0 * mag - 8.0))
    mag = torch.where(code >= 8, -mag, mag)
    scale = torch.ldexp(torch.ones_like(scales, dtype=torch.float32), scales.int() - 127)
    return (mag.reshape(*scales.shape, 32) * scale[..., None]).reshape(values.shape[0], -1)


def _finish(y, s):
    if s["glu"]:
        gate, up = y.chunk(2, -1)
        y = gate / (1.0 + torch.exp(-gate)) * up
    return y.to(DTYPE[s["result"]])


def _linear_plain(s):
    return _finish(_quantized(s["x"], s["act"]) @ _dequantized(s["values"], s["scales"]).t(), s)


def _experts_plain(s):
    """pairs gathered by expert into [experts, most, k], one batched product, rows scattered back; dropped pairs are zero"""
    flat = s["ids"].reshape(-1).long()
    pairs, e = flat.numel(), s["experts"]
    order = torch.argsort(torch.where(flat < 0, e, flat), stable=True)
    group = flat[order]
    first = torch.searchsorted(torch.where(group < 0, e, group), torch.arange(e, device=flat.device))
    place = torch.arange(pairs, device=flat.device) - first[group.clamp(min=0)]
    slot = torch.where(group < 0, e * s["most"], group * s["most"] + place)
    x = _quantized(s["x"], s["act"])
    src = order if s["routed"] else order // s["top_k"]
    xe = torch.zeros(e * s["most"] + 1, s["k"], device=x.device)
    xe[slot] = x[src]
    xt = xe[:-1].reshape(e, s["most"], s["k"]).transpose(1, 2).contiguous()
    w = _dequantized(s["values"], s["scales"]).reshape(e, s["out"], s["k"])
    ye = torch.bmm(w, xt).transpose(1, 2).reshape(e * s["most"], s["out"])
    y = torch.zeros(pairs, s["out"], device=x.device)
    y[order] = torch.where((group < 0)[:, None], torch.zeros((), device=x.device), ye[slot.clamp(max=e * s["most"] - 1)])
    return _finish(y, s).reshape(s["rows"], s["top_k"], -1)


# ---- the calls -------------------------------------------------------------------------------------------------------
def run(state):
    s = state
    if own:
        from tyloquant_amd import runtime_moe as RM
        from tyloquant_amd import runtime_mx as RX
        act, result = ACT[s["act"]], DTYPE[s.get("result", "fp32")]
        if s["kind"] == "quantize":
            return RX.mx_quantize(s["x"], act).dequantize(s["x"].dtype)
        if s["kind"] == "linear":
            if s["glu"]:
                return RX.mx_scaled_glu(s["w"], s["x"], act=act, out_dtype=result)
            return RX.mx_scaled_matmul(s["w"], s["x"], act=act, out_dtype=result)
        route = RM.build_moe_route_plan(s["ids"], s["experts"])
        if s["glu"]:
            return RX.mx_moe_glu(s["w"], s["x"], route, act=act, out_dtype=result)
        return RX.mx_moe_matmul(s["w"], s["x"], route, act=act, routed=s["routed"], out_dtype=result)
    if s["kind"] == "quantize":
        return _quantized(s["x"], s["act"]).to(s["x"].dtype)
    return _linear_plain(s) if s["kind"] == "linear" else _experts_plain(s)


# ---- what a pass cannot do without -----------------------------------------------------------------------------------
def work(case):
    """Inputs read once and outputs written once: weights of the experts that a batch hits on average, activations, results;
    of a quantisation also the codes and scales that it leaves."""
    c = case
    size = {"bf16": 2, "fp16": 2, "fp32": 4}
    coded = {"a4": 17 / 32, "a6": 25 / 32}[c["act"]]
    if c["kind"] == "quantize":
        n = c["rows"] * c["k"]
        return {"bytes": n * (2 * size[c["dtype"]] + coded), "flops": 0}
    cols = c["out"] // 2 if c["glu"] else c["out"]
    weight, rows, x_rows = c["out"] * c["k"] * 17 / 32, c["rows"], c["rows"]
    if c["kind"] == "experts":
        rows *= c["top_k"]
        weight *= c["experts"] * (1.0 - (1.0 - c["top_k"] * (1.0 - c["dropped"]) / c["experts"]) ** c["rows"])
        x_rows = rows if c["routed"] else c["rows"]
    return {"bytes": weight + x_rows * c["k"] * size[c["dtype"]] + rows * cols * size[c["result"]],
            "flops": 2.0 * rows * (1.0 - c.get("dropped", 0.0)) * c["out"] * c["k"]}


# ---- 64 bits -----------------------------------------------------------------------------------------------------------
def _grid(act):
    """every magnitude of the element type, in the order of its codes"""
    if act == "a4":
        return [0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0]
    return [(m / 8 if e == 0 else 1 + m / 8) * 2.0 ** (max(e, 1) - 1) for e in range(4) for m in range(8)]


def _rounded64(x, act):
    """nearest value of the grid by comparing with the midpoints; a value on a midpoint takes the even code"""
    grid = torch.tensor(_grid(act), dtype=torch.float64, device=x.device)
    mid = (grid[1:] + grid[:-1]) / 2
    even_above = torch.arange(1, len(grid), device=x.device) % 2 == 0
    parts = []
    for v in x.split(max(1, (1 << 25) // x.shape[1])):
        v = v.double().reshape(v.shape[0], -1, 32)
        most = v.abs().amax(-1, keepdim=True)
        unit = torch.exp2((torch.floor(torch.log2(most)) - 2).clamp(min=-127.0))
        a = v.abs() / unit
        below = torch.searchsorted(mid, a.contiguous(), right=False)  # midpoints under the value
        at = below.clamp(max=len(mid) - 1)
        code = below + ((mid[at] == a) & (below < len(mid)) & even_above[at])
        parts.append((grid[code] * torch.sign(v) * unit).reshape(v.shape[0], -1))
    return torch.cat(parts)


def _weight64(values, scales):
    table = torch.tensor(_grid("a4") + [-v for v in _grid("a4")], dtype=torch.float64, device=values.device)
    w = torch.empty(values.shape[0], 2 * values.shape[1], dtype=torch.float64, device=values.device)
    w[:, 0::2] = table[(values % 16).long()]
    w[:, 1::2] = table[(values // 16).long()]
    return w * torch.exp2(scales.double() - 127.0).repeat_interleave(32, dim=1)


def exact(case, seed):
    s = prepare(case, seed)
    x = _rounded64(s["x"], s["act"])
    if s["kind"] == "quantize":
        return x
    if s["kind"] == "linear":
        y = x @ _weight64(s["values"], s["scales"]).T
    else:
        ids = s["ids"].reshape(-1).cpu().numpy()
        y = torch.zeros(len(ids), s["out"], dtype=torch.float64, device="cuda")
        for e in np.unique(ids[ids >= 0]):
            own_pairs = torch.from_numpy(np.flatnonzero(ids == e)).cuda()
            rows = slice(int(e) * s["out"], (int(e) + 1) * s["out"])
            y[own_pairs] = x[own_pairs if s["routed"] else own_pairs // s["top_k"]] @ _weight64(s["values"][rows], s["scales"][rows]).T
    if s["glu"]:
        half = s["out"] // 2
        y = y[:, :half] * torch.sigmoid(y[:, :half]) * y[:, half:]
    return y if s["kind"] == "linear" else y.reshape(s["rows"], s["top_k"], -1)
