"""Refusals of the FP8 products, the layer of experts and the log probabilities: all before anything is launched, so they need no GPU."""
import ctypes as C

import pytest
import torch

from tyloquant_amd import _lib as L

P, ODD = 1 << 12, (1 << 12) + 2      # an aligned address that nobody reads, and one that is not


@pytest.fixture(scope="module")
def lib():
    return L.lib()


def refused(lib, rc, code, text):
    assert rc == code, (rc, lib.mfq_hip_last_error())
    assert text in lib.mfq_hip_last_error().decode(), lib.mfq_hip_last_error()


def test_quantize(lib):
    f = lib.mfq_hip_mx8_quantize_rows
    refused(lib, f(None, 0, 128, 1, 128, P, P, None), L.ERR_INVALID, "null")
    refused(lib, f(P, 3, 128, 1, 128, P, P, None), L.ERR_INVALID, "x_dtype")
    refused(lib, f(P, 0, 160, 1, 160, P, P, None), L.ERR_INVALID, "divisible by 128")
    refused(lib, f(P, 0, 127, 2, 128, P, P, None), L.ERR_INVALID, "ldx")
    refused(lib, f(P, 0, 128, 0, 128, P, P, None), L.ERR_INVALID, "[0, 128]")
    refused(lib, f(P, 0, 128, 2, 128, ODD, P, None), L.ERR_INVALID, "aligned")
    refused(lib, f(P + 1, 0, 128, 2, 128, P, P, None), L.ERR_INVALID, "aligned")
    g = lib.mfq_hip_mx8_dequant_quantized
    refused(lib, g(P, P, 1, 128, 5, P, 128, None), L.ERR_INVALID, "out_dtype")
    refused(lib, g(P, P, 2, 128, 0, P, 100, None), L.ERR_INVALID, "ldo")
    assert lib.mfq_hip_mx8_scale_bytes(3, 640) == 2 * 3 * 4 and lib.mfq_hip_mx8_scale_bytes(3, 100) == 0


def gemm(lib, **kw):
    a = dict(values=P, scales=P, rows=256, cols=256, row0=0, nrows=256, x=P, x_dtype=0, ldx=256, x_scales=None, M=40, glu=0, activation=0, y=P, y_dtype=0, ldy=256,
             ws=P, bytes=1 << 30)
    a.update(kw)
    return lib.mfq_hip_mx8_scaled_gemm_rows(*a.values(), None)


@pytest.mark.parametrize("kw,code,text", [
    (dict(values=None), L.ERR_INVALID, "null"), (dict(y=None), L.ERR_INVALID, "null"), (dict(M=0), L.ERR_INVALID, "M=0"),
    (dict(x_dtype=7), L.ERR_INVALID, "x_dtype"), (dict(y_dtype=-1), L.ERR_INVALID, "y_dtype"), (dict(cols=200, ldx=200), L.ERR_INVALID, "divisible by 128"),
    (dict(values=ODD), L.ERR_INVALID, "16-byte"), (dict(x_scales=ODD), L.ERR_INVALID, "4-byte"), (dict(x=P + 1), L.ERR_INVALID, "unaligned x"),
    (dict(ldx=255), L.ERR_INVALID, "ldx"), (dict(ldy=255), L.ERR_INVALID, "ldy"), (dict(row0=64, nrows=128), L.ERR_INVALID, "multiple of 128"),
    (dict(row0=128), L.ERR_INVALID, "128 + 256 of 256"), (dict(glu=1, y_dtype=2), L.ERR_INVALID, "16-bit"), (dict(glu=1, activation=9), L.ERR_INVALID, "activation"),
    (dict(glu=1, nrows=255, rows=255), L.ERR_INVALID, "gate and up"), (dict(bytes=10), L.ERR_WORKSPACE, "workspace"), (dict(ws=None), L.ERR_WORKSPACE, "workspace"),
    (dict(ws=P + 8), L.ERR_WORKSPACE, "unaligned"), (dict(cols=1 << 18, ldx=1 << 18), L.ERR_UNSUPPORTED, "columns"),
    (dict(rows=1 << 17, nrows=1 << 17, cols=1 << 17, ldx=1 << 17, glu=1, ldy=1 << 17), L.ERR_UNSUPPORTED, "gated"),
])
def test_linear(lib, kw, code, text):
    refused(lib, gemm(lib, **kw), code, text)


def moe(lib, **kw):
    a = dict(values=P, scales=P, rows=512, cols=256, out=128, slot=None, E=4, x=P, x_dtype=0, ldx=256, x_scales=None, routed=0, ids=P, T=40, R=2, dst=P, bounds=P,
             glu=0, activation=0, y=P, y_dtype=0, ldy=128, ws=P, bytes=1 << 30)
    a.update(kw)
    return lib.mfq_hip_mx8_moe_matmul(*a.values(), None)


@pytest.mark.parametrize("kw,code,text", [
    (dict(ids=None), L.ERR_INVALID, "ids"), (dict(dst=None), L.ERR_INVALID, "both"), (dict(T=0), L.ERR_INVALID, "0 tokens"), (dict(E=5), L.ERR_INVALID, "experts"),
    (dict(out=100, rows=400, ldy=100), L.ERR_INVALID, "whole blocks"), (dict(out=96), L.ERR_INVALID, "not 4 experts"), (dict(ldy=100), L.ERR_INVALID, "ldy"),
    (dict(bytes=0), L.ERR_WORKSPACE, "workspace"), (dict(ws=P + 8), L.ERR_WORKSPACE, "unaligned"), (dict(glu=1, y_dtype=2), L.ERR_INVALID, "16-bit"),
    (dict(dst=None, bounds=None, cols=20608, ldx=20608), L.ERR_UNSUPPORTED, "without a route map"),
    (dict(T=1 << 20, R=8, routed=1, cols=8192, ldx=8192), L.ERR_UNSUPPORTED, "rows"),
])
def test_experts(lib, kw, code, text):
    refused(lib, moe(lib, **kw), code, text)


def layer(lib, w=(), **kw):
    desc = dict(kind=8, experts=8, hidden=256, inter=128, shared_inter=0, reserved=0, gate_up=P, gate_up_scales=P, down=P, down_scales=P, sgu=None, sgus=None, sdn=None, sdns=None)
    desc.update(w)
    a = dict(x=P, x_dtype=0, ldx=256, T=4, logits=P, bias=None, k=2, mode=0, normalize=0, floor=1e-20, scale=1.0, activation=0, gate=None, ids=P, weights=P, y=P,
             y_dtype=2, ldy=256, ws=P, bytes=1 << 30)
    a.update(kw)
    return lib.mfq_hip_mx_moe_layer(C.byref(L.MxLayer(*desc.values())), *a.values(), None)


@pytest.mark.parametrize("w,kw,code,text", [
    ({}, dict(x=None), L.ERR_INVALID, "null"), (dict(kind=6), {}, L.ERR_INVALID, "kind=6"), (dict(down=None), {}, L.ERR_INVALID, "null tensor"),
    (dict(hidden=192), {}, L.ERR_INVALID, "divisible by 128"), (dict(kind=4, inter=48), {}, L.ERR_INVALID, "divisible by 32"),
    (dict(shared_inter=128), {}, L.ERR_INVALID, "shared"), (dict(experts=1025), {}, L.ERR_UNSUPPORTED, "1025 experts"),
    ({}, dict(x_dtype=2), L.ERR_INVALID, "x_dtype"), ({}, dict(y_dtype=4), L.ERR_INVALID, "y_dtype"), ({}, dict(T=17), L.ERR_UNSUPPORTED, "17 tokens"),
    ({}, dict(T=0), L.ERR_UNSUPPORTED, "0 tokens"), ({}, dict(k=9), L.ERR_INVALID, "top_k"), ({}, dict(mode=5), L.ERR_INVALID, "mode"),
    ({}, dict(mode=3, normalize=1), L.ERR_INVALID, "mutually exclusive"), ({}, dict(activation=2), L.ERR_INVALID, "activation"), ({}, dict(ldx=255), L.ERR_INVALID, "ldx"),
    (dict(gate_up=ODD), {}, L.ERR_INVALID, "16-byte"), (dict(kind=4, down_scales=P + 4), {}, L.ERR_INVALID, "8-byte"), ({}, dict(bytes=64), L.ERR_WORKSPACE, "workspace"),
    ({}, dict(ws=P + 8), L.ERR_WORKSPACE, "unaligned"), (dict(hidden=1 << 17, inter=1 << 16), dict(ldx=1 << 17, ldy=1 << 17), L.ERR_UNSUPPORTED, "experts of"),
])
def test_layer(lib, w, kw, code, text):
    refused(lib, layer(lib, w, **kw), code, text)


def logprobs(lib, **kw):
    a = dict(logits=P, dtype=2, ldl=1000, M=3, V=1000, tokens=P, top=5, lp=P, rank=P, entropy=P, ids=P, best=P, ws=P, bytes=1 << 30)
    a.update(kw)
    return lib.mfq_hip_token_logprobs(*a.values(), None)


@pytest.mark.parametrize("kw,code,text", [
    (dict(logits=None), L.ERR_INVALID, "null"), (dict(tokens=None), L.ERR_INVALID, "null"), (dict(dtype=3), L.ERR_INVALID, "dtype"), (dict(M=0), L.ERR_INVALID, "[0,"),
    (dict(ldl=999), L.ERR_INVALID, "ldl"), (dict(top=65), L.ERR_INVALID, "alternatives"), (dict(top=-1), L.ERR_INVALID, "alternatives"),
    (dict(top=8, V=7), L.ERR_INVALID, "alternatives"), (dict(ids=None), L.ERR_INVALID, "top_ids"), (dict(logits=ODD), L.ERR_INVALID, "unaligned"),
])
def test_logprobs(lib, kw, code, text):
    refused(lib, logprobs(lib, **kw), code, text)


def test_logprobs_workspace(lib):
    lib.mfq_hip_set_cu_count(256)
    try:
        need = lib.mfq_hip_token_logprobs_workspace_bytes(1, 151936, 20)
        assert need > 0 and lib.mfq_hip_token_logprobs_workspace_bytes(4096, 151936, 20) == 0
        refused(lib, logprobs(lib, M=1, V=151936, ldl=151936, top=20, bytes=need - 1), L.ERR_WORKSPACE, "workspace")
        refused(lib, logprobs(lib, M=1, V=151936, ldl=151936, top=20, ws=P + 8), L.ERR_WORKSPACE, "unaligned")
    finally:
        lib.mfq_hip_set_cu_count(0)


def test_host_layer():
    from tyloquant_amd import formats as F
    from tyloquant_amd import runtime as R
    from tyloquant_amd import runtime_moe as RM
    from tyloquant_amd import runtime_mx8 as R8
    from tyloquant_amd.runtime_mx import MxWeight

    def weight(dtype, rows, cols, out=None):
        storage, scale = F.mx_shapes(dtype, rows, cols)
        v, s = torch.zeros(storage, dtype=torch.uint8), torch.zeros(scale, dtype=torch.uint8)
        return MxWeight(F.MxHeader(dtype, 4 if dtype == "MXFP4" else 8, rows, cols, 0, v.numel(), v.numel(), s.numel()), v, s, out)

    x = torch.zeros(3, 256, dtype=torch.bfloat16)
    with pytest.raises(ValueError, match="divisible by 128"):
        R8.mx8_quantize(x[:, :200])
    with pytest.raises(TypeError, match="float32, bfloat16 or float16"):
        R8.mx8_quantize(x.double())
    with pytest.raises(ValueError, match="current GPU, got cpu"):
        R8.mx8_quantize(x)
    with pytest.raises(ValueError, match="must be contiguous uint8"):
        R8.Mx8Rows(torch.zeros(3, 256, dtype=torch.uint8), torch.zeros(3, 2, dtype=torch.uint8), (3, 256))
    w8, w4 = weight("MXFP8", 256, 256), weight("MXFP4", 256, 256)
    with pytest.raises(ValueError, match="use mx_scaled_matmul"):
        R8.mx8_scaled_matmul(w4, x)
    with pytest.raises(ValueError, match="width 128 != neuron length 256"):
        R8.mx8_scaled_matmul(w8, x[:, :128])
    with pytest.raises(TypeError, match="results are"):
        R8.mx8_scaled_matmul(w8, x, out_dtype=torch.float64)
    with pytest.raises(ValueError, match="16-bit type"):
        R8.mx8_scaled_glu(w8, x, out_dtype=torch.float32)
    with pytest.raises(IndexError):
        R8.mx8_scaled_matmul(w8, x, expert=1)
    with pytest.raises(ValueError, match="current GPU"):
        R8.mx8_scaled_matmul(w8, x)
    route = RM.MoeRoutePlan(torch.zeros(3, 2, dtype=torch.int32), 2)
    with pytest.raises(ValueError, match="3 rows for 3 tokens of 2 routes"):
        R8.mx8_moe_matmul(weight("MXFP8", 256, 256, 128), x, route, routed=True)
    with pytest.raises(ValueError, match="1 experts, a route plan for 2"):
        R8.mx8_moe_matmul(w8, x, route)

    gate_up, down, logits = weight("MXFP8", 4 * 256, 256, 256), weight("MXFP8", 4 * 256, 128, 256), torch.zeros(3, 4)
    call = lambda gu=gate_up, dn=down, x=x, z=logits, k=2, **kw: RM.mx_moe_ffn_forward(gu, dn, x, z, k, **kw)
    with pytest.raises(ValueError, match="current GPU, got cpu"):
        call()
    with pytest.raises(ValueError, match="all MXFP8 or all MXFP4"):
        call(shared=(weight("MXFP8", 256, 256), Kind4()))
    with pytest.raises(ValueError, match="incompatible gate_up"):
        call(dn=weight("MXFP8", 3 * 256, 128, 256))
    with pytest.raises(ValueError, match="incompatible shared"):
        call(shared=(weight("MXFP8", 128, 256), weight("MXFP8", 256, 128)))
    with pytest.raises(ValueError, match="at most 16 tokens, got 17"):
        call(x=torch.zeros(17, 256, dtype=torch.bfloat16), z=torch.zeros(17, 4))
    with pytest.raises(ValueError, match="top_k"):
        call(k=5)
    with pytest.raises(ValueError, match="router logits"):
        call(z=torch.zeros(3, 5))
    with pytest.raises(ValueError, match="shared_gate"):
        call(shared_gate=torch.zeros(3))
    with pytest.raises(ValueError, match="mutually exclusive"):
        call(use_sigmoid=True, use_sqrt_softplus=True)
    with pytest.raises(TypeError, match="bfloat16 or float16"):
        call(x=torch.zeros(3, 256))

    z, tokens = torch.zeros(3, 100), torch.zeros(3, dtype=torch.int64)
    with pytest.raises(ValueError, match="current GPU"):
        R.token_logprobs(z, tokens)
    with pytest.raises(TypeError, match="logits must be"):
        R.token_logprobs(z.double(), tokens)
    with pytest.raises(ValueError, match="one for each row"):
        R.token_logprobs(z, tokens[:2])
    with pytest.raises(ValueError, match="one for each row"):
        R.token_logprobs(z, tokens.int())
    for top in (-1, 65, 101):
        with pytest.raises(ValueError, match="top must be"):
            R.token_logprobs(z, tokens, top)


class Kind4:
    """an MXFP4 tensor whose scales are laid already"""
    kind, dtype, rows, neuron_len, out, n_experts = 4, "MXFP4", 256, 128, 256, 1
    values = scales = torch.zeros(1, dtype=torch.uint8)

    def laid_scales(self):
        return self.scales
