"""MXFP4 / MXFP8 weights of full-precision MFQ files and their matmul (see runtime.py).

Mirrors the reference's Mxfp8Weight / mxfp8_matmul_f32 (cpp_runtime/mfq_decode.cpp:2060-2100, 8784-8802) and, for MXFP4
expert pools, dequant_mxfp4_cpu / select_mxfp4_cpu_rows (:1920-1975): the payload's value and scale bytes are used on the
device as they lie in the file.

Products of two microscaled operands (mx_quantize, mx_scaled_matmul, mx_scaled_glu, mx_moe_matmul, mx_moe_glu) have no
counterpart there: activations are quantised to MXFP4 or MXFP6 with a scale for every 32 columns, and the matrix cores
multiply the codes."""
from __future__ import annotations

import torch

from . import _lib as L
from . import formats as F
from .runtime import _Workspace, _as_2d, _like_rows, _ptr, _stream, _upload, _x_dtype, borrow


class MxWeight:
    """[rows, cols] (a linear), or a pool of experts of `out` rows each when `out` is given."""

    def __init__(self, header: F.MxHeader, values: torch.Tensor, scales: torch.Tensor, out: int | None = None):
        self.header, self.values, self.scales = header, values, scales
        self.dtype, self.kind, self.rows, self.neuron_len = header.dtype, header.kind, header.rows, header.cols
        self.out = self.rows if out is None else int(out)
        if self.out <= 0 or self.rows % self.out:
            raise ValueError(f"{self.dtype}: {self.rows} rows are not a whole number of experts of {self.out}")
        if self.kind == 8 and self.out != self.rows and self.out % 128:
            raise ValueError("MXFP8 expert slices must preserve 128-row blocks")
        self.n_experts = self.rows // self.out
        self.data = values                      # the device tensor other weights call `data`
        self._ws = _Workspace()
        self._laid = self._laid_of = self._laid_version = None   # scales of laid_scales, and those that they were made from
        self._needs = {}

    @property
    def payload_bytes(self) -> int:
        return self.header.values_bytes + self.header.scales_bytes

    @staticmethod
    def from_tensors(dtype: str, values: torch.Tensor, scales: torch.Tensor, out: int | None = None) -> "MxWeight":
        """The two byte matrices of a payload that are on the device already (uint8, contiguous, used as they are)."""
        if values.dim() != 2 or scales.dim() != 2 or values.dtype != torch.uint8 or scales.dtype != torch.uint8:
            raise ValueError(f"{dtype}: values and scales must be uint8 matrices")
        cols = values.shape[1] * (2 if dtype == "MXFP4" else 1)
        storage, scale = F.mx_shapes(dtype, values.shape[0], cols)
        if tuple(values.shape) != tuple(storage) or tuple(scales.shape) != tuple(scale):
            raise ValueError(f"{dtype}: values {tuple(values.shape)} and scales {tuple(scales.shape)} must be {tuple(storage)} and {tuple(scale)}")
        if not (values.is_cuda and scales.is_cuda and values.device == scales.device and values.is_contiguous() and scales.is_contiguous()):
            raise ValueError(f"{dtype}: values and scales must be contiguous and on one GPU")
        h = F.MxHeader(dtype, 4 if dtype == "MXFP4" else 8, values.shape[0], cols, 0, values.numel(), values.numel(), scales.numel())
        return MxWeight(h, values, scales, out)

    def laid_scales(self, again: bool = False) -> torch.Tensor:
        """Scales as the products of microscaled operands read them (mfq_hip_mx_lay_scales), laid out at the first call and kept:
        1/16 of the values' bytes.  Scales that torch operations have rewritten in place since are laid out again, to the same place, so
        that captured products see them too; writes that torch does not count (of other libraries, or where the scales are an inference
        tensor) need a call with `again`.  A graph cannot be the first to ask: what it writes is there only after a replay."""
        scales = self.scales
        if self._laid is not None and not again and self._laid_of is scales and (self._laid_version is None or self._laid_version == scales._version):
            return self._laid
        if self.kind != 4:
            raise ValueError(f"products of microscaled operands take MXFP4 weights, not {self.dtype}: use mx_matmul")
        _here(scales)
        if torch.cuda.is_current_stream_capturing():
            raise RuntimeError(f"{self.dtype}: call laid_scales() (lay_scales() of a tensor of experts) before a graph is captured")
        version = None if scales.is_inference() else scales._version
        laid = self._laid if self._laid is not None else torch.empty(_scale_bytes(self.rows, self.neuron_len), dtype=torch.uint8, device=scales.device)
        L.check(L.lib().mfq_hip_mx_lay_scales(_ptr(scales), self.rows, self.neuron_len, _ptr(laid), _stream()))
        torch.cuda.current_stream().synchronize()   # later calls may come on other streams
        self._laid, self._laid_of, self._laid_version = laid, scales, version
        return laid

    def note_need(self, key, need: int) -> int:
        """Remembers the workspace of a call's sizes; a program whose every call has other sizes starts over now and then."""
        if len(self._needs) >= 1024:
            self._needs.clear()
        self._needs[key] = need
        return need

    @staticmethod
    def from_blob(dtype: str, blob, device="cuda", out: int | None = None) -> "MxWeight":
        h = F.parse_mx(dtype, blob)
        device = torch.device(device)
        values = _upload(blob, h.values_off, h.values_bytes, device)
        scales = _upload(blob, h.scales_off, h.scales_bytes, device)
        torch.cuda.current_stream().synchronize()
        return MxWeight(h, values, scales, out)

    def _rows(self, expert: int):
        if not 0 <= expert < self.n_experts:
            raise IndexError(f"{self.dtype}: expert {expert} of {self.n_experts}")
        return expert * self.out, self.out

    def dequantize(self, expert: int = 0, dtype=torch.float32) -> torch.Tensor:
        """fp32: element x scale; fp16: that rounded once more, as the reference's device copy is."""
        row0, nrows = self._rows(expert)
        if dtype not in (torch.float32, torch.float16):
            raise ValueError(f"MX weights dequantize to fp32 or fp16, not {dtype}")
        w = torch.empty((nrows, self.neuron_len), dtype=dtype, device=self.values.device)
        L.check(L.lib().mfq_hip_mx_dequant_rows(self.kind, _ptr(self.values), _ptr(self.scales), self.rows, self.neuron_len,
                                                row0, nrows, L.X_F32 if dtype == torch.float32 else L.X_F16, _ptr(w),
                                                self.neuron_len, _stream()))
        return w


def mx_matmul(w: MxWeight, x: torch.Tensor, expert: int = 0) -> torch.Tensor:
    """x @ W^T in fp32 (mxfp8_matmul_f32, cpp_runtime/mfq_decode.cpp:8784-8802): the matrix-core kernels up to 256 rows (a
    wave per neuron for activations they cannot read in 16-byte pieces), the prefill tile kernel above and, for bf16 rows,
    from where it is cheaper (33 rows and more, by size)."""
    row0, nrows = w._rows(expert)
    x2 = _as_2d(x, w.neuron_len)
    M = x2.shape[0]
    y = torch.empty((M, nrows), dtype=torch.float32, device=x.device)
    if M == 0:
        return _like_rows(y, x)
    lib = L.lib()
    need = lib.mfq_hip_mx_gemm_rows_workspace_bytes(w.neuron_len, nrows, M)
    ws = w._ws.get(need, x.device)
    L.check(lib.mfq_hip_mx_gemm_rows(w.kind, _ptr(w.values), _ptr(w.scales), w.rows, w.neuron_len, row0, nrows, _ptr(x2),
                                     _x_dtype(x2), x2.stride(0), M, _ptr(y), nrows, _ptr(ws), need, _stream()))
    return _like_rows(y, x)


# ---------------------------------------------------------------------------------------
# Products of two microscaled operands
# ---------------------------------------------------------------------------------------
_ACT = {"MXFP4": 4, "MXFP6": 6}
_OUT = {torch.float32: L.X_F32, torch.bfloat16: L.X_BF16, torch.float16: L.X_F16}


def _row_bytes(kind: int, K: int) -> int:
    return -(-K // 256) * (128 if kind == 4 else 192)


def _scale_bytes(rows: int, K: int) -> int:
    return -(-rows // 32) * -(-K // 256) * 256


def _out_dtype(dtype) -> int:
    code = _OUT.get(dtype)
    if code is None:
        raise TypeError(f"results are float32, bfloat16 or float16, not {dtype}")
    return code


def check_act(act: str) -> int:
    """kind of a type that activations are quantised to; refuses others"""
    kind = _ACT.get(act)
    if kind is None:
        raise ValueError(f"activations are quantised to MXFP4 or MXFP6, not {act}")
    return kind


class MxRows:
    """Quantised activations [.., neuron_len]: value bytes of rows of whole groups of 256 columns (uint8 [M, 128 or 192 a group], the
    layout of mfq_hip_mx_quantize_rows) and E8M0 scales (uint8, by 32 rows and groups); `shape` is that of the rows before
    quantisation."""

    def __init__(self, dtype: str, values: torch.Tensor, scales: torch.Tensor, shape):
        shape = tuple(shape)
        kind = check_act(dtype)
        if not shape or shape[-1] <= 0 or shape[-1] % 32:
            raise ValueError(f"{dtype} columns must be divisible by 32: {shape}")
        rows = torch.Size(shape[:-1]).numel()
        want = (rows, _row_bytes(kind, shape[-1])), (_scale_bytes(rows, shape[-1]),)
        if values.dtype != torch.uint8 or scales.dtype != torch.uint8 or (tuple(values.shape), tuple(scales.shape)) != want or \
                not (values.is_contiguous() and scales.is_contiguous()) or values.device != scales.device:
            raise ValueError(f"{dtype} rows of {shape}: values {tuple(values.shape)} and scales {tuple(scales.shape)} must be contiguous uint8 "
                             f"{want[0]} and {want[1]} on one device")
        self._set(dtype, kind, values, scales, shape, rows)

    def _set(self, dtype, kind, values, scales, shape, rows):
        self.dtype, self.kind, self.values, self.scales, self.shape = dtype, kind, values, scales, shape
        self.rows, self.neuron_len = rows, shape[-1]
        return self

    def dequantize(self, dtype=torch.float32) -> torch.Tensor:
        """element x scale in fp32, rounded once to `dtype`."""
        code = _out_dtype(dtype)
        out = torch.empty(self.shape, dtype=dtype, device=self.values.device)
        if self.rows:
            _here(out)
            L.check(L.lib().mfq_hip_mx_dequant_quantized(self.kind, self.values.data_ptr(), self.scales.data_ptr(), self.rows, self.neuron_len, code,
                                                         out.data_ptr(), self.neuron_len, _stream()))
        return out


def _here(t: torch.Tensor) -> None:
    """Launches go to the current device's stream: refuse tensors that are elsewhere."""
    if not t.is_cuda:
        raise ValueError(f"tensors must be on the current GPU, got {t.device}")
    if t.get_device() != torch._C._cuda_getDevice():
        raise ValueError(f"tensors must be on the current GPU (cuda:{torch._C._cuda_getDevice()}), got {t.device}")


def _raw_rows(x: torch.Tensor, K: int) -> torch.Tensor:
    """[rows, K] with neighbouring columns side by side, and rows that do not lie on one another (a broadcast one is copied)"""
    if x.dtype not in _OUT:
        raise TypeError(f"activations must be float32, bfloat16 or float16, got {x.dtype}")
    x2 = _as_2d(x, K)
    return x2 if x2.shape[0] == 1 or x2.stride(0) >= K else x2.contiguous()


def mx_quantize(x: torch.Tensor, dtype: str = "MXFP4") -> MxRows:
    """Rows of bf16, fp16 or fp32 [..., K] to MXFP4 or MXFP6 with a power of two for every 32 columns: 2^(e - 2), e = the
    exponent of the block's largest magnitude; elements to nearest, ties to even, the largest where they are beyond it.  A block
    that holds an infinity or a NaN becomes NaN."""
    kind, shape = check_act(dtype), tuple(x.shape)
    K = shape[-1] if shape else 0
    if K % 32 or K == 0:
        raise ValueError(f"{dtype} columns must be divisible by 32, got {K}")
    x2 = _raw_rows(x, K)
    _here(x2)
    M = x2.shape[0]
    values = torch.empty((M, _row_bytes(kind, K)), dtype=torch.uint8, device=x2.device)
    scales = torch.empty(_scale_bytes(M, K), dtype=torch.uint8, device=x2.device)
    if M:
        L.check(L.lib().mfq_hip_mx_quantize_rows(kind, x2.data_ptr(), _OUT[x2.dtype], x2.stride(0), M, K, values.data_ptr(), scales.data_ptr(), _stream()))
    return MxRows.__new__(MxRows)._set(dtype, kind, values, scales, shape, M)


def _operand(x, K: int, act: str):
    """(kind, tensor, x_dtype, row stride, scales or None, rows, shape) of activations that come quantised or not"""
    if isinstance(x, MxRows):
        if x.neuron_len != K:
            raise ValueError(f"activation width {x.neuron_len} != neuron length {K}")
        return x.kind, x.values, 0, 0, x.scales, x.rows, x.shape
    x2 = _raw_rows(x, K)
    return check_act(act), x2, _OUT[x2.dtype], x2.stride(0), None, x2.shape[0], x.shape


def _result_dtype(w: MxWeight, rows: int, glu: int, out_dtype) -> int:
    code = _out_dtype(out_dtype)
    if glu and (rows % 2 or code == L.X_F32):
        raise ValueError(f"{w.dtype}: a gated product takes a 16-bit type and as many gate as up rows, not {out_dtype} and {rows} rows")
    return code


def _scaled(w: MxWeight, x, act: str, expert: int, glu: int, activation: int, out_dtype) -> torch.Tensor:
    row0, nrows = w._rows(expert)
    K = w.neuron_len
    kind, x2, xd, ldx, xs, M, shape = _operand(x, K, act)
    yd = _result_dtype(w, nrows, glu, out_dtype)
    laid = w.laid_scales()
    _here(x2)
    _here(w.values)
    width = nrows // 2 if glu else nrows
    y = torch.empty((M, width), dtype=out_dtype, device=x2.device)
    if M:
        lib = L.lib()
        key = (kind, nrows, M, xs is None)
        need = w._needs.get(key)
        if need is None:
            need = w.note_need(key, lib.mfq_hip_mx_scaled_gemm_workspace_bytes(kind, nrows, K, M, xs is not None))
        ws = borrow(need, x2.device)
        L.check(lib.mfq_hip_mx_scaled_gemm_rows(w.values.data_ptr(), laid.data_ptr(), w.rows, K, row0, nrows, kind, x2.data_ptr(), xd, ldx,
                                                _ptr(xs), M, glu, activation, y.data_ptr(), yd, width, _ptr(ws), need if ws is not None else 0,
                                                _stream()))
    return y if len(shape) == 2 else y.reshape(*shape[:-1], width)


def mx_scaled_matmul(w: MxWeight, x, act: str = "MXFP6", expert: int = 0, out_dtype=torch.float32) -> torch.Tensor:
    """q(x) @ W^T of an MXFP4 tensor, fp32 sums rounded once to `out_dtype`.  x: bf16, fp16 or fp32 [..., K], quantised to `act` by the
    call, or MxRows (their own type).  mx_matmul is the product with unquantised activations."""
    return _scaled(w, x, act, expert, 0, 0, out_dtype)


def mx_scaled_glu(w: MxWeight, x, act: str = "MXFP6", activation: int = L.GLU_SILU, expert: int = 0, out_dtype=torch.bfloat16) -> torch.Tensor:
    """act(gate) * up of an MXFP4 gate/up tensor (gate rows first), in 16 bits."""
    return _scaled(w, x, act, expert, 1, int(activation), out_dtype)


def mx_moe_into(w: MxWeight, x, route, out: torch.Tensor, act: str = "MXFP6", routed: bool = False, glu: bool = False, activation: int = L.GLU_SILU,
                slot: torch.Tensor | None = None) -> torch.Tensor:
    """The rows out[t, r] of the pairs whose expert `w` holds: expert e is the pool's slot[e] (device int32, -1 for the experts of other
    pools, whose rows are left as they are), or e itself without `slot`; rows of ids that are none become zeros."""
    K, T, R = w.neuron_len, route.tokens, route.routes
    kind, x2, xd, ldx, xs, M, _ = _operand(x, K, act)
    if M != (T * R if routed else T):
        raise ValueError(f"MoE activations must be [{'tokens * routes' if routed else 'tokens'}, K]: {M} rows for {T} tokens of {R} routes")
    if slot is None and w.n_experts != route.n_experts:
        raise ValueError(f"{w.n_experts} experts, a route plan for {route.n_experts}")
    if slot is not None and (slot.dtype != torch.int32 or slot.numel() != route.n_experts or not slot.is_contiguous()):
        raise ValueError("expert slots must be int32 [experts] side by side")
    yd = _result_dtype(w, w.out, glu, out.dtype)
    laid = w.laid_scales()
    width = w.out // 2 if glu else w.out
    if tuple(out.shape) != (T, R, width) or not out.is_contiguous():
        raise ValueError(f"MoE results must be contiguous {(T, R, width)}, got {tuple(out.shape)}")
    for t in (x2, w.values, out, route.ids) if slot is None else (x2, w.values, out, route.ids, slot):
        _here(t)
    if T * R:
        lib = L.lib()
        mapped = route.ids_dst is not None
        key = (kind, M, T * R, route.n_experts, mapped, xs is None)
        need = w._needs.get(key)
        if need is None:
            need = w.note_need(key, lib.mfq_hip_mx_moe_workspace_bytes(kind, K, M, T * R, route.n_experts, mapped, xs is not None))
        ws = borrow(need, x2.device)
        L.check(lib.mfq_hip_mx_moe_matmul(w.values.data_ptr(), laid.data_ptr(), w.rows, K, w.out, _ptr(slot), route.n_experts, kind, x2.data_ptr(), xd,
                                          ldx, _ptr(xs), int(routed), route.ids.data_ptr(), T, R, _ptr(route.ids_dst) if mapped else None,
                                          _ptr(route.expert_bounds) if mapped else None, int(glu), int(activation), out.data_ptr(), yd, width, _ptr(ws),
                                          need if ws is not None else 0, _stream()))
    return out


def _moe_out(w: MxWeight, route, width: int, out_dtype) -> torch.Tensor:
    _out_dtype(out_dtype)
    return torch.empty((route.tokens, route.routes, width), dtype=out_dtype, device=w.values.device)


def mx_moe_matmul(w: MxWeight, x, route, act: str = "MXFP6", routed: bool = False, out_dtype=torch.float32) -> torch.Tensor:
    """[tokens, routes, out] of a pool of MXFP4 experts: every (token, route) pair of `route` (build_moe_route_plan) against its expert;
    zeros where the id is none.  x has a row per token, with `routed` one per pair; quantised to `act` by the call, or MxRows."""
    return mx_moe_into(w, x, route, _moe_out(w, route, w.out, out_dtype), act, routed)


def mx_moe_glu(w: MxWeight, x, route, act: str = "MXFP6", activation: int = L.GLU_SILU, routed: bool = False, out_dtype=torch.bfloat16) -> torch.Tensor:
    """act(gate) * up of a pool of gate/up tensors, 16-bit [tokens, routes, out / 2]."""
    return mx_moe_into(w, x, route, _moe_out(w, route, w.out // 2, out_dtype), act, routed, True, activation)
