"""Dense layers beside the packed experts: gated feed-forward blocks and 8-bit integer linears.

A MoE checkpoint packs its routed experts to int4 and leaves other layers alone: the dense blocks in
front, a shared expert kept in 16 bits, linears in the "int-quantized" 8-bit form.

    gated_ffn(x, w_gate, w_up, w_down, act)     y = (act(x Wg^T) * (x Wu^T)) Wd^T, bf16 / fp16, with
                                                gradients for x and the three weights
    quantize_int8(x)                            int8 codes and one scale per token
    int8_linear(codes, scale, weight, weight_scale, bias, dtype)
                                                int8 product with a scale per token and per output
                                                channel
    int8_gated_ffn(x, w_gate, gate_scale, ...)  the gated block on int8 weights, activations
                                                quantised per token inside

All run on the calling device's current stream, allocate through torch, and never synchronise --
except `check=True`, which reads the call's device error flags afterwards and raises RuntimeError
when a device-side wait ran out.  They may be captured in a CUDA graph.
"""
from __future__ import annotations

import ctypes

import torch

from . import _lib

ACTIVATIONS = {"silu": 0, "gelu_tanh": 1}
_FLOATS = (torch.bfloat16, torch.float16, torch.float32)


def _act_code(act: str, what: str) -> int:
    code = ACTIVATIONS.get(act)
    if code is None:
        raise NotImplementedError(f"{what}: activation {act!r} (one of {', '.join(ACTIVATIONS)})")
    return code


def _rows(x: torch.Tensor, unit: int) -> torch.Tensor:
    """x as [tokens, width] rows that start on 16-byte boundaries (`unit` elements): a view where the
    strides allow it, else a copy."""
    x = x.reshape(-1, x.shape[-1])
    if x.stride(1) != 1 or x.data_ptr() % 16 or (x.shape[0] > 1 and (x.stride(0) % unit or x.stride(0) < x.shape[1])):
        x = x.clone(memory_format=torch.contiguous_format)
    return x


def _stride(x: torch.Tensor) -> int:
    return x.stride(0) if x.shape[0] > 1 else x.shape[1]


def _aligned(w: torch.Tensor) -> torch.Tensor:
    w = w.contiguous()
    return w.clone() if w.data_ptr() % 16 else w


def _check_ffn(x, w_gate, w_up, w_down, what: str) -> None:
    if x.dim() < 1 or w_gate.dim() != 2 or w_up.shape != w_gate.shape or w_down.shape != w_gate.shape[::-1]:
        raise ValueError(f"{what}: weights {tuple(w_gate.shape)}, {tuple(w_up.shape)}, {tuple(w_down.shape)} "
                         "are not [inter, hidden], [inter, hidden], [hidden, inter]")
    if x.shape[-1] != w_gate.shape[1]:
        raise ValueError(f"{what}: x {tuple(x.shape)} does not fit hidden {w_gate.shape[1]}")


def _output(out, shape, dtype, dev, what: str) -> torch.Tensor:
    """`out` checked, or a new tensor."""
    if out is None:
        return torch.empty(shape, dtype=dtype, device=dev)
    if out.shape != torch.Size(shape) or out.dtype != dtype:
        raise ValueError(f"{what}: out {tuple(out.shape)} {out.dtype}, expected {tuple(shape)} {dtype}")
    if not out.is_contiguous() and (out.dim() != 2 or out.stride(1) != 1 or out.stride(0) < out.shape[1]):
        raise ValueError(f"{what}: out must be contiguous, or a 2-D view with unit column stride")
    return out


def _flags(dev, check: bool) -> "torch.Tensor | None":
    return torch.zeros(1, dtype=torch.int32, device=dev) if check else None


def _raise_on(flags: "torch.Tensor | None", what: str) -> None:
    if flags is not None and (v := int(flags.item())):
        raise RuntimeError(f"{what}: device error flags {v:#x} (a device-side wait ran out); the output is not valid")


# ── gated feed-forward, 16-bit ───────────────────────────────────────────────────────────────


def _ffn_call(x, w_gate, w_up, w_down, act: int) -> _lib.FfnCall:
    c = _lib.FfnCall()
    c.act_dtype, c.activation = _lib.DTYPE_CODE[x.dtype], act
    c.n_tokens, c.hidden, c.inter = x.shape[0], x.shape[1], w_gate.shape[0]
    c.x, c.x_row_stride = x.data_ptr(), _stride(x)
    c.w_gate, c.w_up, c.w_down = w_gate.data_ptr(), w_up.data_ptr(), w_down.data_ptr()
    return c


def _run_ffn(c: _lib.FfnCall, backward: bool, dev) -> None:
    lib = _lib.lib()
    what = "gated_ffn backward" if backward else "gated_ffn"
    with torch.cuda.device(dev):
        c.workspace_bytes = lib.vy_gated_ffn_workspace_size(ctypes.byref(c), int(backward))
        ws = torch.empty(c.workspace_bytes, dtype=torch.uint8, device=dev)
        c.workspace = ws.data_ptr()
        fn = lib.vy_gated_ffn_backward if backward else lib.vy_gated_ffn_forward
        _lib.check(fn(ctypes.byref(c), _lib.stream_of(dev)), what)


def _ffn_forward(x, w_gate, w_up, w_down, act: int, out, save: bool, check: bool):
    """(out [T, hidden], saved or None) for 2-D rows x."""
    dev = x.device
    c = _ffn_call(x, w_gate, w_up, w_down, act)
    c.out, c.out_row_stride = out.data_ptr(), _stride(out)
    saved = None
    if save:
        saved = torch.empty(_lib.lib().vy_gated_ffn_saved_floats(c.n_tokens, c.inter), dtype=torch.float32, device=dev)
        c.saved = saved.data_ptr()
    flags = _flags(dev, check)
    c.flags = _lib.ptr(flags)
    _run_ffn(c, False, dev)
    _raise_on(flags, "gated_ffn")
    return saved


class _GatedFfn(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, w_gate, w_up, w_down, act, check):
        rows, wg, wu, wd = _rows(x, 8), _aligned(w_gate), _aligned(w_up), _aligned(w_down)
        out = torch.empty(rows.shape[0], wd.shape[0], dtype=x.dtype, device=x.device)
        saved = _ffn_forward(rows, wg, wu, wd, act, out, True, check)
        ctx.save_for_backward(x, w_gate, w_up, w_down, saved)
        ctx.act, ctx.check = act, check
        return out.view(x.shape)

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, d_out):
        x, w_gate, w_up, w_down, saved = ctx.saved_tensors
        rows, dy = _rows(x, 8), _rows(d_out, 8)
        wg, wu, wd = _aligned(w_gate), _aligned(w_up), _aligned(w_down)
        c = _ffn_call(rows, wg, wu, wd, ctx.act)
        c.saved = saved.data_ptr()
        c.d_out, c.d_out_row_stride = dy.data_ptr(), _stride(dy)
        grads = [torch.empty(t.shape, dtype=t.dtype, device=t.device) if need else None
                 for t, need in zip((rows, wg, wu, wd), ctx.needs_input_grad)]
        c.d_x, c.d_w_gate, c.d_w_up, c.d_w_down = map(_lib.ptr, grads)
        c.d_x_row_stride = rows.shape[1]
        flags = _flags(x.device, ctx.check)
        c.flags = _lib.ptr(flags)
        _run_ffn(c, True, x.device)
        _raise_on(flags, "gated_ffn backward")
        if grads[0] is not None:
            grads[0] = grads[0].view(x.shape)
        return (*grads, None, None)


def gated_ffn(x: torch.Tensor, w_gate: torch.Tensor, w_up: torch.Tensor, w_down: torch.Tensor,
              act: str = "silu", out: "torch.Tensor | None" = None, *, check: bool = False) -> torch.Tensor:
    """y = (act(x Wg^T) * (x Wu^T)) Wd^T.

    x [..., hidden]; w_gate, w_up [inter, hidden]; w_down [hidden, inter]; all bf16 or all fp16,
    hidden and inter multiples of 8; act "silu" or "gelu_tanh".  Returns [..., hidden] in x's type
    (`out`, when given, receives it).  Sums are fp32; h = act(g) * u is rounded once, as the second
    product's operand.  Differentiable once in x and the weights: with gradients on, the call keeps g
    and u (8 bytes per token and intermediate channel) for the backward pass; `out` is refused then.
    Rows of x may be strided; rows or weights that do not start on 16-byte boundaries are copied."""
    what = "gated_ffn"
    code = _act_code(act, what)
    _check_ffn(x, w_gate, w_up, w_down, what)
    if x.dtype not in (torch.bfloat16, torch.float16) or any(w.dtype != x.dtype for w in (w_gate, w_up, w_down)):
        raise NotImplementedError(f"{what}: x {x.dtype}, weights {w_gate.dtype}, {w_up.dtype}, {w_down.dtype} "
                                  "(all bf16 or all fp16)")
    if x.shape[-1] % 8 or w_gate.shape[0] % 8:
        raise NotImplementedError(f"{what}: hidden {x.shape[-1]} and inter {w_gate.shape[0]} must be multiples of 8")
    dev = _lib.require_cuda(x, w_gate, w_up, w_down, out, what=what)
    if torch.is_grad_enabled() and any(t.requires_grad for t in (x, w_gate, w_up, w_down)):
        if out is not None:
            raise RuntimeError(f"{what}: out= with gradients")
        return _GatedFfn.apply(x, w_gate, w_up, w_down, code, check)
    rows = _rows(x, 8)
    y = _output(out, x.shape, x.dtype, dev, what)
    flat = y.view(-1, x.shape[-1]) if y.is_contiguous() else y
    if flat.data_ptr() % 16 or (flat.shape[0] > 1 and flat.stride(0) % 8):
        raise ValueError(f"{what}: out rows must start on 16-byte boundaries")
    _ffn_forward(rows, _aligned(w_gate), _aligned(w_up), _aligned(w_down), code, flat, False, check)
    return y


# ── int8 ─────────────────────────────────────────────────────────────────────────────────────


def quantize_int8(x: torch.Tensor) -> tuple:
    """(codes int8 [..., K], scale fp32 [..., 1]): one scale per row of x (bf16 / fp16 / fp32, any K).

    scale = amax(|x|) / 127 rounded to fp32; code = the nearest integer of the exact quotient
    x / scale (ties to even), so the codes do not depend on how the division is carried out.  A zero
    row has codes 0 and scale 0; a row with an infinity or NaN has codes 0 and scale NaN."""
    what = "quantize_int8"
    if x.dtype not in _FLOATS:
        raise NotImplementedError(f"{what}: x dtype {x.dtype} (bf16, fp16 or fp32)")
    if x.dim() < 1 or x.shape[-1] == 0:
        raise ValueError(f"{what}: x {tuple(x.shape)} has no values in a row")
    dev = _lib.require_cuda(x, what=what)
    rows = x.reshape(-1, x.shape[-1])
    if rows.stride(1) != 1:
        rows = rows.contiguous()
    codes = torch.empty(x.shape, dtype=torch.int8, device=dev)
    scale = torch.empty(*x.shape[:-1], 1, dtype=torch.float32, device=dev)
    with torch.cuda.device(dev):
        _lib.check(_lib.lib().vy_int8_quantize(rows.data_ptr(), _lib.DTYPE_CODE[x.dtype], _stride(rows), rows.shape[0],
                                               rows.shape[1], codes.data_ptr(), scale.data_ptr(), _lib.stream_of(dev)),
                   what)
    return codes, scale


def _scales(scale: torch.Tensor, n: int, what: str) -> torch.Tensor:
    if scale.numel() != n or not scale.is_floating_point():
        raise ValueError(f"{what}: {tuple(scale.shape)} {scale.dtype} scales for {n} rows")
    return scale.reshape(-1).to(torch.float32).contiguous()


def _int8(t: torch.Tensor, what: str) -> None:
    if t.dtype != torch.int8:
        raise NotImplementedError(f"{what}: codes of dtype {t.dtype} (int8)")


def int8_linear(codes: torch.Tensor, scale: torch.Tensor, weight: torch.Tensor, weight_scale: torch.Tensor,
                bias: "torch.Tensor | None" = None, dtype: torch.dtype = torch.bfloat16,
                out: "torch.Tensor | None" = None, *, check: bool = False) -> torch.Tensor:
    """y[..., n] = (sum_k codes[..., k] weight[n, k]) * scale[...] * weight_scale[n] (+ bias[n]).

    codes [..., K] int8 with one scale per row (`quantize_int8`'s pair); weight [N, K] int8 with one
    scale per output channel ([N] or [N, 1]); K a multiple of 16 below 131072, any N.  The sum is
    exact (int32); the scales and the bias are applied in fp32, in that order, and the result is
    rounded once to `dtype` (bf16, fp16 or fp32)."""
    what = "int8_linear"
    _int8(codes, what), _int8(weight, what)
    if codes.dim() < 1 or weight.dim() != 2 or weight.shape[1] != codes.shape[-1]:
        raise ValueError(f"{what}: codes {tuple(codes.shape)} and weight {tuple(weight.shape)}")
    if dtype not in _FLOATS or (bias is not None and bias.dtype not in _FLOATS):
        raise NotImplementedError(f"{what}: dtype {dtype}, bias {None if bias is None else bias.dtype}")
    n, k = weight.shape
    if k % 16 or not 0 < k < 131072 or n == 0:
        raise NotImplementedError(f"{what}: K {k} must be a multiple of 16 below 131072 (N {n})")
    if bias is not None and bias.shape != (n,):
        raise ValueError(f"{what}: bias {tuple(bias.shape)} for {n} output channels")
    dev = _lib.require_cuda(codes, scale, weight, weight_scale, bias, out, what=what)
    rows, w = _rows(codes, 16), _aligned(weight)
    bias = None if bias is None else bias.contiguous()
    sx, sw = _scales(scale, rows.shape[0], what), _scales(weight_scale, n, what)
    y = _output(out, (*codes.shape[:-1], n), dtype, dev, what)
    flat = y.view(-1, n) if y.is_contiguous() else y
    c = _lib.Int8LinearCall()
    c.n_tokens, c.k, c.n = rows.shape[0], rows.shape[1], n
    c.codes, c.codes_row_stride, c.scales = rows.data_ptr(), _stride(rows), sx.data_ptr()
    c.weight, c.weight_scales = w.data_ptr(), sw.data_ptr()
    if bias is not None:
        c.bias, c.bias_dtype = bias.data_ptr(), _lib.DTYPE_CODE[bias.dtype]
    c.out_dtype, c.out, c.out_row_stride = _lib.DTYPE_CODE[dtype], flat.data_ptr(), _stride(flat)
    flags = _flags(dev, check)
    c.flags = _lib.ptr(flags)
    lib = _lib.lib()
    with torch.cuda.device(dev):
        c.workspace_bytes = lib.vy_int8_linear_workspace_size(ctypes.byref(c))
        ws = torch.empty(c.workspace_bytes, dtype=torch.uint8, device=dev) if c.workspace_bytes else None
        c.workspace = _lib.ptr(ws)
        _lib.check(lib.vy_int8_linear(ctypes.byref(c), _lib.stream_of(dev)), what)
    _raise_on(flags, what)
    return y


def int8_gated_ffn(x: torch.Tensor, w_gate: torch.Tensor, gate_scale: torch.Tensor, w_up: torch.Tensor,
                   up_scale: torch.Tensor, w_down: torch.Tensor, down_scale: torch.Tensor, act: str = "silu",
                   out: "torch.Tensor | None" = None, *, check: bool = False) -> torch.Tensor:
    """The gated block on int8 weights with one scale per output channel: x is quantised per token,
    h = act(g) * u stays in fp32 and is quantised per token for the second product.

    x [..., hidden] bf16 or fp16; w_gate, w_up int8 [inter, hidden]; w_down int8 [hidden, inter];
    hidden and inter multiples of 16; scales [rows] or [rows, 1].  Returns [..., hidden] in x's type.
    No gradients."""
    what = "int8_gated_ffn"
    code = _act_code(act, what)
    for w in (w_gate, w_up, w_down):
        _int8(w, what)
    _check_ffn(x, w_gate, w_up, w_down, what)
    if x.dtype not in (torch.bfloat16, torch.float16):
        raise NotImplementedError(f"{what}: x dtype {x.dtype} (bf16 or fp16)")
    if any(d % 16 or not 0 < d < 131072 for d in w_gate.shape):
        raise NotImplementedError(f"{what}: inter and hidden {tuple(w_gate.shape)} must be multiples of 16 below 131072")
    dev = _lib.require_cuda(x, w_gate, gate_scale, w_up, up_scale, w_down, down_scale, out, what=what)
    rows = x.reshape(-1, x.shape[-1])
    if rows.stride(1) != 1:
        rows = rows.contiguous()
    wg, wu, wd = _aligned(w_gate), _aligned(w_up), _aligned(w_down)
    inter, hidden = wg.shape
    sg, su, sd = _scales(gate_scale, inter, what), _scales(up_scale, inter, what), _scales(down_scale, hidden, what)
    y = _output(out, x.shape, x.dtype, dev, what)
    flat = y.view(-1, hidden) if y.is_contiguous() else y
    c = _lib.Int8FfnCall()
    c.act_dtype, c.activation = _lib.DTYPE_CODE[x.dtype], code
    c.n_tokens, c.hidden, c.inter = rows.shape[0], hidden, inter
    c.x, c.x_row_stride = rows.data_ptr(), _stride(rows)
    c.w_gate, c.w_up, c.w_down = wg.data_ptr(), wu.data_ptr(), wd.data_ptr()
    c.gate_scales, c.up_scales, c.down_scales = sg.data_ptr(), su.data_ptr(), sd.data_ptr()
    c.out, c.out_row_stride = flat.data_ptr(), _stride(flat)
    flags = _flags(dev, check)
    c.flags = _lib.ptr(flags)
    lib = _lib.lib()
    with torch.cuda.device(dev):
        c.workspace_bytes = lib.vy_int8_gated_ffn_workspace_size(ctypes.byref(c))
        ws = torch.empty(c.workspace_bytes, dtype=torch.uint8, device=dev)
        c.workspace = ws.data_ptr()
        _lib.check(lib.vy_int8_gated_ffn(ctypes.byref(c), _lib.stream_of(dev)), what)
    _raise_on(flags, what)
    return y
