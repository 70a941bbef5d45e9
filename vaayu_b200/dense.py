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
when a device-side wait ran out (without it such a call's output is unfinished and nobody says so).
They may be captured in a CUDA graph.  Forward-mode derivatives (dual tensors) are refused; `out=`
counts as a write to that tensor and is refused where gradients are wanted.
"""
from __future__ import annotations

import ctypes
import struct
import threading

import torch

from . import _lib

ACTIVATIONS = {"silu": 0, "gelu_tanh": 1}
_BF16, _F16, _F32, _INT8 = torch.bfloat16, torch.float16, torch.float32, torch.int8
_CODE = {_BF16: _lib.BF16, _F16: _lib.F16, _F32: _lib.F32}
_MAX_K = 131072      # an int32 sum of fewer int8 products cannot overflow
_MAX_N = 0x7FFFFF00

# The call structures of include/vaayu_b200.h, packed in one go: a ctypes structure filled field by
# field costs more host time than the launch of a small call.
_FFN = struct.Struct("@iiqiiPqPPPPqPPNPPqPqPPP")
_LINEAR = struct.Struct("@qiiPqPPPPiiPqP")
_INT8_FFN = struct.Struct("@iiqiiPqPPPPPPPqPNP")

_HOST = None
_HOST_LOCK = threading.Lock()
_HOST_ENTRIES = ("vy_last_error", "vy_gated_ffn_saved_floats", "vy_gated_ffn_workspace_size", "vy_gated_ffn_forward",
                 "vy_gated_ffn_backward", "vy_int8_quantize", "vy_int8_linear", "vy_int8_gated_ffn_workspace_size",
                 "vy_int8_gated_ffn")


def _host():
    """The extension that makes ordinary calls (contiguous and aligned operands on the current device)
    without Python in between; it returns None for any other, which the code below takes."""
    global _HOST
    if _HOST is None:
        with _HOST_LOCK:
            if _HOST is None:
                try:
                    from . import _dense_host as host
                except ImportError as e:
                    raise RuntimeError(f"_dense_host does not load ({e}); run `python -m vaayu_b200.build`") from e
                lib = _lib.lib()
                host.bind([ctypes.cast(getattr(lib, n), ctypes.c_void_p).value for n in _HOST_ENTRIES])
                _HOST = host
    return _HOST


_forward_ad = torch.autograd.forward_ad
_current_device = torch._C._cuda_getDevice
_raw_stream = torch._C._cuda_getCurrentRawStream


def _device(what: str, first: torch.Tensor, *others) -> int:
    """The index of the CUDA device all tensors are on; raises as `_lib.require_cuda` does."""
    index = first.get_device()
    for t in others:
        if t is not None and t.get_device() != index:
            index = -1
    if index < 0:
        _lib.require_cuda(first, *others, what=what)      # raises: CPU tensors, or two devices
    return index


def _enqueue(fn, what: str, index: int, *args) -> None:
    """One C call on the device's current stream, with that device current."""
    if index == _current_device():
        status = fn(*args, _raw_stream(index))
    else:
        with torch.cuda.device(index):
            status = fn(*args, _raw_stream(index))
    if status:
        _lib.check(status, what)


def _activation(act: str, what: str) -> int:
    code = ACTIVATIONS.get(act)
    if code is None:
        raise NotImplementedError(f"{what}: activation {act!r} (one of {', '.join(ACTIVATIONS)})")
    return code


def _rows(x: torch.Tensor, unit: int) -> tuple:
    """(x as [tokens, width] with rows that start on 16-byte boundaries (`unit` elements), its row
    stride): a view where the strides allow it, else a copy."""
    if x.is_neg():
        x = x.resolve_neg()
    if x.dim() != 2:
        x = x.reshape(-1, x.shape[-1])
    tokens, width = x.shape
    if x.data_ptr() & 15 == 0:
        row, col = x.stride()
        if tokens <= 1:
            if col == 1 or width == 1:
                return x, -(-width // unit) * unit
        elif col == 1 and row % unit == 0 and row >= width:
            return x, row
    return x.clone(memory_format=torch.contiguous_format), width


def _unit_rows(x: torch.Tensor) -> tuple:
    """(x as [tokens, width] with a unit column stride, its row stride)."""
    if x.is_neg():
        x = x.resolve_neg()
    if x.dim() != 2:
        x = x.reshape(-1, x.shape[-1])
    row, col = x.stride()
    if col != 1:
        x = x.contiguous()
        row = x.shape[1]
    return x, (row if x.shape[0] > 1 else x.shape[1])


def _aligned(w: torch.Tensor) -> torch.Tensor:
    """w itself when it is contiguous and starts on a 16-byte boundary, else a copy that does."""
    if w.is_neg():
        w = w.resolve_neg()
    if not w.is_contiguous():
        return w.contiguous()
    return w.clone() if w.data_ptr() & 15 else w


def _check_ffn(x, w_gate, w_up, w_down, what: str) -> tuple:
    """(hidden, inter) of a block whose operands fit together."""
    shape = w_gate.shape
    if len(shape) == 2 and w_up.shape == shape:
        inter, hidden = shape
        down = w_down.shape
        if len(down) == 2 and down[0] == hidden and down[1] == inter:
            if x.dim() < 1 or x.shape[-1] != hidden:
                raise ValueError(f"{what}: x {tuple(x.shape)} does not fit hidden {hidden}")
            return hidden, inter
    raise ValueError(f"{what}: weights {tuple(shape)}, {tuple(w_up.shape)}, {tuple(w_down.shape)} "
                     "are not [inter, hidden], [inter, hidden], [hidden, inter]")


def _like(x: torch.Tensor) -> torch.Tensor:
    """A new contiguous tensor of x's shape and type.  (empty_like of a contiguous tensor, and new_empty
    with its sizes spelt out, take half the host time of torch.empty with a shape.)"""
    return torch.empty_like(x) if x.is_contiguous() else x.new_empty(x.shape)


def _given(out, shape, dtype, what: str) -> tuple:
    """(the caller's out as [tokens, width], its row stride)."""
    if out.shape != shape or out.dtype != dtype:
        raise ValueError(f"{what}: out {tuple(out.shape)} {out.dtype}, expected {tuple(shape)} {dtype}")
    if out.is_neg():
        raise ValueError(f"{what}: out is a negated view")
    if not out.is_contiguous():
        if out.dim() != 2 or out.stride(1) != 1 or out.stride(0) < out.shape[1]:
            raise ValueError(f"{what}: out must be contiguous, or a 2-D view with unit column stride")
        return out, out.stride(0)
    return out.view(-1, shape[-1]), shape[-1]


def _written(out: torch.Tensor) -> None:
    """Counts up the version of the caller's out: a backward pass that still needs what it held notices."""
    if not out.is_inference():
        torch.autograd.graph.increment_version(out)


_SIZES: dict = {}      # an entry point's sizes -> its workspace bytes


def _remember(key: tuple, size: int) -> int:
    if len(_SIZES) >= 4096:
        _SIZES.clear()
    _SIZES[key] = size
    return size


def _flags(like: torch.Tensor, check: bool) -> "torch.Tensor | None":
    return torch.zeros(1, dtype=torch.int32, device=like.device) if check else None


def _ptr(t: "torch.Tensor | None") -> int:
    return 0 if t is None else t.data_ptr()


def _raise_on(flags: torch.Tensor, what: str) -> None:
    if v := int(flags.item()):
        raise RuntimeError(f"{what}: device error flags {v:#x} (a device-side wait ran out); the output is not valid")


def _no_tangents(what: str, *tensors) -> None:
    """Refuses dual tensors: the kernels would drop their tangents, a derivative of zero."""
    if _forward_ad._current_level < 0:      # no dual tensors now (asked by hand: unpack_dual costs 1 us a tensor)
        return
    for t in tensors:
        if t is not None and t.is_floating_point() and _forward_ad.unpack_dual(t).tangent is not None:
            raise NotImplementedError(f"{what}: no forward-mode derivatives (an operand is a dual tensor)")


def _undifferentiable(results: tuple, message: bytes) -> tuple:
    """The results (None among them), with a node behind them that raises `message` in a backward pass."""
    given = [t.detach().requires_grad_(True) for t in results if t is not None]
    if not given:
        return results
    marked = torch._C._functions.DelayedError(message, len(given))(*given)
    marked = iter(marked if isinstance(marked, tuple) else (marked,))
    return tuple(t if t is None else next(marked) for t in results)


# ── gated feed-forward, 16-bit ───────────────────────────────────────────────────────────────


def _ffn_workspace(tokens: int, hidden: int, inter: int, backward: int) -> int:
    key = (tokens, hidden, inter, backward)
    size = _SIZES.get(key)
    if size is None:
        call = _FFN.pack(0, 0, tokens, hidden, inter, *(0,) * 18)
        size = _remember(key, _lib.lib().vy_gated_ffn_workspace_size(call, backward))
    return size


def _ffn_saved(tokens: int, inter: int) -> int:
    key = (tokens, inter)
    return _SIZES.get(key) or _remember(key, _lib.lib().vy_gated_ffn_saved_floats(tokens, inter))


def _ffn_forward(x, w_gate, w_up, w_down, hidden: int, inter: int, act: int, flat, out_stride: int, index: int,
                 save: bool, check: bool):
    """The forward call into `flat`; returns what the backward pass needs when `save`."""
    rows, x_stride = _rows(x, 8)
    wg, wu, wd = _aligned(w_gate), _aligned(w_up), _aligned(w_down)
    tokens = rows.shape[0]
    lib = _lib.lib()
    size = _ffn_workspace(tokens, hidden, inter, 0)
    ws = rows.new_empty((size + 1) // 2)
    saved = rows.new_empty(_ffn_saved(tokens, inter), dtype=_F32) if save else None
    flags = _flags(rows, check)
    call = _FFN.pack(_CODE[rows.dtype], act, tokens, hidden, inter, rows.data_ptr(), x_stride, wg.data_ptr(),
                     wu.data_ptr(), wd.data_ptr(), flat.data_ptr(), out_stride, _ptr(saved), ws.data_ptr(), size,
                     _ptr(flags), 0, 0, 0, 0, 0, 0, 0)
    _enqueue(lib.vy_gated_ffn_forward, "gated_ffn", index, call)
    if check:
        _raise_on(flags, "gated_ffn")
    return saved


def _ffn_backward(ctx, d_out):
    x, w_gate, w_up, w_down, saved = ctx.saved_tensors
    # what a hook on saved tensors gives back, or a node called by hand is given, may be anything
    what, dtype = "gated_ffn backward", x.dtype
    hidden, inter = _check_ffn(x, w_gate, w_up, w_down, what)
    _device(what, x, w_gate, w_up, w_down, saved, d_out)
    _no_tangents(what, x, w_gate, w_up, w_down, saved, d_out)
    if (dtype not in (_BF16, _F16) or not (w_gate.dtype is w_up.dtype is w_down.dtype is d_out.dtype is dtype)
            or saved.dtype is not _F32):
        raise NotImplementedError(f"{what}: {x.dtype}, {w_gate.dtype}, {w_up.dtype}, {w_down.dtype}, {saved.dtype}, "
                                  f"{d_out.dtype}")
    if d_out.shape != x.shape or saved.numel() != _ffn_saved(x.numel() // hidden, inter):
        raise ValueError(f"{what}: tensors of other sizes than the forward call's")
    saved = _aligned(saved)
    (rows, x_stride), (dy, dy_stride) = _rows(x, 8), _rows(d_out, 8)
    wg, wu, wd = _aligned(w_gate), _aligned(w_up), _aligned(w_down)
    tokens = rows.shape[0]
    need = ctx.needs_input_grad
    grads = [_like(t) if n else None for t, n in zip((x, w_gate, w_up, w_down), need)]
    size = _ffn_workspace(tokens, hidden, inter, 1)
    ws, flags = rows.new_empty((size + 1) // 2), _flags(rows, ctx.check)
    call = _FFN.pack(_CODE[rows.dtype], ctx.act, tokens, hidden, inter, rows.data_ptr(), x_stride,
                     wg.data_ptr(), wu.data_ptr(), wd.data_ptr(), 0, 0, saved.data_ptr(), ws.data_ptr(), size,
                     _ptr(flags), dy.data_ptr(), dy_stride, _ptr(grads[0]), hidden, *map(_ptr, grads[1:]))
    _enqueue(_lib.lib().vy_gated_ffn_backward, what, x.get_device(), call)
    if ctx.check:
        _raise_on(flags, what)
    return (*grads, None, None)


class _GatedFfn(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, w_gate, w_up, w_down, act, check):
        inter, hidden = w_gate.shape
        out = _like(x)
        saved = _ffn_forward(x, w_gate, w_up, w_down, hidden, inter, act, out, hidden, x.get_device(), True, check)
        ctx.save_for_backward(x, w_gate, w_up, w_down, saved)
        ctx.act, ctx.check = act, check
        return out

    @staticmethod
    def backward(ctx, d_out):
        if not torch.is_grad_enabled():
            return _ffn_backward(ctx, d_out)
        # create_graph: the gradients depend on x and the weights even where d_out does not require
        # gradients (a sum's does not), so they are marked whatever d_out is
        with torch.no_grad():
            grads = _ffn_backward(ctx, d_out)
        return _undifferentiable(grads, b"trying to differentiate twice a function that was marked with "
                                        b"@once_differentiable")


def gated_ffn(x: torch.Tensor, w_gate: torch.Tensor, w_up: torch.Tensor, w_down: torch.Tensor,
              act: str = "silu", out: "torch.Tensor | None" = None, *, check: bool = False) -> torch.Tensor:
    """y = (act(x Wg^T) * (x Wu^T)) Wd^T.

    x [..., hidden]; w_gate, w_up [inter, hidden]; w_down [hidden, inter]; all bf16 or all fp16,
    hidden and inter multiples of 8; act "silu" or "gelu_tanh".  Returns [..., hidden] in x's type
    (`out`, when given, receives it).  Sums are fp32.  h = act(g) * u is the second product's operand:
    rounded once to x's type, or up to 32 tokens to a sum of two such values; in fp16 an h beyond 65504
    is infinite (dg and du likewise), and its token's result not finite.  Differentiable once in x and the weights: with gradients on, the call keeps g
    and u (8 bytes per token and intermediate channel) for the backward pass; `out` is refused then.
    Rows of x may be strided; rows or weights that do not start on 16-byte boundaries are copied."""
    what = "gated_ffn"
    code = _activation(act, what)
    if out is None and not check and (y := (_HOST or _host()).gated_ffn(x, w_gate, w_up, w_down, code)) is not None:
        return y
    hidden, inter = _check_ffn(x, w_gate, w_up, w_down, what)
    dtype = x.dtype
    if (dtype is not _BF16 and dtype is not _F16) or not (w_gate.dtype is w_up.dtype is w_down.dtype is dtype):
        raise NotImplementedError(f"{what}: x {dtype}, weights {w_gate.dtype}, {w_up.dtype}, {w_down.dtype} "
                                  "(all bf16 or all fp16)")
    if hidden % 8 or inter % 8 or not hidden or not inter:
        raise NotImplementedError(f"{what}: hidden {hidden} and inter {inter} must be multiples of 8")
    index = _device(what, x, w_gate, w_up, w_down, out)
    _no_tangents(what, x, w_gate, w_up, w_down, out)
    if torch.is_grad_enabled() and (x.requires_grad or w_gate.requires_grad or w_up.requires_grad
                                    or w_down.requires_grad or (out is not None and out.requires_grad)):
        if out is not None:
            raise RuntimeError(f"{what}: out= with gradients")
        return _GatedFfn.apply(x, w_gate, w_up, w_down, code, check)
    if out is None:
        out, stride = _like(x), hidden
        flat = out                      # contiguous: only its address is used
    else:
        flat, stride = _given(out, x.shape, dtype, what)
        if flat.data_ptr() & 15 or stride % 8:
            raise ValueError(f"{what}: out rows must start on 16-byte boundaries")
        _written(out)
    _ffn_forward(x, w_gate, w_up, w_down, hidden, inter, code, flat, stride, index, False, check)
    return out


# ── int8 ─────────────────────────────────────────────────────────────────────────────────────


def _cut_off(what: str, out, *tensors) -> bool:
    """Whether gradients are wanted for an operand of a call that has none; its result is then marked
    (`_undifferentiable`) instead of dropping out of the graph without a word."""
    if torch.is_grad_enabled():
        for t in (out, *tensors):
            if t is not None and t.requires_grad:
                if out is not None:
                    raise RuntimeError(f"{what}: out= with gradients")
                return True
    return False


def quantize_int8(x: torch.Tensor) -> tuple:
    """(codes int8 [..., K], scale fp32 [..., 1]): one scale per row of x (bf16 / fp16 / fp32, any K).

    scale = amax(|x|) / 127 rounded to fp32; code = the nearest integer of the exact quotient
    x / scale (ties to even), so the codes do not depend on how the division is carried out.  A zero
    row has codes 0 and scale 0; a row with an infinity or NaN has codes 0 and scale NaN.  No gradients:
    a backward pass through the scale raises."""
    pair = (_HOST or _host()).quantize_int8(x)
    if pair is not None:
        return pair
    what = "quantize_int8"
    code = _CODE.get(x.dtype)
    if code is None:
        raise NotImplementedError(f"{what}: x dtype {x.dtype} (bf16, fp16 or fp32)")
    shape = x.shape
    if not shape or shape[-1] == 0:
        raise ValueError(f"{what}: x {tuple(shape)} has no values in a row")
    index = _device(what, x)
    _no_tangents(what, x)
    rows, stride = _unit_rows(x)
    tokens, width = rows.shape
    codes = torch.empty_like(x, dtype=_INT8) if x.is_contiguous() else x.new_empty(shape, dtype=_INT8)
    scale = x.new_empty(tokens, 1, dtype=_F32) if len(shape) == 2 else x.new_empty((*shape[:-1], 1), dtype=_F32)
    _enqueue(_lib.lib().vy_int8_quantize, what, index, rows.data_ptr(), code, stride, tokens, width,
             codes.data_ptr(), scale.data_ptr())
    if _cut_off(what, None, x):
        scale, = _undifferentiable((scale,), b"quantize_int8 has no gradients")
    return codes, scale


def _scales(scale: torch.Tensor, n: int, what: str) -> torch.Tensor:
    if scale.numel() != n or not scale.is_floating_point():
        raise ValueError(f"{what}: {tuple(scale.shape)} {scale.dtype} scales for {n} rows")
    if scale.is_neg():
        scale = scale.resolve_neg()
    if scale.dtype is not _F32:
        scale = scale.to(_F32)
    return scale if scale.is_contiguous() else scale.contiguous()


def int8_linear(codes: torch.Tensor, scale: torch.Tensor, weight: torch.Tensor, weight_scale: torch.Tensor,
                bias: "torch.Tensor | None" = None, dtype: torch.dtype = torch.bfloat16,
                out: "torch.Tensor | None" = None, *, check: bool = False) -> torch.Tensor:
    """y[..., n] = (sum_k codes[..., k] weight[n, k]) * scale[...] * weight_scale[n] (+ bias[n]).

    codes [..., K] int8 with one scale per row (`quantize_int8`'s pair); weight [N, K] int8 with one
    scale per output channel ([N] or [N, 1]); K a multiple of 16 below 131072, any N.  The sum is
    exact (int32); the scales and the bias are applied in fp32, in that order, and the result is
    rounded once to `dtype` (bf16, fp16 or fp32).  No gradients: a backward pass through it raises."""
    what = "int8_linear"
    if out is None and not check:
        y = (_HOST or _host()).int8_linear(codes, scale, weight, weight_scale, bias, _CODE.get(dtype, -1))
        if y is not None:
            return y
    if codes.dtype is not _INT8 or weight.dtype is not _INT8:
        raise NotImplementedError(f"{what}: codes {codes.dtype}, weight {weight.dtype} (int8)")
    shape = codes.shape
    if not shape or weight.dim() != 2 or weight.shape[1] != shape[-1]:
        raise ValueError(f"{what}: codes {tuple(codes.shape)} and weight {tuple(weight.shape)}")
    out_code = _CODE.get(dtype)
    if out_code is None or (bias is not None and bias.dtype not in _CODE):
        raise NotImplementedError(f"{what}: dtype {dtype}, bias {None if bias is None else bias.dtype}")
    n, k = weight.shape
    if k % 16 or not 0 < k < _MAX_K or not 0 < n <= _MAX_N:
        raise NotImplementedError(f"{what}: K {k} must be a multiple of 16 below {_MAX_K}, N {n} up to {_MAX_N}")
    bias_code = 0
    if bias is not None:
        if bias.dim() != 1 or bias.shape[0] != n:
            raise ValueError(f"{what}: bias {tuple(bias.shape)} for {n} output channels")
        bias, bias_code = bias.resolve_neg().contiguous(), _CODE[bias.dtype]
    index = _device(what, codes, scale, weight, weight_scale, bias, out)
    _no_tangents(what, scale, weight_scale, bias, out)
    cut = _cut_off(what, out, scale, weight_scale, bias)
    (rows, stride), w = _rows(codes, 16), _aligned(weight)
    tokens = rows.shape[0]
    sx, sw = _scales(scale, tokens, what), _scales(weight_scale, n, what)
    if out is None:
        out = codes.new_empty(tokens, n, dtype=dtype) if len(shape) == 2 else codes.new_empty((*shape[:-1], n), dtype=dtype)
        flat, out_stride = out, n
    else:
        flat, out_stride = _given(out, (*shape[:-1], n), dtype, what)
        _written(out)
    flags = _flags(codes, check)
    call = _LINEAR.pack(tokens, k, n, rows.data_ptr(), stride, sx.data_ptr(), w.data_ptr(), sw.data_ptr(),
                        _ptr(bias), bias_code, out_code, flat.data_ptr(), out_stride, _ptr(flags))
    _enqueue(_lib.lib().vy_int8_linear, what, index, call)
    if check:
        _raise_on(flags, what)
    return _undifferentiable((out,), b"int8_linear has no gradients")[0] if cut else out


def _int8_ffn_workspace(tokens: int, hidden: int, inter: int) -> int:
    key = ("int8", tokens, hidden, inter)
    size = _SIZES.get(key)
    if size is None:
        call = _INT8_FFN.pack(0, 0, tokens, hidden, inter, *(0,) * 13)
        size = _remember(key, _lib.lib().vy_int8_gated_ffn_workspace_size(call))
    return size


def int8_gated_ffn(x: torch.Tensor, w_gate: torch.Tensor, gate_scale: torch.Tensor, w_up: torch.Tensor,
                   up_scale: torch.Tensor, w_down: torch.Tensor, down_scale: torch.Tensor, act: str = "silu",
                   out: "torch.Tensor | None" = None, *, check: bool = False) -> torch.Tensor:
    """The gated block on int8 weights with one scale per output channel: x is quantised per token,
    h = act(g) * u stays in fp32 and is quantised per token for the second product.

    x [..., hidden] bf16 or fp16; w_gate, w_up int8 [inter, hidden]; w_down int8 [hidden, inter];
    hidden and inter multiples of 16; scales [rows] or [rows, 1].  Returns [..., hidden] in x's type.
    No gradients: a backward pass through it raises."""
    what = "int8_gated_ffn"
    code = _activation(act, what)
    if out is None and not check:
        y = (_HOST or _host()).int8_gated_ffn(x, w_gate, gate_scale, w_up, up_scale, w_down, down_scale, code)
        if y is not None:
            return y
    if not (w_gate.dtype is w_up.dtype is w_down.dtype is _INT8):
        raise NotImplementedError(f"{what}: weights {w_gate.dtype}, {w_up.dtype}, {w_down.dtype} (int8)")
    hidden, inter = _check_ffn(x, w_gate, w_up, w_down, what)
    dtype = x.dtype
    if dtype is not _BF16 and dtype is not _F16:
        raise NotImplementedError(f"{what}: x dtype {dtype} (bf16 or fp16)")
    if hidden % 16 or inter % 16 or not 0 < hidden < _MAX_K or not 0 < inter < _MAX_K:
        raise NotImplementedError(f"{what}: hidden {hidden} and inter {inter} must be multiples of 16 below {_MAX_K}")
    index = _device(what, x, w_gate, gate_scale, w_up, up_scale, w_down, down_scale, out)
    _no_tangents(what, x, gate_scale, up_scale, down_scale, out)
    cut = _cut_off(what, out, x, gate_scale, up_scale, down_scale)
    (rows, stride), wg, wu, wd = _unit_rows(x), _aligned(w_gate), _aligned(w_up), _aligned(w_down)
    if stride < hidden:      # rows on top of one another (an expanded row)
        rows, stride = rows.contiguous(), hidden
    sg, su, sd = _scales(gate_scale, inter, what), _scales(up_scale, inter, what), _scales(down_scale, hidden, what)
    if out is None:
        out, out_stride = _like(x), hidden
        flat = out
    else:
        flat, out_stride = _given(out, x.shape, dtype, what)
        _written(out)
    tokens = rows.shape[0]
    size = _int8_ffn_workspace(tokens, hidden, inter)
    ws, flags = rows.new_empty((size + 1) // 2), _flags(rows, check)
    call = _INT8_FFN.pack(_CODE[dtype], code, tokens, hidden, inter, rows.data_ptr(), stride, wg.data_ptr(),
                          wu.data_ptr(), wd.data_ptr(), sg.data_ptr(), su.data_ptr(), sd.data_ptr(), flat.data_ptr(),
                          out_stride, ws.data_ptr(), size, _ptr(flags))
    _enqueue(_lib.lib().vy_int8_gated_ffn, what, index, call)
    if check:
        _raise_on(flags, what)
    return _undifferentiable((out,), b"int8_gated_ffn has no gradients")[0] if cut else out
