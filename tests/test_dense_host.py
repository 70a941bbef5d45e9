"""Dense operators without a GPU: refusals of the Python entry points and of the C ABI (nothing is
launched: every call fails in its argument checks), structure layouts, workspace sizes."""
import ctypes
import subprocess
from pathlib import Path

import pytest
import torch

import vaayu_b200 as vb
from vaayu_b200 import _lib, dense

HEADER = Path(__file__).resolve().parent.parent / "include" / "vaayu_b200.h"
BF16 = torch.bfloat16


def ffn_args(hidden=16, inter=32, dtype=BF16, tokens=2):
    return (torch.zeros(tokens, hidden, dtype=dtype), torch.zeros(inter, hidden, dtype=dtype),
            torch.zeros(inter, hidden, dtype=dtype), torch.zeros(hidden, inter, dtype=dtype))


def test_gated_ffn_refuses_what_it_does_not_take():
    x, wg, wu, wd = ffn_args()
    with pytest.raises(NotImplementedError, match="activation"):
        vb.gated_ffn(x, wg, wu, wd, act="relu")
    with pytest.raises(ValueError, match="are not"):
        vb.gated_ffn(x, wg, wu[:16], wd)
    with pytest.raises(ValueError, match="are not"):
        vb.gated_ffn(x, wg, wu, wd.T)
    with pytest.raises(ValueError, match="does not fit"):
        vb.gated_ffn(x[:, :8], wg, wu, wd)
    with pytest.raises(NotImplementedError, match="all bf16 or all fp16"):
        vb.gated_ffn(x.half(), wg, wu, wd)
    with pytest.raises(NotImplementedError, match="all bf16 or all fp16"):
        vb.gated_ffn(*ffn_args(dtype=torch.float32))
    with pytest.raises(NotImplementedError, match="multiples of 8"):
        vb.gated_ffn(*ffn_args(hidden=12))
    with pytest.raises(NotImplementedError, match="multiples of 8"):
        vb.gated_ffn(*ffn_args(inter=20))
    with pytest.raises(RuntimeError, match="CUDA tensors only"):
        vb.gated_ffn(x, wg, wu, wd)


def test_quantize_int8_refuses_what_it_does_not_take():
    with pytest.raises(NotImplementedError, match="dtype"):
        vb.quantize_int8(torch.zeros(2, 4, dtype=torch.float64))
    with pytest.raises(ValueError, match="no values"):
        vb.quantize_int8(torch.zeros(2, 0))
    with pytest.raises(RuntimeError, match="CUDA tensors only"):
        vb.quantize_int8(torch.zeros(2, 4))


def int8_args(k=32, n=5, tokens=2):
    return (torch.zeros(tokens, k, dtype=torch.int8), torch.zeros(tokens, 1),
            torch.zeros(n, k, dtype=torch.int8), torch.zeros(n))


def test_int8_linear_refuses_what_it_does_not_take():
    codes, scale, w, ws = int8_args()
    with pytest.raises(NotImplementedError, match="int8"):
        vb.int8_linear(codes.float(), scale, w, ws)
    with pytest.raises(NotImplementedError, match="int8"):
        vb.int8_linear(codes, scale, w.to(torch.uint8), ws)
    with pytest.raises(ValueError, match="codes"):
        vb.int8_linear(codes[:, :16], scale, w, ws)
    with pytest.raises(NotImplementedError, match="dtype"):
        vb.int8_linear(codes, scale, w, ws, dtype=torch.float64)
    with pytest.raises(NotImplementedError, match="multiple of 16"):
        vb.int8_linear(*int8_args(k=24))
    with pytest.raises(NotImplementedError, match="multiple of 16"):
        vb.int8_linear(*int8_args(k=131072, n=1, tokens=1))
    with pytest.raises(ValueError, match="bias"):
        vb.int8_linear(codes, scale, w, ws, bias=torch.zeros(4))
    with pytest.raises(RuntimeError, match="CUDA tensors only"):
        vb.int8_linear(codes, scale, w, ws)


def test_int8_gated_ffn_refuses_what_it_does_not_take():
    x, wg, wu, wd = ffn_args()
    q = [w.to(torch.int8) for w in (wg, wu, wd)]
    si, sh = torch.ones(32), torch.ones(16)
    with pytest.raises(NotImplementedError, match="int8"):
        vb.int8_gated_ffn(x, wg, si, q[1], si, q[2], sh)
    with pytest.raises(NotImplementedError, match="x dtype"):
        vb.int8_gated_ffn(x.float(), q[0], si, q[1], si, q[2], sh)
    with pytest.raises(NotImplementedError, match="activation"):
        vb.int8_gated_ffn(x, q[0], si, q[1], si, q[2], sh, act="gelu")
    y = [w.to(torch.int8) for w in ffn_args(hidden=24)[1:]]
    with pytest.raises(NotImplementedError, match="multiples of 16"):
        vb.int8_gated_ffn(ffn_args(hidden=24)[0], y[0], si, y[1], si, y[2], torch.ones(24))
    with pytest.raises(RuntimeError, match="CUDA tensors only"):
        vb.int8_gated_ffn(x, q[0], si, q[1], si, q[2], sh)


# ── the C entry points ───────────────────────────────────────────────────────────────────────

A = 1 << 20      # an aligned address that is never read


def good_ffn():
    c = _lib.FfnCall()
    c.act_dtype, c.activation, c.n_tokens, c.hidden, c.inter = _lib.BF16, 0, 4, 64, 32
    c.x, c.x_row_stride, c.w_gate, c.w_up, c.w_down = A, 64, A, A, A
    c.out, c.out_row_stride, c.saved = A, 64, A
    c.d_out, c.d_out_row_stride, c.d_x, c.d_x_row_stride = A, 64, A, 64
    return c


@pytest.mark.parametrize("field,value,status", [
    ("act_dtype", _lib.F32, -1), ("activation", 7, -1), ("n_tokens", -1, -2), ("hidden", 0, -2), ("hidden", 60, -1),
    ("inter", 36, -1), ("x", None, -2), ("x", A + 8, -3), ("x_row_stride", 32, -3), ("x_row_stride", 68, -3),
    ("w_gate", None, -2), ("w_down", A + 2, -3), ("workspace_bytes", 16, -4), ("n_tokens", 1 << 31, -1)])
def test_ffn_entry_points_refuse(field, value, status):
    lib = _lib.lib()
    for fn, backward in ((lib.vy_gated_ffn_forward, 0), (lib.vy_gated_ffn_backward, 1)):
        c = good_ffn()
        c.workspace, c.workspace_bytes = A, lib.vy_gated_ffn_workspace_size(ctypes.byref(c), backward)
        setattr(c, field, value)
        assert fn(ctypes.byref(c), None) == status
        assert lib.vy_last_error()
        assert fn(None, None) == -2


@pytest.mark.parametrize("field,value,status", [("out", None, -2), ("out", A + 4, -3), ("out_row_stride", 4, -3)])
def test_ffn_forward_refuses(field, value, status):
    lib, c = _lib.lib(), good_ffn()
    c.workspace, c.workspace_bytes = A, 1 << 30
    setattr(c, field, value)
    assert lib.vy_gated_ffn_forward(ctypes.byref(c), None) == status


@pytest.mark.parametrize("field,value,status", [
    ("saved", None, -2), ("d_out", None, -2), ("d_out", A + 4, -3), ("d_out_row_stride", 8, -3), ("d_x", A + 2, -3),
    ("d_x_row_stride", 60, -3), ("d_w_gate", A + 2, -3), ("d_w_up", A + 2, -3), ("d_w_down", A + 2, -3)])
def test_ffn_backward_refuses(field, value, status):
    lib, c = _lib.lib(), good_ffn()
    c.workspace, c.workspace_bytes = A, 1 << 30
    setattr(c, field, value)
    assert lib.vy_gated_ffn_backward(ctypes.byref(c), None) == status


@pytest.mark.parametrize("field,value,status", [
    ("n_tokens", -1, -2), ("k", 40, -1), ("k", 131072, -1), ("n", 0, -2), ("codes", None, -2), ("codes", A + 8, -3),
    ("codes_row_stride", 72, -3), ("codes_row_stride", 48, -3), ("scales", None, -2), ("weight", A + 1, -3),
    ("weight_scales", None, -2), ("out", None, -2), ("out_dtype", _lib.E4M3, -1), ("out_row_stride", 4, -2)])
def test_int8_linear_entry_point_refuses(field, value, status):
    lib, c = _lib.lib(), _lib.Int8LinearCall()
    c.n_tokens, c.k, c.n = 3, 64, 5
    c.codes, c.codes_row_stride, c.scales, c.weight, c.weight_scales = A, 64, A, A, A
    c.out_dtype, c.out, c.out_row_stride = _lib.BF16, A, 5
    setattr(c, field, value)
    assert lib.vy_int8_linear(ctypes.byref(c), None) == status


@pytest.mark.parametrize("field,value,status", [
    ("act_dtype", _lib.F32, -1), ("activation", 3, -1), ("n_tokens", -1, -2), ("hidden", 40, -1), ("inter", 8, -1),
    ("inter", 131072, -1), ("x", None, -2), ("w_up", None, -2), ("w_gate", A + 8, -3), ("down_scales", None, -2),
    ("x_row_stride", 8, -2), ("workspace_bytes", 100, -4)])
def test_int8_ffn_entry_point_refuses(field, value, status):
    lib, c = _lib.lib(), _lib.Int8FfnCall()
    c.act_dtype, c.activation, c.n_tokens, c.hidden, c.inter = _lib.BF16, 0, 3, 64, 32
    c.x, c.x_row_stride, c.w_gate, c.w_up, c.w_down = A, 64, A, A, A
    c.gate_scales = c.up_scales = c.down_scales = A
    c.out, c.out_row_stride = A, 64
    c.workspace, c.workspace_bytes = A, 1 << 30
    setattr(c, field, value)
    assert lib.vy_int8_gated_ffn(ctypes.byref(c), None) == status


def test_quantize_entry_point_refuses():
    q = _lib.lib().vy_int8_quantize
    assert q(A, _lib.E4M3, 8, 2, 8, A, A, None) == -1
    assert q(A, _lib.BF16, 8, -2, 8, A, A, None) == -2
    assert q(A, _lib.BF16, 8, 2, 0, A, A, None) == -2
    assert q(A, _lib.BF16, 8, 1 << 31, 8, A, A, None) == -1
    assert q(None, _lib.BF16, 8, 2, 8, A, A, None) == -2
    assert q(None, _lib.BF16, 8, 0, 8, None, None, None) == 0


@pytest.mark.skipif(not Path("/usr/bin/gcc").exists(), reason="gcc not available")
def test_ctypes_structures_match_the_c_layout(tmp_path):
    structs = {"vy_ffn_call": _lib.FfnCall, "vy_int8_linear_call": _lib.Int8LinearCall,
               "vy_int8_ffn_call": _lib.Int8FfnCall}
    lines = ['#include <stdio.h>', '#include <stddef.h>', f'#include "{HEADER}"', "int main(void){"]
    for st, cls in structs.items():
        lines.append(f'printf("{st} %zu\\n", sizeof({st}));')
        lines += [f'printf("{st}.{n} %zu\\n", offsetof({st}, {n}));' for n, _t in cls._fields_]
    (tmp_path / "layout.c").write_text("\n".join(lines + ["return 0;}"]))
    subprocess.run(["gcc", "-o", str(tmp_path / "layout"), str(tmp_path / "layout.c")], check=True)
    out = subprocess.run([str(tmp_path / "layout")], capture_output=True, text=True, check=True).stdout
    got = dict(line.split() for line in out.splitlines())
    for packer, cls in ((dense._FFN, _lib.FfnCall), (dense._LINEAR, _lib.Int8LinearCall),
                        (dense._INT8_FFN, _lib.Int8FfnCall)):
        # the packed form puts the same values at the same places as the structure does
        fields = [(n, i + 1) for i, (n, _t) in enumerate(cls._fields_)]
        c = cls(**dict(fields))
        assert packer.pack(*(v for _n, v in fields)) == bytes(c)
    for st, cls in structs.items():
        assert int(got[st]) == ctypes.sizeof(cls)
        for n, _t in cls._fields_:
            assert int(got[f"{st}.{n}"]) == getattr(cls, n).offset, f"{st}.{n}"
