"""Refusals of the dense operators' C entry points that keep a kernel from a bad access or an unfinished
wait (no GPU: every call fails in its argument checks)."""
import ctypes

import pytest
import torch

import vaayu_b200 as vb
from vaayu_b200 import _lib

A = 1 << 20      # an aligned address that is never read


def ffn_call(backward):
    lib, c = _lib.lib(), _lib.FfnCall()
    c.act_dtype, c.activation, c.n_tokens, c.hidden, c.inter = _lib.BF16, 0, 4, 64, 32
    c.x, c.x_row_stride, c.w_gate, c.w_up, c.w_down = A, 64, A, A, A
    c.out, c.out_row_stride, c.saved = A, 64, A
    c.d_out, c.d_out_row_stride, c.d_x, c.d_x_row_stride = A, 64, A, 64
    c.workspace, c.workspace_bytes = A, 1 << 62
    return c, lib.vy_gated_ffn_backward if backward else lib.vy_gated_ffn_forward


@pytest.mark.parametrize("backward", [False, True])
@pytest.mark.parametrize("off", [2, 4, 8, 12])
def test_saved_must_be_aligned(backward, off):
    """g and u move as 16-byte vectors; a float array inside a larger buffer may start anywhere."""
    c, fn = ffn_call(backward)
    c.saved = A + off
    assert fn(ctypes.byref(c), None) == -3
    assert b"saved" in _lib.lib().vy_last_error()


def test_sums_that_could_outlast_a_bounded_wait_are_refused():
    """A tile's sum of more than 2^27 products may take longer than its epilogue waits (2 s), and would
    leave the tile unwritten."""
    for backward, field, value in ((False, "hidden", (1 << 27) + 8), (False, "inter", (1 << 26) + 8),
                                   (True, "hidden", (1 << 27) + 8), (True, "inter", (1 << 26) + 8)):
        c, fn = ffn_call(backward)
        setattr(c, field, value)
        c.x_row_stride = c.out_row_stride = c.d_out_row_stride = c.d_x_row_stride = 1 << 28
        assert fn(ctypes.byref(c), None) == -1
        assert b"2^27" in _lib.lib().vy_last_error()
    for name in ("d_w_gate", "d_w_up", "d_w_down"):
        c, fn = ffn_call(True)
        c.n_tokens = (1 << 27) + 1
        setattr(c, name, A)
        assert fn(ctypes.byref(c), None) == -1
        assert b"2^27" in _lib.lib().vy_last_error()


@pytest.mark.parametrize("tokens", [1, 500])
def test_more_output_channels_than_an_int_rounds_up(tokens):
    """n within a tile of 2^31 overflowed when it was rounded up to whole tiles, and the launch had a
    grid of its own."""
    lib, c = _lib.lib(), _lib.Int8LinearCall()
    c.n_tokens, c.k, c.n = tokens, 16, 0x7FFFFF01
    c.codes, c.codes_row_stride, c.scales, c.weight, c.weight_scales = A, 16, A, A, A
    c.out_dtype, c.out, c.out_row_stride = _lib.BF16, A, 1 << 31
    assert lib.vy_int8_linear(ctypes.byref(c), None) == -1
    assert b"above" in lib.vy_last_error()


@pytest.mark.parametrize("n", [0x7FFFFF01, 1 << 31, 1 << 40])
def test_int8_linear_refuses_them_by_name(n):
    codes, w = torch.zeros(2, 16, dtype=torch.int8), torch.zeros(1, dtype=torch.int8).expand(n, 16)
    with pytest.raises(NotImplementedError, match="up to"):
        vb.int8_linear(codes, torch.ones(2, 1), w, torch.ones(1).expand(n))
