"""Dense operators on the GPU against plain 64-bit forms (tests/dense_reference.py), with bounds that
follow the roundings; the int8 product and the quantisation are compared bit for bit."""
import pytest
import torch

import vaayu_b200 as vb
from tests import dense_reference as R
from tests.helpers import make_blobs

pytestmark = pytest.mark.gpu
BF16, F16, F32 = torch.bfloat16, torch.float16, torch.float32


def make(tokens, hidden, inter, dtype, seed=0, grad=False):
    gen = torch.Generator(device="cuda").manual_seed(seed)

    def randn(*shape):
        return torch.randn(*shape, generator=gen, device="cuda")

    x = randn(tokens, hidden).to(dtype)
    ws = [(randn(a, b) / b ** 0.5).to(dtype) for a, b in ((inter, hidden), (inter, hidden), (hidden, inter))]
    dy = randn(tokens, hidden).to(dtype)
    return [t.requires_grad_(grad) for t in (x, *ws)], dy


# ── gated_ffn ────────────────────────────────────────────────────────────────────────────────

SIZES = [(1, 8, 8), (1, 1024, 512), (2, 72, 40), (3, 1024, 512), (7, 136, 1000), (8, 8, 8), (15, 2048, 768), (16, 64, 64),
         (17, 200, 72), (31, 512, 264), (33, 1032, 520), (64, 256, 128), (65, 256, 136), (127, 128, 256), (128, 264, 1032),
         (129, 520, 72), (160, 520, 1032), (161, 136, 72), (192, 64, 2048), (255, 392, 120), (256, 256, 256), (257, 24, 1032), (700, 1024, 512),
         (1003, 2048, 768)]


@pytest.mark.parametrize("tokens,hidden,inter", SIZES)
@pytest.mark.parametrize("dtype,act", [(BF16, "silu"), (F16, "gelu_tanh")])
def test_forward(tokens, hidden, inter, dtype, act):
    ops, _ = make(tokens, hidden, inter, dtype)
    y = vb.gated_ffn(*ops, act=act, check=True)
    want, bound, _ = R.ffn(*ops, act, dtype)
    assert y.dtype == dtype
    R.assert_within(y, want, bound, "y")


@pytest.mark.parametrize("tokens,hidden,inter", SIZES)
@pytest.mark.parametrize("dtype,act", [(BF16, "gelu_tanh"), (F16, "silu")])
def test_gradients(tokens, hidden, inter, dtype, act):
    ops, dy = make(tokens, hidden, inter, dtype, grad=True)
    y = vb.gated_ffn(*ops, act=act, check=True)
    want, bound, parts = R.ffn(*ops, act, dtype)
    R.assert_within(y, want, bound, "y")
    got = torch.autograd.grad(y, ops, dy)
    for name, g, (v, e) in zip(("dx", "dw_gate", "dw_up", "dw_down"), got, R.ffn_gradients(parts, dy, dtype)):
        assert g.dtype == dtype
        R.assert_within(g, v, e, name)


@pytest.mark.parametrize("act", ["silu", "gelu_tanh"])
def test_gradients_against_differences(act):
    """<grad, v> against the central difference of the 64-bit forward along v: the difference is off
    by O(step^2), taken as 1e-6 of the terms' sizes."""
    ops, dy = make(9, 64, 40, F16, grad=True)
    grads = torch.autograd.grad(vb.gated_ffn(*ops, act=act), ops, dy)
    bounds = [e for _v, e in R.ffn_gradients(R.ffn(*ops, act, F16)[2], dy, F16)]

    def loss(ts):
        x, wg, wu, wd = ts
        return ((R.act_and_slope(x @ wg.T, act)[0] * (x @ wu.T)) @ wd.T * dy.double()).sum()

    base = [t.detach().double() for t in ops]
    for i in range(4):
        v = torch.randn(base[i].shape, dtype=torch.float64, device="cuda",
                        generator=torch.Generator(device="cuda").manual_seed(i))
        step = 1e-5
        moved = [loss([t + s * step * v if j == i else t for j, t in enumerate(base)]) for s in (1, -1)]
        slope = (moved[0] - moved[1]) / (2 * step)
        size = (grads[i].double().abs() * v.abs()).sum()
        assert (slope - (grads[i].double() * v).sum()).abs() <= (bounds[i] * v.abs()).sum() + 1e-6 * size


def test_a_thread_that_has_made_no_cuda_call():
    """The first call of a fresh host thread (autograd's own threads are such) finds no bound context."""
    import threading
    ops, _ = make(2, 64, 40, BF16)
    want, got = vb.gated_ffn(*ops), []
    out = torch.empty(2, 64, dtype=BF16, device="cuda")
    torch.cuda.synchronize()
    thread = threading.Thread(target=lambda: got.append(vb.gated_ffn(*ops, out=out)))
    thread.start()
    thread.join()
    assert torch.equal(got[0], want)


@pytest.mark.parametrize("check", [False, True])
def test_gradients_are_not_differentiable_again(check):
    """Under create_graph the gradients come as ever; differentiating them raises instead of giving zeros."""
    ops, dy = make(6, 64, 40, BF16, grad=True)
    want = torch.autograd.grad(vb.gated_ffn(*ops), ops, dy)
    dy.requires_grad_(True)
    got = torch.autograd.grad(vb.gated_ffn(*ops, check=check), ops, dy, create_graph=True)
    assert all(torch.equal(a, b) for a, b in zip(want, got))
    with pytest.raises(RuntimeError, match="once_differentiable"):
        got[0].sum().backward()


@pytest.mark.parametrize("check", [False, True])
def test_only_wanted_gradients(check):
    for wanted in ((0,), (1,), (2,), (3,), (1, 3), (0, 2)):
        ops, dy = make(40, 128, 72, BF16)
        for i in wanted:
            ops[i].requires_grad_(True)
        y = vb.gated_ffn(*ops, check=check)
        parts = R.ffn(*ops, "silu", BF16)[2]
        ref = R.ffn_gradients(parts, dy, BF16)
        got = torch.autograd.grad(y, [ops[i] for i in wanted], dy)
        for i, g in zip(wanted, got):
            R.assert_within(g, *ref[i], f"gradient {i} of {wanted}")


def test_layouts():
    """Strided rows, rows off a 16-byte boundary, three dimensions, transposed weights, an expanded
    output gradient, out= and a strided out=: the same numbers as the contiguous call."""
    ops, _ = make(21, 128, 72, BF16)
    x, wg, wu, wd = ops
    want = vb.gated_ffn(*ops)
    wide = torch.zeros(21, 200, dtype=BF16, device="cuda")
    for at in (0, 8, 3):
        wide[:, at:at + 128] = x
        assert torch.equal(vb.gated_ffn(wide[:, at:at + 128], wg, wu, wd), want)
    assert torch.equal(vb.gated_ffn(x.t().contiguous().t(), wg, wu, wd), want)
    assert torch.equal(vb.gated_ffn(x, wg.t().contiguous().t(), wu, wd.t().contiguous().t()), want)
    off = torch.empty(72 * 128 + 1, dtype=BF16, device="cuda")[1:].view(72, 128).copy_(wg)
    assert torch.equal(vb.gated_ffn(x, off, wu, wd), want)
    assert torch.equal(vb.gated_ffn(x.view(3, 7, 128), wg, wu, wd), want.view(3, 7, 128))
    assert torch.equal(vb.gated_ffn(x[0], wg, wu, wd), vb.gated_ffn(x[:1], wg, wu, wd)[0])
    out = torch.full((21, 136), 7.0, dtype=BF16, device="cuda")
    assert vb.gated_ffn(x, wg, wu, wd, out=out[:, :128]).data_ptr() == out.data_ptr()
    assert torch.equal(out[:, :128], want) and (out[:, 128:] == 7).all()
    x.requires_grad_(True)
    y = vb.gated_ffn(x, wg, wu, wd)
    a, = torch.autograd.grad(y.sum(), x, retain_graph=True)
    b, = torch.autograd.grad(y, x, torch.ones_like(y))
    assert torch.equal(a, b)


def test_refusals_on_the_gpu():
    ops, _ = make(4, 64, 40, BF16)
    with pytest.raises(ValueError, match="out"):
        vb.gated_ffn(*ops, out=torch.empty(4, 64, dtype=F16, device="cuda"))
    with pytest.raises(ValueError, match="16-byte"):
        vb.gated_ffn(*ops, out=torch.empty(4 * 64 + 1, dtype=BF16, device="cuda")[1:].view(4, 64))
    with pytest.raises(RuntimeError, match="CUDA tensors only"):
        vb.gated_ffn(ops[0], ops[1], ops[2].cpu(), ops[3])
    ops[0].requires_grad_(True)
    with pytest.raises(RuntimeError, match="out="):
        vb.gated_ffn(*ops, out=torch.empty(4, 64, dtype=BF16, device="cuda"))


def test_no_tokens():
    ops, dy = make(0, 64, 40, BF16, grad=True)
    y = vb.gated_ffn(*ops)
    assert y.shape == (0, 64)
    grads = torch.autograd.grad(y, ops, dy)
    assert grads[0].shape == (0, 64) and all((g == 0).all() for g in grads[1:])
    with torch.no_grad():
        assert vb.gated_ffn(*ops).shape == (0, 64)
    c, s = vb.quantize_int8(torch.empty(0, 48, device="cuda"))
    assert c.shape == (0, 48) and s.shape == (0, 1)
    w, ws = vb.quantize_int8(torch.randn(64, 48, device="cuda"))
    assert vb.int8_linear(c, s, w, ws).shape == (0, 64)
    wd, sd = vb.quantize_int8(torch.randn(48, 64, device="cuda"))
    assert vb.int8_gated_ffn(torch.empty(0, 48, device="cuda", dtype=BF16), w, ws, w, ws, wd, sd).shape == (0, 48)


@pytest.mark.parametrize("tokens", [5, 40, 300])
@pytest.mark.parametrize("bad", [float("nan"), float("inf")])
def test_a_bad_row_stays_alone(tokens, bad):
    ops, _ = make(tokens, 136, 72, BF16)
    want = vb.gated_ffn(*ops)
    x = ops[0].clone()
    x[2, 5] = bad
    y = vb.gated_ffn(x, *ops[1:])
    keep = torch.arange(tokens, device="cuda") != 2
    assert torch.equal(y[keep], want[keep])
    assert not torch.isfinite(y[2]).any()


def test_large_activations():
    """Gate values far out on both sides: silu and gelu_tanh saturate, gradients stay finite."""
    for act in ("silu", "gelu_tanh"):
        ops, dy = make(20, 64, 40, BF16, grad=True)
        with torch.no_grad():
            ops[1].mul_(3e4)
        y = vb.gated_ffn(*ops, act=act)
        want, bound, parts = R.ffn(*ops, act, BF16)
        R.assert_within(y, want, bound, "y")
        for g, (v, e) in zip(torch.autograd.grad(y, ops, dy), R.ffn_gradients(parts, dy, BF16)):
            R.assert_within(g, v, e, act)


@pytest.mark.parametrize("tokens", [1, 48, 300])
def test_repeatable_and_on_a_side_stream(tokens):
    ops, dy = make(tokens, 512, 264, BF16, grad=True)

    def step():
        y = vb.gated_ffn(*ops)
        return [y, *torch.autograd.grad(y, ops, dy)]

    want = step()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = [step() for _ in range(3)]
    again = step()               # both streams at work
    torch.cuda.synchronize()
    for other in (*got, again):
        assert all(torch.equal(a, b) for a, b in zip(want, other))


@pytest.mark.parametrize("tokens", [1, 48, 300])
def test_captured_steps_replay(tokens):
    """A forward and backward pass captured into two graphs, replayed on changed inputs."""
    ops, dy = make(tokens, 512, 264, BF16, grad=True)
    x = ops[0]

    def step():
        y = vb.gated_ffn(*ops)
        return [y, *torch.autograd.grad(y, ops, dy)]

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step()
    torch.cuda.current_stream().wait_stream(side)
    graphs, results = [], []
    for _ in range(2):
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            results.append(step())
        graphs.append(g)
    with torch.no_grad():
        x.copy_(make(tokens, 512, 264, BF16, seed=3)[0][0])
    for g in graphs:
        g.replay()
    want = step()
    torch.cuda.synchronize()
    for got in results:
        assert all(torch.equal(a, b) for a, b in zip(want, got))


def test_more_values_than_32_bits_count():
    """2.2e9 intermediate values: offsets of h, and of the int8 block's h, pass 2^31."""
    tokens, hidden, inter = 140_000, 16, 16_384
    ops, _ = make(tokens, hidden, inter, BF16)
    rows = torch.tensor([0, 1, 70_000, 131_071, 131_072, 139_998, 139_999], device="cuda")
    y = vb.gated_ffn(*ops)
    want, bound, _ = R.ffn(ops[0][rows], *ops[1:], "silu", BF16)
    R.assert_within(y[rows], want, bound, "y")
    q = [vb.quantize_int8(w) for w in ops[1:]]
    y = vb.int8_gated_ffn(ops[0], *q[0], *q[1], *q[2])
    flat = [t.reshape(-1) if t.dtype == F32 else t for pair in q for t in pair]
    want, bound = R.int8_ffn(ops[0][rows], *flat, "silu", BF16)
    R.assert_within(y[rows], want, bound, "int8 y")


# ── quantize_int8 ────────────────────────────────────────────────────────────────────────────


@pytest.mark.parametrize("dtype", [BF16, F16, F32])
@pytest.mark.parametrize("tokens,width", [(1, 1), (1, 7168), (2, 33), (3, 16), (5, 7168), (7, 771), (64, 4096), (9, 14336),
                                          (300, 520), (2, 16400), (3, 40000), (1000, 48)])
def test_quantize(tokens, width, dtype):
    gen = torch.Generator(device="cuda").manual_seed(width)
    x = (torch.randn(tokens, width, generator=gen, device="cuda")
         * torch.exp(2 * torch.randn(tokens, 1, generator=gen, device="cuda"))).to(dtype)
    codes, scale = vb.quantize_int8(x)
    want, ws = R.quantize(x)
    assert codes.dtype == torch.int8 and scale.shape == (tokens, 1)
    assert torch.equal(scale, ws)
    assert torch.equal(codes, want)


def test_quantize_ties_and_special_rows():
    big = torch.finfo(F32).max
    rows = torch.zeros(10, 64, device="cuda")
    rows[1] = torch.arange(64, device="cuda") + 0.5            # amax 127 below: exact ties
    rows[1, 0] = 127.0
    rows[2] = -(torch.arange(64, device="cuda") + 0.5)
    rows[2, 0] = -127.0
    rows[3, 3] = float("nan")
    rows[4, 5] = float("inf")
    rows[5, 60] = -float("inf")
    rows[6] = big
    rows[6, ::2] = -big / 3
    rows[7] = 1e-44                                            # a scale that underflows to zero
    rows[8] = torch.arange(64, device="cuda") * 1e-41          # a subnormal scale
    rows[9] = torch.arange(64, device="cuda") * 3e-36          # a scale whose reciprocal is near the top
    codes, scale = vb.quantize_int8(rows)
    want, ws = R.quantize(rows)
    fine = [0, 1, 2, 6, 7, 8, 9]
    assert torch.equal(scale[fine], ws[fine]) and torch.equal(codes[fine], want[fine])
    assert (codes[[0, 3, 4, 5, 7]] == 0).all()
    assert torch.isnan(scale[[3, 4, 5]]).all()
    # the bad rows' products are NaN, the others' are not touched
    w, wsc = vb.quantize_int8(torch.randn(24, 64, device="cuda"))
    y = vb.int8_linear(codes, scale, w, wsc, dtype=F32)
    assert torch.isnan(y[[3, 4, 5]]).all() and torch.isfinite(y[[0, 1, 2, 7, 8, 9]]).all()


def test_quantize_layouts():
    x = torch.randn(12, 300, device="cuda").to(BF16)
    want = vb.quantize_int8(x[:, 8:280].contiguous())
    for view in (x[:, 8:280], x[:, 8:280].t().contiguous().t()):
        got = vb.quantize_int8(view)
        assert all(torch.equal(a, b) for a, b in zip(got, want))
    odd = vb.quantize_int8(x[:, 3:200])
    ref = R.quantize(x[:, 3:200])
    assert torch.equal(odd[0], ref[0]) and torch.equal(odd[1], ref[1])
    c3, s3 = vb.quantize_int8(x.view(3, 4, 300))
    c, s = vb.quantize_int8(x)
    assert torch.equal(c3.view(12, 300), c) and s3.shape == (3, 4, 1) and torch.equal(s3.view(12, 1), s)
    same = vb.quantize_int8(x[:1].expand(5, 300))
    assert torch.equal(same[0], c[:1].expand(5, 300))


# ── int8_linear ──────────────────────────────────────────────────────────────────────────────

LINEAR = [(1, 16, 1), (1, 4096, 300), (2, 32, 7), (3, 272, 97), (8, 128, 128), (15, 1040, 129), (16, 4096, 1000),
          (17, 48, 255), (33, 7168, 256), (64, 528, 513), (65, 256, 1024), (100, 14336, 64), (128, 144, 384),
          (129, 128, 2048), (160, 1040, 300), (161, 528, 97), (256, 512, 256), (300, 272, 97), (777, 1040, 1001), (1003, 2048, 768)]


def int8_operands(tokens, k, n, seed=0):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    codes = torch.randint(-128, 128, (tokens, k), generator=gen, device="cuda", dtype=torch.int8)
    w = torch.randint(-128, 128, (n, k), generator=gen, device="cuda", dtype=torch.int8)
    scale = torch.rand(tokens, 1, generator=gen, device="cuda") * 0.02
    ws = torch.rand(n, generator=gen, device="cuda") * 0.01
    bias = torch.randn(n, generator=gen, device="cuda")
    return codes, scale, w, ws, bias


@pytest.mark.parametrize("tokens,k,n", LINEAR)
@pytest.mark.parametrize("dtype,biased", [(BF16, False), (F16, True), (F32, True)])
def test_int8_linear(tokens, k, n, dtype, biased):
    codes, scale, w, ws, bias = int8_operands(tokens, k, n)
    bias = bias.to(dtype) if biased else None
    y = vb.int8_linear(codes, scale, w, ws, bias=bias, dtype=dtype, check=True)
    assert torch.equal(y, R.int8_product(codes, scale, w, ws, bias).to(dtype))


def test_int8_linear_largest_sums():
    """K just below the limit with every product +-16384: sums up to 2.1e9 stay exact."""
    k = 131_056
    codes = torch.full((3, k), -128, dtype=torch.int8, device="cuda")
    codes[1] = 127
    w = torch.full((40, k), -128, dtype=torch.int8, device="cuda")
    w[7] = 127
    one3, one40 = torch.ones(3, 1, device="cuda"), torch.ones(40, device="cuda")
    for c in (codes, codes.repeat(50, 1)):
        s = one3.repeat(c.shape[0] // 3, 1)
        assert torch.equal(vb.int8_linear(c, s, w, one40, dtype=F32), R.int8_product(c, s, w, one40))


def test_int8_linear_layouts():
    codes, scale, w, ws, bias = int8_operands(20, 288, 50)
    want = vb.int8_linear(codes, scale, w, ws)
    wide = torch.zeros(20, 400, dtype=torch.int8, device="cuda")
    for at in (0, 16, 5):
        wide[:, at:at + 288] = codes
        assert torch.equal(vb.int8_linear(wide[:, at:at + 288], scale, w, ws), want)
    assert torch.equal(vb.int8_linear(codes, scale.view(20), w.t().contiguous().t(), ws.view(50, 1)), want)
    assert torch.equal(vb.int8_linear(codes.view(4, 5, 288), scale.view(4, 5, 1), w, ws), want.view(4, 5, 50))
    for cols in (50, 53, 56):
        out = torch.full((20, cols), 3.0, dtype=BF16, device="cuda")
        vb.int8_linear(codes, scale, w, ws, out=out[:, :50])
        assert torch.equal(out[:, :50], want) and (out[:, 50:] == 3).all()
    half = ws.to(BF16)
    assert torch.equal(vb.int8_linear(codes, scale, w, half), vb.int8_linear(codes, scale, w, half.float()))
    with pytest.raises(ValueError, match="scales"):
        vb.int8_linear(codes, scale[:3], w, ws)


# ── int8_gated_ffn ───────────────────────────────────────────────────────────────────────────


@pytest.mark.parametrize("tokens,hidden,inter", [(1, 16, 16), (1, 1024, 512), (2, 144, 48), (1, 14336, 256), (2, 8192, 144),
                                                 (3, 4096, 1040), (4, 4112, 272), (9, 1040, 4096), (15, 272, 2064),
                                                 (16, 1024, 16), (16, 7168, 2048), (17, 64, 1040),
                                                 (33, 528, 272), (64, 256, 128), (129, 272, 80), (257, 1040, 528),
                                                 (1003, 2048, 768)])
@pytest.mark.parametrize("dtype,act", [(BF16, "silu"), (F16, "gelu_tanh")])
def test_int8_gated_ffn(tokens, hidden, inter, dtype, act):
    ops, _ = make(tokens, hidden, inter, dtype)
    q = [vb.quantize_int8(w) for w in ops[1:]]
    y = vb.int8_gated_ffn(ops[0], *q[0], *q[1], *q[2], act=act, check=True)
    flat = [t.reshape(-1) if t.dtype == F32 else t for pair in q for t in pair]
    want, bound = R.int8_ffn(ops[0], *flat, act, dtype)
    R.assert_within(y, want, bound, "y")


@pytest.mark.parametrize("tokens", [1, 12, 24, 300])
def test_int8_gated_ffn_layouts_and_capture(tokens):
    ops, _ = make(tokens, 272, 144, BF16)
    x = ops[0]
    q = [t for w in ops[1:] for t in vb.quantize_int8(w)]
    want = vb.int8_gated_ffn(x, *q)
    wide = torch.zeros(tokens, 301, dtype=BF16, device="cuda")
    for at in (5, 8):
        wide[:, at:at + 272] = x
        assert torch.equal(vb.int8_gated_ffn(wide[:, at:at + 272], *q), want)
    out = torch.full((tokens, 275), 2.0, dtype=BF16, device="cuda")
    vb.int8_gated_ffn(x.view(tokens, 272), *q, out=out[:, :272])
    assert torch.equal(out[:, :272], want) and (out[:, 272:] == 2).all()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        vb.int8_gated_ffn(x, *q)
    torch.cuda.current_stream().wait_stream(side)
    graphs, outs = [torch.cuda.CUDAGraph(), torch.cuda.CUDAGraph()], []
    for g in graphs:
        with torch.cuda.graph(g):
            outs.append(vb.int8_gated_ffn(x, *q))
    x.copy_(make(tokens, 272, 144, BF16, seed=5)[0][0])
    for g in graphs:
        g.replay()
    want = vb.int8_gated_ffn(x, *q)
    assert all(torch.equal(o, want) for o in outs)


@pytest.mark.parametrize("tokens", [2, 9, 40, 300])
def test_int8_gated_ffn_odd_rows_stay_alone(tokens):
    """A zero row gives zeros, a row with a NaN or an infinity NaN, and no other row changes."""
    ops, _ = make(tokens, 272, 144, BF16)
    q = [t for w in ops[1:] for t in vb.quantize_int8(w)]
    want = vb.int8_gated_ffn(ops[0], *q)
    for bad in (0.0, float("nan"), -float("inf")):
        x = ops[0].clone()
        x[1] = 0.0
        x[1, 7] = bad
        y = vb.int8_gated_ffn(x, *q)
        keep = torch.arange(tokens, device="cuda") != 1
        assert torch.equal(y[keep], want[keep])
        assert (y[1] == 0).all() if bad == 0.0 else torch.isnan(y[1]).all()


@pytest.mark.parametrize("tokens", [3, 100, 400])
def test_two_streams_at_once(tokens):
    ops, _ = make(tokens, 1040, 528, BF16)
    q = [t for w in ops[1:] for t in vb.quantize_int8(w)]
    codes, scale = vb.quantize_int8(ops[0])

    def calls():
        return vb.gated_ffn(*ops), vb.int8_gated_ffn(ops[0], *q), vb.int8_linear(codes, scale, q[0], q[1])

    want = calls()
    torch.cuda.synchronize()
    streams, results = [torch.cuda.Stream() for _ in range(2)], []
    for _ in range(5):
        for s in streams:
            with torch.cuda.stream(s):
                results.append(calls())
    torch.cuda.synchronize()
    for got in results:
        assert all(torch.equal(a, b) for a, b in zip(want, got))


@pytest.mark.skipif("torch.cuda.device_count() < 2")
def test_a_device_that_is_not_current():
    ops, dy = make(40, 256, 136, BF16, grad=True)
    there = [t.detach().to("cuda:1").requires_grad_(True) for t in ops]
    y, z = vb.gated_ffn(*ops), vb.gated_ffn(*there)
    assert torch.equal(y.cpu(), z.cpu())
    for a, b in zip(torch.autograd.grad(y, ops, dy), torch.autograd.grad(z, there, dy.to("cuda:1"))):
        assert torch.equal(a.cpu(), b.cpu())
    with pytest.raises(RuntimeError, match="tensors on"):
        vb.gated_ffn(ops[0], *there[1:])


@pytest.mark.parametrize("tokens", [1, 20, 200])
def test_both_host_paths_make_the_same_calls(tokens):
    """The extension (ordinary calls) and the Python path (here: check=True, or a row stride) run the
    same kernels: equal bits, gradients among them."""
    ops, dy = make(tokens, 272, 144, F16, grad=True)
    a, b = vb.gated_ffn(*ops), vb.gated_ffn(*ops, check=True)
    assert type(a.grad_fn).__name__ != type(b.grad_fn).__name__
    assert torch.equal(a, b)
    for g, h in zip(torch.autograd.grad(a, ops, dy), torch.autograd.grad(b, ops, dy)):
        assert torch.equal(g, h)
    x, (wg, wu, wd) = ops[0].detach(), (w.detach() for w in ops[1:])
    with torch.no_grad():
        assert torch.equal(vb.gated_ffn(*ops), a) and not vb.gated_ffn(*ops).requires_grad
    wide = torch.zeros(tokens, 288, dtype=F16, device="cuda")
    wide[:, :272] = x
    for p, q in zip(vb.quantize_int8(x), vb.quantize_int8(wide[:, :272])):
        assert torch.equal(p, q)
    codes, scale = vb.quantize_int8(x)
    q = [t for w in (wg, wu, wd) for t in vb.quantize_int8(w)]
    assert torch.equal(vb.int8_linear(codes, scale, q[0], q[1], dtype=F32),
                       vb.int8_linear(codes, scale, q[0], q[1], dtype=F32, check=True))
    assert torch.equal(vb.int8_gated_ffn(x, *q), vb.int8_gated_ffn(x, *q, check=True))
    x3 = x.view(1, tokens, 272)
    assert vb.int8_gated_ffn(x3, *q).shape == x3.shape and vb.quantize_int8(x3)[1].shape == (1, tokens, 1)


# ── together ─────────────────────────────────────────────────────────────────────────────────


@pytest.mark.parametrize("tokens", [1, 20, 260])
def test_a_block_of_dense_and_packed_layers(tokens):
    """A token batch through an int8 projection, a dense block, the packed experts and a 16-bit shared
    expert, each fed the previous one's output without a synchronisation in between."""
    hidden, inter = 256, 128
    (x, wg, wu, wd), _ = make(tokens, hidden, inter, BF16)
    q = [t for w in (wg, wu, wd) for t in vb.quantize_int8(w)]
    proj = vb.quantize_int8(make(hidden, hidden, 8, BF16, seed=1)[0][0])
    table = vb.ExpertTable(make_blobs(hidden, inter, 8))
    logits = torch.randn(tokens, 8, device="cuda", generator=torch.Generator(device="cuda").manual_seed(2))

    def step():
        codes, scale = vb.quantize_int8(x)
        z = vb.int8_linear(codes, scale, *proj)
        dense = vb.gated_ffn(z, wg, wu, wd)
        packed = vb.moe_forward(dense, *reversed(vb.topk_softmax(logits, 2)), table)
        shared = vb.gated_ffn(dense, wg, wu, wd, act="gelu_tanh")
        return z, dense, packed, shared, vb.int8_gated_ffn(dense, *q)

    z, dense, packed, shared, last = step()
    torch.cuda.synchronize()
    assert torch.equal(z, R.int8_product(*R.quantize(x), *proj).to(BF16))
    R.assert_within(dense, *R.ffn(z, wg, wu, wd, "silu", BF16)[:2], "dense")
    R.assert_within(shared, *R.ffn(dense, wg, wu, wd, "gelu_tanh", BF16)[:2], "shared")
    flat = [t.reshape(-1) if t.dtype == F32 else t for t in q]
    R.assert_within(last, *R.int8_ffn(dense, *flat, "silu", BF16), "int8 block")
    alone = vb.moe_forward(dense.clone(), *reversed(vb.topk_softmax(logits, 2)), table)
    torch.cuda.synchronize()
    assert torch.equal(packed, alone)
    assert all(torch.equal(a, b) for a, b in zip(step(), (z, dense, packed, shared, last)))
