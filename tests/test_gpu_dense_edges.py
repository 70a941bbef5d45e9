"""Dense operators on the GPU at their edges: derivatives finer than a 16-bit rounding, what autograd
may ask for beyond one backward pass, unusual views and operands, the two-part hidden rows."""
import pytest
import torch

import vaayu_b200 as vb
from tests import dense_reference as R

pytestmark = pytest.mark.gpu
BF16, F16, F32, F64 = torch.bfloat16, torch.float16, torch.float32, torch.float64


def randn(*shape, seed=0):
    return torch.randn(*shape, generator=torch.Generator(device="cuda").manual_seed(seed), device="cuda")


def block(tokens, hidden, inter, dtype, grad=False):
    """x, w_gate, w_up, w_down of a block with unit-variance sums."""
    x = randn(tokens, hidden).to(dtype)
    ws = [(randn(a, b, seed=i + 1) / b ** 0.5).to(dtype)
          for i, (a, b) in enumerate(((inter, hidden), (inter, hidden), (hidden, inter)))]
    return [t.requires_grad_(grad) for t in (x, *ws)]


# ── derivatives ──────────────────────────────────────────────────────────────────────────────


@pytest.mark.parametrize("act,check", [("gelu_tanh", False), ("gelu_tanh", True), ("silu", False)])
def test_the_gates_derivative_in_32_bits(act, check):
    """act'(g) to fp32 accuracy, through a d_x whose leading bits cancel: column 7 of d_x is
    16 (256 act'(g) + hi + lo), where two more channels, whose act' is exactly 1 (g = 40), carry
    256 act'(g) rounded to hi + lo in fp16.  Up to 32 tokens dg keeps 22 bits.

    Bound, u = 2^-24: the sigmoid's argument z is off by 7 u |z| (seven roundings, constants among
    them), exp by 4 u more, the sum and the approximate quotient by 5 u; a' = s + g s (1 - s) z' follows
    s, with 9 u on the second term, its 1 - s, and a rounding each of the sum and of s; dg's two parts
    are off by 2^-22, the sums of d_x by R.sum_error(16) of their terms; then the result's rounding."""
    u = 2.0 ** -24
    tokens = 20
    g = (-4.5 + 0.125 * torch.arange(tokens, device="cuda", dtype=F64))
    want = R.act_and_slope(g, act)[1]
    k, c = 1.5957691216057308, 0.044715
    z = g if act == "silu" else k * (g + c * g ** 3)
    dz = torch.ones_like(g) if act == "silu" else k * (1 + 3 * c * g * g)
    s = torch.sigmoid(z)
    rel_s = (1 - s) * (7 * u * z.abs() + 4 * u) + 5 * u
    term = (g * s * (1 - s) * dz).abs()
    off = want.abs() * rel_s + term * (9 * u + s / (1 - s) * rel_s + u) + (s + want.abs()) * u
    off = off + want.abs() * (2.0 ** -22 + 2 * R.sum_error(16))

    hi = (-256 * want).to(F16)
    lo = (-256 * want - hi.double()).to(F16)
    x = torch.zeros(tokens, 8, device="cuda", dtype=F16)
    x[:, 0], x[:, 1], x[:, 2], x[:, 3], x[:, 4] = g.to(F16), 40, hi, lo, 256
    assert torch.equal(x[:, 0].double(), g)
    wg, wu, wd = (torch.zeros(8, 8, device="cuda", dtype=F16) for _ in range(3))
    wg[0, 0] = wg[1, 1] = wg[2, 1] = 1
    wg[:3, 7] = 1
    wu[0, 4] = wu[1, 2] = wu[2, 3] = 1
    wd[0, :3] = 1
    dy = torch.zeros_like(x)
    dy[:, 0] = 16
    x.requires_grad_(True)
    y = vb.gated_ffn(x, wg, wu, wd, act=act, check=check)
    dx, = torch.autograd.grad(y, x, dy)
    exact = 16 * (256 * want + hi.double() + lo.double())
    bound = (4096 * off) * (1 + R.unit(F16)) + R.unit(F16) * exact.abs() + R.tiny(F16)
    R.assert_within(dx[:, 7], exact, bound, "the cancelled column")


@pytest.mark.parametrize("how", ["ordinary", "check", "strided"])
def test_no_second_derivative_without_a_differentiable_incoming_gradient(how):
    """y.sum()'s gradient is a constant, and the gradients that come of it under create_graph still
    depend on x and the weights: a second backward pass raises, whichever host path made the call."""
    x, wg, wu, wd = block(6, 64, 40, BF16, grad=True)
    want = torch.autograd.grad(vb.gated_ffn(x, wg, wu, wd).sum(), (x, wg, wu, wd))
    z = x
    if how == "strided":
        wide = torch.zeros(6, 72, dtype=BF16, device="cuda")
        wide[:, :64] = x.detach()
        z = wide[:, :64].requires_grad_(True)
    y = vb.gated_ffn(z, wg, wu, wd, check=how == "check")
    got = torch.autograd.grad(y.sum(), (z, wg, wu, wd), create_graph=True)
    assert all(torch.equal(a, b) for a, b in zip(want, got))
    for g in got:
        assert g.requires_grad
        with pytest.raises(RuntimeError, match="once_differentiable"):
            (y.sum() + g.float().pow(2).sum()).backward(retain_graph=True)
    only, = torch.autograd.grad(vb.gated_ffn(z, wg, wu, wd, check=how == "check").sum(), wu, create_graph=True)
    with pytest.raises(RuntimeError, match="once_differentiable"):
        only.sum().backward()


@pytest.mark.parametrize("check", [False, True])
def test_forward_mode_derivatives_are_refused(check):
    """A dual tensor would come out without its tangent, a derivative of zero; it is refused."""
    fwd = torch.autograd.forward_ad
    ops = block(5, 64, 48, BF16)
    q = [t for w in ops[1:] for t in vb.quantize_int8(w)]
    codes, scale = vb.quantize_int8(ops[0])
    bias = randn(48)
    want = vb.gated_ffn(*ops)
    with fwd.dual_level():
        def dual(ts, i):
            return [fwd.make_dual(t, torch.ones_like(t)) if j == i else t for j, t in enumerate(ts)]

        for i in range(4):
            with pytest.raises(NotImplementedError, match="forward-mode"):
                vb.gated_ffn(*dual(ops, i), check=check)
        with pytest.raises(NotImplementedError, match="forward-mode"):
            vb.quantize_int8(dual(ops, 0)[0])
        linear = (codes, scale, q[0], q[1], bias)
        for i in (1, 3, 4):
            with pytest.raises(NotImplementedError, match="forward-mode"):
                vb.int8_linear(*dual(linear, i), check=check)
        block_ops = (ops[0], *q)
        for i in (0, 2, 4, 6):
            with pytest.raises(NotImplementedError, match="forward-mode"):
                vb.int8_gated_ffn(*dual(block_ops, i), check=check)
        assert torch.equal(vb.gated_ffn(*ops, check=check), want)      # no dual operand: as ever
        leaf = ops[0].clone().requires_grad_(True)
        y = vb.gated_ffn(leaf, *ops[1:], check=check)
        with pytest.raises(NotImplementedError, match="forward-mode"):
            torch.autograd.grad(y, leaf, dual(ops, 0)[0])
        with pytest.raises(NotImplementedError, match="forward-mode"):
            vb.gated_ffn(*ops, out=fwd.make_dual(torch.ones_like(want), torch.ones_like(want)))
    assert torch.equal(vb.gated_ffn(*ops, check=check), want)


@pytest.mark.parametrize("check", [False, True])
def test_int8_calls_say_that_they_have_no_gradients(check):
    """The int8 calls run on operands that require gradients, with the same bits, and a backward pass
    through their results raises: it would silently leave the operands without their share."""
    ops = block(5, 64, 48, BF16)
    q = [t for w in ops[1:] for t in vb.quantize_int8(w)]
    codes, scale = vb.quantize_int8(ops[0])
    linear = (codes, scale, q[0], q[1], randn(48))
    whole = (ops[0], *q)

    def grad_of(ts, i):
        return [t.clone().requires_grad_(True) if j == i else t for j, t in enumerate(ts)]

    calls = [(vb.int8_linear, linear, (1, 3, 4)), (vb.int8_gated_ffn, whole, (0, 2, 4, 6))]
    for fn, operands, places in calls:
        want = fn(*operands, check=check)
        assert not want.requires_grad
        for i in places:
            with_grad = grad_of(operands, i)
            y = fn(*with_grad, check=check)
            assert torch.equal(y, want) and y.requires_grad
            with pytest.raises(RuntimeError, match="no gradients"):
                y.float().sum().backward()
            assert with_grad[i].grad is None
            with torch.no_grad():
                assert not fn(*with_grad, check=check).requires_grad
            with pytest.raises(RuntimeError, match="out="):
                fn(*with_grad, out=torch.empty_like(want))
    x = ops[0].clone().requires_grad_(True)
    c, s = vb.quantize_int8(x)
    assert torch.equal(c, codes) and torch.equal(s, scale) and not c.requires_grad
    y = vb.int8_linear(c, s, q[0], q[1], check=check)
    for result in (s, y):
        with pytest.raises(RuntimeError, match="no gradients"):
            result.float().sum().backward()
    empty = vb.quantize_int8(torch.empty(0, 48, device="cuda", requires_grad=True))
    assert empty[1].requires_grad and empty[1].shape == (0, 1)


# ── errors ───────────────────────────────────────────────────────────────────────────────────


def test_a_refused_call_of_the_extension_raises():
    """A C entry that answers with an error (here a stand-in for the quantisation's) raises, with its
    status, and the next call works."""
    import ctypes
    from vaayu_b200 import _lib, dense
    x = randn(3, 64)
    want = vb.quantize_int8(x)
    host, lib = dense._host(), _lib.lib()
    real = [ctypes.cast(getattr(lib, n), ctypes.c_void_p).value for n in dense._HOST_ENTRIES]
    restype, argtypes = _lib.SIGNATURES["vy_int8_quantize"]
    stand_in = ctypes.CFUNCTYPE(restype, *argtypes)(lambda *a: -5)
    fake = list(real)
    fake[dense._HOST_ENTRIES.index("vy_int8_quantize")] = ctypes.cast(stand_in, ctypes.c_void_p).value
    host.bind(fake)
    try:
        with pytest.raises(RuntimeError, match=r"quantize_int8 failed \(status -5\)"):
            vb.quantize_int8(x)
    finally:
        host.bind(real)
    assert all(torch.equal(a, b) for a, b in zip(vb.quantize_int8(x), want))


# ── views and operands ───────────────────────────────────────────────────────────────────────


@pytest.mark.parametrize("tokens", [2, 12, 24, 300])
def test_rows_that_overlap(tokens):
    """Rows on top of one another (an expanded row) or overlapping: the same numbers as their copy."""
    x, wg, wu, wd = block(tokens, 272, 144, BF16)
    q = [t for w in (wg, wu, wd) for t in vb.quantize_int8(w)]
    line = randn(272 + 16 * tokens, seed=9).to(BF16)
    codes, _ = vb.quantize_int8(line.view(1, -1))
    for rows in (x[:1].expand(tokens, 272), line.as_strided((tokens, 272), (16, 1)),
                 line.as_strided((tokens, 272), (3, 1)), line.as_strided((tokens, 272), (1, 1))):
        assert torch.equal(vb.int8_gated_ffn(rows, *q), vb.int8_gated_ffn(rows.contiguous(), *q))
        assert torch.equal(vb.gated_ffn(rows, wg, wu, wd), vb.gated_ffn(rows.contiguous(), wg, wu, wd))
        for a, b in zip(vb.quantize_int8(rows), vb.quantize_int8(rows.contiguous())):
            assert torch.equal(a, b)
    scale = torch.rand(tokens, 1, device="cuda")
    rows = codes.view(-1).as_strided((tokens, 272), (16, 1))
    assert torch.equal(vb.int8_linear(rows, scale, q[0], q[1]), vb.int8_linear(rows.contiguous(), scale, q[0], q[1]))


@pytest.mark.parametrize("check", [False, True])
def test_saved_tensors_that_hooks_give_back(check):
    """Hooks on saved tensors may hand the backward pass equal tensors of another layout: the same
    gradients.  Tensors elsewhere, of another type or size are refused before any address is taken."""
    ops = block(40, 128, 72, BF16, grad=True)
    dy = randn(40, 128, seed=4).to(BF16)
    want = torch.autograd.grad(vb.gated_ffn(*ops), ops, dy)

    def grads(pack, unpack):
        with torch.autograd.graph.saved_tensors_hooks(pack, unpack):
            y = vb.gated_ffn(*ops, check=check)
        return torch.autograd.grad(y, ops, dy)

    def off_a_boundary(t):
        return torch.empty(t.numel() + 1, dtype=t.dtype, device=t.device)[1:].view(t.shape).copy_(t)

    def across(t):
        return t.t().contiguous().t() if t.dim() == 2 else torch.stack((t, t), 1)[:, 0]

    same = [lambda t: t, lambda t: t.clone(), across, off_a_boundary]
    for unpack in same:
        for a, b in zip(grads(lambda t: t, unpack), want):
            assert torch.equal(a, b)
    for a, b in zip(grads(lambda t: t.cpu(), lambda t: t.cuda()), want):
        assert torch.equal(a, b)
    with torch.autograd.graph.save_on_cpu():
        y = vb.gated_ffn(*ops, check=check)
    assert all(torch.equal(a, b) for a, b in zip(torch.autograd.grad(y, ops, dy), want))
    for wrong in (lambda t: t.cpu(), lambda t: t.double(), lambda t: t[:-1], lambda t: t.reshape(1, -1),
                  lambda t: t.cpu() if t.dtype == F32 else t, lambda t: t[:-4] if t.dtype == F32 else t,
                  lambda t: t[:33] if t.shape[0] == 40 else t, lambda t: t.half() if t.dtype == BF16 else t):
        with pytest.raises((RuntimeError, ValueError, NotImplementedError)):
            grads(lambda t: t, wrong)


@pytest.mark.parametrize("check", [False, True])
def test_a_node_called_by_hand(check):
    ops = block(9, 64, 40, BF16, grad=True)
    dy = randn(9, 64, seed=4).to(BF16)
    y = vb.gated_ffn(*ops, check=check)
    node = y.grad_fn.apply if check else y.grad_fn
    want = torch.autograd.grad(y, ops, dy, retain_graph=True)
    assert all(torch.equal(a, b) for a, b in zip(node(dy), want))
    assert all(torch.equal(a, b) for a, b in zip(node(dy.t().contiguous().t()), want))
    for wrong in (dy.cpu(), dy.float(), dy[:8], dy[:, :32], dy.view(-1)):
        with pytest.raises((RuntimeError, ValueError, NotImplementedError)):
            node(wrong)


@pytest.mark.parametrize("check", [False, True])
@pytest.mark.parametrize("reentrant", [False, True])
def test_under_activation_checkpoints(check, reentrant):
    """Recomputed in the backward pass (which ends a recomputation early by raising inside a pack hook)."""
    from torch.utils.checkpoint import checkpoint
    ops = block(40, 128, 72, BF16, grad=True)
    dy = randn(40, 128, seed=4).to(BF16)

    def two(x, wg, wu, wd):
        return vb.gated_ffn(vb.gated_ffn(x, wg, wu, wd, check=check), wg, wu, wd, check=check)

    want = torch.autograd.grad(two(*ops), ops, dy)
    checkpoint(two, *ops, use_reentrant=reentrant).backward(dy)
    assert all(torch.equal(t.grad, w) for t, w in zip(ops, want))


def test_an_exception_of_a_hook_comes_through():
    class Stop(Exception):
        pass

    def pack(_t):
        raise Stop

    ops = block(4, 64, 40, BF16, grad=True)
    for check in (False, True):
        with pytest.raises(Stop), torch.autograd.graph.saved_tensors_hooks(pack, lambda t: t):
            vb.gated_ffn(*ops, check=check)
        with torch.autograd.graph.saved_tensors_hooks(lambda t: t, pack):
            y = vb.gated_ffn(*ops, check=check)
        with pytest.raises(Stop):
            y.sum().backward()


def test_out_counts_as_a_write():
    """A tensor that a backward pass still needs and that then receives a result through out= is
    noticed, as for torch's own out=; an out that requires gradients is refused."""
    ops = block(4, 64, 48, BF16)
    q = [t for w in ops[1:] for t in vb.quantize_int8(w)]
    codes, scale = vb.quantize_int8(ops[0])
    calls = [lambda out: vb.gated_ffn(*ops, out=out), lambda out: vb.int8_gated_ffn(ops[0], *q, out=out),
             lambda out: vb.int8_linear(codes, scale, q[0], q[1], out=out)]
    for call, width in zip(calls, (64, 64, 48)):
        out = torch.ones(4, width, dtype=BF16, device="cuda")
        w = torch.ones(4, width, dtype=BF16, device="cuda", requires_grad=True)
        y = (w * out).sum()
        before = out._version
        assert call(out) is out and out._version == before + 1
        with pytest.raises(RuntimeError, match="modified by an inplace operation"):
            y.backward()
        leaf = torch.ones(4, width, dtype=BF16, device="cuda", requires_grad=True)
        with pytest.raises(RuntimeError, match="out="):
            call(leaf)
        with torch.no_grad():
            call(leaf)
        with torch.inference_mode():
            call(torch.ones(4, width, dtype=BF16, device="cuda"))


def test_views_with_the_negative_bit():
    """A view that torch marks as negated (an imaginary part of a conjugate is one) is taken at its value."""
    x, wg, wu, wd = block(5, 64, 48, BF16)
    neg = torch._neg_view
    want = vb.gated_ffn(-x, wg, wu, wd)
    for check in (False, True):
        assert torch.equal(vb.gated_ffn(neg(x), wg, wu, wd, check=check), want)
        assert torch.equal(vb.gated_ffn(x, wg, neg(wu), wd, check=check), vb.gated_ffn(x, wg, -wu, wd))
        assert torch.equal(vb.gated_ffn(x, wg, wu, neg(wd), check=check), vb.gated_ffn(x, wg, wu, -wd))
    for a, b in zip(vb.quantize_int8(neg(x)), vb.quantize_int8(-x)):
        assert torch.equal(a, b)
    q = [t for w in (wg, wu, wd) for t in vb.quantize_int8(w)]
    codes, scale = vb.quantize_int8(x)
    bias = randn(48)
    assert torch.equal(vb.int8_linear(neg(codes), scale, q[0], neg(q[1]), neg(bias)),
                       vb.int8_linear(-codes, scale, q[0], -q[1], -bias))
    assert torch.equal(vb.int8_gated_ffn(neg(x), *q), vb.int8_gated_ffn(-x, *q))
    leaf = x.clone().requires_grad_(True)
    a, = torch.autograd.grad(vb.gated_ffn(leaf, wg, wu, wd), leaf, neg(x))
    b, = torch.autograd.grad(vb.gated_ffn(leaf, wg, wu, wd, check=True), leaf, neg(x))
    c, = torch.autograd.grad(vb.gated_ffn(leaf, wg, wu, wd), leaf, -x)
    assert torch.equal(a, c) and torch.equal(b, c)
    with pytest.raises(ValueError, match="out"):
        vb.gated_ffn(x, wg, wu, wd, out=neg(torch.zeros_like(x)))


# ── two-part hidden rows ─────────────────────────────────────────────────────────────────────


@pytest.mark.parametrize("tokens,hidden,inter", [(1, 1024, 512), (3, 520, 264), (16, 512, 1032), (32, 1024, 512),
                                                 (33, 1024, 512)])
@pytest.mark.parametrize("dtype,act", [(BF16, "silu"), (F16, "gelu_tanh"), (BF16, "gelu_tanh")])
def test_hidden_rows_in_two_parts_up_to_32_tokens(tokens, hidden, inter, dtype, act):
    """Up to 32 tokens h, dg and du go through their products as a sum of two 16-bit values, so the
    results carry the rounding of the result alone.

    e is the RMS error against 64 bits, e0 that of the 64-bit results rounded once.  Two parts keep
    2^-16 (bf16) or better, fp32 sums 2^-19 of their terms: less than a tenth of the rounding's RMS
    (u / 2), so e <= sqrt(1 + 0.1^2) e0 < 1.05 e0.  One part adds an error of the rounding's own size:
    sqrt(2) e0, which the 64-bit forms on rounded h, dg and du show to be over 1.2 e0 at these sizes."""
    ops = block(tokens, hidden, inter, dtype, grad=True)
    dy = randn(tokens, hidden, seed=7).to(dtype)
    y = vb.gated_ffn(*ops, act=act)
    got = [y.detach(), *torch.autograd.grad(y, ops, dy)]

    x, wg, wu, wd = (t.detach().double() for t in ops)
    a, da = R.act_and_slope(x @ wg.T, act)
    up, dh = x @ wu.T, dy.double() @ wd
    exact_rows = (a * up, dh * up * da, dh * a)

    def results(h, dg, du):
        return [h @ wd.T, dg @ wg + du @ wu, dg.T @ x, du.T @ x, dy.double().T @ h]

    def rms(t):
        return t.pow(2).mean().sqrt().item()

    exact = results(*exact_rows)
    one_part = results(*(t.to(dtype).double() for t in exact_rows))
    for name, g, v, p in zip(("y", "dx", "dw_gate", "dw_up", "dw_down"), got, exact, one_part):
        e0 = rms(v.to(dtype).double() - v)
        assert rms(p.to(dtype).double() - v) > 1.2 * e0, name
        e = rms(g.double() - v)
        assert e <= (1.05 if tokens <= 32 else 1.6) * e0, f"{name}: {e / e0:.3f} times the rounding's error"


# ── sizes and ranges ─────────────────────────────────────────────────────────────────────────


def test_gradients_of_more_values_than_32_bits_count():
    """2.2e9 intermediate values: offsets of g and u, dg, du and h pass 2^31.  Only some rows of dy are
    not zero, so the weight gradients are theirs alone."""
    tokens, hidden, inter = 140_000, 16, 16_384
    ops = block(tokens, hidden, inter, BF16, grad=True)
    rows = torch.tensor([0, 1, 70_000, 131_071, 131_072, 139_998, 139_999], device="cuda")
    dy = torch.zeros(tokens, hidden, dtype=BF16, device="cuda")
    dy[rows] = randn(7, hidden, seed=5).to(BF16)
    y = vb.gated_ffn(*ops)
    dx, *dws = torch.autograd.grad(y, ops, dy)
    few = [ops[0].detach()[rows], *(w.detach() for w in ops[1:])]
    want, bound, parts = R.ffn(*few, "silu", BF16)
    R.assert_within(y[rows], want, bound, "y")
    refs = R.ffn_gradients(parts, dy[rows], BF16)
    R.assert_within(dx[rows], *refs[0], "dx")
    rest = torch.ones(tokens, dtype=torch.bool, device="cuda")
    rest[rows] = False
    assert (dx[rest] == 0).all()
    for name, g, (v, e) in zip(("dw_gate", "dw_up", "dw_down"), dws, refs[1:]):
        R.assert_within(g, v, e, name)


@pytest.mark.parametrize("tokens", [3, 40, 300])
def test_fp16_rows_out_of_range_stay_alone(tokens):
    """h = act(g) u is an fp16 operand of the second product (two up to 32 tokens): beyond 65504 it is
    infinite and its token's result not finite, though the sum itself would be; no other token changes."""
    x, wg, wu, wd = block(tokens, 136, 72, F16)
    want = vb.gated_ffn(x, wg, wu, wd)
    x = x.clone()
    x[1] *= 400 / (x[1].float() @ wg.float().T).abs().amax()
    x[1] = x[1] * 2
    g, up = x[1].double() @ wg.double().T, x[1].double() @ wu.double().T
    h = R.act_and_slope(g, "silu")[0] * up
    assert h.abs().max() > 7e4
    y = vb.gated_ffn(x, wg, wu, wd)
    keep = torch.arange(tokens, device="cuda") != 1
    assert torch.equal(y[keep], want[keep]) and not torch.isfinite(y[1]).any()
