"""Plain 64-bit forms of the dense operators, with bounds on what a right kernel may be off.

A bound follows the roundings one by one.  u is half a step of the 16-bit type relative to the value
(bf16 2^-8... as finfo.eps / 2), `tiny` half its smallest subnormal.  An fp32 sum of K products on
the tensor cores is off by at most (K / 16 + 8) 2^-23 sum |a b|: one truncation to an fp32 step for
each group of 16 products, and a few for joining partial sums; the elementwise fp32 steps (activation
and products) by 2^-20 relative.  act' <= 1.13 and |act''| <= 0.8 for both activations."""
import math

import torch

SLOPE, CURVE, STEP32 = 1.13, 0.8, 2.0 ** -20


def unit(dtype):
    return torch.finfo(dtype).eps / 2


def tiny(dtype):
    return torch.finfo(dtype).smallest_normal * torch.finfo(dtype).eps / 2 if dtype == torch.float16 else 0.0


def sum_error(k):
    return (k / 16 + 8) * 2.0 ** -23


def act_and_slope(g, act):
    if act == "silu":
        s = torch.sigmoid(g)
        return g * s, s * (1 + g * (1 - s))
    c = math.sqrt(2 / math.pi)
    t = torch.tanh(c * (g + 0.044715 * g ** 3))
    return 0.5 * g * (1 + t), 0.5 * (1 + t) + 0.5 * g * (1 - t * t) * c * (1 + 3 * 0.044715 * g * g)


def ffn(x, wg, wu, wd, act, dtype):
    """(y, bound on |y - kernel's y|) and the pieces the gradients need, all fp64."""
    x, wg, wu, wd = (t.detach().double() for t in (x, wg, wu, wd))
    u = unit(dtype)
    g, up = x @ wg.T, x @ wu.T
    eg, eu = (sum_error(x.shape[1]) * (x.abs() @ w.abs().T) for w in (wg, wu))
    a, da = act_and_slope(g, act)
    h = a * up
    eh = SLOPE * eg * up.abs() + a.abs() * eu + SLOPE * eg * eu + STEP32 * h.abs()
    eh = eh * (1 + u) + u * h.abs() + tiny(dtype)
    y = h @ wd.T
    ey = eh @ wd.abs().T + sum_error(wd.shape[1]) * (h.abs() @ wd.abs().T)
    ey = ey * (1 + u) + u * y.abs() + tiny(dtype)
    return y, ey, dict(x=x, wg=wg, wu=wu, wd=wd, g=g, up=up, eg=eg, eu=eu, a=a, da=da, h=h, eh=eh)


def ffn_gradients(p, dy, dtype):
    """[(gradient, bound)] for x, w_gate, w_up, w_down."""
    dy, u, t = dy.double(), unit(dtype), tiny(dtype)
    dh = dy @ p["wd"]
    edh = sum_error(dy.shape[1]) * (dy.abs() @ p["wd"].abs())
    dg, du = dh * p["up"] * p["da"], dh * p["a"]
    # products of perturbed factors: |ab - a'b'| <= |a| eb + |b| ea + ea eb, twice
    fu, efu = p["up"].abs() * p["da"].abs(), None
    eda = CURVE * p["eg"]
    efu = p["up"].abs() * eda + p["da"].abs() * p["eu"] + eda * p["eu"]
    edg = dh.abs() * efu + fu * edh + edh * efu + 2 * STEP32 * dh.abs() * p["up"].abs() * SLOPE
    ea = SLOPE * p["eg"]
    edu = dh.abs() * ea + p["a"].abs() * edh + edh * ea + STEP32 * du.abs()
    edg = edg * (1 + u) + u * dg.abs() + t
    edu = edu * (1 + u) + u * du.abs() + t
    out = []

    def product(a, ea_, b, eb_, k):
        v = a @ b
        e = ea_ @ b.abs() + a.abs() @ eb_ + sum_error(k) * (a.abs() @ b.abs())
        return v, e

    zero = torch.zeros_like
    v1, e1 = product(dg, edg, p["wg"], zero(p["wg"]), 2 * dg.shape[1])
    v2, e2 = product(du, edu, p["wu"], zero(p["wu"]), 2 * du.shape[1])
    out.append((v1 + v2, e1 + e2))
    out.append(product(dg.T, edg.T, p["x"], zero(p["x"]), dg.shape[0]))
    out.append(product(du.T, edu.T, p["x"], zero(p["x"]), du.shape[0]))
    out.append(product(dy.T, zero(dy.T), p["h"], p["eh"], dy.shape[0]))
    return [(v, e * (1 + u) + u * v.abs() + t) for v, e in out]


def assert_within(got, want, bound, what):
    got = got.detach().double()
    assert got.shape == want.shape, f"{what}: {tuple(got.shape)} for {tuple(want.shape)}"
    assert torch.isfinite(got).all(), f"{what}: not finite"
    over = (got - want).abs() - bound
    worst = over.max().item() if over.numel() else 0.0
    assert worst <= 0, f"{what}: {worst:.3e} over the bound (of {bound.max().item():.3e} at most)"


def quantize(x):
    """(codes int8, scale fp32): nearest integers of the exact quotients, ties to even."""
    top = x.double().abs().amax(dim=-1, keepdim=True)
    scale = (top / 127).float()
    q = torch.round(x.double() / torch.where(scale > 0, scale, 1.0).double()).clamp(-127, 127)
    return torch.where(scale > 0, q, 0.0).to(torch.int8), scale


def int8_product(codes, scale, weight, weight_scale, bias=None):
    """The scaled product as the operator defines it: exact sum, then single fp32 roundings."""
    acc = (codes.double() @ weight.double().T)              # integers below 2^53: exact
    y = acc.float() * scale.reshape(-1, 1).float() * weight_scale.reshape(1, -1).float()
    return y if bias is None else y + bias.float()


def int8_ffn(x, wg, sg, wu, su, wd, sd, act, dtype):
    """(y, bound) of the int8 block, fp64.  g and u carry three fp32 roundings; a code of h may be off
    by one where its quotient lies nearer to a tie than the error of that quotient."""
    u = unit(dtype)
    codes, scale = quantize(x)
    g = (codes.double() @ wg.double().T) * scale.double() * sg.double()[None]
    up = (codes.double() @ wu.double().T) * scale.double() * su.double()[None]
    a = act_and_slope(g, act)[0]
    h = a * up
    eh = (SLOPE * g.abs() * up.abs() + a.abs() * up.abs()) * 2.0 ** -22 + STEP32 * h.abs()
    top = h.abs().amax(dim=-1, keepdim=True)
    s = (top / 127).float().double()
    rel = torch.where(top > 0, eh.amax(dim=-1, keepdim=True) / torch.where(top > 0, top, 1.0), 0.0) + 2.0 ** -23
    q = h / torch.where(s > 0, s, 1.0)
    eq = eh / torch.where(s > 0, s, 1.0) + q.abs() * rel
    near = ((q - torch.floor(q) - 0.5).abs() <= eq).double()
    codes_h = torch.round(q).clamp(-127, 127)
    wds = wd.double() * sd.double()[:, None]
    y = (codes_h @ wd.double().T) * s * sd.double()[None]      # integer sums: exact, zeros stay zero
    ey = (near * s) @ wds.abs().T * (1 + rel) + y.abs() * (rel + 2.0 ** -22) + (near * s) @ wds.abs().T * rel
    return y, ey * (1 + u) + u * y.abs() + tiny(dtype)
