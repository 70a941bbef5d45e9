"""Cases that the dense feed-forward and 8-bit integer operators are measured on.

The MoE models that the packed-int4 experts come from hold layers that are not packed: the dense
feed-forward blocks in front of the expert layers, shared experts that a checkpoint keeps in 16
bits, and linears in the 8-bit "int-quantized" form.  Four operators serve those:

    ffn, ffn_train   gated_ffn          y = (act(x Wg^T) * (x Wu^T)) Wd^T, and its gradients
    quantize         quantize_int8      one int8 scale per token
    int8_linear      int8_linear        int8 product, scales for each token and output channel
    int8_ffn         int8_gated_ffn     the gated block on int8 weights and int8 activations

Sizes are those of the repository's own layers: 4096 x 14336 (Mixtral-shaped), 2048 x 768
(Qwen3-30B-A3B-shaped), 7168 x 2048 (DeepSeek-V3-shaped), 1024 x 512 (the small layer).
"""
import math

import torch

own = False

DTYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}


def listed():
    return [
        # one decode token through a Mixtral-shaped dense block: the weights' bytes are the cost
        {"name": "ffn decode 1x4096x14336", "op": "ffn", "tokens": 1, "hidden": 4096, "inter": 14336,
         "dtype": "bf16", "act": "silu"},
        # a few tokens (speculative tokens) through the small layer: launch latency
        {"name": "ffn small 3x1024x512", "op": "ffn", "tokens": 3, "hidden": 1024, "inter": 512,
         "dtype": "fp16", "act": "gelu_tanh"},
        # a prompt of 2048 tokens: tensor-core rate
        {"name": "ffn prefill 2048x4096x14336", "op": "ffn", "tokens": 2048, "hidden": 4096, "inter": 14336,
         "dtype": "bf16", "act": "silu"},
        # fine-tuning step of a small block on a ragged packed batch
        {"name": "train ragged 1003x2048x768", "op": "ffn_train", "tokens": 1003, "hidden": 2048, "inter": 768,
         "dtype": "fp16", "act": "gelu_tanh"},
        # fine-tuning step of a Mixtral-shaped dense block
        {"name": "train 2048x4096x14336", "op": "ffn_train", "tokens": 2048, "hidden": 4096, "inter": 14336,
         "dtype": "bf16", "act": "silu"},
        # activations of a decode batch, quantised before an int8 linear: launch latency
        {"name": "quantize 5x7168", "op": "quantize", "tokens": 5, "width": 7168, "dtype": "fp16"},
        # activations of a long prompt in front of a down projection
        {"name": "quantize 4096x14336", "op": "quantize", "tokens": 4096, "width": 14336, "dtype": "bf16"},
        # one decode token through an up projection
        {"name": "int8 linear 1x4096->14336", "op": "int8_linear", "tokens": 1, "width": 4096, "out": 14336,
         "bias": False, "dtype": "bf16"},
        # a ragged decode batch through a shared expert's gate projection, with a bias
        {"name": "int8 linear 37x7168->2048", "op": "int8_linear", "tokens": 37, "width": 7168, "out": 2048,
         "bias": True, "dtype": "fp16"},
        # a prompt through a down projection
        {"name": "int8 linear 2048x14336->4096", "op": "int8_linear", "tokens": 2048, "width": 14336, "out": 4096,
         "bias": False, "dtype": "bf16"},
        # a decode batch through a DeepSeek-V3-shaped shared expert
        {"name": "int8 ffn 16x7168x2048", "op": "int8_ffn", "tokens": 16, "hidden": 7168, "inter": 2048,
         "dtype": "bf16", "act": "silu"},
        # a long prompt through a Mixtral-shaped dense block
        {"name": "int8 ffn 4096x4096x14336", "op": "int8_ffn", "tokens": 4096, "hidden": 4096, "inter": 14336,
         "dtype": "bf16", "act": "silu"},
    ]


def _spread(rng, lo, hi, step=1):
    """A multiple of `step` in [lo, hi], spread over the logarithm of the range."""
    v = math.exp(rng.uniform(math.log(lo), math.log(hi)))
    return max(lo, min(hi, int(v) // step * step))


def draw(rng):
    op = rng.choice(["ffn", "ffn_train", "quantize", "int8_linear", "int8_ffn"])
    dtype = rng.choice(["bf16", "fp16"])
    if op == "quantize":                      # any row length, odd ones too
        width = _spread(rng, 33, 16384)
        return {"op": op, "tokens": _spread(rng, 1, min(8192, 4096 * 14336 // width)), "width": width,
                "dtype": rng.choice(["bf16", "fp16", "fp32"])}
    if op == "int8_linear":                   # K in steps of 16, any number of output channels
        width = _spread(rng, 256, 14336, 16)
        out = _spread(rng, 97, 4096 * 14336 // width if width > 4096 else 14336)
        return {"op": op, "tokens": _spread(rng, 1, min(8192, 2048 * 14336 * 4096 // (width * out))), "width": width,
                "out": out, "bias": rng.random() < 0.5, "dtype": rng.choice(["bf16", "fp16", "fp32"])}
    step = 16 if op == "int8_ffn" else 8
    hidden = _spread(rng, 512, 8192, step)
    inter = _spread(rng, 256, min(16384, 4096 * 14336 // hidden), step)
    most = (4096 if op == "int8_ffn" else 2048) * 4096 * 14336 // (hidden * inter)
    return {"op": op, "tokens": _spread(rng, 1, min(8192, most)), "hidden": hidden, "inter": inter, "dtype": dtype,
            "act": rng.choice(["silu", "gelu_tanh"])}


def _channel_codes(w):
    """Int8 codes and fp32 scales of a weight, one scale for each output channel."""
    scale = w.abs().amax(dim=1) / 127.0
    return torch.clamp(torch.round(w / scale[:, None]), -127, 127).to(torch.int8), scale


def prepare(case, seed):
    gen = torch.Generator(device="cuda").manual_seed(seed)

    def randn(*shape):
        return torch.randn(*shape, generator=gen, device="cuda")

    def weight(rows, cols):                   # unit-variance outputs for unit-variance inputs
        return randn(rows, cols) / math.sqrt(cols)

    op, t, dt = case["op"], case["tokens"], DTYPES[case["dtype"]]
    state = {"op": op, "act": case.get("act"), "dtype": dt}
    if op in ("ffn", "ffn_train"):
        h, i = case["hidden"], case["inter"]
        train = op == "ffn_train"
        state["x"] = randn(t, h).to(dt).requires_grad_(train)
        state["wg"] = weight(i, h).to(dt).requires_grad_(train)
        state["wu"] = weight(i, h).to(dt).requires_grad_(train)
        state["wd"] = weight(h, i).to(dt).requires_grad_(train)
        if train:
            state["dy"] = randn(t, h).to(dt)
    elif op == "quantize":
        # token rows of different sizes, as hidden states have
        state["x"] = (randn(t, case["width"]) * torch.exp(randn(t, 1))).to(dt)
    elif op == "int8_linear":
        state["codes"], state["scale"] = _channel_codes(randn(t, case["width"]))
        state["scale"] = state["scale"][:, None]
        state["w"], state["ws"] = _channel_codes(weight(case["out"], case["width"]))
        state["bias"] = randn(case["out"]).to(dt) if case["bias"] else None
    else:
        h, i = case["hidden"], case["inter"]
        state["x"] = randn(t, h).to(dt)
        state["wg"], state["sg"] = _channel_codes(weight(i, h))
        state["wu"], state["su"] = _channel_codes(weight(i, h))
        state["wd"], state["sd"] = _channel_codes(weight(h, i))
    return state


# ── the operators in their plain form ────────────────────────────────────────────────────────


def _act(g, name):
    """The activation and its derivative."""
    if name == "silu":
        s = 1 / (1 + torch.exp(-g))
        return g * s, s * (1 + g * (1 - s))
    c = math.sqrt(2 / math.pi)
    t = torch.tanh(c * (g + 0.044715 * g * g * g))
    return 0.5 * g * (1 + t), 0.5 * (1 + t) + 0.5 * g * (1 - t * t) * c * (1 + 3 * 0.044715 * g * g)


def _plain_ffn(s):
    x, wg, wu, wd = (s[k].detach().float() for k in ("x", "wg", "wu", "wd"))
    g, u = x @ wg.T, x @ wu.T
    a, da = _act(g, s["act"])
    h = a * u
    y = (h @ wd.T).to(s["dtype"])
    if s["op"] == "ffn":
        return y
    dy = s["dy"].float()
    dh = dy @ wd
    dg, du = dh * u * da, dh * a
    dx = dg @ wg + du @ wu
    return [v.to(s["dtype"]) for v in (y, dx, dg.T @ x, du.T @ x, dy.T @ h)]


def _plain_quantize(x):
    """Codes: the nearest integers of the exact quotient x / scale, ties to even (64 bits, since
    the quotients lie next to ties)."""
    scale = (x.float().abs().amax(dim=-1, keepdim=True).double() / 127).float()
    codes = torch.round(x.double() / scale.double()).clamp(-127, 127)
    return torch.where(scale > 0, codes, 0.0).to(torch.int8), scale


def _plain_product(codes, scale, w, ws):
    """Int8 products summed exactly (64 bits: the sums pass 2^24), then scaled in 32."""
    return (codes.double() @ w.double().T).float() * scale * ws.float()[None, :]


def _plain(s):
    if s["op"] in ("ffn", "ffn_train"):
        return _plain_ffn(s)
    if s["op"] == "quantize":
        return _plain_quantize(s["x"])
    if s["op"] == "int8_linear":
        y = _plain_product(s["codes"], s["scale"], s["w"], s["ws"])
        return (y if s["bias"] is None else y + s["bias"].float()).to(s["dtype"])
    codes, scale = _plain_quantize(s["x"])
    g = _plain_product(codes, scale, s["wg"], s["sg"])
    h = _act(g, s["act"])[0] * _plain_product(codes, scale, s["wu"], s["su"])
    return _plain_product(*_plain_quantize(h), s["wd"], s["sd"]).to(s["dtype"])


def _own(s):
    import vaayu_b200 as vb

    if s["op"] == "ffn":
        return vb.gated_ffn(s["x"], s["wg"], s["wu"], s["wd"], act=s["act"])
    if s["op"] == "ffn_train":
        leaves = (s["x"], s["wg"], s["wu"], s["wd"])
        y = vb.gated_ffn(*leaves, act=s["act"])
        return [y, *torch.autograd.grad(y, leaves, s["dy"])]
    if s["op"] == "quantize":
        return vb.quantize_int8(s["x"])
    if s["op"] == "int8_linear":
        return vb.int8_linear(s["codes"], s["scale"], s["w"], s["ws"], bias=s["bias"], dtype=s["dtype"])
    return vb.int8_gated_ffn(s["x"], s["wg"], s["sg"], s["wu"], s["su"], s["wd"], s["sd"], act=s["act"])


def run(state):
    return _own(state) if own else _plain(state)


def work(case):
    t, size = case["tokens"], {"bf16": 2, "fp16": 2, "fp32": 4}[case["dtype"]]
    if case["op"] == "quantize":
        return {"bytes": t * (case["width"] * (size + 1) + 4), "flops": 3 * t * case["width"]}
    if case["op"] == "int8_linear":
        k, n = case["width"], case["out"]
        return {"bytes": t * (k + 4) + n * (k + 4 + size * case["bias"]) + t * n * size, "flops": 2 * t * k * n}
    h, i = case["hidden"], case["inter"]
    if case["op"] == "int8_ffn":
        return {"bytes": 3 * h * i + 4 * (2 * i + h) + 2 * t * h * size, "flops": 6 * t * h * i}
    if case["op"] == "ffn":
        return {"bytes": size * (3 * h * i + 2 * t * h), "flops": 6 * t * h * i}
    return {"bytes": size * (6 * h * i + 4 * t * h), "flops": 18 * t * h * i}


# ── the definitions in 64 bits ───────────────────────────────────────────────────────────────


def _exact_gate(g, act):
    if act == "silu":
        return g * torch.sigmoid(g)
    return g * 0.5 * (1.0 + torch.tanh(0.7978845608028654 * g * (1.0 + 0.044715 * g ** 2)))


def _exact_codes(x):
    """(codes, scale) as float64: the scale is a 32-bit number, the quotient and its rounding are
    exact (an integer q with |x - q s| smallest, even where two tie)."""
    s = (x.abs().amax(-1, keepdim=True) / 127.0).float().double()
    q = x / torch.where(s > 0, s, torch.ones_like(s))
    low = torch.floor(q)
    rest = q - low
    up = (rest > 0.5) | ((rest == 0.5) & (torch.remainder(low, 2.0) == 1.0))
    return torch.where(s > 0, (low + up.double()).clamp(-127.0, 127.0), torch.zeros_like(q)), s


def exact(case, seed):
    s = prepare(case, seed)
    op = s["op"]
    if op == "quantize":
        codes, scale = _exact_codes(s["x"].double())
        return codes.to(torch.int8), scale
    if op == "int8_linear":
        y = torch.einsum("tk,nk->tn", s["codes"].double() * s["scale"].double(),
                         s["w"].double() * s["ws"].double()[:, None])
        return y if s["bias"] is None else y + s["bias"].double()
    if op == "int8_ffn":
        c, sc = _exact_codes(s["x"].double())
        gate = torch.einsum("tk,nk->tn", c * sc, s["wg"].double() * s["sg"].double()[:, None])
        up = torch.einsum("tk,nk->tn", c * sc, s["wu"].double() * s["su"].double()[:, None])
        c, sc = _exact_codes(_exact_gate(gate, case["act"]) * up)
        return torch.einsum("tk,nk->tn", c * sc, s["wd"].double() * s["sd"].double()[:, None])
    x, wg, wu, wd = (s[k].detach().double().requires_grad_(op == "ffn_train") for k in ("x", "wg", "wu", "wd"))
    hidden = _exact_gate(torch.nn.functional.linear(x, wg), case["act"]) * torch.nn.functional.linear(x, wu)
    y = torch.nn.functional.linear(hidden, wd)
    if op == "ffn":
        return y
    return [y.detach(), *torch.autograd.grad(y, (x, wg, wu, wd), s["dy"].double())]
