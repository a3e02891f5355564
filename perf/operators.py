"""What is measured of the gated feed-forward projections and of the linear layers over 4-bit weights: the cases, their
inputs, their plain form in elementary torch operations, the calls of the framework that compute the same, and the
definition in 64 bits.

Operators (x ``[T, K]``, one row for each token):

``gated``        ``h = act(x G^T) * (x U^T)`` with G, U the first and the second half of the rows of ``gate_up [2I, K]``
``gated_train``  the same, and for a gradient ``dh`` of h the gradients of x and of gate_up
``int4``         ``y = x W^T`` with ``W[n, k] = scale[n, k/g] * (code[n, k] - zero[n, k/g])``, codes of 4 bits, groups of g
``int4_gated``   ``h = act(x G^T) * (x U^T)`` with the 2I rows of gate_up in 4 bits
"""
import math

import torch

own = False

_DTYPES = {"bf16": torch.bfloat16, "fp16": torch.float16}


def listed():
    return [
        # one token of a decoder layer's feed-forward: the weights are read once, nothing else counts
        {"name": "gated_1_token", "op": "gated", "t": 1, "k": 4096, "i": 14336, "act": "silu", "dtype": "bf16", "pad": 0},
        # a decode batch, whose rows are a slice of a wider buffer
        {"name": "gated_100_tokens", "op": "gated", "t": 100, "k": 7168, "i": 2048, "act": "silu", "dtype": "bf16",
         "pad": 128},
        # a prompt of odd length
        {"name": "gated_1037_tokens", "op": "gated", "t": 1037, "k": 4096, "i": 14336, "act": "gelu_tanh", "dtype": "fp16",
         "pad": 0},
        # a training step of a small layer with sizes off every tile
        {"name": "train_333_tokens", "op": "gated_train", "t": 333, "k": 1032, "i": 2744, "act": "gelu", "dtype": "fp16",
         "pad": 0},
        # a training step of a narrow expert
        {"name": "train_2000_tokens", "op": "gated_train", "t": 2000, "k": 7168, "i": 2048, "act": "silu", "dtype": "bf16",
         "pad": 0},
        # a training step of a wide layer
        {"name": "train_8192_tokens", "op": "gated_train", "t": 8192, "k": 4096, "i": 14336, "act": "silu", "dtype": "bf16",
         "pad": 0},
        # the smallest call of a decode step: an output projection for one token
        {"name": "int4_1_token_square", "op": "int4", "t": 1, "k": 4096, "n": 4096, "group": 128, "zero": False,
         "dtype": "bf16"},
        # a down projection for one token
        {"name": "int4_1_token_down", "op": "int4", "t": 1, "k": 14336, "n": 4096, "group": 128, "zero": True,
         "dtype": "fp16"},
        # a decode batch on a wide projection, small groups
        {"name": "int4_16_tokens", "op": "int4", "t": 16, "k": 4096, "n": 28672, "group": 64, "zero": True, "dtype": "bf16"},
        # the feed-forward of one token
        {"name": "int4_gated_1_token", "op": "int4_gated", "t": 1, "k": 4096, "i": 14336, "group": 128, "zero": True,
         "act": "silu", "dtype": "bf16"},
        # five sequences on a narrow expert, the smallest groups
        {"name": "int4_gated_5_tokens", "op": "int4_gated", "t": 5, "k": 7168, "i": 2048, "group": 32, "zero": False,
         "act": "gelu_tanh", "dtype": "fp16"},
        # a larger decode batch
        {"name": "int4_gated_48_tokens", "op": "int4_gated", "t": 48, "k": 4096, "i": 14336, "group": 128, "zero": True,
         "act": "silu", "dtype": "bf16"},
    ]


def draw(rng):
    def spread(lo, hi):
        return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))

    op = rng.choice(["gated", "gated_train", "int4", "int4_gated"])
    case = {"op": op, "dtype": rng.choice(["bf16", "fp16"])}
    if op in ("gated", "gated_train"):
        k, i = 8 * spread(64, 1024), 8 * spread(64, 2048)
        i += rng.choice([0, 0, 0, 1, 5])
        # no more products than the largest listed case
        case.update(t=min(spread(1, 8192), 8192 * 4096 * 14336 // (k * i)), k=k, i=i,
                    act=rng.choice(["silu", "gelu", "gelu_tanh"]), pad=rng.choice([0, 0, 8, 256]))
    else:
        g = rng.choice([32, 64, 128])
        case.update(t=spread(1, 64), k=g * spread(512 // g, 14336 // g), group=g, zero=rng.random() < 0.5)
        rows = spread(512, 28672) + rng.choice([0, 0, 1])
        if op == "int4":
            case.update(n=rows)
        else:
            case.update(i=(rows + 1) // 2, act=rng.choice(["silu", "gelu", "gelu_tanh"]))
    return case


def _four_bits(w, group, zero):
    """Codes, scales and zero points of w by rounding to the nearest step of each group: what a checkpoint stores."""
    n, k = w.shape
    v = w.view(n, k // group, group)
    if zero:
        lo, hi = v.amin(-1).clamp(max=0), v.amax(-1).clamp(min=0)
        scale = ((hi - lo) / 15).clamp(min=1e-6)
        z = torch.round(-lo / scale).clamp(0, 15)
    else:
        scale = (v.abs().amax(-1) / 7.5).clamp(min=1e-6)
        z = torch.full_like(scale, 8)
    q = (torch.round(v / scale[..., None]) + z[..., None]).clamp(0, 15).to(torch.uint8).view(n, k // 2, 2)
    return q[..., 0] | (q[..., 1] << 4), scale, z.to(torch.uint8) if zero else None


def prepare(case, seed):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    dtype = _DTYPES[case["dtype"]]
    t, k = case["t"], case["k"]

    def normal(*shape, std=1.0):
        return std * torch.randn(*shape, generator=gen, device="cuda")

    state = {"op": case["op"], "act": case.get("act")}
    if case["op"] in ("gated", "gated_train"):
        i = case["i"]
        x = normal(t, k + case["pad"]).to(dtype)[:, :k]
        gate_up = normal(2 * i, k, std=0.02).to(dtype)
        if case["op"] == "gated_train":
            state["dh"] = normal(t, i).to(dtype)
            x, gate_up = x.detach().requires_grad_(), gate_up.requires_grad_()
        return dict(state, x=x, gate_up=gate_up)
    rows = case["n"] if case["op"] == "int4" else 2 * case["i"]
    codes, scale, zero = _four_bits(normal(rows, k, std=0.02), case["group"], case["zero"])
    state.update(x=normal(t, k).to(dtype), codes=codes, scale=scale.to(dtype), zero=zero)
    if own:  # the handle that a program makes of a checkpoint once, when it loads it
        import fish_scales_ops_b200 as fso

        state["weight"] = fso.int4.prepare_weight(codes, state["scale"], zero)
    return state


def _act(g, act):
    if act == "silu":
        return g / (1 + torch.exp(-g))
    if act == "gelu":
        return 0.5 * g * (1 + torch.erf(g * math.sqrt(0.5)))
    return 0.5 * g * (1 + torch.tanh(math.sqrt(2 / math.pi) * (g + 0.044715 * g * g * g)))


def _act_slope(g, act):
    if act == "silu":
        s = 1 / (1 + torch.exp(-g))
        return s * (1 + g * (1 - s))
    if act == "gelu":
        return 0.5 * (1 + torch.erf(g * math.sqrt(0.5))) + g * torch.exp(-0.5 * g * g) / math.sqrt(2 * math.pi)
    c = math.sqrt(2 / math.pi)
    th = torch.tanh(c * (g + 0.044715 * g * g * g))
    return 0.5 * (1 + th) + 0.5 * g * (1 - th * th) * c * (1 + 3 * 0.044715 * g * g)


def _weights(codes, scale, zero):
    q = torch.stack((codes & 15, codes >> 4), dim=-1).view(*scale.shape, -1).float()
    z = 8 if zero is None else zero.float()[..., None]
    return ((q - z) * scale.float()[..., None]).flatten(1)


def _run_own(s):
    import fish_scales_ops_b200 as fso

    if s["op"] == "gated":
        return fso.ffn.gated_linear(s["x"], s["gate_up"], activation=s["act"])
    if s["op"] == "gated_train":
        h = fso.ffn.gated_linear(s["x"], s["gate_up"], activation=s["act"])
        dx, dw = torch.autograd.grad(h, (s["x"], s["gate_up"]), s["dh"])
        return {"h": h.detach(), "dx": dx, "dgate_up": dw}
    if s["op"] == "int4":
        return fso.int4.linear(s["x"], s["weight"])
    return fso.int4.gated_linear(s["x"], s["weight"], activation=s["act"])


@torch.no_grad()
def _run_plain(s):
    dtype = s["x"].dtype
    x = s["x"].float()
    if s["op"] == "int4":
        return (x @ _weights(s["codes"], s["scale"], s["zero"]).t()).to(dtype)
    w = s["gate_up"].float() if "gate_up" in s else _weights(s["codes"], s["scale"], s["zero"])
    inter = w.shape[0] // 2
    wg, wu = w[:inter], w[inter:]
    g, u = x @ wg.t(), x @ wu.t()
    a = _act(g, s["act"])
    h = (a * u).to(dtype)
    if s["op"] != "gated_train":
        return h
    dh = s["dh"].float()
    dg, du = dh * u * _act_slope(g, s["act"]), dh * a
    return {"h": h, "dx": (dg @ wg + du @ wu).to(dtype), "dgate_up": torch.cat((dg.t() @ x, du.t() @ x)).to(dtype)}


def run(state):
    return _run_own(state) if own else _run_plain(state)


def work(case):
    t, k = case["t"], case["k"]
    if case["op"] == "gated":
        i = case["i"]
        return {"bytes": 2 * (t * k + 2 * i * k + t * i), "flops": 4 * t * k * i}
    if case["op"] == "gated_train":
        i = case["i"]  # x, gate_up and dh in; h and the gradients of x and gate_up out; three products of one size
        return {"bytes": 2 * (2 * t * k + 2 * 2 * i * k + 2 * t * i), "flops": 12 * t * k * i}
    rows, out = (case["n"], case["n"]) if case["op"] == "int4" else (2 * case["i"], case["i"])
    groups = rows * k // case["group"]
    return {"bytes": rows * k // 2 + groups * (3 if case["zero"] else 2) + 2 * t * (k + out), "flops": 2 * t * rows * k}


@torch.no_grad()
def exact(case, seed):
    """The definition in 64 bits, products by blocks of 2048 weight rows; gradients by the chain rule on each block."""
    s = prepare(case, seed)
    x = s["x"].detach().double()
    t, k = case["t"], case["k"]

    def rows_of(lo, hi):
        if "gate_up" in s:
            return s["gate_up"][lo:hi].detach().double()
        w = torch.empty(hi - lo, k, dtype=torch.float64, device="cuda")
        w[:, 0::2], w[:, 1::2] = (s["codes"][lo:hi] % 16).double(), (s["codes"][lo:hi] // 16).double()
        z = s["zero"][lo:hi].double() if s["zero"] is not None else torch.tensor(8.0, dtype=torch.float64, device="cuda").expand(
            hi - lo, k // case["group"])
        w -= z.repeat_interleave(case["group"], dim=1)
        w *= s["scale"][lo:hi].double().repeat_interleave(case["group"], dim=1)
        return w

    if case["op"] == "int4":
        y = torch.empty(t, case["n"], dtype=torch.float64, device="cuda")
        for lo in range(0, case["n"], 2048):
            hi = min(case["n"], lo + 2048)
            y[:, lo:hi] = torch.einsum("tk,nk->tn", x, rows_of(lo, hi))
        return y
    i = case["i"]
    h = torch.empty(t, i, dtype=torch.float64, device="cuda")
    train = case["op"] == "gated_train"
    if train:
        dx, dw, dh = torch.zeros_like(x), torch.empty(2 * i, k, dtype=torch.float64, device="cuda"), s["dh"].double()
    for lo in range(0, i, 2048):
        hi = min(i, lo + 2048)
        wg, wu = rows_of(lo, hi), rows_of(i + lo, i + hi)
        g, u = torch.einsum("tk,nk->tn", x, wg), torch.einsum("tk,nk->tn", x, wu)
        if case["act"] == "silu":
            cdf = torch.sigmoid(g)
            slope = cdf + g * cdf * torch.sigmoid(-g)
        elif case["act"] == "gelu":
            cdf = 0.5 * torch.erfc(-g / math.sqrt(2.0))
            slope = cdf + g * torch.exp(-g.square() / 2) / math.sqrt(2 * math.pi)
        else:  # 0.5 (1 + tanh z) = 1 / (1 + exp(-2 z))
            inner = 2 * math.sqrt(2 / math.pi) * (g + 0.044715 * g ** 3)
            cdf = torch.sigmoid(inner)
            slope = cdf + g * cdf * torch.sigmoid(-inner) * 2 * math.sqrt(2 / math.pi) * (1 + 0.134145 * g.square())
        h[:, lo:hi] = g * cdf * u
        if train:
            dg, du = dh[:, lo:hi] * u * slope, dh[:, lo:hi] * g * cdf
            dx += torch.einsum("tn,nk->tk", dg, wg) + torch.einsum("tn,nk->tk", du, wu)
            dw[lo:hi], dw[i + lo:i + hi] = torch.einsum("tn,tk->nk", dg, x), torch.einsum("tn,tk->nk", du, x)
    return {"h": h, "dx": dx, "dgate_up": dw} if train else h
