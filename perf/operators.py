"""The operators around the expert FFN whose speed is tracked, called as a training or serving program calls them.

  grouped  products of ragged row segments with one weight per expert (``capi.grouped_linear`` and its gradients)
  linear   a product with bias, activation and residual: the gate projection and the shared expert
           (``capi.linear`` and its gradients)
  norm     layer norm of the hidden states and its gradients (``capi.layer_norm``)

With ``own`` false ``run`` computes the same in elementary torch operations in 32 bits.
"""

import math

import torch

own = False

DEVICE = "cuda:0"
TYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}
EPS = 1e-5

# contraction and output size of one expert's products: gate+up and down of the layer with hidden 7168 and
# intermediate 2048, the same for an intermediate slice of 256 (tensor parallel over 8), the default configuration's
# hidden 4096 with its slice of 384, and small odd ones
EXPERT_SHAPES = ((7168, 4096), (2048, 7168), (7168, 512), (256, 7168), (4096, 768), (384, 4096), (520, 333), (256, 512))
EXPERTS = (1, 5, 16, 32, 64)
# gate projections over 64 and 256 experts, the shared expert's two products, small odd ones
LINEAR_SHAPES = ((7168, 256), (4096, 64), (7168, 2048), (2048, 7168), (4096, 384), (1000, 61), (72, 515))
ACTIVATIONS = ("none", "relu", "silu", "gelu", "gelu_tanh")
HIDDEN = (7168, 4096, 2048, 1031, 512, 100)
MOST_FLOPS = 2 * 32768 * 7168 * 4096


def _grouped(name, direction, dtype, rows, experts, k, n, load="uniform"):
    case = {"op": "grouped", "direction": direction, "dtype": dtype, "rows": rows, "experts": experts, "k": k, "n": n, "load": load}
    return dict(case, name=name) if name else case


def _linear(name, direction, dtype, rows, k, n, activation="none", bias=False, residual=False, out="same", slope=False):
    case = {"op": "linear", "direction": direction, "dtype": dtype, "rows": rows, "k": k, "n": n, "activation": activation,
            "bias": bias, "residual": residual, "out": out, "slope": slope}
    return dict(case, name=name) if name else case


def _norm(name, direction, dtype, rows, hidden):
    case = {"op": "norm", "direction": direction, "dtype": dtype, "rows": rows, "hidden": hidden}
    return dict(case, name=name) if name else case


def listed():
    return [
        # one decode step of 128 sequences on each of 8 expert-parallel ranks: about 32 rows for each of this rank's
        # 32 experts, the weights' stream counts
        _grouped("experts_decode_bf16", "forward", "bf16", 1024, 32, 7168, 4096),
        # a large prefill of the same rank: 1024 rows per expert, the tensor cores count
        _grouped("experts_prefill_bf16", "forward", "bf16", 32768, 32, 7168, 4096),
        # a training step's gradients of the down projection, 512 rows per expert
        _grouped("experts_backward_bf16", "backward", "bf16", 16384, 32, 2048, 7168),
        # the default configuration in half precision with a ragged batch and unequal experts, 777 tokens x 8
        _grouped("experts_backward_fp16_ragged", "backward", "fp16", 6216, 64, 4096, 768, "skewed"),
        # router logits of one decoded token: the smallest call
        _linear("gate_decode_1", "forward", "bf16", 1, 7168, 256, bias=True, out="fp32"),
        # the shared expert's first product for an odd decode batch
        _linear("shared_decode_131", "forward", "bf16", 131, 7168, 2048, "silu"),
        # its second product in a prefill, added to what the routed experts gave
        _linear("shared_prefill_8192", "forward", "bf16", 8192, 2048, 7168, residual=True),
        # its gradients in a training step: input, weight and bias through the activation
        _linear("shared_backward_4096", "backward", "bf16", 4096, 7168, 2048, "gelu_tanh", bias=True, slope=True),
        # layer norm of a small decode batch
        _norm("norm_decode_8", "forward", "bf16", 8, 7168),
        # of a large prefill
        _norm("norm_prefill_32768", "forward", "bf16", 32768, 7168),
        # its gradients in a training step
        _norm("norm_backward_16384", "backward", "bf16", 16384, 7168),
        # the same with an odd width in half precision
        _norm("norm_backward_fp16_odd", "backward", "fp16", 1777, 1031),
    ]


def _log_uniform(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    op = rng.choice(["grouped", "grouped", "linear", "linear", "norm"])
    direction = rng.choice(["forward", "backward"])
    if op == "norm":
        return _norm(None, direction, rng.choice(["bf16", "bf16", "fp16", "fp32"]), _log_uniform(rng, 1, 32768), rng.choice(HIDDEN))
    dtype = rng.choice(["bf16", "bf16", "fp16"])
    times = 4 if direction == "backward" else 2
    if op == "grouped":
        k, n = rng.choice(EXPERT_SHAPES)
        rows = _log_uniform(rng, 1, min(32768, MOST_FLOPS // (times * k * n)))
        return _grouped(None, direction, dtype, rows, rng.choice(EXPERTS), k, n, rng.choice(["uniform", "uniform", "skewed", "sparse"]))
    k, n = rng.choice(LINEAR_SHAPES)
    rows = _log_uniform(rng, 1, 16384)
    activation = rng.choice(ACTIVATIONS)
    if direction == "backward":
        return _linear(None, direction, dtype, rows, k, n, activation, bias=True, slope=activation != "none")
    return _linear(None, direction, dtype, rows, k, n, activation, bias=rng.random() < 0.5, residual=rng.random() < 0.5,
                   out=rng.choice(["same", "same", "fp32"]),
                   # relu's derivative jumps at 0, where the last bit of a sum decides
                   slope=activation not in ("none", "relu") and rng.random() < 0.5)


def _sizes(case, gen):
    """Rows per expert: every row draws its expert; "skewed" prefers the first ones, "sparse" leaves every other one empty."""
    e = case["experts"]
    rank = torch.arange(e, device=DEVICE, dtype=torch.float32)
    p = torch.ones(e, device=DEVICE)
    if case["load"] == "skewed":
        p = (rank + 1.0) ** -0.5
    elif case["load"] == "sparse":
        p = ((rank % 2) == 0).float()
    drawn = torch.multinomial(p, case["rows"], replacement=True, generator=gen)
    return torch.bincount(drawn, minlength=e)


def prepare(case, seed):
    """The tensors that a user's program holds before the call.  ``sizes`` are the segment lengths on the host."""
    gen = torch.Generator(device=DEVICE)
    gen.manual_seed(seed)
    dtype = TYPES[case["dtype"]]

    def normal(*shape, scale=1.0, shift=0.0, to=dtype):
        return torch.randn(*shape, device=DEVICE, generator=gen).mul_(scale).add_(shift).to(to)

    rows = case["rows"]
    if case["op"] == "norm":
        h = case["hidden"]
        s = {"case": case, "x": normal(rows, h, scale=1.5, shift=0.2), "weight": normal(h, scale=0.2, shift=1.0), "bias": normal(h, scale=0.1)}
        if case["direction"] == "backward":
            x = s["x"].double()
            mean = x.mean(1)
            s["mean"] = mean.float()
            s["rstd"] = torch.rsqrt((x - mean[:, None]).square().mean(1) + EPS).float()
            s["dy"] = normal(rows, h, scale=0.1)
        return s
    k, n = case["k"], case["n"]
    s = {"case": case, "x": normal(rows, k)}
    if case["op"] == "grouped":
        sizes = _sizes(case, gen)
        s["offsets"] = torch.nn.functional.pad(sizes.cumsum(0), (1, 0)).to(torch.int32)
        s["sizes"] = sizes.tolist()
        s["w"] = torch.empty(case["experts"], n, k, device=DEVICE, dtype=dtype)
        for e in range(case["experts"]):
            s["w"][e] = normal(n, k, scale=k ** -0.5)
        if case["direction"] == "backward":
            s["dy"] = normal(rows, n, scale=0.1)
        return s
    s["w"] = normal(n, k, scale=k ** -0.5)
    if case["direction"] == "backward":
        s["dy"] = normal(rows, n, scale=0.1)
        s["slope"] = None
        if case["slope"]:
            s["slope"] = _activation(case["activation"], normal(rows, n, to=torch.float32))[1].to(dtype)
        return s
    s["bias"] = normal(n, scale=0.5) if case["bias"] else None
    s["residual"] = normal(rows, n) if case["residual"] else None
    return s


def _activation(name, z):
    """The activation and its derivative."""
    if name == "relu":
        return z.clamp(min=0), (z > 0).to(z.dtype)
    if name == "silu":
        p = 1 / (1 + torch.exp(-z))
        return z * p, p * (1 + z * (1 - p))
    if name == "gelu":
        c = 0.5 * (1 + torch.erf(z * 0.5 ** 0.5))
        return z * c, c + z * torch.exp(-0.5 * z * z) * (0.5 / math.pi) ** 0.5
    if name == "gelu_tanh":
        a = (2 / math.pi) ** 0.5
        t = torch.tanh(a * (z + 0.044715 * z * z * z))
        return 0.5 * z * (1 + t), 0.5 * (1 + t) + 0.5 * z * (1 - t * t) * a * (1 + 3 * 0.044715 * z * z)
    return z, torch.ones_like(z)


def run(state):
    if own:
        return _run_own(state)
    case = state["case"]
    if case["op"] == "grouped":
        return _plain_grouped(state, case)
    if case["op"] == "linear":
        return _plain_linear(state, case)
    return _plain_norm(state, case)


def _run_own(state):
    from moe_bench_b200 import capi

    case = state["case"]
    backward = case["direction"] == "backward"
    if case["op"] == "grouped":
        if backward:
            return capi.grouped_linear_backward(state["dy"], state["x"], state["w"], state["offsets"])
        return capi.grouped_linear(state["x"], state["w"], state["offsets"])
    if case["op"] == "linear":
        if backward:
            return capi.linear_backward(state["dy"], state["x"], state["w"], slope=state["slope"])
        return capi.linear(state["x"], state["w"], bias=state["bias"], activation=case["activation"], residual=state["residual"],
                           out_dtype=torch.float32 if case["out"] == "fp32" else None, want_slope=case["slope"])
    if backward:
        return capi.layer_norm_backward(state["dy"], state["x"], state["mean"], state["rstd"], state["weight"])
    return capi.layer_norm(state["x"], state["weight"], state["bias"], eps=EPS)


def _plain_grouped(state, case):
    x, w, o = state["x"], state["w"].float(), state["offsets"].long()
    # every segment padded to the longest one, a batched product, the rows taken back out
    place = o[:-1, None] + torch.arange(max(max(state["sizes"]), 1), device=x.device)
    real = place < o[1:, None]
    place = place.clamp(max=x.shape[0] - 1)
    xp = x.float()[place] * real[:, :, None]
    if case["direction"] == "forward":
        return torch.bmm(xp, w.transpose(1, 2))[real].to(x.dtype)
    dyp = state["dy"].float()[place] * real[:, :, None]
    dx = torch.bmm(dyp, w)[real].to(x.dtype)
    return dx, torch.bmm(dyp.transpose(1, 2), xp).to(x.dtype)


def _plain_linear(state, case):
    x, w = state["x"].float(), state["w"].float()
    dtype = state["x"].dtype
    if case["direction"] == "backward":
        dz = state["dy"].float()
        if state["slope"] is not None:
            dz = dz * state["slope"].float()
        return (dz @ w).to(dtype), (dz.t() @ x).to(dtype), dz.sum(0)
    z = x @ w.t()
    if state["bias"] is not None:
        z = z + state["bias"].float()
    y, slope = _activation(case["activation"], z)
    if state["residual"] is not None:
        y = y + state["residual"].float()
    y = y.to(torch.float32 if case["out"] == "fp32" else dtype)
    return (y, slope.to(dtype)) if case["slope"] else y


def _plain_norm(state, case):
    x, weight = state["x"].float(), state["weight"].float()
    dtype = state["x"].dtype
    if case["direction"] == "forward":
        mean = x.mean(1)
        centred = x - mean[:, None]
        rstd = torch.rsqrt(centred.square().mean(1) + EPS)
        return (centred * rstd[:, None] * weight + state["bias"].float()).to(dtype), mean, rstd
    dy = state["dy"].float()
    rstd = state["rstd"][:, None]
    h = (x - state["mean"][:, None]) * rstd
    g = dy * weight
    dx = rstd * (g - g.mean(1, keepdim=True) - h * (g * h).mean(1, keepdim=True))
    return dx.to(dtype), (dy * h).sum(0), dy.sum(0)


def _touched(case):
    """Expected number of experts that get a row."""
    e, rows = case["experts"], case["rows"]
    p = [(i + 1.0) ** -0.5 if case["load"] == "skewed" else 1.0 if case["load"] == "uniform" or i % 2 == 0 else 0.0 for i in range(e)]
    return sum(1 - (1 - v / sum(p)) ** rows for v in p)


def work(case):
    size = 4 if case["dtype"] == "fp32" else 2
    rows = case["rows"]
    if case["op"] == "norm":
        h = case["hidden"]
        if case["direction"] == "forward":
            return {"bytes": 2 * rows * h * size + 2 * h * size + 8 * rows, "flops": 8 * rows * h}
        return {"bytes": 3 * rows * h * size + h * (size + 8) + 8 * rows, "flops": 14 * rows * h}
    k, n = case["k"], case["n"]
    if case["op"] == "grouped":
        weights = _touched(case) * n * k * size
        if case["direction"] == "forward":
            return {"bytes": int(rows * (k + n) * size + weights), "flops": 2 * rows * k * n}
        return {"bytes": int(rows * (2 * k + n) * size + weights + case["experts"] * n * k * size), "flops": 4 * rows * k * n}
    if case["direction"] == "backward":
        return {"bytes": (rows * (2 * k + n * (2 if case["slope"] else 1)) + 2 * n * k) * size + 4 * n, "flops": 4 * rows * k * n}
    out = rows * n * (4 if case["out"] == "fp32" else 2) + rows * n * 2 * (case["residual"] + case["slope"])
    return {"bytes": (rows * k + n * k + n * case["bias"]) * size + out, "flops": 2 * rows * k * n}


def exact(case, seed):
    """What ``run`` returns, in 64 bits: segment by segment, derivatives by the chain rule written out."""
    s = prepare(case, seed)
    x = s["x"].double()
    if case["op"] == "grouped":
        parts, grads, begin = [], [], 0
        for e, size in enumerate(s["sizes"]):
            w, rows = s["w"][e].double(), slice(begin, begin + size)
            begin += size
            if case["direction"] == "forward":
                parts.append(x[rows] @ w.t())
            else:
                dy = s["dy"][rows].double()
                parts.append(dy @ w)
                grads.append(torch.einsum("rn,rk->nk", dy, x[rows]).float())  # 64-bit sums, kept in 32
        return torch.cat(parts) if case["direction"] == "forward" else (torch.cat(parts), torch.stack(grads))
    if case["op"] == "linear":
        w = s["w"].double()
        if case["direction"] == "backward":
            dz = s["dy"].double() if s["slope"] is None else s["dy"].double() * s["slope"].double()
            return dz @ w, torch.einsum("rn,rk->nk", dz, x), dz.sum(0)
        z = torch.einsum("rk,nk->rn", x, w)
        if s["bias"] is not None:
            z += s["bias"].double()
        name = case["activation"]
        if name == "relu":
            y, slope = torch.where(z > 0, z, 0.0), torch.where(z > 0, 1.0, 0.0).double()
        elif name == "silu":
            p = torch.sigmoid(z)
            y, slope = z * p, p + z * p * torch.sigmoid(-z)
        elif name == "gelu":
            c = 0.5 * torch.special.erfc(-z / math.sqrt(2.0))
            y, slope = z * c, c + z * torch.exp(-z * z / 2) / math.sqrt(2 * math.pi)
        elif name == "gelu_tanh":
            u = math.sqrt(2 / math.pi) * (z + 0.044715 * z ** 3)
            c = torch.sigmoid(2 * u)  # (1 + tanh u) / 2
            y, slope = z * c, c + 2 * z * c * torch.sigmoid(-2 * u) * math.sqrt(2 / math.pi) * (1 + 0.134145 * z * z)
        else:
            y, slope = z, torch.ones_like(z)
        if s["residual"] is not None:
            y = y + s["residual"].double()
        return (y, slope) if case["slope"] else y
    weight = s["weight"].double()
    if case["direction"] == "forward":
        mean = x.sum(1) / x.shape[1]
        rstd = (x.var(1, unbiased=False) + EPS) ** -0.5
        return torch.addcmul(s["bias"].double(), (x - mean[:, None]) * rstd[:, None], weight), mean, rstd
    dy, rstd = s["dy"].double(), s["rstd"].double()[:, None]
    h = (x - s["mean"].double()[:, None]) * rstd
    g = dy * weight
    inner = (g.sum(1, keepdim=True) + h * torch.einsum("rh,rh->r", g, h)[:, None]) / x.shape[1]
    return (g - inner) * rstd, torch.einsum("rh,rh->h", dy, h), dy.sum(0)
