"""Cases and plain forms of the operators of a gated feed-forward block: the gated projection pair, counter-based dropout
and the root-mean-square norm, forward and backward.

    listed()            the fixed cases
    draw(rng)           one more case of the same ranges
    prepare(case, seed) what a program holds before the call
    run(state)          one pass: the plain form (own == False) or this package's operators (own == True)
    exact(case, seed)   the same outputs from the definition in 64 bits
    work(case)          bytes and operations that a pass cannot do without

Formulas (x [rows, cols], w = the gate and the up projection stacked [2, cols, width]):
    gated forward    pre_b = x w_b;  h = dropout(act(pre_0) * pre_1)
    gated backward   d = dropout'(dz);  dpre_0 = d pre_1 act'(pre_0);  dpre_1 = d act(pre_0);
                     dx = sum_b dpre_b w_b^T;  dw_b = x^T dpre_b
    dropout          y = residual + keep(i) x / (1 - p);  dx = keep(i) dy / (1 - p)
    keep(i)          word i % 4 of Philox4x32-10 (Salmon, Moraes, Dror, Shaw: Parallel random numbers: as easy as 1, 2, 3,
                     SC 2011) at counter (i / 4, offset) under key = seed is at least p * 2^32
    norm forward     rstd = 1 / sqrt(mean(x^2) + eps);  y = x rstd weight
    norm backward    u = dy weight;  dx = rstd (u - x rstd mean(u x rstd));  dweight = sum over rows of dy x rstd
"""
import math

import torch

own = False

_MASK = 0xFFFFFFFF
_EPS = 1e-6
_DTYPES = {"fp16": torch.float16, "fp32": torch.float32}
_context = None


# ------------------------------------------------------------------------------------------------------------ cases
def listed():
    return [
        # One token through the block's up-projections while a model answers: the sizes of the two-layer product that
        # bench.py runs (4096 -> 16384).  Bound by reading the weights.
        {"name": "gated_token", "op": "gated_forward", "dtype": "fp16", "rows": 1, "cols": 4096, "width": 16384, "act": "silu",
         "keep_pre": False, "p": 0.0},
        # One step for 48 sequences that are answered together: still bound by the weights, more than a vector.
        {"name": "gated_batch48", "op": "gated_forward", "dtype": "fp16", "rows": 48, "cols": 2048, "width": 5504, "act": "silu",
         "keep_pre": False, "p": 0.0},
        # Training, the per-GPU shard of bench.py's two-layer product (8192 rows), projections kept for the backward pass.
        {"name": "gated_train", "op": "gated_forward", "dtype": "fp16", "rows": 8192, "cols": 4096, "width": 16384, "act": "silu",
         "keep_pre": True, "p": 0.0},
        # Training a smaller model on packed sequences (a row count that is no multiple of anything) with dropout inside.
        {"name": "gated_train_dropout", "op": "gated_forward", "dtype": "fp16", "rows": 1531, "cols": 1024, "width": 4096,
         "act": "gelu_tanh", "keep_pre": True, "p": 0.1},
        # 32-bit training with sizes that leave every row off a 16-byte boundary.
        {"name": "gated_train_fp32_odd", "op": "gated_forward", "dtype": "fp32", "rows": 333, "cols": 250, "width": 1001, "act": "gelu",
         "keep_pre": True, "p": 0.0},
        # The gradients of gated_train.
        {"name": "gated_backward", "op": "gated_backward", "dtype": "fp16", "rows": 8192, "cols": 4096, "width": 16384, "act": "silu",
         "p": 0.0},
        # The gradients of a small 32-bit block with dropout inside.
        {"name": "gated_backward_fp32", "op": "gated_backward", "dtype": "fp32", "rows": 640, "cols": 384, "width": 1536, "act": "silu",
         "p": 0.1},
        # Dropout of a block's output onto the residual stream, 8192 tokens of 4096 features.
        {"name": "dropout_residual", "op": "dropout_forward", "dtype": "fp16", "rows": 8192, "cols": 4096, "p": 0.1, "residual": True},
        # Its gradient in 32 bits over a count that is no multiple of the generator's four words.
        {"name": "dropout_backward_odd", "op": "dropout_backward", "dtype": "fp32", "rows": 1, "cols": 4000003, "p": 0.25},
        # The norm in front of the block for one token: latency.
        {"name": "norm_token", "op": "norm_forward", "dtype": "fp16", "rows": 1, "cols": 4096},
        # The norm in training, 32 bits, an odd row count.
        {"name": "norm_train_fp32", "op": "norm_forward", "dtype": "fp32", "rows": 12289, "cols": 1000},
        # Its gradients for 8192 tokens of 4096 features.
        {"name": "norm_backward", "op": "norm_backward", "dtype": "fp16", "rows": 8192, "cols": 4096},
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(["gated_forward", "gated_forward", "gated_backward", "gated_backward", "dropout_forward", "dropout_backward",
                     "norm_forward", "norm_backward"])
    case = {"op": op, "dtype": rng.choice(["fp16", "fp16", "fp32"])}
    if op in ("gated_forward", "gated_backward"):
        # a serving step (few rows), or a training step; the projections' sizes run from a toy model to the largest listed
        serving = op == "gated_forward" and rng.random() < 0.4
        case["rows"] = _log(rng, 1, 256) if serving else _log(rng, 64, 8192)
        step = rng.choice([1, 8, 64, 64])
        case["cols"] = max(step, _log(rng, 64, 4096) // step * step)
        case["width"] = max(step, min(16384, int(case["cols"] * rng.uniform(1.5, 4.0))) // step * step)
        case["act"] = rng.choice(["silu", "gelu", "gelu_tanh", "relu", "sigmoid"])
        case["p"] = rng.choice([0.0, 0.0, 0.1]) if not serving else 0.0
        if op == "gated_forward":
            case["keep_pre"] = not serving
    else:
        case["rows"] = _log(rng, 1, 8192)
        case["cols"] = _log(rng, 64, 4096)
        if rng.random() < 0.5:
            case["cols"] = max(64, case["cols"] // 64 * 64)
        if op.startswith("dropout"):
            case["p"] = rng.choice([0.05, 0.1, 0.25, 0.5])
        if op == "dropout_forward":
            case["residual"] = rng.random() < 0.5
    return case


def work(case):
    size = 2 if case["dtype"] == "fp16" else 4
    rows, cols = case["rows"], case["cols"]
    n = rows * cols
    op = case["op"]
    if op.startswith("gated"):
        width = case["width"]
        product = 2 * rows * cols * width
        weights, hidden = 2 * cols * width, rows * width
        if op == "gated_forward":
            return {"bytes": size * (n + weights + hidden * (3 if case["keep_pre"] else 1)), "flops": 2 * product}
        # read x, w, pre, dz; write dx, dw
        return {"bytes": size * (n + weights + 3 * hidden + n + weights), "flops": 4 * product}
    if op == "dropout_forward":
        return {"bytes": size * n * (3 if case["residual"] else 2), "flops": 2 * n}
    if op == "dropout_backward":
        return {"bytes": size * n * 2, "flops": n}
    if op == "norm_forward":
        return {"bytes": size * (2 * n + cols) + 4 * rows, "flops": 4 * n}
    return {"bytes": size * (3 * n + 2 * cols) + 4 * rows, "flops": 9 * n}


# ------------------------------------------------------------------------------------------------------------ inputs
def _normal(gen, shape, dtype, std=1.0):
    t = torch.randn(shape, generator=gen, device="cuda", dtype=torch.float32)
    return t.mul_(std).to(dtype)


def _inputs(case, seed):
    gen = torch.Generator(device="cuda")
    gen.manual_seed(seed)
    dtype = _DTYPES[case["dtype"]]
    rows, cols = case["rows"], case["cols"]
    s = dict(case)
    # the key and the call number of the generator: full 64-bit values
    s["seed"] = (seed * 0x9E3779B97F4A7C15 + 0x1234567) & 0xFFFFFFFFFFFFFFFF
    s["offset"] = (seed * 7919 + 3) & 0xFFFFFFFFFFFFFFFF
    op = case["op"]
    if op.startswith("gated"):
        width = case["width"]
        s["x"] = _normal(gen, (1, rows, cols), dtype)                            # normalised activations
        s["w"] = _normal(gen, (2, cols, width), dtype, 1.0 / math.sqrt(cols))
        if op == "gated_backward":
            s["pre"] = _normal(gen, (2, rows, width), dtype)                     # what the forward pass kept
            s["dz"] = _normal(gen, (1, rows, width), dtype, 0.01)
    elif op == "dropout_forward":
        s["x"] = _normal(gen, (rows, cols), dtype)
        s["residual_in"] = _normal(gen, (rows, cols), dtype, 2.0) if case["residual"] else None
    elif op == "dropout_backward":
        s["dy"] = _normal(gen, (rows, cols), dtype, 0.01)
    else:
        s["x"] = _normal(gen, (rows, cols), dtype, 3.0)                          # a residual stream, not yet normalised
        s["weight"] = (1.0 + 0.1 * torch.randn((cols,), generator=gen, device="cuda")).to(dtype)
        if op == "norm_backward":
            s["dy"] = _normal(gen, (rows, cols), dtype, 0.01)
            s["rstd"] = torch.rsqrt((s["x"].float() ** 2).mean(1) + _EPS)        # what the forward pass kept
    return s


def prepare(case, seed):
    s = _inputs(case, seed)
    if own:
        global _context
        import deep8_b200
        if _context is None:
            _context = deep8_b200.Context(torch.cuda.current_device())
        s["ctx"] = _context
        s["dropout"] = deep8_b200.Dropout(case["p"], s["seed"], s["offset"]) if case.get("p") else None
        # a training program keeps its gradient and workspace buffers from step to step
        if case["op"] == "gated_backward":
            s["dx"], s["dw"], s["dpre"] = torch.empty_like(s["x"]), torch.empty_like(s["w"]), torch.empty_like(s["pre"])
        elif case["op"] == "dropout_backward":
            s["dx"] = torch.empty_like(s["dy"])
        elif case["op"] == "norm_backward":
            s["dx"], s["dweight"] = torch.empty_like(s["x"]), torch.empty_like(s["weight"])
    return s


# ------------------------------------------------------------------------------------------------------------ a pass
def run(state):
    return _run_own(state) if own else _run_plain(state)


def _run_own(s):
    ctx, op = s["ctx"], s["op"]
    if op == "gated_forward":
        if not s["keep_pre"]:
            return ctx.gated_forward(s["x"], s["w"], s["act"])
        pre = torch.empty((2, s["rows"], s["width"]), dtype=s["x"].dtype, device=s["x"].device)
        return {"h": ctx.gated_forward(s["x"], s["w"], s["act"], pre=pre, dropout=s["dropout"]), "pre": pre}
    if op == "gated_backward":
        ctx.gated_backward(s["x"], s["w"], s["pre"], s["dz"], s["dx"], s["dw"], s["act"], dpre=s["dpre"], accumulate=False,
                           dropout=s["dropout"])
        return {"dx": s["dx"], "dw": s["dw"]}
    if op == "dropout_forward":
        return ctx.dropout_forward(s["x"], s["dropout"], residual=s["residual_in"])
    if op == "dropout_backward":
        return ctx.dropout_backward(s["dx"], s["dy"], s["dropout"], accumulate=False)
    if op == "norm_forward":
        rstd = torch.empty((s["rows"],), dtype=torch.float32, device=s["x"].device)
        return {"y": ctx.rms_norm_forward(s["x"], s["weight"], _EPS, rstd=rstd), "rstd": rstd}
    ctx.rms_norm_backward(s["x"], s["weight"], s["rstd"], s["dx"], s["dweight"], s["dy"], accumulate=False)
    return {"dx": s["dx"], "dweight": s["dweight"]}


def _philox(seed, offset, n, device):
    """The first n words of the generator's stream, as int64 values below 2^32."""
    g = torch.arange((n + 3) // 4, dtype=torch.int64, device=device)
    c0, c1 = g & _MASK, g >> 32
    c2, c3 = torch.full_like(g, offset & _MASK), torch.full_like(g, offset >> 32)
    k0, k1 = seed & _MASK, seed >> 32
    for _ in range(10):
        a, b = c0 * 0xD2511F53, c2 * 0xCD9E8D57  # 64-bit products; the sign bit is masked out of the high word
        c0, c1, c2, c3 = ((b >> 32) & _MASK) ^ c1 ^ k0, b & _MASK, ((a >> 32) & _MASK) ^ c3 ^ k1, a & _MASK
        k0, k1 = (k0 + 0x9E3779B9) & _MASK, (k1 + 0xBB67AE85) & _MASK
    return torch.stack((c0, c1, c2, c3), 1).reshape(-1)[:n]


def _keep(s, like):
    words = _philox(s["seed"], s["offset"], like.numel(), like.device)
    return (words >= int(round(s["p"] * 4294967296.0))).reshape(like.shape)


def _drop(s, t):
    return torch.where(_keep(s, t), t * (1.0 / (1.0 - s["p"])), torch.zeros_like(t)) if s["p"] else t


def _act(name, a):
    """act(a) and its derivative."""
    if name == "relu":
        on = (a > 0).to(a.dtype)
        return a * on, on
    if name in ("silu", "sigmoid"):
        sig = 1.0 / (1.0 + torch.exp(-a))
        if name == "sigmoid":
            return sig, sig * (1.0 - sig)
        return a * sig, sig * (1.0 + a * (1.0 - sig))
    if name == "gelu":
        cdf = 0.5 * torch.erfc(a * -math.sqrt(0.5))
        return a * cdf, cdf + a * torch.exp(-0.5 * a * a) / math.sqrt(2.0 * math.pi)
    c = math.sqrt(2.0 / math.pi)
    t = torch.tanh(c * (a + 0.044715 * a * a * a))
    return 0.5 * a * (1.0 + t), 0.5 * (1.0 + t) + 0.5 * a * (1.0 - t * t) * c * (1.0 + 3 * 0.044715 * a * a)


def _run_plain(s):
    op = s["op"]
    if op == "gated_forward":
        x, w = s["x"][0].float(), s["w"].float()
        gate, up = x @ w[0], x @ w[1]
        h = _drop(s, _act(s["act"], gate)[0] * up).to(s["x"].dtype)[None]
        return {"h": h, "pre": torch.stack((gate, up)).to(s["x"].dtype)} if s["keep_pre"] else h
    if op == "gated_backward":
        x, w = s["x"][0].float(), s["w"].float()
        gate, up = s["pre"][0].float(), s["pre"][1].float()
        d = _drop(s, s["dz"][0].float())
        value, slope = _act(s["act"], gate)
        dgate, dup = d * up * slope, d * value
        dx = dgate @ w[0].t() + dup @ w[1].t()
        dw = torch.stack((x.t() @ dgate, x.t() @ dup))
        return {"dx": dx.to(s["x"].dtype)[None], "dw": dw.to(s["w"].dtype)}
    if op == "dropout_forward":
        y = _drop(s, s["x"].float())
        if s["residual_in"] is not None:
            y = s["residual_in"].float() + y
        return y.to(s["x"].dtype)
    if op == "dropout_backward":
        return _drop(s, s["dy"].float()).to(s["dy"].dtype)
    x, weight = s["x"].float(), s["weight"].float()
    if op == "norm_forward":
        rstd = 1.0 / torch.sqrt((x * x).mean(1) + _EPS)
        return {"y": (x * rstd[:, None] * weight).to(s["x"].dtype), "rstd": rstd}
    dy, rstd = s["dy"].float(), s["rstd"][:, None]
    xhat = x * rstd
    u = dy * weight
    dx = rstd * (u - xhat * (u * xhat).mean(1, keepdim=True))
    return {"dx": dx.to(s["x"].dtype), "dweight": (dy * xhat).sum(0).to(s["weight"].dtype)}


# ------------------------------------------------------------------------------------------------------------ 64 bits
def _exact_keep(seed, offset, p, n):
    """The generator again, every 32 x 32-bit product built from 16-bit halves so that nothing passes 2^50."""
    def mul(v, m):
        lo, hi = (v & 0xFFFF) * m, (v >> 16) * m
        low = lo + ((hi & 0xFFFF) << 16)
        return (hi >> 16) + (low >> 32), low & _MASK

    index = torch.arange(n, dtype=torch.int64, device="cuda")
    group, lane = index[::4] // 4, index % 4
    words = [group & _MASK, group >> 32, group * 0 + (offset & _MASK), group * 0 + (offset >> 32)]
    for r in range(10):
        key0, key1 = ((seed & _MASK) + r * 0x9E3779B9) & _MASK, ((seed >> 32) + r * 0xBB67AE85) & _MASK
        hi0, lo0 = mul(words[0], 0xD2511F53)
        hi1, lo1 = mul(words[2], 0xCD9E8D57)
        words = [hi1 ^ words[1] ^ key0, lo1, hi0 ^ words[3] ^ key1, lo0]
    keep = torch.empty(n, dtype=torch.bool, device="cuda")
    for k in range(4):
        count = len(range(k, n, 4))
        keep[lane == k] = words[k][:count] >= round(p * 2 ** 32)
    return keep


def _exact_act(name, a):
    if name == "relu":
        return a.clamp(min=0), torch.heaviside(a, torch.zeros((), dtype=a.dtype, device=a.device))
    if name == "sigmoid":
        return torch.sigmoid(a), torch.sigmoid(a) * torch.sigmoid(-a)
    if name == "silu":
        return a * torch.sigmoid(a), torch.sigmoid(a) + a * torch.sigmoid(a) * torch.sigmoid(-a)
    if name == "gelu":
        normal = torch.special.ndtr(a)
        return a * normal, normal + a * torch.exp(-a * a / 2) / math.sqrt(2 * math.pi)
    z = math.sqrt(2 / math.pi) * (a + 0.044715 * a ** 3)
    slope = math.sqrt(2 / math.pi) * (1 + 0.134145 * a ** 2)
    sig = torch.sigmoid(2 * z)  # (1 + tanh z) / 2
    return a * sig, sig + 2 * a * sig * torch.sigmoid(-2 * z) * slope


def exact(case, seed):
    s = _inputs(case, seed)
    op = case["op"]

    def dropped(t):
        if not case.get("p"):
            return t
        keep = _exact_keep(s["seed"], s["offset"], case["p"], t.numel()).view(t.shape)
        return (t / (1 - case["p"])).masked_fill(~keep, 0.0)

    if op == "gated_forward":
        pre = torch.matmul(s["x"].double(), s["w"].double())
        h = dropped(_exact_act(case["act"], pre[0])[0] * pre[1]).unsqueeze(0)
        return {"h": h, "pre": pre} if case["keep_pre"] else h
    if op == "gated_backward":
        pre, d = s["pre"].double(), dropped(s["dz"][0].double())
        value, slope = _exact_act(case["act"], pre[0])
        dpre = torch.stack((d * pre[1] * slope, d * value))
        del pre, d, value, slope
        dx = torch.matmul(dpre, s["w"].double().transpose(1, 2)).sum(0, keepdim=True)
        return {"dx": dx, "dw": torch.matmul(s["x"].double().transpose(1, 2), dpre)}
    if op == "dropout_forward":
        y = dropped(s["x"].double())
        return y if s["residual_in"] is None else y + s["residual_in"].double()
    if op == "dropout_backward":
        return dropped(s["dy"].double())
    x, weight = s["x"].double(), s["weight"].double()
    if op == "norm_forward":
        rstd = (x.pow(2).sum(1) / x.shape[1] + _EPS).rsqrt()
        return {"y": x * weight * rstd.unsqueeze(1), "rstd": rstd}
    dy, rstd = s["dy"].double(), s["rstd"].double().unsqueeze(1)
    along = (dy * weight * x).sum(1, keepdim=True) * rstd.pow(3) / x.shape[1]
    return {"dx": rstd * dy * weight - x * along, "dweight": torch.einsum("rc,rc->c", dy, x * rstd)}
