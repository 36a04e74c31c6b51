"""Operators of the block's rows in 8 bits and in training: the linear layers as products of 8-bit blocks, the
gradients that use the 8-bit activations kept by the forward, LayerNorm and GELU forward and backward.

`run` computes a case with elementary torch operations, or, where `own` is set, with the framework's operators;
`exact` gives the same outputs in 64 bits from the definitions.

8-bit blocks: 128 consecutive values of a row (128 x 128 of a weight) share the smallest power of two 2^s with
max |v| <= 448 * 2^s; a value is kept as e4m3 of v / 2^s, ties to even.
"""
import math

import torch

own = False

BLOCK = 128
DTYPES = {"bf16": torch.bfloat16, "f16": torch.float16, "f32": torch.float32}
GELU_C, GELU_A = math.sqrt(2.0 / math.pi), 0.044715


# ---------------------------------------------------------------- cases
def listed():
    return [
        # LayerNorm in training.  One token per frame of a chunk: the rows of the modulation's own layers.
        dict(name="ln_rows_3", op="ln", B=1, L=3, C=1536, dtype="bf16", keep8=False),
        # odd row count and channels outside whole blocks, fp32 master activations
        dict(name="ln_odd_f32", op="ln", B=2, L=777, C=1000, dtype="f32", keep8=False),
        # one chunk of three latent frames at 480 x 832 in the 1.3B model, normalised rows kept in 8 bits
        dict(name="ln_chunk_keep8", op="ln", B=1, L=4680, C=1536, dtype="bf16", keep8=True),
        # a whole video of 21 frames: gradients of the modulated norm, scale and shift per frame
        dict(name="ln_mod_video", op="ln_mod", B=1, F=21, rows=1560, C=1536, dtype="bf16"),
        # serving, one token through the wide layer of the feed-forward (weights laid out once)
        dict(name="token_1536_8960", op="linear", M=1, K=1536, N=8960, dtype="bf16", epilogue="none"),
        # serving, ragged in every direction
        dict(name="ragged_f16", op="linear", M=1111, K=1000, N=777, dtype="f16", epilogue="none"),
        # serving, one chunk through the feed-forward's first layer of the 1.3B model
        dict(name="chunk_ffn_1p3b", op="linear", M=4680, K=1536, N=8960, dtype="bf16", epilogue="gelu_tanh"),
        # serving, the same chunk in the 14B model
        dict(name="chunk_ffn_14b", op="linear", M=4680, K=5120, N=13824, dtype="bf16", epilogue="none"),
        # a training step of a small ragged layer: product, gradients of rows, weight and bias
        dict(name="step_ragged_f16", op="step", M=333, K=520, N=264, dtype="f16"),
        # a training step of the feed-forward's first layer on one chunk
        dict(name="step_ffn_1p3b", op="step", M=4680, K=1536, N=8960, dtype="bf16"),
        # GELU in training with its input kept in 8 bits: a short ragged call, and the feed-forward's own
        dict(name="gelu_odd_f16", op="gelu", M=77, C=1000, dtype="f16"),
        dict(name="gelu_ffn_1p3b", op="gelu", M=4680, C=8960, dtype="bf16"),
    ]


def _log(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    op = rng.choice(["ln", "ln_mod", "linear", "linear", "step", "gelu"])
    half = rng.choice(["bf16", "bf16", "f16"])
    if op == "ln":
        return dict(op=op, B=rng.choice([1, 1, 2]), L=_log(rng, 1, 8000), C=8 * _log(rng, 8, 640), dtype=rng.choice(["bf16", "f16", "f32"]),
                    keep8=rng.random() < 0.5)
    if op == "ln_mod":
        return dict(op=op, B=rng.choice([1, 2]), F=rng.choice([1, 3, 7, 21]), rows=_log(rng, 1, 1560), C=8 * _log(rng, 8, 192), dtype=half)
    if op == "gelu":
        return dict(op=op, M=_log(rng, 1, 4680), C=_log(rng, 32, 8960), dtype=half)
    K, N = _log(rng, 64, 8960), _log(rng, 64, 8960)
    if rng.random() < 0.5:
        K, N = 64 * -(-K // 64), 64 * -(-N // 64)
    if op == "step":
        return dict(op=op, M=_log(rng, 1, 4680), K=K, N=min(N, 8960 * 1536 // K + 1), dtype=half)
    return dict(op=op, M=_log(rng, 1, 4680), K=K, N=N, dtype=half, epilogue=rng.choice(["none", "gelu_tanh"]))


# ---------------------------------------------------------------- inputs
def _rows(shape, g, dtype, spread=0.5):
    """Activation rows: channels of different strength, a few of them far above the rest, and a common offset."""
    strength = torch.exp(spread * torch.randn(shape[-1], generator=g, device=g.device))
    return (torch.randn(shape, generator=g, device=g.device) * strength + 0.1).to(dtype)


def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(int(seed))
    dt = DTYPES[case["dtype"]]
    op = case["op"]
    s = {"case": case}
    if op in ("ln", "ln_mod"):
        L = case["L"] if op == "ln" else case["F"] * case["rows"]
        s["x"] = _rows((case["B"], L, case["C"]), g, dt)
        s["dy"] = torch.randn(s["x"].shape, generator=g, device="cuda").to(dt)
        if op == "ln":
            s["weight"] = (1 + 0.1 * torch.randn(case["C"], generator=g, device="cuda")).to(dt).requires_grad_()
            s["bias"] = (0.1 * torch.randn(case["C"], generator=g, device="cuda")).to(dt).requires_grad_()
            s["x"].requires_grad_()
        else:
            s["scale"] = (0.3 * torch.randn((case["B"], case["F"], 1, case["C"]), generator=g, device="cuda")).to(dt)
        return s
    if op == "gelu":
        s["x"] = _rows((1, case["M"], case["C"]), g, dt).requires_grad_()
        s["dy"] = torch.randn(s["x"].shape, generator=g, device="cuda").to(dt)
        return s
    M, K, N = case["M"], case["K"], case["N"]
    s["x"] = _rows((1, M, K), g, dt)
    w = (torch.randn((N, K), generator=g, device="cuda") / math.sqrt(K)).to(dt)
    s["bias"] = (0.1 * torch.randn(N, generator=g, device="cuda")).to(dt)
    if op == "step":
        s["weight"] = w.requires_grad_()
        s["dy"] = torch.randn((1, M, N), generator=g, device="cuda").to(dt)
        s["x"].requires_grad_()
        s["bias"].requires_grad_()
    elif own:       # a serving program keeps the weights laid out in 8 bits ...
        from self_forcing_amd import linear8
        s["weight"] = linear8.pack(w)
    else:           # ... the plain form their values
        s["weight"] = _values(w.float(), True)
    return s


# ---------------------------------------------------------------- plain form, 32 bits
def _values(x, square=False):
    """The values that x [R, K] (fp32) has in 8-bit blocks; `square`: blocks of 128 x 128."""
    R, K = x.shape
    rb = BLOCK if square else 1
    p = torch.nn.functional.pad(x, (0, -K % BLOCK, 0, -R % rb))
    t = p.view(p.shape[0] // rb, rb, p.shape[1] // BLOCK, BLOCK)
    top = torch.where(torch.isfinite(t), t.abs(), torch.zeros_like(t)).amax((1, 3), keepdim=True)
    mant, ex = torch.frexp(top)                                 # top = mant 2^ex, 448 = 0.875 * 2^9
    s = torch.where(top == 0, torch.zeros_like(ex), torch.where(mant <= 0.875, ex - 9, ex - 8)).clamp_min(-126)
    up = ((s + 127) << 23).view(torch.float32)                  # 2^s
    down = ((127 - s) << 23).view(torch.float32)                # 2^-s
    q = (t * down).to(torch.float8_e4m3fn).float() * up
    return q.view(p.shape)[:R, :K]


def _gelu(x):
    return 0.5 * x * (1 + torch.tanh(GELU_C * (x + GELU_A * x * x * x)))


def _gelu_slope(x):
    t = torch.tanh(GELU_C * (x + GELU_A * x * x * x))
    return 0.5 * (1 + t) + 0.5 * x * (1 - t * t) * GELU_C * (1 + 3 * GELU_A * x * x)


def _plain_ln(s):
    case, dt = s["case"], s["x"].dtype
    x, dy, w, b = s["x"].detach().float(), s["dy"].float(), s["weight"].detach().float(), s["bias"].detach().float()
    c = x - x.mean(-1, keepdim=True)
    r = torch.rsqrt((c * c).mean(-1, keepdim=True) + 1e-6)
    xh = c * r
    y = xh * w + b
    if case["keep8"]:
        xh = _values(xh.flatten(0, 1)).view(x.shape)
    g = dy * w
    dx = r * (g - g.mean(-1, keepdim=True) - xh * (g * xh).mean(-1, keepdim=True))
    return [y.to(dt), dx.to(dt), (dy * xh).sum((0, 1)).to(dt), dy.sum((0, 1)).to(dt)]


def _plain_ln_mod(s):
    dt, e = s["x"].dtype, s["scale"].float()
    B, F, _, C = e.shape
    x, dy = s["x"].float().view(B, F, -1, C), s["dy"].float().view(B, F, -1, C)
    c = x - x.mean(-1, keepdim=True)
    r = torch.rsqrt((c * c).mean(-1, keepdim=True) + 1e-6)
    xh = c * r
    g = dy * (1 + e)
    dx = r * (g - g.mean(-1, keepdim=True) - xh * (g * xh).mean(-1, keepdim=True))
    return [dx.view(s["x"].shape).to(dt), (dy * xh).sum(2, keepdim=True).to(dt), dy.sum(2, keepdim=True).to(dt)]


def _plain_linear(s):
    y = _values(s["x"][0].float()) @ s["weight"].t() + s["bias"].float()
    if s["case"]["epilogue"] == "gelu_tanh":
        y = _gelu(y)
    return [y.to(s["x"].dtype)[None]]


def _plain_step(s):
    dt = s["x"].dtype
    x, w, dy = _values(s["x"].detach()[0].float()), _values(s["weight"].detach().float(), True), s["dy"][0].float()
    y = x @ w.t() + s["bias"].detach().float()
    return [y.to(dt)[None], (_values(dy) @ w).to(dt)[None], (dy.t() @ x).to(dt), dy.sum(0).to(dt)]


def _plain_gelu(s):
    x = s["x"].detach()[0].float()
    return [_gelu(x).to(s["x"].dtype)[None], (s["dy"][0].float() * _gelu_slope(_values(x))).to(s["x"].dtype)[None]]


# ---------------------------------------------------------------- the framework's operators
def _own(s):
    from self_forcing_amd import block_ops, linear8
    case, op = s["case"], s["case"]["op"]
    if op == "ln":
        y = block_ops.ln_affine(s["x"], s["weight"], s["bias"], 1e-6, checkpoint8=case["keep8"])
        return [y, *torch.autograd.grad(y, (s["x"], s["weight"], s["bias"]), s["dy"])]
    if op == "ln_mod":
        return list(block_ops.ln_modulate_backward(s["dy"], s["x"], s["scale"], 1e-6))
    if op == "linear":
        return [linear8.linear8(s["x"], s["weight"], s["bias"], epilogue=case["epilogue"])]
    if op == "step":
        y = linear8.linear8(s["x"], s["weight"], s["bias"])
        return [y, *torch.autograd.grad(y, (s["x"], s["weight"], s["bias"]), s["dy"])]
    y = block_ops.gelu_tanh(s["x"], checkpoint8=True)
    return [y, *torch.autograd.grad(y, (s["x"],), s["dy"])]


def run(state):
    if own:
        return _own(state)
    with torch.no_grad():
        return {"ln": _plain_ln, "ln_mod": _plain_ln_mod, "linear": _plain_linear, "step": _plain_step, "gelu": _plain_gelu}[state["case"]["op"]](state)


# ---------------------------------------------------------------- the definitions in 64 bits
def _binade(a):
    """floor(log2(a)) of positive normal float64 numbers, from their bits."""
    return (a.view(torch.int64) >> 52) - 1023


def _two_to(n):
    return ((n + 1023) << 52).view(torch.float64)


def _blocks64(v, square=False):
    """What the 8-bit blocks hold of v [R, K] (float64): the power of two by comparison, the mantissa's step by the value's own binade."""
    R, K = v.shape
    kb = torch.arange(K, device=v.device) // BLOCK
    rb = torch.arange(R, device=v.device) // (BLOCK if square else 1)
    top = torch.zeros(int(rb[-1]) + 1, int(kb[-1]) + 1, dtype=v.dtype, device=v.device)
    idx = (rb[:, None] * top.shape[1] + kb[None, :]).reshape(-1)
    top = top.view(-1).scatter_reduce(0, idx, v.abs().reshape(-1), "amax").view(top.shape)
    s = _binade(top.clamp_min(1e-300)) - 10
    for _ in range(3):
        s = torch.where(top > 448.0 * _two_to(s), s + 1, s)
    s = torch.where(top == 0, torch.zeros_like(s), s)
    unit = _two_to(s)[rb][:, kb]
    a = v.abs() / unit
    step = _two_to(_binade(a.clamp_min(2.0 ** -6)) - 3)
    return torch.sign(v) * torch.round(a / step) * step * unit


def _gelu64(x):
    return x * torch.sigmoid(2 * GELU_C * (x + GELU_A * x ** 3))


def _gelu64_slope(x):
    p = torch.sigmoid(2 * GELU_C * (x + GELU_A * x ** 3))
    return p + x * p * (1 - p) * 2 * GELU_C * (1 + 3 * GELU_A * x ** 2)


def exact(case, seed):
    global own
    was, own = own, False           # the weights as they are given, not a laid-out form of them
    try:
        s = prepare({**case, "op": "step"} if case["op"] == "linear" else case, seed)
    finally:
        own = was
    op = case["op"]
    d = {k: v.detach().double() for k, v in s.items() if isinstance(v, torch.Tensor)}
    if op in ("ln", "ln_mod"):
        x, dy = d["x"], d["dy"]
        var, mean = torch.var_mean(x, -1, correction=0, keepdim=True)
        r = (var + 1e-6) ** -0.5
        xh = (x - mean) * r
        if op == "ln":
            w = d["weight"]
            y = torch.addcmul(d["bias"], xh, w)
            if case["keep8"]:
                xh = _blocks64(xh.reshape(-1, x.shape[-1])).reshape(x.shape)
        else:
            w = (1 + d["scale"]).expand(-1, -1, case["rows"], -1).reshape(x.shape)
        g, C = dy * w, x.shape[-1]
        dx = r / C * (C * g - g.sum(-1, keepdim=True) - xh * torch.linalg.vecdot(g, xh).unsqueeze(-1))
        if op == "ln":
            flat = dy.reshape(-1, C)
            return [y, dx, (flat * xh.reshape(-1, C)).sum(0), flat.sum(0)]
        frames = (case["B"], case["F"], case["rows"], C)
        return [dx, (dy * xh).view(frames).sum(2, keepdim=True), dy.view(frames).sum(2, keepdim=True)]
    if op == "gelu":
        x = d["x"][0]
        return [_gelu64(x)[None], (d["dy"][0] * _gelu64_slope(_blocks64(x)))[None]]
    x, w = _blocks64(d["x"][0]), _blocks64(d["weight"], True)
    y = torch.addmm(d["bias"], x, w.t())
    if op == "linear":
        return [(_gelu64(y) if case["epilogue"] == "gelu_tanh" else y)[None]]
    dy = d["dy"][0]
    return [y[None], torch.mm(_blocks64(dy), w)[None], torch.mm(dy.t(), x), dy.sum(0)]


# ---------------------------------------------------------------- what a pass cannot do without
def work(case):
    e = 4 if case["dtype"] == "f32" else 2
    op = case["op"]
    if op == "ln":          # x and dy in, y and dx out
        n = case["B"] * case["L"] * case["C"]
        return {"bytes": 4 * e * n + 4 * e * case["C"], "flops": 20 * n}
    if op == "ln_mod":      # x and dy in, dx out, the modulation rows
        n = case["B"] * case["F"] * case["rows"] * case["C"]
        return {"bytes": 3 * e * n + 3 * e * case["B"] * case["F"] * case["C"], "flops": 16 * n}
    if op == "gelu":
        n = case["M"] * case["C"]
        return {"bytes": 4 * e * n, "flops": 40 * n}
    M, K, N = case["M"], case["K"], case["N"]
    if op == "linear":      # weights are a byte a value and a scale per block
        return {"bytes": e * M * K + N * K + -(-N // BLOCK) * -(-K // BLOCK) + e * N + e * M * N, "flops": 2 * M * N * K}
    return {"bytes": 2 * e * (M * K + N * K + M * N + N), "flops": 6 * M * N * K}
