"""What is measured of the 8-bit integer path: rows quantised with a scale each (alone, or as the end of the residual
addition and RMSNorm in front of a projection), the product of such rows with 8-bit weights that have a scale per output
channel, and that product with the SwiGLU epilogue of the MLP.

With `own` false, run() computes the operators from elementary torch operations; with `own` true it calls the library.
Sizes are those of the 1.7B talker (hidden 2048, intermediate 6144, q/k/v 4096 columns) from one decode row to the
largest packed prompt batch (max_num_batched_tokens = 16384), and ragged ones.
"""
import math

import torch

own = False

TINY = 2.0 ** -126      # the smallest scale: rows of zeros (and of denormal numbers) keep a finite reciprocal
EPS = 1e-6

# The most a drawn case may cost, in the units of _cost(): what the largest listed ones do.
MOST_PRODUCT = 16384 * 2048 * 6144
MOST_ROWS = 8192 * 6144


def listed():
    return [
        # the q/k/v projection of one stream's decode step
        dict(name="linear 1 row", op="linear", M=1, N=4096, K=2048, bias=False, residual=False),
        # down_proj of a decode step of 16 streams, into the residual stream
        dict(name="linear 16 rows", op="linear", M=16, N=2048, K=6144, bias=False, residual=True),
        # the q/k/v projection of a 200-token prompt
        dict(name="linear 200 rows", op="linear", M=200, N=4096, K=2048, bias=False, residual=False),
        # nothing a multiple of a tile: an adapter or a pruned layer over a few packed prompts
        dict(name="linear ragged", op="linear", M=777, N=1000, K=1111, bias=True, residual=True),
        # down_proj of the largest packed prompt batch
        dict(name="linear 16384 rows", op="linear", M=16384, N=2048, K=6144, bias=False, residual=True),
        # gate/up of the MLP: a decode step of 8 streams, a 200-token prompt, a large packed prompt batch
        dict(name="swiglu 8 rows", op="swiglu", M=8, I=6144, K=2048),
        dict(name="swiglu 200 rows", op="swiglu", M=200, I=6144, K=2048),
        dict(name="swiglu 8192 rows", op="swiglu", M=8192, I=6144, K=2048),
        # the residual addition and norm in front of a projection: a decode step of 8 streams, the largest batch
        dict(name="rmsnorm 8 rows", op="rmsnorm", M=8, H=2048, delta=True),
        dict(name="rmsnorm 16384 rows", op="rmsnorm", M=16384, H=2048, delta=True),
        # the SwiGLU output on its way into down_proj: ragged, and a large packed prompt batch
        dict(name="quantize ragged", op="quantize", M=333, K=1111),
        dict(name="quantize 8192 rows", op="quantize", M=8192, K=6144),
    ]


def _size(rng, low, high):
    """Log-uniform in [low, high]; every other one a multiple of 64 as model sizes are, the rest as they fall."""
    v = int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))
    return max(64, v // 64 * 64) if low >= 64 and rng.random() < 0.5 else v


def draw(rng):
    op = rng.choice(["linear", "linear", "swiglu", "rmsnorm", "quantize"])
    while True:
        M = _size(rng, 1, 16384)
        if op == "linear":
            c = dict(op=op, M=M, N=_size(rng, 64, 8192), K=_size(rng, 64, 8192), bias=rng.random() < 0.5,
                     residual=rng.random() < 0.5)
            if M * c["N"] * c["K"] <= MOST_PRODUCT:
                return c
        elif op == "swiglu":
            c = dict(op=op, M=M, I=_size(rng, 64, 8192), K=_size(rng, 64, 8192))
            if 2 * M * c["I"] * c["K"] <= MOST_PRODUCT:
                return c
        elif op == "rmsnorm":
            c = dict(op=op, M=M, H=_size(rng, 64, 8192), delta=rng.random() < 0.75)
            if M * c["H"] <= 16384 * 2048:
                return c
        else:
            c = dict(op=op, M=M, K=_size(rng, 64, 8192))
            if M * c["K"] <= MOST_ROWS:
                return c


# ---------------------------------------------------------------- inputs
def _gen(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def _activations(g, M, K, spread=1.0):
    """bf16 rows as a decoder's hidden states are: rows of different size, and a few channels far larger than the rest."""
    x = torch.randn(M, K, generator=g, device="cuda")
    x *= torch.exp(spread * 0.5 * torch.randn(M, 1, generator=g, device="cuda"))
    x *= torch.where(torch.rand(K, generator=g, device="cuda") < 0.004, 12.0, 1.0)
    return x.to(torch.bfloat16)


def _int8(x):
    """A checkpoint's or a previous operator's 8-bit rows: values and a scale per row."""
    s = (x.abs().amax(-1) / 127).clamp_min(TINY)
    return (x / s[:, None]).round_().clamp_(-127, 127).to(torch.int8), s


def _rows(q):
    """The rows as the library's own operators leave them: a row takes a multiple of 16 bytes."""
    M, K = q.shape
    buf = torch.zeros(M, (K + 15) // 16 * 16, dtype=torch.int8, device=q.device)
    buf[:, :K] = q
    return buf[:, :K]


def prepare(case, seed):
    g, op, M = _gen(seed), case["op"], case["M"]
    s = {"op": op}
    if op in ("linear", "swiglu"):
        K = case["K"]
        q, s["xs"] = _int8(_activations(g, M, K).float())
        s["x"] = _rows(q)
        if op == "linear":
            N = case["N"]
            s["w"], s["ws"] = _int8(torch.randn(N, K, generator=g, device="cuda") * 0.03)
            s["bias"] = torch.randn(N, generator=g, device="cuda").to(torch.bfloat16) if case["bias"] else None
            s["residual"] = _activations(g, M, N) if case["residual"] else None
            if own:
                from nano_qwen3tts_vllm import hip
                s["packed"] = hip.pack_weight_int8(s["w"])
        else:
            I = case["I"]
            s["gate"], s["gs"] = _int8(torch.randn(I, K, generator=g, device="cuda") * 0.03)
            s["up"], s["us"] = _int8(torch.randn(I, K, generator=g, device="cuda") * 0.03)
            if own:
                from nano_qwen3tts_vllm import hip
                s["packed"] = hip.pack_gate_up_int8(s["gate"], s["up"])
    elif op == "rmsnorm":
        H = case["H"]
        s["x"] = _activations(g, M, H)
        s["delta"] = (0.3 * torch.randn(M, H, generator=g, device="cuda")).to(torch.bfloat16) if case["delta"] else None
        s["w"] = (1 + 0.1 * torch.randn(H, generator=g, device="cuda")).to(torch.bfloat16)
    else:
        s["x"] = _activations(g, M, case["K"])
    return s


# ---------------------------------------------------------------- one pass
def _values(q, scales):
    """The numbers that 8-bit rows stand for."""
    out = torch.empty(q.shape, dtype=torch.bfloat16, device=q.device)
    return torch.mul(q, scales[:, None], out=out)


def _plain_quantize(y):
    s = (y.abs().amax(-1) / 127).clamp_min(TINY)
    return (y / s[:, None]).round().clamp(-127, 127).to(torch.int8), s


def _plain_product(x, xs, w, ws):
    return (x.float() @ w.float().t()) * xs[:, None] * ws


def run(s):
    op = s["op"]
    if own:
        from nano_qwen3tts_vllm import hip
    if op == "linear":
        if own:
            return hip.linear_int8(s["x"], s["xs"], s["packed"], s["ws"], s["ws"].shape[0], bias=s["bias"],
                                   residual=s["residual"])
        y = _plain_product(s["x"], s["xs"], s["w"], s["ws"])
        if s["bias"] is not None:
            y = y + s["bias"].float()
        if s["residual"] is not None:
            y = y + s["residual"].float()
        return y.to(torch.bfloat16)
    if op == "swiglu":
        if own:
            return hip.linear_swiglu_int8(s["x"], s["xs"], s["packed"], s["gs"], s["us"], s["gs"].shape[0])
        g = _plain_product(s["x"], s["xs"], s["gate"], s["gs"])
        u = _plain_product(s["x"], s["xs"], s["up"], s["us"])
        return (g / (1 + torch.exp(-g)) * u).to(torch.bfloat16)
    if op == "rmsnorm":
        if own:
            r = hip.rmsnorm_int8(s["x"], s["w"], EPS, delta=s["delta"])
            return {"values": _values(r[0], r[1]), "scales": r[1], "sum": r[2] if s["delta"] is not None else None}
        h = s["x"]
        if s["delta"] is not None:
            h = (h.float() + s["delta"].float()).to(torch.bfloat16)
        f = h.float()
        y = f / torch.sqrt((f * f).mean(-1, keepdim=True) + EPS) * s["w"].float()
        q, scales = _plain_quantize(y)
        return {"values": _values(q, scales), "scales": scales, "sum": h if s["delta"] is not None else None}
    q, scales = hip.quantize_int8(s["x"]) if own else _plain_quantize(s["x"].float())
    return {"values": _values(q, scales), "scales": scales}


# ---------------------------------------------------------------- what a pass cannot do without
def work(case):
    M = case["M"]
    if case["op"] == "linear":
        N, K = case["N"], case["K"]
        b = M * K + N * K + 4 * M + 4 * N + 2 * M * N + 2 * N * case["bias"] + 2 * M * N * case["residual"]
        return {"bytes": b, "flops": 2 * M * N * K}
    if case["op"] == "swiglu":
        I, K = case["I"], case["K"]
        return {"bytes": M * K + 2 * I * K + 4 * M + 8 * I + 2 * M * I, "flops": 4 * M * I * K + 5 * M * I}
    if case["op"] == "rmsnorm":
        H = case["H"]
        return {"bytes": M * H * (2 + 1) + 2 * H + 4 * M + 4 * M * H * case["delta"], "flops": 8 * M * H}
    return {"bytes": 3 * M * case["K"] + 4 * M, "flops": 4 * M * case["K"]}


# ---------------------------------------------------------------- in 64 bits
def _exact_rows(y):
    scale = torch.clamp(y.abs().max(dim=1).values / 127.0, min=TINY)
    steps = torch.clamp(torch.round(y / scale.unsqueeze(1)), -127.0, 127.0)
    return steps * scale.unsqueeze(1), scale


def _exact_product(x, xs, w, ws):
    acc = torch.empty(x.shape[0], w.shape[0], dtype=torch.float64, device=x.device)
    wt = w.double().t().contiguous()
    for a in range(0, x.shape[0], 4096):
        acc[a:a + 4096] = torch.mm(x[a:a + 4096].double(), wt)
    return acc.mul_(xs.double().unsqueeze(1)).mul_(ws.double().unsqueeze(0))


def exact(case, seed):
    s = prepare(case, seed)
    if case["op"] == "linear":
        y = _exact_product(s["x"], s["xs"], s["w"], s["ws"])
        for more in ("bias", "residual"):
            if s[more] is not None:
                y = y + s[more].double()
        return y
    if case["op"] == "swiglu":
        g = _exact_product(s["x"], s["xs"], s["gate"], s["gs"])
        return g * torch.sigmoid(g) * _exact_product(s["x"], s["xs"], s["up"], s["us"])
    if case["op"] == "rmsnorm":
        h, total = s["x"].double(), None
        if s["delta"] is not None:
            total = h + s["delta"].double()
            h = total.to(torch.bfloat16).double()     # the norm reads the residual stream as it is kept
        rms = torch.linalg.vector_norm(h, dim=1, keepdim=True).square() / h.shape[1]
        values, scales = _exact_rows(h * torch.rsqrt(rms + EPS) * s["w"].double())
        return {"values": values, "scales": scales, "sum": total}
    values, scales = _exact_rows(s["x"].double())
    return {"values": values, "scales": scales}
