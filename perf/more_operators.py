"""What a token's step needs beside the key/value cache, as cases that can be
timed and compared: the norm that adds the residual, rows in 8 bits, the product
of 8-bit rows with 8-bit weights, rotary positions, and the draw of a token.

8 bits are e4m3 codes with one power-of-two scale a row: the smallest, 2^-100 or
more, that takes the row's largest magnitude into +-448.
"""
import math
import random

import torch

own = False

MOST_BYTES = 270e6  # what a drawn case reads and writes at most
MOST_FLOPS = 2.7e11
MOST_LOGITS = 2e7  # a drawn case's logits, which the plain form sorts

TYPES = {"f16": torch.float16, "bf16": torch.bfloat16, "f32": torch.float32}
SIZE = {"f16": 2, "bf16": 2, "f32": 4, "e4m3": 1}
EPS = 1e-6


def listed():
    return [
        # 16 streams' newest tokens before a layer's first product: launches and latency.
        dict(name="norm a token each", kind="norm", rows=16, width=1024, type="bf16",
             residual="f32", out="e4m3"),
        # The same for the prompts that a server takes in at once.
        dict(name="norm prompts", kind="norm", rows=16384, width=1024, type="bf16",
             residual="bf16", out="e4m3"),
        # A chunk's feed-forward activations, gated on their way into 8 bits.
        dict(name="quantize gated", kind="quantize", rows=580, width=4096, type="f16", gated=True),
        # A checkpoint's float32 matrix turned into 8-bit weights.
        dict(name="quantize weights", kind="quantize", rows=6144, width=1024, type="f32",
             gated=False),
        # q|k|v of 16 streams' newest tokens: the weights are read, little is computed.
        dict(name="linear a token each", kind="linear", rows=16, width=1024, out=4096,
             type="bf16"),
        # The output projection of a 10 s utterance under guidance (580 rows).
        dict(name="linear chunk", kind="linear", rows=580, width=2048, out=1024, type="f32"),
        # Prompts through a wide layer: the matrix cores.
        dict(name="linear prompts", kind="linear", rows=4096, width=4096, out=8192, type="bf16"),
        # Queries and keys of 48 streams far into their texts, normed as they are rotated.
        dict(name="rotate a token each", kind="rotary", rows=48, heads=16, kv_heads=8, dim=128,
             rotary=128, interleaved=False, normed=True, far=90000, type="f16"),
        # Prompts, neighbouring dims as pairs, half of every head.
        dict(name="rotate prompts", kind="rotary", rows=12000, heads=16, kv_heads=8, dim=128,
             rotary=64, interleaved=True, normed=False, far=12000, type="bf16"),
        # Codes of a 10 s utterance under guidance (250 frames of 8 codebooks), the best 50.
        dict(name="sample codes", kind="sample", rows=2000, vocab=1025, guided=True, filters="k",
             type="f32"),
        # 64 streams' next text tokens, each with settings of its own.
        dict(name="sample streams", kind="sample", rows=64, vocab=151936, guided=False,
             filters="each", type="bf16"),
        # A text scored by drawing at every place, nothing cut off.
        dict(name="sample text", kind="sample", rows=300, vocab=151936, guided=False,
             filters="none", type="bf16"),
    ]


def _log(rng, low, high):
    return int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))


def draw(rng):
    kind = rng.choice(["norm", "quantize", "linear", "linear", "rotary", "sample", "sample"])
    while True:
        dtype = rng.choice(["f16", "bf16", "f32"])
        if kind == "norm":
            case = dict(kind=kind, rows=_log(rng, 1, 30000), type=dtype,
                        width=rng.choice([8 * _log(rng, 8, 1024), _log(rng, 64, 9000)]),
                        residual=rng.choice(["", dtype, "f32"]),
                        out=rng.choice(["e4m3", "e4m3", "f16" if dtype == "f32" else dtype]))
        elif kind == "quantize":
            case = dict(kind=kind, rows=_log(rng, 1, 30000), type=dtype,
                        width=rng.choice([16 * _log(rng, 4, 800), _log(rng, 64, 13000)]),
                        gated=rng.random() < 0.5)
        elif kind == "linear":
            case = dict(kind=kind, type=dtype,
                        rows=rng.choice([_log(rng, 1, 64), _log(rng, 64, 8192)]),
                        width=16 * _log(rng, 4, 640),
                        out=rng.choice([64 * _log(rng, 1, 160), _log(rng, 16, 12000)]))
        elif kind == "rotary":
            dim = rng.choice([64, 80, 96, 128, 128, 256])
            kv_heads = rng.choice([1, 2, 4, 8])
            case = dict(kind=kind, rows=_log(rng, 1, 30000), heads=kv_heads * rng.choice([1, 2, 4]),
                        kv_heads=kv_heads, dim=dim,
                        rotary=rng.choice([dim, dim, dim // 2, 2 * rng.randint(1, dim // 2)]),
                        interleaved=rng.random() < 0.5, normed=rng.random() < 0.4,
                        far=_log(rng, 100, 1000000), type=dtype)
        else:
            case = dict(kind=kind, rows=_log(rng, 1, 4000), vocab=_log(rng, 60, 200000),
                        guided=rng.random() < 0.3, type=dtype,
                        filters=rng.choice(["none", "k", "p", "each", "each"]))
            if case["rows"] * case["vocab"] > MOST_LOGITS:
                continue
        w = work(case)
        if w["bytes"] <= MOST_BYTES and w["flops"] <= MOST_FLOPS:
            return case


def work(case):
    kind, rows, size = case["kind"], float(case["rows"]), SIZE[case["type"]]
    if kind == "norm":
        values = rows * case["width"]
        held = 2 * SIZE[case["residual"]] if case["residual"] else 0  # read, and the sum
        return dict(bytes=values * (size + held + SIZE[case["out"]]) + 4.0 * case["width"] +
                    (4.0 * rows if case["out"] == "e4m3" else 0.0), flops=5.0 * values)
    if kind == "quantize":
        values = rows * case["width"]
        return dict(bytes=values * (size * (2 if case["gated"] else 1) + 1) + 4.0 * rows,
                    flops=3.0 * values)
    if kind == "linear":
        n, k = float(case["out"]), float(case["width"])
        return dict(bytes=rows * k + n * k + rows * n * size + 4.0 * (rows + n),
                    flops=2.0 * rows * n * k)
    if kind == "rotary":
        values = rows * (case["heads"] + case["kv_heads"]) * case["dim"]
        return dict(bytes=2.0 * values * size + 4.0 * rows, flops=3.0 * values)
    values = rows * case["vocab"]
    return dict(bytes=values * size * (2 if case["guided"] else 1) + 8.0 * rows,
                flops=10.0 * values)


# ------------------------------------------------------------------ what a program holds

def _scale(amax):
    """The smallest power of two, 2^-100 or more, that takes amax into +-448."""
    m, e = torch.frexp(amax)
    e = torch.where(m > 0, e - 9 + (m > 0.875).to(e.dtype), -100)
    return ((e.clamp(min=-100) + 127) << 23).view(torch.float32)


def _codes(y):
    """e4m3 codes and scales of rows of float32 or float64 numbers."""
    scales = _scale(y.abs().amax(-1))
    return (y / scales[:, None]).float().to(torch.float8_e4m3fn), scales


def prepare(case, seed):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    dtype, kind, rows = TYPES[case["type"]], case["kind"], case["rows"]

    def normal(*shape):
        return torch.randn(*shape, generator=gen, device="cuda")

    def uniform(*shape):
        return torch.rand(*shape, generator=gen, device="cuda")

    def codes(count, width):
        # Rows of different loudness, as tokens and output channels have.
        q, s = _codes(normal(count, width) * torch.exp(0.5 * normal(count, 1)))
        return q, s

    state = dict(case=case)
    if kind == "norm":
        width = case["width"]
        # A few loud channels, as a trained model's stream has.
        loud = 1.0 + 20.0 * (uniform(width) > 0.99)
        state.update(x=(normal(rows, width) * 0.5).to(dtype), weight=1.0 + 0.3 * normal(width),
                     residual=None, total=None, scales=None)
        if case["residual"]:
            held = (normal(rows, width) * loud).to(TYPES[case["residual"]])
            state.update(residual=held, total=torch.zeros_like(held))
        if case["out"] == "e4m3":
            state.update(out=torch.zeros(rows, width, dtype=torch.float8_e4m3fn, device="cuda"),
                         scales=torch.zeros(rows, device="cuda"))
        else:
            state.update(out=torch.zeros(rows, width, dtype=TYPES[case["out"]], device="cuda"))
    elif kind == "quantize":
        width = case["width"]
        level = torch.exp(0.5 * normal(rows, 1))
        state.update(x=(normal(rows, width) * level).to(dtype), gate=None,
                     codes=torch.zeros(rows, width, dtype=torch.float8_e4m3fn, device="cuda"),
                     scales=torch.zeros(rows, device="cuda"))
        if case["gated"]:
            state.update(gate=(normal(rows, width) * 2.0).to(dtype))
    elif kind == "linear":
        x, x_scales = codes(rows, case["width"])
        w, w_scales = codes(case["out"], case["width"])
        # Weights as a checkpoint's: columns of unit length or so.
        w_scales = w_scales * 2.0 ** round(-0.5 * math.log2(case["width"]))
        state.update(x=x, x_scales=x_scales, w=w, w_scales=w_scales,
                     y=torch.zeros(rows, case["out"], dtype=dtype, device="cuda"))
    elif kind == "rotary":
        dim, heads, kv_heads = case["dim"], case["heads"], case["kv_heads"]
        half = case["rotary"] // 2
        f = 1e6 ** -(torch.arange(half, dtype=torch.float64, device="cuda") / half)
        # q|k|v rows as a product leaves them, rotated into tensors of their own.
        fused = normal(rows, heads + 2 * kv_heads, dim).to(dtype)
        state.update(q=fused[:, :heads], k=fused[:, heads:heads + kv_heads],
                     q_out=torch.zeros(rows, heads, dim, dtype=dtype, device="cuda"),
                     k_out=torch.zeros(rows, kv_heads, dim, dtype=dtype, device="cuda"),
                     frequencies=f.float(), q_norm=None, k_norm=None,
                     positions=torch.randint(0, case["far"] + 1, (rows,), generator=gen,
                                             device="cuda", dtype=torch.int32))
        if case["normed"]:
            state.update(q_norm=1.0 + 0.3 * normal(dim), k_norm=1.0 + 0.3 * normal(dim))
    else:
        vocab = case["vocab"]
        # Peaked as a trained model's are: a few entries stand out of each row.
        logits = normal(rows, vocab).mul_(2.0)
        best = torch.randint(0, vocab, (rows, 6), generator=gen, device="cuda")
        logits.scatter_add_(1, best, normal(rows, 6).mul_(2.0).add_(8.0))
        state.update(logits=logits.to(dtype), uncond=None, mask=None, random=uniform(rows),
                     tokens=torch.zeros(rows, dtype=torch.int32, device="cuda"),
                     temperature=0.9, top_k=0, top_p=1.0, min_p=0.0)
        if case["guided"]:
            state.update(uncond=(logits + normal(rows, vocab)).to(dtype), mask=vocab - 1)
        if case["filters"] == "k":
            state.update(top_k=50)
        elif case["filters"] == "p":
            state.update(top_p=0.9)
        elif case["filters"] == "each":
            pick = torch.randint(0, 4, (4, rows), generator=gen, device="cuda")

            def choice(k, values, dtype=torch.float32):
                return torch.tensor(values, dtype=dtype, device="cuda")[pick[k]].contiguous()

            state.update(temperature=choice(0, [0.0, 0.7, 1.0, 1.3]),
                         top_k=choice(1, [0, 20, 100, 1000], torch.int32),
                         top_p=choice(2, [1.0, 0.95, 0.9, 0.6]),
                         min_p=choice(3, [0.0, 0.0, 0.02, 0.1]))
    return state


# ------------------------------------------------------------------ a pass

def run(state):
    if own:
        return _run_own(state)
    return PLAIN[state["case"]["kind"]](state)


def _run_own(state):
    import omnivoice_amd as ov
    case = state["case"]
    kind = case["kind"]
    if kind == "norm":
        ov.op_add_rmsnorm(state["x"], state["weight"], state["out"], EPS,
                          residual=state["residual"], total=state["total"],
                          scales=state["scales"])
        return [state[n] for n in ("total", "out", "scales")]
    if kind == "quantize":
        ov.op_quantize8(state["x"], state["codes"], state["scales"], gate=state["gate"])
        return [state["codes"], state["scales"]]
    if kind == "linear":
        ov.op_linear8(state["x"], state["x_scales"], state["w"], state["w_scales"], state["y"])
        return state["y"]
    if kind == "rotary":
        ov.op_rotary(state["q"], state["q_out"], state["k"], state["k_out"],
                     state["frequencies"], positions=state["positions"],
                     interleaved=case["interleaved"], q_norm=state["q_norm"],
                     k_norm=state["k_norm"], eps=EPS)
        return [state["q_out"], state["k_out"]]
    ov.op_sample(state["logits"], state["random"], state["tokens"],
                 temperature=state["temperature"], top_k=state["top_k"], top_p=state["top_p"],
                 min_p=state["min_p"], uncond=state["uncond"],
                 guidance=2.0 if case["guided"] else 0.0, mask_id=state["mask"])
    return state["tokens"]


def _norm(x, weight):
    return weight * x * torch.rsqrt(x.square().mean(-1, keepdim=True) + EPS)


def _plain_norm(state):
    s, total = state["x"].float(), None
    if state["residual"] is not None:
        total = (s + state["residual"].float()).to(state["residual"].dtype)
        s = total.float()
    y = _norm(s, state["weight"])
    if state["scales"] is None:
        return [total, y.to(state["out"].dtype), None]
    return [total, *_codes(y)]


def _plain_quantize(state):
    y = state["x"].float()
    if state["gate"] is not None:
        g = state["gate"].float()
        y = y * (g / (1.0 + torch.exp(-g)))
    return list(_codes(y))


def _plain_linear(state):
    y = state["x"].float() @ state["w"].float().t()
    return (y * state["x_scales"][:, None] * state["w_scales"]).to(state["y"].dtype)


def _plain_rotary(state):
    case = state["case"]
    # Far positions lose their angle in 32 bits.
    angle = state["positions"].double()[:, None] * state["frequencies"].double()
    cos, sin = torch.cos(angle).float()[:, None], torch.sin(angle).float()[:, None]
    outs = []
    for x, weight in ((state["q"], state["q_norm"]), (state["k"], state["k_norm"])):
        y = x.float()
        if weight is not None:
            y = _norm(y, weight)
        turned, rest = y[..., :case["rotary"]], y[..., case["rotary"]:]
        if case["interleaved"]:
            a, b = turned[..., 0::2], turned[..., 1::2]
            turned = torch.stack([a * cos - b * sin, b * cos + a * sin], -1).flatten(-2)
        else:
            a, b = turned.chunk(2, -1)
            turned = torch.cat([a * cos - b * sin, b * cos + a * sin], -1)
        outs.append(torch.cat([turned, rest], -1).to(x.dtype))
    return outs


def _per_row(value, rows, dtype):
    if isinstance(value, torch.Tensor):
        return value[:, None].to(dtype)
    return torch.full((rows, 1), value, dtype=torch.float32, device="cuda").to(dtype)


def _plain_sample(state):
    z = state["logits"].float()
    rows, vocab = z.shape
    if state["uncond"] is not None:
        z = z + 2.0 * (z - state["uncond"].float())
    if state["mask"] is not None:
        z[:, state["mask"]] = -math.inf
    t = _per_row(state["temperature"], rows, torch.float64)
    k = _per_row(state["top_k"], rows, torch.int64)
    p = _per_row(state["top_p"], rows, torch.float64)
    m = _per_row(state["min_p"], rows, torch.float64)
    z, ids = torch.sort(z, dim=-1, descending=True, stable=True)
    # The sums decide where a draw falls, and at which token a share is reached: 64 bits.
    w = torch.exp((z.double() - z[:, :1].double()) / torch.where(t > 0, t, 1.0))
    rank = torch.arange(vocab, device="cuda")
    w = torch.where((k <= 0) | (rank < k), w, 0.0)
    cum = w.cumsum(-1)
    before = torch.nn.functional.pad(cum[:, :-1], (1, 0))
    w = torch.where((rank == 0) | (((p >= 1) | (before < p * cum[:, -1:])) & (w >= m)), w, 0.0)
    w = torch.where((t > 0) | (rank == 0), w, 0.0)
    cum = torch.zeros_like(w).scatter_(1, ids, w).cumsum(-1)
    target = state["random"].double()[:, None] * cum[:, -1:]
    return (cum <= target).sum(-1).to(torch.int32)


PLAIN = dict(norm=_plain_norm, quantize=_plain_quantize, linear=_plain_linear,
             rotary=_plain_rotary, sample=_plain_sample)


# ------------------------------------------------------------------ in 64 bits

def _round_e4m3(x):
    """x to the nearest multiple of its binade's step, ties to even."""
    e = torch.floor(torch.log2(x.abs().clamp(min=1e-300))).clamp(min=-6)
    step = torch.exp2(e - 3)
    return (torch.round(x / step) * step).clamp(-448, 448)


def _exact_codes(y):
    amax = y.abs().amax(-1)
    s = torch.exp2(torch.ceil(torch.log2(amax / 448)).clamp(min=-100))
    return _round_e4m3(y / s[:, None]), s


def exact(case, seed):
    """From the definitions, in 64 bits; none for the drawn tokens, which are whole numbers."""
    if case["kind"] == "sample":
        return None
    state = prepare(case, seed)
    x = state["q"].double() if case["kind"] == "rotary" else state["x"].double()
    if case["kind"] == "norm":
        total = None
        if state["residual"] is not None:
            total = x + state["residual"].double()
            # What is normed is what the sum's type holds.
            x = total.to(state["residual"].dtype).double()
        y = x / torch.sqrt((x * x).sum(-1, keepdim=True) / case["width"] + EPS)
        y = y * state["weight"].double()
        return [total, *_exact_codes(y)] if case["out"] == "e4m3" else [total, y, None]
    if case["kind"] == "quantize":
        if case["gated"]:
            x = x * state["gate"].double() * torch.sigmoid(state["gate"].double())
        return list(_exact_codes(x))
    if case["kind"] == "linear":
        x = x * state["x_scales"].double()[:, None]
        return x @ (state["w"].double() * state["w_scales"].double()[:, None]).t()
    outs = []
    turn = torch.polar(torch.ones_like(state["frequencies"], dtype=torch.float64)[None],
                       state["positions"].double()[:, None] * state["frequencies"].double())
    n = case["rotary"]
    for name in ("q", "k"):
        x = state[name].double()
        if case["normed"]:
            x = x / torch.sqrt(x.pow(2).mean(-1, keepdim=True) + EPS)
            x = x * state[name + "_norm"].double()
        order = torch.arange(n, device="cuda")
        pairs = order.view(-1, 2) if case["interleaved"] else order.view(2, -1).t()
        z = torch.complex(x[..., pairs[:, 0]], x[..., pairs[:, 1]]) * turn[:, None]
        y = x.clone()
        y[..., pairs[:, 0]], y[..., pairs[:, 1]] = z.real, z.imag
        outs.append(y)
    return outs
