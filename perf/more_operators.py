"""The operators of microscaled 4-bit floating point (e2m1 elements, a power of two per 32 of them), as measurable cases.

``quantize``  activations to the 4-bit format and back (``mxfp4_quantize``, ``mxfp4_dequantize``)
``norm``      residual add, RMS norm and quantisation in one, with no rounding to 16 bits between them (``skip_rmsnorm_mxfp4``)
``product``   a projection: activations quantised on the way, weights in the format, sums in 32 bits (``mxfp4_matmul``)
``mlp``       a gated feed-forward: the activation and its quantisation follow from the first product's sums (``mxfp4_matmul``)
``experts``   routed experts: tokens sorted by expert, both products, and back with the routing weights (``fused_moe_mxfp4``)

A block of 32 consecutive elements of a row shares the scale 2^(byte - 127), the largest power of two not above its largest
magnitude, over 4; elements are 0, 0.5, 1, 1.5, 2, 3, 4 or 6 times that with a sign, rounded to the nearest (ties to the even code).
Element 2i of a row is the low half of byte i.  Scale bytes lie in tiles of 128 rows x 128 elements, the order that the tensor
cores read: ``[row tile][k tile][row % 32][row % 128 / 32][block % 4]``, filled up with zeros.  Gate and up rows of a feed-forward alternate
in runs of 64.

``run`` computes the plain form, or with ``own`` calls the framework.
"""

from __future__ import annotations

import math

import torch

own = False

DTYPES = {"fp16": torch.float16, "bf16": torch.bfloat16}
# hidden and feed-forward sizes of the presets (lite_llama_b200/executor/model_config.py)
SIZES = ((4096, 14336), (3584, 18944), (896, 4864), (4096, 12288))
# (experts, chosen, hidden, expert size) of the presets with routed experts
EXPERTS = ((128, 8, 2048, 768), (8, 2, 256, 128))
RUN = 64                                                # gate rows, then as many up rows
VALUES = (0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0)


def listed() -> list[dict]:
    return [
        # one user's token: latency
        {"name": "quantize_1x4096", "kind": "quantize", "tokens": 1, "width": 4096, "dtype": "fp16"},
        # activations of a prompt batch in front of a down projection
        {"name": "quantize_2000x14336", "kind": "quantize", "tokens": 2000, "width": 14336, "dtype": "bf16"},
        # a decode step of 32 requests
        {"name": "norm_32x4096", "kind": "norm", "tokens": 32, "width": 4096, "dtype": "fp16"},
        # a ragged prompt batch
        {"name": "norm_1999x3584", "kind": "norm", "tokens": 1999, "width": 3584, "dtype": "bf16"},
        # q, k and v of one user's token
        {"name": "product_1x6144x4096", "kind": "product", "tokens": 1, "out": 6144, "width": 4096, "bias": False, "dtype": "fp16"},
        # the down projection of a decode step
        {"name": "product_32x4096x14336", "kind": "product", "tokens": 32, "out": 4096, "width": 14336, "bias": False, "dtype": "bf16"},
        # q, k and v with their bias for an odd prompt
        {"name": "product_777x4608x3584", "kind": "product", "tokens": 777, "out": 4608, "width": 3584, "bias": True, "dtype": "bf16"},
        # gate and up of a full prompt batch
        {"name": "product_4000x28672x4096", "kind": "product", "tokens": 4000, "out": 28672, "width": 4096, "bias": False,
         "dtype": "fp16"},
        # a few requests of the small model
        {"name": "mlp_7x896x4864", "kind": "mlp", "tokens": 7, "width": 896, "inner": 4864, "dtype": "fp16"},
        # a prompt of a thousand tokens
        {"name": "mlp_1000x4096x14336", "kind": "mlp", "tokens": 1000, "width": 4096, "inner": 14336, "dtype": "bf16"},
        # a decode step over routed experts: most experts see two tokens
        {"name": "experts_32", "kind": "experts", "tokens": 32, "experts": 128, "chosen": 8, "width": 2048, "inner": 768, "dtype": "fp16"},
        # a prompt batch over routed experts
        {"name": "experts_2000", "kind": "experts", "tokens": 2000, "experts": 128, "chosen": 8, "width": 2048, "inner": 768,
         "dtype": "bf16"},
    ]


def _log_int(rng, lo: int, hi: int) -> int:
    return max(lo, min(hi, round(math.exp(rng.uniform(math.log(lo), math.log(hi + 1))))))


def draw(rng) -> dict:
    kind = rng.choice(("quantize", "norm", "product", "product", "product", "mlp", "mlp", "experts", "experts"))
    case = {"kind": kind, "dtype": rng.choice(("fp16", "bf16"))}
    if kind == "experts":
        case["experts"], case["chosen"], case["width"], case["inner"] = rng.choice(EXPERTS)
        case["tokens"] = _log_int(rng, 1, 2000)
        return case
    hidden, inner = rng.choice(SIZES)
    if kind == "mlp":
        case.update(width=hidden, inner=inner, tokens=_log_int(rng, 1, 1000))
    elif kind == "norm":
        case.update(width=hidden, tokens=_log_int(rng, 1, 4000))
    elif kind == "quantize":
        case.update(width=rng.choice((hidden, inner, 32 * rng.randint(1, 300))), tokens=_log_int(rng, 1, 2000))
    else:
        out, width = rng.choice(((hidden, inner), (2 * inner, hidden), (hidden, hidden),
                                 (rng.randint(33, 9000), 32 * rng.randint(2, 280))))
        case.update(out=out, width=width, bias=rng.random() < 0.3, tokens=_log_int(rng, 1, min(4000, 450_000_000_000 // (out * width))))
    return case


# --------------------------------------------------------------------------------------------------- the format
def _quantise(x: torch.Tensor):
    """Codes (one per byte) and scale bytes of ``x [..., K]`` in its own type: ``[..., K/32, 32]``, ``[..., K/32]``."""
    g = x.unflatten(-1, (-1, 32))
    top = g.abs().amax(-1)
    field = torch.frexp(top.double())[1] + 126          # the exponent field of a 32-bit float
    byte = (field - 2).clamp(0, 254)
    byte = torch.where(top > 0, byte, torch.zeros_like(byte))
    byte = torch.where(top.isfinite(), byte, torch.full_like(byte, 255))
    t = torch.ldexp(g, (127 - byte)[..., None])
    m = t.abs()
    code = (m > 0.25).to(torch.uint8)
    code += m >= 0.75
    code += m > 1.25
    code += m >= 1.75
    code += m > 2.5
    code += m >= 3.5
    code += m > 5
    code += (t < 0).to(torch.uint8) << 3
    code = torch.where((byte == 255)[..., None], torch.zeros_like(code), code)
    return code, byte.to(torch.uint8)


def _scale(byte: torch.Tensor, wide: torch.dtype) -> torch.Tensor:
    bits = byte.to(torch.int32) << 23
    bits = torch.where(byte == 0, 0x00400000, bits)
    bits = torch.where(byte == 255, 0x7FC00000, bits)
    return bits.to(torch.int32).view(torch.float32).to(wide)


def _value(code: torch.Tensor, byte: torch.Tensor, wide: torch.dtype) -> torch.Tensor:
    """What codes ``[..., K/32, 32]`` and scale bytes ``[..., K/32]`` stand for: ``[..., K]``."""
    table = torch.tensor(VALUES + tuple(-v for v in VALUES), dtype=wide, device=code.device)
    return (table[code.int()] * _scale(byte, wide)[..., None]).flatten(-2)


def _store(code: torch.Tensor, byte: torch.Tensor):
    """Weights as they are kept: codes ``[..., N, K/2]`` and scale tiles ``[..., N/128, K/128, 32, 4, 4]``."""
    nib = code.flatten(-2)
    rows, blocks = byte.shape[-2:]
    b = torch.nn.functional.pad(byte, (0, -blocks % 4, 0, -rows % 128))
    tiles = b.unflatten(-1, (-1, 4)).unflatten(-3, (-1, 4, 32))          # [..., N/128, 4, 32, K/128, 4]
    return (nib[..., 0::2] | (nib[..., 1::2] << 4)).contiguous(), tiles.movedim(-2, -4).transpose(-3, -2).contiguous()


def _load(codes: torch.Tensor, tiles: torch.Tensor, wide: torch.dtype) -> torch.Tensor:
    """The values of stored weights: ``[..., N, K]``."""
    rows, blocks = codes.shape[-2], codes.shape[-1] // 16
    byte = tiles.transpose(-3, -2).movedim(-4, -2).flatten(-2).flatten(-4, -2)[..., :rows, :blocks]
    return _value(torch.stack((codes & 15, codes >> 4), -1).flatten(-2).unflatten(-1, (-1, 32)), byte, wide)


def _rounded(x: torch.Tensor, wide: torch.dtype) -> torch.Tensor:
    return _value(*_quantise(x), wide)


# --------------------------------------------------------------------------------------------------- inputs
def prepare(case: dict, seed: int) -> dict:
    dev = "cuda"
    gen = torch.Generator(device=dev).manual_seed(seed)
    s, dtype, tokens, width = dict(case), DTYPES[case["dtype"]], case["tokens"], case["width"]

    def normal(*shape):
        return torch.empty(shape, device=dev).normal_(generator=gen)

    def activations(n, k):
        """A few strong channels, the same in every token, and tokens of different strength."""
        strong = torch.where(torch.rand(k, device=dev, generator=gen) < 0.01, 8.0, 1.0)
        return (normal(n, k) * strong * normal(n, 1).mul_(0.3).exp_()).to(dtype)

    def weights(n, k):
        return _quantise(normal(n, k) * 0.02)

    def gated(inner, k):
        """Gate and up rows in alternating runs."""
        gate, up = weights(inner, k), weights(inner, k)
        return tuple(torch.stack((g.unflatten(0, (-1, RUN)), u.unflatten(0, (-1, RUN))), 1).flatten(0, 2) for g, u in zip(gate, up))

    s["x"] = activations(tokens, width)
    if case["kind"] == "norm":
        s["residual"] = (activations(tokens, width).float() * 3).to(dtype)
        s["weight"] = (1 + 0.2 * normal(width)).to(dtype)
        s["sum"] = torch.empty_like(s["residual"])
        s["eps"] = 1e-5
    elif case["kind"] == "product":
        s["w"] = _store(*weights(case["out"], width))
        s["b"] = normal(case["out"]).to(dtype) if case["bias"] else None
    elif case["kind"] == "mlp":
        s["w1"] = _store(*gated(case["inner"], width))
        s["w2"] = _store(*weights(width, case["inner"]))
    elif case["kind"] == "experts":
        experts, inner = case["experts"], case["inner"]
        per = [(_store(*gated(inner, width)), _store(*weights(width, inner))) for _ in range(experts)]
        s["w1"], s["w2"] = (tuple(torch.stack([p[i][j] for p in per]) for j in range(2)) for i in range(2))
        logits = normal(tokens, experts) + 0.5 * normal(experts)         # some experts are liked better
        top = torch.softmax(logits, -1).topk(case["chosen"], -1)
        s["weights"], s["ids"] = (top.values / top.values.sum(-1, keepdim=True)).to(dtype), top.indices
        s["most"] = int(torch.bincount(top.indices.flatten(), minlength=experts).max())      # room for an expert's tokens
    return s


# --------------------------------------------------------------------------------------------------- operators
def run(s: dict):
    return {"quantize": _quantize, "norm": _norm, "product": _product, "mlp": _mlp, "experts": _experts}[s["kind"]](s)


def _quantize(s):
    if own:
        from lite_llama_b200 import kernels as K

        return K.mxfp4_dequantize(K.mxfp4_quantize(s["x"]), s["x"].dtype)
    return _rounded(s["x"].float(), torch.float32).to(s["x"].dtype)


def _norm(s):
    if own:
        from lite_llama_b200 import kernels as K

        q, total = K.skip_rmsnorm_mxfp4(s["x"], s["residual"], s["weight"], s["eps"], out_residual=s["sum"])
        return K.mxfp4_dequantize(q, s["x"].dtype), total
    dtype = s["x"].dtype
    total = s["x"].double() + s["residual"].double()    # in 64 bits: values next to a border
    y = total / (total.square().mean(-1, keepdim=True) + s["eps"]).sqrt() * s["weight"].double()
    s["sum"].copy_(total)
    return _rounded(y, torch.float32).to(dtype), s["sum"]


def _product(s):
    if own:
        from lite_llama_b200 import kernels as K

        return K.mxfp4_matmul(s["x"], K.MXFP4(*s["w"]), bias=s["b"])
    y = _rounded(s["x"].float(), torch.float32) @ _load(*s["w"], torch.float32).t()
    return (y if s["b"] is None else y + s["b"].float()).to(s["x"].dtype)


def _unit(y):
    """``silu(gate) * up`` of sums whose columns alternate in runs."""
    g, u = y.unflatten(-1, (-1, 2, RUN)).unbind(-2)
    return (g / (1 + (-g).exp()) * u).flatten(-2)


def _mlp(s):
    if own:
        from lite_llama_b200 import kernels as K

        return K.mxfp4_matmul(K.mxfp4_matmul(s["x"], K.MXFP4(*s["w1"]), swiglu=True), K.MXFP4(*s["w2"]), out_dtype=s["x"].dtype)
    # the first product in 64 bits: the values that are rounded next lie next to borders
    y = _rounded(s["x"].double(), torch.float64) @ _load(*s["w1"], torch.float64).t()
    return (_rounded(_unit(y), torch.float32) @ _load(*s["w2"], torch.float32).t()).to(s["x"].dtype)


def _experts(s):
    if own:
        from lite_llama_b200 import kernels as K

        return K.fused_moe_mxfp4(s["x"], K.MXFP4(*s["w1"]), K.MXFP4(*s["w2"]), s["weights"], s["ids"])
    dev, tokens, chosen, most = s["x"].device, s["tokens"], s["chosen"], s["most"]
    slot = s["ids"].flatten()
    order = torch.argsort(slot, stable=True)
    first = torch.searchsorted(slot[order], torch.arange(s["experts"], device=dev))
    place = torch.empty_like(slot)                      # of a slot among its expert's rows
    place[order] = torch.arange(slot.numel(), device=dev) - first[slot[order]]
    rows = torch.zeros(s["experts"], most, s["width"], device=dev, dtype=torch.float64)
    rows[slot, place] = _rounded(s["x"].double(), torch.float64).repeat_interleave(chosen, 0)
    y = torch.bmm(rows, _load(*s["w1"], torch.float64).transpose(1, 2))
    y = torch.bmm(_rounded(_unit(y), torch.float32), _load(*s["w2"], torch.float32).transpose(1, 2))
    out = y[slot, place].view(tokens, chosen, -1) * s["weights"].float()[..., None]
    return out.sum(1).to(s["x"].dtype)


# --------------------------------------------------------------------------------------------------- floors
def work(case: dict) -> dict:
    """Inputs read once, outputs written once; an element of the format takes half a byte and a 32nd."""
    t, k, q = case["tokens"], case["width"], 17 / 32
    if case["kind"] == "quantize":
        return {"bytes": t * k * (2 + 2), "flops": 4 * t * k}
    if case["kind"] == "norm":
        return {"bytes": t * k * (2 + 2 + 2 + 2) + 2 * k, "flops": 9 * t * k}
    if case["kind"] == "product":
        n = case["out"]
        return {"bytes": n * k * q + 2 * t * k + 2 * t * n, "flops": 2 * t * n * k}
    i = case["inner"]
    if case["kind"] == "mlp":
        return {"bytes": 3 * i * k * q + 4 * t * k, "flops": 6 * t * i * k}
    seen = case["experts"] * (1 - (1 - case["chosen"] / case["experts"]) ** t)
    return {"bytes": seen * 3 * i * k * q + 4 * t * k + 10 * t * case["chosen"], "flops": 6 * t * case["chosen"] * i * k}


# --------------------------------------------------------------------------------------------------- definitions in 64 bits
def _grid(x: torch.Tensor) -> torch.Tensor:
    """``x [..., K]`` (64 bits) on the format's grid, by arithmetic."""
    b = x.reshape(*x.shape[:-1], -1, 32)
    high = b.abs().max(-1, keepdim=True).values
    power = torch.floor(torch.log2(high.clamp_min(1e-300)))
    power = power + (high >= 2.0 ** (power + 1)).double() - (high < 2.0 ** power).double()            # log2 rounds
    scale = 2.0 ** (power - 2).clamp(min=-127)
    size = (b / scale).abs()
    step = torch.where(size < 2, 0.5, torch.where(size < 4, 1.0, 2.0))
    return (torch.sign(b) * torch.clamp(torch.round(size / step) * step, max=6) * scale).reshape(x.shape)


def _stored(w) -> torch.Tensor:
    codes, tiles = w
    n, k = codes.shape[0], codes.shape[1] * 2
    e = torch.empty(n, k, dtype=torch.float64, device=codes.device)
    for half in (0, 1):
        c = (codes // 16 if half else codes % 16).double()
        size = c % 8
        size = torch.where(size < 4, size / 2, torch.where(size < 6, size - 2, 2 * size - 8))
        e[:, half::2] = torch.where(c >= 8, -size, size)
    row, block = torch.arange(n, device=codes.device)[:, None], torch.arange(k // 32, device=codes.device)
    byte = tiles[row // 128, block // 4, row % 32, row % 128 // 32, block % 4]
    return e * (2.0 ** (byte.double() - 127)).repeat_interleave(32, 1)


def _halves(w, inner: int):
    full = _stored(w)
    row = torch.arange(inner, device=full.device)
    row = row // RUN * 2 * RUN + row % RUN
    return full[row], full[row + RUN]


def exact(case: dict, seed: int):
    s = prepare(case, seed)
    x = s["x"].double()
    if case["kind"] == "quantize":
        return _grid(x)
    if case["kind"] == "norm":
        x = x + s["residual"].double()
        mean = torch.einsum("tk,tk->t", x, x) / case["width"]
        return _grid(x * torch.rsqrt(mean + s["eps"])[:, None] * s["weight"].double()), x
    if case["kind"] == "product":
        y = torch.einsum("tk,nk->tn", _grid(x), _stored(s["w"]))
        return y if s["b"] is None else y + s["b"].double()

    def feed_forward(rows, w1, w2):
        gate, up = (torch.einsum("tk,nk->tn", rows, w) for w in _halves(w1, case["inner"]))
        return torch.einsum("tk,nk->tn", _grid(torch.sigmoid(gate) * gate * up), _stored(w2))

    if case["kind"] == "mlp":
        return feed_forward(_grid(x), s["w1"], s["w2"])
    out, rows = torch.zeros_like(x), _grid(x)
    for e in range(case["experts"]):
        token, choice = torch.nonzero(s["ids"] == e, as_tuple=True)
        if token.numel():
            y = feed_forward(rows[token], [w[e] for w in s["w1"]], [w[e] for w in s["w2"]])
            out.index_add_(0, token, y * s["weights"][token, choice].double()[:, None])
    return out
