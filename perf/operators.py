"""The operators of a key/value cache held in 4 bits, as measurable cases.

``write``   rotary positions on a step's q and k, K and V quantised into the cache rows of their tokens, and those rows read back
            (``rope_kv_write_int4``, ``read_kv_buffer_int4``)
``decode``  one query per sequence over its cached tokens (``flash_decoding_int4``)
``prompt``  portions of prompts, causal over what is cached of each sequence and over themselves (``flash_attention_int4``)
``maps``    the row of every new token, its position and the request table, from the requests' lengths (``build_slot_maps``)

A cache row holds one token: for every kv head the codes of K and of V (4 bits each, element 2i in the low half of byte i), then K's
and V's (scale, minimum) per group of elements, in the activations' type; the row is filled up to a multiple of 16 bytes.  An
element is ``minimum + scale * code``, where scale = (maximum - minimum) / 15 rounded to that type.

``run`` computes the plain form, or with ``own`` calls the framework.
"""

from __future__ import annotations

import math

import torch

own = False

DTYPES = {"fp16": torch.float16, "bf16": torch.bfloat16}
# (query heads, key/value heads, head size) of the presets (lite_llama_b200/executor/model_config.py)
HEADS = ((32, 8, 128), (28, 4, 128), (14, 2, 64), (32, 4, 128))


def listed() -> list[dict]:
    return [
        # one decode step of a serving batch of 32: a launch between two projections
        {"name": "write_step_32", "kind": "write", "heads": 32, "kv_heads": 8, "head_dim": 128, "group": 64, "batch": 32, "seq": 1,
         "dtype": "fp16"},
        # a padded prompt batch on its way into the cache
        {"name": "write_prompt_4x2000", "kind": "write", "heads": 28, "kv_heads": 4, "head_dim": 128, "group": 64, "batch": 4,
         "seq": 2000, "dtype": "bf16"},
        # one prompt of the small model
        {"name": "write_prompt_777_d64", "kind": "write", "heads": 14, "kv_heads": 2, "head_dim": 64, "group": 32, "batch": 1,
         "seq": 777, "dtype": "fp16"},
        # a single user's chat: latency
        {"name": "decode_1x201", "kind": "decode", "heads": 32, "kv_heads": 8, "head_dim": 128, "group": 64, "batch": 1,
         "context": 201, "rows": "slots", "dtype": "fp16"},
        # the serving batch, requests of different ages, rows handed out by the pool
        {"name": "decode_32x2000", "kind": "decode", "heads": 32, "kv_heads": 8, "head_dim": 128, "group": 64, "batch": 32,
         "context": 2000, "rows": "paged", "dtype": "fp16"},
        # two long documents, which a cache of 16 bits would not leave room for
        {"name": "decode_2x30000", "kind": "decode", "heads": 28, "kv_heads": 4, "head_dim": 128, "group": 128, "batch": 2,
         "context": 30000, "rows": "slots", "dtype": "bf16"},
        # many requests of the small model: short cache rows
        {"name": "decode_150x400_d64", "kind": "decode", "heads": 14, "kv_heads": 2, "head_dim": 64, "group": 32, "batch": 150,
         "context": 400, "rows": "paged", "dtype": "fp16"},
        # the next portion of a long prompt
        {"name": "prompt_1x512_over_7500", "kind": "prompt", "heads": 32, "kv_heads": 8, "head_dim": 128, "group": 64, "batch": 1,
         "new": 512, "context": 7500, "rows": "slots", "dtype": "fp16"},
        # follow-up turns of several chats at once, ragged
        {"name": "prompt_6x150_over_1200", "kind": "prompt", "heads": 28, "kv_heads": 4, "head_dim": 128, "group": 64, "batch": 6,
         "new": 150, "context": 1200, "rows": "paged", "dtype": "bf16"},
        # a few proposed tokens per request to be checked in one step
        {"name": "prompt_16x5_over_900", "kind": "prompt", "heads": 32, "kv_heads": 4, "head_dim": 128, "group": 32, "batch": 16,
         "new": 5, "context": 900, "rows": "paged", "dtype": "fp16"},
        # a decode step of 256 requests in fixed slots
        {"name": "maps_step_256", "kind": "maps", "batch": 256, "new": 1, "width": 4096, "rows": "slots"},
        # portions of seven prompts, rows from the pool
        {"name": "maps_prompt_7x1100", "kind": "maps", "batch": 7, "new": 1100, "width": 8192, "rows": "paged"},
    ]


def _log_int(rng, lo: int, hi: int) -> int:
    return max(lo, min(hi, round(math.exp(rng.uniform(math.log(lo), math.log(hi + 1))))))


def draw(rng) -> dict:
    kind = rng.choice(("write", "decode", "decode", "decode", "prompt", "prompt", "prompt", "maps"))
    if kind == "maps":
        batch = _log_int(rng, 1, 400)
        return {"kind": kind, "batch": batch, "new": _log_int(rng, 1, max(1, 8000 // batch)), "width": rng.choice((2048, 4096, 8192)),
                "rows": rng.choice(("slots", "paged"))}
    heads, kv_heads, head_dim = rng.choice(HEADS)
    case = {"kind": kind, "heads": heads, "kv_heads": kv_heads, "head_dim": head_dim,
            "group": rng.choice([g for g in (32, 64, 128) if g <= head_dim])}
    if kind == "write":
        case["batch"] = _log_int(rng, 1, 64)
        case["seq"] = rng.choice((1, _log_int(rng, 2, max(2, 4000 // case["batch"]))))
    else:
        case["rows"] = rng.choice(("slots", "paged"))
        if kind == "decode":
            case["batch"] = _log_int(rng, 1, 128)
            case["context"] = _log_int(rng, 1, min(30000, 50000 // case["batch"]))
        else:
            case["batch"] = _log_int(rng, 1, 16)
            case["new"] = _log_int(rng, 2, max(2, 512 // case["batch"]))
            case["context"] = _log_int(rng, 1, min(7500, 20000 // case["batch"]))
    case["dtype"] = rng.choice(("fp16", "bf16"))
    return case


# --------------------------------------------------------------------------------------------------- inputs
def _lengths(case, what: str) -> list[int]:
    """One length per request: the first is the case's, the others lie between half of it and it, the same for every seed."""
    n, batch = case[what], case["batch"]
    gen = torch.Generator().manual_seed(len(what) + 31 * batch + n)
    return [n, *torch.randint((n + 1) // 2, n + 1, (batch,), generator=gen).tolist()[1:]]


def _row_bytes(case) -> int:
    per_head = case["head_dim"] + 8 * (case["head_dim"] // case["group"])
    return (case["kv_heads"] * per_head + 15) // 16 * 16


def _quantise(x: torch.Tensor, group: int, wide: torch.dtype):
    """Codes, scale and minimum of ``x [..., D]`` in groups, computed in ``wide``: ``[..., D/group, group]``, ``[..., D/group]`` twice."""
    g = x.reshape(*x.shape[:-1], -1, group)
    lo, hi = torch.aminmax(g, dim=-1)
    scale = ((hi.to(wide) - lo.to(wide)) / 15).to(x.dtype)
    step = scale.to(wide)[..., None]
    code = ((g.to(wide) - lo.to(wide)[..., None]) / step).round().clamp(0, 15)
    code = torch.where(step > 0, code, torch.zeros_like(code)).to(torch.uint8)
    return code, scale, lo


def _pack(codes, scale, lo, heads: int, row_bytes: int) -> torch.Tensor:
    """Cache rows ``[tokens, row_bytes]`` of codes ``[tokens, 2 * heads, D/group, group]`` (K's heads, then V's)."""
    n = codes.shape[0]
    nib = codes.reshape(n, 2, heads, -1)
    code_bytes = (nib[..., 0::2] | (nib[..., 1::2] << 4)).permute(0, 2, 1, 3).reshape(n, heads, -1)
    params = torch.stack((scale, lo), dim=-1).reshape(n, 2, heads, -1).permute(0, 2, 1, 3).contiguous()
    rows = torch.cat((code_bytes, params.view(torch.uint8).reshape(n, heads, -1)), dim=-1).reshape(n, -1)
    return torch.nn.functional.pad(rows, (0, row_bytes - rows.shape[1]))


def _unpack(rows: torch.Tensor, heads: int, head_dim: int, group: int, dtype: torch.dtype, wide: torch.dtype) -> torch.Tensor:
    """The values that cache rows ``[..., row_bytes]`` stand for, in ``wide``: ``[..., 2, heads, D]`` (K, V)."""
    lead, groups = rows.shape[:-1], head_dim // group
    per_head = head_dim + 8 * groups
    r = rows[..., :heads * per_head].reshape(*lead, heads, per_head)
    codes = r[..., :head_dim].reshape(*lead, heads, 2, head_dim // 2)
    nib = torch.stack((codes & 15, codes >> 4), dim=-1).reshape(*lead, heads, 2, groups, group).to(wide)
    params = r[..., head_dim:].contiguous().view(dtype).reshape(*lead, heads, 2, groups, 2).to(wide)
    x = params[..., 1:] + params[..., :1] * nib
    return x.reshape(*lead, heads, 2, head_dim).transpose(-2, -3)


def _rotary(case, dev):
    positions = torch.arange(case["seq"], device=dev, dtype=torch.float64) + 100
    freqs = 5e5 ** (-torch.arange(0, case["head_dim"], 2, device=dev, dtype=torch.float64) / case["head_dim"])
    angle = (positions[:, None] * freqs).repeat(case["batch"], 1, 2)
    dtype = DTYPES[case["dtype"]]
    return angle.cos().to(dtype), angle.sin().to(dtype)


def prepare(case: dict, seed: int) -> dict:
    dev = "cuda"
    gen, host = torch.Generator(device=dev).manual_seed(seed), torch.Generator().manual_seed(seed)
    s = dict(case)
    if case["kind"] == "maps":
        batch, width = case["batch"], case["width"]
        new = _lengths(case, "new")
        ctx = torch.randint(1, width - max(new) + 1, (batch,), generator=host)
        s["total"] = sum(new) + 3                      # the flat batch is padded to a captured size
        requests = batch + 2
        s["req"] = torch.randperm(requests, generator=host)[:batch].to(torch.int32).to(dev)
        s["ctx"], s["new_len"] = ctx.to(torch.int32).to(dev), torch.tensor(new, dtype=torch.int32, device=dev)
        s["table"] = torch.arange(requests * width, dtype=torch.int32, device=dev).view(requests, width)
        s["pool"] = None
        if case["rows"] == "paged":
            s["pool"] = torch.randperm(requests * width, generator=gen, device=dev)[:s["total"]].to(torch.int32)
        return s
    dtype = DTYPES[case["dtype"]]
    hq, hkv, d = case["heads"], case["kv_heads"], case["head_dim"]

    def normal(*shape):
        return torch.empty(shape, device=dev).normal_(generator=gen)

    # keys have a few strong channels, the same in every token
    channel = normal(hkv, d).abs() * 0.5 + 0.75
    channel = torch.where(torch.rand(hkv, d, device=dev, generator=gen) < 0.03, channel * 4, channel)
    channel = torch.cat((channel, torch.ones(hkv, d, device=dev)))
    if case["kind"] == "write":
        tokens = case["batch"] * case["seq"]
        kv = normal(tokens, 2 * hkv, d) * channel
        s["qkv"] = torch.cat((normal(tokens, hq * d), kv.reshape(tokens, -1)), dim=1).to(dtype)
        s["cos"], s["sin"] = _rotary(case, dev)
        s["index"] = torch.randperm(tokens + 500, generator=gen, device=dev)[:tokens].to(torch.int32)
        s["cache"] = torch.zeros(tokens + 500, _row_bytes(case), dtype=torch.uint8, device=dev)
        s["q_out"] = torch.empty(tokens, hq, d, dtype=dtype, device=dev)
        s["k_out"] = torch.empty(tokens, hkv, d, dtype=dtype, device=dev)
        return s
    batch = case["batch"]
    new = _lengths(case, "new") if case["kind"] == "prompt" else [1] * batch
    cached = _lengths(case, "context")
    lens = [c + n for c, n in zip(cached, new)] if case["kind"] == "prompt" else cached
    width = (max(lens) + 255) // 256 * 256             # the bucket of a captured step
    requests = batch + 1
    total = requests * width if case["rows"] == "slots" else sum(lens) + 200
    cache = torch.empty(total, _row_bytes(case), dtype=torch.uint8, device=dev)
    for lo in range(0, total, 16384):
        n = min(total, lo + 16384) - lo
        x = (normal(n, 2 * hkv, d) * channel).to(dtype)
        cache[lo:lo + n] = _pack(*_quantise(x, case["group"], torch.float32), hkv, cache.shape[1])
    s["cache"] = cache
    if case["rows"] == "slots":
        s["table"] = torch.arange(total, dtype=torch.int32, device=dev).view(requests, width)
    else:
        s["table"] = torch.zeros(requests, width, dtype=torch.int32, device=dev)
    req = torch.randperm(requests, generator=host)[:batch].tolist()
    if case["rows"] == "paged":
        order = torch.randperm(total, generator=gen, device=dev).to(torch.int32)
        at = 0
        for r, n in zip(req, lens):
            s["table"][r, :n] = order[at:at + n]
            at += n
    s["req"] = torch.tensor(req, dtype=torch.int32, device=dev)
    s["len"] = torch.tensor(lens, dtype=torch.int32, device=dev)
    s["new_len"] = torch.tensor(new, dtype=torch.int32, device=dev)
    s["start"] = torch.cumsum(s["new_len"], 0, dtype=torch.int32) - s["new_len"]
    s["max_len"], s["max_new"] = width, max(new)
    tokens = sum(new)
    qkv = normal(tokens, (hq + 2 * hkv) * d).to(dtype)  # q where the projection left it
    s["q"] = qkv[:, :hq * d].view(tokens, hq, d)
    s["scale"] = d ** -0.5
    return s


# --------------------------------------------------------------------------------------------------- operators
def run(s: dict):
    return {"write": _write, "decode": _decode, "prompt": _prompt, "maps": _maps}[s["kind"]](s)


def _write(s):
    hq, hkv, d, dtype = s["heads"], s["kv_heads"], s["head_dim"], s["qkv"].dtype
    tokens = s["qkv"].shape[0]
    q = s["qkv"][:, :hq * d].view(tokens, hq, d)
    k = s["qkv"][:, hq * d:(hq + hkv) * d].view(tokens, hkv, d)
    v = s["qkv"][:, (hq + hkv) * d:].view(tokens, hkv, d)
    if own:
        from lite_llama_b200 import kernels as K

        q, k = K.rope_kv_write_int4(q, k, v, s["cos"], s["sin"], s["index"], s["cache"], s["batch"], s["seq"], s["group"],
                                    out_q=s["q_out"], out_k=s["k_out"])
        return q, k, K.read_kv_buffer_int4(s["cache"], s["index"], hkv, d, dtype, s["group"])
    q, k = _rotate(q, s, torch.float32), _rotate(k, s, torch.float32)
    index = s["index"].long()
    s["cache"][index] = _pack(*_quantise(torch.cat((k, v), dim=1), s["group"], torch.float64), hkv, s["cache"].shape[1])
    return q, k, _unpack(s["cache"][index], hkv, d, s["group"], dtype, torch.float32).reshape(tokens, 2 * hkv, d).to(dtype)


def _rotate(x, s, wide):
    half = x.shape[-1] // 2
    cos = s["cos"].reshape(x.shape[0], 1, -1)[..., :half].to(wide)
    sin = s["sin"].reshape(x.shape[0], 1, -1)[..., :half].to(wide)
    a, b = x[..., :half].to(wide), x[..., half:].to(wide)
    return torch.cat((a * cos - b * sin, b * cos + a * sin), dim=-1).to(x.dtype)


def _attend(q, kv, visible, scale):
    """``q [B, m, Hq, D]``, ``kv [B, n, 2, Hkv, D]``, ``visible [B, m, n]``, all in one wide type."""
    batch, m, hq, d = q.shape
    hkv = kv.shape[3]
    k, v = kv[:, :, 0].permute(0, 2, 3, 1), kv[:, :, 1].permute(0, 2, 1, 3)        # [B, Hkv, D, n], [B, Hkv, n, D]
    qg = q.reshape(batch, m, hkv, hq // hkv, d).permute(0, 2, 3, 1, 4).reshape(batch, hkv, -1, d)
    score = torch.matmul(qg, k).view(batch, hkv, hq // hkv, m, -1).mul_(scale)
    score.masked_fill_(~visible[:, None, None], -math.inf)
    p = (score - score.amax(-1, keepdim=True)).exp_()
    out = torch.matmul(p.view(batch, hkv, -1, p.shape[-1]), v).view(batch, hkv, -1, m, d)
    out = out / p.sum(-1)[..., None]
    return out.permute(0, 3, 1, 2, 4).reshape(batch, m, hq, d)


def _cached(s, longest, wide):
    rows = s["cache"][s["table"][s["req"].long(), :longest].long()]
    return _unpack(rows, s["kv_heads"], s["head_dim"], s["group"], DTYPES[s["dtype"]], wide)


def _decode(s):
    if own:
        from lite_llama_b200 import kernels as K

        return K.flash_decoding_int4(s["q"], s["cache"], s["scale"], s["table"], s["req"], s["len"], s["max_len"], s["kv_heads"],
                                     s["group"])
    return _decode_plain(s, torch.float32).to(s["q"].dtype)


def _decode_plain(s, wide):
    keys = torch.arange(s["max_len"], device=s["q"].device)
    visible = (keys < s["len"][:, None])[:, None]
    return _attend(s["q"].to(wide)[:, None], _cached(s, s["max_len"], wide), visible, s["scale"])[:, 0]


def _prompt(s):
    if own:
        from lite_llama_b200 import kernels as K

        return K.flash_attention_int4(s["q"], s["cache"], s["scale"], s["start"], s["new_len"], s["table"], s["req"], s["len"],
                                      s["max_new"], s["max_len"], s["kv_heads"], s["group"])
    dev, m = s["q"].device, s["max_new"]
    token = torch.arange(m, device=dev)
    flat = (s["start"][:, None] + token).clamp(max=s["q"].shape[0] - 1)              # [B, m]
    position = s["len"][:, None] - s["new_len"][:, None] + token
    visible = torch.arange(s["max_len"], device=dev) <= position[..., None]
    out = _attend(s["q"][flat].float(), _cached(s, s["max_len"], torch.float32), visible, s["scale"])
    return out[token < s["new_len"][:, None]].to(s["q"].dtype)


def _maps(s):
    if own:
        from lite_llama_b200 import kernels as K

        rows, position, start, length = K.build_slot_maps(s["req"], s["ctx"], s["new_len"], s["table"], s["total"], s["pool"])
        return rows, position, start, length, s["table"]
    end = torch.cumsum(s["new_len"], 0, dtype=torch.int64)
    token = torch.arange(s["total"], device=end.device)
    which = torch.searchsorted(end, token, right=True)
    valid = which < end.shape[0]
    which = which.clamp(max=end.shape[0] - 1)
    start = end - s["new_len"]
    position = torch.where(valid, s["ctx"].long()[which] + token - start[which], 0)
    place = torch.where(valid, s["req"].long()[which] * s["table"].shape[1] + position, 0)
    table = s["table"].view(-1)
    if s["pool"] is not None:                           # the tail writes what the first token writes
        table.index_copy_(0, torch.where(valid, place, place[0]), torch.where(valid, s["pool"], s["pool"][0]))
    rows = torch.where(valid, table[place], -1)
    return rows, position, start.to(torch.int32), s["ctx"] + s["new_len"], s["table"]


# --------------------------------------------------------------------------------------------------- floors
def work(case: dict) -> dict:
    """Inputs read once, outputs written once; lengths between half of the case's and it count as three quarters."""
    batch = case["batch"]
    mean = lambda n: n * (1 + 0.75 * (batch - 1)) / batch  # noqa: E731
    if case["kind"] == "maps":
        total = batch * mean(case["new"])
        return {"bytes": total * (4 + 8 + 4) + batch * 20, "flops": 0}
    hq, hkv, d = case["heads"], case["kv_heads"], case["head_dim"]
    row = _row_bytes(case)
    if case["kind"] == "write":
        tokens = batch * case["seq"]
        ins = (hq + 2 * hkv) * d * 2 + 2 * d * 2 + 4
        outs = (hq + hkv) * d * 2 + row + 2 * hkv * d * 2
        return {"bytes": tokens * (ins + outs), "flops": tokens * d * (3 * hq + 13 * hkv)}
    if case["kind"] == "decode":
        new, length = 1, mean(case["context"])
        pairs = batch * length
    else:
        new = mean(case["new"])
        length = mean(case["context"]) + new
        pairs = batch * new * (length - new / 2)
    return {"bytes": batch * (length * (row + 4) + 2 * new * hq * d * 2), "flops": 4 * pairs * hq * d}


# --------------------------------------------------------------------------------------------------- definitions in 64 bits
def exact(case: dict, seed: int):
    if case["kind"] == "maps":
        return None
    s = prepare(case, seed)
    hq, hkv, d, group = case["heads"], case["kv_heads"], case["head_dim"], case["group"]
    if case["kind"] == "write":
        x = s["qkv"].double().view(-1, hq + 2 * hkv, d)
        turned, half = x[:, :hq + hkv].clone(), d // 2
        cos, sin = (s[n].double().view(-1, 1, d)[..., :half] for n in ("cos", "sin"))
        turned[..., :half] = x[:, :hq + hkv, :half] * cos - x[:, :hq + hkv, half:] * sin
        turned[..., half:] = x[:, :hq + hkv, half:] * cos + x[:, :hq + hkv, :half] * sin
        # the cache holds what the rounded keys and the values come to on a grid of 16 steps between a group's ends
        kv = torch.cat((turned[:, hq:].to(s["qkv"].dtype).double(), x[:, hq + hkv:]), dim=1).unflatten(-1, (-1, group))
        low = kv.min(-1, keepdim=True).values
        step = ((kv.max(-1, keepdim=True).values - low) / 15).to(s["qkv"].dtype).double()
        steps = torch.clamp(torch.round((kv - low) / step), 0, 15)
        return turned[:, :hq], turned[:, hq:], (low + steps * step).flatten(-2)
    out = []
    bits = s["cache"].view(torch.uint8)
    per_head, groups = d + 8 * (d // group), d // group
    for b in range(case["batch"]):
        n, new, at = int(s["len"][b]), int(s["new_len"][b]), int(s["start"][b])
        rows = bits[s["table"][int(s["req"][b]), :n].long(), :hkv * per_head].view(n, hkv, per_head)
        both = []
        for side in (0, 1):
            code = rows[..., side * d // 2:(side + 1) * d // 2]
            code = torch.stack((code % 16, code // 16), -1).reshape(n, hkv, groups, group).double()
            at_params = d + side * 4 * groups
            params = rows[..., at_params:at_params + 4 * groups].contiguous().view(s["q"].dtype).view(n, hkv, groups, 2).double()
            both.append((code * params[..., 0, None] + params[..., 1, None]).view(n, hkv, d).repeat_interleave(hq // hkv, 1))
        q = s["q"][at:at + new].double()
        seen = torch.arange(n, device=q.device) <= torch.arange(n - new, n, device=q.device)[:, None]
        parts = []
        for h0 in range(0, hq, 4):                      # a few heads at a time: room for 64 bits
            weight = torch.einsum("mhd,nhd->hmn", q[:, h0:h0 + 4], both[0][:, h0:h0 + 4]) * s["scale"]
            weight = torch.softmax(torch.where(seen, weight, -math.inf), -1)
            parts.append(torch.einsum("hmn,nhd->mhd", weight, both[1][:, h0:h0 + 4]))
        out.append(torch.cat(parts, 1))
    return torch.cat(out)
