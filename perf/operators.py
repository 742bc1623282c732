"""Cases of the 8-bit transformer operators: what they compute in plain torch operations, in 64 bits, and the calls that a
program makes of the library.

Operators, all on uint8 codes with (scale, zero point) pairs, value = scale * (code - zero point):

  tokens     Quantize every row of a matrix with parameters of its own, and read the values back.
  linear     y = x w^T + b with x quantised per row (token) on the fly and w held in 8 bits per row (output channel).
  append     New keys and values of several sequences into a paged cache with one scale per block of tokens and head.
  attention  Causal attention of the newest tokens of several sequences over that cache.
"""
import math
import random

import torch

own = False

TINY = 2.0 ** -126  # smallest normal float: no scale is smaller
DTYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
BYTES = {"f32": 4, "f16": 2, "bf16": 2}


def listed():
    return [
        # a handful of tokens between two layers of a decode step: latency
        dict(name="tokens_small", op="tokens", tokens=7, features=4096, dtype="bf16"),
        # rows of an odd length, full precision
        dict(name="tokens_odd_f32", op="tokens", tokens=2053, features=1021, dtype="f32"),
        # a long prompt's activations
        dict(name="tokens_large", op="tokens", tokens=16384, features=8192, dtype="bf16"),
        # one token through a feed-forward matrix: weight streaming
        dict(name="linear_one_token", op="linear", tokens=1, features=4096, out_features=11008, dtype="bf16", bias=False),
        # a decode batch that is not a multiple of anything, odd output width
        dict(name="linear_batch_odd", op="linear", tokens=77, features=4096, out_features=4099, dtype="f16", bias=True),
        # a prompt through a square layer
        dict(name="linear_square", op="linear", tokens=4096, features=4096, out_features=4096, dtype="bf16", bias=True),
        # a large batch of prompts, full-precision output
        dict(name="linear_large_f32", op="linear", tokens=8192, features=8192, out_features=8192, dtype="f32", bias=False),
        # every sequence of a decode batch gets one more token; blocks part-filled, scales that have to grow among them
        dict(name="append_decode", op="append", seqs=64, new=1, longest=48, kv_heads=8, block=32, head_dim=128, dtype="bf16", ragged=1),
        # ragged prompts arrive
        dict(name="append_prompt", op="append", seqs=5, new=3500, longest=3700, kv_heads=8, block=64, head_dim=128, dtype="f16", ragged=2),
        # one short conversation, one token: latency
        dict(name="attention_short", op="attention", seqs=1, new=1, longest=777, q_heads=32, kv_heads=8, block=16, head_dim=128, dtype="bf16", ragged=3),
        # a ragged decode batch, grouped heads
        dict(name="attention_decode", op="attention", seqs=64, new=1, longest=8192, q_heads=64, kv_heads=8, block=64, head_dim=128, dtype="bf16", ragged=4),
        # a chunk of a prompt behind a long context
        dict(name="attention_chunk", op="attention", seqs=2, new=1500, longest=6000, q_heads=32, kv_heads=8, block=64, head_dim=128, dtype="f16", ragged=5),
    ]


def _log(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    op = rng.choice(["tokens", "linear", "linear", "append", "attention", "attention", "attention"])
    dtype = rng.choice(["bf16", "bf16", "f16", "f32"])
    if op == "tokens":
        features = _log(rng, 64, 12000)
        return dict(op=op, tokens=_log(rng, 1, min(16384, 100_000_000 // features)), features=features, dtype=dtype)
    if op == "linear":
        # widths a layer has, mostly multiples of 16 or 128, now and then odd (those up to a few thousand)
        step = rng.choice([128, 128, 16, 1])
        features = max(step, _log(rng, 256, 8192 if step > 1 else 2000) // step * step)
        out = _log(rng, 64, 11008)
        if rng.random() < 0.7:
            out = max(16, out // 16 * 16)
        most = 2.0e11 if step > 1 else 4.0e9
        return dict(op=op, tokens=_log(rng, 1, max(1, min(8192, int(most / (features * out))))), features=features, out_features=out,
                    dtype=dtype, bias=rng.random() < 0.5)
    head_dim = rng.choice([64, 128, 128, 96, 256])
    kv_heads = rng.choice([1, 2, 4, 8])
    block = rng.choice([16, 32, 64, 128])
    ragged = rng.randrange(1 << 20)
    if op == "append":
        seqs = _log(rng, 1, 64)
        new = rng.choice([1, _log(rng, 1, max(1, 16000 // seqs))])
        return dict(op=op, seqs=seqs, new=new, longest=new + rng.randrange(0, 300), kv_heads=kv_heads, block=block, head_dim=head_dim,
                    dtype=dtype, ragged=ragged)
    q_heads = kv_heads * rng.choice([1, 2, 4, 7, 8, 12])
    if rng.random() < 0.7:  # decode and short drafts
        seqs, new = _log(rng, 1, 64), rng.choice([1, 1, 1, 2, 5])
        longest = _log(rng, 16, max(16, min(32000, 64 * 8192 * 8 * 128 // (4 * seqs * kv_heads * head_dim))))
    else:
        seqs = rng.choice([1, 2, 3])
        longest = _log(rng, 64, 6000 // seqs)
        new = _log(rng, 8, max(8, min(longest, 90_000_000 // (longest * q_heads * seqs))))
    return dict(op=op, seqs=seqs, new=min(new, longest), longest=longest, q_heads=q_heads, kv_heads=kv_heads, block=block, head_dim=head_dim,
                dtype=dtype, ragged=ragged)


def _ragged(case):
    """(new tokens, length in all) of every sequence: the first has the longest, the others anything below."""
    r = random.Random(case["ragged"])
    got = []
    for i in range(case["seqs"]):
        length = case["longest"] if i == 0 else r.randint(max(1, case["longest"] // 4), case["longest"])
        new = case["new"] if i == 0 or case["new"] <= 5 else r.randint(max(1, case["new"] // 4), case["new"])
        got.append((min(new, length), length))
    return got


def _generator(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def _randn(g, *shape):
    return torch.randn(shape, generator=g, device="cuda")


def _activations(g, tokens, features, dtype):
    """Rows of different size with a few channels that stick out, as between transformer layers."""
    x = _randn(g, tokens, features)
    x *= torch.exp(0.5 * _randn(g, tokens, 1))
    loud = torch.randint(0, features, (max(1, features // 256),), generator=g, device="cuda")
    x[:, loud] *= 12.0
    return x.to(dtype)


def _pairs(scale, zero):
    """(scale, zero point) pairs in the library's 8-byte form."""
    p = torch.zeros(*scale.shape, 8, dtype=torch.uint8, device=scale.device)
    p.view(torch.float32)[..., 0] = scale
    p[..., 4] = zero
    return p


def _scale_of(p):
    return p.view(torch.float32)[..., 0]


def prepare(case, seed):
    g = _generator(seed)
    dtype = DTYPES[case["dtype"]]
    s = {"case": case}
    if case["op"] in ("tokens", "linear"):
        s["x"] = _activations(g, case["tokens"], case["features"], dtype)
        if case["op"] == "linear":
            n, k = case["out_features"], case["features"]
            s["w"] = torch.randint(0, 256, (n, k), generator=g, device="cuda", dtype=torch.uint8)
            zero = torch.randint(118, 138, (n,), generator=g, device="cuda", dtype=torch.uint8)
            s["w_pairs"] = _pairs(0.0004 * torch.exp(0.3 * _randn(g, n)), zero)
            s["bias"] = _randn(g, n) if case["bias"] else None
            if own:
                import sys
                sys.path.insert(0, "light-tensor_b200/python") if "light-tensor_b200/python" not in sys.path else None
                import ltq
                s["layer"] = ltq.FullyConnected_t(s["w"], s["w_pairs"], s["bias"])
        return s
    spans = _ragged(case)
    per = [-(-length // case["block"]) for _, length in spans]
    blocks, width = sum(per) + 3, max(per)
    order = torch.randperm(blocks, generator=g, device="cuda").to(torch.int32)
    table = torch.zeros(len(spans), width, dtype=torch.int32)
    order = order.cpu()
    at = 0
    for i, n in enumerate(per):
        table[i, :n] = order[at:at + n]
        at += n
    s["table"] = table.cuda()
    s["lengths"] = torch.tensor([length for _, length in spans], dtype=torch.int32, device="cuda")
    offsets = [0]
    for new, _ in spans:
        offsets.append(offsets[-1] + new)
    s["offsets"] = torch.tensor(offsets, dtype=torch.int32, device="cuda")
    s["max_new"] = max(new for new, _ in spans)
    shape = (blocks, case["kv_heads"], case["block"], case["head_dim"])
    for name in ("k", "v"):
        s[name] = torch.empty(shape, dtype=torch.uint8, device="cuda")
        for i in range(0, blocks, 512):
            part = s[name][i:i + 512]
            part.copy_((128 + 36 * _randn(g, *part.shape)).round_().clamp_(1, 255))
        size = 0.03 if name == "k" else 0.02
        s[name + "_pairs"] = _pairs(size * torch.exp(0.4 * _randn(g, blocks, case["kv_heads"])), torch.full((blocks, case["kv_heads"]), 128, device="cuda"))
    total = offsets[-1]
    if case["op"] == "append":
        for name in ("new_k", "new_v"):
            s[name] = (1.2 * _randn(g, total, case["kv_heads"], case["head_dim"])).to(dtype)
    else:
        s["q"] = _randn(g, total, case["q_heads"], case["head_dim"]).to(dtype)
    if own:
        import sys
        sys.path.insert(0, "light-tensor_b200/python") if "light-tensor_b200/python" not in sys.path else None
        import ltq
        s["cache"] = ltq.KVCache(s["k"], s["k_pairs"], s["v"], s["v_pairs"])
    return s


# ---- plain forms ------------------------------------------------------------------------------------------------------

def _round_away(v):
    """Nearest whole number, halves away from zero, for v >= 0 (in 64 bits: v + 0.5 must not round up by itself)."""
    return torch.floor(v.double() + 0.5)


def _over(x, number):
    """x / number as one correctly rounded division (a float tensor over a Python number is a product with its reciprocal)."""
    return (x.double() / number).float()


def _quantize(x, scale, zero):
    v = zero + x / scale
    return _round_away(v.clamp(0.0, 255.0)).float()


def _quantize_rows(x):
    """codes (as floats), scale, zero point of every row."""
    x = x.float()
    lo, hi = x.amin(1, keepdim=True).clamp(max=0.0), x.amax(1, keepdim=True).clamp(min=0.0)
    scale = _over(hi - lo, 255.0).clamp(min=TINY)
    zero = _round_away(0.0 - lo / scale).float()
    return _quantize(x, scale, zero), scale, zero


def _plain_append(s):
    block = s["case"]["block"]
    total = s["new_k"].shape[0]
    seq = torch.searchsorted(s["offsets"], torch.arange(total, device="cuda", dtype=torch.int32), right=True) - 1
    new = s["offsets"][1:] - s["offsets"][:-1]
    first = (s["lengths"] - new)[seq]                     # the first position this call writes in the token's sequence
    pos = torch.arange(total, device="cuda") - s["offsets"][seq] + first
    page = s["table"][seq, pos // block].long()
    start = pos - pos % block
    kept = (first - start).clamp(min=0)                  # tokens in the block from earlier calls
    out = {}
    for name in ("k", "v"):
        x = s["new_" + name].float()
        codes, pairs = s[name], s[name + "_pairs"]
        need = _over(torch.zeros(codes.shape[:2], device="cuda").index_reduce_(0, page, x.abs().amax(2), "amax"), 127.0)
        older = torch.zeros(codes.shape[0], dtype=torch.long, device="cuda").index_reduce_(0, page, kept, "amax")
        touched = torch.zeros(codes.shape[0], dtype=torch.bool, device="cuda").index_fill_(0, page, True)
        old = _scale_of(pairs)
        fresh = (older == 0)[:, None]
        scale = torch.where(fresh, need.clamp(min=TINY), torch.maximum(old, need))
        scale = torch.where(touched[:, None], scale, old)
        grown = (scale > old) & touched[:, None] & ~fresh
        earlier = torch.arange(block, device="cuda")[None, None, :] < older[:, None, None]
        again = _quantize(old[..., None, None] * (codes.float() - 128.0), scale[..., None, None], 128.0)
        codes.copy_(torch.where((grown[..., None] & earlier)[..., None], again, codes.float()))
        codes[page, :, pos % block] = _quantize(x, scale[page][..., None], 128.0).to(torch.uint8)
        pairs.copy_(_pairs(scale, torch.where(touched[:, None], 128, pairs[..., 4])))
        out[name] = scale[..., None, None] * (codes.float() - pairs[..., 4, None, None].float())
        out[name + "_scale"] = scale
    return out


def _plain_attention(s):
    case = s["case"]
    group = case["q_heads"] // case["kv_heads"]
    new = (s["offsets"][1:] - s["offsets"][:-1]).long()
    seqs, most = new.shape[0], s["max_new"]
    t = torch.arange(most, device="cuda")
    at = (s["offsets"][:-1, None] + t).long()             # row of q, sequence by new token
    real = t < new[:, None]
    q = s["q"].float()[torch.where(real, at, 0)]          # [seqs, most, q_heads, head_dim]
    q = q.reshape(seqs, most, case["kv_heads"], group, -1).permute(0, 2, 3, 1, 4).reshape(seqs, case["kv_heads"], group * most, -1)

    def values(name):
        pages = s["table"].long()
        x = _scale_of(s[name + "_pairs"])[pages][..., None, None] * (s[name][pages].float() - s[name + "_pairs"][pages][..., 4, None, None].float())
        return x.permute(0, 2, 1, 3, 4).flatten(2, 3)     # [seqs, kv_heads, keys, head_dim]

    scores = q @ values("k").transpose(2, 3) / math.sqrt(case["head_dim"])
    pos = (s["lengths"].long() - new)[:, None] + t        # [seqs, most]
    seen = torch.arange(scores.shape[3], device="cuda") <= pos[..., None]
    seen = seen[:, None, None].expand(-1, -1, group, -1, -1).flatten(2, 3)
    scores = scores.masked_fill(~seen, -math.inf)
    p = torch.exp(scores - scores.amax(3, keepdim=True))
    o = (p @ values("v")) / p.sum(3, keepdim=True)
    o = o.reshape(seqs, case["kv_heads"], group, most, -1).permute(0, 3, 1, 2, 4).reshape(seqs, most, case["q_heads"], -1)
    return o[real].to(s["q"].dtype)


def run(state):
    case = state["case"]
    op = case["op"]
    if own:
        import ltq
        if op == "tokens":
            codes, pairs, _ = ltq.quantize_tokens(state["x"])
            return {"values": ltq.dequantize_tokens(codes, pairs, state["x"].dtype), "scale": _scale_of(pairs), "zero": pairs[:, 4]}
        if op == "linear":
            return state["layer"].forward(state["x"])
        if op == "append":
            cache = state["cache"]
            cache.append(state["new_k"], state["new_v"], state["table"], state["lengths"], state["offsets"], state["max_new"])
            k, v = cache.values()
            return {"k": k, "k_scale": _scale_of(state["k_pairs"]), "v": v, "v_scale": _scale_of(state["v_pairs"])}
        return state["cache"].attention(state["q"], state["table"], state["lengths"], state["offsets"], state["max_new"])
    if op == "tokens":
        codes, scale, zero = _quantize_rows(state["x"])
        return {"values": (scale * (codes - zero)).to(state["x"].dtype), "scale": scale[:, 0], "zero": zero[:, 0].to(torch.uint8)}
    if op == "linear":
        codes, scale, zero = _quantize_rows(state["x"])
        y = (codes - zero) @ (state["w"].float() - state["w_pairs"][:, 4:5].float()).t()
        y = y * scale * _scale_of(state["w_pairs"])
        if state["bias"] is not None:
            y = y + state["bias"]
        return y.to(state["x"].dtype)
    if op == "append":
        return _plain_append(state)
    return _plain_attention(state)


def work(case):
    op = case["op"]
    size = BYTES[case["dtype"]]
    if op == "tokens":
        n = case["tokens"] * case["features"]
        return {"bytes": 2 * n * size + 2 * n + 16 * case["tokens"], "flops": 6.0 * n}
    if op == "linear":
        m, n, k = case["tokens"], case["out_features"], case["features"]
        return {"bytes": size * m * k + n * k + 8 * n + (4 * n if case["bias"] else 0) + size * m * n, "flops": 2.0 * m * n * k}
    spans = _ragged(case)
    row = case["kv_heads"] * case["head_dim"]
    total = sum(new for new, _ in spans)
    if op == "append":
        blocks = sum(-(-length // case["block"]) for _, length in spans) + 3
        cache = 2 * blocks * case["block"] * row
        # new tokens in, their codes out; then the whole cache read back as float32 values
        return {"bytes": 2 * total * row * (size + 1) + cache * 5 + 2 * 16 * blocks * case["kv_heads"], "flops": 6.0 * total * row + 2.0 * cache}
    pairs = sum(new * length - new * (new - 1) // 2 for new, length in spans)
    held = sum(length for _, length in spans)
    blocks = sum(-(-length // case["block"]) for _, length in spans)
    return {"bytes": 2 * held * row + 16 * blocks * case["kv_heads"] + 4 * blocks + 2 * total * case["q_heads"] * case["head_dim"] * size,
            "flops": 4.0 * pairs * case["q_heads"] * case["head_dim"]}


# ---- 64 bits ------------------------------------------------------------------------------------------------------------
# The parameters and codes are defined with single-precision roundings (a scale is stored as a float, a quotient and its sum with
# the zero point are rounded to float before the code is taken); those roundings are part of the definition and are made here
# explicitly, everything else stays in 64 bits.

def _f32(v):
    return v.to(torch.float32).double()


def _exact_codes(x, scale, zero):
    v = _f32(zero + _f32(x / scale)).clamp(0.0, 255.0)
    return torch.trunc(v + 0.5)


def _exact_rows(x):
    x = x.double()
    zeros = torch.zeros_like(x[:, :1])
    lo = torch.minimum(x.min(dim=1, keepdim=True).values, zeros)
    hi = torch.maximum(x.max(dim=1, keepdim=True).values, zeros)
    scale = torch.maximum(_f32(_f32(hi - lo) / 255.0), zeros + TINY)
    zero = torch.trunc(_f32(-_f32(lo / scale)) + 0.5)
    return _exact_codes(x, scale, zero), scale, zero


def exact(case, seed):
    s = prepare(case, seed)
    op = case["op"]
    if op == "tokens":
        codes, scale, zero = _exact_rows(s["x"])
        return {"values": scale * (codes - zero), "scale": scale[:, 0], "zero": None}
    if op == "linear":
        codes, scale, zero = _exact_rows(s["x"])
        w = (s["w"].double() - s["w_pairs"][:, 4].double()[:, None]) * _scale_of(s["w_pairs"]).double()[:, None]
        y = torch.einsum("mk,nk->mn", scale * (codes - zero), w)
        return y if s["bias"] is None else y + s["bias"].double()
    spans, block = _ragged(case), case["block"]
    table = s["table"].tolist()
    if op == "append":
        out = {}
        for name in ("k", "v"):
            codes, scales = s[name].double(), _scale_of(s[name + "_pairs"]).double().clone()
            begin = 0
            for i, (new, length) in enumerate(spans):
                x = s["new_" + name][begin:begin + new].double()
                begin += new
                p = length - new
                while p < length:
                    page, used = table[i][p // block], p % block
                    take = min(block - used, length - p)
                    part = x[p - (length - new):p - (length - new) + take].transpose(0, 1)   # [heads, take, head_dim]
                    need = _f32(part.abs().flatten(1).max(dim=1).values / 127.0)
                    floor = scales[page].clone() if used else torch.full_like(need, TINY)
                    scale = torch.maximum(floor, need)
                    if used:
                        grown = scale > scales[page]
                        held = _f32(scales[page][:, None, None] * (codes[page, :, :used] - 128.0))
                        codes[page, :, :used] = torch.where(grown[:, None, None], _exact_codes(held, scale[:, None, None], 128.0), codes[page, :, :used])
                    codes[page, :, used:used + take] = _exact_codes(part, scale[:, None, None], 128.0)
                    scales[page] = scale
                    p += take
            out[name] = scales[..., None, None] * (codes - 128.0)
            out[name + "_scale"] = scales
        return out
    group = case["q_heads"] // case["kv_heads"]
    rows, begin = [], 0
    for i, (new, length) in enumerate(spans):
        pages = torch.tensor(table[i][:-(-length // block)], device="cuda")
        q = s["q"][begin:begin + new].double()
        begin += new
        heads = []
        for h in range(case["kv_heads"]):
            k, v = ((_scale_of(s[n + "_pairs"])[pages, h].double()[:, None, None] * (s[n][pages, h].double() - 128.0)).reshape(-1, case["head_dim"])[:length] for n in ("k", "v"))
            logits = torch.einsum("tgd,kd->gtk", q[:, h * group:(h + 1) * group], k) * case["head_dim"] ** -0.5
            hidden = torch.ones(new, length, dtype=torch.bool, device="cuda").triu(length - new + 1)
            logits[:, hidden] = -math.inf
            heads.append(torch.einsum("gtk,kd->tgd", torch.softmax(logits, dim=2), v))
        rows.append(torch.cat(heads, dim=1))
    return torch.cat(rows)
