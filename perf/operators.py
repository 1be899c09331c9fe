"""A paged key / value cache held in 8 bits, as the rollout engine uses it: rows appended to it, single tokens and chunks of
prompts attending to it.

The cache of a layer is ``codes [blocks, 2, Hkv, 64, D]`` (e4m3; keys, then values) and ``scales [blocks, 2, Hkv]`` (fp32,
powers of two): a cached value is code times scale.  A sequence's tokens lie in the blocks that its row of ``table`` names.

* ``append``: the q and k heads of the new tokens' projection are rotated in place, k and v heads go to the cache.  The scale of
  a block and head is the smallest power of two that keeps all it has met within e4m3's range: where new rows raise it, the
  block's other rows are rounded to it; a row at offset 0 starts its block anew, with zeros in the rows that the call does not
  write.  ``slabs`` > 0: the projection comes as fp32 partial sums, which are added up with its bias on the way.
* ``decode``: one query row per sequence against its cached context; sequences of length 0 are idle slots and give zeros.
* ``prefix``: the rows of chunks of prompts, whose keys and values have been appended, against all tokens up to their own.

Head layouts (query heads, kv heads, width) are those of the presets ``qwen2.5-0.5b``, ``qwen2.5-7b``, ``qwen3-30b-a3b``,
and of decoders with 32 / 8 and 16 / 16 heads."""
import math

import torch

own = False
BLOCK, LARGEST = 64, 448.0  # tokens of a cache block, largest e4m3 number
HEADS = {"14/2x64": (14, 2, 64), "28/4x128": (28, 4, 128), "32/4x128": (32, 4, 128), "32/8x128": (32, 8, 128),
         "16/16x128": (16, 16, 128), "8/2x64": (8, 2, 64)}


def _append(heads, sequences, least, longest, fresh, slabs):
    """``sequences`` chunks of ``least`` to ``longest`` new rows; ``fresh``: at position 0, else behind an earlier context."""
    return {"op": "append", "heads": heads, "sequences": sequences, "least": least, "longest": longest, "fresh": fresh,
            "slabs": slabs}


def _decode(heads, sequences, least, longest, idle):
    return {"op": "decode", "heads": heads, "sequences": sequences, "least": least, "longest": longest, "idle": idle}


def _prefix(heads, sequences, least, longest, prefix):
    """Chunks of ``least`` to ``longest`` rows behind up to ``prefix`` cached tokens."""
    return {"op": "prefix", "heads": heads, "sequences": sequences, "least": least, "longest": longest, "prefix": prefix}


def listed():
    return [
        # a decoding step of the headline rollout: 32 prompts x 8 samples, one token each
        dict(_append("28/4x128", 256, 1, 1, False, 0), name="append-decode-256"),
        # a decoding step of a small policy whose projection was split over its contraction
        dict(_append("14/2x64", 61, 1, 1, False, 3), name="append-decode-split-61"),
        # a batch of whole prompts
        dict(_append("28/4x128", 24, 1, 701, True, 0), name="append-prompts-24"),
        # later turns of many long conversations
        dict(_append("32/8x128", 16, 1500, 2500, False, 0), name="append-turns-16"),
        # interactive use of a small policy: one sequence, nothing but latency
        dict(_decode("14/2x64", 1, 513, 513, 0), name="decode-1x513"),
        # the middle of a rollout: samples of all lengths, some slots idle
        dict(_decode("28/4x128", 64, 1, 2100, 5), name="decode-64x2100"),
        # a few long contexts
        dict(_decode("32/8x128", 8, 20001, 32768, 0), name="decode-8x32768"),
        # the end of the headline rollout
        dict(_decode("28/4x128", 256, 1300, 5120, 0), name="decode-256x5120"),
        # a short question behind a short prompt
        dict(_prefix("14/2x64", 1, 9, 9, 130), name="prefix-1x9"),
        # next turns of conversations whose earlier blocks the prefix cache holds
        dict(_prefix("28/4x128", 16, 17, 160, 2500), name="prefix-16x160"),
        # a chunk of a long prompt
        dict(_prefix("28/4x128", 1, 2048, 2048, 6144), name="prefix-1x2048"),
        # chunks of two very long prompts
        dict(_prefix("32/8x128", 2, 1900, 2148, 14000), name="prefix-2x2148"),
    ]


def _between(rng, lo, hi):
    """A whole number between ``lo`` and ``hi``, spread over its logarithm."""
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op, heads = rng.choice(["append", "decode", "prefix"]), rng.choice(sorted(HEADS))
    if op == "append":
        if rng.random() < 0.5:
            return _append(heads, _between(rng, 1, 256), 1, 1, False, rng.choice([0, 0, 1, 2, 5]))
        longest = _between(rng, 2, 2500)
        return _append(heads, _between(rng, 1, max(1, 32000 // longest) if longest > 125 else 256), rng.randint(1, longest),
                       longest, rng.random() < 0.5, 0)
    if op == "decode":
        hq, hkv, d = HEADS[heads]
        longest = _between(rng, 1, 32768)
        # at most 10^9 cached numbers
        sequences = _between(rng, 1, max(1, min(256, 900_000_000 // (2 * longest * hkv * d))))
        return _decode(heads, sequences, _between(rng, 1, longest), longest, rng.randint(0, sequences // 4))
    longest = _between(rng, 1, 2048)
    prefix = _between(rng, 1, 14000)
    sequences = _between(rng, 1, max(1, min(32, 50_000_000 // (longest * (longest + prefix)))))
    return _prefix(heads, sequences, rng.randint(1, longest), longest, prefix)


# ---- sizes --------------------------------------------------------------------------------------
def _spread(n, lo, hi, shift):
    """``n`` unequal whole numbers in ``[lo, hi]``; part of the case, not of its random values."""
    return [lo + int((hi - lo + 1) * (((i + 1) * 0.6180339887 + shift) % 1.0)) for i in range(n)]


def _lengths(case):
    """(new rows, earlier tokens) of every sequence."""
    n = case["sequences"]
    if case["op"] == "decode":
        lens = _spread(n, case["least"], case["longest"], 0.3)
        if n == 1:
            lens = [case["longest"]]
        for i in range(case["idle"]):
            lens[(i * 7 + 3) % n] = 0
        return [1] * n, lens
    new = _spread(n, case["least"], case["longest"], 0.1)
    if case["op"] == "prefix":
        return new, _spread(n, case["prefix"] - case["prefix"] // 4, case["prefix"], 0.5)
    return new, [0] * n if case["fresh"] else _spread(n, 1, 1500, 0.7)


def work(case):
    hq, hkv, d = HEADS[case["heads"]]
    new, old = _lengths(case)
    rows, width = sum(new), (hq + 2 * hkv) * d
    if case["op"] == "append":
        # the projection once, the rotated heads (of partial sums: all heads) and the cached rows once
        if case["slabs"]:
            moved = rows * width * (4 * case["slabs"] + 2)
        else:
            moved = rows * (2 * width + 2 * (hq + hkv) * d)
        return {"bytes": moved + rows * (2 * hkv * d + 4 * d), "flops": 6 * rows * (hq + hkv) * d}
    if case["op"] == "decode":
        seen, pairs = sum(old), sum(old)
    else:
        seen, pairs = rows + sum(old), sum(n * p + n * (n + 1) // 2 for n, p in zip(new, old))
    return {"bytes": seen * 2 * hkv * d + 2 * rows * 2 * hq * d, "flops": 4 * hq * d * pairs}


# ---- inputs -------------------------------------------------------------------------------------
def _quantized(x):
    """Codes and scales of whole blocks ``x [..., 64, D]``."""
    top, exp = torch.frexp(x.abs().amax((-2, -1)))
    exp = torch.where(top == 0, torch.full_like(exp, -126), exp - 9 + (top > 0.875))
    scales = torch.ldexp(torch.ones_like(top), exp)
    return (x / scales[..., None, None]).to(torch.float8_e4m3fn), scales


def prepare(case, seed):
    hq, hkv, d = HEADS[case["heads"]]
    new, old = _lengths(case)
    gen = torch.Generator(device="cuda").manual_seed(seed)
    n, rows, dev = len(new), sum(new), "cuda"
    held = [o if case["op"] == "decode" else a + o for a, o in zip(new, old)]
    need = [-(-t // BLOCK) for t in held]
    most = max(max(need), 1) + 3  # tables are as wide as the longest sequence that the engine admits
    blocks = sum(need) + 5
    order = torch.randperm(blocks, generator=gen, device=dev).tolist()
    table = torch.full((n, most), -1, dtype=torch.int32)
    at = 0
    for i, k in enumerate(need):
        table[i, :k] = torch.tensor(order[at:at + k], dtype=torch.int32)
        at += k
    # keys have channels of unlike size, values blocks of unlike size
    codes = torch.empty(blocks, 2, hkv, BLOCK, d, dtype=torch.float8_e4m3fn, device=dev)
    scales = torch.empty(blocks, 2, hkv, device=dev)
    gain = torch.exp(0.4 * torch.randn(hkv, 1, d, generator=gen, device=dev))
    step = max(1, 100_000_000 // (2 * hkv * BLOCK * d))
    for b in range(0, blocks, step):
        x = torch.randn(min(step, blocks - b), 2, hkv, BLOCK, d, generator=gen, device=dev)
        x[:, 0] *= gain
        x[:, 1] *= torch.exp(0.5 * torch.randn(len(x), hkv, 1, 1, generator=gen, device=dev))
        codes[b:b + step], scales[b:b + step] = _quantized(x)
    s = {"heads": (hq, hkv, d), "op": case["op"], "codes": codes, "scales": scales, "table": table.to(dev)}
    width = (hq + 2 * hkv) * d
    if case["op"] == "append":
        s["seq"] = torch.repeat_interleave(torch.arange(n, dtype=torch.int32), torch.tensor(new)).to(dev)
        s["pos"] = torch.cat([torch.arange(o, o + a, dtype=torch.int32) for a, o in zip(new, old)]).to(dev)
        ang = torch.arange(max(held), dtype=torch.float64)[:, None] * 1e6 ** (-torch.arange(0, d, 2, dtype=torch.float64) / d)
        s["cos"], s["sin"] = ang.cos().float().to(dev), ang.sin().float().to(dev)
        s["bias"] = None
        if case["slabs"]:
            s["bias"] = (0.5 * torch.randn(width, generator=gen, device=dev)).bfloat16()
            s["qkv"] = torch.randn(case["slabs"], rows, width, generator=gen, device=dev) / math.sqrt(case["slabs"])
        else:
            s["qkv"] = torch.randn(rows, width, generator=gen, device=dev).bfloat16()
        return s
    s["qkv"] = torch.randn(n if case["op"] == "decode" else rows, width, generator=gen, device=dev).bfloat16()
    if case["op"] == "decode":
        s["lens"] = torch.tensor(old, dtype=torch.int32, device=dev)
    else:
        s["new"], s["old"], s["slots"] = new, old, list(range(n))
    return s


# ---- the operators ------------------------------------------------------------------------------
def run(s):
    hq, hkv, d = s["heads"]
    if own:
        from siirl_b200.ops import kv_cache as kvc
        cache = kvc.Cache8(s["codes"], s["scales"])
        if s["op"] == "append":
            qkv = kvc.rope_kv_append(s["qkv"], s["pos"], s["cos"], s["sin"], None, s["seq"], s["pos"], s["table"], cache, hq,
                                     hkv, d, s["bias"])
            return {"qkv": qkv, "codes": s["codes"], "scales": s["scales"]}
        if s["op"] == "decode":
            return kvc.decode_attention(s["qkv"], cache, s["lens"], s["table"], hq, hkv, d)
        return kvc.prefill_attention_with_prefix(s["qkv"], s["new"], s["old"], s["slots"], cache, s["table"], hq, hkv, d)
    if s["op"] == "append":
        return _plain_append(s)
    return _plain_decode(s) if s["op"] == "decode" else _plain_prefix(s)


def _plain_append(s):
    hq, hkv, d = s["heads"]
    rows = s["pos"].numel()
    x = s["qkv"].float() if s["bias"] is None else s["qkv"].sum(0) + s["bias"].float()
    x = x.view(rows, hq + 2 * hkv, d)
    cos, sin = s["cos"][s["pos"].long()][:, None], s["sin"][s["pos"].long()][:, None]
    a, b = x[:, :hq + hkv, :d // 2], x[:, :hq + hkv, d // 2:]
    turned = torch.cat([a * cos - b * sin, b * cos + a * sin], -1)
    kv = torch.stack([turned[:, hq:], x[:, hq + hkv:]], 1)  # [rows, 2, Hkv, D]
    if s["bias"] is None:
        qkv = s["qkv"]
        qkv[:, :(hq + hkv) * d] = turned.view(rows, -1).to(qkv.dtype)
    else:
        qkv = torch.cat([turned, x[:, hq + hkv:]], 1).view(rows, -1).bfloat16()
    place, off = s["table"][s["seq"].long(), (s["pos"] // BLOCK).long()].long(), (s["pos"] % BLOCK).long()
    blocks, which = torch.unique(place, return_inverse=True)
    top = torch.zeros(len(blocks), 2, hkv, device=kv.device).index_reduce_(0, which, kv.abs().amax(-1), "amax")
    half, exp = torch.frexp(top)
    need = torch.ldexp(torch.ones_like(top), torch.where(half == 0, torch.full_like(exp, -126), exp - 9 + (half > 0.875)))
    anew = torch.zeros(len(blocks), dtype=torch.bool, device=kv.device)
    anew[which[off == 0]] = True
    kept = torch.where(anew[:, None, None], torch.zeros_like(top), s["scales"][blocks])
    scale = torch.maximum(kept, need)
    codes = s["codes"][blocks].float() * (kept / scale)[..., None, None]
    codes[which, :, :, off] = (kv / scale[which][..., None]).clamp(-LARGEST, LARGEST)
    s["codes"][blocks], s["scales"][blocks] = codes.to(torch.float8_e4m3fn), scale
    return {"qkv": qkv, "codes": s["codes"], "scales": s["scales"]}


def _cached(s, slots, most):
    """Keys and values ``[sequences, Hkv, tokens, D]`` in 32 bits."""
    hq, hkv, d = s["heads"]
    places = s["table"][slots][:, :-(-most // BLOCK)].clamp(min=0).long()
    x = s["codes"][places].float() * s["scales"][places][..., None, None]  # [n, blocks, 2, Hkv, 64, D]
    return x.permute(2, 0, 3, 1, 4, 5).reshape(2, len(places), hkv, -1, d)


def _soft(z, mask):
    z = z.masked_fill_(~mask, -math.inf)
    z = z.sub_(z.amax(-1, keepdim=True).clamp(min=-3e38)).exp_()
    return z.div_(z.sum(-1, keepdim=True).clamp(min=1e-30))


def _plain_decode(s):
    hq, hkv, d = s["heads"]
    n = len(s["lens"])
    k, v = _cached(s, slice(None), s["table"].shape[1] * BLOCK)
    q = s["qkv"][:, :hq * d].float().view(n, hkv, hq // hkv, d)
    mask = torch.arange(k.shape[2], device=k.device) < s["lens"][:, None, None, None]
    p = _soft(q @ k.transpose(-1, -2) / math.sqrt(d), mask)
    return (p @ v).view(n, hq * d).to(s["qkv"].dtype)


def _plain_prefix(s):
    hq, hkv, d = s["heads"]
    n, most = len(s["new"]), max(s["new"])
    dev = s["qkv"].device
    new, old = torch.tensor(s["new"], device=dev), torch.tensor(s["old"], device=dev)
    k, v = _cached(s, s["slots"], max(a + b for a, b in zip(s["new"], s["old"])))
    row = torch.arange(most, device=dev)
    real = row < new[:, None]  # [n, most]
    q = torch.zeros(n, most, hq, d, device=dev)
    q[real] = s["qkv"][:, :hq * d].float().view(-1, hq, d)
    q = q.transpose(1, 2).reshape(n, hkv, hq // hkv * most, d)
    seen = torch.arange(k.shape[2], device=dev) <= (old[:, None] + row)[..., None]  # [n, most, tokens]
    z = (q @ k.transpose(-1, -2)).mul_(1 / math.sqrt(d)).view(n, hq, most, -1)
    p = _soft(z, seen[:, None])
    o = (p.view(n, hkv, hq // hkv * most, -1) @ v).view(n, hq, most, d).transpose(1, 2)
    return o[real].reshape(-1, hq * d).to(s["qkv"].dtype)


# ---- the definition in 64 bits ------------------------------------------------------------------
def exact(case, seed):
    s = prepare(case, seed)
    hq, hkv, d = s["heads"]
    if case["op"] == "append":
        return _exact_append(s)
    out = torch.zeros(s["qkv"].shape[0], hq, d, dtype=torch.float64, device="cuda")
    at = 0
    for i in range(case["sequences"]):
        a = 1 if case["op"] == "decode" else s["new"][i]
        total = int(s["lens"][i]) if case["op"] == "decode" else a + s["old"][i]
        if total:
            places = s["table"][i, :-(-total // BLOCK)].long()
            x = s["codes"][places].double() * s["scales"][places].double()[..., None, None]
            for h in range(hq):
                k, v = (x[:, j, h // (hq // hkv)].reshape(-1, d)[:total] for j in range(2))
                z = torch.einsum("ad,td->at", s["qkv"][at:at + a, h * d:(h + 1) * d].double(), k) * d ** -0.5
                z += torch.full_like(z, -math.inf).triu_(total - a + 1)
                out[at:at + a, h] = torch.einsum("at,td->ad", torch.softmax(z, -1), v)
        at += a
    return out.view(-1, hq * d)


def _exact_append(s):
    hq, hkv, d = s["heads"]
    x = s["qkv"].double()
    if s["bias"] is not None:
        x = x.sum(0) + s["bias"].double()
    rows = x.shape[0]
    x = x.view(rows, hq + 2 * hkv, 2, d // 2)
    turn = torch.complex(s["cos"].double(), s["sin"].double())[s["pos"].long()][:, None]
    z = torch.complex(x[:, :hq + hkv, 0], x[:, :hq + hkv, 1]) * turn
    x = torch.cat([torch.stack([z.real, z.imag], 2), x[:, hq + hkv:]], 1).view(rows, hq + 2 * hkv, d)
    values = s["codes"].double() * s["scales"].double()[..., None, None]
    scales = s["scales"].double()
    seq, pos, table = s["seq"].tolist(), s["pos"].tolist(), s["table"].tolist()
    first = 0
    while first < rows:  # the rows of one block
        end = first + 1
        while end < rows and seq[end] == seq[first] and pos[end] // BLOCK == pos[first] // BLOCK:
            end += 1
        blk, off = table[seq[first]][pos[first] // BLOCK], pos[first] % BLOCK
        if off == 0:
            values[blk], scales[blk] = 0, 0
        kv = x[first:end, hq:].view(end - first, 2, hkv, d).permute(1, 2, 0, 3)
        need = torch.exp2(torch.ceil(torch.log2(kv.abs().amax((-2, -1)) / LARGEST)).clamp(min=-126))
        scales[blk] = torch.maximum(scales[blk], need)
        values[blk, :, :, off:off + end - first] = kv
        first = end
    # to the nearest e4m3 number, ties to even: steps of 2^(e-3), and of 2^-9 below 2^-6
    codes = values / scales[..., None, None]
    step = torch.exp2((torch.frexp(codes)[1].double() - 4).clamp(min=-9))
    return {"qkv": x.view(rows, -1), "codes": torch.round(codes / step) * step, "scales": scales}
