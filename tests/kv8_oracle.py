"""The 8-bit cache's operators in 64 bits, row by row and head by head, from their definitions."""
import math

import torch

LARGEST = 448.0


def e4m3(x):
    """Nearest e4m3 number, ties to even, +-448 beyond the range: steps of 2^(e - 3), of 2^-9 below 2^-6."""
    step = torch.exp2((torch.frexp(x.abs().clamp(max=LARGEST))[1].double() - 4).clamp(min=-9))
    return (torch.round(x / step) * step).clamp(-LARGEST, LARGEST)


def scale_for(top):
    e = -126
    while top > LARGEST * 2.0 ** e:
        e += 1
    return 2.0 ** e


def rotate(x, cos, sin):
    """``x [heads, D]``, ``cos, sin [D / 2]``."""
    a, b = x[:, :x.shape[1] // 2], x[:, x.shape[1] // 2:]
    return torch.cat([a * cos - b * sin, b * cos + a * sin], 1)


def append(rows, rope_pos, cos, sin, section, seq, pos, table, codes, scales, hq, hkv, d):
    """``rows [T, width]`` in 64 bits -> (rotated rows, values before rounding of the written places (NaN elsewhere),
    codes, scales, amax that decided each scale, one place's rows in order).  ``codes`` and ``scales`` are the old state."""
    codes, scales = codes.double().clone(), scales.double().clone()
    raw = torch.full_like(codes, math.nan)
    tops = torch.zeros_like(scales)
    rows = rows.double().clone()
    touched = {}
    for t in range(rows.shape[0]):
        x = rows[t].view(hq + 2 * hkv, d)
        if cos is not None:
            i = torch.arange(d // 2)
            p = rope_pos[t].expand(d // 2) if rope_pos.dim() == 1 else rope_pos[torch.where(
                i < section[0], 0, torch.where(i < section[0] + section[1], 1, 2)), t]
            x[:hq + hkv] = rotate(x[:hq + hkv], cos.double()[p.long(), i], sin.double()[p.long(), i])
        s, at = int(seq[t]), int(pos[t])
        if s < 0 or at < 0 or at // 64 >= table.shape[1] or s >= table.shape[0]:
            continue
        b = int(table[s, at // 64])
        if 0 <= b < codes.shape[0]:
            touched.setdefault(b, []).append((at % 64, x[hq:].view(2, hkv, d)))
    for b, new in touched.items():
        if any(o == 0 for o, _ in new):
            codes[b], scales[b] = 0, 0
        for j in range(2):
            for h in range(hkv):
                tops[b, j, h] = max(float(v[j, h][torch.isfinite(v[j, h])].abs().max()) if torch.isfinite(v[j, h]).any() else 0.0
                                    for _, v in new)
                old, need = float(scales[b, j, h]), scale_for(float(tops[b, j, h]))
                scale = max(old, need)
                codes[b, j, h] = e4m3(codes[b, j, h] * (old / scale))
                scales[b, j, h] = scale
                for o, v in new:
                    raw[b, j, h, o] = v[j, h]
                    codes[b, j, h, o] = e4m3(v[j, h] / scale)
    return rows, raw, codes, scales, tops


def attention(q, codes, scales, blocks, seen, hq, hkv, d, scale):
    """``q [rows, hq * d]``; row i sees the first ``seen[i]`` tokens of the blocks.  Returns (output, sum of weight * |value|)."""
    out, size = (torch.zeros(q.shape[0], hq, d, dtype=torch.float64) for _ in range(2))
    if not len(blocks):
        return out.view(len(q), hq * d), size.view(len(q), hq * d)
    x = codes[blocks].double() * scales[blocks].double()[..., None, None]
    for h in range(hq):
        g = h // (hq // hkv)
        k, v = x[:, 0, g].reshape(-1, d), x[:, 1, g].reshape(-1, d)
        for i, n in enumerate(seen):
            if n:
                w = torch.softmax(k[:n] @ q[i, h * d:(h + 1) * d].double() * scale, 0)
                out[i, h], size[i, h] = w @ v[:n], w @ v[:n].abs()
    return out.view(len(q), hq * d), size.view(len(q), hq * d)


def engine_by_hand(model, logits, ids, cuts, steps):
    """Greedy tokens and log-probabilities of one prompt, as a rollout engine with an 8-bit cache has to get them: the prompt in
    portions that end at ``cuts``, each behind the ones before, then token by token, on a cache of its own."""
    from siirl_b200.ops.attention import SeqInfo
    from siirl_b200.ops.kv_cache import Cache8
    cfg, dev = model.cfg, next(model.parameters()).device
    n = -(-(len(ids) + steps) // 64)
    cache = [Cache8.zeros(n + 1, cfg.num_kv_heads, cfg.head_dim, dev) for _ in range(cfg.num_layers)]
    table = torch.arange(n, 0, -1, dtype=torch.int32, device=dev)[None]
    a = 0
    for b in cuts:
        info, seq = SeqInfo([b - a], device=dev), torch.zeros(b - a, dtype=torch.int32, device=dev)
        at = {} if a == 0 else {"prefix_lens": [a], "prefill_slots": [0]}
        hidden = model.forward_cached(torch.tensor(ids[a:b], device=dev), info.positions + a, cache, table, seq, prefill_info=info, **at)
        a = b
    tokens, probs, one = [], [], torch.zeros(1, dtype=torch.int32, device=dev)
    for n in range(len(ids), len(ids) + steps):
        z = logits(hidden[-1:])[0].detach().double()
        tokens.append(int(z.argmax()))
        probs.append(float(torch.log_softmax(z, 0)[tokens[-1]]))
        hidden = model.forward_cached(torch.tensor(tokens[-1:], device=dev), one + n, cache, table, one, seq_lens=one + n + 1)
    return tokens, probs


def record_cuts(engine):
    """{number of the prompt: (from, to) of its portions} of the prefills to come."""
    cuts, prefill = {}, engine._prefill

    def recorded(seqs, chunks, starts=None, *args, **kw):
        for i, c in enumerate(chunks):
            a = starts[i] if starts is not None else 0
            cuts.setdefault(seqs[i].prompt_index, []).append((a, a + len(c)))
        return prefill(seqs, chunks, starts, *args, **kw)
    engine._prefill = recorded
    return cuts
