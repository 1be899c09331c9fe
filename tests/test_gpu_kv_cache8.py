"""Paged cache in 8 bits: the kernels against the definitions in 64 bits."""
import math

import pytest
import torch

import kv8_oracle as oracle
from siirl_b200.ops import kv_cache as kvc
from siirl_b200.ops import lib
from siirl_b200.ops import reference as ref
from siirl_b200.ops.kv_cache import Cache8

pytestmark = pytest.mark.gpu
DEV = "cuda"
BF16 = 2.0 ** -8        # half a step of bf16, relative to the value


def _random_cache(nb, hkv, d, spread=1.0):
    """Codes over their whole range, scales of unlike blocks."""
    codes = (torch.randn(nb, 2, hkv, 64, d) * 100).clamp(-448, 448).to(torch.float8_e4m3fn)
    scales = 2.0 ** torch.round(-7 + spread * torch.randn(nb, 2, hkv))
    return Cache8(codes, scales)


def _gpu(cache):
    return Cache8(cache.codes.to(DEV), cache.scales.to(DEV))


def _check_append(cache, rows, pos, section, seq, at, table, hq, hkv, d, slabs=0, bias=None, rope=True):
    """One call on the GPU against the definition.  Bounds: a rotated value is a * c - b * s in 32 bits (three roundings of
    2^-24 of |a| + |b|), sums of S partial sums add S + 1 more; bf16 rows half a step, codes half a step of e4m3."""
    cos, sin = ref.rope_tables(d, 1600, 1e4)
    if rope is False:
        cos = sin = None
    g = _gpu(cache)
    t = lambda x: None if x is None else x.to(DEV)  # noqa: E731
    full = rows.double() if not slabs else rows.double().sum(0) + (0 if bias is None else bias.double())
    dev_rows = t(rows)
    if rope:
        out = kvc.rope_kv_append(dev_rows, t(pos), t(cos), t(sin), section, t(seq), t(at), t(table), g, hq, hkv, d, t(bias))
    else:
        kvc.kv_append(dev_rows, t(seq), t(at), t(table), g, hq, hkv, d)
        out = dev_rows
    want, raw, codes, scales, tops = oracle.append(full, pos, cos, sin, section, seq, at, table, *cache, hq, hkv, d)
    out = out.cpu().double()
    width = (hq + hkv) * d
    reach = (rows.double().abs().sum(0) + (0 if bias is None else bias.double().abs())) if slabs else full.abs()
    r = reach.view(len(reach), hq + 2 * hkv, 2, d // 2)
    reach = (r + r.flip(2)).view_as(reach)
    fine = torch.isfinite(want)
    err = (3 + slabs + 1) * 2.0 ** -23 * reach if rope else torch.zeros_like(reach)     # without rotation: exact
    assert bool(((out - want).abs() <= BF16 * want.abs() + err)[fine].all())
    if not slabs:
        assert torch.equal(out[:, width:][fine[:, width:]], full[:, width:][fine[:, width:]])
    got_s = g.scales.cpu().double()
    # the kernel's largest value may be off by its rounding: where the border lies within that, either scale is right
    edge = torch.zeros_like(scales, dtype=torch.bool)
    for i in (tops > 0).nonzero().tolist():
        top = float(tops[tuple(i)])
        edge[tuple(i)] = abs(math.remainder(math.log2(top / 448.0), 1.0)) < 2.0 ** -18
    assert torch.equal(got_s[~edge], scales[~edge])
    kept = torch.isnan(raw) & torch.isfinite(codes)
    kept &= (got_s == scales)[..., None, None]
    got = g.codes.cpu().double()
    assert torch.equal(got[kept], codes[kept])
    new = torch.isfinite(raw)
    s = got_s[..., None, None].expand_as(raw)
    bound = torch.maximum(2.0 ** -4 * raw.abs(), 2.0 ** -10 * s) + 2.0 ** -19 * (raw.abs().nan_to_num().amax(-1, keepdim=True) + s * 2.0 ** -9)
    assert bool(((got * s - raw).abs() <= bound)[new].all())
    inf = torch.isinf(raw)
    assert bool((got[inf] == 448 * torch.sign(raw[inf])).all())
    lib.check_status()
    return g, out


@pytest.mark.parametrize("hq,hkv,d", [(28, 4, 128), (14, 2, 64), (3, 3, 128), (2, 1, 64)])
@pytest.mark.parametrize("rows", [1, 7, 61])
def test_append_single_rows(hq, hkv, d, rows):
    """A decoding step: every sequence at its own place, first, inner and last rows of blocks, idle slots."""
    nb, most = 2 * rows + 3, 3
    cache = _random_cache(nb, hkv, d)
    order = torch.randperm(nb).to(torch.int32)
    table = torch.full((rows, most), -1, dtype=torch.int32)
    table[:, :2] = order[:2 * rows].view(rows, 2)
    at = torch.tensor([[0, 63, 64, 127, 1, 100, 30][i % 7] for i in range(rows)], dtype=torch.int32)
    seq = torch.arange(rows, dtype=torch.int32)
    if rows > 7:
        seq[9], at[12], at[20] = -1, -1, 128     # idle, idle, no block
    x = torch.randn(rows, (hq + 2 * hkv) * d) * torch.exp(2 * torch.randn(rows, 1))
    _check_append(cache, x.bfloat16(), at.clamp(min=0) + 5, None, seq, at, table, hq, hkv, d)


@pytest.mark.parametrize("hq,hkv,d", [(6, 2, 128), (6, 1, 64)])
def test_append_partial_sums_of_chunks(hq, hkv, d):
    lens, width = (150, 70, 1), (hq + 2 * hkv) * d
    cache = _random_cache(8, hkv, d)
    table = torch.tensor([[0, 1, 2, 3], [4, 5, -1, -1], [6, 7, -1, -1]], dtype=torch.int32)
    seq = torch.repeat_interleave(torch.arange(3, dtype=torch.int32), torch.tensor(lens))
    at = torch.cat([torch.arange(s, s + n, dtype=torch.int32) for n, s in zip(lens, (40, 0, 64))])
    _check_append(cache, torch.randn(2, sum(lens), width), at, None, seq, at, table, hq, hkv, d, 2, torch.randn(width).bfloat16())


@pytest.mark.parametrize("hq,hkv,d,slabs,bias", [(28, 4, 128, 3, True), (14, 2, 64, 1, False), (2, 2, 64, 5, True)])
def test_append_partial_sums(hq, hkv, d, slabs, bias):
    rows, width = 13, (hq + 2 * hkv) * d
    cache = _random_cache(rows, hkv, d)
    table = torch.arange(rows, dtype=torch.int32)[:, None].contiguous()
    at = torch.randint(0, 64, (rows,), dtype=torch.int32)
    b = torch.randn(width).bfloat16() if bias else None
    _check_append(cache, torch.randn(slabs, rows, width), at, None, torch.arange(rows, dtype=torch.int32), at, table, hq, hkv, d,
                  slabs, b)


@pytest.mark.parametrize("hq,hkv,d", [(28, 4, 128), (14, 2, 64), (1, 1, 128)])
@pytest.mark.parametrize("lens,starts", [((1, 2, 63, 64, 65, 200), (0, 0, 0, 0, 0, 0)), ((5, 130, 64, 1), (61, 30, 64, 63)),
                                         ((300,), (1,))])
def test_append_chunks(hq, hkv, d, lens, starts):
    """Whole prompts and later chunks: blocks that begin, go on and end in the call; rows with positions of three axes."""
    need = [(s + n + 63) // 64 for n, s in zip(lens, starts)]
    cache = _random_cache(sum(need) + 2, hkv, d, 3.0)
    table = torch.full((len(lens), max(need) + 1), -1, dtype=torch.int32)
    order, a = torch.randperm(sum(need)).to(torch.int32), 0
    for i, k in enumerate(need):
        table[i, :k] = order[a:a + k]
        a += k
    seq = torch.repeat_interleave(torch.arange(len(lens), dtype=torch.int32), torch.tensor(lens))
    at = torch.cat([torch.arange(s, s + n, dtype=torch.int32) for n, s in zip(lens, starts)])
    x = torch.randn(len(seq), (hq + 2 * hkv) * d) * torch.exp(torch.randn(len(seq), 1))
    _check_append(cache, x.bfloat16(), at, None, seq, at, table, hq, hkv, d)
    pos = torch.stack([at, at // 2, at // 3 + 7])
    _check_append(cache, x.bfloat16(), pos, (d // 8, d // 4, d // 8), seq, at, table, hq, hkv, d)
    _check_append(cache, x.bfloat16(), pos, None, seq, at, table, hq, hkv, d, rope=False)


@pytest.mark.parametrize("hq,hkv,d", [(5, 1, 128), (6, 2, 64)])
def test_append_long_batches(hq, hkv, d):
    """More rows than the ranges of small batches, runs of every kind in one range, idle rows among them, runs of one place."""
    lens, starts = [900, 1, 1, 7, 9, 64, 8, 1100, 70, 3], [5, 63, 0, 60, 0, 64, 10, 0, 130, 126]
    test_append_chunks(hq, hkv, d, lens, starts)
    n, nb = 2500, 80
    cache = _random_cache(nb, hkv, d)
    table = torch.randperm(nb).to(torch.int32).view(8, 10)
    seq, at = torch.full((n,), -1, dtype=torch.int32), torch.zeros(n, dtype=torch.int32)
    place = 0
    for i, (b, rows) in enumerate([(0, 1), (1, 100), (2, 8), (3, 65), (4, 64), (5, 9), (6, 7), (7, 200), (8, 70)] * 4):
        j = b + 9 * (i // 9)
        seq[place + 2:place + 2 + rows] = j // 10
        at[place + 2:place + 2 + rows] = j % 10 * 64 + torch.randint(0, 64, (rows,))      # places named twice
        place += rows + 2
    assert place < n
    x = torch.randn(n, (hq + 2 * hkv) * d).bfloat16()
    _check_append(cache, x, at, None, seq, at, table, hq, hkv, d)


def test_append_odd_values_and_places_named_twice():
    hq, hkv, d = 4, 2, 128
    cache = _random_cache(4, hkv, d)
    table = torch.tensor([[2, 0], [3, 1]], dtype=torch.int32)
    seq = torch.tensor([0, 0, 0, 0, 1, 1], dtype=torch.int32)
    at = torch.tensor([5, 6, 5, 70, 0, 9], dtype=torch.int32)
    x = torch.randn(6, (hq + 2 * hkv) * d)
    x[1, hq * d + 3], x[1, hq * d + 9], x[4, -1] = math.inf, -math.inf, math.nan
    x[3, (hq + hkv) * d:] = 0
    x[5, hq * d:] *= 1e30
    x = x.bfloat16()
    _check_append(cache, x, at, None, seq, at, table, hq, hkv, d, rope=False)


def test_append_takes_rows_of_a_wider_buffer():
    hq, hkv, d = 4, 2, 64
    cache, table = _gpu(_random_cache(3, hkv, d)), torch.zeros(1, 1, dtype=torch.int32, device=DEV)
    cos, sin = (x.to(DEV) for x in ref.rope_tables(d, 64, 1e4))
    wide = torch.randn(9, (hq + 2 * hkv) * d + 22, device=DEV).bfloat16()
    rows, at = wide[:, 8:8 + (hq + 2 * hkv) * d], torch.arange(20, 29, dtype=torch.int32, device=DEV)
    seq = torch.zeros(9, dtype=torch.int32, device=DEV)
    other = Cache8(cache.codes.clone(), cache.scales.clone())
    want = kvc.rope_kv_append(rows.contiguous(), at, cos, sin, None, seq, at, table, other, hq, hkv, d)
    edges = wide[:, :8].clone(), wide[:, 8 + rows.shape[1]:].clone()
    got = kvc.rope_kv_append(rows, at, cos, sin, None, seq, at, table, cache, hq, hkv, d)
    assert torch.equal(got, want) and torch.equal(cache.codes.view(torch.uint8), other.codes.view(torch.uint8))
    assert torch.equal(wide[:, :8], edges[0]) and torch.equal(wide[:, 8 + rows.shape[1]:], edges[1])


def _decode(lens, hq, hkv, d, max_blocks, spread=1.0, q_scale=1.0, stride=0):
    need = [(n + 63) // 64 for n in lens]
    cache = _random_cache(sum(need) + 3, hkv, d, spread)
    table = torch.full((len(lens), max_blocks), -1, dtype=torch.int32)
    order, a = torch.randperm(sum(need) + 3).to(torch.int32), 0
    for i, k in enumerate(need):
        table[i, :k] = order[a:a + k]
        a += k
    q = (q_scale * torch.randn(len(lens), (hq + 2 * hkv) * d + stride)).bfloat16()
    return cache, table, q, torch.tensor(lens, dtype=torch.int32)


def _check_decode(cache, table, q, lens, hq, hkv, d, scale=None):
    """Bounds: the output is rounded to bf16.  A weight of 2^e to 2^(e + 1) is kept as three e5m2 terms: the first is off by at most
    2^(e - 3), so that the second is below 2^(e - 3) and off by at most 2^(e - 7), and the third, likewise, by 2^(e - 11): 2^-11 of
    the weight, or 2^-36 of the largest one.  Scores carry 2^-22 sum |q k| and 2^-20 of themselves; these and sums of 32 bits
    over n tokens stay below 2^-11 together."""
    g = _gpu(cache)
    out = kvc.decode_attention(q.to(DEV), g, lens.to(DEV), table.to(DEV), hq, hkv, d, scale)
    lib.check_status()
    again = kvc.decode_attention(q.to(DEV), g, lens.to(DEV), table.to(DEV), hq, hkv, d, scale)
    assert torch.equal(out, again)
    for b, n in enumerate(lens.tolist()):
        want, size = oracle.attention(q[b:b + 1, :hq * d], *cache, table[b, :-(-n // 64)].long(), [n], hq, hkv, d,
                                      d ** -0.5 if scale is None else scale)
        x = cache.dequantize(table[b, :-(-n // 64)].long(), torch.float64)[:, 1].transpose(0, 1).reshape(hkv, -1, d)[:, :n]
        least = 2.0 ** -36 * x.abs().sum(1).repeat_interleave(hq // hkv, 0).reshape(-1)
        err = (out[b].cpu().double() - want[0]).abs()
        assert bool((err <= least + BF16 * want[0].abs() + 2.0 ** -10 * size[0]).all()), (b, n, float((err / (size[0] + 1e-300)).max()))


HEADS = [(28, 4, 128), (14, 2, 64), (4, 4, 128), (32, 1, 128), (9, 1, 64), (24, 2, 128)]


@pytest.mark.parametrize("hq,hkv,d", HEADS)
@pytest.mark.parametrize("lens,width", [((1,), 1), ((64, 0, 65, 127, 128, 129), 4), ((2, 1000, 0, 513), 20), ((0, 0), 2)])
def test_decode_attention(hq, hkv, d, lens, width):
    _check_decode(*_decode(lens, hq, hkv, d, width), hq, hkv, d)


@pytest.mark.parametrize("hq,hkv,d", [(28, 4, 128), (14, 2, 64), (32, 2, 128)])
def test_decode_attention_of_many_and_long_sequences(hq, hkv, d):
    _check_decode(*_decode([3000 - 41 * i if i % 5 else 0 for i in range(70)], hq, hkv, d, 50), hq, hkv, d)
    _check_decode(*_decode([9001], hq, hkv, d, 150), hq, hkv, d)


@pytest.mark.parametrize("hq,hkv,d", [(28, 4, 128), (14, 2, 64), (32, 2, 128)])
def test_decode_attention_of_sharp_scores_and_unlike_scales(hq, hkv, d):
    """Scores whose maximum moves from block to block, scales 2^12 apart, a scale given by the caller; values of zero."""
    _check_decode(*_decode([700, 64, 1], hq, hkv, d, 20, 4.0, 8.0), hq, hkv, d)
    _check_decode(*_decode([333, 90], hq, hkv, d, 20, 1.0, 0.3), hq, hkv, d, 1.0)
    cache, table, q, lens = _decode([400, 130], hq, hkv, d, 8)
    cache.codes.view(torch.uint8)[table[0, 3].long(), 1] = 0
    cache.scales[table[0, 3].long(), 1] = 2.0 ** -126
    cache.scales[table[1, 0].long(), 0] = 2.0 ** -126
    _check_decode(cache, table, q, lens, hq, hkv, d)


@pytest.mark.parametrize("hq,hkv,d", [(28, 4, 128), (14, 2, 64)])
def test_decode_attention_of_many_small_weights_beside_a_large_one(hq, hkv, d):
    """A first token that takes nearly all weight and has values near zero: the result is what thousands of tokens add, each with
    less than a millionth of the largest weight."""
    n = 6000
    cache, table, q, lens = _decode([n], hq, hkv, d, 100)
    cache.codes[:, 0] = (torch.randn(len(cache.codes), hkv, 64, d) * 30).to(torch.float8_e4m3fn)
    cache.scales[:, 0] = 2.0 ** -9
    q[0, :hq * d] = (0.1 * torch.randn(hq * d)).bfloat16()
    sink = table[0, 0].long()
    for h in range(hkv):
        mean = q[0, :hq * d].float().view(hkv, hq // hkv, d)[h].mean(0)
        cache.codes[sink, 0, h, 0] = (440 * torch.sign(mean)).to(torch.float8_e4m3fn)
        cache.scales[sink, 0, h] = 2.0 ** -3
        cache.codes[sink, 0, h, 1:] = 0
    cache.codes[sink, 1, :, 0] = 0
    want, _ = oracle.attention(q[:, :hq * d], *cache, table[0, :-(-n // 64)].long(), [n], hq, hkv, d, d ** -0.5)
    x = cache.dequantize(table[0, :-(-n // 64)].long())
    lead = torch.einsum("hrd,hd->hr", q[0, :hq * d].float().view(hkv, hq // hkv, d), x[0, 0, :, 0]) * d ** -0.5
    assert float(lead.max()) > 14       # 2^-20 of the largest weight and less for the others
    _check_decode(cache, table, q, lens, hq, hkv, d)
    assert float(want.abs().max()) > 0


@pytest.mark.parametrize("hq,hkv,d", [(28, 4, 128), (14, 2, 64), (32, 2, 128)])
def test_decode_attention_ignores_what_it_does_not_see(hq, hkv, d):
    """NaN codes behind the last token, blocks of no sequence, idle slots with tables of anything."""
    lens = [70, 0, 129, 1, 63]
    cache, table, q, n = _decode(lens, hq, hkv, d, 4)
    clean = kvc.decode_attention(q.to(DEV), _gpu(cache), n.to(DEV), table.to(DEV), hq, hkv, d)
    codes = cache.codes.view(torch.uint8)
    for b, k in enumerate(lens):
        if k % 64:
            codes[table[b, k // 64].long(), :, :, k % 64:] = 0x7f
    used = torch.zeros(len(codes), dtype=torch.bool)
    used[table[table >= 0].long()] = True
    codes[~used] = 0xff
    cache.scales[~used] = math.nan
    table[1] = torch.tensor([10 ** 6, -7, 2 ** 31 - 1, 0])
    got = kvc.decode_attention(q.to(DEV), _gpu(cache), n.to(DEV), table.to(DEV), hq, hkv, d)
    assert torch.equal(got, clean)


def test_decode_attention_of_strided_rows_on_another_stream_and_in_a_graph():
    hq, hkv, d = 28, 4, 128
    cache, table, q, n = _decode([300, 65, 0, 1500], hq, hkv, d, 30, stride=24)
    g, q, n, table = _gpu(cache), q.to(DEV), n.to(DEV), table.to(DEV)
    want = kvc.decode_attention(q.contiguous(), g, n, table, hq, hkv, d)
    out = torch.full((4, hq * d), 7.0, device=DEV, dtype=torch.bfloat16)
    assert kvc.decode_attention(q, g, n, table, hq, hkv, d, out=out) is out and torch.equal(out, want)
    odd = torch.cat([q[:, :2], q], 1)[:, 2:]        # rows that start 4 bytes behind a boundary
    assert torch.equal(kvc.decode_attention(odd, g, n, table, hq, hkv, d), want)
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        other = kvc.decode_attention(q, g, n, table, hq, hkv, d)
    torch.cuda.current_stream().wait_stream(s)
    assert torch.equal(other, want)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        held = kvc.decode_attention(q, g, n, table, hq, hkv, d)
    n.copy_(torch.tensor([1, 64, 500, 0]))
    graph.replay()
    assert torch.equal(held[[0, 1, 3]], kvc.decode_attention(q, g, n, table, hq, hkv, d)[[0, 1, 3]])
    lib.check_status()


def test_decode_attention_in_graphs_that_take_turns():
    """Two graphs of two calls each and calls outside of them, replayed in any order; a larger call behind a smaller one."""
    hq, hkv, d = 28, 4, 128
    cache, table, q, n = _decode([2000, 65, 900, 1500], hq, hkv, d, 40)
    g, q, n, table = _gpu(cache), q.to(DEV), n.to(DEV), table.to(DEV)

    def call(k):
        return kvc.decode_attention(q[:k], g, n[:k], table[:k], hq, hkv, d)
    want = {k: call(k).clone() for k in (1, 2, 4)}
    graphs = []
    for _ in range(2):
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            held = [call(1), call(4)]
        graphs.append((graph, held))
    for i in (0, 1, 1, 0):
        for t in graphs[i][1]:
            t.zero_()
        graphs[i][0].replay()
        assert torch.equal(call(2), want[2])
        assert torch.equal(graphs[i][1][0], want[1]) and torch.equal(graphs[i][1][1], want[4])
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        others = [call(4) for _ in range(5)]
    here = [call(4) for _ in range(5)]
    torch.cuda.current_stream().wait_stream(s)
    assert all(torch.equal(x, want[4]) for x in others + here)
    lib.check_status()


def _check_prefix(new, old, hq, hkv, d, spread=1.0, q_scale=1.0):
    """Bounds: weights and output are rounded to 16 bits; see _check_decode for the rest."""
    total = [a + b for a, b in zip(new, old)]
    need = [(n + 63) // 64 for n in total]
    cache = _random_cache(sum(need) + 2, hkv, d, spread)
    n = len(new)
    table = torch.full((n + 2, max(need) + 1), -1, dtype=torch.int32)
    slots = [int(x) for x in torch.randperm(n + 2)[:n]]
    order, a = torch.randperm(sum(need)).to(torch.int32), 0
    for i, k in zip(slots, need):
        table[i, :k] = order[a:a + k]
        a += k
    rows = (q_scale * torch.randn(sum(new), (hq + 2 * hkv) * d)).bfloat16()
    out = kvc.prefill_attention_with_prefix(rows.to(DEV), new, old, slots, _gpu(cache), table.to(DEV), hq, hkv, d).cpu().double()
    lib.check_status()
    assert out.shape == (sum(new), hq * d)
    at = 0
    for i, a, o, k in zip(slots, new, old, need):
        seen = [o + j + 1 for j in range(a)]
        pick = sorted(set(list(range(min(a, 3))) + list(range(0, a, 37)) + [a - 1])) if a else []
        want, size = oracle.attention(rows[[at + j for j in pick], :hq * d], *cache, table[i, :k].long(), [seen[j] for j in pick],
                                      hq, hkv, d, d ** -0.5)
        err = (out[[at + j for j in pick]] - want).abs()
        assert bool((err <= BF16 * want.abs() + (BF16 + 2.0 ** -10) * size).all()), (a, o)
        at += a


@pytest.mark.parametrize("hq,hkv,d", [(28, 4, 128), (14, 2, 64), (2, 2, 128), (4, 1, 64)])
@pytest.mark.parametrize("new,old", [((1,), (64,)), ((9,), (130,)), ((64, 1, 200), (1, 700, 64)), ((128, 129), (128, 63)),
                                     ((300, 5), (0, 1000)), ((257,), (255,))])
def test_prefix_attention(hq, hkv, d, new, old):
    _check_prefix(new, old, hq, hkv, d)


def test_prefix_attention_of_sharp_scores_and_unlike_scales():
    _check_prefix((100, 30), (200, 90), 28, 4, 128, 4.0, 8.0)
    _check_prefix((100, 30), (200, 90), 14, 2, 64, 4.0, 8.0)


def test_copied_blocks_bring_their_scales():
    cache = _gpu(_random_cache(6, 1, 64))
    idx = lambda *x: torch.tensor(x, dtype=torch.int32, device=DEV)  # noqa: E731
    want = cache.dequantize(idx(1, 3).long())
    rest = cache.dequantize(idx(1, 2, 3, 5).long())
    kvc.kv_copy_blocks(cache, idx(1, 3, 2), idx(0, 4, 99))
    assert torch.equal(cache.dequantize(idx(0, 4).long()), want)
    assert torch.equal(cache.dequantize(idx(1, 2, 3, 5).long()), rest)


def test_refusals():
    hq, hkv, d = 4, 2, 64
    cache = _gpu(_random_cache(4, hkv, d))
    table, lens = torch.zeros(2, 2, dtype=torch.int32, device=DEV), torch.ones(2, dtype=torch.int32, device=DEV)
    q = torch.randn(2, (hq + 2 * hkv) * d, device=DEV).bfloat16()
    wide = Cache8.zeros(4, hkv, 96, DEV)
    for call in (lambda: kvc.decode_attention(q.float(), cache, lens, table, hq, hkv, d),
                 lambda: kvc.decode_attention(q, cache, lens.cpu(), table, hq, hkv, d),
                 lambda: kvc.decode_attention(q, Cache8(cache.codes.cpu(), cache.scales), lens, table, hq, hkv, d),
                 lambda: kvc.decode_attention(q, wide, lens, table, 2, hkv, 96),
                 lambda: kvc.decode_attention(torch.zeros(2, 66 * d, device=DEV).bfloat16(), Cache8.zeros(4, 1, d, DEV), lens, table, 66, 1, d),
                 lambda: kvc.kv_append(q.float(), lens, lens, table, cache, hq, hkv, d),
                 lambda: kvc.prefill_attention_with_prefix(q.float(), [2], [3], [0], cache, table, hq, hkv, d),
                 lambda: kvc.prefill_attention_with_prefix(q, [2], [127], [0], cache, table, hq, hkv, d),
                 lambda: kvc.prefill_attention_with_prefix(q, [2], [3], [2], cache, table, hq, hkv, d),
                 lambda: kvc.prefill_attention_with_prefix(q, [3], [3], [0], cache, table, hq, hkv, d)):
        with pytest.raises(ValueError, match="8-bit cache"):
            call()


def test_engine_on_the_8_bit_cache():
    """Prompts, shared and forked blocks, reused prompts and decoding steps from a graph, through the rollout engine."""
    from siirl_b200.engine.rollout.native_engine import RolloutEngine, SamplingParams
    from siirl_b200.models.config import get_config
    from siirl_b200.models.decoder import build_model
    model = build_model(get_config("tiny-gpu"), dtype=torch.bfloat16, device=DEV, seed=1)
    prompts = [list(range(5, 5 + n)) for n in (7, 70, 130, 3)]
    sp = SamplingParams(n=2, temperature=0.0, max_new_tokens=70, eos_token_id=None)
    kw = dict(max_num_seqs=8, max_model_len=512, num_blocks=64, sync_interval=4)
    eager = RolloutEngine(model, use_cuda_graph=False, kv_cache_dtype="fp8", **kw)
    outs = eager.generate(prompts, sp)
    graph = RolloutEngine(model, use_cuda_graph=True, kv_cache_dtype="fp8", **kw)
    assert [o.token_ids for o in graph.generate(prompts, sp)] == [o.token_ids for o in outs]
    plain = RolloutEngine(model, use_cuda_graph=False, **kw).generate(prompts, sp)
    lib.check_status()
    # whole prompts attend to their unrounded keys
    assert [o.token_ids[0] for o in plain] == [o.token_ids[0] for o in outs]
    assert all(o.token_ids == p.token_ids for o, p in zip(outs[::2], outs[1::2]))      # greedy samples of a prompt
    assert eager.generate([p + [9, 8] for p in prompts], sp) is not None
    assert eager.stats["prefix_cache_hit_tokens"] >= 64 + 128
    lib.check_status()
    assert eager.alloc.num_free == eager.alloc.num_blocks


@pytest.mark.parametrize("hq,hkv,d", [(28, 4, 128), (14, 2, 64), (4, 1, 64)])
@pytest.mark.parametrize("new,old", [((5,), (3000,)), ((300, 40), (70, 0)), ((2300,), (1,))])
def test_prefix_attention_keeps_nan_from_rows_that_do_not_see_it(hq, hkv, d, new, old):
    """A key, and values of some columns, of tokens of the chunks and of a prefix: NaN in the rows that see them, and nowhere else."""
    total = [a + b for a, b in zip(new, old)]
    need = [(n + 63) // 64 for n in total]
    cache = _random_cache(sum(need), hkv, d)
    nan = cache.codes.view(torch.uint8)
    table, first = torch.full((len(new), max(need)), -1, dtype=torch.int32), 0
    for i, k in enumerate(need):
        table[i, :k] = torch.arange(first, first + k)
        t = total[i] - 3
        nan[first + t // 64, 1, 0, t % 64, [3, d - 1]] = 0x7f
        t = total[i] - 2
        nan[first + t // 64, 1, hkv - 1, t % 64, 17] = 0xff
        t = total[i] - 1
        nan[first + t // 64, 0, 0, t % 64, 5] = 0x7f
        first += k
    nan[0, 1, hkv - 1, 0, 40] = 0x7f        # all rows of the first sequence
    rows = torch.randn(sum(new), (hq + 2 * hkv) * d).bfloat16()
    out = kvc.prefill_attention_with_prefix(rows.to(DEV), new, old, list(range(len(new))), _gpu(cache), table.to(DEV), hq, hkv, d)
    out = out.cpu().double()
    lib.check_status()
    at = 0
    for i, (a, o, k) in enumerate(zip(new, old, need)):
        pick = sorted(set(range(0, a, 97)) | set(range(max(0, a - 5), a)))
        want, size = oracle.attention(rows[[at + j for j in pick], :hq * d], *cache, table[i, :k].long(), [o + j + 1 for j in pick],
                                      hq, hkv, d, d ** -0.5)
        got = out[[at + j for j in pick]]
        assert torch.equal(got.isnan(), want.isnan())
        err = (got - want).abs()
        assert bool((err <= BF16 * want.abs() + (BF16 + 2.0 ** -10) * size)[~want.isnan()].all())
        at += a


@pytest.mark.parametrize("hq,hkv,d", [(4, 2, 64), (16, 1, 128)])
def test_attention_of_more_sequences_than_a_launch_takes(hq, hkv, d):
    """Single tokens of 1300 sequences, some idle; chunks of 110, some empty."""
    n, most = 1300, 3
    cache = _random_cache(n, hkv, d)
    table = torch.randint(0, n, (n, most), dtype=torch.int32)
    lens = torch.randint(0, 64 * most + 1, (n,), dtype=torch.int32)
    lens[::7] = 0
    q = torch.randn(n, hq * d).bfloat16()
    out = kvc.decode_attention(q.to(DEV), _gpu(cache), lens.to(DEV), table.to(DEV), hq, hkv, d).cpu().double()
    for i in (0, 1, 500, 1022, 1023, 1024, 1025, 1298, 1299):
        want, size = oracle.attention(q[i:i + 1], *cache, table[i].long(), [int(lens[i])], hq, hkv, d, d ** -0.5)
        assert bool(((out[i:i + 1] - want).abs() <= BF16 * want.abs() + 2.0 ** -10 * size).all()), i
    assert not out[lens == 0].any()
    _check_prefix([(5 * i) % 23 if i % 9 else 0 for i in range(110)], [(31 * i) % 130 for i in range(110)], hq, hkv, d)


def test_calls_of_nothing():
    hq, hkv, d = 4, 2, 64
    cache = _gpu(_random_cache(4, hkv, d))
    before = cache.codes.view(torch.uint8).clone()
    i = lambda *x: torch.tensor(x, dtype=torch.int32, device=DEV)  # noqa: E731
    table, width = torch.zeros(2, 2, dtype=torch.int32, device=DEV), (hq + 2 * hkv) * d
    none = torch.empty(0, width, device=DEV, dtype=torch.bfloat16)
    cos, sin = (x.to(DEV) for x in ref.rope_tables(d, 64, 1e4))
    assert kvc.decode_attention(none, cache, i(), table[:0], hq, hkv, d).shape == (0, hq * d)
    assert not kvc.decode_attention(torch.ones(2, hq * d, device=DEV).bfloat16(), cache, i(0, 0), table, hq, hkv, d).any()
    kvc.kv_append(none, i(), i(), table, cache, hq, hkv, d)
    assert kvc.rope_kv_append(none, i(), cos, sin, None, i(), i(), table, cache, hq, hkv, d).shape == (0, width)
    kvc.kv_copy_blocks(cache, i(), i())
    assert kvc.prefill_attention_with_prefix(none, [], [], [], cache, table, hq, hkv, d).shape == (0, hq * d)
    assert kvc.prefill_attention_with_prefix(none, [0, 0], [0, 70], [0, 1], cache, table, hq, hkv, d).shape == (0, hq * d)
    row = torch.randn(1, width, device=DEV).bfloat16()
    kept = row.clone()
    kvc.kv_append(row, i(-1), i(3), table, cache, hq, hkv, d)       # a row of no sequence
    kvc.kv_append(row, i(0), i(128), table, cache, hq, hkv, d)      # and one behind the table
    torch.cuda.synchronize()
    assert torch.equal(cache.codes.view(torch.uint8), before) and torch.equal(row, kept)


def test_lengths_beyond_the_table_end_with_it():
    hq, hkv, d = 4, 2, 128
    cache = _gpu(_random_cache(5, hkv, d))
    table = torch.tensor([[4, 1], [0, 3]], dtype=torch.int32, device=DEV)
    q = torch.randn(2, hq * d, device=DEV).bfloat16()
    i = lambda *x: torch.tensor(x, dtype=torch.int32, device=DEV)  # noqa: E731
    want = kvc.decode_attention(q, cache, i(128, 0), table, hq, hkv, d)
    assert torch.equal(kvc.decode_attention(q, cache, i(2 ** 31 - 1, -5), table, hq, hkv, d), want)
    here = kvc.decode_attention(q.cpu(), Cache8(*(x.cpu() for x in cache)), i(2 ** 31 - 1, -5).cpu(), table.cpu(), hq, hkv, d)
    # two roundings to bf16, and the kernel's own error
    assert float((here.float() - want.cpu().float()).abs().max()) <= 2.0 ** -6 * float(want.abs().max())


def test_refusals_of_what_starts_at_odd_places():
    hq, hkv, d = 4, 2, 64
    cache, width = _gpu(_random_cache(4, hkv, d)), (4 + 2 * 2) * 64
    table, lens = torch.zeros(2, 2, dtype=torch.int32, device=DEV), torch.ones(2, dtype=torch.int32, device=DEV)
    cos, sin = (x.to(DEV) for x in ref.rope_tables(d, 64, 1e4))
    q = torch.randn(2, width, device=DEV).bfloat16()
    out = torch.empty(2 * hq * d + 8, dtype=torch.bfloat16, device=DEV)[3:3 + 2 * hq * d].view(2, hq * d)
    sums = torch.zeros(2 * width + 1, device=DEV)[1:].view(1, 2, width)
    odd = torch.zeros(2 * width + 1, dtype=torch.bfloat16, device=DEV)[1:].view(2, width)
    for call in (lambda: kvc.decode_attention(q, cache, lens, table, hq, hkv, d, out=out),
                 lambda: kvc.rope_kv_append(sums, lens, cos, sin, None, lens, lens, table, cache, hq, hkv, d),
                 lambda: kvc.rope_kv_append(odd, lens, cos, sin, None, lens, lens, table, cache, hq, hkv, d)):
        with pytest.raises(ValueError, match="8-bit cache"):
            call()
    want = kvc.decode_attention(q, cache, lens, table, hq, hkv, d)      # query rows may start anywhere
    odd.copy_(q)
    assert torch.equal(kvc.decode_attention(odd, cache, lens, table, hq, hkv, d), want)
    odd_q = torch.zeros(2 * hq * d + 1, dtype=torch.bfloat16, device=DEV)[1:].view(2, hq * d)
    odd_q.copy_(q[:, :hq * d])
    assert torch.equal(kvc.decode_attention(odd_q, cache, lens, table, hq, hkv, d), want)
    n, p, s = [2], [3], [0]
    assert torch.equal(kvc.prefill_attention_with_prefix(odd, n, p, s, cache, table, hq, hkv, d),
                       kvc.prefill_attention_with_prefix(q, n, p, s, cache, table, hq, hkv, d))


@pytest.mark.parametrize("hq,hkv,d", [(28, 4, 128), (14, 2, 64), (2, 2, 128), (16, 1, 128)])
@pytest.mark.parametrize("new,old", [((5,), (3000,)), ((300, 40), (70, 0)), ((700,), (1,))])
def test_attention_does_not_feel_large_values_that_it_does_not_see(hq, hkv, d, new, old):
    """The last three tokens of each sequence have the largest keys and values that a cache can hold: rows before them stay within
    the bounds that they have without these.  (Not to the bit: what the tensor cores keep of a sum depends on the largest exponent that
    takes part, also where the other factor is zero.)"""
    total = [a + b for a, b in zip(new, old)]
    need = [(n + 63) // 64 for n in total]
    cache = _random_cache(sum(need), hkv, d)
    table, first = torch.full((len(new), max(need)), -1, dtype=torch.int32), 0
    for i, (n, k) in enumerate(zip(total, need)):
        table[i, :k] = torch.arange(first, first + k)
        first += k
        assert n % 64 >= 3
        cache.codes[first - 1] = 0
        cache.codes[first - 1, :, :, n % 64 - 3:] = 448.0
        cache.scales[first - 1] = 2.0 ** 118
    rows = torch.randn(sum(new), (hq + 2 * hkv) * d).bfloat16()
    ends, q = torch.tensor(total, dtype=torch.int32) - 3, torch.randn(len(new), hq * d).bfloat16()
    g = _gpu(cache)
    chunks = kvc.prefill_attention_with_prefix(rows.to(DEV), new, old, list(range(len(new))), g, table.to(DEV), hq, hkv, d).cpu().double()
    single = kvc.decode_attention(q.to(DEV), g, ends.to(DEV), table.to(DEV), hq, hkv, d).cpu().double()
    lib.check_status()
    at = 0
    for i, (a, o, k) in enumerate(zip(new, old, need)):
        pick = sorted(set(range(0, a - 3, 97)) | set(range(max(0, a - 8), a - 3)))
        want, size = oracle.attention(rows[[at + j for j in pick], :hq * d], *cache, table[i, :k].long(), [o + j + 1 for j in pick], hq, hkv, d,
                                      d ** -0.5)
        err = (chunks[[at + j for j in pick]] - want).abs()
        assert bool((err <= BF16 * want.abs() + (BF16 + 2.0 ** -10) * size).all())
        want, size = oracle.attention(q[i:i + 1], *cache, table[i, :k].long(), [int(ends[i])], hq, hkv, d, d ** -0.5)
        assert bool(((single[i:i + 1] - want).abs() <= BF16 * want.abs() + 2.0 ** -10 * size).all())
        at += a


@pytest.mark.parametrize("hq,hkv,d", [(28, 4, 128), (32, 1, 64), (32, 1, 128)])
@pytest.mark.parametrize("scale", [0.0, -0.07])
def test_decode_attention_with_scales_of_any_sign(hq, hkv, d, scale):
    _check_decode(*_decode([700, 1, 0, 129], hq, hkv, d, 12), hq, hkv, d, scale)


@pytest.mark.parametrize("hq,hkv,d", [(28, 4, 128), (14, 2, 64), (9, 1, 64)])
@pytest.mark.parametrize("new,old", [((5,), (100,)), ((5,), (3000,)), ((300, 40), (4000, 0))])
def test_queries_that_are_not_finite_spoil_their_head_alone(hq, hkv, d, new, old):
    """NaN and infinities in some heads of some rows, keys split over several blocks or not: these heads are NaN, as soft-max has
    it, and all others hold the bounds of _check_prefix and _check_decode."""
    total = [a + b for a, b in zip(new, old)]
    need = [(n + 63) // 64 for n in total]
    cache = _random_cache(sum(need), hkv, d)
    table, first = torch.full((len(new), max(need)), -1, dtype=torch.int32), 0
    for i, k in enumerate(need):
        table[i, :k] = torch.arange(first, first + k)
        first += k
    rows = torch.randn(sum(new), (hq + 2 * hkv) * d).bfloat16()
    bad = torch.zeros(len(rows), hq, dtype=torch.bool)
    for r, h, at, x in ((0, 0, 5, math.nan), (1, hq - 1, 0, math.inf), (3, 1, d - 1, -math.inf), (len(rows) - 1, hq // 2, 9, math.nan)):
        rows[r, h * d + at] = x
        bad[r, h] = True
    bad = bad.repeat_interleave(d, 1)
    g = _gpu(cache)
    out = kvc.prefill_attention_with_prefix(rows.to(DEV), new, old, list(range(len(new))), g, table.to(DEV), hq, hkv, d).cpu().double()
    assert torch.equal(out.isnan(), bad)
    at = 0
    for i, (a, o, k) in enumerate(zip(new, old, need)):
        pick = sorted({0, 1, 2, 3, 4, a // 2, a - 1})
        good = ~bad[[at + j for j in pick]]
        want, size = oracle.attention(rows[[at + j for j in pick], :hq * d], *cache, table[i, :k].long(), [o + j + 1 for j in pick],
                                      hq, hkv, d, d ** -0.5)
        err = (out[[at + j for j in pick]] - want).abs()
        assert bool((err <= BF16 * want.abs() + (BF16 + 2.0 ** -10) * size)[good].all())
        at += a
    q, ends = rows[[0, 2][:len(new)]], torch.tensor(total, dtype=torch.int32)      # one with a NaN, one without
    out = kvc.decode_attention(q.to(DEV), g, ends.to(DEV), table.to(DEV), hq, hkv, d).cpu().double()
    lib.check_status()
    assert torch.equal(out.isnan(), bad[[0, 2][:len(new)]])
    for i, (n, k) in enumerate(zip(total, need)):
        want, size = oracle.attention(q[i:i + 1, :hq * d], *cache, table[i, :k].long(), [n], hq, hkv, d, d ** -0.5)
        x = cache.dequantize(table[i, :k].long(), torch.float64)[:, 1].transpose(0, 1).reshape(hkv, -1, d)[:, :n]
        least = 2.0 ** -36 * x.abs().sum(1).repeat_interleave(hq // hkv, 0).reshape(-1)
        ok = (out[i] - want[0]).abs() <= least + BF16 * want[0].abs() + 2.0 ** -10 * size[0]
        assert bool(ok[~out[i].isnan()].all())


@pytest.mark.parametrize("hq,hkv,d", [(2, 1, 128), (2, 1, 64)])
@pytest.mark.parametrize("old", [60, 3000])
@pytest.mark.parametrize("largest", [(), (6, 7), (2, 6), (0,)])
def test_an_infinite_query_is_nan_whichever_keys_it_meets(hq, hkv, d, old, largest):
    """Scores that are infinite: all of them -inf (``largest`` empty), or +inf for the tokens whose number modulo 8 is named."""
    need = (old + 1 + 63) // 64
    cache = _random_cache(need, hkv, d)
    key = torch.full((64,), -3.0)
    for i in largest:
        key[i::8] = 3.0
    cache.codes[:, 0, 0, :, 0] = key.to(torch.float8_e4m3fn)
    table = torch.arange(need, dtype=torch.int32)[None]
    rows = torch.zeros(1, (hq + 2 * hkv) * d)
    rows[0, 0] = math.inf
    g = _gpu(cache)
    out = kvc.prefill_attention_with_prefix(rows.bfloat16().to(DEV), [1], [old], [0], g, table.to(DEV), hq, hkv, d)
    assert bool(out[:, :d].isnan().all()) and bool(torch.isfinite(out[:, d:]).all())
    one = kvc.decode_attention(rows.bfloat16().to(DEV), g, torch.tensor([old + 1], dtype=torch.int32, device=DEV), table.to(DEV), hq, hkv, d)
    assert bool(one[:, :d].isnan().all()) and bool(torch.isfinite(one[:, d:]).all())
    lib.check_status()


def test_threads_on_one_stream():
    """Chunks and single tokens of four threads, all on the default stream."""
    import threading
    hq, hkv, d = 14, 2, 64
    lists, calls = [([9], [130]), ([5], [700]), ([64, 1], [1, 300])], []
    for new, old in lists:
        total = [a + b for a, b in zip(new, old)]
        need = [(n + 63) // 64 for n in total]
        g, table, first = _gpu(_random_cache(sum(need), hkv, d)), torch.full((len(new), max(need)), -1, dtype=torch.int32), 0
        for i, k in enumerate(need):
            table[i, :k] = torch.arange(first, first + k)
            first += k
        q, table = torch.randn(sum(new), (hq + 2 * hkv) * d).bfloat16().to(DEV), table.to(DEV)
        ends = torch.tensor(total, dtype=torch.int32, device=DEV)
        calls.append(lambda q=q, new=new, old=old, g=g, table=table: kvc.prefill_attention_with_prefix(
            q, new, old, list(range(len(new))), g, table, hq, hkv, d))
        calls.append(lambda q=q[:len(new)], ends=ends, g=g, table=table: kvc.decode_attention(q, g, ends, table, hq, hkv, d))
    want = [call() for call in calls]
    torch.cuda.synchronize()
    wrong = []

    def work(shift):
        for i in range(300):
            j = (i + shift) % len(calls)
            got = calls[j]()
            if i % 7 == shift and not torch.equal(got, want[j]):
                wrong.append((shift, i, j))
    threads = [threading.Thread(target=work, args=(k,)) for k in range(4)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    lib.check_status()
    assert not wrong


@pytest.mark.parametrize("hq,hkv,d", [(28, 4, 128), (14, 2, 64)])
def test_prefill_attention_of_mixed_batches(hq, hkv, d):
    """Sequences without earlier tokens attend to the rows' own keys and values, the others to the cache.  Bounds: _check_prefix."""
    from siirl_b200.ops.attention import SeqInfo
    new, old, slots = [5, 170, 1, 90], [100, 0, 700, 0], [2, 1, 0, 3]
    cache = _random_cache(30, hkv, d)
    table = torch.randperm(28).to(torch.int32).view(4, 7).repeat(1, 2).contiguous()
    rows = torch.randn(sum(new), (hq + 2 * hkv) * d).bfloat16()
    info = SeqInfo(new, device=torch.device(DEV))
    out = kvc.prefill_attention(rows.to(DEV), info, old, slots, _gpu(cache), table.to(DEV), hq, hkv, d).cpu().double()
    lib.check_status()
    for n, o, slot, got, x in zip(new, old, slots, out.split(new), rows.split(new)):
        k = -(-(n + o) // 64)
        held, blocks = cache, table[slot, :k].long()
        if o == 0:      # a cache of the rows themselves, without rounding
            kv = torch.zeros(k * 64, 2, hkv, d, dtype=torch.float64)
            kv[:n] = x[:, hq * d:].double().view(n, 2, hkv, d)
            held, blocks = Cache8(kv.view(k, 64, 2, hkv, d).permute(0, 2, 3, 1, 4), torch.ones(k, 2, hkv)), torch.arange(k)
        pick = sorted({0, n // 2, n - 1})
        want, size = oracle.attention(x[pick, :hq * d], *held, blocks, [o + j + 1 for j in pick], hq, hkv, d, d ** -0.5)
        assert bool(((got[pick] - want).abs() <= BF16 * want.abs() + (BF16 + 2.0 ** -10) * size).all())


def test_engine_chunks_and_reused_blocks_follow_from_the_cache():
    """One prompt at a time, so that the same kernels run on as many rows: in portions, and behind blocks of the prefix cache, with the
    tokens that the same portions give by hand.  Log-probabilities: of 32-bit logits, whose sums over the vocabulary may be in
    another order."""
    from siirl_b200.engine.rollout.native_engine import RolloutEngine, SamplingParams
    from siirl_b200.models.config import get_config
    from siirl_b200.models.decoder import build_model
    model, steps = build_model(get_config("tiny-gpu"), dtype=torch.bfloat16, device=DEV, seed=1), 20
    sp = SamplingParams(n=1, temperature=0.0, max_new_tokens=steps, ignore_eos=True)
    kw = dict(max_num_seqs=1, max_model_len=512, num_blocks=32, use_cuda_graph=False, kv_cache_dtype="fp8")
    eng = RolloutEngine(model, **kw)
    for n in (130, 70):
        prompt = list(range(5, 5 + n))
        eng.generate([prompt], sp)
        prompt, old = prompt + [9, 8], n // 64 * 64
        kept, cuts = eng._prefill, oracle.record_cuts(eng)
        got = eng.generate([prompt], sp)[0]
        eng._prefill = kept
        assert cuts == {0: [(old, n + 2)]}
        want, probs = oracle.engine_by_hand(model, eng._logits, prompt, [old, n + 2], steps)
        assert got.token_ids == want and all(abs(a - b) < 1e-4 for a, b in zip(got.logprobs, probs))
    eng = RolloutEngine(model, max_num_batched_tokens=64, enable_chunked_prefill=True, **kw)
    cuts = oracle.record_cuts(eng)
    got = eng.generate([prompt], sp)[0]
    assert cuts == {0: [(0, 64), (64, 72)]}
    want, probs = oracle.engine_by_hand(model, eng._logits, prompt, [64, 72], steps)
    assert got.token_ids == want and all(abs(a - b) < 1e-4 for a, b in zip(got.logprobs, probs))
    lib.check_status()


def test_append_to_rows_that_are_far_apart():
    """Two rows 2^31 + 8 numbers apart: the distance does not fit 32 bits."""
    hq, hkv, d = 4, 2, 64
    width, far = (hq + 2 * hkv) * d, 2 ** 31 + 8
    if torch.cuda.mem_get_info()[0] < 3 * far:
        pytest.skip("4 GB of rows")
    cache, table = _gpu(_random_cache(3, hkv, d)), torch.tensor([[1], [2]], dtype=torch.int32, device=DEV)
    other = Cache8(cache.codes.clone(), cache.scales.clone())
    cos, sin = (x.to(DEV) for x in ref.rope_tables(d, 64, 1e4))
    at, seq = torch.tensor([7, 30], dtype=torch.int32, device=DEV), torch.tensor([0, 1], dtype=torch.int32, device=DEV)
    near = torch.randn(2, width, device=DEV).bfloat16()
    rows = torch.empty(far + width, dtype=torch.bfloat16, device=DEV).as_strided((2, width), (far, 1))
    rows.copy_(near)
    want = kvc.rope_kv_append(near, at, cos, sin, None, seq, at, table, other, hq, hkv, d)
    got = kvc.rope_kv_append(rows, at, cos, sin, None, seq, at, table, cache, hq, hkv, d)
    assert torch.equal(got, want) and torch.equal(cache.codes.view(torch.uint8), other.codes.view(torch.uint8))
    assert torch.equal(cache.scales, other.scales)


@pytest.mark.parametrize("hq,hkv,d", [(4, 2, 64), (28, 4, 128)])
def test_calls_without_a_table_or_without_blocks(hq, hkv, d):
    """A table of no blocks, a cache of none: nothing is seen, by single tokens as on the CPU."""
    q, i = torch.randn(3, hq * d, device=DEV).bfloat16(), lambda *x: torch.tensor(x, dtype=torch.int32, device=DEV)  # noqa: E731
    cache, none = _gpu(_random_cache(2, hkv, d)), Cache8.zeros(0, hkv, d, DEV)
    table, lens = torch.zeros(3, 2, dtype=torch.int32, device=DEV), i(0, 5, 128)
    for c, t, n in ((cache, table[:, :0].contiguous(), lens), (cache, table[:, :0].contiguous(), i(0, 0, 0)), (none, table, lens)):
        out = torch.full((3, hq * d), 7.0, device=DEV, dtype=torch.bfloat16)
        assert kvc.decode_attention(q, c, n, t, hq, hkv, d, out=out) is out and not out.any()
    rows = torch.randn(2, (hq + 2 * hkv) * d, device=DEV).bfloat16()
    kept = rows.clone()
    kvc.kv_append(rows, i(0, 1), i(3, 4), table, none, hq, hkv, d)
    kvc.kv_append(rows, i(0, 1), i(3, 4), table[:, :0].contiguous(), cache, hq, hkv, d)
    kvc.kv_copy_blocks(none, i(0), i(1))
    assert torch.equal(rows, kept)
    lib.check_status()


@pytest.mark.parametrize("hq,hkv,d", [(28, 4, 128), (14, 2, 64), (5, 1, 128)])
@pytest.mark.parametrize("new,old", [((130, 41), (2500, 700)), ((2048, 3), (6000, 40)), ((9, 9), (130, 60))])
def test_chunks_repeat_themselves_whatever_ran_before(hq, hkv, d, new, old):
    """To the bit, after kernels that leave other numbers in shared memory; and whatever the other sequences' queries are: tiles of
    128 rows are not full where the heads of a kv head do not divide 128, or a sequence ends."""
    total = [a + b for a, b in zip(new, old)]
    need = [(n + 63) // 64 for n in total]
    cache, table, first = _random_cache(sum(need), hkv, d), torch.full((2, max(need)), -1, dtype=torch.int32), 0
    for i, k in enumerate(need):
        table[i, :k] = torch.arange(first, first + k)
        first += k
    g, table = _gpu(cache), table.to(DEV)
    rows = (3 * torch.randn(sum(new), (hq + 2 * hkv) * d)).bfloat16().to(DEV)

    def call(x):
        return kvc.prefill_attention_with_prefix(x, new, old, [0, 1], g, table, hq, hkv, d)
    want = call(rows)
    for i, size in enumerate((1.0, 30.0, 1000.0, 0.01)):
        call((size * torch.randn(rows.shape)).bfloat16().to(DEV))
        assert torch.equal(call(rows), want), i
    for i in range(2):
        other = rows.clone()
        other[new[0] * i:new[0] + new[1] * i] *= 100
        keep = slice(new[0], None) if i == 0 else slice(0, new[0])
        assert torch.equal(call(other)[keep], want[keep]), i
    lib.check_status()


def test_appended_chunks_in_graphs_that_take_turns():
    """Appending and chunks, with a workspace that is kept and with one of the call's own, captured twice and replayed on new
    numbers between calls outside of the graphs, and from another stream."""
    hq, hkv, d = 14, 2, 64
    cos, sin = (x.to(DEV) for x in ref.rope_tables(d, 4200, 1e4))
    width, i32 = (hq + 2 * hkv) * d, dict(dtype=torch.int32, device=DEV)
    lists = [([9], [130]), ([300, 2], [4000, 65])]
    calls = []
    for new, old in lists:
        need = [(a + b + 63) // 64 for a, b in zip(new, old)]
        table, first = torch.full((len(new), max(need)), -1, dtype=torch.int32), 0
        for i, k in enumerate(need):
            table[i, :k] = torch.arange(first, first + k)
            first += k
        at = torch.cat([torch.arange(b, b + a) for a, b in zip(new, old)]).to(**i32)
        seq = torch.repeat_interleave(torch.arange(len(new)), torch.tensor(new)).to(**i32)
        held, table, rows = _gpu(_random_cache(first, hkv, d)), table.to(DEV), torch.zeros(sum(new), width, device=DEV).bfloat16()

        def call(rows, cache, new=new, old=old, at=at, seq=seq, table=table):
            kvc.rope_kv_append(rows, at, cos, sin, None, seq, at, table, cache, hq, hkv, d)
            return kvc.prefill_attention_with_prefix(rows, new, old, list(range(len(new))), cache, table, hq, hkv, d)
        call(rows.clone(), Cache8(*(x.clone() for x in held)))
        calls.append((call, rows, held))
    graphs = []
    for _ in range(2):
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            graphs.append((graph, [call(rows, held) for call, rows, held in calls]))
    side = torch.cuda.Stream()
    for step, n in enumerate((0, 1, 1, 0)):
        fresh = [torch.randn(rows.shape, device=DEV).bfloat16() for _, rows, _ in calls]
        other = [Cache8(held.codes.clone(), held.scales.clone()) for _, _, held in calls]
        for (_, rows, _), x in zip(calls, fresh):
            rows.copy_(x)
        want = [call(x, c) for (call, _, _), x, c in zip(calls, fresh, other)]
        if step % 2:
            side.wait_stream(torch.cuda.current_stream())
            with torch.cuda.stream(side):
                graphs[n][0].replay()
            torch.cuda.current_stream().wait_stream(side)
        else:
            graphs[n][0].replay()
        for (_, rows, held), got, x, y, c in zip(calls, graphs[n][1], want, fresh, other):
            assert torch.equal(got, x) and torch.equal(rows, y) and torch.equal(held.scales, c.scales)
            assert torch.equal(held.codes.view(torch.uint8), c.codes.view(torch.uint8))
    lib.check_status()


def test_a_thread_whose_first_calls_are_captured():
    """Nothing that a thread's first call sets up may end a capture."""
    import threading
    hq, hkv, d = 14, 2, 64
    cache, table, q, n = _decode([300, 5], hq, hkv, d, 8)
    g, q, n, table = _gpu(cache), q.to(DEV), n.to(DEV), table.to(DEV)

    def calls():
        return [kvc.decode_attention(q, g, n, table, hq, hkv, d), kvc.prefill_attention_with_prefix(q, [2], [3], [0], g, table, hq, hkv, d)]
    want, got = calls(), []

    def work():
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            held = calls()
        graph.replay()
        torch.cuda.synchronize()
        got.extend(x.clone() for x in held)
    torch.cuda.synchronize()
    t = threading.Thread(target=work)
    t.start()
    t.join()
    lib.check_status()
    assert len(got) == 2 and all(torch.equal(a, b) for a, b in zip(got, want))
