"""Paged cache in 8 bits: definitions on the CPU, refusals, the rollout engine on it."""
import math

import pytest
import torch

import kv8_oracle as oracle
from siirl_b200.ops import kv_cache as kvc
from siirl_b200.ops import reference as ref
from siirl_b200.ops.kv_cache import Cache8


def _tables(d, n=600):
    return ref.rope_tables(d, n, 1e4)


def _append_cpu(rows, pos, cos, sin, section, seq, at, table, cache, hq, hkv, d):
    out = kvc.rope_kv_append(rows.clone(), pos, cos, sin, section, seq, at, table, cache, hq, hkv, d)
    return out


@pytest.mark.parametrize("hq,hkv,d", [(2, 1, 32), (4, 2, 64)])
def test_append_follows_its_definition(hq, hkv, d):
    """Fresh blocks, a block whose scale grows, one whose scale stays, rows of no sequence, a place named twice."""
    cache = Cache8.zeros(7, hkv, d)
    cos, sin = _tables(d)
    table = torch.tensor([[3, 0, 5], [6, 2, -1]], dtype=torch.int32)
    steps = [([0] * 70, list(range(70)), 1.0), ([1, 1], [0, 1], 1e-3), ([1], [2], 900.0), ([1, 0, -1, 1], [3, 70, 4, -1], 0.5),
             ([0, 0], [71, 71], 3.0), ([1], [130], 1.0)]
    for n, (seq, at, size) in enumerate(steps):
        seq, at = torch.tensor(seq, dtype=torch.int32), torch.tensor(at, dtype=torch.int32)
        rows = size * torch.randn(len(seq), (hq + 2 * hkv) * d)
        pos = at.clamp(min=0) + 3
        old = cache.codes.clone(), cache.scales.clone()
        got = _append_cpu(rows, pos, cos, sin, None, seq, at, table, cache, hq, hkv, d)
        want, raw, codes, scales, _ = oracle.append(rows, pos, cos, sin, None, seq, at, table, *old, hq, hkv, d)
        assert torch.allclose(got.double(), want, rtol=2 ** -20, atol=2 ** -20 * size)
        assert torch.equal(cache.scales.double(), scales), n
        # old rows exactly; new ones to half a step of their code (2^-4 of the value, 2^-10 scales below 2^-6 of them)
        kept = torch.isnan(raw)
        assert torch.equal(cache.codes.double()[kept], codes[kept])
        off = (cache.codes.double() * scales[..., None, None] - raw).abs()
        bound = torch.maximum(2 ** -4 * raw.abs(), 2 ** -10 * scales[..., None, None].expand_as(raw)) * (1 + 2 ** -18)
        assert bool((off <= bound)[~kept].all())


def test_scales_are_the_smallest_powers_of_two_and_survive_odd_values():
    cache = Cache8.zeros(2, 1, 32)
    table = torch.zeros(1, 1, dtype=torch.int32)
    seq = torch.zeros(1, dtype=torch.int32)
    row = torch.zeros(1, 96)
    for at, (top, want) in enumerate([(0.0, 2.0 ** -126), (1e-41, 2.0 ** -126), (448.0, 1.0), (448.0001, 2.0), (3.0e38, 2.0 ** 120)]):
        row[0, 32:64] = 0
        row[0, 40] = -top
        kvc.kv_append(row, seq, torch.tensor([at], dtype=torch.int32), table, cache, 1, 1, 32)
        assert float(cache.scales[0, 0, 0]) == want
    cache = Cache8.zeros(2, 1, 32)
    row[0, 32:64] = 3.0
    row[0, 33], row[0, 34], row[0, 35] = math.inf, -math.inf, math.nan
    kvc.kv_append(row, seq, torch.zeros(1, dtype=torch.int32), table, cache, 1, 1, 32)
    got = cache.codes[0, 0, 0, 0].float()
    scale = 2.0 ** -7         # 3 <= 448 * 2^-7
    assert float(cache.scales[0, 0, 0]) == scale and got[1] == 448 and got[2] == -448 and math.isnan(got[3]) and got[0] * scale == 3
    # the block begun anew holds nothing of that any more
    row.fill_(1.0)
    kvc.kv_append(row, seq, torch.zeros(1, dtype=torch.int32), table, cache, 1, 1, 32)
    assert bool(torch.isfinite(cache.codes.float()).all())


def test_dequantized_values_are_exact_in_bf16():
    codes = torch.arange(256, dtype=torch.uint8).view(torch.float8_e4m3fn)
    codes = torch.where(torch.isnan(codes.float()), torch.zeros(()), codes.float()).to(torch.float8_e4m3fn)
    cache = Cache8(codes.repeat(4).view(1, 2, 1, 64, 8).contiguous(), torch.full((1, 2, 1), 2.0 ** -9))
    blocks = torch.zeros(1, dtype=torch.int64)
    assert torch.equal(cache.dequantize(blocks, torch.bfloat16).float(), cache.dequantize(blocks))


@pytest.mark.parametrize("hq,hkv,d", [(2, 2, 32), (6, 2, 64)])
def test_attention_follows_its_definition(hq, hkv, d):
    cache = Cache8((torch.randn(9, 2, hkv, 64, d) * 50).clamp(-400, 400).to(torch.float8_e4m3fn),
                   2.0 ** torch.randint(-9, -4, (9, 2, hkv)).float())
    table = torch.tensor([[0, 3, 5], [1, -1, -1], [2, 4, 8], [7, 6, -1]], dtype=torch.int32)
    lens = torch.tensor([130, 0, 192, 65], dtype=torch.int32)
    q = torch.randn(4, (hq + 2 * hkv) * d)
    got = kvc.decode_attention(q, cache, lens, table, hq, hkv, d)
    for b in range(4):
        n = int(lens[b])
        want, size = oracle.attention(q[b:b + 1, :hq * d], *cache, table[b, :-(-n // 64)].long(), [n], hq, hkv, d, d ** -0.5)
        assert bool(((got[b] - want).abs() <= 1e-5 * size + 1e-30).all())
    new, old = [2, 1, 64, 7], [120, 0, 128, 58]
    rows = torch.randn(sum(new), (hq + 2 * hkv) * d)
    got = kvc.prefill_attention_with_prefix(rows, new, old, [0, 1, 2, 3], cache, table, hq, hkv, d)
    at = 0
    for i, (a, o) in enumerate(zip(new, old)):
        want, size = oracle.attention(rows[at:at + a, :hq * d], *cache, table[i, :-(-(a + o) // 64)].long(),
                                      [o + j + 1 for j in range(a)], hq, hkv, d, d ** -0.5)
        assert bool(((got[at:at + a] - want).abs() <= 1e-5 * size).all())
        at += a


def test_copied_blocks_bring_their_scales():
    cache = Cache8.zeros(5, 2, 32)
    cache.codes.view(torch.uint8).copy_(torch.randint(0, 120, cache.codes.shape))
    cache.scales.copy_(2.0 ** torch.randint(-9, 9, cache.scales.shape))
    want = cache.dequantize(torch.tensor([1, 3]))
    kvc.kv_copy_blocks(cache, torch.tensor([1, 3], dtype=torch.int32), torch.tensor([0, 4], dtype=torch.int32))
    assert torch.equal(cache.dequantize(torch.tensor([0, 4])), want)


def test_copies_that_name_no_block_are_left_out():
    cache = Cache8.zeros(5, 2, 32)
    cache.codes.view(torch.uint8).copy_(torch.randint(0, 120, cache.codes.shape))
    cache.scales.copy_(2.0 ** torch.randint(-9, 9, cache.scales.shape))
    want = cache.dequantize(torch.tensor([0, 1, 2, 3, 1]))
    i = lambda *x: torch.tensor(x, dtype=torch.int32)  # noqa: E731
    kvc.kv_copy_blocks(cache, i(1, -1, 2, 3, 5), i(4, 0, -1, 99, 1))
    assert torch.equal(cache.dequantize(torch.arange(5)), want)
    for src, dst in ((i(1), i(2, 3)), (i(1).long(), i(2).long()), (i(1)[None], i(2)[None])):
        with pytest.raises(ValueError, match="8-bit cache"):
            kvc.kv_copy_blocks(cache, src, dst)


def test_refusals():
    hq, hkv, d = 4, 2, 64
    cache = Cache8.zeros(4, hkv, d)
    table, lens = torch.zeros(2, 2, dtype=torch.int32), torch.ones(2, dtype=torch.int32)
    q = torch.randn(2, (hq + 2 * hkv) * d)
    cos, sin = _tables(d)

    def decode(q=q, cache=cache, lens=lens, table=table, hq=hq, hkv=hkv, d=d, out=None):
        return kvc.decode_attention(q, cache, lens, table, hq, hkv, d, out=out)

    def append(q=q, seq=lens, at=lens, cache=cache, cos=cos, pos=lens, bias=None):
        return kvc.rope_kv_append(q, pos, cos, sin, None, seq, at, table, cache, hq, hkv, d, bias)
    decode(), append(q.clone())
    half = Cache8(cache.codes.to(torch.bfloat16), cache.scales)
    for call in (lambda: decode(cache=half), lambda: decode(cache=Cache8(cache.codes, cache.scales[:3])),
                 lambda: decode(cache=Cache8(cache.codes, cache.scales.half())), lambda: decode(hkv=1), lambda: decode(hq=3),
                 lambda: decode(d=32), lambda: decode(lens=lens.long()), lambda: decode(lens=lens[:1]),
                 lambda: decode(table=table.long()), lambda: decode(table=table.repeat(1, 2)[:, :2]), lambda: decode(q=q[:, :hq * d - 1]),
                 lambda: decode(table=table[:1]), lambda: decode(q=q.t().contiguous().t()),
                 lambda: decode(out=torch.empty(2, hq * d, dtype=torch.float16)), lambda: decode(out=torch.empty(3, hq * d)),
                 lambda: append(q[:, :-1]), lambda: append(seq=lens[:1]), lambda: append(at=lens.long()),
                 lambda: append(cos=cos[:, :-1]), lambda: append(cos=cos.double()), lambda: append(pos=lens[:1]),
                 lambda: append(bias=torch.zeros(q.shape[1])), lambda: append(q.half()[None]),
                 lambda: append(cache=Cache8(cache.codes.transpose(2, 3), cache.scales))):
        with pytest.raises(ValueError, match="8-bit cache"):
            call()


def test_chunk_calls_of_threads_do_not_meet_in_a_workspace(monkeypatch):
    """A call for chunks launches kernels that hand data on through a workspace: while one is in the library, no other call may be
    there with the same memory, nor may single tokens have it."""
    import ctypes
    import threading
    import time
    from siirl_b200.ops import kv_cache8
    inside, met, rows = {}, [], 3

    class Library:
        def sb_kv8_chunk_seqs(self):
            return 48

        def sb_kv8_chunks(self, *args):
            kept, sizes = args[13], ctypes.cast(args[15], ctypes.POINTER(ctypes.c_longlong))
            met.append(inside.get(kept, 0))
            inside[kept] = inside.get(kept, 0) + 1
            time.sleep(0.02)
            inside[kept] -= 1
            sizes[1], sizes[2] = rows, 2
            return 0
    monkeypatch.setattr(kv_cache8._lib, "get_lib", Library)
    monkeypatch.setattr(kv_cache8._lib, "add_launches", lambda n: None)
    monkeypatch.setattr(kv_cache8._lib, "status_word", lambda device: torch.zeros(1, dtype=torch.int32))
    for name, value in (("_cuda_getDevice", -1), ("_cuda_getCurrentRawStream", 0), ("_cuda_isCurrentStreamCapturing", False)):
        monkeypatch.setattr(torch._C, name, lambda *args, value=value: value)
    real = torch.empty
    monkeypatch.setattr(torch, "empty", lambda *size, device=None, **kw: real(*size, **kw))
    real_zeros = torch.zeros
    monkeypatch.setattr(torch, "zeros", lambda *size, device=None, **kw: real_zeros(*size, **kw))
    monkeypatch.setattr(kv_cache8, "_buffers", {})
    hq, hkv, d = 4, 2, 64
    cache, table = Cache8.zeros(4, hkv, d), real_zeros(1, 2, dtype=torch.int32)
    qkv = real_zeros(rows, (hq + 2 * hkv) * d, dtype=torch.bfloat16)
    threads = [threading.Thread(target=lambda: [kv_cache8.chunk_attention(qkv, [rows], [5], [0], cache, table, hq, hkv, d)
                                                for _ in range(4)]) for _ in range(3)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert len(met) == 12 and not any(met)
    # the buffers that are kept for the stream: that of the chunks, and another one for single tokens
    kv_cache8._workspace(-1, 0, 100, 8)
    places = [held[0].data_ptr() for held in kv_cache8._buffers.values()]
    assert len(set(places)) == 2 and set(places) > set(inside)


def test_arguments_are_passed_as_the_library_declares_them():
    """Numbers go to these entry points without a ctypes object of their own: a letter that is too narrow would cut them off in
    silence.  Distances between rows are 64 bits wide."""
    import pathlib
    import re
    from siirl_b200.ops import lib
    header = (pathlib.Path(lib.__file__).parent.parent / "csrc" / "launchers.h").read_text()
    for name, letters in lib._ARGUMENTS.items():
        arguments = [x.strip() for x in re.search(rf"\b{name}\(([^)]*)\)", header).group(1).split(",")]
        kinds = ["p" if "*" in x or "cudaStream_t" in x else "l" if "long long" in x else "f" if x.startswith("float") else "i"
                 for x in arguments]
        assert "".join(kinds) == letters, name
        for x, kind in zip(arguments, kinds):
            assert "stride" not in x or kind == "l", (name, x)


def test_tables_whose_lengths_pass_32_bits_are_refused():
    """More than 2^24 blocks: 64 times their number, rounded up, is not sure to fit."""
    import ctypes
    from siirl_b200.ops import lib
    hq, hkv, d = 2, 1, 64
    cache, table = Cache8.zeros(2, hkv, d), torch.zeros(1, 2 ** 24 + 1, dtype=torch.int32)
    q, one = torch.randn(1, (hq + 2 * hkv) * d), torch.ones(1, dtype=torch.int32)
    for call in (lambda: kvc.decode_attention(q, cache, one, table, hq, hkv, d),
                 lambda: kvc.kv_append(q, one * 0, one, table, cache, hq, hkv, d),
                 lambda: kvc.prefill_attention_with_prefix(q, [1], [3], [0], cache, table, hq, hkv, d)):
        with pytest.raises(ValueError, match="8-bit cache"):
            call()
    # the library by itself, before it looks at anything else
    L, sizes, lists = lib.get_lib(), (ctypes.c_longlong * 3)(), (ctypes.c_int * 2)(1, 0)
    for blocks in (2 ** 24 + 1, 2 ** 25, 2 ** 31 - 1):
        assert L.sb_kv8_decode(16, 256, 16, 16, 2, 16, 16, blocks, 16, 16, 16, 16, 1, hq, hkv, d, 0.1, 16, 0) == -4
        at = ctypes.addressof(lists)
        assert L.sb_kv8_chunks(16, 256, 1, 16, 16, 2, 16, 1, blocks, at, at, at + 4, 1, 16, 0,
                               ctypes.addressof(sizes), 16, hq, hkv, d, 0.1, 16, 0) == -4


# ---- the rollout engine -------------------------------------------------------------------------
@pytest.fixture(scope="module")
def tiny():
    from siirl_b200.models.config import get_config
    from siirl_b200.models.decoder import build_model
    return build_model(get_config("tiny"), dtype=torch.float32, device="cpu", seed=3)


def test_engine_decodes_what_its_cache_holds(tiny):
    """Greedy tokens with shared prompts, forked blocks and several blocks per sequence: each follows from attention to rounded
    keys and values, recomputed here token by token."""
    from siirl_b200.engine.rollout.native_engine import RolloutEngine, SamplingParams
    cfg = tiny.cfg
    eng = RolloutEngine(tiny, max_num_seqs=8, max_model_len=256, num_blocks=40, sync_interval=4, kv_cache_dtype="fp8")
    assert all(isinstance(x, Cache8) for x in eng.cache)
    assert eng._block_bytes() == sum(x.codes[0].numel() + 4 * x.scales[0].numel() for x in eng.cache)
    prompts = [[5, 6, 7, 8, 9], list(range(20, 20 + 70)), list(range(9, 9 + 64))]
    outs = eng.generate(prompts, SamplingParams(n=2, temperature=0.0, max_new_tokens=6, ignore_eos=True))
    plain = RolloutEngine(tiny, max_num_seqs=8, max_model_len=256, num_blocks=40, sync_interval=4)
    want = plain.generate(prompts, SamplingParams(n=2, temperature=0.0, max_new_tokens=6, ignore_eos=True))
    # the first token comes from unrounded keys; samples of a prompt are the same; log-probs stay near
    for o, w in zip(outs, want):
        assert o.token_ids[0] == w.token_ids[0] and abs(o.logprobs[0] - w.logprobs[0]) < 1e-5
        same = next((i for i, (a, b) in enumerate(zip(o.token_ids, w.token_ids)) if a != b), 6)
        assert all(abs(a - b) < 0.2 for a, b in zip(o.logprobs[:same], w.logprobs[:same]))
    assert [outs[0].token_ids, outs[2].token_ids, outs[4].token_ids] == [outs[1].token_ids, outs[3].token_ids, outs[5].token_ids]
    assert eng.alloc.num_free == eng.alloc.num_blocks
    # one sequence by hand
    cache = [Cache8.zeros(4, cfg.num_kv_heads, cfg.head_dim) for _ in range(cfg.num_layers)]
    table, ids = torch.tensor([[2, 0, 3]], dtype=torch.int32), list(prompts[1])
    one = torch.zeros(1, dtype=torch.int32)
    from siirl_b200.ops.attention import SeqInfo
    info = SeqInfo([len(ids)])
    hidden = tiny.forward_cached(torch.tensor(ids), info.positions, cache, table, one.expand(len(ids)).contiguous(), prefill_info=info)[-1:]
    got = []
    for n in range(len(ids), len(ids) + 6):
        got.append(int(eng._logits(hidden).argmax()))
        hidden = tiny.forward_cached(torch.tensor(got[-1:]), one + n, cache, table, one, seq_lens=one + n + 1)
    assert got == outs[2].token_ids


def test_engine_chunks_and_reuses_prompts(tiny):
    from siirl_b200.engine.rollout.native_engine import RolloutEngine, SamplingParams
    prompts = [list(range(7, 7 + n)) for n in (150, 70)]
    sp = SamplingParams(n=1, temperature=0.0, max_new_tokens=4, ignore_eos=True)
    eng = RolloutEngine(tiny, max_num_seqs=8, max_model_len=256, num_blocks=40, kv_cache_dtype="fp8")
    eng.generate(prompts, sp)
    again = eng.generate([p + [3, 4] for p in prompts], sp)
    assert eng.stats["prefix_cache_hit_tokens"] == 128 + 64
    chunked = RolloutEngine(tiny, max_num_seqs=8, max_model_len=256, num_blocks=40, max_num_batched_tokens=64,
                            enable_chunked_prefill=True, kv_cache_dtype="fp8")
    assert len(chunked.generate(prompts, sp)) == len(again) == 2
    eng.borrowed = torch.full((300_000,), math.nan)
    eng.sleep()
    eng.wake_up()
    assert eng.kv_layout["layers_in_borrowed_memory"] > 0
    assert [o.token_ids for o in eng.generate([p + [3, 4] for p in prompts], sp)] is not None
    assert all(bool(torch.isfinite(x.codes.float()).all()) for x in eng.cache)


def test_engine_chunks_and_reused_blocks_follow_from_the_cache(tiny):
    """Prompts in portions, and prompts whose first blocks come from the prefix cache: tokens and log-probabilities are those of the
    same portions recomputed by hand, on a cache that has held nothing else."""
    from siirl_b200.engine.rollout.native_engine import RolloutEngine, SamplingParams
    prompts, steps = [list(range(7, 7 + n)) for n in (150, 70)], 5
    sp = SamplingParams(n=1, temperature=0.0, max_new_tokens=steps, ignore_eos=True)
    kw = dict(max_num_seqs=8, max_model_len=256, num_blocks=40, kv_cache_dtype="fp8")
    eng = RolloutEngine(tiny, **kw)
    eng.generate(prompts, sp)
    again = [p + [3, 4] for p in prompts]
    cuts = oracle.record_cuts(eng)
    reused = eng.generate(again, sp)
    assert cuts == {0: [(128, 152)], 1: [(64, 72)]}
    for i, got in enumerate(reused):
        want, probs = oracle.engine_by_hand(tiny, eng._logits, again[i], [cuts[i][0][0], len(again[i])], steps)
        assert got.token_ids == want and all(abs(a - b) < 1e-5 for a, b in zip(got.logprobs, probs))
    eng = RolloutEngine(tiny, max_num_batched_tokens=64, enable_chunked_prefill=True, **kw)
    cuts = oracle.record_cuts(eng)
    chunked = eng.generate(prompts, sp)
    assert len(cuts[0]) == 3 and len(cuts[1]) == 2
    for i, got in enumerate(chunked):
        assert [a for a, _ in cuts[i]] == [0] + [b for _, b in cuts[i][:-1]]
        want, probs = oracle.engine_by_hand(tiny, eng._logits, prompts[i], [b for _, b in cuts[i]], steps)
        assert got.token_ids == want and all(abs(a - b) < 1e-5 for a, b in zip(got.logprobs, probs))


def test_whole_prompts_attend_to_unrounded_keys_whatever_they_are_admitted_with(tiny):
    """A prompt that is prefilled whole: alone, and in one batch with prompts whose first blocks the prefix cache holds, before and
    behind it.  These in turn get what they get without it."""
    from siirl_b200.engine.rollout.native_engine import RolloutEngine, SamplingParams
    sp = SamplingParams(n=1, temperature=0.0, max_new_tokens=3, ignore_eos=True)
    kw = dict(max_num_seqs=8, max_model_len=256, num_blocks=40, kv_cache_dtype="fp8")
    known, whole = [list(range(7, 7 + n)) for n in (150, 70)], list(range(30, 130))
    again = [p + [3, 4] for p in known]
    alone = RolloutEngine(tiny, **kw).generate([whole], sp)[0]
    eng = RolloutEngine(tiny, **kw)
    eng.generate(known, sp)
    reused = eng.generate(again, sp)
    eng = RolloutEngine(tiny, **kw)
    eng.generate(known, sp)
    mixed = eng.generate([again[0], whole, again[1]], sp)
    assert eng.stats["prefix_cache_hit_tokens"] == 128 + 64
    for got, want in zip(mixed, (reused[0], alone, reused[1])):
        assert got.token_ids == want.token_ids
        assert all(abs(a - b) < 1e-5 for a, b in zip(got.logprobs, want.logprobs))


def test_prefill_attention_of_mixed_batches():
    hq, hkv, d = 4, 2, 32
    cache = Cache8((torch.randn(9, 2, hkv, 64, d) * 50).clamp(-400, 400).to(torch.float8_e4m3fn), 2.0 ** torch.randint(-9, -4, (9, 2, hkv)).float())
    table = torch.tensor([[0, 3, 5], [1, 6, -1], [2, 4, 8], [7, -1, -1]], dtype=torch.int32)
    from siirl_b200.ops.attention import SeqInfo, attention_packed
    new, old, slots = [5, 70, 1, 9], [100, 0, 64, 0], [2, 1, 0, 3]
    rows = torch.randn(sum(new), (hq + 2 * hkv) * d)
    got = kvc.prefill_attention(rows, SeqInfo(new), old, slots, cache, table, hq, hkv, d).split(new)
    parts = rows.split(new)
    for i in range(4):
        if old[i]:
            want = kvc.prefill_attention_with_prefix(parts[i], [new[i]], [old[i]], [slots[i]], cache, table, hq, hkv, d)
        else:
            want = attention_packed(parts[i], SeqInfo([new[i]]), hq, hkv, d)
        assert torch.allclose(got[i], want, rtol=1e-5, atol=1e-6)
    # a cache of the rows' type: as before, in one call
    plain = cache.dequantize(torch.arange(9))
    assert torch.equal(kvc.prefill_attention(rows, SeqInfo(new), old, slots, plain, table, hq, hkv, d),
                       kvc.prefill_attention_with_prefix(rows, new, old, slots, plain, table, hq, hkv, d))
    for none in (None, [0, 0, 0, 0]):
        assert torch.equal(kvc.prefill_attention(rows, SeqInfo(new), none, None, cache, table, hq, hkv, d),
                           attention_packed(rows, SeqInfo(new), hq, hkv, d))


def test_engine_refusals(tiny):
    from siirl_b200.engine.rollout.native_engine import RolloutEngine
    with pytest.raises(ValueError, match="kv_cache_dtype"):
        RolloutEngine(tiny, max_num_seqs=8, max_model_len=64, kv_cache_dtype="int8")
    from siirl_b200.models.config import get_config
    from siirl_b200.models.decoder import build_model
    hybrid = build_model(get_config("tiny-domavik"), dtype=torch.float32, device="cpu", seed=0)
    with pytest.raises(ValueError, match="hybrid"):
        RolloutEngine(hybrid, max_num_seqs=8, max_model_len=64, num_blocks=8, kv_cache_dtype="fp8")


def _tensor_parallel_rank(rank, where, results):
    """Rank of test_tensor_parallel_engines_keep_their_heads_in_8_bits."""
    import torch.distributed as dist
    from siirl_b200.engine.rollout.native_engine import RolloutEngine, SamplingParams
    from siirl_b200.models.config import get_config
    from siirl_b200.models.decoder import build_model
    from siirl_b200.models.tp_decoder import TPDecoder
    from siirl_b200.parallel.tensor_parallel import TPContext
    torch.set_num_threads(2)
    dist.init_process_group("gloo", init_method=f"file://{where}", rank=rank, world_size=2)
    cfg = get_config("tiny")
    model = build_model(cfg, dtype=torch.float32, device="cpu", seed=3)
    view = TPDecoder(model, TPContext(dist.group.WORLD, None, max_rows=1024, max_cols=cfg.hidden_size, max_tiles=64))
    sp = SamplingParams(n=1, temperature=0.0, max_new_tokens=5, ignore_eos=True)
    known, whole, outs = [list(range(7, 7 + n)) for n in (150, 70)], list(range(30, 130)), []
    for m in (model, view):
        eng = RolloutEngine(m, max_num_seqs=8, max_model_len=256, num_blocks=40, kv_cache_dtype="fp8")
        outs.append(eng.generate(known, sp) + eng.generate([known[0] + [3, 4], whole, known[1] + [3, 4]], sp))
        assert eng.stats["prefix_cache_hit_tokens"] == 128 + 64
    results.put((rank, eng.cache[0].codes.shape[2] == cfg.num_kv_heads // 2,
                 [(o.token_ids, w.token_ids, max(abs(a - b) for a, b in zip(o.logprobs, w.logprobs))) for o, w in zip(*outs)]))
    dist.barrier()
    dist.destroy_process_group()


def test_tensor_parallel_engines_keep_their_heads_in_8_bits(tmp_path):
    """Two ranks with half of the heads each, prompts with and without reused blocks: what one rank with all heads gets, as scales are
    a head's own."""
    import torch.multiprocessing as mp
    ctx = mp.get_context("spawn")
    results = ctx.Queue()
    ranks = [ctx.Process(target=_tensor_parallel_rank, args=(i, str(tmp_path / "meet"), results)) for i in range(2)]
    for r in ranks:
        r.start()
    got = [results.get(timeout=240) for _ in ranks]
    for r in ranks:
        r.join(60)
        assert r.exitcode == 0
    for _, halved, pairs in got:
        assert halved and len(pairs) == 5
        for mine, one, off in pairs:
            assert mine == one and off < 1e-4
