"""Paged key / value cache in 8 bits with a scale for each block of tokens and head.

:class:`Cache8` stands where the functions of :mod:`siirl_b200.ops.kv_cache` take the cache of a layer (``rope_kv_append``,
``kv_append``, ``decode_attention``, ``prefill_attention_with_prefix``, ``kv_copy_blocks``); those call what is here.  It holds
``codes [num_blocks, 2, Hkv, 64, D]`` (e4m3; keys, then values) and ``scales [num_blocks, 2, Hkv]`` (fp32): a cached value is
code times scale, half the bytes of the bf16 cache.  Scales are powers of two; of others, which only a caller's own cache can
have, chunks round the values to bf16.

Appending keeps each scale at the smallest power of two (at least 2^-126) with which every finite value that its block and
head have met fits e4m3's range, ``|x| <= 448 * scale``.  New values are rounded once, from the rotated 32-bit ones, to the
nearest code; infinities become +-448 times the scale, NaN stays NaN.  Where new rows raise a scale, the block's other rows are
rounded to it.  A row at offset 0 of a block starts it anew: rows that the call does not write become zeros.  Rows of one call
that lie in the same block have to follow one another; where one place is named twice, its last row counts."""
from __future__ import annotations

import array
import ctypes
import math
import threading
from typing import NamedTuple, Optional

import torch

from . import lib as _lib

BLOCK = 64
LARGEST = 448.0             # of e4m3
HEAD_DIMS = (64, 128)       # of the kernels; the CPU statements take any
ROWS = 1024                 # sequences of one launch of the single-token kernel
TABLE = 2 ** 24             # blocks of a sequence: lengths and what they are rounded up to stay within 32 bits
CHUNK_BYTES = 2 ** 20       # chunks that need no more take a workspace that is kept


class Cache8(NamedTuple):
    """Cache of one layer: a cached value is ``codes`` times the block's and head's scale in ``scales``."""
    codes: torch.Tensor
    scales: torch.Tensor

    @classmethod
    def zeros(cls, num_blocks: int, n_kv_heads: int, head_dim: int, device=None) -> "Cache8":
        return cls(torch.zeros(num_blocks, 2, n_kv_heads, BLOCK, head_dim, dtype=torch.uint8,
                               device=device).view(torch.float8_e4m3fn),
                   torch.zeros(num_blocks, 2, n_kv_heads, dtype=torch.float32, device=device))

    def dequantize(self, blocks: torch.Tensor, dtype: torch.dtype = torch.float32) -> torch.Tensor:
        """Values ``[len(blocks), 2, Hkv, 64, D]`` of some blocks; exact in bf16, too, where the scales are powers of two."""
        codes = self.codes.view(torch.uint8)[blocks].view(torch.float8_e4m3fn)
        return (codes.float() * self.scales[blocks][..., None, None]).to(dtype)


def block_bytes(n_kv_heads: int, head_dim: int) -> int:
    """Bytes of one block of one layer, scales included."""
    return 2 * n_kv_heads * (BLOCK * head_dim + 4)


def _refuse(what: str) -> None:
    raise ValueError(f"8-bit cache: {what}")


# The checks below run before every call of a decoding step: one expression each, and words only where it fails.
def _check(cache: Cache8, n_heads: int, n_kv_heads: int, head_dim: int, rows: torch.Tensor) -> None:
    codes, scales = cache
    shape = codes.shape
    if codes.dtype is not torch.float8_e4m3fn or scales.dtype is not torch.float32:
        _refuse(f"codes are float8_e4m3fn, scales float32, got {codes.dtype}, {scales.dtype}")
    if shape != (shape[0], 2, n_kv_heads, BLOCK, head_dim) or scales.shape != (shape[0], 2, n_kv_heads):
        _refuse(f"codes are [blocks, 2, {n_kv_heads}, {BLOCK}, {head_dim}], scales [blocks, 2, {n_kv_heads}], got "
                f"{tuple(codes.shape)}, {tuple(scales.shape)}")
    if not codes.is_contiguous() or not scales.is_contiguous():
        _refuse("codes and scales are contiguous")
    if n_heads <= 0 or n_heads % n_kv_heads:
        _refuse(f"{n_heads} query heads on {n_kv_heads} kv heads")
    dev = rows.get_device()
    if codes.get_device() != dev or scales.get_device() != dev:
        _refuse("cache and rows are on one device")
    if dev >= 0 and (head_dim not in HEAD_DIMS or n_heads > 32 * n_kv_heads or codes.data_ptr() % 16):
        _refuse(f"the kernels take head widths {HEAD_DIMS}, at most 32 query heads per kv head and codes that start on a 16-byte "
                f"boundary, not {head_dim}, {n_heads} / {n_kv_heads}, {codes.data_ptr() % 16}")


def _check_ints(rows: torch.Tensor, *ints: torch.Tensor) -> None:
    dev = rows.get_device()
    for t in ints:
        if t.dtype is not torch.int32 or t.get_device() != dev or not t.is_contiguous():
            _refuse("lengths, ids, positions and block tables are contiguous int32 tensors on the rows' device")


# ---- appending ----------------------------------------------------------------------------------
def _scale_of(amax: torch.Tensor) -> torch.Tensor:
    half, exp = torch.frexp(amax)       # amax = half * 2^exp, 448 = 0.875 * 2^9
    exp = torch.where(half == 0, torch.full_like(exp, -126), (exp - 9 + (half > 0.875)).clamp(min=-126))
    return torch.ldexp(torch.ones_like(amax), exp)


def _append_cpu(kv: torch.Tensor, seq_ids, positions, block_table, cache: Cache8) -> None:
    """``kv [T, 2, Hkv, D]`` in fp32, rotated."""
    codes, scales = cache
    sequences, width = block_table.shape
    ok = (seq_ids >= 0) & (seq_ids < sequences) & (positions >= 0) & (positions < width * BLOCK)
    kv, seq_ids, positions = kv[ok], seq_ids[ok].long(), positions[ok].long()
    blk = block_table[seq_ids, positions // BLOCK].long()
    ok = (blk >= 0) & (blk < codes.shape[0])
    kv, blk, off = kv[ok], blk[ok], positions[ok] % BLOCK
    top = kv.abs()
    top = torch.where(torch.isfinite(top), top, torch.zeros_like(top)).amax(-1)
    for b in blk.unique().tolist():
        rows = (blk == b).nonzero()[:, 0]
        at = off[rows]
        anew = bool((at == 0).any())
        kept = torch.zeros_like(scales[b]) if anew else scales[b]
        scale = torch.maximum(kept, _scale_of(top[rows].amax(0)))
        values = torch.zeros(codes.shape[1:]) if anew else codes[b].float() * (kept / scale)[..., None, None]
        for r, o in zip(rows.tolist(), at.tolist()):
            values[:, :, o] = kv[r] / scale[..., None]
        codes[b] = values.clamp(-LARGEST, LARGEST).to(codes.dtype)
        scales[b] = scale


def append(qkv: torch.Tensor, rope, seq_ids: torch.Tensor, positions: torch.Tensor, block_table: torch.Tensor,
           cache: Cache8, n_heads: int, n_kv_heads: int, head_dim: int, bias: Optional[torch.Tensor] = None) -> torch.Tensor:
    """Appends the k and v heads of ``qkv [T, (Hq + 2 Hkv) * D]`` to the cache.  ``rope`` (``positions [T] or [3, T], cos, sin,
    mrope_section``, or None): rotates the q and k heads in place first.  ``qkv [S, T, width]``: partial sums, whose sum with
    ``bias`` is rotated and returned as bf16 rows."""
    slabs = qkv if qkv.dim() == 3 else None
    T, width = qkv.shape[-2:]
    if width != (n_heads + 2 * n_kv_heads) * head_dim:
        _refuse(f"rows are {(n_heads + 2 * n_kv_heads) * head_dim} wide, got {width}")
    if seq_ids.shape != (T,) or positions.shape != (T,) or block_table.dim() != 2 or block_table.shape[1] > TABLE:
        _refuse(f"one sequence and position for each of {T} rows, and a table of at most {TABLE} blocks for each sequence")
    _check(cache, n_heads, n_kv_heads, head_dim, qkv)
    _check_ints(qkv, seq_ids, positions, block_table)
    dev = qkv.get_device()
    if slabs is None:
        if bias is not None:
            _refuse("a bias is added to partial sums only")
    elif slabs.dtype is not torch.float32 or not slabs.is_contiguous() or slabs.shape[0] == 0 or slabs.data_ptr() % 8:
        _refuse("partial sums are contiguous float32 from an 8-byte boundary on")
    elif bias is not None and (bias.shape != (width,) or not bias.is_contiguous() or bias.get_device() != dev or
                               bias.dtype is not torch.bfloat16):
        _refuse(f"the bias is {width} bf16 numbers")
    pos = cos = sin = None
    s0 = s1 = rows = 0
    if rope is not None:
        pos, cos, sin, section = rope
        if pos.dtype is not torch.int32 or not pos.is_contiguous():
            pos = pos.to(torch.int32).contiguous()
        rows = 1 if pos.dim() == 1 else pos.shape[0]
        if pos.shape[-1] != T or pos.numel() != rows * T or rows not in (1, 3) or pos.get_device() != dev:
            _refuse(f"rope positions are [{T}] or [3, {T}]")
        table = cos.shape
        if len(table) != 2 or table[1] != head_dim // 2 or not table[0] or sin.shape != table or \
                cos.dtype is not torch.float32 or sin.dtype is not torch.float32 or not cos.is_contiguous() or \
                not sin.is_contiguous() or cos.get_device() != dev or sin.get_device() != dev:
            _refuse(f"cos and sin are contiguous float32 tables of width {head_dim // 2}")
        if rows == 3:
            if section is None or len(section) < 2:
                _refuse("positions of three axes come with the sections of the rotated pairs")
            s0, s1 = section[0], section[0] + section[1]
    if not qkv.is_cuda:
        if slabs is not None:
            qkv = slabs.sum(0) + (0 if bias is None else bias.float())
        x = qkv.float()
        if rope is not None:
            from . import reference as ref
            n = (n_heads + n_kv_heads) * head_dim
            turned = ref.rope(x[:, :n].reshape(T, n_heads + n_kv_heads, head_dim), pos if rows == 3 else pos.reshape(-1), cos,
                              sin, rope[3])
            x = torch.cat([turned.reshape(T, n), x[:, n:]], 1)
        _append_cpu(x[:, n_heads * head_dim:].reshape(T, 2, n_kv_heads, head_dim), seq_ids, positions, block_table, cache)
        if slabs is not None:
            return x.to(torch.bfloat16)
        if rope is not None:
            qkv.copy_(x)
        return qkv
    if dev != torch._C._cuda_getDevice():
        with torch.cuda.device(dev):
            return append(qkv, rope, seq_ids, positions, block_table, cache, n_heads, n_kv_heads, head_dim, bias)
    if slabs is not None:
        qkv = torch.empty(T, width, dtype=torch.bfloat16, device=slabs.device)
    stride, one = qkv.stride()
    if qkv.dtype is not torch.bfloat16 or one != 1 or stride % 2 or qkv.data_ptr() % 4 or stride < width and T > 1:
        _refuse("rows are bf16 numbers next to one another, from an even one on, and do not overlap")
    codes, scales = cache
    sequences, max_blocks = block_table.shape
    _lib.check(_lib.get_lib().sb_kv8_append(
        qkv.data_ptr(), stride, 0 if slabs is None else slabs.data_ptr(), T * width, 0 if slabs is None else slabs.shape[0],
        0 if bias is None else bias.data_ptr(), 0 if pos is None else pos.data_ptr(), rows, s0, s1, 0 if cos is None else table[0],
        0 if cos is None else cos.data_ptr(), 0 if sin is None else sin.data_ptr(), seq_ids.data_ptr(), positions.data_ptr(),
        block_table.data_ptr(), sequences, max_blocks, codes.data_ptr(), scales.data_ptr(), codes.shape[0], T, n_heads, n_kv_heads,
        head_dim, torch._C._cuda_getCurrentRawStream(dev)), "sb_kv8_append")
    return qkv


def copy_blocks(cache: Cache8, src: torch.Tensor, dst: torch.Tensor) -> None:
    """Blocks ``src[i]`` with their scales to ``dst[i]``; pairs that name no block are left out.  The destinations differ from one
    another and from all sources: pairs are copied at the same time."""
    codes, scales = cache
    heads = codes.shape[2] if codes.dim() == 5 else 0
    _check(cache, heads, heads, codes.shape[-1], codes)
    _check_ints(codes, src, dst)
    if src.shape != dst.shape or src.dim() != 1:
        _refuse("as many sources as destinations")
    if not codes.is_cuda:
        ok = (src >= 0) & (src < len(codes)) & (dst >= 0) & (dst < len(codes))
        src, dst = src[ok].long(), dst[ok].long()
        codes.view(torch.uint8)[dst] = codes.view(torch.uint8)[src]
        scales[dst] = scales[src]
        return
    with torch.cuda.device(codes.get_device()):
        _lib.check(_lib.get_lib().sb_kv8_copy_blocks(
            _lib.ptr(codes), _lib.ptr(scales), _lib.ptr(src), _lib.ptr(dst), src.numel(), codes.shape[0], 2 * codes.shape[2],
            ctypes.c_longlong(codes.shape[2:].numel() * 2), _lib.stream()), "sb_kv8_copy_blocks")


# ---- workspaces ---------------------------------------------------------------------------------
# Workspaces, and counters of pieces, which every call leaves as zeros: of each stream, whose kernels run one after the other,
# and of each stream of a capture, since a graph may be replayed beside anything.  A capture's are kept until the stream's next
# one, so that nothing else in the graph gets their memory, and its first call clears the counters in every replay.
# Threads may share a stream.  A launch for single tokens needs nothing of another one.  A call for chunks launches several kernels
# that hand data on through the workspace, which nobody else may write in between: it is the chunks' own, and their calls go to the
# library one at a time.
_buffers: dict = {}
_chunk_calls = threading.Lock()


def _workspace(dev: int, stream: int, floats: int, counts: int, use: str = "pieces"):
    capture = _lib.get_lib().sb_capture_id(stream) if torch._C._cuda_isCurrentStreamCapturing() else 0
    key = dev, stream, capture != 0, use
    held = _buffers.get(key)
    if held is None or held[2] != capture or held[0].numel() < floats or held[1].numel() < counts:
        more = (0, 0) if held is None or held[2] != capture else (held[0].numel(), held[1].numel())
        held = (torch.empty(max(floats, more[0]), dtype=torch.float32, device=f"cuda:{dev}"),
                torch.zeros(max(counts, more[1]), dtype=torch.int32, device=f"cuda:{dev}"), capture)
        _buffers[key] = held
    return held[:2]


# a kernel that gave up a wait may have left counters behind
_lib.on_status_error(_buffers.clear)


# ---- single tokens ------------------------------------------------------------------------------
def decode_attention(q_rows: torch.Tensor, cache: Cache8, seq_lens: torch.Tensor, block_table: torch.Tensor, n_heads: int,
                     n_kv_heads: int, head_dim: int, scale: Optional[float] = None,
                     out: Optional[torch.Tensor] = None) -> torch.Tensor:
    """:func:`siirl_b200.ops.kv_cache.decode_attention` on an 8-bit cache."""
    shape, width = q_rows.shape, n_heads * head_dim
    scale = scale if scale is not None else 1.0 / math.sqrt(head_dim)
    _check(cache, n_heads, n_kv_heads, head_dim, q_rows)
    _check_ints(q_rows, seq_lens, block_table)
    if len(shape) != 2 or shape[1] < width or q_rows.stride(1) != 1:
        _refuse(f"query rows are at least {width} wide")
    B, table = shape[0], block_table.shape
    if seq_lens.shape != (B,) or len(table) != 2 or table[0] < B or table[1] > TABLE:
        _refuse(f"a length and a row of the table, of at most {TABLE} blocks, for each of {B} rows")
    if out is None:
        out = torch.empty(B, width, dtype=q_rows.dtype, device=q_rows.device)
    elif out.shape != (B, width) or not out.is_contiguous() or out.dtype != q_rows.dtype or out.get_device() != q_rows.get_device():
        _refuse(f"the output is a contiguous [{B}, {width}] of the rows' type")
    if not q_rows.is_cuda:
        rep = n_heads // n_kv_heads
        out.zero_()
        for b in range(B):
            n = min(int(seq_lens[b]), BLOCK * block_table.shape[1])
            if n <= 0:
                continue
            x = cache.dequantize(block_table[b, :(n + BLOCK - 1) // BLOCK].long())
            k, v = (x[:, i].permute(1, 0, 2, 3).reshape(n_kv_heads, -1, head_dim)[:, :n].repeat_interleave(rep, 0) for i in (0, 1))
            s = torch.einsum("hd,hnd->hn", q_rows[b, :width].reshape(n_heads, head_dim).float(), k) * scale
            out[b] = torch.einsum("hn,hnd->hd", torch.softmax(s, -1), v).reshape(-1).to(out.dtype)
        return out
    if q_rows.dtype is not torch.bfloat16 or out.data_ptr() % 16:
        _refuse("query rows are bf16, and the output starts on a 16-byte boundary")
    if not table[1] or not cache.codes.shape[0]:
        return out.zero_()      # nothing to be seen
    dev = q_rows.get_device()
    if dev != torch._C._cuda_getDevice():
        with torch.cuda.device(dev):
            return decode_attention(q_rows, cache, seq_lens, block_table, n_heads, n_kv_heads, head_dim, scale, out)
    stride, q = q_rows.stride(0), q_rows.data_ptr()
    if stride % 2 or q % 4:      # contiguous rows may be the odd ones
        q_rows = q_rows[:, :width].clone(memory_format=torch.contiguous_format)
        stride, q = width, q_rows.data_ptr()
    L = _lib.get_lib()
    codes, scales = cache
    max_blocks = table[1]
    rows = 8 if n_heads <= 8 * n_kv_heads or head_dim == 64 else 16
    part = 2 * L.sb_kv8_decode_grid() * rows        # rows of partial results: two for each block of the grid
    entries = n_kv_heads * -(-(n_heads // n_kv_heads) // rows)
    stream = torch._C._cuda_getCurrentRawStream(dev)
    floats, counts = _workspace(dev, stream, part * (head_dim + 4), 4 * min(B, ROWS) * entries)
    for at in range(0, B, ROWS):
        n = min(ROWS, B - at)
        _lib.check(L.sb_kv8_decode(
            q + 2 * at * stride, stride, codes.data_ptr(), scales.data_ptr(), codes.shape[0],
            seq_lens.data_ptr() + 4 * at, block_table.data_ptr() + 4 * at * max_blocks, max_blocks,
            out.data_ptr() + 2 * at * width, floats.data_ptr(), floats.data_ptr() + 4 * part * head_dim, counts.data_ptr(), n,
            n_heads, n_kv_heads, head_dim, scale, _lib.status_word(q_rows.device).data_ptr(), stream), "sb_kv8_decode")
    return out


# ---- chunks of prompts --------------------------------------------------------------------------
def check_chunks(qkv: torch.Tensor, chunk_lens, prefix_lens, slots, cache: Cache8, block_table: torch.Tensor, n_heads: int,
                 n_kv_heads: int, head_dim: int) -> None:
    """Refuses chunks that the cache or the rows cannot hold."""
    _check(cache, n_heads, n_kv_heads, head_dim, qkv)
    _check_ints(qkv, block_table)
    if not len(chunk_lens) == len(prefix_lens) == len(slots):
        _refuse("a chunk, a prefix and a slot for each sequence")
    rows, width = sum(chunk_lens), (n_heads + 2 * n_kv_heads) * head_dim
    if qkv.shape != (rows, width):
        _refuse(f"{rows} rows of {width} numbers, got {tuple(qkv.shape)}")
    if block_table.dim() != 2 or block_table.shape[1] > TABLE:
        _refuse(f"a table of at most {TABLE} blocks for each sequence")
    slots_held, tokens_held = block_table.shape[0], block_table.shape[1] * BLOCK
    for c, p, s in zip(chunk_lens, prefix_lens, slots):
        if c < 0 or p < 0 or not 0 <= s < slots_held or c + p > tokens_held:
            _refuse(f"slot {s} of {slots_held} with {p} + {c} tokens of {tokens_held}")
    if qkv.is_cuda and qkv.dtype is not torch.bfloat16:
        _refuse("rows are bf16")


def chunk_attention(qkv: torch.Tensor, chunk_lens, prefix_lens, slots, cache: Cache8, block_table: torch.Tensor, n_heads: int,
                    n_kv_heads: int, head_dim: int) -> torch.Tensor:
    """:func:`siirl_b200.ops.kv_cache.prefill_attention_with_prefix` on an 8-bit cache, on the GPU.  The visible keys and values
    are unpacked to bf16 once per call: ``4 * Hkv * D`` bytes for every token up to the next multiple of 128, beside the
    output."""
    _check(cache, n_heads, n_kv_heads, head_dim, qkv)
    _check_ints(qkv, block_table)
    rows, width = qkv.shape
    lists = [array.array("i", v) for v in (chunk_lens, prefix_lens, slots)]
    total = len(lists[0])
    if width != (n_heads + 2 * n_kv_heads) * head_dim or qkv.dtype is not torch.bfloat16 or block_table.dim() != 2 or \
            block_table.shape[1] > TABLE or total != len(lists[1]) or total != len(lists[2]) or sum(lists[0]) != rows:
        check_chunks(qkv, *lists, cache, block_table, n_heads, n_kv_heads, head_dim)
    dev = qkv.get_device()
    if dev != torch._C._cuda_getDevice():
        with torch.cuda.device(dev):
            return chunk_attention(qkv, chunk_lens, prefix_lens, slots, cache, block_table, n_heads, n_kv_heads, head_dim)
    held, max_blocks = block_table.shape
    heads = n_heads * head_dim
    out = torch.empty(rows, heads, dtype=qkv.dtype, device=qkv.device)
    stride, one = qkv.stride()
    if one != 1 or stride % 8 or stride < width or qkv.data_ptr() % 16:
        qkv = qkv.clone(memory_format=torch.contiguous_format)      # contiguous rows may be the odd ones
        stride = qkv.shape[1]
    L = _lib.get_lib()
    most, at = L.sb_kv8_chunk_seqs(), 0
    sizes, stream = array.array("q", (0, 0, 0)), torch._C._cuda_getCurrentRawStream(dev)
    codes, scales = cache
    starts = [v.buffer_info()[0] for v in lists]
    with _chunk_calls:
        ws = _workspace(dev, stream, CHUNK_BYTES // 4, 0, "chunks")[0]
        for i in range(0, total, most):
            n = min(most, total - i)
            while True:
                rc = L.sb_kv8_chunks(
                    qkv.data_ptr() + 2 * at * stride, stride, rows - at, codes.data_ptr(), scales.data_ptr(), codes.shape[0],
                    block_table.data_ptr(), held, max_blocks, starts[0] + 4 * i, starts[1] + 4 * i, starts[2] + 4 * i, n,
                    ws.data_ptr(), 4 * ws.numel(), sizes.buffer_info()[0], out.data_ptr() + 2 * at * heads, n_heads, n_kv_heads,
                    head_dim, 1.0 / math.sqrt(head_dim), _lib.status_word(qkv.device).data_ptr(), stream)
                if rc != -6:
                    break
                ws = torch.empty(sizes[0] // 4, dtype=torch.float32, device=qkv.device)     # of the call's own
            if rc == -5:
                check_chunks(qkv, *lists, cache, block_table, n_heads, n_kv_heads, head_dim)
            _lib.check(rc, "sb_kv8_chunks")
            _lib.add_launches(sizes[2])
            at += sizes[1]
    return out
