// Attention of chunks of prompts against a paged cache of e4m3 codes (kv_cache8.cu): row i of a chunk behind a prefix of P
// tokens sees tokens 0 .. P + i.
//
// unpack8_kernel writes the visible tokens' keys and values once as bf16 rows [2, Hkv, rows, D] (code times scale, exact where
// the scale is a power of two), every sequence from a multiple of 128 rows on, zeros behind its last token.  It moves 5 bytes per
// cached number, against 4 * Hq / Hkv * chunk flops per number that the products take; converting in every block of the product
// kernel instead would cost it shared memory bandwidth, of which its operands take three quarters.  A code that is NaN is written
// as zero and its block of 64 rows marked: in a tile that some rows see in part, zero times a value that is NaN would reach rows
// before it.  The rows that do see it get their NaN at the end, from the codes.
//
// fmha_chunk_kernel: a block takes 128 rows of one kv head, a row being (position, query head of the kv head): heads that share
// keys share a block, so that short chunks fill it, too, and keys are fetched once for all of them.  For every 64 keys:
//   S = Q K_j^T      tcgen05.mma 128 x 64 x D -> TMEM, one of two places: the next scores are computed meanwhile
//   soft-max         one warpgroup, thread = row; weights (bf16) replace the scores in TMEM, in two halves, each handed to the
//                    products at once
//   O += P V_j       tcgen05.mma 128 x D x 64, P from TMEM, V through an MN-major descriptor
// Two blocks of an SM share its tensor cores: one computes weights while the other's products run.  (One block with two tiles of
// 128 keys each, which read a third less from shared memory: 2 sequences of up to 2148 rows, 32 / 8 heads, 740 us against 704, and
// more blocks that are not full.)
// The reference of a row's weights is raised only when its maximum grows by 2^8, so the output is rarely rescaled.
// The exponentials (16 a cycle and SM) take as long as the products, at D = 64 twice as long: every fourth pair, at D = 64 every
// second one, is computed on the fused-multiply-add units (2048 rows of one prompt, 28 / 4 heads: 155 us, 162 without; 4 sequences
// of up to 2000 rows, 14 / 2 heads, D = 64: 254, 266 without): 2^x = 2^n 2^f with n the nearest integer and a cubic in f,
// |f| <= 1/2, fitted for the smallest largest relative error (7.5e-5, a fiftieth of a bf16 step) by iteratively reweighted
// least squares.
// Bound by the tensor cores and the power limit: 2 sequences of up to 2148 rows behind up to 14,000 tokens: 704 us in short loops, 1.23
// PFLOP/s, 75 % of a library product's 1.64; 800 us in long ones, whose clock the limit lowers, 1.08 PFLOP/s, 78 % of its 1.39.
// Where there are few blocks, the key tiles are split over several, whose results chunk_merge_kernel joins.
#include <cuda_fp8.h>

#include <algorithm>

#include "common.cuh"
#include "launchers.h"

namespace sb {

constexpr int kChunkKeys = 64;       // keys of a tile
constexpr int kChunkCtas = 2;        // blocks of an SM
constexpr int kChunkSeqs = 48;       // sequences of one launch: what goes with it costs the host time

struct ChunkSeqs {
  int n, rows, tiles;                // rows: of the unpacked keys; tiles: of `span` positions, over all sequences
  int slot[kChunkSeqs], total[kChunkSeqs], prefix[kChunkSeqs];
  int q_row[kChunkSeqs];             // first row of the chunk
  int kv_row[kChunkSeqs], tile[kChunkSeqs];      // first unpacked row, first tile
};
// last i with first[i] <= x
__device__ __forceinline__ int find_seq(const int* first, int n, int x) {
  int lo = 0, hi = n;
  while (hi - lo > 1) {
    const int mid = (lo + hi) >> 1;
    if (first[mid] <= x) lo = mid;
    else hi = mid;
  }
  return lo;
}

__device__ __forceinline__ uint2 bf16_of(uint32_t codes, float scale) {
  const __half2_raw lo = __nv_cvt_fp8x2_to_halfraw2((__nv_fp8x2_storage_t)(codes & 0xffffu), __NV_E4M3);
  const __half2_raw hi = __nv_cvt_fp8x2_to_halfraw2((__nv_fp8x2_storage_t)(codes >> 16), __NV_E4M3);
  const float2 a = __half22float2(*reinterpret_cast<const __half2*>(&lo)), b = __half22float2(*reinterpret_cast<const __half2*>(&hi));
  return make_uint2(pack_bf16x2(a.x * scale, a.y * scale), pack_bf16x2(b.x * scale, b.y * scale));
}

// bytes of four codes: 0xff where one is NaN
__device__ __forceinline__ uint32_t nan_codes(uint32_t c) { return __vcmpeq4(c & 0x7f7f7f7fu, 0x7f7f7f7fu); }

// block x: 64 rows; block y: k and v heads; marks: [2 * Hkv, rows / 64]
template <int D>
__global__ void __launch_bounds__(256) unpack8_kernel(const __grid_constant__ ChunkSeqs q, const uint8_t* codes, const float* scales,
                                                      int num_blocks, const int* block_table, int max_blocks, int Hkv,
                                                      __nv_bfloat16* out, int* marks) {
  chain_sync();
  const int row = blockIdx.x * 64, i = find_seq(q.kv_row, q.n, row), t0 = row - q.kv_row[i], left = q.total[i] - t0;
  const int hd = blockIdx.y, kv = hd >= Hkv;
  int blk = left > 0 ? block_table[(size_t)q.slot[i] * max_blocks + t0 / 64] : -1;
  if (blk >= num_blocks) blk = -1;
  const size_t at = blk < 0 ? 0 : ((size_t)blk * 2 + kv) * Hkv + (hd - kv * Hkv);
  const float scale = blk < 0 ? 0.f : scales[at];
  const uint2* src = reinterpret_cast<const uint2*>(codes + at * 64 * D);
  uint4* dst = reinterpret_cast<uint4*>(out + ((size_t)hd * q.rows + row) * D);
  constexpr int N = D / 32;      // eight numbers at a time: a warp writes whole sectors
  uint2 c[N];
#pragma unroll
  for (int k = 0; k < N; ++k) {
    const int u = k * 256 + threadIdx.x;
    c[k] = blk >= 0 && u * 8 / D < left ? src[u] : make_uint2(0, 0);
  }
  uint32_t nan = 0;
#pragma unroll
  for (int k = 0; k < N; ++k) {
    const uint2 m = make_uint2(nan_codes(c[k].x), nan_codes(c[k].y));
    nan |= m.x | m.y;
    const uint2 p0 = bf16_of(c[k].x & ~m.x, scale), p1 = bf16_of(c[k].y & ~m.y, scale);
    dst[k * 256 + threadIdx.x] = make_uint4(p0.x, p0.y, p1.x, p1.y);
  }
  const int any = __syncthreads_or(nan != 0);
  if (threadIdx.x == 0) marks[hd * (q.rows / 64) + blockIdx.x] = any;
}

// NaN for a row of the output where it sees one, in a key for all columns: tokens t0 (a block's first) .. t1 - 1.  `codes`: of the key
// head in block 0, those of its values `values` further on; `marks`: of its block of t0 and those behind it, likewise
template <int D, typename T>
__device__ __noinline__ void mark_nan(const int* marks, int value_marks, const uint8_t* codes, size_t values, size_t block_bytes,
                                      const int* blocks, int t0, int t1, T* row) {
  for (int t = t0; t < t1; ++t) {
    const int key = marks[(t - t0) / 64], value = marks[value_marks + (t - t0) / 64];
    if (!key && !value) {
      t |= 63;
      continue;
    }
    const uint32_t* c = reinterpret_cast<const uint32_t*>(codes + blocks[t / 64] * block_bytes + t % 64 * D);
    uint32_t any = 0;
    for (int k = 0; key && k < D / 4; ++k) any |= nan_codes(c[k]);
    for (int k = 0; k < D / 4; ++k) {
      const uint32_t m = any ? 0xffffffffu : value ? nan_codes(c[values / 4 + k]) : 0u;
      for (int i = 0; m && i < 4; ++i)
        if (m >> (8 * i) & 1) row[4 * k + i] = T(__int_as_float(0x7fc00000));
    }
    if (any) return;
  }
}

struct ChunkParams {
  __nv_bfloat16* out;      // [chunk rows, Hq * D]
  float* ws_o;             // [tile, kv head, split, query tile, 128, D], where splits > 1
  float* ws_lse;           // [.., 128]
  const int* marks;        // unpack8_kernel's
  const uint8_t* codes;
  const int* block_table;
  int max_blocks;
  int Hq, Hkv, rep, span, splits;      // span: positions of 128 rows
  float scale_log2;
  int* status;
};

template <int D>
struct ChunkSmem {
  static constexpr int kQBytes = 128 * D * 2, kKvBytes = kChunkKeys * D * 2;
  static constexpr int kStages = 4;
  static constexpr int kBarOff = kQBytes + kStages * kKvBytes;  // q, s_full[2], p_full[2][2], o_full, o_step, full[], empty[]
  static constexpr int kTotal = kBarOff + (9 + 2 * kStages) * 8 + 16;
};

// the larger one, NaN where one is NaN
__device__ __forceinline__ float max_nan(float a, float b) {
  float y;
  asm("max.NaN.f32 %0, %1, %2;" : "=f"(y) : "f"(a), "f"(b));
  return y;
}
// two of 2^x: see above.  0 from -127 down: a weight of what a row does not see times a large value would be seen.  NaN stays NaN
__device__ __forceinline__ float2 poly_exp2(float2 x) {
  x.x = max_nan(x.x, -127.f);
  x.y = max_nan(x.y, -127.f);
  const float2 big = make_float2(12582912.f, 12582912.f), small = make_float2(-12582912.f, -12582912.f);      // 1.5 * 2^23
  const float2 t = add_f32x2(x, big), n = add_f32x2(t, small), minus = make_float2(-1.f, -1.f);
  const float2 f = fma_f32x2(n, minus, x);
  float2 p = fma_f32x2(f, make_float2(0.0551716817f, 0.0551716817f), make_float2(0.24261115979f, 0.24261115979f));
  p = fma_f32x2(p, f, make_float2(0.69326098678f, 0.69326098678f));
  p = fma_f32x2(p, f, make_float2(0.99992807130f, 0.99992807130f));
  return mul_f32x2(p, make_float2(__int_as_float(0x3f800000 + (__float_as_int(t.x) << 23)), __int_as_float(0x3f800000 + (__float_as_int(t.y) << 23))));
}

// One thread's MMAs, of operands whose descriptors have the high word of 128-byte swizzle and 1024 bytes between groups of eight
// rows.  A in shared memory, and in TMEM
constexpr uint32_t kDescHigh = (1024u >> 4) | 1u << 14 | 2u << 29;
__device__ __forceinline__ void umma_bf16_ss_lo(uint32_t tmem_d, uint32_t a_lo, uint32_t b_lo, uint32_t idesc, uint32_t accumulate) {
  asm volatile(
      "{\n\t.reg .pred p;\n\t.reg .b64 a, b;\n\t"
      "mov.b64 a, {%1, %4};\n\tmov.b64 b, {%2, %4};\n\t"
      "setp.ne.b32 p, %5, 0;\n\t"
      "tcgen05.mma.cta_group::1.kind::f16 [%0], a, b, %3, p;\n\t}"
      ::"r"(tmem_d), "r"(a_lo), "r"(b_lo), "r"(idesc), "r"(kDescHigh), "r"(accumulate)
      : "memory");
}
__device__ __forceinline__ void umma_bf16_ts_lo(uint32_t tmem_d, uint32_t tmem_a, uint32_t b_lo, uint32_t idesc, uint32_t accumulate) {
  asm volatile(
      "{\n\t.reg .pred p;\n\t.reg .b64 b;\n\t"
      "mov.b64 b, {%2, %4};\n\t"
      "setp.ne.b32 p, %5, 0;\n\t"
      "tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], b, %3, p;\n\t}"
      ::"r"(tmem_d), "r"(tmem_a), "r"(b_lo), "r"(idesc), "r"(kDescHigh), "r"(accumulate)
      : "memory");
}

// Four warps for the soft-max (thread = row), then one for TMA and the MMA issuer.
template <int D>
__global__ void __launch_bounds__(192, kChunkCtas)
fmha_chunk_kernel(const __grid_constant__ CUtensorMap map_q, const __grid_constant__ CUtensorMap map_kv,
                  const __grid_constant__ ChunkSeqs seqs, ChunkParams p) {
  using L = ChunkSmem<D>;
  constexpr int KV = kChunkKeys, kDChunks = D / 64, kStages = L::kStages, kTmaWarp = 4, kMmaWarp = 5;
  constexpr uint32_t kTmemCols = 256;      // two places of scores, then the output
  extern __shared__ __align__(1024) uint8_t smem_raw[];
  uint8_t* smem = smem_raw;
  if (smem_u32(smem) & 1023u) {
    if (threadIdx.x == 0) atomicCAS(p.status, 0, (int)kStatusBadArgument);
    return;
  }
  uint8_t* sQ = smem;
  uint8_t* ring = smem + L::kQBytes;
  uint64_t* bar_q = reinterpret_cast<uint64_t*>(smem + L::kBarOff);
  uint64_t* s_full = bar_q + 1;                                      // [place] scores are in TMEM
  uint64_t* p_full = bar_q + 3;                                      // [place][2] halves of the weights have replaced the scores
  uint64_t* o_full = bar_q + 7;                                      // the output is complete
  uint64_t* o_step = bar_q + 8;                                      // it has the products of one more tile
  uint64_t* full = bar_q + 9;                                        // [kStages] ring of K and V tiles
  uint64_t* empty = full + kStages;
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(empty + kStages);
  int* s_nan = reinterpret_cast<int*>(tmem_slot + 1);

  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  if (tid == 0) {
    tma_prefetch_desc(&map_q);
    tma_prefetch_desc(&map_kv);
    for (int i = 0; i < 9; ++i) mbar_init(&bar_q[i], i >= 3 && i < 7 ? 4 : 1);
    for (int i = 0; i < 2 * kStages; ++i) mbar_init(&full[i], 1);
    fence_barrier_init();
  }
  if (warp == kMmaWarp) {
    tmem_alloc(tmem_slot, kTmemCols);
    tmem_relinquish();
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem_base = *tmem_slot;
  chain_sync();
  // block -> (tile, kv head, share of the keys); a sequence's last tiles, which see most, first
  const int split = (int)(blockIdx.x % p.splits), g = (int)(blockIdx.x / p.splits % p.Hkv);
  const int tile = (int)(blockIdx.x / p.splits / p.Hkv), seq = find_seq(seqs.tile, seqs.n, tile);
  const int prefix = seqs.prefix[seq], total = seqs.total[seq];
  const int tile_end = seq + 1 < seqs.n ? seqs.tile[seq + 1] : seqs.tiles;
  const int c0 = (tile_end - 1 - tile) * p.span, first = prefix + c0;      // first position, in the chunk and in the sequence
  const int all = (min(first + p.span, total) + KV - 1) / KV;
  const int j0 = (int)((long long)all * split / p.splits), n = (int)((long long)all * (split + 1) / p.splits) - j0;      // key tiles
  const int* marks = p.marks + g * (seqs.rows / 64) + (seqs.kv_row[seq] + j0 * KV) / 64;

  if (warp == kTmaWarp) {
    // ------------------------------ TMA producer ------------------------------
    if (lane == 0 && n > 0) {
      const int k_row = g * seqs.rows + seqs.kv_row[seq] + j0 * KV, v_row = k_row + p.Hkv * seqs.rows;
      mbar_arrive_expect_tx(bar_q, (uint32_t)(kDChunks * p.rep * p.span * 128));
#pragma unroll
      for (int c = 0; c < kDChunks; ++c) tma_load_3d(sQ + c * 16384, &map_q, bar_q, c * 64, g * p.rep, seqs.q_row[seq] + c0);
      int i = 0;
      for (; i < 2 * n; ++i) {  // K0 V0 K1 V1 ...
        const int st = i % kStages;
        if (!mbar_wait(&empty[st], ((i / kStages) & 1) ^ 1, p.status, kStatusTimeoutProducer)) break;
        uint8_t* dst = ring + st * L::kKvBytes;
        const int row = ((i & 1) ? v_row : k_row) + (i >> 1) * KV;
        mbar_arrive_expect_tx(&full[st], L::kKvBytes);
#pragma unroll
        for (int c = 0; c < kDChunks; ++c) tma_load_2d(dst + c * (KV * 128), &map_kv, &full[st], c * 64, row);
      }
      if (i < 2 * n) {  // gave up: no copy may land in shared memory that has been handed on
        mbar_wait(bar_q, 0, nullptr, 0);
        for (int k = max(0, i - kStages); k < i; ++k) mbar_wait(&full[k % kStages], (k / kStages) & 1, nullptr, 0);
      }
    }
    // while the last tiles are worked on: whether one of the keys and values is NaN
    __syncwarp();
    int any = 0;
    for (int i = lane; i < n * (KV / 64); i += 32) any |= marks[i] | marks[p.Hkv * (seqs.rows / 64) + i];
    any = __any_sync(0xffffffffu, any);
    if (lane == 0) *s_nan = any;
  } else if (warp == kMmaWarp) {
    // ------------------------------ MMA issuer: one thread ------------------------------
    // The soft-max warps leave it few issue slots: descriptors differ in their low words only, which are kept and stepped
    if (elect_one()) {
      constexpr uint32_t idesc_s = umma_idesc_bf16(128, KV, 0, 0);
      constexpr uint32_t idesc_o = umma_idesc_bf16(128, D, 0, 1);
      constexpr uint32_t kStep = L::kKvBytes >> 4;
      const uint32_t q_lo = (uint32_t)umma_smem_desc(smem_u32(sQ), 16, 1024), k_lo = (uint32_t)umma_smem_desc(smem_u32(ring), 16, 1024);
      const uint32_t v_lo = (uint32_t)umma_smem_desc(smem_u32(ring), KV * 128, 1024);
      auto wait = [&](uint64_t* bar, uint32_t parity) { return mbar_wait(bar, parity, p.status, kStatusTimeoutMma); };
      auto scores = [&](int place, int stage) {
        const uint32_t b = k_lo + stage * kStep;
#pragma unroll
        for (int kk = 0; kk < D / 16; ++kk)
          umma_bf16_ss_lo(tmem_base + place * KV, q_lo + (kk / 4) * 1024 + (kk % 4) * 2, b + (kk / 4) * (KV * 8) + (kk % 4) * 2, idesc_s, kk > 0);
        umma_commit(&s_full[place]);
        umma_commit(&empty[stage]);
      };
      auto products = [&](int place, int stage, int parity, bool first) {
        const uint32_t v = v_lo + stage * kStep;
#pragma unroll
        for (int part = 0; part < 2; ++part) {
          if (!wait(&p_full[2 * place + part], parity)) return false;
          tc_fence_after();
#pragma unroll
          for (int k = 0; k < KV / 32; ++k) {
            const int kk = part * (KV / 32) + k;
            umma_bf16_ts_lo(tmem_base + 2 * KV, tmem_base + place * KV + kk * 8, v + kk * 128, idesc_o, kk > 0 || !first);
          }
        }
        umma_commit(&empty[stage]);
        return true;
      };
      int ks = 0, vs = 1;                  // ring places of K_j and V_j
      uint32_t k_phase = 0, v_phase = 0;
      auto step = [&](int& at, uint32_t& phase) {
        at += 2;
        if (at >= kStages) {
          at -= kStages;
          phase ^= 1;
        }
      };
      bool ok = n > 0 && wait(bar_q, 0) && wait(&full[0], 0);
      tc_fence_after();
      if (ok) scores(0, 0);
      for (int j = 0; j < n && ok; ++j) {
        step(ks, k_phase);
        const bool more = j + 1 < n;
        if (more) ok = wait(&full[ks], k_phase);
        if (more && ok) scores(j + 1 & 1, ks);
        ok = ok && wait(&full[vs], v_phase) && products(j & 1, vs, j >> 1 & 1, j == 0);
        if (!ok) break;
        umma_commit(more ? o_step : o_full);
        step(vs, v_phase);
      }
    }
    __syncwarp();
  } else {
    // ------------------------------ softmax and output: thread = row ------------------------------
    const int row = tid, at = row / p.rep, head = row - at * p.rep;
    const uint32_t lane_off = (uint32_t)(warp * 32) << 16, tmem_o = tmem_base + lane_off + 2 * KV;
    const int qpos = first + at;      // position within the sequence
    // Of a row of the tile that is none of the chunk's, shared memory has other numbers, which rows of its warp must not feel: their
    // references are raised together
    const bool row_valid = at < p.span && qpos < total;
    const float sc = p.scale_log2;
    float m_ref = -INFINITY;          // reference of the weights, scaled
    float2 l_run[2] = {make_float2(0.f, 0.f), make_float2(0.f, 0.f)};
    bool ok = true;
    for (int j = 0; j < n; ++j) {
      const int place = j & 1;
      const uint32_t tmem_s = tmem_base + lane_off + place * KV;
      ok = __all_sync(0xffffffffu, mbar_wait(&s_full[place], j >> 1 & 1, p.status, kStatusTimeoutEpilogue));
      if (!ok) break;
      tc_fence_after();
      uint32_t s[KV / 32][32];
#pragma unroll
      for (int c = 0; c < KV / 32; ++c) tmem_ld_32x32(tmem_s + c * 32, s[c]);
      tmem_ld_wait();
      const int kv0 = (j0 + j) * KV;
      if (kv0 + KV - 1 > first) {
        const int visible = min(qpos + 1, total) - kv0;
#pragma unroll
        for (int i = 0; i < KV; ++i)
          if (i >= visible) s[i / 32][i % 32] = 0xff800000u;  // -inf
      }
      float mx[4] = {-INFINITY, -INFINITY, -INFINITY, -INFINITY};
#pragma unroll
      for (int i = 0; i < KV; ++i) mx[i & 3] = fmaxf(mx[i & 3], __uint_as_float(s[i / 32][i % 32]));
      const float top = row_valid ? fmaxf(fmaxf(mx[0], mx[1]), fmaxf(mx[2], mx[3])) * sc : -INFINITY;
      if (__any_sync(0xffffffffu, top > m_ref + 8.f)) {
        // The barrier of the scores also said that the products of the tile before the last one are done: o_step is at most one
        // phase behind
        if (j > 0) {
          ok = __all_sync(0xffffffffu, mbar_wait(o_step, j - 1 & 1, p.status, kStatusTimeoutEpilogue));
          if (!ok) break;
          tc_fence_after();
        }
        const float m_new = fmaxf(m_ref, top), alpha = fast_exp2(m_ref - (m_new == -INFINITY ? 0.f : m_new));
        m_ref = m_new;
#pragma unroll
        for (int i = 0; i < 2; ++i) {
          l_run[i].x *= alpha;
          l_run[i].y *= alpha;
        }
        if (j > 0) {
#pragma unroll 1
          for (int c = 0; c < D / 8; ++c) {      // few columns at a time: the scores hold most registers
            uint32_t r[8];
            tmem_ld_32x8(tmem_o + c * 8, r);
            tmem_ld_wait();
#pragma unroll
            for (int i = 0; i < 8; ++i) r[i] = __float_as_uint(__uint_as_float(r[i]) * alpha);
            tmem_st_32x8(tmem_o + c * 8, r);
          }
        }
      }
      const float ref = m_ref == -INFINITY ? 0.f : m_ref;
      const float2 sc2 = make_float2(sc, sc), neg = make_float2(-ref, -ref);
#pragma unroll
      for (int part = 0; part < 2; ++part) {
#pragma unroll
        for (int i0 = part * (KV / 2); i0 < (part + 1) * (KV / 2); i0 += 32) {
          uint32_t pk[16];
#pragma unroll
          for (int i = i0; i < i0 + 32; i += 2) {
            float2 x = make_float2(__uint_as_float(s[i / 32][i % 32]), __uint_as_float(s[i / 32][i % 32 + 1]));
            x = fma_f32x2(x, sc2, neg);
            if (i % 8 == 6 || D == 64 && i % 8 == 2) {
              x = poly_exp2(x);
            } else {
              x.x = fast_exp2(x.x);
              x.y = fast_exp2(x.y);
            }
            l_run[i / 2 & 1] = add_f32x2(l_run[i / 2 & 1], x);
            pk[(i - i0) / 2] = pack_bf16x2(x.x, x.y);
          }
          tmem_st_32x16(tmem_s + i0 / 2, pk);
        }
        tmem_st_wait();
        tc_fence_before();
        __syncwarp();
        if (lane == 0) mbar_arrive(&p_full[2 * place + part]);
      }
    }
    if (ok && n > 0) ok = __all_sync(0xffffffffu, mbar_wait(o_full, 0, p.status, kStatusTimeoutEpilogue));
    // ---- O / l -> bf16, or the share's normalised result (TMEM loads are warp-collective; only the stores are predicated) ----
    if (ok) {
      tc_fence_after();
      // 0: all scores are -inf, of a share's keys that the row does not see, or of all its keys, where 0 / 0 is soft-max's answer.
      // Scores that are NaN do not raise the reference, but make the sum NaN
      const float l = (l_run[0].x + l_run[0].y) + (l_run[1].x + l_run[1].y), inv_l = 1.f / l;
      const size_t part = (((size_t)tile * p.Hkv + g) * p.splits + split) * 128 + row;
      const size_t out_row = (size_t)seqs.q_row[seq] + (row_valid ? qpos - prefix : 0);
      __nv_bfloat16* orow = p.out + out_row * (size_t)(p.Hq * D) + (size_t)(g * p.rep + head) * D;
      if (n > 0) {
#pragma unroll 1
        for (int c = 0; c < D / 32; ++c) {
          uint32_t r[32];
          tmem_ld_32x32(tmem_o + c * 32, r);
          tmem_ld_wait();
          if (!row_valid) continue;
          if (p.splits > 1) {
            float4* wrow = reinterpret_cast<float4*>(p.ws_o + part * D + c * 32);
#pragma unroll
            for (int q = 0; q < 8; ++q)
              wrow[q] = make_float4(__uint_as_float(r[4 * q]) * inv_l, __uint_as_float(r[4 * q + 1]) * inv_l,
                                    __uint_as_float(r[4 * q + 2]) * inv_l, __uint_as_float(r[4 * q + 3]) * inv_l);
          } else {
#pragma unroll
            for (int q = 0; q < 4; ++q) {
              uint4 o;
              o.x = pack_bf16x2(__uint_as_float(r[q * 8 + 0]) * inv_l, __uint_as_float(r[q * 8 + 1]) * inv_l);
              o.y = pack_bf16x2(__uint_as_float(r[q * 8 + 2]) * inv_l, __uint_as_float(r[q * 8 + 3]) * inv_l);
              o.z = pack_bf16x2(__uint_as_float(r[q * 8 + 4]) * inv_l, __uint_as_float(r[q * 8 + 5]) * inv_l);
              o.w = pack_bf16x2(__uint_as_float(r[q * 8 + 6]) * inv_l, __uint_as_float(r[q * 8 + 7]) * inv_l);
              *reinterpret_cast<uint4*>(orow + c * 32 + q * 8) = o;
            }
          }
        }
      }
      if (p.splits > 1 && row_valid) p.ws_lse[part] = l == 0.f ? -INFINITY : l != l ? l : m_ref + log2f(l);
    }
  }
  tc_fence_before();
  __syncthreads();
  if (warp == kMmaWarp) {
    tc_fence_after();
    tmem_dealloc(tmem_base, kTmemCols);
  }
  if (*s_nan && warp < kTmaWarp) {      // over what the thread has written
    const int row = tid, at = row / p.rep, qpos = first + at, t0 = j0 * KV, t1 = min(qpos + 1, t0 + n * KV);
    if (at < p.span && qpos < total) {
      const size_t values = (size_t)p.Hkv * 64 * D, part = (((size_t)tile * p.Hkv + g) * p.splits + split) * 128 + row;
      const uint8_t* codes = p.codes + (size_t)g * 64 * D;
      const int* blocks = p.block_table + (size_t)seqs.slot[seq] * p.max_blocks;
      const int more = p.Hkv * (seqs.rows / 64);
      if (p.splits > 1)
        mark_nan<D>(marks, more, codes, values, 2 * values, blocks, t0, t1, p.ws_o + part * D);
      else
        mark_nan<D>(marks, more, codes, values, 2 * values, blocks, t0, t1,
                    p.out + ((size_t)seqs.q_row[seq] + qpos - prefix) * (p.Hq * D) + (size_t)(g * p.rep + row - at * p.rep) * D);
    }
  }
}

// Mean of the shares' results, weighted by 2^(log-sum-exp).  A block takes 16 rows, half a warp each: first the largest weight,
// then all shares at once, so that their reads are under way together.
template <int D>
__global__ void __launch_bounds__(256) chunk_merge_kernel(const __grid_constant__ ChunkSeqs seqs, ChunkParams p) {
  chain_sync();
  const int unit = blockIdx.x / 8, row = blockIdx.x % 8 * 16 + (threadIdx.x >> 4), l = threadIdx.x & 15;
  const int g = unit % p.Hkv, tile = unit / p.Hkv, seq = find_seq(seqs.tile, seqs.n, tile);
  const int tile_end = seq + 1 < seqs.n ? seqs.tile[seq + 1] : seqs.tiles;
  const int at = row / p.rep, pos = (tile_end - 1 - tile) * p.span + at;
  if (at >= p.span || pos >= seqs.total[seq] - seqs.prefix[seq]) return;
  constexpr int N = D / 64;      // groups of four columns of a lane
  const size_t first = (size_t)unit * p.splits * 128 + row, step = 128;
  float top = -INFINITY, sum = 0.f;
  for (int s = 0; s < p.splits; ++s) top = fmaxf(top, p.ws_lse[first + s * step]);
  float4 acc[N] = {};
#pragma unroll 8
  for (int s = 0; s < p.splits; ++s) {
    const float lse = p.ws_lse[first + s * step];
    const bool there = lse != -INFINITY;      // else its share may not have been written
    const float e = there ? exp2f(lse - top) : 0.f;
    sum += e;
#pragma unroll
    for (int k = 0; k < N; ++k) {
      float4 o = make_float4(0.f, 0.f, 0.f, 0.f);
      if (there) o = *reinterpret_cast<const float4*>(p.ws_o + (first + s * step) * D + (k * 16 + l) * 4);
      acc[k].x += e * o.x; acc[k].y += e * o.y; acc[k].z += e * o.z; acc[k].w += e * o.w;
    }
  }
  const float inv = 1.f / sum;      // every row sees a token: a sum of 0 is one of scores that are all -inf, and the result NaN
  __nv_bfloat16* out = p.out + (size_t)(seqs.q_row[seq] + pos) * (p.Hq * D) + (size_t)(g * p.rep + row - at * p.rep) * D;
#pragma unroll
  for (int k = 0; k < N; ++k)
    *reinterpret_cast<uint2*>(out + (k * 16 + l) * 4) =
        make_uint2(pack_bf16x2(acc[k].x * inv, acc[k].y * inv), pack_bf16x2(acc[k].z * inv, acc[k].w * inv));
}

// What a call does, from the host's lists alone
struct ChunkPlan {
  ChunkSeqs s;
  int span, splits;
};
// 16-bit numbers of the unpacked keys and values, and of the marks behind them
static long long unpacked(const ChunkPlan& c, int Hkv, int D) { return 2ll * Hkv * c.s.rows * D; }
static long long marks_of(const ChunkPlan& c, int Hkv) { return ((long long)Hkv * (c.s.rows / 32) + 3) / 4 * 8; }
static int make_chunk_plan(ChunkPlan& c, const int* chunk, const int* prefix, const int* slot, int n, int Hq, int Hkv, int D) {
  const int rep = Hq / Hkv;
  c.span = 128 / rep;
  int order[kChunkSeqs], first[kChunkSeqs];
  long long rows = 0, positions = 0;
  int live = 0;
  for (int i = 0; i < n; ++i) {
    first[i] = (int)positions;
    positions += chunk[i];
    if (chunk[i] > 0) order[live++] = i;
  }
  // those that see most first
  std::sort(order, order + live, [&](int a, int b) { return prefix[a] + chunk[a] > prefix[b] + chunk[b]; });
  c.s.n = live;
  int tiles = 0, longest = 0;
  long long all = 0;      // tiles of keys that the tiles of positions walk over
  for (int k = 0; k < live; ++k) {
    const int i = order[k], total = prefix[i] + chunk[i];
    c.s.slot[k] = slot[i]; c.s.total[k] = total; c.s.prefix[k] = prefix[i]; c.s.q_row[k] = first[i];
    c.s.kv_row[k] = (int)rows; c.s.tile[k] = tiles;
    rows += (total + 127) / 128 * 128;
    const int rows_of = (chunk[i] + c.span - 1) / c.span;
    tiles += rows_of;
    all += rows_of * ((prefix[i] + chunk[i] / 2) / (long long)kChunkKeys + 1);
    longest = std::max(longest, (total + kChunkKeys - 1) / kChunkKeys);
    if (rows * 2 * Hkv > 0x7fffffffll) return -4;
  }
  c.s.rows = (int)rows;
  c.s.tiles = tiles;
  // Shares of the keys: each costs its blocks about what twelve tiles of keys do (results in 32 bits, written and read), and spares
  // the last blocks to run alone.  In tiles:
  const long long blocks = (long long)tiles * Hkv, room = (long long)num_sms() * kChunkCtas;
  c.splits = 1;
  float best = 3.0e38f;
  for (int s = 1; s <= 16 && s <= std::max(1, longest / 8); ++s) {
    const float waves = (float)(blocks * s) / room, share = (float)longest / s;
    const float time = (waves <= 1.f ? share : (float)all * Hkv / room + 0.5f * share) + (s > 1 ? 12.f * std::max(1.f, waves) + 6.f : 0.f);
    if (time < best) {
      best = time;
      c.splits = s;
    }
  }
  if (blocks * c.splits > 0x7fffffffll / 32) return -4;
  return 0;
}

template <int D>
static int launch_chunk(const CUtensorMap& mq, const CUtensorMap& mkv, const ChunkPlan& c, const ChunkParams& p, cudaStream_t stream) {
  using L = ChunkSmem<D>;
  auto kernel = fmha_chunk_kernel<D>;
  static int configured = -1;
  int dev = 0;
  cudaGetDevice(&dev);
  if (configured != dev) {
    cudaError_t e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, L::kTotal);
    if (e != cudaSuccess) return (int)e;
    configured = dev;
  }
  const unsigned blocks = (unsigned)(c.s.tiles * p.Hkv * c.splits);
  const int rc = launch_chained(kernel, blocks, 192, L::kTotal, stream, mq, mkv, c.s, p);
  if (rc || c.splits == 1) return rc;
  return launch_chained(chunk_merge_kernel<D>, (unsigned)(c.s.tiles * p.Hkv * 8), 256, 0, stream, c.s, p);
}

}  // namespace sb

using namespace sb;

extern "C" int sb_kv8_chunk_seqs() { return kChunkSeqs; }

// Chunks of n sequences, at most kChunkSeqs, one behind the other in `qkv` (q heads first, row_stride apart), whose keys and values
// are in the cache.  The lists are the host's.  sizes[0]: bytes that the workspace has to have (16-byte aligned), sizes[1]: rows of
// the chunks, sizes[2]: kernels launched.  -5: chunks that `rows` rows, or a table of `slots` rows of `max_blocks` blocks, cannot
// hold; -6: the workspace is too small, and nothing has been launched.
extern "C" int sb_kv8_chunks(const void* qkv, long long row_stride, int rows, const void* codes, const float* scales, int num_blocks,
                             const int* block_table, int slots, int max_blocks, const int* chunk, const int* prefix, const int* slot,
                             int n, void* ws, long long ws_bytes, long long* sizes, void* out, int Hq, int Hkv, int D, float scale,
                             int* status, cudaStream_t stream) {
  sizes[0] = sizes[1] = sizes[2] = 0;
  if (D != 64 && D != 128) return -2;
  if (max_blocks > 1 << 24) return -4;      // lengths, rounded up to tiles: 32 bits
  if (n > kChunkSeqs || Hq % Hkv || Hq / Hkv > 32 || row_stride % 8 || reinterpret_cast<uintptr_t>(qkv) % 16 || !(scale > 0.f)) return -3;
  long long sum = 0;
  for (int i = 0; i < n; ++i) {
    if (chunk[i] < 0 || prefix[i] < 0 || slot[i] < 0 || slot[i] >= slots || (long long)prefix[i] + chunk[i] > max_blocks * 64ll) return -5;
    sum += chunk[i];
  }
  if (sum > rows) return -5;
  sizes[1] = sum;
  ChunkPlan c;
  int r = make_chunk_plan(c, chunk, prefix, slot, n, Hq, Hkv, D);
  if (r || c.s.tiles == 0) return r;
  // unpacked keys and values, marks, results of shares
  const long long kv_bytes = 2 * unpacked(c, Hkv, D), marks_bytes = 2 * marks_of(c, Hkv);
  const long long parts = c.splits > 1 ? (long long)c.s.tiles * Hkv * c.splits * 128 : 0;
  sizes[0] = kv_bytes + marks_bytes + parts * (D + 1) * 4;
  if (sizes[0] > ws_bytes) return -6;
  bind_context();
  CUtensorMap mq, mkv;
  r = make_tensor_map_bf16_3d(&mq, qkv, D, Hq, sum, D, row_stride, 64, Hq / Hkv, c.span);
  if (r) return r;
  r = make_tensor_map_bf16_2d(&mkv, ws, D, 2ll * Hkv * c.s.rows, D, 64, kChunkKeys);
  if (r) return r;
  int* marks = reinterpret_cast<int*>((char*)ws + kv_bytes);
  r = launch_chained(D == 128 ? unpack8_kernel<128> : unpack8_kernel<64>, dim3(c.s.rows / 64, 2 * Hkv), 256, 0, stream, c.s,
                     (const uint8_t*)codes, scales, num_blocks, block_table, max_blocks, Hkv, (__nv_bfloat16*)ws, marks);
  if (r) return r;
  ChunkParams p;
  p.out = (__nv_bfloat16*)out; p.ws_o = reinterpret_cast<float*>((char*)ws + kv_bytes + marks_bytes);
  p.ws_lse = p.ws_o + parts * D;
  sizes[2] = c.splits > 1 ? 3 : 2;
  p.marks = marks; p.codes = (const uint8_t*)codes; p.block_table = block_table; p.max_blocks = max_blocks;
  p.Hq = Hq; p.Hkv = Hkv; p.rep = Hq / Hkv; p.span = c.span; p.splits = c.splits;
  p.scale_log2 = scale * 1.4426950408889634f; p.status = status;
  return D == 128 ? launch_chunk<128>(mq, mkv, c, p, stream) : launch_chunk<64>(mq, mkv, c, p, stream);
}
