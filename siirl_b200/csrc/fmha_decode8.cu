// Single-token attention against a paged cache of e4m3 codes (kv_cache8.cu), on the 8-bit tensor cores.
//
// o = sum_t softmax(scale q . k_t)_t v_t with k_t = ks * code, v_t = vs * code, one ks and vs per cache block and head.  Both
// products run on codes as they lie in the cache: nothing is converted on the way.  What meets the codes is split instead, into
// 8-bit terms that are columns of one product and are added up afterwards:
//   * a query row, divided by a power of two, into two e4m3 terms, the second 16 times enlarged: 4 + 4 bits hold all that a bf16
//     number has, down to 2^-22 of the row's largest;
//   * a weight into three e5m2 terms, each remainder 16 times enlarged: off by at most 2^-11 of itself or 2^-36 of the largest
//     weight.  e5m2 for its range: thousands of small weights may stand beside one large one whose value is near zero.
// The block's scales go into the score and into the weight, in 32 bits.  So a block with a large scale and small codes would take
// the weights' range from the others: a piece whose blocks' value scales are more than 2^16 apart (those below 2^-60 aside) is
// computed again in 32 bits by the output warps (d8_exact), at 20 to 30 us for 32 tokens: a call takes a hundred times as long, also
// where only one sequence needs it, whose heads are one CTA's (256 x 1300-5120, 28 / 4 heads: 14.4 ms with one block of one sequence,
// 18.4 with one of each, 135 us without; 8 x 20001-32768, 32 / 8: 8.4, 8.8 and 0.074 ms).
//
// A tile is 128 rows of 128 bytes: two cache blocks at D = 128; at D = 64, where a row holds two tokens, four.
//   S^T[row, (token of the row, term, head)] = K Q^T     A = the K tile, B = the terms of all query heads of a kv head
//   O^T[byte of a row, (token of the row, term, head)] += V^T W^T    A = the V tile, B = the weights' terms, a tile row's side by
//                                                        side as its thread writes them, both through MN-major descriptors
// The tile fills the 128 rows of the MMA whatever the number of heads, and shared memory is read once per product.  At D = 64
// only the diagonal (token of the row) blocks of O^T mean something; the query terms of the other token's half are zeros.
//
// The tiles of all (sequence, kv head, group of at most NR query heads) form one list, and every CTA of a persistent grid of
// one CTA per SM takes an equal range of it.  A range is a few pieces, each a run of tiles of one entry.  A piece that is not
// the whole entry leaves a normalised result and its log-sum-exp in a workspace, two slots per CTA, and counts itself; whoever
// finds that all others have joins them.  A second kernel for that would cost the host as much again as this one.
// Up to 32 sequences, if there are few tiles, are cut instead into pieces of at most so many tiles that each CTA gets one: a second
// piece costs a CTA about 1.6 us, a join 3, a tile 0.7 (28 / 4 heads, 300 tokens: 7.2 us whole, 11.0 in equal ranges; 32 x 1000: 11.4
// and 15.3).  32, as a warp's lanes take a sequence each, not because more would not gain: 33 x 300 take 14.4 us where 32 take 8.8,
// 33 x 1000 16.4 and 12.4.
// The warps:
//   0..7   soft-max in two groups, each with an O^T and weights' references of its own.  D = 128: thread = row of the tile, the
//          first four warps take the even tiles of the range, the others the odd ones, so that two tiles are under way.
//          D = 64: the groups take the first and the second tokens of every tile's rows.  A vote of the group per tile says
//          whether a reference has to be raised (a weight above 2^14; a fresh one puts the largest weight at 2^11)
//   8..11  output: joins the two O^T of a piece while the next piece's tiles are under way (double-buffered)
//   12     producer: a ring of K and V tiles, ids and scales of the next 32 cache blocks of the list in registers
//   13, 14 MMA issuers: scores; weighted sums
//   15     query terms of the next pieces
#include <cuda_fp8.h>

#include "common.cuh"
#include "launchers.h"

namespace sb {

constexpr int kQ8Rows = 1024;        // sequences of one launch
constexpr int kQ8Smem = 227 * 1024;
constexpr int kQ8MinTiles = 2;       // tiles of a range, where there are so few that not every SM gets as many
constexpr float kQ8Spread = 16.f, kQ8Low = -60.f;      // log2 of value scales: apart, and of those that do not count
constexpr float kQ8None = -3.0e38f;  // reference before anything has been seen

// mbar_wait() with all but the first look in one place: sixteen warps run seven programs here, and what each of them takes of the
// instruction cache counts
__device__ __noinline__ bool bar_wait_on(uint64_t* bar, uint32_t parity, int* status, int code) {
  return mbar_wait(bar, parity, status, code);
}
__device__ __forceinline__ bool bar_wait(uint64_t* bar, uint32_t parity, int* status, int code) {
  return mbar_try_wait(bar, parity) || bar_wait_on(bar, parity, status, code);
}

__device__ __forceinline__ void umma_e4m3_ss_if(uint32_t leader, uint32_t tmem_d, uint64_t desc_a, uint64_t desc_b,
                                                uint32_t idesc, uint32_t accumulate) {
  asm volatile(
      "{\n\t.reg .pred p, q;\n\t"
      "setp.ne.b32 p, %4, 0;\n\t"
      "setp.ne.b32 q, %5, 0;\n\t"
      "@q tcgen05.mma.cta_group::1.kind::f8f6f4 [%0], %1, %2, %3, p;\n\t}"
      ::"r"(tmem_d), "l"(desc_a), "l"(desc_b), "r"(idesc), "r"(accumulate), "r"(leader)
      : "memory");
}
// kind::f8f6f4 with e4m3 operands, or B in e5m2, and fp32 accumulation
__host__ __device__ constexpr uint32_t umma_idesc_e4m3(int m, int n, int a_mn, int b_mn, int b_e5m2) {
  return (1u << 4) | ((uint32_t)b_e5m2 << 10) | ((uint32_t)a_mn << 15) | ((uint32_t)b_mn << 16) | ((uint32_t)(n >> 3) << 17) | ((uint32_t)(m >> 4) << 24);
}
// descriptor of an MN-major tile whose rows have 32 or 64 bytes: 32- or 64-byte swizzle, groups of eight rows one behind the other
__device__ __forceinline__ uint64_t umma_desc_rows(uint32_t smem_addr, int row_bytes) {
  return (uint64_t)((smem_addr & 0x3FFFF) >> 4) | (uint64_t)1 << 16 | (uint64_t)(row_bytes * 8 >> 4) << 32 | (uint64_t)1 << 46 |
         (uint64_t)(row_bytes == 32 ? 6 : 4) << 61;
}
// largest of a warp
__device__ __forceinline__ float redux_max(float x) {
  float y;
  asm volatile("redux.sync.max.f32 %0, %1, 0xffffffff;" : "=f"(y) : "f"(x));
  return y;
}
// whether `any` is set in one of the 128 threads of four soft-max warps
__device__ __forceinline__ bool vote_128(int group, bool any) {
  uint32_t r;
  asm volatile(
      "{\n\t.reg .pred p, q;\n\t"
      "setp.ne.b32 p, %1, 0;\n\t"
      "barrier.cta.red.or.pred q, %2, 128, p;\n\t"
      "selp.u32 %0, 1, 0, q;\n\t}"
      : "=r"(r)
      : "r"((uint32_t)any), "r"(1 + group)
      : "memory");
  return r != 0;
}
__device__ __forceinline__ uint32_t e4m3x2(float a, float b) {
  return (uint32_t)__nv_cvt_float2_to_fp8x2(make_float2(a, b), __NV_SATFINITE, __NV_E4M3);
}
__device__ __forceinline__ float2 from_e4m3x2(uint32_t codes) {
  const __half2_raw h = __nv_cvt_fp8x2_to_halfraw2((__nv_fp8x2_storage_t)codes, __NV_E4M3);
  return __half22float2(*reinterpret_cast<const __half2*>(&h));
}

__device__ __forceinline__ uint32_t e5m2x2(float a, float b) {
  return (uint32_t)__nv_cvt_float2_to_fp8x2(make_float2(a, b), __NV_SATFINITE, __NV_E5M2);
}
__device__ __forceinline__ float2 from_e5m2x2(uint32_t codes) {
  const __half2_raw h = __nv_cvt_fp8x2_to_halfraw2((__nv_fp8x2_storage_t)codes, __NV_E5M2);
  return __half22float2(*reinterpret_cast<const __half2*>(&h));
}

struct Decode8Params {
  const __nv_bfloat16* q;   // [B, row_stride], q heads first
  long long row_stride;
  const uint8_t* codes;     // [num_blocks, 2, Hkv, 64, D]
  const float* scales;      // [num_blocks, 2, Hkv]
  const int* seq_lens;      // [B]
  const int* block_table;   // [B, max_blocks]
  int num_blocks, max_blocks, B, Hq, Hkv, groups;
  __nv_bfloat16* out;       // [B, Hq * D]
  float* ws_o;              // [2 * grid][NR][D]
  float* ws_lse;            // [2 * grid][4][NR]: each output warp's own
  int* counts;              // [B * entries][4] pieces that have been left, zeros before and after
  float scale_log2;
  int* status;
};

// NR: query heads of a group (rows of a piece), 8 or, at D = 128, 16
template <int D, int NR>
struct D8 {
  static constexpr int PACK = 128 / D;             // tokens of a 128-byte row
  static constexpr int RPB = 64 / PACK;            // rows of a cache block
  static constexpr int BPT = 2 * PACK;             // cache blocks of a tile
  static constexpr int TT = 64 * BPT;              // tokens of a tile
  static constexpr int NS = PACK * 2 * NR;         // columns of S^T
  static constexpr int NO = PACK * 4 * NR;         // columns of O^T, bytes of a row of the weights' terms: 32 or 64, the last
                                                   // quarter of a token's unused
  static constexpr int NQ = NS <= 32 ? 4 : 2;      // query buffers
  static constexpr int kQBytes = NS * 128, kPBytes = NO * 128, kStage = 32768;
  static constexpr int kXBytes = PACK == 2 ? 64 * NR * 4 : 0; // the second tokens' share of a result
  static constexpr int kFixed = NQ * kQBytes + 2 * kPBytes + kXBytes + (2 * kQ8Rows + 1 + 32) * 4 + 4096;
  static constexpr int kStages = (kQ8Smem - kFixed) / kStage < 6 ? (kQ8Smem - kFixed) / kStage : 6;
  static constexpr int kQOff = kStages * kStage, kPOff = kQOff + NQ * kQBytes, kXOff = kPOff + 2 * kPBytes;
  static constexpr int kBlockOff = kXOff + kXBytes;                    // [stages][BPT] {ks, log2 vs, visible tokens}
  static constexpr int kPieceOff = kBlockOff + kStages * BPT * 16;     // [NQ] {sequence, entry, first tile, tiles}
  static constexpr int kRedOff = kPieceOff + NQ * 16;                  // [2 groups][4][NR] {max z, max z + log2 vs}
  static constexpr int kStatOff = kRedOff + 2 * 4 * NR * 8;            // [2 buffers][2 groups]: l [4][NR], m [NR], M [NR]
  static constexpr int kSpreadOff = kStatOff + 4 * 6 * NR * 4;         // [2 buffers][8 warps] {least, largest log2 vs} of the piece
  static constexpr int kFactorOff = kSpreadOff + 16 * 8;               // [NQ][NR] factor of the scores
  static constexpr int kBarOff = kFactorOff + NQ * NR * 4;
  static constexpr int kBars = 3 * kStages + 2 * NQ + 14;
  static constexpr int kPreOff = kBarOff + kBars * 8 + 24;
  static constexpr int kTotal = kPreOff + (2 * kQ8Rows + 1 + 32) * 4;
  // TMEM columns: S^T of two tiles, O^T of two pieces
  static constexpr int kTmemS = 0, kTmemO = 2 * NS;
  static constexpr int kOBuffer = (3 - PACK) * NO;                     // columns of O^T of a piece: each group's own
  static constexpr int kTmemCols = 2 * (NS + kOBuffer) <= 256 ? 256 : 512;
};

struct D8Piece {
  int row, entry, t0, n, tiles;    // entry: kv head * groups + group
};
// the piece at list position `cur` of a range that ends at `end`; pre[b] = tiles of one entry of the sequences before b
__device__ __forceinline__ D8Piece d8_piece(const int* pre, int B, int entries, int cur, int end) {
  int lo = 0, hi = B;       // the last sequence that begins at or before cur (those without tiles have no width)
  while (hi - lo > 1) {
    const int mid = (lo + hi) >> 1;
    if (pre[mid] * entries <= cur) lo = mid;
    else hi = mid;
  }
  D8Piece q;
  q.row = lo;
  q.tiles = pre[lo + 1] - pre[lo];
  const int at = cur - pre[lo] * entries;
  q.entry = at / q.tiles;
  q.t0 = at - q.entry * q.tiles;
  q.n = min(q.tiles - q.t0, end - cur);
  return q;
}
// the piece behind q, which begins at `cur` < end
__device__ __forceinline__ void d8_next(const int* pre, int entries, D8Piece& q, int cur, int end) {
  q.t0 = 0;
  if (++q.entry == entries) {
    q.entry = 0;
    do q.tiles = pre[q.row + 2] - pre[q.row + 1];
    while (++q.row, q.tiles == 0);
  }
  q.n = min(q.tiles, end - cur);
}
// ranges of the list, and the first position of one
__device__ __forceinline__ int d8_ranges(int total, int grid) { return min(grid, max(1, total / kQ8MinTiles)); }
__device__ __forceinline__ int d8_begin(int total, int cta, int ranges) { return (int)((long long)total * min(cta, ranges) / ranges); }

// At most 32 sequences, one for each lane of a warp, of `tiles` tiles, `sum` up to the lane's: if there are few, what this CTA takes
// in mine[0 .. 3]: list positions from, to; number of its piece, pieces of that entry.  Else mine[0] = -1.
__device__ __noinline__ void d8_alone(int tiles, int sum, int entries, int* mine) {
  const int lane = threadIdx.x & 31, grid = gridDim.x, cta = blockIdx.x;
  const int most = __reduce_max_sync(0xffffffffu, tiles), all = __shfl_sync(0xffffffffu, sum, 31);
  // the fewest tiles of a piece with which there are enough CTAs; whole entries, where they are short
  int r = most <= 4 ? most : 2;
  while (r > 0 && r <= 16 && (long long)__reduce_add_sync(0xffffffffu, (tiles + r - 1) / r) * entries > grid) r += r < 4 ? 1 : r < 8 ? 2 : 4;
  if (r == 0 || r > 16 || r > (long long)all * entries / grid + 4) {
    if (lane == 0) mine[0] = -1;
    return;
  }
  const int pieces = (tiles + r - 1) / r;
  int upto = pieces;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const int u = __shfl_up_sync(0xffffffffu, upto, o);
    if (lane >= o) upto += u;
  }
  const int before = (upto - pieces) * entries;
  if (pieces && before <= cta && cta < upto * entries) {
    const int e = (cta - before) / pieces, k = (cta - before) % pieces, first = (sum - tiles) * entries + e * tiles;
    mine[0] = first + k * tiles / pieces;
    mine[1] = first + (k + 1) * tiles / pieces;
    mine[2] = k;
    mine[3] = pieces;
  }
  if (lane == 31 && cta >= upto * entries) mine[0] = mine[1] = 0;
}

template <int N>
__device__ __forceinline__ void tmem_ld_heads(uint32_t taddr, uint32_t (&r)[N]) {
  if constexpr (N == 8) tmem_ld_32x8(taddr, r);
  else tmem_ld_32x16(taddr, r);
}
template <int N>
__device__ __forceinline__ void tmem_st_heads(uint32_t taddr, const uint32_t (&r)[N]) {
  if constexpr (N == 8) tmem_st_32x8(taddr, r);
  else tmem_st_32x16(taddr, r);
}

// a query row times the first D codes of row r of a K tile, in 32 bits
template <int D>
__device__ __noinline__ float d8_dot(const __nv_bfloat16* q, const uint8_t* k, int r) {
  float s = 0.f;
#pragma unroll 1
  for (int d = 0; d < D; ++d) s = fmaf(__bfloat162float(q[d]), from_e4m3x2(k[(((d >> 4) ^ (r & 7)) << 4) + (d & 15)]).x, s);
  return s;
}

// A warp has left its columns of one of the pieces of an entry, which CTAs c0 .. c1 have (c0 in its slot `own`).  If it is the last
// one: mean of all, weighted by 2^(log-sum-exp), to the output.  `parts` and `lses` point at the lane's column and the warp's
// sums of slot 0.
template <int D, int NR>
__device__ __noinline__ void d8_join(const float* parts, const float* lses, int* count, int c0, int c1, int own, int heads,
                                     __nv_bfloat16* orow) {
  __threadfence();      // what this lane has written, before the warp counts
  __syncwarp();
  int before = 0;
  const bool one = (threadIdx.x & 31) == 0;
  if (one) before = atomicAdd(count, 1);
  if (__shfl_sync(0xffffffffu, before, 0) != c1 - c0) return;
  __threadfence();
  if (one) *count = 0;
  constexpr int U = 16 / NR;      // pieces whose reads are under way together
  float top[NR], sum[NR], acc[NR];
#pragma unroll
  for (int h = 0; h < NR; ++h) {
    top[h] = -INFINITY;
    sum[h] = acc[h] = 0.f;
  }
#pragma unroll 1
  for (int c = c0; c <= c1; c += U) {
    float o[U][NR], lse[U][NR];
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const size_t slot = 2 * min(c + u, c1) + (c + u == c0 ? own : 0);
#pragma unroll
      for (int h = 0; h < NR; ++h) {
        o[u][h] = h < heads ? __ldcg(parts + (slot * NR + h) * D) : 0.f;
        lse[u][h] = c + u <= c1 ? __ldcg(lses + slot * 4 * NR + h) : -INFINITY;
      }
    }
#pragma unroll
    for (int h = 0; h < NR; ++h) {
      float now = top[h];
#pragma unroll
      for (int u = 0; u < U; ++u) now = fmaxf(now, lse[u][h]);
      const float f = top[h] == -INFINITY ? 0.f : fast_exp2(top[h] - now);
      sum[h] *= f;
      acc[h] *= f;
#pragma unroll
      for (int u = 0; u < U; ++u) {
        const float e = lse[u][h] == -INFINITY ? 0.f : fast_exp2(lse[u][h] - now);
        sum[h] += e;
        acc[h] += e == 0.f ? 0.f : e * o[u][h];
      }
      top[h] = now;
    }
  }
#pragma unroll
  for (int h = 0; h < NR; ++h)
    if (h < heads) orow[h * D] = __float2bfloat16(sum[h] == 0.f ? 0.f : acc[h] / sum[h]);
}

// Tokens t0 .. t1 - 1 of a kv head for `heads` query rows in 32 bits, by one warp: o[h] of column d, lse of the lane's head.
// A lane takes the scores of every 32nd token, and column d of the weighted sum.
template <int D, int NR>
__device__ __noinline__ void d8_exact(const __nv_bfloat16* q, int heads, const uint8_t* codes, const float* scales, const int* blocks,
                                      int num_blocks, int Hkv, int kv_head, int t0, int t1, float scale_log2, int d, float (&o)[NR],
                                      float& lse) {
  const int lane = threadIdx.x & 31;
  lse = -INFINITY;
  float m[NR], l[NR], w[NR], acc[NR];
#pragma unroll
  for (int h = 0; h < NR; ++h) {
    m[h] = kQ8None;
    l[h] = acc[h] = 0.f;
  }
#pragma unroll 1
  for (int base = t0; base < t1; base += 32) {
    const int t = base + lane;
    int id = t < t1 ? blocks[t / 64] : -1;
    if (id >= num_blocks) id = -1;
    const size_t at = id < 0 ? 0 : (size_t)id * 2 * Hkv + kv_head;
    const uint32_t* k = reinterpret_cast<const uint32_t*>(codes + (at * 64 + t % 64) * D);
    const float vs = id < 0 ? 0.f : scales[at + Hkv];
#pragma unroll
    for (int h = 0; h < NR; ++h) w[h] = 0.f;
    if (id >= 0) {
#pragma unroll 1
      for (int c = 0; c < D / 4; ++c) {
        const uint32_t x = k[c];
        const float2 a = from_e4m3x2(x & 0xffffu), b = from_e4m3x2(x >> 16);
#pragma unroll
        for (int h = 0; h < NR; ++h)
          if (h < heads) {
            const __nv_bfloat162* r = reinterpret_cast<const __nv_bfloat162*>(q + h * D + 4 * c);
            const float2 e = __bfloat1622float2(r[0]), f = __bfloat1622float2(r[1]);
            w[h] = fmaf(e.x, a.x, fmaf(e.y, a.y, fmaf(f.x, b.x, fmaf(f.y, b.y, w[h]))));
          }
      }
    }
    const float ks = id < 0 ? 0.f : scales[at] * scale_log2;
#pragma unroll
    for (int h = 0; h < NR; ++h) {
      const float z = id < 0 ? -INFINITY : w[h] * ks, now = fmaxf(m[h], redux_max(z)), f = fast_exp2(m[h] - now);
      w[h] = fast_exp2(z - now);
      l[h] = fmaf(l[h], f, w[h]);      // of the lane's tokens
      acc[h] *= f;
      m[h] = now;
    }
#pragma unroll 1
    for (int j = 0; j < 32 && base + j < t1; ++j) {
      const int block = __shfl_sync(0xffffffffu, id, j);
      const float s = __shfl_sync(0xffffffffu, vs, j);
      if (block < 0) continue;
      const float v = s * from_e4m3x2(codes[(((size_t)block * 2 + 1) * Hkv + kv_head) * 64 * D + (size_t)((base + j) % 64) * D + d]).x;
#pragma unroll
      for (int h = 0; h < NR; ++h) acc[h] = fmaf(__shfl_sync(0xffffffffu, w[h], j), v, acc[h]);
    }
  }
#pragma unroll
  for (int h = 0; h < NR; ++h) {
#pragma unroll
    for (int i = 16; i > 0; i >>= 1) l[h] += __shfl_xor_sync(0xffffffffu, l[h], i);
    o[h] = l[h] == 0.f ? 0.f : acc[h] / l[h];
    if (lane == h) lse = l[h] == 0.f ? -INFINITY : m[h] + log2f(l[h]);
  }
}

constexpr int kQ8Threads = 16 * 32;

template <int D, int NR>
__global__ void __launch_bounds__(kQ8Threads, 1) fmha_decode8_kernel(const __grid_constant__ CUtensorMap map_c, Decode8Params p) {
  using L = D8<D, NR>;
  constexpr int PACK = L::PACK, NST = L::kStages, BPT = L::BPT, NQ = L::NQ;
  extern __shared__ __align__(1024) uint8_t smem_raw[];
  uint8_t* smem = smem_raw;
  if (smem_u32(smem) & 1023u) {
    if (threadIdx.x == 0) atomicCAS(p.status, 0, (int)kStatusBadArgument);
    return;
  }
  uint8_t *sQ = smem + L::kQOff, *sP = smem + L::kPOff;
  float* s_x = reinterpret_cast<float*>(smem + L::kXOff);
  float4* s_block = reinterpret_cast<float4*>(smem + L::kBlockOff);
  int4* s_piece = reinterpret_cast<int4*>(smem + L::kPieceOff);
  float2* s_red = reinterpret_cast<float2*>(smem + L::kRedOff);
  float* s_stat = reinterpret_cast<float*>(smem + L::kStatOff);
  float2* s_spread = reinterpret_cast<float2*>(smem + L::kSpreadOff);
  float* s_factor = reinterpret_cast<float*>(smem + L::kFactorOff);
  uint64_t* k_full = reinterpret_cast<uint64_t*>(smem + L::kBarOff);
  uint64_t* v_full = k_full + NST;
  uint64_t* kv_empty = v_full + NST;
  uint64_t* q_full = kv_empty + NST;    // [NQ]
  uint64_t* q_empty = q_full + NQ;
  uint64_t* s_full = q_empty + NQ;      // pairs from here on
  uint64_t* s_empty = s_full + 2;
  uint64_t* p_full = s_empty + 2;
  uint64_t* p_empty = p_full + 2;
  uint64_t* o_full = p_empty + 2;       // the piece's MMAs have completed, its statistics are there
  uint64_t* o_empty = o_full + 2;       // the output warps have read O^T and the statistics
  uint64_t* x_full = o_empty + 2;       // second tokens' share
  uint64_t* x_empty = x_full + 1;
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(x_empty + 1);
  volatile int* s_fail = reinterpret_cast<volatile int*>(tmem_slot + 1);   // [4]: by group and vote of a tile
  int* s_pre = reinterpret_cast<int*>(smem + L::kPreOff);
  int* s_tot = s_pre + kQ8Rows + 1;
  int* s_len = s_tot + 32;
  int* s_mine = s_tot + 4;      // where a single total is there: what d8_alone() writes

  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  const int entries = p.Hkv * p.groups, rep = p.Hq / p.Hkv, per_group = (rep + p.groups - 1) / p.groups;
  // of an entry: kv head, first query head, query heads
  auto kv_head = [&](int entry) { return p.groups == 1 ? entry : entry / p.groups; };
  auto group_of = [&](int entry) { return p.groups == 1 ? 0 : entry % p.groups; };
  auto first_head = [&](int entry) { return kv_head(entry) * rep + group_of(entry) * per_group; };
  auto heads_of = [&](int entry) { return min(per_group, rep - group_of(entry) * per_group); };
  if (tid == 0) {
    tma_prefetch_desc(&map_c);
    for (int i = 0; i < 3 * NST; ++i) mbar_init(&k_full[i], 1);
    for (int i = 0; i < NQ; ++i) {
      mbar_init(&q_full[i], 1);
      mbar_init(&q_empty[i], 9);     // the MMAs, the soft-max warps
    }
    for (int i = 0; i < 2; ++i) {
      mbar_init(&s_full[i], 1);
      mbar_init(&s_empty[i], 4 * PACK);
      mbar_init(&p_full[i], 4 * PACK);
      mbar_init(&p_empty[i], 1);
      mbar_init(&o_full[i], 9);      // the MMAs, the statistics of the soft-max warps
      mbar_init(&o_empty[i], 4);
    }
    mbar_init(x_full, 2);
    mbar_init(x_empty, 2);
    for (int i = 0; i < 4; ++i) s_fail[i] = 0;
    fence_barrier_init();
  }
  if (warp == 13) {
    tmem_alloc(tmem_slot, L::kTmemCols);
    tmem_relinquish();
  }
  if (NR == 16)      // the unused quarters
    for (int i = tid; i < 2 * L::kPBytes / 16; i += kQ8Threads) reinterpret_cast<uint4*>(sP)[i] = make_uint4(0, 0, 0, 0);
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem_base = *tmem_slot;
  chain_sync();
  // running sum of the sequences' tiles: chunks of 32 by warp, then their totals
  const int chunks = (p.B + 31) / 32;
  for (int c = warp; c < chunks; c += kQ8Threads / 32) {
    const int b = c * 32 + lane, n = b < p.B ? min(max(p.seq_lens[b], 0), p.max_blocks * 64) : 0;
    int v = (n + L::TT - 1) / L::TT;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const int u = __shfl_up_sync(0xffffffffu, v, o);
      if (lane >= o) v += u;
    }
    if (b < p.B) {
      s_len[b] = n;
      s_pre[b + 1] = v;
    }
    if (lane == 31) s_tot[c] = v;
    if (p.B <= 32) d8_alone((n + L::TT - 1) / L::TT, v, entries, s_mine);
  }
  if (tid == 0) s_pre[0] = 0;
  __syncthreads();
  if (chunks > 1) {
    for (int c = warp; c < chunks; c += kQ8Threads / 32) {
      const int before = __reduce_add_sync(0xffffffffu, lane < c ? s_tot[lane] : 0);      // at most 32 chunks
      const int b = c * 32 + lane;
      if (b < p.B) s_pre[b + 1] += before;
    }
    __syncthreads();
  }
  const int total = s_pre[p.B] * entries, ranges = d8_ranges(total, gridDim.x);
  const bool alone = p.B <= 32 && s_mine[0] >= 0;
  const int begin = alone ? s_mine[0] : d8_begin(total, blockIdx.x, ranges);
  const int end = alone ? s_mine[1] : d8_begin(total, blockIdx.x + 1, ranges);

  if (warp == 12) {
    // ------------------------------ producer ------------------------------
    // lane i: cache block i % BPT of the tile i / BPT places on in the list
    constexpr int kAhead = 32 / BPT;
    struct Block {
      int id, head, left;      // left: tokens of the sequence from this block on
      float ks, vs;
    };
    auto find = [&](int at) {
      Block x = {-1, 0, 0, 0.f, 0.f};
      const int cur = at + lane / BPT;
      if (cur >= end) return x;
      const D8Piece q = d8_piece(s_pre, p.B, entries, cur, end);
      const int j = q.t0 * BPT + lane % BPT;
      x.head = kv_head(q.entry);
      x.left = s_len[q.row] - j * 64;
      if (x.left > 0) x.id = p.block_table[(size_t)q.row * p.max_blocks + j];
      return x;
    };
    auto scales = [&](Block& x) {
      if (x.id < 0 || x.id >= p.num_blocks) return;
      const float* s = p.scales + (size_t)x.id * 2 * p.Hkv + x.head;
      x.ks = s[0];
      x.vs = s[p.Hkv];
    };
    uint32_t tile_no = 0;
    bool ok = true;
    Block x = find(begin), y = x;
    scales(x);
    for (int at = begin; at < end && ok; at += kAhead) {
      const int n = min(kAhead, end - at);
      const int seen = x.id >= 0 && x.id < p.num_blocks ? min(x.left, 64) : 0;
      for (int k = 0; k < n; ++k, ++tile_no) {
        const int stage = tile_no % NST;
        if (!__all_sync(0xffffffffu, bar_wait(&kv_empty[stage], ((tile_no / NST) & 1) ^ 1, p.status, kStatusTimeoutProducer))) {
          ok = false;
          break;
        }
        const bool mine = lane / BPT == k;
        const uint32_t bytes = __popc(__ballot_sync(0xffffffffu, mine && seen)) * (uint32_t)(L::RPB * 128);
        const int part = lane % BPT;
        if (mine && seen) {
          uint8_t* dst = smem + stage * L::kStage + part * (L::RPB * 128);
          const int row = (x.id * 2 * p.Hkv + x.head) * L::RPB;
          tma_load_2d(dst, &map_c, &k_full[stage], 0, row);
          tma_load_2d(dst + 16384, &map_c, &v_full[stage], 0, row + p.Hkv * L::RPB);
        }
        if (mine) s_block[stage * BPT + part] = make_float4(x.ks, seen ? __log2f(x.vs) : 0.f, __int_as_float(seen), 0.f);
        __syncwarp();
        if (lane == 0) {      // the copies may be there already: a phase ends with its arrival
          mbar_arrive_expect_tx(&k_full[stage], bytes);
          mbar_arrive_expect_tx(&v_full[stage], bytes);
        }
        if (k == 0) y = find(at + kAhead);
        if (k == n / 2) scales(y);
      }
      x = y;
    }
    if (!ok) {      // no copy may be in flight when shared memory is given back
      const uint32_t first = tile_no > (uint32_t)NST ? tile_no - NST : 0;
      for (uint32_t j = first; j < tile_no; ++j) {
        bar_wait(&k_full[j % NST], (j / NST) & 1, nullptr, 0);
        bar_wait(&v_full[j % NST], (j / NST) & 1, nullptr, 0);
      }
    }
  } else if (warp == 13) {
    // ------------------------------ scores (the whole warp, converged; one lane issues) ------------------------------
    const uint32_t leader = elect_one() ? 1u : 0u;
    constexpr uint32_t idesc = umma_idesc_e4m3(128, L::NS, 0, 0, 0);
    const uint64_t dk = umma_smem_desc(smem_u32(smem), 16, 1024), dq = umma_smem_desc(smem_u32(sQ), 16, 1024);
    uint32_t piece_no = 0;
    int left = 0, stage = 0;
    uint32_t phase = 0;
    bool ok = true;
    auto wait = [&](uint64_t* bar, uint32_t parity) {
      return __all_sync(0xffffffffu, bar_wait(bar, parity, p.status, kStatusTimeoutMma)) != 0;
    };
    for (int i = 0; i < end - begin && ok; ++i) {
      const uint32_t b = i & 1, iq = piece_no % NQ;
      if (left == 0) {
        ok = wait(&q_full[iq], (piece_no / NQ) & 1);
        left = s_piece[iq].w;
      }
      ok = ok && wait(&s_empty[b], ((i >> 1) & 1) ^ 1) && wait(&k_full[stage], phase);
      if (!ok) break;
      tc_fence_after();
#pragma unroll
      for (int kk = 0; kk < 4; ++kk)
        umma_e4m3_ss_if(leader, tmem_base + L::kTmemS + b * L::NS, dk + (uint32_t)stage * (L::kStage >> 4) + 2 * kk,
                        dq + iq * (L::kQBytes >> 4) + 2 * kk, idesc, kk ? 1u : 0u);
      umma_commit_if(leader, &s_full[b]);
      if (--left == 0) {
        umma_commit_if(leader, &q_empty[iq]);
        ++piece_no;
      }
      if (++stage == NST) {
        stage = 0;
        phase ^= 1;
      }
    }
  } else if (warp == 14) {
    // ------------------------------ weighted sums ------------------------------
    const uint32_t leader = elect_one() ? 1u : 0u;
    constexpr uint32_t idesc = umma_idesc_e4m3(128, L::NO, 1, 1, 1);
    const uint64_t dv = umma_smem_desc(smem_u32(smem) + 16384, 16384, 1024), dp = umma_desc_rows(smem_u32(sP), L::NO);
    uint32_t piece_no = 0, fresh = 3;      // fresh: parts of the piece's O^T that nothing has been added to
    int stage = 0;
    uint32_t phase = 0;
    bool ok = true;
    auto wait = [&](uint64_t* bar, uint32_t parity) {
      return __all_sync(0xffffffffu, bar_wait(bar, parity, p.status, kStatusTimeoutMma)) != 0;
    };
    D8Piece q;
    if (begin < end) q = d8_piece(s_pre, p.B, entries, begin, end);
    int left = 0;
    for (int i = 0; i < end - begin && ok; ++i) {
      const uint32_t b = i & 1, ib = piece_no & 1;
      if (left == 0) {
        if (i) d8_next(s_pre, entries, q, begin + i, end);
        left = __shfl_sync(0xffffffffu, q.n, 0);
        ok = wait(&o_empty[ib], ((piece_no >> 1) & 1) ^ 1);
      }
      ok = ok && wait(&v_full[stage], phase) && wait(&p_full[b], (i >> 1) & 1);
      if (!ok) break;
      tc_fence_after();
      const uint32_t part = PACK == 1 ? b : 0, add = ~fresh >> part & 1;
#pragma unroll
      for (int kk = 0; kk < 4; ++kk)
        umma_e4m3_ss_if(leader, tmem_base + L::kTmemO + ib * L::kOBuffer + part * L::NO, dv + (uint32_t)stage * (L::kStage >> 4) + 256 * kk,
                        dp + b * (L::kPBytes >> 4) + kk * (32 * L::NO >> 4), idesc, kk ? 1u : add);
      umma_commit_if(leader, &kv_empty[stage]);
      umma_commit_if(leader, &p_empty[b]);
      fresh &= ~(1u << part);
      if (--left == 0) {
        umma_commit_if(leader, &o_full[ib]);
        ++piece_no;
        fresh = 3;
      }
      if (++stage == NST) {
        stage = 0;
        phase ^= 1;
      }
    }
  } else if (warp == 15) {
    // ------------------------------ query terms; the next piece's rows are asked for first ------------------------------
    constexpr int E = D / 32;       // elements of a lane
    auto load = [&](const D8Piece& q, uint32_t (&raw)[NR][E / 2]) {
      const int left = heads_of(q.entry);
      const __nv_bfloat16* src = p.q + (size_t)q.row * p.row_stride + (size_t)first_head(q.entry) * D + lane * E;
#pragma unroll
      for (int r = 0; r < NR; ++r)
#pragma unroll
        for (int e = 0; e < E / 2; ++e) raw[r][e] = r < left ? *reinterpret_cast<const uint32_t*>(src + (size_t)r * D + 2 * e) : 0u;
    };
    uint32_t piece_no = 0, raw[NR][E / 2], ahead[NR][E / 2];
    D8Piece q, next;
    if (begin < end) {
      q = d8_piece(s_pre, p.B, entries, begin, end);
      load(q, raw);
    }
    for (int cur = begin; cur < end; ++piece_no) {
      cur += q.n;
      if (cur < end) {
        next = q;
        d8_next(s_pre, entries, next, cur, end);
        load(next, ahead);
      }
      const int iq = piece_no % NQ;
      if (!__all_sync(0xffffffffu, bar_wait(&q_empty[iq], ((piece_no / NQ) & 1) ^ 1, p.status, kStatusTimeoutProducer))) break;
      if (lane == 0) s_piece[iq] = make_int4(q.row, q.entry, q.t0, q.n);
      uint8_t* dst = sQ + iq * L::kQBytes;
#pragma unroll
      for (int h = 0; h < NR; ++h) {
        // largest |x| as a bf16 number's bits: infinities and NaN are the largest
        uint32_t top = 0;
#pragma unroll
        for (int e = 0; e < E / 2; ++e) top = max(top, max(raw[h][e] & 0x7fffu, raw[h][e] >> 16 & 0x7fffu));
        top = __reduce_max_sync(0xffffffffu, top) << 16;
        // a power of two s with largest / s in (224, 448] (or s = 2^-126)
        const int ex = (int)(top >> 23) - 8 + ((top & 0x7fffffu) > 0x600000u);
        const float s = __uint_as_float((uint32_t)max(ex, 1) << 23), inv = __uint_as_float((uint32_t)(254 - max(ex, 1)) << 23);
        uint32_t hi = 0, lo = 0;
#pragma unroll
        for (int e = 0; e < E; e += 2) {
          const float a = __uint_as_float(raw[h][e / 2] << 16) * inv, b = __uint_as_float(raw[h][e / 2] & 0xffff0000u) * inv;
          const uint32_t c = e4m3x2(a, b);
          const float2 f = from_e4m3x2(c);
          hi |= c << (8 * e);
          lo |= e4m3x2((a - f.x) * 16.f, (b - f.y) * 16.f) << (8 * e);
        }
        // row (token of the row, term, head); 16-byte pieces lie at their number xor the row's, modulo 8
#pragma unroll
        for (int c = 0; c < PACK; ++c)
#pragma unroll
          for (int term = 0; term < 2; ++term) {
            const int row = (c * 2 + term) * NR + h;
#pragma unroll
            for (int half = 0; half < PACK; ++half) {
              const int byte = half * D + lane * E;
              uint8_t* at = dst + row * 128 + (((byte >> 4) ^ (row & 7)) << 4) + (byte & 15);
              const uint32_t v = half == c ? (term ? lo : hi) : 0u;
              if (E == 4) *reinterpret_cast<uint32_t*>(at) = v;
              else *reinterpret_cast<uint16_t*>(at) = (uint16_t)v;
            }
          }
        if (lane == 0) s_factor[iq * NR + h] = top >= 0x7f800000u ? __int_as_float(0x7fc00000) : s * p.scale_log2;
      }
      fence_proxy_async_smem();
      __syncwarp();
      if (lane == 0) mbar_arrive(&q_full[iq]);
      q = next;
#pragma unroll
      for (int r = 0; r < NR; ++r)
#pragma unroll
        for (int e = 0; e < E / 2; ++e) raw[r][e] = ahead[r][e];
    }
  } else if (warp < 8) {
    // ------------------------------ soft-max ------------------------------
    const int g = warp >> 2, quarter = warp & 3;
    const int r = quarter * 32 + lane, part = r / L::RPB;                     // row of the tile, its cache block
    const int at = (r % L::RPB) * PACK + (PACK == 2 ? g : 0);                 // the thread's token, in its block
    const uint32_t tmem = tmem_base + ((uint32_t)(quarter * 32) << 16), col = PACK == 2 ? g * 2 * NR : 0;
    const int twist = L::NO == 32 ? r >> 2 & 1 : r >> 1 & 3;      // 16-byte pieces of a row of the weights lie at their number xor this
    float2* red = s_red + g * 4 * NR;
    int tn = 0;                // first tile of the piece, in the range
    int stage = PACK == 1 ? g : 0;      // ring place of the group's next tile, and its turn
    uint32_t round = 0;
    uint32_t piece_no = 0;
    bool ok = true, gone = false;
    auto wait = [&](uint64_t* bar, uint32_t parity) {
      return __all_sync(0xffffffffu, bar_wait(bar, parity, p.status, kStatusTimeoutEpilogue)) != 0;
    };
    for (; tn < end - begin && !gone; ++piece_no) {
      const uint32_t ib = piece_no & 1, iq = piece_no % NQ;
      const uint32_t tmem_o = tmem + L::kTmemO + ib * L::kOBuffer + g * 4 * NR;
      ok = ok && wait(&q_full[iq], (piece_no / NQ) & 1);
      const int4 piece = s_piece[iq];
      const float2* factor = reinterpret_cast<const float2*>(s_factor + iq * NR);
      // a warp that has given up says so in the next vote
      const int stop = ok ? tn + piece.w : tn + 2;
      // two heads in each: references of the sums and of the weights, with their signs turned, and the sums
      float2 m[NR / 2], M[NR / 2], l[NR / 2];
#pragma unroll
      for (int i = 0; i < NR / 2; ++i) {
        m[i] = M[i] = make_float2(-kQ8None, -kQ8None);
        l[i] = make_float2(0.f, 0.f);
      }
      bool first = true;
      float least = INFINITY, largest = -INFINITY;      // of log2 vs; lane 0 has the warp's, as what is seen begins with its row
      for (int t = PACK == 1 ? tn + ((tn ^ g) & 1) : tn; t < stop; t += 3 - PACK) {
        const uint32_t b = t & 1, phase = t >> 1 & 1;
        ok = ok && wait(&s_full[b], phase);
        tc_fence_after();
        float4 block;
        int left;      // tokens of the block from this one on
        float2 z[NR / 2];
        {
          uint32_t raw[2][NR];
          tmem_ld_heads(tmem + L::kTmemS + b * L::NS + col, raw[0]);
          tmem_ld_heads(tmem + L::kTmemS + b * L::NS + col + NR, raw[1]);
          // meanwhile: the tile's scales (its keys' barrier has long turned), and the weighted sum of the tile two before, which
          // has read the buffer that the weights go to
          ok = ok && wait(&k_full[stage], round) && wait(&p_empty[b], phase ^ 1);
          if (!ok) s_fail[2 * g] = 1;
          block = s_block[stage * BPT + part];
          left = __float_as_int(block.z) - at;
          tmem_ld_wait();
#pragma unroll
          for (int i = 0; i < NR / 2; ++i) {
            const float2 hi = make_float2(__uint_as_float(raw[0][2 * i]), __uint_as_float(raw[0][2 * i + 1]));
            const float2 lo = make_float2(__uint_as_float(raw[1][2 * i]), __uint_as_float(raw[1][2 * i + 1]));
            z[i] = mul_f32x2(fma_f32x2(lo, make_float2(0.0625f, 0.0625f), hi), mul_f32x2(factor[i], make_float2(block.x, block.x)));
          }
        }
        tc_fence_before();
        __syncwarp();
        if (lane == 0) mbar_arrive(&s_empty[b]);
        const float lv = block.y;
        const bool seen = left > 0, whole = __all_sync(0xffffffffu, seen);
        if (!whole) {
#pragma unroll
          for (int i = 0; i < NR / 2; ++i)
            if (!seen) z[i] = make_float2(-INFINITY, -INFINITY);
        }
        if (seen && lv > kQ8Low) {
          least = fminf(least, lv);
          largest = fmaxf(largest, lv);
        }
        if constexpr (PACK == 2) {
          if (g == 0 && __any_sync(0xffffffffu, left == 1)) {
            // The last token shares its row with what lies behind it: where that is NaN, zero times it has spoilt the sums, and
            // the scores are computed here
            bool spoilt = false;
#pragma unroll
            for (int i = 0; i < NR / 2; ++i) spoilt |= z[i].x != z[i].x || z[i].y != z[i].y;
            if (spoilt && left == 1) {
              const uint8_t* k = smem + stage * L::kStage + r * 128;
              const int heads = heads_of(piece.y);
              const __nv_bfloat16* src = p.q + (size_t)piece.x * p.row_stride + (size_t)first_head(piece.y) * D;
              const float f = block.x * p.scale_log2;
#pragma unroll
              for (int i = 0; i < NR / 2; ++i)
                z[i] = make_float2(2 * i < heads ? d8_dot<D>(src + (size_t)(2 * i) * D, k, r) * f : 0.f,
                                   2 * i + 1 < heads ? d8_dot<D>(src + (size_t)(2 * i + 1) * D, k, r) * f : 0.f);
            }
          }
        }
        // exponents of the sums' and of the weights' terms
        float2 e[NR / 2], d[NR / 2];
        float top_e = -INFINITY, top_d = -INFINITY;
        auto exponents = [&]() {
#pragma unroll
          for (int i = 0; i < NR / 2; ++i) {
            e[i] = add_f32x2(z[i], m[i]);
            d[i] = add_f32x2(add_f32x2(z[i], M[i]), make_float2(lv, lv));
          }
        };
        exponents();
#pragma unroll
        for (int i = 0; i < NR / 2; ++i) {
          top_e = fmaxf(top_e, fmaxf(e[i].x, e[i].y));
          top_d = fmaxf(top_d, fmaxf(d[i].x, d[i].y));
        }
        // a weight beyond 2^14, or a sum that grows out of its reference's reach
        if (vote_128(g, first || !ok || top_d > 14.f || top_e > 64.f)) {
          // a wait that ran out: all four warps leave together, or the others would stay in a vote.  One flag per vote: a
          // warp may be ahead of the others by what lies between two votes
          gone = s_fail[2 * g];
          if (gone) break;
          float top = -INFINITY;
#pragma unroll
          for (int h = 0; h < NR; ++h) {
            const float a = redux_max(h & 1 ? z[h / 2].y : z[h / 2].x);
            if (lane == h) top = a;
          }
          if (lane < NR) red[quarter * NR + lane] = make_float2(top, top + lv);      // the warp's rows lie in one cache block
          // O^T is scaled below: the products of the group's tile before have to be in it
          if (PACK == 2 && !first) ok = wait(&p_empty[b ^ 1], (t - 1) >> 1 & 1);
          if (!ok) s_fail[2 * g + 1] = 1;
          vote_128(g, false);
          gone = s_fail[2 * g + 1];
          if (gone) break;
          // lane h: head h's new references (0 where there is none to turn)
          float a = -kQ8None, v = -kQ8None;
          if (lane < NR) {
#pragma unroll
            for (int w = 0; w < 4; ++w) {
              const float2 x = red[w * NR + lane];
              a = fminf(a, -x.x);
              v = fminf(v, 11.f - x.y);
            }
          }
          bool moved = false;
          float2 alpha[NR / 2];
#pragma unroll
          for (int i = 0; i < NR / 2; ++i) {
            const float2 m2 = make_float2(fminf(m[i].x, __shfl_sync(0xffffffffu, a, 2 * i)), fminf(m[i].y, __shfl_sync(0xffffffffu, a, 2 * i + 1)));
            const float2 M2 = make_float2(fminf(M[i].x, __shfl_sync(0xffffffffu, v, 2 * i)), fminf(M[i].y, __shfl_sync(0xffffffffu, v, 2 * i + 1)));
            if (!first) {
              l[i].x *= fast_exp2(m2.x - m[i].x);
              l[i].y *= fast_exp2(m2.y - m[i].y);
              alpha[i] = make_float2(fast_exp2(M2.x - M[i].x), fast_exp2(M2.y - M[i].y));
              moved |= M2.x != M[i].x || M2.y != M[i].y;
            }
            m[i] = m2;
            M[i] = M2;
          }
          if (moved) {
            tc_fence_after();
#pragma unroll 1
            for (int i = 0; i < 3; ++i) {
              uint32_t o[NR];
              tmem_ld_heads(tmem_o + i * NR, o);
              tmem_ld_wait();
#pragma unroll
              for (int h = 0; h < NR; ++h) o[h] = __float_as_uint(__uint_as_float(o[h]) * (h & 1 ? alpha[h / 2].y : alpha[h / 2].x));
              tmem_st_heads(tmem_o + i * NR, o);
            }
            tmem_st_wait();
          }
          exponents();
        }
        first = false;
        uint8_t* dst = sP + b * L::kPBytes + r * L::NO;
#pragma unroll
        for (int h8 = 0; h8 < NR; h8 += 8) {
          uint32_t code[3][4];      // of two heads each
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            const int j = h8 / 2 + i;
            l[j] = add_f32x2(l[j], make_float2(fast_exp2(e[j].x), fast_exp2(e[j].y)));
            float2 w = make_float2(fast_exp2(d[j].x), fast_exp2(d[j].y));
#pragma unroll
            for (int term = 0; term < 3; ++term) {
              code[term][i] = e5m2x2(w.x, w.y);
              w = fma_f32x2(from_e5m2x2(code[term][i]), make_float2(-16.f, -16.f), mul_f32x2(w, make_float2(16.f, 16.f)));
            }
          }
          auto join = [](const uint32_t (&x)[4]) { return make_uint2(x[0] | x[1] << 16, x[2] | x[3] << 16); };
          const uint2 a = join(code[0]), b = join(code[1]), c = join(code[2]);
          if constexpr (NR == 8) {
            *reinterpret_cast<uint4*>(dst + ((PACK == 2 ? g * 2 : 0) ^ twist) * 16) = make_uint4(a.x, a.y, b.x, b.y);
            *reinterpret_cast<uint4*>(dst + (((PACK == 2 ? g * 2 : 0) + 1) ^ twist) * 16) = make_uint4(c.x, c.y, 0u, 0u);
          } else {
            *reinterpret_cast<uint2*>(dst + (0 ^ twist) * 16 + h8) = a;
            *reinterpret_cast<uint2*>(dst + (1 ^ twist) * 16 + h8) = b;
            *reinterpret_cast<uint2*>(dst + (2 ^ twist) * 16 + h8) = c;
          }
        }
        // what lies behind the last token may be anything, NaN too: zero weights alone would not do
        if (!whole) {
          ok = ok && wait(&v_full[stage], round);
          uint8_t* v = smem + stage * L::kStage + 16384 + r * 128;
          if (!seen)
#pragma unroll
            for (int i = 0; i < 8 / PACK; ++i)
              *reinterpret_cast<uint4*>(v + ((((PACK == 2 ? g * 4 : 0) + i) ^ (r & 7)) << 4)) = make_uint4(0, 0, 0, 0);
        }
        fence_proxy_async_smem();
        tc_fence_before();
        __syncwarp();
        if (lane == 0) mbar_arrive(&p_full[b]);
        stage += 3 - PACK;
        if (stage >= NST) {
          stage -= NST;
          round ^= 1;
        }
      }
      if (gone) break;
      tn = stop;
      // sums over the warp: half of the heads go to the other half of the lanes at every step
      float sum[NR];
#pragma unroll
      for (int h = 0; h < NR; ++h) sum[h] = h & 1 ? l[h / 2].y : l[h / 2].x;
#pragma unroll
      for (int n = NR, o = 16; o > 0; o >>= 1) {
        if (n > 1) {
          n >>= 1;
#pragma unroll
          for (int i = 0; i < NR / 2; ++i)
            if (i < n) {
              const bool up = lane & o;
              const float mine = up ? sum[i + n] : sum[i], other = up ? sum[i] : sum[i + n];
              sum[i] = mine + __shfl_xor_sync(0xffffffffu, other, o);
            }
        } else {
          sum[0] += __shfl_xor_sync(0xffffffffu, sum[0], o);
        }
      }
      float* stat = s_stat + (ib * 2 + g) * 6 * NR;
      ok = ok && wait(&o_empty[ib], ((piece_no >> 1) & 1) ^ 1);
      constexpr int kLow = NR == 8 ? 2 : 1;      // lane bits below are copies
      if ((lane & ((1 << kLow) - 1)) == 0) stat[quarter * NR + (lane >> kLow)] = sum[0];
      if (quarter == 0) {
#pragma unroll
        for (int i = 0; i < NR / 2; ++i)
          if (lane == i) {
            *reinterpret_cast<float2*>(stat + 4 * NR + 2 * i) = make_float2(-m[i].x, -m[i].y);
            *reinterpret_cast<float2*>(stat + 5 * NR + 2 * i) = make_float2(-M[i].x, -M[i].y);
          }
      }
      if (lane == 0) s_spread[ib * 8 + warp] = make_float2(least, largest);
      __syncwarp();
      if (lane == 0) {
        mbar_arrive(&q_empty[iq]);
        mbar_arrive(&o_full[ib]);
      }
    }
  } else {
    // ------------------------------ idle slots, then output: thread = byte of a row ------------------------------
    const int quarter = warp & 3, byte = quarter * 32 + lane, d = byte % D, c = byte / D;
    const uint32_t lane_off = (uint32_t)(quarter * 32) << 16;
    for (int b = blockIdx.x * 4 + quarter; b < p.B; b += gridDim.x * 4) {
      if (s_len[b] > 0) continue;
      uint4* row = reinterpret_cast<uint4*>(p.out + (size_t)b * p.Hq * D);
      for (int i = lane; i < p.Hq * D / 8; i += 32) row[i] = make_uint4(0u, 0u, 0u, 0u);
    }
    uint32_t piece_no = 0;
    D8Piece q;
    if (begin < end) q = d8_piece(s_pre, p.B, entries, begin, end);
    for (int cur = begin; cur < end; ++piece_no) {
      if (cur != begin) d8_next(s_pre, entries, q, cur, end);
      const uint32_t ib = piece_no & 1;
      if (!__all_sync(0xffffffffu, bar_wait(&o_full[ib], (piece_no >> 1) & 1, p.status, kStatusTimeoutEpilogue))) break;
      tc_fence_after();
      float2 spread = s_spread[ib * 8];
#pragma unroll
      for (int w = 1; w < 8; ++w) {
        const float2 x = s_spread[ib * 8 + w];
        spread = make_float2(fminf(spread.x, x.x), fmaxf(spread.y, x.y));
      }
      // lane h: head h's factors of the two O^T, and its log-sum-exp
      float f[2] = {0.f, 0.f}, lse = -INFINITY;
      if (lane < NR) {
        const float* stat = s_stat + ib * 12 * NR + lane;
        float l[2], m = kQ8None, sum = 0.f;
#pragma unroll
        for (int g = 0; g < 2; ++g) {
          const float* x = stat + g * 6 * NR;
          l[g] = (x[0] + x[NR]) + (x[2 * NR] + x[3 * NR]);
          m = fmaxf(m, x[4 * NR]);
        }
#pragma unroll
        for (int g = 0; g < 2; ++g) sum += l[g] == 0.f ? 0.f : l[g] * fast_exp2(stat[(6 * g + 4) * NR] - m);
#pragma unroll
        for (int g = 0; g < 2; ++g) f[g] = l[g] == 0.f ? 0.f : fast_exp2(stat[(6 * g + 5) * NR] - m) / sum;
        lse = sum == 0.f ? -INFINITY : m + log2f(sum);
      }
      float o[NR];
#pragma unroll
      for (int h = 0; h < NR; ++h) o[h] = 0.f;
      // D = 128: both groups' O^T; D = 64: of the tokens that stand where the thread's byte does
#pragma unroll 1
      for (int g = PACK == 2 ? c : 0; g < (PACK == 2 ? c + 1 : 2); ++g) {
        if (PACK == 1 && q.n == 1 && g != (cur - begin & 1)) continue;      // one tile: the other group's has not been written
        uint32_t x[3][NR];
        const uint32_t at = tmem_base + lane_off + L::kTmemO + ib * L::kOBuffer + g * 4 * NR;
#pragma unroll
        for (int term = 0; term < 3; ++term) tmem_ld_heads(at + term * NR, x[term]);
        tmem_ld_wait();
#pragma unroll
        for (int h = 0; h < NR; ++h) {
          const float a = fmaf(fmaf(__uint_as_float(x[2][h]), 0.0625f, __uint_as_float(x[1][h])), 0.0625f, __uint_as_float(x[0][h]));
          const float w = __shfl_sync(0xffffffffu, g ? f[1] : f[0], h);
          o[h] += w == 0.f ? 0.f : a * w;
        }
      }
      tc_fence_before();
      __syncwarp();
      if (lane == 0) mbar_arrive(&o_empty[ib]);
      if constexpr (PACK == 2) {
        // the odd tokens' warps hand their share to the even tokens'
        if (c == 1) {
          if (!__all_sync(0xffffffffu, bar_wait(x_empty, (piece_no & 1) ^ 1, p.status, kStatusTimeoutEpilogue))) break;
#pragma unroll
          for (int h = 0; h < NR; ++h) s_x[h * 64 + d] = o[h];
          __syncwarp();
          if (lane == 0) mbar_arrive(x_full);
        } else {
          if (!__all_sync(0xffffffffu, bar_wait(x_full, piece_no & 1, p.status, kStatusTimeoutEpilogue))) break;
#pragma unroll
          for (int h = 0; h < NR; ++h) o[h] += s_x[h * 64 + d];
          __syncwarp();
          if (lane == 0) mbar_arrive(x_empty);
        }
      }
      if (c == 0) {
        const int left = heads_of(q.entry);
        const int slot = 2 * blockIdx.x + (cur == begin ? 0 : 1);
        const bool whole = q.n == q.tiles;
        if (spread.y - spread.x > kQ8Spread) {
          float exact[NR], exact_lse;      // o and lse stay in registers
          d8_exact<D, NR>(p.q + (size_t)q.row * p.row_stride + (size_t)first_head(q.entry) * D, left, p.codes, p.scales,
                          p.block_table + (size_t)q.row * p.max_blocks, p.num_blocks, p.Hkv, kv_head(q.entry), q.t0 * L::TT,
                          min(s_len[q.row], (q.t0 + q.n) * L::TT), p.scale_log2, d, exact, exact_lse);
#pragma unroll
          for (int h = 0; h < NR; ++h) o[h] = exact[h];
          lse = exact_lse;
        }
        __nv_bfloat16* orow = p.out + ((size_t)q.row * p.Hq + first_head(q.entry)) * D + d;
        float* wrow = p.ws_o + (size_t)slot * NR * D + d;
#pragma unroll
        for (int h = 0; h < NR; ++h)
          if (h < left) {
            if (whole) orow[h * D] = __float2bfloat16(o[h]);
            else wrow[h * D] = o[h];
          }
        if (!whole) {
          if (lane < NR) p.ws_lse[((size_t)slot * 4 + quarter) * NR + lane] = lse;
          // the range that holds position x is the last one that begins at or before it
          const int first = s_pre[q.row] * entries + q.entry * q.tiles;
          const int c0 = alone ? blockIdx.x - s_mine[2] : (int)(((long long)(first + 1) * ranges - 1) / total);
          const int c1 = alone ? c0 + s_mine[3] - 1 : (int)(((long long)(first + q.tiles) * ranges - 1) / total);
          d8_join<D, NR>(p.ws_o + d, p.ws_lse + quarter * NR, p.counts + ((size_t)q.row * entries + q.entry) * 4 + quarter, c0, c1,
                         alone || d8_begin(total, c0, ranges) >= first ? 0 : 1, left, orow);
        }
      }
      cur += q.n;
    }
  }
  tc_fence_before();
  __syncthreads();
  if (warp == 13) {
    tc_fence_after();
    tmem_dealloc(tmem_base, L::kTmemCols);
  }
}

template <int D, int NR>
static int launch_decode8(const CUtensorMap& mc, const Decode8Params& p, int grid, cudaStream_t stream) {
  using L = D8<D, NR>;
  static_assert(L::kStages >= 4 && L::kTotal <= kQ8Smem && 2 * (L::NS + L::kOBuffer) <= 512 && L::kTotal % 4 == 0, "");
  auto kernel = fmha_decode8_kernel<D, NR>;
  static int configured = -1;
  int dev = 0;
  cudaGetDevice(&dev);
  if (configured != dev) {
    cudaError_t e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, L::kTotal);
    if (e != cudaSuccess) return (int)e;
    configured = dev;
  }
  return launch_chained(kernel, (unsigned)grid, kQ8Threads, L::kTotal, stream, mc, p);
}

}  // namespace sb

using namespace sb;

// Number of the capture that `stream` takes part in, 0 outside of one
extern "C" unsigned long long sb_capture_id(cudaStream_t stream) {
  cudaStreamCaptureStatus status = cudaStreamCaptureStatusNone;
  unsigned long long id = 0;
  if (cudaStreamGetCaptureInfo(stream, &status, &id) != cudaSuccess) cudaGetLastError();
  return status == cudaStreamCaptureStatusActive ? id : 0;
}

extern "C" int sb_kv8_decode_grid() { return num_sms(); }

// Workspaces: with rows = 8 where at most 8 query heads share a kv head or D = 64, else 16, ws_o has 2 * grid * rows * D floats,
// ws_lse 8 * grid * rows; counts B * Hkv * ceil(Hq / Hkv / rows) * 4 ints, which are zeros and stay zeros after every call, but one
// whose waits ran out.
//
// One query row per sequence (at most 1024) against its cached context of seq_lens[b] tokens, the current one included; 0: idle
// slot, its output row is zero.  Rows start on 4-byte boundaries.
extern "C" int sb_kv8_decode(const void* q, long long row_stride, const void* codes, const float* scales, int num_blocks,
                             const int* seq_lens, const int* block_table, int max_blocks, void* out, float* ws_o,
                             float* ws_lse, int* counts, int B, int Hq, int Hkv, int D, float scale, int* status,
                             cudaStream_t stream) {
  if (B == 0) return 0;
  if (D != 64 && D != 128) return -2;
  if (B > kQ8Rows || Hq % Hkv || Hq / Hkv > 32 || row_stride % 2 || reinterpret_cast<uintptr_t>(q) % 4 || reinterpret_cast<uintptr_t>(out) % 16 || max_blocks < 1 || num_blocks < 1) return -3;
  const long long rows = (long long)num_blocks * 2 * Hkv * (D / 2), tiles = (max_blocks + 1ll) / 2 * B * Hkv * 4;
  if (rows > 0x7fffffffll || tiles > 0x7fffffffll || max_blocks > 1 << 24) return -4;      // lengths, rounded up to tiles: 32 bits
  bind_context();
  // rows of 128 bytes, as 64 16-bit numbers; a box is a cache block of one head
  CUtensorMap mc;
  const int r = make_tensor_map_bf16_2d(&mc, codes, 64, rows, 64, 64, D / 2);
  if (r) return r;
  Decode8Params p;
  p.q = (const __nv_bfloat16*)q; p.row_stride = row_stride; p.codes = (const uint8_t*)codes; p.scales = scales; p.seq_lens = seq_lens;
  p.block_table = block_table; p.num_blocks = num_blocks; p.max_blocks = max_blocks; p.B = B; p.Hq = Hq; p.Hkv = Hkv;
  const int most = Hq / Hkv <= 8 || D == 64 ? 8 : 16;
  p.groups = (Hq / Hkv + most - 1) / most;
  p.out = (__nv_bfloat16*)out; p.ws_o = ws_o; p.ws_lse = ws_lse; p.counts = counts;
  p.scale_log2 = scale * 1.4426950408889634f; p.status = status;
  const int grid = num_sms();
  if (D == 64) return launch_decode8<64, 8>(mc, p, grid, stream);
  return most == 8 ? launch_decode8<128, 8>(mc, p, grid, stream) : launch_decode8<128, 16>(mc, p, grid, stream);
}
