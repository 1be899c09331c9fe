// Paged key / value cache in 8 bits: appending rows, forking blocks.
//
// Cache of one layer: codes [num_blocks, 2 (k|v), Hkv, 64 tokens, D] in e4m3, scales [num_blocks, 2, Hkv] in fp32; a cached
// value is code * scale.  A scale is the smallest power of two with which every finite value that its block and head have met
// fits e4m3's range (|x| <= 448 * scale): a power of two because e4m3 is a floating-point format, so that a finer scale would
// buy no relative precision, because dividing by it is exact, and because codes that have to follow a growing scale then
// only lose what falls below e4m3's smallest step.  Values are rounded once, from the 32-bit rotated ones.
#include <cuda_fp8.h>

#include "common.cuh"
#include "launchers.h"

namespace sb {

constexpr int kB8 = 64;  // tokens per cache block

// ---------------------------------------------------------------------------------------
// scales and codes
// ---------------------------------------------------------------------------------------
// |x| where that is finite, else 0: infinities saturate at the block's largest value, they do not set its scale
__device__ __forceinline__ float finite_abs(float x) {
  const float a = fabsf(x);
  return a <= 3.402823466e38f ? a : 0.f;
}
// smallest power of two s (at least 2^-126) with amax <= 448 s: 448 = 1.75 * 2^8
__device__ __forceinline__ float scale_of(float amax) {
  const uint32_t u = __float_as_uint(amax);
  const int e = (int)(u >> 23) - 8 + ((u & 0x7fffffu) > 0x600000u);   // biased exponent
  return __uint_as_float((uint32_t)max(e, 1) << 23);
}
// two values divided by their scale, as codes; beyond the range: +-448
__device__ __forceinline__ uint32_t codes_of(float a, float b) {
  return (uint32_t)__nv_cvt_float2_to_fp8x2(make_float2(a, b), __NV_SATFINITE, __NV_E4M3);
}
__device__ __forceinline__ float2 values_of(uint32_t codes) {
  const __half2_raw h = __nv_cvt_fp8x2_to_halfraw2((__nv_fp8x2_storage_t)(codes & 0xffffu), __NV_E4M3);
  return __half22float2(*reinterpret_cast<const __half2*>(&h));
}
// four codes of a block whose scale has grown
__device__ __forceinline__ uint32_t rescaled(uint32_t codes, float ratio) {
  const float2 a = values_of(codes), b = values_of(codes >> 16);
  return codes_of(a.x * ratio, a.y * ratio) | codes_of(b.x * ratio, b.y * ratio) << 16;
}

struct Append8Params {
  __nv_bfloat16* qkv;      // [T, row_stride]: heads q | k | v
  int row_stride;
  const float* slabs;      // the projection's partial sums [splits, T, heads * D], slab_stride floats apart, or null
  long long slab_stride;
  int splits;
  const __nv_bfloat16* bias;
  const int* rope_pos;     // [pos_rows, T], or null: no rotation
  int pos_rows, sec0, sec1, table_rows;
  const float *cos_tab, *sin_tab;
  const int *seq_ids, *cache_pos, *block_table;
  int sequences, max_blocks;
  uint8_t* codes;
  float* scales;
  int num_blocks, T, Hq, Hkv;
};

// cache block of row t, or -1 where the row is not cached
__device__ __forceinline__ int block_of(const Append8Params& p, int t) {
  const int seq = p.seq_ids[t], cp = p.cache_pos[t];
  if (seq < 0 || seq >= p.sequences || cp < 0 || cp / kB8 >= p.max_blocks) return -1;
  const int blk = p.block_table[(size_t)seq * p.max_blocks + cp / kB8];
  return blk < p.num_blocks ? blk : -1;
}

// row of the tables for element c of row r
__device__ __forceinline__ int table_row(const Append8Params& p, int r, int c) {
  const int axis = p.pos_rows == 3 ? (c < p.sec0 ? 0 : c < p.sec1 ? 1 : 2) : 0;
  return min(max(p.rope_pos[(size_t)axis * p.T + r], 0), p.table_rows - 1);
}

// ---------------------------------------------------------------------------------------
// D / 4 lanes for a head: a lane holds elements 2 l, 2 l + 1 and their partners D / 2 further on
// ---------------------------------------------------------------------------------------
template <int D>
struct RowLanes {
  static constexpr int N = D / 4, half = D / 2;
  const Append8Params& p;
  int head, l;
  uint32_t mask;      // of the lanes
  bool turns;

  __device__ __forceinline__ RowLanes(const Append8Params& q, int h) : p(q), head(h) {
    const int lane = threadIdx.x & 31;
    l = lane % N;
    mask = N == 32 ? 0xffffffffu : 0xffffu << (lane & 16);
    turns = p.rope_pos != nullptr && head < p.Hq + p.Hkv;
  }

  __device__ __forceinline__ void load(int r, float (&x)[4]) const {   // x[0..1]: elements, x[2..3]: their partners; rotated
    if (p.slabs) {
      const float* src = p.slabs + ((size_t)r * (p.Hq + 2 * p.Hkv) + head) * D + 2 * l;
#pragma unroll
      for (int i = 0; i < 4; ++i) x[i] = 0.f;
#pragma unroll 4
      for (int s = 0; s < p.splits; ++s, src += p.slab_stride) {
        const float2 a = *reinterpret_cast<const float2*>(src), b = *reinterpret_cast<const float2*>(src + half);
        x[0] += a.x; x[1] += a.y; x[2] += b.x; x[3] += b.y;
      }
      if (p.bias) {
        const __nv_bfloat16* b = p.bias + head * D + 2 * l;
#pragma unroll
        for (int i = 0; i < 2; ++i) {
          x[i] += __bfloat162float(b[i]);
          x[2 + i] += __bfloat162float(b[half + i]);
        }
      }
    } else {
      const __nv_bfloat16* src = p.qkv + (size_t)r * p.row_stride + (size_t)head * D + 2 * l;
      const float2 a = __bfloat1622float2(*reinterpret_cast<const __nv_bfloat162*>(src));
      const float2 b = __bfloat1622float2(*reinterpret_cast<const __nv_bfloat162*>(src + half));
      x[0] = a.x; x[1] = a.y; x[2] = b.x; x[3] = b.y;
    }
    if (turns) {
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        const int c = 2 * l + i;
        const size_t at = (size_t)table_row(p, r, c) * half + c;
        const float cs = p.cos_tab[at], sn = p.sin_tab[at], a = x[i];
        x[i] = a * cs - x[2 + i] * sn;
        x[2 + i] = x[2 + i] * cs + a * sn;
      }
    }
  }

  __device__ __forceinline__ void write_back(int r, const float (&x)[4]) const {
    if (!p.slabs && !turns) return;
    __nv_bfloat16* dst = p.qkv + (size_t)r * p.row_stride + (size_t)head * D + 2 * l;
    *reinterpret_cast<uint32_t*>(dst) = pack_bf16x2(x[0], x[1]);
    *reinterpret_cast<uint32_t*>(dst + half) = pack_bf16x2(x[2], x[3]);
  }

  __device__ __forceinline__ void turn_only(int r) const {
    if (!p.slabs && !turns) return;
    float x[4];
    load(r, x);
    write_back(r, x);
  }

  // rows t .. end - 1, which all lie in block `blk`: one after the other, so that a place named twice gets its last values
  __device__ __forceinline__ void append(int t, int end, int blk) const {
    const int kv = head >= p.Hq + p.Hkv ? 1 : 0;
    const size_t at = ((size_t)blk * 2 + kv) * p.Hkv + (head - p.Hq - kv * p.Hkv);
    const float before = p.scales[at];      // asked for ahead of the rows
    float x[4], amax = 0.f;
    unsigned long long written = 0;
    for (int r = t; r < end; ++r) {
      load(r, x);
#pragma unroll
      for (int i = 0; i < 4; ++i) amax = fmaxf(amax, finite_abs(x[i]));
      written |= 1ull << (p.cache_pos[r] % kB8);
    }
#pragma unroll
    for (int o = N / 2; o > 0; o >>= 1) amax = fmaxf(amax, __shfl_xor_sync(mask, amax, o));
    uint8_t* dst = p.codes + at * kB8 * D;
    const bool anew = written & 1;
    const float kept = anew ? 0.f : before;
    const float scale = fmaxf(kept, scale_of(amax));
    if (scale != kept) {
      __syncwarp(mask);      // every lane has read the old scale
      const float ratio = kept / scale;
#pragma unroll 8
      for (int r = 0; r < kB8; ++r) {
        if (written >> r & 1) continue;
        uint32_t* c = reinterpret_cast<uint32_t*>(dst + r * D) + l;
        *c = anew ? 0u : rescaled(*c, ratio);
      }
      if (l == 0) p.scales[at] = scale;
    }
    const float inv = 1.f / scale;
    const bool one = end == t + 1;
    for (int r = t; r < end; ++r) {
      if (!one) load(r, x);
      write_back(r, x);
      uint8_t* c = dst + (p.cache_pos[r] % kB8) * D + 2 * l;
      *reinterpret_cast<uint16_t*>(c) = (uint16_t)codes_of(x[0] * inv, x[1] * inv);
      *reinterpret_cast<uint16_t*>(c + half) = (uint16_t)codes_of(x[2] * inv, x[3] * inv);
    }
  }
};

// Rows of any alignment: the lanes that meet the first of the adjacent rows of a cache block do all of them.
template <int D>
__global__ void __launch_bounds__(256) append8_lanes_kernel(Append8Params p) {
  chain_sync();
  const int heads = p.Hq + 2 * p.Hkv;
  const long long unit = (blockIdx.x * 256ll + threadIdx.x) / (D / 4);
  if (unit >= (long long)p.T * heads) return;
  const int t = (int)(unit / heads), head = (int)(unit % heads);
  const RowLanes<D> lanes(p, head);
  const int blk = head < p.Hq ? -1 : block_of(p, t);
  if (blk < 0) {
    lanes.turn_only(t);
    return;
  }
  if (t > 0 && block_of(p, t - 1) == blk) return;
  int end = t + 1;
  while (end < p.T && block_of(p, end) == blk) ++end;
  lanes.append(t, end, blk);
}

// ---------------------------------------------------------------------------------------
// Rows on 16-byte boundaries.  The first blocks of the grid take k and v heads: one head of `range` rows, of which those that
// are the first of a cache block's adjacent rows count (the block that has the first has all of them, up to 64, also where
// they reach beyond its range).  Runs of few rows go to D / 4 lanes each; of longer ones every thread holds a quarter of a row
// in registers while the block finds the largest value, so that rows are read once.  The other blocks rotate q heads: a thread
// keeps the eight angles of its pairs for `per` heads.
//
// Bound by memory: 28 / 4 heads, D = 128, 8992 rows of prompts: NOTE us for 170 MB.
// ---------------------------------------------------------------------------------------
constexpr int kRun = 8;      // rows from which on a run takes the whole block

// eight pairs from element i0 on of one head of row r: the sum of the partial sums, or the row; not rotated
template <int D>
__device__ __forceinline__ void load_pairs(const Append8Params& p, int r, int head, int i0, float (&x)[8], float (&y)[8]) {
  if (p.slabs) {
    const float* src = p.slabs + ((size_t)r * (p.Hq + 2 * p.Hkv) + head) * D + i0;
    slab_sum8(src, p.slab_stride, p.splits, x);
    slab_sum8(src + D / 2, p.slab_stride, p.splits, y);
    if (p.bias) {
      const __nv_bfloat16* b = p.bias + head * D + i0;
#pragma unroll
      for (int k = 0; k < 8; ++k) {
        x[k] += __bfloat162float(b[k]);
        y[k] += __bfloat162float(b[D / 2 + k]);
      }
    }
  } else {
    const __nv_bfloat16* src = p.qkv + (size_t)r * p.row_stride + (size_t)head * D + i0;
    const uint4 a = *reinterpret_cast<const uint4*>(src), b = *reinterpret_cast<const uint4*>(src + D / 2);
    const uint32_t u[4] = {a.x, a.y, a.z, a.w}, v[4] = {b.x, b.y, b.z, b.w};
#pragma unroll
    for (int k = 0; k < 4; ++k) {
      x[2 * k] = __uint_as_float(u[k] << 16); x[2 * k + 1] = __uint_as_float(u[k] & 0xffff0000u);
      y[2 * k] = __uint_as_float(v[k] << 16); y[2 * k + 1] = __uint_as_float(v[k] & 0xffff0000u);
    }
  }
}
template <int D>
__device__ __forceinline__ void load_angles(const Append8Params& p, int r, int i0, float (&c)[8], float (&s)[8]) {
  if (p.pos_rows == 3) {
#pragma unroll
    for (int k = 0; k < 8; ++k) {
      const size_t at = (size_t)table_row(p, r, i0 + k) * (D / 2) + i0 + k;
      c[k] = p.cos_tab[at];
      s[k] = p.sin_tab[at];
    }
    return;
  }
  const size_t at = (size_t)table_row(p, r, 0) * (D / 2) + i0;
#pragma unroll
  for (int k = 0; k < 8; k += 4) {
    const float4 a = *reinterpret_cast<const float4*>(p.cos_tab + at + k), b = *reinterpret_cast<const float4*>(p.sin_tab + at + k);
    c[k] = a.x; c[k + 1] = a.y; c[k + 2] = a.z; c[k + 3] = a.w;
    s[k] = b.x; s[k + 1] = b.y; s[k + 2] = b.z; s[k + 3] = b.w;
  }
}
__device__ __forceinline__ void turn_pairs(float (&x)[8], float (&y)[8], const float (&c)[8], const float (&s)[8]) {
#pragma unroll
  for (int k = 0; k < 8; ++k) {
    const float a = x[k];
    x[k] = a * c[k] - y[k] * s[k];
    y[k] = y[k] * c[k] + a * s[k];
  }
}
template <int D>
__device__ __forceinline__ void store_pairs(const Append8Params& p, int r, int head, int i0, const float (&x)[8], const float (&y)[8]) {
  __nv_bfloat16* dst = p.qkv + (size_t)r * p.row_stride + (size_t)head * D + i0;
  *reinterpret_cast<uint4*>(dst) = make_uint4(pack_bf16x2(x[0], x[1]), pack_bf16x2(x[2], x[3]), pack_bf16x2(x[4], x[5]), pack_bf16x2(x[6], x[7]));
  *reinterpret_cast<uint4*>(dst + D / 2) = make_uint4(pack_bf16x2(y[0], y[1]), pack_bf16x2(y[2], y[3]), pack_bf16x2(y[4], y[5]), pack_bf16x2(y[6], y[7]));
}
__device__ __forceinline__ uint2 codes_of8(const float (&x)[8], float inv) {
  return make_uint2(codes_of(x[0] * inv, x[1] * inv) | codes_of(x[2] * inv, x[3] * inv) << 16,
                    codes_of(x[4] * inv, x[5] * inv) | codes_of(x[6] * inv, x[7] * inv) << 16);
}

template <int D>
__global__ void __launch_bounds__(256) append8_kernel(Append8Params p, int kv_blocks, int range, int per) {
  __shared__ int s_blk[2 * kB8 + 2];      // cache blocks of rows r0 - 1 .. r0 + range + 63
  __shared__ int s_last[kB8];             // last row of the run at each offset
  __shared__ uint32_t s_begin[5], s_top[8];
  chain_sync();
  const int tid = threadIdx.x;
  if ((int)blockIdx.x >= kv_blocks) {
    // ------------------------------ q heads ------------------------------
    constexpr int TPR = D / 16, ROWS = 256 / TPR;
    const int b = blockIdx.x - kv_blocks, parts = (p.Hq + per - 1) / per;
    const int r = b / parts * ROWS + tid / TPR, h0 = b % parts * per, i0 = tid % TPR * 8;
    if (r >= p.T) return;
    float c[8], s[8];
    if (p.rope_pos) load_angles<D>(p, r, i0, c, s);
#pragma unroll 4
    for (int h = h0; h < min(h0 + per, p.Hq); ++h) {
      float x[8], y[8];
      load_pairs<D>(p, r, h, i0, x, y);
      if (p.rope_pos) turn_pairs(x, y, c, s);
      store_pairs<D>(p, r, h, i0, x, y);
    }
    return;
  }
  // ------------------------------ k and v heads ------------------------------
  const int kv_heads = 2 * p.Hkv, hd = blockIdx.x % kv_heads, r0 = blockIdx.x / kv_heads * range;
  const int head = p.Hq + hd, rows = min(range, p.T - r0);
  for (int i = tid; i < range + kB8 + 1; i += 256) {
    const int t = r0 - 1 + i;
    s_blk[i] = t >= 0 && t < p.T ? block_of(p, t) : -1;
  }
  __syncthreads();
  // bit i: row r0 + i lies in another block than the one before
  if (tid < 5 * 32) {
    const bool other = tid < range + kB8 && (r0 + tid >= p.T || s_blk[tid + 1] != s_blk[tid]);
    const uint32_t bits = __ballot_sync(0xffffffffu, other);
    if ((tid & 31) == 0) s_begin[tid >> 5] = bits;
  }
  __syncthreads();
  auto next = [&](int i) {      // first row from i on that begins a run
    uint32_t bits = s_begin[i >> 5] >> (i & 31) << (i & 31);
    int w = i >> 5;
    while (!bits && ++w < 5) bits = s_begin[w];
    return bits ? w * 32 + __ffs(bits) - 1 : range + kB8;
  };
  const RowLanes<D> lanes(p, head);
  constexpr int LPH = D / 4;
  for (int i = tid / LPH; i < rows; i += 256 / LPH) {
    const int blk = s_blk[i + 1], t = r0 + i;
    if (blk < 0) {
      lanes.turn_only(t);
      continue;
    }
    if (s_blk[i] == blk) continue;
    int end = r0 + next(i + 1);
    if (end - t >= kRun && end - t <= kB8) continue;
    if (end - t > kB8)      // some place is named twice
      while (end < p.T && block_of(p, end) == blk) ++end;
    lanes.append(t, end, blk);
  }
  const int kv = hd >= p.Hkv ? 1 : 0;
  const bool turns = p.rope_pos && !kv;
  for (int i = next(0), e; i < rows; i = e) {
    e = next(i + 1);
    const int blk = s_blk[i + 1], t = r0 + i, n = e - i;
    if (blk < 0 || n < kRun || n > kB8) continue;
    // a quarter of a row per thread: 16 pairs (D = 128) or 8
    constexpr int U = D / 64;
    const int row = tid >> 2, q = tid & 3, r = t + row;
    const bool mine = row < n;
    const size_t at = ((size_t)blk * 2 + kv) * p.Hkv + (hd - kv * p.Hkv);
    const float before = p.scales[at];
    if (tid < kB8) s_last[tid] = -1;
    float x[U][8], y[U][8], amax = 0.f;
    int off = 0;
    if (mine) {
      off = p.cache_pos[r] % kB8;
#pragma unroll
      for (int u = 0; u < U; ++u) load_pairs<D>(p, r, head, (u * 4 + q) * 8, x[u], y[u]);
      if (turns) {
#pragma unroll
        for (int u = 0; u < U; ++u) {
          float c[8], s[8];
          load_angles<D>(p, r, (u * 4 + q) * 8, c, s);
          turn_pairs(x[u], y[u], c, s);
        }
      }
#pragma unroll
      for (int u = 0; u < U; ++u)
#pragma unroll
        for (int k = 0; k < 8; ++k) amax = fmaxf(amax, fmaxf(finite_abs(x[u][k]), finite_abs(y[u][k])));
    }
    const uint32_t top = __reduce_max_sync(0xffffffffu, __float_as_uint(amax));      // of numbers >= 0, bits order as they do
    if ((tid & 31) == 0) s_top[tid >> 5] = top;
    __syncthreads();
    if (mine && q == 0) atomicMax(&s_last[off], row);
    __syncthreads();
    uint32_t all = 0;
#pragma unroll
    for (int w = 0; w < 8; ++w) all = max(all, s_top[w]);
    const bool anew = s_last[0] >= 0;
    const float kept = anew ? 0.f : before, scale = fmaxf(kept, scale_of(__uint_as_float(all))), inv = 1.f / scale;
    uint8_t* dst = p.codes + at * kB8 * D;
    if (scale != kept) {
      if (s_last[row] < 0) {      // thread's quarter of the row at this offset
        const float ratio = kept / scale;
        uint32_t* c = reinterpret_cast<uint32_t*>(dst + row * D) + q * (D / 16);
#pragma unroll
        for (int k = 0; k < D / 16; ++k) c[k] = anew ? 0u : rescaled(c[k], ratio);
      }
      if (tid == 0) p.scales[at] = scale;
    }
    if (mine) {
#pragma unroll
      for (int u = 0; u < U; ++u) {
        const int i0 = (u * 4 + q) * 8;
        if (s_last[off] == row) {
          *reinterpret_cast<uint2*>(dst + off * D + i0) = codes_of8(x[u], inv);
          *reinterpret_cast<uint2*>(dst + off * D + D / 2 + i0) = codes_of8(y[u], inv);
        }
        if (turns || p.slabs) store_pairs<D>(p, r, head, i0, x[u], y[u]);
      }
    }
    __syncthreads();
  }
}

// copies blocks with their scales (src[i] -> dst[i]); pairs that name no block are left out
__global__ void __launch_bounds__(256) copy8_blocks_kernel(uint8_t* codes, float* scales, const int* src, const int* dst,
                                                           int n_pairs, int num_blocks, int per_block, long long bytes) {
  for (int i = blockIdx.y; i < n_pairs; i += gridDim.y) {
    const int a = src[i], b = dst[i];
    if (a < 0 || a >= num_blocks || b < 0 || b >= num_blocks) continue;
    const uint4* s = reinterpret_cast<const uint4*>(codes + (size_t)a * bytes);
    uint4* d = reinterpret_cast<uint4*>(codes + (size_t)b * bytes);
    for (long long k = blockIdx.x * 256ll + threadIdx.x; k < bytes / 16; k += gridDim.x * 256ll) d[k] = s[k];
    if (blockIdx.x == 0)
      for (int k = threadIdx.x; k < per_block; k += 256) scales[(size_t)b * per_block + k] = scales[(size_t)a * per_block + k];
  }
}

}  // namespace sb

using namespace sb;

// Rows of one cache block have to follow one another.  rope_pos null: nothing is rotated.
extern "C" int sb_kv8_append(void* qkv, int row_stride, const float* slabs, long long slab_stride, int splits,
                             const void* bias, const int* rope_pos, int pos_rows, int sec0, int sec1, int table_rows,
                             const float* cos_tab, const float* sin_tab, const int* seq_ids, const int* cache_pos,
                             const int* block_table, int sequences, int max_blocks, void* codes, float* scales,
                             int num_blocks, int T, int Hq, int Hkv, int D, cudaStream_t stream) {
  if (T == 0) return 0;
  if (D != 64 && D != 128) return -2;
  if (row_stride % 2 || (slabs && (splits < 1 || slab_stride % 2)) || (rope_pos && table_rows < 1)) return -3;
  Append8Params p;
  p.qkv = (__nv_bfloat16*)qkv; p.row_stride = row_stride; p.slabs = slabs; p.slab_stride = slab_stride; p.splits = splits;
  p.bias = (const __nv_bfloat16*)bias; p.rope_pos = rope_pos; p.pos_rows = pos_rows; p.sec0 = sec0; p.sec1 = sec1;
  p.table_rows = table_rows; p.cos_tab = cos_tab; p.sin_tab = sin_tab; p.seq_ids = seq_ids; p.cache_pos = cache_pos;
  p.block_table = block_table; p.sequences = sequences; p.max_blocks = max_blocks; p.codes = (uint8_t*)codes;
  p.scales = scales; p.num_blocks = num_blocks; p.T = T; p.Hq = Hq; p.Hkv = Hkv;
  auto on = [](const void* x) { return reinterpret_cast<uintptr_t>(x) % 16 == 0; };
  if (row_stride % 8 || !on(qkv) || !on(slabs) || slab_stride % 4 || !on(cos_tab) || !on(sin_tab)) {
    const long long blocks = ((long long)T * (Hq + 2 * Hkv) * (D / 4) + 255) / 256;
    if (blocks > 0x7fffffffll) return -4;
    return launch_chained(D == 128 ? append8_lanes_kernel<128> : append8_lanes_kernel<64>, (unsigned)blocks, 256, 0, stream, p);
  }
  const int range = T <= 2048 ? 8 : kB8, per = T <= 2048 ? 1 : 4, rows = 256 / (D / 16);
  const long long kv = (long long)((T + range - 1) / range) * 2 * Hkv;
  const long long q = rope_pos || slabs ? (long long)((T + rows - 1) / rows) * ((Hq + per - 1) / per) : 0;
  if (kv + q > 0x7fffffffll) return -4;
  return launch_chained(D == 128 ? append8_kernel<128> : append8_kernel<64>, (unsigned)(kv + q), 256, 0, stream, p, (int)kv, range, per);
}

extern "C" int sb_kv8_copy_blocks(void* codes, float* scales, const int* src, const int* dst, int n_pairs, int num_blocks,
                                  int per_block, long long bytes, cudaStream_t stream) {
  if (n_pairs == 0) return 0;
  if (bytes % 16) return -3;
  copy8_blocks_kernel<<<dim3(8, n_pairs < 4096 ? n_pairs : 4096), 256, 0, stream>>>((uint8_t*)codes, scales, src, dst, n_pairs,
                                                                                     num_blocks, per_block, bytes);
  return (int)cudaGetLastError();
}
