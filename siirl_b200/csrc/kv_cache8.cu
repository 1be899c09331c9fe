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
  long long row_stride;
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

  // of the head in block `blk`: its place among the scales, and its scale once the numbers of `amax` have joined; the rows that
  // `written` does not name follow a new one
  __device__ __forceinline__ size_t place(int blk) const {
    const int kv = head >= p.Hq + p.Hkv ? 1 : 0;
    return ((size_t)blk * 2 + kv) * p.Hkv + (head - p.Hq - kv * p.Hkv);
  }
  __device__ __forceinline__ float rescale(size_t at, float before, float amax, unsigned long long written) const {
#pragma unroll
    for (int o = N / 2; o > 0; o >>= 1) amax = fmaxf(amax, __shfl_xor_sync(mask, amax, o));
    const bool anew = written & 1;
    const float kept = anew ? 0.f : before, scale = fmaxf(kept, scale_of(amax));
    if (scale != kept) {
      __syncwarp(mask);      // every lane has read the old scale
      const float ratio = kept / scale;
      uint32_t* c = reinterpret_cast<uint32_t*>(p.codes + at * kB8 * D) + l;
#pragma unroll 4
      for (int r = 0; r < kB8; ++r)
        if (!(written >> r & 1)) c[r * N] = anew ? 0u : rescaled(c[r * N], ratio);
      if (l == 0) p.scales[at] = scale;
    }
    return 1.f / scale;
  }
  __device__ __forceinline__ void store(size_t at, int off, const float (&x)[4], float inv) const {
    uint8_t* c = p.codes + (at * kB8 + off) * D + 2 * l;
    *reinterpret_cast<uint16_t*>(c) = (uint16_t)codes_of(x[0] * inv, x[1] * inv);
    *reinterpret_cast<uint16_t*>(c + half) = (uint16_t)codes_of(x[2] * inv, x[3] * inv);
  }
  __device__ __forceinline__ static float largest(const float (&x)[4]) {
    return fmaxf(fmaxf(finite_abs(x[0]), finite_abs(x[1])), fmaxf(finite_abs(x[2]), finite_abs(x[3])));
  }

  // row t in block `blk`, whose scale is `before`
  __device__ __forceinline__ void append(int t, int blk, const float (&x)[4], float before) const {
    const int off = p.cache_pos[t] % kB8;
    const size_t at = place(blk);
    const float inv = rescale(at, before, largest(x), 1ull << off);
    write_back(t, x);
    store(at, off, x, inv);
  }
  // rows t .. end - 1, one after the other, so that a place named twice gets its last values
  __device__ __forceinline__ void append(int t, int end, int blk) const {
    const size_t at = place(blk);
    const float before = p.scales[at];
    float x[4], amax = 0.f;
    unsigned long long written = 0;
#pragma unroll 1
    for (int r = t; r < end; ++r) {
      load(r, x);
      amax = fmaxf(amax, largest(x));
      written |= 1ull << (p.cache_pos[r] % kB8);
    }
    const float inv = rescale(at, before, amax, written);
#pragma unroll 1
    for (int r = t; r < end; ++r) {
      load(r, x);
      write_back(r, x);
      store(at, p.cache_pos[r] % kB8, x, inv);
    }
  }
};

// Few rows, or rows of any alignment.  A block takes 1024 / D rows of a k or v head, D / 4 lanes each; single rows, as in a
// decoding step, are done without meeting the others: everything they read is asked for first, so that three round trips lead
// to the store (positions; block and angles; scale).  Of a run, the block that has its first row takes all rows at once.  The
// other blocks rotate q heads.  Short on purpose: a step's time is latency, that of fetching the code too.
template <int D>
__global__ void __launch_bounds__(256) append8_rows_kernel(Append8Params p, int kv_blocks) {
  constexpr int LPH = D / 4, S = 256 / LPH;
  __shared__ int s_first[S], s_last[kB8];
  __shared__ uint32_t s_same[3], s_top[8];
  chain_sync();
  const int tid = threadIdx.x, sub = tid / LPH;
  if ((int)blockIdx.x >= kv_blocks) {
    const long long unit = (blockIdx.x - kv_blocks) * (long long)S + sub;
    if (unit < (long long)p.T * p.Hq) RowLanes<D>(p, (int)(unit % p.Hq)).turn_only((int)(unit / p.Hq));
    return;
  }
  const int hd = blockIdx.x % (2 * p.Hkv), r0 = blockIdx.x / (2 * p.Hkv) * S, t = r0 + sub;
  const RowLanes<D> lanes(p, p.Hq + hd);
  bool several = false;
  if (t < p.T) {
    float x[4];
    const int blk = block_of(p, t), prev = t > 0 ? block_of(p, t - 1) : -1, next = t + 1 < p.T ? block_of(p, t + 1) : -1;
    if (blk < 0 || (blk != prev && blk != next)) {
      lanes.load(t, x);
      if (blk < 0) lanes.write_back(t, x);
      else lanes.append(t, blk, x, p.scales[lanes.place(blk)]);
    }
    several = blk >= 0 && blk != prev && blk == next;
  }
  if (tid % LPH == 0) s_first[sub] = several ? t : -1;
  if (!__syncthreads_or(several)) return;
  for (int i = 0; i < S; ++i) {
    const int first = s_first[i];
    if (first < 0) continue;
    const int blk = block_of(p, first);
    __syncthreads();      // the run before has been done
    if (tid < 96) {
      const int r = first + tid;
      const uint32_t same = __ballot_sync(0xffffffffu, tid <= kB8 && r < p.T && block_of(p, r) == blk);
      if ((tid & 31) == 0) s_same[tid >> 5] = same;
    }
    if (tid < kB8) s_last[tid] = -1;
    __syncthreads();
    // rows of the run: up to the first that is elsewhere
    const int n = ~s_same[0] ? __ffs(~s_same[0]) - 1 : ~s_same[1] ? 31 + __ffs(~s_same[1]) : 63 + __ffs(~s_same[2]);
    if (n > kB8) {        // some place is named twice, and the last row counts
      if (sub == 0) {
        int end = first + n;
        while (end < p.T && block_of(p, end) == blk) ++end;
        lanes.append(first, end, blk);
      }
      continue;
    }
    const size_t at = lanes.place(blk);
    const float before = p.scales[at];
    constexpr int M = kB8 / S;
    float x[M][4], amax = 0.f;
#pragma unroll
    for (int k = 0; k < M; ++k) {
      const int row = k * S + sub;
      if (row >= n) continue;
      lanes.load(first + row, x[k]);
      amax = fmaxf(amax, lanes.largest(x[k]));
      if (tid % LPH == 0) atomicMax(&s_last[p.cache_pos[first + row] % kB8], row);
    }
    const uint32_t top = __reduce_max_sync(0xffffffffu, __float_as_uint(amax));      // of numbers >= 0, bits order as they do
    if ((tid & 31) == 0) s_top[tid >> 5] = top;
    __syncthreads();
    uint32_t all = 0;
#pragma unroll
    for (int w = 0; w < 8; ++w) all = max(all, s_top[w]);
    const bool anew = s_last[0] >= 0;
    const float kept = anew ? 0.f : before, scale = fmaxf(kept, scale_of(__uint_as_float(all))), inv = 1.f / scale;
    if (scale != kept) {
      uint32_t* c = reinterpret_cast<uint32_t*>(p.codes + at * kB8 * D) + lanes.l;
#pragma unroll 4
      for (int r = sub; r < kB8; r += S)
        if (s_last[r] < 0) c[r * LPH] = anew ? 0u : rescaled(c[r * LPH], kept / scale);
      if (tid == 0) p.scales[at] = scale;
    }
#pragma unroll
    for (int k = 0; k < M; ++k) {
      const int row = k * S + sub;
      if (row >= n) continue;
      lanes.write_back(first + row, x[k]);
      const int off = p.cache_pos[first + row] % kB8;
      if (s_last[off] == row) lanes.store(at, off, x[k], inv);
    }
  }
}

// ---------------------------------------------------------------------------------------
// Rows on 16-byte boundaries.  The first blocks of the grid take k and v heads: some heads of 64 rows, of which those that
// are the first of a cache block's adjacent rows count (the block that has the first has all of them, up to 64, also where
// they reach beyond its range).  Single rows go to D / 4 lanes each; of more, every thread holds eight pairs in registers
// while the block finds the largest value, so that rows are read once.  The other blocks rotate q heads: a thread
// keeps the eight angles of its pairs for `per` heads.
//
// Bound by memory: 32 / 8 heads, D = 128, 32653 rows (819 MB): 145 us, 5.6 TB/s (with rows held in registers instead of asked for
// four heads ahead, 177); 28 / 4 heads, 8992 rows of 24 prompts (170 MB): 38 us; 421 rows of three partial sums (28 MB): 12.4 us.
// ---------------------------------------------------------------------------------------

// Eight pairs from element i0 on of one head of a row, not rotated.  bf16 rows are asked for several heads ahead: a thread's
// own places in shared memory take what would need registers, and nobody else reads them.  Partial sums (SLABS) are added up
// when they are needed.
constexpr int kAheadHeads = 4;
template <int D, bool SLABS>
struct Pairs {
  static constexpr int kThreads = 4 * D;
  static constexpr int kBytes = SLABS ? 0 : kAheadHeads * 2 * kThreads * 16;
  uint4* own;      // [kAheadHeads][2][threads], from this thread's place on
  __device__ __forceinline__ void ask(const Append8Params& p, int slot, bool any, int r, int head, int i0) const {
    if constexpr (!SLABS) {
      if (any) {
        const __nv_bfloat16* src = p.qkv + (size_t)r * p.row_stride + (size_t)head * D + i0;
#pragma unroll
        for (int half = 0; half < 2; ++half)
          asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(smem_u32(own + (slot * 2 + half) * kThreads)), "l"(src + half * (D / 2))
                       : "memory");
      }
      asm volatile("cp.async.commit_group;" ::: "memory");
    }
  }
  // what was asked for kAheadHeads calls of ask() ago, or before
  __device__ __forceinline__ void get(const Append8Params& p, int slot, int r, int head, int i0, float (&x)[8], float (&y)[8]) const {
    if constexpr (SLABS) {
      const float* src = p.slabs + ((size_t)r * (p.Hq + 2 * p.Hkv) + head) * D + i0;
      slab_sum8(src, p.slab_stride, p.splits, x);
      slab_sum8(src + D / 2, p.slab_stride, p.splits, y);
      if (p.bias) {
        const __nv_bfloat16* v = p.bias + head * D + i0;
#pragma unroll
        for (int k = 0; k < 8; ++k) {
          x[k] += __bfloat162float(v[k]);
          y[k] += __bfloat162float(v[D / 2 + k]);
        }
      }
    } else {
      asm volatile("cp.async.wait_group %0;" ::"n"(kAheadHeads - 1) : "memory");
      const uint4 a = own[slot * 2 * kThreads], b = own[(slot * 2 + 1) * kThreads];
      const uint32_t c[4] = {a.x, a.y, a.z, a.w}, d[4] = {b.x, b.y, b.z, b.w};
#pragma unroll
      for (int k = 0; k < 4; ++k) {
        x[2 * k] = __uint_as_float(c[k] << 16); x[2 * k + 1] = __uint_as_float(c[k] & 0xffff0000u);
        y[2 * k] = __uint_as_float(d[k] << 16); y[2 * k + 1] = __uint_as_float(d[k] & 0xffff0000u);
      }
    }
  }
};
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

template <int D, bool SLABS>
__global__ void __launch_bounds__(4 * D, SLABS ? 1 : 1024 / (4 * D)) append8_kernel(Append8Params p, int kv_blocks, int per_kv,
                                                                                   int per_q) {
  constexpr int range = kB8;              // rows of a block
  __shared__ int s_blk[2 * kB8 + 2];      // cache blocks of rows r0 - 1 .. r0 + range + 63
  __shared__ int s_last[kB8];             // last row of the run at each offset
  __shared__ uint32_t s_begin[5], s_top[2][D / 8];
  constexpr int TPR = D / 16;             // threads of a row, eight pairs each
  chain_sync();
  extern __shared__ uint4 s_ahead[];
  const int tid = threadIdx.x, q = tid % TPR, i0 = q * 8;
  const Pairs<D, SLABS> pairs{s_ahead + tid};
  // blocks of the two kinds take turns, so that the ones that wait and the ones that stream share the SMs
  const int i_kv = (int)((long long)blockIdx.x * kv_blocks / gridDim.x);
  if ((int)((long long)(blockIdx.x + 1) * kv_blocks / gridDim.x) == i_kv) {
    // ------------------------------ q heads ------------------------------
    const int b = blockIdx.x - i_kv, parts = (p.Hq + per_q - 1) / per_q;
    const int r = b / parts * 64 + tid / TPR, h0 = b % parts * per_q;
    if (r >= p.T) return;
    float c[8], s[8];
    const int h1 = min(h0 + per_q, p.Hq);
    for (int k = 0; k < kAheadHeads; ++k) pairs.ask(p, k, h0 + k < h1, r, h0 + k, i0);
    if (p.rope_pos) load_angles<D>(p, r, i0, c, s);
    for (int h = h0; h < h1; ++h) {
      const int slot = (h - h0) % kAheadHeads;
      float x[8], y[8];
      pairs.get(p, slot, r, h, i0, x, y);
      if (p.rope_pos) turn_pairs(x, y, c, s);
      pairs.ask(p, slot, h + kAheadHeads < h1, r, h + kAheadHeads, i0);
      store_pairs<D>(p, r, h, i0, x, y);
    }
    return;
  }
  // ------------------------------ k or v heads ------------------------------
  const int parts = (p.Hkv + per_kv - 1) / per_kv, kv = i_kv % (2 * parts) / parts;
  const int g0 = i_kv % parts * per_kv, g1 = min(g0 + per_kv, p.Hkv);                    // kv heads
  const int r0 = i_kv / (2 * parts) * range, rows = min(range, p.T - r0);
  const int head0 = p.Hq + kv * p.Hkv;
  if (tid < range + kB8 + 1) {
    const int t = r0 - 1 + tid;
    s_blk[tid] = t >= 0 && t < p.T ? block_of(p, t) : -1;
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
  // single rows, and runs that name a place twice
  for (int i = tid / (D / 4); i < rows; i += 16) {
    const int blk = s_blk[i + 1], t = r0 + i;
    int end = t;
    if (blk >= 0) {
      if (s_blk[i] == blk) continue;
      end = r0 + next(i + 1);
      if (end - t > 1 && end - t <= kB8) continue;
      if (end - t > kB8)
        while (end < p.T && block_of(p, end) == blk) ++end;
    }
    for (int g = g0; g < g1; ++g) {
      const RowLanes<D> lanes(p, head0 + g);
      if (blk < 0) {
        lanes.turn_only(t);
      } else if (end > t + 1) {
        lanes.append(t, end, blk);
      } else {
        float x[4];
        lanes.load(t, x);
        lanes.append(t, blk, x, p.scales[lanes.place(blk)]);
      }
    }
  }
  const bool turns = p.rope_pos && !kv;
  for (int i = next(0), e; i < rows; i = e) {
    e = next(i + 1);
    const int blk = s_blk[i + 1], t = r0 + i, n = e - i;
    if (blk < 0 || n < 2 || n > kB8) continue;
    const int row = tid / TPR, r = t + row;
    const bool mine = row < n;
    const size_t at0 = ((size_t)blk * 2 + kv) * p.Hkv;
    float c[8], s[8], before = p.scales[at0 + g0];
    int off = 0;
    for (int k = 0; k < kAheadHeads; ++k) pairs.ask(p, k, mine && g0 + k < g1, r, head0 + g0 + k, i0);      // all: per_kv is at most that
    if (mine) {
      off = p.cache_pos[r] % kB8;
      if (turns) load_angles<D>(p, r, i0, c, s);
    }
    __syncthreads();      // the run before has been done
    if (tid < kB8) s_last[tid] = -1;
    __syncthreads();
    if (mine && q == 0) atomicMax(&s_last[off], row);
    for (int g = g0; g < g1; ++g) {
      float x[8], y[8], amax = 0.f;
      if (mine) {
        pairs.get(p, g - g0, r, head0 + g, i0, x, y);
        if (turns) turn_pairs(x, y, c, s);
#pragma unroll
        for (int k = 0; k < 8; ++k) amax = fmaxf(amax, fmaxf(finite_abs(x[k]), finite_abs(y[k])));
      }
      // of numbers >= 0, bits order as they do
      const uint32_t top = __reduce_max_sync(0xffffffffu, __float_as_uint(amax));
      if ((tid & 31) == 0) s_top[g & 1][tid >> 5] = top;
      pairs.ask(p, 0, false, 0, 0, 0);      // counts as a turn
      const float now = before;
      if (g + 1 < g1) before = p.scales[at0 + g + 1];      // while this one's largest value is found
      __syncthreads();
      uint32_t all = 0;
#pragma unroll
      for (int w = 0; w < D / 8; ++w) all = max(all, s_top[g & 1][w]);
      const bool anew = s_last[0] >= 0;
      const float kept = anew ? 0.f : now, scale = fmaxf(kept, scale_of(__uint_as_float(all))), inv = 1.f / scale;
      uint8_t* dst = p.codes + (at0 + g) * kB8 * D;
      if (scale != kept) {
        if (s_last[row] < 0) {      // the row at this offset is not the call's
          const float ratio = kept / scale;
          uint4* to = reinterpret_cast<uint4*>(dst + row * D) + q;
          const uint4 v = *to;
          *to = anew ? make_uint4(0u, 0u, 0u, 0u)
                     : make_uint4(rescaled(v.x, ratio), rescaled(v.y, ratio), rescaled(v.z, ratio), rescaled(v.w, ratio));
        }
        if (tid == 0) p.scales[at0 + g] = scale;
      }
      if (mine) {
        if (s_last[off] == row) {
          *reinterpret_cast<uint2*>(dst + off * D + i0) = codes_of8(x, inv);
          *reinterpret_cast<uint2*>(dst + off * D + D / 2 + i0) = codes_of8(y, inv);
        }
        if (turns || SLABS) store_pairs<D>(p, r, head0 + g, i0, x, y);
      }
    }
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
extern "C" int sb_kv8_append(void* qkv, long long row_stride, const float* slabs, long long slab_stride, int splits,
                             const void* bias, const int* rope_pos, int pos_rows, int sec0, int sec1, int table_rows,
                             const float* cos_tab, const float* sin_tab, const int* seq_ids, const int* cache_pos,
                             const int* block_table, int sequences, int max_blocks, void* codes, float* scales,
                             int num_blocks, int T, int Hq, int Hkv, int D, cudaStream_t stream) {
  if (T == 0) return 0;
  if (D != 64 && D != 128) return -2;
  if (row_stride % 2 || reinterpret_cast<uintptr_t>(qkv) % 4 || reinterpret_cast<uintptr_t>(slabs) % 8 || (slabs && (splits < 1 || slab_stride % 2)) || (rope_pos && table_rows < 1)) return -3;
  Append8Params p;
  p.qkv = (__nv_bfloat16*)qkv; p.row_stride = row_stride; p.slabs = slabs; p.slab_stride = slab_stride; p.splits = splits;
  p.bias = (const __nv_bfloat16*)bias; p.rope_pos = rope_pos; p.pos_rows = pos_rows; p.sec0 = sec0; p.sec1 = sec1;
  p.table_rows = table_rows; p.cos_tab = cos_tab; p.sin_tab = sin_tab; p.seq_ids = seq_ids; p.cache_pos = cache_pos;
  p.block_table = block_table; p.sequences = sequences; p.max_blocks = max_blocks; p.codes = (uint8_t*)codes;
  p.scales = scales; p.num_blocks = num_blocks; p.T = T; p.Hq = Hq; p.Hkv = Hkv;
  auto on = [](const void* x) { return reinterpret_cast<uintptr_t>(x) % 16 == 0; };
  // At most as many rows as the table has sequences may be a decoding step, where the second kernel would go from row to row (256
  // rows, 28 / 4 heads, D = 128: 7.4 us against 22.7; 1000: 24 against 28).  More rows come in runs (60 rows of one prompt: 7.9 either
  // way).  What the rows are is not known here: prompts of more than 128 rows but no more than the table has sequences take the
  // first kernel as well, which is slower for them (three prompts, table of 1024: 460 rows 13.5 us against 9.2, 886: 21.0 against 10.7).
  if (T <= 128 || T <= sequences || row_stride % 8 || !on(qkv) || !on(slabs) || slab_stride % 4 || !on(cos_tab) || !on(sin_tab)) {
    const int rows = 1024 / D;
    const long long kv = (long long)((T + rows - 1) / rows) * 2 * Hkv;
    const long long q = rope_pos || slabs ? ((long long)T * Hq + rows - 1) / rows : 0;
    if (kv + q > 0x7fffffffll) return -4;
    return launch_chained(D == 128 ? append8_rows_kernel<128> : append8_rows_kernel<64>, (unsigned)(kv + q), 256, 0, stream, p, (int)kv);
  }
  // Several heads for what a block finds out about its rows, as long as every SM gets two blocks (8992 rows, 28 / 4 heads: 38 us; four
  // blocks: 43)
  const int ranges = (T + kB8 - 1) / kB8;
  auto blocks_of = [](long long n, int heads, int per) { return n * ((heads + per - 1) / per); };
  int per_kv = kAheadHeads, per_q = 16;
  while (per_kv > 1 && blocks_of(2 * ranges, Hkv, per_kv) < 2 * num_sms()) per_kv /= 2;
  while (per_q > 1 && blocks_of(ranges, Hq, per_q) < 2 * num_sms()) per_q /= 2;
  const long long kv = blocks_of(2 * ranges, Hkv, per_kv);
  const long long q = rope_pos || slabs ? blocks_of(ranges, Hq, per_q) : 0;
  if (kv + q > 0x7fffffffll) return -4;
  auto launch = [&](auto kernel, int bytes) {
    const cudaError_t e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, bytes);
    if (e != cudaSuccess) return (int)e;
    return launch_chained(kernel, (unsigned)(kv + q), 4 * D, bytes, stream, p, (int)kv, per_kv, per_q);
  };
  if (slabs) return D == 128 ? launch(append8_kernel<128, true>, 0) : launch(append8_kernel<64, true>, 0);
  return D == 128 ? launch(append8_kernel<128, false>, Pairs<128, false>::kBytes) : launch(append8_kernel<64, false>, Pairs<64, false>::kBytes);
}

extern "C" int sb_kv8_copy_blocks(void* codes, float* scales, const int* src, const int* dst, int n_pairs, int num_blocks,
                                  int per_block, long long bytes, cudaStream_t stream) {
  if (n_pairs == 0) return 0;
  if (bytes % 16) return -3;
  copy8_blocks_kernel<<<dim3(8, n_pairs < 4096 ? n_pairs : 4096), 256, 0, stream>>>((uint8_t*)codes, scales, src, dst, n_pairs,
                                                                                     num_blocks, per_block, bytes);
  return (int)cudaGetLastError();
}
