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

// ---------------------------------------------------------------------------------------
// D / 4 lanes per (row, head): a lane holds elements 2 l, 2 l + 1 and their partners D / 2 further on.  The lanes that meet
// the first of the adjacent rows of a cache block do all of them, one after the other, so that one pass knows the block's
// new scale and a row named twice gets its last values.
// ---------------------------------------------------------------------------------------
template <int D>
__global__ void __launch_bounds__(256) append8_rows_kernel(Append8Params p) {
  chain_sync();
  constexpr int LPH = D / 4, half = D / 2;
  const int heads = p.Hq + 2 * p.Hkv;
  const int lane = threadIdx.x & 31, l = lane % LPH;
  const uint32_t mask = LPH == 32 ? 0xffffffffu : 0xffffu << (lane & 16);
  const long long unit = (blockIdx.x * 256ll + threadIdx.x) / LPH;
  if (unit >= (long long)p.T * heads) return;
  const int t = (int)(unit / heads), head = (int)(unit % heads);
  const bool turns = p.rope_pos != nullptr && head < p.Hq + p.Hkv;

  auto load = [&](int r, float (&x)[4]) {   // x[0..1]: elements 2 l, 2 l + 1, x[2..3]: their partners; rotated
    if (p.slabs) {
      const float* src = p.slabs + ((size_t)r * heads + head) * D + 2 * l;
#pragma unroll
      for (int i = 0; i < 4; ++i) x[i] = 0.f;
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
        const int prow = p.pos_rows == 3 ? (c < p.sec0 ? 0 : c < p.sec1 ? 1 : 2) : 0;
        const int at = min(max(p.rope_pos[(size_t)prow * p.T + r], 0), p.table_rows - 1);
        const float cs = p.cos_tab[(size_t)at * half + c], sn = p.sin_tab[(size_t)at * half + c];
        const float a = x[i];
        x[i] = a * cs - x[2 + i] * sn;
        x[2 + i] = x[2 + i] * cs + a * sn;
      }
    }
  };
  auto write_back = [&](int r, const float (&x)[4]) {
    if (!p.slabs && !turns) return;
    __nv_bfloat16* dst = p.qkv + (size_t)r * p.row_stride + (size_t)head * D + 2 * l;
    *reinterpret_cast<uint32_t*>(dst) = pack_bf16x2(x[0], x[1]);
    *reinterpret_cast<uint32_t*>(dst + half) = pack_bf16x2(x[2], x[3]);
  };

  float x[4];
  const int blk = head < p.Hq ? -1 : block_of(p, t);
  if (blk < 0) {
    load(t, x);
    write_back(t, x);
    return;
  }
  if (t > 0 && block_of(p, t - 1) == blk) return;   // the first row's lanes do this one
  int end = t;
  float amax = 0.f;
  unsigned long long written = 0;
  do {
    load(end, x);
#pragma unroll
    for (int i = 0; i < 4; ++i) amax = fmaxf(amax, finite_abs(x[i]));
    written |= 1ull << (p.cache_pos[end] % kB8);
    ++end;
  } while (end < p.T && block_of(p, end) == blk);
#pragma unroll
  for (int o = LPH / 2; o > 0; o >>= 1) amax = fmaxf(amax, __shfl_xor_sync(mask, amax, o));

  const int kv = head >= p.Hq + p.Hkv ? 1 : 0;
  const size_t at = ((size_t)blk * 2 + kv) * p.Hkv + (head - p.Hq - kv * p.Hkv);
  uint8_t* dst = p.codes + at * kB8 * D;
  const bool anew = written & 1;
  const float kept = anew ? 0.f : p.scales[at];
  const float scale = fmaxf(kept, scale_of(amax));
  __syncwarp(mask);
  if (scale != kept) {
    const float ratio = kept / scale;
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
  const long long blocks = ((long long)T * (Hq + 2 * Hkv) * (D / 4) + 255) / 256;
  if (blocks > 0x7fffffffll) return -4;
  return launch_chained(D == 128 ? append8_rows_kernel<128> : append8_rows_kernel<64>, (unsigned)blocks, 256, 0, stream, p);
}

extern "C" int sb_kv8_copy_blocks(void* codes, float* scales, const int* src, const int* dst, int n_pairs, int num_blocks,
                                  int per_block, long long bytes, cudaStream_t stream) {
  if (n_pairs == 0) return 0;
  if (bytes % 16) return -3;
  copy8_blocks_kernel<<<dim3(8, n_pairs < 4096 ? n_pairs : 4096), 256, 0, stream>>>((uint8_t*)codes, scales, src, dst, n_pairs,
                                                                                     num_blocks, per_block, bytes);
  return (int)cudaGetLastError();
}
