// 8-bit key/value cache in pages: quantising write and dequantising read.
//
//   write: a = max(max |x|, 2^-100) over a row's head, scale = a / M,
//          code = round(x * (M / a)), M = 448 (e4m3) or 127 (int8)
//   read:  y = 16-bit(code * scale)
//
// One 32-bit scale per row and head (4 bytes beside 128 codes).  M / a is one
// IEEE division a row; the product's rounding is followed by the 8-bit one.
// The floor 2^-100 keeps M / a finite and makes a row of zeros zeros.  A row
// with inf or NaN gets an infinite or NaN scale and reads back as NaN
// throughout, in int8 too, which has no code for it.
//
// Both kernels move 16 bits and 8 bits per value and no more, and are bound by
// HBM: a thread holds 8 values (16 bytes of the 16-bit row, 8 of codes), a row
// of 128 is 16 lanes.  A CTA takes all heads of a few rows, whose page lookups
// it does once.  Two rows a thread and eight CTAs an SM: reading 32760 rows of
// 40 heads back (1.02 GB moved) 165 us, 6.2 TB/s, writing 4680 rows (145 MB)
// 31.5 us, 20000 rows 107 us (5.8 TB/s); four rows a thread and fewer CTAs take
// 167-196 us to read, streaming stores 174-179.
#include "ps_b200.h"
#include "internal.h"
#include "ptx.cuh"

#include <cuda_bf16.h>
#include <cuda_fp16.h>

namespace psb {
namespace cache {

constexpr int kThreads = 256;
constexpr int kMaxTokens = 32;  // rows of one CTA
constexpr float kFloor = 7.888609052210118e-31f;  // 2^-100

__device__ __forceinline__ float max_nan(float a, float b) {
  float d;
  asm("max.NaN.f32 %0, %1, %2;" : "=f"(d) : "f"(a), "f"(b));
  return d;
}

template <bool kFp16>
__device__ __forceinline__ void widen8(const uint4& v, float (&f)[8]) {
  const uint32_t w[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    if constexpr (kFp16) {
      const float2 t = __half22float2(*reinterpret_cast<const __half2*>(&w[i]));
      f[2 * i] = t.x;
      f[2 * i + 1] = t.y;
    } else {
      f[2 * i] = __uint_as_float(w[i] << 16);
      f[2 * i + 1] = __uint_as_float(w[i] & 0xffff0000u);
    }
  }
}

template <bool kFp16>
__device__ __forceinline__ uint4 narrow8(const float (&f)[8]) {
  uint32_t w[4];
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    if constexpr (kFp16) {
      const __half2 t = __floats2half2_rn(f[2 * i], f[2 * i + 1]);
      w[i] = *reinterpret_cast<const uint32_t*>(&t);
    } else {
      const __nv_bfloat162 t = __floats2bfloat162_rn(f[2 * i], f[2 * i + 1]);
      w[i] = *reinterpret_cast<const uint32_t*>(&t);
    }
  }
  return make_uint4(w[0], w[1], w[2], w[3]);
}

// inv is 0 (of inf) or NaN in a row that has inf or NaN.
template <bool kInt8>
__device__ __forceinline__ uint2 encode8(const float (&f)[8], float inv) {
  uint32_t w[2];
#pragma unroll
  for (int i = 0; i < 2; ++i) {
    float y[4];
    if constexpr (kInt8) {
      // Adding 1.5 * 2^23 rounds to a whole number and leaves it in the low bits.
      // (In pairs the two instructions become one fused one, which rounds once.)
#pragma unroll
      for (int j = 0; j < 4; ++j) y[j] = __fadd_rn(__fmul_rn(f[4 * i + j], inv), 12582912.f);
      const uint32_t lo = __byte_perm(__float_as_uint(y[0]), __float_as_uint(y[1]), 0x0040);
      const uint32_t hi = __byte_perm(__float_as_uint(y[2]), __float_as_uint(y[3]), 0x0040);
      w[i] = inv > 0.f ? __byte_perm(lo, hi, 0x5410) : 0u;
    } else {
      mul2(y[0], y[1], f[4 * i], f[4 * i + 1], inv);
      mul2(y[2], y[3], f[4 * i + 2], f[4 * i + 3], inv);
      uint16_t lo, hi;
      asm("cvt.rn.satfinite.e4m3x2.f32 %0, %1, %2;" : "=h"(lo) : "f"(y[1]), "f"(y[0]));
      asm("cvt.rn.satfinite.e4m3x2.f32 %0, %1, %2;" : "=h"(hi) : "f"(y[3]), "f"(y[2]));
      w[i] = lo | (static_cast<uint32_t>(hi) << 16);
    }
  }
  return make_uint2(w[0], w[1]);
}

template <bool kInt8>
__device__ __forceinline__ void decode8(const uint2& v, float scale, float (&f)[8]) {
  const uint32_t w[2] = {v.x, v.y};
#pragma unroll
  for (int i = 0; i < 2; ++i) {
    if constexpr (kInt8) {
#pragma unroll
      for (int j = 0; j < 4; ++j) f[4 * i + j] = static_cast<float>(static_cast<int8_t>(w[i] >> (8 * j))) * scale;
    } else {
#pragma unroll
      for (int j = 0; j < 2; ++j) {
        uint32_t h;
        asm("cvt.rn.f16x2.e4m3x2 %0, %1;" : "=r"(h) : "h"(static_cast<uint16_t>(w[i] >> (16 * j))));
        const float2 t = __half22float2(*reinterpret_cast<const __half2*>(&h));
        mul2(f[4 * i + 2 * j], f[4 * i + 2 * j + 1], t.x, t.y, scale);
      }
    }
  }
}

// Pool row of position first + i of a sequence; -1 outside its table or pages.
__device__ __forceinline__ int64_t pool_row(const CacheArgs& a, int batch, int64_t pos) {
  if (pos < 0) return -1;
  const int64_t at = pos / a.page_rows;
  if (at >= a.table_len) return -1;
  const int page = a.table[batch * a.table_st + at];
  if (page < 0 || page >= a.num_pages) return -1;
  return static_cast<int64_t>(page) * a.page_rows + (pos - at * a.page_rows);
}

// The largest magnitude of two rows in one reduction: the bits of |x| order
// like the numbers (NaN above inf), so the rows' maxima are the 16-bit halves
// of a word.  Half of a row's lanes then work on each row's scale.  (Row by row
// in 32 bits, instructions were issued in 78 % of the cycles: 33.8 us and 122 us
// for the sizes above.)
//
// grid: (groups of `tokens` rows, batch, K or V)
template <bool kFp16, bool kInt8, int kLanes>
__global__ void __launch_bounds__(kThreads, 8) cache_write_kernel(const CacheArgs a, int tokens, unsigned magic) {
  constexpr int kDim = kLanes * 8, kRows = kThreads / kLanes;
  __shared__ int64_t slot[kMaxTokens];  // of head 0, or -1
  const int batch = blockIdx.y, t = blockIdx.z;
  const int i0 = blockIdx.x * tokens;
  if (threadIdx.x < tokens) {
    const int i = i0 + threadIdx.x;
    const int used = a.count ? min(a.count[batch], a.n) : a.n;
    const int64_t row = i < used ? pool_row(a, batch, int64_t(i) + (a.first ? a.first[batch] : 0)) : -1;
    slot[threadIdx.x] = row < 0 ? -1 : row * a.heads;
  }
  __syncthreads();
  const int lane = threadIdx.x % kLanes, grp = threadIdx.x / kLanes;
  const int rows = min(tokens, a.n - i0) * a.heads;
  const uint16_t* x = static_cast<const uint16_t*>(a.rows[t]) + batch * a.st[t][0] + i0 * a.st[t][1] + lane * 8;
  constexpr float kMost = kInt8 ? 127.f : 448.f;
  for (int j0 = 0; j0 < rows; j0 += kRows * 2) {
    uint4 v[2];
    int64_t at[2];
    uint32_t big[2];
#pragma unroll
    for (int u = 0; u < 2; ++u) {
      const int j = j0 + u * kRows + grp;
      at[u] = -1;
      v[u] = make_uint4(0, 0, 0, 0);
      if (j < rows) {
        const int tok = a.heads == 1 ? j : __umulhi(j, magic), h = j - tok * a.heads;
        if (slot[tok] >= 0) {
          at[u] = slot[tok] + h;
          v[u] = __ldcs(reinterpret_cast<const uint4*>(x + tok * a.st[t][1] + h * a.st[t][2]));
        }
      }
    }
#pragma unroll
    for (int u = 0; u < 2; ++u)
      big[u] = __vmaxu2(__vmaxu2(v[u].x & 0x7fff7fffu, v[u].y & 0x7fff7fffu),
                        __vmaxu2(v[u].z & 0x7fff7fffu, v[u].w & 0x7fff7fffu));
    uint32_t both = __vmaxu2(__byte_perm(big[0], big[1], 0x5410), __byte_perm(big[0], big[1], 0x7632));
#pragma unroll
    for (int o = kLanes / 2; o; o >>= 1) both = __vmaxu2(both, __shfl_xor_sync(0xffffffffu, both, o));
    const bool second = lane & (kLanes / 2);
    float m;
    if constexpr (kFp16) {
      const float2 f = __half22float2(*reinterpret_cast<const __half2*>(&both));
      m = second ? f.y : f.x;
    } else {
      m = __uint_as_float(second ? both & 0xffff0000u : both << 16);
    }
    m = max_nan(m, kFloor);
    const float inv = __fdiv_rn(kMost, m);
    const int64_t mine = second ? at[1] : at[0];
    if (lane % (kLanes / 2) == 0 && mine >= 0) a.scales[t][mine] = m * (1.f / kMost);
#pragma unroll
    for (int u = 0; u < 2; ++u) {
      const float by = __shfl_sync(0xffffffffu, inv, u * (kLanes / 2), kLanes);
      if (at[u] < 0) continue;
      float f[8];
      widen8<kFp16>(v[u], f);
      static_cast<uint2*>(a.pages[t])[at[u] * (kDim / 8) + lane] = encode8<kInt8>(f, by);
    }
  }
}

template <bool kFp16, bool kInt8, int kLanes>
__global__ void __launch_bounds__(kThreads, 8) cache_read_kernel(const CacheArgs a, int tokens, unsigned magic) {
  constexpr int kDim = kLanes * 8, kRows = kThreads / kLanes, kUnroll = 2;
  constexpr int64_t kSkip = -2;  // behind the sequence: left as it is
  __shared__ int64_t slot[kMaxTokens];
  const int batch = blockIdx.y, t = blockIdx.z;
  const int i0 = blockIdx.x * tokens;
  if (threadIdx.x < tokens) {
    const int i = i0 + threadIdx.x;
    const int64_t pos = int64_t(i) + (a.first ? a.first[batch] : 0);
    const int64_t row = i < a.n && pos < a.count[batch] ? pool_row(a, batch, pos) : kSkip;
    slot[threadIdx.x] = row < 0 ? row : row * a.heads;
  }
  __syncthreads();
  const int lane = threadIdx.x % kLanes, grp = threadIdx.x / kLanes;
  const int rows = min(tokens, a.n - i0) * a.heads;
  uint16_t* y = static_cast<uint16_t*>(a.rows[t]) + batch * a.st[t][0] + i0 * a.st[t][1] + lane * 8;
  for (int j0 = 0; j0 < rows; j0 += kRows * kUnroll) {
    uint2 v[kUnroll];
    float scale[kUnroll];
    uint16_t* to[kUnroll];
#pragma unroll
    for (int u = 0; u < kUnroll; ++u) {
      const int j = j0 + u * kRows + grp;
      to[u] = nullptr;
      v[u] = make_uint2(0, 0);  // a position without a page reads as zeros
      scale[u] = 0.f;
      if (j < rows) {
        const int tok = a.heads == 1 ? j : __umulhi(j, magic), h = j - tok * a.heads;
        if (slot[tok] != kSkip) to[u] = y + tok * a.st[t][1] + h * a.st[t][2];
        if (slot[tok] >= 0) {
          const int64_t at = slot[tok] + h;
          v[u] = __ldcs(static_cast<const uint2*>(a.pages[t]) + at * (kDim / 8) + lane);
          scale[u] = a.scales[t][at];
        }
      }
    }
#pragma unroll
    for (int u = 0; u < kUnroll; ++u) {
      if (!to[u]) continue;
      float f[8];
      decode8<kInt8>(v[u], scale[u], f);
      *reinterpret_cast<uint4*>(to[u]) = narrow8<kFp16>(f);
    }
  }
}

template <bool kWrite, bool kFp16, bool kInt8, int kLanes>
int launch(const CacheArgs& a, cudaStream_t stream) {
  // About 128 rows of one head a CTA; fewer, down to one pass, while all CTAs
  // still (nearly) run at a time, 8 on each of 148 SMs.  (us, 128 rows and fewer:
  // writing 8 rows of 12 heads 3.8 and 2.5, 3 x 311 of 10 5.8 and 4.1, 2 x 1000 of
  // 4 heads of 256 7.4 and 4.5; reading 1000 of 40 7.6 and 6.8, but 4 x 2000 of 8
  // heads of 64 in two rounds 5.8 and 6.4.)
  constexpr int kOnce = 2 * kThreads / kLanes;  // rows of one pass
  const int64_t all = int64_t(a.n) * a.batch * a.heads * 2;
  int per = 128;
  while (per > kOnce && all <= int64_t(per) * 5 * 148) per /= 2;
  int tokens = (per + a.heads - 1) / a.heads;
  tokens = tokens > kMaxTokens ? kMaxTokens : tokens;
  const int64_t groups = (int64_t(a.n) + tokens - 1) / tokens;
  const dim3 grid(static_cast<unsigned>(groups), static_cast<unsigned>(a.batch), 2);
  // j / heads for j < 2^16 as a high product
  const unsigned magic = a.heads > 1 ? static_cast<unsigned>((uint64_t(1) << 32) / a.heads + 1) : 0;
  if constexpr (kWrite)
    cache_write_kernel<kFp16, kInt8, kLanes><<<grid, kThreads, 0, stream>>>(a, tokens, magic);
  else
    cache_read_kernel<kFp16, kInt8, kLanes><<<grid, kThreads, 0, stream>>>(a, tokens, magic);
  const cudaError_t err = cudaGetLastError();
  if (err != cudaSuccess) return set_cuda_error(kWrite ? "cache write launch" : "cache read launch", err);
  count_launch();
  return 0;
}

template <bool kWrite, bool kFp16, bool kInt8>
int by_dim(const CacheArgs& a, cudaStream_t stream) {
  switch (a.head_dim) {
    case 64: return launch<kWrite, kFp16, kInt8, 8>(a, stream);
    case 128: return launch<kWrite, kFp16, kInt8, 16>(a, stream);
    case 256: return launch<kWrite, kFp16, kInt8, 32>(a, stream);
  }
  return set_error(PS_B200_ERR_UNSUPPORTED, "the cache holds heads of 64, 128 or 256 (got %d)", a.head_dim);
}

template <bool kWrite>
int by_type(const CacheArgs& a, bool fp16, bool int8, cudaStream_t stream) {
  if (fp16) return int8 ? by_dim<kWrite, true, true>(a, stream) : by_dim<kWrite, true, false>(a, stream);
  return int8 ? by_dim<kWrite, false, true>(a, stream) : by_dim<kWrite, false, false>(a, stream);
}

}  // namespace cache

int launch_cache_write(const CacheArgs& a, bool fp16, bool int8, cudaStream_t stream) {
  return cache::by_type<true>(a, fp16, int8, stream);
}

int launch_cache_read(const CacheArgs& a, bool fp16, bool int8, cudaStream_t stream) {
  return cache::by_type<false>(a, fp16, int8, stream);
}

}  // namespace psb
