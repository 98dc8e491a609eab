// Which blocks of keys a block of queries attends: the mean row of each block,
// the score of every (query block, key block) pair, and the best of them.
//
//   mean_j  = (1/n) sum of the n rows in use of block j            (held in 32 bits)
//   s_ij    = <mean_q_i, mean_k_j>                                 (64 bits)
//   list_i  = the `keep` key blocks with the largest s_ij among those block i
//             may see; of equal scores the lower index wins; ascending order
//
// The scores are 64-bit sums of exact products of 32-bit means, and the means
// come from 64-bit sums, so that which block wins does not hang on the order
// of an addition: a score's rounding (2^-53) is far below the gap between two
// neighbours of a few thousand scores, where 32-bit sums (2^-24) would swap a
// pair in every few thousand lists.
#include "ps_b200.h"
#include "internal.h"
#include "ptx.cuh"

#include <cuda_fp16.h>

namespace psb {
namespace sparse {

constexpr int kHeadDim = 128;
constexpr int kThreads = 256;
constexpr int kWarps = kThreads / 32;
constexpr int kScoreRows = 64, kScoreKeys = 16 * kWarps;  // of one CTA of score_kernel

template <bool kFp16>
__device__ __forceinline__ void add8(double (&a)[8], const uint4& v) {
  const uint32_t w[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const float2 f = kFp16 ? __half22float2(*reinterpret_cast<const __half2*>(&w[i]))
                           : make_float2(__uint_as_float(w[i] << 16), __uint_as_float(w[i] & 0xffff0000u));
    a[2 * i] += static_cast<double>(f.x);
    a[2 * i + 1] += static_cast<double>(f.y);
  }
}

// A warp sums up to 32 rows of one block and pair of heads, 512 bytes a row;
// the warps that share a block lie in one CTA and add up through shared memory.
// Every value is added in 64 bits, as in the selection where it takes the
// queries' means itself: sums of values within 2^30 of each other are exact, so
// that both give the same means, and none overflows.  Bound by HBM and, close
// behind, the conversions to 64 bits (16 a clock and SM): every value is read
// once, 16 loads a thread in flight and three CTAs an SM.  97 MB in 23.2 us, 168 in
// 36.7, 335 in 64.7 (5.2 TB/s); adding four values in 32 bits first, which loses
// what they cancel, takes 20.7, 33.5 and 59.5, building the 64-bit numbers with
// whole-number instructions 23.0, 37.1 and 65.9; 8 loads 24.9, 37.4 and 67.8.
template <bool kFp16>
__global__ void __launch_bounds__(kThreads, 3) block_means_kernel(const MeansArgs args) {
  __shared__ double part[kWarps][32 * 9];
  launch_dependents();
  int64_t cta = blockIdx.x;
  const int t = cta >= args.t[0].ctas;
  if (t) cta -= args.t[0].ctas;
  const MeansTensor& x = args.t[t];
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int per = x.warps;  // warps of one block
  const int64_t item0 = cta * (kWarps / per);  // items: (batch, block, pair of heads)
  auto rows_of = [&](int64_t item, int& batch, int& blk, int& pair) {
    pair = static_cast<int>(item % x.head_pairs);
    const int64_t rest = item / x.head_pairs;
    blk = static_cast<int>(rest % x.blocks);
    batch = static_cast<int>(rest / x.blocks);
    const int len = x.lens ? min(max(x.lens[batch], 0), x.len) : x.len;
    return static_cast<int>(min(max(len - static_cast<int64_t>(blk) * x.block, int64_t(0)), int64_t(x.block)));
  };
  double sum[8] = {0, 0, 0, 0, 0, 0, 0, 0};
  if (item0 + warp / per < x.items) {
    int batch, blk, pair;
    const int rows = rows_of(item0 + warp / per, batch, blk, pair);
    const int head = pair * 2 + (lane >> 4);
    if (head < x.heads) {
      const char* base = static_cast<const char*>(x.x) +
                         2 * (batch * x.st[0] + static_cast<int64_t>(blk) * x.block * x.st[1] + head * x.st[2] +
                              (lane & 15) * 8);
      const int64_t step = x.st[1] * 2;
#pragma unroll 4
      for (int r = warp % per; r < rows; r += 4 * per) {
        uint4 v[4];
#pragma unroll
        for (int u = 0; u < 4; ++u) {
          const int row = r + u * per;
          v[u] = row < rows ? load_once(base + row * step) : make_uint4(0, 0, 0, 0);
        }
#pragma unroll
        for (int u = 0; u < 4; ++u) add8<kFp16>(sum, v[u]);
      }
    }
  }
#pragma unroll
  for (int e = 0; e < 8; ++e) part[warp][lane * 9 + e] = sum[e];
  __syncthreads();
  const int col = threadIdx.x;  // of the two heads' 256
  for (int g = 0; g < kWarps / per && item0 + g < x.items; ++g) {
    int batch, blk, pair;
    const int rows = rows_of(item0 + g, batch, blk, pair);
    if (pair * 2 + (col >> 7) >= x.heads) continue;
    double total = 0;
    for (int w = 0; w < per; ++w) total += part[g * per + w][(col >> 3) * 9 + (col & 7)];
    const int64_t at = (static_cast<int64_t>(batch) * x.blocks + blk) * x.heads + pair * 2;
    x.out[at * kHeadDim + col] = rows ? static_cast<float>(total / rows) : 0.f;
  }
}

// Whole numbers in the order of the scores; 0 is a block that may not be chosen.
// Of 64-bit scores, NaN is above every number (a block with NaN in it is
// attended, so that NaN is not hidden by the selection); of 32-bit ones it only
// says that the 64-bit score is needed, and ~0u is left free.
__device__ __forceinline__ unsigned long long order_key(double s) {
  if (s != s) return ~0ull;
  const unsigned long long u = static_cast<unsigned long long>(__double_as_longlong(s + 0.0));  // -0 is 0
  return (u >> 63) ? ~u : (u | (1ull << 63));
}
__device__ __forceinline__ uint32_t order_key(float s) {
  if (s != s) return ~0u - 1;
  const uint32_t u = __float_as_uint(s + 0.f);
  return (u >> 31) ? ~u : (u | (1u << 31));
}
__device__ __forceinline__ float of_key(uint32_t k) {
  return __uint_as_float((k >> 31) ? (k & 0x7fffffffu) : ~k);
}

// x = hi + lo + at most 2^-17 x, two bf16 numbers (of 8 bits: lo is at most 2^-8 x); pairs of them packed for the tensor cores.
__device__ __forceinline__ void split_bf16(float x, float y, uint32_t& hi, uint32_t& lo) {
  hi = pack_bf16x2(x, y);
  lo = pack_bf16x2(x - __uint_as_float(hi << 16), y - __uint_as_float(hi & 0xffff0000u));
}

__device__ __forceinline__ void mma_bf16(float (&c)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
  asm volatile(
      "mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
      : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
      : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}

__device__ __forceinline__ int blocks_in_use(const int* len, int batch, int block, int blocks) {
  if (!len) return blocks;
  const int64_t n = max(len[batch], 0);
  return static_cast<int>(min(static_cast<int64_t>(blocks), (n + block - 1) / block));
}

// Scores of 64 rows (query blocks of the query heads that share a key head; one
// list each) against 128 key blocks, and the largest squared length of their means.
//
// On the tensor cores: each mean is split into two bf16 terms and the three
// larger products are summed in 32 bits, which is off by less than E = 2^-14
// |q| max |k| (the terms leave 2 * 2^-17, the dropped product 2^-16; 8 sums of
// the main products, 17 terms each, lose at most 2^-23 of their largest a term:
// 2^-15.9; the sums of the small products 2^-8 of that) plus what may underflow.
// pick_kernel turns to 64 bits where that decides.  (Two tf32 terms are closer,
// but take twice the products and, split between them, six times the other
// arithmetic: 24 against 11 us for 1182 key blocks and 296 query blocks of 5
// heads.)
//
// A tile is 16 key blocks x 8 rows.  The order of the 128 products is free, so
// a thread loads 16 bytes of a mean for one k-step of 16; a warp's 16 key means
// go from L2 to registers once, split, for all 64 rows.
__global__ void __launch_bounds__(kThreads, 2) score_kernel(const SelectArgs a) {
  constexpr int kPad = 32 + 4;  // of a row's 32 (hi, hi, lo, lo): 8 lanes' reads fall in different banks
  __shared__ uint4 qs[kScoreRows * kPad];
  __shared__ uint32_t longest;  // bits of the largest |k|^2 of this CTA's key blocks
  launch_dependents();
  wait_for_previous();  // the means
  const int rows = a.group * a.q_blocks;  // of one key head
  const int kv = (a.first_unit + blockIdx.z) % a.kv_heads;
  const int batch = (a.first_unit + blockIdx.z) / a.kv_heads;
  const int heads = a.kv_heads * a.group;
  const int row0 = blockIdx.y * kScoreRows;
  const int rows_here = min(kScoreRows, rows - row0);
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int g = lane >> 2, tig = lane & 3;
  const int k_blocks = blocks_in_use(a.k_len, batch, a.key_block, a.k_blocks);
  if (a.zeros && blockIdx.x + blockIdx.y + blockIdx.z == 0)
    for (int i = threadIdx.x; i < a.n_zeros; i += kThreads) a.zeros[i] = 0;

  if (threadIdx.x == 0) longest = 0;

  // The warp's key means, while the queries' are put in shared memory.
  const int n0 = blockIdx.x * kScoreKeys + warp * 16 + g;
  const float4* km = reinterpret_cast<const float4*>(a.k_means) +
                     (static_cast<int64_t>(batch) * a.k_blocks * a.kv_heads + kv) * (kHeadDim / 4) + tig;
  uint32_t kh[8][4], kl[8][4];
  float sq[2] = {0, 0};
#pragma unroll
  for (int half = 0; half < 2; ++half) {
    float4 v[2][4];
#pragma unroll
    for (int i = 0; i < 2; ++i)
#pragma unroll
      for (int j = 0; j < 4; ++j)
        v[i][j] = n0 + 8 * i < k_blocks ? __ldg(km + static_cast<int64_t>(n0 + 8 * i) * a.kv_heads * (kHeadDim / 4) +
                                                4 * (4 * half + j))
                                        : make_float4(0, 0, 0, 0);
#pragma unroll
    for (int i = 0; i < 2; ++i)
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const float4 x = v[i][j];
        sq[i] = fmaf(x.x, x.x, fmaf(x.y, x.y, fmaf(x.z, x.z, fmaf(x.w, x.w, sq[i]))));
        split_bf16(x.x, x.y, kh[4 * half + j][i], kl[4 * half + j][i]);
        split_bf16(x.z, x.w, kh[4 * half + j][2 + i], kl[4 * half + j][2 + i]);
      }
  }

  for (int r = warp; r < (rows_here + 7) / 8 * 8; r += kWarps) {
    const int row = row0 + r;
    float4 m = make_float4(0, 0, 0, 0);
    if (r < rows_here) {
      const int h = kv * a.group + row / a.q_blocks, qb = row % a.q_blocks;
      const int64_t at = ((static_cast<int64_t>(batch) * a.q_blocks + qb) * heads + h) * (kHeadDim / 4) + lane;
      if (a.q) {  // few query rows: their mean is taken here
        const int len = a.q_len ? min(max(a.q_len[batch], 0), a.len_q) : a.len_q;
        const int n = min(max(len - qb * a.query_block, 0), a.query_block);
        const uint16_t* x = static_cast<const uint16_t*>(a.q) + batch * a.q_st[0] +
                            static_cast<int64_t>(qb) * a.query_block * a.q_st[1] + h * a.q_st[2] + 4 * lane;
        double sum[4] = {0, 0, 0, 0};
#pragma unroll 4
        for (int i = 0; i < n; ++i) {
          const uint2 w2 = __ldg(reinterpret_cast<const uint2*>(x + i * a.q_st[1]));
          const uint32_t w[2] = {w2.x, w2.y};
#pragma unroll
          for (int e = 0; e < 2; ++e) {
            const float2 f = a.fp16 ? __half22float2(*reinterpret_cast<const __half2*>(&w[e]))
                                    : make_float2(__uint_as_float(w[e] << 16), __uint_as_float(w[e] & 0xffff0000u));
            sum[2 * e] += static_cast<double>(f.x);
            sum[2 * e + 1] += static_cast<double>(f.y);
          }
        }
        if (n) m = make_float4(float(sum[0] / n), float(sum[1] / n), float(sum[2] / n), float(sum[3] / n));
        if (blockIdx.x == 0) reinterpret_cast<float4*>(a.q_means)[at] = m;
      } else {
        m = __ldg(reinterpret_cast<const float4*>(a.q_means) + at);
      }
    }
    uint4 t;
    split_bf16(m.x, m.y, t.x, t.z);
    split_bf16(m.z, m.w, t.y, t.w);
    qs[r * kPad + lane] = t;
  }
  __syncthreads();

  const int64_t unit = blockIdx.z;
  if (blockIdx.y == 0) {
    uint32_t most = 0;
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      sq[i] += __shfl_xor_sync(0xffffffffu, sq[i], 1);
      sq[i] += __shfl_xor_sync(0xffffffffu, sq[i], 2);
      most = max(most, __float_as_uint(fabsf(sq[i])));  // NaN is above inf
    }
    most = __reduce_max_sync(0xffffffffu, most);
    if (lane == 0) atomicMax(&longest, most);
    __syncthreads();
    if (threadIdx.x == 0) a.k_sq[unit * gridDim.x + blockIdx.x] = longest;
  }
  float* scores = a.scores + (unit * rows + row0) * a.k_blocks;
#pragma unroll 2
  for (int t = 0; t < rows_here; t += 8) {
    float c[4] = {0, 0, 0, 0}, rest[4] = {0, 0, 0, 0};
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      const uint4 b = qs[(t + g) * kPad + 4 * j + tig];
      mma_bf16(c, kh[j], b.x, b.y);
      mma_bf16(rest, kl[j], b.x, b.y);
      mma_bf16(rest, kh[j], b.z, b.w);
    }
#pragma unroll
    for (int i = 0; i < 2; ++i)
#pragma unroll
      for (int e = 0; e < 2; ++e) {
        const int r = t + 2 * tig + e;
        if (r < rows_here && n0 + 8 * i < a.k_blocks)
          scores[static_cast<int64_t>(r) * a.k_blocks + n0 + 8 * i] = c[2 * i + e] + rest[2 * i + e];
      }
  }
}

// Sums over the CTA; consecutive calls alternate between two halves of `part`.
template <int kWarps>
struct CtaSum {
  int (*part)[kWarps];
  int phase;
  __device__ __forceinline__ int operator()(int v) {
    v = __reduce_add_sync(0xffffffffu, v);
    int* p = part[phase];
    phase ^= 1;
    if ((threadIdx.x & 31) == 0) p[threadIdx.x >> 5] = v;
    __syncthreads();
    int total = 0;
#pragma unroll
    for (int w = 0; w < kWarps; ++w) total += p[w];
    return total;
  }
};

// One CTA picks one list; a thread holds kPer of the scores, as keys in their
// order (block (warp * kPer + j) * 32 + lane).
//
// With T the keep-th largest score, a block above T + 2E is chosen and one
// below T - 2E is not, in 64 bits too; only the blocks between (the T block
// alone, in half of the lists) are scored again in 64 bits.
//
// T is found by counting the keys above a cut, first where the keep-th of as
// many normal scores lies, then where the counts at the ends put it on a
// straight line, every fourth time in the middle of the key range, until
// exactly `keep` lie above: 4.3 counts of 1182 normal scores, against 15 with
// bisection alone.
template <int kWarps, int kPer>
__global__ void __launch_bounds__(32 * kWarps) pick_kernel(const SelectArgs a) {
  extern __shared__ __align__(16) unsigned long long exact[];  // [k_blocks], used with many ties only
  __shared__ int part[2][kWarps];
  __shared__ uint32_t ends[3][kWarps];
  __shared__ float sums[2][kWarps];
  __shared__ int open_at[32];
  __shared__ unsigned long long open_key[32];
  __shared__ int n_open;
  launch_dependents();
  wait_for_previous();  // the scores
  const int rows = a.group * a.q_blocks;
  const int unit = blockIdx.x / rows, row = blockIdx.x - unit * rows;
  const int batch = (a.first_unit + unit) / a.kv_heads, kv = a.first_unit + unit - batch * a.kv_heads;
  const int heads = a.kv_heads * a.group;
  const int h = kv * a.group + row / a.q_blocks, qb = row % a.q_blocks;
  const int64_t list = (static_cast<int64_t>(batch) * heads + h) * a.q_blocks + qb;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const bool in_use = qb < blocks_in_use(a.q_len, batch, a.query_block, a.q_blocks);
  const int n_used = in_use ? blocks_in_use(a.k_len, batch, a.key_block, a.k_blocks) : 0;
  const int first = warp * kPer * 32 + lane;  // block of the thread's first key

  const float* score = a.scores + (static_cast<int64_t>(unit) * rows + row) * a.k_blocks;
  const uint8_t* allowed = a.allowed ? a.allowed + batch * a.allowed_st[0] + h * a.allowed_st[1] + qb * a.allowed_st[2]
                                     : nullptr;
  uint32_t key[kPer];
  uint32_t least = ~0u, most = 0;
  int n_may = 0;
  float s1 = 0, s2 = 0;  // sums of the scores and their squares
  {
    float x[kPer];
#pragma unroll
    for (int j = 0; j < kPer; ++j) x[j] = first + 32 * j < n_used ? __ldg(score + first + 32 * j) : 0.f;
#pragma unroll
    for (int j = 0; j < kPer; ++j) {
      const int i = first + 32 * j;
      const bool may = i < n_used && (!allowed || allowed[i * a.allowed_st[3]] != 0);
      key[j] = may ? order_key(x[j]) : 0u;
      n_may += may;
      s1 += may ? x[j] : 0.f;
      s2 += may ? x[j] * x[j] : 0.f;
      least = min(least, key[j] - 1);  // 0 becomes the largest
      most = max(most, key[j]);
    }
  }
  least = __reduce_min_sync(0xffffffffu, least);
  most = __reduce_max_sync(0xffffffffu, most);
#pragma unroll
  for (int o = 16; o; o >>= 1) {
    s1 += __shfl_xor_sync(0xffffffffu, s1, o);
    s2 += __shfl_xor_sync(0xffffffffu, s2, o);
  }
  if (lane == 0) {
    ends[0][warp] = least;
    ends[1][warp] = most;
    sums[0][warp] = s1;
    sums[1][warp] = s2;
  }
  if (threadIdx.x == 0) n_open = 0;
  CtaSum<kWarps> sum{part, 0};
  n_may = sum(n_may);  // and a barrier

  unsigned long long chosen = 0;  // bit j: key j
  if (n_may <= a.keep) {
#pragma unroll
    for (int j = 0; j < kPer; ++j) chosen |= static_cast<unsigned long long>(key[j] != 0) << j;
  } else {
    // T, the smallest key above `floor`.
    s1 = s2 = 0;
#pragma unroll
    for (int w = 0; w < kWarps; ++w) {
      least = min(least, ends[0][w]);
      most = max(most, ends[1][w]);
      s1 += sums[0][w];
      s2 += sums[1][w];
    }
    s1 = __fdividef(s1, static_cast<float>(n_may));
    const float spread = sqrtf(fmaxf(__fdividef(s2, static_cast<float>(n_may)) - s1 * s1, 0.f));
    float f = s1 - spread * normcdfinvf(__fdividef(static_cast<float>(a.keep), static_cast<float>(n_may)));
    uint32_t lo = least + 1, hi = most, floor = 0;
    int from_lo = n_may, above = 0;  // keys from lo up, keys above hi
    for (int round = 1;; ++round) {
      if (lo >= hi) {
        floor = lo - 1;
        break;
      }
      uint32_t mid = lo + ((hi - lo) >> 1) + 1;  // lo < mid <= hi
      if ((round & 3) && isfinite(f)) mid = min(max(order_key(f), lo + 1), hi);
      int c = 0;
#pragma unroll
      for (int j = 0; j < kPer; ++j) c += key[j] >= mid;
      c = sum(c);
      if (c == a.keep) {
        floor = mid - 1;
        break;
      }
      if (c > a.keep) {
        lo = mid;
        from_lo = c;
      } else {
        hi = mid - 1;
        above = c;
      }
      const float u = of_key(lo), v = of_key(hi);
      f = u + (v - u) * __fdividef(static_cast<float>(from_lo - a.keep), static_cast<float>(from_lo - above));
    }
    uint32_t kth = ~0u;
#pragma unroll
    for (int j = 0; j < kPer; ++j) kth = key[j] > floor ? min(kth, key[j]) : kth;
    kth = __reduce_min_sync(0xffffffffu, kth);
    if (lane == 0) ends[2][warp] = kth;
    const float4 q = __ldg(reinterpret_cast<const float4*>(a.q_means) +
                           ((static_cast<int64_t>(batch) * a.q_blocks + qb) * heads + h) * (kHeadDim / 4) + lane);
    float q_sq = fmaf(q.x, q.x, fmaf(q.y, q.y, fmaf(q.z, q.z, q.w * q.w)));
#pragma unroll
    for (int o = 16; o; o >>= 1) q_sq += __shfl_xor_sync(0xffffffffu, q_sq, o);
    uint32_t longest = 0;
    const int k_chunks = (a.k_blocks + kScoreKeys - 1) / kScoreKeys;
    for (int i = lane; i < k_chunks; i += 32) longest = max(longest, __ldg(a.k_sq + static_cast<int64_t>(unit) * k_chunks + i));
    longest = __reduce_max_sync(0xffffffffu, longest);
    __syncthreads();
#pragma unroll
    for (int w = 0; w < kWarps; ++w) kth = min(kth, ends[2][w]);
    const float T = of_key(kth);
    const float len_q = sqrtf(q_sq), len_k = sqrtf(__uint_as_float(longest));
    const float E2 = 1.220703125e-04f * len_q * len_k + 7.70371978e-34f * (1.f + len_q + len_k);  // 2^-13, 2^-110
    uint32_t lo_key = 1, hi_key = ~0u - 1;  // undecided: every block, where E says nothing
    // (Squares below 2^-100 of the lengths may have lost what they were made of to underflow.)
    const float least_sq = fminf(q_sq, __uint_as_float(longest));
    if (kth < ~0u - 1 && least_sq > 7.888609052210118e-31f && len_q * len_k < 1e38f && isfinite(T - E2) &&
        isfinite(T + E2)) {
      lo_key = order_key(T - E2);
      hi_key = order_key(T + E2);
    }
    int sure = 0;
#pragma unroll
    for (int j = 0; j < kPer; ++j) {
      sure += key[j] > hi_key;
      chosen |= static_cast<unsigned long long>(key[j] > hi_key) << j;
      if (key[j] >= lo_key && key[j] <= hi_key) {
        const int at = atomicAdd(&n_open, 1);  // in any order: they are ranked below
        if (at < 32) open_at[at] = first + 32 * j;
      }
    }
    const int wanted = a.keep - sum(sure);
    const int open = n_open;
    const float4* km = reinterpret_cast<const float4*>(a.k_means) +
                       (static_cast<int64_t>(batch) * a.k_blocks * a.kv_heads + kv) * (kHeadDim / 4);
    auto score64 = [&](int i) {  // by one warp
      const float4 k = __ldg(km + static_cast<int64_t>(i) * a.kv_heads * (kHeadDim / 4) + lane);
      double d = fma(double(q.x), double(k.x), double(q.y) * double(k.y)) +
                 fma(double(q.z), double(k.z), double(q.w) * double(k.w));
#pragma unroll
      for (int o = 16; o; o >>= 1) d += __shfl_xor_sync(0xffffffffu, d, o);
      return order_key(d);
    };
    if (open == wanted) {
#pragma unroll
      for (int j = 0; j < kPer; ++j) chosen |= static_cast<unsigned long long>(key[j] >= lo_key) << j;
    } else if (open <= 32) {
      for (int e = warp; e < open; e += kWarps) {
        const unsigned long long k = score64(open_at[e]);
        if (lane == 0) open_key[e] = k;
      }
      __syncthreads();
      for (int e = 0; e < open; ++e) {
        // Every thread ranks every open block and keeps its own.
        const int at = open_at[e];
        int better = 0;
        for (int o = lane; o < open; o += 32)
          better += open_key[o] > open_key[e] || (open_key[o] == open_key[e] && open_at[o] < at);
        better = __reduce_add_sync(0xffffffffu, better);
        const int j = (at - first) >> 5;
        if (better < wanted && ((at ^ first) & 31) == 0 && j >= 0 && j < kPer) chosen |= 1ull << j;
      }
    } else {
      // Many equal or overflowing scores: all that are open in 64 bits, and
      // the bisection of 64-bit keys (0: not open) for the wanted-th of them.
      for (int j = 0; j < kPer; ++j) {
        const int i0 = warp * kPer * 32 + 32 * j;
        for (int l = 0; l < 32 && i0 + l < a.k_blocks; ++l) {
          const uint32_t k = __shfl_sync(0xffffffffu, key[j], l);
          unsigned long long e = 0;
          if (k >= lo_key && k <= hi_key) e = score64(i0 + l);
          if (lane == 0) exact[i0 + l] = e;
        }
      }
      __syncwarp();
      const int begin = min(warp * kPer * 32, a.k_blocks), end = min(begin + kPer * 32, a.k_blocks);
      unsigned long long lo64 = 1, hi64 = ~0ull;
      int left = 0, over = 0;  // ties to be chosen; keys above hi64
      bool found = false;
      while (lo64 < hi64) {
        const unsigned long long mid = lo64 + ((hi64 - lo64) >> 1) + 1;
        int c = 0;
        for (int i = begin + lane; i < end; i += 32) c += exact[i] >= mid;
        c = sum(c);
        if (c == wanted) {
          lo64 = mid;
          found = true;
          break;
        }
        if (c > wanted) {
          lo64 = mid;
        } else {
          hi64 = mid - 1;
          over = c;
        }
      }
      // Chosen: keys above lo64, and as many that equal it as are still wanted
      // (all of them where the cut was exact), by index across the warps.
      int same = 0;
      for (int i = begin + lane; i < end; i += 32) same += exact[i] == lo64;
      same = __reduce_add_sync(0xffffffffu, same);
      __syncthreads();  // `part` may still be read
      if (lane == 0) part[0][warp] = same;
      __syncthreads();
      left = found ? a.k_blocks : wanted - over;
      for (int w = 0; w < warp; ++w) left = max(left - part[0][w], 0);
      for (int j = 0; j < kPer; ++j) {
        const int i = first + 32 * j;
        const unsigned long long e = i < end ? exact[i] : 0ull;
        const unsigned m = __ballot_sync(0xffffffffu, e == lo64);
        if (e > lo64 || (e == lo64 && __popc(m & ((1u << lane) - 1)) < left)) chosen |= 1ull << j;
        left = max(left - __popc(m), 0);
      }
    }
  }

  // The chosen in ascending order.
  int mine = __reduce_add_sync(0xffffffffu, __popcll(chosen));
  __syncthreads();  // `part` may still be read
  if (lane == 0) part[0][warp] = mine;
  __syncthreads();
  int done = 0, total = 0;
#pragma unroll
  for (int w = 0; w < kWarps; ++w) {
    if (w < warp) done += part[0][w];
    total += part[0][w];
  }
  int* out = a.blocks + list * a.keep;
#pragma unroll
  for (int j = 0; j < kPer; ++j) {
    const bool take = (chosen >> j) & 1;
    const unsigned m = __ballot_sync(0xffffffffu, take);
    if (take) out[done + __popc(m & ((1u << lane) - 1))] = first + 32 * j;
    done += __popc(m);
  }
  for (int i = total + threadIdx.x; i < a.keep; i += 32 * kWarps) out[i] = -1;
  if (threadIdx.x == 0) a.counts[list] = total;
}

// Few key blocks: scores and list in one kernel, all in 64 bits.
//
// A CTA makes one list.  Eight lanes take a key mean, 16 values each; then each
// block's place is the number of better ones, counted by as many threads as
// there are for it.  Against the two kernels above that saves a launch and the
// wait between them, but every CTA reads and converts the key means again and
// makes k_blocks^2 comparisons.  Measured (us, here and there): 12 lists of 32
// blocks 2.8 and 8-10, 192 of 32 3.5 and 10, 720 of 79 10.1 and 17.5, 40 of 250
// 8.4 and 11.3, 640 of 128 12.1 and 16.7; 160 of 256 13.6 and 11.9, 3000 of 64
// 26.6 and 24.2, 1280 of 256 38 and 22.
constexpr int kRankBlocks = 256;

__global__ void __launch_bounds__(kThreads, 4) rank_kernel(const SelectArgs a) {
  __shared__ __align__(16) double qs[kHeadDim];
  __shared__ double sums[kWarps][kHeadDim];
  __shared__ unsigned long long keys[kRankBlocks];
  __shared__ int better[kRankBlocks];
  __shared__ int taken[kWarps];  // chosen of each 32 blocks
  launch_dependents();
  wait_for_previous();  // the means
  const int rows = a.group * a.q_blocks;  // of one key head
  const int unit = blockIdx.x / rows, row = blockIdx.x - unit * rows;
  const int batch = unit / a.kv_heads, kv = unit - batch * a.kv_heads;
  const int heads = a.kv_heads * a.group;
  const int h = kv * a.group + row / a.q_blocks, qb = row % a.q_blocks;
  const int64_t list = (static_cast<int64_t>(batch) * heads + h) * a.q_blocks + qb;
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  const int n_used = qb < blocks_in_use(a.q_len, batch, a.query_block, a.q_blocks)
                         ? blocks_in_use(a.k_len, batch, a.key_block, a.k_blocks)
                         : 0;
  if (a.zeros && blockIdx.x == 0)
    for (int i = tid; i < a.n_zeros; i += kThreads) a.zeros[i] = 0;

  const int part = lane & 7;
  const float4* km = reinterpret_cast<const float4*>(a.k_means) +
                     (static_cast<int64_t>(batch) * a.k_blocks * a.kv_heads + kv) * (kHeadDim / 4) + part;
  auto load = [&](int j, float4 (&v)[4]) {
#pragma unroll
    for (int c = 0; c < 4; ++c)
      v[c] = j < n_used ? __ldg(km + static_cast<int64_t>(j) * a.kv_heads * (kHeadDim / 4) + 8 * c) : make_float4(0, 0, 0, 0);
  };
  float4 v[4];
  load(warp * 4 + (lane >> 3), v);

  if (a.q) {  // few query rows: their mean is taken here, a row to a warp
    const int len = a.q_len ? min(max(a.q_len[batch], 0), a.len_q) : a.len_q;
    const int n = min(max(len - qb * a.query_block, 0), a.query_block);
    const uint16_t* x = static_cast<const uint16_t*>(a.q) + batch * a.q_st[0] +
                        static_cast<int64_t>(qb) * a.query_block * a.q_st[1] + h * a.q_st[2] + 4 * lane;
    double sum[4] = {0, 0, 0, 0};
#pragma unroll 4
    for (int i = warp; i < n; i += kWarps) {
      const uint2 w2 = __ldg(reinterpret_cast<const uint2*>(x + i * a.q_st[1]));
      const uint32_t w[2] = {w2.x, w2.y};
#pragma unroll
      for (int e = 0; e < 2; ++e) {
        const float2 f = a.fp16 ? __half22float2(*reinterpret_cast<const __half2*>(&w[e]))
                                : make_float2(__uint_as_float(w[e] << 16), __uint_as_float(w[e] & 0xffff0000u));
        sum[2 * e] += static_cast<double>(f.x);
        sum[2 * e + 1] += static_cast<double>(f.y);
      }
    }
#pragma unroll
    for (int e = 0; e < 4; ++e) sums[warp][4 * lane + e] = sum[e];
    __syncthreads();
    if (tid < kHeadDim) {
      double total = 0;
#pragma unroll
      for (int w = 0; w < kWarps; ++w) total += sums[w][tid];
      qs[tid] = n ? static_cast<double>(static_cast<float>(total / n)) : 0.0;
    }
  } else if (tid < kHeadDim) {
    qs[tid] = static_cast<double>(
        __ldg(a.q_means + ((static_cast<int64_t>(batch) * a.q_blocks + qb) * heads + h) * kHeadDim + tid));
  }
  better[tid] = 0;
  __syncthreads();

  double q[16];  // the lane's pieces part, part + 8, ... of 16 bytes
#pragma unroll
  for (int i = 0; i < 16; ++i) q[i] = qs[4 * (part + 8 * (i >> 2)) + (i & 3)];
  const uint8_t* allowed = a.allowed ? a.allowed + batch * a.allowed_st[0] + h * a.allowed_st[1] + qb * a.allowed_st[2]
                                     : nullptr;
  for (int j0 = 0; j0 < a.k_blocks; j0 += 4 * kWarps) {
    const int j = j0 + warp * 4 + (lane >> 3);
    bool may = j < n_used;
    if (may && allowed && part == 0) may = allowed[j * a.allowed_st[3]] != 0;
    double d[2] = {0, 0};
#pragma unroll
    for (int c = 0; c < 4; ++c) {
      d[0] = fma(q[4 * c], double(v[c].x), d[0]);
      d[1] = fma(q[4 * c + 1], double(v[c].y), d[1]);
      d[0] = fma(q[4 * c + 2], double(v[c].z), d[0]);
      d[1] = fma(q[4 * c + 3], double(v[c].w), d[1]);
    }
    load(j + 4 * kWarps, v);
    d[0] += d[1];
#pragma unroll
    for (int o = 4; o; o >>= 1) d[0] += __shfl_xor_sync(0xffffffffu, d[0], o);
    if (part == 0 && j < a.k_blocks) keys[j] = may ? order_key(d[0]) : 0ull;
  }
  __syncthreads();

  // Thread tid counts a share of the blocks better than block tid % span.
  const int span = (a.k_blocks + 31) & ~31, shares = kThreads / span;
  const int share = tid / span, j = tid - share * span;
  if (share < shares && j < a.k_blocks) {
    // Of equals the lower index is better: before the warp's 32 blocks a key
    // counts from `key` on, behind them above it.  (What 0 counts does not matter, it is never chosen.)
    const unsigned long long key = keys[j], below = key - 1;
    const int begin = a.k_blocks * share / shares, end = a.k_blocks * (share + 1) / shares;
    const int own = j & ~31;
    int n = 0, i = begin;
#pragma unroll 8
    for (; i < min(own, end); ++i) n += keys[i] > below;
    for (; i < min(own + 32, end); ++i) n += keys[i] > (i < j ? below : key);
#pragma unroll 8
    for (; i < end; ++i) n += keys[i] > key;
    if (shares == 1)
      better[j] = n;
    else if (n)
      atomicAdd(&better[j], n);
  }
  __syncthreads();
  const bool take = tid < a.k_blocks && keys[tid] != 0 && better[tid] < a.keep;
  const unsigned m = __ballot_sync(0xffffffffu, take);
  if (lane == 0) taken[warp] = __popc(m);
  __syncthreads();
  int before = 0, total = 0;
#pragma unroll
  for (int w = 0; w < kWarps; ++w) {
    before += w < warp ? taken[w] : 0;
    total += taken[w];
  }
  int* out = a.blocks + list * a.keep;
  if (take) out[before + __popc(m & ((1u << lane) - 1))] = tid;
  for (int i = total + tid; i < a.keep; i += kThreads) out[i] = -1;
  if (tid == 0) a.counts[list] = total;
}

}  // namespace sparse

bool select_is_small(int64_t lists, int k_blocks) {
  return k_blocks <= sparse::kRankBlocks && lists * k_blocks * (k_blocks + 256) <= (1 << 25);
}

int launch_block_means(const MeansArgs& a, bool fp16, cudaStream_t stream) {
  using namespace sparse;
  const int64_t ctas = a.t[0].ctas + a.t[1].ctas;
  if (ctas == 0) return 0;
  if (ctas > 0x7fffffff) return set_error(PS_B200_ERR_UNSUPPORTED, "block_means: more than 2^31 blocks");
  if (fp16)
    block_means_kernel<true><<<static_cast<unsigned>(ctas), kThreads, 0, stream>>>(a);
  else
    block_means_kernel<false><<<static_cast<unsigned>(ctas), kThreads, 0, stream>>>(a);
  const cudaError_t err = cudaGetLastError();
  if (err != cudaSuccess) return set_cuda_error("block_means launch", err);
  count_launch();
  return 0;
}

int launch_block_select(SelectArgs a, cudaStream_t stream) {
  using namespace sparse;
  // Warps and keys a thread by the number of key blocks: 20 keys in registers
  // as long as eight warps hold the list, 64 beyond.
  const size_t smem = size_t(a.k_blocks) * 8;
  const int form = a.k_blocks <= 2 * 20 * 32 ? 0 : a.k_blocks <= 8 * 20 * 32 ? 1 : 2;
  void (*const pick)(const SelectArgs) = form == 0 ? pick_kernel<2, 20> : form == 1 ? pick_kernel<8, 20> : pick_kernel<8, 64>;
  static_assert(8 * 64 * 32 == kSelectMaxBlocks, "the largest list");
  static bool done[64] = {false};
  int dev = 0;
  if (cudaGetDevice(&dev) != cudaSuccess || dev < 0 || dev >= 64) dev = 0;
  if (form == 2 && !done[dev]) {  // the others stay below 48 KB
    const cudaError_t err =
        cudaFuncSetAttribute(pick_kernel<8, 64>, cudaFuncAttributeMaxDynamicSharedMemorySize, kSelectMaxBlocks * 8);
    if (err != cudaSuccess) return set_cuda_error("block_select: cudaFuncSetAttribute", err);
    done[dev] = true;
  }
  const int64_t rows = int64_t(a.group) * a.q_blocks;
  const int64_t row_chunks = (rows + kScoreRows - 1) / kScoreRows;
  if (row_chunks > 65535) return set_error(PS_B200_ERR_UNSUPPORTED, "block_select: more than 2^22 lists a key head");
  const int units = a.batch * a.kv_heads;
  if (select_is_small(units * rows, a.k_blocks)) {
    const cudaError_t err = launch_after(rank_kernel, dim3(static_cast<unsigned>(units * rows)), dim3(kThreads), 0,
                                         stream, a.after_means, a);
    if (err != cudaSuccess) return set_cuda_error("block_select launch", err);
    count_launch();
    return 0;
  }
  const int step = select_units(a.batch, a.kv_heads, a.group, a.q_blocks, a.k_blocks);
  for (a.first_unit = 0; a.first_unit < units; a.first_unit += step) {
    const int n = units - a.first_unit < step ? units - a.first_unit : step;
    const dim3 grid(static_cast<unsigned>((a.k_blocks + kScoreKeys - 1) / kScoreKeys), static_cast<unsigned>(row_chunks),
                    static_cast<unsigned>(n));
    cudaError_t err = launch_after(score_kernel, grid, dim3(kThreads), 0, stream, a.after_means, a);
    if (err != cudaSuccess) return set_cuda_error("block_select scores launch", err);
    count_launch();
    err = launch_after(pick, dim3(static_cast<unsigned>(n * rows)), dim3(form == 0 ? 64 : 256), smem, stream, true, a);
    if (err != cudaSuccess) return set_cuda_error("block_select launch", err);
    count_launch();
  }
  return 0;
}

}  // namespace psb
