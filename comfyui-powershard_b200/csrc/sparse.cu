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

template <bool kFp16>
__device__ __forceinline__ void add8(float (&a)[8], const uint4& v) {
  const uint32_t w[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    if constexpr (kFp16) {
      const float2 f = __half22float2(*reinterpret_cast<const __half2*>(&w[i]));
      a[2 * i] += f.x;
      a[2 * i + 1] += f.y;
    } else {
      a[2 * i] += __uint_as_float(w[i] << 16);
      a[2 * i + 1] += __uint_as_float(w[i] & 0xffff0000u);
    }
  }
}

// One CTA per (block, pair of heads, batch row) of up to two tensors: a warp
// reads the 512 bytes that two heads of a row hold, the warps take the block's
// rows in turn, four rows at a time.  Four values are added in 32 bits (exact
// for 16-bit values within a few binades) before the 64-bit sum, which keeps
// the conversions to 64 bits (16 a clock and SM) at a quarter of the values.
template <bool kFp16>
__global__ void __launch_bounds__(kThreads) block_means_kernel(const MeansArgs args) {
  __shared__ double part[kWarps][32 * 9];
  launch_dependents();
  int64_t cta = blockIdx.x;
  const int t = cta >= args.t[0].ctas;
  if (t) cta -= args.t[0].ctas;
  const MeansTensor& x = args.t[t];
  const int pair = static_cast<int>(cta % x.head_pairs);
  cta /= x.head_pairs;
  const int blk = static_cast<int>(cta % x.blocks);
  const int batch = static_cast<int>(cta / x.blocks);
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int len = x.lens ? min(max(x.lens[batch], 0), x.len) : x.len;
  const int64_t first = static_cast<int64_t>(blk) * x.block;
  const int rows = static_cast<int>(min(max(len - first, int64_t(0)), int64_t(x.block)));
  const int head = pair * 2 + (lane >> 4);
  double sum[8] = {0, 0, 0, 0, 0, 0, 0, 0};
  if (head < x.heads) {
    const char* base = static_cast<const char*>(x.x) +
                       2 * (batch * x.st[0] + first * x.st[1] + head * x.st[2] + (lane & 15) * 8);
    const int64_t step = x.st[1] * 2;
#pragma unroll 2
    for (int r = warp; r < rows; r += 4 * kWarps) {
      uint4 v[4];
#pragma unroll
      for (int u = 0; u < 4; ++u) {
        const int row = r + u * kWarps;
        v[u] = row < rows ? __ldg(reinterpret_cast<const uint4*>(base + row * step)) : make_uint4(0, 0, 0, 0);
      }
      float a[8] = {0, 0, 0, 0, 0, 0, 0, 0};
#pragma unroll
      for (int u = 0; u < 4; ++u) add8<kFp16>(a, v[u]);
#pragma unroll
      for (int e = 0; e < 8; ++e) sum[e] += static_cast<double>(a[e]);
    }
  }
#pragma unroll
  for (int e = 0; e < 8; ++e) part[warp][lane * 9 + e] = sum[e];
  __syncthreads();
  const int col = threadIdx.x;  // of the two heads' 256
  if (pair * 2 + (col >> 7) < x.heads) {
    double total = 0;
#pragma unroll
    for (int w = 0; w < kWarps; ++w) total += part[w][(col >> 3) * 9 + (col & 7)];
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

// x = hi + lo: the upper 10 bits of the mantissa, and the rest, of which the
// product drops what is below its own 10 (both by truncation, without a
// conversion: those run at 16 a clock and SM).
__device__ __forceinline__ void split_tf32(float x, uint32_t& hi, uint32_t& lo) {
  hi = __float_as_uint(x) & 0xffffe000u;
  lo = __float_as_uint(x - __uint_as_float(hi));
}

__device__ __forceinline__ void mma_tf32(float (&c)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
  asm volatile(
      "mma.sync.aligned.m16n8k8.row.col.f32.tf32.tf32.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
      : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
      : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}

// The keep-th largest of n keys (of those above 0, more than keep), by
// bisection of their range: `floor` and how many that equal floor + 1 belong
// to it are returned so that chosen = above floor + 1, plus the first `ties`
// equal to it; ties 0: all above floor.  It ends as soon as exactly `keep` lie
// above the middle (10 to 20 counts for scores that differ).
template <typename Key>
__device__ __forceinline__ void kth_largest(const Key* key, int n, int keep, Key lo, Key hi, int lane, Key& floor,
                                            int& ties) {
  int above = 0;  // keys above hi
  ties = 0;
  while (lo < hi) {
    const Key mid = lo + ((hi - lo) >> 1) + 1;  // lo < mid <= hi
    int c = 0;
#pragma unroll 8
    for (int i = lane; i < n; i += 32) c += key[i] >= mid;
    c = __reduce_add_sync(0xffffffffu, c);
    if (c == keep) {
      floor = mid - 1;
      return;
    }
    if (c > keep) {
      lo = mid;
    } else {
      hi = mid - 1;
      above = c;
    }
  }
  floor = lo - 1;
  ties = keep - above;
}

// Writes a row's chosen indices in ascending order (one warp): keys above
// floor + 1, and the first `ties` equal to it (ties 0: keys above floor).
template <typename Key>
__device__ __forceinline__ void write_list(const Key* key, int n, Key floor, int ties, int keep, int* out, int* count,
                                           int lane) {
  const unsigned below = (1u << lane) - 1;
  const Key equal = floor + 1;
  const bool tied = ties > 0;
  int done = 0;
#pragma unroll 4
  for (int n0 = 0; n0 < n; n0 += 32) {
    const int i = n0 + lane;
    const Key k = i < n ? key[i] : Key(0);
    bool take = k > floor;
    if (tied) {
      const unsigned m = __ballot_sync(0xffffffffu, take && k == equal);
      if (take && k == equal) take = __popc(m & below) < ties;
      ties -= min(ties, __popc(m));
    }
    const unsigned m = __ballot_sync(0xffffffffu, take);
    if (take) out[done + __popc(m & below)] = i;
    done += __popc(m);
  }
  for (int i = done + lane; i < keep; i += 32) out[i] = -1;
  if (lane == 0) *count = done;
}

// One CTA scores up to eight rows (query blocks of the query heads that share a
// key head) against every key block, then a warp selects for each row.
//
// The scores are first taken on the tensor cores: each mean is split into two
// tf32 terms and the three larger products are summed in 32 bits, which is off
// by less than E = 2^-16 |q| max |k| (the dropped terms are 3 * 2^-20 |q||k|, 16
// sums of the main products, nine terms each, keep 24 bits of their largest:
// 2^-16.8; the sums of the small products are 2^-10 of that) plus what may
// underflow.  With T the keep-th largest of these, a block above
// T + 2E is chosen and one below T - 2E is not, in 64 bits too; only the blocks
// between (the T block alone, in all but every few rows) are scored in 64 bits.
// Measured at 75600 tokens, 5 heads, 1182 key blocks, 118 kept: all scores in
// 64-bit FMAs 120 us (bound by their operands' shared-memory reads).
//
// Tiles are 16 key blocks x 8 rows.  The order of the 128 products is free, so
// a thread loads 16 bytes of a mean and uses them in two products' k-steps: the
// key means go from L2 to registers once per CTA, without shared memory.
__global__ void __launch_bounds__(kThreads, 2) block_select_kernel(const SelectArgs a) {
  extern __shared__ __align__(16) unsigned char smem[];
  unsigned long long* exact = reinterpret_cast<unsigned long long*>(smem);  // [k_blocks], for rows with many ties
  uint32_t* keys = reinterpret_cast<uint32_t*>(exact + a.k_blocks);         // [rows_per_cta][k_blocks]
  __shared__ __align__(16) float means[8][kHeadDim];  // of the queries
  __shared__ uint32_t longest;      // bits of max |k|^2
  __shared__ uint32_t redo[8];      // rows whose undecided blocks are many: lo key, or 0
  __shared__ uint32_t redo_hi[8];

  launch_dependents();
  wait_for_previous();  // the means
  const int rows = a.group * a.q_blocks;  // of one key head
  const int chunks = (rows + a.rows_per_cta - 1) / a.rows_per_cta;
  const int chunk = blockIdx.x % chunks;
  const int kv = (blockIdx.x / chunks) % a.kv_heads;
  const int batch = blockIdx.x / chunks / a.kv_heads;
  const int heads = a.kv_heads * a.group;
  const int row0 = chunk * a.rows_per_cta;
  const int rows_here = min(a.rows_per_cta, rows - row0);
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int g = lane >> 2, tig = lane & 3;

  int k_blocks = a.k_blocks;
  if (a.k_len) {
    const int64_t len = max(a.k_len[batch], 0);
    k_blocks = static_cast<int>(min(int64_t(k_blocks), (len + a.key_block - 1) / a.key_block));
  }
  int q_blocks = a.q_blocks;
  if (a.q_len) {
    const int64_t len = max(a.q_len[batch], 0);
    q_blocks = static_cast<int>(min(int64_t(q_blocks), (len + a.query_block - 1) / a.query_block));
  }
  if (threadIdx.x == 0) longest = 0;
  if (threadIdx.x < 8) redo[threadIdx.x] = 0;
  if (warp < rows_here) {
    const int row = row0 + warp;
    const int h = kv * a.group + row / a.q_blocks, qb = row % a.q_blocks;
    float4 m = make_float4(0, 0, 0, 0);
    if (a.q) {  // few query rows: their mean is taken here
      const int len = a.q_len ? min(max(a.q_len[batch], 0), a.len_q) : a.len_q;
      const int n = min(max(len - qb * a.query_block, 0), a.query_block);
      const uint16_t* x = static_cast<const uint16_t*>(a.q) + batch * a.q_st[0] +
                          static_cast<int64_t>(qb) * a.query_block * a.q_st[1] + h * a.q_st[2] + 4 * lane;
      double sum[4] = {0, 0, 0, 0};
#pragma unroll 4
      for (int i = 0; i < n; ++i) {
        const uint2 v = __ldg(reinterpret_cast<const uint2*>(x + i * a.q_st[1]));
        const uint32_t w[2] = {v.x, v.y};
#pragma unroll
        for (int e = 0; e < 2; ++e) {
          const float2 f = a.fp16 ? __half22float2(*reinterpret_cast<const __half2*>(&w[e]))
                                  : make_float2(__uint_as_float(w[e] << 16), __uint_as_float(w[e] & 0xffff0000u));
          sum[2 * e] += static_cast<double>(f.x);
          sum[2 * e + 1] += static_cast<double>(f.y);
        }
      }
      if (n) m = make_float4(float(sum[0] / n), float(sum[1] / n), float(sum[2] / n), float(sum[3] / n));
    } else {
      m = __ldg(reinterpret_cast<const float4*>(a.q_means) +
                ((static_cast<int64_t>(batch) * a.q_blocks + qb) * heads + h) * (kHeadDim / 4) + lane);
    }
    reinterpret_cast<float4*>(means[warp])[lane] = m;
  }
  __syncthreads();

  auto q_mean = [&](int r) { return reinterpret_cast<const float4*>(means[r]); };  // of row r of this CTA
  const float4* km = reinterpret_cast<const float4*>(a.k_means) +
                     (static_cast<int64_t>(batch) * a.k_blocks * a.kv_heads + kv) * (kHeadDim / 4);
  const int64_t kstep = static_cast<int64_t>(a.kv_heads) * (kHeadDim / 4);

  float q_sq = 0;  // |q|^2 of row g, after the sum over the four lanes that share it
  {
    float4 q[8];
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      q[j] = g < rows_here ? q_mean(g)[4 * j + tig] : make_float4(0, 0, 0, 0);
      q_sq = fmaf(q[j].x, q[j].x, fmaf(q[j].y, q[j].y, fmaf(q[j].z, q[j].z, fmaf(q[j].w, q[j].w, q_sq))));
    }
    // What each of this thread's two result columns (rows 2 tig, 2 tig + 1) may see.
    const uint8_t* allowed[2] = {nullptr, nullptr};
    bool in_use[2];
#pragma unroll
    for (int c = 0; c < 2; ++c) {
      const int r = 2 * tig + c, row = row0 + r;
      in_use[c] = r < rows_here && row % a.q_blocks < q_blocks;
      if (a.allowed && in_use[c])
        allowed[c] = a.allowed + batch * a.allowed_st[0] + (kv * a.group + row / a.q_blocks) * a.allowed_st[1] +
                     (row % a.q_blocks) * a.allowed_st[2];
    }
    uint32_t most = 0;
    for (int t = warp * 16; t < a.k_blocks; t += kWarps * 16) {
      float c[4] = {0, 0, 0, 0}, small[4] = {0, 0, 0, 0};
      float sq[2] = {0, 0};
#pragma unroll
      for (int half = 0; half < 2; ++half) {
        float4 v[2][4];
#pragma unroll
        for (int i = 0; i < 2; ++i) {
          const int n = t + g + 8 * i;
#pragma unroll
          for (int j = 0; j < 4; ++j)
            v[i][j] = n < k_blocks ? __ldg(km + n * kstep + 4 * (4 * half + j) + tig) : make_float4(0, 0, 0, 0);
        }
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          const float f[2][4] = {{v[0][j].x, v[0][j].y, v[0][j].z, v[0][j].w},
                                 {v[1][j].x, v[1][j].y, v[1][j].z, v[1][j].w}};
          const float4 qj = q[4 * half + j];
          const float qf[4] = {qj.x, qj.y, qj.z, qj.w};
#pragma unroll
          for (int u = 0; u < 2; ++u) {
            uint32_t ah[4], al[4], bh[2], bl[2];
            split_tf32(f[0][2 * u], ah[0], al[0]);
            split_tf32(f[1][2 * u], ah[1], al[1]);
            split_tf32(f[0][2 * u + 1], ah[2], al[2]);
            split_tf32(f[1][2 * u + 1], ah[3], al[3]);
            split_tf32(qf[2 * u], bh[0], bl[0]);
            split_tf32(qf[2 * u + 1], bh[1], bl[1]);
            mma_tf32(c, ah, bh[0], bh[1]);
            mma_tf32(small, al, bh[0], bh[1]);
            mma_tf32(small, ah, bl[0], bl[1]);
#pragma unroll
            for (int i = 0; i < 2; ++i)
              sq[i] = fmaf(f[i][2 * u], f[i][2 * u], fmaf(f[i][2 * u + 1], f[i][2 * u + 1], sq[i]));
          }
        }
      }
#pragma unroll
      for (int i = 0; i < 4; ++i) c[i] += small[i];
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        sq[i] += __shfl_xor_sync(0xffffffffu, sq[i], 1);
        sq[i] += __shfl_xor_sync(0xffffffffu, sq[i], 2);
        most = max(most, __float_as_uint(fabsf(sq[i])));  // NaN is above inf
        const int n = t + g + 8 * i;
        if (n >= a.k_blocks) continue;
#pragma unroll
        for (int e = 0; e < 2; ++e) {
          if (2 * tig + e >= rows_here) continue;
          const bool may = in_use[e] && n < k_blocks && (!allowed[e] || allowed[e][n * a.allowed_st[3]] != 0);
          keys[(2 * tig + e) * a.k_blocks + n] = may ? order_key(c[2 * i + e]) : 0u;
        }
      }
    }
    most = __reduce_max_sync(0xffffffffu, most);
    if (lane == 0) atomicMax(&longest, most);
    q_sq += __shfl_xor_sync(0xffffffffu, q_sq, 1);
    q_sq += __shfl_xor_sync(0xffffffffu, q_sq, 2);
  }
  __syncthreads();

  auto list_of = [&](int r) {
    const int row = row0 + r;
    return (static_cast<int64_t>(batch) * heads + kv * a.group + row / a.q_blocks) * a.q_blocks + row % a.q_blocks;
  };
  if (warp < rows_here) {
    const int r = warp;
    uint32_t* key = keys + r * a.k_blocks;
    const int64_t list = list_of(r);
    uint32_t least = ~0u, most = 0;
    int n_may = 0;
#pragma unroll 8
    for (int n = lane; n < a.k_blocks; n += 32) {
      const uint32_t k = key[n];
      n_may += k != 0;
      least = min(least, k - 1);  // 0 becomes the largest
      most = max(most, k);
    }
    n_may = __reduce_add_sync(0xffffffffu, n_may);
    uint32_t floor = 0;
    bool settled = true;
    if (n_may > a.keep) {
      least = __reduce_min_sync(0xffffffffu, least) + 1;
      most = __reduce_max_sync(0xffffffffu, most);
      int ties;
      kth_largest(key, a.k_blocks, a.keep, least, most, lane, floor, ties);
      // T: the smallest key above floor.
      uint32_t kth = ~0u;
#pragma unroll 8
      for (int n = lane; n < a.k_blocks; n += 32) {
        const uint32_t k = key[n];
        if (k > floor) kth = min(kth, k);
      }
      kth = __reduce_min_sync(0xffffffffu, kth);
      const float T = of_key(kth);
      const float len_q = sqrtf(__shfl_sync(0xffffffffu, q_sq, 4 * r));
      const float len_k = sqrtf(__uint_as_float(longest));
      const float E2 = 3.0517578125e-05f * len_q * len_k + 7.70371978e-34f * (1.f + len_q + len_k);  // 2^-15, 2^-110
      uint32_t lo_key = 1, hi_key = ~0u - 1;  // undecided: every block, where E says nothing
      if (kth < ~0u - 1 && isfinite(T - E2) && isfinite(T + E2)) {
        lo_key = order_key(T - E2);
        hi_key = order_key(T + E2);
      }
      int sure = 0, open = 0;
#pragma unroll 8
      for (int n = lane; n < a.k_blocks; n += 32) {
        const uint32_t k = key[n];
        sure += k > hi_key;
        open += k >= lo_key && k <= hi_key;
      }
      sure = __reduce_add_sync(0xffffffffu, sure);
      open = __reduce_add_sync(0xffffffffu, open);
      const int wanted = a.keep - sure;
      if (open == wanted) {
        floor = lo_key - 1;
      } else if (open <= 32) {
        // Lane i takes the i-th undecided block, in the order of their indices.
        int mine = -1, seen = 0;
        for (int n0 = 0; n0 < a.k_blocks && seen < open; n0 += 32) {
          const uint32_t k = n0 + lane < a.k_blocks ? key[n0 + lane] : 0u;
          unsigned m = __ballot_sync(0xffffffffu, k >= lo_key && k <= hi_key);
          for (; m; m &= m - 1, ++seen)
            if (lane == seen) mine = n0 + __ffs(m) - 1;
        }
        const float4 qv = q_mean(r)[lane];
        unsigned long long score = 0;
        for (int e = 0; e < open; ++e) {
          const float4 kk = __ldg(km + __shfl_sync(0xffffffffu, mine, e) * kstep + lane);
          double d = fma(double(qv.x), double(kk.x), double(qv.y) * double(kk.y)) +
                     fma(double(qv.z), double(kk.z), double(qv.w) * double(kk.w));
#pragma unroll
          for (int o = 16; o; o >>= 1) d += __shfl_xor_sync(0xffffffffu, d, o);
          if (lane == e) score = order_key(d);
        }
        int better = 0;
        for (int e = 0; e < open; ++e) {
          const unsigned long long other = __shfl_sync(0xffffffffu, score, e);
          better += other > score || (other == score && e < lane);
        }
        __syncwarp();
        if (lane < open) key[mine] = better < wanted ? ~0u : 0u;
        __syncwarp();
        floor = hi_key;
      } else {
        settled = false;
        if (lane == 0) {
          redo[r] = lo_key;
          redo_hi[r] = hi_key;
        }
      }
    }
    if (settled) write_list(key, a.k_blocks, floor, 0, a.keep, a.blocks + list * a.keep, a.counts + list, lane);
  }
  __syncthreads();
  // Rows with more than 32 undecided blocks (equal or overflowing scores): the
  // CTA scores them in 64 bits, one warp selects.
  for (int r = 0; r < rows_here; ++r) {
    const uint32_t lo_key = redo[r], hi_key = redo_hi[r];
    if (!lo_key) continue;
    const float4* q = q_mean(r);
    for (int n = threadIdx.x; n < a.k_blocks; n += kThreads) {
      const uint32_t k = keys[r * a.k_blocks + n];
      unsigned long long e = k > hi_key ? ~0ull : 0ull;
      if (k >= lo_key && k <= hi_key) {
        double d = 0;
        for (int u = 0; u < kHeadDim / 4; ++u) {
          const float4 x = q[u], y = __ldg(km + n * kstep + u);
          d = fma(double(x.x), double(y.x), d);
          d = fma(double(x.y), double(y.y), d);
          d = fma(double(x.z), double(y.z), d);
          d = fma(double(x.w), double(y.w), d);
        }
        e = order_key(d);
      }
      exact[n] = e;
    }
    __syncthreads();
    if (warp == 0) {
      unsigned long long floor;
      int ties;
      kth_largest(exact, a.k_blocks, a.keep, 1ull, ~0ull, lane, floor, ties);
      const int64_t list = list_of(r);
      write_list(exact, a.k_blocks, floor, ties, a.keep, a.blocks + list * a.keep, a.counts + list, lane);
    }
    __syncthreads();
  }
}

inline size_t select_smem(int rows, int k_blocks) { return size_t(k_blocks) * (8 + 4 * size_t(rows)); }

}  // namespace sparse

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
  static bool done[64] = {false};
  int dev = 0;
  if (cudaGetDevice(&dev) != cudaSuccess || dev < 0 || dev >= 64) dev = 0;
  if (!done[dev]) {
    const cudaError_t err = cudaFuncSetAttribute(block_select_kernel, cudaFuncAttributeMaxDynamicSharedMemorySize,
                                                 static_cast<int>(kSelectSmemLimit));
    if (err != cudaSuccess) return set_cuda_error("block_select: cudaFuncSetAttribute", err);
    done[dev] = true;
  }
  // Eight rows share a CTA's reads of the key means where their keys fit shared memory.
  a.rows_per_cta = select_smem(8, a.k_blocks) <= kSelectSmemLimit ? 8 : 1;
  const int64_t chunks = (int64_t(a.group) * a.q_blocks + a.rows_per_cta - 1) / a.rows_per_cta;
  const int64_t ctas = chunks * a.kv_heads * a.batch;
  if (ctas > 0x7fffffff) return set_error(PS_B200_ERR_UNSUPPORTED, "block_select: more than 2^31 lists");
  const cudaError_t err = launch_after(block_select_kernel, dim3(static_cast<unsigned>(ctas)), dim3(kThreads),
                                       select_smem(a.rows_per_cta, a.k_blocks), stream, a.after_means, a);
  if (err != cudaSuccess) return set_cuda_error("block_select launch", err);
  count_launch();
  return 0;
}

}  // namespace psb
