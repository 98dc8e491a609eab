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

// 64-bit keys in the order of the scores: 0 for a block that may not be
// chosen, above every number for NaN (a block with NaN in it is attended, so
// that NaN is not hidden by the selection).
__device__ __forceinline__ unsigned long long order_key(double s) {
  if (s != s) return ~0ull;
  const unsigned long long u = static_cast<unsigned long long>(__double_as_longlong(s + 0.0));  // -0 is 0
  return (u >> 63) ? ~u : (u | (1ull << 63));
}

// Sums and prefixes over the threads that share a row: a warp, or the CTA.
template <int kGroup>
struct Group {
  int* scratch;  // [2][kWarps], for the CTA
  int phase = 0;
  __device__ __forceinline__ int sum(int v) {
    v = __reduce_add_sync(0xffffffffu, v);
    if constexpr (kGroup == 32) return v;
    int* s = scratch + kWarps * phase;  // the other half may still be read
    phase ^= 1;
    if ((threadIdx.x & 31) == 0) s[threadIdx.x >> 5] = v;
    __syncthreads();
    int total = 0;
#pragma unroll
    for (int w = 0; w < kWarps; ++w) total += s[w];
    return total;
  }
  // Threads of the group ahead of this one with `p` set; `total`: all of them.
  __device__ __forceinline__ int rank(bool p, int& total) {
    const unsigned m = __ballot_sync(0xffffffffu, p);
    int before = __popc(m & ((1u << (threadIdx.x & 31)) - 1));
    total = __popc(m);
    if constexpr (kGroup == 32) return before;
    int* s = scratch + kWarps * phase;
    phase ^= 1;
    if ((threadIdx.x & 31) == 0) s[threadIdx.x >> 5] = total;
    __syncthreads();
    total = 0;
#pragma unroll
    for (int w = 0; w < kWarps; ++w) {
      if (w < static_cast<int>(threadIdx.x >> 5)) before += s[w];
      total += s[w];
    }
    return before;
  }
};

// One CTA scores kRows rows (query blocks of the query heads that share a key
// head) against every key block, then selects: a warp per row, or with one row
// the whole CTA.
//
// The k-th largest key is found by bisection of the 64-bit key range between
// the row's least and greatest key; it ends as soon as exactly `keep` keys lie
// above the middle (about log2 of a score's spacing: 10 to 20 counts of the
// row in shared memory).
template <int kRows>
__global__ void __launch_bounds__(kThreads) block_select_kernel(const SelectArgs a) {
  constexpr int kGroup = kRows == 1 ? kThreads : 32;
  extern __shared__ __align__(16) unsigned char smem[];
  double* qs = reinterpret_cast<double*>(smem);                                             // [128][kRows]
  unsigned long long* keys = reinterpret_cast<unsigned long long*>(qs + kHeadDim * kRows);  // [kRows][k_blocks]
  __shared__ int scratch[2 * kWarps];

  const int rows = a.group * a.q_blocks;  // of one key head
  const int chunks = (rows + kRows - 1) / kRows;
  const int chunk = blockIdx.x % chunks;
  const int kv = (blockIdx.x / chunks) % a.kv_heads;
  const int batch = blockIdx.x / chunks / a.kv_heads;
  const int heads = a.kv_heads * a.group;
  const int row0 = chunk * kRows;
  const int tid = threadIdx.x;

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

  for (int i = tid; i < kHeadDim * kRows; i += kThreads) {
    const int r = i / kHeadDim, d = i % kHeadDim;
    const int row = row0 + r;
    double v = 0;
    if (row < rows) {
      const int h = kv * a.group + row / a.q_blocks, qb = row % a.q_blocks;
      v = a.q_means[((static_cast<int64_t>(batch) * a.q_blocks + qb) * heads + h) * kHeadDim + d];
    }
    qs[d * kRows + r] = v;
  }
  __syncthreads();

  const float4* km = reinterpret_cast<const float4*>(a.k_means) +
                     (static_cast<int64_t>(batch) * a.k_blocks * a.kv_heads + kv) * (kHeadDim / 4);
  const int64_t kstep = static_cast<int64_t>(a.kv_heads) * (kHeadDim / 4);
  auto put = [&](int r, int n, double s) {
    const int row = row0 + r;
    if (row >= rows) return;
    const int qb = row % a.q_blocks;
    bool may = n < k_blocks && qb < q_blocks;
    if (may && a.allowed)
      may = a.allowed[batch * a.allowed_st[0] + (kv * a.group + row / a.q_blocks) * a.allowed_st[1] +
                      qb * a.allowed_st[2] + n * a.allowed_st[3]] != 0;
    keys[static_cast<int64_t>(r) * a.k_blocks + n] = may ? order_key(s) : 0ull;
  };
  if constexpr (kRows == 1) {
    // Four lanes share a key block, 16 bytes of its mean each in turn.
    const int sub = tid & 3;
    for (int n0 = 0; n0 < a.k_blocks; n0 += kThreads / 4) {
      const int n = n0 + (tid >> 2);
      double s0 = 0, s1 = 0;
      if (n < k_blocks) {
        const float4* p = km + n * kstep;
#pragma unroll
        for (int u = 0; u < 8; ++u) {
          const float4 v = __ldg(p + 4 * u + sub);
          const double* q = qs + (4 * u + sub) * 4;
          s0 = fma(static_cast<double>(v.x), q[0], s0);
          s1 = fma(static_cast<double>(v.y), q[1], s1);
          s0 = fma(static_cast<double>(v.z), q[2], s0);
          s1 = fma(static_cast<double>(v.w), q[3], s1);
        }
      }
      double s = s0 + s1;
      s += __shfl_xor_sync(0xffffffffu, s, 1);
      s += __shfl_xor_sync(0xffffffffu, s, 2);
      if (sub == 0 && n < a.k_blocks) put(0, n, s);
    }
  } else {
    // A thread per key block, kRows scores each: the query means come from
    // shared memory as broadcasts, a key mean's line stays in L1 for its 512 B.
    for (int n = tid; n < a.k_blocks; n += kThreads) {
      double s[kRows];
#pragma unroll
      for (int r = 0; r < kRows; ++r) s[r] = 0;
      if (n < k_blocks) {
        const float4* p = km + n * kstep;
#pragma unroll 4
        for (int u = 0; u < kHeadDim / 4; ++u) {
          const float4 v = __ldg(p + u);
          const double f[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            const double2* q = reinterpret_cast<const double2*>(qs + (4 * u + e) * kRows);
#pragma unroll
            for (int r = 0; r < kRows / 2; ++r) {
              const double2 w = q[r];
              s[2 * r] = fma(f[e], w.x, s[2 * r]);
              s[2 * r + 1] = fma(f[e], w.y, s[2 * r + 1]);
            }
          }
        }
      }
#pragma unroll
      for (int r = 0; r < kRows; ++r) put(r, n, s[r]);
    }
  }
  __syncthreads();

  const int r = kRows == 1 ? 0 : tid >> 5;
  const int me = kRows == 1 ? tid : tid & 31;
  const int row = row0 + r;
  if (row >= rows) return;  // a whole warp; with one row it never holds
  const unsigned long long* key = keys + static_cast<int64_t>(r) * a.k_blocks;
  Group<kGroup> group{scratch};
  unsigned long long least = ~0ull, most = 0;
  int n_may = 0;
  for (int n = me; n < a.k_blocks; n += kGroup) {
    const unsigned long long k = key[n];
    if (k) {
      ++n_may;
      least = min(least, k);
      most = max(most, k);
    }
  }
  n_may = group.sum(n_may);
  // Chosen: every key above `floor`, and the first `ties` that equal it.
  unsigned long long floor = 0;
  int ties = 0;
  if (n_may > a.keep) {
    // In the CTA form each warp's bounds would differ: the whole key range
    // costs a few counts more.
    unsigned long long lo = 1, hi = ~0ull;
    if constexpr (kGroup == 32) {
#pragma unroll
      for (int o = 16; o; o >>= 1) {
        least = min(least, __shfl_xor_sync(0xffffffffu, least, o));
        most = max(most, __shfl_xor_sync(0xffffffffu, most, o));
      }
      lo = least;
      hi = most;
    }
    int above = 0;  // keys above hi
    bool found = false;
    while (lo < hi) {
      const unsigned long long mid = lo + ((hi - lo) >> 1) + 1;  // lo < mid <= hi
      int c = 0;
      for (int n = me; n < a.k_blocks; n += kGroup) c += key[n] >= mid;
      c = group.sum(c);
      if (c == a.keep) {
        floor = mid - 1;
        found = true;
        break;
      }
      if (c > a.keep) {
        lo = mid;
      } else {
        hi = mid - 1;
        above = c;
      }
    }
    if (!found) {
      floor = lo;
      ties = a.keep - above;
    }
  }
  const int h = kv * a.group + row / a.q_blocks, qb = row % a.q_blocks;
  const int64_t list = (static_cast<int64_t>(batch) * heads + h) * a.q_blocks + qb;
  int* out = a.blocks + list * a.keep;
  int done = 0;
  for (int n0 = 0; n0 < a.k_blocks; n0 += kGroup) {
    const int n = n0 + me;
    const unsigned long long k = n < a.k_blocks ? key[n] : 0ull;
    bool take = k > floor;
    int all;
    if (ties > 0) {  // the same for the whole group
      const int before = group.rank(k == floor && k != 0, all);
      take |= k == floor && k != 0 && before < ties;
      ties -= min(ties, all);
    }
    const int at = done + group.rank(take, all);
    if (take) out[at] = n;
    done += all;
  }
  for (int i = done + me; i < a.keep; i += kGroup) out[i] = -1;
  if (me == 0) a.counts[list] = done;
}

// Shared memory of one CTA with `rows` rows of k_blocks keys.
inline size_t select_smem(int rows, int k_blocks) {
  return size_t(rows) * (kHeadDim + size_t(k_blocks)) * sizeof(double);
}

template <int kRows>
int launch_select(const SelectArgs& a, cudaStream_t stream) {
  static bool done[64] = {false};
  int dev = 0;
  if (cudaGetDevice(&dev) != cudaSuccess || dev < 0 || dev >= 64) dev = 0;
  if (!done[dev]) {
    const cudaError_t err = cudaFuncSetAttribute(block_select_kernel<kRows>, cudaFuncAttributeMaxDynamicSharedMemorySize,
                                                 static_cast<int>(kSelectSmemLimit));
    if (err != cudaSuccess) return set_cuda_error("block_select: cudaFuncSetAttribute", err);
    done[dev] = true;
  }
  const int64_t chunks = (int64_t(a.group) * a.q_blocks + kRows - 1) / kRows;
  const int64_t ctas = chunks * a.kv_heads * a.batch;
  if (ctas > 0x7fffffff) return set_error(PS_B200_ERR_UNSUPPORTED, "block_select: more than 2^31 lists");
  block_select_kernel<kRows>
      <<<static_cast<unsigned>(ctas), kThreads, select_smem(kRows, a.k_blocks), stream>>>(a);
  const cudaError_t err = cudaGetLastError();
  if (err != cudaSuccess) return set_cuda_error("block_select launch", err);
  count_launch();
  return 0;
}

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

int launch_block_select(const SelectArgs& a, cudaStream_t stream) {
  using namespace sparse;
  // Eight rows a CTA read each key mean once for eight scores; with fewer
  // rows than half of that, or rows too long for shared memory, one row a CTA.
  const bool eight = int64_t(a.group) * a.q_blocks >= 4 && select_smem(8, a.k_blocks) <= kSelectSmemLimit;
  return eight ? launch_select<8>(a, stream) : launch_select<1>(a, stream);
}

}  // namespace psb
