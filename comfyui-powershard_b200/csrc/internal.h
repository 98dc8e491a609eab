// Internal declarations shared by the kernel translation units and the C ABI.
#pragma once

#include <cuda.h>
#include <cuda_runtime.h>
#include <stdint.h>

namespace psb {

constexpr int kMaxSegs = 64;  // segments (source ranks) per attention call

// Arguments of the attention kernel that are not tensor maps.
struct AttnArgs {
  void* seg_out[kMaxSegs];  // output element (batch 0, row 0, head 0, d 0) of each query segment:
                            // slices of one tensor, or other GPUs' buffers (peer exchange)
  int64_t o_stride[4];   // batch, (unused), row, head strides in elements (d stride 1)
  int seg_rows_q;        // rows allocated per query segment
  int nsegs_q;           // query segments
  int q_tiles_per_seg;   // ceil(seg_rows_q / 128)
  int num_q_tiles;       // prefix tiles + nsegs_q * q_tiles_per_seg
  int seg_rows_k;
  int nsegs_k;
  int num_kv_tiles;      // prefix tiles + sum over key segments of ceil(valid_k / 128)
  int valid_q[kMaxSegs]; // valid rows of each query segment (a prefix of its rows)
  int valid_k[kMaxSegs];
  int group;             // query heads per key/value head (GQA)
  float scale_log2;      // softmax_scale * log2(e)
  int out_fp32;          // 1: output fp32, 0: output in the input 16-bit type
  int* status;           // device status word (0 = ok), may be null
  // Optional prefix range (Flux text tokens): query and key rows [0, pre_len)
  // come from the prefix maps, ahead of the segmented rows; num_q_tiles and
  // num_kv_tiles count both ranges.  pre_len == 0: no prefix.
  int pre_len;
  int pre_tiles;         // ceil(pre_len / 128)
  void* pre_out;         // prefix output row 0, head 0
  int64_t pre_o_stride[4];  // batch, (unused), row, head strides in elements
  // Work units: (query tile pair, head, batch), pair fastest; the grid is 1-D.
  // Units [0, full_units) run whole; each later unit (the last, partial wave)
  // runs as `split` CTAs over consecutive parts of the key range, writing
  // partials that attn_combine_kernel merges.
  int npairs;            // ceil(num_q_tiles / 2)
  int grid_heads;
  int full_units;
  int split;             // 1: no split
  float* ws_o;           // [slot][2][128][128] fp32: O / l of one part, slot = (unit - full_units) * split + part
  float* ws_lse;         // [slot][2][128] fp32: m + log2(l) of one part (log2 units of the scaled scores)
  float2* ws_ml;         // in its place m and l of one part (sparse_attn.cu): their sum would round l away where m is
                         // large, and with it how much parts of like maxima weigh; or null
  // Block lists (sparse_attn.cu only).  Query block i of head h of batch row b attends the key
  // blocks blocks[((b * grid_heads + h) * list_rows + i) * list_len + ...]; one segment of queries and keys.
  const int* blocks;
  const int* counts;     // [batch][heads][list_rows] entries in use of each list, or null: list_len
  int list_rows;         // query blocks of one head
  int list_len;          // entries of one list
  int pairs_per_list;    // query block rows / 256
  int key_block;         // rows of a key block
  int key_blocks;        // ceil(seg_rows_k / key_block); a listed block outside [0, key_blocks) holds no key
  int piece;             // rows of one K/V load: 128, or 64 when key_block is not a multiple of 128
  const int* q_len;      // [batch] query rows in use, or null: all; output rows behind them are zero
  const int* k_len;      // [batch] key rows in use, or null: all; what lies behind them is not used
  int* tickets;          // few queries: [split units] zeros, the last part of a unit merges it; or null: a kernel of its own does
};

constexpr int kMaxSplit = 8;
constexpr int kMaxSparseSplit = 32;
constexpr int kMergeRows = 16;  // query rows up to which sparse attention runs in its form for few queries
// ... and up to which the parts of a split unit are merged in it, by the warp
// that ends last.  That saves a launch, but the warp takes two rows after the
// other: 12 lists of 8 tiles, 1 row 15.0 us and (merged by a kernel) as much, with
// the host in the steady state 18.0 and 19.9; 4 rows 16.0 and 16.1; 8 rows 18.7 and
// 16.7; 16 rows 24.4 and 16.9.
constexpr int kTicketRows = 4;
// Workspace bytes for up to 160 SMs: one partial (O, lse) per CTA of a wave.
constexpr int64_t kAttnWorkspaceBytes = int64_t(160) * 2 * 128 * (128 + 1) * 4;

// Launches the attention grid (full_units + split units * split CTAs) and,
// when units are split, the combine kernel after it on the same stream.
int launch_attention(const CUtensorMap& tq, const CUtensorMap& tk, const CUtensorMap& tv,
                     const CUtensorMap& tqp, const CUtensorMap& tkp, const CUtensorMap& tvp,
                     const AttnArgs& args, int64_t total_units, bool fp16, cudaStream_t stream);
// Merges the parts of `split_units` units (overlap: right after the kernel that writes them).
int launch_combine(const AttnArgs& args, int64_t split_units, bool fp16, bool overlap, cudaStream_t stream);
// The same over the block lists of `args` (sparse_attn.cu).
int launch_sparse_attention(const CUtensorMap& tq, const CUtensorMap& tk, const CUtensorMap& tv, const AttnArgs& args,
                            int64_t total_units, bool fp16, bool after_select, cudaStream_t stream);

// Process-wide count of kernels this library launched (ps_b200_kernel_launches).
void count_launch();

struct PrepassArgs {
  const void* x[3];        // q, k, v projection outputs, [batch][n_local][heads*head_dim]
  int64_t x_batch_stride[3]; // elements between consecutive batch rows
  int64_t x_row_stride[3]; // elements between consecutive tokens
  int64_t x_head_stride[3];// elements between consecutive heads of a token (head_dim: [n][H*D] rows)
  const void* w[2];        // RMSNorm weights of q and k, [heads*head_dim]
  int w_fp32;              // 1: weights are fp32, 0: same 16-bit type as x
  const float* freqs;      // [batch][n_local][head_dim/2][2][2] fp32
  int64_t freqs_batch_stride; // floats between consecutive batch rows (0: one table for the batch)
  int64_t freqs_row_stride;// floats between consecutive tokens
  void* dst[kMaxSegs];     // block [3][batch][seg_rows][heads_per_rank][head_dim] for each destination
                           // rank: slices of the local send buffer, or peers' receive buffers
  int batch, world, n_local, seg_rows, heads, heads_per_rank, head_dim;
  float eps;
  int norm_rope;           // 0: plain pack, 1: full-width RMSNorm + RoPE, 2: per-head RMSNorm + RoPE
  int rope_style;          // 0: interleaved pairs (2j, 2j+1) over the head; 1: split half (j, j+rope_pairs)
  int rope_pairs;          // rotated pairs per head (head_dim/2 for style 0; a multiple of 8 for style 1)
  // Token-mode fan-out (kv_fanout > 0, world 1, heads_per_rank == heads): q rows go to q_out
  // [batch][seg_rows][heads][head_dim]; k and v rows go to each of dst[0..kv_fanout-1], blocks
  // [2][batch][seg_rows][heads][head_dim] (the all-gather of K/V as stores).
  void* q_out;
  int kv_fanout;
};

int launch_prepass(const PrepassArgs& a, bool fp16, cudaStream_t stream);

struct UnpackArgs {
  const void* recv;        // head block src, batch b, row i at recv + src*src_stride + b*batch_stride
                           // + i*row_stride (elements)
  int64_t src_stride, batch_stride, row_stride;
  void* out;               // [batch][n_local][heads][head_dim] (strides below)
  int64_t out_batch_stride;// elements between consecutive batch rows of out
  int64_t out_row_stride;  // elements between consecutive tokens of out
  int batch, world, n_local, seg_rows, heads, heads_per_rank, head_dim;
  int out_fp32;            // 1: write fp32, 0: same 16-bit type as recv
};

int launch_unpack(const UnpackArgs& a, bool fp16, cudaStream_t stream);

// Arguments of the projection GEMMs (proj.cu) that are not tensor maps.
struct ProjArgs {
  int n;                   // rows of A: batch * n_local (epi 1) or this rank's tokens (epi 0)
  int batch;               // epi 1: batch rows; GEMM row m is token m % n_local of batch row m / n_local
  int n_local;             // epi 1: tokens per batch row
  int64_t freqs_batch_stride;  // epi 1: floats between the rotation tables of batch rows (0: shared)
  int kdim;                // K: input features (a multiple of 64)
  int width;               // output features of one projection (a multiple of 256)
  int ntile_n;             // width / 256: column tiles of one projection
  int row_blocks;          // ceil(n / 256): row blocks of the 256-row pair tiles
  int a_mode;              // 0: A is [n][kdim] rows; 1: A is [src][n][a_block_k] blocks (k = src*a_block_k + c)
  int a_block_k;           // columns per source block (a multiple of 64) for a_mode 1
  int epi;                 // 0: y = A W^T + b stored row-major; 1: q/k/v with RMSNorm, RoPE and the Ulysses pack
  const void* bias[3];     // per projection, [width], may be null
  int bias_fp32;           // 1: fp32 biases, 0: the 16-bit activation type
  const void* normw[2];    // RMSNorm weights of q and k, [width]
  int normw_fp32;
  const float* freqs;      // [n][head_dim/2][2][2] rotation table
  int64_t freqs_row_stride;
  float eps;
  void* dst[kMaxSegs];     // epi 1: destination d's block [3][batch][seg_rows][heads_per_rank][head_dim]
  int world, seg_rows, heads, heads_per_rank, head_dim;
  void* out;               // epi 0: [n][width] (row stride out_row_stride elements)
  int64_t out_row_stride;
  int out_fp32;
  // Scheduling (persistent CTA pairs, one task = one 256 x 256 pair tile per round):
  int total_groups;        // epi 1: 2 * row_blocks q/k groups of pair tiles
  int total_tiles;         // epi 0: row_blocks * ntile_n; epi 1: 3 * row_blocks * ntile_n
  int rounds;
  // RMSNorm statistics per 128-row block (two per pair row block):
  float* ss_part;          // epi 1: [4 * row_blocks][ntile_n][128] partial sums of squares
  unsigned* counters;      // epi 1: [4 * row_blocks] tiles that posted their partials (zeroed)
  int* status;             // device status word, may be null
};

// Launches the projection GEMM: `clusters` pairs of CTAs (cooperative
// cluster launch: every CTA resident, one per SM).
int launch_proj(const CUtensorMap& ta, const CUtensorMap& tw0, const CUtensorMap& tw1, const CUtensorMap& tw2,
                const ProjArgs& args, bool fp16, int clusters, cudaStream_t stream);
// CTA pairs the device keeps resident at once (0 on error, recorded).
int proj_clusters(bool fp16);

struct BroadcastArgs {
  const void* src;         // 16-byte vectors to copy
  void* dst[kMaxSegs];     // destinations (this GPU's memory or a peer's)
  int ndst;
  int64_t vectors;
};

int launch_broadcast(const BroadcastArgs& a, cudaStream_t stream);

// Block means (sparse.cu) of one tensor [batch][len][heads][128].
struct MeansTensor {
  const void* x;
  int64_t st[3];           // batch, row, head strides in elements
  int len, heads, block;
  int blocks;              // ceil(len / block)
  int head_pairs;          // ceil(heads / 2)
  int warps;               // that share a block (1, 2, 4 or 8), about 32 rows each
  int64_t items;           // batch * blocks * head_pairs
  int64_t ctas;            // of eight warps
  const int* lens;         // [batch] rows in use, or null: len
  float* out;              // [batch][blocks][heads][128]
};
struct MeansArgs {
  MeansTensor t[2];        // the second one is empty (ctas 0) or of the same type and batch
};
int launch_block_means(const MeansArgs& a, bool fp16, cudaStream_t stream);

constexpr int kSelectMaxBlocks = 16384;  // 8 bytes of shared memory each
// Pairs of batch row and key head whose scores are held at a time, in at most 64 MB where one fits in that.
inline int select_units(int64_t batch, int64_t kv_heads, int64_t group, int64_t q_blocks, int64_t k_blocks) {
  const int64_t one = group * q_blocks * k_blocks * 4;
  int64_t n = (int64_t(64) << 20) / (one > 0 ? one : 1);
  n = n < 1 ? 1 : (n > 65535 ? 65535 : n);
  return static_cast<int>(n < batch * kv_heads ? n : batch * kv_heads);
}
// Workspace of launch_block_select: the scores of those pairs, and the largest of the key means' squared lengths.
inline int64_t select_score_floats(int64_t batch, int64_t kv_heads, int64_t group, int64_t q_blocks, int64_t k_blocks) {
  return select_units(batch, kv_heads, group, q_blocks, k_blocks) * (group * q_blocks + 1) * k_blocks;
}
struct SelectArgs {
  float* q_means;          // [batch][q_blocks][kv_heads * group][128]
  const float* k_means;    // [batch][k_blocks][kv_heads][128]
  int batch, kv_heads, group, q_blocks, k_blocks, keep;
  int query_block, key_block;
  const int* q_len;        // [batch] rows in use, or null
  const int* k_len;
  const uint8_t* allowed;  // truth value of (batch, head, query block, key block) under these strides, or null
  int64_t allowed_st[4];
  int* blocks;             // [batch][heads][q_blocks][keep]
  int* counts;             // [batch][heads][q_blocks]
  float* scores;           // workspace: [units at a time][group * q_blocks][k_blocks]
  uint32_t* k_sq;          // ... and behind it, bits of the largest |k|^2 of every 128 key blocks [units][chunks]
  int first_unit;          // set by the launch
  // Queries [batch][len_q][kv_heads * group][128] (16-bit) whose means the kernel takes itself and writes
  // to q_means, or null.
  const void* q;
  int64_t q_st[3];         // batch, row, head strides in elements
  int len_q;
  int fp16;
  bool after_means;        // launched right after the kernel that writes the means: starts while that one ends (after
                           // the attention of an earlier call that costs 1.4 us of 27 instead)
  int* zeros;              // n_zeros words that the kernels behind the selection want zeroed
  int n_zeros;
};
int launch_block_select(SelectArgs a, cudaStream_t stream);
bool select_is_small(int64_t lists, int k_blocks);  // one kernel makes the lists (rank_kernel)

// 8-bit key/value cache (cache.cu).
struct CacheArgs {
  void* pages[2];          // K and V codes [pages][page_rows][heads][head_dim], 8 bits each
  float* scales[2];        // [pages][page_rows][heads]
  void* rows[2];           // 16-bit rows: read from by the write, written to by the read
  int64_t st[2][3];        // batch, row, head strides of the 16-bit rows in elements
  int batch, n;            // rows of each sequence in `rows`
  int heads, head_dim;
  int num_pages, page_rows;
  const int* table;        // [batch][table_len] page of each page_rows positions
  int64_t table_st;
  int table_len;
  const int* first;        // [batch] position of row 0, or null: 0
  const int* count;        // write: [batch] rows in use, or null: n; read: [batch] positions held
};
int launch_cache_write(const CacheArgs& a, bool fp16, bool int8, cudaStream_t stream);
int launch_cache_read(const CacheArgs& a, bool fp16, bool int8, cudaStream_t stream);

// Error bookkeeping (thread-local message, returned code).
int set_error(int code, const char* fmt, ...);
int set_cuda_error(const char* what, cudaError_t err);

}  // namespace psb
