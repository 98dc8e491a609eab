// Block-sparse attention forward: each block of queries over the key blocks
// that its list names (tiles, UMMAs and softmax as in attention.cu).
//
// A unit of work is two 128-row query tiles of one head and its list, or, of
// the units of the last wave, one part of the list.  A key tile is one 128-row
// load or two 64-row loads from anywhere in the sequence.  A query block is a
// multiple of 256 rows: both query tiles share the list, so each K/V tile is
// loaded once for 256 queries, as in the dense form (a list for each 128 rows
// would double the K/V loads: 64 KB per 128 x 128 tile pair is ~52 B/clk per
// SM, above the L2's share).
//
// Lists are short (a unit of the dense kernel walks every key), so what a CTA
// costs beside its tiles counts: with one CTA per unit, ~10 us of launch, TMEM
// allocation, first loads and epilogue against 2 us a tile.  CTAs here keep
// their barriers and TMEM and take unit after unit from the not yet started
// CTAs of their own grid (the hardware's work stealing, which also levels lists
// of different lengths); while the softmax warps write one unit's output, the
// next one's Q, K and V load and its first scores are computed.
//
// Rows past a sequence's key length are not used, whatever they hold: their
// scores are masked, and as 0 * NaN is NaN in the PV product, V rows of a
// partly used tile are overwritten with zeros in shared memory before it.
//
// Warp roles (320 threads) as in the dense kernel: 0-3 / 4-7 softmax and
// epilogue of query tile 0 / 1, 8 producer (the whole warp: it also zeroes V
// rows), 9 UMMA issuer.  Where a unit has one query tile (the last pair of an
// odd count), group 1 sits it out.
//
// The form for few queries (kFew: at most 16 rows, one tile of which one warp's
// rows hold them) is bound by the keys it reads and, per CTA, by the latency of
// load, scores, softmax and output product in turn.  So warps 0 and 4 take the
// key tiles by turns, each with its own S, P and O; the issue order S_n,
// PV_{n-1}, S_{n+1} keeps two tiles under way, and the shared memory of the
// second query tile and of the output staging are a third K and V stage (the
// 1.5 us and more that a load takes under way are then spread over three
// tiles).  At a unit's end warp 0 adds the two up, through the part of the
// query tile that holds no query.
// Measured, 48 tiles a list: 120 lists 2.0 us a tile with one group alone, 1.35
// in turns; 148 lists 1.6 us (6.0 TB/s: bound by HBM), 1.1 us where L2 holds the
// keys (9 TB/s).
#include "attn_tile.cuh"

namespace psb {
namespace attn {
namespace {

constexpr int kStageBytes = 4096;  // output staging of one softmax warp: 32 rows x 64 columns
constexpr int kRing = 4;           // FREE signals: K_{n+4} is never loaded before FREE(n) is waited for
constexpr int kMetaRing = 8;       // published rows: tile n+8 is published after FREE(n+5), so n has been read

enum SparseBar : int {
  kQ = 0,
  kKFull = 1,
  kVFull = kKFull + 3,
  kS = kVFull + 3,         // [2] S_t computed
  kFree = kS + 2,          // [kRing] FREE[n%4]: every S of tile n observed complete -> K_n free, and V_{n-1}
                           // (few queries: V_{n-2}), whose PV was issued before
  kP = kFree + kRing,      // [2] P_t written
  kPH = kP + 2,            // [2][kPParts-1]
  kO = kPH + 2 * (kPParts - 1),  // [2] O_t of a unit final; of units in which group t has a tile: such a unit's P_t
                                 // comes after the last one's O_t, so that no phase passes a waiting group by
  kDrain = kO + 2,
  kTail = kDrain + 1,      // V rows of a partly used tile loaded
  kMeta = kTail + 1,       // [kMetaRing] rows in use of a tile published
  kWork = kMeta + kMetaRing,  // [2] a unit published
  kTaken = kWork + 2,      // [2] ... and read by the issuer and the softmax warps
  kNext = kTaken + 2,      // the grid's answer
  kOther = kNext + 1,      // few queries: group 1's rows of a unit staged
  kOtherRead = kOther + 1, // ... and read
  kCount = kOtherRead + 1
};
constexpr int kStageOff = kSmemQ + kSmemK + kSmemV;
constexpr int kBarOff = kStageOff + 8 * kStageBytes;
// Few queries: one Q tile, of which the first 32 rows are loaded (the others
// give rows of S and O that nothing reads), and three K and V stages.
constexpr int kFewStages = 3;
constexpr int kFewQRows = 32;
constexpr int kMergePad = kHeadDim + 4;     // floats of a staged row of O
constexpr int kMergeOff = kFewQRows * 128;  // behind those rows of the tile's first 64 columns
static_assert(kMergeOff + kMergeRows * (kMergePad + 2) * 4 <= kHalfTile && kMergeRows <= kFewQRows, "staged rows");
static_assert(kTileBytes + 2 * kFewStages * kTileBytes == kBarOff, "both forms end at the barriers");
constexpr int kSmem = kBarOff + 512 + 1024;  // barriers and small words, 1 KiB align slack
static_assert(kSmem <= 227 * 1024, "shared memory of one CTA");

enum SparseErr : int { kErrWork = 108, kErrMeta = 109 };

struct Work {
  int unit;  // -1: none left
  int slot;  // of the split workspace, or -1: a whole unit
  int tiles;
  int rows;  // query rows in use of the sequence
};

struct Small {  // behind the barriers
  Work work[2];
  int meta[kMetaRing];  // rows in use of a tile's lower 64 | upper 64 << 8
  uint32_t tmem;
  int abort;
  __align__(16) int answer[4];
};
static_assert(kCount * 8 + sizeof(Small) <= 512, "barrier block overflow");

struct Coord {
  int pair, head, batch;
  __device__ __forceinline__ Coord(const AttnArgs& a, int unit) {
    pair = unit % a.npairs;
    const int rest = unit / a.npairs;
    head = rest % a.grid_heads;
    batch = rest / a.grid_heads;
  }
};

// The pieces of one unit's list, in order: a block is cut into pieces of
// args.piece rows, a 128-row tile holds 128 / piece consecutive ones.
struct BlockList {
  const int* list;
  int count;     // entries in use
  int len_k;     // key rows in use
  int per;       // pieces of one block
  int entry, sub;  // of the next piece

  struct Piece {
    int block, sub;
  };
  // The load of the block's number is under way until the piece is used.
  __device__ __forceinline__ Piece next() {
    const Piece p{entry < count ? __ldg(list + entry) : -1, sub};
    if (++sub == per) {
      sub = 0;
      ++entry;
    }
    return p;
  }
  // First row of a piece, and in `valid` its rows in use.  A piece without any
  // starts behind the tensor: its load fills with zeros.
  __device__ __forceinline__ int row(const AttnArgs& a, const Piece& p, int& valid) const {
    valid = 0;
    if (p.block < 0 || p.block >= a.key_blocks) return a.seg_rows_k;
    const int64_t r = static_cast<int64_t>(p.block) * a.key_block + p.sub * a.piece;
    if (r >= len_k) return a.seg_rows_k;
    valid = min(a.piece, len_k - static_cast<int>(r));
    return static_cast<int>(r);
  }
};

// The unit (or part of one) that grid index x stands for, and its list from
// the first tile on.
__device__ __forceinline__ Work find_work(const AttnArgs& a, int x, BlockList& b) {
  Work w;
  const bool partial = x >= a.full_units;
  w.slot = partial ? x - a.full_units : -1;
  w.unit = partial ? a.full_units + w.slot / a.split : x;
  const int parts = partial ? a.split : 1;
  const int part = partial ? w.slot % a.split : 0;
  const Coord c(a, w.unit);
  w.rows = a.q_len ? min(max(a.q_len[c.batch], 0), a.seg_rows_q) : a.seg_rows_q;
  b.len_k = a.k_len ? min(max(a.k_len[c.batch], 0), a.seg_rows_k) : a.seg_rows_k;
  const int64_t at = (static_cast<int64_t>(c.batch) * a.grid_heads + c.head) * a.list_rows + c.pair / a.pairs_per_list;
  b.list = a.blocks + at * a.list_len;
  b.count = a.counts ? min(max(a.counts[at], 0), a.list_len) : a.list_len;
  if (c.pair * 2 * kBlockM >= w.rows || b.len_k == 0) b.count = 0;
  b.per = a.key_block / a.piece;
  const int64_t tiles = (static_cast<int64_t>(b.count) * a.key_block + kBlockN - 1) / kBlockN;
  const int begin = static_cast<int>(part * tiles / parts);
  w.tiles = static_cast<int>((part + 1) * tiles / parts) - begin;
  const int first = begin * (kBlockN / a.piece);
  b.entry = first / b.per;
  b.sub = first - b.entry * b.per;
  return w;
}

template <bool kFp16, bool kFew>
__global__ void __launch_bounds__(kThreads, 1)
    sparse_attn_kernel(const __grid_constant__ CUtensorMap tm_q, const __grid_constant__ CUtensorMap tm_k,
                       const __grid_constant__ CUtensorMap tm_v, const AttnArgs args) {
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  uint8_t* sQ = smem;
  constexpr int kKSt = kFew ? kFewStages : kKStages, kVSt = kFew ? kFewStages : kVStages;
  uint8_t* sK = smem + (kFew ? kTileBytes : kSmemQ);
  uint8_t* sV = sK + kKSt * kTileBytes;
  uint64_t* bars = reinterpret_cast<uint64_t*>(smem + kBarOff);
  Small* small = reinterpret_cast<Small*>(bars + kCount + (kCount & 1));
  volatile int* abort_flag = &small->abort;
  const int warp = threadIdx.x >> 5;
  const int lane = threadIdx.x & 31;
  int* status = args.status;
  auto bar = [&](int i) { return smem_u32(&bars[i]); };

  launch_dependents();
  if (threadIdx.x == 0) {
    small->abort = 0;
    mbar_init(bar(kQ), 1);
    for (int i = 0; i < 2; ++i) {
      mbar_init(bar(kS + i), 1);
      mbar_init(bar(kP + i), kFew ? 32 : 128);
      for (int q = 0; q + 1 < kPParts; ++q) mbar_init(bar(kPH + i * (kPParts - 1) + q), kFew ? 32 : 128);
      mbar_init(bar(kWork + i), 1);
      mbar_init(bar(kTaken + i), kFew ? 3 : 9);
    }
    for (int i = 0; i < kKSt; ++i) mbar_init(bar(kKFull + i), 1);
    for (int i = 0; i < kVSt; ++i) mbar_init(bar(kVFull + i), 1);
    for (int i = 0; i < kRing; ++i) {
      mbar_init(bar(kFree + i), 1);
    }
    for (int i = 0; i < kMetaRing; ++i) mbar_init(bar(kMeta + i), 1);
    mbar_init(bar(kO), 1);
    mbar_init(bar(kO + 1), 1);
    mbar_init(bar(kDrain), 1);
    mbar_init(bar(kTail), 1);
    mbar_init(bar(kNext), 1);
    mbar_init(bar(kOther), 1);
    mbar_init(bar(kOtherRead), 1);
    fence_mbar_init();
  }
  if (warp == 9) {
    tmem_alloc(smem_u32(&small->tmem), 512);
    tmem_relinquish();
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = small->tmem;
  wait_for_previous();  // the lists

  // Tiles are numbered through all units of the CTA (n): K and V stages, FREE
  // and the published rows go by n, S_t and P_t by the tiles of group t.
  if (warp == 8) {
    // ------------------------------------------------------------ producer
    if (lane == 0) {
      tma_prefetch_desc(&tm_q);
      tma_prefetch_desc(&tm_k);
      tma_prefetch_desc(&tm_v);
    }
    const int pieces = kBlockN / args.piece;
    const int piece_bytes = args.piece * 128;  // of one 64-column half
    int x = blockIdx.x;
    int n = 0, loaded = 0;  // tiles; units with tiles
    int k_loads = 0, v_loads = 0;
    uint32_t tail_phase = 0;
    int open_request = -1;  // phase of an answer not yet read
    bool ok = true;
    for (int u = 0;; ++u) {
      const int b = u & 1;
      BlockList list;
      Work w{-1, -1, 0, 0};
      if (x >= 0) w = find_work(args, x, list);
      if (u >= 2) ok = warp_wait(bar(kTaken + b), ((u >> 1) - 1) & 1u, abort_flag, status, kErrWork);
      if (!ok) break;
      if (lane == 0) {
        small->work[b] = w;
        mbar_arrive(bar(kWork + b));
      }
      if (x < 0) break;
      if (lane == 0) {
        mbar_arrive_expect_tx(bar(kNext), 16);
        request_cta(smem_u32(small->answer), bar(kNext));
      }
      open_request = u & 1;
      if (w.tiles > 0) {
        const Coord c(args, w.unit);
        const int kv_head = c.head / args.group;
        // The last unit's scores are all computed once its last tile is free.
        auto free_wait = [&](int tile) {
          return warp_wait(bar(kFree + tile % kRing), (tile / kRing) & 1u, abort_flag, status, kErrEmpty);
        };
        if (n > 0) ok = free_wait(n - 1);
        if (!ok) break;
        if (lane == 0) {
          const int t0 = c.pair * 2;
          const bool two = t0 + 1 < args.num_q_tiles;
          mbar_arrive_expect_tx(bar(kQ), kFew ? 2 * kFewQRows * 128 : two ? 2 * kTileBytes : kTileBytes);
          for (int h = 0; h < 2; ++h) {
            tma_load_5d(smem_u32(sQ + h * kHalfTile), &tm_q, bar(kQ), h * 64, c.head, t0 * kBlockM, 0, c.batch);
            if (two)
              tma_load_5d(smem_u32(sQ + kTileBytes + h * kHalfTile), &tm_q, bar(kQ), h * 64, c.head,
                          (t0 + 1) * kBlockM, 0, c.batch);
          }
        }
        ++loaded;
        auto load = [&](uint8_t* stage, const CUtensorMap* map, int full, const int (&row)[2]) {
          if (lane == 0) {
            mbar_arrive_expect_tx(bar(full), kTileBytes);
#pragma unroll
            for (int p = 0; p < 2; ++p)
              if (p < pieces)
                for (int h = 0; h < 2; ++h)
                  tma_load_5d(smem_u32(stage + h * kHalfTile + p * piece_bytes), map, bar(full), h * 64, kv_head,
                              row[p], 0, c.batch);
          }
        };
        // The blocks of a tile are looked up a tile ahead of its K, and K goes a
        // tile ahead of V.
        BlockList::Piece ahead[2];
        auto look = [&] {
          ahead[0] = list.next();
          if (pieces == 2) ahead[1] = list.next();
        };
        int row[2], valid[2], next_row[2] = {0, 0}, next_valid[2] = {0, 0};
        auto load_k = [&](int tile) -> bool {  // and looks up the tile after it
#pragma unroll
          for (int p = 0; p < 2; ++p)
            if (p < pieces) next_row[p] = list.row(args, ahead[p], next_valid[p]);
          look();
          if (tile >= kKSt && !free_wait(tile - kKSt)) return false;
          if (lane == 0) {
            const int lo = pieces == 1 ? min(next_valid[0], 64) : next_valid[0];
            const int hi = pieces == 1 ? max(next_valid[0] - 64, 0) : next_valid[1];
            small->meta[tile % kMetaRing] = lo | (hi << 8);
            mbar_arrive(bar(kMeta + tile % kMetaRing));
          }
          load(sK + tile % kKSt * kTileBytes, &tm_k, kKFull + tile % kKSt, next_row);
          k_loads = tile + 1;
          return true;
        };
        look();
        ok = load_k(n);
        for (int i = 0; i < w.tiles && ok; ++i, ++n) {
          const int vst = n % kVSt;
          bool tail = false;  // rows of the tensor that are not in use reach the tile
#pragma unroll
          for (int p = 0; p < 2; ++p) {
            row[p] = next_row[p];
            valid[p] = next_valid[p];
            tail |= valid[p] > 0 && valid[p] < args.piece && list.len_k < args.seg_rows_k;
          }
          if (i + 1 < w.tiles) ok = load_k(n + 1);
          // V_{n-kVSt} is read: S_{n-1} is complete, and every PV issued before it.
          if (ok && n >= kVSt) ok = free_wait(n - 1);
          if (!ok) break;
          if (!tail) {
            load(sV + vst * kTileBytes, &tm_v, kVFull + vst, row);
          } else {
            uint8_t* stage = sV + vst * kTileBytes;
            load(stage, &tm_v, kTail, row);
            drain_wait(bar(kTail), tail_phase, status);
            tail_phase ^= 1u;
            __syncwarp();
#pragma unroll
            for (int p = 0; p < 2; ++p) {
              if (valid[p] == 0) continue;  // no such piece, or filled with zeros by its load
              const int chunks = (args.piece - valid[p]) * 8;  // 16 bytes each, of one half
              for (int h = 0; h < 2; ++h) {
                uint4* dst = reinterpret_cast<uint4*>(stage + h * kHalfTile + p * piece_bytes + valid[p] * 128);
                for (int j = lane; j < chunks; j += 32) dst[j] = make_uint4(0, 0, 0, 0);
              }
            }
            fence_proxy_async();
            __syncwarp();
            if (lane == 0) mbar_arrive(bar(kVFull + vst));
          }
          v_loads = n + 1;
        }
        if (!ok) break;
      }
      ok = warp_wait(bar(kNext), u & 1u, abort_flag, status, kErrWork);
      if (!ok) break;
      open_request = -1;
      x = granted_cta(smem_u32(small->answer));
      fence_proxy_async();  // read before the next answer is written
      __syncwarp();
    }
    // Every copy issued must land before the CTA may exit.
    if (open_request >= 0) drain_wait(bar(kNext), static_cast<uint32_t>(open_request), status);
    if (loaded) drain_wait(bar(kQ), (loaded - 1) & 1u, status);
    for (int i = max(0, k_loads - kKSt); i < k_loads; ++i) drain_wait(bar(kKFull + i % kKSt), (i / kKSt) & 1u, status);
    for (int i = max(0, v_loads - kVSt); i < v_loads; ++i) drain_wait(bar(kVFull + i % kVSt), (i / kVSt) & 1u, status);
  } else if (warp == 9) {
    // ------------------------------------------------------------ UMMA issuer (one lane; elected, not chosen by
    // its number, it issues a UMMA every 39 cycles instead of 45, and launches end 3-5 % sooner)
    if (elect_one()) {
      const TileMma mma = TileMma::make<kFp16>(tmem, sQ, sK, sV);
      // P_t arrives in parts; each part's UMMAs are issued as soon as it is written.
      auto pv = [&](int t, int st, uint32_t parity, bool accumulate) -> bool {
#pragma unroll
        for (int q = 0; q < kPParts; ++q) {
          const int b = q + 1 < kPParts ? kPH + t * (kPParts - 1) + q : kP + t;
          if (!mbar_wait(bar(b), parity, abort_flag, status, kErrP)) return false;
          tc_fence_after();
          mma.pv(t, st, q, accumulate);
        }
        return true;
      };
      int n = 0, n1 = 0, loaded = 0;  // tiles; tiles of group 1; units with tiles
      bool ok = true;
      for (int u = 0; ok; ++u) {
        const int b = u & 1;
        if (!mbar_wait(bar(kWork + b), (u >> 1) & 1u, abort_flag, status, kErrWork)) break;
        const Work w = small->work[b];
        mbar_arrive(bar(kTaken + b));
        if (w.unit < 0) break;
        if (w.tiles == 0) continue;
        const bool two = (w.unit % args.npairs) * 2 + 1 < args.num_q_tiles;
        ok = mbar_wait(bar(kQ), loaded & 1u, abort_flag, status, kErrQ);
        ++loaded;
        if constexpr (kFew) {
          // Tile j belongs to group j & 1: PV_{j-2}, S_j, PV_{j-1}, S_{j+1}, ...
          const int n0 = n;
          for (int j = n0; j < n0 + w.tiles + 2 && ok; ++j) {
            const int d = j - 2;
            if (d >= n0) {
              ok = mbar_wait(bar(kVFull + d % kVSt), (d / kVSt) & 1u, abort_flag, status, kErrFull);
              if (ok) ok = pv(d & 1, d % kVSt, (d >> 1) & 1u, d - n0 >= 2);
              if (!ok) break;
            }
            if (j < n0 + w.tiles) {
              ok = mbar_wait(bar(kKFull + j % kKSt), (j / kKSt) & 1u, abort_flag, status, kErrFull);
              if (!ok) break;
              tc_fence_after();
              mma.s(j & 1, 0, j % kKSt);
              umma_commit(bar(kS + (j & 1)));
            }
          }
          n = n0 + w.tiles;
          for (int t = 0; t < 2 && ok; ++t)
            if (w.tiles > 1 || (n0 & 1) == t) umma_commit(bar(kO + t));
        } else {
          // Issue order per key tile: S0_i, PV1_{i-1}, S1_i, PV0_i.  The first S
          // of a unit follow the last PV of the one before on the tensor pipe.
          for (int i = 0; i < w.tiles && ok; ++i, ++n) {
            const int st = n & 1;
            ok = mbar_wait(bar(kKFull + st), (n >> 1) & 1u, abort_flag, status, kErrFull);
            if (!ok) break;
            tc_fence_after();
            mma.s(0, st);
            umma_commit(bar(kS + 0));
            if (two) {
              if (i > 0) ok = pv(1, (n - 1) & 1, (n1 - 1) & 1u, i > 1);
              if (!ok) break;
              mma.s(1, st);
              umma_commit(bar(kS + 1));
              ++n1;
            }
            ok = mbar_wait(bar(kVFull + st), (n >> 1) & 1u, abort_flag, status, kErrFull);
            if (ok) ok = pv(0, st, n & 1u, i > 0);
          }
          if (ok && two) ok = pv(1, (n - 1) & 1, (n1 - 1) & 1u, w.tiles > 1);
          if (ok) umma_commit(bar(kO));
          if (ok && two) umma_commit(bar(kO + 1));
        }
      }
      // All issued UMMAs complete before TMEM is released.
      umma_commit(bar(kDrain));
      drain_wait(bar(kDrain), 0, status);
    }
  } else if (kFew) {
    // ------------------------------------------------------------ softmax, few queries
    const int t = warp >> 2;
    const uint32_t s_addr = tmem + 128 * t, o_addr = tmem + 256 + 128 * t;
    float* rows_o = reinterpret_cast<float*>(smem + kMergeOff);  // of group 1: [kMergeRows][kMergePad], then m, l
    float* rows_ml = rows_o + kMergeRows * kMergePad;
    int n = 0, loaded = 0, own = 0;  // tiles; units with tiles; units with tiles of this group
    for (int u = 0; (warp & 3) == 0; ++u) {
      const int b = u & 1;
      if (!warp_wait(bar(kWork + b), (u >> 1) & 1u, abort_flag, status, kErrWork)) break;
      const int tiles = small->work[b].tiles;
      if (small->work[b].unit < 0) break;
      float m = -1e30f, l = 0.f;
      bool ok = true, any = false;
      const int end = n + tiles;
      for (int j = n + ((n ^ t) & 1); j < end; j += 2) {
        const int slot = j % kMetaRing;
        ok = warp_wait(bar(kMeta + slot), (j / kMetaRing) & 1u, abort_flag, status, kErrMeta);
        if (!ok) break;
        const int used = small->meta[slot];
        ok = warp_wait(bar(kS + t), (j >> 1) & 1u, abort_flag, status, kErrS);
        if (!ok) break;
        if (lane == 0) mbar_arrive(bar(kFree + j % kRing));
        tc_fence_after();
        uint32_t sr[128];
        tmem_ld32_at<0>(s_addr + 0, sr);
        tmem_ld32_at<32>(s_addr + 32, sr);
        tmem_ld32_at<64>(s_addr + 64, sr);
        tmem_ld32_at<96>(s_addr + 96, sr);
        tmem_wait_ld();
        float s[128];
#pragma unroll
        for (int i = 0; i < 128; ++i) s[i] = __uint_as_float(sr[i]);
        if (used != (64 | (64 << 8))) {
          const int lo = used & 0xff, hi = used >> 8;
#pragma unroll
          for (int i = 0; i < 128; ++i)
            if ((i & 63) >= (i < 64 ? lo : hi)) s[i] = -INFINITY;
        }
        softmax_row<kFp16, true, false>(s, !any, args.scale_log2, s_addr, o_addr, bar(kPH + t * (kPParts - 1)), bar(kP + t), m, l);
        any = true;
      }
      n = end;
      if (tiles > 0) {
        if (ok && any) ok = warp_wait(bar(kO + t), own++ & 1u, abort_flag, status, kErrO);
        // Group 1's staged rows: free to write, or written.
        if (ok && t == 0) ok = warp_wait(bar(kOther), loaded & 1u, abort_flag, status, kErrO);
        if (ok && t == 1 && loaded > 0) ok = warp_wait(bar(kOtherRead), (loaded - 1) & 1u, abort_flag, status, kErrO);
        ++loaded;
      }
      if (!ok) break;
      const Work w = small->work[b];
      __syncwarp();
      if (lane == 0) mbar_arrive(bar(kTaken + b));
      tc_fence_after();
      const Coord c(args, w.unit);
      const int rows = args.seg_rows_q;
      // out = (w0 O_0 + w1 O_1) / (w0 l_0 + w1 l_1), w_t = 2^(m_t - max); a group
      // without a tile never wrote its O.
      // (Without one, group 1 may write here while S_0 reads the query tile: rows of S that nothing reads.)
      if (t == 1) {
        if (tiles == 0) continue;
#pragma unroll
        for (int q = 0; q < 4; ++q) {
          uint32_t o[32];
          tmem_ld32(o_addr + 32 * q, o);
          tmem_wait_ld();
          if (lane < rows) {
#pragma unroll
            for (int i = 0; i < 8; ++i)
              *reinterpret_cast<float4*>(rows_o + lane * kMergePad + 32 * q + 4 * i) =
                  any ? make_float4(__uint_as_float(o[4 * i]), __uint_as_float(o[4 * i + 1]),
                                    __uint_as_float(o[4 * i + 2]), __uint_as_float(o[4 * i + 3]))
                      : make_float4(0, 0, 0, 0);
          }
        }
        if (lane < rows) {
          rows_ml[2 * lane] = m;
          rows_ml[2 * lane + 1] = l;
        }
        __syncwarp();
        if (lane == 0) mbar_arrive(bar(kOther));
      } else {
        const bool live = tiles > 0 && lane < w.rows;
        const float m1 = lane < rows ? rows_ml[2 * lane] : -1e30f, l1 = lane < rows ? rows_ml[2 * lane + 1] : 0.f;
        const float top = fmaxf(m, m1);
        const float w0 = ex2_approx(m - top), w1 = ex2_approx(m1 - top);
        const float total = fmaf(w0, l, w1 * l1);
        const float inv_l = total > 0.f ? 1.f / total : 0.f;
        const float f0 = w0 * inv_l, f1 = w1 * inv_l;
        const int64_t at = static_cast<int64_t>(w.slot) * 2 * kBlockM + lane;  // of the split workspace
        uint16_t* out = static_cast<uint16_t*>(args.seg_out[0]) + c.batch * args.o_stride[0] + c.head * args.o_stride[3];
#pragma unroll
        for (int q = 0; q < 4; ++q) {
          uint32_t o[32];
          tmem_ld32(o_addr + 32 * q, o);
          tmem_wait_ld();
          if (lane < rows) {
#pragma unroll
            for (int i = 0; i < 4; ++i) {
              const float4 a = *reinterpret_cast<const float4*>(rows_o + lane * kMergePad + 32 * q + 8 * i);
              const float4 e = *reinterpret_cast<const float4*>(rows_o + lane * kMergePad + 32 * q + 8 * i + 4);
              const float other[8] = {a.x, a.y, a.z, a.w, e.x, e.y, e.z, e.w};
              float v[8];
#pragma unroll
              for (int x = 0; x < 8; ++x) {
                const float own = any ? __uint_as_float(o[8 * i + x]) : 0.f;
                v[x] = live ? fmaf(own, f0, other[x] * f1) : 0.f;
              }
              if (w.slot >= 0) {
                float4* dst = reinterpret_cast<float4*>(args.ws_o + at * kHeadDim + 32 * q + 8 * i);
                dst[0] = make_float4(v[0], v[1], v[2], v[3]);
                dst[1] = make_float4(v[4], v[5], v[6], v[7]);
              } else {
                *reinterpret_cast<uint4*>(out + lane * args.o_stride[2] + 32 * q + 8 * i) =
                    make_uint4(pack2<kFp16>(v[0], v[1]), pack2<kFp16>(v[2], v[3]), pack2<kFp16>(v[4], v[5]),
                               pack2<kFp16>(v[6], v[7]));
              }
            }
          }
        }
        if (w.slot >= 0 && lane < rows) args.ws_ml[at] = live ? make_float2(top, total) : make_float2(-1e30f, 0.f);
        __syncwarp();
        if (lane == 0 && tiles > 0) mbar_arrive(bar(kOtherRead));
        if (w.slot >= 0 && args.tickets) {
          // Whichever part is written last merges them, in the order of the
          // parts (a launch less: 3 us of a 25 us call).
          const int split_unit = w.slot / args.split;
          __threadfence();
          __syncwarp();
          int done = 0;
          if (lane == 0) done = atomicAdd(&args.tickets[split_unit], 1);
          done = __shfl_sync(0xffffffffu, done, 0);
          if (done == args.split - 1) {
            __threadfence();
            const int col = (lane & 15) * 8;
            for (int r = lane >> 4; r < rows; r += 2) {
              float acc[8];
              const float inv = merge_parts(args, split_unit, 0, r, col, acc);
              *reinterpret_cast<uint4*>(out + r * args.o_stride[2] + col) =
                  make_uint4(pack2<kFp16>(acc[0] * inv, acc[1] * inv), pack2<kFp16>(acc[2] * inv, acc[3] * inv),
                             pack2<kFp16>(acc[4] * inv, acc[5] * inv), pack2<kFp16>(acc[6] * inv, acc[7] * inv));
            }
          }
        }
      }
      tc_fence_before();  // O is read before the next unit's P is released
    }
  } else {
    // ------------------------------------------------------------ softmax
    const int t = warp >> 2;
    const int quarter = warp & 3;
    const int row = quarter * 32 + lane;
    const uint32_t lane_off = static_cast<uint32_t>(quarter * 32) << 16;
    const uint32_t s_addr = tmem + lane_off + 128 * t;
    const uint32_t o_addr = tmem + lane_off + 256 + 128 * t;
    const float scale_log2 = args.scale_log2;
    int n = 0, nt = 0, own = 0;  // tiles; tiles of this group; units with tiles of this group
    for (int u = 0;; ++u) {
      const int b = u & 1;
      if (!warp_wait(bar(kWork + b), (u >> 1) & 1u, abort_flag, status, kErrWork)) break;
      const int unit = small->work[b].unit, tiles = small->work[b].tiles;
      if (unit < 0) break;
      const bool two = (unit % args.npairs) * 2 + 1 < args.num_q_tiles;
      const bool mine = t == 0 || two;
      float m = -INFINITY, l = 0.f;
      bool ok = true;
      if (mine) {
        for (int i = 0; i < tiles; ++i, ++nt) {
          const int slot = (n + i) % kMetaRing;
          ok = warp_wait(bar(kMeta + slot), ((n + i) / kMetaRing) & 1u, abort_flag, status, kErrMeta);
          if (!ok) break;
          const int used = small->meta[slot];
          ok = warp_wait(bar(kS + t), nt & 1u, abort_flag, status, kErrS);
          if (!ok) break;
          // The group whose S comes last says that the tile's K is free.
          if (quarter == 0 && lane == 0 && t == (two ? 1 : 0)) mbar_arrive(bar(kFree + (n + i) % kRing));
          tc_fence_after();
          uint32_t sr[128];
          tmem_ld32_at<0>(s_addr + 0, sr);
          tmem_ld32_at<32>(s_addr + 32, sr);
          tmem_ld32_at<64>(s_addr + 64, sr);
          tmem_ld32_at<96>(s_addr + 96, sr);
          tmem_wait_ld();
          float s[128];
#pragma unroll
          for (int j = 0; j < 128; ++j) s[j] = __uint_as_float(sr[j]);
          if (used != (64 | (64 << 8))) {
            const int lo = used & 0xff, hi = used >> 8;
#pragma unroll
            for (int j = 0; j < 128; ++j)
              if ((j & 63) >= (j < 64 ? lo : hi)) s[j] = -INFINITY;
          }
          softmax_row<kFp16, true, true>(s, i == 0, scale_log2, s_addr, o_addr, bar(kPH + t * (kPParts - 1)), bar(kP + t), m, l);
        }
      }
      n += tiles;
      if (ok && mine && tiles > 0) ok = warp_wait(bar(kO + t), own++ & 1u, abort_flag, status, kErrO);
      if (!ok) break;
      const Work w = small->work[b];
      __syncwarp();
      if (lane == 0) mbar_arrive(bar(kTaken + b));
      if (!mine) continue;
      tc_fence_after();
      const Coord c(args, w.unit);
      const int tile = c.pair * 2 + t;
      const int row0 = tile * kBlockM;
      const int rows = min(kBlockM, args.seg_rows_q - row0);  // of the tensor in this tile
      // Rows behind the sequence's queries and rows that saw no key are zeros
      // (the accumulator of a unit without tiles was not written).
      const bool live = w.tiles > 0 && row0 + row < w.rows;
      const float inv_l = l > 0.f ? 1.f / l : 0.f;
      if (w.slot >= 0) {
        // One part of a list: O / l in fp32, m and l, merged by
        // attn_combine_kernel, which reads the rows of the tensor only.
        const int64_t at = (static_cast<int64_t>(w.slot) * 2 + t) * kBlockM + row;
        float4* dst = reinterpret_cast<float4*>(args.ws_o + at * kHeadDim);
        if (row - lane < rows) {  // uniform across the warp
#pragma unroll
          for (int q = 0; q < 4; ++q) {
            uint32_t o[32];
            tmem_ld32(o_addr + 32 * q, o);
            tmem_wait_ld();
            if (row < rows) {
#pragma unroll
              for (int j = 0; j < 8; ++j) {
                float4 v = make_float4(__uint_as_float(o[4 * j + 0]) * inv_l, __uint_as_float(o[4 * j + 1]) * inv_l,
                                       __uint_as_float(o[4 * j + 2]) * inv_l, __uint_as_float(o[4 * j + 3]) * inv_l);
                dst[8 * q + j] = live ? v : make_float4(0, 0, 0, 0);
              }
            }
          }
          if (row < rows) args.ws_ml[at] = live ? make_float2(m, l) : make_float2(-1e30f, 0.f);
        }
      } else {
        // Each warp stages 64 columns of its 32 rows (row r, 16-byte chunk k at
        // r*128 + ((k ^ (r & 7)) << 4)), then 8 threads store 128 bytes of a row.
        uint8_t* stage = smem + kStageOff + warp * kStageBytes;
        const int64_t base = c.batch * args.o_stride[0] + static_cast<int64_t>(row0 + quarter * 32) * args.o_stride[2] +
                             c.head * args.o_stride[3];
        uint16_t* out = static_cast<uint16_t*>(args.seg_out[0]) + base;
        const int k = lane & 7;
#pragma unroll
        for (int h = 0; h < 2; ++h) {
#pragma unroll
          for (int q = 0; q < 2; ++q) {
            uint32_t o[32];
            tmem_ld32(o_addr + 64 * h + 32 * q, o);
            tmem_wait_ld();
#pragma unroll
            for (int j = 0; j < 4; ++j) {
              uint4 v;
              v.x = pack2<kFp16>(__uint_as_float(o[8 * j + 0]) * inv_l, __uint_as_float(o[8 * j + 1]) * inv_l);
              v.y = pack2<kFp16>(__uint_as_float(o[8 * j + 2]) * inv_l, __uint_as_float(o[8 * j + 3]) * inv_l);
              v.z = pack2<kFp16>(__uint_as_float(o[8 * j + 4]) * inv_l, __uint_as_float(o[8 * j + 5]) * inv_l);
              v.w = pack2<kFp16>(__uint_as_float(o[8 * j + 6]) * inv_l, __uint_as_float(o[8 * j + 7]) * inv_l);
              if (!live) v = make_uint4(0, 0, 0, 0);
              *reinterpret_cast<uint4*>(stage + lane * 128 + (((4 * q + j) ^ (lane & 7)) << 4)) = v;
            }
          }
          __syncwarp();
#pragma unroll
          for (int p = 0; p < 8; ++p) {
            const int r = p * 4 + (lane >> 3);
            if (quarter * 32 + r < rows)
              *reinterpret_cast<uint4*>(out + r * args.o_stride[2] + h * 64 + 8 * k) =
                  *reinterpret_cast<const uint4*>(stage + r * 128 + ((k ^ (r & 7)) << 4));
          }
          __syncwarp();
        }
      }
      tc_fence_before();  // O is read before the next unit's P is released
    }
  }

  tc_fence_before();
  __syncthreads();
  if (warp == 9) {
    tc_fence_after();
    tmem_dealloc(tmem, 512);
  }
}

template <bool kFp16, bool kFew>
int launch(const CUtensorMap& tq, const CUtensorMap& tk, const CUtensorMap& tv, const AttnArgs& args, int64_t units,
           bool after_select, cudaStream_t stream) {
  static bool done[64] = {false};
  int dev = 0;
  if (cudaGetDevice(&dev) != cudaSuccess || dev < 0 || dev >= 64) dev = 0;
  if (!done[dev]) {
    const cudaError_t err =
        cudaFuncSetAttribute(sparse_attn_kernel<kFp16, kFew>, cudaFuncAttributeMaxDynamicSharedMemorySize, kSmem);
    if (err != cudaSuccess) return set_cuda_error("sparse attention: cudaFuncSetAttribute", err);
    done[dev] = true;
  }
  const int64_t split_units = args.split > 1 ? units - args.full_units : 0;
  const int64_t ctas = args.full_units + (split_units > 0 ? split_units * args.split : units - args.full_units);
  if (ctas <= 0) return 0;
  if (ctas > 0x7fffffff) return set_error(PS_B200_ERR_UNSUPPORTED, "attention grid above 2^31 CTAs");
  const cudaError_t err = launch_after(sparse_attn_kernel<kFp16, kFew>, dim3(static_cast<unsigned>(ctas)), dim3(kThreads),
                                       kSmem, stream, after_select, tq, tk, tv, args);
  if (err != cudaSuccess) return set_cuda_error("sparse attention launch", err);
  count_launch();
  if (split_units > 0 && !args.tickets) return launch_combine(args, split_units, kFp16, true, stream);
  return 0;
}

}  // namespace
}  // namespace attn

int launch_sparse_attention(const CUtensorMap& tq, const CUtensorMap& tk, const CUtensorMap& tv, const AttnArgs& args,
                            int64_t total_units, bool fp16, bool after_select, cudaStream_t stream) {
  const bool few = args.seg_rows_q <= kMergeRows;
  auto launch = fp16 ? (few ? attn::launch<true, true> : attn::launch<true, false>)
                     : (few ? attn::launch<false, true> : attn::launch<false, false>);
  return launch(tq, tk, tv, args, total_units, after_select, stream);
}

}  // namespace psb
