// Attention of packed query rows on the tensor cores, for prompts of
// different lengths (packed_attn.cu) and for drafted trees over the paged
// cache (tree_attn.cu): O = softmax(scale Q K^T + mask) V per kv head, one
// pass over the keys with the running maximum and sum of the softmax.
//
// Rows. All query heads that share a kv head are rows of the same tile: row
// r of a tile is token r / group, head r % group (one 3-D TMA box), so a
// short sequence or a small tree fills a tile and K/V are read once for the
// whole group. A work item has up to two tiles of 128 rows ("streams").
//
//   warps 0-3, 4-7   softmax of stream 0 and 1, one thread per row: S row
//                    from TMEM to registers, mask, running max m and sum l,
//                    P = 2^(s - m) rounded to the input type into TMEM; at the
//                    end O / l to global memory
//   warps 8, 9       MMA issuer (one lane) of stream 0 and 1: S_x = Q_x K_j^T
//                    (shared memory operands), O_x += P_x V_j (P from TMEM:
//                    shared memory carries Q, K and V reads only, 96 bytes a
//                    clock at full MMA rate instead of 160)
//   warps 10, 14     TMA producers of the K and of the V tiles, a ring each
//   warp 11 (1 lane) TMA producer of the Q tiles
//   warp 12          looks over each V tile that some row must not see whole
//   warp 13 (1 lane) works out the CTA's next items for the other warps: a ring
//                    of kRowItems descriptions in shared memory
//
// Two streams keep the tensor cores fed: while one does its softmax, the
// other's P V and next Q K^T run. In PAIR items the streams are two Q tiles
// that read the same K/V tiles. An item with one Q tile runs as ALT: both
// streams hold that tile and take the even and the odd key tiles, and stream
// 0 merges the two results at the end. Each stream has its own issuing warp:
// with one thread issuing for both, its waits and commits (2000 cycles a
// step) came between the products (16383 tokens of 32 + 4 heads: 2.97 ms).
//
// With 128-wide heads TMEM is full and P overwrites S in place, so S_x(j+1) is
// issued after P V_x(j): MMAs of one thread execute in order. For the same
// reason S_x(j+1) being complete means that P V_x(j) is, and O_x may then be
// rescaled without another barrier. With 64-wide heads P has its own columns:
// S_x(j+1) goes out as soon as S_x(j) has been read, under the powers (16383
// tokens of 32 + 4 heads: 1.81 -> 1.58 ms), and a barrier tells when P V_x(j)
// is done. O is rescaled only when a row's max grew by more than 2^8 since its
// P values were scaled (P <= 2^8 is exact in range for bf16 and fp16, and l is
// fp32).
//
// Masked keys: scores are replaced, not added to, so NaN or infinite keys
// cannot reach a row that does not see them. Values are different, as 0 * NaN
// = NaN in the product: warp 12 zeroes what is not finite in V tiles that
// some row sees only in part (and rows past the sequence's end), and the
// epilogue adds those elements to the rows that do see them. (An infinite value
// whose weight rounds to 0 in P is NaN from a tile seen whole, as 0 * inf, and
// infinity from one seen in part; neither is promised.)
//
// Measured (B200): 16383 tokens of 32 + 4 heads of 128 in 2.0-2.27 ms, 970 to
// 1090 TFLOP/s of causal products, of 1641 that cuBLAS reaches in a burst and
// 1388 under the power cap; 32 trees of 16 nodes over 2000-4096 keys in 86-98
// us with the joins, 4.1-4.7 TB/s of K and V. What bounds it is the chain of a
// stream's scores, softmax and products (1950 cycles of softmax and as many of
// waiting a tile), for trees the stream of K/V tiles (what holds it below the
// copy rate is not known; a third V stage helped, a second Q tile's place is
// all that is left for another). The code is kept short (waits counted in
// polls, loops rolled): at 106 KB a sixth of its instruction requests missed.
//
// Every wait is bounded; a timeout sets the device status and the kernel
// drains.
#pragma once

#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include <atomic>
#include <type_traits>

#include "ptx.cuh"
#include "runtime.h"

namespace kvm {

constexpr int kRowThreads = 512;
// Registers a thread after the warps have split up: 128 * 512 at launch.
constexpr int kRowSoftmaxRegs = 200;    // warps 0-7
constexpr int kRowControlRegs = 56;     // warps 8-15
constexpr float kRowRescale = 8.0f;     // log2 units
constexpr int kRowMaxSeqs = 1024;       // sequences of one call (tables in shared memory)
constexpr int kRowMaxDirty = 10;        // V tiles of an item that a row sees in part
constexpr int kRowItems = 4;            // item descriptions in the ring
constexpr int kRowItemUsers = 14;       // warps that give one back: 0-12 and 14
constexpr int kRowBadWords = kRowMaxDirty * 4 + 4;  // their bad values' keys; any; padding
constexpr int kRowMaxNodes = 1024;

// Shared memory of one CTA for head width D. ONE: no item has a second Q tile,
// whose place then goes to the V ring.
template <int D, bool TREE, bool ONE>
struct RowSmem {
  static constexpr int kHalves = D / 64;
  // A step's products go out under a lock, one stream's after the other's, in
  // items of kLockTiles key tiles and more, where the tensor cores are nearly the
  // bound (16383 tokens: 2.1 ms with, 2.50 without); not in shorter ones, which
  // wait for their softmax, nor for trees of one Q tile, which wait for memory
  // (32 trees: 96 us with, 94 without), nor where S does not wait for P V.
  static constexpr bool kLock = !ONE && D == 128;
  static constexpr int kLockTiles = 6;
  // TMEM columns: S_0 and S_1 (128 each), O_0 and O_1 (D each). With 64-wide
  // heads P_0 and P_1 (64 each) have their own; with 128 they lie over S.
  static constexpr bool kOwnP = D == 64;
  static constexpr uint32_t kColO = 256, kColP = kOwnP ? 384 : 0, kStepP = kOwnP ? 64 : 128;
  static constexpr uint32_t kHalf = 128 * 64 * 2;            // 128 rows x 64 columns
  static constexpr uint32_t kTile = kHalves * kHalf;
  static constexpr int kStagesK = D == 128 ? 2 : 4;
  static constexpr int kStagesV = kStagesK + (ONE ? 1 : 0);
  static constexpr uint32_t kOffQ = 0;                       // [2], one with ONE
  static constexpr uint32_t kOffK = (ONE ? 1 : 2) * kTile;   // [kStagesK]
  static constexpr uint32_t kOffV = kOffK + kStagesK * kTile;
  static constexpr uint32_t kOffTab = kOffV + kStagesV * kTile;
  static constexpr uint32_t kTabBytes = kRowMaxSeqs * (TREE ? 4 : 10) + 16;
  static constexpr uint32_t kOffBad = kOffTab + kTabBytes;
  static constexpr uint32_t kOffItems = kOffBad + kRowItems * kRowBadWords * 4;
  static constexpr uint32_t kOffMl = kOffItems + kRowItems * 64;
  static constexpr uint32_t kOffPages = kOffMl + 2 * 128 * 8;
  static constexpr uint32_t kPageSlots = 128;                // page ids a producer reads ahead
  static constexpr uint32_t kOffOut = kOffPages + 2 * kPageSlots * 4;  // [8 warps][32 rows][64 B]
  static constexpr uint32_t kOffBar = kOffOut + 8 * 2048;
  // q_full[2] q_empty[2] k_full[] k_empty[] v_full[] v_empty[] s_full[2] p_full[2]
  // o_full[2] o_free[2] alt_ml[2] looked[I] it_full[I] it_empty[I] drain[2] s_read[2]
  // pv_done[2]
  static constexpr int kBars = 2 * (kStagesK + kStagesV) + 20 + 3 * kRowItems;
  static constexpr size_t bytes() { return 1024 + kOffBar + kBars * 8 + 16; }
};

struct RowParams {
  int S, HQ, HKV, group;
  int tile_tokens;       // tokens of a Q tile: 128 / group
  int rows;              // rows of q and out
  float scale_log2;
  void* out;
  long long ldo;
  const int* q_off;      // [S+1]
  int* status;
  // values again, for the epilogue's rare path
  const void* v;
  long long ldv;
  // ---- trees over the paged cache
  const int* q_pos;      // [S] cached tokens before the tree
  const unsigned* mask;  // [rows, words]
  int words, max_nodes, max_keys;
  int whole;             // items are not cut
  const int* bt;
  const int* bt_off;
  int bt_len;            // entries of bt
  int block_size, block_log2, box_rows, num_pages, layer;
  long long page_rows, layer_rows, kv_rows;  // strides in token slots
  float* ws_o;           // [2 * grid][256][128]
  float* ws_ml;          // [2 * grid][256][2]
  struct RowJoin* ws_join;  // [grid]
};

// What the joining kernel does for a CTA: the item that the CTA begins and the
// next ones go on with (ntok0 = 0: none).
struct RowJoin {
  int row0, kh, ntok0, ntok1;
  int part, last;        // the CTA's slot; the last CTA, which has its part in slot 2 * last
  int s, tok0;
};

// A stretch of work: tiles [t0, t0 + n) of the keys for up to two Q tiles.
struct RowItem {
  int s, kh;
  int row0;              // row of q of stream 0's first token
  int tok0;              // that token's index in its sequence (node index of a tree)
  int ntok0, ntok1;      // tokens of the two Q tiles
  int key0;              // prompts: row of the sequence's first key
  int ctx, nodes;        // trees
  int keys;              // keys of the sequence
  int t0, n, n0, n1;
  int alt;
  int part;              // slot of a partial result, -1: the whole result

  __device__ __forceinline__ int count(int x) const {
    return alt ? (x ? n >> 1 : (n + 1) >> 1) : (x ? n1 : n0);
  }
  __device__ __forceinline__ int tile(int x, int i) const { return alt ? 2 * i + x : i; }
  // Whether both streams use the item's key tile j.
  __device__ __forceinline__ bool shared(int j) const { return !alt && j < n0 && j < n1; }
};

// Tables in shared memory, built once per CTA from the offsets on the device.
struct RowTables {
  int* start;            // prompts: first item of rank r's block; trees: first tile (item) of s
  int* count;            // prompts: items of the sequence of rank r
  unsigned short* order; // prompts: sequence of rank r
  int* total;            // items (prompts) or tiles (trees)
};

template <typename L>
__device__ __forceinline__ RowTables row_tables(uint8_t* smem) {
  RowTables t;
  uint8_t* p = smem + L::kOffTab;
  t.start = reinterpret_cast<int*>(p);
  t.count = reinterpret_cast<int*>(p + kRowMaxSeqs * 4);            // prompts
  t.order = reinterpret_cast<unsigned short*>(p + kRowMaxSeqs * 8);  // prompts
  t.total = reinterpret_cast<int*>(p + L::kTabBytes - 16);
  return t;
}

// ------------------------------------------------------------- prompts ---
//
// Items of a sequence of n items are its Q tile pairs; the i-th costs about i
// key tiles. They are dealt heaviest first: by i from the longest sequence's
// last down to 0, every sequence that has an i-th item in turn. With the
// sequences ranked by n descending, r + 1 of them have the items of the
// levels (n_{r+1}, n_r], which start at item sum_{i<r} (n_i - n_r).
__device__ __forceinline__ void build_prompt_tables(const RowParams& p, RowTables t,
                                                    int* scratch) {
  const int per = 2 * p.tile_tokens;
  // Sequences before the first bad one are disjoint, which bounds the items;
  // the bad one and all after it are left out.
  int* good = t.total;
  if (threadIdx.x == 0) *good = p.S;
  __syncthreads();
#pragma unroll 1
  for (int s = threadIdx.x; s < p.S; s += kRowThreads) {
    const int a = p.q_off[s], b = p.q_off[s + 1];
    const bool bad = a < 0 || b < a || b > p.rows;
    if (bad) atomicMin(good, s);
    scratch[s] = bad ? 0 : static_cast<int>((static_cast<long long>(b - a) + per - 1) / per);
  }
  __syncthreads();
  const int n_good = *good;
  if (n_good < p.S && blockIdx.x == 0 && threadIdx.x == 0) atomicOr(p.status, kDevBadInput);
#pragma unroll 1
  for (int s = n_good + threadIdx.x; s < p.S; s += kRowThreads) scratch[s] = 0;
  __syncthreads();
#pragma unroll 1
  for (int s = threadIdx.x; s < p.S; s += kRowThreads) {
    const int n = scratch[s];
    int rank = 0;
#pragma unroll 1
    for (int i = 0; i < p.S; ++i) {
      const int m = scratch[i];
      rank += m > n || (m == n && i < s);
    }
    t.order[rank] = static_cast<unsigned short>(s);
    t.count[rank] = n;
  }
  __syncthreads();
  if (threadIdx.x < 32) {
    int before = 0;  // items of the ranks before this chunk
#pragma unroll 1
    for (int r0 = 0; r0 < p.S; r0 += 32) {
      const int r = r0 + threadIdx.x;
      const int n = r < p.S ? t.count[r] : 0;
      int sum = n;
#pragma unroll
      for (int o = 1; o < 32; o <<= 1) {
        const int up = __shfl_up_sync(0xffffffffu, sum, o);
        if (static_cast<int>(threadIdx.x) >= o) sum += up;
      }
      if (r < p.S) t.start[r] = before + sum - n - r * n;
      before += __shfl_sync(0xffffffffu, sum, 31);
    }
    if (threadIdx.x == 0) *t.total = before;
  }
  __syncthreads();
}

struct PromptItems {
  int round = 0;
  // The CTA's next item: rounds of one item per CTA, every other one in
  // reverse, so no CTA always gets a round's heaviest.
  __device__ __forceinline__ bool next(const RowParams& p, const RowTables& t, RowItem& it) {
    const int G = gridDim.x, b = blockIdx.x;
    const int w = round * G + (round & 1 ? G - 1 - b : b);
    ++round;
    if (w >= *t.total * p.HKV) return false;
    it.kh = w % p.HKV;
    const int u = w / p.HKV;
    int lo = 0, hi = p.S - 1;
#pragma unroll 1
    while (lo < hi) {
      const int mid = (lo + hi + 1) >> 1;
      if (t.start[mid] <= u) lo = mid; else hi = mid - 1;
    }
    const int i = u - t.start[lo];
    const int q_item = t.count[lo] - 1 - i / (lo + 1);
    it.s = t.order[i % (lo + 1)];
    it.key0 = p.q_off[it.s];
    it.keys = p.q_off[it.s + 1] - it.key0;
    it.tok0 = q_item * 2 * p.tile_tokens;
    it.row0 = it.key0 + it.tok0;
    const int left = it.keys - it.tok0;
    it.ntok0 = min(left, p.tile_tokens);
    it.ntok1 = max(0, min(left - p.tile_tokens, p.tile_tokens));
    it.ctx = it.nodes = 0;
    it.t0 = 0;
    it.n0 = (it.tok0 + it.ntok0 + 127) >> 7;
    it.n1 = it.ntok1 > 0 ? (it.tok0 + it.ntok0 + it.ntok1 + 127) >> 7 : 0;
    it.n = max(it.n0, it.n1);
    it.alt = it.ntok1 == 0 && it.n > 1;
    it.part = -1;
    return true;
  }
};

// --------------------------------------------------------------- trees ---
//
// The key tiles of all (sequence, query tile pair, kv head) in a row, in that
// order, are cut into one stretch of equal length per CTA: every CTA streams
// the same number of K/V tiles whatever the contexts. A stretch that begins
// or ends inside an item leaves a partial result; the joining kernel joins
// them. A few short items (`whole`) are dealt out uncut instead, one to a CTA.
__device__ __forceinline__ int tree_pairs(const RowParams& p, int nodes) {
  return (nodes + 2 * p.tile_tokens - 1) / (2 * p.tile_tokens);
}

// Whether a sequence's rows [a, b) are no rows of q.
__device__ __forceinline__ bool tree_bad_rows(const RowParams& p, int a, int b) {
  return a < 0 || b < a || b > p.rows;
}

// Key tiles of sequence s, 0 for one that is empty or refused.
__device__ __forceinline__ int tree_tiles(const RowParams& p, int s, int& nodes, int& ctx,
                                          bool report) {
  const int a = p.q_off[s], b = p.q_off[s + 1];
  ctx = p.q_pos[s];
  nodes = b - a;
  const bool bad = tree_bad_rows(p, a, b) || ctx < 0 || nodes > p.max_nodes ||
                   ctx > p.max_keys - nodes;
  if (bad && report) atomicOr(p.status, kDevBadInput);
  if (bad || nodes == 0) { nodes = 0; return 0; }
  return (ctx + nodes + 127) >> 7;
}

// Sequences before the first one with bad rows own disjoint rows; that one and
// all after it are left out, as they could write rows of the others.
__device__ __forceinline__ void build_tree_tables(const RowParams& p, RowTables t, bool report) {
  if (threadIdx.x < 32) {
    int before = 0;
    bool left_out = false;  // by a sequence of an earlier chunk
#pragma unroll 1
    for (int s0 = 0; s0 < p.S; s0 += 32) {
      const int s = s0 + threadIdx.x;
      int n = 0;
      bool bad_rows = false;
      if (s < p.S) {
        int nodes, ctx;
        const int tiles = tree_tiles(p, s, nodes, ctx, report);
        n = (p.whole ? tiles > 0 : tiles) * tree_pairs(p, nodes) * p.HKV;
        bad_rows = tree_bad_rows(p, p.q_off[s], p.q_off[s + 1]);
      }
      const unsigned from = __ballot_sync(0xffffffffu, bad_rows);
      if (left_out || (from & ((2u << threadIdx.x) - 1u)) != 0) n = 0;
      left_out = left_out || from != 0;
      int sum = n;
#pragma unroll
      for (int o = 1; o < 32; o <<= 1) {
        const int up = __shfl_up_sync(0xffffffffu, sum, o);
        if (static_cast<int>(threadIdx.x) >= o) sum += up;
      }
      if (s < p.S) t.start[s] = before + sum - n;
      before += __shfl_sync(0xffffffffu, sum, 31);
    }
    if (threadIdx.x == 0) *t.total = before;
  }
  __syncthreads();
}

// Tiles per CTA: at least 4, so that small calls are not cut to pieces.
__device__ __forceinline__ int tree_share(int total, int ctas) {
  return max(4, (total + ctas - 1) / ctas);
}

struct TreeItems {
  int pos = -1, end = 0, first = 1, share = 1;
  __device__ __forceinline__ bool next(const RowParams& p, const RowTables& t, RowItem& it) {
    if (pos < 0) {
      const int total = *t.total;
      share = p.whole ? 1 : tree_share(total, gridDim.x);
      const long long b = static_cast<long long>(blockIdx.x) * share;
      pos = b < total ? static_cast<int>(b) : total;
      end = min(pos + share, total);
    }
    if (pos >= end) return false;
    int lo = 0, hi = p.S - 1;
#pragma unroll 1
    while (lo < hi) {
      const int mid = (lo + hi + 1) >> 1;
      if (t.start[mid] <= pos) lo = mid; else hi = mid - 1;
    }
    it.s = lo;
    const int tiles = tree_tiles(p, lo, it.nodes, it.ctx, false);
    const int at = pos - t.start[lo];
    const int item = p.whole ? at : at / tiles;
    it.kh = item % p.HKV;
    it.tok0 = item / p.HKV * 2 * p.tile_tokens;
    it.key0 = 0;
    it.row0 = p.q_off[lo] + it.tok0;
    it.keys = it.ctx + it.nodes;
    it.t0 = p.whole ? 0 : at - item * tiles;
    it.n = p.whole ? tiles : min(tiles - it.t0, end - pos);
    const int left = it.nodes - it.tok0;
    it.ntok0 = min(left, p.tile_tokens);
    it.ntok1 = max(0, min(left - p.tile_tokens, p.tile_tokens));
    it.n0 = it.n;
    it.n1 = it.ntok1 > 0 ? it.n : 0;
    it.alt = it.ntok1 == 0 && it.n > 1;
    it.part = it.n == tiles ? -1 : 2 * int(blockIdx.x) + (first ? 0 : 1);
    first = 0;
    pos = p.whole ? end : pos + it.n;
    return true;
  }
};

// -------------------------------------------------------------- pieces ---

// D[tmem] (+)= A[tmem] x B[smem desc]^T, kind::f16; A holds 128 rows of 16-bit
// pairs, one row per lane.
__device__ __forceinline__ void mma_f16_ts(uint32_t d_tmem, uint32_t a_tmem, uint64_t b_desc,
                                           uint32_t idesc, uint32_t accumulate) {
  asm volatile(
      "{\n\t.reg .pred p;\n\t"
      "setp.ne.b32 p, %4, 0;\n\t"
      "tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], %2, %3, p;\n\t}" ::"r"(d_tmem),
      "r"(a_tmem), "l"(b_desc), "r"(idesc), "r"(accumulate)
      : "memory");
}

// Bounded waits, counted in polls instead of by the clock: there are many of
// them, and the kernel's code has to stay in the instruction cache.
constexpr uint32_t kRowPolls = 1u << 26;  // of 20 ns and more: over a second
__device__ __forceinline__ bool row_wait(uint64_t* bar, uint32_t parity, volatile int* abort) {
#pragma unroll 1
  for (uint32_t left = kRowPolls; left != 0; --left) {
    if (mbar_try_wait(bar, parity)) return true;
    if ((left & 63u) == 0 && *abort) return false;
  }
  *abort = 1;
  return false;
}

// A count in shared memory that one warp raises and others wait for.
__device__ __forceinline__ void st_release_cta(uint32_t* p, uint32_t v) {
  asm volatile("st.release.cta.shared::cta.u32 [%0], %1;" ::"r"(smem_u32(p)), "r"(v) : "memory");
}
__device__ __forceinline__ uint32_t ld_acquire_cta(const uint32_t* p) {
  uint32_t v;
  asm volatile("ld.acquire.cta.shared::cta.u32 %0, [%1];" : "=r"(v) : "r"(smem_u32(p)) : "memory");
  return v;
}
__device__ __forceinline__ bool count_wait(const uint32_t* p, uint32_t at_least,
                                           volatile int* abort) {
#pragma unroll 1
  for (uint32_t left = kRowPolls; left != 0; --left) {
    if (static_cast<int32_t>(ld_acquire_cta(p) - at_least) >= 0) return true;
    if ((left & 255u) == 0 && *abort) return false;
  }
  *abort = 1;
  return false;
}

// A lock in shared memory between two threads of the CTA that each hold it
// for a bounded time. Returns false when the wait gave up.
__device__ __forceinline__ bool lock_take(uint32_t* p, volatile int* abort) {
#pragma unroll 1
  for (uint32_t left = kRowPolls; left != 0; --left) {
    uint32_t was;
    asm volatile("atom.relaxed.cta.shared::cta.cas.b32 %0, [%1], 0, 1;"
                 : "=r"(was) : "r"(smem_u32(p)) : "memory");
    if (was == 0) return true;
    if ((left & 255u) == 0 && *abort) return false;
  }
  *abort = 1;
  return false;
}

__device__ __forceinline__ bool mbar_test(uint64_t* bar, uint32_t parity) {
  uint32_t ok;
  asm volatile(
      "{\n\t.reg .pred p;\n\t"
      "mbarrier.test_wait.parity.shared::cta.b64 p, [%1], %2;\n\t"
      "selp.u32 %0, 1, 0, p;\n\t}"
      : "=r"(ok) : "r"(smem_u32(bar)), "r"(parity) : "memory");
  return ok != 0;
}

__device__ __forceinline__ void st_global_if(bool on, unsigned long long to, uint4 v) {
  asm volatile(
      "{\n\t.reg .pred p;\n\t"
      "setp.ne.u32 p, %0, 0;\n\t"
      "@p st.global.v4.b32 [%1], {%2, %3, %4, %5};\n\t}" ::"r"(static_cast<uint32_t>(on)),
      "l"(to), "r"(v.x), "r"(v.y), "r"(v.z), "r"(v.w)
      : "memory");
}

// 3-D tiled TMA load (x innermost).
__device__ __forceinline__ void tma_load_3d(void* dst, const void* tmap, uint64_t* bar,
                                            int32_t x, int32_t y, int32_t z) {
  asm volatile(
      "cp.async.bulk.tensor.3d.shared::cluster.global.tile.mbarrier::complete_tx::bytes "
      "[%0], [%1, {%3, %4, %5}], [%2];" ::"r"(smem_u32(dst)),
      "l"(tmap), "r"(smem_u32(bar)), "r"(x), "r"(y), "r"(z)
      : "memory");
}

// Maxima that are NaN when an argument is: a row that sees a NaN score is NaN.
__device__ __forceinline__ float max3(float a, float b, float c) {
  float r;
  asm("max.NaN.f32 %0, %1, %2, %3;" : "=f"(r) : "f"(a), "f"(b), "f"(c));
  return r;
}
__device__ __forceinline__ float max2(float a, float b) {
  float r;
  asm("max.NaN.f32 %0, %1, %2;" : "=f"(r) : "f"(a), "f"(b));
  return r;
}

template <int N>
__device__ __forceinline__ void reg_give() {
  asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(N));
}
template <int N>
__device__ __forceinline__ void reg_take() {
  asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(N));
}

template <bool F16>
__device__ __forceinline__ uint32_t pack16(float a, float b) {
  if constexpr (F16) {
    const __half2 h = __floats2half2_rn(a, b);
    return *reinterpret_cast<const uint32_t*>(&h);
  } else {
    const __nv_bfloat162 h = __floats2bfloat162_rn(a, b);
    return *reinterpret_cast<const uint32_t*>(&h);
  }
}

template <bool F16>
__host__ __device__ constexpr uint32_t row_idesc(int n, int b_mn) {
  const uint32_t type = F16 ? 0u : 1u;
  return (1u << 4) | (type << 7) | (type << 10) | (static_cast<uint32_t>(b_mn) << 16) |
         (static_cast<uint32_t>(n >> 3) << 17) | (static_cast<uint32_t>(128 >> 4) << 24);
}

// Bits of the mask of one tree row for the 32 keys from `rel` (the key's index
// minus the cached ones) on: cached keys all seen, drafted ones by the mask.
__device__ __forceinline__ unsigned tree_bits(const unsigned* mask, int words, int nodes,
                                              int rel) {
  if (rel <= -32) return 0xffffffffu;
  if (rel >= nodes) return 0u;
  const int w = rel >> 5;
  const unsigned lo = w < 0 ? 0xffffffffu : w < words ? mask[w] : 0u;
  const unsigned hi = w + 1 < words ? mask[w + 1] : 0u;
  unsigned bits = __funnelshift_r(lo, hi, rel & 31);
  const int left = nodes - rel;  // keys of the sequence from rel on
  if (left < 32) bits &= (1u << left) - 1u;
  return bits;
}

// Whether row (token t of its sequence) sees key k.
template <bool TREE>
__device__ __forceinline__ bool row_sees(const RowItem& it, const unsigned* mask, int words,
                                         int token, int k) {
  if constexpr (!TREE) return k <= token;
  if (k < it.ctx) return true;
  const int j = k - it.ctx;
  return j < it.nodes && (j >> 5) < words && (mask[j >> 5] >> (j & 31) & 1u);
}

// First key tile (relative to the item's) that some row sees only in part.
template <bool TREE>
__device__ __forceinline__ int first_dirty(const RowItem& it) {
  const int k = TREE ? it.ctx : it.tok0 + 1;  // first key not seen by all
  return max(0, (k >> 7) - it.t0);
}

// Pages in sequence s's table, none if it leaves the list.
__device__ __forceinline__ int table_entries(const RowParams& p, int s) {
  const int a = p.bt_off[s], b = p.bt_off[s + 1];
  return a < 0 || b > p.bt_len ? 0 : b - a;
}

// Address of the value row of key k (the epilogue's rare path), or NULL.
template <bool TREE>
__device__ __forceinline__ const uint16_t* value_row(const RowParams& p, const RowItem& it,
                                                     int D, int k) {
  long long row = it.key0 + k;
  if constexpr (TREE) {
    const int idx = k >> p.block_log2, b0 = p.bt_off[it.s];
    const int page = idx < table_entries(p, it.s) ? p.bt[b0 + idx] : -1;
    if (page < 0 || page >= p.num_pages) return nullptr;
    row = page * p.page_rows + p.layer * p.layer_rows + p.kv_rows + k % p.block_size;
  }
  return static_cast<const uint16_t*>(p.v) + row * p.ldv + static_cast<long long>(it.kh) * D;
}

template <bool F16>
__device__ __forceinline__ bool nonfinite16(uint16_t b) {
  constexpr uint16_t top = F16 ? 0x7C00 : 0x7F80;
  return (b & top) == top;
}
template <bool F16>
__device__ __forceinline__ float widen16(uint16_t b) {
  if constexpr (F16) return __half2float(*reinterpret_cast<const __half*>(&b));
  else return __uint_as_float(static_cast<uint32_t>(b) << 16);
}

// -------------------------------------------------------------- kernel ---

template <int D, bool F16, bool TREE, bool ONE>
__global__ void __launch_bounds__(kRowThreads, 1)
    row_attn_kernel(const __grid_constant__ CUtensorMap tmQ,
                    const __grid_constant__ CUtensorMap tmK,
                    const __grid_constant__ CUtensorMap tmV, const __grid_constant__ RowParams p) {
  using L = RowSmem<D, TREE, ONE>;
  using Items = typename std::conditional<TREE, TreeItems, PromptItems>::type;
  constexpr int NK = L::kStagesK, NV = L::kStagesV;
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>(
      (reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  uint64_t* bars = reinterpret_cast<uint64_t*>(smem + L::kOffBar);
  uint64_t* q_full = bars;                      // [2]
  uint64_t* q_empty = q_full + 2;               // [2]
  uint64_t* k_full = q_empty + 2;               // [NK]
  uint64_t* k_empty = k_full + NK;              // [NK] 2 arrivals
  uint64_t* v_full = k_empty + NK;              // [NV]
  uint64_t* v_empty = v_full + NV;              // [NV] 2 arrivals
  uint64_t* s_full = v_empty + NV;              // [2]
  uint64_t* p_full = s_full + 2;                // [2] 128 arrivals
  uint64_t* o_full = p_full + 2;                // [2]
  uint64_t* o_free = o_full + 2;                // [2] 128 arrivals
  uint64_t* alt_ml = o_free + 2;                // [2] 128 arrivals
  uint64_t* looked = alt_ml + 2;                // [kRowItems]
  uint64_t* it_full = looked + kRowItems;       // [kRowItems]
  uint64_t* it_empty = it_full + kRowItems;     // [kRowItems] kRowItemUsers arrivals
  uint64_t* drain = it_empty + kRowItems;       // [2]
  uint64_t* s_read = drain + 2;                 // [2] 128 arrivals (kOwnP)
  uint64_t* pv_done = s_read + 2;               // [2] (kOwnP)
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(bars + L::kBars);
  volatile int* abort_flag = reinterpret_cast<volatile int*>(tmem_slot + 1);
  uint32_t* v_count = tmem_slot + 2;            // V tiles looked over, ever
  uint32_t* mma_lock = tmem_slot + 3;
  unsigned* bad_words = reinterpret_cast<unsigned*>(smem + L::kOffBad);
  float2* alt_buf = reinterpret_cast<float2*>(smem + L::kOffMl);   // [2][128]
  const RowTables tab = row_tables<L>(smem);

  RowItem* ring = reinterpret_cast<RowItem*>(smem + L::kOffItems);
  static_assert(sizeof(RowItem) == 64, "one 64-byte slot each");
  // The next item for a warp (or its one lane): the ord-th of the CTA. False
  // at the end, or when the wait gave up. A slot is given back by every user.
  auto next_item = [&](uint32_t ord, RowItem& it) {
    const uint32_t slot = ord % kRowItems;
    if (!row_wait(&it_full[slot], (ord / kRowItems) & 1, abort_flag)) return false;
    it = ring[slot];
    return it.n > 0;
  };
  auto item_done = [&](uint32_t ord) { mbar_arrive(&it_empty[ord % kRowItems]); };

  const int warp = threadIdx.x / 32;
  const int lane = threadIdx.x % 32;

  if (threadIdx.x == 0) {
    *abort_flag = 0;
    *v_count = 0;
    *mma_lock = 0;
    for (int i = 0; i < 2; ++i) {
      mbar_init(&q_full[i], 1);
      mbar_init(&q_empty[i], 2 - i);
      mbar_init(&drain[i], 1);
      mbar_init(&s_read[i], 128);
      mbar_init(&pv_done[i], 1);
      mbar_init(&s_full[i], 1);
      mbar_init(&p_full[i], 128);
      mbar_init(&o_full[i], 1);
      mbar_init(&o_free[i], 128);
      mbar_init(&alt_ml[i], 128);
    }
    for (int i = 0; i < NK; ++i) {
      mbar_init(&k_full[i], 1);
      mbar_init(&k_empty[i], 2);
    }
    for (int i = 0; i < NV; ++i) {
      mbar_init(&v_full[i], 1);
      mbar_init(&v_empty[i], 2);
    }
    for (int i = 0; i < kRowItems; ++i) {
      mbar_init(&looked[i], 1);
      mbar_init(&it_full[i], 1);
      mbar_init(&it_empty[i], kRowItemUsers);
    }
    fence_mbar_init();
    tma_prefetch_desc(&tmQ);
    tma_prefetch_desc(&tmK);
    tma_prefetch_desc(&tmV);
  }
  if (warp == 8) {
    tmem_alloc(tmem_slot, 512);
    tmem_relinquish();
  }
  // All before this may overlap the kernel ahead in the stream; what follows
  // reads what it may have written.
  pdl_wait();
  pdl_trigger();
  if constexpr (TREE) build_tree_tables(p, tab, blockIdx.x == 0);
  else build_prompt_tables(p, tab, reinterpret_cast<int*>(smem + L::kOffK));
  fence_async_smem();  // the tables' scratch becomes a tile of the ring
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = *tmem_slot;

  if (warp >= 8) {
    reg_give<kRowControlRegs>();
    if (warp == 10 || warp == 14) {
      // ------------------------------------------------ K and V producers
      const int kv = warp == 14;
      const uint32_t N = kv ? NV : NK;
      uint64_t* full = kv ? v_full : k_full;
      uint64_t* empty = kv ? v_empty : k_empty;
      uint8_t* tiles = smem + (kv ? L::kOffV : L::kOffK);
      const void* map = kv ? &tmV : &tmK;
      int* page_ids = reinterpret_cast<int*>(smem + L::kOffPages) + kv * L::kPageSlots;
      RowItem it;
      uint32_t st = 0, phase = 1;  // the ring's next slot
      bool ok = true;
#pragma unroll 1
      for (uint32_t ord = 0; ok && __all_sync(0xffffffffu, next_item(ord, it)); ++ord) {
        __syncwarp();
        if (lane == 0) item_done(ord);
        int have = -1;  // page ids [have, have + kPageSlots) of the sequence are in shared memory
#pragma unroll 1
        for (int j = 0; j < it.n && ok; ++j) {
          const int k0 = (it.t0 + j) * 128;
          uint8_t* dst = tiles + st * L::kTile;
          if constexpr (TREE) {
            const int k1 = min(k0 + 128, it.keys);
            const int pg0 = k0 >> p.block_log2, pg1 = (k1 - 1) >> p.block_log2;
            if (have < 0 || pg1 >= have + static_cast<int>(L::kPageSlots)) {
              have = pg0;
              const int bt0 = p.bt_off[it.s], bt_n = table_entries(p, it.s);
              const int last = min(have + static_cast<int>(L::kPageSlots),
                                   ((it.keys - 1) >> p.block_log2) + 1);
              __syncwarp();
#pragma unroll 1
              for (int i = have + lane; i < last; i += 32) {
                const int page = i < bt_n ? p.bt[bt0 + i] : -1;
                // Pages outside the pool or the table are reported and not
                // loaded: every access stays inside the pool, and what the
                // sequence's rows get is undefined.
                const bool good = page >= 0 && page < p.num_pages;
                if (!good) atomicOr(p.status, kDevBadInput);
                page_ids[i - have] = good ? page : -1;
              }
              __syncwarp();
            }
            // lane i issues the boxes of the tile's i-th page
            const int segs = p.block_log2 >= 7 ? 1 : (k1 - k0 + p.box_rows - 1) >> p.block_log2;
            const int tok = k0 + lane * p.box_rows;
            const int page = lane < segs ? page_ids[(tok >> p.block_log2) - have] : -1;
            const uint32_t boxes = __popc(__ballot_sync(0xffffffffu, page >= 0));
            bool got = true;
            if (lane == 0) {
              got = row_wait(&empty[st], phase, abort_flag);
              if (got) mbar_arrive_expect_tx(&full[st], boxes * p.box_rows * (D * 2u));
            }
            ok = __shfl_sync(0xffffffffu, got, 0);
            if (!ok) break;
            if (page >= 0) {
              const int row = static_cast<int>(page * p.page_rows + p.layer * p.layer_rows +
                                               kv * p.kv_rows + (tok & (p.block_size - 1)));
              dst += lane * p.box_rows * 128u;
#pragma unroll
              for (int h = 0; h < L::kHalves; ++h)
                tma_load_2d(dst + h * L::kHalf, map, &full[st], it.kh * D + h * 64, row);
            }
          } else if (lane == 0) {
            if (!row_wait(&empty[st], phase, abort_flag)) {
              ok = false;
              break;
            }
            mbar_arrive_expect_tx(&full[st], L::kTile);
#pragma unroll
            for (int h = 0; h < L::kHalves; ++h)
              tma_load_2d(dst + h * L::kHalf, map, &full[st], it.kh * D + h * 64, it.key0 + k0);
          }
          if (++st == N) {
            st = 0;
            phase ^= 1;
          }
        }
        // Of prompts only lane 0 waits. When its wait gave up all lanes leave
        // together: the others would be in the next vote without it for ever.
        if constexpr (TREE) __syncwarp();
        else ok = __shfl_sync(0xffffffffu, ok, 0) != 0;
      }
    } else if (warp == 11) {
      if (lane == 0) {
        // ---------------------------------------------- Q producer
        RowItem it;
        uint32_t uses0 = 0, uses1 = 0;
        const uint32_t bytes = L::kHalves * 64u * 2u * p.group * p.tile_tokens;
        bool ok = true;
#pragma unroll 1
        for (uint32_t ord = 0; ok && next_item(ord, it); ++ord) {
          item_done(ord);
#pragma unroll 1
          for (int x = 0; x < 2 && ok; ++x) {
            if (x == 1 && it.n1 == 0) break;
            uint32_t& uses = x ? uses1 : uses0;
            if (!row_wait(&q_empty[x], (uses & 1) ^ 1, abort_flag)) { ok = false; break; }
            ++uses;
            mbar_arrive_expect_tx(&q_full[x], bytes);
            for (int h = 0; h < L::kHalves; ++h)
              tma_load_3d(smem + L::kOffQ + x * L::kTile + h * L::kHalf, &tmQ, &q_full[x],
                          h * 64, it.kh * p.group, it.row0 + x * p.tile_tokens);
          }
        }
      }
    } else if (warp == 12) {
      // ------------------------------------------------ value tiles
      RowItem it;
      uint32_t c = 0;
      bool ok = true;
#pragma unroll 1
      for (uint32_t ord = 0; ok && __all_sync(0xffffffffu, next_item(ord, it)); ++ord) {
        const int dirty = first_dirty<TREE>(it);
        unsigned any = 0;
        unsigned* bad = bad_words + (ord % kRowItems) * kRowBadWords;
#pragma unroll 1
        for (int j = 0; j < it.n; ++j, ++c) {
          const uint32_t st = c % NV;
          const bool in = row_wait(&v_full[st], (c / NV) & 1, abort_flag);
          if (!__all_sync(0xffffffffu, in)) { ok = false; break; }
          if (j >= dirty) {
            uint8_t* tile = smem + L::kOffV + st * L::kTile;
#pragma unroll 1
            for (int q = 0; q < 4; ++q) {
              const int r = q * 32 + lane;
              const int key = (it.t0 + j) * 128 + r;
              bool found = false;
#pragma unroll 1
              for (int h = 0; h < L::kHalves; ++h) {
                uint8_t* row = tile + h * L::kHalf + r * 128;
                if (key >= it.keys) {
#pragma unroll 1
                  for (int ch = 0; ch < 8; ++ch)
                    *reinterpret_cast<uint4*>(row + ((ch ^ (r & 7)) << 4)) =
                        make_uint4(0, 0, 0, 0);
                } else {
                  // the largest magnitude of the half row, two values at a time
                  unsigned top = 0;
#pragma unroll
                  for (int ch = 0; ch < 8; ++ch) {
                    const uint4 w = *reinterpret_cast<const uint4*>(row + ((ch ^ (r & 7)) << 4));
                    top = __vmaxu2(top, __vmaxu2(__vmaxu2(w.x & 0x7FFF7FFFu, w.y & 0x7FFF7FFFu),
                                                 __vmaxu2(w.z & 0x7FFF7FFFu, w.w & 0x7FFF7FFFu)));
                  }
                  constexpr unsigned inf = F16 ? 0x7C00u : 0x7F80u;
                  if ((top & 0xFFFFu) >= inf || (top >> 16) >= inf) {
                    found = true;
                    uint16_t* e = reinterpret_cast<uint16_t*>(row);
#pragma unroll 1
                    for (int i = 0; i < 64; ++i)
                      if (nonfinite16<F16>(e[i])) e[i] = 0;
                  }
                }
              }
              const unsigned word = __ballot_sync(0xffffffffu, found);
              any |= word;
              if (lane == 0 && j - dirty < kRowMaxDirty) bad[(j - dirty) * 4 + q] = word;
            }
            fence_async_smem();
          }
          __syncwarp();
          if (lane == 0) st_release_cta(v_count, c + 1);
        }
        if (!ok) break;
        __syncwarp();
        if (lane == 0) {
          bad[kRowMaxDirty * 4] = any;
          mbar_arrive(&looked[ord % kRowItems]);
          item_done(ord);
        }
      }
    } else if (warp == 13) {
      if (lane == 0) {
        // ---------------------------------------------- items
        Items items;
        RowItem it;
#pragma unroll 1
        for (uint32_t ord = 0;; ++ord) {
          const uint32_t slot = ord % kRowItems;
          if (!row_wait(&it_empty[slot], ((ord / kRowItems) & 1) ^ 1, abort_flag)) break;
          const bool more = items.next(p, tab, it);
          if constexpr (TREE) {
            if (!p.whole && ord == 0) p.ws_join[blockIdx.x] = RowJoin{};  // none so far
            if (more && it.part >= 0 && it.t0 == 0) {
              const int end = items.pos - it.n + ((it.keys + 127) >> 7);
              p.ws_join[blockIdx.x] = {it.row0, it.kh, it.ntok0, it.ntok1, it.part,
                                       (end - 1) / items.share, it.s, it.tok0};
            }
          }
          if (!more) it.n = 0;
          ring[slot] = it;
          mbar_arrive(&it_full[slot]);
          if (!more) break;
        }
      }
    } else if (warp < 10 && lane == 0) {
      // ------------------------------------------------ MMA issuer
      constexpr uint32_t kIdescQK = row_idesc<F16>(128, 0);
      constexpr uint32_t kIdescPV = row_idesc<F16>(D, 1);
      const int x = warp - 8;
      const uint32_t tS = tmem + x * 128, tO = tmem + L::kColO + x * D;
      const uint32_t tP = tmem + L::kColP + x * L::kStepP;
      RowItem it;
      uint32_t base = 0;          // key tiles of the items before
      uint32_t ord0 = 0, ord1 = 0;  // items before; those with a Q tile 1
      uint32_t tiles = 0, mine = 0;  // tiles and items of the stream before
      bool ok = true;
#pragma unroll 1
      for (; ok && next_item(ord0, it); base += it.n, ++ord0, ord1 += it.n1 > 0) {
        item_done(ord0);
        const int cnt = it.count(x);
        const int qt = it.alt ? 0 : x;
        // Both streams look at Q tile 0 of every item, and both give it back:
        // neither can be a phase of any barrier ahead of the other's items.
        if (!row_wait(&q_full[0], ord0 & 1, abort_flag)) break;
        if (x == 1 && !it.alt) mbar_arrive(&q_empty[0]);
        const uint64_t q_desc = sdesc_sw128(smem_u32(smem + L::kOffQ + qt * L::kTile), 0, 1024);
        auto k_ready = [&](int i) {
          const uint32_t g = base + it.tile(x, i);
          return mbar_test(&k_full[g % NK], (g / NK) & 1);
        };
        // K of the stream's i-th tile (and its Q tile) are in shared memory.
        auto wait_k = [&](int i) {
          const uint32_t g = base + it.tile(x, i);
          return (i > 0 || !qt || row_wait(&q_full[1], ord1 & 1, abort_flag)) &&
                 row_wait(&k_full[g % NK], (g / NK) & 1, abort_flag);
        };
        if (cnt == 0) continue;
        const bool locked = L::kLock && it.n >= L::kLockTiles;
        // Step i issues P V of tile i - 1 and S of tile i together: the streams'
        // products then follow one another, and one's softmax runs under the
        // other's products, instead of both at half speed side by side. Only
        // when K of tile i is not there yet, P V goes ahead alone.
        bool held = false, ahead = false;
#pragma unroll 1
        for (int i = 0; i <= cnt; ++i) {
          // Products of step i: with P in its own columns S of tile i, as soon as
          // the scores of tile i - 1 have been read, then P V of tile i - 1; with P
          // over S first P V, then S. `ahead`: S of tile i has gone out already.
          auto issue_s = [&]() {
            const int j = it.tile(x, i);
            const uint32_t st = (base + j) % NK;
            const uint64_t k_desc = sdesc_sw128(smem_u32(smem + L::kOffK + st * L::kTile), 0, 1024);
#pragma unroll
            for (int kk = 0; kk < D / 16; ++kk) {
              const uint32_t off = ((kk >> 2) * L::kHalf + (kk & 3) * 32) >> 4;
              mma_f16_ss(tS, q_desc + off, k_desc + off, kIdescQK, kk > 0);
            }
            mma_commit(&s_full[x]);
            // Two arrivals free a slot: one of each stream, or both of its only one.
            mma_commit(&k_empty[st]);
            if (!it.shared(j)) mma_commit(&k_empty[st]);
            if (i == cnt - 1) mma_commit(&q_empty[qt]);
          };
          ahead = false;
          if (i > 0) {
            const int j = it.tile(x, i - 1);
            const uint32_t st = (base + j) % NV;
            if (L::kOwnP && i < cnt) {
              if (!row_wait(&s_read[x], tiles & 1, abort_flag)) { ok = false; break; }
              if (k_ready(i)) {
                tc_fence_after();
                issue_s();
                ahead = true;
              }
            }
            if (!count_wait(v_count, base + j + 1, abort_flag) ||
                (i == 1 && !row_wait(&o_free[x], (mine & 1) ^ 1, abort_flag)) ||
                !row_wait(&p_full[x], tiles & 1, abort_flag)) {
              ok = false;
              break;
            }
            ++tiles;
            const bool both = !L::kOwnP && i < cnt && k_ready(i);
            if (locked && !lock_take(mma_lock, abort_flag)) { ok = false; break; }
            held = true;
            tc_fence_after();
            const uint64_t v_desc =
                sdesc_sw128(smem_u32(smem + L::kOffV + st * L::kTile), L::kHalf, 1024);
#pragma unroll
            for (int kk = 0; kk < 8; ++kk)
              mma_f16_ts(tO, tP + kk * 8, v_desc + kk * (2048 >> 4), kIdescPV,
                         (i > 1 || kk > 0) ? 1u : 0u);
            mma_commit(&v_empty[st]);
            if (!it.shared(j)) mma_commit(&v_empty[st]);
            if (L::kOwnP) mma_commit(&pv_done[x]);
            if (i == cnt) mma_commit(&o_full[x]);
            if (!both) {
              if (locked) st_release_cta(mma_lock, 0);
              held = false;
            }
          }
          if (i < cnt && !ahead) {
            if (!held) {
              if (!wait_k(i) || (locked && !lock_take(mma_lock, abort_flag))) {
                ok = false;
                break;
              }
              tc_fence_after();
            }
            issue_s();
            if (locked) st_release_cta(mma_lock, 0);
            held = false;
          }
        }
        ++mine;
      }
      // Every MMA issued above must finish before TMEM is released.
      mma_commit(&drain[x]);
      volatile int local_abort = 0;
      row_wait(&drain[x], 0, &local_abort);
    }
  } else {
    // ------------------------------------------------ softmax / epilogue
    reg_take<kRowSoftmaxRegs>();
    const int x = warp >> 2;
    const int quarter = warp & 3;               // TMEM lane quarter
    const int r = quarter * 32 + lane;          // row of the Q tile
    const uint32_t lanes = static_cast<uint32_t>(quarter * 32) << 16;
    const uint32_t tS = tmem + x * 128 + lanes, tO = tmem + L::kColO + x * D + lanes;
    const uint32_t tP = tmem + L::kColP + x * L::kStepP + lanes;
    const float sl2 = p.scale_log2;
    const int r_tok = r / p.group, r_head = r - r_tok * p.group;
    RowItem it;
    uint32_t tiles = 0, mine = 0, act1 = 0, alts = 0, ord = 0;
    bool ok = true;
#pragma unroll 1
    for (; ok && __all_sync(0xffffffffu, next_item(ord, it)); ++ord) {
      const int cnt = it.count(x);
      if (cnt == 0) {
        __syncwarp();
        if (lane == 0) item_done(ord);
        continue;
      }
      const int q_tile = it.alt ? 0 : x;
      const int token = it.tok0 + q_tile * p.tile_tokens + r_tok;   // in its sequence
      const unsigned* mask = nullptr;
      if constexpr (TREE)  // rows past the tree's end read the last node's mask
        mask = p.mask + static_cast<long long>(p.q_off[it.s] + min(token, it.nodes - 1)) * p.words;
      const bool counts = r_tok < (q_tile ? it.ntok1 : it.ntok0) && r_tok < p.tile_tokens;
      float m = -INFINITY, msl = 0.f;
      float2 l2[2] = {make_float2(0.f, 0.f), make_float2(0.f, 0.f)};
#pragma unroll 1
      for (int i = 0; i < cnt; ++i) {
        const bool ready = row_wait(&s_full[x], tiles & 1, abort_flag);
        ++tiles;
        if (!__all_sync(0xffffffffu, ready)) { ok = false; break; }
        tc_fence_after();
        float s[128];
#pragma unroll
        for (int c4 = 0; c4 < 4; ++c4)
          tmem_ld32(tS + c4 * 32, *reinterpret_cast<uint32_t(*)[32]>(&s[c4 * 32]));
        tmem_wait_ld();
        if (L::kOwnP) {
          tc_fence_before();
          mbar_arrive(&s_read[x]);
        }
        const int k0 = (it.t0 + it.tile(x, i)) * 128;
        const bool masked = TREE ? k0 + 128 > it.ctx
                                 : k0 + 127 > it.tok0 + q_tile * p.tile_tokens;
        if (masked) {
#pragma unroll
          for (int c4 = 0; c4 < 4; ++c4) {
            unsigned bits;  // the keys the row sees
            if constexpr (TREE) {
              bits = tree_bits(mask, p.words, it.nodes, k0 + c4 * 32 - it.ctx);
            } else {
              const int lim = token - k0 - c4 * 32;
              bits = lim < 0 ? 0u : lim > 30 ? 0xffffffffu : (2u << lim) - 1u;
            }
#pragma unroll
            for (int c = 0; c < 32; ++c)
              if (!(bits & (1u << c))) s[c4 * 32 + c] = -INFINITY;
          }
        }
        // Row max as four chains (max is exact in any order), two values a step.
        float mx[4] = {s[0], s[1], s[2], s[3]};
#pragma unroll
        for (int c = 4; c < 124; c += 8)
#pragma unroll
          for (int u = 0; u < 4; ++u) mx[u] = max3(mx[u], s[c + u], s[c + 4 + u]);
#pragma unroll
        for (int u = 0; u < 4; ++u) mx[u] = max2(mx[u], s[124 + u]);
        const float mt = max2(max3(mx[0], mx[1], mx[2]), mx[3]);
        if (L::kOwnP && tiles > 1) {  // the tile before has left P and reached O
          const bool free = row_wait(&pv_done[x], tiles & 1, abort_flag);
          if (!__all_sync(0xffffffffu, free)) { ok = false; break; }
          tc_fence_after();
        }
        if (i == 0) {
          m = mt;
          msl = m == -INFINITY ? 0.f : m * sl2;
        } else if (__any_sync(0xffffffffu, counts && !((mt - m) * sl2 <= kRowRescale))) {
          // (rows of no token take no part in the vote: what they hold, and with it
          // the roundings of the rows beside them, would differ from call to call)
          const float mn = max2(m, mt);
          const float nsl = mn == -INFINITY ? 0.f : mn * sl2;
          const float alpha = m == -INFINITY ? 0.f : ex2_approx(msl - nsl);
#pragma unroll 1
          for (int c = 0; c < D; c += 16) {
            uint32_t u[16];
            tmem_ld16(tO + c, u);
            tmem_wait_ld();
#pragma unroll
            for (int q = 0; q < 16; ++q)
              u[q] = __float_as_uint(__uint_as_float(u[q]) * alpha);
            tmem_st16(tO + c, u);
          }
          l2[0].x *= alpha; l2[0].y *= alpha; l2[1].x *= alpha; l2[1].y *= alpha;
          m = mn;
          msl = nsl;
        }
        // P = 2^(s scale - m), two at a time, rounded to the input type for the
        // product with V; l sums the unrounded values.
        const float2 sc = make_float2(sl2, sl2), neg = make_float2(-msl, -msl);
#pragma unroll
        for (int c4 = 0; c4 < 4; ++c4) {
          uint32_t u[16];
#pragma unroll
          for (int c = 0; c < 16; ++c) {
            float2 e = __ffma2_rn(make_float2(s[c4 * 32 + 2 * c], s[c4 * 32 + 2 * c + 1]), sc, neg);
            e.x = ex2_approx(e.x);
            e.y = ex2_approx(e.y);
            l2[c & 1] = __fadd2_rn(l2[c & 1], e);
            u[c] = pack16<F16>(e.x, e.y);
          }
          tmem_st16(tP + c4 * 16, u);
        }
        tmem_wait_st();
        tc_fence_before();
        mbar_arrive(&p_full[x]);
      }
      if (!ok) break;
      float l = (l2[0].x + l2[0].y) + (l2[1].x + l2[1].y);
      if (it.alt && x == 1) {
        alt_buf[(alts & 1) * 128 + r] = make_float2(m == -INFINITY ? m : msl, l);
        mbar_arrive(&alt_ml[alts & 1]);
        __syncwarp();
        if (lane == 0) item_done(ord);
        ++alts;
        ++mine;
        continue;
      }
      // ---- epilogue
      bool fin = row_wait(&o_full[x], mine & 1, abort_flag);
      float a0 = 1.f, a1 = 0.f;                  // weights of the two streams' O
      float ml = m == -INFINITY ? m : msl;       // running max, log2 units
      if (it.alt) {
        // (stream 1's statistics first: by then its earlier items are through)
        fin = fin && row_wait(&alt_ml[alts & 1], (alts >> 1) & 1, abort_flag) &&
              row_wait(&o_full[1], act1 & 1, abort_flag);
        if (__all_sync(0xffffffffu, fin)) {
          const float2 o = alt_buf[(alts & 1) * 128 + r];
          const float mm = max2(ml, o.x);
          // a stream that saw nothing has m = -inf and O = 0
          a0 = ml == -INFINITY ? (mm == -INFINITY ? 1.f : 0.f) : ex2_approx(ml - mm);
          a1 = o.x == -INFINITY ? 0.f : ex2_approx(o.x - mm);
          l = l * a0 + o.y * a1;
          ml = mm;
        }
        ++alts;
      }
      fin = fin && row_wait(&looked[ord % kRowItems], (ord / kRowItems) & 1, abort_flag);
      if (!__all_sync(0xffffffffu, fin)) { ok = false; break; }
      ++mine;
      act1 += it.count(1) > 0;
      tc_fence_after();
      const int row = it.row0 + q_tile * p.tile_tokens + r_tok;
      const int head = it.kh * p.group + r_head;
      // Values that are not finite, of keys this row sees (words of the item's
      // dirty tiles; all zero but for broken inputs).
      const unsigned* bad = bad_words + (ord % kRowItems) * kRowBadWords;
      const int dirty = first_dirty<TREE>(it);
      const int bad_n = min(max(it.n - dirty, 0), kRowMaxDirty) * 4;
      const unsigned any_bad = bad[kRowMaxDirty * 4];
      float inv = 1.0f;
      uint8_t* stage = smem + L::kOffOut + warp * 2048;
      unsigned long long dst = 0;  // where the row goes
      if (counts)
        dst = it.part >= 0
                  ? reinterpret_cast<unsigned long long>(
                        p.ws_o + (static_cast<long long>(it.part) * 256 + q_tile * 128 + r) * 128)
                  : reinterpret_cast<unsigned long long>(
                        static_cast<uint16_t*>(p.out) + row * p.ldo +
                        static_cast<long long>(head) * D);
      // the pieces this lane stores: 16 bytes of the rows lane / 4 + 8 k
      unsigned long long to[4];
#pragma unroll
      for (int k = 0; k < 4; ++k) {
        to[k] = __shfl_sync(0xffffffffu, dst, k * 8 + (lane >> 2));
        if (to[k] != 0) to[k] += (lane & 3) * 16;
      }
      if (it.part < 0) {
        inv = 1.0f / l;
        if constexpr (TREE) {
          if (l == 0.f) {  // a row that sees no key at all is zero
            bool sees = it.ctx > 0;
#pragma unroll 1
            for (int w = 0; w < p.words && !sees; ++w)
              sees = tree_bits(mask, p.words, it.nodes, w * 32) != 0;
            if (!sees) inv = 0.f;
          }
        }
      }
#pragma unroll 1
      for (int c4 = 0; c4 < D / 32; ++c4) {
        uint32_t u[32];
        tmem_ld32(tO + c4 * 32, u);
        tmem_wait_ld();
        float o[32];
#pragma unroll
        for (int q = 0; q < 32; ++q) o[q] = __uint_as_float(u[q]);
        if (it.alt) {
          tmem_ld32(tO + D + c4 * 32, u);
          tmem_wait_ld();
#pragma unroll
          for (int q = 0; q < 32; ++q) o[q] = o[q] * a0 + __uint_as_float(u[q]) * a1;
        }
        // 64 bytes of a row per lane, turned in shared memory so that four lanes
        // store each row's piece together (a row per lane would touch 32 lines
        // with every store).
        auto put = [&](const uint32_t (&w)[16], int at) {
          __syncwarp();
#pragma unroll
          for (int c = 0; c < 4; ++c)
            *reinterpret_cast<uint4*>(stage + lane * 64 + ((c ^ (lane >> 1 & 3)) << 4)) =
                make_uint4(w[4 * c], w[4 * c + 1], w[4 * c + 2], w[4 * c + 3]);
          __syncwarp();
          uint4 v[4];
#pragma unroll
          for (int k = 0; k < 4; ++k) {
            const int from = k * 8 + (lane >> 2);
            v[k] = *reinterpret_cast<const uint4*>(
                stage + from * 64 + (((lane & 3) ^ (from >> 1 & 3)) << 4));
          }
#pragma unroll
          for (int k = 0; k < 4; ++k) st_global_if(to[k] != 0, to[k] + at, v[k]);
        };
        if (TREE && it.part >= 0) {
#pragma unroll
          for (int h = 0; h < 2; ++h) {
            uint32_t w[16];
#pragma unroll
            for (int q = 0; q < 16; ++q) w[q] = __float_as_uint(o[h * 16 + q]);
            put(w, c4 * 128 + h * 64);
          }
        } else {
          uint32_t w[16];
#pragma unroll
          for (int q = 0; q < 16; ++q) w[q] = pack16<F16>(o[2 * q] * inv, o[2 * q + 1] * inv);
          put(w, c4 * 64);
        }
      }
      if (any_bad != 0) {
        // After the row's own stores: finite + infinity is infinity, and NaN
        // and opposite infinities come out as they should.
        __syncwarp();
#pragma unroll 1
        for (int w = 0; counts && w < bad_n; ++w) {
#pragma unroll 1
          for (unsigned b = bad[w]; b != 0; b &= b - 1) {
            const int k = (it.t0 + dirty) * 128 + w * 32 + __ffs(b) - 1;
            const uint16_t* vr = value_row<TREE>(p, it, D, k);
            if (vr == nullptr || !row_sees<TREE>(it, mask, p.words, token, k)) continue;
#pragma unroll 1
            for (int d = 0; d < D; ++d) {
              if (!nonfinite16<F16>(vr[d])) continue;
              const float add = widen16<F16>(vr[d]);
              if (it.part >= 0) {
                reinterpret_cast<float*>(dst)[d] += add;
              } else {
                uint16_t* e = reinterpret_cast<uint16_t*>(dst) + d;
                *e = static_cast<uint16_t>(pack16<F16>(widen16<F16>(*e) + add, 0.f));
              }
            }
          }
        }
      }
      if (it.part >= 0 && counts)
        reinterpret_cast<float2*>(p.ws_ml)[static_cast<long long>(it.part) * 256 + q_tile * 128 +
                                           r] = make_float2(ml, l);
      tc_fence_before();
      mbar_arrive(&o_free[x]);
      if (it.alt) mbar_arrive(&o_free[1]);
      __syncwarp();
      if (lane == 0) item_done(ord);
    }
  }

  __syncthreads();
  if (*abort_flag) {
    // Let copies already in flight land before the CTA exits.
    const uint64_t t0 = globaltimer_ns();
    while (globaltimer_ns() - t0 < 1000000ull) __nanosleep(1000);
    if (threadIdx.x == 0) atomicOr(p.status, kDevWaitTimeout);
  }
  if (warp == 8) {
    __syncwarp();
    tc_fence_after();
    tmem_dealloc(tmem, 512);
  }
}

// Before a kernel's first launch on a device: its shared memory, and that it
// was built with the registers its warps hand over to one another (setmaxnreg
// draws on those of the launch, and a share that is not there is waited for
// without end). `ready` is the kernel's own flag word, a bit per device.
template <typename Kern>
int row_kernel_ready(Kern* kern, size_t smem, std::atomic<uint64_t>& ready) {
  int dev = 0;
  KVM_CUDA_TRY(cudaGetDevice(&dev));
  const uint64_t bit = 1ull << (dev & 63);
  if (ready.load(std::memory_order_acquire) & bit) return KVM_OK;
  cudaFuncAttributes a;
  KVM_CUDA_TRY(cudaFuncGetAttributes(&a, kern));
  if (a.numRegs * kRowThreads < 256 * kRowSoftmaxRegs + 256 * kRowControlRegs)
    return fail(KVM_ERR_UNSUPPORTED, "attention kernel built with too few registers");
  KVM_CUDA_TRY(cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, int(smem)));
  ready.fetch_or(bit, std::memory_order_release);
  return KVM_OK;
}

}  // namespace kvm
