// Upkeep of a paged KV pool on the device, all layers, K and V in one launch:
// page copies (a fork's own copy of its parent's last page, pages moved
// towards the front of the pool) and the compaction of a drafted tree's
// accepted tokens to consecutive slots. Both read kernel.kvcache's pool
// (src/ir/dialect/kernel/dialect.cpp:69-70, src/ir/graph_config.h:20-39).
//
// Both only move bytes. Copies are bound by HBM: 96 pages of 2 MB in 67-69 us
// (5.9 TB/s) from 96 sources, in 63-64 us from 64 of them that repeat (5.3 TB/s
// of what has to be read and written). Compaction is bound by the launch and by
// reads that wait for one another, the lists, the tables and the rows (48
// sequences of up to eight kept tokens, 24 layers: 10.4-10.8 us for 5.8 us of
// bytes). Neither decides anything by the order in which blocks run.
#include "kv_layout.h"
#include "runtime.h"

namespace kvm {
namespace {

constexpr int kCopyThreads = 256;
constexpr int kCopyVecs = 8;                           // 16-byte vectors per thread
constexpr int kCopyChunk = kCopyThreads * kCopyVecs;   // vectors (32 KB) per step of a block

// A page as nested runs of 16-byte vectors, contiguous dimensions merged:
// vector v lies at (v / inner / n1) * s2 + (v / inner % n1) * s1 + v % inner
// from the page's start.
struct PageRuns {
  long long page;       // vectors between pages
  long long s1, s2;
  unsigned inner, n1;
  unsigned total;       // vectors of a page
};

__device__ __forceinline__ long long run_offset(const PageRuns& r, unsigned v) {
  const unsigned run = v / r.inner;
  return (run / r.n1) * r.s2 + (run % r.n1) * r.s1 + (v - run * r.inner);
}

// A block takes consecutive steps of (pair, chunk); on a new pair it looks
// through the lists, so that a pair whose destination is out of range, is
// written by another pair or is read by another one is skipped and reported,
// and the result never depends on which block ran first.
__global__ void __launch_bounds__(kCopyThreads)
    copy_pages_kernel(uint4* __restrict__ pool, const __grid_constant__ PageRuns r,
                      const int* __restrict__ src, const int* __restrict__ dst, int n,
                      int num_pages, int chunks, long long steps, int* status) {
  pdl_wait();
  pdl_trigger();
  const long long per = (steps + gridDim.x - 1) / gridDim.x;
  const long long begin = blockIdx.x * per, end = min(begin + per, steps);
  int pair = -1;
  bool ok = false;
  const uint4* from = nullptr;
  uint4* to = nullptr;
  for (long long w = begin; w < end; ++w) {
    const int i = static_cast<int>(w / chunks);
    if (i != pair) {
      pair = i;
      const int a = src[i], b = dst[i];
      bool bad = a < 0 || a >= num_pages || b < 0 || b >= num_pages;
      for (int j = threadIdx.x; j < n; j += kCopyThreads)
        if (j != i && (dst[j] == b || (src[j] == b && a != b))) bad = true;
      bad = __syncthreads_or(bad);
      if (bad && threadIdx.x == 0) atomicOr(status, kDevBadInput);
      ok = !bad && a != b;
      from = pool + a * r.page;
      to = pool + b * r.page;
    }
    if (!ok) continue;
    const unsigned v0 = static_cast<unsigned>(w - static_cast<long long>(i) * chunks) * kCopyChunk +
                        threadIdx.x;
    uint4 x[kCopyVecs];
    long long at[kCopyVecs];
#pragma unroll
    for (int u = 0; u < kCopyVecs; ++u) {
      const unsigned v = v0 + u * kCopyThreads;
      if (v < r.total) {
        at[u] = run_offset(r, v);
        x[u] = from[at[u]];
      }
    }
#pragma unroll
    for (int u = 0; u < kCopyVecs; ++u)
      if (v0 + u * kCopyThreads < r.total) to[at[u]] = x[u];
  }
}

constexpr int kCompactThreads = 128;
constexpr int kCompactBatch = 64;   // kept tokens whose addresses are held at a time
constexpr int kCompactFly = 8;      // rows in flight per thread

// One block per (sequence, layer, K or V). A thread owns 16-byte columns of
// the row and walks the kept tokens in order, eight loads ahead of their
// stores: with kept strictly increasing, slot i is never the source of a
// token after the i-th, so moving in place in this order is safe.
__global__ void __launch_bounds__(kCompactThreads)
    compact_kernel(uint4* __restrict__ pool, const __grid_constant__ kvm_kv_layout L,
                   int layers, const int* __restrict__ kept, int n_kept,
                   const int* __restrict__ kept_off, const int* __restrict__ q_pos,
                   const int* __restrict__ bt, int table_len, const int* __restrict__ bt_off,
                   int* status) {
  __shared__ long long from[kCompactBatch], to[kCompactBatch];
  pdl_wait();
  pdl_trigger();
  const int unit = blockIdx.x;
  const int kv = unit & 1, layer = L.layer + (unit >> 1) % layers, s = (unit >> 1) / layers;
  const int k0 = kept_off[s], m = kept_off[s + 1] - k0;
  if (m == 0) return;
  if (k0 < 0 || m < 0 || m > n_kept - k0) {
    if (threadIdx.x == 0) atomicOr(status, kDevBadInput);
    return;
  }
  const int p0 = q_pos[s], b0 = bt_off[s], b1 = bt_off[s + 1];
  const long long slots =
      b0 < 0 || b1 > table_len ? 0 : (static_cast<long long>(b1) - b0) * L.block_size;
  // page of a position, or -1
  auto page_of = [&](long long pos) {
    if (pos < 0 || pos >= slots) return -1;
    const int pg = bt[b0 + pos / L.block_size];
    return pg >= 0 && pg < L.num_pages ? pg : -1;
  };
  bool bad = p0 < 0;
  for (int i = threadIdx.x; i < m && !bad; i += kCompactThreads) {
    const int j = kept[k0 + i];
    bad = j < i || (i > 0 && j <= kept[k0 + i - 1]) || page_of(p0 + static_cast<long long>(j)) < 0 ||
          page_of(p0 + static_cast<long long>(i)) < 0;
  }
  if (__syncthreads_or(bad)) {   // the sequence stays as it is
    if (threadIdx.x == 0) atomicOr(status, kDevBadInput);
    return;
  }
  const int vecs = L.width / 8;
  const long long base = (layer * L.layer_stride + kv * L.kv_stride) / 8;
  auto place = [&](long long pos) {
    return base + (page_of(pos) * L.page_stride + pos % L.block_size * L.token_stride) / 8;
  };
  for (int i0 = 0; i0 < m; i0 += kCompactBatch) {
    const int nb = min(kCompactBatch, m - i0);
    __syncthreads();
    for (int i = threadIdx.x; i < nb; i += kCompactThreads) {
      from[i] = place(p0 + static_cast<long long>(kept[k0 + i0 + i]));
      to[i] = place(p0 + static_cast<long long>(i0 + i));
    }
    __syncthreads();
    for (int c = threadIdx.x; c < vecs; c += kCompactThreads) {
      for (int i = 0; i < nb; i += kCompactFly) {
        uint4 x[kCompactFly];
#pragma unroll
        for (int u = 0; u < kCompactFly; ++u)
          if (i + u < nb && from[i + u] != to[i + u]) x[u] = pool[from[i + u] + c];
#pragma unroll
        for (int u = 0; u < kCompactFly; ++u)
          if (i + u < nb && from[i + u] != to[i + u]) pool[to[i + u] + c] = x[u];
      }
    }
  }
}

}  // namespace
}  // namespace kvm

using namespace kvm;

extern "C" int kvm_sm100_kvcache_copy_pages(void* cache, const kvm_kv_layout* L, int layers,
                                            const int32_t* src, const int32_t* dst, int n,
                                            kvm_stream_t stream) {
  if (int rc = check_kv_layout(L)) return rc;
  if (layers <= 0 || n < 0 || !cache || !aligned16(cache))
    return fail(KVM_ERR_INVALID_ARG, "kvcache_copy_pages: bad argument");
  if (n == 0) return KVM_OK;
  if (!src || !dst) return fail(KVM_ERR_INVALID_ARG, "kvcache_copy_pages: bad argument");
  const long long total = static_cast<long long>(layers) * 2 * L->block_size * (L->width / 8);
  if (total >= (1ll << 31))
    return fail(KVM_ERR_UNSUPPORTED, "kvcache_copy_pages: a page of 32 GB or more");
  const DeviceInfo* dev = device_info();
  if (!dev) return KVM_ERR_CUDA;
  // (layer, kv, slot, vector), innermost dimensions merged while contiguous
  PageRuns r{};
  const long long ts = L->token_stride / 8, ks = L->kv_stride / 8, ls = L->layer_stride / 8;
  const unsigned w8 = L->width / 8, bs = L->block_size;
  r.page = L->page_stride / 8;
  r.total = static_cast<unsigned>(total);
  const bool slots = ts == w8;                        // a page's slots are one run
  const bool kvs = slots && ks == static_cast<long long>(bs) * w8;
  const bool all = kvs && ls == 2ll * bs * w8;
  if (all) {
    r.inner = r.total; r.n1 = 1;
  } else if (kvs) {
    r.inner = 2 * bs * w8; r.n1 = 1; r.s2 = ls;
  } else if (slots) {
    r.inner = bs * w8; r.n1 = 2; r.s1 = ks; r.s2 = ls;
  } else {
    return fail(KVM_ERR_UNSUPPORTED,
                "kvcache_copy_pages: token_stride must equal width");
  }
  uint4* base = static_cast<uint4*>(cache) + L->layer * ls;
  const int chunks = static_cast<int>((total + kCopyChunk - 1) / kCopyChunk);
  const long long steps = static_cast<long long>(n) * chunks;
  const long long most = dev->sm_count * 8ll;
  const int grid = static_cast<int>(steps < most ? steps : most);
  KVM_CUDA_TRY(launch_ex(true, copy_pages_kernel, dim3(grid), dim3(kCopyThreads), 0,
                         static_cast<cudaStream_t>(stream), base, r, src, dst, n, L->num_pages,
                         chunks, steps, dev->status));
  return KVM_OK;
}

extern "C" int kvm_sm100_kvcache_compact(void* cache, const kvm_kv_layout* L, int layers,
                                         const int32_t* kept, int n_kept,
                                         const int32_t* kept_offsets,
                                         const int32_t* q_positions,
                                         const int32_t* block_table, int table_len,
                                         const int32_t* bt_offsets, int S,
                                         kvm_stream_t stream) {
  if (int rc = check_kv_layout(L)) return rc;
  if (layers <= 0 || S < 0 || n_kept < 0 || table_len < 0 || !cache || !aligned16(cache))
    return fail(KVM_ERR_INVALID_ARG, "kvcache_compact: bad argument");
  if (S == 0 || n_kept == 0) return KVM_OK;
  if (!kept || !kept_offsets || !q_positions || (!block_table && table_len > 0) || !bt_offsets)
    return fail(KVM_ERR_INVALID_ARG, "kvcache_compact: bad argument");
  const long long blocks = 2ll * layers * S;
  if (blocks >= (1ll << 31))
    return fail(KVM_ERR_INVALID_ARG, "kvcache_compact: too many sequences and layers");
  const DeviceInfo* dev = device_info();
  if (!dev) return KVM_ERR_CUDA;
  KVM_CUDA_TRY(launch_ex(true, compact_kernel, dim3(static_cast<unsigned>(blocks)),
                         dim3(kCompactThreads), 0, static_cast<cudaStream_t>(stream),
                         static_cast<uint4*>(cache), *L, layers, kept, n_kept, kept_offsets,
                         q_positions, block_table, table_len, bt_offsets, dev->status));
  return KVM_OK;
}
