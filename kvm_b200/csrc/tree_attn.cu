// Attention for a tree of drafted tokens over the paged KV cache: the form of
// kernel.attn.decode (src/ir/dialect/kernel/dialect.cpp:39) whose new rows
// need not be a chain. Row i of a sequence sees the cached tokens before the
// tree and the drafted tokens its mask names. The kernel is row_attn.cuh's;
// this file joins the partial results of items cut between CTAs.
#include <cmath>

#include "kv_layout.h"
#include "row_attn.cuh"

namespace kvm {
namespace {

constexpr int kTreeMaxCtas = 148;   // stretches the key tiles are cut into, at most
constexpr int kJoinThreads = 256;
constexpr int kJoinRows = 32;       // rows of a block of the joining kernel

// One CTA c per stretch and block of rows: if the last item of stretch c goes
// on in the next ones, and began in c, its parts are joined here. Stretch c
// holds its part in slot 2c when the item is its first, else 2c + 1; the
// following ones, which begin inside the item, in slot 2c'. A warp per row:
//   M = max m_c, out = sum O_c 2^(m_c - M) / sum l_c 2^(m_c - M).
__global__ void __launch_bounds__(kJoinThreads)
    tree_join_kernel(const __grid_constant__ RowParams p, int ctas) {
  __shared__ int start[kRowMaxSeqs], total_s;
  RowTables t{start, nullptr, nullptr, &total_s};
  build_tree_tables(p, t, false);
  const int total = total_s, share = tree_share(total, ctas), c = blockIdx.x;
  const long long begin = static_cast<long long>(c) * share;
  const long long end = begin + share;
  // The partial results are the kernel's before this one. (The offsets are not:
  // it has waited for their writers before letting this one start.) No block
  // may leave before: this kernel would then end before that one does.
  pdl_wait();
  pdl_trigger();
  if (end >= total) return;          // nothing goes on after the last stretch
  int lo = 0, hi = p.S - 1;
  while (lo < hi) {
    const int mid = (lo + hi + 1) >> 1;
    if (start[mid] <= end - 1) lo = mid; else hi = mid - 1;
  }
  int nodes, ctx;
  const int tiles = tree_tiles(p, lo, nodes, ctx, false);
  const int item = static_cast<int>(end - 1 - start[lo]) / tiles;
  const long long i0 = start[lo] + static_cast<long long>(item) * tiles, i1 = i0 + tiles;
  if (i1 <= end || i0 < begin) return;
  const int kh = item % p.HKV, tok0 = item / p.HKV * 2 * p.tile_tokens;
  const int last = static_cast<int>((i1 - 1) / share);
  const int slot0 = 2 * c + (i0 == begin ? 0 : 1);
  const int lane = threadIdx.x % 32;
  for (int r = blockIdx.y * kJoinRows + threadIdx.x / 32; r < (blockIdx.y + 1) * kJoinRows;
       r += kJoinThreads / 32) {
    const int q_tile = r >> 7, in_tile = r & 127;
    const int r_tok = in_tile / p.group;
    const int token = tok0 + q_tile * p.tile_tokens + r_tok;
    if (r_tok >= p.tile_tokens || token >= nodes) continue;
    const float2* ml = reinterpret_cast<const float2*>(p.ws_ml);
    float M = ml[slot0 * 256ll + r].x;
    for (int d = c + 1; d <= last; ++d) M = fmaxf(M, ml[2ll * d * 256 + r].x);
    float L = 0.f;
    float4 acc = make_float4(0.f, 0.f, 0.f, 0.f);
    for (int d = c; d <= last; ++d) {
      const long long at = (d == c ? slot0 : 2ll * d) * 256 + r;
      const float2 v = ml[at];
      // a part whose keys the row does not see holds m = -inf and O = 0
      if (v.x == -INFINITY && M > -INFINITY) continue;
      const float f = v.x == M ? 1.f : ex2_approx(v.x - M);
      const float4 o = reinterpret_cast<const float4*>(p.ws_o)[at * 32 + lane];
      L += v.y * f;
      acc.x += o.x * f; acc.y += o.y * f; acc.z += o.z * f; acc.w += o.w * f;
    }
    float inv = 1.0f / L;
    if (L == 0.f) {
      bool sees = ctx > 0;
      const unsigned* mask = p.mask + static_cast<long long>(p.q_off[lo] + token) * p.words;
      for (int w = 0; w < p.words && !sees; ++w) sees = tree_bits(mask, p.words, nodes, w * 32) != 0;
      if (!sees) inv = 0.f;
    }
    const long long row = p.q_off[lo] + token;
    const int head = kh * p.group + in_tile - r_tok * p.group;
    uint2 v;
    v.x = pack16<false>(acc.x * inv, acc.y * inv);
    v.y = pack16<false>(acc.z * inv, acc.w * inv);
    reinterpret_cast<uint2*>(static_cast<uint16_t*>(p.out) + row * p.ldo + head * 128ll)[lane] = v;
  }
}

template <bool ONE>
int launch_tree(const CUtensorMap& tq, const CUtensorMap& tkv, const RowParams& p, int ctas,
                cudaStream_t st) {
  auto kern = row_attn_kernel<128, false, true, ONE>;
  constexpr size_t smem = RowSmem<128, true, ONE>::bytes();
  static std::atomic<uint64_t> ready{0};
  if (int rc = row_kernel_ready(kern, smem, ready)) return rc;
  KVM_CUDA_TRY(launch_ex(true, kern, dim3(ctas), dim3(kRowThreads), smem, st, tq, tkv, tkv, p));
  return KVM_OK;
}

// How a call is cut up, from its bounds alone.
struct TreeCut {
  int64_t ctas;
  bool whole;
};
TreeCut tree_cut(int64_t S, int HKV, int group, int max_q_rows, int max_keys) {
  const int64_t per = 2 * (128 / group);
  const int64_t items = S * HKV * ((max_q_rows + per - 1) / per);
  const int64_t tiles = (int64_t(max_keys) + 127) / 128;
  // Items that fit the CTAs one each, of at most eight key tiles, stay whole:
  // cutting them saves at most half of their few microseconds and costs the
  // joining launch.
  if (items <= kTreeMaxCtas && tiles <= 8) return {items, true};
  const int64_t ctas = (items * tiles + 3) / 4;  // four key tiles each, at least
  return {ctas < kTreeMaxCtas ? ctas : kTreeMaxCtas, false};
}

}  // namespace
}  // namespace kvm

using namespace kvm;

extern "C" int64_t kvm_sm100_attention_tree_workspace(int S, int HQ, int HKV, int max_q_rows,
                                                      int max_keys) {
  if (S <= 0 || HQ <= 0 || HKV <= 0 || HQ % HKV || HQ / HKV > 128 || max_q_rows <= 0 ||
      max_keys <= 0 || max_keys > (1 << 30))
    return 0;
  const TreeCut cut = tree_cut(S, HKV, HQ / HKV, max_q_rows, max_keys);
  return cut.whole ? 0 : cut.ctas * 2 * 256 * (128 + 2) * 4;
}

extern "C" int kvm_sm100_attention_tree_paged(
    const void* q, int64_t ldq, const void* cache, const kvm_kv_layout* L, void* out,
    int64_t ldo, const int32_t* q_offsets, const int32_t* q_positions, const uint32_t* mask,
    int mask_words, const int32_t* block_table, int table_len, const int32_t* bt_offsets, int S,
    int rows,
    int HQ, int max_q_rows, int max_keys, float scale, void* workspace,
    int64_t workspace_bytes, kvm_stream_t stream) {
  if (int rc = check_kv_layout(L)) return rc;
  if (S < 0 || rows < 0 || table_len < 0 || HQ <= 0 || L->width % 128 || HQ % (L->width / 128))
    return fail(KVM_ERR_INVALID_ARG,
                "attention_tree: head_dim 128, width = HKV*128, HQ a multiple of HKV");
  const int HKV = L->width / 128, group = HQ / HKV, bs = L->block_size;
  if (group > 128)
    return fail(KVM_ERR_UNSUPPORTED, "attention_tree: at most 128 query heads per kv head");
  if (S > kRowMaxSeqs)
    return fail(KVM_ERR_UNSUPPORTED, "attention_tree: at most 1024 sequences a call");
  if (bs < 16 || (bs & (bs - 1)) != 0)
    return fail(KVM_ERR_UNSUPPORTED,
                "attention_tree: block_size must be a power of two >= 16");
  if (L->page_stride % L->token_stride || L->layer_stride % L->token_stride ||
      L->kv_stride % L->token_stride)
    return fail(KVM_ERR_INVALID_ARG,
                "attention_tree: page, layer and kv strides must be whole token slots");
  if (!std::isfinite(scale)) return fail(KVM_ERR_INVALID_ARG, "attention_tree: bad scale");
  if (S == 0 || rows == 0) return KVM_OK;
  if (max_q_rows <= 0 || max_q_rows > kRowMaxNodes || max_keys <= 0 || max_keys > (1 << 30))
    return fail(KVM_ERR_INVALID_ARG,
                "attention_tree: max_q_rows 1..1024 and max_keys 1..2^30");
  if (mask_words <= 0 || int64_t(mask_words) * 32 < max_q_rows)
    return fail(KVM_ERR_INVALID_ARG, "attention_tree: the mask holds fewer than max_q_rows bits");
  if (!q || !cache || !out || !q_offsets || !q_positions || !mask || !block_table ||
      !bt_offsets || !aligned16(q) || !aligned16(cache) || !aligned16(out) ||
      ldq < int64_t(HQ) * 128 || ldo < int64_t(HQ) * 128 || ldq % 8 || ldo % 8)
    return fail(KVM_ERR_INVALID_ARG, "attention_tree: bad pointer or row stride");
  const int64_t per = 2 * (128 / group);
  if (int64_t(S) * HKV * ((max_q_rows + per - 1) / per) * ((int64_t(max_keys) + 127) / 128) >=
      (1ll << 30))
    return fail(KVM_ERR_INVALID_ARG, "attention_tree: too large");
  // The pool as rows of token slots: page a, layer l, K or V x, slot i is row
  // a*page_rows + l*layer_rows + x*kv_rows + i.
  const int64_t pool_rows = (int64_t(L->num_pages) - 1) * (L->page_stride / L->token_stride) +
                            int64_t(L->layer) * (L->layer_stride / L->token_stride) + L->kv_stride / L->token_stride + bs;
  if (pool_rows >= (1ll << 31))
    return fail(KVM_ERR_UNSUPPORTED, "attention_tree: pool too large for 32-bit rows");
  const TreeCut cut = tree_cut(S, HKV, group, max_q_rows, max_keys);
  const int64_t ctas = cut.ctas;
  const int64_t need = kvm_sm100_attention_tree_workspace(S, HQ, HKV, max_q_rows, max_keys);
  if (need > 0 && (!workspace || workspace_bytes < need || !aligned16(workspace)))
    return fail(KVM_ERR_INVALID_ARG, "attention_tree: workspace too small");
  const DeviceInfo* dev = device_info();
  if (!dev) return KVM_ERR_CUDA;
  RowParams p{};
  p.S = S; p.HQ = HQ; p.HKV = HKV; p.group = group;
  p.tile_tokens = 128 / group;
  p.rows = rows;
  p.scale_log2 = (scale > 0.f ? scale : 1.0f / sqrtf(128.0f)) * 1.4426950408889634f;
  p.out = out; p.ldo = ldo; p.q_off = q_offsets; p.status = dev->status;
  p.v = cache; p.ldv = L->token_stride;
  p.q_pos = q_positions; p.mask = mask; p.words = mask_words;
  p.max_nodes = max_q_rows; p.max_keys = max_keys; p.whole = cut.whole;
  p.bt = block_table; p.bt_off = bt_offsets; p.bt_len = table_len;
  p.block_size = bs; p.block_log2 = __builtin_ctz(bs); p.box_rows = bs < 128 ? bs : 128;
  p.num_pages = L->num_pages; p.layer = L->layer;
  p.page_rows = L->page_stride / L->token_stride;
  p.layer_rows = L->layer_stride / L->token_stride;
  p.kv_rows = L->kv_stride / L->token_stride;
  p.ws_o = static_cast<float*>(workspace);
  p.ws_ml = need > 0 ? p.ws_o + ctas * 2 * 256 * 128 : nullptr;
  CUtensorMap tq, tkv;
  if (int rc = encode_tmap_3d(&tq, q, {128, uint64_t(HQ), uint64_t(rows)},
                              {256, uint64_t(ldq) * 2},
                              {64, uint32_t(group), uint32_t(p.tile_tokens)},
                              CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, CU_TENSOR_MAP_SWIZZLE_128B))
    return rc;
  if (int rc = encode_tmap_2d(&tkv, cache, L->width, pool_rows, L->token_stride * 2, 64,
                              p.box_rows, CU_TENSOR_MAP_DATA_TYPE_BFLOAT16,
                              CU_TENSOR_MAP_SWIZZLE_128B))
    return rc;
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  // Trees that fit one Q tile leave the second one's place to the V ring.
  const int rc = max_q_rows <= p.tile_tokens ? launch_tree<true>(tq, tkv, p, int(ctas), st)
                                             : launch_tree<false>(tq, tkv, p, int(ctas), st);
  if (rc != KVM_OK) return rc;
  if (!cut.whole && ctas > 1) {
    const int most = int64_t(max_q_rows) < per ? max_q_rows : int(per);
    const int last_row = most <= p.tile_tokens ? most * group : 128 + (most - p.tile_tokens) * group;
    const dim3 grid(unsigned(ctas - 1), (last_row + kJoinRows - 1) / kJoinRows);
    KVM_CUDA_TRY(launch_ex(true, tree_join_kernel, grid, dim3(kJoinThreads), 0, st, p, int(ctas)));
  }
  return KVM_OK;
}
