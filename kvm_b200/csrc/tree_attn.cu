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
constexpr int kJoinRows = kJoinThreads / 32;  // a warp per row

// Joins the parts of the item that stretch c begins and later ones go on with
// (the attention kernel has left its description):
//   M = max m_d, out = sum O_d 2^(m_d - M) / sum l_d 2^(m_d - M).
// Lane d looks after part d's statistics; the parts' rows are loaded four at a
// time. (With the description worked out again by every block, four rows a warp
// and one part after the other, 3 trees of 60 nodes took 97 us, 77 of them the
// attention kernel.)
__global__ void __launch_bounds__(kJoinThreads)
    tree_join_kernel(const __grid_constant__ RowParams p) {
  pdl_wait();
  pdl_trigger();
  const int c = blockIdx.x;
  const RowJoin job = p.ws_join[c];
  const int r = blockIdx.y * kJoinRows + threadIdx.x / 32, lane = threadIdx.x % 32;
  const int q_tile = r >> 7, in_tile = r & 127;
  const int r_tok = in_tile / p.group;
  if (job.ntok0 == 0 || r_tok >= p.tile_tokens || r_tok >= (q_tile ? job.ntok1 : job.ntok0))
    return;
  const int parts = job.last - c + 1;
  // slot of part d: the first where its CTA put it, the others first in theirs
  auto slot = [&](int d) {
    return (d == 0 ? static_cast<long long>(job.part) : 2ll * (c + d)) * 256 + r;
  };
  const float2* ml = reinterpret_cast<const float2*>(p.ws_ml);
  const float4* o = reinterpret_cast<const float4*>(p.ws_o) + lane;
  float M = -INFINITY, L = 0.f;
  float4 acc = make_float4(0.f, 0.f, 0.f, 0.f);
  for (int d0 = 0; d0 < parts; d0 += 32) {
    const int n = min(32, parts - d0);
    const float2 mine = lane < n ? ml[slot(d0 + lane)] : make_float2(-INFINITY, 0.f);
    float top = mine.x;
#pragma unroll
    for (int s = 16; s >= 1; s >>= 1)
      top = max2(top, __shfl_xor_sync(0xffffffffu, top, s));
    const float now = max2(M, top);
    // a part whose keys the row does not see has m = -inf and O = 0
    const float old = M == now ? 1.f : M == -INFINITY ? 0.f : ex2_approx(M - now);
    const float f = mine.x == -INFINITY ? 0.f : mine.x == now ? 1.f : ex2_approx(mine.x - now);
    M = now;
    float sum = mine.y * f;
#pragma unroll
    for (int s = 16; s >= 1; s >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, s);
    L = L * old + sum;
    acc.x *= old; acc.y *= old; acc.z *= old; acc.w *= old;
    for (int d = 0; d < n; d += 4) {
      float4 v[4];
#pragma unroll
      for (int u = 0; u < 4; ++u)
        v[u] = d + u < n ? o[slot(d0 + d + u) * 32] : make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
      for (int u = 0; u < 4; ++u) {
        const float g = __shfl_sync(0xffffffffu, f, (d + u) & 31);
        if (d + u < n) {
          acc.x += v[u].x * g; acc.y += v[u].y * g; acc.z += v[u].z * g; acc.w += v[u].w * g;
        }
      }
    }
  }
  const int token = job.tok0 + q_tile * p.tile_tokens + r_tok;
  float inv = 1.0f / L;
  if (L == 0.f) {  // a row that sees no key at all is zero
    bool sees = p.q_pos[job.s] > 0;
    const int nodes = p.q_off[job.s + 1] - p.q_off[job.s];
    const unsigned* mask = p.mask + static_cast<long long>(p.q_off[job.s] + token) * p.words;
    for (int w = 0; w < p.words && !sees; ++w) sees = tree_bits(mask, p.words, nodes, w * 32) != 0;
    if (!sees) inv = 0.f;
  }
  const long long row = job.row0 + q_tile * p.tile_tokens + r_tok;
  const int head = job.kh * p.group + in_tile - r_tok * p.group;
  uint2 w;
  w.x = pack16<false>(acc.x * inv, acc.y * inv);
  w.y = pack16<false>(acc.z * inv, acc.w * inv);
  reinterpret_cast<uint2*>(static_cast<uint16_t*>(p.out) + row * p.ldo + head * 128ll)[lane] = w;
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
  return cut.whole ? 0 : cut.ctas * (2 * 256 * (128 + 2) * 4 + int64_t(sizeof(RowJoin)));
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
  if (!q || !cache || !out || !q_offsets || !q_positions || !mask ||
      (!block_table && table_len > 0) || !bt_offsets || !aligned16(q) || !aligned16(cache) || !aligned16(out) ||
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
  p.ws_join = need > 0 ? reinterpret_cast<RowJoin*>(p.ws_ml + ctas * 2 * 256 * 2) : nullptr;
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
    KVM_CUDA_TRY(launch_ex(true, tree_join_kernel, grid, dim3(kJoinThreads), 0, st, p));
  }
  return KVM_OK;
}
