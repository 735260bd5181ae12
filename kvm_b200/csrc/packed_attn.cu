// Causal grouped-query attention over packed sequences of different lengths:
// kernel.attn.prefill (src/ir/dialect/kernel/dialect.cpp:38) with the row
// offsets an attn_meta value carries (src/ir/dialect/kernel/values.h:83-117).
// The kernel is row_attn.cuh's.
#include <cmath>

#include "row_attn.cuh"

namespace kvm {
namespace {

template <int D, bool F16>
int launch_packed(const CUtensorMap& tq, const CUtensorMap& tk, const CUtensorMap& tv,
                  const RowParams& p, int grid, cudaStream_t st) {
  auto kern = row_attn_kernel<D, F16, false, false>;
  constexpr size_t smem = RowSmem<D, false, false>::bytes();
  static std::atomic<uint64_t> ready{0};
  if (int rc = row_kernel_ready(kern, smem, ready)) return rc;
  KVM_CUDA_TRY(launch_ex(true, kern, dim3(grid), dim3(kRowThreads), smem, st, tq, tk, tv, p));
  return KVM_OK;
}

}  // namespace
}  // namespace kvm

using namespace kvm;

extern "C" int kvm_sm100_attention_packed(const void* q, int64_t ldq, const void* k,
                                          int64_t ldk, const void* v, int64_t ldv, void* out,
                                          int64_t ldo, const int32_t* offsets, int S, int rows,
                                          int HQ, int HKV, int head_dim, int dtype, float scale,
                                          kvm_stream_t stream) {
  if (S < 0 || rows < 0 || HQ <= 0 || HKV <= 0 || HQ % HKV != 0)
    return fail(KVM_ERR_INVALID_ARG,
                "attention_packed: need S, rows >= 0 and HQ a multiple of HKV");
  if (head_dim != 64 && head_dim != 128)
    return fail(KVM_ERR_UNSUPPORTED, "attention_packed: head_dim 64 or 128");
  if (dtype != KVM_EW_BF16 && dtype != KVM_EW_F16)
    return fail(KVM_ERR_UNSUPPORTED, "attention_packed: bf16 or f16");
  if (HQ / HKV > 128)
    return fail(KVM_ERR_UNSUPPORTED, "attention_packed: at most 128 query heads per kv head");
  if (S > kRowMaxSeqs)
    return fail(KVM_ERR_UNSUPPORTED, "attention_packed: at most 1024 sequences a call");
  if (!std::isfinite(scale)) return fail(KVM_ERR_INVALID_ARG, "attention_packed: bad scale");
  if (S == 0 || rows == 0) return KVM_OK;
  if (!q || !k || !v || !out || !offsets || !aligned16(q) || !aligned16(k) || !aligned16(v) ||
      !aligned16(out))
    return fail(KVM_ERR_INVALID_ARG, "attention_packed: NULL or unaligned pointer");
  const int64_t wq = int64_t(HQ) * head_dim, wk = int64_t(HKV) * head_dim;
  if (ldq < wq || ldo < wq || ldk < wk || ldv < wk || ldq % 8 || ldk % 8 || ldv % 8 || ldo % 8)
    return fail(KVM_ERR_INVALID_ARG,
                "attention_packed: row strides must hold the heads and be multiples of 8");
  const DeviceInfo* dev = device_info();
  if (!dev) return KVM_ERR_CUDA;
  RowParams p{};
  p.S = S; p.HQ = HQ; p.HKV = HKV; p.group = HQ / HKV;
  p.tile_tokens = 128 / p.group;
  p.rows = rows;
  p.scale_log2 = (scale > 0.f ? scale : 1.0f / sqrtf(float(head_dim))) * 1.4426950408889634f;
  p.out = out; p.ldo = ldo; p.q_off = offsets; p.status = dev->status;
  p.v = v; p.ldv = ldv;
  const bool f16 = dtype == KVM_EW_F16;
  const auto elem = f16 ? CU_TENSOR_MAP_DATA_TYPE_FLOAT16 : CU_TENSOR_MAP_DATA_TYPE_BFLOAT16;
  CUtensorMap tq, tk, tv;
  if (int rc = encode_tmap_3d(&tq, q, {uint64_t(head_dim), uint64_t(HQ), uint64_t(rows)},
                              {uint64_t(head_dim) * 2, uint64_t(ldq) * 2},
                              {64, uint32_t(p.group), uint32_t(p.tile_tokens)}, elem,
                              CU_TENSOR_MAP_SWIZZLE_128B))
    return rc;
  if (int rc = encode_tmap_2d(&tk, k, wk, rows, ldk * 2, 64, 128, elem,
                              CU_TENSOR_MAP_SWIZZLE_128B))
    return rc;
  if (int rc = encode_tmap_2d(&tv, v, wk, rows, ldv * 2, 64, 128, elem,
                              CU_TENSOR_MAP_SWIZZLE_128B))
    return rc;
  // The number of items is known on the device; this bounds it.
  const int64_t per = 2ll * p.tile_tokens;
  const int64_t items = HKV * ((rows + per - 1) / per + S);
  if (items >= (1ll << 30))
    return fail(KVM_ERR_INVALID_ARG, "attention_packed: too many rows and heads");
  const int grid = items < dev->sm_count ? int(items) : dev->sm_count;
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  if (head_dim == 128)
    return f16 ? launch_packed<128, true>(tq, tk, tv, p, grid, st)
               : launch_packed<128, false>(tq, tk, tv, p, grid, st);
  return f16 ? launch_packed<64, true>(tq, tk, tv, p, grid, st)
             : launch_packed<64, false>(tq, tk, tv, p, grid, st);
}
