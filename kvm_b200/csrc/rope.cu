// Rotary position embedding with a position per row: the general form of
// kernel.attn.rope (src/ir/dialect/kernel/dialect.cpp:40), for the query and
// the key heads of a batch in one launch.
//
// For the pair i < d/2 of a head's first d = rotary_dim columns,
//   theta = position * f_i,   (a, b) -> m (a cos - b sin, b cos + a sin),
// the pair being columns (2i, 2i+1) or (i, i + d/2); the other columns pass.
//
// The angle. A 32-bit product position * f_i is off by position * 2^-25 of
// f_i, several hundredths of a radian at a million tokens. So f_i / 2 pi is
// held as a 64-bit fraction of a turn and multiplied in integers: whole turns
// fall off the top, the fraction is exact up to position * 2^-65, and its top
// 32 bits go to sincospif (angle error 2^-25 turns from the conversion to 24
// bits). One 64-bit multiply replaces a powf and a wide range reduction.
//
// Bound by HBM: every element is read once and written once (8192 rows of 72
// heads of 128, bf16: 49.0-49.4 us interleaved, 6.1 TB/s; 46.5-47.7 us split;
// fp32: 90.3 us in both layouts, 6.7 TB/s). A block takes one row and up to
// kRopeUnroll units a thread, whose loads are issued before the row's d/2 sines
// are computed (one thread each, into shared memory) and consumed after; a
// thread keeps the same columns in every head, so it reads its sines once.
// Units are 16 bytes of a head (two of them, d/2 apart, in the split layout);
// where sizes, strides or pointers leave 16-byte units uneven, units of one pair
// are used.
#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include <cmath>
#include <cstring>

#include "runtime.h"

namespace kvm {
namespace {

constexpr int kRopeThreads = 256;
// Units in flight per thread: of 2, 3 and 4, 3 was the fastest in both layouts
// (split, 8192 rows of 72 heads: 57.3, 47.7, 48.5 us), with at least 6 and 4
// blocks an SM (interleaved with 4, 5, 6, 7: 51.9, 52.7, 49.4, 50.2 us).
constexpr int kRopeUnroll = 3;

struct RopeSide {
  const void* x;
  void* y;
  long long ldx, ldy;
  int heads;
};

struct RopeParams {
  RopeSide q, k;
  const void* positions;
  int pos64;
  int head_dim, rot;     // rot = rotary columns
  int units, slots;      // units per head; heads a block works on at a time
  int rot_units;         // the first of them rotate, the rest are copied
  int heads_per_block;   // slots * iterations
  float sign;            // -1: the transposed rotation
};

__device__ __forceinline__ float to_f(float v) { return v; }
__device__ __forceinline__ float to_f(__half v) { return __half2float(v); }
__device__ __forceinline__ float to_f(__nv_bfloat16 v) { return __bfloat162float(v); }
template <typename T> __device__ __forceinline__ T from_f(float v);
template <> __device__ __forceinline__ float from_f<float>(float v) { return v; }
template <> __device__ __forceinline__ __half from_f<__half>(float v) { return __float2half_rn(v); }
template <> __device__ __forceinline__ __nv_bfloat16 from_f<__nv_bfloat16>(float v) {
  return __float2bfloat16_rn(v);
}

// Two neighbours at a time: one instruction packs both.
__device__ __forceinline__ float2 load2(const __half* e) {
  return __half22float2(*reinterpret_cast<const __half2*>(e));
}
__device__ __forceinline__ float2 load2(const __nv_bfloat16* e) {
  return __bfloat1622float2(*reinterpret_cast<const __nv_bfloat162*>(e));
}
__device__ __forceinline__ float2 load2(const float* e) { return make_float2(e[0], e[1]); }
__device__ __forceinline__ void store2(__half* e, float x, float y) {
  *reinterpret_cast<__half2*>(e) = __floats2half2_rn(x, y);
}
__device__ __forceinline__ void store2(__nv_bfloat16* e, float x, float y) {
  *reinterpret_cast<__nv_bfloat162*>(e) = __floats2bfloat162_rn(x, y);
}
__device__ __forceinline__ void store2(float* e, float x, float y) {
  e[0] = x;
  e[1] = y;
}

// V elements moved as one access when they fill 16 bytes, else one by one.
template <typename T, int V>
struct alignas(sizeof(T) * V == 16 ? 16 : alignof(T)) Vec {
  T e[V];
};

// V: elements of a vector. Split layout: a rotating unit is the vectors at j
// and j + rot/2; interleaved: one vector holding V/2 pairs.
template <typename T, int V, bool INTER>
__global__ void __launch_bounds__(kRopeThreads, INTER ? 6 : 4)
    rope_rows_kernel(const __grid_constant__ RopeParams p,
                     const __grid_constant__ kvm_rope_table t) {
  __shared__ float2 cs[KVM_ROPE_MAX_PAIRS];
  using W = Vec<T, V>;
  const long long row = blockIdx.x;
  const int unit = threadIdx.x % p.units, slot = threadIdx.x / p.units;
  const int h0 = blockIdx.y * p.heads_per_block;
  const int heads = min(p.q.heads + p.k.heads, h0 + p.heads_per_block);
  const bool rotates = unit < p.rot_units;
  const int half = p.rot / 2;
  const int col = rotates ? unit * V : p.rot + (unit - p.rot_units) * V;

  pdl_wait();
  pdl_trigger();
  constexpr int U = kRopeUnroll;
  W a[U], b[U];
#pragma unroll
  for (int u = 0; u < U; ++u) {
    const int h = h0 + slot + u * p.slots;
    if (slot < p.slots && h < heads) {
      const bool is_q = h < p.q.heads;
      const RopeSide& s = is_q ? p.q : p.k;
      const T* x = static_cast<const T*>(s.x) + row * s.ldx +
                   static_cast<long long>(is_q ? h : h - p.q.heads) * p.head_dim + col;
      a[u] = *reinterpret_cast<const W*>(x);
      if (!INTER && rotates) b[u] = *reinterpret_cast<const W*>(x + half);
    }
  }

  constexpr int NP = INTER ? V / 2 : V;  // pairs of a unit
  const long long pos = p.pos64 ? static_cast<const long long*>(p.positions)[row]
                                : static_cast<const int*>(p.positions)[row];
  for (int i = threadIdx.x; i < t.pairs; i += blockDim.x) {
    const unsigned long long turn = static_cast<unsigned long long>(pos) * t.turns[i];
    // top 32 bits as a signed fraction of a turn, in half turns for sincospi
    const float half_turns = static_cast<float>(static_cast<int>(turn >> 32)) * 0x1p-31f;
    float sn, cn;
    sincospif(half_turns, &sn, &cn);
    // a unit's pairs rot_units apart: the units of a warp read without conflicts
    cs[i % NP * p.rot_units + i / NP] = make_float2(cn * t.magnitude, sn * t.magnitude * p.sign);
  }
  __syncthreads();

  float2 w[NP];
  if (rotates) {
#pragma unroll
    for (int i = 0; i < NP; ++i) w[i] = cs[i * p.rot_units + unit];
  }
#pragma unroll
  for (int u = 0; u < U; ++u) {
    const int h = h0 + slot + u * p.slots;
    if (slot < p.slots && h < heads) {
      const bool is_q = h < p.q.heads;
      const RopeSide& s = is_q ? p.q : p.k;
      T* y = static_cast<T*>(s.y) + row * s.ldy +
             static_cast<long long>(is_q ? h : h - p.q.heads) * p.head_dim + col;
      if (rotates) {
        if constexpr (sizeof(T) * V == 16 && INTER) {
#pragma unroll
          for (int i = 0; i < NP; ++i) {
            const float2 f = load2(a[u].e + 2 * i);
            store2(a[u].e + 2 * i, f.x * w[i].x - f.y * w[i].y, f.y * w[i].x + f.x * w[i].y);
          }
        } else if constexpr (sizeof(T) * V == 16) {
#pragma unroll
          for (int i = 0; i < NP; i += 2) {
            const float2 fa = load2(a[u].e + i), fb = load2(b[u].e + i);
            store2(a[u].e + i, fa.x * w[i].x - fb.x * w[i].y,
                   fa.y * w[i + 1].x - fb.y * w[i + 1].y);
            store2(b[u].e + i, fb.x * w[i].x + fa.x * w[i].y,
                   fb.y * w[i + 1].x + fa.y * w[i + 1].y);
          }
        } else {  // one pair
          T& ra = a[u].e[0];
          T& rb = INTER ? a[u].e[V - 1] : b[u].e[0];
          const float fa = to_f(ra), fb = to_f(rb);
          ra = from_f<T>(fa * w[0].x - fb * w[0].y);
          rb = from_f<T>(fb * w[0].x + fa * w[0].y);
        }
        *reinterpret_cast<W*>(y) = a[u];
        if (!INTER) *reinterpret_cast<W*>(y + half) = b[u];
      } else {
        *reinterpret_cast<W*>(y) = a[u];
      }
    }
  }
}

template <typename T, bool INTER>
cudaError_t rope_launch(RopeParams p, const kvm_rope_table& t, int rows, int sms,
                        cudaStream_t st) {
  constexpr int V16 = 16 / sizeof(T);
  auto even = [](const RopeSide& s) {
    return s.heads == 0 || (aligned16(s.x) && aligned16(s.y) && s.ldx % V16 == 0 &&
                            s.ldy % V16 == 0);
  };
  const bool vec = even(p.q) && even(p.k) && p.head_dim % V16 == 0 && p.rot % V16 == 0 &&
                   (INTER || (p.rot / 2) % V16 == 0);
  constexpr int V1 = INTER ? 2 : 1;
  const int v = vec ? V16 : V1;
  p.rot_units = (INTER ? p.rot : p.rot / 2) / v;
  p.units = p.rot_units + (p.head_dim - p.rot) / v;
  const int total = p.q.heads + p.k.heads;
  const int most = kRopeThreads / p.units < total ? kRopeThreads / p.units : total;
  // One pass of the slots per block while that leaves SMs idle, else up to
  // kRopeUnroll, which spreads a row's sines over more of its heads. Of the
  // upper half of the possible slot counts, the one that leaves the fewest
  // heads' worth of threads idle (72 heads on 16 slots would run as 64 + 8).
  int it = 1;
  p.slots = most;
  if (static_cast<long long>(rows) * ((total + most - 1) / most) > 2ll * sms) {
    int least = 1 << 30;
    for (int slots = most; slots > most / 2; --slots) {
      const int passes = (total + slots - 1) / slots;
      const int blocks = (passes + kRopeUnroll - 1) / kRopeUnroll;
      const int per = (passes + blocks - 1) / blocks;
      const int idle = slots * per * blocks - total;
      if (idle < least) {
        least = idle;
        it = per;
        p.slots = slots;
      }
    }
  }
  p.heads_per_block = p.slots * it;
  const dim3 grid(rows, (total + p.heads_per_block - 1) / p.heads_per_block);
  const int threads = (p.slots * p.units + 31) / 32 * 32;
  return launch_ex(true, vec ? rope_rows_kernel<T, V16, INTER> : rope_rows_kernel<T, V1, INTER>,
                   grid, dim3(threads), 0, st, p, t);
}

}  // namespace
}  // namespace kvm

using namespace kvm;

extern "C" int kvm_sm100_rope_table(const kvm_rope_config* c, kvm_rope_table* t) {
  if (!c || !t) return fail(KVM_ERR_INVALID_ARG, "rope_table: NULL argument");
  const int d = c->rotary_dim;
  if (d <= 0 || d % 2 || d / 2 > KVM_ROPE_MAX_PAIRS)
    return fail(KVM_ERR_INVALID_ARG, "rope_table: rotary_dim must be even, 2..256");
  const int kind = c->scaling;
  if (kind < KVM_ROPE_NONE || kind > KVM_ROPE_DIVISORS)
    return fail(KVM_ERR_INVALID_ARG, "rope_table: unknown scaling");
  if (!(c->base > 1.0) || !std::isfinite(c->base))
    return fail(KVM_ERR_INVALID_ARG, "rope_table: base must be a finite number above 1");
  const bool scaled = kind != KVM_ROPE_NONE && kind != KVM_ROPE_DIVISORS;
  if (scaled && (!(c->factor >= 1.0) || !std::isfinite(c->factor)))
    return fail(KVM_ERR_INVALID_ARG, "rope_table: factor must be a finite number >= 1");
  if ((kind == KVM_ROPE_BANDS || kind == KVM_ROPE_YARN) &&
      (!(c->original_len > 0) || !(c->low > 0) || !(c->high > c->low) ||
       !std::isfinite(c->original_len) || !std::isfinite(c->high)))
    return fail(KVM_ERR_INVALID_ARG,
                "rope_table: bands and yarn need original_len > 0 and 0 < low < high");
  if (kind == KVM_ROPE_NTK && d == 2)
    return fail(KVM_ERR_INVALID_ARG, "rope_table: ntk needs rotary_dim > 2");
  // (compared as it is held: a magnitude that fp32 makes infinite or zero is none)
  if (!std::isfinite(static_cast<float>(c->magnitude)) || c->magnitude < 0 ||
      (c->magnitude > 0 && static_cast<float>(c->magnitude) == 0.f))
    return fail(KVM_ERR_INVALID_ARG, "rope_table: magnitude must be 0 or a positive fp32 number");
  if (kind == KVM_ROPE_DIVISORS) {
    if (!c->divisors) return fail(KVM_ERR_INVALID_ARG, "rope_table: divisors is NULL");
    for (int i = 0; i < d / 2; ++i)
      if (!(c->divisors[i] > 0) || !std::isfinite(c->divisors[i]))
        return fail(KVM_ERR_INVALID_ARG, "rope_table: divisors must be finite and positive");
  }
  const long double two_pi = 6.283185307179586476925286766559L;
  long double base = c->base;
  if (kind == KVM_ROPE_NTK)
    base *= powl(static_cast<long double>(c->factor), static_cast<long double>(d) / (d - 2));
  // yarn: the pair index at which a wavelength fits original_len `turns` times
  auto at = [&](double turns) {
    return d * logl(c->original_len / (two_pi * turns)) / (2 * logl(base));
  };
  long double lo = 0, hi = 0;
  if (kind == KVM_ROPE_YARN) {
    lo = fmaxl(floorl(at(c->high)), 0);
    hi = fminl(ceill(at(c->low)), d - 1);
  }
  std::memset(t, 0, sizeof(*t));
  t->pairs = d / 2;
  t->magnitude = c->magnitude > 0 ? static_cast<float>(c->magnitude)
                 : kind == KVM_ROPE_YARN
                     ? static_cast<float>(0.1L * logl(c->factor) + 1.0L)
                     : 1.0f;
  for (int i = 0; i < d / 2; ++i) {
    long double f = powl(base, -2.0L * i / d);
    long double keep = 1;  // share of the unscaled frequency; the rest is f / factor
    if (kind == KVM_ROPE_LINEAR) keep = 0;
    if (kind == KVM_ROPE_BANDS) {
      const long double turns = c->original_len * f / two_pi;
      keep = (turns - c->low) / (static_cast<long double>(c->high) - c->low);
    }
    if (kind == KVM_ROPE_YARN) keep = 1 - (i - lo) / fmaxl(hi - lo, 1e-3L);
    keep = fminl(fmaxl(keep, 0), 1);
    if (scaled && kind != KVM_ROPE_NTK) f = f * keep + f / c->factor * (1 - keep);
    if (kind == KVM_ROPE_DIVISORS) f /= c->divisors[i];
    const long double turn = fmodl(f / two_pi, 1.0L);
    t->turns[i] = static_cast<uint64_t>(ldexpl(turn, 64));
  }
  return KVM_OK;
}

extern "C" int kvm_sm100_rope(const kvm_rope_table* table, const void* q, int64_t ldq,
                              void* out_q, int64_t ldoq, int heads_q, const void* k,
                              int64_t ldk, void* out_k, int64_t ldok, int heads_k, int rows,
                              int head_dim, int interleaved, int backward, int dtype,
                              const void* positions, int positions_64, kvm_stream_t stream) {
  if (!table || table->pairs <= 0 || table->pairs > KVM_ROPE_MAX_PAIRS)
    return fail(KVM_ERR_INVALID_ARG, "rope: table not made by kvm_sm100_rope_table");
  if (rows < 0 || heads_q <= 0 || heads_k < 0 || head_dim <= 0 || head_dim > 256 ||
      head_dim % 2 || 2 * table->pairs > head_dim)
    return fail(KVM_ERR_INVALID_ARG,
                "rope: need heads > 0 and an even head_dim of at most 256 that holds "
                "rotary_dim");
  if (heads_q > (1 << 14) || heads_k > (1 << 14))
    return fail(KVM_ERR_INVALID_ARG, "rope: too many heads");
  if (dtype != KVM_EW_BF16 && dtype != KVM_EW_F16 && dtype != KVM_EW_F32)
    return fail(KVM_ERR_INVALID_ARG, "rope: dtype must be bf16, f16 or f32");
  const size_t elem = dtype == KVM_EW_F32 ? 4 : 2;
  auto bad = [&](const void* x, int64_t ldx, const void* y, int64_t ldy, int heads) {
    const int64_t w = int64_t(heads) * head_dim;
    return !x || !y || reinterpret_cast<uintptr_t>(x) % elem ||
           reinterpret_cast<uintptr_t>(y) % elem || (rows > 1 && (ldx < w || ldy < w)) ||
           (x == y && ldx != ldy && rows > 1);
  };
  if (rows == 0) return KVM_OK;
  if (bad(q, ldq, out_q, ldoq, heads_q) ||
      (heads_k > 0 && bad(k, ldk, out_k, ldok, heads_k)) || !positions ||
      reinterpret_cast<uintptr_t>(positions) % (positions_64 ? 8 : 4))
    return fail(KVM_ERR_INVALID_ARG,
                "rope: NULL or misaligned pointer, a row stride below heads * head_dim, or "
                "an in-place call with two row strides");
  const DeviceInfo* dev = device_info();
  if (!dev) return KVM_ERR_CUDA;
  RopeParams p{};
  p.q = {q, out_q, ldq, ldoq, heads_q};
  p.k = {k, out_k, ldk, ldok, heads_k};
  p.positions = positions;
  p.pos64 = positions_64;
  p.head_dim = head_dim;
  p.rot = 2 * table->pairs;
  p.sign = backward ? -1.f : 1.f;
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  auto go = [&](auto tag) {
    using T = decltype(tag);
    return interleaved ? rope_launch<T, true>(p, *table, rows, dev->sm_count, st)
                       : rope_launch<T, false>(p, *table, rows, dev->sm_count, st);
  };
  if (dtype == KVM_EW_F32) KVM_CUDA_TRY(go(float()));
  else if (dtype == KVM_EW_F16) KVM_CUDA_TRY(go(__half()));
  else KVM_CUDA_TRY(go(__nv_bfloat16()));
  return KVM_OK;
}
