// Rows into and out of the paged 4-bit KV cache (layout: kv_int4.cuh).
//
// write: per (token, KV head, 64 dims)
//     zero = max. bf16 <= min(x);  step = min. bf16 >= fl((max(x) - zero) / 15)
//     c    = clamp(rint(fl(fl(x - zero) / step)), 0, 15)        (0 when step = 0)
//   zero is rounded down and step up, so every x lies in [zero, zero + 15 step]
//   and the stored value is within half a step of it.  Every rounding is an
//   IEEE fp32 operation, so the codes are the same on every device.  8 lanes
//   hold a group, 8 dims each; min and max are three shuffles.
// read: zero + c * step, one fused multiply-add (the product is exact).
//
// Both are bound by memory traffic: one 16-byte load (write) or store (read)
// per thread and the packed word on the other side.
#include "kv_int4.cuh"
#include "launchers.h"

namespace afd {
namespace kv4 {

constexpr int kThreads = 256;

template <typename T>
AFD_DEVICE void load8(float (&x)[8], const T* p, bool vec) {
  if (vec) {
    if constexpr (sizeof(T) == 2) {
      const Vec16<T> v = load16(p);
#pragma unroll
      for (int i = 0; i < 8; ++i) x[i] = to_f32(v.v[i]);
    } else {
      const Vec16<T> a = load16(p), b = load16(p + 4);
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        x[i] = to_f32(a.v[i]);
        x[i + 4] = to_f32(b.v[i]);
      }
    }
  } else {
#pragma unroll
    for (int i = 0; i < 8; ++i) x[i] = to_f32(p[i]);
  }
}

// grid.x covers (token, head, D / 8) and grid.y is 0 for K, 1 for V.  A thread's
// 8 lanes of a group are neighbours and in range together (D % 64 == 0).
template <typename T>
__global__ void __launch_bounds__(kThreads) write_kernel(Kv4WriteParams p) {
  const int parts = p.dim / 8;
  const int64_t idx = (int64_t)blockIdx.x * kThreads + threadIdx.x;
  const bool live = idx < (int64_t)p.tokens * p.kv_heads * parts;
  const int64_t at = live ? idx : 0;
  const int part = (int)(at % parts);
  const int64_t row = at / parts;
  const int head = (int)(row % p.kv_heads);
  const int64_t tok = row / p.kv_heads;
  const bool is_v = blockIdx.y != 0;
  const T* src = reinterpret_cast<const T*>(is_v ? p.v : p.k) + tok * (is_v ? p.v_st : p.k_st) +
                 head * (is_v ? p.v_sh : p.k_sh) + part * 8;
  float x[8];
  load8(x, src, p.vec != 0);
  float lo = x[0], hi = x[0];
#pragma unroll
  for (int i = 1; i < 8; ++i) {
    lo = fminf(lo, x[i]);
    hi = fmaxf(hi, x[i]);
  }
#pragma unroll
  for (int o = 1; o < 8; o <<= 1) {
    lo = fminf(lo, __shfl_xor_sync(0xffffffffu, lo, o));
    hi = fmaxf(hi, __shfl_xor_sync(0xffffffffu, hi, o));
  }
  if (!live) return;
  const int64_t slot = p.slots[tok];
  if (slot < 0 || slot >= p.num_slots) {
    if (part == 0 && p.status != nullptr) atomicExch(p.status, kStatusBadIndex);
    return;
  }
  const float zero = bf16_down(lo);
  const float step = bf16_up_nonneg(__fdiv_rn(hi - zero, 15.f));
  uint32_t word = 0;
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    const float c = step > 0.f ? rintf(__fdiv_rn(x[i] - zero, step)) : 0.f;
    word |= (uint32_t)fminf(fmaxf(c, 0.f), 15.f) << (4 * i);
  }
  const int64_t blk = slot / p.block_size, off = slot % p.block_size;
  const int64_t dst = (blk * p.kv_heads + head) * p.block_size + off;
  uint8_t* codes = is_v ? p.v_codes : p.k_codes;
  uint32_t* scale = is_v ? p.v_scale : p.k_scale;
  reinterpret_cast<uint32_t*>(codes + dst * (p.dim / 2))[part] = word;
  if (part % 8 == 0)
    scale[dst * (p.dim / kGroup) + part / 8] = __float_as_uint(step) >> 16 | (__float_as_uint(zero) & 0xFFFF0000u);
  if (p.scores != nullptr && !is_v && part == 0) p.scores[dst] = 0.f;
}

template <typename T>
__global__ void __launch_bounds__(kThreads) read_kernel(Kv4ReadParams p) {
  const int parts = p.dim / 8;
  const int64_t idx = (int64_t)blockIdx.x * kThreads + threadIdx.x;
  if (idx >= (int64_t)p.tokens * p.kv_heads * parts) return;
  const int part = (int)(idx % parts);
  const int64_t row = idx / parts;
  const int head = (int)(row % p.kv_heads);
  const int64_t slot = p.slots[row / p.kv_heads];
  const bool is_v = blockIdx.y != 0;
  T* dst = reinterpret_cast<T*>(is_v ? p.v : p.k) + idx * 8;
  float x[8] = {};
  if (slot < 0 || slot >= p.num_slots) {
    if (part == 0 && p.status != nullptr) atomicExch(p.status, kStatusBadIndex);
  } else {
    const int64_t src = (slot / p.block_size * p.kv_heads + head) * p.block_size + slot % p.block_size;
    const uint32_t word = reinterpret_cast<const uint32_t*>((is_v ? p.v_codes : p.k_codes) + src * (p.dim / 2))[part];
    const uint32_t pair = (is_v ? p.v_scale : p.k_scale)[src * (p.dim / kGroup) + part / 8];
    const float step = pair_step(pair), zero = pair_zero(pair);
#pragma unroll
    for (int i = 0; i < 8; ++i) x[i] = fmaf((float)((word >> (4 * i)) & 15u), step, zero);
  }
  constexpr int N = Vec16<T>::N;
#pragma unroll
  for (int u = 0; u < 8 / N; ++u) {
    Vec16<T> v;
#pragma unroll
    for (int i = 0; i < N; ++i) v.v[i] = from_f32<T>(x[u * N + i]);
    store16(dst + u * N, v);
  }
}

}  // namespace kv4
}  // namespace afd

using namespace afd;

void launch_kv4_write(const Kv4WriteParams& p, int dtype, cudaStream_t s) {
  const int64_t n = (int64_t)p.tokens * p.kv_heads * (p.dim / 8);
  const dim3 grid((unsigned)((n + kv4::kThreads - 1) / kv4::kThreads), 2);
  switch (dtype) {
    case kF32: kv4::write_kernel<float><<<grid, kv4::kThreads, 0, s>>>(p); break;
    case kF16: kv4::write_kernel<__half><<<grid, kv4::kThreads, 0, s>>>(p); break;
    default: kv4::write_kernel<__nv_bfloat16><<<grid, kv4::kThreads, 0, s>>>(p); break;
  }
}

void launch_kv4_read(const Kv4ReadParams& p, int dtype, cudaStream_t s) {
  const int64_t n = (int64_t)p.tokens * p.kv_heads * (p.dim / 8);
  const dim3 grid((unsigned)((n + kv4::kThreads - 1) / kv4::kThreads), 2);
  switch (dtype) {
    case kF32: kv4::read_kernel<float><<<grid, kv4::kThreads, 0, s>>>(p); break;
    case kF16: kv4::read_kernel<__half><<<grid, kv4::kThreads, 0, s>>>(p); break;
    default: kv4::read_kernel<__nv_bfloat16><<<grid, kv4::kThreads, 0, s>>>(p); break;
  }
}
