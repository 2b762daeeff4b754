// Rows into and out of the paged 4-bit KV cache (layout: kv_int4.cuh).
//
// write: per (token, KV head, 64 dims)
//     zero = max. bf16 <= min(x);  step = min. bf16 >= fl((max(x) - zero) / 15)
//     c    = clamp(rint(fl(fl(x - zero) / step)), 0, 15)        (0 when step = 0)
//   zero is rounded down and step up, so every x lies in [zero, zero + 15 step]
//   and the stored value is within half a step of it.  Every rounding is an
//   IEEE fp32 operation, so the codes are the same on every device.  A group
//   with a NaN, an infinity or a range that overflows fp32 reads back as NaN:
//   its step is infinite, or step and zero are NaN.  8 lanes hold a group, 8
//   dims each; min and max are three shuffles.
// read: zero + c * step, one fused multiply-add (the product is exact).
//
// Their floor is memory traffic.  A thread takes K and V of its part of a row,
// which halves the index arithmetic: 16001 tokens x 8 heads of 128, bf16, are
// written in 32 us (84 MB, 2.6 TB/s; instruction issue bounds it, 3.3 of 4 per
// clock) and read as fp32 in 34 us (150 MB, 4.4 TB/s).
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

// d / s, correctly rounded, with r the correctly rounded 1 / s: a quotient
// within an ulp and one exact remainder (Markstein 1990).  Holds because s has
// 8 significant bits (its mantissa is not all ones) and both are far from the
// ends of the exponent range.
AFD_DEVICE float quotient(float d, float s, float r) {
  const float q = d * r;
  return fmaf(fmaf(-q, s, d), r, q);
}

// Row (block, head, offset) of a slot in the cache; a power-of-two block size is a shift.
AFD_DEVICE int64_t cache_row(int64_t slot, uint32_t head, int kv_heads, int block_size, int shift) {
  int64_t blk;
  int off;
  if (shift >= 0) {
    blk = slot >> shift;
    off = (int)slot & (block_size - 1);
  } else {
    blk = slot / block_size;
    off = (int)(slot - blk * block_size);
  }
  return (blk * kv_heads + head) * block_size + off;
}

// Quantises the 8 values of this lane with the 64 of its 8 neighbours and
// stores its word and, from the group's first lane, the (step, zero) pair.
AFD_DEVICE void store_group(const float (&x)[8], bool live, uint32_t* word_at, uint32_t* pair_at, bool first) {
  float lo = x[0], hi = x[0];
#pragma unroll
  for (int i = 1; i < 8; ++i) {
    lo = min_nan(lo, x[i]);
    hi = max_nan(hi, x[i]);
  }
#pragma unroll
  for (int o = 1; o < 8; o <<= 1) {
    lo = min_nan(lo, __shfl_xor_sync(0xffffffffu, lo, o));
    hi = max_nan(hi, __shfl_xor_sync(0xffffffffu, hi, o));
  }
  if (!live) return;
  const float zero = bf16_down(lo);
  const float exact = __fdiv_rn(hi - zero, 15.f);
  const float step = bf16_up_nonneg(exact);
  uint32_t word = 0, pair = __float_as_uint(step) >> 16 | (__float_as_uint(zero) & 0xFFFF0000u);
  if (exact != exact) {  // a NaN in the group, or nothing but one infinity
    pair = 0x7FC07FC0u;
  } else if (step > 1e-25f && step < 1e25f) {
    // Adding 1.5 * 2^23 rounds to a whole number, ties to even, in the low bits
    // of 0x4B400000.  zero <= x and the step's rounding keep it in 0 .. 15.
    const float r = __frcp_rn(step);
    constexpr uint32_t kOnes = 0x11111111u;
#pragma unroll
    for (int i = 0; i < 8; ++i)
      word += __float_as_uint(quotient(x[i] - zero, step, r) + 12582912.f) * (1u << (4 * i));
    word -= 0x4B400000u * kOnes;
  } else if (step > 0.f) {
#pragma unroll
    for (int i = 0; i < 8; ++i)
      word |= (uint32_t)fminf(fmaxf(rintf(__fdiv_rn(x[i] - zero, step)), 0.f), 15.f) << (4 * i);
  }
  *word_at = word;
  if (first) *pair_at = pair;
}

// A block takes kThreads / parts rows (token, head), K and V of each.  D / 8
// lanes hold a row, so the 8 lanes of a group are neighbours.
template <typename T, int D>
__global__ void __launch_bounds__(kThreads) write_kernel(Kv4WriteParams p) {
  constexpr int kParts = D / 8, kRows = kThreads / kParts;
  const uint32_t part = threadIdx.x % kParts;
  uint32_t row = blockIdx.x * kRows + threadIdx.x / kParts;
  bool live = row < (uint32_t)p.tokens * (uint32_t)p.kv_heads;
  row = live ? row : 0;
  const uint32_t tok = row / (uint32_t)p.kv_heads, head = row - tok * (uint32_t)p.kv_heads;
  const T* k = reinterpret_cast<const T*>(p.k) + (int64_t)tok * p.k_st + (int64_t)head * p.k_sh + part * 8;
  const T* v = reinterpret_cast<const T*>(p.v) + (int64_t)tok * p.v_st + (int64_t)head * p.v_sh + part * 8;
  const int64_t slot = p.slots[tok];
  float x[8], y[8];
  load8(x, k, p.vec != 0);
  load8(y, v, p.vec != 0);
  if (slot < 0 || slot >= p.num_slots) {
    if (live && part == 0 && p.status != nullptr) atomicExch(p.status, kStatusBadIndex);
    live = false;
  }
  const int64_t dst = live ? cache_row(slot, head, p.kv_heads, p.block_size, p.block_shift) : 0;
  const int64_t word = dst * kParts + part, pair = dst * (D / kGroup) + part / 8;
  store_group(x, live, reinterpret_cast<uint32_t*>(p.k_codes) + word, p.k_scale + pair, part % 8 == 0);
  store_group(y, live, reinterpret_cast<uint32_t*>(p.v_codes) + word, p.v_scale + pair, part % 8 == 0);
  if (p.scores != nullptr && live && part == 0) p.scores[dst] = 0.f;
}

// A thread writes one 16-byte vector of K and of V: neighbouring lanes,
// neighbouring vectors.
template <typename T, int D>
__global__ void __launch_bounds__(kThreads) read_kernel(Kv4ReadParams p) {
  constexpr int N = Vec16<T>::N, kParts = D / N, kRows = kThreads / kParts;
  const uint32_t part = threadIdx.x % kParts;
  const uint32_t row = blockIdx.x * kRows + threadIdx.x / kParts;
  if (row >= (uint32_t)p.tokens * (uint32_t)p.kv_heads) return;
  const uint32_t tok = row / (uint32_t)p.kv_heads, head = row - tok * (uint32_t)p.kv_heads;
  const int64_t slot = p.slots[tok];
  uint32_t kw = 0, kp = 0, vw = 0, vp = 0;  // a zero step and zero: zeros
  if (slot < 0 || slot >= p.num_slots) {
    if (part == 0 && p.status != nullptr) atomicExch(p.status, kStatusBadIndex);
  } else {
    const int64_t src = cache_row(slot, head, p.kv_heads, p.block_size, p.block_shift);
    const int64_t word = src * (D / 8) + part * N / 8, pair = src * (D / kGroup) + part * N / kGroup;
    kw = reinterpret_cast<const uint32_t*>(p.k_codes)[word] >> (part * N % 8 * 4);
    vw = reinterpret_cast<const uint32_t*>(p.v_codes)[word] >> (part * N % 8 * 4);
    kp = p.k_scale[pair];
    vp = p.v_scale[pair];
  }
  Vec16<T> k, v;
#pragma unroll
  for (int i = 0; i < N; ++i) {
    k.v[i] = from_f32<T>(fmaf((float)((kw >> (4 * i)) & 15u), pair_step(kp), pair_zero(kp)));
    v.v[i] = from_f32<T>(fmaf((float)((vw >> (4 * i)) & 15u), pair_step(vp), pair_zero(vp)));
  }
  const int64_t at = (int64_t)row * D + part * N;
  store16(reinterpret_cast<T*>(p.k) + at, k);
  store16(reinterpret_cast<T*>(p.v) + at, v);
}

// The grid over rows of D values, N of them a thread.
template <int D, int N> dim3 row_grid(int64_t rows) {
  constexpr int kRows = kThreads / (D / N);
  return dim3((unsigned)((rows + kRows - 1) / kRows));
}
int shift_of(int block_size) { return (block_size & (block_size - 1)) == 0 ? __builtin_ctz(block_size) : -1; }

template <typename T>
void write(Kv4WriteParams p, cudaStream_t s) {
  const int64_t rows = (int64_t)p.tokens * p.kv_heads;
  p.block_shift = shift_of(p.block_size);
  switch (p.dim) {
    case 64: write_kernel<T, 64><<<row_grid<64, 8>(rows), kThreads, 0, s>>>(p); break;
    case 128: write_kernel<T, 128><<<row_grid<128, 8>(rows), kThreads, 0, s>>>(p); break;
    default: write_kernel<T, 256><<<row_grid<256, 8>(rows), kThreads, 0, s>>>(p);
  }
}
template <typename T>
void read(Kv4ReadParams p, cudaStream_t s) {
  const int64_t rows = (int64_t)p.tokens * p.kv_heads;
  p.block_shift = shift_of(p.block_size);
  switch (p.dim) {
    case 64: read_kernel<T, 64><<<row_grid<64, Vec16<T>::N>(rows), kThreads, 0, s>>>(p); break;
    case 128: read_kernel<T, 128><<<row_grid<128, Vec16<T>::N>(rows), kThreads, 0, s>>>(p); break;
    default: read_kernel<T, 256><<<row_grid<256, Vec16<T>::N>(rows), kThreads, 0, s>>>(p);
  }
}

}  // namespace kv4
}  // namespace afd

using namespace afd;

void launch_kv4_write(const Kv4WriteParams& p, int dtype, cudaStream_t s) {
  switch (dtype) {
    case kF32: kv4::write<float>(p, s); break;
    case kF16: kv4::write<__half>(p, s); break;
    default: kv4::write<__nv_bfloat16>(p, s); break;
  }
}

void launch_kv4_read(const Kv4ReadParams& p, int dtype, cudaStream_t s) {
  switch (dtype) {
    case kF32: kv4::read<float>(p, s); break;
    case kF16: kv4::read<__half>(p, s); break;
    default: kv4::read<__nv_bfloat16>(p, s); break;
  }
}
