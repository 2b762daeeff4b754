// The paged 4-bit KV cache: layout and device helpers.
//
// Per block, KV head and position the cache holds D / 2 bytes of codes (dim 2 i
// in the low nibble of byte i) and, per 64 dims, a bf16 pair (step, zero).  A
// code c stands for  zero + c * step.  Codes and pairs are two tensors,
//   codes [blocks, kv_heads, block_size, D / 2]      uint8
//   scale [blocks, kv_heads, block_size, D / 64, 2]  bf16
// head-major inside a block, so that the positions one (sequence, head) reads
// are contiguous runs: 16 positions are 1 KB of codes and 128 B of pairs at
// D = 128.
#pragma once

#include "common.cuh"

namespace afd {
namespace kv4 {

constexpr int kGroup = 64;  // dims that share one (step, zero)

// Rounded to bf16 toward +inf / -inf, as fp32.  Only the low 16 bits of the
// encoding are cut, so a magnitude grows by adding 0xFFFF before the cut.
AFD_DEVICE float bf16_up_nonneg(float x) { return __uint_as_float((__float_as_uint(x) + 0xFFFFu) & 0xFFFF0000u); }
AFD_DEVICE float bf16_down(float x) {
  const uint32_t b = __float_as_uint(x);
  return __uint_as_float((b >> 31 ? b + 0xFFFFu : b) & 0xFFFF0000u);
}

// The low / high half of a (step, zero) pair as fp32.
AFD_DEVICE float pair_step(uint32_t p) { return __uint_as_float(p << 16); }
// The same by a product with 65536, for kernels whose logic pipe is the busy one.
AFD_DEVICE float pair_step(uint32_t p, uint32_t shl16) { return __uint_as_float(p * shl16); }
AFD_DEVICE float pair_zero(uint32_t p) { return __uint_as_float(p & 0xFFFF0000u); }

}  // namespace kv4
}  // namespace afd
