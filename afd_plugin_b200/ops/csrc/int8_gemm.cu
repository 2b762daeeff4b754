// Linear layer in 8-bit integers:  y[t, n] = xs[t] ws[n] sum_k xq[t, k] w[n, k].
//
// quantize   per token  xs = amax / 127,  xq = clamp(rint(x * (127 / amax)))
//            with amax = max(|x|, 2^-100); one block per token, which keeps
//            a row's first 8192 values in registers (what is longer is read
//            twice, the second time from cache).  4099 x 7168 bf16: 22.6 us,
//            3.9 TB/s; its loads all wait for one another at the row's maximum.
// gemm       tcgen05.mma kind::i8 on TMA-fed 128B-swizzled tiles, int32
//            accumulators in TMEM.  int32 sums are exact, so the order and the
//            split of K do not show in the result; the scales are applied in
//            fp32 as the accumulators are read.
//
// Tile: 128 tokens (MMA M, TMEM lanes) x BN output channels (MMA N, columns),
// 128 bytes of K per stage.  A lane holds one token's consecutive channels, so
// the epilogue stores 16-byte vectors without a transpose.  Rows of either
// operand past the end are filled with zeros by TMA, as is K past its end.
//
// Warps: 0 TMA producer, 1 MMA issuer, 2-5 epilogue.  Weights do not depend on
// the quantize kernel: the producer starts on them before it waits for that
// grid (programmatic dependent launch).
//
// What bounds it.  4099 x 36864 x 7168: 700 us in isolation (3.1 POPS), 824 us
// back to back under the power cap (2.6 POPS; twice cuBLAS's sustained bf16
// rate is 2.8).  256 x 2048 x 10944: 17.5 us, of which 4 us wait for the
// quantize kernel and about 6 us feed 90 MB from L2; its floor is 4.4 us of
// HBM.  5 x 5120 x 2048: 8.3 us, latencies (floor 1.6 us), and 10 us with the
// quantize kernel before it.
//
// Beside the framework's bf16 linear layer (5120 x 2048, graphs): 10.2 us against
// 6.5 at 1 - 64 tokens, 17.4 against 10.2 at 512, 60.8 against 62.1 at 4096.  It
// halves the weights' memory; it is faster for prompts only.
//
// Every wait is bounded; on expiry the CTA records kStatusWaitTimeout, waits
// (bounded) for its MMAs in flight and winds down.
#include <cooperative_groups.h>
#include <cudaTypedefs.h>

#include <algorithm>

#include "common.cuh"
#include "device_state.h"
#include "launchers.h"

namespace afd {
PFN_cuTensorMapEncodeTiled_v12000 get_tensor_map_encoder();

namespace i8 {
namespace cg = cooperative_groups;

constexpr int kBM = 128;
constexpr int kBK = 128;  // bytes of K per stage: one swizzle row
constexpr int kThreads = 6 * 32;
constexpr int kXBytes = kBM * kBK;

// ------------------------------------------------------------------ quantize
constexpr int kQThreads = 256;

// 8 consecutive elements, as loaded.
template <typename T>
struct Chunk {
  T v[8];
  AFD_DEVICE void load(const T* p, bool vec) {
    if (vec) {
      constexpr int N = Vec16<T>::N;
#pragma unroll
      for (int u = 0; u < 8 / N; ++u) *reinterpret_cast<uint4*>(v + u * N) = *reinterpret_cast<const uint4*>(p + u * N);
    } else {
#pragma unroll
      for (int i = 0; i < 8; ++i) v[i] = p[i];
    }
  }
  AFD_DEVICE float amax(float m) const {
#pragma unroll
    for (int i = 0; i < 8; ++i) m = max_nan(m, fabsf(to_f32(v[i])));
    return m;
  }
  AFD_DEVICE uint2 quantized(float inv) const {
    uint32_t w[2] = {0, 0};
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      const int c = max(-127, min(127, __float2int_rn(to_f32(v[i]) * inv)));  // NaN converts to 0; its scale is NaN
      w[i / 4] |= (uint32_t)(c & 255) << (8 * (i % 4));
    }
    return make_uint2(w[0], w[1]);
  }
};

constexpr int kQHeld = 4;  // chunks of a row a thread keeps in registers: 8192 values are read once

template <typename T>
__global__ void __launch_bounds__(kQThreads) quantize_kernel(int8_t* __restrict__ q, float* __restrict__ scale,
                                                             const T* __restrict__ x, int64_t ld, int k, int vec) {
  __shared__ float s_max[kQThreads / 32];
  pdl_launch_dependents();
  constexpr int kStride = kQThreads * 8;
  const T* row = x + blockIdx.x * ld;
  int8_t* out = q + (int64_t)blockIdx.x * k;
  const int i0 = threadIdx.x * 8;
  Chunk<T> held[kQHeld];
  float amax = 0.f;
#pragma unroll
  for (int u = 0; u < kQHeld; ++u)
    if (i0 + u * kStride < k) held[u].load(row + i0 + u * kStride, vec != 0);
#pragma unroll
  for (int u = 0; u < kQHeld; ++u)
    if (i0 + u * kStride < k) amax = held[u].amax(amax);
  for (int i = i0 + kQHeld * kStride; i < k; i += kStride) {
    Chunk<T> c;
    c.load(row + i, vec != 0);
    amax = c.amax(amax);
  }
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) amax = max_nan(amax, __shfl_xor_sync(0xffffffffu, amax, o));
  if ((threadIdx.x & 31) == 0) s_max[threadIdx.x / 32] = amax;
  __syncthreads();
  amax = 7.888609052210118e-31f;  // 2^-100
#pragma unroll
  for (int w = 0; w < kQThreads / 32; ++w) amax = max_nan(amax, s_max[w]);
  const float inv = __fdiv_rn(127.f, amax);
  if (threadIdx.x == 0) scale[blockIdx.x] = __fdiv_rn(amax, 127.f);
#pragma unroll
  for (int u = 0; u < kQHeld; ++u)
    if (i0 + u * kStride < k) *reinterpret_cast<uint2*>(out + i0 + u * kStride) = held[u].quantized(inv);
  for (int i = i0 + kQHeld * kStride; i < k; i += kStride) {
    Chunk<T> c;
    c.load(row + i, vec != 0);
    *reinterpret_cast<uint2*>(out + i) = c.quantized(inv);
  }
}

// ---------------------------------------------------------------------- gemm
// K-major, 128B-swizzled operand descriptor (8-row groups 1024 B apart).
AFD_DEVICE uint64_t make_desc(uint32_t saddr) {
  return (uint64_t)((saddr & 0x3FFFF) >> 4) | (uint64_t)1 << 16 | (uint64_t)(1024 >> 4) << 32 | (uint64_t)1 << 46 |
         (uint64_t)2 << 61;
}
// kind::i8 instruction descriptor: s8 x s8 -> s32, both K-major.
AFD_DEVICE constexpr uint32_t make_idesc(int m, int n) {
  return (2u << 4) | (1u << 7) | (1u << 10) | ((uint32_t)(n >> 3) << 17) | ((uint32_t)(m >> 4) << 24);
}
AFD_DEVICE void mma_i8(uint32_t tmem_d, uint64_t adesc, uint64_t bdesc, uint32_t idesc, uint32_t accumulate) {
  asm volatile(
      "{\n .reg .pred p;\n setp.ne.b32 p, %4, 0;\n"
      " tcgen05.mma.cta_group::1.kind::i8 [%0], %1, %2, %3, p;\n}\n" ::"r"(tmem_d),
      "l"(adesc), "l"(bdesc), "r"(idesc), "r"(accumulate));
}
AFD_DEVICE void mma_commit(uint64_t* bar) {
  asm volatile("tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [%0];" ::"r"(smem_u32(bar))
               : "memory");
}
AFD_DEVICE void tc_fence_before() { asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory"); }
AFD_DEVICE void tc_fence_after() { asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory"); }
AFD_DEVICE void tmem_ld32(uint32_t taddr, int (&r)[32]) {
  asm volatile(
      "tcgen05.ld.sync.aligned.32x32b.x32.b32 {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16,%17,%18,%19,"
      "%20,%21,%22,%23,%24,%25,%26,%27,%28,%29,%30,%31}, [%32];"
      : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]), "=r"(r[8]),
        "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15]), "=r"(r[16]),
        "=r"(r[17]), "=r"(r[18]), "=r"(r[19]), "=r"(r[20]), "=r"(r[21]), "=r"(r[22]), "=r"(r[23]), "=r"(r[24]),
        "=r"(r[25]), "=r"(r[26]), "=r"(r[27]), "=r"(r[28]), "=r"(r[29]), "=r"(r[30]), "=r"(r[31])
      : "r"(taddr));
  asm volatile("tcgen05.wait::ld.sync.aligned;" ::: "memory");
}

template <int BN, int STAGES>
struct Smem {
  alignas(1024) uint8_t x[STAGES][kXBytes];
  alignas(1024) uint8_t w[STAGES][BN * kBK];
  alignas(16) float ws[2][BN];  // channel scales of the tile in each accumulator
  uint64_t full[STAGES];
  uint64_t empty[STAGES];
  uint64_t acc_full[2];
  uint64_t acc_empty[2];
  uint32_t tmem_base;
};

// Of gemm_pair_kernel: 6 stages of 32 KB, channel scales, barriers, padded to 1 KB.
constexpr size_t kPairSmem = 6 * 2 * kXBytes + 3 * 1024;

struct Args {
  void* y;
  const float* xs;
  const float* ws;
  int* status;
  int t, n, k_blocks;
  int m_tiles, n_tiles;
  int band;      // m tiles walked before the next n tile
  int x_rows;    // rows of a token tile that TMA fetches
  int out_vec;   // rows of y start on 16-byte boundaries
};

// Tiles in order: bands of `band` token tiles; inside a band channels outer,
// tokens inner, so a band's tokens stay in L2 while the weights pass once.
AFD_DEVICE void tile_at(const Args& a, int i, int& m, int& n) {
  const int per = a.band * a.n_tiles;
  const int b = i / per, r = i - b * per;
  const int rows = min(a.band, a.m_tiles - b * a.band);
  n = r / rows;
  m = b * a.band + (r - n * rows);
}

// Scales 32 accumulators of one token and stores them from channel n0 on.
template <typename T>
AFD_DEVICE void store32(const Args& a, const int (&v)[32], const float* ws, float xs, int row, int n0) {
  if (row >= a.t || n0 >= a.n) return;
  T* y = reinterpret_cast<T*>(a.y) + (int64_t)row * a.n + n0;
  if (a.out_vec && n0 + 32 <= a.n) {
    constexpr int N = Vec16<T>::N;
#pragma unroll
    for (int u = 0; u < 32 / N; ++u) {
      Vec16<T> o;
#pragma unroll
      for (int i = 0; i < N; ++i) o.v[i] = from_f32<T>((float)v[u * N + i] * (xs * ws[u * N + i]));
      store16(y + u * N, o);
    }
  } else {
#pragma unroll
    for (int i = 0; i < 32; ++i)
      if (n0 + i < a.n) y[i] = from_f32<T>((float)v[i] * (xs * ws[i]));
  }
}

// Barrier of the four epilogue warps that also ands `pred` over them: all of
// them see a wait's outcome alike, so all leave or none.
AFD_DEVICE bool epi_all(bool pred) {
  uint32_t out;
  asm volatile(
      "{\n .reg .pred p, q;\n setp.ne.u32 p, %1, 0;\n bar.red.and.pred q, 1, 128, p;\n selp.u32 %0, 1, 0, q;\n}\n"
      : "=r"(out)
      : "r"((uint32_t)pred)
      : "memory");
  return out != 0;
}
AFD_DEVICE void report_timeout(const Args& a) {
  if (a.status != nullptr) atomicExch(a.status, kStatusWaitTimeout);
}

// Persistent: CTA c takes tiles c, c + grid, ...; the accumulator is double
// buffered, so a tile's epilogue overlaps the next one's MMAs.  With kSplit, a
// cluster works on one tile: each CTA sums its share of K, and each then adds
// up its share of the channels over the cluster through distributed shared
// memory.
template <typename T, int BN, int STAGES, bool kSplit>
__global__ void __launch_bounds__(kThreads, 1) gemm_kernel(const __grid_constant__ CUtensorMap x_map,
                                                           const __grid_constant__ CUtensorMap w_map, const Args a) {
  using SmemT = Smem<BN, STAGES>;
  constexpr int kAccBufs = kSplit ? 1 : 2;
  constexpr uint32_t kCols = kAccBufs * BN < 32 ? 32 : kAccBufs * BN;
  extern __shared__ uint8_t smem_raw[];
  SmemT& sm = *reinterpret_cast<SmemT*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  const int warp = threadIdx.x / 32, lane = threadIdx.x & 31;
  if (threadIdx.x == 0) {
    for (int s = 0; s < STAGES; ++s) {
      mbar_init(&sm.full[s], 1);
      mbar_init(&sm.empty[s], 1);
    }
    for (int b = 0; b < 2; ++b) {
      mbar_init(&sm.acc_full[b], 1);
      mbar_init(&sm.acc_empty[b], 4);
    }
    fence_barrier_init();
  }
  if (warp == 1) {
    asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(&sm.tmem_base)),
                 "r"(kCols));
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;");
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = sm.tmem_base;

  // This CTA's tiles and K blocks.
  int first = blockIdx.x, stride = gridDim.x, kb0 = 0, kb1 = a.k_blocks;
  int split_rank = 0, splits = 1;
  if constexpr (kSplit) {
    splits = (int)cg::this_cluster().num_blocks();
    split_rank = (int)cg::this_cluster().block_rank();
    first = blockIdx.x / splits;
    stride = a.m_tiles * a.n_tiles;  // one tile per cluster
    const int per = (a.k_blocks + splits - 1) / splits;
    kb0 = min(a.k_blocks, split_rank * per);
    kb1 = min(a.k_blocks, kb0 + per);
  }
  const int tiles = a.m_tiles * a.n_tiles;

  if (warp == 0) {
    if (lane == 0) {
      prefetch_tensormap(&x_map);
      prefetch_tensormap(&w_map);
      const uint32_t tx = a.x_rows * kBK + BN * kBK;
      int ahead = 0;  // stages whose weights are on their way before the quantized rows are ready
      {
        int m, n;
        if (first < tiles) {
          tile_at(a, first, m, n);
          for (; ahead < STAGES && kb0 + ahead < kb1; ++ahead) {
            mbar_expect_tx(&sm.full[ahead], tx);
            tma_load_2d(sm.w[ahead], &w_map, &sm.full[ahead], (kb0 + ahead) * kBK, n * BN);
          }
        }
      }
      pdl_wait();
      int it = 0;
      bool ok = true;
      for (int i = first; i < tiles && ok; i += stride) {
        int m, n;
        tile_at(a, i, m, n);
        for (int kb = kb0; kb < kb1; ++kb, ++it) {
          const int st = it % STAGES;
          if (it >= ahead) {
            if (!mbar_wait_bounded(&sm.empty[st], ((it / STAGES) & 1) ^ 1)) {
              report_timeout(a);
              ok = false;
              break;
            }
            mbar_expect_tx(&sm.full[st], tx);
            tma_load_2d(sm.w[st], &w_map, &sm.full[st], kb * kBK, n * BN);
          }
          tma_load_2d(sm.x[st], &x_map, &sm.full[st], kb * kBK, m * kBM);
        }
      }
      // no copy may still be in flight when the CTA ends (at once, unless a wait gave up)
      for (int j = it < STAGES ? 0 : it - STAGES; j < it; ++j) mbar_wait_bounded(&sm.full[j % STAGES], (j / STAGES) & 1);
    }
  } else if (warp == 1) {
    if (lane == 0) {
      constexpr uint32_t idesc = make_idesc(kBM, BN);
      int it = 0, acc = 0;
      bool ok = true;
      for (int i = first; i < tiles && ok; i += stride, ++acc) {
        const int ab = acc % kAccBufs;
        if (!mbar_wait_bounded(&sm.acc_empty[ab], ((acc / kAccBufs) & 1) ^ 1)) ok = false;
        tc_fence_after();
        for (int kb = kb0; kb < kb1 && ok; ++kb, ++it) {
          const int st = it % STAGES;
          if (!mbar_wait_bounded(&sm.full[st], (it / STAGES) & 1)) {
            ok = false;
            break;
          }
          tc_fence_after();
          const uint32_t xa = smem_u32(sm.x[st]), wa = smem_u32(sm.w[st]);
#pragma unroll
          for (int kk = 0; kk < kBK / 32; ++kk)
            mma_i8(tmem + ab * BN, make_desc(xa + kk * 32), make_desc(wa + kk * 32), idesc, ((kb - kb0) | kk) != 0);
          mma_commit(&sm.empty[st]);
        }
        if (ok) {
          mma_commit(&sm.acc_full[ab]);
        } else {
          report_timeout(a);
          // a commit's arrival marks every MMA before it complete: none may still
          // write TMEM when it is freed
          mma_commit(&sm.acc_full[ab]);
          mbar_wait_bounded(&sm.acc_full[ab], (acc / kAccBufs) & 1);
        }
      }
    }
  } else {
    const int quarter = warp & 3;  // TMEM lanes 32 * quarter .. + 31
    pdl_wait();                    // the token scales
    int acc = 0;
    for (int i = first; i < tiles; i += stride, ++acc) {
      const int ab = acc % kAccBufs;
      int m, n;
      tile_at(a, i, m, n);
      const int row = m * kBM + quarter * 32 + lane;
      const float xs = row < a.t ? a.xs[row] : 0.f;
      for (int c = (warp - 2) * 32 + lane; c < BN; c += 128) sm.ws[ab][c] = n * BN + c < a.n ? a.ws[n * BN + c] : 0.f;
      if (!epi_all(mbar_wait_bounded(&sm.acc_full[ab], (acc / kAccBufs) & 1))) {
        if (lane == 0) report_timeout(a);
        break;
      }
      tc_fence_after();
      const uint32_t tacc = tmem + ab * BN + ((uint32_t)(quarter * 32) << 16);
      if constexpr (kSplit) {
        // the ring is drained: it holds this CTA's sums, [channel][token]
        int* part = reinterpret_cast<int*>(sm.x[0]);
#pragma unroll 1
        for (int c0 = 0; c0 < BN; c0 += 32) {
          int v[32];
          if (kb1 > kb0) {
            tmem_ld32(tacc + c0, v);
          } else {  // no K blocks left for this CTA: nothing was accumulated
#pragma unroll
            for (int j = 0; j < 32; ++j) v[j] = 0;
          }
#pragma unroll
          for (int j = 0; j < 32; ++j)
            if (row < a.t) part[(c0 + j) * kBM + quarter * 32 + lane] = v[j];
        }
      } else {
#pragma unroll 1
        for (int c0 = 0; c0 < BN; c0 += 32) {
          int v[32];
          tmem_ld32(tacc + c0, v);
          store32<T>(a, v, sm.ws[ab] + c0, xs, row, n * BN + c0);
        }
        tc_fence_before();
        if (lane == 0) mbar_arrive(&sm.acc_empty[ab]);
      }
    }
  }
  if constexpr (kSplit) {
    cg::cluster_group cluster = cg::this_cluster();
    cluster.sync();
    int m, n;
    tile_at(a, first, m, n);
    // Units of 8 channels of 4 tokens; CTA r takes channel octets r, r +
    // splits, ..., its threads tokens innermost.
    const int toks = min(kBM, a.t - m * kBM), quads = (toks + 3) / 4;
    const int octets = (BN / 8 - split_rank + splits - 1) / splits;
    for (int i = threadIdx.x; i < quads * octets; i += kThreads) {
      const int tok = i % quads * 4, c = (split_rank + i / quads * splits) * 8;
      const int n0 = n * BN + c;
      if (n0 >= a.n) continue;
      int v[4][8] = {};
      for (int r = 0; r < splits; ++r) {
        const int* part = cluster.map_shared_rank(reinterpret_cast<int*>(sm.x[0]), r) + c * kBM + tok;
#pragma unroll
        for (int j = 0; j < 8; ++j) {
          const int4 x = *reinterpret_cast<const int4*>(part + j * kBM);
          v[0][j] += x.x;
          v[1][j] += x.y;
          v[2][j] += x.z;
          v[3][j] += x.w;
        }
      }
#pragma unroll
      for (int q = 0; q < 4; ++q) {
        const int row = m * kBM + tok + q;
        if (row >= a.t) break;
        const float xs = a.xs[row];
        T* y = reinterpret_cast<T*>(a.y) + (int64_t)row * a.n + n0;
        if (a.out_vec && n0 + 8 <= a.n) {
          constexpr int N = Vec16<T>::N;
#pragma unroll
          for (int u = 0; u < 8 / N; ++u) {
            Vec16<T> o;
#pragma unroll
            for (int j = 0; j < N; ++j) o.v[j] = from_f32<T>((float)v[q][u * N + j] * (xs * sm.ws[0][c + u * N + j]));
            store16(y + u * N, o);
          }
        } else {
#pragma unroll
          for (int j = 0; j < 8; ++j)
            if (n0 + j < a.n) y[j] = from_f32<T>((float)v[q][j] * (xs * sm.ws[0][c + j]));
        }
      }
    }
    cluster.sync();  // no CTA's shared memory goes away while another reads it
  }
  tc_fence_before();
  __syncthreads();
  if (warp == 1) {
    tc_fence_after();
    asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(kCols));
  }
}

// Large products: two SMs on one 256 x 256 tile (cta_group::2).  Each CTA of
// the pair holds half of the tokens (MMA M) and half of the channels (N) in its
// shared memory; one MMA reads both, so a byte of weights is fetched by one SM
// for 256 tokens instead of 128, which is what bounds the one-CTA kernel: its
// tensor pipe is fed 58 B per clock and SM where it could take 94.  CTA 0 issues
// the MMAs; both CTAs' copies complete on its barriers, and its commits signal
// both.  Each CTA has its 128 tokens x 256 channels in its own TMEM.
AFD_DEVICE uint32_t leader_addr(const void* p) {  // the same object in CTA 0 of the cluster
  uint32_t a;
  asm("mapa.shared::cluster.u32 %0, %1, 0;" : "=r"(a) : "r"(smem_u32(p)));
  return a;
}
AFD_DEVICE void tma_pair(void* dst, const CUtensorMap* map, uint32_t bar, int x, int y) {
  asm volatile(
      "cp.async.bulk.tensor.2d.cta_group::2.shared::cluster.global.tile.mbarrier::complete_tx::bytes [%0], [%1, {%3, "
      "%4}], [%2];" ::"r"(smem_u32(dst)),
      "l"(map), "r"(bar), "r"(x), "r"(y)
      : "memory");
}
AFD_DEVICE void mma_pair(uint32_t tmem_d, uint64_t adesc, uint64_t bdesc, uint32_t idesc, uint32_t accumulate) {
  asm volatile(
      "{\n .reg .pred p;\n setp.ne.b32 p, %4, 0;\n"
      " tcgen05.mma.cta_group::2.kind::i8 [%0], %1, %2, %3, p;\n}\n" ::"r"(tmem_d),
      "l"(adesc), "l"(bdesc), "r"(idesc), "r"(accumulate));
}
AFD_DEVICE void commit_pair(uint64_t* bar) {  // arrives on this barrier of both CTAs
  asm volatile(
      "tcgen05.commit.cta_group::2.mbarrier::arrive::one.shared::cluster.multicast::cluster.b64 [%0], %1;" ::"r"(
          smem_u32(bar)),
      "h"((uint16_t)3)
      : "memory");
}

constexpr int kPairStages = 6;

template <typename T>
__global__ void __launch_bounds__(kThreads, 1) gemm_pair_kernel(const __grid_constant__ CUtensorMap x_map,
                                                                const __grid_constant__ CUtensorMap w_map,
                                                                const Args a) {
  constexpr int BN = 256, STAGES = kPairStages;
  struct SmemT {
    alignas(1024) uint8_t x[STAGES][kXBytes];
    alignas(1024) uint8_t w[STAGES][BN / 2 * kBK];
    alignas(16) float ws[2][BN];
    uint64_t full[STAGES];
    uint64_t empty[STAGES];
    uint64_t acc_full[2];
    uint64_t acc_empty[2];
    uint32_t tmem_base;
  };
  static_assert(sizeof(SmemT) == kPairSmem, "the launcher's size");
  extern __shared__ uint8_t smem_raw[];
  SmemT& sm = *reinterpret_cast<SmemT*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  cg::cluster_group cluster = cg::this_cluster();
  const int rank = (int)cluster.block_rank();
  const int warp = threadIdx.x / 32, lane = threadIdx.x & 31;
  if (threadIdx.x == 0) {
    for (int s = 0; s < STAGES; ++s) {
      mbar_init(&sm.full[s], 1);
      mbar_init(&sm.empty[s], 1);
    }
    for (int b = 0; b < 2; ++b) {
      mbar_init(&sm.acc_full[b], 1);
      mbar_init(&sm.acc_empty[b], 8);  // the epilogue warps of both CTAs
    }
    fence_barrier_init();
  }
  if (warp == 1) {
    asm volatile("tcgen05.alloc.cta_group::2.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(&sm.tmem_base)),
                 "r"(2 * BN));
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::2.sync.aligned;");
  }
  tc_fence_before();
  cluster.sync();  // barriers and TMEM of both CTAs are ready
  tc_fence_after();
  const uint32_t tmem = sm.tmem_base;
  const int tiles = a.m_tiles * a.n_tiles, first = blockIdx.x / 2, stride = gridDim.x / 2;

  if (warp == 0) {
    if (lane == 0) {
      prefetch_tensormap(&x_map);
      prefetch_tensormap(&w_map);
      constexpr uint32_t tx = 2 * (kXBytes + BN / 2 * kBK);  // both CTAs' halves
      int ahead = 0;  // stages whose weights are on their way before the quantized rows are ready
      if (first < tiles) {
        int m, n;
        tile_at(a, first, m, n);
        for (; ahead < STAGES && ahead < a.k_blocks; ++ahead) {
          if (rank == 0) mbar_expect_tx(&sm.full[ahead], tx);
          tma_pair(sm.w[ahead], &w_map, leader_addr(&sm.full[ahead]), ahead * kBK, n * BN + rank * (BN / 2));
        }
      }
      pdl_wait();
      int it = 0;
      bool ok = true;
      for (int i = first; i < tiles && ok; i += stride) {
        int m, n;
        tile_at(a, i, m, n);
        for (int kb = 0; kb < a.k_blocks; ++kb, ++it) {
          const int st = it % STAGES;
          const uint32_t bar = leader_addr(&sm.full[st]);
          if (it >= ahead) {
            if (!mbar_wait_bounded(&sm.empty[st], ((it / STAGES) & 1) ^ 1)) {
              report_timeout(a);
              ok = false;
              break;
            }
            if (rank == 0) mbar_expect_tx(&sm.full[st], tx);
            tma_pair(sm.w[st], &w_map, bar, kb * kBK, n * BN + rank * (BN / 2));
          }
          tma_pair(sm.x[st], &x_map, bar, kb * kBK, (2 * m + rank) * kBM);
        }
      }
      // no copy of either CTA may still be in flight when they end (at once, unless a wait gave up)
      if (rank == 0)
        for (int j = it < STAGES ? 0 : it - STAGES; j < it; ++j)
          mbar_wait_bounded(&sm.full[j % STAGES], (j / STAGES) & 1);
    }
  } else if (warp == 1) {
    if (lane == 0 && rank == 0) {
      constexpr uint32_t idesc = make_idesc(2 * kBM, BN);
      int it = 0, acc = 0;
      bool ok = true;
      for (int i = first; i < tiles && ok; i += stride, ++acc) {
        const int ab = acc % 2;
        if (!mbar_wait_bounded(&sm.acc_empty[ab], ((acc / 2) & 1) ^ 1)) ok = false;
        tc_fence_after();
        for (int kb = 0; kb < a.k_blocks && ok; ++kb, ++it) {
          const int st = it % STAGES;
          if (!mbar_wait_bounded(&sm.full[st], (it / STAGES) & 1)) {
            ok = false;
            break;
          }
          tc_fence_after();
          const uint32_t xa = smem_u32(sm.x[st]), wa = smem_u32(sm.w[st]);
#pragma unroll
          for (int kk = 0; kk < kBK / 32; ++kk)
            mma_pair(tmem + ab * BN, make_desc(xa + kk * 32), make_desc(wa + kk * 32), idesc, (kb | kk) != 0);
          commit_pair(&sm.empty[st]);
        }
        commit_pair(&sm.acc_full[ab]);
        if (!ok) {
          report_timeout(a);
          mbar_wait_bounded(&sm.acc_full[ab], (acc / 2) & 1);  // no MMA may still write TMEM when it is freed
        }
      }
    }
  } else {
    const int quarter = warp & 3;  // TMEM lanes 32 * quarter .. + 31
    pdl_wait();                    // the token scales
    int acc = 0;
    for (int i = first; i < tiles; i += stride, ++acc) {
      const int ab = acc % 2;
      int m, n;
      tile_at(a, i, m, n);
      const int row = (2 * m + rank) * kBM + quarter * 32 + lane;
      const float xs = row < a.t ? a.xs[row] : 0.f;
      for (int c = (warp - 2) * 32 + lane; c < BN; c += 128) sm.ws[ab][c] = n * BN + c < a.n ? a.ws[n * BN + c] : 0.f;
      if (!epi_all(mbar_wait_bounded(&sm.acc_full[ab], (acc / 2) & 1))) {
        if (lane == 0) report_timeout(a);
        break;
      }
      tc_fence_after();
      const uint32_t tacc = tmem + ab * BN + ((uint32_t)(quarter * 32) << 16);
#pragma unroll 1
      for (int c0 = 0; c0 < BN; c0 += 32) {
        int v[32];
        tmem_ld32(tacc + c0, v);
        store32<T>(a, v, sm.ws[ab] + c0, xs, row, n * BN + c0);
      }
      tc_fence_before();
      if (lane == 0)
        asm volatile("mbarrier.arrive.release.cluster.shared::cluster.b64 _, [%0];" ::"r"(leader_addr(&sm.acc_empty[ab]))
                     : "memory");
    }
  }
  tc_fence_before();
  cluster.sync();  // neither CTA's shared memory or TMEM goes away while the other uses it
  if (warp == 1) {
    tc_fence_after();
    asm volatile("tcgen05.dealloc.cta_group::2.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(2 * BN));
  }
}

bool encode(CUtensorMap* map, const void* base, int64_t rows, int k, int box_rows) {
  const cuuint64_t dims[2] = {(cuuint64_t)k, (cuuint64_t)rows};
  const cuuint64_t strides[1] = {(cuuint64_t)k};
  const cuuint32_t box[2] = {kBK, (cuuint32_t)box_rows};
  const cuuint32_t estr[2] = {1, 1};
  return get_tensor_map_encoder()(map, CU_TENSOR_MAP_DATA_TYPE_UINT8, 2, const_cast<void*>(base), dims, strides, box,
                                  estr, CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B,
                                  CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
                                  CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}

template <typename T, int BN, int STAGES, bool kSplit>
cudaError_t launch(const Int8GemmParams& p, Args a, int splits, cudaStream_t s) {
  a.n_tiles = (p.n + BN - 1) / BN;
  CUtensorMap xm, wm;
  if (!encode(&xm, p.xq, p.t, p.k, a.x_rows) || !encode(&wm, p.w, p.n, p.k, BN)) return cudaErrorInvalidValue;
  auto* kernel = gemm_kernel<T, BN, STAGES, kSplit>;
  const size_t smem = sizeof(Smem<BN, STAGES>) + 1024;
  static PerDeviceOnce attr;
  cudaError_t e = attr.run([&] {
    return cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)smem);
  });
  if (e != cudaSuccess) return e;
  const int64_t tiles = (int64_t)a.m_tiles * a.n_tiles;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3((unsigned)(kSplit ? tiles * splits : tiles < device_sm_count() ? tiles : device_sm_count()));
  cfg.blockDim = dim3(kThreads);
  cfg.dynamicSmemBytes = smem;
  cfg.stream = s;
  cudaLaunchAttribute at[2];
  at[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  at[0].val.programmaticStreamSerializationAllowed = pdl_enabled() ? 1 : 0;
  at[1].id = cudaLaunchAttributeClusterDimension;
  at[1].val.clusterDim.x = splits;
  at[1].val.clusterDim.y = at[1].val.clusterDim.z = 1;
  cfg.attrs = at;
  cfg.numAttrs = kSplit ? 2 : 1;
  return cudaLaunchKernelEx(&cfg, kernel, xm, wm, a);
}

template <typename T>
cudaError_t launch_pair(const Int8GemmParams& p, Args a, cudaStream_t s) {
  a.m_tiles = (p.t + 2 * kBM - 1) / (2 * kBM);
  a.n_tiles = (p.n + 255) / 256;
  a.band = (a.band + 1) / 2;
  a.x_rows = kBM;
  CUtensorMap xm, wm;
  if (!encode(&xm, p.xq, p.t, p.k, kBM) || !encode(&wm, p.w, p.n, p.k, 128)) return cudaErrorInvalidValue;
  auto* kernel = gemm_pair_kernel<T>;
  const size_t smem = kPairSmem + 1024;
  static PerDeviceOnce attr;
  cudaError_t e = attr.run([&] {
    return cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)smem);
  });
  if (e != cudaSuccess) return e;
  const int64_t tiles = (int64_t)a.m_tiles * a.n_tiles;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3((unsigned)(2 * std::min<int64_t>(tiles, device_sm_count() / 2)));
  cfg.blockDim = dim3(kThreads);
  cfg.dynamicSmemBytes = smem;
  cfg.stream = s;
  cudaLaunchAttribute at[2];
  at[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  at[0].val.programmaticStreamSerializationAllowed = pdl_enabled() ? 1 : 0;
  at[1].id = cudaLaunchAttributeClusterDimension;
  at[1].val.clusterDim.x = 2;
  at[1].val.clusterDim.y = at[1].val.clusterDim.z = 1;
  cfg.attrs = at;
  cfg.numAttrs = 2;
  return cudaLaunchKernelEx(&cfg, kernel, xm, wm, a);
}

template <typename T>
cudaError_t run(const Int8GemmParams& p, cudaStream_t s) {
  Args a{};
  a.y = p.y;
  a.xs = p.xs;
  a.ws = p.ws;
  a.status = p.status;
  a.t = p.t;
  a.n = p.n;
  a.k_blocks = (p.k + kBK - 1) / kBK;
  a.m_tiles = (p.t + kBM - 1) / kBM;
  a.x_rows = p.t < kBM ? (p.t + 7) / 8 * 8 : kBM;
  a.out_vec = (int64_t)p.n * sizeof(T) % 16 == 0 && reinterpret_cast<uintptr_t>(p.y) % 16 == 0;
  const int64_t fit = (int64_t)48 << 20;  // token rows of a band: well inside L2
  a.band = (int)(fit / ((int64_t)kBM * p.k));
  a.band = a.band < 1 ? 1 : (a.band > a.m_tiles ? a.m_tiles : a.band);
  const int sms = device_sm_count();
  // Enough 256 x 256 tiles for every pair of SMs: 832 us against 928 with one SM
  // a tile at 4099 x 36864 x 7168, 2.6 POPS (twice the bf16 rate that cuBLAS
  // sustains there is 2.8).  With at most 128 tokens half a pair would idle.
  if (a.m_tiles > 1 && (int64_t)((a.m_tiles + 1) / 2) * ((p.n + 255) / 256) >= sms / 2) return launch_pair<T>(p, a, s);
  if ((int64_t)a.m_tiles * ((p.n + 255) / 256) >= sms) return launch<T, 256, 4, false>(p, a, 1, s);
  // Fewer tiles than SMs.  A long contraction is split over a cluster (a share
  // of at least 16 stages: shorter ones cost more to add up than they save); a
  // short one takes narrower tiles.  Measured: 256 x 2048 x 10944, 30.2, 23.1
  // and 17.6 us with 1, 2 and 4 shares; 5 x 5120 x 2048, 8.3 us with 64-wide
  // tiles, 8.7 with 128-wide ones, 9.5 and 13.2 with those in 2 and 4 shares.
  const int tiles = a.m_tiles * ((p.n + 127) / 128);
  const int splits = std::min({8, sms / tiles, a.k_blocks / 16});
  if (splits > 1) return launch<T, 128, 6, true>(p, a, splits, s);
  if (2 * tiles <= sms) return launch<T, 64, 6, false>(p, a, 1, s);
  return launch<T, 128, 6, false>(p, a, 1, s);
}

}  // namespace i8
}  // namespace afd

using namespace afd;

int launch_int8_quantize(int8_t* q, float* scale, const void* x, int64_t ld, int t, int k, int vec, int dtype,
                         cudaStream_t s) {
  switch (dtype) {
    case kF32: i8::quantize_kernel<float><<<t, i8::kQThreads, 0, s>>>(q, scale, (const float*)x, ld, k, vec); break;
    case kF16: i8::quantize_kernel<__half><<<t, i8::kQThreads, 0, s>>>(q, scale, (const __half*)x, ld, k, vec); break;
    default:
      i8::quantize_kernel<__nv_bfloat16><<<t, i8::kQThreads, 0, s>>>(q, scale, (const __nv_bfloat16*)x, ld, k, vec);
  }
  return (int)cudaGetLastError();
}

int launch_int8_gemm(const Int8GemmParams& p, int dtype, cudaStream_t s) {
  switch (dtype) {
    case kF32: return (int)i8::run<float>(p, s);
    case kF16: return (int)i8::run<__half>(p, s);
    default: return (int)i8::run<__nv_bfloat16>(p, s);
  }
}
