// Grouped-query paged decode over the 4-bit KV cache (layout: kv_int4.cuh).
//
//   s[h, t] = scale * q_h . k_t        k_t = zk_t + ck_t * stepk_t   per 64 dims
//   o_h     = sum_t softmax_t(s[h, :]) v_t
//
// With codes shifted to c - 8 (and zero to zero + 8 step) the products split:
//   q . k_t = sum_groups step_t,j * (q_j . c_t,j) + zero_t,j * sum(q_j)
//   o       = sum_groups (p_t step_t,j) c_t,j + p_t zero_t,j
// so the tensor cores multiply q (scaled by a power of two per head, exact in
// fp16) and p * step (rounded to fp16's 11 bits, or 22 for fp16 results, see
// take_tiles) with small integers, and the scales stay outside in fp32, as do
// the running maximum and sum.
//
// What bounds it: the floor is the packed rows, 144 B per position and KV head
// at D = 128, at the HBM rate; what it spends is the latency of about 400
// instructions a 16-position tile, a third of them the unpacking of codes, at
// 12 warps per SM (2.4 instructions a clock of 4; the logic pipe is half busy,
// the tensor pipe a fifth).  16 sequences of 50 - 131 K positions, 32 query
// heads on 4 KV heads of 128, bf16: 835 MB in 215 us, 3.9 TB/s, 59% of the
// measured copy bandwidth (64% inside the kernel).
//
// A warp unpacks the codes it needs straight into MMA operand registers, so
// the tile is the A operand (16 positions x 16 dims, or 16 dims x 16
// positions) and the query heads are the 8 columns of B: a group of 8 query
// heads needs half the MMAs that padding the heads to 16 rows would.  Each
// warp owns whole tiles: a private ring of cp.async stages, no block barrier
// in the loop, running maximum and sum per warp; the warps of a CTA merge once
// at the end, while the next piece's tiles are on their way.
//
// Work split: a tile is 16 positions of one (sequence, KV head).  All tiles of
// the batch, in (sequence, head, position) order, are dealt to one wave of
// CTAs in equal contiguous shares, whatever the lengths; a share that covers
// part of a (sequence, head) leaves a partial (unnormalised o, max, sum) that
// a second small kernel joins.  Short tables take one CTA per (sequence, head)
// instead and write the result at once: one launch (kv4_decode_plan).
//
// Scores: the decode leaves its logits, and a small kernel adds each position's
// probability under the joined log-sum-exp, summed over the group's query
// heads, to its score.  Batches whose logits would take more than 512 MB read K
// once more instead.  Beside the decode alone the two cost 4.3 and 13.9 us at
// 16 sequences of 0.8 - 2 K positions (16 heads on 16), 13.0 and 17.7 us at 4
// of 20 - 33 K (64 on 4).
#include <algorithm>
#include <cfloat>
#include <type_traits>

#include "device_state.h"
#include "kv_int4.cuh"
#include "launchers.h"

namespace afd {
namespace kv4 {

constexpr int kTile = 16;
constexpr int kWarps = 4;
constexpr int kStages = 3;       // of kTiles tiles each
constexpr int kScoreStages = 4;  // of one tile's K
constexpr int kDecThreads = kWarps * 32;
constexpr int kMaxBatch = 256;       // sequences per launch (their prefix sums sit in shared memory)
constexpr float kLowest = -FLT_MAX;  // a maximum before any logit: finite, so that differences stay defined
constexpr float kStepTop = 512.f;    // scaled steps stay below this (times 2^kLazy: fp16 factors below 2^15)
constexpr int kScaleTop = 117;       // steps of 2^-108 and more set their own scale, smaller ones keep 2^117
constexpr float kLazy = 6.f;         // the running maximum moves when it is exceeded by 2^6
// What a piece costs beside its tiles (pipeline fill, query, merge), in tiles,
// and the steps of all warps that tiles come in.  Measured at 256 sequences of
// 1 - 4001 positions, D = 256: 119, 107, 101 and 97 us with 4, 10, 16 and 24;
// at 16 of 2050 and of 50 - 131 K positions 10 and more are alike.
constexpr int kPieceCost = 16;
constexpr int kRound = 8;
constexpr int kMinShare = 8;         // a CTA's share of tiles is not cut below this

template <int D>
struct Ring {
  static constexpr int G = D / kGroup;
  static constexpr int kCodes = kTile * D / 2;  // bytes of one tile's codes
  static constexpr int kPairs = kTile * G * 4;
  static constexpr int kHalf = kCodes + kPairs;  // K codes, K pairs; then the same of V
  static constexpr int kStageBytes = 2 * kHalf;
};

// 16-byte chunk of a row of codes -> chunk in shared memory.  The MMA operand
// loads of one instruction touch rows {0, 1, 2, 3}, {4, .., 7} (V) or
// {0, 4, 1, 5}, {2, 6, 3, 7} (K); this spreads each set over all banks.  Dim
// group j is reached by an XOR with 32 j, row r + 4 by one with kRow4.
template <int D>
AFD_DEVICE constexpr int swz(int row, int chunk) {
  if (D == 256) return chunk ^ (((row & 3) ^ ((row >> 1) & 2)) << 1);
  if (D == 128) return chunk ^ ((((row >> 1) ^ (row >> 2)) & 1) << 1);
  return chunk;
}
// Tiles a warp takes at once: two where the registers allow it, so that their
// chains of dependent operations interleave.
template <int D, int NT> constexpr int kTiles = D * NT <= 128 ? 2 : 1;
// CTAs one SM holds (their registers bound it).  At 16 sequences of 50 - 131 K
// positions and D = 128, four CTAs of one tile a step in 128 registers took
// 239 us, three in 168 registers 220 us.
template <int D, int NT> constexpr int kResident = D * NT <= 128 ? 3 : 2;
// Row lengths of query heads and of results in shared memory, padded so that
// the lanes of one access fall on different banks.
template <int D> constexpr int kQueryLd = D + 8;
template <int D> constexpr int kRedLd = D + 4;
template <int D> constexpr int kRow4 = D == 256 ? 64 : (D == 128 ? 32 : 0);

// The 8 codes of a word as fp16 pairs c - 8: v[i] = codes i and i + 4.  OR-ing
// a code into the mantissa of 1024 adds it (or 16 times it, from the nibble
// above); one multiply-add brings it down, exactly.  Masks and base come from
// the kernel's parameters: as literals they would cost two logic operations
// each instead of one (an instruction takes one literal).
struct Unpack {
  uint32_t lo, hi, base;
  AFD_DEVICE void operator()(uint32_t (&v)[4], uint32_t w) const {
    const uint32_t x = w >> 8;
    v[0] = sub((w & lo) | base);
    v[1] = down((w & hi) | base);
    v[2] = sub((x & lo) | base);
    v[3] = down((x & hi) | base);
  }
  static AFD_DEVICE uint32_t sub(uint32_t m) {
    const __half2 v = __hsub2(*reinterpret_cast<const __half2*>(&m), __floats2half2_rn(1032.f, 1032.f));
    return *reinterpret_cast<const uint32_t*>(&v);
  }
  static AFD_DEVICE uint32_t down(uint32_t m) {
    const __half2 v = __hfma2(*reinterpret_cast<const __half2*>(&m), __floats2half2_rn(0.0625f, 0.0625f),
                              __floats2half2_rn(-72.f, -72.f));
    return *reinterpret_cast<const uint32_t*>(&v);
  }
};

AFD_DEVICE void mma_f16(float (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1) {
  asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
      : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
      : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}
AFD_DEVICE uint32_t pack_f16(float lo, float hi) {
  const __half2 v = __floats2half2_rn(lo, hi);
  return *reinterpret_cast<const uint32_t*>(&v);
}
// x's binary exponent, from the encoding, as -112 .. 127: 2^(5 - it), 2^(14 - it)
// and their inverses are normal numbers, for subnormal and infinite x too.
AFD_DEVICE int exponent_of(float x) { return min(max((int)(__float_as_uint(x) >> 23) & 255, 15), 254) - 127; }
AFD_DEVICE float pow2(int e) { return __uint_as_float((uint32_t)(e + 127) << 23); }

// 8x8 transpose of 16-bit values held one row pair per lane.
AFD_DEVICE uint32_t transpose8(uint32_t v) {
  uint32_t d;
  asm("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(d) : "r"(v));
  return d;
}
AFD_DEVICE float fast_exp2(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}
AFD_DEVICE void cp16(uint32_t dst, const void* src) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(dst), "l"(src) : "memory");
}
AFD_DEVICE void cp_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int N> AFD_DEVICE void cp_wait() { asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory"); }
AFD_DEVICE void lds64(uint32_t& a, uint32_t& b, uint32_t addr) {
  asm volatile("ld.shared.v2.u32 {%0, %1}, [%2];" : "=r"(a), "=r"(b) : "r"(addr));
}
AFD_DEVICE uint32_t lds32(uint32_t addr) {
  uint32_t a;
  asm volatile("ld.shared.u32 %0, [%1];" : "=r"(a) : "r"(addr));
  return a;
}
template <int G>
AFD_DEVICE void lds_pairs(uint32_t (&v)[G], uint32_t addr) {  // one position's (step, zero) pairs
  if constexpr (G == 1) {
    v[0] = lds32(addr);
  } else if constexpr (G == 2) {
    lds64(v[0], v[1], addr);
  } else {
    asm volatile("ld.shared.v4.u32 {%0, %1, %2, %3}, [%4];"
                 : "=r"(v[0]), "=r"(v[1]), "=r"(v[2]), "=r"(v[3])
                 : "r"(addr));
  }
}

// Sequence length as the kernels use it: never negative, never past the table.
AFD_DEVICE int seq_len_of(const Kv4DecodeParams& p, int b) {
  const int n = p.seq_lens[b];
  return n < 0 ? 0 : min(n, p.max_blocks * p.block_size);
}

// Row of a tile that MMA row (or k index) i stands for: rows are taken in the
// order 0 4 1 5 2 6 3 7 (+ 8), which keeps both operands' loads conflict-free.
AFD_DEVICE int tile_row(int i) { return (i & 8) | ((i & 7) >> 1) | ((i & 1) << 2); }

AFD_DEVICE int tiles_of(int n) { return (n + kTile - 1) / kTile; }
// Length of a (sequence, head chunk) in the order the shares are cut from.
AFD_DEVICE int cost_of(int tiles) { return tiles > 0 ? (tiles + kRound - 1) / kRound * kRound + kPieceCost : 0; }

// Inclusive prefix sums of the sequences' costs into cum[1 .. batch]
// (cum[0] = 0); every thread of the block calls this.
AFD_DEVICE void cost_prefix(const Kv4DecodeParams& p, int* cum, int* warp_sums) {
  const int lane = threadIdx.x & 31, warp = threadIdx.x / 32, nw = blockDim.x / 32;
  int carry = 0;
  if (threadIdx.x == 0) cum[0] = 0;
  for (int b0 = 0; b0 < p.batch; b0 += blockDim.x) {
    const int b = b0 + threadIdx.x;
    int v = b < p.batch ? cost_of(tiles_of(seq_len_of(p, b))) : 0;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const int u = __shfl_up_sync(0xffffffffu, v, o);
      if (lane >= o) v += u;
    }
    if (lane == 31) warp_sums[warp] = v;
    __syncthreads();
    int before = carry, total = 0;
    for (int w = 0; w < nw; ++w) {
      if (w < warp) before += warp_sums[w];
      total += warp_sums[w];
    }
    if (b < p.batch) cum[b + 1] = before + v;
    carry += total;
    __syncthreads();
  }
  __syncthreads();
}

// The share of the batch's cost a CTA takes (the same expression wherever it is
// needed).  One wave of CTAs: two or four waves of shorter shares measured 2 and
// 11% slower at 16 sequences of 50 - 131 K positions, each CTA's start costing
// more than the evener finish gains.
AFD_DEVICE int64_t share_of(int64_t total, int ctas) {
  const int64_t s = (total + ctas - 1) / ctas;
  return s < kMinShare + kPieceCost ? kMinShare + kPieceCost : s;
}

// One piece: tiles [t0, t1) of (sequence b, head chunk hv).
struct Piece {
  int b, hv, t0, t1, tiles;
  int64_t next;  // where the next piece starts
};

// The piece that starts at position `at` of the batch's order and ends at `end`
// or at its (sequence, head)'s end.  It may hold no tile (t0 == t1), when only
// a (sequence, head)'s fixed cost fell into the share.
AFD_DEVICE Piece piece_at(const Kv4DecodeParams& p, const int* cum, int heads_v, int64_t at, int64_t end) {
  int lo = 0, hi = p.batch - 1;  // largest b with cum[b] * heads_v <= at
  while (lo < hi) {
    const int mid = (lo + hi + 1) >> 1;
    if ((int64_t)cum[mid] * heads_v <= at) lo = mid;
    else hi = mid - 1;
  }
  const int cost = cum[lo + 1] - cum[lo];
  const int64_t rem = at - (int64_t)cum[lo] * heads_v;
  Piece pc;
  pc.b = lo;
  pc.hv = (int)(rem / cost);
  const int v0 = (int)(rem - (int64_t)pc.hv * cost);
  const int v1 = (int)min((int64_t)cost, v0 + (end - at));
  pc.tiles = tiles_of(seq_len_of(p, lo));
  pc.t0 = min(pc.tiles, max(0, v0 - kPieceCost));
  pc.t1 = min(pc.tiles, max(0, v1 - kPieceCost));
  pc.next = at + (v1 - v0);
  return pc;
}

// A warp's walk over the tiles of one (sequence, KV head) in the cache: U
// neighbouring tiles from `first` on, then those U * kWarps further, and so on.
// Block ids are fetched one step ahead.
template <int D, int U>
struct TileWalk {
  const uint8_t *kc, *vc, *sc;  // this lane's bytes of the head's first row: K codes, V codes, pairs
  const int32_t* table;
  uint32_t block_codes, block_pairs;  // bytes of a block's codes and pairs
  int pg, in, per_block, last_block, blk[U];

  AFD_DEVICE void start(const Kv4DecodeParams& p, int b, int kv_head, int first, int lane) {
    table = p.block_table + (int64_t)b * p.table_stride;
    last_block = p.num_blocks - 1;
    const uint32_t rows = (uint32_t)kv_head * p.block_size;
    kc = p.k_codes + (size_t)rows * (D / 2) + lane * 16;
    vc = p.v_codes + (size_t)rows * (D / 2) + lane * 16;
    // the lower half warp copies K's pairs, the upper half V's
    sc = reinterpret_cast<const uint8_t*>(lane < 16 ? p.k_scale : p.v_scale) + (size_t)rows * (D / kGroup * 4) +
         (lane & 15) * 16;
    block_codes = (uint32_t)p.kv_heads * p.block_size * (D / 2);
    block_pairs = (uint32_t)p.kv_heads * p.block_size * (D / kGroup * 4);
    per_block = p.block_size / kTile;
    pg = first / per_block;
    in = first - pg * per_block;
  }
  // Page and place in it of the step's u-th tile.
  AFD_DEVICE void at(int u, int& page, int& place) const {
    const bool over = in + u >= per_block;  // u <= 1
    page = pg + over;
    place = over ? in + u - per_block : in + u;
  }
  // Reads the block ids of the step's first `n` tiles (see check_blocks for bad ones).
  AFD_DEVICE void fetch(int n) {
#pragma unroll
    for (int u = 0; u < U; ++u) {
      int page, place;
      at(u, page, place);
      if (u < n) blk[u] = (int)min((unsigned)table[page], (unsigned)last_block);
    }
  }
  AFD_DEVICE void advance() {
    in += U * kWarps;
    while (in >= per_block) {
      in -= per_block;
      ++pg;
    }
  }
  // `dst`: this lane's swizzled place in a stage (Places::cp).
  template <bool kWithV>
  AFD_DEVICE void load(int u, uint32_t stage, uint32_t dst, int lane) const {
    using R = Ring<D>;
    int page, place;
    at(u, page, place);
    const size_t off = (size_t)blk[u] * block_codes + (uint32_t)(place * R::kCodes);
#pragma unroll
    for (int i = 0; i < R::kCodes / 512; ++i) {
      // 32 chunks on: the row grows by 8 (D = 128) or 4 (D = 256)
      const uint32_t to = stage + ((D == 256 && (i & 1)) ? dst ^ 64u : dst) + i * 512;
      cp16(to, kc + off + i * 512);
      if (kWithV) cp16(to + R::kHalf, vc + off + i * 512);
    }
    if ((lane & 15) < R::kPairs / 16 && (kWithV || lane < 16))
      cp16(stage + R::kCodes + (lane < 16 ? 0 : R::kHalf) + (lane & 15) * 16,
           sc + (size_t)blk[u] * block_pairs + (uint32_t)(place * R::kPairs));
  }
};

// Reports block ids of tiles [t0, t1) that lie outside the pool (the walk reads
// the pool's last block in their place).
AFD_DEVICE void check_blocks(const Kv4DecodeParams& p, int b, int t0, int t1) {
  const int32_t* table = p.block_table + (int64_t)b * p.table_stride;
  const int per_block = p.block_size / kTile;
  for (int pg = t0 / per_block + (int)threadIdx.x; pg * per_block < t1; pg += kDecThreads)
    if ((unsigned)table[pg] >= (unsigned)p.num_blocks && p.status != nullptr) atomicExch(p.status, kStatusBadIndex);
}

// Where this lane copies to and reads from inside a stage.
template <int D>
struct Places {
  uint32_t cp, k, v, pair;
  AFD_DEVICE explicit Places(int lane) {
    constexpr int kChunks = D / 32;
    const int g = lane >> 2, c = lane & 3, r0 = tile_row(g);
    cp = lane / kChunks * (D / 2) + swz<D>(lane / kChunks, lane % kChunks) * 16;
    k = r0 * (D / 2) + swz<D>(r0, c >> 1) * 16 + (c & 1) * 8;
    v = Ring<D>::kHalf + c * (D / 2) + swz<D>(c, g >> 2) * 16 + (g & 3) * 4;
    pair = Ring<D>::kCodes + r0 * (D / kGroup) * 4;
  }
};

// The query heads of one chunk as B operands, and their sums per dim group.
// Column n of tile t is head t * 8 + n of the chunk (zero beyond `heads`).
// Each head is scaled by a power of two, its largest value to [2^14, 2^15):
// a bf16 value fits fp16 exactly then, down to 2^-31 of the head's largest
// (an fp16 one down to 2^-28).
template <typename T, int D, int NT>
struct Query {
  static constexpr int G = D / kGroup;
  uint32_t f[NT][G * 4][2];
  float sum[NT][G][2];  // of heads 2c, 2c + 1, times scale * log2(e)
  float unit[NT][2];    // what one unit of the scaled q . codes stands for, in the same

  AFD_DEVICE void load(const T* sq, float scale_log2, int lane) {
    const int g = lane >> 2, c = lane & 3;
#pragma unroll
    for (int t = 0; t < NT; ++t) {
      const T* row = sq + (t * 8 + g) * kQueryLd<D> + c * 16;
      float amax = 0.f;
#pragma unroll
      for (int j = 0; j < G; ++j) {
        Vec16<T> x[2];
        x[0] = load16(row + j * kGroup);
        x[1] = load16(row + j * kGroup + 8);
        float acc = 0.f;
#pragma unroll
        for (int i = 0; i < 16; ++i) {
          const float v = to_f32(x[i >> 3].v[i & 7]);
          acc += v;
          amax = fmaxf(amax, fabsf(v));
        }
        acc += __shfl_xor_sync(0xffffffffu, acc, 1);
        acc += __shfl_xor_sync(0xffffffffu, acc, 2);
        acc *= scale_log2;
        sum[t][j][0] = __shfl_sync(0xffffffffu, acc, c * 8);
        sum[t][j][1] = __shfl_sync(0xffffffffu, acc, c * 8 + 4);
      }
      amax = fmaxf(amax, __shfl_xor_sync(0xffffffffu, amax, 1));
      amax = fmaxf(amax, __shfl_xor_sync(0xffffffffu, amax, 2));
      const int e = 14 - exponent_of(amax);
      const float up = pow2(e), down = pow2(-e) * scale_log2;
      unit[t][0] = __shfl_sync(0xffffffffu, down, c * 8);
      unit[t][1] = __shfl_sync(0xffffffffu, down, c * 8 + 4);
#pragma unroll
      for (int j = 0; j < G; ++j) {
#pragma unroll
        for (int w = 0; w < 2; ++w) {  // the lane's word w, code pairs 0 .. 3
          const Vec16<T> x = load16(row + j * kGroup + w * 8);
          float v[8];
#pragma unroll
          for (int i = 0; i < 8; ++i) v[i] = to_f32(x.v[i]) * up;
          f[t][j * 4 + w * 2][0] = pack_f16(v[0], v[4]);
          f[t][j * 4 + w * 2][1] = pack_f16(v[1], v[5]);
          f[t][j * 4 + w * 2 + 1][0] = pack_f16(v[2], v[6]);
          f[t][j * 4 + w * 2 + 1][1] = pack_f16(v[3], v[7]);
        }
      }
    }
  }
};

// s[t][i] for this lane: rows tile_row(g) (i = 0, 1) and tile_row(g) + 8
// (i = 2, 3), heads t * 8 + 2c + (i & 1); in the log2 domain.
template <typename T, int D, int NT>
AFD_DEVICE void tile_logits(float (&s)[NT][4], const Query<T, D, NT>& q, uint32_t stage, const Places<D>& at,
                            const Unpack& codes, uint32_t shl16) {
  constexpr int G = D / kGroup;
  uint32_t p0[G], p1[G];
  lds_pairs<G>(p0, stage + at.pair);
  lds_pairs<G>(p1, stage + at.pair + 8 * G * 4);
  float z[NT][4];
#pragma unroll
  for (int j = 0; j < G; ++j) {
    uint32_t w0[2], w1[2];
    const uint32_t from = (stage + at.k) ^ (j * 32);
    lds64(w0[0], w0[1], from);
    lds64(w1[0], w1[1], from + 8 * (D / 2));
    float acc[NT][4];
#pragma unroll
    for (int t = 0; t < NT; ++t) acc[t][0] = acc[t][1] = acc[t][2] = acc[t][3] = 0.f;
#pragma unroll
    for (int k = 0; k < 2; ++k) {
      uint32_t x[4], y[4];
      codes(x, w0[k]);
      codes(y, w1[k]);
#pragma unroll
      for (int t = 0; t < NT; ++t) {
        mma_f16(acc[t], x[0], y[0], x[1], y[1], q.f[t][j * 4 + 2 * k][0], q.f[t][j * 4 + 2 * k][1]);
        mma_f16(acc[t], x[2], y[2], x[3], y[3], q.f[t][j * 4 + 2 * k + 1][0], q.f[t][j * 4 + 2 * k + 1][1]);
      }
    }
    const float st0 = pair_step(p0[j], shl16), st1 = pair_step(p1[j], shl16);
    const float z0 = fmaf(8.f, st0, pair_zero(p0[j])), z1 = fmaf(8.f, st1, pair_zero(p1[j]));
#pragma unroll
    for (int t = 0; t < NT; ++t) {
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const float st = i < 2 ? st0 : st1, zz = i < 2 ? z0 : z1;
        s[t][i] = j == 0 ? st * acc[t][i] : fmaf(st, acc[t][i], s[t][i]);
        z[t][i] = j == 0 ? zz * q.sum[t][j][i & 1] : fmaf(zz, q.sum[t][j][i & 1], z[t][i]);
      }
    }
  }
#pragma unroll
  for (int t = 0; t < NT; ++t)
#pragma unroll
    for (int i = 0; i < 4; ++i) s[t][i] = fmaf(s[t][i], q.unit[t][i & 1], z[t][i]);
}

// Stage the chunk's query heads in shared memory (rows beyond them zero).
template <typename T, int D, int NT>
AFD_DEVICE void stage_query(T* sq, const Kv4DecodeParams& p, int b, int head0, int heads) {
  const T* q = reinterpret_cast<const T*>(p.q) + b * p.q_sb + head0 * p.q_sh;
  for (int i = threadIdx.x; i < NT * 8 * D; i += blockDim.x) {
    const int h = i / D, d = i % D;
    sq[h * kQueryLd<D> + d] = h < heads ? q[h * p.q_sh + d] : from_f32<T>(0.f);
  }
}

// Unnormalised result of a piece in shared memory -> output (slot -1) or partial.
template <typename T, int D, int NT>
AFD_DEVICE void write_result(const Kv4DecodeParams& p, int b, int head0, int heads, int64_t slot, const float* red,
                             const float* ml, int nact) {
  // ml: [kWarps][NT * 8] maxima, then sums; red: [nact][NT * 8][D], already on the common maximum
  constexpr int H = NT * 8;
  for (int i = threadIdx.x; i < heads * (D / 4); i += kDecThreads) {
    const int h = i / (D / 4), d4 = i % (D / 4) * 4;
    float m = kLowest, l = 0.f;
    for (int w = 0; w < nact; ++w) m = fmaxf(m, ml[w * H + h]);
    float4 o = make_float4(0.f, 0.f, 0.f, 0.f);
    for (int w = 0; w < nact; ++w) {
      const float f = fast_exp2(ml[w * H + h] - m);
      l = fmaf(ml[(kWarps + w) * H + h], f, l);
      const float4 v = *reinterpret_cast<const float4*>(red + (w * H + h) * kRedLd<D> + d4);
      o.x = fmaf(v.x, f, o.x);
      o.y = fmaf(v.y, f, o.y);
      o.z = fmaf(v.z, f, o.z);
      o.w = fmaf(v.w, f, o.w);
    }
    if (slot < 0) {
      const float inv = l > 0.f ? 1.f / l : (l == 0.f ? 0.f : l);
      T* out = reinterpret_cast<T*>(p.out) + ((int64_t)b * p.heads + head0 + h) * D + d4;
      out[0] = from_f32<T>(o.x * inv);
      out[1] = from_f32<T>(o.y * inv);
      out[2] = from_f32<T>(o.z * inv);
      out[3] = from_f32<T>(o.w * inv);
      if (d4 == 0 && p.lse != nullptr)
        p.lse[(int64_t)b * p.heads + head0 + h] = (m + log2f(l)) * 0.6931471805599453f;
    } else {
      *reinterpret_cast<float4*>(p.part_o + (slot * H + h) * D + d4) = o;
      if (d4 == 0) {
        p.part_ml[(slot * H + h) * 2] = m;
        p.part_ml[(slot * H + h) * 2 + 1] = l;
      }
    }
  }
}

// The running state of one warp: its 8 NT heads' maxima and sums, and o.
template <int D, int NT>
struct Acc {
  static constexpr int G = D / kGroup;
  float o[NT][G * 4][4], zo[NT][G][2], m[NT][2], l[NT][2];
  float scale[G];  // power of two that o's group j is multiplied by
  AFD_DEVICE void clear() {
#pragma unroll
    for (int t = 0; t < NT; ++t) {
#pragma unroll
      for (int i = 0; i < G * 4; ++i) o[t][i][0] = o[t][i][1] = o[t][i][2] = o[t][i][3] = 0.f;
#pragma unroll
      for (int j = 0; j < G; ++j) zo[t][j][0] = zo[t][j][1] = 0.f;
      m[t][0] = m[t][1] = kLowest;
      l[t][0] = l[t][1] = 0.f;
    }
#pragma unroll
    for (int j = 0; j < G; ++j) scale[j] = pow2(kScaleTop);
  }
};

// The tiles of one step, in a stage of the ring.  `left` positions from the
// first tile on exist (kTail: fewer than the step's): the others weigh nothing,
// whatever their bytes hold.
//
// The second product takes p * step in fp16, 11 bits: half a step of that is an
// eighth of the half step of a bf16 result.  An fp16 result, whose half step it
// would equal, takes what the first factor leaves as a second one (22 bits): at
// 16 sequences of 50 - 131 K positions 239 us instead of 217, at 16 of 0.8 - 2 K
// with scores 34.5 instead of 32.7; the error against 64 bits is 1.9 - 2.1e-4,
// the result's own rounding, instead of 2.6e-4.  p is at most 2^kLazy,
// and a power of two per dim group (kept per warp, lowered when a larger step
// comes) holds the steps below 2^9, so the factors stay below 2^15.  A step
// that set the scale gets 2^5 at least: factors keep full precision down to
// 2^-19 of it, and below that are off by at most 2^-30 of it.
template <typename T, int D, int NT, bool kLogits, bool kTail>
AFD_DEVICE void take_tiles(Acc<D, NT>& acc, const Query<T, D, NT>& q, uint32_t stage, const Places<D>& at,
                           const Unpack& codes, uint32_t shl16, int left, int lane, float* logits, int64_t logits_ld,
                           int heads) {
  using R = Ring<D>;
  constexpr int G = D / kGroup, U = kTiles<D, NT>;
  constexpr int kParts = std::is_same<T, __half>::value ? 2 : 1;
  float s[U][NT][4];
#pragma unroll
  for (int u = 0; u < U; ++u) tile_logits<T, D, NT>(s[u], q, stage + u * R::kStageBytes, at, codes, shl16);
  const int r0 = tile_row(lane >> 2);
  if constexpr (kLogits) {  // `logits`: this step's first position, head 0 of the chunk
#pragma unroll
    for (int u = 0; u < U; ++u)
#pragma unroll
      for (int t = 0; t < NT; ++t)
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const int h = t * 8 + (lane & 3) * 2 + (i & 1), r = u * kTile + r0 + (i >> 1) * 8;
          if (h < heads && (!kTail || r < left)) logits[h * logits_ld + r] = s[u][t][i];
        }
  }
  uint32_t pr[U][2][G];          // (step, zero) of rows r0 and r0 + 8
  float st[U][2][G], k[U][2][G]; // their steps, and scaled
  bool grow = false;
#pragma unroll
  for (int u = 0; u < U; ++u) {
#pragma unroll
    for (int r = 0; r < 2; ++r) {
      lds_pairs<G>(pr[u][r], stage + u * R::kStageBytes + R::kHalf + at.pair + r * 8 * G * 4);
      const bool in = !kTail || u * kTile + r0 + r * 8 < left;
#pragma unroll
      for (int j = 0; j < G; ++j) {
        // positions past the end hold anything: their factors are zero, not 0 * that
        if (kTail && !in) pr[u][r][j] = 0;
        st[u][r][j] = pair_step(pr[u][r][j], shl16);
        k[u][r][j] = st[u][r][j] * acc.scale[j];
      }
      if (kTail && !in) {
#pragma unroll
        for (int t = 0; t < NT; ++t) s[u][t][2 * r] = s[u][t][2 * r + 1] = -INFINITY;
      }
    }
  }
#pragma unroll
  for (int j = 0; j < G; ++j) {
    float mx = fmaxf(k[0][0][j], k[0][1][j]);
#pragma unroll
    for (int u = 1; u < U; ++u) mx = fmaxf(mx, fmaxf(k[u][0][j], k[u][1][j]));
    grow |= mx >= kStepTop;
  }
#pragma unroll
  for (int t = 0; t < NT; ++t) {
#pragma unroll
    for (int e = 0; e < 2; ++e) {
      float mx = fmaxf(s[0][t][e], s[0][t][2 + e]);
#pragma unroll
      for (int u = 1; u < U; ++u) mx = fmaxf(mx, fmaxf(s[u][t][e], s[u][t][2 + e]));
      grow |= mx > acc.m[t][e] + kLazy;
    }
  }
  if (__any_sync(0xffffffffu, grow)) {
    float by[G];  // what o's scale changes by
#pragma unroll
    for (int j = 0; j < G; ++j) {
      float mx = 0.f;
#pragma unroll
      for (int u = 0; u < U; ++u) mx = fmaxf(mx, fmaxf(st[u][0][j], st[u][1][j]));
#pragma unroll
      for (int x = 4; x < 32; x <<= 1) mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, x));
      by[j] = 1.f;
      if (mx * acc.scale[j] >= kStepTop) {  // the largest step to [2^5, 2^6): three binades of room
        const int e = 5 - exponent_of(mx);
        by[j] = pow2(e) / acc.scale[j];
        acc.scale[j] = pow2(e);
#pragma unroll
        for (int u = 0; u < U; ++u)
#pragma unroll
          for (int r = 0; r < 2; ++r) k[u][r][j] = st[u][r][j] * acc.scale[j];
      }
    }
#pragma unroll
    for (int t = 0; t < NT; ++t) {
#pragma unroll
      for (int e = 0; e < 2; ++e) {
        float mx = acc.m[t][e];
#pragma unroll
        for (int u = 0; u < U; ++u) mx = fmaxf(mx, fmaxf(s[u][t][e], s[u][t][2 + e]));
#pragma unroll
        for (int x = 4; x < 32; x <<= 1) mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, x));
        const float f = fast_exp2(acc.m[t][e] - mx);
        acc.m[t][e] = mx;
        acc.l[t][e] *= f;
#pragma unroll
        for (int j = 0; j < G; ++j) {
          acc.zo[t][j][e] *= f;
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            acc.o[t][j * 4 + i][e] *= f * by[j];
            acc.o[t][j * 4 + i][2 + e] *= f * by[j];
          }
        }
      }
    }
  }
#pragma unroll
  for (int u = 0; u < U; ++u) {
#pragma unroll
    for (int t = 0; t < NT; ++t) {
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        s[u][t][i] = fast_exp2(s[u][t][i] - acc.m[t][i & 1]);
        acc.l[t][i & 1] += s[u][t][i];
      }
    }
    // P V: the probabilities, scaled per dim group, are the B operand.
#pragma unroll
    for (int j = 0; j < G; ++j) {
      const float z0 = fmaf(8.f, st[u][0][j], pair_zero(pr[u][0][j]));
      const float z1 = fmaf(8.f, st[u][1][j], pair_zero(pr[u][1][j]));
      uint32_t b[NT][kParts][2];
#pragma unroll
      for (int t = 0; t < NT; ++t) {
        const float* p = s[u][t];
        acc.zo[t][j][0] = fmaf(p[0], z0, fmaf(p[2], z1, acc.zo[t][j][0]));
        acc.zo[t][j][1] = fmaf(p[1], z0, fmaf(p[3], z1, acc.zo[t][j][1]));
#pragma unroll
        for (int r = 0; r < 2; ++r) {
          const float lo = p[2 * r] * k[u][r][j], hi = p[2 * r + 1] * k[u][r][j];
          const uint32_t top = pack_f16(lo, hi);
          b[t][0][r] = transpose8(top);
          if constexpr (kParts == 2) {
            const float2 took = __half22float2(*reinterpret_cast<const __half2*>(&top));
            b[t][1][r] = transpose8(pack_f16(lo - took.x, hi - took.y));
          }
        }
      }
      // k indices 2c, 2c + 1, 2c + 8, 2c + 9 are rows c, c + 4, c + 8, c + 12
      const uint32_t even = ((stage + at.v) ^ (j * 32)) + u * R::kStageBytes;
      const uint32_t odd = ((stage + at.v) ^ (j * 32) ^ kRow4<D>) + 4 * (D / 2) + u * R::kStageBytes;
      const uint32_t w0 = lds32(even), w1 = lds32(odd), w2 = lds32(even + 8 * (D / 2)), w3 = lds32(odd + 8 * (D / 2));
      // codes 0 .. 3 (dims) of two positions, then codes 4 .. 7
      uint32_t x0[4], x1[4], x2[4], x3[4];
      codes(x0, __byte_perm(w0, w1, 0x5410));
      codes(x1, __byte_perm(w0, w1, 0x7632));
      codes(x2, __byte_perm(w2, w3, 0x5410));
      codes(x3, __byte_perm(w2, w3, 0x7632));
#pragma unroll
      for (int i = 0; i < 4; ++i)
#pragma unroll
        for (int t = 0; t < NT; ++t)
#pragma unroll
          for (int part = 0; part < kParts; ++part)
            mma_f16(acc.o[t][j * 4 + i], x0[i], x1[i], x2[i], x3[i], b[t][part][0], b[t][part][1]);
    }
  }
}

// Shared memory of a decode CTA: the warps' rings; their results of a piece,
// merged while the next piece's first tiles are on their way; a chunk of query
// heads; the batch's prefix sums.  At D = 128 with 8 heads it is 75.3 KB: three
// CTAs fill the SM's 227 KB.
template <typename T, int D, int NT>
struct DecodeSmem {
  static constexpr int kRing = kWarps * kStages * kTiles<D, NT> * Ring<D>::kStageBytes;
  static constexpr int kRed = kWarps * NT * 8 * kRedLd<D> * 4;
  static constexpr int kQuery = NT * 8 * kQueryLd<D> * (int)sizeof(T);
  static int bytes(int batch, bool direct) { return kRing + kRed + kQuery + (direct ? 0 : (batch + 1) * 4); }
};

// What a piece is to the loop: its tiles, and whose they are.
struct Work {
  int b, t0, t1, n;                  // n: positions of the sequence
  int kv_head, head0, heads, slot;   // slot: where a partial result goes, or -1 if it is the whole
};

template <typename T, int D, int NT, bool kLogits>
__global__ void __launch_bounds__(kDecThreads, (kResident<D, NT>)) decode_kernel(Kv4DecodeParams p) {
  using R = Ring<D>;
  using S = DecodeSmem<T, D, NT>;
  constexpr int G = D / kGroup, H = NT * 8, U = kTiles<D, NT>;
  extern __shared__ __align__(128) uint8_t smem[];
  __shared__ int s_warp[kWarps];
  __shared__ float s_ml[2 * kWarps * H];
  float* const red = reinterpret_cast<float*>(smem + S::kRing);
  T* const sq = reinterpret_cast<T*>(smem + S::kRing + S::kRed);
  int* cum = reinterpret_cast<int*>(smem + S::kRing + S::kRed + S::kQuery);
  const int warp = threadIdx.x / 32, lane = threadIdx.x & 31;
  const int g = lane >> 2, c = lane & 3;
  const int heads_v = p.kv_heads * p.chunks;
  const Places<D> place(lane);
  const Unpack codes{p.mask_lo, p.mask_hi, p.base_f16};

  int64_t at = 0, end = 1, share = 1;  // direct: one (sequence, head chunk) per CTA
  if (!p.direct) {
    cost_prefix(p, cum, s_warp);
    const int64_t total = (int64_t)cum[p.batch] * heads_v;
    share = share_of(total, gridDim.x);
    at = min(total, blockIdx.x * share);
    end = min(total, at + share);
    // empty sequences have no piece: their results are written here
    for (int b = blockIdx.x; b < p.batch; b += gridDim.x)
      if (seq_len_of(p, b) == 0) {
        T* out = reinterpret_cast<T*>(p.out) + (int64_t)b * p.heads * D;
        for (int i = threadIdx.x; i < p.heads * D; i += kDecThreads) out[i] = from_f32<T>(0.f);
        if (p.lse != nullptr)
          for (int i = threadIdx.x; i < p.heads; i += kDecThreads) p.lse[(int64_t)b * p.heads + i] = -INFINITY;
      }
  }
  int4 split = make_int4(0, 0, 0, 0);  // for the join: sequence, first head, heads, pieces
  // The next piece of this CTA's share, if there is one.
  auto take = [&](Work& w) {
    Piece pc;
    while (true) {
      if (at >= end) return false;
      if (p.direct) {
        pc.b = blockIdx.x / heads_v;
        pc.hv = blockIdx.x % heads_v;
        pc.t0 = 0;
        pc.t1 = pc.tiles = tiles_of(seq_len_of(p, pc.b));
        at = end;
        break;
      }
      pc = piece_at(p, cum, heads_v, at, end);
      at = pc.next;
      if (pc.t0 < pc.t1) break;
    }
    const int group = p.heads / p.kv_heads, h_in = pc.hv % p.chunks * H;
    w.b = pc.b;
    w.t0 = pc.t0;
    w.t1 = pc.t1;
    w.n = seq_len_of(p, pc.b);
    w.kv_head = pc.hv / p.chunks;
    w.head0 = w.kv_head * group + h_in;
    w.heads = min(H, group - h_in);
    // Only a share's first and last pieces can be parts of a (sequence, head):
    // one that begins with its first tile goes to the CTA's second slot.
    w.slot = pc.t0 == 0 && pc.t1 == pc.tiles ? -1 : 2 * (int)blockIdx.x + (pc.t0 == 0 ? 1 : 0);
    if (pc.t0 == 0 && pc.t1 < pc.tiles)  // goes on in the CTAs after this one, to that of its last tile
      split = make_int4(w.b, w.head0, w.heads, 1 + (int)((pc.tiles - pc.t1 + share - 1) / share));
    return true;
  };

  // Each warp fills its own ring.  Steps of U tiles of a piece are dealt to the
  // warps in turn.
  constexpr uint32_t kStep = U * R::kStageBytes, kLast = (kStages - 1) * kStep;
  const uint32_t base = smem_u32(smem) + warp * kStages * kStep;
  TileWalk<D, U> walk;
  int issue = 0, issue_end = 0;
  auto copy_next = [&](uint32_t into) {
    if (issue < issue_end) {
#pragma unroll
      for (int u = 0; u < U; ++u)
        if (issue + u < issue_end) walk.template load<true>(u, into + u * R::kStageBytes, place.cp, lane);
      issue += U * kWarps;
      walk.advance();
      walk.fetch(issue_end - issue);
    }
    cp_commit();
  };
  auto begin = [&](const Work& w) {
    issue = w.t0 + warp * U;
    issue_end = w.t1;
    walk.start(p, w.b, w.kv_head, issue, lane);
    walk.fetch(issue_end - issue);
#pragma unroll
    for (int s = 0; s < kStages - 1; ++s) copy_next(base + s * kStep);
    check_blocks(p, w.b, w.t0, w.t1);
  };

  Work w, next;
  bool more = take(w);
  if (more) {
    begin(w);
    stage_query<T, D, NT>(sq, p, w.b, w.head0, w.heads);
  }
  while (more) {
    __syncthreads();  // this piece's query is staged, the last one's results are written
    Query<T, D, NT> q;
    q.load(sq, p.scale_log2, lane);
    Acc<D, NT> acc;
    acc.clear();
    float* logits = nullptr;
    if constexpr (kLogits) logits = p.logits + (int64_t)(w.b * p.heads + w.head0) * p.logits_ld;
    uint32_t st = base, into = base + kLast;
    for (int tile = w.t0 + warp * U; tile < w.t1; tile += U * kWarps) {
      cp_wait<kStages - 2>();
      __syncwarp();
      copy_next(into);  // into the stage that the previous step has left
      // a piece that ends before its sequence may end inside a step
      const int left = min(w.n, w.t1 * kTile) - tile * kTile;
      float* const lg = kLogits ? logits + tile * kTile : nullptr;
      if (left >= U * kTile)
        take_tiles<T, D, NT, kLogits, false>(acc, q, st, place, codes, p.shl16, left, lane, lg, p.logits_ld, w.heads);
      else
        take_tiles<T, D, NT, kLogits, true>(acc, q, st, place, codes, p.shl16, left, lane, lg, p.logits_ld, w.heads);
      into = st;
      st = st == base + kLast ? base : st + kStep;
      __syncwarp();  // every lane is done with this stage before it is refilled
    }
    more = take(next);
    if (more) begin(next);  // on its way while this piece is merged

    const int nact = min(kWarps, (w.t1 - w.t0 + U - 1) / U);
    if (warp < nact) {
#pragma unroll
      for (int t = 0; t < NT; ++t) {
#pragma unroll
        for (int e = 0; e < 2; ++e) {
          float ls = acc.l[t][e], z[G];
#pragma unroll
          for (int j = 0; j < G; ++j) z[j] = acc.zo[t][j][e];
#pragma unroll
          for (int x = 4; x < 32; x <<= 1) {
            ls += __shfl_xor_sync(0xffffffffu, ls, x);
#pragma unroll
            for (int j = 0; j < G; ++j) z[j] += __shfl_xor_sync(0xffffffffu, z[j], x);
          }
          const int h = t * 8 + 2 * c + e;
          if (g == 0) {
            s_ml[warp * H + h] = acc.m[t][e];
            s_ml[(kWarps + warp) * H + h] = ls;
          }
          float* to = red + (warp * H + h) * kRedLd<D> + g * 8;
#pragma unroll
          for (int j = 0; j < G; ++j) {
            const auto& o = acc.o[t];
            const float u = 1.f / acc.scale[j];
            *reinterpret_cast<float4*>(to + j * kGroup) =
                make_float4(fmaf(o[j * 4][e], u, z[j]), fmaf(o[j * 4 + 1][e], u, z[j]), fmaf(o[j * 4 + 2][e], u, z[j]),
                            fmaf(o[j * 4 + 3][e], u, z[j]));
            *reinterpret_cast<float4*>(to + j * kGroup + 4) =
                make_float4(fmaf(o[j * 4][2 + e], u, z[j]), fmaf(o[j * 4 + 1][2 + e], u, z[j]),
                            fmaf(o[j * 4 + 2][2 + e], u, z[j]), fmaf(o[j * 4 + 3][2 + e], u, z[j]));
          }
        }
      }
    }
    __syncthreads();
    if (more) stage_query<T, D, NT>(sq, p, next.b, next.head0, next.heads);
    write_result<T, D, NT>(p, w.b, w.head0, w.heads, w.slot, red, s_ml, nact);
    w = next;
  }
  cp_wait<0>();
  if (!p.direct && threadIdx.x == 0) *reinterpret_cast<int4*>(p.splits + 4 * blockIdx.x) = split;
}

// Joins the partials of the (sequences, head chunks) that more than one CTA
// worked on: block c those of the one that begins in CTA c's share and goes on
// in the next, if there is one.  kJoinWarps / H warps take a head's pieces in
// turn and merge through shared memory.
constexpr int kJoinWarps = 32;
template <typename T, int D, int NT>
__global__ void __launch_bounds__(kJoinWarps * 32) join_kernel(Kv4DecodeParams p) {
  constexpr int H = NT * 8, W = kJoinWarps / H, V = D / 32;  // warps of a head, dims a lane holds
  __shared__ float s_ml[kJoinWarps][2], s_o[kJoinWarps][D];
  const int warp = threadIdx.x / 32, lane = threadIdx.x & 31, h = warp / W, part = warp % W;
  pdl_wait();
  const int4 split = *reinterpret_cast<const int4*>(p.splits + 4 * blockIdx.x);  // sequence, first head, heads, pieces
  if (split.w == 0) return;
  float m = kLowest, l = 0.f, o[V] = {};
  if (h < split.z) {
#pragma unroll 8
    for (int k = part; k < split.w; k += W) {
      // the first piece is in its CTA's second slot, the others begin shares
      const int64_t slot = (2 * (int64_t)(blockIdx.x + k) + (k == 0 ? 1 : 0)) * H + h;
      const float2 ml = *reinterpret_cast<const float2*>(p.part_ml + slot * 2);
      float v[V];
#pragma unroll
      for (int i = 0; i < V; ++i) v[i] = p.part_o[slot * D + i * 32 + lane];
      const float mx = fmaxf(m, ml.x), f = fast_exp2(m - mx), g = fast_exp2(ml.x - mx);
      m = mx;
      l = l * f + ml.y * g;
#pragma unroll
      for (int i = 0; i < V; ++i) o[i] = o[i] * f + v[i] * g;
    }
  }
  if (lane == 0) {
    s_ml[warp][0] = m;
    s_ml[warp][1] = l;
  }
#pragma unroll
  for (int i = 0; i < V; ++i) s_o[warp][i * 32 + lane] = o[i];
  __syncthreads();
  if (part != 0 || h >= split.z) return;
#pragma unroll
  for (int w = 1; w < W; ++w) m = fmaxf(m, s_ml[warp + w][0]);
  l = 0.f;
#pragma unroll
  for (int i = 0; i < V; ++i) o[i] = 0.f;
#pragma unroll
  for (int w = 0; w < W; ++w) {
    const float f = fast_exp2(s_ml[warp + w][0] - m);
    l = fmaf(s_ml[warp + w][1], f, l);
#pragma unroll
    for (int i = 0; i < V; ++i) o[i] = fmaf(s_o[warp + w][i * 32 + lane], f, o[i]);
  }
  const float inv = l > 0.f ? 1.f / l : (l == 0.f ? 0.f : l);
  const int64_t row = (int64_t)split.x * p.heads + split.y + h;
  T* out = reinterpret_cast<T*>(p.out) + row * D;
#pragma unroll
  for (int i = 0; i < V; ++i) out[i * 32 + lane] = from_f32<T>(o[i] * inv);
  if (lane == 0 && p.lse != nullptr) p.lse[row] = (m + log2f(l)) * 0.6931471805599453f;
}

// Scores from the logits that the decode left (log2 domain, [batch, heads,
// logits_ld]): a thread takes a position of one (sequence, KV head) and sums the
// probabilities of the group's heads.  Adds, not stores: sequences may share
// blocks.
constexpr int kScoreThreads = 128, kScorePositions = 256;  // of a block: many small ones, to have many loads in flight
__global__ void __launch_bounds__(kScoreThreads) add_scores_kernel(Kv4DecodeParams p) {
  const int b = blockIdx.x / p.kv_heads, kv_head = blockIdx.x % p.kv_heads;
  const int n = seq_len_of(p, b), group = p.heads / p.kv_heads;
  const int64_t head = (int64_t)b * p.heads + kv_head * group;
  pdl_wait();
  for (int64_t first = (int64_t)blockIdx.y * kScorePositions; first < n; first += (int64_t)gridDim.y * kScorePositions) {
    const int t0 = (int)first + threadIdx.x, t1 = t0 + kScoreThreads;
    const float* at = p.logits + head * p.logits_ld;
    float w0 = 0.f, w1 = 0.f;
#pragma unroll 8
    for (int h = 0; h < group; ++h) {
      const float lse = p.lse[head + h] * 1.4426950408889634f;
      if (t0 < n) w0 += fast_exp2(at[h * p.logits_ld + t0] - lse);
      if (t1 < n) w1 += fast_exp2(at[h * p.logits_ld + t1] - lse);
    }
#pragma unroll
    for (int u = 0; u < 2; ++u) {
      const int t = u ? t1 : t0;
      if (t < n) {
        const int pg = t / p.block_size;
        const uint32_t blk = min((unsigned)p.block_table[(int64_t)b * p.table_stride + pg], (unsigned)p.num_blocks - 1u);
        atomicAdd(p.scores + ((int64_t)blk * p.kv_heads + kv_head) * p.block_size + (t - pg * p.block_size), u ? w1 : w0);
      }
    }
  }
}

// The same without stored logits, from K once more: for batches whose logits
// would not fit the workspace.
// Adds every position's probability to its score.  The same shares of tiles;
// nothing to merge, since a position is in one tile.
template <typename T, int D, int NT>
__global__ void __launch_bounds__(kDecThreads, 4) score_kernel(Kv4DecodeParams p) {
  using R = Ring<D>;
  constexpr int H = NT * 8;
  extern __shared__ __align__(128) uint8_t smem[];
  __shared__ int s_warp[kWarps];
  T* sq = reinterpret_cast<T*>(smem + p.ring_bytes);
  int* cum = reinterpret_cast<int*>(smem + p.ring_bytes + H * kQueryLd<D> * sizeof(T));
  const int warp = threadIdx.x / 32, lane = threadIdx.x & 31;
  const int c = lane & 3, r0 = tile_row(lane >> 2);
  const int heads_v = p.kv_heads * p.chunks;
  const Places<D> place(lane);
  const Unpack codes{p.mask_lo, p.mask_hi, p.base_f16};
  cost_prefix(p, cum, s_warp);
  const int64_t total = (int64_t)cum[p.batch] * heads_v;
  const int64_t share = share_of(total, gridDim.x);
  int64_t at = min(total, blockIdx.x * share);
  const int64_t end = min(total, at + share);
  pdl_wait();  // the log-sum-exps of the decode
  while (at < end) {
    const Piece pc = piece_at(p, cum, heads_v, at, end);
    at = pc.next;
    if (pc.t0 == pc.t1) continue;
    const int n = seq_len_of(p, pc.b);
    const int kv_head = pc.hv / p.chunks, group = p.heads / p.kv_heads;
    const int h_in = pc.hv % p.chunks * H;
    const int heads = min(H, group - h_in);
    const int head0 = kv_head * group + h_in;
    const uint32_t base = smem_u32(smem) + warp * kScoreStages * R::kHalf;
    int issue = pc.t0 + warp;
    TileWalk<D, 1> walk;
    walk.start(p, pc.b, kv_head, issue, lane);
    walk.fetch(pc.t1 - issue);
    auto copy_next = [&](uint32_t into) {
      if (issue < pc.t1) {
        walk.template load<false>(0, into, place.cp, lane);
        issue += kWarps;
        walk.advance();
        walk.fetch(pc.t1 - issue);
      }
      cp_commit();
    };
#pragma unroll
    for (int s = 0; s < kScoreStages - 1; ++s) copy_next(base + s * R::kHalf);
    stage_query<T, D, NT>(sq, p, pc.b, head0, heads);
    __syncthreads();
    Query<T, D, NT> q;
    q.load(sq, p.scale_log2, lane);
    float lse[NT][2];  // log2 domain; heads beyond the group weigh nothing
#pragma unroll
    for (int t = 0; t < NT; ++t)
#pragma unroll
      for (int e = 0; e < 2; ++e) {
        const int h = t * 8 + 2 * c + e;
        lse[t][e] = h < heads ? p.lse[(int64_t)pc.b * p.heads + head0 + h] * 1.4426950408889634f : INFINITY;
      }
    // a second walk, for the scores' addresses
    TileWalk<D, 1> to;
    to.start(p, pc.b, kv_head, pc.t0 + warp, lane);
    float* const scores = p.scores + (size_t)kv_head * p.block_size;
    constexpr uint32_t kLast = (kScoreStages - 1) * R::kHalf;
    uint32_t st = base, into = base + kLast;
    for (int tile = pc.t0 + warp; tile < pc.t1; tile += kWarps) {
      to.fetch(1);
      cp_wait<kScoreStages - 2>();
      __syncwarp();
      copy_next(into);
      float s[NT][4];
      tile_logits<T, D, NT>(s, q, st, place, codes, p.shl16);
      into = st;
      st = st == base + kLast ? base : st + R::kHalf;
      float w0 = 0.f, w1 = 0.f;
#pragma unroll
      for (int t = 0; t < NT; ++t) {
        w0 += fast_exp2(s[t][0] - lse[t][0]) + fast_exp2(s[t][1] - lse[t][1]);
        w1 += fast_exp2(s[t][2] - lse[t][0]) + fast_exp2(s[t][3] - lse[t][1]);
      }
      w0 += __shfl_xor_sync(0xffffffffu, w0, 1);
      w1 += __shfl_xor_sync(0xffffffffu, w1, 1);
      w0 += __shfl_xor_sync(0xffffffffu, w0, 2);
      w1 += __shfl_xor_sync(0xffffffffu, w1, 2);
      // Adds, not stores: head chunks and sequences that share blocks meet here.
      if (c < 2) {
        const int r = r0 + c * 8;
        if (tile * kTile + r < n)
          atomicAdd(scores + (size_t)to.blk[0] * ((uint32_t)p.kv_heads * p.block_size) + to.in * kTile + r,
                    c == 0 ? w0 : w1);
      }
      to.advance();
      __syncwarp();
    }
    cp_wait<0>();
    __syncthreads();
  }
}

template <typename T, int D, int NT, bool kLogits>
cudaError_t launch_decode(const Kv4DecodeParams& p, cudaStream_t s) {
  using S = DecodeSmem<T, D, NT>;
  auto* kernel = decode_kernel<T, D, NT, kLogits>;
  static PerDeviceOnce attr;
  cudaError_t e = attr.run([&] {
    return cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, S::bytes(kMaxBatch, false));
  });
  if (e != cudaSuccess) return e;
  kernel<<<p.ctas, kDecThreads, S::bytes(p.batch, p.direct), s>>>(p);
  if (!p.direct) {
    e = launch_pdl(join_kernel<T, D, NT>, dim3((unsigned)p.ctas), dim3(kJoinWarps * 32), 0, s, p);
    if (e != cudaSuccess) return e;
  }
  return cudaGetLastError();
}

template <typename T, int D, int NT>
cudaError_t launch_score(Kv4DecodeParams p, cudaStream_t s) {
  constexpr int H = NT * 8;
  p.ring_bytes = kWarps * kScoreStages * Ring<D>::kHalf;
  const int smem = p.ring_bytes + H * kQueryLd<D> * (int)sizeof(T) + (p.batch + 1) * 4;
  static PerDeviceOnce attr;
  cudaError_t e = attr.run([&] {
    return cudaFuncSetAttribute(score_kernel<T, D, NT>, cudaFuncAttributeMaxDynamicSharedMemorySize,
                                p.ring_bytes + H * kQueryLd<D> * (int)sizeof(T) + (kMaxBatch + 1) * 4);
  });
  if (e != cudaSuccess) return e;
  return launch_pdl(score_kernel<T, D, NT>, dim3(4 * device_sm_count()), dim3(kDecThreads), (size_t)smem, s, p);
}

template <typename T, int D, int NT>
cudaError_t run(const Kv4DecodeParams& p, cudaStream_t s) {
  const cudaError_t e = p.logits != nullptr ? launch_decode<T, D, NT, true>(p, s) : launch_decode<T, D, NT, false>(p, s);
  if (e != cudaSuccess || p.scores == nullptr) return e;
  if (p.logits == nullptr) return launch_score<T, D, NT>(p, s);
  // blocks for every position there may be, up to 64 waves; the rest in turn
  const int64_t chunks = ((int64_t)p.max_blocks * p.block_size + kScorePositions - 1) / kScorePositions;
  const int64_t most = 1 + (int64_t)64 * 16 * device_sm_count() / (p.batch * p.kv_heads);
  return launch_pdl(add_scores_kernel,
                    dim3((unsigned)(p.batch * p.kv_heads), (unsigned)std::min<int64_t>({chunks, most, 65535})),
                    dim3(kScoreThreads), 0, s, p);
}

template <typename T>
cudaError_t dispatch(Kv4DecodeParams p, cudaStream_t s) {
  p.mask_lo = 0x000F000Fu;
  p.mask_hi = 0x00F000F0u;
  p.base_f16 = 0x64006400u;
  p.shl16 = 65536u;
  const bool wide = p.head_tiles == 2;
  switch (p.dim) {
    case 64: return wide ? run<T, 64, 2>(p, s) : run<T, 64, 1>(p, s);
    case 128: return wide ? run<T, 128, 2>(p, s) : run<T, 128, 1>(p, s);
    default: return run<T, 256, 1>(p, s);
  }
}

}  // namespace kv4
}  // namespace afd

using namespace afd;

Kv4Plan kv4_decode_plan(int batch, int heads, int kv_heads, int dim, int max_len) {
  Kv4Plan plan;
  const int group = heads / kv_heads;
  // 16 heads share one unpacking of the codes: 38.8 us against 41.1 us in two
  // passes of 8 at 4 sequences of 20 - 33 K positions, 64 heads on 4.  At
  // D = 256 their accumulators would not fit in registers.
  plan.head_tiles = dim <= 128 && group > 8 ? 2 : 1;
  const int per = 8 * plan.head_tiles;
  plan.chunks = (group + per - 1) / per;
  const int64_t items = (int64_t)batch * kv_heads * plan.chunks;
  // Up to 512 positions a CTA takes a whole (sequence, head): 6.1 us against
  // 8.9 us in shares and their join at 2 sequences of up to 61 positions, 10.8
  // against 15.7 us at 64 of 100 - 512, 27.0 against 35.1 us at 256 of 1 - 512.
  constexpr int kDirectTiles = 32;
  plan.direct = (max_len + kv4::kTile - 1) / kv4::kTile <= kDirectTiles;
  const int resident = dim * plan.head_tiles <= 128 ? 3 : 2;  // kResident
  plan.ctas = plan.direct ? (int)items : resident * device_sm_count();
  // the prefix sums of a launch stay below 2^31 whatever the lengths
  const int64_t most = INT32_MAX / ((int64_t)max_len / kv4::kTile + kv4::kRound + kv4::kPieceCost);
  plan.max_batch = (int)std::min<int64_t>(kv4::kMaxBatch, most);
  return plan;
}

int launch_gqa_decode_int4(const Kv4DecodeParams& p, int dtype, cudaStream_t s) {
  return (int)(dtype == kF16 ? kv4::dispatch<__half>(p, s) : kv4::dispatch<__nv_bfloat16>(p, s));
}
