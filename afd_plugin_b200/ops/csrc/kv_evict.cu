// Eviction from the paged 4-bit KV cache by accumulated attention weight.
//
// A sequence of n > budget positions keeps, for each KV head, its last
// `recent` positions and the budget - recent best scored of the others (ties
// go to the earlier position).  The kept rows move, in order, to the
// sequence's first `budget` positions, in place; the scores move with them.
//
// One cluster of CTAs works on one (sequence, KV head):
//   1. the CTAs take equal runs of positions and turn scores into 32-bit keys
//      that order like the scores (in shared memory, as far as they fit);
//   2. four passes over 8 bits each find the key of the last kept position
//      (the first as the scores arrive): shared-memory histograms, summed over
//      the cluster through distributed shared memory;
//   3. each warp counts its run, a prefix over warps and CTAs gives every kept
//      position its rank;
//   4. rows move in chunks: all CTAs load a chunk into registers, a cluster
//      barrier, then they store it.  Row i comes from a position >= i, so a
//      chunk's stores only overwrite rows that this chunk or an earlier one
//      has loaded, and the next chunk's loads are issued before the barrier.
//
// What bounds it: the moved rows, read and written once (148 B each way at
// D = 128), and one read of the scores.  32 sequences of 20 - 33 K positions
// cut to 8192 (4 KV heads of 128): 328 MB in 113 us, 2.9 TB/s; 43 us of it are
// the selection, whose passes wait for one another, and the move alone runs at
// 4.4 TB/s.  Three sequences just over 1024: 15 us, nearly all of them those
// waits.  The cluster size spreads small batches over the SMs.
#include <cooperative_groups.h>

#include "device_state.h"
#include "kv_int4.cuh"
#include "launchers.h"

namespace afd {
namespace kv4 {
namespace cg = cooperative_groups;

constexpr int kEvThreads = 512;
constexpr int kEvWarps = kEvThreads / 32;
constexpr int kUnits = 4;  // 16-byte units of codes a thread moves per chunk

// Orders like the float; NaN counts as -inf, -0 as 0.
AFD_DEVICE uint32_t order_key(float x) {
  if (x != x) x = -INFINITY;
  const uint32_t u = __float_as_uint(x + 0.f);
  return u >> 31 ? ~u : u | 0x80000000u;
}

struct EvictView {
  const Kv4EvictParams& p;
  const int32_t* table;
  int64_t head_off, block_rows;
  AFD_DEVICE EvictView(const Kv4EvictParams& q, int b, int h)
      : p(q), table(q.block_table + (int64_t)b * q.table_stride), head_off((int64_t)h * q.block_size),
        block_rows((int64_t)q.kv_heads * q.block_size) {}
  // Cache row of a position.  A block id outside the pool is reported and replaced by the padding block.
  AFD_DEVICE int64_t row(int pos) const {
    const int pg = p.block_shift >= 0 ? pos >> p.block_shift : pos / p.block_size;
    int blk = table[pg];
    if ((unsigned)blk >= (unsigned)p.num_blocks) {
      if (p.status != nullptr) atomicExch(p.status, kStatusBadIndex);
      blk = 0;
    }
    return blk * block_rows + head_off + (pos - pg * p.block_size);
  }
};

template <int D>
__global__ void __launch_bounds__(kEvThreads) evict_kernel(Kv4EvictParams p) {
  constexpr int G = D / kGroup;
  constexpr int kRowUnits = 2 * D / 32;                     // 16-byte units of codes of a row, K then V
  constexpr int kRows = kUnits * kEvThreads / kRowUnits;    // rows a CTA moves per chunk
  constexpr int kRowWords = 2 * G + 1;                      // (step, zero) pairs of K and V, and the score
  constexpr int kWords = (kRows * kRowWords + kEvThreads - 1) / kEvThreads;
  extern __shared__ __align__(16) uint32_t s_keys[];
  __shared__ uint32_t s_hist[2][256];
  __shared__ uint32_t s_pick[2];              // digit, positions still to take from it
  __shared__ int s_warp[2][kEvWarps];         // kept-for-sure / tied positions of each warp's run
  __shared__ int s_cta[2];                    // the CTA's totals, read by the others
  __shared__ uint32_t s_scan[8];
  __shared__ int64_t s_src[2][kRows];         // source rows of this chunk and the next
  __shared__ int64_t s_dst[3][kRows];         // destination rows, of the last chunk too (see the move)

  cg::cluster_group cluster = cg::this_cluster();
  const int cs = (int)cluster.num_blocks(), rank = (int)cluster.block_rank();
  const int item = blockIdx.x / cs;
  const int b = item / p.kv_heads, h = item % p.kv_heads;
  const int tid = threadIdx.x, warp = tid / 32, lane = tid & 31;
  int n = p.seq_lens[b];
  n = n < 0 ? 0 : min(n, p.max_blocks * p.block_size);
  int32_t* kept = p.kept + (int64_t)item * p.budget;
  if (h == 0 && rank == 0 && tid == 0) p.new_lens[b] = min(n, p.budget);
  if (n <= p.budget) {  // the same for the whole cluster
    for (int i = rank * kEvThreads + tid; i < p.budget; i += cs * kEvThreads) kept[i] = i < n ? i : -1;
    return;
  }
  const EvictView view(p, b, h);
  const int m = n - p.recent;             // candidates
  const int need = p.budget - p.recent;   // of them to keep: 0 <= need < m
  // Runs of whole quads: four positions are one load and one look at the table.
  const int per = ((m + cs - 1) / cs + 3) & ~3;
  const int lo = min(m, rank * per), cnt = min(m, lo + per) - lo;
  const int quads = (cnt + 3) / 4;

  uint4* const keys = reinterpret_cast<uint4*>(s_keys);
  const int held = p.key_cap / 4;  // quads in shared memory; the rest are read again each time
  auto load_quad = [&](int i) {    // a block's rows come in multiples of 16, so a quad stays inside its block
    const float4 x = *reinterpret_cast<const float4*>(p.scores + view.row(lo + 4 * i));
    return make_uint4(order_key(x.x), order_key(x.y), order_key(x.z), order_key(x.w));
  };
  auto quad_at = [&](int i) { return i < held ? keys[i] : load_quad(i); };
  for (int i = tid; i < 2 * 256; i += kEvThreads) (&s_hist[0][0])[i] = 0;
  __syncthreads();

  // Adds the digit of one key per lane.  Scores crowd in few exponents: one add
  // where the warp agrees.  Whole warps call this.
  auto count_digit = [&](uint32_t* hist, bool in, uint32_t digit) {
    const uint32_t act = __ballot_sync(0xffffffffu, in);
    if (act == 0) return;
    const uint32_t first = __shfl_sync(0xffffffffu, digit, __ffs(act) - 1);
    if (__all_sync(0xffffffffu, !in || digit == first)) {
      if (lane == 0) atomicAdd(&hist[first], (uint32_t)__popc(act));
    } else if (in) {
      atomicAdd(&hist[digit], 1u);
    }
  };

  // The key of the last position kept (`bound`) and how many of its ties are.
  uint32_t bound = 0, left = (uint32_t)need;
  const int padded = (quads + 31) & ~31;
#pragma unroll 1
  for (int pass = 0; pass < 4; ++pass) {
    const int shift = 24 - 8 * pass;
    uint32_t* hist = s_hist[pass & 1];
#pragma unroll 2
    for (int i = tid; i < padded; i += kEvThreads) {  // whole warps enter
      uint4 k4 = make_uint4(0, 0, 0, 0);
      if (i < quads) {
        k4 = pass == 0 ? load_quad(i) : quad_at(i);
        if (pass == 0 && i < held) keys[i] = k4;
      }
      const uint32_t k[4] = {k4.x, k4.y, k4.z, k4.w};
      bool in[4], any = false;
#pragma unroll
      for (int q = 0; q < 4; ++q) {
        in[q] = 4 * i + q < cnt && (pass == 0 || ((k[q] ^ bound) >> (shift + 8)) == 0);
        any |= in[q];
      }
      if (!__any_sync(0xffffffffu, any)) continue;
#pragma unroll
      for (int q = 0; q < 4; ++q) count_digit(hist, in[q], (k[q] >> shift) & 255u);
    }
    cluster.sync();
    uint32_t sum = 0, above = 0;
    if (tid < 256) {  // thread t looks at digit 255 - t: descending order
#pragma unroll
      for (int r = 0; r < 8; ++r)  // all loads in flight at once
        if (r < cs) sum += cluster.map_shared_rank(hist, r)[255 - tid];
      above = sum;
#pragma unroll
      for (int o = 1; o < 32; o <<= 1) {
        const uint32_t u = __shfl_up_sync(0xffffffffu, above, o);
        if (lane >= o) above += u;
      }
      if (lane == 31) s_scan[warp] = above;
    }
    __syncthreads();
    if (tid < 256) {
      for (int w = 0; w < warp; ++w) above += s_scan[w];
      above -= sum;  // positions with a higher digit
      if (above < left && left <= above + sum) {
        s_pick[0] = 255 - tid;
        s_pick[1] = left - above;
      }
      if (left == 0 && tid == 0) {  // nothing to take: a bound above every key
        s_pick[0] = 255;
        s_pick[1] = 0;
      }
    }
    // the other buffer was read before this pass's barrier: clear it for the next pass
    if (tid >= 256) s_hist[(pass + 1) & 1][tid - 256] = 0;
    __syncthreads();
    bound |= s_pick[0] << shift;
    left = s_pick[1];
    __syncthreads();
  }
  // left = ties of `bound` to keep, the earliest ones (0 only when need is 0).
  const bool none = need == 0;

  // Each warp's run of quads: its sure and tied counts (low and high half of one
  // word), then ranks.
  const int seg = ((quads + kEvWarps - 1) / kEvWarps + 31) & ~31;
  const int w0 = min(quads, warp * seg), w1 = min(quads, w0 + seg);
  auto classes = [&](int i, uint32_t (&c)[4]) {  // 1: above the bound, 1 << 16: tied, 0: out
    const uint4 k4 = i < w1 ? quad_at(i) : make_uint4(0, 0, 0, 0);
    const uint32_t k[4] = {k4.x, k4.y, k4.z, k4.w};
    uint32_t sum = 0;
#pragma unroll
    for (int q = 0; q < 4; ++q) {
      const bool live = !none && i < w1 && 4 * i + q < cnt;
      c[q] = live && k[q] > bound ? 1u : (live && k[q] == bound ? 1u << 16 : 0u);
      sum += c[q];
    }
    return sum;
  };
  int gt = 0, eq = 0;
  uint32_t c[4];
  for (int i0 = w0; i0 < w1; i0 += 32) {
    const uint32_t sum = classes(i0 + lane, c);
    gt += sum & 0xFFFF;
    eq += sum >> 16;
  }
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) {
    gt += __shfl_xor_sync(0xffffffffu, gt, o);
    eq += __shfl_xor_sync(0xffffffffu, eq, o);
  }
  if (lane == 0) {
    s_warp[0][warp] = gt;
    s_warp[1][warp] = eq;
  }
  __syncthreads();
  int gt_before = 0, eq_before = 0;
  for (int w = 0; w < warp; ++w) {
    gt_before += s_warp[0][w];
    eq_before += s_warp[1][w];
  }
  if (tid == kEvThreads - 1) {
    s_cta[0] = gt_before + gt;
    s_cta[1] = eq_before + eq;
  }
  cluster.sync();
#pragma unroll
  for (int r = 0; r < 7; ++r)
    if (r < rank) {
      const int* other = cluster.map_shared_rank(s_cta, r);
      gt_before += other[0];
      eq_before += other[1];
    }
  for (int i0 = w0; i0 < w1; i0 += 32) {
    const int i = i0 + lane;
    const uint32_t mine = classes(i, c);
    uint32_t upto = mine;  // at most 128 of each in a step: the halves do not meet
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const uint32_t u = __shfl_up_sync(0xffffffffu, upto, o);
      if (lane >= o) upto += u;
    }
    const uint32_t total = __shfl_sync(0xffffffffu, upto, 31), before = upto - mine;
    int g = gt_before + (int)(before & 0xFFFF), e = eq_before + (int)(before >> 16);
#pragma unroll
    for (int q = 0; q < 4; ++q) {
      if (c[q] == 1u || (c[q] != 0 && e < (int)left)) kept[g + min(e, (int)left)] = lo + 4 * i + q;
      g += c[q] & 0xFFFF;
      e += c[q] >> 16;
    }
    gt_before += total & 0xFFFF;
    eq_before += total >> 16;
  }
  for (int i = rank * kEvThreads + tid; i < p.recent; i += cs * kEvThreads) kept[need + i] = m + i;
  cluster.sync();  // the list is complete, and visible to the cluster

  // Move.  16-byte units of codes and 4-byte words of pairs and scores.  Each
  // row's source and destination are looked up once, by one thread, a chunk
  // ahead of their use.  What orders the lists, with only the cluster barrier
  // B(i) of chunk i between the threads:
  //   s_src: chunk i's is written before B(i - 1), read between B(i - 1) and
  //          B(i), and overwritten (by chunk i + 2's) after B(i): two buffers.
  //   s_dst: chunk i's is written before B(i - 1) and read by its stores, which
  //          are between B(i) and B(i + 1), as is the look-up of chunk i + 2.
  //          That one has a buffer of its own; chunk i + 3's comes after
  //          B(i + 1): three buffers.
  uint4* const kc = reinterpret_cast<uint4*>(p.k_codes);
  uint4* const vc = reinterpret_cast<uint4*>(p.v_codes);
  auto unit = [&](int64_t row, int u) {
    return u < D / 32 ? kc + row * (D / 32) + u : vc + row * (D / 32) + (u - D / 32);
  };
  auto word = [&](int64_t row, int w) {
    return w < G ? p.k_scale + row * G + w
                 : (w < 2 * G ? p.v_scale + row * G + (w - G) : reinterpret_cast<uint32_t*>(p.scores) + row);
  };
  const int step = cs * kRows, skip = rank * kRows;
  const bool is_dst = tid >= kEvThreads / 2;
  auto look_up = [&](int src, int dst, int r0) {  // rows r0 .. r0 + kRows - 1, into these buffers
    for (int r = tid & (kEvThreads / 2 - 1); r < kRows; r += kEvThreads / 2)
      if (r0 + r < p.budget) (is_dst ? s_dst[dst] : s_src[src])[r] = view.row(is_dst ? r0 + r : kept[r0 + r]);
  };
  look_up(0, 0, skip);
  __syncthreads();
  int src = 0, dst = 0;
  for (int r0 = skip; r0 - skip < p.budget; r0 += step) {
    const int next_dst = dst == 2 ? 0 : dst + 1;
    uint4 x[kUnits];
    uint32_t y[kWords];
#pragma unroll
    for (int k = 0; k < kUnits; ++k) {
      const int j = k * kEvThreads + tid, r = j / kRowUnits;
      if (r0 + r < p.budget) x[k] = *unit(s_src[src][r], j % kRowUnits);
    }
#pragma unroll
    for (int k = 0; k < kWords; ++k) {
      const int j = k * kEvThreads + tid, r = j / kRowWords;
      if (j < kRows * kRowWords && r0 + r < p.budget) y[k] = *word(s_src[src][r], j % kRowWords);
    }
    look_up(src ^ 1, next_dst, r0 + step);
    cluster.sync();
#pragma unroll
    for (int k = 0; k < kUnits; ++k) {
      const int j = k * kEvThreads + tid, r = j / kRowUnits;
      if (r0 + r < p.budget) *unit(s_dst[dst][r], j % kRowUnits) = x[k];
    }
#pragma unroll
    for (int k = 0; k < kWords; ++k) {
      const int j = k * kEvThreads + tid, r = j / kRowWords;
      if (j < kRows * kRowWords && r0 + r < p.budget) *word(s_dst[dst][r], j % kRowWords) = y[k];
    }
    src ^= 1;
    dst = next_dst;
  }
}

template <int D>
cudaError_t launch_evict(Kv4EvictParams p, int cs, size_t smem, cudaStream_t s) {
  static PerDeviceOnce attr;
  cudaError_t e =
      attr.run([&] { return cudaFuncSetAttribute(evict_kernel<D>, cudaFuncAttributeMaxDynamicSharedMemorySize, 46080 * 4); });
  if (e != cudaSuccess) return e;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3((unsigned)(p.batch * p.kv_heads * cs));
  cfg.blockDim = dim3(kEvThreads);
  cfg.dynamicSmemBytes = smem;
  cfg.stream = s;
  cudaLaunchAttribute a[1];
  a[0].id = cudaLaunchAttributeClusterDimension;
  a[0].val.clusterDim.x = cs;
  a[0].val.clusterDim.y = a[0].val.clusterDim.z = 1;
  cfg.attrs = a;
  cfg.numAttrs = 1;
  return cudaLaunchKernelEx(&cfg, evict_kernel<D>, p);
}

}  // namespace kv4
}  // namespace afd

using namespace afd;

int launch_kv_evict_int4(Kv4EvictParams p, int dim, cudaStream_t s) {
  // As many CTAs on each (sequence, head) as keep all of them resident at once,
  // two per SM.  Measured at 128 (sequences x heads) of 20 - 33 K positions:
  // 170, 123, 133 and 159 us with 1, 2, 4 and 8, where the rule takes 2; at 12
  // of 1.1 K 20.7, 15.7, 13.2 and 14.1 us, where it takes 8, a microsecond from
  // the best.
  int cs = 1;
  while (cs < 8 && (int64_t)p.batch * p.kv_heads * cs * 2 <= 2 * device_sm_count()) cs *= 2;
  const int per = ((p.max_blocks * p.block_size + cs - 1) / cs + 3) & ~3;
  p.block_shift = (p.block_size & (p.block_size - 1)) == 0 ? __builtin_ctz(p.block_size) : -1;
  p.key_cap = per < 46080 ? per : 46080;  // 180 KB
  const size_t smem = (size_t)p.key_cap * 4;
  switch (dim) {
    case 64: return (int)kv4::launch_evict<64>(p, cs, smem, s);
    case 128: return (int)kv4::launch_evict<128>(p, cs, smem, s);
    default: return (int)kv4::launch_evict<256>(p, cs, smem, s);
  }
}
