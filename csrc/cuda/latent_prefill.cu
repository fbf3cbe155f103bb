// Expanded latent attention: a chunk of new tokens over a paged latent cache.
//
// One kernel expands the context rows [c (R) | k_r (64)] out of their pages to every head's key
// and value rows (kv = w_h c, [128 | 128] a head), and the attention runs with keys
// [k_h (128) | k_r (64, shared)] and values of 128:
//   out_i = sum_j softmax_j(scale q_i . k_j) v_j  over j <= position of i.
//
// Roundings: the expanded keys and values are bf16, the type of the query's rows that the first
// product takes and half the bytes of fp32, and so is P, the second product's operand (sums
// are fp32).  fp16 would keep 3 bits more, but not every model's values are within its range.  With the
// output's own, three roundings of 2^-8 at most: an output is 0.0029 from 64-bit arithmetic
// in the mean square, where one rounded once at the end is 0.0017.
#include <algorithm>

#include "common.cuh"
#include "kernels.h"
#include "tcgen05.cuh"

namespace kapsl {
using namespace tc;

using bf16 = __nv_bfloat16;

namespace {

constexpr int kNope = 128, kRot = 64, kVal = 128;
constexpr float kLog2e = 1.4426950408889634f;

// Bounded wait (2 s): polls the barrier, and reads the clock and the CTA's abort flag rarely
// (both are slow beside a poll).  A time-out records `code` and ends the CTA's other waits.
template <class Smem>
__device__ __forceinline__ bool wait_or_abort(Smem& s, uint64_t* bar, uint32_t parity, int* err, int code) {
  uint64_t t0 = 0;
  for (uint32_t spin = 1;; ++spin) {
    if (mbar_test_wait(bar, parity)) return true;
    if ((spin & 1023) == 0) {
      const uint64_t now = globaltimer_ns();
      if (t0 == 0) t0 = now;
      if (s.abort_flag) return false;
      if (now - t0 > 2000000000ull) {
        atomicCAS(err, 0, code);
        s.abort_flag = 1;
        return false;
      }
    }
  }
}

// ------------------------------------------------------------------ expansion
//
// kv[row, head] = w_head (256 x R) . c_row for every context row: a GEMM whose A rows come straight
// out of the pages.  A CTA pair (cluster of 2) works on units of (256 context rows, head) with
// cta_group::2 MMAs (M = 256, N = 256): each CTA holds 128 rows of one sequence and half of the
// head's weights, so a CTA loads 16 KB of weights for 512 cycles of products (one CTA alone needs
// 32 KB, and beside 128 KB of rows only two such stages fit: 1.45 x the time at 20k rows x
// 128 heads).  The units, rows outermost, are cut into equal stretches, one a pair; the rows stay in
// shared memory while the heads' weights stream past them, and two accumulators of 256 TMEM
// columns let one unit's epilogue run beside the next one's products.
// The epilogue turns 32-row slabs in shared memory so that every global store instruction
// writes whole 128-byte lines.  Rows behind a context (up to the next multiple of 16) are
// written as zeros, whatever their page slots hold; the head-0 unit also copies the rows'
// rotary keys.
constexpr int kExpandThreads = 192;  // warp 0 TMA, warp 1 MMA, warps 2-5 epilogue
constexpr int kSlabPitch = 144;      // 64 bf16 and 16 bytes against bank conflicts

template <int R>
struct alignas(1024) ExpandSmem {
  static constexpr int kChunks = R / 64;
  static constexpr int kStages = R == 512 ? 5 : 8;
  uint8_t a[kChunks][128 * 128];
  uint8_t b[kStages][128 * 128];
  uint8_t slab[4][32 * kSlabPitch];
  uint64_t a_full, a_empty, b_full[kStages], b_empty[kStages], acc_full[2], acc_empty[2], drained;
  uint32_t tmem_base;
  volatile int abort_flag;
};

// The `page`-row group of cache row j of a sequence: its first row, or the row past the cache.
__device__ __forceinline__ int64_t page_row(const int32_t* bt, int j, int page, int64_t num_blocks, int* err) {
  const int blk = bt[j / page];
  if (blk >= 0 && blk < num_blocks) return (int64_t)blk * page;
  atomicCAS(err, 0, 82);
  return num_blocks * page;
}

__device__ __forceinline__ uint32_t cta_rank() {
  uint32_t r;
  asm volatile("mov.u32 %0, %%cluster_ctarank;" : "=r"(r));
  return r;
}
__device__ __forceinline__ void cluster_sync() {
  asm volatile("barrier.cluster.arrive.release.aligned;\n\tbarrier.cluster.wait.acquire.aligned;" ::: "memory");
}
// arrives on the leader CTA's copy of a barrier
__device__ __forceinline__ void arrive_leader(uint64_t* bar) {
  asm volatile(
      "{\n\t.reg .b32 a;\n\tmapa.shared::cluster.u32 a, %0, 0;\n\t"
      "mbarrier.arrive.release.cluster.shared::cluster.b64 _, [a];\n\t}" ::"r"(smem_u32(bar))
      : "memory");
}
// a load of this CTA whose bytes count on the leader's barrier (peer bit of the address cleared)
__device__ __forceinline__ void tma_load_pair(void* dst, const CUtensorMap* m, uint64_t* bar, int32_t x, int32_t y) {
  asm volatile(
      "cp.async.bulk.tensor.2d.cta_group::2.shared::cluster.global.mbarrier::complete_tx::bytes"
      " [%0], [%1, {%3, %4}], [%2];" ::"r"(smem_u32(dst)),
      "l"(reinterpret_cast<uint64_t>(m)), "r"(smem_u32(bar) & 0xFEFFFFFFu), "r"(x), "r"(y)
      : "memory");
}
__device__ __forceinline__ void mma_pair(uint32_t d, uint64_t a, uint64_t b, uint32_t idesc, uint32_t accumulate) {
  asm volatile(
      "{\n\t.reg .pred p;\n\tsetp.ne.b32 p, %4, 0;\n\t"
      "tcgen05.mma.cta_group::2.kind::f16 [%0], %1, %2, %3, p;\n\t}" ::"r"(d),
      "l"(a), "l"(b), "r"(idesc), "r"(accumulate)
      : "memory");
}
__device__ __forceinline__ void commit_pair(uint64_t* bar) {  // arrives on both CTAs' barrier
  asm volatile(
      "tcgen05.commit.cta_group::2.mbarrier::arrive::one.shared::cluster.multicast::cluster.b64 [%0], %1;" ::"r"(
          smem_u32(bar)),
      "h"((uint16_t)3)
      : "memory");
}

template <int R>
__global__ void __cluster_dims__(2, 1, 1) __launch_bounds__(kExpandThreads, 1)
    latent_expand_kernel(const __grid_constant__ CUtensorMap c_map, const __grid_constant__ CUtensorMap w_map,
                         const bf16* cache, int64_t num_blocks, int page, const int32_t* work, int nwork,
                         const int32_t* seq_info, const int32_t* block_tables, int max_blocks, int heads,
                         bf16* kv, int64_t kv_stride, bf16* k_rope, int* err) {
  griddep_entry();
  using S = ExpandSmem<R>;
  extern __shared__ __align__(1024) uint8_t smem_raw[];
  S& s = *reinterpret_cast<S*>(smem_raw);
  const int warp = __shfl_sync(0xffffffffu, threadIdx.x / 32, 0), lane = threadIdx.x % 32;
  const int rank = (int)cta_rank();
  const int pairs = gridDim.x / 2, me = blockIdx.x / 2;
  const int64_t units = (int64_t)((nwork + 1) / 2) * heads;
  const int64_t u0 = units * me / pairs, u1 = units * (me + 1) / pairs;
  if (u0 >= u1) return;
  if (smem_u32(smem_raw) & 1023) {
    if (threadIdx.x == 0) atomicCAS(err, 0, 90);
    return;
  }
  if (threadIdx.x == 0) {
    s.abort_flag = 0;
    mbar_init(&s.a_full, 1);
    mbar_init(&s.a_empty, 1);
    for (int i = 0; i < S::kStages; ++i) {
      mbar_init(&s.b_full[i], 1);
      mbar_init(&s.b_empty[i], 1);
    }
    for (int i = 0; i < 2; ++i) {
      mbar_init(&s.acc_full[i], 1);
      mbar_init(&s.acc_empty[i], 8);  // 4 warps x 2 CTAs
    }
    mbar_init(&s.drained, 1);
    fence_barrier_init();
  }
  if (warp == 1) {
    asm volatile("tcgen05.alloc.cta_group::2.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(&s.tmem_base)),
                 "r"(512)
                 : "memory");
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::2.sync.aligned;" ::: "memory");
  }
  tc_fence_before();
  cluster_sync();  // both CTAs' barriers stand before the other uses them
  tc_fence_after();
  const uint32_t tmem = __shfl_sync(0xffffffffu, s.tmem_base, 0);
  int tile = (int)(u0 / heads) * 2 + rank, head = (int)(u0 % heads);  // an odd last tile has no partner
  const int n_units = (int)(u1 - u0);

  if (warp == 0) {
    if (elect_one()) {
      int sent = 0, na = 0;
      bool ok = true;
      for (int i = 0; ok && i < n_units; ++i) {
        if (i == 0 || head == 0) {
          if (na > 0 && !(ok = wait_or_abort(s, &s.a_empty, (na - 1) & 1, err, 97))) break;
          const bool real = tile < nwork;
          const int32_t* si = seq_info + 5 * (real ? work[2 * tile] : 0);
          const int r0 = real ? work[2 * tile + 1] : 0, ctx = real ? si[2] : 0;
          const int32_t* bt = block_tables + (int64_t)si[3] * max_blocks;
          if (rank == 0) mbar_arrive_expect_tx(&s.a_full, 2 * S::kChunks * 128 * 128);
          int y[8];  // the block ids first: their loads are independent of each other
#pragma unroll
          for (int g = 0; g < 8; ++g) {
            const int r = g * page;
            y[g] = (int)(r < 128 && r0 + r < ctx ? page_row(bt, r0 + r, page, num_blocks, err) : num_blocks * page);
          }
#pragma unroll
          for (int g = 0; g < 8; ++g)
            if (g * page < 128)
#pragma unroll
              for (int c = 0; c < S::kChunks; ++c)
                tma_load_pair(s.a[c] + g * page * 128, &c_map, &s.a_full, c * 64, y[g]);
          ++na;
        }
        for (int ks = 0; ks < S::kChunks; ++ks, ++sent) {
          const int st = sent % S::kStages;
          if (sent >= S::kStages) ok = wait_or_abort(s, &s.b_empty[st], (sent / S::kStages - 1) & 1, err, 97);
          if (!ok) break;
          if (rank == 0) mbar_arrive_expect_tx(&s.b_full[st], 2 * 128 * 128);
          tma_load_pair(s.b[st], &w_map, &s.b_full[st], ks * 64, head * 256 + rank * 128);
        }
        if (++head == heads) head = 0, tile += 2;
      }
      // both CTAs' copies in flight end before the pair does, on the way out of a time-out too
      if (rank == 0) {
        if (na > 0) mbar_wait_sleep(&s.a_full, (na - 1) & 1);
        for (int i = max(0, sent - S::kStages); i < sent; ++i)
          mbar_wait_sleep(&s.b_full[i % S::kStages], (i / S::kStages) & 1);
      }
    }
  } else if (warp == 1) {
    if (rank == 0 && elect_one()) {
      constexpr uint32_t idesc = idesc_bf16<256, 256>();
      const uint64_t a_desc = smem_desc_sw128(smem_u32(s.a[0])), b_desc = smem_desc_sw128(smem_u32(s.b[0]));
      int seen = 0, na = 0;
      bool ok = true;
      for (int i = 0; ok && i < n_units; ++i) {
        if (i == 0 || head == 0) ok = wait_or_abort(s, &s.a_full, na++ & 1, err, 98);
        if (i >= 2) ok = ok && wait_or_abort(s, &s.acc_empty[i & 1], ((i >> 1) - 1) & 1, err, 98);
        const uint32_t d = tmem + (i & 1) * 256;
        for (int ks = 0; ok && ks < S::kChunks; ++ks, ++seen) {
          const int st = seen % S::kStages;
          ok = wait_or_abort(s, &s.b_full[st], (seen / S::kStages) & 1, err, 98);
          if (!ok) break;
          tc_fence_after();
          const uint64_t a = a_desc + ks * 1024, b = b_desc + st * 1024;
#pragma unroll
          for (int kk = 0; kk < 4; ++kk) mma_pair(d, a + kk * 2, b + kk * 2, idesc, ks + kk > 0);
          commit_pair(&s.b_empty[st]);
        }
        if (!ok) break;
        commit_pair(&s.acc_full[i & 1]);
        if (++head == heads) {
          head = 0;
          commit_pair(&s.a_empty);
        }
      }
      commit_pair(&s.drained);
    }
  } else {
    const int quad = warp & 3;
    uint8_t* slab = s.slab[quad];
    const uint32_t lane_off = (uint32_t)(quad * 32) << 16;
    for (int i = 0; i < n_units; ++i) {
      const bool real = tile < nwork;
      const int32_t* si = seq_info + 5 * (real ? work[2 * tile] : 0);
      const int r0 = real ? work[2 * tile + 1] + quad * 32 : 0, ctx = real ? si[2] : 0;  // this warp's 32 rows
      const int64_t row0 = (int64_t)si[4] + r0;
      const int valid = ctx - r0, padded = min(32, (ctx + 15) / 16 * 16 - r0);
      if (head == 0 && k_rope != nullptr) {
        const int32_t* bt = block_tables + (int64_t)si[3] * max_blocks;
#pragma unroll
        for (int k = 0; k < 8; ++k) {  // 4 rows x 8 lanes
          const int r = 4 * k + (lane >> 3), seg = lane & 7;
          if (r < padded) {
            uint4 x = make_uint4(0, 0, 0, 0);
            if (r < valid) {
              const int64_t at = page_row(bt, r0 + r, page, num_blocks, err) + (r0 + r) % page;
              if (at < num_blocks * page)
                x = *reinterpret_cast<const uint4*>(cache + at * (R + kRot) + R + seg * 8);
            }
            *reinterpret_cast<uint4*>(k_rope + (row0 + r) * kRot + seg * 8) = x;
          }
        }
      }
      const bool ok = wait_or_abort(s, &s.acc_full[i & 1], (i >> 1) & 1, err, 99);
      if (!__all_sync(0xffffffffu, ok)) break;
      tc_fence_after();
      bf16* dst = kv + row0 * kv_stride + head * 256;
#pragma unroll 1
      for (int c = 0; c < 256; c += 64) {
        uint4* mine = reinterpret_cast<uint4*>(slab + lane * kSlabPitch);
#pragma unroll
        for (int half = 0; half < 2; ++half) {
          float v[32];
          tmem_ld32w(tmem + lane_off + (i & 1) * 256 + c + half * 32, v);
          if (lane >= valid) {
#pragma unroll
            for (int e = 0; e < 32; ++e) v[e] = 0.f;
          }
#pragma unroll
          for (int q = 0; q < 4; ++q)
            mine[half * 4 + q] =
                make_uint4(pack_bf16(v[8 * q], v[8 * q + 1]), pack_bf16(v[8 * q + 2], v[8 * q + 3]),
                           pack_bf16(v[8 * q + 4], v[8 * q + 5]), pack_bf16(v[8 * q + 6], v[8 * q + 7]));
        }
        __syncwarp();
        if (c == 192) {  // the accumulator has been read
          tc_fence_before();
          if (lane == 0) arrive_leader(&s.acc_empty[i & 1]);
        }
#pragma unroll
        for (int k = 0; k < 8; ++k) {
          const int r = 4 * k + (lane >> 3), seg = lane & 7;
          if (r < padded)
            *reinterpret_cast<uint4*>(dst + r * kv_stride + c + seg * 8) =
                *reinterpret_cast<const uint4*>(slab + r * kSlabPitch + seg * 16);
        }
        __syncwarp();
      }
      if (++head == heads) head = 0, tile += 2;
    }
  }
  tc_fence_before();
  __syncthreads();
  if (threadIdx.x == 32) mbar_wait_sleep(&s.drained, 0);  // every MMA has finished before tensor memory is freed
  __syncthreads();
  cluster_sync();  // no CTA leaves while its peer may still signal it
  tc_fence_after();
  if (warp == 1)
    asm volatile("tcgen05.dealloc.cta_group::2.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(512) : "memory");
}

// ------------------------------------------------------------------ attention
//
// One CTA per (256 query tokens of a sequence, head): two tiles of 128 rows share every K and V
// tile of 128 keys.  Per row tile t and key tile j:
//   S_t = Q_t K_j^T     tcgen05.mma, K-major operands in shared memory -> 128 TMEM columns
//   P_t = 2^(S_t - m)   one thread a row, packed to bf16 (the MMA's operand type; the row
//                       sums are of the fp32 values) over S_t's columns
//   O_t += P_t V_j      tcgen05.mma, P from TMEM, V MN-major from shared memory
// The MMA thread issues PV_0(j), S_0(j+1), PV_1(j), S_1(j+1): while one row tile's softmax runs, the
// tensor cores work on the other.  K (3 x 16 KB) and V (2 x 16 KB) tiles go through a
// ring of eight 16 KB slots, 128 keys x 64 dims each.
//
// S_t(j + 1) is issued after PV_t(j) by the same thread, so once its scores are complete O_t is at
// rest: the softmax warps themselves rescale it, and only when a score exceeds the running
// maximum by 8 (in log2; p <= 256 loses nothing in bf16 or fp32).
// A CTA with 128 rows or fewer gives its two halves the even and the odd key tiles of the same
// rows instead (and the second half's m, l and O join the first's at the end): the chain of
// scores, softmax and product that bounds a lone row tile is half as long.
//
// Where the CTAs are too few for the GPU, the longest row tiles have their keys cut into parts of
// part_tiles key tiles, a CTA each, that give fp32 partial results per row, which
// latent_prefill_join_kernel joins.  Row tiles no longer than a part stay whole.
//
// Keys past a row's position have p = 0.  PV stops at the row tile's last key, rounded up
// to 16; the rows there are the expansion's zeros, so nothing behind a sequence is read.
constexpr int kThreads = 384;  // warp 0 TMA, warp 1 MMA, warps 4-7 and 8-11 softmax of row tile 0 and 1
constexpr int kSlots = 8;
constexpr uint32_t kSlotBytes = 128 * 128;
constexpr float kRaise = 8.f;
constexpr float kNoMax = -1e30f;

struct alignas(1024) PrefillSmem {
  uint8_t q[2][3][kSlotBytes];
  uint8_t ring[kSlots][kSlotBytes];
  uint64_t q_full, k_full[2], k_empty[2], v_full[2], v_empty[2], s_full[2], p_full[2], o_full[2], drained;
  uint32_t tmem_base;
  volatile int abort_flag;
};

__device__ __forceinline__ float ex2(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}

// Two fp32 values as one 64-bit operand of the packed instructions (one issue slot for both).
__device__ __forceinline__ uint64_t pair(float a, float b) {
  uint64_t r;
  asm("mov.b64 %0, {%1, %2};" : "=l"(r) : "f"(a), "f"(b));
  return r;
}
__device__ __forceinline__ void unpair(uint64_t v, float& a, float& b) {
  asm("mov.b64 {%0, %1}, %2;" : "=f"(a), "=f"(b) : "l"(v));
}
__device__ __forceinline__ uint64_t fma2(uint64_t a, uint64_t b, uint64_t c) {
  uint64_t r;
  asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(r) : "l"(a), "l"(b), "l"(c));
  return r;
}
__device__ __forceinline__ uint64_t add2(uint64_t a, uint64_t b) {
  uint64_t r;
  asm("add.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b));
  return r;
}
__device__ __forceinline__ float max3(float a, float b, float c) {
  float r;
  asm("max.f32 %0, %1, %2, %3;" : "=f"(r) : "f"(a), "f"(b), "f"(c));
  return r;
}

// P of one row of a key tile relative to the running maximum m: 128 scores from TMEM, 64
// packed bf16 pairs, their fp32 sum, and the largest relative score.  The load of the
// next 32 columns is under way while 32 are worked on.  The scaled scores are rounded before m is
// taken off, as m's own was, so that the largest is 0 at any size: scale * s - m in one
// rounding is up to half of m's last place there, from 2^28 on more than kRaise whatever m is.  (A packed
// product by itself was seen to be contracted with the packed sum; an fma is not.)
template <bool MASKED>
__device__ __forceinline__ float row_pass(uint32_t s_tmem, float scale_log2, float m, int limit, uint32_t (&p)[64],
                                          float& sum) {
  const uint64_t sc = pair(scale_log2, scale_log2), off = pair(-m, -m), zero = pair(0.f, 0.f);
  float top = -INFINITY;
  uint64_t acc = pair(0.f, 0.f);
  uint32_t v[2][32];
  tmem_ld_start(s_tmem, v[0]);
#pragma unroll
  for (int c = 0; c < 4; ++c) {
    tmem_ld_wait(v[c & 1]);
    if (c < 3) tmem_ld_start(s_tmem + (c + 1) * 32, v[(c + 1) & 1]);
#pragma unroll
    for (int i = 0; i < 32; i += 2) {
      float x0, x1;
      unpair(add2(fma2(pair(__uint_as_float(v[c & 1][i]), __uint_as_float(v[c & 1][i + 1])), sc, zero), off), x0, x1);
      if (MASKED) {
        if (c * 32 + i > limit) x0 = -INFINITY;
        if (c * 32 + i + 1 > limit) x1 = -INFINITY;
      }
      top = max3(top, x0, x1);
      const float p0 = ex2(x0), p1 = ex2(x1);
      acc = add2(acc, pair(p0, p1));
      p[c * 16 + i / 2] = pack_bf16(p0, p1);
    }
  }
  float a, b;
  unpair(acc, a, b);
  sum = a + b;
  return top;
}

__global__ void __launch_bounds__(kThreads, 1)
    latent_prefill_kernel(const __grid_constant__ CUtensorMap q_map, const __grid_constant__ CUtensorMap kv_map,
                          const __grid_constant__ CUtensorMap rope_map, const int32_t* work,
                          const int32_t* seq_info, int64_t q_rows, float scale_log2,
                          bf16* out, int64_t out_stride, int cut, int part_tiles, int slots, float* part_o,
                          float2* part_ml, int* err) {
  griddep_entry();
  extern __shared__ __align__(1024) uint8_t smem_raw[];
  PrefillSmem& s = *reinterpret_cast<PrefillSmem*>(smem_raw);
  const int warp = __shfl_sync(0xffffffffu, threadIdx.x / 32, 0), lane = threadIdx.x % 32;
  const int h = blockIdx.y;
  // `slots` CTAs a row tile that is cut, one for each of the others
  const int cut_ctas = cut * slots, bx = blockIdx.x;
  const bool parted = bx < cut_ctas;
  const int tile = parted ? bx / slots : cut + bx - cut_ctas, part = parted ? bx - tile * slots : 0;
  const int32_t* si = seq_info + 5 * work[2 * tile];
  const int t0 = work[2 * tile + 1];
  const int row0 = si[0] + t0, n = si[1] - t0;  // n: rows from t0 on
  // this CTA's key tiles; keys and positions count from its first key
  const int all_keys = si[2] - si[1] + t0 + min(n, 256), all_tiles = (all_keys + 127) / 128;
  const int range = 128 * (parted ? part_tiles : all_tiles), key0 = part * range;
  const int pos0 = si[2] - si[1] + t0 - key0, kv0 = si[4] + key0;
  // keys of the two halves, key tiles of the CTA and of each half
  const bool split = n <= 128;
  const int keys0 = max(0, min(range, pos0 + min(n, 128)));
  const int keys1 = split ? keys0 : max(0, min(range, pos0 + min(n, 256)));
  const int nt = (keys1 + 127) / 128;
  const int nt0 = split ? (nt + 1) / 2 : (keys0 + 127) / 128, nt1 = split ? nt / 2 : nt;
  const int64_t part_row = ((int64_t)(part * gridDim.y + h) * cut + tile) * 256;
  if ((smem_u32(smem_raw) & 1023) || row0 < 0 || row0 + min(n, 256) > q_rows || n <= 0) {
    if (threadIdx.x == 0) atomicCAS(err, 0, 90);
    return;
  }
  if (key0 >= all_keys) return;  // this row tile has fewer parts than the longest

  if (threadIdx.x == 0) {
    s.abort_flag = 0;
    mbar_init(&s.q_full, 1);
    for (int i = 0; i < 2; ++i) {
      mbar_init(&s.k_full[i], 1);
      mbar_init(&s.k_empty[i], 1);
      mbar_init(&s.v_full[i], 1);
      mbar_init(&s.v_empty[i], 1);
      mbar_init(&s.s_full[i], 1);
      mbar_init(&s.p_full[i], 4);
      mbar_init(&s.o_full[i], 1);
    }
    mbar_init(&s.drained, 1);
    fence_barrier_init();
  }
  if (warp == 1) tmem_alloc(&s.tmem_base, 512);
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = __shfl_sync(0xffffffffu, s.tmem_base, 0);  // S_0, S_1, O_0, O_1: 128 columns each

  if (warp == 0) {
    // ------------------------------------------------------------ TMA producer
    if (elect_one()) {
      const int tiles_q = split ? 1 : 2;
      mbar_arrive_expect_tx(&s.q_full, tiles_q * 3 * kSlotBytes);
      for (int t = 0; t < tiles_q; ++t)
        for (int c = 0; c < 3; ++c) tma_load_2d(s.q[t][c], &q_map, &s.q_full, h * 192 + c * 64, row0 + t * 128);
      // Slots of tile j: keys 5j .. 5j + 2, values 5j + 3, 5j + 4 (mod 8).  Those of K_j were
      // last used by K_{j-2} and V_{j-2}, those of V_j by K_{j-1}, which is free once the last
      // scores of tile j - 1 are complete.  The empty barriers go by the tile's parity: their
      // next phase needs a tile that this thread has not sent yet, so none can be missed.
      bool ok = true;
      int j = 0;
      for (; j < nt; ++j) {
        if (j >= 2 && !wait_or_abort(s, &s.v_empty[j & 1], ((j >> 1) - 1) & 1, err, 91)) { ok = false; break; }
        uint64_t* bar = &s.k_full[j & 1];
        mbar_arrive_expect_tx(bar, 3 * kSlotBytes);
        tma_load_2d(s.ring[(5 * j) % kSlots], &kv_map, bar, h * 256, kv0 + j * 128);
        tma_load_2d(s.ring[(5 * j + 1) % kSlots], &kv_map, bar, h * 256 + 64, kv0 + j * 128);
        tma_load_2d(s.ring[(5 * j + 2) % kSlots], &rope_map, bar, 0, kv0 + j * 128);
        if (j >= 1 && !wait_or_abort(s, &s.k_empty[(j - 1) & 1], ((j - 1) >> 1) & 1, err, 91)) { ok = false; break; }
        bar = &s.v_full[j & 1];
        mbar_arrive_expect_tx(bar, 2 * kSlotBytes);
        tma_load_2d(s.ring[(5 * j + 3) % kSlots], &kv_map, bar, h * 256 + 128, kv0 + j * 128);
        tma_load_2d(s.ring[(5 * j + 4) % kSlots], &kv_map, bar, h * 256 + 192, kv0 + j * 128);
      }
      // the copies in flight end before the CTA does, on the way out of a time-out too
      mbar_wait_sleep(&s.q_full, 0);
      for (int i = max(0, j - 2); i < j; ++i) {
        mbar_wait_sleep(&s.k_full[i & 1], (i >> 1) & 1);
        mbar_wait_sleep(&s.v_full[i & 1], (i >> 1) & 1);
      }
      if (!ok) mbar_wait_sleep(&s.k_full[j & 1], (j >> 1) & 1, 10000000ull);  // if it was sent
    }
  } else if (warp == 1) {
    // -------------------------------------------------------------- MMA issuer
    if (elect_one()) {
      constexpr uint32_t idesc_s = idesc_bf16<128, 128>();
      constexpr uint32_t idesc_o = idesc_bf16<128, 128>() | kIdescBMn;
      constexpr uint64_t kSlotStep = kSlotBytes >> 4;
      const uint64_t q_desc = smem_desc_sw128(smem_u32(s.q[0][0])), k_desc = smem_desc_sw128(smem_u32(s.ring[0]));
      const uint64_t v_desc = smem_desc_mn_sw128(smem_u32(s.ring[0]), kSlotBytes, 1024);
      bool ok = wait_or_abort(s, &s.q_full, 0, err, 92);
      auto issue_s = [&](int t, int j) {  // scores of half t
        ok = ok && wait_or_abort(s, &s.k_full[j & 1], (j >> 1) & 1, err, 93);
        if (!ok) return;
        tc_fence_after();
#pragma unroll
        for (int c = 0; c < 3; ++c) {
          const uint64_t a = q_desc + (split ? c : t * 3 + c) * kSlotStep;
          const uint64_t b = k_desc + ((5 * j + c) % kSlots) * kSlotStep;
#pragma unroll
          for (int kk = 0; kk < 4; ++kk) mma_bf16(tmem + t * 128, a + kk * 2, b + kk * 2, idesc_s, c + kk > 0);
        }
        mma_commit(&s.s_full[t]);
        if (split || t == 1) mma_commit(&s.k_empty[j & 1]);  // the tile's last scores
      };
      auto issue_pv = [&](int t, int j, int keys, bool last) {
        const int i = split ? j >> 1 : j;  // the half's own count of tiles
        ok = ok && wait_or_abort(s, &s.v_full[j & 1], (j >> 1) & 1, err, 93);
        ok = ok && wait_or_abort(s, &s.p_full[t], i & 1, err, 94);
        if (!ok) return;
        tc_fence_after();
        // the two value chunks may wrap around the ring's end: one descriptor step between them
        const int s0 = (5 * j + 3) % kSlots, s1 = (5 * j + 4) % kSlots;
        const int steps = min(8, (keys - j * 128 + 15) / 16);
        const uint64_t v = v_desc + s0 * kSlotStep;
        if (s1 > s0 && steps == 8) {
#pragma unroll
          for (int kk = 0; kk < 8; ++kk)
            mma_bf16_tmem_a(tmem + 256 + t * 128, tmem + t * 128 + kk * 8, v + kk * 128, idesc_o, i + kk > 0);
        } else {
          constexpr uint32_t idesc_h = idesc_bf16<128, 64>() | kIdescBMn;
          for (int c = 0; c < 2; ++c)
            for (int kk = 0; kk < steps; ++kk)
              mma_bf16_tmem_a(tmem + 256 + t * 128 + c * 64, tmem + t * 128 + kk * 8,
                              v_desc + (c ? s1 : s0) * kSlotStep + kk * 128, idesc_h, i + kk > 0);
        }
        if (last) mma_commit(&s.v_empty[j & 1]);
      };
      if (nt0 > 0) issue_s(0, 0);
      if (!split || nt > 1) issue_s(1, split ? 1 : 0);
      for (int j = 0; ok && j < nt; ++j) {
        if (split) {
          const int t = j & 1;
          issue_pv(t, j, keys0, true);
          if (j + 2 < nt) {
            issue_s(t, j + 2);
          } else if (ok) {
            mma_commit(&s.o_full[t]);
          }
          continue;
        }
        if (j < nt0) {
          issue_pv(0, j, keys0, false);
          if (j + 1 < nt0) {
            issue_s(0, j + 1);
          } else if (ok) {
            mma_commit(&s.o_full[0]);
          }
        }
        issue_pv(1, j, keys1, true);
        if (j + 1 < nt) {
          issue_s(1, j + 1);
        } else if (ok) {
          mma_commit(&s.o_full[1]);
        }
      }
      // every MMA issued has finished before the tensor memory is freed
      mma_commit(&s.drained);
      mbar_wait_sleep(&s.drained, 0);
    }
  } else if (warp >= 4) {
    // ------------------------------------------------------- softmax, epilogue
    const int t = (warp - 4) / 4, quad = warp & 3;
    const int row = quad * 32 + lane + (split ? 0 : t * 128);
    const int keys = t ? keys1 : keys0, tiles = t ? nt1 : nt0;
    const int last_key = min(pos0 + row, keys - 1);  // this row's; rows past the chunk see the tile's keys
    const uint32_t s_tmem = tmem + t * 128 + ((uint32_t)(quad * 32) << 16);
    const uint32_t o_tmem = s_tmem + 256;
    float m = kNoMax, l = 0.f;
    bool fresh = true;  // any row of the warp without a maximum
    bool ok = true;
    for (int i = 0; i < tiles; ++i) {
      ok = wait_or_abort(s, &s.s_full[t], i & 1, err, 95);
      if (!__all_sync(0xffffffffu, ok)) {
        ok = false;
        break;
      }
      tc_fence_after();
      const int limit = last_key - (split ? 2 * i + t : i) * 128;  // columns up to this one count
      const bool masked = __any_sync(0xffffffffu, limit < 127);
      uint32_t p[64];
      float sum = 0.f;
      // The maximum is looked for where a row has none (the first tile, or later where its scores are all
      // -inf) and where a score passed the running one too far.  No score is above it then, and
      // the pass after it is the last.  One place for the pass: its code is long, and fetched
      // anew by every CTA.
      bool look = fresh;
#pragma unroll 1
      while (true) {
        if (look) {
          float top = -INFINITY;
#pragma unroll 1
          for (int c = 0; c < 4; ++c) {
            float v[32];
            tmem_ld32w(s_tmem + c * 32, v);
#pragma unroll
            for (int e = 0; e < 32; ++e) top = fmaxf(top, c * 32 + e > limit ? -INFINITY : v[e] * scale_log2);
          }
          float mn = fmaxf(m, top), f = ex2(m - mn);
          // a row without keys in the tile has none later: any reference
          if (m == kNoMax) mn = limit < 0 ? 0.f : top == -INFINITY ? kNoMax : top, f = 1.f;
          m = mn;
          fresh = __any_sync(0xffffffffu, m == kNoMax);
          if (i > 0 && __any_sync(0xffffffffu, f != 1.f)) {
            l *= f;
#pragma unroll 1
            for (int c = 0; c < 8; ++c) {
              float o[16];
              uint32_t u[16];
              tmem_ld16(o_tmem + c * 16, o);
#pragma unroll
              for (int e = 0; e < 16; ++e) u[e] = __float_as_uint(o[e] * f);
              tmem_st16(o_tmem + c * 16, u);
            }
          }
        }
        const float top = masked ? row_pass<true>(s_tmem, scale_log2, m, limit, p, sum)
                                 : row_pass<false>(s_tmem, scale_log2, m, limit, p, sum);
        if (look || !__any_sync(0xffffffffu, top > kRaise)) break;
        look = true;
      }
      l += sum;
#pragma unroll
      for (int c = 0; c < 4; ++c) {
        uint32_t u[16];
#pragma unroll
        for (int i = 0; i < 16; ++i) u[i] = p[c * 16 + i];
        tmem_st16(s_tmem + c * 16, u);
      }
      tmem_wait_st();
      tc_fence_before();
      __syncwarp();
      if (lane == 0) mbar_arrive(&s.p_full[t]);
    }
    if (ok && tiles > 0) ok = wait_or_abort(s, &s.o_full[t], 0, err, 96);
    ok = __all_sync(0xffffffffu, ok && tiles > 0);
    tc_fence_after();
    float f0 = 1.f, f1 = 0.f, m_out = m;  // factors of the halves' O, the maximum they count from
    // the second half's O [dim][row], m and l go through the ring: every tile of it has been used
    float* other = reinterpret_cast<float*>(s.ring[0]);
    const int at = quad * 32 + lane;
    if (split) {
      if (t == 1) {
        if (!ok) l = 0.f;
        wait_or_abort(s, &s.o_full[0], 0, err, 96);  // the first half's tiles are in the ring too
        __syncwarp();
        if (ok) {
#pragma unroll 1
          for (int c = 0; c < 8; ++c) {
            float o[16];
            tmem_ld16(o_tmem + c * 16, o);
#pragma unroll
            for (int e = 0; e < 16; ++e) other[(c * 16 + e) * 128 + at] = o[e];
          }
        }
        other[128 * 128 + at] = m;
        other[129 * 128 + at] = l;
      }
      asm volatile("bar.sync 1, 256;" ::: "memory");
      if (t == 0) {
        const float m1 = other[128 * 128 + at], l1 = other[129 * 128 + at];
        if (l1 != 0.f) {  // a row without keys in the second half, or a half without tiles: 0
          const float top = l == 0.f ? m1 : fmaxf(m, m1);
          f0 = l == 0.f ? 0.f : ex2(m - top), f1 = ex2(m1 - top);
          l = l * f0 + l1 * f1;
          m_out = top;
        }
      }
    }
    if (parted) {
      if (!(split && t == 1)) {
        const float inv = !ok || l == 0.f ? 0.f : 1.f / l;
        part_ml[part_row + row] = !ok || l == 0.f ? make_float2(-INFINITY, 0.f) : make_float2(m_out, l);
        if (split) part_ml[part_row + row + 128] = make_float2(-INFINITY, 0.f);
        float* dst = part_o + (part_row + row) * kVal;
        for (int c = 0; ok && c < 8; ++c) {
          float o[16];
          tmem_ld16(o_tmem + c * 16, o);
          if (__any_sync(0xffffffffu, f1 != 0.f)) {
#pragma unroll
            for (int e = 0; e < 16; ++e)
              o[e] = o[e] * f0 + (f1 != 0.f ? other[(c * 16 + e) * 128 + at] * f1 : 0.f);
          }
#pragma unroll
          for (int e = 0; e < 16; e += 4)
            *reinterpret_cast<float4*>(dst + c * 16 + e) =
                make_float4(o[e] * inv, o[e + 1] * inv, o[e + 2] * inv, o[e + 3] * inv);
        }
      }
    } else if (ok && !(split && t == 1)) {
      const float inv = l == 0.f ? 0.f : 1.f / l;  // a row without a finite score: zeros, as in the other forms
      bf16* dst = out + (int64_t)(row0 + row) * out_stride + (int64_t)h * kVal;
#pragma unroll 1
      for (int c = 0; c < 8; ++c) {
        float o[16];
        tmem_ld16(o_tmem + c * 16, o);
        if (__any_sync(0xffffffffu, f1 != 0.f)) {
#pragma unroll
          for (int e = 0; e < 16; ++e)
            o[e] = o[e] * f0 + (f1 != 0.f ? other[(c * 16 + e) * 128 + at] * f1 : 0.f);
        }
        if (row < n) {
#pragma unroll
          for (int e = 0; e < 16; ++e) o[e] *= inv;
#pragma unroll
          for (int e = 0; e < 16; e += 8)
            *reinterpret_cast<uint4*>(dst + c * 16 + e) =
                make_uint4(pack_bf16(o[e], o[e + 1]), pack_bf16(o[e + 2], o[e + 3]), pack_bf16(o[e + 4], o[e + 5]),
                           pack_bf16(o[e + 6], o[e + 7]));
        }
      }
    }
  }
  tc_fence_before();
  __syncthreads();
  if (warp == 1) {
    tc_fence_after();
    tmem_dealloc(tmem, 512);
  }
}

// out = sum_z w_z o_z / sum_z w_z over the parts z of a row tile's keys, w_z = l_z 2^(m_z - M) of their maxima and sums
// (kept apart: m_z + log2 l_z would round l_z to m_z's last place): one warp per (row of a
// row tile, head), 4 dims a lane.
__global__ void __launch_bounds__(256) latent_prefill_join_kernel(const float* part_o, const float2* part_ml,
                                                                  int part_tiles, int slots, const int32_t* work,
                                                                  const int32_t* seq_info, bf16* out,
                                                                  int64_t out_stride) {
  griddep_entry();
  const int row = blockIdx.z * 8 + (threadIdx.x >> 5), lane = threadIdx.x & 31, h = blockIdx.y;
  const int32_t* si = seq_info + 5 * work[2 * blockIdx.x];
  const int t0 = work[2 * blockIdx.x + 1];
  if (t0 + row >= si[1]) return;
  const int keys = si[2] - si[1] + t0 + min(si[1] - t0, 256);
  const bool mine = lane < slots && lane * part_tiles * 128 < keys;  // lane z: part z
  const int parts = __popc(__ballot_sync(0xffffffffu, mine));
  const int64_t first = ((int64_t)h * gridDim.x + blockIdx.x) * 256 + row, step = (int64_t)gridDim.y * gridDim.x * 256;
  const float2 ml = mine ? part_ml[first + lane * step] : make_float2(-INFINITY, 0.f);
  float M = warp_max(ml.x);
  if (M == -INFINITY) M = 0.f;
  const float e = ml.y * ex2(ml.x - M), L = warp_sum(e);
  const float w = L == 0.f ? 0.f : e / L;
  float4 x = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll 4
  for (int z = 0; z < parts; ++z) {
    const float f = __shfl_sync(0xffffffffu, w, z);
    if (f != 0.f) {  // a part without keys of this row may have written no result
      const float4 y = *reinterpret_cast<const float4*>(part_o + (first + z * step) * kVal + lane * 4);
      x.x += f * y.x, x.y += f * y.y, x.z += f * y.z, x.w += f * y.w;
    }
  }
  *reinterpret_cast<uint2*>(out + (int64_t)(si[0] + t0 + row) * out_stride + h * kVal + lane * 4) =
      make_uint2(pack_bf16(x.x, x.y), pack_bf16(x.z, x.w));
}

}  // namespace

void launch_latent_expand(const LatentExpand& a, cudaStream_t st) {
  if (a.nwork == 0 || a.heads == 0) return;
  auto go = [&](auto kern, size_t smem, std::atomic<uint64_t>& attr_devs) {
    ensure_smem_attr(attr_devs, kern, smem);
    const CUtensorMap tc = make_tmap_2d_bf16(a.cache, (uint64_t)a.num_blocks * a.page, a.R + kRot, a.R + kRot, a.page, 64, true);
    const CUtensorMap tw = make_tmap_2d_bf16(a.w, (uint64_t)a.heads * 256, a.R, a.R, 128, 64, true);
    const int grid = 2 * (int)std::max<int64_t>(1, std::min<int64_t>(a.num_sms / 2, (int64_t)((a.nwork + 1) / 2) * a.heads));
    launch_k(kern, dim3(grid), kExpandThreads, smem, st, tc, tw, a.cache, a.num_blocks, a.page, a.work, a.nwork,
             a.seq_info, a.block_tables, a.max_blocks, a.heads, a.kv, a.kv_stride, a.k_rope, a.err);
    KAPSL_LAUNCH_CHECK();
    note_launch();
  };
  static_assert(sizeof(ExpandSmem<512>) <= 232448 && sizeof(ExpandSmem<256>) <= 232448, "shared memory of one CTA");
  static std::atomic<uint64_t> attr512{0}, attr256{0};
  if (a.R == 512) {
    go(latent_expand_kernel<512>, sizeof(ExpandSmem<512>), attr512);
  } else if (a.R == 256) {
    go(latent_expand_kernel<256>, sizeof(ExpandSmem<256>), attr256);
  } else {
    throw std::runtime_error("latent prefill: the latent must have 256 or 512 values");
  }
}

void launch_latent_prefill(const LatentPrefill& a, cudaStream_t st) {
  if (a.nwork == 0 || a.heads == 0) return;
  const size_t smem = sizeof(PrefillSmem);
  static_assert(sizeof(PrefillSmem) <= 232448, "shared memory of one CTA");
  static std::atomic<uint64_t> attr_devs{0};
  ensure_smem_attr(attr_devs, latent_prefill_kernel, smem);
  const CUtensorMap tq = make_tmap_2d_bf16(a.q, a.T, (uint64_t)a.heads * (kNope + kRot), a.q_stride, 128, 64, true);
  const CUtensorMap tkv = make_tmap_2d_bf16(a.kv, a.kv_rows, (uint64_t)a.heads * (kNope + kVal), a.kv_stride, 128, 64, true);
  const CUtensorMap tr = make_tmap_2d_bf16(a.k_rope, a.kv_rows, kRot, kRot, 128, 64, true);
  launch_k(latent_prefill_kernel, dim3(a.cut * a.slots + a.nwork - a.cut, a.heads), kThreads, smem, st, tq, tkv, tr,
           a.work, a.seq_info, a.T, a.scale * kLog2e, a.out, a.out_stride, a.cut, a.part_tiles, a.slots, a.part_o,
           a.part_ml, a.err);
  KAPSL_LAUNCH_CHECK();
  note_launch();
  if (a.cut == 0) return;
  launch_k(latent_prefill_join_kernel, dim3(a.cut, a.heads, 32), 256, 0, st, a.part_o, a.part_ml, a.part_tiles, a.slots,
           a.work, a.seq_info, a.out, a.out_stride);
  KAPSL_LAUNCH_CHECK();
  note_launch();
}

}  // namespace kapsl
