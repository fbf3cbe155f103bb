// Absorbed latent attention for single tokens over a paged latent cache.
//
// A cache row is [c (R) | k_r (64)], shared by every head.  Head h has the key
// expansion K_h = w[h, :128] and the value expansion V_h = w[h, 128:], both [128, R].
// With the key expansion moved to the query's side,
//   qa_h = [K_h^T q_h[:128] | q_h[128:]],   s_j = scale * qa_h . row_j,
//   o_h = sum_j softmax(s)_j c_j,           out_h = V_h o_h,
// so the cache is read once for all heads and nothing is expanded per token.
//
// Three launches: absorb (qa), attention over splits of the context (fp32 partials of
// o), and one that joins the splits and applies V_h.
#include <algorithm>

#include "common.cuh"
#include "kernels.h"
#include "tcgen05.cuh"

namespace kapsl {
using namespace tc;

using bf16 = __nv_bfloat16;

namespace {

constexpr int kNope = 128, kRot = 64, kVal = 128;
constexpr int kMaxSplits = 64;
constexpr float kLog2e = 1.4426950408889634f;

// ------------------------------------------------------------------ attention
//
// One CTA per (split, up to 64 heads, sequence).  The products are transposed so
// that the heads are the MMA's N, which may be 16, 32 or 64 without wasted rows:
//   S^T [64 keys, heads] = K . qa^T    (M = 64, K tile K-major)
//   O^T [R dims, heads] += c^T . P^T   (M = 128 x R / 128; the same K tile read MN-major)
// so a key tile is loaded once and serves both products, and O^T of 64 heads takes 256
// of the 512 TMEM columns, which leaves room for two S^T tiles.
//
// Warp 0 loads 64-key tiles by TMA into a ring, warp 1 issues the MMAs, warps 2-5
// do the softmax: a tile's column maxima by register/shuffle exchange and shared
// memory, P rounded to bf16 (the operand type of the second product; the row sums are
// of the fp32 values).  The running maximum is raised, and O^T rescaled in TMEM, only
// when a score exceeds it by 2^8: p <= 256 loses nothing in bf16 or fp32, and the
// final division uses the same maximum.  Keys past the context have p = 0 and their
// cache rows are cleared in shared memory, since 0 * NaN of a stale row would count.
constexpr int kKeys = 64;
constexpr int kSoft = 4;  // softmax warps
constexpr int kThreads = (2 + kSoft) * 32;
constexpr float kRaise = 8.f;

template <int R, int NT>
struct Shape {
  static constexpr int W = R + kRot;
  static constexpr int kChunks = W / 64;
  static constexpr uint32_t kChunkBytes = kKeys * 128;        // 64 keys x 64 dims
  static constexpr uint32_t kTileBytes = kChunks * kChunkBytes;
  static constexpr uint32_t kQChunk = NT * 128;
  static constexpr uint32_t kQBytes = kChunks * kQChunk;
  static constexpr int kStages = R == 512 ? 2 : 4;  // what 227 KB hold beside 64 heads' queries
  static constexpr uint32_t kP = kKeys * 128;
};

template <int R, int NT>
struct DecodeSmem {
  using S = Shape<R, NT>;
  alignas(1024) uint8_t k[S::kStages][S::kTileBytes];
  alignas(1024) uint8_t q[S::kQBytes];
  alignas(1024) uint8_t p[S::kP];
  float red[2][kSoft][NT];  // per warp column maxima (tiles alternate), then sums
  uint64_t q_full, kv_full[S::kStages], kv_empty[S::kStages], s_full[2], s_free[2], p_full, pv_done, drained;
  uint32_t tmem_base;
  volatile int abort_flag;
};

// Bounded wait (2 s); a time-out records `code`, and every other wait of the CTA gives up
// with it.  The softmax warps go on through their loop after one (they share block
// barriers), on whatever the buffers hold.
template <class Smem>
__device__ __forceinline__ bool wait_or_abort(Smem& s, uint64_t* bar, uint32_t parity, int* err, int code) {
  if (mbar_try_wait(bar, parity)) return true;
  const uint64_t t0 = globaltimer_ns();
  while (!s.abort_flag) {
    if (mbar_try_wait_sleep(bar, parity, 20000u)) return true;
    if (globaltimer_ns() - t0 > 2000000000ull) {
      atomicCAS(err, 0, code);
      s.abort_flag = 1;
    }
  }
  return false;
}

__device__ __forceinline__ void soft_barrier() { asm volatile("bar.sync 1, %0;" ::"n"(kSoft * 32) : "memory"); }

// Reduces v[n] over the 8 lanes that share lane % 4 (rows of an accumulator fragment)
// and leaves in v[0 .. out) the results of columns `first ..`: each step a lane keeps half of
// its columns and sends the other half, 14 shuffles for 16 columns instead of 48.
template <int V, class F>
__device__ __forceinline__ int reduce_columns(float (&v)[V], F f) {
  const int lane = threadIdx.x & 31;
  int first = 0;
  int n = V;
#pragma unroll
  for (int mask = 16; mask >= 4; mask >>= 1) {
    const bool hi = (lane & mask) != 0;
    if (n > 1) {
      n >>= 1;
#pragma unroll
      for (int i = 0; i < V / 2; ++i) {
        if (i < n) {
          const float keep = hi ? v[i + n] : v[i], send = hi ? v[i] : v[i + n];
          v[i] = f(keep, __shfl_xor_sync(0xffffffffu, send, mask));
        }
      }
      first += hi ? n : 0;
    } else {
      v[0] = f(v[0], __shfl_xor_sync(0xffffffffu, v[0], mask));
    }
  }
  return first;
}

// column of a thread's n-th column value (pairs of adjacent columns, 8 apart)
__device__ __forceinline__ int frag_col(int n) { return (n >> 1) * 8 + (threadIdx.x & 3) * 2 + (n & 1); }

// The values of columns c .. c + 15 in every lane, from the lanes that hold them (v indexed as
// frag_col).
template <int V>
__device__ __forceinline__ void columns16(const float (&v)[V], int c, float (&out)[16]) {
#pragma unroll
  for (int n = 0; n < 16; ++n)
    out[n] = __shfl_sync(0xffffffffu, v[((c + n) >> 3) * 2 + (n & 1)], (n & 7) >> 1);
}

template <int R, int NT>
__global__ void __launch_bounds__(kThreads, 1)
    latent_attn_kernel(const __grid_constant__ CUtensorMap q_map, const __grid_constant__ CUtensorMap c_map,
                       int64_t num_blocks, int page, const int32_t* __restrict__ block_tables, int max_blocks,
                       const int32_t* __restrict__ ctx_lens, float* __restrict__ part_o,
                       float* __restrict__ part_lse, int H, int heads_per_cta, int nsplit, float scale_log2,
                       int* __restrict__ err) {
  griddep_entry();
  using S = Shape<R, NT>;
  extern __shared__ __align__(1024) uint8_t smem_raw[];
  DecodeSmem<R, NT>& s = *reinterpret_cast<DecodeSmem<R, NT>*>(smem_raw);
  const int warp = threadIdx.x / 32, lane = threadIdx.x % 32;
  const int split = blockIdx.x, b = blockIdx.z;
  const int h0 = blockIdx.y * heads_per_cta, nheads = min(heads_per_cta, H - h0);
  const int ctx = max(0, min(ctx_lens[b], max_blocks * page));
  const int tiles_all = (ctx + kKeys - 1) / kKeys;
  const int per = (tiles_all + nsplit - 1) / nsplit;
  const int tile0 = split * per;
  const int ntiles = max(0, min(tiles_all, tile0 + per) - tile0);
  const int64_t part0 = ((int64_t)b * H + h0) * nsplit + split;  // + head * nsplit
  if (ntiles == 0) {
    if (threadIdx.x < nheads) part_lse[part0 + (int64_t)threadIdx.x * nsplit] = -INFINITY;
    return;
  }
  if (smem_u32(smem_raw) & 1023) {  // the swizzled tiles need it
    if (threadIdx.x == 0) atomicCAS(err, 0, 83);
    return;
  }

  if (threadIdx.x == 0) {
    s.abort_flag = 0;
    mbar_init(&s.q_full, 1);
    for (int i = 0; i < S::kStages; ++i) {
      mbar_init(&s.kv_full[i], 1);
      mbar_init(&s.kv_empty[i], 1);
    }
    for (int i = 0; i < 2; ++i) {
      mbar_init(&s.s_full[i], 1);
      mbar_init(&s.s_free[i], kSoft * 32);
    }
    mbar_init(&s.p_full, kSoft * 32);
    mbar_init(&s.pv_done, 1);
    mbar_init(&s.drained, 1);
    fence_barrier_init();
  }
  if (warp == 1) tmem_alloc(&s.tmem_base, 512);
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = s.tmem_base;
  const uint32_t tmem_o = tmem + 2 * NT;

  if (warp == 0) {
    // ------------------------------------------------------------ TMA producer
    const int pages = kKeys / page;  // per tile: 1, 2 or 4
    const int32_t* bt = block_tables + (int64_t)b * max_blocks;
    const int nblk = (ctx + page - 1) / page;
    const int oob = (int)(num_blocks * page);  // a row past the cache reads as zeros
    if (lane == 0) mbar_arrive_expect_tx(&s.q_full, S::kQBytes);
    __syncwarp();
    if (lane < S::kChunks) tma_load_2d(s.q + lane * S::kQChunk, &q_map, &s.q_full, lane * 64, b * H + h0);
    int sent = 0;
    for (; sent < ntiles; ++sent) {
      const int st = sent % S::kStages;
      int y = oob;  // lane l < pages: first row of the tile's page l
      const int j = (tile0 + sent) * pages + lane;
      if (lane < pages && j < nblk) {
        const int blk = bt[j];
        if (blk >= 0 && blk < num_blocks) {
          y = blk * page;
        } else {
          atomicCAS(err, 0, 82);
        }
      }
      bool ok = !s.abort_flag;
      if (ok && sent >= S::kStages) ok = wait_or_abort(s, &s.kv_empty[st], (sent / S::kStages - 1) & 1, err, 84);
      if (!__all_sync(0xffffffffu, ok)) break;
      if (lane == 0) mbar_arrive_expect_tx(&s.kv_full[st], S::kTileBytes);
      __syncwarp();
      for (int i0 = 0; i0 < pages * S::kChunks; i0 += 32) {
        const int i = i0 + lane, pg = min(i / S::kChunks, pages - 1), c = i % S::kChunks;
        const int yy = __shfl_sync(0xffffffffu, y, pg);
        if (i < pages * S::kChunks)
          tma_load_2d(s.k[st] + c * S::kChunkBytes + pg * page * 128, &c_map, &s.kv_full[st], c * 64, yy);
      }
    }
    // the copies in flight end before the CTA does, on the way out of a time-out too
    if (lane == 0) {
      mbar_wait_sleep(&s.q_full, 0);
      for (int i = max(0, sent - S::kStages); i < sent; ++i)
        mbar_wait_sleep(&s.kv_full[i % S::kStages], (i / S::kStages) & 1);
    }
  } else if (warp == 1) {
    // -------------------------------------------------------------- MMA issuer
    if (lane == 0) {
      constexpr uint32_t idesc_s = idesc_bf16<64, NT>();
      constexpr uint32_t idesc_o = idesc_bf16<128, NT>() | kIdescAMn | kIdescBMn;
      const uint32_t q_addr = smem_u32(s.q), p_addr = smem_u32(s.p);
      auto issue_s = [&](int j) {  // the tile has landed
        tc_fence_after();
        const uint32_t k_addr = smem_u32(s.k[j % S::kStages]);
#pragma unroll
        for (int c = 0; c < S::kChunks; ++c)
#pragma unroll
          for (int kk = 0; kk < 4; ++kk)
            mma_bf16(tmem + (j & 1) * NT, smem_desc_sw128(k_addr + c * S::kChunkBytes + kk * 32),
                     smem_desc_sw128(q_addr + c * S::kQChunk + kk * 32), idesc_s, c + kk > 0);
        mma_commit(&s.s_full[j & 1]);
      };
      auto full = [&](int j) -> uint64_t* { return &s.kv_full[j % S::kStages]; };
      auto full_ph = [&](int j) -> uint32_t { return (j / S::kStages) & 1; };
      bool ok = wait_or_abort(s, &s.q_full, 0, err, 85) && wait_or_abort(s, full(0), 0, err, 85);
      if (ok) issue_s(0);
      for (int j = 0; ok && j < ntiles; ++j) {
        // the next tile's scores as soon as it has landed, this tile's second product as
        // soon as P is there, whichever comes first
        bool next = j + 1 >= ntiles, p_ready = false;
        const uint64_t t_start = globaltimer_ns();
        while (!p_ready) {
          if (!next && mbar_try_wait(full(j + 1), full_ph(j + 1)) &&
              (j + 1 < 2 || mbar_try_wait(&s.s_free[(j + 1) & 1], (((j + 1) >> 1) - 1) & 1))) {
            issue_s(j + 1);
            next = true;
          }
          p_ready = mbar_try_wait(&s.p_full, j & 1);
          if (!p_ready && (s.abort_flag || globaltimer_ns() - t_start > 2000000000ull)) {
            if (!s.abort_flag) atomicCAS(err, 0, 86);
            s.abort_flag = 1;
            ok = false;
            break;
          }
        }
        if (!ok) break;
        tc_fence_after();
        const uint32_t k_addr = smem_u32(s.k[j % S::kStages]);
#pragma unroll
        for (int m = 0; m < R / 128; ++m)
#pragma unroll
          for (int kk = 0; kk < kKeys / 16; ++kk)
            mma_bf16(tmem_o + m * NT,
                     smem_desc_mn_sw128(k_addr + 2 * m * S::kChunkBytes + kk * 2048, S::kChunkBytes, 1024),
                     smem_desc_mn_sw128(p_addr + kk * 2048, 1024, 1024), idesc_o, j > 0 || kk > 0);
        mma_commit(&s.pv_done);
        mma_commit(&s.kv_empty[j % S::kStages]);
        if (!next) {
          ok = wait_or_abort(s, full(j + 1), full_ph(j + 1), err, 85) &&
               (j + 1 < 2 || wait_or_abort(s, &s.s_free[(j + 1) & 1], (((j + 1) >> 1) - 1) & 1, err, 87));
          if (ok) issue_s(j + 1);
        }
      }
      // every MMA issued has finished before the tensor memory is freed
      mma_commit(&s.drained);
      mbar_wait_sleep(&s.drained, 0);
    }
  } else {
    // ------------------------------------------------------- softmax, epilogue
    const int quad = warp & 3;  // TMEM lane quadrant
    const int sw = warp - 2;
    constexpr int V = NT / 4;  // columns a thread holds
    const int row = quad * 16 + (lane >> 2);  // keys row and row + 8 of the tile
    const uint32_t lane_off = (uint32_t)(quad * 32) << 16;
    float m_ref[V], l[V];
#pragma unroll
    for (int n = 0; n < V; ++n) m_ref[n] = -INFINITY, l[n] = 0.f;
    for (int i = 0; i < ntiles; ++i) {
      wait_or_abort(s, &s.s_full[i & 1], (i >> 1) & 1, err, 88);
      __syncwarp();
      tc_fence_after();
      float v[NT / 8][4];
      tmem_ld_frag<NT / 8>(tmem + lane_off + (i & 1) * NT, v);
      tc_fence_before();
      mbar_arrive(&s.s_free[i & 1]);
      const int valid = ctx - (tile0 + i) * kKeys;  // keys of this tile
      const bool in0 = row < valid, in1 = row + 8 < valid;
      float mx[V];
#pragma unroll
      for (int n = 0; n < V; ++n) {
        float& a = v[n >> 1][n & 1];
        float& c = v[n >> 1][2 + (n & 1)];
        a = in0 ? a * scale_log2 : -INFINITY;
        c = in1 ? c * scale_log2 : -INFINITY;
        mx[n] = fmaxf(a, c);
      }
      const int first = reduce_columns<V>(mx, [](float x, float y) { return fmaxf(x, y); });
      constexpr int VF = V >= 8 ? V / 8 : 1;
#pragma unroll
      for (int n = 0; n < VF; ++n) s.red[i & 1][sw][frag_col(first + n)] = mx[n];
      soft_barrier();
      float mt[V];
      bool raise = false;
#pragma unroll
      for (int g = 0; g < V / 2; ++g) {
        const int c = g * 8 + (lane & 3) * 2;
        float2 x = *reinterpret_cast<const float2*>(&s.red[i & 1][0][c]);
#pragma unroll
        for (int w = 1; w < kSoft; ++w) {
          const float2 y = *reinterpret_cast<const float2*>(&s.red[i & 1][w][c]);
          x.x = fmaxf(x.x, y.x), x.y = fmaxf(x.y, y.y);
        }
        mt[2 * g] = x.x, mt[2 * g + 1] = x.y;
        raise |= x.x > m_ref[2 * g] + kRaise || x.y > m_ref[2 * g + 1] + kRaise;
      }
      // every warp sees every column, so all of them decide alike
      raise = __any_sync(0xffffffffu, raise);
      if (i > 0) wait_or_abort(s, &s.pv_done, (i - 1) & 1, err, 89);
      __syncwarp();
      if (raise) {
#pragma unroll
        for (int n = 0; n < V; ++n) {
          const float mn = fmaxf(m_ref[n], mt[n]);
          mt[n] = mn == -INFINITY ? 1.f : exp2f(m_ref[n] - mn);  // now the factor
          m_ref[n] = mn;
          l[n] *= mt[n];
        }
        if (i > 0) {
          tc_fence_after();
#pragma unroll
          for (int c = 0; c < NT; c += 16) {
            float f[16];
            columns16(mt, c, f);
#pragma unroll 1
            for (int m = 0; m < R / 128; ++m) {
              float o[16];
              uint32_t u[16];
              const uint32_t at = tmem_o + lane_off + m * NT + c;
              tmem_ld16(at, o);
#pragma unroll
              for (int n = 0; n < 16; ++n) u[n] = __float_as_uint(o[n] * f[n]);
              tmem_st16(at, u);
            }
          }
          tmem_wait_st();
        }
      }
#pragma unroll
      for (int g = 0; g < V / 2; ++g) {
        const float m0 = m_ref[2 * g] == -INFINITY ? 0.f : m_ref[2 * g];
        const float m1 = m_ref[2 * g + 1] == -INFINITY ? 0.f : m_ref[2 * g + 1];
        const float a0 = exp2f(v[g][0] - m0), a1 = exp2f(v[g][1] - m1);
        const float b0 = exp2f(v[g][2] - m0), b1 = exp2f(v[g][3] - m1);
        l[2 * g] += a0 + b0;
        l[2 * g + 1] += a1 + b1;
        uint8_t* dst = s.p + (lane & 3) * 4;
        *reinterpret_cast<uint32_t*>(dst + sw128_offset(row, g)) = pack_bf16(a0, a1);
        *reinterpret_cast<uint32_t*>(dst + sw128_offset(row + 8, g)) = pack_bf16(b0, b1);
      }
      if (valid < kKeys) {  // the last tile: rows past the context
        wait_or_abort(s, &s.kv_full[i % S::kStages], (i / S::kStages) & 1, err, 88);
        uint8_t* kt = s.k[i % S::kStages];
        const int t = threadIdx.x - 64, per_row = R / 8;  // 16-byte vectors of a row's latent
        for (int e = t; e < (kKeys - valid) * per_row; e += kSoft * 32) {
          const int r = valid + e / per_row, x = e % per_row;
          *reinterpret_cast<uint4*>(kt + (x >> 3) * S::kChunkBytes + r * 128 + (x & 7) * 16) = make_uint4(0, 0, 0, 0);
        }
      }
      fence_proxy_async_smem();
      tc_fence_before();
      mbar_arrive(&s.p_full);
    }
    wait_or_abort(s, &s.pv_done, (ntiles - 1) & 1, err, 89);
    __syncwarp();
    tc_fence_after();
    float (&red)[kSoft][NT] = s.red[ntiles & 1];  // the last tile's maxima are in the other one
    {
      float part[V];
#pragma unroll
      for (int n = 0; n < V; ++n) part[n] = l[n];
      const int first = reduce_columns<V>(part, [](float x, float y) { return x + y; });
      constexpr int VF = V >= 8 ? V / 8 : 1;
#pragma unroll
      for (int n = 0; n < VF; ++n) red[sw][frag_col(first + n)] = part[n];
    }
    soft_barrier();
#pragma unroll
    for (int n = 0; n < V; ++n) {
      const int c = frag_col(n);
      float sum = 0.f;
#pragma unroll
      for (int w = 0; w < kSoft; ++w) sum += red[w][c];
      l[n] = sum == 0.f ? 0.f : 1.f / sum;
      if (sw == 0 && lane < 4 && c < nheads)
        part_lse[part0 + (int64_t)c * nsplit] = sum == 0.f ? -INFINITY : m_ref[n] + log2f(sum);
    }
#pragma unroll
    for (int c = 0; c < NT; c += 16) {
      float f[16];
      columns16(l, c, f);
#pragma unroll 1
      for (int m = 0; m < R / 128; ++m) {
        float o[16];
        tmem_ld16(tmem_o + lane_off + m * NT + c, o);
        // a warp writes 32 consecutive dims of one head at a time
        float* dst = part_o + (part0 + (int64_t)c * nsplit) * R + m * 128 + quad * 32 + lane;
#pragma unroll
        for (int n = 0; n < 16; ++n)
          if (c + n < nheads) dst[(int64_t)n * nsplit * R] = o[n] * f[n];
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

// -------------------------------------------------------------- head products
//
// y[b, h, n] = sum_k x[b, h, k] w_h[k, n], small matrices per head: bound by the weights
// (64 KB + 64 KB a head at R = 512) until hundreds of rows share them, which mma.sync
// serves at the speed of the loads; a 128-row tcgen05 tile would be mostly padding.

__device__ __forceinline__ void cp16(void* dst, const void* src) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(smem_u32(dst)), "l"(src) : "memory");
}
__device__ __forceinline__ void cp_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int N>
__device__ __forceinline__ void cp_wait() { asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory"); }

// qa[b, h, :R] = q[b, h, :128] . w[h, :128, :], qa[b, h, R:] = q[b, h, 128:].
// One CTA per (64 columns, head, MROWS rows); qa is bf16, the tensor cores' operand type.
template <int R, int MROWS>
__global__ void __launch_bounds__(128) latent_absorb_kernel(const bf16* __restrict__ q, int64_t q_stride,
                                                            const bf16* __restrict__ w, bf16* __restrict__ qa, int B,
                                                            int H) {
  griddep_entry();
  constexpr int kPitchW = 64 + 8, kPitchX = kNope + 8;  // 16 bytes of padding: conflict-free ldmatrix
  __shared__ __align__(16) bf16 ws[kNope * kPitchW];
  __shared__ __align__(16) bf16 xs[MROWS * kPitchX];
  const int n0 = blockIdx.x * 64, h = blockIdx.y, b0 = blockIdx.z * MROWS;
  const int t = threadIdx.x, warp = t >> 5, lane = t & 31;
  const bf16* wk = w + (int64_t)h * (kNope + kVal) * R + n0;
  for (int i = t; i < kNope * 8; i += 128) cp16(ws + (i >> 3) * kPitchW + (i & 7) * 8, wk + (int64_t)(i >> 3) * R + (i & 7) * 8);
  for (int i = t; i < MROWS * 16; i += 128) {
    const int r = i >> 4;
    if (b0 + r < B)
      cp16(xs + r * kPitchX + (i & 15) * 8, q + (int64_t)(b0 + r) * q_stride + (int64_t)h * (kNope + kRot) + (i & 15) * 8);
  }
  cp_commit();
  if (blockIdx.x == 0) {  // the rotary part
    for (int i = t; i < MROWS * 8; i += 128) {
      const int b = b0 + (i >> 3);
      if (b < B)
        *reinterpret_cast<uint4*>(qa + ((int64_t)b * H + h) * (R + kRot) + R + (i & 7) * 8) =
            *reinterpret_cast<const uint4*>(q + (int64_t)b * q_stride + (int64_t)h * (kNope + kRot) + kNope + (i & 7) * 8);
    }
  }
  cp_wait<0>();
  __syncthreads();
  // MROWS = 64: a warp per 16 rows, 64 columns; 16: a warp per 16 columns
  constexpr int NP = MROWS == 64 ? 4 : 1;  // 16-column pairs of n-tiles a warp
  const int r0 = MROWS == 64 ? warp * 16 : 0, c0 = MROWS == 64 ? 0 : warp * 16;
  float acc[NP][2][4] = {};
#pragma unroll
  for (int ks = 0; ks < kNope / 16; ++ks) {
    uint32_t a[4];
    ldmatrix_x4(a, smem_u32(xs + (r0 + (lane & 15)) * kPitchX + ks * 16 + (lane >> 4) * 8));
#pragma unroll
    for (int p = 0; p < NP; ++p) {
      uint32_t bb[4];
      ldmatrix_x4_trans(bb, smem_u32(ws + (ks * 16 + (lane & 15)) * kPitchW + c0 + p * 16 + (lane >> 4) * 8));
      mma_bf16_16816(acc[p][0], a, {bb[0], bb[1]});
      mma_bf16_16816(acc[p][1], a, {bb[2], bb[3]});
    }
  }
#pragma unroll
  for (int p = 0; p < NP; ++p)
#pragma unroll
    for (int nt = 0; nt < 2; ++nt)
#pragma unroll
      for (int e = 0; e < 2; ++e) {
        const int b = b0 + r0 + (lane >> 2) + e * 8;
        if (b < B)
          *reinterpret_cast<uint32_t*>(qa + ((int64_t)b * H + h) * (R + kRot) + n0 + c0 + p * 16 + nt * 8 + (lane & 3) * 2) =
              pack_bf16(acc[p][nt][2 * e], acc[p][nt][2 * e + 1]);
      }
}

// Joins the splits and applies V_h: out[b, h, n] = sum_r o[b, h, r] w[h, 128 + n, r] with
//   o = sum_s 2^(lse_s - M) o_s / sum_s 2^(lse_s - M).
// o enters the product as hi + lo, two bf16 whose sum keeps 16 bits of it: the
// second MMA costs nothing beside the loads, and one rounding less reaches the output.
// One CTA per (NCOLS columns, head, MROWS rows), K in chunks of 128.
template <int R, int MROWS, int NCOLS>
__global__ void __launch_bounds__(MROWS == 64 ? 256 : 128)
    latent_out_kernel(const float* __restrict__ part_o, const float* __restrict__ part_lse,
                      const bf16* __restrict__ w, bf16* __restrict__ out, int64_t out_stride, int B, int H,
                      int nsplit) {
  griddep_entry();
  constexpr int kThr = MROWS == 64 ? 256 : 128;
  constexpr int kPitch = 128 + 8;
  constexpr int kSteps = R / 128;
  extern __shared__ __align__(16) uint8_t raw[];
  bf16* ws = reinterpret_cast<bf16*>(raw);             // [2][NCOLS][kPitch]
  bf16* xh = ws + 2 * NCOLS * kPitch;                  // [MROWS][kPitch]
  bf16* xl = xh + MROWS * kPitch;
  float* wt = reinterpret_cast<float*>(xl + MROWS * kPitch);  // [MROWS][nsplit] split weights
  const int n0 = blockIdx.x * NCOLS, h = blockIdx.y, b0 = blockIdx.z * MROWS;
  const int t = threadIdx.x, warp = t >> 5, lane = t & 31;
  const bf16* wv = w + ((int64_t)h * (kNope + kVal) + kNope + n0) * R;
  auto load_w = [&](int c) {
    for (int i = t; i < NCOLS * 16; i += kThr)
      cp16(ws + ((c & 1) * NCOLS + (i >> 4)) * kPitch + (i & 15) * 8, wv + (int64_t)(i >> 4) * R + c * 128 + (i & 15) * 8);
    cp_commit();
  };
  load_w(0);
  for (int r = warp; r < MROWS; r += kThr / 32) {  // a warp per row
    const int b = b0 + r;
    const float* lse = part_lse + ((int64_t)min(b, B - 1) * H + h) * nsplit;
    const float a0 = lane < nsplit ? lse[lane] : -INFINITY, a1 = lane + 32 < nsplit ? lse[lane + 32] : -INFINITY;
    const float M = warp_max(fmaxf(a0, a1));
    // no split has a key: weights 0; a NaN in any split reaches the row
    const float e0 = M == -INFINITY && a0 == a0 ? 0.f : exp2f(a0 - M), e1 = M == -INFINITY && a1 == a1 ? 0.f : exp2f(a1 - M);
    const float L = warp_sum(e0 + e1);
    const float inv = L == 0.f ? 0.f : 1.f / L;
    if (lane < nsplit) wt[r * nsplit + lane] = e0 * inv;
    if (lane + 32 < nsplit) wt[r * nsplit + lane + 32] = e1 * inv;
  }
  constexpr int WN = MROWS == 64 ? NCOLS / 2 : NCOLS / 4;  // columns a warp
  constexpr int NT8 = WN / 8;
  const int r0 = MROWS == 64 ? (warp & 3) * 16 : 0, c0 = (MROWS == 64 ? warp >> 2 : warp) * WN;
  float acc[NT8][4] = {};
  __syncthreads();
  for (int c = 0; c < kSteps; ++c) {
    if (c + 1 < kSteps) load_w(c + 1);
    for (int i = t; i < MROWS * 32; i += kThr) {
      const int r = i >> 5, k = (i & 31) * 4;
      float4 x = make_float4(0.f, 0.f, 0.f, 0.f);
      if (b0 + r < B) {
        const float* src = part_o + (((int64_t)(b0 + r) * H + h) * nsplit) * R + c * 128 + k;
        for (int s = 0; s < nsplit; ++s) {
          const float f = wt[r * nsplit + s];
          if (f != 0.f) {  // a split without keys wrote no partial
            const float4 y = *reinterpret_cast<const float4*>(src + (int64_t)s * R);
            x.x += f * y.x, x.y += f * y.y, x.z += f * y.z, x.w += f * y.w;
          }
        }
      }
      const uint32_t h0 = pack_bf16(x.x, x.y), h1 = pack_bf16(x.z, x.w);
      const float2 f0 = __bfloat1622float2(*reinterpret_cast<const __nv_bfloat162*>(&h0));
      const float2 f1 = __bfloat1622float2(*reinterpret_cast<const __nv_bfloat162*>(&h1));
      *reinterpret_cast<uint2*>(xh + r * kPitch + k) = make_uint2(h0, h1);
      *reinterpret_cast<uint2*>(xl + r * kPitch + k) =
          make_uint2(pack_bf16(x.x - f0.x, x.y - f0.y), pack_bf16(x.z - f1.x, x.w - f1.y));
    }
    if (c + 1 < kSteps) {
      cp_wait<1>();
    } else {
      cp_wait<0>();
    }
    __syncthreads();
    const bf16* wc = ws + (c & 1) * NCOLS * kPitch;
#pragma unroll
    for (int ks = 0; ks < 8; ++ks) {
      uint32_t ah[4], al[4];
      const int at = (r0 + (lane & 15)) * kPitch + ks * 16 + (lane >> 4) * 8;
      ldmatrix_x4(ah, smem_u32(xh + at));
      ldmatrix_x4(al, smem_u32(xl + at));
#pragma unroll
      for (int n = 0; n < NT8; ++n) {
        uint32_t bb[2];
        // rows n, 16 bytes at k and k + 8
        asm volatile("ldmatrix.sync.aligned.m8n8.x2.shared.b16 {%0,%1}, [%2];"
                     : "=r"(bb[0]), "=r"(bb[1])
                     : "r"(smem_u32(wc + (c0 + n * 8 + (lane & 7)) * kPitch + ks * 16 + ((lane >> 3) & 1) * 8)));
        mma_bf16_16816(acc[n], ah, bb);
        mma_bf16_16816(acc[n], al, bb);
      }
    }
    __syncthreads();  // the x tile is rewritten next
  }
#pragma unroll
  for (int n = 0; n < NT8; ++n)
#pragma unroll
    for (int e = 0; e < 2; ++e) {
      const int b = b0 + r0 + (lane >> 2) + e * 8;
      if (b < B)
        *reinterpret_cast<uint32_t*>(out + (int64_t)b * out_stride + (int64_t)h * kVal + n0 + c0 + n * 8 + (lane & 3) * 2) =
            pack_bf16(acc[n][2 * e], acc[n][2 * e + 1]);
    }
}

template <int R, int MROWS, int NCOLS>
void run_out(const LatentDecode& a, const float* part_o, const float* part_lse, cudaStream_t st) {
  auto kern = latent_out_kernel<R, MROWS, NCOLS>;
  const size_t fixed = (size_t)(2 * NCOLS + 2 * MROWS) * 136 * 2;
  static std::atomic<uint64_t> attr_devs{0};
  ensure_smem_attr(attr_devs, kern, fixed + (size_t)MROWS * kMaxSplits * 4);
  launch_k(kern, dim3(kVal / NCOLS, a.H, (a.B + MROWS - 1) / MROWS), MROWS == 64 ? 256 : 128,
           fixed + (size_t)MROWS * a.nsplit * 4, st, part_o, part_lse, a.w, a.out, a.out_stride, a.B, a.H, a.nsplit);
  KAPSL_LAUNCH_CHECK();
}

template <int R, int NT>
void run_attn(const LatentDecode& a, const bf16* qa, float* part_o, float* part_lse, int head_tiles, cudaStream_t st) {
  using S = Shape<R, NT>;
  auto kern = latent_attn_kernel<R, NT>;
  const size_t smem = sizeof(DecodeSmem<R, NT>);
  static_assert(sizeof(DecodeSmem<R, NT>) <= 232448, "shared memory of one CTA");
  static std::atomic<uint64_t> attr_devs{0};
  ensure_smem_attr(attr_devs, kern, smem);
  const CUtensorMap tq = make_tmap_2d_bf16(qa, (uint64_t)a.B * a.H, S::W, S::W, NT, 64, true);
  const CUtensorMap tc = make_tmap_2d_bf16(a.cache, (uint64_t)a.num_blocks * a.page, S::W, S::W, a.page, 64, true);
  launch_k(kern, dim3(a.nsplit, head_tiles, a.B), kThreads, smem, st, tq, tc, a.num_blocks, a.page, a.block_tables,
           a.max_blocks, a.ctx_lens, part_o, part_lse, a.H, (a.H + head_tiles - 1) / head_tiles, a.nsplit,
           a.scale * kLog2e, a.err);
  KAPSL_LAUNCH_CHECK();
}

int head_tiles_of(int H) { return (H + 63) / 64; }

template <int R>
void run(const LatentDecode& a, cudaStream_t st) {
  bf16* qa = static_cast<bf16*>(a.workspace);
  float* part_o = reinterpret_cast<float*>(qa + (int64_t)a.B * a.H * (R + kRot));
  float* part_lse = part_o + (int64_t)a.B * a.H * a.nsplit * R;
  if (a.B <= 16) {
    launch_k(latent_absorb_kernel<R, 16>, dim3(R / 64, a.H, 1), 128, 0, st, a.q, a.q_stride, a.w, qa, a.B, a.H);
  } else {
    launch_k(latent_absorb_kernel<R, 64>, dim3(R / 64, a.H, (a.B + 63) / 64), 128, 0, st, a.q, a.q_stride, a.w, qa,
             a.B, a.H);
  }
  KAPSL_LAUNCH_CHECK();
  const int ht = head_tiles_of(a.H), hpc = (a.H + ht - 1) / ht;
  if (hpc <= 16) {
    run_attn<R, 16>(a, qa, part_o, part_lse, ht, st);
  } else if (hpc <= 32) {
    run_attn<R, 32>(a, qa, part_o, part_lse, ht, st);
  } else {
    run_attn<R, 64>(a, qa, part_o, part_lse, ht, st);
  }
  if (a.B <= 16) {
    run_out<R, 16, 32>(a, part_o, part_lse, st);
  } else {
    run_out<R, 64, 128>(a, part_o, part_lse, st);
  }
  note_launch(3);
}

}  // namespace

int latent_decode_num_splits(int B, int H, int R, int max_ctx, int num_sms) {
  const int ctas = std::max(1, B * head_tiles_of(std::max(1, H)));
  int s = (4 * num_sms + ctas - 1) / ctas;
  s = std::min(s, std::max(1, (max_ctx + 511) / 512));
  return std::max(1, std::min(s, kMaxSplits));
}

size_t latent_decode_workspace_bytes(int B, int H, int R, int nsplit) {
  const size_t bh = (size_t)B * H;
  return bh * (R + kRot) * 2 + bh * nsplit * ((size_t)R + 1) * 4;
}

void launch_latent_decode(const LatentDecode& a, cudaStream_t st) {
  if (a.B == 0) return;
  if (a.R == 512) {
    run<512>(a, st);
  } else if (a.R == 256) {
    run<256>(a, st);
  } else {
    throw std::runtime_error("latent decode: the latent must have 256 or 512 values");
  }
}

}  // namespace kapsl
