// Absorbed latent attention for single tokens over a paged latent cache.
//
// A cache row is [c (R) | k_r (64)], shared by every head.  Head h has the key
// expansion K_h = w[h, :128] and the value expansion V_h = w[h, 128:], both [128, R].
// With the key expansion moved to the query's side,
//   qa_h = [K_h^T q_h[:128] | q_h[128:]],   s_j = scale * qa_h . row_j,
//   o_h = sum_j softmax(s)_j c_j,           out_h = V_h o_h,
// so the cache is read once for all heads and nothing is expanded per token.
//
// Four launches: absorb (qa, and the schedule), attention over pieces of the contexts (fp32
// partials of o), the join of the pieces, and the product with V_h.
//
// Roundings: qa and P become bf16 because the cache does not change its type and both
// operands of an MMA share theirs; halves of more bits would cost a second pass over every key
// tile's products, which bound the kernel above some 32 heads.  With few heads it waits for DRAM
// and such a pass might hide; one precision is kept, so that a model's accuracy does not depend on
// how its heads are sharded.  The joined o keeps 16 bits in two bf16.  Each rounding is 2^-8 of
// a value at most and 0.0017 in the mean square: an output is 0.0024-0.0028 from 64-bit
// arithmetic, where one rounded once at the end is 0.0017.
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

// -------------------------------------------------------------------- schedule
//
// The tiles (64 keys) of all sequences form one line, and each CTA of a head tile takes an
// equal stretch of it, whatever the lengths: stretches cross sequence ends, sequences
// cross stretches.  A piece is the part of sequence b that CTA c holds; b + c grows along
// the line, so it numbers the pieces' partial results.  Head tiles of the same
// sequences run side by side (cache tiles are read from DRAM once).
//
// table: [0] tiles a CTA takes, [1 + b] first tile of sequence b, [1 + B] all tiles.
// `quota` is at least a 32nd of the longest sequence: no row joins more than kMaxPieces.
constexpr int kKeys = 64;
constexpr int kMaxPieces = 33;

__host__ __device__ constexpr int table_ints(int B) { return (B + 2 + 31) / 32 * 32; }

__device__ __forceinline__ int seq_tiles(const int32_t* ctx_lens, int b, int limit, int keys) {
  return (max(0, min(ctx_lens[b], limit)) + keys - 1) / keys;
}

// One block writes the table (`limit`: tokens the block tables hold).
__device__ void write_schedule(const int32_t* ctx_lens, int B, int limit, int keys, int ctas, int32_t* table) {
  __shared__ int sums[33], longest;
  const int t = threadIdx.x, lane = t & 31, warp = t >> 5, nw = blockDim.x >> 5;
  if (t == 0) longest = 0;
  int base = 0;
  for (int b0 = 0; b0 < B; b0 += blockDim.x) {
    const int n = b0 + t < B ? seq_tiles(ctx_lens, b0 + t, limit, keys) : 0;
    int x = n;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const int y = __shfl_up_sync(0xffffffffu, x, o);
      if (lane >= o) x += y;
    }
    __syncthreads();
    if (lane == 31) sums[warp] = x;
    atomicMax(&longest, n);
    __syncthreads();
    int before = base;
    for (int w = 0; w < nw; ++w) {
      if (w < warp) before += sums[w];
      base += sums[w];
    }
    if (b0 + t < B) table[1 + b0 + t] = before + x - n;
  }
  __syncthreads();
  if (t == 0) {
    table[1 + B] = base;
    table[0] = max(1, max((base + ctas - 1) / ctas, (longest + 31) / 32));
  }
}

// ------------------------------------------------------------------ attention
//
// A CTA works on up to 64 heads.  The products are transposed so that the heads are the
// MMA's N, which may be 16, 32 or 64 without wasted rows:
//   S^T [64 keys, heads] = K . qa^T    (M = 64, K tile K-major)
//   O^T [R dims, heads] += c^T . P^T   (M = 128 x R / 128; the same K tile read MN-major)
// so a key tile is loaded once and serves both products, and O^T of 64 heads takes 256
// of the 512 TMEM columns, which leaves room for two S^T tiles.
//
// Tiles are loaded by TMA in groups of 128 latent dims (the rotary dims with the first),
// one producer warp and one ring of barriers a group: the scores of a group start when it
// lands, its slot is free again when the second product has read it.  One warp issues the
// MMAs, four do the softmax.
//
// Single-thread roles are entered by elect.sync.  Measured per SM: MMAs of M = 64, N = 16-64
// issued from a `lane == 0` branch took 44 cycles each, elected 23-32; 2 KB boxes (16-token
// pages) issued by nine lanes of one warp arrived at 17 B/clk, by one elected thread at 31, by
// four warps' elected threads at 90 (8 KB boxes: 80).
//
// Softmax: scores (times log2 e) are compared with the running maximum; only when one
// exceeds it by 8 (a vote over the four warps) is the maximum raised - column maxima by
// register and shared-memory exchange - and O^T rescaled in TMEM.  p <= 256 loses nothing in bf16 or
// fp32, and the final division uses the same maximum.  The scaled scores are rounded before the
// maximum, one of them, is taken off: in one rounding scale * s - m would be up to half of m's
// last place at the maximum, and 2^ of that infinite from 2^31 on.  P is rounded to bf16, the
// operand type of the second product; the row sums are of the fp32 values.  Keys past the context
// have p = 0 and their cache rows are cleared in shared memory, since 0 * NaN of a
// stale row would count.
constexpr int kSoft = 4;  // softmax warps
template <int R>
constexpr int kAttnThreads = (R / 128 + 1 + kSoft) * 32;
constexpr float kRaise = 8.f;
constexpr float kNoMax = -1e30f;

template <int R, int NT>
struct Shape {
  static constexpr int W = R + kRot;
  static constexpr int kChunks = W / 64;
  static constexpr int kGroups = R / 128;
  static constexpr uint32_t kChunkBytes = kKeys * 128;  // 64 keys x 64 dims
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
  float red[kSoft][NT];      // per warp column maxima, or sums
  float mcol[NT], fac[NT];   // the columns' running maxima; factors on O^T
  uint64_t q_full, q_empty, kv_full[S::kStages][S::kGroups], kv_empty[S::kStages][S::kGroups], s_full[2], s_free[2],
      p_full, pv_done, drained;
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

__device__ __forceinline__ float ex2(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}

__device__ __forceinline__ void soft_barrier() { asm volatile("bar.sync 1, %0;" ::"n"(kSoft * 32) : "memory"); }
__device__ __forceinline__ bool soft_any(bool v) {  // any thread of the softmax warps
  uint32_t r;
  asm volatile(
      "{\n\t.reg .pred p, q;\n\tsetp.ne.b32 q, %1, 0;\n\tbar.red.or.pred p, 1, %2, q;\n\tselp.u32 %0, 1, 0, p;\n\t}"
      : "=r"(r)
      : "r"((uint32_t)v), "n"(kSoft * 32)
      : "memory");
  return r != 0;
}

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

// A CTA's stretch of the line, piece by piece.  The next sequence's place and length are loaded
// while the present one is worked on.
struct Pieces {
  const int32_t *start, *ctx_lens;  // start = table + 1
  int B, limit, at, end, b, s0, s1, s2, len, len1;
  __device__ Pieces(const int32_t* table, const int32_t* lens, int B_, int limit_, int c)
      : start(table + 1), ctx_lens(lens), B(B_), limit(limit_) {  // called by whole warps
    const int quota = table[0], all = table[1 + B], lane = threadIdx.x & 31;
    at = (int)min((int64_t)c * quota, (int64_t)all);
    end = min(at + quota, all);
    b = 0;  // last sequence that starts at or before `at`, 32 candidates at a time
    for (int n = B; n > 1;) {
      const int step = (n + 31) / 32, i = lane * step;
      const bool le = i < n && start[b + i] <= at;
      const int k = __popc(__ballot_sync(0xffffffffu, le)) - 1;
      b += k * step;
      n = min(step, n - k * step);
    }
    s0 = start[b];
    s1 = start[b + 1];
    len = ctx_lens[b];
    ahead();
  }
  __device__ void ahead() {
    s2 = start[min(b + 2, B)];
    len1 = ctx_lens[min(b + 1, B - 1)];
  }
  __device__ bool more() const { return at < end; }
  __device__ int first() const { return at - s0; }  // tile within the sequence
  __device__ int tiles() const { return min(end, s1) - at; }
  __device__ int keys() const { return min(len, limit); }
  __device__ void next() {
    at = min(end, s1);
    while (at < end && s1 <= at) {  // sequences without keys take no tiles
      ++b;
      s0 = s1;
      s1 = s2;
      len = len1;
      ahead();
    }
  }
};

template <int R, int NT>
__global__ void __launch_bounds__(kAttnThreads<R>, 1)
    latent_attn_kernel(const __grid_constant__ CUtensorMap q_map, const __grid_constant__ CUtensorMap c_map,
                       int64_t num_blocks, int page, const int32_t* block_tables, int max_blocks,
                       const int32_t* table_rows, int num_tables,
                       const int32_t* ctx_lens, const int32_t* table,
                       float* part_o, float2* part_ml, int B, int H, int heads_per_cta,
                       int head_tiles, float scale_log2, int* err) {
  griddep_launch();
  using S = Shape<R, NT>;
  constexpr int kMma = S::kGroups;  // warps: producers, MMA issuer, softmax
  extern __shared__ __align__(1024) uint8_t smem_raw[];
  DecodeSmem<R, NT>& s = *reinterpret_cast<DecodeSmem<R, NT>*>(smem_raw);
  const int warp = __shfl_sync(0xffffffffu, threadIdx.x / 32, 0), lane = threadIdx.x % 32;
  const int ht = blockIdx.x % head_tiles, c = blockIdx.x / head_tiles;
  const int ctas = gridDim.x / head_tiles;
  const int h0 = ht * heads_per_cta, nheads = min(heads_per_cta, H - h0);
  if (smem_u32(smem_raw) & 1023) {  // the swizzled tiles need it
    if (threadIdx.x == 0) atomicCAS(err, 0, 83);
    return;
  }

  if (threadIdx.x == 0) {
    s.abort_flag = 0;
    mbar_init(&s.q_full, 1);
    mbar_init(&s.q_empty, 1);
    for (int i = 0; i < S::kStages; ++i)
      for (int g = 0; g < S::kGroups; ++g) {
        mbar_init(&s.kv_full[i][g], 1);
        mbar_init(&s.kv_empty[i][g], 1);
      }
    for (int i = 0; i < 2; ++i) {
      mbar_init(&s.s_full[i], 1);
      mbar_init(&s.s_free[i], kSoft);
    }
    mbar_init(&s.p_full, kSoft);
    mbar_init(&s.pv_done, 1);
    mbar_init(&s.drained, 1);
    fence_barrier_init();
  }
  griddep_wait();  // before the allocation: a CTA of the grid waited for may still need its own
  if (warp == kMma) tmem_alloc(&s.tmem_base, 512);
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = __shfl_sync(0xffffffffu, s.tmem_base, 0);
  const uint32_t tmem_o = tmem + 2 * NT;
  Pieces pc(table, ctx_lens, B, max_blocks * page, c);  // without pieces, every role falls through its loop

  if (warp < S::kGroups) {
    // ------------------------------------------- TMA producer of dims [128 g, 128 g + 128)
    const int g = warp;
    const int pages = kKeys / page;  // per tile: 1, 2 or 4
    const int oob = (int)(num_blocks * page);  // a row past the cache reads as zeros
    int sent = 0, nq = 0;
    bool ok = true;
    // lane l < pages: first row of page l of a tile
    auto page_row = [&](int trow, int tile) {
      const int j = tile * pages + lane;
      if (lane >= pages || j >= (pc.keys() + page - 1) / page) return oob;
      const int blk = trow >= 0 && trow < num_tables ? block_tables[(int64_t)trow * max_blocks + j] : -1;
      if (blk >= 0 && blk < num_blocks) return blk * page;
      atomicCAS(err, 0, 82);
      return oob;
    };
    for (; ok && pc.more(); pc.next()) {
      const int b = pc.b, t0 = pc.first(), n = pc.tiles();
      const int trow = table_rows != nullptr ? table_rows[b] : b;
      int y = page_row(trow, t0), y1 = n > 1 ? page_row(trow, t0 + 1) : oob;
      if (g == 0) {
        if (nq > 0) ok = wait_or_abort(s, &s.q_empty, (nq - 1) & 1, err, 84);
        if (!__all_sync(0xffffffffu, ok)) break;
        if (elect_one()) {
          mbar_arrive_expect_tx(&s.q_full, S::kQBytes);
#pragma unroll
          for (int ch = 0; ch < S::kChunks; ++ch)
            tma_load_2d(s.q + ch * S::kQChunk, &q_map, &s.q_full, ch * 64, b * H + h0);
        }
        ++nq;
      }
      for (int i = 0; i < n; ++i, ++sent) {
        const int st = sent % S::kStages;
        const int y2 = i + 2 < n ? page_row(trow, t0 + i + 2) : oob;
        int yy[4], zz[4];
#pragma unroll
        for (int pg = 0; pg < 4; ++pg) {
          yy[pg] = __shfl_sync(0xffffffffu, y, pg);
          zz[pg] = __shfl_sync(0xffffffffu, y1, pg);
        }
        if (elect_one()) {  // the next tile comes into L2 while its slot is still in use
#pragma unroll
          for (int pg = 0; pg < 4; ++pg) {
            if (pg < pages && zz[pg] < oob) {
              tma_prefetch_2d(&c_map, 128 * g, zz[pg]);
              tma_prefetch_2d(&c_map, 128 * g + 64, zz[pg]);
              if (g == 0) tma_prefetch_2d(&c_map, R, zz[pg]);
            }
          }
        }
        __syncwarp();
        if (sent >= S::kStages) ok = wait_or_abort(s, &s.kv_empty[st][g], (sent / S::kStages - 1) & 1, err, 84);
        if (!__all_sync(0xffffffffu, ok)) {
          ok = false;
          break;
        }
        if (elect_one()) {
          uint64_t* bar = &s.kv_full[st][g];
          mbar_arrive_expect_tx(bar, (g == 0 ? 3 : 2) * S::kChunkBytes);
#pragma unroll
          for (int pg = 0; pg < 4; ++pg) {
            if (pg < pages) {
              uint8_t* dst = s.k[st] + pg * page * 128;
              tma_load_2d(dst + 2 * g * S::kChunkBytes, &c_map, bar, 128 * g, yy[pg]);
              tma_load_2d(dst + (2 * g + 1) * S::kChunkBytes, &c_map, bar, 128 * g + 64, yy[pg]);
              if (g == 0) tma_load_2d(dst + (S::kChunks - 1) * S::kChunkBytes, &c_map, bar, R, yy[pg]);
            }
          }
        }
        __syncwarp();
        y = y1;
        y1 = y2;
      }
    }
    // the copies in flight end before the CTA does, on the way out of a time-out too
    if (lane == 0) {
      if (nq > 0) mbar_wait_sleep(&s.q_full, (nq - 1) & 1);
      for (int i = max(0, sent - S::kStages); i < sent; ++i)
        mbar_wait_sleep(&s.kv_full[i % S::kStages][g], (i / S::kStages) & 1);
    }
  } else if (warp == kMma) {
    // -------------------------------------------------------------- MMA issuer
    if (elect_one()) {
      constexpr uint32_t idesc_s = idesc_bf16<64, NT>();
      constexpr uint32_t idesc_o = idesc_bf16<128, NT>() | kIdescAMn | kIdescBMn;
      // Descriptors differ in the 14-bit address field only (16-byte units): one 64-bit base per
      // operand and constant steps, so that an MMA costs two additions.
      constexpr uint64_t kChunkStep = S::kChunkBytes >> 4, kTileStep = S::kTileBytes >> 4, kQStep = S::kQChunk >> 4;
      const uint64_t k_desc = smem_desc_sw128(smem_u32(s.k[0])), q_desc = smem_desc_sw128(smem_u32(s.q));
      const uint64_t v_desc = smem_desc_mn_sw128(smem_u32(s.k[0]), S::kChunkBytes, 1024);
      const uint64_t p_desc = smem_desc_mn_sw128(smem_u32(s.p), 1024, 1024);
      // two cursors over the same tiles: scores (sc) and second products (pv)
      Pieces sp = pc;
      int sc = 0, grp = 0, left_s = sp.more() ? sp.tiles() : 0, nq = 0;
      bool s_open = true, q_open = false;
      const int total = pc.end - pc.at;
      int left_p = left_s;
      bool first_p = true;
      uint64_t t_last = 0;
      uint32_t idle = 0;
      for (int pv = 0; pv < total;) {
        bool moved = false;
        // the second product first: it frees the slots that the next loads wait for
        if (pv < sc && mbar_test_wait(&s.p_full, pv & 1)) {
          tc_fence_after();
          const int st = pv % S::kStages;
          const uint64_t v0 = v_desc + st * kTileStep;
#pragma unroll
          for (int m = 0; m < S::kGroups; ++m) {
#pragma unroll
            for (int kk = 0; kk < kKeys / 16; ++kk)
              mma_bf16(tmem_o + m * NT, v0 + 2 * m * kChunkStep + kk * 128, p_desc + kk * 128, idesc_o,
                       !(first_p && kk == 0));
            mma_commit(&s.kv_empty[st][m]);
          }
          mma_commit(&s.pv_done);
          first_p = false;
          ++pv;
          if (--left_p == 0) {
            pc.next();
            left_p = pc.more() ? pc.tiles() : 0;
            first_p = true;
          }
          moved = true;
        }
        if (sc < total && sc < pv + 2) {  // two score tiles ahead, only the second product can go on
          if (!q_open) q_open = mbar_test_wait(&s.q_full, nq & 1);
          if (!s_open) s_open = mbar_test_wait(&s.s_free[sc & 1], ((sc >> 1) - 1) & 1);
          const int st = sc % S::kStages;
          if (q_open && s_open && mbar_test_wait(&s.kv_full[st][grp], (sc / S::kStages) & 1)) {
            tc_fence_after();
            const uint64_t k0 = k_desc + st * kTileStep, kg = k0 + 2 * grp * kChunkStep, qg = q_desc + 2 * grp * kQStep;
            const uint32_t d = tmem + (sc & 1) * NT;
            const uint32_t fresh = grp == 0;
#pragma unroll
            for (int ch = 0; ch < 2; ++ch)
#pragma unroll
              for (int kk = 0; kk < 4; ++kk)
                mma_bf16(d, kg + ch * kChunkStep + kk * 2, qg + ch * kQStep + kk * 2, idesc_s, ch + kk > 0 || !fresh);
            if (grp == 0)
#pragma unroll
              for (int kk = 0; kk < 4; ++kk)
                mma_bf16(d, k0 + (S::kChunks - 1) * kChunkStep + kk * 2, q_desc + (S::kChunks - 1) * kQStep + kk * 2,
                         idesc_s, 1);
            if (++grp == S::kGroups) {
              mma_commit(&s.s_full[sc & 1]);
              grp = 0;
              ++sc;
              s_open = sc < 2;
              if (--left_s == 0) {  // the piece's last scores: its queries are free
                mma_commit(&s.q_empty);
                ++nq;
                q_open = false;
                sp.next();
                left_s = sp.more() ? sp.tiles() : 0;
              }
            }
            moved = true;
          }
        }
        if (moved) {
          idle = 0;
        } else if ((++idle & 1023) == 0) {  // the clock is read rarely: it is slow
          const uint64_t now = globaltimer_ns();
          if (idle == 1024) t_last = now;
          if (s.abort_flag || now - t_last > 2000000000ull) {
            if (!s.abort_flag) atomicCAS(err, 0, 86);
            s.abort_flag = 1;
            break;
          }
        }
      }
      // every MMA issued has finished before the tensor memory is freed
      mma_commit(&s.drained);
      mbar_wait_sleep(&s.drained, 0);
    }
  } else {
    // ------------------------------------------------------- softmax, epilogue
    const int quad = warp & 3;  // TMEM lane quadrant
    const int sw = warp - kMma - 1, tid = sw * 32 + lane;
    constexpr int V = NT / 4;  // columns a thread holds
    constexpr int VF = V >= 8 ? V / 8 : 1;
    const int row = quad * 16 + (lane >> 2);  // keys row and row + 8 of the tile
    const uint32_t lane_off = (uint32_t)(quad * 32) << 16;
    int tile = 0;  // of the CTA
    for (; pc.more(); pc.next()) {
      const int b = pc.b, n_tiles = pc.tiles();
      const int left = pc.keys() - pc.first() * kKeys;  // keys from the piece's first on
      float m_ref[V], l[V];
#pragma unroll
      for (int n = 0; n < V; ++n) m_ref[n] = 0.f, l[n] = 0.f;
      for (int i = 0; i < n_tiles; ++i, ++tile) {
        wait_or_abort(s, &s.s_full[tile & 1], (tile >> 1) & 1, err, 88);
        __syncwarp();
        tc_fence_after();
        float v[NT / 8][4];
        tmem_ld_frag<NT / 8>(tmem + lane_off + (tile & 1) * NT, v);
        tc_fence_before();
        __syncwarp();
        if (lane == 0) mbar_arrive(&s.s_free[tile & 1]);  // one arrival a warp: 128 on one word serialise
        const int valid = left - i * kKeys;  // keys of this tile
        const bool in0 = row < valid, in1 = row + 8 < valid;
        float x[NT / 8][4], top = -INFINITY;
        auto scores = [&](bool relative) {  // log2 scores, less the running maximum
#pragma unroll
          for (int g = 0; g < NT / 8; ++g)
#pragma unroll
            for (int e = 0; e < 4; ++e)
              x[g][e] = __fadd_rn(__fmul_rn(v[g][e], scale_log2), relative ? -m_ref[2 * g + (e & 1)] : 0.f);
          if (valid < kKeys) {
#pragma unroll
            for (int g = 0; g < NT / 8; ++g)
#pragma unroll
              for (int e = 0; e < 4; ++e)
                if (!(e < 2 ? in0 : in1)) x[g][e] = -INFINITY;
          }
        };
        scores(true);
#pragma unroll
        for (int g = 0; g < NT / 8; ++g)
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            top = fmaxf(top, x[g][e]);
            x[g][e] = ex2(x[g][e]);
          }
        const bool raise = soft_any(i == 0 || top > kRaise);
        if (tile > 0) wait_or_abort(s, &s.pv_done, (tile - 1) & 1, err, 89);  // P is free, O^T at rest
        __syncwarp();
        if (raise) {
          float mx[V];
          scores(false);
#pragma unroll
          for (int n = 0; n < V; ++n) mx[n] = fmaxf(x[n >> 1][n & 1], x[n >> 1][2 + (n & 1)]);
          const int first = reduce_columns<V>(mx, [](float a, float c) { return fmaxf(a, c); });
#pragma unroll
          for (int n = 0; n < VF; ++n) s.red[sw][frag_col(first + n)] = mx[n];
          soft_barrier();
          if (tid < NT) {  // one thread a column
            float mn = fmaxf(fmaxf(s.red[0][tid], s.red[1][tid]), fmaxf(s.red[2][tid], s.red[3][tid]));
            const float old = i == 0 ? 0.f : s.mcol[tid];
            // no finite score yet: a reference that the first one passes
            mn = i == 0 ? (mn == -INFINITY ? kNoMax : mn) : fmaxf(mn, old);
            s.mcol[tid] = mn;
            s.fac[tid] = i == 0 ? 1.f : ex2(old - mn);  // (2^-mn may be infinite, and l is 0 yet)
          }
          soft_barrier();
#pragma unroll
          for (int n = 0; n < V; ++n) {
            m_ref[n] = s.mcol[frag_col(n)];
            l[n] *= s.fac[frag_col(n)];
          }
          if (i > 0) {
            tc_fence_after();
#pragma unroll 1
            for (int k = 0; k < S::kGroups * (NT / 16); ++k) {  // 16 columns of 128 dims at a time
              const int col = k % (NT / 16) * 16;
              const uint32_t at = tmem_o + lane_off + k / (NT / 16) * NT + col;
              float o[16];
              uint32_t u[16];
              tmem_ld16(at, o);
#pragma unroll
              for (int n = 0; n < 16; ++n) u[n] = __float_as_uint(o[n] * s.fac[col + n]);
              tmem_st16(at, u);
            }
            tmem_wait_st();
          }
          scores(true);
#pragma unroll
          for (int g = 0; g < NT / 8; ++g)
#pragma unroll
            for (int e = 0; e < 4; ++e) x[g][e] = ex2(x[g][e]);
        }
#pragma unroll
        for (int g = 0; g < NT / 8; ++g) {
          l[2 * g] += x[g][0] + x[g][2];
          l[2 * g + 1] += x[g][1] + x[g][3];
          uint8_t* dst = s.p + (lane & 3) * 4;
          *reinterpret_cast<uint32_t*>(dst + sw128_offset(row, g)) = pack_bf16(x[g][0], x[g][1]);
          *reinterpret_cast<uint32_t*>(dst + sw128_offset(row + 8, g)) = pack_bf16(x[g][2], x[g][3]);
        }
        if (valid < kKeys) {  // the sequence's last tile: rows past the context
          const int st = tile % S::kStages;
          for (int g = 0; g < S::kGroups; ++g)
            wait_or_abort(s, &s.kv_full[st][g], (tile / S::kStages) & 1, err, 88);
          const int per_row = R / 8;  // 16-byte vectors of a row's latent
          for (int e = tid; e < (kKeys - valid) * per_row; e += kSoft * 32) {
            const int r = valid + e / per_row, x = e % per_row;
            *reinterpret_cast<uint4*>(s.k[st] + (x >> 3) * S::kChunkBytes + r * 128 + (x & 7) * 16) =
                make_uint4(0, 0, 0, 0);
          }
        }
        fence_proxy_async_smem();
        tc_fence_before();
        __syncwarp();
        if (lane == 0) mbar_arrive(&s.p_full);
      }
      // ---- the piece's partial result
      wait_or_abort(s, &s.pv_done, (tile - 1) & 1, err, 89);
      __syncwarp();
      tc_fence_after();
      const int64_t slot = ((int64_t)ht * (B + ctas) + b + c) * heads_per_cta;
      {
        float part[V];
#pragma unroll
        for (int n = 0; n < V; ++n) part[n] = l[n];
        const int first = reduce_columns<V>(part, [](float x, float y) { return x + y; });
#pragma unroll
        for (int n = 0; n < VF; ++n) s.red[sw][frag_col(first + n)] = part[n];
      }
      soft_barrier();
      if (tid < NT) {
        const float sum = s.red[0][tid] + s.red[1][tid] + s.red[2][tid] + s.red[3][tid];
        s.fac[tid] = sum == 0.f ? 0.f : __fdividef(1.f, sum);
        if (tid < nheads) part_ml[slot + tid] = make_float2(sum == 0.f ? -INFINITY : s.mcol[tid], sum);
      }
      soft_barrier();
#pragma unroll 1
      for (int k = 0; k < S::kGroups * (NT / 16); ++k) {
        const int col = k % (NT / 16) * 16, m = k / (NT / 16);
        float o[16];
        tmem_ld16(tmem_o + lane_off + m * NT + col, o);
        // a warp writes 32 consecutive dims of one head at a time
        float* dst = part_o + (slot + col) * R + m * 128 + quad * 32 + lane;
#pragma unroll
        for (int n = 0; n < 16; ++n)
          if (col + n < nheads) dst[n * R] = o[n] * s.fac[col + n];
      }
      tc_fence_before();  // O^T has been read: ordered before the next p_full
    }
  }
  tc_fence_before();
  __syncthreads();
  if (warp == kMma) {
    tc_fence_after();
    tmem_dealloc(tmem, 512);
  }
}

// ------------------------------------------------------------- attention, CTA pairs
//
// Up to 128 heads of a rank-512 latent.  Here the heads are the MMA's M:
//   S [128 heads, 64 keys] = qa . K^T     O [128 heads, 256 dims] += P . c
// A cluster of two CTAs takes tiles of 128 keys.  Each computes the scores of its own 64 and
// the output's own 256 dims over all 128, so the scores' operand qa may come from tensor memory
// (O takes 256 columns, two thirds of qa 192, S 64) and no product is done twice: an MMA reads
// its 2 KB of keys for 32 cycles of work, where the 64-head form reads 4 KB of operands.
// The two CTAs exchange the rows' maxima (st.async, one float a row and tile) and P (4 KB a
// warp, copied from shared memory to shared memory): both scale a row by the same maximum.
// The values of the other CTA's keys come from L2 a second time (13 chunks of 64 keys x 64 dims
// a tile instead of 9).
//
// S(t + 1) is issued before the second product of t: the softmax warps (one thread a head) take
// S(t) into registers at once, so one S tile in tensor memory is enough, and maxima, exponentials
// and the exchange of P run behind S(t + 1).  The chunks live in three rings, each in the order
// in which it is freed: a: the 5 that only the scores read, b: the 4 of the own keys and dims,
// which both products read (two tiles), c: the 4 of the other's keys.
//
// Whole calls, 64-head tiles and pairs: 192 x 8192 tokens x 128 heads 674 and 508 us, 64 x 4096 x 128 145
// and 119, 64 x 500 x 128 56 and 51, 16 x 1000 x 80 31 and 30; at 64 heads and fewer, where half
// of the MMA's rows would be empty, 151 and 189 (64 x 8192 x 64).  With L2 flushed 8 x 2048 x 128 41 and
// 41, 4 x 1000 x 128 37 and 35; a lone request loses by the pairs' longer set-up and piece's
// end, 1 x 2048 x 128 33 and 34, 1 x 2048 x 80 29 and 31, 1 x 512 x 128 29 and 33.  A tile takes 4,100 cycles where its
// MMAs alone would take 2,500 (S 1,460, second product 1,050): operands, arriving chunks and P
// share the shared memory, and loads from L2 run at 5.9 TB/s over the GPU.  The end of a piece
// (queries to tensor memory, partial result) takes 19,000 cycles; a form that turned the queries in
// shared memory and overlapped more of it took as long over whole calls.
constexpr int kPairThreads = 256;  // warps 0-2 TMA (a, b, c), 3 MMA, 4-7 softmax
constexpr int kPairKeys = 128;
constexpr int kPairHeads = 64;  // more heads than this take pairs
constexpr uint32_t kChunk = 64 * 128;  // 64 keys x 64 dims

struct alignas(1024) PairSmem {
  uint8_t a[6][kChunk];
  uint8_t b[2][4][kChunk];
  uint8_t c[4][kChunk];
  uint8_t q[3][128 * 128];
  uint8_t p[2][128 * 128];  // by the CTA whose keys they are of
  float other[2][128];      // the other CTA's maxima (or sums)
  uint64_t a_full[6], a_empty[6], b_full[2], b_empty[2], c_full, c_empty, q_full, q_empty, s_full, s_free, p_full,
      p_free, other_full[2][4], drained;
  uint32_t tmem_base;
  volatile int abort_flag;
};

__device__ __forceinline__ uint32_t pair_rank() {
  uint32_t r;
  asm volatile("mov.u32 %0, %%cluster_ctarank;" : "=r"(r));
  return r;
}
__device__ __forceinline__ void pair_sync() {
  asm volatile("barrier.cluster.arrive.release.aligned;\n\tbarrier.cluster.wait.acquire.aligned;" ::: "memory");
}
__device__ __forceinline__ uint32_t in_cta(const void* p, uint32_t rank) {  // the same place in a CTA of the cluster
  uint32_t a;
  asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(a) : "r"(smem_u32(p)), "r"(rank));
  return a;
}
// wait_or_abort that polls: the clock and the abort flag are read rarely (both are slow beside a poll)
__device__ __forceinline__ bool poll_or_abort(PairSmem& s, uint64_t* bar, uint32_t parity, int* err, int code) {
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
__device__ __forceinline__ bool try_wait_cluster(uint64_t* bar, uint32_t parity) {
  uint32_t ok;
  asm volatile(
      "{\n\t.reg .pred p;\n\t"
      "mbarrier.try_wait.parity.acquire.cluster.shared::cta.b64 p, [%1], %2;\n\t"
      "selp.u32 %0, 1, 0, p;\n\t}"
      : "=r"(ok)
      : "r"(smem_u32(bar)), "r"(parity)
      : "memory");
  return ok != 0;
}

__global__ void __cluster_dims__(2, 1, 1) __launch_bounds__(kPairThreads, 1)
    latent_attn_pair_kernel(const __grid_constant__ CUtensorMap q_map, const __grid_constant__ CUtensorMap c_map,
                            const bf16* qa, const bf16* cache, int64_t num_blocks, int page,
                            const int32_t* block_tables, int max_blocks, const int32_t* table_rows, int num_tables,
                            const int32_t* ctx_lens, const int32_t* table, float* part_o, float2* part_ml, int B, int H,
                            int heads_per_cta, int head_tiles, float scale_log2, int* err) {
  griddep_launch();
  constexpr int R = 512, W = R + kRot;
  extern __shared__ __align__(1024) uint8_t smem_raw[];
  PairSmem& s = *reinterpret_cast<PairSmem*>(smem_raw);
  const int warp = __shfl_sync(0xffffffffu, threadIdx.x / 32, 0), lane = threadIdx.x % 32;
  const int rank = (int)pair_rank(), pair = blockIdx.x / 2;
  const int ht = pair % head_tiles, c = pair / head_tiles;
  const int pairs = gridDim.x / 2 / head_tiles;
  const int h0 = ht * heads_per_cta, nheads = min(heads_per_cta, H - h0);
  if (smem_u32(smem_raw) & 1023) {  // the same in both CTAs
    if (threadIdx.x == 0) atomicCAS(err, 0, 83);
    return;
  }
  if (threadIdx.x == 0) {
    s.abort_flag = 0;
    for (int i = 0; i < 6; ++i) {
      mbar_init(&s.a_full[i], 1);
      mbar_init(&s.a_empty[i], 1);
    }
    for (int i = 0; i < 2; ++i) {
      mbar_init(&s.b_full[i], 1);
      mbar_init(&s.b_empty[i], 1);
      for (int w = 0; w < 4; ++w) mbar_init(&s.other_full[i][w], 1);
    }
    mbar_init(&s.c_full, 1);
    mbar_init(&s.c_empty, 1);
    mbar_init(&s.q_full, 5);  // the copies, and four warps' part in tensor memory
    mbar_init(&s.q_empty, 1);
    mbar_init(&s.s_full, 1);
    mbar_init(&s.s_free, 4);
    mbar_init(&s.p_full, 4);  // and the bytes of the other CTA's P
    mbar_init(&s.p_free, 2);  // both CTAs' second product
    mbar_init(&s.drained, 1);
    fence_barrier_init();
  }
  griddep_wait();  // before the allocation: a CTA of the grid waited for may still need its own
  if (warp == 3) tmem_alloc(&s.tmem_base, 512);
  tc_fence_before();
  pair_sync();  // both CTAs' barriers stand before the other uses them
  tc_fence_after();
  const uint32_t tmem = __shfl_sync(0xffffffffu, s.tmem_base, 0);
  const uint32_t tmem_q = tmem + 64, tmem_o = tmem + 256;
  Pieces pc(table, ctx_lens, B, max_blocks * page, c);
  // The chunk of 64 dims that is the i-th in the scores' product: the rotary dims, the other CTA's
  // 256 dims, the own.  The first three of qa are in shared memory, the rest in tensor memory.
  auto dims = [&](int i) { return i == 0 ? R : i < 5 ? 256 * (1 - rank) + 64 * (i - 1) : 256 * rank + 64 * (i - 5); };

  if (warp < 3) {
    // ------------------------------------------------------------ TMA producers
    const int half = warp == 2 ? 1 - rank : rank;  // whose keys of the tile
    const int pages = kKeys / page;
    const int oob = (int)(num_blocks * page);  // a row past the cache reads as zeros
    int sent = 0, chunks = 0, nq = 0;
    bool ok = true;
    auto page_row = [&](int trow, int tile) {  // lane l < pages: first row of page l of the 64 keys
      const int j = (2 * tile + half) * pages + lane;
      if (lane >= pages || j >= (pc.keys() + page - 1) / page) return oob;
      const int blk = trow >= 0 && trow < num_tables ? block_tables[(int64_t)trow * max_blocks + j] : -1;
      if (blk >= 0 && blk < num_blocks) return blk * page;
      atomicCAS(err, 0, 82);
      return oob;
    };
    for (; ok && pc.more(); pc.next()) {
      const int b = pc.b, t0 = pc.first(), n = pc.tiles();
      const int trow = table_rows != nullptr ? table_rows[b] : b;
      int y = page_row(trow, t0), y1 = n > 1 ? page_row(trow, t0 + 1) : oob;
      if (warp == 0) {
        if (nq > 0) ok = wait_or_abort(s, &s.q_empty, (nq - 1) & 1, err, 84);
        if (!__all_sync(0xffffffffu, ok)) break;
        if (elect_one()) {
          mbar_arrive_expect_tx(&s.q_full, sizeof(s.q));
          for (int i = 0; i < 3; ++i) tma_load_2d(s.q[i], &q_map, &s.q_full, dims(i), b * H + h0);
        }
        ++nq;
      }
      for (int i = 0; i < n; ++i, ++sent) {
        const int y2 = i + 2 < n ? page_row(trow, t0 + i + 2) : oob;
        int yy[4];
#pragma unroll
        for (int pg = 0; pg < 4; ++pg) yy[pg] = __shfl_sync(0xffffffffu, y, pg);
        if (warp == 1 && y2 < oob)  // whole pages come into L2 two tiles ahead, a lane each
          asm volatile("cp.async.bulk.prefetch.L2.global [%0], %1;" ::"l"(cache + (int64_t)y2 * W), "r"(page * W * 2)
                       : "memory");
        auto load = [&](uint8_t* dst, uint64_t* bar, int x) {
#pragma unroll
          for (int pg = 0; pg < 4; ++pg)
            if (pg < pages) tma_load_2d(dst + pg * page * 128, &c_map, bar, x, yy[pg]);
        };
        if (warp == 0) {
          for (int k = 0; ok && k < 5; ++k) {
            const int st = chunks % 6;
            if (chunks >= 6) ok = wait_or_abort(s, &s.a_empty[st], (chunks / 6 - 1) & 1, err, 84);
            ok = __all_sync(0xffffffffu, ok);
            if (!ok) break;
            if (elect_one()) {
              mbar_arrive_expect_tx(&s.a_full[st], kChunk);
              load(s.a[st], &s.a_full[st], dims(k));
            }
            __syncwarp();
            ++chunks;
          }
          if (!ok) break;
        } else {
          const int st = warp == 1 ? sent & 1 : 0;
          uint64_t* full = warp == 1 ? &s.b_full[st] : &s.c_full;
          if (warp == 1 && sent >= 2) ok = wait_or_abort(s, &s.b_empty[st], ((sent >> 1) - 1) & 1, err, 84);
          if (warp == 2 && sent >= 1) ok = wait_or_abort(s, &s.c_empty, (sent - 1) & 1, err, 84);
          ok = __all_sync(0xffffffffu, ok);
          if (!ok) break;
          if (elect_one()) {
            mbar_arrive_expect_tx(full, 4 * kChunk);
            for (int k = 0; k < 4; ++k) load(warp == 1 ? s.b[st][k] : s.c[k], full, 256 * rank + 64 * k);
          }
          __syncwarp();
        }
        y = y1;
        y1 = y2;
      }
    }
    // the copies in flight end before the CTA does, on the way out of a time-out too
    if (lane == 0) {
      if (warp == 0) {
        if (nq > 0) {  // the other arrivals of q_full may be missing after a time-out: chunks alone tell
          for (int i = max(0, chunks - 6); i < chunks; ++i) mbar_wait_sleep(&s.a_full[i % 6], (i / 6) & 1);
          mbar_wait_sleep(&s.q_full, (nq - 1) & 1);
        }
      } else if (warp == 1) {
        for (int i = max(0, sent - 2); i < sent; ++i) mbar_wait_sleep(&s.b_full[i & 1], (i >> 1) & 1);
      } else if (sent > 0) {
        mbar_wait_sleep(&s.c_full, (sent - 1) & 1);
      }
    }
  } else if (warp == 3) {
    // -------------------------------------------------------------- MMA issuer
    if (elect_one()) {
      constexpr uint32_t idesc_s = idesc_bf16<128, 64>();
      constexpr uint32_t idesc_o = idesc_bf16<128, 256>() | kIdescBMn;
      constexpr uint64_t kStep = kChunk >> 4;
      const uint64_t a_desc = smem_desc_sw128(smem_u32(s.a[0])), b_desc = smem_desc_sw128(smem_u32(s.b[0][0]));
      const uint64_t q_desc = smem_desc_sw128(smem_u32(s.q[0]));
      const uint64_t p_own = smem_desc_sw128(smem_u32(s.p[rank])), p_other = smem_desc_sw128(smem_u32(s.p[1 - rank]));
      const uint64_t v_own = smem_desc_mn_sw128(smem_u32(s.b[0][0]), kChunk, 1024);
      const uint64_t v_other = smem_desc_mn_sw128(smem_u32(s.c[0]), kChunk, 1024);
      const int total = pc.end - pc.at;
      Pieces sp = pc;
      int left_s = sp.more() ? sp.tiles() : 0, left_p = left_s, nq = 0, chunks = 0;
      bool ok = true, first_s = true, first_p = true;
      for (int t = 0; ok && t <= total; ++t) {
        if (t < total) {
          if (first_s) ok = poll_or_abort(s, &s.q_full, nq & 1, err, 86);
          if (t > 0) ok = ok && poll_or_abort(s, &s.s_free, (t - 1) & 1, err, 86);
          for (int k = 0; ok && k < 5; ++k, ++chunks) {
            const int st = chunks % 6;
            ok = poll_or_abort(s, &s.a_full[st], (chunks / 6) & 1, err, 86);
            if (!ok) break;
            tc_fence_after();
            if (k < 3) {
#pragma unroll
              for (int kk = 0; kk < 4; ++kk)
                mma_bf16(tmem, q_desc + k * 1024 + kk * 2, a_desc + st * kStep + kk * 2, idesc_s, k + kk > 0);
            } else {
#pragma unroll
              for (int kk = 0; kk < 4; ++kk)
                mma_bf16_tmem_a(tmem, tmem_q + (k - 3) * 32 + kk * 8, a_desc + st * kStep + kk * 2, idesc_s, 1);
            }
            mma_commit(&s.a_empty[st]);
          }
          ok = ok && poll_or_abort(s, &s.b_full[t & 1], (t >> 1) & 1, err, 86);
          if (!ok) break;
          tc_fence_after();
#pragma unroll
          for (int k = 0; k < 4; ++k)
#pragma unroll
            for (int kk = 0; kk < 4; ++kk)
              mma_bf16_tmem_a(tmem, tmem_q + (k + 2) * 32 + kk * 8, b_desc + ((t & 1) * 4 + k) * kStep + kk * 2,
                              idesc_s, 1);
          mma_commit(&s.s_full);
          first_s = false;
          if (--left_s == 0) {  // the piece's last scores: its queries are free
            mma_commit(&s.q_empty);
            ++nq;
            first_s = true;
            sp.next();
            left_s = sp.more() ? sp.tiles() : 0;
          }
        }
        if (t > 0) {
          const int u = t - 1;
          ok = poll_or_abort(s, &s.p_full, u & 1, err, 86) && poll_or_abort(s, &s.c_full, u & 1, err, 86);
          if (!ok) break;
          tc_fence_after();
#pragma unroll
          for (int kk = 0; kk < 4; ++kk)
            mma_bf16(tmem_o, p_own + kk * 2, v_own + (u & 1) * 4 * kStep + kk * 128, idesc_o, !(first_p && kk == 0));
          mma_commit(&s.b_empty[u & 1]);
#pragma unroll
          for (int kk = 0; kk < 4; ++kk) mma_bf16(tmem_o, p_other + kk * 2, v_other + kk * 128, idesc_o, 1);
          mma_commit(&s.c_empty);
          asm volatile(  // on both CTAs' barrier
              "tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.multicast::cluster.b64 [%0], %1;" ::"r"(
                  smem_u32(&s.p_free)),
              "h"((uint16_t)3)
              : "memory");
          first_p = false;
          if (--left_p == 0) {
            pc.next();
            left_p = pc.more() ? pc.tiles() : 0;
            first_p = true;
          }
        }
      }
      // every MMA issued has finished before the tensor memory is freed
      mma_commit(&s.drained);
      mbar_wait_sleep(&s.drained, 0);
    }
  } else {
    // ------------------------------------------------------- softmax, epilogue
    const int quad = warp & 3, row = quad * 32 + lane;  // head h0 + row
    const uint32_t lane_off = (uint32_t)(quad * 32) << 16;
    const uint32_t peer_val = in_cta(&s.other[0][row], 1 - rank), peer_bar = in_cta(&s.other_full[0][quad], 1 - rank);
    const uint32_t peer_p = in_cta(s.p[rank] + quad * 4096, 1 - rank), peer_p_full = in_cta(&s.p_full, 1 - rank);
    int xch = 0;  // exchanges with the other CTA
    // A thread sends x + 1 after it has read x: two places are enough.
    auto send = [&](float v) {
      const int at = xch & 1;
      if (lane == 0) mbar_arrive_expect_tx(&s.other_full[at][quad], 128);
      asm volatile("st.async.shared::cluster.mbarrier::complete_tx::bytes.b32 [%0], %1, [%2];" ::"r"(
                       peer_val + at * 512),
                   "r"(__float_as_uint(v)), "r"(peer_bar + at * 32)
                   : "memory");
    };
    auto receive = [&]() {
      const int at = xch & 1;
      uint64_t* bar = &s.other_full[at][quad];
      const uint64_t t0 = globaltimer_ns();
      while (!try_wait_cluster(bar, (xch >> 1) & 1) && !s.abort_flag) {
        if (globaltimer_ns() - t0 > 2000000000ull) {
          atomicCAS(err, 0, 87);
          s.abort_flag = 1;
        }
      }
      __syncwarp();
      ++xch;
      return s.other[at][row];
    };
    auto load_q = [&](int b) {  // qa's later six chunks of this thread's head -> tensor memory
      const bf16* src = qa + ((int64_t)b * H + h0 + row) * W;
#pragma unroll 1
      for (int g = 0; g < 3; ++g) {
        uint4 v[16];
#pragma unroll
        for (int k = 0; k < 16; ++k)
          v[k] = row < nheads ? *reinterpret_cast<const uint4*>(src + dims(3 + 2 * g + k / 8) + k % 8 * 8)
                              : make_uint4(0, 0, 0, 0);
#pragma unroll
        for (int k = 0; k < 4; ++k) {
          uint32_t u[16];
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            u[4 * e] = v[4 * k + e].x, u[4 * e + 1] = v[4 * k + e].y;
            u[4 * e + 2] = v[4 * k + e].z, u[4 * e + 3] = v[4 * k + e].w;
          }
          tmem_st16(tmem_q + lane_off + g * 64 + k * 16, u);
        }
      }
      tmem_wait_st();
      tc_fence_before();
      __syncwarp();
      if (lane == 0) mbar_arrive(&s.q_full);
    };
    if (pc.more()) load_q(pc.b);
    int tile = 0;  // of the pair
    bool live = true;  // false after a time-out
    while (pc.more()) {
      const int b = pc.b, n_tiles = pc.tiles();
      const int left = pc.keys() - pc.first() * kPairKeys;  // keys from the piece's first on
      float m = -INFINITY, l = 0.f;
      for (int i = 0; i < n_tiles; ++i, ++tile) {
        live = __all_sync(0xffffffffu, wait_or_abort(s, &s.s_full, tile & 1, err, 88) && !s.abort_flag);
        if (!live) break;
        tc_fence_after();
        float v[2][32];
        {
          uint32_t r0[32], r1[32];
          tmem_ld_start(tmem + lane_off, r0);
          tmem_ld_start(tmem + lane_off + 32, r1);
          tmem_ld_wait(r0);
          tmem_ld_wait(r1);
#pragma unroll
          for (int n = 0; n < 32; ++n) {
            v[0][n] = __uint_as_float(r0[n]) * scale_log2;
            v[1][n] = __uint_as_float(r1[n]) * scale_log2;
          }
        }
        tc_fence_before();
        __syncwarp();
        if (lane == 0) mbar_arrive(&s.s_free);
        const int valid = left - i * kPairKeys - rank * 64;  // of this CTA's keys
        if (valid < 64) {
#pragma unroll
          for (int n = 0; n < 64; ++n)
            if (n >= valid) v[n >> 5][n & 31] = -INFINITY;
        }
        float top4[4] = {-INFINITY, -INFINITY, -INFINITY, -INFINITY};
#pragma unroll
        for (int n = 0; n < 64; ++n) top4[n & 3] = fmaxf(top4[n & 3], v[n >> 5][n & 31]);
        const float top = fmaxf(fmaxf(top4[0], top4[1]), fmaxf(top4[2], top4[3]));
        send(top);
        uint32_t p[32];
        float sum;
        auto exps = [&]() {
          const float ref = m == -INFINITY ? 0.f : m;  // no finite score yet: every p is 0 or NaN
          float add[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
          for (int n = 0; n < 64; n += 2) {
            const float e0 = ex2(v[n >> 5][n & 31] - ref), e1 = ex2(v[n >> 5][(n & 31) + 1] - ref);
            add[n & 2] += e0;
            add[(n & 2) + 1] += e1;
            p[n >> 1] = pack_bf16(e0, e1);
          }
          sum = (add[0] + add[1]) + (add[2] + add[3]);
        };
        if (i > 0) exps();  // with the present maximum, while the other CTA's is under way
        const float M = fmaxf(top, receive());
        const bool up = M > m + kRaise;
        const bool raise = __any_sync(0xffffffffu, up);
        if (tile > 0) wait_or_abort(s, &s.p_free, (tile - 1) & 1, err, 89);  // P is free, O at rest
        __syncwarp();
        if (raise && i > 0) {
          const float fac = up ? ex2(m - M) : 1.f;
          l *= fac;
          tc_fence_after();
#pragma unroll 1
          for (int k = 0; k < 16; ++k) {
            float o[16];
            uint32_t u[16];
            tmem_ld16(tmem_o + lane_off + k * 16, o);
#pragma unroll
            for (int n = 0; n < 16; ++n) u[n] = __float_as_uint(o[n] * fac);
            tmem_st16(tmem_o + lane_off + k * 16, u);
          }
          tmem_wait_st();
        }
        if (up) m = M;
        if (raise || i == 0) exps();
        l += sum;
#pragma unroll
        for (int k = 0; k < 8; ++k)
          *reinterpret_cast<uint4*>(s.p[rank] + sw128_offset(row, k)) =
              make_uint4(p[4 * k], p[4 * k + 1], p[4 * k + 2], p[4 * k + 3]);
        if (left - i * kPairKeys < kPairKeys) {  // the sequence's last tile: value rows past the context
          wait_or_abort(s, &s.b_full[tile & 1], (tile >> 1) & 1, err, 88);
          wait_or_abort(s, &s.c_full, tile & 1, err, 88);
#pragma unroll 1
          for (int own = 0; own < 2; ++own) {
            const int first = max(0, left - i * kPairKeys - (own ? rank : 1 - rank) * 64);
            uint8_t* at = own ? s.b[tile & 1][0] : s.c[0];
            for (int e = row; e < (64 - first) * 32; e += 128)  // 16-byte vectors of a row's 256 dims
              *reinterpret_cast<uint4*>(at + (e & 31) / 8 * kChunk + (first + (e >> 5)) * 128 + (e & 7) * 16) =
                  make_uint4(0, 0, 0, 0);
          }
        }
        fence_proxy_async_smem();
        tc_fence_before();
        __syncwarp();
        if (lane == 0) {
          asm volatile(
              "cp.async.bulk.shared::cluster.shared::cta.mbarrier::complete_tx::bytes [%0], [%1], %2, [%3];" ::"r"(
                  peer_p),
              "r"(smem_u32(s.p[rank] + quad * 4096)), "r"(4096), "r"(peer_p_full)
              : "memory");
          if (quad == 0) {
            mbar_arrive_expect_tx(&s.p_full, 128 * 128);
          } else {
            mbar_arrive(&s.p_full);
          }
        }
      }
      if (!live) break;
      // ---- the piece's partial result; the next piece's queries first
      send(l);
      pc.next();
      if (pc.more()) load_q(pc.b);
      l += receive();
      wait_or_abort(s, &s.p_free, (tile - 1) & 1, err, 89);
      __syncwarp();
      tc_fence_after();
      const int64_t slot = ((int64_t)ht * (B + pairs) + b + c) * heads_per_cta;
      if (rank == 0 && row < nheads) part_ml[slot + row] = make_float2(l == 0.f ? -INFINITY : m, l);
      const float inv = l == 0.f ? 0.f : __fdividef(1.f, l);
      uint8_t* turn = s.p[rank] + quad * 4096;  // 32 rows x 32 dims, turned for whole-line stores
#pragma unroll 1
      for (int k = 0; k < 8; ++k) {
        float o[32];
        tmem_ld32w(tmem_o + lane_off + k * 32, o);
#pragma unroll
        for (int q = 0; q < 8; ++q)
          *reinterpret_cast<float4*>(turn + lane * 128 + ((q ^ (lane & 7)) * 16)) =
              make_float4(o[4 * q] * inv, o[4 * q + 1] * inv, o[4 * q + 2] * inv, o[4 * q + 3] * inv);
        __syncwarp();
#pragma unroll
        for (int q = 0; q < 8; ++q) {
          const int r = 4 * q + (lane >> 3), seg = lane & 7;
          if (quad * 32 + r < nheads)
            *reinterpret_cast<float4*>(part_o + (slot + quad * 32 + r) * R + rank * 256 + k * 32 + seg * 4) =
                *reinterpret_cast<const float4*>(turn + r * 128 + ((seg ^ (r & 7)) * 16));
        }
        __syncwarp();
      }
      tc_fence_before();  // O has been read: ordered before the next p_full
    }
  }
  tc_fence_before();
  __syncthreads();
  if (s.abort_flag && threadIdx.x == 0)  // after a time-out: copies to the other CTA have long landed
    for (const uint64_t t0 = globaltimer_ns(); globaltimer_ns() - t0 < 100000;) {
    }
  pair_sync();  // no CTA leaves while its peer may still write to it
  if (warp == 3) {
    tc_fence_after();
    tmem_dealloc(tmem, 512);
  }
}

// -------------------------------------------------------------- head products
//
// y[b, h, n] = sum_k x[b, h, k] w_h[k, n], small matrices per head, bound by the weights (128 KB +
// 128 KB a head at R = 512) and the rows' traffic.  Few rows: mma.sync on 16-row tiles, many
// small CTAs, since latency is all that counts.  Else: tcgen05 on 128-row tiles fed by
// TMA; at 64 rows x 128 heads the mma.sync form took 13 us for either product, held back by its
// shared-memory loads, where this one takes 10 (absorb, which writes 9 MB) and 7 us.

__device__ __forceinline__ void cp16(void* dst, const void* src) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(smem_u32(dst)), "l"(src) : "memory");
}
__device__ __forceinline__ void cp_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int N>
__device__ __forceinline__ void cp_wait() { asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory"); }

// qa[b, h, R:] = q[b, h, 128:] for ROWS rows, by 128 threads: all loads before the first store (the
// compiler cannot tell that they do not overlap).
template <int R, int ROWS>
__device__ __forceinline__ void copy_rotary(const bf16* q, int64_t q_stride, bf16* qa, int rows, int H, int h) {
  constexpr int N = ROWS * 8 / 128;
  uint4 v[N];
  const int seg = threadIdx.x & 7;
#pragma unroll
  for (int i = 0; i < N; ++i) {
    const int b = (i * 128 + threadIdx.x) >> 3;
    if (b < rows)
      v[i] = *reinterpret_cast<const uint4*>(q + (int64_t)b * q_stride + (int64_t)h * (kNope + kRot) + kNope + seg * 8);
  }
#pragma unroll
  for (int i = 0; i < N; ++i) {
    const int b = (i * 128 + threadIdx.x) >> 3;
    if (b < rows) *reinterpret_cast<uint4*>(qa + ((int64_t)b * H + h) * (R + kRot) + R + seg * 8) = v[i];
  }
}

// qa[b, h, :R] = q[b, h, :128] . w[h, :128, :], qa[b, h, R:] = q[b, h, 128:].
// One CTA per (64 columns, head, 16 rows); qa is bf16, the tensor cores' operand type.
template <int R>
__global__ void __launch_bounds__(128) latent_absorb_kernel(const bf16* q, int64_t q_stride,
                                                            const bf16* w, bf16* qa, int B,
                                                            int H, const int32_t* ctx_lens, int limit, int keys,
                                                            int ctas, int32_t* table) {
  griddep_entry();
  constexpr int MROWS = 16;
  if (blockIdx.x == gridDim.x - 1 && blockIdx.y == 0 && blockIdx.z == 0)
    write_schedule(ctx_lens, B, limit, keys, ctas, table);
  constexpr int kPitchW = 64 + 8, kPitchX = kNope + 8;  // 16 bytes of padding: conflict-free ldmatrix
  __shared__ __align__(16) bf16 ws[kNope * kPitchW];
  __shared__ __align__(16) bf16 xs[MROWS * kPitchX];
  const int n0 = blockIdx.x * 64, h = blockIdx.y, b0 = blockIdx.z * MROWS;
  const int rows = min(MROWS, B - b0);
  q += (int64_t)b0 * q_stride;
  qa += (int64_t)b0 * H * (R + kRot);
  const int t = threadIdx.x, warp = t >> 5, lane = t & 31;
  const bf16* wk = w + (int64_t)h * (kNope + kVal) * R + n0;
  for (int i = t; i < kNope * 8; i += 128)
    cp16(ws + (i >> 3) * kPitchW + (i & 7) * 8, wk + (int64_t)(i >> 3) * R + (i & 7) * 8);
  for (int i = t; i < MROWS * 16; i += 128) {
    const int r = i >> 4;
    if (r < rows)
      cp16(xs + r * kPitchX + (i & 15) * 8, q + (int64_t)r * q_stride + (int64_t)h * (kNope + kRot) + (i & 15) * 8);
  }
  cp_commit();
  if (blockIdx.x == 0) {  // the rotary part
    copy_rotary<R, MROWS>(q, q_stride, qa, rows, H, h);
  }
  cp_wait<0>();
  __syncthreads();
  const int c0 = warp * 16;  // a warp's columns
  float acc[2][4] = {};
#pragma unroll
  for (int ks = 0; ks < kNope / 16; ++ks) {
    uint32_t a[4], bb[4];
    ldmatrix_x4(a, smem_u32(xs + (lane & 15) * kPitchX + ks * 16 + (lane >> 4) * 8));
    ldmatrix_x4_trans(bb, smem_u32(ws + (ks * 16 + (lane & 15)) * kPitchW + c0 + (lane >> 4) * 8));
    mma_bf16_16816(acc[0], a, {bb[0], bb[1]});
    mma_bf16_16816(acc[1], a, {bb[2], bb[3]});
  }
  __syncthreads();  // the result takes the queries' place, then leaves in whole 128-byte rows
#pragma unroll
  for (int nt = 0; nt < 2; ++nt)
#pragma unroll
    for (int e = 0; e < 2; ++e)
      *reinterpret_cast<uint32_t*>(xs + ((lane >> 2) + e * 8) * kPitchX + c0 + nt * 8 + (lane & 3) * 2) =
          pack_bf16(acc[nt][2 * e], acc[nt][2 * e + 1]);
  __syncthreads();
  for (int i = t; i < MROWS * 8; i += 128) {
    const int b = i >> 3;
    if (b < rows)
      *reinterpret_cast<uint4*>(qa + ((int64_t)b * H + h) * (R + kRot) + n0 + (i & 7) * 8) =
          *reinterpret_cast<const uint4*>(xs + (i >> 3) * kPitchX + (i & 7) * 8);
  }
}

// Joins a row's pieces: o[b, h] = sum_c w_c o_c / sum_c w_c, w_c = l_c 2^(m_c - M), written as hi + lo,
// two bf16 whose sum keeps 16 bits of it: the product below then rounds nothing else.  A piece
// brings its maximum m_c and sum l_c apart: the sum of m_c and log2 l_c would round l_c to m_c's
// last place, 2^-6 at scores of 2^17.  One
// thread per 8 dims of ROWS rows, whole warps a row: the pieces' weights are spread over the
// lanes, and P pieces of every row are requested at once (few rows have many pieces: P = 8;
// many rows have one or two: P = 2, and two rows a thread).
template <int R, int P, int ROWS>
__global__ void __launch_bounds__(128)
    latent_join_kernel(const float* part_o, const float2* part_ml, const int32_t* table, bf16* hi, bf16* lo, int B,
                       int H, int heads_per_cta, int ctas) {
  griddep_entry();
  constexpr int kRowThreads = R / 8;
  const int lane = threadIdx.x & 31;
  const int64_t rows = (int64_t)B * H;
  const int64_t row0 = ((int64_t)blockIdx.x * (128 / kRowThreads) + threadIdx.x / kRowThreads) * ROWS;  // b * H + h
  const int k = threadIdx.x % kRowThreads * 8;
  const int64_t step = (int64_t)heads_per_cta * R;
  const int quota = table[0];
  int n[ROWS], most = 0;
  const float* src[ROWS];
  float e0[ROWS], e1[ROWS], l0[ROWS], l1[ROWS], inv[ROWS], x[ROWS][8] = {};
  float4 y[ROWS][P][2];
  auto load = [&](int p0) {
#pragma unroll
    for (int i = 0; i < ROWS; ++i)
#pragma unroll
      for (int p = 0; p < P; ++p)
        if (p0 + p < n[i]) {
          const float4* at = reinterpret_cast<const float4*>(src[i] + (p0 + p) * step);
          y[i][p][0] = at[0];
          y[i][p][1] = at[1];
        } else {  // its weight is 0
          y[i][p][0] = y[i][p][1] = make_float4(0.f, 0.f, 0.f, 0.f);
        }
  };
#pragma unroll
  for (int i = 0; i < ROWS; ++i) {
    n[i] = 0;
    src[i] = part_o;
    e0[i] = e1[i] = -INFINITY;
    l0[i] = l1[i] = 0.f;
    if (row0 + i < rows) {
      const int b = (int)((row0 + i) / H), h = (int)((row0 + i) % H);
      const int s0 = table[1 + b], s1 = table[2 + b], c0 = s0 / quota;
      n[i] = s1 > s0 ? (s1 - 1) / quota - c0 + 1 : 0;
      const int64_t slot = ((int64_t)(h / heads_per_cta) * (B + ctas) + b + c0) * heads_per_cta + h % heads_per_cta;
      src[i] = part_o + slot * R + k;
      if (lane < n[i]) {
        const float2 ml = part_ml[slot + (int64_t)lane * heads_per_cta];
        e0[i] = ml.x, l0[i] = ml.y;
      }
      if (lane + 32 < n[i]) {
        const float2 ml = part_ml[slot + (int64_t)(lane + 32) * heads_per_cta];
        e1[i] = ml.x, l1[i] = ml.y;
      }
    }
    most = max(most, n[i]);
  }
  load(0);  // under way with the weights
#pragma unroll
  for (int i = 0; i < ROWS; ++i) {
    float M = warp_max(fmaxf(e0[i], e1[i]));
    if (M == -INFINITY) M = 0.f;  // no finite score in the row: weights 0 (or NaN, which reaches the row)
    e0[i] = l0[i] * ex2(e0[i] - M), e1[i] = l1[i] * ex2(e1[i] - M);
    const float L = warp_sum(e0[i] + e1[i]);
    inv[i] = L == 0.f ? 0.f : 1.f / L;
  }
  for (int p0 = 0; p0 < most; p0 += P) {
    if (p0 > 0) load(p0);
#pragma unroll
    for (int i = 0; i < ROWS; ++i)
#pragma unroll
      for (int p = 0; p < P; ++p) {
        const float f = __shfl_sync(0xffffffffu, p0 < 32 ? e0[i] : e1[i], (p0 + p) & 31);
        const float4 u = y[i][p][0], v = y[i][p][1];
        x[i][0] += f * u.x, x[i][1] += f * u.y, x[i][2] += f * u.z, x[i][3] += f * u.w;
        x[i][4] += f * v.x, x[i][5] += f * v.y, x[i][6] += f * v.z, x[i][7] += f * v.w;
      }
  }
#pragma unroll
  for (int i = 0; i < ROWS; ++i) {
    if (row0 + i >= rows) return;
    uint32_t top[4], low[4];
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const float u = x[i][2 * j] * inv[i], v = x[i][2 * j + 1] * inv[i];
      top[j] = pack_bf16(u, v);
      const float2 f = __bfloat1622float2(*reinterpret_cast<const __nv_bfloat162*>(&top[j]));
      low[j] = pack_bf16(u - f.x, v - f.y);
    }
    *reinterpret_cast<uint4*>(hi + (row0 + i) * R + k) = make_uint4(top[0], top[1], top[2], top[3]);
    *reinterpret_cast<uint4*>(lo + (row0 + i) * R + k) = make_uint4(low[0], low[1], low[2], low[3]);
  }
}

// out[b, h, n] = sum_r (hi + lo)[b, h, r] w[h, 128 + n, r]: one CTA per (32 columns, head, 16 rows),
// everything it needs requested at once.
template <int R>
__global__ void __launch_bounds__(128)
    latent_out_kernel(const bf16* hi, const bf16* lo, const bf16* w,
                      bf16* out, int64_t out_stride, int B, int H) {
  griddep_entry();
  constexpr int MROWS = 16, NCOLS = 32, THREADS = 128;
  constexpr int kPitch = 128 + 8;
  constexpr int kSteps = R / 128, STAGES = kSteps + 1;
  constexpr int kStage = (NCOLS + 2 * MROWS) * kPitch;
  extern __shared__ __align__(16) uint8_t raw[];
  bf16* sm = reinterpret_cast<bf16*>(raw);  // a stage: [NCOLS] w, [MROWS] hi, [MROWS] lo rows
  const int n0 = blockIdx.x * NCOLS, h = blockIdx.y, b0 = blockIdx.z * MROWS, rows = min(MROWS, B - b0);
  const int t = threadIdx.x, warp = t >> 5, lane = t & 31;
  const bf16* wv = w + ((int64_t)h * (kNope + kVal) + kNope + n0) * R;
  auto load = [&](int c) {
    if (c < kSteps) {
      bf16* st = sm + (c % STAGES) * kStage;
      for (int i = t; i < NCOLS * 16; i += THREADS)
        cp16(st + (i >> 4) * kPitch + (i & 15) * 8, wv + (int64_t)(i >> 4) * R + c * 128 + (i & 15) * 8);
      for (int i = t; i < 2 * MROWS * 16; i += THREADS) {
        const int r = (i >> 4) % MROWS;
        if (r < rows)
          cp16(st + (NCOLS + (i >> 4)) * kPitch + (i & 15) * 8,
               (i >= MROWS * 16 ? lo : hi) + ((int64_t)(b0 + r) * H + h) * R + c * 128 + (i & 15) * 8);
      }
    }
    cp_commit();
  };
#pragma unroll
  for (int c = 0; c < STAGES - 1; ++c) load(c);
  const int c0 = warp * 8;  // a warp's columns
  float acc[4] = {};
  for (int c = 0; c < kSteps; ++c) {
    cp_wait<STAGES - 2>();
    __syncthreads();  // the chunk is here, and the stage loaded next has been read
    load(c + STAGES - 1);
    const bf16* wc = sm + (c % STAGES) * kStage;
    const bf16* xh = wc + NCOLS * kPitch;
#pragma unroll
    for (int ks = 0; ks < 8; ++ks) {
      uint32_t ah[4], al[4];
      const int at = (lane & 15) * kPitch + ks * 16 + (lane >> 4) * 8;
      ldmatrix_x4(ah, smem_u32(xh + at));
      ldmatrix_x4(al, smem_u32(xh + MROWS * kPitch + at));
      uint32_t bb[2];  // rows n, 16 bytes at k and k + 8
      asm volatile("ldmatrix.sync.aligned.m8n8.x2.shared.b16 {%0,%1}, [%2];"
                   : "=r"(bb[0]), "=r"(bb[1])
                   : "r"(smem_u32(wc + (c0 + (lane & 7)) * kPitch + ks * 16 + ((lane >> 3) & 1) * 8)));
      mma_bf16_16816(acc, ah, bb);
      mma_bf16_16816(acc, al, bb);
    }
  }
#pragma unroll
  for (int e = 0; e < 2; ++e) {
    const int b = (lane >> 2) + e * 8;
    if (b < rows)
      *reinterpret_cast<uint32_t*>(out + (int64_t)(b0 + b) * out_stride + (int64_t)h * kVal + n0 + c0 + (lane & 3) * 2) =
          pack_bf16(acc[2 * e], acc[2 * e + 1]);
  }
}

// ---- the same on tcgen05: 128-row tiles, thread = row of the accumulator's quadrant

// Stores 32 rows x 64 columns of an accumulator (this warp's lanes, columns from taddr) as bf16
// rows of 128 bytes: through a shared-memory slab, so that a store instruction writes whole lines.
constexpr int kSlabPitch = 144;  // 64 bf16 and 16 bytes against bank conflicts
__device__ __forceinline__ void store_slab(uint32_t taddr, uint8_t* slab, bf16* dst, int64_t pitch, int rows) {
  const int lane = threadIdx.x & 31;
  uint4* mine = reinterpret_cast<uint4*>(slab + lane * kSlabPitch);
#pragma unroll
  for (int half = 0; half < 2; ++half) {
    float v[32];
    tmem_ld32w(taddr + half * 32, v);
#pragma unroll
    for (int q = 0; q < 4; ++q)
      mine[half * 4 + q] = make_uint4(pack_bf16(v[8 * q], v[8 * q + 1]), pack_bf16(v[8 * q + 2], v[8 * q + 3]),
                                      pack_bf16(v[8 * q + 4], v[8 * q + 5]), pack_bf16(v[8 * q + 6], v[8 * q + 7]));
  }
  __syncwarp();
#pragma unroll
  for (int k = 0; k < 8; ++k) {
    const int r = 4 * k + (lane >> 3), seg = lane & 7;
    if (r < rows)
      *reinterpret_cast<uint4*>(dst + r * pitch + seg * 8) =
          *reinterpret_cast<const uint4*>(slab + r * kSlabPitch + seg * 16);
  }
  __syncwarp();
}

struct AbsorbSmem {
  alignas(1024) uint8_t x[2][128 * 128];  // 128 rows x 64 of k
  alignas(1024) uint8_t w[4][128 * 128];  // 128 of k x 64 columns
  uint64_t full, done;
  uint32_t tmem_base;
  volatile int abort_flag;
};

// One CTA per (256 columns, head, 128 rows); w is read MN-major, as it lies in memory.
template <int R>
__global__ void __launch_bounds__(128) latent_absorb_tc_kernel(const __grid_constant__ CUtensorMap q_map,
                                                               const __grid_constant__ CUtensorMap w_map, const bf16* q,
                                                               int64_t q_stride, bf16* qa, int B, int H,
                                                               const int32_t* ctx_lens, int limit, int keys, int ctas,
                                                               int32_t* table, int* err) {
  griddep_launch();
  extern __shared__ __align__(1024) uint8_t smem_raw[];
  AbsorbSmem& s = *reinterpret_cast<AbsorbSmem*>(smem_raw);
  const int n0 = blockIdx.x * 256, h = blockIdx.y, b0 = blockIdx.z * 128;
  const int warp = __shfl_sync(0xffffffffu, threadIdx.x / 32, 0), lane = threadIdx.x % 32;
  if (smem_u32(smem_raw) & 1023) {
    if (threadIdx.x == 0) atomicCAS(err, 0, 83);
    return;
  }
  if (threadIdx.x == 0) {
    s.abort_flag = 0;
    mbar_init(&s.full, 1);
    mbar_init(&s.done, 1);
    fence_barrier_init();
  }
  griddep_wait();  // before the allocation: a CTA of the grid waited for may still need its own
  if (warp == 0) tmem_alloc(&s.tmem_base, 256);
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = __shfl_sync(0xffffffffu, s.tmem_base, 0);
  if (warp == 0 && elect_one()) {
    mbar_arrive_expect_tx(&s.full, 6 * 128 * 128);
#pragma unroll
    for (int c = 0; c < 2; ++c) tma_load_2d(s.x[c], &q_map, &s.full, h * (kNope + kRot) + c * 64, b0);
#pragma unroll
    for (int c = 0; c < 4; ++c) tma_load_2d(s.w[c], &w_map, &s.full, n0 + c * 64, h * (kNope + kVal));
    if (wait_or_abort(s, &s.full, 0, err, 84)) {
      tc_fence_after();
      constexpr uint32_t idesc = idesc_bf16<128, 256>() | kIdescBMn;
      const uint64_t a = smem_desc_sw128(smem_u32(s.x[0])), b = smem_desc_mn_sw128(smem_u32(s.w[0]), 128 * 128, 1024);
#pragma unroll
      for (int kk = 0; kk < 8; ++kk) mma_bf16(tmem, a + (kk >> 2) * 1024 + (kk & 3) * 2, b + kk * 128, idesc, kk > 0);
    }
    mma_commit(&s.done);
  }
  __syncwarp();
  if (blockIdx.x == 0) {  // the rotary part
    copy_rotary<R, 128>(q + (int64_t)b0 * q_stride, q_stride, qa + (int64_t)b0 * H * (R + kRot), B - b0, H, h);
  }
  if (blockIdx.x == gridDim.x - 1 && blockIdx.y == 0 && blockIdx.z == 0)
    write_schedule(ctx_lens, B, limit, keys, ctas, table);
  wait_or_abort(s, &s.done, 0, err, 85);
  __syncwarp();
  tc_fence_after();
  // the operands have been read: their place serves as the slabs
  uint8_t* slab = s.x[0] + warp * 32 * kSlabPitch;
  const int r0 = b0 + warp * 32;
  bf16* dst = qa + ((int64_t)r0 * H + h) * (R + kRot) + n0;
#pragma unroll 1
  for (int c = 0; c < 256; c += 64)
    store_slab(tmem + ((uint32_t)(warp * 32) << 16) + c, slab, dst + c, (int64_t)H * (R + kRot), B - r0);
  tc_fence_before();
  __syncthreads();
  if (warp == 0) {
    tc_fence_after();
    tmem_dealloc(tmem, 256);
  }
}

constexpr int kOutStages = 4;
struct OutSmem {
  alignas(1024) uint8_t st[kOutStages][3][128 * 128];  // hi, lo rows and value weights, 64 of k
  uint64_t full[kOutStages], empty[kOutStages], done;
  uint32_t tmem_base;
  volatile int abort_flag;
};

// out[b, h, n] = sum_r (hi + lo)[b, h, r] w[h, 128 + n, r]: one CTA per (head, 128 rows).
template <int R>
__global__ void __launch_bounds__(128, 1) latent_out_tc_kernel(const __grid_constant__ CUtensorMap hi_map,
                                                            const __grid_constant__ CUtensorMap lo_map,
                                                            const __grid_constant__ CUtensorMap w_map, bf16* out,
                                                            int64_t out_stride, int B, int* err) {
  griddep_launch();
  constexpr int kSteps = R / 64;
  extern __shared__ __align__(1024) uint8_t smem_raw[];
  OutSmem& s = *reinterpret_cast<OutSmem*>(smem_raw);
  const int h = blockIdx.x, b0 = blockIdx.y * 128;
  const int warp = __shfl_sync(0xffffffffu, threadIdx.x / 32, 0);
  if (smem_u32(smem_raw) & 1023) {
    if (threadIdx.x == 0) atomicCAS(err, 0, 83);
    return;
  }
  if (threadIdx.x == 0) {
    s.abort_flag = 0;
    for (int i = 0; i < kOutStages; ++i) {
      mbar_init(&s.full[i], 1);
      mbar_init(&s.empty[i], 1);
    }
    mbar_init(&s.done, 1);
    fence_barrier_init();
  }
  griddep_wait();  // before the allocation: a CTA of the grid waited for may still need its own
  if (warp == 0) tmem_alloc(&s.tmem_base, 128);
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = __shfl_sync(0xffffffffu, s.tmem_base, 0);
  if (warp == 0) {
    if (elect_one()) {
      bool ok = true;
      int k = 0;
      for (; k < kSteps; ++k) {
        const int st = k % kOutStages;
        if (k >= kOutStages && !(ok = wait_or_abort(s, &s.empty[st], (k / kOutStages - 1) & 1, err, 84))) break;
        mbar_arrive_expect_tx(&s.full[st], 3 * 128 * 128);
        tma_load_2d(s.st[st][2], &w_map, &s.full[st], k * 64, h * (kNope + kVal) + kNope);
        tma_load_2d(s.st[st][0], &hi_map, &s.full[st], h * R + k * 64, b0);
        tma_load_2d(s.st[st][1], &lo_map, &s.full[st], h * R + k * 64, b0);
      }
      if (!ok)  // the copies in flight end before the CTA does
        for (int i = max(0, k - kOutStages); i < k; ++i) mbar_wait_sleep(&s.full[i % kOutStages], (i / kOutStages) & 1);
    }
  } else if (warp == 1) {
    if (elect_one()) {
      constexpr uint32_t idesc = idesc_bf16<128, 128>();
      const uint64_t d0 = smem_desc_sw128(smem_u32(s.st[0][0]));
      for (int k = 0; k < kSteps; ++k) {
        const int st = k % kOutStages;
        if (!wait_or_abort(s, &s.full[st], (k / kOutStages) & 1, err, 85)) break;
        tc_fence_after();
        const uint64_t a = d0 + st * 3 * 1024, b = a + 2 * 1024;
#pragma unroll
        for (int kk = 0; kk < 4; ++kk) {
          mma_bf16(tmem, a + kk * 2, b + kk * 2, idesc, k + kk > 0);
          mma_bf16(tmem, a + 1024 + kk * 2, b + kk * 2, idesc, 1);
        }
        mma_commit(&s.empty[st]);
      }
      mma_commit(&s.done);
    }
  }
  __syncwarp();
  wait_or_abort(s, &s.done, 0, err, 86);
  __syncwarp();
  tc_fence_after();
  // every operand has been read: the stages' place serves as the slabs
  uint8_t* slab = s.st[0][0] + warp * 32 * kSlabPitch;
  const int r0 = b0 + warp * 32;
  bf16* dst = out + (int64_t)r0 * out_stride + (int64_t)h * kVal;
#pragma unroll 1
  for (int c = 0; c < 128; c += 64)
    store_slab(tmem + ((uint32_t)(warp * 32) << 16) + c, slab, dst + c, out_stride, B - r0);
  tc_fence_before();
  __syncthreads();
  if (warp == 0) {
    tc_fence_after();
    tmem_dealloc(tmem, 128);
  }
}

// Heads are cut into equal tiles of at most 64, or 128 where CTA pairs do the attention; each gets an
// equal share of the SMs (or pairs), and no more CTAs than B contexts of max_ctx tokens have tiles.
struct Plan {
  bool pairs;
  int keys, head_tiles, heads_per_cta, ctas;
  Plan(int B, int H, int R, int max_ctx, int num_sms)
      : pairs(R == 512 && H > kPairHeads && num_sms >= 2),
        keys(pairs ? kPairKeys : kKeys),
        head_tiles(pairs ? (H + 127) / 128 : (H + 63) / 64),
        heads_per_cta((H + head_tiles - 1) / head_tiles) {
    const int64_t tiles = (int64_t)B * std::max(1, max_ctx / keys + (max_ctx % keys != 0));
    ctas = (int)std::max<int64_t>(1, std::min<int64_t>(num_sms / (pairs ? 2 : 1) / head_tiles, tiles));
  }
};

// Workspace: qa, the schedule, the joined rows' low halves, the pieces' (m, l) and o (each part 128-byte aligned).
struct Layout {
  size_t table, low, ml, part, bytes;
  Layout(int B, int H, int R, const Plan& p) {
    const size_t slots = (size_t)p.head_tiles * (B + p.ctas) * p.heads_per_cta;
    auto up = [](size_t n) { return (n + 127) / 128 * 128; };
    table = up((size_t)B * H * (R + kRot) * 2);
    low = table + up((size_t)table_ints(B) * 4);
    ml = low + up((size_t)B * H * R * 2);
    part = ml + up(slots * 8);
    bytes = part + slots * R * 4;
  }
};

template <class Kernel, class... Args>
void run_smem(Kernel kern, std::atomic<uint64_t>& attr_devs, dim3 grid, size_t smem, cudaStream_t st, Args... args) {
  ensure_smem_attr(attr_devs, kern, smem);
  launch_k(kern, grid, 128, smem, st, args...);
  KAPSL_LAUNCH_CHECK();
}

template <int R, int NT>
void run_attn(const LatentDecode& a, const Plan& p, const bf16* qa, float* part_o, float2* part_ml,
              const int32_t* table, cudaStream_t st) {
  using S = Shape<R, NT>;
  auto kern = latent_attn_kernel<R, NT>;
  constexpr size_t smem = sizeof(DecodeSmem<R, NT>);
  static_assert(smem <= 232448, "shared memory of one CTA");
  static std::atomic<uint64_t> attr_devs{0};
  ensure_smem_attr(attr_devs, kern, smem);
  const CUtensorMap tq = make_tmap_2d_bf16(qa, (uint64_t)a.B * a.H, S::W, S::W, NT, 64, true);
  const CUtensorMap tc = make_tmap_2d_bf16(a.cache, (uint64_t)a.num_blocks * a.page, S::W, S::W, a.page, 64, true);
  launch_k(kern, dim3(p.ctas * p.head_tiles), kAttnThreads<R>, smem, st, tq, tc, a.num_blocks, a.page, a.block_tables,
           a.max_blocks, a.table_rows, a.num_tables, a.ctx_lens, table, part_o, part_ml, a.B, a.H, p.heads_per_cta,
           p.head_tiles, a.scale * kLog2e, a.err);
  KAPSL_LAUNCH_CHECK();
}

void run_pairs(const LatentDecode& a, const Plan& p, const bf16* qa, float* part_o, float2* part_ml,
               const int32_t* table, cudaStream_t st) {
  static_assert(sizeof(PairSmem) <= 232448, "shared memory of one CTA");
  static std::atomic<uint64_t> attr_devs{0};
  ensure_smem_attr(attr_devs, latent_attn_pair_kernel, sizeof(PairSmem));
  const int W = a.R + kRot;
  const CUtensorMap tq = make_tmap_2d_bf16(qa, (uint64_t)a.B * a.H, W, W, 128, 64, true);
  const CUtensorMap tc = make_tmap_2d_bf16(a.cache, (uint64_t)a.num_blocks * a.page, W, W, a.page, 64, true);
  launch_k(latent_attn_pair_kernel, dim3(2 * p.ctas * p.head_tiles), kPairThreads, sizeof(PairSmem), st, tq, tc, qa,
           static_cast<const bf16*>(a.cache), a.num_blocks, a.page, a.block_tables, a.max_blocks, a.table_rows,
           a.num_tables, a.ctx_lens, table, part_o, part_ml, a.B, a.H, p.heads_per_cta, p.head_tiles,
           a.scale * kLog2e, a.err);
  KAPSL_LAUNCH_CHECK();
}

template <int R>
void run(const LatentDecode& a, cudaStream_t st) {
  const Plan p(a.B, a.H, R, a.max_ctx, a.num_sms);
  const Layout l(a.B, a.H, R, p);
  uint8_t* ws = static_cast<uint8_t*>(a.workspace);
  bf16* qa = reinterpret_cast<bf16*>(ws);
  int32_t* table = reinterpret_cast<int32_t*>(ws + l.table);
  float2* part_ml = reinterpret_cast<float2*>(ws + l.ml);
  float* part_o = reinterpret_cast<float*>(ws + l.part);
  const int limit = a.max_blocks * a.page;
  // Tiles of 16 rows while their CTAs are few (a whole call of 33 rows x 20 heads 27 us, with the 128-row
  // tiles 32; of 64 rows x 128 heads 118 and 101 us).
  const bool small = (a.B + 15) / 16 * a.H <= 256;
  const unsigned tiles16 = (a.B + 15) / 16;
  const CUtensorMap tw = make_tmap_2d_bf16(a.w, (uint64_t)a.H * (kNope + kVal), R, R, 128, 64, true);
  if (small) {
    launch_k(latent_absorb_kernel<R>, dim3(R / 64, a.H, tiles16), 128, 0, st, a.q, a.q_stride, a.w, qa, a.B, a.H,
             a.ctx_lens, limit, p.keys, p.ctas, table);
    KAPSL_LAUNCH_CHECK();
  } else {
    const CUtensorMap tq = make_tmap_2d_bf16(a.q, a.B, (uint64_t)a.H * (kNope + kRot), a.q_stride, 128, 64, true);
    static std::atomic<uint64_t> devs{0};
    run_smem(latent_absorb_tc_kernel<R>, devs, dim3(R / 256, a.H, (a.B + 127) / 128), sizeof(AbsorbSmem), st, tq, tw,
             a.q, a.q_stride, qa, a.B, a.H, a.ctx_lens, limit, p.keys, p.ctas, table, a.err);
  }
  if (p.pairs) {
    run_pairs(a, p, qa, part_o, part_ml, table, st);
  } else if (p.heads_per_cta <= 16) {
    run_attn<R, 16>(a, p, qa, part_o, part_ml, table, st);
  } else if (p.heads_per_cta <= 32) {
    run_attn<R, 32>(a, p, qa, part_o, part_ml, table, st);
  } else {
    run_attn<R, 64>(a, p, qa, part_o, part_ml, table, st);
  }
  // qa has been read: the high halves take its place
  bf16* lo = reinterpret_cast<bf16*>(ws + l.low);
  const int64_t rows = (int64_t)a.B * a.H, per = 1024 / R * (small ? 1 : 2);
  launch_k(small ? latent_join_kernel<R, 8, 1> : latent_join_kernel<R, 2, 2>, dim3((unsigned)((rows + per - 1) / per)),
           128, 0, st, part_o, part_ml, table, qa, lo, a.B, a.H, p.heads_per_cta, p.ctas);
  KAPSL_LAUNCH_CHECK();
  static std::atomic<uint64_t> devs{0}, devs_tc{0};
  if (small) {
    constexpr size_t smem = (size_t)(R / 128 + 1) * (32 + 2 * 16) * 136 * 2;
    run_smem(latent_out_kernel<R>, devs, dim3(kVal / 32, a.H, tiles16), smem, st, qa, lo, a.w, a.out, a.out_stride, a.B, a.H);
  } else {
    const uint64_t width = (uint64_t)a.H * R;
    const CUtensorMap th = make_tmap_2d_bf16(qa, a.B, width, width, 128, 64, true);
    const CUtensorMap tl = make_tmap_2d_bf16(lo, a.B, width, width, 128, 64, true);
    run_smem(latent_out_tc_kernel<R>, devs_tc, dim3(a.H, (a.B + 127) / 128), sizeof(OutSmem), st, th, tl, tw, a.out,
             a.out_stride, a.B, a.err);
  }
  note_launch(4);
}

}  // namespace

size_t latent_decode_workspace_bytes(int B, int H, int R, int max_ctx, int num_sms) {
  return Layout(B, H, R, Plan(B, H, R, max_ctx, num_sms)).bytes;
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
