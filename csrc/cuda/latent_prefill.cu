// Expanded latent attention: a chunk of new tokens over a paged latent cache.
//
// The context rows [c (R) | k_r (64)] are gathered out of the pages, one GEMM expands
// them to every head's key and value rows (kv = c w_h^T, [128 | 128] a head), and the
// attention runs with keys [k_h (128) | k_r (64, shared)] and values of 128:
//   out_i = sum_j softmax_j(scale q_i . k_j) v_j  over j <= position of i.
#include <algorithm>

#include "common.cuh"
#include "kernels.h"

namespace kapsl {

using bf16 = __nv_bfloat16;

namespace {

constexpr int kNope = 128, kRot = 64, kVal = 128;
constexpr float kLog2e = 1.4426950408889634f;

// One warp per output row; rows between sequences (padding to 16) become zero.
__global__ void __launch_bounds__(256) latent_gather_kernel(const bf16* __restrict__ cache, int64_t num_blocks,
                                                            int page, int W, const int32_t* __restrict__ seq_info,
                                                            int nseq, const int32_t* __restrict__ block_tables,
                                                            int max_blocks, bf16* __restrict__ rows, int64_t total,
                                                            int* __restrict__ err) {
  griddep_entry();
  const int64_t row = (int64_t)blockIdx.x * 8 + (threadIdx.x >> 5);
  const int lane = threadIdx.x & 31;
  if (row >= total) return;
  int lo = 0, hi = nseq - 1;  // last sequence whose first row is <= row
  while (lo < hi) {
    const int mid = (lo + hi + 1) / 2;
    if (seq_info[mid * 5 + 4] <= row) lo = mid;
    else hi = mid - 1;
  }
  const int j = (int)(row - seq_info[lo * 5 + 4]);
  const uint4* src = nullptr;
  if (j < seq_info[lo * 5 + 2]) {
    const int blk = block_tables[(int64_t)seq_info[lo * 5 + 3] * max_blocks + j / page];
    if (blk >= 0 && blk < num_blocks) {
      src = reinterpret_cast<const uint4*>(cache + ((int64_t)blk * page + j % page) * W);
    } else if (lane == 0) {
      atomicCAS(err, 0, 82);
    }
  }
  uint4* dst = reinterpret_cast<uint4*>(rows + row * W);
  for (int c = lane; c < W / 8; c += 32) dst[c] = src ? src[c] : make_uint4(0, 0, 0, 0);
}

// One warp per (token, head), keys one at a time.
__global__ void __launch_bounds__(256) latent_prefill_kernel(const LatentPrefill a) {
  griddep_entry();
  const int seq = a.work[2 * blockIdx.x], t0 = a.work[2 * blockIdx.x + 1], h = blockIdx.y;
  const int32_t* si = a.seq_info + 5 * seq;
  const int row0 = si[0], n = si[1], ctx = si[2], kv0 = si[4];
  const int lane = threadIdx.x & 31;
  const int W = a.R + kRot;
  for (int t = t0 + (threadIdx.x >> 5); t < min(n, t0 + 256); t += 8) {
    const __nv_bfloat162* q = reinterpret_cast<const __nv_bfloat162*>(a.q + (int64_t)(row0 + t) * a.q_stride + h * 192);
    const float2 q0 = __bfloat1622float2(q[lane]), q1 = __bfloat1622float2(q[32 + lane]),
                 q2 = __bfloat1622float2(q[64 + lane]);
    float2 o0 = make_float2(0.f, 0.f), o1 = o0;
    float m = -INFINITY, l = 0.f;
    const int last = ctx - n + t;
    for (int j = 0; j <= last; ++j) {
      const __nv_bfloat162* kv = reinterpret_cast<const __nv_bfloat162*>(a.kv + (int64_t)(kv0 + j) * a.kv_stride + h * 256);
      const __nv_bfloat162* kr = reinterpret_cast<const __nv_bfloat162*>(a.rows + (int64_t)(kv0 + j) * W + a.R);
      const float2 k0 = __bfloat1622float2(kv[lane]), k1 = __bfloat1622float2(kv[32 + lane]),
                   k2 = __bfloat1622float2(kr[lane]);
      const float s = a.scale * kLog2e *
                      warp_sum(q0.x * k0.x + q0.y * k0.y + q1.x * k1.x + q1.y * k1.y + q2.x * k2.x + q2.y * k2.y);
      const float2 v0 = __bfloat1622float2(kv[64 + lane]), v1 = __bfloat1622float2(kv[96 + lane]);
      const float mn = fmaxf(m, s);
      const float f = m == -INFINITY ? 0.f : exp2f(m - mn), p = mn == -INFINITY ? 0.f : exp2f(s - mn);
      m = mn;
      l = l * f + p;
      o0 = make_float2(o0.x * f + p * v0.x, o0.y * f + p * v0.y);
      o1 = make_float2(o1.x * f + p * v1.x, o1.y * f + p * v1.y);
    }
    const float inv = l > 0.f ? 1.f / l : 0.f;
    __nv_bfloat162* dst = reinterpret_cast<__nv_bfloat162*>(a.out + (int64_t)(row0 + t) * a.out_stride + h * kVal);
    dst[lane] = __floats2bfloat162_rn(o0.x * inv, o0.y * inv);
    dst[32 + lane] = __floats2bfloat162_rn(o1.x * inv, o1.y * inv);
  }
}

}  // namespace

void launch_latent_gather(const bf16* cache, int64_t num_blocks, int page, int R, const int32_t* seq_info, int nseq,
                          const int32_t* block_tables, int max_blocks, bf16* rows, int64_t total, int* err,
                          cudaStream_t st) {
  if (total == 0 || nseq == 0) return;
  launch_k(latent_gather_kernel, dim3((unsigned)((total + 7) / 8)), 256, 0, st, cache, num_blocks, page, R + kRot,
           seq_info, nseq, block_tables, max_blocks, rows, total, err);
  KAPSL_LAUNCH_CHECK();
  note_launch();
}

void launch_latent_prefill(const LatentPrefill& a, cudaStream_t st) {
  if (a.nwork == 0 || a.heads == 0) return;
  launch_k(latent_prefill_kernel, dim3(a.nwork, a.heads), 256, 0, st, a);
  KAPSL_LAUNCH_CHECK();
  note_launch();
}

}  // namespace kapsl
