// Absorbed latent attention for single tokens over a paged latent cache.
//
// A cache row is [c (R) | k_r (64)], shared by every head.  Head h has the key
// expansion K_h = w[h, :128] and the value expansion V_h = w[h, 128:], both [128, R].
// With the key expansion moved to the query's side,
//   qa_h = [K_h^T q_h[:128] | q_h[128:]],   s_j = scale * qa_h . row_j,
//   o_h = sum_j softmax(s)_j c_j,           out_h = V_h o_h,
// so the cache is read once for all heads and nothing is expanded per token.
#include <algorithm>

#include "common.cuh"
#include "kernels.h"

namespace kapsl {

using bf16 = __nv_bfloat16;

namespace {

constexpr int kNope = 128, kRot = 64, kVal = 128;
constexpr float kLog2e = 1.4426950408889634f;

// qa[b, h, :] (bf16: the tensor cores' operand type)
template <int R>
__global__ void __launch_bounds__(128) latent_absorb_kernel(const bf16* __restrict__ q, int64_t q_stride,
                                                            const bf16* __restrict__ w, bf16* __restrict__ qa,
                                                            int H) {
  griddep_entry();
  const int h = blockIdx.x, b = blockIdx.y;
  const bf16* qr = q + (int64_t)b * q_stride + (int64_t)h * (kNope + kRot);
  const bf16* wk = w + (int64_t)h * (kNope + kVal) * R;
  bf16* dst = qa + ((int64_t)b * H + h) * (R + kRot);
  for (int r = threadIdx.x; r < R; r += blockDim.x) {
    float acc = 0.f;
    for (int d = 0; d < kNope; ++d) acc += __bfloat162float(qr[d]) * __bfloat162float(wk[(int64_t)d * R + r]);
    dst[r] = __float2bfloat16(acc);
  }
  if (threadIdx.x < kRot) dst[R + threadIdx.x] = qr[kNope + threadIdx.x];
}

// One warp per head, 8 heads a CTA; each lane holds (R + 64) / 32 query values and R / 32
// accumulators, keys are taken one at a time.
template <int R>
__global__ void __launch_bounds__(256) latent_attn_kernel(const bf16* __restrict__ qa,
                                                          const bf16* __restrict__ cache, int64_t num_blocks,
                                                          int page, const int32_t* __restrict__ block_tables,
                                                          int max_blocks, const int32_t* __restrict__ ctx_lens,
                                                          float* __restrict__ part_o, float* __restrict__ part_lse,
                                                          int H, int nsplit, float scale_log2,
                                                          int* __restrict__ err) {
  griddep_entry();
  constexpr int W = R + kRot, NQ = W / 64, NO = R / 64;  // bf16 pairs a lane
  const int split = blockIdx.x, b = blockIdx.z, lane = threadIdx.x & 31;
  const int h = blockIdx.y * 8 + (threadIdx.x >> 5);
  if (h >= H) return;
  const int ctx = min(ctx_lens[b], max_blocks * page);
  const int per = ((ctx + nsplit - 1) / nsplit + 15) / 16 * 16;
  const int j0 = split * per, j1 = min(ctx, j0 + per);
  float2 qv[NQ], o[NO];
  const __nv_bfloat162* qr = reinterpret_cast<const __nv_bfloat162*>(qa + ((int64_t)b * H + h) * W);
#pragma unroll
  for (int i = 0; i < NQ; ++i) qv[i] = __bfloat1622float2(qr[i * 32 + lane]);
#pragma unroll
  for (int i = 0; i < NO; ++i) o[i] = make_float2(0.f, 0.f);
  float m = -INFINITY, l = 0.f;
  for (int j = j0; j < j1; ++j) {
    const int blk = block_tables[(int64_t)b * max_blocks + j / page];
    if (blk < 0 || blk >= num_blocks) {
      if (lane == 0) atomicCAS(err, 0, 82);
      continue;
    }
    const __nv_bfloat162* row =
        reinterpret_cast<const __nv_bfloat162*>(cache + ((int64_t)blk * page + j % page) * W);
    float2 kv[NQ];
    float s = 0.f;
#pragma unroll
    for (int i = 0; i < NQ; ++i) {
      kv[i] = __bfloat1622float2(row[i * 32 + lane]);
      s += kv[i].x * qv[i].x + kv[i].y * qv[i].y;
    }
    s = warp_sum(s) * scale_log2;
    const float mn = fmaxf(m, s);
    const float f = m == -INFINITY ? 0.f : exp2f(m - mn), p = mn == -INFINITY ? 0.f : exp2f(s - mn);
    m = mn;
    l = l * f + p;
#pragma unroll
    for (int i = 0; i < NO; ++i) o[i] = make_float2(o[i].x * f + p * kv[i].x, o[i].y * f + p * kv[i].y);
  }
  const int64_t pi = ((int64_t)b * H + h) * nsplit + split;
  const float inv = l > 0.f ? 1.f / l : 0.f;
#pragma unroll
  for (int i = 0; i < NO; ++i)
    reinterpret_cast<float2*>(part_o + pi * R)[i * 32 + lane] = make_float2(o[i].x * inv, o[i].y * inv);
  if (lane == 0) part_lse[pi] = l > 0.f ? m + log2f(l) : -INFINITY;
}

template <int R>
__global__ void __launch_bounds__(128) latent_combine_kernel(const float* __restrict__ part_o,
                                                             const float* __restrict__ part_lse,
                                                             const bf16* __restrict__ w, bf16* __restrict__ out,
                                                             int64_t out_stride, int H, int nsplit) {
  griddep_entry();
  const int h = blockIdx.x, b = blockIdx.y;
  __shared__ float o[R];
  const int64_t base = ((int64_t)b * H + h) * nsplit;
  float M = -INFINITY;
  for (int s = 0; s < nsplit; ++s) M = fmaxf(M, part_lse[base + s]);
  for (int r = threadIdx.x; r < R; r += blockDim.x) {
    float L = 0.f, acc = 0.f;
    for (int s = 0; s < nsplit && M != -INFINITY; ++s) {
      const float f = exp2f(part_lse[base + s] - M);
      L += f;
      acc += f * part_o[(base + s) * R + r];
    }
    o[r] = L > 0.f ? acc / L : 0.f;
  }
  __syncthreads();
  const bf16* wv = w + ((int64_t)h * (kNope + kVal) + kNope + threadIdx.x) * R;
  float acc = 0.f;
  for (int r = 0; r < R; ++r) acc += o[r] * __bfloat162float(wv[r]);
  out[(int64_t)b * out_stride + h * kVal + threadIdx.x] = __float2bfloat16(acc);
}

template <int R>
void run(const LatentDecode& a, cudaStream_t st) {
  bf16* qa = static_cast<bf16*>(a.workspace);
  float* part_o = reinterpret_cast<float*>(qa + (int64_t)a.B * a.H * (R + kRot));
  float* part_lse = part_o + (int64_t)a.B * a.H * a.nsplit * R;
  launch_k(latent_absorb_kernel<R>, dim3(a.H, a.B), 128, 0, st, a.q, a.q_stride, a.w, qa, a.H);
  KAPSL_LAUNCH_CHECK();
  launch_k(latent_attn_kernel<R>, dim3(a.nsplit, (a.H + 7) / 8, a.B), 256, 0, st, qa, a.cache, a.num_blocks, a.page,
           a.block_tables, a.max_blocks, a.ctx_lens, part_o, part_lse, a.H, a.nsplit, a.scale * kLog2e, a.err);
  KAPSL_LAUNCH_CHECK();
  launch_k(latent_combine_kernel<R>, dim3(a.H, a.B), 128, 0, st, part_o, part_lse, a.w, a.out, a.out_stride, a.H,
           a.nsplit);
  KAPSL_LAUNCH_CHECK();
  note_launch(3);
}

}  // namespace

int latent_decode_num_splits(int B, int H, int R, int max_ctx, int num_sms) {
  const int ctas = std::max(1, B * ((H + 7) / 8));
  int s = (2 * num_sms + ctas - 1) / ctas;
  s = std::min(s, std::max(1, (max_ctx + 255) / 256));
  return std::max(1, std::min(s, 64));
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
