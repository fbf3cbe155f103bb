// Rotary positions for strided heads, and the cache write of latent attention.
//
// rope: y = x with the dims [offset, offset + P) of every head rotated by the
// token's angles, P = the width of the cos | sin table.  Pairs are (i, i + P/2)
// (half layout) or (2i, 2i + 1) (interleaved):
//   y_a = x_a cos_i - x_b sin_i,   y_b = x_b cos_i + x_a sin_i   (fp32, one rounding)
//
// rope_latent_write: one token's compressed KV row kv = [c (R) | k (P)] becomes the
// cache row [c / sqrt(mean(c^2) + eps) * w | rope(k)], and the query heads' rotary
// part is rotated in the same launch.
#include <cuda_fp16.h>

#include <algorithm>

#include "common.cuh"
#include "kernels.h"

namespace kapsl {

using bf16 = __nv_bfloat16;

namespace {

template <class T>
__device__ __forceinline__ float to_f(T v);
template <>
__device__ __forceinline__ float to_f<float>(float v) { return v; }
template <>
__device__ __forceinline__ float to_f<bf16>(bf16 v) { return __bfloat162float(v); }
template <>
__device__ __forceinline__ float to_f<__half>(__half v) { return __half2float(v); }
template <class T>
__device__ __forceinline__ T from_f(float v);
template <>
__device__ __forceinline__ float from_f<float>(float v) { return v; }
template <>
__device__ __forceinline__ bf16 from_f<bf16>(float v) { return __float2bfloat16(v); }
template <>
__device__ __forceinline__ __half from_f<__half>(float v) { return __float2half(v); }

// N elements moved at once; the one-pair units of the narrow path are only element-aligned.
template <class T, int N>
struct alignas(N == 2 ? sizeof(T) : sizeof(T) * N) Vec {
  T v[N];
};

// N consecutive table values; the table's rows are 16-byte aligned when N > 1.
template <int N>
__device__ __forceinline__ void load_cs(const float* p, float (&o)[N]) {
  if constexpr (N % 4 == 0) {
#pragma unroll
    for (int i = 0; i < N; i += 4) {
      const float4 f = *reinterpret_cast<const float4*>(p + i);
      o[i] = f.x, o[i + 1] = f.y, o[i + 2] = f.z, o[i + 3] = f.w;
    }
  } else if constexpr (N % 2 == 0) {
#pragma unroll
    for (int i = 0; i < N; i += 2) {
      const float2 f = *reinterpret_cast<const float2*>(p + i);
      o[i] = f.x, o[i + 1] = f.y;
    }
  } else {
#pragma unroll
    for (int i = 0; i < N; ++i) o[i] = p[i];
  }
}

// The angles of one unit of a head: N elements (interleaved: N/2 pairs), or N pairs (a[k], b[k])
// in the half layout; `i` is the unit's first angle index.
template <int N, bool IL>
struct Angles {
  static constexpr int M = IL ? N / 2 : N;
  float c[M], s[M];
  __device__ __forceinline__ Angles(const float* cs, int half, int i) {
    load_cs<M>(cs + i, c);
    load_cs<M>(cs + half + i, s);
  }
  template <class T>
  __device__ __forceinline__ void rotate(Vec<T, N>& a, Vec<T, N>& b) const {
#pragma unroll
    for (int k = 0; k < M; ++k) {
      T& p = IL ? a.v[2 * k] : a.v[k];
      T& q = IL ? a.v[(2 * k + 1) % N] : b.v[k % N];
      const float x = to_f(p), y = to_f(q);
      p = from_f<T>(x * c[k] - y * s[k]);
      q = from_f<T>(y * c[k] + x * s[k]);
    }
  }
};

// One thread column (threadIdx.x) per unit of a head, one thread row per (token, head)
// row, several rows a thread so that several independent 16-byte loads are in
// flight.  Units [0, nrot) rotate, the rest (out of place only) copy elements of the
// dims outside the rotated part (one element on the narrow path).
template <class T, bool IL>
constexpr int kRopeRows = sizeof(T) == 2 && !IL ? 2 : 4;

template <class T, int N, bool IL>
__device__ __forceinline__ void rope_rows(int64_t block, const T* x, int64_t xs_t, int64_t xs_h, T* y, int64_t ys_t,
                                          int64_t ys_h, const int32_t* positions, const float* __restrict__ cos_sin,
                                          int max_pos, int64_t rows, int H, int D, int P, int offset, bool in_place,
                                          int* err) {
  constexpr int kRows = kRopeRows<T, IL>;
  const int half = P >> 1;
  const int nrot = IL ? P / N : half / N;
  constexpr int NC = sizeof(T) * N == 16 ? N : 1;  // elements a copying unit moves
  const int nunit = nrot + (in_place ? 0 : (D - P) / NC);
  const int64_t r0 = block * blockDim.y * kRows + threadIdx.y;
  for (int u = threadIdx.x; u < nunit; u += blockDim.x) {
    const bool rot = u < nrot;
    // element offsets inside the head
    const int c = (u - nrot) * NC;
    const int e0 = rot ? offset + u * N : (c < offset ? c : c + P);
    Vec<T, N> a[kRows], b[kRows];
    int pos[kRows];
    T* dst[kRows];
#pragma unroll
    for (int k = 0; k < kRows; ++k) {
      const int64_t r = r0 + (int64_t)k * blockDim.y;
      dst[k] = nullptr;
      if (r < rows) {
        const int64_t t = r / H;
        const int h = (int)(r - t * H);
        const T* src = x + t * xs_t + h * xs_h + e0;
        dst[k] = y + t * ys_t + h * ys_h + e0;
        if (rot || NC == N) {
          a[k] = *reinterpret_cast<const Vec<T, N>*>(src);
        } else {
          a[k].v[0] = *src;
        }
        if (!IL && rot) b[k] = *reinterpret_cast<const Vec<T, N>*>(src + half);
        if (rot) pos[k] = positions[t];
      }
    }
#pragma unroll
    for (int k = 0; k < kRows; ++k) {
      if (dst[k] == nullptr) continue;
      if (rot) {
        if (pos[k] >= 0 && pos[k] < max_pos) {
          Angles<N, IL>(cos_sin + (int64_t)pos[k] * P, half, IL ? u * N / 2 : u * N).rotate(a[k], b[k]);
        } else {
          atomicCAS(err, 0, 80);  // no such table row: the head keeps its values
        }
        if (!IL) *reinterpret_cast<Vec<T, N>*>(dst[k] + half) = b[k];
      }
      if (rot || NC == N) {
        *reinterpret_cast<Vec<T, N>*>(dst[k]) = a[k];
      } else {
        *dst[k] = a[k].v[0];
      }
    }
  }
}

template <class T, int N, bool IL>
__global__ void __launch_bounds__(256) rope_kernel(const T* x, int64_t xs_t, int64_t xs_h, T* y, int64_t ys_t,
                                                   int64_t ys_h, const int32_t* positions,
                                                   const float* __restrict__ cos_sin, int max_pos, int64_t rows, int H,
                                                   int D, int P, int offset, bool in_place, int* err) {
  griddep_entry();
  rope_rows<T, N, IL>(blockIdx.x, x, xs_t, xs_h, y, ys_t, ys_h, positions, cos_sin, max_pos, rows, H, D, P, offset,
                      in_place, err);
}

template <class T, int N, bool IL>
void rope_launch(const RopeArgs& a, cudaStream_t st) {
  const int nrot = IL ? a.P / N : a.P / 2 / N;
  constexpr int NC = sizeof(T) * N == 16 ? N : 1;
  const int nunit = std::max(1, nrot + (a.in_place ? 0 : (a.D - a.P) / NC));
  const int bx = std::min(nunit, 256);
  const int by = std::max(1, 256 / bx);
  const int64_t rows = a.T * a.H;
  const int64_t grid = (rows + (int64_t)by * kRopeRows<T, IL> - 1) / ((int64_t)by * kRopeRows<T, IL>);
  if (grid > 0x7fffffff) throw std::runtime_error("rope: too many rows");
  launch_k(rope_kernel<T, N, IL>, dim3((unsigned)grid), dim3(bx, by), 0, st, static_cast<const T*>(a.x), a.xs_t,
           a.xs_h, static_cast<T*>(a.y), a.ys_t, a.ys_h, a.positions, a.cos_sin, a.max_pos, rows, a.H, a.D, a.P,
           a.offset, a.in_place, a.err);
  KAPSL_LAUNCH_CHECK();
  note_launch();
}

template <class T>
void rope_dispatch(const RopeArgs& a, cudaStream_t st) {
  // 16-byte units where every stride, offset and base address allows them, else the
  // smallest unit (one pair).
  constexpr int N = 16 / sizeof(T);
  const int64_t unit = a.interleaved ? a.P : a.P / 2;
  const bool wide = unit % N == 0 && a.offset % N == 0 && (a.in_place || a.D % N == 0) && a.xs_t % N == 0 &&
                    a.xs_h % N == 0 && a.ys_t % N == 0 && a.ys_h % N == 0 &&
                    (reinterpret_cast<uintptr_t>(a.x) & 15) == 0 && (reinterpret_cast<uintptr_t>(a.y) & 15) == 0 &&
                    (reinterpret_cast<uintptr_t>(a.cos_sin) & 15) == 0 && a.P % 4 == 0 && (a.P / 2) % 4 == 0;
  if (wide) {
    a.interleaved ? rope_launch<T, N, true>(a, st) : rope_launch<T, N, false>(a, st);
  } else if (a.interleaved) {
    rope_launch<T, 2, true>(a, st);
  } else {
    rope_launch<T, 1, false>(a, st);
  }
}

// ------------------------------------------------------- latent cache write
// The first blocks take a token a warp: the latent is normalised (R / 256 16-byte vectors a
// lane, sum of squares by shuffles) and the shared key rotated.  The others take a token each
// and rotate its query heads: a thread keeps the angles of its unit for all its heads, two
// heads' loads in flight, asked for beside the angles (67 us where they waited for them).  8191 tokens
// x 128 heads, out of place: 60 us, 4.8 TB/s of the bytes it needs; 6 % less with contiguous heads
// instead of every third 128 bytes of q, so most of what is above DRAM's 44 us is a block's chain
// of position, then data and angles.  rope_kernel's row order, which loads the angles again for
// every head, took 70-87 us.
template <int R, bool IL>
__global__ void __launch_bounds__(256) rope_latent_write_kernel(
    const bf16* q, int64_t qs_t, int64_t qs_h, bf16* qo, int64_t qo_t, int64_t qo_h, const bf16* kv, int64_t kv_stride,
    const int32_t* positions, const int64_t* slots, const float* __restrict__ cos_sin, int max_pos,
    const bf16* w, float eps, bf16* cache, int64_t num_slots, int T, int H, int latent_blocks, int* err) {
  griddep_entry();
  constexpr int P = 64, N = 8, half = P / 2;
  constexpr int NU = IL ? P / N : half / N;  // rotating units a head
  if (blockIdx.x >= latent_blocks) {
    const int t = blockIdx.x - latent_blocks, u = threadIdx.x % NU, step = blockDim.x / NU;
    const int pos = positions[t];
    const bool ok = pos >= 0 && pos < max_pos;
    const bf16* src = q + t * qs_t + (int64_t)u * N;
    bf16* dst = qo + t * qo_t + (int64_t)u * N;
    if (!ok) {  // nothing is read from the table, which may have no rows at all
      if (src != dst)
        for (int h = threadIdx.x / NU; h < H; h += step) {
          *reinterpret_cast<Vec<bf16, N>*>(dst + h * qo_h) = *reinterpret_cast<const Vec<bf16, N>*>(src + h * qs_h);
          if (!IL)
            *reinterpret_cast<Vec<bf16, N>*>(dst + h * qo_h + half) =
                *reinterpret_cast<const Vec<bf16, N>*>(src + h * qs_h + half);
        }
      return;
    }
    const Angles<N, IL> angles(cos_sin + (int64_t)pos * P, half, IL ? u * N / 2 : u * N);
    for (int h = threadIdx.x / NU; h < H; h += 2 * step) {
      Vec<bf16, N> a[2], b[2];
#pragma unroll
      for (int k = 0; k < 2; ++k) {
        if (h + k * step < H) {
          const bf16* at = src + (h + k * step) * qs_h;
          a[k] = *reinterpret_cast<const Vec<bf16, N>*>(at);
          if (!IL) b[k] = *reinterpret_cast<const Vec<bf16, N>*>(at + half);
        }
      }
#pragma unroll
      for (int k = 0; k < 2; ++k) {
        if (h + k * step < H) {
          bf16* at = dst + (h + k * step) * qo_h;
          angles.rotate(a[k], b[k]);
          *reinterpret_cast<Vec<bf16, N>*>(at) = a[k];
          if (!IL) *reinterpret_cast<Vec<bf16, N>*>(at + half) = b[k];
        }
      }
    }
    return;
  }
  const int lane = threadIdx.x & 31, t = blockIdx.x * (blockDim.x >> 5) + (threadIdx.x >> 5);
  if (t >= T) return;
  const int pos = positions[t];
  const int64_t slot = slots[t];
  const bool ok = pos >= 0 && pos < max_pos;
  if (slot < 0) return;  // a padded row, whatever its position
  if (!ok && lane == 0) atomicCAS(err, 0, 80);
  if (slot >= num_slots) {
    if (lane == 0) atomicCAS(err, 0, 81);
    return;
  }
  const bf16* src = kv + (int64_t)t * kv_stride;
  bf16* dst = cache + slot * (R + P);
  Vec<bf16, N> v[R / 256], ww[R / 256];
  Vec<bf16, N> a, b;
#pragma unroll
  for (int i = 0; i < R / 256; ++i) v[i] = *reinterpret_cast<const Vec<bf16, N>*>(src + (i * 32 + lane) * N);
#pragma unroll
  for (int i = 0; i < R / 256; ++i) ww[i] = *reinterpret_cast<const Vec<bf16, N>*>(w + (i * 32 + lane) * N);
  if (lane < NU) {
    a = *reinterpret_cast<const Vec<bf16, N>*>(src + R + lane * N);
    if (!IL) b = *reinterpret_cast<const Vec<bf16, N>*>(src + R + half + lane * N);
  }
  float ss = 0.f;
#pragma unroll
  for (int i = 0; i < R / 256; ++i)
#pragma unroll
    for (int k = 0; k < N; ++k) ss += to_f(v[i].v[k]) * to_f(v[i].v[k]);
  const float inv = rsqrtf(warp_sum(ss) / (float)R + eps);
#pragma unroll
  for (int i = 0; i < R / 256; ++i) {
#pragma unroll
    for (int k = 0; k < N; ++k) v[i].v[k] = from_f<bf16>(to_f(v[i].v[k]) * inv * to_f(ww[i].v[k]));
    *reinterpret_cast<Vec<bf16, N>*>(dst + (i * 32 + lane) * N) = v[i];
  }
  if (lane < NU) {
    if (ok) Angles<N, IL>(cos_sin + (int64_t)pos * P, half, IL ? lane * N / 2 : lane * N).rotate(a, b);
    *reinterpret_cast<Vec<bf16, N>*>(dst + R + lane * N) = a;
    if (!IL) *reinterpret_cast<Vec<bf16, N>*>(dst + R + half + lane * N) = b;
  }
}

}  // namespace

void launch_rope(const RopeArgs& a, int dtype, cudaStream_t st) {
  if (a.T == 0 || a.H == 0) return;
  if (dtype == 0) {
    rope_dispatch<bf16>(a, st);
  } else if (dtype == 1) {
    rope_dispatch<__half>(a, st);
  } else {
    rope_dispatch<float>(a, st);
  }
}

void launch_rope_latent_write(const RopeArgs& a, const bf16* kv, int64_t kv_stride, const int64_t* slots,
                              const bf16* w, float eps, bf16* cache, int64_t num_slots, int R, cudaStream_t st) {
  if (a.T == 0) return;
  const int units = a.H * (a.interleaved ? 8 : 4);  // of 16 bytes (half layout: a pair of them) a token
  const int threads = std::min(256, std::max(32, (units + 31) / 32 * 32));
  const int latent_blocks = (int)((a.T * 32 + threads - 1) / threads);
  const int64_t q_blocks = a.H > 0 ? a.T : 0;
  if (latent_blocks + q_blocks > 0x7fffffff) throw std::runtime_error("rope_latent_write: too many rows");
  auto go = [&](auto kern) {
    launch_k(kern, dim3((unsigned)(latent_blocks + q_blocks)), dim3(threads), 0, st,
             static_cast<const bf16*>(a.x), a.xs_t, a.xs_h, static_cast<bf16*>(a.y), a.ys_t, a.ys_h, kv, kv_stride,
             a.positions, slots, a.cos_sin, a.max_pos, w, eps, cache, num_slots, (int)a.T, a.H, latent_blocks, a.err);
  };
  if (R == 512) {
    a.interleaved ? go(rope_latent_write_kernel<512, true>) : go(rope_latent_write_kernel<512, false>);
  } else if (R == 256) {
    a.interleaved ? go(rope_latent_write_kernel<256, true>) : go(rope_latent_write_kernel<256, false>);
  } else {
    throw std::runtime_error("rope_latent_write: the latent must have 256 or 512 values");
  }
  KAPSL_LAUNCH_CHECK();
  note_launch();
}

}  // namespace kapsl
