// Python bindings of the rotary and latent-attention kernels (registered by bindings.cpp).
#include <ATen/cuda/CUDAContext.h>
#include <c10/cuda/CUDAGuard.h>
#include <torch/extension.h>

#include <algorithm>
#include <utility>
#include <vector>

#include "common.cuh"
#include "kernels.h"

namespace {

using torch::Tensor;

constexpr int64_t kNope = 128, kRot = 64, kVal = 128;

inline __nv_bfloat16* bf(const Tensor& t) { return reinterpret_cast<__nv_bfloat16*>(t.data_ptr()); }
inline cudaStream_t cur_stream() { return at::cuda::getCurrentCUDAStream().stream(); }

// Numbers in messages go through this: an integer streamed into TORCH_CHECK's message crashed
// the process with this compiler and torch build instead of raising.
inline std::string num(int64_t v) { return std::to_string(v); }

void check(const Tensor& t, at::ScalarType dt, const Tensor& like, const char* op, const char* name) {
  TORCH_CHECK(t.is_cuda() && t.device() == like.device(), op, ": ", name, " must be on ", like.device().str());
  TORCH_CHECK(t.scalar_type() == dt, op, ": ", name, " must be ", toString(dt), ", got ", toString(t.scalar_type()));
}

// Byte range a tensor touches (dense upper bound of a strided view).
std::pair<uintptr_t, uintptr_t> span(const Tensor& t) {
  int64_t last = 0;
  for (int64_t d = 0; d < t.dim(); ++d) last += (t.size(d) - 1) * t.stride(d);
  const uintptr_t p = reinterpret_cast<uintptr_t>(t.data_ptr());
  return {p, p + (uintptr_t)(last + 1) * t.element_size()};
}

bool ranges_meet(const Tensor& a, const Tensor& b) {
  if (a.numel() == 0 || b.numel() == 0) return false;
  const auto x = span(a), y = span(b);
  return x.first < y.second && y.first < x.second;
}

bool same_view(const Tensor& a, const Tensor& b) {
  return a.data_ptr() == b.data_ptr() && a.sizes() == b.sizes() && a.strides() == b.strides();
}

// Strides of dims of one index never step, whatever they say.
int64_t step(const Tensor& t, int64_t d) { return t.size(d) > 1 ? t.stride(d) : 0; }

// Whether two indexes of a view may share an element: dim by dim, smallest stride first, each has to
// step over everything inside it.
bool overlaps_itself(const Tensor& t) {
  std::vector<std::pair<int64_t, int64_t>> dims;  // stride, size
  for (int64_t d = 0; d < t.dim(); ++d) {
    if (t.size(d) == 0) return false;
    if (t.size(d) > 1) dims.push_back({t.stride(d), t.size(d)});
  }
  std::sort(dims.begin(), dims.end());
  int64_t extent = 1;
  for (const auto& [stride, size] : dims) {
    if (stride < extent) return true;
    extent += (size - 1) * stride;
  }
  return false;
}

// Whether kv [T, n] shares elements with the heads q [T, H, D] of the same buffer's rows (a fused
// projection's), each row's heads taken as one stretch.  Views of other row pitches are not compared.
bool rows_meet(const Tensor& kv, const Tensor& q) {
  if (!ranges_meet(kv, q)) return false;
  const int64_t heads = step(q, 1) * (q.size(1) - 1) + q.size(2), width = kv.size(1);
  int64_t at = ((const char*)kv.data_ptr() - (const char*)q.data_ptr()) / q.element_size();
  if (q.size(0) == 1) return at < heads && at + width > 0;
  const int64_t pitch = q.stride(0);
  if (kv.stride(0) != pitch || heads > pitch) return false;
  at = (at % pitch + pitch) % pitch;  // kv's start behind the heads', in a row
  return at < heads || at + width > pitch;
}

// Row pitch of a [rows, width] view, for kernels and tensor maps: that of a lone row never counts.
int64_t pitch(const Tensor& t) { return t.size(0) > 1 ? t.stride(0) : t.size(1); }

// Rows that share memory (an expanded query) are copied: a tensor map's rows lie apart.
Tensor rows_apart(const Tensor& t) {
  if (t.size(0) <= 1 || t.stride(0) >= t.size(1)) return t;
  const c10::cuda::CUDAGuard g(t.device());
  return t.contiguous();
}

kapsl::RopeArgs rope_args(const char* op, const Tensor& x, const Tensor& y, const Tensor& positions,
                          const Tensor& cos_sin, int64_t offset, bool interleaved, const Tensor& err) {
  TORCH_CHECK(x.is_cuda(), op, ": x must be a CUDA tensor");
  TORCH_CHECK(x.dim() == 3 && (x.size(2) <= 1 || x.stride(2) == 1), op, ": x must be [T, H, D] with contiguous heads");
  check(y, x.scalar_type(), x, op, "out");
  TORCH_CHECK(y.sizes() == x.sizes() && (y.size(2) <= 1 || y.stride(2) == 1), op, ": out must have x's shape");
  TORCH_CHECK(!overlaps_itself(y), op, ": out must not be expanded or overlap itself");
  check(positions, at::kInt, x, op, "positions");
  TORCH_CHECK(positions.dim() == 1 && positions.is_contiguous() && positions.size(0) >= x.size(0), op,
              ": positions must hold an int32 per token");
  check(cos_sin, at::kFloat, x, op, "cos_sin");
  TORCH_CHECK(cos_sin.dim() == 2 && cos_sin.is_contiguous() && cos_sin.size(1) >= 2 && cos_sin.size(1) % 2 == 0 &&
                  cos_sin.size(0) <= INT32_MAX,
              op, ": cos_sin must be [positions, rotated dims] with an even width");
  TORCH_CHECK(offset >= 0 && offset + cos_sin.size(1) <= x.size(2), op, ": the rotated dims [", num(offset), ", ",
              num(offset + cos_sin.size(1)), ") leave the head of ", num(x.size(2)));
  TORCH_CHECK(x.size(1) <= INT32_MAX && x.size(2) <= INT32_MAX, op, ": sizes out of range");
  check(err, at::kInt, x, op, "err");
  const bool in_place = same_view(x, y);
  TORCH_CHECK(in_place || !ranges_meet(x, y), op, ": out must be x itself or not overlap it");
  kapsl::RopeArgs a;
  a.x = x.data_ptr();
  a.y = y.data_ptr();
  a.xs_t = step(x, 0);
  a.xs_h = step(x, 1);
  a.ys_t = step(y, 0);
  a.ys_h = step(y, 1);
  a.positions = positions.data_ptr<int32_t>();
  a.cos_sin = cos_sin.data_ptr<float>();
  a.max_pos = (int)cos_sin.size(0);
  a.T = x.size(0);
  a.H = (int)x.size(1);
  a.D = (int)x.size(2);
  a.P = (int)cos_sin.size(1);
  a.offset = (int)offset;
  a.interleaved = interleaved;
  a.in_place = in_place;
  a.err = err.data_ptr<int>();
  return a;
}

void rope(Tensor y, Tensor x, Tensor positions, Tensor cos_sin, int64_t offset, bool interleaved, Tensor err) {
  const at::ScalarType dt = x.scalar_type();
  TORCH_CHECK(dt == at::kBFloat16 || dt == at::kHalf || dt == at::kFloat, "rope: x must be bf16, fp16 or fp32");
  const kapsl::RopeArgs a = rope_args("rope", x, y, positions, cos_sin, offset, interleaved, err);
  const c10::cuda::CUDAGuard g(x.device());
  kapsl::launch_rope(a, dt == at::kBFloat16 ? 0 : dt == at::kHalf ? 1 : 2, cur_stream());
}

// cache [blocks, page, R + 64]; returns R
int64_t check_cache(const char* op, const Tensor& cache, const Tensor& like) {
  check(cache, at::kBFloat16, like, op, "cache");
  TORCH_CHECK(cache.dim() == 3 && cache.is_contiguous() && cache.size(0) >= 1, op, ": cache must be [blocks, page, R + 64] contiguous");
  const int64_t R = cache.size(2) - kRot, page = cache.size(1);
  TORCH_CHECK(R == 256 || R == 512, op, ": the latent must have 256 or 512 values (cache rows of 320 or 576), got rows of ",
              num(cache.size(2)));
  TORCH_CHECK(page == 16 || page == 32 || page == 64, op, ": pages must hold 16, 32 or 64 tokens, got ", num(page));
  TORCH_CHECK(cache.size(0) * page <= INT32_MAX, op, ": cache has too many rows");
  TORCH_CHECK((reinterpret_cast<uintptr_t>(cache.data_ptr()) & 15) == 0, op, ": cache must be 16-byte aligned");
  return R;
}

void check_rows16(const char* op, const Tensor& t, const char* name) {
  TORCH_CHECK((reinterpret_cast<uintptr_t>(t.data_ptr()) & 15) == 0, op, ": ", name, " must be 16-byte aligned");
  for (int64_t d = 0; d + 1 < t.dim(); ++d)
    TORCH_CHECK(step(t, d) % 8 == 0, op, ": ", name, " rows must be 16-byte aligned");
}

void rope_latent_write(Tensor q, Tensor q_out, Tensor kv, Tensor positions, Tensor slots, Tensor cos_sin, Tensor w,
                       double eps, Tensor cache, bool interleaved, Tensor err) {
  const char* op = "rope_latent_write";
  TORCH_CHECK(q.scalar_type() == at::kBFloat16, op, ": q must be bf16");
  const kapsl::RopeArgs a = rope_args(op, q, q_out, positions, cos_sin, 0, interleaved, err);
  TORCH_CHECK(a.D == kRot && a.P == kRot, op, ": q must be [T, H, 64] (the rotary part) with a table of width 64");
  check_rows16(op, q, "q");
  check_rows16(op, q_out, "q_out");
  const int64_t R = check_cache(op, cache, q);
  check(kv, at::kBFloat16, q, op, "kv");
  TORCH_CHECK(kv.dim() == 2 && kv.stride(1) == 1 && kv.size(0) == q.size(0) && kv.size(1) == R + kRot, op,
              ": kv must be [T, ", num(R + kRot), "]");
  check_rows16(op, kv, "kv");
  check(w, at::kBFloat16, q, op, "weight");
  TORCH_CHECK(w.dim() == 1 && w.size(0) == R && w.is_contiguous() && (reinterpret_cast<uintptr_t>(w.data_ptr()) & 15) == 0,
              op, ": weight must be [", num(R), "], contiguous and 16-byte aligned");
  check(slots, at::kLong, q, op, "slots");
  TORCH_CHECK(slots.dim() == 1 && slots.is_contiguous() && slots.size(0) >= q.size(0), op,
              ": slots must hold an int64 per token");
  TORCH_CHECK((reinterpret_cast<uintptr_t>(cos_sin.data_ptr()) & 15) == 0, op, ": cos_sin must be 16-byte aligned");
  TORCH_CHECK(q.size(0) <= INT32_MAX, op, ": too many tokens");
  TORCH_CHECK(!ranges_meet(cache, kv) && !ranges_meet(cache, q_out), op, ": the cache must not overlap kv or q");
  TORCH_CHECK(a.in_place ? !rows_meet(kv, q) : !ranges_meet(kv, q_out), op,
              ": the query heads written must not overlap kv");
  const c10::cuda::CUDAGuard g(q.device());
  kapsl::launch_rope_latent_write(a, bf(kv), kv.size(0) > 1 ? kv.stride(0) : 0, slots.data_ptr<int64_t>(), bf(w),
                                  (float)eps, bf(cache), cache.size(0) * cache.size(1), (int)R, cur_stream());
}

// Workspace of latent_decode_attention for these rows of q.
int64_t latent_workspace_bytes(Tensor q, int64_t H, int64_t R, int64_t max_ctx) {
  TORCH_CHECK(q.is_cuda() && q.dim() == 2 && q.size(0) <= 65535 && H >= 1 && H <= 1024 && (R == 256 || R == 512),
              "latent_decode_attention: q, num_heads or the cache's row width out of range");
  const c10::cuda::CUDAGuard g(q.device());
  return (int64_t)kapsl::latent_decode_workspace_bytes((int)q.size(0), (int)H, (int)R,
                                                       (int)std::min<int64_t>(std::max<int64_t>(max_ctx, 0), INT32_MAX),
                                                       kapsl::gemm_num_sms());
}

// q / out [rows, heads * width] and w [H, 256, R]
void check_heads(const char* op, const Tensor& q, const Tensor& cache, const Tensor& w, const Tensor& out, int64_t H,
                 int64_t R) {
  TORCH_CHECK(H >= 1 && H <= 1024, op, ": num_heads out of range");
  TORCH_CHECK(q.dim() == 2 && q.size(1) == H * (kNope + kRot) && (q.size(1) == 0 || q.stride(1) == 1), op, ": q must be [T, ",
              num(H * (kNope + kRot)), "] (128 + 64 dims a head)");
  check_rows16(op, q, "q");
  check(out, at::kBFloat16, q, op, "out");
  TORCH_CHECK(out.dim() == 2 && out.size(1) == H * kVal && out.stride(1) == 1 && out.size(0) == q.size(0), op,
              ": out must be [T, ", num(H * kVal), "]");
  check_rows16(op, out, "out");
  TORCH_CHECK(!overlaps_itself(out), op, ": out must not be expanded or overlap itself");
  check(w, at::kBFloat16, q, op, "w_kv_b");
  TORCH_CHECK(w.numel() == H * (kNope + kVal) * R && w.size(-1) == R && w.is_contiguous(), op, ": w_kv_b must be [", num(H),
              " * 256, ", num(R), "] contiguous");
  TORCH_CHECK((reinterpret_cast<uintptr_t>(w.data_ptr()) & 15) == 0, op, ": w_kv_b must be 16-byte aligned");
  TORCH_CHECK(!ranges_meet(q, out) && !ranges_meet(cache, out) && !ranges_meet(w, out), op,
              ": out must not overlap q, the cache or w_kv_b");
}

void latent_decode_attention(Tensor q, Tensor cache, Tensor w, Tensor block_tables, Tensor ctx_lens, Tensor out,
                             int64_t H, double scale, int64_t max_ctx, Tensor workspace,
                             c10::optional<Tensor> table_rows, Tensor err) {
  const char* op = "latent_decode_attention";
  TORCH_CHECK(q.is_cuda(), op, ": q must be a CUDA tensor");
  check(q, at::kBFloat16, q, op, "q");
  const int64_t R = check_cache(op, cache, q);
  check_heads(op, q, cache, w, out, H, R);
  const int64_t B = q.size(0);
  check(block_tables, at::kInt, q, op, "block_tables");
  TORCH_CHECK(block_tables.dim() == 2 && block_tables.is_contiguous() &&
                  (table_rows.has_value() || block_tables.size(0) >= B) && (block_tables.size(1) >= 1 || B == 0),
              op, ": block_tables must be [B, max_blocks] contiguous");
  // the kernels count tokens of a row, rounded up to a tile, and tiles of all rows in 32 bits
  const int64_t tokens = block_tables.size(1) * cache.size(1);
  TORCH_CHECK(tokens <= INT32_MAX - 128, op, ": block_tables too wide");
  TORCH_CHECK(B * ((tokens + 63) / 64) <= 1 << 30, op, ": ", num(B), " rows of up to ", num(tokens),
              " tokens are too many for one call");
  check(ctx_lens, at::kInt, q, op, "ctx_lens");
  TORCH_CHECK(ctx_lens.dim() == 1 && ctx_lens.is_contiguous() && ctx_lens.size(0) >= B, op,
              ": ctx_lens must hold an int32 per row");
  TORCH_CHECK(B <= 65535, op, ": at most 65535 rows");
  check(workspace, at::kByte, q, op, "workspace");
  TORCH_CHECK(workspace.is_contiguous() && workspace.numel() >= latent_workspace_bytes(q, H, R, max_ctx) &&
                  (reinterpret_cast<uintptr_t>(workspace.data_ptr()) & 127) == 0,
              op, ": workspace too small or not 128-byte aligned");
  check(err, at::kInt, q, op, "err");
  q = rows_apart(q);
  const c10::cuda::CUDAGuard g(q.device());
  kapsl::LatentDecode a;
  if (table_rows.has_value()) {
    check(*table_rows, at::kInt, q, op, "table_rows");
    TORCH_CHECK(table_rows->dim() == 1 && table_rows->is_contiguous() && table_rows->size(0) >= B, op,
                ": table_rows must hold an int32 per row");
    a.table_rows = table_rows->data_ptr<int32_t>();
  }
  a.num_tables = (int)block_tables.size(0);
  a.q = bf(q);
  a.q_stride = pitch(q);
  a.cache = bf(cache);
  a.num_blocks = cache.size(0);
  a.page = (int)cache.size(1);
  a.R = (int)R;
  a.w = bf(w);
  a.block_tables = block_tables.data_ptr<int32_t>();
  a.max_blocks = (int)block_tables.size(1);
  a.ctx_lens = ctx_lens.data_ptr<int32_t>();
  a.out = bf(out);
  a.out_stride = pitch(out);
  a.B = (int)B;
  a.H = (int)H;
  a.max_ctx = (int)std::min<int64_t>(std::max<int64_t>(max_ctx, 0), INT32_MAX);
  a.num_sms = kapsl::gemm_num_sms();
  a.scale = (float)scale;
  a.workspace = workspace.data_ptr();
  a.err = err.data_ptr<int>();
  kapsl::launch_latent_decode(a, cur_stream());
}

// kv [n, heads * 256] and, where given, k_rope [n, 64] of the plan's context rows; w [heads * 256, R]
void latent_expand(Tensor cache, Tensor w, Tensor work, Tensor seq_info, Tensor block_tables, Tensor kv,
                   c10::optional<Tensor> k_rope, Tensor err) {
  const char* op = "latent_expand";
  TORCH_CHECK(cache.is_cuda(), op, ": cache must be a CUDA tensor");
  const int64_t R = check_cache(op, cache, cache);
  check(w, at::kBFloat16, cache, op, "w");
  check(kv, at::kBFloat16, cache, op, "kv");
  check(work, at::kInt, cache, op, "work");
  check(seq_info, at::kInt, cache, op, "seq_info");
  check(block_tables, at::kInt, cache, op, "block_tables");
  check(err, at::kInt, cache, op, "err");
  TORCH_CHECK(w.dim() == 2 && w.is_contiguous() && w.size(1) == R && w.size(0) % 256 == 0 && w.size(0) > 0, op,
              ": w must be [heads * 256, R]");
  const int64_t heads = w.size(0) / 256;
  TORCH_CHECK(kv.dim() == 2 && kv.stride(1) == 1 && kv.size(1) == heads * 256 && kv.stride(0) >= kv.size(1), op,
              ": kv must be [n, heads * 256]");
  check_rows16(op, kv, "kv");
  check_rows16(op, w, "w");
  TORCH_CHECK(work.dim() == 2 && work.size(1) == 2 && work.is_contiguous(), op, ": work [n, 2]");
  TORCH_CHECK(seq_info.dim() == 2 && seq_info.size(1) == 5 && seq_info.is_contiguous(), op, ": seq_info [S, 5]");
  TORCH_CHECK(block_tables.dim() == 2 && block_tables.is_contiguous(), op, ": block_tables [S, max_blocks]");
  kapsl::LatentExpand a;
  if (k_rope.has_value()) {
    check(*k_rope, at::kBFloat16, cache, op, "k_rope");
    TORCH_CHECK(k_rope->dim() == 2 && k_rope->is_contiguous() && k_rope->size(1) == kRot && k_rope->size(0) == kv.size(0),
                op, ": k_rope must be [n, 64]");
    a.k_rope = bf(*k_rope);
  }
  const c10::cuda::CUDAGuard g(cache.device());
  a.cache = bf(cache);
  a.num_blocks = cache.size(0);
  a.page = (int)cache.size(1);
  a.R = (int)R;
  a.w = bf(w);
  a.work = work.data_ptr<int32_t>();
  a.nwork = (int)work.size(0);
  a.seq_info = seq_info.data_ptr<int32_t>();
  a.block_tables = block_tables.data_ptr<int32_t>();
  a.max_blocks = (int)block_tables.size(1);
  a.heads = (int)heads;
  a.num_sms = kapsl::gemm_num_sms();
  a.kv = bf(kv);
  a.kv_stride = pitch(kv);
  a.err = err.data_ptr<int>();
  kapsl::launch_latent_expand(a, cur_stream());
}

void check_latent_prefill(Tensor q, Tensor cache, Tensor w, Tensor block_tables, Tensor out, int64_t H, int64_t rows,
                          int64_t tables, int64_t max_ctx) {
  const char* op = "latent_prefill_attention";
  TORCH_CHECK(q.is_cuda(), op, ": q must be a CUDA tensor");
  check(q, at::kBFloat16, q, op, "q");
  const int64_t R = check_cache(op, cache, q);
  check_heads(op, q, cache, w, out, H, R);
  check(block_tables, at::kInt, q, op, "block_tables");
  TORCH_CHECK(block_tables.dim() == 2 && block_tables.is_contiguous(), op, ": block_tables must be contiguous");
  TORCH_CHECK(q.size(0) >= rows, op, ": the plan covers ", num(rows), " rows of q, which has ",
              num(q.size(0)));
  TORCH_CHECK(block_tables.size(0) >= tables, op, ": the plan reads ", num(tables), " block tables, given ",
              num(block_tables.size(0)));
  TORCH_CHECK(block_tables.size(1) * cache.size(1) >= max_ctx, op, ": block_tables hold ",
              num(block_tables.size(1) * cache.size(1)), " tokens a sequence, the plan needs ", num(max_ctx));
}

// attention of `heads` heads: q / out already narrowed to them
void latent_prefill(Tensor q, Tensor kv, Tensor k_rope, Tensor work, Tensor seq_info, Tensor out, int64_t heads,
                    double scale, int64_t cut, int64_t part_tiles, int64_t slots, c10::optional<Tensor> parts,
                    Tensor err) {
  const char* op = "latent_prefill";
  TORCH_CHECK(q.is_cuda(), op, ": q must be a CUDA tensor");
  check(q, at::kBFloat16, q, op, "q");
  check(kv, at::kBFloat16, q, op, "kv");
  check(k_rope, at::kBFloat16, q, op, "k_rope");
  check(out, at::kBFloat16, q, op, "out");
  check(work, at::kInt, q, op, "work");
  check(seq_info, at::kInt, q, op, "seq_info");
  check(err, at::kInt, q, op, "err");
  TORCH_CHECK(heads >= 1 && heads <= 65535, op, ": heads out of range");
  TORCH_CHECK(q.dim() == 2 && q.stride(1) == 1 && q.size(1) == heads * (kNope + kRot), op, ": q [T, heads * 192]");
  TORCH_CHECK(kv.dim() == 2 && kv.stride(1) == 1 && kv.size(1) == heads * (kNope + kVal), op, ": kv [n, heads * 256]");
  TORCH_CHECK(k_rope.dim() == 2 && k_rope.is_contiguous() && k_rope.size(1) == kRot && k_rope.size(0) == kv.size(0), op,
              ": k_rope [n, 64]");
  TORCH_CHECK(out.dim() == 2 && out.stride(1) == 1 && out.size(1) == heads * kVal && out.size(0) == q.size(0), op,
              ": out [T, heads * 128]");
  TORCH_CHECK(work.dim() == 2 && work.size(1) == 2 && work.is_contiguous(), op, ": work [n, 2]");
  TORCH_CHECK(seq_info.dim() == 2 && seq_info.size(1) == 5 && seq_info.is_contiguous(), op, ": seq_info [S, 5]");
  check_rows16(op, q, "q");
  check_rows16(op, kv, "kv");
  check_rows16(op, k_rope, "k_rope");
  check_rows16(op, out, "out");
  q = rows_apart(q);
  const c10::cuda::CUDAGuard g(q.device());
  kapsl::LatentPrefill a;
  a.q = bf(q);
  a.q_stride = pitch(q);
  a.T = q.size(0);
  a.kv = bf(kv);
  a.kv_stride = pitch(kv);
  a.kv_rows = kv.size(0);
  if (cut > 0) {
    TORCH_CHECK(cut <= work.size(0) && part_tiles >= 1 && part_tiles <= INT32_MAX && slots >= 1 && slots <= 32, op,
                ": row tiles or parts out of range");
    const int64_t rows = slots * heads * cut * 256;
    TORCH_CHECK(parts.has_value(), op, ": key ranges need room for partial results");
    check(*parts, at::kFloat, q, op, "parts");
    TORCH_CHECK(parts->is_contiguous() && parts->numel() >= rows * (kVal + 2), op, ": parts too small");
    a.cut = (int)cut;
    a.part_tiles = (int)part_tiles;
    a.slots = (int)slots;
    a.part_o = parts->data_ptr<float>();
    a.part_ml = reinterpret_cast<float2*>(a.part_o + rows * kVal);
  }
  a.k_rope = bf(k_rope);
  a.work = work.data_ptr<int32_t>();
  a.nwork = (int)work.size(0);
  a.seq_info = seq_info.data_ptr<int32_t>();
  a.out = bf(out);
  a.out_stride = pitch(out);
  a.heads = (int)heads;
  a.scale = (float)scale;
  a.err = err.data_ptr<int>();
  kapsl::launch_latent_prefill(a, cur_stream());
}

}  // namespace

void register_latent(pybind11::module_& m) {
  m.def("rope", &rope, "rotary positions of strided heads (half / interleaved, part of the head)");
  m.def("rope_latent_write", &rope_latent_write, "latent norm + rotary key -> paged latent cache, query rotary part");
  m.def("latent_decode_attention", &latent_decode_attention, "absorbed latent attention over a paged cache");
  m.def("latent_workspace_bytes", &latent_workspace_bytes);
  m.def("latent_expand", &latent_expand, "keys and values of every head from the paged latent cache");
  m.def("check_latent_prefill", &check_latent_prefill);
  m.def("latent_prefill", &latent_prefill, "causal attention over expanded latent keys and values");
}
