// PyTorch-ROCm operators over the C ABI in include/kv_cache.h: the appends to
// the paged caches and the attention over the 4-bit one. In the manner of
// gqa_decode_ext.cpp: checks that raise RuntimeError, outputs and workspace
// from the caching allocator, a device guard, the current stream, the
// launcher's code checked. Host-only C++; the device code is in the
// hipcc-built library. python/kv_cache.py documents the operators.
#include <torch/extension.h>

#include <c10/core/DeviceGuard.h>
#include <c10/hip/HIPStream.h>

#include <cmath>
#include <optional>

#include "kv_cache.h"

namespace {

using torch::Tensor;
using OptTensor = std::optional<Tensor>;

constexpr int64_t kDim = 128, kLatent = 512, kRope = 64;

void check_launch(int err, const char* op) {
  TORCH_CHECK(err == 0, op, " failed: ", hipGetErrorString(static_cast<hipError_t>(err)),
              " (hipError_t ", err, ")");
}

uint16_t* bf16(const Tensor& t) { return reinterpret_cast<uint16_t*>(t.data_ptr()); }
hipStream_t stream_of(const Tensor& t) {
  return c10::hip::getCurrentHIPStream(t.device().index()).stream();
}

void check_rows(const Tensor& t, const char* name, int64_t dims, const char* shape) {
  TORCH_CHECK(t.is_cuda(), name, " must be a CUDA tensor");
  TORCH_CHECK(t.scalar_type() == torch::kBFloat16, name, " must be bf16");
  TORCH_CHECK(t.dim() == (dims == 0 ? 2 : 3), name, " must be ", shape);
  TORCH_CHECK(t.numel() == 0 || t.stride(-1) == 1, name, " must have contiguous dims (stride 1)");
  TORCH_CHECK(t.dim() < 3 || (t.stride(0) >= 0 && t.stride(1) >= 0), name,
              " must not have negative strides");
}

void check_index(const Tensor& t, const char* name, int64_t dim, const Tensor& like) {
  TORCH_CHECK(t.is_cuda(), name, " must be a CUDA tensor");
  TORCH_CHECK(t.scalar_type() == torch::kInt32, name, " must be int32");
  TORCH_CHECK(t.is_contiguous(), name, " must be contiguous");
  TORCH_CHECK(t.dim() == dim, name, " must have ", dim, " dimension(s)");
  TORCH_CHECK(t.device() == like.device(), "all tensors must be on the same device");
}

void check_same_device(const Tensor& t, const Tensor& like) {
  TORCH_CHECK(t.device() == like.device(), "all tensors must be on the same device");
}

int narrow(int64_t x, const char* what) {
  TORCH_CHECK(x >= 0 && x <= INT32_MAX, what, " is too large");
  return (int)x;
}

// A strided array of rows: [T, heads] rows of `width` elements.
struct Rows {
  const char* name;
  int64_t base, T, heads, st, sh, width;  // base in elements (addresses are multiples of 2)

  int64_t token_width() const { return heads > 0 ? (heads - 1) * sh + width : 0; }
  int64_t extent() const { return T > 0 ? (T - 1) * st + token_width() : 0; }
};

Rows rows_of(const char* name, const Tensor& t) {
  const bool heads = t.dim() == 3;
  return {name, (int64_t)(reinterpret_cast<uintptr_t>(t.data_ptr()) / 2), t.size(0),
          heads ? t.size(1) : 1, t.stride(0), heads ? t.stride(1) : 0, t.size(-1)};
}

// The stride of a dimension that two arrays share, -1 if they differ. (Of a dimension
// of size 1 it can be anything and means nothing.)
int64_t common_stride(int64_t sx, int64_t nx, int64_t sy, int64_t ny) {
  return nx <= 1 ? sy : ny <= 1 || sx == sy ? sx : -1;
}

// Whether x and y surely have no element in common: apart as a whole, or, with
// the same token (and head) stride, in every period of it (two views of one
// projection's output).
bool disjoint(const Rows& x, const Rows& y) {
  if (x.extent() == 0 || y.extent() == 0) return true;
  if (x.base + x.extent() <= y.base || y.base + y.extent() <= x.base) return true;
  const auto apart = [](int64_t d, int64_t period, int64_t wx, int64_t wy) {
    if (period <= 0) return false;
    const int64_t m = ((d % period) + period) % period;
    return wx <= m && m + wy <= period;
  };
  const int64_t d = y.base - x.base;
  const int64_t st = common_stride(x.st, x.T, y.st, y.T);
  const int64_t sh = common_stride(x.sh, x.heads, y.sh, y.heads);
  if (apart(d, st, x.token_width(), y.token_width())) return true;
  const bool one_token = x.T == 1 && y.T == 1;
  return st >= 0 && sh > 0 && (one_token || st % sh == 0) && apart(d, sh, x.width, y.width);
}

void check_no_overlap(const Rows& x, const Rows& y) {
  TORCH_CHECK(disjoint(x, y), x.name, " and ", y.name, " must not overlap");
}

// A written tensor whose own rows overlap (an expanded view) has no one result.
void check_written(const Rows& x) {
  const bool heads_apart = x.heads <= 1 || x.sh >= x.width;
  const bool tokens_apart = x.T <= 1 || x.st >= x.token_width() ||
                            (x.st >= x.width && (x.heads <= 1 || x.sh >= (x.T - 1) * x.st + x.width));
  TORCH_CHECK(x.extent() == 0 || (heads_apart && tokens_apart), x.name,
              " must not overlap itself");
}

// A contiguous cache as one row.
Rows whole(const Tensor& cache, const char* name) {
  const int64_t elements = (int64_t)(cache.numel() * cache.element_size() + 1) / 2;
  return {name, (int64_t)(reinterpret_cast<uintptr_t>(cache.data_ptr()) / 2), 1, 1, 0, 0, elements};
}

void check_cache_apart(const Tensor& cache, const char* name, std::initializer_list<Rows> others) {
  for (const Rows& r : others) check_no_overlap(r, whole(cache, name));
}

void check_aligned(const Tensor& t, const char* name, uintptr_t to) {
  TORCH_CHECK(reinterpret_cast<uintptr_t>(t.data_ptr()) % to == 0, name, " must be ", to,
              "-byte aligned");
}

struct Index {
  int T, B, max_blocks;
  const int *table, *lens, *cu, *rope;
};

Index check_tokens(int64_t T, const Tensor& block_table, const Tensor& seq_lens,
                   const OptTensor& cu_seqlens, const OptTensor& positions, const Tensor& like) {
  check_index(block_table, "block_table", 2, like);
  check_index(seq_lens, "seq_lens", 1, like);
  const int64_t B = seq_lens.size(0);
  TORCH_CHECK(block_table.size(0) == B, "block_table batch dim must match seq_lens");
  TORCH_CHECK(block_table.size(1) > 0, "block_table must have at least one column");
  TORCH_CHECK(T <= KV_MAX_TOKENS, "at most ", KV_MAX_TOKENS, " new tokens a call");
  Index ix{narrow(T, "the number of tokens"), narrow(B, "the batch"),
           narrow(block_table.size(1), "block_table"), block_table.data_ptr<int>(),
           seq_lens.data_ptr<int>(), nullptr, nullptr};
  if (cu_seqlens) {
    check_index(*cu_seqlens, "cu_seqlens", 1, like);
    TORCH_CHECK(cu_seqlens->size(0) == B + 1, "cu_seqlens must be [B + 1]");
    ix.cu = cu_seqlens->data_ptr<int>();
  } else {
    TORCH_CHECK(T == B, "without cu_seqlens there must be one new token a request");
  }
  if (positions) {
    check_index(*positions, "positions", 1, like);
    TORCH_CHECK(positions->size(0) == T, "positions must be [T]");
    ix.rope = positions->data_ptr<int>();
  }
  return ix;
}

const float* check_angles(const Tensor& t, const Tensor& like) {
  TORCH_CHECK(t.is_cuda(), "cos_sin must be a CUDA tensor");
  TORCH_CHECK(t.scalar_type() == torch::kFloat32, "cos_sin must be fp32");
  TORCH_CHECK(t.dim() == 2 && t.is_contiguous(),
              "cos_sin must be a contiguous [positions, rotary_dim] tensor");
  check_same_device(t, like);
  return t.data_ptr<float>();
}

const void* check_weight(const OptTensor& w, const char* name, int64_t dims, const Tensor& like,
                         int& type) {
  type = KV_WEIGHT_BF16;
  if (!w) return nullptr;
  TORCH_CHECK(w->is_cuda(), name, " must be a CUDA tensor");
  TORCH_CHECK(w->scalar_type() == torch::kBFloat16 || w->scalar_type() == torch::kFloat32, name,
              " must be bf16 or fp32");
  TORCH_CHECK(w->dim() == 1 && w->size(0) == dims && w->is_contiguous(), name,
              " must be a contiguous [", dims, "] tensor");
  check_same_device(*w, like);
  if (w->scalar_type() == torch::kFloat32) type = KV_WEIGHT_FP32;
  return w->data_ptr();
}

void check_mxfp4(const Tensor& cache, const Tensor& like) {
  TORCH_CHECK(cache.is_cuda(), "kv_cache must be a CUDA tensor");
  TORCH_CHECK(cache.scalar_type() == torch::kUInt8, "kv_cache must be uint8");
  TORCH_CHECK(cache.is_contiguous(), "kv_cache must be contiguous");
  TORCH_CHECK(cache.dim() == 4 && cache.size(1) > 0 && cache.size(2) > 0 &&
                  cache.size(3) == KV_MXFP4_TILE_BYTES,
              "kv_cache must be [num_blocks, Hkv, block_size / 16, 2176]");
  check_aligned(cache, "kv_cache", 16);
  check_same_device(cache, like);
}

// q_out as given, or a new tensor of q's shape.
Tensor output_for(const Tensor& q, const OptTensor& q_out, const char* shape) {
  if (!q_out) return torch::empty(q.sizes(), q.options());
  check_rows(*q_out, "q_out", 1, shape);
  TORCH_CHECK(q_out->sizes() == q.sizes(), "q_out must have q's shape");
  check_same_device(*q_out, q);
  return *q_out;
}

void check_output(const Rows& q, const Rows& out, std::initializer_list<Rows> inputs) {
  check_written(out);
  const bool in_place = q.base == out.base && (q.T <= 1 || q.st == out.st) &&
                        (q.heads <= 1 || q.sh == out.sh);
  if (!in_place) check_no_overlap(q, out);
  for (const Rows& r : inputs) check_no_overlap(r, out);
}

Tensor append(bool mx, const Tensor& q, const Tensor& k, const Tensor& v, const Tensor& k_cache,
              const OptTensor& v_cache, const Tensor& block_table, const Tensor& seq_lens,
              const OptTensor& cos_sin, const OptTensor& cu_seqlens, const OptTensor& positions,
              const OptTensor& q_weight, const OptTensor& k_weight, double eps, bool interleaved,
              const OptTensor& q_out) {
  check_rows(q, "q", 1, "[T, Hq, 128]");
  check_rows(k, "k", 1, "[T, Hkv, 128]");
  check_rows(v, "v", 1, "[T, Hkv, 128]");
  TORCH_CHECK(q.size(2) == kDim && k.size(2) == kDim && v.size(2) == kDim,
              "q, k and v must have head dim 128");
  TORCH_CHECK(k.sizes() == v.sizes(), "k and v must have the same shape");
  TORCH_CHECK(q.size(0) == k.size(0), "q, k and v must have the same number of tokens");
  check_same_device(k, q);
  check_same_device(v, q);
  const int64_t Hq = q.size(1), Hkv = k.size(1);
  TORCH_CHECK(Hq > 0 && Hkv > 0 && Hq <= 4096 && Hkv <= 4096, "between 1 and 4096 heads");
  kv_append_args a{};
  if (mx) {
    check_mxfp4(k_cache, q);
    TORCH_CHECK(k_cache.size(1) == Hkv, "kv_cache must have k's number of heads");
    a.mxfp4_cache = k_cache.data_ptr<uint8_t>();
    a.num_blocks = narrow(k_cache.size(0), "kv_cache");
    a.block_size = narrow(k_cache.size(2) * KV_MXFP4_TILE_TOKENS, "block_size");
  } else {
    TORCH_CHECK(k_cache.is_cuda() && v_cache->is_cuda(), "k_cache/v_cache must be CUDA tensors");
    TORCH_CHECK(k_cache.scalar_type() == torch::kBFloat16 &&
                    v_cache->scalar_type() == torch::kBFloat16,
                "k_cache/v_cache must be bf16");
    TORCH_CHECK(k_cache.is_contiguous() && v_cache->is_contiguous(),
                "k_cache/v_cache must be contiguous");
    TORCH_CHECK(k_cache.dim() == 4 && k_cache.size(1) > 0 && k_cache.size(2) == Hkv &&
                    k_cache.size(3) == kDim,
                "k_cache must be [num_blocks, block_size, Hkv, 128]");
    TORCH_CHECK(k_cache.sizes() == v_cache->sizes(),
                "k_cache and v_cache must have the same shape");
    check_same_device(k_cache, q);
    check_same_device(*v_cache, q);
    check_aligned(k_cache, "k_cache", 16);
    check_aligned(*v_cache, "v_cache", 16);
    a.k_cache = bf16(k_cache);
    a.v_cache = bf16(*v_cache);
    a.num_blocks = narrow(k_cache.size(0), "k_cache");
    a.block_size = narrow(k_cache.size(1), "block_size");
  }
  const Index ix = check_tokens(q.size(0), block_table, seq_lens, cu_seqlens, positions, q);
  if (cos_sin) {
    a.cos_sin = check_angles(*cos_sin, q);
    TORCH_CHECK(cos_sin->size(1) >= 16 && cos_sin->size(1) <= kDim && cos_sin->size(1) % 16 == 0,
                "rotary_dim must be a multiple of 16 between 16 and 128");
    TORCH_CHECK(cos_sin->size(0) > 0, "cos_sin must have at least one position");
    a.table_rows = narrow(cos_sin->size(0), "cos_sin");
    a.rotary_dim = (int)cos_sin->size(1);
  }
  a.q_weight = check_weight(q_weight, "q_weight", kDim, q, a.q_weight_type);
  a.k_weight = check_weight(k_weight, "k_weight", kDim, q, a.k_weight_type);
  const c10::DeviceGuard guard(q.device());
  Tensor out = output_for(q, q_out, "[T, Hq, 128]");
  const Rows rq = rows_of("q", q), rk = rows_of("k", k), rv = rows_of("v", v),
             ro = rows_of("q_out", out);
  check_output(rq, ro, {rk, rv});
  check_cache_apart(k_cache, mx ? "kv_cache" : "k_cache", {rq, rk, rv, ro});
  if (!mx) {
    check_cache_apart(*v_cache, "v_cache", {rq, rk, rv, ro});
    check_cache_apart(k_cache, "k_cache", {whole(*v_cache, "v_cache")});
  }
  a.q = bf16(q), a.k = bf16(k), a.v = bf16(v), a.q_out = bf16(out);
  a.q_token_stride = rq.st, a.q_head_stride = rq.sh;
  a.k_token_stride = rk.st, a.k_head_stride = rk.sh;
  a.v_token_stride = rv.st, a.v_head_stride = rv.sh;
  a.q_out_token_stride = ro.st, a.q_out_head_stride = ro.sh;
  a.block_table = ix.table, a.seq_lens = ix.lens, a.cu_seqlens = ix.cu, a.rope_positions = ix.rope;
  a.T = ix.T, a.B = ix.B, a.max_blocks = ix.max_blocks;
  a.Hq = (int)Hq, a.Hkv = (int)Hkv;
  a.interleaved = interleaved;
  a.eps = (float)eps;
  if (mx)
    check_launch(kv_append_mxfp4_launch(&a, stream_of(q)), "kv_append_mxfp4_launch");
  else
    check_launch(kv_append_launch(&a, stream_of(q)), "kv_append_launch");
  return out;
}

Tensor kv_append(Tensor q, Tensor k, Tensor v, Tensor k_cache, Tensor v_cache, Tensor block_table,
                 Tensor seq_lens, OptTensor cos_sin, OptTensor cu_seqlens, OptTensor positions,
                 OptTensor q_weight, OptTensor k_weight, double eps, bool interleaved,
                 OptTensor q_out) {
  return append(false, q, k, v, k_cache, v_cache, block_table, seq_lens, cos_sin, cu_seqlens,
                positions, q_weight, k_weight, eps, interleaved, q_out);
}

Tensor kv_append_mxfp4(Tensor q, Tensor k, Tensor v, Tensor kv_cache, Tensor block_table,
                       Tensor seq_lens, OptTensor cos_sin, OptTensor cu_seqlens,
                       OptTensor positions, OptTensor q_weight, OptTensor k_weight, double eps,
                       bool interleaved, OptTensor q_out) {
  return append(true, q, k, v, kv_cache, std::nullopt, block_table, seq_lens, cos_sin, cu_seqlens,
                positions, q_weight, k_weight, eps, interleaved, q_out);
}

std::tuple<Tensor, Tensor> kv_read_mxfp4(Tensor kv_cache, Tensor block_table, Tensor seq_lens,
                                         OptTensor cu_seqlens, std::optional<int64_t> num_tokens) {
  check_mxfp4(kv_cache, kv_cache);
  TORCH_CHECK(seq_lens.dim() == 1, "seq_lens must have 1 dimension(s)");
  TORCH_CHECK(num_tokens || !cu_seqlens, "cu_seqlens needs num_tokens");
  const int64_t T = num_tokens ? *num_tokens : seq_lens.size(0);
  TORCH_CHECK(T >= 0, "num_tokens must not be negative");
  const Index ix = check_tokens(T, block_table, seq_lens, cu_seqlens, std::nullopt, kv_cache);
  const c10::DeviceGuard guard(kv_cache.device());
  const auto opts = kv_cache.options().dtype(torch::kBFloat16);
  const int64_t Hkv = kv_cache.size(1);
  Tensor k = torch::empty({T, Hkv, kDim}, opts), v = torch::empty({T, Hkv, kDim}, opts);
  check_launch(kv_read_mxfp4_launch(
                   kv_cache.data_ptr<uint8_t>(), ix.table, ix.lens, ix.cu, bf16(k), bf16(v), ix.T,
                   ix.B, narrow(Hkv, "Hkv"), narrow(kv_cache.size(0), "kv_cache"),
                   narrow(kv_cache.size(2) * KV_MXFP4_TILE_TOKENS, "block_size"), ix.max_blocks,
                   stream_of(kv_cache)),
               "kv_read_mxfp4_launch");
  return {k, v};
}

Tensor mla_append(Tensor q_pe, Tensor c_kv, Tensor k_pe, Tensor kv_cache, Tensor block_table,
                  Tensor seq_lens, Tensor cos_sin, OptTensor cu_seqlens, OptTensor positions,
                  OptTensor c_weight, double eps, bool interleaved, OptTensor q_out) {
  check_rows(q_pe, "q_pe", 1, "[T, h_q, 64]");
  check_rows(c_kv, "c_kv", 0, "[T, 512]");
  check_rows(k_pe, "k_pe", 0, "[T, 64]");
  TORCH_CHECK(q_pe.size(2) == kRope, "q_pe must be [T, h_q, 64]");
  TORCH_CHECK(c_kv.size(1) == kLatent, "c_kv must be [T, 512]");
  TORCH_CHECK(k_pe.size(1) == kRope, "k_pe must be [T, 64]");
  TORCH_CHECK(q_pe.size(0) == c_kv.size(0) && q_pe.size(0) == k_pe.size(0),
              "q_pe, c_kv and k_pe must have the same number of tokens");
  TORCH_CHECK(q_pe.size(1) > 0 && q_pe.size(1) <= 4096, "between 1 and 4096 heads");
  check_same_device(c_kv, q_pe);
  check_same_device(k_pe, q_pe);
  TORCH_CHECK(kv_cache.is_cuda(), "kv_cache must be a CUDA tensor");
  TORCH_CHECK(kv_cache.scalar_type() == torch::kBFloat16, "kv_cache must be bf16");
  TORCH_CHECK(kv_cache.is_contiguous(), "kv_cache must be contiguous");
  TORCH_CHECK(kv_cache.dim() == 4 && kv_cache.size(1) > 0 && kv_cache.size(2) == 1 &&
                  kv_cache.size(3) == kLatent + kRope,
              "kv_cache must be [num_blocks, block_size, 1, 576]");
  check_aligned(kv_cache, "kv_cache", 16);
  check_same_device(kv_cache, q_pe);
  const Index ix = check_tokens(q_pe.size(0), block_table, seq_lens, cu_seqlens, positions, q_pe);
  kv_append_mla_args a{};
  a.cos_sin = check_angles(cos_sin, q_pe);
  TORCH_CHECK(cos_sin.size(1) == kRope && cos_sin.size(0) > 0, "cos_sin must be [positions, 64]");
  a.c_weight = check_weight(c_weight, "c_weight", kLatent, q_pe, a.c_weight_type);
  const c10::DeviceGuard guard(q_pe.device());
  Tensor out = output_for(q_pe, q_out, "[T, h_q, 64]");
  const Rows rq = rows_of("q_pe", q_pe), rc = rows_of("c_kv", c_kv), rk = rows_of("k_pe", k_pe),
             ro = rows_of("q_out", out);
  check_output(rq, ro, {rc, rk});
  check_cache_apart(kv_cache, "kv_cache", {rq, rc, rk, ro});
  a.q_pe = bf16(q_pe), a.c = bf16(c_kv), a.k_pe = bf16(k_pe), a.q_out = bf16(out);
  a.q_token_stride = rq.st, a.q_head_stride = rq.sh;
  a.c_token_stride = rc.st, a.k_token_stride = rk.st;
  a.q_out_token_stride = ro.st, a.q_out_head_stride = ro.sh;
  a.kv_cache = bf16(kv_cache);
  a.block_table = ix.table, a.seq_lens = ix.lens, a.cu_seqlens = ix.cu, a.rope_positions = ix.rope;
  a.T = ix.T, a.B = ix.B, a.h_q = (int)q_pe.size(1), a.max_blocks = ix.max_blocks;
  a.num_blocks = narrow(kv_cache.size(0), "kv_cache");
  a.block_size = narrow(kv_cache.size(1), "block_size");
  a.table_rows = narrow(cos_sin.size(0), "cos_sin");
  a.interleaved = interleaved;
  a.eps = (float)eps;
  check_launch(kv_append_mla_launch(&a, stream_of(q_pe)), "kv_append_mla_launch");
  return out;
}

Tensor gqa_decode_mxfp4(Tensor q, Tensor kv_cache, Tensor block_table, Tensor seq_lens,
                        double scale, int64_t num_workgroups) {
  TORCH_CHECK(q.is_cuda(), "q must be a CUDA tensor");
  TORCH_CHECK(q.scalar_type() == torch::kBFloat16, "q must be bf16");
  TORCH_CHECK(q.is_contiguous(), "q must be contiguous");
  TORCH_CHECK(q.dim() == 3 && q.size(2) == kDim, "q must be [B, Hq, 128]");
  check_mxfp4(kv_cache, q);
  check_index(block_table, "block_table", 2, q);
  check_index(seq_lens, "seq_lens", 1, q);
  const int64_t B = q.size(0), Hq = q.size(1), Hkv = kv_cache.size(1);
  TORCH_CHECK(Hq > 0 && Hq % Hkv == 0, "Hq must be divisible by Hkv");
  TORCH_CHECK(block_table.size(0) == B, "block_table batch dim must match q");
  TORCH_CHECK(seq_lens.size(0) == B, "seq_lens batch dim must match q");
  TORCH_CHECK(block_table.size(1) > 0, "block_table must have at least one column");
  TORCH_CHECK(num_workgroups >= 0 && num_workgroups <= 65536,
              "num_workgroups must be in [0, 65536] (0: chosen)");
  TORCH_CHECK(std::isfinite(scale), "scale must be finite");
  const int block_size = narrow(kv_cache.size(2) * KV_MXFP4_TILE_TOKENS, "block_size");
  const int max_blocks = narrow(block_table.size(1), "block_table");
  const c10::DeviceGuard guard(q.device());
  Tensor qa = q;
  if (reinterpret_cast<uintptr_t>(q.data_ptr()) % 16 != 0) qa = q.clone();
  Tensor out = torch::empty(q.sizes(), q.options());
  if (B == 0) return out;
  const size_t bytes =
      kv_decode_mxfp4_workspace_bytes(narrow(B, "the batch"), narrow(Hq, "Hq"), narrow(Hkv, "Hkv"),
                                      block_size, max_blocks, (int)num_workgroups);
  Tensor ws;
  if (bytes > 0)
    ws = torch::empty({(int64_t)bytes}, torch::TensorOptions().dtype(torch::kUInt8).device(q.device()));
  check_launch(kv_decode_mxfp4_launch(bf16(qa), kv_cache.data_ptr<uint8_t>(),
                                      block_table.data_ptr<int>(), seq_lens.data_ptr<int>(),
                                      bf16(out), (int)B, (int)Hq, (int)Hkv,
                                      narrow(kv_cache.size(0), "kv_cache"), block_size, max_blocks,
                                      (float)scale, (int)num_workgroups,
                                      bytes > 0 ? ws.data_ptr() : nullptr, bytes, stream_of(q)),
               "kv_decode_mxfp4_launch");
  return out;
}

}  // namespace

PYBIND11_MODULE(TORCH_EXTENSION_NAME, m) {
  const auto none = py::none();
  m.def("kv_append", &kv_append, "append to the paged bf16 caches, with norm and rotation",
        py::arg("q"), py::arg("k"), py::arg("v"), py::arg("k_cache"), py::arg("v_cache"),
        py::arg("block_table"), py::arg("seq_lens"), py::arg("cos_sin") = none,
        py::arg("cu_seqlens") = none, py::arg("positions") = none, py::arg("q_weight") = none,
        py::arg("k_weight") = none, py::arg("eps") = 1e-6, py::arg("interleaved") = false,
        py::arg("q_out") = none);
  m.def("kv_append_mxfp4", &kv_append_mxfp4,
        "append to the paged 4-bit cache, with norm and rotation", py::arg("q"), py::arg("k"),
        py::arg("v"), py::arg("kv_cache"), py::arg("block_table"), py::arg("seq_lens"),
        py::arg("cos_sin") = none, py::arg("cu_seqlens") = none, py::arg("positions") = none,
        py::arg("q_weight") = none, py::arg("k_weight") = none, py::arg("eps") = 1e-6,
        py::arg("interleaved") = false, py::arg("q_out") = none);
  m.def("kv_read_mxfp4", &kv_read_mxfp4, "rows of the paged 4-bit cache as bf16",
        py::arg("kv_cache"), py::arg("block_table"), py::arg("seq_lens"),
        py::arg("cu_seqlens") = none, py::arg("num_tokens") = none);
  m.def("mla_append", &mla_append, "append to the paged MLA cache, with norm and rotation",
        py::arg("q_pe"), py::arg("c_kv"), py::arg("k_pe"), py::arg("kv_cache"),
        py::arg("block_table"), py::arg("seq_lens"), py::arg("cos_sin"),
        py::arg("cu_seqlens") = none, py::arg("positions") = none, py::arg("c_weight") = none,
        py::arg("eps") = 1e-6, py::arg("interleaved") = true, py::arg("q_out") = none);
  m.def("gqa_decode_mxfp4", &gqa_decode_mxfp4, "GQA decode over the paged 4-bit cache",
        py::arg("q"), py::arg("kv_cache"), py::arg("block_table"), py::arg("seq_lens"),
        py::arg("scale"), py::arg("num_workgroups") = 0);
}
