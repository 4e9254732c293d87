// Python entry points of the paged-cache operators (paged.py, speculative.py):
// the checks of the arguments and the launch in C++ on at::Tensor arguments,
// through the C ABI of libqi4_b200.so. A decode step calls them once or twice
// per layer, so their host cost is part of the step.
//
// Errors: ValueError / TypeError before any launch, RuntimeError with the
// library's message when a launch fails. Inputs that the kernels cannot read
// in place (a last dimension with gaps, an unaligned start) are copied; pages
// are never copied.
#include <ATen/ATen.h>
#include <c10/cuda/CUDAGuard.h>
#include <c10/cuda/CUDAStream.h>
#include <torch/extension.h>

#include <string>

#include "../../include/qi4_b200.h"

namespace py = pybind11;

namespace {

using OptTensor = c10::optional<at::Tensor>;

[[noreturn]] void raise_status(int rc, const char* what) {
  char buf[512];
  qi4_last_error(buf, sizeof(buf));
  const char* name = rc == QI4_ERR_ARGUMENT    ? "ARGUMENT"
                     : rc == QI4_ERR_DTYPE     ? "DTYPE"
                     : rc == QI4_ERR_SHAPE     ? "SHAPE"
                     : rc == QI4_ERR_ALIGNMENT ? "ALIGNMENT"
                     : rc == QI4_ERR_LAUNCH    ? "LAUNCH"
                     : rc == QI4_ERR_DEVICE    ? "DEVICE"
                                               : "UNKNOWN";
  const std::string msg = std::string(what) + " failed (" + name + "): " + buf;
  if (rc == QI4_ERR_ARGUMENT || rc == QI4_ERR_SHAPE || rc == QI4_ERR_ALIGNMENT) throw py::value_error(msg);
  if (rc == QI4_ERR_DTYPE) throw py::type_error(msg);
  throw std::runtime_error(msg);
}

void want(bool ok, const char* message) {
  if (!ok) throw py::value_error(message);
}
void want_type(bool ok, const char* message) {
  if (!ok) throw py::type_error(message);
}

bool aligned16(const at::Tensor& t) { return reinterpret_cast<uintptr_t>(t.data_ptr()) % 16 == 0; }

// [T, heads, D] as the kernels read it: D contiguous, the start 16-byte
// aligned, strides in whole 16 bytes and not zero (an expanded tensor); copied
// otherwise.
at::Tensor rows(const at::Tensor& t) {
  auto fits = [&](int64_t dim) { return t.stride(dim) % 8 == 0 && (t.stride(dim) > 0 || t.size(dim) == 1); };
  if (t.stride(2) == 1 && aligned16(t) && fits(0) && fits(1)) return t;
  const at::Tensor c = t.contiguous();
  return aligned16(c) ? c : c.clone();
}

at::Tensor dense(const at::Tensor& t) { return t.is_contiguous() ? t : t.contiguous(); }

const int32_t* ints(const OptTensor& t, at::Tensor& keep) {
  if (!t) return nullptr;
  keep = dense(*t);
  return static_cast<const int32_t*>(keep.data_ptr());
}

void check_ints(const at::Tensor& t, int64_t n, const at::Tensor& like, const char* message) {
  want_type(t.scalar_type() == at::kInt, "lengths, cu_tokens, positions, block tables and counts must be int32 tensors");
  want(t.dim() == 1 && t.size(0) == n, message);
  want(t.is_cuda() && t.get_device() == like.get_device(), "all tensors must be on one CUDA device");
}

// The pages and their table as the C ABI takes them; `table` keeps a copy alive where one was needed.
qi4_paged_kv pages_of(const at::Tensor& k, const at::Tensor& v, const at::Tensor& block_table, at::Tensor& table) {
  want(k.dim() == 4 && v.sizes() == k.sizes(), "k_cache and v_cache must be [pages, kv_heads, page_size, head_dim]");
  want_type((k.scalar_type() == at::kBFloat16 || k.scalar_type() == at::kHalf) && v.scalar_type() == k.scalar_type(),
            "the caches must both be BF16 or both FP16");
  want(k.is_cuda() && v.is_cuda() && block_table.is_cuda() && v.get_device() == k.get_device() &&
           block_table.get_device() == k.get_device(),
       "all tensors must be on one CUDA device");
  want_type(block_table.scalar_type() == at::kInt,
            "lengths, cu_tokens, positions, block tables and counts must be int32 tensors");
  want(block_table.dim() == 2 && block_table.size(0) > 0 && block_table.size(1) > 0,
       "block_table must be [batch, pages of a sequence]");
  for (int64_t i = 0; i < 4; ++i)
    want(k.size(i) > 0 && k.size(i) < (int64_t(1) << 31) && (k.size(i) == 1 || k.stride(i) == v.stride(i)),
         "k_cache and v_cache must have the same strides");
  want(k.stride(3) == 1 || k.size(3) == 1, "the caches' last dimension must be contiguous");
  table = block_table.stride(1) == 1 || block_table.size(1) == 1 ? block_table : block_table.contiguous();
  qi4_paged_kv kv;
  kv.k = k.data_ptr();
  kv.v = v.data_ptr();
  kv.block_table = static_cast<const int32_t*>(table.data_ptr());
  kv.table_stride = table.size(0) > 1 ? table.stride(0) : 0;
  // (The stride of a dimension of size 1 is not used.)
  kv.page_stride = k.size(0) > 1 ? k.stride(0) : 0;
  kv.head_stride = k.size(1) > 1 ? k.stride(1) : 0;
  kv.slot_stride = k.size(2) > 1 ? k.stride(2) : k.size(3);
  kv.dtype = k.scalar_type() == at::kHalf ? QI4_DTYPE_F16 : QI4_DTYPE_BF16;
  kv.pages = static_cast<int32_t>(k.size(0));
  kv.kv_heads = static_cast<int32_t>(k.size(1));
  kv.page_size = static_cast<int32_t>(k.size(2));
  kv.head_dim = static_cast<int32_t>(k.size(3));
  kv.table_width = static_cast<int32_t>(table.size(1));
  return kv;
}

void check_rows(const at::Tensor& t, int64_t T, const at::Tensor& cache, const char* message) {
  want(t.dim() == 3 && t.size(0) == T && t.size(2) == cache.size(3), message);
  want_type(t.scalar_type() == cache.scalar_type(), "q, k and v must have the caches' type");
  want(t.is_cuda() && t.get_device() == cache.get_device(), "all tensors must be on one CUDA device");
}

void check_batch(const OptTensor& cu_tokens, const at::Tensor& lengths, int64_t T, int64_t B, const at::Tensor& like) {
  check_ints(lengths, B, like, "lengths must have one entry per row of block_table");
  if (cu_tokens)
    check_ints(*cu_tokens, B + 1, like, "cu_tokens must have one entry more than block_table has rows");
  else
    want(T % B == 0, "without cu_tokens every sequence must have the same number of tokens");
}

at::Tensor rope_paged_append(const at::Tensor& q, const at::Tensor& k, const at::Tensor& v, const at::Tensor& k_cache,
                             const at::Tensor& v_cache, const at::Tensor& block_table, const at::Tensor& lengths,
                             const OptTensor& cos, const OptTensor& sin, const OptTensor& cu_tokens,
                             const OptTensor& positions, bool interleaved, const OptTensor& q_out) {
  at::Tensor table, keep[3];
  const qi4_paged_kv kv = pages_of(k_cache, v_cache, block_table, table);
  want(k.dim() == 3, "k must be [tokens, kv_heads, head_dim]");
  const int64_t T = k.size(0), B = block_table.size(0);
  check_rows(q, T, k_cache, "q must be [tokens, query heads, head_dim] with k's tokens and the caches' head_dim");
  check_rows(k, T, k_cache, "k must be [tokens, kv_heads, head_dim] with the caches' head_dim");
  check_rows(v, T, k_cache, "v must be [tokens, kv_heads, head_dim] with k's tokens and the caches' head_dim");
  want(k.size(1) == kv.kv_heads && v.size(1) == kv.kv_heads, "k and v must have the caches' kv_heads");
  check_batch(cu_tokens, lengths, T, B, k_cache);
  want(cos.has_value() == sin.has_value(), "cos and sin must be given together");
  at::Tensor c, s;
  if (cos) {
    want(cos->dim() == 2 && sin->sizes() == cos->sizes(), "cos and sin must be [rows, rotary dims / 2]");
    want_type(cos->scalar_type() == at::kFloat && sin->scalar_type() == at::kFloat, "cos and sin must be FP32");
    want(cos->is_cuda() && sin->is_cuda() && cos->get_device() == k.get_device() && sin->get_device() == k.get_device(),
         "all tensors must be on one CUDA device");
    c = dense(*cos);
    s = dense(*sin);
    if (c.numel() && !aligned16(c)) c = c.clone();
    if (s.numel() && !aligned16(s)) s = s.clone();
  }
  if (positions) check_ints(*positions, T, k_cache, "positions must have one entry per token");
  const at::Tensor q2 = rows(q), k2 = rows(k), v2 = rows(v);
  at::Tensor out;
  if (q_out) {
    out = *q_out;
    check_rows(out, T, k_cache, "q_out must have q's shape");
    want(out.size(1) == q.size(1), "q_out must have q's shape");
    want(out.numel() == 0 || (out.stride(2) == 1 && aligned16(out) && out.stride(0) % 8 == 0 && out.stride(1) % 8 == 0),
         "q_out must be 16-byte aligned with head_dim contiguous and strides that are multiples of 8");
  } else {
    out = at::empty({T, q.size(1), q.size(2)}, q.options());
  }
  if (T == 0) return out;
  const c10::cuda::CUDAGuard guard(k.device());
  const int rc = qi4_rope_paged_append(
      &kv, q2.data_ptr(), q2.stride(0), q2.stride(1), k2.data_ptr(), k2.stride(0), k2.stride(1), v2.data_ptr(),
      v2.stride(0), v2.stride(1), out.data_ptr(), out.stride(0), out.stride(1), T, B, q.size(1),
      ints(cu_tokens, keep[0]), ints(lengths, keep[1]), ints(positions, keep[2]),
      cos ? static_cast<const float*>(c.data_ptr()) : nullptr, cos ? static_cast<const float*>(s.data_ptr()) : nullptr,
      cos ? c.size(0) : 0, cos ? static_cast<int>(2 * c.size(1)) : 0, interleaved ? 1 : 0,
      c10::cuda::getCurrentCUDAStream(k.get_device()).stream());
  if (rc) raise_status(rc, "qi4_rope_paged_append");
  return out;
}

at::Tensor attend(const at::Tensor& q, const at::Tensor& k_cache, const at::Tensor& v_cache,
                  const OptTensor& prefix_table, int64_t prefix_length, const at::Tensor& block_table,
                  const at::Tensor& lengths, const OptTensor& cu_tokens, c10::optional<int64_t> max_tokens,
                  c10::optional<double> scale, bool causal, const OptTensor& out_, const OptTensor& workspace) {
  at::Tensor table, prefix, keep[2];
  const qi4_paged_kv kv = pages_of(k_cache, v_cache, block_table, table);
  want(q.dim() == 3, "q must be [tokens, query heads, head_dim]");
  const int64_t T = q.size(0), B = block_table.size(0), Hq = q.size(1);
  check_rows(q, T, k_cache, "q must be [tokens, query heads, head_dim] with the caches' head_dim");
  want(Hq > 0 && Hq % kv.kv_heads == 0, "the query heads must be a multiple of the caches' kv_heads");
  check_batch(cu_tokens, lengths, T, B, k_cache);
  want(!max_tokens || *max_tokens >= 0, "max_tokens must not be negative");
  if (prefix_table) {
    check_ints(*prefix_table, prefix_table->dim() == 1 ? prefix_table->size(0) : -1, k_cache,
               "prefix_table must be one row of pages");
    want(prefix_length >= 0 && prefix_length <= prefix_table->size(0) * kv.page_size,
         "prefix_length must lie within the pages of prefix_table");
    prefix = dense(*prefix_table);
  }
  const at::Tensor q2 = rows(q);
  at::Tensor out;
  if (out_) {
    out = *out_;
    check_rows(out, T, k_cache, "out must have q's shape");
    want(out.size(1) == Hq && out.is_contiguous() && (T == 0 || reinterpret_cast<uintptr_t>(out.data_ptr()) % 32 == 0),
         "out must have q's shape, contiguous and 32-byte aligned");
  } else {
    out = at::empty({T, Hq, q.size(2)}, q.options());
  }
  if (T == 0) return out;
  const c10::cuda::CUDAGuard guard(q.device());
  const int64_t most = max_tokens ? *max_tokens : 0;
  at::Tensor ws;
  if (workspace) {
    ws = *workspace;
    want_type(ws.scalar_type() == at::kByte, "workspace must be a uint8 tensor");
    want(ws.is_cuda() && ws.get_device() == q.get_device() && ws.is_contiguous(),
         "workspace must be contiguous, on the tensors' device");
  } else {
    const size_t bytes = qi4_paged_attention_workspace(T, Hq, kv.kv_heads, kv.head_dim, cu_tokens ? most : T / B,
                                                       prefix_length > 0);
    ws = at::empty({static_cast<int64_t>(bytes)}, q.options().dtype(at::kByte));
  }
  const cudaStream_t stream = c10::cuda::getCurrentCUDAStream(q.get_device()).stream();
  const float sc = static_cast<float>(scale ? *scale : 1.0 / std::sqrt(static_cast<double>(q.size(2))));
  const int rc =
      prefix_table
          ? qi4_shared_prefix_attention(&kv, q2.data_ptr(), q2.stride(0), q2.stride(1), out.data_ptr(), T, B, Hq,
                                        static_cast<const int32_t*>(prefix.data_ptr()), prefix.size(0), prefix_length,
                                        ints(cu_tokens, keep[0]), ints(lengths, keep[1]), most, sc, ws.data_ptr(),
                                        ws.numel(), stream)
          : qi4_paged_attention(&kv, q2.data_ptr(), q2.stride(0), q2.stride(1), out.data_ptr(), T, B, Hq,
                                ints(cu_tokens, keep[0]), ints(lengths, keep[1]), most, sc, causal ? 1 : 0,
                                ws.data_ptr(), ws.numel(), stream);
  if (rc) raise_status(rc, prefix_table ? "qi4_shared_prefix_attention" : "qi4_paged_attention");
  return out;
}

py::tuple verify_draft(const at::Tensor& draft_tokens, const at::Tensor& target, const at::Tensor& uniforms,
                       const OptTensor& draft, const OptTensor& counts) {
  want(target.dim() == 3 && target.size(1) >= 1 && target.size(2) >= 1,
       "target_probs must be [batch, drafts + 1, vocabulary]");
  const int64_t B = target.size(0), K = target.size(1) - 1, V = target.size(2);
  const at::ScalarType t = target.scalar_type();
  want_type(t == at::kFloat || t == at::kBFloat16 || t == at::kHalf, "probabilities must be FP32, BF16 or FP16");
  want_type(draft_tokens.scalar_type() == at::kLong, "draft_tokens must be int64");
  want(draft_tokens.dim() == 2 && draft_tokens.size(0) == B && draft_tokens.size(1) == K,
       "draft_tokens must be [batch, drafts]");
  want_type(uniforms.scalar_type() == at::kFloat, "uniforms must be FP32");
  want(uniforms.dim() == 2 && uniforms.size(0) == B && uniforms.size(1) == K + 1,
       "uniforms must be [batch, drafts + 1]");
  if (draft) {
    want_type(draft->scalar_type() == t, "draft_probs must have target_probs' type");
    want(draft->dim() == 3 && draft->size(0) == B && draft->size(1) == K && draft->size(2) == V,
         "draft_probs must be [batch, drafts, vocabulary]");
  }
  want(target.is_cuda(), "all tensors must be on one CUDA device");
  for (const at::Tensor* x : {&draft_tokens, &uniforms, draft ? &*draft : &target})
    want(x->is_cuda() && x->get_device() == target.get_device(), "all tensors must be on one CUDA device");
  if (counts) check_ints(*counts, B, target, "draft_counts must have one entry per sequence");
  at::Tensor keep;
  const at::Tensor p = target.stride(2) == 1 || V == 1 ? target : target.contiguous();
  const at::Tensor q = !draft ? at::Tensor() : draft->stride(2) == 1 || V == 1 ? *draft : draft->contiguous();
  const at::Tensor d = dense(draft_tokens), u = dense(uniforms);
  at::Tensor out = at::empty({B, K + 1}, draft_tokens.options());
  at::Tensor accepted = at::empty({B}, draft_tokens.options().dtype(at::kInt));
  if (B == 0) return py::make_tuple(out, accepted);
  const c10::cuda::CUDAGuard guard(target.device());
  const int rc = qi4_verify_draft(
      static_cast<const int64_t*>(d.data_ptr()), p.data_ptr(), p.stride(0), p.stride(1),
      draft && K > 0 ? q.data_ptr() : nullptr, draft ? q.stride(0) : 0, draft ? q.stride(1) : 0,
      t == at::kFloat ? QI4_DTYPE_F32 : t == at::kHalf ? QI4_DTYPE_F16 : QI4_DTYPE_BF16,
      static_cast<const float*>(u.data_ptr()), ints(counts, keep), B, K, V, static_cast<int64_t*>(out.data_ptr()),
      static_cast<int32_t*>(accepted.data_ptr()), c10::cuda::getCurrentCUDAStream(target.get_device()).stream());
  if (rc) raise_status(rc, "qi4_verify_draft");
  return py::make_tuple(out, accepted);
}

}  // namespace

void bind_paged(py::module_& m) {
  m.def("rope_paged_append", &rope_paged_append, "Rotary positions and append to a paged cache (b200_rope_paged_append)");
  m.def("attend", &attend, "Paged and shared-prefix attention (b200_paged_attention, b200_shared_prefix_attention)");
  m.def("verify_draft", &verify_draft, "Draft verification (b200_verify_draft)");
}
