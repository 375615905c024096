// abi_serving.cu — the extern "C" entry points of the serving operators
// (packed prompts and the paged key-value cache): argument checks, then the
// kernels on the context's stream.  Index arrays live on the device; what
// they hold is checked by the kernels (hs_sync reports it).
#include <math.h>

#include <exception>
#include <string>

#include "../../include/headshot_cuda.h"
#include "hs_abi_ctx.h"
#include "hs_internal.h"

namespace hs {
namespace {

hs_status invalid(const char* name, const char* what) {
  return abi_fail(HS_ERR_INVALID, std::string(name) + ": " + what);
}

bool aligned(const void* p, uintptr_t to) { return (reinterpret_cast<uintptr_t>(p) & (to - 1)) == 0; }

// Checks shared by the three operators.
hs_status check_common(const char* name, hs_ctx* ctx, uint32_t Hq, uint32_t Hkv, uint32_t D, hs_dtype dtype) {
  if (!ctx) return invalid(name, "null context");
  if (dtype != HS_F32 && dtype != HS_F16 && dtype != HS_BF16) return invalid(name, "unknown dtype");
  if (dtype == HS_F32) return abi_fail(HS_ERR_UNSUPPORTED, std::string(name) + ": f16 and bf16 storage only");
  if (D != 64 && D != 128)
    return abi_fail(HS_ERR_UNSUPPORTED, std::string(name) + ": head_dim " + std::to_string(D) +
                                            " unsupported (this build implements 64, 128)");
  if (Hkv == 0) return invalid(name, "Hkv must be positive");
  if (Hq % Hkv != 0) return invalid(name, "Hq must be a multiple of Hkv");
  if (Hq > 1024 || Hkv > 1024) return invalid(name, "more than 1024 heads");
  return HS_OK;
}

// A token stride in elements: 0 selects `heads * D`; others must cover the
// heads and keep rows 16-byte aligned.
hs_status fix_stride(const char* name, const char* which, uint32_t heads, uint32_t D, uint64_t* stride) {
  const uint64_t row = static_cast<uint64_t>(heads) * D;
  if (*stride == 0) *stride = row;
  if (*stride < row || *stride % 8 || *stride > (1ull << 32))
    return invalid(name, (std::string(which) + " stride must be a multiple of 8 elements and cover the heads").c_str());
  return HS_OK;
}

// Head vectors of n tokens, 16-bit elements.
struct Rows {
  const void* at;
  uint64_t n, stride, row;
  uint64_t begin() const { return reinterpret_cast<uintptr_t>(at); }
  uint64_t end() const { return at && n && row ? begin() + 2 * ((n - 1) * stride + row) : begin(); }
};
bool overlap(const Rows& a, const Rows& b) {
  return a.begin() < a.end() && b.begin() < b.end() && a.begin() < b.end() && b.begin() < a.end();
}
// Whether `out` may be written while `in` is read: apart, or the same rows,
// since each of them is read whole before its own place is written.
bool apart_or_same(const Rows& out, const Rows& in) {
  return !overlap(out, in) || (out.at == in.at && (in.stride == out.stride || in.n == 1) && in.row == out.row);
}

hs_status check_cache(const char* name, const void* k_cache, const void* v_cache, const int* block_table,
                      const int* kv_lens, uint32_t n_pages, uint32_t page_size, uint32_t max_pages) {
  if (!k_cache || !v_cache || !block_table || !kv_lens) return invalid(name, "null cache pointer");
  if (!aligned(k_cache, 16) || !aligned(v_cache, 16)) return invalid(name, "cache pointers must be 16-byte aligned");
  if (!aligned(block_table, 4) || !aligned(kv_lens, 4)) return invalid(name, "index pointers must be 4-byte aligned");
  if (page_size == 0) return invalid(name, "page_size must be positive");
  if (n_pages > 0x7fffffffu) return invalid(name, "n_pages does not fit an int");
  if (static_cast<uint64_t>(max_pages) * page_size > 0x7fffffffull)
    return invalid(name, "max_pages * page_size does not fit an int");
  return HS_OK;
}

// No C++ exception crosses the boundary.
template <typename F>
hs_status guarded(const char* name, F&& f) {
  try {
    return f();
  } catch (const std::exception&) {
    try {
      return abi_fail(HS_ERR_OOM, std::string(name) + ": host allocation failed");
    } catch (...) {
      return HS_ERR_OOM;
    }
  }
}

}  // namespace
}  // namespace hs

using namespace hs;

extern "C" {

hs_status hs_kv_append(hs_ctx* ctx, const void* q, const void* k, const void* v, void* q_out, void* k_out,
                       void* k_cache, void* v_cache, const int* block_table, const int* kv_lens, const int* cu_new,
                       uint64_t q_stride, uint64_t k_stride, uint64_t v_stride, uint32_t n_tokens, uint32_t n_seqs,
                       uint32_t Hq, uint32_t Hkv, uint32_t D, uint32_t n_pages, uint32_t page_size,
                       uint32_t max_pages, hs_dtype dtype, const float* rope_sin, const float* rope_cos,
                       uint32_t rope_rows, uint32_t prefix, uint32_t tokens_per_frame) {
  const char* name = "hs_kv_append";
  return guarded(name, [&]() -> hs_status {
    hs_status r = check_common(name, ctx, q ? Hq : Hkv, Hkv, D, dtype);
    if (r != HS_OK) return r;
    if (n_tokens > 0x7fffffffu || n_seqs > 0x7ffffffeu) return invalid(name, "too many tokens or sequences");
    if (!cu_new && n_tokens != n_seqs) return invalid(name, "without cu_new there is one token per sequence");
    if (n_tokens == 0 || n_seqs == 0) return HS_OK;
    if (!k || !v) return invalid(name, "null tensor pointer");
    if ((q != nullptr) != (q_out != nullptr)) return invalid(name, "q and q_out go together");
    if ((rope_sin != nullptr) != (rope_cos != nullptr)) return invalid(name, "rope_sin and rope_cos go together");
    if (!aligned(q, 16) || !aligned(k, 16) || !aligned(v, 16) || !aligned(q_out, 16) || !aligned(k_out, 16) ||
        !aligned(rope_sin, 16) || !aligned(rope_cos, 16))
      return invalid(name, "tensor pointers must be 16-byte aligned");
    if (!aligned(cu_new, 4)) return invalid(name, "index pointers must be 4-byte aligned");
    if (rope_sin && tokens_per_frame) {
      if (prefix > tokens_per_frame) return invalid(name, "prefix > tokens_per_frame");
      if (rope_rows < tokens_per_frame - prefix) return invalid(name, "rope tables shorter than tokens_per_frame - prefix");
    }
    r = check_cache(name, k_cache, v_cache, block_table, kv_lens, n_pages, page_size, max_pages);
    if (r != HS_OK) return r;
    if (q && (r = fix_stride(name, "q", Hq, D, &q_stride)) != HS_OK) return r;
    if ((r = fix_stride(name, "k", Hkv, D, &k_stride)) != HS_OK) return r;
    if ((r = fix_stride(name, "v", Hkv, D, &v_stride)) != HS_OK) return r;
    const uint64_t q_row = static_cast<uint64_t>(Hq) * D, k_row = static_cast<uint64_t>(Hkv) * D;
    const Rows rq{q, n_tokens, q_stride, q_row}, rk{k, n_tokens, k_stride, k_row}, rv{v, n_tokens, v_stride, k_row};
    const Rows rqo{q_out, n_tokens, q_row, q_row}, rko{k_out, n_tokens, k_row, k_row};
    if (q && !apart_or_same(rqo, rq)) return invalid(name, "in place q needs contiguous tokens");
    if (k_out && !apart_or_same(rko, rk)) return invalid(name, "in place k needs contiguous tokens");
    if ((q && (overlap(rqo, rk) || overlap(rqo, rv))) ||
        (k_out && (overlap(rko, rv) || (q && (overlap(rko, rq) || overlap(rko, rqo))))))
      return invalid(name, "q_out and k_out must not overlap other tensors");
    KvAppend a;
    a.q = q;
    a.k = k;
    a.v = v;
    a.q_out = q_out;
    a.k_out = k_out;
    a.q_stride = q_stride;
    a.k_stride = k_stride;
    a.v_stride = v_stride;
    a.cu_new = cu_new;
    a.n_tokens = n_tokens;
    a.q_heads = q ? Hq : 0;
    a.sin_t = rope_sin;
    a.cos_t = rope_cos;
    a.rope_rows = rope_rows;
    a.prefix = prefix;
    a.tokens_per_frame = tokens_per_frame;
    const PagedCache c{k_cache, v_cache, block_table, kv_lens, n_seqs, n_pages, page_size, max_pages, Hkv};
    DeviceGuard guard(ctx->device);
    ProfScope prof(ctx, ctx_stream(ctx), "kv_append");
    const cudaError_t e = launch_kv_append(ctx_stream(ctx), static_cast<int>(dtype), D, a, c, ctx->d_status);
    return e == cudaSuccess ? HS_OK : abi_cuda_fail(e, name);
  });
}

hs_status hs_attention_varlen(hs_ctx* ctx, const void* q, const void* k, const void* v, void* out, uint64_t q_stride,
                              uint64_t k_stride, uint64_t v_stride, const int* cu_q, const int* cu_k,
                              uint32_t total_q, uint32_t total_k, uint32_t n_seqs, uint32_t Hq, uint32_t Hkv,
                              uint32_t D, int causal, hs_dtype dtype, float scale) {
  const char* name = "hs_attention_varlen";
  return guarded(name, [&]() -> hs_status {
    hs_status r = check_common(name, ctx, Hq, Hkv, D, dtype);
    if (r != HS_OK) return r;
    if (Hq / Hkv > 128) return abi_fail(HS_ERR_UNSUPPORTED, std::string(name) + ": more than 128 query heads per key head");
    if (total_q > 0x7fffffffu || total_k > 0x7fffffffu || n_seqs > 0x7ffffffeu)
      return invalid(name, "too many tokens or sequences");
    if (total_q == 0 || n_seqs == 0 || Hq == 0) return HS_OK;
    if (!cu_k && total_k != total_q) return invalid(name, "without cu_k, k and v have as many tokens as q");
    if (!q || !out || !cu_q || (total_k && (!k || !v))) return invalid(name, "null tensor pointer");
    if (!aligned(q, 16) || !aligned(k, 16) || !aligned(v, 16) || !aligned(out, 16))
      return invalid(name, "tensor pointers must be 16-byte aligned");
    if (!aligned(cu_q, 4) || !aligned(cu_k, 4)) return invalid(name, "index pointers must be 4-byte aligned");
    if ((r = fix_stride(name, "q", Hq, D, &q_stride)) != HS_OK) return r;
    if ((r = fix_stride(name, "k", Hkv, D, &k_stride)) != HS_OK) return r;
    if ((r = fix_stride(name, "v", Hkv, D, &v_stride)) != HS_OK) return r;
    const uint64_t q_row = static_cast<uint64_t>(Hq) * D, k_row = static_cast<uint64_t>(Hkv) * D;
    const Rows ro{out, total_q, q_row, q_row};
    if (!apart_or_same(ro, Rows{q, total_q, q_stride, q_row}) || overlap(ro, Rows{k, total_k, k_stride, k_row}) ||
        overlap(ro, Rows{v, total_k, v_stride, k_row}))
      return invalid(name, "out must not overlap k or v, and q only as the same contiguous rows");
    if (!(scale > 0.f) || !isfinite(scale)) scale = 1.0f / sqrtf(static_cast<float>(D));
    VarlenIO io;
    io.q = q;
    io.k = k;
    io.v = v;
    io.out = out;
    io.q_stride = q_stride;
    io.k_stride = k_stride;
    io.v_stride = v_stride;
    io.cu_q = cu_q;
    io.cu_k = cu_k ? cu_k : cu_q;
    io.total_q = total_q;
    io.total_k = total_k;
    io.n_seqs = n_seqs;
    io.q_heads = Hq;
    io.kv_heads = Hkv;
    io.causal = causal != 0;
    DeviceGuard guard(ctx->device);
    std::string err;
    cudaError_t e;
    {
      ProfScope prof(ctx, ctx_stream(ctx), "attention_varlen");
      e = launch_attention_varlen(ctx_stream(ctx), static_cast<int>(dtype), D, io, scale, ctx->d_status,
                                  ctx_timeout_ns(ctx), &err);
    }
    if (e == cudaSuccess) return HS_OK;
    return err.empty() ? abi_cuda_fail(e, name) : invalid(name, err.c_str());
  });
}

hs_status hs_attention_paged_workspace(hs_ctx* ctx, size_t* bytes) {
  const char* name = "hs_attention_paged_workspace";
  return guarded(name, [&]() -> hs_status {
    if (!ctx || !bytes) return invalid(name, "null argument");
    DeviceGuard guard(ctx->device);
    *bytes = attention_paged_workspace_bytes();
    return HS_OK;
  });
}

hs_status hs_attention_paged(hs_ctx* ctx, const void* q, void* out, const void* k_cache, const void* v_cache,
                             const int* block_table, const int* kv_lens, uint64_t q_stride, uint32_t n_seqs,
                             uint32_t Hq, uint32_t Hkv, uint32_t D, uint32_t n_pages, uint32_t page_size,
                             uint32_t max_pages, hs_dtype dtype, float scale, void* workspace,
                             size_t workspace_bytes) {
  const char* name = "hs_attention_paged";
  return guarded(name, [&]() -> hs_status {
    hs_status r = check_common(name, ctx, Hq, Hkv, D, dtype);
    if (r != HS_OK) return r;
    if (static_cast<uint64_t>(n_seqs) * Hq > 0x3fffffffull) return invalid(name, "n_seqs * Hq too large");
    if (n_seqs == 0 || Hq == 0) return HS_OK;
    if (!q || !out) return invalid(name, "null tensor pointer");
    if (!aligned(q, 16) || !aligned(out, 16)) return invalid(name, "tensor pointers must be 16-byte aligned");
    r = check_cache(name, k_cache, v_cache, block_table, kv_lens, n_pages, page_size, max_pages);
    if (r != HS_OK) return r;
    if ((r = fix_stride(name, "q", Hq, D, &q_stride)) != HS_OK) return r;
    const uint64_t q_row = static_cast<uint64_t>(Hq) * D;
    if (!apart_or_same(Rows{out, n_seqs, q_row, q_row}, Rows{q, n_seqs, q_stride, q_row}))
      return invalid(name, "in place q needs contiguous tokens");
    if (!(scale > 0.f) || !isfinite(scale)) scale = 1.0f / sqrtf(static_cast<float>(D));
    DeviceGuard guard(ctx->device);
    if (!workspace || !aligned(workspace, 16) || workspace_bytes < attention_paged_workspace_bytes())
      return invalid(name, "workspace null, misaligned or smaller than hs_attention_paged_workspace says");
    PagedIO io;
    io.q = q;
    io.out = out;
    io.q_stride = q_stride;
    io.q_heads = Hq;
    io.workspace = workspace;
    const PagedCache c{const_cast<void*>(k_cache), const_cast<void*>(v_cache), block_table, kv_lens, n_seqs, n_pages,
                       page_size, max_pages, Hkv};
    ProfScope prof(ctx, ctx_stream(ctx), "attention_paged");
    const cudaError_t e =
        launch_attention_paged(ctx_stream(ctx), static_cast<int>(dtype), D, io, c, scale, ctx->d_status);
    return e == cudaSuccess ? HS_OK : abi_cuda_fail(e, name);
  });
}

}  // extern "C"
