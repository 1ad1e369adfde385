// C entry points of the serving operators (include/xt_b200.h): argument
// checks on the host, then the launchers of serve.h.
#include <cuda_runtime.h>

#include <limits>
#include <string>

#include "../../include/xt_b200.h"
#include "serve.h"

namespace xt {
int record_error(int code, const std::string& msg);  // capi.cpp
int device_error_word(uint32_t** out);               // capi.cpp
uint64_t thread_wait_limit_cycles();                 // capi.cpp
}  // namespace xt

namespace {

using xt::record_error;

constexpr int64_t kMaxInt = std::numeric_limits<int32_t>::max();

bool is_float(int elem) { return elem == XT_ELEM_F32 || elem == XT_ELEM_BF16; }
int64_t size_of(int elem) { return elem == XT_ELEM_F32 ? 4 : elem == XT_ELEM_BF16 ? 2 : 1; }
uint8_t code_of(int elem) {
  return elem == XT_ELEM_F32 ? xt::dev::kF32 : elem == XT_ELEM_BF16 ? xt::dev::kBF16 : xt::dev::kI8;
}
bool aligned(const void* p, int64_t bytes) { return reinterpret_cast<uintptr_t>(p) % bytes == 0; }

int bad(const char* who, const std::string& what) { return record_error(XT_EARGUMENT, std::string(who) + ": " + what); }

int finish(const char* who, cudaError_t e) {
  return e == cudaSuccess ? XT_OK : record_error(XT_ECUDA, std::string(who) + ": " + cudaGetErrorString(e));
}

int check_cache(const char* who, const xt_cache& c) {
  if (!c.k || !c.v || !c.k_scale || !c.v_scale) return bad(who, "null cache array");
  if (c.pages < 1 || c.heads < 1 || c.page < 1 || c.block < 1) return bad(who, "the cache's extents must be positive");
  if (c.heads > 65535 || c.pages > kMaxInt / c.heads) return bad(who, "the cache has too many heads or pages");
  if (c.page > kMaxInt / 256) return bad(who, "the cache's pages are too long");
  if (c.page % c.block != 0) return bad(who, "a cache page must hold whole blocks");
  if (c.dim < 16 || c.dim > 256 || c.dim % 16 != 0) return bad(who, "the cache's dim must be a multiple of 16 up to 256");
  if (!aligned(c.k, 16) || !aligned(c.v, 16)) return bad(who, "the cache is not 16-byte aligned");
  return XT_OK;
}

int check_batch(const char* who, const xt_batch& b, int page) {
  if (b.seqs < 0 || b.tokens < 0 || b.table_width < 0 || b.table_stride < 0) return bad(who, "negative batch extent");
  if (b.seqs > 0 && (!b.starts || !b.lengths || (b.table_width > 0 && !b.table))) return bad(who, "null batch array");
  // positions are 32-bit and a sequence's last tile may reach past its last token
  if (static_cast<int64_t>(b.table_width) * page > kMaxInt - 256) return bad(who, "the page table is too wide");
  return XT_OK;
}

xt::dev::CacheView view(const xt_cache& c) {
  return {c.k, c.v, c.k_scale, c.v_scale, c.pages, c.heads, c.page, c.dim, c.block};
}
xt::dev::BatchView view(const xt_batch& b) {
  return {b.starts, b.lengths, b.table, b.seqs, b.tokens, b.table_width, b.table_stride};
}

xt::dev::AttendArgs attend_args(const xt_cache_attention_args& a, uint32_t* error_word) {
  return {view(a.cache), view(a.batch), a.q, a.out, a.q_token, a.q_head, a.out_token, a.out_head, a.q_heads, a.max_new,
          a.window, a.scale, a.softcap, code_of(a.elem), a.workspace, a.workspace_bytes, error_word,
          xt::thread_wait_limit_cycles()};
}

int check_attention(const char* who, const xt_cache_attention_args* a) {
  if (!a) return bad(who, "null argument");
  if (int st = check_cache(who, a->cache)) return st;
  if (int st = check_batch(who, a->batch, a->cache.page)) return st;
  if (!is_float(a->elem)) return bad(who, "q must be f32 or bf16");
  if (a->q_heads < 1 || a->q_heads % a->cache.heads != 0) return bad(who, "q_heads must be a multiple of the cache's heads");
  if (static_cast<int64_t>(a->batch.tokens) * a->q_heads > kMaxInt - 256) return bad(who, "too many query rows");
  if (a->window < 0 || a->max_new < 0) return bad(who, "negative window or max_new");
  if (!(a->softcap >= 0.0f && a->softcap <= std::numeric_limits<float>::max()))
    return bad(who, "softcap must be 0 or positive, and finite");
  return XT_OK;
}

}  // namespace

extern "C" {

int xt_rms_norm(const xt_rms_norm_args* a, void* stream) {
  const char* who = "xt_rms_norm";
  if (!a) return bad(who, "null argument");
  if (a->rows < 0 || a->cols < 1) return bad(who, "rows must not be negative and cols must be positive");
  if (a->rows > kMaxInt || a->cols > kMaxInt / 2) return bad(who, "too many rows or columns");
  if (!is_float(a->elem) || !is_float(a->weight_elem)) return bad(who, "x and weight must be f32 or bf16");
  if (!is_float(a->y_elem) && a->y_elem != XT_ELEM_I8) return bad(who, "y must be f32, bf16 or i8");
  if (a->rows == 0) return XT_OK;
  if (!a->x || !a->weight || !a->y) return bad(who, "null array");
  if (a->y_elem == XT_ELEM_I8 && !a->scales) return bad(who, "int8 rows need scales");
  const int64_t size = size_of(a->elem);
  if (!aligned(a->x, size) || !aligned(a->residual, size) || !aligned(a->sum, size) ||
      !aligned(a->weight, size_of(a->weight_elem)) || !aligned(a->y, size_of(a->y_elem)) || !aligned(a->scales, 4))
    return bad(who, "an array is not aligned to its element");
  xt::dev::NormArgs n{a->x,    a->residual, a->weight,   a->y,
                      a->sum,  a->scales,   a->rows,     a->cols,
                      a->x_stride, a->residual_stride, a->y_stride, a->sum_stride,
                      code_of(a->elem), code_of(a->weight_elem), code_of(a->y_elem), a->eps};
  return finish(who, xt::dev::launch_rms_norm(n, static_cast<cudaStream_t>(stream)));
}

int xt_rope(const xt_rope_args* a, void* stream) {
  const char* who = "xt_rope";
  if (!a) return bad(who, "null argument");
  if (a->tokens < 0 || a->heads < 0 || a->dim < 2 || a->dim % 2) return bad(who, "dim must be even and positive");
  if (a->rot < 0 || a->rot % 2 || a->rot > a->dim) return bad(who, "rot must be even and at most dim");
  if (a->tokens > kMaxInt || a->heads > kMaxInt / a->dim) return bad(who, "too many tokens or elements of a token");
  if (!is_float(a->elem) || !is_float(a->y_elem) || (a->elem == XT_ELEM_BF16 && a->y_elem != XT_ELEM_BF16))
    return bad(who, "types are f32 to f32 or bf16, or bf16 to bf16");
  if (a->tokens == 0 || a->heads == 0) return XT_OK;
  if (!a->x || !a->y || (a->rot > 0 && (!a->positions || !a->table))) return bad(who, "null array");
  if (!aligned(a->x, size_of(a->elem)) || !aligned(a->y, size_of(a->y_elem)) || !aligned(a->table, 8))
    return bad(who, "an array is not aligned to its element");
  uint32_t* word = nullptr;
  if (int st = xt::device_error_word(&word)) return st;
  xt::dev::RopeArgs r{a->x,      a->y,      a->positions, reinterpret_cast<const float2*>(a->table),
                      a->tokens, a->heads,  a->dim,       a->rot,
                      a->table_rows, a->x_token, a->x_head, a->y_token, a->y_head,
                      code_of(a->elem), code_of(a->y_elem),
                      static_cast<uint8_t>(a->interleaved != 0), static_cast<uint8_t>(a->inverse != 0), word};
  return finish(who, xt::dev::launch_rope(r, static_cast<cudaStream_t>(stream)));
}

int xt_cache_append(const xt_cache_append_args* a, void* stream) {
  const char* who = "xt_cache_append";
  if (!a) return bad(who, "null argument");
  if (int st = check_cache(who, a->cache)) return st;
  if (int st = check_batch(who, a->batch, a->cache.page)) return st;
  if (!is_float(a->elem)) return bad(who, "k and v must be f32 or bf16");
  if (a->rope && (a->rot < 2 || a->rot % 2 || a->rot > a->cache.dim)) return bad(who, "rot must be even, positive and at most dim");
  if (a->rope && a->rope_rows < 1) return bad(who, "the rotation table has no positions");
  if (a->batch.tokens == 0 || a->batch.seqs == 0) return XT_OK;
  if (!a->k || !a->v) return bad(who, "null array");
  if (!aligned(a->k, size_of(a->elem)) || !aligned(a->v, size_of(a->elem)) || !aligned(a->rope, 8))
    return bad(who, "an array is not aligned to its element");
  uint32_t* word = nullptr;
  if (int st = xt::device_error_word(&word)) return st;
  xt::dev::AppendArgs p{view(a->cache), view(a->batch), a->k, a->v, a->k_token, a->k_head, a->v_token, a->v_head,
                        reinterpret_cast<const float2*>(a->rope), a->rope ? a->rot : 0, a->rope_rows,
                        code_of(a->elem), static_cast<uint8_t>(a->interleaved != 0), word};
  return finish(who, xt::dev::launch_cache_append(p, static_cast<cudaStream_t>(stream)));
}

int xt_cache_attention_workspace(const xt_cache_attention_args* a, size_t* out_bytes) {
  const char* who = "xt_cache_attention_workspace";
  if (!out_bytes) return bad(who, "null argument");
  if (int st = check_attention(who, a)) return st;
  *out_bytes = xt::dev::attend_workspace_bytes(attend_args(*a, nullptr));
  return XT_OK;
}

int xt_cache_attention(const xt_cache_attention_args* a, void* stream) {
  const char* who = "xt_cache_attention";
  if (int st = check_attention(who, a)) return st;
  if (a->batch.tokens == 0 || a->batch.seqs == 0) return XT_OK;
  if (!a->q || !a->out) return bad(who, "null array");
  const int64_t bytes = 4 * size_of(a->elem);
  if (!aligned(a->q, bytes) || !aligned(a->out, bytes) || a->q_token % 4 || a->q_head % 4 || a->out_token % 4 || a->out_head % 4)
    return bad(who, "q and out must be aligned to four elements, and their strides multiples of four");
  const size_t need = xt::dev::attend_workspace_bytes(attend_args(*a, nullptr));
  if (need > 0 && (!a->workspace || !aligned(a->workspace, 16) || a->workspace_bytes < need))
    return bad(who, "the workspace must be 16-byte aligned and hold " + std::to_string(need) + " bytes");
  uint32_t* word = nullptr;
  if (int st = xt::device_error_word(&word)) return st;
  return finish(who, xt::dev::launch_cache_attention(attend_args(*a, word), static_cast<cudaStream_t>(stream)));
}

int xt_dequantize(const int8_t* q, const float* scales, void* out, int64_t n, int64_t run, int elem, void* stream) {
  const char* who = "xt_dequantize";
  if (n < 0 || run < 1) return bad(who, "n must not be negative and run must be positive");
  if (!is_float(elem)) return bad(who, "out must be f32 or bf16");
  if (n % run != 0) return bad(who, "n must be whole runs");
  if (n == 0) return XT_OK;
  if (!q || !scales || !out) return bad(who, "null array");
  if (!aligned(q, 16) || !aligned(out, 16) || !aligned(scales, 4)) return bad(who, "q and out must be 16-byte aligned");
  xt::dev::DequantArgs d{q, scales, out, n, run, code_of(elem)};
  return finish(who, xt::dev::launch_dequantize(d, static_cast<cudaStream_t>(stream)));
}

}  // extern "C"
