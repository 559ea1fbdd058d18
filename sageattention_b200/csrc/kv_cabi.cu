// extern "C" boundary of the 4-bit key/value cache (declared in include/sage3_b200.h): argument checks and launches.
#include "../../include/sage3_b200.h"

#include <cuda_runtime.h>

#include "kernels.h"

namespace {

inline bool aligned(const void* p, size_t n) { return (reinterpret_cast<uintptr_t>(p) & (n - 1)) == 0; }

int check_cache(const sage3_kv_cache* c) {
  if (c == nullptr || c->data == nullptr || !aligned(c->data, 16) || !aligned(c->k_offset, 16)) return SAGE3_ERR_ARGUMENT;
  if (c->num_pages <= 0 || c->num_kv_heads <= 0) return SAGE3_ERR_ARGUMENT;
  if (c->page_size != 16 && c->page_size != 32 && c->page_size != 64 && c->page_size != 128) return SAGE3_ERR_UNSUPPORTED;
  if (c->head_dim <= 0 || c->head_dim % 8 != 0 || c->head_dim > c->head_dim_stored) return SAGE3_ERR_UNSUPPORTED;
  if (c->head_dim_stored != 64 && c->head_dim_stored != 128) return SAGE3_ERR_UNSUPPORTED;
  return SAGE3_OK;
}

// of a page size that check_cache has let through
inline int shift_of(int page_size) { return page_size == 16 ? 4 : page_size == 32 ? 5 : page_size == 64 ? 6 : 7; }

// rows of 16-byte vectors
int check_rows(const sage3_tensor& t) {
  if (!aligned(t.ptr, 16) || t.stride_b % 8 || t.stride_h % 8 || t.stride_n % 8) return SAGE3_ERR_ARGUMENT;
  return SAGE3_OK;
}

sage3::KvRows rows_of(const sage3_tensor& t) { return sage3::KvRows{t.ptr, t.stride_b, t.stride_h, t.stride_n}; }

// without offsets every sequence has one token
inline int longest_q(const sage3_kv_attention_args* a) { return a->cu_seqlens_q != nullptr ? a->max_seqlen_q : 1; }

inline bool takes_prefill(const sage3_kv_attention_args* a) {
  return sage3::kv_prefill_takes(a->Hq, a->cache->num_kv_heads, a->cache->head_dim_stored, longest_q(a));
}

int check_attention(const sage3_kv_attention_args* a) {
  if (a == nullptr) return SAGE3_ERR_ARGUMENT;
  if (int st = check_cache(a->cache)) return st;
  if (a->B <= 0 || a->Hq <= 0 || a->max_seqlen_q <= 0 || a->max_seqlen_k <= 0 || a->total_q < 0 || a->columns <= 0) return SAGE3_ERR_ARGUMENT;
  if (a->Hq % a->cache->num_kv_heads != 0) return SAGE3_ERR_UNSUPPORTED;
  const int64_t rows = (int64_t)longest_q(a) * (a->Hq / a->cache->num_kv_heads);
  if (rows >= (1ll << 30) || a->max_seqlen_k > (1 << 30)) return SAGE3_ERR_UNSUPPORTED;
  if (takes_prefill(a) ? !sage3::kv_prefill_fits(a->B, a->Hq, a->cache->num_kv_heads, longest_q(a))
                       : !sage3::kv_decode_fits(a->B, a->Hq, a->cache->num_kv_heads, longest_q(a), a->max_seqlen_k))
    return SAGE3_ERR_UNSUPPORTED;
  return SAGE3_OK;
}

}  // namespace

extern "C" {

int sage3_kv_block_tables(const sage3_kv_tables_args* a, void* stream) {
  if (a == nullptr || a->B <= 0 || a->columns <= 0 || a->num_free < 0 || a->num_tokens < 0 || a->row_stride < a->columns) return SAGE3_ERR_ARGUMENT;
  if (!a->lens_before || !a->lens_new || !a->block_table || !a->kv_lens || !a->cu_seqlens_q || !a->pages_taken) return SAGE3_ERR_ARGUMENT;
  if ((a->num_free > 0 && !a->free_pages) || (a->num_tokens > 0 && (!a->positions || !a->slots))) return SAGE3_ERR_ARGUMENT;
  if (a->page_size != 16 && a->page_size != 32 && a->page_size != 64 && a->page_size != 128) return SAGE3_ERR_UNSUPPORTED;
  if (a->B > sage3::kTableMost) return SAGE3_ERR_UNSUPPORTED;
  sage3::KvTablesArgs k{};
  k.before = a->lens_before; k.fresh = a->lens_new; k.free_pages = a->free_pages;
  k.table = a->block_table; k.table_stride = a->row_stride;
  k.B = a->B; k.cols = a->columns; k.num_free = a->num_free; k.page_size = a->page_size; k.num_tokens = a->num_tokens;
  k.kv_lens = a->kv_lens; k.cu = a->cu_seqlens_q; k.positions = a->positions; k.slots = a->slots; k.taken = a->pages_taken;
  cudaError_t e = sage3::launch_block_tables(k, (cudaStream_t)stream);
  return e == cudaSuccess ? SAGE3_OK : sage3::cuda_fail(e);
}

int sage3_kv_tokens(const sage3_kv_tokens_args* a, void* stream) {
  if (a == nullptr || a->B < 0 || a->N < 0 || a->Hq < 0 || a->Hkv <= 0) return SAGE3_ERR_ARGUMENT;
  if (a->D <= 0 || a->D > 128 || a->D % 8 != 0) return SAGE3_ERR_UNSUPPORTED;
  if (a->k.ptr == nullptr || (a->Hq > 0 && (a->q.ptr == nullptr || a->q_out.ptr == nullptr))) return SAGE3_ERR_ARGUMENT;
  if (a->k_out.ptr == nullptr && a->cache == nullptr) return SAGE3_ERR_ARGUMENT;
  for (const sage3_tensor* t : {&a->q, &a->k, &a->v, &a->q_out, &a->k_out})
    if (int st = check_rows(*t)) return st;
  if (!aligned(a->q_weight, 16) || !aligned(a->k_weight, 16) || !aligned(a->cos, 16) || !aligned(a->sin, 16)) return SAGE3_ERR_ARGUMENT;
  if (a->rot_dim < 0 || a->rot_dim > a->D || a->rot_dim % 8 != 0) return SAGE3_ERR_UNSUPPORTED;
  if (a->rot_dim > 0 && (!a->cos || !a->sin || a->places <= 0)) return SAGE3_ERR_ARGUMENT;
  if ((a->q_weight || a->k_weight) && !(a->eps >= 0.f)) return SAGE3_ERR_ARGUMENT;
  sage3::KvTokensArgs k{};
  k.DS = a->D <= 64 ? 64 : 128;
  if (a->cache != nullptr) {
    if (int st = check_cache(a->cache)) return st;
    if (a->v.ptr == nullptr || a->slots == nullptr) return SAGE3_ERR_ARGUMENT;
    if (a->cache->num_kv_heads != a->Hkv || a->cache->head_dim != a->D) return SAGE3_ERR_ARGUMENT;
    k.DS = a->cache->head_dim_stored;
    k.data = (uint8_t*)a->cache->data; k.slots = a->slots; k.k_offset = a->cache->k_offset;
    k.page_size = a->cache->page_size; k.page_shift = shift_of(a->cache->page_size); k.num_slots = a->cache->num_pages * a->cache->page_size;
    k.v = a->v.ptr;
  }
  if ((int64_t)a->B * a->N >= (1ll << 31) - 64 || (int64_t)a->Hq + 2ll * a->Hkv > 65535 * 8) return SAGE3_ERR_UNSUPPORTED;
  if ((int64_t)a->B * a->N == 0) return SAGE3_OK;
  k.q = rows_of(a->q); k.k = rows_of(a->k); k.vr = rows_of(a->v); k.q_out = rows_of(a->q_out); k.k_out = rows_of(a->k_out);
  k.B = a->B; k.N = a->N; k.Hq = a->Hq; k.Hkv = a->Hkv; k.D = a->D;
  k.weight[0] = a->q_weight; k.weight[1] = a->k_weight;
  k.eps = a->eps; k.inv_d = 1.0f / (float)a->D;
  k.cos = a->cos; k.sin = a->sin; k.places = a->places; k.rot = a->rot_dim; k.adjacent = a->adjacent_pairs != 0;
  k.positions = a->positions; k.positions64 = a->positions_int64 != 0;
  // keys and values that only go to the cache have a kernel of their own
  const bool as_is = a->Hq == 0 && a->B == 1 && a->k_out.ptr == nullptr && a->k_weight == nullptr && a->rot_dim == 0;
  if (as_is && a->Hkv > 32767) return SAGE3_ERR_UNSUPPORTED;
  cudaError_t e = as_is ? sage3::launch_kv_append(k, (cudaStream_t)stream) : sage3::launch_kv_tokens(k, (cudaStream_t)stream);
  return e == cudaSuccess ? SAGE3_OK : sage3::cuda_fail(e);
}

int sage3_kv_read(const sage3_kv_cache* cache, const int64_t* slots, int64_t T, void* k, void* v, void* stream) {
  if (int st = check_cache(cache)) return st;
  if (T < 0) return SAGE3_ERR_ARGUMENT;
  if (T == 0) return SAGE3_OK;
  if (T >= (1ll << 31) - 64 || cache->num_kv_heads > 32767) return SAGE3_ERR_UNSUPPORTED;      // (a CTA counts up to 63 tokens beyond the last)
  if (!slots || !k || !v || !aligned(k, 16) || !aligned(v, 16)) return SAGE3_ERR_ARGUMENT;
  sage3::KvReadArgs a{};
  a.data = (const uint8_t*)cache->data; a.slots = slots; a.T = T; a.num_slots = cache->num_pages * cache->page_size;
  a.Hkv = cache->num_kv_heads; a.D = cache->head_dim; a.DS = cache->head_dim_stored; a.page_shift = shift_of(cache->page_size);
  a.k_offset = cache->k_offset; a.k = k; a.v = v;
  cudaError_t e = sage3::launch_kv_read(a, (cudaStream_t)stream);
  return e == cudaSuccess ? SAGE3_OK : sage3::cuda_fail(e);
}

int sage3_kv_attention_workspace(const sage3_kv_attention_args* a, size_t* bytes) {
  if (int st = check_attention(a)) return st;
  if (bytes == nullptr) return SAGE3_ERR_ARGUMENT;
  int sms;
  if (cudaError_t e = sage3::sm_count(&sms); e != cudaSuccess) return sage3::cuda_fail(e);
  const auto size = takes_prefill(a) ? sage3::kv_prefill_workspace : sage3::kv_decode_workspace;
  *bytes = size(a->B, a->Hq, a->cache->num_kv_heads, a->cache->head_dim_stored, longest_q(a), a->max_seqlen_k, sms);
  return SAGE3_OK;
}

int sage3_kv_attention(const sage3_kv_attention_args* a, void* stream) {
  if (int st = check_attention(a)) return st;
  if (a->total_q == 0) return SAGE3_OK;
  if (!a->q || !a->out || !a->kv_lens || !a->block_table || (!a->workspace && a->workspace_bytes > 0)) return SAGE3_ERR_ARGUMENT;
  if (!aligned(a->q, 16) || !aligned(a->out, 16) || !aligned(a->workspace, 256)) return SAGE3_ERR_ARGUMENT;
  if (a->q_stride_n % 8 || a->q_stride_h % 8 || a->out_stride_n % 8 || a->out_stride_h % 8) return SAGE3_ERR_ARGUMENT;
  if (a->cu_seqlens_q == nullptr && a->total_q < a->B) return SAGE3_ERR_ARGUMENT;
  size_t need;
  if (int st = sage3_kv_attention_workspace(a, &need)) return st;
  if (a->workspace_bytes < need) return SAGE3_ERR_ARGUMENT;
  const sage3_kv_cache& c = *a->cache;
  sage3::KvAttnArgs k{};
  k.data = (const uint8_t*)c.data; k.num_pages = c.num_pages; k.Hkv = c.num_kv_heads; k.page_size = c.page_size;
  k.D = c.head_dim; k.DS = c.head_dim_stored; k.k_offset = c.k_offset;
  k.q = a->q; k.q_sn = a->q_stride_n; k.q_sh = a->q_stride_h;
  k.out = a->out; k.o_sn = a->out_stride_n; k.o_sh = a->out_stride_h; k.lse = a->lse;
  k.cu_q = a->cu_seqlens_q; k.kv_lens = a->kv_lens; k.table = a->block_table; k.table_stride = a->row_stride;
  k.B = a->B; k.Hq = a->Hq; k.cols = a->columns; k.tokens = a->total_q;
  k.max_q = longest_q(a); k.max_k = a->max_seqlen_k; k.causal = a->is_causal != 0;
  k.sm_scale = a->sm_scale > 0.f ? a->sm_scale : 1.0f / sqrtf((float)c.head_dim);
  k.workspace = a->workspace; k.status = a->device_status;
  cudaError_t e = cudaSuccess;
  if (a->device_status != nullptr) e = cudaMemsetAsync(a->device_status, 0, sizeof(int32_t), (cudaStream_t)stream);
  if (e == cudaSuccess) e = takes_prefill(a) ? sage3::launch_kv_prefill(k, (cudaStream_t)stream) : sage3::launch_kv_decode(k, (cudaStream_t)stream);
  return e == cudaSuccess ? SAGE3_OK : sage3::cuda_fail(e);
}

}  // extern "C"
