// C ABI of the decoder operators (declared in include/lunara_b200_decoder.h):
// argument checks on the host, then one launcher each. No entry point allocates.
#include <cuda_runtime.h>

#include <cmath>

#include "decoder.h"
#include "kernels.h"

using namespace lunara;

namespace {

// Sizes that device code holds in 32 bits.
constexpr int64_t kMaxTokens = int64_t{1} << 30;
constexpr int64_t kMaxDim = int64_t{1} << 16;
constexpr int64_t kMaxHeads = 65535;   // grid.y
constexpr int64_t kMaxSlots = int64_t{1} << 31;

bool valid_dtype(int64_t d) { return d == LUNARA_F16 || d == LUNARA_BF16 || d == LUNARA_F32; }
int64_t dtype_bytes(int64_t d) { return d == LUNARA_F32 ? 4 : 2; }
bool aligned(const void* p, uintptr_t n) { return reinterpret_cast<uintptr_t>(p) % n == 0; }

// Each check returns a status; LUNARA_OK leaves the message alone.
int check_rotary(const char* fn, const lunarad_rotary_table& r, int64_t dim) {
  if (r.rot < 0 || r.rot > dim || r.rot % 2 != 0)
    return fail(LUNARA_ERR_INVALID_ARG, "%s: rot %lld is not an even number in [0, %lld]", fn, (long long)r.rot,
                (long long)dim);
  if (r.layout != LUNARAD_ROTARY_HALF && r.layout != LUNARAD_ROTARY_INTERLEAVED)
    return fail(LUNARA_ERR_INVALID_ARG, "%s: bad rotary layout %lld", fn, (long long)r.layout);
  if (r.rot > 0) {
    if (r.table == nullptr || r.positions <= 0)
      return fail(LUNARA_ERR_INVALID_ARG, "%s: rotary table is empty", fn);
    if (!aligned(r.table, 16)) return fail(LUNARA_ERR_INVALID_ARG, "%s: rotary table is not 16-byte aligned", fn);
  }
  return LUNARA_OK;
}

int check_view(const char* fn, const char* name, const lunarad_view& v, int64_t dtype) {
  if (v.data == nullptr) return fail(LUNARA_ERR_INVALID_ARG, "%s: %s is NULL", fn, name);
  if (!aligned(v.data, dtype_bytes(dtype)))
    return fail(LUNARA_ERR_INVALID_ARG, "%s: %s is not aligned to its elements", fn, name);
  return LUNARA_OK;
}

int check_dense(const char* fn, int64_t batch, int64_t heads, int64_t seq, int64_t dim, int64_t dtype) {
  if (!valid_dtype(dtype)) return fail(LUNARA_ERR_INVALID_ARG, "%s: bad dtype %lld", fn, (long long)dtype);
  if (batch < 0 || heads < 0 || seq < 0 || dim < 0) return fail(LUNARA_ERR_INVALID_ARG, "%s: negative shape", fn);
  if (batch > kMaxTokens || seq > kMaxTokens || batch * seq > kMaxTokens || heads > kMaxHeads || dim > kMaxDim)
    return fail(LUNARA_ERR_UNSUPPORTED, "%s: batch * seq above 2^30, heads above 65535 or dim above 65536", fn);
  return LUNARA_OK;
}

int check_positions(const char* fn, const void* positions, int64_t bytes) {
  if (positions == nullptr) return fail(LUNARA_ERR_INVALID_ARG, "%s: positions is NULL", fn);
  if (bytes != 4 && bytes != 8)
    return fail(LUNARA_ERR_INVALID_ARG, "%s: position_bytes %lld is neither 4 nor 8", fn, (long long)bytes);
  if (!aligned(positions, static_cast<uintptr_t>(bytes)))
    return fail(LUNARA_ERR_INVALID_ARG, "%s: positions are not aligned", fn);
  return LUNARA_OK;
}

int check_cache(const char* fn, const lunarad_cache* c) {
  if (c == nullptr) return fail(LUNARA_ERR_INVALID_ARG, "%s: cache is NULL", fn);
  const bool e2m1 = c->kind == LUNARAD_KIND_E2M1;
  if (!e2m1 && !valid_dtype(c->kind)) return fail(LUNARA_ERR_INVALID_ARG, "%s: bad cache kind %lld", fn, (long long)c->kind);
  if (c->num_pages < 0 || c->kv_heads < 1 || c->page_size < 1 || c->dim < 1)
    return fail(LUNARA_ERR_INVALID_ARG, "%s: bad cache shape", fn);
  if (c->num_pages >= kMaxSlots || c->kv_heads > kMaxHeads || c->page_size > (int64_t{1} << 20) || c->dim > kMaxDim)
    return fail(LUNARA_ERR_UNSUPPORTED, "%s: cache too large (pages below 2^31, heads 65535, page size 2^20)", fn);
  if (c->num_pages > 0 && (c->k == nullptr || c->v == nullptr))
    return fail(LUNARA_ERR_INVALID_ARG, "%s: cache pages are NULL", fn);
  if (e2m1) {
    if (c->dim % 16 != 0)
      return fail(LUNARA_ERR_INVALID_ARG, "%s: a 4-bit cache needs a head dim that is a multiple of 16", fn);
    if (c->num_pages > 0 && (c->k_scales == nullptr || c->v_scales == nullptr))
      return fail(LUNARA_ERR_INVALID_ARG, "%s: a 4-bit cache needs scales", fn);
    if (!aligned(c->k, 8) || !aligned(c->v, 8) || c->k_page_stride % 8 || c->k_head_stride % 8 ||
        c->v_page_stride % 8 || c->v_head_stride % 8)
      return fail(LUNARA_ERR_INVALID_ARG, "%s: 4-bit pages need 8-byte alignment", fn);
    if (!(c->k_gain > 0) || !(c->v_gain > 0) || !std::isfinite(1.0f / (float)c->k_gain) ||
        !std::isfinite(1.0f / (float)c->v_gain) || !std::isfinite((float)c->k_gain) || !std::isfinite((float)c->v_gain))
      return fail(LUNARA_ERR_INVALID_ARG, "%s: gains must be positive fp32 numbers", fn);
  } else if (!aligned(c->k, dtype_bytes(c->kind)) || !aligned(c->v, dtype_bytes(c->kind))) {
    return fail(LUNARA_ERR_INVALID_ARG, "%s: cache pages are not aligned to their elements", fn);
  }
  return LUNARA_OK;
}

int check_sequences(const char* fn, const lunarad_sequences& s) {
  if (s.batch < 0 || s.tokens < 0 || s.max_pages < 0) return fail(LUNARA_ERR_INVALID_ARG, "%s: negative sizes", fn);
  if (s.batch > kMaxTokens || s.tokens > kMaxTokens || s.max_pages >= kMaxSlots)
    return fail(LUNARA_ERR_UNSUPPORTED, "%s: more than 2^30 tokens or sequences, or 2^31 pages", fn);
  if (s.batch == 0 || s.tokens == 0) return LUNARA_OK;
  if (s.seq_starts == nullptr || s.seq_lens == nullptr || (s.page_table == nullptr && s.max_pages > 0))
    return fail(LUNARA_ERR_INVALID_ARG, "%s: page_table, seq_starts or seq_lens is NULL", fn);
  if (!aligned(s.seq_starts, 4) || !aligned(s.seq_lens, 4) || !aligned(s.page_table, 4))
    return fail(LUNARA_ERR_INVALID_ARG, "%s: page_table, seq_starts or seq_lens is not aligned", fn);
  if (s.batch > 1 && s.table_stride < s.max_pages)
    return fail(LUNARA_ERR_INVALID_ARG, "%s: page table rows overlap", fn);
  return LUNARA_OK;
}

int check_attention(const char* fn, const lunarad_paged_attention_args* a) {
  int rc = check_cache(fn, a->cache);
  if (rc == LUNARA_OK) rc = check_sequences(fn, a->seqs);
  if (rc != LUNARA_OK) return rc;
  const lunarad_cache& c = *a->cache;
  if (!valid_dtype(a->dtype)) return fail(LUNARA_ERR_INVALID_ARG, "%s: bad dtype %lld", fn, (long long)a->dtype);
  if (c.kind != LUNARAD_KIND_E2M1 && c.kind != a->dtype)
    return fail(LUNARA_ERR_INVALID_ARG, "%s: queries and cache differ in dtype", fn);
  if (a->q_heads < 1 || a->q_heads % c.kv_heads != 0)
    return fail(LUNARA_ERR_INVALID_ARG, "%s: %lld query heads are no multiple of %lld key heads", fn,
                (long long)a->q_heads, (long long)c.kv_heads);
  if (a->q_heads > kMaxHeads || a->seqs.tokens * a->q_heads >= kMaxSlots)
    return fail(LUNARA_ERR_UNSUPPORTED, "%s: more than 65535 heads or 2^31 query rows", fn);
  if (c.dim > 256) return fail(LUNARA_ERR_UNSUPPORTED, "%s: head dim %lld > 256", fn, (long long)c.dim);
  if (c.page_size * a->seqs.max_pages >= kMaxSlots - 4096)   // (the kernels look a batch of keys ahead)
    return fail(LUNARA_ERR_UNSUPPORTED, "%s: page table covers nearly 2^31 positions or more", fn);
  if (a->window < 0 || a->window >= kMaxSlots) return fail(LUNARA_ERR_INVALID_ARG, "%s: bad window", fn);
  if (a->max_q_len < 0) return fail(LUNARA_ERR_INVALID_ARG, "%s: negative max_q_len", fn);
  if (!std::isfinite(a->scale)) return fail(LUNARA_ERR_INVALID_ARG, "%s: scale is not finite", fn);
  // The kernels hold scale * gain, and that times log2(e), in fp32.
  const double factor = a->scale * (c.kind == LUNARAD_KIND_E2M1 ? c.k_gain : 1.0);
  if (!std::isfinite(static_cast<float>(1.4426950408889634 * factor)))
    return fail(LUNARA_ERR_INVALID_ARG, "%s: scale %g (with the keys' gain %g) is not finite in fp32", fn, a->scale, factor);
  return LUNARA_OK;
}

// The arguments with a bare dtype, and whether LUNARAD_ZERO_REST was in it.
template <typename Args>
Args take_zero_rest(const Args& a, bool& zero_rest) {
  Args bare = a;
  zero_rest = (a.dtype & LUNARAD_ZERO_REST) != 0;
  bare.dtype &= ~int64_t{LUNARAD_ZERO_REST};
  return bare;
}

// A call without sequences or without tokens: nothing runs.
int no_work(const char* fn, const lunarad_sequences& s, bool zero_rest) {
  if (zero_rest && s.tokens > 0) return fail(LUNARA_ERR_INVALID_ARG, "%s: rows of no sequence are zeroed beside a sequence's only", fn);
  return ok();
}

cudaStream_t as_stream(void* s) { return static_cast<cudaStream_t>(s); }

}  // namespace

extern "C" {

int lunarad_rotary(const lunarad_rotary_args* a, void* stream) {
  static const char* fn = "lunarad_rotary";
  if (a == nullptr) return fail(LUNARA_ERR_INVALID_ARG, "%s: args is NULL", fn);
  int rc = check_dense(fn, a->batch, a->heads, a->seq, a->dim, a->dtype);
  if (rc == LUNARA_OK) rc = check_rotary(fn, a->rotary, a->dim);
  if (rc != LUNARA_OK) return rc;
  if (a->batch == 0 || a->heads == 0 || a->seq == 0 || a->dim == 0) return ok();
  rc = check_positions(fn, a->positions, a->position_bytes);
  if (rc == LUNARA_OK) rc = check_view(fn, "X", a->x, a->dtype);
  if (rc == LUNARA_OK) rc = check_view(fn, "Y", a->y, a->dtype);
  if (rc != LUNARA_OK) return rc;
  return from_cuda(launch_rotary(*a, as_stream(stream)), fn);
}

int lunarad_qk_norm_rotary(const lunarad_qk_norm_rotary_args* a, void* stream) {
  static const char* fn = "lunarad_qk_norm_rotary";
  if (a == nullptr) return fail(LUNARA_ERR_INVALID_ARG, "%s: args is NULL", fn);
  int rc = check_dense(fn, a->batch, a->q_heads, a->seq, a->dim, a->dtype);
  if (rc == LUNARA_OK) rc = check_dense(fn, a->batch, a->k_heads, a->seq, a->dim, a->dtype);
  if (rc == LUNARA_OK && a->q_heads + a->k_heads > kMaxHeads)
    rc = fail(LUNARA_ERR_UNSUPPORTED, "%s: more than 65535 heads", fn);
  if (rc == LUNARA_OK) rc = check_rotary(fn, a->rotary, a->dim);
  if (rc != LUNARA_OK) return rc;
  if (!(a->eps >= 0) || !std::isfinite(a->eps)) return fail(LUNARA_ERR_INVALID_ARG, "%s: eps must be >= 0", fn);
  if (a->batch == 0 || a->seq == 0 || a->dim == 0 || a->q_heads + a->k_heads == 0) return ok();
  rc = check_positions(fn, a->positions, a->position_bytes);
  if (rc == LUNARA_OK && a->q_heads > 0) rc = check_view(fn, "Q", a->q, a->dtype);
  if (rc == LUNARA_OK && a->q_heads > 0) rc = check_view(fn, "Q's output", a->q_out, a->dtype);
  if (rc == LUNARA_OK && a->k_heads > 0) rc = check_view(fn, "K", a->k, a->dtype);
  if (rc == LUNARA_OK && a->k_heads > 0) rc = check_view(fn, "K's output", a->k_out, a->dtype);
  if (rc != LUNARA_OK) return rc;
  if (!aligned(a->q_weight, dtype_bytes(a->dtype)) || !aligned(a->k_weight, dtype_bytes(a->dtype)))
    return fail(LUNARA_ERR_INVALID_ARG, "%s: weights are not aligned to their elements", fn);
  return from_cuda(launch_qk_norm_rotary(*a, as_stream(stream)), fn);
}

int lunarad_kv_append(const lunarad_kv_append_args* args, void* stream) {
  static const char* fn = "lunarad_kv_append";
  if (args == nullptr) return fail(LUNARA_ERR_INVALID_ARG, "%s: args is NULL", fn);
  bool zero_rest;
  const lunarad_kv_append_args bare = take_zero_rest(*args, zero_rest), *a = &bare;
  int rc = check_cache(fn, a->cache);
  if (rc == LUNARA_OK) rc = check_sequences(fn, a->seqs);
  if (rc != LUNARA_OK) return rc;
  const lunarad_cache& c = *a->cache;
  if (!valid_dtype(a->dtype)) return fail(LUNARA_ERR_INVALID_ARG, "%s: bad dtype %lld", fn, (long long)a->dtype);
  if (c.kind != LUNARAD_KIND_E2M1 && c.kind != a->dtype)
    return fail(LUNARA_ERR_INVALID_ARG, "%s: keys and cache differ in dtype", fn);
  rc = check_rotary(fn, a->rotary, c.dim);
  if (rc != LUNARA_OK) return rc;
  if (a->q_heads < 0) return fail(LUNARA_ERR_INVALID_ARG, "%s: negative q_heads", fn);
  if (a->q_heads + 2 * c.kv_heads > kMaxHeads) return fail(LUNARA_ERR_UNSUPPORTED, "%s: more than 65535 heads", fn);
  if (c.kind == LUNARAD_KIND_E2M1 && c.dim > 512)
    return fail(LUNARA_ERR_UNSUPPORTED, "%s: head dim %lld > 512 into a 4-bit cache", fn, (long long)c.dim);
  if (a->seqs.batch == 0 || a->seqs.tokens == 0) return no_work(fn, a->seqs, zero_rest);
  rc = check_view(fn, "K", a->k, a->dtype);
  if (rc == LUNARA_OK) rc = check_view(fn, "V", a->v, a->dtype);
  if (rc == LUNARA_OK && a->q_heads > 0) rc = check_view(fn, "Q", a->q, a->dtype);
  if (rc == LUNARA_OK && a->q_heads > 0) rc = check_view(fn, "Q's output", a->q_out, a->dtype);
  if (rc != LUNARA_OK) return rc;
  return from_cuda(launch_kv_append(*a, zero_rest, as_stream(stream)), fn);
}

int lunarad_kv_read(const lunarad_kv_read_args* args, void* stream) {
  static const char* fn = "lunarad_kv_read";
  if (args == nullptr) return fail(LUNARA_ERR_INVALID_ARG, "%s: args is NULL", fn);
  bool zero_rest;
  const lunarad_kv_read_args bare = take_zero_rest(*args, zero_rest), *a = &bare;
  int rc = check_cache(fn, a->cache);
  if (rc == LUNARA_OK) rc = check_sequences(fn, a->seqs);
  if (rc != LUNARA_OK) return rc;
  if (!valid_dtype(a->dtype)) return fail(LUNARA_ERR_INVALID_ARG, "%s: bad dtype %lld", fn, (long long)a->dtype);
  if (a->cache->kind != LUNARAD_KIND_E2M1 && a->cache->kind != a->dtype)
    return fail(LUNARA_ERR_INVALID_ARG, "%s: output and cache differ in dtype", fn);
  if (a->seqs.batch == 0 || a->seqs.tokens == 0) return no_work(fn, a->seqs, zero_rest);
  if (a->k_out == nullptr || a->v_out == nullptr) return fail(LUNARA_ERR_INVALID_ARG, "%s: output is NULL", fn);
  if (!aligned(a->k_out, dtype_bytes(a->dtype)) || !aligned(a->v_out, dtype_bytes(a->dtype)))
    return fail(LUNARA_ERR_INVALID_ARG, "%s: output is not aligned to its elements", fn);
  return from_cuda(launch_kv_read(*a, zero_rest, as_stream(stream)), fn);
}

int64_t lunarad_paged_attention_workspace(const lunarad_paged_attention_args* args, int device) {
  static const char* fn = "lunarad_paged_attention_workspace";
  if (args == nullptr) return -fail(LUNARA_ERR_INVALID_ARG, "%s: args is NULL", fn);
  bool zero_rest;
  const lunarad_paged_attention_args bare = take_zero_rest(*args, zero_rest), *a = &bare;
  const int rc = check_attention(fn, a);
  if (rc != LUNARA_OK) return -rc;
  ok();
  if (a->seqs.batch == 0 || a->seqs.tokens == 0) return 0;
  return paged_attention_workspace(*a, device_num_sms_of(device));
}

int lunarad_paged_attention(const lunarad_paged_attention_args* args, void* workspace, int64_t workspace_bytes,
                            void* stream) {
  static const char* fn = "lunarad_paged_attention";
  if (args == nullptr) return fail(LUNARA_ERR_INVALID_ARG, "%s: args is NULL", fn);
  bool zero_rest;
  const lunarad_paged_attention_args bare = take_zero_rest(*args, zero_rest), *a = &bare;
  int rc = check_attention(fn, a);
  if (rc != LUNARA_OK) return rc;
  if (a->seqs.batch == 0 || a->seqs.tokens == 0) return no_work(fn, a->seqs, zero_rest);
  rc = check_view(fn, "Q", a->q, a->dtype);
  if (rc == LUNARA_OK) rc = check_view(fn, "O", a->o, a->dtype);
  if (rc != LUNARA_OK) return rc;
  const int64_t need = paged_attention_workspace(*a, device_num_sms());
  if (need > 0 && (workspace == nullptr || workspace_bytes < need || !aligned(workspace, 16)))
    return fail(LUNARA_ERR_INVALID_ARG, "%s: needs a 16-byte aligned workspace of %lld bytes", fn, (long long)need);
  return from_cuda(launch_paged_attention(*a, zero_rest, workspace, as_stream(stream)), fn);
}

}  // extern "C"
