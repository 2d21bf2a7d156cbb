// Attention over the paged key/value cache.
//
//   O[t] = sum_j softmax_j(scale q_t . k_j) v_j   over the keys j that the
//   query's position sees: j <= p, and with a window j > p - window.
//
// Simple kernel (any dtype and head dimension up to 256): one warp per query
// token and head, lanes over the head dimension, one key after the other with
// the running maximum and sum of the softmax in fp32.
#include "kernels.h"
#include "paged.cuh"

namespace lunara {
namespace {

struct PagedParams {
  const void* q;
  void* o;
  int64_t q_head, q_tok, o_head, o_tok;   // strides
  const void* k;
  const void* v;
  const void* ks;
  const void* vs;
  int64_t k_page, k_head, v_page, v_head, ks_page, ks_head, vs_page, vs_head;
  int num_pages, kv_heads, page_size, dim, q_heads, group;
  Seqs seqs;
  int window;
  float scale;   // softmax scale times the keys' gain
  float v_gain;
  unsigned int* err;
};

// The keys that a position sees, as [lo, hi), cut to the page table.
__device__ __forceinline__ void visible(const PagedParams& p, int64_t pos, int& lo, int& hi) {
  const int64_t cap = static_cast<int64_t>(p.seqs.max_pages) * p.page_size;
  int64_t e = pos + 1;
  if (e > cap) {
    atomicCAS(p.err, 0u, static_cast<unsigned>(kErrCachePosition));
    e = cap;
  }
  hi = static_cast<int>(e);
  lo = p.window > 0 && pos + 1 > p.window ? static_cast<int>(min(pos + 1 - p.window, e)) : 0;
}

constexpr int kSimpleThreads = 128;
constexpr int kPer = 8;   // elements per lane: head dimension up to 256

// One element of a cached row; e2m1 without the gain.
template <typename T, bool E2M1>
__device__ __forceinline__ float cached(const void* pages, const void* scales, int64_t at, int64_t scale_at, int d) {
  if constexpr (E2M1) {
    const uint32_t byte = static_cast<const uint8_t*>(pages)[at + (d >> 1)];
    const float2 v = __half22float2(e2m1x2_to_half2(byte));
    return (d & 1 ? v.y : v.x) * e4m3_to_float(static_cast<const uint8_t*>(scales)[scale_at + (d >> 4)]);
  } else {
    return Io<T>::to_f(static_cast<const T*>(pages)[at + d]);
  }
}

template <typename T, bool E2M1>
__global__ void __launch_bounds__(kSimpleThreads) paged_simple_kernel(const __grid_constant__ PagedParams p) {
  pdl_wait();
  pdl_launch_dependents();
  const int token = static_cast<int>(blockIdx.x) * (kSimpleThreads / 32) + (static_cast<int>(threadIdx.x) >> 5);
  const int lane = static_cast<int>(threadIdx.x) & 31;
  const int h = static_cast<int>(blockIdx.y), kh = h / p.group;
  if (token >= p.seqs.tokens) return;
  int seq;
  int64_t pos;
  if (!find_token(p.seqs, token, seq, pos)) return;
  const T* q = static_cast<const T*>(p.q) + token * p.q_tok + h * p.q_head;
  float qv[kPer], ov[kPer];
#pragma unroll
  for (int e = 0; e < kPer; ++e) {
    const int d = lane + 32 * e;
    qv[e] = d < p.dim ? Io<T>::to_f(q[d]) * p.scale : 0.f;
    ov[e] = 0.f;
  }
  int lo = 0, hi = 0;
  if (pos >= 0) visible(p, pos, lo, hi);
  float m = -INFINITY, l = 0.f;
  for (int j = lo; j < hi; ++j) {
    int slot;
    const int64_t page = find_page(p.seqs, seq, j, p.num_pages, slot, p.err);
    if (page < 0) continue;
    const int64_t row = E2M1 ? p.dim / 2 : p.dim, srow = p.dim / 16;
    const int64_t ka = page * p.k_page + kh * p.k_head + slot * row, va = page * p.v_page + kh * p.v_head + slot * row;
    const int64_t ksa = page * p.ks_page + kh * p.ks_head + slot * srow, vsa = page * p.vs_page + kh * p.vs_head + slot * srow;
    float s = 0.f;
#pragma unroll
    for (int e = 0; e < kPer; ++e) {
      const int d = lane + 32 * e;
      if (d < p.dim) s = fmaf(qv[e], cached<T, E2M1>(p.k, p.ks, ka, ksa, d), s);
    }
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) s += __shfl_xor_sync(0xffffffffu, s, o);
    const float m_new = fmax_nan(m, s);
    const float base = m_new == -INFINITY ? 0.f : m_new;
    const float corr = __expf(m - base);
    const float pj = __expf(s - base);
    l = l * corr + pj;
#pragma unroll
    for (int e = 0; e < kPer; ++e) {
      const int d = lane + 32 * e;
      if (d < p.dim) ov[e] = fmaf(ov[e], corr, pj * cached<T, E2M1>(p.v, p.vs, va, vsa, d));
    }
    m = m_new;
  }
  T* out = static_cast<T*>(p.o) + token * p.o_tok + h * p.o_head;
  const float inv = l == 0.f ? 0.f : p.v_gain / l;
#pragma unroll
  for (int e = 0; e < kPer; ++e) {
    const int d = lane + 32 * e;
    if (d < p.dim) out[d] = Io<T>::from_f(l == 0.f ? 0.f : ov[e] * inv);
  }
}

template <typename T, bool E2M1>
cudaError_t run_simple(const PagedParams& p, cudaStream_t s) {
  const dim3 grid(static_cast<unsigned>(ceil_div64(p.seqs.tokens, kSimpleThreads / 32)), p.q_heads);
  return launch_pdl(paged_simple_kernel<T, E2M1>, grid, dim3(kSimpleThreads), 0, s, p);
}

template <typename T>
cudaError_t run(const PagedParams& p, bool e2m1, cudaStream_t s) {
  return e2m1 ? run_simple<T, true>(p, s) : run_simple<T, false>(p, s);
}

}  // namespace

int64_t paged_attention_workspace(const lunarad_paged_attention_args&) { return 0; }

cudaError_t launch_paged_attention(const lunarad_paged_attention_args& a, cudaStream_t stream) {
  const lunarad_cache& c = *a.cache;
  PagedParams p{};
  p.q = a.q.data;
  p.o = const_cast<void*>(a.o.data);
  p.q_head = a.q.head_stride;
  p.q_tok = a.q.seq_stride;
  p.o_head = a.o.head_stride;
  p.o_tok = a.o.seq_stride;
  p.k = c.k;
  p.v = c.v;
  p.ks = c.k_scales;
  p.vs = c.v_scales;
  p.k_page = c.k_page_stride;
  p.k_head = c.k_head_stride;
  p.v_page = c.v_page_stride;
  p.v_head = c.v_head_stride;
  p.ks_page = c.ks_page_stride;
  p.ks_head = c.ks_head_stride;
  p.vs_page = c.vs_page_stride;
  p.vs_head = c.vs_head_stride;
  p.num_pages = static_cast<int>(c.num_pages);
  p.kv_heads = static_cast<int>(c.kv_heads);
  p.page_size = static_cast<int>(c.page_size);
  p.dim = static_cast<int>(c.dim);
  p.q_heads = static_cast<int>(a.q_heads);
  p.group = static_cast<int>(a.q_heads / c.kv_heads);
  p.seqs = make_seqs(a.seqs, c.page_size);
  p.window = static_cast<int>(a.window);
  const bool e2m1 = c.kind == LUNARAD_KIND_E2M1;
  p.scale = static_cast<float>(a.scale * (e2m1 ? c.k_gain : 1.0));
  p.v_gain = e2m1 ? static_cast<float>(c.v_gain) : 1.f;
  p.err = device_error_word();
  if (p.err == nullptr) return cudaErrorInvalidDevice;
  if (a.dtype == LUNARA_F16) return run<__half>(p, e2m1, stream);
  if (a.dtype == LUNARA_BF16) return run<__nv_bfloat16>(p, e2m1, stream);
  return run<float>(p, e2m1, stream);
}

}  // namespace lunara
