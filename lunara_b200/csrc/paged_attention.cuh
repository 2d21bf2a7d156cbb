// Parameters and helpers shared by the kernels of the paged attention.
#pragma once

#include "paged.cuh"

namespace lunara {

struct PagedParams {
  const void* q;
  void* o;
  int64_t q_head, q_tok, o_head, o_tok;   // strides
  const void* k;
  const void* v;
  const void* ks;
  const void* vs;
  int64_t k_page, k_head, v_page, v_head, ks_page, ks_head, vs_page, vs_head;
  // The same for the streaming kernel: strides in units of `unit` bytes, of the
  // scales in 16 bytes.
  uint32_t unit, k_page_u, v_page_u, row_u, ks_page_u, vs_page_u;
  int num_pages, kv_heads, page_size, dim, q_heads, group;
  Seqs seqs;
  int window;
  float scale;   // softmax scale times the keys' gain
  float v_gain;
  // Sequences with min_rows <= (their tokens * group) < max_rows are this kernel's.
  int64_t min_rows, max_rows;
  int nt;   // 8-row tiles per row tile of the streaming kernel
  // Split work: partial results of each worker (two slots of a row tile).
  float* part_o;
  float* part_ml;
  int workers;
  unsigned int* err;
};

// One sequence as the attention kernels see it.
struct SeqInfo {
  int first;      // its first token
  int n;          // its tokens
  int64_t pos0;   // position of the first one (negative: padding before position 0)
  int hi;         // keys that its last token sees, cut to the page table
  int lo;         // first key that its first real token sees
};

__device__ __forceinline__ SeqInfo load_seq(const PagedParams& p, int b) {
  SeqInfo s;
  const int a = p.seqs.starts[b], e = p.seqs.starts[b + 1], len = p.seqs.lens[b];
  s.first = max(0, min(a, p.seqs.tokens));
  s.n = max(0, min(e, p.seqs.tokens) - s.first);
  s.pos0 = static_cast<int64_t>(len) - (static_cast<int64_t>(e) - s.first);
  const int64_t cap = static_cast<int64_t>(p.seqs.max_pages) * p.page_size;
  int64_t hi = s.pos0 + s.n;   // == len unless seq_starts runs past the tokens
  if (hi > cap) {
    if (s.n > 0) atomicCAS(p.err, 0u, static_cast<unsigned>(kErrCachePosition));
    hi = cap;
  }
  s.hi = static_cast<int>(max(hi, int64_t{0}));
  const int64_t q0 = max(s.pos0, int64_t{0});
  s.lo = p.window > 0 && q0 + 1 > p.window ? static_cast<int>(min(q0 + 1 - p.window, static_cast<int64_t>(s.hi))) : 0;
  return s;
}

// The keys [lo, hi) that a position sees, cut to the page table.
__device__ __forceinline__ void visible(const PagedParams& p, int64_t pos, int& lo, int& hi) {
  const int64_t cap = static_cast<int64_t>(p.seqs.max_pages) * p.page_size;
  const int64_t e = max(int64_t{0}, min(pos + 1, cap));
  hi = static_cast<int>(e);
  lo = p.window > 0 && pos + 1 > p.window ? static_cast<int>(min(pos + 1 - p.window, e)) : 0;
}

// Many query rows per sequence (paged_prefill.cu): 16-bit caches with head
// dimension 64 or 128.
int64_t paged_prefill_workspace(int dim, int sms);
cudaError_t launch_paged_prefill(PagedParams p, int dtype, void* workspace, cudaStream_t stream);

}  // namespace lunara
