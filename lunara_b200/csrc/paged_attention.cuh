// Parameters and helpers shared by the kernels of the paged attention.
#pragma once

#include <atomic>

#include "kernels.h"
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
  int zero_before, zero_behind;   // clear the rows before the first sequence, behind the last
  // Split work: partial results of each worker (two slots of a row tile).
  float* part_o;    // unnormalised output rows
  float* part_ml;   // kPartMl floats per row: largest score, sum, factor
  struct Cut* cuts;   // of each worker
  int workers;
  unsigned int* err;
};

// A part's exponents are (score - largest score) * factor, in log2; its row's
// parts have the same factor. The largest score is kept as it is, not times the
// factor: for scores of 2^17 that product's rounding would move a part's weight
// by half a percent against the other parts'.
constexpr int kPartMl = 4;

// The factor of a row's exponents, (score - largest score) * factor in log2: the
// scale times log2(e), and times what its queries were divided by. It takes part
// as a positive fp32 number of any size. Zero would make NaN of the distance of
// the first score from -inf: it becomes the smallest number, which leaves every
// distance between fp32 numbers at nothing, as zero would. Infinity, which only
// scores beyond fp32 can need, becomes the largest.
__device__ __forceinline__ float exponent_factor(float f) { return fminf(fmaxf(f, 1.4e-45f), 3.402823466e38f); }

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

// Written by every worker for the kernel that joins the parts: the row tile
// that its run began at the first key tile of and did not finish. Its parts are
// this worker's, in `slot`, and those of the next parts - 1 workers in slot 0.
struct Cut {
  int parts;   // 0: there is none
  int slot, rows, first_token, row0, kv_head;
  int pad[2];
};

// Clears the output rows of token; by a whole block.
template <typename T>
__device__ __forceinline__ void clear_token(const PagedParams& p, int token) {
  const int width = p.q_heads * p.dim;
  for (int e = threadIdx.x; e < width; e += blockDim.x)
    static_cast<T*>(p.o)[token * p.o_tok + e / p.dim * p.o_head + e % p.dim] = Io<T>::from_f(0.f);
}

// Clears the output rows of the sequences that are this kernel's and have no
// keys, and of the tokens that no sequence owns where that is asked for; by
// whole blocks, each its share.
template <typename T>
__device__ __forceinline__ void clear_empty(const PagedParams& p) {
  if (p.zero_before)
    for (int token = blockIdx.x, end = min(p.seqs.starts[0], p.seqs.tokens); token < end; token += gridDim.x) clear_token<T>(p, token);
  if (p.zero_behind)
    for (int64_t token = int64_t{max(p.seqs.starts[p.seqs.batch], 0)} + blockIdx.x; token < p.seqs.tokens; token += gridDim.x)
      clear_token<T>(p, static_cast<int>(token));
  for (int b = blockIdx.x; b < p.seqs.batch; b += gridDim.x) {
    const SeqInfo s = load_seq(p, b);
    const int64_t rows = static_cast<int64_t>(s.n) * p.group;
    if (rows < p.min_rows || rows >= p.max_rows || s.hi > s.lo) continue;
    for (int token = s.first; token < s.first + s.n; ++token) clear_token<T>(p, token);
  }
}

// The keys [lo, hi) that a position sees, cut to the page table.
__device__ __forceinline__ void visible(const PagedParams& p, int64_t pos, int& lo, int& hi) {
  const int64_t cap = static_cast<int64_t>(p.seqs.max_pages) * p.page_size;
  const int64_t e = max(int64_t{0}, min(pos + 1, cap));
  hi = static_cast<int>(e);
  lo = p.window > 0 && pos + 1 > p.window ? static_cast<int>(min(pos + 1 - p.window, e)) : 0;
}

// Joins the parts of the cut row tiles. Block x looks at every gridDim.x-th
// worker's cut, at most 32 of them (a block for each worker cost 10 us in
// launches alone, most of them for nothing), and takes the share blockIdx.y of the rows of each. Lanes load the maxima and sums of 32 parts at once; the sums of O
// then are independent loads, many of them in flight. The warps of a row meet in
// shared memory.
constexpr int kJoinThreads = 128;

template <typename T, int DP>
__global__ void __launch_bounds__(kJoinThreads) paged_join_kernel(const __grid_constant__ PagedParams p, int tile_rows) {
  constexpr int kWarps = kJoinThreads / 32, kE = DP / 32;
  __shared__ float s_o[kWarps][DP];
  __shared__ float2 s_ml[kWarps];
  pdl_wait();
  const int lane = static_cast<int>(threadIdx.x) & 31, warp = static_cast<int>(threadIdx.x) >> 5;
  const int candidate = static_cast<int>(blockIdx.x) + lane * static_cast<int>(gridDim.x);
  uint32_t found = __ballot_sync(0xffffffffu, candidate < p.workers && p.cuts[candidate].parts > 0);
  for (; found != 0u; found &= found - 1u) {
    const int w0 = static_cast<int>(blockIdx.x) + (__ffs(found) - 1) * static_cast<int>(gridDim.x);
    const Cut cut = p.cuts[w0];
    const int share = (cut.rows + static_cast<int>(gridDim.y) - 1) / static_cast<int>(gridDim.y);
    const int r_first = static_cast<int>(blockIdx.y) * share, r_end = min(cut.rows, r_first + share);
    if (r_first >= r_end) continue;
    // `at_once` rows at a time, `splits` warps to each.
    const int splits = r_end - r_first >= kWarps ? 1 : kWarps / (r_end - r_first), at_once = kWarps / splits;
    const int split = warp / at_once;
    for (int r0 = r_first; r0 < r_end; r0 += at_once) {
      const int r = r0 + warp % at_once;
      const bool use = split < splits && r < r_end;
      auto at = [&](int i) {   // row r of part i
        return (static_cast<int64_t>(w0 + i) * 2 + (i == 0 ? cut.slot : 0)) * tile_rows + r;
      };
      float m = -INFINITY, l = 0.f, factor = 0.f, o[kE];
#pragma unroll
      for (int e = 0; e < kE; ++e) o[e] = 0.f;
      if (use) {
        for (int i0 = split; i0 < cut.parts; i0 += 32 * splits) {
          // Lane k: part i0 + k splits.
          const int n = min(32, (cut.parts - i0 + splits - 1) / splits);
          float4 ml = make_float4(-INFINITY, 0.f, 0.f, 0.f);
          if (lane < n) ml = *reinterpret_cast<const float4*>(p.part_ml + kPartMl * at(i0 + lane * splits));
          factor = __shfl_sync(0xffffffffu, ml.z, 0);
          float top = ml.x;
#pragma unroll
          for (int k = 16; k > 0; k >>= 1) top = fmax_nan(top, __shfl_xor_sync(0xffffffffu, top, k));
          const float next = fmax_nan(m, top), base = next == -INFINITY ? 0.f : next;
          const float keep = ex2_approx((m - base) * factor), f = ex2_approx((ml.x - base) * factor);
          m = next;
          l = l * keep + ml.y * f;   // of this lane's parts, summed below
#pragma unroll
          for (int e = 0; e < kE; ++e) o[e] *= keep;
#pragma unroll 8
          for (int k = 0; k < n; ++k) {
            const float* src = p.part_o + at(i0 + k * splits) * DP + kE * lane;
            const float w = __shfl_sync(0xffffffffu, f, k);
            if constexpr (kE == 4) {
              const float4 v = *reinterpret_cast<const float4*>(src);
              o[0] = fmaf(v.x, w, o[0]); o[1] = fmaf(v.y, w, o[1]); o[2] = fmaf(v.z, w, o[2]); o[3] = fmaf(v.w, w, o[3]);
            } else {
              const float2 v = *reinterpret_cast<const float2*>(src);
              o[0] = fmaf(v.x, w, o[0]); o[1] = fmaf(v.y, w, o[1]);
            }
          }
        }
#pragma unroll
        for (int k = 16; k > 0; k >>= 1) l += __shfl_xor_sync(0xffffffffu, l, k);
      }
      if (splits > 1) {
        __syncthreads();   // the rows before have been read
#pragma unroll
        for (int e = 0; e < kE; ++e) s_o[warp][kE * lane + e] = o[e];
        if (lane == 0) s_ml[warp] = make_float2(m, l);
        __syncthreads();
        if (use && split == 0)
          for (int k = 1; k < splits; ++k) {
            const float2 ml = s_ml[warp + k * at_once];
            const float next = fmax_nan(m, ml.x), base = next == -INFINITY ? 0.f : next;
            const float fa = ex2_approx((m - base) * factor), fb = ex2_approx((ml.x - base) * factor);   // (split 0 has had a part)
            m = next;
            l = l * fa + ml.y * fb;
#pragma unroll
            for (int e = 0; e < kE; ++e) o[e] = o[e] * fa + s_o[warp + k * at_once][kE * lane + e] * fb;
          }
      }
      if (use && split == 0) {
        const float inv = l == 0.f ? 0.f : p.v_gain / l;
        const int row = cut.row0 + r, i = row / p.group;
        T* out = static_cast<T*>(p.o) + (cut.first_token + i) * p.o_tok + (cut.kv_head * p.group + row - i * p.group) * p.o_head + kE * lane;
#pragma unroll
        for (int e = 0; e < kE; ++e)
          if (kE * lane + e < p.dim) out[e] = Io<T>::from_f(l == 0.f ? 0.f : o[e] * inv);
      }
    }
  }
}

// Blocks along x for a join over `workers` runs.
inline unsigned join_blocks(int workers) {
  const int few = 2 * device_num_sms(), need = (workers + 31) / 32;
  return static_cast<unsigned>(workers < few ? workers : need > few ? need : few);
}

// Prepares a kernel (its shared memory, and with regs > 0 a check that it was
// built with that many registers) once per device: the calls cost a microsecond
// or two, which a decode step would pay every time. `done` is the caller's, one
// per kernel, a bit for each device.
template <typename Kernel>
cudaError_t prepare_once(Kernel kern, std::atomic<uint64_t>& done, int smem, int regs) {
  int dev = 0;
  cudaError_t e = cudaGetDevice(&dev);
  if (e != cudaSuccess) return e;
  const uint64_t bit = dev < 64 ? uint64_t{1} << dev : 0;
  if ((done.load(std::memory_order_acquire) & bit) != 0) return cudaSuccess;
  if (regs > 0) {
    cudaFuncAttributes fa{};
    e = cudaFuncGetAttributes(&fa, kern);
    if (e != cudaSuccess) return e;
    if (fa.numRegs != regs) return cudaErrorInvalidConfiguration;
  }
  e = cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, smem);
  if (e == cudaSuccess) done.fetch_or(bit, std::memory_order_release);
  return e;
}

// Many query rows per sequence (paged_prefill.cu): 16-bit caches, head dimension
// a multiple of 8 up to 128, scale not negative.
int64_t paged_prefill_workspace(int dim, int sms);
cudaError_t launch_paged_prefill(PagedParams p, int dtype, void* workspace, cudaStream_t stream);

}  // namespace lunara
