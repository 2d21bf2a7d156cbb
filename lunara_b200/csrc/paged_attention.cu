// Attention over the paged key/value cache.
//
//   O[t] = sum_j softmax_j(scale q_t . k_j) v_j   over the keys j that the
//   query's position sees: j <= p, and with a window j > p - window.
//
// Streaming kernel (16-bit and 4-bit caches): the query rows of one sequence
// and key head (its tokens times the query heads of the group) make tiles of 8 or
// 16 rows; their keys are cut into tiles of KT, and all tiles of the batch, in
// the order (sequence, key head, row tile, key tile), are dealt to the warps of
// a persistent grid in equal contiguous runs. Bound by HBM: a decode step reads
// each cached byte once for group * 4 operations per element. Measured on B200:
// 64 sequences of up to 8191 keys, 32/8 heads of 128 in bf16, 188 us for 1.18 GB
// (6.3 TB/s); with 4 bits 438 MB of codes in 108 us (4.0 TB/s, 64 % of the issue
// slots: conversions and products that wait for one another).
//   * Every warp works alone (no block barrier after the start): it copies its
//     tiles with cp.async into a ring of its own in shared memory. The order of
//     the head dimension inside the scores and of the columns of V is free; it is
//     chosen so that a lane's mma fragments are contiguous in memory, and no
//     ldmatrix is needed.
//   * S^T = K Q^T and O^T += V^T P^T by mma.sync m16n8k16 with fp32 accumulators:
//     keys and elements fill the 16 rows of an instruction, so that 8 query rows
//     fill the rest. These products need a fraction of the legacy tensor rate
//     while HBM delivers its 23 bytes per clock and SM; where there are enough
//     rows for tcgen05, paged_prefill.cu takes them.
//   * The running maximum is raised only when a row's maximum grows by more
//     than 2^8 (a warp vote), so O is rescaled a few times per row in all. P
//     rounded to the products' type, as V has it, is off by half a step of it.
//   * 4-bit caches: codes become f16 pairs by one cvt per pair, times their
//     e4m3 scale by one half2 product, exactly (6 significant bits; 2^-10 ..
//     2688); the products run in f16 whatever the queries' type. bf16 queries
//     are brought into f16's range row by row with a power of two, which drops
//     bits below 2^-24 of the row's largest element only.
// Runs that cut a (sequence, key head, row tile) leave partial O, maximum and
// sum in the workspace, and a second kernel joins them; all others write O. The
// split depends on the lengths only, so results repeat bit for bit.
//
// Simple kernel (fp32, and head dimensions or strides the streaming kernel does
// not take): one warp per query row, one key after the other.
#include <type_traits>

#include "kernels.h"
#include "paged_attention.cuh"
#include "scale_copy.h"

namespace lunara {
namespace {

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
  if (!find_token(p.seqs, token, seq, pos)) {
    if (p.zero_behind)
      for (int d = lane; d < p.dim; d += 32) static_cast<T*>(p.o)[token * p.o_tok + h * p.o_head + d] = Io<T>::from_f(0.f);
    return;
  }
  const T* q = static_cast<const T*>(p.q) + token * p.q_tok + h * p.q_head;
  float qv[kPer], ov[kPer];
#pragma unroll
  for (int e = 0; e < kPer; ++e) {
    const int d = lane + 32 * e;
    qv[e] = d < p.dim ? Io<T>::to_f(q[d]) * p.scale : 0.f;
    ov[e] = 0.f;
  }
  int lo, hi;
  visible(p, pos, lo, hi);
  if (hi <= pos) atomicCAS(p.err, 0u, static_cast<unsigned>(kErrCachePosition));
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
    // expf is off by 2 ulp at any argument, so that fp32 calls get fp32 weights.
    const float corr = expf(m - base);
    const float pj = expf(s - base);
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

// ------------------------------------------------------- streaming kernel --
constexpr int kWarps = 4;
constexpr int kStreamThreads = 32 * kWarps;
constexpr int kMaxBatch = 1024;          // sequences per launch (their prefix sums stand in shared memory)
constexpr float kRescaleLog2 = 8.0f;

// Sizes of one instance; DP is the head dimension rounded up to 64 or 128, NT
// the 8-row tiles of queries that share the keys.
template <bool E2M1, int DP, int NT>
struct Shape {
  static constexpr int kRows = 8 * NT;
  static constexpr int KT = E2M1 || DP == 64 ? 32 : 16;   // keys per tile
  static constexpr int kSteps = DP / 16;                  // k-steps of K Q^T
  static constexpr int kRun = E2M1 ? DP / 8 : 8;          // neighbouring columns of V that a lane holds
  static constexpr int kRow = E2M1 ? DP / 2 : 2 * DP;             // bytes of a row, codes or elements
  static constexpr int kKBytes = KT * kRow, kVBytes = KT * kRow;
  static constexpr int kScaleBytes = E2M1 ? KT * (DP / 16) : 0;   // of K, and of V
  static constexpr int kStageBytes = kKBytes + kVBytes + 2 * kScaleBytes;
  static constexpr int kStages = NT == 1 ? 2 : 3;
  static constexpr int kRingBytes = kStages * kStageBytes;        // per warp
  static constexpr int kCtasPerSm = (E2M1 ? 3 : 2) + (NT == 1 ? 1 : 0);
};

// 16 bytes to shared memory, or zeros (then nothing is read).
__device__ __forceinline__ void copy_async(uint32_t dst, const void* src, bool in) {
  asm volatile("cp.async.cg.shared.global.L2::128B [%0], [%1], 16, %2;" ::"r"(dst), "l"(src), "r"(in ? 16 : 0) : "memory");
}
__device__ __forceinline__ void copy_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int N>
__device__ __forceinline__ void copy_wait() { asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory"); }

__device__ __forceinline__ uint4 lds128(uint32_t a) {
  uint4 u;
  asm volatile("ld.shared.v4.u32 {%0, %1, %2, %3}, [%4];" : "=r"(u.x), "=r"(u.y), "=r"(u.z), "=r"(u.w) : "r"(a) : "memory");
  return u;
}
__device__ __forceinline__ uint2 lds64(uint32_t a) {
  uint2 u;
  asm volatile("ld.shared.v2.u32 {%0, %1}, [%2];" : "=r"(u.x), "=r"(u.y) : "r"(a) : "memory");
  return u;
}
__device__ __forceinline__ uint32_t lds32(uint32_t a) {
  uint32_t u;
  asm volatile("ld.shared.u32 %0, [%1];" : "=r"(u) : "r"(a) : "memory");
  return u;
}
__device__ __forceinline__ uint32_t lds16(uint32_t a) {
  uint16_t u;
  asm volatile("ld.shared.u16 %0, [%1];" : "=h"(u) : "r"(a) : "memory");
  return u;
}
__device__ __forceinline__ uint32_t lds8(uint32_t a) {
  uint32_t u;
  asm volatile("ld.shared.u8 %0, [%1];" : "=r"(u) : "r"(a) : "memory");
  return u;
}

// Places in a stage of the 16-byte piece `piece` of K's and V's row r. The rows
// stand one behind the other, so that 8 neighbouring lanes copy one 128-byte
// line of memory to one 128-byte line here: a copy whose two sides do not match
// line by line is cut into a request per sector (measured: 1.5 times the
// sectors, 4.8 instead of 6 TB/s). Within a line the pieces are permuted so that
// the lanes of a product read from different banks.
template <typename S, bool E2M1>
__device__ __forceinline__ uint32_t k_place(int r, int piece) {
  if constexpr (E2M1) return r * S::kRow + 16 * piece;
  else return r * S::kRow + (piece >> 3) * 128 + (((piece & 7) ^ (4 * (r & 1))) << 4);
}
template <typename S, bool E2M1>
__device__ __forceinline__ uint32_t v_place(int r, int piece) {
  constexpr int kPerLine = S::kRow >= 128 ? 1 : 128 / S::kRow;   // rows per line
  if constexpr (kPerLine == 1) return r * S::kRow + (piece >> 3) * 128 + (((piece & 7) ^ (r & 6)) << 4);
  else if constexpr (kPerLine == 2) return (r >> 1) * 128 + ((((r & 1) * 4 + piece) ^ (r & 6)) << 4);
  else return (r >> 2) * 128 + ((((r & 3) * 2 + piece) ^ (2 * ((r >> 2) & 1))) << 4);
}

__device__ __forceinline__ void sts8(uint32_t a, uint32_t v) {
  asm volatile("st.shared.u8 [%0], %1;" ::"r"(a), "r"(v) : "memory");
}

// The 8 x 8 matrix of 16-bit elements whose rows the lanes 4 r .. 4 r + 3 hold, transposed.
__device__ __forceinline__ uint32_t transpose8x8(uint32_t x) {
  uint32_t r;
  asm volatile("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(r) : "r"(x));
  return r;
}

// D += A B, m16n8k16: A row-major, B column-major, 16-bit, fp32 accumulators.
template <typename T>
__device__ __forceinline__ void mma16816(float (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0,
                                         uint32_t b1) {
  if constexpr (std::is_same<T, __half>::value)
    asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
        : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
        : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
  else
    asm("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
        : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
        : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}

__device__ __forceinline__ uint32_t hmul2(uint32_t a, uint32_t b) {
  uint32_t r;
  asm("mul.rn.f16x2 %0, %1, %2;" : "=r"(r) : "r"(a), "r"(b));
  return r;
}
// The four bytes of codes in w as f16 pairs.
__device__ __forceinline__ void codes_to_half2(uint32_t w, uint32_t (&h)[4]) {
  asm("{\n\t.reg .b8 t0, t1, t2, t3;\n\t"
      "mov.b32 {t0, t1, t2, t3}, %4;\n\t"
      "cvt.rn.f16x2.e2m1x2 %0, t0;\n\t"
      "cvt.rn.f16x2.e2m1x2 %1, t1;\n\t"
      "cvt.rn.f16x2.e2m1x2 %2, t2;\n\t"
      "cvt.rn.f16x2.e2m1x2 %3, t3;\n\t}"
      : "=r"(h[0]), "=r"(h[1]), "=r"(h[2]), "=r"(h[3])
      : "r"(w));
}
// Two e4m3 bytes as an f16 pair.
__device__ __forceinline__ uint32_t scales_to_half2(uint32_t two) {
  uint32_t r;
  asm("cvt.rn.f16x2.e4m3x2 %0, %1;" : "=r"(r) : "h"(static_cast<uint16_t>(two)));
  return r;
}

// Row tiles of a sequence, and the key tiles of each of them.
struct Tiling {
  int KT, rows;   // keys and rows of a tile
};
__device__ __forceinline__ void seq_tiles(const PagedParams& p, const SeqInfo& s, Tiling tl, int& row_tiles, int& tiles) {
  const int64_t rows = static_cast<int64_t>(s.n) * p.group;
  if (rows < p.min_rows || rows >= p.max_rows || s.hi <= s.lo) {
    row_tiles = tiles = 0;
    return;
  }
  row_tiles = static_cast<int>((rows + tl.rows - 1) / tl.rows);
  tiles = (s.hi + tl.KT - 1) / tl.KT - s.lo / tl.KT;
}

// prefix[b] = tiles of the sequences before b (batch + 1 entries in shared
// memory), by the whole block.
__device__ __forceinline__ void prefix_tiles(const PagedParams& p, Tiling tl, int64_t* prefix, int64_t* warp_sums) {
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, warps = blockDim.x >> 5;
  int64_t carry = 0;
  for (int b0 = 0; b0 < p.seqs.batch; b0 += blockDim.x) {
    const int b = b0 + static_cast<int>(threadIdx.x);
    int64_t inc = 0;
    if (b < p.seqs.batch) {
      int rt, nt;
      seq_tiles(p, load_seq(p, b), tl, rt, nt);
      inc = static_cast<int64_t>(p.kv_heads) * rt * nt;
    }
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const int64_t y = __shfl_up_sync(0xffffffffu, inc, o);
      if (lane >= o) inc += y;
    }
    if (lane == 31) warp_sums[warp] = inc;
    __syncthreads();
    int64_t before = carry;
    for (int w = 0; w < warps; ++w) {
      if (w < warp) before += warp_sums[w];
      carry += warp_sums[w];
    }
    if (b < p.seqs.batch) prefix[b + 1] = before + inc;
    __syncthreads();
  }
  if (threadIdx.x == 0) prefix[0] = 0;
  __syncthreads();
}

// Worker w of `workers` takes the tiles [run_start(w), run_start(w + 1)); there
// are never more workers than tiles, so that none of them has an empty run (the
// join reads a part of every worker between a row's first and last one).
__device__ __forceinline__ int used_workers(const PagedParams& p, int64_t total) {
  return static_cast<int>(min(total, static_cast<int64_t>(p.workers)));
}
__device__ __forceinline__ int64_t run_start(int64_t total, int workers, int w) { return total * w / workers; }
// The worker whose run holds tile t.
__device__ __forceinline__ int run_of(int64_t total, int workers, int64_t t) {
  return static_cast<int>(((t + 1) * workers + total - 1) / total) - 1;
}

// EXACT: the head dimension is DP, a constant.
template <typename T, bool E2M1, int DP, int NT, bool EXACT>
__global__ void __launch_bounds__(kStreamThreads, Shape<E2M1, DP, NT>::kCtasPerSm)
    paged_stream_kernel(const __grid_constant__ PagedParams p) {
  using S = Shape<E2M1, DP, NT>;
  using M = typename std::conditional<E2M1, __half, T>::type;   // type of the products
  constexpr int KT = S::KT;
  constexpr Tiling kTiling{S::KT, S::kRows};
  extern __shared__ __align__(16) uint8_t smem[];
  __shared__ int64_t warp_sums[kWarps];
  int64_t* prefix = reinterpret_cast<int64_t*>(smem + kWarps * S::kRingBytes);
  const int lane = static_cast<int>(threadIdx.x) & 31, warp = static_cast<int>(threadIdx.x) >> 5;
  const int g = lane >> 2, c = lane & 3;
  const uint32_t ring = smem_u32(smem) + warp * S::kRingBytes;
  pdl_wait();
  pdl_launch_dependents();
  prefix_tiles(p, kTiling, prefix, warp_sums);
  const int64_t total = prefix[p.seqs.batch];
  const int workers = used_workers(p, total), worker = static_cast<int>(blockIdx.x) * kWarps + warp;
  clear_empty<T>(p);
  if (worker >= workers) {
    if (lane == 0) p.cuts[worker].parts = 0;
    return;
  }
  const int64_t t_first = run_start(total, workers, worker), t_end = run_start(total, workers, worker + 1);
  const bool grouped = E2M1 || (p.page_size & 7) == 0;   // 8 neighbouring keys stand in one page
  constexpr int kElem = E2M1 ? 1 : 2;
  const int dim = EXACT ? DP : p.dim;
  const int row_bytes = E2M1 ? dim / 2 : dim * 2, srow = dim / 16;

  for (int64_t t = t_first; t < t_end;) {
    // ------------------------------------------------ where the run stands --
    int b = 0;
    for (int end = p.seqs.batch; b + 1 < end;) {   // last b with prefix[b] <= t
      const int mid = (b + end) >> 1;
      if (prefix[mid] <= t) b = mid; else end = mid;
    }
    const SeqInfo s = load_seq(p, b);
    int row_tiles, seg_tiles;
    seq_tiles(p, s, kTiling, row_tiles, seg_tiles);
    const int64_t in_seq = t - prefix[b];
    const int seg = static_cast<int>(in_seq / seg_tiles);
    const int tile0 = static_cast<int>(in_seq - static_cast<int64_t>(seg) * seg_tiles);
    const int kh = seg / row_tiles, rt = seg - kh * row_tiles;
    const int n_tiles = static_cast<int>(min(static_cast<int64_t>(seg_tiles - tile0), t_end - t));
    const int key0 = (s.lo / KT + tile0) * KT;
    const int row0 = rt * S::kRows, rows = min(S::kRows, s.n * p.group - row0);

    // Keys that the lane's query columns 2 c and 2 c + 1 (of each 8-row tile) see.
    int lo[NT][2], hi[NT][2];
#pragma unroll
    for (int n = 0; n < NT; ++n)
#pragma unroll
      for (int r = 0; r < 2; ++r) visible(p, s.pos0 + (row0 + min(8 * n + 2 * c + r, rows - 1)) / p.group, lo[n][r], hi[n][r]);
    // Keys that some row sees, and that all rows see.
    int any_lo, any_hi, all_lo, all_hi;
    visible(p, s.pos0 + (row0 + rows - 1) / p.group, all_lo, any_hi);
    visible(p, s.pos0 + row0 / p.group, any_lo, all_hi);

    // -------------------------------------------------------------- pages --
    // Lane l looks up the l-th group of 8 keys of a batch of 256 (grouped) or
    // the l-th key of a tile, a batch ahead of its use, and keeps where it
    // stands in K, V and the scales, in units of p.unit bytes (32 bits reach
    // 64 or 256 GiB).
    const int32_t* table = p.seqs.page_table + b * p.seqs.table_stride;
    const int per_lane = grouped ? 8 : 1, batch_keys = grouped ? 256 : KT;
    auto load_page = [&](int first) {
      const int key = first + per_lane * lane;
      if (key + per_lane <= any_lo || key >= any_hi) return -1;   // nothing of it is read
      const int page = table[p.seqs.page_div.div(key)];
      if (page >= 0 && page < p.num_pages) return page;
      atomicCAS(p.err, 0u, static_cast<unsigned>(kErrCachePage));
      return -1;
    };
    uint32_t k_at = 0, v_at = 0, ks_at = 0, vs_at = 0, have = 0;   // have: a bit per lane whose lookup found a page
    int batch0 = key0 - batch_keys, page_next = load_page(key0);
    auto next_batch = [&] {
      const int page = page_next;
      batch0 += batch_keys;
      page_next = load_page(batch0 + batch_keys);
      have = __ballot_sync(0xffffffffu, page >= 0);
      const int key = batch0 + per_lane * lane;
      const uint32_t slot = static_cast<uint32_t>(key - p.seqs.page_div.div(key) * p.page_size);
      const uint32_t pg = static_cast<uint32_t>(max(page, 0)), use = page >= 0 ? 1u : 0u;
      k_at = (pg * p.k_page_u + slot * p.row_u) * use;
      v_at = (pg * p.v_page_u + slot * p.row_u) * use;
      if constexpr (E2M1) {   // groups of 8 scale rows: pieces of 16 bytes
        ks_at = (pg * p.ks_page_u + (slot >> 3) * static_cast<uint32_t>(srow >> 1)) * use;
        vs_at = (pg * p.vs_page_u + (slot >> 3) * static_cast<uint32_t>(srow >> 1)) * use;
      }
    };
    const char* kb = static_cast<const char*>(p.k) + kh * p.k_head * kElem;
    const char* vb = static_cast<const char*>(p.v) + kh * p.v_head * kElem;
    auto place = [&](const char* base, uint32_t at) { return base + static_cast<uint64_t>(at) * p.unit; };

    // Starts the copies of tile i into its stage; returns a bit for each of its
    // keys that takes part. All others are zero-filled: neither a stale slot's
    // NaN nor a bad page may reach a product.
    auto issue = [&](int i, int stage) -> uint32_t {
      const int first = key0 + i * KT;
      if (first - batch0 >= batch_keys) next_batch();
      const int g0 = (first - batch0) >> 3;   // grouped: the tile's first group in the batch
      uint32_t ok = have;
      if (grouped) {
        const uint32_t x = (ok >> g0) & ((1u << (KT / 8)) - 1u);   // a bit for each group -> a byte
        ok = ((x & 1u) | ((x & 2u) << 7) | ((x & 4u) << 14) | ((x & 8u) << 21)) * 0xFFu;
      }
      if (any_lo > first) ok &= any_lo - first < 32 ? ~0u << (any_lo - first) : 0u;
      if (any_hi < first + 32) ok &= any_hi > first ? (1u << (any_hi - first)) - 1u : 0u;
      if (KT < 32) ok &= (1u << (KT & 31)) - 1u;
      const uint32_t at = ring + stage * S::kStageBytes;
      if constexpr (E2M1) {
        constexpr int kPieces = DP / 32;   // 16-byte pieces of a row of codes
        const int piece = lane % kPieces, in_group = (lane / kPieces) & 7;
        const bool lane_in = EXACT || 16 * piece < row_bytes;
        const int from = in_group * row_bytes + (lane_in ? 16 * piece : 0);   // (a copy of nothing names a place in the cache too)
        const char* kl = kb + from;
        const char* vl = vb + from;
#pragma unroll
        for (int j = 0; j < KT * kPieces / 32; ++j) {
          const int local = (lane + 32 * j) / kPieces, src = g0 + (local >> 3);
          const uint32_t ka = __shfl_sync(0xffffffffu, k_at, src), va = __shfl_sync(0xffffffffu, v_at, src);
          const bool in = ((ok >> local) & 1u) != 0u && lane_in;
          copy_async(at + k_place<S, true>(local, piece), place(kl, ka), in);
          copy_async(at + S::kKBytes + v_place<S, true>(local, piece), place(vl, va), in);
        }
        // The scales of a group of 8 keys are srow / 2 pieces of 16 bytes. A
        // group with a masked key is copied whole; V's are cleared below.
        const ScaleCopy sc = scale_copy<KT, DP>(lane, srow);
        const uint32_t ka = __shfl_sync(0xffffffffu, ks_at, g0 + sc.group), va = __shfl_sync(0xffffffffu, vs_at, g0 + sc.group);
        if (sc.copies) {
          const bool in = ((ok >> (8 * sc.group)) & 0xFFu) != 0u;
          const uint8_t* src = sc.kv == 0 ? static_cast<const uint8_t*>(p.ks) + kh * p.ks_head + static_cast<uint64_t>(ka) * 16
                                          : static_cast<const uint8_t*>(p.vs) + kh * p.vs_head + static_cast<uint64_t>(va) * 16;
          copy_async(at + S::kKBytes + S::kVBytes + sc.kv * S::kScaleBytes + sc.place, src + 16 * sc.piece, in);
        }
      } else {
        constexpr int kPieces = DP / 8, kAtOnce = 32 / kPieces;
        const int piece = lane % kPieces, sub = lane / kPieces;
        const bool lane_in = EXACT || 16 * piece < row_bytes;
        const int from = lane_in ? 16 * piece : 0;
#pragma unroll
        for (int i8 = 0; i8 < KT / 8; ++i8) {
          const uint32_t ka = __shfl_sync(0xffffffffu, k_at, (g0 + i8) & 31), va = __shfl_sync(0xffffffffu, v_at, (g0 + i8) & 31);
          const char* kg = place(kb + sub * row_bytes + from, ka);
          const char* vg = place(vb + sub * row_bytes + from, va);
#pragma unroll
          for (int it = 0; it < 8 / kAtOnce; ++it) {
            const int r = it * kAtOnce + sub, local = 8 * i8 + r;
            const bool in = ((ok >> local) & 1u) != 0u && lane_in;
            const char* ksrc = kg + it * kAtOnce * row_bytes;
            const char* vsrc = vg + it * kAtOnce * row_bytes;
            if (!grouped) {   // every row by its own page
              ksrc = place(kb + from, __shfl_sync(0xffffffffu, k_at, local));
              vsrc = place(vb + from, __shfl_sync(0xffffffffu, v_at, local));
            }
            copy_async(at + k_place<S, false>(local, piece), ksrc, in);
            copy_async(at + S::kKBytes + v_place<S, false>(local, piece), vsrc, in);
          }
        }
      }
      copy_commit();
      return ok;
    };

    uint32_t ok_of[S::kStages];   // of the tiles in flight, oldest first
#pragma unroll
    for (int i = 0; i < S::kStages - 1; ++i) {
      ok_of[i] = 0u;
      if (i < n_tiles) ok_of[i] = issue(i, i);
      else copy_commit();
    }

    // ------------------------------------------------------------ queries --
    // Q^T as the B operand: the lane holds query row g of each 8-row tile.
    uint32_t qf[NT][S::kSteps][2];
    // The maximum below needs a positive factor: a negative scale turns the
    // queries' signs instead.
    float sl2[NT][2];   // of the columns 2 c, 2 c + 1
    const float scale_log2 = fabsf(p.scale) * 1.4426950408889634f;
    const uint32_t flip = p.scale < 0.f ? 0x80008000u : 0u;
#pragma unroll
    for (int n = 0; n < NT; ++n) {
      const int row = row0 + min(8 * n + g, rows - 1), i = row / p.group;
      const T* q = static_cast<const T*>(p.q) + (s.first + i) * p.q_tok + (kh * p.group + row - i * p.group) * p.q_head;
#pragma unroll
      for (int j = 0; j < DP / 32; ++j) {
        // The lane's j-th 8 elements: with 16 bits piece c + 4 j of the row,
        // with 4 bits the j-th 8 of DP / 4 neighbouring ones.
        const int d = E2M1 ? (DP / 4) * c + 8 * j : 8 * (c + 4 * j);
        uint4 u = make_uint4(0u, 0u, 0u, 0u);
        if (d < dim) u = *reinterpret_cast<const uint4*>(q + d);
        qf[n][2 * j][0] = u.x ^ flip; qf[n][2 * j][1] = u.y ^ flip;
        qf[n][2 * j + 1][0] = u.z ^ flip; qf[n][2 * j + 1][1] = u.w ^ flip;
      }
      float up = 1.f;
      if constexpr (E2M1 && std::is_same<T, __nv_bfloat16>::value) {
        float top = 0.f;
#pragma unroll
        for (int w = 0; w < S::kSteps; ++w)
#pragma unroll
          for (int k = 0; k < 2; ++k) {
            const float2 f = Io<T>::unpack2(qf[n][w][k]);
            top = fmaxf(top, fmaxf(fabsf(f.x), fabsf(f.y)));
          }
        top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 1));
        top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 2));
        // Times 2^-e for 2^e <= top < 2^(e + 1), and the scores times 2^e; rows of
        // zeros or subnormals stay as they are. An infinite element stays one, and
        // the finite ones beside it come into f16's range like those of 2^127.
        const uint32_t e = min(__float_as_uint(top) >> 23, 254u);
        const bool use = e > 0u;
        const float down = use ? __uint_as_float(e < 254u ? (254u - e) << 23 : 0x00400000u) : 1.f;   // 2^-127 is subnormal
        up = use ? __uint_as_float(e << 23) : 1.f;
#pragma unroll
        for (int w = 0; w < S::kSteps; ++w)
#pragma unroll
          for (int k = 0; k < 2; ++k) {
            const float2 f = Io<T>::unpack2(qf[n][w][k]);
            qf[n][w][k] = Io<__half>::pack2(f.x * down, f.y * down);
          }
      }
#pragma unroll
      for (int r = 0; r < 2; ++r) sl2[n][r] = exponent_factor(scale_log2 * __shfl_sync(0xffffffffu, up, 4 * (2 * c + r)));
    }

    // ---------------------------------------------------------- key tiles --
    // O^T: m-tile j holds, in rows g and g + 8, the lane's elements 2 j and
    // 2 j + 1 of V's row, for the query columns 2 c and 2 c + 1.
    constexpr int kMTiles = DP / 16;
    float acc[NT][kMTiles][4];
#pragma unroll
    for (int n = 0; n < NT; ++n)
#pragma unroll
      for (int j = 0; j < kMTiles; ++j)
#pragma unroll
        for (int e = 0; e < 4; ++e) acc[n][j][e] = 0.f;
    // Per column: maximum of the unscaled scores, and this lane's part of the sum.
    // Exponents are (score - maximum) * factor, so the largest is exactly 0
    // however large the scores are (score * factor - maximum * factor in one FMA
    // is off by the rounding of the maximum's product).
    float m[NT][2], l[NT][2];
#pragma unroll
    for (int n = 0; n < NT; ++n) {
      m[n][0] = m[n][1] = -INFINITY;
      l[n][0] = l[n][1] = 0.f;
    }

    int stage = 0;
    for (int i = 0; i < n_tiles; ++i) {
      const int ahead = stage == 0 ? S::kStages - 1 : stage - 1;   // (stage + kStages - 1) % kStages
      if (i + S::kStages - 1 < n_tiles) ok_of[S::kStages - 1] = issue(i + S::kStages - 1, ahead);
      else {
        ok_of[S::kStages - 1] = 0u;
        copy_commit();
      }
      copy_wait<S::kStages - 1>();
      __syncwarp();   // rows copied by other lanes
      const uint32_t ok = ok_of[0];
#pragma unroll
      for (int k = 0; k + 1 < S::kStages; ++k) ok_of[k] = ok_of[k + 1];
      const uint32_t at = ring + stage * S::kStageBytes;
      const int first = key0 + i * KT;
      constexpr uint32_t kFull = KT == 32 ? ~0u : (1u << (KT & 31)) - 1u;
      if (ok != 0u) {
        if constexpr (E2M1) {
          // A masked key's scales may be anything, NaN too: V's must not meet
          // the zero probability of that key. (K's only touch its own scores.)
          if (ok != kFull) {
            if (((ok >> lane) & 1u) == 0u)
              for (int k = 0; k < srow; ++k) sts8(at + S::kKBytes + S::kVBytes + S::kScaleBytes + lane * srow + k, 0u);
            __syncwarp();
          }
        }
        // S^T = K Q^T: m-tiles of 16 keys (rows g and g + 8 of each).
        float sc[NT][KT / 16][4];
#pragma unroll
        for (int n = 0; n < NT; ++n)
#pragma unroll
          for (int a = 0; a < KT / 16; ++a)
#pragma unroll
            for (int e = 0; e < 4; ++e) sc[n][a][e] = 0.f;
        if constexpr (E2M1) {
          const uint32_t k_scales = at + S::kKBytes + S::kVBytes;
          constexpr int kWords = DP / 32;   // words of 8 codes per lane and key
#pragma unroll
          for (int a = 0; a < KT / 16; ++a) {
            uint32_t w[2][kWords], sx[2][2];   // of keys g and g + 8
#pragma unroll
            for (int h = 0; h < 2; ++h) {
              const int key = 16 * a + 8 * h + g;
              if constexpr (DP == 128) {
                const uint4 u = lds128(at + k_place<S, true>(key, c));
                w[h][0] = u.x; w[h][1] = u.y; w[h][2] = u.z; w[h][3] = u.w;
                const uint32_t s01 = scales_to_half2(EXACT || 2 * c < srow ? lds16(k_scales + key * srow + 2 * c) : 0u);
                sx[h][0] = __byte_perm(s01, s01, 0x1010);
                sx[h][1] = __byte_perm(s01, s01, 0x3232);
              } else {
                const uint2 u = lds64(at + k_place<S, true>(key, c >> 1) + 8 * (c & 1));
                w[h][0] = u.x; w[h][1] = u.y;
                sx[h][0] = sx[h][1] = scales_to_half2((EXACT || c < srow ? lds8(k_scales + key * srow + c) : 0u) * 0x101u);
              }
            }
#pragma unroll
            for (int q = 0; q < kWords; ++q) {
              uint32_t x[4], y[4];
              codes_to_half2(w[0][q], x);
              codes_to_half2(w[1][q], y);
              const uint32_t s0 = sx[0][2 * q / kWords], s1 = sx[1][2 * q / kWords];
#pragma unroll
              for (int k = 0; k < 4; ++k) {
                x[k] = hmul2(x[k], s0);
                y[k] = hmul2(y[k], s1);
              }
#pragma unroll
              for (int n = 0; n < NT; ++n) {
                mma16816<M>(sc[n][a], x[0], y[0], x[1], y[1], qf[n][2 * q][0], qf[n][2 * q][1]);
                mma16816<M>(sc[n][a], x[2], y[2], x[3], y[3], qf[n][2 * q + 1][0], qf[n][2 * q + 1][1]);
              }
            }
          }
        } else {
#pragma unroll
          for (int j = 0; j < DP / 32; ++j)
#pragma unroll
            for (int a = 0; a < KT / 16; ++a) {
              const uint4 u = lds128(at + k_place<S, false>(16 * a + g, c + 4 * j));
              const uint4 v = lds128(at + k_place<S, false>(16 * a + 8 + g, c + 4 * j));
#pragma unroll
              for (int n = 0; n < NT; ++n) {
                mma16816<M>(sc[n][a], u.x, v.x, u.y, v.y, qf[n][2 * j][0], qf[n][2 * j][1]);
                mma16816<M>(sc[n][a], u.z, v.z, u.w, v.w, qf[n][2 * j + 1][0], qf[n][2 * j + 1][1]);
              }
            }
        }
        // Masks, where the tile has a key that not every row sees. Element e of
        // m-tile a: key 16 a + 8 (e / 2) + g, column 2 c + e % 2.
        if (ok != kFull || first < all_lo || first + KT > all_hi) {
#pragma unroll
          for (int n = 0; n < NT; ++n)
#pragma unroll
            for (int a = 0; a < KT / 16; ++a)
#pragma unroll
              for (int e = 0; e < 4; ++e) {
                const int local = 16 * a + 8 * (e >> 1) + g, key = first + local;
                if (((ok >> local) & 1u) == 0u || key < lo[n][e & 1] || key >= hi[n][e & 1]) sc[n][a][e] = -INFINITY;
              }
        }
        // Running maxima; NaN propagates, so a NaN score makes its row NaN.
        float top[NT][2];
        bool grown = false;
#pragma unroll
        for (int n = 0; n < NT; ++n)
#pragma unroll
          for (int r = 0; r < 2; ++r) {
            float x = fmax_nan(sc[n][0][r], sc[n][0][2 + r]);
#pragma unroll
            for (int a = 1; a < KT / 16; ++a) x = fmax3_nan(x, sc[n][a][r], sc[n][a][2 + r]);
            x = fmax_nan(x, __shfl_xor_sync(0xffffffffu, x, 4));
            x = fmax_nan(x, __shfl_xor_sync(0xffffffffu, x, 8));
            x = fmax_nan(x, __shfl_xor_sync(0xffffffffu, x, 16));
            top[n][r] = x;
            grown |= !((x - m[n][r]) * sl2[n][r] <= kRescaleLog2);   // (true for NaN, and while a row has seen no key)
          }
        if (__any_sync(0xffffffffu, grown)) {
#pragma unroll
          for (int n = 0; n < NT; ++n)
#pragma unroll
            for (int r = 0; r < 2; ++r) {
              const float next = fmax_nan(m[n][r], top[n][r]);
              const float alpha = next == -INFINITY ? 1.f : ex2_approx((m[n][r] - next) * sl2[n][r]);
              m[n][r] = next;
              l[n][r] *= alpha;
#pragma unroll
              for (int j = 0; j < kMTiles; ++j) {
                acc[n][j][r] *= alpha;
                acc[n][j][2 + r] *= alpha;
              }
            }
        }
        // P^T as the B operand of V^T P^T: 8 x 8 blocks transposed.
        uint32_t pf[NT][KT / 16][2];
#pragma unroll
        for (int n = 0; n < NT; ++n) {
          const float off0 = m[n][0] == -INFINITY ? 0.f : m[n][0], off1 = m[n][1] == -INFINITY ? 0.f : m[n][1];
#pragma unroll
          for (int a = 0; a < KT / 16; ++a) {
#pragma unroll
            for (int e = 0; e < 4; ++e)
              sc[n][a][e] = ex2_approx((sc[n][a][e] - ((e & 1) == 0 ? off0 : off1)) * sl2[n][e & 1]);
            l[n][0] += sc[n][a][0] + sc[n][a][2];
            l[n][1] += sc[n][a][1] + sc[n][a][3];
            pf[n][a][0] = transpose8x8(Io<M>::pack2(sc[n][a][0], sc[n][a][1]));
            pf[n][a][1] = transpose8x8(Io<M>::pack2(sc[n][a][2], sc[n][a][3]));
          }
        }
        // O^T += V^T P^T
#pragma unroll
        for (int a = 0; a < KT / 16; ++a) {
          if constexpr (E2M1) {
            // This lane's columns lie in one scale block. (Where it is behind
            // the head dimension another key's scale is read; those columns
            // are not stored.)
            const uint32_t v_scales = at + S::kKBytes + S::kVBytes + S::kScaleBytes + (DP == 128 ? g : g >> 1);
            uint32_t sx[2];
#pragma unroll
            for (int h = 0; h < 2; ++h) {
              const int key = 16 * a + 8 * h + 2 * c;
              sx[h] = scales_to_half2(lds8(v_scales + key * srow) | (lds8(v_scales + (key + 1) * srow) << 8));
            }
            constexpr int kW = DP / 64;   // words of codes per lane and key
            uint32_t w[2][2][kW];
#pragma unroll
            for (int h = 0; h < 2; ++h)
#pragma unroll
              for (int e = 0; e < 2; ++e) {
                const int key = 16 * a + 8 * h + 2 * c + e;
                if constexpr (DP == 128) {
                  const uint2 u = lds64(at + S::kKBytes + v_place<S, true>(key, g >> 1) + 8 * (g & 1));
                  w[h][e][0] = u.x;
                  w[h][e][1] = u.y;
                } else {
                  w[h][e][0] = lds32(at + S::kKBytes + v_place<S, true>(key, g >> 2) + 4 * (g & 3));
                }
              }
#pragma unroll
            for (int q = 0; q < kW; ++q) {
              // Bytes that pair the codes of two keys: even and odd elements.
              uint32_t ev[2][4], od[2][4];
#pragma unroll
              for (int h = 0; h < 2; ++h) {
                const uint32_t x = w[h][0][q], y = w[h][1][q];
                codes_to_half2((x & 0x0F0F0F0Fu) | ((y << 4) & 0xF0F0F0F0u), ev[h]);
                codes_to_half2(((x >> 4) & 0x0F0F0F0Fu) | (y & 0xF0F0F0F0u), od[h]);
#pragma unroll
                for (int j = 0; j < 4; ++j) {
                  ev[h][j] = hmul2(ev[h][j], sx[h]);
                  od[h][j] = hmul2(od[h][j], sx[h]);
                }
              }
#pragma unroll
              for (int j = 0; j < 4; ++j)
#pragma unroll
                for (int n = 0; n < NT; ++n)
                  mma16816<M>(acc[n][4 * q + j], ev[0][j], od[0][j], ev[1][j], od[1][j], pf[n][a][0], pf[n][a][1]);
            }
          } else {
#pragma unroll
            for (int j = 0; j < DP / 64; ++j) {
              uint32_t w[4][4];   // [key][word]
#pragma unroll
              for (int e = 0; e < 4; ++e) {
                const uint4 u = lds128(at + S::kKBytes + v_place<S, false>(16 * a + 8 * (e >> 1) + 2 * c + (e & 1), g + 8 * j));
                w[e][0] = u.x; w[e][1] = u.y; w[e][2] = u.z; w[e][3] = u.w;
              }
#pragma unroll
              for (int q = 0; q < 4; ++q) {
                const uint32_t a0 = __byte_perm(w[0][q], w[1][q], 0x5410), a1 = __byte_perm(w[0][q], w[1][q], 0x7632);
                const uint32_t a2 = __byte_perm(w[2][q], w[3][q], 0x5410), a3 = __byte_perm(w[2][q], w[3][q], 0x7632);
#pragma unroll
                for (int n = 0; n < NT; ++n) mma16816<M>(acc[n][4 * j + q], a0, a1, a2, a3, pf[n][a][0], pf[n][a][1]);
              }
            }
          }
        }
      }
      __syncwarp();   // the stage may be written again
      stage = stage + 1 == S::kStages ? 0 : stage + 1;
    }
    copy_wait<0>();

    // ------------------------------------------------------------- results --
#pragma unroll
    for (int n = 0; n < NT; ++n)
#pragma unroll
      for (int r = 0; r < 2; ++r)
#pragma unroll
        for (int o = 4; o < 32; o <<= 1) l[n][r] += __shfl_xor_sync(0xffffffffu, l[n][r], o);
    const bool whole = tile0 == 0 && n_tiles == seg_tiles;
    const int64_t part = static_cast<int64_t>(worker) * 2 + (t == t_first ? 0 : 1);
#pragma unroll
    for (int n = 0; n < NT; ++n)
#pragma unroll
      for (int r = 0; r < 2; ++r) {
        const int in_tile = 8 * n + 2 * c + r, row = row0 + in_tile;
        if (in_tile < rows) {
          const bool none = l[n][r] == 0.f;
          const float f = whole ? p.v_gain / l[n][r] : 1.f;
          const int i = row / p.group;
          T* out = static_cast<T*>(p.o) + (s.first + i) * p.o_tok + (kh * p.group + row - i * p.group) * p.o_head;
          float* po = p.part_o + (part * S::kRows + in_tile) * DP;
          // The lane's kRun neighbouring elements kRun g + 64 k ..
#pragma unroll
          for (int k = 0; k < DP / (8 * S::kRun); ++k)
#pragma unroll
            for (int d8 = 0; d8 < S::kRun; d8 += 8) {
              const int d = 64 * k + S::kRun * g + d8, j0 = (S::kRun * k + d8) / 2;
              float x[8];
#pragma unroll
              for (int e = 0; e < 8; ++e) x[e] = none ? 0.f : acc[n][j0 + (e >> 1)][2 * (e & 1) + r] * f;
              if (whole) {
                if (d < dim)
                  *reinterpret_cast<uint4*>(out + d) = make_uint4(Io<T>::pack2(x[0], x[1]), Io<T>::pack2(x[2], x[3]),
                                                                  Io<T>::pack2(x[4], x[5]), Io<T>::pack2(x[6], x[7]));
              } else {
                *reinterpret_cast<float4*>(po + d) = make_float4(x[0], x[1], x[2], x[3]);
                *reinterpret_cast<float4*>(po + d + 4) = make_float4(x[4], x[5], x[6], x[7]);
              }
            }
          if (!whole && g == 0)
            *reinterpret_cast<float4*>(p.part_ml + (part * S::kRows + in_tile) * kPartMl) = make_float4(m[n][r], l[n][r], sl2[n][r], 0.f);
        }
      }
    t += n_tiles;
    if (t >= t_end && lane == 0) {
      Cut cut{};
      if (tile0 == 0 && n_tiles < seg_tiles) {
        cut.parts = run_of(total, workers, t - n_tiles + seg_tiles - 1) - worker + 1;
        cut.slot = t - n_tiles == t_first ? 0 : 1;
        cut.rows = rows;
        cut.first_token = s.first;
        cut.row0 = row0;
        cut.kv_head = kh;
      }
      p.cuts[worker] = cut;
    }
  }
}

// ------------------------------------------------------------------- host --
template <typename T, bool E2M1>
cudaError_t run_simple(const PagedParams& p, cudaStream_t s) {
  const dim3 grid(static_cast<unsigned>(ceil_div64(p.seqs.tokens, kSimpleThreads / 32)), p.q_heads);
  return launch_pdl(paged_simple_kernel<T, E2M1>, grid, dim3(kSimpleThreads), 0, s, p);
}

int padded_dim(int64_t dim) { return dim <= 64 ? 64 : 128; }

// 8-row tiles that share the keys, by the likely query rows of a sequence (the
// caller's hint, else the mean). One tile needs half the accumulators and
// exponentials and leaves room for more warps, two read the keys once for 16 rows.
// With 4 bits each key is converted again for every row tile, so two pay from 9
// rows on (four 131072-key contexts of 4 rows: 155 us with two, 132 with one). With
// 16 bits they pay from 17 rows on where the second reading comes from L2 (8 x 4096
// keys, 8 key heads of 128, 134 MB: 16 rows 42 us with one, 54 with two; 32 rows 64
// and 57), and from 9 on in larger caches (32 sequences of up to 4096 keys, at most
// 537 MB: 16 rows 98 and 89; 2 x 32768 keys, 268 MB: 108 and 109, 32 rows 183 and
// 106). The page table bounds the size.
int row_tiles_of(const lunarad_paged_attention_args& a) {
  const lunarad_cache& c = *a.cache;
  const int64_t mean = (a.seqs.tokens + a.seqs.batch - 1) / a.seqs.batch;
  const int64_t hint = a.max_q_len < a.seqs.tokens ? a.max_q_len : a.seqs.tokens;
  const int64_t rows = (hint > 0 ? hint : mean) * (a.q_heads / c.kv_heads);
  const double bytes = 4.0 * static_cast<double>(c.kv_heads * c.dim) * static_cast<double>(c.page_size * a.seqs.max_pages) *
                       static_cast<double>(a.seqs.batch);
  return rows <= (c.kind != LUNARAD_KIND_E2M1 && bytes < 200e6 ? 16 : 8) ? 1 : 2;
}
int stream_workers(bool e2m1, int nt, int sms) { return sms * kWarps * ((e2m1 ? 3 : 2) + (nt == 1 ? 1 : 0)); }

bool al16(const void* p) { return (reinterpret_cast<uintptr_t>(p) & 15u) == 0; }

// Bytes of the unit in which the streaming kernel keeps where a page and row
// stands, in 32 bits: 64 where all strides allow it (so that 256 GiB are
// reached), else 16. 0 when a page stands beyond that.
int place_unit(const lunarad_cache& c) {
  const bool e2m1 = c.kind == LUNARAD_KIND_E2M1;
  const int64_t elem = e2m1 ? 1 : 2, row = e2m1 ? c.dim / 2 : c.dim * 2;
  const int64_t step = c.page_size % 8 == 0 ? 8 * row : row;   // rows are looked up by groups of 8, or one by one
  const int64_t kp = c.k_page_stride * elem, vp = c.v_page_stride * elem;
  const int64_t unit = step % 64 == 0 && row % 64 == 0 && kp % 64 == 0 && vp % 64 == 0 ? 64 : 16;
  const int64_t most = int64_t{1} << 31, pages = c.num_pages;
  if (kp < 0 || vp < 0 || c.ks_page_stride < 0 || c.vs_page_stride < 0) return 0;
  const int64_t used = c.page_size * row / unit + 1;
  if (kp / unit * pages + used >= 2 * most || vp / unit * pages + used >= 2 * most) return 0;
  if (e2m1 && (c.ks_page_stride / 16 * pages + c.page_size * c.dim / 256 + 1 >= 2 * most ||
               c.vs_page_stride / 16 * pages + c.page_size * c.dim / 256 + 1 >= 2 * most))
    return 0;
  return static_cast<int>(unit);
}

// 16-byte copies of whole rows: aligned bases and strides, rows of 16-byte
// pieces; for 4 bits also pages of whole groups of 8 keys. A cache without pages
// has no place that a copy of nothing could name.
bool stream_ok(const lunarad_paged_attention_args& a) {
  const lunarad_cache& c = *a.cache;
  const bool e2m1 = c.kind == LUNARAD_KIND_E2M1;
  if (a.dtype == LUNARA_F32 || c.dim > 128 || c.num_pages == 0) return false;
  if (!al16(a.q.data) || a.q.head_stride % 8 || a.q.seq_stride % 8) return false;
  if (!al16(a.o.data) || a.o.head_stride % 8 || a.o.seq_stride % 8) return false;
  if (!al16(c.k) || !al16(c.v) || place_unit(c) == 0) return false;
  const int64_t vec = e2m1 ? 16 : 8;
  if (c.k_page_stride % vec || c.k_head_stride % vec || c.v_page_stride % vec || c.v_head_stride % vec) return false;
  if (!e2m1) return c.dim % 8 == 0;
  return c.dim % 32 == 0 && c.page_size % 8 == 0 && al16(c.k_scales) && al16(c.v_scales) && c.ks_page_stride % 16 == 0 &&
         c.ks_head_stride % 16 == 0 && c.vs_page_stride % 16 == 0 && c.vs_head_stride % 16 == 0;
}

// Sequences with this many query rows go to the tcgen05 kernel where it takes
// the cache: there the streaming kernel would read the keys a third time (8 x 4096
// keys, 8 key heads of 128: 32 rows 57 us streaming, 68 on tcgen05, 48 rows 73 and
// 69; 2 x 32768 keys: 106 and 95, 165 and 96).
constexpr int64_t kPrefillRows = 33;

bool prefill_ok(const lunarad_paged_attention_args& a) {
  const lunarad_cache& c = *a.cache;
  const int64_t group = a.q_heads / c.kv_heads;
  // Tokens of a sequence at most, as far as is known. No more tokens than
  // sequences: a decode step, which the second pair of launches would cost 8 us
  // (the streaming kernel is right for any sequence).
  int64_t most = a.seqs.tokens <= a.seqs.batch ? 1 : a.seqs.tokens;
  if (a.max_q_len > 0) most = a.max_q_len < a.seqs.tokens ? a.max_q_len : a.seqs.tokens;
  return stream_ok(a) && a.scale >= 0 && c.kind != LUNARAD_KIND_E2M1 && most * group >= kPrefillRows;
}

int64_t stream_workspace(const lunarad_paged_attention_args& a, int sms) {
  const int nt = row_tiles_of(a);
  const int64_t rows = int64_t{2} * stream_workers(a.cache->kind == LUNARAD_KIND_E2M1, nt, sms) * 8 * nt;
  return rows * (padded_dim(a.cache->dim) + kPartMl) * static_cast<int64_t>(sizeof(float)) + rows / (16 * nt) * static_cast<int64_t>(sizeof(Cut));
}

template <typename T, bool E2M1, int DP, int NT, bool EXACT>
cudaError_t run_stream(PagedParams p, cudaStream_t s) {
  using S = Shape<E2M1, DP, NT>;
  const size_t prefix = sizeof(int64_t) * (static_cast<size_t>(p.seqs.batch < kMaxBatch ? p.seqs.batch : kMaxBatch) + 2);
  const size_t smem = static_cast<size_t>(kWarps) * S::kRingBytes + prefix;
  static_assert(kWarps * S::kRingBytes + 8 * (kMaxBatch + 2) + 1280 <= 228 * 1024 / S::kCtasPerSm, "shared memory per SM");
  auto kern = paged_stream_kernel<T, E2M1, DP, NT, EXACT>;
  static std::atomic<uint64_t> prepared{0};
  cudaError_t e = prepare_once(kern, prepared, kWarps * S::kRingBytes + 8 * (kMaxBatch + 2), 0);
  if (e != cudaSuccess) return e;
  const int batch = p.seqs.batch, zero_rest = p.zero_behind;
  const Seqs all = p.seqs;
  for (int b0 = 0; b0 < batch; b0 += kMaxBatch) {   // more sequences than the prefix sums hold: one after the other
    p.seqs.batch = batch - b0 < kMaxBatch ? batch - b0 : kMaxBatch;
    p.seqs.page_table = all.page_table + b0 * all.table_stride;
    p.seqs.starts = all.starts + b0;
    p.seqs.lens = all.lens + b0;
    p.zero_before = zero_rest && b0 == 0;
    p.zero_behind = zero_rest && b0 + p.seqs.batch == batch;
    e = launch_pdl(kern, dim3(p.workers / kWarps), dim3(kStreamThreads), smem, s, p);
    if (e != cudaSuccess) return e;
    e = launch_pdl(paged_join_kernel<T, DP>, dim3(join_blocks(p.workers), 4), dim3(kJoinThreads), 0, s, p, int{S::kRows});
    if (e != cudaSuccess) return e;
  }
  return cudaSuccess;
}

template <typename T, bool E2M1, int NT>
cudaError_t run_stream_dim(const PagedParams& p, cudaStream_t s) {
  if (p.dim == 64) return run_stream<T, E2M1, 64, NT, true>(p, s);
  if (p.dim < 64) return run_stream<T, E2M1, 64, NT, false>(p, s);
  return p.dim == 128 ? run_stream<T, E2M1, 128, NT, true>(p, s) : run_stream<T, E2M1, 128, NT, false>(p, s);
}

template <typename T>
cudaError_t run(const PagedParams& p, bool stream_kernel, bool e2m1, cudaStream_t s) {
  if constexpr (!std::is_same<T, float>::value) {
    if (stream_kernel) {
      if (e2m1) return p.nt == 1 ? run_stream_dim<T, true, 1>(p, s) : run_stream_dim<T, true, 2>(p, s);
      return p.nt == 1 ? run_stream_dim<T, false, 1>(p, s) : run_stream_dim<T, false, 2>(p, s);
    }
  }
  return e2m1 ? run_simple<T, true>(p, s) : run_simple<T, false>(p, s);
}

}  // namespace

int64_t paged_attention_workspace(const lunarad_paged_attention_args& a, int sms) {
  if (!stream_ok(a)) return 0;
  return stream_workspace(a, sms) + (prefill_ok(a) ? paged_prefill_workspace(static_cast<int>(a.cache->dim), sms) : 0);
}

cudaError_t launch_paged_attention(const lunarad_paged_attention_args& a, bool zero_rest, void* workspace, cudaStream_t stream) {
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
  p.min_rows = 0;
  p.max_rows = INT64_MAX;
  const bool stream_kernel = stream_ok(a);
  if (stream_kernel) {
    p.unit = static_cast<uint32_t>(place_unit(c));
    const int64_t elem = e2m1 ? 1 : 2;
    p.k_page_u = static_cast<uint32_t>(c.k_page_stride * elem / p.unit);
    p.v_page_u = static_cast<uint32_t>(c.v_page_stride * elem / p.unit);
    p.row_u = static_cast<uint32_t>((e2m1 ? c.dim / 2 : c.dim * 2) / p.unit);
    p.ks_page_u = static_cast<uint32_t>(c.ks_page_stride / 16);
    p.vs_page_u = static_cast<uint32_t>(c.vs_page_stride / 16);
    p.nt = row_tiles_of(a);
    p.workers = stream_workers(e2m1, p.nt, device_num_sms());
    p.part_o = static_cast<float*>(workspace);
    p.part_ml = p.part_o + int64_t{2} * p.workers * 8 * p.nt * padded_dim(c.dim);
    p.cuts = reinterpret_cast<Cut*>(p.part_ml + int64_t{2} * p.workers * 8 * p.nt * kPartMl);
  }
  p.err = device_error_word();
  if (p.err == nullptr) return cudaErrorInvalidDevice;
  if (prefill_ok(a)) {   // (the rows of no sequence are the other kernel's)
    PagedParams q = p;
    q.min_rows = p.max_rows = kPrefillRows;
    const cudaError_t e = launch_paged_prefill(q, static_cast<int>(a.dtype),
                                               static_cast<char*>(workspace) + stream_workspace(a, device_num_sms()), stream);
    if (e != cudaSuccess) return e;
  }
  p.zero_before = p.zero_behind = zero_rest;
  if (a.dtype == LUNARA_F16) return run<__half>(p, stream_kernel, e2m1, stream);
  if (a.dtype == LUNARA_BF16) return run<__nv_bfloat16>(p, stream_kernel, e2m1, stream);
  return run<float>(p, stream_kernel, e2m1, stream);
}

}  // namespace lunara
