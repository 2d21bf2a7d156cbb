// Device helpers shared by the kernels that deal with ragged sequences and the
// paged key/value cache.
#pragma once

#include "common.cuh"
#include "decoder.h"

namespace lunara {

// Quotient by a divisor fixed at launch, for 0 <= n < 2^31 (Granlund and
// Montgomery, "Division by invariant integers using multiplication", 1994):
// with l = ceil(log2 d) and m = floor(2^32 (2^l - d) / d) + 1,
// n / d = (umulhi(m, n) + n) >> l. The sum stays below 2^32 for such n.
struct FastDiv {
  uint32_t d, m, l;
  __host__ void init(uint32_t div) {
    d = div;
    l = 0;
    while ((uint64_t{1} << l) < div) ++l;
    m = static_cast<uint32_t>(((uint64_t{1} << 32) * ((uint64_t{1} << l) - div)) / div + 1);
  }
  __device__ __forceinline__ int div(int n) const {
    const uint32_t u = static_cast<uint32_t>(n);
    return static_cast<int>((__umulhi(m, u) + u) >> l);
  }
};

// Device form of lunarad_sequences.
struct Seqs {
  const int32_t* page_table;
  const int32_t* starts;
  const int32_t* lens;
  int64_t table_stride;
  int max_pages, batch, tokens;
  FastDiv page_div;   // by the page size
};

inline Seqs make_seqs(const lunarad_sequences& s, int64_t page_size) {
  Seqs d{};
  d.page_table = s.page_table;
  d.starts = s.seq_starts;
  d.lens = s.seq_lens;
  d.table_stride = s.table_stride;
  d.max_pages = static_cast<int>(s.max_pages);
  d.batch = static_cast<int>(s.batch);
  d.tokens = static_cast<int>(s.tokens);
  d.page_div.init(static_cast<uint32_t>(page_size));
  return d;
}

// The sequence that owns `token`, and its position in it. False when no
// sequence owns it (behind the last one). Whatever the arrays hold, `seq` is
// in [0, batch). The first probe assumes one token per sequence, which a
// decode step has: there it answers after one memory latency.
__device__ __forceinline__ bool find_token(const Seqs& s, int token, int& seq, int64_t& pos) {
  const int guess = token < s.batch ? token : s.batch - 1;
  int s1 = s.starts[guess + 1];
  int len = s.lens[guess];
  seq = guess;
  if (!(s.starts[guess] <= token && token < s1)) {
    int lo = 0, hi = s.batch;   // last b in [0, batch) with starts[b] <= token
    while (lo + 1 < hi) {
      const int mid = (lo + hi) >> 1;
      if (s.starts[mid] <= token) lo = mid; else hi = mid;
    }
    seq = lo;
    s1 = s.starts[lo + 1];
    if (token >= s1 || token < s.starts[lo]) return false;
    len = s.lens[lo];
  }
  pos = static_cast<int64_t>(len) - (static_cast<int64_t>(s1) - token);
  return true;
}

// Page number and slot of a position of a sequence; -1 with a device error for
// a position behind the page table or a page outside the cache. pos >= 0.
__device__ __forceinline__ int find_page(const Seqs& s, int seq, int64_t pos, int num_pages, int& slot,
                                         unsigned int* err) {
  if (pos >= (int64_t{1} << 31) || s.page_div.div(static_cast<int>(pos)) >= s.max_pages) {
    atomicCAS(err, 0u, static_cast<unsigned>(kErrCachePosition));
    return -1;
  }
  const int pi = s.page_div.div(static_cast<int>(pos));
  slot = static_cast<int>(pos) - pi * static_cast<int>(s.page_div.d);
  const int page = s.page_table[seq * s.table_stride + pi];
  if (page < 0 || page >= num_pages) {
    atomicCAS(err, 0u, static_cast<unsigned>(kErrCachePage));
    return -1;
  }
  return page;
}

// ---------------------------------------------------------- 4-bit formats --
// Two e2m1 codes of a byte as an f16 pair (low nibble in the low half), exact.
__device__ __forceinline__ __half2 e2m1x2_to_half2(uint32_t byte) {
  uint32_t r;
  asm("{\n\t.reg .b8 t, u;\n\t"
      "cvt.u8.u32 t, %1;\n\t"
      "cvt.rn.f16x2.e2m1x2 %0, t;\n\t}"
      : "=r"(r)
      : "r"(byte));
  return *reinterpret_cast<__half2*>(&r);
}

// The nearest e2m1 codes (ties to even, saturating at 6) of a pair as a byte.
__device__ __forceinline__ uint32_t float2_to_e2m1x2(float lo, float hi) {
  uint32_t r;
  asm("{\n\t.reg .b8 t;\n\t"
      "cvt.rn.satfinite.e2m1x2.f32 t, %2, %1;\n\t"
      "cvt.u32.u8 %0, t;\n\t}"
      : "=r"(r)
      : "f"(lo), "f"(hi));
  return r;
}

__device__ __forceinline__ uint32_t float_to_e4m3(float v) {
  uint16_t r;
  asm("cvt.rn.satfinite.e4m3x2.f32 %0, %1, %2;" : "=h"(r) : "f"(0.f), "f"(v));
  return r & 0xFFu;
}

__device__ __forceinline__ float e4m3_to_float(uint32_t byte) {
  uint32_t r;
  asm("cvt.rn.f16x2.e4m3x2 %0, %1;" : "=r"(r) : "h"(static_cast<uint16_t>(byte)));
  return __low2float(*reinterpret_cast<__half2*>(&r));
}

}  // namespace lunara
