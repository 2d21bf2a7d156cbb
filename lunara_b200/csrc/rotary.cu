// Rotary positions, per-head query/key norms with the rotation, and appending
// to and reading from the paged key/value cache: kernels that move rows of one
// head's elements ("rows") once, bound by HBM when there are many tokens and by
// memory latency in a decode step.
//
// Mathematics. A pair (a, b) of a row at position p becomes
//   (a cos - b sin, b cos + a sin),  (cos, sin) = table[p][pair]
// with pairs (i, i + rot/2) or (2i, 2i + 1), elements from rot on unchanged;
// the norm before it is x * rsqrt(mean(x^2) + eps) * w. All of it in fp32 with
// one rounding at the end. The rotation's products and sums are rounded one by
// one (no contraction into FMAs), so that the 4-bit codes made from them are
// the same in any implementation of the definition.
//
// Work split. A lane holds two 8-element vectors of a row, one in each half of
// the rotated elements (or of those behind them), so a pair of either layout
// never crosses lanes, rotation in place is safe, and neighbouring lanes access
// neighbouring 16 bytes. The (cos, sin) of its 8 pairs stay in registers while
// the lane walks over kHeads heads of the token: the fp32 table (64 bytes per
// lane) is read once for them instead of once per head. The rows are loaded
// before anything is known of the position, so that the chain of dependent
// loads is (sequence, page) or position, table, and nothing more.
#include "kernels.h"
#include "paged.cuh"

namespace lunara {
namespace {

constexpr int kThreads = 128;

// 8 consecutive elements (16-byte aligned) as loaded, as floats, and back.
template <typename T>
struct Raw8 {
  uint4 v[sizeof(T) / 2];
};

template <typename T>
__device__ __forceinline__ Raw8<T> load_raw(const T* p) {
  Raw8<T> r;
#pragma unroll
  for (int i = 0; i < static_cast<int>(sizeof(T) / 2); ++i) r.v[i] = reinterpret_cast<const uint4*>(p)[i];
  return r;
}

template <typename T>
__device__ __forceinline__ void unpack(const Raw8<T>& r, float (&f)[8]) {
  const uint4 u = r.v[0];
  if constexpr (sizeof(T) == 4) {
    const uint4 v = r.v[1];
    f[0] = __uint_as_float(u.x); f[1] = __uint_as_float(u.y); f[2] = __uint_as_float(u.z); f[3] = __uint_as_float(u.w);
    f[4] = __uint_as_float(v.x); f[5] = __uint_as_float(v.y); f[6] = __uint_as_float(v.z); f[7] = __uint_as_float(v.w);
  } else {
    const float2 a = Io<T>::unpack2(u.x), b = Io<T>::unpack2(u.y), c = Io<T>::unpack2(u.z), d = Io<T>::unpack2(u.w);
    f[0] = a.x; f[1] = a.y; f[2] = b.x; f[3] = b.y; f[4] = c.x; f[5] = c.y; f[6] = d.x; f[7] = d.y;
  }
}

template <typename T>
__device__ __forceinline__ void load8(const T* p, float (&f)[8]) {
  unpack<T>(load_raw(p), f);
}

template <typename T>
__device__ __forceinline__ void store8(T* p, const float (&f)[8]) {
  if constexpr (sizeof(T) == 4) {
    *reinterpret_cast<float4*>(p) = make_float4(f[0], f[1], f[2], f[3]);
    *reinterpret_cast<float4*>(p + 4) = make_float4(f[4], f[5], f[6], f[7]);
  } else {
    uint4 u;
    u.x = Io<T>::pack2(f[0], f[1]);
    u.y = Io<T>::pack2(f[2], f[3]);
    u.z = Io<T>::pack2(f[4], f[5]);
    u.w = Io<T>::pack2(f[6], f[7]);
    *reinterpret_cast<uint4*>(p) = u;
  }
}

__device__ __forceinline__ void turn(float& a, float& b, float c, float s) {
  const float x = __fsub_rn(__fmul_rn(a, c), __fmul_rn(b, s));
  b = __fadd_rn(__fmul_rn(b, c), __fmul_rn(a, s));
  a = x;
}

// One group of heads: strided rows in, strided rows or cache slots out.
struct RowSet {
  const void* src;
  void* dst;
  int64_t sb, sh, ss;      // source strides (batch, head, seq)
  int64_t db, dh, ds;      // destination strides; paged: db = page, dh = head, ds = slot (dim)
  const void* weight;      // norm weight or NULL
  int heads;
  int rotate, paged;
};

struct RowsParams {
  RowSet set[3];
  int group_end[3];        // head groups of sets 0..i, cumulated
  // positions: given, or from the sequences
  const void* positions;
  int position_bytes;
  int64_t position_batch_stride;
  Seqs seqs;
  int num_pages;
  const float* table;
  int64_t table_positions;
  int rot, dim, units, lanes_log2;
  int tokens, seq;         // tokens = batch * seq
  int inverse;
  int zero_rest;           // rows of tokens that no sequence owns: zero, not left alone
  float eps;
  unsigned int* err;
};

// Where a token stands: its batch index and seq index in the views, its
// position, and (paged) its page and slot.
struct TokenPlace {
  int b, s, page, slot;
  int64_t pos;
  bool owned;    // false: nothing of the token is touched
  bool valid;    // false: its rows are zero, nothing goes to the cache
};

template <bool PAGED>
__device__ __forceinline__ TokenPlace place_token(const RowsParams& p, int token, bool needs_table) {
  TokenPlace t;
  t.owned = token < p.tokens;
  t.valid = false;
  t.page = -1;
  t.slot = 0;
  t.pos = 0;
  t.b = 0;
  t.s = token;
  if (!t.owned) return t;
  if constexpr (PAGED) {
    int seq;
    if (!find_token(p.seqs, token, seq, t.pos)) {
      t.owned = p.zero_rest != 0;
      return t;
    }
    if (t.pos < 0) return t;
    t.page = find_page(p.seqs, seq, t.pos, p.num_pages, t.slot, p.err);
    t.valid = t.page >= 0;
  } else {
    t.b = token / p.seq;
    t.s = token - t.b * p.seq;
    const int64_t i = t.b * p.position_batch_stride + t.s;
    t.pos = p.position_bytes == 8 ? static_cast<const int64_t*>(p.positions)[i]
                                  : static_cast<const int32_t*>(p.positions)[i];
    t.valid = true;
  }
  if (t.valid && needs_table && (t.pos < 0 || t.pos >= p.table_positions)) {
    atomicCAS(p.err, 0u, static_cast<unsigned>(kErrRotaryPosition));
    t.valid = false;
  }
  return t;
}

// The 4-bit form of a scale block of 16 elements.
struct QuantParams {
  RowsParams r;
  void* scales[3];
  int64_t sc_page[3], sc_head[3];
  float inv_gain[3];
  int blocks;   // dim / 16
};

// code = e2m1(y / s), the quotient rounded to nearest as IEEE division does:
// with r = RN(1/s), q0 = RN(y r) and the exact remainder q0 s - y, RN(q0 -
// remainder * r) is the correctly rounded quotient (Markstein, 1990; s has 4
// significant bits, so the all-ones exception of the theorem cannot arise).
// The remainder is taken with this sign so that a negative zero stays one: its
// remainder is +0, and -0 - 0 r = -0 (with y - q0 s the sum would be +0).
__device__ __forceinline__ float quotient(float y, float s, float r) {
  const float q0 = __fmul_rn(y, r);
  return __fmaf_rn(-__fmaf_rn(q0, s, -y), r, q0);
}

// The e4m3 scale of a block whose largest magnitude is amax (saturates at 448,
// keeps NaN), and the codes of N of its elements, 4 bits each.
template <int N>
__device__ __forceinline__ uint32_t quantise(const float (&y)[N], int first, float amax, uint32_t& scale) {
  // amax / 6 correctly rounded in the same way (beyond 1e30 it saturates anyway).
  const float top = amax > 1e30f ? 1e30f : amax;
  scale = float_to_e4m3(quotient(top, 6.0f, 1.0f / 6.0f));
  const float s = e4m3_to_float(scale);
  uint32_t w = 0u;
  if (s > 0.f) {
    const float r = __frcp_rn(s);
    if (amax < 1e30f) {
#pragma unroll
      for (int i = 0; i < 8; i += 2)
        w |= float2_to_e2m1x2(quotient(y[first + i], s, r), quotient(y[first + i + 1], s, r)) << (4 * i);
    } else {   // the quotient's remainder may overflow: there, any quotient saturates or is tiny
#pragma unroll 1
      for (int i = 0; i < 8; i += 2)
        w |= float2_to_e2m1x2(__fdiv_rn(y[first + i], s), __fdiv_rn(y[first + i + 1], s)) << (4 * i);
    }
  }
  return w;
}

// QUANT: paged rows go to a 4-bit cache; a scale block belongs to two
// neighbouring lanes.
template <typename T, int LAYOUT, bool NORM, bool PAGED, bool QUANT, int HEADS>
__global__ void __launch_bounds__(kThreads) rows_kernel(const __grid_constant__ QuantParams q) {
  const RowsParams& p = q.r;
  pdl_wait();
  pdl_launch_dependents();
  const int lanes = 1 << p.lanes_log2;
  const int token = static_cast<int>(blockIdx.x) * (kThreads >> p.lanes_log2) + (static_cast<int>(threadIdx.x) >> p.lanes_log2);
  const int u = static_cast<int>(threadIdx.x) & (lanes - 1);
  int which = 0;
  while (which < 2 && static_cast<int>(blockIdx.y) >= p.group_end[which]) ++which;
  const RowSet& set = p.set[which];
  const int h0 = (static_cast<int>(blockIdx.y) - (which ? p.group_end[which - 1] : 0)) * HEADS;
  const int nh = min(HEADS, set.heads - h0);
  const bool lane_in = token < p.tokens && u < p.units;
  const bool turns = 16 * u < p.rot;
  const int o0 = turns ? 8 * u : p.rot / 2 + 8 * u;                                  // rot + 8 (u - rot / 16)
  const int o1 = turns ? p.rot / 2 + 8 * u : p.dim / 2 + 8 * u;                      // rot + (dim - rot) / 2 + 8 (u - rot / 16)
  Raw8<T> ra[HEADS], rb[HEADS];
  if (lane_in) {
    const int sb = PAGED ? 0 : token / p.seq, ss = PAGED ? token : token - sb * p.seq;
    const T* src = static_cast<const T*>(set.src) + sb * set.sb + ss * set.ss + h0 * set.sh;
#pragma unroll
    for (int h = 0; h < HEADS; ++h)
      if (h < nh) {
        ra[h] = load_raw(src + h * set.sh + o0);
        rb[h] = load_raw(src + h * set.sh + o1);
      }
  }
  const TokenPlace t = place_token<PAGED>(p, token, p.rot > 0);
  const bool rotate = set.rotate && turns;
  float cs[16];
  if (lane_in && t.valid && rotate) {
    const float* row = p.table + t.pos * p.rot;
    const float* c0 = row + (LAYOUT == LUNARAD_ROTARY_HALF ? 16 * u : o0);
    const float* c1 = LAYOUT == LUNARAD_ROTARY_HALF ? c0 + 8 : row + o1;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const float4 v = __ldg(reinterpret_cast<const float4*>(i < 2 ? c0 : c1) + (i & 1));
      cs[4 * i] = v.x; cs[4 * i + 1] = v.y; cs[4 * i + 2] = v.z; cs[4 * i + 3] = v.w;
    }
    if (p.inverse) {
#pragma unroll
      for (int i = 0; i < 8; ++i) cs[2 * i + 1] = -cs[2 * i + 1];
    }
  }
  Raw8<T> rw0, rw1;
  const bool weighted = NORM && set.weight != nullptr;
  if (weighted && lane_in) {
    rw0 = load_raw(static_cast<const T*>(set.weight) + o0);
    rw1 = load_raw(static_cast<const T*>(set.weight) + o1);
  }
  const float inv_dim = 1.0f / static_cast<float>(p.dim);
  const bool stores = lane_in && t.owned && (t.valid || !set.paged);
  char* dst = static_cast<char*>(set.dst);
  const int elem = QUANT && set.paged ? 1 : static_cast<int>(sizeof(T));
  if (stores) dst += (set.paged ? t.page * set.db + t.slot * set.ds : t.b * set.db + t.s * set.ds) * elem + h0 * set.dh * elem;
#pragma unroll
  for (int h = 0; h < HEADS; ++h) {
    if (h >= nh) break;   // the same in all lanes
    float a[8], b[8];
    unpack<T>(ra[h], a);
    unpack<T>(rb[h], b);
    if constexpr (NORM) {
      float ss = 0.f;
      if (lane_in) {
#pragma unroll
        for (int i = 0; i < 8; ++i) ss = fmaf(a[i], a[i], fmaf(b[i], b[i], ss));
      }
      for (int o = lanes >> 1; o > 0; o >>= 1) ss += __shfl_xor_sync(0xffffffffu, ss, o);
      const float r = rsqrtf(fmaf(ss, inv_dim, p.eps));
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        a[i] *= r;
        b[i] *= r;
      }
      if (weighted) {
        float w[8];
        unpack<T>(rw0, w);
#pragma unroll
        for (int i = 0; i < 8; ++i) a[i] *= w[i];
        unpack<T>(rw1, w);
#pragma unroll
        for (int i = 0; i < 8; ++i) b[i] *= w[i];
      }
    }
    if (!t.valid) {
#pragma unroll
      for (int i = 0; i < 8; ++i) a[i] = b[i] = 0.f;
    } else if (rotate) {
      if (LAYOUT == LUNARAD_ROTARY_HALF) {
#pragma unroll
        for (int i = 0; i < 8; ++i) turn(a[i], b[i], cs[2 * i], cs[2 * i + 1]);
      } else {
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          turn(a[2 * i], a[2 * i + 1], cs[2 * i], cs[2 * i + 1]);
          turn(b[2 * i], b[2 * i + 1], cs[8 + 2 * i], cs[8 + 2 * i + 1]);
        }
      }
    }
    char* row = dst + h * set.dh * elem;
    if (QUANT && set.paged) {   // (the same in all lanes)
      float top[2] = {0.f, 0.f};
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        a[i] = __fmul_rn(a[i], q.inv_gain[which]);
        b[i] = __fmul_rn(b[i], q.inv_gain[which]);
        top[0] = fmax_nan(top[0], fabsf(a[i]));
        top[1] = fmax_nan(top[1], fabsf(b[i]));
      }
#pragma unroll
      for (int k = 0; k < 2; ++k) top[k] = fmax_nan(top[k], __shfl_xor_sync(0xffffffffu, top[k], 1));
      uint32_t s0, s1;
      const uint32_t w0 = quantise(a, 0, top[0], s0), w1 = quantise(b, 0, top[1], s1);
      if (stores) {
        *reinterpret_cast<uint32_t*>(row + o0 / 2) = w0;
        *reinterpret_cast<uint32_t*>(row + o1 / 2) = w1;
        if ((u & 1) == 0) {
          uint8_t* sc = static_cast<uint8_t*>(q.scales[which]) + t.page * q.sc_page[which] + (h0 + h) * q.sc_head[which] +
                        static_cast<int64_t>(t.slot) * q.blocks;
          sc[o0 / 16] = static_cast<uint8_t>(s0);
          sc[o1 / 16] = static_cast<uint8_t>(s1);
        }
      }
    } else if (stores) {
      store8(reinterpret_cast<T*>(row) + o0, a);
      store8(reinterpret_cast<T*>(row) + o1, b);
    }
  }
}

// Any head dimension, alignment and rot: one warp per row, lanes over pairs
// and then over the elements behind rot, element by element.
template <typename T, bool NORM, bool PAGED>
__global__ void __launch_bounds__(kThreads) rows_any_kernel(const __grid_constant__ RowsParams p, int layout) {
  pdl_wait();
  pdl_launch_dependents();
  const int token = static_cast<int>(blockIdx.x) * (kThreads / 32) + (static_cast<int>(threadIdx.x) >> 5);
  const int lane = static_cast<int>(threadIdx.x) & 31;
  int which = 0;
  while (which < 2 && static_cast<int>(blockIdx.y) >= p.group_end[which]) ++which;
  const RowSet& set = p.set[which];
  const int h = static_cast<int>(blockIdx.y) - (which ? p.group_end[which - 1] : 0);
  const TokenPlace t = place_token<PAGED>(p, token, p.rot > 0);
  if (!t.owned || (set.paged && !t.valid)) return;
  const T* src = static_cast<const T*>(set.src) + t.b * set.sb + t.s * set.ss + h * set.sh;
  T* dst = static_cast<T*>(set.dst) +
           (set.paged ? t.page * set.db + t.slot * set.ds : t.b * set.db + t.s * set.ds) + h * set.dh;
  if (!t.valid) {
    for (int d = lane; d < p.dim; d += 32) dst[d] = Io<T>::from_f(0.f);
    return;
  }
  float r = 1.f;
  const T* w = static_cast<const T*>(set.weight);
  if constexpr (NORM) {
    float ss = 0.f;
    for (int d = lane; d < p.dim; d += 32) {
      const float x = Io<T>::to_f(src[d]);
      ss = fmaf(x, x, ss);
    }
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) ss += __shfl_xor_sync(0xffffffffu, ss, o);
    r = rsqrtf(ss / static_cast<float>(p.dim) + p.eps);
  }
  auto value = [&](int d) {
    float x = Io<T>::to_f(src[d]);
    if constexpr (NORM) x = x * r * (w != nullptr ? Io<T>::to_f(w[d]) : 1.f);
    return x;
  };
  const int rot = set.rotate ? p.rot : 0;
  for (int i = lane; i < rot / 2; i += 32) {
    const int d0 = layout == LUNARAD_ROTARY_HALF ? i : 2 * i;
    const int d1 = layout == LUNARAD_ROTARY_HALF ? rot / 2 + i : 2 * i + 1;
    float a = value(d0), b = value(d1);
    const float* cs = p.table + (t.pos * (p.rot / 2) + i) * 2;
    turn(a, b, cs[0], p.inverse ? -cs[1] : cs[1]);
    dst[d0] = Io<T>::from_f(a);
    dst[d1] = Io<T>::from_f(b);
  }
  for (int d = rot + lane; d < p.dim; d += 32) dst[d] = Io<T>::from_f(value(d));
}

// ------------------------------------------------- append to a 4-bit cache --
// Any rot and alignment: a thread makes the 16 elements of one scale block of a
// cached row (fetching their partners too), element by element.
template <typename T>
__global__ void __launch_bounds__(kThreads) append_e2m1_any_kernel(const __grid_constant__ QuantParams q, int layout) {
  pdl_wait();
  pdl_launch_dependents();
  const RowsParams& p = q.r;
  const int lanes = 1 << p.lanes_log2;
  const int token = static_cast<int>(blockIdx.x) * (kThreads >> p.lanes_log2) + (static_cast<int>(threadIdx.x) >> p.lanes_log2);
  const int u = static_cast<int>(threadIdx.x) & (lanes - 1);
  int which = 0;
  while (which < 2 && static_cast<int>(blockIdx.y) >= p.group_end[which]) ++which;
  const RowSet& set = p.set[which];
  const int h = static_cast<int>(blockIdx.y) - (which ? p.group_end[which - 1] : 0);
  const TokenPlace t = place_token<true>(p, token, p.rot > 0);
  if (!t.owned || u >= q.blocks || !t.valid) return;
  const T* src = static_cast<const T*>(set.src) + t.s * set.ss + h * set.sh;
  const int d0 = 16 * u;
  float y[16];
  const int rot = set.rotate ? p.rot : 0;
  const float* row = p.table + t.pos * p.rot;
#pragma unroll
  for (int i = 0; i < 16; ++i) {
    const int d = d0 + i;
    float x = Io<T>::to_f(src[d]);
    if (d < rot) {
      const bool first = layout == LUNARAD_ROTARY_HALF ? d < rot / 2 : (d & 1) == 0;
      const int other = layout == LUNARAD_ROTARY_HALF ? (first ? d + rot / 2 : d - rot / 2) : (d ^ 1);
      const int pair = layout == LUNARAD_ROTARY_HALF ? (first ? d : d - rot / 2) : d >> 1;
      const float z = Io<T>::to_f(src[other]);
      float a = first ? x : z, b = first ? z : x;
      turn(a, b, row[2 * pair], row[2 * pair + 1]);
      x = first ? a : b;
    }
    y[i] = x;
  }
  float amax = 0.f;
#pragma unroll
  for (int i = 0; i < 16; ++i) {
    y[i] = __fmul_rn(y[i], q.inv_gain[which]);
    amax = fmax_nan(amax, fabsf(y[i]));
  }
  uint32_t sb;
  const uint32_t w0 = quantise(y, 0, amax, sb), w1 = quantise(y, 8, amax, sb);
  uint8_t* dst = static_cast<uint8_t*>(set.dst) + t.page * set.db + h * set.dh + t.slot * set.ds + 8 * u;
  *reinterpret_cast<uint2*>(dst) = make_uint2(w0, w1);
  static_cast<uint8_t*>(q.scales[which])[t.page * q.sc_page[which] + h * q.sc_head[which] +
                                         static_cast<int64_t>(t.slot) * q.blocks + u] = static_cast<uint8_t>(sb);
}

// --------------------------------------------------------------- read back --
struct ReadParams {
  Seqs seqs;
  const void* src[2];
  const void* scales[2];
  int64_t page_stride[2], head_stride[2], sc_page[2], sc_head[2];
  float gain[2];
  void* dst[2];
  int heads, dim, units, lanes_log2, num_pages, tokens, zero_rest;
  unsigned int* err;
};

// blockIdx.y = group of HEADS heads, blockIdx.z = 0 keys / 1 values; a lane
// moves 8 neighbouring elements of each head, so that both the codes and the
// rows are accessed without gaps, and all heads' loads are in flight at once.
template <typename T, bool E2M1, int HEADS>
__global__ void __launch_bounds__(kThreads) read_kernel(const __grid_constant__ ReadParams p) {
  pdl_wait();
  pdl_launch_dependents();
  const int lanes = 1 << p.lanes_log2;
  const int token = static_cast<int>(blockIdx.x) * (kThreads >> p.lanes_log2) + (static_cast<int>(threadIdx.x) >> p.lanes_log2);
  if (token >= p.tokens) return;
  const int h0 = static_cast<int>(blockIdx.y) * HEADS, kv = static_cast<int>(blockIdx.z), nh = min(HEADS, p.heads - h0);
  int seq, slot = 0, page = -1;
  int64_t pos;
  if (!find_token(p.seqs, token, seq, pos)) {
    if (!p.zero_rest) return;
    pos = -1;
  }
  if (pos >= 0) page = find_page(p.seqs, seq, pos, p.num_pages, slot, p.err);
  T* dst = static_cast<T*>(p.dst[kv]) + (static_cast<int64_t>(token) * p.heads + h0) * p.dim;
  const int64_t at = page * p.page_stride[kv] + h0 * p.head_stride[kv];
  for (int u = static_cast<int>(threadIdx.x) & (lanes - 1); u < p.units; u += lanes) {
    if constexpr (E2M1) {
      uint32_t w[HEADS], s[HEADS];
#pragma unroll
      for (int h = 0; h < HEADS; ++h) {
        w[h] = s[h] = 0u;
        if (page >= 0 && h < nh) {
          w[h] = __ldg(reinterpret_cast<const uint32_t*>(static_cast<const uint8_t*>(p.src[kv]) + at + h * p.head_stride[kv] +
                                                         static_cast<int64_t>(slot) * (p.dim / 2)) + u);
          s[h] = __ldg(static_cast<const uint8_t*>(p.scales[kv]) + page * p.sc_page[kv] + (h0 + h) * p.sc_head[kv] +
                       static_cast<int64_t>(slot) * (p.dim / 16) + (u >> 1));
        }
      }
#pragma unroll
      for (int h = 0; h < HEADS; ++h)
        if (h < nh) {
          const float scale = __fmul_rn(e4m3_to_float(s[h]), p.gain[kv]);
          float x[8];
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            const float2 v = __half22float2(e2m1x2_to_half2((w[h] >> (8 * i)) & 0xFFu));
            x[2 * i] = __fmul_rn(v.x, scale);
            x[2 * i + 1] = __fmul_rn(v.y, scale);
          }
          store8(dst + h * p.dim + 8 * u, x);
        }
    } else {
      float x[HEADS][8];
#pragma unroll
      for (int h = 0; h < HEADS; ++h) {
#pragma unroll
        for (int i = 0; i < 8; ++i) x[h][i] = 0.f;
        if (page >= 0 && h < nh)
          load8(static_cast<const T*>(p.src[kv]) + at + h * p.head_stride[kv] + static_cast<int64_t>(slot) * p.dim + 8 * u, x[h]);
      }
#pragma unroll
      for (int h = 0; h < HEADS; ++h)
        if (h < nh) store8(dst + h * p.dim + 8 * u, x[h]);
    }
  }
}

// Any head dimension and alignment, element by element (4 bits: by scale blocks).
template <typename T, bool E2M1>
__global__ void __launch_bounds__(kThreads) read_any_kernel(const __grid_constant__ ReadParams p) {
  pdl_wait();
  pdl_launch_dependents();
  const int token = static_cast<int>(blockIdx.x) * (kThreads / 32) + (static_cast<int>(threadIdx.x) >> 5);
  if (token >= p.tokens) return;
  const int h = static_cast<int>(blockIdx.y), kv = static_cast<int>(blockIdx.z);
  int seq, slot = 0, page = -1;
  int64_t pos;
  if (!find_token(p.seqs, token, seq, pos)) {
    if (!p.zero_rest) return;
    pos = -1;
  }
  if (pos >= 0) page = find_page(p.seqs, seq, pos, p.num_pages, slot, p.err);
  T* dst = static_cast<T*>(p.dst[kv]) + (static_cast<int64_t>(token) * p.heads + h) * p.dim;
  const int64_t at = page * p.page_stride[kv] + h * p.head_stride[kv];
  for (int d = static_cast<int>(threadIdx.x) & 31; d < p.dim; d += 32) {
    T x = Io<T>::from_f(0.f);
    if (page >= 0) {
      if constexpr (E2M1) {
        const uint8_t byte = static_cast<const uint8_t*>(p.src[kv])[at + static_cast<int64_t>(slot) * (p.dim / 2) + (d >> 1)];
        const uint8_t sb = static_cast<const uint8_t*>(p.scales[kv])[page * p.sc_page[kv] + h * p.sc_head[kv] +
                                                                     static_cast<int64_t>(slot) * (p.dim / 16) + (d >> 4)];
        const float2 v = __half22float2(e2m1x2_to_half2(byte));
        x = Io<T>::from_f(__fmul_rn(d & 1 ? v.y : v.x, __fmul_rn(e4m3_to_float(sb), p.gain[kv])));
      } else {
        x = static_cast<const T*>(p.src[kv])[at + static_cast<int64_t>(slot) * p.dim + d];
      }
    }
    dst[d] = x;
  }
}

// ------------------------------------------------------------------- host --
bool al16(const void* p) { return (reinterpret_cast<uintptr_t>(p) & 15u) == 0; }

int log2_ceil(int n) {
  int l = 0;
  while ((1 << l) < n) ++l;
  return l;
}

// Whether the 16-byte row kernel takes the sets: whole units (into a 4-bit cache
// pairs of them), 16-byte aligned rows.
bool rows_vector_ok(const RowsParams& p, int n_sets, int elem, bool quant) {
  const int whole = quant ? 32 : 16;
  if (p.dim % whole != 0 || p.rot % whole != 0 || p.dim > 512) return false;
  if (p.rot > 0 && !al16(p.table)) return false;
  const int64_t vec = 16 / elem;
  for (int i = 0; i < n_sets; ++i) {
    const RowSet& s = p.set[i];
    if (!al16(s.src) || !al16(s.weight)) return false;
    for (int64_t v : {s.sb, s.sh, s.ss})
      if (v % vec != 0) return false;
    if (quant && s.paged) continue;   // words of codes: the library's entry has checked their alignment
    if (!al16(s.dst)) return false;
    for (int64_t v : {s.db, s.dh, s.ds})
      if (v % vec != 0) return false;
  }
  return true;
}

void set_groups(RowsParams& p, int n_sets, int per) {
  int end = 0;
  for (int i = 0; i < 3; ++i) {
    if (i < n_sets) end += (p.set[i].heads + per - 1) / per;
    p.group_end[i] = end;
  }
}

// Heads per lane, measured on B200: rotating 4111 x 24 rows of 128 bf16 took
// 13.9 us with 1, 12.0 with 2, 16.9 with 4 (registers leave too few warps);
// reading 88720 tokens of a 4-bit cache, 8 heads of 128, 116 us with 2, 90 with 4, 82 with 8.
constexpr int kHeads = 2, kReadHeads = 8;

template <typename T, bool NORM, bool PAGED, bool QUANT, int HEADS>
cudaError_t run_rows_vector(const QuantParams& q, int layout, dim3 grid, cudaStream_t s) {
  return layout == LUNARAD_ROTARY_HALF
             ? launch_pdl(rows_kernel<T, LUNARAD_ROTARY_HALF, NORM, PAGED, QUANT, HEADS>, grid, dim3(kThreads), 0, s, q)
             : launch_pdl(rows_kernel<T, LUNARAD_ROTARY_INTERLEAVED, NORM, PAGED, QUANT, HEADS>, grid, dim3(kThreads), 0, s, q);
}

template <typename T, bool NORM, bool PAGED, bool QUANT>
cudaError_t run_rows(QuantParams q, int n_sets, int layout, cudaStream_t s) {
  RowsParams& p = q.r;
  p.err = device_error_word();
  if (p.err == nullptr) return cudaErrorInvalidDevice;
  const bool vector = rows_vector_ok(p, n_sets, sizeof(T), QUANT);
  if (!vector) {
    if constexpr (QUANT) {
      // The cached rows block by block, the query rows (which may be rotated in
      // place) pair by pair.
      set_groups(p, 2, 1);
      q.blocks = p.dim / 16;
      p.lanes_log2 = log2_ceil(q.blocks);
      const dim3 blocks(static_cast<unsigned>(ceil_div64(p.tokens, kThreads >> p.lanes_log2)), p.group_end[2]);
      const cudaError_t e = launch_pdl(append_e2m1_any_kernel<T>, blocks, dim3(kThreads), 0, s, q, layout);
      if (e != cudaSuccess || n_sets < 3) return e;
      QuantParams rest = q;
      rest.r.set[0] = q.r.set[2];
      return run_rows<T, NORM, PAGED, false>(rest, 1, layout, s);
    } else {
      set_groups(p, n_sets, 1);
      const dim3 grid(static_cast<unsigned>(ceil_div64(p.tokens, kThreads / 32)), p.group_end[2]);
      return launch_pdl(rows_any_kernel<T, NORM, PAGED>, grid, dim3(kThreads), 0, s, p, layout);
    }
  }
  p.units = p.dim / 16;
  q.blocks = p.dim / 16;
  p.lanes_log2 = log2_ceil(p.units);
  const int per_block = kThreads >> p.lanes_log2;
  const unsigned gx = static_cast<unsigned>(ceil_div64(p.tokens, per_block));
  // One head per lane while all blocks fit the SMs at once (latency counts: reading
  // 1006 tokens of 12 heads took 8 us instead of 12); several beyond, see kHeads.
  set_groups(p, n_sets, 1);
  const bool few = static_cast<int64_t>(gx) * p.group_end[2] <= int64_t{device_num_sms()} * 16;
  if (!few) set_groups(p, n_sets, kHeads);
  const dim3 grid(gx, p.group_end[2]);
  return few ? run_rows_vector<T, NORM, PAGED, QUANT, 1>(q, layout, grid, s)
             : run_rows_vector<T, NORM, PAGED, QUANT, kHeads>(q, layout, grid, s);
}

template <bool NORM, bool PAGED, bool QUANT>
cudaError_t run_rows_dtype(const QuantParams& q, int n_sets, int layout, int64_t dtype, cudaStream_t s) {
  if (dtype == LUNARA_F16) return run_rows<__half, NORM, PAGED, QUANT>(q, n_sets, layout, s);
  if (dtype == LUNARA_BF16) return run_rows<__nv_bfloat16, NORM, PAGED, QUANT>(q, n_sets, layout, s);
  return run_rows<float, NORM, PAGED, QUANT>(q, n_sets, layout, s);
}

void set_rotary(RowsParams& p, const lunarad_rotary_table& r) {
  p.table = r.table;
  p.table_positions = r.positions;
  p.rot = static_cast<int>(r.rot);
}

RowSet view_set(const lunarad_view& in, const lunarad_view& out, const void* weight, int64_t heads) {
  RowSet s{};
  s.src = in.data;
  s.sb = in.batch_stride;
  s.sh = in.head_stride;
  s.ss = in.seq_stride;
  s.dst = const_cast<void*>(out.data);
  s.db = out.batch_stride;
  s.dh = out.head_stride;
  s.ds = out.seq_stride;
  s.weight = weight;
  s.heads = static_cast<int>(heads);
  s.rotate = 1;
  return s;
}

template <typename T, bool E2M1>
cudaError_t run_read(ReadParams p, cudaStream_t s) {
  p.err = device_error_word();
  if (p.err == nullptr) return cudaErrorInvalidDevice;
  const int64_t e = 16 / sizeof(T);
  bool vec = p.dim % 16 == 0;
  for (int i = 0; i < 2; ++i) {
    vec = vec && al16(p.dst[i]);
    if (!E2M1) vec = vec && al16(p.src[i]) && p.page_stride[i] % e == 0 && p.head_stride[i] % e == 0;
  }
  if (!vec) {
    const dim3 grid(static_cast<unsigned>(ceil_div64(p.tokens, kThreads / 32)), p.heads, 2);
    return launch_pdl(read_any_kernel<T, E2M1>, grid, dim3(kThreads), 0, s, p);
  }
  p.units = p.dim / 8;
  p.lanes_log2 = log2_ceil(p.units);
  if (p.lanes_log2 > 5) p.lanes_log2 = 5;
  const unsigned gx = static_cast<unsigned>(ceil_div64(p.tokens, kThreads >> p.lanes_log2));
  if (static_cast<int64_t>(gx) * p.heads * 2 <= int64_t{device_num_sms()} * 16)
    return launch_pdl(read_kernel<T, E2M1, 1>, dim3(gx, p.heads, 2), dim3(kThreads), 0, s, p);
  return launch_pdl(read_kernel<T, E2M1, kReadHeads>, dim3(gx, (p.heads + kReadHeads - 1) / kReadHeads, 2), dim3(kThreads), 0, s, p);
}

template <typename T>
cudaError_t run_read_kind(const ReadParams& p, bool e2m1, cudaStream_t s) {
  return e2m1 ? run_read<T, true>(p, s) : run_read<T, false>(p, s);
}

}  // namespace

cudaError_t launch_rotary(const lunarad_rotary_args& a, cudaStream_t stream) {
  QuantParams q{};
  RowsParams& p = q.r;
  p.set[0] = view_set(a.x, a.y, nullptr, a.heads);
  p.positions = a.positions;
  p.position_bytes = static_cast<int>(a.position_bytes);
  p.position_batch_stride = a.position_batch_stride;
  set_rotary(p, a.rotary);
  p.dim = static_cast<int>(a.dim);
  p.tokens = static_cast<int>(a.batch * a.seq);
  p.seq = static_cast<int>(a.seq);
  p.inverse = a.inverse != 0;
  return run_rows_dtype<false, false, false>(q, 1, static_cast<int>(a.rotary.layout), a.dtype, stream);
}

cudaError_t launch_qk_norm_rotary(const lunarad_qk_norm_rotary_args& a, cudaStream_t stream) {
  QuantParams q{};
  RowsParams& p = q.r;
  p.set[0] = view_set(a.q, a.q_out, a.q_weight, a.q_heads);
  p.set[1] = view_set(a.k, a.k_out, a.k_weight, a.k_heads);
  p.positions = a.positions;
  p.position_bytes = static_cast<int>(a.position_bytes);
  p.position_batch_stride = a.position_batch_stride;
  set_rotary(p, a.rotary);
  p.dim = static_cast<int>(a.dim);
  p.tokens = static_cast<int>(a.batch * a.seq);
  p.seq = static_cast<int>(a.seq);
  p.eps = static_cast<float>(a.eps);
  return run_rows_dtype<true, false, false>(q, 2, static_cast<int>(a.rotary.layout), a.dtype, stream);
}

cudaError_t launch_kv_append(const lunarad_kv_append_args& a, bool zero_rest, cudaStream_t stream) {
  const lunarad_cache& c = *a.cache;
  const bool e2m1 = c.kind == LUNARAD_KIND_E2M1;
  QuantParams q{};
  RowsParams& p = q.r;
  const lunarad_view none{};
  int n = 0;
  auto cache_set = [&](const lunarad_view& in, void* pages, int64_t ps, int64_t hs, void* scales, int64_t sps,
                       int64_t shs, double gain, bool rotate) {
    RowSet s = view_set(in, none, nullptr, c.kv_heads);
    s.sb = 0;
    s.dst = pages;
    s.db = ps;
    s.dh = hs;
    s.ds = e2m1 ? c.dim / 2 : c.dim;
    s.rotate = rotate && a.rotary.rot > 0;
    s.paged = 1;
    q.scales[n] = scales;
    q.sc_page[n] = sps;
    q.sc_head[n] = shs;
    q.inv_gain[n] = 1.0f / static_cast<float>(gain);
    p.set[n++] = s;
  };
  cache_set(a.k, c.k, c.k_page_stride, c.k_head_stride, c.k_scales, c.ks_page_stride, c.ks_head_stride, c.k_gain, true);
  cache_set(a.v, c.v, c.v_page_stride, c.v_head_stride, c.v_scales, c.vs_page_stride, c.vs_head_stride, c.v_gain, false);
  if (a.q_heads > 0) {
    RowSet s = view_set(a.q, a.q_out, nullptr, a.q_heads);
    s.sb = s.db = 0;
    p.set[n++] = s;
  }
  p.seqs = make_seqs(a.seqs, c.page_size);
  p.num_pages = static_cast<int>(c.num_pages);
  set_rotary(p, a.rotary);
  p.dim = static_cast<int>(c.dim);
  p.tokens = static_cast<int>(a.seqs.tokens);
  p.seq = p.tokens;
  p.zero_rest = zero_rest;
  const int layout = static_cast<int>(a.rotary.layout);
  return e2m1 ? run_rows_dtype<false, true, true>(q, n, layout, a.dtype, stream)
              : run_rows_dtype<false, true, false>(q, n, layout, a.dtype, stream);
}

cudaError_t launch_kv_read(const lunarad_kv_read_args& a, bool zero_rest, cudaStream_t stream) {
  const lunarad_cache& c = *a.cache;
  ReadParams p{};
  p.seqs = make_seqs(a.seqs, c.page_size);
  p.src[0] = c.k;
  p.src[1] = c.v;
  p.scales[0] = c.k_scales;
  p.scales[1] = c.v_scales;
  p.page_stride[0] = c.k_page_stride;
  p.page_stride[1] = c.v_page_stride;
  p.head_stride[0] = c.k_head_stride;
  p.head_stride[1] = c.v_head_stride;
  p.sc_page[0] = c.ks_page_stride;
  p.sc_page[1] = c.vs_page_stride;
  p.sc_head[0] = c.ks_head_stride;
  p.sc_head[1] = c.vs_head_stride;
  p.gain[0] = static_cast<float>(c.k_gain);
  p.gain[1] = static_cast<float>(c.v_gain);
  p.dst[0] = a.k_out;
  p.dst[1] = a.v_out;
  p.heads = static_cast<int>(c.kv_heads);
  p.dim = static_cast<int>(c.dim);
  p.num_pages = static_cast<int>(c.num_pages);
  p.tokens = static_cast<int>(a.seqs.tokens);
  p.zero_rest = zero_rest;
  const bool e2m1 = c.kind == LUNARAD_KIND_E2M1;
  if (a.dtype == LUNARA_F16) return run_read_kind<__half>(p, e2m1, stream);
  if (a.dtype == LUNARA_BF16) return run_read_kind<__nv_bfloat16>(p, e2m1, stream);
  return run_read_kind<float>(p, e2m1, stream);
}

}  // namespace lunara
