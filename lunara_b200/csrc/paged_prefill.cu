// Attention over the paged cache for many query rows per sequence (prompts and
// chunks of prompts), on tcgen05.
//
// The query rows of a sequence and key head (its tokens times the query heads
// of the group) make items of 256 rows: two tiles of 128 that share every key
// block. Bound by the tensor and exponential pipes: 4 * 256 * 128 * D
// operations per 128-key block against 2 * 128 * D cached elements read.
//   * Equal runs: the key blocks of all items, in the order (sequence, key head,
//     row tile, block), are dealt to the persistent CTAs in equal contiguous
//     runs, so neither ragged lengths nor causal triangles nor few items leave
//     SMs idle. How many blocks precede a row tile is a sum of floors of a
//     linear function, taken in closed form. Items that a run cuts leave
//     partial O, maximum and sum in the workspace, and a second kernel joins
//     them.
//   * warps 0-3, 4-7   softmax of tile 0 and 1 (thread = row)
//     warps 8, 9       tcgen05.mma issuers of tile 0 and 1
//                        S_w = Q_w K^T  (128 x 128 x D, operands in shared memory)
//                        O_w += P_w V   (128 x D x 128, P_w from TMEM)
//     warps 12-15      copy Q, K and V with cp.async, any page size, into
//                        128-byte-swizzled tiles; rows that no query of the item
//                        sees, and rows of bad pages, become zeros there
//   * TMEM: S_w 128 columns each, O_w D columns each; P_w (16-bit pairs) takes
//     the first half of S_w's columns once the row is in registers. The next
//     S_w is issued when P_w V has completed; meanwhile the other tile's
//     products run.
#include <type_traits>

#include "kernels.h"
#include "paged_attention.cuh"

namespace lunara {
namespace {

constexpr int kItemRows = 256;
constexpr int kTileRows = 128;
constexpr int kBlock = 128;              // keys per block
constexpr int kThreads = 512;
constexpr int kMaxBatch = 1024;          // sequences per launch
constexpr float kRescaleLog2 = 8.0f;
// setmaxnreg split of the launch's 512 x 128 registers.
constexpr int kLaunchRegs = 128;
constexpr int kSoftmaxRegs = 200, kIssueRegs = 40, kCopyRegs = 72;
static_assert(256 * kSoftmaxRegs + 128 * kIssueRegs + 128 * kCopyRegs <= kThreads * kLaunchRegs, "register split");
constexpr int kPolyPairs = 4;            // of 16 exponential pairs on the FMA pipe, as in attention.cu
constexpr int kMaskRing = 16;            // blocks whose key masks are kept; more than the ring can run ahead

template <int D>
struct Layout {
  static constexpr int kHalves = D / 64;                       // 64-element column blocks of a tile
  static constexpr uint32_t kHalfBytes = kBlock * 128;         // 128 rows of 128 bytes
  static constexpr uint32_t kSlotBytes = kHalves * kHalfBytes; // one K or V block
  static constexpr uint32_t kQBytes = 2 * kSlotBytes;          // two row tiles
  static constexpr int kSlots = D == 128 ? 5 : 8;              // ring of K and V blocks: K0, V0, K1, V1, ...
  static constexpr int kLag = 2;                               // slots whose copies stay in flight
  static constexpr uint32_t kSmem = kQBytes + kSlots * kSlotBytes + kMaskRing * 16 + 512 + 1024;
  static constexpr uint32_t kTmemS = 0, kTmemO = 256, kTmemCols = 512;
};

// Sum over i < n of floor((a i + b) / m), a, b >= 0 (the Euclid-like recursion
// of Graham, Knuth and Patashnik, Concrete Mathematics, 3.5).
__device__ int64_t floor_sum(int64_t n, int64_t m, int64_t a, int64_t b) {
  int64_t sum = 0;
  while (n > 0) {
    if (a >= m) {
      sum += n * (n - 1) / 2 * (a / m);
      a %= m;
    }
    if (b >= m) {
      sum += n * (b / m);
      b %= m;
    }
    const int64_t top = a * n + b;
    if (top < m) break;
    n = top / m;
    b = top % m;
    const int64_t x = m;
    m = a;
    a = x;
  }
  return sum;
}

// Key blocks of the items of one sequence: those of row tile r are
// [block_lo(r), block_hi(r)), a superset of what its rows see.
struct Plan {
  int row_tiles;
  int64_t pos0;   // of the first token, cut to [0, positions of the page table]
  int64_t rows;
  int G, W;       // group; window, 0 where it cuts nothing or the sequence begins with padding
  __device__ __forceinline__ int64_t hi_num(int64_t r) const { return kItemRows * r + kItemRows - 1 + G * (pos0 + kBlock); }
  __device__ __forceinline__ int64_t lo_num(int64_t r) const { return kItemRows * r + G * (pos0 + 1 - W); }
  __device__ __forceinline__ int block_hi(int r) const {
    const int64_t last = min(static_cast<int64_t>(kItemRows) * (r + 1), rows) - 1;
    return static_cast<int>((pos0 + last / G) / kBlock) + 1;
  }
  __device__ __forceinline__ int block_lo(int r) const {
    if (W == 0) return 0;
    const int64_t x = pos0 + static_cast<int64_t>(kItemRows) * r / G + 1 - W;
    return x > 0 ? static_cast<int>(x / kBlock) : 0;
  }
  __device__ __forceinline__ int blocks(int r) const { return block_hi(r) - block_lo(r); }
  // Blocks of the row tiles before r.
  __device__ __forceinline__ int64_t before(int r) const {
    int64_t tail = 0;
    if (r == row_tiles && r > 0) {   // the last tile may be short
      --r;
      tail = blocks(r);
    }
    int64_t x = floor_sum(r, static_cast<int64_t>(kBlock) * G, kItemRows, hi_num(0));
    if (W > 0) {
      const int64_t first = lo_num(0) >= 0 ? 0 : (-lo_num(0) + kItemRows - 1) / kItemRows;   // tiles before it start at block 0
      if (r > first) x -= floor_sum(r - first, static_cast<int64_t>(kBlock) * G, kItemRows, lo_num(first));
    }
    return x + tail;
  }
};

__device__ __forceinline__ Plan make_plan(const PagedParams& p, const SeqInfo& s) {
  Plan x;
  x.rows = static_cast<int64_t>(s.n) * p.group;
  x.row_tiles = x.rows < p.min_rows || x.rows >= p.max_rows || s.hi <= s.lo ? 0 : static_cast<int>((x.rows + kItemRows - 1) / kItemRows);
  x.pos0 = min(max(s.pos0, int64_t{0}), static_cast<int64_t>(p.seqs.max_pages) * p.page_size);
  x.G = p.group;
  x.W = s.pos0 < 0 ? 0 : p.window;
  return x;
}

// prefix[b] = blocks of the sequences before b, by the whole CTA.
__device__ __forceinline__ void prefix_blocks(const PagedParams& p, int64_t* prefix, int64_t* warp_sums) {
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, warps = blockDim.x >> 5;
  int64_t carry = 0;
  for (int b0 = 0; b0 < p.seqs.batch; b0 += blockDim.x) {
    const int b = b0 + static_cast<int>(threadIdx.x);
    int64_t inc = 0;
    if (b < p.seqs.batch) {
      const Plan x = make_plan(p, load_seq(p, b));
      inc = p.kv_heads * x.before(x.row_tiles);
    }
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const int64_t y = __shfl_up_sync(0xffffffffu, inc, o);
      if (lane >= o) inc += y;
    }
    if (lane == 31) warp_sums[warp] = inc;
    __syncthreads();
    int64_t before = carry, all = 0;
    for (int w = 0; w < warps; ++w) {
      if (w < warp) before += warp_sums[w];
      all += warp_sums[w];
    }
    if (b < p.seqs.batch) prefix[b + 1] = before + inc;
    carry += all;
    __syncthreads();
  }
  if (threadIdx.x == 0) prefix[0] = 0;
  __syncthreads();
}

// Worker w takes the blocks [run_start(w), run_start(w + 1)); run_of(t) takes block t.
__device__ __forceinline__ int64_t run_start(int64_t total, int workers, int w) { return total * w / workers; }
__device__ __forceinline__ int run_of(int64_t total, int workers, int64_t t) {
  return static_cast<int>(((t + 1) * workers + total - 1) / total) - 1;
}

// An item, or the part of it that a run holds.
struct Item {
  int b, kh, rt;
  int item_blocks;   // of the whole item
  int first;         // first block of the part within the item
  int n;             // blocks of the part
  int block0;        // the part's first key block
  SeqInfo s;
};

// Walks the items of the run [t, end).
struct Cursor {
  Plan plan;
  Item x;

  __device__ void load(const PagedParams& p, int b) {
    x.b = b;
    x.s = load_seq(p, b);
    plan = make_plan(p, x.s);
  }
  // The item that holds block t.
  __device__ void seek(const PagedParams& p, const int64_t* prefix, int64_t t) {
    int b = 0;
    for (int e = p.seqs.batch; b + 1 < e;) {   // last b with prefix[b] <= t
      const int mid = (b + e) >> 1;
      if (prefix[mid] <= t) b = mid; else e = mid;
    }
    load(p, b);
    const int64_t in_seq = t - prefix[b];
    const int64_t per_head = plan.before(plan.row_tiles);
    x.kh = static_cast<int>(in_seq / per_head);
    const int64_t in_head = in_seq - x.kh * per_head;
    int r = 0;
    for (int e = plan.row_tiles; r + 1 < e;) {
      const int mid = (r + e) >> 1;
      if (plan.before(mid) <= in_head) r = mid; else e = mid;
    }
    x.rt = r;
    x.item_blocks = plan.blocks(r);
    x.first = static_cast<int>(in_head - plan.before(r));
  }
  __device__ __forceinline__ void clip(int64_t left) {
    x.n = static_cast<int>(min(static_cast<int64_t>(x.item_blocks - x.first), left));
    x.block0 = plan.block_lo(x.rt) + x.first;
  }
  // To the next item (there is one).
  __device__ void next(const PagedParams& p) {
    if (++x.rt == plan.row_tiles) {
      x.rt = 0;
      if (++x.kh == p.kv_heads) {
        x.kh = 0;
        do load(p, x.b + 1); while (plan.row_tiles == 0);
      }
    }
    x.item_blocks = plan.blocks(x.rt);
    x.first = 0;
  }
};

__device__ __forceinline__ void copy16(uint32_t dst, const void* src, bool in) {
  asm volatile("cp.async.cg.shared.global.L2::128B [%0], [%1], 16, %2;" ::"r"(dst), "l"(src), "r"(in ? 16 : 0) : "memory");
}

// Keys that some row of a tile pair sees.
__device__ __forceinline__ void item_keys(const PagedParams& p, const Item& x, int& lo, int& hi) {
  const int64_t rows = static_cast<int64_t>(x.s.n) * p.group;
  const int64_t r0 = static_cast<int64_t>(x.rt) * kItemRows, r1 = min(r0 + kItemRows, rows) - 1;
  int a, b;
  visible(p, x.s.pos0 + r0 / p.group, lo, a);
  visible(p, x.s.pos0 + r1 / p.group, b, hi);
}

template <typename T, int D>
__global__ void __launch_bounds__(kThreads, 1) paged_prefill_kernel(const __grid_constant__ PagedParams p) {
  using L = Layout<D>;
  constexpr bool kBF16 = std::is_same<T, __nv_bfloat16>::value;
  constexpr uint32_t IDESC_S = idesc_f16(128, kBlock, kBF16, false, false);
  constexpr uint32_t IDESC_PV = idesc_f16(128, D, kBF16, false, true);

  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t{1023});
  uint8_t* sQ = smem;
  uint8_t* sRing = sQ + L::kQBytes;
  uint32_t* s_mask = reinterpret_cast<uint32_t*>(sRing + L::kSlots * L::kSlotBytes);   // [kMaskRing][4]
  uint64_t* bars = reinterpret_cast<uint64_t*>(s_mask + kMaskRing * 4);
  uint64_t* q_full = bars;
  uint64_t* q_free = q_full + 1;            // both issuers done with Q
  uint64_t* full = q_free + 1;              // [kSlots]
  uint64_t* empty = full + L::kSlots;       // [kSlots] both issuers done with the slot
  uint64_t* s_full = empty + L::kSlots;     // [2]
  uint64_t* p_ready = s_full + 2;           // [2]
  uint64_t* o_full = p_ready + 2;           // [2]
  uint64_t* o_free = o_full + 2;            // [2] the item's O_w is read
  uint64_t* drain_bar = o_free + 2;         // [2]
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(drain_bar + 2);
  volatile int* abort_flag = reinterpret_cast<volatile int*>(tmem_slot + 1);
  // The prefix sums stand in the ring until the roles begin.
  int64_t* prefix = reinterpret_cast<int64_t*>(sRing);
  __shared__ int64_t warp_sums[kThreads / 32];
  __shared__ Cursor s_cursor;

  const int warp = threadIdx.x >> 5;
  const int lane = threadIdx.x & 31;
  if (threadIdx.x == 0) {
    mbar_init(q_full, 128);
    mbar_init(q_free, 2);
    for (int i = 0; i < L::kSlots; ++i) {
      mbar_init(&full[i], 128);
      mbar_init(&empty[i], 2);
    }
    for (int w = 0; w < 2; ++w) {
      mbar_init(&s_full[w], 1);
      mbar_init(&p_ready[w], kTileRows);
      mbar_init(&o_full[w], 1);
      mbar_init(&o_free[w], kTileRows);
      mbar_init(&drain_bar[w], 1);
    }
    *abort_flag = 0;
    fence_mbar_init();
  }
  if (warp == 8) {
    tmem_alloc(tmem_slot, L::kTmemCols);
    tmem_relinquish();
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem_base = *tmem_slot;
  pdl_wait();
  pdl_launch_dependents();
  prefix_blocks(p, prefix, warp_sums);
  const int64_t total = prefix[p.seqs.batch];
  const int workers = static_cast<int>(min(total, static_cast<int64_t>(p.workers)));
  const int worker = static_cast<int>(blockIdx.x);
  int64_t t_first = 0, t_end = 0;
  clear_empty<T>(p);
  if (worker >= workers) {
    if (threadIdx.x == 0) p.cuts[worker].parts = 0;
  } else {
    t_first = run_start(total, workers, worker);
    t_end = run_start(total, workers, worker + 1);
    if (threadIdx.x == 0) s_cursor.seek(p, prefix, t_first);
  }
  __syncthreads();   // the prefix sums are used up: the ring may be written

  if (warp >= 12) {
    reg_dealloc<kCopyRegs>();
    // -------------------------------------------------------------- copies --
    // A warp copies 32 rows of every block; lane l looks up the place of row
    // 32 warp + l, and D / 8 neighbouring lanes copy one row.
    const int cw = warp - 12;
    constexpr int kPer = D / 8, kRowsAtOnce = 32 / kPer;
    const int chunk = lane % kPer, sub = lane / kPer;
    const uint32_t ring = smem_u32(sRing);
    int slot = 0;
    uint32_t phase = 0;        // of empty[slot]
    int issued = 0, arrived = 0;   // slots
    auto arrive_oldest = [&] {     // its copies have landed
      fence_proxy_async_smem();
      mbar_arrive(&full[arrived % L::kSlots]);
      ++arrived;
    };
    bool ok = true;
    Cursor cur = s_cursor;
    int block_count = 0;
    uint32_t items = 0;
    for (int64_t t = t_first; ok && t < t_end; ++items) {
      cur.clip(t_end - t);
      const Item& x = cur.x;
      int lo, hi;
      item_keys(p, x, lo, hi);
      // Q: row r of the item is token r / group, head r % group of the pair.
      if (!mbar_wait_warp(q_free, (items & 1u) ^ 1u, abort_flag, p.err, kErrPagedWait)) { ok = false; break; }
      {
        const int64_t rows = static_cast<int64_t>(x.s.n) * p.group - static_cast<int64_t>(x.rt) * kItemRows;
        for (int it = 0; it < kItemRows / 4 / kRowsAtOnce; ++it) {
          const int r = (kItemRows / 4) * cw + it * kRowsAtOnce + sub;
          const bool in = r < rows;
          const int64_t row = static_cast<int64_t>(x.rt) * kItemRows + (in ? r : 0);
          const int i = static_cast<int>(row / p.group);
          const int head = x.kh * p.group + static_cast<int>(row - static_cast<int64_t>(i) * p.group);
          const T* src = static_cast<const T*>(p.q) + (x.s.first + i) * p.q_tok + head * p.q_head + 8 * chunk;
          copy16(smem_u32(sQ) + (r >> 7) * L::kSlotBytes + (chunk >> 3) * L::kHalfBytes + (r & 127) * 128 + (((chunk & 7) ^ (r & 7)) << 4),
                 src, in);
        }
      }
      asm volatile("cp.async.commit_group;" ::: "memory");
      asm volatile("cp.async.wait_group 0;" ::: "memory");
      while (arrived < issued) arrive_oldest();
      fence_proxy_async_smem();
      mbar_arrive(q_full);
      const int32_t* table = p.seqs.page_table + x.b * p.seqs.table_stride;
      const char* bases[2] = {static_cast<const char*>(p.k) + x.kh * p.k_head * 2, static_cast<const char*>(p.v) + x.kh * p.v_head * 2};
      const int row_bytes = D * 2;
      auto find = [&](int block, int& row_slot) {   // page of this lane's row, or -1
        const int key = block * kBlock + 32 * cw + lane;
        if (key < lo || key >= hi) return -1;
        const int pi = p.seqs.page_div.div(key);
        row_slot = key - pi * p.page_size;
        const int page = table[pi];
        if (page >= 0 && page < p.num_pages) return page;
        atomicCAS(p.err, 0u, static_cast<unsigned>(kErrCachePage));
        return -1;
      };
      int next_slot = 0, next_page = find(x.block0, next_slot);
      for (int j = 0; j < x.n && ok; ++j, ++block_count) {
        const int page = next_page, row_slot = next_slot;
        if (j + 1 < x.n) next_page = find(x.block0 + j + 1, next_slot);
        const uint32_t use = __ballot_sync(0xffffffffu, page >= 0);
        if (lane == 0) s_mask[(block_count % kMaskRing) * 4 + cw] = use;
#pragma unroll
        for (int kv = 0; kv < 2; ++kv) {
          if (!mbar_wait_warp(&empty[slot], phase ^ 1u, abort_flag, p.err, kErrPagedWait)) { ok = false; break; }
          const int64_t stride = (kv == 0 ? p.k_page : p.v_page) * 2;
          const uint32_t dst = ring + slot * L::kSlotBytes + (chunk >> 3) * L::kHalfBytes;
#pragma unroll 4
          for (int it = 0; it < 32 / kRowsAtOnce; ++it) {
            const int r = it * kRowsAtOnce + sub;
            const int pg = __shfl_sync(0xffffffffu, page, r), sl = __shfl_sync(0xffffffffu, row_slot, r);
            const int row = 32 * cw + r;
            const bool in = pg >= 0;
            copy16(dst + row * 128 + (((chunk & 7) ^ (row & 7)) << 4),
                   in ? bases[kv] + pg * stride + static_cast<int64_t>(sl) * row_bytes + 16 * chunk : bases[kv], in);
          }
          asm volatile("cp.async.commit_group;" ::: "memory");
          ++issued;
          if (issued - arrived > L::kLag) {
            asm volatile("cp.async.wait_group %0;" ::"n"(L::kLag) : "memory");
            arrive_oldest();
          }
          if (++slot == L::kSlots) { slot = 0; phase ^= 1u; }
        }
      }
      asm volatile("cp.async.wait_group 0;" ::: "memory");
      while (arrived < issued) arrive_oldest();
      t += x.n;
      if (t < t_end) cur.next(p);
    }
    asm volatile("cp.async.wait_group 0;" ::: "memory");
  } else if (warp == 8 || warp == 9) {
    reg_dealloc<kIssueRegs>();
    // ---------------------------------------------------------- MMA issuers --
    const int w = warp - 8;
    const bool leader = elect_one_sync();
    auto wait = [&](uint64_t* bar, uint32_t parity) {
      return mbar_wait_warp(bar, parity, abort_flag, p.err, kErrPagedWait);
    };
    const uint64_t qd = sw128_desc(smem_u32(sQ) + w * L::kSlotBytes, 16, 1024);
    const uint64_t kd0 = sw128_desc(smem_u32(sRing), 16, 1024);
    const uint64_t vd0 = sw128_desc(smem_u32(sRing), L::kHalfBytes, 1024);
    const uint32_t d_s = tmem_base + L::kTmemS + w * 128;
    const uint32_t d_o = tmem_base + L::kTmemO + w * D;
    auto issue_s = [&](int slot) {
      const uint64_t kd = kd0 + static_cast<uint64_t>(slot) * (L::kSlotBytes >> 4);
#pragma unroll
      for (int kk = 0; kk < D / 16; ++kk) {
        const uint64_t off = (kk >> 2) * (L::kHalfBytes >> 4) + 2 * (kk & 3);
        umma_f16_ss(d_s, qd + off, kd + off, IDESC_S, kk > 0 ? 1u : 0u);
      }
    };
    auto issue_pv = [&](int slot, bool first) {
      const uint64_t vd = vd0 + static_cast<uint64_t>(slot) * (L::kSlotBytes >> 4);
#pragma unroll
      for (int kk = 0; kk < kBlock / 16; ++kk)
        umma_f16_ts(d_o, d_s + kk * 8, vd + 128 * kk, IDESC_PV, (!first || kk > 0) ? 1u : 0u);
    };
    bool ok = true;
    Cursor cur = s_cursor;
    uint32_t items = 0, blocks = 0;   // items and blocks so far
    uint32_t used = 0;                // ring slots so far
    for (int64_t t = t_first; ok && t < t_end; ++items) {
      cur.clip(t_end - t);
      const int n = cur.x.n;
      if (!wait(q_full, items & 1u)) { ok = false; break; }
      for (int j = 0; j < n && ok; ++j, ++blocks) {
        const int ks = static_cast<int>(used % L::kSlots), vs = static_cast<int>((used + 1) % L::kSlots);
        const uint32_t kp = (used / L::kSlots) & 1u, vp = ((used + 1) / L::kSlots) & 1u;
        // S of block j: K is there, and P V of the block before has read P
        // (which shares S's columns).
        if (!wait(&full[ks], kp)) { ok = false; break; }
        if (j > 0 && !wait(&o_full[w], (blocks - 1) & 1u)) { ok = false; break; }
        tc_fence_after();
        if (leader) {
          issue_s(ks);
          umma_commit(&s_full[w]);
          umma_commit(&empty[ks]);
          if (j + 1 == n) umma_commit(q_free);
        }
        __syncwarp();
        if (!wait(&full[vs], vp)) { ok = false; break; }
        if (!wait(&p_ready[w], blocks & 1u)) { ok = false; break; }
        // The item's first P V overwrites O: the item before must have been read.
        if (j == 0 && items > 0 && !wait(&o_free[w], (items - 1) & 1u)) { ok = false; break; }
        tc_fence_after();
        if (leader) {
          issue_pv(vs, j == 0);
          umma_commit(&o_full[w]);
          umma_commit(&empty[vs]);
        }
        __syncwarp();
        used += 2;
      }
      // The next item's S must not overwrite P before the last P V has read it.
      if (ok && !wait(&o_full[w], (blocks - 1) & 1u)) ok = false;
      t += n;
      if (ok && t < t_end) cur.next(p);
    }
    if (!ok) {
      if (leader) umma_commit(&drain_bar[w]);
      __syncwarp();
      mbar_drain_wait(&drain_bar[w], 0, 1000000000ull);
    }
  } else if (warp >= 8) {
    reg_dealloc<kIssueRegs>();   // idle warps of the issuers' warpgroup
  } else {
    reg_alloc<kSoftmaxRegs>();
    // ------------------------------------------------------------- softmax --
    const int w = warp >> 2, quarter = warp & 3, r = quarter * 32 + lane;
    const uint32_t lane_off = static_cast<uint32_t>(quarter * 32) << 16;
    const uint32_t tS = tmem_base + lane_off + L::kTmemS + w * 128;
    const uint32_t tO = tmem_base + lane_off + L::kTmemO + w * D;
    // The maximum needs a positive factor: a negative scale turns the scores'
    // signs, a zero one becomes too small to matter.
    const float sl2 = fmaxf(fabsf(p.scale) * 1.4426950408889634f, 1e-30f);
    const bool negative = p.scale < 0.f;
    bool ok = true;
    Cursor cur = s_cursor;
    uint32_t blocks = 0;
    for (int64_t t = t_first; ok && t < t_end;) {
      cur.clip(t_end - t);
      const Item& x = cur.x;
      const int64_t rows = static_cast<int64_t>(x.s.n) * p.group;
      const int64_t row = static_cast<int64_t>(x.rt) * kItemRows + w * kTileRows + r;
      const bool real = row < rows;
      const int i = static_cast<int>((real ? row : rows - 1) / p.group);
      int lo, hi;
      visible(p, x.s.pos0 + i, lo, hi);
      const int n = x.n, block0 = x.block0;
      float m = -INFINITY, l = 0.f;
      for (int j = 0; j < n; ++j, ++blocks) {
        if (!mbar_wait_warp(&s_full[w], blocks & 1u, abort_flag, p.err, kErrPagedWait)) { ok = false; break; }
        tc_fence_after();
        uint32_t sc[4][32];
#pragma unroll
        for (int cc = 0; cc < 4; ++cc) tmem_ld_32x32b_x32(tS + cc * 32, sc[cc]);
        const uint4 keep = *reinterpret_cast<const uint4*>(&s_mask[(blocks % kMaskRing) * 4]);
        tmem_ld_wait_regs(sc[0]);
        reg_fence(sc[1]);
        reg_fence(sc[2]);
        reg_fence(sc[3]);
        const int kv0 = (block0 + j) * kBlock;
        if (negative) {
#pragma unroll
          for (int cc = 0; cc < 4; ++cc)
#pragma unroll
            for (int e = 0; e < 32; ++e) sc[cc][e] ^= 0x80000000u;
        }
        const bool masked = (keep.x & keep.y & keep.z & keep.w) != ~0u || __any_sync(0xffffffffu, kv0 < lo || kv0 + kBlock > hi);
        if (masked) {
          const uint32_t words[4] = {keep.x, keep.y, keep.z, keep.w};
#pragma unroll
          for (int cc = 0; cc < 4; ++cc) {
            // Bits of the columns that this row sees.
            const int a = lo - kv0 - 32 * cc, b = hi - kv0 - 32 * cc;
            uint32_t bits = words[cc];
            if (a > 0) bits &= a < 32 ? ~0u << a : 0u;
            if (b < 32) bits &= b > 0 ? (1u << b) - 1u : 0u;
#pragma unroll
            for (int e = 0; e < 32; ++e)
              if (((bits >> e) & 1u) == 0u) sc[cc][e] = __float_as_uint(-INFINITY);
          }
        }
        float mxp[8];
#pragma unroll
        for (int q = 0; q < 8; ++q) mxp[q] = -INFINITY;
#pragma unroll
        for (int cc = 0; cc < 4; ++cc)
#pragma unroll
          for (int e = 0; e < 32; e += 2)
            mxp[(e >> 1) & 7] = fmax3_nan(mxp[(e >> 1) & 7], __uint_as_float(sc[cc][e]), __uint_as_float(sc[cc][e + 1]));
        const float mx = fmax3_nan(fmax3_nan(mxp[0], mxp[1], mxp[2]), fmax3_nan(mxp[3], mxp[4], mxp[5]), fmax_nan(mxp[6], mxp[7]));
        const float cand = mx * sl2;
        if (j == 0) {
          m = cand;
        } else if (__any_sync(0xffffffffu, !(cand <= m + kRescaleLog2))) {
          // P V of the block before is complete (S of this block was issued after it).
          const float next = fmax_nan(m, cand);
          const float alpha = next == -INFINITY ? 1.f : ex2_approx(m - next);
          l *= alpha;
          m = next;
          const uint64_t a2 = f2_pack(alpha, alpha);
#pragma unroll
          for (int c = 0; c < D / 16; ++c) {
            uint32_t ov[16];
            tmem_ld_32x32b_x16(tO + c * 16, ov);
            asm volatile("tcgen05.wait::ld.sync.aligned;"
                         : "+r"(ov[0]), "+r"(ov[1]), "+r"(ov[2]), "+r"(ov[3]), "+r"(ov[4]), "+r"(ov[5]), "+r"(ov[6]), "+r"(ov[7]),
                           "+r"(ov[8]), "+r"(ov[9]), "+r"(ov[10]), "+r"(ov[11]), "+r"(ov[12]), "+r"(ov[13]), "+r"(ov[14]), "+r"(ov[15])
                         :
                         : "memory");
#pragma unroll
            for (int e = 0; e < 16; e += 2) {
              const float2 v = f2_unpack(f2_mul(f2_pack(__uint_as_float(ov[e]), __uint_as_float(ov[e + 1])), a2));
              ov[e] = __float_as_uint(v.x);
              ov[e + 1] = __float_as_uint(v.y);
            }
            tmem_st_32x32b_x16(tO + c * 16, ov);
          }
        }
        const float off = m == -INFINITY ? 0.f : m;
        const uint64_t sl2x2 = f2_pack(sl2, sl2), neg2 = f2_pack(-off, -off);
        uint64_t sum2[4] = {0ull, 0ull, 0ull, 0ull};
#pragma unroll
        for (int c = 0; c < 4; ++c) {
          uint32_t pk[16];
#pragma unroll
          for (int g0 = 0; g0 < 16; g0 += 8) {
            uint64_t x2[8], e2[8];
#pragma unroll
            for (int q = 0; q < 8; ++q) {
              const int e = 2 * (g0 + q);
              x2[q] = f2_fma(f2_pack(__uint_as_float(sc[c][e]), __uint_as_float(sc[c][e + 1])), sl2x2, neg2);
            }
#pragma unroll
            for (int q = 0; q < 8; ++q) {
              const int pair = g0 + q;
              if (((pair * kPolyPairs) % 16) < kPolyPairs) {
                e2[q] = ex2_poly2_clamped(x2[q]);
              } else {
                const float2 v = f2_unpack(x2[q]);
                e2[q] = f2_pack(ex2_approx(v.x), ex2_approx(v.y));
              }
            }
            if (masked) {
              // The cubic gives 2^-126 for a masked score; it must count as nothing
              // (a row whose block is all masked keeps its maximum of -inf).
#pragma unroll
              for (int q = 0; q < 8; ++q) {
                const int pair = g0 + q;
                if (((pair * kPolyPairs) % 16) < kPolyPairs) {
                  const int e = 2 * pair;
                  const float2 v = f2_unpack(e2[q]);
                  e2[q] = f2_pack(sc[c][e] == 0xFF800000u ? 0.f : v.x, sc[c][e + 1] == 0xFF800000u ? 0.f : v.y);
                }
              }
            }
#pragma unroll
            for (int q = 0; q < 8; ++q) {
              const int pair = g0 + q;
              sum2[pair & 3] = f2_add(sum2[pair & 3], e2[q]);
              const float2 v = f2_unpack(e2[q]);
              pk[pair] = Io<T>::pack2(v.x, v.y);
            }
          }
          tmem_st_32x32b_x16(tS + c * 16, pk);
        }
        const float2 ls = f2_unpack(f2_add(f2_add(sum2[0], sum2[1]), f2_add(sum2[2], sum2[3])));
        l += ls.x + ls.y;
        tmem_st_wait();
        tc_fence_before();
        mbar_arrive(&p_ready[w]);
      }
      if (ok) ok = mbar_wait_warp(&o_full[w], (blocks - 1) & 1u, abort_flag, p.err, kErrPagedWait);
      if (!ok) break;
      tc_fence_after();
      // ------------------------------------------------------------ results --
      const bool whole = x.first == 0 && n == x.item_blocks;
      const float f = whole ? (l == 0.f ? 0.f : 1.0f / l) : 1.f;
      const int head = x.kh * p.group + static_cast<int>((real ? row : rows - 1) - static_cast<int64_t>(i) * p.group);
      T* out = static_cast<T*>(p.o) + (x.s.first + i) * p.o_tok + head * p.o_head;
      const int64_t part = (static_cast<int64_t>(worker) * 2 + (t == t_first ? 0 : 1)) * kItemRows + w * kTileRows + r;
      float* po = p.part_o + part * D;
#pragma unroll
      for (int c = 0; c < D / 32; ++c) {
        uint32_t ov[32];
        tmem_ld_32x32b_x32(tO + c * 32, ov);
        tmem_ld_wait_regs(ov);
        if (real) {
          if (whole) {
#pragma unroll
            for (int q = 0; q < 4; ++q) {
              float v[8];
#pragma unroll
              for (int e = 0; e < 8; ++e) v[e] = l == 0.f ? 0.f : __uint_as_float(ov[8 * q + e]) * f;
              *reinterpret_cast<uint4*>(out + 32 * c + 8 * q) =
                  make_uint4(Io<T>::pack2(v[0], v[1]), Io<T>::pack2(v[2], v[3]), Io<T>::pack2(v[4], v[5]), Io<T>::pack2(v[6], v[7]));
            }
          } else {
#pragma unroll
            for (int q = 0; q < 8; ++q) {
              const bool none = l == 0.f;
              *reinterpret_cast<float4*>(po + 32 * c + 4 * q) =
                  make_float4(none ? 0.f : __uint_as_float(ov[4 * q]), none ? 0.f : __uint_as_float(ov[4 * q + 1]),
                              none ? 0.f : __uint_as_float(ov[4 * q + 2]), none ? 0.f : __uint_as_float(ov[4 * q + 3]));
            }
          }
        }
      }
      if (real && !whole) *reinterpret_cast<float2*>(p.part_ml + part * 2) = make_float2(m, l);
      tc_fence_before();
      mbar_arrive(&o_free[w]);
      if (t + n >= t_end && threadIdx.x == 0) {
        Cut cut{};
        if (x.first == 0 && !whole) {
          cut.parts = run_of(total, workers, t + x.item_blocks - 1) - worker + 1;
          cut.slot = t == t_first ? 0 : 1;
          cut.rows = static_cast<int>(min(rows - static_cast<int64_t>(x.rt) * kItemRows, static_cast<int64_t>(kItemRows)));
          cut.first_token = x.s.first;
          cut.row0 = x.rt * kItemRows;
          cut.kv_head = x.kh;
        }
        p.cuts[worker] = cut;
      }
      t += n;
      if (t < t_end) cur.next(p);
    }
  }

  tc_fence_before();
  __syncthreads();
  if (warp == 8) {
    __syncwarp();
    tc_fence_after();
    tmem_dealloc(tmem_base, L::kTmemCols);
  }
}

template <typename T, int D>
cudaError_t run_prefill(PagedParams p, cudaStream_t s) {
  using L = Layout<D>;
  static_assert(L::kSmem + 1024 <= 227 * 1024 && 8 * (kMaxBatch + 1) <= L::kSlots * L::kSlotBytes, "shared memory");
  auto kern = paged_prefill_kernel<T, D>;
  cudaFuncAttributes fa{};
  cudaError_t e = cudaFuncGetAttributes(&fa, kern);
  if (e != cudaSuccess) return e;
  if (fa.numRegs != kLaunchRegs) return cudaErrorInvalidConfiguration;   // the setmaxnreg split counts on it
  e = cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, L::kSmem);
  if (e != cudaSuccess) return e;
  const int batch = p.seqs.batch;
  const Seqs all = p.seqs;
  for (int b0 = 0; b0 < batch; b0 += kMaxBatch) {
    p.seqs.batch = batch - b0 < kMaxBatch ? batch - b0 : kMaxBatch;
    p.seqs.page_table = all.page_table + b0 * all.table_stride;
    p.seqs.starts = all.starts + b0;
    p.seqs.lens = all.lens + b0;
    e = launch_pdl(kern, dim3(p.workers), dim3(kThreads), static_cast<size_t>(L::kSmem), s, p);
    if (e != cudaSuccess) return e;
    e = launch_pdl(paged_join_kernel<T, D>, dim3(join_blocks(p.workers), 16), dim3(kJoinThreads), 0, s, p, int{kItemRows});
    if (e != cudaSuccess) return e;
  }
  return cudaSuccess;
}

}  // namespace

int64_t paged_prefill_workspace(int dim, int sms) {
  return int64_t{2} * sms * kItemRows * (dim + 2) * static_cast<int64_t>(sizeof(float)) + sms * static_cast<int64_t>(sizeof(Cut));
}

cudaError_t launch_paged_prefill(PagedParams p, int dtype, void* workspace, cudaStream_t stream) {
  p.workers = device_num_sms();
  p.part_o = static_cast<float*>(workspace);
  p.part_ml = p.part_o + int64_t{2} * p.workers * kItemRows * p.dim;
  p.cuts = reinterpret_cast<Cut*>(p.part_ml + int64_t{2} * p.workers * kItemRows * 2);
  if (dtype == LUNARA_BF16)
    return p.dim == 64 ? run_prefill<__nv_bfloat16, 64>(p, stream) : run_prefill<__nv_bfloat16, 128>(p, stream);
  return p.dim == 64 ? run_prefill<__half, 64>(p, stream) : run_prefill<__half, 128>(p, stream);
}

}  // namespace lunara
