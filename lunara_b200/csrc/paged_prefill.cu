// Attention over the paged cache for many query rows per sequence (prompts and
// chunks of prompts), on tcgen05.
//
// The query rows of a sequence and key head (its tokens times the query heads
// of the group) make items of 256 rows: two tiles of 128 that share every key
// block: 4 * 256 * 128 * D operations per 128-key block against 2 * 128 * D cached
// elements read. Bound by the chain S, softmax, P of a tile, which is longer than
// the other tile's products (tensor pipe 44 %, exponentials 34 %). Measured on
// B200: 1024 tokens each of 3 sequences of 4060 to 16384 keys, 32/8 heads of 128 in
// bf16, 0.59 ms for 533 GFLOP (0.90 PFLOP/s), 0.66 ms in a row of calls.
//   * Equal runs: the key blocks of all items, in the order (sequence, key head,
//     row tile, block), are dealt to the persistent CTAs in equal contiguous
//     runs, so neither ragged lengths nor causal triangles nor few items leave
//     SMs idle. How many blocks precede a row tile is a sum of floors of a
//     linear function, taken in closed form. Items that a run cuts leave
//     partial O, maximum and sum in the workspace, and a second kernel joins
//     them.
//   * warps 0-3, 4-7   softmax of tile 0 and 1 (thread = row)
//     warp 8           tcgen05.mma issuer
//                        S_w = Q_w K^T  (128 x 128 x D, operands in shared memory)
//                        O_w += P_w V   (128 x D x 128, P_w from TMEM)
//                        in the order P_0 V, next S_0, P_1 V, next S_1: one tile's
//                        products run whole while the other's softmax has the
//                        issue slots (an issuer per tile interleaved them: 4030
//                        instead of 3200 cycles a block)
//     warps 10, 11     copy K and V (and Q between them) into 128-byte-swizzled
//                        tiles: a block whose keys all take part by TMA, a box
//                        per page; one at the ends of what the item sees, with
//                        bad pages, or of pages that do not tile a block, row by
//                        row with cp.async, with zeros for the keys left out
//   * TMEM: S_w 128 columns each, O_w D columns each; P_w (16-bit pairs) takes
//     the first half of S_w's columns once the row is in registers. The next
//     S_w is issued right behind P_w V; meanwhile the other tile's products run.
#include <cudaTypedefs.h>

#include <type_traits>

#include "kernels.h"
#include "paged_attention.cuh"

namespace lunara {
namespace {

constexpr int kItemRows = 256;
constexpr int kTileRows = 128;
constexpr int kBlock = 128;              // keys per block
constexpr int kThreads = 384;
constexpr int kCopyWarps = 2;
constexpr int kMaxBatch = 1024;          // sequences per launch
constexpr float kRescaleLog2 = 8.0f;
// setmaxnreg split of the launch's 384 x 168 registers.
constexpr int kLaunchRegs = 168;
constexpr int kSoftmaxRegs = 224, kOtherRegs = 56;
static_assert(256 * kSoftmaxRegs + 128 * kOtherRegs <= kThreads * kLaunchRegs, "register split");
// Of 16 exponential pairs these are on the FMA pipe, as in attention.cu: a cubic,
// off by 7.5e-5 where rounding a probability to 16 bits is by up to 4.9e-4 (f16)
// or 3.9e-3 (bf16).
constexpr int kPolyPairs = 4;
constexpr int kMaskRing = 16;            // blocks whose key masks are kept; more than the ring can run ahead
constexpr int kItemRing = 4;             // items whose block counts are kept; the copies run one item ahead at most

// D: the head dimension rounded up to 64 or 128; columns behind it are zeros in
// shared memory (TMA fills what lies outside the tensor) and are not stored.
template <int D>
struct Layout {
  static constexpr int kHalves = D / 64;                       // 64-element column blocks of a tile
  static constexpr uint32_t kHalfBytes = kBlock * 128;         // 128 rows of 128 bytes
  static constexpr uint32_t kSlotBytes = kHalves * kHalfBytes; // one K or V block
  static constexpr uint32_t kQBytes = 2 * kSlotBytes;          // two row tiles
  static constexpr int kSlots = D == 128 ? 5 : 8;              // ring of K and V blocks: K0, V0, K1, V1, ...
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
__global__ void __launch_bounds__(kThreads, 1)
    paged_prefill_kernel(const __grid_constant__ PagedParams p, const __grid_constant__ CUtensorMap tk,
                         const __grid_constant__ CUtensorMap tv, int box_rows) {
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
  uint64_t* q_free = q_full + 1;            // the item's last S is done
  uint64_t* full = q_free + 1;              // [kSlots]
  uint64_t* empty = full + L::kSlots;       // [kSlots] the products are done with the slot
  uint64_t* s_full = empty + L::kSlots;     // [2]
  uint64_t* p_ready = s_full + 2;           // [2]
  uint64_t* o_full = p_ready + 2;           // [2]
  uint64_t* o_free = o_full + 2;            // [2] the item's O_w is read
  uint64_t* drain_bar = o_free + 2;
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(drain_bar + 1);
  volatile int* abort_flag = reinterpret_cast<volatile int*>(tmem_slot + 1);
  int* s_blocks = reinterpret_cast<int*>(tmem_slot + 2);   // [kItemRing] blocks of an item's part
  // The prefix sums stand in the ring until the roles begin.
  int64_t* prefix = reinterpret_cast<int64_t*>(sRing);
  __shared__ int64_t warp_sums[kThreads / 32];
  __shared__ Cursor s_cursor;

  const int warp = threadIdx.x >> 5;
  const int lane = threadIdx.x & 31;
  if (threadIdx.x == 0) {
    mbar_init(q_full, kCopyWarps);
    mbar_init(q_free, 1);
    for (int i = 0; i < L::kSlots; ++i) {
      mbar_init(&full[i], 1);
      mbar_init(&empty[i], 1);
    }
    for (int w = 0; w < 2; ++w) {
      mbar_init(&s_full[w], 1);
      mbar_init(&p_ready[w], kTileRows);
      mbar_init(&o_full[w], 1);
      mbar_init(&o_free[w], kTileRows);
    }
    mbar_init(drain_bar, 1);
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
  if (threadIdx.x == 0) p.cuts[worker].parts = 0;   // until the run's end says otherwise
  if (worker < workers) {
    t_first = run_start(total, workers, worker);
    t_end = run_start(total, workers, worker + 1);
    if (threadIdx.x == 0) s_cursor.seek(p, prefix, t_first);
  }
  // The prefix sums are used up: the ring may be written, by TMA too, whose
  // writes have no order with the plain ones before them without the fence.
  fence_proxy_async_smem();
  __syncthreads();

  if (warp >= 10) {
    reg_dealloc<kOtherRegs>();
    // -------------------------------------------------------------- copies --
    // Warp 10 fills the ring's K slots, warp 11 its V slots.
    const int kv = warp - 10;
    constexpr int kPer = D / 8, kRowsAtOnce = 32 / kPer;   // lanes to a row, rows at once
    const int chunk = lane % kPer, sub = lane / kPer;
    const uint32_t lane_dst = (chunk >> 3) * L::kHalfBytes;
    const int boxes = box_rows > 0 ? kBlock / box_rows : 0;
    const CUtensorMap* map = kv == 0 ? &tk : &tv;
    if (lane == 0 && boxes > 0) tma_prefetch_desc(map);   // (without boxes there is no map)
    const uint32_t page_u = kv == 0 ? p.k_page_u : p.v_page_u;
    bool ok = true;
    Cursor cur = s_cursor;
    int slot = kv;             // ring slot of this warp's next block, and the phase of its empty barrier
    uint32_t phase = 0, block_count = 0, items = 0;
    uint32_t filled = 0, filled_phase = 0;   // bits of the slots that TMA was started on, and of their phases
    for (int64_t t = t_first; ok && t < t_end; ++items) {
      cur.clip(t_end - t);
      const Item& x = cur.x;
      int lo, hi;
      item_keys(p, x, lo, hi);
      // Q: row r of the item is token r / group, head r % group; a warp copies a tile.
      if (!mbar_wait_warp(q_free, (items & 1u) ^ 1u, abort_flag, p.err, kErrPagedWait)) { ok = false; break; }
      {
        // Lane l finds the places of rows 32 h + l (32-bit: tokens * heads is below 2^31).
        const int row0 = x.rt * kItemRows + kTileRows * kv, rows = x.s.n * p.group;
        const uint32_t dst = smem_u32(sQ) + kv * L::kSlotBytes + lane_dst;
#pragma unroll 1
        for (int h = 0; h < 4; ++h) {
          const int row = row0 + 32 * h + lane;
          const uint32_t use = __ballot_sync(0xffffffffu, row < rows);
          const int i = (row < rows ? row : 0) / p.group, head = x.kh * p.group + (row < rows ? row : 0) - i * p.group;
          const bool in_row = 8 * chunk < p.dim;
          const char* src = static_cast<const char*>(p.q) + ((x.s.first + i) * p.q_tok + head * p.q_head) * 2;
          const uint32_t src_lo = static_cast<uint32_t>(reinterpret_cast<uint64_t>(src)), src_hi = static_cast<uint32_t>(reinterpret_cast<uint64_t>(src) >> 32);
#pragma unroll 4
          for (int it = 0; it < 32 / kRowsAtOnce; ++it) {
            const int r = it * kRowsAtOnce + sub;
            const uint64_t at = (static_cast<uint64_t>(__shfl_sync(0xffffffffu, src_hi, r)) << 32) | __shfl_sync(0xffffffffu, src_lo, r);
            copy16(dst + (32 * h + r) * 128 + (((chunk & 7) ^ (r & 7)) << 4), reinterpret_cast<const char*>(at) + (in_row ? 16 * chunk : 0),
                   ((use >> r) & 1u) != 0u && in_row);
          }
        }
      }
      asm volatile("cp.async.commit_group;" ::: "memory");
      asm volatile("cp.async.wait_group 0;" ::: "memory");
      fence_proxy_async_smem();
      __syncwarp();
      if (lane == 0) {
        if (kv == 0) s_blocks[items % kItemRing] = x.n;
        mbar_arrive(q_full);
      }
      const int32_t* table = p.seqs.page_table + x.b * p.seqs.table_stride;
      auto page_of = [&](int key) {   // -1: no page, or one outside the cache
        const int page = table[p.seqs.page_div.div(key)];
        if (page >= 0 && page < p.num_pages) return page;
        atomicCAS(p.err, 0u, static_cast<unsigned>(kErrCachePage));
        return -1;
      };
      // The lane's box of a block, looked up a block ahead.
      auto box_page = [&](int block) {
        const int key = block * kBlock + lane * box_rows;
        return lane < boxes && block * kBlock >= lo && block * kBlock + kBlock <= hi ? page_of(key) : -1;
      };
      int next = box_page(x.block0);
      for (int j = 0; j < x.n; ++j, ++block_count) {
        const int key0 = (x.block0 + j) * kBlock, page = next;
        if (j + 1 < x.n) next = box_page(x.block0 + j + 1);
        if (!mbar_wait_warp(&empty[slot], phase ^ 1u, abort_flag, p.err, kErrPagedWait)) { ok = false; break; }
        uint8_t* tile = sRing + slot * L::kSlotBytes;
        const bool whole = boxes > 0 && __popc(__ballot_sync(0xffffffffu, page >= 0)) == boxes;
        if (whole) {
          if (lane == 0) {
            if (kv == 0) *reinterpret_cast<uint4*>(&s_mask[(block_count % kMaskRing) * 4]) = make_uint4(~0u, ~0u, ~0u, ~0u);
            mbar_arrive_expect_tx(&full[slot], L::kSlotBytes);
          }
          __syncwarp();
          if (lane < boxes) {
            const int key = key0 + lane * box_rows, in_page = key - p.seqs.page_div.div(key) * p.page_size;
#pragma unroll
            for (int h = 0; h < L::kHalves; ++h)
              tma_load_4d(tile + h * L::kHalfBytes + lane * box_rows * 128, map, &full[slot], 64 * h, in_page, x.kh, page);
          }
          filled |= 1u << slot;
          filled_phase = (filled_phase & ~(1u << slot)) | (phase << slot);
        } else {
          const bool in_row = 8 * chunk < p.dim;
          const char* base = static_cast<const char*>(kv == 0 ? p.k : p.v) + x.kh * (kv == 0 ? p.k_head : p.v_head) * 2 + (in_row ? 16 * chunk : 0);
#pragma unroll 1
          for (int h = 0; h < 4; ++h) {
            const int key = key0 + 32 * h + lane;
            const int pg = key >= lo && key < hi ? page_of(key) : -1;
            const uint32_t use = __ballot_sync(0xffffffffu, pg >= 0);
            if (kv == 0 && lane == 0) s_mask[(block_count % kMaskRing) * 4 + h] = use;
            // Where the lane's row stands, in units of p.unit bytes.
            const uint32_t in_page = static_cast<uint32_t>(key - p.seqs.page_div.div(key) * p.page_size) * p.row_u;
            const uint32_t at = pg >= 0 ? static_cast<uint32_t>(pg) * page_u + in_page : 0u;
            const uint32_t dst = smem_u32(tile) + lane_dst + 32 * h * 128;
#pragma unroll 4
            for (int it = 0; it < 32 / kRowsAtOnce; ++it) {
              const int r = it * kRowsAtOnce + sub;
              const uint32_t row_at = __shfl_sync(0xffffffffu, at, r);
              copy16(dst + r * 128 + (((chunk & 7) ^ (r & 7)) << 4), base + static_cast<uint64_t>(row_at) * p.unit,
                     ((use >> r) & 1u) != 0u && in_row);
            }
          }
          asm volatile("cp.async.commit_group;" ::: "memory");
          asm volatile("cp.async.wait_group 0;" ::: "memory");
          fence_proxy_async_smem();
          __syncwarp();
          if (lane == 0) mbar_arrive(&full[slot]);
        }
        slot += 2;
        if (slot >= L::kSlots) { slot -= L::kSlots; phase ^= 1u; }
      }
      t += x.n;
      if (ok && t < t_end) cur.next(p);
    }
    if (!ok)   // the copies in flight are waited for
      for (int i = 0; i < L::kSlots; ++i)
        if ((filled >> i) & 1u) mbar_drain_wait(&full[i], (filled_phase >> i) & 1u, 200000000ull);
  } else if (warp >= 8) {
    reg_dealloc<kOtherRegs>();
    // ----------------------------------------------------------- MMA issuer --
    const bool leader = elect_one_sync();
    auto wait = [&](uint64_t* bar, uint32_t parity) {
      return mbar_wait_warp(bar, parity, abort_flag, p.err, kErrPagedWait);
    };
    const uint64_t qd0 = sw128_desc(smem_u32(sQ), 16, 1024);
    const uint64_t kd0 = sw128_desc(smem_u32(sRing), 16, 1024);
    const uint64_t vd0 = sw128_desc(smem_u32(sRing), L::kHalfBytes, 1024);
    auto issue_s = [&](int w, int slot) {
      const uint64_t qd = qd0 + w * (L::kSlotBytes >> 4), kd = kd0 + static_cast<uint64_t>(slot) * (L::kSlotBytes >> 4);
#pragma unroll
      for (int kk = 0; kk < D / 16; ++kk) {
        const uint64_t off = (kk >> 2) * (L::kHalfBytes >> 4) + 2 * (kk & 3);
        umma_f16_ss(tmem_base + L::kTmemS + w * 128, qd + off, kd + off, IDESC_S, kk > 0 ? 1u : 0u);
      }
    };
    auto issue_pv = [&](int w, int slot, bool first) {
      const uint64_t vd = vd0 + static_cast<uint64_t>(slot) * (L::kSlotBytes >> 4);
#pragma unroll
      for (int kk = 0; kk < kBlock / 16; ++kk)
        umma_f16_ts(tmem_base + L::kTmemO + w * D, tmem_base + L::kTmemS + w * 128 + kk * 8, vd + 128 * kk, IDESC_PV,
                    (!first || kk > 0) ? 1u : 0u);
    };
    bool ok = warp == 8;              // (the warpgroup's other warp idles)
    uint32_t items = 0, blocks = 0;   // items and blocks so far
    int ks = 0;                       // ring slot of the next K, and its phase
    uint32_t kp = 0;
    for (int left = __shfl_sync(0xffffffffu, static_cast<int>(t_end - t_first), 0); ok && left > 0; ++items) {
      if (!wait(q_full, items & 1u)) { ok = false; break; }
      // (The shuffle tells the compiler that the count, and with it the ring slot
      // and the descriptors, are the same in all lanes.)
      const int n = __shfl_sync(0xffffffffu, *reinterpret_cast<volatile int*>(&s_blocks[items % kItemRing]), 0);
      left -= n;
      if (!wait(&full[ks], kp)) { ok = false; break; }
      tc_fence_after();
      if (leader) {
        issue_s(0, ks);
        umma_commit(&s_full[0]);
        issue_s(1, ks);
        umma_commit(&s_full[1]);
        umma_commit(&empty[ks]);
        if (n == 1) umma_commit(q_free);
      }
      __syncwarp();
      for (int j = 0; j < n && ok; ++j, ++blocks) {
        const int vs = ks + 1 == L::kSlots ? 0 : ks + 1, next = vs + 1 == L::kSlots ? 0 : vs + 1;
        const uint32_t vp = vs == 0 ? kp ^ 1u : kp, np = next == 0 ? vp ^ 1u : vp;
        const bool more = j + 1 < n;
        if (!wait(&full[vs], vp)) { ok = false; break; }
        if (more && !wait(&full[next], np)) { ok = false; break; }
#pragma unroll
        for (int w = 0; w < 2; ++w) {
          if (!wait(&p_ready[w], blocks & 1u)) { ok = false; break; }
          // The item's first P V overwrites O: the item before must have been read.
          if (j == 0 && items > 0 && !wait(&o_free[w], (items - 1) & 1u)) { ok = false; break; }
          tc_fence_after();
          if (leader) {
            issue_pv(w, vs, j == 0);
            umma_commit(&o_full[w]);
            if (w == 1) umma_commit(&empty[vs]);
            if (more) {
              // S overwrites P, which shares its columns: the tensor core runs
              // the products of one thread in their order of issue, so P V has
              // read P by then.
              issue_s(w, next);
              umma_commit(&s_full[w]);
              if (w == 1) {
                umma_commit(&empty[next]);
                if (j + 2 == n) umma_commit(q_free);
              }
            }
          }
          __syncwarp();
        }
        ks = next;
        kp = np;
      }
    }
    if (!ok && warp == 8) {
      if (leader) umma_commit(drain_bar);
      __syncwarp();
      mbar_drain_wait(drain_bar, 0, 1000000000ull);
    }
  } else {
    reg_alloc<kSoftmaxRegs>();
    // ------------------------------------------------------------- softmax --
    const int w = warp >> 2, quarter = warp & 3, r = quarter * 32 + lane;
    const uint32_t lane_off = static_cast<uint32_t>(quarter * 32) << 16;
    const uint32_t tS = tmem_base + lane_off + L::kTmemS + w * 128;
    const uint32_t tO = tmem_base + lane_off + L::kTmemO + w * D;
    const float sl2 = exponent_factor(p.scale * 1.4426950408889634f);   // (the scale is not negative here)
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
      // The largest score so far (as of the last rescaling), its product with the
      // factor, and the sum. Exponents are score * factor - off in one FMA, off by
      // the rounding of `off`, 2^-24 of it. That cancels out as long as all of a
      // row's terms share it; where it could be felt in the differences (|off|
      // above 8192: "far"), `top` is taken off the scores first.
      float top = -INFINITY, off = -INFINITY, l = 0.f;
      auto far_off = [](float x) { return fabsf(x) > 8192.f; };
      // What the exponents' base is above top * factor.
      auto excess = [&](float t, float x) { return far_off(x) ? 0.f : fmaf(-t, sl2, x); };
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
        float mx = fmax3_nan(fmax3_nan(mxp[0], mxp[1], mxp[2]), fmax3_nan(mxp[3], mxp[4], mxp[5]), fmax_nan(mxp[6], mxp[7]));
        // inf - inf makes NaN of a row with a score of +inf, as its softmax is; the
        // cubic's clamp would drop it where such a key stands in its columns.
        if (mx == INFINITY) mx = NAN;
        if (j == 0) {
          top = mx;
          off = mx * sl2;
        } else if (__any_sync(0xffffffffu, !(mx <= top || (mx - top) * sl2 <= kRescaleLog2))) {
          // O is rescaled once P V of the block before has completed (as it has:
          // S of this block ran after it).
          if (!mbar_wait_warp(&o_full[w], (blocks - 1) & 1u, abort_flag, p.err, kErrPagedWait)) { ok = false; break; }
          tc_fence_after();
          const float next = fmax_nan(top, mx), next_off = next * sl2;
          const float alpha = next == -INFINITY ? 1.f : ex2_approx(fmaf(top - next, sl2, excess(top, off) - excess(next, next_off)));
          l *= alpha;
          top = next;
          off = next_off;
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
        const bool far = far_off(off);   // (a row that has seen no key too: nothing is taken off its -inf)
        if (__any_sync(0xffffffffu, far)) {
          const float sub = far && top != -INFINITY ? top : 0.f;
#pragma unroll
          for (int cc = 0; cc < 4; ++cc)
#pragma unroll
            for (int e = 0; e < 32; ++e) sc[cc][e] = __float_as_uint(__uint_as_float(sc[cc][e]) - sub);
        }
        const float minus = far ? 0.f : -off;
        const uint64_t sl2x2 = f2_pack(sl2, sl2), neg2 = f2_pack(minus, minus);
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
                // The cubic's result below -126, masked scores' too, is dropped by
                // fp16's rounding. bf16 would hold it, and values may be as large
                // (2^-126 of a finite 2^121 is 1/32): there it is taken off, which
                // leaves exactly 0 and moves no other result by more than it.
                e2[q] = ex2_poly2_clamped(x2[q]);
                if constexpr (kBF16) e2[q] = f2_add(e2[q], f2_pack(-ex2_poly2_floor(), -ex2_poly2_floor()));
              } else {
                const float2 v = f2_unpack(x2[q]);
                e2[q] = f2_pack(ex2_approx(v.x), ex2_approx(v.y));
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
      // With fp16 a masked score adds 2^-126 at most (the cubic's smallest), which
      // is nothing beside a row's largest, but the whole sum of a row that saw no
      // key: such a row keeps its maximum of -inf.
      if (top == -INFINITY) l = 0.f;
      const bool whole = x.first == 0 && n == x.item_blocks;
      // A part's exponents are brought to the base top * factor, the same in all parts.
      const float f = l == 0.f ? 0.f : whole ? 1.0f / l : ex2_approx(excess(top, off));
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
              if (32 * c + 8 * q < p.dim)
                *reinterpret_cast<uint4*>(out + 32 * c + 8 * q) =
                  make_uint4(Io<T>::pack2(v[0], v[1]), Io<T>::pack2(v[2], v[3]), Io<T>::pack2(v[4], v[5]), Io<T>::pack2(v[6], v[7]));
            }
          } else {
#pragma unroll
            for (int q = 0; q < 8; ++q) {
              const bool none = l == 0.f;
              *reinterpret_cast<float4*>(po + 32 * c + 4 * q) =
                  make_float4(none ? 0.f : __uint_as_float(ov[4 * q]) * f, none ? 0.f : __uint_as_float(ov[4 * q + 1]) * f,
                              none ? 0.f : __uint_as_float(ov[4 * q + 2]) * f, none ? 0.f : __uint_as_float(ov[4 * q + 3]) * f);
            }
          }
        }
      }
      if (real && !whole) *reinterpret_cast<float4*>(p.part_ml + part * kPartMl) = make_float4(top, l * f, sl2, 0.f);
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

// Tensor map of the pages, a box of `rows` rows of 64 elements.
bool encode_pages(CUtensorMap* map, const void* pages, int dtype, const PagedParams& p, int64_t page, int64_t head, int rows) {
  auto encode = reinterpret_cast<PFN_cuTensorMapEncodeTiled>(tensor_map_encoder());
  if (encode == nullptr) return false;
  const cuuint64_t dims[4] = {static_cast<cuuint64_t>(p.dim), static_cast<cuuint64_t>(p.page_size),
                              static_cast<cuuint64_t>(p.kv_heads), static_cast<cuuint64_t>(p.num_pages)};
  // A dimension of extent 1 is never stepped: any stride will do.
  const cuuint64_t row = static_cast<cuuint64_t>(p.dim) * 2;
  const cuuint64_t strides[3] = {row, p.kv_heads == 1 ? row : static_cast<cuuint64_t>(head) * 2,
                                 p.num_pages == 1 ? row : static_cast<cuuint64_t>(page) * 2};
  for (cuuint64_t v : strides)
    if (v == 0 || v % 16 != 0 || v >= (cuuint64_t{1} << 40)) return false;
  const cuuint32_t box[4] = {64, static_cast<cuuint32_t>(rows), 1, 1};
  const cuuint32_t step[4] = {1, 1, 1, 1};
  return encode(map, dtype == LUNARA_BF16 ? CU_TENSOR_MAP_DATA_TYPE_BFLOAT16 : CU_TENSOR_MAP_DATA_TYPE_FLOAT16, 4,
                const_cast<void*>(pages), dims, strides, box, step, CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B,
                CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}

template <typename T, int D>
cudaError_t run_prefill(PagedParams p, cudaStream_t s) {
  using L = Layout<D>;
  static_assert(L::kSmem + 1024 <= 227 * 1024 && 8 * (kMaxBatch + 1) <= L::kSlots * L::kSlotBytes, "shared memory");
  auto kern = paged_prefill_kernel<T, D>;
  static std::atomic<uint64_t> prepared{0};
  cudaError_t e = prepare_once(kern, prepared, static_cast<int>(L::kSmem), kLaunchRegs);   // the setmaxnreg split counts on the registers
  if (e != cudaSuccess) return e;
  // TMA where pages tile a 128-key block in boxes of whole swizzle atoms (8
  // rows); row by row elsewhere (box_rows 0).
  const int ps = p.page_size;
  int box_rows = ps >= 8 && (ps % kBlock == 0 || kBlock % ps == 0) ? (ps < kBlock ? ps : kBlock) : 0;
  CUtensorMap mk{}, mv{};
  const int dtype = std::is_same<T, __nv_bfloat16>::value ? LUNARA_BF16 : LUNARA_F16;
  if (box_rows > 0 && (!encode_pages(&mk, p.k, dtype, p, p.k_page, p.k_head, box_rows) ||
                       !encode_pages(&mv, p.v, dtype, p, p.v_page, p.v_head, box_rows)))
    box_rows = 0;
  const int batch = p.seqs.batch;
  const Seqs all = p.seqs;
  for (int b0 = 0; b0 < batch; b0 += kMaxBatch) {
    p.seqs.batch = batch - b0 < kMaxBatch ? batch - b0 : kMaxBatch;
    p.seqs.page_table = all.page_table + b0 * all.table_stride;
    p.seqs.starts = all.starts + b0;
    p.seqs.lens = all.lens + b0;
    e = launch_pdl(kern, dim3(p.workers), dim3(kThreads), static_cast<size_t>(L::kSmem), s, p, mk, mv, box_rows);
    if (e != cudaSuccess) return e;
    e = launch_pdl(paged_join_kernel<T, D>, dim3(join_blocks(p.workers), 16), dim3(kJoinThreads), 0, s, p, int{kItemRows});
    if (e != cudaSuccess) return e;
  }
  return cudaSuccess;
}

}  // namespace

int64_t paged_prefill_workspace(int dim, int sms) {
  return int64_t{2} * sms * kItemRows * ((dim <= 64 ? 64 : 128) + kPartMl) * static_cast<int64_t>(sizeof(float)) + sms * static_cast<int64_t>(sizeof(Cut));
}

cudaError_t launch_paged_prefill(PagedParams p, int dtype, void* workspace, cudaStream_t stream) {
  p.workers = device_num_sms();
  p.part_o = static_cast<float*>(workspace);
  p.part_ml = p.part_o + int64_t{2} * p.workers * kItemRows * (p.dim <= 64 ? 64 : 128);
  p.cuts = reinterpret_cast<Cut*>(p.part_ml + int64_t{2} * p.workers * kItemRows * kPartMl);
  if (dtype == LUNARA_BF16)
    return p.dim <= 64 ? run_prefill<__nv_bfloat16, 64>(p, stream) : run_prefill<__nv_bfloat16, 128>(p, stream);
  return p.dim <= 64 ? run_prefill<__half, 64>(p, stream) : run_prefill<__half, 128>(p, stream);
}

}  // namespace lunara
