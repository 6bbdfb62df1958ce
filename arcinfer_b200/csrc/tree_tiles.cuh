// Tree attention on the tensor cores: tiles of 128 rows (a node and a query head each) against tiles of
// keys and values that come from their pages by tiled copies.
#pragma once
#include "cache.cuh"
#include "tcgen05.cuh"

namespace arcs {

struct TreeDev {
  CacheDev c;  // k and v: the layer's
  const char* q;
  char* out;
  int64_t q_token_stride, q_head_stride, out_token_stride, out_head_stride;  // bytes
  float* lse;
  const int32_t* node_off;
  const unsigned long long* mask;
  int32_t T, Hq, group, max_nodes;
  float scale_log2;  // scale * log2 e
  // the tile kernel's
  int32_t by_row, page_rows, head_rows, no_row;  // where a page's rows lie in the tensor maps; a row behind the last
  int32_t part_rows;                             // rows of a block of partial results
  uint32_t* prefix;                              // [slots + 2] units of work before a slot, and what an item counts for itself
  float2* part_stat;                             // [CTAs][2][part_rows] (maximum in log2, sum)
  float4* part;                                  // [CTAs][2][dim / 4][part_rows]: a warp's rows side by side where they are written
};

// How the two groups of softmax warps share the work. kSplit: one tile of rows, the tiles of keys
// go to the groups in turn, each with sums of its own that meet at the end. kPair: two tiles of rows,
// one a group, over the same keys. kShare: as kSplit, with one set of sums (at dim 256 it takes half of
// the tensor memory): the groups hand the reference of the weights on from tile to tile.
enum { kSplit = 0, kPair = 1, kShare = 2 };

template <int DIM, int MODE>
struct TilePlan {
  static constexpr int kKeys = 128;                            // keys in a tile
  static constexpr int kRows = MODE == kPair ? 256 : 128;      // rows of an item
  // Pieces of a tile in the ring: at dim 256 the keys come as two halves of 128 values each, the values as
  // two halves of 64 keys. (Tiles of 64 keys instead cost a third more: a product of 128 x 64 x 16 takes
  // 56 cycles, not the half of 64, because the queries are read again for every one.)
  static constexpr int kSub = DIM == 256 ? 2 : 1;
  static constexpr int kQBytes = kRows * DIM * 2;
  static constexpr int kTile = kKeys * DIM * 2 / kSub;         // 32 KB, at dim 64 16 KB
  // slots of the ring: 160 KB a CTA keep the memory busy (24 MB under way on all of them). kSplit leaves room
  // beside them for a CTA of join_kernel; at dim 256 a fifth slot gains more (84 -> 79 us for 24 nodes over 131071).
  static constexpr int kSlots = DIM == 64 ? 10 : 5;
  static constexpr int kSmem = kQBytes + kSlots * kTile + 2048 + 1024;
  static constexpr uint32_t kScore1 = kKeys;                   // columns: scores 0, scores 1, sums from 256 on
  static constexpr uint32_t kSums = 256;
  // What a tile of keys costs, and an item for its beginning and end (queries, the last tile's way through,
  // results): fitted to the ends of all CTAs. With two tiles of rows 2.73 us, with one of them 2.28, an item
  // 8.8; with one tile of rows 1.35 us and an item 5.0.
  static constexpr int kCost = MODE == kPair ? 6 : 1, kCostOne = MODE == kPair ? 5 : 1, kItemCost = MODE == kPair ? 18 : 4;
};
static_assert(TilePlan<128, kSplit>::kSmem <= 232448 && TilePlan<128, kPair>::kSmem <= 232448 && TilePlan<256, kShare>::kSmem <= 232448 &&
              TilePlan<64, kPair>::kSmem <= 232448, "227 KB of shared memory");
// 8 softmax warps, two that copy keys and values, one that issues the products, one that brings the queries
constexpr int kTileThreads = 384;
constexpr int kCtas = kSmCount;  // one a SM

struct SlotWork {
  int off, n, len, tiles, blocks;  // rows of the step, nodes, settled tokens; tiles of keys, blocks of rows a key head
  bool bad;
};
template <typename P>
__device__ __forceinline__ void size_up(const TreeDev& a, SlotWork& w) {
  w.tiles = w.n > 0 ? (w.len + w.n + P::kKeys - 1) / P::kKeys : 0;
  w.blocks = w.n > 0 ? (w.n * a.group + P::kRows - 1) / P::kRows : 0;
}
template <typename P>
__device__ __forceinline__ SlotWork slot_work(const TreeDev& a, int s) {
  SlotWork w;
  const int r1 = a.node_off[s + 1], used = a.c.used[s];
  w.off = a.node_off[s];
  w.n = r1 - w.off;
  w.len = a.c.len[s];
  w.bad = w.off < 0 || r1 < w.off || r1 > a.T || w.n > a.max_nodes ||
          (w.n > 0 && (w.len < 0 || used < 0 || used > a.c.max_pages || (int64_t)w.len + w.n > ((int64_t)used << a.c.page_shift)));
  if (w.bad) w.n = 0;
  size_up<P>(a, w);
  return w;
}

// The work is dealt out evenly in units of cost: all slots' items (key head, block of rows) lie in a row,
// each `extra` units for itself and then its tiles; CTA c of G takes what begins in [total c / G,
// total (c + 1) / G), so the lengths need not be known on the host. An item that lies in one CTA is
// finished there; one that is cut leaves partial results, joined by join_kernel. `extra` is zero where a CTA
// gets fewer than 16 tiles: there an even share of tiles counts for more.
template <typename P>
struct Costs {
  int first, head, last;  // units of an item with all its rows, of a key head's items; of a tile in the head's last item
  __device__ __forceinline__ Costs(const TreeDev& a, const SlotWork& w, int extra) {
    last = w.n * a.group - (w.blocks - 1) * P::kRows <= 128 ? P::kCostOne : P::kCost;
    first = w.tiles * P::kCost + extra;
    head = w.blocks > 0 ? (w.blocks - 1) * first + w.tiles * last + extra : 0;
  }
};
__device__ __forceinline__ uint32_t first_unit(uint32_t total, int c, int ctas) { return (uint32_t)((uint64_t)total * (uint32_t)c / (uint32_t)ctas); }
__device__ __forceinline__ int cta_of_unit(uint32_t total, uint32_t u, int ctas) { return (int)(((uint64_t)(u + 1) * (uint32_t)ctas - 1) / total); }
template <typename P>
__device__ __forceinline__ int extra_units(uint32_t plain_total, int ctas) { return plain_total >= 16u * P::kCost * (uint32_t)ctas ? P::kItemCost : 0; }

struct Place {  // of an item
  int head, block, cost;
  uint32_t begins;  // its first unit
};
// the item that unit x of a slot belongs to
template <typename P>
__device__ __forceinline__ Place place_of(const SlotWork& w, const Costs<P>& c, uint32_t base, int x) {
  Place p;
  p.head = x / c.head;
  const int y = x - p.head * c.head;
  p.block = min(y / c.first, w.blocks - 1);
  p.cost = p.block == w.blocks - 1 ? c.last : P::kCost;
  p.begins = base + (uint32_t)(p.head * c.head + p.block * c.first);
  return p;
}

struct Piece {  // of an item: tiles [t0, t1)
  int head, block, t0, t1;
};
template <typename P>
struct Walk {
  uint32_t u, u1, base;
  int s, extra;
  SlotWork w;
  __device__ __forceinline__ bool next(const TreeDev& a, Piece& p) {
    while (u < u1) {
      Costs<P> c(a, w, extra);
      while (u >= base + (uint32_t)(c.head * a.c.heads)) {
        base += (uint32_t)(c.head * a.c.heads);
        w = slot_work<P>(a, ++s);
        c = Costs<P>(a, w, extra);
      }
      const Place at = place_of<P>(w, c, base, (int)(u - base));
      const int from = (int)(u - at.begins) - extra, ends = w.tiles * at.cost, to = min((int)(u1 - at.begins) - extra, ends);
      p.head = at.head;
      p.block = at.block;
      p.t0 = from <= 0 ? 0 : (from + at.cost - 1) / at.cost;
      p.t1 = to <= 0 ? 0 : (to + at.cost - 1) / at.cost;
      u = at.begins + (uint32_t)(to + extra);
      if (p.t0 < p.t1) return true;
    }
    return false;
  }
};

// Bounded wait; when one runs out, every other wait of the CTA ends too.
__device__ __forceinline__ uint64_t clock_ns() {
  uint64_t t;
  asm volatile("mov.u64 %0, %globaltimer;" : "=l"(t));
  return t;
}
__device__ __forceinline__ bool hold(uint64_t* bar, uint32_t parity, volatile int* fail) {
  if (mbar_try_wait(bar, parity)) return true;
  const uint64_t began = clock_ns();
  for (;;) {
#pragma unroll 1
    for (int i = 0; i < 64; ++i)
      if (mbar_try_wait(bar, parity)) return true;
    if (*fail) return false;
    if (clock_ns() - began > 2000000000ull) break;  // two seconds
  }
  *fail = 1;
  return false;
}
__device__ __forceinline__ bool hold_warp(uint64_t* bar, uint32_t parity, volatile int* fail) {
  return __all_sync(0xFFFFFFFFu, hold(bar, parity, fail));
}

// one arrival for a whole warp's work (the arrivals of a barrier are taken one after the other)
__device__ __forceinline__ void arrive_warp(uint64_t* bar) {
  __syncwarp();
  if ((threadIdx.x & 31) == 0) mbar_arrive(bar);
}

// The rows of an item to shared memory, swizzled as the tiles of keys are: thread `at` of `by`.
template <int DIM, int ROWS>
__device__ __forceinline__ void bring_queries(const TreeDev& a, const SlotWork& w, const Piece& p, char* sq, int at, int by) {
  constexpr int kChunks = DIM / 8;
  const int rows = min(ROWS, w.n * a.group - p.block * ROWS), c = at % kChunks, step = by / kChunks;
  int r = at / kChunks;
  const int x = p.block * ROWS + r;
  int node = x / a.group, g = x - node * a.group;
  const char* from = a.q + (int64_t)w.off * a.q_token_stride + (int64_t)(p.head * a.group) * a.q_head_stride + c * 16;
  for (; r < rows; r += step) {
    copy16(sq + (r >> 7) * (128 * DIM * 2) + (c >> 3) * 16384 + (r & 127) * 128 + (((c & 7) ^ (r & 7)) << 4), from + node * a.q_token_stride + g * a.q_head_stride);
    for (g += step; g >= a.group; g -= a.group) ++node;
  }
}

template <typename T> struct Weight;
template <> struct Weight<__nv_bfloat16> {
  static constexpr bool kBf16 = true;
  static constexpr float kShift = 0.0f, kSlack = 8.0f;
  static constexpr uint32_t kExp = 0x7F80u;
  static __device__ __forceinline__ uint32_t pack(float a, float b) {
    const __nv_bfloat162 h = __floats2bfloat162_rn(a, b);
    return *reinterpret_cast<const uint32_t*>(&h);
  }
  static __device__ __forceinline__ float widen(uint32_t bits) { return __uint_as_float(bits << 16); }
};
// fp16 weights are carried 2^11 times as large: a weight of 2^-25 of the largest would else be
// rounded to nothing, and a hundred thousand of them are not nothing
template <> struct Weight<__half> {
  static constexpr bool kBf16 = false;
  static constexpr float kShift = 11.0f, kSlack = 4.0f;  // 2^15 at most: fp16 ends at 65504
  static constexpr uint32_t kExp = 0x7C00u;
  static __device__ __forceinline__ uint32_t pack(float a, float b) {
    const __half2 h = __floats2half2_rn(a, b);
    return *reinterpret_cast<const uint32_t*>(&h);
  }
  static __device__ __forceinline__ float widen(uint32_t bits) {
    const __half h = __ushort_as_half((unsigned short)bits);
    return __half2float(h);
  }
};

// Among four neighbouring lanes: lane b gets part b of all four lanes' y (y[e]: that of lane e).
__device__ __forceinline__ void swap_words(uint32_t& low, uint32_t& high, bool up, int mask) {
  // the lane with the bit gives the lower of two, the other the upper
  const uint32_t got = __shfl_xor_sync(0xFFFFFFFFu, up ? low : high, mask);
  low = up ? got : low;
  high = up ? high : got;
}
__device__ __forceinline__ void transpose4(uint4 (&y)[4], int lane) {
#pragma unroll
  for (int s = 1; s < 4; s <<= 1) {
    const bool up = (lane & s) != 0;
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      if (e & s) continue;
      swap_words(y[e].x, y[e | s].x, up, s);
      swap_words(y[e].y, y[e | s].y, up, s);
      swap_words(y[e].z, y[e | s].z, up, s);
      swap_words(y[e].w, y[e | s].w, up, s);
    }
  }
}

// 2^x, but never nothing: what it weighs may be infinite, and a finite sum times this is nothing anyway
__device__ __forceinline__ float weight_of(float x) { return fmaxf(exp2_approx(x), 1.17549435e-38f); }

// Up to 128 slots, a warp on its own: four slots a lane, the units before each, and the units in all.
template <typename P>
__device__ __forceinline__ uint32_t add_up(const TreeDev& a, int ctas, SlotWork (&w)[4], uint32_t (&before)[4], uint32_t (&own)[4], int& extra) {
  const int lane = threadIdx.x & 31;
  uint32_t plain = 0;
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    w[i].n = 0;
    w[i].bad = false;
    if (i * 32 + lane < a.c.slots) w[i] = slot_work<P>(a, i * 32 + lane);
    else size_up<P>(a, w[i]);
    plain += (uint32_t)(Costs<P>(a, w[i], 0).head * a.c.heads);
  }
  extra = extra_units<P>(__reduce_add_sync(0xFFFFFFFFu, plain), ctas);
  uint32_t total = 0;
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    before[i] = own[i] = 0;
    if (i * 32 >= a.c.slots) continue;
    own[i] = (uint32_t)(Costs<P>(a, w[i], extra).head * a.c.heads);
    uint32_t x = own[i];
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const uint32_t y = __shfl_up_sync(0xFFFFFFFFu, x, o);
      if (lane >= o) x += y;
    }
    before[i] = total + x - own[i];
    total += __shfl_sync(0xFFFFFFFFu, x, 31);
  }
  return total;
}

template <typename T, int DIM, int MODE>
__global__ void __maxnreg__(152)
    tree_tiles_kernel(const __grid_constant__ CUtensorMap map_k, const __grid_constant__ CUtensorMap map_v, const TreeDev a) {
  using P = TilePlan<DIM, MODE>;
  using W = Weight<T>;
  constexpr int kKeys = P::kKeys, kRows = P::kRows, kRing = P::kSlots, kNT = kTileThreads;
  extern __shared__ __align__(1024) char smem[];
  char* sq = smem;
  char* ring = smem + P::kQBytes;
  float2* stat = reinterpret_cast<float2*>(ring + kRing * P::kTile);  // [2][128]
  float* handed = reinterpret_cast<float*>(stat + 256);               // [128] (kShare) the reference after the last tile
  uint64_t* bars = reinterpret_cast<uint64_t*>(handed + 128);
  uint64_t *full = bars, *empty = bars + kRing, *s_full = empty + kRing, *p_half = s_full + 2, *p_full = p_half + 2, *ref_set = p_full + 2 /* [2][4] */, *q_first = ref_set + 8, *q_full = q_first + 1, *q_empty = q_full + 1,
           *item_done = q_empty + 1, *sums_done = item_done + 1, *stat_full = sums_done + 1, *sums_free = stat_full + 1, *drain = sums_free + 1;
  unsigned long long* odd = reinterpret_cast<unsigned long long*>(drain + 1);  // [4] nodes whose values are not all finite: piece k's are in odd[k & 3]
  uint32_t* s_tmem = reinterpret_cast<uint32_t*>(odd + 4);
  volatile int* fail = reinterpret_cast<volatile int*>(s_tmem + 1);
  uint32_t* s_begin = s_tmem + 2;  // [2] first slot, units before it
  uint32_t* s_sums = s_tmem + 5;   // [12]
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, cta = blockIdx.x, ctas = gridDim.x;
  pdl_trigger();
  if (smem_addr(smem) & 1023u) {  // (the tiles' swizzle goes by the address)
    if (cta == 0 && tid == 0) raise_status(a.c.status, ARCS_ERR_CUDA);
    return;
  }

  // ---- where this CTA's units begin. Up to 128 slots every warp adds up on its own, which asks for no
  // barrier but the one behind the set-up; more are added up by the whole CTA, in the ring's memory.
  Walk<P> walk;
  uint32_t total = 0;
  const bool few = a.c.slots <= 128;
  if (warp == 9) {
    tmem_alloc(s_tmem, 512);
    if (lane == 0) {
      for (int i = 0; i < kRing; ++i) {
        mbar_init(&full[i], 1);
        mbar_init(&empty[i], 1);
      }
      for (int i = 0; i < 2; ++i) {
        mbar_init(&s_full[i], 1);
        mbar_init(&p_half[i], 4);
        mbar_init(&p_full[i], 4);
      }
      for (int i = 0; i < 4; ++i) odd[i] = 0;
      for (int i = 0; i < 8; ++i) mbar_init(&ref_set[i], 1);
      mbar_init(q_first, 8);
      mbar_init(q_full, 1);
      mbar_init(q_empty, 1);
      mbar_init(item_done, 1);
      mbar_init(sums_done, 1);
      mbar_init(stat_full, 8);
      mbar_init(sums_free, 8);
      mbar_init(drain, 1);
      *fail = 0;
      mbar_init_fence();
    }
    __syncwarp();
  }
  walk.s = -1;
  if (few) {
    SlotWork w[4];
    uint32_t before[4], own[4];
    total = add_up<P>(a, ctas, w, before, own, walk.extra);
    walk.u = first_unit(total, cta, ctas);
    walk.u1 = first_unit(total, cta + 1, ctas);
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      if (i * 32 >= a.c.slots) break;
      const unsigned hit = __ballot_sync(0xFFFFFFFFu, before[i] <= walk.u && walk.u < before[i] + own[i]);
      if (hit) {
        const int from = __ffs((int)hit) - 1;
        walk.s = i * 32 + from;
        walk.base = __shfl_sync(0xFFFFFFFFu, before[i], from);
        walk.w.off = __shfl_sync(0xFFFFFFFFu, w[i].off, from);
        walk.w.n = __shfl_sync(0xFFFFFFFFu, w[i].n, from);
        walk.w.len = __shfl_sync(0xFFFFFFFFu, w[i].len, from);
      }
      if (w[i].bad && cta == 0 && warp == 0) raise_status(a.c.status, ARCS_ERR_PAGE);
    }
    size_up<P>(a, walk.w);
  } else {
    uint32_t* pre = reinterpret_cast<uint32_t*>(ring);
    walk.extra = 0;
    for (int turn = 0; turn < 2; ++turn) {  // the plain total first, which decides `extra`
      total = 0;
      for (int s0 = 0; s0 < a.c.slots; s0 += kNT) {
        const int s = s0 + tid;
        uint32_t mine = 0;
        if (s < a.c.slots) {
          const SlotWork w = slot_work<P>(a, s);
          if (w.bad && cta == 0) raise_status(a.c.status, ARCS_ERR_PAGE);
          mine = (uint32_t)(Costs<P>(a, w, walk.extra).head * a.c.heads);
        }
        uint32_t x = mine;
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
          const uint32_t y = __shfl_up_sync(0xFFFFFFFFu, x, o);
          if (lane >= o) x += y;
        }
        if (lane == 31) s_sums[warp] = x;
        __syncthreads();
        uint32_t before = 0, all = 0;
        for (int i = 0; i < kNT / 32; ++i) {
          const uint32_t v = s_sums[i];
          if (i < warp) before += v;
          all += v;
        }
        if (s < a.c.slots) pre[s] = total + before + x - mine;
        total += all;
        __syncthreads();
      }
      if (turn == 0) walk.extra = extra_units<P>(total, ctas);
    }
    if (tid == 0) pre[a.c.slots] = total;
    __syncthreads();
    if (cta == 0) {
      for (int s = tid; s <= a.c.slots; s += kNT) a.prefix[s] = pre[s];
      if (tid == 0) a.prefix[a.c.slots + 1] = (uint32_t)walk.extra;
    }
    walk.u = first_unit(total, cta, ctas);
    walk.u1 = first_unit(total, cta + 1, ctas);
    for (int s = tid; s < a.c.slots; s += kNT)
      if (pre[s] <= walk.u && walk.u < pre[s + 1]) {
        s_begin[0] = (uint32_t)s;
        s_begin[1] = pre[s];
      }
    fence_proxy_async();
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = *s_tmem;
  if (walk.u == walk.u1) {  // nothing for this CTA
    if (warp == 9) tmem_free(tmem, 512);
    return;
  }
  if (!few) {
    walk.s = (int)s_begin[0];
    walk.base = s_begin[1];
    walk.w = slot_work<P>(a, walk.s);
  }
  Piece p;

  // (384 threads of 152 registers at the start; the softmax warps take what the other four need not hold)
  if (warp >= 8) {
    asm volatile("setmaxnreg.dec.sync.aligned.u32 56;");
    if (warp == 8 || warp == 10) {
      // ============================================== copies: keys (warp 8) and values (warp 10) of the pieces, in a ring that they fill in
      // the order in which the products ask for them. One warp alone, some 600 cycles a tile, could not
      // keep the memory busy with small pages.
      const bool is_k = warp == 8;
      const CUtensorMap* map = is_k ? &map_k : &map_v;
      constexpr int kSub = P::kSub, kPart = kKeys / kSub;  // (keys in a piece of a value tile)
      const int box = min(a.c.page_size, is_k ? kKeys : kPart);
      uint32_t rc0 = 0, last = 0;
      bool ok = true;
      while (ok && walk.next(a, p)) {
        const int n = p.t1 - p.t0, end = walk.w.len + walk.w.n;
        const int32_t* list = a.c.table + (int64_t)walk.s * a.c.max_pages;
        // the page that this lane copies of what begins at `place`
        auto page_of = [&](int place, int keys) {
          return lane * box < keys && place + lane * box < end ? list[(place + lane * box) >> a.c.page_shift] : 0;
        };
        const int keys = is_k ? kKeys : kPart, place0 = p.t0 * kKeys;
        int id_next = page_of(place0, keys), id = 0;
        for (int i = 0; ok && i < n * kSub; ++i) {
          const int j = i / kSub, h = i % kSub;
          const int place = place0 + (is_k ? j * kKeys : i * kPart);
          if (!is_k || h == 0) {
            id = id_next;
            if (i + 1 < n * kSub) id_next = page_of(place + keys, keys);
          }
          // (a key tile is asked for one step ahead of the value tile before it)
          const uint32_t entry = MODE == kPair ? 2 * j + !is_k : is_k ? max(0, 2 * j - 1) : min(2 * j + 2, 2 * n - 1), rc = rc0 + entry * kSub + h;
          const int slot = rc % kRing;
          if (!hold_warp(&empty[slot], ((rc / kRing) & 1u) ^ 1u, fail)) {
            ok = false;
            break;
          }
          const int boxes = (max(0, min(keys, end - place)) + box - 1) / box;
          if (lane == 0) mbar_expect_tx(&full[slot], (uint32_t)(boxes * box * (is_k ? DIM / kSub : DIM) * 2));
          if (lane < boxes) {
            int row = a.no_row;
            if (id >= 0 && id < a.c.n_pages) row = id * a.page_rows + p.head * a.head_rows + (place & (a.c.page_size - 1));
            else raise_status(a.c.status, ARCS_ERR_PAGE);
            const int y = a.by_row ? row : p.head, z = a.by_row ? 0 : row;
            char* dst = ring + slot * P::kTile + lane * box * 128;
            if (is_k) {
#pragma unroll
              for (int c = 0; c < DIM / 64 / kSub; ++c) tile_load3(dst + c * (kKeys * 128), map, (h * (DIM / 64 / kSub) + c) * 64, y, z, &full[slot]);
            } else {
#pragma unroll
              for (int c = 0; c < DIM / 64; ++c) tile_load3(dst + c * (kPart * 128), map, c * 64, y, z, &full[slot]);
            }
          }
          __syncwarp();
          last = rc + 1;
        }
        rc0 += 2 * n * kSub;
      }
      if (!ok && lane == 0)  // the copies in flight land before the CTA's memory goes to another
        for (uint32_t i = last > (uint32_t)kRing ? last - kRing : 0; i < last; ++i) mbar_wait(&full[i % kRing], (i / kRing) & 1u);
    } else if (warp == 9) {
      // ============================================== products
      {
        const uint32_t on = elect_one();
        constexpr uint32_t kScores = mma_desc(128, kKeys, W::kBf16, false), kValues = mma_desc(128, DIM, W::kBf16, true);
        uint32_t rc = 0, k = 0, turn = 0;  // (turn: a bit a score tile, the phase its barriers are in)
        bool ok = true;
        constexpr int kSub = P::kSub, kPart = kKeys / kSub;
        auto commit = [&](uint64_t* bar) { mma_commit(on, bar); };
        auto there = [&](uint32_t at) { return hold_warp(&full[at % kRing], (at / kRing) & 1u, fail); };
        // rows of queries `tile` x the keys from ring position `at` on; `last`: the slots are free afterwards
        auto scores = [&](int b, int tile, uint32_t at, bool last) {
          const uint32_t qa = smem_addr(sq) + tile * (128 * DIM * 2);
#pragma unroll
          for (int h = 0; h < kSub; ++h) {
            const uint32_t ka = smem_addr(ring) + (at + h) % kRing * P::kTile;
            if (kSub > 1 && !there(at + h)) return false;
#pragma unroll
            for (int i = 0; i < DIM / kSub / 16; ++i)
              mma_ss(on, tmem + b * P::kScore1, smem_desc(qa + h * (DIM / kSub / 64) * 16384 + (i / 4) * 16384 + (i % 4) * 32, 16, 1024),
                     smem_desc(ka + (i / 4) * (kKeys * 128) + (i % 4) * 32, 16, 1024), kScores, h + i > 0);
            if (kSub > 1) commit(&empty[(at + h) % kRing]);
          }
          commit(&s_full[b]);
          if (kSub == 1 && last) commit(&empty[at % kRing]);
          return true;
        };
        // weights of score tile b x the values from ring position `at` on: the first half of the keys as soon
        // as their weights are there
        auto values = [&](int b, int sums, uint32_t at, bool first, bool last) {
#pragma unroll
          for (int h = 0; h < 2; ++h) {
            const uint32_t slot = (at + (kSub > 1 ? h : 0)) % kRing, va = smem_addr(ring) + slot * P::kTile + (kSub > 1 ? 0 : h * (kKeys / 32) * 2048);
            if (kSub > 1 && !there(at + h)) return false;
            if (!hold_warp(h ? &p_full[b] : &p_half[b], (turn >> b) & 1u, fail)) return false;
            tc_fence_after();
#pragma unroll
            for (int i = 0; i < kKeys / 32; ++i)
              mma_ts(on, tmem + P::kSums + sums * DIM, tmem + b * P::kScore1 + (h * (kKeys / 32) + i) * 8, smem_desc(va + i * 2048, kPart * 128, 1024), kValues,
                     !(first && h + i == 0));
            if (kSub > 1 || (last && h == 1)) commit(&empty[slot]);
          }
          turn ^= 1u << b;
          return true;
        };
        while (ok && walk.next(a, p)) {
          const int n = p.t1 - p.t0;
          const bool two = MODE == kPair && walk.w.n * a.group - p.block * kRows > 128;
          ok = k == 0 ? hold_warp(q_first, 0, fail) : hold_warp(q_full, (k - 1u) & 1u, fail);
          tc_fence_after();
          uint32_t k_at = 0, v_at = 0;
          for (int j = 0; ok && j <= n; ++j) {
            // (the sums of the piece before have been read: asked before the first product into them)
            if (j == 1 && k > 0 && !(ok = hold_warp(sums_free, (k - 1u) & 1u, fail))) break;
            if (MODE == kPair) {
              // (what is copied is looked at before the weights are waited for, not between two products)
              if (j >= 1) {
                v_at = rc++;
                ok = there(v_at);
              }
              if (ok && j < n) {
                k_at = rc++;
                ok = there(k_at);
              }
              if (ok && j >= 1) ok = values(0, 0, v_at, j == 1, !two);
              if (ok && j < n) ok = scores(0, 0, k_at, !two);
              if (ok && two && j >= 1) ok = values(1, 1, v_at, j == 1, true);
              if (ok && two && j < n) ok = scores(1, 1, k_at, true);
              if (ok && j == n - 1) commit(q_empty);
            } else {
              if (j < n) {
                ok = (kSub > 1 || there(rc)) && scores(j & 1, 0, rc, true);
                rc += kSub;
                if (ok && j == n - 1) commit(q_empty);
              }
              if (ok && j >= 1) {
                const int b = (j - 1) & 1;
                ok = (kSub > 1 || there(rc)) && values(b, MODE == kSplit ? b : 0, rc, MODE == kSplit ? j <= 2 : j == 1, true);
                rc += kSub;
                if (MODE == kShare) commit(sums_done);
              }
            }
          }
          if (!ok) break;
          commit(item_done);
          ++k;
        }
        if (!ok) {
          commit(drain);
          if (lane == 0) mbar_wait(drain, 0);
        }
      }
      __syncwarp();
    } else {
      // ============================================== queries of the next piece, once the products have done with those of this one
      // (those of the first piece are brought by the softmax warps, which have nothing else to do then)
      uint32_t k = 0;
      while (walk.next(a, p)) {
        if (k > 0) {
          if (!hold_warp(q_empty, (k - 1u) & 1u, fail)) break;
          bring_queries<DIM, kRows>(a, walk.w, p, sq, lane, 32);
          copy16_wait();
          fence_proxy_async();
          arrive_warp(q_full);
        }
        ++k;
      }
    }
  } else {
    asm volatile("setmaxnreg.inc.sync.aligned.u32 200;");
    // ================================================ softmax: a thread a row
    const int grp = warp >> 2, row_t = tid & 127;
    const uint32_t lanes = tmem + ((uint32_t)(warp & 3) << 21);  // this warp's 32 lanes of tensor memory
    const int first_row = MODE == kPair ? grp * 128 : 0, my = first_row + row_t;
    const float sl2 = a.scale_log2;
    const uint64_t scale2 = pair_of(sl2, sl2);
    // ring position; phase of the score tile; pieces; (kShare) tiles of both groups, references that the other group has set
    uint32_t rc0 = 0, turn = 0, k = 0, done = 0, set = 0;
    bool ok = true;
    while (ok && walk.next(a, p)) {
      const int n = p.t1 - p.t0, len = walk.w.len, end = len + walk.w.n, off = walk.w.off;
      const int rows = min(kRows, walk.w.n * a.group - p.block * kRows);
      if (k == 0) {
        bring_queries<DIM, kRows>(a, walk.w, p, sq, tid, 256);
        copy16_wait();
        fence_proxy_async();
        arrive_warp(q_first);
      }
      const bool warp_live = first_row + (warp & 3) * 32 < rows, live = my < rows;
      const int x = p.block * kRows + (live ? my : 0), node = x / a.group, head_q = p.head * a.group + x - node * a.group;
      unsigned long long bits = 0;
      if (live) bits = a.mask ? a.mask[off + node] : (2ull << node) - 1ull;
      if (walk.w.n < 64) bits &= (1ull << walk.w.n) - 1ull;

      float m = -INFINITY, l = 0.0f;  // the reference of this row's weights (at most kSlack below the largest score, in log2), their sum
      const int mine = MODE == kPair && grp == 1 && rows <= 128 ? 0 : n;
      for (int j = MODE == kPair ? 0 : grp; j < mine; j += MODE == kPair ? 1 : 2) {
        const uint32_t score = lanes + grp * P::kScore1;
        if (!hold_warp(&s_full[grp], turn & 1u, fail)) {
          ok = false;
          break;
        }
        turn ^= 1u;
        tc_fence_after();
        const int p0 = (p.t0 + j) * kKeys;
        const bool tail = p0 + kKeys > len;
        if (warp_live) {
          uint32_t s[kKeys / 32][32];
#pragma unroll
          for (int i = 0; i < kKeys / 32; ++i) tmem_ld32(s[i], score + i * 32);
          tmem_wait_ld();
#pragma unroll
          for (int i = 0; i < kKeys / 32; ++i) tmem_use(s[i]);
          if (tail) {  // column c is place p0 + c: a settled token, a node (its bit decides), or nothing
#pragma unroll
            for (int i = 0; i < kKeys / 32; ++i) {
              const int rel = len - p0 - 32 * i;  // columns of these 32 that are settled tokens
              const uint32_t settled = rel >= 32 ? ~0u : rel <= 0 ? 0u : (1u << rel) - 1u;
              const uint32_t nodes = rel >= 32 ? 0u : rel >= 0 ? (uint32_t)(bits << rel) : rel > -64 ? (uint32_t)(bits >> -rel) : 0u;
              const uint32_t see = settled | nodes;
#pragma unroll
              for (int c = 0; c < 32; ++c)
                if (!((see >> c) & 1u)) s[i][c] = 0xFF800000u;
            }
          }
          float top[4] = {-INFINITY, -INFINITY, -INFINITY, -INFINITY};
#pragma unroll
          for (int i = 0; i < kKeys / 32; ++i)
#pragma unroll
            for (int c = 0; c < 32; c += 2) top[(c >> 1) & 3] = max3(top[(c >> 1) & 3], __uint_as_float(s[i][c]), __uint_as_float(s[i][c + 1]));
          const float most = max3(fmaxf(top[0], top[1]), top[2], top[3]) * sl2;
          // The reference moves only when a weight would pass 2^kSlack: the sums rarely have to be
          // brought down, and nothing is lost, because weights and sums carry the same factor.
          float before = m;
          if (MODE == kShare && j > 0) {
            if (!hold_warp(&ref_set[(grp ^ 1) * 4 + (warp & 3)], set++ & 1u, fail)) {
              ok = false;
              break;
            }
            before = handed[row_t];
          }
          const bool moves = live && most > before + W::kSlack;
          const float now = moves ? most : before;
          if (MODE == kShare) {
            handed[row_t] = now;
            arrive_warp(&ref_set[grp * 4 + (warp & 3)]);
          }
          if (MODE == kShare || __any_sync(0xFFFFFFFFu, moves)) {
            l *= now != m ? exp2_approx(m - now) : 1.0f;
            m = now;
          }
          if (j >= (MODE == kSplit ? 2 : 1) && __any_sync(0xFFFFFFFFu, moves)) {  // there are sums to bring down
            if (MODE == kShare) {
              if (!hold_warp(sums_done, (done + j - 1u) & 1u, fail)) {
                ok = false;
                break;
              }
              tc_fence_after();
            }
            const float f = moves ? exp2_approx(before - now) : 1.0f;
            const uint64_t f2 = pair_of(f, f);
            const uint32_t sums = lanes + P::kSums + (MODE == kShare ? 0 : grp * DIM);
#pragma unroll 1
            for (int i = 0; i < DIM / 16; ++i) {
              uint32_t o[16];
              tmem_ld16(o, sums + i * 16);
              tmem_wait_ld();
              tmem_use(o);
#pragma unroll
              for (int c = 0; c < 16; c += 2) {
                float y0, y1;
                pair_out(mul_pair(pair_of(__uint_as_float(o[c]), __uint_as_float(o[c + 1])), f2), y0, y1);
                o[c] = __float_as_uint(y0);
                o[c + 1] = __float_as_uint(y1);
              }
              tmem_st16(sums + i * 16, o);
            }
          }
          const float ref = W::kShift - (m == -INFINITY ? 0.0f : m);
          const uint64_t ref2 = pair_of(ref, ref);
          // The weights are rounded to 16 bits, once, because the product with the values takes both operands in one 16-bit
          // type; their sum is taken before that. It costs half a step of each weight: bf16 results are off by 2.3e-3 of
          // their length where the rounding of the result alone makes 1.7e-3, fp16 ones by 2.8e-4 and 2.1e-4. A second
          // product with what was rounded off would take it away, and double the time of the products with the values.
          uint64_t sum[2] = {0ull, 0ull};
#pragma unroll
          for (int i = 0; i < kKeys / 32; ++i) {
            uint32_t w[16];
#pragma unroll
            for (int c = 0; c < 32; c += 2) {
              float e0, e1;
              pair_out(fma_pair(pair_of(__uint_as_float(s[i][c]), __uint_as_float(s[i][c + 1])), scale2, ref2), e0, e1);
              e0 = exp2_approx(e0);
              e1 = exp2_approx(e1);
              sum[(c >> 1) & 1] = add_pair(sum[(c >> 1) & 1], pair_of(e0, e1));
              w[c >> 1] = W::pack(e0, e1);
            }
            tmem_st16(score + i * 16, w);
            if (i == kKeys / 64 - 1 && !tail) {  // half of the weights are there
              tmem_wait_st();
              tc_fence_before();
              arrive_warp(&p_half[grp]);
            }
          }
          float l0, l1;
          pair_out(add_pair(sum[0], sum[1]), l0, l1);
          l += l0 + l1;
          tmem_wait_st();
        } else if (!tail) {
          arrive_warp(&p_half[grp]);
        }
        if (tail && (MODE != kPair || grp == 0)) {
          // Values behind the last node are whatever the page holds, and 0 times NaN is NaN: they become
          // zeros. A node's value that is not finite, too: it is added at the end to the rows that see the node.
          constexpr int kSub = P::kSub, kPart = kKeys / kSub;
          const uint32_t at = rc0 + (MODE == kPair ? 2 * j + 1 : min(2 * j + 2, 2 * n - 1)) * kSub;
#pragma unroll
          for (int h = 0; h < kSub; ++h) ok = hold_warp(&full[(at + h) % kRing], ((at + h) / kRing) & 1u, fail) && ok;
          if (!ok) break;
          const int lo = max(0, len - p0);
          for (int i = row_t; i < (kKeys - lo) * (DIM / 8); i += 128) {
            const int r = lo + i / (DIM / 8), c = i % (DIM / 8);
            uint4* v = reinterpret_cast<uint4*>(ring + (at + r / kPart) % kRing * P::kTile + (c >> 3) * (kPart * 128) + r % kPart * 128 + (c & 7) * 16);
            if (p0 + r >= end) {
              *v = make_uint4(0, 0, 0, 0);
              continue;
            }
            uint4 y = *v;
            bool hit = false;
            auto clean = [&](uint32_t w) {
              if ((w & W::kExp) == W::kExp) { w &= 0xFFFF0000u; hit = true; }
              if ((w & (W::kExp << 16)) == (W::kExp << 16)) { w &= 0x0000FFFFu; hit = true; }
              return w;
            };
            y = make_uint4(clean(y.x), clean(y.y), clean(y.z), clean(y.w));
            if (hit) {
              *v = y;
              atomicOr(&odd[k & 3u], 1ull << (p0 + r - len));
            }
          }
          fence_proxy_async();
        }
        tc_fence_before();
        if (tail) arrive_warp(&p_half[grp]);
        arrive_warp(&p_full[grp]);
      }
      if (!ok) break;

      // ---- the end of the piece
      if (!hold_warp(item_done, k & 1u, fail)) {
        ok = false;
        break;
      }
      tc_fence_after();
      if (MODE != kPair) stat[grp * 128 + row_t] = make_float2(m, l);
      arrive_warp(stat_full);
      if (!hold_warp(stat_full, k & 1u, fail)) {
        ok = false;
        break;
      }
      float f0 = 1.0f, f1 = 0.0f;
      if (MODE != kPair) {
        const float2 s0 = stat[row_t], s1 = stat[128 + row_t];
        m = fmaxf(s0.x, s1.x);
        const float ref = m == -INFINITY ? 0.0f : m;
        f0 = weight_of(s0.x - ref);
        f1 = weight_of(s1.x - ref);
        l = f0 * s0.y + f1 * s1.y;
      }
      if (warp_live && mine > 0) {
        const bool whole = p.t0 == 0 && p.t1 == walk.w.tiles, sees = l > 0.0f || l != l;
        const float inv = !whole ? 1.0f : sees ? 1.0f / l : 0.0f;
        if (MODE != kSplit) f0 = 1.0f;  // (kShare: the sums are those of both groups)
        const uint64_t g0 = pair_of(f0 * inv, f0 * inv), g1 = pair_of(f1 * inv, f1 * inv);
        const int64_t block = (int64_t)cta * 2 + (p.t0 == 0);
        const unsigned long long fix = odd[k & 3u] & bits;
        constexpr int kCols = MODE == kPair ? DIM : DIM / 2;
        const int c0 = MODE == kPair ? 0 : grp * kCols;
        if (live && (MODE == kPair || grp == 0)) {
          if (!whole) a.part_stat[block * a.part_rows + my] = make_float2(m - W::kShift, l);
          else if (a.lse) a.lse[(int64_t)(off + node) * a.Hq + head_q] = sees ? (m - W::kShift + log2f(l)) * 0.6931471805599453f : -INFINITY;
        }
#pragma unroll 2
        for (int i = 0; i < kCols / 32; ++i) {
          const int col = c0 + i * 32;
          uint32_t o[32];
          tmem_ld32(o, lanes + P::kSums + (MODE == kPair ? grp * DIM : 0) + col);
          if (MODE == kSplit && n > 1) {  // (with one tile the other group has no sums)
            uint32_t o1[32];
            tmem_ld32(o1, lanes + P::kSums + DIM + col);
            tmem_wait_ld();
            tmem_use(o);
            tmem_use(o1);
#pragma unroll
            for (int c = 0; c < 32; c += 2) {
              float y0, y1;
              pair_out(fma_pair(pair_of(__uint_as_float(o1[c]), __uint_as_float(o1[c + 1])), g1, mul_pair(pair_of(__uint_as_float(o[c]), __uint_as_float(o[c + 1])), g0)), y0, y1);
              o[c] = __float_as_uint(y0);
              o[c + 1] = __float_as_uint(y1);
            }
          } else {
            tmem_wait_ld();
            tmem_use(o);
#pragma unroll
            for (int c = 0; c < 32; c += 2) {
              float y0, y1;
              pair_out(mul_pair(pair_of(__uint_as_float(o[c]), __uint_as_float(o[c + 1])), g0), y0, y1);
              o[c] = __float_as_uint(y0);
              o[c + 1] = __float_as_uint(y1);
            }
          }
          if (fix) {
            for (unsigned long long f = fix; f; f &= f - 1) {
              const int place = len + __ffsll((long long)f) - 1, pg = a.c.table[(int64_t)walk.s * a.c.max_pages + (place >> a.c.page_shift)];
              if (pg < 0 || pg >= a.c.n_pages) continue;
              const unsigned short* v =
                  reinterpret_cast<const unsigned short*>(a.c.v + pg * a.c.page_stride + p.head * a.c.head_stride + (place & (a.c.page_size - 1)) * a.c.token_stride) + col;
#pragma unroll
              for (int c = 0; c < 32; ++c) {
                const uint32_t y = v[c];
                if ((y & W::kExp) == W::kExp) o[c] = __float_as_uint(__uint_as_float(o[c]) + W::widen(y));
              }
            }
          }
          if (whole) {
            // Four lanes hand their rows' 16-byte parts to one another, so that a store writes 64 bytes of a row: one
            // that writes 16 bytes of 32 rows keeps the store path four times as long.
            uint4 y[4];
#pragma unroll
            for (int e = 0; e < 4; ++e) {
              uint32_t z[4];
#pragma unroll
              for (int f = 0; f < 4; ++f)
                z[f] = sees ? W::pack(__uint_as_float(o[8 * e + 2 * f]), __uint_as_float(o[8 * e + 2 * f + 1])) : 0u;
              y[e] = make_uint4(z[0], z[1], z[2], z[3]);
            }
            transpose4(y, lane);
            const int64_t row_at = (off + node) * a.out_token_stride + head_q * a.out_head_stride + col * 2;
#pragma unroll
            for (int e = 0; e < 4; ++e) {
              const int from = (lane & ~3) + e;
              const int64_t at = __shfl_sync(0xFFFFFFFFu, row_at, from);
              if (first_row + (warp & 3) * 32 + from < rows) *reinterpret_cast<uint4*>(a.out + at + (lane & 3) * 16) = y[e];
            }
          } else if (live) {
            float4* dst = a.part + (block * (DIM / 4) + col / 4) * a.part_rows + my;
#pragma unroll
            for (int c = 0; c < 32; c += 4)
              dst[(int64_t)(c / 4) * a.part_rows] = make_float4(__uint_as_float(o[c]), __uint_as_float(o[c + 1]), __uint_as_float(o[c + 2]), __uint_as_float(o[c + 3]));
          }
          __syncwarp();
        }
      }
      // (the other warps may be at work on piece k + 1 by now and set its bits; none is in piece k + 2 before this warp, too,
      // has arrived at the stat_full of k + 1, and none is still in piece k - 2)
      if (tid == 0) odd[(k + 2) & 3u] = 0;
      tc_fence_before();
      arrive_warp(sums_free);
      rc0 += 2 * n * P::kSub;
      done += n;
      if (MODE == kShare && warp_live && (n & 1) == grp) ++set;  // (the piece's last tile was the other group's: nobody asked for its reference)
      ++k;
    }
  }
  __syncthreads();
  if (tid == 0 && *fail) raise_status(a.c.status, ARCS_ERR_TIMEOUT);
  if (warp == 9) tmem_free(tmem, 512);
}

// The pieces of items that were cut, joined. FEW: few items of maybe a hundred pieces each; blockIdx.x is
// the item (slot, key head, block). Else many: every item that is cut begins in one CTA and goes on in the
// next, so blockIdx.x names the CTA in which it begins. A warp takes kCols x 4 columns of 2^row_bits rows
// (blockIdx.y): as the pieces lie, a lane a row, and where the rows are fewer than the lanes, these
// share a row's pieces (FEW: the four warps do, too). It asks for some pieces at a time, their statistics
// beside them: what bounds it is the latency of one such round, 1.7 us for pieces that other SMs have just
// written. Small enough
// (56 registers, 128 threads) to be on the SM, its way found, while the last pieces are still worked on, where the
// tiles leave it shared memory: with kSplit, and at dim 64 (195 KB of 228). With kPair at dim 128 and kShare the
// tiles take all of it, and a CTA of this kernel begins when one of theirs has left.
constexpr int kJoinThreads = 128;
template <int DIM, bool FEW>
struct JoinPlan {
  static constexpr int kCols = FEW ? 1 : 4;                   // of four values each
  static constexpr int kAtOnce = FEW ? 5 : 2;                 // pieces
  static constexpr int kParts = DIM / 4 / kCols / (FEW ? 1 : 4);  // CTAs for a group of rows
};
template <typename T, int DIM, int MODE, bool FEW>
__global__ void __launch_bounds__(kJoinThreads, 9) join_kernel(const TreeDev a, int ctas, int blocks, int row_bits) {
  using P = TilePlan<DIM, MODE>;
  using W = Weight<T>;
  using J = JoinPlan<DIM, FEW>;
  constexpr int kCols = J::kCols;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  uint32_t total = 0, base = 0, u = 0;
  int s = FEW ? (int)blockIdx.x / (a.c.heads * blocks) : -1, extra = 0;
  const bool few = FEW || a.c.slots <= 128;  // (few items are of few slots)
  if (few) {
    SlotWork w[4];
    uint32_t before[4], own[4];
    total = add_up<P>(a, ctas, w, before, own, extra);
    u = first_unit(total, (int)blockIdx.x + 1, ctas);
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const bool mine = FEW ? i * 32 + lane == s : before[i] <= u && u < before[i] + own[i];
      const unsigned hit = __ballot_sync(0xFFFFFFFFu, mine);
      if (hit) {
        s = i * 32 + __ffs((int)hit) - 1;
        base = __shfl_sync(0xFFFFFFFFu, before[i], __ffs((int)hit) - 1);
      }
    }
  } else {
    pdl_wait();
    total = __ldcg(a.prefix + a.c.slots);
    extra = (int)__ldcg(a.prefix + a.c.slots + 1);
    u = first_unit(total, (int)blockIdx.x + 1, ctas);
    int lo = 0, n = a.c.slots;  // the last slot with prefix <= u (those without units share theirs with the next)
    while (n > 1) {
      const int step = (n + 31) / 32, at = lo + lane * step;
      const unsigned b = __ballot_sync(0xFFFFFFFFu, at < lo + n && __ldcg(a.prefix + at) <= u);
      const int j = b ? 31 - __clz(b) : 0;
      n = min(step, lo + n - (lo + j * step));
      lo += j * step;
    }
    s = lo;
    base = __ldcg(a.prefix + s);
  }
  // (every CTA waits before it ends: what follows on the stream begins when this grid is done, and must not
  // find the tiles still at work)
  if (s < 0 || (!FEW && u >= total)) return pdl_wait();
  const SlotWork w = slot_work<P>(a, s);
  if (w.n == 0) return pdl_wait();
  const Costs<P> costs(a, w, extra);
  int x = (int)(u - base);
  if (FEW) {
    const int i = (int)blockIdx.x - s * a.c.heads * blocks, head = i / blocks;
    if (i - head * blocks >= w.blocks) return pdl_wait();
    x = head * costs.head + (i - head * blocks) * costs.first;
  }
  const Place at = place_of<P>(w, costs, base, x);
  const int head = at.head, block = at.block;
  const uint32_t tile0 = at.begins + (uint32_t)extra;  // where the item's first tile begins
  const int c0 = cta_of_unit(total, tile0, ctas), c1 = cta_of_unit(total, tile0 + (uint32_t)((w.tiles - 1) * at.cost), ctas);
  if (c0 == c1 || (!FEW && c0 != (int)blockIdx.x)) return pdl_wait();  // not cut, or cut before
  // CTA c0 + 32 i + lane has a tile of the item: bit `lane` of pieces[i] (with hardly more units than CTAs
  // some of them have none)
  unsigned pieces[(kCtas + 31) / 32];
#pragma unroll
  for (int i = 0; i < (kCtas + 31) / 32; ++i) {
    const int c = c0 + 32 * i + lane;
    bool has = c <= c1;
    if (has && total < (uint32_t)ctas * (P::kCost + 1)) {
      const uint32_t u0 = first_unit(total, c, ctas), u1 = first_unit(total, c + 1, ctas);
      const int from = max(0, (int)(u0 - tile0)), to = min((int)(u1 - tile0), w.tiles * at.cost);
      has = (from + at.cost - 1) / at.cost < (to + at.cost - 1) / at.cost;
    }
    pieces[i] = __ballot_sync(0xFFFFFFFFu, has);
  }
  const int rows = min(P::kRows, w.n * a.group - block * P::kRows);
  const int rr = ((int)blockIdx.y / J::kParts << row_bits) + (lane & ((1 << row_bits) - 1));
  const int share = FEW ? (lane >> row_bits) * 4 + warp : lane >> row_bits, shares = (32 >> row_bits) * (FEW ? 4 : 1);
  const int col = FEW ? (int)blockIdx.y % J::kParts : ((int)blockIdx.y % J::kParts * 4 + warp) * kCols;  // in steps of four values
  const bool live = rr < rows;
  if (few) pdl_wait();
  float m = -INFINITY, l = 0.0f, o[kCols][4];
#pragma unroll
  for (int d = 0; d < kCols; ++d) o[d][0] = o[d][1] = o[d][2] = o[d][3] = 0.0f;
  for (int b = c0 + share; b <= c1; b += J::kAtOnce * shares) {
    float4 y[J::kAtOnce][kCols];
    float2 st[J::kAtOnce];
#pragma unroll
    for (int i = 0; i < J::kAtOnce; ++i) {
      const int c = b + i * shares;
      unsigned word = pieces[0];
#pragma unroll
      for (int e = 1; e < (kCtas + 31) / 32; ++e)
        if ((c - c0) >> 5 == e) word = pieces[e];
      const bool there = live && c <= c1 && ((word >> ((c - c0) & 31)) & 1u);
      const int64_t blk = (int64_t)c * 2 + (c == c0);
      st[i] = make_float2(-INFINITY, 0.0f);
#pragma unroll
      for (int d = 0; d < kCols; ++d) y[i][d] = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
      if (there) {
        st[i] = __ldcg(a.part_stat + blk * a.part_rows + rr);
#pragma unroll
        for (int d = 0; d < kCols; ++d) y[i][d] = __ldcg(a.part + (blk * (DIM / 4) + col + d) * a.part_rows + rr);
      }
    }
    float top = m;
#pragma unroll
    for (int i = 0; i < J::kAtOnce; ++i) top = fmaxf(top, st[i].x);
    const float ref = top == -INFINITY ? 0.0f : top, f = weight_of(m - ref);
    m = top;
    l = f * l;
#pragma unroll
    for (int d = 0; d < kCols; ++d)
#pragma unroll
      for (int e = 0; e < 4; ++e) o[d][e] = f * o[d][e];
#pragma unroll
    for (int i = 0; i < J::kAtOnce; ++i) {
      const float wt = weight_of(st[i].x - ref);
      l += wt * st[i].y;
#pragma unroll
      for (int d = 0; d < kCols; ++d) {
        o[d][0] += wt * y[i][d].x;
        o[d][1] += wt * y[i][d].y;
        o[d][2] += wt * y[i][d].z;
        o[d][3] += wt * y[i][d].w;
      }
    }
  }
  for (int x = 16; x >= 1 << row_bits; x >>= 1) {  // the lanes' shares of a row
    const float top = fmaxf(m, __shfl_xor_sync(0xFFFFFFFFu, m, x)), ref = top == -INFINITY ? 0.0f : top, f = weight_of(m - ref);
    m = top;
    l = f * l;
    l += __shfl_xor_sync(0xFFFFFFFFu, l, x);
#pragma unroll
    for (int d = 0; d < kCols; ++d)
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        o[d][e] = f * o[d][e];
        o[d][e] += __shfl_xor_sync(0xFFFFFFFFu, o[d][e], x);
      }
  }
  if (FEW) {  // the warps'
    __shared__ float meet[3][6][32];
    if (warp > 0) {
      float* mine = &meet[warp - 1][0][lane];
      mine[0] = m;
      mine[32] = l;
#pragma unroll
      for (int e = 0; e < 4; ++e) mine[64 + 32 * e] = o[0][e];
    }
    __syncthreads();
    if (warp > 0) return;
    float top = m;
#pragma unroll
    for (int i = 0; i < 3; ++i) top = fmaxf(top, meet[i][0][lane]);
    const float ref = top == -INFINITY ? 0.0f : top, f = weight_of(m - ref);
    m = top;
    l = f * l;
#pragma unroll
    for (int e = 0; e < 4; ++e) o[0][e] = f * o[0][e];
#pragma unroll
    for (int i = 0; i < 3; ++i) {
      const float wt = weight_of(meet[i][0][lane] - ref);
      l += wt * meet[i][1][lane];
#pragma unroll
      for (int e = 0; e < 4; ++e) o[0][e] += wt * meet[i][2 + e][lane];
    }
  }
  if (!live || lane >> row_bits) return;
  const bool sees = l > 0.0f || l != l;
  const float inv = sees ? 1.0f / l : 0.0f;
  const int row = block * P::kRows + rr, node = row / a.group, h = head * a.group + row - node * a.group;
  char* dst = a.out + (w.off + node) * a.out_token_stride + h * a.out_head_stride + col * 8;
#pragma unroll
  for (int d = 0; d < kCols; ++d)
    *reinterpret_cast<uint2*>(dst + d * 8) = sees ? make_uint2(W::pack(o[d][0] * inv, o[d][1] * inv), W::pack(o[d][2] * inv, o[d][3] * inv)) : make_uint2(0u, 0u);
  if (a.lse && col == 0) a.lse[(int64_t)(w.off + node) * a.Hq + h] = sees ? (m + log2f(l)) * 0.6931471805599453f : -INFINITY;
}

}  // namespace arcs
