// The paged cache: room for more tokens, copies that share pages, pages given back, the kept nodes
// of a verified tree moved together, and the norm and rotation that bring queries and keys there.
#include "cache.cuh"

namespace arcs {

// ---------------------------------------------------------------- pages taken (reserve, fork)
// One CTA, because pages go out in order: slot after slot, the lowest free number first. (1) what
// every slot needs, and the running sum of it; (2) one walk over the pages' counts, 8192 at a time
// and no further than the last page needed: the r-th free page belongs to the slot whose stretch of
// the running sum r lies in; (3) the slots' lists. No list of free pages is kept, so none can
// go stale, and the same pages go out whatever was given back in which order before.
constexpr int kAllocThreads = 1024;

// (in 64 bits: 4096 slots may ask for more pages than an int counts)
__device__ __forceinline__ long long block_scan_exclusive(long long v, long long* warp_sums, long long* total) {
  const int lane = threadIdx.x & 31, w = threadIdx.x >> 5;
  long long x = v;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const long long y = __shfl_up_sync(0xFFFFFFFFu, x, o);
    if (lane >= o) x += y;
  }
  if (lane == 31) warp_sums[w] = x;
  __syncthreads();
  if (w == 0) {
    long long y = warp_sums[lane];
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const long long z = __shfl_up_sync(0xFFFFFFFFu, y, o);
      if (lane >= o) y += z;
    }
    warp_sums[lane] = y;
  }
  __syncthreads();
  *total = warp_sums[31];
  const long long before = (w ? warp_sums[w - 1] : 0) + x - v;
  __syncthreads();
  return before;
}

// `ask`: extra[] of reserve, parent[] of fork. done: fork's [slots], 1 where a copy was made.
template <bool FORK>
__global__ void __launch_bounds__(kAllocThreads) alloc_kernel(const CacheDev c, const int32_t* __restrict__ ask, int32_t* __restrict__ done) {
  __shared__ int pre[kMaxSlots + 1];   // pages that the slots before this one take (at most INT_MAX: more than there are)
  __shared__ int base[kMaxSlots];      // where in the slot's list the first new page goes; -1: nothing is done for the slot
  __shared__ long long warp_sums[32];
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  if (FORK) pdl_trigger();

  // (the first stretch of the pages' counts is on its way before anything else is known)
  const int w0 = warp * 256;
  int32_t count[8];
#pragma unroll
  for (int j = 0; j < 8; ++j) count[j] = w0 + j * 32 + lane < c.n_pages ? c.ref[w0 + j * 32 + lane] : 1;

  // what each slot needs: pre[s], and base[s]
  for (int s = tid; s < c.slots; s += kAllocThreads) {
    const int a = ask[s], used = c.used[s], len = c.len[s];
    int need = 0, at = -1;
    if (!FORK && a > 0) {
      if (used < 0 || used > c.max_pages || len < 0) {
        raise_status(c.status, ARCS_ERR_PAGE);
      } else {
        const int64_t want = ((int64_t)len + a + c.page_size - 1) >> c.page_shift;
        if (want > c.max_pages) raise_status(c.status, ARCS_ERR_FULL);
        else if (want > used) { need = (int)want - used; at = used; }
      }
    }
    if (FORK && a >= 0) {
      bool fine = a < c.slots && a != s && used == 0;
      if (fine) {
        const int from_len = c.len[a], from_used = c.used[a];
        fine = ask[a] < 0 && from_len >= 0 && from_used >= 0 && from_used <= c.max_pages && (int64_t)from_len <= ((int64_t)from_used << c.page_shift);
        if (fine) { at = from_len >> c.page_shift; need = (from_len & (c.page_size - 1)) != 0; }
      }
      if (!fine) raise_status(c.status, ARCS_ERR_PAGE);
    }
    pre[s] = need;
    base[s] = at;
  }
  __syncthreads();
  if (FORK) {  // the lists of pages are looked over by a warp each, before anything is promised
    for (int s = warp; s < c.slots; s += kAllocThreads / 32) {
      const int at = base[s], n = at + pre[s];
      if (at < 0) continue;
      const int32_t* from = c.table + (int64_t)ask[s] * c.max_pages;
      bool fine = true;
      for (int i = lane; i < n; i += 32) {
        const int p = from[i];
        fine = fine && p >= 0 && p < c.n_pages && c.ref[p] > 0;
      }
      if (!__all_sync(0xFFFFFFFFu, fine) && lane == 0) {
        base[s] = -1;
        pre[s] = 0;
        raise_status(c.status, ARCS_ERR_PAGE);
      }
    }
    __syncthreads();
  }
  long long asked = 0;
  for (int s0 = 0; s0 < c.slots; s0 += kAllocThreads) {
    const int s = s0 + tid;
    long long all;
    const long long before = block_scan_exclusive(s < c.slots ? pre[s] : 0, warp_sums, &all);
    if (s < c.slots) pre[s] = (int)min(asked + before, 0x7FFFFFFFll);
    asked += all;
  }
  const int sum = (int)min(asked, 0x7FFFFFFFll);
  if (tid == 0) pre[c.slots] = sum;
  __syncthreads();

  int found = 0;  // free pages seen so far
  for (int p0 = 0; p0 < c.n_pages && found < sum; p0 += kAllocThreads * 8) {
    unsigned b[8];
    int mine = 0;
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      const int p = p0 + w0 + j * 32 + lane;
      if (p0 > 0) count[j] = p < c.n_pages ? c.ref[p] : 1;
    }
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      b[j] = __ballot_sync(0xFFFFFFFFu, count[j] == 0);
      mine += __popc(b[j]);
    }
    long long all;
    int r0 = found + (int)block_scan_exclusive(lane == 0 ? mine : 0, warp_sums, &all);
    r0 = __shfl_sync(0xFFFFFFFFu, r0, 0);
    found += (int)all;
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      const int r = r0 + __popc(b[j] & ((1u << lane) - 1u));
      r0 += __popc(b[j]);
      if (!((b[j] >> lane) & 1u) || r >= sum) continue;
      int lo = 0, hi = c.slots;  // the last slot with pre[slot] <= r
      while (hi - lo > 1) {
        const int mid = (lo + hi) >> 1;
        if (pre[mid] <= r) lo = mid;
        else hi = mid;
      }
      const int p = p0 + w0 + j * 32 + lane;
      c.table[(int64_t)lo * c.max_pages + base[lo] + r - pre[lo]] = p;
      c.ref[p] = 1;
    }
  }
  __syncthreads();
  if (tid == 0 && found < sum) raise_status(c.status, ARCS_ERR_FULL);

  // the slots' lists: a warp each
  for (int s = warp; s < c.slots; s += kAllocThreads / 32) {
    const int at = base[s], need = pre[s + 1] - pre[s];
    int32_t* list = c.table + (int64_t)s * c.max_pages;
    bool ok = at >= 0;
    if (ok && need > 0 && pre[s + 1] > found) {  // the pages did not suffice: those this slot had been given go back
      for (int i = lane; i < found - pre[s]; i += 32) {
        c.ref[list[at + i]] = 0;
        list[at + i] = -1;
      }
      ok = false;
    }
    if (FORK) {
      if (ok) {
        const int32_t* from = c.table + (int64_t)ask[s] * c.max_pages;
        for (int i = lane; i < at; i += 32) {
          const int p = from[i];
          list[i] = p;
          atomicAdd(&c.ref[p], 1);
        }
        if (lane == 0) {
          c.used[s] = at + need;
          c.len[s] = c.len[ask[s]];
        }
      }
      if (lane == 0) done[s] = ok;
    } else if (ok && lane == 0) {
      c.used[s] = at + need;
    }
  }
}

// ---------------------------------------------------------------- fork: the rest of the last page
// A CTA takes one (layer, pool, head) of one copy: `rest` rows of dim values, 16 bytes a thread. The
// slots are the fast index of the grid, so that the copies of one parent read its rows at about the same
// time, and all but the first of them find them in the L2 cache.
__global__ void __launch_bounds__(256) fork_copy_kernel(const CacheDev c, const int32_t* __restrict__ parent, const int32_t* __restrict__ done) {
  pdl_wait();
  const int s = blockIdx.x;
  if (!done[s]) return;
  const int len = c.len[s], rest = len & (c.page_size - 1), last = len >> c.page_shift;
  if (rest == 0) return;
  const int from = c.table[(int64_t)parent[s] * c.max_pages + last], to = c.table[(int64_t)s * c.max_pages + last];
  const int h = blockIdx.y % c.heads, lv = blockIdx.y / c.heads;
  char* pool = ((lv & 1) ? c.v : c.k) + (lv >> 1) * c.layer_stride + h * c.head_stride;
  const char* src = pool + from * c.page_stride;
  char* dst = pool + to * c.page_stride;
  const int row = c.dim / 8, n = rest * row;  // 16-byte chunks
  const int shift = 31 - __clz(row);
  for (int i0 = threadIdx.x; i0 < n; i0 += 256 * 4) {
    uint4 x[4];
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const int i = i0 + j * 256;
      if (i < n) x[j] = *reinterpret_cast<const uint4*>(src + (i >> shift) * c.token_stride + (i & (row - 1)) * 16);
    }
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const int i = i0 + j * 256;
      if (i < n) *reinterpret_cast<uint4*>(dst + (i >> shift) * c.token_stride + (i & (row - 1)) * 16) = x[j];
    }
  }
}

// ---------------------------------------------------------------- free
__device__ __forceinline__ void give_back(const CacheDev& c, int32_t* list, int i) {
  const int p = list[i];
  if (p < 0 || p >= c.n_pages) {
    raise_status(c.status, ARCS_ERR_PAGE);
  } else if (atomicSub(&c.ref[p], 1) < 1) {  // nobody held it
    atomicAdd(&c.ref[p], 1);
    raise_status(c.status, ARCS_ERR_PAGE);
  }
  list[i] = -1;
}

__global__ void __launch_bounds__(256) free_kernel(const CacheDev c, const int32_t* __restrict__ which) {
  const int s = blockIdx.x * 8 + (threadIdx.x >> 5), lane = threadIdx.x & 31;
  if (s >= c.slots || which[s] == 0) return;
  const int used = c.used[s];
  if (used < 0 || used > c.max_pages) {
    if (lane == 0) raise_status(c.status, ARCS_ERR_PAGE);
    return;
  }
  for (int i = lane; i < used; i += 32) give_back(c, c.table + (int64_t)s * c.max_pages, i);
  if (lane == 0) {
    c.used[s] = 0;
    c.len[s] = 0;
  }
}

// ---------------------------------------------------------------- compact
// Two launches: the rows move, then the lists change. A slot that the first one refuses is marked in its
// `used` (a bit that no count has), because what it was refused for, a page with other holders, may
// look different once the second one gives pages back: every CTA of the first that reads the mark
// refuses too, and the second takes it off again.
constexpr int32_t kRefused = 1 << 30;

// Whether a slot's path can be followed; asked by a whole warp, the same answer in every lane. from, to:
// where the rows of the nodes lane and lane + 32 lie and go (bytes into a (layer, pool, head)); first: the
// first node that moves (kept: none does).
struct Path {
  int64_t from[2], to[2];
  int first;
};
template <bool HOLDERS>
__device__ __forceinline__ bool follow(const CacheDev& c, int s, int used, int len, int kept, const int32_t* __restrict__ path, int path_stride, Path& p) {
  const int lane = threadIdx.x & 31;
  bool fine = kept <= ARCS_TREE_MAX && kept <= path_stride && len >= 0 && used >= 0 && used <= c.max_pages && (int64_t)len <= ((int64_t)used << c.page_shift);
  p.first = kept;
  if (fine) {
    const int32_t* list = c.table + (int64_t)s * c.max_pages;
    int from[2] = {0, 0}, to[2] = {0, 0}, node[2] = {-1, -1}, before[2] = {-1, -1};
#pragma unroll
    for (int e = 0; e < 2; ++e) {
      const int i = lane + 32 * e;
      if (i < kept) {
        node[e] = path[i];
        if (i) before[e] = path[i - 1];
      }
    }
#pragma unroll
    for (int e = 0; e < 2; ++e) {
      const int i = lane + 32 * e;
      if (i >= kept) continue;
      // (ascending nodes have node >= i, so that the place len + i lies in the slot's pages, too; a list that
      // is not ascending is found out by some lane, and none reads outside)
      if (node[e] <= before[e] || node[e] < i || node[e] >= ARCS_TREE_MAX || (int64_t)len + node[e] >= ((int64_t)used << c.page_shift)) {
        fine = false;
        continue;
      }
      from[e] = list[(len + node[e]) >> c.page_shift];
      to[e] = list[(len + i) >> c.page_shift];
    }
#pragma unroll
    for (int e = 0; e < 2; ++e) {
      const int i = lane + 32 * e;
      if (i >= kept || !fine) continue;
      if (from[e] < 0 || from[e] >= c.n_pages || to[e] < 0 || to[e] >= c.n_pages) {
        fine = false;
        continue;
      }
      if (node[e] > i) {
        p.first = min(p.first, i);
        if (HOLDERS && c.ref[to[e]] != 1) fine = false;
      }
      p.from[e] = from[e] * c.page_stride + ((len + node[e]) & (c.page_size - 1)) * c.token_stride;
      p.to[e] = to[e] * c.page_stride + ((len + i) & (c.page_size - 1)) * c.token_stride;
    }
  }
  p.first = __reduce_min_sync(0xFFFFFFFFu, p.first);
  return __all_sync(0xFFFFFFFFu, fine);
}

// Rows move towards the front only (node >= its place), and a thread keeps to one 16-byte column of
// one (layer, pool, head) at a time: it reads up to eight rows before it writes them, in ascending order,
// so no row is written before it has been read. The way to the rows is three dependent trips to
// memory (path, pages, their holders), so a CTA takes as many columns as fill the machine twice
// over rather than one a thread. 64 slots x 8192 columns x 7 rows: 21.6 us, 5.4 TB/s.
__global__ void __launch_bounds__(256) compact_move_kernel(const CacheDev c, const int32_t* __restrict__ kept_, const int32_t* __restrict__ path_, int path_stride) {
  pdl_trigger();
  __shared__ int64_t from[ARCS_TREE_MAX], to[ARCS_TREE_MAX];
  __shared__ int s_first;
  const int s = blockIdx.y, tid = threadIdx.x;
  const int kept = kept_[s];
  if (tid < 32) {
    const int used = *(volatile int32_t*)(c.used + s), len = c.len[s];
    Path p;
    const bool fine = kept <= 0 || follow<true>(c, s, used, len, kept, path_ + (int64_t)s * path_stride, path_stride, p);
    if (!fine && blockIdx.x == 0 && tid == 0 && used >= 0 && used <= c.max_pages) c.used[s] = used | kRefused;
    if (fine && kept > 0)
#pragma unroll
      for (int e = 0; e < 2; ++e)
        if (tid + 32 * e < kept) {
          from[tid + 32 * e] = p.from[e];
          to[tid + 32 * e] = p.to[e];
        }
    if (tid == 0) s_first = fine && kept > 0 ? p.first : kept;
  }
  __syncthreads();
  const int first = s_first;
  if (first >= kept) return;
  const int row = c.dim / 8, cols = c.layers * 2 * c.heads * row;
  for (int col = blockIdx.x * 256 + tid; col < cols; col += gridDim.x * 256) {
    const int d = col & (row - 1), x = col / row, h = x % c.heads, lv = x / c.heads;
    char* pool = ((lv & 1) ? c.v : c.k) + (lv >> 1) * c.layer_stride + h * c.head_stride + d * 16;
    for (int i0 = first; i0 < kept; i0 += 8) {
      uint4 y[8];
#pragma unroll
      for (int j = 0; j < 8; ++j)
        if (i0 + j < kept) y[j] = *reinterpret_cast<const uint4*>(pool + from[i0 + j]);
#pragma unroll
      for (int j = 0; j < 8; ++j)
        if (i0 + j < kept) *reinterpret_cast<uint4*>(pool + to[i0 + j]) = y[j];
    }
  }
}

// (what it needs to know of the lists it finds out before it waits for the rows: the first launch changes
// nothing in them but the mark)
__global__ void __launch_bounds__(256) compact_lists_kernel(const CacheDev c, const int32_t* __restrict__ kept_, const int32_t* __restrict__ path_, int path_stride,
                                                            int32_t* len_out) {
  const int s = blockIdx.x * 8 + (threadIdx.x >> 5), lane = threadIdx.x & 31;
  if (s >= c.slots) return;
  const int kept = max(0, kept_[s]), len = c.len[s], seen = *(volatile int32_t*)(c.used + s);
  Path p;
  bool fine = follow<false>(c, s, seen & ~kRefused, len, kept, path_ + (int64_t)s * path_stride, path_stride, p);
  pdl_wait();
  const int used = *(volatile int32_t*)(c.used + s);
  fine = fine && used >= 0 && used <= c.max_pages;
  __syncwarp();
  if (!fine) {
    if (lane == 0) {
      if (used >= kRefused && used <= kRefused + c.max_pages) c.used[s] = used - kRefused;
      raise_status(c.status, ARCS_ERR_PAGE);
      len_out[s] = len;
    }
    return;
  }
  const int left = (len + kept + c.page_size - 1) >> c.page_shift;
  for (int i = left + lane; i < used; i += 32) give_back(c, c.table + (int64_t)s * c.max_pages, i);
  __syncwarp();
  if (lane == 0) {
    if (left < used) c.used[s] = left;
    len_out[s] = len + kept;
  }
}

// ---------------------------------------------------------------- append
struct AppendDev {
  CacheDev c;  // k and v: the layer's
  const char* q;
  const char* k;
  const char* v;
  char* q_out;
  int64_t q_stride, k_stride, v_stride, q_out_stride;  // bytes
  const float* q_weight;
  const float* k_weight;
  float eps;
  int32_t T, Hq, rot, interleaved;
  const double* inv_freq;
  const int32_t* pos;
  const int32_t* node_off;
};

template <typename T> struct Half2Of;
template <> struct Half2Of<__nv_bfloat16> {
  static __device__ __forceinline__ float2 widen(uint32_t w) { return __bfloat1622float2(*reinterpret_cast<__nv_bfloat162*>(&w)); }
  static __device__ __forceinline__ uint32_t pack(float a, float b) {
    const __nv_bfloat162 h = __floats2bfloat162_rn(a, b);
    return *reinterpret_cast<const uint32_t*>(&h);
  }
};
template <> struct Half2Of<__half> {
  static __device__ __forceinline__ float2 widen(uint32_t w) { return __half22float2(*reinterpret_cast<__half2*>(&w)); }
  static __device__ __forceinline__ uint32_t pack(float a, float b) {
    const __half2 h = __floats2half2_rn(a, b);
    return *reinterpret_cast<const uint32_t*>(&h);
  }
};

// A CTA takes ROWS rows (four where there are many: the way to a row's place, four dependent trips to memory,
// is what bounds a CTA with one). A head is DIM / 8 neighbouring lanes with twice four values each; a lane
// stays with a head for all rows, so that weights and addresses are found once, and its next head's rows
// are always asked for. Lane l < rot / 8 has the values 4 l .. and rot / 2 + 4 l .. (interleaved: 8 l ..), so that
// both of a pair are its own and its turns are 4 l .., the other lanes what is not rotated: with 16 bytes in a
// row instead, eight shuffles a head brought the pairs together, and 14,700 rows of 48 heads of 128 took
// 125 us. Meanwhile, at the start, a warp a row finds the place, and the others the turns of
// the rotation, once for all heads: in fp64, pos * inv_freq / 2 pi less its whole part, so that a
// position of any size leaves an angle exact to fp32. What bounds it is the memory, each value once in
// and once out, and hardly less the instructions.
constexpr int kAppendRows = 4;
template <typename T, int DIM, int ROWS>
__global__ void __launch_bounds__(256, ROWS == 1 ? 5 : 4) append_kernel(const AppendDev a) {
  __shared__ __align__(16) float2 turn[ROWS][DIM / 2];
  __shared__ int64_t s_at[ROWS];  // bytes into a head of the layer; -1: nowhere, -2: not even the query
  constexpr int kLanes = DIM / 8, kGroups = 256 / kLanes;
  const int t0 = blockIdx.x * ROWS, rows = min(ROWS, a.T - t0), tid = threadIdx.x;
  const int lane = tid % kLanes, all = a.Hq + 2 * a.c.heads, half = a.rot / 2;
  const bool turns_here = lane < a.rot / 8;
  const int e0 = a.interleaved ? 8 * lane : turns_here ? 4 * lane : a.rot + 8 * (lane - a.rot / 8), e1 = a.interleaved || !turns_here ? e0 + 4 : half + 4 * lane;
  auto load = [&](int g, uint4 (&x)[ROWS]) {
    const bool is_q = g < a.Hq, is_v = g >= a.Hq + a.c.heads;
    const int64_t stride = is_q ? a.q_stride : is_v ? a.v_stride : a.k_stride;
    const int h = is_q ? g : is_v ? g - a.Hq - a.c.heads : g - a.Hq;
    const char* src = (is_q ? a.q : is_v ? a.v : a.k) + t0 * stride + h * (DIM * 2);
#pragma unroll
    for (int r = 0; r < ROWS; ++r) {
      x[r] = make_uint4(0, 0, 0, 0);
      if (g < all && r < rows) {
        if (a.interleaved) {
          x[r] = *reinterpret_cast<const uint4*>(src + e0 * 2);
        } else {
          const uint2 lo = *reinterpret_cast<const uint2*>(src + e0 * 2), hi = *reinterpret_cast<const uint2*>(src + e1 * 2);
          x[r] = make_uint4(lo.x, lo.y, hi.x, hi.y);
        }
      }
      src += stride;
    }
  };
  uint4 ahead[ROWS];
  load(tid / kLanes, ahead);
  if (tid < 32 * ROWS) {
    const int r = tid / 32;
    if (r < rows) {
      const int t = t0 + r, s = slot_of_row(a.node_off, a.c.slots, t);
      if (tid % 32 == 0) {
        int64_t at = -2;
        if (s >= 0) {
          const int64_t place = (int64_t)a.c.len[s] + (t - a.node_off[s]), list = place >> a.c.page_shift;
          int page = -1;
          if (place >= 0 && list < a.c.used[s] && list < a.c.max_pages) page = a.c.table[(int64_t)s * a.c.max_pages + list];
          if (page < 0 || page >= a.c.n_pages) {
            at = -1;
            raise_status(a.c.status, ARCS_ERR_PAGE);
          } else {
            at = page * a.c.page_stride + (place & (a.c.page_size - 1)) * a.c.token_stride;
          }
        }
        s_at[r] = at;
      }
    }
  } else if (half > 0) {
    for (int i = tid - 32 * ROWS; i < rows * half; i += 256 - 32 * ROWS) {
      const int r = i / half, e = i - r * half;
      const double turns = (double)a.pos[t0 + r] * a.inv_freq[e] * 0.15915494309189533577;
      float sn, cs;
      sincospif((float)(2.0 * (turns - rint(turns))), &sn, &cs);
      turn[r][e] = make_float2(cs, sn);
    }
  }
  __syncthreads();
  for (int g0 = 0; g0 < all; g0 += kGroups) {
    const int g = g0 + tid / kLanes;
    const bool is_q = g < a.Hq, is_v = g >= a.Hq + a.c.heads, live = g < all;
    const int h = is_q ? g : is_v ? g - a.Hq - a.c.heads : g - a.Hq;
    uint4 x[ROWS];
#pragma unroll
    for (int r = 0; r < ROWS; ++r) x[r] = ahead[r];
    load(g + kGroups, ahead);
    const float* w = is_q ? a.q_weight : is_v ? nullptr : a.k_weight;
    const bool norms = a.q_weight || a.k_weight, copied = __all_sync(0xFFFFFFFFu, is_v || !live);
    float4 w0 = make_float4(1.0f, 1.0f, 1.0f, 1.0f), w1 = w0;
    if (w && live) {
      w0 = __ldg(reinterpret_cast<const float4*>(w + e0));
      w1 = __ldg(reinterpret_cast<const float4*>(w + e1));
    }
    char* dst = is_q ? a.q_out + t0 * a.q_out_stride + h * (DIM * 2) : (is_v ? a.c.v : a.c.k) + h * a.c.head_stride;
#pragma unroll
    for (int r = 0; r < ROWS; ++r) {
      if (r >= rows) break;
      if (!copied) {
        float y[8];
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          const float2 f = Half2Of<T>::widen(j == 0 ? x[r].x : j == 1 ? x[r].y : j == 2 ? x[r].z : x[r].w);
          y[2 * j] = f.x;
          y[2 * j + 1] = f.y;
        }
        if (norms) {
          float ss = 0.0f;
#pragma unroll
          for (int j = 0; j < 8; ++j) ss = fmaf(y[j], y[j], ss);
#pragma unroll
          for (int o = kLanes / 2; o > 0; o >>= 1) ss += __shfl_xor_sync(0xFFFFFFFFu, ss, o);
          const float n = w ? rsqrtf(ss * (1.0f / DIM) + a.eps) : 1.0f;
          y[0] *= n * w0.x;
          y[1] *= n * w0.y;
          y[2] *= n * w0.z;
          y[3] *= n * w0.w;
          y[4] *= n * w1.x;
          y[5] *= n * w1.y;
          y[6] *= n * w1.z;
          y[7] *= n * w1.w;
        }
        if (turns_here) {
          const float4 f0 = *reinterpret_cast<const float4*>(&turn[r][4 * lane]), f1 = *reinterpret_cast<const float4*>(&turn[r][4 * lane + 2]);
          auto rotate = [](float& u, float& v, float c, float s) {
            const float w = u * c - v * s;
            v = u * s + v * c;
            u = w;
          };
          if (a.interleaved) {
            rotate(y[0], y[1], f0.x, f0.y);
            rotate(y[2], y[3], f0.z, f0.w);
            rotate(y[4], y[5], f1.x, f1.y);
            rotate(y[6], y[7], f1.z, f1.w);
          } else {
            rotate(y[0], y[4], f0.x, f0.y);
            rotate(y[1], y[5], f0.z, f0.w);
            rotate(y[2], y[6], f1.x, f1.y);
            rotate(y[3], y[7], f1.z, f1.w);
          }
        }
        if (!is_v) x[r] = make_uint4(Half2Of<T>::pack(y[0], y[1]), Half2Of<T>::pack(y[2], y[3]), Half2Of<T>::pack(y[4], y[5]), Half2Of<T>::pack(y[6], y[7]));
      }
      if (live) {
        const int64_t at = s_at[r];
        if (at >= (is_q ? -1 : 0)) {
          char* to = dst + (is_q ? r * a.q_out_stride : at);
          if (a.interleaved) {
            *reinterpret_cast<uint4*>(to + e0 * 2) = x[r];
          } else {
            *reinterpret_cast<uint2*>(to + e0 * 2) = make_uint2(x[r].x, x[r].y);
            *reinterpret_cast<uint2*>(to + e1 * 2) = make_uint2(x[r].z, x[r].w);
          }
        }
      }
    }
  }
}

}  // namespace arcs

using namespace arcs;

extern "C" int arcs_cache_reserve(const arcs_cache* cache, const int32_t* extra, void* stream) {
  if (int inj = fault_injected()) return inj;
  if (const char* f = cache_fault(cache, true)) return bad_argument("cache_reserve", f);
  if (!extra) return bad_argument("cache_reserve", "no list of extra tokens");
  alloc_kernel<false><<<1, kAllocThreads, 0, static_cast<cudaStream_t>(stream)>>>(cache_dev(cache), extra, nullptr);
  return check_launch("cache_reserve");
}

extern "C" int arcs_cache_fork(const arcs_cache* cache, const int32_t* parent, int32_t* done, void* stream) {
  if (int inj = fault_injected()) return inj;
  if (const char* f = cache_fault(cache, true)) return bad_argument("cache_fork", f);
  if (!parent || !done) return bad_argument("cache_fork", "no list of parents, or none for what was done");
  if ((int64_t)cache->layers * 2 * cache->heads > 65535) return bad_argument("cache_fork", "layers x heads of the cache is above 32767");
  const CacheDev c = cache_dev(cache);
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  alloc_kernel<true><<<1, kAllocThreads, 0, st>>>(c, parent, done);
  if (int rc = check_launch("cache_fork")) return rc;
  const dim3 grid((unsigned)c.slots, (unsigned)(c.layers * 2 * c.heads));
  launch_behind(fork_copy_kernel, grid, dim3(256), 0, st, c, parent, done);
  return check_launch("cache_fork");
}

extern "C" int arcs_cache_free(const arcs_cache* cache, const int32_t* which, void* stream) {
  if (int inj = fault_injected()) return inj;
  if (const char* f = cache_fault(cache, true)) return bad_argument("cache_free", f);
  if (!which) return bad_argument("cache_free", "no list of slots");
  free_kernel<<<(unsigned)((cache->slots + 7) / 8), 256, 0, static_cast<cudaStream_t>(stream)>>>(cache_dev(cache), which);
  return check_launch("cache_free");
}

extern "C" int arcs_cache_compact(const arcs_cache* cache, const int32_t* kept, const int32_t* path, int32_t path_stride, int32_t* len_out, void* stream) {
  if (int inj = fault_injected()) return inj;
  if (const char* f = cache_fault(cache, true)) return bad_argument("cache_compact", f);
  if (!kept || !path || !len_out || path_stride < 1) return bad_argument("cache_compact", "no paths, or nowhere to write the lengths");
  const CacheDev c = cache_dev(cache);
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  const int64_t cols = (int64_t)c.layers * 2 * c.heads * (c.dim / 8);
  if (cols > 0x3FFFFFFFll) return bad_argument("cache_compact", "layers x heads x dim is too large");
  const int64_t most = (cols + 255) / 256, fill = (4 * kSmCount + c.slots - 1) / c.slots;
  compact_move_kernel<<<dim3((unsigned)(most < fill ? most : fill), (unsigned)c.slots), 256, 0, st>>>(c, kept, path, path_stride);
  if (int rc = check_launch("cache_compact")) return rc;
  launch_behind(compact_lists_kernel, dim3((unsigned)((c.slots + 7) / 8)), dim3(256), 0, st, c, kept, path, path_stride, len_out);
  return check_launch("cache_compact");
}

extern "C" int arcs_cache_append(const arcs_append_args* g, void* stream) {
  if (int inj = fault_injected()) return inj;
  if (!g) return bad_argument("cache_append", "no arguments");
  if (const char* f = cache_fault(g->cache, false)) return bad_argument("cache_append", f);
  const arcs_cache* c = g->cache;
  if (g->layer < 0 || g->layer >= c->layers) return bad_argument("cache_append", "no such layer");
  if (g->T < 0 || g->Hq < 1 || g->Hq > 65536) return bad_argument("cache_append", "T or Hq out of range");
  if (g->T == 0) return ARCS_OK;
  if (!g->q || !g->k || !g->v || !g->q_out || !g->pos || !g->node_off || (g->rot > 0 && !g->inv_freq)) return bad_argument("cache_append", "a null pointer");
  if (g->rot < 0 || g->rot > c->dim || g->rot % 16) return bad_argument("cache_append", "rot is not a multiple of 16 up to dim");
  const int64_t qrow = (int64_t)g->Hq * c->dim, krow = (int64_t)c->heads * c->dim;
  if (((g->q_stride | g->k_stride | g->v_stride | g->q_out_stride) & 7) || g->q_stride < qrow || g->q_out_stride < qrow || g->k_stride < krow || g->v_stride < krow)
    return bad_argument("cache_append", "a stride is not a multiple of 8 elements, or shorter than a row");
  if ((reinterpret_cast<uintptr_t>(g->q) | reinterpret_cast<uintptr_t>(g->k) | reinterpret_cast<uintptr_t>(g->v) | reinterpret_cast<uintptr_t>(g->q_out) |
       reinterpret_cast<uintptr_t>(g->q_weight) | reinterpret_cast<uintptr_t>(g->k_weight)) & 15)
    return bad_argument("cache_append", "a tensor is not 16-byte aligned");
  if (!(g->eps >= 0.0f)) return bad_argument("cache_append", "eps is negative");
  AppendDev a;
  a.c = cache_dev(c);
  a.c.k += g->layer * a.c.layer_stride;
  a.c.v += g->layer * a.c.layer_stride;
  a.q = static_cast<const char*>(g->q);
  a.k = static_cast<const char*>(g->k);
  a.v = static_cast<const char*>(g->v);
  a.q_out = static_cast<char*>(g->q_out);
  a.q_stride = g->q_stride * 2;
  a.k_stride = g->k_stride * 2;
  a.v_stride = g->v_stride * 2;
  a.q_out_stride = g->q_out_stride * 2;
  a.q_weight = g->q_weight;
  a.k_weight = g->k_weight;
  a.eps = g->eps;
  a.T = g->T;
  a.Hq = g->Hq;
  a.rot = g->rot;
  a.interleaved = g->interleaved;
  a.inv_freq = g->inv_freq;
  a.pos = g->pos;
  a.node_off = g->node_off;
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  // (four rows a CTA where all SMs have their four CTAs of four rows one and a half times over: of 48 heads of 128, 500 rows took 6.2 us with one and 8.8 with
  // four, 2400 rows 18.6 and 19.2, 5000 rows 37.9 and 34.9, 14,700 rows 102 and 83)
  const bool many = g->T > kSmCount * 4 * kAppendRows * 3 / 2;
  const unsigned grid = (unsigned)(many ? (g->T + kAppendRows - 1) / kAppendRows : g->T);
#define ARCS_ROWS(TYPE, D)                                                                \
  do {                                                                                    \
    if (many) append_kernel<TYPE, D, kAppendRows><<<grid, 256, 0, st>>>(a);               \
    else append_kernel<TYPE, D, 1><<<grid, 256, 0, st>>>(a);                              \
  } while (0)
#define ARCS_LAUNCH(TYPE)                        \
  do {                                           \
    if (c->dim == 64) ARCS_ROWS(TYPE, 64);       \
    else if (c->dim == 128) ARCS_ROWS(TYPE, 128); \
    else ARCS_ROWS(TYPE, 256);                   \
  } while (0)
  if (c->dtype == ARCS_BF16) ARCS_LAUNCH(__nv_bfloat16);
  else ARCS_LAUNCH(__half);
#undef ARCS_LAUNCH
#undef ARCS_ROWS
  return check_launch("cache_append");
}
