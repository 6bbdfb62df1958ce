// Attention of the nodes of drafted trees over a paged cache.
#include "tree_tiles.cuh"

namespace arcs {

// For pools whose rows no tensor map can name (strides that are not multiples of one another): one warp a
// row, a running maximum and sum over the places it sees, the values added up as they come. What bounds it is one
// trip to memory after the other for every place: one token over 4096 takes 2.6 ms (18 us on the tensor cores), 24
// nodes of 16 heads of 256 over 131071 tokens 153 ms (88 us).
template <typename T, int DIM>
__global__ void __launch_bounds__(128) tree_rows_kernel(const TreeDev a) {
  constexpr int kPer = DIM / 32;
  const int64_t row = (int64_t)blockIdx.x * 4 + (threadIdx.x >> 5);
  const int lane = threadIdx.x & 31;
  const int t = (int)(row / a.Hq), h = (int)(row % a.Hq);
  if (t >= a.T) return;
  const int s = slot_of_row(a.node_off, a.c.slots, t);
  if (s < 0) return;
  const int i = t - a.node_off[s], n = a.node_off[s + 1] - a.node_off[s], len = a.c.len[s], used = a.c.used[s];
  if (n > a.max_nodes || a.node_off[s + 1] > a.T || len < 0 || used < 0 || used > a.c.max_pages || (int64_t)len + n > ((int64_t)used << a.c.page_shift)) {
    if (lane == 0) raise_status(a.c.status, ARCS_ERR_PAGE);
    return;
  }
  const unsigned long long bits = a.mask ? a.mask[t] : (2ull << i) - 1ull;
  float q[kPer], o[kPer];
  const T* qp = reinterpret_cast<const T*>(a.q + t * a.q_token_stride + h * a.q_head_stride) + lane * kPer;
#pragma unroll
  for (int d = 0; d < kPer; ++d) {
    q[d] = (float)qp[d];
    o[d] = 0.0f;
  }
  float m = -INFINITY, l = 0.0f;
  const int32_t* list = a.c.table + (int64_t)s * a.c.max_pages;
  for (int p = 0; p < len + n; ++p) {
    if (p >= len && !((bits >> (p - len)) & 1ull)) continue;
    const int page = list[p >> a.c.page_shift];
    if (page < 0 || page >= a.c.n_pages) {
      if (lane == 0) raise_status(a.c.status, ARCS_ERR_PAGE);
      return;
    }
    const int64_t at = page * a.c.page_stride + (h / a.group) * a.c.head_stride + (p & (a.c.page_size - 1)) * a.c.token_stride;
    const T* k = reinterpret_cast<const T*>(a.c.k + at) + lane * kPer;
    const T* v = reinterpret_cast<const T*>(a.c.v + at) + lane * kPer;
    float x = 0.0f;
#pragma unroll
    for (int d = 0; d < kPer; ++d) x = fmaf(q[d], (float)k[d], x);
#pragma unroll
    for (int w = 16; w > 0; w >>= 1) x += __shfl_xor_sync(0xFFFFFFFFu, x, w);
    x *= a.scale_log2;
    if (x > m) {
      const float f = exp2f(m - x);
      l *= f;
#pragma unroll
      for (int d = 0; d < kPer; ++d) o[d] *= f;
      m = x;
    }
    const float w = x == -INFINITY ? 0.0f : exp2f(x - m);
    l += w;
#pragma unroll
    for (int d = 0; d < kPer; ++d) o[d] = fmaf(w, (float)v[d], o[d]);
  }
  T* op = reinterpret_cast<T*>(a.out + t * a.out_token_stride + h * a.out_head_stride) + lane * kPer;
#pragma unroll
  for (int d = 0; d < kPer; ++d) op[d] = (T)(l > 0.0f || l != l ? o[d] / l : 0.0f);
  if (a.lse && lane == 0) a.lse[(int64_t)t * a.Hq + h] = l > 0.0f || l != l ? (m + log2f(l)) * 0.6931471805599453f : -INFINITY;
}

}  // namespace arcs

namespace {

using namespace arcs;

typedef CUresult (*EncodeTiled)(CUtensorMap*, CUtensorMapDataType, cuuint32_t, void*, const cuuint64_t*, const cuuint64_t*, const cuuint32_t*, const cuuint32_t*,
                                CUtensorMapInterleave, CUtensorMapSwizzle, CUtensorMapL2promotion, CUtensorMapFloatOOBfill);
EncodeTiled encode_tiled() {
  static const EncodeTiled fn = [] {
    void* p = nullptr;
    cudaDriverEntryPointQueryResult found;
    if (cudaGetDriverEntryPoint("cuTensorMapEncodeTiled", &p, cudaEnableDefault, &found) != cudaSuccess || found != cudaDriverEntryPointSuccess) p = nullptr;
    return reinterpret_cast<EncodeTiled>(p);
  }();
  return fn;
}

// How a pool's rows lie: as rows `token` apart that pages and heads are whole numbers of, or, with a
// token's heads side by side, as such rows of heads. false: neither.
struct RowPlan {
  bool by_row;
  int64_t page_rows, head_rows, rows;
};
bool plan_rows(const arcs_cache* c, RowPlan* r) {
  const int64_t ts = c->token_stride, ps = c->n_pages > 1 ? c->page_stride : 0, hs = c->heads > 1 ? c->head_stride : 0;
  if (ps % ts) return false;
  r->page_rows = ps / ts;
  r->by_row = hs % ts == 0;
  r->head_rows = r->by_row ? hs / ts : 0;
  if (!r->by_row && (ts % hs || hs * c->heads > ts)) return false;
  r->rows = (c->n_pages - 1) * r->page_rows + (c->heads - 1) * r->head_rows + c->page_size;
  return r->rows < 0x7FFFFF00ll && ts * 2 < (1ll << 40);
}

bool make_map(CUtensorMap* map, const arcs_cache* c, const void* base, const RowPlan& r, int keys) {
  const int box = c->page_size < keys ? c->page_size : keys;
  const int64_t hs = c->heads > 1 ? c->head_stride : c->dim;
  const cuuint64_t dims[3] = {(cuuint64_t)c->dim, (cuuint64_t)(r.by_row ? r.rows : c->heads), (cuuint64_t)(r.by_row ? 1 : r.rows)};
  const cuuint64_t strides[2] = {(cuuint64_t)(r.by_row ? c->token_stride : hs) * 2, (cuuint64_t)c->token_stride * 2};
  const cuuint32_t boxes[3] = {64, (cuuint32_t)(r.by_row ? box : 1), (cuuint32_t)(r.by_row ? 1 : box)}, steps[3] = {1, 1, 1};
  return encode_tiled()(map, c->dtype == ARCS_BF16 ? CU_TENSOR_MAP_DATA_TYPE_BFLOAT16 : CU_TENSOR_MAP_DATA_TYPE_FLOAT16, 3, const_cast<void*>(base), dims, strides, boxes, steps,
                        CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}

int mode_of(int dim, int rows) { return dim == 256 ? kShare : rows > 128 ? kPair : kSplit; }
int rows_of(int mode) { return mode == kPair ? 256 : 128; }
// Units of cost that the tile kernel may have to count (in 31 bits, on the device): every slot as long as its list of pages.
// Below 2^63: 2^12 slots x 2^10 heads x 2^5 blocks x (2^24 tiles x 6 + 18).
int64_t most_units(const arcs_cache* c, int rows, int mode) {
  const bool pair = mode == kPair;
  const int64_t tiles = ((int64_t)c->max_pages * c->page_size + TilePlan<128, kPair>::kKeys - 1) / TilePlan<128, kPair>::kKeys;
  const int64_t items = (int64_t)c->slots * c->heads * ((rows + rows_of(mode) - 1) / rows_of(mode));
  return items * (tiles * (pair ? TilePlan<128, kPair>::kCost : TilePlan<128, kSplit>::kCost) + (pair ? TilePlan<128, kPair>::kItemCost : TilePlan<128, kSplit>::kItemCost));
}
size_t round16(size_t n) { return (n + 15) / 16 * 16; }

template <typename K>
cudaError_t ensure_carveout(K kernel, std::atomic<unsigned long long>& done) {
  int dev = 0;
  cudaError_t e = cudaGetDevice(&dev);
  if (e != cudaSuccess) return e;
  const unsigned long long bit = 1ull << (dev & 63);
  if (done.load(std::memory_order_acquire) & bit) return cudaSuccess;
  e = cudaFuncSetAttribute(kernel, cudaFuncAttributePreferredSharedMemoryCarveout, cudaSharedmemCarveoutMaxShared);
  if (e == cudaSuccess) done.fetch_or(bit, std::memory_order_release);
  return e;
}

template <typename T, int DIM, int MODE>
int launch_tiles(const CUtensorMap& mk, const CUtensorMap& mv, const TreeDev& a, cudaStream_t st) {
  using P = TilePlan<DIM, MODE>;
  static std::atomic<unsigned long long> attr_done{0}, room_done{0};
  cudaError_t e = ensure_dynamic_smem(tree_tiles_kernel<T, DIM, MODE>, P::kSmem, attr_done);
  // (all of the SM's memory to be shared memory, not as much as this kernel asks for: with kSplit, and at dim 64, join_kernel's CTA is to fit beside)
  if (e == cudaSuccess) e = ensure_carveout(tree_tiles_kernel<T, DIM, MODE>, room_done);
  if (e != cudaSuccess) return set_error(ARCS_ERR_CUDA, cudaGetErrorString(e));
  tree_tiles_kernel<T, DIM, MODE><<<kCtas, kTileThreads, P::kSmem, st>>>(mk, mv, a);
  if (int rc = check_launch("tree_attention")) return rc;
  const int blocks = (a.max_nodes * a.group + P::kRows - 1) / P::kRows;
  const int64_t items = (int64_t)a.c.slots * a.c.heads * blocks;
  int row_bits = 0;
  while (row_bits < 5 && 1 << row_bits < a.part_rows) ++row_bits;
  const unsigned groups = (unsigned)((a.part_rows + (1 << row_bits) - 1) >> row_bits);
  if (items <= kCtas / 2)
    launch_behind(join_kernel<T, DIM, MODE, true>, dim3((unsigned)items, groups * JoinPlan<DIM, true>::kParts), dim3(kJoinThreads), 0, st, a, kCtas, blocks, row_bits);
  else
    launch_behind(join_kernel<T, DIM, MODE, false>, dim3(kCtas - 1, groups * JoinPlan<DIM, false>::kParts), dim3(kJoinThreads), 0, st, a, kCtas, blocks, row_bits);
  return check_launch("tree_attention");
}

}  // namespace

extern "C" size_t arcs_tree_attention_workspace_bytes(int32_t slots, int32_t heads, int32_t Hq, int32_t dim, int32_t max_nodes) {
  if (slots < 1 || heads < 1 || Hq < heads || Hq % heads || Hq / heads > 64 || (dim != 64 && dim != 128 && dim != 256) || max_nodes < 1 || max_nodes > ARCS_TREE_MAX) return 0;
  const int rows = max_nodes * (Hq / heads), most = rows_of(mode_of(dim, rows));
  const size_t blocks = (size_t)kCtas * 2 * (rows < most ? rows : most);
  return round16(((size_t)slots + 2) * 4) + round16(blocks * 8) + blocks * dim * 4;
}

extern "C" int arcs_tree_attention(const arcs_tree_attention_args* g, void* stream) {
  if (int inj = fault_injected()) return inj;
  if (!g) return bad_argument("tree_attention", "no arguments");
  if (const char* f = cache_fault(g->cache, false)) return bad_argument("tree_attention", f);
  const arcs_cache* c = g->cache;
  if (g->layer < 0 || g->layer >= c->layers) return bad_argument("tree_attention", "no such layer");
  if (g->T < 0 || g->Hq < 1 || g->Hq % c->heads || g->Hq / c->heads > 64) return bad_argument("tree_attention", "T or Hq out of range, or Hq not a multiple of the key heads");
  if (g->max_nodes < 1 || g->max_nodes > ARCS_TREE_MAX) return bad_argument("tree_attention", "max_nodes is not 1 .. 64");
  if (!(g->scale > 0.0f) || g->scale * 1.4426950408889634f > 3.4028235e38f) return bad_argument("tree_attention", "scale is not a positive number");
  if (g->T == 0) return ARCS_OK;
  if (!g->q || !g->out || !g->node_off) return bad_argument("tree_attention", "a null pointer");
  if (((g->q_token_stride | g->q_head_stride | g->out_token_stride | g->out_head_stride) & 7) || g->q_token_stride < c->dim || g->q_head_stride < c->dim ||
      g->out_token_stride < c->dim || g->out_head_stride < c->dim)
    return bad_argument("tree_attention", "a stride is not a multiple of 8 elements, or below dim");
  if ((reinterpret_cast<uintptr_t>(g->q) | reinterpret_cast<uintptr_t>(g->out)) & 15) return bad_argument("tree_attention", "a tensor is not 16-byte aligned");
  RowPlan r;
  const bool tiled = plan_rows(c, &r);
  const int rows = g->max_nodes * (g->Hq / c->heads), mode = mode_of(c->dim, rows), most = rows_of(mode);
  if (tiled && most_units(c, rows, mode) > 0x7FFFFFFFll) return bad_argument("tree_attention", "slots x places x heads x nodes is too large");
  if (!g->workspace || g->workspace_bytes < arcs_tree_attention_workspace_bytes(c->slots, c->heads, g->Hq, c->dim, g->max_nodes) ||
      (reinterpret_cast<uintptr_t>(g->workspace) & 15))
    return set_error(ARCS_ERR_WORKSPACE, "tree_attention: workspace too small, or not 16-byte aligned");
  TreeDev a;
  a.c = cache_dev(c);
  a.c.k += g->layer * a.c.layer_stride;
  a.c.v += g->layer * a.c.layer_stride;
  a.q = static_cast<const char*>(g->q);
  a.out = static_cast<char*>(g->out);
  a.q_token_stride = g->q_token_stride * 2;
  a.q_head_stride = g->q_head_stride * 2;
  a.out_token_stride = g->out_token_stride * 2;
  a.out_head_stride = g->out_head_stride * 2;
  a.lse = g->lse;
  a.node_off = g->node_off;
  a.mask = reinterpret_cast<const unsigned long long*>(g->mask);
  a.T = g->T;
  a.Hq = g->Hq;
  a.group = g->Hq / c->heads;
  a.max_nodes = g->max_nodes;
  a.scale_log2 = g->scale * 1.4426950408889634f;
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  const int64_t all_rows = (int64_t)g->T * g->Hq;
  if (all_rows > 0x1FFFFFFF0ll) return bad_argument("tree_attention", "too many rows");

  if (tiled) {
    const int keys = 128, part = c->dim == 256 ? 64 : 128;  // (as in TilePlan)
    if (!encode_tiled()) return set_error(ARCS_ERR_CUDA, "tree_attention: the driver makes no tensor maps");
    CUtensorMap mk, mv;
    if (!make_map(&mk, c, a.c.k, r, keys) || !make_map(&mv, c, a.c.v, r, part)) return set_error(ARCS_ERR_CUDA, "tree_attention: no tensor map for these pools");
    a.by_row = r.by_row;
    a.page_rows = (int32_t)r.page_rows;
    a.head_rows = (int32_t)r.head_rows;
    a.no_row = (int32_t)r.rows;
    a.part_rows = rows < most ? rows : most;
    char* ws = static_cast<char*>(g->workspace);
    const size_t blocks = (size_t)kCtas * 2 * a.part_rows;
    a.prefix = reinterpret_cast<uint32_t*>(ws);
    a.part_stat = reinterpret_cast<float2*>(ws + round16(((size_t)c->slots + 2) * 4));
    a.part = reinterpret_cast<float4*>(ws + round16(((size_t)c->slots + 2) * 4) + round16(blocks * 8));
#define ARCS_LAUNCH(TYPE)                                                                \
  do {                                                                                   \
    if (c->dim == 256) return launch_tiles<TYPE, 256, kShare>(mk, mv, a, st);           \
    if (c->dim == 128 && mode == kPair) return launch_tiles<TYPE, 128, kPair>(mk, mv, a, st); \
    if (c->dim == 128) return launch_tiles<TYPE, 128, kSplit>(mk, mv, a, st);            \
    if (mode == kPair) return launch_tiles<TYPE, 64, kPair>(mk, mv, a, st);              \
    return launch_tiles<TYPE, 64, kSplit>(mk, mv, a, st);                                \
  } while (0)
    if (c->dtype == ARCS_BF16) ARCS_LAUNCH(__nv_bfloat16);
    else ARCS_LAUNCH(__half);
#undef ARCS_LAUNCH
  }
  const unsigned grid = (unsigned)((all_rows + 3) / 4);
#define ARCS_LAUNCH(TYPE)                                                       \
  do {                                                                          \
    if (c->dim == 64) tree_rows_kernel<TYPE, 64><<<grid, 128, 0, st>>>(a);      \
    else if (c->dim == 128) tree_rows_kernel<TYPE, 128><<<grid, 128, 0, st>>>(a); \
    else tree_rows_kernel<TYPE, 256><<<grid, 128, 0, st>>>(a);                  \
  } while (0)
  if (c->dtype == ARCS_BF16) ARCS_LAUNCH(__nv_bfloat16);
  else ARCS_LAUNCH(__half);
#undef ARCS_LAUNCH
  return check_launch("tree_attention");
}
