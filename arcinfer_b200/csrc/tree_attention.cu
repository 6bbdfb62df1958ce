// Attention of the nodes of drafted trees over a paged cache.
#include "cache.cuh"

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
};

// One warp a row (a node and a query head): a running maximum and sum over the places it sees, the
// values added up as they come.
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

using namespace arcs;

extern "C" size_t arcs_tree_attention_workspace_bytes(int32_t slots, int32_t heads, int32_t Hq, int32_t dim, int32_t max_nodes) {
  if (slots < 1 || heads < 1 || Hq < heads || Hq % heads || (dim != 64 && dim != 128 && dim != 256) || max_nodes < 1 || max_nodes > ARCS_TREE_MAX) return 0;
  return 256;
}

extern "C" int arcs_tree_attention(const arcs_tree_attention_args* g, void* stream) {
  if (int inj = fault_injected()) return inj;
  if (!g) return bad_argument("tree_attention", "no arguments");
  if (const char* f = cache_fault(g->cache, false)) return bad_argument("tree_attention", f);
  const arcs_cache* c = g->cache;
  if (g->layer < 0 || g->layer >= c->layers) return bad_argument("tree_attention", "no such layer");
  if (g->T < 0 || g->Hq < 1 || g->Hq % c->heads || g->Hq / c->heads > 64) return bad_argument("tree_attention", "T or Hq out of range, or Hq not a multiple of the key heads");
  if (g->max_nodes < 1 || g->max_nodes > ARCS_TREE_MAX) return bad_argument("tree_attention", "max_nodes is not 1 .. 64");
  if (!(g->scale > 0.0f) || g->scale > 3e38f) return bad_argument("tree_attention", "scale is not a positive number");
  if (g->T == 0) return ARCS_OK;
  if (!g->q || !g->out || !g->node_off) return bad_argument("tree_attention", "a null pointer");
  if (((g->q_token_stride | g->q_head_stride | g->out_token_stride | g->out_head_stride) & 7) || g->q_token_stride < c->dim || g->q_head_stride < c->dim ||
      g->out_token_stride < c->dim || g->out_head_stride < c->dim)
    return bad_argument("tree_attention", "a stride is not a multiple of 8 elements, or below dim");
  if ((reinterpret_cast<uintptr_t>(g->q) | reinterpret_cast<uintptr_t>(g->out)) & 15) return bad_argument("tree_attention", "a tensor is not 16-byte aligned");
  if (!g->workspace || g->workspace_bytes < arcs_tree_attention_workspace_bytes(c->slots, c->heads, g->Hq, c->dim, g->max_nodes))
    return set_error(ARCS_ERR_WORKSPACE, "tree_attention: workspace too small");
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
  const int64_t rows = (int64_t)g->T * g->Hq;
  if (rows > 0x1FFFFFFF0ll) return bad_argument("tree_attention", "too many rows");
  const unsigned grid = (unsigned)((rows + 3) / 4);
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
