// The paged cache's argument block on the device, and what the calls over it share.
#pragma once
#include <cuda_fp16.h>

#include "common.cuh"
#include "plan.h"

namespace arcs {

constexpr int kMaxSlots = 4096;

struct CacheDev {
  char* k;   // pools, in bytes from here on: all strides below are in bytes
  char* v;
  int64_t layer_stride, page_stride, head_stride, token_stride;
  int32_t layers, n_pages, page_size, page_shift, heads, dim, slots, max_pages;
  int32_t* table;
  int32_t* used;
  int32_t* ref;
  int32_t* len;
  int32_t* status;
};

// null when the block is in order, else what is wrong with it
inline const char* cache_fault(const arcs_cache* c, bool needs_ref) {
  if (!c) return "no cache";
  if (!c->k || !c->v || !c->table || !c->used || !c->len || (needs_ref && !c->ref)) return "the cache lacks a pool or a list";
  if (c->dtype != ARCS_BF16 && c->dtype != ARCS_F16) return "the cache's dtype is neither bf16 nor fp16";
  if (c->dim != 64 && c->dim != 128 && c->dim != 256) return "the cache's dim is not 64, 128 or 256";
  if (c->page_size < 16 || c->page_size > 256 || (c->page_size & (c->page_size - 1))) return "the cache's page_size is not 16, 32, 64, 128 or 256";
  if (c->layers < 1 || c->n_pages < 1 || c->heads < 1 || c->heads > 1024 || c->max_pages < 1) return "a size of the cache is below 1, or heads above 1024";
  if (c->slots < 1 || c->slots > kMaxSlots) return "the cache's slots are not 1 .. 4096";
  if ((int64_t)c->max_pages * c->page_size > 0x7FFF0000ll) return "a slot of the cache could hold more than 2^31 tokens";
  if (((c->layer_stride | c->page_stride | c->head_stride | c->token_stride) & 7) || c->layer_stride < 0 || c->page_stride < 0 ||
      c->head_stride < c->dim || c->token_stride < c->dim || (c->layers > 1 && c->layer_stride < c->dim) || (c->n_pages > 1 && c->page_stride < c->dim))
    return "a stride of the cache is not a multiple of 8 elements, or below dim";
  if ((reinterpret_cast<uintptr_t>(c->k) | reinterpret_cast<uintptr_t>(c->v)) & 15) return "a pool of the cache is not 16-byte aligned";
  return nullptr;
}

inline CacheDev cache_dev(const arcs_cache* c) {
  CacheDev d;
  d.k = static_cast<char*>(c->k);
  d.v = static_cast<char*>(c->v);
  d.layer_stride = c->layer_stride * 2;
  d.page_stride = c->page_stride * 2;
  d.head_stride = c->head_stride * 2;
  d.token_stride = c->token_stride * 2;
  d.layers = c->layers;
  d.n_pages = c->n_pages;
  d.page_size = c->page_size;
  d.page_shift = __builtin_ctz((unsigned)c->page_size);
  d.heads = c->heads;
  d.dim = c->dim;
  d.slots = c->slots;
  d.max_pages = c->max_pages;
  d.table = c->table;
  d.used = c->used;
  d.ref = c->ref;
  d.len = c->len;
  d.status = c->status;
  return d;
}

inline int bad_argument(const char* call, const char* what) {
  snprintf(error_buffer(), 256, "%s: %s", call, what);
  return ARCS_ERR_ARG;
}

// a launch that may begin while the kernel before it on the stream still runs (it waits in pdl_wait)
template <typename... P, typename... A>
inline cudaError_t launch_behind(void (*kernel)(P...), dim3 grid, dim3 block, size_t smem, cudaStream_t st, A... args) {
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = grid;
  cfg.blockDim = block;
  cfg.dynamicSmemBytes = smem;
  cfg.stream = st;
  cudaLaunchAttribute at[1];
  at[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  at[0].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = at;
  cfg.numAttrs = 1;
  return cudaLaunchKernelEx(&cfg, kernel, P(args)...);
}

// The slot whose rows [off[s], off[s + 1]) hold row t, or -1; asked by a whole warp. Every round
// narrows the range 32-fold, so that 4096 slots take three trips to memory.
__device__ __forceinline__ int slot_of_row(const int32_t* __restrict__ off, int slots, int t) {
  const int lane = threadIdx.x & 31;
  int lo = 0, n = slots;  // the last s in [lo, lo + n) with off[s] <= t is looked for
  while (n > 1) {
    const int step = (n + 31) / 32, at = lo + lane * step;
    const bool reached = at < lo + n && __ldg(off + at) <= t;
    const unsigned b = __ballot_sync(0xFFFFFFFFu, reached);
    const int j = b ? 31 - __clz(b) : 0;
    n = min(step, lo + n - (lo + j * step));
    lo += j * step;
  }
  return __ldg(off + lo) <= t && t < __ldg(off + lo + 1) ? lo : -1;
}

}  // namespace arcs
