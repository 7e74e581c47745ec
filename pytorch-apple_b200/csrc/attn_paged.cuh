// Shared between the kernels of attention over a paged KV cache.
#pragma once
#include "common.cuh"

namespace b200 {

struct PagedParams {
  const void *q, *k_pages, *v_pages;
  void* out;                       // [token, Hq, D]
  const int32_t *q_start, *kv_len, *table;
  int64_t B, N, num_pages, table_stride;
  int64_t qs[2], ks[3];            // element strides: q over (token, head), pages over (page, head, row)
  int Hq, Hkv, G, page_size;
  int64_t window;                  // keys a token sees back from its own (0: all)
  float scale;
};

// A sequence's first token, how many it has and how many keys.  What the device arrays hold is cut to what the buffers hold, so that
// no value in them leads outside a buffer.
struct PagedSeq { int64_t first; int T; int64_t n; };
__device__ __forceinline__ PagedSeq paged_seq(const PagedParams& p, int64_t b) {
  int64_t lo = __ldg(p.q_start + b), hi = __ldg(p.q_start + b + 1), n = __ldg(p.kv_len + b);
  lo = lo < 0 ? 0 : lo > p.N ? p.N : lo;
  hi = hi < lo ? lo : hi > p.N ? p.N : hi;
  const int64_t room = p.table_stride * p.page_size;
  n = n < 0 ? 0 : n > room ? room : n;
  return {lo, static_cast<int>(hi - lo), n};
}

}  // namespace b200
