// Attention of every sequence's new tokens over the pages of its KV cache.
#include "attn_paged.cuh"

namespace b200 {

namespace {

constexpr float LOG2E = 1.4426950408889634f;

// One warp per (token, query head), one key at a time.
template <typename T, int D>
__global__ void __launch_bounds__(128) attn_paged_kernel(const __grid_constant__ PagedParams p) {
  constexpr int E = D / 32;
  const int lane = threadIdx.x & 31;
  const int64_t w = static_cast<int64_t>(blockIdx.x) * 4 + (threadIdx.x >> 5), n = w / p.Hq;
  const int h = static_cast<int>(w - n * p.Hq);
  pdl_trigger();
  pdl_wait();
  if (n >= p.N) return;
  int64_t lo = 0, hi = p.B;   // the sequence: the last one that starts at or before this token
  while (hi - lo > 1) {
    const int64_t mid = (lo + hi) / 2;
    if (__ldg(p.q_start + mid) <= n) lo = mid; else hi = mid;
  }
  const PagedSeq s = paged_seq(p, lo);
  if (n < s.first || n >= s.first + s.T) return;   // behind the last sequence
  const int64_t pos = s.n - s.T + (n - s.first);
  const int64_t j0 = p.window > 0 && pos - p.window + 1 > 0 ? pos - p.window + 1 : 0;
  float q[E], o[E], m = -INFINITY, l = 0.f;
  const T* qr = static_cast<const T*>(p.q) + n * p.qs[0] + h * p.qs[1] + lane * E;
  for (int e = 0; e < E; ++e) { q[e] = to_f32<T>(qr[e]) * (p.scale * LOG2E); o[e] = 0.f; }
  const int64_t head = static_cast<int64_t>(h / p.G) * p.ks[1] + lane * E;
  for (int64_t j = j0; j <= pos; ++j) {
    const int64_t page = __ldg(p.table + lo * p.table_stride + j / p.page_size);
    const bool there = page >= 0 && page < p.num_pages;
    const int64_t at = (there ? page : 0) * p.ks[0] + head + (j % p.page_size) * p.ks[2];
    float d = 0.f, v[E];
    for (int e = 0; e < E; ++e) {
      d += q[e] * (there ? to_f32<T>(static_cast<const T*>(p.k_pages)[at + e]) : 0.f);
      v[e] = there ? to_f32<T>(static_cast<const T*>(p.v_pages)[at + e]) : 0.f;
    }
    d = warp_sum(d);
    const float mn = fmaxf(m, d), c = exp2f(m - mn), w_ = exp2f(d - mn);
    for (int e = 0; e < E; ++e) o[e] = o[e] * c + w_ * v[e];
    l = l * c + w_;
    m = mn;
  }
  T* out = static_cast<T*>(p.out) + (n * p.Hq + h) * D + lane * E;
  for (int e = 0; e < E; ++e) out[e] = from_f32<T>(l > 0.f ? o[e] / l : 0.f);
}

}  // namespace
}  // namespace b200

using namespace b200;

extern "C" int64_t b200_attn_paged_workspace_bytes(int64_t max_q, int Hq, int Hkv, int D) {
  return 0;
}

extern "C" int b200_attn_paged(const void* q, const void* k_pages, const void* v_pages, void* out, const int32_t* q_start, const int32_t* kv_len,
                               const int32_t* page_table, int64_t B, int64_t n_tokens, int64_t max_q, int Hq, int Hkv, int D, int64_t num_pages,
                               int page_size, int64_t table_stride, const int64_t q_strides[2], const int64_t kv_strides[3], int64_t window, float scale,
                               int dtype, void* workspace, int64_t workspace_bytes, void* stream) {
  B200_CHECK_ARG(q && k_pages && v_pages && out && q_start && kv_len && page_table && q_strides && kv_strides && B >= 0 && n_tokens >= 0 && max_q >= 0 &&
                 Hq > 0 && Hkv > 0 && num_pages > 0 && table_stride > 0 && window >= 0, "b200_attn_paged: bad arguments");
  B200_CHECK_ARG(D == 64 || D == 128, "b200_attn_paged: head_dim %d not supported (64 and 128 only)", D);
  B200_CHECK_ARG(Hq % Hkv == 0 && Hq / Hkv <= 128, "b200_attn_paged: query heads per KV head must divide and be <= 128");
  B200_CHECK_ARG(page_size > 0 && page_size % 16 == 0, "b200_attn_paged: page size %d is not a multiple of 16", page_size);
  if (!(table_stride * page_size < (1ll << 31) && n_tokens < (1ll << 31) && B < (1ll << 31)))
    B200_FAIL(B200_ELIMIT, "b200_attn_paged: more than 2^31 - 1 tokens, sequences or keys of a sequence");
  bool ok = aligned16(q) && aligned16(k_pages) && aligned16(v_pages) && aligned16(out);
  PagedParams p;
  for (int i = 0; i < 2; ++i) { p.qs[i] = q_strides[i]; ok = ok && q_strides[i] % 8 == 0 && q_strides[i] >= 0; }
  for (int i = 0; i < 3; ++i) { p.ks[i] = kv_strides[i]; ok = ok && kv_strides[i] % 8 == 0 && kv_strides[i] >= 0; }
  if (!ok) B200_FAIL(B200_EALIGN, "b200_attn_paged: operands must be 16-byte aligned with strides multiple of 8");
  if (B == 0 || n_tokens == 0 || max_q == 0) return B200_OK;
  p.q = q; p.k_pages = k_pages; p.v_pages = v_pages; p.out = out; p.q_start = q_start; p.kv_len = kv_len; p.table = page_table;
  p.B = B; p.N = n_tokens; p.num_pages = num_pages; p.table_stride = table_stride; p.Hq = Hq; p.Hkv = Hkv; p.G = Hq / Hkv; p.page_size = page_size;
  p.window = window; p.scale = scale;
  const unsigned grid = static_cast<unsigned>(ceil_div(n_tokens * Hq, 4));
  B200_DISPATCH_HALF(dtype, T, {
    launch_pdl(D == 128 ? attn_paged_kernel<T, 128> : attn_paged_kernel<T, 64>, dim3(grid), dim3(128), 0, static_cast<cudaStream_t>(stream), p);
  });
  B200_CHECK_LAUNCH("attn_paged_kernel");
  return B200_OK;
}
