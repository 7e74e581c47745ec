// Keys and values of a step's new tokens -> pages of the KV cache, with the position rotation of queries and keys on the way:
//   x'[d] = x[d] cos[d] - x[d + D/2] sin[d],   x'[d + D/2] = x[d + D/2] cos[d + D/2] + x[d] sin[d + D/2]     (d < D/2)
// in fp32 with one rounding, to the activation type.  (The rotation of the static-cache path rounds both products too, because
// the unfused graph that it replaces does; this one replaces nothing, and the errors would be twice as large.)
//
// One thread per 8 dims of both halves of a (token, head): everything it reads it has read before it writes, so queries may be
// rotated in place.  64 tokens of 12 + 2 + 2 heads of 128: 2.0 us, all of it launch and one round trip to memory (0.1 us of bytes); 2048 tokens in fp16 with
// fp32 tables: 4.4 us for 18.9 MB (2.9 us at the 6.46 TB/s of a copy), where 64-bit divisions and a slot looked up ahead of the loads made 4.8.
#include "common.cuh"

namespace b200 {

namespace {

struct AppendParams {
  const void* x[3];      // q, k, v: [token, head, D], D contiguous
  int64_t xs[3][2];      // element strides over (token, head)
  const void *cos_t, *sin_t;
  void *q_out, *k_pages, *v_pages;
  const int64_t* slots;
  int64_t N, n_slots;
  int64_t ps[3];         // element strides of the pages over (page, head, row)
  int Hq, Hkv, D, page_size, table_dtype;
};

__device__ __forceinline__ void load_table(const void* t, int64_t i, int dtype, float (&f)[8]) {
  if (dtype == B200_F32) {
    const float4 a = __ldg(reinterpret_cast<const float4*>(static_cast<const float*>(t) + i)), b = __ldg(reinterpret_cast<const float4*>(static_cast<const float*>(t) + i) + 1);
    f[0] = a.x; f[1] = a.y; f[2] = a.z; f[3] = a.w; f[4] = b.x; f[5] = b.y; f[6] = b.z; f[7] = b.w;
  } else if (dtype == B200_BF16) {
    unpack8<__nv_bfloat16>(__ldg(reinterpret_cast<const uint4*>(static_cast<const __nv_bfloat16*>(t) + i)), f);
  } else {
    unpack8<__half>(__ldg(reinterpret_cast<const uint4*>(static_cast<const __half*>(t) + i)), f);
  }
}

template <typename T>
__global__ void __launch_bounds__(128) paged_append_kernel(const __grid_constant__ AppendParams p) {
  const int hp = p.D >> 4, H = p.Hq + 2 * p.Hkv;   // pairs of packs per head
  const int64_t gid = static_cast<int64_t>(blockIdx.x) * blockDim.x + threadIdx.x;
  int64_t n;
  int h, pk;
  if (gid >> 32 == 0) {   // (a division in 64 bits takes longer than all the rest of the arithmetic)
    const uint32_t row = static_cast<uint32_t>(gid) / static_cast<uint32_t>(hp), token = row / static_cast<uint32_t>(H);
    pk = static_cast<int>(static_cast<uint32_t>(gid) - row * hp);
    h = static_cast<int>(row - token * H);
    n = token;
  } else {
    const int64_t row = gid / hp;
    pk = static_cast<int>(gid - row * hp);
    n = row / H;
    h = static_cast<int>(row - n * H);
  }
  if (n >= p.N) return;
  const int which = h < p.Hq ? 0 : (h < p.Hq + p.Hkv ? 1 : 2);
  if (which == 1) h -= p.Hq;
  if (which == 2) h -= p.Hq + p.Hkv;
  pdl_wait();
  pdl_trigger();
  // all that is read is on its way at once
  const int64_t slot = which == 0 ? 0 : __ldg(p.slots + n);
  const uint4* src = reinterpret_cast<const uint4*>(static_cast<const T*>(p.x[which]) + n * p.xs[which][0] + h * p.xs[which][1]);
  uint4 lo = src[pk], hi = src[pk + hp];
  if (which != 2 && p.cos_t) {
    float a[8], b[8], c0[8], s0[8], c1[8], s1[8], o[8];
    const int64_t t = n * p.D + pk * 8;
    load_table(p.cos_t, t, p.table_dtype, c0);
    load_table(p.sin_t, t, p.table_dtype, s0);
    load_table(p.cos_t, t + (p.D >> 1), p.table_dtype, c1);
    load_table(p.sin_t, t + (p.D >> 1), p.table_dtype, s1);
    unpack8<T>(lo, a);
    unpack8<T>(hi, b);
#pragma unroll
    for (int k = 0; k < 8; ++k) o[k] = a[k] * c0[k] - b[k] * s0[k];
    lo = pack8<T>(o);
#pragma unroll
    for (int k = 0; k < 8; ++k) o[k] = b[k] * c1[k] + a[k] * s1[k];
    hi = pack8<T>(o);
  }
  T* dst;
  if (which == 0) {
    dst = static_cast<T*>(p.q_out) + (n * p.Hq + h) * p.D;
  } else {
    if (slot < 0 || slot >= p.n_slots) return;   // a row of padding
    const int64_t page = p.n_slots >> 32 == 0 ? static_cast<uint32_t>(slot) / static_cast<uint32_t>(p.page_size) : slot / p.page_size;
    dst = static_cast<T*>(which == 1 ? p.k_pages : p.v_pages) + page * p.ps[0] + h * p.ps[1] + (slot - page * p.page_size) * p.ps[2];
  }
  reinterpret_cast<uint4*>(dst)[pk] = lo;
  reinterpret_cast<uint4*>(dst)[pk + hp] = hi;
}

}  // namespace
}  // namespace b200

using namespace b200;

extern "C" int b200_paged_append(const b200_paged_append_args* a, void* stream) {
  B200_CHECK_ARG(a && a->k && a->v && a->k_pages && a->v_pages && a->slots && a->n_tokens >= 0 && a->Hq >= 0 && a->Hkv > 0 && a->num_pages > 0 &&
                 a->page_size > 0, "b200_paged_append: bad arguments");
  B200_CHECK_ARG(a->Hq == 0 || (a->q && a->q_out), "b200_paged_append: query heads without queries or a place for them");
  B200_CHECK_ARG(!a->cos_t == !a->sin_t, "b200_paged_append: cos and sin tables come together");
  B200_CHECK_ARG(a->D > 0 && a->D % 16 == 0, "b200_paged_append: head_dim %d is not a multiple of 16", a->D);
  if (a->cos_t && a->table_dtype != B200_F32 && a->table_dtype != a->dtype)
    B200_FAIL(B200_ENOTSUP, "b200_paged_append: tables are f32 or of the activation type (got dtype %d)", a->table_dtype);
  bool ok = aligned16(a->k) && aligned16(a->v) && aligned16(a->k_pages) && aligned16(a->v_pages) && aligned16(a->cos_t) && aligned16(a->sin_t);
  AppendParams p;
  p.x[0] = a->q; p.x[1] = a->k; p.x[2] = a->v;
  if (a->Hq > 0) ok = ok && aligned16(a->q) && aligned16(a->q_out);
  for (int i = 0; i < 2; ++i) {
    p.xs[0][i] = a->Hq > 0 ? a->q_strides[i] : 0; p.xs[1][i] = a->k_strides[i]; p.xs[2][i] = a->v_strides[i];
    ok = ok && p.xs[0][i] % 8 == 0 && p.xs[1][i] % 8 == 0 && p.xs[2][i] % 8 == 0;
  }
  const int64_t kv_len[3] = {a->num_pages, a->Hkv, a->page_size};
  for (int i = 0; i < 3; ++i) { p.ps[i] = a->kv_strides[i]; ok = ok && a->kv_strides[i] % 8 == 0 && (a->kv_strides[i] > 0 || kv_len[i] <= 1); }
  if (!ok) B200_FAIL(B200_EALIGN, "b200_paged_append: operands must be 16-byte aligned with strides multiple of 8, those of the pages positive");
  if (a->n_tokens == 0) return B200_OK;
  p.cos_t = a->cos_t; p.sin_t = a->sin_t; p.q_out = a->q_out; p.k_pages = a->k_pages; p.v_pages = a->v_pages; p.slots = a->slots;
  p.N = a->n_tokens; p.n_slots = a->num_pages * a->page_size; p.Hq = a->Hq; p.Hkv = a->Hkv; p.D = a->D; p.page_size = a->page_size;
  p.table_dtype = a->table_dtype;
  const int64_t blocks = ceil_div(a->n_tokens * (a->Hq + 2 * static_cast<int64_t>(a->Hkv)) * (a->D >> 4), 128);
  if (blocks >= (1ll << 31)) B200_FAIL(B200_ELIMIT, "b200_paged_append: too many tokens");
  B200_DISPATCH_HALF(a->dtype, T, { launch_pdl(paged_append_kernel<T>, dim3(static_cast<unsigned>(blocks)), dim3(128), 0, static_cast<cudaStream_t>(stream), p); });
  B200_CHECK_LAUNCH("paged_append_kernel");
  return B200_OK;
}
