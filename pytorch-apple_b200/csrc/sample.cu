// Drawing one token per row of logits: temperature, top-k, top-p, min-p, and a given random number.
//
// With z the row, m its largest element and T the temperature, a token weighs w = exp((z - m) / T).  In the order "larger first, of equal
// ones the lower index first" top-k keeps the first k tokens, top-p of those the ones before which less than top_p of their sum lies (the
// first always), min-p what weighs at least min_p.  The token drawn is the first one, by index, at which the running sum of what is kept
// passes u times the whole sum.
//
// Weights are whole numbers in units of 2^-40 (their sums over a row stay below 2^62), good to about 2^-31 of themselves: integer sums
// do not depend on the order of the additions, so the same row gives the same token however it is dealt to blocks, and a sum over
// 150 000 tokens is as exact as its terms (in fp32 a boundary between two tokens would move by 2^-24 of the sum, more than a
// rare token is wide).  Thresholds are found on the logits themselves, never on weights.
//
// A row belongs to the CTAs of a cluster, each with a contiguous range of columns; what they find out they tell one another through
// distributed shared memory.
#include "common.cuh"
#include "tc5.cuh"

namespace b200 {

namespace {

using u64 = unsigned long long;
constexpr int ST = 512, SW = ST / 32;        // threads and warps of a CTA
constexpr int MAX_CTAS = 8;                  // of a row
constexpr int64_t MAX_COLS = 1 << 22;        // sums of weights stay below 2^62
constexpr u64 ONE = 1ull << 40;              // weight of the row's maximum

struct SampleParams {
  const void* logits;
  int64_t* out;
  int64_t row_stride;
  const float *temperature, *top_p, *min_p, *uniform;
  const int32_t* top_k;
  int cols, seg;   // columns of the row and of a CTA's range
};

// Keys order like the logits they come from: equal keys, equal values (-0 counts as 0); NaN comes last, like -infinity.
__device__ __forceinline__ uint32_t key_of(float x) {
  if (x != x) return 0;
  const uint32_t b = __float_as_uint(x + 0.f);
  return b & 0x80000000u ? ~b : b | 0x80000000u;
}
constexpr uint32_t KEY_NEG_INF = 0x007fffffu;   // key_of(-infinity)

// exp((z - m) / T) = 2^-t, t = (m - z) log2(e) / T, by the table method (P. T. P. Tang, 1989): t to 32 binary places, 2^-(i / 256) from a table for
// the first eight, a cubic for the rest (its next term is below 2^-38).  The difference and its product with log2(e) / T are carried as
// pairs of fp32 numbers: a rounding of t = 30 alone would be 2^-20 of the weight.
struct Weigher {
  float m, c_hi, c_lo;
  const uint32_t* table;   // 2^31 2^-(i / 256)
  __device__ __forceinline__ u64 operator()(float z) const {
    if (z == m) return ONE;
    const float dh = m - z, bv = m - dh, dl = (m - (dh + bv)) + (bv - z);
    const float p = __fmul_rn(dh, c_hi);
    if (!(p < 60.f)) return 0;   // (a NaN or an infinite difference as well)
    const float e = fmaf(dh, c_hi, -p) + fmaf(dh, c_lo, dl * c_hi);
    const float ip = floorf(p);
    int64_t t = (static_cast<int64_t>(ip) << 32) + static_cast<int64_t>(__float2uint_rz((p - ip) * 4294967296.f)) + static_cast<int64_t>(__float2int_rn(e * 4294967296.f));
    t = t < 0 ? 0 : t;
    const uint32_t f = static_cast<uint32_t>(t);
    const float a = static_cast<float>(f & 0xffffffu) * (0.6931471805599453f / 4294967296.f);
    const float q = a - a * a * (0.5f - a * (1.f / 6.f));   // 1 - 2^-r
    const uint32_t tab = table[f >> 24];
    const uint32_t w = tab - static_cast<uint32_t>((static_cast<u64>(tab) * __float2uint_rn(q * 4294967296.f) + 0x80000000ull) >> 32);
    return (static_cast<u64>(w) << 9) >> static_cast<int>(t >> 32);
  }
};

struct Shared {
  uint32_t table[256];
  u64 part[SW];
  u64 total;
  u64 told[2][MAX_CTAS];   // values of all CTAs of the row, two exchanges deep
};

// A thread's share of the CTA's columns: warp w has a contiguous range, 256 columns at a time, eight per lane.
template <typename T> struct Row {
  const T* x;
  int begin, end;   // of this warp
  bool vec;
  __device__ __forceinline__ void load(int c, float (&f)[8]) const {   // columns c .. c + 7; those past the end as NaN
    if (vec && c + 8 <= end) {
      if constexpr (sizeof(T) == 2) {
        unpack8<T>(__ldg(reinterpret_cast<const uint4*>(x + c)), f);
      } else {
        const float4 a = __ldg(reinterpret_cast<const float4*>(x + c)), b = __ldg(reinterpret_cast<const float4*>(x + c) + 1);
        f[0] = a.x; f[1] = a.y; f[2] = a.z; f[3] = a.w; f[4] = b.x; f[5] = b.y; f[6] = b.z; f[7] = b.w;
      }
    } else {
#pragma unroll
      for (int k = 0; k < 8; ++k) f[k] = c + k < end ? to_f32<T>(x[c + k]) : __uint_as_float(0x7fffffffu);
    }
  }
  template <typename F> __device__ __forceinline__ void each(F&& f) const {
    for (int c = begin + (threadIdx.x & 31) * 8; c < end; c += 256) {
      float v[8];
      load(c, v);
#pragma unroll
      for (int k = 0; k < 8; ++k) f(v[k], c + k);
    }
  }
};

__device__ __forceinline__ u64 warp_add(u64 v) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
  return v;
}
__device__ __forceinline__ u64 warp_top(u64 v) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) {
    const u64 w = __shfl_xor_sync(0xffffffffu, v, o);
    v = w > v ? w : v;
  }
  return v;
}

// Sum or maximum over all threads of the row, known to all of them.  sh.told holds the CTAs' values afterwards, in slot `turn`.
template <bool TOP> __device__ u64 row_reduce(u64 v, Shared& sh, int ctas, int& turn) {
  v = TOP ? warp_top(v) : warp_add(v);
  if ((threadIdx.x & 31) == 0) sh.part[threadIdx.x >> 5] = v;
  __syncthreads();
  if (threadIdx.x < 32) {
    u64 s = threadIdx.x < SW ? sh.part[threadIdx.x] : 0;
    s = TOP ? warp_top(s) : warp_add(s);
    if (ctas == 1) {
      if (threadIdx.x == 0) sh.told[turn][0] = s;
    } else if (static_cast<int>(threadIdx.x) < ctas) {
      const uint32_t to = tc5::map_to_rank(tc5::smem_addr(&sh.told[turn][tc5::cluster_ctarank()]), threadIdx.x);
      asm volatile("st.shared::cluster.u64 [%0], %1;" ::"r"(to), "l"(s) : "memory");
    }
  }
  if (ctas == 1) __syncthreads(); else tc5::cluster_sync();
  u64 r = 0;
  for (int i = 0; i < ctas; ++i) r = TOP ? (sh.told[turn][i] > r ? sh.told[turn][i] : r) : r + sh.told[turn][i];
  turn ^= 1;
  return r;
}

template <typename T>
__global__ void __launch_bounds__(ST) sample_rows_kernel(const __grid_constant__ SampleParams p) {
  __shared__ Shared sh;
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, ctas = gridDim.x, rank = blockIdx.x;
  const int64_t r = blockIdx.y;
  int turn = 0;
  if (threadIdx.x < 256) sh.table[threadIdx.x] = static_cast<uint32_t>(exp2(-static_cast<double>(threadIdx.x) / 256.) * 2147483648. + 0.5);
  pdl_trigger();
  if (ctas > 1) tc5::cluster_sync();   // every CTA of the row runs before anyone writes into a peer
  pdl_wait();
  const T* x = static_cast<const T*>(p.logits) + r * p.row_stride;
  const int c0 = min(p.cols, rank * p.seg), c1 = min(p.cols, c0 + p.seg);
  const int span = (((c1 - c0 + SW - 1) / SW) + 255) & ~255;   // columns of a warp
  Row<T> row;
  row.x = x;
  row.begin = min(c1, c0 + warp * span);
  row.end = min(c1, row.begin + span);
  row.vec = (reinterpret_cast<uintptr_t>(x) & 15u) == 0;

  // ---- the maximum, and of equal ones the lowest index ----
  u64 best = 0;
  row.each([&](float z, int c) {
    const u64 v = static_cast<u64>(key_of(z)) << 32 | static_cast<uint32_t>(~c);
    if (v > best && c < row.end) best = v;
  });
  best = row_reduce<true>(best, sh, ctas, turn);
  const uint32_t top = static_cast<uint32_t>(best >> 32);
  const int first = static_cast<int>(~static_cast<uint32_t>(best));
  const float T_ = p.temperature ? __ldg(p.temperature + r) : 1.f;
  if (!(T_ > 0.f) || top <= KEY_NEG_INF) {   // greedy; a row without any weight gives its first token
    if (rank == 0 && threadIdx.x == 0) p.out[r] = top <= KEY_NEG_INF ? 0 : first;
    return;
  }
  const double c = 1.4426950408889634074 / static_cast<double>(T_);
  Weigher weight;
  weight.m = __uint_as_float(top & 0x80000000u ? top & 0x7fffffffu : ~top);
  weight.c_hi = static_cast<float>(c);
  weight.c_lo = static_cast<float>(c - static_cast<double>(weight.c_hi));
  weight.table = sh.table;

  // What is kept: keys above `cut`, and of those equal to it the indices up to `last`
  uint32_t cut = 0;
  int last = p.cols;
  // the (need)th lowest index among the columns whose key is `cut`
  auto index_limit = [&](u64 need) {
    int at = 0;
#pragma unroll 1
    for (int bit = 1 << 21; bit > 0; bit >>= 1) {
      const int next = at | bit;
      u64 n = 0;
      row.each([&](float z, int i) { n += (i < next && i < last + 1 && key_of(z) == cut && i < row.end) ? 1 : 0; });
      if (row_reduce<false>(n, sh, ctas, turn) < need) at = next;
    }
    return at;
  };

  const int k = p.top_k ? __ldg(p.top_k + r) : 0;
  if (k > 0 && k < p.cols) {
#pragma unroll 1
    for (uint32_t bit = 0x80000000u; bit > 0; bit >>= 1) {
      u64 n = 0;
      row.each([&](float z, int i) { n += (i < row.end && key_of(z) >= (cut | bit)) ? 1 : 0; });
      if (row_reduce<false>(n, sh, ctas, turn) >= static_cast<u64>(k)) cut |= bit;
    }
    u64 above = 0;
    row.each([&](float z, int i) { above += (i < row.end && key_of(z) > cut) ? 1 : 0; });
    above = row_reduce<false>(above, sh, ctas, turn);
    last = index_limit(static_cast<u64>(k) - above);
  }
  const float tp = p.top_p ? __ldg(p.top_p + r) : 1.f;
  if (tp < 1.f) {
    auto mass_from = [&](uint32_t from) {   // of what is kept so far, with keys of at least `from`
      u64 s = 0;
      row.each([&](float z, int i) {
        const uint32_t key = key_of(z);
        if (i < row.end && key >= from && (key > cut || (key == cut && i <= last))) s += weight(z);
      });
      return row_reduce<false>(s, sh, ctas, turn);
    };
    const double limit = fmax(static_cast<double>(tp) * static_cast<double>(mass_from(0)), 0.5);
    uint32_t at = 0;
#pragma unroll 1
    for (uint32_t bit = 0x80000000u; bit > 0; bit >>= 1)
      if (static_cast<double>(mass_from(at | bit)) >= limit) at |= bit;
    const u64 above = at == 0xffffffffu ? 0 : mass_from(at + 1);
    if (at != cut) { cut = at; last = p.cols; }
    const u64 w = weight(__uint_as_float(at & 0x80000000u ? at & 0x7fffffffu : ~at));
    last = min(last, index_limit(static_cast<u64>(ceil((limit - static_cast<double>(above)) / static_cast<double>(w)))));
  }
  const float mp = p.min_p ? __ldg(p.min_p + r) : 0.f;
  const u64 least = mp > 0.f ? static_cast<u64>(ceil(static_cast<double>(fminf(mp, 1.f)) * static_cast<double>(ONE))) : 0;

  // ---- the draw: sums of the warps' ranges, then the range in which the running sum passes the target ----
  auto kept = [&](float z, int i) -> u64 {
    const uint32_t key = key_of(z);
    if (i >= row.end || key < cut || (key == cut && i > last)) return 0;
    const u64 w = weight(z);
    return w >= least ? w : 0;
  };
  u64 mine = 0;
  row.each([&](float z, int i) { mine += kept(z, i); });
  mine = warp_add(mine);
  const int slot = turn;
  const u64 total = row_reduce<false>(lane == 0 ? mine : 0, sh, ctas, turn);
  const double d = static_cast<double>(p.uniform ? __ldg(p.uniform + r) : 0.f) * static_cast<double>(total);
  u64 target = d > 0. ? (d < static_cast<double>(total) ? static_cast<u64>(d) : total - 1) : 0;
  target = target < total ? target : total - 1;
  u64 before = 0;
  for (int i = 0; i < rank; ++i) before += sh.told[slot][i];
  for (int i = 0; i < warp; ++i) before += sh.part[i];
  if (target < before || target >= before + mine) return;
  for (int c = row.begin + lane * 8; ; c += 256) {   // (the whole warp goes round together)
    float v[8];
    u64 w[8], s = 0;
    if (c < row.end) row.load(c, v);
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      w[e] = c < row.end ? kept(v[e], c + e) : 0;
      s += w[e];
    }
    u64 upto = s;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const u64 t = __shfl_up_sync(0xffffffffu, upto, o);
      if (lane >= o) upto += t;
    }
    const unsigned passed = __ballot_sync(0xffffffffu, before + upto > target);
    if (passed) {
      if (lane == __ffs(passed) - 1) {
        u64 run = before + upto - s;
        int e = 0;
        while (e < 7 && run + w[e] <= target) run += w[e++];
        p.out[r] = c + e;
      }
      return;
    }
    before += __shfl_sync(0xffffffffu, upto, 31);
  }
}

}  // namespace
}  // namespace b200

using namespace b200;

extern "C" int b200_sample_rows(const void* logits, int64_t* out, int64_t rows, int64_t cols, int64_t row_stride, const float* temperature,
                                const int32_t* top_k, const float* top_p, const float* min_p, const float* uniform, int dtype, void* stream) {
  B200_CHECK_ARG(logits && out && uniform && rows >= 0 && cols > 0 && row_stride >= 0, "b200_sample_rows: bad arguments");
  if (cols > MAX_COLS || rows > 65535) B200_FAIL(B200_ELIMIT, "b200_sample_rows: more than %lld columns or 65535 rows", (long long)MAX_COLS);
  if (rows == 0) return B200_OK;
  SampleParams p;
  p.logits = logits; p.out = out; p.row_stride = row_stride; p.temperature = temperature; p.top_k = top_k; p.top_p = top_p; p.min_p = min_p;
  p.uniform = uniform; p.cols = static_cast<int>(cols);
  int ctas = 1;
  while (ctas < MAX_CTAS && 2 * ctas * rows <= 148 && cols > 4096 * ctas) ctas *= 2;
  p.seg = static_cast<int>(ceil_div(ceil_div(cols, ctas), 256) * 256);
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(static_cast<unsigned>(ctas), static_cast<unsigned>(rows));
  cfg.blockDim = dim3(ST);
  cfg.stream = static_cast<cudaStream_t>(stream);
  cudaLaunchAttribute attrs[2];
  int n = 0;
  attrs[n].id = cudaLaunchAttributeClusterDimension;
  attrs[n].val.clusterDim.x = static_cast<unsigned>(ctas);
  attrs[n].val.clusterDim.y = 1;
  attrs[n++].val.clusterDim.z = 1;
  if (pdl_enabled()) {
    attrs[n].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attrs[n++].val.programmaticStreamSerializationAllowed = 1;
  }
  cfg.attrs = attrs;
  cfg.numAttrs = n;
  B200_DISPATCH_FLOAT(dtype, T, { cudaLaunchKernelEx(&cfg, sample_rows_kernel<T>, p); });
  B200_CHECK_LAUNCH("sample_rows_kernel");
  return B200_OK;
}
