// Drawing one token per row of logits: temperature, top-k, top-p, min-p, and a given random number.
//
// With z the row, m its largest element and T the temperature, a token weighs w = exp((z - m) / T).  In the order "larger first, of equal
// ones the lower index first" top-k keeps the first k tokens, top-p of those the ones before which less than top_p of their sum lies (the
// first always), min-p what weighs at least min_p.  The token drawn is the first one, by index, at which the running sum of what is kept
// passes u times the whole sum.
//
// Weights are whole numbers in units of 2^-40 (their sums over a row are at most 2^62): integer sums do not depend on the order of the additions,
// so the same row gives the same token however it is dealt to blocks, and a sum over 150 000 tokens is as exact as its terms (in
// fp32 a boundary between two tokens would move by 2^-24 of the sum, more than a rare token is wide).  Thresholds are found on the logits
// themselves, never on weights.
//
// A row belongs to the CTAs of a cluster, each with a contiguous range of columns that it brings into shared memory once where it fits and the row starts on a 16-byte
// boundary (a bulk copy per warp; other rows are read from memory in every pass, element by element) and then goes through a few times: for the maximum; for the sum of the weights where it is needed; for the tokens that are large enough to matter. How
// large that is the maxima of the threads' own tokens tell: the k-th largest of them has at least k tokens at or above it, and hardly more. Those tokens are
// sorted by one CTA, which mostly finds everything that is kept among them and finishes alone. Where it does not (flat rows, thousands of tokens kept), counts or
// weights in 16 intervals of z, then in 16 parts of the one in which the last token kept lies, and so on, lead to a list of tokens around it, and the row is
// drawn from by sums over ranges.
//
// us per call, twenty to a graph, rows of 151 936 tokens in bf16 (64 of them 19.4 MB, 3 us of memory; normal with a spread of 2.2 and some 300 likelier tokens), all at
// temperature 1 but for the greedy and the flat ones (temperature 3):
//            greedy  top-k 50  top-k 400  no filter  top-p 0.9  min-p 0.05  top-k 2000  flat, top-p 0.95
//   1 row       4.3      11.1       14.6        8.5       14.9         7.8        25.4        54.4
//   64 rows     6.6      14.3       22.6       16.3       22.0        11.5        70.9       115
//   200 rows   16.6      29.6       53.2       45.1       57.4        28.1       180         394
//   64 rows of 151 937 (seven of eight start off a 16-byte boundary): 22.8, 29.9, no filter 31.1, top-p 44.8, flat 176; of 50 257 against 50 256: 10.5 / 4.9, 18.1 / 12.9,
//   15.3 / 10.1, 24.5 / 16.9.
// Not the memory is the bound: launch and copy are 4.5 of it, every meeting of a row's CTAs is 1 (there are two to six), the sum of the weights 6 (76 000 tokens per SM, an
// exponential and about 18 instructions each), sorting and the draw 2 to 8.
#include <type_traits>

#include "common.cuh"
#include "mma.cuh"
#include "tc5.cuh"

namespace b200 {

namespace {

using u64 = unsigned long long;
template <typename T> struct Pair;
template <> struct Pair<__half> { using type = __half2; };
template <> struct Pair<__nv_bfloat16> { using type = __nv_bfloat162; };
constexpr int ST = 512, SW = ST / 32;        // threads and warps of a CTA
constexpr int MAX_CTAS = 8;                  // of a row
constexpr int64_t MAX_COLS = 1 << 22;        // sums of weights are at most 2^62
constexpr u64 ONE = 1ull << 40;              // weight of the row's maximum
constexpr int BINS = 16;
constexpr int CAP = 2048;                    // tokens of a list
constexpr int BIN_BYTES = SW * BINS * 32 * 8;   // a counter per warp, bin and lane; later the lists
constexpr int STAGE_BYTES = 152 * 1024;      // of a CTA's columns at most
static_assert(BIN_BYTES >= 3 * CAP * 8, "the lists lie over the counters");
static_assert(MAX_COLS / (MAX_CTAS * ST) <= 1024, "a lane's columns: Weigher::Sum");

struct SampleParams {
  const void* logits;
  int64_t* out;
  int64_t row_stride;
  const float *temperature, *top_p, *min_p, *uniform;
  const int32_t* top_k;
  int cols, seg;   // columns of the row and of a CTA's range
  int staged;      // the range is brought into shared memory
};

// code left by a bounded wait that ran out
__device__ int g_sample_error = 0;

// Keys order like the logits they come from: equal keys, equal values (-0 counts as 0); NaN comes first.
__device__ __forceinline__ uint32_t key_of(float x) {
  if (x != x) return 0xffffffffu;
  const uint32_t b = __float_as_uint(x + 0.f);
  return b & 0x80000000u ? ~b : b | 0x80000000u;
}

// Two fp32 numbers in a pair of registers, and the instructions for both at once
struct Two { u64 v; };
__device__ __forceinline__ Two two(float a, float b) {
  Two r;
  asm("mov.b64 %0, {%1, %2};" : "=l"(r.v) : "f"(a), "f"(b));
  return r;
}
__device__ __forceinline__ float first(Two a) { return __uint_as_float(static_cast<uint32_t>(a.v)); }
__device__ __forceinline__ float second(Two a) { return __uint_as_float(static_cast<uint32_t>(a.v >> 32)); }
__device__ __forceinline__ Two fma2(Two a, Two b, Two c) {
  Two r;
  asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(r.v) : "l"(a.v), "l"(b.v), "l"(c.v));
  return r;
}
__device__ __forceinline__ Two mul2(Two a, Two b) {
  Two r;
  asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(r.v) : "l"(a.v), "l"(b.v));
  return r;
}
__device__ __forceinline__ Two add2_down(Two a, Two b) {   // rounded towards zero
  Two r;
  asm("add.rz.f32x2 %0, %1, %2;" : "=l"(r.v) : "l"(a.v), "l"(b.v));
  return r;
}
__device__ __forceinline__ float exp2_fast(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}

// exp((z - m) / T) = 2^-t, t = (m - z) log2(e) / T.  log2(e) / T is carried as a pair of fp32 numbers, and the difference where it need not be whole:
// a rounding of t = 30 alone would be 2^-20 of the weight.  Two ways:
// - the few tokens that the row's sum mostly consists of (t below 12, less at temperatures above 1, where the sum spreads over more) by the table method
//   (P. T. P. Tang, 1989): t to 32 binary places, 2^-(i / 256) from a table for the first eight, a cubic for the rest (its next term is below 2^-38).  The
//   sum at every later boundary moves with their errors, and most of 150 000 tokens are less than 2^-22 of it wide: with the other way for them too,
//   one draw in a hundred from a row without filters would give a neighbour of the right token; so it is one in 30 000.
// - all others by the fast exponential of t's distance from the nearest whole number, good to 2^-22 of itself: errors of many small weights, as good as
//   independent.  Straight through and without conversions (they share their unit with the exponential).
template <typename T> struct Weigher {
  float m, c_hi, c_lo;
  float end, near;         // differences at which t is 43 (an eighth of a unit: no weight), and below which the table is used
  const uint32_t* table;   // 2^31 2^-(i / 256)
  // m - z, not above `end`
  __device__ __forceinline__ float difference(float z) const { return fminf(m - z, end); }
  __device__ __forceinline__ float rest(float z, float dh) const {   // (m - z) - dh
    const float bv = m - dh;
    return (m - (dh + bv)) + (bv - z);
  }
  // weight = (hi - 0x4b000000) 2^20 + lo - 0x4b000000, both whole numbers up to 2^21, for a difference of z or `end`
  __device__ __forceinline__ void parts(float z, float dh, uint32_t& hi, uint32_t& lo) const {
    const float shifted = fmaf(dh, c_hi, 12582912.f);      // + 1.5 2^23: t to the nearest whole number
    float x = fmaf(dh, c_lo, fmaf(dh, c_hi, -(shifted - 12582912.f)));
    if constexpr (sizeof(T) == 4) x = dh < end ? fmaf(rest(z, dh), c_hi, x) : x;   // (differences of 16-bit logits are whole but for those next to zero)
    float y = exp2_fast(-x);
    y *= __uint_as_float((147u << 23) - (__float_as_uint(shifted) << 23));   // 2^(20 - whole): the weight in units of 2^-20
    const float h = __fadd_rz(y, 8388608.f);
    hi = __float_as_uint(h);
    lo = __float_as_uint(fmaf(y - (h - 8388608.f), 1048576.f, 8388608.f));   // (rounded: cut off, 150 000 small weights would lose 2^-24 of the sum)
  }
  __device__ __forceinline__ u64 other(float z, float dh) const {
    uint32_t hi, lo;
    parts(z, dh, hi, lo);
    return (static_cast<u64>(hi - 0x4b000000u) << 20) + (lo - 0x4b000000u);
  }
  __device__ __forceinline__ u64 large(float z) const {   // (ONE for z == m)
    const float dh = m - z, p = __fmul_rn(dh, c_hi);
    const float e = fmaf(dh, c_hi, -p) + fmaf(dh, c_lo, rest(z, dh) * c_hi);
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
  __device__ __forceinline__ u64 operator()(float z) const {
    const float dh = difference(z);
    return dh < near ? large(z) : other(z, dh);
  }
  // f(token, its place among the eight) for those whose bit is set, a token of each lane at a time (a warp goes round as often as its lane with most of them has some)
  template <typename F> static __device__ __forceinline__ void each_set(uint32_t set, const float (&z)[8], F&& f) {
    while (set) {
      const int at = __ffs(set) - 1;
      set &= set - 1;
      float v = z[0];
#pragma unroll
      for (int k = 1; k < 8; ++k) v = at == k ? z[k] : v;
      f(v, at);
    }
  }
  // Sum of the weights, of at least `least`, of those of eight tokens that keep(token, column) lets through
  template <typename K> __device__ __forceinline__ u64 sum(const float (&z)[8], int c, u64 least, K&& keep) const {
    uint32_t close = 0;
    u64 t = 0;
#pragma unroll
    for (int k = 0; k < 8; ++k) {
      const float dh = difference(z[k]);
      const bool kept = keep(z[k], c + k);
      close |= (kept && dh < near ? 1u : 0u) << k;
      const u64 w = other(z[k], kept && dh >= near ? dh : end);
      t += w >= least ? w : 0;
    }
    each_set(close, z, [&](float v, int) {
      const u64 w = large(v);
      t += w >= least ? w : 0;
    });
    return t;
  }
  // Running sum of a lane's weights: its two parts (with 0x4b000000 for every token so far: up to 1024 of them, below 2^31), and what near tokens weigh
  // more than in the parts
  struct Sum {
    uint32_t hi = 0, lo = 0, tokens = 0;
    u64 near = 0;
    __device__ __forceinline__ u64 total() const { return (static_cast<u64>(hi - tokens * 0x4b000000u) << 20) + (lo - tokens * 0x4b000000u) + near; }
  };
  // Adds the weights of eight tokens, the largest of which is `top`: the other way for all of them, two at a time (as parts() to the bit), then the few near
  // ones once more
  __device__ __forceinline__ void add(Sum& sum, const float (&z)[8], float top) const {
    const Two m2 = two(m, m), nch = two(-c_hi, -c_hi), ncl = two(-c_lo, -c_lo), minus = two(-1.f, -1.f), half = two(12582912.f, 12582912.f);
    const Two unit = two(8388608.f, 8388608.f), low = two(1048576.f, 1048576.f);
#pragma unroll
    for (int k = 0; k < 8; k += 2) {
      const Two z2 = two(z[k], z[k + 1]);
      Two d = fma2(z2, minus, m2);
      d = two(fminf(first(d), end), fminf(second(d), end));
      const Two shifted = fma2(d, nch, half);              // t's nearest whole number, counted down
      Two x = fma2(d, ncl, fma2(d, nch, fma2(shifted, minus, half)));   // - (t - the nearest whole number)
      if constexpr (sizeof(T) == 4) {
        const Two one = two(1.f, 1.f), bv = fma2(d, minus, m2), a = fma2(fma2(d, one, bv), minus, m2), b = fma2(z2, minus, bv);
        const Two y = fma2(fma2(a, one, b), nch, x);
        x = two(first(d) < end ? first(y) : first(x), second(d) < end ? second(y) : second(x));
      }
      Two y = two(exp2_fast(first(x)), exp2_fast(second(x)));
      y = mul2(y, two(__uint_as_float((__float_as_uint(first(shifted)) << 23) + (147u << 23)), __uint_as_float((__float_as_uint(second(shifted)) << 23) + (147u << 23))));
      const Two h = add2_down(y, unit), l = fma2(fma2(fma2(unit, minus, h), minus, y), low, unit);
      sum.hi += __float_as_uint(first(h)) + __float_as_uint(second(h));
      sum.lo += __float_as_uint(first(l)) + __float_as_uint(second(l));
    }
    sum.tokens += 8;
    if (difference(top) < near) {
      uint32_t close = 0;
#pragma unroll
      for (int k = 0; k < 8; ++k) close |= (difference(z[k]) < near ? 1u : 0u) << k;
      each_set(close, z, [&](float v, int) { sum.near += large(v) - other(v, difference(v)); });
    }
  }
};

struct Shared {
  uint32_t table[256];
  u64 part[SW];
  u64 told[2][MAX_CTAS];   // values of all CTAs of the row, two exchanges deep
  u64 bin_mass[SW][BINS], told_mass[2][MAX_CTAS][BINS];
  uint32_t bin_count[SW][32], told_count[2][MAX_CTAS][32];
  u64 cut_last;            // from the list: key << 32 | index of the last token kept
  int listed;
  int pick[2], settled;
  __align__(8) uint64_t full[SW];
};

// NaN where one of the two is
__device__ __forceinline__ float max_nan(float a, float b) {
  float r;
  asm("max.NaN.f32 %0, %1, %2;" : "=f"(r) : "f"(a), "f"(b));
  return r;
}
template <typename T> __device__ __forceinline__ uint32_t max2(uint32_t a, uint32_t b) {   // of pairs of 16-bit numbers
  if constexpr (sizeof(T) == 4) {
    return a;
  } else {
    using P = typename Pair<T>::type;
    const P r = __hmax2_nan(reinterpret_cast<const P&>(a), reinterpret_cast<const P&>(b));
    return reinterpret_cast<const uint32_t&>(r);
  }
}

// A thread's share of the CTA's columns: warp w has a contiguous range, 256 columns at a time, eight per lane.
template <typename T> struct Row {
  const T* x;
  const T* copy;             // of this warp's range, or nullptr
  int begin, end, copied;    // columns begin .. copied - 1 are in the copy
  bool vec;
  bool infinite = false;     // the maximum is +infinity: as if it were 0 and all else -infinity
  __device__ __forceinline__ void load(int c, float (&f)[8]) const {   // columns c .. c + 7; those past the end as -infinity
    fetch(c, f);
    if (infinite)
#pragma unroll
      for (int k = 0; k < 8; ++k) f[k] = f[k] == INFINITY ? 0.f : -INFINITY;
  }
  __device__ __forceinline__ void fetch(int c, float (&f)[8]) const {
    if (c + 8 <= copied) {
      unpack(copy + (c - begin), f);
    } else if (vec && c + 8 <= end) {
      unpack(x + c, f);
    } else {
#pragma unroll
      for (int k = 0; k < 8; ++k) f[k] = c + k < end ? to_f32<T>(x[c + k]) : -INFINITY;
    }
  }
  // f(the largest of columns c .. c + 7, NaN where there is one; c) for the warp's columns from `from` up to `to`
  template <typename F> __device__ __forceinline__ void tops(int from, int to, F&& f) const {
    int c = from + (threadIdx.x & 31) * 8;
    to = min(to, end);
    const auto of = [](const float (&z)[8]) {
      return max_nan(max_nan(max_nan(z[0], z[1]), max_nan(z[2], z[3])), max_nan(max_nan(z[4], z[5]), max_nan(z[6], z[7])));
    };
    if (!infinite && (copied > begin || vec)) {   // 128, then 64 bytes of a thread under way
      const T* const at = copied > begin ? copy - begin : x;
      const int all = min(to, copied > begin ? copied : end);
      const auto some = [&](auto count) {
        constexpr int N = decltype(count)::value;
        for (; c + (N - 1) * 256 + 8 <= all; c += N * 256) {
          if constexpr (sizeof(T) == 2) {
            uint4 w[N];
#pragma unroll
            for (int i = 0; i < N; ++i) w[i] = *reinterpret_cast<const uint4*>(at + c + 256 * i);
#pragma unroll
            for (int i = 0; i < N; ++i) {
              float a, b;
              unpack2<T>(max2<T>(max2<T>(w[i].x, w[i].y), max2<T>(w[i].z, w[i].w)), a, b);
              f(max_nan(a, b), c + 256 * i);
            }
          } else {
            float z[N][8];
#pragma unroll
            for (int i = 0; i < N; ++i) unpack(at + c + 256 * i, z[i]);
#pragma unroll
            for (int i = 0; i < N; ++i) f(of(z[i]), c + 256 * i);
          }
        }
      };
      some(std::integral_constant<int, 16 / sizeof(T)>());
      some(std::integral_constant<int, 8 / sizeof(T)>());
    }
    for (; c < to; c += 256) {
      float z[8];
      load(c, z);
      f(of(z), c);
    }
  }
  // f(eight tokens, the largest of them, their first column) for all of the warp's columns
  template <typename F> __device__ __forceinline__ void eights(F&& f) const {
    const auto of = [](const float (&z)[8]) { return fmaxf(fmaxf(fmaxf(z[0], z[1]), fmaxf(z[2], z[3])), fmaxf(fmaxf(z[4], z[5]), fmaxf(z[6], z[7]))); };
    int c = begin + (threadIdx.x & 31) * 8;
    if (!infinite && (copied > begin || vec)) {   // the next load is under way meanwhile
      const T* const at = copied > begin ? copy - begin : x;
      const int all = copied > begin ? copied : end;
      using Raw = std::conditional_t<sizeof(T) == 2, uint4, float4>;
      Raw w[8 * sizeof(T) / 16];
      if (c + 8 <= all) {
#pragma unroll
        for (int i = 0; i < static_cast<int>(sizeof(T) / 2); ++i) w[i] = *(reinterpret_cast<const Raw*>(at + c) + i);
      }
#pragma unroll 1
      for (; c + 8 <= all; c += 256) {
        float z[8], top;
        if constexpr (sizeof(T) == 2) {
          unpack8<T>(w[0], z);
          float a, b;
          unpack2<T>(max2<T>(max2<T>(w[0].x, w[0].y), max2<T>(w[0].z, w[0].w)), a, b);
          top = fmaxf(a, b);
        } else {
          z[0] = w[0].x; z[1] = w[0].y; z[2] = w[0].z; z[3] = w[0].w; z[4] = w[1].x; z[5] = w[1].y; z[6] = w[1].z; z[7] = w[1].w;
          top = of(z);
        }
        if (c + 256 + 8 <= all) {
#pragma unroll
          for (int i = 0; i < static_cast<int>(sizeof(T) / 2); ++i) w[i] = *(reinterpret_cast<const Raw*>(at + c + 256) + i);
        }
        f(z, top, c);
      }
    }
    for (; c < end; c += 256) {
      float z[8];
      load(c, z);
      f(z, of(z), c);
    }
  }
  // f(eight tokens, their first column) for those eights that have one of at least `floor`: first where there is any at all, 32 of a lane at a time, then
  // those one after the other (a warp has few where few tokens matter, but hardly 256 columns without one: k = 400 in 64 rows 2 us instead of 7.5)
  template <typename F> __device__ __forceinline__ void from(float floor, F&& f) const {
#pragma unroll 1
    for (int base = begin; base < end; base += 32 * 256) {
      uint32_t some = 0;
      tops(base, base + 32 * 256, [&](float z, int c) { some |= (z >= floor ? 1u : 0u) << ((c - base) >> 8); });
      while (some) {
        const int c = base + (__ffs(some) - 1) * 256 + (threadIdx.x & 31) * 8;
        some &= some - 1;
        float z[8];
        load(c, z);
        f(z, c);
      }
    }
  }
  static __device__ __forceinline__ void unpack(const T* at, float (&f)[8]) {
    if constexpr (sizeof(T) == 2) {
      unpack8<T>(*reinterpret_cast<const uint4*>(at), f);
    } else {
      const float4 a = *reinterpret_cast<const float4*>(at), b = *(reinterpret_cast<const float4*>(at) + 1);
      f[0] = a.x; f[1] = a.y; f[2] = a.z; f[3] = a.w; f[4] = b.x; f[5] = b.y; f[6] = b.z; f[7] = b.w;
    }
  }
  template <typename F> __device__ __forceinline__ void each(F&& f) const {
#pragma unroll 2
    for (int c = begin + (threadIdx.x & 31) * 8; c < end; c += 256) {
      float v[8];
      load(c, v);
#pragma unroll
      for (int k = 0; k < 8; ++k) f(v[k], c + k);
    }
  }
};

__device__ __forceinline__ u64 warp_add(u64 v) {   // (v at most 2^62; in three parts the warp's own instruction does it)
  const uint32_t a = __reduce_add_sync(0xffffffffu, static_cast<uint32_t>(v) & 0x3ffffffu), b = __reduce_add_sync(0xffffffffu, static_cast<uint32_t>(v >> 26) & 0x3ffffffu);
  return a + (static_cast<u64>(b) << 26) + (static_cast<u64>(__reduce_add_sync(0xffffffffu, static_cast<uint32_t>(v >> 52))) << 52);
}

// Sum, or maximum (of 32 bits), over all threads of the row, known to all of them.  sh.told holds the CTAs' values afterwards, in slot `turn`.
template <bool TOP> __device__ u64 row_reduce(u64 v, Shared& sh, int ctas, int& turn) {
  v = TOP ? __reduce_max_sync(0xffffffffu, static_cast<uint32_t>(v)) : warp_add(v);
  if ((threadIdx.x & 31) == 0) sh.part[threadIdx.x >> 5] = v;
  __syncthreads();
  if (threadIdx.x < 32) {
    u64 s = threadIdx.x < SW ? sh.part[threadIdx.x] : 0;
    s = TOP ? __reduce_max_sync(0xffffffffu, static_cast<uint32_t>(s)) : warp_add(s);
    if (ctas == 1) {
      if (threadIdx.x == 0) sh.told[turn][0] = s;
    } else if (static_cast<int>(threadIdx.x) < ctas) {
      const uint32_t to = tc5::map_to_rank(tc5::smem_addr(&sh.told[turn][tc5::cluster_ctarank()]), threadIdx.x);
      asm volatile("st.shared::cluster.u64 [%0], %1;" ::"r"(to), "l"(s) : "memory");
    }
    __syncwarp();
  }
  if (ctas == 1) __syncthreads(); else tc5::cluster_sync();
  u64 r = 0;
  for (int i = 0; i < ctas; ++i) r = TOP ? (sh.told[turn][i] > r ? sh.told[turn][i] : r) : r + sh.told[turn][i];
  turn ^= 1;
  return r;
}

// list[0 .. n) in descending order.  All threads; begins and ends with a barrier; list[n] up to the next multiple of 256 may be overwritten.
// Every warp sorts 32 elements at a time by shuffles, then four runs at a time become one: an element's place is its own plus those that the other three runs
// have ahead of it, looked for by halving.  Meanwhile element i lies at i ^ (i / 16 % 16): steps by 16 and more would all meet in one bank.  (us for 110 and 490 elements: 1.0 and 2.7, where steps over all of the list took 2.9 and 4.6.)
template <int E> __device__ __forceinline__ void sort_elements(u64* list, int n) {
  const int i = threadIdx.x, lane = i & 31;
  const auto place = [](int at) { return at ^ ((at >> 4) & 15); };
  u64 v[E];
#pragma unroll
  for (int e = 0; e < E; ++e) v[e] = i + ST * e < n ? list[i + ST * e] : 0;
  n = (n + 31) & ~31;
#pragma unroll
  for (int size = 2; size <= 32; size <<= 1)
#pragma unroll
    for (int step = size >> 1; step > 0; step >>= 1) {
      const bool larger = ((lane & step) == 0) == ((lane & size) == 0 || size == 32);   // the larger of the two stays here
#pragma unroll
      for (int e = 0; e < E; ++e) {
        const u64 w = __shfl_xor_sync(0xffffffffu, v[e], step);
        v[e] = larger == (w > v[e]) ? w : v[e];
      }
    }
#pragma unroll
  for (int e = 0; e < E; ++e)
    if (i + ST * e < n) list[n > 32 ? place(i + ST * e) : i] = v[e];
  __syncthreads();
#pragma unroll 1
  for (int run = 32; run < n; run <<= 2) {
    int to[E];
#pragma unroll
    for (int e = 0; e < E; ++e) {
      const int at = i + ST * e, four = at & ~(4 * run - 1), own = (at - four) & ~(run - 1);
      to[e] = at - own;
      if (at < n) {   // (a whole warp is, or is not)
        int ahead[3] = {0, 0, 0};
#pragma unroll 1
        for (int step = run; step > 0; step >>= 1)
#pragma unroll
          for (int o = 0; o < 3; ++o) {   // the other runs (no two elements are equal but the filling, which is all in one run)
            const int last = ahead[o] + step - 1, there = four + o * run + (o * run >= own ? run : 0) + last;
            const bool in = last < run && there < n;
            const u64 w = list[place(in ? there : at)];
            ahead[o] += in && w > v[e] ? step : 0;
          }
        to[e] += ahead[0] + ahead[1] + ahead[2];
      }
    }
    __syncthreads();
#pragma unroll
    for (int e = 0; e < E; ++e)
      if (i + ST * e < n) list[4 * run < n ? place(to[e]) : to[e]] = v[e];
    __syncthreads();
    if (4 * run < n) {
#pragma unroll
      for (int e = 0; e < E; ++e) v[e] = i + ST * e < n ? list[place(i + ST * e)] : 0;
    }
  }
}
__device__ void sort_list(u64* list, int n) {
  __syncthreads();
  if (n <= ST) sort_elements<1>(list, n);
  else if (n <= 2 * ST) sort_elements<2>(list, n);
  else sort_elements<4>(list, n);
}
static_assert(CAP == 4 * ST, "sort_list");

// sums[i] = val(0) + .. + val(i) for i < n <= CAP.  All threads; ends with a barrier.
template <typename F> __device__ void scan_list(u64* sums, int n, Shared& sh, F&& val) {
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, per = (n + ST - 1) / ST;
  u64 run = 0;
  for (int e = 0; e < per; ++e) {
    const int i = threadIdx.x * per + e;
    if (i < n) {
      run += val(i);
      sums[i] = run;
    }
  }
  u64 upto = run;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const u64 t = __shfl_up_sync(0xffffffffu, upto, o);
    if (lane >= o) upto += t;
  }
  __syncthreads();
  if (lane == 31) sh.part[warp] = upto;
  __syncthreads();
  u64 before = upto - run;
#pragma unroll
  for (int w = 0; w < SW; ++w) before += w < warp ? sh.part[w] : 0;
  for (int e = 0; e < per; ++e) {
    const int i = threadIdx.x * per + e;
    if (i < n) sums[i] += before;
  }
  __syncthreads();
}

__device__ __forceinline__ float value_of(uint32_t key) { return __uint_as_float(key & 0x80000000u ? key & 0x7fffffffu : ~key); }

template <typename T>
__global__ void __launch_bounds__(ST, 1) sample_rows_kernel(const __grid_constant__ SampleParams p) {
  extern __shared__ __align__(16) uint8_t dsm[];
  __shared__ Shared sh;
  u64* const bins = reinterpret_cast<u64*>(dsm);
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, ctas = gridDim.x, rank = blockIdx.x;
  const int64_t r = blockIdx.y;
  int turn = 0;
  const T* x = static_cast<const T*>(p.logits) + r * p.row_stride;
  const int c0 = min(p.cols, rank * p.seg), c1 = min(p.cols, c0 + p.seg);
  const int span = (((c1 - c0 + SW - 1) / SW) + 255) & ~255;   // columns of a warp
  Row<T> row;
  row.x = x;
  row.begin = min(c1, c0 + warp * span);
  row.end = min(c1, row.begin + span);
  row.vec = (reinterpret_cast<uintptr_t>(x) & 15u) == 0;
  row.copied = row.begin;
  row.copy = reinterpret_cast<const T*>(dsm + BIN_BYTES) + (row.begin - c0);
  if (ctas > 1) tc5::cluster_arrive();   // (this CTA runs: its shared memory may be written to)
  if (lane == 0) tc5::mbar_init(&sh.full[warp], 1);
  if (threadIdx.x == 0) sh.listed = 0;
  tc5::fence_barrier_init();
  __syncwarp();
  pdl_trigger();
  pdl_wait();
  if (p.staged && row.vec) {
    const uint32_t bytes = static_cast<uint32_t>(row.end - row.begin) * sizeof(T) & ~15u;
    row.copied = row.begin + bytes / sizeof(T);
    if (bytes && lane == 0) {
      tc5::mbar_arrive_expect_tx(&sh.full[warp], bytes);
      asm volatile("cp.async.bulk.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1], %2, [%3];"
                   ::"r"(tc5::smem_addr(row.copy)), "l"(x + row.begin), "r"(bytes), "r"(tc5::smem_addr(&sh.full[warp])) : "memory");
    }
  }
  if (threadIdx.x < 256) sh.table[threadIdx.x] = static_cast<uint32_t>(exp2(-static_cast<double>(threadIdx.x) / 256.) * 2147483648. + 0.5);
  const float T_ = p.temperature ? __ldg(p.temperature + r) : 1.f, tp = p.top_p ? __ldg(p.top_p + r) : 1.f, mp = p.min_p ? __ldg(p.min_p + r) : 0.f;
  const int k = p.top_k ? __ldg(p.top_k + r) : 0;
  const float uniform = __ldg(p.uniform + r);
  // (temperatures past 1e30 and below 5e-39 count as those: differences of logits are not told apart any more, or not there at all)
  const double c_ = fmin(1.4426950408889634074 / fmin(static_cast<double>(T_), 1e30), 3e38);
  Weigher<T> weight;
  weight.m = 0.f;
  weight.c_hi = static_cast<float>(c_);
  weight.c_lo = static_cast<float>(c_ - static_cast<double>(weight.c_hi));
  weight.end = static_cast<float>(43. / c_);
  weight.near = static_cast<float>(12. / c_) / fmaxf(T_, 1.f);
  weight.table = sh.table;
  const u64 least = mp > 0.f ? static_cast<u64>(ceil(static_cast<double>(fminf(mp, 1.f)) * static_cast<double>(ONE))) : 0;
  if (row.copied > row.begin && !tc5::mbar_wait(&sh.full[warp], 0) && lane == 0) atomicExch(&g_sample_error, 70);

  // ---- the maximum ----
  float top = -INFINITY;   // of this thread's tokens
  row.tops(row.begin, row.end, [&](float z, int) { top = max_nan(top, z); });
  __syncwarp();
  if (ctas > 1) tc5::cluster_wait();   // every CTA of the row runs
  const u64 best = row_reduce<true>(key_of(top), sh, ctas, turn);   // (its barriers are the table's too)
  float m = value_of(static_cast<uint32_t>(best));
  const bool none = !(m > -INFINITY);     // a row without any weight, or with a NaN: there is nothing to draw from
  if (!(T_ > 0.f) || none) {              // greedy: the first of the largest
    u64 at = 0;
    if (!none) {
      row.from(m, [&](const float (&z)[8], int c) {
#pragma unroll
        for (int e = 7; e >= 0; --e)
          if (z[e] == m && static_cast<uint32_t>(~(c + e)) > at) at = static_cast<uint32_t>(~(c + e));
      });
      at = row_reduce<true>(at, sh, ctas, turn);
    }
    if (rank == 0 && threadIdx.x == 0) p.out[r] = none ? 0 : static_cast<int>(~static_cast<uint32_t>(at));
    return;
  }
  if (m == INFINITY) {
    row.infinite = true;
    top = top == m ? 0.f : -INFINITY;
    m = 0.f;
  }
  weight.m = m;
  auto target_of = [&](u64 total) -> u64 {
    const double d = static_cast<double>(uniform) * static_cast<double>(total);
    const u64 t = d > 0. ? (d < static_cast<double>(total) ? static_cast<u64>(d) : total - 1) : 0;
    return t < total ? t : total - 1;
  };

  // What is kept: logits above that of key `cut`, and of those equal to it the indices up to `last`
  uint32_t cut = 0;
  int last = p.cols;
  auto stays = [&](float z, int i) {
    const uint32_t key = key_of(z);
    return key > cut || (key == cut && i <= last);
  };

  // The place of a logit below the maximum, from its difference: t in units of 2^-17, 23 bits.  It falls as logits rise (every step of its arithmetic
  // does), equal places need not mean equal logits.  Those at `end` weigh nothing and count as not there.
  constexpr int PLACE_BITS = 23;
  constexpr uint32_t LAST_PLACE = (1u << PLACE_BITS) - 1u;
  auto place = [&](float dh) { return __float_as_uint(fmaf(__fmul_rn(dh, weight.c_hi), 131072.f, 8388608.f)) & LAST_PLACE; };

  // Looks for the token that the filter ends with: the k-th (count), or the one at which the running sum reaches `limit`.  Result: 0 nothing is cut off,
  // 1 all that is kept is in the list of CTA 0, 2 (cut, last) are found, 3 they are to be found bit by bit.
  u64 whole = 0;         // sum of what is kept before top-p
  bool few = false;      // the search knows that hardly an eighth of a warp's tokens can still matter: Row::from() instead of Row::eights()
  auto limit_of = [&](u64 sum) { return fmax(static_cast<double>(tp) * static_cast<double>(sum), 0.5); };
  const bool restricted_by_k = k > 0 && k < p.cols;
  auto lowest = [&](uint32_t hi) {   // no token with a place up to `hi` is below this
    return weight.m - fminf((static_cast<float>(hi) + 8.f) * (1.0001f / 131072.f) / weight.c_hi, weight.end) - fabsf(weight.m) * 5e-7f;
  };
  auto collect = [&](uint32_t lo, uint32_t hi) {   // tokens with places in [lo, hi], to CTA 0: into a list of each CTA's own, then in one piece
    // (a bound on the logits with some room: places are looked at only behind it)
    const float above = lo == 0 ? INFINITY : weight.m - (static_cast<float>(lo) - 8.f) * (0.9999f / 131072.f) / weight.c_hi + fabsf(weight.m) * 5e-7f;
    const float bound = lowest(hi);
    const auto take = [&](const float (&z)[8], int c) {
      uint32_t some = 0;
#pragma unroll
      for (int k = 0; k < 8; ++k) some |= (z[k] >= bound && z[k] <= above ? 1u : 0u) << k;
      weight.each_set(some, z, [&](float v, int k) {
        const float dh = weight.difference(v);
        const uint32_t X = place(dh);
        if (dh < weight.end && X <= hi && X >= lo && stays(v, c + k)) {
          const int at = atomicAdd(&sh.listed, 1);
          if (at < CAP) bins[at] = static_cast<u64>(key_of(v)) << 32 | static_cast<uint32_t>(~(c + k));
        }
      });
    };
    if (lo == 0 || few) row.from(bound, take); else row.eights([&](const float (&z)[8], float, int c) { take(z, c); });
    __syncthreads();
    if (ctas == 1) return;
    // Everybody learns how many the others have: a CTA's go behind those of the ones before it
    const int mine = sh.listed;
    if (static_cast<int>(threadIdx.x) < ctas)
      asm volatile("st.shared::cluster.u64 [%0], %1;" ::"r"(tc5::map_to_rank(tc5::smem_addr(&sh.told[turn][rank]), threadIdx.x)), "l"(static_cast<u64>(mine)) : "memory");
    __syncwarp();
    tc5::cluster_sync();
    int at = 0, total = 0;
    for (int i = 0; i < ctas; ++i) {
      const int n = static_cast<int>(sh.told[turn][i]);
      at += i < rank ? n : 0;
      total += n;
    }
    turn ^= 1;
    if (rank != 0) {
      const int n = min(min(mine, CAP), CAP - at);
      const uint32_t to = tc5::map_to_rank(tc5::smem_addr(bins), 0);
      for (int i = threadIdx.x; i < n; i += ST) asm volatile("st.shared::cluster.u64 [%0], %1;" ::"r"(to + (at + i) * 8), "l"(bins[i]) : "memory");
    }
    if (threadIdx.x == 0) sh.listed = rank == 0 ? total : 0;
    __syncwarp();
    tc5::cluster_sync();
  };
  auto sorted = [&]() {   // CTA 0: its list in order; the number of tokens
    const int n = min(sh.listed, CAP);
    sort_list(bins, n);
    return n;
  };
  auto search = [&](const bool by_mass) __attribute__((always_inline)) -> int {
    uint32_t first = 0, end = LAST_PLACE, above = 0;   // places that are looked at, tokens before them
    u64 above_mass = 0;
    double limit = 0.;
    const float at_least = cut == 0 ? -INFINITY : value_of(cut);   // (what top-k has left)
    few = few && cut != 0;
#pragma unroll 1
    for (int shift = PLACE_BITS - 4; ; shift = shift >= 4 ? shift - 4 : 0) {
      u64* const own = bins + warp * BINS * 32 + lane;
#pragma unroll
      for (int b = 0; b < BINS; ++b) own[b * 32] = 0;
      // (a lane has fewer than 2^12 columns of a row, each below 2^40 + 1: 12 bits count, 52 add up)
      const auto count_in = [&](const float (&z)[8], int c) {
        uint32_t close = 0;
#pragma unroll
        for (int e = 0; e < 8; ++e) {
          const float dh = weight.difference(z[e]);
          const uint32_t X = place(dh) - first;
          bool in = dh < weight.end && X <= end - first;
          if (by_mass && restricted_by_k) in = in && stays(z[e], c + e);
          u64 add = 1ull << 52;
          if (by_mass) {
            close |= (in && dh < weight.near ? 1u : 0u) << e;
            in = in && dh >= weight.near;
            add += weight.other(z[e], dh);
          }
          own[in ? (X >> shift) * 32 : 0] += in ? add : 0;   // (without a branch)
        }
        weight.each_set(close, z, [&](float v, int) { own[((place(weight.difference(v)) - first) >> shift) * 32] += (1ull << 52) + weight.large(v); });
      };
      const float floor = end == LAST_PLACE ? at_least : fmaxf(at_least, lowest(end));
      if (few) row.from(floor, count_in); else row.eights([&](const float (&z)[8], float top_, int c) {
        if (top_ >= floor) count_in(z, c);
      });
      __syncwarp();
      {
        const int b = lane >> 1;
        uint32_t count = 0;
        u64 mass = 0;
#pragma unroll
        for (int e = 0; e < 16; ++e) {
          const u64 v = bins[(warp * BINS + b) * 32 + (lane & 1) * 16 + ((e + b) & 15)];
          count += static_cast<uint32_t>(v >> 52);
          mass += v & ((1ull << 52) - 1);
        }
        count += __shfl_xor_sync(0xffffffffu, count, 1);
        mass += __shfl_xor_sync(0xffffffffu, mass, 1);
        if (!(lane & 1)) { sh.bin_count[warp][b] = count; sh.bin_mass[warp][b] = mass; }
      }
      __syncthreads();
      if (static_cast<int>(threadIdx.x) < BINS * ctas) {
        const int b = threadIdx.x & (BINS - 1), to = threadIdx.x / BINS;
        uint32_t count = 0;
        u64 mass = 0;
        for (int w = 0; w < SW; ++w) { count += sh.bin_count[w][b]; mass += sh.bin_mass[w][b]; }
        if (ctas == 1) {
          sh.told_count[turn][0][b] = count;
          sh.told_mass[turn][0][b] = mass;
        } else {
          const uint32_t me = tc5::cluster_ctarank();
          asm volatile("st.shared::cluster.u32 [%0], %1;" ::"r"(tc5::map_to_rank(tc5::smem_addr(&sh.told_count[turn][me][b]), to)), "r"(count) : "memory");
          asm volatile("st.shared::cluster.u64 [%0], %1;" ::"r"(tc5::map_to_rank(tc5::smem_addr(&sh.told_mass[turn][me][b]), to)), "l"(mass) : "memory");
        }
      }
      if (ctas == 1) __syncthreads(); else tc5::cluster_sync();
      // lane b of every warp: bin b over all CTAs, then running sums
      uint32_t count = 0;
      u64 mass = 0;
      for (int i = 0; i < ctas; ++i) { count += sh.told_count[turn][i][lane & 15]; mass += sh.told_mass[turn][i][lane & 15]; }
      turn ^= 1;
      uint32_t n = count;
      u64 s = mass;
#pragma unroll
      for (int o = 1; o < BINS; o <<= 1) {
        const uint32_t a = __shfl_up_sync(0xffffffffu, n, o);
        const u64 t = __shfl_up_sync(0xffffffffu, s, o);
        if ((lane & 15) >= o) { n += a; s += t; }
      }
      if (shift == PLACE_BITS - 4 && by_mass) {
        whole = __shfl_sync(0xffffffffu, s, 15);
        limit = limit_of(whole);
      }
      const bool reached = by_mass ? static_cast<double>(above_mass + s) >= limit : above + n >= static_cast<uint32_t>(k);
      const unsigned hit = __ballot_sync(0xffffffffu, reached && lane < BINS);
      if (!hit) return 0;   // (fewer than k tokens weigh anything)
      const int b = __ffs(hit) - 1;
      const uint32_t here = __shfl_sync(0xffffffffu, count, b);
      above += __shfl_sync(0xffffffffu, n, b) - here;
      above_mass += __shfl_sync(0xffffffffu, s, b) - __shfl_sync(0xffffffffu, mass, b);
      first += static_cast<uint32_t>(b) << shift;
      end = first + ((1u << shift) - 1u);
      few = (above + here) * 32 < static_cast<uint32_t>(p.cols);
      if (above + here <= CAP) { collect(0, end); return 1; }
      if (here <= CAP && (above > CAP - CAP / 8 || shift == 0)) {   // the last token kept is among these
        collect(first, end);
        if (rank == 0) {
          const int n_ = sorted();
          u64* const sums = bins + CAP;   // (over the running sums)
          int want;
          if (by_mass) {
            scan_list(sums, n_, sh, [&](int i) { return weight(value_of(static_cast<uint32_t>(bins[i] >> 32))); });
            int mine = n_;   // the first at which the running sum reaches the limit
            for (int i = threadIdx.x; i < n_; i += ST)
              if (static_cast<double>(above_mass + sums[i]) >= limit) { mine = i; break; }
            if (threadIdx.x == 0) sh.pick[0] = n_ - 1;
            __syncthreads();
            atomicMin(&sh.pick[0], mine);
            __syncthreads();
            want = sh.pick[0];
          } else {
            want = static_cast<int>(static_cast<uint32_t>(k) - above) - 1;
          }
          if (static_cast<int>(threadIdx.x) < ctas) {
            const u64 v = bins[want];
            if (ctas == 1) sh.cut_last = v;
            else asm volatile("st.shared::cluster.u64 [%0], %1;" ::"r"(tc5::map_to_rank(tc5::smem_addr(&sh.cut_last), threadIdx.x)), "l"(v) : "memory");
          }
          if (threadIdx.x == 0) sh.listed = 0;
        }
        if (ctas == 1) __syncthreads(); else tc5::cluster_sync();
        cut = static_cast<uint32_t>(sh.cut_last >> 32);
        last = static_cast<int>(~static_cast<uint32_t>(sh.cut_last));
        return 2;
      }
      if (shift == 0) return 3;   // more equal places than a list holds
    }
  };

  // The thresholds bit by bit, a pass over the row for each bit of key and index: for rows with thousands of equal logits at the border
  auto index_limit = [&](u64 need) {   // the (need)th lowest index among the columns whose key is `cut`
    int at = 0;
#pragma unroll 1
    for (int bit = 1 << 21; bit > 0; bit >>= 1) {
      const int next = at | bit;
      u64 n = 0;
      row.each([&](float z, int i) { n += (i < next && i <= last && i < row.end && key_of(z) == cut) ? 1 : 0; });
      if (row_reduce<false>(n, sh, ctas, turn) < need) at = next;
    }
    return at;
  };
  auto top_k_by_bits = [&]() {
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
  };
  auto top_p_by_bits = [&]() {
    auto mass_from = [&](uint32_t from) {   // of what is kept so far, with keys of at least `from`
      u64 s = 0;
      row.each([&](float z, int i) {
        if (i < row.end && stays(z, i) && key_of(z) >= from) s += weight(z);
      });
      return row_reduce<false>(s, sh, ctas, turn);
    };
    const double limit = limit_of(whole);
    uint32_t at = 0;
#pragma unroll 1
    for (uint32_t bit = 0x80000000u; bit > 0; bit >>= 1)
      if (static_cast<double>(mass_from(at | bit)) >= limit) at |= bit;
    const u64 above = at == 0xffffffffu ? 0 : mass_from(at + 1);
    if (at != cut) { cut = at; last = p.cols; }
    last = min(last, index_limit(static_cast<u64>(ceil((limit - static_cast<double>(above)) / static_cast<double>(weight(value_of(at)))))));
  };

  // Places up to which at least `want` of the threads' largest tokens lie, hardly more (all places where there are not that many)
  auto reach = [&](uint32_t want) -> uint32_t {
    const float dh = weight.difference(top);
    const uint32_t X = dh < weight.end ? place(dh) : 1u << PLACE_BITS;
    uint32_t first = 0, above = 0;
#pragma unroll 1
    for (int shift = PLACE_BITS - 5; ; shift -= 5) {
      const uint32_t b = X >= first ? (X - first) >> shift : 32u;   // 32 and more: elsewhere
      uint32_t count = 0;
#pragma unroll
      for (int e = 0; e < 32; ++e) {
        const uint32_t n = __popc(__ballot_sync(0xffffffffu, b == e));
        count = lane == e ? n : count;
      }
      sh.bin_count[warp][lane] = count;
      __syncthreads();
      if (static_cast<int>(threadIdx.x) < 32 * ctas) {
        const int to = threadIdx.x / 32;
        uint32_t n = 0;
#pragma unroll
        for (int w = 0; w < SW; ++w) n += sh.bin_count[w][lane];
        if (ctas == 1) sh.told_count[turn][0][lane] = n;
        else asm volatile("st.shared::cluster.u32 [%0], %1;" ::"r"(tc5::map_to_rank(tc5::smem_addr(&sh.told_count[turn][rank][lane]), to)), "r"(n) : "memory");
      }
      if (ctas == 1) __syncthreads(); else tc5::cluster_sync();
      uint32_t n = 0;
      for (int i = 0; i < ctas; ++i) n += sh.told_count[turn][i][lane];
      turn ^= 1;
      const uint32_t here = n;
#pragma unroll
      for (int o = 1; o < 32; o <<= 1) {
        const uint32_t a = __shfl_up_sync(0xffffffffu, n, o);
        if (lane >= o) n += a;
      }
      const unsigned hit = __ballot_sync(0xffffffffu, above + n >= want);
      if (!hit) return LAST_PLACE;
      const int at = __ffs(hit) - 1;
      const uint32_t upto = above + __shfl_sync(0xffffffffu, n, at), size = __shfl_sync(0xffffffffu, here, at);
      first += static_cast<uint32_t>(at) << shift;
      if (upto <= want + want / 16 + 24 || shift <= 3) return first + ((1u << shift) - 1u);
      above = upto - size;
    }
  };

  const int threads = ctas * ST;
  int found = 0;
  bool all_k = false;    // the list holds the k tokens themselves
  u64 *const sums = bins + CAP, *const order = bins + 2 * CAP;
  // CTA 0: cuts the sorted list (of n tokens, with the running sums of their weights) off behind the last token kept, and draws in the order of the indices
  auto finish = [&](int n) {
    int kept = all_k && k < n ? k : n;
    const double limit = tp < 1.f ? limit_of(all_k ? sums[kept - 1] : whole) : 0.;
    if (threadIdx.x == 0) sh.pick[0] = sh.pick[1] = kept;
    __syncthreads();
    for (int i = threadIdx.x; i < kept; i += ST) {
      const u64 before = i > 0 ? sums[i - 1] : 0;
      if ((tp < 1.f && i > 0 && static_cast<double>(before) >= limit) || sums[i] - before < least) { atomicMin(&sh.pick[0], i); break; }
    }
    __syncthreads();
    kept = sh.pick[0];
    for (int i = threadIdx.x; i < kept; i += ST) order[i] = bins[i] << 32 | static_cast<uint32_t>(i);   // ~index, place in the list
    sort_list(order, kept);
    const u64 total = sums[kept - 1];
    scan_list(bins, kept, sh, [&](int i) {   // (the keys are not needed any more: weights come from the sums)
      const uint32_t j = static_cast<uint32_t>(order[i]);
      return sums[j] - (j > 0 ? sums[j - 1] : 0);
    });
    const u64 target = target_of(total);
    for (int i = threadIdx.x; i < kept; i += ST)
      if (bins[i] > target) { atomicMin(&sh.pick[1], i); break; }
    __syncthreads();
    if (threadIdx.x == 0) p.out[r] = static_cast<int>(~static_cast<uint32_t>(order[min(sh.pick[1], kept - 1)] >> 32));
  };

  // ---- the short way: the largest tokens, as many as k or as a nucleus mostly has ----
  // (k of the threads have one of the tokens that reach the k-th largest maximum, so there are threads ln(threads / (threads - k)) of them where tokens come as they
  // like: 200 rows with top-k 400, one CTA each, 53 us this way and 101 the other)
  const bool few_k = restricted_by_k && k < threads && k <= CAP / 2 &&
                     static_cast<float>(threads) * logf(static_cast<float>(threads) / static_cast<float>(threads - k)) <= 0.7f * CAP;
  if (few_k || (tp < 1.f && !restricted_by_k)) {
    if (!few_k) {
      typename Weigher<T>::Sum s;
      row.eights([&](const float (&z)[8], float top_, int) { weight.add(s, z, top_); });
      whole = row_reduce<false>(s.total(), sh, ctas, turn);
    }
    const uint32_t upto = reach(few_k ? static_cast<uint32_t>(k) : 96u);
    collect(0, upto);
    if (rank == 0) {
      const bool fits = sh.listed <= CAP;
      bool all = fits && few_k;
      int n = 0;
      if (fits) {
        n = sorted();
        scan_list(sums, n, sh, [&](int i) { return weight(value_of(static_cast<uint32_t>(bins[i] >> 32))); });
        if (!few_k) all = upto == LAST_PLACE || static_cast<double>(sums[n - 1]) >= limit_of(whole);
      }
      if (static_cast<int>(threadIdx.x) < ctas) {
        const int v = all ? 1 : 0;
        if (ctas == 1) sh.settled = v;
        else asm volatile("st.shared::cluster.u32 [%0], %1;" ::"r"(tc5::map_to_rank(tc5::smem_addr(&sh.settled), threadIdx.x)), "r"(v) : "memory");
      }
      __syncthreads();
      if (threadIdx.x == 0) sh.listed = 0;
      all_k = all && few_k;
      if (all) finish(n);
    }
    if (ctas > 1) tc5::cluster_sync(); else __syncthreads();
    if (sh.settled) return;
  }

  // ---- the long way ----
  if (restricted_by_k) {
    found = search(false);
    all_k = found == 1;
    if (found == 3) top_k_by_bits();
  }
  if (tp < 1.f && found != 1) {
    found = search(true);
    if (found == 3) top_p_by_bits();
  }
  if (found == 1) {
    if (rank != 0) return;
    const int n = sorted();
    scan_list(sums, n, sh, [&](int i) { return weight(value_of(static_cast<uint32_t>(bins[i] >> 32))); });
    finish(n);
    return;
  }

  // ---- the draw: sums of the warps' ranges, then of parts of the one in which the running sum passes the target ----
  auto kept = [&](float z, int i) -> u64 {
    if (!stays(z, i)) return 0;
    const u64 w = weight(z);
    return w >= least ? w : 0;
  };
  u64 mine = 0;
  const float at_cut = value_of(cut);
  const auto all = [](float, int) { return true; };
  const auto some = [&](float v, int i) { return v > at_cut || (v == at_cut && i <= last); };
  const auto add = [&](typename Weigher<T>::Sum& s, const float (&z)[8], float top_, int c) {
    if (cut == 0) {
      weight.add(s, z, top_);
    } else if (top_ >= at_cut) {
      float v[8];
#pragma unroll
      for (int e = 0; e < 8; ++e) v[e] = some(z[e], c + e) ? z[e] : -INFINITY;
      weight.add(s, v, top_);
    }
  };
  // (no token that weighs `least` is below this: the weight is at least half of it)
  const float enough = least > 0 ? weight.m - fminf((41.01f - log2f(static_cast<float>(least))) * 1.0001f / weight.c_hi, weight.end) - fabsf(weight.m) * 5e-7f : -INFINITY;
  if (least == 0 && !(few && cut != 0)) {
    typename Weigher<T>::Sum s;
    row.eights([&](const float (&z)[8], float top_, int c) { add(s, z, top_, c); });
    mine = s.total();
  } else if (cut == 0) row.from(enough, [&](const float (&z)[8], int c) { mine += weight.sum(z, c, least, all); });
  else row.from(fmaxf(enough, at_cut), [&](const float (&z)[8], int c) { mine += weight.sum(z, c, least, some); });
  const auto sum_of = [&](const float (&z)[8], int c) -> u64 {
    if (least != 0) return weight.sum(z, c, least, stays);
    typename Weigher<T>::Sum s;
    add(s, z, fmaxf(fmaxf(fmaxf(z[0], z[1]), fmaxf(z[2], z[3])), fmaxf(fmaxf(z[4], z[5]), fmaxf(z[6], z[7]))), c);
    return s.total();
  };
  mine = warp_add(mine);
  const int slot = turn;
  const u64 total = row_reduce<false>(lane == 0 ? mine : 0, sh, ctas, turn);
  const u64 target = target_of(total);
  u64 before = 0;
  for (int i = 0; i < rank; ++i) before += sh.told[slot][i];
  if (target < before || target >= before + sh.told[slot][rank]) return;   // another CTA's
  int w_ = 0;
  while (before + sh.part[w_] <= target) before += sh.part[w_++];
  // the range of warp w_, 256 columns of it to each warp at a time
  Row<T> part = row;
  part.begin = min(c1, c0 + w_ * span);
  part.end = min(c1, part.begin + span);
  part.copy = reinterpret_cast<const T*>(dsm + BIN_BYTES) + (part.begin - c0);
  part.copied = p.staged && row.vec ? part.begin + static_cast<int>((static_cast<uint32_t>(part.end - part.begin) * sizeof(T) & ~15u) / sizeof(T)) : part.begin;
  for (int b_ = part.begin; b_ < part.end; b_ += SW * 256) {
    const int c = b_ + warp * 256 + lane * 8;
    float v[8];
    u64 s = 0;
    if (c < part.end) {
      part.load(c, v);
      s = sum_of(v, c);
    }
    u64 upto = s;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const u64 t = __shfl_up_sync(0xffffffffu, upto, o);
      if (lane >= o) upto += t;
    }
    __syncthreads();   // (what was in sh.part has been read)
    if (lane == 31) sh.part[warp] = upto;
    __syncthreads();
    u64 mine_ = before;
#pragma unroll
    for (int i = 0; i < SW; ++i) {
      const u64 t = sh.part[i];
      mine_ += i < warp ? t : 0;
      before += t;
    }
    const unsigned passed = __ballot_sync(0xffffffffu, mine_ + upto > target);
    if (target >= mine_ && passed) {   // one of the eight tokens of lane `src`: a lane for each of them
      const int src = __ffs(passed) - 1, c_ = b_ + warp * 256 + src * 8;
      part.load(c_, v);
      float z = v[0];
#pragma unroll
      for (int e = 1; e < 8; ++e) z = (lane & 7) == e ? v[e] : z;
      u64 run = kept(z, c_ + (lane & 7));
#pragma unroll
      for (int o = 1; o < 8; o <<= 1) {
        const u64 t = __shfl_up_sync(0xffffffffu, run, o);
        if ((lane & 7) >= o) run += t;
      }
      const unsigned reached = __ballot_sync(0xffffffffu, __shfl_sync(0xffffffffu, mine_ + upto - s, src) + run > target) & 0x7fu;
      if (lane == 0) p.out[r] = c_ + (reached ? __ffs(reached) - 1 : 7);
    }
    if (target < before) return;
  }
}

// Clusters of 2, 4 and 8 CTAs that a device runs at once (SMs come in groups that a cluster cannot leave: 37 of 4 do not all fit on 148)
struct SampleWave {
  int rows[4] = {0, 0, 0, 0};   // [log2 of the CTAs]; 0: not known yet
};

template <typename T> int launch_sample(SampleParams p, int64_t rows, cudaStream_t st) {
  constexpr int smem = BIN_BYTES + STAGE_BYTES;
  static PerDevice<SampleWave> wave_on;
  SampleWave* const wave = wave_on.slot();
  if (!wave) B200_FAIL(B200_ELAUNCH, "sample_rows_kernel: no current device");
  if (!wave->rows[0]) {
    const cudaError_t e = cudaFuncSetAttribute(sample_rows_kernel<T>, cudaFuncAttributeMaxDynamicSharedMemorySize, smem);
    if (e != cudaSuccess) B200_FAIL(B200_ELAUNCH, "sample_rows_kernel attribute: %s", cudaGetErrorString(e));
    for (int i = 3; i > 0; --i) {
      cudaLaunchConfig_t cfg = {};
      cfg.gridDim = dim3(1u << i, 64);
      cfg.blockDim = dim3(ST);
      cfg.dynamicSmemBytes = smem;
      cudaLaunchAttribute attr;
      attr.id = cudaLaunchAttributeClusterDimension;
      attr.val.clusterDim.x = 1u << i;
      attr.val.clusterDim.y = attr.val.clusterDim.z = 1;
      cfg.attrs = &attr;
      cfg.numAttrs = 1;
      if (cudaOccupancyMaxActiveClusters(&wave->rows[i], sample_rows_kernel<T>, &cfg) != cudaSuccess) {
        cudaGetLastError();
        wave->rows[i] = 0;
      }
    }
    wave->rows[0] = 148;
  }
  // As many CTAs per row as all run at once; rows of a CTA that do not fit into its shared memory are read anew in each pass, which is less than a second
  // wave takes (us: 64 rows in fp32 with top-k 50 19 against 29, 128 in bf16 without filters 25 against 30).
  const auto seg_of = [&](int ctas) { return ceil_div(ceil_div(static_cast<int64_t>(p.cols), ctas), 256) * 256; };
  int log_ctas = 0;
  while (log_ctas < 3 && p.cols > (2048 << log_ctas) && rows <= wave->rows[log_ctas + 1]) ++log_ctas;
  // (sums of the weights stay small enough for a lane's counters: Weigher::Sum)
  while (log_ctas < 3 && seg_of(1 << log_ctas) > 1024 * ST) ++log_ctas;
  const int ctas = 1 << log_ctas;
  p.seg = static_cast<int>(seg_of(ctas));
  p.staged = p.seg * sizeof(T) <= STAGE_BYTES ? 1 : 0;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(static_cast<unsigned>(ctas), static_cast<unsigned>(rows));
  cfg.blockDim = dim3(ST);
  cfg.dynamicSmemBytes = BIN_BYTES + (p.staged ? static_cast<size_t>(p.seg) * sizeof(T) : 0);
  cfg.stream = st;
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
  cudaLaunchKernelEx(&cfg, sample_rows_kernel<T>, p);
  B200_CHECK_LAUNCH("sample_rows_kernel");
  return B200_OK;
}

}  // namespace

int sample_error(bool clear) {
  int v = 0;
  if (cudaMemcpyFromSymbol(&v, g_sample_error, sizeof(int)) != cudaSuccess) return -1;
  if (clear && v) {
    const int zero = 0;
    cudaMemcpyToSymbol(g_sample_error, &zero, sizeof(int));
  }
  return v;
}

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
  B200_DISPATCH_FLOAT(dtype, T, { return launch_sample<T>(p, rows, static_cast<cudaStream_t>(stream)); });
  return B200_OK;
}
