// Shared between the kernels of attention over a paged KV cache: arguments, how the work is dealt to blocks, and the partial results.
#pragma once
#include "common.cuh"

namespace b200 {

struct PagedParams {
  const void *q, *k_pages, *v_pages;
  void* out;                       // [token, Hq, D]
  const int32_t *q_start, *kv_len, *table;
  int64_t B, N, num_pages, table_stride;
  int64_t qs[2], ks[3];            // element strides: q over (token, head), pages over (page, head, row)
  int Hq, Hkv, G, page_size, page_shift;   // page_shift: log2 of the page size, negative where that is no power of two
  int64_t window;                  // keys a token sees back from its own (0: all)
  float scale;
  int whole;                       // items are not cut: a block takes those that begin in its range
  // partial results (paged_workspace)
  int4* head;                      // [PAGED_CTAS]: {pieces, first token, KV head, rows} of the item that begins in a block and ends in a later one
  float2* ml;                      // [PAGED_CTAS][2][rows]: (maximum in the log2 domain, sum)
  float* acc;                      // [PAGED_CTAS][2][rows][D], with tiles of 128 rows [PAGED_CTAS][2][D / 4][rows][4]
};

constexpr int PAGED_CTAS = 148;        // blocks that share the work (fixed, so that the workspace does not depend on the device)
constexpr int PAGED_MAX_SEQS = 4096;   // of a call: their running costs are kept in shared memory
constexpr int PAGED_MAX_PIECES = 32;   // of a block at a time

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

// ---- how the work is dealt out --------------------------------------------------------------------------------
// An item is (sequence, KV head, tile of `tpt` tokens): the tokens' G query heads of that KV head are the rows of one tile, row = token * G + head, so
// that keys and values are read once for all of them.  It costs its key tiles of KT keys plus OV for what it does once.  All items, one behind
// the other, are cut into equal ranges, one per block; a block's piece of an item that it does not have alone becomes a partial
// result.  Lengths are read on the device (a captured call follows them), every block works the cuts out for itself, and sequences
// of any lengths load all blocks alike.
struct PagedPiece {
  int32_t b, hk, token, tokens;   // sequence, KV head, first token (index into q) and how many
  int32_t p0, j0, cnt, flags;   // position of the first token, first key tile and number of them, 1: the item begins here, 2: it ends here
};

// (A block has these on its way to its first key, where a division by a number that only the caller knows is 0.05 to 0.2 us)
__device__ __forceinline__ int paged_page(const PagedParams& p, int key) { return p.page_shift >= 0 ? key >> p.page_shift : key / p.page_size; }
__device__ __forceinline__ int paged_tiles(int T, int tpt) { return T <= tpt ? (T > 0 ? 1 : 0) : (T + tpt - 1) / tpt; }
__device__ __forceinline__ int64_t paged_divide(int64_t a, int64_t b) {   // (neither is negative)
  return ((a | b) >> 32) == 0 ? static_cast<int64_t>(static_cast<uint32_t>(a) / static_cast<uint32_t>(b)) : a / b;
}

struct PagedTile { int t0, t1, j0, cnt; int64_t p0; };
template <int KT> __device__ __forceinline__ PagedTile paged_tile(const PagedParams& p, int T, int64_t n, int i, int tpt) {
  PagedTile t;
  t.t0 = i * tpt;
  t.t1 = min(T, t.t0 + tpt);
  t.p0 = n - T + t.t0;
  const int64_t hi = n - T + t.t1, lo = p.window > 0 && t.p0 - p.window + 1 > 0 ? t.p0 - p.window + 1 : 0;
  t.j0 = hi > lo ? static_cast<int>(lo / KT) : 0;
  t.cnt = hi > lo ? static_cast<int>((hi + KT - 1) / KT) - t.j0 : 1;   // no key: one tile in which everything is masked
  return t;
}

__device__ __forceinline__ int64_t warp_sum64(int64_t v) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
  return v;
}

// What every block keeps of the sequences while it looks for its pieces (shared memory)
struct PagedWork {
  int64_t* pre;        // [B + 1]: cost of the sequences before b
  int32_t *first, *n;  // [B]: first token, keys
  int32_t* T;          // [B]: tokens
};
constexpr int paged_work_bytes = PAGED_MAX_SEQS * 20 + 8;
__device__ __forceinline__ PagedWork paged_work(void* at, int seqs) {   // 20 bytes per sequence and 8
  PagedWork w;
  w.pre = static_cast<int64_t*>(at);
  w.first = reinterpret_cast<int32_t*>(w.pre + seqs + 1);
  w.n = w.first + seqs;
  w.T = w.n + seqs;
  return w;
}

// Fills `w`; returns pre[B].  All THREADS threads (up to 32 sequences: the first warp alone, the others get no answer); ends with a barrier
// (of the warp).
template <int KT, int OV, int THREADS> __device__ int64_t paged_prefix(const PagedParams& p, int tpt, const PagedWork& w, int64_t* warp_total) {
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, B = static_cast<int>(p.B);
  const int chunk = (B + THREADS - 1) / THREADS;
  if (B <= 32 && warp > 0) return 0;
  int64_t run = 0;
  for (int c = 0; c < chunk; ++c) {
    const int b = threadIdx.x * chunk + c;
    PagedSeq s = {0, 0, 0};
    if (b < B) {
      s = paged_seq(p, b);
      w.first[b] = static_cast<int>(s.first);
      w.n[b] = static_cast<int>(s.n);
      w.T[b] = s.T;
    }
    const int tiles = paged_tiles(s.T, tpt);
    int64_t cost = 0;
    if (tiles == 1) cost = paged_tile<KT>(p, s.T, s.n, 0, tpt).cnt + OV;
    // a prompt's many tiles: the whole warp adds them up
    for (unsigned many = __ballot_sync(0xffffffffu, tiles > 1); many; many &= many - 1) {
      const int src = __ffs(many) - 1, T = __shfl_sync(0xffffffffu, s.T, src), nt = (T + tpt - 1) / tpt;
      const int64_t n = __shfl_sync(0xffffffffu, s.n, src);
      int64_t sum = 0;
      for (int i = lane; i < nt; i += 32) sum += paged_tile<KT>(p, T, n, i, tpt).cnt + OV;
      sum = warp_sum64(sum);
      if (lane == src) cost = sum;
    }
    run += cost * p.Hkv;
    if (b < B) w.pre[b + 1] = run;
  }
  int64_t upto = run;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const int64_t t = __shfl_up_sync(0xffffffffu, upto, o);
    if (lane >= o) upto += t;
  }
  if (B <= 32) {
    if (lane < B) w.pre[lane + 1] = upto;
    if (lane == 0) w.pre[0] = 0;
    __syncwarp();
    return __shfl_sync(0xffffffffu, upto, 31);
  }
  if (lane == 31) warp_total[warp] = upto;
  __syncthreads();
  int64_t before = upto - run, total = 0;
#pragma unroll
  for (int v = 0; v < THREADS / 32; ++v) {
    if (v < warp) before += warp_total[v];
    total += warp_total[v];
  }
  for (int c = 0; c < chunk; ++c) {
    const int b = threadIdx.x * chunk + c;
    if (b < B) w.pre[b + 1] += before;
  }
  if (threadIdx.x == 0) w.pre[0] = 0;
  __syncthreads();
  return total;
}

// The pieces of items in the costs [u0, u1), at most PAGED_MAX_PIECES; returns where to go on (u1: that was all).  One whole warp.
// head is written where an item begins in this block and does not end in it: whose rows they are, and (ends) where it ends.
template <int KT, int OV>
__device__ int64_t paged_pieces(const PagedParams& p, int tpt, const PagedWork& w, int64_t u0, int64_t u1, PagedPiece* list, int& count, int4& head, int64_t& ends) {
  const int lane = threadIdx.x & 31, B = static_cast<int>(p.B);
  count = 0;
  int lo = 0, hi = B;   // the last sequence that begins at or before u0 (and so is not empty)
  while (hi - lo > 1) {
    const int mid = (lo + hi) >> 1;
    if (w.pre[mid] <= u0) lo = mid; else hi = mid;
  }
  for (int b = lo; b < B && w.pre[b] < u1; ++b) {
    const int64_t begin = w.pre[b], all = w.pre[b + 1] - begin;
    if (begin + all <= u0 || all == 0) continue;
    const int T = w.T[b], first = w.first[b], tiles = paged_tiles(T, tpt);
    const int64_t n = w.n[b];
    int skip = 0;   // heads ahead of u0
    int64_t base = begin;
    if (u0 > begin && p.Hkv > 1) {
      const int64_t per_head = tiles == 1 ? paged_tile<KT>(p, T, n, 0, tpt).cnt + OV : paged_divide(all, p.Hkv), off = u0 - begin;
      skip = p.Hkv <= 32 ? __popc(__ballot_sync(0xffffffffu, lane < p.Hkv && (lane + 1) * per_head <= off)) : static_cast<int>(paged_divide(off, per_head));
      base += skip * per_head;
    }
    const int items = p.Hkv * tiles;
    for (int e0 = skip * tiles; e0 < items && base < u1; e0 += 32) {
      const int e = e0 + lane, h = tiles == 1 ? e : e / tiles;
      PagedTile t = {0, 0, 0, 0, 0};
      if (e < items) t = paged_tile<KT>(p, T, n, e - h * tiles, tpt);
      const int64_t cost = e < items ? t.cnt + OV : 0;
      int64_t upto = cost;
      if (tiles == 1) {   // (all items of a decoding sequence cost the same)
        upto = static_cast<int64_t>(min(lane + 1, items - e0)) * __shfl_sync(0xffffffffu, t.cnt + OV, 0);
      } else {
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
          const int64_t v = __shfl_up_sync(0xffffffffu, upto, o);
          if (lane >= o) upto += v;
        }
      }
      const int64_t start = base + upto - cost + OV, end = base + upto;
      const bool here = start >= u0 && start < u1;
      const int64_t a = p.whole ? start : u0 > start ? u0 : start, z = p.whole ? (here ? end : start) : u1 < end ? u1 : end;
      const unsigned mine = __ballot_sync(0xffffffffu, e < items && a < z);
      const int at = count + __popc(mine & ((1u << lane) - 1u));
      const bool taken = ((mine >> lane) & 1u) && at < PAGED_MAX_PIECES;
      if (taken) {
        PagedPiece f;
        f.b = b;
        f.hk = h;
        f.token = first + t.t0;
        f.tokens = t.t1 - t.t0;
        f.p0 = static_cast<int>(t.p0);
        f.j0 = t.j0 + static_cast<int>(a - start);
        f.cnt = static_cast<int>(z - a);
        f.flags = (a == start ? 1 : 0) | (z == end ? 2 : 0);
        list[at] = f;
      }
      // (at most one per block, and the last of its pieces)
      const unsigned opens = __ballot_sync(0xffffffffu, taken && a == start && z < end);
      if (opens) {
        const int src = __ffs(opens) - 1;
        ends = __shfl_sync(0xffffffffu, end, src);
        head.x = 1;
        head.y = __shfl_sync(0xffffffffu, first + t.t0, src);
        head.z = __shfl_sync(0xffffffffu, h, src);
        head.w = __shfl_sync(0xffffffffu, (t.t1 - t.t0) * p.G, src);
      }
      count += __popc(mine);
      if (count > PAGED_MAX_PIECES) {   // go on behind the last one taken
        const unsigned last = __ballot_sync(0xffffffffu, taken && at == PAGED_MAX_PIECES - 1);
        count = PAGED_MAX_PIECES;
        return last ? __shfl_sync(0xffffffffu, p.whole ? start + 1 : z, __ffs(last) - 1) : base;   // (none of these 32 was taken: they begin at base or later)
      }
      base += __shfl_sync(0xffffffffu, upto, 31);
    }
  }
  return u1;
}

// Where a piece's partial result goes: slot 1 for the one that an item begins with, slot 0 for the others.
__device__ __forceinline__ int64_t paged_slot(int cta, bool begins, int rows_max) { return (static_cast<int64_t>(cta) * 2 + (begins ? 1 : 0)) * rows_max; }

// tcgen05 kernel (attn_paged_tc5.cu); B200_ENOTSUP where a tensor map cannot be made
int attn_paged_tc5(const PagedParams& p, int D, int dtype, cudaStream_t stream);
int attn_paged_tc5_error(bool clear);
// code left by a bounded wait of either kernel that ran out (0 = none); optionally cleared
int attn_paged_error(bool clear);

constexpr int PAGED_TC5_ROWS = 128;

}  // namespace b200
