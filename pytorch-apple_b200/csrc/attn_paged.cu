// Attention of every sequence's new tokens over the pages of its KV cache: the kernel for few rows per KV head (decoding sequences, a few
// drafted tokens), the one that joins partial results, and the entry point.  Chunks and prompts: attn_paged_tc5.cu.
#include "attn_paged.cuh"
#include "gemm_tc5.cuh"
#include "mma.cuh"
#include "tc5.cuh"

namespace b200 {

namespace {

constexpr float LOG2E = 1.4426950408889634f;

// ===========================================================================
// Few rows: up to 8 NT rows (tokens times query heads) share each KV head.  The problem is transposed so that the rows lie on the
// 8-wide side of the m16n8k16 MMA (mma.sync: at 4 flop per byte and row this is bound by memory):
//   S^T[16 keys x 8 rows] = K[16 x D] Q^T,   O^T[D x 8 rows] += V^T[D x 16] P^T.
// A block of eight warps walks through its pieces (attn_paged.cuh) with a warp per 16 keys; every warp has a ring of its own
// in shared memory, filled by TMA (one box of 16 rows of a page each for K and V, 128-byte swizzle), so that nothing in the loop
// waits for another warp.  At the end of a piece each warp parks its accumulators in the ring stage that it has just read (which is
// refilled afterwards; the others are on their way meanwhile) and the block adds them up.
//
// us: one sequence of 613 keys 8.4 (launch 2.3, lengths and pages 3, keys 2, sums 1), of 20001 keys 10.9; 64 of 512 to 4352 keys 28.5, of which 17 are the
// keys at 6.5 TB/s, 4.3 what precedes the first copy and 4.5 the joining kernel.  A warp has 24 KB on its way, 196 KB per SM.
//
// Probabilities are rounded to the activation type, which the MMA takes (sums are of the unrounded ones, in fp32): against 64 bits the output is off by 0.22 % in bf16
// (root mean square), 0.16 of which is its own rounding.  At 18 % of the issue slots the MMAs are not the bound, but two for each would lengthen the chain per block of keys.
// ===========================================================================
constexpr int FEW_WARPS = 8, FEW_KEYS = 16;
// What an item costs besides its 16-key blocks, in blocks (a round of the eight warps is eight).  us at 4 / 8 / 16 / 28: 64 ragged sequences 29.6 / 29.1 / 28.6 / 28.1,
// 200 of 100 to 1500 keys 34.3 / 33.4 / 30.5 / 29.6, one of 2000 10.9 / 10.1 / 9.1 / 10.7, eight of 500 to 8000 12.5 / 11.6 / 10.3 / 11.5, eight of 4097 11.9 / 13.9 / 12.8 / 12.0.
constexpr int FEW_OV = 16;
constexpr int FEW_MIN_SHARE = 16;  // blocks (and OVs) of a CTA at least
constexpr float FEW_STEP = 8.f;    // the stored maximum follows the true one when that has grown by more (log2)
constexpr int FEW_RING = 24576;    // bytes of a warp's ring

__device__ int g_few_error = 0;    // left by a bounded wait that ran out

template <typename T, int D, int NT>
__global__ void __launch_bounds__(FEW_WARPS * 32, 1)
    attn_paged_few_kernel(const __grid_constant__ CUtensorMap map_k, const __grid_constant__ CUtensorMap map_v, const __grid_constant__ PagedParams p, const int tpt) {
  constexpr int BLOCK = 2 * FEW_KEYS * D * 2, HALF = BLOCK / 2, STAGES = FEW_RING / BLOCK;   // 16 keys of K and of V
  constexpr int ROWS = 8 * NT, KS = D / 16;
  extern __shared__ uint8_t smem_raw[];
  uint8_t* const smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~static_cast<uintptr_t>(1023));
  __shared__ __align__(8) uint64_t full[FEW_WARPS][STAGES];
  __shared__ __align__(16) PagedPiece s_piece[PAGED_MAX_PIECES];
  __shared__ int s_first[PAGED_MAX_PIECES + 1];   // blocks ahead of each piece of the list
  __shared__ float s_m[FEW_WARPS][ROWS], s_l[FEW_WARPS][ROWS];
  __shared__ int s_park[FEW_WARPS];               // where a warp has parked its accumulators (ring stage, -1: it has none)
  __shared__ int64_t s_total[FEW_WARPS], s_small[(32 * 20 + 8) / 8];
  __shared__ int s_count, s_more;

  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, g = lane >> 2, t = lane & 3, cta = blockIdx.x;
  uint8_t* const ring = smem + warp * FEW_RING;
  if (lane == 0) {
    for (int s = 0; s < STAGES; ++s) tc5::mbar_init(&full[warp][s], 1);
    tc5::fence_barrier_init();
  }
  if (threadIdx.x == 0) { tc5::prefetch_tensormap(&map_k); tc5::prefetch_tensormap(&map_v); }
  pdl_trigger();
  pdl_wait();   // lengths, pages, queries and cache rows come from earlier kernels
  const bool small = p.B <= 32;   // the first warp's own matter (paged_prefix), in a place of its own; others lie over the rings, which are still empty
  const PagedWork work = small ? paged_work(s_small, 32) : paged_work(smem, PAGED_MAX_SEQS);
  int64_t u0 = 0, u1 = 0, share = 1, ends = 0;
  auto deal = [&]() {   // this block's range of costs (as far as it is known to this warp)
    const int64_t total = paged_prefix<FEW_KEYS, FEW_OV, FEW_WARPS * 32>(p, tpt, work, s_total);
    const int64_t even = (total + PAGED_CTAS - 1) / PAGED_CTAS;
    share = even > FEW_MIN_SHARE ? even : FEW_MIN_SHARE;
    u1 = (cta + 1) * share < total ? (cta + 1) * share : total;
  };
  deal();
  u0 = cta * share;
  int4 head = make_int4(0, 0, 0, 0);
  const float sl = p.scale * LOG2E;
  uint32_t phase = 0;   // parity of each stage's next completion
  int st = 0;           // stage of the next block to be read
  uint32_t patience = 1u << 22;

  // ldmatrix: lane supplies one row address of 8x8 matrix (lane >> 3); a panel holds 64 dims of 16 rows, chunk c of row r at c ^ (r & 7)
  const int mi = lane >> 3, mr = lane & 7;
  const uint32_t ring_addr = smem_u32(ring);
  const uint32_t k_row = (8 * (mi & 1) + mr) * 128, v_row = (8 * (mi >> 1) + mr) * 128;

  while (true) {
    if (warp == 0) {
      int count = 0;
      if (u0 < u1) u0 = paged_pieces<FEW_KEYS, FEW_OV>(p, tpt, work, u0, u1, s_piece, count, head, ends);
      __syncwarp();
      if (lane == 0) {
        s_more = u0 < u1;
        s_count = count;
        int run = 0;
        for (int f = 0; f < count; ++f) { s_first[f] = run; run += s_piece[f].cnt; }
        s_first[count] = run;
      }
    }
    __syncthreads();
    const int F = s_count;
    const bool more = s_more;
    if (F == 0) break;   // (a range that no item begins or goes on in)
    const int X = s_first[F];

    // Copies: block x of the list is warp x % 8's; its page and row are looked up 32 blocks ahead, one per lane
    int id_page = 0, id_row = 0, id_hk = 0, next_page = 0, next_row = 0, next_hk = 0;
    auto look = [&](int x, int& page, int& row, int& hk) {
      page = row = hk = 0;
      if (x < X) {
        int f = 0;
        while (x >= s_first[f + 1]) ++f;
        const int key = (s_piece[f].j0 + x - s_first[f]) * FEW_KEYS, i = paged_page(p, key);
        row = key - i * p.page_size;
        hk = s_piece[f].hk;
        const int hi = s_piece[f].p0 + s_piece[f].tokens;
        page = key < hi ? __ldg(p.table + s_piece[f].b * p.table_stride + i) : -1;   // (an item without keys has no page either)
        if (page < 0 || page >= p.num_pages) page = static_cast<int>(p.num_pages);   // outside the tensor: zeros
      }
    };
    int x_copy = warp, st_copy = st;   // next block to be copied, and into which stage
    auto copy = [&]() {
      const int i = (x_copy / FEW_WARPS) & 31;
      if (i == 0 && x_copy >= FEW_WARPS * 32) { id_page = next_page; id_row = next_row; id_hk = next_hk; }
      if (i == 0) look(x_copy + FEW_WARPS * (32 + lane), next_page, next_row, next_hk);
      const int page = __shfl_sync(0xffffffffu, id_page, i), row = __shfl_sync(0xffffffffu, id_row, i), hk = __shfl_sync(0xffffffffu, id_hk, i);
      if (lane == 0 && x_copy < X) {
        uint64_t* const bar = &full[warp][st_copy];
        tc5::mbar_arrive_expect_tx(bar, BLOCK);
        tc5::tma_load_5d(ring + st_copy * BLOCK, &map_k, bar, 0, row, 0, hk, page);
        tc5::tma_load_5d(ring + st_copy * BLOCK + HALF, &map_v, bar, 0, row, 0, hk, page);
      }
      x_copy += FEW_WARPS;
      st_copy = st_copy + 1 == STAGES ? 0 : st_copy + 1;
    };
    look(warp + FEW_WARPS * lane, id_page, id_row, id_hk);
    if (!small) {
      tc5::fence_proxy_async();
      __syncthreads();   // (everybody is through with the running costs)
    }
    for (int s = 0; s < STAGES; ++s) copy();

    // Q^T fragments: row 8 j + g, dims 16 ks + 2 t, +1 and 16 ks + 2 t + 8, +9
    uint32_t qf[KS][NT][2];
    auto load_q = [&](const PagedPiece& c) {
      const int rows = c.tokens * p.G;
#pragma unroll
      for (int j = 0; j < NT; ++j) {
        const int r = 8 * j + g;
        const T* qr = static_cast<const T*>(p.q) + (static_cast<int64_t>(c.token) + r / p.G) * p.qs[0] + (c.hk * p.G + r % p.G) * p.qs[1] + 2 * t;
#pragma unroll
        for (int ks = 0; ks < KS; ++ks) {
          qf[ks][j][0] = r < rows ? *reinterpret_cast<const uint32_t*>(qr + 16 * ks) : 0u;
          qf[ks][j][1] = r < rows ? *reinterpret_cast<const uint32_t*>(qr + 16 * ks + 8) : 0u;
        }
      }
    };
    load_q(s_piece[0]);
    int x = warp;   // this warp's next block
#pragma unroll 1
    for (int f = 0; f < F; ++f) {
      const PagedPiece c = s_piece[f];
      const int rows = c.tokens * p.G, hi = c.p0 + c.tokens;   // keys from here on nobody sees
      const int lo = p.window > 0 && c.p0 - p.window + 1 > 0 ? static_cast<int>(c.p0 - p.window + 1) : 0;
      const int x_end = s_first[f + 1], key_base = (c.j0 - s_first[f]) * FEW_KEYS;
      float m[NT][2], l[NT][2], o[KS][NT][4];
#pragma unroll
      for (int j = 0; j < NT; ++j) m[j][0] = m[j][1] = -INFINITY, l[j][0] = l[j][1] = 0.f;
      int parked = -1;
      if (x < x_end) {
        // rows 8 j + 2 t, + 1 are this lane's columns of S^T; their keys end before see and begin at from
        int see[NT][2], from[NT][2], see_min = hi, from_max = lo;
#pragma unroll
        for (int j = 0; j < NT; ++j)
#pragma unroll
          for (int e = 0; e < 2; ++e) {
            const int r = 8 * j + 2 * t + e;
            see[j][e] = r < rows ? c.p0 + r / p.G + 1 : hi;
            from[j][e] = p.window > 0 && see[j][e] - p.window > 0 ? static_cast<int>(see[j][e] - p.window) : 0;
            see_min = min(see_min, see[j][e]);
            from_max = max(from_max, from[j][e]);
          }
#pragma unroll
        for (int ks = 0; ks < KS; ++ks)
#pragma unroll
          for (int j = 0; j < NT; ++j) o[ks][j][0] = o[ks][j][1] = o[ks][j][2] = o[ks][j][3] = 0.f;

#pragma unroll 1
        while (true) {
          const int key0 = key_base + x * FEW_KEYS;
          const uint32_t sk = ring_addr + st * BLOCK, sv = sk + HALF;
          if (!tc5::mbar_wait(&full[warp][st], (phase >> st) & 1u, patience)) {   // (a copy that never comes: the result is void, nothing hangs)
            patience = 1u << 10;
            if (lane == 0) atomicExch(&g_few_error, 60);
          }
          phase ^= 1u << st;
          if (key0 + FEW_KEYS > hi || key0 < lo) {   // clear the rows of V that no row sees
            const int row = lane >> 1, key = key0 + row;
            if (key >= hi || key < lo) {
              uint4* const v = reinterpret_cast<uint4*>(ring + st * BLOCK + HALF + (D == 128 ? (lane & 1) * 2048 + row * 128 : row * 128 + (lane & 1) * 64));
#pragma unroll
              for (int e = 0; e < D / 16; ++e) v[e] = make_uint4(0, 0, 0, 0);
            }
            tc5::fence_proxy_async();   // before the stage is copied into again
            __syncwarp();
          }
          // ---- S^T = K Q^T (two accumulators halve the dependent chain) ----
          float sa[NT][4], sb[NT][4];
#pragma unroll
          for (int j = 0; j < NT; ++j)
#pragma unroll
            for (int e = 0; e < 4; ++e) sa[j][e] = sb[j][e] = 0.f;
#pragma unroll
          for (int ks = 0; ks < KS; ks += 2) {
            uint32_t a0[4], a1[4];
            ldmatrix_x4(a0, sk + (ks >> 2) * 2048 + k_row + (((2 * (ks & 3) + (mi >> 1)) ^ mr) << 4));
            ldmatrix_x4(a1, sk + (ks >> 2) * 2048 + k_row + (((2 * (ks & 3) + 2 + (mi >> 1)) ^ mr) << 4));
#pragma unroll
            for (int j = 0; j < NT; ++j) {
              MmaType<T>::mma(sa[j], a0, qf[ks][j]);
              MmaType<T>::mma(sb[j], a1, qf[ks + 1][j]);
            }
          }
          float v[NT][4];   // keys g (0, 1) and g + 8 (2, 3) x rows 8 j + 2 t (0, 2) and + 1 (1, 3)
#pragma unroll
          for (int j = 0; j < NT; ++j)
#pragma unroll
            for (int e = 0; e < 4; ++e) v[j][e] = (sa[j][e] + sb[j][e]) * sl;
          if (key0 + FEW_KEYS > see_min || key0 < from_max) {
#pragma unroll
            for (int j = 0; j < NT; ++j)
#pragma unroll
              for (int e = 0; e < 4; ++e) {
                const int key = key0 + g + (e >> 1) * 8;
                if (key >= see[j][e & 1] || key < from[j][e & 1]) v[j][e] = -INFINITY;
              }
          }
          // ---- the running maximum moves only when some score has outgrown it ----
          bool grown = false;
#pragma unroll
          for (int j = 0; j < NT; ++j)
#pragma unroll
            for (int e = 0; e < 4; ++e) grown = grown || v[j][e] > m[j][e & 1] + FEW_STEP || (m[j][e & 1] == -INFINITY && v[j][e] > -INFINITY);
          if (__any_sync(0xffffffffu, grown)) {
#pragma unroll
            for (int j = 0; j < NT; ++j) {
              float mx[2] = {fmaxf(v[j][0], v[j][2]), fmaxf(v[j][1], v[j][3])};
#pragma unroll
              for (int off = 4; off < 32; off <<= 1) {
                mx[0] = fmaxf(mx[0], __shfl_xor_sync(0xffffffffu, mx[0], off));
                mx[1] = fmaxf(mx[1], __shfl_xor_sync(0xffffffffu, mx[1], off));
              }
#pragma unroll
              for (int e = 0; e < 2; ++e) {
                const float mn = fmaxf(m[j][e], mx[e]), f_ = ex2_approx(m[j][e] - (mn == -INFINITY ? 0.f : mn));
                m[j][e] = mn;
                l[j][e] *= f_;
#pragma unroll
                for (int ks = 0; ks < KS; ++ks) { o[ks][j][e] *= f_; o[ks][j][e + 2] *= f_; }
              }
            }
          }
          // ---- O^T += V^T P^T ----
          uint32_t pb[NT][2];
#pragma unroll
          for (int j = 0; j < NT; ++j) {
            const float u0_ = m[j][0] == -INFINITY ? 0.f : m[j][0], u1_ = m[j][1] == -INFINITY ? 0.f : m[j][1];
            const float p0 = ex2_approx(v[j][0] - u0_), p1 = ex2_approx(v[j][1] - u1_), p2 = ex2_approx(v[j][2] - u0_), p3 = ex2_approx(v[j][3] - u1_);
            l[j][0] += p0 + p2;
            l[j][1] += p1 + p3;
            pb[j][0] = movmatrix_trans(pack2<T>(p0, p1));
            pb[j][1] = movmatrix_trans(pack2<T>(p2, p3));
          }
#pragma unroll
          for (int ks = 0; ks < KS; ++ks) {
            uint32_t a[4];
            ldmatrix_x4_trans(a, sv + (ks >> 2) * 2048 + v_row + (((2 * (ks & 3) + (mi & 1)) ^ mr) << 4));
#pragma unroll
            for (int j = 0; j < NT; ++j) MmaType<T>::mma(o[ks][j], a, pb[j]);
          }
          __syncwarp();   // every lane has read the stage
          x += FEW_WARPS;
          const int was = st;
          st = st + 1 == STAGES ? 0 : st + 1;
          if (x >= x_end) { parked = was; break; }
          copy();
        }
        if (f + 1 < F) load_q(s_piece[f + 1]);   // (on its way while this piece's sums are added up)
#pragma unroll
        for (int j = 0; j < NT; ++j)
#pragma unroll
          for (int off = 4; off < 32; off <<= 1) {
            l[j][0] += __shfl_xor_sync(0xffffffffu, l[j][0], off);
            l[j][1] += __shfl_xor_sync(0xffffffffu, l[j][1], off);
          }
        // [row][D] floats, dim d of row r at d ^ (r's 2 t and j) * 8: lanes that differ in t store to other banks
        float* const slab = reinterpret_cast<float*>(ring + parked * BLOCK);
#pragma unroll
        for (int ks = 0; ks < KS; ++ks)
#pragma unroll
          for (int j = 0; j < NT; ++j)
#pragma unroll
            for (int e = 0; e < 4; ++e) {
              const int r = 8 * j + 2 * t + (e & 1);
              slab[r * D + ((16 * ks + g + (e >> 1) * 8) ^ (t << 3))] = o[ks][j][e];
            }
        if (g == 0) {
#pragma unroll
          for (int j = 0; j < NT; ++j)
#pragma unroll
            for (int e = 0; e < 2; ++e) { s_m[warp][8 * j + 2 * t + e] = m[j][e]; s_l[warp][8 * j + 2 * t + e] = l[j][e]; }
        }
      }
      if (parked < 0 && f + 1 < F) load_q(s_piece[f + 1]);
      if (lane == 0) s_park[warp] = parked;
      __syncthreads();
      // ---- the block's sums: a thread per four dims of a row ----
      {
        constexpr int LPR = D / 4;
        const int d = threadIdx.x % LPR * 4;
        const bool whole = c.flags == 3;
        const int64_t slot = paged_slot(cta, c.flags & 1, ROWS);
        for (int r = threadIdx.x / LPR; r < rows; r += FEW_WARPS * 32 / LPR) {
          float mw[FEW_WARPS], top = -INFINITY;
          float4 a[FEW_WARPS];
#pragma unroll
          for (int w = 0; w < FEW_WARPS; ++w) {
            const int at = s_park[w];
            mw[w] = at >= 0 ? s_m[w][r] : -INFINITY;
            a[w] = at >= 0 ? *reinterpret_cast<const float4*>(smem + w * FEW_RING + at * BLOCK + (r * D + (d ^ (((r & 7) >> 1) << 3))) * 4) : make_float4(0.f, 0.f, 0.f, 0.f);
            top = fmaxf(top, mw[w]);
          }
          const float ref = top == -INFINITY ? 0.f : top;
          float4 acc = make_float4(0.f, 0.f, 0.f, 0.f);
          float sum = 0.f;
#pragma unroll
          for (int w = 0; w < FEW_WARPS; ++w) {
            const float f_ = ex2_approx(mw[w] - ref);
            acc.x += a[w].x * f_; acc.y += a[w].y * f_; acc.z += a[w].z * f_; acc.w += a[w].w * f_;
            sum += s_park[w] >= 0 ? s_l[w][r] * f_ : 0.f;
          }
          if (whole) {   // (a row without keys gives zeros)
            const float inv = sum > 0.f ? 1.f / sum : 0.f;
            *reinterpret_cast<uint2*>(static_cast<T*>(p.out) + ((static_cast<int64_t>(c.token) + r / p.G) * p.Hq + c.hk * p.G + r % p.G) * D + d) =
                make_uint2(pack2<T>(acc.x * inv, acc.y * inv), pack2<T>(acc.z * inv, acc.w * inv));
          } else {
            *reinterpret_cast<float4*>(p.acc + (slot + r) * D + d) = acc;
            if (d == 0) p.ml[slot + r] = make_float2(top, sum);
          }
        }
      }
      tc5::fence_proxy_async();   // what was parked, ahead of the copies into the same stages
      __syncthreads();
      if (parked >= 0) copy();
    }
    if (!more) break;
    deal();   // (the rings lay over the running costs)
  }
  if (threadIdx.x == 0 && !p.whole) {
    if (head.x) head.x = static_cast<int>(paged_divide(ends - 1, share)) - cta + 1;   // blocks with pieces of the item that begins here and ends in another
    p.head[cta] = head;
  }
}

// ===========================================================================
// Joins the pieces of the item that begins in block blockIdx.x of the kernel before and goes on in the next ones, in the order of the blocks (their
// sums are the same whoever adds them up).  Bound by latency: the wait for the kernel before, the item, then its pieces (3 to 5 us).
//
// Few rows: row blockIdx.y, a thread per four dims, the pieces dealt to the 256 / (D / 4)ths of the block, so that a thread's chain of loads stays short
// (71 pieces: 17.2 us with a thread per piece and dim).
// ===========================================================================
struct PagedSum {   // of a thread's four dims: relative to m
  float m = -INFINITY, l = 0.f;
  float4 acc = {0.f, 0.f, 0.f, 0.f};
  // pieces first, first + step, .. of `pieces`, BATCH of them under way; read(piece, ml, acc) fetches one
  template <int BATCH, typename F> __device__ __forceinline__ void add(int first, int step, int pieces, F&& read) {
    for (int i0 = first; i0 < pieces; i0 += BATCH * step) {
      float2 ml[BATCH];
      float4 a[BATCH];
#pragma unroll
      for (int i = 0; i < BATCH; ++i) {
        ml[i] = make_float2(-INFINITY, 0.f);
        a[i] = make_float4(0.f, 0.f, 0.f, 0.f);
        if (i0 + i * step < pieces) read(i0 + i * step, ml[i], a[i]);
      }
      float top = m;
#pragma unroll
      for (int i = 0; i < BATCH; ++i) top = fmaxf(top, ml[i].x);
      const float ref = top == -INFINITY ? 0.f : top, c = ex2_approx(m - ref);
      l *= c; acc.x *= c; acc.y *= c; acc.z *= c; acc.w *= c;
#pragma unroll
      for (int i = 0; i < BATCH; ++i) {
        const float f = ex2_approx(ml[i].x - ref);
        l += ml[i].y * f;
        acc.x += a[i].x * f; acc.y += a[i].y * f; acc.z += a[i].z * f; acc.w += a[i].w * f;
      }
      m = top;
    }
  }
  template <typename T> __device__ __forceinline__ uint2 result() const {   // (no key: zeros; a sum that is no number stays none)
    const float inv = l == 0.f ? 0.f : 1.f / l;
    return make_uint2(pack2<T>(acc.x * inv, acc.y * inv), pack2<T>(acc.z * inv, acc.w * inv));
  }
};

template <typename T, int D, int ROWS>
__global__ void __launch_bounds__(256) attn_paged_merge_kernel(const __grid_constant__ PagedParams p) {
  constexpr int LPR = D / 4, GROUPS = 256 / LPR;
  __shared__ float4 s_acc[GROUPS][LPR];
  __shared__ float2 s_ml[GROUPS];
  pdl_trigger();
  pdl_wait();
  const int4 it = __ldg(p.head + blockIdx.x);
  const int g = threadIdx.x / LPR, c = threadIdx.x % LPR, r = blockIdx.y;
  if (it.x == 0 || r >= it.w) return;
  PagedSum sum;
  sum.add<10>(g, GROUPS, it.x, [&](int piece, float2& ml, float4& a) {
    const int64_t slot = paged_slot(blockIdx.x + piece, piece == 0, ROWS) + r;
    ml = __ldg(p.ml + slot);
    a = __ldg(reinterpret_cast<const float4*>(p.acc + slot * D) + c);
  });
  s_acc[g][c] = sum.acc;
  if (c == 0) s_ml[g] = make_float2(sum.m, sum.l);
  __syncthreads();
  if (threadIdx.x >= LPR) return;
  PagedSum all;
  all.add<GROUPS>(0, 1, GROUPS, [&](int e, float2& ml, float4& a) { ml = s_ml[e]; a = s_acc[e][c]; });
  *reinterpret_cast<uint2*>(static_cast<T*>(p.out) + ((static_cast<int64_t>(it.y) + r / p.G) * p.Hq + it.z * p.G + r % p.G) * D + c * 4) = all.result<T>();
}

// Tiles of 128 rows, whose sums lie as [D / 4][rows] of four each: 1024 / D rows from blockIdx.y * (1024 / D) on, a thread per row and four dims.  Many pieces too
// (a few tokens over a very long history): eight threads to share them, with a barrier per eighth of the dims, took 46 against 34 us for 128 tokens over 20000
// keys, 34 against 28 for 21 over 30000; eight pieces on their way instead of four 35 and 29.
template <typename T, int D>
__global__ void __launch_bounds__(256) attn_paged_merge_rows_kernel(const __grid_constant__ PagedParams p) {
  constexpr int LPR = D / 4, RPB = 256 / LPR, ROWS = PAGED_TC5_ROWS;
  pdl_trigger();
  pdl_wait();
  const int4 it = __ldg(p.head + blockIdx.x);
  const int r = blockIdx.y * RPB + threadIdx.x % RPB, c = threadIdx.x / RPB;
  if (it.x == 0 || r >= it.w) return;
  PagedSum sum;
  sum.add<4>(0, 1, it.x, [&](int piece, float2& ml, float4& a) {
    const int64_t slot = paged_slot(blockIdx.x + piece, piece == 0, ROWS);
    ml = __ldg(p.ml + slot + r);
    a = __ldg(reinterpret_cast<const float4*>(p.acc + slot * D) + c * ROWS + r);
  });
  *reinterpret_cast<uint2*>(static_cast<T*>(p.out) + ((static_cast<int64_t>(it.y) + r / p.G) * p.Hq + it.z * p.G + r % p.G) * D + c * 4) = sum.result<T>();
}

// ===========================================================================
// Where the tensor-core kernels are switched off (or a tensor map cannot be made): one warp per (token, query head), one key at a time.
// ===========================================================================
template <typename T, int D>
__global__ void __launch_bounds__(128) attn_paged_plain_kernel(const __grid_constant__ PagedParams p) {
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
  for (int e = 0; e < E; ++e) out[e] = from_f32<T>(l == 0.f ? 0.f : o[e] / l);
}

template <typename T, int D, int NT> int launch_few(const PagedParams& p, int dtype, cudaStream_t st) {
  constexpr int smem = FEW_WARPS * FEW_RING + 1024;
  static PerDevice<bool> configured_on;
  bool* configured = configured_on.slot();
  if (!configured) return B200_ENOTSUP;
  if (!*configured) {
    if (cudaFuncSetAttribute(attn_paged_few_kernel<T, D, NT>, cudaFuncAttributeMaxDynamicSharedMemorySize, smem) != cudaSuccess) {
      cudaGetLastError();
      return B200_ENOTSUP;
    }
    *configured = true;
  }
  CUtensorMap mk, mv;
  auto bytes = [](int64_t elems) { return elems > 0 ? static_cast<uint64_t>(elems) * 2 : static_cast<uint64_t>(D) * 2; };   // (0: an axis of length one)
  const uint64_t dims[5] = {64, static_cast<uint64_t>(p.page_size), D / 64, static_cast<uint64_t>(p.Hkv), static_cast<uint64_t>(p.num_pages)};
  const uint64_t str[4] = {bytes(p.ks[2]), 128, bytes(p.ks[1]), bytes(p.ks[0])};
  const uint32_t box[5] = {64, FEW_KEYS, D / 64, 1, 1};
  if (!tma_encode_sw128(&mk, dtype, 5, p.k_pages, dims, str, box) || !tma_encode_sw128(&mv, dtype, 5, p.v_pages, dims, str, box)) return B200_ENOTSUP;
  return launch_pdl(attn_paged_few_kernel<T, D, NT>, dim3(PAGED_CTAS), dim3(FEW_WARPS * 32), smem, st, mk, mv, p, 8 * NT / p.G) == cudaSuccess ? B200_OK : B200_ELAUNCH;
}

// rows per KV head of the kernel that takes a call
int rows_of(int64_t max_q, int G) {
  if (G <= 8 && max_q * G <= 8) return 8;
  if (G <= 16 && max_q * G <= 16) return 16;
  return PAGED_TC5_ROWS;
}

int64_t workspace_parts(int rows, int D, int64_t* ml, int64_t* acc) {   // byte offsets of the arrays; returns the size
  *ml = PAGED_CTAS * 16;
  *acc = *ml + static_cast<int64_t>(PAGED_CTAS) * 2 * rows * 8;
  return *acc + static_cast<int64_t>(PAGED_CTAS) * 2 * rows * D * 4;
}

}  // namespace

int attn_paged_error(bool clear) {
  int v = 0;
  if (cudaMemcpyFromSymbol(&v, g_few_error, sizeof(int)) != cudaSuccess) return -1;
  if (clear && v) {
    const int zero = 0;
    cudaMemcpyToSymbol(g_few_error, &zero, sizeof(int));
  }
  const int other = attn_paged_tc5_error(clear);
  return v ? v : other;
}

}  // namespace b200

using namespace b200;

extern "C" int64_t b200_attn_paged_workspace_bytes(int64_t max_q, int Hq, int Hkv, int D) {
  if (max_q <= 0 || Hq <= 0 || Hkv <= 0 || D <= 0) return 0;
  int64_t ml, acc;
  return workspace_parts(rows_of(max_q, Hq / Hkv), D, &ml, &acc);
}

extern "C" int b200_attn_paged(const b200_attn_paged_args* args, void* stream) {
  B200_CHECK_ARG(args, "b200_attn_paged: bad arguments");
  const b200_attn_paged_args& a = *args;
  const int Hq = a.Hq, Hkv = a.Hkv, D = a.D, dtype = a.dtype;
  B200_CHECK_ARG(a.q && a.k_pages && a.v_pages && a.out && a.q_start && a.kv_len && a.page_table && a.B >= 0 && a.n_tokens >= 0 && a.max_q >= 0 &&
                 Hq > 0 && Hkv > 0 && a.num_pages > 0 && a.table_stride > 0 && a.window >= 0, "b200_attn_paged: bad arguments");
  B200_CHECK_ARG(D == 64 || D == 128, "b200_attn_paged: head_dim %d not supported (64 and 128 only)", D);
  B200_CHECK_ARG(Hq % Hkv == 0 && Hq / Hkv <= 128, "b200_attn_paged: query heads per KV head must divide and be <= 128");
  B200_CHECK_ARG(a.page_size > 0 && a.page_size % 16 == 0, "b200_attn_paged: page size %d is not a multiple of 16", a.page_size);
  if (!(a.table_stride < (1ll << 30) && a.table_stride * a.page_size < (1ll << 30) && a.n_tokens * Hq < (1ll << 31) && a.B <= PAGED_MAX_SEQS))
    B200_FAIL(B200_ELIMIT, "b200_attn_paged: more than %d sequences, 2^30 keys of one or 2^31 rows of queries", PAGED_MAX_SEQS);
  bool ok = aligned16(a.q) && aligned16(a.k_pages) && aligned16(a.v_pages) && aligned16(a.out) && aligned16(a.workspace);
  PagedParams p;
  const int64_t q_len[2] = {a.n_tokens, Hq}, kv_len[3] = {a.num_pages, Hkv, a.page_size};
  for (int i = 0; i < 2; ++i) { p.qs[i] = a.q_strides[i]; ok = ok && a.q_strides[i] % 8 == 0 && (a.q_strides[i] > 0 || q_len[i] <= 1); }
  for (int i = 0; i < 3; ++i) { p.ks[i] = a.kv_strides[i]; ok = ok && a.kv_strides[i] % 8 == 0 && (a.kv_strides[i] > 0 || kv_len[i] <= 1); }
  if (!ok) B200_FAIL(B200_EALIGN, "b200_attn_paged: operands must be 16-byte aligned with positive strides that are multiples of 8");
  if (dtype != B200_BF16 && dtype != B200_F16) B200_FAIL(B200_ENOTSUP, "b200_attn_paged: dtype %d is not f16/bf16", dtype);
  if (a.B == 0 || a.n_tokens == 0 || a.max_q == 0) return B200_OK;
  const int G = Hq / Hkv, rows = rows_of(a.max_q, G);
  int64_t ml, acc;
  const int64_t need = workspace_parts(rows, D, &ml, &acc);
  if (!a.workspace || a.workspace_bytes < need)
    B200_FAIL(B200_EINVAL, "b200_attn_paged: workspace of %lld bytes required (got %lld)", (long long)need, (long long)a.workspace_bytes);
  p.q = a.q; p.k_pages = a.k_pages; p.v_pages = a.v_pages; p.out = a.out; p.q_start = a.q_start; p.kv_len = a.kv_len; p.table = a.page_table;
  p.B = a.B; p.N = a.n_tokens; p.num_pages = a.num_pages; p.table_stride = a.table_stride; p.Hq = Hq; p.Hkv = Hkv; p.G = G; p.page_size = a.page_size;
  p.page_shift = (a.page_size & (a.page_size - 1)) == 0 ? __builtin_ctz(a.page_size) : -1;
  p.window = a.window < (1ll << 30) ? a.window : 0;   // (no sequence is that long)
  p.scale = a.scale;
  p.head = static_cast<int4*>(a.workspace);
  p.ml = reinterpret_cast<float2*>(static_cast<char*>(a.workspace) + ml);
  p.acc = reinterpret_cast<float*>(static_cast<char*>(a.workspace) + acc);
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  // Short tables: a block of its own for each item takes hardly longer than joining pieces does, and saves a launch on the host.  By the table's width, as the lengths are on the
  // device: a wide table over short sequences gets pieces.  us, pieces -> whole, tables as wide as the sequences are long:
  //   1 sequence of 300 / 613 / 800 / 1024 / 2000 keys 8.7 -> 7.0, 8.8 -> 8.4, 8.8 -> 9.4, 8.8 -> 10.0, 9.0 -> 14.8; 8 of up to 1000 9.4 -> 9.9, 64 14.6 -> 15.0, 200 27.5 -> 27.1;
  //   19 with four tokens each, 64 dims, up to 1024 / 2000 keys 14.8 -> 11.7, 18.7 -> 16.6; tiles of 128 rows: 22 tokens over 512 / 1000 keys 13.3 -> 12.2, 14.2 -> 17.0,
  //   128 over 512 / 1000 15.1 -> 13.6, 16.0 -> 18.2, 512 over 512 / 1000 15.8 -> 14.0, 18.5 -> 18.5.
  p.whole = a.table_stride * a.page_size * D <= (rows == PAGED_TC5_ROWS ? 512 : 1024) * 128 ? 1 : 0;
  int rc = B200_ENOTSUP;
  if (tc5_enabled()) {
    if (rows == PAGED_TC5_ROWS) {
      rc = attn_paged_tc5(p, D, dtype, st);
    } else {
      B200_DISPATCH_HALF(dtype, T, {
        rc = rows == 8 ? (D == 128 ? launch_few<T, 128, 1>(p, dtype, st) : launch_few<T, 64, 1>(p, dtype, st))
                       : (D == 128 ? launch_few<T, 128, 2>(p, dtype, st) : launch_few<T, 64, 2>(p, dtype, st));
      });
    }
  }
  if (rc == B200_ELAUNCH) B200_CHECK_LAUNCH("attn_paged");
  if (rc == B200_ENOTSUP) {
    B200_DISPATCH_HALF(dtype, T, {
      launch_pdl(D == 128 ? attn_paged_plain_kernel<T, 128> : attn_paged_plain_kernel<T, 64>, dim3(static_cast<unsigned>(ceil_div(a.n_tokens * Hq, 4))),
                 dim3(128), 0, st, p);
    });
  } else if (!p.whole) {
    B200_DISPATCH_HALF(dtype, T, {
      const auto merge = [&](auto kernel, int groups) { launch_pdl(kernel, dim3(PAGED_CTAS, static_cast<unsigned>(groups)), dim3(256), 0, st, p); };
      if (rows == 8) { if (D == 128) merge(attn_paged_merge_kernel<T, 128, 8>, 8); else merge(attn_paged_merge_kernel<T, 64, 8>, 8); }
      else if (rows == 16) { if (D == 128) merge(attn_paged_merge_kernel<T, 128, 16>, 16); else merge(attn_paged_merge_kernel<T, 64, 16>, 16); }
      else { if (D == 128) merge(attn_paged_merge_rows_kernel<T, 128>, 16); else merge(attn_paged_merge_rows_kernel<T, 64>, 8); }
    });
  }
  B200_CHECK_LAUNCH("attn_paged");
  return B200_OK;
}
