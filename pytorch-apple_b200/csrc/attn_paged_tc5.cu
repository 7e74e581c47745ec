// Attention over a paged KV cache on the 5th-generation tensor cores (tcgen05.mma, accumulators in tensor memory, operands by TMA): chunks
// of prompts, whole prompts, and batches in which some sequences decode.
//
// The rows of a tile are up to 128 / G tokens times the G query heads that share a KV head (row = token * G + head), so that a key tile is
// fetched once for all of them; one TMA box per 64 dims brings them in that order.  Keys and values come in tiles of 128 keys, one box per
// piece of a page (the largest power of two that divides the page size, at most 128 rows), through rings of two stages each.
// What is attended follows from positions alone: a tile that reaches past a row's last key or ahead of its window is masked in
// registers, rows of V that no row of the tile may see are cleared in shared memory (0 times what lies there need not be 0).
//
// Two groups of four softmax warps share a tile, group g on its keys 64 g .. 64 g + 63 with running maxima and an accumulator of its
// own, one thread per row; the stored maximum follows the true one when that has grown by more than RESCALE_STEP.  The probabilities
// stay in tensor memory: they replace the scores that they come from and are the A operand of the second product from there (through shared memory a tile moved
// 224 KB of it instead of 160, and there was no room for a second stage of queries).  A block walks through its pieces (attn_paged.cuh) without draining: the scores of
// the next item's first tile are computed while the last one's rows are written.
//
// Probabilities are rounded to the activation type, which the tensor cores take (sums are of the unrounded ones, in fp32): an error of half a step of each, as large as
// the one that the output's own rounding makes.  Against 64 bits 0.20 to 0.23 % of the output in bf16 (root mean square), where rounding the output alone leaves 0.16; a
// second product for what the rounding cuts off would double the work with V for the difference.
//
// A tile of 128 rows x 128 keys takes 1.3 us, two of them under way, so one goes round in 2.6 (stamps of the global timer in a copy, 512 tokens over 4608 keys and a prompt of
// 2048): 0.8 to 1.0 from its scores to its last probability, 0.2 for their stores, 0.2 to 0.3 until the issuing thread knows that both groups have arrived (the
// slower one holds up the product of the other, and with it the next scores), 0.5 to issue the product with V, 0.5 for the scores of the tile after next, up to 0.3 until those
// are seen.  Its products are 0.55 us at the nominal rate and its exponentials 0.55: neither unit is full (the tensor pipe 27 % of the call), the way round is the bound.
//
// Warp roles: warps 0-3 and 4-7 the softmax groups, warp 8 MMA issuer and owner of the tensor memory, warps 9 and 10 TMA producers (Q and K; V), a box per lane.  Every
// barrier wait is bounded; on a time-out the block records a code, stops issuing, waits for its copies, frees its tensor memory and returns.
#include "attn_paged.cuh"
#include "gemm_tc5.cuh"
#include "tc5.cuh"

namespace b200 {

__device__ int g_attn_paged_error = 0;

namespace {

constexpr int BKV = 128;
constexpr int PANEL = 128 * 128;               // [128 rows][128 bytes]: 64 columns of an operand tile
constexpr int THREADS = 352;
// What an item costs besides its tiles, in tiles.  us at 2 / 3 / 4 / 5, a microsecond more than now each: 512 tokens over 4608 keys 32.1 / 31.0 / 31.4 / 31.6, a
// prompt of 2048 37.1 / 35.4 / 35.2 / 36.6, 32 sequences of which two are prompts 26.8 / 26.7 / 28.2 / 28.5.
constexpr int OV = 3;
constexpr int MIN_SHARE = 2;                   // tiles (and OVs) of a block at least
constexpr float LOG2E_F = 1.4426950408889634f;
constexpr float RESCALE_STEP = 8.f;
constexpr int TMEM_COLS = 512;                 // two buffers of S (128 columns each), O of both groups

template <typename T> struct Fmt;
template <> struct Fmt<__half> { static constexpr int value = 0; };
template <> struct Fmt<__nv_bfloat16> { static constexpr int value = 1; };

__device__ __forceinline__ float ex2(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}
__device__ __forceinline__ void mbar_arrive1(uint64_t* bar) {
  asm volatile("mbarrier.arrive.shared::cta.b64 _, [%0];" ::"r"(tc5::smem_addr(bar)) : "memory");
}

constexpr int OUT_BYTES = 2 * PANEL;           // where rows are turned round on their way out, 4 KB per softmax warp
constexpr int smem_bytes(int D) { return 6 * (D / 64) * PANEL + OUT_BYTES + 1024; }   // Q, K, V twice each, rows, alignment
static_assert(smem_bytes(64) >= paged_work_bytes + 1024, "the sequences' costs lie over the tiles");

template <typename T, int D>
__global__ void __launch_bounds__(THREADS, 1)
    attn_paged_tc5_kernel(const __grid_constant__ CUtensorMap map_q, const __grid_constant__ CUtensorMap map_k, const __grid_constant__ CUtensorMap map_v,
                          const __grid_constant__ PagedParams p, const int tpt, const int log_box) {
  const int box = 1 << log_box;                   // keys of a copy
  constexpr int NP = D / 64, TILE = NP * PANEL;   // panels and bytes of a K, V or Q tile
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~static_cast<uintptr_t>(1023));
  uint8_t* q_s = smem;
  uint8_t* k_s = smem + 2 * TILE;
  uint8_t* v_s = smem + 4 * TILE;
  uint8_t* out_s = smem + 6 * TILE;
  // tile n of the block lives in stages and buffers n & 1, the queries of piece f in stage f & 1.  A stage of K is free when the scores made from it
  // are there, one of V when the product is: the producers wait for what the softmax threads wait for (the next phase of these barriers
  // needs the copy that they are about to issue, so they cannot miss one).
  __shared__ __align__(8) uint64_t q_full[2], q_empty[2], k_full[2], v_full[2], s_full[2], p_ready[2], o_full[2];
  __shared__ uint32_t tmem_holder;
  __shared__ __align__(16) PagedPiece s_piece[PAGED_MAX_PIECES];
  __shared__ int64_t s_total[THREADS / 32];
  __shared__ int s_count, s_more, failed;

  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, cta = blockIdx.x;
  if (warp == 9 && lane == 0) {
    failed = 0;
    for (int s = 0; s < 2; ++s) {
      tc5::mbar_init(&q_full[s], 1);
      tc5::mbar_init(&q_empty[s], 1);
      tc5::mbar_init(&k_full[s], 1);
      tc5::mbar_init(&v_full[s], 1);
      tc5::mbar_init(&s_full[s], 1);
      tc5::mbar_init(&p_ready[s], 256);
      tc5::mbar_init(&o_full[s], 1);
    }
    tc5::fence_barrier_init();
    tc5::prefetch_tensormap(&map_q);
    tc5::prefetch_tensormap(&map_k);
    tc5::prefetch_tensormap(&map_v);
  }
  if (warp == 8) { tc5::tmem_alloc(&tmem_holder, TMEM_COLS); tc5::tmem_relinquish(); }
  pdl_trigger();
  pdl_wait();   // lengths, pages, queries and cache rows come from earlier kernels
  const PagedWork work = paged_work(smem, PAGED_MAX_SEQS);   // (no tile has been copied yet)
  int64_t u0 = 0, u1 = 0, share = 1, ends = 0;
  auto deal = [&]() {   // this block's range of costs (as far as it is known to this warp)
    const int64_t total = paged_prefix<BKV, OV, THREADS>(p, tpt, work, s_total);
    const int64_t even = (total + PAGED_CTAS - 1) / PAGED_CTAS;
    share = even > MIN_SHARE ? even : MIN_SHARE;
    u1 = (cta + 1) * share < total ? (cta + 1) * share : total;
  };
  deal();
  u0 = cta * share;
  int4 head = make_int4(0, 0, 0, 0);
  uint32_t tmem_base = 0;
  int n = 0, fg = 0;   // tiles and pieces behind this block, the same in every role

  while (true) {
    if (warp == 0) {
      int count = 0;
      if (u0 < u1) u0 = paged_pieces<BKV, OV>(p, tpt, work, u0, u1, s_piece, count, head, ends);
      if (lane == 0) { s_more = u0 < u1; s_count = count; }
    }
    tc5::fence_proxy_async();   // the tiles are copied over what has been written here
    tc5::tc_fence_before();
    __syncthreads();
    tc5::tc_fence_after();
    tmem_base = tmem_holder;
    const int F = s_count;
    const bool more = s_more;
    if (F == 0) break;   // (a range that no item begins or goes on in)

    if (warp >= 9) {   // ---- TMA producers, of Q and K and of V: lane l brings rows [l * box, (l + 1) * box) of a tile ----
      const bool is_k = warp == 9;
      const CUtensorMap* const map = is_k ? &map_k : &map_v;
      uint64_t *const full = is_k ? k_full : v_full, *const empty = is_k ? s_full : o_full;
      uint8_t* const tiles = (is_k ? k_s : v_s) + lane * box * 128;
      bool ok = true;
      int q_at = fg, kv_at = n;   // copies issued
      auto wait = [&](uint64_t* bar, uint32_t parity, int code) {
        const bool got = __all_sync(0xffffffffu, tc5::mbar_wait(bar, parity));
        const bool gone = *reinterpret_cast<volatile int*>(&failed) != 0;
        if (!got && !gone && lane == 0) { failed = 1; atomicExch(&g_attn_paged_error, code); }
        return __all_sync(0xffffffffu, got && !gone);
      };
      // Boxes of the next 32 / per_tile tiles of a piece, one per lane: page and first row (a page number is a round trip to L2: looked up a batch ahead)
      struct Rows { int page, row; };
      const int log_boxes = 7 - log_box, batch = 32 >> log_boxes;   // boxes of a tile, tiles looked up at a time
      auto locate = [&](const PagedPiece& c, int k0) {
        const int hi = c.p0 + c.tokens;   // keys from here on nobody sees
        const int lo = p.window > 0 && c.p0 - p.window + 1 > 0 ? static_cast<int>(c.p0 - p.window + 1) : 0;
        const int k = k0 + (lane >> log_boxes), key = (c.j0 + k) * BKV + (lane & ((1 << log_boxes) - 1)) * box;
        Rows a = {0, -1};
        if (k < c.cnt && key < hi && key + box > lo) {
          const int i = paged_page(p, key);
          a.row = key - i * p.page_size;
          a.page = __ldg(p.table + c.b * p.table_stride + i);
        }
        return a;
      };
      int at = n;
      PagedPiece c = s_piece[0];
      Rows next = locate(c, 0), cur = next;
      for (int f = 0; f < F && ok; ++f) {
        const int cnt = c.cnt, hk = c.hk, token = c.token;
        for (int k = 0; k < cnt && ok; ++k, ++at) {
          const int st = at & 1, in_batch = k & (batch - 1);
          if (in_batch == 0) {
            cur = next;
            if (k + batch < cnt) next = locate(c, k + batch);
            else if (f + 1 < F) { c = s_piece[f + 1]; next = locate(c, 0); }
          }
          const int src = (in_batch << log_boxes) + (lane & ((1 << log_boxes) - 1));
          const int page_ = __shfl_sync(0xffffffffu, cur.page, src), row = __shfl_sync(0xffffffffu, cur.row, src);
          const bool there = lane < (1 << log_boxes) && row >= 0;
          const uint32_t bytes = static_cast<uint32_t>(__popc(__ballot_sync(0xffffffffu, there))) * box * 128 * NP;
          if (is_k && k == 0) {
            const int qs = (fg + f) & 1, turn = (fg + f) >> 1;
            if (turn > 0 && !(ok = wait(&q_empty[qs], (turn & 1) ^ 1, 51))) break;
            if (lane == 0) {
              tc5::mbar_arrive_expect_tx(&q_full[qs], static_cast<uint32_t>(p.G) * tpt * 128 * NP);
              for (int h = 0; h < NP; ++h) tc5::tma_load_4d(q_s + qs * TILE + h * PANEL, &map_q, &q_full[qs], 0, hk * p.G, token, h);
            }
            ++q_at;
          }
          if (at >= 2 && !(ok = wait(&empty[st], ((at >> 1) & 1) ^ 1, is_k ? 50 : 52))) break;
          if (lane == 0) tc5::mbar_arrive_expect_tx(&full[st], bytes);
          __syncwarp();
          if (there) {
            const int page = page_ < 0 || page_ >= p.num_pages ? static_cast<int>(p.num_pages) : page_;   // outside the tensor: zeros
            for (int h = 0; h < NP; ++h) tc5::tma_load_5d(tiles + st * TILE + h * PANEL, map, &full[st], 0, row, h, hk, page);
          }
          kv_at = at + 1;
        }
      }
      // on a failure elsewhere the copies in flight must land before the block leaves
      if (*reinterpret_cast<volatile int*>(&failed)) {
        for (int i = q_at > 2 ? q_at - 2 : 0; is_k && i < q_at; ++i) tc5::mbar_wait(&q_full[i & 1], (i >> 1) & 1, 1u << 16);
        for (int i = kv_at > 2 ? kv_at - 2 : 0; i < kv_at; ++i) tc5::mbar_wait(&full[i & 1], (i >> 1) & 1, 1u << 16);
      }
    } else if (warp == 8) {
      if (lane == 0) {   // ---- MMA issuer ----
        constexpr uint32_t idesc_s = tc5::umma_idesc(128, BKV, Fmt<T>::value);
        constexpr uint32_t idesc_o = tc5::umma_idesc(128, D, Fmt<T>::value) | (1u << 16);   // B operand MN-major
        const uint32_t q_first = tc5::desc_sw128_lo(tc5::smem_addr(q_s));
        bool ok = true;
        // scores run up to two tiles ahead of the products with V: (sf, sk) is the next tile whose scores are to be issued
        int sf = 0, sk = 0, sn = n;
        auto issue_s = [&](bool look) {   // look: the K tile has not been looked for by the softmax threads
          const int st = sn & 1, qs = (fg + sf) & 1;
          if (sk == 0 && !tc5::mbar_wait(&q_full[qs], ((fg + sf) >> 1) & 1)) return false;
          if (look && !tc5::mbar_wait(&k_full[st], (sn >> 1) & 1)) return false;
          tc5::tc_fence_after();
          const uint32_t k_lo = tc5::desc_sw128_lo(tc5::smem_addr(k_s + st * TILE)), q_lo = q_first + qs * (TILE >> 4);
#pragma unroll
          for (int h = 0; h < NP; ++h) tc5::umma_f16_kblock(tmem_base + 128 * st, q_lo + h * (PANEL >> 4), k_lo + h * (PANEL >> 4), idesc_s, h > 0);
          tc5::umma_commit(&s_full[st]);
          if (++sk == s_piece[sf].cnt) {
            tc5::umma_commit(&q_empty[qs]);
            ++sf;
            sk = 0;
          }
          ++sn;
          return true;
        };
        for (int i = 0; i < 2 && ok && sf < F; ++i) ok = issue_s(true);
        int at = n;
        for (int f = 0; f < F && ok; ++f) {
          const int cnt = s_piece[f].cnt;
          for (int k = 0; k < cnt && ok; ++k, ++at) {
            const int st = at & 1;
            const uint32_t v_addr = tc5::smem_addr(v_s + st * TILE);
            if (!(ok = tc5::mbar_wait(&p_ready[st], (at >> 1) & 1))) break;
            tc5::tc_fence_after();
#pragma unroll
            for (int e = 0; e < 8; ++e) {     // 16 keys per instruction = two 8-key groups of the V panels
              const uint64_t db = tc5::umma_desc_sw128_mn(v_addr + e * 2048, PANEL, 1024);
              tc5::umma_f16_ta(tmem_base + 256 + 128 * (e >> 2), tmem_base + 128 * st + 64 * (e >> 2) + 8 * (e & 3), db, idesc_o, k > 0 || (e & 3) != 0);
            }
            tc5::umma_commit(&o_full[st]);
            if (sf < F) ok = issue_s(false);
          }
        }
        if (!ok && !*reinterpret_cast<volatile int*>(&failed)) { failed = 1; atomicExch(&g_attn_paged_error, 53); }
      }
      __syncwarp();
    } else {
      // ---- softmax: one thread per row and group, group g on keys 64 g .. of a tile ----
      const int g = warp >> 2, quarter = warp & 3;
      const int r = 32 * quarter + lane;   // the tensor-memory lane this thread may read
      const uint32_t t_lane = tmem_base + (static_cast<uint32_t>(32 * quarter) << 16);
      const uint32_t t_o = t_lane + 256 + 128 * g;
      const float c = p.scale * LOG2E_F;   // scores in the log2 domain
      bool alive = true;
      auto wait_all = [&](uint64_t* bar, uint32_t parity, int code) {
        bool got = tc5::mbar_try_wait(bar, parity);
        if (!__all_sync(0xffffffffu, got)) got = __all_sync(0xffffffffu, tc5::mbar_wait(bar, parity));
        if (!got && lane == 0 && !*reinterpret_cast<volatile int*>(&failed)) { failed = 1; atomicExch(&g_attn_paged_error, code); }
        return got;
      };
      int at = n, left = 0;   // tiles of this list still to come
      for (int f = 0; f < F; ++f) left += s_piece[f].cnt;
#pragma unroll 1
      for (int f = 0; f < F; ++f) {   // (a thread that has given up still meets the others at the end of every piece)
        const PagedPiece pc = s_piece[f];
        const int rows = pc.tokens * p.G;
        const bool row_live = r < rows, warp_live = 32 * quarter < rows;
        const int see = row_live ? pc.p0 + r / p.G + 1 : 0;   // keys from here on this row does not see
        const int from = p.window > 0 && see - p.window > 0 ? static_cast<int>(see - p.window) : 0;   // nor those ahead of this one
        const int hi = pc.p0 + pc.tokens, lo = p.window > 0 && pc.p0 - p.window + 1 > 0 ? static_cast<int>(pc.p0 - p.window + 1) : 0;   // nor any row
        float m_run = -INFINITY, l_run = 0.f;   // maximum that the row's sums are relative to, sum of the probabilities
#pragma unroll 1
        for (int k = 0; k < pc.cnt && alive; ++k, ++at, --left) {
          const int st = at & 1, key0 = (pc.j0 + k) * BKV;
          const uint32_t t_s = t_lane + 128 * st + 64 * g;   // this thread's scores, and where its probabilities replace them
          if (!wait_all(&s_full[st], (at >> 1) & 1, 54)) { alive = false; break; }
          tc5::tc_fence_after();
          // A tile that all rows see all of: the probabilities follow the scores at once, relative to the maximum so far; where a row has outgrown it the
          // tile is done again below (S is still there, and nobody has been told of the probabilities).
          bool done = false;
          if (warp_live && k > 0 && c > 0.f && key0 + BKV <= pc.p0 + 1 && (p.window == 0 || key0 + p.window >= pc.p0 + pc.tokens)) {
            const float m_use = m_run == -INFINITY ? 0.f : m_run;
            float sum[4] = {0.f, 0.f, 0.f, 0.f}, mx[4] = {-INFINITY, -INFINITY, -INFINITY, -INFINITY};
            uint32_t w[32];
            auto probabilities = [&](float (&u)[32], int q0) {
#pragma unroll
              for (int q = 0; q < 4; ++q) {
                float pr[8];
#pragma unroll
                for (int e = 0; e < 8; e += 2) {
                  float a = u[8 * q + e], d = u[8 * q + e + 1];
                  mx[e >> 1] = fmaxf(mx[e >> 1], fmaxf(a, d));
                  tc5::fma2(a, d, c, -m_use, -m_use);
                  pr[e] = ex2(a);
                  pr[e + 1] = ex2(d);
                  tc5::add2(sum[e & 2], sum[(e & 2) + 1], pr[e], pr[e + 1]);
                }
                const uint4 v = pack8<T>(pr);
                w[4 * (q0 + q)] = v.x; w[4 * (q0 + q) + 1] = v.y; w[4 * (q0 + q) + 2] = v.z; w[4 * (q0 + q) + 3] = v.w;
              }
            };
            float u0_[32], u1_[32];
            tc5::tmem_ld_32x32_async(t_s, u0_);
            tc5::tmem_ld_wait();
            tc5::tmem_ld_32x32_async(t_s + 32, u1_);
            probabilities(u0_, 0);
            tc5::tmem_ld_wait();
            probabilities(u1_, 4);
            const float top = fmaxf(fmaxf(mx[0], mx[1]), fmaxf(mx[2], mx[3])) * c;
            done = !__any_sync(0xffffffffu, row_live && (top > m_run + RESCALE_STEP || (m_run == -INFINITY && top > m_run)));
            if (done) {
              l_run += (sum[0] + sum[1]) + (sum[2] + sum[3]);
              tc5::tmem_st_32x32_raw(t_s, w);
            }
          }
          if (warp_live && !done) {
            float u[64];
            tc5::tmem_ld_32x32_async(t_s, *reinterpret_cast<float(*)[32]>(&u[0]));
            tc5::tmem_ld_32x32_async(t_s + 32, *reinterpret_cast<float(*)[32]>(&u[32]));
            tc5::tmem_ld_wait();
            float to_log2 = c;
            if (c <= 0.f) {   // (with the factor left for later the maximum would be the minimum, and 0 times a masked key's -infinity no number)
#pragma unroll
              for (int e = 0; e < 64; e += 2) tc5::mul2(u[e], u[e + 1], c);
              to_log2 = 1.f;
            }
            const int end = see - key0 - 64 * g, begin = from - key0 - 64 * g;
            if (end < 64 || begin > 0) {
#pragma unroll
              for (int e = 0; e < 64; ++e)
                if (e >= end || e < begin) u[e] = -INFINITY;
            }
            float mx[4] = {-INFINITY, -INFINITY, -INFINITY, -INFINITY};
#pragma unroll
            for (int e = 0; e < 64; e += 8)
#pragma unroll
              for (int q = 0; q < 4; ++q) mx[q] = fmaxf(mx[q], fmaxf(u[e + 2 * q], u[e + 2 * q + 1]));
            const float top = fmaxf(fmaxf(mx[0], mx[1]), fmaxf(mx[2], mx[3])) * to_log2;
            const bool moved = top > m_run + RESCALE_STEP || (m_run == -INFINITY && top > m_run);
            const float m_new = moved ? top : m_run;
            const float m_use = m_new == -INFINITY ? 0.f : m_new;
            if (k > 0 && __any_sync(0xffffffffu, moved)) {   // rescale this warp's rows, once the product before has finished
              if (!wait_all(&o_full[st ^ 1], ((at - 1) >> 1) & 1, 55)) { alive = false; break; }
              const float alpha = moved ? ex2(m_run - m_use) : 1.f;   // 0 for the first maximum of a row
              tc5::tc_fence_after();
#pragma unroll 1
              for (int q = 0; q < D; q += 16) {
                float t[16];
                tc5::tmem_ld_32x16(t_o + q, t);
                tc5::tmem_ld_wait();
#pragma unroll
                for (int e = 0; e < 16; e += 2) tc5::mul2(t[e], t[e + 1], alpha);
                tc5::tmem_st_32x16(t_o + q, t);
              }
              tc5::tmem_st_wait();
              l_run *= alpha;
            }
            m_run = m_new;
            float sum[4] = {0.f, 0.f, 0.f, 0.f};
            uint32_t w[32];
#pragma unroll
            for (int q = 0; q < 8; ++q) {
              float pr[8];
#pragma unroll
              for (int e = 0; e < 8; e += 2) {
                float a = u[8 * q + e], d = u[8 * q + e + 1];
                tc5::fma2(a, d, to_log2, -m_use, -m_use);
                pr[e] = ex2(a);
                pr[e + 1] = ex2(d);
                tc5::add2(sum[e & 2], sum[(e & 2) + 1], pr[e], pr[e + 1]);
              }
              const uint4 v = pack8<T>(pr);
              w[4 * q] = v.x; w[4 * q + 1] = v.y; w[4 * q + 2] = v.z; w[4 * q + 3] = v.w;
            }
            l_run += (sum[0] + sum[1]) + (sum[2] + sum[3]);
            tc5::tmem_st_32x32_raw(t_s, w);
          }
          if (key0 + BKV > hi || key0 < lo) {   // clear the rows of V that no row sees
            if (!wait_all(&v_full[st], (at >> 1) & 1, 56)) { alive = false; break; }
            const int row = threadIdx.x >> 1, half = threadIdx.x & 1, key = key0 + row;
            if (key >= hi || key < lo) {
              uint8_t* const at_v = v_s + st * TILE + (NP == 2 ? half * PANEL + row * 128 : row * 128 + half * 64);
#pragma unroll
              for (int e = 0; e < 4 * NP; ++e) reinterpret_cast<uint4*>(at_v)[e] = make_uint4(0, 0, 0, 0);
            }
            tc5::fence_proxy_async();   // (the tensor core reads through the async proxy)
          }
          if (warp_live) tc5::tmem_st_wait();
          tc5::tc_fence_before();     // this thread's tcgen05.ld / st are complete before its probabilities are read, S and O touched again
          // what the products of this tile and the scores of the one after next read has landed: looked for by one warp per group
          if (quarter == 0) {
            if (g == 0 ? !wait_all(&v_full[st], (at >> 1) & 1, 57) : left > 2 && !wait_all(&k_full[st], ((at + 2) >> 1) & 1, 58)) { alive = false; break; }
          }
          mbar_arrive1(&p_ready[st]);
        }
        // ---- the piece's rows: the half of the head dimension that this group writes, from both accumulators ----
        if (alive) alive = wait_all(&o_full[(at - 1) & 1], ((at - 1) >> 1) & 1, 59);
        float* const ml = reinterpret_cast<float*>(out_s + g * 1024);
        ml[r] = m_run;
        ml[128 + r] = l_run;
        tc5::tc_fence_before();
        asm volatile("bar.sync 1, 256;" ::: "memory");
        tc5::tc_fence_after();
        const float *ml_0 = reinterpret_cast<const float*>(out_s) + r, *ml_1 = reinterpret_cast<const float*>(out_s + 1024) + r;
        const float m_0 = ml_0[0], m_1 = ml_1[0], l_0 = ml_0[128], l_1 = ml_1[128];
        asm volatile("bar.sync 1, 256;" ::: "memory");
        if (alive && warp_live) {
          const float m_all = fmaxf(m_0, m_1), m_ref = m_all == -INFINITY ? 0.f : m_all;
          float w_0 = ex2(m_0 - m_ref), w_1 = ex2(m_1 - m_ref);
          const float l_all = l_0 * w_0 + l_1 * w_1;
          const bool whole = pc.flags == 3;
          if (whole) {
            const float inv = l_all > 0.f ? 1.f / l_all : 0.f;   // a row without keys gives zeros
            w_0 *= inv;
            w_1 *= inv;
          }
          const int64_t slot = paged_slot(cta, pc.flags & 1, PAGED_TC5_ROWS);
          if (!whole && g == 0 && row_live) p.ml[slot + r] = make_float2(m_all, l_all);
          // Sums go as [D / 4][rows] of four each, so that a warp's rows make whole lines; results through 4 KB of the warp's (chunk c of row r at c ^ (r & 7))
          uint8_t* const own = out_s + warp * 4096;
          const int live = rows - 32 * quarter < 32 ? rows - 32 * quarter : 32;   // rows of this warp
          const int64_t to = ((static_cast<int64_t>(pc.token) + r / p.G) * p.Hq + pc.hk * p.G + r % p.G) * D + g * (D / 2);
          float4* const part = reinterpret_cast<float4*>(p.acc + slot * D) + r;
#pragma unroll
          for (int q = 0; q < D / 2; q += 32) {
            float t0[32], t1[32];
            tc5::tmem_ld_32x32_async(t_lane + 256 + g * (D / 2) + q, t0);
            tc5::tmem_ld_32x32_async(t_lane + 384 + g * (D / 2) + q, t1);
            tc5::tmem_ld_wait();
#pragma unroll
            for (int e = 0; e < 32; e += 2) { t0[e] = fmaf(t1[e], w_1, t0[e] * w_0); t0[e + 1] = fmaf(t1[e + 1], w_1, t0[e + 1] * w_0); }
            if (whole) {
#pragma unroll
              for (int e = 0; e < 4; ++e)
                *reinterpret_cast<uint4*>(own + lane * 128 + (((q / 8 + e) ^ (r & 7)) << 4)) = pack8<T>(*reinterpret_cast<float(*)[8]>(&t0[8 * e]));
            } else if (row_live) {
#pragma unroll
              for (int e = 0; e < 8; ++e) part[((g * (D / 2) + q) / 4 + e) * PAGED_TC5_ROWS] = *reinterpret_cast<float4*>(&t0[4 * e]);
            }
          }
          tc5::tc_fence_before();
          if (whole) {
            constexpr int CH = D / 16;   // 16-byte chunks of half a row
            __syncwarp();
#pragma unroll
            for (int it = 0; it < CH; ++it) {
              const int row = it * (32 / CH) + lane / CH, ch = lane % CH;
              const int64_t dst = __shfl_sync(0xffffffffu, to, row);
              if (row < live)
                *reinterpret_cast<uint4*>(static_cast<T*>(p.out) + dst + ch * 8) = *reinterpret_cast<const uint4*>(own + row * 128 + ((ch ^ (row & 7)) << 4));
            }
          }
          __syncwarp();
        }
      }
    }
    for (int f = 0; f < F; ++f) n += s_piece[f].cnt;
    fg += F;
    if (__syncthreads_or(*reinterpret_cast<volatile int*>(&failed))) break;   // (what the threads see may differ: they agree)
    if (!more) break;
    deal();   // (the tiles lay over it)
  }
  if (threadIdx.x == 0 && !p.whole) {
    if (head.x) head.x = static_cast<int>(paged_divide(ends - 1, share)) - cta + 1;   // blocks with pieces of the item that begins here and ends in another
    p.head[cta] = head;
  }
  tc5::tc_fence_before();
  __syncthreads();
  if (warp == 8) { tc5::tc_fence_after(); tc5::tmem_dealloc(tmem_base, TMEM_COLS); }
}

template <typename T, int D> int launch(const PagedParams& p, int dtype, cudaStream_t st) {
  static PerDevice<bool> configured_on;
  bool* configured = configured_on.slot();
  if (!configured) return B200_ENOTSUP;
  if (!*configured) {
    if (cudaFuncSetAttribute(attn_paged_tc5_kernel<T, D>, cudaFuncAttributeMaxDynamicSharedMemorySize, smem_bytes(D)) != cudaSuccess) {
      cudaGetLastError();
      return B200_ENOTSUP;
    }
    *configured = true;
  }
  const int tpt = 128 / p.G;
  int log_box = 4;
  while (log_box < 7 && p.page_size % (2 << log_box) == 0) ++log_box;
  CUtensorMap mq, mk, mv;
  auto bytes = [](int64_t elems) { return elems > 0 ? static_cast<uint64_t>(elems) * 2 : static_cast<uint64_t>(D) * 2; };   // (0: an axis of length one)
  {
    const uint64_t dims[4] = {64, static_cast<uint64_t>(p.Hq), static_cast<uint64_t>(p.N), D / 64};
    const uint64_t str[3] = {bytes(p.qs[1]), bytes(p.qs[0]), 128};
    const uint32_t b[4] = {64, static_cast<uint32_t>(p.G), static_cast<uint32_t>(tpt), 1};
    if (!tma_encode_sw128(&mq, dtype, 4, p.q, dims, str, b)) return B200_ENOTSUP;
  }
  for (int i = 0; i < 2; ++i) {
    const uint64_t dims[5] = {64, static_cast<uint64_t>(p.page_size), D / 64, static_cast<uint64_t>(p.Hkv), static_cast<uint64_t>(p.num_pages)};
    const uint64_t str[4] = {bytes(p.ks[2]), 128, bytes(p.ks[1]), bytes(p.ks[0])};
    const uint32_t b[5] = {64, 1u << log_box, 1, 1, 1};
    if (!tma_encode_sw128(i ? &mv : &mk, dtype, 5, i ? p.v_pages : p.k_pages, dims, str, b)) return B200_ENOTSUP;
  }
  return launch_pdl(attn_paged_tc5_kernel<T, D>, dim3(PAGED_CTAS), dim3(THREADS), smem_bytes(D), st, mq, mk, mv, p, tpt, log_box) == cudaSuccess ? B200_OK : B200_ELAUNCH;
}

}  // namespace

int attn_paged_tc5_error(bool clear) {
  int v = 0;
  if (cudaMemcpyFromSymbol(&v, g_attn_paged_error, sizeof(int)) != cudaSuccess) return -1;
  if (clear && v) {
    const int zero = 0;
    cudaMemcpyToSymbol(g_attn_paged_error, &zero, sizeof(int));
  }
  return v;
}

int attn_paged_tc5(const PagedParams& p, int D, int dtype, cudaStream_t st) {
  if (p.num_pages >= (1ll << 31) - 1) return B200_ENOTSUP;
  if (dtype == B200_BF16) return D == 128 ? launch<__nv_bfloat16, 128>(p, dtype, st) : launch<__nv_bfloat16, 64>(p, dtype, st);
  return D == 128 ? launch<__half, 128>(p, dtype, st) : launch<__half, 64>(p, dtype, st);
}

}  // namespace b200
