// Attention over a paged cache for chunks of many query rows (prompts in pieces): pairs of 128-row tiles on tcgen05.
//
// The same sums as paged_decode.cu, bound by the tensor cores and the exponentials where rows are many. Rows of a tile are (token, head of the group), so the
// heads that share a key head read its keys once: with rep heads per group a tile holds 128 / rep tokens, one TMA box {64 columns, rep heads, 128 / rep tokens}
// per 64 columns. A CTA walks its share of the line of units (paged.cuh) with everything in flight across items: per pair of tiles and block of 128 keys
//   warp 0      : TMA: queries once per item, keys one block ahead in two stages, values; a box per page
//   warp 1      : S = Q K^T, block by block, tile 0 then tile 1, into one S buffer: a product is issued when the rows of the one before have been read
//   warp 3      : O += P V as the rows of P arrive (a warp of its own: one that issued both waited for one tile's barriers while the other's were ready)
//   warp 2      : clears the value rows behind a sequence's last token before they are multiplied (what lies there may be anything)
//   warps 4-11  : softmax and sums of tile 0 and tile 1, a thread per row: the whole S row in registers, P as packed bf16 in tensor memory, where the product takes
//                 it from (through shared memory P cost 160 of the 384 KB that a block moves there, 128 bytes a cycle), O in tensor memory
// The softmax warps hold a whole S row, P's words and the sums at once: 416 bytes of spill stores, 588 of loads (600 with 64-wide heads).
// Tensor memory: S 128 | P 2 x 64 | O 2 x HDP columns. Parts of items go to scratch in fp32 and are joined by a second launch. Every wait is bounded.
//
// 2048 tokens over 16384, 32 heads on 8 of 128: 443 to 520 us (box and power), 1000 to 1160 TFLOP/s; prompts of six users with a window of 1024, 40 heads on 8 of 128:
// 139 us, 450 TFLOP/s of what is visible. A block takes a pair of tiles 3.3 to 3.6 thousand cycles, of which the tensor cores need 2048 and the exponentials 2048; the
// softmax warps never wait for a product. An item's end (last product, output, the next item's rows) costs about 9 thousand more, masked blocks half again as long.
#include "elfa_native.h"
#include "paged.cuh"

namespace elfa {

int make_paged_tmap(CUtensorMap* tm, const void* pages, long long P, int Hkv, int page, int hd, int box_rows);
bool paged_units_fit(const PagedGeom& g, int block);

namespace {

constexpr int PBLK = 128, PTHREADS = 384, PSUB = 128 * 128;

struct PrefillArgs {
  PagedGeom g;
  const __nv_bfloat16 *q, *pages;
  __nv_bfloat16* out;
  float *part, *stat;                  // [2 G][2 tiles][HDP / 4][128] float4, [2 G][2 tiles][128] (maximum, sum)
  PagedJoin* notes;                    // [G]
  long long qs;
  float scale;
  int tile_toks;                       // tokens of one of the two tiles
};

enum { PB_Q = 0, PB_QFREE, PB_KFULL, PB_KFREE = PB_KFULL + 2, PB_VFULL = PB_KFREE + 2, PB_VFREE = PB_VFULL + 2, PB_VTAIL = PB_VFREE + 2,
       PB_SFULL = PB_VTAIL + 2, PB_SREAD = PB_SFULL + 2, PB_PREADY, PB_OFULL = PB_PREADY + 2, PB_COUNT = PB_OFULL + 2 };

template <int HDP>
struct PrefillSmem {
  static constexpr int NSUB = HDP / 64;
  static constexpr int Q = 0, K = Q + 2 * NSUB * PSUB, V = K + 2 * NSUB * PSUB, OUT = V + 2 * NSUB * PSUB, BAR = OUT + 8 * 4096;
  static constexpr int TOTAL = BAR + PB_COUNT * 8 + 16 + 4 * (PTHREADS / 32);
  static constexpr int DYN = TOTAL + 1024;
  static_assert(paged_line_bytes(PAGED_MAX_SEQS) <= 8 * 4096, "the line of units lies where outputs will");
};

// what a CTA does of an item: blocks i0 .. i1 of its list; tile 0 takes part up to n0, tile 1 up to n1
struct Part {
  int i0, i1, n0, n1;
};
__device__ __forceinline__ Part part_of(const PagedGeom& g, const PagedItem& it, unsigned u, unsigned u_end) {
  Part p;
  p.i0 = (int)(u - it.u0);
  p.i1 = (int)(min(u_end, it.u0 + it.span.n) - it.u0);
  const int half = g.tile_rows >> 1, r0 = it.t * g.tile_rows, rows = min(g.tile_rows, it.s.n * g.rep - r0);
  if (rows <= half) {
    p.n0 = p.i1;
    p.n1 = p.i0;
  } else {
    const int hi = max(it.s.kv - it.s.n + g.by_rep(r0 + half - 1) + 1, 0), b = (hi + PBLK - 1) / PBLK;      // blocks up to tile 0's last row
    const int n = b >= it.span.w0 ? it.span.ns + b - it.span.w0 : min(it.span.ns, b);
    p.n0 = min(max(n, p.i0), p.i1);
    p.n1 = p.i1;
  }
  return p;
}

// the lowest n bits, n clamped to 0 .. 32
__device__ __forceinline__ uint32_t first_bits(int n) { return n <= 0 ? 0u : (n >= 32 ? 0xffffffffu : (1u << n) - 1u); }

template <int HDP>
__global__ void __launch_bounds__(PTHREADS, 1) paged_prefill_kernel(const __grid_constant__ CUtensorMap tmQ, const __grid_constant__ CUtensorMap tmKV,
                                                                    const __grid_constant__ PrefillArgs a) {
  using L = PrefillSmem<HDP>;
  constexpr int NSUB = L::NSUB;
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  uint64_t* bars = reinterpret_cast<uint64_t*>(smem + L::BAR);
  uint32_t* tmem_holder = reinterpret_cast<uint32_t*>(bars + PB_COUNT);
  volatile int* abort_flag = reinterpret_cast<volatile int*>(tmem_holder + 1);
  const uint32_t sbase = smem_u32(smem), bar0 = smem_u32(bars);
  auto bar = [&](int i) { return bar0 + 8u * i; };
  const PagedGeom& g = a.g;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int half_rows = g.tile_rows >> 1;

  if (threadIdx.x == 0) {
    prefetch_tmap(&tmQ);
    prefetch_tmap(&tmKV);
    for (int i = 0; i < PB_COUNT; ++i)
      mbar_init(bar(i), i == PB_SREAD || i == PB_PREADY || i == PB_PREADY + 1 ? 4 : 1);
    *abort_flag = 0;
    fence_barrier_init();
  }
  if (warp == 1) {
    tmem_alloc(smem_u32(tmem_holder), 512);
    tmem_relinquish();
  }
  // query rows that no box fills (rep does not divide 128) stay zero
  for (int i = half_rows * 8 + threadIdx.x; i < 128 * 8; i += PTHREADS)
#pragma unroll
    for (int s = 0; s < 2 * NSUB; ++s)
      asm volatile("st.shared.v4.b32 [%0], {%1, %1, %1, %1};" ::"r"(sbase + L::Q + s * PSUB + i * 16), "r"(0) : "memory");
  fence_proxy_async();
  const PagedLine line = paged_line(smem + L::OUT, g.B, tmem_holder + 4);
  const unsigned W = paged_prefix<PBLK, PTHREADS>(g, line, true);
  if (blockIdx.x == 0) paged_rest(g, a.out, line.seqs[0], line.seqs[g.B - 1]);
  const int G = (int)min(W, gridDim.x);
  const PagedShares shares(W, G);
  const unsigned u_begin = (int)blockIdx.x < G ? shares.first(blockIdx.x) : 0, u_end = (int)blockIdx.x < G ? shares.first(blockIdx.x + 1) : 0;
  PagedItem it{};
  if (u_begin < u_end) it = paged_find<PBLK>(g, line, u_begin);
  if (threadIdx.x == 0) paged_join_note(g, a.notes, it, shares, blockIdx.x, u_begin < u_end && u_begin > it.u0);
  pdl_next();
  tc_fence_before();
  __syncthreads();                                         // the prefix makes room for outputs
  tc_fence_after();
  const uint32_t tmem_base = *tmem_holder;
  const uint32_t TM_S = tmem_base, TM_P[2] = {tmem_base + 128, tmem_base + 192};
  const uint32_t TM_O[2] = {tmem_base + 256, tmem_base + 256 + HDP};

  if (warp < 4) {
    reg_dec<80>();
    if (warp == 0) {
      // ---------------------------------------------------------------- loads
      const int box_rows = min(1 << g.page_shift, PBLK), boxes = PBLK / box_rows, box = lane / NSUB, sub = lane % NSUB;
      const bool mine = box < boxes;
      const int none = 2 * g.P * g.Hkv;                    // past the pool's end: zeros
      bool ok = true;
      uint32_t kc = 0, vc = 0, qc = 0;
      auto wait = [&](int b, uint32_t parity) { ok = ok && __all_sync(0xffffffffu, mbar_wait(bar(b), parity, abort_flag, g.status)); };
      auto page_of = [&](const PagedItem& x, int i) {
        const int key = x.span.block(i) * PBLK + box * box_rows;
        return mine && key < x.s.kv ? paged_page(g, x.b, key) : -1;
      };
      auto load_q = [&](const PagedItem& x) {
        if (qc) wait(PB_QFREE, (qc - 1) & 1);
        ++qc;
        if (!ok) return;
        const int tiles = min(g.tile_rows, x.s.n * g.rep - x.t * g.tile_rows) > half_rows ? 2 : 1;
        if (lane == 0) mbar_expect_tx(bar(PB_Q), tiles * NSUB * half_rows * 128);
        __syncwarp();
        if (lane < tiles * NSUB)
          tma_load_3d(sbase + L::Q + lane * PSUB, &tmQ, (lane % NSUB) * 64, x.h * g.rep, x.s.q0 + (2 * x.t + lane / NSUB) * a.tile_toks, bar(PB_Q));
        __syncwarp();
      };
      auto load = [&](const PagedItem& x, int i, int id, int kv, uint32_t dst, int b) {
        if (lane == 0) mbar_expect_tx(bar(b), NSUB * PSUB);
        __syncwarp();
        if (mine)
          tma_load_3d(dst + sub * PSUB + box * box_rows * 128, &tmKV, sub * 64, (x.span.block(i) * PBLK + box * box_rows) & ((1 << g.page_shift) - 1),
                      id < 0 ? none : (2 * id + kv) * g.Hkv + x.h, bar(b));
        __syncwarp();
      };
      auto load_k = [&](const PagedItem& x, int i, int id) {
        const int st = kc & 1;
        if (kc >= 2) wait(PB_KFREE + st, ((kc >> 1) - 1) & 1);
        ++kc;
        if (ok) load(x, i, id, 0, sbase + L::K + st * NSUB * PSUB, PB_KFULL + st);
      };
      if (u_begin < u_end) {
        int id = page_of(it, (int)(u_begin - it.u0));
        load_q(it);
        load_k(it, (int)(u_begin - it.u0), id);
        for (unsigned u = u_begin; u < u_end && ok; ++u) {
          const PagedItem cur = it;
          const int i = (int)(u - cur.u0);
          int next_id = -1;
          if (u + 1 < u_end) {
            const bool fresh = u + 1 >= it.u0 + it.span.n;
            if (fresh) paged_next<PBLK>(g, it);
            next_id = page_of(it, (int)(u + 1 - it.u0));
            if (fresh) load_q(it);
            load_k(it, (int)(u + 1 - it.u0), next_id);
          }
          const int st = vc & 1;
          if (vc >= 2) wait(PB_VFREE + st, ((vc >> 1) - 1) & 1);
          ++vc;
          if (ok) load(cur, i, id, 1, sbase + L::V + st * NSUB * PSUB, ((cur.span.block(i) + 1) * PBLK > cur.s.kv ? PB_VTAIL : PB_VFULL) + st);
          id = next_id;
        }
      }
    } else if (warp == 1 || warp == 3) {
      // ---------------------------------------------------------------- products: S from warp 1, O from warp 3
      bool ok = true;
      auto wait = [&](int b, uint32_t parity) { ok = ok && __all_sync(0xffffffffu, mbar_wait(bar(b), parity, abort_flag, g.status)); };
      auto commit = [&](int b) {
        if (elect_one()) tc_commit(bar(b));
        __syncwarp();
      };
      uint32_t blocks = 0, parts = 0, done = 0, pI[2] = {0, 0};
      for (unsigned u = u_begin; u < u_end && ok;) {
        const Part p = part_of(g, it, u, u_end);
        for (int i = p.i0; i < p.i1 && ok; ++i, ++blocks) {
          const int st = blocks & 1;
          const uint32_t parity = (blocks >> 1) & 1;
          if (warp == 1) {
            constexpr uint32_t idesc = make_idesc_bf16(128, 128, false, false);
            const uint64_t dq = make_smem_desc(sbase + L::Q, 16, 1024, 2), dk = make_smem_desc(sbase + L::K + st * NSUB * PSUB, 16, 1024, 2);
            const uint32_t q_lo = (uint32_t)dq, q_hi = (uint32_t)(dq >> 32), k_lo = (uint32_t)dk, k_hi = (uint32_t)(dk >> 32);
            wait(PB_KFULL + st, parity);
            if (i == p.i0) wait(PB_Q, parts++ & 1);
#pragma unroll
            for (int t = 0; t < 2; ++t) {
              if (i >= (t ? p.n1 : p.n0)) continue;
              if (done) wait(PB_SREAD, (done - 1) & 1);    // the one S buffer: the rows of the product before have been read
              ++done;
              if (!ok) break;
              tc_fence_after();
              if (elect_one()) {
#pragma unroll
                for (int kk = 0; kk < HDP / 16; ++kk) {
                  const uint32_t off = ((kk / 4) * PSUB + (kk % 4) * 32) >> 4;
                  tc_mma_f16_lh(TM_S, q_lo + ((t * NSUB * PSUB) >> 4) + off, q_hi, k_lo + off, k_hi, idesc, kk != 0);
                }
                tc_commit(bar(PB_SFULL + t));
              }
              __syncwarp();
            }
            if (ok) commit(PB_KFREE + st);
            if (ok && i + 1 == p.i1) commit(PB_QFREE);
          } else {
            constexpr uint32_t idesc = make_idesc_bf16(128, HDP, false, true);
            const uint64_t dv = make_smem_desc(sbase + L::V + st * NSUB * PSUB, PSUB, 1024, 2);
            const uint32_t v_lo = (uint32_t)dv, v_hi = (uint32_t)(dv >> 32);
            wait(PB_VFULL + st, parity);
#pragma unroll
            for (int t = 0; t < 2; ++t) {
              if (i >= (t ? p.n1 : p.n0)) continue;
              wait(PB_PREADY + t, pI[t]++ & 1);
              if (!ok) break;
              tc_fence_after();
              if (elect_one()) {
#pragma unroll
                for (int kk = 0; kk < 8; ++kk) tc_mma_f16_ts_lh(TM_O[t], TM_P[t] + kk * 8, v_lo + ((kk * 2048) >> 4), v_hi, idesc, i != p.i0 || kk != 0);
                tc_commit(bar(PB_OFULL + t));
              }
              __syncwarp();
            }
            if (ok) commit(PB_VFREE + st);
          }
        }
        u = it.u0 + p.i1;
        if (u < u_end) paged_next<PBLK>(g, it);
      }
    } else if (warp == 2) {
      // ---------------------------------------------------------------- value rows that hold no token
      uint32_t tails[2] = {0, 0}, blocks = 0;
      for (unsigned u = u_begin; u < u_end;) {
        const unsigned ue = min(u_end, it.u0 + it.span.n);
        bool ok = true;
        for (int i = (int)(u - it.u0); i < (int)(ue - it.u0) && ok; ++i) {
          const int key0 = it.span.block(i) * PBLK, st = blocks++ & 1;
          if (key0 + PBLK <= it.s.kv) continue;
          ok = __all_sync(0xffffffffu, mbar_wait(bar(PB_VTAIL + st), (st ? tails[1] : tails[0]) & 1, abort_flag, g.status));
          if (st) ++tails[1];
          else ++tails[0];
          if (!ok) break;
          for (int x = max(it.s.kv - key0, 0) * 8 + lane; x < PBLK * 8; x += 32)
#pragma unroll
            for (int s = 0; s < NSUB; ++s)
              asm volatile("st.shared.v4.b32 [%0], {%1, %1, %1, %1};" ::"r"(sbase + L::V + (st * NSUB + s) * PSUB + x * 16), "r"(0) : "memory");
          fence_proxy_async();
          __syncwarp();
          if (lane == 0) mbar_arrive(bar(PB_VFULL + st));
        }
        if (!ok) break;
        u = ue;
        if (u < u_end) paged_next<PBLK>(g, it);
      }
    }
  } else {
    reg_inc<208>();
    // ---------------------------------------------------------------- softmax and sums
    const int t = (warp - 4) >> 2, quarter = warp & 3, row_local = quarter * 32 + lane;
    const uint32_t lane_addr = (uint32_t)(quarter * 32) << 16;
    const uint32_t stage = sbase + L::OUT + (warp - 4) * 4096;             // this warp's 32 rows of 64 columns on their way out
    const float sl2 = a.scale * 1.4426950408889634f;
    uint32_t sc = 0, oc = 0;                               // S rows taken, P tiles handed over
    bool ok = true;
    for (unsigned u = u_begin; u < u_end && ok;) {
      const Part p = part_of(g, it, u, u_end);
      const int n_t = t ? p.n1 : p.n0;
      const int first_row = it.t * g.tile_rows + t * half_rows, rows = min(half_rows, it.s.n * g.rep - first_row);   // rows <= 0: no such tile
      const int pos0 = it.s.kv - it.s.n;
      const int r = first_row + min(row_local, max(rows, 1) - 1), tok = min(g.by_rep(r), it.s.n - 1), pos = pos0 + tok;
      const int pos_min = pos0 + g.by_rep(first_row), pos_max = pos0 + g.by_rep(first_row + max(rows, 1) - 1);
      const int lower = g.window ? pos - g.window + 1 : 0;
      float m = -INFINITY, l = 0.f;
      // the pages of each 16 keys, read a block ahead and looked at when it is their turn
      const int* pages_of = g.table + (long long)it.b * g.N;
      auto look = [&](int i) {
        const int key = it.span.block(i) * PBLK + lane * 16;
        return lane < 8 && key < it.s.kv ? __ldg(pages_of + (key >> g.page_shift)) : -1;
      };
      int id = p.i0 < n_t ? look(p.i0) : -1;
      for (int i = p.i0; i < n_t; ++i) {
        const int key0 = it.span.block(i) * PBLK;
        ok = __all_sync(0xffffffffu, mbar_wait(bar(PB_SFULL + t), sc & 1, abort_flag, g.status));
        ++sc;
        if (!ok) break;
        tc_fence_after();
        uint32_t s[128];
#pragma unroll
        for (int c = 0; c < 4; ++c) tmem_ld32(TM_S + lane_addr + c * 32, *reinterpret_cast<uint32_t(*)[32]>(&s[c * 32]));
        tmem_ld_wait();
        tc_fence_before();
        __syncwarp();
        if (lane == 0) mbar_arrive(bar(PB_SREAD));
        const uint32_t there = __ballot_sync(0xffffffffu, id >= 0 && id < g.P) & 0xffu;
        if (i + 1 < n_t) id = look(i + 1);
        bool landed = i == p.i0;                           // whether the product before is known to be complete (an item's end waits for it)
        if (there != 0xffu || key0 + PBLK - 1 > pos_min || (g.window && key0 < pos_max - g.window + 1 && key0 + PBLK > g.sinks)) {
          // a word of visible keys per 32 columns, then a select by one bit each: tests of every column in turn took 7 us a block where these take 0.3
#pragma unroll
          for (int c = 0; c < 4; ++c) {
            const int base = key0 + c * 32;
            uint32_t see = first_bits(pos + 1 - base) & ((there >> (2 * c) & 1u ? 0xffffu : 0u) | (there >> (2 * c + 1) & 1u ? 0xffff0000u : 0u));
            if (g.window) see &= ~first_bits(lower - base) | first_bits(g.sinks - base);
#pragma unroll
            for (int x = 0; x < 32; ++x) s[c * 32 + x] = see >> x & 1u ? s[c * 32 + x] : 0xff800000u;      // -inf
          }
        }
        auto row_max = [&]() {
          float mx4[4] = {-INFINITY, -INFINITY, -INFINITY, -INFINITY};
#pragma unroll
          for (int x = 0; x < 128; x += 2) mx4[(x >> 1) & 3] = max3(mx4[(x >> 1) & 3], __uint_as_float(s[x]), __uint_as_float(s[x + 1]));
          return fmaxf(fmaxf(mx4[0], mx4[1]), fmaxf(mx4[2], mx4[3])) * sl2;
        };
        // The exponentials do not wait for the row's maximum. Their reference may lag behind it: as long as a block's sum stays below 2^8 none of them is above that.
        // Where it does not (rare behind an item's first blocks), or nothing has been seen yet, the maximum is found, the sums are scaled and the row is done again.
        bool fresh = i == p.i0;
        for (;;) {
          if (fresh) {
            const float mx = row_max();
            const bool grow = mx > m;
            const float m_new = grow ? mx : m, alpha = grow ? fast_exp2(m - m_new) : 1.f;
            if (i > p.i0) {
              if (!landed) ok = __all_sync(0xffffffffu, mbar_wait(bar(PB_OFULL + t), (oc - 1) & 1, abort_flag, g.status));
              if (!ok) break;
              landed = true;
              tc_fence_after();
#pragma unroll 1
              for (int c = 0; c < HDP / 16; ++c) {         // narrow pieces: the S row stays in registers meanwhile
                uint32_t o[16];
                tmem_ld16(TM_O[t] + lane_addr + c * 16, o);
                tmem_ld_wait();
#pragma unroll
                for (int x = 0; x < 16; ++x) o[x] = __float_as_uint(__uint_as_float(o[x]) * alpha);
                tmem_st16(TM_O[t] + lane_addr + c * 16, o);
              }
              tmem_st_wait();
            }
            l *= alpha;
            m = m_new;
          }
          const float neg_m = m == -INFINITY ? 0.f : -m;
          const uint64_t sc2 = pack_f32x2(sl2, sl2), neg2 = pack_f32x2(neg_m, neg_m);
          uint64_t ls[2] = {0ull, 0ull};
#pragma unroll
          for (int c = 0; c < 4; ++c) {
            uint32_t w[16];
#pragma unroll
            for (int x = 0; x < 32; x += 2) {
              float x0, x1;
              unpack_f32x2(fma_f32x2(pack_f32x2(__uint_as_float(s[c * 32 + x]), __uint_as_float(s[c * 32 + x + 1])), sc2, neg2), x0, x1);
              const float e0 = fast_exp2(x0), e1 = fast_exp2(x1);
              ls[(x >> 1) & 1] = add_f32x2(ls[(x >> 1) & 1], pack_f32x2(e0, e1));
              w[x >> 1] = pack_bf16(e0, e1);
            }
            if (c == 0 && !landed) {                       // P is still the operand of the product before
              ok = __all_sync(0xffffffffu, mbar_wait(bar(PB_OFULL + t), (oc - 1) & 1, abort_flag, g.status));
              landed = true;
              tc_fence_after();
            }
            if (ok) tmem_st16(TM_P[t] + lane_addr + c * 16, w);
          }
          if (!ok) break;
          float a0, a1, a2, a3;
          unpack_f32x2(ls[0], a0, a1);
          unpack_f32x2(ls[1], a2, a3);
          const float block = (a0 + a1) + (a2 + a3);
          if (fresh || !__any_sync(0xffffffffu, block > 256.f || m == -INFINITY)) {
            l += block;
            break;
          }
          fresh = true;
        }
        if (!ok) break;
        tmem_st_wait();
        tc_fence_before();
        __syncwarp();
        if (lane == 0) mbar_arrive(bar(PB_PREADY + t));
        ++oc;
      }
      const bool any = n_t > p.i0, whole = p.i0 == 0 && p.i1 == it.span.n;
      u = min(u_end, it.u0 + it.span.n);
      PagedItem next = it;
      if (u < u_end) paged_next<PBLK>(g, next);            // its lengths arrive while the last product runs
      if (ok && any) {
        ok = __all_sync(0xffffffffu, mbar_wait(bar(PB_OFULL + t), (oc - 1) & 1, abort_flag, g.status));
        tc_fence_after();
      }
      if (ok && rows > 0) {
        const bool valid = row_local < rows;
        const long long at = it.s.q0 + tok;
        const int head = it.h * g.rep + r - tok * g.rep;
        const float inv = l == 0.f ? 0.f : 1.f / l;
        const long long orow = (at * g.H + head) * g.hd;
        const long long ps = (2LL * blockIdx.x + (p.i0 == 0)) * 2 + t;
        float4* prow = reinterpret_cast<float4*>(a.part) + ps * (HDP / 4) * 128 + row_local;
        const uint64_t inv2 = pack_f32x2(inv, inv), zero2 = 0ull;
        uint64_t odd = 0ull;
#pragma unroll 1
        for (int c = 0; c < HDP / 32; ++c) {
          uint32_t o[32];
          if (any) {
            tmem_ld32(TM_O[t] + lane_addr + c * 32, o);
            tmem_ld_wait();
          } else {
#pragma unroll
            for (int x = 0; x < 32; ++x) o[x] = 0u;
          }
          if (whole) {
            // through shared memory, 64 columns at a time: the 16-byte pieces of a row next to each other make whole lines (a thread's row at a time: 32 lines per
            // instruction, 3 us an item)
#pragma unroll
            for (int x = 0; x < 4; ++x) {
              uint32_t w[4];
#pragma unroll
              for (int y = 0; y < 4; ++y) {
                const uint64_t v = mul_f32x2(pack_f32x2(__uint_as_float(o[x * 8 + 2 * y]), __uint_as_float(o[x * 8 + 2 * y + 1])), inv2);
                odd = fma_f32x2(v, zero2, odd);            // infinity and NaN times zero
                float v0, v1;
                unpack_f32x2(v, v0, v1);
                w[y] = pack_bf16(v0, v1);
              }
              asm volatile("st.shared.v4.b32 [%0], {%1, %2, %3, %4};" ::"r"(stage + lane * 128 + ((((c & 1) * 4 + x) ^ (lane & 7)) << 4)), "r"(w[0]), "r"(w[1]),
                           "r"(w[2]), "r"(w[3]) : "memory");
            }
            if (c & 1) {
              __syncwarp();
#pragma unroll
              for (int y = 0; y < 8; ++y) {
                const int x = y * 4 + (lane >> 3), piece = lane & 7, col = (c >> 1) * 64 + piece * 8;
                const long long to = __shfl_sync(0xffffffffu, orow, x);
                uint4 v;
                asm volatile("ld.shared.v4.b32 {%0, %1, %2, %3}, [%4];" : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w)
                             : "r"(stage + x * 128 + ((piece ^ (x & 7)) << 4)) : "memory");
                if (quarter * 32 + x < rows && col < g.hd) *reinterpret_cast<uint4*>(a.out + to + col) = v;
              }
            }
          } else if (valid) {
#pragma unroll
            for (int x = 0; x < 8; ++x)
              prow[(c * 8 + x) * 128] = make_float4(__uint_as_float(o[x * 4]), __uint_as_float(o[x * 4 + 1]), __uint_as_float(o[x * 4 + 2]), __uint_as_float(o[x * 4 + 3]));
          }
          __syncwarp();
        }
        if (!whole && valid) reinterpret_cast<float2*>(a.stat)[ps * 128 + row_local] = make_float2(m, l);
        __syncwarp();
        float odd0, odd1;
        unpack_f32x2(odd, odd0, odd1);
        unsigned bad = __ballot_sync(0xffffffffu, whole && valid && (odd0 != 0.f || odd1 != 0.f));
        while (bad) {
          const int x = __ffs(bad) - 1, rx = first_row + quarter * 32 + x, tx = g.by_rep(rx);
          bad &= bad - 1;
          const int hx = it.h * g.rep + rx - tx * g.rep;
          const long long ax = it.s.q0 + tx;
          float res[HDP / 32];
          paged_row<HDP>(g, a.q + ax * a.qs + hx * g.hd, a.pages, it.b, it.h, pos0 + tx, a.scale, res);
#pragma unroll
          for (int c = 0; c < HDP / 32; ++c)
            if (lane + 32 * c < g.hd) a.out[(ax * g.H + hx) * g.hd + lane + 32 * c] = __float2bfloat16(res[c]);
        }
        tc_fence_before();
        __syncwarp();
      }
      it = next;
    }
  }

  __syncwarp();
  tc_fence_before();
  __syncthreads();
  if (warp == 1) {
    tc_fence_after();
    tmem_dealloc(tmem_base, 512);
  }
}

// Block (c - 1, y, z) joins 32 rows (y) of the item that CTA c has noted, a thread per row, its warps taking four columns each in turn (of the z-th share of them).
template <int HDP>
__global__ void __launch_bounds__(256) paged_prefill_join_kernel(const __grid_constant__ PrefillArgs a) {
  constexpr int VECS = HDP / 4, TURNS = VECS / 8;
  __shared__ float most[8][32], sums[8][32], weight[32][32];
  __shared__ uint2 tile[32][VECS + 1];
  __shared__ unsigned bad_rows;
  const PagedGeom& g = a.g;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  pdl_wait();
  const int c = blockIdx.x + 1;
  const PagedJoin j = a.notes[c];
  const int half_rows = g.tile_rows >> 1, t = blockIdx.y >> 2, first = (blockIdx.y & 3) * 32, local = first + lane;
  if (first >= half_rows || t * half_rows + first >= j.rows) return;
  const bool live = local < half_rows && t * half_rows + local < j.rows;
  const float2* stat = reinterpret_cast<const float2*>(a.stat);
  const float4* part = reinterpret_cast<const float4*>(a.part);
  const int n = j.last - c + 2;                                        // parts: CTAs c - 1 to last
  auto slot = [&](int i) { return (i == 0 ? 2LL * c - 1 : 2LL * (c - 1 + i)) * 2 + t; };
  float M = -INFINITY;
  for (int i = warp; i < n && live; i += 8) M = fmaxf(M, stat[slot(i) * 128 + local].x);
  most[warp][lane] = M;
  if (threadIdx.x == 0) bad_rows = 0;
  __syncthreads();
#pragma unroll
  for (int w = 0; w < 8; ++w) M = fmaxf(M, most[w][lane]);
  float den = 0.f;
  float4 num[TURNS];
#pragma unroll
  for (int k = 0; k < TURNS; ++k) num[k] = make_float4(0.f, 0.f, 0.f, 0.f);
  const int k0 = blockIdx.z * TURNS / gridDim.z, k1 = (blockIdx.z + 1) * TURNS / gridDim.z;
  for (int i0 = 0; i0 < n; i0 += 32) {
    const int m = min(32, n - i0);
    for (int i = warp; i < m; i += 8) {
      const float2 st = live ? stat[slot(i0 + i) * 128 + local] : make_float2(-INFINITY, 0.f);
      const float w = st.x == -INFINITY ? 1.f : fast_exp2(st.x - M);   // without a maximum: sums of zero, or a NaN to hand on
      weight[i][lane] = w;
      den += w * st.y;
    }
    __syncthreads();
    if (live)
#pragma unroll 2
      for (int i = 0; i < m; ++i) {
        const float w = weight[i][lane];
#pragma unroll
        for (int k = 0; k < TURNS; ++k) {
          if (k < k0 || k >= k1) continue;
          const float4 x = part[(slot(i0 + i) * VECS + k * 8 + warp) * 128 + local];
          num[k].x += w * x.x; num[k].y += w * x.y; num[k].z += w * x.z; num[k].w += w * x.w;
        }
      }
    __syncthreads();
  }
  sums[warp][lane] = den;
  __syncthreads();
  den = 0.f;
#pragma unroll
  for (int w = 0; w < 8; ++w) den += sums[w][lane];
  const float inv = den == 0.f ? 0.f : 1.f / den;
  bool finite = true;
#pragma unroll
  for (int k = 0; k < TURNS; ++k) {
    if (k < k0 || k >= k1) continue;
    const float x = num[k].x * inv, y = num[k].y * inv, z = num[k].z * inv, w = num[k].w * inv;
    finite = finite & isfinite(x) & isfinite(y) & isfinite(z) & isfinite(w);
    tile[lane][k * 8 + warp] = make_uint2(pack_bf16(x, y), pack_bf16(z, w));
  }
  if (live && !finite) atomicOr(&bad_rows, 1u << lane);
  __syncthreads();
  const unsigned bad = bad_rows;
  for (int x = warp; x < 32; x += 8) {
    const int r = j.r0 + t * half_rows + first + x;
    if (first + x >= half_rows || t * half_rows + first + x >= j.rows) continue;
    const int tok = g.by_rep(r), head = j.h * g.rep + r - tok * g.rep;
    const long long at = j.q0 + tok;
    __nv_bfloat16* po = a.out + (at * g.H + head) * g.hd;
    if (bad >> x & 1u) {
      float res[HDP / 32];
      paged_row<HDP>(g, a.q + at * a.qs + head * g.hd, a.pages, j.b, j.h, j.pos0 + tok, a.scale, res);
#pragma unroll
      for (int k = 0; k < HDP / 32; ++k) {
        const int col = lane + 32 * k;
        if (col < g.hd && col / 32 >= k0 && col / 32 < k1) po[col] = __float2bfloat16(res[k]);
      }
    } else if (lane < VECS && lane * 4 < g.hd && lane / 8 >= k0 && lane / 8 < k1) {
      *reinterpret_cast<uint2*>(po + lane * 4) = tile[x][lane];
    }
  }
}

template <int HDP>
int launch_prefill(PrefillArgs& a, int page, int join_z, cudaStream_t st) {
  CUtensorMap tmQ, tmKV;
  int rc = make_paged_tmap(&tmKV, a.pages, a.g.P, a.g.Hkv, page, a.g.hd, page < PBLK ? page : PBLK);
  if (rc != ELFA_OK) return rc;
  const uint64_t dims[3] = {(uint64_t)a.g.hd, (uint64_t)a.g.H, (uint64_t)a.g.T};
  const uint64_t strides[2] = {(uint64_t)a.g.hd * 2, (uint64_t)a.qs * 2};
  const uint32_t box[3] = {64, (uint32_t)a.g.rep, (uint32_t)a.tile_toks};
  rc = make_tmap_nd_bf16(&tmQ, a.q, 3, dims, strides, box);
  if (rc != ELFA_OK) return rc;
  ELFA_REQUIRE(paged_units_fit(a.g, PBLK), "paged_attention: too much work for one call (2^32 tiles of 256 rows by 128 keys)");
  ELFA_CUDA(allow_shared<paged_prefill_kernel<HDP>>(PrefillSmem<HDP>::DYN));
  const int grid = 148;
  paged_prefill_kernel<HDP><<<grid, PTHREADS, PrefillSmem<HDP>::DYN, st>>>(tmQ, tmKV, a);
  ELFA_CUDA(cudaGetLastError());
  ::elfa::count_launches(1);
  PdlScope scope(true);
  ELFA_CUDA(launch_chain(paged_prefill_join_kernel<HDP>, dim3(grid - 1, 8, join_z), dim3(256), 0, st, 1, a));
  ELFA_CUDA(cudaGetLastError());
  ::elfa::count_launches(1);
  return ELFA_OK;
}

}  // namespace

long long paged_prefill_scratch(int hd) { return 148LL * (2 * 2 * 128 * ((hd <= 64 ? 64 : 128) + 2) + 8); }

int paged_prefill(PagedGeom g, const void* q, long long qs, const void* pages, void* out, float* scratch, int page, float scale, cudaStream_t st) {
  PrefillArgs a{};
  a.g = g;
  a.q = static_cast<const __nv_bfloat16*>(q);
  a.pages = static_cast<const __nv_bfloat16*>(pages);
  a.out = static_cast<__nv_bfloat16*>(out);
  a.qs = qs;
  a.scale = scale;
  a.tile_toks = 128 / g.rep;
  a.g.tile_rows = 2 * a.tile_toks * g.rep;
  a.g.by_tile = div_by((unsigned)a.g.tile_rows);
  a.part = scratch;
  a.stat = scratch + 2LL * 148 * 2 * 128 * (g.hd <= 64 ? 64 : 128);
  a.notes = reinterpret_cast<PagedJoin*>(a.stat + 2LL * 148 * 2 * 128 * 2);
  // few items have many parts each: their columns go to several blocks too (a slice of 32 columns each)
  const long long items = g.Hkv * ((long long)g.T * g.rep / a.g.tile_rows + 1);
  const int join_z = items < 16 ? (g.hd <= 64 ? 2 : 4) : 1;
  return g.hd <= 64 ? launch_prefill<64>(a, page, join_z, st) : launch_prefill<128>(a, page, join_z, st);
}

}  // namespace elfa
