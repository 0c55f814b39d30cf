// Attention over a paged cache for a few query rows per key head (decoding, a few proposed tokens): tiles of 16 rows on `mma.sync`.
//
// o = sum_j softmax_j(q k_j scale) v_j over the keys that a row sees, one pass over keys and values with a running maximum and sum. Bound by the
// memory: every key and value is read once and meets 16 rows, 16 x 4 operations per element where the tensor cores would take hundreds. So
// a warp fetches for itself: blocks of 32 keys by TMA into a ring of its own, three blocks deep (12 x 16 KB in flight per SM at 128-wide heads),
// no barrier between the warps until an item ends, where their four partial results meet in shared memory. What a CTA leaves of an item
// that others share goes to scratch in fp32; a second small launch joins those (in the order of the CTAs, so one call's result does not depend on timing). Where items are
// alike, a cluster of up to eight CTAs takes each instead and joins its parts through distributed shared memory: no line to count, no second launch.
// The exponent's reference may lag behind the row's maximum by up to 2^8 before sums are scaled again.
// Probabilities are rounded to bf16 for the second product (relative 2^-8 at most, as the result will be); their sum is taken before that.
// 48 sequences of up to 8191 tokens, 32 heads on 8 of 128: 867 MB in 144 to 148 us, 6 TB/s (the first keys arrive after 4.5 us, the join takes 5).
// 16 sequences, a window of 4096: 65 MB in 20.5 us (in clusters of four; as a line of units 24). One sequence of 129 tokens: a 4 us kernel in a call that the host takes 13 us to issue.
#include "elfa_native.h"
#include "mma_sync.cuh"
#include "paged.cuh"

namespace elfa {

int make_paged_tmap(CUtensorMap* tm, const void* pages, long long P, int Hkv, int page, int hd, int box_rows);

namespace {

constexpr int DBLK = 32, DWARPS = 4, DST = 3, DROWS = 16;

struct DecodeArgs {
  PagedGeom g;
  const __nv_bfloat16 *q, *pages;
  __nv_bfloat16* out;
  float *part, *stat;                  // [2 G][16][HDP], [2 G][16][2] (maximum, sum)
  PagedJoin* notes;                    // [G]
  long long qs;                        // elements from a token's queries to the next one's
  float scale;
  int wide, whole;                     // a warp per sequence for the prefix; whole: that many CTAs (a cluster) take an item, 0: the line of units
  int min_units;
};

template <int HDP>
struct DecodeSmem {
  static constexpr int NSUB = HDP / 64, HALF = NSUB * DBLK * 128, UNIT = 2 * HALF;
  static constexpr int MERGE = DWARPS * DST * UNIT;                  // [2][16][HDP] fp32
  static constexpr int STAT = MERGE + 2 * DROWS * HDP * 4;           // [4][16][2]
  static constexpr int BAR = STAT + DWARPS * DROWS * 8;
  static constexpr int TOT = BAR + DWARPS * DST * 8;                 // warp totals, abort flag
  static constexpr int LINE = TOT + DWARPS * 4 + 16;
  static constexpr int bytes(int B) { return LINE + paged_line_bytes(B) + 1024; }
};

__device__ __forceinline__ int decode_ctas(unsigned W, int grid, int min_units) { return (int)min((W + min_units - 1) / min_units, (unsigned)grid); }

// The CTAs of a cluster have an item's parts in shared memory, [16][HDP] and (maximum, sum): row r is joined by CTA r mod their number, in their order.
template <int HDP>
__device__ __noinline__ void join_cluster(const DecodeArgs& a, PagedItem it, float* part, float2* stat, bool any) {
  constexpr int VEC = HDP / 4, SIDE = DWARPS * 32 / VEC;               // threads of a row, rows side by side
  __shared__ unsigned bad;
  const PagedGeom& g = a.g;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, n = a.whole, rank = (int)cluster_ctarank();
  const int r0 = it.t * DROWS, rows = min(DROWS, it.s.n * g.rep - r0);
  if (!any) {                                                          // fewer blocks than CTAs
    for (int i = threadIdx.x; i < DROWS * HDP; i += DWARPS * 32) part[i] = 0.f;
    if (threadIdx.x < DROWS) stat[threadIdx.x] = make_float2(-INFINITY, 0.f);
  }
  if (threadIdx.x == 0) bad = 0;
  cluster_sync_all();
  const int v = threadIdx.x % VEC;
  const uint32_t part_at = smem_u32(part), stat_at = smem_u32(stat);
  for (int r = rank + n * (threadIdx.x / VEC); r < rows; r += n * SIDE) {
    float2 st[8];
    float M = -INFINITY;
#pragma unroll
    for (int c = 0; c < 8; ++c)
      if (c < n) {
        st[c] = ld_cluster_f2(map_to_cta(stat_at + r * 8, c));
        M = fmaxf(M, st[c].x);
      }
    float4 num = make_float4(0.f, 0.f, 0.f, 0.f);
    float den = 0.f;
#pragma unroll
    for (int c = 0; c < 8; ++c)
      if (c < n) {
        const float4 x = ld_cluster_f4(map_to_cta(part_at + (r * HDP + v * 4) * 4, c));
        const float w = st[c].x == -INFINITY ? 1.f : fast_exp2(st[c].x - M);           // without a maximum: sums of zero, or a NaN to hand on
        den += w * st[c].y;
        num.x += w * x.x; num.y += w * x.y; num.z += w * x.z; num.w += w * x.w;
      }
    const float inv = den == 0.f ? 0.f : 1.f / den;
    num.x *= inv; num.y *= inv; num.z *= inv; num.w *= inv;
    if (v * 4 < g.hd) {
      const int tok = g.by_rep(r0 + r), head = it.h * g.rep + r0 + r - tok * g.rep;
      *reinterpret_cast<uint2*>(a.out + ((long long)(it.s.q0 + tok) * g.H + head) * g.hd + v * 4) = make_uint2(pack_bf16(num.x, num.y), pack_bf16(num.z, num.w));
      if (!(isfinite(num.x) && isfinite(num.y) && isfinite(num.z) && isfinite(num.w))) atomicOr(&bad, 1u << r);
    }
  }
  __syncthreads();
  for (int r = warp; r < rows; r += DWARPS) {
    if (!(bad >> r & 1u)) continue;
    const int tok = g.by_rep(r0 + r), head = it.h * g.rep + r0 + r - tok * g.rep;
    const long long at = it.s.q0 + tok;
    float res[HDP / 32];
    paged_row<HDP>(g, a.q + at * a.qs + head * g.hd, a.pages, it.b, it.h, it.s.kv - it.s.n + tok, a.scale, res);
#pragma unroll
    for (int x = 0; x < HDP / 32; ++x)
      if (lane + 32 * x < g.hd) a.out[(at * g.H + head) * g.hd + lane + 32 * x] = __float2bfloat16(res[x]);
  }
  cluster_sync_all();                                                  // nobody's shared memory goes while another reads it
}

template <int HDP>
__global__ void __launch_bounds__(DWARPS * 32) paged_decode_kernel(const __grid_constant__ CUtensorMap tm, const __grid_constant__ DecodeArgs a) {
  using L = DecodeSmem<HDP>;
  constexpr int NSUB = L::NSUB;
  constexpr unsigned FRONT = paged_front<DBLK>;
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  float* merge = reinterpret_cast<float*>(smem + L::MERGE);
  float2* stat = reinterpret_cast<float2*>(smem + L::STAT);
  volatile int* abort_flag = reinterpret_cast<volatile int*>(smem + L::TOT + DWARPS * 4);
  const PagedGeom& g = a.g;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, gr = lane >> 2, qd = lane & 3;
  const uint32_t ring = smem_u32(smem) + warp * DST * L::UNIT, bars = smem_u32(smem + L::BAR) + warp * DST * 8;

  if (threadIdx.x == 0) {
    prefetch_tmap(&tm);
    *abort_flag = 0;
  }
  if (lane < DST) mbar_init(bars + 8 * lane, 1);
  fence_barrier_init();
  unsigned u_begin, u_end;
  PagedItem first{};
  if (a.whole) {
    const int item = blockIdx.x / a.whole, rank = blockIdx.x - item * a.whole;
    first.b = item / g.Hkv;
    first.h = item - first.b * g.Hkv;
    first.t = 0;
    first.s = paged_seq(g, first.b);
    first.tiles = paged_tiles(g, first.s);
    first.span = paged_span<DBLK>(g, first.s, 0);
    first.u0 = 0u - FRONT;                               // no empty units
    const unsigned n = first.tiles ? first.span.n - FRONT : 0;
    u_begin = n * rank / a.whole;
    u_end = n * (rank + 1) / a.whole;
    if (first.h == 0 && rank == 0) {
      if (first.b == 0 && (g.ends & 1)) paged_zero_rows(g, a.out, 0, first.s.q0);
      if (first.b == g.B - 1 && (g.ends & 2)) paged_zero_rows(g, a.out, first.s.q0 + first.s.n, g.T);
    }
    __syncthreads();
  } else {
    const PagedLine line = paged_line(smem + L::LINE, g.B, reinterpret_cast<unsigned*>(smem + L::TOT));
    const unsigned W = paged_prefix<DBLK, DWARPS * 32>(g, line, a.wide);
    if (blockIdx.x == 0) paged_rest(g, a.out, line.seqs[0], line.seqs[g.B - 1]);
    const int G = decode_ctas(W, gridDim.x, a.min_units);
    const PagedShares shares(W, G);
    u_begin = (int)blockIdx.x < G ? shares.first(blockIdx.x) : 0;
    u_end = (int)blockIdx.x < G ? shares.first(blockIdx.x + 1) : 0;
    if (u_begin < u_end) first = paged_find<DBLK>(g, line, u_begin);
    if (threadIdx.x == 0) paged_join_note(g, a.notes, first, shares, blockIdx.x, u_begin < u_end && u_begin > first.u0);
  }
  pdl_next();
  if (u_begin >= u_end && !(a.whole > 1 && first.tiles)) return;           // a cluster stays together

  // ---- the warp's own loads: unit u_begin + warp, then every fourth; the page of the next one is looked up a turn ahead
  PagedItem pi = first;
  unsigned pu = u_begin + warp;
  const int rows_per_box = min(1 << g.page_shift, DBLK), boxes = DBLK / rows_per_box;
  const int box = lane / (2 * NSUB), sub = (lane >> 1) % NSUB, kv = lane & 1;
  uint32_t there = 0;                                    // two bits per ring slot: which half's page is there
  struct Ahead {
    int id, row, h;
    bool any;
  };
  auto look = [&]() {
    Ahead n{-1, 0, 0, false};
    for (; pu < u_end; pu += DWARPS) {
      while (pu - pi.u0 >= (unsigned)pi.span.n) paged_next<DBLK>(g, pi);
      if (pu - pi.u0 < FRONT) continue;
      const int key = pi.span.block((int)(pu - pi.u0 - FRONT)) * DBLK + box * rows_per_box;
      n.row = key & ((1 << g.page_shift) - 1);
      n.h = pi.h;
      n.any = true;
      if (box < boxes && key < pi.s.kv) n.id = __ldg(g.table + (long long)pi.b * g.N + (key >> g.page_shift));
      pu += DWARPS;
      break;
    }
    return n;
  };
  auto issue = [&](int slot, const Ahead& n) {
    if (!n.any) return;
    const uint32_t bar = bars + 8 * slot, dst = ring + slot * L::UNIT;
    if (lane == 0) mbar_expect_tx(bar, L::UNIT);
    const bool ok = n.id >= 0 && n.id < g.P;
    if (n.id >= g.P) atomicOr(g.status, (unsigned)ELFA_ST_BAD_PAGE);
    __syncwarp();
    if (box < boxes)                                     // an absent page is read past the pool's end, which gives zeros
      tma_load_3d(dst + kv * L::HALF + (sub * DBLK + box * rows_per_box) * 128, &tm, sub * 64, n.row,
                  ok ? (2 * n.id + kv) * g.Hkv + n.h : 2 * g.P * g.Hkv, bar);
    const unsigned who = __ballot_sync(0xffffffffu, ok);
    const uint32_t two = (who & 1u) | ((boxes > 1 ? who >> (2 * NSUB) & 1u : who & 1u) << 1);
    there = (there & ~(3u << (2 * slot))) | two << (2 * slot);
  };
  Ahead ahead;
  {
    Ahead n[DST];                                        // the first ones asked for together
#pragma unroll
    for (int s = 0; s < DST; ++s) {
      n[s] = look();
    }
    ahead = look();
#pragma unroll
    for (int s = 0; s < DST; ++s) issue(s, n[s]);
  }

  const float sl2 = a.scale * 1.4426950408889634f;
  PagedItem it = first;
  int slot = 0;
  uint32_t phase = 0;
  bool ok = true;
  for (unsigned u = u_begin; u < u_end;) {
    const unsigned ue = min(u_end, it.u0 + it.span.n);
    const int r0 = it.t * DROWS, rows = min(DROWS, it.s.n * g.rep - r0), pos0 = it.s.kv - it.s.n;
    if (!a.whole && ue - it.u0 <= FRONT) {                 // a share that ends before the item's first block: a part of nothing, for the join
      const long long ps = 2LL * blockIdx.x + (u == it.u0);
      for (int i = threadIdx.x; i < rows * HDP; i += DWARPS * 32) a.part[ps * DROWS * HDP + i] = 0.f;
      if ((int)threadIdx.x < rows) reinterpret_cast<float2*>(a.stat)[ps * DROWS + threadIdx.x] = make_float2(-INFINITY, 0.f);
      u = ue;
      continue;
    }
    // rows behind the last one repeat it
    const int ra = r0 + min(gr, rows - 1), rb = r0 + min(gr + 8, rows - 1), ta = g.by_rep(ra), tb = g.by_rep(rb);
    const int pa = pos0 + ta, pb = pos0 + tb, pos_min = pos0 + g.by_rep(r0), pos_max = pos0 + g.by_rep(r0 + rows - 1);
    uint32_t qf[HDP / 16][4];
    {
      const __nv_bfloat16* qa = a.q + (it.s.q0 + ta) * a.qs + (it.h * g.rep + ra - ta * g.rep) * g.hd;
      const __nv_bfloat16* qb = a.q + (it.s.q0 + tb) * a.qs + (it.h * g.rep + rb - tb * g.rep) * g.hd;
#pragma unroll
      for (int kk = 0; kk < HDP / 16; ++kk) {
        const int c = kk * 16 + qd * 2;
        qf[kk][0] = c < g.hd ? *reinterpret_cast<const uint32_t*>(qa + c) : 0u;
        qf[kk][1] = c < g.hd ? *reinterpret_cast<const uint32_t*>(qb + c) : 0u;
        qf[kk][2] = c + 8 < g.hd ? *reinterpret_cast<const uint32_t*>(qa + c + 8) : 0u;
        qf[kk][3] = c + 8 < g.hd ? *reinterpret_cast<const uint32_t*>(qb + c + 8) : 0u;
      }
    }
    float o[HDP / 8][4];
#pragma unroll
    for (int d = 0; d < HDP / 8; ++d) o[d][0] = o[d][1] = o[d][2] = o[d][3] = 0.f;
    float m[2] = {-INFINITY, -INFINITY}, l[2] = {0.f, 0.f};

    const unsigned lead = (warp - (u - u_begin)) & (DWARPS - 1);       // this warp's first unit of the item
    for (unsigned x = u + lead; x < ue; x += DWARPS) {
      if (x - it.u0 < FRONT) continue;
      const int key0 = it.span.block((int)(x - it.u0 - FRONT)) * DBLK;
      ok = ok && __all_sync(0xffffffffu, mbar_wait(bars + 8 * slot, phase, abort_flag, g.status));
      if (!ok) break;
      const uint32_t kbase = ring + slot * L::UNIT, vbase = kbase + L::HALF;
      const uint32_t two = there >> (2 * slot) & 3u;
      if (key0 + DBLK > it.s.kv) {
        // rows of the last page that hold no token yet: whatever lies there must not meet a probability of zero
        const int from = max(it.s.kv - key0, 0);
        for (int i = from * 8 + lane; i < DBLK * 8; i += 32)
#pragma unroll
          for (int s = 0; s < NSUB; ++s)
            asm volatile("st.shared.v4.b32 [%0], {%1, %1, %1, %1};" ::"r"(vbase + s * DBLK * 128 + i * 16), "r"(0) : "memory");
        fence_proxy_async();                                           // the ring's next copy into this slot comes behind
        __syncwarp();
      }
      float s[4][4];
#pragma unroll
      for (int n = 0; n < 4; ++n) s[n][0] = s[n][1] = s[n][2] = s[n][3] = 0.f;
#pragma unroll
      for (int kk = 0; kk < HDP / 16; ++kk)
#pragma unroll
        for (int np = 0; np < 2; ++np) {
          const int key = np * 16 + (lane >> 4) * 8 + (lane & 7), chunk = (kk & 3) * 2 + (lane >> 3 & 1);
          uint32_t b[4];
          ldsm4(b, kbase + (kk >> 2) * DBLK * 128 + key * 128 + ((chunk ^ (key & 7)) << 4));
          mma_bf16(s[2 * np], qf[kk], b[0], b[1]);
          mma_bf16(s[2 * np + 1], qf[kk], b[2], b[3]);
        }
      const bool need = two != 3u || key0 + DBLK - 1 > pos_min || (g.window && key0 <= pos_max - g.window && key0 + DBLK > g.sinks);
      if (need) {
#pragma unroll
        for (int n = 0; n < 4; ++n)
#pragma unroll
          for (int j = 0; j < 4; ++j) {
            const int key = key0 + n * 8 + qd * 2 + (j & 1);
            if (!(two >> (n >> 1) & 1u) || !paged_sees(g, key, j < 2 ? pa : pb)) s[n][j] = -INFINITY;
          }
      }
#pragma unroll
      for (int r = 0; r < 2; ++r) {
        float mx = fmaxf(fmaxf(fmaxf(s[0][2 * r], s[0][2 * r + 1]), fmaxf(s[1][2 * r], s[1][2 * r + 1])),
                         fmaxf(fmaxf(s[2][2 * r], s[2][2 * r + 1]), fmaxf(s[3][2 * r], s[3][2 * r + 1])));
        mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 1));
        mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 2)) * sl2;
        const bool grow = mx - m[r] > 8.f;
        if (__any_sync(0xffffffffu, grow)) {
          const float mn = grow ? mx : m[r], alpha = grow ? fast_exp2(m[r] - mn) : 1.f;
#pragma unroll
          for (int d = 0; d < HDP / 8; ++d) {
            o[d][2 * r] *= alpha;
            o[d][2 * r + 1] *= alpha;
          }
          l[r] *= alpha;
          m[r] = mn;
        }
        const float neg = m[r] == -INFINITY ? 0.f : -m[r];             // nothing seen yet: exp2(-inf) without inf - inf
#pragma unroll
        for (int n = 0; n < 4; ++n)
#pragma unroll
          for (int j = 0; j < 2; ++j) {
            s[n][2 * r + j] = fast_exp2(fmaf(s[n][2 * r + j], sl2, neg));
            l[r] += s[n][2 * r + j];
          }
      }
#pragma unroll
      for (int ks = 0; ks < 2; ++ks) {
        const uint32_t p[4] = {pack_bf16(s[2 * ks][0], s[2 * ks][1]), pack_bf16(s[2 * ks][2], s[2 * ks][3]),
                               pack_bf16(s[2 * ks + 1][0], s[2 * ks + 1][1]), pack_bf16(s[2 * ks + 1][2], s[2 * ks + 1][3])};
#pragma unroll
        for (int dp = 0; dp < HDP / 16; ++dp) {
          const int key = ks * 16 + (lane >> 3 & 1) * 8 + (lane & 7), chunk = (dp & 3) * 2 + (lane >> 4);
          uint32_t b[4];
          ldsm4_t(b, vbase + (dp >> 2) * DBLK * 128 + key * 128 + ((chunk ^ (key & 7)) << 4));
          mma_bf16(o[2 * dp], p, b[0], b[1]);
          mma_bf16(o[2 * dp + 1], p, b[2], b[3]);
        }
      }
      __syncwarp();                                                    // every lane has read the slot
      issue(slot, ahead);
      ahead = look();
      if (++slot == DST) {
        slot = 0;
        phase ^= 1;
      }
    }

    // ---- the four warps' results meet
#pragma unroll
    for (int r = 0; r < 2; ++r) {
      l[r] += __shfl_xor_sync(0xffffffffu, l[r], 1);
      l[r] += __shfl_xor_sync(0xffffffffu, l[r], 2);
      if (qd == 0) stat[warp * DROWS + gr + 8 * r] = make_float2(m[r], l[r]);
    }
    __syncthreads();
    float M[2], sum[2];
#pragma unroll
    for (int r = 0; r < 2; ++r) {
      M[r] = -INFINITY;
      sum[r] = 0.f;
#pragma unroll
      for (int w = 0; w < DWARPS; ++w) M[r] = fmaxf(M[r], stat[w * DROWS + gr + 8 * r].x);
#pragma unroll
      for (int w = 0; w < DWARPS; ++w) {
        const float2 st = stat[w * DROWS + gr + 8 * r];
        sum[r] += st.y * (st.x == -INFINITY ? 1.f : fast_exp2(st.x - M[r]));   // a NaN sum without a maximum is handed on
      }
      const float f = m[r] == -INFINITY ? 1.f : fast_exp2(m[r] - M[r]);
#pragma unroll
      for (int d = 0; d < HDP / 8; ++d) {
        o[d][2 * r] *= f;
        o[d][2 * r + 1] *= f;
      }
    }
    auto put = [&](float* buf) {
#pragma unroll
      for (int d = 0; d < HDP / 8; ++d) {
        *reinterpret_cast<float2*>(buf + gr * HDP + ((d ^ (gr & 3)) * 8) + qd * 2) = make_float2(o[d][0], o[d][1]);
        *reinterpret_cast<float2*>(buf + (gr + 8) * HDP + ((d ^ (gr & 3)) * 8) + qd * 2) = make_float2(o[d][2], o[d][3]);
      }
    };
    auto add = [&](const float* buf) {
#pragma unroll
      for (int d = 0; d < HDP / 8; ++d) {
        const float2 x = *reinterpret_cast<const float2*>(buf + gr * HDP + ((d ^ (gr & 3)) * 8) + qd * 2);
        const float2 y = *reinterpret_cast<const float2*>(buf + (gr + 8) * HDP + ((d ^ (gr & 3)) * 8) + qd * 2);
        o[d][0] += x.x; o[d][1] += x.y; o[d][2] += y.x; o[d][3] += y.y;
      }
    };
    if (warp >= 2) put(merge + (warp - 2) * DROWS * HDP);
    __syncthreads();
    if (warp < 2) add(merge + warp * DROWS * HDP);
    if (warp == 1) put(merge + DROWS * HDP);                           // the half that only this warp reads
    __syncthreads();
    if (warp == 0) {
      add(merge + DROWS * HDP);
      if (a.whole > 1) {                                               // for the cluster to read
#pragma unroll
        for (int d = 0; d < HDP / 8; ++d) {
          *reinterpret_cast<float2*>(merge + gr * HDP + d * 8 + qd * 2) = make_float2(o[d][0], o[d][1]);
          *reinterpret_cast<float2*>(merge + (gr + 8) * HDP + d * 8 + qd * 2) = make_float2(o[d][2], o[d][3]);
        }
        if (qd == 0) {
          stat[gr] = make_float2(M[0], sum[0]);
          stat[gr + 8] = make_float2(M[1], sum[1]);
        }
      } else if (a.whole || (u == it.u0 && ue == it.u0 + it.span.n)) {
        unsigned bad = 0;
#pragma unroll
        for (int r = 0; r < 2; ++r) {
          const float inv = sum[r] == 0.f ? 0.f : 1.f / sum[r];        // a row that sees nothing gives zero
          const int tok = r ? tb : ta, head = it.h * g.rep + (r ? rb : ra) - tok * g.rep;
          __nv_bfloat16* po = a.out + ((long long)(it.s.q0 + tok) * g.H + head) * g.hd;
          bool finite = true;
#pragma unroll
          for (int d = 0; d < HDP / 8; ++d) {
            const float x = o[d][2 * r] * inv, y = o[d][2 * r + 1] * inv;
            finite = finite && isfinite(x) && isfinite(y);
            if (gr + 8 * r < rows && d * 8 < g.hd) *reinterpret_cast<uint32_t*>(po + d * 8 + qd * 2) = pack_bf16(x, y);
          }
          const unsigned who = __ballot_sync(0xffffffffu, !finite);
#pragma unroll
          for (int i = 0; i < 8; ++i) bad |= (who >> (4 * i) & 15u ? 1u : 0u) << (i + 8 * r);
        }
        bad &= (1u << rows) - 1u;
        __syncwarp();
        while (bad) {                                                  // all lanes hold the same word
          const int r = __ffs(bad) - 1;
          bad &= bad - 1;
          const int tok = g.by_rep(r0 + r), head = it.h * g.rep + r0 + r - tok * g.rep;
          const long long at = it.s.q0 + tok;
          float res[HDP / 32];
          paged_row<HDP>(g, a.q + at * a.qs + head * g.hd, a.pages, it.b, it.h, pos0 + tok, a.scale, res);
#pragma unroll
          for (int x = 0; x < HDP / 32; ++x)
            if (lane + 32 * x < g.hd) a.out[(at * g.H + head) * g.hd + lane + 32 * x] = __float2bfloat16(res[x]);
        }
      } else {
        const long long ps = 2LL * blockIdx.x + (u == it.u0);
        float* po = a.part + ps * DROWS * HDP;
#pragma unroll
        for (int d = 0; d < HDP / 8; ++d) {
          if (gr < rows) *reinterpret_cast<float2*>(po + gr * HDP + d * 8 + qd * 2) = make_float2(o[d][0], o[d][1]);
          if (gr + 8 < rows) *reinterpret_cast<float2*>(po + (gr + 8) * HDP + d * 8 + qd * 2) = make_float2(o[d][2], o[d][3]);
        }
        if (qd == 0) {
          float2* st = reinterpret_cast<float2*>(a.stat) + ps * DROWS;
          st[gr] = make_float2(M[0], sum[0]);
          st[gr + 8] = make_float2(M[1], sum[1]);
        }
      }
    }
    u = ue;
    if (u < u_end) paged_next<DBLK>(g, it);
  }
  if (a.whole > 1) join_cluster<HDP>(a, it, merge, stat, u_begin < u_end);
}

// Block c - 1 joins the item that CTA c has noted. Rows, and of few rows the parts too, go to groups of HDP / 4 threads with four columns each.
template <int HDP>
__global__ void __launch_bounds__(256) paged_decode_join_kernel(const __grid_constant__ DecodeArgs a) {
  constexpr int VEC = HDP / 4, GROUPS = 256 / VEC;
  __shared__ float4 sum[GROUPS][VEC];
  __shared__ float total[GROUPS];
  __shared__ unsigned bad;
  const PagedGeom& g = a.g;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, group = threadIdx.x / VEC, v = threadIdx.x % VEC;
  pdl_wait();
  const int c = blockIdx.x + 1;
  const PagedJoin j = a.notes[c];
  if (j.rows == 0) return;
  if (threadIdx.x == 0) bad = 0;
  const int n = j.last - c + 2;                                        // parts: CTAs c - 1 to last
  const int wide = min(j.rows <= 1 ? 1 : 1 << (32 - __clz(j.rows - 1)), GROUPS), subs = GROUPS / wide;   // rows side by side, groups per row
  const int sub = group / wide;
  const float2* stat = reinterpret_cast<const float2*>(a.stat);
  const float4* part = reinterpret_cast<const float4*>(a.part);
  auto slot = [&](int i) { return i == 0 ? 2LL * c - 1 : 2LL * (c - 1 + i); };
  for (int base = 0; base < j.rows; base += wide) {
    const int r = base + group % wide;
    const bool live = r < j.rows;
    float M = -INFINITY;
    for (int i = v; i < n && live; i += VEC) M = fmaxf(M, stat[slot(i) * DROWS + r].x);
#pragma unroll
    for (int o = VEC / 2; o > 0; o >>= 1) M = fmaxf(M, __shfl_xor_sync(0xffffffffu, M, o));
    float4 num = make_float4(0.f, 0.f, 0.f, 0.f);
    float den = 0.f;
    if (live) {
#pragma unroll 4
      for (int i = sub; i < n; i += subs) {
        const float2 st = stat[slot(i) * DROWS + r];
        const float4 x = part[(slot(i) * DROWS + r) * VEC + v];
        const float w = st.x == -INFINITY ? 1.f : fast_exp2(st.x - M); // without a maximum: sums of zero, or a NaN to hand on
        den += w * st.y;
        num.x += w * x.x; num.y += w * x.y; num.z += w * x.z; num.w += w * x.w;
      }
    }
    sum[group][v] = num;
    if (v == 0) total[group] = den;
    __syncthreads();
    if (sub == 0 && live) {
      for (int s = 1; s < subs; ++s) {
        const float4 x = sum[group + s * wide][v];
        num.x += x.x; num.y += x.y; num.z += x.z; num.w += x.w;
        den += total[group + s * wide];
      }
      const float inv = den == 0.f ? 0.f : 1.f / den;
      num.x *= inv; num.y *= inv; num.z *= inv; num.w *= inv;
      if (v * 4 < g.hd) {
        const int tok = g.by_rep(j.r0 + r), head = j.h * g.rep + (j.r0 + r) - tok * g.rep;
        *reinterpret_cast<uint2*>(a.out + ((long long)(j.q0 + tok) * g.H + head) * g.hd + v * 4) = make_uint2(pack_bf16(num.x, num.y), pack_bf16(num.z, num.w));
        if (!(isfinite(num.x) && isfinite(num.y) && isfinite(num.z) && isfinite(num.w))) atomicOr(&bad, 1u << r);
      }
    }
    __syncthreads();
  }
  for (int r = warp; r < j.rows; r += 8) {
    if (!(bad >> r & 1u)) continue;
    const int tok = g.by_rep(j.r0 + r), head = j.h * g.rep + (j.r0 + r) - tok * g.rep;
    const long long at = j.q0 + tok;
    float res[HDP / 32];
    paged_row<HDP>(g, a.q + at * a.qs + head * g.hd, a.pages, j.b, j.h, j.pos0 + tok, a.scale, res);
#pragma unroll
    for (int x = 0; x < HDP / 32; ++x)
      if (lane + 32 * x < g.hd) a.out[(at * g.H + head) * g.hd + lane + 32 * x] = __float2bfloat16(res[x]);
  }
}

// The number of CTAs is rounded up, so a share has at least half of these (15 units make shares of 8 and 7): it may lie within an item's empty units, and is a part
// of nothing then.
constexpr int MIN_UNITS = 4 + paged_front<DBLK>;

int decode_grid(int hd) { return 148 * (hd <= 64 ? 2 : 1); }
// CTAs per item (a cluster) where items are alike or cannot be long, 0 for the line of units. us, line against clusters (their size), 16 heads of 64, in a graph (the GPU's part)
// and as a call among others (the line has two launches and scratch for the host to see to): 1 sequence of 2000 11.2, 10.0 and 24, 13 (8); of 8000 12.8, 15.6 and 18, 18 (8); of
// 10000 14.3, 17.9 and 18, 21 (8); 4 of 2000 12.8, 11.6 and 18, 14 (4); 16 of 1000 19.0, 14.2 and 22, 17 (1). So one sequence of 8000 to 10000 would be the line's by now, and from
// 10240 on it is. 32000 keys: 34 and 42. 16 of 2000: 35 and 29, but then, as among 4 of 8000, one long sequence among short ones would hold up the others.
int decode_whole(int B, int Hkv, int hd, int max_new, int rep, long long cache, int window, int sinks) {
  if ((long long)max_new * rep > DROWS) return 0;
  const long long items = (long long)B * Hkv, seen = (long long)window + max_new + sinks + 2 * DBLK, most = window && seen < cache ? seen : cache;
  if (most <= 512) return 1;
  for (int n = 8; n > 1; n /= 2)           // clusters that run at once: one CTA per SM (two of 64-wide heads), and clusters of eight leave some out
    if (items * n <= (hd <= 64 ? 256 : 128) && most >= 256 * n && most <= 1280 * n && (window || B == 1 || most <= 2048)) return n;
  return most <= 1024 && items >= 64;
}

template <int HDP>
int launch_decode(DecodeArgs& a, int page, cudaStream_t st) {
  CUtensorMap tm;
  const int rc = make_paged_tmap(&tm, a.pages, a.g.P, a.g.Hkv, page, a.g.hd, page < DBLK ? page : DBLK);
  if (rc != ELFA_OK) return rc;
  const int smem = DecodeSmem<HDP>::bytes(a.whole ? 0 : a.g.B);
  ELFA_CUDA(allow_shared<paged_decode_kernel<HDP>>(DecodeSmem<HDP>::bytes(PAGED_MAX_SEQS)));
  const int grid = a.whole ? a.g.B * a.g.Hkv * a.whole : decode_grid(a.g.hd);
  cudaLaunchConfig_t cfg{};
  cfg.gridDim = dim3((unsigned)grid);
  cfg.blockDim = dim3(DWARPS * 32);
  cfg.dynamicSmemBytes = smem;
  cfg.stream = st;
  cudaLaunchAttribute at[1];
  at[0].id = cudaLaunchAttributeClusterDimension;
  at[0].val.clusterDim.x = a.whole;
  at[0].val.clusterDim.y = at[0].val.clusterDim.z = 1;
  cfg.attrs = at;
  cfg.numAttrs = a.whole > 1 ? 1 : 0;
  ELFA_CUDA(cudaLaunchKernelEx(&cfg, paged_decode_kernel<HDP>, tm, a));
  ELFA_CUDA(cudaGetLastError());
  ::elfa::count_launches(1);
  if (a.whole) return ELFA_OK;
  PdlScope scope(true);
  ELFA_CUDA(launch_chain(paged_decode_join_kernel<HDP>, dim3(grid - 1), dim3(256), 0, st, 1, a));
  ELFA_CUDA(cudaGetLastError());
  ::elfa::count_launches(1);
  return ELFA_OK;
}

}  // namespace

// Pages as [P * 2 * Hkv][page][hd]: a box is `box_rows` tokens of one page and head, 64 columns.
int make_paged_tmap(CUtensorMap* tm, const void* pages, long long P, int Hkv, int page, int hd, int box_rows) {
  const uint64_t dims[3] = {(uint64_t)hd, (uint64_t)page, (uint64_t)(2 * P * Hkv)};
  const uint64_t strides[2] = {(uint64_t)hd * 2, (uint64_t)hd * page * 2};
  const uint32_t box[3] = {64, (uint32_t)box_rows, 1};
  return make_tmap_nd_bf16(tm, pages, 3, dims, strides, box);
}

// Checks that both forms of the attention and the write share, and the geometry.
int paged_geom(PagedGeom* g, const void* pages, const int* table, const int* q_start, const int* kv_len, int B, int N, int P, int page, int T, int H,
               int Hkv, int hd, int max_new, int window, int sinks) {
  ELFA_REQUIRE(pages && table && q_start && kv_len, "paged: null pointer");
  ELFA_REQUIRE(B > 0 && N > 0 && P > 0 && T > 0 && Hkv > 0 && H > 0 && H % Hkv == 0 && max_new > 0, "paged: bad sizes");
  ELFA_REQUIRE(page >= 16 && page <= 256 && (page & (page - 1)) == 0, "paged: tokens per page must be 16, 32, 64, 128 or 256");
  ELFA_REQUIRE(hd >= 8 && hd <= 128 && hd % 8 == 0, "paged: head dimension must be a multiple of 8 up to 128");
  ELFA_REQUIRE((long long)P * 2 * Hkv < 0x7fffffffLL && (long long)N * page < 0x7fffff00LL, "paged: too many pages");
  ELFA_REQUIRE((long long)T * (H / Hkv) < 0x7ffff000LL, "paged: too many query rows");
  ELFA_REQUIRE(window >= 0 && sinks >= 0, "paged: negative window or sinks");
  ELFA_REQUIRE((reinterpret_cast<uintptr_t>(pages) & 15) == 0, "paged: pages must be 16-byte aligned");
  g->status = status_word();
  ELFA_REQUIRE(g->status != nullptr, "paged: no status word");
  g->table = table; g->q_start = q_start; g->kv_len = kv_len;
  g->B = B; g->N = N; g->P = P; g->T = T; g->max_new = max_new;
  g->page_shift = __builtin_ctz((unsigned)page);
  g->H = H; g->Hkv = Hkv; g->rep = H / Hkv; g->hd = hd;
  g->by_rep = div_by((unsigned)g->rep);
  g->window = window > (1 << 30) ? 0 : window;
  g->sinks = sinks > (1 << 30) ? 1 << 30 : sinks;
  g->ends = 3;
  return ELFA_OK;
}

// paged_prefill.cu
long long paged_prefill_scratch(int hd);
int paged_prefill(PagedGeom g, const void* q, long long qs, const void* pages, void* out, float* scratch, int page, float scale, cudaStream_t st);

// Units are counted in 32 bits.
bool paged_units_fit(const PagedGeom& g, int block) {
  const double tiles = (double)g.T * g.rep / g.tile_rows + g.B, blocks = ((double)g.N * (1 << g.page_shift)) / block + 2 + paged_front<32>;
  return tiles * blocks * g.Hkv < 4.0e9;
}

// Which calls go to the tiles of 2 x 128 rows, by the rows of a key head. 16-row tiles read the keys again for every 16 rows, 128-row tiles take as long for one row as for
// all. us, 16-row tiles against 128-row tiles: 8 sequences of 3000, 16 heads of 128: 16 rows 49, 60; 24 rows 73, 60; 48 rows 97, 61. Heads of 64: 32 rows 45, 51; 48 rows 55, 51.
// 32 of 2000, 32 heads on 8 of 128: 16 rows 59, 76; 24 rows 97, 78. One of 30000: 16 rows 42, 49; 24 rows 50, 50; 48 rows 67, 51. Where the bound is far above what most
// sequences have (up to 32 rows, half of that on average) 16-row tiles would be the faster ones, 50 against 57 us; the host knows the bound only. It is why
// 64-wide heads change forms above 48 rows, where a call that has all of the bound's rows would at 48.
static bool many_rows(int max_new, int rep, int hd) { return (long long)max_new * rep > (hd > 64 ? 16 : 48) && rep <= 128; }

}  // namespace elfa

using namespace elfa;

// Floats of scratch that elfa_paged_attention wants for a call of these sizes.
ELFA_API int elfa_paged_attention_scratch(int B, int N, int page, int H, int Hkv, int hd, int max_new, int window, int sinks) {
  if (B <= 0 || N <= 0 || page <= 0 || Hkv <= 0 || H % Hkv || max_new <= 0) return 0;
  if (many_rows(max_new, H / Hkv, hd)) return (int)paged_prefill_scratch(hd);
  const int full = B < PAGED_MAX_SEQS ? B : PAGED_MAX_SEQS, rest = B % PAGED_MAX_SEQS;      // sequences of the launches
  const long long cache = (long long)N * page;
  if (decode_whole(full, Hkv, hd, max_new, H / Hkv, cache, window, sinks) && (!rest || decode_whole(rest, Hkv, hd, max_new, H / Hkv, cache, window, sinks))) return 0;
  return decode_grid(hd) * (2 * DROWS * ((hd <= 64 ? 64 : 128) + 2) + 8);
}

namespace {

// One launch (and its join), of at most PAGED_MAX_SEQS sequences.
int paged_part(const PagedGeom& g, const void* q, long long qs, const void* pages, void* out, float* scratch, int page, float scale, cudaStream_t st) {
  if (many_rows(g.max_new, g.rep, g.hd)) {
    ELFA_REQUIRE(scratch && (reinterpret_cast<uintptr_t>(scratch) & 15) == 0, "paged_attention: no scratch, or not 16-byte aligned");
    return paged_prefill(g, q, qs, pages, out, scratch, page, scale, st);
  }
  DecodeArgs a{};
  a.g = g;
  a.q = static_cast<const __nv_bfloat16*>(q);
  a.pages = static_cast<const __nv_bfloat16*>(pages);
  a.out = static_cast<__nv_bfloat16*>(out);
  a.qs = qs;
  a.scale = scale;
  a.g.tile_rows = DROWS;
  a.g.by_tile = div_by(DROWS);
  a.whole = decode_whole(g.B, g.Hkv, g.hd, g.max_new, g.rep, (long long)g.N * page, g.window, g.sinks);
  a.wide = ((long long)g.max_new * g.rep + DROWS - 1) / DROWS > 4;
  a.min_units = MIN_UNITS;
  ELFA_REQUIRE(paged_units_fit(a.g, DBLK), "paged_attention: too much work for one call (2^32 tiles of 16 rows by 32 keys)");
  ELFA_REQUIRE(a.whole || (scratch && (reinterpret_cast<uintptr_t>(scratch) & 15) == 0), "paged_attention: no scratch, or not 16-byte aligned");
  a.part = scratch;
  a.stat = scratch + 2LL * decode_grid(g.hd) * DROWS * (g.hd <= 64 ? 64 : 128);
  a.notes = reinterpret_cast<PagedJoin*>(a.stat + 2LL * decode_grid(g.hd) * DROWS * 2);
  return g.hd <= 64 ? launch_decode<64>(a, page, st) : launch_decode<128>(a, page, st);
}

}  // namespace

// q: rows [T] of H heads, `qs` elements apart, heads packed, 16-byte aligned; out: [T, H * hd] contiguous. max_new: at least the most new tokens of a sequence.
ELFA_API int elfa_paged_attention(const void* q, long long qs, const void* pages, const int* table, const int* q_start, const int* kv_len, void* out,
                                  float* scratch, int B, int N, int P, int page, int T, int H, int Hkv, int hd, int max_new, int window, int sinks,
                                  float scale, void* stream) {
  PagedGeom g{};
  int rc = paged_geom(&g, pages, table, q_start, kv_len, B, N, P, page, T, H, Hkv, hd, max_new, window, sinks);
  if (rc != ELFA_OK) return rc;
  ELFA_REQUIRE(q && out, "paged_attention: null pointer");
  ELFA_REQUIRE(qs % 8 == 0 && (reinterpret_cast<uintptr_t>(q) & 15) == 0 && (reinterpret_cast<uintptr_t>(out) & 15) == 0,
               "paged_attention: query rows must lie on 16-byte boundaries");
  for (int b = 0; b < B; b += PAGED_MAX_SEQS) {            // q_start counts from the first row of the whole call in every launch
    PagedGeom part = g;
    part.B = B - b < PAGED_MAX_SEQS ? B - b : PAGED_MAX_SEQS;
    part.table = table + (long long)b * N;
    part.q_start = q_start + b;
    part.kv_len = kv_len + b;
    part.ends = (b == 0 ? 1 : 0) | (part.B == B - b ? 2 : 0);
    rc = paged_part(part, q, qs, pages, out, scratch, page, scale, static_cast<cudaStream_t>(stream));
    if (rc != ELFA_OK) return rc;
  }
  return ELFA_OK;
}
