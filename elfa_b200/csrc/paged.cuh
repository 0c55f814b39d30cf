// What the kernels over a paged key / value cache share: the geometry of a call and how its work is cut.
//
// pages [P, 2, Hkv, page, hd] bf16; table [B, N] int32 names the pages of each sequence in order (negative: absent); sequence b brings the new
// tokens q_start[b] .. q_start[b + 1] of the call and has kv_len[b] tokens with them, so its i-th new token stands at kv_len - n + i. A query at
// `pos` sees the keys that lie in pages that are there and for which key <= pos and (key > pos - window or key < sinks).
//
// Work is counted in units: one tile of query rows (rows are (token, head of the group) pairs, token first, so a key is read once for all heads
// that share it) against one block of keys. The units of all (sequence, tile, key head) items stand in one line, blocks innermost, and each of G
// CTAs takes W / G of them (the first ones one more each): the same number whatever the sequences' lengths are, and the host needs to know none of
// them. An item that a CTA does not hold whole leaves a partial result: slot 2 c + 1 for the part that begins it, slot 2 c for a later part.
#pragma once
#include "common.cuh"

namespace elfa {

constexpr int PAGED_MAX_SEQS = 1024;       // of a launch of the attention, whose CTAs keep all sequences in shared memory; larger batches are cut into launches

// x / d for 0 <= x < 2^31 and a d that the host knows: with 2^s the power of two from d on and m = floor(2^32 (2^s - d) / d) + 1, (mulhi(x, m) + x) >> s
// (the round-up method for invariant divisors). A division costs some 40 instructions, and the walk over items is made of them.
struct DivBy {
  unsigned d, m, s;
  __device__ __forceinline__ int operator()(int x) const { return (int)((__umulhi((unsigned)x, m) + (unsigned)x) >> s); }
};
inline DivBy div_by(unsigned d) {
  unsigned s = 0;
  while ((1u << s) < d) ++s;
  return {d, (unsigned)((((unsigned long long)1 << 32) * ((1ull << s) - d)) / d + 1), s};
}

struct PagedGeom {
  const int *table, *q_start, *kv_len;
  int B, N, P, page_shift, T, max_new;     // T: rows of q; max_new: the most new tokens that the host has planned for
  int H, Hkv, rep, hd;
  int window, sinks;                       // window 0: none
  int tile_rows;                           // query rows of a tile
  DivBy by_rep, by_tile;                   // / rep, / tile_rows
  int ends;                                // 1: this launch has the call's first sequence, which begins at row 0; 2: its last, which ends at row T
  unsigned int* status;
};

struct PagedSeq {
  int q0, n, kv;                           // first new token, new tokens, tokens with them
};

// in_order: whether the sequence's rows are a piece of the call's. Where those of all sequences are, no row has two sequences (each starts where the one before ends).
__device__ __forceinline__ PagedSeq paged_seq(const PagedGeom& g, int b, bool* in_order = nullptr) {
  const int a = g.q_start[b], e = g.q_start[b + 1], kv = g.kv_len[b];
  const long long most = (long long)g.N << g.page_shift;
  PagedSeq s;
  s.q0 = min(max(a, 0), g.T);
  s.n = min(max(e, s.q0), g.T) - s.q0;
  s.kv = (int)min((long long)max(kv, 0), min(most, 0x7fffff00LL));
  if (s.q0 != a || s.q0 + s.n != e || s.kv != kv || s.n > s.kv || s.n > g.max_new || (b == 0 && (g.ends & 1) && a != 0) || (b == g.B - 1 && (g.ends & 2) && e != g.T))
    atomicOr(g.status, (unsigned)ELFA_ST_BAD_PAGE);
  if (in_order) *in_order = s.q0 == a && s.q0 + s.n == e;
  return s;
}
// Rows that no sequence has give zeros: those in front of the launch's first sequence and behind its last one, by all threads of one block.
// Out of line: the decoding kernel has no register to spare (inlined, it spills 36 bytes).
template <int = 0>
__device__ __noinline__ void paged_zero_rows(const PagedGeom& g, __nv_bfloat16* out, int from, int to) {
  uint4* p = reinterpret_cast<uint4*>(out);
  const long long row = (long long)g.H * g.hd / 8;
  for (long long i = from * row + threadIdx.x; i < to * row; i += blockDim.x) p[i] = make_uint4(0u, 0u, 0u, 0u);
}
__device__ __forceinline__ void paged_rest(const PagedGeom& g, __nv_bfloat16* out, const PagedSeq& first, const PagedSeq& last) {
  if (g.ends & 1) paged_zero_rows(g, out, 0, first.q0);
  if (g.ends & 2) paged_zero_rows(g, out, last.q0 + last.n, g.T);
}
__device__ __forceinline__ int paged_tiles(const PagedGeom& g, const PagedSeq& s) {
  return g.by_tile(s.n * g.rep + g.tile_rows - 1);
}

// An item's end (partial results meet, the result is written) takes as long as some blocks: with 16-row tiles it stands in the line as that many empty units in
// front of the item, or a CTA whose share is many short items would be the last by far. us with 0, 3, 5, 7, 10, 14 of them: 48 sequences to 8191, 32 heads on 8 of
// 128: 165, 157, 150, 147, 147, 150; 64 to 1500: 91, 69, 58, 56, 52, 52; 16 to 1500, 16 heads of 64: 47, 28, 23, 23, 23, 24.
template <int BLK>
constexpr int paged_front = BLK == 32 ? 10 : 0;

// key blocks that the rows of a tile see: i < ns is block i (sinks), later ones are w0 + i - ns. A tile that sees nothing still has one block.
struct PagedSpan {
  int ns, w0, n;                           // n: units, with the empty ones in front
  __device__ __forceinline__ int block(int i) const { return i < ns ? i : w0 + i - ns; }
};
template <int BLK>
__device__ __forceinline__ PagedSpan paged_span(const PagedGeom& g, const PagedSeq& s, int t) {
  const int r0 = t * g.tile_rows, lo_tok = g.by_rep(r0), hi_tok = g.by_rep(min(r0 + g.tile_rows, s.n * g.rep) - 1);
  const int pos0 = s.kv - s.n, hi = max(pos0 + hi_tok + 1, 0);
  const int lo = g.window ? max(0, pos0 + lo_tok - g.window + 1) : 0;
  PagedSpan p;
  p.w0 = lo / BLK;
  p.ns = g.window ? min((min(g.sinks, hi) + BLK - 1) / BLK, p.w0) : 0;
  p.n = max(p.ns + (hi + BLK - 1) / BLK - p.w0, 1) + paged_front<BLK>;
  return p;
}

// units of a sequence (all tiles, all key heads); `lane` of `lanes` threads adds up every lanes-th tile. The host has seen to it that all units of a call fit 32 bits.
template <int BLK>
__device__ __forceinline__ unsigned paged_units(const PagedGeom& g, const PagedSeq& s, int lane, int lanes) {
  const int tiles = paged_tiles(g, s);
  unsigned u = 0;
  for (int t = lane; t < tiles; t += lanes) u += paged_span<BLK>(g, s, t).n;
  return u * g.Hkv;
}

// What every CTA works out for itself, in shared memory: prefix[b] = units before sequence b, prefix[B] = W, and the sequences.
struct PagedLine {
  unsigned* prefix;                        // [B + 1]
  PagedSeq* seqs;                          // [B]
  unsigned* warp_tot;                      // [warps]
};
constexpr int paged_line_bytes(int B) { return 4 * (B + 1) + (int)sizeof(PagedSeq) * B; }
__device__ __forceinline__ PagedLine paged_line(void* at, int B, unsigned* warp_tot) {
  unsigned* p = static_cast<unsigned*>(at);
  return {p, reinterpret_cast<PagedSeq*>(p + B + 1), warp_tot};
}
// By all threads of the block (ends with a barrier); returns W. Rows that several sequences claim would make more units than the host has allowed for (more than 32
// bits hold): such a call has no units, and the status word says why. wide: a warp per sequence (many tiles each).
template <int BLK, int THREADS>
__device__ __forceinline__ unsigned paged_prefix(const PagedGeom& g, const PagedLine& line, bool wide) {
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  constexpr int WARPS = THREADS / 32;
  bool in_order = true;
  if (wide) {
    for (int b = warp; b < g.B; b += WARPS) {
      bool here;
      const PagedSeq s = paged_seq(g, b, &here);
      in_order = in_order && here;
      const unsigned u = __reduce_add_sync(0xffffffffu, paged_units<BLK>(g, s, lane, 32));
      if (lane == 0) {
        line.prefix[b + 1] = u;
        line.seqs[b] = s;
      }
    }
    __syncthreads();
  }
  unsigned run = 0;
  for (int b0 = 0; b0 < g.B; b0 += THREADS) {
    const int b = b0 + threadIdx.x;
    unsigned u = 0;
    if (b < g.B) {
      if (wide) {
        u = line.prefix[b + 1];
      } else {
        bool here;
        const PagedSeq s = paged_seq(g, b, &here);
        in_order = in_order && here;
        line.seqs[b] = s;
        u = paged_units<BLK>(g, s, 0, 1);
      }
    }
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const unsigned v = __shfl_up_sync(0xffffffffu, u, o);
      if (lane >= o) u += v;
    }
    if (g.B > 32) {                        // else the first warp has all of them
      if (lane == 31) line.warp_tot[warp] = u;
      __syncthreads();
      unsigned before = run;
#pragma unroll
      for (int w = 0; w < WARPS; ++w) {
        if (w < warp) before += line.warp_tot[w];
        run += line.warp_tot[w];
      }
      u += before;
      if (b0 + THREADS < g.B) __syncthreads();
    }
    if (b < g.B) line.prefix[b + 1] = u;
  }
  if (threadIdx.x == 0) line.prefix[0] = 0;
  return __syncthreads_and(in_order) ? line.prefix[g.B] : 0;
}

struct PagedItem {
  int b, t, h;
  PagedSeq s;
  PagedSpan span;
  unsigned u0;                             // unit of its block 0
  int tiles;
};

// the item that unit u belongs to; all lanes of a warp call it together
template <int BLK>
__device__ __forceinline__ PagedItem paged_find(const PagedGeom& g, const PagedLine& line, unsigned u) {
  int lo = 0, hi = g.B;                    // prefix[lo] <= u < prefix[hi]
  while (hi - lo > 1) {
    const int mid = (lo + hi) >> 1;
    if (line.prefix[mid] <= u) lo = mid;
    else hi = mid;
  }
  PagedItem it;
  it.b = lo;
  it.s = line.seqs[lo];
  it.tiles = paged_tiles(g, it.s);
  const int lane = threadIdx.x & 31;
  unsigned base = line.prefix[lo];
  it.t = 0;
  if (it.tiles > 1) {
    for (int t0 = 0;; t0 += 32) {
      const int t = t0 + lane;
      const unsigned mine = t < it.tiles ? (unsigned)paged_span<BLK>(g, it.s, t).n * g.Hkv : 0;
      unsigned incl = mine;
#pragma unroll
      for (int o = 1; o < 32; o <<= 1) {
        const unsigned v = __shfl_up_sync(0xffffffffu, incl, o);
        if (lane >= o) incl += v;
      }
      const unsigned hit = __ballot_sync(0xffffffffu, base + incl > u && t < it.tiles);
      if (hit || t0 + 32 >= it.tiles) {
        const int l = hit ? __ffs(hit) - 1 : it.tiles - 1 - t0;
        it.t = t0 + l;
        base += __shfl_sync(0xffffffffu, incl - mine, l);
        break;
      }
      base += __shfl_sync(0xffffffffu, incl, 31);
    }
  }
  it.span = paged_span<BLK>(g, it.s, it.t);
  it.h = (int)((u - base) / (unsigned)it.span.n);
  it.u0 = base + (unsigned)it.h * it.span.n;
  return it;
}
// the next item in line (there is one as long as its first unit is below W)
template <int BLK>
__device__ __forceinline__ void paged_next(const PagedGeom& g, PagedItem& it) {
  it.u0 += it.span.n;
  if (++it.h < g.Hkv) return;
  it.h = 0;
  if (++it.t >= it.tiles) {
    it.t = 0;
    do {
      if (++it.b >= g.B) {                 // behind the last one
        it.b = g.B - 1;
        break;
      }
      it.s = paged_seq(g, it.b);
      it.tiles = paged_tiles(g, it.s);
    } while (it.tiles == 0);
  }
  it.span = paged_span<BLK>(g, it.s, it.t);
}

// The shares of G CTAs (G <= W).
struct PagedShares {
  unsigned each, more;                     // units of a CTA; how many of them have one more
  __device__ __forceinline__ PagedShares(unsigned W, unsigned G) : each(G ? W / G : 0), more(G ? W - each * G : 0) {}
  __device__ __forceinline__ unsigned first(unsigned c) const { return c * each + min(c, more); }
  __device__ __forceinline__ int owner(unsigned u) const {
    const unsigned front = more * (each + 1);
    return (int)(u < front ? u / (each + 1) : more + (u - front) / each);
  }
};

// What joins an item that several CTAs have parts of, written by the CTA that the item's first cut lies in front of: its parts are slot 2 first + 1 and
// slots 2 c for first < c <= last. rows 0: nothing to join here.
struct alignas(16) PagedJoin {
  int rows, last, b, h, r0, q0, pos0, unused;
};
__device__ __forceinline__ void paged_join_note(const PagedGeom& g, PagedJoin* notes, const PagedItem& it, const PagedShares& shares, int c, bool cut) {
  PagedJoin j{};
  if (cut && shares.owner(it.u0) == c - 1) {
    j.rows = min(g.tile_rows, it.s.n * g.rep - it.t * g.tile_rows);
    j.last = shares.owner(it.u0 + it.span.n - 1);
    j.b = it.b;
    j.h = it.h;
    j.r0 = it.t * g.tile_rows;
    j.q0 = it.s.q0;
    j.pos0 = it.s.kv - it.s.n;
  }
  notes[c] = j;
}

__device__ __forceinline__ bool paged_sees(const PagedGeom& g, int key, int pos) {
  return key <= pos && (!g.window || key > pos - g.window || key < g.sinks);
}
// page of a key, negative when absent or outside the pool (which is recorded)
__device__ __forceinline__ int paged_page(const PagedGeom& g, int b, int key) {
  const int col = key >> g.page_shift;
  if (col >= g.N) return -1;
  const int id = g.table[(long long)b * g.N + col];
  if (id >= g.P) {
    atomicOr(g.status, (unsigned)ELFA_ST_BAD_PAGE);
    return -1;
  }
  return id;
}

// One query row by one warp, key after key, nothing but what it sees: for rows whose result in the matrix form is not finite, which a
// hidden value that is not finite makes of it too (0 times infinity). Lane l gets the columns l, l + 32, ...
template <int HDP>
__device__ __noinline__ void paged_row(const PagedGeom& g, const __nv_bfloat16* q, const __nv_bfloat16* pages, int b, int h, int pos, float scale,
                                       float (&out)[HDP / 32]) {
  const int lane = threadIdx.x & 31;
  const long long head = (long long)g.hd << g.page_shift;                    // elements of one head of a page
  const int mask = (1 << g.page_shift) - 1;
  auto row_of = [&](int id, int key, int kv) { return pages + (((long long)id * 2 + kv) * g.Hkv + h) * head + (long long)(key & mask) * g.hd; };
  auto score = [&](int key, bool& seen) {
    seen = paged_sees(g, key, pos);
    const int id = seen ? paged_page(g, b, key) : -1;
    seen = id >= 0;
    float a = 0.f;
    if (seen) {
      const __nv_bfloat16* k = row_of(id, key, 0);
      for (int c = 0; c < g.hd; ++c) a += __bfloat162float(q[c]) * __bfloat162float(k[c]);
    }
    return a * scale;
  };
  float m = -INFINITY, l = 0.f;
  const int lo = g.window ? max(0, pos - g.window + 1) : 0, skip = g.window ? min(min(g.sinks, lo), pos + 1) : 0;
  const int count = pos < 0 ? 0 : skip + pos + 1 - lo;                       // visible keys: 0 .. skip, lo .. pos
  auto key_at = [&](int i) { return i < skip ? i : lo + i - skip; };
  for (int i = lane; i < count; i += 32) {
    bool seen;
    const float s = score(key_at(i), seen);
    if (seen) m = fmaxf(m, s);                                               // a NaN score comes back with its exponential
  }
  m = warp_max(m);
  const float ref = m == -INFINITY ? 0.f : m;
  for (int x = 0; x < HDP / 32; ++x) out[x] = 0.f;
  for (int i0 = 0; i0 < count; i0 += 32) {
    bool seen = false;
    const int key = i0 + lane < count ? key_at(i0 + lane) : -1;
    float p = 0.f;
    if (key >= 0) {
      const float s = score(key, seen);
      if (seen) p = expf(s - ref);
    }
    l += p;
    const unsigned who = __ballot_sync(0xffffffffu, seen);
    for (int j = 0; j < 32; ++j) {
      const float w = __shfl_sync(0xffffffffu, p, j);
      const int kj = __shfl_sync(0xffffffffu, key, j);
      if (!(who >> j & 1)) continue;
      const __nv_bfloat16* v = row_of(paged_page(g, b, kj), kj, 1);
#pragma unroll
      for (int x = 0; x < HDP / 32; ++x)
        if (lane + 32 * x < g.hd) out[x] += w * __bfloat162float(v[lane + 32 * x]);
    }
  }
  l = warp_sum(l);
#pragma unroll
  for (int x = 0; x < HDP / 32; ++x) out[x] = count == 0 || l == 0.f ? 0.f : out[x] / l;
}

}  // namespace elfa
