// One token per row of logits: temperature, top-k, top-p, min-p, drawn with given exponential variates.
//
// w_i = exp((x_i - max x) / T). In the order of falling x (equal ones by index) every filter keeps a prefix: the first k; of those the
// shortest one with mass >= p of theirs; of those the ones with w_i >= min_p. What is kept races: the token with the largest w_i / e_i wins, which
// for independent exponential variates e_i is token i with probability w_i / sum w (the lowest index where two are equal). T <= 0 takes the first largest logit, and so
// does a row of which nothing races (min_p above 1; variates that are NaN). A NaN logit counts as -inf; a row without any number above -inf gives -1.
//
// Sums are of fp32 weights, joined in fp32 or fp64; what decides between two tokens is fp32. Counts and places are integers, so a result does not depend on the order in
// which threads come. Bound by latency where rows are few (a dozen meetings of a row's CTAs: one row of 32000, all filters, 20 us) and by the passes' instructions
// where they are many: 96 rows of 131072, top-p, 75 us out of the L2 and 84 from memory, of a CTA's row maximum 12, counting 19, window 8, race 30, sort 5.
// Where a nucleus ends is decided by sums of exponentials that are off by 2^-22 each: where its line passes within some 10^-6 of the mass of a token's edge either may be
// the last.
#include <math_constants.h>

#include <type_traits>

#include "common.cuh"
#include "elfa_native.h"

namespace elfa {
namespace {

struct SampleArgs {
  const void* logits;
  const float* noise;
  long long ld, ldn;
  const float* temperature;
  const int* top_k;
  const float *top_p, *min_p;
  float temperature_all, top_p_all, min_p_all;           // for all rows where the pointer is null
  int top_k_all;
  long long* out;
  int V;
};

// increasing in x; -inf (and NaN, which loads replace by it) is the smallest
__device__ __forceinline__ uint32_t order_key(float x) {
  const uint32_t u = __float_as_uint(x + 0.f);           // -0 and 0 are equal
  return u & 0x80000000u ? ~u : u | 0x80000000u;
}

constexpr int ST = 512, SW = ST / 32;      // threads of a CTA
constexpr int BINS = 8192, LIST = 4096;    // bins of width T / 256 below the maximum; tokens that are sorted
constexpr float BINS_PER = 256.f;
// Vectors of 16 bytes that a thread asks for at once, tokens of the race's batches: about what 64 registers hold (the kernel around the passes spills 162 bytes of fp32
// rows, 34 of bf16 ones; twice as many of either cost 7 to 25 %).
constexpr int EACH = 2, RACE = 8;

// (key, index) as one number: larger is earlier in the order of falling logits, equal ones by index. Never 0.
__device__ __forceinline__ unsigned long long place(float x, int i) { return (unsigned long long)order_key(x) << 32 | (uint32_t)~i; }
__device__ __forceinline__ int index_of(unsigned long long c) { return (int)~(uint32_t)c; }
__device__ __forceinline__ float value_of(unsigned long long c) {
  const uint32_t u = (uint32_t)(c >> 32);
  return __uint_as_float(u & 0x80000000u ? u & 0x7fffffffu : ~u);
}

struct SampleShared {
  union {
    unsigned int hist[BINS];               // tokens per bin of this CTA's part of the row
    unsigned long long list[LIST];         // places of its tokens in the window; in the first CTA then of all of them, in order
  };
  unsigned int merged[BINS];               // tokens per bin of the row, in the first CTA
  unsigned long long swap[LIST];
  double2 mail[2][8];                      // what the CTAs of the row send each other, by turns
  double2 red[SW];
  double2 scan[SW];
  unsigned long long cut;                  // the last token that is kept
  double mass, target;
  long long before, upto;                  // tokens before and up to the end of the window
  int b1, b2;                              // the window: bins that a filter's line may run through
  int fill, pos, mode;                     // entries of the list; kept ones of them; what comes next
};
enum { SORT_ALL, SORT_WINDOW, SEARCH };

// A CTA's part of a row: single elements up to a 16-byte boundary (the first CTA's), vectors of 16 bytes, single ones behind the last vector (the last CTA's).
template <typename T>
struct Part {
  static constexpr int PER = 16 / sizeof(T);
  const T* x;
  int V, head, vecs, v0, v1;
  bool front, back;

  __device__ __forceinline__ static float value(T v) {     // of a NaN and -inf the latter
    if constexpr (std::is_same<T, float>::value) return fmaxf(v, -CUDART_INF_F);
    else return fmaxf(__bfloat162float(v), -CUDART_INF_F);
  }
  __device__ __forceinline__ const uint4* vectors() const { return reinterpret_cast<const uint4*>(x + head); }
  // f(index) of the single ones
  template <typename F>
  __device__ __forceinline__ void singles(F&& f) const {
    if (front && threadIdx.x < head) f((int)threadIdx.x);
    const int tail = head + vecs * PER + threadIdx.x;
    if (back && tail < V) f(tail);
  }
  // f(value, index), U vectors asked for at once and a batch ahead
  template <int U, typename F>
  __device__ __forceinline__ void each(F&& f) const {
    singles([&](int i) { f(value(x[i]), i); });
    const uint4* xv = vectors();
    uint4 w[U];
#pragma unroll
    for (int u = 0; u < U; ++u)
      if (v0 + (int)threadIdx.x + u * ST < v1) w[u] = __ldg(xv + v0 + threadIdx.x + u * ST);
    for (int v = v0 + threadIdx.x; v < v1; v += U * ST) {
      uint4 now[U];
#pragma unroll
      for (int u = 0; u < U; ++u) now[u] = w[u];
#pragma unroll
      for (int u = 0; u < U; ++u)
        if (v + (U + u) * ST < v1) w[u] = __ldg(xv + v + (U + u) * ST);
#pragma unroll
      for (int u = 0; u < U; ++u) {
        if (v + u * ST >= v1) break;
        const T* e = reinterpret_cast<const T*>(&now[u]);
#pragma unroll
        for (int k = 0; k < PER; ++k) f(value(e[k]), head + (v + u * ST) * PER + k);
      }
    }
  }
};

struct Weights {
  float mx, temp, per;
  __device__ __forceinline__ float exact(float v) const { return v == mx ? 1.f : expf((v - mx) / temp); }
  // y = 256 (mx - v) / T, 0 for the largest whatever it is (inf - inf is a NaN), never falling as v falls; exp(-y / 256) for the sums: 2^-22 of each
  __device__ __forceinline__ float depth(float v) const { return fmaxf(mx - v, 0.f) * per; }
  __device__ __forceinline__ static float rough(float y) { return fast_exp2(y * (-1.4426950408889634f / BINS_PER)); }
};

__device__ __forceinline__ void enter_race(unsigned long long& win, float w, float e, int i) {
  const float sc = w / e;
  if (sc >= 0.f) win = max(win, (unsigned long long)__float_as_uint(sc) << 32 | (uint32_t)~i);
}

// The passes over a row are functions of their own, with all registers for a loop each.
template <typename T>
__device__ __noinline__ float part_max(Part<T> p) {
  float mx = -CUDART_INF_F;
  p.template each<6>([&](float v, int) { mx = fmaxf(mx, v); });
  return mx;
}

// -> the place of the first token with that value, of the thread's ones; 0 for none.
template <typename T>
__device__ __noinline__ unsigned long long part_first(Part<T> p, float mx) {
  unsigned long long first = 0;
  p.template each<EACH>([&](float v, int i) {
    if (v == mx) first = max(first, place(v, i));
  });
  return first;
}

// Tokens per bin; -> the mass.
template <typename T>
__device__ __noinline__ float part_count(Part<T> p, Weights w, unsigned int* hist) {
  float sum = 0.f;
  unsigned int rest = 0;                   // what weighs less than 2^-46, often most of the row, would meet in one word
  p.template each<EACH>([&](float v, int) {
    const float y = w.depth(v);
    if (y >= BINS - 1.f) ++rest;
    else atomicAdd(&hist[__float_as_uint(__fadd_rd(y, 8388608.f)) - 0x4b000000u], 1u);               // its whole part
    sum += Weights::rough(y);
  });
  if (rest) atomicAdd(&hist[BINS - 1], rest);
  return sum;
}

// What a thread has found of the race: the mass of its tokens, the best rough score, that token, the next best; and of the exact ones the best.
struct Raced {
  float sum, bar, second;
  int bar_at;
  unsigned long long win;
};
struct RaceRules {
  float min_p, from, to;                   // bins in front of which tokens race, and in front of which they are collected
  float last_value;                        // the last token that is kept so far
  int last_index;
  __device__ __forceinline__ bool kept(float v, int i) const { return v > last_value || (v == last_value && i <= last_index); }
};
enum { FRONT, KEPT, EVERY };
// The race of the tokens in front of bin `from`, of those that are kept or of every one: a rough score of each. Tokens at the line of min_p are few: their exact scores are
// taken at once. Those in the bins behind, few as well, go to the list.
template <typename T, int WHO>
__device__ __noinline__ Raced part_race(Part<T> p, Weights ws, const float* noise, RaceRules rules, SampleShared* s) {
  constexpr int PER = Part<T>::PER, RUNS = RACE / PER;
  Raced out{0.f, -1.f, -1.f, 0, 0};
  const float floor_p = fmaxf(rules.min_p, 0.f), least = floor_p * (1.f - 1e-5f), sure = floor_p * (1.f + 1e-5f);
  const bool rest = rules.to == CUDART_INF_F;
  auto in = [&](float v, int i, float y) { return WHO == EVERY || (WHO == KEPT ? rules.kept(v, i) : y < rules.from); };
  auto rare = [&](int i) {
    const float v = p.value(p.x[i]);
    if (in(v, i, ws.depth(v))) {
      const float w = ws.exact(v);
      if (w >= rules.min_p) enter_race(out.win, w, noise[i], i);
    } else if (rules.kept(v, i)) {
      const int at = atomicAdd(&s->fill, 1);               // the window's count fits
      if (at < LIST) s->list[at] = place(v, i);
    }
  };
  // -> whether it is one of the few
  auto take = [&](float v, int i, float e) {
    const float y = ws.depth(v), r = Weights::rough(y);
    const bool now = in(v, i, y);
    out.sum += now ? r : 0.f;
    float inv;
    asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(inv) : "f"(e));
    const float sc = now && r >= sure ? r * inv : -1.f;
    if (sc > out.bar) out.bar_at = i;
    out.second = fmaxf(out.second, fminf(sc, out.bar));
    out.bar = fmaxf(out.bar, sc);
    return now ? r >= least && r < sure : WHO == FRONT && (y < rules.to || rest);
  };
  p.singles([&](int i) {
    if (take(p.value(p.x[i]), i, noise[i])) rare(i);
  });
  const uint4* xv = p.vectors();
  const float* ev = noise + p.head;
  const bool even = (reinterpret_cast<uintptr_t>(ev) & 15) == 0;
  uint4 w[RUNS];                           // asked for a batch ahead, with their variates
  float4 e[RUNS][PER / 4];
  auto ask = [&](int v) {
#pragma unroll
    for (int u = 0; u < RUNS; ++u) {
      const int at = v + u * ST;
      if (at >= p.v1) continue;
      w[u] = __ldg(xv + at);
#pragma unroll
      for (int h = 0; h < PER / 4; ++h) {
        const float* from = ev + (long long)at * PER + 4 * h;
        e[u][h] = even ? __ldg(reinterpret_cast<const float4*>(from)) : make_float4(__ldg(from), __ldg(from + 1), __ldg(from + 2), __ldg(from + 3));
      }
    }
  };
  const int start = p.v0 + threadIdx.x;
  ask(start);
  for (int v = start; v < p.v1; v += RUNS * ST) {
    uint4 now[RUNS];
    float4 en[RUNS][PER / 4];
#pragma unroll
    for (int u = 0; u < RUNS; ++u) {
      now[u] = w[u];
#pragma unroll
      for (int h = 0; h < PER / 4; ++h) en[u][h] = e[u][h];
    }
    ask(v + RUNS * ST);
    unsigned few = 0;
#pragma unroll
    for (int u = 0; u < RUNS; ++u) {
      if (v + u * ST >= p.v1) break;
      const T* el = reinterpret_cast<const T*>(&now[u]);
      const float* ee = reinterpret_cast<const float*>(en[u]);
#pragma unroll
      for (int q = 0; q < PER; ++q)
        if (take(p.value(el[q]), p.head + (v + u * ST) * PER + q, ee[q])) few |= 1u << (u * PER + q);
    }
    while (few) {
      const int q = __ffs(few) - 1;
      few &= few - 1;
      rare(p.head + (v + q / PER * ST) * PER + q % PER);
    }
  }
  return out;
}

// A row belongs to a cluster of C CTAs: CTA r reads the r-th part of it, in every pass. Passes: the maximum; tokens per bin (and the whole mass); the race over
// the tokens in front of the few bins that a filter's line runs through, whose tokens the first CTA sorts to find out which of them race too. Where the sorted list
// holds all that can be kept, it races alone. The row is read again from the L2 in each pass (a row of 131072 fp32 logits is 512 KB). What does not fit the
// list (many equal logits) is searched bit by bit, and then races in a pass of its own.
template <typename T>
__global__ void __launch_bounds__(ST, 2) sample_kernel(const __grid_constant__ SampleArgs a, int C) {
  extern __shared__ __align__(16) uint8_t smem_raw[];
  SampleShared& s = *reinterpret_cast<SampleShared*>(smem_raw);
  const int rank = C > 1 ? (int)cluster_ctarank() : 0, b = blockIdx.x / C, tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, V = a.V;
  const T* x = static_cast<const T*>(a.logits) + b * a.ld;
  const float* noise = a.noise ? a.noise + b * a.ldn : nullptr;
  auto peer = [&](auto* p, int r) {        // the same thing in CTA r of the cluster
    if (C == 1) return p;
    uint64_t out;
    asm("mapa.u64 %0, %1, %2;" : "=l"(out) : "l"(reinterpret_cast<uint64_t>(p)), "r"(r));
    return reinterpret_cast<decltype(p)>(out);
  };
  auto meet = [&]() {
    if (C > 1) cluster_sync_all();
    else __syncthreads();
  };

  Part<T> part;
  part.x = x;
  part.V = V;
  part.head = min(V, (int)((16 - (reinterpret_cast<uintptr_t>(x) & 15)) % 16 / sizeof(T)));
  part.vecs = (V - part.head) / Part<T>::PER;
  part.v0 = (int)((long long)part.vecs * rank / C);
  part.v1 = (int)((long long)part.vecs * (rank + 1) / C);
  part.front = rank == 0;
  part.back = rank == C - 1;
  auto each = [&](auto&& f) { part.template each<EACH>(f); };
  // ---- sums and maxima over the row, the same in every thread of the cluster
  int turn = 0;
  auto gather = [&](double2 mine, auto&& join) {
    if (lane == 0) s.red[warp] = mine;
    __syncthreads();
    double2 all = s.red[0];
    for (int w = 1; w < SW; ++w) all = join(all, s.red[w]);
    if (C > 1) {
      if (tid < C) *peer(&s.mail[turn][rank], tid) = all;
      cluster_sync_all();
      all = s.mail[turn][0];
      for (int r = 1; r < C; ++r) all = join(all, s.mail[turn][r]);
      turn ^= 1;
    } else {
      __syncthreads();
    }
    return all;
  };
  auto total = [&](double u, double v) {
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) {
      u += __shfl_xor_sync(0xffffffffu, u, o);
      v += __shfl_xor_sync(0xffffffffu, v, o);
    }
    return gather(make_double2(u, v), [](double2 p, double2 q) { return make_double2(p.x + q.x, p.y + q.y); });
  };
  auto most = [&](unsigned long long v) {
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) v = max(v, __shfl_xor_sync(0xffffffffu, v, o));
    const double2 r = gather(make_double2(__longlong_as_double((long long)v), 0.0), [](double2 p, double2 q) {
      return (unsigned long long)__double_as_longlong(p.x) >= (unsigned long long)__double_as_longlong(q.x) ? p : q;
    });
    return (unsigned long long)__double_as_longlong(r.x);
  };

  // the sum of u and, in one number, that of n over the CTAs and the largest f
  auto race_total = [&](double u, int n, float f) {
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) {
      u += __shfl_xor_sync(0xffffffffu, u, o);
      f = fmaxf(f, __shfl_xor_sync(0xffffffffu, f, o));
    }
    return gather(make_double2(u, __hiloint2double(__float_as_int(f), warp == 0 ? n : 0)), [](double2 p, double2 q) {
      const float top = fmaxf(__int_as_float(__double2hiint(p.y)), __int_as_float(__double2hiint(q.y)));
      return make_double2(p.x + q.x, __hiloint2double(__float_as_int(top), __double2loint(p.y) + __double2loint(q.y)));
    });
  };
  auto race_top = [](double2 all) { return __int_as_float(__double2hiint(all.y)); };

  const int kr = a.top_k ? a.top_k[b] : a.top_k_all, k = kr > 0 && kr < V ? kr : V;
  const float asked = a.temperature ? a.temperature[b] : a.temperature_all, temp = fminf(asked, 1e30f), asked_p = a.top_p ? a.top_p[b] : a.top_p_all,
              asked_min = a.min_p ? a.min_p[b] : a.min_p_all;
  const float p = fmaxf(asked_p, 0.f), min_p = isnan(asked_min) ? CUDART_INF_F : asked_min;            // of a NaN: the first token, none in the race
  if (C > 1) cluster_sync_all();           // every CTA of the row has started
  const float mx = value_of(most(place(part_max<T>(part), 0)));
  if (mx == -CUDART_INF_F || !(asked > 0.f)) {
    const unsigned long long first = most(mx == -CUDART_INF_F ? 0 : part_first<T>(part, mx));
    if (rank == 0 && tid == 0) a.out[b] = index_of(first);             // -1 of 0
    return;
  }
  const Weights ws{mx, temp, fminf(BINS_PER / temp, 1e30f)};
  auto weight = [&](float v) { return ws.exact(v); };
  auto depth = [&](float v) { return ws.depth(v); };
  auto rough = [&](float y) { return Weights::rough(y); };
  unsigned long long win = 0;
  auto race = [&](float w, int i) { enter_race(win, w, noise[i], i); };
  // what is kept: cut and all before it in the order
  unsigned long long cut = 0;
  RaceRules rules{min_p, 0.f, 0.f, -CUDART_INF_F, V};
  auto keep_to = [&](unsigned long long c) {
    if (c == 0) return;
    rules.last_value = value_of(c);
    rules.last_index = index_of(c);
  };
  auto kept = [&](float v, int i) { return rules.kept(v, i); };

  // The exact score where a thread's best is within 10^-4 of the row's, more than the rough scores are off: of that token, or of all of the CTA's where a thread
  // has another one as near (few rows do).
  Raced found_by_me{0.f, -1.f, -1.f, 0, 0};
  float top = -1.f;                        // the best of the row's
  bool raced = false;
  auto settle = [&](auto&& in) {           // by all threads of a CTA
    win = max(win, found_by_me.win);
    const bool plain = top > 1e-30f && top < CUDART_INF_F; // else some may have left the range in which they are that good
    const float near = plain ? top * (1.f - 1e-4f) : top < 0.f ? 0.f : -2.f;
    const bool mine = found_by_me.bar >= near;
    if (__syncthreads_or(mine && (!plain || found_by_me.second >= near))) {
      each([&](float v, int i) {
        if (!in(v, i, depth(v))) return;
        const float w = weight(v);
        if (w >= min_p) race(w, i);
      });
    } else if (mine) {
      race(weight(part.value(x[found_by_me.bar_at])), found_by_me.bar_at);
    }
  };

  if (k < V || p < 1.f) {
    for (int i = tid; i < BINS; i += ST) s.hist[i] = 0;
    if (tid == 0) s.fill = 0;
    __syncthreads();
    const bool want_all = p < 1.f && k == V;
    const float sum = part_count<T>(part, ws, s.hist);
    double mass = 0.0;                                     // of what top-k keeps
    if (want_all) mass = total(sum, 0.0).x;
    else meet();
    // all of the row is counted
    // ---- each CTA adds a share of the bins up, for the row's first one: there 16 neighbouring bins per thread
    constexpr int OWN = BINS / ST;
    for (int i = BINS / 4 * rank / C + tid; i < BINS / 4 * (rank + 1) / C; i += ST) {
      uint4 h[8];
#pragma unroll
      for (int r = 0; r < 8; ++r)
        if (r < C) h[r] = reinterpret_cast<const uint4*>(peer(s.hist, r))[i];
      uint4 sum4 = h[0];
#pragma unroll
      for (int r = 1; r < 8; ++r)
        if (r < C) {
          sum4.x += h[r].x; sum4.y += h[r].y; sum4.z += h[r].z; sum4.w += h[r].w;
        }
      reinterpret_cast<uint4*>(peer(s.merged, 0))[i] = sum4;
    }
    meet();                                                // from here on the list may take the bins' place
    auto load_counts = [&](unsigned int (&cnt)[OWN]) {
#pragma unroll
      for (int j = 0; j < OWN / 4; ++j) {
        const uint4 v = reinterpret_cast<const uint4*>(s.merged)[tid * (OWN / 4) + j];
        cnt[4 * j] = v.x; cnt[4 * j + 1] = v.y; cnt[4 * j + 2] = v.z; cnt[4 * j + 3] = v.w;
      }
    };
    // sums before this thread: v over the first CTA's threads
    auto before_me = [&](double& u, double& v) {
      auto scan = [&](double a, int upto) {                // inclusive, over `upto` lanes
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
          const double b = __shfl_up_sync(0xffffffffu, a, o);
          if (o < upto && lane >= o) a += b;
        }
        return a;
      };
      const double iu = scan(u, 32), iv = scan(v, 32);
      __syncthreads();
      if (lane == 31) s.scan[warp] = make_double2(iu, iv);
      __syncthreads();
      const double2 all = lane < SW ? s.scan[lane] : make_double2(0.0, 0.0);
      const double wu = __shfl_sync(0xffffffffu, scan(all.x, SW), warp ? warp - 1 : 0), wv = __shfl_sync(0xffffffffu, scan(all.y, SW), warp ? warp - 1 : 0);
      u = iu - u + (warp ? wu : 0.0);
      v = iv - v + (warp ? wv : 0.0);
    };
    // Of tokens (exact) and mass (fp32, its error far below the windows' margins): what lies before this thread and what up to its end, which is where the next one
    // starts; and all of the mass and of sq.
    struct Span {
      unsigned before, upto;
      float front, back, all, sq;
    };
    auto spans = [&](unsigned n, float mass, float sq) {
      auto scan = [&](auto v) {
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
          const auto u = __shfl_up_sync(0xffffffffu, v, o);
          if (lane >= o) v += u;
        }
        return v;
      };
      const unsigned in = scan(n);
      const float im = scan(mass);
#pragma unroll
      for (int o = 16; o > 0; o >>= 1) sq += __shfl_xor_sync(0xffffffffu, sq, o);
      __syncthreads();
      if (lane == 31) s.scan[warp] = make_double2(__hiloint2double(__float_as_int(im), (int)in), sq);
      __syncthreads();
      const double2 all = lane < SW ? s.scan[lane] : make_double2(0.0, 0.0);
      const unsigned wn = scan((unsigned)__double2loint(all.x));
      const float wm = scan(__int_as_float(__double2hiint(all.x)));
      sq = (float)all.y;
#pragma unroll
      for (int o = 16; o > 0; o >>= 1) sq += __shfl_xor_sync(0xffffffffu, sq, o);
      const unsigned n0 = __shfl_sync(0xffffffffu, wn, warp ? warp - 1 : 0), n1 = __shfl_sync(0xffffffffu, wn, warp);
      const float m0 = __shfl_sync(0xffffffffu, wm, warp ? warp - 1 : 0), m1 = __shfl_sync(0xffffffffu, wm, warp);
      const unsigned bn = warp ? n0 : 0u;
      const float bm = warp ? m0 : 0.f;
      const unsigned pn = __shfl_up_sync(0xffffffffu, in, 1);
      const float pm = __shfl_up_sync(0xffffffffu, im, 1);
      return Span{lane ? bn + pn : bn, lane == 31 ? n1 : bn + in, lane ? bm + pm : bm, lane == 31 ? m1 : bm + im, __shfl_sync(0xffffffffu, wm, SW - 1), sq};
    };
    const int bin0 = tid * OWN;
    // The window (first CTA): where the number of tokens reaches `want`, or the mass may. A bin's tokens weigh between exp(-(bin + 1) / 256) and
    // exp(-bin / 256); those of bin `last`, of which not all may count, between nothing and that. `wide` takes the bounds; else the middle of the bin stands for
    // them (the largest token's weight is known), as shares of their sum where that is the whole. Places within a bin are as good as even, so a sum is off by
    // 1 / (256 sqrt 12) of sqrt(sum w^2), of bf16 logits, where a bin holds one or two values, of sqrt(sum (n w)^2): four times that to either side hold nearly always
    // and leave 10 to 500 tokens to sort; what the list then holds shows whether they did.
    auto window_of_count = [&](unsigned want) {
      unsigned int cnt[OWN], n = 0;
      load_counts(cnt);
#pragma unroll
      for (int j = 0; j < OWN; ++j) n += cnt[j];
      unsigned at = spans(n, 0.f, 0.f).before;
#pragma unroll
      for (int j = 0; j < OWN; ++j) {
        if (at < want && at + cnt[j] >= want) {
          s.b1 = s.b2 = bin0 + j;
          s.before = at;
          s.upto = at + cnt[j];
        }
        at += cnt[j];
      }
      __syncthreads();
    };
    auto window_of_mass = [&](double target, int last, bool wide) {
      unsigned int cnt[OWN];
      load_counts(cnt);
      constexpr float RATIO = 0.99610137f;                 // exp(-1 / 256)
      const float edge = expf(-bin0 / BINS_PER) * (wide ? 1.f : 0.99804878f);          // exp(-1 / 512)
      constexpr bool FINE = std::is_same<T, float>::value;
      const float shrink = wide ? RATIO : 1.f;
      const float largest = wide || tid ? 0.f : 1.f - edge;
      float w = edge, sum = largest, sq = FINE && largest > 0.f ? -edge * edge : 0.f;
      unsigned int n = 0;
#pragma unroll
      for (int j = 0; j < OWN; ++j) {
        if (bin0 + j <= last) {
          n += cnt[j];
          sum += cnt[j] * w;
          sq += cnt[j] * w * (FINE ? w : cnt[j] * w);
        }
        w *= RATIO;
      }
      if (tid == 0) {                                      // should rounding hide the line: more than a list holds
        s.b1 = s.b2 = last;
        s.before = 0;
        s.upto = 1LL << 40;
      }
      const Span at = spans(n, sum, sq);                   // (with a barrier)
      const float want = !wide && k == V ? p * at.all : (float)target;
      // 2e-5: more than the sums' and the weights' rounding
      const float gap = 2e-5f + (wide ? 0.f : fminf(4.f / (256.f * 3.4641f) * sqrtf(fmaxf(at.sq, 0.f)) / want, 0x1p-9f));
      const float up = want * (1.f - gap), down = want * (1.f + gap);
      const bool ends_here = bin0 <= last && bin0 + OWN > last;
      if ((at.front < up && at.back >= up) || (at.front * shrink < down && at.back * shrink >= down) || ends_here) {
        w = edge;
        float high = at.front;
        unsigned count = at.before;
#pragma unroll
        for (int j = 0; j < OWN; ++j) {
          const int bin = bin0 + j;
          if (bin > last) continue;
          const float next = j == OWN - 1 || bin == last ? fmaxf(high, at.back) : high + cnt[j] * w + (j == 0 ? largest : 0.f);
          if (high < up && (next >= up || bin == last)) {
            s.b1 = bin;
            s.before = count;
          }
          if (high * shrink < down && (next * shrink >= down || bin == last)) {
            s.b2 = bin;
            s.upto = count + cnt[j];
          }
          count += cnt[j];
          high = next;
          w *= RATIO;
        }
      }
      __syncthreads();
    };
    // first CTA, thread 0: what comes next, to the others
    auto tell = [&](int mode) {
      for (int r = 0; r < C; ++r) {
        SampleShared* d = peer(&s, r);
        d->b1 = s.b1;
        d->b2 = s.b2;
        d->mode = mode;
      }
    };
    // The window's tokens (those that are kept so far) to the list; the mass of the ones before it, which race here if this filter is the last one.
    auto before_window = [&](float, int, float y) { return y < s.b1; };
    auto collect = [&](bool last) {
      rules.from = (float)s.b1;
      rules.to = s.b2 == BINS - 1 ? CUDART_INF_F : (float)(s.b2 + 1);
      float sum = 0.f;
      if (last) {
        found_by_me = part_race<T, FRONT>(part, ws, noise, rules, &s);
        sum = found_by_me.sum;
      } else {
        each([&](float v, int i) {
          const float y = depth(v);
          if (y < rules.from) {
            sum += rough(y);
          } else if ((y < rules.to || rules.to == CUDART_INF_F) && kept(v, i)) {
            const int at = atomicAdd(&s.fill, 1);          // the window's count fits
            if (at < LIST) s.list[at] = place(v, i);
          }
        });
      }
      __syncthreads();
      const int fill = min(s.fill, LIST);
      const double2 all = race_total(sum, fill, found_by_me.bar);
      top = race_top(all);
      if (C > 1) {                                         // behind those of the CTAs before, in the first one
        int at = 0;
        for (int r = 0; r < rank; ++r) at += __double2loint(s.mail[turn ^ 1][r].y);
        unsigned long long* to0 = peer(s.swap, 0);
        for (int i = tid; i < fill && at + i < LIST; i += ST) to0[at + i] = s.list[i];
        cluster_sync_all();
      } else {
        for (int i = tid; i < fill; i += ST) s.swap[i] = s.list[i];
        __syncthreads();
      }
      return make_double2(all.x, min(__double2loint(all.y), LIST));
    };
    // first CTA: all lists to one, in order: a bitonic network, E neighbouring entries per thread in registers, exchanges between warps through shared memory
    auto order = [&](auto per_thread, int m) {
      constexpr int E = per_thread.value;
      unsigned long long e[E];
#pragma unroll
      for (int j = 0; j < E; ++j) e[j] = s.swap[tid * E + j];
      unsigned long long* buf = s.list;
      for (int size = 2; size <= m; size <<= 1)
        for (int step = size >> 1; step > 0; step >>= 1) {
          if (step < E) {
#pragma unroll
            for (int st = 1; st < E; st <<= 1) {
              if (st != step) continue;
#pragma unroll
              for (int j = 0; j < E; ++j)
                if (!(j & st)) {
                  const bool fall = ((tid * E + j) & size) == 0;
                  const unsigned long long u = e[j], v = e[j | st];
                  if ((u < v) == fall) {
                    e[j] = v;
                    e[j | st] = u;
                  }
                }
            }
          } else {
            if (step >= 32 * E) {
#pragma unroll
              for (int j = 0; j < E; ++j) buf[j * ST + tid] = e[j];
              __syncthreads();
            }
#pragma unroll
            for (int j = 0; j < E; ++j) {
              const int i = tid * E + j;
              const unsigned long long o = step >= 32 * E ? buf[j * ST + (tid ^ (step / E))] : __shfl_xor_sync(0xffffffffu, e[j], step / E);
              const bool larger = ((i & step) == 0) == ((i & size) == 0);
              e[j] = larger ? max(e[j], o) : min(e[j], o);
            }
            if (step >= 32 * E) buf = buf == s.swap ? s.list : s.swap;       // the next exchange's place: nobody reads it any more behind its barrier
          }
        }
      __syncthreads();
#pragma unroll
      for (int j = 0; j < E; ++j) s.list[tid * E + j] = e[j];
      __syncthreads();
    };
    auto sort = [&](int n) {
      int m = 2;
      while (m < n) m <<= 1;
      const int room = max(m, ST);
      for (int i = n + tid; i < room; i += ST) s.swap[i] = 0;
      __syncthreads();
      if (m <= ST) order(std::integral_constant<int, 1>{}, m);
      else if (m <= 2 * ST) order(std::integral_constant<int, 2>{}, m);
      else if (m <= 4 * ST) order(std::integral_constant<int, 4>{}, m);
      else order(std::integral_constant<int, 8>{}, m);
    };
    // first CTA: the mass of the first n of the list, and how many of them it takes until base + mass >= want (n, if that is not reached) in s.pos
    auto prefix = [&](int n, double base, double want) {
      const int each_n = (n + ST - 1) / ST, i0 = min(n, tid * each_n), i1 = min(n, i0 + each_n);
      double at = 0.0, none = 0.0;
      for (int i = i0; i < i1; ++i) at += weight(value_of(s.list[i]));
      if (tid == 0) s.pos = n;
      before_me(at, none);
      double run = base + at;
      for (int i = i0; i < i1; ++i) {
        const double next = run + weight(value_of(s.list[i]));
        if (run < want && next >= want) s.pos = i + 1;
        run = next;
      }
      if (i1 == n && i1 > i0) s.mass = run;
      __syncthreads();
      return s.mass;
    };
    auto race_list = [&](int n) {
      for (int i = tid; i < n; i += ST) {
        const float w = weight(value_of(s.list[i]));
        if (w >= min_p) race(w, index_of(s.list[i]));
      }
    };
    // bit by bit: the last token that is kept when `reach(least)` of them have to be: the largest place with reach(place) >= want
    auto search = [&](double want, auto&& count) {
      unsigned long long c = 0;
      const int low_bits = 32 - __clz(V - 1 | 1);
      for (int bit = 63; bit >= 0; --bit) {
        if (bit < 32 && bit >= low_bits) {                 // ~index: ones
          c |= 1ull << bit;
          continue;
        }
        const unsigned long long y = c | 1ull << bit;
        double n = 0;
        each([&](float v, int i) {
          const unsigned long long at = place(v, i);
          if (at >= y && at >= cut) n += count(v);
        });
        if (total(n, 0.0).x >= want) c = y;
      }
      return c;
    };

    if (k < V) {
      if (rank == 0) {
        window_of_count(k);
        const bool all = s.upto <= LIST;
        __syncthreads();
        if (tid == 0) {
          if (all) s.b1 = 0;
          tell(all ? SORT_ALL : (s.upto - s.before <= LIST ? SORT_WINDOW : SEARCH));
        }
      }
      meet();
      const int mode = s.mode, last = s.b2;
      if (mode == SEARCH) {
        cut = search(k, [](float) { return 1.0; });
        if (p < 1.f) {
          double m = 0;
          each([&](float v, int i) { m += place(v, i) >= cut ? (double)rough(depth(v)) : 0.0; });
          mass = total(m, 0.0).x;
        }
      } else {
        const double2 got = collect(mode == SORT_WINDOW && p >= 1.f);
        const double above = got.x;
        if (mode == SORT_ALL) {                            // the list holds all that can be kept
          if (rank != 0) return;
          sort((int)got.y);
          int n = min((int)got.y, k);
          if (p < 1.f) {
            const double m = prefix(n, 0.0, -1.0);
            prefix(n, 0.0, fmax((double)p * m, 1e-30));
            n = s.pos;
          }
          race_list(n);
#pragma unroll
          for (int o = 16; o > 0; o >>= 1) win = max(win, __shfl_xor_sync(0xffffffffu, win, o));
          if (lane == 0) s.swap[warp] = win;
          __syncthreads();
          if (tid == 0) {
            for (int w = 0; w < SW; ++w) win = max(win, s.swap[w]);
            a.out[b] = index_of(win ? win : s.list[0]);    // the first largest where none of them raced
          }
          return;
        }
        if (rank == 0) {
          sort((int)got.y);
          const int n = (int)(k - s.before);
          const double m = p < 1.f ? prefix(n, above, 1e300) : 0.0;
          if (p >= 1.f) race_list(n);
          if (tid < C) {
            SampleShared* d = peer(&s, tid);
            d->cut = s.list[n - 1];
            d->mass = m;
          }
        }
        meet();
        cut = s.cut;
        mass = s.mass;
        if (p >= 1.f) {
          settle(before_window);
          raced = true;
        }
        __syncthreads();
        if (tid == 0) s.fill = 0;          // for the next window; read and counted on behind the barriers before that
      }
      if (rank == 0 && tid == 0) s.b2 = last;
    }
    if (p < 1.f) {
      const double want = fmax((double)p * mass, 1e-30);   // a share of nothing still takes the first token
      int last = BINS - 1;
      if (k < V) {
        __syncthreads();
        last = s.b2;
        __syncthreads();
      }
      bool found = false;
      // bf16 logits of one bin are one or two numbers: its middle says too little of them, but as shares
      for (int wide = std::is_same<T, float>::value || k == V ? 0 : 1; wide < 2 && !found; ++wide) {
        if (rank == 0) {
          window_of_mass(want, last, wide);
          if (tid == 0) tell(s.upto - s.before <= LIST ? SORT_WINDOW : SEARCH);
        }
        meet();
        if (s.mode == SEARCH) break;
        keep_to(cut);
        const double2 got = collect(true);
        if (rank == 0) {
          const int n = (int)got.y;
          sort(n);
          bool holds = n > 0;
          if (n > 0) {
            const double m = prefix(n, got.x, want);
            holds = got.x < want && m >= want;
          }
          if (tid < C) peer(&s, tid)->cut = holds ? s.list[s.pos - 1] : 0;
          if (holds) race_list(s.pos);
          __syncthreads();
        }
        if (tid == 0) s.fill = 0;
        meet();
        if (s.cut) {
          found = raced = true;
          settle(before_window);
        }
      }
      if (!found) cut = max(cut, search(want, [&](float v) { return (double)rough(depth(v)); }));
    }
  }
  if (!raced) {
    keep_to(cut);
    auto all = [&](float v, int i, float) { return kept(v, i); };
    found_by_me = cut ? part_race<T, KEPT>(part, ws, noise, rules, &s) : part_race<T, EVERY>(part, ws, noise, rules, &s);
    top = race_top(race_total(0.0, 0, found_by_me.bar));
    settle(all);
  }
  win = most(win);
  if (win == 0) win = most(part_first<T>(part, mx));       // nothing raced: the first largest (the same turn in every thread of the row)
  if (rank == 0 && tid == 0) a.out[b] = index_of(win);
}

template <typename T>
int launch_sample(const SampleArgs& a, int B, cudaStream_t st) {
  // CTAs per row: while each has an SM of its own and 8192 logits, twice as many. Measured, us on 1, 2, 4, 8 (top-p, but for the 8192): 1 row of 131072: 65, 49, 38, 32;
  // 40: 71, 53, 54, 72; 96: 74, 76, 89, 127; 120: 91, 80, 109, 163; 64 of 32000 bf16: 33, 32, 37, 66; 150 of 50000: 58, 73, 94, 153; 32 of 8192: 17, 19, 19, 23. Where two CTAs
  // would share SMs the sizes above differ in sign, and rows stay with one.
  int C = 1;
  while (C < 8 && a.V > 8192LL * C && (long long)B * C * 2 <= 148) C *= 2;
  ELFA_CUDA(allow_shared<sample_kernel<T>>((int)sizeof(SampleShared)));
  cudaLaunchConfig_t cfg{};
  cfg.gridDim = dim3((unsigned)B * C);
  cfg.blockDim = dim3(ST);
  cfg.dynamicSmemBytes = sizeof(SampleShared);
  cfg.stream = st;
  cudaLaunchAttribute at[1];
  at[0].id = cudaLaunchAttributeClusterDimension;
  at[0].val.clusterDim.x = C;
  at[0].val.clusterDim.y = at[0].val.clusterDim.z = 1;
  cfg.attrs = at;
  cfg.numAttrs = 1;
  ELFA_CUDA(cudaLaunchKernelEx(&cfg, sample_kernel<T>, a, C));
  ELFA_CUDA(cudaGetLastError());
  ::elfa::count_launches(1);
  return ELFA_OK;
}

}  // namespace
}  // namespace elfa

using namespace elfa;

// logits: [B] rows of V, ld apart (type 0 bf16, 1 fp32); noise: [B] rows of V fp32, ldn apart; the four settings per row, or where
// their pointer is null one for all; out: [B]. noise may be null where the temperature is 0 for all rows.
ELFA_API int elfa_sample(const void* logits, int type, long long ld, const float* noise, long long ldn, const float* temperature, const int* top_k,
                         const float* top_p, const float* min_p, float temperature_all, int top_k_all, float top_p_all, float min_p_all, long long* out,
                         int B, int V, void* stream) {
  ELFA_REQUIRE(logits && out && (noise || (!temperature && !(temperature_all > 0.f))), "sample: null pointer");
  ELFA_REQUIRE(B > 0 && B <= (1 << 27) && V > 0 && V < 0x7fffffff - 65536 && (type == 0 || type == 1), "sample: bad sizes");
  const SampleArgs a{logits, noise, ld, ldn, temperature, top_k, top_p, min_p, temperature_all, top_p_all, min_p_all, top_k_all, out, V};
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  return type == 0 ? launch_sample<__nv_bfloat16>(a, B, st) : launch_sample<float>(a, B, st);
}
