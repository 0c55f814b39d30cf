// One token per row of logits: temperature, top-k, top-p, min-p, drawn with given exponential variates.
//
// w_i = exp((x_i - max x) / T). In the order of falling x (equal ones by index) every filter keeps a prefix: the first k; of those the
// shortest one with mass >= p of theirs; of those the ones with w_i >= min_p. What is kept races: the token with the largest w_i / e_i wins, which
// for independent exponential variates e_i is token i with probability w_i / sum w (the lowest index where two are equal). T <= 0 takes the first largest logit.
// A NaN counts as -inf; a row without any number above -inf gives -1.
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
    unsigned long long list[LIST];         // places, in the row's first CTA
  };
  double2 mail[2][8];                      // what the CTAs of the row send each other, by turns
  double2 red[SW];
  double scan[3][SW];
  unsigned long long cut;                  // the last token that is kept
  double mass, target;
  long long before, upto;                  // tokens before and up to the end of the window
  int b1, b2;                              // the window: bins that a filter's line may run through
  int fill, pos, mode;                     // entries of the list; kept ones of them; what comes next
};
enum { SORT_ALL, SORT_WINDOW, SEARCH };

// A row belongs to a cluster of C CTAs: CTA r reads the r-th part of it, in every pass. Passes: the maximum; tokens per bin (and the whole mass); the tokens of
// the few bins that the line runs through, which the first CTA sorts; and the race over what is kept, or over the sorted list alone where it holds all of it.
// The row is read again from the L2 in each (a row of 131072 fp32 logits is 512 KB). What does not fit the list (many equal logits) is searched bit by bit.
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

  // ---- every element of this CTA's part: single ones up to a 16-byte boundary, then vectors
  constexpr int PER = 16 / sizeof(T);
  const int head = min(V, (int)((16 - (reinterpret_cast<uintptr_t>(x) & 15)) % 16 / sizeof(T)));
  const int vecs = (V - head) / PER, v0 = (int)((long long)vecs * rank / C), v1 = (int)((long long)vecs * (rank + 1) / C);
  auto each = [&](auto&& f) {
    auto value = [](T v) {
      float y;
      if constexpr (std::is_same<T, float>::value) y = v;
      else y = __bfloat162float(v);
      return y != y ? -CUDART_INF_F : y;
    };
    if (rank == 0 && tid < head) f(value(x[tid]), tid);
    const int tail = head + vecs * PER;
    if (rank == C - 1 && tail + tid < V) f(value(x[tail + tid]), tail + tid);
    const uint4* xv = reinterpret_cast<const uint4*>(x + head);
    constexpr int U = 4;
    for (int v = v0 + tid; v < v1; v += U * ST) {
      uint4 w[U];
#pragma unroll
      for (int u = 0; u < U; ++u)
        if (v + u * ST < v1) w[u] = __ldg(xv + v + u * ST);
#pragma unroll
      for (int u = 0; u < U; ++u) {
        if (v + u * ST >= v1) break;
        const T* e = reinterpret_cast<const T*>(&w[u]);
#pragma unroll
        for (int k = 0; k < PER; ++k) f(value(e[k]), head + (v + u * ST) * PER + k);
      }
    }
  };
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

  const int kr = a.top_k ? a.top_k[b] : a.top_k_all, k = kr > 0 && kr < V ? kr : V;
  const float temp = a.temperature ? a.temperature[b] : a.temperature_all, p = a.top_p ? a.top_p[b] : a.top_p_all,
              min_p = a.min_p ? a.min_p[b] : a.min_p_all;
  if (C > 1) cluster_sync_all();           // every CTA of the row has started
  unsigned long long best = 0;
  each([&](float v, int i) { best = max(best, place(v, i)); });
  best = most(best);
  const float mx = value_of(best);
  if (mx == -CUDART_INF_F || !(temp > 0.f)) {
    if (rank == 0 && tid == 0) a.out[b] = mx == -CUDART_INF_F ? -1 : index_of(best);
    return;
  }
  auto weight = [&](float v) { return v == mx ? 1.f : expf((v - mx) / temp); };
  const float fast = 1.4426950408889634f / temp;
  auto rough = [&](float v) { return v == mx ? 1.f : fast_exp2((v - mx) * fast); };       // for the sums: 2^-22 of each, of what weighs little a bit more
  unsigned long long win = (uint32_t)best;                                                // score 0 of the first largest, should no other compare
  auto race = [&](float w, int i) {
    const float sc = w / noise[i];
    if (sc >= 0.f) win = max(win, (unsigned long long)__float_as_uint(sc) << 32 | (uint32_t)~i);
  };
  unsigned long long cut = 0;

  if (k < V || p < 1.f) {
    const float per = BINS_PER / temp;
    auto bin_of = [&](float v) { return v == mx ? 0 : (int)fminf((mx - v) * per, BINS - 1.f); };     // never falls as v falls, whatever it rounds to
    for (int i = tid; i < BINS; i += ST) s.hist[i] = 0;
    if (tid == 0) s.fill = 0;
    __syncthreads();
    const bool want_all = p < 1.f && k == V;
    float sum = 0.f;
    unsigned int rest = 0;                                 // what weighs less than 2^-46, often most of the row, would meet in one word
    each([&](float v, int) {
      const int bin = bin_of(v);
      if (bin == BINS - 1) ++rest;
      else atomicAdd(&s.hist[bin], 1u);
      if (want_all) sum += rough(v);
    });
    if (rest) atomicAdd(&s.hist[BINS - 1], rest);
    double mass = want_all ? total(sum, 0.0).x : 0.0;      // of what top-k keeps
    meet();                                                // all of the row is counted
    // ---- the row's first CTA adds the bins up: 16 neighbouring ones per thread
    constexpr int OWN = BINS / ST;
    unsigned int cnt[OWN];
    if (rank == 0) {
#pragma unroll
      for (int j = 0; j < OWN; ++j) cnt[j] = 0;
      for (int r = 0; r < C; ++r) {
        const uint4* h = reinterpret_cast<const uint4*>(peer(s.hist, r)) + tid * (OWN / 4);
#pragma unroll
        for (int j = 0; j < OWN / 4; ++j) {
          const uint4 v = h[j];
          cnt[4 * j] += v.x; cnt[4 * j + 1] += v.y; cnt[4 * j + 2] += v.z; cnt[4 * j + 3] += v.w;
        }
      }
      __syncthreads();                                     // the list may take the bins' place
    }
    // sums before this thread: v over the first CTA's threads
    auto before_me = [&](double (&v)[3]) {
      double incl[3] = {v[0], v[1], v[2]};
#pragma unroll
      for (int o = 1; o < 32; o <<= 1)
#pragma unroll
        for (int q = 0; q < 3; ++q) {
          const double u = __shfl_up_sync(0xffffffffu, incl[q], o);
          if (lane >= o) incl[q] += u;
        }
      __syncthreads();
      if (lane == 31)
#pragma unroll
        for (int q = 0; q < 3; ++q) s.scan[q][warp] = incl[q];
      __syncthreads();
#pragma unroll
      for (int q = 0; q < 3; ++q) {
        v[q] = incl[q] - v[q];
        for (int w = 0; w < warp; ++w) v[q] += s.scan[q][w];
      }
    };
    const int bin0 = tid * OWN;
    // The window (first CTA): where the number of tokens reaches `want`, or bounds of the mass do. A bin's tokens weigh between exp(-(bin + 1) / 256) and
    // exp(-bin / 256); those of bin `last`, of which not all may count, between nothing and that.
    auto window_of_count = [&](double want) {
      double at[3] = {0, 0, 0};
#pragma unroll
      for (int j = 0; j < OWN; ++j) at[0] += cnt[j];
      before_me(at);
#pragma unroll
      for (int j = 0; j < OWN; ++j) {
        if (at[0] < want && at[0] + cnt[j] >= want) {
          s.b1 = s.b2 = bin0 + j;
          s.before = (long long)at[0];
          s.upto = (long long)(at[0] + cnt[j]);
        }
        at[0] += cnt[j];
      }
      __syncthreads();
    };
    auto window_of_mass = [&](double want, int last) {
      auto high = [&](int j) { return cnt[j] * (double)expf(-(bin0 + j) / BINS_PER); };
      auto low = [&](int j) { return bin0 + j < last ? cnt[j] * (double)expf(-(bin0 + j + 1) / BINS_PER) : 0.0; };
      double at[3] = {0, 0, 0};
#pragma unroll
      for (int j = 0; j < OWN; ++j) {
        if (bin0 + j > last) continue;
        at[0] += cnt[j];
        at[1] += high(j);
        at[2] += low(j);
      }
      before_me(at);
      const double up = want * (1 - 1e-5), down = want * (1 + 1e-5);         // more than the sums' and the weights' rounding
#pragma unroll
      for (int j = 0; j < OWN; ++j) {
        const int bin = bin0 + j;
        if (bin > last) continue;
        if (at[1] < up && (at[1] + high(j) >= up || bin == last)) {
          s.b1 = bin;
          s.before = (long long)at[0];
        }
        if (at[2] < down && (at[2] + low(j) >= down || bin == last)) {
          s.b2 = bin;
          s.upto = (long long)(at[0] + cnt[j]);
        }
        at[0] += cnt[j];
        at[1] += high(j);
        at[2] += low(j);
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
    // the window's tokens (those not behind `least`) to the list; the mass of the ones before the window
    auto collect = [&](unsigned long long least) {
      const int b1 = s.b1, b2 = s.b2;
      int* fill = peer(&s.fill, 0);
      unsigned long long* list = peer(s.list, 0);
      float sum = 0.f;
      each([&](float v, int i) {
        const int bin = bin_of(v);
        if (bin < b1) sum += rough(v);
        else if (bin <= b2 && place(v, i) >= least) {
          const int at = atomicAdd(fill, 1);
          if (at < LIST) list[at] = place(v, i);
        }
      });
      return total(sum, 0.0).x;
    };
    // first CTA: the list in order
    auto sort = [&]() {
      const int n = min(s.fill, LIST);
      int m = 2;
      while (m < n) m <<= 1;
      for (int i = n + tid; i < m; i += ST) s.list[i] = 0;
      for (int size = 2; size <= m; size <<= 1)
        for (int step = size >> 1; step > 0; step >>= 1) {
          __syncthreads();
          for (int i = tid; i < m / 2; i += ST) {
            const int l = 2 * i - (i & (step - 1)), h = l + step;
            const unsigned long long u = s.list[l], v = s.list[h];
            if ((u < v) == ((l & size) == 0)) {            // falling
              s.list[l] = v;
              s.list[h] = u;
            }
          }
        }
      __syncthreads();
      return n;
    };
    // first CTA: the mass of the first n of the list, and how many of them it takes until base + mass >= want (n, if that is not reached) in s.pos
    auto prefix = [&](int n, double base, double want) {
      const int each_n = (n + ST - 1) / ST, i0 = min(n, tid * each_n), i1 = min(n, i0 + each_n);
      double at[3] = {0, 0, 0};
      for (int i = i0; i < i1; ++i) at[0] += weight(value_of(s.list[i]));
      if (tid == 0) s.pos = n;
      before_me(at);
      double run = base + at[0];
      for (int i = i0; i < i1; ++i) {
        const double next = run + weight(value_of(s.list[i]));
        if (run < want && next >= want) s.pos = i + 1;
        run = next;
      }
      if (i1 == n && i1 > i0) s.mass = run;
      __syncthreads();
      return s.mass;
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
          each([&](float v, int i) { m += place(v, i) >= cut ? (double)rough(v) : 0.0; });
          mass = total(m, 0.0).x;
        }
      } else {
        const double above = collect(0);
        if (mode == SORT_ALL) {                            // the list holds all that can be kept
          if (rank != 0) return;
          int n = min(sort(), k);
          if (p < 1.f) {
            const double m = prefix(n, 0.0, -1.0);
            prefix(n, 0.0, fmax((double)p * m, 1e-30));
            n = s.pos;
          }
          for (int i = tid; i < n; i += ST) {
            const float w = weight(value_of(s.list[i]));
            if (w >= min_p) race(w, index_of(s.list[i]));
          }
#pragma unroll
          for (int o = 16; o > 0; o >>= 1) win = max(win, __shfl_xor_sync(0xffffffffu, win, o));
          __syncthreads();
          if (lane == 0) s.list[warp] = win;
          __syncthreads();
          if (tid == 0) {
            for (int w = 0; w < SW; ++w) win = max(win, s.list[w]);
            a.out[b] = index_of(win);
          }
          return;
        }
        if (rank == 0) {
          sort();
          const int n = (int)(k - s.before);
          const double m = p < 1.f ? prefix(n, above, 1e300) : 0.0;
          if (tid < C) {
            SampleShared* d = peer(&s, tid);
            d->cut = s.list[n - 1];
            d->mass = m;
          }
          __syncthreads();
          if (tid == 0) s.fill = 0;
        }
        meet();
        cut = s.cut;
        mass = s.mass;
      }
      if (rank == 0 && tid == 0) s.b2 = last;
    }
    if (p < 1.f) {
      const double want = fmax((double)p * mass, 1e-30);   // a share of nothing still takes the first token
      if (rank == 0) {
        __syncthreads();
        const int last = k < V ? s.b2 : BINS - 1;
        __syncthreads();
        window_of_mass(want, last);
        if (tid == 0) tell(s.upto - s.before <= LIST ? SORT_WINDOW : SEARCH);
      }
      meet();
      const double above = s.mode == SEARCH ? 0.0 : collect(cut);
      int found = 0;
      if (s.mode != SEARCH) {
        if (rank == 0) {
          const int n = sort();
          if (n > 0) prefix(n, above, want);
          if (tid < C) {
            SampleShared* d = peer(&s, tid);
            d->cut = n > 0 ? s.list[s.pos - 1] : 0;
          }
        }
        meet();
        if (s.cut) {
          cut = s.cut;
          found = 1;
        }
      }
      if (!found) cut = max(cut, search(want, [&](float v) { return (double)rough(v); }));
    }
  }
  each([&](float v, int i) {
    if (place(v, i) < cut) return;
    const float w = weight(v);
    if (w >= min_p) race(w, i);
  });
  win = most(win);
  if (rank == 0 && tid == 0) a.out[b] = index_of(win);
}

template <typename T>
int launch_sample(const SampleArgs& a, int B, cudaStream_t st) {
  // CTAs per row: a part of 16384 logits or less each, and while the rows leave SMs idle, down to 4096
  int C = 1;
  while (C < 8 && ((long long)a.V > 16384LL * C || (B * C * 2 <= 148 && (long long)a.V > 4096LL * C))) C *= 2;
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
