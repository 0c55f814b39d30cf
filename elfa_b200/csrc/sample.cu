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

constexpr int ST = 1024;

template <typename T>
__global__ void __launch_bounds__(ST) sample_kernel(const __grid_constant__ SampleArgs a) {
  __shared__ double redd[32];
  __shared__ unsigned long long redu[32];
  const int b = blockIdx.x, warp = threadIdx.x >> 5, lane = threadIdx.x & 31, V = a.V;
  const T* x = static_cast<const T*>(a.logits) + b * a.ld;
  const float* noise = a.noise ? a.noise + b * a.ldn : nullptr;
  auto load = [&](int i) {
    float v;
    if constexpr (std::is_same<T, float>::value) v = x[i];
    else v = __bfloat162float(x[i]);
    return v != v ? -CUDART_INF_F : v;
  };
  auto sum = [&](double v) {
    for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
    __syncthreads();
    if (lane == 0) redd[warp] = v;
    __syncthreads();
    v = redd[lane];
    for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
    return v;
  };
  auto most = [&](unsigned long long v) {
    for (int o = 16; o > 0; o >>= 1) v = max(v, __shfl_xor_sync(0xffffffffu, v, o));
    __syncthreads();
    if (lane == 0) redu[warp] = v;
    __syncthreads();
    v = redu[lane];
    for (int o = 16; o > 0; o >>= 1) v = max(v, __shfl_xor_sync(0xffffffffu, v, o));
    return v;
  };
  // (key, index) as one number whose largest is the largest key at its lowest index
  unsigned long long best = 0;
  for (int i = threadIdx.x; i < V; i += ST) best = max(best, (unsigned long long)order_key(load(i)) << 32 | (uint32_t)(~i));
  best = most(best);
  const int arg = (int)~(uint32_t)best;
  const float mx = load(arg), temp = a.temperature ? a.temperature[b] : a.temperature_all;
  if (mx == -CUDART_INF_F || !(temp > 0.f)) {
    if (threadIdx.x == 0) a.out[b] = mx == -CUDART_INF_F ? -1 : arg;
    return;
  }
  auto weight = [&](float v) { return v == mx ? 1.f : expf((v - mx) / temp); };
  const int kr = a.top_k ? a.top_k[b] : a.top_k_all, k = kr > 0 && kr < V ? kr : V;
  const float p = a.top_p ? a.top_p[b] : a.top_p_all, min_p = a.min_p ? a.min_p[b] : a.min_p_all;
  // kept: key > cut, and of key == cut those with index < bound
  uint32_t cut = 0;
  int bound = V;
  double ties = -1.0;                                    // how many of key == cut (negative: all)
  if (k < V) {
    for (int bit = 31; bit >= 0; --bit) {
      const uint32_t c = cut | 1u << bit;
      double n = 0;
      for (int i = threadIdx.x; i < V; i += ST) n += order_key(load(i)) >= c;
      if (sum(n) >= k) cut = c;
    }
    double n = 0;
    for (int i = threadIdx.x; i < V; i += ST) n += order_key(load(i)) > cut;
    ties = k - sum(n);
  }
  if (p < 1.f) {
    double above = 0, at = 0, wt = 0;
    for (int i = threadIdx.x; i < V; i += ST) {
      const float v = load(i);
      const uint32_t key = order_key(v);
      if (key > cut) above += weight(v);
      if (key == cut) {
        at += 1;
        wt = weight(v);
      }
    }
    above = sum(above);
    at = sum(at);
    wt = at > 0 ? __longlong_as_double(most(__double_as_longlong(wt))) : 0;
    const double have = ties < 0 ? at : ties, target = (double)p * (above + have * wt);
    if (above >= target && above > 0) {                  // the nucleus ends above the cut
      uint32_t c2 = 0;
      for (int bit = 31; bit >= 0; --bit) {
        const uint32_t c = c2 | 1u << bit;
        double s = 0;
        if (c > cut)
          for (int i = threadIdx.x; i < V; i += ST) {
            const float v = load(i);
            if (order_key(v) >= c) s += weight(v);
          }
        if (c <= cut || sum(s) >= target) c2 = c;
      }
      // c2 is the largest bound that still holds the mass (it may be no key itself); a target of 0 wants the first token
      if (c2 > (uint32_t)(best >> 32)) c2 = (uint32_t)(best >> 32);
      cut = c2;
      above = 0; at = 0; wt = 0;
      for (int i = threadIdx.x; i < V; i += ST) {
        const float v = load(i);
        const uint32_t key = order_key(v);
        if (key > cut) above += weight(v);
        if (key == cut) {
          at += 1;
          wt = weight(v);
        }
      }
      above = sum(above);
      at = sum(at);
      wt = at > 0 ? __longlong_as_double(most(__double_as_longlong(wt))) : 0;
      ties = at;
    } else {
      ties = have;
    }
    if (wt > 0) ties = fmin(ties, fmax(1.0, ceil((target - above) / wt)));
  }
  if (ties >= 0) {                                       // the index before which the first `ties` of the equal ones lie
    int lo = 0, hi = V;                                  // count(equal, index < hi) >= ties
    while (lo < hi) {
      const int mid = (lo + hi) >> 1;
      double n = 0;
      for (int i = threadIdx.x; i < mid; i += ST) n += order_key(load(i)) == cut;
      if (sum(n) >= ties) hi = mid;
      else lo = mid + 1;
    }
    bound = lo;
  }
  unsigned long long win = (uint32_t)~arg;               // the first largest logit, should nothing else compare
  for (int i = threadIdx.x; i < V; i += ST) {
    const float v = load(i);
    const uint32_t key = order_key(v);
    const float w = weight(v);
    if (key < cut || (key == cut && i >= bound) || w < min_p) continue;
    const float s = w / noise[i];
    if (s >= 0.f) win = max(win, (unsigned long long)__float_as_uint(s) << 32 | (uint32_t)(~i));
  }
  win = most(win);
  if (threadIdx.x == 0) a.out[b] = (int)~(uint32_t)win;
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
  ELFA_REQUIRE(B > 0 && V > 0 && V < 0x7fffffff - 4096 && (type == 0 || type == 1), "sample: bad sizes");
  const SampleArgs a{logits, noise, ld, ldn, temperature, top_k, top_p, min_p, temperature_all, top_p_all, min_p_all, top_k_all, out, V};
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  if (type == 0) sample_kernel<__nv_bfloat16><<<B, ST, 0, st>>>(a);
  else sample_kernel<float><<<B, ST, 0, st>>>(a);
  ELFA_CUDA(cudaGetLastError());
  ::elfa::count_launches(1);
  return ELFA_OK;
}
