// Moving keys and values into and between the pages of a cache (layout: see paged.cuh). Both kernels only copy: bound by the memory, or by the
// launch where they move little.
#include <cstdlib>
#include <cstring>

#include "elfa_native.h"
#include "paged.cuh"

namespace elfa {

int paged_geom(PagedGeom* g, const void* pages, const int* table, const int* q_start, const int* kv_len, int B, int N, int P, int page, int T, int H,
               int Hkv, int hd, int max_new, int window, int sinks);

namespace {

// A block takes `per` tokens: their places are looked up once (a search for the sequence, then the table); then a thread has a 16-byte piece of a token, works out once
// where it goes and moves it for all of the tokens, their loads ahead of their stores. 12 thousand tokens of 8 heads of 128 (99 MB): 20.5 us,
// 4.8 TB/s (22.8 with a division per piece and token, which two thirds of the issue slots went to).
struct WriteArgs {
  PagedGeom g;
  const uint4 *k, *v;
  uint4* pages;
  long long ks, vs;                        // 16-byte vectors from a token to the next
};
template <int PER>
__global__ void __launch_bounds__(256) paged_write_kernel(const __grid_constant__ WriteArgs a) {
  __shared__ long long place[PER];      // vector index of (page, key half, head 0, row), -1: nowhere
  const PagedGeom& g = a.g;
  const int t0 = blockIdx.x * PER, count = min(PER, g.T - t0), page = 1 << g.page_shift, hv = g.hd / 8;
  if ((int)threadIdx.x < count) {
    const int t = t0 + threadIdx.x;
    int lo = 0, hi = g.B;                  // the last sequence that starts at or before t (empty ones start where the next one does)
    while (hi - lo > 1) {
      const int mid = (lo + hi) >> 1;
      if (g.q_start[mid] <= t) lo = mid;
      else hi = mid;
    }
    bool fits;                             // else the clamped lengths would lead to the places of other tokens
    const PagedSeq s = paged_seq(g, lo, &fits);
    fits = fits && s.kv == g.kv_len[lo] && s.n <= s.kv;
    const int pos = s.kv - s.n + t - s.q0;
    long long at = -1;
    if (fits && t >= s.q0 && t < s.q0 + s.n) {
      const int id = paged_page(g, lo, pos);
      if (id >= 0) at = ((long long)id * 2 * g.Hkv * page + (pos & (page - 1))) * hv;
    }
    if (at < 0) atomicOr(g.status, (unsigned)ELFA_ST_BAD_PAGE);      // a new token without a page would be lost
    place[threadIdx.x] = at;
  }
  __syncthreads();
  const int row = g.Hkv * hv, all = 2 * row;
  const long long head = (long long)page * hv;
  for (int c = threadIdx.x; c < all; c += 256) {
    const int half = c >= row, x = c - half * row, h = x / hv;
    const uint4* from = half ? a.v + t0 * a.vs + x : a.k + t0 * a.ks + x;
    uint4* to = a.pages + ((long long)half * g.Hkv + h) * head + (x - h * hv);
    const long long step = half ? a.vs : a.ks;
    uint4 val[PER];
#pragma unroll
    for (int t = 0; t < PER; ++t)
      if (t < count) val[t] = __ldcs(from + t * step);
#pragma unroll
    for (int t = 0; t < PER; ++t)
      if (t < count && place[t] >= 0) to[place[t]] = val[t];
  }
}

// The page numbers travel with the launch: no copy to the device, and nothing that a later call could overwrite while this one waits. 300 pages of 256 KB in 8
// layers: 197 us, 6.4 TB/s, the rate of a plain copy.
constexpr int COPY_PAIRS = 480, COPY_VECS = 4;
struct CopyArgs {
  uint4* pages;
  long long layer, page;                   // vectors per layer and page
  int pair[COPY_PAIRS][2];
};
// grid (pieces of a page, pairs, layers)
__global__ void __launch_bounds__(256) copy_pages_kernel(const __grid_constant__ CopyArgs a) {
  const int from = a.pair[blockIdx.y][0], to = a.pair[blockIdx.y][1];
  uint4* base = a.pages + blockIdx.z * a.layer;
  const uint4* s = base + from * a.page;
  uint4* d = base + to * a.page;
  const long long i0 = (long long)blockIdx.x * 256 * COPY_VECS + threadIdx.x;
  uint4 v[COPY_VECS];
#pragma unroll
  for (int x = 0; x < COPY_VECS; ++x)
    if (i0 + x * 256 < a.page) v[x] = __ldcs(s + i0 + x * 256);
#pragma unroll
  for (int x = 0; x < COPY_VECS; ++x)
    if (i0 + x * 256 < a.page) __stcs(d + i0 + x * 256, v[x]);
}

}  // namespace
}  // namespace elfa

using namespace elfa;

// k, v: rows [T] of Hkv packed heads, ks / vs elements apart, 16-byte aligned.
ELFA_API int elfa_paged_write(const void* k, long long ks, const void* v, long long vs, void* pages, const int* table, const int* q_start,
                              const int* kv_len, int B, int N, int P, int page, int T, int Hkv, int hd, void* stream) {
  WriteArgs a{};
  const int rc = paged_geom(&a.g, pages, table, q_start, kv_len, B, N, P, page, T, Hkv, Hkv, hd, T, 0, 0);
  if (rc != ELFA_OK) return rc;
  ELFA_REQUIRE(k && v, "paged_write: null pointer");
  ELFA_REQUIRE(ks % 8 == 0 && vs % 8 == 0 && ((reinterpret_cast<uintptr_t>(k) | reinterpret_cast<uintptr_t>(v)) & 15) == 0,
               "paged_write: rows must lie on 16-byte boundaries");
  a.k = static_cast<const uint4*>(k);
  a.v = static_cast<const uint4*>(v);
  a.pages = static_cast<uint4*>(pages);
  a.ks = ks / 8;
  a.vs = vs / 8;
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  if (T >= 148 * 32) paged_write_kernel<8><<<(T + 7) / 8, 256, 0, st>>>(a);
  else if (T >= 148 * 4) paged_write_kernel<2><<<(T + 1) / 2, 256, 0, st>>>(a);
  else paged_write_kernel<1><<<T, 256, 0, st>>>(a);
  ELFA_CUDA(cudaGetLastError());
  ::elfa::count_launches(1);
  return ELFA_OK;
}

// pages: [L][P] pages of page_bytes each, layer_bytes from a layer to the next. pairs: host array of n (from, to). Copies all of them in all layers;
// a page is written once at most and no page that is written is read, so their order does not matter.
ELFA_API int elfa_copy_pages(void* pages, long long layer_bytes, long long page_bytes, int L, int P, const int* from, const int* to, int n, void* stream) {
  ELFA_REQUIRE(pages && from && to, "copy_pages: null pointer");
  ELFA_REQUIRE(L > 0 && L <= 65535 && P > 0 && n >= 0 && page_bytes > 0, "copy_pages: bad sizes");
  ELFA_REQUIRE(page_bytes % 16 == 0 && layer_bytes % 16 == 0 && (reinterpret_cast<uintptr_t>(pages) & 15) == 0,
               "copy_pages: pages must be multiples of 16 bytes on 16-byte boundaries");
  const long long vecs = page_bytes / 16, pieces = (vecs + 256 * COPY_VECS - 1) / (256 * COPY_VECS);
  ELFA_REQUIRE(pieces < 0x7fffffffLL, "copy_pages: pages are too large");
  if (n == 0) return ELFA_OK;
  unsigned char* mark = static_cast<unsigned char*>(calloc((size_t)P, 1));
  ELFA_REQUIRE(mark != nullptr, "copy_pages: out of memory");
  const char* wrong = nullptr;
  for (int i = 0; i < n && !wrong; ++i) {
    if (from[i] < 0 || from[i] >= P || to[i] < 0 || to[i] >= P) wrong = "copy_pages: a page outside the pool";
    else mark[from[i]] |= 1;
  }
  for (int i = 0; i < n && !wrong; ++i) {
    if (mark[to[i]] & 1) wrong = "copy_pages: a page is both read and written";
    else if (mark[to[i]] & 2) wrong = "copy_pages: a page is written twice";
    mark[to[i]] |= 2;
  }
  free(mark);
  ELFA_REQUIRE(!wrong, wrong);
  CopyArgs a;
  a.pages = static_cast<uint4*>(pages);
  a.layer = layer_bytes / 16;
  a.page = vecs;
  for (int i0 = 0; i0 < n; i0 += COPY_PAIRS) {
    const int m = n - i0 < COPY_PAIRS ? n - i0 : COPY_PAIRS;
    for (int i = 0; i < m; ++i) {
      a.pair[i][0] = from[i0 + i];
      a.pair[i][1] = to[i0 + i];
    }
    copy_pages_kernel<<<dim3((unsigned)pieces, m, L), 256, 0, static_cast<cudaStream_t>(stream)>>>(a);
    ELFA_CUDA(cudaGetLastError());
    ::elfa::count_launches(1);
  }
  return ELFA_OK;
}
