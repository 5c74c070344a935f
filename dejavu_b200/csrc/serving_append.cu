// New tokens enter a paged cache: rotation of q and k, store of k and v into their pages, in one pass over the rows.
//
// A block takes one row: its angles are shared by all heads. The row is in registers before the angles are known (16-byte loads that
// depend on nothing), so what a block waits for is one round of loads, the position's own short chain beside it, and its stores.
// Bound by HBM for prompts, by that one round for a few rows.
//
// Angles: position * frequency is exact in 64 bits up to positions of 2^29; what is left of it after whole turns are taken off in 64
// bits is rounded to 32 and goes through sincosf, so that far positions are as exact as near ones (in 32 bits the angle of position
// 131071 would be off by 2^-8).
#include <math.h>

#include "serving.cuh"

namespace djv {

__device__ unsigned g_append_faults;

constexpr int AP_MAX_HALF = 1024;

struct AppendArgs {
  void *q_out, *k_out, *k_pages, *v_pages;
  const void *q, *k, *v;
  long long ldq, hq, ldk, hk, ldv, hv;
  Pool pool;
  int pages, page;
  Divider by_page;
  const int *table;
  long long ld_table;
  int width;
  const long long *pos;
  const int *cu;
  const float *freqs;
  float amp;
  int half, B, H, G, D;
};

// Row t's position and page, by one thread. p < 0: no such token.
struct AppendPlace {
  long long p, at;  // at: offset of (page, slot), head 0, or -1
};
__device__ __forceinline__ AppendPlace append_place(const AppendArgs &a, int t) {
  const int b = a.cu == nullptr ? t : sequence_of(a.cu, a.B, t);
  AppendPlace w{-1, -1};
  if (b < 0) return w;
  w.p = a.pos[b] + (a.cu == nullptr ? 0 : t - a.cu[b]);
  if (w.p < 0) return w;
  int slot;
  const PageMap m{a.table + b * a.ld_table, a.width, a.page, a.pages, a.by_page};
  const long long page = page_of(m, w.p, slot);
  if (page == NO_PAGE) atomicAdd(&g_append_faults, 1u);
  else w.at = page * a.pool.ld_page + slot * a.pool.ld_slot;
  return w;
}

__device__ __forceinline__ void append_angles(const AppendArgs &a, long long p, float *cs) {
  for (int i = threadIdx.x; i < a.half; i += blockDim.x) {
    const double turn = 6.283185307179586477, angle = (double)p * (double)a.freqs[i];
    const double rest = angle - turn * rint(angle / turn);
    float s, c;
    sincosf((float)rest, &s, &c);
    cs[i] = c * a.amp;
    cs[a.half + i] = s * a.amp;
  }
}

// One element pair at a time: any strides and any address.
template <typename T>
__global__ void append_simple_kernel(AppendArgs a, int interleaved) {
  __shared__ float cs[2 * AP_MAX_HALF];
  __shared__ AppendPlace place;
  pdl_prologue();
  const int t = blockIdx.x;
  if (threadIdx.x == 0) place = append_place(a, t);
  __syncthreads();
  const AppendPlace w = place;
  if (a.half && w.p >= 0) append_angles(a, w.p, cs);
  __syncthreads();
  const int heads = a.q_out ? a.H : 0, total = (heads + 2 * a.G) * a.D;
  for (int i = threadIdx.x; i < total; i += blockDim.x) {
    const int h = i / a.D, d = i - h * a.D;
    const T *src = h < heads ? static_cast<const T *>(a.q) + t * a.ldq + h * a.hq
                   : h < heads + a.G ? static_cast<const T *>(a.k) + t * a.ldk + (h - heads) * a.hk
                                     : static_cast<const T *>(a.v) + t * a.ldv + (h - heads - a.G) * a.hv;
    T r = src[d];
    if (w.p < 0) {
      r = from_f<T>(0.f);
    } else if (h < heads + a.G && d < 2 * a.half) {
      const int pair = interleaved ? d / 2 : (d < a.half ? d : d - a.half);
      const bool second = interleaved ? (d & 1) != 0 : d >= a.half;
      const float x = to_f(src[interleaved ? 2 * pair : pair]), y = to_f(src[interleaved ? 2 * pair + 1 : pair + a.half]);
      r = from_f<T>(second ? y * cs[pair] + x * cs[a.half + pair] : x * cs[pair] - y * cs[a.half + pair]);
    }
    if (h < heads) {
      static_cast<T *>(a.q_out)[((long long)t * a.H + h) * a.D + d] = r;
    } else if (h < heads + a.G) {
      const int g = h - heads;
      if (a.k_out) static_cast<T *>(a.k_out)[((long long)t * a.G + g) * a.D + d] = r;
      if (w.at >= 0) static_cast<T *>(a.k_pages)[w.at + g * a.pool.ld_head + d] = r;
    } else if (w.at >= 0) {
      static_cast<T *>(a.v_pages)[w.at + (h - heads - a.G) * a.pool.ld_head + d] = r;
    }
  }
}

unsigned append_faults() {
  unsigned v = 0;
  if (cudaMemcpyFromSymbol(&v, g_append_faults, sizeof(v)) != cudaSuccess) {
    cudaGetLastError();
    return 0;
  }
  return v;
}

}  // namespace djv

using namespace djv;

extern "C" unsigned djv_paged_faults(void) { return append_faults() + decode_faults(); }

extern "C" unsigned djv_serving_timeouts(void) { return decode_timeouts() + packed_timeouts(); }

extern "C" int djv_paged_append(int dtype, void *q_out, void *k_out, const void *q, long long ldq, long long hq, const void *k,
                                long long ldk, long long hk, const void *v, long long ldv, long long hv, void *k_pages,
                                void *v_pages, long long ld_page, long long ld_head, long long ld_slot, int pages, int page,
                                const int32_t *table, long long ld_table, int width, const long long *pos, const int32_t *cu,
                                const float *freqs, float amp, int half, int interleaved, int B, int T, int H, int G, int D,
                                void *stream) {
  DJV_REQUIRE(is_dtype(dtype), "paged_append: dtype %d", dtype);
  DJV_REQUIRE(k && v && k_pages && v_pages && table && pos && (!q_out || q) && (half == 0 || freqs), "paged_append: null pointer");
  const int chunk = 16 / (int)dtype_bytes(dtype);
  DJV_REQUIRE(B >= 1 && T >= 0 && (cu || T == B) && G >= 1 && H >= (q_out ? 1 : 0) && pages >= 1 && page >= 1 && width >= 1 &&
                  (long long)width * page < (1ll << 31) && D >= 1 && D <= 2 * AP_MAX_HALF && half >= 0 && 2 * half <= D &&
                  (long long)(H + 2 * G) * D < (1ll << 30),
              "paged_append: B=%d T=%d H=%d G=%d D=%d half=%d pages=%d of %d, table %d wide", B, T, H, G, D, half, pages, page, width);
  DJV_REQUIRE(D % chunk == 0 && aligned16(k_pages) && aligned16(v_pages) && ld_page % chunk == 0 && ld_head % chunk == 0 &&
                  ld_slot % chunk == 0,
              "paged_append: rows of the pages start on multiples of 16 bytes");
  if (T == 0) return DJV_OK;
  const AppendArgs a{q_out, k_out, k_pages, v_pages, q, k, v, ldq, hq, ldk, hk, ldv, hv, {ld_page, ld_head, ld_slot}, pages, page,
                     divider_of(page), table, ld_table, width, pos, cu, freqs, amp, half, B, H, G, D};
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  if (dtype == DJV_DTYPE_F16) djv::launch_kernel(append_simple_kernel<__half>, dim3(T), dim3(256), 0, st, a, interleaved);
  else if (dtype == DJV_DTYPE_BF16) djv::launch_kernel(append_simple_kernel<bf16>, dim3(T), dim3(256), 0, st, a, interleaved);
  else djv::launch_kernel(append_simple_kernel<float>, dim3(T), dim3(256), 0, st, a, interleaved);
  count_launch();
  return check_launch("paged_append");
}
