// New tokens enter a paged cache: rotation of q and k, store of k and v into their pages, in one pass over the rows.
//
// A block of 128 threads takes one row: its angles are shared by all heads. What it reads of q, k and v, 16 bytes at a time, depends on
// nothing and is asked for first; beside it runs the chain offsets -> position -> angles, page, which every warp goes through for
// itself, so that the block meets once, over the angles. Small blocks, many of them on a multiprocessor, hide that chain.
// Bound by HBM for prompts (8191 rows of 32 + 2 x 8 heads of 128, bf16: 41 us for 218 MB, 0.81 of the copy rate; element by element 180;
// fp32 82 us), by the chain for a few rows (one row: 3.4 us in a graph, fp32 5.1). Layouts that 16-byte accesses cannot read go element by element.
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

// The sequence of row t, or -1. By a warp.
__device__ __forceinline__ int sequence_of(const int *cu, int B, int t) {
  const int lane = threadIdx.x % WARP;
  SequenceSearch s{0, B};
  while (!s.done()) {
    const int at = s.probe(lane);
    s.narrow(32 - __clz(__ballot_sync(0xffffffffu, at < s.hi && cu[at] <= t)));
  }
  return cu[s.lo] <= t && t < cu[s.lo + 1] ? s.lo : -1;
}

// Row t's position and page, by all lanes of a warp. p < 0: no such token.
struct AppendPlace {
  long long p, at;  // at: offset of (page, slot), head 0, or -1
};
__device__ __forceinline__ AppendPlace append_place(const AppendArgs &a, int t) {
  const int b = a.cu == nullptr ? t : sequence_of(a.cu, a.B, t);
  AppendPlace w{-1, -1};
  if (b < 0) return w;
  const long long begin = a.pos[b], row = a.cu == nullptr ? 0 : t - a.cu[b], most = 0x7fffffffffffffffll;
  w.p = begin > most - row ? most : begin + row;  // (behind every table all the same)
  if (w.p < 0) return w;
  int slot;
  const PageMap m{a.table + b * a.ld_table, a.width, a.page, a.pages, a.by_page};
  const long long page = page_of(m, w.p, slot);
  if (page != NO_PAGE) w.at = page * a.pool.ld_page + slot * a.pool.ld_slot;
  else if (threadIdx.x == 0) atomicAdd(&g_append_faults, 1u);
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
  pdl_prologue();
  const int t = blockIdx.x;
  const AppendPlace w = append_place(a, t);
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

constexpr int AP_THREADS = 128, AP_DEEP = 4;  // pieces of a thread that are asked for before the angles are known

// 16 bytes at a time. A piece is two chunks that are rotated with each other, one of neighbouring pairs (NEXT), or one that is copied.
template <typename T, bool NEXT>
__global__ void __launch_bounds__(AP_THREADS) append_kernel(AppendArgs a) {
  constexpr int N = Chunk<T>::N;
  extern __shared__ float cs[];  // cos[half], sin[half]
  pdl_prologue();
  const int t = blockIdx.x, heads = a.q_out ? a.H : 0;
  const int rot = (NEXT ? 2 * a.half : a.half) / N, rest = (a.D - 2 * a.half) / N, whole = a.D / N;  // pieces of a head
  const int n_rot = (heads + a.G) * rot, n_rest = (heads + a.G) * rest, total = n_rot + n_rest + a.G * whole;
  struct Piece {
    int h, d;  // head: q's, then k's, then v's; first dimension
    bool turned;
  };
  auto piece = [&](int i) {
    Piece p;
    if (i < n_rot) {
      p.h = i / rot;
      p.d = (i - p.h * rot) * N;
      p.turned = true;
    } else if (i < n_rot + n_rest) {
      i -= n_rot;
      p.h = i / rest;
      p.d = 2 * a.half + (i - p.h * rest) * N;
      p.turned = false;
    } else {
      i -= n_rot + n_rest;
      p.h = i / whole;
      p.d = (i - p.h * whole) * N;
      p.h += heads + a.G;
      p.turned = false;
    }
    return p;
  };
  auto source = [&](const Piece &p) {
    return (p.h < heads ? static_cast<const T *>(a.q) + (long long)t * a.ldq + p.h * a.hq
            : p.h < heads + a.G ? static_cast<const T *>(a.k) + (long long)t * a.ldk + (p.h - heads) * a.hk
                                : static_cast<const T *>(a.v) + (long long)t * a.ldv + (p.h - heads - a.G) * a.hv) + p.d;
  };
  auto ask = [&](int i, uint4 &x, uint4 &y) {
    if (i >= total) return;
    const Piece p = piece(i);
    const T *src = source(p);
    x = ld_cached16(src);
    if (!NEXT && p.turned) y = ld_cached16(src + a.half);
  };
  uint4 x[AP_DEEP] = {}, y[AP_DEEP] = {};
#pragma unroll
  for (int i = 0; i < AP_DEEP; ++i) ask(i * AP_THREADS + threadIdx.x, x[i], y[i]);
  const AppendPlace w = append_place(a, t);
  if (w.p >= 0) append_angles(a, w.p, cs);
  __syncthreads();
  auto put = [&](int i, uint4 x, uint4 y) {
    if (i >= total) return;
    const Piece p = piece(i);
    const bool two = !NEXT && p.turned;
    if (w.p < 0) {
      x = y = make_uint4(0, 0, 0, 0);
    } else if (p.turned) {
      float u[N], v[N];
      T ru[N], rv[N];
      unpack_chunk<T>(x, u);
      if (NEXT) {
#pragma unroll
        for (int e = 0; e < N; e += 2) {
          const float c = cs[(p.d + e) / 2], s = cs[a.half + (p.d + e) / 2];
          ru[e] = from_f<T>(u[e] * c - u[e + 1] * s);
          ru[e + 1] = from_f<T>(u[e + 1] * c + u[e] * s);
        }
      } else {
        unpack_chunk<T>(y, v);
#pragma unroll
        for (int e = 0; e < N; ++e) {
          const float c = cs[p.d + e], s = cs[a.half + p.d + e];
          ru[e] = from_f<T>(u[e] * c - v[e] * s);
          rv[e] = from_f<T>(v[e] * c + u[e] * s);
        }
        y = *reinterpret_cast<uint4 *>(rv);
      }
      x = *reinterpret_cast<uint4 *>(ru);
    }
    auto store = [&](T *dst) {
      *reinterpret_cast<uint4 *>(dst) = x;
      if (two) *reinterpret_cast<uint4 *>(dst + a.half) = y;
    };
    if (p.h < heads) {
      store(static_cast<T *>(a.q_out) + ((long long)t * a.H + p.h) * a.D + p.d);
    } else if (p.h < heads + a.G) {
      const int g = p.h - heads;
      if (a.k_out) store(static_cast<T *>(a.k_out) + ((long long)t * a.G + g) * a.D + p.d);
      if (w.at >= 0) store(static_cast<T *>(a.k_pages) + w.at + g * a.pool.ld_head + p.d);
    } else if (w.at >= 0) {
      store(static_cast<T *>(a.v_pages) + w.at + (p.h - heads - a.G) * a.pool.ld_head + p.d);
    }
  };
#pragma unroll
  for (int i = 0; i < AP_DEEP; ++i) put(i * AP_THREADS + threadIdx.x, x[i], y[i]);
  for (int i = AP_DEEP * AP_THREADS + threadIdx.x; i < total; i += AP_THREADS) {
    uint4 p = {}, q = {};
    ask(i, p, q);
    put(i, p, q);
  }
}

template <typename T>
static cudaError_t launch_append(const AppendArgs &a, int rows, bool vec, int interleaved, cudaStream_t st) {
  if (!vec) return djv::launch_kernel(append_simple_kernel<T>, dim3(rows), dim3(256), 0, st, a, interleaved);
  return interleaved ? djv::launch_kernel(append_kernel<T, true>, dim3(rows), dim3(AP_THREADS), a.half * 8, st, a)
                     : djv::launch_kernel(append_kernel<T, false>, dim3(rows), dim3(AP_THREADS), a.half * 8, st, a);
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
  const auto fits = [&](const void *p, long long ld, long long head) { return aligned16(p) && ld % chunk == 0 && head % chunk == 0; };
  const bool vec = fits(k, ldk, hk) && fits(v, ldv, hv) && (!q_out || (fits(q, ldq, hq) && aligned16(q_out))) && aligned16(k_out) &&
                   (interleaved ? 2 * half : half) % chunk == 0;
  if (dtype == DJV_DTYPE_F16) launch_append<__half>(a, T, vec, interleaved, st);
  else if (dtype == DJV_DTYPE_BF16) launch_append<bf16>(a, T, vec, interleaved, st);
  else launch_append<float>(a, T, vec, interleaved, st);
  count_launch();
  return check_launch("paged_append");
}
