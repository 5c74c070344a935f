// Attention of one new token per sequence over its paged cache.
#include "serving.cuh"

namespace djv {

__device__ unsigned g_decode_faults;

struct DecodeArgs {
  void *out;
  const void *q, *k, *v;
  long long ldq, hq;
  Pool pool;
  int pages, page;
  const int *table;
  long long ld_table;
  int width;
  const long long *pos;
  int B, H, G, D;
  float scale;
};

// A block takes one head of one sequence, its warps every fourth token with a softmax of their own, joined at the end.
template <typename T>
__global__ void __launch_bounds__(128) decode_simple_kernel(DecodeArgs a) {
  __shared__ float sm[4], sl[4], so[4][256];
  pdl_prologue();
  const int h = blockIdx.x, b = blockIdx.y, g = h / (a.H / a.G), warp = threadIdx.x / WARP, lane = threadIdx.x % WARP;
  long long n = a.pos[b] + 1;
  const long long room = (long long)a.width * a.page;
  if (n > room) {
    if (threadIdx.x == 0 && h == 0) atomicAdd(&g_decode_faults, 1u);
    n = room;
  }
  const T *q = static_cast<const T *>(a.q) + b * a.ldq + h * a.hq;
  float qr[8], o[8], m = -INFINITY, l = 0.f;
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    qr[i] = lane + i * 32 < a.D ? to_f(q[lane + i * 32]) : 0.f;
    o[i] = 0.f;
  }
  const PageMap map{a.table + b * a.ld_table, a.width, a.page, a.pages};
  for (long long t = warp; t < n; t += 4) {
    int slot;
    const long long page = page_of(map, t, slot);
    if (page == NO_PAGE) {
      if (lane == 0 && h == 0 && (slot == 0 || t == n - 1)) atomicAdd(&g_decode_faults, 1u);
      continue;
    }
    const long long at = page * a.pool.ld_page + g * a.pool.ld_head + slot * a.pool.ld_slot;
    const T *k = static_cast<const T *>(a.k) + at, *v = static_cast<const T *>(a.v) + at;
    float s = 0.f;
#pragma unroll
    for (int i = 0; i < 8; ++i)
      if (lane + i * 32 < a.D) s = fmaf(qr[i], to_f(k[lane + i * 32]), s);
    s = warp_sum(s) * a.scale;
    const float top = fmaxf(m, s), base = top == -INFINITY ? 0.f : top;
    const float corr = expf(m - base), p = expf(s - base);
    m = top;
    l = l * corr + p;
#pragma unroll
    for (int i = 0; i < 8; ++i)
      if (lane + i * 32 < a.D) o[i] = fmaf(p, to_f(v[lane + i * 32]), o[i] * corr);
  }
  if (lane == 0) {
    sm[warp] = m;
    sl[warp] = l;
  }
#pragma unroll
  for (int i = 0; i < 8; ++i)
    if (lane + i * 32 < a.D) so[warp][lane + i * 32] = o[i];
  __syncthreads();
  float top = -INFINITY, sum = 0.f;
  for (int w = 0; w < 4; ++w) top = fmaxf(top, sm[w]);
  if (top == -INFINITY) top = 0.f;
  for (int w = 0; w < 4; ++w) sum += sl[w] * expf(sm[w] - top);
  for (int d = threadIdx.x; d < a.D; d += blockDim.x) {
    float x = 0.f;
    for (int w = 0; w < 4; ++w) x += so[w][d] * expf(sm[w] - top);
    static_cast<T *>(a.out)[((long long)b * a.H + h) * a.D + d] = from_f<T>(sum == 0.f ? 0.f : x / sum);
  }
}

unsigned decode_faults() {
  unsigned v = 0;
  if (cudaMemcpyFromSymbol(&v, g_decode_faults, sizeof(v)) != cudaSuccess) {
    cudaGetLastError();
    return 0;
  }
  return v;
}

}  // namespace djv

using namespace djv;

extern "C" size_t djv_paged_attention_scratch_bytes(int, int, int, int, int, int, int) { return 0; }

extern "C" int djv_paged_attention(int dtype, void *out, const void *q, long long ldq, long long hq, const void *k_pages,
                                   const void *v_pages, long long ld_page, long long ld_head, long long ld_slot, int pages, int page,
                                   const int32_t *table, long long ld_table, int width, const long long *pos, int B, int H, int G,
                                   int D, float scale, void *scratch, size_t scratch_bytes, void *stream) {
  DJV_REQUIRE(is_dtype(dtype), "paged_attention: dtype %d", dtype);
  DJV_REQUIRE(out && q && k_pages && v_pages && table && pos, "paged_attention: null pointer");
  const int chunk = 16 / (int)dtype_bytes(dtype);
  DJV_REQUIRE(B >= 0 && B <= 65535 && G >= 1 && H >= 1 && H % G == 0 && H <= 65536 && pages >= 1 && page >= 1 && width >= 1 &&
                  (long long)width * page < (1ll << 31) && D >= 1 && D <= 256,
              "paged_attention: B=%d H=%d G=%d D=%d pages=%d of %d, table %d wide", B, H, G, D, pages, page, width);
  DJV_REQUIRE(D % chunk == 0 && aligned16(k_pages) && aligned16(v_pages) && ld_page % chunk == 0 && ld_head % chunk == 0 &&
                  ld_slot % chunk == 0 && aligned16(q) && ldq % chunk == 0 && hq % chunk == 0 && aligned16(out),
              "paged_attention: rows start on multiples of 16 bytes");
  DJV_REQUIRE(scale == scale && scale - scale == 0.f, "paged_attention: scale %f", scale);
  if (B == 0) return DJV_OK;
  if (scratch_bytes < djv_paged_attention_scratch_bytes(dtype, B, H, G, D, page, width) || !aligned16(scratch)) {
    set_error("paged_attention: scratch");
    return DJV_ERR_SCRATCH;
  }
  const DecodeArgs a{out, q, k_pages, v_pages, ldq, hq, {ld_page, ld_head, ld_slot}, pages, page, table, ld_table, width, pos,
                     B, H, G, D, scale};
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  if (dtype == DJV_DTYPE_F16) djv::launch_kernel(decode_simple_kernel<__half>, dim3(H, B), dim3(128), 0, st, a);
  else if (dtype == DJV_DTYPE_BF16) djv::launch_kernel(decode_simple_kernel<bf16>, dim3(H, B), dim3(128), 0, st, a);
  else djv::launch_kernel(decode_simple_kernel<float>, dim3(H, B), dim3(128), 0, st, a);
  count_launch();
  return check_launch("paged_attention");
}
