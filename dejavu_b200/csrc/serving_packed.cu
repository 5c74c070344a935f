// Causal attention over packed prompts on the CUDA cores, whatever the element type, strides and alignment.
//
// A block takes 64 queries of one head and walks the key tiles of 32 up to its last query; a thread keeps 4 rows x 4 keys of the scores
// and 4 rows x D / 8 columns of the sums in registers, everything in fp32.
#include "serving_packed.cuh"

namespace djv {

constexpr int PS_Q = 64, PS_K = 32, PS_THREADS = 128;

template <typename T, int DP>  // DP: D rounded up
__global__ void __launch_bounds__(PS_THREADS) packed_simple_kernel(PackedArgs a) {
  extern __shared__ float smem[];
  constexpr int LD = DP + 4;
  float *sq = smem, *sk = sq + PS_Q * LD, *sv = sk + PS_K * LD, *sp = sv + PS_K * LD;  // sp (64, 33)
  __shared__ PackedTile tile;
  pdl_prologue();
  const int tid = threadIdx.x, ty = tid / 8, tx = tid % 8, h = blockIdx.y, g = h / (a.H / a.G);
  if (tid < WARP) {
    const PackedTile w = packed_tile<PS_Q>(a, blockIdx.x);
    if (tid == 0) tile = w;
  }
  __syncthreads();
  const PackedTile w = tile;
  if (w.rows <= 0) return;
  T *out = static_cast<T *>(a.out) + ((long long)(w.first + w.q0) * a.H + h) * a.D;
  if (w.rest) {
    if (!a.keep_rest)
      for (int i = tid; i < w.rows * a.D; i += PS_THREADS) out[(long long)(i / a.D) * a.H * a.D + i % a.D] = from_f<T>(0.f);
    return;
  }
  const T *q = static_cast<const T *>(a.q) + (long long)(w.first + w.q0) * a.ldq + h * a.hq;
  const T *k = static_cast<const T *>(a.k) + (long long)w.first * a.ldk + g * a.hk;
  const T *v = static_cast<const T *>(a.v) + (long long)w.first * a.ldv + g * a.hv;
  for (int i = tid; i < PS_Q * DP; i += PS_THREADS) {
    const int r = i / DP, d = i % DP;
    sq[r * LD + d] = r < w.rows && d < a.D ? to_f(q[r * a.ldq + d]) : 0.f;
  }
  float o[4][DP / 8], m[4], l[4];
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    m[i] = -INFINITY;
    l[i] = 0.f;
#pragma unroll
    for (int j = 0; j < DP / 8; ++j) o[i][j] = 0.f;
  }
  const int end = w.q0 + w.rows;  // keys that the last query sees
  for (int j0 = 0; j0 < end; j0 += PS_K) {
    __syncthreads();
    for (int i = tid; i < PS_K * DP; i += PS_THREADS) {
      const int r = i / DP, d = i % DP;
      const bool ok = j0 + r < end && d < a.D;
      sk[r * LD + d] = ok ? to_f(k[(j0 + r) * a.ldk + d]) : 0.f;
      sv[r * LD + d] = ok ? to_f(v[(j0 + r) * a.ldv + d]) : 0.f;
    }
    __syncthreads();
    float s[4][4] = {};
#pragma unroll 4
    for (int d = 0; d < DP; d += 4) {
      float4 x[4], y[4];
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        x[i] = *reinterpret_cast<const float4 *>(sq + (ty * 4 + i) * LD + d);
        y[i] = *reinterpret_cast<const float4 *>(sk + (tx + i * 8) * LD + d);
      }
#pragma unroll
      for (int i = 0; i < 4; ++i)
#pragma unroll
        for (int j = 0; j < 4; ++j)
          s[i][j] = fmaf(x[i].w, y[j].w, fmaf(x[i].z, y[j].z, fmaf(x[i].y, y[j].y, fmaf(x[i].x, y[j].x, s[i][j]))));
    }
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const int row = w.q0 + ty * 4 + i;
      float top = m[i];
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        s[i][j] = j0 + tx + j * 8 <= row ? s[i][j] * a.scale : -INFINITY;
        top = fmaxf(top, s[i][j]);
      }
#pragma unroll
      for (int x = 4; x > 0; x >>= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, x));
      const float base = top == -INFINITY ? 0.f : top, corr = expf(m[i] - base);
      m[i] = top;
      l[i] *= corr;
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const float p = expf(s[i][j] - base);
        l[i] += p;
        sp[(ty * 4 + i) * (PS_K + 1) + tx + j * 8] = p;
      }
#pragma unroll
      for (int j = 0; j < DP / 8; ++j) o[i][j] *= corr;
    }
    __syncwarp();  // (a row's weights are made and read by one warp)
    // a key that a row does not see weighs nothing, whatever its value is
    const bool edge = j0 + PS_K - 1 > w.q0 + ty * 4;
    for (int c = 0; c < PS_K; ++c) {
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        if (edge && j0 + c > w.q0 + ty * 4 + i) continue;
        const float p = sp[(ty * 4 + i) * (PS_K + 1) + c];
#pragma unroll
        for (int j = 0; j < DP / 8; ++j) o[i][j] = fmaf(p, sv[c * LD + tx + j * 8], o[i][j]);
      }
    }
  }
#pragma unroll
  for (int i = 0; i < 4; ++i) {
#pragma unroll
    for (int x = 4; x > 0; x >>= 1) l[i] += __shfl_xor_sync(0xffffffffu, l[i], x);
    const int r = ty * 4 + i;
    if (r >= w.rows) continue;
    const float inv = l[i] == 0.f ? 0.f : 1.f / l[i];
#pragma unroll
    for (int j = 0; j < DP / 8; ++j)
      if (tx + j * 8 < a.D) out[(long long)r * a.H * a.D + tx + j * 8] = from_f<T>(o[i][j] * inv);
  }
}

template <typename T, int DP>
static cudaError_t launch_packed_simple(const PackedArgs &a, cudaStream_t st) {
  constexpr int smem = ((PS_Q + 2 * PS_K) * (DP + 4) + PS_Q * (PS_K + 1)) * 4;
  static DevicePrep prep;
  const int(*unused)[4];
  cudaError_t e = prep.get(
      [&](int(&)[4]) { return cudaFuncSetAttribute(packed_simple_kernel<T, DP>, cudaFuncAttributeMaxDynamicSharedMemorySize, smem); },
      unused);
  if (e != cudaSuccess) return e;
  return djv::launch_kernel(packed_simple_kernel<T, DP>, dim3(packed_tiles<PS_Q>(a.T, a.B), a.H), dim3(PS_THREADS), smem, st, a);
}
template <typename T>
static cudaError_t launch_packed_simple(const PackedArgs &a, cudaStream_t st) {
  return a.D <= 64 ? launch_packed_simple<T, 64>(a, st)
                   : a.D <= 128 ? launch_packed_simple<T, 128>(a, st) : launch_packed_simple<T, 256>(a, st);
}

}  // namespace djv

using namespace djv;

extern "C" int djv_packed_attention(int dtype, void *out, const void *q, long long ldq, long long hq, const void *k, long long ldk,
                                    long long hk, const void *v, long long ldv, long long hv, const int32_t *cu, int B, int T, int H,
                                    int G, int D, float scale, int keep_rest, void *stream) {
  DJV_REQUIRE(is_dtype(dtype), "packed_attention: dtype %d", dtype);
  DJV_REQUIRE(out && q && k && v && cu, "packed_attention: null pointer");
  DJV_REQUIRE(B >= 1 && B <= (1 << 24) && T >= 0 && T <= (1 << 30) && G >= 1 && H >= 1 && H % G == 0 && H <= 65535 && D >= 1 && D <= 256,
              "packed_attention: B=%d T=%d H=%d G=%d D=%d", B, T, H, G, D);
  DJV_REQUIRE(scale == scale && scale - scale == 0.f, "packed_attention: scale %f", scale);
  if (T == 0) return DJV_OK;
  const PackedArgs a{out, q, k, v, ldq, hq, ldk, hk, ldv, hv, cu, B, T, H, G, D, scale, keep_rest};
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  if (packed_tc_supported(dtype, a)) return packed_tc(dtype, a, st);
  const cudaError_t e = dtype == DJV_DTYPE_F16    ? launch_packed_simple<__half>(a, st)
                        : dtype == DJV_DTYPE_BF16 ? launch_packed_simple<bf16>(a, st)
                                                  : launch_packed_simple<float>(a, st);
  if (e != cudaSuccess) {
    cudaGetLastError();
    set_error("packed_attention: CUDA error %d (%s)", (int)e, cudaGetErrorString(e));
    return DJV_ERR_CUDA;
  }
  count_launch();
  return check_launch("packed_attention");
}
