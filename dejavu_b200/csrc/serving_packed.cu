// Causal attention over packed prompts on the CUDA cores, whatever the element type, strides and alignment.
//
// A block takes 64 queries of one head and walks the key tiles of 32 up to its last query; a thread keeps 4 rows x 4 keys of the scores
// and 4 rows x D / 8 columns of the sums in registers, everything in fp32.
#include "pairs.cuh"
#include "serving_packed.cuh"

namespace djv {

constexpr int PS_Q = 128, PS_THREADS = 256, PS_ROWS = 8;  // queries of a block; rows of a thread

template <typename T, int DP>  // DP: D rounded up
__global__ void __launch_bounds__(PS_THREADS) packed_simple_kernel(PackedArgs a) {
  extern __shared__ __align__(16) float smem[];
  constexpr int KEYS = DP > 128 ? 32 : 64, LD = DP + 4, LP = KEYS + 4, J = KEYS / 16, N = DP / 64;
  float *sq = smem, *sk = sq + PS_Q * LD, *sv = sk + KEYS * LD, *sp = sv + KEYS * LD;  // sp (128, LP)
  __shared__ PackedTile tile;
  pdl_prologue();
  const int tid = threadIdx.x, ty = tid / 16, tx = tid % 16, h = blockIdx.y, g = h / (a.H / a.G);
  if (tid < WARP) {
    const PackedTile w = packed_tile<PS_Q>(a, gridDim.x - 1 - blockIdx.x);  // (a sequence's longest tiles go first)
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
#pragma unroll 8
  for (int i = tid; i < PS_Q * DP; i += PS_THREADS) {
    const int r = i / DP, d = i % DP;
    sq[r * LD + d] = r < w.rows && d < a.D ? to_f(q[r * a.ldq + d]) : 0.f;
  }
  // a thread's rows are ty * 8 .., its keys tx + 16 j, its columns tx * 4 + 64 n ..; products go two to an instruction
  uint64_t o[PS_ROWS][2 * N];
  float m[PS_ROWS], l[PS_ROWS];
#pragma unroll
  for (int i = 0; i < PS_ROWS; ++i) {
    m[i] = -INFINITY;
    l[i] = 0.f;
#pragma unroll
    for (int n = 0; n < 2 * N; ++n) o[i][n] = 0;
  }
  const int end = w.q0 + w.rows, depth = (a.D + 3) / 4 * 4;  // keys that the last query sees
  for (int j0 = 0; j0 < end; j0 += KEYS) {
    __syncthreads();
#pragma unroll 8
    for (int i = tid; i < KEYS * DP; i += PS_THREADS) {
      const int r = i / DP, d = i % DP;
      const bool ok = j0 + r < end && d < a.D;
      sk[r * LD + d] = ok ? to_f(k[(j0 + r) * a.ldk + d]) : 0.f;
      sv[r * LD + d] = ok ? to_f(v[(j0 + r) * a.ldv + d]) : 0.f;
    }
    __syncthreads();
    uint64_t s2[PS_ROWS][J] = {};
#pragma unroll 2
    for (int d = 0; d < depth; d += 4) {
      ulonglong2 y[J];
#pragma unroll
      for (int j = 0; j < J; ++j) y[j] = *reinterpret_cast<const ulonglong2 *>(sk + (tx + j * 16) * LD + d);
#pragma unroll
      for (int i = 0; i < PS_ROWS; ++i) {
        const ulonglong2 x = *reinterpret_cast<const ulonglong2 *>(sq + (ty * PS_ROWS + i) * LD + d);
#pragma unroll
        for (int j = 0; j < J; ++j) s2[i][j] = fma2(x.y, y[j].y, fma2(x.x, y[j].x, s2[i][j]));
      }
    }
#pragma unroll
    for (int i = 0; i < PS_ROWS; ++i) {
      const int row = w.q0 + ty * PS_ROWS + i;
      float s[J], top = m[i];
#pragma unroll
      for (int j = 0; j < J; ++j) {
        float lo, hi;
        unpack2(s2[i][j], lo, hi);
        s[j] = j0 + tx + j * 16 <= row ? (lo + hi) * a.scale : -INFINITY;
        top = fmaxf(top, s[j]);
      }
#pragma unroll
      for (int x = 8; x > 0; x >>= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, x));
      const float base = top == -INFINITY ? 0.f : top, corr = expf(m[i] - base);
      m[i] = top;
      l[i] *= corr;
#pragma unroll
      for (int j = 0; j < J; ++j) {
        const float p = expf(s[j] - base);
        l[i] += p;
        sp[(ty * PS_ROWS + i) * LP + tx + j * 16] = p;
      }
      const uint64_t corr2 = pack2(corr, corr);
#pragma unroll
      for (int n = 0; n < 2 * N; ++n) o[i][n] = fma2(o[i][n], corr2, 0);
    }
    __syncwarp();  // (a row's weights are made and read by one warp)
    auto add = [&](int i, int c, float p) {
      const uint64_t p2 = pack2(p, p);
#pragma unroll
      for (int n = 0; n < N; ++n) {
        const ulonglong2 y = *reinterpret_cast<const ulonglong2 *>(sv + c * LD + n * 64 + tx * 4);
        o[i][2 * n] = fma2(p2, y.x, o[i][2 * n]);
        o[i][2 * n + 1] = fma2(p2, y.y, o[i][2 * n + 1]);
      }
    };
    if (j0 + KEYS - 1 <= w.q0 + ty * PS_ROWS) {
#pragma unroll 1
      for (int c = 0; c < KEYS; c += 4) {
        float p[PS_ROWS][4];
#pragma unroll
        for (int i = 0; i < PS_ROWS; ++i) *reinterpret_cast<float4 *>(p[i]) = *reinterpret_cast<const float4 *>(sp + (ty * PS_ROWS + i) * LP + c);
#pragma unroll
        for (int e = 0; e < 4; ++e)
#pragma unroll
          for (int i = 0; i < PS_ROWS; ++i) add(i, c + e, p[i][e]);
      }
    } else {  // a key that a row does not see weighs nothing, whatever its value is
#pragma unroll 1
      for (int c = 0; c < KEYS; ++c)
#pragma unroll
        for (int i = 0; i < PS_ROWS; ++i)
          if (j0 + c <= w.q0 + ty * PS_ROWS + i) add(i, c, sp[(ty * PS_ROWS + i) * LP + c]);
    }
  }
#pragma unroll
  for (int i = 0; i < PS_ROWS; ++i) {
#pragma unroll
    for (int x = 8; x > 0; x >>= 1) l[i] += __shfl_xor_sync(0xffffffffu, l[i], x);
    const int r = ty * PS_ROWS + i;
    if (r >= w.rows) continue;
    const float inv = l[i] == 0.f ? 0.f : 1.f / l[i];
#pragma unroll
    for (int n = 0; n < 2 * N; ++n) {
      const int d = n / 2 * 64 + tx * 4 + n % 2 * 2;
      float x, y;
      unpack2(o[i][n], x, y);
      if (d < a.D) out[(long long)r * a.H * a.D + d] = from_f<T>(x * inv);
      if (d + 1 < a.D) out[(long long)r * a.H * a.D + d + 1] = from_f<T>(y * inv);
    }
  }
}

template <typename T, int DP>
static cudaError_t launch_packed_simple(const PackedArgs &a, cudaStream_t st) {
  constexpr int keys = DP > 128 ? 32 : 64, smem = ((PS_Q + 2 * keys) * (DP + 4) + PS_Q * (keys + 4)) * 4;
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
