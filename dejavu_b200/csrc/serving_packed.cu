// Causal attention over packed prompts on the CUDA cores, whatever the element type, strides and alignment.
//
// A block takes 128 queries of one head and walks the key tiles of 64 up to its last query; a thread keeps 8 rows x 4 keys of the scores
// and 8 rows x D / 16 columns of the sums in registers, everything in fp32. What bounds it are the loads of operands from shared memory,
// 12 of 16 bytes for 64 instructions of two products each in the scores. fp32, one prompt of 4096 tokens, 16 heads over 8: heads of
// 64 1.26 ms, of 128 2.6 ms (27 TFLOP/s), of 256 5.5 ms (25; library products of whole score matrices take 5.0). With 64 queries, 4 rows and a key
// tile of 32: 2.6, 4.8 and 22.6 ms.
#include "pairs.cuh"
#include "serving_packed.cuh"

namespace djv {

constexpr int PS_Q = 128, PS_KEYS = 64, PS_THREADS = 256, PS_ROWS = 8;  // queries of a block, keys of a tile; rows of a thread

template <typename T, int DP>  // DP: D rounded up
__global__ void __launch_bounds__(PS_THREADS) packed_simple_kernel(PackedArgs a) {
  extern __shared__ __align__(16) float smem[];
  // Key and value tiles are staged by up to 128 columns at a time; where that is all there are, both at once.
  constexpr int KEYS = PS_KEYS, COLS = DP < 128 ? DP : 128, PARTS = DP / COLS, LD = DP + 4, LK = COLS + 4, LP = KEYS + 4, J = KEYS / 16, N = DP / 64;
  float *sq = smem, *sk = sq + PS_Q * LD, *sv = PARTS > 1 ? sk : sk + KEYS * LK, *sp = sv + KEYS * LK;  // sp (128, LP)
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
  auto stage = [&](float *to, const T *from, long long ld, int j0, int part) {
    constexpr int EACH = KEYS * COLS / PS_THREADS, STEP = PS_THREADS / COLS;  // a thread's column, and rows; all of its loads are on their way at once
    const int r0 = tid / COLS, c = tid % COLS, d = c + part * COLS;
    const T *at = from + (j0 + r0) * ld + d;
    T x[EACH];
#pragma unroll
    for (int i = 0; i < EACH; ++i) x[i] = j0 + r0 + i * STEP < end && d < a.D ? at[i * STEP * ld] : from_f<T>(0.f);
#pragma unroll
    for (int i = 0; i < EACH; ++i) to[(r0 + i * STEP) * LK + c] = to_f(x[i]);
  };
  for (int j0 = 0; j0 < end; j0 += KEYS) {
    uint64_t s2[PS_ROWS][J] = {};
#pragma unroll 1
    for (int part = 0; part < PARTS; ++part) {
      __syncthreads();
      stage(sk, k, a.ldk, j0, part);
      if (PARTS == 1) stage(sv, v, a.ldv, j0, 0);
      __syncthreads();
      const float *x0 = sq + ty * PS_ROWS * LD + part * COLS;
      const int limit = min(COLS, depth - part * COLS);
#pragma unroll 2
      for (int d = 0; d < limit; d += 4) {
        ulonglong2 y[J];
#pragma unroll
        for (int j = 0; j < J; ++j) y[j] = *reinterpret_cast<const ulonglong2 *>(sk + (tx + j * 16) * LK + d);
#pragma unroll
        for (int i = 0; i < PS_ROWS; ++i) {
          const ulonglong2 x = *reinterpret_cast<const ulonglong2 *>(x0 + i * LD + d);
#pragma unroll
          for (int j = 0; j < J; ++j) s2[i][j] = fma2(x.y, y[j].y, fma2(x.x, y[j].x, s2[i][j]));
        }
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
#pragma unroll
    for (int part = 0; part < PARTS; ++part) {
      if (PARTS > 1) {
        if (part * COLS >= a.D) break;
        __syncthreads();
        stage(sv, v, a.ldv, j0, part);
        __syncthreads();
      }
      auto row = [&](int c, ulonglong2(&y)[COLS / 64]) {
#pragma unroll
        for (int n = 0; n < COLS / 64; ++n) y[n] = *reinterpret_cast<const ulonglong2 *>(sv + c * LK + n * 64 + tx * 4);
      };
      auto add = [&](int i, float p, const ulonglong2(&y)[COLS / 64]) {
        const uint64_t p2 = pack2(p, p);
#pragma unroll
        for (int n = 0; n < COLS / 64; ++n) {
          uint64_t *to = o[i] + 2 * (part * (COLS / 64) + n);
          to[0] = fma2(p2, y[n].x, to[0]);
          to[1] = fma2(p2, y[n].y, to[1]);
        }
      };
      const int own = w.q0 + ty * PS_ROWS - j0;  // the key that the thread's first row sees last
      ulonglong2 y[COLS / 64];
      if (own >= KEYS - 1) {
#pragma unroll 1
        for (int c = 0; c < KEYS; c += 4) {
          float p[PS_ROWS][4];
#pragma unroll
          for (int i = 0; i < PS_ROWS; ++i) *reinterpret_cast<float4 *>(p[i]) = *reinterpret_cast<const float4 *>(sp + (ty * PS_ROWS + i) * LP + c);
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            row(c + e, y);
#pragma unroll
            for (int i = 0; i < PS_ROWS; ++i) add(i, p[i][e], y);
          }
        }
      } else {  // a key that a row does not see weighs nothing, whatever its value is
#pragma unroll 1
        for (int c = 0; c < min(KEYS, own + PS_ROWS); ++c) {
          row(c, y);
#pragma unroll
          for (int i = 0; i < PS_ROWS; ++i)
            if (c <= own + i) add(i, sp[(ty * PS_ROWS + i) * LP + c], y);
        }
      }
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
  constexpr int smem = (PS_Q * (DP + 4) + (DP > 128 ? 1 : 2) * PS_KEYS * ((DP < 128 ? DP : 128) + 4) + PS_Q * (PS_KEYS + 4)) * 4;
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
