// Causal attention over packed prompts on the 5th-generation tensor cores (bf16, fp16).
//
// Persistent blocks, one per multiprocessor, walk items of 256 queries of one head: two tiles of 128 that share the key and value
// tiles they pass, so that one tile's softmax runs while the tensor cores work for the other. Roles:
//   warps 0-3, 4-7  softmax and results of a query tile each, a thread per row: S (TMEM, fp32) -> weights in the inputs' type, over S
//   warp 8          one thread loads: Q tiles, and K and V tiles of 128 keys into a ring, by TMA
//   warp 9          one thread issues the products: S = Q K^T, O (TMEM) += P V
//   warps 10, 11    look through the value tiles that hold keys some row does not see (the last one or two of an item)
// With one score tile per query tile in TMEM (S 2 x 128 + O 2 x 128 columns are all there is) a tile's steps are a chain: QK, softmax, PV;
// the two tiles' chains interleave.
//
// O is only rescaled when a row's maximum grows by more than 2^8 (the division by the sum makes up for the rest), by the softmax
// threads themselves: the barrier that says S is there also says that the product before it is complete.
//
// What a row does not see must not reach it: scores are masked by comparison, but a weight of 0 times an infinity would be NaN. So
// entries of those value tiles that are not finite are set to 0 before the products, and joined again at the end for the rows that
// see them.
#include "pairs.cuh"
#include "serving_packed.cuh"
#include "tcgen05.cuh"
#include "tensor_map.cuh"

namespace djv {

constexpr int PT_THREADS = 384, PT_M = 128, PT_N = 128, PT_Q = 2 * PT_M;  // rows of a query tile, of a key tile, of an item
constexpr int PT_LOADER = 8, PT_ISSUER = 9, PT_SCAN = 10;

__device__ unsigned g_packed_timeouts;  // bounded waits that ran out (never, in a healthy run)

// a box of 64 elements x 1 head x 128 rows
__device__ __forceinline__ void tma_load_rows(uint32_t dst, const CUtensorMap *map, int d, int head, int row, uint64_t *bar) {
  asm volatile(
      "cp.async.bulk.tensor.3d.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3, %4}], [%5];" ::"r"(dst), "l"(map),
      "r"(d), "r"(head), "r"(row), "r"(smem_u32(bar))
      : "memory");
}

template <typename T>
__device__ __forceinline__ uint32_t pack_pair(float lo, float hi);
template <>
__device__ __forceinline__ uint32_t pack_pair<bf16>(float lo, float hi) { return pack_bf16(lo, hi); }
template <>
__device__ __forceinline__ uint32_t pack_pair<__half>(float lo, float hi) {
  __half2 h = __floats2half2_rn(lo, hi);
  return *reinterpret_cast<uint32_t *>(&h);
}

// the bits of a 16-bit pair's exponents, and of the lowest of them
template <typename T>
struct Exponent;
template <>
struct Exponent<bf16> {
  static constexpr uint32_t MASK = 0x7f807f80u, ONE = 0x00800080u;
};
template <>
struct Exponent<__half> {
  static constexpr uint32_t MASK = 0x7c007c00u, ONE = 0x04000400u;
};

template <typename T, int KB, int STAGES>  // KB: blocks of 64 elements in a row
__global__ void __launch_bounds__(PT_THREADS, 1)
packed_tc_kernel(const __grid_constant__ CUtensorMap map_q, const __grid_constant__ CUtensorMap map_k,
                 const __grid_constant__ CUtensorMap map_v, PackedArgs a, int tiles) {
  extern __shared__ unsigned char smem_raw[];
  __shared__ __align__(8) uint64_t q_full[2], q_empty[2], full[STAGES], empty[STAGES], s_full[2], p_full[2], o_full[2],
      clean[STAGES], taken[2][2], drained;
  __shared__ uint32_t tmem_slot;
  __shared__ int odd[2][2][2];  // by the item's parity: what each of the two warps found in each of the two value tiles
  constexpr uint32_t TILE = KB * PT_N * 128;
  const int tid = threadIdx.x, warp = tid / WARP, lane = tid % WARP;
  unsigned char *base = reinterpret_cast<unsigned char *>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~(uintptr_t)1023);
  const uint32_t q_sm = smem_u32(base), ring = q_sm + 2 * TILE;
  if (tid == 0) {
    for (int t = 0; t < 2; ++t) {
      mbar_init(&q_full[t], 1);
      mbar_init(&q_empty[t], 1);
      mbar_init(&s_full[t], 1);
      mbar_init(&p_full[t], PT_M);
      mbar_init(&o_full[t], 1);
      mbar_init(&taken[0][t], 4);
      mbar_init(&taken[1][t], 4);
    }
    for (int s = 0; s < STAGES; ++s) {
      mbar_init(&full[s], 1);
      mbar_init(&empty[s], 3);  // the products that read it, and the two warps that look through it
      mbar_init(&clean[s], 2 * WARP);
    }
    mbar_init(&drained, 1);
    mbar_fence_init();
  }
  if (warp == PT_ISSUER) tmem_alloc(&tmem_slot, 512);
  pdl_prologue();
  tmem_fence_before();
  __syncthreads();
  tmem_fence_after();
  const uint32_t tm = tmem_slot;
  const int items = tiles * a.H;
  // Items in the order of falling work (later queries see more keys), dealt out back and forth
  auto item_of = [&](int round) {
    const int i = round * (int)gridDim.x + ((round & 1) ? (int)gridDim.x - 1 - (int)blockIdx.x : (int)blockIdx.x);
    return i < items ? i : -1;
  };
  auto tile_of = [&](int item) { return packed_tile<PT_Q>(a, tiles - 1 - item / a.H); };  // whole warp
  const int rounds = (items + (int)gridDim.x - 1) / (int)gridDim.x;
  bool dead = false;  // a wait ran out: wait no more, finish and report

  if (warp < 8) {
    asm volatile("setmaxnreg.inc.sync.aligned.u32 208;");
    const int t = warp / 4, r = tid % PT_M;
    const uint32_t lane_base = (uint32_t)(warp % 4 * 32) << 16, tm_s = tm + t * PT_N + lane_base, tm_o = tm + 2 * PT_N + t * (KB * 64) + lane_base;
    const float c = a.scale * 1.4426950408889634f, ca = c == 0.f ? 1e-30f : fabsf(c);  // scores in units of log 2
    const uint64_t ca2 = pack2(ca, ca);
    int steps = 0, done = 0;  // phases of s_full and o_full
    int parity = 0;
    for (int round = 0; round < rounds; ++round) {
      const int item = item_of(round);
      if (item < 0) break;
      const PackedTile w = tile_of(item);
      const int h = item % a.H, rows = w.rows - t * PT_M;  // of this query tile
      if (w.rows <= 0) continue;
      T *out = static_cast<T *>(a.out) + ((long long)(w.first + w.q0 + t * PT_M + r) * a.H + h) * a.D;
      if (w.rest) {
        if (!a.keep_rest && r < rows)
          for (int d = 0; d < a.D; d += 8) *reinterpret_cast<uint4 *>(out + d) = make_uint4(0, 0, 0, 0);
        continue;
      }
      parity ^= 1;
      if (rows <= 0) continue;
      const int last = w.q0 / PT_N + t;  // the key tile of the row's own key
      float m = 0.f, l = 0.f;
      for (int j = 0; j <= last; ++j, ++steps) {
        if (!dead) dead = !mbar_wait(&s_full[t], steps & 1);
        __syncwarp();
        tmem_fence_after();
        uint32_t s[4][32];
#pragma unroll
        for (int q = 0; q < 4; ++q) tmem_ld32(s[q], tm_s + q * 32);
        tmem_wait_ld();
        if (c < 0.f) {
#pragma unroll
          for (int q = 0; q < 4; ++q)
#pragma unroll
            for (int e = 0; e < 32; ++e) s[q][e] ^= 0x80000000u;
        }
        if (j == last) {  // keys behind the row's own
#pragma unroll
          for (int q = 0; q < 4; ++q)
#pragma unroll
            for (int e = 0; e < 32; ++e)
              if (q * 32 + e > r) s[q][e] = 0xff800000u;
        }
        float mm[4] = {-INFINITY, -INFINITY, -INFINITY, -INFINITY};
#pragma unroll
        for (int q = 0; q < 4; ++q)
#pragma unroll
          for (int e = 0; e < 32; ++e) mm[e % 4] = fmaxf(mm[e % 4], __uint_as_float(s[q][e]));
        const float mx = fmaxf(fmaxf(mm[0], mm[1]), fmaxf(mm[2], mm[3])) * ca;
        if (j == 0) {
          m = mx == -INFINITY ? 0.f : mx;
        } else {
          const bool grow = mx > m + 8.f;
          if (__any_sync(0xffffffffu, grow)) {
            const float corr = grow ? exp2_approx(m - mx) : 1.f;
            if (grow) m = mx;
            l *= corr;
#pragma unroll
            for (int q = 0; q < KB * 64; q += 16) {
              uint32_t o[16];
              tmem_ld16(o, tm_o + q);
              tmem_wait_ld();
#pragma unroll
              for (int e = 0; e < 16; ++e) o[e] = __float_as_uint(__uint_as_float(o[e]) * corr);
              tmem_st16(tm_o + q, o);
            }
          }
        }
        const uint64_t nm2 = pack2(-m, -m);
        uint64_t l2[2] = {0, 0};
#pragma unroll
        for (int q = 0; q < 4; ++q) {
          uint32_t p[16];
#pragma unroll
          for (int e = 0; e < 16; ++e) {
            float x, y;
            unpack2(fma2(pack2(__uint_as_float(s[q][2 * e]), __uint_as_float(s[q][2 * e + 1])), ca2, nm2), x, y);
            x = exp2_approx(x);
            y = exp2_approx(y);
            l2[e % 2] = add2(l2[e % 2], pack2(x, y));
            p[e] = pack_pair<T>(x, y);
          }
          tmem_st16(tm_s + q * 16, p);
        }
        float x, y;
        unpack2(add2(l2[0], l2[1]), x, y);
        l += x + y;
        tmem_wait_st();
        tmem_fence_before();
        mbar_arrive(&p_full[t]);
      }
      if (!dead) dead = !mbar_wait(&o_full[t], done & 1);
      ++done;
      __syncwarp();
      tmem_fence_after();
      const float inv = l == 0.f ? 0.f : 1.f / l;
      const bool odd0 = (odd[parity][0][0] | odd[parity][0][1]) != 0, odd1 = (odd[parity][1][0] | odd[parity][1][1]) != 0;
      __syncwarp();
      if (lane == 0) mbar_arrive(&taken[parity][t]);
#pragma unroll 1
      for (int q = 0; q < a.D; q += 16) {
        uint32_t o[16];
        tmem_ld16(o, tm_o + q);
        tmem_wait_ld();
        float f[16];
#pragma unroll
        for (int e = 0; e < 16; ++e) f[e] = __uint_as_float(o[e]) * inv;
        if ((odd0 || odd1) && r < rows) {  // values that are not finite, for who sees them
          const int i = w.q0 + t * PT_M + r, g = h / (a.H / a.G);
          for (int d2 = 0; d2 < 2; ++d2) {
            if (!(d2 ? odd1 : odd0)) continue;
            const int j0 = w.q0 + d2 * PT_N;
            for (int j = j0; j <= min(i, j0 + PT_N - 1); ++j) {
              const T *v = static_cast<const T *>(a.v) + (long long)(w.first + j) * a.ldv + g * a.hv;
#pragma unroll
              for (int e = 0; e < 16; ++e) {
                const float x = q + e < a.D ? to_f(v[q + e]) : 0.f;
                if (!(fabsf(x) <= 3.402823466e38f)) f[e] += x;
              }
            }
          }
        }
        if (r < rows) {
#pragma unroll
          for (int e = 0; e < 16; e += 8)
            if (q + e < a.D)
              *reinterpret_cast<uint4 *>(out + q + e) = make_uint4(pack_pair<T>(f[e], f[e + 1]), pack_pair<T>(f[e + 2], f[e + 3]),
                                                                   pack_pair<T>(f[e + 4], f[e + 5]), pack_pair<T>(f[e + 6], f[e + 7]));
        }
        __syncwarp();
      }
      tmem_fence_before();  // (the next item's first product into O waits for this thread's next weights)
    }
  } else {
    asm volatile("setmaxnreg.dec.sync.aligned.u32 88;");
    int slot = 0;              // ring slots passed so far; slot n is stage n % STAGES in its n / STAGES-th use
    int used[2] = {0, 0};      // items that used query tile 0, 1
    unsigned looked = 0;       // phases of clean, a bit each
    int parity = 0, seen[2][2] = {};  // phases of taken
    int stepped[2] = {0, 0};   // phases of p_full
    for (int round = 0; round < rounds && !dead; ++round) {
      const int item = item_of(round);
      if (item < 0) break;
      const PackedTile w = tile_of(item);
      if (w.rows <= 0 || w.rest) continue;
      const int h = item % a.H, g = h / (a.H / a.G), d0 = w.q0 / PT_N;
      const bool both = w.rows > PT_M;
      const int n = d0 + (both ? 2 : 1);  // key tiles
      parity ^= 1;
      if (warp == PT_LOADER) {
        if (lane == 0) {
          auto load = [&](const CUtensorMap *map, int head, int row) {
            const int s = slot % STAGES;
            if (slot >= STAGES && !dead) dead = !mbar_wait(&empty[s], (slot / STAGES - 1) & 1);
            if (dead) return;
            mbar_arrive_expect_tx(&full[s], TILE);
            for (int b = 0; b < KB; ++b) tma_load_rows(ring + s * TILE + b * PT_N * 128, map, b * 64, head, row, &full[s]);
            ++slot;
          };
          for (int t = 0; t < (both ? 2 : 1); ++t) {
            if (used[t] && !dead) dead = !mbar_wait(&q_empty[t], (used[t] - 1) & 1);
            if (dead) break;
            ++used[t];
            mbar_arrive_expect_tx(&q_full[t], TILE);
            for (int b = 0; b < KB; ++b)
              tma_load_rows(q_sm + t * TILE + b * PT_M * 128, &map_q, b * 64, h, w.first + w.q0 + t * PT_M, &q_full[t]);
            if (t == 0) load(&map_k, g, w.first);
          }
          for (int j = 0; j < n && !dead; ++j) {
            if (j) load(&map_k, g, w.first + j * PT_N);
            load(&map_v, g, w.first + j * PT_N);
          }
        }
        dead = __shfl_sync(0xffffffffu, (int)dead, 0) != 0;
      } else if (warp == PT_ISSUER) {
        if (lane == 0) {
          constexpr bool FP16 = sizeof(T) == 2 && !__is_same(T, bf16);
          const uint32_t idesc_s = mma_idesc(PT_M, PT_N, false, false, FP16), idesc_o = mma_idesc(PT_M, (a.D + 15) / 16 * 16, false, true, FP16);
          const int k_steps = (a.D + 15) / 16;
          auto wait = [&](uint64_t *bar, int phase) {
            if (!dead) dead = !mbar_wait(bar, phase & 1);
            tmem_fence_after();
          };
          auto scores = [&](int t, int at) {
            const uint64_t q = desc_k_major(q_sm + t * TILE, PT_M, 0), k = desc_k_major(ring + at % STAGES * TILE, PT_N, 0);
#pragma unroll
            for (int x = 0; x < KB * 4; ++x) {
              const uint32_t step = (x / 4) * (PT_N * 128 / 16) + (x % 4) * 2;  // descriptor units of 16 bytes
              if (x < k_steps) mma_ss(tm + t * PT_N, q + step, k + step, idesc_s, x > 0);
            }
            mma_commit(&s_full[t]);
          };
          // slots of this item: K0, V0, K1, V1, ...
          const int first = slot;
          wait(&full[first % STAGES], first / STAGES);
          for (int t = 0; t < (both ? 2 : 1); ++t) {
            wait(&q_full[t], used[t]);
            ++used[t];
            scores(t, first);
          }
          mma_commit(&empty[first % STAGES]);
          for (int j = 0; j < n; ++j) {
            const int vs = first + 2 * j + 1, ks = vs + 1;
            wait(&full[vs % STAGES], vs / STAGES);
            if (j >= d0) {
              wait(&clean[vs % STAGES], looked >> (vs % STAGES));
              looked ^= 1u << (vs % STAGES);
            }
            bool more = false;
            for (int t = 0; t < (both ? 2 : 1); ++t) {
              const int last = d0 + t;
              if (j > last) continue;
              wait(&p_full[t], stepped[t]);
              ++stepped[t];
              const uint64_t v = desc_mn_major(ring + vs % STAGES * TILE, PT_N, 0);
#pragma unroll
              for (int x = 0; x < PT_N / 16; ++x)
                mma_ts(tm + 2 * PT_N + t * (KB * 64), tm + t * PT_N + x * 8, v + (uint64_t)(x * 128), idesc_o, j > 0 || x > 0);
              if (j == last) {
                mma_commit(&o_full[t]);
                continue;
              }
              if (!more) wait(&full[ks % STAGES], ks / STAGES);
              more = true;
              scores(t, ks);
              if (j + 1 == last) mma_commit(&q_empty[t]);
            }
            mma_commit(&empty[vs % STAGES]);
            if (more) mma_commit(&empty[ks % STAGES]);
          }
          if (d0 == 0) mma_commit(&q_empty[0]);  // (a tile with one key tile)
          slot += 2 * n;
        }
        dead = __shfl_sync(0xffffffffu, (int)dead, 0) != 0;
      } else {
        const int me = tid - PT_SCAN * WARP, mine = warp - PT_SCAN;
        for (int t = 0; t < 2; ++t) {  // what was found in the item before the last has been read
          if (seen[parity][t] && !dead) dead = !mbar_wait(&taken[parity][t], (seen[parity][t] - 1) & 1);
          if (t == 0 || both) ++seen[parity][t];
        }
        dead = __any_sync(0xffffffffu, dead);
        if (lane == 0) odd[parity][1][mine] = 0;
        for (int x = 0; x < 2 * n; ++x) {
          const int vs = slot + x, j = x / 2;
          if (!dead) dead = !mbar_wait(&full[vs % STAGES], (vs / STAGES) & 1);
          dead = __any_sync(0xffffffffu, dead);
          if (x % 2 == 0 || j < d0) {
            if (lane == 0) mbar_arrive(&empty[vs % STAGES]);
            continue;
          }
          uint4 *v = reinterpret_cast<uint4 *>(base + 2 * TILE + vs % STAGES * TILE);
          bool any = false;
          for (int i = me; i < (int)(TILE / 16); i += 2 * WARP) {
            uint4 x = v[i];
            uint32_t *e = reinterpret_cast<uint32_t *>(&x);
            bool here = false;
#pragma unroll
            for (int y = 0; y < 4; ++y) {
              const uint32_t top = ((e[y] & Exponent<T>::MASK) + Exponent<T>::ONE) & 0x80008000u;
              here |= top != 0;
              if (top & 0x8000u) e[y] &= 0xffff0000u;
              if (top & 0x80000000u) e[y] &= 0x0000ffffu;
            }
            if (here) v[i] = x;
            any |= here;
          }
          any = __any_sync(0xffffffffu, any);
          if (lane == 0) odd[parity][j - d0][mine] = any;
          fence_proxy_async_smem();
          mbar_arrive(&clean[vs % STAGES]);
          if (lane == 0) mbar_arrive(&empty[vs % STAGES]);
        }
        slot += 2 * n;
      }
    }
    if (warp == PT_LOADER && lane == 0) {  // copies that nobody waited for still land
      for (int s = slot < STAGES ? 0 : slot - STAGES; s < slot; ++s) mbar_wait(&full[s % STAGES], (s / STAGES) & 1);
      for (int t = 0; t < 2; ++t)
        if (used[t]) mbar_wait(&q_full[t], (used[t] - 1) & 1);
    }
    if (warp == PT_ISSUER && lane == 0 && dead) {
      mma_commit(&drained);
      mbar_wait(&drained, 0);
    }
  }
  if (dead && lane == 0) atomicAdd(&g_packed_timeouts, 1u);
  __syncwarp();
  tmem_fence_before();
  __syncthreads();
  if (warp == PT_ISSUER) {
    tmem_fence_after();
    tmem_dealloc(tm, 512);
  }
}

// rows of heads of D elements: boxes of 64 elements x 1 head x 128 rows with the 128-byte swizzle, zeros outside
static bool rows_map(CUtensorMap *map, bool fp16, const void *p, long long ld, long long hs, int T, int heads, int D) {
  const cuuint64_t dims[3] = {(cuuint64_t)D, (cuuint64_t)heads, (cuuint64_t)T},
                   strides[2] = {(cuuint64_t)(heads > 1 ? hs : ld) * 2, (cuuint64_t)ld * 2};
  const cuuint32_t box[3] = {64, 1, PT_M}, unit[3] = {1, 1, 1};
  return encode_tiled()(map, fp16 ? CU_TENSOR_MAP_DATA_TYPE_FLOAT16 : CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, 3, const_cast<void *>(p), dims,
                        strides, box, unit, CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
                        CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}

// Whether TMA can read the rows: strides are positive multiples of 16 bytes.
static bool rows_fit(const void *p, long long ld, long long hs, int heads) {
  return aligned16(p) && ld > 0 && ld % 8 == 0 && ld < (1ll << 36) && (heads == 1 || (hs > 0 && hs % 8 == 0 && hs < (1ll << 36)));
}
bool packed_tc_supported(int dtype, const PackedArgs &a) {
  return dtype != DJV_DTYPE_F32 && a.D % 8 == 0 && a.D <= 128 && rows_fit(a.q, a.ldq, a.hq, a.H) && rows_fit(a.k, a.ldk, a.hk, a.G) &&
         rows_fit(a.v, a.ldv, a.hv, a.G) && aligned16(a.out) && (long long)packed_tiles<PT_Q>(a.T, a.B) * a.H < (1ll << 30) && encode_tiled();
}

template <typename T, int KB>
static int launch_packed_tc(const PackedArgs &a, cudaStream_t st) {
  constexpr int STAGES = KB == 1 ? 8 : 4, smem = 1024 + (2 + STAGES) * KB * PT_N * 128;
  constexpr bool FP16 = !__is_same(T, bf16);
  CUtensorMap q, k, v;
  if (!rows_map(&q, FP16, a.q, a.ldq, a.hq, a.T, a.H, a.D) || !rows_map(&k, FP16, a.k, a.ldk, a.hk, a.T, a.G, a.D) ||
      !rows_map(&v, FP16, a.v, a.ldv, a.hv, a.T, a.G, a.D)) {
    set_error("packed_attention: a tensor map was refused");
    return DJV_ERR_CUDA;
  }
  static DevicePrep prep;
  const int(*unused)[4];
  cudaError_t e = prep.get(
      [&](int(&)[4]) { return cudaFuncSetAttribute(packed_tc_kernel<T, KB, STAGES>, cudaFuncAttributeMaxDynamicSharedMemorySize, smem); },
      unused);
  const int tiles = packed_tiles<PT_Q>(a.T, a.B), items = tiles * a.H, grid = items < sm_count() ? items : sm_count();
  if (e == cudaSuccess)
    e = djv::launch_kernel(packed_tc_kernel<T, KB, STAGES>, dim3(grid), dim3(PT_THREADS), smem, st, q, k, v, a, tiles);
  if (e != cudaSuccess) {
    cudaGetLastError();
    set_error("packed_attention: CUDA error %d (%s)", (int)e, cudaGetErrorString(e));
    return DJV_ERR_CUDA;
  }
  count_launch();
  return check_launch("packed_attention");
}

int packed_tc(int dtype, const PackedArgs &a, cudaStream_t st) {
  if (dtype == DJV_DTYPE_F16) return a.D <= 64 ? launch_packed_tc<__half, 1>(a, st) : launch_packed_tc<__half, 2>(a, st);
  return a.D <= 64 ? launch_packed_tc<bf16, 1>(a, st) : launch_packed_tc<bf16, 2>(a, st);
}

unsigned packed_timeouts() {
  unsigned v = 0;
  if (cudaMemcpyFromSymbol(&v, g_packed_timeouts, sizeof(v)) != cudaSuccess) {
    cudaGetLastError();
    return 0;
  }
  return v;
}

}  // namespace djv
