// Causal attention over packed prompts on the 5th-generation tensor cores (bf16, fp16).
//
// Persistent blocks, one per multiprocessor, walk items of 256 queries of one head: two tiles of 128 that share the key and value
// tiles they pass, so that one tile's softmax runs while the tensor cores work for the other. Roles:
//   warps 0-3, 4-7  softmax and results of a query tile each, a thread per row: S (TMEM, fp32) -> weights in the inputs' type, over S
//   warp 8          one thread loads: Q tiles, and K and V tiles of 128 keys into a ring, by TMA
//   warp 9          issues the products: S = Q K^T, O (TMEM) += P V
//   warps 10, 11    look through the value tiles that hold keys some row does not see (the last one or two of an item)
// With one score tile per query tile in TMEM (S 2 x 128 + O 2 x 128 columns are all there is) a tile's steps are a chain: QK, softmax, PV;
// the two tiles' chains interleave. Heads of more than 128 have one query tile (O takes 256 columns, Q 64 KB) and tiles of 64 keys, four of
// which fit beside it: nothing runs behind the chain.
//
// O is only rescaled when a row's maximum grows by more than 2^8 (the division by the sum makes up for the rest), by the softmax
// threads themselves: the barrier that says S is there also says that the product before it is complete. fp16 ends at 2^-24 and goes up to
// 2^16, so its weights, up to 2^8, are made 2^7 times as large, and so are their sums: from 2^-21 of the largest on they have all their
// bits, below that they are off by 2^-32 of the largest at most.
//
// Few items go out in the order of falling work, many from the last sequence's last one on, back and forth over the blocks; sequences
// may have any lengths.
//
// The weights enter the second product as one term, rounded by half a step at most (2^-8 of a bf16 weight, 2^-11 of an fp16 one),
// as the results are: off from 64 bits by 2.0e-3 (bf16) and 2.5e-4 (fp16) in all, where rounding the results alone makes 1.6e-3 and 2.0e-4.
// A second term for what they lack would make the products with V twice as many: 16001 tokens 1.93 -> 3.31 ms, 24 prompts 0.33 -> 0.53.
//
// Measured (32 heads over 8, 128 dimensions, bf16): 16001 tokens 1.71 ms, 1.23 PFLOP/s, and 1.93 ms when the power cap has the clocks at
// 1.61 GHz; 24 prompts of 16384 tokens in all 0.32 ms, 0.69 PFLOP/s. A step of an item takes about 3000 cycles, the exponentials of its two
// tiles 2048 of the special units and its products 2048 of the tensor cores. What did not pay: two threads per row, exponentials by
// polynomials, turns between the tiles, values' products that begin with half the weights, waits that spin.
// 16 heads over 8 of 256 dimensions: 4096 tokens 0.19 ms, 0.74 PFLOP/s (5.5 on the CUDA cores), 16384 tokens 2.6 ms, 0.85 PFLOP/s.
//
// What a row does not see must not reach it: scores are masked by comparison, but a weight of 0 times an infinity would be NaN. So
// entries of those value tiles that are not finite are set to 0 before the products, and joined again at the end for the rows that
// see them. In the tiles that all rows see the products take them as they are; where a weight (or what O is rescaled by) has been rounded
// to 0 that is NaN too, and a warp whose results are not finite, though the sum of the weights is, goes through the values once more (looking at
// each 16 columns as they are stored took 2 % more; at the end of them it takes nothing).
#include "pairs.cuh"
#include "serving_packed.cuh"
#include "tcgen05.cuh"
#include "tensor_map.cuh"

namespace djv {

constexpr int PT_THREADS = 384, PT_M = 128;  // rows of a query tile
constexpr int PT_SOFT = 8, PT_LOADER = 8, PT_ISSUER = 9, PT_SCAN = 10;  // softmax warps, and the others
constexpr int PT_TABLE = 1024;  // items per head that are put in order
constexpr int PT_ROUNDS = 256;  // items of a block that are looked up at a time

// Products and commits by one thread of a warp that runs as one: what they are given stays in uniform registers (from one thread's own
// branch every operand of every product would have to be moved there, 60 to 130 cycles for each).
__device__ __forceinline__ void warp_mma_ss(uint32_t d, uint64_t a, uint64_t b, uint32_t idesc, uint32_t accumulate) {
  asm volatile(
      "{\n"
      ".reg .pred p, e;\n"
      "elect.sync _|e, 0xffffffff;\n"
      "setp.ne.b32 p, %4, 0;\n"
      "@e tcgen05.mma.cta_group::1.kind::f16 [%0], %1, %2, %3, p;\n"
      "}\n" ::"r"(d),
      "l"(a), "l"(b), "r"(idesc), "r"(accumulate)
      : "memory");
}
__device__ __forceinline__ void warp_mma_ts(uint32_t d, uint32_t a, uint64_t b, uint32_t idesc, uint32_t accumulate) {
  asm volatile(
      "{\n"
      ".reg .pred p, e;\n"
      "elect.sync _|e, 0xffffffff;\n"
      "setp.ne.b32 p, %4, 0;\n"
      "@e tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], %2, %3, p;\n"
      "}\n" ::"r"(d),
      "r"(a), "l"(b), "r"(idesc), "r"(accumulate)
      : "memory");
}
__device__ __forceinline__ void warp_commit(uint64_t *bar) {
  asm volatile(
      "{\n"
      ".reg .pred e;\n"
      "elect.sync _|e, 0xffffffff;\n"
      "@e tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [%0];\n"
      "}\n" ::"r"(smem_u32(bar))
      : "memory");
}
__device__ __forceinline__ float max3(float a, float b, float c) {
  float d;
  asm("max.f32 %0, %1, %2, %3;" : "=f"(d) : "f"(a), "f"(b), "f"(c));
  return d;
}

__device__ unsigned g_packed_timeouts;  // bounded waits that ran out (never, in a healthy run)

// a box of 64 elements x 1 head x the map's rows
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

// KB: blocks of 64 elements in a row; FULL: all of them are in use, and results start on 32 bytes; NT: query tiles of an item; KN: keys of a tile
template <typename T, int KB, bool FULL, int NT, int KN, int STAGES>
__global__ void __launch_bounds__(PT_THREADS, 1)
packed_tc_kernel(const __grid_constant__ CUtensorMap map_q, const __grid_constant__ CUtensorMap map_k,
                 const __grid_constant__ CUtensorMap map_v, PackedArgs a, int most) {
  extern __shared__ unsigned char smem_raw[];
  __shared__ __align__(8) uint64_t q_full[2], q_empty[2], full[STAGES], empty[STAGES], s_full[2], p_full[2], o_full[2],
      clean[STAGES], taken[2][2], drained;
  __shared__ uint32_t tmem_slot;
  __shared__ int2 table[PT_TABLE];    // sequence and item in it, by falling work
  __shared__ int4 mine[PT_ROUNDS];    // the block's items: the sequence's first row, first query in it, queries, head
  __shared__ int odd[2][2][2];  // by the item's parity: what each of the two warps found in each of the two value tiles
  constexpr uint32_t Q_TILE = KB * PT_M * 128, TILE = KB * KN * 128, O_AT = NT * KN;  // bytes; columns of TMEM in front of O
  constexpr float LIFT = __is_same(T, bf16) ? 0.f : 7.f;  // weights and sums are 2^LIFT times what they stand for
  constexpr int PT_Q = NT * PT_M;
  const int tid = threadIdx.x, warp = tid / WARP, lane = tid % WARP;
  unsigned char *base = reinterpret_cast<unsigned char *>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~(uintptr_t)1023);
  const uint32_t q_sm = smem_u32(base), ring = q_sm + NT * Q_TILE;
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
  // How many items there are, and if they are few their order: by falling number in the sequence, which is what they take.
  // (Offsets that do not ascend can make more than `most`, which is all that offsets that do can make: the rest is left out.)
  const int total = packed_total<PT_Q>(a, 0, a.B), tiles = total < 0 || total > most ? most : total;
  // Every block makes the order for itself, in tiles * B steps or so, and what it evens out grows less with more sequences. 32 heads of 128, in
  // order and not, by tiles * B: 444 128 and 136 us, 1848 241 and 250, 2592 222 and 256, 4608 550 and 570, 6528 200 and 192, 7344 483 and 472,
  // 18944 216 and 207.
  const bool ordered = tiles == total && tiles <= PT_TABLE && a.B <= 5 * 1024 && tiles * a.B <= 5 * 1024;
  if (ordered) {
    for (int i = warp; i < tiles; i += PT_THREADS / WARP) {
      const PackedTile w = packed_tile<PT_Q>(a, i);
      const int q = w.q0 / PT_Q;
      int before = 0;
      for (int b = lane; b < a.B; b += WARP) {
        const int lo = max(0, min(a.cu[b], a.T)), n = max(0, min(a.cu[b + 1], a.T) - lo), t = (n + PT_Q - 1) / PT_Q;
        before += max(0, t - q - 1) + (b < w.b && t > q);
      }
      before = __reduce_add_sync(0xffffffffu, before);
      if (lane == 0) table[before] = make_int2(w.b, q);
    }
  }
  // Else how many there are in front of every `segment` sequences, and they go out from the last sequence's last one.
  const int segment = ((a.B + PT_TABLE - 1) / PT_TABLE + WARP - 1) / WARP * WARP, segments = (a.B + segment - 1) / segment;
  if (!ordered) {
    for (int i = warp; i < segments; i += PT_THREADS / WARP) {
      const int n = packed_total<PT_Q>(a, i * segment, min(a.B, (i + 1) * segment));
      if (lane == 0) table[i].x = n;
    }
    __syncthreads();
    if (warp == 0) {
      int run = 0;
      for (int i0 = 0; i0 < segments; i0 += WARP) {
        const int n = i0 + lane < segments ? table[i0 + lane].x : 0;
        int sum = n;
#pragma unroll
        for (int o = 1; o < WARP; o <<= 1) {
          const int up = __shfl_up_sync(0xffffffffu, sum, o);
          if (lane >= o) sum += up;
        }
        if (i0 + lane < segments) table[i0 + lane].x = run + sum - n;
        run += __shfl_sync(0xffffffffu, sum, WARP - 1);
      }
    }
  }
  tmem_fence_before();
  __syncthreads();
  tmem_fence_after();
  const uint32_t tm = tmem_slot;
  const int items = tiles * a.H;
  // items are dealt out back and forth
  auto item_of = [&](int round) {
    const int i = round * (int)gridDim.x + ((round & 1) ? (int)gridDim.x - 1 - (int)blockIdx.x : (int)blockIdx.x);
    return i < items ? i : -1;
  };
  auto tile_of = [&](int item) {  // whole warp
    if (!ordered) {
      const int index = tiles - 1 - item / a.H;
      int lo = 0, hi = segments;  // the last segment that does not begin after it
      while (hi - lo > 1) {
        const int mid = (lo + hi) / 2;
        if (table[mid].x <= index) lo = mid;
        else hi = mid;
      }
      return packed_tile<PT_Q>(a, index, lo * segment, table[lo].x);
    }
    const int2 x = table[item / a.H];
    const int first = max(0, min(a.cu[x.x], a.T)), q0 = x.y * PT_Q;
    return PackedTile{first, q0, min(PT_Q, min(a.cu[x.x + 1], a.T) - first - q0), 0, x.x};
  };
  const int rounds = (items + (int)gridDim.x - 1) / (int)gridDim.x;
  // Looked up before the roles begin, and again after so many items: none of their loops has the search in it.
  auto look_up = [&](int base, int from, int step) {
    for (int i = from; i < PT_ROUNDS && base + i < rounds; i += step) {
      const int item = item_of(base + i);
      PackedTile w{0, 0, 0, 0, 0};
      if (item >= 0) w = tile_of(item);
      if (lane == 0) mine[i] = make_int4(w.first, w.q0, w.rows, item % a.H);
    }
  };
  look_up(0, warp, PT_THREADS / WARP);
  __syncthreads();
  auto meet = [] { asm volatile("barrier.cta.sync 1, %0;" ::"n"(PT_THREADS) : "memory"); };
  bool dead = false;  // a wait ran out: wait no more, finish and report

  if (warp < PT_SOFT) {
    asm volatile("setmaxnreg.inc.sync.aligned.u32 208;");
    const int t = warp / 4, r = tid % PT_M;
    const uint32_t lane_base = (uint32_t)(warp % 4 * 32) << 16;
    // the row's scores, over which it puts its weights, and its sums
    const uint32_t tm_s = tm + t * KN + lane_base, tm_o = tm + O_AT + t * (KB * 64) + lane_base;
    const float c = a.scale * 1.4426950408889634f, ca = c == 0.f ? 1e-30f : fabsf(c);  // scores in units of log 2
    const uint64_t ca2 = pack2(ca, ca);
    if (!a.keep_rest) {  // rows of no sequence
      const int head = max(0, min(a.cu[0], a.T)), tail = max(head, min(a.cu[a.B], a.T)), pieces = a.H * a.D / 8;
      for (int i = blockIdx.x; i < head + a.T - tail; i += gridDim.x) {
        uint4 *row = reinterpret_cast<uint4 *>(static_cast<T *>(a.out) + (long long)(i < head ? i : i - head + tail) * a.H * a.D);
        for (int d = tid; d < pieces; d += PT_SOFT * WARP) row[d] = make_uint4(0, 0, 0, 0);
      }
    }
    int steps = 0, done = 0;  // phases of s_full and o_full
    int parity = 0;
    for (int round = 0; round < rounds; ++round) {
      if (round > 0 && round % PT_ROUNDS == 0) {
        meet();
        meet();  // (between: the other warps look up the next ones)
      }
      const int4 w = mine[round % PT_ROUNDS];
      const int first = w.x, q0 = w.y, h = w.w, rows = w.z - t * PT_M;  // of this query tile
      if (w.z <= 0) continue;
      parity ^= 1;
      if (rows <= 0) continue;
      const int last = (q0 + min(w.z, (t + 1) * PT_M) - 1) / KN;  // the key tile of the tile's last key
      float m = 0.f, l = 0.f;
      for (int j = 0; j <= last; ++j, ++steps) {
        if (!dead) dead = !mbar_wait(&s_full[t], steps & 1);
        __syncwarp();
        tmem_fence_after();
        uint32_t s[KN / 32][32];
#pragma unroll
        for (int q = 0; q < KN / 32; ++q) tmem_ld32(s[q], tm_s + q * 32);
        tmem_wait_ld();
        if (c < 0.f) {
#pragma unroll
          for (int q = 0; q < KN / 32; ++q)
#pragma unroll
            for (int e = 0; e < 32; ++e) s[q][e] ^= 0x80000000u;
        }
        if ((j + 1) * KN > q0 + t * PT_M) {  // keys behind the row's own
          const int own = q0 + t * PT_M + r - j * KN;
#pragma unroll
          for (int q = 0; q < KN / 32; ++q)
#pragma unroll
            for (int e = 0; e < 32; ++e)
              if (q * 32 + e > own) s[q][e] = 0xff800000u;
        }
        float mm[4] = {-INFINITY, -INFINITY, -INFINITY, -INFINITY};
#pragma unroll
        for (int q = 0; q < KN / 32; ++q)
#pragma unroll
          for (int e = 0; e < 32; e += 2) mm[e / 2 % 4] = max3(mm[e / 2 % 4], __uint_as_float(s[q][e]), __uint_as_float(s[q][e + 1]));
        const float mx = fmaxf(max3(mm[0], mm[1], mm[2]), mm[3]) * ca;
        if (j == 0) {
          m = mx == -INFINITY ? -3e38f : mx;  // (a tile that weighs nothing: any later maximum is more)
        } else {
          const bool grow = mx > m + 8.f;
          if (__any_sync(0xffffffffu, grow)) {
            const float corr = grow ? exp2_approx(m - mx) : 1.f;
            if (grow) m = mx;
            l *= corr;
#pragma unroll 1
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
        const uint64_t nm2 = pack2(LIFT - m, LIFT - m);
        uint64_t l2[2] = {0, 0};
#pragma unroll
        for (int q = 0; q < KN / 32; ++q) {
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
      T *out = static_cast<T *>(a.out) + ((long long)(first + q0 + t * PT_M + r) * a.H + h) * a.D;
      float z = 0.f;  // or NaN: a result is not finite
      auto results = [&](int q, bool again) {
        uint32_t o[16];
        tmem_ld16(o, tm_o + q);
        tmem_wait_ld();
        float f[16];
#pragma unroll
        for (int e = 0; e < 16; ++e) f[e] = __uint_as_float(o[e]) * inv;
        if (!again) {
#pragma unroll
          for (int e = 0; e < 16; ++e) z = fmaf(f[e], 0.f, z);
        } else {  // values of whole tiles that are not finite
          float x[16] = {};
          const T *v = static_cast<const T *>(a.v) + (long long)first * a.ldv + h / (a.H / a.G) * a.hv + q;
#pragma unroll 4
          for (int j = lane; j < q0; j += WARP)
#pragma unroll
            for (int e = 0; e < 16; e += 8) {
              if (q + e >= a.D) continue;
              float y[8];
              unpack_chunk<T>(*reinterpret_cast<const uint4 *>(v + j * a.ldv + e), y);
#pragma unroll
              for (int i = 0; i < 8; ++i)
                if (!(fabsf(y[i]) < INFINITY)) x[e + i] += y[i];
            }
#pragma unroll
          for (int e = 0; e < 16; ++e) {
#pragma unroll
            for (int d = 16; d > 0; d >>= 1) x[e] += __shfl_xor_sync(0xffffffffu, x[e], d);
            if (f[e] != f[e] && x[e] != 0.f) f[e] = x[e];
          }
        }
        if ((odd0 || odd1) && r < rows) {  // values that are not finite, for who sees them
          const int i = q0 + t * PT_M + r, g = h / (a.H / a.G);
          for (int d2 = 0; d2 < 2; ++d2) {
            if (!(d2 ? odd1 : odd0)) continue;
            const int j0 = (q0 / KN + d2) * KN;
            for (int j = j0; j <= min(i, j0 + KN - 1); ++j) {
              const T *v = static_cast<const T *>(a.v) + (long long)(first + j) * a.ldv + g * a.hv;
#pragma unroll
              for (int e = 0; e < 16; ++e) {
                const float x = q + e < a.D ? to_f(v[q + e]) : 0.f;
                if (!(fabsf(x) <= 3.402823466e38f)) f[e] += x;
              }
            }
          }
        }
        if (r < rows) {
          uint32_t p[8];
#pragma unroll
          for (int e = 0; e < 8; ++e) p[e] = pack_pair<T>(f[2 * e], f[2 * e + 1]);
          if (FULL) {  // a sector in one: every lane writes to a line of its own
            asm volatile("st.global.v8.b32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8};" ::"l"(out + q), "r"(p[0]), "r"(p[1]), "r"(p[2]), "r"(p[3]),
                         "r"(p[4]), "r"(p[5]), "r"(p[6]), "r"(p[7])
                         : "memory");
          } else {
            if (q < a.D) *reinterpret_cast<uint4 *>(out + q) = make_uint4(p[0], p[1], p[2], p[3]);
            if (q + 8 < a.D) *reinterpret_cast<uint4 *>(out + q + 8) = make_uint4(p[4], p[5], p[6], p[7]);
          }
        }
        __syncwarp();
      };
#pragma unroll 1
      for (int q = 0; q < a.D; q += 16) results(q, false);
      if (__any_sync(0xffffffffu, z != 0.f && l == l && r < rows)) {
#pragma unroll 1
        for (int q = 0; q < a.D; q += 16) results(q, true);
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
    for (int round = 0; round < rounds; ++round) {
      if (round > 0 && round % PT_ROUNDS == 0) {
        meet();
        look_up(round, warp - PT_SOFT, PT_THREADS / WARP - PT_SOFT);
        meet();
      }
      const int4 w = mine[round % PT_ROUNDS];
      if (w.z <= 0 || dead) continue;
      const int row0 = w.x, q0 = w.y, h = w.w, g = h / (a.H / a.G), d0 = q0 / KN;
      const bool both = w.z > PT_M;
      // the last key tiles of the query tiles, and how many there are; from d0 on not every row sees all of a tile
      const int last0 = (q0 + min(w.z, PT_M) - 1) / KN, n = (q0 + w.z - 1) / KN + 1;
      parity ^= 1;
      if (warp == PT_LOADER) {
        if (lane == 0) {
          auto load = [&](const CUtensorMap *map, int head, int row) {
            const int s = slot % STAGES;
            if (slot >= STAGES && !dead) dead = !mbar_wait(&empty[s], (slot / STAGES - 1) & 1);
            if (dead) return;
            mbar_arrive_expect_tx(&full[s], TILE);
            for (int b = 0; b < KB; ++b) tma_load_rows(ring + s * TILE + b * KN * 128, map, b * 64, head, row, &full[s]);
            ++slot;
          };
          for (int t = 0; t < (both ? 2 : 1); ++t) {
            if (used[t] && !dead) dead = !mbar_wait(&q_empty[t], (used[t] - 1) & 1);
            if (dead) break;
            ++used[t];
            mbar_arrive_expect_tx(&q_full[t], Q_TILE);
            for (int b = 0; b < KB; ++b)
              tma_load_rows(q_sm + t * Q_TILE + b * PT_M * 128, &map_q, b * 64, h, row0 + q0 + t * PT_M, &q_full[t]);
            if (t == 0) load(&map_k, g, row0);
          }
          for (int j = 0; j < n && !dead; ++j) {
            if (j) load(&map_k, g, row0 + j * KN);
            load(&map_v, g, row0 + j * KN);
          }
        }
        dead = __shfl_sync(0xffffffffu, (int)dead, 0) != 0;
      } else if (warp == PT_ISSUER) {
        constexpr bool FP16 = !__is_same(T, bf16);
        const uint32_t idesc_s = mma_idesc(PT_M, KN, false, false, FP16), idesc_o = mma_idesc(PT_M, FULL ? KB * 64 : (a.D + 15) / 16 * 16, false, true, FP16);
        const int k_steps = FULL ? KB * 4 : (a.D + 15) / 16;
        const uint64_t qd = desc_k_major(q_sm, PT_M, 0), k0 = desc_k_major(ring, KN, 0), v0 = desc_mn_major(ring, KN, 0);
        auto wait = [&](uint64_t *bar, int phase) {
          if (!dead && !mbar_try_wait(bar, phase & 1)) dead = !mbar_wait(bar, phase & 1);
          __syncwarp();
          tmem_fence_after();
        };
        auto scores = [&](int t, int at) {
          const uint64_t q = qd + t * (Q_TILE / 16), k = k0 + at % STAGES * (TILE / 16);
#pragma unroll
          for (int x = 0; x < KB * 4; ++x) {
            // (descriptor units of 16 bytes)
            if (FULL || x < k_steps)
              warp_mma_ss(tm + t * KN, q + (x / 4) * (PT_M * 128 / 16) + (x % 4) * 2, k + (x / 4) * (KN * 128 / 16) + (x % 4) * 2, idesc_s, x > 0);
          }
          warp_commit(&s_full[t]);
        };
        auto values = [&](int t, int at, bool begun) {
          const uint64_t v = v0 + at % STAGES * (TILE / 16);
#pragma unroll
          for (int x = 0; x < KN / 16; ++x)
            warp_mma_ts(tm + O_AT + t * (KB * 64), tm + t * KN + x * 8, v + (uint64_t)(x * 128), idesc_o,
                        x > 0 ? 1u : (uint32_t)begun);
        };
        // slots of this item: K0, V0, K1, V1, ... Those of the next step are waited for behind this step's products.
        const int first = slot;
        auto arrive = [&](int j) {  // V of step j, K of step j + 1
          const int vs = first + 2 * j + 1;
          wait(&full[vs % STAGES], vs / STAGES);
          if (j >= d0) {
            wait(&clean[vs % STAGES], looked >> (vs % STAGES));
            looked ^= 1u << (vs % STAGES);
          }
          if (j + 1 < n) wait(&full[(vs + 1) % STAGES], (vs + 1) / STAGES);
        };
        wait(&full[first % STAGES], first / STAGES);
        for (int t = 0; t < (both ? 2 : 1); ++t) {
          wait(&q_full[t], used[t]);
          ++used[t];
          scores(t, first);
        }
        warp_commit(&empty[first % STAGES]);
        arrive(0);
        for (int j = 0; j < n; ++j) {
          const int vs = first + 2 * j + 1;
          if (j <= last0) {
            wait(&p_full[0], stepped[0]);
            ++stepped[0];
            values(0, vs, j > 0);
            if (j < last0) {
              scores(0, vs + 1);
              if (j + 1 == last0) warp_commit(&q_empty[0]);
            } else {
              warp_commit(&o_full[0]);
              if (j == 0) warp_commit(&q_empty[0]);  // (a tile with one key tile)
            }
          }
          if (both) {
            wait(&p_full[1], stepped[1]);
            ++stepped[1];
            values(1, vs, j > 0);
          }
          warp_commit(&empty[vs % STAGES]);
          if (j + 1 < n) {
            if (both) {
              scores(1, vs + 1);
              if (j + 2 == n) warp_commit(&q_empty[1]);
            }
            warp_commit(&empty[(vs + 1) % STAGES]);
            arrive(j + 1);
          } else if (both) {
            warp_commit(&o_full[1]);
          }
        }
        slot += 2 * n;
        dead = __any_sync(0xffffffffu, dead);
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
          uint4 *v = reinterpret_cast<uint4 *>(base + NT * Q_TILE + vs % STAGES * TILE);
          // the largest magnitude, two 16-bit numbers at a time: infinities and NaN are above all others
          uint32_t large[4] = {0, 0, 0, 0};
#pragma unroll 4
          for (int i = me; i < (int)(TILE / 16); i += 2 * WARP) {
            const uint4 y = v[i];
            large[0] = __vmaxu2(large[0], y.x & 0x7fff7fffu);
            large[1] = __vmaxu2(large[1], y.y & 0x7fff7fffu);
            large[2] = __vmaxu2(large[2], y.z & 0x7fff7fffu);
            large[3] = __vmaxu2(large[3], y.w & 0x7fff7fffu);
          }
          const uint32_t most = __vmaxu2(__vmaxu2(large[0], large[1]), __vmaxu2(large[2], large[3]));
          bool any = (((most & Exponent<T>::MASK) + Exponent<T>::ONE) & 0x80008000u) != 0;
          if (any) {
            for (int i = me; i < (int)(TILE / 16); i += 2 * WARP) {
              uint4 y = v[i];
              uint32_t *e = reinterpret_cast<uint32_t *>(&y);
#pragma unroll
              for (int z = 0; z < 4; ++z) {
                const uint32_t top = ((e[z] & Exponent<T>::MASK) + Exponent<T>::ONE) & 0x80008000u;
                if (top & 0x8000u) e[z] &= 0xffff0000u;
                if (top & 0x80000000u) e[z] &= 0x0000ffffu;
              }
              v[i] = y;
            }
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
    if (warp == PT_ISSUER && dead) {
      warp_commit(&drained);
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

// rows of heads of D elements: boxes of 64 elements x 1 head x `rows` rows with the 128-byte swizzle, zeros outside
static bool rows_map(CUtensorMap *map, bool fp16, const void *p, long long ld, long long hs, int T, int heads, int D, int rows) {
  const cuuint64_t dims[3] = {(cuuint64_t)D, (cuuint64_t)heads, (cuuint64_t)T},
                   strides[2] = {(cuuint64_t)(heads > 1 ? hs : ld) * 2, (cuuint64_t)ld * 2};
  const cuuint32_t box[3] = {64, 1, (cuuint32_t)rows}, unit[3] = {1, 1, 1};
  return encode_tiled()(map, fp16 ? CU_TENSOR_MAP_DATA_TYPE_FLOAT16 : CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, 3, const_cast<void *>(p), dims,
                        strides, box, unit, CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
                        CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}

// Whether TMA can read the rows: strides are positive multiples of 16 bytes.
static bool rows_fit(const void *p, long long ld, long long hs, int heads) {
  return aligned16(p) && ld > 0 && ld % 8 == 0 && ld < (1ll << 36) && (heads == 1 || (hs > 0 && hs % 8 == 0 && hs < (1ll << 36)));
}
bool packed_tc_supported(int dtype, const PackedArgs &a) {
  return dtype != DJV_DTYPE_F32 && a.D % 8 == 0 && a.D <= 256 && rows_fit(a.q, a.ldq, a.hq, a.H) && rows_fit(a.k, a.ldk, a.hk, a.G) &&
         rows_fit(a.v, a.ldv, a.hv, a.G) && aligned16(a.out) &&
         (long long)packed_tiles<PT_M>(a.T, a.B) * a.H < (1ll << 30) && encode_tiled();
}

template <typename T, int KB, bool FULL>
static int launch_packed_tc(const PackedArgs &a, cudaStream_t st) {
  // Heads of more than 128: O takes 256 columns of TMEM, so that there is room for one query tile, and tiles of 64 keys for four stages.
  constexpr int NT = KB > 2 ? 1 : 2, KN = KB > 2 ? 64 : 128, STAGES = KB == 1 ? 8 : 4;
  constexpr int smem = 1024 + NT * KB * PT_M * 128 + STAGES * KB * KN * 128;
  constexpr bool FP16 = !__is_same(T, bf16);
  const auto kernel = packed_tc_kernel<T, KB, FULL, NT, KN, STAGES>;
  CUtensorMap q, k, v;
  if (!rows_map(&q, FP16, a.q, a.ldq, a.hq, a.T, a.H, a.D, PT_M) || !rows_map(&k, FP16, a.k, a.ldk, a.hk, a.T, a.G, a.D, KN) ||
      !rows_map(&v, FP16, a.v, a.ldv, a.hv, a.T, a.G, a.D, KN)) {
    set_error("packed_attention: a tensor map was refused");
    return DJV_ERR_CUDA;
  }
  static DevicePrep prep;
  const int(*unused)[4];
  cudaError_t e = prep.get([&](int(&)[4]) { return cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, smem); }, unused);
  // (no fewer than there can be)
  const int tiles = packed_tiles<NT * PT_M>(a.T, a.B), grid = tiles * a.H < sm_count() ? tiles * a.H : sm_count();
  if (e == cudaSuccess) e = djv::launch_kernel(kernel, dim3(grid), dim3(PT_THREADS), smem, st, q, k, v, a, tiles);
  if (e != cudaSuccess) {
    cudaGetLastError();
    set_error("packed_attention: CUDA error %d (%s)", (int)e, cudaGetErrorString(e));
    return DJV_ERR_CUDA;
  }
  count_launch();
  return check_launch("packed_attention");
}

int packed_tc(int dtype, const PackedArgs &a, cudaStream_t st) {
  const auto of = [&](auto t) {
    using T = decltype(t);
    const bool sectors = (reinterpret_cast<uintptr_t>(a.out) & 31) == 0;  // whole heads are stored 32 bytes at a time
    if (a.D <= 64) return a.D == 64 && sectors ? launch_packed_tc<T, 1, true>(a, st) : launch_packed_tc<T, 1, false>(a, st);
    if (a.D <= 128) return a.D == 128 && sectors ? launch_packed_tc<T, 2, true>(a, st) : launch_packed_tc<T, 2, false>(a, st);
    return a.D == 256 && sectors ? launch_packed_tc<T, 4, true>(a, st) : launch_packed_tc<T, 4, false>(a, st);
  };
  return dtype == DJV_DTYPE_F16 ? of(__half()) : of(bf16());
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
