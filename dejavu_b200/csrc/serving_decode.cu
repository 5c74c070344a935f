// Attention of one new token per sequence over its paged cache: every cached byte is read once, so HBM is the bound, or, for short
// caches, the chain position -> page -> keys -> softmax -> values -> join.
//
// The cached tokens of all sequences and key/value heads are cut into units of 64 and dealt out evenly to the blocks that are resident
// at once (serving_plan.cuh), whatever the lengths are; the lengths are only known on the device. An item (key/value head of a
// sequence, with up to 16 of the query heads that share it) that one block has all of goes straight to the output; parts of
// others go to scratch and a second kernel, launched programmatically, joins them in order. Where the table has no room for more
// than a few units a block takes an item and there is no second kernel.
//
// A block's four warps take 16 tokens at a time, each with a softmax of its own, joined in shared memory at the item's end. Rows of K and V
// arrive in a ring per warp by 16-byte asynchronous copies (any page size, any strides), swizzled for ldmatrix; the ring runs on from
// item to item, so that the next one's rows are on their way while one ends, and the page of a tile is
// looked up a tile ahead. fp16 and bf16 go through mma.sync, 16 query heads x 16 tokens: tcgen05 would have to pad the heads to
// 64 or 128 rows, and the tensor work is a small part of the time either way. The weights enter the second product as two terms
// of the cache's type, hi + lo, so that they keep 16 bits (bf16), or 22 (fp16) down to 2^-18 of the largest, below which they are off by 2^-38
// of the largest at most: fp16 ends at 2^-24, so its weights are 2^15 times as large, and so are their sums. fp32 goes through the CUDA cores, 4 heads and 8 or 16
// tokens at a time.
//
// A value that is not finite and is seen makes its dimension so: hi is rounded towards 0, so that lo is not negative, and neither is 0
// where it stands for something (0 times an infinity is NaN). In fp16 that holds however small the weight is, in bf16 and fp32 for weights
// of 2^-126 of the largest and more, which is what 32 bits hold. (A look at the sums at the end of an item costs 2 us of 49 with short
// items: code that is fetched once.)
//
// Measured (bf16, pages of 16, 32 query heads over 8 of 128 dimensions): one cache of 131071 tokens 95 us, 5.7 TB/s; 64 of up to 8192 tokens 173 us,
// 5.9 TB/s; 16 of 32 heads, fp16, up to 2048 tokens 51 us, 5.0 TB/s (101 before an item's beginning and end counted as units); 137
// tokens of 12 heads of 64 5.2 us in a graph. fp32, 16 caches of up to 4000 tokens, 32 heads over 8 of 128: 72 us, 4.0 TB/s (96 with queries from L1,
// branches for the rows and 16 tokens): exponentials and shuffles of tiles of 8 tokens. Heads of 256, bf16, over the same lengths: 78 us,
// 3.7 TB/s, as shared memory has room for one block.
#include <math.h>
#include <type_traits>

#include "mma.cuh"
#include "pairs.cuh"
#include "ring.cuh"
#include "serving.cuh"
#include "tensor_map.cuh"

namespace djv {

__device__ unsigned g_decode_faults;
__device__ unsigned g_decode_timeouts;  // bounded waits that ran out (never, in a healthy run)

constexpr int DE_WARPS = 4, DE_THREADS = DE_WARPS * WARP;

struct DecodeArgs {
  void *out;
  const void *q, *k, *v;
  long long ldq, hq;
  Pool pool;
  int pages, page;
  Divider by_page;
  const int *table;
  long long ld_table;
  int width;
  const long long *pos;
  int B, H, G, D;
  float scale;
  float *parts;  // two slots for each block: of the item that it ends and of the one that it begins; NULL: no item is split
  int groups;    // groups of query heads that share a key/value head
};

// Tokens of sequence b.
__device__ __forceinline__ long long decode_tokens(const DecodeArgs &a, int b) {
  const long long p = a.pos[b], room = (long long)a.width * a.page;
  return p < 0 ? 0 : (p >= room ? room : p + 1);
}

struct DecodePlace {
  int b;
  long long base, total;  // the first unit of sequence b, units of the batch
};
// The sequence that unit x is in, by all of the block; `of(total)` says which unit that is.
template <typename F>
__device__ __forceinline__ DecodePlace decode_locate(const DecodeArgs &a, F of, long long *slots) {
  const int tid = threadIdx.x, lane = tid % WARP, warp = tid / WARP, share = a.G * a.groups;
  long long mine = 0, first = 0;
  for (int b = tid; b < a.B; b += DE_THREADS) {
    const long long u = units_of(decode_tokens(a, b)) * share;
    if (b == tid) first = u;
    mine += u;
  }
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) mine += __shfl_xor_sync(0xffffffffu, mine, o);
  if (lane == 0) slots[warp] = mine;
  __syncthreads();
  long long total = 0;
#pragma unroll
  for (int w = 0; w < DE_WARPS; ++w) total += slots[w];
  const long long x = of(total);
  long long run = 0;
  if (tid == 0) slots[DE_WARPS] = -1;
  for (int b0 = 0; b0 < a.B; b0 += DE_THREADS) {
    const int b = b0 + tid;
    const long long u = b >= a.B ? 0 : (b0 == 0 ? first : units_of(decode_tokens(a, b)) * share);
    long long sum = u;
#pragma unroll
    for (int o = 1; o < WARP; o <<= 1) {
      const long long up = __shfl_up_sync(0xffffffffu, sum, o);
      if (lane >= o) sum += up;
    }
    __syncthreads();
    if (lane == WARP - 1) slots[warp] = sum;
    __syncthreads();
    long long before = run;
#pragma unroll
    for (int w = 0; w < DE_WARPS; ++w) {
      if (w < warp) before += slots[w];
      run += slots[w];
    }
    if (u > 0 && x >= before + sum - u && x < before + sum) {
      slots[DE_WARPS] = b;
      slots[DE_WARPS + 1] = before + sum - u;
    }
    if (x < run) break;
  }
  __syncthreads();
  return {(int)slots[DE_WARPS], slots[DE_WARPS + 1], total};
}

template <typename T>
struct DecodeRows {  // query heads of an item
  static constexpr int N = sizeof(T) == 4 ? 4 : 16;
};

// One warp's share of an item: running maximum (in units of log 2), sum and weighted values of its tokens.
template <typename T, int DP>
struct DecodeSums;

// Of a 16-byte chunk in a tile: blocks of 128 bytes of every row, swizzled as TMA does and as ldmatrix reads without bank conflicts.
template <int ROWS>
__device__ __forceinline__ uint32_t tile_offset(int row, int chunk) {
  return (uint32_t)((chunk >> 3) * (ROWS * 128) + row * 128 + (((chunk & 7) ^ (row & 7)) << 4));
}

// a box of one tile's rows and 128 bytes of each: slots of a page of one head
__device__ __forceinline__ void tma_load_slots(uint32_t dst, const CUtensorMap *map, int d, int slot, int head, int page, uint64_t *bar) {
  asm volatile(
      "cp.async.bulk.tensor.4d.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3, %4, %5}], [%6];" ::"r"(dst), "l"(map),
      "r"(d), "r"(slot), "r"(head), "r"(page), "r"(smem_u32(bar))
      : "memory");
}

template <typename T>
__device__ __forceinline__ uint32_t pair_of(float lo, float hi);
template <>
__device__ __forceinline__ uint32_t pair_of<bf16>(float lo, float hi) { return pack_bf16(lo, hi); }
template <>
__device__ __forceinline__ uint32_t pair_of<__half>(float lo, float hi) {
  __half2 h = __floats2half2_rn(lo, hi);
  return *reinterpret_cast<uint32_t *>(&h);
}
// rounded towards 0
template <typename T>
__device__ __forceinline__ uint32_t pair_below(float lo, float hi);
template <>
__device__ __forceinline__ uint32_t pair_below<bf16>(float lo, float hi) {
  uint32_t v;
  asm("cvt.rz.bf16x2.f32 %0, %1, %2;" : "=r"(v) : "f"(hi), "f"(lo));
  return v;
}
template <>
__device__ __forceinline__ uint32_t pair_below<__half>(float lo, float hi) {
  uint32_t v;
  asm("cvt.rz.f16x2.f32 %0, %1, %2;" : "=r"(v) : "f"(hi), "f"(lo));
  return v;
}
// the smallest number above 0 where it is less
template <typename T>
__device__ __forceinline__ uint32_t above_zero(uint32_t v);
template <>
__device__ __forceinline__ uint32_t above_zero<bf16>(uint32_t v) {
  asm("max.bf16x2 %0, %0, %1;" : "+r"(v) : "r"(0x00010001u));
  return v;
}
template <>
__device__ __forceinline__ uint32_t above_zero<__half>(uint32_t v) {
  asm("max.f16x2 %0, %0, %1;" : "+r"(v) : "r"(0x00010001u));
  return v;
}
template <typename T>
__device__ __forceinline__ float2 floats_of(uint32_t u);
template <>
__device__ __forceinline__ float2 floats_of<bf16>(uint32_t u) { return b2f(u); }
template <>
__device__ __forceinline__ float2 floats_of<__half>(uint32_t u) { return h2f(u); }

// fp16, bf16: lane (g, t) has rows g and g + 8 of the 16 heads, two columns of every 8 dimensions
template <typename T, int DP>
struct MmaSums {
  static constexpr int TOKENS = 16;
  static constexpr float LIFT = std::is_same<T, __half>::value ? 15.f : 0.f;  // weights and sums are 2^LIFT times what they stand for
  // what sums of lower maxima are scaled by: not 0 in fp16, whose sums stay below 2^80
  __device__ __forceinline__ static float factor(float f) { return LIFT > 0 ? fmaxf(f, 1.17549435e-38f) : f; }
  uint32_t q[DP / 16][4];
  float o[DP / 8][4], m[2], l[2];
  uint32_t k_at[4], v_at[4];  // where the lane's rows and chunks of the operands are, in a 128-byte block of a tile

  __device__ __forceinline__ MmaSums() {
    const int lane = threadIdx.x % WARP;
#pragma unroll
    for (int x = 0; x < 4; ++x) {
      k_at[x] = tile_offset<TOKENS>((lane >> 4) * 8 + lane % 8, x * 2 + ((lane >> 3) & 1));
      v_at[x] = tile_offset<TOKENS>(((lane >> 3) & 1) * 8 + lane % 8, x * 2 + (lane >> 4));
    }
  }

  __device__ __forceinline__ void start(const T *query, long long hq, int rows, int D) {
    const int g = threadIdx.x % WARP / 4, t = threadIdx.x % 4;
#pragma unroll
    for (int k = 0; k < DP / 16; ++k)
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        const int row = g + (e & 1) * 8, d = k * 16 + t * 2 + (e >> 1) * 8;
        q[k][e] = row < rows && d < D ? *reinterpret_cast<const uint32_t *>(query + row * hq + d) : 0u;
      }
#pragma unroll
    for (int i = 0; i < DP / 8; ++i)
#pragma unroll
      for (int e = 0; e < 4; ++e) o[i][e] = 0.f;
    m[0] = m[1] = -INFINITY;
    l[0] = l[1] = 0.f;
  }
  // c: scale in units of log 2; seen: a bit for each of the 16 tokens
  __device__ __forceinline__ void tile(uint32_t k_sm, uint32_t v_sm, unsigned seen, float c) {
    const int t = threadIdx.x % 4;
    float s[2][4] = {};
#pragma unroll
    for (int k = 0; k < DP / 16; ++k) {
      uint32_t b[4];
      ldmatrix_x4(b, k_sm + k_at[k % 4] + k / 4 * (TOKENS * 128));
      mma_m16n8k16_t<T>(s[0], q[k][0], q[k][1], q[k][2], q[k][3], b[0], b[1]);
      mma_m16n8k16_t<T>(s[1], q[k][0], q[k][1], q[k][2], q[k][3], b[2], b[3]);
    }
#pragma unroll
    for (int n = 0; n < 2; ++n)
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        s[n][e] *= c;
        if (seen != 0xffffu && !((seen >> (n * 8 + t * 2 + (e & 1))) & 1)) s[n][e] = -INFINITY;
      }
    float corr[2];
#pragma unroll
    for (int r = 0; r < 2; ++r) {
      float top = fmaxf(fmaxf(s[0][2 * r], s[0][2 * r + 1]), fmaxf(s[1][2 * r], s[1][2 * r + 1]));
      top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 1));
      top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 2));
      top = fmaxf(top, m[r]);
      const float base = top == -INFINITY ? 0.f : top, low = base - LIFT;
      corr[r] = factor(exp2_approx(m[r] - base));
      m[r] = top;
#pragma unroll
      for (int n = 0; n < 2; ++n)
#pragma unroll
        for (int e = 2 * r; e < 2 * r + 2; ++e) s[n][e] = exp2_approx(s[n][e] - low);
      l[r] = l[r] * corr[r] + ((s[0][2 * r] + s[0][2 * r + 1]) + (s[1][2 * r] + s[1][2 * r + 1]));
    }
    if (__any_sync(0xffffffffu, corr[0] != 1.f || corr[1] != 1.f)) {
#pragma unroll
      for (int i = 0; i < DP / 8; ++i)
#pragma unroll
        for (int e = 0; e < 4; ++e) o[i][e] *= corr[e >> 1];
    }
    uint32_t hi[4], lo[4];
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      const float x = s[e >> 1][(e & 1) * 2], y = s[e >> 1][(e & 1) * 2 + 1];
      hi[e] = pair_below<T>(x, y);
      if (LIFT > 0) hi[e] = above_zero<T>(hi[e]);  // (values behind the last token are zeros)
      const float2 h = floats_of<T>(hi[e]);
      lo[e] = above_zero<T>(pair_of<T>(x - h.x, y - h.y));
    }
#pragma unroll
    for (int i = 0; i < DP / 16; ++i) {
      uint32_t b[4];
      ldmatrix_x4_trans(b, v_sm + v_at[i % 4] + i / 4 * (TOKENS * 128));
      mma_m16n8k16_t<T>(o[2 * i], hi[0], hi[1], hi[2], hi[3], b[0], b[1]);
      mma_m16n8k16_t<T>(o[2 * i + 1], hi[0], hi[1], hi[2], hi[3], b[2], b[3]);
      mma_m16n8k16_t<T>(o[2 * i], lo[0], lo[1], lo[2], lo[3], b[0], b[1]);
      mma_m16n8k16_t<T>(o[2 * i + 1], lo[0], lo[1], lo[2], lo[3], b[2], b[3]);
    }
  }
  __device__ __forceinline__ void finish() {
#pragma unroll
    for (int r = 0; r < 2; ++r) {
      l[r] += __shfl_xor_sync(0xffffffffu, l[r], 1);
      l[r] += __shfl_xor_sync(0xffffffffu, l[r], 2);
    }
  }
  // another warp's sums join this one's
  __device__ __forceinline__ void absorb(const float *sums, const float *sm, const float *sl) {
    const int lane = threadIdx.x % WARP, g = lane / 4, t = lane % 4;
#pragma unroll
    for (int r = 0; r < 2; ++r) {
      const float other = sm[g + r * 8], top = fmaxf(m[r], other), base = top == -INFINITY ? 0.f : top;
      const float mine = factor(exp2_approx(m[r] - base)), its = factor(exp2_approx(other - base));
      m[r] = top;
      l[r] = l[r] * mine + sl[g + r * 8] * its;
#pragma unroll
      for (int i = 0; i < DP / 8; ++i) {
        const float2 y = *reinterpret_cast<const float2 *>(sums + (g + r * 8) * DP + ((i ^ g) * 8 + t * 2));
        o[i][2 * r] = o[i][2 * r] * mine + y.x * its;
        o[i][2 * r + 1] = o[i][2 * r + 1] * mine + y.y * its;
      }
    }
  }
  // the result, where the item is whole (slot NULL), or what the second kernel joins
  __device__ __forceinline__ void emit(T *out, float *slot, int rows, int D) const {
    const int lane = threadIdx.x % WARP, g = lane / 4, t = lane % 4;
#pragma unroll
    for (int r = 0; r < 2; ++r) {
      const int row = g + r * 8;
      if (row >= rows) continue;
      const float inv = l[r] == 0.f ? 0.f : 1.f / l[r];
#pragma unroll
      for (int i = 0; i < DP / 8; ++i) {
        if (i * 8 >= D) continue;
        if (slot == nullptr) *reinterpret_cast<uint32_t *>(out + row * D + i * 8 + t * 2) = pair_of<T>(o[i][2 * r] * inv, o[i][2 * r + 1] * inv);
        else *reinterpret_cast<float2 *>(slot + row * DP + i * 8 + t * 2) = make_float2(o[i][2 * r], o[i][2 * r + 1]);
      }
      if (slot != nullptr && t == 0) {
        slot[16 * DP + row] = m[r];
        slot[16 * DP + 16 + row] = l[r];
      }
    }
  }
  // sums (rows, DP), 8-column pieces of a row in an order of its own (no bank conflicts), and the rows' maxima and sums
  __device__ __forceinline__ void store(float *sums, float *sm, float *sl) const {
    const int lane = threadIdx.x % WARP, g = lane / 4, t = lane % 4;
#pragma unroll
    for (int r = 0; r < 2; ++r) {
      if (t == 0) {
        sm[g + r * 8] = m[r];
        sl[g + r * 8] = l[r];
      }
#pragma unroll
      for (int i = 0; i < DP / 8; ++i)
        *reinterpret_cast<float2 *>(sums + (g + r * 8) * DP + ((i ^ g) * 8 + t * 2)) = make_float2(o[i][2 * r], o[i][2 * r + 1]);
    }
  }
};
template <int DP>
struct DecodeSums<bf16, DP> : MmaSums<bf16, DP> {};
template <int DP>
struct DecodeSums<__half, DP> : MmaSums<__half, DP> {};

// fp32: for the scores a lane has a token and every PARTS-th chunk of it (of wide heads two tokens, one after the other), so that its share of
// the queries takes 128 registers; for the values it has DP / 32 adjacent dimensions (or two times four). Products go two to an instruction.
template <int DP>
struct DecodeSums<float, DP> {
  static constexpr int TOKENS = DP > 64 ? 8 : 16, TURNS = DP > 128 ? 2 : 1, AT_ONCE = TOKENS / TURNS, PARTS = WARP / AT_ONCE, W = DP / 32,
                       EACH = DP / 4 / PARTS;  // EACH: chunks of a lane
  int rows;
  ulonglong2 q[EACH][4];
  float m[4], l[4];
  union {
    uint64_t o2[4][W / 2];
    float o[4][W];
  };

  // the dimension of a lane's i-th sum
  __device__ __forceinline__ static int dim(int i) {
    const int lane = threadIdx.x % WARP;
    return W <= 4 ? lane * W + i : i / 4 * 128 + lane * 4 + i % 4;
  }
  // a lane's i-th chunk (eight lanes that read at once have eight different columns of the swizzle)
  __device__ __forceinline__ static int chunk(int i) {
    const int part = threadIdx.x % WARP / AT_ONCE;
    return TURNS == 1 ? i * PARTS + part : i * PARTS + part / 2 + part % 2 * 4;
  }
  __device__ __forceinline__ void start(const float *first, long long h, int n, int D) {
    rows = n;
#pragma unroll
    for (int r = 0; r < 4; ++r) {
      m[r] = -INFINITY;
      l[r] = 0.f;
#pragma unroll
      for (int i = 0; i < W / 2; ++i) o2[r][i] = 0;
#pragma unroll
      for (int i = 0; i < EACH; ++i)
        q[i][r] = r < rows && chunk(i) * 4 < D ? __ldg(reinterpret_cast<const ulonglong2 *>(first + r * h + chunk(i) * 4)) : make_ulonglong2(0, 0);
    }
  }
  __device__ __forceinline__ static ulonglong2 at(uint32_t sm) {
    ulonglong2 v;
    asm volatile("ld.shared.v2.u64 {%0,%1}, [%2];" : "=l"(v.x), "=l"(v.y) : "r"(sm) : "memory");
    return v;
  }
  __device__ __forceinline__ void tile(uint32_t k_sm, uint32_t v_sm, unsigned seen, float c) {
    if (rows == 1) tile_of<1>(k_sm, v_sm, seen, c);
    else if (rows == 2) tile_of<2>(k_sm, v_sm, seen, c);
    else tile_of<4>(k_sm, v_sm, seen, c);
  }
  template <int R>  // rows (of four the last may be zeros): no branches, so that their chains overlap
  __device__ __forceinline__ void tile_of(uint32_t k_sm, uint32_t v_sm, unsigned seen, float c) {
    const int lane = threadIdx.x % WARP, mine = lane % AT_ONCE;
    float s[TURNS][R];
#pragma unroll
    for (int n = 0; n < TURNS; ++n) {
      uint64_t s2[R] = {};
#pragma unroll
      for (int i = 0; i < EACH; ++i) {
        const ulonglong2 k = at(k_sm + tile_offset<TOKENS>(n * AT_ONCE + mine, chunk(i)));
#pragma unroll
        for (int r = 0; r < R; ++r) s2[r] = fma2(q[i][r].y, k.y, fma2(q[i][r].x, k.x, s2[r]));
      }
#pragma unroll
      for (int r = 0; r < R; ++r) {
        float x, y;
        unpack2(s2[r], x, y);
        s[n][r] = x + y;
      }
    }
    float top[R];
#pragma unroll
    for (int x = AT_ONCE; x < WARP; x <<= 1)
#pragma unroll
      for (int n = 0; n < TURNS; ++n)
#pragma unroll
        for (int r = 0; r < R; ++r) s[n][r] += __shfl_xor_sync(0xffffffffu, s[n][r], x);
#pragma unroll
    for (int r = 0; r < R; ++r) {
      top[r] = m[r];
#pragma unroll
      for (int n = 0; n < TURNS; ++n) {
        s[n][r] = (seen >> (n * AT_ONCE + mine)) & 1 ? s[n][r] * c : -INFINITY;
        top[r] = fmaxf(top[r], s[n][r]);
      }
    }
#pragma unroll
    for (int x = AT_ONCE / 2; x > 0; x >>= 1)
#pragma unroll
      for (int r = 0; r < R; ++r) top[r] = fmaxf(top[r], __shfl_xor_sync(0xffffffffu, top[r], x));
#pragma unroll
    for (int r = 0; r < R; ++r) {
      const float base = top[r] == -INFINITY ? 0.f : top[r], corr = exp2f(m[r] - base);
      m[r] = top[r];
      l[r] *= corr;
#pragma unroll
      for (int n = 0; n < TURNS; ++n) {
        s[n][r] = exp2f(s[n][r] - base);
        if (lane < AT_ONCE) l[r] += s[n][r];
      }
      const uint64_t corr2 = pack2(corr, corr);
#pragma unroll
      for (int i = 0; i < W / 2; ++i) o2[r][i] = fma2(o2[r][i], corr2, 0);
    }
#pragma unroll
    for (int t = 0; t < TOKENS; ++t) {
      uint64_t v[W / 2];
      if (W == 2) {
        asm volatile("ld.shared.u64 %0, [%1];" : "=l"(v[0]) : "r"(v_sm + tile_offset<TOKENS>(t, lane / 2) + lane % 2 * 8) : "memory");
      } else {
#pragma unroll
        for (int i = 0; i < W / 4; ++i) {
          const ulonglong2 x = at(v_sm + tile_offset<TOKENS>(t, i * WARP + lane));
          v[2 * i % (W / 2)] = x.x;
          v[(2 * i + 1) % (W / 2)] = x.y;
        }
      }
#pragma unroll
      for (int r = 0; r < R; ++r) {
        const float p = __shfl_sync(0xffffffffu, s[t / AT_ONCE][r], t % AT_ONCE);
        const uint64_t p2 = pack2(p, p);
#pragma unroll
        for (int i = 0; i < W / 2; ++i) o2[r][i] = fma2(p2, v[i], o2[r][i]);
      }
    }
  }
  __device__ __forceinline__ void finish() {
#pragma unroll
    for (int r = 0; r < 4; ++r) l[r] = warp_sum(l[r]);
  }
  __device__ __forceinline__ void absorb(const float *sums, const float *sm, const float *sl) {
#pragma unroll
    for (int r = 0; r < 4; ++r) {
      const float top = fmaxf(m[r], sm[r]), base = top == -INFINITY ? 0.f : top, mine = exp2f(m[r] - base), its = exp2f(sm[r] - base);
      m[r] = top;
      l[r] = l[r] * mine + sl[r] * its;
#pragma unroll
      for (int i = 0; i < W; ++i) o[r][i] = o[r][i] * mine + sums[r * DP + i * WARP + threadIdx.x % WARP] * its;  // (any order, as store has it)
    }
  }
  __device__ __forceinline__ void emit(float *out, float *slot, int n, int D) const {
    const int lane = threadIdx.x % WARP;
#pragma unroll
    for (int r = 0; r < 4; ++r) {
      if (r >= n) continue;
      const float inv = l[r] == 0.f ? 0.f : 1.f / l[r];
#pragma unroll
      for (int i = 0; i < W; ++i) {
        const int d = dim(i);
        if (d >= D) continue;
        if (slot == nullptr) out[r * D + d] = o[r][i] * inv;
        else slot[r * DP + d] = o[r][i];
      }
      if (slot != nullptr && lane == 0) {
        slot[4 * DP + r] = m[r];
        slot[4 * DP + 4 + r] = l[r];
      }
    }
  }
  __device__ __forceinline__ void store(float *sums, float *sm, float *sl) const {
    const int lane = threadIdx.x % WARP;
#pragma unroll
    for (int r = 0; r < 4; ++r) {
      if (lane == 0) {
        sm[r] = m[r];
        sl[r] = l[r];
      }
#pragma unroll
      for (int i = 0; i < W; ++i) sums[r * DP + i * WARP + lane] = o[r][i];
    }
  }
};

template <typename T, int DP>
struct DecodeRing {
  static constexpr int TILE = DecodeSums<T, DP>::TOKENS * DP * (int)sizeof(T);  // bytes of a tile of keys, or of values
  // as many blocks and stages as shared memory has room for: 16 to 24 KB in flight per warp, 96 to 192 KB per multiprocessor
  static constexpr int BLOCKS = TILE <= 2048 ? 3 : (TILE <= 4096 ? 2 : 1), STAGES = TILE <= 2048 ? 4 : 3;
  static constexpr int BYTES = DE_WARPS * STAGES * 2 * TILE, SUMS = DecodeRows<T>::N * DP;  // sums: floats of one warp's
  struct Rest {
    uint64_t full[DE_WARPS][STAGES];
    long long slots[DE_WARPS + 2];
    float sm[2][DecodeRows<T>::N], sl[2][DecodeRows<T>::N];
    unsigned seen[DE_WARPS][STAGES];
  };
  static constexpr int SMEM = BYTES + 2 * SUMS * 4 + (int)sizeof(Rest);
};

// Where a block is in its units.
struct DecodeCursor {
  long long x, end, base;  // next unit, the last one's end, the sequence's first unit
  int b, tokens, units;    // of an item of the sequence
  int item, from, to;      // the part: units from .. to - 1 of the item, whose key/value head is
  int head;
  int t0, t1;
  int tiles, i;  // rounds of four tiles of this part, and the next of them
};

// BOXES: pages are whole tiles, which TMA brings, one thread asking; else every lane copies 16-byte chunks.
template <typename T, int DP, bool BOXES>
__global__ void __launch_bounds__(DE_THREADS, DecodeRing<T, DP>::BLOCKS)
decode_kernel(const __grid_constant__ CUtensorMap map_k, const __grid_constant__ CUtensorMap map_v, DecodeArgs a, int least) {
  using Sums = DecodeSums<T, DP>;
  using Ring = DecodeRing<T, DP>;
  constexpr int ROWS = DecodeRows<T>::N, TOKENS = Sums::TOKENS, STAGES = Ring::STAGES, TILE = Ring::TILE;
  constexpr int N = Chunk<T>::N, CHUNKS = DP / N;                              // of a row
  constexpr int AT_ONCE = CHUNKS >= WARP ? 1 : WARP / CHUNKS, WIDE = CHUNKS > WARP ? CHUNKS / WARP : 1;
  extern __shared__ __align__(1024) unsigned char ring[];
  float *const joined = reinterpret_cast<float *>(ring + Ring::BYTES);
  // (not of their own beside the ring: what stands in front of it would be padded to its alignment)
  auto &rest = *reinterpret_cast<typename Ring::Rest *>(joined + 2 * Ring::SUMS);
  auto &full = rest.full;
  auto &sm = rest.sm, &sl = rest.sl;
  auto &seen = rest.seen;
  long long *const slots = rest.slots;
  const int tid = threadIdx.x, lane = tid % WARP, warp = tid / WARP;
  if (BOXES) {
    if (lane == 0) {
      for (int i = 0; i < STAGES; ++i) mbar_init(&full[warp][i], 1);
      mbar_fence_init();
    }
    __syncwarp();
  }
  // (in this order: what the second kernel reads ahead of its wait, the positions, is complete when it starts)
  asm volatile("griddepcontrol.wait;" ::: "memory");
  asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
  const int share = a.G * a.groups, R = a.H / a.G;
  auto sequence = [&](DecodeCursor &c) {
    c.tokens = (int)decode_tokens(a, c.b);
    c.units = (int)units_of(c.tokens);
  };
  auto open = [&](DecodeCursor &c) {  // the part that begins at c.x
    const DecodePart p = decode_part(c.x, c.end, c.base, c.units);
    c.item = (int)p.item;
    c.head = c.item / a.groups;
    c.from = (int)p.from;
    c.to = (int)p.to;
    c.t0 = (int)tokens_before(p.from, c.tokens);
    c.t1 = (int)tokens_before(p.to, c.tokens);
    c.tiles = c.t1 > c.t0 ? (c.t1 - c.t0 + DE_WARPS * TOKENS - 1) / (DE_WARPS * TOKENS) : 1;
    c.i = 0;
  };
  auto close = [&](DecodeCursor &c) {  // on to the next part; false: there is none
    c.x += c.to - c.from;
    if (c.x >= c.end) return false;
    if (c.x == c.base + (long long)c.units * share) {
      c.base = c.x;
      ++c.b;
      sequence(c);
    }
    open(c);
    return true;
  };
  DecodeCursor at;  // of the products
  if (a.parts == nullptr) {  // an item each
    at.b = blockIdx.x / share;
    at.base = 0;
    sequence(at);
    at.x = (long long)(blockIdx.x - at.b * share) * at.units;
    at.end = at.x + at.units;
  } else {
    long long per;
    const DecodePlace w = decode_locate(a, [&](long long total) {
      per = units_per_block(total, gridDim.x, least);
      return blockIdx.x * per;
    }, slots);
    at.x = blockIdx.x * per;
    at.end = at.x + per < w.total ? at.x + per : w.total;
    if (at.x >= at.end || w.b < 0) return;
    at.b = w.b;
    at.base = w.base;
    sequence(at);
  }
  open(at);
  DecodeCursor ahead = at;  // of the loads
  bool more = true;
  const uint32_t warp_ring = smem_addr(ring) + warp * STAGES * 2 * TILE;
  const float c = a.scale * 1.4426950408889634f;

  const PageMap no_map{nullptr, a.width, a.page, a.pages, a.by_page};
  // The first token of the warp's next tile; where its row is in the pools (BOXES: the page and, in the upper half, the slot), or -1.
  // Without BOXES the lane's own token's, lanes beyond the tile's tokens repeat them.
  auto row_ahead = [&]() -> long long {
    const int at = (ahead.i * DE_WARPS + warp) * TOKENS + (BOXES ? 0 : lane % TOKENS);
    if (!more || at >= ahead.t1 - ahead.t0) return -1;  // (the tile's tokens may pass 2^31)
    const int t = ahead.t0 + at;
    int slot;
    PageMap map = no_map;
    map.table = a.table + ahead.b * a.ld_table;
    const long long page = page_of(map, t, slot);
    if (page != NO_PAGE) return BOXES ? (long long)slot << 32 | page : page * a.pool.ld_page + slot * a.pool.ld_slot;
    if (ahead.item == 0 && lane < (BOXES ? 1 : TOKENS) && (slot == 0 || lane == 0)) atomicAdd(&g_decode_faults, 1u);
    return -1;
  };
  long long row = row_ahead();
  unsigned asked = 0, taken = 0;  // phases of the stages' barriers, a bit each
  unsigned there = 0;             // stages that have a tile
  bool dead = false;              // a wait ran out: wait no more, finish and report
  auto load = [&](int stage) {
    if (more) {
      const uint32_t dst = warp_ring + stage * 2 * TILE;
      const int g = ahead.head;
      if (BOXES) {
        const unsigned bit = 1u << stage;
        there &= ~bit;
        if (row >= 0) {
          there |= bit;
          asked ^= bit;
          if (lane == 0) {
            mbar_arrive_expect_tx(&full[warp][stage], 2 * TILE);
#pragma unroll
            for (int x = 0; x < DP * (int)sizeof(T) / 128; ++x) {
              const int d = x * (128 / (int)sizeof(T));
              tma_load_slots(dst + x * TOKENS * 128, &map_k, d, (int)(row >> 32), g, (int)row, &full[warp][stage]);
              tma_load_slots(dst + TILE + x * TOKENS * 128, &map_v, d, (int)(row >> 32), g, (int)row, &full[warp][stage]);
            }
          }
        }
      } else {
        const unsigned bits = __ballot_sync(0xffffffffu, row >= 0) & ((1u << TOKENS) - 1);
        if (lane == 0) seen[warp][stage] = bits;
        const long long head = g * a.pool.ld_head;
        const T *k = static_cast<const T *>(a.k), *v = static_cast<const T *>(a.v);
#pragma unroll
        for (int p = 0; p < TOKENS / AT_ONCE; ++p) {
          const int r = p * AT_ONCE + (CHUNKS >= WARP ? 0 : lane / CHUNKS);
          const long long off = __shfl_sync(0xffffffffu, row, r);
#pragma unroll
          for (int y = 0; y < WIDE; ++y) {
            const int ch = CHUNKS >= WARP ? y * WARP + lane : lane % CHUNKS;
            const bool ok = off >= 0 && ch * N < a.D;
            const long long from = ok ? off + head + ch * N : 0;
            const uint32_t to = dst + tile_offset<TOKENS>(r, ch);
            cp_async16_zfill(to, k + from, ok ? 16 : 0);
            cp_async16_zfill(to + TILE, v + from, ok ? 16 : 0);
          }
        }
      }
      if (++ahead.i == ahead.tiles) more = close(ahead);
      row = row_ahead();
    }
    if (!BOXES) cp_async_commit();
  };
  // Waits for a stage; its tokens that are there. Values that are not (behind the sequence's last token) become zeros.
  auto arrived = [&](int stage, int i) -> unsigned {
    if (!BOXES) {
      cp_async_wait<STAGES - 1>();
      __syncwarp();
      return seen[warp][stage];
    }
    const int left = at.t1 - at.t0 - (i * DE_WARPS + warp) * TOKENS;
    const unsigned bits = !((there >> stage) & 1) ? 0u : (left >= TOKENS ? (1u << TOKENS) - 1 : (1u << left) - 1);
    if (bits) {
      if (!dead) dead = !mbar_wait(&full[warp][stage], (taken >> stage) & 1);
      taken ^= 1u << stage;
      if (bits != (1u << TOKENS) - 1) {
        const int first = __popc(bits);  // (they are the last ones)
        for (int i = lane; i < (TOKENS - first) * CHUNKS; i += WARP)
          asm volatile("st.shared.v4.b32 [%0], {%1, %1, %1, %1};" ::"r"(warp_ring + stage * 2 * TILE + TILE +
                                                                         tile_offset<TOKENS>(first + i / CHUNKS, i % CHUNKS)),
                       "r"(0)
                       : "memory");
        fence_proxy_async_smem();
        __syncwarp();
      }
    }
    return bits;
  };
#pragma unroll 1
  for (int i = 0; i < STAGES - 1; ++i) load(i);

  Sums sums;
  int stage = 0;
  for (;;) {
    const int g = at.head, h0 = (at.item - g * a.groups) * ROWS, rows = min(ROWS, R - h0), h = g * R + h0;
    if (tid == 0 && at.item == 0 && at.from == 0 && a.pos[at.b] >= (long long)a.width * a.page) atomicAdd(&g_decode_faults, 1u);
    sums.start(static_cast<const T *>(a.q) + at.b * a.ldq + h * a.hq, a.hq, rows, a.D);
#pragma unroll 1
    for (int i = 0; i < at.tiles; ++i) {
      load(stage == 0 ? STAGES - 1 : stage - 1);
      const unsigned bits = arrived(stage, i);
      if (bits) sums.tile(warp_ring + stage * 2 * TILE, warp_ring + stage * 2 * TILE + TILE, bits, c);
      __syncwarp();
      stage = stage == STAGES - 1 ? 0 : stage + 1;
    }
    // the four warps' sums: two and two, then the two that are left
    sums.finish();
    __syncthreads();  // (the last item's sums have been read)
    if (warp >= 2) sums.store(joined + (warp - 2) * Ring::SUMS, sm[warp - 2], sl[warp - 2]);
    __syncthreads();
    if (warp < 2) sums.absorb(joined + warp * Ring::SUMS, sm[warp], sl[warp]);
    __syncwarp();
    if (warp == 1) sums.store(joined + Ring::SUMS, sm[1], sl[1]);
    __syncthreads();
    if (warp == 0) {
      sums.absorb(joined + Ring::SUMS, sm[1], sl[1]);
      const bool whole = at.from == 0 && at.to == at.units;
      // the slot of a part: 1 of an item that begins here, 0 of one that began in a block before
      float *slot = whole ? nullptr : a.parts + (blockIdx.x * 2 + (at.from == 0 ? 1 : 0)) * (long long)(ROWS * (DP + 2));
      sums.emit(static_cast<T *>(a.out) + ((long long)at.b * a.H + h) * a.D, slot, rows, a.D);
    }
    if (!close(at)) break;
  }
  cp_async_wait<0>();
  if (BOXES && dead) {  // copies that nobody waited for still land
    for (int i = 0; i < STAGES; ++i)
      if (asked != 0 || taken != 0) mbar_wait(&full[warp][i], ((asked >> i) & 1) ^ 1);
    if (lane == 0) atomicAdd(&g_decode_timeouts, 1u);
  }
}

// A sum times a factor from 0 to 1; an infinite one stays, whatever the factor has been rounded to.
__device__ __forceinline__ float scaled(float y, float f) { return fabsf(y) == INFINITY ? y : y * f; }

// Joins the parts of the item that begins in block blockIdx.x of `blocks` and ends in a later one, if there is one: row blockIdx.y, the
// parts dealt out to the warps, four dimensions to a lane.
template <typename T, int DP>
__global__ void __launch_bounds__(DE_THREADS) decode_join_kernel(DecodeArgs a, int blocks, int least) {
  constexpr int ROWS = DecodeRows<T>::N, WIDE = DP > 128 ? 2 : 1;
  constexpr long long SLOT = ROWS * (DP + 2);
  __shared__ long long slots[DE_WARPS + 2];
  __shared__ float4 so[DE_WARPS][WIDE * WARP];
  __shared__ float sm[DE_WARPS], sl[DE_WARPS];
  const int lane = threadIdx.x % WARP, warp = threadIdx.x / WARP;
  asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
  long long per;
  const int R = a.H / a.G;
  // (positions and their like are those the first kernel worked with: it let this one start when they were complete)
  const DecodePlace w = decode_locate(a, [&](long long total) {
    per = units_per_block(total, blocks, least);
    return (blockIdx.x + 1) * per - 1;
  }, slots);
  const long long last = (blockIdx.x + 1) * per - 1;  // this block's last unit
  bool mine = last + 1 < w.total && w.b >= 0;
  long long item = 0;
  int more = 0;  // parts after the first, 2 * SLOT apart
  if (mine) {
    const long long units = units_of(decode_tokens(a, w.b));
    item = (last - w.base) / units;
    const long long from = w.base + item * units, to = from + units;
    mine = to > last + 1 && from >= blockIdx.x * per;  // else it ends here, or began in a block before
    more = (int)((to - 1) / per) - (int)blockIdx.x;
  }
  asm volatile("griddepcontrol.wait;" ::: "memory");
  const int g = (int)(item / a.groups), h0 = (int)(item % a.groups) * ROWS, r = blockIdx.y;
  if (!mine || r >= min(ROWS, R - h0)) return;
  const float *begin = a.parts + (blockIdx.x * 2 + 1) * SLOT, *rest = a.parts + blockIdx.x * 2 * SLOT;  // part s > 0: rest + s * 2 * SLOT
  float m = -INFINITY, l = 0.f;
  float4 o[WIDE] = {};
  for (int s0 = warp; s0 <= more; s0 += 4 * DE_WARPS) {  // four parts at a time
    float pm[4], pl[4];
    float4 y[4][WIDE];
#pragma unroll
    for (int x = 0; x < 4; ++x) {
      const int s = s0 + x * DE_WARPS;
      const float *p = s == 0 ? begin : rest + s * 2 * SLOT;
      pm[x] = s <= more ? p[ROWS * DP + r] : -INFINITY;
      pl[x] = s <= more ? p[ROWS * DP + ROWS + r] : 0.f;
#pragma unroll
      for (int z = 0; z < WIDE; ++z) {
        const int d = (z * WARP + lane) * 4;
        y[x][z] = s <= more && d < a.D ? *reinterpret_cast<const float4 *>(p + r * DP + d) : make_float4(0.f, 0.f, 0.f, 0.f);
      }
    }
    float top = m;
#pragma unroll
    for (int x = 0; x < 4; ++x) top = fmaxf(top, pm[x]);
    const float base = top == -INFINITY ? 0.f : top, corr = exp2f(m - base);
    m = top;
    l *= corr;
#pragma unroll
    for (int z = 0; z < WIDE; ++z) o[z] = make_float4(scaled(o[z].x, corr), scaled(o[z].y, corr), scaled(o[z].z, corr), scaled(o[z].w, corr));
#pragma unroll
    for (int x = 0; x < 4; ++x) {
      const float f = exp2f(pm[x] - base);
      l = fmaf(pl[x], f, l);
#pragma unroll
      for (int z = 0; z < WIDE; ++z)
        o[z] = make_float4(o[z].x + scaled(y[x][z].x, f), o[z].y + scaled(y[x][z].y, f), o[z].z + scaled(y[x][z].z, f), o[z].w + scaled(y[x][z].w, f));
    }
  }
#pragma unroll
  for (int z = 0; z < WIDE; ++z) so[warp][z * WARP + lane] = o[z];
  if (lane == 0) {
    sm[warp] = m;
    sl[warp] = l;
  }
  __syncthreads();
  float top = -INFINITY, sum = 0.f;
#pragma unroll
  for (int x = 0; x < DE_WARPS; ++x) top = fmaxf(top, sm[x]);
  const float base = top == -INFINITY ? 0.f : top;
  for (int d = threadIdx.x; d < a.D; d += DE_THREADS) {
    float y = 0.f;
    sum = 0.f;
#pragma unroll
    for (int x = 0; x < DE_WARPS; ++x) {
      const float f = exp2f(sm[x] - base);
      sum = fmaf(sl[x], f, sum);
      y += scaled(reinterpret_cast<const float *>(so[x])[d], f);
    }
    static_cast<T *>(a.out)[((long long)w.b * a.H + g * R + h0 + r) * a.D + d] = from_f<T>(sum == 0.f ? 0.f : y / sum);
  }
}

// How a call is dealt out.
struct DecodePlan {
  int groups, blocks, least;
  size_t scratch;
  bool split;
};
// Units of an item up to which it is not split, by what the table has room for, as the lengths are on the device: three of tokens, 192 (that
// one block reads them takes no longer than a second kernel does: 137 tokens of 12 heads, in a graph, 5.2 us whole and 9.4 split, which a table
// with room for 193 and more makes them), and units that a block gets at least where items are split (2000 tokens of 8 heads, cold: 16 us
// with two of them tokens, 18 with three, 21 with five).
constexpr int DE_WHOLE = DECODE_ITEM + 3, DE_LEAST = DECODE_ITEM + 2;
template <typename T, int DP>
static DecodePlan decode_plan(int B, int H, int G, int page, int width) {
  constexpr int ROWS = DecodeRows<T>::N;
  DecodePlan p;
  p.groups = ceil_div(H / G, ROWS);
  const long long items = (long long)B * G * p.groups, most = units_of((long long)width * page);  // units of an item
  p.split = most > DE_WHOLE;
  p.least = DE_LEAST;
  const long long resident = (long long)sm_count() * DecodeRing<T, DP>::BLOCKS, needed = (items * most + DE_LEAST - 1) / DE_LEAST;
  p.blocks = (int)(p.split ? (needed < resident ? needed : resident) : items);
  p.scratch = p.split ? (size_t)p.blocks * 2 * ROWS * (DP + 2) * 4 : 0;
  return p;
}

// A pool as TMA reads it: boxes of 128 bytes x `rows` slots of a page of a head. False: strides that TMA does not take.
template <typename T>
static bool slots_map(CUtensorMap *map, const void *p, const DecodeArgs &a, int rows) {
  // (a stride that nothing depends on can be anything)
  const auto bytes = [](long long stride, int n) { return n > 1 ? stride * (long long)sizeof(T) : 16ll; };
  const long long slot = bytes(a.pool.ld_slot, a.page), head = bytes(a.pool.ld_head, a.G), page = bytes(a.pool.ld_page, a.pages);
  for (long long s : {slot, head, page})
    if (s <= 0 || s % 16 || s >= (1ll << 40)) return false;
  const cuuint64_t dims[4] = {(cuuint64_t)a.D, (cuuint64_t)a.page, (cuuint64_t)a.G, (cuuint64_t)a.pages},
                   strides[3] = {(cuuint64_t)slot, (cuuint64_t)head, (cuuint64_t)page};
  const cuuint32_t box[4] = {128 / (cuuint32_t)sizeof(T), (cuuint32_t)rows, 1, 1}, unit[4] = {1, 1, 1, 1};
  const CUtensorMapDataType type = sizeof(T) == 4 ? CU_TENSOR_MAP_DATA_TYPE_FLOAT32
                                   : std::is_same<T, bf16>::value ? CU_TENSOR_MAP_DATA_TYPE_BFLOAT16 : CU_TENSOR_MAP_DATA_TYPE_FLOAT16;
  return encode_tiled() && encode_tiled()(map, type, 4, const_cast<void *>(p), dims, strides, box, unit, CU_TENSOR_MAP_INTERLEAVE_NONE,
                                          CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
                                          CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}

template <typename T, int DP>
static cudaError_t launch_decode(DecodeArgs a, void *scratch, cudaStream_t st) {
  using Ring = DecodeRing<T, DP>;
  static DevicePrep prep;
  const int(*unused)[4];
  cudaError_t e = prep.get(
      [&](int(&)[4]) {
        cudaError_t f = cudaFuncSetAttribute(decode_kernel<T, DP, true>, cudaFuncAttributeMaxDynamicSharedMemorySize, Ring::SMEM);
        return f != cudaSuccess ? f : cudaFuncSetAttribute(decode_kernel<T, DP, false>, cudaFuncAttributeMaxDynamicSharedMemorySize, Ring::SMEM);
      },
      unused);
  if (e != cudaSuccess) return e;
  constexpr int TOKENS = DecodeSums<T, DP>::TOKENS;
  CUtensorMap k{}, v{};
  const bool boxes = a.page % TOKENS == 0 && slots_map<T>(&k, a.k, a, TOKENS) && slots_map<T>(&v, a.v, a, TOKENS);
  const DecodePlan p = decode_plan<T, DP>(a.B, a.H, a.G, a.page, a.width);
  a.groups = p.groups;
  a.parts = p.split ? static_cast<float *>(scratch) : nullptr;
  e = djv::launch_kernel(boxes ? decode_kernel<T, DP, true> : decode_kernel<T, DP, false>, dim3(p.blocks), dim3(DE_THREADS), Ring::SMEM, st,
                         k, v, a, p.least);
  count_launch();
  if (e == cudaSuccess && p.split && p.blocks > 1) {
    e = djv::launch_kernel(decode_join_kernel<T, DP>, dim3(p.blocks - 1, a.H / a.G < DecodeRows<T>::N ? a.H / a.G : DecodeRows<T>::N),
                           dim3(DE_THREADS), 0, st, a, p.blocks, p.least);
    count_launch();
  }
  return e;
}

// f<T, DP>() for the type and the head size
template <typename F>
static auto decode_form(int dtype, int D, F f) {
  const auto of = [&](auto t) {
    using T = decltype(t);
    return D <= 64 ? f(t, std::integral_constant<int, 64>()) : D <= 128 ? f(t, std::integral_constant<int, 128>())
                                                                       : f(t, std::integral_constant<int, 256>());
  };
  return dtype == DJV_DTYPE_F16 ? of(__half()) : dtype == DJV_DTYPE_BF16 ? of(bf16()) : of(float());
}

unsigned decode_faults() {
  unsigned v = 0;
  if (cudaMemcpyFromSymbol(&v, g_decode_faults, sizeof(v)) != cudaSuccess) {
    cudaGetLastError();
    return 0;
  }
  return v;
}
unsigned decode_timeouts() {
  unsigned v = 0;
  if (cudaMemcpyFromSymbol(&v, g_decode_timeouts, sizeof(v)) != cudaSuccess) {
    cudaGetLastError();
    return 0;
  }
  return v;
}

}  // namespace djv

using namespace djv;

extern "C" size_t djv_paged_attention_scratch_bytes(int dtype, int B, int H, int G, int D, int page, int width) {
  if (!is_dtype(dtype) || B < 1 || G < 1 || H < G || D < 1 || D > 256 || page < 1 || width < 1) return 0;
  return decode_form(dtype, D, [&](auto t, auto dp) { return decode_plan<decltype(t), decltype(dp)::value>(B, H, G, page, width).scratch; });
}

extern "C" int djv_paged_attention(int dtype, void *out, const void *q, long long ldq, long long hq, const void *k_pages,
                                   const void *v_pages, long long ld_page, long long ld_head, long long ld_slot, int pages, int page,
                                   const int32_t *table, long long ld_table, int width, const long long *pos, int B, int H, int G,
                                   int D, float scale, void *scratch, size_t scratch_bytes, void *stream) {
  DJV_REQUIRE(is_dtype(dtype), "paged_attention: dtype %d", dtype);
  DJV_REQUIRE(out && q && k_pages && v_pages && table && pos, "paged_attention: null pointer");
  const int chunk = 16 / (int)dtype_bytes(dtype);
  DJV_REQUIRE(B >= 0 && G >= 1 && H >= 1 && H % G == 0 && H <= 65536 && (long long)B * H < (1ll << 30) && pages >= 1 && page >= 1 &&
                  width >= 1 && (long long)width * page < (1ll << 31) && D >= 1 && D <= 256,
              "paged_attention: B=%d H=%d G=%d D=%d pages=%d of %d, table %d wide", B, H, G, D, pages, page, width);
  DJV_REQUIRE(D % chunk == 0 && aligned16(k_pages) && aligned16(v_pages) && ld_page % chunk == 0 && ld_head % chunk == 0 &&
                  ld_slot % chunk == 0 && aligned16(q) && ldq % chunk == 0 && hq % chunk == 0 && aligned16(out),
              "paged_attention: rows start on multiples of 16 bytes");
  DJV_REQUIRE(scale == scale && scale - scale == 0.f, "paged_attention: scale %f", scale);
  if (B == 0) return DJV_OK;
  const size_t need = djv_paged_attention_scratch_bytes(dtype, B, H, G, D, page, width);
  if (scratch_bytes < need || !aligned16(scratch) || (need && !scratch)) {
    set_error("paged_attention: scratch of %zu bytes, %zu needed, 16-byte aligned", scratch_bytes, need);
    return DJV_ERR_SCRATCH;
  }
  const DecodeArgs a{out, q, k_pages, v_pages, ldq, hq, {ld_page, ld_head, ld_slot}, pages, page, divider_of(page), table, ld_table, width, pos,
                     B, H, G, D, scale, nullptr, 1};
  const cudaError_t e = decode_form(
      dtype, D, [&](auto t, auto dp) { return launch_decode<decltype(t), decltype(dp)::value>(a, scratch, static_cast<cudaStream_t>(stream)); });
  if (e != cudaSuccess) {
    cudaGetLastError();
    set_error("paged_attention: CUDA error %d (%s)", (int)e, cudaGetErrorString(e));
    return DJV_ERR_CUDA;
  }
  return check_launch("paged_attention");
}
