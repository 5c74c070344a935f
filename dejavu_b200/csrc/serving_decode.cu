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
// arrive in a ring per warp by 16-byte asynchronous copies (any page size, any strides), swizzled for ldmatrix; the page of a tile is
// looked up a tile ahead. fp16 and bf16 go through mma.sync, 16 query heads x 16 tokens: tcgen05 would have to pad the heads to
// 64 or 128 rows, and the tensor work is a small part of the time either way. The weights enter the second product as two terms
// of the cache's type, hi + lo, so that they keep 16 (bf16) or 22 bits. fp32 goes through the CUDA cores, 4 heads at a time.
#include <math.h>
#include <type_traits>

#include "mma.cuh"
#include "pairs.cuh"
#include "serving.cuh"

namespace djv {

__device__ unsigned g_decode_faults;

constexpr int DE_WARPS = 4, DE_THREADS = DE_WARPS * WARP;

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
  float *parts;  // two slots for each block: of the item that it ends and of the one that it begins; NULL: no item is split
  int groups;    // groups of query heads that share a key/value head
};

// Tokens of sequence b.
__device__ __forceinline__ long long decode_tokens(const DecodeArgs &a, int b) {
  const long long n = a.pos[b] + 1, room = (long long)a.width * a.page;
  return n < 0 ? 0 : (n > room ? room : n);
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

template <typename T, int DP>
__device__ __forceinline__ uint32_t tile_offset(int row, int chunk) {  // of a 16-byte chunk in a tile
  return (uint32_t)(row * DP * (int)sizeof(T) + ((chunk ^ (row & 7)) << 4));
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
  uint32_t q[DP / 16][4];
  float o[DP / 8][4], m[2], l[2];

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
  __device__ __forceinline__ void tile(uint32_t k_sm, uint32_t v_sm, unsigned seen, float c, int D) {
    const int lane = threadIdx.x % WARP, t = lane % 4;
    float s[2][4] = {};
#pragma unroll
    for (int k = 0; k < DP / 16; ++k) {
      if (k * 16 >= D) break;
      uint32_t b[4];
      ldmatrix_x4(b, k_sm + tile_offset<T, DP>((lane >> 4) * 8 + lane % 8, k * 2 + ((lane >> 3) & 1)));
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
      const float base = top == -INFINITY ? 0.f : top;
      corr[r] = exp2_approx(m[r] - base);
      m[r] = top;
#pragma unroll
      for (int n = 0; n < 2; ++n)
#pragma unroll
        for (int e = 2 * r; e < 2 * r + 2; ++e) s[n][e] = exp2_approx(s[n][e] - base);
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
      hi[e] = pair_of<T>(x, y);
      const float2 h = floats_of<T>(hi[e]);
      lo[e] = pair_of<T>(x - h.x, y - h.y);
    }
#pragma unroll
    for (int i = 0; i < DP / 16; ++i) {
      if (i * 16 >= D) break;
      uint32_t b[4];
      ldmatrix_x4_trans(b, v_sm + tile_offset<T, DP>(((lane >> 3) & 1) * 8 + lane % 8, i * 2 + (lane >> 4)));
      mma_m16n8k16_t<T>(o[2 * i], hi[0], hi[1], hi[2], hi[3], b[0], b[1]);
      mma_m16n8k16_t<T>(o[2 * i + 1], hi[0], hi[1], hi[2], hi[3], b[2], b[3]);
      mma_m16n8k16_t<T>(o[2 * i], lo[0], lo[1], lo[2], lo[3], b[0], b[1]);
      mma_m16n8k16_t<T>(o[2 * i + 1], lo[0], lo[1], lo[2], lo[3], b[2], b[3]);
    }
  }
  // sums (rows, DP), and the maxima and sums of the rows
  __device__ __forceinline__ void store(float *sums, float *sm, float *sl) {
    const int lane = threadIdx.x % WARP, g = lane / 4, t = lane % 4;
#pragma unroll
    for (int r = 0; r < 2; ++r) {
      l[r] += __shfl_xor_sync(0xffffffffu, l[r], 1);
      l[r] += __shfl_xor_sync(0xffffffffu, l[r], 2);
      if (t == 0) {
        sm[g + r * 8] = m[r];
        sl[g + r * 8] = l[r];
      }
#pragma unroll
      for (int i = 0; i < DP / 8; ++i)
        *reinterpret_cast<float2 *>(sums + (g + r * 8) * DP + i * 8 + t * 2) = make_float2(o[i][2 * r], o[i][2 * r + 1]);
    }
  }
};
template <int DP>
struct DecodeSums<bf16, DP> : MmaSums<bf16, DP> {};
template <int DP>
struct DecodeSums<__half, DP> : MmaSums<__half, DP> {};

// fp32: for the scores a lane has a token and every PARTS-th chunk of it, for the values DP / 32 dimensions
template <int DP>
struct DecodeSums<float, DP> {
  static constexpr int TOKENS = DP > 128 ? 8 : 16, PARTS = WARP / TOKENS, W = DP / 32;
  const float *query;
  long long hq;
  int rows;
  float o[4][W], m[4], l[4];

  __device__ __forceinline__ void start(const float *q, long long h, int n, int) {
    query = q;
    hq = h;
    rows = n;
#pragma unroll
    for (int r = 0; r < 4; ++r) {
      m[r] = -INFINITY;
      l[r] = 0.f;
#pragma unroll
      for (int i = 0; i < W; ++i) o[r][i] = 0.f;
    }
  }
  __device__ __forceinline__ static float4 at(uint32_t sm) {
    float4 v;
    asm volatile("ld.shared.v4.f32 {%0,%1,%2,%3}, [%4];" : "=f"(v.x), "=f"(v.y), "=f"(v.z), "=f"(v.w) : "r"(sm) : "memory");
    return v;
  }
  __device__ __forceinline__ void tile(uint32_t k_sm, uint32_t v_sm, unsigned seen, float c, int D) {
    const int lane = threadIdx.x % WARP, token = lane % TOKENS, part = lane / TOKENS;
    float s[4] = {};
    for (int ch = part; ch * 4 < D; ch += PARTS) {
      const float4 k = at(k_sm + tile_offset<float, DP>(token, ch));
#pragma unroll
      for (int r = 0; r < 4; ++r) {
        if (r >= rows) break;
        const float4 q = __ldg(reinterpret_cast<const float4 *>(query + r * hq + ch * 4));
        s[r] = fmaf(q.x, k.x, fmaf(q.y, k.y, fmaf(q.z, k.z, fmaf(q.w, k.w, s[r]))));
      }
    }
#pragma unroll
    for (int r = 0; r < 4; ++r) {
      if (r >= rows) break;
#pragma unroll
      for (int x = TOKENS; x < WARP; x <<= 1) s[r] += __shfl_xor_sync(0xffffffffu, s[r], x);
      s[r] = (seen >> token) & 1 ? s[r] * c : -INFINITY;
      float top = s[r];
#pragma unroll
      for (int x = TOKENS / 2; x > 0; x >>= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, x));
      top = fmaxf(top, m[r]);
      const float base = top == -INFINITY ? 0.f : top, corr = exp2f(m[r] - base);
      m[r] = top;
      s[r] = exp2f(s[r] - base);
      l[r] = l[r] * corr + (part == 0 ? s[r] : 0.f);
#pragma unroll
      for (int i = 0; i < W; ++i) o[r][i] *= corr;
    }
#pragma unroll
    for (int t = 0; t < TOKENS; ++t) {
      float p[4];
#pragma unroll
      for (int r = 0; r < 4; ++r) p[r] = __shfl_sync(0xffffffffu, s[r], t);
#pragma unroll
      for (int i = 0; i < W; ++i) {
        float v;
        const int d = i * WARP + lane;
        asm volatile("ld.shared.f32 %0, [%1];" : "=f"(v) : "r"(v_sm + tile_offset<float, DP>(t, d / 4) + (d % 4) * 4) : "memory");
#pragma unroll
        for (int r = 0; r < 4; ++r) o[r][i] = fmaf(p[r], v, o[r][i]);
      }
    }
  }
  __device__ __forceinline__ void store(float *sums, float *sm, float *sl) {
    const int lane = threadIdx.x % WARP;
#pragma unroll
    for (int r = 0; r < 4; ++r) {
      l[r] = warp_sum(l[r]);
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
  static constexpr int SMEM = DE_WARPS * STAGES * 2 * TILE;
};

template <typename T, int DP>
__global__ void __launch_bounds__(DE_THREADS, DecodeRing<T, DP>::BLOCKS) decode_kernel(DecodeArgs a, int least) {
  using Sums = DecodeSums<T, DP>;
  using Ring = DecodeRing<T, DP>;
  constexpr int ROWS = DecodeRows<T>::N, TOKENS = Sums::TOKENS, STAGES = Ring::STAGES, TILE = Ring::TILE;
  constexpr int N = Chunk<T>::N, CHUNKS = DP / N;                              // of a row
  constexpr int AT_ONCE = CHUNKS >= WARP ? 1 : WARP / CHUNKS, WIDE = CHUNKS > WARP ? CHUNKS / WARP : 1;
  extern __shared__ __align__(128) unsigned char ring[];
  __shared__ float sm[DE_WARPS][ROWS], sl[DE_WARPS][ROWS];
  __shared__ long long slots[DE_WARPS + 2];
  const int tid = threadIdx.x, lane = tid % WARP, warp = tid / WARP;
  pdl_prologue();
  const int share = a.G * a.groups, R = a.H / a.G;
  long long x, end, base, units, tokens;
  int b;
  long long mine = 0;  // first unit of this block
  if (a.parts == nullptr) {  // an item each
    b = blockIdx.x / share;
    tokens = decode_tokens(a, b);
    units = units_of(tokens);
    base = 0;
    x = (blockIdx.x - (long long)b * share) * units;
    end = x + units;
  } else {
    long long per;
    const DecodePlace w = decode_locate(a, [&](long long total) {
      per = units_per_block(total, gridDim.x, least);
      return blockIdx.x * per;
    }, slots);
    x = mine = blockIdx.x * per;
    end = x + per < w.total ? x + per : w.total;
    if (x >= end || w.b < 0) return;
    b = w.b;
    base = w.base;
    tokens = decode_tokens(a, b);
    units = units_of(tokens);
  }
  if (tid == 0 && a.pos[b] >= (long long)a.width * a.page && x == base) atomicAdd(&g_decode_faults, 1u);
  const uint32_t warp_ring = smem_addr(ring) + warp * STAGES * 2 * TILE;
  float *warp_sums = reinterpret_cast<float *>(ring + warp * STAGES * 2 * TILE);
  const float c = a.scale * 1.4426950408889634f;

  while (x < end) {
    const DecodePart part = decode_part(x, end, base, units);
    const int g = (int)(part.item / a.groups), h0 = (int)(part.item % a.groups) * ROWS, rows = min(ROWS, R - h0), h = g * R + h0;
    const long long t0 = part.from * DECODE_UNIT, t1 = min(tokens, part.to * DECODE_UNIT);
    const PageMap map{a.table + b * a.ld_table, a.width, a.page, a.pages};
    const T *k = static_cast<const T *>(a.k) + g * a.pool.ld_head, *v = static_cast<const T *>(a.v) + g * a.pool.ld_head;
    const int tiles = t1 > t0 ? (int)((t1 - t0 + DE_WARPS * TOKENS - 1) / (DE_WARPS * TOKENS)) : 0;
    auto first_of = [&](int i) { return t0 + (long long)(i * DE_WARPS + warp) * TOKENS; };
    // where the row of the lane's token of tile i is (lanes beyond the tokens repeat them), or -1
    auto row_of = [&](int i) -> long long {
      const long long t = first_of(i) + lane % TOKENS;
      if (i >= tiles || t >= t1) return -1;
      int slot;
      const long long page = page_of(map, t, slot);
      if (page != NO_PAGE) return page * a.pool.ld_page + slot * a.pool.ld_slot;
      if (part.item == 0 && lane < TOKENS && (slot == 0 || lane == 0)) atomicAdd(&g_decode_faults, 1u);
      return -1;
    };
    unsigned seen[STAGES];
    auto load = [&](int i, long long row, unsigned &bits) {
      bits = __ballot_sync(0xffffffffu, row >= 0) & (TOKENS == 32 ? 0xffffffffu : (1u << TOKENS) - 1);
      if (i < tiles) {
        const uint32_t dst = warp_ring + i % STAGES * 2 * TILE;
#pragma unroll
        for (int p = 0; p < TOKENS / AT_ONCE; ++p) {
          const int r = p * AT_ONCE + (CHUNKS >= WARP ? 0 : lane / CHUNKS);
          const long long at = __shfl_sync(0xffffffffu, row, r);
#pragma unroll
          for (int y = 0; y < WIDE; ++y) {
            const int ch = CHUNKS >= WARP ? y * WARP + lane : lane % CHUNKS;
            const bool ok = at >= 0 && ch * N < a.D;
            const uint32_t to = dst + tile_offset<T, DP>(r, ch);
            cp_async16_zfill(to, ok ? k + at + ch * N : k, ok ? 16 : 0);
            cp_async16_zfill(to + TILE, ok ? v + at + ch * N : v, ok ? 16 : 0);
          }
        }
      }
      cp_async_commit();
    };
    Sums sums;
    long long next = row_of(0);
    sums.start(static_cast<const T *>(a.q) + b * a.ldq + h * a.hq, a.hq, rows, a.D);
#pragma unroll
    for (int i = 0; i < STAGES - 1; ++i) {
      load(i, next, seen[i]);
      next = row_of(i + 1);
    }
    for (int i0 = 0; i0 < tiles; i0 += STAGES) {
#pragma unroll
      for (int y = 0; y < STAGES; ++y) {
        const int i = i0 + y;
        if (i >= tiles) break;
        cp_async_wait<STAGES - 2>();
        __syncwarp();
        load(i + STAGES - 1, next, seen[(y + STAGES - 1) % STAGES]);
        next = row_of(i + STAGES);
        if (seen[y]) sums.tile(warp_ring + y * 2 * TILE, warp_ring + y * 2 * TILE + TILE, seen[y], c, a.D);
        __syncwarp();
      }
    }
    cp_async_wait<0>();
    __syncwarp();
    sums.store(warp_sums, sm[warp], sl[warp]);
    __syncthreads();
    const bool whole = part.from == 0 && part.to == units;
    // the slot of a part: 1 of an item that begins here, 0 of one that began in a block before
    float *slot = whole ? nullptr : a.parts + (blockIdx.x * 2 + (part.from == 0 ? 1 : 0)) * (long long)(ROWS * (DP + 2));
    for (int i = tid; i < rows * (DP / 4); i += DE_THREADS) {
      const int r = i / (DP / 4), d = i % (DP / 4) * 4;
      if (d >= a.D) continue;
      float top = -INFINITY, sum = 0.f;
#pragma unroll
      for (int w = 0; w < DE_WARPS; ++w) top = fmaxf(top, sm[w][r]);
      const float down = top == -INFINITY ? 0.f : top;
      float4 o = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
      for (int w = 0; w < DE_WARPS; ++w) {
        const float f = exp2f(sm[w][r] - down);
        const float4 y = *reinterpret_cast<const float4 *>(reinterpret_cast<const float *>(ring + w * STAGES * 2 * TILE) + r * DP + d);
        sum += sl[w][r] * f;
        o.x += y.x * f;
        o.y += y.y * f;
        o.z += y.z * f;
        o.w += y.w * f;
      }
      if (whole) {
        const float inv = sum == 0.f ? 0.f : 1.f / sum;
        T *out = static_cast<T *>(a.out) + ((long long)b * a.H + h + r) * a.D + d;
        T r4[4] = {from_f<T>(o.x * inv), from_f<T>(o.y * inv), from_f<T>(o.z * inv), from_f<T>(o.w * inv)};
        if (sizeof(T) == 4) *reinterpret_cast<uint4 *>(out) = *reinterpret_cast<uint4 *>(r4);
        else *reinterpret_cast<uint2 *>(out) = *reinterpret_cast<uint2 *>(r4);
      } else {
        *reinterpret_cast<float4 *>(slot + r * DP + d) = o;
        if (d == 0) {
          slot[ROWS * DP + r] = top;
          slot[ROWS * DP + ROWS + r] = sum;
        }
      }
    }
    __syncthreads();
    x += part.to - part.from;
    if (x < end && x == base + units * share) {
      base = x;
      ++b;
      tokens = decode_tokens(a, b);
      units = units_of(tokens);
      if (tid == 0 && a.pos[b] >= (long long)a.width * a.page) atomicAdd(&g_decode_faults, 1u);
    }
  }
  (void)mine;
}

// Joins the parts of the item that begins in block blockIdx.x of `blocks` and ends in a later one, if there is one.
template <typename T, int DP>
__global__ void __launch_bounds__(DE_THREADS) decode_join_kernel(DecodeArgs a, int blocks, int least) {
  constexpr int ROWS = DecodeRows<T>::N;
  constexpr long long SLOT = ROWS * (DP + 2);
  __shared__ long long slots[DE_WARPS + 2];
  pdl_prologue();
  long long per;
  const int share = a.G * a.groups, R = a.H / a.G;
  const DecodePlace w = decode_locate(a, [&](long long total) {
    per = units_per_block(total, blocks, least);
    return (blockIdx.x + 1) * per - 1;
  }, slots);
  const long long last = (blockIdx.x + 1) * per - 1;  // this block's last unit
  if (last + 1 >= w.total || w.b < 0) return;
  const long long units = units_of(decode_tokens(a, w.b)), item = (last - w.base) / units, from = w.base + item * units, to = from + units;
  if (to == last + 1 || from < blockIdx.x * per) return;  // it ends here, or began in a block before
  const int end = (int)((to - 1) / per);
  const int g = (int)(item / a.groups), h0 = (int)(item % a.groups) * ROWS, rows = min(ROWS, R - h0);
  const float *begin = a.parts + (blockIdx.x * 2 + 1) * SLOT, *rest = a.parts + (blockIdx.x + 1) * 2 * SLOT;
  const int more = end - blockIdx.x;  // slots after the first, 2 * SLOT apart
  for (int i = threadIdx.x; i < rows * (DP / 4); i += DE_THREADS) {
    const int r = i / (DP / 4), d = i % (DP / 4) * 4;
    if (d >= a.D) continue;
    float top = begin[ROWS * DP + r];
    for (int s = 0; s < more; ++s) top = fmaxf(top, rest[s * 2 * SLOT + ROWS * DP + r]);
    const float down = top == -INFINITY ? 0.f : top;
    float4 o = make_float4(0.f, 0.f, 0.f, 0.f);
    float sum = 0.f;
    for (int s = -1; s < more; ++s) {
      const float *p = s < 0 ? begin : rest + s * 2 * SLOT;
      const float f = exp2f(p[ROWS * DP + r] - down);
      const float4 y = *reinterpret_cast<const float4 *>(p + r * DP + d);
      sum += p[ROWS * DP + ROWS + r] * f;
      o.x += y.x * f;
      o.y += y.y * f;
      o.z += y.z * f;
      o.w += y.w * f;
    }
    const float inv = sum == 0.f ? 0.f : 1.f / sum;
    T *out = static_cast<T *>(a.out) + ((long long)w.b * a.H + g * R + h0 + r) * a.D + d;
    T r4[4] = {from_f<T>(o.x * inv), from_f<T>(o.y * inv), from_f<T>(o.z * inv), from_f<T>(o.w * inv)};
    if (sizeof(T) == 4) *reinterpret_cast<uint4 *>(out) = *reinterpret_cast<uint4 *>(r4);
    else *reinterpret_cast<uint2 *>(out) = *reinterpret_cast<uint2 *>(r4);
  }
}

// How a call is dealt out.
struct DecodePlan {
  int groups, blocks, least;
  size_t scratch;
  bool split;
};
constexpr int DE_LEAST = 4;  // units of a block, where items are split
template <typename T, int DP>
static DecodePlan decode_plan(int B, int H, int G, int page, int width) {
  constexpr int ROWS = DecodeRows<T>::N;
  DecodePlan p;
  p.groups = ceil_div(H / G, ROWS);
  const long long items = (long long)B * G * p.groups, most = units_of((long long)width * page);  // units of an item
  p.split = most > DE_LEAST;
  p.least = DE_LEAST;
  const long long resident = (long long)sm_count() * DecodeRing<T, DP>::BLOCKS, needed = (items * most + DE_LEAST - 1) / DE_LEAST;
  p.blocks = (int)(p.split ? (needed < resident ? needed : resident) : items);
  p.scratch = p.split ? (size_t)p.blocks * 2 * ROWS * (DP + 2) * 4 : 0;
  return p;
}

template <typename T, int DP>
static cudaError_t launch_decode(DecodeArgs a, void *scratch, cudaStream_t st) {
  static DevicePrep prep;
  const int(*unused)[4];
  cudaError_t e = prep.get(
      [&](int(&)[4]) { return cudaFuncSetAttribute(decode_kernel<T, DP>, cudaFuncAttributeMaxDynamicSharedMemorySize, DecodeRing<T, DP>::SMEM); },
      unused);
  if (e != cudaSuccess) return e;
  const DecodePlan p = decode_plan<T, DP>(a.B, a.H, a.G, a.page, a.width);
  a.groups = p.groups;
  a.parts = p.split ? static_cast<float *>(scratch) : nullptr;
  e = djv::launch_kernel(decode_kernel<T, DP>, dim3(p.blocks), dim3(DE_THREADS), DecodeRing<T, DP>::SMEM, st, a, p.least);
  count_launch();
  if (e == cudaSuccess && p.split && p.blocks > 1) {
    e = djv::launch_kernel(decode_join_kernel<T, DP>, dim3(p.blocks - 1), dim3(DE_THREADS), 0, st, a, p.blocks, p.least);
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
  const DecodeArgs a{out, q, k_pages, v_pages, ldq, hq, {ld_page, ld_head, ld_slot}, pages, page, table, ld_table, width, pos,
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
