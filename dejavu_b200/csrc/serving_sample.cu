// Sampling of one token per row of logits: temperature, top-k, top-p, min-p, from a given random number.
//
// Entries are ordered without being sorted. (logit, index) is a 64-bit number, larger for what comes first, so that every cut is a
// threshold on it and ties need no rule of their own. A row is swept a few times (from L2 after the first):
//   1. its largest entry;  2. a histogram of 2048 equal steps of the logit, counts only;
//   3. what lies in the step of the k-th entry: collected and sorted in shared memory, which gives the threshold of top-k;
//   4. the same for top-p, where counts and the steps' borders bound the sums from both sides: the entries between the bounds are
//      collected, those outside summed;
//   5. the sum of what is kept, warp by warp in index order, and the place where the running sum passes u times it.
// If too many entries are in the way (ties), the range is cut into 2048 steps again, now of the 64-bit number, until few are left.
// Weights are 32-bit numbers with an error of at most 4e-7 (exp2f's, beside an exponent that is kept in two terms), sums 64-bit
// ones. A comparison that comes out closer than the weights' errors allow makes the row start again with 64-bit weights: the token is
// that of the 64-bit definition.
#include <math.h>
#include <string.h>

#include "serving.cuh"

namespace djv {

constexpr int SA_THREADS = 512, SA_WARPS = SA_THREADS / WARP, SA_BINS = 2048, SA_LIST = 2048;
constexpr double SA_CLOSE = 8e-7;   // what counts as close, of a sum of 32-bit weights: twice their relative error
constexpr float SA_FAR = 45.f;      // temperatures below the largest entry from where on nothing counts (e^-45 = 3e-20)

struct SampleArgs {
  long long *token;
  const void *logits;
  long long ld;
  const float *u, *temperature;
  double temperature0;
  const int *top_k;
  int top_k0;
  const float *top_p;
  double top_p0;
  const float *min_p;
  double min_p0;
  int V;
};

using u64 = unsigned long long;

// Larger for larger logits; NaN counts as -inf, -0 as 0.
__device__ __forceinline__ uint32_t order_of(float x) {
  if (x != x) x = -INFINITY;
  const uint32_t u = __float_as_uint(x + 0.f);
  return u ^ ((uint32_t)((int)u >> 31) | 0x80000000u);
}
__device__ __forceinline__ float logit_of(uint32_t key) {
  return __uint_as_float(key & 0x80000000u ? key ^ 0x80000000u : ~key);
}
constexpr uint32_t SA_NONE = 0x007fffffu;  // order_of(-inf)
__device__ __forceinline__ u64 place_of(uint32_t key, int i) { return (u64)key << 32 | (uint32_t)~i; }

struct SampleShared {
  u64 list[SA_LIST];
  unsigned count[SA_BINS];
  double mass[SA_BINS];
  double part[SA_WARPS];
  u64 wide[SA_WARPS];
  int listed;
  int found[4];
  u64 lo, hi, place;
  double sums[3];
};

// ---- what a block does together -------------------------------------------------------------------------------------
template <typename V, typename F>
__device__ __forceinline__ V block_all(V v, V *slots, F f) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) v = f(v, __shfl_xor_sync(0xffffffffu, v, o));
  __syncthreads();
  if (threadIdx.x % WARP == 0) slots[threadIdx.x / WARP] = v;
  __syncthreads();
  v = slots[0];
#pragma unroll 4
  for (int w = 1; w < SA_WARPS; ++w) v = f(v, slots[w]);
  return v;
}
__device__ __forceinline__ double block_total(double v, SampleShared &s) {
  return block_all(v, s.part, [](double a, double b) { return a + b; });
}

// f(x, index) for the row's entries from lo to hi (multiples of the chunk, or the row's end), a thread every `step`-th chunk
template <typename T, bool VEC, typename F>
__device__ __forceinline__ void sweep(const T *row, int lo, int hi, int at, int step, F f) {
  constexpr int N = VEC ? Chunk<T>::N : 1, DEEP = 4;
  int i = lo + at * N;
  if (VEC) {
    for (; i + (DEEP - 1) * step * N + N <= hi; i += DEEP * step * N) {
      uint4 v[DEEP];
#pragma unroll
      for (int d = 0; d < DEEP; ++d) v[d] = *reinterpret_cast<const uint4 *>(row + i + d * step * N);
#pragma unroll
      for (int d = 0; d < DEEP; ++d) {
        float x[N];
        unpack_chunk<T>(v[d], x);
#pragma unroll
        for (int e = 0; e < N; ++e) f(x[e], i + d * step * N + e);
      }
    }
  }
  for (; i < hi; i += step * N)
    for (int e = 0; e < N; ++e)
      if (i + e < hi) f(to_f(row[i + e]), i + e);
}

// Sorts list[0 .. n), largest first; n <= SA_LIST.
__device__ void sort_list(SampleShared &s, int n) {
  int size = 32;
  while (size < n) size *= 2;
  for (int i = n + threadIdx.x; i < size; i += SA_THREADS) s.list[i] = 0;
  __syncthreads();
  for (int k = 2; k <= size; k *= 2)
    for (int j = k / 2; j > 0; j /= 2) {
      for (int i = threadIdx.x; i < size / 2; i += SA_THREADS) {
        const int a = 2 * i - (i & (j - 1)), b = a + j;
        const u64 x = s.list[a], y = s.list[b];
        if ((x < y) == ((a & k) == 0)) {
          s.list[a] = y;
          s.list[b] = x;
        }
      }
      __syncthreads();
    }
}

// ---- one row ----------------------------------------------------------------------------------------------------------
template <typename T, bool VEC>
struct SampleRow {
  const T *row;
  int V;
  SampleShared &s;
  float top, inv;       // largest logit, steps per unit of the logit
  double temperature;
  float c_hi, c_lo;     // log2(e) / temperature
  float reach;          // entries further below the largest are dropped

  template <bool EXACT>
  __device__ __forceinline__ double weight(float x) const {
    if (x == top) return 1.0;  // (+inf among them)
    if (EXACT) return exp(((double)x - (double)top) / temperature);
    const float t = x - top, v = t - x, e = (x - (t - v)) - (top + v);  // x - top = t + e
    const float y = t * c_hi, rest = fmaf(t, c_hi, -y) + fmaf(t, c_lo, e * c_hi);
    const float w = exp2f(y);
    return fmaf(w, rest * 0.69314718f, w);
  }
  __device__ __forceinline__ bool counts(float x) const { return x >= -3.402823466e38f && !(top - x > reach); }
  __device__ __forceinline__ int bin_of(float x) const { return min(SA_BINS - 1, (int)((top - x) * inv)); }

  template <typename F>
  __device__ __forceinline__ void all(F f) const {
    sweep<T, VEC>(row, 0, V, threadIdx.x, SA_THREADS, f);
  }

  // Of the entries between places lo and hi (inclusive), those in front first: the place of entry number `rank` (from 0), or, by
  // mass, of the last entry in front of which less than `mass` lies. Cuts the range until what is left fits the list.
  template <bool EXACT, bool MASS>
  __device__ u64 narrow(u64 lo, u64 hi, int rank, double mass, double total, bool &close) {
    for (;;) {
      __syncthreads();
      if (threadIdx.x == 0) {
        s.listed = 0;
        s.lo = ~0ull;
        s.hi = 0;
      }
      __syncthreads();
      u64 first = 0, last = ~0ull;
      all([&](float x, int i) {
        const u64 p = place_of(order_of(x), i);
        if (p < lo || p > hi || !counts(x)) return;
        first = p > first ? p : first;
        last = p < last ? p : last;
        const int at = atomicAdd(&s.listed, 1);
        if (at < SA_LIST) s.list[at] = p;
      });
      __syncthreads();
      const int n = s.listed;
      if (n <= SA_LIST) break;
      hi = block_all(first, s.wide, [](u64 a, u64 b) { return a > b ? a : b; });
      lo = block_all(last, s.wide, [](u64 a, u64 b) { return a < b ? a : b; });
      int shift = 0;
      while (((hi - lo) >> shift) >= SA_BINS) ++shift;
      for (int i = threadIdx.x; i < SA_BINS; i += SA_THREADS) {
        s.count[i] = 0;
        s.mass[i] = 0;
      }
      __syncthreads();
      all([&](float x, int i) {
        const u64 p = place_of(order_of(x), i);
        if (p < lo || p > hi || !counts(x)) return;
        const int bin = (int)((hi - p) >> shift);
        if (MASS) atomicAdd(&s.mass[bin], weight<EXACT>(x));
        else atomicAdd(&s.count[bin], 1u);
      });
      __syncthreads();
      if (threadIdx.x == 0) {
        int bin = 0;
        if (MASS) {  // the last step in front of which less than `mass` lies and that holds anything
          double run = 0;
          int best = 0;
          double before = 0;
          for (; bin < SA_BINS; ++bin) {
            if (s.mass[bin] == 0) continue;
            if (bin > 0 && run >= mass) break;
            best = bin;
            before = run;
            run += s.mass[bin];
          }
          s.found[0] = best;
          s.sums[0] = before;
          // the step's borders have to be clear of the errors
          s.found[1] = !EXACT && (fabs(before - mass) <= SA_CLOSE * total || fabs(run - mass) <= SA_CLOSE * total);
        } else {
          int run = 0;
          while (bin < SA_BINS - 1 && run + (int)s.count[bin] <= rank) run += s.count[bin++];
          s.found[0] = bin;
          s.found[1] = run;
        }
      }
      __syncthreads();
      const int bin = s.found[0];
      if (MASS) {
        mass -= s.sums[0];
        close |= s.found[1] != 0;
      } else {
        rank -= s.found[1];
      }
      const u64 step = 1ull << shift, up = hi - (u64)bin * step;
      lo = up - lo >= step ? up - (step - 1) : lo;
      hi = up;
    }
    const int n = s.listed;
    sort_list(s, n);
    if (!MASS) {
      const u64 p = s.list[rank];
      __syncthreads();
      return p;
    }
    // running sums of the list's weights, a warp 32 at a time
    if (threadIdx.x < WARP) {
      double run = 0;
      u64 place = s.list[0];
      bool near = false;
      for (int i0 = 0; i0 < n; i0 += WARP) {
        const int i = i0 + threadIdx.x;
        const double w = i < n ? weight<EXACT>(logit_of((uint32_t)(s.list[i] >> 32))) : 0.0;
        double sum = w;
#pragma unroll
        for (int o = 1; o < WARP; o <<= 1) {
          const double up = __shfl_up_sync(0xffffffffu, sum, o);
          if ((int)threadIdx.x >= o) sum += up;
        }
        const double before = run + sum - w;
        const bool in = i < n && (before < mass || i == 0);
        near |= __any_sync(0xffffffffu, i < n && i > 0 && fabs(before - mass) <= SA_CLOSE * total) != 0;
        const unsigned kept = __ballot_sync(0xffffffffu, in);
        if (kept) place = s.list[i0 + 31 - __clz(kept)];
        if (kept != 0xffffffffu) break;
        run += __shfl_sync(0xffffffffu, sum, WARP - 1);
      }
      if (threadIdx.x == 0) {
        s.place = place;
        s.found[0] = near;
      }
    }
    __syncthreads();
    const u64 place = s.place;
    if (!EXACT) close |= s.found[0] != 0;
    __syncthreads();
    return place;
  }

  // The place of the last entry that top-p keeps. cut: the place of the last one that top-k keeps. counts of the steps: s.count,
  // those of the last step with any kept entry among them.
  template <bool EXACT>
  __device__ u64 nucleus(u64 cut, double p, bool &close) {
    // bounds of the running sums at the steps' borders, by warp 0
    const float width = inv > 0.f ? 1.f / inv : 0.f;
    if (threadIdx.x < WARP) {
      const int lane = threadIdx.x;
      double total_lo = 0, total_hi = 0;
      for (int b = lane; b < SA_BINS; b += WARP) {
        if (!s.count[b]) continue;
        total_hi += s.count[b] * exp2((double)c_hi * -(b * (double)width) * (1 - 1e-6));
        total_lo += s.count[b] * exp2((double)c_hi * -((b + 1) * (double)width) * (1 + 1e-6));
      }
#pragma unroll
      for (int o = 16; o > 0; o >>= 1) {
        total_lo += __shfl_xor_sync(0xffffffffu, total_lo, o);
        total_hi += __shfl_xor_sync(0xffffffffu, total_hi, o);
      }
      total_lo *= 1 - 1e-5;
      total_hi *= 1 + 1e-5;
      // first: the first step at whose end the sum can have reached p of the total; last: the first at whose end it has to have
      double run_lo = 0, run_hi = 0;
      int first = -1, last = -1, end = 0;
      for (int b0 = 0; b0 < SA_BINS && last < 0; b0 += WARP) {
        const int b = b0 + lane;
        const unsigned n = s.count[b];
        double hi = n ? n * exp2((double)c_hi * -(b * (double)width) * (1 - 1e-6)) * (1 + 1e-5) : 0.0;
        double lo = n ? n * exp2((double)c_hi * -((b + 1) * (double)width) * (1 + 1e-6)) * (1 - 1e-5) : 0.0;
#pragma unroll
        for (int o = 1; o < WARP; o <<= 1) {
          const double x = __shfl_up_sync(0xffffffffu, hi, o), y = __shfl_up_sync(0xffffffffu, lo, o);
          if (lane >= o) {
            hi += x;
            lo += y;
          }
        }
        const unsigned can = __ballot_sync(0xffffffffu, run_hi + hi >= p * total_lo), must = __ballot_sync(0xffffffffu, run_lo + lo >= p * total_hi);
        const unsigned any = __ballot_sync(0xffffffffu, n != 0);
        if (first < 0 && can) first = b0 + __ffs(can) - 1;
        if (last < 0 && must) last = b0 + __ffs(must) - 1;
        if (any) end = b0 + 31 - __clz(any);
        run_hi += __shfl_sync(0xffffffffu, hi, WARP - 1);
        run_lo += __shfl_sync(0xffffffffu, lo, WARP - 1);
      }
      if (lane == 0) {
        s.found[0] = first < 0 ? end : first;
        s.found[1] = last < 0 ? SA_BINS - 1 : last;
      }
    }
    __syncthreads();
    const int first = s.found[0], last = s.found[1];
    double in_front = 0, between = 0, behind = 0;
    u64 hi = 0, lo = ~0ull;
    all([&](float x, int i) {
      if (!counts(x)) return;
      const u64 at = place_of(order_of(x), i);
      if (at < cut) return;
      const int bin = bin_of(x);
      const double w = weight<EXACT>(x);
      if (bin < first) {
        in_front += w;
      } else if (bin > last) {
        behind += w;
      } else {
        between += w;
        hi = at > hi ? at : hi;
        lo = at < lo ? at : lo;
      }
    });
    in_front = block_total(in_front, s);
    between = block_total(between, s);
    behind = block_total(behind, s);
    hi = block_all(hi, s.wide, [](u64 a, u64 b) { return a > b ? a : b; });
    lo = block_all(lo, s.wide, [](u64 a, u64 b) { return a < b ? a : b; });
    const double total = in_front + between + behind;
    if (lo > hi) return cut;  // nothing between the bounds: no entry is dropped
    return narrow<EXACT, true>(lo, hi, 0, p * total - in_front, total, close);
  }

  // The token: the first index at which the running sum of what is kept passes u times its total.
  template <bool EXACT>
  __device__ int draw(u64 cut, double u, double min_p, bool &close) {
    const int warp = threadIdx.x / WARP, lane = threadIdx.x % WARP;
    constexpr int N = VEC ? Chunk<T>::N : 1;
    const int share = ((V + SA_WARPS - 1) / SA_WARPS + WARP * N - 1) / (WARP * N) * (WARP * N);
    const int lo = min(V, warp * share), hi = min(V, lo + share);
    auto kept = [&](float x, int i) -> double {
      if (!counts(x) || place_of(order_of(x), i) < cut) return 0.0;
      const double w = weight<EXACT>(x);
      if (min_p > 0 && w < min_p * (1 + 1e-5) && (w < min_p * (1 - 1e-5) || weight<true>(x) < min_p)) return 0.0;
      return w;
    };
    double sum = 0;
    sweep<T, VEC>(row, lo, hi, lane, WARP, [&](float x, int i) { sum += kept(x, i); });
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
    __syncthreads();
    if (lane == 0) s.part[warp] = sum;
    if (threadIdx.x == 0) s.found[0] = -1;
    __syncthreads();
    double total = 0, before = 0, target;
    for (int w = 0; w < SA_WARPS; ++w) total += s.part[w];
    target = u * total;
    int mine = SA_WARPS;  // the warp whose part the target falls into: the first whose running sum exceeds it
    int last = 0;         // the last warp that keeps anything
    for (int w = 0; w < SA_WARPS; ++w) {
      if (s.part[w] > 0) last = w;
      if (mine == SA_WARPS && before + s.part[w] > target) mine = w;
      if (mine == SA_WARPS) before += s.part[w];
    }
    if (mine == SA_WARPS) {  // (rounding: the last entry that is kept)
      mine = last;
      target = INFINITY;
      before = 0;
    }
    if (warp == mine) {
      double run = before;
      int token = -1, latest = -1;
      bool near = false;
      for (int i0 = lo; i0 < hi && token < 0; i0 += WARP) {
        const int i = i0 + lane;
        const double w = i < hi ? kept(to_f(row[i]), i) : 0.0;
        if (__ballot_sync(0xffffffffu, w > 0) == 0) continue;
        double sum = w;
#pragma unroll
        for (int o = 1; o < WARP; o <<= 1) {
          const double up = __shfl_up_sync(0xffffffffu, sum, o);
          if (lane >= o) sum += up;
        }
        const unsigned over = __ballot_sync(0xffffffffu, w > 0 && run + sum > target);
        near |= __any_sync(0xffffffffu, w > 0 && fabs(run + sum - target) <= SA_CLOSE * total) != 0;
        latest = i0 + 31 - __clz(__ballot_sync(0xffffffffu, w > 0));
        if (over) token = i0 + __ffs(over) - 1;
        run += __shfl_sync(0xffffffffu, sum, WARP - 1);
      }
      if (lane == 0) {
        s.found[0] = token >= 0 ? token : latest;
        s.found[1] = near || fabs(before - target) <= SA_CLOSE * total;
      }
    }
    __syncthreads();
    const int token = s.found[0];
    if (!EXACT && mine != SA_WARPS) close |= s.found[1] != 0;
    __syncthreads();
    return token;
  }
};

template <typename T, bool VEC>
__global__ void __launch_bounds__(SA_THREADS, 2) sample_kernel(SampleArgs a) {
  extern __shared__ __align__(16) unsigned char smem_raw[];
  SampleShared &s = *reinterpret_cast<SampleShared *>(smem_raw);
  pdl_prologue();
  const int b = blockIdx.x;
  const double temperature = a.temperature ? (double)a.temperature[b] : a.temperature0;
  const double p = a.top_p ? (double)a.top_p[b] : a.top_p0, min_p = a.min_p ? (double)a.min_p[b] : a.min_p0;
  const int k = a.top_k ? a.top_k[b] : a.top_k0;
  const double u = a.u[b];
  SampleRow<T, VEC> r{static_cast<const T *>(a.logits) + b * a.ld, a.V, s};
  u64 best = 0;
  uint32_t least = 0xffffffffu;
  r.all([&](float x, int i) {
    const uint32_t key = order_of(x);
    const u64 place = place_of(key, i);
    if (key <= SA_NONE) return;
    best = place > best ? place : best;
    least = min(least, key);
  });
  best = block_all(best, s.wide, [](u64 x, u64 y) { return x > y ? x : y; });
  const int arg = best ? (int)~(uint32_t)best : -1;
  if (arg < 0 || !(temperature > 0) || k == 1) {
    if (threadIdx.x == 0) a.token[b] = arg;
    return;
  }
  const uint32_t bottom = (uint32_t)block_all((u64)least, s.wide, [](u64 x, u64 y) { return x < y ? x : y; });
  r.top = logit_of((uint32_t)(best >> 32));
  r.temperature = temperature;
  const double c = 1.4426950408889634 / temperature;
  r.c_hi = (float)c;
  r.c_lo = (float)(c - (double)r.c_hi);
  r.reach = (float)fmin(SA_FAR * temperature, 3e38);
  const float range = fminf(r.top - logit_of(bottom), r.reach);
  r.inv = range > 0.f && range < 3e38f ? SA_BINS / range * 0.99999f : 0.f;
  const bool by_rank = k > 0 && k < a.V, by_mass = p < 1;
  bool close = false;
  u64 cut = 0;
  if (by_rank || by_mass) {
    for (int i = threadIdx.x; i < SA_BINS; i += SA_THREADS) s.count[i] = 0;
    __syncthreads();
    r.all([&](float x, int) {
      if (r.counts(x)) atomicAdd(&s.count[r.bin_of(x)], 1u);
    });
    __syncthreads();
  }
  if (by_rank) {
    if (threadIdx.x < WARP) {
      const int lane = threadIdx.x;
      int run = 0, bin = -1, before = 0;
      for (int b0 = 0; b0 < SA_BINS && bin < 0; b0 += WARP) {
        int n = s.count[b0 + lane], sum = n;
#pragma unroll
        for (int o = 1; o < WARP; o <<= 1) {
          const int up = __shfl_up_sync(0xffffffffu, sum, o);
          if (lane >= o) sum += up;
        }
        const unsigned over = __ballot_sync(0xffffffffu, run + sum >= k);
        if (over) {
          bin = b0 + __ffs(over) - 1;
          before = run + __shfl_sync(0xffffffffu, sum - n, __ffs(over) - 1);
        }
        run += __shfl_sync(0xffffffffu, sum, WARP - 1);
      }
      if (lane == 0) {
        s.found[2] = bin;
        s.found[3] = before;
      }
    }
    __syncthreads();
    const int bin = s.found[2], before = s.found[3];
    if (bin >= 0) {  // else there are fewer than k
      u64 first = 0, last = ~0ull;
      r.all([&](float x, int i) {
        if (!r.counts(x) || r.bin_of(x) != bin) return;
        const u64 at = place_of(order_of(x), i);
        first = at > first ? at : first;
        last = at < last ? at : last;
      });
      first = block_all(first, s.wide, [](u64 x, u64 y) { return x > y ? x : y; });
      last = block_all(last, s.wide, [](u64 x, u64 y) { return x < y ? x : y; });
      bool none = false;
      // (the histogram is needed again)
      cut = r.template narrow<true, false>(last, first, k - 1 - before, 0, 0, none);
      if (by_mass) {
        for (int i = threadIdx.x; i < SA_BINS; i += SA_THREADS) s.count[i] = 0;
        __syncthreads();
        r.all([&](float x, int i) {
          if (r.counts(x) && place_of(order_of(x), i) >= cut) atomicAdd(&s.count[r.bin_of(x)], 1u);
        });
        __syncthreads();
      }
    }
  }
  const u64 by_k = cut;
  if (by_mass) cut = r.template nucleus<false>(by_k, p, close);
  int token = -1;
  if (!close) token = r.template draw<false>(cut, u, min_p, close);
  if (close) {
    if (by_mass) {
      // the steps' counts may have been used up
      for (int i = threadIdx.x; i < SA_BINS; i += SA_THREADS) s.count[i] = 0;
      __syncthreads();
      r.all([&](float x, int i) {
        if (r.counts(x) && place_of(order_of(x), i) >= by_k) atomicAdd(&s.count[r.bin_of(x)], 1u);
      });
      __syncthreads();
      cut = r.template nucleus<true>(by_k, p, close);
    }
    token = r.template draw<true>(cut, u, min_p, close);
  }
  if (threadIdx.x == 0) a.token[b] = token;
}

template <typename T>
static cudaError_t launch_sample(const SampleArgs &a, int B, bool vec, cudaStream_t st) {
  constexpr int smem = sizeof(SampleShared);
  static DevicePrep prep;
  const int(*unused)[4];
  cudaError_t e = prep.get(
      [&](int(&)[4]) {
        cudaError_t f = cudaFuncSetAttribute(sample_kernel<T, true>, cudaFuncAttributeMaxDynamicSharedMemorySize, smem);
        return f != cudaSuccess ? f : cudaFuncSetAttribute(sample_kernel<T, false>, cudaFuncAttributeMaxDynamicSharedMemorySize, smem);
      },
      unused);
  if (e != cudaSuccess) return e;
  return vec ? djv::launch_kernel(sample_kernel<T, true>, dim3(B), dim3(SA_THREADS), smem, st, a)
             : djv::launch_kernel(sample_kernel<T, false>, dim3(B), dim3(SA_THREADS), smem, st, a);
}

static double double_of(long long bits) {
  double v;
  memcpy(&v, &bits, sizeof(v));
  return v;
}

}  // namespace djv

using namespace djv;

extern "C" int djv_sample(int dtype, long long *token, const void *logits, long long ld, const float *u, const float *temperature,
                          long long temperature_bits, const int32_t *top_k, int top_k_all, const float *top_p, long long top_p_bits,
                          const float *min_p, long long min_p_bits, int B, int V, void *stream) {
  DJV_REQUIRE(is_dtype(dtype), "sample: dtype %d", dtype);
  DJV_REQUIRE(token && logits && u, "sample: null pointer");
  DJV_REQUIRE(B >= 0 && V >= 1 && V <= (1 << 30) && ld >= V, "sample: B=%d V=%d ld=%lld", B, V, ld);
  const SampleArgs a{token, logits, ld, u, temperature, double_of(temperature_bits), top_k, top_k_all, top_p, double_of(top_p_bits),
                     min_p, double_of(min_p_bits), V};
  DJV_REQUIRE((temperature || (a.temperature0 >= 0 && a.temperature0 < 1e30)) && (top_k || top_k_all >= 0) && (top_p || a.top_p0 >= 0) &&
                  (min_p || (a.min_p0 >= 0 && a.min_p0 <= 1)),
              "sample: temperature %g, top_k %d, top_p %g, min_p %g", a.temperature0, top_k_all, a.top_p0, a.min_p0);
  if (B == 0) return DJV_OK;
  const bool vec = aligned16(logits) && ld % (16 / (int)dtype_bytes(dtype)) == 0;
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  const cudaError_t e = dtype == DJV_DTYPE_F16    ? launch_sample<__half>(a, B, vec, st)
                        : dtype == DJV_DTYPE_BF16 ? launch_sample<bf16>(a, B, vec, st)
                                                  : launch_sample<float>(a, B, vec, st);
  if (e != cudaSuccess) {
    cudaGetLastError();
    set_error("sample: CUDA error %d (%s)", (int)e, cudaGetErrorString(e));
    return DJV_ERR_CUDA;
  }
  count_launch();
  return check_launch("sample");
}
