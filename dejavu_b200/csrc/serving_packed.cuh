// Packed prompts: which rows a block takes.
#pragma once
#include "serving.cuh"

namespace djv {

struct PackedArgs {
  void *out;
  const void *q, *k, *v;
  long long ldq, hq, ldk, hk, ldv, hv;
  const int *cu;
  int B, T, H, G, D;
  float scale;
  int keep_rest;
};

// the tensor-core form: fp16 and bf16, rows that TMA can read, results that start on 16 bytes
bool packed_tc_supported(int dtype, const PackedArgs &a);
int packed_tc(int dtype, const PackedArgs &a, cudaStream_t st);

struct PackedTile {
  int first, q0, rows;  // the sequence's first row, the tile's first query in it, its queries (<= 0: no tile)
  int rest;             // 1: rows of no sequence
  int b;                // the sequence
};

// Tiles of Q rows that B sequences of T rows in all can make, those of no sequence among them.
template <int Q>
inline int packed_tiles(int T, int B) { return T / Q + B + 2 < T + 2 ? T / Q + B + 2 : T + 2; }

// Tiles of Q rows that sequences from .. to - 1 make. Whole warp.
template <int Q>
__device__ __forceinline__ int packed_total(const PackedArgs &a, int from, int to) {
  int t = 0;
  for (int b = from + (int)(threadIdx.x % WARP); b < to; b += WARP) {
    const int lo = max(0, min(a.cu[b], a.T));
    t += (max(0, min(a.cu[b + 1], a.T) - lo) + Q - 1) / Q;
  }
  return __reduce_add_sync(0xffffffffu, t);
}

// Tile number `index`: tiles of the sequences in order, then of the rows in front of the first and behind the last. from, seen: a sequence
// that the tile is not in front of, and the tiles before that. Whole warp. Whatever cu holds, rows are within 0 .. T - 1.
template <int Q>
__device__ __forceinline__ PackedTile packed_tile(const PackedArgs &a, int index, int from = 0, int seen = 0) {
  const int lane = threadIdx.x % WARP;
  for (int b0 = from; b0 < a.B; b0 += WARP) {
    const int b = b0 + lane;
    int lo = 0, n = 0;
    if (b < a.B) {
      lo = max(0, min(a.cu[b], a.T));
      n = max(0, min(a.cu[b + 1], a.T) - lo);
    }
    const int t = (n + Q - 1) / Q;
    int s = t;
#pragma unroll
    for (int o = 1; o < WARP; o <<= 1) {
      const int up = __shfl_up_sync(0xffffffffu, s, o);
      if (lane >= o) s += up;
    }
    const unsigned here = __ballot_sync(0xffffffffu, index < seen + s);
    if (here) {
      const int who = __ffs(here) - 1;
      const int first = __shfl_sync(0xffffffffu, lo, who), rows = __shfl_sync(0xffffffffu, n, who);
      const int before = seen + __shfl_sync(0xffffffffu, s - t, who), q0 = (index - before) * Q;
      return {first, q0, min(Q, rows - q0), 0, b0 + who};
    }
    seen += __shfl_sync(0xffffffffu, s, WARP - 1);
  }
  const int head = max(0, min(a.cu[0], a.T)), tail = max(0, min(a.cu[a.B], a.T));
  const long long at = (long long)(index - seen) * Q;
  const int in_head = (head + Q - 1) / Q * Q;
  if (at < in_head) return {0, (int)at, min(Q, head - (int)at), 1, -1};
  const long long left = a.T - tail - (at - in_head);
  if (left <= 0) return {0, 0, 0, 1, -1};
  return {tail, (int)(at - in_head), left < Q ? (int)left : Q, 1, -1};
}

}  // namespace djv
