// What the prefill kernels share: their arguments, where a tile's rows are, and the join of a tile's parts.
#pragma once

#include <algorithm>
#include <climits>

#include "paged_read.cuh"

namespace bpt {

struct PrefillArgs {
  PagedSource src;
  const void* q;  // [T, Hq, D], f16 or bf16
  int q_dtype;
  int64_t q_st, q_sh;
  const int32_t* cu;           // [B + 1]: sequence b's new tokens are rows cu[b] .. cu[b + 1] - 1 of q
  const int32_t* lengths;      // [B]: tokens in the cache, the new ones included
  const int32_t* positions;    // [T] or null: a new token's position; null: the new tokens are the last of their sequence
  const int32_t* key_starts;   // [T] or null
  const int32_t* prefix_lens;  // [B] or null
  const float* slopes;         // [Hq] or null
  float softcap, sm_scale;
  int window;
  int T, B, Hq, D, rep;
  int split, n_splits;
  void* out;  // [T, Hq, D] in q's type
  int* part_count;  // [tiles, Hkv]: the parts that a tile was cut into (1: it is in out already)
  float* part_out;  // [tiles, Hkv, n_splits, rows, D]
  float* part_lse;  // [tiles, Hkv, n_splits, rows], base 2
};

constexpr int kPrefillTcRows = 128;  // packed rows per CTA of the tensor-core kernel
int prefill_tc(const PrefillArgs& a, int kind, int64_t tiles, int flags, cudaStream_t stream);

// A tile of packed rows (token * rep + head) of one sequence.
struct TileAt {
  int b;        // the sequence, -1 where the grid has more tiles than there are
  int token0;   // its first new token (a row of q)
  int tokens;   // how many it has
  int row0;     // the tile's first packed row
};

// The `x`-th tile of `rows` packed rows, the longest-reaching of every sequence first (under a causal mask they take
// longest). Every warp searches on its own: 32 sequences at a time.
__device__ __forceinline__ TileAt find_tile(const PrefillArgs& a, int rows, int x) {
  const int lane = threadIdx.x & 31;
  int seen = 0;
  for (int b0 = 0; b0 < a.B; b0 += 32) {
    const int b = b0 + lane;
    int start = 0, n = 0;
    if (b < a.B) {
      start = a.cu[b];
      n = a.cu[b + 1] - start;
      if (start < 0 || n < 0 || n > a.T - start) n = 0;  // offsets that do not fit q: nothing is computed for them
    }
    const int mine = (n * a.rep + rows - 1) / rows;
    int upto = mine;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const int v = __shfl_up_sync(0xffffffffu, upto, o);
      if (lane >= o) upto += v;
    }
    const unsigned hit = __ballot_sync(0xffffffffu, seen + upto > x);
    if (hit) {
      const int w = __ffs(hit) - 1;
      TileAt at;
      at.b = b0 + w;
      at.token0 = __shfl_sync(0xffffffffu, start, w);
      at.tokens = __shfl_sync(0xffffffffu, n, w);
      const int tiles = __shfl_sync(0xffffffffu, mine, w);
      const int before = seen + __shfl_sync(0xffffffffu, upto, w) - tiles;
      at.row0 = (tiles - 1 - (x - before)) * rows;
      return at;
    }
    seen += __shfl_sync(0xffffffffu, upto, 31);
  }
  return TileAt{-1, 0, 0, 0};
}

// A sequence's length, cut to what its table has pages for.
__device__ __forceinline__ int sequence_length(const PrefillArgs& a, int b, bool tells) {
  const int room = int(min(int64_t(a.src.bt_width) << a.src.bs_log2, int64_t(1) << 30));
  const int len = a.lengths[b];
  if (len > room && tells) record_error(kDevErrBlockIndex);
  return min(len, room);
}

struct RowAt {
  int64_t q, out;  // element offsets of its query and its output, -1 for a row past the sequence's end
  int code;        // the same row counted from its tile's first token and head: tokens << 16 | heads, -1 for none
  int pos, lo, hi;
  float slope;  // minus the head's slope, in base 2
};

__device__ __forceinline__ RowAt row_at(const PrefillArgs& a, const TileAt& at, int r, int hk, int len) {
  RowAt x;
  const int t = r / a.rep, h = hk * a.rep + r - t * a.rep;
  if (t >= at.tokens) return RowAt{-1, -1, -1, 0, 0, 0, 0.f};
  const int token = at.token0 + t;
  x.q = int64_t(token) * a.q_st + int64_t(h) * a.q_sh;
  x.out = (int64_t(token) * a.Hq + h) * a.D;
  x.code = ((t - at.row0 / a.rep) << 16) | (r - t * a.rep);
  x.pos = a.positions ? min(max(a.positions[token], -1), 1 << 30) : len - at.tokens + t;
  x.lo = a.key_starts ? max(a.key_starts[token], 0) : 0;
  if (a.window > 0) x.lo = max(x.lo, x.pos - a.window + 1);
  x.hi = x.pos + 1;
  if (a.prefix_lens) x.hi = max(x.hi, a.prefix_lens[at.b]);
  x.hi = min(x.hi, len);
  x.slope = a.slopes ? -a.slopes[h] * kLog2e : 0.f;
  return x;
}

__device__ __forceinline__ float load_16(const void* p, int dtype, int64_t i) {
  if (dtype == BPT_DTYPE_F16) return __half2float(static_cast<const __half*>(p)[i]);
  return __bfloat162float(static_cast<const __nv_bfloat16*>(p)[i]);
}
__device__ __forceinline__ void store_16(void* p, int dtype, int64_t i, float v) {
  if (dtype == BPT_DTYPE_F16) static_cast<__half*>(p)[i] = __float2half_rn(v);
  else static_cast<__nv_bfloat16*>(p)[i] = __float2bfloat16_rn(v);
}

}  // namespace bpt
