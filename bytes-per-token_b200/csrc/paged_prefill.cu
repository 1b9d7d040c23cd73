// Prefill attention over a paged cache of any format: the new tokens of a ragged batch attend over their sequences' pages, with
// score caps, distance bias, sliding windows, documents (a first visible key per token) and a shared prefix.
//
//   s_j = cap tanh(scale q.k_j / cap) - slope |p - j|,  out = sum_j softmax(s)_j v_j  over  lo <= j < hi,
//   lo = max(0, start, p - window + 1), hi = min(length, max(p + 1, prefix));  no visible key gives 0.
//
// One pass over the keys with the running maximum and sum. The query heads of a KV head are packed with their tokens into
// rows (row = token * rep + head), so every key and value brought in serves all of them; a row carries its own interval
// [lo, hi), and a tile of rows visits only the keys between its smallest lo and largest hi.
//
// Every format but int8 takes csrc/paged_prefill_tc.cu. The kernel here serves int8 pages, whose scale per key goes on the
// scores (a factor per column of S) and on the probabilities (a factor per column of P), so that the codes themselves are the
// operands. A power of two per row keeps a row's largest product of a probability and a scale in f16's range however small
// the values are. It multiplies with mma.sync: 64 rows per CTA (16 per warp), 64 keys per step, two cp.async stages. It is bound by
// the latency of the legacy products and the codes' conversion at 8 warps an SM (no pipe above 19%): twelve ragged prompts, 16 + 8
// heads of 128, 676 us (B200), where the tcgen05 kernel takes 124 over bf16 pages. This file also holds, for both kernels, the plan and the join: where there
// are few tiles, each takes several CTAs, with a part of its keys each, and a second kernel, launched dependently, joins them.
#include "paged_prefill.cuh"

namespace bpt {
namespace {

constexpr int kWarps = 4;
constexpr int kThreads = 32 * kWarps;
constexpr int kRows = 16 * kWarps;
constexpr int kKeys = 64;

constexpr int KIND = BPT_KV_INT8;

template <int D>
struct PrefillShape {
  static constexpr int RB = D * kElemBytes<KIND>;
  static constexpr int kScaleBytes = kKeys * 4;                     // 16 K then 16 V scales (fp16) per 16 keys
  static constexpr int kStage = 2 * kKeys * RB + kScaleBytes + 16;  // keys, values, scales, a flag per 16 keys
  static constexpr int kQ = kWarps * (D / 16) * 32 * 16;            // the q fragments
  static constexpr int kStages = 2;
  static constexpr int kSmem = kStages * kStage + kQ;
};

template <int D>
__global__ void __launch_bounds__(kThreads) paged_prefill_kernel(const PrefillArgs a) {
  using S = PrefillShape<D>;
  constexpr int RB = S::RB;
  extern __shared__ __align__(1024) uint8_t smem[];
  __shared__ int s_range[2][kWarps];
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, g = lane >> 2, t = lane & 3;
  const int hk = blockIdx.y, sp = blockIdx.z;
  pdl_launch_dependents();
  pdl_wait();
  const TileAt at = find_tile(a, kRows, int(blockIdx.x));
  const int64_t tile = int64_t(blockIdx.x) * a.src.Hkv + hk;
  if (at.b < 0) {
    if (a.n_splits > 1 && sp == 0 && tid == 0) a.part_count[tile] = 0;
    return;
  }
  const int b = at.b;
  const int len = sequence_length(a, b, tid == 0 && hk == 0 && sp == 0);

  // this lane's rows g and g + 8 of its warp's 16
  RowAt row[2];
#pragma unroll
  for (int i = 0; i < 2; ++i) row[i] = row_at(a, at, at.row0 + warp * 16 + g + 8 * i, hk, len);
  {  // the keys that the CTA's rows, and that all rows of this warp, see
    int lo = INT_MAX, hi = 0;
#pragma unroll
    for (int i = 0; i < 2; ++i)
      if (row[i].hi > row[i].lo) {
        lo = min(lo, row[i].lo);
        hi = max(hi, row[i].hi);
      }
    lo = __reduce_min_sync(0xffffffffu, lo);
    hi = __reduce_max_sync(0xffffffffu, hi);
    if (lane == 0) {
      s_range[0][warp] = lo;
      s_range[1][warp] = hi;
    }
  }
  const int all_lo = __reduce_max_sync(0xffffffffu, max(row[0].lo, row[1].lo));
  const int all_hi = __reduce_min_sync(0xffffffffu, min(row[0].hi, row[1].hi));
  __syncthreads();
  int lo = s_range[0][0], hi = s_range[1][0];
#pragma unroll
  for (int w = 1; w < kWarps; ++w) {
    lo = min(lo, s_range[0][w]);
    hi = max(hi, s_range[1][w]);
  }
  const int base = lo == INT_MAX ? 0 : lo & ~15;
  const int parts = hi > base ? min(a.n_splits, (hi - base + a.split - 1) / a.split) : 0;
  if (a.n_splits > 1 && sp == 0 && tid == 0) a.part_count[tile] = parts;
  if (sp >= max(parts, 1)) return;
  const int from = base + sp * a.split;  // of the part; keys below lo are masked by the rows
  const int to = parts == 0 ? from : sp == parts - 1 ? hi : from + a.split;
  const int steps = (to - from + kKeys - 1) / kKeys;

  const uint32_t smem_u = smem_u32(smem);
  auto stage = [&](int st) { return smem_u + st * S::kStage; };
  auto scales_of = [&](int st, int w) {
    return reinterpret_cast<uint16_t*>(smem + st * S::kStage + 2 * kKeys * RB) + 32 * w;
  };
  auto flag_of = [&](int st) { return reinterpret_cast<uint32_t*>(smem + st * S::kStage + 2 * kKeys * RB + S::kScaleBytes); };
  // warp w brings keys 16 w .. 16 w + 15 of a step
  GroupLoader<KIND, D> loader(a.src, hk, kKeys, lane);
  loader.begin(b, from + 16 * warp, steps, max(from, lo), to);
  auto request = [&](int i, int st) {
    if (i < steps)
      loader.request(i, stage(st) + warp * 16 * RB, stage(st) + (kKeys + warp * 16) * RB, flag_of(st) + warp);
    cp_async_commit();
  };
  request(0, 0);

  // q as A fragments in shared memory, [k-step][lane]: scaled by a power of two into [-1, 1] for f16 products of bf16
  // queries (exact, but for parts 2^-24 below the row's largest), as it is otherwise
  uint4* qs = reinterpret_cast<uint4*>(smem + S::kStages * S::kStage) + warp * (D / 16) * 32;
  float unit[2];
  {
    float amax[2] = {0.f, 0.f};
    if (a.q_dtype == BPT_DTYPE_BF16) {
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        if (row[i].q >= 0)
          for (int j = 0; j < D / 16; ++j)
#pragma unroll
            for (int e = 0; e < 4; ++e)
              amax[i] = fmaxf(amax[i], fabsf(load_16(a.q, a.q_dtype, row[i].q + q_dim<KIND>(j, t, e))));
        amax[i] = fmaxf(amax[i], __shfl_xor_sync(0xffffffffu, amax[i], 1));
        amax[i] = fmaxf(amax[i], __shfl_xor_sync(0xffffffffu, amax[i], 2));
      }
    }
    const float2 u0 = unit_range(amax[0]), u1 = unit_range(amax[1]);
    unit[0] = u0.y;
    unit[1] = u1.y;
    for (int j = 0; j < D / 16; ++j) {
      uint32_t f[4];
#pragma unroll
      for (int e = 0; e < 2; ++e)
#pragma unroll
        for (int i = 0; i < 2; ++i) {
          float x = 0.f, y = 0.f;
          if (row[i].q >= 0) {
            x = load_16(a.q, a.q_dtype, row[i].q + q_dim<KIND>(j, t, 2 * e)) * (i ? u1.x : u0.x);
            y = load_16(a.q, a.q_dtype, row[i].q + q_dim<KIND>(j, t, 2 * e + 1)) * (i ? u1.x : u0.x);
          }
          f[2 * e + i] = pack2<KIND>(x, y);
        }
      qs[j * 32 + lane] = make_uint4(f[0], f[1], f[2], f[3]);
    }
    __syncwarp();
  }
  const bool cap = a.softcap > 0.f;
  const float cap_out = a.softcap * kLog2e;
  float mul[2];
#pragma unroll
  for (int i = 0; i < 2; ++i) {
    const float raw = a.sm_scale * unit[i] * a.src.k_scale;
    mul[i] = cap ? raw * 2.f * kLog2e / a.softcap : raw * kLog2e;
  }

  float m[2] = {-INFINITY, -INFINITY}, l[2] = {0.f, 0.f};
  // a row's largest product of a probability and a value scale so far, and the power of two under which o holds them
  float most[2] = {0.f, 0.f}, fit[2] = {1.f, 1.f};
  float o[D / 8][4];
#pragma unroll
  for (int n = 0; n < D / 8; ++n)
#pragma unroll
    for (int i = 0; i < 4; ++i) o[n][i] = 0.f;

  for (int i = 0; i < steps; ++i) {
    const int st = i & 1, key0 = from + i * kKeys;
    loader.place(scales_of(st, warp));
    __syncthreads();  // everyone is done with the stage refilled next
    request(i + 1, st ^ 1);
    cp_async_wait<1>();
    __syncthreads();  // this step's keys and values have landed
    float s[kKeys / 8][4];
#pragma unroll
    for (int n = 0; n < kKeys / 8; ++n)
#pragma unroll
      for (int e = 0; e < 4; ++e) s[n][e] = 0.f;
#pragma unroll
    for (int n = 0; n < kKeys / 16; ++n) {
      scores16<KIND, D>(stage(st) + n * 16 * RB, lane, [&](int j) {
        const uint4 u = qs[j * 32 + lane];
        return MmaRows{{u.x, u.y, u.z, u.w}};
      }, s[2 * n], s[2 * n + 1]);
    }
    const bool masked = key0 < all_lo || key0 + kKeys > all_hi;
    const uint4 bad = *reinterpret_cast<const uint4*>(flag_of(st));
    const bool any_bad = (bad.x | bad.y | bad.z | bad.w) != 0u;
    float top[2] = {-INFINITY, -INFINITY};
#pragma unroll
    for (int n = 0; n < kKeys / 8; ++n) {
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        const int i2 = e >> 1, key = key0 + 8 * n + 2 * t + (e & 1);
        float x = s[n][e];
        x *= __half2float(reinterpret_cast<const __half*>(scales_of(st, n >> 1))[8 * (n & 1) + 2 * t + (e & 1)]) * mul[i2];
        if (cap) x = capped(x, cap_out);
        if (a.slopes) x = fmaf(row[i2].slope, fabsf(float(key - row[i2].pos)), x);
        if (masked && (key < row[i2].lo || key >= row[i2].hi)) x = -INFINITY;
        if (any_bad) {
          const uint32_t w = n >> 1 == 0 ? bad.x : n >> 1 == 1 ? bad.y : n >> 1 == 2 ? bad.z : bad.w;
          if (w >> (n & 1) & 1u) x = -INFINITY;
        }
        s[n][e] = x;
        top[i2] = fmaxf(top[i2], x);
      }
    }
    float off[2];
#pragma unroll
    for (int i2 = 0; i2 < 2; ++i2) {
      top[i2] = fmaxf(top[i2], __shfl_xor_sync(0xffffffffu, top[i2], 1));
      top[i2] = fmaxf(top[i2], __shfl_xor_sync(0xffffffffu, top[i2], 2));
      const float to_m = fmaxf(m[i2], top[i2]);
      off[i2] = to_m == -INFINITY ? 0.f : to_m;
      const float shrink = exp2_approx(m[i2] - off[i2]);
      m[i2] = to_m;
      l[i2] *= shrink;
      most[i2] *= shrink;
      // the probabilities, and what they bring to the output: times their values' scales
      float here = 0.f;
#pragma unroll
      for (int n = 0; n < kKeys / 8; ++n) {
        const __half2 vs = *reinterpret_cast<const __half2*>(scales_of(st, n >> 1) + 16 + 8 * (n & 1) + 2 * t);
        const float x = exp2_approx(s[n][2 * i2] - off[i2]), y = exp2_approx(s[n][2 * i2 + 1] - off[i2]);
        l[i2] += x + y;
        s[n][2 * i2] = x * __low2float(vs);
        s[n][2 * i2 + 1] = y * __high2float(vs);
        here = fmaxf(here, fmaxf(s[n][2 * i2], s[n][2 * i2 + 1]));
      }
      here = fmaxf(here, __shfl_xor_sync(0xffffffffu, here, 1));
      here = fmaxf(here, __shfl_xor_sync(0xffffffffu, here, 2));
      most[i2] = fmaxf(most[i2], here);
      const float to_fit = most[i2] > 0.f ? value_range(most[i2]) : fit[i2], change = shrink * (to_fit * inverse_power(fit[i2]));
      fit[i2] = to_fit;
#pragma unroll
      for (int n = 0; n < D / 8; ++n) {
        o[n][2 * i2] *= change;
        o[n][2 * i2 + 1] *= change;
      }
    }
#pragma unroll
    for (int n = 0; n < kKeys / 16; ++n) {
      // They enter the product rounded to 16 bits (as any operand of these matrix instructions), a row's largest brought to
      // [2^9, 2^10) by a power of two; the sum that divides them is taken before the rounding, in fp32.
      uint32_t p[4];
#pragma unroll
      for (int k = 0; k < 2; ++k)
#pragma unroll
        for (int i2 = 0; i2 < 2; ++i2)
          p[2 * k + i2] = pack2<KIND>(s[2 * n + k][2 * i2] * fit[i2], s[2 * n + k][2 * i2 + 1] * fit[i2]);
      values16<KIND, D>(stage(st) + (kKeys + n * 16) * RB, lane, p, o);
    }
  }
  cp_async_wait<0>();
  float inv[2];
#pragma unroll
  for (int i = 0; i < 2; ++i) {
    l[i] += __shfl_xor_sync(0xffffffffu, l[i], 1);
    l[i] += __shfl_xor_sync(0xffffffffu, l[i], 2);
    inv[i] = l[i] == 0.f ? 0.f : inverse_power(fit[i]) / l[i];
  }
  if (parts <= 1) {
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      if (row[i].out < 0) continue;
#pragma unroll
      for (int n = 0; n < D / 8; ++n) {
        const float x = o[n][2 * i] * inv[i], y = o[n][2 * i + 1] * inv[i];
        const int64_t dst = row[i].out + v_dim<KIND, D>(n, t, 0);
        store_16(a.out, a.q_dtype, dst, x);
        store_16(a.out, a.q_dtype, row[i].out + v_dim<KIND, D>(n, t, 1), y);
      }
    }
    return;
  }
  // a part: [rows][D] and the rows' log2-sum-exp2 of tile (blockIdx.x, hk), part sp
  float* part = a.part_out + (tile * a.n_splits + sp) * (kRows * D);
  float* part_lse = a.part_lse + (tile * a.n_splits + sp) * kRows;
#pragma unroll
  for (int i = 0; i < 2; ++i) {
    if (row[i].out < 0) continue;
    const int r = warp * 16 + g + 8 * i;
#pragma unroll
    for (int n = 0; n < D / 8; ++n) {
      part[r * D + v_dim<KIND, D>(n, t, 0)] = o[n][2 * i] * inv[i];
      part[r * D + v_dim<KIND, D>(n, t, 1)] = o[n][2 * i + 1] * inv[i];
    }
    if (t == 0) part_lse[r] = l[i] == 0.f ? -INFINITY : (m[i] == -INFINITY ? 0.f : m[i]) + log2f(l[i]);
  }
}

// Joins the parts of a tile into out: a warp per row, D / 32 columns per lane.
template <int D>
__global__ void __launch_bounds__(256) prefill_join_kernel(const PrefillArgs a, int rows) {
  constexpr int V = D / 32;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, r = int(blockIdx.y) * 8 + warp;
  pdl_launch_dependents();
  pdl_wait();
  const int64_t tile = blockIdx.x;
  const int x = int(tile / a.src.Hkv), hk = int(tile - int64_t(x) * a.src.Hkv);
  const int parts = a.part_count[tile];
  if (parts <= 1) return;
  const TileAt at = find_tile(a, rows, x);
  const int pr = at.row0 + r, t = pr / a.rep;
  if (t >= at.tokens) return;
  const float* lse = a.part_lse + tile * a.n_splits * rows + r;
  const float* outs = a.part_out + (tile * a.n_splits * rows + r) * D + lane;
  float top = -INFINITY;
  for (int i = lane; i < parts; i += 32) top = fmaxf(top, lse[int64_t(i) * rows]);
  top = warp_max(top);
  const float off = top == -INFINITY ? 0.f : top;
  float sum = 0.f, acc[V];
#pragma unroll
  for (int e = 0; e < V; ++e) acc[e] = 0.f;
#pragma unroll 8
  for (int i = 0; i < parts; ++i) {
    const float f = exp2_approx(lse[int64_t(i) * rows] - off);
    sum += f;
#pragma unroll
    for (int e = 0; e < V; ++e) acc[e] = fmaf(f, outs[int64_t(i) * rows * D + 32 * e], acc[e]);
  }
  const float inv = sum == 0.f ? 0.f : 1.f / sum;
  const int64_t dst = (int64_t(at.token0 + t) * a.Hq + hk * a.rep + pr - t * a.rep) * D + lane;
#pragma unroll
  for (int e = 0; e < V; ++e) store_16(a.out, a.q_dtype, dst + 32 * e, acc[e] * inv);
}

int launch_join(const PrefillArgs& a, int64_t tiles, int rows, cudaStream_t stream) {
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(unsigned(tiles * a.src.Hkv), unsigned((rows + 7) / 8));
  cfg.blockDim = dim3(256);
  cfg.stream = stream;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  const cudaError_t err = a.D == 64    ? cudaLaunchKernelEx(&cfg, prefill_join_kernel<64>, a, rows)
                          : a.D == 128 ? cudaLaunchKernelEx(&cfg, prefill_join_kernel<128>, a, rows)
                                       : cudaLaunchKernelEx(&cfg, prefill_join_kernel<256>, a, rows);
  if (err != cudaSuccess) return set_error(BPT_ERR_CUDA, "paged prefill launch: %s", cudaGetErrorString(err));
  return BPT_OK;
}

template <int D>
int launch_prefill(const PrefillArgs& a, int64_t tiles, int flags, cudaStream_t stream) {
  using S = PrefillShape<D>;
  static std::atomic<uint64_t> ready{0};
  const int st = set_max_smem_once(reinterpret_cast<const void*>(paged_prefill_kernel<D>), S::kSmem, ready);
  if (st) return st;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(unsigned(tiles), unsigned(a.src.Hkv), unsigned(a.n_splits));
  cfg.blockDim = dim3(kThreads);
  cfg.dynamicSmemBytes = S::kSmem;
  cfg.stream = stream;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = attr;
  cfg.numAttrs = (flags & BPT_FLAG_PDL) ? 1 : 0;
  const cudaError_t err = cudaLaunchKernelEx(&cfg, paged_prefill_kernel<D>, a);
  if (err != cudaSuccess) return set_error(BPT_ERR_CUDA, "paged prefill launch: %s", cudaGetErrorString(err));
  return BPT_OK;
}

int prefill_int8(const PrefillArgs& a, int64_t tiles, int flags, cudaStream_t stream) {
  if (a.D == 64) return launch_prefill<64>(a, tiles, flags, stream);
  if (a.D == 128) return launch_prefill<128>(a, tiles, flags, stream);
  return launch_prefill<256>(a, tiles, flags, stream);
}

// How a call is cut: which kernel, rows per tile, the most tiles that the rows can make, keys per part and parts.
struct Plan {
  bool tc;
  int rows;
  int64_t tiles;
  int64_t split, n_splits;
};

Plan plan_prefill(int64_t T, int64_t B, int64_t Hq, int64_t Hkv, int64_t D, int kind, int64_t tokens) {
  Plan p;
  p.tc = kind != BPT_KV_INT8;
  p.rows = p.tc ? kPrefillTcRows : kRows;
  p.tiles = T * (Hq / Hkv) / p.rows + B;
  // Fewer CTAs than fill the GPU (two per SM, one of heads of 256 on the tensor-core kernel): each tile's keys in parts of at
  // least 256 until there are.
  const int64_t ctas = p.tiles * Hkv, want = (p.tc && D == 256 ? 1 : 2) * int64_t(num_sms());
  p.n_splits = std::max<int64_t>(std::min(want / ctas, (tokens + 255) / 256), 1);
  p.split = ((tokens + p.n_splits - 1) / p.n_splits + 127) / 128 * 128;
  return p;
}

// Of a workspace, behind the tickets of other reads: the tiles' counts of parts, the parts' sums, the parts.
int64_t count_bytes(const Plan& p, int64_t Hkv) { return (p.tiles * Hkv * 4 + 255) / 256 * 256; }
int64_t lse_bytes(const Plan& p, int64_t Hkv) { return (p.tiles * Hkv * p.n_splits * p.rows * 4 + 255) / 256 * 256; }

}  // namespace
}  // namespace bpt

using namespace bpt;

extern "C" int64_t bpt_paged_prefill_workspace_bytes(int64_t T, int64_t B, int64_t Hq, int64_t Hkv, int64_t D, int kind,
                                                     int64_t tokens) {
  if (T < 1 || B < 1 || Hkv < 1 || Hq < Hkv || tokens < 1) return 0;
  const Plan p = plan_prefill(T, B, Hq, Hkv, D, kind, tokens);
  return p.n_splits > 1 ? kTicketBytes + count_bytes(p, Hkv) + lse_bytes(p, Hkv) + p.tiles * Hkv * p.n_splits * p.rows * D * 4 : 0;
}

extern "C" int bpt_paged_prefill(const bpt_paged_prefill_args* args) {
  BPT_REQUIRE(args, BPT_ERR_INVALID, "paged prefill: null arguments");
  const void* const q = args->q;
  const int q_dtype = int(args->q_dtype);
  const int64_t q_stride_t = args->q_stride_t;
  const int64_t q_stride_h = args->q_stride_h;
  const void* const k_pool = args->k_pool;
  const void* const v_pool = args->v_pool;
  const int kind = int(args->kind);
  const float k_scale = float(args->k_scale);
  const float v_scale = float(args->v_scale);
  const void* const k_scales = args->k_scales;
  const void* const v_scales = args->v_scales;
  const int32_t* const block_table = args->block_table;
  const int64_t bt_stride = args->bt_stride;
  const int64_t bt_width = args->bt_width;
  const int32_t* const cu_seqlens = args->cu_seqlens;
  const int32_t* const lengths = args->lengths;
  const int32_t* const positions = args->positions;
  const int32_t* const key_starts = args->key_starts;
  const int32_t* const prefix_lens = args->prefix_lens;
  const float* const alibi_slopes = args->alibi_slopes;
  const float softcap = float(args->softcap);
  const int64_t window = args->window;
  const int64_t T = args->T;
  const int64_t B = args->B;
  const int64_t Hq = args->Hq;
  const int64_t Hkv = args->Hkv;
  const int64_t D = args->D;
  const int64_t block_size = args->block_size;
  const int64_t num_blocks = args->num_blocks;
  const int64_t tokens = args->tokens;
  const float sm_scale = float(args->sm_scale);
  void* const out = args->out;
  void* const workspace = args->workspace;
  const int64_t workspace_bytes = args->workspace_bytes;
  const int flags = int(args->flags);
  void* const stream = args->stream;
  const char* who = "paged prefill";
  BPT_REQUIRE(T >= 0 && T < (1ll << 30) && B >= 0 && B < (1 << 20), BPT_ERR_INVALID, "%s: T=%lld B=%lld", who, (long long)T,
              (long long)B);
  if (T == 0 || B == 0) return BPT_OK;
  BPT_REQUIRE(q && cu_seqlens && lengths && out, BPT_ERR_INVALID, "%s: null pointer argument", who);
  PrefillArgs a;
  const int bad = paged_source(a.src, who, k_pool, v_pool, kind, k_scale, v_scale, k_scales, v_scales, block_table, bt_stride,
                               bt_width, Hkv, D, block_size, num_blocks);
  if (bad) return bad;
  BPT_REQUIRE(q_dtype == BPT_DTYPE_F16 || q_dtype == BPT_DTYPE_BF16, BPT_ERR_INVALID, "%s: q dtype %d (f16 or bf16)", who,
              q_dtype);
  BPT_REQUIRE((kind != BPT_KV_F16 || q_dtype == BPT_DTYPE_F16) && (kind != BPT_KV_BF16 || q_dtype == BPT_DTYPE_BF16),
              BPT_ERR_UNSUPPORTED, "%s: 16-bit pages take queries of their own type", who);
  BPT_REQUIRE(Hq >= 1 && Hq % Hkv == 0 && Hq < (1 << 15), BPT_ERR_INVALID, "%s: Hq=%lld is not a multiple of Hkv=%lld", who,
              (long long)Hq, (long long)Hkv);
  BPT_REQUIRE(T * (Hq / Hkv) < (1ll << 31) - 1024, BPT_ERR_INVALID, "%s: too many rows", who);
  BPT_REQUIRE(tokens >= 1 && tokens < (1ll << 30), BPT_ERR_INVALID, "%s: tokens=%lld", who, (long long)tokens);
  BPT_REQUIRE(window >= 0, BPT_ERR_INVALID, "%s: window=%lld", who, (long long)window);
  BPT_REQUIRE(softcap >= 0.f && softcap < INFINITY, BPT_ERR_INVALID, "%s: softcap must be finite and not negative", who);
  BPT_REQUIRE(q_stride_t % 8 == 0 && q_stride_h % 8 == 0 && aligned16(q) && aligned16(out), BPT_ERR_ALIGNMENT,
              "%s: rows must start on 16 bytes", who);
  a.q = q;
  a.q_dtype = q_dtype;
  a.q_st = q_stride_t;
  a.q_sh = q_stride_h;
  a.cu = cu_seqlens;
  a.lengths = lengths;
  a.positions = positions;
  a.key_starts = key_starts;
  a.prefix_lens = prefix_lens;
  a.slopes = alibi_slopes;
  a.softcap = softcap;
  a.sm_scale = sm_scale;
  a.window = window < (1 << 30) ? int(window) : 0;
  a.T = int(T);
  a.B = int(B);
  a.Hq = int(Hq);
  a.D = int(D);
  a.rep = int(Hq / Hkv);
  a.out = out;
  const Plan p = plan_prefill(T, B, Hq, Hkv, D, kind, tokens);
  a.split = int(p.split);
  a.n_splits = int(p.n_splits);
  BPT_REQUIRE(p.tiles < (1ll << 31) && Hkv < 65536 && p.n_splits < 65536, BPT_ERR_INVALID, "%s: too many rows", who);
  a.part_count = nullptr;
  a.part_lse = nullptr;
  a.part_out = nullptr;
  if (p.n_splits > 1) {
    const int64_t need = bpt_paged_prefill_workspace_bytes(T, B, Hq, Hkv, D, kind, tokens);
    BPT_REQUIRE(workspace, BPT_ERR_WORKSPACE, "%s: no workspace", who);
    BPT_REQUIRE(aligned16(workspace), BPT_ERR_ALIGNMENT, "%s: workspace must be 16-byte aligned", who);
    BPT_REQUIRE(workspace_bytes >= need, BPT_ERR_WORKSPACE, "%s: workspace of %lld bytes, need %lld", who,
                (long long)workspace_bytes, (long long)need);
    uint8_t* ws = static_cast<uint8_t*>(workspace) + kTicketBytes;
    a.part_count = reinterpret_cast<int*>(ws);
    a.part_lse = reinterpret_cast<float*>(ws + count_bytes(p, Hkv));
    a.part_out = reinterpret_cast<float*>(ws + count_bytes(p, Hkv) + lse_bytes(p, Hkv));
  }
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  const int st = p.tc ? prefill_tc(a, kind, p.tiles, flags, s) : prefill_int8(a, p.tiles, flags, s);
  return st || p.n_splits == 1 ? st : launch_join(a, p.tiles, p.rows, s);
}
