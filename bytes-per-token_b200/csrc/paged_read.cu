// Decode attention over a paged cache of any format, with score caps, distance bias, sliding windows and a first visible
// key: one query token per sequence.
//
//   s_j = cap tanh(scale q.k_j / cap) - slope |p - j|,  out = sum_j softmax(s)_j v_j  over  max(0, start, p - window + 1) <= j
//   <= p, p = length - 1; no visible key gives 0.
//
// Bound by memory: each visible key and value is read once. A CTA takes a run of keys of one (sequence, KV head, eight of its
// query heads) with four warps that never wait for one another until the end: each walks every fourth group of 16 keys with
// its own ring of cp.async stages, its own running maximum and sum. A group's rows arrive whole (D elements of one head);
// rows outside the visible run are not read, their places hold zeros. The eight query heads fill only half of an MMA's 16
// rows, so the other half carries what rounding takes off: rows 0-7 hold q (then the probabilities) rounded to the product's
// 16-bit type, rows 8-15 the rounded-off rest, and both halves' sums are added in fp32. Products are thus good to 16 (bf16)
// or 22 bits at no cost. The warps join in shared memory; where a sequence takes several CTAs, each writes its part and the
// last to finish (a ticket) joins them.
#include "paged_read.cuh"

namespace bpt {

namespace {

constexpr int kWarps = 4;
constexpr int kThreads = 32 * kWarps;
constexpr int64_t kTickets = 65536;
constexpr int64_t kTicketBytes = kTickets * 4;

struct ReadArgs {
  PagedSource src;
  const void* q;
  int q_dtype;
  int64_t q_sb, q_sh;
  const int32_t* lengths;
  const int32_t* key_starts;  // [B] or null
  const float* slopes;        // [Hq] or null
  float softcap, sm_scale;
  int window;
  int B, Hq, rep, tiles;  // tiles: groups of 8 query heads per KV head
  int split, n_splits;
  int merge;  // 1: parts start at the first visible key's group and are joined into out; 0: parts start at key 0
  void* out;
  int out_dtype;
  float* part_out;  // [B, Hq, n_splits, D]
  float* part_lse;  // [B, Hq, n_splits], natural logarithm
  unsigned int* tickets;
};

__device__ __forceinline__ float load_any(const void* p, int dtype, int64_t i) {
  if (dtype == BPT_DTYPE_F32) return static_cast<const float*>(p)[i];
  if (dtype == BPT_DTYPE_F16) return __half2float(static_cast<const __half*>(p)[i]);
  return __bfloat162float(static_cast<const __nv_bfloat16*>(p)[i]);
}
__device__ __forceinline__ void store_any(void* p, int dtype, int64_t i, float v) {
  if (dtype == BPT_DTYPE_F32) static_cast<float*>(p)[i] = v;
  else if (dtype == BPT_DTYPE_F16) static_cast<__half*>(p)[i] = __float2half_rn(v);
  else static_cast<__nv_bfloat16*>(p)[i] = __float2bfloat16_rn(v);
}

template <int KIND, int D>
struct ReadShape {
  static constexpr int RB = D * kElemBytes<KIND>;
  static constexpr int kScaleBytes = KIND == BPT_KV_INT8 ? 64 : 0;  // 16 K and 16 V scales (fp16) of a group
  static constexpr int kStage = 2 * 16 * RB + kScaleBytes + 16;  // keys, values, scales, the bad-block flag
  // Stages per warp: what keeps the memory busy. 16-bit heads of 128: 3 stages x 8 KB x 4 warps = 96 KB, two CTAs per SM.
  static constexpr int kStages = RB >= 512 ? 3 : RB == 256 ? 3 : 4;
  static constexpr int kRing = kStages * kStage;
  static constexpr int kJoin = 8 * D * 4 + 8 * 8;  // a warp's part: o [8][D], m and l [8]
  static constexpr int kPerWarp = kRing > kJoin ? kRing : kJoin;
  static constexpr int kSmem = kWarps * kPerWarp;
};

template <int KIND, int D>
__global__ void __launch_bounds__(kThreads) paged_read_kernel(const ReadArgs a) {
  using S = ReadShape<KIND, D>;
  constexpr int RB = S::RB, NST = S::kStages;
  extern __shared__ __align__(1024) uint8_t smem[];
  __shared__ int s_last;
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, g = lane >> 2, t = lane & 3;
  const int b = blockIdx.z, hk = int(blockIdx.y) / a.tiles, tile = int(blockIdx.y) - hk * a.tiles, sp = blockIdx.x;
  pdl_launch_dependents();
  pdl_wait();
  const int room = int(min(int64_t(a.src.bt_width) << a.src.bs_log2, int64_t(1) << 30));
  int len = a.lengths[b];
  if (len > room) {  // more tokens than the table has pages for
    if (tid == 0) record_error(kDevErrBlockIndex);
    len = room;
  }
  const int pos = len - 1;
  int lo = a.key_starts ? max(a.key_starts[b], 0) : 0;
  if (a.window > 0) lo = max(lo, pos - a.window + 1);
  const int hi = max(len, 0);
  const int base = a.merge ? lo & ~15 : 0;
  const int parts = hi > lo ? min(a.n_splits, (hi - base + a.split - 1) / a.split) : 0;
  const int h0 = hk * a.rep + tile * 8;        // this CTA's first query head
  const int heads = min(8, a.rep - tile * 8);  // and how many
  if (a.merge && sp >= max(parts, 1)) return;
  const int64_t from64 = int64_t(base) + int64_t(sp) * a.split;
  const int from = max(lo, int(min(from64, int64_t(hi))));
  const int to = sp == a.n_splits - 1 ? hi : int(min(int64_t(hi), from64 + a.split));
  const int first = from & ~15;
  const int groups = to > from ? (to - first + 15) / 16 : 0;
  const int mine = groups > warp ? (groups - warp + kWarps - 1) / kWarps : 0;  // this warp's groups: warp, warp + 4, ...

  uint8_t* ring = smem + warp * S::kPerWarp;
  const uint32_t ring_u = smem_u32(ring);
  auto scales_of = [&](int st) { return reinterpret_cast<uint16_t*>(ring + st * S::kStage + 32 * RB); };
  auto flag_of = [&](int st) { return reinterpret_cast<uint32_t*>(ring + st * S::kStage + 32 * RB + S::kScaleBytes); };
  GroupLoader<KIND, D> loader(a.src, b, hk, first + 16 * warp, 16 * kWarps, mine, from, to, lane);
  auto request = [&](int i, int st) {
    if (i < mine) loader.request(i, ring_u + st * S::kStage, ring_u + st * S::kStage + 16 * RB, flag_of(st));
    cp_async_commit();
  };
#pragma unroll
  for (int i = 0; i < NST - 1; ++i) {
    request(i, i);
    if (i < NST - 2) loader.place(scales_of(i));
  }

  // q: the A fragments of head h0 + g, rounded in rows 0-7 and what rounding took off in rows 8-15
  uint32_t qf[D / 16][4];
  float q_unit = 1.f;
  {
    const int64_t at = int64_t(b) * a.q_sb + int64_t(h0 + g) * a.q_sh;
    float amax = 0.f;
    if constexpr (KIND != BPT_KV_BF16) {  // f16 products: q scaled by a power of two into [-1, 1]
      if (g < heads)
        for (int j = 0; j < D / 16; ++j)
#pragma unroll
          for (int i = 0; i < 4; ++i) amax = fmaxf(amax, fabsf(load_any(a.q, a.q_dtype, at + q_dim<KIND>(j, t, i))));
      amax = fmaxf(amax, __shfl_xor_sync(0xffffffffu, amax, 1));
      amax = fmaxf(amax, __shfl_xor_sync(0xffffffffu, amax, 2));
    }
    const float2 unit = KIND == BPT_KV_BF16 ? make_float2(1.f, 1.f) : unit_range(amax);
    q_unit = unit.y;
#pragma unroll
    for (int j = 0; j < D / 16; ++j) {
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        float x = 0.f, y = 0.f;
        if (g < heads) {
          x = load_any(a.q, a.q_dtype, at + q_dim<KIND>(j, t, 2 * i)) * unit.x;
          y = load_any(a.q, a.q_dtype, at + q_dim<KIND>(j, t, 2 * i + 1)) * unit.x;
        }
        const uint32_t hi2 = pack2<KIND>(x, y);
        const float2 r = unpack2<KIND>(hi2);
        qf[j][2 * i] = hi2;
        qf[j][2 * i + 1] = a.q_dtype == BPT_DTYPE_F32 || KIND == BPT_KV_BF16 && a.q_dtype == BPT_DTYPE_F16
                               ? pack2<KIND>(x - r.x, y - r.y) : 0u;
      }
    }
  }
  const float raw = a.sm_scale * q_unit * a.src.k_scale;  // a product as a score
  const bool cap = a.softcap > 0.f;
  const float mul = cap ? raw * 2.f * kLog2e / a.softcap : raw * kLog2e;
  const float cap_out = a.softcap * kLog2e;
  const float slope = a.slopes && g < heads ? a.slopes[h0 + g] * kLog2e : 0.f;

  float m = -INFINITY, l = 0.f;
  float o[D / 8][4];
#pragma unroll
  for (int n = 0; n < D / 8; ++n)
#pragma unroll
    for (int i = 0; i < 4; ++i) o[n][i] = 0.f;

  int st = 0, st_in = NST - 1;
  for (int i = 0; i < mine; ++i) {
    cp_async_wait<NST - 2>();
    if (i + NST - 2 < mine) loader.place(scales_of(st_in == 0 ? NST - 1 : st_in - 1));  // the group requested last
    __syncwarp();  // every lane's copies of this group have landed; everyone is done with the stage refilled next
    request(i + NST - 1, st_in);
    const int key0 = first + 16 * (warp + kWarps * i);
    const uint32_t tile_u = ring_u + st * S::kStage;
    float s0[4] = {0.f, 0.f, 0.f, 0.f}, s1[4] = {0.f, 0.f, 0.f, 0.f};
    scores16<KIND, D>(tile_u, lane, [&](int j) { return MmaRows{{qf[j][0], qf[j][1], qf[j][2], qf[j][3]}}; }, s0, s1);
    float s[4] = {s0[0] + s0[2], s0[1] + s0[3], s1[0] + s1[2], s1[1] + s1[3]};  // keys 2t, 2t + 1, 2t + 8, 2t + 9
    float vs[4] = {1.f, 1.f, 1.f, 1.f};
    if constexpr (KIND == BPT_KV_INT8) {
      const __half* sc = reinterpret_cast<const __half*>(scales_of(st));
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        const int r = 2 * t + (e & 1) + (e >> 1) * 8;
        s[e] *= __half2float(sc[r]);
        vs[e] = __half2float(sc[16 + r]);
      }
    }
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      const int key = key0 + 2 * t + (e & 1) + (e >> 1) * 8;
      s[e] *= mul;
      if (cap) s[e] = capped(s[e], cap_out);
      s[e] = fmaf(slope, float(key - pos), s[e]);
      if (key < from || key >= to) s[e] = -INFINITY;
    }
    const uint32_t bad = *flag_of(st);  // keys of a block that the table names out of range are left out
    if (bad & 1u) s[0] = s[1] = -INFINITY;
    if (bad & 2u) s[2] = s[3] = -INFINITY;
    float top = fmaxf(fmaxf(s[0], s[1]), fmaxf(s[2], s[3]));
    top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 1));
    top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 2));
    if (__any_sync(0xffffffffu, top > m)) {
      const float to_m = fmaxf(m, top);
      const float shrink = to_m == -INFINITY ? 1.f : exp2_approx(m - to_m);
      m = to_m;
      l *= shrink;
#pragma unroll
      for (int n = 0; n < D / 8; ++n)
#pragma unroll
        for (int e = 0; e < 4; ++e) o[n][e] *= shrink;
    }
    const float off = m == -INFINITY ? 0.f : m;
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      s[e] = exp2_approx(s[e] - off);
      l += s[e];
      s[e] *= vs[e];
    }
    uint32_t p[4];
    p[0] = pack2<KIND>(s[0], s[1]);
    p[2] = pack2<KIND>(s[2], s[3]);
    const float2 r0 = unpack2<KIND>(p[0]), r1 = unpack2<KIND>(p[2]);
    p[1] = pack2<KIND>(s[0] - r0.x, s[1] - r0.y);
    p[3] = pack2<KIND>(s[2] - r1.x, s[3] - r1.y);
    values16<KIND, D>(tile_u + 16 * RB, lane, p, o);
    st = st + 1 == NST ? 0 : st + 1;
    st_in = st_in + 1 == NST ? 0 : st_in + 1;
  }
  cp_async_wait<0>();
  l += __shfl_xor_sync(0xffffffffu, l, 1);
  l += __shfl_xor_sync(0xffffffffu, l, 2);
  __syncwarp();

  // the four warps' parts, joined: o [8][D] and (m, l) [8] of each in its own ring's place
  float* my = reinterpret_cast<float*>(ring);
#pragma unroll
  for (int n = 0; n < D / 8; ++n)
#pragma unroll
    for (int e = 0; e < 2; ++e) my[g * D + v_dim<KIND, D>(n, t, e)] = o[n][e] + o[n][2 + e];
  if (t == 0) {
    my[8 * D + g] = m;
    my[8 * D + 8 + g] = l;
  }
  __syncthreads();
  const bool direct = a.merge && parts <= 1;
  constexpr int V = D / 32;  // a warp writes rows warp and warp + 4, V columns (32 apart) per lane
  for (int r = warp; r < heads; r += kWarps) {
    float ms[kWarps], top = -INFINITY, sum = 0.f, acc[V];
#pragma unroll
    for (int w = 0; w < kWarps; ++w) {
      ms[w] = reinterpret_cast<const float*>(smem + w * S::kPerWarp)[8 * D + r];
      top = fmaxf(top, ms[w]);
    }
    const float off = top == -INFINITY ? 0.f : top;
#pragma unroll
    for (int i = 0; i < V; ++i) acc[i] = 0.f;
#pragma unroll
    for (int w = 0; w < kWarps; ++w) {
      const float* part = reinterpret_cast<const float*>(smem + w * S::kPerWarp);
      const float f = exp2_approx(ms[w] - off);
      sum = fmaf(f, part[8 * D + 8 + r], sum);
#pragma unroll
      for (int i = 0; i < V; ++i) acc[i] = fmaf(f, part[r * D + lane + 32 * i], acc[i]);
    }
    const float inv = sum == 0.f ? 0.f : a.src.v_scale / sum;
    const int64_t row = int64_t(b) * a.Hq + h0 + r;
    if (direct) {
#pragma unroll
      for (int i = 0; i < V; ++i) store_any(a.out, a.out_dtype, row * D + lane + 32 * i, acc[i] * inv);
    } else {
      float* dst = a.part_out + (row * a.n_splits + sp) * D;
#pragma unroll
      for (int i = 0; i < V; ++i) dst[lane + 32 * i] = acc[i] * inv;
      if (lane == 0) a.part_lse[row * a.n_splits + sp] = sum == 0.f ? -INFINITY : (off + log2f(sum)) / kLog2e;
    }
  }
  if (!a.merge || direct) return;

  // the last CTA of this (sequence, heads) to finish joins the parts
  __threadfence();
  __syncthreads();
  if (tid == 0) {
    const unsigned int ticket = atomicAdd(&a.tickets[(int64_t(b) * a.src.Hkv + hk) * a.tiles + tile], 1u);
    s_last = ticket == unsigned(parts - 1);
  }
  __syncthreads();
  if (!s_last) return;
  __threadfence();
  for (int r = warp; r < heads; r += kWarps) {
    const int64_t row = int64_t(b) * a.Hq + h0 + r;
    const float* lse = a.part_lse + row * a.n_splits;
    const float* outs = a.part_out + row * a.n_splits * D;
    float top = -INFINITY;
    for (int i = lane; i < parts; i += 32) top = fmaxf(top, __ldcg(lse + i));
    top = warp_max(top);
    const float off = top == -INFINITY ? 0.f : top;
    float sum = 0.f, acc[V];
#pragma unroll
    for (int i = 0; i < V; ++i) acc[i] = 0.f;
#pragma unroll 4
    for (int i = 0; i < parts; ++i) {
      const float f = exp2_approx((__ldcg(lse + i) - off) * kLog2e);
      sum += f;
#pragma unroll
      for (int e = 0; e < V; ++e) acc[e] = fmaf(f, __ldcg(outs + int64_t(i) * D + lane + 32 * e), acc[e]);
    }
    const float inv = sum == 0.f ? 0.f : 1.f / sum;
#pragma unroll
    for (int e = 0; e < V; ++e) store_any(a.out, a.out_dtype, row * D + lane + 32 * e, acc[e] * inv);
  }
  if (tid == 0) a.tickets[(int64_t(b) * a.src.Hkv + hk) * a.tiles + tile] = 0u;
}

template <int KIND, int D>
int launch_read(const ReadArgs& a, int flags, cudaStream_t stream) {
  using S = ReadShape<KIND, D>;
  static std::atomic<uint64_t> ready{0};
  const int st = set_max_smem_once(reinterpret_cast<const void*>(paged_read_kernel<KIND, D>), S::kSmem, ready);
  if (st) return st;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(unsigned(a.n_splits), unsigned(a.src.Hkv * a.tiles), unsigned(a.B));
  cfg.blockDim = dim3(kThreads);
  cfg.dynamicSmemBytes = S::kSmem;
  cfg.stream = stream;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = attr;
  cfg.numAttrs = (flags & BPT_FLAG_PDL) ? 1 : 0;
  const cudaError_t err = cudaLaunchKernelEx(&cfg, paged_read_kernel<KIND, D>, a);
  if (err != cudaSuccess) return set_error(BPT_ERR_CUDA, "paged read launch: %s", cudaGetErrorString(err));
  return BPT_OK;
}

template <int KIND>
int read_dim(const ReadArgs& a, int64_t D, int flags, cudaStream_t stream) {
  if (D == 64) return launch_read<KIND, 64>(a, flags, stream);
  if (D == 128) return launch_read<KIND, 128>(a, flags, stream);
  return launch_read<KIND, 256>(a, flags, stream);
}

int64_t read_workspace(int64_t B, int64_t Hq, int64_t D, int64_t n_splits) {
  const int64_t lse = ((B * Hq * n_splits * 4 + 255) / 256) * 256;
  return kTicketBytes + lse + B * Hq * n_splits * D * 4;
}

}  // namespace

int paged_source(PagedSource& s, const char* who, const void* k_pool, const void* v_pool, int kind, float k_scale,
                 float v_scale, const void* k_scales, const void* v_scales, const int32_t* block_table, int64_t bt_stride,
                 int64_t bt_width, int64_t Hkv, int64_t D, int64_t block_size, int64_t num_blocks) {
  BPT_REQUIRE(k_pool && v_pool && block_table, BPT_ERR_INVALID, "%s: null pointer argument", who);
  BPT_REQUIRE(kind == BPT_KV_FP8 || kind == BPT_KV_INT8 || kind == BPT_KV_F16 || kind == BPT_KV_BF16, BPT_ERR_INVALID,
              "%s: kind %d", who, kind);
  BPT_REQUIRE(D == 64 || D == 128 || D == 256, BPT_ERR_UNSUPPORTED, "%s: D=%lld (64, 128 or 256)", who, (long long)D);
  BPT_REQUIRE(Hkv >= 1 && Hkv < (1 << 14), BPT_ERR_INVALID, "%s: Hkv=%lld", who, (long long)Hkv);
  BPT_REQUIRE(block_size >= 8 && block_size <= 1024 && (block_size & (block_size - 1)) == 0, BPT_ERR_UNSUPPORTED,
              "%s: block_size=%lld (a power of two from 8 to 1024)", who, (long long)block_size);
  BPT_REQUIRE(num_blocks >= 1 && num_blocks < (1ll << 31), BPT_ERR_INVALID, "%s: num_blocks=%lld", who, (long long)num_blocks);
  BPT_REQUIRE(bt_width >= 1 && bt_width < (1ll << 31) && bt_stride >= bt_width, BPT_ERR_INVALID,
              "%s: block table of width %lld, stride %lld", who, (long long)bt_width, (long long)bt_stride);
  if (kind == BPT_KV_FP8)
    BPT_REQUIRE(k_scale > 0.f && v_scale > 0.f, BPT_ERR_INVALID, "%s: FP8 scales must be positive", who);
  if (kind == BPT_KV_INT8) BPT_REQUIRE(k_scales && v_scales, BPT_ERR_INVALID, "%s: INT8 needs scale pools", who);
  BPT_REQUIRE(aligned16(k_pool) && aligned16(v_pool), BPT_ERR_ALIGNMENT, "%s: pools must be 16-byte aligned", who);
  s.k_pool = static_cast<const uint8_t*>(k_pool);
  s.v_pool = static_cast<const uint8_t*>(v_pool);
  s.k_scales = static_cast<const __half*>(k_scales);
  s.v_scales = static_cast<const __half*>(v_scales);
  s.block_table = block_table;
  s.bt_stride = bt_stride;
  s.num_blocks = num_blocks;
  s.bt_width = int(bt_width);
  s.bs_log2 = 0;
  while ((1 << s.bs_log2) < block_size) ++s.bs_log2;
  s.Hkv = int(Hkv);
  s.k_scale = kind == BPT_KV_FP8 ? k_scale : 1.f;
  s.v_scale = kind == BPT_KV_FP8 ? v_scale : 1.f;
  return BPT_OK;
}

}  // namespace bpt

using namespace bpt;

extern "C" int64_t bpt_paged_read_workspace_bytes(int64_t B, int64_t Hq, int64_t D, int64_t n_splits) {
  return n_splits > 1 ? read_workspace(B, Hq, D, n_splits) : 0;
}

extern "C" int bpt_paged_read(const bpt_paged_read_args* args) {
  BPT_REQUIRE(args, BPT_ERR_INVALID, "paged read: null arguments");
  const void* const q = args->q;
  const int q_dtype = int(args->q_dtype);
  const int64_t q_stride_b = args->q_stride_b;
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
  const int32_t* const lengths = args->lengths;
  const int32_t* const key_starts = args->key_starts;
  const float* const alibi_slopes = args->alibi_slopes;
  const float softcap = float(args->softcap);
  const int64_t window = args->window;
  const int64_t B = args->B;
  const int64_t Hq = args->Hq;
  const int64_t Hkv = args->Hkv;
  const int64_t D = args->D;
  const int64_t block_size = args->block_size;
  const int64_t num_blocks = args->num_blocks;
  const int64_t split = args->split;
  const int64_t n_splits = args->n_splits;
  const float sm_scale = float(args->sm_scale);
  void* const out = args->out;
  const int out_dtype = int(args->out_dtype);
  float* const out_partial = args->out_partial;
  float* const lse_partial = args->lse_partial;
  void* const workspace = args->workspace;
  const int64_t workspace_bytes = args->workspace_bytes;
  const int flags = int(args->flags);
  void* const stream = args->stream;
  const char* who = "paged read";
  BPT_REQUIRE(B >= 0 && B < 65536, BPT_ERR_INVALID, "%s: B=%lld", who, (long long)B);
  if (B == 0) return BPT_OK;
  BPT_REQUIRE(q && lengths, BPT_ERR_INVALID, "%s: null pointer argument", who);
  BPT_REQUIRE(q_dtype == BPT_DTYPE_F32 || q_dtype == BPT_DTYPE_F16 || q_dtype == BPT_DTYPE_BF16, BPT_ERR_INVALID,
              "%s: q dtype %d", who, q_dtype);
  ReadArgs a;
  const int bad = paged_source(a.src, who, k_pool, v_pool, kind, k_scale, v_scale, k_scales, v_scales, block_table, bt_stride,
                               bt_width, Hkv, D, block_size, num_blocks);
  if (bad) return bad;
  BPT_REQUIRE(Hq >= 1 && Hq % Hkv == 0 && Hq < (1 << 15), BPT_ERR_INVALID, "%s: Hq=%lld is not a multiple of Hkv=%lld", who,
              (long long)Hq, (long long)Hkv);
  BPT_REQUIRE(split >= 16 && split % 16 == 0 && split < (1ll << 30) && n_splits >= 1 && n_splits < (1 << 20), BPT_ERR_INVALID,
              "%s: split=%lld (a multiple of 16), n_splits=%lld", who, (long long)split, (long long)n_splits);
  BPT_REQUIRE(window >= 0, BPT_ERR_INVALID, "%s: window=%lld", who, (long long)window);
  BPT_REQUIRE(softcap >= 0.f && softcap < INFINITY, BPT_ERR_INVALID, "%s: softcap must be finite and not negative", who);
  a.merge = out_partial == nullptr;
  a.q = q;
  a.q_dtype = q_dtype;
  a.q_sb = q_stride_b;
  a.q_sh = q_stride_h;
  a.lengths = lengths;
  a.key_starts = key_starts;
  a.slopes = alibi_slopes;
  a.softcap = softcap;
  a.sm_scale = sm_scale;
  a.window = window < (1 << 30) ? int(window) : 0;
  a.B = int(B);
  a.Hq = int(Hq);
  a.rep = int(Hq / Hkv);
  a.tiles = (a.rep + 7) / 8;
  a.split = int(split);
  a.n_splits = int(n_splits);
  a.out = out;
  a.out_dtype = out_dtype;
  a.part_out = out_partial;
  a.part_lse = lse_partial;
  a.tickets = nullptr;
  BPT_REQUIRE(Hkv * a.tiles < 65536, BPT_ERR_INVALID, "%s: too many heads", who);
  if (a.merge) {
    BPT_REQUIRE(out, BPT_ERR_INVALID, "%s: null output", who);
    BPT_REQUIRE(out_dtype == BPT_DTYPE_F32 || out_dtype == BPT_DTYPE_F16 || out_dtype == BPT_DTYPE_BF16, BPT_ERR_INVALID,
                "%s: out dtype %d", who, out_dtype);
    if (n_splits > 1) {
      BPT_REQUIRE(B * Hkv * a.tiles <= kTickets, BPT_ERR_UNSUPPORTED, "%s: %lld sequence heads to join (at most %lld)", who,
                  (long long)(B * Hkv * a.tiles), (long long)kTickets);
      BPT_REQUIRE(workspace, BPT_ERR_WORKSPACE, "%s: no workspace", who);
      BPT_REQUIRE(aligned16(workspace), BPT_ERR_ALIGNMENT, "%s: workspace must be 16-byte aligned", who);
      const int64_t need = read_workspace(B, Hq, D, n_splits);
      BPT_REQUIRE(workspace_bytes >= need, BPT_ERR_WORKSPACE, "%s: workspace of %lld bytes, need %lld", who,
                  (long long)workspace_bytes, (long long)need);
      uint8_t* ws = static_cast<uint8_t*>(workspace);
      a.tickets = reinterpret_cast<unsigned int*>(ws);
      a.part_lse = reinterpret_cast<float*>(ws + kTicketBytes);
      a.part_out = reinterpret_cast<float*>(ws + kTicketBytes + ((B * Hq * n_splits * 4 + 255) / 256) * 256);
    }
  } else {
    BPT_REQUIRE(lse_partial, BPT_ERR_INVALID, "%s: null output", who);
  }
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  switch (kind) {
    case BPT_KV_FP8: return read_dim<BPT_KV_FP8>(a, D, flags, s);
    case BPT_KV_INT8: return read_dim<BPT_KV_INT8>(a, D, flags, s);
    case BPT_KV_F16: return read_dim<BPT_KV_F16>(a, D, flags, s);
    default: return read_dim<BPT_KV_BF16>(a, D, flags, s);
  }
}
