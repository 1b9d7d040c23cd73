// rope_kv_append: new tokens' queries and keys rotated by their positions (after an optional RMSNorm per head), keys and
// values stored at their slots of a paged cache, in one pass over q, k and v.
//
//   x' = x * rsqrt(mean(x^2) + eps) * w                       (q and k, where a norm weight is given)
//   y[i] = x'[i] c[i] - x'[j] s[i],  y[j] = x'[j] c[i] + x'[i] s[i]     over the first R dims, the rest copied,
//   (i, j) = (i, i + R/2) or, interleaved, (2i, 2i + 1);  c, s = row `position` of the cos / sin tables (fp32)
//
// q goes to q_out in its own type; k and v go to slot (block, offset) as 16-bit values, as E4M3 codes of y / scale or as
// int8 codes under an fp16 scale per (token, KV head). Everything between the load and that one rounding is fp32: the
// quantized codes are taken from the fp32 rotation, not from a 16-bit copy of it.
//
// Without queries (Hq 0) nothing rotates and positions are not read: keys and values are stored as they come.
//
// Bound by memory at many tokens and by launch and load latency at few: 16-byte loads and stores only. A lane owns 16 values
// of a head, 8 and the 8 that rotate with them, so the rotation needs no shuffle; D / 16 lanes hold a head (4, 8 or 16 at D
// 64, 128, 256) and a warp 32 / (D / 16) heads of one token at a time. A warp takes `per_warp` such groups of one
// token, keeping the token's cos and sin in registers.
//
// Measured (B200, 6,558 GB/s copy): 8,192 tokens of 16 + 8 + 8 heads of 128 with norms into bf16 pages 38 us, 3.6 TB/s (the
// floor is 21 us: a warp's groups load one after another, and 71 registers leave 24 warps an SM; held to 40 warps by
// __launch_bounds__ 35 us, but 2,001 tokens into E4M3 pages 10.5 us instead of 8); into INT8 pages 62 us (the head's maximum
// and the quotients on top); 64 tokens 4.2 us, launch and latency.
#include "common.cuh"

namespace bpt {
namespace {

struct AppendArgs {
  const void* q;
  const void* k;
  const void* v;
  int64_t q_st, q_sh, k_st, k_sh, v_st, v_sh;  // strides in elements: token, head
  const int32_t* positions;
  const float* cos;
  const float* sin;
  int64_t table_rows;
  const void* q_norm;
  const void* k_norm;
  void* q_out;
  const int32_t* blocks;
  const int32_t* offsets;
  uint8_t* k_pool;
  uint8_t* v_pool;
  __half* k_scales;
  __half* v_scales;
  float k_scale, v_scale, eps;
  int T, Hq, Hkv, rotary, block_size;
  int chunks;    // work items per token
  int per_warp;  // head groups per item
  int64_t num_blocks;
};

template <int DT>
__device__ __forceinline__ void load8(const void* p, int64_t i, float (&x)[8]) {
  if constexpr (DT == BPT_DTYPE_F32) {
    const float4* f = reinterpret_cast<const float4*>(static_cast<const float*>(p) + i);
    const float4 a = f[0], b = f[1];
    x[0] = a.x; x[1] = a.y; x[2] = a.z; x[3] = a.w; x[4] = b.x; x[5] = b.y; x[6] = b.z; x[7] = b.w;
  } else {
    const uint4 w = *reinterpret_cast<const uint4*>(static_cast<const uint16_t*>(p) + i);
    const uint32_t wv[4] = {w.x, w.y, w.z, w.w};
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      float2 f;
      if constexpr (DT == BPT_DTYPE_BF16) {
        f = make_float2(__uint_as_float(wv[j] << 16), __uint_as_float(wv[j] & 0xFFFF0000u));
      } else {
        f = __half22float2(*reinterpret_cast<const __half2*>(&wv[j]));
      }
      x[2 * j] = f.x;
      x[2 * j + 1] = f.y;
    }
  }
}

template <int DT>
__device__ __forceinline__ void store8(void* p, int64_t i, const float (&x)[8]) {
  if constexpr (DT == BPT_DTYPE_F32) {
    float4* f = reinterpret_cast<float4*>(static_cast<float*>(p) + i);
    f[0] = make_float4(x[0], x[1], x[2], x[3]);
    f[1] = make_float4(x[4], x[5], x[6], x[7]);
  } else {
    uint32_t w[4];
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      if constexpr (DT == BPT_DTYPE_BF16) {
        const __nv_bfloat162 b = __floats2bfloat162_rn(x[2 * j], x[2 * j + 1]);
        w[j] = *reinterpret_cast<const uint32_t*>(&b);
      } else {
        const __half2 h = __floats2half2_rn(x[2 * j], x[2 * j + 1]);
        w[j] = *reinterpret_cast<const uint32_t*>(&h);
      }
    }
    *reinterpret_cast<uint4*>(static_cast<uint16_t*>(p) + i) = make_uint4(w[0], w[1], w[2], w[3]);
  }
}

// x / s with x's sign on a zero quotient (E4M3 keeps it); an infinite or NaN quotient stays what it is, where the
// remainder of div_by would turn an infinity into a NaN.
__device__ __forceinline__ float quotient(float x, float s, float rs) {
  const float q = __fmul_rn(x, rs);
  return fabsf(q) < INFINITY ? copysignf(__fmaf_rn(__fmaf_rn(-q, s, x), rs, q), x) : q;
}

template <int DT, int D, int KIND, bool INTERLEAVED>
__global__ void __launch_bounds__(256) rope_append_kernel(const AppendArgs a) {
  constexpr int LPH = D / 16;    // lanes per head
  constexpr int HPW = 32 / LPH;  // heads per warp and group
  pdl_launch_dependents();
  pdl_wait();
  const uint32_t item = blockIdx.x * 8u + (threadIdx.x >> 5);
  if (item >= uint32_t(a.T) * uint32_t(a.chunks)) return;  // whole warps leave together
  const int lane = threadIdx.x & 31, l = lane % LPH;
  const int t = int(item / uint32_t(a.chunks)), chunk = int(item - uint32_t(t) * uint32_t(a.chunks));
  const int blk = a.blocks[t], off = a.offsets[t], pos = a.positions ? a.positions[t] : 0;
  if (blk == -1) return;  // a padding token
  if (a.positions && (pos < 0 || pos >= a.table_rows)) {
    if (lane == 0) record_error(kDevErrPosition);
    return;
  }
  const bool bad = blk < 0 || blk >= a.num_blocks || off < 0 || off >= a.block_size;
  if (bad && chunk == 0 && lane == 0)
    record_error(blk < 0 || blk >= a.num_blocks ? kDevErrBlockIndex : kDevErrSlotIndex);
  const int half = a.rotary / 2;
  const bool rotates = 16 * l < a.rotary;
  // this lane's two runs of 8: partners of the rotation in the half form, 16 consecutive values otherwise
  const int o0 = !INTERLEAVED && rotates ? 8 * l : 16 * l;
  const int o1 = !INTERLEAVED && rotates ? half + 8 * l : 16 * l + 8;
  float c[8], s[8];
  if (rotates) {
    load8<BPT_DTYPE_F32>(a.cos, int64_t(pos) * half + 8 * l, c);
    load8<BPT_DTYPE_F32>(a.sin, int64_t(pos) * half + 8 * l, s);
  }
  const int heads = a.Hq + 2 * a.Hkv;
  const int64_t slot = (int64_t(blk) * a.block_size + off) * a.Hkv;
  for (int g = 0; g < a.per_warp; ++g) {
    const int first = (chunk * a.per_warp + g) * HPW;
    if (first >= heads) break;
    const int h = first + lane / LPH;
    const bool on = h < heads;
    const bool is_q = h < a.Hq, is_v = h >= a.Hq + a.Hkv;
    const int hk = is_q ? h : is_v ? h - a.Hq - a.Hkv : h - a.Hq;
    float x0[8] = {}, x1[8] = {};
    if (on) {
      const void* src = is_q ? a.q : is_v ? a.v : a.k;
      const int64_t at = int64_t(t) * (is_q ? a.q_st : is_v ? a.v_st : a.k_st) +
                         int64_t(hk) * (is_q ? a.q_sh : is_v ? a.v_sh : a.k_sh);
      load8<DT>(src, at + o0, x0);
      load8<DT>(src, at + o1, x1);
    }
    if (a.q_norm || a.k_norm) {
      float ss = 0.f;
#pragma unroll
      for (int i = 0; i < 8; ++i) ss = fmaf(x0[i], x0[i], fmaf(x1[i], x1[i], ss));
#pragma unroll
      for (int o = LPH / 2; o > 0; o >>= 1) ss += __shfl_xor_sync(0xffffffffu, ss, o);
      const void* w = is_q ? a.q_norm : is_v ? nullptr : a.k_norm;
      if (on && w) {
        const float inv = rsqrtf(ss / float(D) + a.eps);
        float w0[8], w1[8];
        load8<DT>(w, o0, w0);
        load8<DT>(w, o1, w1);
#pragma unroll
        for (int i = 0; i < 8; ++i) {
          x0[i] = x0[i] * inv * w0[i];
          x1[i] = x1[i] * inv * w1[i];
        }
      }
    }
    if (rotates && !is_v) {
      if constexpr (INTERLEAVED) {
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const float e = x0[2 * i], f = x0[2 * i + 1], m = x1[2 * i], n = x1[2 * i + 1];
          x0[2 * i] = fmaf(e, c[i], -f * s[i]);
          x0[2 * i + 1] = fmaf(f, c[i], e * s[i]);
          x1[2 * i] = fmaf(m, c[4 + i], -n * s[4 + i]);
          x1[2 * i + 1] = fmaf(n, c[4 + i], m * s[4 + i]);
        }
      } else {
#pragma unroll
        for (int i = 0; i < 8; ++i) {
          const float e = x0[i], f = x1[i];
          x0[i] = fmaf(e, c[i], -f * s[i]);
          x1[i] = fmaf(f, c[i], e * s[i]);
        }
      }
    }
    if (on && is_q) {
      const int64_t at = (int64_t(t) * a.Hq + h) * D;
      store8<DT>(a.q_out, at + o0, x0);
      store8<DT>(a.q_out, at + o1, x1);
    }
    const int64_t row = (slot + hk) * D;
    uint8_t* pool = is_v ? a.v_pool : a.k_pool;
    const bool stores = on && !is_q && !bad;
    if constexpr (KIND == BPT_KV_F16 || KIND == BPT_KV_BF16) {
      constexpr int PT = KIND == BPT_KV_F16 ? BPT_DTYPE_F16 : BPT_DTYPE_BF16;
      if (stores) {
        store8<PT>(pool, row + o0, x0);
        store8<PT>(pool, row + o1, x1);
      }
    } else {
      uint32_t w[4];
      if constexpr (KIND == BPT_KV_FP8) {
        const float sc = is_v ? a.v_scale : a.k_scale, rs = __frcp_rn(sc);
#pragma unroll
        for (int i = 0; i < 2; ++i) {
          w[i] = uint32_t(float2_to_e4m3x2(quotient(x0[4 * i], sc, rs), quotient(x0[4 * i + 1], sc, rs))) |
                 (uint32_t(float2_to_e4m3x2(quotient(x0[4 * i + 2], sc, rs), quotient(x0[4 * i + 3], sc, rs))) << 16);
          w[2 + i] = uint32_t(float2_to_e4m3x2(quotient(x1[4 * i], sc, rs), quotient(x1[4 * i + 1], sc, rs))) |
                     (uint32_t(float2_to_e4m3x2(quotient(x1[4 * i + 2], sc, rs), quotient(x1[4 * i + 3], sc, rs))) << 16);
        }
      } else {
        float amax = 0.f;
#pragma unroll
        for (int i = 0; i < 8; ++i) amax = fmaxf(amax, fmaxf(fabsf(x0[i]), fabsf(x1[i])));
#pragma unroll
        for (int o = LPH / 2; o > 0; o >>= 1) amax = fmaxf(amax, __shfl_xor_sync(0xffffffffu, amax, o));
        __half s16 = __float2half_rn(__fdiv_rn(amax, 127.0f));
        if (!(__half2float(s16) > 0.f)) s16 = __float2half_rn(1.0f);
        const float sc = __half2float(s16), rs = __frcp_rn(sc);
        auto code = [&](float x) { return uint32_t(int(fminf(fmaxf(rintf(quotient(x, sc, rs)), -128.f), 127.f))) & 0xFFu; };
#pragma unroll
        for (int i = 0; i < 2; ++i) {
          w[i] = code(x0[4 * i]) | (code(x0[4 * i + 1]) << 8) | (code(x0[4 * i + 2]) << 16) | (code(x0[4 * i + 3]) << 24);
          w[2 + i] = code(x1[4 * i]) | (code(x1[4 * i + 1]) << 8) | (code(x1[4 * i + 2]) << 16) | (code(x1[4 * i + 3]) << 24);
        }
        if (stores && l == 0) (is_v ? a.v_scales : a.k_scales)[slot + hk] = s16;
      }
      if (stores) {
        *reinterpret_cast<uint2*>(pool + row + o0) = make_uint2(w[0], w[1]);
        *reinterpret_cast<uint2*>(pool + row + o1) = make_uint2(w[2], w[3]);
      }
    }
  }
}

template <int DT, int D, int KIND>
int launch_append(const AppendArgs& args, bool interleaved, int flags, cudaStream_t stream) {
  AppendArgs a = args;
  const int groups = (a.Hq + 2 * a.Hkv + 32 / (D / 16) - 1) / (32 / (D / 16));
  // Few tokens: a group per warp, so that every load of the call is in flight at once. Many: several of a token's groups in
  // one warp, which reads its cos and sin once, as long as every SM has 8 warps: 2,001 tokens into E4M3 pages 7.9 us (8.4
  // with a group per warp), 8,192 tokens 39 us either way.
  const int64_t fill = int64_t(num_sms()) * 8;
  a.per_warp = 1;
  while (a.per_warp < groups && int64_t(a.T) * ((groups + 2 * a.per_warp - 1) / (2 * a.per_warp)) >= fill) a.per_warp *= 2;
  a.chunks = (groups + a.per_warp - 1) / a.per_warp;
  const int64_t ctas = (int64_t(a.T) * a.chunks + 7) / 8;
  BPT_REQUIRE(int64_t(a.T) * a.chunks < (1ll << 32) - 8, BPT_ERR_INVALID, "rope_kv_append: too many tokens");
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(unsigned(ctas));
  cfg.blockDim = dim3(256);
  cfg.stream = stream;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = attr;
  cfg.numAttrs = (flags & BPT_FLAG_PDL) ? 1 : 0;
  const cudaError_t err = interleaved ? cudaLaunchKernelEx(&cfg, rope_append_kernel<DT, D, KIND, true>, a)
                                      : cudaLaunchKernelEx(&cfg, rope_append_kernel<DT, D, KIND, false>, a);
  if (err != cudaSuccess) return set_error(BPT_ERR_CUDA, "rope_kv_append launch: %s", cudaGetErrorString(err));
  return BPT_OK;
}

template <int DT, int D>
int append_kind(const AppendArgs& a, int kind, bool interleaved, int flags, cudaStream_t s) {
  switch (kind) {
    case BPT_KV_FP8: return launch_append<DT, D, BPT_KV_FP8>(a, interleaved, flags, s);
    case BPT_KV_INT8: return launch_append<DT, D, BPT_KV_INT8>(a, interleaved, flags, s);
    case BPT_KV_F16: return launch_append<DT, D, BPT_KV_F16>(a, interleaved, flags, s);
    default: return launch_append<DT, D, BPT_KV_BF16>(a, interleaved, flags, s);
  }
}

template <int DT>
int append_dim(const AppendArgs& a, int64_t D, int kind, bool interleaved, int flags, cudaStream_t s) {
  if (D == 64) return append_kind<DT, 64>(a, kind, interleaved, flags, s);
  if (D == 128) return append_kind<DT, 128>(a, kind, interleaved, flags, s);
  return append_kind<DT, 256>(a, kind, interleaved, flags, s);
}

}  // namespace
}  // namespace bpt

using namespace bpt;

extern "C" int bpt_rope_kv_append(const bpt_rope_kv_append_args* args) {
  BPT_REQUIRE(args, BPT_ERR_INVALID, "rope_kv_append: null arguments");
  const void* const q = args->q;
  const void* const k = args->k;
  const void* const v = args->v;
  const int dtype = int(args->dtype);
  const int64_t q_stride_t = args->q_stride_t;
  const int64_t q_stride_h = args->q_stride_h;
  const int64_t k_stride_t = args->k_stride_t;
  const int64_t k_stride_h = args->k_stride_h;
  const int64_t v_stride_t = args->v_stride_t;
  const int64_t v_stride_h = args->v_stride_h;
  const int64_t T = args->T;
  const int64_t Hq = args->Hq;
  const int64_t Hkv = args->Hkv;
  const int64_t D = args->D;
  const int64_t rotary = args->rotary;
  const int32_t* const positions = args->positions;
  const float* const cos = args->cos;
  const float* const sin = args->sin;
  const int64_t table_rows = args->table_rows;
  const int interleaved = int(args->interleaved);
  const void* const q_norm = args->q_norm;
  const void* const k_norm = args->k_norm;
  const float eps = float(args->eps);
  void* const q_out = args->q_out;
  const int32_t* const write_blocks = args->write_blocks;
  const int32_t* const write_offsets = args->write_offsets;
  void* const k_pool = args->k_pool;
  void* const v_pool = args->v_pool;
  const int kind = int(args->kind);
  const float k_scale = float(args->k_scale);
  const float v_scale = float(args->v_scale);
  void* const k_scales = args->k_scales;
  void* const v_scales = args->v_scales;
  const int64_t block_size = args->block_size;
  const int64_t num_blocks = args->num_blocks;
  const int flags = int(args->flags);
  void* const stream = args->stream;
  BPT_REQUIRE(T >= 0 && T < (1ll << 31), BPT_ERR_INVALID, "rope_kv_append: T=%lld", (long long)T);
  if (T == 0) return BPT_OK;
  const bool store_only = Hq == 0;
  BPT_REQUIRE((store_only || (q && positions && cos && sin && q_out)) && k && v && write_blocks && write_offsets && k_pool && v_pool,
              BPT_ERR_INVALID, "rope_kv_append: null pointer argument");
  BPT_REQUIRE(dtype == BPT_DTYPE_F32 || dtype == BPT_DTYPE_F16 || dtype == BPT_DTYPE_BF16, BPT_ERR_INVALID,
              "rope_kv_append: dtype %d", dtype);
  BPT_REQUIRE(kind == BPT_KV_FP8 || kind == BPT_KV_INT8 || kind == BPT_KV_F16 || kind == BPT_KV_BF16, BPT_ERR_INVALID,
              "rope_kv_append: kind %d", kind);
  BPT_REQUIRE(D == 64 || D == 128 || D == 256, BPT_ERR_UNSUPPORTED, "rope_kv_append: D=%lld (64, 128 or 256)",
              (long long)D);
  BPT_REQUIRE(!store_only || (rotary == 0 && !positions && !q_norm && !k_norm), BPT_ERR_INVALID,
              "rope_kv_append: without queries nothing rotates (rotary 0, no positions, no norms)");
  BPT_REQUIRE(store_only || (rotary >= 16 && rotary <= D && rotary % 16 == 0), BPT_ERR_UNSUPPORTED,
              "rope_kv_append: rotary=%lld must be a multiple of 16 from 16 to D", (long long)rotary);
  BPT_REQUIRE(Hq >= 0 && Hkv >= 1 && Hq < (1ll << 16) && Hkv < (1ll << 16), BPT_ERR_INVALID,
              "rope_kv_append: Hq=%lld Hkv=%lld", (long long)Hq, (long long)Hkv);
  BPT_REQUIRE(store_only || table_rows >= 1, BPT_ERR_INVALID, "rope_kv_append: empty cos / sin table");
  BPT_REQUIRE(block_size >= 1 && block_size < (1ll << 31) && num_blocks >= 1 && num_blocks < (1ll << 31), BPT_ERR_INVALID,
              "rope_kv_append: bad pool shape");
  if (kind == BPT_KV_FP8)
    BPT_REQUIRE(k_scale > 0.f && v_scale > 0.f, BPT_ERR_INVALID, "rope_kv_append: FP8 scales must be positive");
  if (kind == BPT_KV_INT8)
    BPT_REQUIRE(k_scales && v_scales, BPT_ERR_INVALID, "rope_kv_append: INT8 needs scale pools");
  const int64_t unit = dtype == BPT_DTYPE_F32 ? 4 : 8;  // elements in 16 bytes
  BPT_REQUIRE(aligned16(q) && aligned16(k) && aligned16(v) && aligned16(q_out) && aligned16(k_pool) &&
                  aligned16(v_pool) && aligned16(cos) && aligned16(sin) && (!q_norm || aligned16(q_norm)) &&
                  (!k_norm || aligned16(k_norm)) && q_stride_t % unit == 0 && q_stride_h % unit == 0 &&
                  k_stride_t % unit == 0 && k_stride_h % unit == 0 && v_stride_t % unit == 0 && v_stride_h % unit == 0,
              BPT_ERR_ALIGNMENT, "rope_kv_append: rows must start on 16 bytes");
  AppendArgs a;
  a.q = q;
  a.k = k;
  a.v = v;
  a.q_st = q_stride_t;
  a.q_sh = q_stride_h;
  a.k_st = k_stride_t;
  a.k_sh = k_stride_h;
  a.v_st = v_stride_t;
  a.v_sh = v_stride_h;
  a.positions = positions;
  a.cos = cos;
  a.sin = sin;
  a.table_rows = table_rows;
  a.q_norm = q_norm;
  a.k_norm = k_norm;
  a.q_out = q_out;
  a.blocks = write_blocks;
  a.offsets = write_offsets;
  a.k_pool = static_cast<uint8_t*>(k_pool);
  a.v_pool = static_cast<uint8_t*>(v_pool);
  a.k_scales = static_cast<__half*>(k_scales);
  a.v_scales = static_cast<__half*>(v_scales);
  a.k_scale = k_scale;
  a.v_scale = v_scale;
  a.eps = eps;
  a.T = int(T);
  a.Hq = int(Hq);
  a.Hkv = int(Hkv);
  a.rotary = int(rotary);
  a.block_size = int(block_size);
  a.num_blocks = num_blocks;
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  if (dtype == BPT_DTYPE_F32) return append_dim<BPT_DTYPE_F32>(a, D, kind, interleaved != 0, flags, s);
  if (dtype == BPT_DTYPE_F16) return append_dim<BPT_DTYPE_F16>(a, D, kind, interleaved != 0, flags, s);
  return append_dim<BPT_DTYPE_BF16>(a, D, kind, interleaved != 0, flags, s);
}
