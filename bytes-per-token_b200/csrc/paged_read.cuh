// Shared pieces of the kernels that read a paged KV cache of any format (bf16, f16, E4M3 codes, int8 codes) through
// mma.sync: the shared-memory layout of a run of 16 keys, the K and V operand fragments taken from it, and the scores.
//
// A key row of D elements is RB bytes; its 16-byte chunks are swizzled so that the fragment loads meet no bank conflict
// (at D = 64 with 8-bit codes two rows share 128 bytes: two-way). 16-bit rows: chunk c of row r at c ^ (r mod 8), read with
// ldmatrix. 8-bit rows are read with plain vector loads: QK sums over the head dim and PV leaves it alone, so both
// may take the dims in any order that both operands share, and each lane takes the dims whose codes sit next to each
// other. Codes become f16 exactly (E4M3 and int8 both fit); their scales stay outside the products.
#pragma once

#include "common.cuh"

namespace bpt {

template <int KIND>
constexpr bool kIs16 = KIND == BPT_KV_F16 || KIND == BPT_KV_BF16;
template <int KIND>
constexpr int kElemBytes = kIs16<KIND> ? 2 : 1;

struct PagedSource {
  const uint8_t* k_pool;  // [num_blocks, block_size, Hkv, D]
  const uint8_t* v_pool;
  const __half* k_scales;  // int8: [num_blocks, block_size, Hkv]
  const __half* v_scales;
  const int32_t* block_table;
  int64_t bt_stride;
  int64_t num_blocks;
  int bt_width;
  int bs_log2;  // block_size = 1 << bs_log2
  int Hkv;
  float k_scale, v_scale;  // E4M3: per tensor; 1 otherwise
};

__device__ __forceinline__ void cp_async16(uint32_t dst, const void* src, bool take) {
  const int bytes = take ? 16 : 0;  // nothing is read where not taken: the 16 bytes become zeros
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst), "l"(src), "r"(bytes) : "memory");
}
__device__ __forceinline__ void cp_async16(uint32_t dst, const void* src) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(dst), "l"(src) : "memory");
}
__device__ __forceinline__ void cp_async_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int N>
__device__ __forceinline__ void cp_async_wait() {
  asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory");
}

// The place of 16-byte chunk c of row r.
template <int KIND, int D>
__device__ __forceinline__ int swizzled(int r, int c) {
  if constexpr (kIs16<KIND>) return c ^ (r & 7);
  if constexpr (D == 64) return c ^ ((r >> 1) & 3);
  return c ^ ((((r >> 1) & 3) << 1) ^ ((r & 1) << 2));
}

struct MmaRows {  // an A fragment: 16 rows of a k-step
  uint32_t v[4];
};

template <int KIND>
__device__ __forceinline__ void mma_16816(float (&c)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
  if constexpr (KIND == BPT_KV_BF16) {
    asm volatile(
        "mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
        : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
        : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
  } else {
    asm volatile(
        "mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
        : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
        : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
  }
}

// Two floats as a pair of the product's type, x in the low half.
template <int KIND>
__device__ __forceinline__ uint32_t pack2(float x, float y) {
  if constexpr (KIND == BPT_KV_BF16) {
    const __nv_bfloat162 v = __floats2bfloat162_rn(x, y);
    return *reinterpret_cast<const uint32_t*>(&v);
  } else {
    const __half2 v = __floats2half2_rn(x, y);
    return *reinterpret_cast<const uint32_t*>(&v);
  }
}
template <int KIND>
__device__ __forceinline__ float2 unpack2(uint32_t u) {
  if constexpr (KIND == BPT_KV_BF16) {
    return make_float2(__uint_as_float(u << 16), __uint_as_float(u & 0xFFFF0000u));
  } else {
    return __half22float2(*reinterpret_cast<const __half2*>(&u));
  }
}

// The head dim of slot i (0, 1: k = 2t, 2t + 1; 2, 3: k = 2t + 8, 2t + 9) of k-step j for the lanes with lane % 4 == t.
template <int KIND>
__device__ __forceinline__ int q_dim(int j, int t, int i) {
  if constexpr (kIs16<KIND>) return 16 * j + 2 * t + (i & 1) + (i >> 1) * 8;
  return 64 * (j >> 2) + 16 * t + 4 * (j & 3) + i;
}

// Four codes as two f16 pairs: bytes 0, 1 and bytes 2, 3.
template <int KIND>
__device__ __forceinline__ uint2 codes_to_f16(uint32_t four) {
  uint2 h;
  if constexpr (KIND == BPT_KV_FP8) {
    asm("{\n\t.reg .b16 lo, hi;\n\t"
        "mov.b32 {lo, hi}, %2;\n\t"
        "cvt.rn.f16x2.e4m3x2 %0, lo;\n\t"
        "cvt.rn.f16x2.e4m3x2 %1, hi;\n\t}"
        : "=r"(h.x), "=r"(h.y)
        : "r"(four));
  } else {  // 1024 + (code + 128) as f16 bits, less 1152
    const uint32_t u = four ^ 0x80808080u, m0 = __byte_perm(u, 0x64646464u, 0x4140), m1 = __byte_perm(u, 0x64646464u, 0x4342);
    const __half2 off = __floats2half2_rn(1152.f, 1152.f);
    const __half2 v0 = __hsub2(*reinterpret_cast<const __half2*>(&m0), off), v1 = __hsub2(*reinterpret_cast<const __half2*>(&m1), off);
    h.x = *reinterpret_cast<const uint32_t*>(&v0);
    h.y = *reinterpret_cast<const uint32_t*>(&v1);
  }
  return h;
}

__device__ __forceinline__ void ldmatrix4(uint32_t (&r)[4], uint32_t addr) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0, %1, %2, %3}, [%4];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
               : "r"(addr)
               : "memory");
}
__device__ __forceinline__ void ldmatrix4_trans(uint32_t (&r)[4], uint32_t addr) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0, %1, %2, %3}, [%4];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
               : "r"(addr)
               : "memory");
}
__device__ __forceinline__ uint4 lds128(uint32_t addr) {
  uint4 v;
  asm volatile("ld.shared.v4.u32 {%0, %1, %2, %3}, [%4];" : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w) : "r"(addr) : "memory");
  return v;
}
__device__ __forceinline__ uint2 lds64(uint32_t addr) {
  uint2 v;
  asm volatile("ld.shared.v2.u32 {%0, %1}, [%2];" : "=r"(v.x), "=r"(v.y) : "r"(addr) : "memory");
  return v;
}

// s0, s1 += q . K^T for 16 keys at `tile` (rows 0-7 -> s0, 8-15 -> s1). q(j): the A fragment of k-step j. Even and odd
// k-steps are summed apart: four chains of dependent products instead of two, half as long.
template <int KIND, int D, typename Q>
__device__ __forceinline__ void scores16(uint32_t tile, int lane, const Q& q, float (&s0)[4], float (&s1)[4]) {
  constexpr int RB = D * kElemBytes<KIND>;
  float t0[4] = {0.f, 0.f, 0.f, 0.f}, t1[4] = {0.f, 0.f, 0.f, 0.f};
  if constexpr (kIs16<KIND>) {
    const int row = (lane & 7) + ((lane >> 4) << 3), c = (lane >> 3) & 1;
    const uint32_t base = tile + row * RB;
#pragma unroll
    for (int j = 0; j < D / 16; ++j) {
      uint32_t b[4];
      ldmatrix4(b, base + swizzled<KIND, D>(row, 2 * j + c) * 16);
      const MmaRows qj = q(j);
      mma_16816<KIND>(j & 1 ? t0 : s0, qj.v, b[0], b[1]);
      mma_16816<KIND>(j & 1 ? t1 : s1, qj.v, b[2], b[3]);
    }
  } else {
    const int g = lane >> 2, t = lane & 3;
#pragma unroll
    for (int j4 = 0; j4 < D / 64; ++j4) {
      const uint4 x = lds128(tile + g * RB + swizzled<KIND, D>(g, 4 * j4 + t) * 16);
      const uint4 y = lds128(tile + (g + 8) * RB + swizzled<KIND, D>(g + 8, 4 * j4 + t) * 16);
      const uint32_t xs[4] = {x.x, x.y, x.z, x.w}, ys[4] = {y.x, y.y, y.z, y.w};
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const MmaRows qj = q(4 * j4 + i);
        const uint2 x2 = codes_to_f16<KIND>(xs[i]), y2 = codes_to_f16<KIND>(ys[i]);
        mma_16816<KIND>(i & 1 ? t0 : s0, qj.v, x2.x, x2.y);
        mma_16816<KIND>(i & 1 ? t1 : s1, qj.v, y2.x, y2.y);
      }
    }
  }
#pragma unroll
  for (int e = 0; e < 4; ++e) {
    s0[e] += t0[e];
    s1[e] += t1[e];
  }
}

// o[n] += P . V for 16 keys at `tile`; p: the A fragment (rows x 16 keys). Column n of a lane's o is head dim v_dim(n, .).
template <int KIND, int D>
__device__ __forceinline__ void values16(uint32_t tile, int lane, const uint32_t (&p)[4], float (&o)[D / 8][4]) {
  constexpr int RB = D * kElemBytes<KIND>;
  if constexpr (kIs16<KIND>) {
    const int row = lane & 15, c = lane >> 4;
    const uint32_t base = tile + row * RB;
#pragma unroll
    for (int n = 0; n < D / 8; n += 2) {
      uint32_t b[4];
      ldmatrix4_trans(b, base + swizzled<KIND, D>(row, n + c) * 16);
      mma_16816<KIND>(o[n], p, b[0], b[1]);
      mma_16816<KIND>(o[n + 1], p, b[2], b[3]);
    }
  } else {
    const int g = lane >> 2, t = lane & 3;
    const int rows[4] = {2 * t, 2 * t + 1, 2 * t + 8, 2 * t + 9};
    constexpr int W = D == 64 ? 2 : 4;  // words of codes per row and pass
#pragma unroll
    for (int pass = 0; pass < (D == 256 ? 2 : 1); ++pass) {
      uint32_t w[4][W];
#pragma unroll
      for (int r = 0; r < 4; ++r) {
        if constexpr (D == 64) {
          const uint2 u = lds64(tile + rows[r] * RB + swizzled<KIND, D>(rows[r], g >> 1) * 16 + (g & 1) * 8);
          w[r][0] = u.x;
          w[r][1] = u.y;
        } else {
          const uint4 u = lds128(tile + rows[r] * RB + swizzled<KIND, D>(rows[r], 8 * pass + g) * 16);
          w[r][0] = u.x;
          w[r][1] = u.y;
          w[r][2] = u.z;
          w[r][3] = u.w;
        }
      }
#pragma unroll
      for (int i = 0; i < W; ++i) {
        // bytes j of rows 2t and 2t + 1 next to each other (and of rows 2t + 8, 2t + 9), two j per word
        const uint32_t a0 = __byte_perm(w[0][i], w[1][i], 0x5140), a1 = __byte_perm(w[0][i], w[1][i], 0x7362);
        const uint32_t c0 = __byte_perm(w[2][i], w[3][i], 0x5140), c1 = __byte_perm(w[2][i], w[3][i], 0x7362);
        const uint2 x0 = codes_to_f16<KIND>(a0), x1 = codes_to_f16<KIND>(a1), y0 = codes_to_f16<KIND>(c0), y1 = codes_to_f16<KIND>(c1);
        const int n = 4 * W * pass + 4 * i;
        mma_16816<KIND>(o[n], p, x0.x, y0.x);
        mma_16816<KIND>(o[n + 1], p, x0.y, y0.y);
        mma_16816<KIND>(o[n + 2], p, x1.x, y1.x);
        mma_16816<KIND>(o[n + 3], p, x1.y, y1.y);
      }
    }
  }
}

// One warp's copies of groups of 16 keys from the pages into shared memory: its i-th group is keys first + step * i ..
// first + step * i + 15 of KV head hk (`first`, `step` multiples of 16). Keys outside [from, to), and those of a block that
// the table names out of range, are not read: their places hold zeros, and flag bits 0 (keys 0-7) and 1 (keys 8-15) tell
// of bad blocks. Entries of pages with no key in [from, to) are not looked at: a page given back behind a window may hold
// anything there. Lane n holds the blocks of the group 32 i + n, so a group's rows need no load of the table.
template <int KIND, int D>
struct GroupLoader {
  static constexpr int RB = D * kElemBytes<KIND>;
  const PagedSource& src;
  const int32_t* table;
  int64_t row_bytes, head_bytes;
  int first, step, count, from, to, hk, lane;
  int held = -1, held2 = -1;
  uint32_t scale_bits = 0;

  __device__ __forceinline__ GroupLoader(const PagedSource& s, int hk_, int step_, int lane_)
      : src(s), table(nullptr), row_bytes(int64_t(s.Hkv) * RB), head_bytes(int64_t(hk_) * RB), first(0), step(step_), count(0),
        from(0), to(0), hk(hk_), lane(lane_) {}

  // `count` groups of sequence b from key `first_` on.
  __device__ __forceinline__ void begin(int b, int first_, int count_, int from_, int to_) {
    table = src.block_table + int64_t(b) * src.bt_stride;
    first = first_;
    count = count_;
    from = from_;
    to = to_;
  }
  __device__ __forceinline__ int block_at(int key, int keys) const {  // of keys key .. key + keys - 1
    if (key >= to || key + keys <= from) return -1;
    const int blk = table[key >> src.bs_log2];
    if (blk < 0 || blk >= src.num_blocks) {
      record_error(kDevErrBlockIndex);
      return -1;
    }
    return blk;
  }
  // Requests group i: rows of K at k_dst and of V at v_dst (shared addresses). Called by the whole warp, groups in order.
  __device__ __forceinline__ void request(int i, uint32_t k_dst, uint32_t v_dst, uint32_t* flag) {
    const bool two = src.bs_log2 == 3;  // pages of 8 keys: a group spans two
    if ((i & 31) == 0) {
      const int n = i + lane, key = first + step * n;
      held = n < count ? block_at(key, two ? 8 : 16) : -1;
      if (two) held2 = n < count ? block_at(key + 8, 8) : -1;
    }
    const int key0 = first + step * i;
    const int blk = __shfl_sync(0xffffffffu, held, i & 31);
    const int blk2 = two ? __shfl_sync(0xffffffffu, held2, i & 31) : blk;
    const int inside = key0 & ((1 << src.bs_log2) - 1);
    const int64_t slot = (int64_t(max(blk, 0)) << src.bs_log2) + inside;
    const int64_t slot2 = two ? (int64_t(max(blk2, 0)) << 3) - 8 : slot;  // so that row r of the group is slot2 + r
    const int64_t at = slot * row_bytes + head_bytes, at2 = slot2 * row_bytes + head_bytes;
    if (lane == 0) *flag = (blk < 0 && key0 < to ? 1u : 0u) | (blk2 < 0 && key0 + 8 < to ? 2u : 0u);  // (or unseen)
    constexpr int CPR = RB / 16;
    const int r0 = lane / CPR, c0 = lane % CPR;  // this lane's chunk of the first rows; a pass of the warp takes STEP rows
    constexpr int STEP = CPR >= 32 ? 1 : 32 / CPR;
    if (key0 >= from && key0 + 16 <= to && blk >= 0 && blk2 >= 0) {  // all of it
      const int64_t mine = r0 * row_bytes + c0 * 16;
      const uint8_t *k0 = src.k_pool + at + mine, *k1 = src.k_pool + at2 + mine, *v0 = src.v_pool + at + mine, *v1 = src.v_pool + at2 + mine;
#pragma unroll
      for (int n = 0; n < 16 / STEP; ++n) {
        const uint32_t d = (STEP * n + r0) * RB + swizzled<KIND, D>(STEP * n + r0, c0) * 16;
        const int64_t down = STEP * n * row_bytes;
        cp_async16(k_dst + d, (STEP * n < 8 ? k0 : k1) + down);
        cp_async16(v_dst + d, (STEP * n < 8 ? v0 : v1) + down);
      }
    } else {
#pragma unroll
      for (int n = 0; n < 16 / STEP; ++n) {
        const int r = STEP * n + r0;
        const bool take = key0 + r >= from && key0 + r < to && (STEP * n < 8 ? blk : blk2) >= 0;
        const int64_t off = take ? (STEP * n < 8 ? at : at2) + r * row_bytes + c0 * 16 : 0;
        const uint32_t d = r * RB + swizzled<KIND, D>(r, c0) * 16;
        cp_async16(k_dst + d, src.k_pool + off, take);
        cp_async16(v_dst + d, src.v_pool + off, take);
      }
    }
    if constexpr (KIND == BPT_KV_INT8) {  // lanes 0-15 the group's K scales, 16-31 its V scales; stored by place()
      const int r = lane & 15;
      const bool take = key0 + r >= from && key0 + r < to && (r < 8 ? blk : blk2) >= 0;
      const int64_t at_scale = ((r < 8 ? slot : slot2) + r) * src.Hkv + hk;
      scale_bits = take ? __half_as_ushort((lane < 16 ? src.k_scales : src.v_scales)[at_scale]) : 0u;
    }
  }
  // The scales requested last, into shared memory (called when they have had time to arrive).
  __device__ __forceinline__ void place(uint16_t* scales) const {
    if constexpr (KIND == BPT_KV_INT8) scales[lane] = uint16_t(scale_bits);
  }
};

// The head dim of column 2t + e of n-tile n.
template <int KIND, int D>
__device__ __forceinline__ int v_dim(int n, int t, int e) {
  const int g = 2 * t + e;
  if constexpr (kIs16<KIND>) return 8 * n + g;
  if constexpr (D == 64) return 8 * g + n;
  return 128 * (n >> 4) + 16 * g + (n & 15);
}

constexpr float kLog2e = 1.4426950408889634f;

__device__ __forceinline__ float exp2_approx(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}

// cap tanh(x / cap) as a base-2 score, from y = 2 log2(e) x / cap; `cap_out` = cap log2 e. tanh = 1 - 2 / (2^y + 1): its
// absolute error is a few 2^-24, so the score's is a few 2^-24 of the cap.
__device__ __forceinline__ float capped(float y, float cap_out) {
  return cap_out - __fdividef(2.f * cap_out, exp2_approx(y) + 1.f);
}

// The power of two that brings |x| <= amax to at most 1, as (factor, its inverse): keeps any q inside f16's range.
__device__ __forceinline__ float2 unit_range(float amax) {
  const uint32_t bits = __float_as_uint(amax);
  const int e = int(bits >> 23) - 126;  // amax < 2^e
  if (amax == 0.f || e <= -126 || e > 126) return make_float2(1.f, 1.f);
  return make_float2(__uint_as_float(uint32_t(127 - e) << 23), __uint_as_float(uint32_t(127 + e) << 23));
}

// The power of two that brings `most` > 0, a row's largest probability times the scale of its key's int8 values, to
// [2^9, 2^10): scales of small values (max / 127 in f16) would otherwise take the products below what f16 holds. Between 2^-7
// and 2^70, so that ratios of two such powers, by which sums move from one to the next, stay in fp32's range.
__device__ __forceinline__ float value_range(float most) {
  const int e = min(max(int(__float_as_uint(most) >> 23) - 126, -60), 17);
  return __uint_as_float(uint32_t(137 - e) << 23);
}
// 1 / f of a power of two, exactly.
__device__ __forceinline__ float inverse_power(float f) { return __uint_as_float(0x7F000000u - __float_as_uint(f)); }

// The checks and fields that every reader of a paged cache of any format shares.
int paged_source(PagedSource& s, const char* who, const void* k_pool, const void* v_pool, int kind, float k_scale,
                 float v_scale, const void* k_scales, const void* v_scales, const int32_t* block_table, int64_t bt_stride,
                 int64_t bt_width, int64_t Hkv, int64_t D, int64_t block_size, int64_t num_blocks);

}  // namespace bpt
