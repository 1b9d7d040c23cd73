// Prefill attention on the 5th-generation tensor cores (tcgen05, sm_100a only), for head dims 64 and 128: the same
// operation, rows, intervals and parts as csrc/paged_prefill.cu.
//
// A CTA takes 256 packed rows (token * rep + head) of one KV head as two tiles of 128 and walks their keys 128 at a time:
//   S = Q K^T    both operands in shared memory (128-byte swizzle), fp32 S in tensor memory;
//   P = 2^(s - m) rounded to the pages' 16-bit type over S's own columns in tensor memory;
//   O += P V     P from tensor memory, V as it lies in its pages ([key][dim], the transposed operand form), fp32 O in tensor
//                memory.
// Four warpgroups: two do the softmax, each of one tile, a thread per row (so neither maximum nor sum crosses threads); one
// brings pages into a ring of shared-memory stages, K and V of a step in stages of their own, by cp.async (rows of any page
// size; keys that are not visible become zeros); of the last, one thread issues the XX
//
// A row's m is the true maximum of its first 64 keys and moves only when the sum of 2^(s - m) over 64 keys passes 2^15: until then
// every P is below 2^15, which both 16-bit types hold, and is divided by the sum of the same powers, so nothing is lost by
// an m that lags. A step thus takes no maximum: one pass from S to P and its sum, and O in tensor memory is rescaled a few
// times per row, if at all.
//
// Every wait is bounded; a thread whose wait runs out records it and leaves its loop, the others follow by their own limits,
// and the CTA still awaits its copies and products, frees its tensor memory and returns.
#define BPT_WHOLE_PROGRAM  // compiled without relocatable device code
#include <type_traits>

#include "paged_prefill.cuh"

namespace bpt {
namespace {

constexpr int kThreads = 512;     // warpgroups: softmax of tile 0, softmax of tile 1, producer, matrix products
constexpr int kTileRows = 128;
constexpr int kRows = 2 * kTileRows;
static_assert(kRows == kPrefillTcRows, "the tiles that the caller counts");
constexpr int kKeys = 128;        // per step
constexpr int kSoftmaxRegs = 200;  // 2 x 128 x 200 + 2 x 128 x 56 = 512 x 128: the split of the registers at launch
constexpr int kOtherRegs = 56;
constexpr int kLaunchRegs = 128;
static_assert(256 * kSoftmaxRegs + 256 * kOtherRegs <= kThreads * kLaunchRegs, "setmaxnreg draws on the launch's registers");
constexpr int kFlagSteps = 16;     // steps whose bad-block flags are kept (the ring runs at most 5 steps ahead)
constexpr float kMostSum = 32768.f;  // a step's sum of powers beyond which a row's maximum moves

template <int KIND, int D>
struct TcShape {
  static constexpr int kRowBytes = D * kElemBytes<KIND>;  // a key's row in its page
  static constexpr int kTileBytes = kTileRows * D * 2;  // a Q tile; a K or V stage
  static constexpr int kStages = D == 128 ? 5 : 8;
  static constexpr int kQ = 2 * kTileBytes;
  static constexpr int kBars = 2 * kStages + 18;  // an even number: the flags behind them start on 16 bytes
  static constexpr int kSmem = 1024 + kQ + kStages * kTileBytes + kBars * 8 + kFlagSteps * 16 + 64;
  static constexpr uint32_t kO = 256;     // columns: S0, S1 at 0, 128; O0, O1 at 256, 256 + D
  static_assert(256 + 2 * D <= 512, "tensor memory");
};

__device__ __forceinline__ void tmem_load32(uint32_t addr, uint32_t (&v)[32]) {
  asm volatile(
      "tcgen05.ld.sync.aligned.32x32b.x32.b32 {%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, "
      "%15, %16, %17, %18, %19, %20, %21, %22, %23, %24, %25, %26, %27, %28, %29, %30, %31}, [%32];\n\t"
      "tcgen05.wait::ld.sync.aligned;"
      : "=r"(v[0]), "=r"(v[1]), "=r"(v[2]), "=r"(v[3]), "=r"(v[4]), "=r"(v[5]), "=r"(v[6]), "=r"(v[7]),
        "=r"(v[8]), "=r"(v[9]), "=r"(v[10]), "=r"(v[11]), "=r"(v[12]), "=r"(v[13]), "=r"(v[14]), "=r"(v[15]),
        "=r"(v[16]), "=r"(v[17]), "=r"(v[18]), "=r"(v[19]), "=r"(v[20]), "=r"(v[21]), "=r"(v[22]), "=r"(v[23]),
        "=r"(v[24]), "=r"(v[25]), "=r"(v[26]), "=r"(v[27]), "=r"(v[28]), "=r"(v[29]), "=r"(v[30]), "=r"(v[31])
      : "r"(addr)
      : "memory");
}
__device__ __forceinline__ void tmem_load64(uint32_t addr, uint32_t (&v)[64]) {
  asm volatile(
      "tcgen05.ld.sync.aligned.32x32b.x64.b32 {%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, "
      "%15, %16, %17, %18, %19, %20, %21, %22, %23, %24, %25, %26, %27, %28, %29, %30, %31, %32, %33, %34, %35, "
      "%36, %37, %38, %39, %40, %41, %42, %43, %44, %45, %46, %47, %48, %49, %50, %51, %52, %53, %54, %55, %56, "
      "%57, %58, %59, %60, %61, %62, %63}, [%64];\n\t"
      "tcgen05.wait::ld.sync.aligned;"
      : "=r"(v[0]), "=r"(v[1]), "=r"(v[2]), "=r"(v[3]), "=r"(v[4]), "=r"(v[5]), "=r"(v[6]), "=r"(v[7]),
        "=r"(v[8]), "=r"(v[9]), "=r"(v[10]), "=r"(v[11]), "=r"(v[12]), "=r"(v[13]), "=r"(v[14]), "=r"(v[15]),
        "=r"(v[16]), "=r"(v[17]), "=r"(v[18]), "=r"(v[19]), "=r"(v[20]), "=r"(v[21]), "=r"(v[22]), "=r"(v[23]),
        "=r"(v[24]), "=r"(v[25]), "=r"(v[26]), "=r"(v[27]), "=r"(v[28]), "=r"(v[29]), "=r"(v[30]), "=r"(v[31]),
        "=r"(v[32]), "=r"(v[33]), "=r"(v[34]), "=r"(v[35]), "=r"(v[36]), "=r"(v[37]), "=r"(v[38]), "=r"(v[39]),
        "=r"(v[40]), "=r"(v[41]), "=r"(v[42]), "=r"(v[43]), "=r"(v[44]), "=r"(v[45]), "=r"(v[46]), "=r"(v[47]),
        "=r"(v[48]), "=r"(v[49]), "=r"(v[50]), "=r"(v[51]), "=r"(v[52]), "=r"(v[53]), "=r"(v[54]), "=r"(v[55]),
        "=r"(v[56]), "=r"(v[57]), "=r"(v[58]), "=r"(v[59]), "=r"(v[60]), "=r"(v[61]), "=r"(v[62]), "=r"(v[63])
      : "r"(addr)
      : "memory");
}
__device__ __forceinline__ void tmem_store32(uint32_t addr, const uint32_t (&v)[32]) {
  asm volatile(
      "tcgen05.st.sync.aligned.32x32b.x32.b32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, "
      "%15, %16, %17, %18, %19, %20, %21, %22, %23, %24, %25, %26, %27, %28, %29, %30, %31, %32};" ::"r"(addr),
      "r"(v[0]), "r"(v[1]), "r"(v[2]), "r"(v[3]), "r"(v[4]), "r"(v[5]), "r"(v[6]), "r"(v[7]), "r"(v[8]),
      "r"(v[9]), "r"(v[10]), "r"(v[11]), "r"(v[12]), "r"(v[13]), "r"(v[14]), "r"(v[15]), "r"(v[16]), "r"(v[17]),
      "r"(v[18]), "r"(v[19]), "r"(v[20]), "r"(v[21]), "r"(v[22]), "r"(v[23]), "r"(v[24]), "r"(v[25]), "r"(v[26]),
      "r"(v[27]), "r"(v[28]), "r"(v[29]), "r"(v[30]), "r"(v[31])
      : "memory");
}


__device__ __forceinline__ void tmem_wait_store() { asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory"); }
__device__ __forceinline__ void tc_fence_before() { asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory"); }
__device__ __forceinline__ void tc_fence_after() { asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory"); }
__device__ __forceinline__ void tc_commit(uint64_t* bar) {
  asm volatile("tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [%0];" ::"r"(smem_u32(bar))
               : "memory");
}

// Shared-memory descriptors of 128-byte-swizzled tiles whose rows are 128 bytes, in atoms of 8 rows (1024 bytes). With the
// contraction along the row (Q, K): the next 8 rows 1024 bytes on. With the contraction across rows (V): the next 8 keys
// 1024 bytes on, the next 64 dims `half` bytes on.
__device__ __forceinline__ uint64_t desc_along(uint32_t addr) {
  return uint64_t((addr >> 4) & 0x3FFFu) | (uint64_t(1) << 16) | (uint64_t(1024 >> 4) << 32) | (uint64_t(1) << 46) |
         (uint64_t(2) << 61);
}
__device__ __forceinline__ uint64_t desc_across(uint32_t addr, uint32_t half) {
  return uint64_t((addr >> 4) & 0x3FFFu) | (uint64_t(half >> 4) << 16) | (uint64_t(1024 >> 4) << 32) | (uint64_t(1) << 46) |
         (uint64_t(2) << 61);
}
// Instruction descriptor, kind::f16: D f32 (bits 4-5 = 1), A and B f16 or bf16 (bits 7-9, 10-12 = 0 or 1), B's rows across
// the contraction (bit 16), N >> 3 at bits 17-22, M >> 4 at bits 24-28.
template <int KIND>
constexpr uint32_t tc_idesc(int m, int n, bool across) {
  return (1u << 4) | (KIND == BPT_KV_BF16 ? (1u << 7) | (1u << 10) : 0u) | (across ? 1u << 16 : 0u) | (uint32_t(n >> 3) << 17) |
         (uint32_t(m >> 4) << 24);
}
// One thread of a converged warp. The products are issued under it, with everything they take computed by the whole warp: the
// descriptors then stay in uniform registers, where the instruction wants them (issued by `lane == 0` they are moved
// there one by one: 100 cycles a product instead of a few).
__device__ __forceinline__ bool elect_one() {
  uint32_t one;
  asm volatile(
      "{\n\t.reg .pred p;\n\t"
      "elect.sync _|p, 0xffffffff;\n\t"
      "selp.u32 %0, 1, 0, p;\n\t}"
      : "=r"(one));
  return one != 0;
}
__device__ __forceinline__ void tc_mma_ss(uint32_t d, uint64_t a, uint64_t b, uint32_t idesc, uint32_t acc) {
  asm volatile(
      "{\n\t.reg .pred p;\n\t"
      "setp.ne.b32 p, %4, 0;\n\t"
      "tcgen05.mma.cta_group::1.kind::f16 [%0], %1, %2, %3, p;\n\t}" ::"r"(d),
      "l"(a), "l"(b), "r"(idesc), "r"(acc)
      : "memory");
}
__device__ __forceinline__ void tc_mma_ts(uint32_t d, uint32_t a, uint64_t b, uint32_t idesc, uint32_t acc) {
  asm volatile(
      "{\n\t.reg .pred p;\n\t"
      "setp.ne.b32 p, %4, 0;\n\t"
      "tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], %2, %3, p;\n\t}" ::"r"(d),
      "r"(a), "l"(b), "r"(idesc), "r"(acc)
      : "memory");
}

// Item n of the ring (K of step n / 2 where n is even, V where odd): its stage and the parity of the lap it fills.
template <int STAGES>
struct Item {
  int stage = 0;
  uint32_t lap = 0;
  __device__ __forceinline__ void next() {
    if (++stage == STAGES) {
      stage = 0;
      lap ^= 1u;
    }
  }
};

__device__ __forceinline__ float2 fadd2(float2 a, float2 b) {
  float2 d;
  asm("{\n\t.reg .b64 ra, rb, rd;\n\t"
      "mov.b64 ra, {%2, %3};\n\t"
      "mov.b64 rb, {%4, %5};\n\t"
      "add.rn.f32x2 rd, ra, rb;\n\t"
      "mov.b64 {%0, %1}, rd;\n\t}"
      : "=f"(d.x), "=f"(d.y)
      : "f"(a.x), "f"(a.y), "f"(b.x), "f"(b.y));
  return d;
}

// What a softmax warpgroup does for tile i: its queries into shared memory, then every step's maximum, probabilities and
// sum, and at the end its rows of O (or of a part) to memory. Thread = row = lane of tensor memory.
template <int KIND, int D, bool CAP, bool SLOPED>
__device__ __forceinline__ void softmax_rows(const PrefillArgs& a, const TileAt& at, const RowAt& row, int hk, int sp, int parts,
                                             int from, int first, int last, int i, uint32_t tmem, uint8_t* smem, uint64_t* q_full,
                                             uint64_t* s_full, uint64_t* p_full, uint64_t* o_done,
                                             uint64_t* started, const uint32_t* flags) {
  using S = TcShape<KIND, D>;
  const int r = threadIdx.x & 127, warp = r >> 5, lane = threadIdx.x & 31;
  float q_unit = 1.f;
  {
    // 32 / CPR rows per pass of the warp, a row's 16-byte chunks side by side
    constexpr int CPR = D / 8, RPP = 32 / CPR;
    uint8_t* tile = smem + i * S::kTileBytes;
    const int c = lane % CPR;
    uint4 x[CPR];
    // (loads without conditions, so that all are in flight at once: rows that are none read the tile's first and become zeros)
    const int64_t q0 = int64_t(at.token0 + at.row0 / a.rep) * a.q_st + int64_t(hk * a.rep) * a.q_sh + 8 * c;
#pragma unroll
    for (int k = 0; k < CPR; ++k) {
      const int code = max(__shfl_sync(0xffffffffu, row.code, RPP * k + lane / CPR), 0);
      const int64_t from_q0 = int64_t(code >> 16) * a.q_st + (code & 0xFFFF) * a.q_sh;
      x[k] = __ldg(reinterpret_cast<const uint4*>(static_cast<const uint16_t*>(a.q) + q0 + from_q0));
    }
    const uint32_t rows = __ballot_sync(0xffffffffu, row.code >= 0);
#pragma unroll
    for (int k = 0; k < CPR; ++k)
      if (!(rows >> (RPP * k + lane / CPR) & 1u)) x[k] = make_uint4(0u, 0u, 0u, 0u);
    if constexpr (!kIs16<KIND>) {
      // f16 products of bf16 queries: a row is brought into [-1, 1] by a power of two (exact, but for parts 2^-24 below its
      // largest); the score's factor takes it back
      if (a.q_dtype == BPT_DTYPE_BF16) {
#pragma unroll
        for (int k = 0; k < CPR; ++k) {
          const uint32_t u[4] = {x[k].x, x[k].y, x[k].z, x[k].w};
          float2 f[4];
          float amax = 0.f;
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            f[e] = unpack2<BPT_KV_BF16>(u[e]);
            amax = fmaxf(amax, fmaxf(fabsf(f[e].x), fabsf(f[e].y)));
          }
#pragma unroll
          for (int o = CPR / 2; o > 0; o >>= 1) amax = fmaxf(amax, __shfl_xor_sync(0xffffffffu, amax, o));
          const float2 unit = unit_range(amax);
          x[k] = make_uint4(pack2<KIND>(f[0].x * unit.x, f[0].y * unit.x), pack2<KIND>(f[1].x * unit.x, f[1].y * unit.x),
                            pack2<KIND>(f[2].x * unit.x, f[2].y * unit.x), pack2<KIND>(f[3].x * unit.x, f[3].y * unit.x));
          const float back = __shfl_sync(0xffffffffu, unit.y, (lane % RPP) * CPR);  // of row RPP k + lane mod RPP
          if (lane / RPP == k) q_unit = back;
        }
      }
    }
#pragma unroll
    for (int k = 0; k < CPR; ++k) {
      const int rr = 32 * warp + RPP * k + lane / CPR;
      *reinterpret_cast<uint4*>(tile + (c >> 3) * (kTileRows * 128) + rr * 128 + (((c & 7) ^ (rr & 7)) << 4)) = x[k];
    }
    fence_proxy_async_shared();
    __syncwarp();
    if (lane == 0) mbar_arrive(&q_full[i]);
  }
  const float raw = a.sm_scale * a.src.k_scale * q_unit;  // a product as a score
  const float mul = CAP ? raw * 2.f * kLog2e / a.softcap : raw * kLog2e;
  const float cap_out = a.softcap * kLog2e;
  const float mul_now = CAP || SLOPED ? 1.f : mul;  // what is left to multiply once a product has its shape
  const int all_lo = __reduce_max_sync(0xffffffffu, row.lo), all_hi = __reduce_min_sync(0xffffffffu, row.hi);
  const uint32_t lanes = uint32_t(32 * warp) << 16;
  const uint32_t s_at = tmem + lanes + i * 128, o_at = tmem + lanes + S::kO + i * D;

  float m = -INFINITY;  // the maximum in use
  float l = 0.f;
  uint32_t n = 0;
  bool ok = true;
  for (int j = first; j < last; ++j, ++n) {
    const int key0 = from + j * kKeys;
    ok = __all_sync(0xffffffffu, mbar_wait(&s_full[2 * i], n & 1u));
    if (!ok) break;
    if (i == 0 && n == 0 && lane == 0) mbar_arrive(started);
    const uint4 bad = *reinterpret_cast<const uint4*>(flags + (j & (kFlagSteps - 1)) * 4);
    const bool any_bad = (bad.x | bad.y | bad.z | bad.w) != 0u;
    const bool masked = any_bad || key0 < all_lo || key0 + kKeys > all_hi;
    // Columns c .. c + 31 of S, as scores but for the factor mul_now.
    auto shape = [&](int c, uint32_t* x, auto with_mask) {
      if constexpr (CAP) {
#pragma unroll
        for (int e = 0; e < 32; ++e) x[e] = __float_as_uint(capped(__uint_as_float(x[e]) * mul, cap_out));
      } else if constexpr (SLOPED) {
#pragma unroll
        for (int e = 0; e < 32; ++e) x[e] = __float_as_uint(__uint_as_float(x[e]) * mul);
      }
      if constexpr (SLOPED) {
        const float far = float(key0 + c - row.pos);
#pragma unroll
        for (int e = 0; e < 32; ++e) x[e] = __float_as_uint(fmaf(row.slope, fabsf(far + float(e)), __uint_as_float(x[e])));
      }
      if constexpr (decltype(with_mask)::value) {
        const int below = row.lo - key0 - c, above = row.hi - key0 - c;
        const uint32_t w = c == 0 ? bad.x : c == 32 ? bad.y : c == 64 ? bad.z : bad.w;
#pragma unroll
        for (int e = 0; e < 32; ++e)
          if (e < below || e >= above || (w >> (e >> 3) & 1u)) x[e] = 0xFF800000u;
      }
    };
    // The step's keys in halves h: P = 2^(s - m), rounded to 16 bits (as any operand of these matrix instructions), and the
    // fp32 sum of what was rounded. P V of the first half runs while the powers of the second are taken.
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      if (h) ok = __all_sync(0xffffffffu, mbar_wait(&s_full[2 * i + 1], n & 1u));
      if (!ok) break;
      tc_fence_after();
      uint32_t p[32];
      auto powers = [&](float off, auto with_mask) {
        float2 sum = make_float2(0.f, 0.f);
        uint32_t x[64];
        tmem_load64(s_at + 64 * h, x);
#pragma unroll
        for (int k = 0; k < 2; ++k) {
          shape(64 * h + 32 * k, x + 32 * k, with_mask);
#pragma unroll
          for (int e = 0; e < 16; ++e) {
            const float2 y = ffma2(make_float2(__uint_as_float(x[32 * k + 2 * e]), __uint_as_float(x[32 * k + 2 * e + 1])),
                                   make_float2(mul_now, mul_now), make_float2(-off, -off));
            const float2 z = make_float2(exp2_approx(y.x), exp2_approx(y.y));
            sum = fadd2(sum, z);
            p[16 * k + e] = pack2<KIND>(z.x, z.y);
          }
        }
        return sum.x + sum.y;
      };
      // a row that has met no key yet meets some in this half: its first maximum
      const int half0 = key0 + 64 * h;
      const bool fresh = m == -INFINITY && row.lo < half0 + 64 && row.hi > half0;
      float sum = 0.f;
      bool looked = false, known = !__all_sync(0xffffffffu, fresh);  // some row has a maximum to begin with
      for (;;) {
        // (two bodies: as one, its masks would be taken on every step)
        if (known) {
          const float off = m == -INFINITY ? 0.f : m;
          sum = masked ? powers(off, std::true_type()) : powers(off, std::false_type());
        }
        const bool moves = fresh ? m == -INFINITY : !(sum <= kMostSum);
        if (looked || !__any_sync(0xffffffffu, moves)) break;
        // a first half-step, and a few later ones: the row's maximum is looked up and moves
        float top = -INFINITY;
#pragma unroll 1
        for (int c = 64 * h; c < 64 * h + 64; c += 32) {
          uint32_t x[32];
          tmem_load32(s_at + c, x);
          shape(c, x, std::true_type());
#pragma unroll
          for (int e = 0; e < 32; ++e) top = fmaxf(top, __uint_as_float(x[e]));
        }
        top *= mul_now;
        float shrink = 1.f;
        if (moves && top > m) {
          shrink = exp2_approx(m - top);
          m = top;
          l *= shrink;
        }
        if (n > 0 || h > 0) {  // the half-step before this one is in O
          ok = __all_sync(0xffffffffu, mbar_wait(&o_done[2 * i + (h ^ 1)], (h ? n : n - 1) & 1u));
          if (!ok) break;
          tc_fence_after();
#pragma unroll 1
          for (int c = 0; c < D; c += 32) {
            uint32_t o[32];
            tmem_load32(o_at + c, o);
#pragma unroll
            for (int e = 0; e < 32; ++e) o[e] = __float_as_uint(__uint_as_float(o[e]) * shrink);
            tmem_store32(o_at + c, o);
          }
        }
        known = looked = true;
      }
      if (!ok) break;
      l += sum;
      tmem_store32(s_at + 64 * h, p);
      tmem_wait_store();
      tc_fence_before();
      __syncwarp();
      if (lane == 0) mbar_arrive(&p_full[2 * i + h]);
    }
    if (!ok) break;
  }
  if (i == 0 && n == 0 && lane == 0) mbar_arrive(started);  // (a tile that sees no key)
  if (ok && n > 0) ok = __all_sync(0xffffffffu, mbar_wait(&o_done[2 * i + 1], (n - 1) & 1u));
  tc_fence_after();
  const float inv = l == 0.f ? 0.f : a.src.v_scale / l;
  const int64_t tile = int64_t(blockIdx.x) * a.src.Hkv + hk;
  // Rows to memory through the warp's share of the tile's queries (which the last products have read), so that a row's
  // 16-byte chunks are stored side by side: 2 D bytes of 32 rows at a time, all of them in 16 bits or half of a part in fp32.
  constexpr int CPR = D / 8;
  const bool bf16 = a.q_dtype == BPT_DTYPE_BF16;
  auto pack_out = [&](float x, float y) {
    if constexpr (kIs16<KIND>) return pack2<KIND>(x, y);
    return bf16 ? pack2<BPT_KV_BF16>(x, y) : pack2<BPT_KV_F16>(x, y);
  };
  uint8_t* stage = smem + i * S::kTileBytes + warp * (32 * 2 * D);
  const int c = lane % CPR;
  const int64_t out0 = (int64_t(at.token0 + at.row0 / a.rep) * a.Hq + hk * a.rep) * (2 * D);  // of the tile's first row, in bytes
  const int64_t part0 = ((tile * a.n_splits + sp) * kRows + i * kTileRows + 32 * warp) * (4 * D);  // of the warp's first row
#pragma unroll 1
  for (int half = 0; half < (parts > 1 ? 2 : 1); ++half) {
#pragma unroll
    for (int b = 0; b < CPR; b += 8) {  // eight chunks: 64 values of 16 bits or 32 of fp32
      uint32_t o[32];
#pragma unroll
      for (int q = 0; q < 2; ++q) {
        if (parts > 1 && q == 1) break;
        const int col = parts > 1 ? half * (D / 2) + 4 * b : 8 * b + 32 * q;
        if (n > 0) {
          tmem_load32(o_at + col, o);
        } else {
#pragma unroll
          for (int e = 0; e < 32; ++e) o[e] = 0u;
        }
        if (parts > 1) {
#pragma unroll
          for (int e = 0; e < 8; ++e)
            *reinterpret_cast<float4*>(stage + lane * (2 * D) + (((b + e) ^ (lane & 7)) << 4)) =
                make_float4(__uint_as_float(o[4 * e]) * inv, __uint_as_float(o[4 * e + 1]) * inv,
                            __uint_as_float(o[4 * e + 2]) * inv, __uint_as_float(o[4 * e + 3]) * inv);
        } else {
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            uint32_t w[4];
#pragma unroll
            for (int k = 0; k < 4; ++k)
              w[k] = pack_out(__uint_as_float(o[8 * e + 2 * k]) * inv, __uint_as_float(o[8 * e + 2 * k + 1]) * inv);
            *reinterpret_cast<uint4*>(stage + lane * (2 * D) + (((b + 4 * q + e) ^ (lane & 7)) << 4)) =
                make_uint4(w[0], w[1], w[2], w[3]);
          }
        }
      }
    }
    __syncwarp();
#pragma unroll
    for (int k = 0; k < CPR; ++k) {
      const int rr = 32 / CPR * k + lane / CPR;
      const uint4 x = *reinterpret_cast<const uint4*>(stage + rr * (2 * D) + ((c ^ (rr & 7)) << 4));
      const int code = __shfl_sync(0xffffffffu, row.code, rr);
      if (code >= 0 && ok) {
        uint8_t* dst = parts > 1 ? reinterpret_cast<uint8_t*>(a.part_out) + part0 + int64_t(rr) * (4 * D) + half * (2 * D)
                                 : static_cast<uint8_t*>(a.out) + out0 + ((code >> 16) * a.Hq + (code & 0xFFFF)) * (2 * D);
        *reinterpret_cast<uint4*>(dst + 16 * c) = x;
      }
    }
    __syncwarp();
  }
  if (ok && parts > 1 && row.code >= 0)
    a.part_lse[(tile * a.n_splits + sp) * kRows + i * kTileRows + r] = l == 0.f ? -INFINITY : (m == -INFINITY ? 0.f : m) + log2f(l);
}

// CAP: scores are capped. SLOPED: they fall with distance, or their factor is not positive (a maximum of products is then no
// maximum of scores).
template <int KIND, int D, bool CAP, bool SLOPED>
__global__ void __launch_bounds__(kThreads, 1) paged_prefill_tc_kernel(const PrefillArgs a) {
  using S = TcShape<KIND, D>;
  constexpr int NS = S::kStages;
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = smem_raw + ((1024u - (smem_u32(smem_raw) & 1023u)) & 1023u);
  uint8_t* ring = smem + S::kQ;
  uint64_t* bars = reinterpret_cast<uint64_t*>(ring + NS * S::kTileBytes);
  uint64_t* full = bars;             // [NS] a stage's rows have landed (one arrival per producer warp)
  uint64_t* empty = full + NS;       // [NS] both tiles' products that read it are done
  uint64_t* q_full = empty + NS;     // [2] a tile's queries are in shared memory
  uint64_t* s_full = q_full + 2;     // [2][2] a tile's half-step of S is in tensor memory
  uint64_t* p_full = s_full + 4;     // [2][2] a half of P is in tensor memory, O rescaled where needed
  uint64_t* o_done = p_full + 4;     // [2][2] that half's P V is in O
  uint64_t* drained = o_done + 4;    // all products are done
  uint64_t* started = drained + 1;   // tile 0 has its first scores
  uint32_t* flags = reinterpret_cast<uint32_t*>(bars + S::kBars);  // [kFlagSteps][4] bad blocks, a word per producer warp
  int* range = reinterpret_cast<int*>(flags + kFlagSteps * 4);      // [2] lo, [2] hi of the tiles
  uint32_t* slot = reinterpret_cast<uint32_t*>(range + 4);          // tensor-memory address
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, wg = warp >> 2;
  const int hk = blockIdx.y, sp = blockIdx.z;

  if (tid == 0) {
    for (int i = 0; i < NS; ++i) {
      mbar_init(&full[i], 4);
      mbar_init(&empty[i], 2);
    }
    for (int i = 0; i < 2; ++i) {
      mbar_init(&q_full[i], 4);
      for (int h = 0; h < 2; ++h) mbar_init(&s_full[2 * i + h], 2);  // the products' completion, and the issuing thread (whose own waits saw the flags)
      mbar_init(&p_full[2 * i], 4);
      mbar_init(&p_full[2 * i + 1], 4);
      mbar_init(&o_done[2 * i], 1);
      mbar_init(&o_done[2 * i + 1], 1);
      range[i] = INT_MAX;
      range[2 + i] = 0;
    }
    mbar_init(drained, 2);
    mbar_init(started, 4);
    fence_mbar_init();
  }
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
  __syncthreads();

  // the tiles' rows: thread r of a softmax warpgroup holds row r
  RowAt row{-1, -1, -1, 0, 0, 0, 0.f};
  if (wg < 2) {
    row = row_at(a, at, at.row0 + wg * kTileRows + (tid & 127), hk, len);
    const bool any = row.hi > row.lo;
    const int lo = __reduce_min_sync(0xffffffffu, any ? row.lo : INT_MAX);
    const int hi = __reduce_max_sync(0xffffffffu, any ? row.hi : 0);
    if (lane == 0 && hi > 0) {
      atomicMin(&range[wg], lo);
      atomicMax(&range[2 + wg], hi);
    }
  } else if (warp == 12) {  // all of tensor memory (one CTA per SM)
    asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], 512;" ::"r"(smem_u32(slot)) : "memory");
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = *slot;
  auto free_tmem = [&]() {
    asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, 512;" ::"r"(tmem) : "memory");
  };
  const int lo = min(range[0], range[1]), hi = max(range[2], range[3]);
  const int base = lo == INT_MAX ? 0 : lo & ~15;
  const int parts = hi > base ? min(a.n_splits, (hi - base + a.split - 1) / a.split) : 0;
  if (a.n_splits > 1 && sp == 0 && tid == 0) a.part_count[tile] = parts;
  if (sp >= max(parts, 1)) {
    if (warp == 12) free_tmem();
    return;
  }
  const int from = base + sp * a.split;
  const int to = parts == 0 ? from : sp == parts - 1 ? hi : from + a.split;
  const int steps = (to - from + kKeys - 1) / kKeys;
  // the steps that tile i has keys in: first[i] <= j < last[i]
  int first[2], last[2];
#pragma unroll
  for (int i = 0; i < 2; ++i) {
    const int l = max(range[i], from), h = min(range[2 + i], to);
    first[i] = h > l ? (l - from) / kKeys : 0;
    last[i] = h > l ? (h - from + kKeys - 1) / kKeys : 0;
  }
  if (wg == 2) {
    asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(kOtherRegs));
    // ---- producer: warp w brings rows 32 w .. 32 w + 31 of every stage, two groups of 16 keys
    const int w = warp & 3;
    const int32_t* table = a.src.block_table + int64_t(b) * a.src.bt_stride;
    const int64_t row_bytes = int64_t(a.src.Hkv) * S::kRowBytes, head_bytes = int64_t(hk) * S::kRowBytes;
    const bool two = a.src.bs_log2 == 3;
    const int take_from = max(from, lo);
    int held = -1, held2 = -1;  // lane n: the block(s) of group n of the current 16 steps
    auto block_at = [&](int key) -> int {
      if (key >= to) return -1;
      const int blk = table[key >> a.src.bs_log2];
      if (blk < 0 || blk >= a.src.num_blocks) {
        record_error(kDevErrBlockIndex);
        return -1;
      }
      return blk;
    };
    auto hold = [&](int j) {
      const int key = from + kKeys * (j + (lane >> 1)) + 32 * w + 16 * (lane & 1);
      held = block_at(key);
      if (two) held2 = block_at(key + 8);
    };
    // The blocks of group grp of step j (one twice where pages are longer than 8), and what the table names wrongly.
    auto blocks_of = [&](int j, int grp, int& blk, int& blk2, uint32_t& bad) {
      const int key0 = from + kKeys * j + 32 * w + 16 * grp;
      blk = __shfl_sync(0xffffffffu, held, 2 * (j & 15) + grp);
      blk2 = two ? __shfl_sync(0xffffffffu, held2, 2 * (j & 15) + grp) : blk;
      bad |= (blk < 0 && key0 < to ? 1u : 0u) << (2 * grp) | (blk2 < 0 && key0 + 8 < to ? 2u : 0u) << (2 * grp);
    };
    if constexpr (!kIs16<KIND>) {
    // Codes go through registers: 16 codes a load, an f16 each into the stage. An item's loads are issued an item ahead.
    constexpr int CPR = D / 16, RPP = 32 / CPR;  // 16-code chunks of a row; rows per pass of the warp
    const int r0 = lane / CPR, c0 = lane % CPR;
    uint4 codes[2][CPR];
    uint32_t taken[2];
    bool ok = true;
    Item<NS> in;
    // (loads without conditions, so that all are in flight at once; what is not taken reads the pool's start and is dropped)
    auto load = [&](int n, uint4 (&x)[CPR], uint32_t& taken) {
      taken = 0;
      const int j = n >> 1;
      if ((n & 1) == 0 && (j & 15) == 0) hold(j);
      const uint8_t* pool = (n & 1) ? a.src.v_pool : a.src.k_pool;
      uint32_t bad = 0;
#pragma unroll
      for (int grp = 0; grp < 2; ++grp) {
        int blk, blk2;
        blocks_of(j, grp, blk, blk2, bad);
        const int key0 = from + kKeys * j + 32 * w + 16 * grp;
        const int64_t slot0 = (int64_t(max(blk, 0)) << a.src.bs_log2) + (key0 & ((1 << a.src.bs_log2) - 1));
        const int64_t slot1 = two ? (int64_t(max(blk2, 0)) << 3) - 8 : slot0;
#pragma unroll
        for (int k = 0; k < 16 / RPP; ++k) {
          const int r = RPP * k + r0;
          const bool take = key0 + r >= take_from && key0 + r < to && (RPP * k < 8 ? blk : blk2) >= 0;
          const uint8_t* src = pool + (take ? ((RPP * k < 8 ? slot0 : slot1) + r) * row_bytes + head_bytes : 0);
          x[grp * (16 / RPP) + k] = __ldg(reinterpret_cast<const uint4*>(src) + c0);
          taken |= (take ? 1u : 0u) << (grp * (16 / RPP) + k);
        }
      }
      if ((n & 1) == 0 && lane == 0) flags[(j & (kFlagSteps - 1)) * 4 + w] = bad;
    };
    auto store = [&](const uint4 (&x)[CPR], uint32_t taken) {
      uint8_t* dst = ring + in.stage * S::kTileBytes + ((2 * c0) >> 3) * (kKeys * 128);
#pragma unroll
      for (int k = 0; k < CPR; ++k) {
        const int rr = 32 * w + RPP * k + r0;
        const uint32_t keep = taken >> k & 1u ? 0xFFFFFFFFu : 0u, u[4] = {x[k].x & keep, x[k].y & keep, x[k].z & keep, x[k].w & keep};
#pragma unroll
        for (int e = 0; e < 2; ++e)
          *reinterpret_cast<uint4*>(dst + rr * 128 + ((((2 * c0 + e) & 7) ^ (rr & 7)) << 4)) =
              make_uint4(codes_to_f16<KIND>(u[2 * e] & 0xFFFFu), codes_to_f16<KIND>(u[2 * e] >> 16),
                         codes_to_f16<KIND>(u[2 * e + 1] & 0xFFFFu), codes_to_f16<KIND>(u[2 * e + 1] >> 16));
      }
      fence_proxy_async_shared();
      __syncwarp();
      if (lane == 0) mbar_arrive(&full[in.stage]);
    };
    if (steps > 0) load(0, codes[0], taken[0]);
    for (int n = 0; n < 2 * steps && ok; n += 2) {
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        if (n + h + 1 < 2 * steps) load(n + h + 1, codes[h ^ 1], taken[h ^ 1]);
        if (n + h >= NS) ok = __all_sync(0xffffffffu, mbar_wait(&empty[in.stage], in.lap ^ 1u));
        if (!ok) break;
        store(codes[h], taken[h]);
        in.next();
      }
    }
    } else {
    constexpr int CPR = D / 8;  // 16-byte chunks of a row
    constexpr int kLag = 2;     // items in flight before the oldest is announced
    Item<NS> in, out;
    bool ok = true;
    int announced = 0;
    auto announce = [&]() {  // the oldest item's copies of this warp have landed: make them the tensor cores' to read
      fence_proxy_async_shared();
      __syncwarp();
      if (lane == 0) mbar_arrive(&full[out.stage]);
      out.next();
      ++announced;
    };
    for (int n = 0; n < 2 * steps && ok; ++n) {
      const int j = n >> 1;
      if (n >= NS) {
        // before waiting for a stage, announce what is in flight: the products that free it may need just that
        if (!__all_sync(0xffffffffu, mbar_test(&empty[in.stage], in.lap ^ 1u))) {
          cp_async_wait<0>();
          while (announced < n) announce();
          ok = __all_sync(0xffffffffu, mbar_wait(&empty[in.stage], in.lap ^ 1u));
          if (!ok) break;
        }
      }
      if ((n & 1) == 0) {
        if ((j & 15) == 0) hold(j);
      }
      const uint8_t* pool = (n & 1) ? a.src.v_pool : a.src.k_pool;
      const uint32_t dst = smem_u32(ring + in.stage * S::kTileBytes);
      uint32_t bad = 0;
      // this lane's chunk of the first rows of each group, and its place: rows 32 / CPR further on are constants away
      const int r0 = lane / CPR, c0 = lane % CPR;
      const uint32_t dst0 = dst + (c0 >> 3) * (kKeys * 128) + (32 * w + r0) * 128, x0 = uint32_t((c0 & 7) ^ r0);
#pragma unroll
      for (int grp = 0; grp < 2; ++grp) {
        const int key0 = from + kKeys * j + 32 * w + 16 * grp;
        int blk, blk2;
        blocks_of(j, grp, blk, blk2, bad);
        const int64_t slot0 = (int64_t(max(blk, 0)) << a.src.bs_log2) + (key0 & ((1 << a.src.bs_log2) - 1));
        const int64_t slot1 = two ? (int64_t(max(blk2, 0)) << 3) - 8 : slot0;
        constexpr int STEP = 32 / CPR;  // rows per pass of the warp
        const uint8_t* src0 = pool + (slot0 + r0) * row_bytes + head_bytes + c0 * 16;
        const uint8_t* src1 = pool + (slot1 + r0) * row_bytes + head_bytes + c0 * 16;
        const bool whole = key0 >= take_from && key0 + 16 <= to && blk >= 0 && blk2 >= 0;
#pragma unroll
        for (int k = 0; k < 16 / STEP; ++k) {
          const uint32_t d = dst0 + (16 * grp + STEP * k) * 128 + ((x0 ^ uint32_t((STEP * k) & 7)) << 4);
          const uint8_t* src = (STEP * k < 8 ? src0 : src1) + STEP * k * row_bytes;
          if (whole) {
            cp_async16(d, src);
          } else {
            const int key = key0 + STEP * k + r0;
            const bool take = key >= take_from && key < to && (STEP * k < 8 ? blk : blk2) >= 0;
            cp_async16(d, take ? src : pool, take);
          }
        }
      }
      if ((n & 1) == 0 && lane == 0) flags[(j & (kFlagSteps - 1)) * 4 + w] = bad;
      cp_async_commit();
      in.next();
      if (n == 0) {  // the first keys are waited for by everyone
        cp_async_wait<0>();
        announce();
      } else {
        cp_async_wait<kLag>();
        if (announced + kLag <= n) announce();
      }
    }
    cp_async_wait<0>();
    while (ok && announced < 2 * steps) announce();
    }
  } else if (wg == 3) {
    asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(kOtherRegs));
    if (warp < 14) {
      // ---- matrix products: a warp per tile; the whole warp waits, one of its threads issues. A step's keys go in halves:
      // S of the next step's half overwrites the columns of this step's half as soon as its P V has been issued.
      constexpr uint32_t id_s = tc_idesc<KIND>(kTileRows, kKeys / 2, false), id_o = tc_idesc<KIND>(kTileRows, D, true);
      const int i = warp - 12, begin = i ? first[1] : first[0], end = i ? last[1] : last[0];
      const uint64_t q_desc = desc_along(smem_u32(smem + i * S::kTileBytes)), k_desc = desc_along(smem_u32(ring)),
                     v_desc = desc_across(smem_u32(ring), kKeys * 128);
      const uint32_t s_at = tmem + i * 128, o_at = tmem + S::kO + i * D;
      Item<NS> item;  // the ring's next item: K of step j on entering step j = 0, else V of step j - 1, then K of step j
      uint32_t n = 0;  // steps whose Q K^T has been issued
      bool ok = true;
      auto wait = [&](uint64_t* bar, uint32_t parity) { ok = __all_sync(0xffffffffu, mbar_wait(bar, parity)); };
      if (end > begin) wait(&q_full[i], 0u);
      // Tile 1 starts half a step late, and stays so: in step, both tiles would take powers at once and then wait at once.
      if (i == 1 && ok && end > begin) wait(started, 0u);
      for (int j = 0; j <= steps && ok; ++j) {
        const int v_stage = item.stage;
        if (j > 0) {
          wait(&full[v_stage], item.lap);
          if (!ok) break;
          item.next();
        }
        const int k_stage = item.stage;
        if (j < steps) {
          wait(&full[k_stage], item.lap);
          if (!ok) break;
          item.next();
        }
        const bool pv = j > begin && j <= end, qk = j >= begin && j < end;
#pragma unroll
        for (int h = 0; h < 2; ++h) {
          if (pv) wait(&p_full[2 * i + h], (n - 1) & 1u);
          if (!ok) break;
          tc_fence_after();
          if (elect_one()) {
            if (pv) {  // P V of step j - 1
              const uint64_t vd = v_desc + uint32_t(v_stage * (S::kTileBytes >> 4) + h * (kKeys / 2 * 128 >> 4));
#pragma unroll
              for (int k = 0; k < kKeys / 32; ++k)
                tc_mma_ts(o_at, s_at + 64 * h + 8 * k, vd + k * (2048 >> 4), id_o, k > 0 || h > 0 || j - 1 > begin ? 1u : 0u);
              tc_commit(&o_done[2 * i + h]);
            }
            if (qk) {  // Q K^T of step j
              const uint64_t kd = k_desc + uint32_t(k_stage * (S::kTileBytes >> 4) + h * (kKeys / 2 * 128 >> 4));
#pragma unroll
              for (int k = 0; k < D / 16; ++k) {
                const uint32_t at_k = (k & 3) * (32 >> 4), at_q = (k >> 2) * (kTileRows * 128 >> 4) + at_k;
                tc_mma_ss(s_at + 64 * h, q_desc + at_q, kd + (k >> 2) * (kKeys * 128 >> 4) + at_k, id_s, k > 0 ? 1u : 0u);
              }
              tc_commit(&s_full[2 * i + h]);
              mbar_arrive(&s_full[2 * i + h]);
            }
          }
          __syncwarp();
        }
        if (!ok) break;
        if (qk) ++n;
        if (elect_one()) {
          if (j > 0) tc_commit(&empty[v_stage]);
          if (j < steps) tc_commit(&empty[k_stage]);
        }
        __syncwarp();
      }
      if (elect_one()) tc_commit(drained);
      __syncwarp();
    }
  } else {
    asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(kSoftmaxRegs));
    softmax_rows<KIND, D, CAP, SLOPED>(a, at, row, hk, sp, parts, from, first[wg], last[wg], wg, tmem, smem, q_full, s_full, p_full, o_done,
                          started, flags);
  }
  __syncwarp();
  tc_fence_before();
  __syncthreads();
  if (warp == 12) {
    (void)mbar_wait(drained, 0u);  // every product issued is complete before tensor memory is freed
    tc_fence_after();
    free_tmem();
  }
}

template <int KIND, int D, bool CAP, bool SLOPED>
int launch_tc(const PrefillArgs& a, int64_t tiles, int flags, cudaStream_t stream) {
  using S = TcShape<KIND, D>;
  const void* kernel = reinterpret_cast<const void*>(paged_prefill_tc_kernel<KIND, D, CAP, SLOPED>);
  static std::atomic<uint64_t> ready{0};
  if (ready.load(std::memory_order_relaxed) == 0) {
    // setmaxnreg hands out the registers of the launch: a build whose kernel was compiled to fewer would wait for ever
    cudaFuncAttributes attr_of;
    const cudaError_t asked = cudaFuncGetAttributes(&attr_of, kernel);
    if (asked != cudaSuccess) return set_error(BPT_ERR_CUDA, "paged prefill: %s", cudaGetErrorString(asked));
    BPT_REQUIRE(attr_of.numRegs == kLaunchRegs, BPT_ERR_CUDA, "paged prefill: kernel built with %d registers, not %d",
                attr_of.numRegs, kLaunchRegs);
  }
  const int st = set_max_smem_once(kernel, S::kSmem, ready);
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
  const cudaError_t err = cudaLaunchKernelEx(&cfg, paged_prefill_tc_kernel<KIND, D, CAP, SLOPED>, a);
  if (err != cudaSuccess) return set_error(BPT_ERR_CUDA, "paged prefill launch: %s", cudaGetErrorString(err));
  return BPT_OK;
}

template <int KIND, int D>
int launch_shape(const PrefillArgs& a, int64_t tiles, int flags, cudaStream_t stream) {
  const bool cap = a.softcap > 0.f, sloped = a.slopes != nullptr || !(a.sm_scale > 0.f);
  if (cap) return sloped ? launch_tc<KIND, D, true, true>(a, tiles, flags, stream) : launch_tc<KIND, D, true, false>(a, tiles, flags, stream);
  return sloped ? launch_tc<KIND, D, false, true>(a, tiles, flags, stream) : launch_tc<KIND, D, false, false>(a, tiles, flags, stream);
}

}  // namespace

int take_prefill_tc_error() {
  int value = 0;
  const int zero = 0;
  if (cudaMemcpyFromSymbol(&value, g_device_error, sizeof(int)) != cudaSuccess) return -1;
  if (value != 0) cudaMemcpyToSymbol(g_device_error, &zero, sizeof(int));
  return value;
}

int prefill_tc(const PrefillArgs& a, int kind, int64_t tiles, int flags, cudaStream_t stream) {
  if (kind == BPT_KV_FP8)
    return a.D == 64 ? launch_shape<BPT_KV_FP8, 64>(a, tiles, flags, stream) : launch_shape<BPT_KV_FP8, 128>(a, tiles, flags, stream);
  if (kind == BPT_KV_F16)
    return a.D == 64 ? launch_shape<BPT_KV_F16, 64>(a, tiles, flags, stream) : launch_shape<BPT_KV_F16, 128>(a, tiles, flags, stream);
  return a.D == 64 ? launch_shape<BPT_KV_BF16, 64>(a, tiles, flags, stream) : launch_shape<BPT_KV_BF16, 128>(a, tiles, flags, stream);
}

}  // namespace bpt
