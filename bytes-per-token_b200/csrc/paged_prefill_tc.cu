// Prefill attention on the 5th-generation tensor cores (tcgen05, sm_100a only): the same operation, rows, intervals and parts
// as csrc/paged_prefill.cu.
//
// A CTA takes a tile of 128 packed rows (token * rep + head) of one KV head and walks their keys 64 at a time:
//   S = Q K^T    both operands in shared memory (128-byte swizzle), fp32 S in tensor memory, two buffers of 64 columns;
//   P = 2^(s - m) rounded to 16 bits, over the S that it came from;
//   O += P V     P from tensor memory, V as it lies in its pages ([key][dim], the transposed operand form), fp32 O in tensor
//                memory.
// Two warpgroups. One does the softmax, a thread per row, so that neither maximum nor sum crosses threads. Of the other, one
// warp issues the products and the rest bring pages into a ring of shared-memory stages (K and V of a step in stages of their
// own) as TMA boxes, pages past the visible keys out of the map's range and so zero: 16-bit pages as the products take them, a
// box per page, a warp for K and one for V; E4M3 codes by one warp, and through the registers of two to f16. While the softmax takes a step's powers, the tensor
// cores take the products of the step before and the scores of the next. At heads of 64 and 128 two CTAs share an SM, so that
// one's loads, waits and stores run under the other's powers.
//
// Keys go from the last to the first: a row's nearest come first, which a bias by distance favours.
//
// A row's m is the true maximum of the first step that it sees and moves only when a step's sum of 2^(s - m) passes 2^15: until
// then every P is below 2^15, which both 16-bit types hold, and is divided by the sum of the same powers, so nothing is lost
// by an m that lags. A step thus takes no maximum: one pass from S to P and its sum, and O in tensor memory is rescaled a few
// times per row, if at all. Over f16 and E4M3 pages P is f16, whose smallest step is 2^-24: a power below 2^-25 is lost, N
// keys lose at most N 2^-25 of the largest value. (Powers of s - m + 4 or + 8 would reach that much further down, but leave m as
// much less room to lag: heads of 256, capped, 198 and 221 us instead of 168.) Without cap and bias a power's exponent is one
// fused product less the rounded m, off by m's rounding for all keys of a row alike: that is only a common factor of P and
// its sum, and stays in f16's range for scores below 2^27.
//
// Measured (B200: 1,647 TFLOP/s bf16 by library product in a burst, 1,405 sustained; 6,558 GB/s copy): a prompt of 8,192 tokens,
// 32 + 8 heads of 128, bf16: 511 us by itself (1,076 TFLOP/s), 550 to 567 when calls follow each other, at 1,570 MHz under the
// power limit (980 TFLOP/s). Products and exponentials each fill 57% of their pipe; a step's chain S -> P -> O has to hide
// behind the other CTA's. Ragged batches (12 prompts of 17 to 2,000: 124 us) are bound by what is not the loop: about 9 us per
// CTA for its map, first pages, queries and rows out. Heads of 256, capped, 4,096 tokens in a window of 1,024: 166 us, one CTA
// an SM. E4M3: two chunks of about 1,800 tokens over 2,700, 16 + 4 heads of 128, 200 us (bf16 133): the two converting warps.
// For that prompt, on the way here: 256 rows in one CTA per SM 713 us; 128 rows with a box per 64 dims 687, a box per page
// 565, K and V by warps of their own 538; a polynomial in place of a quarter of the exponentials 576 where 572 was without.
//
// Every wait is bounded; a thread whose wait runs out records it and leaves its loop, the others follow by their own limits,
// and the CTA still awaits its copies and products, frees its tensor memory and returns.
#define BPT_WHOLE_PROGRAM  // compiled without relocatable device code
#include <cuda.h>
#include <cudaTypedefs.h>

#include <type_traits>

#include "paged_prefill.cuh"

namespace bpt {
namespace {

constexpr int kThreads = 256;  // warpgroups: softmax; producers (warps 4-6) and products (warp 7)
constexpr int kRows = 128;
static_assert(kRows == kPrefillTcRows, "the tiles that the caller counts");
constexpr int kKeys = 64;  // per step
constexpr int kLaunchRegs = 128;
constexpr int kFlagSteps = 16;       // steps whose bad-block flags are kept (the ring runs at most 4 steps ahead)
constexpr float kMostSum = 32768.f;  // a step's sum of powers beyond which a row's maximum moves

template <int KIND, int D>
struct TcShape {
  static constexpr int kRowBytes = D * kElemBytes<KIND>;  // a key's row in its page
  static constexpr int kQ = kRows * D * 2;
  static constexpr int kStage = kKeys * D * 2;  // [group of 8 keys][part of 64 dims][8][128 bytes, swizzled]
  static constexpr int kGroup = 8 * D * 2;
  static constexpr int kStages = D == 64 ? 8 : D == 128 ? 5 : 4;
  static constexpr int kBars = ((kIs16<KIND> ? 2 : 3) * kStages + 12) / 2 * 2;  // (even: what follows starts on 16 bytes)
  static constexpr int kSmem = kQ + kStages * kStage + kBars * 8 + kFlagSteps * 4 + 16;
  static_assert(D == 256 || kSmem <= 113 * 1024, "two CTAs per SM");
  static constexpr int kProducers = kIs16<KIND> ? 2 : 3;  // warps
  // setmaxnreg: 128 threads x (softmax + other) = 256 x the launch's 128
  static constexpr int kSoftmaxRegs = kIs16<KIND> ? 200 : 168, kOtherRegs = 256 - kSoftmaxRegs;
  static constexpr uint32_t kO = 128;                             // columns: S at 0 and 64, O from 128
  static constexpr uint32_t kColumns = D == 256 ? 512 : 256;  // of tensor memory
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

// Shared-memory descriptors of 128-byte-swizzled tiles, whose rows of 64 values are 128 bytes, in atoms of 8 rows (1024
// bytes). With the contraction along the row (Q, K): the next 8 rows `rows8` bytes on. With the contraction across rows
// (V): the next 8 keys `rows8` bytes on, the next 64 dims `dims64` bytes on.
__device__ __forceinline__ uint64_t desc_along(uint32_t addr, uint32_t rows8) {
  return uint64_t((addr >> 4) & 0x3FFFu) | (uint64_t(1) << 16) | (uint64_t(rows8 >> 4) << 32) | (uint64_t(1) << 46) |
         (uint64_t(2) << 61);
}
__device__ __forceinline__ uint64_t desc_across(uint32_t addr, uint32_t rows8, uint32_t dims64) {
  return uint64_t((addr >> 4) & 0x3FFFu) | (uint64_t(dims64 >> 4) << 16) | (uint64_t(rows8 >> 4) << 32) | (uint64_t(1) << 46) |
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

// A place in the ring: its stage and the parity of the lap that fills it.
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

// One page's keys (64 of a longer one) of a head, by groups of 8: the map's dims are 64 dims of a row, 8 rows, the row's
// D / 64 parts, heads, and groups of 8 tokens of the pool.
__device__ __forceinline__ void tma_box(uint32_t dst, const CUtensorMap* map, int head, int group, uint64_t* bar) {
  asm volatile(
      "cp.async.bulk.tensor.5d.shared::cluster.global.tile.mbarrier::complete_tx::bytes [%0], [%1, {%2, %2, %2, %3, %4}], "
      "[%5];" ::"r"(dst),
      "l"(reinterpret_cast<uint64_t>(map)), "r"(0), "r"(head), "r"(group), "r"(smem_u32(bar))
      : "memory");
}

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

// What the softmax warpgroup does: the tile's queries into shared memory, then every step's probabilities and sum, and at the
// end its rows of O (or of a part) to memory. Thread = row = lane of tensor memory.
template <int KIND, int D, bool CAP, bool SLOPED>
__device__ __forceinline__ void softmax_rows(const PrefillArgs& a, const TileAt& at, const RowAt& row, int hk, int sp, int parts,
                                             int from, int steps, uint32_t tmem, uint8_t* smem, uint64_t* q_full,
                                             uint64_t* s_full, uint64_t* p_full, uint64_t* o_done, const uint32_t* flags) {
  using S = TcShape<KIND, D>;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, r = threadIdx.x;
  float q_unit = 1.f;
  {
    // 32 / CPR rows per pass of the warp, a row's 16-byte chunks side by side
    constexpr int CPR = D / 8, RPP = 32 / CPR;
    uint8_t* tile = smem;
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
      *reinterpret_cast<uint4*>(tile + (c >> 3) * (kRows * 128) + rr * 128 + (((c & 7) ^ (rr & 7)) << 4)) = x[k];
    }
    fence_proxy_async_shared();
    __syncwarp();
    if (lane == 0) mbar_arrive(q_full);
  }
  const float raw = a.sm_scale * a.src.k_scale * q_unit;  // a product as a score
  const float mul = CAP ? raw * 2.f * kLog2e / a.softcap : raw * kLog2e;
  const float cap_out = a.softcap * kLog2e;
  const float mul_now = CAP || SLOPED ? 1.f : mul;  // what is left to multiply once a product has its shape
  const int all_lo = __reduce_max_sync(0xffffffffu, row.lo), all_hi = __reduce_min_sync(0xffffffffu, row.hi);
  const uint32_t lanes = uint32_t(32 * warp) << 16, o_at = tmem + lanes + S::kO;

  float m = -INFINITY;  // the maximum in use
  float l = 0.f;
  bool ok = true;
  for (int j = 0; j < steps; ++j) {
    const int key0 = from + (steps - 1 - j) * kKeys;
    const uint32_t s_at = tmem + lanes + 64 * (j & 1), phase = (j >> 1) & 1;
    ok = __all_sync(0xffffffffu, mbar_wait(&s_full[j & 1], phase));
    if (!ok) break;
    tc_fence_after();
    const uint32_t bad = flags[j & (kFlagSteps - 1)];
    const bool masked = bad != 0u || key0 < all_lo || key0 + kKeys > all_hi;
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
        const uint32_t w = bad >> (c >> 3);
#pragma unroll
        for (int e = 0; e < 32; ++e)
          if (e < below || e >= above || (w >> (e >> 3) & 1u)) x[e] = 0xFF800000u;
      }
    };
    // P = 2^(s - m), rounded to 16 bits (as any operand of these matrix instructions), and the fp32 sum of what was rounded.
    uint32_t p[32];
    auto powers = [&](float off, auto with_mask) {
      float2 sum = make_float2(0.f, 0.f);
      uint32_t x[64];
      tmem_load64(s_at, x);
#pragma unroll
      for (int k = 0; k < 2; ++k) {
        shape(32 * k, x + 32 * k, with_mask);
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
    // a row that has met no key yet meets some in this step: its first maximum
    const bool fresh = m == -INFINITY && row.lo < key0 + kKeys && row.hi > key0;
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
      // a first step, and a few later ones: the row's maximum is looked up and moves
      float top = -INFINITY;
#pragma unroll 1
      for (int c = 0; c < kKeys; c += 32) {
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
      if (j > 0) {  // the step before this one is in O
        ok = __all_sync(0xffffffffu, mbar_wait(&o_done[(j - 1) & 1], ((j - 1) >> 1) & 1u));
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
    tmem_store32(s_at, p);
    tmem_wait_store();
    tc_fence_before();
    __syncwarp();
    if (lane == 0) mbar_arrive(&p_full[j & 1]);
  }
  const int n = steps;
  if (ok && n > 0) ok = __all_sync(0xffffffffu, mbar_wait(&o_done[(n - 1) & 1], ((n - 1) >> 1) & 1u));
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
  uint8_t* stage = smem + warp * (32 * 2 * D);
  const int c = lane % CPR;
  const int64_t out0 = (int64_t(at.token0 + at.row0 / a.rep) * a.Hq + hk * a.rep) * (2 * D);  // of the tile's first row, in bytes
  const int64_t part0 = ((tile * a.n_splits + sp) * kRows + 32 * warp) * (4 * D);  // of the warp's first row
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
                                 : static_cast<uint8_t*>(a.out) + out0 + int64_t((code >> 16) * a.Hq + (code & 0xFFFF)) * (2 * D);
        *reinterpret_cast<uint4*>(dst + 16 * c) = x;
      }
    }
    __syncwarp();
  }
  if (ok && parts > 1 && row.code >= 0)
    a.part_lse[(tile * a.n_splits + sp) * kRows + r] = l == 0.f ? -INFINITY : (m == -INFINITY ? 0.f : m) + log2f(l);
}

// CAP: scores are capped. SLOPED: they fall with distance, or their factor is not positive (a maximum of products is then no
// maximum of scores).
template <int KIND, int D, bool CAP, bool SLOPED>
__global__ void __launch_bounds__(kThreads, 2)
    paged_prefill_tc_kernel(const PrefillArgs a, const __grid_constant__ CUtensorMap tm_k, const __grid_constant__ CUtensorMap tm_v) {
  using S = TcShape<KIND, D>;
  constexpr int NS = S::kStages;
  extern __shared__ __align__(1024) uint8_t smem[];
  uint8_t* ring = smem + S::kQ;
  uint64_t* bars = reinterpret_cast<uint64_t*>(ring + NS * S::kStage);
  uint64_t* full = bars;             // [NS] a stage's rows have landed
  uint64_t* empty = full + NS;       // [NS] the products that read it are done
  uint64_t* q_full = empty + NS;     // the queries are in shared memory
  uint64_t* s_full = q_full + 1;     // [2] S is in its buffer: the products' completion, and the issuing thread (which has
                                     //     waited for the keys, and so seen their flags)
  uint64_t* p_full = s_full + 2;     // [2] P is in its buffer, O rescaled where needed
  uint64_t* o_done = p_full + 2;     // [2] that buffer's P V is in O
  uint64_t* drained = o_done + 2;    // all products are done
  uint64_t* edge = drained + 1;      // a stage whose rows are only partly visible has landed
  uint64_t* raw = edge + 1;          // [NS] a stage's codes have landed (E4M3)
  uint32_t* flags = reinterpret_cast<uint32_t*>(bars + S::kBars);  // [kFlagSteps] a bit per 8 keys of a block out of range
  int* range = reinterpret_cast<int*>(flags + kFlagSteps);          // the smallest lo, the largest hi
  uint32_t* slot = reinterpret_cast<uint32_t*>(range + 2);          // tensor-memory address
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, wg = warp >> 2;
  const int hk = blockIdx.y, sp = blockIdx.z;

  if (smem_u32(smem) & 1023u) {  // (dynamic shared memory starts there: the kernel has no other)
    if (tid == 0) record_error(kDevErrTimeout);
    return;
  }
  if (tid == 32 || tid == 64)  // (a first box waits for its map)
    asm volatile("prefetch.tensormap [%0];" ::"l"(reinterpret_cast<uint64_t>(tid == 32 ? &tm_k : &tm_v)) : "memory");
  if (tid == 0) {
    for (int i = 0; i < NS; ++i) {
      mbar_init(&full[i], kIs16<KIND> ? 1 : 2);
      mbar_init(&empty[i], 1);
      if constexpr (!kIs16<KIND>) mbar_init(&raw[i], 1);
    }
    mbar_init(q_full, 4);
    for (int i = 0; i < 2; ++i) {
      mbar_init(&s_full[i], 2);
      mbar_init(&p_full[i], 4);
      mbar_init(&o_done[i], 1);
    }
    mbar_init(drained, 1);
    mbar_init(edge, 1);
    range[0] = INT_MAX;
    range[1] = 0;
    fence_mbar_init();
  }
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

  // the tile's rows: thread r of the softmax warpgroup holds row r
  RowAt row{-1, -1, -1, 0, 0, 0, 0.f};
  if (wg == 0) {
    row = row_at(a, at, at.row0 + tid, hk, len);
    const bool any = row.hi > row.lo;
    const int lo = __reduce_min_sync(0xffffffffu, any ? row.lo : INT_MAX);
    const int hi = __reduce_max_sync(0xffffffffu, any ? row.hi : 0);
    if (lane == 0 && hi > 0) {
      atomicMin(&range[0], lo);
      atomicMax(&range[1], hi);
    }
  } else if (warp == 7) {
    asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(slot)), "r"(S::kColumns)
                 : "memory");
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = *slot;
  // Every CTA of this grid holds its tensor memory (or has left) before any dependent CTA can start: one that allocated
  // columns which a CTA here still needs would wait for this grid's end, and this grid for the columns.
  pdl_launch_dependents();
  auto free_tmem = [&]() {
    asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(S::kColumns) : "memory");
  };
  const int lo = range[0], hi = range[1];
  const int base = lo == INT_MAX ? 0 : lo & ~(kKeys - 1);
  const int parts = hi > base ? min(a.n_splits, (hi - base + a.split - 1) / a.split) : 0;
  if (a.n_splits > 1 && sp == 0 && tid == 0) a.part_count[tile] = parts;
  if (sp >= max(parts, 1)) {
    if (warp == 7) free_tmem();
    return;
  }
  const int from = base + sp * a.split;
  const int to = parts == 0 ? from : sp == parts - 1 ? hi : from + a.split;
  const int steps = (to - from + kKeys - 1) / kKeys;
  // Ring items in the order that the products take them: K 0, K 1, then V j, K j + 2 for every step j.
  const int items = 2 * steps;
  auto step_of = [&](int n) { return n < 2 ? n : n & 1 ? (n + 1) >> 1 : (n - 2) >> 1; };  // (n odd from 3 on: K)
  auto is_v = [&](int n) { return n >= 2 && (n & 1) == 0; };

  if (wg == 1) {
    asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(S::kOtherRegs));
    if (warp < 4 + S::kProducers) {
      // ---- producers
      const int w = warp - 4;
      const int32_t* table = a.src.block_table + int64_t(b) * a.src.bt_stride;
      const int take_from = max(from, lo);
      // A step's pages: 64 / page size of them (one where pages are longer).
      const int page_log2 = min(a.src.bs_log2, 6), per_log2 = 6 - page_log2, window_log2 = 5 - per_log2;
      auto block_at = [&](int key) -> int {  // -1: no key is visible there, -2: the table names a block out of range
        if (key >= to || key + (1 << page_log2) <= take_from) return -1;
        const int blk = table[key >> a.src.bs_log2];
        if (blk < 0 || blk >= a.src.num_blocks) {
          record_error(kDevErrBlockIndex);
          return -2;
        }
        return blk;
      };
      // Lane i of a window holds page i mod per_step of step first + i / per_step; the next window is loaded while this one is
      // in use.
      auto window = [&](int first) {
        const int back = steps - 1 - first - (lane >> per_log2);  // steps go from the last keys to the first
        return back < 0 ? -1 : block_at(from + (back << 6) + ((lane & ((1 << per_log2) - 1)) << page_log2));
      };
      int k_held = window(0), k_next = window(1 << window_log2), v_held = k_held, v_next = k_next;
      // this lane's page (lane < pages) of step j
      auto page_of = [&](int j, bool v) {
        const int in = j & ((1 << window_log2) - 1);
        if (in == 0 && j > 0) {
          if (v) {
            v_held = v_next;
            v_next = window(j + (1 << window_log2));
          } else {
            k_held = k_next;
            k_next = window(j + (1 << window_log2));
          }
        }
        return __shfl_sync(0xffffffffu, v ? v_held : k_held, (in << per_log2) + (lane & ((1 << per_log2) - 1)));
      };
      // the bits of a step's 8-key units whose block is out of range
      auto flag = [&](int j, int blk) {
        const uint32_t wrong = __ballot_sync(0xffffffffu, blk == -2) & ((1u << (1 << per_log2)) - 1u);
        uint32_t bits = 0;
        if (wrong)
          for (int u = 0; u < 8; ++u) bits |= (wrong >> (u >> (page_log2 - 3)) & 1u) << u;
        if (lane == 0) flags[j & (kFlagSteps - 1)] = bits;
      };
      Item<NS> in;
      bool ok = true;
      if constexpr (kIs16<KIND>) {
        // warp 4 brings K, warp 5 V: every second item of the ring
        const bool v = w == 1;
        const int pages = 1 << per_log2, nowhere = int(a.src.num_blocks << (a.src.bs_log2 - 3));  // a group behind the pool
        const CUtensorMap* map = v ? &tm_v : &tm_k;
        uint32_t edges = 0, asked = 0, laps = 0;  // bits of stages: a copy was asked for, the lap of the last
        int n = v ? min(2, steps) : 0;  // the item of step j
        for (int i = 0; i < n; ++i) in.next();
        for (int j = 0; j < steps; ++j) {
          const int blk = page_of(j, v);
          if (!v) flag(j, blk);
          const int key0 = from + kKeys * (steps - 1 - j);
          const int group =
              blk >= 0 ? (blk << (a.src.bs_log2 - 3)) + ((key0 & ((1 << a.src.bs_log2) - 1)) >> 6 << 3) : nowhere;
          const bool partly = v && (key0 < take_from || key0 + kKeys > to);
          uint64_t* bar = partly ? edge : &full[in.stage];
          const uint32_t dst = smem_u32(ring + in.stage * S::kStage);
          if (n >= NS) ok = __all_sync(0xffffffffu, mbar_wait(&empty[in.stage], in.lap ^ 1u));
          if (!ok) break;
          if (lane == 0) mbar_arrive_expect_tx(bar, S::kStage);
          __syncwarp();
          if (lane < pages)  // (a page that is not there lies behind the pool: its box becomes zeros)
            tma_box(dst + (lane << (page_log2 - 3)) * S::kGroup, map, hk, group, bar);
          if (partly) {  // values next to the visible ones may be anything: their rows become zeros, as P's columns are there
            ok = __all_sync(0xffffffffu, mbar_wait(edge, edges & 1u));
            ++edges;
            if (!ok) break;
            for (int i = lane; i < kKeys * (D / 8); i += 32) {
              const int r = i / (D / 8), c = i % (D / 8);
              if (key0 + r < take_from || key0 + r >= to)
                *reinterpret_cast<uint4*>(ring + in.stage * S::kStage + (r >> 3) * S::kGroup + (c >> 3) * 1024 + (r & 7) * 128 + (c & 7) * 16) =
                    make_uint4(0u, 0u, 0u, 0u);
            }
            fence_proxy_async_shared();
            __syncwarp();
            if (lane == 0) mbar_arrive(&full[in.stage]);
          }
          asked |= 1u << in.stage;
          laps = (laps & ~(1u << in.stage)) | in.lap << in.stage;
          const int ahead = v ? (j == steps - 2 ? 1 : 2) : (j == 0 ? 1 : 2);
          n += ahead;
          in.next();
          if (ahead == 2) in.next();
        }
        // (a wait ran out: the copies asked for land before the CTA ends)
        if (!ok)
          for (int i = 0; i < NS; ++i)
            if (asked >> i & 1u) (void)mbar_wait(&full[i], laps >> i & 1u);
      } else {
        // Warp 6 brings the codes, 8 keys a TMA box, a lane a box, into the second half of the place that their f16 values
        // take; warps 4 and 5 then take four of the eight places each, two at a time: codes into registers, f16 back. (One
        // warp that both brought and converted left the ring empty while it waited: heads of 128 took half as long again.)
        constexpr int CPR = D / 16, PER = CPR * 8 / 32;  // 16-byte chunks of a key's codes; a lane's of 8 keys
        auto order = [&](int n, int& j, bool& v) {
          v = is_v(n) || n >= 2 * steps - 1;
          j = n >= 2 * steps - 1 ? steps - 1 : step_of(n);
        };
        if (w == 2) {
          const int nowhere = int(a.src.num_blocks << (a.src.bs_log2 - 3));  // a group behind the pool
          int n = 0;
          for (; n < items; ++n) {
            int j;
            bool v;
            order(n, j, v);
            const int blk = page_of(j, v);
            if (!v) flag(j, blk);
            const int key = from + kKeys * (steps - 1 - j) + 8 * (lane & 7);
            const int blk8 = __shfl_sync(0xffffffffu, blk, (lane & 7) >> (page_log2 - 3));
            const int group =
                blk8 >= 0 ? (blk8 << (a.src.bs_log2 - 3)) + ((key & ((1 << a.src.bs_log2) - 1)) >> 3) : nowhere;
            if (n >= NS) ok = __all_sync(0xffffffffu, mbar_wait(&empty[in.stage], in.lap ^ 1u));
            if (!ok) break;
            if (lane == 0) mbar_arrive_expect_tx(&raw[in.stage], kKeys * D);
            __syncwarp();
            if (lane < 8)
              tma_box(smem_u32(ring + in.stage * S::kStage) + lane * S::kGroup + 8 * D, v ? &tm_v : &tm_k, hk, group,
                      &raw[in.stage]);
            in.next();
          }
          // (a wait ran out: the copies asked for land before the CTA ends)
          if (!ok)
            for (int i = 0; i < NS; ++i)
              if (i < n) (void)mbar_wait(&raw[i], i < in.stage ? in.lap : in.lap ^ 1u);
        } else {
          for (int n = 0; n < items; ++n) {
            ok = __all_sync(0xffffffffu, mbar_wait(&raw[in.stage], in.lap));
            if (!ok) break;
            int j;
            bool v;
            order(n, j, v);
            const int key0 = from + kKeys * (steps - 1 - j);
            const bool partly = v && (key0 < take_from || key0 + kKeys > to);
#pragma unroll
            for (int i = 0; i < 4; i += 2) {
              uint8_t* const rows = ring + in.stage * S::kStage + (4 * w + i) * S::kGroup;
              uint4 x[2][PER];
#pragma unroll
              for (int k = 0; k < 2; ++k)
#pragma unroll
                for (int e = 0; e < PER; ++e)
                  x[k][e] = *reinterpret_cast<const uint4*>(rows + k * S::kGroup + 8 * D + (lane + 32 * e) * 16);
              if (partly) {  // values next to the visible ones may be anything: zeros
#pragma unroll
                for (int k = 0; k < 2; ++k)
#pragma unroll
                  for (int e = 0; e < PER; ++e) {
                    const int key = key0 + 8 * (4 * w + i + k) + (lane + 32 * e) / CPR;
                    if (key < take_from || key >= to) x[k][e] = make_uint4(0u, 0u, 0u, 0u);
                  }
              }
              __syncwarp();  // the warp has these codes: their places may be written
#pragma unroll
              for (int k = 0; k < 2; ++k)
#pragma unroll
                for (int e = 0; e < PER; ++e) {
                  const int r = (lane + 32 * e) / CPR, c = (lane + 32 * e) % CPR;
                  const uint32_t u[4] = {x[k][e].x, x[k][e].y, x[k][e].z, x[k][e].w};
                  uint8_t* dst = rows + k * S::kGroup + ((2 * c) >> 3) * 1024 + r * 128;
#pragma unroll
                  for (int h = 0; h < 2; ++h) {
                    const uint2 x0 = codes_to_f16<KIND>(u[2 * h]), x1 = codes_to_f16<KIND>(u[2 * h + 1]);
                    *reinterpret_cast<uint4*>(dst + ((((2 * c + h) & 7) ^ r) << 4)) = make_uint4(x0.x, x0.y, x1.x, x1.y);
                  }
                }
            }
            fence_proxy_async_shared();
            __syncwarp();
            if (lane == 0) mbar_arrive(&full[in.stage]);
            in.next();
          }
        }
      }
    } else if (warp == 7) {
      // ---- matrix products: the whole warp waits, one of its threads issues
      constexpr uint32_t id_s = tc_idesc<KIND>(kRows, kKeys, false), id_o = tc_idesc<KIND>(kRows, D, true);
      const uint64_t q_desc = desc_along(smem_u32(smem), 1024), k_desc = desc_along(smem_u32(ring), S::kGroup),
                     v_desc = desc_across(smem_u32(ring), S::kGroup, 1024);
      Item<NS> item;
      bool ok = true;
      auto wait = [&](uint64_t* bar, uint32_t parity) { ok = ok && __all_sync(0xffffffffu, mbar_wait(bar, parity)); };
      auto scores = [&](int j) {  // S = Q K^T of step j
        wait(&full[item.stage], item.lap);
        if (!ok) return;
        tc_fence_after();
        if (elect_one()) {
          const uint64_t kd = k_desc + uint32_t(item.stage * (S::kStage >> 4));
#pragma unroll
          for (int k = 0; k < D / 16; ++k) {
            const uint32_t at_k = (k & 3) * (32 >> 4);
            tc_mma_ss(tmem + 64 * (j & 1), q_desc + (k >> 2) * (kRows * 128 >> 4) + at_k, kd + (k >> 2) * (1024 >> 4) + at_k,
                      id_s, k > 0 ? 1u : 0u);
          }
          tc_commit(&s_full[j & 1]);
          mbar_arrive(&s_full[j & 1]);
          tc_commit(&empty[item.stage]);
        }
        __syncwarp();
        item.next();
      };
      if (steps > 0) wait(q_full, 0u);
      if (steps > 0 && ok) scores(0);
      if (steps > 1 && ok) scores(1);
      for (int j = 0; j < steps && ok; ++j) {  // O += P V of step j, then S of step j + 2 over the P that it took
        wait(&full[item.stage], item.lap);
        wait(&p_full[j & 1], (j >> 1) & 1u);
        if (!ok) break;
        tc_fence_after();
        if (elect_one()) {
          const uint64_t vd = v_desc + uint32_t(item.stage * (S::kStage >> 4));
#pragma unroll
          for (int k = 0; k < kKeys / 16; ++k)
            tc_mma_ts(tmem + S::kO, tmem + 64 * (j & 1) + 8 * k, vd + k * (2 * S::kGroup >> 4), id_o, k > 0 || j > 0 ? 1u : 0u);
          tc_commit(&o_done[j & 1]);
          tc_commit(&empty[item.stage]);
        }
        __syncwarp();
        item.next();
        if (j + 2 < steps) scores(j + 2);
      }
      if (elect_one()) tc_commit(drained);
      __syncwarp();
    }
  } else {
    asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(S::kSoftmaxRegs));
    softmax_rows<KIND, D, CAP, SLOPED>(a, at, row, hk, sp, parts, from, steps, tmem, smem, q_full, s_full, p_full, o_done, flags);
  }
  __syncwarp();
  tc_fence_before();
  __syncthreads();
  if (warp == 7) {
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
  CUtensorMap tm_k, tm_v;
  auto encode = reinterpret_cast<PFN_cuTensorMapEncodeTiled_v12000>(tensor_map_encoder());
  if (!encode) return set_error(BPT_ERR_UNSUPPORTED, "paged prefill: the driver has no tensor-map encoder");
  const int64_t groups = a.src.num_blocks << (a.src.bs_log2 - 3);
  BPT_REQUIRE(groups < (1ll << 31) - 1, BPT_ERR_UNSUPPORTED, "paged prefill: a pool of %lld tokens", (long long)groups * 8);
  // 16-bit pages: a box has a row's parts of 64 dims one after another, swizzled; codes: rows as they are, 8 a box
  constexpr bool k16 = kIs16<KIND>;
  const cuuint64_t row = cuuint64_t(S::kRowBytes), token = row * a.src.Hkv;
  const cuuint64_t dims[5] = {k16 ? 64 : D, 8, k16 ? D / 64 : 1, cuuint64_t(a.src.Hkv), cuuint64_t(groups)};
  const cuuint64_t strides[4] = {token, k16 ? 128 : row, row, 8 * token};
  const cuuint32_t box[5] = {k16 ? 64 : D, 8, k16 ? D / 64 : 1, 1, k16 ? 1u << (std::min(a.src.bs_log2, 6) - 3) : 1u};
  const cuuint32_t ones[5] = {1, 1, 1, 1, 1};
  const CUtensorMapDataType type = KIND == BPT_KV_FP8   ? CU_TENSOR_MAP_DATA_TYPE_UINT8
                                   : KIND == BPT_KV_F16 ? CU_TENSOR_MAP_DATA_TYPE_FLOAT16
                                                        : CU_TENSOR_MAP_DATA_TYPE_BFLOAT16;
  for (int i = 0; i < 2; ++i) {
    const CUresult res = encode(i ? &tm_v : &tm_k, type, 5, const_cast<uint8_t*>(i ? a.src.v_pool : a.src.k_pool), dims, strides,
                                box, ones, CU_TENSOR_MAP_INTERLEAVE_NONE,
                                k16 ? CU_TENSOR_MAP_SWIZZLE_128B : CU_TENSOR_MAP_SWIZZLE_NONE,
                                CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
    if (res != CUDA_SUCCESS) return set_error(BPT_ERR_INVALID, "paged prefill: tensor map: error %d", int(res));
  }
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
  const cudaError_t err = cudaLaunchKernelEx(&cfg, paged_prefill_tc_kernel<KIND, D, CAP, SLOPED>, a, tm_k, tm_v);
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
  auto of = [&](auto k) {
    constexpr int K = decltype(k)::value;
    if (a.D == 64) return launch_shape<K, 64>(a, tiles, flags, stream);
    if (a.D == 128) return launch_shape<K, 128>(a, tiles, flags, stream);
    return launch_shape<K, 256>(a, tiles, flags, stream);
  };
  if (kind == BPT_KV_FP8) return of(std::integral_constant<int, BPT_KV_FP8>());
  if (kind == BPT_KV_F16) return of(std::integral_constant<int, BPT_KV_F16>());
  return of(std::integral_constant<int, BPT_KV_BF16>());
}

}  // namespace bpt
