// Decode attention over a paged cache of any format, with score caps, distance bias, sliding windows and a first visible
// key: one query token per sequence.
//
//   s_j = cap tanh(scale q.k_j / cap) - slope |p - j|,  out = sum_j softmax(s)_j v_j  over  max(0, start, p - window + 1) <= j
//   <= p, p = length - 1; no visible key gives 0.
//
// Bound by memory: each visible key and value is read once. Work is cut into equal shares, one per warp of a full GPU (two
// CTAs of four warps an SM; one CTA where rows of 512 bytes leave no room): a warp takes a contiguous range of groups of 16 keys, of one KV head (and eight of its query heads), across the
// sequences of the batch, so that ragged lengths leave no SM idle; the warps of a CTA hold the heads of one range, whose rows
// lie next to each other in the pages. A warp never waits for another: it has its own ring of cp.async stages, running on
// into its next sequence, and its own running maximum and sum. A group's rows arrive whole (D elements of one head); rows
// outside the visible run are not read, their places hold zeros.
//
// The eight query heads fill only half of an MMA's 16 rows, so the other half carries what rounding takes off: rows 0-7 hold q
// (then the probabilities) rounded to the product's 16-bit type, rows 8-15 the rounded-off rest, and both halves' sums
// are added in fp32. Products are thus good to 16 (bf16) or 22 bits at no cost; f16 probabilities stand at up to 2^15, so that
// a long tail far below the largest keeps its bits too.
// INT8 pages have a scale per key: K's goes on the score, V's on the probability, and a power of two per row keeps a row's
// largest such product in f16's range however small the values are (5% of the time of 8 sequences of 32,768).
//
// A sequence inside one range goes straight to out. One that crosses ranges leaves a part per range, and a second kernel,
// launched dependently, joins them.
//
// Measured (B200, 6,558 GB/s copy; captured): f16, 8 sequences of 32,768, 32 query and 8 KV heads of 128, capped: 186 us,
// 5.8 TB/s (INT8 156 us, 3.5 TB/s); bf16, 32 sequences of 512 to 4,096: 62 us, 4.9 TB/s (start and join); E4M3 in a window of
// 4,096, 17 sequences: 32 us, 1.8 TB/s, bound by the latency of a warp's chain at 8 warps an SM (0.3 instructions a cycle, no
// pipe above 14%); one sequence of 1,000: 14 us, two launches and a dependent chain of loads. A ring of six stages with one
// CTA an SM took 73 us for the batch of 32.
#include <algorithm>

#include "paged_read.cuh"

namespace bpt {

namespace {

constexpr int kWarps = 4;          // per CTA, at most
// What a sequence's start costs a range, in groups of 16 keys. (8: one sequence of 1,000 takes 20.6 us instead of 14.7.)
constexpr int kStartCost = 2;
constexpr int kLeastShare = 2;     // groups; a smaller share would be all start and join

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
  int B, Hq, rep, tiles, heads;  // tiles: groups of 8 query heads per KV head; heads = Hkv * tiles
  int ranges;
  void* out;
  int out_dtype;
  // merged: parts[ranges][heads][2] (0: of the sequence that a range continues, 1: of the one it leaves unfinished), each
  // o [8][D] and base-2 log-sum-exps [8]; meta[places][heads]: a sequence in several ranges as (itself, its first range, its
  // last), (-1, ., .) for none. A place is a sequence where there are no more of them than ranges, else the range that it
  // starts in: the second kernel has a CTA per place and head.
  float* ws_out;
  float* ws_lse;
  int4* ws_meta;
  int by_sequence;
  // partials: out [B, Hq, n_splits, D], lse [B, Hq, n_splits] (natural logarithm) of `split` keys each
  float* part_out;
  float* part_lse;
  int split, n_splits;
};

__device__ __forceinline__ void store_any(void* p, int dtype, int64_t i, float v) {
  if (dtype == BPT_DTYPE_F32) static_cast<float*>(p)[i] = v;
  else if (dtype == BPT_DTYPE_F16) static_cast<__half*>(p)[i] = __float2half_rn(v);
  else static_cast<__nv_bfloat16*>(p)[i] = __float2bfloat16_rn(v);
}

// Two neighbouring elements (the first at an even index) as floats.
template <int DT>
__device__ __forceinline__ float2 load_pair(const void* p, int64_t i) {
  if constexpr (DT == BPT_DTYPE_F32) return *reinterpret_cast<const float2*>(static_cast<const float*>(p) + i);
  const uint32_t u = *reinterpret_cast<const uint32_t*>(static_cast<const uint16_t*>(p) + i);
  return DT == BPT_DTYPE_F16 ? unpack2<BPT_KV_F16>(u) : unpack2<BPT_KV_BF16>(u);
}

// The A fragments of one query row per lane quad: rounded to the product's type in rows 0-7, what rounding took off in rows
// 8-15. For f16 products q is scaled by a power of two into [-1, 1]; returns what undoes it. Every load of a pass is in flight
// at once (the second pass finds the row in L1).
template <int KIND, int D, int DT>
__device__ __forceinline__ float query_rows(const void* q, int64_t at, int t, bool here, uint32_t (&qf)[D / 16][4]) {
  constexpr bool kExact = DT == BPT_DTYPE_BF16 || (DT == BPT_DTYPE_F16 && KIND != BPT_KV_BF16);  // rounding takes nothing off
  float2 unit = make_float2(1.f, 1.f);
  if constexpr (KIND != BPT_KV_BF16 && DT != BPT_DTYPE_F16) {
    float amax = 0.f;
    if (here) {
#pragma unroll
      for (int j = 0; j < D / 16; ++j)
#pragma unroll
        for (int i = 0; i < 2; ++i) {
          const float2 x = load_pair<DT>(q, at + q_dim<KIND>(j, t, 2 * i));
          amax = fmaxf(amax, fmaxf(fabsf(x.x), fabsf(x.y)));
        }
    }
    amax = fmaxf(amax, __shfl_xor_sync(0xffffffffu, amax, 1));
    amax = fmaxf(amax, __shfl_xor_sync(0xffffffffu, amax, 2));
    unit = unit_range(amax);
  }
#pragma unroll
  for (int j = 0; j < D / 16; ++j)
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      float2 x = make_float2(0.f, 0.f);
      if (here) x = load_pair<DT>(q, at + q_dim<KIND>(j, t, 2 * i));
      x.x *= unit.x;
      x.y *= unit.x;
      qf[j][2 * i] = pack2<KIND>(x.x, x.y);
      const float2 r = unpack2<KIND>(qf[j][2 * i]);
      qf[j][2 * i + 1] = kExact ? 0u : pack2<KIND>(x.x - r.x, x.y - r.y);
    }
  return unit.y;
}

template <int KIND, int D>
struct ReadShape {
  static constexpr int RB = D * kElemBytes<KIND>;
  static constexpr int kScaleBytes = KIND == BPT_KV_INT8 ? 64 : 0;  // 16 K and 16 V scales (fp16) of a group
  static constexpr int kStage = 2 * 16 * RB + kScaleBytes + 16;  // keys, values, scales, the bad-block flag
  // Stages per warp: what keeps the memory busy. 16-bit heads of 128: 3 stages x 8 KB x 4 warps = 96 KB, two CTAs per SM.
  static constexpr int kStages = RB >= 512 ? 3 : RB == 256 ? 3 : 4;
  static constexpr int kPerWarp = kStages * kStage;
  static constexpr int kSmem = kWarps * kPerWarp;
  static constexpr int kCtas = RB >= 512 ? 1 : 2;  // per SM
};

// The visible keys of a sequence, cut to the pages that its table has.
struct Visible {
  int pos, lo, hi, base, groups;  // base: lo rounded down to a group; groups of 16 keys from there to hi
};
__device__ __forceinline__ Visible visible_keys(const ReadArgs& a, int b, bool tells = false) {
  Visible v;
  const int room = int(min(int64_t(a.src.bt_width) << a.src.bs_log2, int64_t(1) << 30));
  const int whole = a.lengths[b], len = min(whole, room);
  if (tells && whole > room) record_error(kDevErrBlockIndex);  // more tokens than the table has pages for
  v.pos = len - 1;
  v.lo = a.key_starts ? max(a.key_starts[b], 0) : 0;
  if (a.window > 0) v.lo = max(v.lo, v.pos - a.window + 1);
  v.hi = max(len, 0);
  v.base = v.lo & ~15;
  v.groups = v.hi > v.lo ? (v.hi - v.base + 15) >> 4 : 0;
  return v;
}

// A warp's walk over the sequences of its range [begin, end) of costs: sequence b starts at cost `at`, its groups at
// at + kStartCost.
struct Walk {
  int b;
  int64_t at;
  Visible v;
  int g0, g1;  // its groups in the range
  __device__ __forceinline__ void enter(const ReadArgs& a, int64_t begin, int64_t end) {
    v = visible_keys(a, b);
    const int64_t start = at + kStartCost;
    g0 = int(min(max(begin - start, int64_t(0)), int64_t(v.groups)));
    g1 = int(min(max(end - start, int64_t(0)), int64_t(v.groups)));
  }
  __device__ __forceinline__ void leave() {
    at += kStartCost + v.groups;
    ++b;
  }
};

template <int KIND, int D, bool MERGE>
__global__ void __launch_bounds__(32 * kWarps, ReadShape<KIND, D>::kCtas) paged_read_kernel(const ReadArgs a) {
  using S = ReadShape<KIND, D>;
  constexpr int RB = S::RB, NST = S::kStages;
  extern __shared__ __align__(1024) uint8_t smem[];
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, g = lane >> 2, t = lane & 3;
  pdl_launch_dependents();
  pdl_wait();
  const int64_t id = int64_t(blockIdx.x) * (blockDim.x >> 5) + warp;
  const int64_t unit = id / a.heads;
  const int ht = int(id - unit * a.heads), hk = ht / a.tiles, tile = ht - hk * a.tiles;
  if (unit >= (MERGE ? int64_t(a.ranges) : int64_t(a.B) * a.n_splits)) return;
  const int h0 = hk * a.rep + tile * 8;        // this warp's first query head
  const int heads = min(8, a.rep - tile * 8);  // and how many

  Walk use;  // the sequence whose groups are multiplied
  int64_t begin = 0, end = 0, share = 1;
  const int range = int(unit);
  int sp = 0;
  if constexpr (MERGE) {
    int64_t total = 0;
    int mine = 0;  // of the first 32 sequences
    for (int b0 = 0; b0 < a.B; b0 += 32) {
      const int groups = b0 + lane < a.B ? kStartCost + visible_keys(a, b0 + lane, id == 0).groups : 0;
      if (b0 == 0) mine = groups;
      total += groups;
    }
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) total += __shfl_xor_sync(0xffffffffu, total, o);
    share = max((total + a.ranges - 1) / a.ranges, int64_t(kStartCost + kLeastShare));
    begin = range * share;
    end = min(begin + share, total);
    if (a.ranges > 1 && !a.by_sequence && lane == 0) a.ws_meta[id] = make_int4(-1, 0, 0, 0);
    if (begin >= total) return;
    int64_t before = 0;  // the sequence that holds cost `begin`
    for (int b0 = 0;; b0 += 32) {
      int upto = b0 == 0 ? mine : b0 + lane < a.B ? kStartCost + visible_keys(a, b0 + lane).groups : 0;
      const int own = upto;
#pragma unroll
      for (int o = 1; o < 32; o <<= 1) {
        const int x = __shfl_up_sync(0xffffffffu, upto, o);
        if (lane >= o) upto += x;
      }
      const unsigned hit = __ballot_sync(0xffffffffu, before + upto > begin);
      if (hit) {
        const int w = __ffs(hit) - 1;
        use.b = b0 + w;
        use.at = before + __shfl_sync(0xffffffffu, upto - own, w);
        break;
      }
      before += __shfl_sync(0xffffffffu, upto, 31);
    }
    use.enter(a, begin, end);
  } else {
    use.b = int(unit / a.n_splits);
    use.at = 0;
    sp = int(unit - int64_t(use.b) * a.n_splits);
    use.v = visible_keys(a, use.b, lane == 0 && sp == 0 && ht == 0);
    const int64_t from = int64_t(sp) * a.split, to = sp == a.n_splits - 1 ? int64_t(use.v.hi) : from + a.split;
    use.v.lo = int(max(int64_t(use.v.lo), min(from, int64_t(use.v.hi))));
    use.v.hi = int(min(int64_t(use.v.hi), to));
    use.v.base = use.v.lo & ~15;
    use.v.groups = use.v.hi > use.v.lo ? (use.v.hi - use.v.base + 15) >> 4 : 0;
    use.g0 = 0;
    use.g1 = use.v.groups;
  }

  uint8_t* ring = smem + warp * S::kPerWarp;
  const uint32_t ring_u = smem_u32(ring);
  auto scales_of = [&](int st) { return reinterpret_cast<uint16_t*>(ring + st * S::kStage + 32 * RB); };
  auto flag_of = [&](int st) { return reinterpret_cast<uint32_t*>(ring + st * S::kStage + 32 * RB + S::kScaleBytes); };
  // The loader runs NST - 1 groups ahead of the products, into the sequences that follow.
  GroupLoader<KIND, D> loader(a.src, hk, 16, lane);
  Walk fetch = use;
  int fetched = 0;        // groups of `fetch` requested so far
  bool placed = true;     // int8: the scales requested last are in shared memory
  auto open = [&]() {     // begins the next sequence that has groups in the range
    for (;;) {
      if (fetch.g1 > fetch.g0) {
        loader.begin(fetch.b, fetch.v.base + 16 * fetch.g0, fetch.g1 - fetch.g0, fetch.v.lo, fetch.v.hi);
        fetched = 0;
        return true;
      }
      if (!MERGE) return false;
      fetch.leave();
      if (fetch.b >= a.B || fetch.at >= end) return false;
      fetch.enter(a, begin, end);
    }
  };
  bool more = open();
  auto request = [&](int st) {
    if (more) {
      loader.request(fetched, ring_u + st * S::kStage, ring_u + st * S::kStage + 16 * RB, flag_of(st));
      placed = false;
      if (++fetched == loader.count) {
        fetch.g1 = fetch.g0;  // done with it
        more = open();
      }
    }
    cp_async_commit();
  };
  auto place = [&](int st) {
    if (KIND == BPT_KV_INT8 && !placed) {
      loader.place(scales_of(st));
      placed = true;
    }
  };
#pragma unroll
  for (int i = 0; i < NST - 1; ++i) {
    request(i);
    if (i < NST - 2) place(i);
  }
  // Powers are taken of s - m with m the largest score less kLift: the largest P is 2^15, so that of f16 products a P of 2^-29
  // of it still has 11 bits (bf16 has the range anyway; int8 pages bring theirs into range below). Beyond 2^22, where fp32 would
  // round that difference, m is the score itself; m never falls, so no P passes 2^15 either way.
  constexpr float kLift = KIND == BPT_KV_F16 || KIND == BPT_KV_FP8 ? 15.f : 0.f;
  const bool cap = a.softcap > 0.f;
  const float cap_out = a.softcap * kLog2e;
  const float slope = a.slopes && g < heads ? a.slopes[h0 + g] * kLog2e : 0.f;
  int st = 0, st_in = NST - 1;

  for (;;) {  // the range's sequences
    if (MERGE && use.v.groups == 0 && use.at >= begin && a.by_sequence && a.ranges > 1 && lane == 0)
      a.ws_meta[int64_t(use.b) * a.heads + ht] = make_int4(-1, 0, 0, 0);
    if (MERGE && use.v.groups == 0 && use.at >= begin && lane < D / 8) {  // nothing visible: zeros
      for (int r = 0; r < heads; ++r)
#pragma unroll
        for (int i = 0; i < 8; ++i) store_any(a.out, a.out_dtype, (int64_t(use.b) * a.Hq + h0 + r) * D + lane * 8 + i, 0.f);
    }
    if (!MERGE || use.g1 > use.g0) {
  uint32_t qf[D / 16][4];
  const int64_t q_at = int64_t(use.b) * a.q_sb + int64_t(h0 + g) * a.q_sh;
  const float q_unit = a.q_dtype == BPT_DTYPE_BF16  ? query_rows<KIND, D, BPT_DTYPE_BF16>(a.q, q_at, t, g < heads, qf)
                       : a.q_dtype == BPT_DTYPE_F16 ? query_rows<KIND, D, BPT_DTYPE_F16>(a.q, q_at, t, g < heads, qf)
                                                    : query_rows<KIND, D, BPT_DTYPE_F32>(a.q, q_at, t, g < heads, qf);
  const float raw = a.sm_scale * q_unit * a.src.k_scale;  // a product as a score
  const float mul = cap ? raw * 2.f * kLog2e / a.softcap : raw * kLog2e;

  float m = -INFINITY, l = 0.f;
  // int8: the row's largest product of a probability and a value scale so far, and the power of two under which o holds them
  float most = 0.f, fit = 1.f;
  float o[D / 8][4];
#pragma unroll
  for (int n = 0; n < D / 8; ++n)
#pragma unroll
    for (int i = 0; i < 4; ++i) o[n][i] = 0.f;

  const int from = use.v.lo, to = use.v.hi, pos = use.v.pos;
  for (int i = use.g0; i < use.g1; ++i) {
    cp_async_wait<NST - 2>();
    place(st_in == 0 ? NST - 1 : st_in - 1);
    __syncwarp();  // every lane's copies of this group have landed; everyone is done with the stage refilled next
    request(st_in);
    const int key0 = use.v.base + 16 * i;
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
    if (kLift > 0.f && fabsf(top) < 4194304.f) top -= kLift;
    if (__any_sync(0xffffffffu, top > m)) {
      const float to_m = fmaxf(m, top);
      const float shrink = to_m == -INFINITY ? 1.f : exp2_approx(m - to_m);
      m = to_m;
      l *= shrink;
      if constexpr (KIND == BPT_KV_INT8) most *= shrink;
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
    if constexpr (KIND == BPT_KV_INT8) {
      // The products enter the matrix operands between 2^9 and 2^15 at a row's largest, where f16 and its rest keep 22 bits
      // of it, and 11 of one 2^-23 as large.
      float top_p = fmaxf(fmaxf(s[0], s[1]), fmaxf(s[2], s[3]));
      top_p = fmaxf(top_p, __shfl_xor_sync(0xffffffffu, top_p, 1));
      top_p = fmaxf(top_p, __shfl_xor_sync(0xffffffffu, top_p, 2));
      most = fmaxf(most, top_p);
      const float at = most * fit;
      if (__any_sync(0xffffffffu, at > 32768.f || (at < 512.f && most > 0.f))) {
        const float to_fit = most > 0.f ? value_range(most) : fit, change = to_fit * inverse_power(fit);
        fit = to_fit;
#pragma unroll
        for (int n = 0; n < D / 8; ++n)
#pragma unroll
          for (int e = 0; e < 4; ++e) o[n][e] *= change;
      }
#pragma unroll
      for (int e = 0; e < 4; ++e) s[e] *= fit;
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
  l += __shfl_xor_sync(0xffffffffu, l, 1);
  l += __shfl_xor_sync(0xffffffffu, l, 2);
  const float inv = l == 0.f ? 0.f : KIND == BPT_KV_INT8 ? inverse_power(fit) / l : a.src.v_scale / l;
  const float lse = l == 0.f ? -INFINITY : (m == -INFINITY ? 0.f : m) + log2f(l);
  // where the rows go: straight to out, or to a part
  const int64_t row = int64_t(use.b) * a.Hq + h0 + g;
  float* dst = nullptr;
  if constexpr (MERGE) {
    const bool starts = use.g0 == 0, ends = use.g1 == use.v.groups;
    if (!(starts && ends)) {
      const int64_t part = id * 2 + (starts ? 1 : 0);
      dst = a.ws_out + (part * 8 + g) * D;
      if (t == 0) a.ws_lse[part * 8 + g] = lse;
    }
    if (starts && lane == 0 && a.ranges > 1 && (a.by_sequence || !ends))
      a.ws_meta[a.by_sequence ? int64_t(use.b) * a.heads + ht : id] =
          make_int4(ends ? -1 : use.b, range, int((use.at + kStartCost + use.v.groups - 1) / share), 0);
  } else if (g < heads) {
    dst = a.part_out + (row * a.n_splits + sp) * D;
    if (t == 0) a.part_lse[row * a.n_splits + sp] = lse / kLog2e;
  }
  if (g < heads) {
#pragma unroll
    for (int n = 0; n < D / 8; ++n) {
      const float x = (o[n][0] + o[n][2]) * inv, y = (o[n][1] + o[n][3]) * inv;
      const int dx = v_dim<KIND, D>(n, t, 0), dy = v_dim<KIND, D>(n, t, 1);
      if (dst) {
        if constexpr (kIs16<KIND>) {
          *reinterpret_cast<float2*>(dst + dx) = make_float2(x, y);
        } else {
          dst[dx] = x;
          dst[dy] = y;
        }
      } else {
        store_any(a.out, a.out_dtype, row * D + dx, x);
        store_any(a.out, a.out_dtype, row * D + dy, y);
      }
    }
  }
    }
    if (!MERGE) break;
    use.leave();
    if (use.b >= a.B || use.at >= end) break;
    use.enter(a, begin, end);
  }
  cp_async_wait<0>();
}

// Joins the parts of a place's sequence for one of its heads. Eight warps: as many per row as fit.
template <int D>
__global__ void __launch_bounds__(256) paged_join_kernel(const ReadArgs a) {
  __shared__ float s_sum[8], s_top[8];
  __shared__ float s_acc[8][D];
  pdl_launch_dependents();
  pdl_wait();
  const int64_t id = blockIdx.x;
  const int4 meta = a.ws_meta[id];
  if (meta.x < 0) return;
  const int range = meta.y, ht = int(id % a.heads), hk = ht / a.tiles, tile = ht - hk * a.tiles;
  const int h0 = hk * a.rep + tile * 8, heads = min(8, a.rep - tile * 8), rows = gridDim.y == 1 ? heads : 1;
  if (int(blockIdx.y) >= heads) return;
  const int per_row = rows == 1 ? 8 : rows == 2 ? 4 : rows <= 4 ? 2 : 1;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, r = warp / per_row, first = warp % per_row;
  const int row = rows == 1 ? int(blockIdx.y) : r;
  const int parts = meta.z - range + 1;
  constexpr int V = D / 32;
  float top = -INFINITY, sum = 0.f, acc[V];
#pragma unroll
  for (int e = 0; e < V; ++e) acc[e] = 0.f;
  auto part_at = [&](int i) { return ((int64_t(range + i) * a.heads + ht) * 2 + (i == 0 ? 1 : 0)) * 8 + row; };
  if (r < rows) {
    for (int i = first + per_row * lane; i < parts; i += per_row * 32) top = fmaxf(top, a.ws_lse[part_at(i)]);
    top = warp_max(top);
    const float off = top == -INFINITY ? 0.f : top;
#pragma unroll 8
    for (int i = first; i < parts; i += per_row) {
      const int64_t at = part_at(i);
      const float f = exp2_approx(a.ws_lse[at] - off);
      sum += f;
#pragma unroll
      for (int e = 0; e < V; ++e) acc[e] = fmaf(f, a.ws_out[at * D + lane + 32 * e], acc[e]);
    }
  }
  if (lane == 0) {
    s_top[warp] = top;
    s_sum[warp] = sum;
  }
#pragma unroll
  for (int e = 0; e < V; ++e) s_acc[warp][lane + 32 * e] = acc[e];
  __syncthreads();
  if (r >= rows || first != 0) return;
  float all = top;
  for (int w = 1; w < per_row; ++w) all = fmaxf(all, s_top[warp + w]);
  const float off = all == -INFINITY ? 0.f : all;
  float total = 0.f;
#pragma unroll
  for (int e = 0; e < V; ++e) acc[e] = 0.f;
  for (int w = 0; w < per_row; ++w) {
    const float f = exp2_approx(s_top[warp + w] - off);
    total = fmaf(f, s_sum[warp + w], total);
#pragma unroll
    for (int e = 0; e < V; ++e) acc[e] = fmaf(f, s_acc[warp + w][lane + 32 * e], acc[e]);
  }
  const float inv = total == 0.f ? 0.f : 1.f / total;
#pragma unroll
  for (int e = 0; e < V; ++e)
    store_any(a.out, a.out_dtype, (int64_t(meta.x) * a.Hq + h0 + row) * D + lane + 32 * e, acc[e] * inv);
}

int launch(const void* kernel, dim3 grid, int threads, int smem, bool dependent, const ReadArgs& a, cudaStream_t stream) {
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = grid;
  cfg.blockDim = dim3(unsigned(threads));
  cfg.dynamicSmemBytes = size_t(smem);
  cfg.stream = stream;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = attr;
  cfg.numAttrs = dependent ? 1 : 0;
  ReadArgs copy = a;
  void* args[] = {&copy};
  const cudaError_t err = cudaLaunchKernelExC(&cfg, kernel, args);
  if (err != cudaSuccess) return set_error(BPT_ERR_CUDA, "paged read launch: %s", cudaGetErrorString(err));
  return BPT_OK;
}

// The most ranges of a merged read: as many as give every warp of a full GPU one head of one range (two CTAs per SM, one at
// 16-bit heads of 256; three CTAs of 8-bit heads of 128 took 37 us where two took 35).
int64_t read_ranges(int64_t heads, int64_t D, int kind) {
  const bool wide = D == 256 && (kind == BPT_KV_F16 || kind == BPT_KV_BF16);
  return std::max<int64_t>(int64_t(num_sms()) * (wide ? 1 : 2) * kWarps / heads, 1);
}

template <int KIND, int D, bool MERGE>
int launch_read(const ReadArgs& a, int flags, cudaStream_t stream) {
  using S = ReadShape<KIND, D>;
  const void* kernel = reinterpret_cast<const void*>(paged_read_kernel<KIND, D, MERGE>);
  static std::atomic<uint64_t> ready{0};
  int st = set_max_smem_once(kernel, S::kSmem, ready);
  if (st) return st;
  const int64_t warps = (MERGE ? int64_t(a.ranges) : int64_t(a.B) * a.n_splits) * a.heads;
  // few warps are spread over the SMs
  const int per_cta = int(std::min<int64_t>(kWarps, (warps + num_sms() - 1) / num_sms()));
  const int64_t ctas = (warps + per_cta - 1) / per_cta;
  BPT_REQUIRE(ctas < (1ll << 31), BPT_ERR_INVALID, "paged read: too many parts");
  st = launch(kernel, dim3(unsigned(ctas)), 32 * per_cta, per_cta * S::kPerWarp, (flags & BPT_FLAG_PDL) != 0, a, stream);
  if (st || !MERGE || a.ranges == 1) return st;
  // many ranges per sequence: a CTA per row, so that no warp reads a long row of parts
  const unsigned rows = a.ranges >= 16 * int64_t(a.B) ? unsigned(std::min(a.rep, 8)) : 1u;
  const int64_t places = (a.by_sequence ? a.B : a.ranges) * int64_t(a.heads);
  return launch(reinterpret_cast<const void*>(paged_join_kernel<D>), dim3(unsigned(places), rows), 256, 0, true, a, stream);
}

template <int KIND>
int read_dim(const ReadArgs& a, int64_t D, bool merge, int flags, cudaStream_t stream) {
  if (merge) {
    if (D == 64) return launch_read<KIND, 64, true>(a, flags, stream);
    if (D == 128) return launch_read<KIND, 128, true>(a, flags, stream);
    return launch_read<KIND, 256, true>(a, flags, stream);
  }
  if (D == 64) return launch_read<KIND, 64, false>(a, flags, stream);
  if (D == 128) return launch_read<KIND, 128, false>(a, flags, stream);
  return launch_read<KIND, 256, false>(a, flags, stream);
}

struct ReadWorkspace {
  int64_t meta, lse, out, total;  // offsets of the three parts, behind the tickets of other reads; the size
};
ReadWorkspace read_workspace(int64_t Hq, int64_t Hkv, int64_t D, int kind) {
  const int64_t heads = Hkv * ((Hq / Hkv + 7) / 8), warps = read_ranges(heads, D, kind) * heads;
  ReadWorkspace w;
  w.meta = kTicketBytes;
  w.lse = w.meta + (warps * 16 + 255) / 256 * 256;
  w.out = w.lse + (warps * 2 * 8 * 4 + 255) / 256 * 256;
  w.total = w.out + warps * 2 * 8 * D * 4;
  return w;
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

extern "C" int64_t bpt_paged_read_workspace_bytes(int64_t Hq, int64_t Hkv, int64_t D, int kind) {
  return Hkv >= 1 && Hq >= Hkv && D >= 1 ? read_workspace(Hq, Hkv, D, kind).total : 0;
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
  const int64_t tokens = args->tokens;
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
  BPT_REQUIRE(B >= 0 && B < (1 << 24), BPT_ERR_INVALID, "%s: B=%lld", who, (long long)B);
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
  BPT_REQUIRE(window >= 0, BPT_ERR_INVALID, "%s: window=%lld", who, (long long)window);
  BPT_REQUIRE(q_stride_b % 2 == 0 && q_stride_h % 2 == 0 && reinterpret_cast<uintptr_t>(q) % (q_dtype == BPT_DTYPE_F32 ? 8 : 4) == 0,
              BPT_ERR_ALIGNMENT, "%s: q's rows must start on pairs of elements", who);
  BPT_REQUIRE(softcap >= 0.f && softcap < INFINITY, BPT_ERR_INVALID, "%s: softcap must be finite and not negative", who);
  const bool merge = out_partial == nullptr;
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
  BPT_REQUIRE(Hkv * a.tiles < 65536, BPT_ERR_INVALID, "%s: too many heads", who);
  a.heads = int(Hkv * a.tiles);
  a.out = out;
  a.out_dtype = out_dtype;
  a.part_out = out_partial;
  a.part_lse = lse_partial;
  a.split = a.n_splits = a.ranges = 1;
  a.ws_out = a.ws_lse = nullptr;
  a.ws_meta = nullptr;
  a.by_sequence = 0;
  if (merge) {
    BPT_REQUIRE(out, BPT_ERR_INVALID, "%s: null output", who);
    BPT_REQUIRE(out_dtype == BPT_DTYPE_F32 || out_dtype == BPT_DTYPE_F16 || out_dtype == BPT_DTYPE_BF16, BPT_ERR_INVALID,
                "%s: out dtype %d", who, out_dtype);
    BPT_REQUIRE(tokens >= 1, BPT_ERR_INVALID, "%s: tokens=%lld", who, (long long)tokens);
    const int64_t keys = a.window > 0 ? std::min<int64_t>(tokens, int64_t(a.window) + 15) : tokens;
    const int64_t cost = (std::min<int64_t>(keys, 1 << 30) + 15) / 16 + kStartCost;
    a.ranges = int(std::min(read_ranges(a.heads, D, kind), std::max<int64_t>(B * cost / (kStartCost + kLeastShare), 1)));
    a.by_sequence = B <= a.ranges;
    if (a.ranges > 1) {
      const ReadWorkspace w = read_workspace(Hq, Hkv, D, kind);
      BPT_REQUIRE(workspace, BPT_ERR_WORKSPACE, "%s: no workspace", who);
      BPT_REQUIRE(aligned16(workspace), BPT_ERR_ALIGNMENT, "%s: workspace must be 16-byte aligned", who);
      BPT_REQUIRE(workspace_bytes >= w.total, BPT_ERR_WORKSPACE, "%s: workspace of %lld bytes, need %lld", who,
                  (long long)workspace_bytes, (long long)w.total);
      uint8_t* ws = static_cast<uint8_t*>(workspace);
      a.ws_meta = reinterpret_cast<int4*>(ws + w.meta);
      a.ws_lse = reinterpret_cast<float*>(ws + w.lse);
      a.ws_out = reinterpret_cast<float*>(ws + w.out);
    }
  } else {
    BPT_REQUIRE(lse_partial, BPT_ERR_INVALID, "%s: null output", who);
    BPT_REQUIRE(split >= 16 && split % 16 == 0 && split < (1ll << 30) && n_splits >= 1 && n_splits < (1 << 20),
                BPT_ERR_INVALID, "%s: split=%lld (a multiple of 16), n_splits=%lld", who, (long long)split, (long long)n_splits);
    a.split = int(split);
    a.n_splits = int(n_splits);
  }
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  switch (kind) {
    case BPT_KV_FP8: return read_dim<BPT_KV_FP8>(a, D, merge, flags, s);
    case BPT_KV_INT8: return read_dim<BPT_KV_INT8>(a, D, merge, flags, s);
    case BPT_KV_F16: return read_dim<BPT_KV_F16>(a, D, merge, flags, s);
    default: return read_dim<BPT_KV_BF16>(a, D, merge, flags, s);
  }
}
