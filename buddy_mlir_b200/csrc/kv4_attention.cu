// Attention over the 4-bit KV cache (b200_kv4_attention).
//
// Codes go to the tensor cores as they are: with k = lo + s c per group of 64 dims, a score is  q.k = sum over groups of s (q.c) + lo sum(q),  and
// an output  sum p v = sum (p s) c + sum p lo,  so that scales meet scores and weights (a handful per key) instead of 64 codes each.  A code is one
// f16 exactly; the other operand is one f16 (f32: two, 22 bits of it) after a power of two of its row that puts the row's largest near f16's.
// Codes are the operand with M rows (mma.m16n8k16: sixteen positions, or sixteen dims), the query rows that share a kv head the eight
// columns; words of eight codes lie in the cache as the operand's registers want them, and one AND makes a pair of codes a pair of
// f16: nibbles 0 and 1 of a half-word are the subnormal numbers c 2^-24 and c 2^-20, which the tensor cores multiply exactly.
//
// The reference r of a row's weights is not its largest score but the largest of score + log2 of the key's larger V scale, so that the weights
// that meet codes, p s, are at most 2^12 and near 2^8 where they count, whatever the scales are; sums and totals carry the same factor.  (By their
// magnitude: a group whose minimum was rounded to above its maximum has a negative one.)  f16 ends at 2^-24, 2^-32 of that: where the other group's weights are
// far smaller (kNear), those of f32 and their sums carry a power of two of their own, set when the reference moves and lowered when a weight outgrows it (a group at
// 2^-20 of the other would keep 13 bits).  The 16-bit types, whose one term keeps its 11 bits down to 2^-22 of the other group, go without: that took them 5 to 14 % longer.
//
// Sixteen warps of a CTA share an item's tiles, each with four tiles on their way (cp.async), and join in shared memory.  64 rows of 2000 to 4096 keys, 32
// heads on 8 of 128 dims, bf16: 62 us, 3.7 TB/s, 0.56 of a copy's rate (f32, one tile at a time and twice the products: 93 us).  A tile is some 290 instructions of a warp, 114 clocks of an SM; issue slots are
// half full and the tensor pipe a quarter, so chains of latencies bound it at four warps a scheduler (128 registers a thread: q, sums and two tiles).
#include "kv4_plan.cuh"

#include <algorithm>

namespace b200 {

namespace {

constexpr int kWarps = 16, kThreads = 32 * kWarps;
constexpr int kRows = 8;            // query rows of an item: a position's heads (several positions', if they are few)
constexpr int kSlots = 4;           // tiles that a warp has in flight or in hand
constexpr int kChunkRows = 64;     // query vectors of a sequence and kv head from which on tcgen05 has them
constexpr int kLeastKeys = 512, kSplit = 1000;     // of a CTA, where there are not more CTAs than that asks for
// Of a lane's sum of weights: a key that has more of it is one of few.  (f16, steps of 200 sequences of up to 600 keys, twelve seeds: errors 2.0 to 2.3e-4, where the
// result's own rounding is 2.0 to 2.1e-4; with 0.9 2.2 to 2.65e-4 and 2 % shorter; all weights rounded: 3.0e-4.)
constexpr float kFew = 0.25f;
constexpr float kNear = 6.f, kApart = 64.f;   // log2 of how much smaller a group's largest weight may be than the other's before it is raised; that ratio
constexpr int kMostLift = 40;
constexpr float kLeastScale = 5.9604645e-8f;   // (f16's smallest: a group of equal values that f16 holds has the scale 0)

__host__ __device__ constexpr int part_floats(int D) { return kRows * (D + 4) + 2 * kRows; }   // sums in rows of D + 4, maxima, totals

__device__ __forceinline__ float lg2(float x) {
  float y;
  asm("lg2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}
__device__ __forceinline__ uint32_t transpose8(uint32_t x) {
  uint32_t y;
  asm("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(y) : "r"(x));
  return y;
}
__device__ __forceinline__ void mma(float (&c)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
  asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
      : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
      : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
__device__ __forceinline__ void copy16(void *to, const void *from) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"((uint32_t)__cvta_generic_to_shared(to)), "l"(from) : "memory");
}
__device__ __forceinline__ void copies_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int LEFT> __device__ __forceinline__ void copies_wait() { asm volatile("cp.async.wait_group %0;" ::"n"(LEFT) : "memory"); }

// Codes of the low nibble of each byte-pair of w (bits 0 .. 3 and 16 .. 19) and of the high one, as pairs of f16: c 2^-24 and c 2^-20.
__device__ __forceinline__ uint32_t low_codes(uint32_t w) { return w & 0x000f000fu; }
__device__ __forceinline__ uint32_t high_codes(uint32_t w) { return w & 0x00f000f0u; }
// f32 needs normal operands (the tensor cores line products up by their exponents, and a subnormal number's says little): c - 8 by way of 1024 + c and
// 1024 + 16 c, one operation more.
__device__ __forceinline__ uint32_t low_exact(uint32_t w) {
  uint32_t x = (w & 0x000f000fu) | 0x64006400u;
  asm("add.rn.f16x2 %0, %0, %1;" : "+r"(x) : "r"(0xe408e408u));                            // - 1032
  return x;
}
__device__ __forceinline__ uint32_t high_exact(uint32_t w) {
  uint32_t x = (w & 0x00f000f0u) | 0x64006400u;
  asm("add.rn.f16x2 %0, %0, %1;" : "+r"(x) : "r"(0xe480e480u));                            // - 1152: 16 (c - 8)
  return x;
}
// -8 in both: what centres V's codes.  A sum of n weighted codes then stays as small as the values' own spread, which matters because the tensor
// cores' sums round towards zero.
constexpr uint32_t kMinus8Low = 0x80088008u, kMinus8High = 0x80808080u;
constexpr float kCentre = 8.f;

// x and y as TERMS f16 each
template <int TERMS> __device__ __forceinline__ void split(float x, float y, uint32_t (&t)[TERMS]) {
#pragma unroll
  for (int i = 0; i < TERMS; ++i) {
    t[i] = pack_f16(x, y);
    if (i + 1 < TERMS) {
      const float2 f = halves(t[i]);
      x -= f.x;
      y -= f.y;
    }
  }
}

template <int D, int TYPE> struct Tile {   // of a warp: one item's sums
  static constexpr int GROUPS = D / kKv4Group, STEPS = D / 16, BYTES = kv4_tile_bytes(D);
  static constexpr bool EXACT = TYPE == B200_F32;
  static constexpr int TERMS = EXACT ? 2 : 1;
  static constexpr int KT = EXACT ? 1 : 2;  // tiles at a time
  static constexpr bool LIFTS = EXACT && GROUPS == 2;
  static constexpr float LOW = EXACT ? 1.f : 5.9604645e-8f, HIGH = EXACT ? 16.f : 9.5367432e-7f;   // units of the codes' operands
  uint32_t q[TERMS][STEPS][2];
  float qs[GROUPS][2];                      // sums of q over a group, times the scores' scale, of rows 2 t and 2 t + 1 (t: lane % 4)
  float unit[2];                            // the scores' scale over the row's power of two and the codes' unit
  float o[STEPS][4];                        // dims 16 i + g (+ 8), rows 2 t (+ 1) (g: lane / 4)
  float bias[GROUPS][2], r[2], l[2];        // sums over this lane's keys: p (lo + 8 s), p
  uint32_t lift;                            // LIFTS: byte 2 group + row: log2 of what that group's weights and o are raised by
  bool raised;                              // any of the warp's is

  __device__ __forceinline__ int lift_of(int gr, int e) const { return lift >> 8 * (2 * gr + e) & 255; }
  __device__ __forceinline__ void times(int gr, int e, float f) {
#pragma unroll
    for (int i = 4 * gr; i < 4 * gr + 4; ++i) {
      o[i][e] *= f;
      o[i][2 + e] *= f;
    }
  }
  // The powers of two of both groups' weights, from the largest score + log2 of scale of these keys: set where the keys are among those that count most for the
  // row, otherwise only lowered as far as f16 asks for.
  __device__ __forceinline__ void settle(const uint8_t *tiles, const float (&s)[KT][4]) {
    const int lane = threadIdx.x & 31, g = lane >> 2;
#pragma unroll
    for (int e = 0; e < 2; ++e) {
      float most[2] = {-INFINITY, -INFINITY};
#pragma unroll
      for (int n = 0; n < KT; ++n)
#pragma unroll
        for (int h = 0; h < 2; ++h) {
          const uint2 pairs = *reinterpret_cast<const uint2 *>(tiles + n * BYTES + kv4_v_pairs(D) + (g + 8 * h) * 8);
          most[0] = fmaxf(most[0], s[n][2 * h + e] + lg2(fabsf(halves(pairs.x).x)));
          most[1] = fmaxf(most[1], s[n][2 * h + e] + lg2(fabsf(halves(pairs.y).x)));
        }
#pragma unroll
      for (int x = 4; x < 32; x <<= 1) {
        most[0] = fmaxf(most[0], __shfl_xor_sync(0xffffffffu, most[0], x));
        most[1] = fmaxf(most[1], __shfl_xor_sync(0xffffffffu, most[1], x));
      }
      const bool counts = fmaxf(most[0], most[1]) > r[e] + kKv4Top - kNear;
#pragma unroll
      for (int gr = 0; gr < 2; ++gr) {
        const int have = lift_of(gr, e);
        const float less = r[e] + kKv4Top - most[gr];   // (a group of scales 0 asks for nothing)
        const int to = !(less < 1000.f) ? have : counts ? (less > kNear ? min((int)less, kMostLift) : 0) : min(have, max((int)(less + kNear), 0));
        lift += (uint32_t)(to - have) << 8 * (2 * gr + e);
        times(gr, e, power(to - have));
      }
    }
  }
  __device__ __forceinline__ void clear() {
    lift = 0;
    raised = false;
#pragma unroll
    for (int i = 0; i < STEPS; ++i)
#pragma unroll
      for (int e = 0; e < 4; ++e)
        o[i][e] = 0.f;
#pragma unroll
    for (int e = 0; e < 2; ++e) {
      r[e] = kKv4Seed;
      l[e] = 0.f;
#pragma unroll
      for (int gr = 0; gr < GROUPS; ++gr)
        bias[gr][e] = 0.f;
    }
  }

  // q of this lane's row (lane / 4), or none
  __device__ __forceinline__ void load_q(const Kv4Params &p, bool live, int64_t at) {
    const int lane = threadIdx.x & 31, t = lane & 3;
    float x[STEPS][4], most = 0.f;
#pragma unroll
    for (int k = 0; k < STEPS; ++k) {
      const int d = 32 * (k / 2) + 8 * t + 4 * (k & 1);
#pragma unroll
      for (int e = 0; e < 4; ++e)
        x[k][e] = live && !p.wide_q ? load_as_float(p.a.q, TYPE, at + d + e) : 0.f;
      if (live && p.wide_q)
        load_wide<TYPE>(p.a.q, at + d, x[k]);
#pragma unroll
      for (int e = 0; e < 4; ++e)
        most = fmaxf(most, fabsf(x[k][e]));
    }
    most = fmaxf(most, __shfl_xor_sync(0xffffffffu, most, 1));
    most = fmaxf(most, __shfl_xor_sync(0xffffffffu, most, 2));
    // 2^up: the row's largest comes to 2^14 .. 2^15 (a row below 2^-86 not as far)
    const int up = min(max(14 + 127 - (int)(__float_as_uint(most) >> 23), -113), 100);
    const float factor = __uint_as_float((uint32_t)(127 + up) << 23), over = p.log2_scale * __uint_as_float((uint32_t)(127 - up) << 23) * (1.f / LOW);
#pragma unroll
    for (int e = 0; e < 2; ++e)
      unit[e] = __shfl_sync(0xffffffffu, over, 8 * t + 4 * e);
#pragma unroll
    for (int gr = 0; gr < GROUPS; ++gr) {
      float sum = 0.f;
#pragma unroll
      for (int k = 4 * gr; k < 4 * gr + 4; ++k) {
        float y[4];
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          sum += x[k][e];
          y[e] = x[k][e] * (e / 2 == 0 ? factor : factor * (LOW / HIGH));
        }
        uint32_t lo[TERMS], hi[TERMS];
        split<TERMS>(y[0], y[1], lo);
        split<TERMS>(y[2], y[3], hi);
#pragma unroll
        for (int i = 0; i < TERMS; ++i) {
          q[i][k][0] = lo[i];
          q[i][k][1] = hi[i];
        }
      }
      sum += __shfl_xor_sync(0xffffffffu, sum, 1);
      sum += __shfl_xor_sync(0xffffffffu, sum, 2);
      sum = sum - sum == 0.f ? sum * p.log2_scale : NAN;   // (a row with an infinity has no scores)
#pragma unroll
      for (int e = 0; e < 2; ++e)
        qs[gr][e] = __shfl_sync(0xffffffffu, sum, 8 * t + 4 * e);
    }
  }

  // KT tiles of sixteen keys, from j0[i] on; limit: keys that rows 2 t and 2 t + 1 see (only where MASKED)
  template <bool MASKED> __device__ __forceinline__ void keys(const uint8_t *tiles, const int (&j0)[KT], const int (&limit)[2]) {
    const int lane = threadIdx.x & 31, g = lane >> 2, t = lane & 3;
    float s[KT][4], top[2] = {-INFINITY, -INFINITY};
    bool out[KT][4];   // not seen
#pragma unroll
    for (int n = 0; n < KT; ++n) {
      const uint8_t *tile = tiles + n * BYTES;
      uint32_t kw[2][D / 32], kp[2][GROUPS], vp[2][GROUPS];   // of keys g and g + 8
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        const int j = g + 8 * h;
        if constexpr (D == 128) {
          *reinterpret_cast<uint4 *>(kw[h]) = *reinterpret_cast<const uint4 *>(tile + j * 64 + t * 16);
          *reinterpret_cast<uint2 *>(kp[h]) = *reinterpret_cast<const uint2 *>(tile + kv4_k_pairs(D) + j * 8);
          *reinterpret_cast<uint2 *>(vp[h]) = *reinterpret_cast<const uint2 *>(tile + kv4_v_pairs(D) + j * 8);
        } else {
          *reinterpret_cast<uint2 *>(kw[h]) = *reinterpret_cast<const uint2 *>(tile + j * 32 + t * 8);
          kp[h][0] = *reinterpret_cast<const uint32_t *>(tile + kv4_k_pairs(D) + j * 4);
          vp[h][0] = *reinterpret_cast<const uint32_t *>(tile + kv4_v_pairs(D) + j * 4);
        }
      }
      float dot[4] = {}, low[4] = {};
#pragma unroll
      for (int gr = 0; gr < GROUPS; ++gr) {
        float c[4] = {};
#pragma unroll
        for (int i = 2 * gr; i < 2 * gr + 2; ++i)
#pragma unroll
          for (int u = 0; u < 2; ++u) {
            const uint32_t x = kw[0][i] >> (8 * u), y = kw[1][i] >> (8 * u);
            const uint32_t a[4] = {EXACT ? low_exact(x) : low_codes(x), EXACT ? low_exact(y) : low_codes(y), EXACT ? high_exact(x) : high_codes(x),
                                   EXACT ? high_exact(y) : high_codes(y)};
#pragma unroll
            for (int e = TERMS - 1; e >= 0; --e)
              mma(c, a, q[e][2 * i + u][0], q[e][2 * i + u][1]);
          }
#pragma unroll
        for (int h = 0; h < 2; ++h) {
          const float2 pair = halves(kp[h][gr]);
          const float lo = EXACT ? fmaf(kCentre, pair.x, pair.y) : pair.y;
#pragma unroll
          for (int e = 0; e < 2; ++e) {
            dot[2 * h + e] = fmaf(c[2 * h + e], pair.x, dot[2 * h + e]);
            low[2 * h + e] = fmaf(lo, qs[gr][e], low[2 * h + e]);
          }
        }
      }
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        float largest = kLeastScale;
#pragma unroll
        for (int gr = 0; gr < GROUPS; ++gr)
          largest = fmaxf(largest, fabsf(halves(vp[h][gr]).x));
        const float height = lg2(largest);
#pragma unroll
        for (int e = 0; e < 2; ++e) {
          const int k = 2 * h + e;
          s[n][k] = fmaf(dot[k], unit[e], low[k]);
          float at = s[n][k] + height;
          if constexpr (MASKED) {
            out[n][k] = j0[n] + g + 8 * h >= limit[e];
            s[n][k] = out[n][k] ? -INFINITY : s[n][k];
            at = out[n][k] ? -INFINITY : at;
          }
          top[e] = fmaxf(top[e], at);
        }
      }
    }
    if (__any_sync(0xffffffffu, kv4_moves(top[0], r[0]) || kv4_moves(top[1], r[1]))) {
#pragma unroll
      for (int e = 0; e < 2; ++e) {
#pragma unroll
        for (int x = 4; x < 32; x <<= 1)
          top[e] = fmaxf(top[e], __shfl_xor_sync(0xffffffffu, top[e], x));
        top[e] = kv4_moves(top[e], r[e]) ? kv4_reference(top[e]) : r[e];   // (each row for itself)
        const float keep = ex2(r[e] - top[e]);
        r[e] = top[e];
        l[e] *= keep;
#pragma unroll
        for (int gr = 0; gr < GROUPS; ++gr) {
          bias[gr][e] *= keep;
          times(gr, e, keep);
        }
      }
      if constexpr (LIFTS) {
        bool apart = false;   // keys that are seen, and whose groups are
#pragma unroll
        for (int n = 0; n < KT; ++n)
#pragma unroll
          for (int h = 0; h < 2; ++h) {
            const uint2 pairs = *reinterpret_cast<const uint2 *>(tiles + n * BYTES + kv4_v_pairs(D) + (g + 8 * h) * 8);
            const float a = fabsf(halves(pairs.x).x), b = fabsf(halves(pairs.y).x), least = fminf(a, b);
            apart = apart || (least > 0.f && least * kApart < fmaxf(a, b) && fmaxf(s[n][2 * h], s[n][2 * h + 1]) > -INFINITY);
          }
        raised = raised || __any_sync(0xffffffffu, apart);
      }
    }
    if constexpr (LIFTS)
      if (raised) {
        settle(tiles, s);
        raised = __any_sync(0xffffffffu, lift != 0);
      }
#pragma unroll
    for (int n = 0; n < KT; ++n) {
      const uint8_t *tile = tiles + n * BYTES;
      uint32_t vp[2][GROUPS];
#pragma unroll
      for (int h = 0; h < 2; ++h)
        if constexpr (D == 128)
          *reinterpret_cast<uint2 *>(vp[h]) = *reinterpret_cast<const uint2 *>(tile + kv4_v_pairs(D) + (g + 8 * h) * 8);
        else
          vp[h][0] = *reinterpret_cast<const uint32_t *>(tile + kv4_v_pairs(D) + (g + 8 * h) * 4);
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        s[n][e] = ex2(s[n][e] - r[e & 1]);
        l[e & 1] += s[n][e];
      }
      // Weights are rounded to f16, as the result is; of many keys that averages out.  Where a key is most of a lane's, what the rounding left counts too.
      // (bf16 results are rounded eight times as far, f32 weights have two terms.)
      bool few = false;
      if constexpr (TYPE == B200_F16)
        few = __any_sync(0xffffffffu, fmaxf(s[n][0], s[n][2]) > kFew * l[0] || fmaxf(s[n][1], s[n][3]) > kFew * l[1]);
#pragma unroll
      for (int gr = 0; gr < GROUPS; ++gr) {
        float w[4];
#pragma unroll
        for (int h = 0; h < 2; ++h) {
          const float2 pair = halves(vp[h][gr]);
          const float centre = fmaf(kCentre, pair.x, pair.y);
#pragma unroll
          for (int e = 0; e < 2; ++e) {
            const int k = 2 * h + e;
            w[k] = s[n][k] * pair.x;
            float b = fmaf(s[n][k], centre, bias[gr][e]);
            if constexpr (MASKED) {   // (what is not seen may be NaN)
              w[k] = out[n][k] ? 0.f : w[k];
              b = out[n][k] ? bias[gr][e] : b;
            }
            bias[gr][e] = b;
          }
        }
        if (LIFTS && raised)
#pragma unroll
          for (int k = 0; k < 4; ++k)
            w[k] *= power(lift_of(gr, k & 1));
        uint32_t b0[TERMS], b1[TERMS];
        split<TERMS>(w[0], w[1], b0);
        split<TERMS>(w[2], w[3], b1);
#pragma unroll
        for (int e = 0; e < TERMS; ++e) {
          b0[e] = transpose8(b0[e]);
          b1[e] = transpose8(b1[e]);
        }
        uint32_t vw[4];
        *reinterpret_cast<uint4 *>(vw) = *reinterpret_cast<const uint4 *>(tile + kv4_v_codes(D) + gr * 512 + lane * 16);
        if constexpr (TYPE == B200_F16)
          if (few) {
            const uint32_t kept[2] = {pack_f16(w[0], w[1]), pack_f16(w[2], w[3])};
            const float2 x = halves(kept[0]), y = halves(kept[1]);
            const float left[4] = {w[0] - x.x, w[1] - x.y, w[2] - y.x, w[3] - y.y};
            const uint32_t b2 = transpose8(pack_f16(left[0], left[1])), b3 = transpose8(pack_f16(left[2], left[3]));
#pragma unroll
            for (int e = 0; e < 2; ++e)
              bias[gr][e] = fmaf(-kCentre, left[e] + left[2 + e], bias[gr][e]);
#pragma unroll
            for (int i = 0; i < 4; ++i) {
              const uint32_t a[4] = {low_codes(vw[i]), high_codes(vw[i]), low_codes(vw[i] >> 8), high_codes(vw[i] >> 8)};
              mma(o[4 * gr + i], a, b2, b3);
            }
          }
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          if constexpr (!EXACT) {
            const uint32_t minus8[4] = {kMinus8Low, kMinus8High, kMinus8Low, kMinus8High};
            const uint32_t a[4] = {low_codes(vw[i]), high_codes(vw[i]), low_codes(vw[i] >> 8), high_codes(vw[i] >> 8)};
            mma(o[4 * gr + i], minus8, b0[0], b1[0]);
            mma(o[4 * gr + i], a, b0[0], b1[0]);
          } else {   // a sum of its own, added with rounding to nearest
            const uint32_t a[4] = {low_exact(vw[i]), high_exact(vw[i]), low_exact(vw[i] >> 8), high_exact(vw[i] >> 8)};
            float c[4] = {};
#pragma unroll
            for (int e = TERMS - 1; e >= 0; --e)
              mma(c, a, b0[e], b1[e]);
#pragma unroll
            for (int e = 0; e < 4; ++e)
              o[4 * gr + i][e] += c[e];
          }
        }
      }
    }
  }

  // sums over all keys of the warp
  __device__ __forceinline__ void finish() {
#pragma unroll
    for (int e = 0; e < 2; ++e) {
#pragma unroll
      for (int x = 4; x < 32; x <<= 1) {
        l[e] += __shfl_xor_sync(0xffffffffu, l[e], x);
#pragma unroll
        for (int gr = 0; gr < GROUPS; ++gr)
          bias[gr][e] += __shfl_xor_sync(0xffffffffu, bias[gr][e], x);
      }
#pragma unroll
      for (int i = 0; i < STEPS; ++i) {
        const float lower = LIFTS ? power(-lift_of(i * 16 / kKv4Group, e)) : 1.f;
        o[i][e] = fmaf(o[i][e] * lower, 1.f / LOW, bias[i * 16 / kKv4Group][e]);
        o[i][2 + e] = fmaf(o[i][2 + e] * lower, 1.f / HIGH, bias[i * 16 / kKv4Group][e]);
      }
    }
  }

  __device__ __forceinline__ void store(float *part) const {
    const int lane = threadIdx.x & 31, g = lane >> 2, t = lane & 3;
#pragma unroll
    for (int i = 0; i < STEPS; ++i)
#pragma unroll
      for (int e = 0; e < 4; ++e)
        part[(2 * t + (e & 1)) * (D + 4) + 16 * i + g + 8 * (e >> 1)] = o[i][e];
    if (g == 0)
#pragma unroll
      for (int e = 0; e < 2; ++e) {
        part[kRows * (D + 4) + 2 * t + e] = r[e];
        part[kRows * (D + 4) + kRows + 2 * t + e] = l[e];
      }
  }
};

__device__ __forceinline__ int rows_of(const Kv4Params &p, const Sequence &q, int rt, int slot) {   // of an item
  const int tokens = min(p.tokens, q.n - rt * p.tokens);
  return p.subs == 1 ? tokens * p.heads : min(p.heads, p.G - slot % p.subs * p.heads);
}

// What a warp leaves behind: parts of its first item (that began before it) and of its last (that goes on behind it).
struct Left {
  Place a, b;
  int a_tiles, b_tiles;
  const float *a_part;
  bool has_a, a_ends, has_b;
};

template <int D, int TYPE> __global__ void __launch_bounds__(kThreads, 1) kv4_attention_kernel(const __grid_constant__ Kv4Params p) {
  using T = Tile<D, TYPE>;
  constexpr int BYTES = T::BYTES, PART = part_floats(D), RING = kSlots * BYTES, KT = T::KT, STAGES = kSlots / KT;
  static_assert(RING >= PART * 4, "a part of a warp lies in its ring");
  extern __shared__ __align__(128) uint8_t s_all[];
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, n = p.a.n_seqs, room = p.a.table_stride * p.page;
  __shared__ long long s_sum[2 * kWarps + 1];
  __shared__ Left s_left[kWarps];
  __shared__ int s_ctas[2][3];     // of a shared item that this CTA adds up: whether it does, the CTAs with its first and last part
  kernel_go();
  kernel_wait();

  if (lane == 0)
    s_left[warp].has_a = s_left[warp].has_b = false;
  if (tid < 2)
    s_ctas[tid][0] = 0;
  KeyPlan<4> plan;
  plan.build<kThreads>(p, s_all + kWarps * RING, s_sum, kLeastKeys, kSplit);
  // rows of no sequence
  if (p.fill) {
    const int lo = plan.r0[0], hi = max(lo, plan.r0[n]), none = lo + p.a.rows - hi, cols = p.a.q_heads * D;
    for (int64_t i = (int64_t)blockIdx.x * kThreads + tid; i < (int64_t)none * cols; i += (int64_t)gridDim.x * kThreads) {
      const int r = (int)(i / cols);
      put<TYPE>(p, (int64_t)(r < lo ? r : hi + r - lo) * p.a.out_ld + i % cols, 0.f);
    }
  }

  // ---- this CTA's keys, this warp's keys ----------------------------------------------------------------------------------------
  const long long total = plan.total;
  if (total == 0 || (int)blockIdx.x >= plan.ctas)
    return;
  long long x = plan.border(blockIdx.x + min(lane, 1));   // (a lane each)
  const long long cta_begin = __shfl_sync(0xffffffffu, x, 0), mine = __shfl_sync(0xffffffffu, x, 1) - cta_begin;
  const int act = (int)max(1ll, min((long long)kWarps, mine >> 4));   // the warps that work: sixteen keys each at least (then each begins a tile)
  Place at{n, 0, 0, 0}, stop;
  x = cta_begin + plan.part_of(mine, warp + min(lane, 1), act);
  if (x < total && warp < act)
    at = plan.locate(x);
  stop.s = __shfl_sync(0xffffffffu, at.s, 1);
  stop.slot = __shfl_sync(0xffffffffu, at.slot, 1);
  stop.rt = __shfl_sync(0xffffffffu, at.rt, 1);
  stop.tile = __shfl_sync(0xffffffffu, at.tile, 1);
  at.s = __shfl_sync(0xffffffffu, at.s, 0);
  at.slot = __shfl_sync(0xffffffffu, at.slot, 0);
  at.rt = __shfl_sync(0xffffffffu, at.rt, 0);
  at.tile = __shfl_sync(0xffffffffu, at.tile, 0);

  if (warp < act && mine > 0) {
    uint8_t *ring = s_all + warp * RING;
    T tile;
    while (at.s < n) {
      const Sequence q = plan.sequence(at.s);
      const int all = plan.item_tiles(q, at.rt);
      const bool here = stop.s == at.s && stop.slot == at.slot && stop.rt == at.rt;
      const int t0 = at.tile, t1 = here ? min(stop.tile, all) : all;
      if (here && t0 >= t1)
        break;
      if (t0 >= all) {   // (a border behind an item's last tile)
        plan.next_item(at, q);
        continue;
      }
      // ---- this warp's tiles of the item ----------------------------------------------------------------------------------------
      const int live = rows_of(p, q, at.rt, at.slot), first_token = at.rt * p.tokens, tokens = min(p.tokens, q.n - first_token);
      const int least = clamp((long long)q.base + first_token + 1, 0, room), most = clamp((long long)q.base + first_token + tokens, 0, room);
      auto source = [&](int t) { return t >= t1 || t * kKv4Tile >= most ? -1 : tile_source(p, at.s, at.slot / p.subs, t); };
      int now = source(t0 + lane), next = source(t0 + 32 + lane);
      tile.clear();
      uint32_t none = 0;            // bit of a slot: nothing to see in its tile
      int ahead = 0, hand = 0;      // slots: of the next tiles to ask for, of the tiles in hand
      auto request = [&](int i) {   // tiles t0 + i ..
        if (i > 0 && (i & 31) == 0) {
          now = next;
          next = source(t0 + i + 32 + lane);
        }
#pragma unroll
        for (int k = 0; k < KT; ++k) {
          const int from = __shfl_sync(0xffffffffu, now, (i + k) & 31);
          none = from < 0 ? none | 1u << (ahead + k) : none & ~(1u << (ahead + k));
          if (from >= 0) {
            const uint8_t *src = p.pool + (int64_t)from * BYTES + lane * 16;
            uint8_t *to = ring + (ahead + k) * BYTES + lane * 16;
#pragma unroll
            for (int c = 0; c < BYTES / 512; ++c)
              copy16(to + c * 512, src + c * 512);
            if (BYTES % 512 != 0 && lane < BYTES % 512 / 16)
              copy16(to + BYTES / 512 * 512, src + BYTES / 512 * 512);
          }
        }
        copies_commit();
        ahead = (ahead + KT) % kSlots;
      };
      const int count = t1 - t0;
      __syncwarp();
#pragma unroll
      for (int i = 0; i < STAGES - 1; ++i)
        request(i * KT);
      tile.load_q(p, lane / 4 < live, lane / 4 < live ? row_at(p, q.r0 + first_token, at.slot, lane / 4, p.a.q_ld, D) : 0);
#pragma unroll 1
      for (int i = 0; i < count; i += KT) {
        copies_wait<STAGES - 2>();
        __syncwarp();
        const uint32_t skip = none >> hand & ((1u << KT) - 1);
        const uint8_t *bytes = ring + hand * BYTES;
        hand = (hand + KT) % kSlots;
        request(i + kSlots - KT);
        if (skip == (1u << KT) - 1)
          continue;
        int j0[KT], limit[2] = {0, 0};
#pragma unroll
        for (int k = 0; k < KT; ++k)
          j0[k] = skip >> k & 1 ? room : (t0 + i + k) * kKv4Tile;   // (no row sees a key from `room` on)
        if (j0[KT - 1] + kKv4Tile <= least && skip == 0) {
          tile.template keys<false>(bytes, j0, limit);
        } else {
#pragma unroll
          for (int e = 0; e < 2; ++e) {
            const int row = 2 * (lane & 3) + e;
            limit[e] = row < live ? clamp((long long)q.base + first_token + (row * p.over_heads >> 16) + 1, 0, room) : 0;
          }
          tile.template keys<true>(bytes, j0, limit);
        }
      }
      copies_wait<0>();
      __syncwarp();
      tile.finish();
      // ---- whole, or a part -------------------------------------------------------------------------------------------------------
      if (t0 == 0 && t1 == all) {
        float over[2];
#pragma unroll
        for (int e = 0; e < 2; ++e)
          over[e] = tile.l[e] == 0.f ? 0.f : 1.f / tile.l[e];
#pragma unroll
        for (int e = 0; e < 2; ++e) {
          const int row = 2 * (lane & 3) + e;
          if (row < live) {
            const int64_t to = row_at(p, q.r0 + first_token, at.slot, row, p.a.out_ld, D) + lane / 4;
#pragma unroll
            for (int i = 0; i < D / 16; ++i) {
              put<TYPE>(p, to + 16 * i, tile.l[e] == 0.f ? 0.f : tile.o[i][e] * over[e]);
              put<TYPE>(p, to + 16 * i + 8, tile.l[e] == 0.f ? 0.f : tile.o[i][2 + e] * over[e]);
            }
          }
        }
      } else {   // a part of the first item, or of the last; that of the first has to lie elsewhere where others follow
        float *part = t0 > 0 && !here ? p.parts + ((int64_t)2 * kKv4Ctas + blockIdx.x * kWarps + warp) * PART : reinterpret_cast<float *>(ring);
        tile.store(part);
        if (lane == 0) {
          Left &left = s_left[warp];
          if (t0 > 0) {
            left.has_a = true;
            left.a_ends = t1 == all;
            left.a_tiles = count;
            left.a_part = part;
            left.a = at;
          } else {
            left.has_b = true;
            left.b_tiles = count;
            left.b = at;
          }
        }
      }
      if (here)
        break;
      plan.next_item(at, q);
    }
  }
  __syncthreads();

  // ---- parts of items: over the warps of this CTA, then over CTAs ----------------------------------------------------------------
  const uint32_t has_a = __ballot_sync(0xffffffffu, lane < act && s_left[lane % kWarps].has_a), has_b = __ballot_sync(0xffffffffu, lane < act && s_left[lane % kWarps].has_b);
  const uint32_t ends = __ballot_sync(0xffffffffu, lane < act && s_left[lane % kWarps].has_a && s_left[lane % kWarps].a_ends);
  // A chain: the parts of an item, of neighbouring warps.  One may have begun in another CTA (chain 0, then), the others are opened by the warps of
  // has_b; the last of them may go on in the next CTA.
  const int incoming = has_a & 1, chains = incoming + __popc(has_b);
  if (chains == 0)
    return;
  struct Chain {
    int first, last;
    bool opened, whole;
  };
  auto chain = [&](int k) {
    Chain c;
    c.opened = k >= incoming;
    uint32_t b = has_b;
    for (int i = incoming; i < k; ++i)
      b &= b - 1;
    c.first = c.opened ? __ffs(b) - 1 : 0;
    const uint32_t end = ends >> (c.first + c.opened) << (c.first + c.opened);
    c.last = end != 0 ? __ffs(end) - 1 : act - 1;
    c.whole = c.opened && end != 0;
    return c;
  };
  auto add = [](float4 &o, float &l, float4 v, float pl, float f) {
    l = fmaf(pl, f, l);
    o = make_float4(fmaf(v.x, f, o.x), fmaf(v.y, f, o.y), fmaf(v.z, f, o.z), fmaf(v.w, f, o.w));
  };
  auto write_out = [&](const Place &at, int row, int d, float4 o, float l) {
    const Sequence q = plan.sequence(at.s);
    if (row >= rows_of(p, q, at.rt, at.slot))
      return;
    const float over = l == 0.f ? 0.f : 1.f / l;
    put4<TYPE>(p, row_at(p, q.r0 + at.rt * p.tokens, at.slot, row, p.a.out_ld, D) + d, l == 0.f ? make_float4(0.f, 0.f, 0.f, 0.f) : make_float4(o.x * over, o.y * over, o.z * over, o.w * over));
  };
  // chains side by side, a power of two of them, a warp each at least
  constexpr int FOURS = kRows * D / 4;
  const int lanes = max(32, kThreads >> (32 - __clz(chains - 1)));
  for (int i = tid; i < chains * lanes; i += kThreads) {
    const int k = i / lanes;
    const Chain c = chain(k);
    auto part = [&](int w) { return c.opened && w == c.first ? reinterpret_cast<const float *>(s_all + w * RING) : s_left[w].a_part; };
    // a lane's share of the rows, all of it at once; part by part, to the larger reference
    constexpr int MOST = FOURS / 32;
    float top[MOST], l[MOST];
    float4 o[MOST];
#pragma unroll
    for (int u = 0; u < MOST; ++u) {
      top[u] = kKv4Seed;
      l[u] = 0.f;
      o[u] = make_float4(0.f, 0.f, 0.f, 0.f);
    }
    const int e0 = i % lanes;
    if (lanes >= FOURS) {   // (an element a lane, and many parts: loads side by side)
      const int row = e0 / (D / 4), d = e0 % (D / 4) * 4;
      if (e0 >= FOURS)
        break;
#pragma unroll 4
      for (int w = c.first; w <= c.last; ++w)
        top[0] = fmaxf(top[0], part(w)[kRows * (D + 4) + row]);
#pragma unroll 4
      for (int w = c.first; w <= c.last; ++w) {
        const float *x = part(w);
        add(o[0], l[0], *reinterpret_cast<const float4 *>(x + row * (D + 4) + d), x[kRows * (D + 4) + kRows + row], ex2(x[kRows * (D + 4) + row] - top[0]));
      }
    }
#pragma unroll 1
    for (int w = c.first; w <= c.last && lanes < FOURS; ++w) {
      const float *x = part(w);
#pragma unroll
      for (int u = 0; u < MOST; ++u) {
        const int e = e0 + u * lanes, row = e / (D / 4), d = e % (D / 4) * 4;
        if (e < FOURS) {
          const float r = x[kRows * (D + 4) + row], to = fmaxf(top[u], r), keep = ex2(top[u] - to);
          const float4 v = *reinterpret_cast<const float4 *>(x + row * (D + 4) + d);
          top[u] = to;
          l[u] *= keep;
          o[u] = make_float4(o[u].x * keep, o[u].y * keep, o[u].z * keep, o[u].w * keep);
          add(o[u], l[u], v, x[kRows * (D + 4) + kRows + row], ex2(r - to));
        }
      }
    }
#pragma unroll
    for (int u = 0; u < MOST; ++u) {
      const int e = e0 + u * lanes, row = e / (D / 4), d = e % (D / 4) * 4;
      if (e >= FOURS)
        break;
      if (c.whole) {
        write_out(s_left[c.first].b, row, d, o[u], l[u]);
      } else {
        float *to = p.parts + ((int64_t)blockIdx.x * 2 + c.opened) * PART;
        *reinterpret_cast<float4 *>(to + row * (D + 4) + d) = o[u];
        if (d == 0) {
          to[kRows * (D + 4) + row] = top[u];
          to[kRows * (D + 4) + kRows + row] = l[u];
        }
      }
    }
  }
  const bool outgoing = !chain(chains - 1).whole && chain(chains - 1).opened;
  if (!incoming && !outgoing)
    return;
  __threadfence();
  __syncthreads();
  if (warp < 2 && (warp == 0 ? incoming : outgoing)) {
    const Chain c = chain(warp == 0 ? 0 : chains - 1);
    int tiles = 0, from, to;
    for (int w = c.first; w <= c.last; ++w)
      tiles += c.opened && w == c.first ? s_left[w].b_tiles : s_left[w].a_tiles;
    if (plan.arrive(p.counters, c.opened ? s_left[c.first].b : s_left[0].a, tiles, from, to) && lane == 0) {
      s_ctas[warp][0] = 1;
      s_ctas[warp][1] = from;
      s_ctas[warp][2] = to;
    }
  }
  __syncthreads();
  const int row = tid % FOURS / (D / 4), d = tid % (D / 4) * 4;
  for (int k = tid / FOURS; k < 2; k += kThreads / FOURS) {
    if (s_ctas[k][0] == 0)
      continue;
    __threadfence();
    const Chain c = chain(k == 0 ? 0 : chains - 1);
    const int from = s_ctas[k][1], to = s_ctas[k][2];
    auto part = [&](int b) { return p.parts + ((int64_t)b * 2 + (b == from)) * PART; };
    float top = kKv4Seed, l = 0.f;
    float4 o = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll 4
    for (int b = from; b <= to; ++b)
      top = fmaxf(top, __ldcg(part(b) + kRows * (D + 4) + row));
#pragma unroll 4
    for (int b = from; b <= to; ++b)
      add(o, l, __ldcg(reinterpret_cast<const float4 *>(part(b) + row * (D + 4) + d)), __ldcg(part(b) + kRows * (D + 4) + kRows + row),
          ex2(__ldcg(part(b) + kRows * (D + 4) + row) - top));
    write_out(c.opened ? s_left[c.first].b : s_left[0].a, row, d, o, l);
  }
}

RaisedOn g_raised[6];

template <int D, int TYPE> int attention_launch(RaisedOn &raised, const Kv4Params &p, cudaStream_t st) {
  const int fixed = kWarps * kSlots * kv4_tile_bytes(D);
  if (int rc = raise_shared_limit(raised, (const void *)kv4_attention_kernel<D, TYPE>, fixed + KeyPlan<4>::bytes(B200_KV4_ATTENTION_MAX_SEQS)))
    return rc;
  return launch_after(kv4_attention_kernel<D, TYPE>, dim3(kKv4Ctas), kThreads, fixed + KeyPlan<4>::bytes(p.a.n_seqs), st, p);
}

} // namespace

const int *kv4_attention_error(const void *workspace) { return (const int *)workspace + kKv4Ctas; }

} // namespace b200

using namespace b200;

extern "C" {

int64_t b200_kv4_attention_workspace_bytes(int q_heads, int kv_heads, int head_dim) {
  if (kv_heads < 1 || kv_heads > 1024 || q_heads < 1 || q_heads % kv_heads != 0 || (head_dim != 64 && head_dim != 128))
    return B200_EINVAL;
  return 2048 + (int64_t)kKv4Ctas * std::max<int64_t>((2 + kWarps) * part_floats(head_dim), kv4_chunk_part_floats(head_dim)) * 4;
}

int b200_kv4_attention_status(void *workspace, void *stream) {
  if (!workspace)
    return fail(B200_EINVAL, "kv4_attention_status: null workspace");
  if (int rc = ensure_device())
    return rc;
  int code = 0;
  B200_CUDA(cudaMemcpyAsync(&code, kv4_attention_error(workspace), 4, cudaMemcpyDeviceToHost, (cudaStream_t)stream));
  B200_CUDA(cudaStreamSynchronize((cudaStream_t)stream));
  return code == 0 ? B200_OK : fail(B200_ECUDA, "kv4_attention: a bounded wait gave up (code %d)", code);
}

int b200_kv4_attention(const b200_kv4_cache *c, const b200_kv4_attention_args *a, void *workspace, int64_t workspace_bytes, void *stream) {
  if (int rc = kv4_check("kv4_attention", c))
    return rc;
  if (!a || (a->rows > 0 && (!a->q || !a->out || !workspace || !a->row_start || !a->lens || !a->block_table)))
    return fail(B200_EINVAL, "kv4_attention: null pointer");
  if (a->dtype != B200_F32 && a->dtype != B200_F16 && a->dtype != B200_BF16)
    return fail(B200_EINVAL, "kv4_attention: element type %d", a->dtype);
  if (a->rows < 0 || a->n_seqs < 1 || a->table_stride < 1 || a->q_heads < 1 || a->q_heads % c->kv_heads != 0 || (int64_t)a->table_stride * c->page > 1 << 30)
    return fail(B200_EINVAL, "kv4_attention: %d rows of %d sequences, tables of %d pages, %d heads on %d", a->rows, a->n_seqs, a->table_stride, a->q_heads,
                c->kv_heads);
  if (a->n_seqs > B200_KV4_ATTENTION_MAX_SEQS)
    return fail(B200_ELIMIT, "kv4_attention: %d sequences (at most %d)", a->n_seqs, B200_KV4_ATTENTION_MAX_SEQS);
  const int64_t cols = (int64_t)a->q_heads * c->head_dim;
  if (a->rows > 1 && (a->q_ld < cols || a->out_ld < cols))
    return fail(B200_EINVAL, "kv4_attention: row strides %lld and %lld of rows of %lld", (long long)a->q_ld, (long long)a->out_ld, (long long)cols);
  const uintptr_t mask = a->dtype == B200_F32 ? 3 : 1;
  if (((uintptr_t)a->q | (uintptr_t)a->out) & mask || ((uintptr_t)a->row_start | (uintptr_t)a->lens | (uintptr_t)a->block_table) & 3)
    return fail(B200_EINVAL, "kv4_attention: a pointer is not aligned to its elements");
  if (a->rows == 0)
    return ensure_device();
  if (a->q == a->out)
    return fail(B200_EINVAL, "kv4_attention: q and out overlap");
  if (workspace_bytes < b200_kv4_attention_workspace_bytes(a->q_heads, c->kv_heads, c->head_dim) || (uintptr_t)workspace & 255)
    return fail(B200_EINVAL, "kv4_attention: a workspace of %lld bytes, aligned to 256, is required",
                (long long)b200_kv4_attention_workspace_bytes(a->q_heads, c->kv_heads, c->head_dim));
  if (int rc = ensure_device())
    return rc;
  Kv4Params p{};
  p.pool = (const uint8_t *)c->pool;
  p.n_pages = c->n_pages;
  p.kv_heads = c->kv_heads;
  p.page = c->page;
  p.a = *a;
  p.G = a->q_heads / c->kv_heads;
  p.log2_scale = a->scale * 1.4426950408889634f;
  const int size = a->dtype == B200_F32 ? 4 : 2;
  p.wide_q = (((uintptr_t)a->q | (uintptr_t)(a->q_ld * size)) & (4 * size - 1)) == 0;
  p.wide_q16 = (((uintptr_t)a->q | (uintptr_t)(a->q_ld * size)) & 15) == 0;
  p.wide_out = (((uintptr_t)a->out | (uintptr_t)(a->out_ld * size)) & (4 * size - 1)) == 0;
  p.counters = (int *)workspace;
  p.parts = (float *)((char *)workspace + 2048);
  p.fill = 1;
  p.least_rows = 1;
  p.most_rows = INT32_MAX;
  p.subs = (p.G + kRows - 1) / kRows;
  p.heads = std::min(p.G, kRows);
  p.tokens = p.subs == 1 ? kRows / p.G : 1;
  p.over_heads = (65536 + p.heads - 1) / p.heads;
  cudaStream_t st = (cudaStream_t)stream;
  // Sequences of many rows go to tcgen05, in a launch of their own, if there is enough to do (pairs of a query vector and a key): the form's beginnings and
  // ends take 35 (bf16) or 50 us where the few-rows form has 12.  Who has how many rows is known on the device only, so both launches are made where the sizes
  // leave it open, and both see from the lengths whose the sequences are.
  // (Few rows, many rows, us; 1000 keys, f32 12 heads on 2, else 32 on 8: f32 20 x 22 rows 54 / 59, 20 x 43 96 / 59; bf16 20 x 16 53 / 71, 20 x 32 88 / 73; f16 20 x 32
  // 91 / 103, 20 x 64 162 / 150; one sequence of 11 rows of f32 18 / 49.)
  // Only where there are 24 query vectors of a kv head for every sequence (or place for one): other calls are decode steps, mostly, which would pay for the second
  // launch and its look at the lengths (128 rows of 32 to 4000 keys, 32 heads on 8: bf16 79 us, 98 with it; f16 91 either way; f32 117, 133).  A chunk beside many of them is
  // the price: 512 rows at 4000 keys and 127 rows take 282 us in bf16, 328 in f16, 471 in f32, where tcgen05 would have 210, 275 and 304; beside 63 they have it (182, 238, 257).
  const bool exact = a->dtype != B200_BF16;   // (a bf16 result is rounded eight times as far as f16 operands are)
  const double work = a->dtype == B200_F32 ? 5.5e6 : exact ? 30e6 : 15e6, vectors = (double)a->rows * a->q_heads;
  if ((exact ? kv4_exact_takes(p.G, a->n_seqs) : kv4_chunk_takes(p.G, a->n_seqs)) && (int64_t)a->rows * p.G >= kChunkRows &&
      (int64_t)a->rows * p.G >= 24 * (int64_t)a->n_seqs && vectors * a->table_stride * c->page >= work) {
    const bool only = a->n_seqs == 1 && vectors * a->rows / 2 >= work;   // (rows that see one another, if nothing before them)
    Kv4Params chunk = p;
    chunk.least_rows = (kChunkRows + p.G - 1) / p.G;
    chunk.many = true;
    if (only) {
      chunk.least_rows = 1;
    } else {
      p.most_rows = chunk.least_rows - 1;
      p.many_rows = chunk.many_rows = chunk.least_rows;
      p.least_work = chunk.least_work = std::max<int64_t>(1, (int64_t)(work / a->q_heads));
      chunk.fill = 0;
    }
    if (int rc = exact ? kv4_exact_launch(chunk, c->head_dim, st) : kv4_chunk_launch(chunk, c->head_dim, st))
      return rc;
    if (only)
      return B200_OK;
  }
#define B200_D(D_)                                                                                                                    \
  (a->dtype == B200_F32   ? attention_launch<D_, B200_F32>(g_raised[D_ / 64 - 1], p, st)                                              \
   : a->dtype == B200_F16 ? attention_launch<D_, B200_F16>(g_raised[D_ / 64 + 1], p, st)                                              \
                          : attention_launch<D_, B200_BF16>(g_raised[D_ / 64 + 3], p, st))
  return c->head_dim == 128 ? B200_D(128) : B200_D(64);
#undef B200_D
}

} // extern "C"
