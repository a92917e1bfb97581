// Attention over the 4-bit KV cache for sequences of many f32 or f16 rows (a prompt, or a chunk of one) on the 5th-generation tensor cores.
//
// Products of f32's accuracy out of f16 operands: q and the weights are two f16 terms each (22 bits, after a power of two of the row; q of f16 is one), and so
// is what is left of a value once it is centred.  With v = (c - 8) s + m, m = lo + 8 s,
//   q.k = sum over dims of q (c - 8) s + sum over groups of m (sum of q)       sum p v = sum p (c - 8) s + sum p m:
// (c - 8) s has 15 bits at most, so that its rounding to f16 and what that leaves are two terms without any error, made by a product and an fma; the parts with m
// are a few f32 operations of the thread that has the row.  Three of the four products of terms are summed, the small ones first, and a block's product is added to
// those before it outside the tensor cores, whose sums round towards zero: eight such steps count, of centred values.
//
// Seven warps make the operands of 128 keys: K of a block while the softmax has the one before it, V when the product of the block before is done.  Eight
// do the softmax, two threads per row: scores of half a block each, the larger of their maxima (through shared memory) decides whether the row's
// reference moves, weights.  Scores of two blocks have their own columns (2 x 128), O and its sum D each.
//
// A prompt of 1000 f32 rows, 12 heads on 2 of 128 dims: 53 us (the few-rows form 70), errors 3 to 4e-7 of the result; 4000 rows: 415 us, 118 TFLOP/s.  A block takes some
// 8000 clocks, 5400 of them the softmax, and 2300 for the products: a tile's K takes a maker 2300, its V 1450, and of seven makers one has two tiles.  Eight
// (17 warps of 96 registers) spill, 63 us; one thread per row and eight makers take as long here and 13 % longer at 4000 rows.  Items that CTAs share come together too
// slowly to be worth it (78 us).  f16, 1001 rows at 4000 keys, 32 heads on 8: 265 us (kv4_chunk.cu, whose errors would be 2.5 times f16's rounding: 120).
#include "kv4_rows.cuh"

#include <algorithm>
#include <type_traits>

namespace b200 {

namespace {

constexpr int kSoftmaxWarps = 8, kMakers = 7, kThreads = 32 * (kSoftmaxWarps + kMakers + 1);
constexpr int kNotes = 4;
constexpr uint32_t kCols = 512;
constexpr int kLeastKeys = 256, kSplit = 1200;

template <int D> struct Shape {
  static constexpr int GROUPS = D / kKv4Group, BYTES = kv4_tile_bytes(D);
  static constexpr uint32_t TERM = kRows * D * 2;   // bytes of a term of q, K or V
  static constexpr int PART = rows_part<D, kRows>();
  static constexpr int SMEM = 1024 + 6 * TERM;
  static constexpr uint32_t COL_S = 0, COL_O = 2 * kKeys, COL_SUM = COL_O + kRows;   // (a block's product; those of the blocks before)
};

// What the softmax has to know of a block's keys.
struct Notes {
  __align__(16) float k_mid[2][kKeys], v_mid[2][kKeys];   // m, by group
  // bits of sixteen keys, by tile: any of the next; K not finite; no page; V not finite, by group
  __align__(16) uint16_t special[8];
  uint16_t k_bad[8], hole[8], v_bad[2][8];
  __device__ __forceinline__ static uint32_t word(const uint16_t *x, int c) { return reinterpret_cast<const uint32_t *>(x)[c]; }   // of keys 32 c ..
};
struct Bars {
  uint64_t k_full, v_full, s_full[2], p_ready[2], pv_done, q_full;
  uint32_t tmem_base;
  int abort_flag;
  Meeting meeting;
  float row[kRows][4];         // its scores' factor, sums of q
  float top[2][2][kRows];      // of a row's half of a block: largest score
  float4 half[2][kRows];       // of a row's half of the keys: total, sums with m, marks
  long long sums[2 * (kThreads / 32) + 1];
  Notes notes[kNotes];
};

// c - 8 of the low nibble of each byte-pair of w, and of the high one
__device__ __forceinline__ uint32_t low_codes(uint32_t w) {
  uint32_t x = (w & 0x000f000fu) | 0x64006400u;                        // 1024 + c
  asm("add.rn.f16x2 %0, %0, %1;" : "+r"(x) : "r"(0xe408e408u));
  return x;
}
__device__ __forceinline__ uint32_t high_codes(uint32_t w) { return fma2((w & 0x00f000f0u) | 0x64006400u, 0x2c002c00u, 0xd480d480u); }   // 1024 + 16 c, / 16 - 72
// c s as two terms; HELD: the first within +-65504
template <bool HELD> __device__ __forceinline__ void terms(uint32_t c, uint32_t s, uint32_t &high, uint32_t &low) {
  asm("mul.rn.f16x2 %0, %1, %2;" : "=r"(high) : "r"(c), "r"(s));
  if constexpr (HELD) {
    asm("min.f16x2 %0, %0, %1;" : "+r"(high) : "r"(0x7bff7bffu));
    asm("max.f16x2 %0, %0, %1;" : "+r"(high) : "r"(0xfbfffbffu));
  }
  low = fma2(c, s, high ^ 0x80008000u);
}

template <int D, int TYPE> __global__ void __launch_bounds__(kThreads, 1) kv4_exact_kernel(const __grid_constant__ Kv4Params p) {
  using H = Shape<D>;
  constexpr int GROUPS = H::GROUPS;
  extern __shared__ __align__(1024) uint8_t smem[];
  uint8_t *qs = reinterpret_cast<uint8_t *>(((uintptr_t)smem + 1023) & ~(uintptr_t)1023);
  uint8_t *ks = qs + 2 * H::TERM, *vs = ks + 2 * H::TERM, *s_plan = vs + 2 * H::TERM;   // (the larger terms, then the smaller ones)
  __shared__ Bars bars;
  const int warp = __shfl_sync(0xffffffffu, (int)threadIdx.x >> 5, 0), lane = threadIdx.x & 31;
  volatile int *ab = &bars.abort_flag;
  int *error = p.counters + kKv4Ctas;

  if (threadIdx.x == 0) {
    mbar_init(&bars.k_full, kTiles);
    mbar_init(&bars.v_full, kTiles);
    for (int i = 0; i < 2; ++i) {
      mbar_init(&bars.s_full[i], 1);
      mbar_init(&bars.p_ready[i], kSoftmaxWarps);
    }
    mbar_init(&bars.pv_done, 1);
    mbar_init(&bars.q_full, kSoftmaxWarps);
    bars.abort_flag = 0;
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
  }
  if (warp == kSoftmaxWarps + kMakers) {
    asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(&bars.tmem_base)), "n"(kCols) : "memory");
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
  }
  fence_before();
  __syncthreads();
  fence_after();
  const uint32_t tmem = __shfl_sync(0xffffffffu, bars.tmem_base, 0);
  kernel_go();   // not before the allocation: see tensor_core.cuh
  kernel_wait();
  const int room = p.a.table_stride * p.page;
  RowsPlan plan;
  plan.build<kThreads>(p, s_plan, bars.sums, kLeastKeys, kSplit);
  if (p.fill) {
    const int lo = plan.r0[0], hi = max(lo, plan.r0[plan.n]), none = lo + p.a.rows - hi, cols = p.a.q_heads * D;
    for (int64_t i = (int64_t)blockIdx.x * kThreads + threadIdx.x; i < (int64_t)none * cols; i += (int64_t)gridDim.x * kThreads) {
      const int r = (int)(i / cols);
      put<TYPE>(p, (int64_t)(r < lo ? r : hi + r - lo) * p.a.out_ld + i % cols, 0.f);
    }
  }
  const bool works = plan.total > 0 && (int)blockIdx.x < plan.ctas;
  auto wait = [&](bool &ok, uint64_t *bar, uint32_t parity, int code) {   // whole warps leave the poll; who gave up goes on without waiting
    if (ok)
      ok = __all_sync(0xffffffffu, mbar_wait(bar, parity & 1, ab, error, code));
  };

  if (works && warp < kSoftmaxWarps) {
    // ---- softmax: two threads per row, of half a block's keys each ----------------------------------------------------------------------
    const int row = (warp & 3) * 32 + lane, side = warp >> 2;
    const uint32_t lanes = tmem + ((uint32_t)((warp & 3) * 32) << 16), col_o = lanes + H::COL_O + side * (D / 2), col_sum = lanes + H::COL_SUM + side * (D / 2);
    auto pair_meets = [&]() { asm volatile("bar.sync %0, 64;" ::"r"(2 + (warp & 3)) : "memory"); };   // (the two warps of the same rows)
    bool ok = true;
    uint32_t made = 0;
    Walk walk(plan);
    Segment g;
    while (walk.next(plan, g)) {
      const uint32_t n = g.b1 - g.b0;
      float r = kKv4Seed, l = 0.f, sum_q[GROUPS];
      uint64_t bias[GROUPS] = {};               // sums of p m, over even and odd keys
      uint32_t marks = 0;                       // V groups that become NaN
      const int token = row / p.G;
      const bool live = token < min(g.tokens, p.tokens);
      const int seen_by = live ? clamp((long long)g.base + g.first + token + 1, 0, room) : 0;
      {
        // ---- q: times a power of two, as two f16; row by row, four dims a lane
        constexpr int LANES = D / 4, BATCH = 8;   // lanes of a row (of 64 dims: two rows at once); loads side by side
        const int64_t mine = live ? row_at(p, g.r0 + g.first, g.at.slot, row, p.a.q_ld, D) : -1;
        const int d = 4 * (lane % LANES);
#pragma unroll 1
        for (int from = 0; from < LANES / 2; from += BATCH) {
          float batch[BATCH][4], most[BATCH], sum[BATCH];
          // (this warp's rows: the first or second half of the 32)
          auto which = [&](int b) { return 16 * side + 32 / LANES * (from + b) + lane / LANES; };
#pragma unroll
          for (int b = 0; b < BATCH; ++b) {
            float (&x)[4] = batch[b];
            const int64_t at = __shfl_sync(0xffffffffu, mine, which(b));
#pragma unroll
            for (int e = 0; e < 4; ++e)
              x[e] = 0.f;
            if (at >= 0 && p.wide_q)
              load_wide<TYPE>(p.a.q, at + d, x);
            else if (at >= 0)
#pragma unroll
              for (int e = 0; e < 4; ++e)
                x[e] = load_as_float(p.a.q, TYPE, at + d + e);
          }
#pragma unroll
          for (int b = 0; b < BATCH; ++b) {
            const float (&x)[4] = batch[b];
            most[b] = max3(fmaxf(fabsf(x[0]), fabsf(x[1])), fabsf(x[2]), fabsf(x[3]));
            sum[b] = (x[0] + x[1]) + (x[2] + x[3]);
          }
#pragma unroll
          for (int o = 1; o < LANES; o <<= 1)   // (all rows' steps side by side)
#pragma unroll
            for (int b = 0; b < BATCH; ++b)
              most[b] = fmaxf(most[b], __shfl_xor_sync(0xffffffffu, most[b], o));
#pragma unroll
          for (int o = 1; o < 16; o <<= 1)
#pragma unroll
            for (int b = 0; b < BATCH; ++b)
              sum[b] += __shfl_xor_sync(0xffffffffu, sum[b], o);
#pragma unroll
          for (int b = 0; b < BATCH; ++b) {
            const float (&x)[4] = batch[b];
            const int up = min(max(14 + 127 - (int)(__float_as_uint(most[b]) >> 23), -113), 100), at = (warp & 3) * 32 + which(b);
            const float by = power(up);
            if (lane % LANES == 0)
              bars.row[at][0] = power(-up) * p.log2_scale;
            if (lane % 16 == 0)
              bars.row[at][1 + lane % LANES / 16] = sum[b] * p.log2_scale;
            const float a[4] = {x[0] * by, x[1] * by, x[2] * by, x[3] * by};
            const uint32_t high[2] = {pack_f16(a[0], a[1]), pack_f16(a[2], a[3])};
            const uint32_t to = smem_u32(qs) + at * 128 + d / 64 * (kRows * 128) + ((d / 8 % 8 ^ (at & 7)) << 4) + d % 8 * 2;
            store2(to, high[0], high[1]);
            if constexpr (TYPE == B200_F32) {
              const float2 f = halves(high[0]), h = halves(high[1]);
              store2(to + H::TERM, pack_f16(a[0] - f.x, a[1] - f.y), pack_f16(a[2] - h.x, a[3] - h.y));
            }
          }
        }
        fence_proxy();
        fence_before();
        __syncwarp();
        if (lane == 0)
          mbar_arrive(&bars.q_full);
        pair_meets();
      }
      float factor = bars.row[row][0];
#pragma unroll
      for (int gr = 0; gr < GROUPS; ++gr) {
        sum_q[gr] = bars.row[row][1 + gr];
        if (!(sum_q[gr] - sum_q[gr] == 0.f))    // (a row with an infinity, or NaN, has no scores)
          factor = NAN;
      }
      for (uint32_t j = 0; j < n; ++j) {
        const uint32_t block = made + j, col_s = lanes + H::COL_S + (block & 1) * kKeys + side * (kKeys / 2);
        const int key0 = (g.b0 + j) * kKeys, seen = min(max(seen_by - key0, 0), kKeys);   // keys of the block that this row sees
        if (j > 0) {
          // ---- the block before's product joins the sum, with rounding to nearest
          // (every product is waited for before the next can begin: a wait tells one phase from its neighbours only)
          wait(ok, &bars.pv_done, block - 1, 743);
          fence_after();
#pragma unroll 1
          for (int i = 0; i < D / 2; i += 32) {
            uint32_t w[32], sum[32];
            tmem_load32(col_o + i, w);
            tmem_arrived(w);
            if (j > 1) {
              tmem_load32(col_sum + i, sum);
              tmem_arrived(sum);
#pragma unroll
              for (int e = 0; e < 32; ++e)
                w[e] = __float_as_uint(__uint_as_float(w[e]) + __uint_as_float(sum[e]));
            }
            tmem_store32(col_sum + i, w);
          }
          tmem_wait_store();
        }
        wait(ok, &bars.s_full[block & 1], block >> 1, 741);
        fence_after();
        // (the makers wrote them before the products that have been waited for could begin; another block's come four blocks later)
        const Notes &notes = bars.notes[block % kNotes];
        const uint4 any_special = *reinterpret_cast<const uint4 *>(notes.special);
        const bool special = (any_special.x | any_special.y | any_special.z | any_special.w) != 0;
        const bool masked = special || __any_sync(0xffffffffu, live && seen < kKeys);
        auto sees = [&](int c) {   // of keys 32 c ..: a bit each
          const int k = seen - 32 * c;
          return (k >= 32 ? 0xffffffffu : k <= 0 ? 0u : (1u << k) - 1) & ~Notes::word(notes.hole, c);
        };
        // ---- scores, back in their place, and the largest
        float top = -INFINITY;
        auto score = [&](auto hidden) {
          constexpr bool HIDDEN = decltype(hidden)::value;
          const uint64_t ff = pack2(factor, factor);
#pragma unroll 1
          for (int i = 0; i < 2; ++i) {
            const int c = 2 * side + i;
            uint32_t w[32];
            tmem_load32(col_s + 32 * i, w);
            tmem_arrived(w);
            const uint32_t m = HIDDEN ? sees(c) : 0u;
            float x[4] = {-INFINITY, -INFINITY, -INFINITY, -INFINITY};
#pragma unroll
            for (int k = 0; k < 32; k += 4) {
              uint64_t mid[2] = {};
#pragma unroll
              for (int gr = 0; gr < GROUPS; ++gr) {
                const float4 f = *reinterpret_cast<const float4 *>(notes.k_mid[gr] + 32 * c + k);
                const uint64_t by = pack2(sum_q[gr], sum_q[gr]);
                mid[0] = gr == 0 ? mul_2(pack2(f.x, f.y), by) : fma_2(pack2(f.x, f.y), by, mid[0]);
                mid[1] = gr == 0 ? mul_2(pack2(f.z, f.w), by) : fma_2(pack2(f.z, f.w), by, mid[1]);
              }
#pragma unroll
              for (int e = 0; e < 4; e += 2) {
                const float2 y = unpack2(fma_2(pack2(__uint_as_float(w[k + e]), __uint_as_float(w[k + e + 1])), ff, mid[e / 2]));
                w[k + e] = !HIDDEN || m >> (k + e) & 1 ? __float_as_uint(y.x) : 0xff800000u;
                w[k + e + 1] = !HIDDEN || m >> (k + e + 1) & 1 ? __float_as_uint(y.y) : 0xff800000u;
                x[k / 2 + e / 2 & 3] = max3(x[k / 2 + e / 2 & 3], __uint_as_float(w[k + e]), __uint_as_float(w[k + e + 1]));
              }
            }
            tmem_store32(col_s + 32 * i, w);
            top = fmaxf(top, fmaxf(max3(x[0], x[1], x[2]), x[3]));
          }
        };
        if (masked)
          score(std::true_type());
        else
          score(std::false_type());
        bars.top[block & 1][side][row] = top;
        tmem_wait_store();
        pair_meets();
        top = fmaxf(top, bars.top[block & 1][1 - side][row]);
        // ---- a row's reference moves (both threads know it, and have half of the sums each)
        if (__any_sync(0xffffffffu, kv4_moves(top, r))) {
          const float to = kv4_moves(top, r) ? kv4_reference(ceilf(top)) : r, keep = ex2(r - to);   // (each row for itself)
          r = to;
          l *= keep;
#pragma unroll
          for (int gr = 0; gr < GROUPS; ++gr)
            bias[gr] = mul_2(bias[gr], pack2(keep, keep));
          if (j > 0)
#pragma unroll 1
            for (int i = 0; i < D / 2; i += 32) {
              uint32_t w[32];
              tmem_load32(col_sum + i, w);
              tmem_arrived(w);
#pragma unroll
              for (int e = 0; e < 32; ++e)
                w[e] = __float_as_uint(__uint_as_float(w[e]) * keep);
              tmem_store32(col_sum + i, w);
            }
        }
        // ---- weights, as two f16 in the place of the scores that they were
        auto weigh = [&](auto hidden) {
          constexpr bool HIDDEN = decltype(hidden)::value;
          const uint64_t rr = pack2(-r, -r);
#pragma unroll 1
          for (int i = 0; i < 2; ++i) {
            const int c = 2 * side + i;
            uint32_t w[32], out[32];
            tmem_load32(col_s + 32 * i, w);
            tmem_arrived(w);
            const uint32_t m = HIDDEN ? sees(c) : 0u, bad = HIDDEN ? Notes::word(notes.k_bad, c) & m : 0u;
            uint64_t sum[2] = {};
#pragma unroll
            for (int k = 0; k < 32; k += 4) {
              uint64_t both[2];
#pragma unroll
              for (int e = 0; e < 4; e += 2) {
                float2 y = unpack2(add_2(pack2(__uint_as_float(w[k + e]), __uint_as_float(w[k + e + 1])), rr));
                y.x = ex2(y.x);
                y.y = ex2(y.y);
                if constexpr (HIDDEN) {
                  y.x = bad >> (k + e) & 1 ? NAN : m >> (k + e) & 1 ? y.x : 0.f;
                  y.y = bad >> (k + e + 1) & 1 ? NAN : m >> (k + e + 1) & 1 ? y.y : 0.f;
                }
                both[e / 2] = pack2(y.x, y.y);
                sum[e / 2] = add_2(sum[e / 2], both[e / 2]);
                const uint32_t high = pack_f16(y.x, y.y);
                const float2 f = halves(high);
                out[(k + e) / 2] = high;
                out[16 + (k + e) / 2] = pack_f16(y.x - f.x, y.y - f.y);
              }
#pragma unroll
              for (int gr = 0; gr < GROUPS; ++gr) {
                const float4 f = *reinterpret_cast<const float4 *>(notes.v_mid[gr] + 32 * c + k);
                bias[gr] = fma_2(both[0], pack2(f.x, f.y), bias[gr]);
                bias[gr] = fma_2(both[1], pack2(f.z, f.w), bias[gr]);
              }
            }
            const float2 all = unpack2(add_2(sum[0], sum[1]));
            l += all.x + all.y;
            tmem_store32(col_s + 32 * i, out);
            if constexpr (HIDDEN)
#pragma unroll
              for (int gr = 0; gr < GROUPS; ++gr)
                marks |= (Notes::word(notes.v_bad[gr], c) & m) != 0 ? 1u << gr : 0u;
          }
        };
        if (masked)
          weigh(std::true_type());
        else
          weigh(std::false_type());
        tmem_wait_store();
        fence_before();
        __syncwarp();
        if (lane == 0)
          mbar_arrive(&bars.p_ready[block & 1]);
      }
      made += n;
      // ---- the rows' sums: out, or a part; half of the dims each ----------------------------------------------------------------------
      {
        float b[GROUPS];
#pragma unroll
        for (int gr = 0; gr < GROUPS; ++gr) {
          const float2 f = unpack2(bias[gr]);
          b[gr] = f.x + f.y;
        }
        bars.half[side][row] = make_float4(l, b[0], b[GROUPS - 1], __uint_as_float(marks));
      }
      pair_meets();
      const float4 x = bars.half[0][row], y = bars.half[1][row];
      l = x.x + y.x;
      marks = __float_as_uint(x.w) | __float_as_uint(y.w);
      const int gr = GROUPS == 2 ? side : 0;
      const float b = gr == 0 ? x.y + y.y : x.z + y.z;
      const bool whole = g.b0 == 0 && g.b1 == g.all;
      float *part = p.parts + ((int64_t)blockIdx.x * 2 + (g.b0 == 0)) * H::PART;
      const int64_t to = live ? row_at(p, g.r0 + g.first, g.at.slot, row, p.a.out_ld, D) : 0;
      wait(ok, &bars.pv_done, made - 1, 749);
      fence_after();
#pragma unroll 1
      for (int c = 0; c < D / 2; c += 32) {
        uint32_t w[32];
        tmem_load32(col_o + c, w);
        tmem_arrived(w);
        if (n > 1) {
          uint32_t sum[32];
          tmem_load32(col_sum + c, sum);
          tmem_arrived(sum);
#pragma unroll
          for (int e = 0; e < 32; ++e)
            w[e] = __float_as_uint(__uint_as_float(w[e]) + __uint_as_float(sum[e]));
        }
        if (live) {
#pragma unroll
          for (int e = 0; e < 32; e += 4) {
            const float o[4] = {__uint_as_float(w[e]) + b, __uint_as_float(w[e + 1]) + b, __uint_as_float(w[e + 2]) + b, __uint_as_float(w[e + 3]) + b};
            const int d = side * (D / 2) + c + e;
            if (whole)
              put_over<TYPE>(p, to + d, o, l, marks >> gr & 1);
            else
              __stcg(reinterpret_cast<float4 *>(part) + d / 4 * kRows + row, make_float4(o[0], o[1], o[2], o[3]));
          }
        }
      }
      fence_before();
      if (whole)
        continue;
      if (live && side == 0) {
        float *rest = part + kRows * D;
        rest[row] = r;
        rest[kRows + row] = l;
#pragma unroll
        for (int i = 0; i < GROUPS; ++i)
          rest[(2 + i) * kRows + row] = marks >> i & 1 ? 1.f : 0.f;
      }
      meet<D, TYPE, kRows, 32 * kSoftmaxWarps>(p, plan, g, bars.meeting, row, live, to, side * (D / 2), (side + 1) * (D / 2));
    }
  } else if (works && warp < kSoftmaxWarps + kMakers) {
    // ---- makers: every seventh tile each; K of a tile, then V of the one before ------------------------------------------------------------
    const int mw = warp - kSoftmaxWarps, gq = lane >> 2, t = lane & 3;
    // (rows of K and of V^T that a lane writes are g, modulo eight)
    const uint32_t s_k = smem_u32(ks) + gq * 128, s_v = smem_u32(vs) + gq * 128 + 4 * t;
    struct Raw {
      uint32_t k[2][D / 32], v[D / 16];               // codes of rows g and g + 8; words of V
      uint32_t kp[2][GROUPS], vp[2][2][GROUPS];       // pairs of rows g and g + 8; of keys 2 t + e + 8 u
    };
    auto load = [&](Raw &x, int from) {
      const uint8_t *at = p.pool + (int64_t)max(from, 0) * H::BYTES;   // (a tile that nobody sees: its pairs become zero)
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        const int j = gq + 8 * h;
        if constexpr (D == 128) {
          *reinterpret_cast<uint4 *>(x.k[h]) = *reinterpret_cast<const uint4 *>(at + j * 64 + t * 16);
          *reinterpret_cast<uint4 *>(x.v + 4 * h) = *reinterpret_cast<const uint4 *>(at + kv4_v_codes(D) + h * 512 + lane * 16);
          *reinterpret_cast<uint2 *>(x.kp[h]) = *reinterpret_cast<const uint2 *>(at + kv4_k_pairs(D) + j * 8);
          *reinterpret_cast<uint4 *>(x.vp[h]) = *reinterpret_cast<const uint4 *>(at + kv4_v_pairs(D) + (2 * t + 8 * h) * 8);
        } else {
          *reinterpret_cast<uint2 *>(x.k[h]) = *reinterpret_cast<const uint2 *>(at + j * 32 + t * 8);
          if (h == 0)
            *reinterpret_cast<uint4 *>(x.v) = *reinterpret_cast<const uint4 *>(at + kv4_v_codes(D) + lane * 16);
          x.kp[h][0] = *reinterpret_cast<const uint32_t *>(at + kv4_k_pairs(D) + j * 4);
          *reinterpret_cast<uint2 *>(x.vp[h]) = *reinterpret_cast<const uint2 *>(at + kv4_v_pairs(D) + (2 * t + 8 * h) * 4);
        }
      }
    };
    bool ok = true;
    uint32_t made = 0;
    Walk walk(plan);
    Segment g;
    while (walk.next(plan, g)) {
      const int most = clamp((long long)g.base + g.first + g.tokens, 0, room);   // keys that any row sees
      const int n = g.b1 - g.b0, tiles = kTiles * n;
      auto source = [&](int i) {   // of this warp's i-th tile: its number in the pool, or -1
        const int q = mw + kMakers * i, x = kTiles * g.b0 + q;
        return q >= tiles || x * kKv4Tile >= most ? -1 : tile_source(p, g.at.s, g.at.slot, x);
      };
      int now = source(lane), next = source(32 + lane);
      Raw raw, ahead;
      uint32_t v[D / 16], vp[2][2][GROUPS];   // of the block before
      bool v_beyond = false;
      uint32_t v_block = 0;
      int v_tile = -1;
      int from, then = __shfl_sync(0xffffffffu, now, 0);
      load(ahead, then);
      for (int i = 0, q = mw; q < tiles || v_tile >= 0; ++i, q += kMakers) {
        const bool more = q < tiles;   // (after the last tile its V is left)
        raw = ahead;
        from = then;
        if (((i + 1) & 31) == 0) {
          now = next;
          next = source(i + 33 + lane);
        }
        then = __shfl_sync(0xffffffffu, now, (i + 1) & 31);
        if (more)
          load(ahead, then);   // (behind the last: tile 0 of the pool, not used)
        const uint32_t block = made + q / kTiles;
        const int tile = q % kTiles, key0 = (g.b0 + q / kTiles) * kKeys + kKv4Tile * tile;
        bool beyond = false;
        if (more) {
          // ---- pairs: those of keys that nobody sees, and those that are not finite, are zero
          uint32_t k_bad = 0, v_bad[GROUPS] = {}, strange = 0;
          auto every = [&](auto f) {   // f(pair, key of the tile, mask of what is bad)
#pragma unroll
            for (int gr = 0; gr < GROUPS; ++gr)
#pragma unroll
              for (int u = 0; u < 2; ++u) {
                f(raw.kp[u][gr], gq + 8 * u, k_bad);
#pragma unroll
                for (int e = 0; e < 2; ++e)
                  f(raw.vp[u][e][gr], 2 * t + e + 8 * u, v_bad[gr]);
              }
          };
          every([&](uint32_t &pair, int, uint32_t &) {   // (8 s beyond f16, or something not finite: x - x is not zero)
            uint32_t x;
            asm("mul.rn.f16x2 %0, %1, %2;" : "=r"(x) : "r"(pair), "r"(0x3c004800u));
            const __half2 y = *reinterpret_cast<const __half2 *>(&x), d = __hsub2(y, y);
            strange |= *reinterpret_cast<const uint32_t *>(&d);
          });
          beyond = __any_sync(0xffffffffu, strange != 0);
          bool any_bad = false;
          if (from < 0 || key0 + kKv4Tile > most || beyond) {
            every([&](uint32_t &pair, int key, uint32_t &bad) {
              const bool seen = from >= 0 && key0 + key < most;
              if (!seen || !finite_pair(pair)) {
                bad |= seen ? 1u << key : 0u;
                pair = 0u;
              }
            });
            k_bad = __reduce_or_sync(0xffffffffu, k_bad);
            uint32_t all = k_bad;
#pragma unroll
            for (int gr = 0; gr < GROUPS; ++gr) {
              v_bad[gr] = __reduce_or_sync(0xffffffffu, v_bad[gr]);
              all |= v_bad[gr];
            }
            any_bad = all != 0;
          }
          // ---- K: words of eight dims of a key
          if (block > 0)
            wait(ok, &bars.s_full[(block - 1) & 1], (block - 1) >> 1, 744);
          Notes &notes = bars.notes[block % kNotes];   // (the block four before is done with)
          auto mid = [](uint32_t pair) {
            const float2 f = halves(pair);
            return fmaf(8.f, f.x, f.y);
          };
#pragma unroll
          for (int gr = 0; gr < GROUPS; ++gr)
#pragma unroll
            for (int u = 0; u < 2; ++u) {
              if (t == 0)
                notes.k_mid[gr][kKv4Tile * tile + gq + 8 * u] = mid(raw.kp[u][gr]);
              if (gq == 0)
                *reinterpret_cast<float2 *>(notes.v_mid[gr] + kKv4Tile * tile + 2 * t + 8 * u) = make_float2(mid(raw.vp[u][0][gr]), mid(raw.vp[u][1][gr]));
            }
          if (lane == 0) {
            const uint32_t hole = from < 0 && key0 < most ? 0xffffu : 0u;
            notes.k_bad[tile] = (uint16_t)k_bad;
            notes.hole[tile] = (uint16_t)hole;
#pragma unroll
            for (int gr = 0; gr < GROUPS; ++gr)
              notes.v_bad[gr][tile] = (uint16_t)v_bad[gr];
            notes.special[tile] = (uint16_t)(any_bad ? 1u : hole);
          }
          const uint32_t k_at = s_k + tile * (kKv4Tile * 128);
          auto make_k = [&](auto held) {
            constexpr bool HELD = decltype(held)::value;
#pragma unroll
            for (int h = 0; h < 2; ++h)
#pragma unroll
              for (int gr = 0; gr < GROUPS; ++gr) {
                const uint32_t s = __byte_perm(raw.kp[h][gr], 0, 0x1010);
#pragma unroll
                for (int w = 0; w < 2; ++w) {
                  const uint32_t x = raw.k[h][2 * gr + w], y = x >> 8, at = k_at + gr * (kKeys * 128) + h * 1024 + (((4 * w + t) ^ gq) << 4);
                  uint32_t high[4], low[4];
                  terms<HELD>(low_codes(x), s, high[0], low[0]);
                  terms<HELD>(high_codes(x), s, high[1], low[1]);
                  terms<HELD>(low_codes(y), s, high[2], low[2]);
                  terms<HELD>(high_codes(y), s, high[3], low[3]);
                  store4(at, high[0], high[1], high[2], high[3]);
                  store4(at + H::TERM, low[0], low[1], low[2], low[3]);
                }
              }
          };
          if (beyond)
            make_k(std::true_type());
          else
            make_k(std::false_type());
          fence_proxy();
          __syncwarp();
          if (lane == 0)
            mbar_arrive(&bars.k_full);
        }
        if (v_tile >= 0) {
          // ---- V of the tile before: words of dims 16 w + g (+ 8) and keys 2 t, 2 t + 1 (+ 8)
          if (v_block > 0)
            wait(ok, &bars.pv_done, v_block - 1, 745);
          const int c = v_tile % 4 * 2;
          const uint32_t v_at = s_v + v_tile / 4 * (D * 128);
          auto make_v = [&](auto held) {
            constexpr bool HELD = decltype(held)::value;
#pragma unroll
            for (int gr = 0; gr < GROUPS; ++gr) {
              const uint32_t s[2] = {__byte_perm(vp[0][0][gr], vp[0][1][gr], 0x5410), __byte_perm(vp[1][0][gr], vp[1][1][gr], 0x5410)};
#pragma unroll
              for (int w = 4 * gr; w < 4 * gr + 4; ++w) {
                const uint32_t x = v[w];
#pragma unroll
                for (int u = 0; u < 2; ++u) {
                  const uint32_t at = v_at + w * 2048 + (((c + u) ^ gq) << 4);
                  uint32_t high, low;
                  terms<HELD>(low_codes(x >> 8 * u), s[u], high, low);
                  store1(at, high);
                  store1(at + H::TERM, low);
                  terms<HELD>(high_codes(x >> 8 * u), s[u], high, low);
                  store1(at + 1024, high);
                  store1(at + 1024 + H::TERM, low);
                }
              }
            }
          };
          if (v_beyond)
            make_v(std::true_type());
          else
            make_v(std::false_type());
          fence_proxy();
          __syncwarp();
          if (lane == 0)
            mbar_arrive(&bars.v_full);
        }
        v_tile = more ? tile : -1;
        v_block = block;
        if (more) {
#pragma unroll
          for (int w = 0; w < D / 16; ++w)
            v[w] = raw.v[w];
#pragma unroll
          for (int u = 0; u < 2; ++u)
#pragma unroll
            for (int e = 0; e < 2; ++e)
#pragma unroll
              for (int gr = 0; gr < GROUPS; ++gr)
                vp[u][e][gr] = raw.vp[u][e][gr];
          v_beyond = beyond;
        }
      }
      made += n;
    }
  } else if (works) {
    // ---- tensor core issue --------------------------------------------------------------------------------------------------------
    uint32_t leader;
    asm volatile("{\n .reg .pred p;\n elect.sync _|p, 0xffffffff;\n selp.u32 %0, 1, 0, p;\n}" : "=r"(leader));
    const uint64_t dq = smem_desc(smem_u32(qs)), dk = smem_desc(smem_u32(ks)), dv = smem_desc(smem_u32(vs));
    bool ok = true;
    uint32_t made = 0, segments = 0;
    // the small products first: terms of the first operand and of the second
    constexpr uint32_t FIRST[3] = {1, 0, 0}, SECOND[3] = {0, 1, 0};
    constexpr int LEAST = TYPE == B200_F32 ? 0 : 1;   // (q of f16 is one term)
    auto scores = [&](uint32_t block) {
      wait(ok, &bars.k_full, block, 746);
      if (!ok)
        return;
      fence_after();
#pragma unroll
      for (int i = LEAST; i < 3; ++i)
#pragma unroll
        for (int k = 0; k < D / 16; ++k)
          mma_ss<kKeys>(leader, tmem + H::COL_S + (block & 1) * kKeys, dq + ((FIRST[i] * H::TERM + (k >> 2) * (kRows * 128) + (k & 3) * 32) >> 4),
                        dk + ((SECOND[i] * H::TERM + (k >> 2) * (kKeys * 128) + (k & 3) * 32) >> 4), (i - LEAST | k) != 0);
      if (leader)
        tc_commit(&bars.s_full[block & 1]);
    };
    Walk walk(plan);
    Segment g;
    while (ok && walk.next(plan, g)) {
      const uint32_t n = g.b1 - g.b0;
      wait(ok, &bars.q_full, segments++, 747);
      if (!ok)
        break;
      scores(made);
      for (uint32_t j = 0; j < n && ok; ++j) {
        const uint32_t block = made + j;
        if (j + 1 < n)
          scores(block + 1);
        wait(ok, &bars.p_ready[block & 1], block >> 1, 748);
        wait(ok, &bars.v_full, block, 750);
        if (!ok)
          break;
        fence_after();
#pragma unroll
        for (int i = 0; i < 3; ++i)
#pragma unroll
          for (int k = 0; k < kKeys / 16; ++k)   // (weights: of 32 keys sixteen columns of each term)
            mma_ts<D>(leader, tmem + H::COL_O, tmem + H::COL_S + (block & 1) * kKeys + (k >> 1) * 32 + FIRST[i] * 16 + (k & 1) * 8,
                      dv + ((SECOND[i] * H::TERM + (k >> 2) * (D * 128) + (k & 3) * 32) >> 4), (i | k) != 0);
        if (leader)
          tc_commit(&bars.pv_done);
      }
      made += n;
    }
  }
  fence_before();
  __syncthreads();
  if (warp == kSoftmaxWarps + kMakers) {
    if (*ab) {   // products of an abandoned block may still be in flight: let them land
      const unsigned long long t0 = now_ns();
      while (now_ns() - t0 < 2000000ull) {
      }
    }
    asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "n"(kCols) : "memory");
  }
}

RaisedOn g_raised[4];
constexpr int kMostSeqs = 800;   // whose plan fits beside the operands

template <int D, int TYPE> int exact_launch(RaisedOn &raised, const Kv4Params &p, cudaStream_t st) {
  if (int rc = raise_shared_limit(raised, (const void *)kv4_exact_kernel<D, TYPE>, Shape<D>::SMEM + RowsPlan::bytes(kMostSeqs)))
    return rc;
  return launch_after(kv4_exact_kernel<D, TYPE>, dim3(kKv4Ctas), kThreads, Shape<D>::SMEM + RowsPlan::bytes(p.a.n_seqs), st, p);
}

} // namespace

bool kv4_exact_takes(int G, int n_seqs) { return G <= kRows && n_seqs <= kMostSeqs; }

int kv4_exact_launch(Kv4Params p, int D, cudaStream_t st) {
  p.heads = p.G;
  p.subs = 1;
  p.tokens = kRows / p.G;
  p.over_heads = (65536 + p.heads - 1) / p.heads;
  if (p.a.dtype == B200_F16)
    return D == 128 ? exact_launch<128, B200_F16>(g_raised[0], p, st) : exact_launch<64, B200_F16>(g_raised[1], p, st);
  return D == 128 ? exact_launch<128, B200_F32>(g_raised[2], p, st) : exact_launch<64, B200_F32>(g_raised[3], p, st);
}

} // namespace b200
