// Attention over the 4-bit KV cache for sequences of many bf16 rows (a chunk of a prompt, or all of it) on the 5th-generation tensor cores.
//
// Where many rows meet a key its 128 codes are better made values once: seven warps turn 128 keys into f16 operands (K [128][D], V
// transposed [D][128], swizzled), two times 128 query rows are multiplied with them.  A code becomes f16 by way of 1024 + c; with its group's scale and
// minimum it meets in one fma, so with one rounding: a value of the cache is a multiple of 2^-24, where f16 ends, and half a step off above 2^-13.
// Only a group of the whole range of f16 can reach beyond it, by its scale's rounding, to 65536: that is held at 65504.
//
// One thread per row does the softmax in one pass: 32 scores at a time come from tensor memory, their weights go back in their place as the A operand of
// O += P V, which stays in tensor memory.  Where a score is more than 2^4 above the row's reference, that moves (by whole powers of two), and
// what has been summed and the block's weights so far are multiplied: rare after a row's first keys.
// Two sets of 128 rows take turns: one's products run under the other's softmax.  (S 2 x 128 columns, O 2 x D.)
// A key's values that are not finite are zero in the operands, and what sees them becomes NaN afterwards: nothing reaches rows that do not.
//
// 1001 rows at 4000 keys, 32 heads on 8 of 128 dims, bf16: 120 us, 479 TFLOP/s, 0.29 of a dense product's rate.  A block of 128 keys takes an SM 7000 clocks,
// 1500 of them for its products: a set's softmax (3400) and the way of its weights through both products (2400) follow each other.  The softmax goes through its scores
// in a loop of 32 at a time: straight code with the next 32 on their way took 4 % longer.
#include "kv4_rows.cuh"

#include <algorithm>
#include <type_traits>

namespace b200 {

namespace {

constexpr int kSets = 2;                            // of kRows
constexpr int kSoftmaxWarps = 4 * kSets, kMakers = 7, kThreads = 32 * (kSoftmaxWarps + kMakers + 1);
constexpr int kStages = 2, kNotes = 4;
constexpr uint32_t kCols = 512;
constexpr int kLeastKeys = 256, kSplit = 1200;

template <int D> struct Shape {
  static constexpr int GROUPS = D / kKv4Group, BYTES = kv4_tile_bytes(D);
  static constexpr uint32_t Q_BYTES = kRows * D * 2, KV_BYTES = kKeys * D * 2;
  static constexpr int PART = rows_part<D, kSets * kRows>();
  static constexpr int SMEM = 1024 + kSets * Q_BYTES + 2 * kStages * KV_BYTES;
  static constexpr uint32_t COL_S = 0, COL_O = kSets * kKeys;
};

// What the softmax has to know of a block's keys.
struct Notes {
  // bits of sixteen keys, by tile: any of the next; K not finite; no page; V not finite, by group
  __align__(16) uint16_t special[8];
  uint16_t k_bad[8], hole[8], v_bad[2][8];
  __device__ __forceinline__ static uint32_t word(const uint16_t *x, int c) { return reinterpret_cast<const uint32_t *>(x)[c]; }   // of keys 32 c ..
};
struct Bars {
  uint64_t k_full[kStages], k_empty[kStages], v_full[kStages], v_empty[kStages], s_full[kSets], p_ready[kSets], o_full[kSets], q_full[kSets];
  uint32_t tmem_base;
  int abort_flag;
  Meeting meeting;
  long long sums[2 * (kThreads / 32) + 1];
  Notes notes[kNotes];
};

// Codes of the low nibble of each byte-pair of w, and of the high one.
__device__ __forceinline__ uint32_t low_codes(uint32_t w) {
  uint32_t x = (w & 0x000f000fu) | 0x64006400u;                        // 1024 + c
  asm("add.rn.f16x2 %0, %0, %1;" : "+r"(x) : "r"(0xe400e400u));
  return x;
}
__device__ __forceinline__ uint32_t high_codes(uint32_t w) { return fma2((w & 0x00f000f0u) | 0x64006400u, 0x2c002c00u, 0xd400d400u); }   // 1024 + 16 c, / 16 - 64
// c s + lo; HELD: within +-65504
template <bool HELD> __device__ __forceinline__ uint32_t value2(uint32_t c, uint32_t s, uint32_t lo) {
  uint32_t x = fma2(c, s, lo);
  if constexpr (HELD) {
    asm("min.f16x2 %0, %0, %1;" : "+r"(x) : "r"(0x7bff7bffu));
    asm("max.f16x2 %0, %0, %1;" : "+r"(x) : "r"(0xfbfffbffu));
  }
  return x;
}

template <int D> __global__ void __launch_bounds__(kThreads, 1) kv4_chunk_kernel(const __grid_constant__ Kv4Params p) {
  using H = Shape<D>;
  constexpr int GROUPS = H::GROUPS, TYPE = B200_BF16;
  extern __shared__ __align__(1024) uint8_t smem[];
  uint8_t *qs = reinterpret_cast<uint8_t *>(((uintptr_t)smem + 1023) & ~(uintptr_t)1023);
  uint8_t *ks = qs + kSets * H::Q_BYTES, *vs = ks + kStages * H::KV_BYTES, *s_plan = vs + kStages * H::KV_BYTES;
  __shared__ Bars bars;
  const int warp = __shfl_sync(0xffffffffu, (int)threadIdx.x >> 5, 0), lane = threadIdx.x & 31;
  volatile int *ab = &bars.abort_flag;
  int *error = p.counters + kKv4Ctas;

  if (threadIdx.x == 0) {
    for (int i = 0; i < kStages; ++i) {
      mbar_init(&bars.k_full[i], kTiles);
      mbar_init(&bars.v_full[i], kTiles);
      mbar_init(&bars.k_empty[i], 1);
      mbar_init(&bars.v_empty[i], 1);
    }
    for (int i = 0; i < kSets; ++i) {
      mbar_init(&bars.s_full[i], 1);
      mbar_init(&bars.o_full[i], 1);
      mbar_init(&bars.p_ready[i], 4);
      mbar_init(&bars.q_full[i], 4);
    }
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
  const int half = p.tokens / kSets;   // positions of a set
  auto wait = [&](bool &ok, uint64_t *bar, uint32_t parity, int code) {   // whole warps leave the poll; who gave up goes on without waiting
    if (ok)
      ok = __all_sync(0xffffffffu, mbar_wait(bar, parity, ab, error, code));
  };

  if (works && warp < kSoftmaxWarps) {
    // ---- softmax: a thread per row --------------------------------------------------------------------------------------------
    const int set = warp >> 2, row = (warp & 3) * 32 + lane;
    const uint32_t lanes = tmem + ((uint32_t)((warp & 3) * 32) << 16), col_s = lanes + H::COL_S + set * kKeys, col_o = lanes + H::COL_O + set * D;
    const uint32_t q_at = smem_u32(qs) + set * H::Q_BYTES + row * 128;
    bool ok = true;
    uint32_t blocks = 0, segments = 0, made = 0;   // of this set so far; of the CTA
    Walk walk(plan);
    Segment g;
    while (walk.next(plan, g)) {
      const int mine = g.tokens - set * half;   // positions of this set
      const bool any = mine > 0;
      const uint32_t n = g.b1 - g.b0;
      float r = kKv4Seed, l = 0.f, factor = 0.f;
      bool far = false;                         // a row of this warp has its reference far from zero
      bool marks[GROUPS] = {};                  // V groups that become NaN
      const int token = row / p.G, seen_by = any && token < min(mine, half) ? clamp((long long)g.base + g.first + set * half + token + 1, 0, room) : 0;
      const bool live = any && token < min(mine, half);
      const int64_t q_row = live ? row_at(p, g.r0 + g.first + set * half, g.at.slot, row, p.a.q_ld, D) : 0;
      if (any) {
        // ---- q: times a power of two, as f16; two elements a word
        uint32_t w[D / 2];
        if (live && p.wide_q16) {
#pragma unroll
          for (int c = 0; c < D / 8; ++c)
            *reinterpret_cast<uint4 *>(w + 4 * c) = *(reinterpret_cast<const uint4 *>((const uint16_t *)p.a.q + q_row) + c);
        } else {
#pragma unroll
          for (int c = 0; c < D / 2; ++c)
            w[c] = live ? ((const uint16_t *)p.a.q)[q_row + 2 * c] | (uint32_t)((const uint16_t *)p.a.q)[q_row + 2 * c + 1] << 16 : 0u;
        }
        auto two = [](uint32_t x) { return make_float2(__uint_as_float(x << 16), __uint_as_float(x & 0xffff0000u)); };
        float most = 0.f, sum = 0.f;
#pragma unroll
        for (int c = 0; c < D / 2; ++c) {
          const float2 x = two(w[c]);
          most = max3(most, fabsf(x.x), fabsf(x.y));
          sum = fmaf(x.x, 0.f, fmaf(x.y, 0.f, sum));   // (NaN where one is not finite)
        }
        const int up = min(max(14 + 127 - (int)(__float_as_uint(most) >> 23), -113), 100);
        const float by = p.log2_scale < 0.f ? -power(up) : power(up);
        factor = sum == 0.f ? fabsf(p.log2_scale) * power(-up) : NAN;
#pragma unroll
        for (int c = 0; c < D / 8; ++c) {
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            const float2 x = two(w[4 * c + e]);
            w[4 * c + e] = pack_f16(x.x * by, x.y * by);
          }
          store4(q_at + (c >> 3) * (kRows * 128) + (((c & 7) ^ (row & 7)) << 4), w[4 * c], w[4 * c + 1], w[4 * c + 2], w[4 * c + 3]);
        }
        fence_proxy();
        fence_before();
        __syncwarp();
        if (lane == 0)
          mbar_arrive(&bars.q_full[set]);
      }
      for (uint32_t j = 0; any && j < n; ++j) {
        const int key0 = (g.b0 + j) * kKeys, seen = min(max(seen_by - key0, 0), kKeys);   // keys of the block that this row sees
        wait(ok, &bars.s_full[set], blocks & 1, 731);
        ++blocks;
        fence_after();
        // (the makers wrote them before the products that have been waited for could begin; another block's come four blocks later)
        const Notes &notes = bars.notes[(made + j) % kNotes];
        const uint4 any_special = *reinterpret_cast<const uint4 *>(notes.special);
        const bool special = (any_special.x | any_special.y | any_special.z | any_special.w) != 0;
        const bool masked = special || __any_sync(0xffffffffu, live && seen < kKeys);
        auto sees = [&](int c) {   // of keys 32 c ..: a bit each
          const int k = seen - 32 * c;
          return (k >= 32 ? 0xffffffffu : k <= 0 ? 0u : (1u << k) - 1) & ~Notes::word(notes.hole, c);
        };
        // a row's reference moves, at the keys 32 c and on
        auto move = [&](float top, int c) {
          const float to = kv4_moves(top, r) ? kv4_reference(ceilf(top)) : r, keep = ex2(r - to);   // (each row for itself)
          r = to;
          far = __any_sync(0xffffffffu, fabsf(r) >= kKv4Far / 2 && r != kKv4Seed);
          l *= keep;
          auto times = [&](uint32_t at, bool pairs) {
            uint32_t w[32];
            tmem_load32(at, w);
            tmem_arrived(w);
#pragma unroll
            for (int e = 0; e < 32; ++e)
              if (pairs) {
                const float2 x = halves(w[e]);
                w[e] = pack_f16(x.x * keep, x.y * keep);
              } else {
                w[e] = __float_as_uint(__uint_as_float(w[e]) * keep);
              }
            tmem_store32(at, w);
          };
          if (j > 0)   // (the sums so far are complete: their products came before the scores)
#pragma unroll 1
            for (int i = 0; i < D; i += 32)
              times(col_o + i, false);
          if (c > 0) {
            tmem_wait_store();
            // weights of this block; where they end in the middle of 32 columns, scores that are used no more
            times(col_s, true);
            if (c == 3)
              times(col_s + 32, true);
            tmem_wait_store();
          }
        };
        auto weigh = [&](auto hidden) {
          constexpr bool HIDDEN = decltype(hidden)::value;
#pragma unroll 1
          for (int c = 0; c < 4; ++c) {
            uint32_t w[32];
            tmem_load32(col_s + 32 * c, w);
            tmem_arrived(w);
            const uint32_t m = HIDDEN ? sees(c) : 0u, bad = HIDDEN ? Notes::word(notes.k_bad, c) & m : 0u;
            float x[4] = {-INFINITY, -INFINITY, -INFINITY, -INFINITY};
#pragma unroll
            for (int k = 0; k < 32; k += 2) {
              if constexpr (HIDDEN) {
                w[k] = m >> k & 1 ? w[k] : 0xff800000u;
                w[k + 1] = m >> (k + 1) & 1 ? w[k + 1] : 0xff800000u;
              }
              x[k / 2 & 3] = max3(x[k / 2 & 3], __uint_as_float(w[k]), __uint_as_float(w[k + 1]));
            }
            const float top = fmaxf(max3(x[0], x[1], x[2]), x[3]) * factor;
            if (__any_sync(0xffffffffu, kv4_moves(top, r)))
              move(top, c);
            // Scores less the reference are one fma each.  Far out its exact product and the rounded one that made the reference are steps of f32 apart, and
            // those are whole powers of two of a weight: scores are rounded first.
            float by = factor;
            if (far) {
#pragma unroll
              for (int k = 0; k < 32; ++k)
                w[k] = __float_as_uint(__uint_as_float(w[k]) * factor);
              by = 1.f;
            }
            uint32_t out[16];
            const uint64_t ff = pack2(by, by), rr = pack2(-r, -r);
            uint64_t sum[2] = {};
#pragma unroll
            for (int k = 0; k < 32; k += 2) {
              float2 x = unpack2(fma_2(pack2(__uint_as_float(w[k]), __uint_as_float(w[k + 1])), ff, rr));
              x.x = ex2(x.x);
              x.y = ex2(x.y);
              if constexpr (HIDDEN) {
                x.x = bad >> k & 1 ? NAN : m >> k & 1 ? x.x : 0.f;
                x.y = bad >> (k + 1) & 1 ? NAN : m >> (k + 1) & 1 ? x.y : 0.f;
              }
              sum[k / 2 & 1] = add_2(sum[k / 2 & 1], pack2(x.x, x.y));
              out[k / 2] = pack_f16(x.x, x.y);
            }
            const float2 both = unpack2(add_2(sum[0], sum[1]));
            l += both.x + both.y;
            tmem_store16(col_s + 16 * c, out);
            if constexpr (HIDDEN)
#pragma unroll
              for (int gr = 0; gr < GROUPS; ++gr)
                marks[gr] = marks[gr] || (Notes::word(notes.v_bad[gr], c) & m) != 0;
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
          mbar_arrive(&bars.p_ready[set]);
      }
      made += n;
      // ---- the rows' sums: out, or a part ------------------------------------------------------------------------------------------
      const bool whole = g.b0 == 0 && g.b1 == g.all;
      float *part = p.parts + ((int64_t)blockIdx.x * 2 + (g.b0 == 0)) * H::PART;
      const int at = set * kRows + row;
      const int64_t to = live ? row_at(p, g.r0 + g.first + set * half, g.at.slot, row, p.a.out_ld, D) : 0;
      if (any) {
        wait(ok, &bars.o_full[set], segments & 1, 732);
        ++segments;
        fence_after();
#pragma unroll 1
        for (int c = 0; c < D; c += 32) {
          uint32_t w[32];
          tmem_load32(col_o + c, w);
          tmem_arrived(w);
          if (live) {
#pragma unroll
            for (int e = 0; e < 32; e += 4) {
              const float o[4] = {__uint_as_float(w[e]), __uint_as_float(w[e + 1]), __uint_as_float(w[e + 2]), __uint_as_float(w[e + 3])};
              if (whole)
                put_over<TYPE>(p, to + c + e, o, l, marks[(c + e) / kKv4Group]);
              else
                __stcg(reinterpret_cast<float4 *>(part) + (c + e) / 4 * (kSets * kRows) + at, make_float4(o[0], o[1], o[2], o[3]));
            }
          }
        }
        fence_before();
        if (live && !whole) {
          float *rest = part + kSets * kRows * D;
          rest[at] = r;
          rest[kSets * kRows + at] = l;
#pragma unroll
          for (int gr = 0; gr < GROUPS; ++gr)
            rest[(2 + gr) * kSets * kRows + at] = marks[gr] ? 1.f : 0.f;
        }
      }
      if (!whole)
        meet<D, TYPE, kSets * kRows, 32 * kSoftmaxWarps>(p, plan, g, bars.meeting, at, live, to);
    }
  } else if (works && warp < kSoftmaxWarps + kMakers) {
    // ---- makers: every seventh tile each -------------------------------------------------------------------------------------------
    const int mw = warp - kSoftmaxWarps, gq = lane >> 2, t = lane & 3;
    const uint32_t s_k = smem_u32(ks) + gq * 128, s_v = smem_u32(vs) + gq * 128 + 4 * t;
    struct Raw {
      uint32_t k[2][D / 32], v[D / 16];               // codes of rows g and g + 8; words of V
      uint32_t kp[2][GROUPS], vp[2][2][GROUPS];       // pairs of rows g and g + 8; of keys 2 t + e + 8 u
    };
    auto load = [&](Raw &x, int from) {
      const uint8_t *tile = p.pool + (int64_t)max(from, 0) * H::BYTES;   // (a tile that nobody sees: its pairs become zero)
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        const int j = gq + 8 * h;
        if constexpr (D == 128) {
          *reinterpret_cast<uint4 *>(x.k[h]) = *reinterpret_cast<const uint4 *>(tile + j * 64 + t * 16);
          *reinterpret_cast<uint4 *>(x.v + 4 * h) = *reinterpret_cast<const uint4 *>(tile + kv4_v_codes(D) + h * 512 + lane * 16);
          *reinterpret_cast<uint2 *>(x.kp[h]) = *reinterpret_cast<const uint2 *>(tile + kv4_k_pairs(D) + j * 8);
          *reinterpret_cast<uint4 *>(x.vp[h]) = *reinterpret_cast<const uint4 *>(tile + kv4_v_pairs(D) + (2 * t + 8 * h) * 8);
        } else {
          *reinterpret_cast<uint2 *>(x.k[h]) = *reinterpret_cast<const uint2 *>(tile + j * 32 + t * 8);
          if (h == 0)
            *reinterpret_cast<uint4 *>(x.v) = *reinterpret_cast<const uint4 *>(tile + kv4_v_codes(D) + lane * 16);
          x.kp[h][0] = *reinterpret_cast<const uint32_t *>(tile + kv4_k_pairs(D) + j * 4);
          *reinterpret_cast<uint2 *>(x.vp[h]) = *reinterpret_cast<const uint2 *>(tile + kv4_v_pairs(D) + (2 * t + 8 * h) * 4);
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
        const int q = mw + kMakers * i, tile = kTiles * g.b0 + q;
        return q >= tiles || tile * kKv4Tile >= most ? -1 : tile_source(p, g.at.s, g.at.slot, tile);
      };
      int now = source(lane), next = source(32 + lane);
      Raw raw, ahead;
      int from, then = __shfl_sync(0xffffffffu, now, 0);
      load(ahead, then);
      for (int i = 0, q = mw; q < tiles; ++i, q += kMakers) {
        raw = ahead;
        from = then;
        if (((i + 1) & 31) == 0) {
          now = next;
          next = source(i + 33 + lane);
        }
        then = __shfl_sync(0xffffffffu, now, (i + 1) & 31);
        load(ahead, then);
        const uint32_t block = made + q / kTiles, stage = block % kStages;
        const int tile = q % kTiles, key0 = (g.b0 + q / kTiles) * kKeys + kKv4Tile * tile;
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
#pragma unroll
        for (int gr = 0; gr < GROUPS; ++gr) {   // (the value of code 15, beyond f16 or nothing finite: x - x is not zero)
          const uint32_t at[3][2] = {{raw.kp[0][gr], raw.kp[1][gr]}, {raw.vp[0][0][gr], raw.vp[0][1][gr]}, {raw.vp[1][0][gr], raw.vp[1][1][gr]}};
#pragma unroll
          for (int i = 0; i < 3; ++i) {
            const uint32_t top = fma2(0x4b804b80u, __byte_perm(at[i][0], at[i][1], 0x5410), __byte_perm(at[i][0], at[i][1], 0x7632));
            const __half2 x = *reinterpret_cast<const __half2 *>(&top), d = __hsub2(x, x);
            strange |= *reinterpret_cast<const uint32_t *>(&d);
          }
        }
        const bool beyond = __any_sync(0xffffffffu, strange != 0);
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
        if (block >= kStages)
          wait(ok, &bars.k_empty[stage], (block / kStages - 1) & 1, 733);
        if (lane == 0) {   // (after the wait: the block four before is done with)
          Notes &notes = bars.notes[block % kNotes];
          const uint32_t hole = from < 0 && key0 < most ? 0xffffu : 0u;
          notes.k_bad[tile] = (uint16_t)k_bad;
          notes.hole[tile] = (uint16_t)hole;
#pragma unroll
          for (int gr = 0; gr < GROUPS; ++gr)
            notes.v_bad[gr][tile] = (uint16_t)v_bad[gr];
          notes.special[tile] = (uint16_t)(any_bad ? 1u : hole);
        }
        // (rows of K and of V^T that a lane writes are g, modulo eight)
        const uint32_t k_at = s_k + stage * H::KV_BYTES + tile * (kKv4Tile * 128), v_at = s_v + stage * H::KV_BYTES + tile / 4 * (D * 128);
        auto make_k = [&](auto held) {
#pragma unroll
          for (int h = 0; h < 2; ++h)
#pragma unroll
            for (int gr = 0; gr < GROUPS; ++gr) {
              const uint32_t s = __byte_perm(raw.kp[h][gr], 0, 0x1010), lo = __byte_perm(raw.kp[h][gr], 0, 0x3232);
#pragma unroll
              for (int w = 0; w < 2; ++w) {
                const uint32_t x = raw.k[h][2 * gr + w], y = x >> 8;
                constexpr bool HELD = decltype(held)::value;
                store4(k_at + gr * (kKeys * 128) + h * 1024 + (((4 * w + t) ^ gq) << 4), value2<HELD>(low_codes(x), s, lo), value2<HELD>(high_codes(x), s, lo),
                       value2<HELD>(low_codes(y), s, lo), value2<HELD>(high_codes(y), s, lo));
              }
            }
        };
        if (beyond)
          make_k(std::true_type());
        else
          make_k(std::false_type());
        // ---- V: words of dims 16 w + g (+ 8) and keys 2 t, 2 t + 1 (+ 8)
        if (block >= kStages)
          wait(ok, &bars.v_empty[stage], (block / kStages - 1) & 1, 734);
        const int c = tile % 4 * 2;
        auto make_v = [&](auto held) {
          constexpr bool HELD = decltype(held)::value;
#pragma unroll
          for (int gr = 0; gr < GROUPS; ++gr) {
            uint32_t s[2], lo[2];
#pragma unroll
            for (int u = 0; u < 2; ++u) {
              s[u] = __byte_perm(raw.vp[u][0][gr], raw.vp[u][1][gr], 0x5410);
              lo[u] = __byte_perm(raw.vp[u][0][gr], raw.vp[u][1][gr], 0x7632);
            }
#pragma unroll
            for (int w = 4 * gr; w < 4 * gr + 4; ++w) {
              const uint32_t x = raw.v[w], y = x >> 8;
              const uint32_t to0 = v_at + w * 2048 + ((c ^ gq) << 4), to1 = v_at + w * 2048 + (((c + 1) ^ gq) << 4);
              store1(to0, value2<HELD>(low_codes(x), s[0], lo[0]));
              store1(to0 + 1024, value2<HELD>(high_codes(x), s[0], lo[0]));
              store1(to1, value2<HELD>(low_codes(y), s[1], lo[1]));
              store1(to1 + 1024, value2<HELD>(high_codes(y), s[1], lo[1]));
            }
          }
        };
        if (beyond)
          make_v(std::true_type());
        else
          make_v(std::false_type());
        fence_proxy();
        __syncwarp();
        if (lane == 0) {
          mbar_arrive(&bars.k_full[stage]);
          mbar_arrive(&bars.v_full[stage]);
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
    uint32_t made = 0, ready[kSets] = {}, segments[kSets] = {};
    auto scores = [&](int set, uint32_t block) {
#pragma unroll
      for (int k = 0; k < D / 16; ++k)
        mma_ss<kKeys>(leader, tmem + H::COL_S + set * kKeys, dq + ((set * H::Q_BYTES + (k >> 2) * (kRows * 128) + (k & 3) * 32) >> 4),
                      dk + ((block % kStages * H::KV_BYTES + (k >> 2) * (kKeys * 128) + (k & 3) * 32) >> 4), k != 0);
      if (leader)
        tc_commit(&bars.s_full[set]);
    };
    auto keys_ready = [&](uint32_t block) {
      wait(ok, &bars.k_full[block % kStages], (block / kStages) & 1, 735);
      fence_after();
    };
    Walk walk(plan);
    Segment g;
    while (ok && walk.next(plan, g)) {
      const int sets = g.tokens > half ? 2 : 1;
      const uint32_t n = g.b1 - g.b0;
      for (int set = 0; set < sets; ++set)
        wait(ok, &bars.q_full[set], segments[set]++ & 1, 736);
      keys_ready(made);
      if (!ok)
        break;
      for (int set = 0; set < sets; ++set)
        scores(set, made);
      if (leader)
        tc_commit(&bars.k_empty[made % kStages]);
      for (uint32_t j = 0; j < n && ok; ++j) {
        const uint32_t block = made + j;
#pragma unroll
        for (int set = 0; set < kSets; ++set) {
          if (set >= sets)
            break;
          wait(ok, &bars.p_ready[set], ready[set]++ & 1, 737);
          if (set == 0)
            wait(ok, &bars.v_full[block % kStages], (block / kStages) & 1, 738);
          if (!ok)
            break;
          fence_after();
#pragma unroll
          for (int k = 0; k < kKeys / 16; ++k)
            mma_ts<D>(leader, tmem + H::COL_O + set * D, tmem + H::COL_S + set * kKeys + k * 8,
                      dv + ((block % kStages * H::KV_BYTES + (k >> 2) * (D * 128) + (k & 3) * 32) >> 4), (j | k) != 0);
          if (j + 1 < n) {
            if (set == 0)
              keys_ready(block + 1);
            if (!ok)
              break;
            scores(set, block + 1);
          } else if (leader) {
            tc_commit(&bars.o_full[set]);
          }
        }
        if (ok && leader) {
          tc_commit(&bars.v_empty[block % kStages]);
          if (j + 1 < n)
            tc_commit(&bars.k_empty[(block + 1) % kStages]);
        }
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

RaisedOn g_raised[2];
constexpr int kMostSeqs = 1500;   // whose plan fits beside the operands

template <int D> int chunk_launch(RaisedOn &raised, const Kv4Params &p, cudaStream_t st) {
  if (int rc = raise_shared_limit(raised, (const void *)kv4_chunk_kernel<D>, Shape<D>::SMEM + RowsPlan::bytes(kMostSeqs)))
    return rc;
  return launch_after(kv4_chunk_kernel<D>, dim3(kKv4Ctas), kThreads, Shape<D>::SMEM + RowsPlan::bytes(p.a.n_seqs), st, p);
}

} // namespace

int64_t kv4_chunk_part_floats(int D) { return 2 * (D == 128 ? Shape<128>::PART : Shape<64>::PART); }

bool kv4_chunk_takes(int G, int n_seqs) { return G <= kRows && n_seqs <= kMostSeqs; }

int kv4_chunk_launch(Kv4Params p, int D, cudaStream_t st) {
  p.heads = p.G;
  p.subs = 1;
  p.tokens = kSets * (kRows / p.G);
  p.over_heads = (65536 + p.heads - 1) / p.heads;
  return D == 128 ? chunk_launch<128>(g_raised[0], p, st) : chunk_launch<64>(g_raised[1], p, st);
}

} // namespace b200
