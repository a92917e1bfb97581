// Attention over the 4-bit KV cache for sequences of many rows (a chunk of a prompt, or all of it) on the 5th-generation tensor cores.
//
// Where many rows meet a key its 128 codes are better made values once: four warps turn 128 keys into f16 operands (K [128][D], V
// transposed [D][128], swizzled), two times 128 query rows are multiplied with them.  A tile of sixteen keys has a power of two of its own, so
// that its largest value comes to 2^-8 .. 2^-7: code, scale and minimum then meet in one fma with one rounding (codes as the subnormal
// numbers c 2^-24 and c 2^-20, the scale times 2^24 and 2^20).  K's power goes into the scores' factor, V's into the weights' exponent, whose reference
// counts it too: weights fit f16 whatever the values are, and need no other normalisation.
//
// One thread per row does the softmax: scores come from tensor memory twice (their maximum, then the weights), the weights go back in their
// place as the A operand of O += P V, which stays in tensor memory; it is multiplied only when a row's reference moves by more than 2^4.
// Two sets of 128 rows take turns: one's products run under the other's softmax.  (S 2 x 128 columns, O 2 x D.)
// A key's values that are not finite are zero in the operands, and what sees them becomes NaN afterwards: nothing reaches rows that do not.
#include "kv4_plan.cuh"
#include "tensor_core.cuh"

#include <algorithm>

namespace b200 {

namespace {

constexpr int kRows = 128, kSets = 2;               // query rows of a set
constexpr int kKeys = 128, kShift = 7;              // of a block
constexpr int kSoftmaxWarps = 4 * kSets, kMakers = 4, kThreads = 32 * (kSoftmaxWarps + kMakers + 1);
constexpr int kStages = 2, kNotes = 4;
constexpr uint32_t kCols = 512;
constexpr int kLeastKeys = 256;

template <int D> struct Shape {
  static constexpr int GROUPS = D / kKv4Group, BYTES = kv4_tile_bytes(D);
  static constexpr uint32_t Q_BYTES = kRows * D * 2, KV_BYTES = kKeys * D * 2;
  static constexpr int PART = kSets * kRows * (D + 2 + GROUPS);   // floats: sums [D / 4][rows][4], references, totals, marks
  static constexpr int SMEM = 1024 + kSets * Q_BYTES + 2 * kStages * KV_BYTES;
  static constexpr uint32_t COL_S = 0, COL_O = kSets * kKeys;
};

// What the softmax has to know of a block's keys.
struct Notes {
  float factor[8], height[8], unit[8];   // of a tile: of its scores; log2 of V's power of two, and that itself (inverted)
  uint32_t special[4];                   // any of the words below
  uint32_t k_bad[4], hole[4], v_bad[2][4];   // keys: K not finite; no page; V not finite, by group
};
struct Bars {
  uint64_t k_full[kStages], k_empty[kStages], v_full[kStages], v_empty[kStages], s_full[kSets], p_ready[kSets], o_full[kSets], q_full[kSets];
  uint32_t tmem_base;
  int abort_flag, last, from, to;
  long long sums[kThreads / 32];
  Notes notes[kNotes];
};

// kind::f16 instruction descriptor: D = f32, A = B = f16, both K-major, M = 128.
template <int N> __host__ __device__ constexpr uint32_t idesc() {
  return (1u << 4) | ((uint32_t)(N >> 3) << 17) | ((uint32_t)(kRows >> 4) << 24);
}
// Executed by a whole warp in uniform control flow, issued by the lane whose `leader` is set.
template <int N> __device__ __forceinline__ void mma_ss(uint32_t leader, uint32_t d, uint64_t a, uint64_t b, uint32_t accumulate) {
  asm volatile(
      "{\n .reg .pred p, l;\n setp.ne.b32 p, %4, 0;\n setp.ne.b32 l, %5, 0;\n"
      " @l tcgen05.mma.cta_group::1.kind::f16 [%0], %1, %2, %3, p;\n}" ::"r"(d),
      "l"(a), "l"(b), "r"(idesc<N>()), "r"(accumulate), "r"(leader)
      : "memory");
}
template <int N> __device__ __forceinline__ void mma_ts(uint32_t leader, uint32_t d, uint32_t a, uint64_t b, uint32_t accumulate) {
  asm volatile(
      "{\n .reg .pred p, l;\n setp.ne.b32 p, %4, 0;\n setp.ne.b32 l, %5, 0;\n"
      " @l tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], %2, %3, p;\n}" ::"r"(d),
      "r"(a), "l"(b), "r"(idesc<N>()), "r"(accumulate), "r"(leader)
      : "memory");
}
__device__ __forceinline__ void tmem_store32(uint32_t addr, const uint32_t (&v)[32]) {
  asm volatile("tcgen05.st.sync.aligned.32x32b.x32.b32 [%0], {%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16,%17,%18,%19,%20,%21,%22,%23,%24,%25,"
               "%26,%27,%28,%29,%30,%31,%32};" ::"r"(addr),
               "r"(v[0]), "r"(v[1]), "r"(v[2]), "r"(v[3]), "r"(v[4]), "r"(v[5]), "r"(v[6]), "r"(v[7]), "r"(v[8]), "r"(v[9]), "r"(v[10]), "r"(v[11]), "r"(v[12]),
               "r"(v[13]), "r"(v[14]), "r"(v[15]), "r"(v[16]), "r"(v[17]), "r"(v[18]), "r"(v[19]), "r"(v[20]), "r"(v[21]), "r"(v[22]), "r"(v[23]), "r"(v[24]),
               "r"(v[25]), "r"(v[26]), "r"(v[27]), "r"(v[28]), "r"(v[29]), "r"(v[30]), "r"(v[31])
               : "memory");
}
__device__ __forceinline__ void tmem_wait_store() { asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory"); }
__device__ __forceinline__ void fence_before() { asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory"); }
__device__ __forceinline__ void fence_after() { asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory"); }
__device__ __forceinline__ void fence_proxy() { asm volatile("fence.proxy.async.shared::cta;" ::: "memory"); }
// byte offset of 16-byte chunk c of row r in a tile of 128-byte rows, 128-byte swizzle
__device__ __forceinline__ uint32_t swz(int r, int c) { return (uint32_t)(r * 128 + ((c ^ (r & 7)) << 4)); }
__device__ __forceinline__ uint32_t fma2(uint32_t a, uint32_t b, uint32_t c) {
  uint32_t r;
  asm("fma.rn.f16x2 %0, %1, %2, %3;" : "=r"(r) : "r"(a), "r"(b), "r"(c));
  return r;
}
__device__ __forceinline__ bool finite_pair(uint32_t pair) { return (pair & 0x7c00u) != 0x7c00u && (pair & 0x7c000000u) != 0x7c000000u; }
__device__ __forceinline__ float power(int e) { return __uint_as_float((uint32_t)(127 + e) << 23); }
// of a tile's largest value: the power of two that brings it to 2^-8 .. 2^-7
__device__ __forceinline__ int lift(float largest) { return min(max(119 - (int)(__float_as_uint(largest) >> 23), -40), 40); }

// A CTA's share of an item: blocks b0 .. b1 - 1 of `all`.
struct Segment {
  Place at;
  int b0, b1, all;
  int first, tokens;      // the item's positions
  int base;               // of the sequence
  int r0;
};
// The segments of a CTA, in order; every role walks them by itself.
struct Walk {
  Place at, stop;
  bool over;
  __device__ __forceinline__ Walk(const KeyPlan<kShift> &plan) {
    const int lane = threadIdx.x & 31;
    const long long x = plan.border(blockIdx.x + min(lane, 1));
    over = __shfl_sync(0xffffffffu, x, 0) == __shfl_sync(0xffffffffu, x, 1);
    at = Place{plan.n, 0, 0, 0};
    if (x < plan.total) {
      long long begin, end;
      plan.locate(x, at, begin, end);
    }
    stop.s = __shfl_sync(0xffffffffu, at.s, 1);
    stop.slot = __shfl_sync(0xffffffffu, at.slot, 1);
    stop.rt = __shfl_sync(0xffffffffu, at.rt, 1);
    stop.tile = __shfl_sync(0xffffffffu, at.tile, 1);
    at.s = __shfl_sync(0xffffffffu, at.s, 0);
    at.slot = __shfl_sync(0xffffffffu, at.slot, 0);
    at.rt = __shfl_sync(0xffffffffu, at.rt, 0);
    at.tile = __shfl_sync(0xffffffffu, at.tile, 0);
  }
  __device__ __forceinline__ bool next(const KeyPlan<kShift> &plan, Segment &g) {
    while (!over && at.s < plan.n) {
      const Sequence q = plan.sequence(at.s);
      g.all = plan.item_tiles(q, at.rt);
      if (at.tile >= g.all) {
        plan.next_item(at, q);
        continue;
      }
      const bool here = stop.s == at.s && stop.slot == at.slot && stop.rt == at.rt;
      g.at = at;
      g.b0 = at.tile;
      g.b1 = here ? min(stop.tile, g.all) : g.all;
      g.first = at.rt * plan.tokens;
      g.tokens = min(plan.tokens, q.n - g.first);
      g.base = q.base;
      g.r0 = q.r0;
      over = here;
      if (!here)
        plan.next_item(at, q);
      return g.b0 < g.b1;
    }
    return false;
  }
};

template <int D, int TYPE> __global__ void __launch_bounds__(kThreads, 1) kv4_chunk_kernel(const __grid_constant__ Kv4Params p) {
  using H = Shape<D>;
  constexpr int GROUPS = H::GROUPS;
  extern __shared__ __align__(1024) uint8_t smem[];
  uint8_t *qs = reinterpret_cast<uint8_t *>(((uintptr_t)smem + 1023) & ~(uintptr_t)1023);
  uint8_t *ks = qs + kSets * H::Q_BYTES, *vs = ks + kStages * H::KV_BYTES, *s_plan = vs + kStages * H::KV_BYTES;
  __shared__ Bars bars;
  const int warp = __shfl_sync(0xffffffffu, (int)threadIdx.x >> 5, 0), lane = threadIdx.x & 31;
  volatile int *ab = &bars.abort_flag;
  int *error = p.counters + kKv4Ctas;

  if (threadIdx.x == 0) {
    for (int i = 0; i < kStages; ++i) {
      mbar_init(&bars.k_full[i], kMakers);
      mbar_init(&bars.v_full[i], kMakers);
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
  KeyPlan<kShift> plan;
  plan.build<kThreads>(p, s_plan, bars.sums, kLeastKeys);
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
    uint8_t *q_at = qs + set * H::Q_BYTES;
    bool ok = true;
    uint32_t blocks = 0, segments = 0, made = 0;   // of this set so far; of the CTA
    Walk walk(plan);
    Segment g;
    while (walk.next(plan, g)) {
      const int mine = g.tokens - set * half;   // positions of this set
      const bool any = mine > 0;
      const uint32_t n = g.b1 - g.b0;
      float r = kKv4Seed, l = 0.f, factor = 0.f;
      bool marks[GROUPS] = {};                  // V groups that become NaN
      const int token = row / p.G, seen_by = any && token < min(mine, half) ? clamp((long long)g.base + g.first + set * half + token + 1, 0, room) : 0;
      const bool live = any && token < min(mine, half);
      const int64_t q_row = live ? row_at(p, g.r0 + g.first + set * half, g.at.slot, row, p.a.q_ld, D) : 0;
      if (any) {
        // ---- q: times a power of two, as f16
        float x[4], most = 0.f, sum = 0.f;
        auto load = [&](int d) {
          if (live && p.wide_q)
            load_wide<TYPE>(p.a.q, q_row + d, x);
          else
#pragma unroll
            for (int e = 0; e < 4; ++e)
              x[e] = live ? load_as_float(p.a.q, TYPE, q_row + d + e) : 0.f;
        };
#pragma unroll 4
        for (int d = 0; d < D; d += 4) {
          load(d);
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            most = fmaxf(most, fabsf(x[e]));
            sum += x[e] * 0.f;               // (NaN where one is not finite)
          }
        }
        const int up = min(max(14 + 127 - (int)(__float_as_uint(most) >> 23), -113), 100);
        const float by = p.log2_scale < 0.f ? -power(up) : power(up);
        factor = sum == 0.f ? fabsf(p.log2_scale) * power(-up) : NAN;
#pragma unroll 4
        for (int c = 0; c < D / 8; ++c) {
          uint32_t w[4];
#pragma unroll
          for (int h = 0; h < 2; ++h) {
            load(8 * c + 4 * h);
            w[2 * h] = pack_f16(x[0] * by, x[1] * by);
            w[2 * h + 1] = pack_f16(x[2] * by, x[3] * by);
          }
          *reinterpret_cast<uint4 *>(q_at + (c >> 3) * (kRows * 128) + swz(row, c & 7)) = make_uint4(w[0], w[1], w[2], w[3]);
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
        const bool special = (notes.special[0] | notes.special[1] | notes.special[2] | notes.special[3]) != 0;
        const bool masked = special || __any_sync(0xffffffffu, live && seen < kKeys);
        auto sees = [&](int c) {   // of keys 32 c ..: a bit each
          const int k = seen - 32 * c;
          return (k >= 32 ? 0xffffffffu : k <= 0 ? 0u : (1u << k) - 1) & ~notes.hole[c];
        };
        float top = -INFINITY;
        // ---- the largest of score + log2 of V's power
#pragma unroll
        for (int c = 0; c < 4; ++c) {
          uint32_t w[32];
          tmem_load32(col_s + 32 * c, w);
          tmem_wait_load();
          if (masked) {
            const uint32_t m = sees(c);
#pragma unroll
            for (int e = 0; e < 32; ++e)
              w[e] = m >> e & 1 ? w[e] : 0xff800000u;
          }
#pragma unroll
          for (int h = 0; h < 2; ++h) {
            float x = __uint_as_float(w[16 * h]);
#pragma unroll
            for (int e = 1; e < 16; ++e)
              x = fmaxf(x, __uint_as_float(w[16 * h + e]));
            top = fmaxf(top, fmaf(x, factor * notes.factor[2 * c + h], notes.height[2 * c + h]));
          }
        }
        const bool moves = top > r + (kKv4Top + kKv4Lag);
        if (__any_sync(0xffffffffu, moves)) {
          const float to = moves ? top - kKv4Top : r, keep = ex2(r - to);   // (each row for itself)
          r = to;
          l *= keep;
          if (j > 0) {   // (the sums so far are complete: their products came before the scores)
#pragma unroll 1
            for (int c = 0; c < D; c += 32) {
              uint32_t w[32];
              tmem_load32(col_o + c, w);
              tmem_wait_load();
#pragma unroll
              for (int e = 0; e < 32; ++e)
                w[e] = __float_as_uint(__uint_as_float(w[e]) * keep);
              tmem_store32(col_o + c, w);
            }
          }
        }
        // ---- weights, in place of the scores
#pragma unroll
        for (int c = 0; c < 4; ++c) {
          uint32_t w[32], out[16];
          tmem_load32(col_s + 32 * c, w);
          tmem_wait_load();
          const uint32_t m = masked ? sees(c) : 0xffffffffu, bad = masked ? notes.k_bad[c] & m : 0u;
#pragma unroll
          for (int h = 0; h < 2; ++h) {
            const float f = factor * notes.factor[2 * c + h], b = notes.height[2 * c + h] - r;
            float sum[2] = {};
#pragma unroll
            for (int e = 0; e < 16; e += 2) {
              float x[2];
#pragma unroll
              for (int u = 0; u < 2; ++u) {
                const int k = 16 * h + e + u;
                x[u] = ex2(fmaf(__uint_as_float(w[k]), f, b));
                if (masked)
                  x[u] = bad >> k & 1 ? NAN : m >> k & 1 ? x[u] : 0.f;
                sum[u] += x[u];
              }
              out[8 * h + e / 2] = pack_f16(x[0], x[1]);
            }
            l = fmaf(sum[0] + sum[1], notes.unit[2 * c + h], l);
          }
          tmem_store16(col_s + 16 * c, out);
          if (special)
#pragma unroll
            for (int gr = 0; gr < GROUPS; ++gr)
              marks[gr] = marks[gr] || (notes.v_bad[gr][c] & m) != 0;
        }
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
      auto write_out = [&](int d, const float (&o)[4], float total, const bool (&nan)[GROUPS]) {
        const float over = total == 0.f ? 0.f : 1.f / total;
        float x[4];
#pragma unroll
        for (int e = 0; e < 4; ++e)
          x[e] = nan[d / kKv4Group] ? NAN : total == 0.f ? 0.f : o[e] * over;
        if (p.wide_out) {
          if constexpr (TYPE == B200_F16)
            *reinterpret_cast<uint2 *>((__half *)p.a.out + to + d) = make_uint2(pack_f16(x[0], x[1]), pack_f16(x[2], x[3]));
          else {
            uint32_t lo, hi;
            asm("cvt.rn.bf16x2.f32 %0, %1, %2;" : "=r"(lo) : "f"(x[1]), "f"(x[0]));
            asm("cvt.rn.bf16x2.f32 %0, %1, %2;" : "=r"(hi) : "f"(x[3]), "f"(x[2]));
            *reinterpret_cast<uint2 *>((__nv_bfloat16 *)p.a.out + to + d) = make_uint2(lo, hi);
          }
        } else {
#pragma unroll
          for (int e = 0; e < 4; ++e)
            put<TYPE>(p, to + d + e, x[e]);
        }
      };
      if (any) {
        wait(ok, &bars.o_full[set], segments & 1, 732);
        ++segments;
        fence_after();
#pragma unroll 1
        for (int c = 0; c < D; c += 32) {
          uint32_t w[32];
          tmem_load32(col_o + c, w);
          tmem_wait_load();
          if (live) {
#pragma unroll
            for (int e = 0; e < 32; e += 4) {
              const float o[4] = {__uint_as_float(w[e]), __uint_as_float(w[e + 1]), __uint_as_float(w[e + 2]), __uint_as_float(w[e + 3])};
              if (whole)
                write_out(c + e, o, l, marks);
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
      if (whole)
        continue;
      __threadfence();
      asm volatile("bar.sync 1, %0;" ::"n"(kSoftmaxWarps * 32) : "memory");
      if (warp == 0) {
        int from, until;
        const bool last = plan.arrive(p.counters, g.at, g.b1 - g.b0, from, until);
        if (lane == 0) {
          bars.last = last;
          bars.from = from;
          bars.to = until;
        }
      }
      asm volatile("bar.sync 1, %0;" ::"n"(kSoftmaxWarps * 32) : "memory");
      if (!bars.last || !live)
        continue;
      __threadfence();
      const int from = bars.from, until = bars.to;
      auto other = [&](int b) { return p.parts + ((int64_t)b * 2 + (b == from)) * H::PART; };
      auto rest = [&](int b, int i) { return __ldcg(other(b) + kSets * kRows * (D + i) + at); };
      float top = kKv4Seed, total = 0.f;
      bool nan[GROUPS] = {};
      for (int b = from; b <= until; ++b)
        top = fmaxf(top, rest(b, 0));
      for (int b = from; b <= until; ++b) {
        total = fmaf(rest(b, 1), ex2(rest(b, 0) - top), total);
#pragma unroll
        for (int gr = 0; gr < GROUPS; ++gr)
          nan[gr] = nan[gr] || rest(b, 2 + gr) != 0.f;
      }
#pragma unroll 1
      for (int d = 0; d < D; d += 16) {
        float o[4][4] = {};
        for (int b = from; b <= until; ++b) {
          const float f = ex2(rest(b, 0) - top);
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            const float4 v = __ldcg(reinterpret_cast<const float4 *>(other(b)) + (d / 4 + i) * (kSets * kRows) + at);
            o[i][0] = fmaf(v.x, f, o[i][0]);
            o[i][1] = fmaf(v.y, f, o[i][1]);
            o[i][2] = fmaf(v.z, f, o[i][2]);
            o[i][3] = fmaf(v.w, f, o[i][3]);
          }
        }
#pragma unroll
        for (int i = 0; i < 4; ++i)
          write_out(d + 4 * i, o[i], total, nan);
      }
    }
  } else if (works && warp < kSoftmaxWarps + kMakers) {
    // ---- makers: 32 keys of every block, two tiles, each ------------------------------------------------------------------------
    const int mw = warp - kSoftmaxWarps, gq = lane >> 2, t = lane & 3;
    struct Raw {
      uint32_t k[2][D / 32], v[D / 16], kp[2][GROUPS], vp[2][2][GROUPS];   // rows g and g + 8; words of V; pairs of keys 2 t + e + 8 u
    };
    auto load_k = [&](Raw &x, int from) {
      const uint8_t *tile = p.pool + (int64_t)max(from, 0) * H::BYTES;   // (a tile that nobody sees: its pairs become zero)
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        const int j = gq + 8 * h;
        if constexpr (D == 128) {
          *reinterpret_cast<uint4 *>(x.k[h]) = __ldg(reinterpret_cast<const uint4 *>(tile + j * 64 + t * 16));
          *reinterpret_cast<uint2 *>(x.kp[h]) = __ldg(reinterpret_cast<const uint2 *>(tile + kv4_k_pairs(D) + j * 8));
        } else {
          *reinterpret_cast<uint2 *>(x.k[h]) = __ldg(reinterpret_cast<const uint2 *>(tile + j * 32 + t * 8));
          x.kp[h][0] = __ldg(reinterpret_cast<const uint32_t *>(tile + kv4_k_pairs(D) + j * 4));
        }
      }
    };
    auto load_v = [&](Raw &x, int from) {
      const uint8_t *tile = p.pool + (int64_t)max(from, 0) * H::BYTES;
#pragma unroll
      for (int gr = 0; gr < GROUPS; ++gr)
        *reinterpret_cast<uint4 *>(x.v + 4 * gr) = __ldg(reinterpret_cast<const uint4 *>(tile + kv4_v_codes(D) + gr * 512 + lane * 16));
    };
    auto load_pairs = [&](Raw &x, int from) {
      const uint8_t *tile = p.pool + (int64_t)max(from, 0) * H::BYTES;
#pragma unroll
      for (int u = 0; u < 2; ++u)
        if constexpr (D == 128)
          *reinterpret_cast<uint4 *>(x.vp[u]) = __ldg(reinterpret_cast<const uint4 *>(tile + kv4_v_pairs(D) + (2 * t + 8 * u) * 8));
        else
          *reinterpret_cast<uint2 *>(x.vp[u]) = __ldg(reinterpret_cast<const uint2 *>(tile + kv4_v_pairs(D) + (2 * t + 8 * u) * 4));
    };
    bool ok = true;
    uint32_t made = 0;
    Walk walk(plan);
    Segment g;
    while (walk.next(plan, g)) {
      const int most = clamp((long long)g.base + g.first + g.tokens, 0, room);   // keys that any row sees
      const uint32_t n = g.b1 - g.b0;
      auto source = [&](uint32_t j, int i) {   // of this warp's tile i of block b0 + j
        const int tile = 8 * (g.b0 + (int)j) + 2 * mw + i;
        return j >= n || tile * kKv4Tile >= most ? -1 : tile_source(p, g.at.s, g.at.slot, tile);
      };
      int now = source(lane >> 1, lane & 1), next = source(16 + (lane >> 1), lane & 1);
      Raw raw[2];
      int from[2], then[2];   // numbers of the tiles in hand, and of the next block's
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        from[i] = __shfl_sync(0xffffffffu, now, i);
        load_k(raw[i], from[i]);
        load_v(raw[i], from[i]);
        load_pairs(raw[i], from[i]);
      }
      for (uint32_t j = 0; j < n; ++j, ++made) {
        uint32_t hole = 0;
#pragma unroll
        for (int i = 0; i < 2; ++i)
          if ((g.b0 + (int)j) * kKeys + 32 * mw + 16 * i < most && from[i] < 0)
            hole |= 0xffffu << (16 * i);
        if (((j + 1) & 15) == 0) {
          now = next;
          next = source(j + 17 + (lane >> 1), lane & 1);
        }
#pragma unroll
        for (int i = 0; i < 2; ++i)
          then[i] = __shfl_sync(0xffffffffu, now, ((j + 1) & 15) * 2 + i);
        const uint32_t stage = made % kStages;
        const int key0 = (g.b0 + (int)j) * kKeys + 32 * mw;
        // ---- pairs: those of keys that nobody sees, and those that are not finite, are zero
        uint32_t k_bad = 0, v_bad[GROUPS] = {};
        int k_lift[2], v_lift[2];
#pragma unroll
        for (int i = 0; i < 2; ++i) {
          float largest = 0.f;
          auto look = [&](uint32_t &pair, int key, uint32_t &bad) {   // key: of this warp's 32
            const bool seen = from[i] >= 0 && key0 + key < most;
            if (!seen || !finite_pair(pair)) {
              if (seen)
                bad |= 1u << key;
              pair = 0u;
            }
            const float2 f = halves(pair);
            largest = fmaxf(largest, fmaxf(fabsf(f.y), fabsf(fmaf(15.f, f.x, f.y))));
          };
#pragma unroll
          for (int h = 0; h < 2; ++h)
#pragma unroll
            for (int gr = 0; gr < GROUPS; ++gr)
              look(raw[i].kp[h][gr], 16 * i + gq + 8 * h, k_bad);
          k_lift[i] = lift(__uint_as_float(__reduce_max_sync(0xffffffffu, __float_as_uint(largest))));
          largest = 0.f;
#pragma unroll
          for (int u = 0; u < 2; ++u)
#pragma unroll
            for (int e = 0; e < 2; ++e)
#pragma unroll
              for (int gr = 0; gr < GROUPS; ++gr)
                look(raw[i].vp[u][e][gr], 16 * i + 2 * t + e + 8 * u, v_bad[gr]);
          v_lift[i] = lift(__uint_as_float(__reduce_max_sync(0xffffffffu, __float_as_uint(largest))));
        }
        Notes &notes = bars.notes[made % kNotes];
        uint32_t bad = k_bad;
#pragma unroll
        for (int gr = 0; gr < GROUPS; ++gr)
          bad |= v_bad[gr];
        const bool any_bad = __any_sync(0xffffffffu, bad != 0);
        if (any_bad) {   // (rare)
          k_bad = __reduce_or_sync(0xffffffffu, k_bad);
#pragma unroll
          for (int gr = 0; gr < GROUPS; ++gr)
            v_bad[gr] = __reduce_or_sync(0xffffffffu, v_bad[gr]);
        }
        // ---- K: words of eight dims of a key
        if (made >= kStages)
          wait(ok, &bars.k_empty[stage], (made / kStages - 1) & 1, 733);
        if (lane < 2) {   // (after the wait: the block four before is done with)
          notes.factor[2 * mw + lane] = power(-(lane ? k_lift[1] : k_lift[0]));
          notes.height[2 * mw + lane] = (float)-(lane ? v_lift[1] : v_lift[0]);
          notes.unit[2 * mw + lane] = power(lane ? v_lift[1] : v_lift[0]);
        }
        if (lane == 0) {
          notes.k_bad[mw] = k_bad;
          notes.hole[mw] = hole;
#pragma unroll
          for (int gr = 0; gr < GROUPS; ++gr)
            notes.v_bad[gr][mw] = v_bad[gr];
          notes.special[mw] = (any_bad ? 1u : 0u) | hole;
        }
        uint8_t *k_at = ks + stage * H::KV_BYTES, *v_at = vs + stage * H::KV_BYTES;
#pragma unroll
        for (int i = 0; i < 2; ++i) {
          const float one = power(k_lift[i]);
#pragma unroll
          for (int h = 0; h < 2; ++h)
#pragma unroll
            for (int w = 0; w < D / 32; ++w) {
              const float2 f = halves(raw[i].kp[h][w / 2]);
              const float s = f.x * one, l = f.y * one;
              const uint32_t low = pack_f16(s * 16777216.f, s * 16777216.f), high = pack_f16(s * 1048576.f, s * 1048576.f), lo = pack_f16(l, l);
              const uint32_t x = raw[i].k[h][w], y = x >> 8;
              *reinterpret_cast<uint4 *>(k_at + w / 2 * (kKeys * 128) + swz(32 * mw + 16 * i + gq + 8 * h, 4 * (w & 1) + t)) =
                  make_uint4(fma2(x & 0x000f000fu, low, lo), fma2(x & 0x00f000f0u, high, lo), fma2(y & 0x000f000fu, low, lo), fma2(y & 0x00f000f0u, high, lo));
            }
        }
        fence_proxy();
        __syncwarp();
        if (lane == 0)
          mbar_arrive(&bars.k_full[stage]);
#pragma unroll
        for (int i = 0; i < 2; ++i)
          load_k(raw[i], then[i]);
        // ---- V: words of dims 16 w + g (+ 8) and keys 2 t, 2 t + 1 (+ 8)
        if (made >= kStages)
          wait(ok, &bars.v_empty[stage], (made / kStages - 1) & 1, 734);
#pragma unroll
        for (int i = 0; i < 2; ++i) {
          const float unit = power(v_lift[i]);
#pragma unroll
          for (int gr = 0; gr < GROUPS; ++gr) {
            uint32_t low[2], high[2], lo[2];
#pragma unroll
            for (int u = 0; u < 2; ++u) {
              const float2 a = halves(raw[i].vp[u][0][gr]), b = halves(raw[i].vp[u][1][gr]);
              low[u] = pack_f16(a.x * unit * 16777216.f, b.x * unit * 16777216.f);
              high[u] = pack_f16(a.x * unit * 1048576.f, b.x * unit * 1048576.f);
              lo[u] = pack_f16(a.y * unit, b.y * unit);
            }
#pragma unroll
            for (int w = 4 * gr; w < 4 * gr + 4; ++w) {
              const uint32_t x = raw[i].v[w], y = x >> 8;
              uint8_t *to = v_at + mw / 2 * (D * 128) + 4 * t;
              const int c = mw % 2 * 4 + 2 * i, d = 16 * w + gq;
              *reinterpret_cast<uint32_t *>(to + swz(d, c)) = fma2(x & 0x000f000fu, low[0], lo[0]);
              *reinterpret_cast<uint32_t *>(to + swz(d + 8, c)) = fma2(x & 0x00f000f0u, high[0], lo[0]);
              *reinterpret_cast<uint32_t *>(to + swz(d, c + 1)) = fma2(y & 0x000f000fu, low[1], lo[1]);
              *reinterpret_cast<uint32_t *>(to + swz(d + 8, c + 1)) = fma2(y & 0x00f000f0u, high[1], lo[1]);
            }
          }
        }
        fence_proxy();
        __syncwarp();
        if (lane == 0)
          mbar_arrive(&bars.v_full[stage]);
#pragma unroll
        for (int i = 0; i < 2; ++i) {
          from[i] = then[i];
          load_v(raw[i], from[i]);
          load_pairs(raw[i], from[i]);
        }
      }
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

RaisedOn g_raised[4];
constexpr int kMostSeqs = 1900;   // whose plan fits beside the operands

template <int D, int TYPE> int chunk_launch(RaisedOn &raised, const Kv4Params &p, cudaStream_t st) {
  if (int rc = raise_shared_limit(raised, (const void *)kv4_chunk_kernel<D, TYPE>, Shape<D>::SMEM + KeyPlan<kShift>::bytes(kMostSeqs)))
    return rc;
  return launch_after(kv4_chunk_kernel<D, TYPE>, dim3(kKv4Ctas), kThreads, Shape<D>::SMEM + KeyPlan<kShift>::bytes(p.a.n_seqs), st, p);
}

} // namespace

int64_t kv4_chunk_part_floats(int D) { return 2 * (D == 128 ? Shape<128>::PART : Shape<64>::PART); }

bool kv4_chunk_takes(int dtype, int G, int n_seqs) { return (dtype == B200_F16 || dtype == B200_BF16) && G <= kRows && n_seqs <= kMostSeqs; }

int kv4_chunk_launch(Kv4Params p, int D, cudaStream_t st) {
  p.heads = p.G;
  p.subs = 1;
  p.tokens = kSets * (kRows / p.G);
  if (p.a.dtype == B200_F16)
    return D == 128 ? chunk_launch<128, B200_F16>(g_raised[0], p, st) : chunk_launch<64, B200_F16>(g_raised[1], p, st);
  return D == 128 ? chunk_launch<128, B200_BF16>(g_raised[2], p, st) : chunk_launch<64, B200_BF16>(g_raised[3], p, st);
}

} // namespace b200
