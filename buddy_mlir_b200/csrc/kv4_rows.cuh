// What the forms of the 4-bit cache's attention for sequences of many rows share (kv4_chunk.cu: bf16, kv4_exact.cu: f32 and f16): blocks of 128 keys by 128 query
// rows on tcgen05, an item's parts and how they meet.
#pragma once
#include "kv4_plan.cuh"
#include "tensor_core.cuh"

namespace b200 {

constexpr int kRows = 128;                          // query rows of a product
constexpr int kKeys = 128, kShift = 7;              // of a block
constexpr int kTiles = kKeys / kKv4Tile;            // of a block
using RowsPlan = KeyPlan<kShift>;

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
// (the values are there after the wait, and the compiler takes them from it)
__device__ __forceinline__ void tmem_arrived(uint32_t (&v)[32]) {
  asm volatile("tcgen05.wait::ld.sync.aligned;"
               : "+r"(v[0]), "+r"(v[1]), "+r"(v[2]), "+r"(v[3]), "+r"(v[4]), "+r"(v[5]), "+r"(v[6]), "+r"(v[7]), "+r"(v[8]), "+r"(v[9]), "+r"(v[10]),
                 "+r"(v[11]), "+r"(v[12]), "+r"(v[13]), "+r"(v[14]), "+r"(v[15]), "+r"(v[16]), "+r"(v[17]), "+r"(v[18]), "+r"(v[19]), "+r"(v[20]),
                 "+r"(v[21]), "+r"(v[22]), "+r"(v[23]), "+r"(v[24]), "+r"(v[25]), "+r"(v[26]), "+r"(v[27]), "+r"(v[28]), "+r"(v[29]), "+r"(v[30]),
                 "+r"(v[31])
               :
               : "memory");
}
__device__ __forceinline__ void tmem_wait_store() { asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory"); }
__device__ __forceinline__ void fence_before() { asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory"); }
__device__ __forceinline__ void fence_after() { asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory"); }
__device__ __forceinline__ void fence_proxy() { asm volatile("fence.proxy.async.shared::cta;" ::: "memory"); }
// (Operands in shared memory: rows of 128 bytes, 128-byte swizzle: 16-byte chunk c of row r lies at chunk c ^ (r & 7).)
__device__ __forceinline__ void store4(uint32_t at, uint32_t a, uint32_t b, uint32_t c, uint32_t d) {   // (an address in shared memory)
  asm volatile("st.shared.v4.b32 [%0], {%1, %2, %3, %4};" ::"r"(at), "r"(a), "r"(b), "r"(c), "r"(d) : "memory");
}
__device__ __forceinline__ void store2(uint32_t at, uint32_t a, uint32_t b) { asm volatile("st.shared.v2.b32 [%0], {%1, %2};" ::"r"(at), "r"(a), "r"(b) : "memory"); }
__device__ __forceinline__ void store1(uint32_t at, uint32_t a) { asm volatile("st.shared.b32 [%0], %1;" ::"r"(at), "r"(a) : "memory"); }
__device__ __forceinline__ uint32_t fma2(uint32_t a, uint32_t b, uint32_t c) {
  uint32_t r;
  asm("fma.rn.f16x2 %0, %1, %2, %3;" : "=r"(r) : "r"(a), "r"(b), "r"(c));
  return r;
}
__device__ __forceinline__ float max3(float a, float b, float c) {
  float r;
  asm("max.f32 %0, %1, %2, %3;" : "=f"(r) : "f"(a), "f"(b), "f"(c));
  return r;
}
__device__ __forceinline__ bool finite_pair(uint32_t pair) { return (pair & 0x7c00u) != 0x7c00u && (pair & 0x7c000000u) != 0x7c000000u; }
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
  __device__ __forceinline__ Walk(const RowsPlan &plan) {
    const int lane = threadIdx.x & 31;
    const long long x = plan.border(blockIdx.x + min(lane, 1));
    over = __shfl_sync(0xffffffffu, x, 0) == __shfl_sync(0xffffffffu, x, 1);
    at = Place{plan.n, 0, 0, 0};
    if (x < plan.total)
      at = plan.locate(x);
    stop.s = __shfl_sync(0xffffffffu, at.s, 1);
    stop.slot = __shfl_sync(0xffffffffu, at.slot, 1);
    stop.rt = __shfl_sync(0xffffffffu, at.rt, 1);
    stop.tile = __shfl_sync(0xffffffffu, at.tile, 1);
    at.s = __shfl_sync(0xffffffffu, at.s, 0);
    at.slot = __shfl_sync(0xffffffffu, at.slot, 0);
    at.rt = __shfl_sync(0xffffffffu, at.rt, 0);
    at.tile = __shfl_sync(0xffffffffu, at.tile, 0);
  }
  __device__ __forceinline__ bool next(const RowsPlan &plan, Segment &g) {
    while (!over && at.s < plan.n) {
      const Sequence q = plan.sequence(at.s);
      g.all = plan.item_tiles(q, at.rt);
      const bool here = stop.s == at.s && stop.slot == at.slot && stop.rt == at.rt;
      if (at.tile >= g.all && !here) {
        plan.next_item(at, q);
        continue;
      }
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

// four dims of a row: sums over its total, zero where it saw nothing
template <int TYPE> __device__ __forceinline__ void put_over(const Kv4Params &p, int64_t to, const float (&o)[4], float total, bool nan) {
  const float over = total == 0.f ? 0.f : 1.f / total;
  float x[4];
#pragma unroll
  for (int e = 0; e < 4; ++e)
    x[e] = nan ? NAN : total == 0.f ? 0.f : o[e] * over;
  put4<TYPE>(p, to, make_float4(x[0], x[1], x[2], x[3]));
}
// A part of an item: sums [D / 4][ROWS][4], then each row's reference, total and marks (V groups that become NaN).
template <int D, int ROWS> __host__ __device__ constexpr int rows_part() { return ROWS * (D + 2 + D / kKv4Group); }
struct Meeting {
  int last, from, to;
};
// This CTA's part is in memory; by THREADS threads of its first warps, a row (`at`) each.  Who completes the item adds its parts up, in their order.
template <int D, int TYPE, int ROWS, int THREADS>
__device__ __forceinline__ void meet(const Kv4Params &p, const RowsPlan &plan, const Segment &g, Meeting &m, int at, bool live, int64_t to, int d0 = 0, int d1 = D) {
  constexpr int GROUPS = D / kKv4Group, PART = rows_part<D, ROWS>();
  __threadfence();
  asm volatile("bar.sync 1, %0;" ::"n"(THREADS) : "memory");
  if (threadIdx.x < 32) {
    int from, until;
    const bool last = plan.arrive(p.counters, g.at, g.b1 - g.b0, from, until);
    if (threadIdx.x == 0) {
      m.last = last;
      m.from = from;
      m.to = until;
    }
  }
  asm volatile("bar.sync 1, %0;" ::"n"(THREADS) : "memory");
  if (!m.last || !live)
    return;
  __threadfence();
  const int from = m.from, until = m.to;
  auto other = [&](int b) { return p.parts + ((int64_t)b * 2 + (b == from)) * PART; };
  auto rest = [&](int b, int i) { return __ldcg(other(b) + ROWS * (D + i) + at); };
  float top = kKv4Seed, total = 0.f;
  bool nan[GROUPS] = {};
#pragma unroll 4
  for (int b = from; b <= until; ++b)
    top = fmaxf(top, rest(b, 0));
#pragma unroll 2
  for (int b = from; b <= until; ++b) {
    total = fmaf(rest(b, 1), ex2(rest(b, 0) - top), total);
#pragma unroll
    for (int gr = 0; gr < GROUPS; ++gr)
      nan[gr] = nan[gr] || rest(b, 2 + gr) != 0.f;
  }
#pragma unroll 1
  for (int d = d0; d < d1; d += 32) {
    float o[8][4] = {};
#pragma unroll 2
    for (int b = from; b <= until; ++b) {
      const float f = ex2(rest(b, 0) - top);
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        const float4 v = __ldcg(reinterpret_cast<const float4 *>(other(b)) + (d / 4 + i) * ROWS + at);
        o[i][0] = fmaf(v.x, f, o[i][0]);
        o[i][1] = fmaf(v.y, f, o[i][1]);
        o[i][2] = fmaf(v.z, f, o[i][2]);
        o[i][3] = fmaf(v.w, f, o[i][3]);
      }
    }
#pragma unroll
    for (int i = 0; i < 8; ++i)
      put_over<TYPE>(p, to + d + 4 * i, o[i], total, nan[d / kKv4Group]);
  }
}

} // namespace b200
