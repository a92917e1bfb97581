// Attention over the 4-bit KV cache (b200_kv4_attention).
//
// Codes go to the tensor cores as they are: with k = lo + s c per group of 64 dims, a score is  q.k = sum over groups of s (q.c) + lo sum(q),  and
// an output  sum p v = sum (p s) c + sum p lo,  so that scales meet scores and weights (a handful per key) instead of 64 codes each.  A code is one
// f16 exactly; the other operand is one f16 (f32: two, 22 bits of it) after a power of two of its row that puts the row's largest near f16's.
// Codes are the operand with M rows (mma.m16n8k16: sixteen positions, or sixteen dims), the query rows that share a kv head the eight
// columns; words of eight codes lie in the cache as the operand's registers want them, and one and-or makes a pair of codes a pair of
// f16 (1024 + c, or 1024 + 16 c: the code in the mantissa's low bits).
//
// The reference r of a row's weights is not its largest score but the largest of score + log2 of the key's larger V scale, so that the weights
// that meet codes, p s, are at most 2^12 and near 2^8 where they count, whatever the scales are; sums and totals carry the same factor.
#include "kv4.cuh"

#include <algorithm>

namespace b200 {

namespace {

constexpr int kWarps = 8, kThreads = 32 * kWarps, kCtas = 296;
constexpr int kRows = 8;            // query rows of an item: a position's heads (several positions', if they are few)
constexpr int kStages = 3;          // tiles that a warp has in flight or in hand
constexpr float kTop = 8.f;          // powers of two: what the largest weight p s is at when a row's reference is set,
constexpr float kLag = 4.f;          // and how far above that one may come before it is set again
constexpr float kSeed = -1.0e30f;
constexpr float kLeastScale = 5.9604645e-8f;   // (f16's smallest: a group of equal values has the scale 0)

struct AttentionParams {
  const uint8_t *pool;
  int n_pages, kv_heads, page;
  b200_kv4_attention_args a;
  int G, heads, tokens, subs;       // q heads of a kv head, of an item; positions of an item; items that share a kv head's q heads
  float log2_scale;
  int *counters;                    // [kCtas]
  float *parts;                     // [kCtas][2][part floats]
};

__host__ __device__ constexpr int part_floats(int D) { return kRows * (D + 4) + 2 * kRows; }   // sums in rows of D + 4, maxima, totals

__device__ __forceinline__ int clamp(long long x, int lo, int hi) { return (int)(x < lo ? lo : x > hi ? hi : x); }
__device__ __forceinline__ float ex2(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}
__device__ __forceinline__ float lg2(float x) {
  float y;
  asm("lg2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}
__device__ __forceinline__ uint32_t pack_f16(float lo, float hi) {
  uint32_t r;
  asm("cvt.rn.f16x2.f32 %0, %1, %2;" : "=r"(r) : "f"(hi), "f"(lo));
  return r;
}
__device__ __forceinline__ float2 halves(uint32_t pair) { return __half22float2(*reinterpret_cast<const __half2 *>(&pair)); }
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

// Codes of nibbles p and p + 4 of w >> 8 * (p / 2), p = 0 and 1, as pairs of f16: 1024 + c and 1024 + 16 c as they come, or (CENTRED) c - 8.  All exact.
// Centred operands keep a sum of n weighted codes as small as the values' own spread: the tensor cores' sums round towards zero.
constexpr float kCentre = 8.f;
constexpr float kOffset = 1024.f;   // not centred: of the products with q (lo), and with q / 16 (hi)
template <bool CENTRED> __device__ __forceinline__ void codes(uint32_t w, uint32_t &lo, uint32_t &hi) {
  lo = (w & 0x000f000fu) | 0x64006400u;
  hi = (w & 0x00f000f0u) | 0x64006400u;
  if constexpr (CENTRED) {
    asm("add.rn.f16x2 %0, %0, %1;" : "+r"(lo) : "r"(0xe408e408u));                                   // - 1032
    asm("fma.rn.f16x2 %0, %0, %1, %2;" : "+r"(hi) : "r"(0x2c002c00u), "r"(0xd480d480u));             // / 16 - 72
  }
}

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

// A sequence as its items: its rows `tokens` at a time and, for each kv head (or part of its q heads), a range of keys that ends at the last
// row's own position.  Cost of an item: its keys; of all items before it in a head: before().
struct Sequence {
  int r0, n;            // rows
  int base;             // position of the first row (negative: rows before it see nothing), at most the table's room
  int past, tiles;      // max(base, 0); row tiles
  __device__ __forceinline__ Sequence(const AttentionParams &p, int s, int room) {
    r0 = clamp(p.a.row_start[s], 0, p.a.rows);
    n = clamp(p.a.row_start[s + 1], r0, p.a.rows) - r0;
    base = clamp((long long)p.a.lens[s] - n, -n, room);
    past = max(base, 0);
    tiles = (n + p.tokens - 1) / p.tokens;
  }
  __device__ __forceinline__ long long before(int rt, int tokens) const {
    return rt < tiles ? (long long)rt * past + (long long)tokens * rt * (rt + 1) / 2
                      : tiles == 0 ? 0 : (long long)(tiles - 1) * past + (long long)tokens * tiles * (tiles - 1) / 2 + past + n;
  }
};

template <int D, int TYPE> struct Tile {   // of a warp: one item's sums
  static constexpr int GROUPS = D / kKv4Group, STEPS = D / 16, TERMS = TYPE == B200_F32 ? 2 : 1;
  // K's codes: a score of bf16 queries does not notice that 1024 + c costs it 2^-13 of the sum of |q s|; f16 would
  static constexpr bool K_CENTRED = TYPE != B200_BF16;
  uint32_t q[TERMS][STEPS][2];
  float qs[GROUPS][2];                      // sums of q over a group, times the scores' scale, of rows 2 t and 2 t + 1 (t: lane % 4)
  float minus[K_CENTRED ? 1 : GROUPS][2];   // what the offsets of codes add up to, negative
  float unit[2];                            // the scores' scale over the row's power of two
  float o[STEPS][4];                        // dims 16 i + g (+ 8), rows 2 t (+ 1) (g: lane / 4)
  float bias[GROUPS][2], r[2], l[2];        // sums over this lane's keys: p (lo + 8 s), p

  __device__ __forceinline__ void clear() {
#pragma unroll
    for (int i = 0; i < STEPS; ++i)
#pragma unroll
      for (int e = 0; e < 4; ++e)
        o[i][e] = 0.f;
#pragma unroll
    for (int e = 0; e < 2; ++e) {
      r[e] = kSeed;
      l[e] = 0.f;
#pragma unroll
      for (int gr = 0; gr < GROUPS; ++gr)
        bias[gr][e] = 0.f;
    }
  }

  // q of this lane's row (lane / 4), or none
  __device__ __forceinline__ void load_q(const AttentionParams &p, bool live, int64_t at) {
    const int lane = threadIdx.x & 31, t = lane & 3;
    float x[STEPS][4], most = 0.f;
#pragma unroll
    for (int k = 0; k < STEPS; ++k) {
      const int d = 32 * (k / 2) + 8 * t + 4 * (k & 1);
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        x[k][e] = live ? load_as_float(p.a.q, TYPE, at + d + e) : 0.f;
        most = fmaxf(most, fabsf(x[k][e]));
      }
    }
    most = fmaxf(most, __shfl_xor_sync(0xffffffffu, most, 1));
    most = fmaxf(most, __shfl_xor_sync(0xffffffffu, most, 2));
    // 2^up: the row's largest comes to 2^14 .. 2^15 (a row below 2^-86 not as far)
    const int up = min(max(14 + 127 - (int)(__float_as_uint(most) >> 23), -113), 100);
    const float factor = __uint_as_float((uint32_t)(127 + up) << 23), over = p.log2_scale * __uint_as_float((uint32_t)(127 - up) << 23);
#pragma unroll
    for (int e = 0; e < 2; ++e)
      unit[e] = __shfl_sync(0xffffffffu, over, 8 * t + 4 * e);
#pragma unroll
    for (int gr = 0; gr < GROUPS; ++gr) {
      float sum = 0.f, off = 0.f;
#pragma unroll
      for (int k = 4 * gr; k < 4 * gr + 4; ++k) {
        float y[4];
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          sum += x[k][e];
          y[e] = x[k][e] * factor;
          if constexpr (!K_CENTRED) {
            y[e] = __half2float(__float2half_rn(e / 2 == 0 ? y[e] : y[e] * 0.0625f));
            off = fmaf(kOffset, y[e], off);
          }
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
      if constexpr (!K_CENTRED) {
        off += __shfl_xor_sync(0xffffffffu, off, 1);
        off += __shfl_xor_sync(0xffffffffu, off, 2);
#pragma unroll
        for (int e = 0; e < 2; ++e)
          minus[gr][e] = -__shfl_sync(0xffffffffu, off, 8 * t + 4 * e);
      }
    }
  }

  // sixteen keys from j0 on; limit: keys that rows 2 t and 2 t + 1 see (only where MASKED)
  template <bool MASKED> __device__ __forceinline__ void keys(const uint8_t *tile, int j0, const int (&limit)[2]) {
    const int lane = threadIdx.x & 31, g = lane >> 2, t = lane & 3;
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
      float c[4];
#pragma unroll
      for (int e = 0; e < 4; ++e)
        c[e] = K_CENTRED ? 0.f : minus[K_CENTRED ? 0 : gr][e & 1];
#pragma unroll
      for (int i = 2 * gr; i < 2 * gr + 2; ++i)
#pragma unroll
        for (int u = 0; u < 2; ++u) {
          uint32_t a[4];
          codes<K_CENTRED>(kw[0][i] >> (8 * u), a[0], a[2]);
          codes<K_CENTRED>(kw[1][i] >> (8 * u), a[1], a[3]);
#pragma unroll
          for (int e = TERMS - 1; e >= 0; --e)
            mma(c, a, q[e][2 * i + u][0], q[e][2 * i + u][1]);
        }
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        const float2 pair = halves(kp[h][gr]);
        const float lo = K_CENTRED ? fmaf(kCentre, pair.x, pair.y) : pair.y;
#pragma unroll
        for (int e = 0; e < 2; ++e) {
          dot[2 * h + e] = fmaf(c[2 * h + e], pair.x, dot[2 * h + e]);
          low[2 * h + e] = fmaf(lo, qs[gr][e], low[2 * h + e]);
        }
      }
    }
    float s[4], at[4], vs[GROUPS][2], vb[GROUPS][2];
    bool out[4];   // not seen
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      float largest = kLeastScale;
#pragma unroll
      for (int gr = 0; gr < GROUPS; ++gr) {
        const float2 pair = halves(vp[h][gr]);
        vs[gr][h] = pair.x;
        vb[gr][h] = fmaf(kCentre, pair.x, pair.y);
        largest = fmaxf(largest, pair.x);
      }
      const float height = lg2(largest);
#pragma unroll
      for (int e = 0; e < 2; ++e) {
        const int k = 2 * h + e;
        s[k] = fmaf(dot[k], unit[e], low[k]);
        if constexpr (MASKED) {
          out[k] = j0 + g + 8 * h >= limit[e];
          s[k] = out[k] ? -INFINITY : s[k];
        }
        at[k] = s[k] + height;
        if constexpr (MASKED)
          at[k] = out[k] ? -INFINITY : at[k];
      }
    }
    if (__any_sync(0xffffffffu, fmaxf(at[0], at[2]) > r[0] + (kTop + kLag) || fmaxf(at[1], at[3]) > r[1] + (kTop + kLag))) {
#pragma unroll
      for (int e = 0; e < 2; ++e) {
        float top = fmaxf(at[e], at[2 + e]);
#pragma unroll
        for (int x = 4; x < 32; x <<= 1)
          top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, x));
        top = fmaxf(top - kTop, r[e]);
        const float keep = ex2(r[e] - top);
        r[e] = top;
        l[e] *= keep;
#pragma unroll
        for (int gr = 0; gr < GROUPS; ++gr)
          bias[gr][e] *= keep;
#pragma unroll
        for (int i = 0; i < STEPS; ++i) {
          o[i][e] *= keep;
          o[i][2 + e] *= keep;
        }
      }
    }
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      s[e] = ex2(s[e] - r[e & 1]);
      l[e & 1] += s[e];
    }
#pragma unroll
    for (int gr = 0; gr < GROUPS; ++gr) {
      float w[4];
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        w[e] = s[e] * vs[gr][e >> 1];
        float b = fmaf(s[e], vb[gr][e >> 1], bias[gr][e & 1]);
        if constexpr (MASKED) {   // (what is not seen may be NaN)
          w[e] = out[e] ? 0.f : w[e];
          b = out[e] ? bias[gr][e & 1] : b;
        }
        bias[gr][e & 1] = b;
      }
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
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        uint32_t a[4];
        codes<true>(vw[i], a[0], a[1]);
        codes<true>(vw[i] >> 8, a[2], a[3]);
        if constexpr (TERMS == 1) {
          mma(o[4 * gr + i], a, b0[0], b1[0]);
        } else {   // f32: a sum of its own, added with rounding to nearest
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
        o[i][e] += bias[i * 16 / kKv4Group][e];
        o[i][2 + e] += bias[i * 16 / kKv4Group][e];
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

__device__ __forceinline__ void put(const AttentionParams &p, int64_t at, float x) {
  if (p.a.dtype == B200_F32)
    ((float *)p.a.out)[at] = x;
  else if (p.a.dtype == B200_F16)
    ((__half *)p.a.out)[at] = __float2half_rn(x);
  else
    ((__nv_bfloat16 *)p.a.out)[at] = __float2bfloat16_rn(x);
}
// element of an item's row in q (ld: q's) or out, before its dims
__device__ __forceinline__ int64_t row_at(const AttentionParams &p, int r0, int rt, int slot, int row, int64_t ld, int D) {
  return (r0 + (int64_t)rt * p.tokens + row / p.heads) * ld + (int64_t)((slot / p.subs) * p.G + slot % p.subs * p.heads + row % p.heads) * D;
}
__device__ __forceinline__ int rows_of(const AttentionParams &p, const Sequence &q, int rt, int slot) {   // of an item
  const int tokens = min(p.tokens, q.n - rt * p.tokens);
  return p.subs == 1 ? tokens * p.heads : min(p.heads, p.G - slot % p.subs * p.heads);
}
// Where a warp stands: an item and the next of its tiles.
struct Place {
  int s, slot, rt, tile;
};

// A chain of parts of an item that ends in this CTA, or leaves it (by its last warp).
struct Chain {
  Place at;          // the item
  int first, last;   // warps with its parts
  bool opened;       // here: the first part is that warp's second one
  bool ends;
};

template <int D, int TYPE> __global__ void __launch_bounds__(kThreads, 2) kv4_attention_kernel(const __grid_constant__ AttentionParams p) {
  constexpr int BYTES = kv4_tile_bytes(D), PART = part_floats(D), RING = kStages * BYTES;
  static_assert(RING >= PART * 4, "the second part of a warp lies in its ring");
  extern __shared__ __align__(128) uint8_t s_all[];
  uint8_t *s_ring = s_all;
  float *s_part = reinterpret_cast<float *>(s_all + kWarps * RING);                                // first parts
  long long *s_cost = reinterpret_cast<long long *>(s_all + kWarps * (RING + PART * 4));          // [n_seqs + 1]
  __shared__ long long s_sum[kWarps];
  __shared__ Chain s_chain[kWarps + 1];
  __shared__ bool s_has_a[kWarps], s_a_ends[kWarps], s_has_b[kWarps];
  __shared__ Place s_a[kWarps], s_b[kWarps];
  __shared__ int s_n_chains, s_last;
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, n = p.a.n_seqs, room = p.a.table_stride * p.page, slots = p.kv_heads * p.subs;
  kernel_go();
  kernel_wait();

  // ---- costs of all sequences, added up --------------------------------------------------------------------------------------
  {
    const int per = (n + kThreads - 1) / kThreads, first = min(n, tid * per), last = min(n, first + per);
    long long sum = 0;
    for (int s = first; s < last; ++s) {
      const Sequence q(p, s, room);
      s_cost[s] = sum;
      sum += slots * q.before(q.tiles, p.tokens);
    }
    long long upto = sum;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const long long v = __shfl_up_sync(0xffffffffu, upto, o);
      if (lane >= o)
        upto += v;
    }
    if (lane == 31)
      s_sum[warp] = upto;
    __syncthreads();
    long long before = upto - sum;
    for (int w = 0; w < warp; ++w)
      before += s_sum[w];
    for (int s = first; s < last; ++s)
      s_cost[s] += before;
    if (tid == kThreads - 1)
      s_cost[n] = before + sum;
    __syncthreads();
  }
  // rows of no sequence
  {
    const int lo = clamp(p.a.row_start[0], 0, p.a.rows), hi = clamp(p.a.row_start[n], lo, p.a.rows), none = lo + p.a.rows - hi, cols = p.a.q_heads * D;
    for (int64_t i = (int64_t)blockIdx.x * kThreads + tid; i < (int64_t)none * cols; i += (int64_t)gridDim.x * kThreads) {
      const int r = (int)(i / cols);
      put(p, (int64_t)(r < lo ? r : hi + r - lo) * p.a.out_ld + i % cols, 0.f);
    }
  }
  const long long total = s_cost[n];
  if (total == 0)
    return;
  // the warps that work: sixteen keys each at least (then each begins a tile)
  const long long workers = max(1ll, min((long long)gridDim.x * kWarps, total / 16));
  const long long me = (long long)blockIdx.x * kWarps + warp;
  if ((long long)blockIdx.x * kWarps >= workers)
    return;
  auto place = [&](long long x) {   // the first tile that begins at x or behind it
    Place at;
    int lo = 0, hi = n;
    while (hi - lo > 1) {
      const int mid = (lo + hi) >> 1;
      if (s_cost[mid] <= x)
        lo = mid;
      else
        hi = mid;
    }
    at.s = lo;
    const Sequence q(p, lo, room);
    x -= s_cost[lo];
    const long long head = q.before(q.tiles, p.tokens);
    at.slot = (int)(x / head);
    x -= at.slot * head;
    int a = 0, b = q.tiles;
    while (b - a > 1) {
      const int mid = (a + b) >> 1;
      if (q.before(mid, p.tokens) <= x)
        a = mid;
      else
        b = mid;
    }
    at.rt = a;
    at.tile = (int)((x - q.before(a, p.tokens) + 15) >> 4);
    return at;
  };
  auto item_tiles = [&](const Sequence &q, int rt) { return (q.past + min((rt + 1) * p.tokens, q.n) + 15) >> 4; };
  auto next_item = [&](Place &at, const Sequence &q) {   // (leaves the sequence: true)
    at.tile = 0;
    if (++at.rt < q.tiles)
      return false;
    at.rt = 0;
    if (++at.slot < slots)
      return false;
    at.slot = 0;
    do
      ++at.s;
    while (at.s < n && s_cost[at.s + 1] == s_cost[at.s]);
    return true;
  };
  if (lane == 0)
    s_has_a[warp] = s_has_b[warp] = false;

  if (me < workers) {
    Place at = place(total * me / workers);
    const long long end = total * (me + 1) / workers;
    Place stop{n, 0, 0, 0};
    if (end < total)
      stop = place(end);
    Tile<D, TYPE> tile;
    uint8_t *ring = s_ring + warp * RING;
    while (at.s < n) {
      const Sequence q(p, at.s, room);
      const int T = item_tiles(q, at.rt);
      if (at.tile >= T) {   // (a boundary behind an item's last tile)
        next_item(at, q);
        continue;
      }
      const bool here = stop.s == at.s && stop.slot == at.slot && stop.rt == at.rt;
      const int t0 = at.tile, t1 = here ? min(stop.tile, T) : T;
      if (t0 >= t1)
        break;
      // ---- this warp's tiles of the item ----------------------------------------------------------------------------------------
      const int live = rows_of(p, q, at.rt, at.slot), first_token = at.rt * p.tokens, tokens = min(p.tokens, q.n - first_token);
      const int least = clamp((long long)q.base + first_token + 1, 0, room), most = clamp((long long)q.base + first_token + tokens, 0, room);
      const int kv = at.slot / p.subs, per_page = p.page / kKv4Tile;
      auto source = [&](int t) {   // of lane's tile: its number in the pool, or -1
        if (t >= t1 || t * kKv4Tile >= most)
          return -1;
        const int id = p.a.block_table[(int64_t)at.s * p.a.table_stride + t / per_page];
        return id < 0 || id >= p.n_pages ? -1 : (id * p.kv_heads + kv) * per_page + t % per_page;
      };
      int now = source(t0 + lane), next = source(t0 + 32 + lane);
      tile.clear();
      uint32_t none = 0;   // bit of a stage: nothing to see in its tile
      int ahead = 0, hand = 0;      // stages: of the next tile to ask for, of the tile in hand
      auto request = [&](int i) {   // tile t0 + i
        if (i > 0 && (i & 31) == 0) {
          now = next;
          next = source(t0 + i + 32 + lane);
        }
        const int from = __shfl_sync(0xffffffffu, now, i & 31);
        none = from < 0 ? none | 1u << ahead : none & ~(1u << ahead);
        if (from >= 0) {
          const uint8_t *src = p.pool + (int64_t)from * BYTES + lane * 16;
          uint8_t *to = ring + ahead * BYTES + lane * 16;
#pragma unroll
          for (int c = 0; c < BYTES / 512; ++c)
            copy16(to + c * 512, src + c * 512);
          if (BYTES % 512 != 0 && lane < BYTES % 512 / 16)
            copy16(to + BYTES / 512 * 512, src + BYTES / 512 * 512);
        }
        copies_commit();
        ahead = ahead == kStages - 1 ? 0 : ahead + 1;
      };
      const int count = t1 - t0;
      __syncwarp();
#pragma unroll
      for (int i = 0; i < kStages - 1; ++i)
        request(i);
      tile.load_q(p, lane / 4 < live, lane / 4 < live ? row_at(p, q.r0, at.rt, at.slot, lane / 4, p.a.q_ld, D) : 0);
#pragma unroll 1
      for (int i = 0; i < count; ++i) {
        copies_wait<kStages - 2>();
        __syncwarp();
        const bool skip = none >> hand & 1;
        const uint8_t *bytes = ring + hand * BYTES;
        hand = hand == kStages - 1 ? 0 : hand + 1;
        request(i + kStages - 1);
        if (skip)
          continue;
        const int j0 = (t0 + i) * kKv4Tile;
        int limit[2] = {0, 0};
        if (j0 + kKv4Tile <= least) {
          tile.template keys<false>(bytes, j0, limit);
        } else {
#pragma unroll
          for (int e = 0; e < 2; ++e) {
            const int row = 2 * (lane & 3) + e;
            limit[e] = row < live ? clamp((long long)q.base + first_token + row / p.heads + 1, 0, room) : 0;
          }
          tile.template keys<true>(bytes, j0, limit);
        }
      }
      copies_wait<0>();
      __syncwarp();
      tile.finish();
      // ---- whole, or a part -------------------------------------------------------------------------------------------------------
      if (t0 == 0 && t1 == T) {
        float over[2];
#pragma unroll
        for (int e = 0; e < 2; ++e)
          over[e] = tile.l[e] == 0.f ? 0.f : 1.f / tile.l[e];
#pragma unroll
        for (int e = 0; e < 2; ++e) {
          const int row = 2 * (lane & 3) + e;
          if (row < live) {
            const int64_t to = row_at(p, q.r0, at.rt, at.slot, row, p.a.out_ld, D) + lane / 4;
#pragma unroll
            for (int i = 0; i < D / 16; ++i) {
              put(p, to + 16 * i, tile.l[e] == 0.f ? 0.f : tile.o[i][e] * over[e]);
              put(p, to + 16 * i + 8, tile.l[e] == 0.f ? 0.f : tile.o[i][2 + e] * over[e]);
            }
          }
        }
      } else if (t0 > 0) {   // (only a warp's first item)
        tile.store(s_part + warp * PART);
        if (lane == 0) {
          s_has_a[warp] = true;
          s_a_ends[warp] = t1 == T;
          s_a[warp] = at;
        }
      } else {               // (only its last)
        tile.store(reinterpret_cast<float *>(ring));
        if (lane == 0) {
          s_has_b[warp] = true;
          s_b[warp] = at;
        }
      }
      if (here)
        break;
      next_item(at, q);
    }
  }
  __syncthreads();

  // ---- parts of items: over the warps of this CTA, then over CTAs ----------------------------------------------------------------
  if (tid == 0) {
    int k = 0;
    const int act = (int)min((long long)kWarps, workers - (long long)blockIdx.x * kWarps);
    for (int w = -1; w < act; ++w) {
      if (w < 0 ? !s_has_a[0] : !s_has_b[w])
        continue;
      Chain c;
      c.opened = w >= 0;
      c.at = w < 0 ? s_a[0] : s_b[w];
      c.first = max(w, 0);
      c.last = c.first;
      c.ends = w < 0 && s_a_ends[0];
      while (!c.ends && c.last + 1 < act) {
        ++c.last;
        c.ends = s_a_ends[c.last];
      }
      s_chain[k++] = c;
    }
    s_n_chains = k;
  }
  __syncthreads();
  auto part_of = [&](const Chain &c, int w) { return c.opened && w == c.first ? reinterpret_cast<const float *>(s_ring + w * RING) : s_part + w * PART; };
  for (int k = 0; k < s_n_chains; ++k) {
    const Chain c = s_chain[k];
    const Sequence q(p, c.at.s, room);
    const int live = rows_of(p, q, c.at.rt, c.at.slot);
    const bool whole = c.opened && c.ends;
    float *mine = p.parts + ((int64_t)blockIdx.x * 2 + c.opened) * PART;
    for (int i = tid; i < kRows * D / 4; i += kThreads) {
      const int row = i / (D / 4), d = i % (D / 4) * 4;
      float top = kSeed, l = 0.f;
      float4 o = make_float4(0.f, 0.f, 0.f, 0.f);
      for (int w = c.first; w <= c.last; ++w)
        top = fmaxf(top, part_of(c, w)[kRows * (D + 4) + row]);
      for (int w = c.first; w <= c.last; ++w) {
        const float *part = part_of(c, w), pl = part[kRows * (D + 4) + kRows + row], f = ex2(part[kRows * (D + 4) + row] - top);
        const float4 v = *reinterpret_cast<const float4 *>(part + row * (D + 4) + d);
        l = fmaf(pl, f, l);
        o = make_float4(fmaf(v.x, f, o.x), fmaf(v.y, f, o.y), fmaf(v.z, f, o.z), fmaf(v.w, f, o.w));
      }
      if (whole) {
        if (row < live) {
          const int64_t to = row_at(p, q.r0, c.at.rt, c.at.slot, row, p.a.out_ld, D) + d;
          const float over = l == 0.f ? 0.f : 1.f / l;
          put(p, to, l == 0.f ? 0.f : o.x * over);
          put(p, to + 1, l == 0.f ? 0.f : o.y * over);
          put(p, to + 2, l == 0.f ? 0.f : o.z * over);
          put(p, to + 3, l == 0.f ? 0.f : o.w * over);
        }
      } else {
        *reinterpret_cast<float4 *>(mine + row * (D + 4) + d) = o;
        if (d == 0) {
          mine[kRows * (D + 4) + row] = top;
          mine[kRows * (D + 4) + kRows + row] = l;
        }
      }
    }
    if (whole)
      continue;
    // the CTAs with parts of this item: those of its first and last tile's workers
    const long long begin = s_cost[c.at.s] + c.at.slot * q.before(q.tiles, p.tokens) + q.before(c.at.rt, p.tokens);
    const long long final = begin + 16ll * (item_tiles(q, c.at.rt) - 1);
    const int from = (int)((((begin + 1) * workers - 1) / total) / kWarps), to = (int)((((final + 1) * workers - 1) / total) / kWarps);
    __threadfence();
    __syncthreads();
    if (tid == 0) {
      const int before = atomicAdd(p.counters + from, 1);
      s_last = before == to - from;
      if (s_last)
        p.counters[from] = 0;
    }
    __syncthreads();
    if (!s_last)
      continue;
    __threadfence();
    for (int i = tid; i < kRows * D / 4; i += kThreads) {
      const int row = i / (D / 4), d = i % (D / 4) * 4;
      if (row >= live)
        continue;
      auto part = [&](int b) { return p.parts + ((int64_t)b * 2 + (b == from)) * PART; };
      float top = kSeed, l = 0.f;
      float4 o = make_float4(0.f, 0.f, 0.f, 0.f);
      for (int b = from; b <= to; ++b)
        top = fmaxf(top, __ldcg(part(b) + kRows * (D + 4) + row));
      for (int b = from; b <= to; ++b) {
        const float pl = __ldcg(part(b) + kRows * (D + 4) + kRows + row), f = ex2(__ldcg(part(b) + kRows * (D + 4) + row) - top);
        const float4 v = __ldcg(reinterpret_cast<const float4 *>(part(b) + row * (D + 4) + d));
        l = fmaf(pl, f, l);
        o = make_float4(fmaf(v.x, f, o.x), fmaf(v.y, f, o.y), fmaf(v.z, f, o.z), fmaf(v.w, f, o.w));
      }
      const int64_t at = row_at(p, q.r0, c.at.rt, c.at.slot, row, p.a.out_ld, D) + d;
      const float over = l == 0.f ? 0.f : 1.f / l;
      put(p, at, l == 0.f ? 0.f : o.x * over);
      put(p, at + 1, l == 0.f ? 0.f : o.y * over);
      put(p, at + 2, l == 0.f ? 0.f : o.z * over);
      put(p, at + 3, l == 0.f ? 0.f : o.w * over);
    }
  }
}

RaisedOn g_raised[6];

template <int D, int TYPE> int attention_launch(RaisedOn &raised, const AttentionParams &p, cudaStream_t st) {
  const int fixed = kWarps * (kStages * kv4_tile_bytes(D) + part_floats(D) * 4);
  if (int rc = raise_shared_limit(raised, (const void *)kv4_attention_kernel<D, TYPE>, fixed + 8 * (B200_KV4_ATTENTION_MAX_SEQS + 1)))
    return rc;
  return launch_after(kv4_attention_kernel<D, TYPE>, dim3(kCtas), kThreads, fixed + 8 * (p.a.n_seqs + 1), st, p);
}

} // namespace

} // namespace b200

using namespace b200;

extern "C" {

int64_t b200_kv4_attention_workspace_bytes(int q_heads, int kv_heads, int head_dim) {
  if (kv_heads < 1 || kv_heads > 1024 || q_heads < 1 || q_heads % kv_heads != 0 || (head_dim != 64 && head_dim != 128))
    return B200_EINVAL;
  return 2048 + (int64_t)kCtas * 2 * part_floats(head_dim) * 4;
}

int b200_kv4_attention(const b200_kv4_cache *c, const b200_kv4_attention_args *a, void *workspace, int64_t workspace_bytes, void *stream) {
  if (int rc = kv4_check("kv4_attention", c))
    return rc;
  if (!a || (a->rows > 0 && (!a->q || !a->out || !workspace || !a->row_start || !a->lens || !a->block_table)))
    return fail(B200_EINVAL, "kv4_attention: null pointer");
  if (a->dtype != B200_F32 && a->dtype != B200_F16 && a->dtype != B200_BF16)
    return fail(B200_EINVAL, "kv4_attention: element type %d", a->dtype);
  if (a->rows < 0 || a->n_seqs < 1 || a->table_stride < 1 || a->q_heads < 1 || a->q_heads % c->kv_heads != 0 || (int64_t)a->table_stride * c->page > INT32_MAX)
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
  AttentionParams p{(const uint8_t *)c->pool, c->n_pages, c->kv_heads, c->page, *a};
  p.G = a->q_heads / c->kv_heads;
  p.subs = (p.G + kRows - 1) / kRows;
  p.heads = std::min(p.G, kRows);
  p.tokens = p.subs == 1 ? kRows / p.G : 1;
  p.log2_scale = a->scale * 1.4426950408889634f;
  p.counters = (int *)workspace;
  p.parts = (float *)((char *)workspace + 2048);
  cudaStream_t st = (cudaStream_t)stream;
#define B200_D(D_)                                                                                                                    \
  (a->dtype == B200_F32   ? attention_launch<D_, B200_F32>(g_raised[D_ / 64 - 1], p, st)                                              \
   : a->dtype == B200_F16 ? attention_launch<D_, B200_F16>(g_raised[D_ / 64 + 1], p, st)                                              \
                          : attention_launch<D_, B200_BF16>(g_raised[D_ / 64 + 3], p, st))
  return c->head_dim == 128 ? B200_D(128) : B200_D(64);
#undef B200_D
}

} // extern "C"
