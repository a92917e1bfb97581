// How the attention kernels over the 4-bit cache share out their work: sequences cut into items, the items' keys dealt evenly to CTAs, whatever the
// sequences' lengths (known on the device only).
#pragma once
#include "kv4.cuh"

#include <climits>

namespace b200 {

constexpr int kKv4Ctas = 148;          // of a launch at most
constexpr int kKv4Snap = 256;          // keys that a CTA may have more or fewer, so that it begins with an item (few of many: a quarter)
constexpr int kKv4Many = 4096;
constexpr int kKv4Item = 48;           // keys that take as long as beginning and ending an item
constexpr float kKv4Top = 8.f;         // powers of two: what the largest weight that meets codes is at when a row's reference is set,
constexpr float kKv4Lag = 4.f;         // and how far above that one may come before it is set again
constexpr float kKv4Seed = -3.402823466e38f;   // a row's reference before its first key: no finite score lies below
// Scores from here on are their own reference: a step of f32 is as large as kKv4Top there, and weights must neither vanish nor leave f16 by how a sum was rounded.
constexpr float kKv4Far = 16777216.f;

struct Kv4Params {
  const uint8_t *pool;
  int n_pages, kv_heads, page;
  b200_kv4_attention_args a;
  int G;                            // q heads of a kv head
  int heads, tokens, subs;          // of an item: q heads, positions; items that share a position's kv head
  int over_heads;                   // 2^16 / heads, rounded up
  int least_rows, most_rows;        // sequences of this launch: by their rows
  int many_rows;                    // from how many rows on a sequence counts as one of many;
  long long least_work;             // where less work than this is in those (rows times keys), the few-rows form has them too (0: not looked at)
  bool many;                        // this launch is the many-rows form
  int fill;                         // 1: rows of no sequence are zeroed here
  float log2_scale;
  bool wide_q, wide_out, wide_q16;  // rows are aligned to four elements; to 16 bytes
  int *counters;                    // [kKv4Ctas], then an error word
  float *parts;
};

__device__ __forceinline__ int clamp(long long x, int lo, int hi) { return (int)(x < lo ? lo : x > hi ? hi : x); }
__device__ __forceinline__ float ex2(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}
// Whether a row's reference moves for a score of `top`, and where to.  (By their difference, which is exact where they are near each other.)
__device__ __forceinline__ bool kv4_moves(float top, float r) { return top - r > kKv4Top + kKv4Lag; }
__device__ __forceinline__ float kv4_reference(float top) { return fabsf(top) < kKv4Far ? top - kKv4Top : top; }
__device__ __forceinline__ float power(int e) { return __uint_as_float((uint32_t)(127 + e) << 23); }
__device__ __forceinline__ uint32_t pack_f16(float lo, float hi) {
  uint32_t r;
  asm("cvt.rn.f16x2.f32 %0, %1, %2;" : "=r"(r) : "f"(hi), "f"(lo));
  return r;
}
__device__ __forceinline__ float2 halves(uint32_t pair) { return __half22float2(*reinterpret_cast<const __half2 *>(&pair)); }
// two f32 at once
__device__ __forceinline__ uint64_t pack2(float a, float b) {
  uint64_t r;
  asm("mov.b64 %0, {%1, %2};" : "=l"(r) : "f"(a), "f"(b));
  return r;
}
__device__ __forceinline__ float2 unpack2(uint64_t x) {
  float2 r;
  asm("mov.b64 {%0, %1}, %2;" : "=f"(r.x), "=f"(r.y) : "l"(x));
  return r;
}
__device__ __forceinline__ uint64_t fma_2(uint64_t a, uint64_t b, uint64_t c) {
  uint64_t r;
  asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(r) : "l"(a), "l"(b), "l"(c));
  return r;
}
__device__ __forceinline__ uint64_t add_2(uint64_t a, uint64_t b) {
  uint64_t r;
  asm("add.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b));
  return r;
}
__device__ __forceinline__ uint64_t mul_2(uint64_t a, uint64_t b) {
  uint64_t r;
  asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b));
  return r;
}
template <int TYPE> __device__ __forceinline__ void put(const Kv4Params &p, int64_t at, float x) {
  if constexpr (TYPE == B200_F32)
    ((float *)p.a.out)[at] = x;
  else if constexpr (TYPE == B200_F16)
    ((__half *)p.a.out)[at] = __float2half_rn(x);
  else
    ((__nv_bfloat16 *)p.a.out)[at] = __float2bfloat16_rn(x);
}
template <int TYPE> __device__ __forceinline__ void put4(const Kv4Params &p, int64_t at, float4 x) {
  if (!p.wide_out) {
    put<TYPE>(p, at, x.x);
    put<TYPE>(p, at + 1, x.y);
    put<TYPE>(p, at + 2, x.z);
    put<TYPE>(p, at + 3, x.w);
  } else if constexpr (TYPE == B200_F32) {
    *reinterpret_cast<float4 *>((float *)p.a.out + at) = x;
  } else if constexpr (TYPE == B200_F16) {
    *reinterpret_cast<uint2 *>((__half *)p.a.out + at) = make_uint2(pack_f16(x.x, x.y), pack_f16(x.z, x.w));
  } else {
    uint32_t lo, hi;
    asm("cvt.rn.bf16x2.f32 %0, %1, %2;" : "=r"(lo) : "f"(x.y), "f"(x.x));
    asm("cvt.rn.bf16x2.f32 %0, %1, %2;" : "=r"(hi) : "f"(x.w), "f"(x.z));
    *reinterpret_cast<uint2 *>((__nv_bfloat16 *)p.a.out + at) = make_uint2(lo, hi);
  }
}
// four elements of q, aligned
template <int TYPE> __device__ __forceinline__ void load_wide(const void *q, int64_t at, float (&x)[4]) {
  if constexpr (TYPE == B200_F32) {
    *reinterpret_cast<float4 *>(x) = *reinterpret_cast<const float4 *>((const float *)q + at);
  } else {
    const uint2 v = *reinterpret_cast<const uint2 *>((const uint16_t *)q + at);
#pragma unroll
    for (int e = 0; e < 2; ++e) {
      const uint32_t w = e ? v.y : v.x;
      const float2 f = TYPE == B200_F16 ? halves(w) : make_float2(__uint_as_float(w << 16), __uint_as_float(w & 0xffff0000u));
      x[2 * e] = f.x;
      x[2 * e + 1] = f.y;
    }
  }
}

// A sequence as its items: its rows `tokens` at a time and, for each kv head (or part of its q heads), a range of keys that ends at the last
// row's own position.  Cost of an item: its keys, and some more for its beginning and end; of all items before it in a head: before().
struct Sequence {
  int r0, n;            // rows
  int base;             // position of the first row (negative: rows before it see nothing), at most the table's room
  int past, tiles;      // max(base, 0); row tiles
  __device__ __forceinline__ Sequence(int first, int end, int position, int tokens) : r0(first), n(max(end - first, 0)), base(position) {
    past = max(base, 0);
    tiles = n <= tokens ? min(n, 1) : (n + tokens - 1) / tokens;
  }
  template <typename I = long long> __device__ __forceinline__ I before(int rt, int tokens) const {
    return rt == 0 ? 0
           : rt < tiles ? (I)rt * (past + kKv4Item) + (I)tokens * rt * (rt + 1) / 2
                        : (I)tiles * (past + kKv4Item) + (I)tokens * tiles * (tiles - 1) / 2 + n;
  }
};
// x * a / b, rounded down, for a <= b up to 2^15
template <typename I> __device__ __forceinline__ I share(I x, int a, int b) {
  if constexpr (sizeof(I) == 4) {
    const uint32_t q = (uint32_t)x / (uint32_t)b, r = (uint32_t)x - q * b;
    return (I)(q * a + r * a / (uint32_t)b);
  } else {
    return x / b * a + x % b * a / b;
  }
}

// Rows times keys of the sequences of many rows, by all THREADS of the CTA.  (Out of the way of the kernels' code.)
template <int THREADS> __device__ __noinline__ unsigned long long many_work(const Kv4Params &p, long long *sums) {
  const int room = p.a.table_stride * p.page;
  unsigned long long work = 0;
  for (int s = threadIdx.x; s < p.a.n_seqs; s += THREADS) {
    const int rows = max(clamp(p.a.row_start[s + 1], 0, p.a.rows) - clamp(p.a.row_start[s], 0, p.a.rows), 0);
    if (rows >= p.many_rows)
      work += (unsigned long long)rows * (unsigned)(clamp((long long)p.a.lens[s] - rows, 0, room) + rows / 2);
  }
#pragma unroll
  for (int o = 1; o < 32; o <<= 1)
    work += __shfl_xor_sync(0xffffffffu, work, o);
  if (threadIdx.x % 32 == 0)
    sums[threadIdx.x / 32] = (long long)work;
  __syncthreads();
  work = 0;
  for (int w = 0; w < THREADS / 32; ++w)
    work += (unsigned long long)sums[w];
  __syncthreads();
  return work;
}

// An item and the first of its tiles that is meant.
struct Place {
  int s, slot, rt, tile;
};

// SHIFT: log2 of a tile's keys.  An item that CTAs share costs them what some `split` keys do (its parts' way through L2): where whole items leave
// nobody with that much more than an even share, CTAs have whole items.
template <int SHIFT> struct KeyPlan {
  const long long *cost;   // [n + 1], in shared memory as the others
  const int *r0, *base;    // [n + 1], [n]: a sequence's rows, and the position of the first
  const int *items;        // [n + 1]: items before it
  int n, tokens, slots, ctas, window;
  bool whole, small;       // small: sums fit 32 bits (with room for one more item)
  long long total;
  static constexpr int kNone = 1 << 30;   // more items than are counted

  static __host__ __device__ constexpr int bytes(int n) { return 20 * (n + 1); }

  // By all THREADS of the CTA; sums: 2 * THREADS / 32 + 1 words of shared memory.
  template <int THREADS> __device__ __forceinline__ void build(const Kv4Params &p, void *memory, long long *sums, int least_keys, int split) {
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, room = p.a.table_stride * p.page;
    n = p.a.n_seqs;
    tokens = p.tokens;
    slots = p.kv_heads * p.subs;
    long long *s_cost = reinterpret_cast<long long *>(memory);
    int *s_r0 = reinterpret_cast<int *>(s_cost + n + 1), *s_base = s_r0 + n + 1, *s_items = s_base + n;
    const int per = (n + THREADS - 1) / THREADS, first = min(n, tid * per), last = min(n, first + per);
    int least_rows = p.least_rows, most_rows = p.most_rows;
    if (p.least_work > 0) {   // (both launches come to the same)
      const unsigned long long work = many_work<THREADS>(p, sums);
      if (work < (unsigned long long)p.least_work) {
        least_rows = p.many ? INT_MAX : 0;
        most_rows = INT_MAX;
      }
    }
    long long sum = 0;
    int count = 0, most = 0;
    for (int s = first; s < last; ++s) {
      const int a = clamp(p.a.row_start[s], 0, p.a.rows), b = clamp(p.a.row_start[s + 1], 0, p.a.rows), rows = max(b - a, 0);
      const int at = clamp((long long)p.a.lens[s] - rows, -rows, room);
      s_r0[s] = a;
      s_base[s] = at;
      if (s == n - 1)
        s_r0[n] = b;
      const Sequence q(a, b, at, tokens);
      s_cost[s] = sum;
      s_items[s] = count;
      if (rows >= least_rows && rows <= most_rows) {
        sum += slots * q.before(q.tiles, tokens);
        count = (int)min((long long)count + (long long)slots * q.tiles, (long long)kNone);
        most = max(most, q.past + rows + kKv4Item);
      }
    }
    const int busy = (n - 1) / per / 32;   // the last warp with a sequence
    if (warp <= busy) {
      long long upto = sum;
      int upto_items = count;
#pragma unroll
      for (int o = 1; o < 32; o <<= 1) {
        const long long v = __shfl_up_sync(0xffffffffu, upto, o);
        const int i = __shfl_up_sync(0xffffffffu, upto_items, o);
        if (lane >= o) {
          upto += v;
          upto_items = min(upto_items, kNone) + min(i, kNone);
        }
      }
      upto_items = min(upto_items, kNone);
      most = __reduce_max_sync(0xffffffffu, most);
      if (lane == 31) {
        sums[warp] = upto;
        sums[THREADS / 32 + warp] = (long long)upto_items << 32 | (uint32_t)most;
      }
      sum = upto - sum;
      count = upto_items - count;
    }
    __syncthreads();
    long long before = 0, all = 0;
    int before_items = 0, all_items = 0;
    most = 0;
    for (int w = 0; w <= busy; ++w) {
      if (w == warp) {
        before = all;
        before_items = all_items;
      }
      all += sums[w];
      all_items = min(all_items + (int)(sums[THREADS / 32 + w] >> 32), kNone);
      most = max(most, (int)(uint32_t)sums[THREADS / 32 + w]);
    }
    if (warp <= busy)
      for (int s = first; s < last; ++s) {
        s_cost[s] += before + sum;
        s_items[s] += before_items + count;
      }
    if (tid == 0) {
      s_cost[n] = all;
      s_items[n] = all_items;
    }
    __syncthreads();
    cost = s_cost;
    r0 = s_r0;
    base = s_base;
    items = s_items;
    total = all;
    small = total < (1ll << 30);
    ctas = total >= (long long)gridDim.x * least_keys ? gridDim.x : max(1, (int)total / least_keys);
    const long long chunk = small ? (int)total / ctas : total / ctas;
    window = chunk > kKv4Many ? kKv4Snap / 4 : (int)min((long long)kKv4Snap, chunk / 2 - 1);
    const int each = (all_items + (int)gridDim.x - 1) / (int)gridDim.x;
    whole = all_items < kNone && (long long)each * most <= chunk + split;
    if (whole)
      ctas = max(1, min((int)gridDim.x, all_items));
  }
  __device__ __forceinline__ Sequence sequence(int s) const { return Sequence(r0[s], r0[s + 1], base[s], tokens); }
  __device__ __forceinline__ int item_keys(const Sequence &q, int rt) const { return q.past + min((rt + 1) * tokens, q.n); }
  __device__ __forceinline__ int item_tiles(const Sequence &q, int rt) const { return (item_keys(q, rt) + (1 << SHIFT) - 1) >> SHIFT; }
  // the item with key x of all, from begin to end; at.tile: the first tile from x on (none of the item's, if x lies in its last or behind it)
  template <typename I> __device__ __forceinline__ void locate_in(I x, Place &at, I &begin, I &end) const {
    int lo = 0, hi = n;
    while (hi - lo > 1) {
      const int mid = (lo + hi) >> 1;
      if ((I)cost[mid] <= x)
        lo = mid;
      else
        hi = mid;
    }
    at.s = lo;
    const Sequence q = sequence(lo);
    begin = (I)cost[lo];
    if constexpr (sizeof(I) == 4) {
      const I head = q.template before<I>(q.tiles, tokens);
      at.slot = (uint32_t)(x - begin) / (uint32_t)head;
      begin += at.slot * head;
    } else {
      const I head = q.template before<I>(q.tiles, tokens);
      at.slot = (int)((x - begin) / head);
      begin += at.slot * head;
    }
    int a = 0, b = q.tiles;
    while (b - a > 1) {
      const int mid = (a + b) >> 1;
      if (q.template before<I>(mid, tokens) <= x - begin)
        a = mid;
      else
        b = mid;
    }
    at.rt = a;
    end = begin + q.template before<I>(a + 1, tokens);
    begin += q.template before<I>(a, tokens);
    at.tile = (int)((x - begin + (1 << SHIFT) - 1) >> SHIFT);
  }
  __device__ __forceinline__ Place locate(long long x) const {
    Place at;
    if (small) {
      int begin, end;
      locate_in<int>((int)x, at, begin, end);
    } else {
      long long begin, end;
      locate_in<long long>(x, at, begin, end);
    }
    return at;
  }
  template <typename I> __device__ __forceinline__ long long border_in(int c) const {
    const I x = share<I>((I)total, c, ctas);
    Place at;
    I begin, end;
    locate_in<I>(x, at, begin, end);
    return x - begin <= end - x ? (x - begin <= window ? begin : x) : end - x <= window ? end : x;
  }
  // where CTA c begins: at its share of all keys, or at the item border next to that
  __device__ __forceinline__ long long border(int c) const {
    if (c <= 0 || c >= ctas)
      return c <= 0 ? 0 : total;
    if (whole) {
      const int i = share<int>(items[n], c, ctas);
      int lo = 0, hi = n;
      while (hi - lo > 1) {
        const int mid = (lo + hi) >> 1;
        if (items[mid] <= i)
          lo = mid;
        else
          hi = mid;
      }
      const Sequence q = sequence(lo);
      const int slot = q.tiles == 1 ? i - items[lo] : (i - items[lo]) / q.tiles;
      return cost[lo] + slot * q.before(q.tiles, tokens) + q.before(i - items[lo] - slot * q.tiles, tokens);
    }
    return small ? border_in<int>(c) : border_in<long long>(c);
  }
  // where part c of n of a range of `mine` keys begins
  __device__ __forceinline__ long long part_of(long long mine, int c, int of) const {
    return small ? (long long)share<int>((int)mine, c, of) : share<long long>(mine, c, of);
  }
  __device__ __forceinline__ int nominal(long long x) const { return (int)(((x + 1) * ctas - 1) / total); }   // the CTA that x would lie in without that
  __device__ __forceinline__ void next_item(Place &at, const Sequence &q) const {
    at.tile = 0;
    if (++at.rt < q.tiles)
      return;
    at.rt = 0;
    if (++at.slot < slots)
      return;
    at.slot = 0;
    do
      ++at.s;
    while (at.s < n && cost[at.s + 1] == cost[at.s]);
  }
  // The tiles of an item are counted as its parts arrive, in the counter of the CTA that would begin it were there no borders moved (no two items
  // that are shared have the same).  By a whole warp, `tiles` of them having arrived and being visible: true for who completes the item, with the
  // CTAs of its first and last part.
  __device__ __forceinline__ bool arrive(int *counters, const Place &item, int tiles, int &from, int &to) const {
    const int lane = threadIdx.x & 31;
    const Sequence q = sequence(item.s);
    const int all = item_tiles(q, item.rt);
    const long long first = cost[item.s] + item.slot * q.before(q.tiles, tokens) + q.before(item.rt, tokens), last = first + ((long long)(all - 1) << SHIFT);
    from = nominal(first);
    to = nominal(last);
    int before = 0;
    if (lane == 0)
      before = atomicAdd(counters + from, tiles);
    if (__shfl_sync(0xffffffffu, before, 0) + tiles != all)
      return false;
    if (lane == 0)
      counters[from] = 0;
    const long long x = border(lane == 0 ? from + 1 : lane == 1 ? to : to + 1);   // (a lane each)
    const bool later = __shfl_sync(0xffffffffu, (int)(x <= first), 0), sooner = __shfl_sync(0xffffffffu, (int)(x > last), 1),
               beyond = __shfl_sync(0xffffffffu, (int)(x <= last), 2);
    from += later;
    to += beyond - sooner;
    return true;
  }
};

// element of a row in q (ld: q's) or out, before its dims: row i (0 .. 127) of the position `token` and on, of an item's heads
__device__ __forceinline__ int64_t row_at(const Kv4Params &p, int token, int slot, int i, int64_t ld, int D) {
  const int kv = p.subs == 1 ? slot : slot / p.subs, behind = i * p.over_heads >> 16;   // i / heads
  return (token + behind) * ld + (int64_t)(kv * p.G + (slot - kv * p.subs - behind) * p.heads + i) * D;
}
// number of a tile of sixteen keys of a sequence in the pool, or -1
__device__ __forceinline__ int tile_source(const Kv4Params &p, int s, int kv, int t) {
  const int per_page = p.page / kKv4Tile, id = p.a.block_table[(int64_t)s * p.a.table_stride + t / per_page];
  return id < 0 || id >= p.n_pages ? -1 : (id * p.kv_heads + kv) * per_page + t % per_page;
}

// sequences of many rows, on tcgen05: kv4_chunk.cu (bf16), kv4_exact.cu (f32 and f16)
int64_t kv4_chunk_part_floats(int D);   // of a CTA's two parts
bool kv4_chunk_takes(int G, int n_seqs);
int kv4_chunk_launch(Kv4Params p, int D, cudaStream_t st);
bool kv4_exact_takes(int G, int n_seqs);
int kv4_exact_launch(Kv4Params p, int D, cudaStream_t st);

} // namespace b200
