// The 4-bit KV cache's writer and reader (b200_kv4_write, b200_kv4_read).
//
// A lane has eight dims of a row's K or V, eight lanes a group of 64: a warp takes both groups of K and V of a head of 128 dims at once, or two heads
// of 64.  A group's extremes take three shuffles; eight dims of K are one word of codes, those of V, with a neighbour's, a byte for each of
// eight pairs of dims sixteen apart.  A code's quotient is a product and one correction (quotient.cuh), the same bits as a division.
// What bounds the writer is instructions: 231 of a warp per 256 values, issue slots 71 % full (16001 bf16 rows of 8 x 128: 37 us, 84 MB).  The reader has half as
// many and takes as long (149 MB as f32 with what it writes: 3.9 TB/s).
#include "kv4.cuh"
#include "quotient.cuh"

#include <algorithm>

namespace b200 {

namespace {

constexpr int kThreads = 256;

struct CacheParams {
  uint8_t *pool;
  int64_t positions;     // of the pool
  int kv_heads, page;
  void *k, *v;
  int64_t k_ld, v_ld;
  const int64_t *slots;
  int rows, heads;       // heads: pairs of them for D = 64
  int shares, per_share; // a row's heads are dealt to that many warps, so many each
};

// eight elements of a row, with one load or store where they are aligned to their size
template <typename T, bool WIDE> __device__ __forceinline__ void load8(const T *p, float (&x)[8]) {
  if constexpr (WIDE && sizeof(T) == 4) {
    asm volatile("ld.global.v8.f32 {%0,%1,%2,%3,%4,%5,%6,%7}, [%8];"
                 : "=f"(x[0]), "=f"(x[1]), "=f"(x[2]), "=f"(x[3]), "=f"(x[4]), "=f"(x[5]), "=f"(x[6]), "=f"(x[7])
                 : "l"(p)
                 : "memory");
  } else if constexpr (WIDE) {
    __align__(16) T e[8];
    *reinterpret_cast<uint4 *>(e) = *reinterpret_cast<const uint4 *>(p);
#pragma unroll
    for (int i = 0; i < 8; ++i)
      x[i] = (float)e[i];
  } else {
#pragma unroll
    for (int i = 0; i < 8; ++i)
      x[i] = (float)p[i];
  }
}
template <typename T, bool WIDE> __device__ __forceinline__ void store8(T *p, const float (&x)[8]) {
  if constexpr (WIDE && sizeof(T) == 4) {
    asm volatile("st.global.v8.f32 [%0], {%1,%2,%3,%4,%5,%6,%7,%8};" ::"l"(p), "f"(x[0]), "f"(x[1]), "f"(x[2]), "f"(x[3]), "f"(x[4]), "f"(x[5]),
                 "f"(x[6]), "f"(x[7])
                 : "memory");
  } else if constexpr (WIDE) {
    __align__(16) T e[8];
#pragma unroll
    for (int i = 0; i < 8; ++i)
      e[i] = (T)x[i];
    *reinterpret_cast<uint4 *>(p) = *reinterpret_cast<uint4 *>(e);
  } else {
#pragma unroll
    for (int i = 0; i < 8; ++i)
      p[i] = (T)x[i];
  }
}

__device__ __forceinline__ float least(float a, float b) {   // (a NaN stays)
  float y;
  asm("min.NaN.f32 %0, %1, %2;" : "=f"(y) : "f"(a), "f"(b));
  return y;
}
__device__ __forceinline__ float most(float a, float b) {
  float y;
  asm("max.NaN.f32 %0, %1, %2;" : "=f"(y) : "f"(a), "f"(b));
  return y;
}

// Where a lane's eight dims lie: lanes 0 .. 15 have K's, the others V's; of a head of 128, or of two of 64.
template <int D> struct Lane {
  int group, m, sub;       // m: which eight dims of the group; sub: which head of two
  bool is_k;
  int code, pair, column;  // bytes from the tile on: the lane's codes (V's: without the position), the pair; elements from the heads on
  __device__ __forceinline__ Lane() {
    const int lane = threadIdx.x & 31;
    is_k = lane < 16;
    m = lane & 7;
    group = D == 128 ? lane >> 3 & 1 : 0;
    sub = D == 128 ? 0 : lane >> 3 & 1;
    // V: of the first of the four pairs of dims that this lane stores or loads (64 bytes from one to the next)
    code = is_k ? m % 4 * (D / 8) + (2 * group + m / 4) * 4 : kv4_v_codes(D) + group * 512 + (m & 1) * 256 + m / 2 * 4;
    pair = (is_k ? kv4_k_pairs(D) : kv4_v_pairs(D)) + group * 4;
    column = sub * D + group * kKv4Group + 8 * m;
  }
  __device__ __forceinline__ int code_at(int j) const { return code + (is_k ? j * (D / 2) : j % 8 / 2 * 16 + j % 2 * 2 + j / 8); }
  __device__ __forceinline__ int pair_at(int j) const { return pair + j * (D / kKv4Group) * 4; }
};

// A warp's share: some heads of a row.
template <int D> struct Share {
  int row, head, end;
  int j;                   // the position in its tile
  uint8_t *tile;           // of the first head; null: no position of the pool
  int64_t step;            // to the next head's
  __device__ __forceinline__ Share(const CacheParams &p, int64_t at) {
    row = (int)(at / p.shares);
    head = (int)(at - (int64_t)row * p.shares) * p.per_share;
    end = min(head + p.per_share, p.heads);
    const int64_t slot = p.slots[row];
    step = (int64_t)(p.page / kKv4Tile) * kv4_tile_bytes(D);
    const int64_t id = slot >> 31 ? slot / p.page : (int64_t)((uint32_t)slot / (uint32_t)p.page);
    const int off = (int)(slot - id * p.page);
    j = off & (kKv4Tile - 1);
    tile = slot < 0 || slot >= p.positions ? nullptr : p.pool + id * p.kv_heads * step + off / kKv4Tile * kv4_tile_bytes(D);
  }
};

template <int D, typename T, bool WIDE> __global__ void __launch_bounds__(kThreads) kv4_write_kernel(const __grid_constant__ CacheParams p) {
  constexpr int HEADS = 128 / D;   // of a step
  kernel_go();
  kernel_wait();
  const Lane<D> me;
  for (int64_t at = (int64_t)blockIdx.x * (kThreads / 32) + (threadIdx.x >> 5); at < (int64_t)p.rows * p.shares; at += (int64_t)gridDim.x * (kThreads / 32)) {
    const Share<D> w(p, at);
    if (w.tile == nullptr)
      continue;
    const T *in = (const T *)(me.is_k ? p.k : p.v) + w.row * (me.is_k ? p.k_ld : p.v_ld) + me.column;
    const int code_at = me.code_at(w.j), pair_at = me.pair_at(w.j);
    for (int h = w.head; h < w.end; ++h) {
      const int head = HEADS * h + me.sub;
      float x[8];
      if (head < p.kv_heads) {
        load8<T, WIDE>(in + (int64_t)HEADS * h * D, x);
      } else {
#pragma unroll
        for (int i = 0; i < 8; ++i)
          x[i] = 0.f;
      }
      float mn = x[0], mx = x[0];
#pragma unroll
      for (int i = 1; i < 8; ++i) {
        mn = least(mn, x[i]);
        mx = most(mx, x[i]);
      }
#pragma unroll
      for (int o = 4; o > 0; o >>= 1) {
        mn = least(mn, __shfl_xor_sync(0xffffffffu, mn, o));
        mx = most(mx, __shfl_xor_sync(0xffffffffu, mx, o));
      }
      if (__any_sync(0xffffffffu, mx > kKv4Most || mn < -kKv4Most)) {   // (rare)
        mn = most(least(mn, kKv4Most), -kKv4Most);
        mx = most(least(mx, kKv4Most), -kKv4Most);
#pragma unroll
        for (int i = 0; i < 8; ++i)
          x[i] = most(least(x[i], kKv4Most), -kKv4Most);
      }
      const bool nan = mn != mn;
      const __half lo = __float2half_rn(mn);
      const float l = __half2float(lo), range = __fsub_rn(mx, l), over15 = 1.f / 15.f;
      const __half scale = __float2half_rn(quotient(range, 15.f, over15));
      // The quotient's steps hold for any scale of the format (2^-24 at least) but for numerators below 2^-100, whose code is 0 either way.
      const float s = __half2float(scale), r = __frcp_rn(s);
      uint32_t c[8];
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        const float a = __fsub_rn(x[i], l), q = a * r, code = fmaf(fmaf(-s, q, a), r, q);
        c[i] = __float_as_uint(__fadd_rn(fminf(fmaxf(code, 0.f), 15.f), 12582912.f));   // rounded as rint does, in the low byte
      }
      // K: dim 2 a + h of the eight is nibble a + 4 h; V: dim i is nibble i
      uint32_t word = me.is_k ? __byte_perm(__byte_perm(c[0] + (c[2] << 4), c[4] + (c[6] << 4), 0x0040), __byte_perm(c[1] + (c[3] << 4), c[5] + (c[7] << 4), 0x0040), 0x5410)
                              : __byte_perm(__byte_perm(c[0] + (c[1] << 4), c[2] + (c[3] << 4), 0x0040), __byte_perm(c[4] + (c[5] << 4), c[6] + (c[7] << 4), 0x0040), 0x5410);
      word = s > 0.f && !nan ? word : 0;
      const uint32_t other = __shfl_xor_sync(0xffffffffu, word, 1);
      if (head >= p.kv_heads)
        continue;
      uint8_t *tile = w.tile + head * w.step;
      if (me.is_k) {
        *reinterpret_cast<uint32_t *>(tile + code_at) = word;
      } else {   // dims 16 i + g (low nibbles: the even lane's) and 16 i + 8 + g: four pairs each
        const uint32_t low = me.m & 1 ? other >> 16 : word, high = me.m & 1 ? word >> 16 : other;
        // nibbles of two half-words, interleaved: bytes 0 and 2 of `even`, then of `odd`
        const uint32_t even = (low & 0x0f0f) | (high & 0x0f0f) << 4, odd = (low >> 4 & 0x0f0f) | (high & 0xf0f0);
        tile[code_at] = (uint8_t)even;
        tile[code_at + 64] = (uint8_t)odd;
        tile[code_at + 128] = (uint8_t)(even >> 8);
        tile[code_at + 192] = (uint8_t)(odd >> 8);
      }
      if (me.m == 0)
        *reinterpret_cast<uint32_t *>(tile + pair_at) = nan ? 0x7e000000u : (uint32_t)__half_as_ushort(scale) | (uint32_t)__half_as_ushort(lo) << 16;
    }
  }
}

template <int D, typename T, bool WIDE> __global__ void __launch_bounds__(kThreads) kv4_read_kernel(const __grid_constant__ CacheParams p) {
  constexpr int HEADS = 128 / D;
  kernel_go();
  kernel_wait();
  const Lane<D> me;
  for (int64_t at = (int64_t)blockIdx.x * (kThreads / 32) + (threadIdx.x >> 5); at < (int64_t)p.rows * p.shares; at += (int64_t)gridDim.x * (kThreads / 32)) {
    const Share<D> w(p, at);
    T *out = (T *)(me.is_k ? p.k : p.v) + w.row * (me.is_k ? p.k_ld : p.v_ld) + me.column;
    const int code_at = me.code_at(w.j), pair_at = me.pair_at(w.j);
#pragma unroll 2
    for (int h = w.head; h < w.end; ++h) {
      const int head = HEADS * h + me.sub;
      uint32_t word = 0, pair = 0;   // word of V: dims g (low half) and g + 8 of this lane's four pairs
      if (w.tile != nullptr && head < p.kv_heads) {
        const uint8_t *tile = w.tile + head * w.step;
        pair = *reinterpret_cast<const uint32_t *>(tile + pair_at);
        if (me.is_k) {
          word = *reinterpret_cast<const uint32_t *>(tile + code_at);
        } else {
          const uint32_t even = tile[code_at] | (uint32_t)tile[code_at + 128] << 8, odd = tile[code_at + 64] | (uint32_t)tile[code_at + 192] << 8;
          word = (even & 0x0f0f) | (odd & 0x0f0f) << 4 | (even & 0xf0f0) << 12 | (odd & 0xf0f0) << 16;
        }
      }
      const uint32_t other = __shfl_xor_sync(0xffffffffu, word, 1);
      if (head >= p.kv_heads)
        continue;
      if (!me.is_k)   // the even lane's dims are the low nibbles of both, the odd one's the high
        word = me.m & 1 ? other >> 16 | (word & 0xffff0000u) : (word & 0xffffu) | other << 16;
      const __half2 both = *reinterpret_cast<const __half2 *>(&pair);
      const float s = __low2float(both), l = __high2float(both);
      // in the order of K's nibbles: dims 0 2 4 6 1 3 5 7
      float c[8], x[8];
#pragma unroll
      for (int i = 0; i < 8; ++i)   // (a code as 2^23 + c, less 2^23)
        c[i] = fmaf(s, __uint_as_float((word >> (4 * i) & 15) | 0x4b000000u) - 8388608.f, l);
#pragma unroll
      for (int i = 0; i < 8; ++i)
        x[i] = me.is_k ? c[i / 2 + 4 * (i & 1)] : c[i];
      store8<T, WIDE>(out + (int64_t)HEADS * h * D, x);
    }
  }
}

template <bool WRITE> int cache_launch(const b200_kv4_cache &c, const void *k, int64_t k_ld, const void *v, int64_t v_ld, int dtype, const int64_t *slots,
                                       int rows, cudaStream_t st) {
  if (rows == 0)
    return B200_OK;
  // a warp takes a row's heads one after the other, as many of them as leave every SM 16 warps
  const int heads = c.head_dim == 128 ? c.kv_heads : (c.kv_heads + 1) / 2, warps = kThreads / 32;
  const int per_share = (int)std::min<int64_t>(heads, std::max<int64_t>(1, (int64_t)rows * heads / (148 * 16))), shares = (heads + per_share - 1) / per_share;
  const CacheParams p{(uint8_t *)c.pool, (int64_t)c.n_pages * c.page, c.kv_heads, c.page, (void *)k, (void *)v, k_ld, v_ld, slots, rows, heads, shares, per_share};
  const dim3 grid((unsigned)std::min<int64_t>(((int64_t)rows * shares + warps - 1) / warps, 148 * 64));
  const int size = dtype == B200_F32 ? 4 : 2;
  const bool wide = (((uintptr_t)k | (uintptr_t)v | (uintptr_t)(k_ld * size) | (uintptr_t)(v_ld * size)) & (8 * size - 1)) == 0;
#define B200_KERNEL(D, T, W) (WRITE ? kv4_write_kernel<D, T, W> : kv4_read_kernel<D, T, W>)
#define B200_TYPE(T)                                                                                                                            \
  launch_after(c.head_dim == 128 ? (wide ? B200_KERNEL(128, T, true) : B200_KERNEL(128, T, false)) : (wide ? B200_KERNEL(64, T, true) : B200_KERNEL(64, T, false)), \
               grid, kThreads, 0, st, p)
  return dtype == B200_F32 ? B200_TYPE(float) : dtype == B200_F16 ? B200_TYPE(__half) : B200_TYPE(__nv_bfloat16);
#undef B200_TYPE
#undef B200_KERNEL
}

int check_rows(const char *call, const b200_kv4_cache *c, const void *k, int64_t k_ld, const void *v, int64_t v_ld, int dtype, const int64_t *slots,
               int rows) {
  if (int rc = kv4_check(call, c))
    return rc;
  if (dtype != B200_F32 && dtype != B200_F16 && dtype != B200_BF16)
    return fail(B200_EINVAL, "%s: element type %d", call, dtype);
  if (rows < 0)
    return fail(B200_EINVAL, "%s: %d rows", call, rows);
  if (rows > 0 && (!k || !v || !slots))
    return fail(B200_EINVAL, "%s: null pointer", call);
  const int64_t cols = (int64_t)c->kv_heads * c->head_dim;
  if (rows > 1 && (k_ld < cols || v_ld < cols))
    return fail(B200_EINVAL, "%s: row strides %lld and %lld of rows of %lld", call, (long long)k_ld, (long long)v_ld, (long long)cols);
  const uintptr_t mask = dtype == B200_F32 ? 3 : 1;
  if (((uintptr_t)k | (uintptr_t)v) & mask || (uintptr_t)slots & 7)
    return fail(B200_EINVAL, "%s: a pointer is not aligned to its elements", call);
  return ensure_device();
}

} // namespace

int kv4_check(const char *call, const b200_kv4_cache *c) {
  if (!c || !c->pool)
    return fail(B200_EINVAL, "%s: null pointer", call);
  if (b200_kv4_pool_bytes(c->n_pages, c->kv_heads, c->head_dim, c->page) < 0)
    return fail(B200_EINVAL, "%s: no cache of %d pages of %d positions, %d heads of %d (64 or 128 dims, pages of a multiple of 16 up to 65536)", call,
                c->n_pages, c->page, c->kv_heads, c->head_dim);
  if ((uintptr_t)c->pool & 15)
    return fail(B200_EINVAL, "%s: the pool is not aligned to 16 bytes", call);
  return B200_OK;
}

int kv4_write_launch(const b200_kv4_cache &c, const void *k, int64_t k_ld, const void *v, int64_t v_ld, int dtype, const int64_t *slots, int rows,
                     cudaStream_t st) {
  return cache_launch<true>(c, k, k_ld, v, v_ld, dtype, slots, rows, st);
}

} // namespace b200

using namespace b200;

extern "C" {

int64_t b200_kv4_pool_bytes(int n_pages, int kv_heads, int head_dim, int page) {
  if (n_pages < 1 || kv_heads < 1 || kv_heads > 1024 || (head_dim != 64 && head_dim != 128) || page < kKv4Tile || page % kKv4Tile != 0 || page > 65536 ||
      (int64_t)n_pages * kv_heads * (page / kKv4Tile) > INT32_MAX)
    return B200_EINVAL;
  return (int64_t)n_pages * kv_heads * (page / kKv4Tile) * kv4_tile_bytes(head_dim);
}

int b200_kv4_write(const b200_kv4_cache *c, const void *k, int64_t k_ld, const void *v, int64_t v_ld, int dtype, const int64_t *slots, int rows,
                   void *stream) {
  if (int rc = check_rows("kv4_write", c, k, k_ld, v, v_ld, dtype, slots, rows))
    return rc;
  return kv4_write_launch(*c, k, k_ld, v, v_ld, dtype, slots, rows, (cudaStream_t)stream);
}

int b200_kv4_read(const b200_kv4_cache *c, void *k, int64_t k_ld, void *v, int64_t v_ld, int dtype, const int64_t *slots, int rows, void *stream) {
  if (int rc = check_rows("kv4_read", c, k, k_ld, v, v_ld, dtype, slots, rows))
    return rc;
  return cache_launch<false>(*c, k, k_ld, v, v_ld, dtype, slots, rows, (cudaStream_t)stream);
}

} // extern "C"
