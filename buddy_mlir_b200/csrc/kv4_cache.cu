// The 4-bit KV cache's writer and reader (b200_kv4_write, b200_kv4_read).
//
// A lane has eight dims of a row's K or V, eight lanes a group of 64: a warp takes both groups of K and V of a head of 128 dims at once, or two heads
// of 64.  A group's extremes take three shuffles; eight dims of K are one word of codes, those of V, with a neighbour's, a byte for each of
// eight pairs of dims sixteen apart.  A code's quotient is a product and one correction (quotient.cuh), the same bits as a division.
// What bounds them is instructions (some 190 and 130 of a warp per 256 values), then bytes.
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
};

// eight elements of a row, with 16-byte loads where they are aligned
template <typename T, bool WIDE> __device__ __forceinline__ void load8(const T *p, float (&x)[8]) {
  if constexpr (WIDE && sizeof(T) == 4) {
    *reinterpret_cast<float4 *>(x) = *reinterpret_cast<const float4 *>(p);
    *reinterpret_cast<float4 *>(x + 4) = *reinterpret_cast<const float4 *>(p + 4);
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
    *reinterpret_cast<float4 *>(p) = make_float4(x[0], x[1], x[2], x[3]);
    *reinterpret_cast<float4 *>(p + 4) = make_float4(x[4], x[5], x[6], x[7]);
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

// Where a lane's eight dims lie: lanes 0 .. 15 have K's, the others V's; of a head of 128, or of two of 64.
template <int D> struct Place {
  int head, group, m;      // m: which eight dims of the group
  int j;                   // the position in its tile
  uint8_t *tile;           // null: no position of the pool
  __device__ __forceinline__ Place(const CacheParams &p, int row, int head_of) {
    const int lane = threadIdx.x & 31;
    m = lane & 7;
    group = D == 128 ? lane >> 3 & 1 : 0;
    head = D == 128 ? head_of : 2 * head_of + (lane >> 3 & 1);
    const int64_t slot = p.slots[row];
    if (slot < 0 || slot >= p.positions || head >= p.kv_heads) {
      tile = nullptr;
      j = 0;
      return;
    }
    const int64_t id = slot >> 31 ? slot / p.page : (int64_t)((uint32_t)slot / (uint32_t)p.page);
    const int off = (int)(slot - id * p.page);
    j = off % kKv4Tile;
    tile = p.pool + ((id * p.kv_heads + head) * (p.page / kKv4Tile) + off / kKv4Tile) * kv4_tile_bytes(D);
  }
  __device__ __forceinline__ int column() const { return head * D + group * kKv4Group + 8 * m; }
  __device__ __forceinline__ uint32_t *k_word() const { return reinterpret_cast<uint32_t *>(tile + j * (D / 2) + m % 4 * (D / 8) + (2 * group + m / 4) * 4); }
  // of V: of the first of the four pairs of dims that this lane stores or loads (64 bytes from one to the next)
  __device__ __forceinline__ uint8_t *v_bytes() const {
    return tile + kv4_v_codes(D) + group * 512 + (m & 1) * 256 + j % 8 / 2 * 16 + m / 2 * 4 + j % 2 * 2 + j / 8;
  }
  __device__ __forceinline__ uint32_t *pair(bool is_k) const {
    return reinterpret_cast<uint32_t *>(tile + (is_k ? kv4_k_pairs(D) : kv4_v_pairs(D)) + (j * (D / kKv4Group) + group) * 4);
  }
};

template <int D, typename T, bool WIDE> __global__ void __launch_bounds__(kThreads) kv4_write_kernel(const __grid_constant__ CacheParams p) {
  kernel_go();
  kernel_wait();
  const int lane = threadIdx.x & 31;
  const bool is_k = lane < 16;
  int row = blockIdx.x;
  for (int h = threadIdx.x >> 5; row < p.rows; h += kThreads / 32) {
    while (h >= p.heads) {
      h -= p.heads;
      row += gridDim.x;
    }
    if (row >= p.rows)
      break;
    const Place<D> g(p, row, h);
    float x[8], mn = kKv4Most, mx = -kKv4Most;
    bool nan = false;
    if (g.head < p.kv_heads) {
      load8<T, WIDE>((const T *)(is_k ? p.k : p.v) + row * (is_k ? p.k_ld : p.v_ld) + g.column(), x);
    } else {
#pragma unroll
      for (int i = 0; i < 8; ++i)
        x[i] = 0.f;
    }
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      nan = nan || x[i] != x[i];
      x[i] = fminf(fmaxf(x[i], -kKv4Most), kKv4Most);
      mn = fminf(mn, x[i]);
      mx = fmaxf(mx, x[i]);
    }
#pragma unroll
    for (int o = 4; o > 0; o >>= 1) {
      mn = fminf(mn, __shfl_xor_sync(0xffffffffu, mn, o));
      mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, o));
    }
    nan = __ballot_sync(0xffffffffu, nan) >> (lane & 24) & 0xff;
    const __half lo = __float2half_rn(mn), scale = __float2half_rn(__fdiv_rn(__fsub_rn(mx, __half2float(lo)), 15.f));
    const float l = __half2float(lo), s = __half2float(scale), b = s * 16777216.f, r = __frcp_rn(b);   // (b >= 1: the smallest scale is 2^-24)
    const bool some = s > 0.f && !nan;
    // dim 2 a + h of the eight: nibble a + 4 h
    uint32_t word = 0;
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      const float a = __fsub_rn(x[i], l) * 16777216.f, q = a * r, code = fmaf(fmaf(-b, q, a), r, q);
      // rounded as rint does: added to 1.5 * 2^23
      word |= (__float_as_uint(__fadd_rn(fminf(fmaxf(code, 0.f), 15.f), 12582912.f)) & 15u) << (is_k ? 4 * (i / 2 + 4 * (i & 1)) : 4 * i);
    }
    word = some ? word : 0;
    const uint32_t other = __shfl_xor_sync(0xffffffffu, word, 1);
    if (g.tile == nullptr)
      continue;
    if (is_k) {
      *g.k_word() = word;
    } else {   // dims 16 i + g (low nibbles: the even lane's) and 16 i + 8 + g: four pairs each
      const uint32_t low = g.m & 1 ? other >> 16 : word, high = g.m & 1 ? word >> 16 : other;
      uint8_t *v = g.v_bytes();
#pragma unroll
      for (int i = 0; i < 4; ++i)
        v[i * 64] = (uint8_t)((low >> (4 * i) & 15) | (high >> (4 * i) & 15) << 4);
    }
    if (g.m == 0)
      *g.pair(is_k) = nan ? 0x7e000000u : (uint32_t)__half_as_ushort(scale) | (uint32_t)__half_as_ushort(lo) << 16;
  }
}

template <int D, typename T, bool WIDE> __global__ void __launch_bounds__(kThreads) kv4_read_kernel(const __grid_constant__ CacheParams p) {
  kernel_go();
  kernel_wait();
  const int lane = threadIdx.x & 31;
  const bool is_k = lane < 16;
  int row = blockIdx.x;
  for (int h = threadIdx.x >> 5; row < p.rows; h += kThreads / 32) {
    while (h >= p.heads) {
      h -= p.heads;
      row += gridDim.x;
    }
    if (row >= p.rows)
      break;
    const Place<D> g(p, row, h);
    uint32_t word = 0, pair = 0;   // word of V: low nibbles (dims g) and high ones of this lane's four pairs
    if (g.tile != nullptr) {
      pair = *g.pair(is_k);
      if (is_k) {
        word = *g.k_word();
      } else {
        const uint8_t *v = g.v_bytes();
#pragma unroll
        for (int i = 0; i < 4; ++i)
          word |= (uint32_t)(v[i * 64] & 15) << (4 * i) | (uint32_t)(v[i * 64] >> 4) << (16 + 4 * i);
      }
    }
    const uint32_t other = __shfl_xor_sync(0xffffffffu, word, 1);
    if (g.head >= p.kv_heads)
      continue;
    if (!is_k)   // the even lane's dims are the low nibbles of both, the odd one's the high
      word = g.m & 1 ? other >> 16 | (word & 0xffff0000u) : (word & 0xffffu) | other << 16;
    const __half2 both = *reinterpret_cast<const __half2 *>(&pair);
    const float s = __low2float(both), l = __high2float(both);
    float x[8];
#pragma unroll
    for (int i = 0; i < 8; ++i)
      x[i] = fmaf(s, (float)(word >> (is_k ? 4 * (i / 2 + 4 * (i & 1)) : 4 * i) & 15), l);
    store8<T, WIDE>((T *)(is_k ? p.k : p.v) + row * (is_k ? p.k_ld : p.v_ld) + g.column(), x);
  }
}

template <bool WRITE> int cache_launch(const b200_kv4_cache &c, const void *k, int64_t k_ld, const void *v, int64_t v_ld, int dtype, const int64_t *slots,
                                       int rows, cudaStream_t st) {
  if (rows == 0)
    return B200_OK;
  const int heads = c.head_dim == 128 ? c.kv_heads : (c.kv_heads + 1) / 2, warps = kThreads / 32;
  const CacheParams p{(uint8_t *)c.pool, (int64_t)c.n_pages * c.page, c.kv_heads, c.page, (void *)k, (void *)v, k_ld, v_ld, slots, rows, heads};
  // a CTA takes rows that are the grid apart, its warps one head after the other
  const int64_t ctas = ((int64_t)rows * heads + warps - 1) / warps;
  const dim3 grid((unsigned)std::min<int64_t>(std::min<int64_t>(ctas, rows), 148 * 8));
  const int size = dtype == B200_F32 ? 4 : 2;
  const bool wide = (((uintptr_t)k | (uintptr_t)v | (uintptr_t)(k_ld * size) | (uintptr_t)(v_ld * size)) & 15) == 0;
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
