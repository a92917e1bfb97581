// The 4-bit KV cache's writer and reader (b200_kv4_write, b200_kv4_read).
//
// A half-warp has a group of 64 dims of one row and head, four dims a lane: its extremes by four shuffles, lo and the scale rounded to
// f16, the codes by one division each.
#include "kv4.cuh"

namespace b200 {

namespace {

constexpr int kThreads = 256;

struct CacheParams {
  uint8_t *pool;
  int64_t positions;     // of the pool
  int kv_heads, D, page;
  void *k, *v;
  int64_t k_ld, v_ld;
  const int64_t *slots;
  int64_t groups;        // rows * kv heads * D / 64
};

template <typename T> struct Four {   // four elements of a row, with one load where they are aligned
  T e[4];
};
template <typename T, bool WIDE> __device__ __forceinline__ void load4(const T *p, float (&x)[4]) {
  Four<T> v;
  if constexpr (WIDE && sizeof(T) == 4)
    *reinterpret_cast<uint4 *>(&v) = *reinterpret_cast<const uint4 *>(p);
  else if constexpr (WIDE)
    *reinterpret_cast<uint2 *>(&v) = *reinterpret_cast<const uint2 *>(p);
  else
    for (int i = 0; i < 4; ++i)
      v.e[i] = p[i];
#pragma unroll
  for (int i = 0; i < 4; ++i)
    x[i] = (float)v.e[i];
}
template <typename T, bool WIDE> __device__ __forceinline__ void store4(T *p, const float (&x)[4]) {
  Four<T> v;
#pragma unroll
  for (int i = 0; i < 4; ++i)
    v.e[i] = (T)x[i];
  if constexpr (WIDE && sizeof(T) == 4)
    *reinterpret_cast<uint4 *>(p) = *reinterpret_cast<uint4 *>(&v);
  else if constexpr (WIDE)
    *reinterpret_cast<uint2 *>(p) = *reinterpret_cast<uint2 *>(&v);
  else
    for (int i = 0; i < 4; ++i)
      p[i] = v.e[i];
}

// Codes of a lane's four dims, and the group's pair (scale in the low half); all 16 lanes of the group call it.
__device__ __forceinline__ uint32_t quantise(const float (&in)[4], uint32_t lanes, int (&code)[4]) {
  float x[4], mn = INFINITY, mx = -INFINITY;
  bool nan = false;
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    nan = nan || in[i] != in[i];
    x[i] = fminf(fmaxf(in[i], -kKv4Most), kKv4Most);
    mn = fminf(mn, x[i]);
    mx = fmaxf(mx, x[i]);
  }
#pragma unroll
  for (int o = 8; o > 0; o >>= 1) {
    mn = fminf(mn, __shfl_xor_sync(lanes, mn, o));
    mx = fmaxf(mx, __shfl_xor_sync(lanes, mx, o));
  }
  nan = __any_sync(lanes, nan);
  const __half lo = __float2half_rn(mn), scale = __float2half_rn(__fdiv_rn(__fsub_rn(mx, __half2float(lo)), 15.f));
  const float l = __half2float(lo), s = __half2float(scale);
#pragma unroll
  for (int i = 0; i < 4; ++i)
    code[i] = nan || !(s > 0.f) ? 0 : (int)fminf(fmaxf(rintf(__fdiv_rn(__fsub_rn(x[i], l), s)), 0.f), 15.f);
  return nan ? 0x7e000000u : (uint32_t)__half_as_ushort(scale) | (uint32_t)__half_as_ushort(lo) << 16;
}

struct Place {   // of a half-warp's group
  int64_t row;
  int head, group, j;      // j: the position in its tile
  uint8_t *tile;           // null: no position of the pool
};
__device__ __forceinline__ Place place_of(const CacheParams &p, int64_t at) {
  const int per_head = p.D / kKv4Group, per_row = p.kv_heads * per_head;
  Place g;
  g.row = at / per_row;
  const int in_row = (int)(at % per_row);
  g.head = in_row / per_head;
  g.group = in_row % per_head;
  const int64_t slot = p.slots[g.row];
  const int64_t page = slot / p.page;
  const int off = (int)(slot % p.page);
  g.j = off % kKv4Tile;
  g.tile = slot < 0 || slot >= p.positions
               ? nullptr
               : p.pool + ((page * p.kv_heads + g.head) * (p.page / kKv4Tile) + off / kKv4Tile) * kv4_tile_bytes(p.D);
  return g;
}

template <typename T, bool WIDE> __global__ void __launch_bounds__(kThreads) kv4_write_kernel(const __grid_constant__ CacheParams p) {
  kernel_go();
  kernel_wait();
  const int r = threadIdx.x & 15;
  const uint32_t lanes = 0xffffu << (threadIdx.x & 16);
  for (int64_t at = ((int64_t)blockIdx.x * kThreads + threadIdx.x) >> 4; at < p.groups; at += (int64_t)gridDim.x * (kThreads / 16)) {
    const Place g = place_of(p, at);
    if (g.tile == nullptr)
      continue;   // (all 16 lanes)
    const int64_t col = (int64_t)g.head * p.D + g.group * kKv4Group + 4 * r;
    float x[4];
    int c[4];
    load4<T, WIDE>((const T *)p.k + g.row * p.k_ld + col, x);
    uint32_t pair = quantise(x, lanes, c);
    // bytes (c0, c2) and (c1, c3) of lanes r (even) and r + 1: one word
    const uint32_t mine = c[0] | c[2] << 4 | (c[1] | c[3] << 4) << 16, other = __shfl_down_sync(lanes, mine, 1, 16);
    if ((r & 1) == 0)
      *reinterpret_cast<uint32_t *>(g.tile + g.j * (p.D / 2) + (r / 2) % 4 * (p.D / 8) + (2 * g.group + r / 8) * 4) = mine | other << 8;
    if (r == 0)
      *reinterpret_cast<uint32_t *>(g.tile + kv4_k_pairs(p.D) + (g.j * (p.D / kKv4Group) + g.group) * 4) = pair;
    load4<T, WIDE>((const T *)p.v + g.row * p.v_ld + col, x);
    pair = quantise(x, lanes, c);
    // dims 16 i + g (low nibble) and 16 i + 8 + g are four lanes' halves apart: lanes r and r ^ 2 store two bytes each
    const uint32_t all = c[0] | c[1] << 8 | c[2] << 16 | c[3] << 24, apart = __shfl_xor_sync(lanes, all, 2);
    const bool high = r & 2;
    const uint32_t both = high ? apart | all << 4 : all | apart << 4;
    uint8_t *v = g.tile + kv4_v_codes(p.D) + g.group * 512 + (r & 1) * 256 + g.j % 8 / 2 * 16 + r / 4 * 4 + g.j % 2 * 2 + g.j / 8;
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      const int e = high ? 2 + i : i;
      v[e * 64] = (uint8_t)(both >> (8 * e));
    }
    if (r == 0)
      *reinterpret_cast<uint32_t *>(g.tile + kv4_v_pairs(p.D) + (g.j * (p.D / kKv4Group) + g.group) * 4) = pair;
  }
}

template <typename T, bool WIDE> __global__ void __launch_bounds__(kThreads) kv4_read_kernel(const __grid_constant__ CacheParams p) {
  kernel_go();
  kernel_wait();
  const int r = threadIdx.x & 15;
  for (int64_t at = ((int64_t)blockIdx.x * kThreads + threadIdx.x) >> 4; at < p.groups; at += (int64_t)gridDim.x * (kThreads / 16)) {
    const Place g = place_of(p, at);
    const int64_t col = (int64_t)g.head * p.D + g.group * kKv4Group + 4 * r;
    float k[4] = {}, v[4] = {};
    if (g.tile != nullptr) {
      const int pair_at = (g.j * (p.D / kKv4Group) + g.group) * 4;
      __half2 pair = *reinterpret_cast<const __half2 *>(g.tile + kv4_k_pairs(p.D) + pair_at);
      const uint32_t word =
          *reinterpret_cast<const uint32_t *>(g.tile + g.j * (p.D / 2) + (r / 2) % 4 * (p.D / 8) + (2 * g.group + r / 8) * 4) >> (8 * (r & 1));
#pragma unroll
      for (int i = 0; i < 4; ++i)
        k[i] = fmaf(__low2float(pair), (float)(word >> (16 * (i & 1) + 4 * (i >> 1)) & 15), __high2float(pair));
      pair = *reinterpret_cast<const __half2 *>(g.tile + kv4_v_pairs(p.D) + pair_at);
      const uint8_t *c = g.tile + kv4_v_codes(p.D) + g.group * 512 + (r & 1) * 256 + g.j % 8 / 2 * 16 + r / 4 * 4 + g.j % 2 * 2 + g.j / 8;
#pragma unroll
      for (int i = 0; i < 4; ++i)
        v[i] = fmaf(__low2float(pair), (float)(c[i * 64] >> (r & 2 ? 4 : 0) & 15), __high2float(pair));
    }
    store4<T, WIDE>((T *)p.k + g.row * p.k_ld + col, k);
    store4<T, WIDE>((T *)p.v + g.row * p.v_ld + col, v);
  }
}

template <bool WRITE> int cache_launch(const b200_kv4_cache &c, const void *k, int64_t k_ld, const void *v, int64_t v_ld, int dtype, const int64_t *slots,
                                       int rows, cudaStream_t st) {
  if (rows == 0)
    return B200_OK;
  const int64_t groups = (int64_t)rows * c.kv_heads * (c.head_dim / kKv4Group);
  const CacheParams p{(uint8_t *)c.pool, (int64_t)c.n_pages * c.page, c.kv_heads, c.head_dim, c.page, (void *)k, (void *)v, k_ld, v_ld, slots, groups};
  const int64_t blocks = (groups + kThreads / 16 - 1) / (kThreads / 16);
  const dim3 grid((unsigned)(blocks < 148 * 64 ? blocks : 148 * 64));
  const int size = dtype == B200_F32 ? 4 : 2;
  const bool wide = (((uintptr_t)k | (uintptr_t)v | (uintptr_t)(k_ld * size) | (uintptr_t)(v_ld * size)) & (4 * size - 1)) == 0;
#define B200_TYPE(T)                                                                                                                       \
  (WRITE ? launch_after(wide ? kv4_write_kernel<T, true> : kv4_write_kernel<T, false>, grid, kThreads, 0, st, p)                          \
         : launch_after(wide ? kv4_read_kernel<T, true> : kv4_read_kernel<T, false>, grid, kThreads, 0, st, p))
  return dtype == B200_F32 ? B200_TYPE(float) : dtype == B200_F16 ? B200_TYPE(__half) : B200_TYPE(__nv_bfloat16);
#undef B200_TYPE
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
