// Attention over the 4-bit KV cache (b200_kv4_attention).
#include "kv4.cuh"

namespace b200 {

namespace {

constexpr int kThreads = 128;

struct AttentionParams {
  const uint8_t *pool;
  int n_pages, kv_heads, page;
  b200_kv4_attention_args a;
};

__device__ __forceinline__ int clamp(int x, int lo, int hi) { return min(max(x, lo), hi); }

// A warp per row and q head, a key after the other.
template <int D> __global__ void __launch_bounds__(kThreads) kv4_attention_kernel(const __grid_constant__ AttentionParams p) {
  constexpr int E = D / 32;   // dims 32 e + lane of a lane
  kernel_go();
  kernel_wait();
  const b200_kv4_attention_args &a = p.a;
  const int lane = threadIdx.x & 31;
  const int64_t at = (int64_t)blockIdx.x * (kThreads / 32) + (threadIdx.x >> 5);
  if (at >= (int64_t)a.rows * a.q_heads)
    return;
  const int row = (int)(at / a.q_heads), head = (int)(at % a.q_heads), kv = head / (a.q_heads / p.kv_heads);
  // the last sequence that begins at or before the row
  int lo = -1, hi = a.n_seqs;
  while (hi - lo > 1) {
    const int mid = (lo + hi) >> 1;
    if (a.row_start[mid] <= row)
      lo = mid;
    else
      hi = mid;
  }
  int seen = 0;
  if (lo >= 0 && row < a.row_start[lo + 1])
    seen = clamp((int)min((int64_t)a.lens[lo] - a.row_start[lo + 1] + row + 1, (int64_t)a.table_stride * p.page), 0, a.table_stride * p.page);
  float q[E], acc[E] = {}, m = -INFINITY, l = 0.f;
  bool any = false;
#pragma unroll
  for (int e = 0; e < E; ++e)
    q[e] = load_as_float(a.q, a.dtype, (int64_t)row * a.q_ld + (int64_t)head * D + 32 * e + lane);
  for (int j = 0; j < seen; ++j) {
    const int id = a.block_table[(int64_t)lo * a.table_stride + j / p.page], off = j % p.page, jj = off % kKv4Tile;
    if (id < 0 || id >= p.n_pages)
      continue;
    const uint8_t *tile = p.pool + (((int64_t)id * p.kv_heads + kv) * (p.page / kKv4Tile) + off / kKv4Tile) * kv4_tile_bytes(D);
    float s = 0.f, v[E];
#pragma unroll
    for (int e = 0; e < E; ++e) {
      const int d = 32 * e + lane, pair = (jj * (D / kKv4Group) + d / kKv4Group) * 4;
      const __half2 kp = *reinterpret_cast<const __half2 *>(tile + kv4_k_pairs(D) + pair), vp = *reinterpret_cast<const __half2 *>(tile + kv4_v_pairs(D) + pair);
      const int kc = tile[jj * (D / 2) + d / 8 % 4 * (D / 8) + d / 32 * 4 + d % 2 * 2 + d % 8 / 4] >> (d % 4 / 2 * 4) & 15;
      const int vc = tile[kv4_v_codes(D) + d / 64 * 512 + d % 8 * 64 + jj % 8 / 2 * 16 + d / 16 % 4 * 4 + jj % 2 * 2 + jj / 8] >> (d % 16 / 8 * 4) & 15;
      s = fmaf(q[e], fmaf(__low2float(kp), (float)kc, __high2float(kp)), s);
      v[e] = fmaf(__low2float(vp), (float)vc, __high2float(vp));
    }
    s = warp_sum(s) * a.scale;
    const float top = fmaxf(m, s), w = expf(s - top), keep = m == -INFINITY ? 0.f : expf(m - top);
    l = fmaf(l, keep, w);
#pragma unroll
    for (int e = 0; e < E; ++e)
      acc[e] = fmaf(acc[e], keep, w * v[e]);
    m = top;
    any = true;
  }
#pragma unroll
  for (int e = 0; e < E; ++e) {
    const float o = any ? acc[e] / l : 0.f;
    const int64_t to = (int64_t)row * a.out_ld + (int64_t)head * D + 32 * e + lane;
    if (a.dtype == B200_F32)
      ((float *)a.out)[to] = o;
    else if (a.dtype == B200_F16)
      ((__half *)a.out)[to] = __float2half_rn(o);
    else
      ((__nv_bfloat16 *)a.out)[to] = __float2bfloat16_rn(o);
  }
}

} // namespace

} // namespace b200

using namespace b200;

extern "C" {

int64_t b200_kv4_attention_workspace_bytes(int q_heads, int kv_heads, int head_dim) {
  if (kv_heads < 1 || kv_heads > 1024 || q_heads < 1 || q_heads % kv_heads != 0 || (head_dim != 64 && head_dim != 128))
    return B200_EINVAL;
  return 256;
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
  const AttentionParams p{(const uint8_t *)c->pool, c->n_pages, c->kv_heads, c->page, *a};
  const dim3 grid((unsigned)(((int64_t)a->rows * a->q_heads + kThreads / 32 - 1) / (kThreads / 32)));
  return c->head_dim == 128 ? launch_after(kv4_attention_kernel<128>, grid, kThreads, 0, (cudaStream_t)stream, p)
                            : launch_after(kv4_attention_kernel<64>, grid, kThreads, 0, (cudaStream_t)stream, p);
}

} // extern "C"
