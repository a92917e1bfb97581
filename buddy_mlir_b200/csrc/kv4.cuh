// The 4-bit KV cache's format and its addresses (buddy_b200.h has both in words): shared by its writer, its reader and its attention.
#pragma once
#include "common.cuh"

namespace b200 {

constexpr int kKv4Group = 64;    // dims with one (scale, lo) pair
constexpr int kKv4Tile = 16;     // positions of a tile
constexpr float kKv4Most = 65504.f;

__host__ __device__ constexpr int kv4_tile_bytes(int D) { return kKv4Tile * (D + D / 8); }
// parts of a tile
__host__ __device__ constexpr int kv4_v_codes(int D) { return 8 * D; }
__host__ __device__ constexpr int kv4_k_pairs(int D) { return 16 * D; }
__host__ __device__ constexpr int kv4_v_pairs(int D) { return 17 * D; }

// Checks of a cache that its calls have in common.
int kv4_check(const char *call, const b200_kv4_cache *c);

// kv4_cache.cu: what is behind b200_page_step and b200_kv4_write, without their checks
int page_step_launch(const b200_page_step_args &a, cudaStream_t st);
int kv4_write_launch(const b200_kv4_cache &c, const void *k, int64_t k_ld, const void *v, int64_t v_ld, int dtype, const int64_t *slots, int rows,
                     cudaStream_t st);
// kv4_attention.cu: the word of a workspace that says which bounded wait gave up (0: none)
const int *kv4_attention_error(const void *workspace);

} // namespace b200
