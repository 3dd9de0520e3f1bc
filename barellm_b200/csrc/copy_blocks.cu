// Page copies inside a paged pool: every layer's K and V slab [Hkv, bs, D] of a
// source block goes to a destination block, and its scales when the pool is 8-bit.
// Bound by HBM: 2 * pairs * layers * 2 * slab bytes read and written.  The block
// ids come from the host and travel in the kernel's parameters, so a call needs
// no upload and can be captured; the host checks that no block is written twice
// or both read and written, so the CTAs' order cannot change the result.  Pairs
// whose slabs hold 3.8 GB read and written: 566 us, 6.6 TB/s.
#include <cstdlib>

#include "common.cuh"

namespace bl {
namespace {

// Pairs in a launch's parameters: 1000 (8000 bytes), or 32 where there are no more,
// since the driver copies all of a kernel's parameters on every launch (8 pairs,
// calls in a row: 8.7 against 9.5 us).
constexpr int kPairsPerLaunch = 1000, kFewPairs = 32;
constexpr int kThreads = 256;
constexpr int kUnroll = 4;  // 16-byte vectors a thread has in flight

template <int N>
struct CopyArgs {
  char* k_pool;
  char* v_pool;
  float* k_scale;
  float* v_scale;
  int64_t num_blocks, slab;  // slab: bytes of one block's K (or V) in one layer
  int32_t hkv, parts;        // parts: CTAs per slab
  int32_t src[N];
  int32_t dst[N];
};

// grid: (pairs * parts, 2, layers)
template <typename V, int N>
__global__ void __launch_bounds__(kThreads) copy_blocks_kernel(const __grid_constant__ CopyArgs<N> a) {
  const int pair = blockIdx.x / a.parts, part = blockIdx.x - pair * a.parts;
  const bool is_v = blockIdx.y;
  const int64_t layer = blockIdx.z;
  const int64_t sb = layer * a.num_blocks + a.src[pair], db = layer * a.num_blocks + a.dst[pair];
  char* pool = is_v ? a.v_pool : a.k_pool;
  const V* src = reinterpret_cast<const V*>(pool + sb * a.slab);
  V* dst = reinterpret_cast<V*>(pool + db * a.slab);
  const int64_t nvec = a.slab / (int64_t)sizeof(V);
  for (int64_t i = (int64_t)part * (kThreads * kUnroll) + threadIdx.x; i < nvec;
       i += (int64_t)a.parts * (kThreads * kUnroll)) {
    V v[kUnroll];
#pragma unroll
    for (int u = 0; u < kUnroll; ++u)
      if (i + u * kThreads < nvec) v[u] = src[i + u * kThreads];
#pragma unroll
    for (int u = 0; u < kUnroll; ++u)
      if (i + u * kThreads < nvec) dst[i + u * kThreads] = v[u];
  }
  float* scale = is_v ? a.v_scale : a.k_scale;
  if (scale && part == 0)
    for (int h = threadIdx.x; h < a.hkv; h += kThreads) scale[db * a.hkv + h] = scale[sb * a.hkv + h];
}

// Refuses ids outside the pool, a destination named twice and a block that is
// both source and destination.  A few pairs are compared with one another; for
// more, a byte per block of the pool says what was seen.
int check_pairs(const bl_copy_blocks_args& a) {
  for (int64_t i = 0; i < a.count; ++i)
    BL_CHECK_ARG(a.src[i] >= 0 && a.src[i] < a.num_blocks && a.dst[i] >= 0 && a.dst[i] < a.num_blocks,
                 "bl_copy_blocks: block id outside the pool (pair %lld: %lld -> %lld, %lld blocks)", (long long)i,
                 (long long)a.src[i], (long long)a.dst[i], (long long)a.num_blocks);
  int64_t twice = -1, both = -1;
  if (a.count <= 32) {
    for (int64_t i = 0; i < a.count; ++i)
      for (int64_t j = 0; j < a.count; ++j) {
        if (j < i && a.dst[i] == a.dst[j]) twice = a.dst[i];
        if (a.dst[i] == a.src[j]) both = a.dst[i];
      }
  } else {
    uint8_t* seen = static_cast<uint8_t*>(calloc((size_t)a.num_blocks, 1));  // 1: read, 2: written
    if (!seen) {
      set_error("bl_copy_blocks: out of host memory");
      return BL_ERR_CAPACITY;
    }
    for (int64_t i = 0; i < a.count; ++i) {
      if (seen[a.dst[i]] & 2) twice = a.dst[i];
      seen[a.src[i]] |= 1;
      seen[a.dst[i]] |= 2;
    }
    for (int64_t i = 0; i < a.count; ++i)
      if (seen[a.dst[i]] & 1) both = a.dst[i];
    free(seen);
  }
  BL_CHECK_ARG(twice < 0, "bl_copy_blocks: block %lld is written twice", (long long)twice);
  BL_CHECK_ARG(both < 0, "bl_copy_blocks: block %lld is both read and written", (long long)both);
  return BL_OK;
}

template <int N>
int launch_copies(const bl_copy_blocks_args& a, cudaStream_t s) {
  CopyArgs<N> k;
  k.k_pool = (char*)a.k_pool;
  k.v_pool = (char*)a.v_pool;
  k.k_scale = a.k_scale;
  k.v_scale = a.v_scale;
  k.num_blocks = a.num_blocks;
  k.slab = a.num_kv_heads * a.block_size * a.head_dim * a.elem_bytes;
  k.hkv = (int32_t)a.num_kv_heads;
  const bool vec = k.slab % 16 == 0 && ((uintptr_t)a.k_pool & 15) == 0 && ((uintptr_t)a.v_pool & 15) == 0;
  const int64_t nvec = vec ? k.slab / 16 : k.slab;
  k.parts = (int32_t)std::min<int64_t>(64, (nvec + kThreads * kUnroll - 1) / (kThreads * kUnroll));
  for (int64_t at = 0; at < a.count; at += N) {
    const int n = (int)std::min<int64_t>(N, a.count - at);
    for (int i = 0; i < n; ++i) {
      k.src[i] = (int32_t)a.src[at + i];
      k.dst[i] = (int32_t)a.dst[at + i];
    }
    dim3 grid((unsigned)(n * k.parts), 2, (unsigned)a.num_layers);
    if (vec)
      copy_blocks_kernel<uint4, N><<<grid, kThreads, 0, s>>>(k);
    else
      copy_blocks_kernel<uint8_t, N><<<grid, kThreads, 0, s>>>(k);
    BL_CHECK_LAUNCH("copy_blocks_kernel");
  }
  return BL_OK;
}

}  // namespace
}  // namespace bl

using namespace bl;

extern "C" int bl_copy_blocks(const bl_copy_blocks_args* args, void* stream) {
  BL_CHECK_ARG(args != nullptr, "bl_copy_blocks: args is null");
  const bl_copy_blocks_args& a = *args;
  BL_CHECK_ARG(a.k_pool && a.v_pool, "bl_copy_blocks: K/V pool pointers must be non-null");
  BL_CHECK_ARG((a.k_scale != nullptr) == (a.v_scale != nullptr), "bl_copy_blocks: give both scale tables or none");
  BL_CHECK_ARG(a.num_layers > 0 && a.num_blocks > 0 && a.num_kv_heads > 0 && a.block_size > 0 && a.head_dim > 0 &&
                   a.elem_bytes > 0,
               "bl_copy_blocks: pool dimensions must be positive");
  BL_CHECK_ARG(a.num_layers <= 65535 && a.num_blocks <= INT32_MAX && a.num_kv_heads <= INT32_MAX,
               "bl_copy_blocks: pool dimensions too large");
  BL_CHECK_ARG(a.count >= 0 && a.count <= a.num_blocks, "bl_copy_blocks: more pairs than blocks");
  if (a.count == 0) return BL_OK;
  BL_CHECK_ARG(a.src && a.dst, "bl_copy_blocks: null block ids");
  const int rc = check_pairs(a);
  if (rc) return rc;
  return a.count <= kFewPairs ? launch_copies<kFewPairs>(a, (cudaStream_t)stream)
                              : launch_copies<kPairsPerLaunch>(a, (cudaStream_t)stream);
}
