// Chunked-prefill attention over an 8-bit paged cache.  Query i of row b (C_b
// queries, total length L_b) sees keys 0 .. L_b - C_b + i, as in prefill.cu;
// K and V are code * scale (fp8.cuh).  Reference counterpart: the prefill SDPA of
// src/barellm/attention/backend.py:52-61 over a dense read of the cache.
//
// Three ways, chosen by shape (use_tc below):
//   expand + prefill_tc_kernel  16-bit q, head_dim a multiple of 8 up to 128.  The rows' pages are
//       dequantised once into a 16-bit paged scratch (bf16: exact, a code has
//       four significant bits; fp16: in units of each row and KV head, half_unit in
//       fp8.cuh), which the tcgen05 kernel of prefill_tc.cu then reads.  The
//       expansion moves 1 + 2 bytes per cached element (1 + 2 n where a KV head
//       becomes n, below); a CTA of the attention kernel reads the 2-byte form,
//       and every 128 query tokens times group re-read it (mostly from L2), so
//       dequantising in that kernel would repeat the conversion for every query
//       tile.  (Few queries over a long prefix pay for that: 8 rows of 4 queries over 8k
//       tokens take 204 us, ten times their codes' bytes.)  Block sizes
//       other than 16 become 16-token pages on the way, and a query group
//       that the kernel is not built for (3, 5, 16, ...) becomes several KV heads
//       with the same contents and a group of 8, 4, 2 or 1.  A head_dim below
//       128 is widened with zeros, which change neither scores nor outputs: K
//       and V on the way, q and out through copies.
//   fp8_prefill_mma_kernel      16-bit q, head_dim a multiple of 16 from 144 to 256.
//   fp8_prefill_simt_kernel     any element type, head_dim <= 256, block size
//       and group: 64 queries x 64 keys a tile in fp32, pages dequantised
//       into shared memory.
// The two on the tensor cores round P to the element type, whose product with V
// the matrix instructions take: half a step (2^-8 in bf16, 2^-11 in fp16) of each
// weight in the numerator; the weights' sum, the maxima and the outputs' sums are fp32.
// A key that a query does not see has weight 0, and 0 * NaN is NaN: a NaN among the
// V of a chunk may reach the chunk's queries before it (never those that see nothing).
#include <cstring>
#include <type_traits>

#include "fp8.cuh"
#include "prefill_tc.cuh"

namespace bl {
namespace {

constexpr float kLog2e = 1.4426950408889634f;
constexpr int kPage = 16;  // tokens of a scratch page
constexpr int kTCDim = 128;

inline size_t align256(size_t x) { return (x + 255) & ~size_t(255); }

// How a call's scratch looks: 16-token pages of `heads` KV heads, each cached
// head repeated `dup` times; q and out widened to 128 dims where head_dim is less.
struct Scratch {
  int64_t width, pages, heads, dup;
  size_t table, order, units, k, v, q, out, total;
};

bool use_tc(int32_t dtype, int64_t d) {
  return (dtype == BL_BF16 || dtype == BL_F16) && d > 0 && d <= kTCDim && d % 8 == 0;
}

bool use_mma(int32_t dtype, int64_t d) {
  return (dtype == BL_BF16 || dtype == BL_F16) && d > kTCDim && d <= 256 && d % 16 == 0;
}

// False when the scratch would not fit the tcgen05 kernel's 32-bit row coordinates
// (the call then takes the SIMT kernel).
bool plan_scratch(int32_t dtype, int64_t batch, int64_t hq, int64_t hkv, int64_t d, int64_t bs, int64_t total_q, int64_t max_seq_len,
                  int64_t total_blocks, Scratch* w) {
  const int64_t g = hq / hkv;
  int64_t gt = 8;
  while (g % gt) gt /= 2;
  w->dup = g / gt;
  w->heads = hkv * w->dup;
  w->width = (max_seq_len + kPage - 1) / kPage;
  // every row ends in at most one partial page; more than batch * width cannot be in use
  const double bound = (double)total_blocks * (double)bs / kPage + (double)batch + 1;
  w->pages = (int64_t)std::min(bound, (double)batch * (double)w->width);
  if ((double)w->pages * w->heads * kPage > (double)(INT32_MAX - 64) || w->heads > 65535) return false;
  const size_t table_bytes = align256((size_t)batch * w->width * sizeof(int32_t));
  w->units = table_bytes + align256((size_t)batch * sizeof(int32_t));
  const size_t off = w->units + (dtype == BL_F16 ? align256((size_t)batch * w->heads * 2 * sizeof(float)) : 0);
  const size_t half = align256((size_t)w->pages * w->heads * kPage * kTCDim * 2);
  w->table = 0;
  w->order = table_bytes;
  w->k = off;
  w->v = off + half;
  const size_t wide = d < kTCDim ? align256((size_t)total_q * hq * kTCDim * 2) : 0;
  w->q = off + 2 * half;
  w->out = w->q + wide;
  w->total = w->out + wide;
  return true;
}

struct ExpandArgs {
  const uint8_t* k_pool;
  const uint8_t* v_pool;
  const float* k_scale;
  const float* v_scale;
  void* k_out;
  void* v_out;
  int32_t* table;  // [batch][width]
  int32_t* order;  // [batch] rows, the longest first
  float* k_unit;   // fp16: [batch, hkv * dup]
  float* v_unit;
  int64_t num_blocks, layer, width, pages, bt_stride, bt_width;
  const int32_t* block_tables;
  const int32_t* row_ids;
  const int32_t* seq_lens;
  const int32_t* q_offsets;
  int64_t max_q, o_sb, o_st, o_sh;
  void* out;
  int32_t hkv, bs, bs_shift, d, dup, hq;  // bs_shift: log2 of the block size, or -1
  int32_t own_units;                      // fp16: every CTA finds its row's units itself
  int32_t* err;
};

constexpr int kExpandThreads = 256;  // one page of one head: 16 tokens x 16 eight-code vectors

// fp16: the units of a row's KV head (half_unit), from the scales of the row's blocks.
// Bound by two dependent loads a block, 256 blocks at a time.  Every warp leaves its
// maxima in `s` (before a __syncthreads); units_of joins them.
struct UnitShared {
  float k[kExpandThreads / 32], v[kExpandThreads / 32];
};
template <typename A>
__device__ __forceinline__ void find_units(const A& a, int64_t row, int64_t len, int h, UnitShared& s) {
  const int64_t blocks = len > 0 ? min((len + a.bs - 1) / a.bs, a.bt_width) : 0;
  float km = 0.f, vm = 0.f;
#pragma unroll 2
  for (int64_t j = threadIdx.x; j < blocks; j += kExpandThreads) {
    const int64_t phys = a.block_tables[row * a.bt_stride + j];
    if (phys < 0 || phys >= a.num_blocks) continue;  // (reported where the block's tokens are read)
    const int64_t slot = (a.layer * a.num_blocks + phys) * a.hkv + h;
    km = fmaxf(km, a.k_scale[slot]);
    vm = fmaxf(vm, a.v_scale[slot]);
  }
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) {
    km = fmaxf(km, __shfl_xor_sync(0xffffffffu, km, o));
    vm = fmaxf(vm, __shfl_xor_sync(0xffffffffu, vm, o));
  }
  if ((threadIdx.x & 31) == 0) s.k[threadIdx.x >> 5] = km, s.v[threadIdx.x >> 5] = vm;
}
__device__ __forceinline__ float2 units_of(const UnitShared& s) {
  float km = s.k[0], vm = s.v[0];
#pragma unroll
  for (int w = 1; w < kExpandThreads / 32; ++w) km = fmaxf(km, s.k[w]), vm = fmaxf(vm, s.v[w]);
  return make_float2(half_unit(km), half_unit(vm));
}
__device__ __forceinline__ void store_units(const ExpandArgs& a, int64_t b, int h, float2 unit) {
  for (int r = threadIdx.x; r < a.dup; r += kExpandThreads) {
    a.k_unit[(b * a.hkv + h) * a.dup + r] = unit.x;
    a.v_unit[(b * a.hkv + h) * a.dup + r] = unit.y;
  }
}

// The units ahead of the expansion, whose first loads are on their way meanwhile.
// Rows of few blocks need no such kernel: every CTA of the expansion finds them by
// itself (ExpandArgs::own_units).
// grid: (hkv, batch)
__global__ void __launch_bounds__(kExpandThreads) fp8_units_kernel(const ExpandArgs a) {
  pdl_trigger();  // the expansion may start; it waits for this grid before it needs a unit
  const int64_t b = blockIdx.y;
  __shared__ UnitShared s;
  find_units(a, a.row_ids ? (int64_t)a.row_ids[b] : b, a.seq_lens[b], blockIdx.x, s);
  __syncthreads();
  store_units(a, b, blockIdx.x, units_of(s));
}

// Bound by HBM: 1 byte read and 2 written per element (8 rows, 41.8k tokens, 8 KV
// heads, head_dim 128: 257 MB in 45..50 us, 5.1..5.7 TB/s).  Four pages a CTA, so
// that 8 loads a thread are in flight while the CTA counts the pages before its row.
constexpr int kExpandPages = 4;  // pages of a CTA
// fp16 rows of at most so many blocks: every CTA finds the units by itself, which saves a
// launch (8 rows of 300 tokens, calls in a row: 25.4 against 28.4 us; of 1000: 40.0 and
// 40.4).  Rows of more are read by too many CTAs (of 4000: 118.6 against 116.1 us; of
// 32k: 917 and 789).
constexpr int64_t kOwnUnitBlocks = 128;

// grid: (ceil(width / kExpandPages), hkv, batch)
template <typename T>
__global__ void __launch_bounds__(kExpandThreads, 4) fp8_expand_kernel(const ExpandArgs a) {
  constexpr bool kUnits = std::is_same<T, __half>::value;
  const int tid = threadIdx.x, h = blockIdx.y;
  const int64_t b = blockIdx.z;
  const int64_t len = max((int64_t)a.seq_lens[b], (int64_t)0);
  if (blockIdx.x == 0 && h == 0) {
    // queries that see no key at all (more queries than tokens): zeros
    int64_t qo = 0, nq = a.max_q;
    if (a.q_offsets) {
      qo = a.q_offsets[b];
      nq = (int64_t)a.q_offsets[b + 1] - qo;
    }
    for (int64_t i = 0; i < nq - len; ++i)
      for (int e = tid; e < a.hq * kTCDim; e += kExpandThreads)
        reinterpret_cast<T*>(a.out)[b * a.o_sb + (qo + i) * a.o_st + (int64_t)(e / kTCDim) * a.o_sh + e % kTCDim] =
            from_f32<T>(0.f);
    if (tid == 0 && len > a.width * kPage) raise_dev(a.err, BL_DEVERR_WORKSPACE);  // longer than max_seq_len
    // The attention kernel's CTAs start in the order of their rows, and one CTA's
    // time goes with its row's length: the longest rows go first.
    __shared__ int s_rank;
    if (tid == 0) s_rank = 0;
    __syncthreads();
    int longer = 0;
    for (int64_t r = tid; r < (int64_t)gridDim.z; r += kExpandThreads) {
      const int64_t l = max((int64_t)a.seq_lens[r], (int64_t)0);
      longer += l > len || (l == len && r < b);
    }
    atomicAdd(&s_rank, longer);
    __syncthreads();
    if (tid == 0) a.order[s_rank] = (int32_t)b;
  }
  const int64_t j0 = (int64_t)blockIdx.x * kExpandPages;
  if (j0 * kPage >= len) {
    if (kUnits) pdl_wait();  // (this grid is complete only when the units are; a no-op without their kernel)
    return;
  }

  const int64_t row = a.row_ids ? (int64_t)a.row_ids[b] : b;
  const int tok = tid >> 4, v = tid & 15;
  uint2 kc[kExpandPages], vc[kExpandPages];
  float ks[kExpandPages], vs[kExpandPages];
  bool ok[kExpandPages];
#pragma unroll
  for (int p = 0; p < kExpandPages; ++p) {
    const int64_t j = j0 + p, t = j * kPage + tok;
    ok[p] = false;
    if (j >= a.width || t >= len) continue;
    const int64_t lb = a.bs_shift >= 0 ? t >> a.bs_shift : t / a.bs;
    if (lb >= a.bt_width) {
      raise_dev(a.err, BL_DEVERR_TABLE);
      continue;
    }
    int64_t phys = a.block_tables[row * a.bt_stride + lb];
    if (phys < 0 || phys >= a.num_blocks) {
      raise_dev(a.err, BL_DEVERR_BLOCK_ID);
      continue;
    }
    const int64_t slot = (a.layer * a.num_blocks + phys) * a.hkv + h;
    if (v * 8 >= a.d) continue;  // (dims that head_dim does not have are zeros)
    const int64_t src = (slot * a.bs + (t - lb * a.bs)) * a.d + v * 8;
    kc[p] = *reinterpret_cast<const uint2*>(a.k_pool + src);
    vc[p] = *reinterpret_cast<const uint2*>(a.v_pool + src);
    ks[p] = a.k_scale[slot];
    vs[p] = a.v_scale[slot];
    ok[p] = true;
  }
  // meanwhile, the first scratch page of the row: the pages of the rows before it
  __shared__ int64_t s_sum[kExpandThreads / 32];
  int64_t base = 0;
  for (int64_t r = tid; r < b; r += kExpandThreads)
    base += (min(max((int64_t)a.seq_lens[r], (int64_t)0), a.width * kPage) + kPage - 1) / kPage;
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) base += __shfl_xor_sync(0xffffffffu, base, o);
  if ((tid & 31) == 0) s_sum[tid >> 5] = base;
  __shared__ UnitShared s_unit;
  if (kUnits && a.own_units) find_units(a, row, len, h, s_unit);
  __syncthreads();
  base = 0;
#pragma unroll
  for (int w = 0; w < kExpandThreads / 32; ++w) base += s_sum[w];
  if (h == 0 && tid < kExpandPages && j0 + tid < a.width && (j0 + tid) * kPage < len) {
    const bool fits = base + j0 + tid < a.pages;
    a.table[b * a.width + j0 + tid] = fits ? (int32_t)(base + j0 + tid) : -1;
    if (!fits) raise_dev(a.err, BL_DEVERR_WORKSPACE);
  }
  if (kUnits) {
    pdl_wait();  // the units are written
    const int64_t at = (b * a.hkv + h) * a.dup;
    float2 unit;
    if (a.own_units) {
      unit = units_of(s_unit);
      if (blockIdx.x == 0) store_units(a, b, h, unit);
    } else {
      unit = make_float2(a.k_unit[at], a.v_unit[at]);
    }
    const float k_inv = pow2_inverse(unit.x), v_inv = pow2_inverse(unit.y);
#pragma unroll
    for (int p = 0; p < kExpandPages; ++p) ks[p] *= k_inv, vs[p] *= v_inv;
  }
#pragma unroll
  for (int p = 0; p < kExpandPages; ++p) {
    const int64_t j = j0 + p;
    if (j >= a.width || base + j >= a.pages || j * kPage >= len) continue;
    // a token whose block cannot be read, and the slots behind the length, become zeros
    uint4 ko = make_uint4(0, 0, 0, 0), vo = ko;
    if (ok[p]) {
      ko = dequant8<T>(kc[p], ks[p]);
      vo = dequant8<T>(vc[p], vs[p]);
    }
    for (int r = 0; r < a.dup; ++r) {
      const int64_t dst = ((((base + j) * a.hkv + h) * a.dup + r) * kPage + tok) * kTCDim + v * 8;
      *reinterpret_cast<uint4*>(reinterpret_cast<T*>(a.k_out) + dst) = ko;
      *reinterpret_cast<uint4*>(reinterpret_cast<T*>(a.v_out) + dst) = vo;
    }
  }
}

// q rows of head_dim d widened to 128 dims with zeros (IN), or the widened out
// rows cut back to d.  One warp per (token, head) row, four dims a lane.  Tokens:
// packed on one axis, or [batch, max_q].
struct WidenArgs {
  void* narrow;
  void* wide;  // [total, hq, 128]
  int64_t sb, st, sh;
  const int32_t* offsets;  // packed: tokens [offsets[0], offsets[batch]) belong to rows
  int64_t batch, max_q, total;
  int32_t hq, d;
};

template <typename T, bool IN>
__global__ void __launch_bounds__(256) fp8_widen_kernel(const WidenArgs a) {
  const int lane = threadIdx.x & 31;
  const int64_t r = (int64_t)blockIdx.x * 8 + (threadIdx.x >> 5);
  const int64_t n = r / a.hq;
  if (n >= a.total) return;
  const int h = (int)(r - n * a.hq);
  int64_t b = 0, t = n;
  if (a.offsets) {
    if (n < a.offsets[0] || n >= a.offsets[a.batch]) return;
  } else {
    b = n / a.max_q;
    t = n - b * a.max_q;
  }
  T* x = reinterpret_cast<T*>(a.narrow) + b * a.sb + t * a.st + (int64_t)h * a.sh;
  T* y = reinterpret_cast<T*>(a.wide) + r * kTCDim + 4 * lane;
#pragma unroll
  for (int e = 0; e < 4; ++e) {
    const int d = 4 * lane + e;
    if (IN)
      y[e] = d < a.d ? x[d] : from_f32<T>(0.f);
    else if (d < a.d)
      x[d] = y[e];
  }
}

template <typename T, bool IN>
int launch_widen(const WidenArgs& k, cudaStream_t s) {
  const int64_t rows = k.total * k.hq;
  fp8_widen_kernel<T, IN><<<(unsigned)((rows + 7) / 8), 256, 0, s>>>(k);
  BL_CHECK_LAUNCH("fp8_widen_kernel");
  return BL_OK;
}

// ---------------------------------------------------------------------------
// head_dims above 128: mma.sync kernel
// ---------------------------------------------------------------------------
constexpr int kMmaRows = 128, kMmaKeys = 64;  // query rows and keys of a tile
constexpr int kMmaDim = 256;
constexpr int kMmaThreads = 256;  // a warp has 16 query rows
constexpr int kMmaRow = kMmaDim * 2;  // bytes of a 16-bit row in shared memory

struct MmaArgs {
  const void* q;
  int64_t q_sb, q_st, q_sh;
  void* out;
  int64_t o_sb, o_st, o_sh;
  const int32_t* q_offsets;
  const int32_t* seq_lens;
  const uint8_t* k_pool;
  const uint8_t* v_pool;
  const float* k_scale;
  const float* v_scale;
  const int32_t* block_tables;
  int64_t bt_stride, bt_width;
  const int32_t* row_ids;
  int64_t num_blocks, layer, max_q;
  int32_t hkv, g, bs, d;
  int32_t q_vec, o_pair;  // q rows can be read 16 bytes at a time, out rows written two elements at a time
  float scale_log2;
  int32_t* err;
};

struct MmaShared {
  uint8_t q[kMmaRows * kMmaRow];
  uint8_t k[kMmaKeys * kMmaRow], v[kMmaKeys * kMmaRow];     // the tile, in q's type
  uint8_t kc[kMmaKeys * kMmaDim], vc[kMmaKeys * kMmaDim];   // its codes, or the next tile's on their way
  int64_t row[2][kMmaKeys];                                 // byte offset of a token's codes, -1: none
  float ks[2][kMmaKeys], vs[2][kMmaKeys];                   // in the units below
  UnitShared unit;
};

// byte offset of 16-byte chunk c of row r: rows are 512 bytes, and eight rows'
// equal chunks lie in different banks
__device__ __forceinline__ uint32_t mma_at(int r, int c) { return (uint32_t)(r * kMmaRow + ((c ^ (r & 7)) << 4)); }

__device__ __forceinline__ void copy16_async(uint32_t dst, const void* src) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(dst), "l"(src) : "memory");
}

// S = Q K^T and O += P V on mma.sync, 128 query rows by 64 keys a tile.  The rows
// of a tile are (token, head of the group) pairs, so that one pass over the keys
// serves the whole group and a short chunk still fills a tile.  Codes come by
// cp.async while the tile before is worked on and become 16-bit rows once per tile.
// (The tcgen05 kernel's tile for 128 dims does not fit 256: its rings of 16-bit
// keys and values would need 256 KB.)  What bounds it: the phases of a tile (widen,
// scores, softmax, values) wait for one another, with 8 warps on an SM.  4 chunks
// of 256..1024 tokens over 0..4k, 32 / 8 heads of 256 dims, bf16, 181 GFLOP: 1.02 ms,
// 177 TFLOP/s (the fp32 SIMT kernel below: 11.0 ms).
// grid: (ceil(max_q * g / kMmaRows), hkv, batch)
template <typename T>
__global__ void __launch_bounds__(kMmaThreads, 1) fp8_prefill_mma_kernel(const MmaArgs a) {
  extern __shared__ __align__(16) unsigned char smem_raw[];
  MmaShared* sh = reinterpret_cast<MmaShared*>(smem_raw + ((128u - (smem_u32(smem_raw) & 127u)) & 127u));
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  const int64_t b = blockIdx.z;
  const int h = blockIdx.y;
  int64_t qo = 0, nq = a.max_q;
  if (a.q_offsets) {
    qo = a.q_offsets[b];
    nq = (int64_t)a.q_offsets[b + 1] - qo;
  }
  const int64_t r0 = ((int64_t)gridDim.x - 1 - blockIdx.x) * kMmaRows;  // the tiles with most keys first
  const int64_t rows = nq * a.g;
  if (r0 >= rows) return;
  const int64_t len = a.seq_lens[b], prefix = len - nq;
  const int64_t kend = prefix + (min(r0 + kMmaRows, rows) - 1) / a.g + 1;  // keys that the last row sees
  const int64_t trow = a.row_ids ? (int64_t)a.row_ids[b] : b;
  const int chunks = a.d / 16;  // 16-byte chunks of a token's codes

  // fp16: the units of the keys that the tile sees (half_unit)
  float k_unit = 1.f, v_unit = 1.f, k_inv = 1.f, v_inv = 1.f;
  if constexpr (std::is_same<T, __half>::value) {
    static_assert(kMmaThreads == kExpandThreads, "find_units");
    find_units(a, trow, kend, h, sh->unit);
    __syncthreads();
    const float2 unit = units_of(sh->unit);
    k_unit = unit.x, v_unit = unit.y;
    k_inv = pow2_inverse(k_unit), v_inv = pow2_inverse(v_unit);
  }
  const float scale_log2 = a.scale_log2 * k_unit;

  auto locate = [&](int64_t k0, int buf) {
    if (tid >= kMmaKeys) return;
    const int64_t t = k0 + tid;
    int64_t r = -1;
    float ks = 0.f, vs = 0.f;
    if (t < kend) {
      const int64_t lb = t / a.bs;
      if (lb >= a.bt_width) {
        raise_dev(a.err, BL_DEVERR_TABLE);
      } else {
        const int64_t phys = a.block_tables[trow * a.bt_stride + lb];
        if (phys < 0 || phys >= a.num_blocks) {
          raise_dev(a.err, BL_DEVERR_BLOCK_ID);
        } else {
          const int64_t slot = (a.layer * a.num_blocks + phys) * a.hkv + h;
          r = (slot * a.bs + (t - lb * a.bs)) * a.d;
          ks = a.k_scale[slot] * k_inv;
          vs = a.v_scale[slot] * v_inv;
        }
      }
    }
    sh->row[buf][tid] = r;
    sh->ks[buf][tid] = ks;
    sh->vs[buf][tid] = vs;
  };
  auto fetch = [&](int buf) {
    for (int e = tid; e < kMmaKeys * 16; e += kMmaThreads) {
      const int t = e >> 4, c = e & 15;
      const int64_t r = sh->row[buf][t];
      if (r >= 0 && c < chunks) {
        copy16_async(smem_u32(sh->kc + t * kMmaDim + c * 16), a.k_pool + r + c * 16);
        copy16_async(smem_u32(sh->vc + t * kMmaDim + c * 16), a.v_pool + r + c * 16);
      }
    }
    asm volatile("cp.async.commit_group;" ::: "memory");
  };
  auto widen = [&](const uint8_t* codes, uint8_t* to, const float* scale, int buf) {
    for (int e = tid; e < kMmaKeys * 16; e += kMmaThreads) {
      const int t = e >> 4, c = e & 15;
      uint4 x[2];
      x[0] = x[1] = make_uint4(0u, 0u, 0u, 0u);
      if (sh->row[buf][t] >= 0 && c < chunks) {
        const uint4 w = *reinterpret_cast<const uint4*>(codes + t * kMmaDim + c * 16);
        x[0] = dequant8<T>(make_uint2(w.x, w.y), scale[t]);
        x[1] = dequant8<T>(make_uint2(w.z, w.w), scale[t]);
      }
      *reinterpret_cast<uint4*>(to + mma_at(t, 2 * c)) = x[0];
      *reinterpret_cast<uint4*>(to + mma_at(t, 2 * c + 1)) = x[1];
    }
  };

  locate(0, 0);
  // the tile's query rows, zeros behind the last one and behind head_dim
  for (int e = tid; e < kMmaRows * 32; e += kMmaThreads) {
    const int i = e >> 5, c = e & 31;
    const int64_t r = r0 + i;
    union {
      T t[8];
      uint4 u;
    } x;
    x.u = make_uint4(0u, 0u, 0u, 0u);
    if (r < rows && c < 2 * chunks) {
      const int64_t t = r / a.g;
      const T* p = reinterpret_cast<const T*>(a.q) + b * a.q_sb + (qo + t) * a.q_st + (h * a.g + (r - t * a.g)) * a.q_sh + c * 8;
      if (a.q_vec) {
        x.u = *reinterpret_cast<const uint4*>(p);
      } else {
#pragma unroll
        for (int j = 0; j < 8; ++j) x.t[j] = p[j];
      }
    }
    *reinterpret_cast<uint4*>(sh->q + mma_at(i, c)) = x.u;
  }
  __syncthreads();
  fetch(0);

  const int g_row = lane >> 2, t4 = lane & 3;
  // the lane's two rows; the last key each sees
  int64_t last[2];
#pragma unroll
  for (int i = 0; i < 2; ++i) {
    const int64_t r = r0 + warp * 16 + g_row + 8 * i;
    last[i] = r < rows ? prefix + r / a.g : -1;
  }
  float m[2] = {-INFINITY, -INFINITY}, l[2] = {0.f, 0.f};
  float o[kMmaDim / 8][4];
#pragma unroll
  for (int j = 0; j < kMmaDim / 8; ++j) o[j][0] = o[j][1] = o[j][2] = o[j][3] = 0.f;

  const uint32_t qs = smem_u32(sh->q), ks = smem_u32(sh->k), vs = smem_u32(sh->v);
  const int q_row = warp * 16 + (lane & 15), q_half = lane >> 4;
  const int k_row = (lane & 7) + ((lane & 16) >> 1), k_half = (lane >> 3) & 1;
  const int v_row = lane & 15, v_half = lane >> 4;

  int buf = 0;
  for (int64_t k0 = 0; k0 < kend; k0 += kMmaKeys, buf ^= 1) {
    asm volatile("cp.async.wait_group 0;" ::: "memory");
    __syncthreads();  // the codes are here; the tile before is no longer read
    widen(sh->kc, sh->k, sh->ks[buf], buf);
    widen(sh->vc, sh->v, sh->vs[buf], buf);
    locate(k0 + kMmaKeys, buf ^ 1);
    __syncthreads();
    fetch(buf ^ 1);

    float s[kMmaKeys / 8][4];
#pragma unroll
    for (int j = 0; j < kMmaKeys / 8; ++j) s[j][0] = s[j][1] = s[j][2] = s[j][3] = 0.f;
#pragma unroll 4
    for (int c = 0; c < kMmaDim / 16; ++c) {
      uint32_t q0, q1, q2, q3;
      ldmatrix_x4(qs + mma_at(q_row, 2 * c + q_half), q0, q1, q2, q3);
#pragma unroll
      for (int j = 0; j < kMmaKeys / 8; j += 2) {
        uint32_t b0, b1, b2, b3;
        ldmatrix_x4(ks + mma_at(j * 8 + k_row, 2 * c + k_half), b0, b1, b2, b3);
        mma_16816<T>(s[j][0], s[j][1], s[j][2], s[j][3], q0, q1, q2, q3, b0, b1);
        mma_16816<T>(s[j + 1][0], s[j + 1][1], s[j + 1][2], s[j + 1][3], q0, q1, q2, q3, b2, b3);
      }
    }
    // softmax in log2 units; keys that a row does not see, or that cannot be read, are out
    float mx[2] = {m[0], m[1]};
#pragma unroll
    for (int j = 0; j < kMmaKeys / 8; ++j)
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        const int key = j * 8 + 2 * t4 + (e & 1), i = e >> 1;
        s[j][e] = k0 + key <= last[i] && sh->row[buf][key] >= 0 ? s[j][e] * scale_log2 : -INFINITY;
        mx[i] = fmaxf(mx[i], s[j][e]);
      }
    float al[2], unit[2];
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      mx[i] = fmaxf(mx[i], __shfl_xor_sync(0xffffffffu, mx[i], 1));
      mx[i] = fmaxf(mx[i], __shfl_xor_sync(0xffffffffu, mx[i], 2));
      al[i] = mx[i] == m[i] ? 1.f : fast_exp2(m[i] - mx[i]);
      unit[i] = mx[i] == -INFINITY ? 0.f : mx[i];
      m[i] = mx[i];
      l[i] *= al[i];
    }
    if (__any_sync(0xffffffffu, al[0] != 1.f || al[1] != 1.f)) {
#pragma unroll
      for (int j = 0; j < kMmaDim / 8; ++j) o[j][0] *= al[0], o[j][1] *= al[0], o[j][2] *= al[1], o[j][3] *= al[1];
    }
#pragma unroll
    for (int c = 0; c < kMmaKeys / 16; ++c) {
      uint32_t p[4];
#pragma unroll
      for (int x = 0; x < 2; ++x) {
        float(&y)[4] = s[2 * c + x];
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          y[e] = fast_exp2(y[e] - unit[e >> 1]);
          l[e >> 1] += y[e];
        }
        p[2 * x] = pack2<T>(y[0], y[1]);
        p[2 * x + 1] = pack2<T>(y[2], y[3]);
      }
#pragma unroll
      for (int j = 0; j < kMmaDim / 8; j += 2) {
        uint32_t b0, b1, b2, b3;
        ldmatrix_x4_trans(vs + mma_at(c * 16 + v_row, j + v_half), b0, b1, b2, b3);
        mma_16816<T>(o[j][0], o[j][1], o[j][2], o[j][3], p[0], p[1], p[2], p[3], b0, b1);
        mma_16816<T>(o[j + 1][0], o[j + 1][1], o[j + 1][2], o[j + 1][3], p[0], p[1], p[2], p[3], b2, b3);
      }
    }
  }
  asm volatile("cp.async.wait_group 0;" ::: "memory");
#pragma unroll
  for (int i = 0; i < 2; ++i) {
    l[i] += __shfl_xor_sync(0xffffffffu, l[i], 1);
    l[i] += __shfl_xor_sync(0xffffffffu, l[i], 2);
    const int64_t r = r0 + warp * 16 + g_row + 8 * i;
    if (r >= rows) continue;
    const int64_t t = r / a.g;
    T* dst = reinterpret_cast<T*>(a.out) + b * a.o_sb + (qo + t) * a.o_st + (h * a.g + (r - t * a.g)) * a.o_sh;
    // 0: no key seen, so zeros whatever the keys of the tile hold; a NaN sum stays NaN
    const bool none = l[i] == 0.f;
    const float inv = none ? 0.f : 1.f / l[i] * v_unit;
#pragma unroll
    for (int j = 0; j < kMmaDim / 8; ++j) {
      const int d = j * 8 + 2 * t4;
      if (d >= a.d) break;
      const float x = none ? 0.f : o[j][2 * i] * inv, y = none ? 0.f : o[j][2 * i + 1] * inv;
      if (a.o_pair) {
        *reinterpret_cast<uint32_t*>(dst + d) = pack2<T>(x, y);
      } else {
        dst[d] = from_f32<T>(x);
        dst[d + 1] = from_f32<T>(y);
      }
    }
  }
}

// ---------------------------------------------------------------------------
// SIMT kernel
// ---------------------------------------------------------------------------
constexpr int kBQ = 64, kBK = 64;
constexpr int kSimtThreads = 256;  // 16 x 16: a thread owns 4 queries x (4 keys | 4 dims of every 64)
constexpr int kPStride = kBK + 4;

struct SimtArgs {
  const void* q;
  int64_t q_sb, q_st, q_sh;
  void* out;
  int64_t o_sb, o_st, o_sh;
  const int32_t* q_offsets;
  const int32_t* seq_lens;
  const uint8_t* k_pool;
  const uint8_t* v_pool;
  const float* k_scale;
  const float* v_scale;
  const int32_t* block_tables;
  int64_t bt_stride, bt_width;
  const int32_t* row_ids;
  int64_t num_blocks, layer, max_q;
  int32_t hkv, g, bs, d, stride;  // stride: floats between rows of a shared tile
  float scale_log2;
  int32_t* err;
};

struct SimtShared {
  int64_t row[kBK];  // byte offset of the token's codes, -1: none
  float ks[kBK], vs[kBK];
};

// Rows of a shared tile start an odd number of 16-byte units apart, so 16
// threads reading 16 rows' float4 touch every bank once.
int tile_stride(int d) {
  int s = (d + 3) / 4 * 4 + 4;
  if ((s / 4) % 2 == 0) s += 4;
  return s;
}
size_t simt_smem(int d) {
  return sizeof(SimtShared) + sizeof(float) * ((size_t)(kBQ + kBK) * tile_stride(d) + kBQ * kPStride);
}

// S = q K^T and O += P V as outer products in registers: a thread's 4 x 4 block
// reads 8 float4 of shared memory for 64 multiplies.  4 chunks of 256..1024 tokens
// over 0..4k, 32 / 8 fp32 heads of 128 dims, 91 GFLOP: 3.7 ms, 24 TFLOP/s, a third of
// the fp32 pipe.  Packed products (two dims an instruction) and codes fetched a
// tile ahead by cp.async changed nothing (3.8, 3.7 ms).
// grid: (ceil(max_q / kBQ), hq, batch).  NC = ceil(head_dim / 64).
template <typename T, int NC>
__global__ void __launch_bounds__(kSimtThreads) fp8_prefill_simt_kernel(const SimtArgs a) {
  extern __shared__ __align__(16) unsigned char smem_raw[];
  SimtShared* sh = reinterpret_cast<SimtShared*>(smem_raw);
  float* qs = reinterpret_cast<float*>(smem_raw + sizeof(SimtShared));
  float* kv = qs + kBQ * a.stride;
  float* ps = kv + kBK * a.stride;
  const int tid = threadIdx.x, ty = tid >> 4, tx = tid & 15;
  const int64_t b = blockIdx.z;
  const int hq = blockIdx.y, h = hq / a.g;
  int64_t qo = 0, nq = a.max_q;
  if (a.q_offsets) {
    qo = a.q_offsets[b];
    nq = (int64_t)a.q_offsets[b + 1] - qo;
  }
  const int64_t q0 = ((int64_t)gridDim.x - 1 - blockIdx.x) * kBQ;  // the tiles with most keys first
  if (q0 >= nq) return;
  const int64_t len = a.seq_lens[b], prefix = len - nq;
  const int64_t kend = prefix + min(q0 + kBQ, nq);
  const int64_t row = a.row_ids ? (int64_t)a.row_ids[b] : b;
  const int d4 = (a.d + 3) / 4;

  const T* qp = reinterpret_cast<const T*>(a.q) + b * a.q_sb + (int64_t)hq * a.q_sh;
  for (int e = tid; e < kBQ * 4 * d4; e += kSimtThreads) {
    const int r = e / (4 * d4), d = e - r * 4 * d4;
    qs[r * a.stride + d] =
        (q0 + r < nq && d < a.d) ? to_f32<T>(qp[(qo + q0 + r) * a.q_st + d]) * a.scale_log2 : 0.f;
  }
  float m[4], l[4], o[4][NC][4];
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    m[i] = -INFINITY;
    l[i] = 0.f;
#pragma unroll
    for (int c = 0; c < NC; ++c) o[i][c][0] = o[i][c][1] = o[i][c][2] = o[i][c][3] = 0.f;
  }

  auto load_tile = [&](const uint8_t* pool, const float* sc) {
    const bool words = (a.d & 3) == 0;
    for (int e = tid; e < kBK * d4; e += kSimtThreads) {
      const int t = e / d4, c = e - t * d4;
      const int64_t r = sh->row[t];
      float4 x = make_float4(0.f, 0.f, 0.f, 0.f);
      if (r >= 0) {
        const float s = sc[t];
        if (words) {
          const uint32_t w = *reinterpret_cast<const uint32_t*>(pool + r + 4 * c);
          const float2 lo = e4m3x2_to_float2((uint16_t)w), hi = e4m3x2_to_float2((uint16_t)(w >> 16));
          x = make_float4(lo.x * s, lo.y * s, hi.x * s, hi.y * s);
        } else {
          const uint8_t* p = pool + r + 4 * c;
          const int n = a.d - 4 * c;
          x.x = e4m3_to_float(p[0]) * s;
          if (n > 1) x.y = e4m3_to_float(p[1]) * s;
          if (n > 2) x.z = e4m3_to_float(p[2]) * s;
          if (n > 3) x.w = e4m3_to_float(p[3]) * s;
        }
      }
      *reinterpret_cast<float4*>(kv + t * a.stride + 4 * c) = x;
    }
  };

  for (int64_t k0 = 0; k0 < kend; k0 += kBK) {
    __syncthreads();  // the previous tile (and ps) is no longer read; qs is complete
    if (tid < kBK) {
      const int64_t t = k0 + tid;
      int64_t r = -1;
      if (t < kend) {
        const int64_t lb = t / a.bs;
        if (lb >= a.bt_width) {
          raise_dev(a.err, BL_DEVERR_TABLE);
        } else {
          const int64_t phys = a.block_tables[row * a.bt_stride + lb];
          if (phys < 0 || phys >= a.num_blocks) {
            raise_dev(a.err, BL_DEVERR_BLOCK_ID);
          } else {
            const int64_t slot = (a.layer * a.num_blocks + phys) * a.hkv + h;
            r = (slot * a.bs + (t - lb * a.bs)) * a.d;
            sh->ks[tid] = a.k_scale[slot];
            sh->vs[tid] = a.v_scale[slot];
          }
        }
      }
      sh->row[tid] = r;
    }
    __syncthreads();
    load_tile(a.k_pool, sh->ks);
    __syncthreads();
    float s[4][4];
#pragma unroll
    for (int i = 0; i < 4; ++i) s[i][0] = s[i][1] = s[i][2] = s[i][3] = 0.f;
    for (int d = 0; d < d4; ++d) {
      float4 qv[4], kx[4];
#pragma unroll
      for (int i = 0; i < 4; ++i) qv[i] = *reinterpret_cast<const float4*>(qs + (ty * 4 + i) * a.stride + 4 * d);
#pragma unroll
      for (int j = 0; j < 4; ++j) kx[j] = *reinterpret_cast<const float4*>(kv + (tx + 16 * j) * a.stride + 4 * d);
#pragma unroll
      for (int i = 0; i < 4; ++i)
#pragma unroll
        for (int j = 0; j < 4; ++j)
          s[i][j] = fmaf(qv[i].x, kx[j].x, fmaf(qv[i].y, kx[j].y, fmaf(qv[i].z, kx[j].z, fmaf(qv[i].w, kx[j].w, s[i][j]))));
    }
    bool live[4];
#pragma unroll
    for (int j = 0; j < 4; ++j) live[j] = sh->row[tx + 16 * j] >= 0;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const int64_t last = prefix + q0 + ty * 4 + i - k0;  // last key of the tile that the query sees
      float mx = -INFINITY;
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        if (!live[j] || tx + 16 * j > last) s[i][j] = -INFINITY;
        mx = fmaxf(mx, s[i][j]);
      }
#pragma unroll
      for (int of = 1; of < 16; of <<= 1) mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, of));
      const float mn = fmaxf(m[i], mx);
      const float al = mn == m[i] ? 1.f : fast_exp2(m[i] - mn);
      const float u = mn == -INFINITY ? 0.f : mn;
      m[i] = mn;
      float sum = 0.f;
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const float p = fast_exp2(s[i][j] - u);
        sum += p;
        ps[(ty * 4 + i) * kPStride + tx + 16 * j] = p;
      }
      l[i] = l[i] * al + sum;  // this thread's keys; the 16 threads' sums are joined at the end
#pragma unroll
      for (int c = 0; c < NC; ++c) o[i][c][0] *= al, o[i][c][1] *= al, o[i][c][2] *= al, o[i][c][3] *= al;
    }
    __syncthreads();
    load_tile(a.v_pool, sh->vs);
    __syncthreads();
    for (int k = 0; k < kBK; k += 4) {
      float4 p[4];
#pragma unroll
      for (int i = 0; i < 4; ++i) p[i] = *reinterpret_cast<const float4*>(ps + (ty * 4 + i) * kPStride + k);
#pragma unroll
      for (int c = 0; c < NC; ++c) {
        const int col = tx * 4 + 64 * c;
        if (col < 4 * d4) {
#pragma unroll
          for (int w = 0; w < 4; ++w) {
            const float4 x = *reinterpret_cast<const float4*>(kv + (k + w) * a.stride + col);
#pragma unroll
            for (int i = 0; i < 4; ++i) {
              const float pw = w == 0 ? p[i].x : w == 1 ? p[i].y : w == 2 ? p[i].z : p[i].w;
              o[i][c][0] = fmaf(pw, x.x, o[i][c][0]);
              o[i][c][1] = fmaf(pw, x.y, o[i][c][1]);
              o[i][c][2] = fmaf(pw, x.z, o[i][c][2]);
              o[i][c][3] = fmaf(pw, x.w, o[i][c][3]);
            }
          }
        }
      }
    }
  }
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    float sum = l[i];
#pragma unroll
    for (int of = 1; of < 16; of <<= 1) sum += __shfl_xor_sync(0xffffffffu, sum, of);
    const int64_t r = q0 + ty * 4 + i;
    if (r >= nq) continue;
    T* op = reinterpret_cast<T*>(a.out) + b * a.o_sb + (qo + r) * a.o_st + (int64_t)hq * a.o_sh;
#pragma unroll
    for (int c = 0; c < NC; ++c)
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        const int d = tx * 4 + 64 * c + e;
        if (d < a.d) op[d] = from_f32<T>(sum == 0.f ? 0.f : o[i][c][e] / sum);
      }
  }
}

template <typename T, int NC>
int launch_simt_nc(const SimtArgs& k, dim3 grid, cudaStream_t s) {
  if (cudaFuncSetAttribute(fp8_prefill_simt_kernel<T, NC>, cudaFuncAttributeMaxDynamicSharedMemorySize,
                           (int)simt_smem(64 * NC)) != cudaSuccess) {
    set_error("fp8_prefill_simt_kernel: %s", cudaGetErrorString(cudaGetLastError()));
    return BL_ERR_LAUNCH;
  }
  fp8_prefill_simt_kernel<T, NC><<<grid, kSimtThreads, simt_smem(k.d), s>>>(k);
  BL_CHECK_LAUNCH("fp8_prefill_simt_kernel");
  return BL_OK;
}

template <typename T>
int launch_simt(const bl_prefill_fp8_args& a, cudaStream_t s) {
  const bl_paged_layer& kv = a.layer.kv;
  SimtArgs k;
  k.q = a.q;
  k.q_sb = a.q_stride_b, k.q_st = a.q_stride_t, k.q_sh = a.q_stride_h;
  k.out = a.out;
  k.o_sb = a.out_stride_b, k.o_st = a.out_stride_t, k.o_sh = a.out_stride_h;
  k.q_offsets = a.q_offsets;
  k.seq_lens = a.seq_lens;
  k.k_pool = (const uint8_t*)kv.k_pool;
  k.v_pool = (const uint8_t*)kv.v_pool;
  k.k_scale = a.layer.k_scale;
  k.v_scale = a.layer.v_scale;
  k.block_tables = kv.block_tables;
  k.bt_stride = kv.bt_stride;
  k.bt_width = kv.bt_width;
  k.row_ids = kv.row_ids;
  k.num_blocks = kv.num_blocks;
  k.layer = kv.layer;
  k.max_q = a.max_q_len;
  k.hkv = (int32_t)kv.num_kv_heads;
  k.g = (int32_t)(a.num_q_heads / kv.num_kv_heads);
  k.bs = (int32_t)kv.block_size;
  k.d = (int32_t)kv.head_dim;
  k.stride = tile_stride(k.d);
  k.scale_log2 = a.scale * kLog2e;
  k.err = a.err;
  dim3 grid((unsigned)((a.max_q_len + kBQ - 1) / kBQ), (unsigned)a.num_q_heads, (unsigned)a.batch);
  switch ((k.d + 63) / 64) {
    case 1: return launch_simt_nc<T, 1>(k, grid, s);
    case 2: return launch_simt_nc<T, 2>(k, grid, s);
    case 3: return launch_simt_nc<T, 3>(k, grid, s);
    default: return launch_simt_nc<T, 4>(k, grid, s);
  }
}

template <typename T>
int launch_mma(const bl_prefill_fp8_args& a, cudaStream_t s) {
  const bl_paged_layer& kv = a.layer.kv;
  MmaArgs k;
  k.q = a.q;
  k.q_sb = a.q_stride_b, k.q_st = a.q_stride_t, k.q_sh = a.q_stride_h;
  k.out = a.out;
  k.o_sb = a.out_stride_b, k.o_st = a.out_stride_t, k.o_sh = a.out_stride_h;
  k.q_offsets = a.q_offsets;
  k.seq_lens = a.seq_lens;
  k.k_pool = (const uint8_t*)kv.k_pool;
  k.v_pool = (const uint8_t*)kv.v_pool;
  k.k_scale = a.layer.k_scale;
  k.v_scale = a.layer.v_scale;
  k.block_tables = kv.block_tables;
  k.bt_stride = kv.bt_stride;
  k.bt_width = kv.bt_width;
  k.row_ids = kv.row_ids;
  k.num_blocks = kv.num_blocks;
  k.layer = kv.layer;
  k.max_q = a.max_q_len;
  k.hkv = (int32_t)kv.num_kv_heads;
  k.g = (int32_t)(a.num_q_heads / kv.num_kv_heads);
  k.bs = (int32_t)kv.block_size;
  k.d = (int32_t)kv.head_dim;
  k.q_vec = ((uintptr_t)a.q & 15) == 0 && a.q_stride_b % 8 == 0 && a.q_stride_t % 8 == 0 && a.q_stride_h % 8 == 0;
  k.o_pair = ((uintptr_t)a.out & 3) == 0 && a.out_stride_b % 2 == 0 && a.out_stride_t % 2 == 0 && a.out_stride_h % 2 == 0;
  k.scale_log2 = a.scale * kLog2e;
  k.err = a.err;
  const int64_t tiles = (a.max_q_len * k.g + kMmaRows - 1) / kMmaRows;
  BL_CHECK_ARG(tiles <= INT32_MAX, "bl_paged_prefill_fp8: too many queries");
  const size_t smem = sizeof(MmaShared) + 128;
  if (cudaFuncSetAttribute(fp8_prefill_mma_kernel<T>, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)smem) !=
      cudaSuccess) {
    set_error("fp8_prefill_mma_kernel: %s", cudaGetErrorString(cudaGetLastError()));
    return BL_ERR_LAUNCH;
  }
  fp8_prefill_mma_kernel<T>
      <<<dim3((unsigned)tiles, (unsigned)k.hkv, (unsigned)a.batch), kMmaThreads, smem, s>>>(k);
  BL_CHECK_LAUNCH("fp8_prefill_mma_kernel");
  return BL_OK;
}

template <typename T>
int launch_tc(const bl_prefill_fp8_args& a, const Scratch& w, cudaStream_t s) {
  const bl_paged_layer& kv = a.layer.kv;
  char* ws = (char*)a.workspace;
  // the attention kernel's q and out: the caller's, or widened copies
  const bool wide = kv.head_dim < kTCDim;
  const void* q = a.q;
  void* out = a.out;
  int64_t q_sb = a.q_stride_b, q_st = a.q_stride_t, q_sh = a.q_stride_h;
  int64_t o_sb = a.out_stride_b, o_st = a.out_stride_t, o_sh = a.out_stride_h;
  WidenArgs x;
  if (wide) {
    x.offsets = a.q_offsets;
    x.batch = a.batch;
    x.max_q = a.max_q_len;
    x.total = a.total_q_len;
    x.hq = (int32_t)a.num_q_heads;
    x.d = (int32_t)kv.head_dim;
    x.narrow = const_cast<void*>(a.q);
    x.wide = ws + w.q;
    x.sb = q_sb, x.st = q_st, x.sh = q_sh;
    const int rc = launch_widen<T, true>(x, s);
    if (rc) return rc;
    q = ws + w.q;
    out = ws + w.out;
    q_sh = o_sh = kTCDim;
    q_st = o_st = a.num_q_heads * kTCDim;
    q_sb = o_sb = a.q_offsets ? 0 : a.max_q_len * q_st;
  }
  ExpandArgs e;
  e.k_pool = (const uint8_t*)kv.k_pool;
  e.v_pool = (const uint8_t*)kv.v_pool;
  e.k_scale = a.layer.k_scale;
  e.v_scale = a.layer.v_scale;
  e.k_out = ws + w.k;
  e.v_out = ws + w.v;
  e.table = (int32_t*)(ws + w.table);
  e.order = (int32_t*)(ws + w.order);
  e.k_unit = (float*)(ws + w.units);
  e.v_unit = e.k_unit + a.batch * w.heads;
  e.num_blocks = kv.num_blocks;
  e.layer = kv.layer;
  e.width = w.width;
  e.pages = w.pages;
  e.bt_stride = kv.bt_stride;
  e.bt_width = kv.bt_width;
  e.block_tables = kv.block_tables;
  e.row_ids = kv.row_ids;
  e.seq_lens = a.seq_lens;
  e.q_offsets = a.q_offsets;
  e.max_q = a.max_q_len;
  e.out = out;
  e.o_sb = o_sb, e.o_st = o_st, e.o_sh = o_sh;
  e.hkv = (int32_t)kv.num_kv_heads;
  e.bs = (int32_t)kv.block_size;
  e.bs_shift = -1;
  for (int i = 0; i <= 16; ++i)
    if (kv.block_size == 1 << i) e.bs_shift = i;
  e.d = (int32_t)kv.head_dim;
  e.dup = (int32_t)w.dup;
  e.hq = (int32_t)a.num_q_heads;
  e.err = a.err;
  dim3 grid((unsigned)((w.width + kExpandPages - 1) / kExpandPages), (unsigned)e.hkv, (unsigned)a.batch);
  e.own_units = std::min(kv.bt_width, (a.max_seq_len + kv.block_size - 1) / kv.block_size) <= kOwnUnitBlocks;
  if (std::is_same<T, __half>::value && !e.own_units) {
    fp8_units_kernel<<<dim3((unsigned)e.hkv, (unsigned)a.batch), kExpandThreads, 0, s>>>(e);
    BL_CHECK_LAUNCH("fp8_units_kernel");
    if (launch_pdl(fp8_expand_kernel<T>, grid, dim3(kExpandThreads), 0, s, e) != cudaSuccess) {
      set_error("fp8_expand_kernel: launch failed: %s", cudaGetErrorString(cudaGetLastError()));
      return BL_ERR_LAUNCH;
    }
  } else {
    fp8_expand_kernel<T><<<grid, kExpandThreads, 0, s>>>(e);
    BL_CHECK_LAUNCH("fp8_expand_kernel");
  }

  bl_prefill_args p;
  memset(&p, 0, sizeof(p));
  p.kv.k_pool = e.k_out;
  p.kv.v_pool = e.v_out;
  p.kv.num_layers = 1;
  p.kv.num_blocks = w.pages;
  p.kv.num_kv_heads = w.heads;
  p.kv.block_size = kPage;
  p.kv.head_dim = kTCDim;
  p.kv.dtype = kv.dtype;
  p.kv.layer = 0;
  p.kv.block_tables = e.table;
  p.kv.bt_stride = w.width;
  p.kv.bt_width = w.width;
  p.kv.row_ids = nullptr;
  p.q = q;
  p.q_stride_b = q_sb, p.q_stride_t = q_st, p.q_stride_h = q_sh;
  p.out = out;
  p.out_stride_b = o_sb, p.out_stride_t = o_st, p.out_stride_h = o_sh;
  p.q_offsets = a.q_offsets;
  p.seq_lens = a.seq_lens;
  p.batch = a.batch;
  p.num_q_heads = a.num_q_heads;
  p.max_q_len = a.max_q_len;
  p.scale = a.scale;
  p.err = a.err;
  const Expansion expansion = {e.order, e.k_unit, e.v_unit};
  const int rc = prefill_tc_launch(p, s, &expansion);
  if (rc || !wide) return rc;
  x.narrow = a.out;
  x.wide = out;
  x.sb = a.out_stride_b, x.st = a.out_stride_t, x.sh = a.out_stride_h;
  return launch_widen<T, false>(x, s);
}

// Strides and pointers that the tcgen05 kernel reads pairs of elements through
// (widened copies have them by themselves).
bool tc_alignment(const bl_prefill_fp8_args& a) {
  if (a.layer.kv.head_dim < kTCDim) return true;
  return ((uintptr_t)a.q & 3) == 0 && ((uintptr_t)a.out & 3) == 0 && a.q_stride_b % 2 == 0 && a.q_stride_t % 2 == 0 &&
         a.q_stride_h % 2 == 0 && a.out_stride_b % 2 == 0 && a.out_stride_t % 2 == 0 && a.out_stride_h % 2 == 0;
}

}  // namespace
}  // namespace bl

using namespace bl;

extern "C" size_t bl_paged_prefill_fp8_workspace_bytes(int32_t dtype, int64_t batch, int64_t num_q_heads,
                                                       int64_t num_kv_heads, int64_t head_dim, int64_t block_size,
                                                       int64_t total_q_len, int64_t max_seq_len, int64_t total_blocks) {
  if (batch <= 0 || total_q_len <= 0 || num_kv_heads <= 0 || num_q_heads <= 0 || num_q_heads % num_kv_heads || block_size <= 0 ||
      max_seq_len <= 0 || total_blocks <= 0 || !use_tc(dtype, head_dim))
    return 0;
  Scratch w;
  return plan_scratch(dtype, batch, num_q_heads, num_kv_heads, head_dim, block_size, total_q_len, max_seq_len, total_blocks, &w)
             ? w.total
             : 0;
}

extern "C" int bl_paged_prefill_fp8(const bl_prefill_fp8_args* args, void* stream) {
  const char* who = "bl_paged_prefill_fp8";
  BL_CHECK_ARG(args != nullptr, "%s: args is null", who);
  const bl_prefill_fp8_args& a = *args;
  const int rc = check_fp8_layer(a.layer, who);
  if (rc) return rc;
  const bl_paged_layer& kv = a.layer.kv;
  BL_CHECK_ARG(a.q && a.out && a.seq_lens, "%s: null q/out/seq_lens", who);
  BL_CHECK_ARG(a.batch > 0 && a.batch <= 65535, "%s: batch must be in [1, 65535]", who);
  BL_CHECK_ARG(a.num_q_heads > 0 && a.num_q_heads <= 65535 && a.num_q_heads % kv.num_kv_heads == 0,
               "num_heads must divide evenly by num_kv_heads");
  BL_CHECK_ARG(a.max_q_len > 0 && a.max_q_len <= INT32_MAX, "K/V sequence length must be greater than zero");
  BL_CHECK_ARG(a.max_seq_len > 0 && a.max_seq_len <= INT32_MAX, "%s: max_seq_len must be in [1, 2^31)", who);
  BL_CHECK_ARG(a.total_blocks > 0, "%s: total_blocks must be positive", who);
  BL_CHECK_ARG(a.total_q_len >= (a.q_offsets ? 1 : a.batch * a.max_q_len) && a.total_q_len <= INT32_MAX,
               "%s: total_q_len does not cover the queries", who);
  const int es = elem_size(kv.dtype);
  BL_CHECK_ARG(((uintptr_t)a.q % es) == 0 && ((uintptr_t)a.out % es) == 0,
               "%s: q/out must be aligned to their element type", who);
  cudaStream_t s = (cudaStream_t)stream;
  Scratch w;
  if (use_tc(kv.dtype, kv.head_dim) && tc_alignment(a) &&
      plan_scratch(kv.dtype, a.batch, a.num_q_heads, kv.num_kv_heads, kv.head_dim, kv.block_size, a.total_q_len, a.max_seq_len,
                   a.total_blocks, &w)) {
    if (!a.workspace || a.workspace_bytes < w.total) {
      set_error("%s: workspace too small (%zu < %zu bytes)", who, a.workspace ? a.workspace_bytes : (size_t)0, w.total);
      return BL_ERR_CAPACITY;
    }
    BL_CHECK_ARG(((uintptr_t)a.workspace & 255) == 0, "%s: workspace must be 256-byte aligned", who);
    return kv.dtype == BL_BF16 ? launch_tc<__nv_bfloat16>(a, w, s) : launch_tc<__half>(a, w, s);
  }
  if (use_mma(kv.dtype, kv.head_dim)) return kv.dtype == BL_BF16 ? launch_mma<__nv_bfloat16>(a, s) : launch_mma<__half>(a, s);
  switch (kv.dtype) {
    case BL_F32: return launch_simt<float>(a, s);
    case BL_F16: return launch_simt<__half>(a, s);
    default: return launch_simt<__nv_bfloat16>(a, s);
  }
}
