// Decode attention over an 8-bit paged cache (one query token per request, GQA):
//   out[b, hq] = softmax_t(scale * q[b, hq] . K[b, h, t]) V[b, h, t],  t < len_b,
// with K = code * k_scale[block, h], V = code * v_scale[block, h] (fp8.cuh).
// 8-bit counterpart of decode.cu; the reference chain it stands for is
// SDPAAttentionBackend.attend, src/barellm/attention/backend.py:34-61.
//
// Kernels
//   fp8_decode_plan_kernel one CTA.  Splits rows into 512-token chunks and lists
//                          the units, full chunks first, then partial ones by
//                          decreasing size.
//   fp8_decode_tc_kernel   bf16 / fp16 q, head_dim a multiple of 16, block_size
//                          one of 8.  Built for 64, 128 and 256 dims; the copies
//                          fill the dims up to the next of these with zeros.
//                          Persistent CTAs claim (chunk, KV head, 8 query heads)
//                          items.  A planner warp describes the next item (query
//                          fragments, page rows, scales) while four consumer
//                          warps work on one, each on every fourth step of 32
//                          tokens, copied by TMA into a ring of its own.
//   fp8_decode_simt_kernel everything else (fp32 q, other head_dims and block
//                          sizes, pools past the tensor map's 2^31 rows): the
//                          same chunks, fp32 multiplies in registers.
//   fp8_decode_reduce_kernel  joins the chunks of rows that have several.
//
// Arithmetic of the tensor-core kernel.  Codes are converted to fp16, which
// holds every e4m3 value exactly, and the two products run on mma.sync
// m16n8k16 with fp32 sums.  q is brought to fp16 by a power of two per head
// (its largest magnitude lands in [1, 2)), so a bf16 element keeps all its bits
// down to 2^-16 of the head's largest and loses at most 2^-25 of that below.
// k_scale multiplies the score in fp32.  P (<= 2^8, see below) is rounded to
// fp16, half a step of 2^-11 relative.  V's scales are powers of two: a tile's is
// folded into its P relative to the tile that set the sums' unit, or applied to
// sums of its own where it is far smaller.
//
// What bounds it (64 requests of 1k..32k tokens, 32 / 8 heads, head_dim 128, bf16:
// 2.12 GB): HBM, while the chip is cool: plan, attention and join together 353 us, 5.99 TB/s,
// the attention kernel alone 339 us, 6.25 TB/s (a copy on this card: 6.56).  Under a
// load that goes on for 100 ms the card reaches its power cap and the SM
// clock falls to 1.6 GHz; the conversions and products then take longer than
// the copies (calls in a loop: 388..406 us, 5.2..5.45 TB/s; without them 343 us).  The
// three CTAs per SM leave 128 registers, of which the 128-dim kernel spills 56
// bytes (68 at block sizes of 8).  Measured and not kept: one
// producer warp for the CTA (375 us without any arithmetic), rings of 4 steps a
// warp or 2 CTAs per SM with larger rings (more than 96 KB in flight per SM is
// slower), 4 CTAs of 96 registers (425 us), static rounds in place of claims (373 us).
#include <cstddef>
#include <cstring>
#include <mutex>
#include <type_traits>

#include "fp8.cuh"

namespace bl {
namespace {

constexpr int kChunk = 512;  // tokens; fixed, so that a row's result does not depend on the batch
constexpr int kChunkTiles = kChunk / 16;
constexpr int32_t kPlanMagic = 0x38504c46;
constexpr float kLog2e = 1.4426950408889634f;

inline size_t align256(size_t x) { return (x + 255) & ~size_t(255); }

// One chunk of a row, as the plan records it.
struct alignas(16) Unit {
  int32_t row, chunk, len, part;  // len: the row's length, at most what its table covers; part: slot of its partial
};

struct WsLayout {
  size_t hdr, row_base, units, lse, o, total;
  int64_t max_units;
};

WsLayout ws_layout(int64_t batch, int64_t hq, int64_t d, int64_t max_seq_len) {
  WsLayout w;
  w.max_units = batch * ((max_seq_len + kChunk - 1) / kChunk);
  size_t off = 0;
  w.hdr = off;      off += align256(8 * sizeof(int32_t));
  w.row_base = off; off += align256((batch + 1) * sizeof(int32_t));
  w.units = off;    off += align256(w.max_units * sizeof(Unit));
  // a row of one chunk leaves no partial
  const int64_t parts = max_seq_len > kChunk ? w.max_units : 0;
  w.lse = off;      off += align256(parts * hq * sizeof(float));
  w.o = off;        off += align256(parts * hq * d * sizeof(float));
  w.total = off;
  return w;
}

// ---------------------------------------------------------------------------
// plan
// ---------------------------------------------------------------------------
constexpr int kPlanThreads = 1024;  // at most; a batch of fewer rows takes fewer

struct PlanArgs {
  const int32_t* seq_lens;
  int32_t batch, max_units;
  int64_t cap;        // tokens a table row covers
  int32_t* hdr;       // [0] units, [1] magic, [2] batch, [3] max_units, [4..5] items claimed, [6] CTAs done
  int32_t* row_base;  // [batch + 1]
  Unit* units;        // [max_units]
  int32_t* err;
};

// Exclusive sums of v over the CTA; total over all.  s: an int per warp.
__device__ __forceinline__ int cta_exclusive(int v, int* s, int& total) {
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  int x = v;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const int y = __shfl_up_sync(0xffffffffu, x, o);
    if (lane >= o) x += y;
  }
  if (lane == 31) s[warp] = x;
  __syncthreads();
  int before = 0;
  total = 0;
  for (int w = 0; w < (int)(blockDim.x >> 5); ++w) {
    const int t = s[w];
    if (w < warp) before += t;
    total += t;
  }
  __syncthreads();
  return before + x - v;
}

__global__ void __launch_bounds__(kPlanThreads) fp8_decode_plan_kernel(const PlanArgs a) {
  pdl_trigger();  // the attention kernel may launch; it waits for this grid (and for those before it) to complete
  // Nothing is read or written before the kernel ahead has completed: it may be what
  // writes the lengths or the row ids, and the workspace may be memory that it still
  // reads (an append's tokens, freed since; the plan of the call before).
  pdl_wait();
  __shared__ int s_sum[kPlanThreads / 32];
  __shared__ int s_count[kChunkTiles], s_next[kChunkTiles];  // partial chunks by size in tiles, minus one
  const int tid = threadIdx.x;
  if (tid < kChunkTiles) s_count[tid] = 0;
  __syncthreads();
  auto put = [&](int pos, int row, int chunk, int len, int base) {
    if ((uint32_t)pos >= (uint32_t)a.max_units) return;  // (rows far past max_seq_len may wrap the sums)
    *reinterpret_cast<int4*>(a.units + pos) = make_int4(row, chunk, len, base + chunk);
  };
  auto length = [&](int b) {
    const int64_t len = a.seq_lens[b];
    return (int)min(max(len, (int64_t)0), a.cap);
  };
  int all = 0, full = 0;
  for (int b0 = 0; b0 < a.batch; b0 += blockDim.x) {
    const int b = b0 + tid;
    const int len = b < a.batch ? length(b) : 0;
    const int nfull = len / kChunk, nall = (int)(((int64_t)len + kChunk - 1) / kChunk);
    int tot_all, tot_full;
    const int my_all = all + cta_exclusive(nall, s_sum, tot_all);
    const int my_full = full + cta_exclusive(nfull, s_sum, tot_full);
    if (b < a.batch) {
      if (a.seq_lens[b] > a.cap) raise_dev(a.err, BL_DEVERR_TABLE);
      a.row_base[b] = my_all;
      for (int c = 0; c < nfull; ++c) put(my_full + c, b, c, len, my_all);
      if (nall > nfull) atomicAdd(&s_count[(len - nfull * kChunk + 15) / 16 - 1], 1);
    }
    all += tot_all;
    full += tot_full;
  }
  __syncthreads();
  if (tid < kChunkTiles) {
    int pos = full;  // partial chunks follow the full ones, the largest first
    for (int s = tid + 1; s < kChunkTiles; ++s) pos += s_count[s];
    s_next[tid] = pos;
  }
  if (tid == 0) {
    if (all > a.max_units) raise_dev(a.err, BL_DEVERR_WORKSPACE);  // a row is longer than max_seq_len
    a.row_base[a.batch] = all;
    a.hdr[0] = min(all, a.max_units);
    a.hdr[1] = kPlanMagic;
    a.hdr[2] = a.batch;
    a.hdr[3] = a.max_units;
    a.hdr[4] = a.hdr[5] = a.hdr[6] = 0;
  }
  __syncthreads();
  // (the order among chunks of one size is left to the atomics: it changes no result)
  for (int b = tid; b < a.batch; b += blockDim.x) {
    const int len = length(b), nfull = len / kChunk, rest = len - nfull * kChunk;
    if (rest > 0)
      put(atomicAdd(&s_next[(rest + 15) / 16 - 1], 1), b, nfull, len, a.row_base[b]);
  }
}

struct Args {
  const void* q;
  int64_t q_sb, q_sh;
  void* out;
  int64_t o_sb, o_sh;
  const uint8_t* k_pool;
  const uint8_t* v_pool;
  const float* k_scale;
  const float* v_scale;
  const int32_t* block_tables;
  int64_t bt_stride, bt_width;
  const int32_t* row_ids;
  const int32_t* seq_lens;
  int64_t num_blocks, layer;
  int32_t batch, hq, hkv, g, bs, d;
  int32_t tile_heads, head_tiles;  // query heads of an item, at most; items of a KV head
  int32_t q_vec, o_vec;  // q (of a head_dim that the kernel is built for) / out go four 16-bit elements at a time
  float scale_log2;
  int32_t* hdr;
  const int32_t* row_base;
  const Unit* units;
  float* ws_lse;
  float* ws_o;
  int32_t max_units, has_parts;
  int32_t planned;  // 0: a small call without a plan; every CTA has at most one item
  int32_t cluster;  // > 0 (a small call): a row's chunks are the CTAs of a cluster of this size, which joins them itself
  int32_t* err;
};

// One item: a chunk of a row, a KV head and up to tile_heads of its query heads.
struct Item {
  int b, h, hq0, heads;
  int t0, t1;     // the chunk's tokens are [t0, t1)
  int nch, part;  // chunks of the row, slot of this one's partial
  int table_row;
};

// Unit u of a small batch (at most 32 rows), found by one warp from the lengths
// alone: row by row, chunk by chunk, as the plan numbers the partials.  Lane b
// stands for row b.  `units`: their number.
__device__ __forceinline__ Unit find_unit(const Args& a, int u, int lane, int& units) {
  int64_t len = lane < a.batch ? (int64_t)a.seq_lens[lane] : 0;
  const int64_t cap = a.bt_width * a.bs;
  if (len > cap) {
    if (blockIdx.x == 0) raise_dev(a.err, BL_DEVERR_TABLE);
    len = cap;
  }
  const int n = len > 0 ? (int)((len + kChunk - 1) / kChunk) : 0;
  int incl = n;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const int y = __shfl_up_sync(0xffffffffu, incl, o);
    if (lane >= o) incl += y;
  }
  units = __shfl_sync(0xffffffffu, incl, 31);
  const uint32_t past = __ballot_sync(0xffffffffu, incl > u);
  Unit r = {};
  r.row = past ? __ffs(past) - 1 : 0;
  r.chunk = u - __shfl_sync(0xffffffffu, incl - n, r.row);
  r.len = __shfl_sync(0xffffffffu, (int)len, r.row);
  r.part = u;
  return r;
}

// The unit of this CTA in a call whose clusters are rows.
__device__ __forceinline__ Unit cluster_unit(const Args& a, bool tell) {
  Unit r = {};
  const int c = blockIdx.x / a.cluster;
  r.chunk = blockIdx.x - c * a.cluster;
  r.row = c / (a.hkv * a.head_tiles);
  int64_t len = a.seq_lens[r.row];
  const int64_t cap = a.bt_width * a.bs;
  if (len > cap) {
    if (tell) raise_dev(a.err, BL_DEVERR_TABLE);
    len = cap;
  }
  if (len > (int64_t)a.cluster * kChunk && tell) raise_dev(a.err, BL_DEVERR_WORKSPACE);  // longer than max_seq_len
  r.len = (int)max(len, (int64_t)0);
  return r;
}

__device__ __forceinline__ Unit load_unit(const Args& a, int64_t item) {
  const int4 x = *reinterpret_cast<const int4*>(a.units + item / (a.hkv * a.head_tiles));
  Unit u;
  u.row = x.x, u.chunk = x.y, u.len = x.z, u.part = x.w;
  return u;
}

// False when the plan names a unit outside the batch or the table.
__device__ __forceinline__ bool make_item(const Args& a, int64_t item, const Unit& u, Item& it) {
  const int r = (int)(item % (a.hkv * a.head_tiles));
  it.h = r / a.head_tiles;
  const int ht = r - it.h * a.head_tiles;
  it.hq0 = it.h * a.g + ht * a.tile_heads;
  it.heads = min(a.tile_heads, a.g - ht * a.tile_heads);
  it.b = u.row;
  it.part = u.part;
  it.t0 = u.chunk * kChunk;
  it.t1 = min(it.t0 + kChunk, u.len);
  it.nch = (u.len + kChunk - 1) / kChunk;
  const bool ok = u.row >= 0 && u.row < a.batch && (uint32_t)u.chunk <= (uint32_t)(INT32_MAX - kChunk) / kChunk &&
                  it.t0 < u.len && u.len <= a.bt_width * a.bs;
  it.table_row = ok && a.row_ids ? a.row_ids[u.row] : u.row;
  if (!ok) it.t0 = it.t1 = it.heads = 0;  // no steps, no outputs
  return ok;
}

__device__ __forceinline__ int plan_units(const Args& a, bool tell) {
  const int units = a.hdr[0];
  if (a.hdr[1] != kPlanMagic || a.hdr[2] != a.batch || a.hdr[3] != a.max_units || units < 0 || units > a.max_units) {
    if (tell && blockIdx.x == 0) raise_dev(a.err, BL_DEVERR_WORKSPACE);
    return 0;
  }
  return units;
}

// Rows without tokens have no unit in the plan: their outputs are zeros.
template <typename T>
__device__ __forceinline__ void zero_empty_rows(const Args& a, int nthreads) {
  for (int b = blockIdx.x; b < a.batch; b += gridDim.x) {
    if (a.seq_lens[b] > 0) continue;
    for (int e = threadIdx.x; e < a.hq * a.d; e += nthreads) {
      const int h = e / a.d;
      reinterpret_cast<T*>(a.out)[(int64_t)b * a.o_sb + (int64_t)h * a.o_sh + (e - h * a.d)] = from_f32<T>(0.f);
    }
  }
}

// Whether the item's partial has a place in the workspace (it has none where a
// row is longer than max_seq_len).
__device__ __forceinline__ bool has_part(const Args& a, const Item& it) {
  return a.has_parts && it.part >= 0 && it.part < a.max_units;
}

// ---------------------------------------------------------------------------
// tensor-core kernel
// ---------------------------------------------------------------------------
constexpr int kNW = 4;                      // consumer warps
constexpr int kThreadsTC = (kNW + 1) * 32;  // + the planner warp
constexpr int kStepTokens = 32;             // tokens a consumer warp takes at a time: two 16-token tiles
constexpr int kTiles = kChunkTiles;         // 16-token tiles of a chunk, one per planner lane
static_assert(kTiles == 32, "a planner lane holds one tile of the chunk");

template <int D>
struct Cfg {
  static constexpr int kRow = D < 128 ? D : 128;  // bytes of a token row in one TMA box
  static constexpr int kHalves = D / kRow;
  static constexpr int kTile = 16 * D;            // K (or V) codes of one tile
  static constexpr int kSlot = 4 * kTile;         // K and V of two tiles
  static constexpr int kDepth = D == 64 ? 4 : 2;  // ring slots of a consumer warp
  static constexpr int kBox = 16 * kRow;
  static constexpr int kKS = D / 16;              // 16-dim steps of the score product
  static constexpr int kLaneDims = kRow / 8;      // output dims a lane owns per half
  static constexpr int kWords = kLaneDims / 4;    // V words a lane reads per token and half
  static constexpr int kVecs = D / 16;            // float4s of sums a lane holds (two heads)
};

// What the planner warp hands to the consumers, an item at a time.  NP: pieces of
// a tile that lie in one block: one of 16 tokens, or two of 8 where the block
// size is no multiple of 16.
template <int D, int NP>
struct alignas(16) ItemSlot {
  float2 f[4];                             // score factors of heads 2t and 2t + 1
  int32_t y[kTiles * NP];                  // pool row of each piece
  float ks[kTiles * NP], vs[kTiles * NP];  // its scales
  Item it;
};

template <int D, int NP>
struct alignas(16) TCShared {  // the query fragments and the merge buffer behind it are read 16 bytes at a time
  ItemSlot<D, NP> items[2];
  float2 ml[kNW][8];  // maximum and sum of each class and head
  uint64_t full[kNW][Cfg<D>::kDepth];
  uint64_t item_full[2], item_empty[2];
  uint64_t comb_full, comb_free;
  int abort;
};

// 16-byte chunk `c` of token row `r` within a box, as TMA's swizzle places it
template <int ROW>
__device__ __forceinline__ int swizzled(int r, int c) {
  return r * ROW + ((ROW == 128 ? (c ^ (r & 7)) : (c ^ ((r >> 1) & 3))) << 4);
}

// D += A(16x16) * B(16x8) in fp16 with fp32 sums.  Not volatile: a pure function
// of its registers, so the compiler may interleave independent products.
__device__ __forceinline__ void mma_f16(float (&c)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0,
                                        uint32_t b1) {
  asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, "
      "{%0, %1, %2, %3};"
      : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
      : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}

// Waits unless the CTA gave up; a wait that runs out (2 s) makes it give up.  A
// waiting warp sleeps in the barrier unit up to the hint's time, so that it does
// not take issue slots from the others.
__device__ __forceinline__ bool wait_or_abort(uint64_t* bar, uint32_t parity, int* abort, int32_t* err) {
  if (mbar_try_wait(bar, parity)) return true;
  const uint64_t t0 = global_timer_ns();
  while (true) {
    uint32_t done;
    asm volatile(
        "{\n\t.reg .pred p;\n\t"
        "mbarrier.try_wait.parity.shared::cta.b64 p, [%1], %2, %3;\n\t"
        "selp.u32 %0, 1, 0, p;\n\t}"
        : "=r"(done)
        : "r"(smem_u32(bar)), "r"(parity), "r"(20000u)
        : "memory");
    if (done) return true;
    if (*(volatile int*)abort) return false;
    if (global_timer_ns() - t0 > 2000000000ull) {
      raise_dev(err, BL_DEVERR_TIMEOUT);
      *(volatile int*)abort = 1;
      return false;
    }
  }
}

// An item on its way to the consumers: lane i holds tile i of the chunk.  begin()
// makes the loads that the plan's record leads to, finish() those behind the
// block id.
template <typename T, int D, int NP>
struct Pending {
  Item it;
  bool valid;
  int tok, lb[NP];
  int32_t phys[NP], y[NP];
  float ks[NP], vs[NP];
  uint2 q[Cfg<D>::kKS];  // dims 16 k + 4 t + {0..3} of head g, as stored

  __device__ __forceinline__ void begin(const Args& a, int64_t item, const Unit& u, int lane) {
    valid = make_item(a, item, u, it);
    tok = it.t0 + 16 * lane;
#pragma unroll
    for (int p = 0; p < NP; ++p) {
      const int t = tok + p * (16 / NP);
      lb[p] = t / a.bs;
      phys[p] = 0;
      if (t < it.t1) phys[p] = a.block_tables[(int64_t)it.table_row * a.bt_stride + lb[p]];
    }
    const int g_row = lane >> 2, t4 = lane & 3;
    const T* qp = reinterpret_cast<const T*>(a.q) + (int64_t)(valid ? it.b : 0) * a.q_sb +
                  (int64_t)(it.hq0 + (g_row < it.heads ? g_row : 0)) * a.q_sh + 4 * t4;
#pragma unroll
    for (int k = 0; k < Cfg<D>::kKS; ++k) {
      if (a.q_vec) {
        q[k] = *reinterpret_cast<const uint2*>(qp + k * 16);
      } else if (k * 16 >= a.d) {
        q[k] = make_uint2(0u, 0u);  // (the codes there are zeros)
      } else {
        const T* p = qp + k * 16;
        q[k] = make_uint2(pack2<T>(to_f32<T>(p[0]), to_f32<T>(p[1])), pack2<T>(to_f32<T>(p[2]), to_f32<T>(p[3])));
      }
    }
  }

  __device__ __forceinline__ void finish(const Args& a) {
#pragma unroll
    for (int p = 0; p < NP; ++p) {
      const int t = tok + p * (16 / NP);
      if (t < it.t1) {
        int64_t b = phys[p];
        if (b < 0 || b >= a.num_blocks) {
          raise_dev(a.err, BL_DEVERR_BLOCK_ID);
          b = 0;
        }
        const int64_t slot = (a.layer * a.num_blocks + b) * a.hkv + it.h;
        ks[p] = a.k_scale[slot];
        vs[p] = a.v_scale[slot];
        y[p] = (int32_t)(slot * a.bs + (t - lb[p] * a.bs));
      } else {
        // a missing second piece repeats the first one (no effect: its codes are masked)
        y[p] = p ? y[0] : 0;
        ks[p] = p ? ks[0] : 1.f;
        vs[p] = p ? vs[0] : 1.f;
      }
    }
  }

  // The query heads as fp16 B fragments and score factors, for this lane.
  // Position k of a 16-dim step stands for dim 16 ks + 4 t + {0, 1} (k = 2t,
  // 2t+1) and + {2, 3} (k = 2t+8, 2t+9): the order in which a lane finds the K
  // codes of one 32-bit word.
  // Lanes of heads that the item does not have store nothing: `qs` has room for
  // min(g, 8) heads, lane by lane.
  __device__ __forceinline__ void stage(const Args& a, int lane, ItemSlot<D, NP>& out, uint2* qs) const {
    const int t4 = lane & 3, room = 4 * min(a.g, 8);
    float amax = 0.f;
#pragma unroll
    for (int k = 0; k < Cfg<D>::kKS; ++k) {
      const float2 x = unpack2<T>(q[k].x), y2 = unpack2<T>(q[k].y);
      amax = fmaxf(fmaxf(amax, fmaxf(finite_abs(x.x), finite_abs(x.y))), fmaxf(finite_abs(y2.x), finite_abs(y2.y)));
    }
    amax = fmaxf(amax, __shfl_xor_sync(0xffffffffu, amax, 1));
    amax = fmaxf(amax, __shfl_xor_sync(0xffffffffu, amax, 2));
    int e = (int)(__float_as_uint(amax) >> 23) - 127;
    e = amax > 0.f ? min(max(e, -126), 126) : 0;
    const float down = exp2_int(-e);
#pragma unroll
    for (int k = 0; k < Cfg<D>::kKS; ++k) {
      const float2 x = unpack2<T>(q[k].x), y2 = unpack2<T>(q[k].y);
      const uint2 v = make_uint2(pack2<__half>(x.x * down, x.y * down), pack2<__half>(y2.x * down, y2.y * down));
      if (lane < room) qs[k * room + lane] = v;
    }
    const float f = exp2_int(e) * a.scale_log2;
    const float f0 = __shfl_sync(0xffffffffu, f, 8 * t4);
    const float f1 = __shfl_sync(0xffffffffu, f, 8 * t4 + 4);
    if (lane < 4) out.f[lane] = make_float2(f0, f1);
    // a step with one tile repeats its V scale for the missing one (no effect: its codes are masked)
    const float before = __shfl_up_sync(0xffffffffu, vs[NP - 1], 1);
#pragma unroll
    for (int p = 0; p < NP; ++p) {
      out.y[lane * NP + p] = y[p];
      out.ks[lane * NP + p] = ks[p];
      out.vs[lane * NP + p] = tok < it.t1 ? vs[p] : before;
    }
    if (lane == 0) out.it = it;
  }
};

__device__ __forceinline__ void cluster_sync() {
  asm volatile("barrier.cluster.arrive.release.aligned;\n\tbarrier.cluster.wait.acquire.aligned;" ::: "memory");
}
__device__ __forceinline__ uint32_t cluster_addr(const void* p, int rank) {
  uint32_t r;
  asm("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(r) : "r"(smem_u32(p)), "r"(rank));
  return r;
}
__device__ __forceinline__ float cluster_load(uint32_t addr) {
  float v;
  asm volatile("ld.shared::cluster.f32 %0, [%1];" : "=f"(v) : "r"(addr) : "memory");
  return v;
}

constexpr int kMaxCluster = 8;  // the portable size
constexpr int kReduceWarps = 4;

// Joins the chunks of a row that a cluster holds: o[head][D] and lse[head] of every
// CTA, in shared memory.  Every thread of the cluster comes here; the outputs
// are dealt to all of them.  The sums go in the order of fp8_decode_reduce_kernel,
// so that a row's result is the same in a call of either kind.
template <typename T, int D>
__device__ __forceinline__ void cluster_join(const Args& a, const float* o, const float2* lse) {
  __syncwarp();
  cluster_sync();
  const int c = blockIdx.x / a.cluster, rank = blockIdx.x - c * a.cluster;
  const int per_row = a.hkv * a.head_tiles, b = c / per_row, r = c - b * per_row;
  const int h = r / a.head_tiles, ht = r - h * a.head_tiles;
  const int hq0 = h * a.g + ht * a.tile_heads, heads = min(a.tile_heads, a.g - ht * a.tile_heads);
  const int64_t len = min((int64_t)a.seq_lens[b], a.bt_width * a.bs);
  const int nch = (int)((max(len, (int64_t)0) + kChunk - 1) / kChunk);
  if (nch > 1 && nch <= a.cluster) {
    for (int e = rank * kThreadsTC + (int)threadIdx.x; e < heads * D; e += a.cluster * kThreadsTC) {
      const int g = e / D, d = e - g * D;
      if (d >= a.d) continue;
      float l[kMaxCluster], x[kMaxCluster], M = -INFINITY, den = 0.f;
      float num[kReduceWarps] = {};
#pragma unroll
      for (int i = 0; i < kMaxCluster; ++i) {
        l[i] = -INFINITY, x[i] = 0.f;
        if (i < nch) l[i] = cluster_load(cluster_addr(&lse[g].x, i)), x[i] = cluster_load(cluster_addr(o + e, i));
      }
#pragma unroll
      for (int i = 0; i < kMaxCluster; ++i) M = fmaxf(M, l[i]);
#pragma unroll
      for (int i = 0; i < kMaxCluster; ++i) {
        const float w = l[i] == -INFINITY ? 0.f : (l[i] == M ? 1.f : fast_exp2(l[i] - M));
        num[i % kReduceWarps] += w * x[i], den += w;
      }
      static_assert(kReduceWarps == 4, "the order of the sums");
      const float all = (num[0] + num[1]) + (num[2] + num[3]);
      reinterpret_cast<T*>(a.out)[(int64_t)b * a.o_sb + (int64_t)(hq0 + g) * a.o_sh + d] =
          from_f32<T>(den == 0.f ? 0.f : all / den);
    }
  }
  cluster_sync();  // no CTA leaves while another reads its sums
}

// ROWS: a call whose clusters are rows (a.cluster > 0); at most one CTA per SM then.
template <typename T, int D, int NP, bool ROWS>
__global__ void __launch_bounds__(kThreadsTC, D == 128 && !ROWS ? 3 : 1)
    fp8_decode_tc_kernel(const Args a, const __grid_constant__ CUtensorMap kmap, const __grid_constant__ CUtensorMap vmap) {
  using C = Cfg<D>;
  using Shared = TCShared<D, NP>;
  using Slot = ItemSlot<D, NP>;
  static_assert(sizeof(Shared) % 16 == 0 && C::kDepth * C::kSlot % 1024 == 0 && C::kKS * 4 * sizeof(uint2) % 16 == 0 &&
                    sizeof(Slot) % 16 == 0 && offsetof(Slot, ks) % 16 == 0 && offsetof(Slot, vs) % 16 == 0,
                "vector accesses to shared memory");
  extern __shared__ __align__(1024) unsigned char smem_raw[];
  unsigned char* slots = smem_raw + ((1024u - (smem_u32(smem_raw) & 1023u)) & 1023u);
  Shared* sh = reinterpret_cast<Shared*>(slots + kNW * C::kDepth * C::kSlot);
  const int room = 4 * min(a.g, 8);                              // lanes of the heads an item can have
  uint2* qs = reinterpret_cast<uint2*>(sh + 1);                  // [2][kKS][room] fragments
  float* comb = reinterpret_cast<float*>(qs + 2 * C::kKS * room);  // [kNW - 1][kVecs][8 * head pairs] float4

  const int warp = threadIdx.x >> 5;
  const int lane = threadIdx.x & 31;
  if (threadIdx.x == 0) {
    for (int s = 0; s < kNW * C::kDepth; ++s) mbar_init(&sh->full[0][0] + s, 1);
    for (int s = 0; s < 2; ++s) {
      mbar_init(&sh->item_full[s], 1);
      mbar_init(&sh->item_empty[s], kNW);
    }
    mbar_init(&sh->comb_full, kNW - 1);
    mbar_init(&sh->comb_free, 1);
    sh->abort = 0;
    fence_mbar_init();
  }
  __syncthreads();

  pdl_wait();     // the plan (and all work before it) is complete and visible

  if (warp == kNW) {
    // ------------------------------ planner ------------------------------
    // Describes item by item to the consumers, one item ahead of them.  After its
    // first item a CTA claims the next one that nobody has: the plan lists the
    // chunks by decreasing size, so the CTAs finish together.  (A claim is made
    // when the consumers begin the item before it, late enough to be fair and a
    // whole item's time ahead of its use.)
    unsigned long long* claimed = reinterpret_cast<unsigned long long*>(a.hdr + 4);
    Pending<T, D, NP> p;
    int64_t item = blockIdx.x, items = 0;
    Unit first = {};
    if (a.planned) {
      first = load_unit(a, item);  // (the grid is no larger than the plan has room for)
      items = (int64_t)plan_units(a, lane == 0) * a.hkv * a.head_tiles;
    }
    for (int n_item = 0;; ++n_item) {
      const int k = n_item & 1;
      if (!__all_sync(0xffffffffu, wait_or_abort(&sh->item_empty[k], ((n_item >> 1) & 1) ^ 1, &sh->abort, a.err))) break;
      Unit unit = {};
      bool end;
      if (a.planned) {
        if (n_item > 0) {
          unsigned long long c = 0;
          if (lane == 0) c = atomicAdd(claimed, 1ull);
          item = (int64_t)__shfl_sync(0xffffffffu, c, 0) + gridDim.x;
          if (item < 0 && lane == 0) raise_dev(a.err, BL_DEVERR_WORKSPACE);  // (no plan's counter)
        }
        end = item < 0 || item >= items;
        if (!end) unit = n_item > 0 ? load_unit(a, item) : first;
      } else {
        end = n_item > 0;
        if (!end && ROWS) {
          unit = cluster_unit(a, lane == 0);
          item = blockIdx.x / a.cluster;
          end = unit.chunk * kChunk >= unit.len;
        } else if (!end) {
          const int per_unit = a.hkv * a.head_tiles;
          int units;
          unit = find_unit(a, (int)(item / per_unit), lane, units);
          end = item >= (int64_t)units * per_unit;
          if (units > a.max_units && blockIdx.x == 0 && lane == 0) raise_dev(a.err, BL_DEVERR_WORKSPACE);
        }
      }
      if (end) {
        pdl_trigger();  // the join kernel's launch may overlap this grid's end, for which it waits
        if (lane == 0) sh->items[k].it.heads = -1;
      } else {
        p.begin(a, item, unit, lane);
        p.finish(a);
        if (!p.valid && lane == 0) raise_dev(a.err, BL_DEVERR_WORKSPACE);
        p.stage(a, lane, sh->items[k], qs + k * C::kKS * room);
      }
      __syncwarp();
      if (lane == 0) mbar_arrive(&sh->item_full[k]);
      if (end) break;
    }
    // The last CTA to make its last claim leaves the counters as the plan did, for
    // the next layer's call with the same plan.
    if (a.planned && lane == 0 && atomicAdd(a.hdr + 6, 1) == (int)gridDim.x - 1) {
      a.hdr[6] = 0;
      *claimed = 0;
    }
    if constexpr (ROWS) cluster_join<T, D>(a, comb, sh->ml[kNW - 1]);
    return;
  }

  // ------------------------------ consumers ------------------------------
  if (lane == 0) {
    prefetch_tensormap(&kmap);
    prefetch_tensormap(&vmap);
  }
  zero_empty_rows<T>(a, kNW * 32);
  constexpr int kKS = C::kKS, kLaneDims = C::kLaneDims, kWords = C::kWords, kDepth = C::kDepth;
  const int g_row = lane >> 2;  // mma group: token (scores), query head (q, P), dim block (output)
  const int t4 = lane & 3;
  unsigned char* ring = slots + warp * kDepth * C::kSlot;
  const int k_row = (lane & 7) + (lane & 8);  // this lane's ldmatrix row of a K tile
  const uint32_t v_off = (uint32_t)((g_row * kLaneDims) & 15);
  // merge buffer: the lanes that hold heads, (head pairs) x 8 of them, side by side
  const int pairs = (min(a.g, 8) + 1) / 2;
  float4* const mine = reinterpret_cast<float4*>(comb) + g_row * pairs + t4;
  const int comb_vec = 8 * pairs;  // float4s between a lane's own
  const uint64_t policy = policy_evict_first();

  // A warp issues its own copies into a ring of its own: kDepth steps of 32
  // tokens.  One producer warp for the CTA had to pass every step through two
  // barriers and could not keep HBM busy (measured: its loop took ~850 cycles a
  // step, 2.7 TB/s from one CTA per SM whatever the ring's size).  The issue
  // cursor (item, step) runs ahead of the steps consumed, into the next item
  // once the planner has described it.
  int issued = 0, taken = 0;       // steps
  int at_item = -1, at_step = 0, at_steps = 0;
  int at_tiles = 0;
  bool at_end = false;
  // Issues the next step if there is one; `may_wait` false: only if its item is
  // described already.  n_item: the item being consumed; the cursor goes at most
  // one item further, since the planner describes that one only after this warp
  // has taken its steps of the item before n_item.
  auto issue = [&](int n_item, bool may_wait) -> bool {
    while (at_step >= at_steps) {
      const int next = at_item + 1;
      if (at_end || next > n_item + 1) return false;
      const int k = next & 1;
      if (!may_wait) {
        if (!__all_sync(0xffffffffu, mbar_try_wait(&sh->item_full[k], (next >> 1) & 1))) return false;
      } else if (!__all_sync(0xffffffffu, wait_or_abort(&sh->item_full[k], (next >> 1) & 1, &sh->abort, a.err))) {
        return false;
      }
      const Item& it = sh->items[k].it;
      if (it.heads < 0) {
        at_end = true;
        return false;
      }
      at_item = next;
      at_tiles = (it.t1 - it.t0 + 15) / 16;
      at_steps = (at_tiles + 1) / 2;
      at_step = (warp + next) & (kNW - 1);
    }
    const int slot = issued % kDepth;
    if (lane == 0) {
      const ItemSlot<D, NP>& is = sh->items[at_item & 1];
      const int n = min(2, at_tiles - 2 * at_step);
      uint64_t* bar = &sh->full[warp][slot];
      fence_proxy_async_smem();  // the warp's reads of the slot come before the copies into it
      mbar_arrive_expect_tx(bar, n * 2 * C::kTile);
      unsigned char* kd = ring + slot * C::kSlot;
      unsigned char* vd = kd + 2 * C::kTile;
#pragma unroll
      for (int x = 0; x < 2; ++x) {
        if (x < n) {
#pragma unroll
          for (int p = 0; p < NP; ++p) {
            const int32_t y = is.y[(2 * at_step + x) * NP + p];
            const int to = x * C::kTile + p * (C::kBox / NP);
#pragma unroll
            for (int hf = 0; hf < C::kHalves; ++hf) {
              tma_load_2d_hint(kd + to + hf * C::kBox, &kmap, bar, hf * 128, y, policy);
              tma_load_2d_hint(vd + to + hf * C::kBox, &vmap, bar, hf * 128, y, policy);
            }
          }
        }
      }
    }
    __syncwarp();
    at_step += kNW;
    ++issued;
    return true;
  };
  bool ok = true;

  for (int n_item = 0; ok; ++n_item) {
    // all waits are per warp and bounded; a CTA that gave up leaves them at once
    const int slot_i = n_item & 1;
    ok = __all_sync(0xffffffffu, wait_or_abort(&sh->item_full[slot_i], (n_item >> 1) & 1, &sh->abort, a.err));
    if (!ok) break;
    const Item it = sh->items[slot_i].it;
    if (it.heads < 0) break;  // no more items
    const float2 fs = sh->items[slot_i].f[t4];
    uint2 qf[kKS];
#pragma unroll
    for (int ks = 0; ks < kKS; ++ks)
      qf[ks] = g_row < it.heads ? qs[(slot_i * kKS + ks) * room + lane] : make_uint2(0u, 0u);
    const float f0 = fs.x, f1 = fs.y;
    const int nsteps = (it.t1 - it.t0 + kStepTokens - 1) / kStepTokens;

    // Running softmax state of this warp, per query head (column).  m follows
    // the maximum lazily: it moves only when a score passes it by 8 (log2
    // units), so P stays <= 2^8 and most steps need no cross-lane maximum.  The
    // output sums are kept in units of vref, the V scale of the tile that last
    // set it; a tile whose scale is close enough folds the (power of two) ratio
    // into its P.
    float m0 = -INFINITY, m1 = -INFINITY, l0 = 0.f, l1 = 0.f, vref = 0.f, vinv = 0.f;
    float o[C::kHalves][2 * kWords][4];
#pragma unroll
    for (int hf = 0; hf < C::kHalves; ++hf)
#pragma unroll
      for (int j = 0; j < 2 * kWords; ++j) o[hf][j][0] = o[hf][j][1] = o[hf][j][2] = o[hf][j][3] = 0.f;

    // The item's steps are dealt to the warps by class (step mod kNW); which warp
    // has which class turns from item to item, so that the warp of class 0, which
    // joins the others' sums below, is not always the same.  A class's sums do not
    // depend on its warp, so a row's result does not depend on what ran before it.
    const int cls = (warp + n_item) & (kNW - 1);
    for (int i = cls; i < nsteps; i += kNW) {
      // The slots freed by earlier steps are filled here, so that copies are in
      // flight for one step beyond this one.  (More does not help: HBM gives these
      // scattered 2 KB pages at its best rate with about 96 KB in flight per SM.)
      while (issued - taken < kDepth && issue(n_item, issued == taken)) {
      }
      const int slot = taken % kDepth;
      ok = issued > taken && __all_sync(0xffffffffu, wait_or_abort(&sh->full[warp][slot], (taken / kDepth) & 1, &sh->abort,
                                                                   a.err));
      if (!ok) break;
      float ksc[2 * NP], vsc[2 * NP];  // scales of the step's pieces
      if constexpr (NP == 1) {
        const float2 ks2 = *reinterpret_cast<const float2*>(&sh->items[slot_i].ks[2 * i]);
        const float2 vs2 = *reinterpret_cast<const float2*>(&sh->items[slot_i].vs[2 * i]);
        ksc[0] = ks2.x, ksc[1] = ks2.y, vsc[0] = vs2.x, vsc[1] = vs2.y;
      } else {
        const float4 ks4 = *reinterpret_cast<const float4*>(&sh->items[slot_i].ks[4 * i]);
        const float4 vs4 = *reinterpret_cast<const float4*>(&sh->items[slot_i].vs[4 * i]);
        ksc[0] = ks4.x, ksc[1] = ks4.y, ksc[2] = ks4.z, ksc[3] = ks4.w;
        vsc[0] = vs4.x, vsc[1] = vs4.y, vsc[2] = vs4.z, vsc[3] = vs4.w;
      }
      const uint32_t kb = smem_u32(ring + slot * C::kSlot);
      const unsigned char* vb = ring + slot * C::kSlot + 2 * C::kTile + v_off;

      // S^T[token][head] = K[token] . q[head], codes times normalised q.  Two chains of
      // sums per tile, joined at the end: the products of a chain wait for one another.
      float s[2][4];
      {
        float z[2][2][4];
#pragma unroll
        for (int x = 0; x < 2; ++x)
#pragma unroll
          for (int e = 0; e < 4; ++e) z[x][0][e] = z[x][1][e] = 0.f;
#pragma unroll
        for (int hf = 0; hf < C::kHalves; ++hf) {
          uint32_t r[2][C::kRow / 32][4];
#pragma unroll
          for (int c = 0; c < C::kRow / 32; ++c)
#pragma unroll
            for (int x = 0; x < 2; ++x)
              ldmatrix_x4(kb + x * C::kTile + hf * C::kBox + swizzled<C::kRow>(k_row, 2 * c + (lane >> 4)), r[x][c][0],
                          r[x][c][1], r[x][c][2], r[x][c][3]);
#pragma unroll
          for (int c = 0; c < C::kRow / 32; ++c)
#pragma unroll
            for (int x = 0; x < 2; ++x) {
              const int ks = hf * (C::kRow / 16) + 2 * c;
              mma_f16(z[x][0], e4m3lo_to_f16x2(r[x][c][0]), e4m3lo_to_f16x2(r[x][c][1]), e4m3hi_to_f16x2(r[x][c][0]),
                      e4m3hi_to_f16x2(r[x][c][1]), qf[ks].x, qf[ks].y);
              mma_f16(z[x][1], e4m3lo_to_f16x2(r[x][c][2]), e4m3lo_to_f16x2(r[x][c][3]), e4m3hi_to_f16x2(r[x][c][2]),
                      e4m3hi_to_f16x2(r[x][c][3]), qf[ks + 1].x, qf[ks + 1].y);
            }
        }
#pragma unroll
        for (int x = 0; x < 2; ++x)
#pragma unroll
          for (int e = 0; e < 4; ++e) s[x][e] = z[x][0][e] + z[x][1][e];
      }
      const int nvalid = it.t1 - (it.t0 + i * kStepTokens);  // tokens of the step that exist
      float c0[2 * NP], c1[2 * NP];  // factors of heads 2t, 2t + 1 for each piece's scores, log2 units
#pragma unroll
      for (int p = 0; p < 2 * NP; ++p) c0[p] = f0 * ksc[p], c1[p] = f1 * ksc[p];
      if (nvalid < kStepTokens) {
#pragma unroll
        for (int x = 0; x < 2; ++x) {
          if (16 * x + g_row >= nvalid) s[x][0] = s[x][1] = -INFINITY;
          if (16 * x + g_row + 8 >= nvalid) s[x][2] = s[x][3] = -INFINITY;
        }
        // (a factor that underflowed would make NaN of the mask)
#pragma unroll
        for (int p = 0; p < 2 * NP; ++p) c0[p] = fmaxf(c0[p], 1.2e-38f), c1[p] = fmaxf(c1[p], 1.2e-38f);
      }
      float mx0, mx1;
      if constexpr (NP == 1) {
        mx0 = fmaxf(fmaxf(s[0][0], s[0][2]) * c0[0], fmaxf(s[1][0], s[1][2]) * c0[1]);
        mx1 = fmaxf(fmaxf(s[0][1], s[0][3]) * c1[0], fmaxf(s[1][1], s[1][3]) * c1[1]);
      } else {
        mx0 = fmaxf(fmaxf(s[0][0] * c0[0], s[0][2] * c0[1]), fmaxf(s[1][0] * c0[2], s[1][2] * c0[3]));
        mx1 = fmaxf(fmaxf(s[0][1] * c1[0], s[0][3] * c1[1]), fmaxf(s[1][1] * c1[2], s[1][3] * c1[3]));
      }
      if (__any_sync(0xffffffffu, mx0 > m0 + 8.f || mx1 > m1 + 8.f)) {
#pragma unroll
        for (int off = 4; off < 32; off <<= 1) {
          mx0 = fmaxf(mx0, __shfl_xor_sync(0xffffffffu, mx0, off));
          mx1 = fmaxf(mx1, __shfl_xor_sync(0xffffffffu, mx1, off));
        }
        const float n0 = fmaxf(m0, mx0), n1 = fmaxf(m1, mx1);
        // (-inf) - (-inf) is NaN: a head whose scores are all -inf so far keeps its (zero) sums
        const float al0 = n0 == m0 ? 1.f : fast_exp2(m0 - n0), al1 = n1 == m1 ? 1.f : fast_exp2(m1 - n1);
        m0 = n0, m1 = n1;
        if (i != cls) {  // (on a warp's first step there are no sums yet)
          l0 *= al0, l1 *= al1;
#pragma unroll
          for (int hf = 0; hf < C::kHalves; ++hf)
#pragma unroll
            for (int j = 0; j < 2 * kWords; ++j) {
              o[hf][j][0] *= al0, o[hf][j][2] *= al0;
              o[hf][j][1] *= al1, o[hf][j][3] *= al1;
            }
        }
      }
      const float u0 = m0 == -INFINITY ? 0.f : -m0, u1 = m1 == -INFINITY ? 0.f : -m1;
      // exponentials and row sums
#pragma unroll
      for (int x = 0; x < 2; ++x) {
        const int a0 = x * NP, a1 = x * NP + NP - 1;  // pieces of the lane's two tokens
        s[x][0] = fast_exp2(fmaf(s[x][0], c0[a0], u0)), s[x][2] = fast_exp2(fmaf(s[x][2], c0[a1], u0));
        s[x][1] = fast_exp2(fmaf(s[x][1], c1[a0], u1)), s[x][3] = fast_exp2(fmaf(s[x][3], c1[a1], u1));
      }
      l0 += (s[0][0] + s[0][2]) + (s[1][0] + s[1][2]);
      l1 += (s[0][1] + s[0][3]) + (s[1][1] + s[1][3]);

      // O^T[dim][head] += V^T[dim][token] P^T[token][head] of tile x.  A lane takes the
      // kLaneDims consecutive dims g_row * kLaneDims of tokens 2t, 2t+1, 2t+8, 2t+9 and
      // pairs two tokens' bytes, so a converted pair is one A register (row =
      // dim, two consecutive tokens).  ONLY: -1, or the half of the tile whose tokens
      // are taken.  APART: the sums are made on their own and added times `ratio`.
      auto pv = [&](int x, float ratio, auto apart, auto only) {
        constexpr bool kApart = decltype(apart)::value;
        constexpr int kOnly = decltype(only)::value;
        // P^T (tokens x heads) -> B fragment (k = token, n = head)
        const uint32_t pb0 = kOnly == 1 ? 0u : movmatrix_trans(pack2<__half>(s[x][0], s[x][1]));
        const uint32_t pb1 = kOnly == 0 ? 0u : movmatrix_trans(pack2<__half>(s[x][2], s[x][3]));
        const int left = nvalid - 16 * x;
#pragma unroll
        for (int hf = 0; hf < C::kHalves; ++hf) {
          uint32_t v[4][kWords];
#pragma unroll
          for (int k = 0; k < 4; ++k) {
            const unsigned char* p = vb + x * C::kTile + hf * C::kBox +
                                     swizzled<C::kRow>(2 * t4 + (k & 1) + 8 * (k >> 1), (g_row * kLaneDims) >> 4);
            if constexpr (kWords == 4) {
              const uint4 u = *reinterpret_cast<const uint4*>(p);
              v[k][0] = u.x, v[k][1] = u.y, v[k][2] = u.z, v[k][3] = u.w;
            } else {
              const uint2 u = *reinterpret_cast<const uint2*>(p);
              v[k][0] = u.x, v[k][1] = u.y;
            }
          }
          if (left < 16) {
            // slots past the length hold stale codes (possibly NaN): 0 * NaN is NaN
#pragma unroll
            for (int k = 0; k < 4; ++k)
#pragma unroll
              for (int j = 0; j < kWords; ++j) v[k][j] = 2 * t4 + (k & 1) + 8 * (k >> 1) < left ? v[k][j] : 0u;
          }
#pragma unroll
          for (int j = 0; j < kWords; ++j) {
            const uint32_t lo01 = __byte_perm(v[0][j], v[1][j], 0x5140), lo23 = __byte_perm(v[0][j], v[1][j], 0x7362);
            const uint32_t hi01 = __byte_perm(v[2][j], v[3][j], 0x5140), hi23 = __byte_perm(v[2][j], v[3][j], 0x7362);
            float(&d0)[4] = o[hf][2 * j];
            float(&d1)[4] = o[hf][2 * j + 1];
            if constexpr (!kApart) {
              mma_f16(d0, e4m3lo_to_f16x2(lo01), e4m3hi_to_f16x2(lo01), e4m3lo_to_f16x2(hi01), e4m3hi_to_f16x2(hi01), pb0,
                      pb1);
              mma_f16(d1, e4m3lo_to_f16x2(lo23), e4m3hi_to_f16x2(lo23), e4m3lo_to_f16x2(hi23), e4m3hi_to_f16x2(hi23), pb0,
                      pb1);
            } else {
              float z0[4] = {0.f, 0.f, 0.f, 0.f}, z1[4] = {0.f, 0.f, 0.f, 0.f};
              mma_f16(z0, e4m3lo_to_f16x2(lo01), e4m3hi_to_f16x2(lo01), e4m3lo_to_f16x2(hi01), e4m3hi_to_f16x2(hi01), pb0,
                      pb1);
              mma_f16(z1, e4m3lo_to_f16x2(lo23), e4m3hi_to_f16x2(lo23), e4m3lo_to_f16x2(hi23), e4m3hi_to_f16x2(hi23), pb0,
                      pb1);
#pragma unroll
              for (int e = 0; e < 4; ++e) d0[e] += ratio * z0[e], d1[e] += ratio * z1[e];
            }
          }
        }
      };
      // A much larger V scale becomes the reference (the sums shrink by a power
      // of two); a much smaller one is added apart.
      float vmax = fmaxf(vsc[0], vsc[1]);
      if constexpr (NP == 2) vmax = fmaxf(vmax, fmaxf(vsc[2], vsc[3]));
      if (vmax > vref * 16.f) {
        const float r = vref * pow2_inverse(vmax);
        vref = vmax;
        vinv = pow2_inverse(vmax);
        if (i != cls) {
#pragma unroll
          for (int hf = 0; hf < C::kHalves; ++hf)
#pragma unroll
            for (int j = 0; j < 2 * kWords; ++j)
#pragma unroll
              for (int e = 0; e < 4; ++e) o[hf][j][e] *= r;
        }
      }
      float r[2 * NP], rmin = INFINITY, rmax = 0.f;
#pragma unroll
      for (int p = 0; p < 2 * NP; ++p) r[p] = vsc[p] * vinv, rmin = fminf(rmin, r[p]), rmax = fmaxf(rmax, r[p]);
      using Both = std::integral_constant<int, -1>;
      if (rmin >= 0.015625f) {
        if (rmin != 1.f || rmax != 1.f) {
#pragma unroll
          for (int x = 0; x < 2; ++x)
#pragma unroll
            for (int e = 0; e < 4; ++e) s[x][e] *= r[x * NP + (e >> 1) * (NP - 1)];
        }
        pv(0, 1.f, std::false_type(), Both());
        pv(1, 1.f, std::false_type(), Both());
      } else if constexpr (NP == 1) {
        pv(0, r[0], std::true_type(), Both());
        pv(1, r[1], std::true_type(), Both());
      } else {
#pragma unroll
        for (int x = 0; x < 2; ++x) {
          pv(x, r[2 * x], std::true_type(), std::integral_constant<int, 0>());
          pv(x, r[2 * x + 1], std::true_type(), std::integral_constant<int, 1>());
        }
      }
      ++taken;
      __syncwarp();
    }
    __syncwarp();
    if (!ok) break;
    // The slot's description is gone once every warp has arrived here: a cursor
    // that has not passed this item (it has no step for this warp) passes it now.
    if (at_item < n_item) {
      at_item = n_item;
      at_step = at_steps = 0;
    }
    if (lane == 0) mbar_arrive(&sh->item_empty[slot_i]);

    // ---- merge the warps: the one with class 0 joins the others' sums to its own ----
#pragma unroll
    for (int off = 4; off < 32; off <<= 1) {
      l0 += __shfl_xor_sync(0xffffffffu, l0, off);
      l1 += __shfl_xor_sync(0xffffffffu, l1, off);
    }
    const int h0 = 2 * t4, h1 = 2 * t4 + 1;
    const bool holds = h0 < it.heads;
    const unsigned holders = ROWS ? __ballot_sync(0xffffffffu, holds) : 0u;
    // the previous item's sums have been read (every warp waits here, so no phase is skipped)
    ok = __all_sync(0xffffffffu, wait_or_abort(&sh->comb_free, (n_item & 1) ^ 1, &sh->abort, a.err));
    if (!ok) break;
    if (cls != 0) {
      const int w = cls - 1;
      if (g_row == 0) {
        sh->ml[w][h0] = make_float2(m0, l0);
        sh->ml[w][h1] = make_float2(m1, l1);
      }
      if (holds) {
        float4* dst = mine + w * C::kVecs * comb_vec;
#pragma unroll
        for (int hf = 0; hf < C::kHalves; ++hf)
#pragma unroll
          for (int j = 0; j < 2 * kWords; ++j) {
            const float(&x)[4] = o[hf][j];
            dst[(hf * 2 * kWords + j) * comb_vec] = make_float4(x[0] * vref, x[1] * vref, x[2] * vref, x[3] * vref);
          }
      }
      __syncwarp();
      if (lane == 0) mbar_arrive(&sh->comb_full);
      continue;
    }
    ok = __all_sync(0xffffffffu, wait_or_abort(&sh->comb_full, n_item & 1, &sh->abort, a.err));
    if (!ok) break;
    if (holds) {
      float M0 = m0, M1 = m1;
      float2 ml0[kNW - 1], ml1[kNW - 1];
#pragma unroll
      for (int w = 0; w < kNW - 1; ++w) {
        ml0[w] = sh->ml[w][h0], ml1[w] = sh->ml[w][h1];
        M0 = fmaxf(M0, ml0[w].x), M1 = fmaxf(M1, ml1[w].x);
      }
      auto weight = [](float m, float M) { return m == -INFINITY ? 0.f : (m == M ? 1.f : fast_exp2(m - M)); };
      const float s0 = weight(m0, M0), s1 = weight(m1, M1);
      float L0 = s0 * l0, L1 = s1 * l1;
      const float r0 = s0 * vref, r1 = s1 * vref;
#pragma unroll
      for (int hf = 0; hf < C::kHalves; ++hf)
#pragma unroll
        for (int j = 0; j < 2 * kWords; ++j) {
          float(&x)[4] = o[hf][j];
          x[0] *= r0, x[2] *= r0, x[1] *= r1, x[3] *= r1;
        }
#pragma unroll
      for (int w = 0; w < kNW - 1; ++w) {
        const float w0 = weight(ml0[w].x, M0), w1 = weight(ml1[w].x, M1);
        L0 += w0 * ml0[w].y, L1 += w1 * ml1[w].y;
        const float4* src = mine + w * C::kVecs * comb_vec;
#pragma unroll
        for (int hf = 0; hf < C::kHalves; ++hf)
#pragma unroll
          for (int j = 0; j < 2 * kWords; ++j) {
            const float4 y = src[(hf * 2 * kWords + j) * comb_vec];
            float(&x)[4] = o[hf][j];
            x[0] += w0 * y.x, x[1] += w1 * y.y, x[2] += w0 * y.z, x[3] += w1 * y.w;
          }
      }
      // (in a cluster the joined sums go where the other warps' were: every lane has read its own)
      if (ROWS) __syncwarp(holders);
      // sum 0: no token (nothing seen); a NaN sum stays NaN
      const float i0 = L0 == 0.f ? 0.f : 1.f / L0, i1 = L1 == 0.f ? 0.f : 1.f / L1;
      const bool parts = it.nch > 1;
      if (parts && !ROWS && !has_part(a, it)) {
        raise_dev(a.err, BL_DEVERR_WORKSPACE);
      } else {
#pragma unroll
        for (int c = 0; c < 2; ++c) {
          if (c == 1 && h1 >= it.heads) break;
          const int hq = it.hq0 + (c ? h1 : h0);
          const float inv = c ? i1 : i0;
          T* dst = reinterpret_cast<T*>(a.out) + (int64_t)it.b * a.o_sb + (int64_t)hq * a.o_sh;
          float* part = ROWS ? comb + (c ? h1 : h0) * D : a.ws_o + ((int64_t)it.part * a.hq + hq) * a.d;
          float* lse = ROWS ? &sh->ml[kNW - 1][c ? h1 : h0].x : a.ws_lse + (int64_t)it.part * a.hq + hq;
          if (parts && g_row == 0)
            *lse = c ? (L1 == 0.f ? -INFINITY : M1 + __log2f(L1))
                     : (L0 == 0.f ? -INFINITY : M0 + __log2f(L0));
#pragma unroll
          for (int hf = 0; hf < C::kHalves; ++hf)
#pragma unroll
            for (int j = 0; j < 2 * kWords; j += 2) {
              const int d = hf * 128 + g_row * kLaneDims + 2 * j;
              if (d >= a.d) break;
              const float v0 = o[hf][j][c] * inv, v1 = o[hf][j][2 + c] * inv;
              const float v2 = o[hf][j + 1][c] * inv, v3 = o[hf][j + 1][2 + c] * inv;
              if (parts) {
                *reinterpret_cast<float4*>(part + d) = make_float4(v0, v1, v2, v3);
              } else if (a.o_vec) {
                *reinterpret_cast<uint2*>(dst + d) = make_uint2(pack2<T>(v0, v1), pack2<T>(v2, v3));
              } else {
                dst[d] = from_f32<T>(v0), dst[d + 1] = from_f32<T>(v1);
                dst[d + 2] = from_f32<T>(v2), dst[d + 3] = from_f32<T>(v3);
              }
            }
        }
      }
    }
    __syncwarp();
    if (lane == 0) mbar_arrive(&sh->comb_free);
  }
  // Drain: every copy this warp issued lands before the CTA can exit (some are
  // left only where the CTA gave up).
  for (; taken < issued; ++taken)
    if (!mbar_wait(&sh->full[warp][taken % kDepth], (taken / kDepth) & 1)) raise_dev(a.err, BL_DEVERR_TIMEOUT);
  if constexpr (ROWS) cluster_join<T, D>(a, comb, sh->ml[kNW - 1]);
}

// ---------------------------------------------------------------------------
// SIMT kernel: any element type, head_dim <= 256, any block size
// ---------------------------------------------------------------------------
constexpr int kSimtThreads = 128;
constexpr int kSimtWarps = kSimtThreads / 32;
constexpr int kSimtTok = 4;    // tokens a lane group has in hand
// resident CTAs per SM that the registers of HG heads allow
__host__ __device__ constexpr int simt_ctas(int heads) { return heads == 4 ? 2 : heads == 2 ? 3 : 4; }
constexpr int kSimtHeads = 4;  // query heads of an item, at most

// the four codes of a word, times s
__device__ __forceinline__ void decode4(uint32_t w, uint64_t s, uint64_t (&x)[2]) {
  const float2 lo = unpack2<__half>(e4m3lo_to_f16x2(w)), hi = unpack2<__half>(e4m3hi_to_f16x2(w));
  x[0] = f2_mul(f2_pack(lo.x, lo.y), s);
  x[1] = f2_mul(f2_pack(hi.x, hi.y), s);
}

template <int HG>
struct alignas(16) SimtShared {
  float4 q[HG][4][16];          // dims 16 l + 4 c + {0..3} of a head at [c][l]: lanes side by side read side by side
  int64_t row[kChunk];          // byte offset of a token's codes, -1: none
  float ks[kChunk], vs[kChunk];
  float2 ml[kSimtWarps][HG];    // maximum and sum of each warp
  float o[kSimtWarps][HG][256];
};

// A group of lanes has a token, each lane 16 dims of it, straight from the pool:
// the codes never pass through shared memory.  HG heads' products with them in
// registers (q from shared memory, the sums of the output in registers), the
// lanes' shares of a score joined by shuffles; every group keeps a softmax of its
// own, and the groups and warps are joined once per chunk.  K codes of the next
// step are on their way during the V half of this one, V codes during the K half.
// What bounds it (64 requests of 1k..8k tokens, 32 / 8 heads of 128 dims, fp32 q,
// 617 MB): issue slots and latency, 352 us, 1.75 TB/s; 2 and 1 heads
// a KV head 2.3 and 3.9 TB/s.  (Through fp32 tiles in shared memory: 889 us.)
// WIDE: head_dim and the pool's rows in whole 16-byte units.
template <typename T, int HG, bool WIDE>
__global__ void __launch_bounds__(kSimtThreads, simt_ctas(HG)) fp8_decode_simt_kernel(const Args a) {
  __shared__ SimtShared<HG> sh;
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  int lpt = 1;  // lanes of a token
  while (16 * lpt < a.d) lpt *= 2;
  const int tpw = 32 / lpt;  // tokens a warp reads at once
  const int lt = lane & (lpt - 1), grp = lane / lpt, dim0 = 16 * lt;
  const bool has_dims = dim0 < a.d;

  pdl_wait();
  const int64_t items = (int64_t)plan_units(a, tid == 0) * a.hkv * a.head_tiles;
  zero_empty_rows<T>(a, kSimtThreads);

  auto load = [&](const uint8_t* pool, int at, uint4 (&w)[kSimtTok]) {
#pragma unroll
    for (int u = 0; u < kSimtTok; ++u) {
      const int t = at + (u * kSimtWarps + warp) * tpw + grp;
      const int64_t r = t < kChunk ? sh.row[t] : -1;
      w[u] = make_uint4(0u, 0u, 0u, 0u);
      if (r < 0 || !has_dims) continue;
      const uint8_t* p = pool + r + dim0;
      if constexpr (WIDE) {
        w[u] = *reinterpret_cast<const uint4*>(p);
      } else {
        uint32_t x[4] = {0u, 0u, 0u, 0u};
        const int n = min(16, a.d - dim0);
        if ((a.d & 3) == 0) {
#pragma unroll
          for (int c = 0; c < 4; ++c)
            if (4 * c < n) x[c] = *reinterpret_cast<const uint32_t*>(p + 4 * c);
        } else {
#pragma unroll
          for (int e = 0; e < 16; ++e)
            if (e < n) x[e >> 2] |= (uint32_t)p[e] << (8 * (e & 3));
        }
        w[u] = make_uint4(x[0], x[1], x[2], x[3]);
      }
    }
  };

  for (int64_t item = blockIdx.x; item < items; item += gridDim.x) {
    Item it;
    if (!make_item(a, item, load_unit(a, item), it)) {
      if (tid == 0) raise_dev(a.err, BL_DEVERR_WORKSPACE);
      continue;
    }
    __syncthreads();  // the previous item's shared state is no longer read
    const int n = it.t1 - it.t0;
    for (int i = tid; i < kChunk; i += kSimtThreads) {
      int64_t r = -1;
      float ks = 0.f, vs = 0.f;
      if (i < n) {
        const int t = it.t0 + i, lb = t / a.bs;
        const int64_t phys = a.block_tables[(int64_t)it.table_row * a.bt_stride + lb];
        if (phys < 0 || phys >= a.num_blocks) {
          raise_dev(a.err, BL_DEVERR_BLOCK_ID);
        } else {
          const int64_t slot = (a.layer * a.num_blocks + phys) * a.hkv + it.h;
          r = (slot * a.bs + (t - lb * a.bs)) * a.d;
          ks = a.k_scale[slot];
          vs = a.v_scale[slot];
        }
      }
      sh.row[i] = r;
      sh.ks[i] = ks;
      sh.vs[i] = vs;
    }
    for (int e = tid; e < HG * 256; e += kSimtThreads) {
      const int h = e >> 8, d = e & 255;
      float x = 0.f;
      if (h < it.heads && d < a.d)
        x = to_f32<T>(reinterpret_cast<const T*>(a.q)[(int64_t)it.b * a.q_sb + (int64_t)(it.hq0 + h) * a.q_sh + d]) *
            a.scale_log2;
      reinterpret_cast<float*>(&sh.q[h][(d >> 2) & 3][d >> 4])[d & 3] = x;
    }
    __syncthreads();

    float m[HG], l[HG];
    uint64_t o[HG][8];
#pragma unroll
    for (int h = 0; h < HG; ++h) {
      m[h] = -INFINITY;
      l[h] = 0.f;
#pragma unroll
      for (int j = 0; j < 8; ++j) o[h][j] = 0ull;
    }
    uint4 kc[kSimtTok], vc[kSimtTok];
    load(a.k_pool, 0, kc);
    load(a.v_pool, 0, vc);
    const int step = kSimtWarps * tpw * kSimtTok;
    for (int at = 0; at < n; at += step) {
      float s[kSimtTok][HG];
      float vs[kSimtTok];
      {
        uint64_t z[kSimtTok][HG], ks[kSimtTok];
#pragma unroll
        for (int u = 0; u < kSimtTok; ++u) {
          const int t = at + (u * kSimtWarps + warp) * tpw + grp;
          const float x = t < kChunk ? sh.ks[t] : 0.f;
          vs[u] = t < kChunk ? sh.vs[t] : 0.f;
          ks[u] = f2_pack(x, x);
#pragma unroll
          for (int h = 0; h < HG; ++h) z[u][h] = 0ull;
        }
#pragma unroll
        for (int c = 0; c < 4; ++c) {
          uint64_t q[HG][2];
#pragma unroll
          for (int h = 0; h < HG; ++h) {
            const ulonglong2 x = *reinterpret_cast<const ulonglong2*>(&sh.q[h][c][lt]);
            q[h][0] = x.x, q[h][1] = x.y;
          }
#pragma unroll
          for (int u = 0; u < kSimtTok; ++u) {
            uint64_t x[2];
            decode4(c == 0 ? kc[u].x : c == 1 ? kc[u].y : c == 2 ? kc[u].z : kc[u].w, ks[u], x);
#pragma unroll
            for (int h = 0; h < HG; ++h) z[u][h] = f2_fma(x[1], q[h][1], f2_fma(x[0], q[h][0], z[u][h]));
          }
        }
        load(a.k_pool, at + step, kc);
#pragma unroll
        for (int u = 0; u < kSimtTok; ++u)
#pragma unroll
          for (int h = 0; h < HG; ++h) {
            const float2 x = f2_unpack(z[u][h]);
            s[u][h] = x.x + x.y;
          }
      }
      for (int off = 1; off < lpt; off <<= 1)
#pragma unroll
        for (int u = 0; u < kSimtTok; ++u)
#pragma unroll
          for (int h = 0; h < HG; ++h) s[u][h] += __shfl_xor_sync(0xffffffffu, s[u][h], off);
      bool moved = false;
      float top[HG];
#pragma unroll
      for (int h = 0; h < HG; ++h) top[h] = m[h];
#pragma unroll
      for (int u = 0; u < kSimtTok; ++u) {
        const int t = at + (u * kSimtWarps + warp) * tpw + grp;
        const bool live = t < kChunk && sh.row[t] >= 0;
#pragma unroll
        for (int h = 0; h < HG; ++h) {
          if (!live) s[u][h] = -INFINITY;
          top[h] = fmaxf(top[h], s[u][h]);
        }
      }
      // the maximum moves only when a score passes it by 8 (log2 units): P <= 2^8
#pragma unroll
      for (int h = 0; h < HG; ++h) moved |= top[h] > m[h] + 8.f;
      if (__any_sync(0xffffffffu, moved)) {
#pragma unroll
        for (int h = 0; h < HG; ++h) {
          const float al = top[h] == m[h] ? 1.f : fast_exp2(m[h] - top[h]);
          m[h] = top[h];
          l[h] *= al;
          const uint64_t al2 = f2_pack(al, al);
#pragma unroll
          for (int j = 0; j < 8; ++j) o[h][j] = f2_mul(o[h][j], al2);
        }
      }
#pragma unroll
      for (int h = 0; h < HG; ++h) {
        const float unit = m[h] == -INFINITY ? 0.f : m[h];
#pragma unroll
        for (int u = 0; u < kSimtTok; ++u) {
          s[u][h] = fast_exp2(s[u][h] - unit);
          l[h] += s[u][h];
        }
      }
#pragma unroll
      for (int u = 0; u < kSimtTok; ++u) {
        const uint64_t v2 = f2_pack(vs[u], vs[u]);
        uint64_t p[HG];
#pragma unroll
        for (int h = 0; h < HG; ++h) p[h] = f2_pack(s[u][h], s[u][h]);
#pragma unroll
        for (int c = 0; c < 4; ++c) {
          uint64_t x[2];
          decode4(c == 0 ? vc[u].x : c == 1 ? vc[u].y : c == 2 ? vc[u].z : vc[u].w, v2, x);
#pragma unroll
          for (int h = 0; h < HG; ++h) {
            o[h][2 * c] = f2_fma(p[h], x[0], o[h][2 * c]);
            o[h][2 * c + 1] = f2_fma(p[h], x[1], o[h][2 * c + 1]);
          }
        }
      }
      load(a.v_pool, at + step, vc);
    }

    // ---- join the groups of the warp, then the warps ----
    auto weight = [](float x, float top) { return x == -INFINITY ? 0.f : (x == top ? 1.f : fast_exp2(x - top)); };
    for (int off = lpt; off < 32; off <<= 1) {
#pragma unroll
      for (int h = 0; h < HG; ++h) {
        const float om = __shfl_xor_sync(0xffffffffu, m[h], off), ol = __shfl_xor_sync(0xffffffffu, l[h], off);
        const float top = fmaxf(m[h], om);
        const float w = weight(m[h], top), ow = weight(om, top);
        m[h] = top;
        l[h] = w * l[h] + ow * ol;
#pragma unroll
        for (int j = 0; j < 8; ++j) {
          const uint64_t x = __shfl_xor_sync(0xffffffffu, o[h][j], off);
          o[h][j] = f2_fma(f2_pack(ow, ow), x, f2_mul(f2_pack(w, w), o[h][j]));
        }
      }
    }
    if (grp == 0) {
#pragma unroll
      for (int h = 0; h < HG; ++h) {
        if (lt == 0) sh.ml[warp][h] = make_float2(m[h], l[h]);
        if (has_dims)
#pragma unroll
          for (int j = 0; j < 8; j += 2)
            *reinterpret_cast<ulonglong2*>(&sh.o[warp][h][dim0 + 2 * j]) = make_ulonglong2(o[h][j], o[h][j + 1]);
      }
    }
    __syncthreads();
    const bool parts = it.nch > 1;
    if (parts && !has_part(a, it)) {
      if (tid == 0) raise_dev(a.err, BL_DEVERR_WORKSPACE);
      continue;
    }
    for (int h = 0; h < it.heads; ++h) {
      float top = -INFINITY, sum = 0.f, w[kSimtWarps];
#pragma unroll
      for (int i = 0; i < kSimtWarps; ++i) top = fmaxf(top, sh.ml[i][h].x);
#pragma unroll
      for (int i = 0; i < kSimtWarps; ++i) {
        w[i] = weight(sh.ml[i][h].x, top);
        sum += w[i] * sh.ml[i][h].y;
      }
      // sum 0: no token (nothing seen); a NaN sum stays NaN
      const int hq = it.hq0 + h;
      T* dst = reinterpret_cast<T*>(a.out) + (int64_t)it.b * a.o_sb + (int64_t)hq * a.o_sh;
      float* part = a.ws_o + ((int64_t)it.part * a.hq + hq) * a.d;
      if (parts && tid == 0) a.ws_lse[(int64_t)it.part * a.hq + hq] = sum == 0.f ? -INFINITY : top + __log2f(sum);
      for (int d = tid; d < a.d; d += kSimtThreads) {
        float x = 0.f;
#pragma unroll
        for (int i = 0; i < kSimtWarps; ++i) x += w[i] * sh.o[i][h][d];
        x = sum == 0.f ? 0.f : x / sum;
        if (parts)
          part[d] = x;
        else
          dst[d] = from_f32<T>(x);
      }
    }
  }
}

// ---------------------------------------------------------------------------
// reduce: rows of several chunks
// ---------------------------------------------------------------------------
constexpr int kReduceThreads = 32 * kReduceWarps;
constexpr int kReduceTile = 512;  // chunks whose weights are in shared memory at a time

// grid: (batch, hq).  Warp w sums every fourth chunk, a lane four consecutive
// dims at a time; the warps' sums are joined in shared memory.
template <typename T>
__global__ void __launch_bounds__(kReduceThreads) fp8_decode_reduce_kernel(const Args a) {
  pdl_wait();  // the partials are complete and visible
  constexpr int kWarps = kReduceThreads / 32;
  const int b = blockIdx.x, hq = blockIdx.y, tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  const int64_t len = min((int64_t)a.seq_lens[b], a.bt_width * a.bs);
  if (len <= kChunk) return;
  const int nch = (int)((len + kChunk - 1) / kChunk);
  int64_t base = 0;
  if (a.planned) {
    base = a.row_base[b];
  } else {
    for (int r = 0; r < b; ++r)
      base += (min(max((int64_t)a.seq_lens[r], (int64_t)0), a.bt_width * a.bs) + kChunk - 1) / kChunk;
  }
  if (base < 0 || base + nch > a.max_units) return;  // flagged by the plan or the attention kernel
  __shared__ float s_w[kReduceTile];
  __shared__ float s_red[kWarps];
  __shared__ float s_num[kWarps][256];
  float M = -INFINITY;
  for (int c = tid; c < nch; c += kReduceThreads) M = fmaxf(M, a.ws_lse[(base + c) * a.hq + hq]);
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) M = fmaxf(M, __shfl_xor_sync(0xffffffffu, M, o));
  if (lane == 0) s_red[warp] = M;
  __syncthreads();
#pragma unroll
  for (int w = 0; w < kWarps; ++w) M = fmaxf(M, s_red[w]);
  float num[2][4] = {}, den = 0.f;
  const int64_t cstride = (int64_t)a.hq * a.d;
  const bool vec = (a.d & 3) == 0;
  for (int c0 = 0; c0 < nch; c0 += kReduceTile) {
    const int n = min(kReduceTile, nch - c0);
    __syncthreads();
    for (int c = tid; c < n; c += kReduceThreads) {
      const float l = a.ws_lse[(base + c0 + c) * a.hq + hq];
      s_w[c] = l == -INFINITY ? 0.f : (l == M ? 1.f : fast_exp2(l - M));
    }
    __syncthreads();
    const float* po = a.ws_o + ((base + c0) * a.hq + hq) * a.d;
#pragma unroll
    for (int k = 0; k < 2; ++k) {
      const int d = 4 * lane + 128 * k;
      if (d >= a.d) break;
      if (vec) {
#pragma unroll 8
        for (int c = warp; c < n; c += kWarps) {
          const float4 x = *reinterpret_cast<const float4*>(po + c * cstride + d);
          const float f = s_w[c];
          num[k][0] += f * x.x, num[k][1] += f * x.y, num[k][2] += f * x.z, num[k][3] += f * x.w;
        }
      } else {
        for (int c = warp; c < n; c += kWarps)
#pragma unroll
          for (int e = 0; e < 4; ++e)
            if (d + e < a.d) num[k][e] += s_w[c] * po[c * cstride + d + e];
      }
    }
    for (int c = 0; c < n; ++c) den += s_w[c];
  }
#pragma unroll
  for (int k = 0; k < 2; ++k)
#pragma unroll
    for (int e = 0; e < 4; ++e) s_num[warp][4 * lane + 128 * k + e] = num[k][e];
  __syncthreads();
  T* dst = reinterpret_cast<T*>(a.out) + (int64_t)b * a.o_sb + (int64_t)hq * a.o_sh;
  for (int d = tid; d < a.d; d += kReduceThreads) {
    const float x = (s_num[0][d] + s_num[1][d]) + (s_num[2][d] + s_num[3][d]);
    dst[d] = from_f32<T>(den == 0.f ? 0.f : x / den);
  }
}

// ---------------------------------------------------------------------------
// host side
// ---------------------------------------------------------------------------
// The tensor-core kernel: 16-bit q, pool rows of whole 16-byte units (a tensor
// map's stride), whole 8-token pieces in a block, and pool rows within the
// tensor map's 32-bit coordinates.  Columns behind head_dim lie outside the map,
// so that the copies fill them with zeros; they cost products but no bytes.
bool use_tc(const bl_paged_layer& kv) {
  const double rows = (double)kv.num_layers * kv.num_blocks * kv.num_kv_heads * kv.block_size;
  return (kv.dtype == BL_BF16 || kv.dtype == BL_F16) && kv.head_dim % 16 == 0 && kv.head_dim <= 256 &&
         kv.block_size % 8 == 0 && rows <= (double)INT32_MAX;
}

template <typename T, int D, int NP, bool ROWS>
int launch_tc(const Args& k, const bl_paged_layer& kv, cudaStream_t s) {
  using C = Cfg<D>;
  CUtensorMap kmap, vmap;
  const uint64_t rows = (uint64_t)kv.num_layers * kv.num_blocks * kv.num_kv_heads * kv.block_size;
  const uint64_t row_bytes = (uint64_t)kv.head_dim;
  if (!make_tmap_rows_8bit(&kmap, kv.k_pool, row_bytes, rows, C::kRow, 16 / NP) ||
      !make_tmap_rows_8bit(&vmap, kv.v_pool, row_bytes, rows, C::kRow, 16 / NP))
    return BL_ERR_LAUNCH;
  const auto smem_for = [](int g) {
    const size_t heads = std::min(g, 8);
    return 1024 + (size_t)kNW * C::kDepth * C::kSlot + sizeof(TCShared<D, NP>) + 2 * C::kKS * 4 * heads * sizeof(uint2) +
           (size_t)(kNW - 1) * C::kVecs * 8 * ((heads + 1) / 2) * sizeof(float4);
  };
  const size_t smem = smem_for(k.g);
  const int64_t items = (int64_t)k.max_units * k.hkv * k.head_tiles;
  // resident CTAs per SM, asked once per device and head tile (the attribute is per device too)
  static std::mutex mu;
  static int occ_cache[64][9] = {};
  int dev = 0, occ = 0;
  cudaGetDevice(&dev);
  {
    std::lock_guard<std::mutex> lk(mu);
    int* slot = dev >= 0 && dev < 64 ? &occ_cache[dev][std::min(k.g, 8)] : &occ;
    if (*slot == 0) {
      int o = 0;
      if (cudaFuncSetAttribute(fp8_decode_tc_kernel<T, D, NP, ROWS>, cudaFuncAttributeMaxDynamicSharedMemorySize,
                               (int)smem_for(8)) != cudaSuccess ||
          cudaOccupancyMaxActiveBlocksPerMultiprocessor(&o, fp8_decode_tc_kernel<T, D, NP, ROWS>, kThreadsTC, smem) !=
              cudaSuccess) {
        set_error("fp8_decode_tc_kernel: %s", cudaGetErrorString(cudaGetLastError()));
        return BL_ERR_LAUNCH;
      }
      *slot = std::max(o, 1);
    }
    occ = *slot;
  }
  const int64_t grid = std::min<int64_t>((int64_t)num_sms() * occ, items);
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3((unsigned)(ROWS ? items : grid));
  cfg.blockDim = dim3(kThreadsTC);
  cfg.dynamicSmemBytes = smem;
  cfg.stream = s;
  cudaLaunchAttribute attr[2];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  attr[1].id = cudaLaunchAttributeClusterDimension;
  attr[1].val.clusterDim.x = (unsigned)k.cluster;
  attr[1].val.clusterDim.y = attr[1].val.clusterDim.z = 1;
  cfg.attrs = attr;
  cfg.numAttrs = ROWS ? 2 : 1;
  if (cudaLaunchKernelEx(&cfg, fp8_decode_tc_kernel<T, D, NP, ROWS>, k, kmap, vmap) != cudaSuccess) {
    set_error("fp8_decode_tc_kernel: launch failed: %s", cudaGetErrorString(cudaGetLastError()));
    return BL_ERR_LAUNCH;
  }
  return BL_OK;
}

template <typename T, int NP, bool ROWS>
int launch_tc_dims(const Args& k, const bl_paged_layer& kv, cudaStream_t s) {
  return k.d <= 64    ? launch_tc<T, 64, NP, ROWS>(k, kv, s)
         : k.d <= 128 ? launch_tc<T, 128, NP, ROWS>(k, kv, s)
                      : launch_tc<T, 256, NP, ROWS>(k, kv, s);
}

template <typename T, int HG>
int launch_simt_heads(const Args& k, cudaStream_t s) {
  const int64_t items = (int64_t)k.max_units * k.hkv * k.head_tiles;
  const int64_t grid = std::min<int64_t>((int64_t)num_sms() * simt_ctas(HG), items);
  const bool wide = k.d % 16 == 0;
  if (launch_pdl(wide ? fp8_decode_simt_kernel<T, HG, true> : fp8_decode_simt_kernel<T, HG, false>, dim3((unsigned)grid),
                 dim3(kSimtThreads), 0, s, k) != cudaSuccess) {
    set_error("fp8_decode_simt_kernel: launch failed: %s", cudaGetErrorString(cudaGetLastError()));
    return BL_ERR_LAUNCH;
  }
  return BL_OK;
}

template <typename T>
int launch_simt(const Args& k, cudaStream_t s) {
  return k.tile_heads == 1   ? launch_simt_heads<T, 1>(k, s)
         : k.tile_heads == 2 ? launch_simt_heads<T, 2>(k, s)
                             : launch_simt_heads<T, 4>(k, s);
}

template <typename T>
int launch_all(const Args& k, const bl_paged_layer& kv, cudaStream_t s) {
  int rc = BL_ERR_UNSUPPORTED;
  if constexpr (sizeof(T) == 2) {
    if (use_tc(kv))
      rc = k.bs % 16 == 0 ? (k.cluster ? launch_tc_dims<T, 1, true>(k, kv, s) : launch_tc_dims<T, 1, false>(k, kv, s))
                          : (k.cluster ? launch_tc_dims<T, 2, true>(k, kv, s) : launch_tc_dims<T, 2, false>(k, kv, s));
    else
      rc = launch_simt<T>(k, s);
  } else {
    rc = launch_simt<T>(k, s);
  }
  if (rc || !k.has_parts || k.cluster) return rc;
  if (launch_pdl(fp8_decode_reduce_kernel<T>, dim3((unsigned)k.batch, (unsigned)k.hq), dim3(kReduceThreads), 0, s, k) !=
      cudaSuccess) {
    set_error("fp8_decode_reduce_kernel: launch failed: %s", cudaGetErrorString(cudaGetLastError()));
    return BL_ERR_LAUNCH;
  }
  return BL_OK;
}

// How a call runs, by its sizes.
struct Way {
  int tile_heads, head_tiles;
  int cluster;   // chunks of a row, joined within a cluster; 0: by the join kernel
  bool planned;
  bool scratch;  // uses the workspace
};

Way way_of(const bl_decode_fp8_args& a) {
  const bl_paged_layer& kv = a.layer.kv;
  const int64_t g = a.num_q_heads / kv.num_kv_heads, chunks = (a.max_seq_len + kChunk - 1) / kChunk;
  const bool tc = use_tc(kv);
  Way w;
  w.tile_heads = tc ? 8 : (int)std::min<int64_t>(g == 3 ? 4 : g, kSimtHeads);
  w.head_tiles = (int)((g + w.tile_heads - 1) / w.tile_heads);
  // A call whose items all fit the GPU at once needs no plan: the order and the
  // claims that it brings would change nothing (one request of 777 tokens: 14.4 us
  // on the device without it, 20.5 us with it).
  w.planned = !(tc && a.batch <= 32 && a.batch * chunks * kv.num_kv_heads * w.head_tiles <= num_sms());
  // Up to kMaxCluster chunks a row, they are joined within a cluster: no join kernel
  // and no workspace either (the same request, calls in a row: 18.0 to 11.4 us).
  w.cluster = !w.planned && chunks > 1 && chunks <= kMaxCluster ? (int)chunks : 0;
  w.scratch = w.planned || (chunks > 1 && !w.cluster);
  return w;
}

}  // namespace
}  // namespace bl

using namespace bl;

extern "C" size_t bl_paged_decode_fp8_workspace_bytes(int64_t batch, int64_t num_q_heads, int64_t head_dim,
                                                      int64_t max_seq_len) {
  if (batch <= 0 || num_q_heads <= 0 || head_dim <= 0 || max_seq_len <= 0) return 0;
  return ws_layout(batch, num_q_heads, head_dim, max_seq_len).total;
}

extern "C" size_t bl_paged_decode_fp8_scratch_bytes(const bl_decode_fp8_args* args) {
  if (!args || check_fp8_layer(args->layer, "bl_paged_decode_fp8_scratch_bytes")) return 0;
  const bl_decode_fp8_args& a = *args;
  const bl_paged_layer& kv = a.layer.kv;
  if (a.batch <= 0 || a.num_q_heads <= 0 || a.num_q_heads % kv.num_kv_heads || a.max_seq_len <= 0) return 0;
  return way_of(a).scratch ? ws_layout(a.batch, a.num_q_heads, kv.head_dim, a.max_seq_len).total : 0;
}

extern "C" int bl_paged_decode_fp8(const bl_decode_fp8_args* args, void* stream) {
  const char* who = "bl_paged_decode_fp8";
  BL_CHECK_ARG(args != nullptr, "%s: args is null", who);
  const bl_decode_fp8_args& a = *args;
  int rc = check_fp8_layer(a.layer, who);
  if (rc) return rc;
  const bl_paged_layer& kv = a.layer.kv;
  BL_CHECK_ARG(a.q && a.out && a.seq_lens, "%s: null q/out/seq_lens", who);
  BL_CHECK_ARG(a.batch > 0 && a.batch <= 65535, "%s: batch must be in [1, 65535]", who);
  BL_CHECK_ARG(a.num_q_heads > 0 && a.num_q_heads <= 65535 && a.num_q_heads % kv.num_kv_heads == 0,
               "num_heads must divide evenly by num_kv_heads");
  BL_CHECK_ARG(a.max_seq_len > 0, "KV cache is empty");
  BL_CHECK_ARG(a.max_seq_len <= INT32_MAX - kChunk, "%s: max_seq_len does not fit in int32", who);
  const int es = elem_size(kv.dtype);
  BL_CHECK_ARG(((uintptr_t)a.q % es) == 0 && ((uintptr_t)a.out % es) == 0,
               "%s: q/out must be aligned to their element type", who);
  const WsLayout w = ws_layout(a.batch, a.num_q_heads, kv.head_dim, a.max_seq_len);
  BL_CHECK_ARG(w.max_units <= INT32_MAX, "%s: too many split-K units", who);
  const Way way = way_of(a);
  if (way.scratch || a.workspace || a.workspace_bytes) {
    if (!a.workspace || a.workspace_bytes < w.total) {
      set_error("%s: workspace too small (%zu < %zu bytes)", who, a.workspace ? a.workspace_bytes : (size_t)0, w.total);
      return BL_ERR_CAPACITY;
    }
    BL_CHECK_ARG(((uintptr_t)a.workspace & 255) == 0, "%s: workspace must be 256-byte aligned", who);
  }
  cudaStream_t s = (cudaStream_t)stream;

  Args k;
  memset(&k, 0, sizeof(k));
  k.q = a.q;
  k.q_sb = a.q_stride_b;
  k.q_sh = a.q_stride_h;
  k.out = a.out;
  k.o_sb = a.out_stride_b;
  k.o_sh = a.out_stride_h;
  k.k_pool = (const uint8_t*)kv.k_pool;
  k.v_pool = (const uint8_t*)kv.v_pool;
  k.k_scale = a.layer.k_scale;
  k.v_scale = a.layer.v_scale;
  k.block_tables = kv.block_tables;
  k.bt_stride = kv.bt_stride;
  k.bt_width = std::min(kv.bt_width, (int64_t)(INT32_MAX - kChunk) / kv.block_size);  // positions are 32-bit
  k.row_ids = kv.row_ids;
  k.seq_lens = a.seq_lens;
  k.num_blocks = kv.num_blocks;
  k.layer = kv.layer;
  k.batch = (int32_t)a.batch;
  k.hq = (int32_t)a.num_q_heads;
  k.hkv = (int32_t)kv.num_kv_heads;
  k.g = k.hq / k.hkv;
  k.tile_heads = way.tile_heads;
  k.head_tiles = way.head_tiles;
  k.planned = way.planned;
  k.cluster = way.cluster;
  k.bs = (int32_t)kv.block_size;
  k.d = (int32_t)kv.head_dim;
  k.q_vec = (k.d == 64 || k.d == 128 || k.d == 256) && ((uintptr_t)a.q & 7) == 0 && a.q_stride_b % 4 == 0 && a.q_stride_h % 4 == 0;
  k.o_vec = ((uintptr_t)a.out & 7) == 0 && a.out_stride_b % 4 == 0 && a.out_stride_h % 4 == 0;
  k.scale_log2 = a.scale * kLog2e;
  char* ws = (char*)a.workspace;
  if (way.scratch) {
    k.hdr = (int32_t*)(ws + w.hdr);
    k.row_base = (const int32_t*)(ws + w.row_base);
    k.units = (const Unit*)(ws + w.units);
    k.ws_lse = (float*)(ws + w.lse);
    k.ws_o = (float*)(ws + w.o);
  }
  k.max_units = (int32_t)w.max_units;
  k.has_parts = a.max_seq_len > kChunk;
  k.err = a.err;

  if (k.planned && !a.plan_ready) {
    PlanArgs p;
    p.seq_lens = a.seq_lens;
    p.batch = k.batch;
    p.max_units = k.max_units;
    p.cap = k.bt_width * kv.block_size;
    p.hdr = (int32_t*)(ws + w.hdr);
    p.row_base = (int32_t*)(ws + w.row_base);
    p.units = (Unit*)(ws + w.units);
    p.err = a.err;
    const int threads = std::min(kPlanThreads, (k.batch + 31) / 32 * 32);  // >= kChunkTiles
    if (launch_pdl(fp8_decode_plan_kernel, dim3(1), dim3(threads), 0, s, p) != cudaSuccess) {
      set_error("fp8_decode_plan_kernel: launch failed: %s", cudaGetErrorString(cudaGetLastError()));
      return BL_ERR_LAUNCH;
    }
  }
  switch (kv.dtype) {
    case BL_F32: return launch_all<float>(k, kv, s);
    case BL_F16: return launch_all<__half>(k, kv, s);
    default: return launch_all<__nv_bfloat16>(k, kv, s);
  }
}
