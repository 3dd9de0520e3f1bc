// Decode attention over an 8-bit paged cache (one query token per request, GQA):
//   out[b, hq] = softmax_t(scale * q[b, hq] . K[b, h, t]) V[b, h, t],  t < len_b,
// with K = code * k_scale[block, h], V = code * v_scale[block, h] (fp8.cuh).
// 8-bit counterpart of decode.cu; the reference chain it stands for is
// SDPAAttentionBackend.attend, src/barellm/attention/backend.py:34-61.
//
// Kernels
//   decode_plan_kernel     (decode.cu) splits rows into 512-token chunks.
//   fp8_decode_tc_kernel   bf16 / fp16 q, head_dim 64, 128 or 256, block_size a
//                          multiple of 16.  Persistent CTAs walk (chunk, KV head,
//                          8 query heads) items.  One producer warp streams 32
//                          tokens of K and V codes a step through a TMA ring;
//                          four consumer warps take every fourth step.
//   fp8_decode_simt_kernel everything else (fp32 q, other head_dims and block
//                          sizes, pools past the tensor map's 2^31 rows): the
//                          same chunks, fp32 multiplies on dequantised tiles.
//   fp8_decode_reduce_kernel  joins the chunks of rows that have several.
//
// Arithmetic of the tensor-core kernel.  Codes are converted to fp16, which
// holds every e4m3 value exactly, and the two products run on mma.sync
// m16n8k16 with fp32 sums.  q is brought to fp16 by a power of two per head
// (its largest magnitude lands in [1, 2)), so a bf16 element keeps all its bits
// down to 2^-16 of the head's largest and loses at most 2^-25 of that below.
// k_scale multiplies the score in fp32.  P (<= 2^8, see below) is rounded to
// fp16, 2^-12 relative.  V's scales are applied to the fp32 sums.
#include <cstring>
#include <mutex>

#include "decode_plan.cuh"
#include "fp8.cuh"

namespace bl {
namespace {

constexpr int kChunk = kDecodeChunkTokens;
constexpr float kLog2e = 1.4426950408889634f;

inline size_t align256(size_t x) { return (x + 255) & ~size_t(255); }

struct WsLayout {
  size_t hdr, row_base, exec, lse, o, total;
  int64_t max_units;
};

WsLayout ws_layout(int64_t batch, int64_t hq, int64_t d, int64_t max_seq_len) {
  WsLayout w;
  w.max_units = batch * ((max_seq_len + kChunk - 1) / kChunk);
  size_t off = 0;
  w.hdr = off;      off += align256(4 * sizeof(int32_t));
  w.row_base = off; off += align256((batch + 1) * sizeof(int32_t));
  w.exec = off;     off += align256(w.max_units * sizeof(int2));
  // a row of one chunk leaves no partial
  const int64_t parts = max_seq_len > kChunk ? w.max_units : 0;
  w.lse = off;      off += align256(parts * hq * sizeof(float));
  w.o = off;        off += align256(parts * hq * d * sizeof(float));
  w.total = off;
  return w;
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
  int32_t batch, hq, hkv, g, head_tiles, bs, d;
  int32_t q_vec;  // q rows can be read four elements at a time
  float scale_log2;
  const int32_t* hdr;
  const int32_t* row_base;
  const int2* exec;
  float* ws_lse;
  float* ws_o;
  int32_t max_units, has_parts;
  int32_t* err;
};

// One item: a chunk of a row, a KV head and up to eight of its query heads.
struct Item {
  int b, chunk, h, hq0, heads;
  int len, t0, t1;  // the chunk's tokens are [t0, t1), t1 <= len
  int nch;          // chunks of the row
};

// False when the plan names a unit outside the batch or the row's length.
__device__ __forceinline__ bool get_item(const Args& a, int64_t item, Item& it) {
  const int per_unit = a.hkv * a.head_tiles;
  const int u = (int)(item / per_unit);
  const int r = (int)(item - (int64_t)u * per_unit);
  it.h = r / a.head_tiles;
  const int ht = r - it.h * a.head_tiles;
  it.hq0 = it.h * a.g + ht * 8;
  it.heads = min(8, a.g - ht * 8);
  const int2 bc = a.exec[u];
  it.b = bc.x;
  it.chunk = bc.y;
  if (bc.x < 0 || bc.x >= a.batch || bc.y < 0) return false;
  const int64_t cap = a.bt_width * a.bs;
  it.len = (int)min((int64_t)a.seq_lens[bc.x], cap);
  const int64_t t0 = (int64_t)bc.y * kChunk;
  if (t0 >= it.len) return false;
  it.t0 = (int)t0;
  it.t1 = (int)min(t0 + kChunk, (int64_t)it.len);
  it.nch = (int)(((int64_t)it.len + kChunk - 1) / kChunk);
  return true;
}

__device__ __forceinline__ int plan_units(const Args& a) {
  const int units = a.hdr[0];
  if (a.hdr[1] != kDecodePlanMagic || a.hdr[2] != a.batch || units < 0 || units > a.max_units) {
    if (threadIdx.x == 0 && blockIdx.x == 0) raise_dev(a.err, BL_DEVERR_WORKSPACE);
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

// One element of an item's result: the output for a row of one chunk, else the
// chunk's partial (o, log2-sum-exp) for the reduce kernel.
template <typename T>
__device__ __forceinline__ void store_result(const Args& a, const Item& it, int hd, int d, float M, float L, float O) {
  const int hq = it.hq0 + hd;
  const float val = L == 0.f ? 0.f : O / L;  // a NaN sum stays NaN
  if (it.nch <= 1) {
    reinterpret_cast<T*>(a.out)[(int64_t)it.b * a.o_sb + (int64_t)hq * a.o_sh + d] = from_f32<T>(val);
    return;
  }
  const int64_t slot = (int64_t)a.row_base[it.b] + it.chunk;
  if (!a.has_parts || slot < 0 || slot >= a.max_units) {  // longer than max_seq_len allows
    if (d == 0) raise_dev(a.err, BL_DEVERR_WORKSPACE);
    return;
  }
  a.ws_o[(slot * a.hq + hq) * a.d + d] = val;
  if (d == 0) a.ws_lse[slot * a.hq + hq] = L == 0.f ? -INFINITY : M + __log2f(L);
}

// ---------------------------------------------------------------------------
// tensor-core kernel
// ---------------------------------------------------------------------------
constexpr int kNW = 4;                      // consumer warps
constexpr int kThreadsTC = (kNW + 1) * 32;  // + the producer warp
constexpr int kStepTokens = 32;             // tokens a consumer warp takes at a time: two 16-token tiles
constexpr int kTiles = kChunk / 16;         // 16-token tiles of a chunk, one per producer lane
static_assert(kTiles == 32, "a producer lane holds one tile of the chunk");

template <int D>
struct Cfg {
  static constexpr int kRow = D < 128 ? D : 128;  // bytes of a token row in one TMA box
  static constexpr int kHalves = D / kRow;
  static constexpr int kTile = 16 * D;            // K (or V) codes of one tile
  static constexpr int kSlot = 4 * kTile;         // K and V of two tiles
  static constexpr int kStages = D == 256 ? 4 : 8;
  static constexpr int kBox = 16 * kRow;
};

template <int D>
struct TCShared {
  uint64_t full[Cfg<D>::kStages];
  uint64_t empty[Cfg<D>::kStages];
  float scales[Cfg<D>::kStages][4];  // k_scale of the two tiles, v_scale of the two tiles
  float ml[kNW][8][2];
  int abort;
};

// 16-byte chunk `c` of token row `r` within a box, as TMA's swizzle places it
template <int ROW>
__device__ __forceinline__ int swizzled(int r, int c) {
  return r * ROW + ((ROW == 128 ? (c ^ (r & 7)) : (c ^ ((r >> 1) & 3))) << 4);
}

template <typename T, int D>
__global__ void __launch_bounds__(kThreadsTC) fp8_decode_tc_kernel(const Args a, const __grid_constant__ CUtensorMap kmap,
                                                                   const __grid_constant__ CUtensorMap vmap) {
  using C = Cfg<D>;
  extern __shared__ __align__(1024) unsigned char smem_raw[];
  unsigned char* slots =
      reinterpret_cast<unsigned char*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  float* comb_o = reinterpret_cast<float*>(slots + C::kStages * C::kSlot);  // [kNW][min(g, 8)][D]
  const int gmax = min(a.g, 8);
  TCShared<D>* sh = reinterpret_cast<TCShared<D>*>(comb_o + kNW * gmax * D);

  const int warp = threadIdx.x >> 5;
  const int lane = threadIdx.x & 31;
  if (threadIdx.x == 0) {
    for (int s = 0; s < C::kStages; ++s) {
      mbar_init(&sh->full[s], 1);
      mbar_init(&sh->empty[s], 1);
    }
    sh->abort = 0;
    fence_mbar_init();
  }
  __syncthreads();

  pdl_wait();  // the plan (and all work before it) is complete and visible
  const int64_t items = (int64_t)plan_units(a) * a.hkv * a.head_tiles;

  if (warp == kNW) {
    // ------------------------------ producer ------------------------------
    if (lane == 0) {
      prefetch_tensormap(&kmap);
      prefetch_tensormap(&vmap);
    }
    const uint64_t policy = policy_evict_first();
    int issued = 0;  // steps issued so far == ring index of the next
    bool ok = true;
    for (int64_t item = blockIdx.x; item < items && ok; item += gridDim.x) {
      Item it;
      if (!get_item(a, item, it)) {
        if (lane == 0) raise_dev(a.err, BL_DEVERR_WORKSPACE);
        continue;
      }
      // lane i holds tile i of the chunk: its pool row and its scales
      const int tok = it.t0 + 16 * lane;
      int32_t y = 0;
      float ks = 1.f, vs = 1.f;
      if (tok < it.t1) {
        const int64_t row = a.row_ids ? (int64_t)a.row_ids[it.b] : (int64_t)it.b;
        const int lb = tok / a.bs;
        int64_t phys = a.block_tables[row * a.bt_stride + lb];
        if (phys < 0 || phys >= a.num_blocks) {
          raise_dev(a.err, BL_DEVERR_BLOCK_ID);
          phys = 0;
        }
        const int64_t slot = (a.layer * a.num_blocks + phys) * a.hkv + it.h;
        ks = a.k_scale[slot];
        vs = a.v_scale[slot];
        y = (int32_t)(slot * a.bs + (tok - lb * a.bs));
      }
      const int ntiles = (it.t1 - it.t0 + 15) / 16;
      for (int t = 0; t < ntiles; t += 2) {
        const int slot = issued % C::kStages;
        if (!__all_sync(0xffffffffu, mbar_wait(&sh->empty[slot], ((issued / C::kStages) & 1) ^ 1))) {
          raise_dev(a.err, BL_DEVERR_TIMEOUT);
          sh->abort = 1;
          ok = false;
          break;
        }
        const int x = lane - t;  // this lane's tile of the step: 0 or 1
        const int n = min(2, ntiles - t);
        if (x >= 0 && x < 2) {
          // a step with one tile repeats its V scale for the missing one (no effect: its codes are masked)
          sh->scales[slot][x] = ks;
          sh->scales[slot][2 + x] = vs;
        }
        const float vs0 = __shfl_sync(0xffffffffu, vs, t);
        __syncwarp();
        if (lane == 0) {
          if (n == 1) sh->scales[slot][3] = vs0;
          mbar_arrive_expect_tx(&sh->full[slot], n * 2 * C::kTile);
        }
        __syncwarp();
        if (x >= 0 && x < n) {
          unsigned char* kd = slots + slot * C::kSlot + x * C::kTile;
          unsigned char* vd = kd + 2 * C::kTile;
#pragma unroll
          for (int hf = 0; hf < C::kHalves; ++hf) {
            tma_load_2d_hint(kd + hf * C::kBox, &kmap, &sh->full[slot], hf * 128, y, policy);
            tma_load_2d_hint(vd + hf * C::kBox, &vmap, &sh->full[slot], hf * 128, y, policy);
          }
        }
        ++issued;
      }
    }
    // Drain: every issued copy lands before the CTA can exit.
    __syncwarp();
    if (lane == 0) {
      for (int s = 0; s < C::kStages && s < issued; ++s) {
        const int last = s + ((issued - 1 - s) / C::kStages) * C::kStages;
        if (!mbar_wait(&sh->full[s], (last / C::kStages) & 1)) raise_dev(a.err, BL_DEVERR_TIMEOUT);
      }
    }
    return;
  }

  // ------------------------------ consumers ------------------------------
  zero_empty_rows<T>(a, kNW * 32);
  constexpr int kKS = D / 16;                // 16-dim steps of the score product
  constexpr int kLaneDims = C::kRow / 8;     // output dims a lane owns per half
  constexpr int kWords = kLaneDims / 4;      // V words a lane reads per token and half
  const int g_row = lane >> 2;  // mma group: token (scores), query head (q, P), dim block (output)
  const int t4 = lane & 3;
  int base = 0;  // ring index of the item's first step

  for (int64_t item = blockIdx.x; item < items; item += gridDim.x) {
    Item it;
    if (!get_item(a, item, it)) continue;  // flagged by the producer
    const int nsteps = (it.t1 - it.t0 + kStepTokens - 1) / kStepTokens;

    // q as fp16 B fragments.  Position k of a 16-dim step stands for dim
    // 16 ks + 4 t + {0, 1} (k = 2t, 2t+1) and + {2, 3} (k = 2t+8, 2t+9): the order
    // in which a lane finds the K codes of one 32-bit word.
    uint32_t qf[kKS][2];
    float f0, f1;  // scale * log2(e) * the head's power of two, heads 2 t4 and 2 t4 + 1
    {
      const bool valid = g_row < it.heads;
      const T* qp = reinterpret_cast<const T*>(a.q) + (int64_t)it.b * a.q_sb +
                    (int64_t)(it.hq0 + (valid ? g_row : 0)) * a.q_sh;
      float qv[kKS][4];
      float amax = 0.f;
#pragma unroll
      for (int ks = 0; ks < kKS; ++ks) {
        const T* p = qp + ks * 16 + 4 * t4;
        if (a.q_vec) {
          const uint2 w = *reinterpret_cast<const uint2*>(p);
          const float2 x = unpack2<T>(w.x), y = unpack2<T>(w.y);
          qv[ks][0] = x.x, qv[ks][1] = x.y, qv[ks][2] = y.x, qv[ks][3] = y.y;
        } else {
#pragma unroll
          for (int e = 0; e < 4; ++e) qv[ks][e] = to_f32<T>(p[e]);
        }
#pragma unroll
        for (int e = 0; e < 4; ++e) amax = fmaxf(amax, finite_abs(qv[ks][e]));
      }
      amax = fmaxf(amax, __shfl_xor_sync(0xffffffffu, amax, 1));
      amax = fmaxf(amax, __shfl_xor_sync(0xffffffffu, amax, 2));
      int e = (int)(__float_as_uint(amax) >> 23) - 127;
      e = amax > 0.f ? min(max(e, -126), 126) : 0;
      const float down = valid ? exp2_int(-e) : 0.f;
#pragma unroll
      for (int ks = 0; ks < kKS; ++ks) {
        qf[ks][0] = pack2<__half>(valid ? qv[ks][0] * down : 0.f, valid ? qv[ks][1] * down : 0.f);
        qf[ks][1] = pack2<__half>(valid ? qv[ks][2] * down : 0.f, valid ? qv[ks][3] * down : 0.f);
      }
      const float f = exp2_int(e) * a.scale_log2;
      f0 = __shfl_sync(0xffffffffu, f, 8 * t4);
      f1 = __shfl_sync(0xffffffffu, f, 8 * t4 + 4);
    }

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

    for (int i = warp; i < nsteps; i += kNW) {
      const int gi = base + i;
      const int slot = gi % C::kStages;
      if (*(volatile int*)&sh->abort) break;
      if (!mbar_wait(&sh->full[slot], (gi / C::kStages) & 1)) {
        raise_dev(a.err, BL_DEVERR_TIMEOUT);
        *(volatile int*)&sh->abort = 1;
        break;
      }
      __syncwarp();
      const float4 sc = *reinterpret_cast<const float4*>(sh->scales[slot]);
      const uint32_t kb = smem_u32(slots + slot * C::kSlot);
      const unsigned char* vb = slots + slot * C::kSlot + 2 * C::kTile;

      // S^T[token][head] = K[token] . q[head]
      float s[2][4];
#pragma unroll
      for (int x = 0; x < 2; ++x) {
        s[x][0] = s[x][1] = s[x][2] = s[x][3] = 0.f;
#pragma unroll
        for (int hf = 0; hf < C::kHalves; ++hf)
#pragma unroll
          for (int c = 0; c < C::kRow / 16; c += 2) {
            uint32_t r0, r1, r2, r3;
            const int r = (lane & 7) + (lane & 8);
            ldmatrix_x4(kb + x * C::kTile + hf * C::kBox + swizzled<C::kRow>(r, c + (lane >> 4)), r0, r1, r2, r3);
            const int ks = hf * (C::kRow / 16) + c;
            mma_16816<__half>(s[x][0], s[x][1], s[x][2], s[x][3], e4m3lo_to_f16x2(r0), e4m3lo_to_f16x2(r1),
                              e4m3hi_to_f16x2(r0), e4m3hi_to_f16x2(r1), qf[ks][0], qf[ks][1]);
            mma_16816<__half>(s[x][0], s[x][1], s[x][2], s[x][3], e4m3lo_to_f16x2(r2), e4m3lo_to_f16x2(r3),
                              e4m3hi_to_f16x2(r2), e4m3hi_to_f16x2(r3), qf[ks + 1][0], qf[ks + 1][1]);
          }
      }
      const int nvalid = it.t1 - (it.t0 + i * kStepTokens);  // tokens of the step that exist
#pragma unroll
      for (int x = 0; x < 2; ++x) {
        const float ks = x ? sc.y : sc.x;
        s[x][0] *= f0 * ks, s[x][1] *= f1 * ks, s[x][2] *= f0 * ks, s[x][3] *= f1 * ks;
      }
      if (nvalid < kStepTokens) {
#pragma unroll
        for (int x = 0; x < 2; ++x) {
          if (16 * x + g_row >= nvalid) s[x][0] = s[x][1] = -INFINITY;
          if (16 * x + g_row + 8 >= nvalid) s[x][2] = s[x][3] = -INFINITY;
        }
      }
      float mx0 = fmaxf(fmaxf(s[0][0], s[0][2]), fmaxf(s[1][0], s[1][2]));
      float mx1 = fmaxf(fmaxf(s[0][1], s[0][3]), fmaxf(s[1][1], s[1][3]));
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
        l0 *= al0, l1 *= al1;
#pragma unroll
        for (int hf = 0; hf < C::kHalves; ++hf)
#pragma unroll
          for (int j = 0; j < 2 * kWords; ++j) {
            o[hf][j][0] *= al0, o[hf][j][2] *= al0;
            o[hf][j][1] *= al1, o[hf][j][3] *= al1;
          }
      }
      const float u0 = m0 == -INFINITY ? 0.f : m0, u1 = m1 == -INFINITY ? 0.f : m1;
      // exponentials and row sums
#pragma unroll
      for (int x = 0; x < 2; ++x) {
        s[x][0] = fast_exp2(s[x][0] - u0), s[x][2] = fast_exp2(s[x][2] - u0);
        s[x][1] = fast_exp2(s[x][1] - u1), s[x][3] = fast_exp2(s[x][3] - u1);
        l0 += s[x][0] + s[x][2];
        l1 += s[x][1] + s[x][3];
      }
#pragma unroll
      for (int x = 0; x < 2; ++x) {
        const float vs = x ? sc.w : sc.z;
        // A much larger scale becomes the reference (the sums shrink by a
        // power of two); a much smaller one is added through its own sums.
        if (vs > vref * 16.f) {
          const float r = vref * pow2_inverse(vs);
          vref = vs;
          vinv = pow2_inverse(vs);
#pragma unroll
          for (int hf = 0; hf < C::kHalves; ++hf)
#pragma unroll
            for (int j = 0; j < 2 * kWords; ++j)
#pragma unroll
              for (int e = 0; e < 4; ++e) o[hf][j][e] *= r;
        }
        const float ratio = vs * vinv;
        const bool fold = ratio >= 0.015625f;
        const float pr = fold ? ratio : 1.f;
        // P^T (tokens x heads) -> B fragment (k = token, n = head)
        const uint32_t pb0 = movmatrix_trans(pack2<__half>(s[x][0] * pr, s[x][1] * pr));
        const uint32_t pb1 = movmatrix_trans(pack2<__half>(s[x][2] * pr, s[x][3] * pr));
        // O^T[dim][head] += V^T[dim][token] P^T[token][head].  A lane reads the
        // 16 (kLaneDims) consecutive dims g_row * kLaneDims of tokens 2t, 2t+1,
        // 2t+8, 2t+9 and pairs two tokens' bytes, so a converted pair is one A
        // register (row = dim, two consecutive tokens).
        const int r0 = 2 * t4;
        const int left = nvalid - 16 * x;
#pragma unroll
        for (int hf = 0; hf < C::kHalves; ++hf) {
          const unsigned char* box = vb + x * C::kTile + hf * C::kBox;
          uint32_t w[4][kWords];
#pragma unroll
          for (int k = 0; k < 4; ++k) {
            const int r = r0 + (k & 1) + 8 * (k >> 1);
            const unsigned char* p =
                box + swizzled<C::kRow>(r, (g_row * kLaneDims) >> 4) + ((g_row * kLaneDims) & 15);
            if constexpr (kWords == 4) {
              const uint4 v = *reinterpret_cast<const uint4*>(p);
              w[k][0] = v.x, w[k][1] = v.y, w[k][2] = v.z, w[k][3] = v.w;
            } else {
              const uint2 v = *reinterpret_cast<const uint2*>(p);
              w[k][0] = v.x, w[k][1] = v.y;
            }
            // slots past the length hold stale codes (possibly NaN): 0 * NaN is NaN
            if (left < 16 && r >= left) {
#pragma unroll
              for (int j = 0; j < kWords; ++j) w[k][j] = 0u;
            }
          }
#pragma unroll
          for (int j = 0; j < kWords; ++j) {
            const uint32_t lo01 = __byte_perm(w[0][j], w[1][j], 0x5140), lo23 = __byte_perm(w[0][j], w[1][j], 0x7362);
            const uint32_t hi01 = __byte_perm(w[2][j], w[3][j], 0x5140), hi23 = __byte_perm(w[2][j], w[3][j], 0x7362);
            float(&d0)[4] = o[hf][2 * j];
            float(&d1)[4] = o[hf][2 * j + 1];
            if (fold) {
              mma_16816<__half>(d0[0], d0[1], d0[2], d0[3], e4m3lo_to_f16x2(lo01), e4m3hi_to_f16x2(lo01),
                                e4m3lo_to_f16x2(hi01), e4m3hi_to_f16x2(hi01), pb0, pb1);
              mma_16816<__half>(d1[0], d1[1], d1[2], d1[3], e4m3lo_to_f16x2(lo23), e4m3hi_to_f16x2(lo23),
                                e4m3lo_to_f16x2(hi23), e4m3hi_to_f16x2(hi23), pb0, pb1);
            } else {
              float z0[4] = {0.f, 0.f, 0.f, 0.f}, z1[4] = {0.f, 0.f, 0.f, 0.f};
              mma_16816<__half>(z0[0], z0[1], z0[2], z0[3], e4m3lo_to_f16x2(lo01), e4m3hi_to_f16x2(lo01),
                                e4m3lo_to_f16x2(hi01), e4m3hi_to_f16x2(hi01), pb0, pb1);
              mma_16816<__half>(z1[0], z1[1], z1[2], z1[3], e4m3lo_to_f16x2(lo23), e4m3hi_to_f16x2(lo23),
                                e4m3lo_to_f16x2(hi23), e4m3hi_to_f16x2(hi23), pb0, pb1);
#pragma unroll
              for (int e = 0; e < 4; ++e) d0[e] += ratio * z0[e], d1[e] += ratio * z1[e];
            }
          }
        }
      }
      __syncwarp();
      if (lane == 0) mbar_arrive(&sh->empty[slot]);
    }
    base += nsteps;

    // ---- merge the warps ----
#pragma unroll
    for (int off = 4; off < 32; off <<= 1) {
      l0 += __shfl_xor_sync(0xffffffffu, l0, off);
      l1 += __shfl_xor_sync(0xffffffffu, l1, off);
    }
    const int h0 = 2 * t4, h1 = 2 * t4 + 1;
    if (g_row == 0) {
      sh->ml[warp][h0][0] = m0, sh->ml[warp][h0][1] = l0;
      sh->ml[warp][h1][0] = m1, sh->ml[warp][h1][1] = l1;
    }
    float* cw = comb_o + warp * gmax * D;
#pragma unroll
    for (int hf = 0; hf < C::kHalves; ++hf)
#pragma unroll
      for (int j = 0; j < 2 * kWords; ++j) {
        const int d0 = hf * 128 + g_row * kLaneDims + 2 * j;
        if (h0 < it.heads) *reinterpret_cast<float2*>(cw + h0 * D + d0) = make_float2(o[hf][j][0] * vref, o[hf][j][2] * vref);
        if (h1 < it.heads) *reinterpret_cast<float2*>(cw + h1 * D + d0) = make_float2(o[hf][j][1] * vref, o[hf][j][3] * vref);
      }
    named_barrier_sync(1, kNW * 32);
    for (int e = threadIdx.x; e < it.heads * D; e += kNW * 32) {
      const int hd = e / D;
      const int d = e - hd * D;
      float M = -INFINITY;
#pragma unroll
      for (int w = 0; w < kNW; ++w) M = fmaxf(M, sh->ml[w][hd][0]);
      float L = 0.f, O = 0.f;
#pragma unroll
      for (int w = 0; w < kNW; ++w) {
        const float mw = sh->ml[w][hd][0];
        const float f = mw == -INFINITY ? 0.f : (mw == M ? 1.f : fast_exp2(mw - M));
        L += f * sh->ml[w][hd][1];
        O += f * comb_o[(w * gmax + hd) * D + d];
      }
      store_result<T>(a, it, hd, d, M, L, O);
    }
    named_barrier_sync(1, kNW * 32);
  }
}

// ---------------------------------------------------------------------------
// SIMT kernel: any element type, head_dim <= 256, any block size
// ---------------------------------------------------------------------------
constexpr int kSimtThreads = 256;
constexpr int kSimtTokens = 32;  // tokens per tile: one per lane in the score phase

struct SimtShared {
  int64_t row[kSimtTokens];  // byte offset of the token's codes, -1: none
  float ks[kSimtTokens], vs[kSimtTokens];
  float p[8][kSimtTokens];
  float alpha[8], l[8], m[8];
};

// Eight warps: in the score phase warp w owns query head w and lane i token i;
// in the P V phase a thread owns one dim of every (256 / Dp)-th head.
template <typename T>
__global__ void __launch_bounds__(kSimtThreads) fp8_decode_simt_kernel(const Args a) {
  extern __shared__ __align__(1024) unsigned char smem_raw[];
  SimtShared* sh = reinterpret_cast<SimtShared*>(smem_raw);
  const int dp1 = a.d + 1;
  float* qs = reinterpret_cast<float*>(smem_raw + sizeof(SimtShared));  // [8][d]
  float* tile = qs + 8 * a.d;                                          // [32][d + 1]
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  int dp = 32;
  while (dp < a.d) dp *= 2;
  const int vd = tid % dp, vh0 = tid / dp, vstep = kSimtThreads / dp;

  pdl_wait();
  const int64_t items = (int64_t)plan_units(a) * a.hkv * a.head_tiles;
  zero_empty_rows<T>(a, kSimtThreads);

  auto load_tile = [&](const uint8_t* pool, const float* sc) {
    const bool words = (a.d & 3) == 0;
    const int per = words ? a.d / 4 : a.d;
    for (int e = tid; e < kSimtTokens * per; e += kSimtThreads) {
      const int t = e / per, c = e - t * per;
      const int64_t r = sh->row[t];
      if (words) {
        float2 x = make_float2(0.f, 0.f), y = x;
        if (r >= 0) {
          const uint32_t w = *reinterpret_cast<const uint32_t*>(pool + r + 4 * c);
          x = e4m3x2_to_float2((uint16_t)w), y = e4m3x2_to_float2((uint16_t)(w >> 16));
        }
        const float s = r >= 0 ? sc[t] : 0.f;
        float* p = tile + t * dp1 + 4 * c;
        p[0] = x.x * s, p[1] = x.y * s, p[2] = y.x * s, p[3] = y.y * s;
      } else {
        tile[t * dp1 + c] = r >= 0 ? e4m3_to_float(pool[r + c]) * sc[t] : 0.f;
      }
    }
  };

  for (int64_t item = blockIdx.x; item < items; item += gridDim.x) {
    Item it;
    if (!get_item(a, item, it)) {
      if (tid == 0) raise_dev(a.err, BL_DEVERR_WORKSPACE);
      continue;
    }
    __syncthreads();  // the previous item's shared state is no longer read
    for (int e = tid; e < it.heads * a.d; e += kSimtThreads) {
      const int h = e / a.d;
      qs[e] = to_f32<T>(reinterpret_cast<const T*>(a.q)[(int64_t)it.b * a.q_sb + (int64_t)(it.hq0 + h) * a.q_sh + (e - h * a.d)]) *
              a.scale_log2;
    }
    float m = -INFINITY, l = 0.f;  // warp w: head w
    float acc[8];
#pragma unroll
    for (int k = 0; k < 8; ++k) acc[k] = 0.f;
    const int64_t row = a.row_ids ? (int64_t)a.row_ids[it.b] : (int64_t)it.b;
    for (int t0 = it.t0; t0 < it.t1; t0 += kSimtTokens) {
      __syncthreads();  // the previous tile is no longer read; qs is complete
      if (tid < kSimtTokens) {
        const int t = t0 + tid;
        int64_t r = -1;
        if (t < it.t1) {
          const int lb = t / a.bs;
          const int64_t phys = a.block_tables[row * a.bt_stride + lb];
          if (phys < 0 || phys >= a.num_blocks) {
            raise_dev(a.err, BL_DEVERR_BLOCK_ID);
          } else {
            const int64_t slot = (a.layer * a.num_blocks + phys) * a.hkv + it.h;
            r = (slot * a.bs + (t - lb * a.bs)) * a.d;
            sh->ks[tid] = a.k_scale[slot];
            sh->vs[tid] = a.v_scale[slot];
          }
        }
        sh->row[tid] = r;
      }
      __syncthreads();
      load_tile(a.k_pool, sh->ks);
      __syncthreads();
      if (warp < it.heads) {
        const float* qh = qs + warp * a.d;
        const float* kt = tile + lane * dp1;
        float s = 0.f;
        for (int d = 0; d < a.d; ++d) s = fmaf(qh[d], kt[d], s);
        if (sh->row[lane] < 0) s = -INFINITY;
        float mx = s;
#pragma unroll
        for (int o = 16; o > 0; o >>= 1) mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, o));
        const float mn = fmaxf(m, mx);
        const float al = mn == m ? 1.f : fast_exp2(m - mn);
        const float p = fast_exp2(s - (mn == -INFINITY ? 0.f : mn));
        float ps = p;
#pragma unroll
        for (int o = 16; o > 0; o >>= 1) ps += __shfl_xor_sync(0xffffffffu, ps, o);
        m = mn;
        l = l * al + ps;
        sh->p[warp][lane] = p;
        if (lane == 0) sh->alpha[warp] = al;
      }
      __syncthreads();
      load_tile(a.v_pool, sh->vs);
      __syncthreads();
      if (vd < a.d) {
#pragma unroll
        for (int k = 0; k < 8; ++k) {
          const int h = vh0 + k * vstep;
          if (h >= it.heads) break;
          float x = acc[k] * sh->alpha[h];
#pragma unroll 8
          for (int t = 0; t < kSimtTokens; ++t) x = fmaf(sh->p[h][t], tile[t * dp1 + vd], x);
          acc[k] = x;
        }
      }
    }
    if (warp < it.heads && lane == 0) {
      sh->m[warp] = m;
      sh->l[warp] = l;
    }
    __syncthreads();
    if (vd < a.d) {
#pragma unroll
      for (int k = 0; k < 8; ++k) {
        const int h = vh0 + k * vstep;
        if (h >= it.heads) break;
        store_result<T>(a, it, h, vd, sh->m[h], sh->l[h], acc[k]);
      }
    }
  }
}

size_t simt_smem(int d) { return sizeof(SimtShared) + sizeof(float) * (8 * (size_t)d + kSimtTokens * (d + 1)); }

// ---------------------------------------------------------------------------
// reduce: rows of several chunks
// ---------------------------------------------------------------------------
constexpr int kReduceThreads = 128;
constexpr int kReduceTile = 512;  // chunks whose weights are in shared memory at a time

// grid: (batch, hq)
template <typename T>
__global__ void __launch_bounds__(kReduceThreads) fp8_decode_reduce_kernel(const Args a) {
  pdl_wait();  // the partials are complete and visible
  const int b = blockIdx.x, hq = blockIdx.y, tid = threadIdx.x;
  const int64_t len = min((int64_t)a.seq_lens[b], a.bt_width * a.bs);
  if (len <= kChunk) return;
  const int nch = (int)((len + kChunk - 1) / kChunk);
  const int64_t base = a.row_base[b];
  if (base < 0 || base + nch > a.max_units) return;  // flagged by the plan or the attention kernel
  __shared__ float s_w[kReduceTile];
  __shared__ float s_red[kReduceThreads / 32];
  float M = -INFINITY;
  for (int c = tid; c < nch; c += kReduceThreads) M = fmaxf(M, a.ws_lse[(base + c) * a.hq + hq]);
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) M = fmaxf(M, __shfl_xor_sync(0xffffffffu, M, o));
  if ((tid & 31) == 0) s_red[tid >> 5] = M;
  __syncthreads();
#pragma unroll
  for (int w = 0; w < kReduceThreads / 32; ++w) M = fmaxf(M, s_red[w]);
  float num[2] = {0.f, 0.f}, den = 0.f;  // head_dim <= 2 * kReduceThreads
  const int64_t cstride = (int64_t)a.hq * a.d;
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
      const int d = tid + k * kReduceThreads;
      if (d >= a.d) break;
#pragma unroll 8
      for (int c = 0; c < n; ++c) num[k] += s_w[c] * po[c * cstride + d];
    }
    for (int c = 0; c < n; ++c) den += s_w[c];
  }
#pragma unroll
  for (int k = 0; k < 2; ++k) {
    const int d = tid + k * kReduceThreads;
    if (d < a.d)
      reinterpret_cast<T*>(a.out)[(int64_t)b * a.o_sb + (int64_t)hq * a.o_sh + d] =
          from_f32<T>(den == 0.f ? 0.f : num[k] / den);
  }
}

// ---------------------------------------------------------------------------
// host side
// ---------------------------------------------------------------------------
// The tensor-core kernel: 16-bit q, a head_dim it is built for, whole 16-token
// tiles in a block, and pool rows within the tensor map's 32-bit coordinates.
bool use_tc(const bl_paged_layer& kv) {
  const double rows = (double)kv.num_layers * kv.num_blocks * kv.num_kv_heads * kv.block_size;
  return (kv.dtype == BL_BF16 || kv.dtype == BL_F16) && (kv.head_dim == 64 || kv.head_dim == 128 || kv.head_dim == 256) &&
         kv.block_size % 16 == 0 && rows <= (double)INT32_MAX;
}

template <typename T, int D>
int launch_tc(const Args& k, const bl_paged_layer& kv, cudaStream_t s) {
  using C = Cfg<D>;
  CUtensorMap kmap, vmap;
  const uint64_t rows = (uint64_t)kv.num_layers * kv.num_blocks * kv.num_kv_heads * kv.block_size;
  if (!make_tmap_rows_8bit(&kmap, kv.k_pool, D, rows, C::kRow, 16) ||
      !make_tmap_rows_8bit(&vmap, kv.v_pool, D, rows, C::kRow, 16))
    return BL_ERR_LAUNCH;
  const size_t fixed = 1024 + (size_t)C::kStages * C::kSlot + sizeof(TCShared<D>);
  const size_t smem = fixed + (size_t)kNW * std::min(k.g, 8) * D * sizeof(float);
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
      if (cudaFuncSetAttribute(fp8_decode_tc_kernel<T, D>, cudaFuncAttributeMaxDynamicSharedMemorySize,
                               (int)(fixed + (size_t)kNW * 8 * D * sizeof(float))) != cudaSuccess ||
          cudaOccupancyMaxActiveBlocksPerMultiprocessor(&o, fp8_decode_tc_kernel<T, D>, kThreadsTC, smem) !=
              cudaSuccess) {
        set_error("fp8_decode_tc_kernel: %s", cudaGetErrorString(cudaGetLastError()));
        return BL_ERR_LAUNCH;
      }
      *slot = std::max(o, 1);
    }
    occ = *slot;
  }
  const int64_t grid = std::min<int64_t>((int64_t)num_sms() * occ, items);
  if (launch_pdl(fp8_decode_tc_kernel<T, D>, dim3((unsigned)grid), dim3(kThreadsTC), smem, s, k, kmap, vmap) !=
      cudaSuccess) {
    set_error("fp8_decode_tc_kernel: launch failed: %s", cudaGetErrorString(cudaGetLastError()));
    return BL_ERR_LAUNCH;
  }
  return BL_OK;
}

template <typename T>
int launch_simt(const Args& k, cudaStream_t s) {
  const size_t smem = simt_smem(k.d);
  const int64_t items = (int64_t)k.max_units * k.hkv * k.head_tiles;
  const int64_t grid = std::min<int64_t>((int64_t)num_sms() * 4, items);
  if (launch_pdl(fp8_decode_simt_kernel<T>, dim3((unsigned)grid), dim3(kSimtThreads), smem, s, k) != cudaSuccess) {
    set_error("fp8_decode_simt_kernel: launch failed: %s", cudaGetErrorString(cudaGetLastError()));
    return BL_ERR_LAUNCH;
  }
  return BL_OK;
}

template <typename T>
int launch_all(const Args& k, const bl_paged_layer& kv, cudaStream_t s) {
  int rc = BL_ERR_UNSUPPORTED;
  if constexpr (sizeof(T) == 2) {
    if (use_tc(kv))
      rc = k.d == 64 ? launch_tc<T, 64>(k, kv, s) : k.d == 128 ? launch_tc<T, 128>(k, kv, s) : launch_tc<T, 256>(k, kv, s);
    else
      rc = launch_simt<T>(k, s);
  } else {
    rc = launch_simt<T>(k, s);
  }
  if (rc || !k.has_parts) return rc;
  if (launch_pdl(fp8_decode_reduce_kernel<T>, dim3((unsigned)k.batch, (unsigned)k.hq), dim3(kReduceThreads), 0, s, k) !=
      cudaSuccess) {
    set_error("fp8_decode_reduce_kernel: launch failed: %s", cudaGetErrorString(cudaGetLastError()));
    return BL_ERR_LAUNCH;
  }
  return BL_OK;
}

}  // namespace
}  // namespace bl

using namespace bl;

extern "C" size_t bl_paged_decode_fp8_workspace_bytes(int64_t batch, int64_t num_q_heads, int64_t head_dim,
                                                      int64_t max_seq_len) {
  if (batch <= 0 || num_q_heads <= 0 || head_dim <= 0 || max_seq_len <= 0) return 0;
  return ws_layout(batch, num_q_heads, head_dim, max_seq_len).total;
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
  BL_CHECK_ARG(a.max_seq_len <= INT32_MAX, "%s: max_seq_len does not fit in int32", who);
  const int es = elem_size(kv.dtype);
  BL_CHECK_ARG(((uintptr_t)a.q % es) == 0 && ((uintptr_t)a.out % es) == 0,
               "%s: q/out must be aligned to their element type", who);
  const WsLayout w = ws_layout(a.batch, a.num_q_heads, kv.head_dim, a.max_seq_len);
  if (!a.workspace || a.workspace_bytes < w.total) {
    set_error("%s: workspace too small (%zu < %zu bytes)", who, a.workspace ? a.workspace_bytes : (size_t)0, w.total);
    return BL_ERR_CAPACITY;
  }
  BL_CHECK_ARG(((uintptr_t)a.workspace & 255) == 0, "%s: workspace must be 256-byte aligned", who);
  BL_CHECK_ARG(w.max_units <= INT32_MAX, "%s: too many split-K units", who);
  char* ws = (char*)a.workspace;
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
  k.bt_width = kv.bt_width;
  k.row_ids = kv.row_ids;
  k.seq_lens = a.seq_lens;
  k.num_blocks = kv.num_blocks;
  k.layer = kv.layer;
  k.batch = (int32_t)a.batch;
  k.hq = (int32_t)a.num_q_heads;
  k.hkv = (int32_t)kv.num_kv_heads;
  k.g = k.hq / k.hkv;
  k.head_tiles = (k.g + 7) / 8;
  k.bs = (int32_t)kv.block_size;
  k.d = (int32_t)kv.head_dim;
  k.q_vec = ((uintptr_t)a.q & 7) == 0 && a.q_stride_b % 4 == 0 && a.q_stride_h % 4 == 0;
  k.scale_log2 = a.scale * kLog2e;
  k.hdr = (const int32_t*)(ws + w.hdr);
  k.row_base = (const int32_t*)(ws + w.row_base);
  k.exec = (const int2*)(ws + w.exec);
  k.ws_lse = (float*)(ws + w.lse);
  k.ws_o = (float*)(ws + w.o);
  k.max_units = (int32_t)w.max_units;
  k.has_parts = a.max_seq_len > kChunk;
  k.err = a.err;

  if (!a.plan_ready) {
    DecodePlanArgs p;
    p.seq_lens = a.seq_lens;
    p.batch = k.batch;
    p.bs = 1;  // chunks are counted in tokens
    p.chunk_blocks = kChunk;
    p.bt_width = (int32_t)std::min<int64_t>(kv.bt_width * kv.block_size, INT32_MAX);
    p.max_units = k.max_units;
    p.hdr = (int32_t*)(ws + w.hdr);
    p.row_base = (int32_t*)(ws + w.row_base);
    p.exec = (int2*)(ws + w.exec);
    p.err = a.err;
    rc = launch_decode_plan(p, s);
    if (rc) return rc;
  }
  switch (kv.dtype) {
    case BL_F32: return launch_all<float>(k, kv, s);
    case BL_F16: return launch_all<__half>(k, kv, s);
    default: return launch_all<__nv_bfloat16>(k, kv, s);
  }
}
