// 8-bit paged cache: quantising append and dequantising gather.
//
// append   one warp per (row, touched block, KV head) and K or V.  The block's
//          new scale is S = max(scale of the tokens it holds already, the scale
//          its new tokens need); new tokens are stored as e4m3(x / S), and only
//          where S grew are the old codes moved to it.  A block belongs to one
//          warp of a call, so nothing is atomic and the result is the same
//          every time.  Counterpart of PagedLayerKV.append_only
//          (src/barellm/engine/paged_kv_cache.py:151-193).
// gather   dense code * scale in the caller's type, zeros behind each length.
//          Counterpart of PagedLayerKV.read (paged_kv_cache.py:215-240).
// Both are bound by HBM: append reads E bytes and writes 1 per element, gather
// reads 1 and writes E.  A call of a few tokens is bound by its launch and three
// dependent loads (row, table entry, tokens): 4.2 us for 4 rows of one token.
#include "fp8.cuh"

namespace bl {
namespace {

constexpr int kAppendWarps = 4;

struct AppendFp8Args {
  uint8_t* k_pool;
  uint8_t* v_pool;
  float* k_scale;
  float* v_scale;
  const char* k_new;
  const char* v_new;
  int64_t num_blocks, layer;
  int64_t ksb, ksh, kst, vsb, vsh, vst;  // strides of the new tokens, in elements
  const int32_t* block_tables;
  int64_t bt_stride, bt_width;
  const int32_t* row_ids;
  const int32_t* start_pos;
  const int32_t* new_offsets;
  int64_t max_new;
  int32_t hkv, bs, d;
  int32_t vpr_shift;  // log2 of a token's 16-byte vectors, or -1
  int32_t* err;
};

// 16 bytes of T as floats
template <typename T>
__device__ __forceinline__ void unpack16(const uint4& v, float* f) {
  if constexpr (sizeof(T) == 2) {
    const uint32_t w[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const float2 p = unpack2<T>(w[i]);
      f[2 * i] = p.x;
      f[2 * i + 1] = p.y;
    }
  } else {
    f[0] = __uint_as_float(v.x), f[1] = __uint_as_float(v.y), f[2] = __uint_as_float(v.z), f[3] = __uint_as_float(v.w);
  }
}

template <typename T>
__device__ __forceinline__ void store_codes(uint8_t* dst, const float* f, float inv) {
  if constexpr (sizeof(T) == 2) {
    uint2 c;
    c.x = pack_e4m3x4(f[0] * inv, f[1] * inv, f[2] * inv, f[3] * inv);
    c.y = pack_e4m3x4(f[4] * inv, f[5] * inv, f[6] * inv, f[7] * inv);
    *reinterpret_cast<uint2*>(dst) = c;
  } else {
    *reinterpret_cast<uint32_t*>(dst) = pack_e4m3x4(f[0] * inv, f[1] * inv, f[2] * inv, f[3] * inv);
  }
}

// The largest magnitude in a 16-byte vector as an integer that orders as the
// magnitudes do: the values' bits without the sign.  16-bit elements go two
// at a time (the result's halves are separate maxima).
template <typename T>
__device__ __forceinline__ uint32_t max_bits(uint32_t m, const uint4& v) {
  if constexpr (sizeof(T) == 2) {
    m = __vmaxu2(m, v.x & 0x7fff7fffu);
    m = __vmaxu2(m, v.y & 0x7fff7fffu);
    m = __vmaxu2(m, v.z & 0x7fff7fffu);
    return __vmaxu2(m, v.w & 0x7fff7fffu);
  } else {
    m = max(m, v.x & 0x7fffffffu);
    m = max(m, v.y & 0x7fffffffu);
    m = max(m, v.z & 0x7fffffffu);
    return max(m, v.w & 0x7fffffffu);
  }
}
// The magnitude that max_bits' result (joined over its halves) stands for;
// +inf or NaN where the vector holds one.
template <typename T> __device__ __forceinline__ float bits_to_magnitude(uint32_t m);
template <> __device__ __forceinline__ float bits_to_magnitude<float>(uint32_t m) { return __uint_as_float(m); }
template <> __device__ __forceinline__ float bits_to_magnitude<__nv_bfloat16>(uint32_t m) {
  return __uint_as_float(max(m & 0xffffu, m >> 16) << 16);
}
template <> __device__ __forceinline__ float bits_to_magnitude<__half>(uint32_t m) {
  return __half2float(__ushort_as_half((unsigned short)max(m & 0xffffu, m >> 16)));
}

// grid: (touched blocks, ceil(2 * hkv / kAppendWarps), batch)
// VEC: rows move as 16-byte vectors (head_dim a multiple of one, everything
// aligned); up to kHeld of them per lane stay in registers between the maximum
// and the store (a 16-token block of head_dim 128 fits), more are read twice.
// A warp per block and head, not per token: the block's scale needs all of its new
// tokens.  40k packed tokens (8 KV heads, head_dim 128, bf16, 247 MB): 47.4 us,
// 5.2 TB/s; with the tokens read twice 69.8 us.
template <typename T, bool VEC>
__global__ void __launch_bounds__(kAppendWarps * 32) append_fp8_kernel(const AppendFp8Args a) {
  pdl_trigger();  // a dependent launch (the decode plan) may start; it waits for this grid
  constexpr int E = VEC ? 16 / (int)sizeof(T) : 1;  // elements per vector
  constexpr int kHeld = VEC ? (sizeof(T) == 2 ? 8 : 16) : 1;
  const int lane = threadIdx.x & 31;
  const int unit = blockIdx.y * kAppendWarps + (threadIdx.x >> 5);
  if (unit >= 2 * a.hkv) return;
  const int h = unit >> 1;
  const bool is_v = unit & 1;
  const int64_t b = blockIdx.z;
  int64_t off = 0, n = a.max_new;
  if (a.new_offsets) {
    off = a.new_offsets[b];
    n = (int64_t)a.new_offsets[b + 1] - off;
  }
  const int64_t start = a.start_pos[b];
  if (start < 0) {
    if (lane == 0) raise_dev(a.err, BL_DEVERR_TABLE);
    return;
  }
  const int64_t lb = start / a.bs + blockIdx.x;
  const int64_t p0 = max(start, lb * a.bs), p1 = min(start + n, (lb + 1) * a.bs);
  if (p0 >= p1) return;
  const int64_t st = is_v ? a.vst : a.kst;
  const T* src = reinterpret_cast<const T*>(is_v ? a.v_new : a.k_new) + b * (is_v ? a.vsb : a.ksb) +
                 (int64_t)h * (is_v ? a.vsh : a.ksh) + (off + p0 - start) * st;
  const int vpr = a.d / E;                  // vectors per token
  const int total = (int)(p1 - p0) * vpr;  // block_size * head_dim <= 2^24
  auto token_of = [&](int idx) { return a.vpr_shift >= 0 ? idx >> a.vpr_shift : idx / vpr; };
  auto vector_at = [&](int idx) {
    const int t = token_of(idx);
    return src + t * st + (idx - t * vpr) * E;
  };
  // the tokens are on their way while the block is looked up
  uint4 held[kHeld];
  const bool fits = VEC && total <= kHeld * 32;
  if (fits) {
#pragma unroll
    for (int i = 0; i < kHeld; ++i) {
      const int idx = lane + 32 * i;
      held[i] = make_uint4(0, 0, 0, 0);
      if (idx < total) held[i] = *reinterpret_cast<const uint4*>(vector_at(idx));
    }
  }
  if (lb >= a.bt_width) {
    if (lane == 0) raise_dev(a.err, BL_DEVERR_TABLE);
    return;
  }
  const int64_t row = a.row_ids ? (int64_t)a.row_ids[b] : b;
  const int64_t phys = a.block_tables[row * a.bt_stride + lb];
  if (phys < 0 || phys >= a.num_blocks) {
    if (lane == 0) raise_dev(a.err, BL_DEVERR_BLOCK_ID);
    return;
  }
  const int64_t slot = (a.layer * a.num_blocks + phys) * a.hkv + h;
  uint8_t* page = (is_v ? a.v_pool : a.k_pool) + slot * a.bs * a.d;
  float* scale_p = (is_v ? a.v_scale : a.k_scale) + slot;
  const int kept = (int)(p0 - lb * a.bs);  // tokens the block holds already
  const float old_scale = kept > 0 ? *scale_p : 0.f;
  uint8_t* dst = page + (int64_t)kept * a.d;

  // largest finite magnitude of the new tokens
  float amax = 0.f;
  if constexpr (VEC) {
    uint32_t bits = 0;
    if (fits) {
#pragma unroll
      for (int i = 0; i < kHeld; ++i) bits = max_bits<T>(bits, held[i]);
    } else {
#pragma unroll 4
      for (int idx = lane; idx < total; idx += 32) bits = max_bits<T>(bits, *reinterpret_cast<const uint4*>(vector_at(idx)));
    }
    amax = bits_to_magnitude<T>(bits);
    if (__any_sync(0xffffffffu, !(amax < INFINITY))) {
      // an infinity or a NaN among the tokens: again, leaving those out
      amax = 0.f;
      for (int idx = lane; idx < total; idx += 32) {
        float f[8];
        unpack16<T>(*reinterpret_cast<const uint4*>(vector_at(idx)), f);
#pragma unroll
        for (int e = 0; e < E; ++e) amax = fmaxf(amax, finite_abs(f[e]));
      }
    }
  } else {
    for (int idx = lane; idx < total; idx += 32) amax = fmaxf(amax, finite_abs(to_f32<T>(*vector_at(idx))));
  }
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) amax = fmaxf(amax, __shfl_xor_sync(0xffffffffu, amax, o));
  const float need = exp2_int(scale_exponent(amax));
  const float scale = fmaxf(need, old_scale);

  // old codes move to the larger scale (a power-of-two ratio, <= 1)
  if (kept > 0 && scale > old_scale) {
    const float ratio = old_scale * pow2_inverse(scale);
    const int bytes = kept * a.d;
    int done = 0;
    if (((uintptr_t)page & 3) == 0) {
      done = bytes & ~3;
      for (int i = lane * 4; i < done; i += 128) {
        const uint32_t w = *reinterpret_cast<const uint32_t*>(page + i);
        const float2 x = e4m3x2_to_float2((uint16_t)w), y = e4m3x2_to_float2((uint16_t)(w >> 16));
        *reinterpret_cast<uint32_t*>(page + i) = pack_e4m3x4(x.x * ratio, x.y * ratio, y.x * ratio, y.y * ratio);
      }
    }
    for (int i = done + lane; i < bytes; i += 32)
      page[i] = (uint8_t)pack_e4m3x2(e4m3_to_float(page[i]) * ratio, 0.f);
  }
  if (lane == 0 && scale != old_scale) *scale_p = scale;

  const float inv = pow2_inverse(scale);
  if (fits) {
#pragma unroll
    for (int i = 0; i < kHeld; ++i) {
      const int idx = lane + 32 * i;
      if (idx < total) {
        float f[8];
        unpack16<T>(held[i], f);
        store_codes<T>(dst + idx * E, f, inv);
      }
    }
  } else {
    for (int idx = lane; idx < total; idx += 32) {
      const T* p = vector_at(idx);
      if constexpr (VEC) {
        float f[8];
        unpack16<T>(*reinterpret_cast<const uint4*>(p), f);
        store_codes<T>(dst + idx * E, f, inv);
      } else {
        dst[idx] = (uint8_t)pack_e4m3x2(to_f32<T>(*p) * inv, 0.f);
      }
    }
  }
}

struct GatherFp8Args {
  const uint8_t* k_pool;
  const uint8_t* v_pool;
  const float* k_scale;
  const float* v_scale;
  char* k_out;
  char* v_out;
  int64_t num_blocks, layer;
  int64_t osb, osh, ost;  // elements
  const int32_t* block_tables;
  int64_t bt_stride, bt_width;
  const int32_t* row_ids;
  const int32_t* seq_lens;
  int64_t max_len;
  int32_t hkv, bs, bs_shift, d, nvec, zero_fill;
  int32_t* err;
};

// E consecutive codes
template <int E> struct CodesT;
template <> struct CodesT<8> { using type = uint2; };
template <> struct CodesT<4> { using type = uint32_t; };
template <> struct CodesT<1> { using type = uint8_t; };
template <int E> using Codes = typename CodesT<E>::type;

// E codes times scale, as one store of E elements of T
template <typename T, int E>
__device__ __forceinline__ void dequant_store(T* dst, const Codes<E>& c, float scale) {
  if constexpr (E == 1) {
    *dst = dequant_to<T>(e4m3_to_float(c) * scale);
  } else {
    float f[E];
    uint32_t w[E / 4];
    if constexpr (E == 8)
      w[0] = c.x, w[1] = c.y;
    else
      w[0] = c;
#pragma unroll
    for (int i = 0; i < E / 4; ++i) {
      const float2 x = unpack2<__half>(e4m3lo_to_f16x2(w[i])), y = unpack2<__half>(e4m3hi_to_f16x2(w[i]));
      f[4 * i] = x.x * scale, f[4 * i + 1] = x.y * scale, f[4 * i + 2] = y.x * scale, f[4 * i + 3] = y.y * scale;
    }
    union {
      T t[E];
      uint4 u;
    } o;
#pragma unroll
    for (int i = 0; i < E; ++i) o.t[i] = dequant_to<T>(f[i]);
    *reinterpret_cast<uint4*>(dst) = o.u;
  }
}

template <typename T, int E>
__device__ __forceinline__ void zero_store(T* dst) {
  if constexpr (E == 1)
    *dst = from_f32<T>(0.f);
  else
    *reinterpret_cast<uint4*>(dst) = make_uint4(0, 0, 0, 0);
}

constexpr int kGatherTok = 2;  // tokens of a thread: their loads are in flight together

// grid: (ceil(max_len / (kGatherTok * blockDim.y)), hkv, batch); threadIdx.x walks the
// vectors of a token, threadIdx.y the tokens.  64 rows of up to 4k tokens (8 KV
// heads, head_dim 128, bf16, 1.35 GB): 215 us, 6.28 TB/s; one token a thread 236 us.
template <typename T, int E>
__global__ void __launch_bounds__(256) gather_fp8_kernel(const GatherFp8Args a) {
  const int64_t b = blockIdx.z;
  const int h = blockIdx.y;
  const int64_t t0 = (int64_t)blockIdx.x * (kGatherTok * blockDim.y) + threadIdx.y;
  const int64_t len = a.seq_lens[b];
  const int64_t row = a.row_ids ? (int64_t)a.row_ids[b] : b;
  T* ko = reinterpret_cast<T*>(a.k_out) + b * a.osb + h * a.osh;
  T* vo = reinterpret_cast<T*>(a.v_out) + b * a.osb + h * a.osh;
  int64_t src[kGatherTok];
  float ks[kGatherTok], vs[kGatherTok];
#pragma unroll
  for (int i = 0; i < kGatherTok; ++i) {
    const int64_t t = t0 + i * blockDim.y;
    src[i] = -1;
    if (t >= len || t >= a.max_len) continue;
    const int64_t lb = a.bs_shift >= 0 ? t >> a.bs_shift : t / a.bs;
    if (lb >= a.bt_width) {
      raise_dev(a.err, BL_DEVERR_TABLE);
      src[i] = -2;
      continue;
    }
    const int64_t phys = a.block_tables[row * a.bt_stride + lb];
    if (phys < 0 || phys >= a.num_blocks) {
      raise_dev(a.err, BL_DEVERR_BLOCK_ID);
      src[i] = -2;
      continue;
    }
    const int64_t slot = (a.layer * a.num_blocks + phys) * a.hkv + h;
    src[i] = (slot * a.bs + (t - lb * a.bs)) * a.d;
    ks[i] = a.k_scale[slot];
    vs[i] = a.v_scale[slot];
  }
  for (int v = threadIdx.x; v < a.nvec; v += blockDim.x) {
    Codes<E> kc[kGatherTok], vc[kGatherTok];
#pragma unroll
    for (int i = 0; i < kGatherTok; ++i)
      if (src[i] >= 0) {
        kc[i] = *reinterpret_cast<const Codes<E>*>(a.k_pool + src[i] + v * E);
        vc[i] = *reinterpret_cast<const Codes<E>*>(a.v_pool + src[i] + v * E);
      }
#pragma unroll
    for (int i = 0; i < kGatherTok; ++i) {
      const int64_t t = t0 + i * blockDim.y;
      if (t >= a.max_len) break;
      if (src[i] >= 0) {
        dequant_store<T, E>(ko + t * a.ost + v * E, kc[i], ks[i]);
        dequant_store<T, E>(vo + t * a.ost + v * E, vc[i], vs[i]);
      } else if (src[i] == -1 && a.zero_fill) {
        zero_store<T, E>(ko + t * a.ost + v * E);
        zero_store<T, E>(vo + t * a.ost + v * E);
      }
    }
  }
}

template <typename T>
int launch_append(const AppendFp8Args& k, bool vec, dim3 grid, cudaStream_t s) {
  if (vec)
    append_fp8_kernel<T, true><<<grid, kAppendWarps * 32, 0, s>>>(k);
  else
    append_fp8_kernel<T, false><<<grid, kAppendWarps * 32, 0, s>>>(k);
  BL_CHECK_LAUNCH("append_fp8_kernel");
  return BL_OK;
}

template <typename T>
int launch_gather(GatherFp8Args k, bool vec, int64_t batch, cudaStream_t s) {
  constexpr int E = 16 / (int)sizeof(T);
  k.nvec = vec ? k.d / E : k.d;
  const int bx = std::min(k.nvec, 256);
  const int by = 256 / bx;
  const int64_t gx = (k.max_len + kGatherTok * by - 1) / (kGatherTok * by);
  dim3 grid((unsigned)gx, (unsigned)k.hkv, (unsigned)batch), block((unsigned)bx, (unsigned)by);
  if (vec)
    gather_fp8_kernel<T, E><<<grid, block, 0, s>>>(k);
  else
    gather_fp8_kernel<T, 1><<<grid, block, 0, s>>>(k);
  BL_CHECK_LAUNCH("gather_fp8_kernel");
  return BL_OK;
}

}  // namespace
}  // namespace bl

using namespace bl;

extern "C" int bl_paged_append_fp8(const bl_append_fp8_args* args, void* stream) {
  BL_CHECK_ARG(args != nullptr, "bl_paged_append_fp8: args is null");
  const bl_append_fp8_args& a = *args;
  const int rc = check_fp8_layer(a.layer, "bl_paged_append_fp8");
  if (rc) return rc;
  const bl_paged_layer& kv = a.layer.kv;
  BL_CHECK_ARG(a.k_new && a.v_new && a.start_pos, "bl_paged_append_fp8: null input pointer");
  BL_CHECK_ARG(a.batch > 0 && a.batch <= 65535, "bl_paged_append_fp8: batch must be in [1, 65535]");
  BL_CHECK_ARG(a.max_new_tokens > 0, "K/V sequence length must be greater than zero");
  BL_CHECK_ARG(a.max_new_tokens <= INT32_MAX, "bl_paged_append_fp8: too many new tokens");
  const int es = elem_size(kv.dtype);
  BL_CHECK_ARG(((uintptr_t)a.k_new % es) == 0 && ((uintptr_t)a.v_new % es) == 0,
               "bl_paged_append_fp8: K/V must be aligned to their element type");
  AppendFp8Args k;
  k.k_pool = (uint8_t*)kv.k_pool;
  k.v_pool = (uint8_t*)kv.v_pool;
  k.k_scale = a.layer.k_scale;
  k.v_scale = a.layer.v_scale;
  k.k_new = (const char*)a.k_new;
  k.v_new = (const char*)a.v_new;
  k.num_blocks = kv.num_blocks;
  k.layer = kv.layer;
  k.ksb = a.new_stride_b, k.ksh = a.new_stride_h, k.kst = a.new_stride_t;
  k.vsb = a.v_stride_b, k.vsh = a.v_stride_h, k.vst = a.v_stride_t;
  k.block_tables = kv.block_tables;
  k.bt_stride = kv.bt_stride;
  k.bt_width = kv.bt_width;
  k.row_ids = kv.row_ids;
  k.start_pos = a.start_pos;
  k.new_offsets = a.new_offsets;
  k.max_new = a.max_new_tokens;
  k.hkv = (int32_t)kv.num_kv_heads;
  k.bs = (int32_t)kv.block_size;
  k.d = (int32_t)kv.head_dim;
  k.err = a.err;
  const int E = 16 / es;
  bool vec = kv.head_dim % E == 0 && ((uintptr_t)a.k_new & 15) == 0 && ((uintptr_t)a.v_new & 15) == 0;
  for (int64_t st : {k.ksb, k.ksh, k.kst, k.vsb, k.vsh, k.vst}) vec = vec && st % E == 0;
  k.vpr_shift = -1;
  for (int i = 0; i < 8; ++i)
    if (vec && kv.head_dim / E == 1 << i) k.vpr_shift = i;
  // blocks that n tokens can touch, from any offset in a block
  const int64_t touched = (a.max_new_tokens + kv.block_size - 2) / kv.block_size + 1;
  dim3 grid((unsigned)touched, (unsigned)((2 * k.hkv + kAppendWarps - 1) / kAppendWarps), (unsigned)a.batch);
  cudaStream_t s = (cudaStream_t)stream;
  switch (kv.dtype) {
    case BL_F32: return launch_append<float>(k, vec, grid, s);
    case BL_F16: return launch_append<__half>(k, vec, grid, s);
    default: return launch_append<__nv_bfloat16>(k, vec, grid, s);
  }
}

extern "C" int bl_paged_gather_fp8(const bl_gather_fp8_args* args, void* stream) {
  BL_CHECK_ARG(args != nullptr, "bl_paged_gather_fp8: args is null");
  const bl_gather_fp8_args& a = *args;
  const int rc = check_fp8_layer(a.layer, "bl_paged_gather_fp8");
  if (rc) return rc;
  const bl_paged_layer& kv = a.layer.kv;
  BL_CHECK_ARG(a.k_out && a.v_out && a.seq_lens, "bl_paged_gather_fp8: null pointer");
  BL_CHECK_ARG(a.batch > 0 && a.batch <= 65535, "bl_paged_gather_fp8: batch must be in [1, 65535]");
  BL_CHECK_ARG(a.max_len > 0, "KV cache is empty");
  BL_CHECK_ARG(a.max_len <= INT32_MAX, "bl_paged_gather_fp8: max_len too large");
  const int es = elem_size(kv.dtype);
  BL_CHECK_ARG(((uintptr_t)a.k_out % es) == 0 && ((uintptr_t)a.v_out % es) == 0,
               "bl_paged_gather_fp8: outputs must be aligned to their element type");
  GatherFp8Args k;
  k.k_pool = (const uint8_t*)kv.k_pool;
  k.v_pool = (const uint8_t*)kv.v_pool;
  k.k_scale = a.layer.k_scale;
  k.v_scale = a.layer.v_scale;
  k.k_out = (char*)a.k_out;
  k.v_out = (char*)a.v_out;
  k.num_blocks = kv.num_blocks;
  k.layer = kv.layer;
  k.osb = a.out_stride_b, k.osh = a.out_stride_h, k.ost = a.out_stride_t;
  k.block_tables = kv.block_tables;
  k.bt_stride = kv.bt_stride;
  k.bt_width = kv.bt_width;
  k.row_ids = kv.row_ids;
  k.seq_lens = a.seq_lens;
  k.max_len = a.max_len;
  k.hkv = (int32_t)kv.num_kv_heads;
  k.bs = (int32_t)kv.block_size;
  k.d = (int32_t)kv.head_dim;
  k.nvec = 0;
  k.bs_shift = -1;
  for (int i = 0; i < 17; ++i)
    if (kv.block_size == (int64_t)1 << i) k.bs_shift = i;
  k.zero_fill = a.zero_fill;
  k.err = a.err;
  const int E = 16 / es;
  const bool vec = kv.head_dim % E == 0 && ((uintptr_t)a.k_out & 15) == 0 && ((uintptr_t)a.v_out & 15) == 0 &&
                   k.osb % E == 0 && k.osh % E == 0 && k.ost % E == 0;
  cudaStream_t s = (cudaStream_t)stream;
  switch (kv.dtype) {
    case BL_F32: return launch_gather<float>(k, vec, a.batch, s);
    case BL_F16: return launch_gather<__half>(k, vec, a.batch, s);
    default: return launch_gather<__nv_bfloat16>(k, vec, a.batch, s);
  }
}
