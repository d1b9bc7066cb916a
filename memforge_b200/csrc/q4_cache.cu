// The 4-bit KV cache's write and read: quantising scatter (mf_q4_reshape_and_cache)
// and dequantising gather (mf_q4_gather_kv).
//
// Write, per row x of D values (one token, kv head, K or V):
//   base  = largest fp16 <= min(x)
//   scale = smallest fp16 with 15 * scale >= max(x) - base
//   code  = (x - base) / scale, rounded to nearest even       (0 .. 15, no clamp)
// The definition is exact, so a code never depends on how it was computed: the
// quotient is formed in fp32 (error below 3e-6 for a quotient up to 15) and decided in fp64 only
// within 1e-4 of a half.  A row with a NaN or a magnitude above 65504 stores NaN
// parameters and reads back as NaN.
//
// Both are bound by memory traffic (the write by its 16- or 32-bit sources, the
// read by its outputs): D / 8 lanes own a row and move 16 bytes of it each.

#include "mf_q4.cuh"

namespace mf {
namespace {

template <typename S>
MF_DEVINL void load8(const S* p, bool vec, float* x) {
  if (vec) {
    if constexpr (sizeof(S) == 2) {
      const uint4 r = __ldg(reinterpret_cast<const uint4*>(p));
      const S* e = reinterpret_cast<const S*>(&r);
#pragma unroll
      for (int i = 0; i < 8; ++i) x[i] = Elt<S>::to_f32(e[i]);
    } else {
      const float4 a = __ldg(reinterpret_cast<const float4*>(p));
      const float4 b = __ldg(reinterpret_cast<const float4*>(p) + 1);
      x[0] = a.x, x[1] = a.y, x[2] = a.z, x[3] = a.w;
      x[4] = b.x, x[5] = b.y, x[6] = b.z, x[7] = b.w;
    }
  } else {
#pragma unroll
    for (int i = 0; i < 8; ++i) x[i] = Elt<S>::to_f32(p[i]);
  }
}

// The code of x: (x - base) / scale to nearest even.
MF_DEVINL uint32_t encode(float x, float base, float scale, float inv) {
  const float t = __fmul_rn(__fsub_rn(x, base), inv);
  const float lo = floorf(t);
  const float f = t - lo;
  uint32_t n = (uint32_t)lo + (f > 0.5f ? 1u : 0u);
  if (fabsf(f - 0.5f) < 1e-4f) {
    const double away = (double)x - (double)base;
    const double mid = ((double)lo + 0.5) * (double)scale;
    n = (uint32_t)lo + (away > mid || (away == mid && ((uint32_t)lo & 1u)) ? 1u : 0u);
  }
  return n;
}

template <typename S, int D>
__global__ void __launch_bounds__(256)
    q4_write_kernel(const S* __restrict__ key, const S* __restrict__ value, int64_t k_st,
                    int64_t k_sh, int64_t v_st, int64_t v_sh, uint8_t* __restrict__ pool,
                    int64_t sb, int64_t sh, int64_t num_slots, const void* __restrict__ slots,
                    int slots64, int num_tokens, int num_heads, bool vec, int32_t* err) {
  grid_launch_dependents();
  constexpr int LPR = D / 8;  // lanes per row
  constexpr int RPW = 32 / LPR;
  const int lane = threadIdx.x & 31, rl = lane % LPR;
  const int64_t rows = 2 * (int64_t)num_tokens * num_heads;
  const int64_t warps = (int64_t)gridDim.x * (blockDim.x >> 5);
  const int64_t w0 = blockIdx.x * (int64_t)(blockDim.x >> 5) + (threadIdx.x >> 5);
  for (int64_t r0 = w0 * RPW; r0 < rows; r0 += warps * RPW) {
    const int64_t r = r0 + lane / LPR;
    const bool have = r < rows;
    const bool is_v = have && r >= rows / 2;
    const int64_t th = have ? (is_v ? r - rows / 2 : r) : 0;
    const int h = (int)(th % num_heads), t = (int)(th / num_heads);
    int64_t slot = -1;
    if (have)
      slot = slots64 ? reinterpret_cast<const int64_t*>(slots)[t]
                     : (int64_t)reinterpret_cast<const int32_t*>(slots)[t];
    const bool live = slot >= 0 && slot < num_slots;
    if (have && !live && slot != -1 && h == 0 && rl == 0) set_err(err, MF_ERR_SLOT);
    float x[8];
    if (live) {
      load8(is_v ? value + t * v_st + h * v_sh + rl * 8 : key + t * k_st + h * k_sh + rl * 8, vec,
            x);
    } else {
#pragma unroll
      for (int i = 0; i < 8; ++i) x[i] = 0.f;
    }
    float lo = x[0], hi = x[0];
    bool fine = true;
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      lo = fminf(lo, x[i]);
      hi = fmaxf(hi, x[i]);
      fine = fine && fabsf(x[i]) <= 65504.f;  // false for NaN
    }
#pragma unroll
    for (int o = LPR / 2; o > 0; o >>= 1) {
      lo = fminf(lo, __shfl_xor_sync(0xffffffffu, lo, o));
      hi = fmaxf(hi, __shfl_xor_sync(0xffffffffu, hi, o));
    }
    const uint32_t bad = __ballot_sync(0xffffffffu, !fine);
    const uint32_t mine = LPR == 32 ? 0xffffffffu : ((1u << (LPR & 31)) - 1u) << (lane - rl);
    const bool row_ok = (bad & mine) == 0;
    if (!live) continue;  // no warp collective below

    uint32_t codes = 0;
    __half scale = __ushort_as_half((unsigned short)0x7E00), base = scale;
    if (row_ok) {
      base = __float2half_rd(lo);
      const float bf = __half2float(base);
      const double span = (double)hi - (double)bf;
      // Nearest fp16 to span / 15, then one step either way to the smallest that
      // covers the span (15 * scale is exact in fp32).
      unsigned short sbits = __half_as_ushort(__float2half_rn((float)span * (1.f / 15.f)));
      auto covers = [&](unsigned short b) {
        return (double)(15.f * __half2float(__ushort_as_half(b))) >= span;
      };
      if (!covers(sbits)) ++sbits;
      if (sbits > 0 && covers(sbits - 1)) --sbits;
      scale = __ushort_as_half(sbits);
      const float sf = __half2float(scale);
      if (sf > 0.f) {
        const float inv = __frcp_rn(sf);
#pragma unroll
        for (int i = 0; i < 8; ++i) codes |= encode(x[i], bf, sf, inv) << (4 * i);
      }
    }
    const int tok = (int)(slot % q4::BLOCK);
    uint8_t* rec = pool + (slot / q4::BLOCK) * sb + h * sh;
    if (!is_v) {
      *reinterpret_cast<uint32_t*>(rec + tok * (D / 2) + rl * 4) = codes;
    } else {
      *reinterpret_cast<uint16_t*>(rec + q4::v_piece<D>(tok, 2 * rl)) = (uint16_t)codes;
      *reinterpret_cast<uint16_t*>(rec + q4::v_piece<D>(tok, 2 * rl + 1)) = (uint16_t)(codes >> 16);
    }
    if (rl == 0)
      *reinterpret_cast<__half2*>(rec + 16 * D + (is_v ? 64 : 0) + tok * 4) =
          __halves2half2(scale, base);
  }
}

// Row order (K or V, head, token), tokens fastest: neighbouring rows of a context
// share a record and its sectors, and an output head's rows are written in a run.
template <typename S, int D>
__global__ void __launch_bounds__(256)
    q4_gather_kernel(const uint8_t* __restrict__ pool, int64_t sb, int64_t sh, int64_t num_slots,
                     const void* __restrict__ index, int index64, int num_tokens, int num_heads,
                     S* __restrict__ ko, S* __restrict__ vo, int64_t o_sh, int64_t o_st, bool vec,
                     int32_t* err) {
  grid_dependency_wait();
  constexpr int LPR = D / 8;
  const int64_t half = (int64_t)num_tokens * num_heads * LPR;
  for (int64_t i = blockIdx.x * (int64_t)blockDim.x + threadIdx.x; i < 2 * half;
       i += (int64_t)gridDim.x * blockDim.x) {
    const bool is_v = i >= half;
    const int64_t ii = is_v ? i - half : i;
    const int rl = (int)(ii % LPR);
    const int64_t ht = ii / LPR;
    const int t = (int)(ht % num_tokens), h = (int)(ht / num_tokens);
    const int64_t slot = index64 ? reinterpret_cast<const int64_t*>(index)[t]
                                 : (int64_t)reinterpret_cast<const int32_t*>(index)[t];
    float x[8];
    if (slot < 0 || slot >= num_slots) {
      if (h == 0 && rl == 0) set_err(err, MF_ERR_SLOT);
#pragma unroll
      for (int j = 0; j < 8; ++j) x[j] = 0.f;
    } else {
      const int tok = (int)(slot % q4::BLOCK);
      const uint8_t* rec = pool + (slot / q4::BLOCK) * sb + h * sh;
      uint32_t codes;
      if (!is_v) {
        codes = *reinterpret_cast<const uint32_t*>(rec + tok * (D / 2) + rl * 4);
      } else {
        codes = *reinterpret_cast<const uint16_t*>(rec + q4::v_piece<D>(tok, 2 * rl)) |
                (uint32_t)*reinterpret_cast<const uint16_t*>(rec + q4::v_piece<D>(tok, 2 * rl + 1))
                    << 16;
      }
      const float2 par = __half22float2(
          *reinterpret_cast<const __half2*>(rec + 16 * D + (is_v ? 64 : 0) + tok * 4));
#pragma unroll
      for (int j = 0; j < 8; ++j) x[j] = fmaf((float)((codes >> (4 * j)) & 15u), par.x, par.y);
    }
    S* dst = (is_v ? vo : ko) + h * o_sh + (int64_t)t * o_st + rl * 8;
    S e[8];
#pragma unroll
    for (int j = 0; j < 8; ++j) e[j] = from_f32<S>(x[j]);
    if (vec) {
#pragma unroll
      for (int j = 0; j < (int)sizeof(S) / 2; ++j)
        reinterpret_cast<uint4*>(dst)[j] = reinterpret_cast<const uint4*>(e)[j];
    } else {
#pragma unroll
      for (int j = 0; j < 8; ++j) dst[j] = e[j];
    }
  }
}

template <typename S>
bool rows_vec(const void* a, const void* b, int64_t s0, int64_t s1, int64_t s2, int64_t s3) {
  auto al = [](const void* p) { return (reinterpret_cast<uintptr_t>(p) & 15) == 0; };
  auto al16 = [](int64_t s) { return (s * (int64_t)sizeof(S)) % 16 == 0; };
  return al(a) && al(b) && al16(s0) && al16(s1) && al16(s2) && al16(s3);
}

int grid_of(int64_t threads) {
  const int64_t blocks = (threads + 255) / 256;
  const int64_t most = (int64_t)current_sm_count() * 32;
  return (int)(blocks < most ? blocks : most);
}

const char* pool_fault(const void* pool, int64_t sb, int64_t sh, int32_t num_blocks,
                       int32_t num_heads, int32_t d) {
  if (!q4::head_dim_ok(d)) return "head_dim must be 64, 128 or 256";
  if (num_blocks <= 0 || num_heads <= 0) return "non-positive block or head count";
  if ((reinterpret_cast<uintptr_t>(pool) | (uintptr_t)sb | (uintptr_t)sh) & 15)
    return "pool base and strides must be multiples of 16 bytes";
  return nullptr;
}

}  // namespace

template <typename S>
static int launch_write(const void* k, const void* v, int64_t kst, int64_t ksh, int64_t vst,
                        int64_t vsh, uint8_t* pool, int64_t sb, int64_t sh, int64_t num_slots,
                        const void* slots, int s64, int T, int H, int D, int32_t* err,
                        cudaStream_t stream) {
  const bool vec = rows_vec<S>(k, v, kst, ksh, vst, vsh);
  const int grid = grid_of(2 * (int64_t)T * H * (D / 8));
  auto go = [&](auto kern) {
    kern<<<grid, 256, 0, stream>>>(static_cast<const S*>(k), static_cast<const S*>(v), kst, ksh,
                                   vst, vsh, pool, sb, sh, num_slots, slots, s64, T, H, vec, err);
  };
  if (D == 64) go(q4_write_kernel<S, 64>);
  else if (D == 128) go(q4_write_kernel<S, 128>);
  else go(q4_write_kernel<S, 256>);
  return check_launch("q4 reshape_and_cache");
}

template <typename S>
static int launch_read(const uint8_t* pool, int64_t sb, int64_t sh, int64_t num_slots,
                       const void* index, int i64, int T, int H, int D, void* ko, void* vo,
                       int64_t osh, int64_t ost, int32_t* err, cudaStream_t stream) {
  const bool vec = rows_vec<S>(ko, vo, osh, ost, 0, 0);
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3((unsigned)grid_of(2 * (int64_t)T * H * (D / 8)));
  cfg.blockDim = dim3(256);
  cfg.stream = stream;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  auto kern = D == 64 ? q4_gather_kernel<S, 64>
                      : D == 128 ? q4_gather_kernel<S, 128> : q4_gather_kernel<S, 256>;
  const cudaError_t e = cudaLaunchKernelEx(&cfg, kern, pool, sb, sh, num_slots, index, i64, T, H,
                                           static_cast<S*>(ko), static_cast<S*>(vo), osh, ost, vec,
                                           err);
  if (e != cudaSuccess)
    return fail(MF_ECUDA, std::string("q4 gather_kv: ") + cudaGetErrorString(e));
  return check_launch("q4 gather_kv");
}

}  // namespace mf

using namespace mf;

extern "C" int64_t mf_q4_record_bytes(int32_t head_dim) {
  if (!q4::head_dim_ok(head_dim)) return fail(MF_EUNSUPPORTED, "q4: head_dim must be 64, 128 or 256");
  return q4::record_bytes(head_dim);
}

extern "C" int mf_q4_reshape_and_cache(const void* key, const void* value, mf_dtype src_dtype,
                                       int64_t k_stride_tok, int64_t k_stride_head,
                                       int64_t v_stride_tok, int64_t v_stride_head, void* pool,
                                       int64_t pool_stride_block, int64_t pool_stride_head,
                                       int32_t num_blocks, const void* slot_mapping,
                                       int32_t slot_mapping_is_int64, int32_t num_tokens,
                                       int32_t num_kv_heads, int32_t head_dim, int32_t* err_flag,
                                       mf_stream_t stream) {
  if (const char* why = pool_fault(pool, pool_stride_block, pool_stride_head, num_blocks,
                                   num_kv_heads, head_dim))
    return fail(MF_EINVAL, std::string("q4 reshape_and_cache: ") + why);
  if (num_tokens < 0) return fail(MF_EINVAL, "q4 reshape_and_cache: negative token count");
  if (num_tokens == 0) return MF_OK;
  if (!key || !value || !pool || !slot_mapping)
    return fail(MF_EINVAL, "q4 reshape_and_cache: null pointer");
  const int64_t num_slots = (int64_t)num_blocks * q4::BLOCK;
  cudaStream_t s = reinterpret_cast<cudaStream_t>(stream);
  auto* pl = static_cast<uint8_t*>(pool);
#define MF_Q4W(S)                                                                             \
  return launch_write<S>(key, value, k_stride_tok, k_stride_head, v_stride_tok, v_stride_head, \
                         pl, pool_stride_block, pool_stride_head, num_slots, slot_mapping,    \
                         slot_mapping_is_int64, num_tokens, num_kv_heads, head_dim, err_flag, s)
  switch (src_dtype) {
    case MF_F32: MF_Q4W(float);
    case MF_F16: MF_Q4W(__half);
    case MF_BF16: MF_Q4W(__nv_bfloat16);
  }
#undef MF_Q4W
  return fail(MF_EINVAL, "q4 reshape_and_cache: unknown dtype");
}

extern "C" int mf_q4_gather_kv(const void* pool, int64_t pool_stride_block,
                               int64_t pool_stride_head, int32_t num_blocks,
                               const void* flat_index, int32_t index_is_int64, int32_t num_tokens,
                               int32_t num_kv_heads, int32_t head_dim, void* key_out,
                               void* value_out, mf_dtype out_dtype, int64_t out_stride_head,
                               int64_t out_stride_tok, int32_t* err_flag, mf_stream_t stream) {
  if (const char* why = pool_fault(pool, pool_stride_block, pool_stride_head, num_blocks,
                                   num_kv_heads, head_dim))
    return fail(MF_EINVAL, std::string("q4 gather_kv: ") + why);
  if (num_tokens < 0) return fail(MF_EINVAL, "q4 gather_kv: negative token count");
  if (num_tokens == 0) return MF_OK;
  if (!pool || !flat_index || !key_out || !value_out)
    return fail(MF_EINVAL, "q4 gather_kv: null pointer");
  const int64_t num_slots = (int64_t)num_blocks * q4::BLOCK;
  cudaStream_t s = reinterpret_cast<cudaStream_t>(stream);
  auto* pl = static_cast<const uint8_t*>(pool);
#define MF_Q4R(S)                                                                            \
  return launch_read<S>(pl, pool_stride_block, pool_stride_head, num_slots, flat_index,      \
                        index_is_int64, num_tokens, num_kv_heads, head_dim, key_out, value_out, \
                        out_stride_head, out_stride_tok, err_flag, s)
  switch (out_dtype) {
    case MF_F32: MF_Q4R(float);
    case MF_F16: MF_Q4R(__half);
    case MF_BF16: MF_Q4R(__nv_bfloat16);
  }
#undef MF_Q4R
  return fail(MF_EINVAL, "q4 gather_kv: unknown dtype");
}
