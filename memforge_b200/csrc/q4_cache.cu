// The 4-bit KV cache's write and read: quantising scatter (mf_q4_reshape_and_cache)
// and dequantising gather (mf_q4_gather_kv).
//
// Write, per row x of D values (one token, kv head, K or V):
//   base  = largest fp16 <= min(x)
//   scale = smallest fp16 with 15 * scale >= max(x) - base
//   code  = (x - base) / scale, rounded to nearest even       (0 .. 15, no clamp)
// The definition is exact, so a code never depends on how it was computed: the quotient is
// formed in fp32 (error below 3e-6 for a quotient up to 15), and within 1e-5 of a half, as the
// scale's condition, decided on error-free fp32 differences.  A row
// with a NaN or a magnitude above 65504 stores NaN parameters and reads back as NaN.
//
// D / 16 lanes own a row, 16 values each.  The bytes would allow 13 us each way for 16004
// tokens of 8 heads, and arithmetic is what binds: wide lanes share a row's parameters,
// addresses and shuffles among more values (8 a lane took a third more), packed minima
// and maxima of 16-bit sources (a maximum and a negated minimum share a register for the
// shuffles), codes rounded and gathered by one multiply-add each, no 64-bit divisions.

#include "mf_q4.cuh"

namespace mf {
namespace {

// max / min of pairs; max keeps a NaN.
template <typename S> MF_DEVINL uint32_t max2_nan(uint32_t a, uint32_t b) {
  uint32_t r;
  if constexpr (std::is_same<S, __half>::value)
    asm("max.NaN.f16x2 %0, %1, %2;" : "=r"(r) : "r"(a), "r"(b));
  else
    asm("max.NaN.bf16x2 %0, %1, %2;" : "=r"(r) : "r"(a), "r"(b));
  return r;
}
template <typename S> MF_DEVINL uint32_t min2(uint32_t a, uint32_t b) {
  uint32_t r;
  if constexpr (std::is_same<S, __half>::value)
    asm("min.f16x2 %0, %1, %2;" : "=r"(r) : "r"(a), "r"(b));
  else
    asm("min.bf16x2 %0, %1, %2;" : "=r"(r) : "r"(a), "r"(b));
  return r;
}
MF_DEVINL float max_nan(float a, float b) {
  float r;
  asm("max.NaN.f32 %0, %1, %2;" : "=f"(r) : "f"(a), "f"(b));
  return r;
}

constexpr int E = 16;  // values of a row per lane

// A lane's source values, and the row's largest and smallest value (over LPR lanes; a NaN
// comes out in hi).
template <typename S, int LPR>
struct RowPart {
  static constexpr int NW = E * sizeof(S) / 4;
  uint32_t raw[NW];  // words of 16-bit pairs, or fp32

  MF_DEVINL float at(int i) const {
    if constexpr (sizeof(S) == 4) return __uint_as_float(raw[i]);
    else return Elt<S>::to_f32(reinterpret_cast<const S*>(raw)[i]);
  }
  MF_DEVINL void load(const S* p, bool live, bool vec) {
#pragma unroll
    for (int i = 0; i < NW; ++i) raw[i] = 0;
    if (!live) return;
    if (vec) {
#pragma unroll
      for (int v = 0; v < NW / 4; ++v) {
        const uint4 r = __ldg(reinterpret_cast<const uint4*>(p) + v);
        raw[4 * v] = r.x, raw[4 * v + 1] = r.y, raw[4 * v + 2] = r.z, raw[4 * v + 3] = r.w;
      }
    } else if constexpr (sizeof(S) == 2) {
      const uint16_t* e = reinterpret_cast<const uint16_t*>(p);
#pragma unroll
      for (int i = 0; i < NW; ++i) raw[i] = e[2 * i] | (uint32_t)e[2 * i + 1] << 16;
    } else {
#pragma unroll
      for (int i = 0; i < NW; ++i) raw[i] = __float_as_uint(p[i]);
    }
  }
};

// The largest and smallest value of K's row in even lanes and of V's in odd ones (a NaN comes
// out in hi): the first exchange of the reduction parts the two, so they share the rest.
template <typename S, int LPR>
MF_DEVINL void ranges(const RowPart<S, LPR>& k, const RowPart<S, LPR>& v, float& hi, float& lo) {
  const bool odd = threadIdx.x & 1;
  if constexpr (sizeof(S) == 2) {
    // (maximum, negated minimum) of a row's part in one register
    auto part = [](const RowPart<S, LPR>& r) {
      uint32_t mx = r.raw[0], mn = r.raw[0];
#pragma unroll
      for (int i = 1; i < RowPart<S, LPR>::NW; ++i) {
        mx = max2_nan<S>(mx, r.raw[i]);
        mn = min2<S>(mn, r.raw[i]);
      }
      mn ^= 0x80008000u;
      return max2_nan<S>(__byte_perm(mx, mn, 0x5410), __byte_perm(mx, mn, 0x7632));
    };
    const uint32_t pk = part(k), pv = part(v);
    uint32_t m = max2_nan<S>(odd ? pv : pk, __shfl_xor_sync(0xffffffffu, odd ? pk : pv, 1));
#pragma unroll
    for (int o = 2; o < LPR; o <<= 1) m = max2_nan<S>(m, __shfl_xor_sync(0xffffffffu, m, o));
    const S* t = reinterpret_cast<const S*>(&m);
    hi = Elt<S>::to_f32(t[0]);
    lo = -Elt<S>::to_f32(t[1]);
  } else {
    float h[2], l[2];
#pragma unroll
    for (int w = 0; w < 2; ++w) {
      const RowPart<S, LPR>& r = w ? v : k;
      h[w] = l[w] = r.at(0);
#pragma unroll
      for (int i = 1; i < E; ++i) h[w] = max_nan(h[w], r.at(i)), l[w] = fminf(l[w], r.at(i));
    }
    hi = max_nan(odd ? h[1] : h[0], __shfl_xor_sync(0xffffffffu, odd ? h[0] : h[1], 1));
    lo = fminf(odd ? l[1] : l[0], __shfl_xor_sync(0xffffffffu, odd ? l[0] : l[1], 1));
#pragma unroll
    for (int o = 2; o < LPR; o <<= 1) {
      hi = max_nan(hi, __shfl_xor_sync(0xffffffffu, hi, o));
      lo = fminf(lo, __shfl_xor_sync(0xffffffffu, lo, o));
    }
  }
}

// Scale and base of a row with values lo .. hi.
MF_DEVINL __half2 row_params(float hi, float lo) {
  const __half base = __float2half_rd(lo);
  const float bf = __half2float(base);
  // span = hi - base = s + e exactly (two-sum)
  const float s = hi - bf, bb = s - hi;
  const float e = (hi - (s - bb)) + (-bf - bb);
  // The nearest fp16 to span / 15 is at most one step from the smallest that covers it
  // (15 * scale and its difference from s are exact in fp32).
  unsigned short bits = __half_as_ushort(__float2half_rn(s * (1.f / 15.f)));
  auto covers = [&](unsigned short b) {
    return 15.f * __half2float(__ushort_as_half(b)) - s >= e;
  };
  if (!covers(bits)) ++bits;
  if (bits > 0 && covers(bits - 1)) --bits;
  return __halves2half2(__ushort_as_half(bits), base);
}

// A lane's codes, eight in a word: (x - base) / scale to nearest even.
template <typename R>
MF_DEVINL void encode(const R& x, float base, float scale, uint32_t* codes) {
  constexpr float MAGIC = 12582912.f;  // 1.5 * 2^23: a sum's low bits are the rounded quotient
  codes[0] = codes[1] = 0;
  if (!(scale > 0.f)) return;
  const float inv = __frcp_rn(scale);
  const uint64_t inv2 = f32x2(inv, inv), neg_base = f32x2(-base, -base), magic = f32x2(MAGIC, MAGIC),
                 minus = f32x2(-1.f, -1.f);
  float far = 0.f;
#pragma unroll
  for (int i = 0; i < E; i += 2) {
    const uint64_t d = f32x2_add(f32x2(x.at(i), x.at(i + 1)), neg_base);
    const uint64_t t = f32x2_fma(d, inv2, magic);
    float r0, r1, t0, t1;  // quotient less its rounding
    f32x2_split(f32x2_fma(d, inv2, f32x2_fma(t, minus, magic)), r0, r1);
    far = fmax3f(far, fabsf(r0), fabsf(r1));
    f32x2_split(t, t0, t1);
    codes[i / 8] += (__float_as_uint(t0) << (4 * (i % 8))) + (__float_as_uint(t1) << (4 * (i % 8) + 4));
  }
  uint32_t magic_bits = 0;
#pragma unroll
  for (int i = 0; i < 8; ++i) magic_bits += 0x4B400000u << (4 * i);
  codes[0] -= magic_bits;
  codes[1] -= magic_bits;
  if (far > 0.49999f) {
    // Some quotient is near a half (in bf16 sources one in a thousand is exactly one):
    // decide all exactly.  x - base = d + e without error (two-sum); (lo + 1/2) * scale has 16
    // bits, so d less it is exact where they are close, and e only decides where they agree.
    codes[0] = codes[1] = 0;
#pragma unroll
    for (int i = 0; i < E; ++i) {
      const float v = x.at(i), d = v - base, bb = d - v;
      const float e = (v - (d - bb)) + (-base - bb);
      const float n = rintf(d * inv);  // at most one off, and only near a half
      const float lo = fmaf(d, inv, -n) < 0.f ? n - 1.f : n;
      const float g = (d - (lo + 0.5f) * scale) + e;
      const uint32_t l = (uint32_t)(int)lo;
      codes[i / 8] |= (l + (g > 0.f || (g == 0.f && (l & 1u)) ? 1u : 0u)) << (4 * (i % 8));
    }
  }
}

// One token of head blockIdx.y per group of D / 16 lanes: its K row and its V row.  V's two
// tokens of a word are usually written together (a prompt's slots follow one another): the
// lanes of such a pair trade halves and store whole words, where 2-byte stores of one token
// each took four times the store transactions (40 us for 16004 tokens of 8 heads).
template <typename S, int D>
__global__ void __launch_bounds__(256)
    q4_write_kernel(const S* __restrict__ key, const S* __restrict__ value, int64_t k_st,
                    int64_t k_sh, int64_t v_st, int64_t v_sh, uint8_t* __restrict__ pool,
                    int64_t sb, int64_t sh, int64_t num_slots, const void* __restrict__ slots,
                    int slots64, int num_tokens, bool vec, int32_t* err) {
  grid_launch_dependents();
  constexpr int LPR = D / E, RPW = 32 / LPR;
  const int lane = threadIdx.x & 31, rl = lane % LPR, h = blockIdx.y;
  const int t = (blockIdx.x * 8 + (threadIdx.x >> 5)) * RPW + lane / LPR;
  int64_t slot = -1;
  if (t < num_tokens)
    slot = slots64 ? __ldg(reinterpret_cast<const long long*>(slots) + t)
                   : (int64_t)__ldg(reinterpret_cast<const int32_t*>(slots) + t);
  const bool live = slot >= 0 && slot < num_slots;
  if (!live && slot != -1 && h == 0 && rl == 0) set_err(err, MF_ERR_SLOT);
  RowPart<S, LPR> row[2];
  row[0].load(key + (live ? t * k_st + h * k_sh + rl * E : 0), live, vec);
  row[1].load(value + (live ? t * v_st + h * v_sh + rl * E : 0), live, vec);
  const int tok = (int)(slot & (q4::BLOCK - 1));
  uint8_t* rec = pool + (live ? (slot / q4::BLOCK) * sb + h * sh : 0);
  float hi, lo;
  ranges(row[0], row[1], hi, lo);
  uint32_t par = 0x7E007E00u;  // even lanes: K's, odd ones: V's
  if (hi <= 65504.f && lo >= -65504.f) {  // false with a NaN
    const __half2 p = row_params(hi, lo);
    par = *reinterpret_cast<const uint32_t*>(&p);
  }
  if (live && rl < 2) *reinterpret_cast<uint32_t*>(rec + 16 * D + rl * 64 + tok * 4) = par;
  uint32_t codes[2][2];
#pragma unroll
  for (int v = 0; v < 2; ++v) {
    const uint32_t mine = __shfl_sync(0xffffffffu, par, (lane & ~1) | v);
    const float2 f = __half22float2(*reinterpret_cast<const __half2*>(&mine));
    encode(row[v], f.y, f.x, codes[v]);  // (codes of a NaN row are 0)
  }
  const bool odd = tok & 1;
  const long long other = __shfl_xor_sync(0xffffffffu, (long long)slot, LPR);
  const uint32_t got = __shfl_xor_sync(0xffffffffu, codes[1][odd ? 0 : 1], LPR);
  if (!live) return;
  *reinterpret_cast<uint2*>(rec + tok * (D / 2) + rl * 8) = make_uint2(codes[0][0], codes[0][1]);
  if (other == (slot ^ 1)) {  // both tokens of the words: even stores the first two, odd the rest
    const uint32_t even_c = odd ? got : codes[1][0], odd_c = odd ? codes[1][1] : got;
    *reinterpret_cast<uint2*>(rec + (q4::v_piece<D>(tok, 4 * rl + (odd ? 2 : 0)) & ~3)) =
        make_uint2(__byte_perm(even_c, odd_c, 0x5410), __byte_perm(even_c, odd_c, 0x7632));
  } else {
#pragma unroll
    for (int w = 0; w < 2; ++w) {
      uint8_t* at = rec + q4::v_piece<D>(tok, 4 * rl + 2 * w);  // and the next word
      *reinterpret_cast<uint16_t*>(at) = (uint16_t)codes[1][w];
      *reinterpret_cast<uint16_t*>(at + 4) = (uint16_t)(codes[1][w] >> 16);
    }
  }
}

// Blocks of 64 tokens (x) of one head (y), K or V (z): neighbouring rows of a context share a
// record and its sectors, and an output head's rows are written in a run.
template <typename S, int D>
__global__ void __launch_bounds__(256)
    q4_gather_kernel(const uint8_t* __restrict__ pool, int64_t sb, int64_t sh, int64_t num_slots,
                     const void* __restrict__ index, int index64, int num_tokens,
                     S* __restrict__ ko, S* __restrict__ vo, int64_t o_sh, int64_t o_st, bool vec,
                     int32_t* err) {
  grid_dependency_wait();
  constexpr int LPR = D / E, ROWS = 256 / LPR, PASSES = 64 / ROWS < 1 ? 1 : 64 / ROWS;
  constexpr int TOKENS = ROWS * PASSES;
  const int rl = threadIdx.x % LPR;
  const bool is_v = blockIdx.z != 0;
  const uint8_t* head = pool + blockIdx.y * sh;
  S* out = (is_v ? vo : ko) + blockIdx.y * o_sh + rl * E;
  uint32_t codes[PASSES][2], par[PASSES];
#pragma unroll
  for (int u = 0; u < PASSES; ++u) {
    const int t = blockIdx.x * TOKENS + u * ROWS + threadIdx.x / LPR;
    codes[u][0] = codes[u][1] = par[u] = 0;
    if (t >= num_tokens) continue;
    const int64_t slot = index64 ? __ldg(reinterpret_cast<const long long*>(index) + t)
                                 : (int64_t)__ldg(reinterpret_cast<const int32_t*>(index) + t);
    if (slot < 0 || slot >= num_slots) {
      if (blockIdx.y == 0 && rl == 0) set_err(err, MF_ERR_SLOT);
      continue;  // zeros
    }
    const int tok = (int)(slot & (q4::BLOCK - 1));
    const uint8_t* rec = head + (slot / q4::BLOCK) * sb;
    if (!is_v) {
      const uint2 v = __ldg(reinterpret_cast<const uint2*>(rec + tok * (D / 2) + rl * 8));
      codes[u][0] = v.x, codes[u][1] = v.y;
    } else {
      // whole words (two tokens'), of which this token's half
#pragma unroll
      for (int w = 0; w < 2; ++w) {
        const uint2 v = __ldg(reinterpret_cast<const uint2*>(
            rec + (q4::v_piece<D>(tok, 4 * rl + 2 * w) & ~3)));
        codes[u][w] = __byte_perm(v.x, v.y, (tok & 1) ? 0x7632 : 0x5410);
      }
    }
    par[u] = __ldg(reinterpret_cast<const uint32_t*>(rec + 16 * D + (is_v ? 64 : 0) + tok * 4));
  }
#pragma unroll
  for (int u = 0; u < PASSES; ++u) {
    const int t = blockIdx.x * TOKENS + u * ROWS + threadIdx.x / LPR;
    if (t >= num_tokens) continue;
    const float2 sb2 = __half22float2(*reinterpret_cast<const __half2*>(&par[u]));
    S* dst = out + (int64_t)t * o_st;
#pragma unroll
    for (int w = 0; w < 2; ++w) {
      float x[8];
#pragma unroll
      for (int i = 0; i < 4; ++i) {  // codes i and i + 4, as 1024 + n under fp16's exponent
        uint32_t p = ((codes[u][w] >> (4 * i)) & 0x000F000Fu) | 0x64006400u;
        asm("sub.rn.f16x2 %0, %0, %1;" : "+r"(p) : "r"(0x64006400u));
        const float2 n = __half22float2(*reinterpret_cast<const __half2*>(&p));
        x[i] = fmaf(n.x, sb2.x, sb2.y);
        x[i + 4] = fmaf(n.y, sb2.x, sb2.y);
      }
      alignas(16) S e[8];
      if constexpr (sizeof(S) == 2) {
        uint32_t* q = reinterpret_cast<uint32_t*>(e);
#pragma unroll
        for (int i = 0; i < 4; ++i) q[i] = Mma<S>::pack(x[2 * i], x[2 * i + 1]);
        if (sb2.x != sb2.x || sb2.y != sb2.y) {  // torch's NaN
#pragma unroll
          for (int i = 0; i < 8; ++i) e[i] = from_f32<S>(NAN);
        }
      } else {
#pragma unroll
        for (int i = 0; i < 8; ++i) e[i] = x[i];
      }
      if (vec) {
#pragma unroll
        for (int i = 0; i < (int)sizeof(S) / 2; ++i)
          reinterpret_cast<uint4*>(dst + 8 * w)[i] = reinterpret_cast<const uint4*>(e)[i];
      } else {
#pragma unroll
        for (int i = 0; i < 8; ++i) dst[8 * w + i] = e[i];
      }
    }
  }
}

template <typename S>
bool rows_vec(const void* a, const void* b, int64_t s0, int64_t s1, int64_t s2, int64_t s3) {
  auto al = [](const void* p) { return (reinterpret_cast<uintptr_t>(p) & 15) == 0; };
  auto al16 = [](int64_t s) { return (s * (int64_t)sizeof(S)) % 16 == 0; };
  return al(a) && al(b) && al16(s0) && al16(s1) && al16(s2) && al16(s3);
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
  if (H > 65535) return fail(MF_EUNSUPPORTED, "q4 reshape_and_cache: more than 65535 heads");
  const int per = 8 * 32 / (D / E);  // tokens a block
  const dim3 grid((unsigned)((T + per - 1) / per), (unsigned)H);
  auto go = [&](auto kern) {
    kern<<<grid, 256, 0, stream>>>(static_cast<const S*>(k), static_cast<const S*>(v), kst, ksh,
                                   vst, vsh, pool, sb, sh, num_slots, slots, s64, T, vec, err);
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
  if (H > 65535) return fail(MF_EUNSUPPORTED, "q4 gather_kv: more than 65535 heads");
  cfg.gridDim = dim3((unsigned)((T + 63) / 64), (unsigned)H, 2);  // 64 tokens a block
  cfg.blockDim = dim3(256);
  cfg.stream = stream;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  auto kern = D == 64 ? q4_gather_kernel<S, 64>
                      : D == 128 ? q4_gather_kernel<S, 128> : q4_gather_kernel<S, 256>;
  const cudaError_t e = cudaLaunchKernelEx(&cfg, kern, pool, sb, sh, num_slots, index, i64, T,
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
