// Long query runs over the 4-bit cache where many row tiles read the same keys: the cache's live
// pages are expanded to fp16 once, into the workspace, and the tcgen05 chunk kernel reads
// them by TMA (attn_prefill_body.cuh, EXP).
//
// The converting form of that kernel redoes the conversion for every 128-row tile, and its
// converters' 3000 instructions a key tile share the SM with the softmax.  Expanding costs 512
// bytes of writes per token and kv head, once.  It is used from five row tiles of a kv head on,
// while the expanded copy (bounded by the tables' width) stays below SCRATCH_MAX.  Expanded :
// converting in us (device, 32/8 heads, every run of the given tiles at the end of its keys):
//
//   tiles                          3          4          5          6          8           16
//   4 sequences of 2000 keys   41 :  43   42 :  43   60 :  76   61 :  78   62 :  77    99 :  141
//   4 of 8000                 121 : 115  122 : 116  189 : 218  189 : 228  189 : 226   325 :  438
//   16 of 2000                117 : 114  134 : 149  154 : 179  174 : 216  191 : 248   322 :  462
//   16 of 8000                381 : 338  453 : 454  525 : 590  599 : 670  670 : 817  1160 : 1498

#include <algorithm>

#include "attn_prefill_body.cuh"
#include "attn_prefill_maps.h"
#include "q4_attn.h"

namespace mf {
namespace pf {

constexpr size_t SCRATCH_MAX = size_t(1) << 30;
constexpr int MIN_TILES = 5;  // row tiles of a kv head

template <typename T, bool MOD>
__global__ void __launch_bounds__(THREADS, 1) q4_expanded_kernel(
    const __grid_constant__ CUtensorMap tmq, const __grid_constant__ CUtensorMap tmk,
    const __grid_constant__ CUtensorMap tmv, const __grid_constant__ Params P) {
  prefill_body<T, MOD, false, true>(&tmq, &tmk, &tmv, &tmk, &tmv, P);
}

// q in fp16, each row times the power of two that brings its largest element to
// [2^14, 2^15), in the order of the run's rows; 16 lanes a row.  Rows of no sequence (behind the
// last one's) become zeros: neither their entries of the row map nor their q are read.
template <typename T>
__global__ void __launch_bounds__(256) q4_expand_q(const __grid_constant__ Params P, __half* out,
                                                   float* scale) {
  grid_launch_dependents();
  grid_dependency_wait();
  const uint32_t at = blockIdx.x * 16 + threadIdx.x / 16, rows = (uint32_t)(P.a.total_q * P.a.hq);
  const int c = threadIdx.x & 15;
  const int r = (int)(at / (uint32_t)P.a.hq), h = (int)(at - (uint32_t)r * (uint32_t)P.a.hq);
  const int first = P.a.cu_q ? P.a.cu_q[0] : 0;
  const int end = P.a.cu_q ? P.a.cu_q[P.a.num_seqs] : P.a.num_seqs * P.a.q_per_seq;
  uint4 in = make_uint4(0, 0, 0, 0);
  if (at < rows && r >= first && r < end) {
    const T* p = static_cast<const T*>(P.a.q) + (int64_t)map_row(P.a, r) * P.a.q_sr +
                 (int64_t)h * P.a.q_sh + c * 8;
    in = __ldg(reinterpret_cast<const uint4*>(p));
  }
  const T* t = reinterpret_cast<const T*>(&in);
  float x[8];
#pragma unroll
  for (int e = 0; e < 8; ++e) x[e] = Elt<T>::to_f32(t[e]);
  float top = 0.f;
#pragma unroll
  for (int e = 0; e < 8; ++e) top = fmaxf(top, fabsf(x[e]));
#pragma unroll
  for (int o = 1; o < 16; o <<= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, o));
  if (at >= rows) return;
  const int ex = (int)(__float_as_uint(top) >> 23);
  const float mul = __uint_as_float((uint32_t)min(max(268 - ex, 1), 240) << 23);
  if (c == 0) scale[at] = P.scale_log2 / mul;
  uint4 v;
  v.x = Mma<__half>::pack(x[0] * mul, x[1] * mul);
  v.y = Mma<__half>::pack(x[2] * mul, x[3] * mul);
  v.z = Mma<__half>::pack(x[4] * mul, x[5] * mul);
  v.w = Mma<__half>::pack(x[6] * mul, x[7] * mul);
  reinterpret_cast<uint4*>(out)[(int64_t)at * 16 + c] = v;
}

// Keys and values in fp16 (one rounding): 64 threads a record.  Tokens behind the
// sequence's last are zeros; pages that no row sees are left out.
__global__ void __launch_bounds__(256) q4_expand_kv(const __grid_constant__ Params P, __half* k,
                                                    __half* v) {
  grid_launch_dependents();
  grid_dependency_wait();
  const int s = blockIdx.y, unit = blockIdx.x * 4 + threadIdx.x / 64, ts = threadIdx.x & 63;
  const int page = unit / P.a.hkv, h = unit - page * P.a.hkv;
  int q_start, q_len;
  seq_rows(P.a, s, q_start, q_len);
  if (q_len <= 0 || (int64_t)q_len * P.G <= P.rows_cap) return;
  const int kv = P.a.kv_lens[s], len = min(kv, P.width * PAGE);
  if (page * PAGE >= len) return;
  q_len = min(q_len, P.a.max_q_len);
  if (P.a.mods.window > 0) {
    const int pfx = P.a.mods.prefix ? P.a.mods.prefix[s] : 0;
    if (page * PAGE >= pfx && page * PAGE + PAGE <= kv - q_len - P.a.mods.window + 1) return;
  }
  int id = __ldg(P.a.tables + (int64_t)s * P.a.table_stride + page);
  if (id < 0 || id >= P.a.num_blocks) {
    if (ts == 0) set_err(P.a.err, MF_ERR_BLOCK_ID);
    id = 0;
  }
  const uint8_t* rec =
      static_cast<const uint8_t*>(P.a.kp) + (int64_t)id * P.a.sb + (int64_t)h * P.a.sh;
  const uint4 kc = __ldg(reinterpret_cast<const uint4*>(rec) + ts);
  const uint4 vc = __ldg(reinterpret_cast<const uint4*>(rec + 8 * D) + ts);
  const int kr = ts >> 2, vr = (ts >> 5) * 8 + 2 * (ts & 3);  // K row, first of two V rows
  const uint32_t* par = reinterpret_cast<const uint32_t*>(rec + 16 * D);  // K's 16, V's 16
  auto params = [&](bool value, int row, uint32_t& sc, uint32_t& ba) {
    const uint32_t of_v = __ldg(par + 16 + row);
    uint32_t pr = !value ? key_params(__ldg(par + row), of_v) : nan_row(of_v) ? 0u : of_v;
    if (page * PAGE + row >= len) pr = 0u;
    sc = __byte_perm(pr, pr, 0x1010);
    ba = __byte_perm(pr, pr, 0x3232);
    return pr;
  };
  const int64_t row0 = ((int64_t)s * P.width + page) * PAGE;
  {
    uint32_t sc, ba;
    const bool past = past_range(params(false, kr, sc, ba));
    uint4* dst = reinterpret_cast<uint4*>(k + ((row0 + kr) * P.a.hkv + h) * D + (ts & 3) * 32);
    const uint32_t* w = &kc.x;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      uint32_t p[4];
      code_pairs(w[i], p);  // (0, 4) (1, 5) (2, 6) (3, 7)
#pragma unroll
      for (int e = 0; e < 4; ++e) p[e] = half2_fma(p[e], sc, ba);
      if (past) {
#pragma unroll
        for (int e = 0; e < 4; ++e) p[e] = held(p[e]);
      }
      dst[i] = make_uint4(__byte_perm(p[0], p[1], 0x5410), __byte_perm(p[2], p[3], 0x5410),
                          __byte_perm(p[0], p[1], 0x7632), __byte_perm(p[2], p[3], 0x7632));
    }
  }
  {
    uint32_t s0, b0, s1, b1;
    const uint32_t p0 = params(true, vr, s0, b0), p1 = params(true, vr + 1, s1, b1);
    const uint32_t sc = __byte_perm(s0, s1, 0x5410), ba = __byte_perm(b0, b1, 0x5410);
    const bool past = past_range(half2_max(p0, p1));
    uint4* d0 = reinterpret_cast<uint4*>(v + ((row0 + vr) * P.a.hkv + h) * D + ((ts & 31) >> 2) * 16);
    uint4* d1 = d0 + P.a.hkv * (D / 8);
    const uint32_t* w = &vc.x;
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      uint32_t p[8];
      code_pairs(w[2 * i], p);  // (even, odd token) of four dims
      code_pairs(w[2 * i + 1], p + 4);
#pragma unroll
      for (int e = 0; e < 8; ++e) p[e] = half2_fma(p[e], sc, ba);
      if (past) {
#pragma unroll
        for (int e = 0; e < 8; ++e) p[e] = held(p[e]);
      }
      d0[i] = make_uint4(__byte_perm(p[0], p[1], 0x5410), __byte_perm(p[2], p[3], 0x5410),
                         __byte_perm(p[4], p[5], 0x5410), __byte_perm(p[6], p[7], 0x5410));
      d1[i] = make_uint4(__byte_perm(p[0], p[1], 0x7632), __byte_perm(p[2], p[3], 0x7632),
                         __byte_perm(p[4], p[5], 0x7632), __byte_perm(p[6], p[7], 0x7632));
    }
  }
}

template <typename T, bool MOD>
static int launch_expanded(const Params& P, const CUtensorMap& mq, const CUtensorMap& mk,
                           const CUtensorMap& mv, __half* q, float* scale, __half* k, __half* v,
                           int64_t grid, cudaStream_t stream) {
  auto kern = q4_expanded_kernel<T, MOD>;
  static thread_local int ready = -1;
  int dev = 0;
  cudaGetDevice(&dev);
  if (ready != dev) {
    const cudaError_t e = cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize,
                                               (int)(smem_bytes(MAX_SEQS) + 1024));
    if (e != cudaSuccess)
      return fail(MF_ECUDA, std::string("q4 attention: ") + cudaGetErrorString(e));
    ready = dev;
  }
  cudaLaunchAttribute attr[1];
  cudaLaunchConfig_t cfg = {};
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  cfg.stream = stream;
  cfg.blockDim = dim3(256);
  cfg.gridDim = dim3((unsigned)(((int64_t)P.a.total_q * P.a.hq + 15) / 16));
  cudaError_t e = cudaLaunchKernelEx(&cfg, q4_expand_q<T>, P, q, scale);
  if (e == cudaSuccess) {
    cfg.gridDim = dim3((unsigned)((P.width * P.a.hkv + 3) / 4), (unsigned)P.a.num_seqs);
    e = cudaLaunchKernelEx(&cfg, q4_expand_kv, P, k, v);
  }
  if (e == cudaSuccess) {
    cfg.gridDim = dim3((unsigned)grid);
    cfg.blockDim = dim3(THREADS);
    cfg.dynamicSmemBytes = smem_bytes(P.a.num_seqs) + 1024;
    e = cudaLaunchKernelEx(&cfg, kern, mq, mk, mv, P);
  }
  if (e != cudaSuccess)
    return fail(MF_ECUDA, std::string("q4 attention: ") + cudaGetErrorString(e));
  return check_launch("q4 attention (expanded)");
}

}  // namespace pf

bool q4_expand_plan(const AttnParams& a, int width, int vec, mf_dtype dtype, Q4Scratch& sc) {
  const int G = a.hq / a.hkv;
  if (!vec || (int64_t)a.total_q * a.hq > 0x7fffffffLL - 16) return false;
  if (!q4_prefill_serves(a, dtype) || G > 16) return false;
  const int ppt = pf::positions_per_tile(G);
  if ((a.max_q_len + ppt - 1) / ppt < pf::MIN_TILES) return false;
  auto up = [](size_t x) { return (x + 255) & ~(size_t)255; };
  const double rows = (double)a.num_seqs * width * q4::BLOCK * a.hkv;
  if (rows * pf::D * 4 > (double)pf::SCRATCH_MAX || a.num_seqs > 65535) return false;
  const size_t kv = (size_t)rows * pf::D * 2;
  sc.q = 0;
  sc.scale = up((size_t)a.total_q * a.hq * pf::D * 2);
  sc.k = sc.scale + up((size_t)a.total_q * a.hq * 4);
  sc.v = sc.k + up(kv);
  sc.bytes = sc.v + up(kv);
  return true;
}

int launch_q4_expanded(const AttnParams& a, int width, int rows_cap, const Q4Scratch& sc,
                       uint8_t* ws, cudaStream_t stream) {
  pf::Params P{};
  P.a = a;
  P.G = a.hq / a.hkv;
  P.rows_cap = rows_cap;
  P.set_scores();
  P.in_fmt = 0;  // fp16 operands
  P.width = width;
  P.vec = 1;
  auto* q = reinterpret_cast<__half*>(ws + sc.q);
  auto* scale = reinterpret_cast<float*>(ws + sc.scale);
  auto* k = reinterpret_cast<__half*>(ws + sc.k);
  auto* v = reinterpret_cast<__half*>(ws + sc.v);
  P.qs = scale;
  const int ppt = pf::positions_per_tile(P.G);
  const uint64_t slots = (uint64_t)a.num_seqs * width * pf::PAGE;
  const uint64_t tok = (uint64_t)a.hkv * pf::D * 2;
  CUtensorMap mq, mk, mv;
  const auto f16 = CU_TENSOR_MAP_DATA_TYPE_FLOAT16;
  if (encode_pf(&mq, q, (uint64_t)a.hq, pf::D * 2, (uint64_t)a.total_q, (uint64_t)a.hq * pf::D * 2,
                (uint32_t)P.G, (uint32_t)ppt, f16) != CUDA_SUCCESS ||
      encode_pf(&mk, k, slots, tok, (uint64_t)a.hkv, pf::D * 2, pf::PAGE, 1, f16) != CUDA_SUCCESS ||
      encode_pf(&mv, v, slots, tok, (uint64_t)a.hkv, pf::D * 2, pf::PAGE, 1, f16) != CUDA_SUCCESS)
    return fail(MF_ECUDA, "q4 attention: tensor map encoding failed");
  const int64_t items = (int64_t)a.num_seqs * ((a.max_q_len + ppt - 1) / ppt) * a.hkv;
  const int64_t grid = std::min<int64_t>(items, current_sm_count());
  const bool mod = a.mods.any();
  return mod ? pf::launch_expanded<__nv_bfloat16, true>(P, mq, mk, mv, q, scale, k, v, grid, stream)
             : pf::launch_expanded<__nv_bfloat16, false>(P, mq, mk, mv, q, scale, k, v, grid, stream);
}

}  // namespace mf
