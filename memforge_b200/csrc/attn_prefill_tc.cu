// Host side of the tcgen05 chunk kernel over 16-bit pools; the kernel is in
// attn_prefill_body.cuh.

#include "attn_prefill_body.cuh"
#include "attn_prefill_maps.h"

namespace mf {
namespace pf {

template <typename T, bool MOD>
__global__ void __launch_bounds__(THREADS, 1) prefill_kernel(
    const __grid_constant__ CUtensorMap tmq, const __grid_constant__ CUtensorMap tmk,
    const __grid_constant__ CUtensorMap tmv, const __grid_constant__ CUtensorMap tmwk,
    const __grid_constant__ CUtensorMap tmwv, const __grid_constant__ Params P) {
  prefill_body<T, MOD, false>(&tmq, &tmk, &tmv, &tmwk, &tmwv, P);
}

}  // namespace pf

// ----------------------------------------------------------------- host side

const char* prefill_tc_unsupported(const AttnParams& p, mf_dtype dtype) {
  if (dtype != MF_BF16 && dtype != MF_F16) return "dtype is not bf16/f16";
  if (p.d != pf::D) return "head_dim is not 128";
  if (p.block_size != pf::PAGE) return "block_size is not 16";
  if (p.sb != (int64_t)pf::PAGE * p.ss) return "pool blocks are not slot-contiguous";
  if ((p.ss * 2) % 16 || (p.sh * 2) % 16) return "pool strides not 16-byte multiples";
  if ((reinterpret_cast<uintptr_t>(p.kp) | reinterpret_cast<uintptr_t>(p.vp) |
       reinterpret_cast<uintptr_t>(p.q) | reinterpret_cast<uintptr_t>(p.out)) & 15)
    return "q/out/pool not 16-byte aligned";
  if ((p.q_sr * 2) % 16 || (p.q_sh * 2) % 16 || (p.o_sr * 2) % 16 || (p.o_sh * 2) % 16)
    return "q/out strides not 16-byte multiples";
  const int G = p.hq / p.hkv;
  if (G < 1 || G > 16) return "GQA group above 16";
  if (p.row_map) return "row_map";
  if (p.wk) {
    if (p.max_q_len > pf::PAGE) return "window longer than 16 rows";
    if ((p.w_sr * 2) % 16 || (p.w_sh * 2) % 16) return "window strides not 16-byte multiples";
    if ((reinterpret_cast<uintptr_t>(p.wk) | reinterpret_cast<uintptr_t>(p.wv)) & 15)
      return "window not 16-byte aligned";
  }
  if (p.num_seqs > pf::MAX_SEQS) return "more than 4096 sequences";
  if (!p.causal) return "non-causal";
  if ((int64_t)p.num_blocks * pf::PAGE > 0x7fffffffLL) return "pool slots exceed int32";
  return nullptr;
}

int launch_attn_prefill_tc(const AttnParams& p, mf_dtype dtype, int rows_cap,
                           cudaStream_t stream) {
  const CUtensorMapDataType dt =
      dtype == MF_BF16 ? CU_TENSOR_MAP_DATA_TYPE_BFLOAT16 : CU_TENSOR_MAP_DATA_TYPE_FLOAT16;
  const int G = p.hq / p.hkv;
  CUtensorMap mq, mk, mv, mwk, mwv;
  const uint64_t slots = (uint64_t)p.num_blocks * pf::PAGE;
  const int ppt = pf::positions_per_tile(G);
  // q: (64, heads, halves, rows), box (64, G heads, 1, floor(128/G) positions)
  CUresult r0 = encode_pf(&mq, p.q, (uint64_t)p.hq, (uint64_t)p.q_sh * 2, (uint64_t)p.total_q,
                          (uint64_t)p.q_sr * 2, (uint32_t)G, (uint32_t)ppt, dt);
  // pool: (64, slots, halves, kv heads), box (64, 16 tokens, 1, 1 head)
  CUresult r1 = encode_pf(&mk, p.kp, slots, (uint64_t)p.ss * 2, (uint64_t)p.hkv,
                          (uint64_t)p.sh * 2, pf::PAGE, 1, dt);
  CUresult r2 = encode_pf(&mv, p.vp, slots, (uint64_t)p.ss * 2, (uint64_t)p.hkv,
                          (uint64_t)p.sh * 2, pf::PAGE, 1, dt);
  // window: (64, rows, halves, kv heads), box (64, 16 rows, 1, 1 head)
  CUresult r3 = CUDA_SUCCESS, r4 = CUDA_SUCCESS;
  if (p.wk) {
    r3 = encode_pf(&mwk, p.wk, (uint64_t)p.total_q, (uint64_t)p.w_sr * 2, (uint64_t)p.hkv,
                   (uint64_t)p.w_sh * 2, pf::PAGE, 1, dt);
    r4 = encode_pf(&mwv, p.wv, (uint64_t)p.total_q, (uint64_t)p.w_sr * 2, (uint64_t)p.hkv,
                   (uint64_t)p.w_sh * 2, pf::PAGE, 1, dt);
  } else {
    mwk = mk;
    mwv = mv;
  }
  if (r0 != CUDA_SUCCESS || r1 != CUDA_SUCCESS || r2 != CUDA_SUCCESS || r3 != CUDA_SUCCESS ||
      r4 != CUDA_SUCCESS)
    return fail(MF_ECUDA, "prefill: tensor map encoding failed");
  pf::Params P;
  P.a = p;
  P.G = G;
  P.rows_cap = rows_cap;
  P.set_scores();
  P.in_fmt = dtype == MF_BF16 ? 1u : 0u;
  P.window = p.wk ? 1 : 0;
  // Persistent grid: one CTA per SM, or fewer when there are fewer items
  // (num_seqs x query tiles of the longest run x kv heads bounds the count).
  const int64_t q_tiles = ((int64_t)p.max_q_len + ppt - 1) / ppt;
  const int64_t items_max = (int64_t)p.num_seqs * q_tiles * p.hkv;
  if (items_max == 0) return MF_OK;
  const int64_t grid = std::min<int64_t>(items_max, current_sm_count());
  const bool mod = p.mods.any();
  auto kern = dtype == MF_BF16
                  ? (mod ? pf::prefill_kernel<__nv_bfloat16, true> : pf::prefill_kernel<__nv_bfloat16, false>)
                  : (mod ? pf::prefill_kernel<__half, true> : pf::prefill_kernel<__half, false>);
  const size_t smem = pf::smem_bytes(p.num_seqs) + 1024;
  static thread_local int configured_dev[4] = {-1, -1, -1, -1};
  int dev = 0;
  cudaGetDevice(&dev);
  const int which = (dtype == MF_BF16 ? 1 : 0) + (mod ? 2 : 0);
  if (configured_dev[which] != dev) {
    cudaError_t e = cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize,
                                         (int)(pf::smem_bytes(pf::MAX_SEQS) + 1024));
    if (e != cudaSuccess) return fail(MF_ECUDA, std::string("prefill: ") + cudaGetErrorString(e));
    configured_dev[which] = dev;
  }
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3((unsigned)grid);
  cfg.blockDim = dim3(pf::THREADS);
  cfg.dynamicSmemBytes = smem;
  cfg.stream = stream;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  cudaError_t le = cudaLaunchKernelEx(&cfg, kern, mq, mk, mv, mwk, mwv, P);
  if (le != cudaSuccess)
    return fail(MF_ECUDA, std::string("prefill: ") + cudaGetErrorString(le));
  return check_launch("paged attention (tcgen05 prefill)");
}

}  // namespace mf
