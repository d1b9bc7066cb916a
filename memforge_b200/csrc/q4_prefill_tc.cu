// Long query runs over the 4-bit cache: the tcgen05 chunk kernel with operands that warps
// convert from the records (attn_prefill_body.cuh, Q4).

#include <algorithm>
#include <atomic>

#include "attn_prefill_body.cuh"
#include "q4_attn.h"

namespace mf {
namespace pf {

template <typename T, bool MOD>
__global__ void __launch_bounds__(Q4_THREADS, 1)
    q4_prefill_kernel(const __grid_constant__ Params P) {
  prefill_body<T, MOD, true>(nullptr, nullptr, nullptr, nullptr, nullptr, P);
}

template <typename T, bool MOD>
static int launch_q4(const Params& P, int64_t grid, cudaStream_t stream) {
  auto kern = q4_prefill_kernel<T, MOD>;
  static thread_local int ready = -1;
  int dev = 0;
  cudaGetDevice(&dev);
  if (ready != dev) {
    const cudaError_t e = cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize,
                                               (int)(smem_bytes(Q4_MAX_SEQS, true) + 1024));
    if (e != cudaSuccess)
      return fail(MF_ECUDA, std::string("q4 attention: ") + cudaGetErrorString(e));
    ready = dev;
  }
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3((unsigned)grid);
  cfg.blockDim = dim3(Q4_THREADS);
  cfg.dynamicSmemBytes = smem_bytes(P.a.num_seqs, true) + 1024;
  cfg.stream = stream;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  const cudaError_t e = cudaLaunchKernelEx(&cfg, kern, P);
  if (e != cudaSuccess)
    return fail(MF_ECUDA, std::string("q4 attention: ") + cudaGetErrorString(e));
  return check_launch("q4 attention (chunks)");
}

}  // namespace pf

// bf16 only: keys, values and P rounded to fp16 stay far below a bf16 output's own rounding (1.03
// times its error against 64 bits), but add up to 2.3 times an fp16 output's.  fp16 runs stay
// with mma.sync, whose codes are exact (1.15 times).
bool q4_prefill_serves(const AttnParams& a, mf_dtype dtype) {
  return dtype == MF_BF16 && a.d == pf::D && a.hq / a.hkv <= pf::BM &&
         a.num_seqs <= pf::Q4_MAX_SEQS;
}

// The kernel's register split is of the 96 registers a thread that ptxas gave it here; a build
// with another number must not run it (setmaxnreg would wait for registers that are not there), and
// leaves such runs to mma.sync.
bool q4_converting_built() {
  static std::atomic<int> known{-1};
  int ok = known.load(std::memory_order_relaxed);
  if (ok < 0) {
    cudaFuncAttributes a, b;
    if (cudaFuncGetAttributes(&a, pf::q4_prefill_kernel<__nv_bfloat16, false>) != cudaSuccess ||
        cudaFuncGetAttributes(&b, pf::q4_prefill_kernel<__nv_bfloat16, true>) != cudaSuccess) {
      cudaGetLastError();
      return false;
    }
    ok = a.numRegs == pf::Q4_REGS_LAUNCH && b.numRegs == pf::Q4_REGS_LAUNCH;
    known.store(ok, std::memory_order_relaxed);
  }
  return ok != 0;
}

int launch_q4_prefill(const AttnParams& a, int width, int vec, int rows_cap,
                      cudaStream_t stream) {
  pf::Params P{};
  P.a = a;
  P.G = a.hq / a.hkv;
  P.rows_cap = rows_cap;
  P.set_scores();
  P.in_fmt = 0;  // fp16 operands
  P.width = width;
  P.vec = vec;
  const int ppt = pf::positions_per_tile(P.G);
  const int64_t items = (int64_t)a.num_seqs * ((a.max_q_len + ppt - 1) / ppt) * a.hkv;
  const int64_t grid = std::min<int64_t>(items, current_sm_count());
  if (grid == 0) return MF_OK;
  const bool mod = a.mods.any();
  return mod ? pf::launch_q4<__nv_bfloat16, true>(P, grid, stream)
             : pf::launch_q4<__nv_bfloat16, false>(P, grid, stream);
}

}  // namespace mf
