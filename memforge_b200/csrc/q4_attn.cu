// Attention over the 4-bit paged KV cache: decode, verify and chunk rows.
//
//   s  = scale * (sk * (q . n) + bk * sum(q))        (key = sk * n + bk, n the codes)
//   out = sum_k p_k (sv_k n_k + bv_k) / sum_k p_k,   p = 2^(s log2(e) - m)
//
// Bound by reading the cache: D + 8 bytes per (token, kv head).  What the design
// saves is the arithmetic of turning 4-bit codes into MMA operands, which would
// otherwise bind first:
//  * A code n in the low bits of an fp16 is the denormal n * 2^-24, exactly.  One
//    AND of a 32-bit word therefore yields two operand elements (mask 0x000F000F, or
//    0x00F000F0 for 16 n, whose factor 1/16 is folded into q or the epilogue); one shift
//    serves the word's other four codes.  No conversion, no scale per element.
//  * The scales stay outside the products: sk and bk enter once per (key, row) after
//    Q K^T, sv is multiplied into p before P V, bv enters as sum p bv.
//  * S^T = K Q^T and O^T = V^T P^T (mma.sync m16n8k16, fp32 accumulate) keep the keys
//    and the head dims on M = 16 and the rows of a GQA group on N = 8, so eight query
//    rows cost what one does.  The record stores V in A-fragment order, so every
//    fragment is a 16-byte shared load.
// q enters as fp16 scaled by a power of two (largest element of the row tile near 2^14), so
// bf16 and fp16 queries are exact down to 2^-28 of that element; fp32 queries and their P
// are split into two fp16 numbers (22 bits), and their codes taken as n - 8: the products
// with n itself are several times the values', and fp32 sums of them would cancel
// (4e-5 relative at a few thousand keys, measured).  P for 16-bit outputs is rounded to fp16 (2^-12
// relative), at or below the output's own rounding; for fp16 outputs the codes are
// centred (a constant A operand sums the rounded P, times 8), else that rounding would
// count at the size of n * sv instead of the value's.
//
// Work: units (sequence, row tile, kv head) of n pages each, concatenated and cut
// into equal contiguous ranges, one per CTA (4 warps, 4 CTAs per SM at NT = 1).  The
// warps of a CTA take the pages of its range in turn, each with its own ring of
// records fetched by untiled bulk copies (one contiguous record per page), so no warp
// waits for another inside a unit; at a unit's end the four partial results are joined
// through shared memory.  A unit cut by a range border leaves fp32 partials in the
// workspace; a second, dependent launch joins those and writes zeros for sequences
// without a visible key.  No counters and no atomics: the workspace needs no
// initial value, and results do not depend on arrival order.
//
// The products add up p * n, all of one sign, and every add of the tensor core rounds toward zero,
// by 1e-7 of the sum so far.  Over a warp's 2048 pages of a 131072-key sequence the sums lost
// 1e-4 of themselves: 6 % of the output where flat weights let the values cancel (bf16; 2.7 %
// in fp16, 0.3 % in fp32).  So every SHIFT pages twice a row's mean sum over the dims moves from
// the accumulators to the row's scalar part (sum p bv), which is summed with rounding to nearest:
// the sums then lie below zero for one span and above it for the next, and what they lose cancels
// (bf16 then 0.19 %, its rounding; fp16 0.03 %, fp32 5e-5; 2 % of the time).
//
// The running maximum is lazy: a tile raises it only when some score exceeds it by
// more than 8 (log2 units), so the common tile has one vote and no shuffles; the same
// vote covers the power of two that keeps p * sv inside fp16.

#include <algorithm>

#include "mf_attn.h"
#include "mf_q4.cuh"
#include "q4_attn.h"

namespace mf {
namespace q4a {

constexpr int PAGE = q4::BLOCK;
constexpr int WARPS = 4;
constexpr int THREADS = WARPS * 32;
constexpr uint64_t WAIT_LIMIT = 2000000000ull;
constexpr float RAISE = 8.f;        // log2 units
constexpr float PV_TOP = 128.f;     // largest sv * kinv; p <= 2^8 makes 2^15 < 65504

struct Params {
  AttnParams a;  // kp: the pool, sb / sh: its block and head strides in bytes
  int G, RT;      // query heads per kv head; most row tiles of a sequence
  uint32_t g_mul; // ceil(2^32 / G): rows are divided by G a few times per unit
  int min_tiles;  // fewest pages a CTA is given
  int rows_cap;   // runs of more rows per kv head belong to another kernel (0: none do)
  int width;      // entries of a block table's row
  int vec;        // q and out rows allow 16-byte loads and 8-byte stores
  int32_t* prefix;   // [num_seqs + 1]
  float* part;
  int part_floats;
};

struct Geo {
  int q_start, q_len, kv, win0;  // kv: visible cache length, win0: position of row 0
  int pfx, pa, gap, n;           // prefix keys, its pages, pages left out after them, pages
  int nrt;
};

// r / G for rows of a run (below 2^24, G at most 255: the host checks), and r % G.
MF_DEVINL int div_g(const Params& P, int r) {
  return P.G == 1 ? r : (int)__umulhi((uint32_t)r, P.g_mul);
}
MF_DEVINL int mod_g(const Params& P, int r) { return r - div_g(P, r) * P.G; }

template <bool MOD>
MF_DEVINL Geo seq_geo(const Params& P, int s, int rows, bool report) {
  Geo g;
  seq_rows(P.a, s, g.q_start, g.q_len);
  int kv = P.a.kv_lens[s];
  const int64_t nrows = (int64_t)g.q_len * P.G;
  g.n = g.pa = g.gap = g.pfx = 0;
  g.nrt = 0;
  g.kv = 0;
  g.win0 = kv - g.q_len;
  if (g.q_len <= 0 || (P.rows_cap && nrows > P.rows_cap)) return g;
  if (g.q_len > P.a.max_q_len) {  // more rows than the launch was sized for
    if (report) set_err(P.a.err, MF_ERR_LENGTH);
    g.q_len = P.a.max_q_len;
  }
  g.nrt = (g.q_len * P.G + rows - 1) / rows;
  if (kv < 0) {
    if (report) set_err(P.a.err, MF_ERR_LENGTH);
    kv = 0;
  }
  if ((kv + (int64_t)PAGE - 1) / PAGE > P.width) {
    if (report) set_err(P.a.err, MF_ERR_TABLE);
    kv = P.width * PAGE;
  }
  g.kv = kv;
  int pages = (int)(((int64_t)kv + PAGE - 1) / PAGE);
  if (MOD) {
    if (P.a.mods.prefix) g.pfx = min(max(P.a.mods.prefix[s], 0), kv);
    g.pa = (g.pfx + PAGE - 1) / PAGE;
    const int lo = P.a.mods.window > 0 ? min(max(g.win0 - P.a.mods.window + 1, 0), kv) : 0;
    g.gap = min(max(lo / PAGE - g.pa, 0), max(pages - g.pa, 0));
  }
  g.n = pages - g.gap;
  return g;
}

// The tile list [0, total) cut into nv equal ranges.  Tiles are counted in 32 bits (the host
// refuses calls whose tables could hold more).
struct Split {
  uint32_t total, nv, base, rem;
  MF_DEVINL uint32_t bound(uint32_t c) const { return c >= nv ? total : c * base + min(c, rem); }
  MF_DEVINL int owner(uint32_t t) const {
    const uint32_t big = (base + 1) * rem;
    return (int)(t < big ? t / (base + 1) : rem + (t - big) / base);
  }
};

MF_DEVINL Split make_split(uint32_t total, uint32_t most, uint32_t min_tiles) {
  Split s;
  s.total = total;
  s.nv = min(max((total + min_tiles - 1) / min_tiles, 1u), most);
  s.base = total / s.nv;
  s.rem = total - s.base * s.nv;
  return s;
}

// A position in a CTA's range: the unit (s, rt, h) and the next of its pages.
template <int R, bool MOD>
struct Cursor {
  uint32_t pos, base;  // start of the piece after this one; first tile of sequence s
  int s, rt, h, k, k0, k1;
  Geo g;
  int hi_max, lo_min;
  bool valid;

  MF_DEVINL void open(const Params& P, uint32_t end) {  // the piece that starts at `pos`
    valid = pos < end;
    if (!valid) return;
    uint32_t in = pos - base;
    while (in >= (uint32_t)(g.n * g.nrt * P.a.hkv)) {
      base += (uint32_t)(g.n * g.nrt * P.a.hkv);
      g = seq_geo<MOD>(P, ++s, R, false);
      in = pos - base;
    }
    const uint32_t u = in / (uint32_t)g.n;
    k0 = (int)(in - u * g.n);
    rt = P.RT == 1 ? 0 : (int)(u / (uint32_t)P.a.hkv);
    h = (int)u - rt * P.a.hkv;
    k1 = (int)min((uint32_t)g.n, k0 + (end - pos));
    pos += k1 - k0;
    const int last = min(rt * R + R, g.q_len * P.G) - 1;
    hi_max = P.a.causal ? g.win0 + div_g(P, last) : g.kv - 1;
    lo_min = MOD && P.a.mods.window > 0 ? g.win0 + div_g(P, rt * R) - P.a.mods.window + 1 : 0;
  }
  MF_DEVINL int page(int i) const { return !MOD || i < g.pa ? i : i + g.gap; }
  MF_DEVINL bool live(int pg) const {  // some row of the tile sees some key of the page
    const int b = pg * PAGE;
    return (MOD && b < g.pfx) || (b <= hi_max && (!MOD || b + PAGE - 1 >= lo_min));
  }
};

MF_DEVINL void bulk_load(uint32_t dst, const void* src, uint32_t bytes, uint64_t* bar,
                         uint64_t policy) {
  asm volatile(
      "cp.async.bulk.shared::cluster.global.mbarrier::complete_tx::bytes.L2::cache_hint "
      "[%0], [%1], %2, [%3], %4;" ::"r"(dst),
      "l"(src), "r"(bytes), "r"(smem_u32(bar)), "l"(policy)
      : "memory");
}

template <int N>
MF_DEVINL void lds_words(uint32_t addr, uint32_t* w) {
  if constexpr (N == 2)
    asm volatile("ld.shared.v2.u32 {%0,%1}, [%2];" : "=r"(w[0]), "=r"(w[1]) : "r"(addr));
  else
    asm volatile("ld.shared.v4.u32 {%0,%1,%2,%3}, [%4];"
                 : "=r"(w[0]), "=r"(w[1]), "=r"(w[2]), "=r"(w[3])
                 : "r"(addr));
}

MF_DEVINL float2 lds_half2(uint32_t addr) {
  uint32_t v;
  asm volatile("ld.shared.u32 %0, [%1];" : "=r"(v) : "r"(addr));
  return __half22float2(*reinterpret_cast<__half2*>(&v));
}

MF_DEVINL uint32_t movm_trans(uint32_t x) {
  uint32_t y;
  asm volatile("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(y) : "r"(x));
  return y;
}

// Operand registers of a code word's low nibbles (mask 0x000F000F) and of 16 times its
// next ones (0x00F000F0).  As denormals, n * 2^-24; SIGNED: 1024 + n as an fp16, less
// 1032, is n - 8 exactly.
template <bool SIGNED, bool HIGH>
MF_DEVINL uint32_t operand(uint32_t w) {
  w &= HIGH ? 0x00F000F0u : 0x000F000Fu;
  if constexpr (SIGNED) {
    w |= 0x64006400u;
    const uint32_t off = HIGH ? 0x64806480u : 0x64086408u;  // 1152, 1032
    asm("sub.rn.f16x2 %0, %0, %1;" : "+r"(w) : "r"(off));
  }
  return w;
}

template <typename T, int D, int NT>
struct Cfg {
  static constexpr bool SPLIT = sizeof(T) == 4;  // fp32: two fp16 parts, signed codes
  static constexpr float UNIT = SPLIT ? 1.f : 16777216.f;  // 1 / an operand's unit
  static constexpr bool CENTRE = std::is_same<T, __half>::value;
  static constexpr int R = 8 * NT;
  static constexpr int SHIFT = 64;  // pages of a warp from one shift of its sums to the next (2^n)
  static constexpr int REC = q4::record_bytes(D);
  // CTAs per SM by registers: 32 accumulators and 16 q registers per 8 rows at D = 128.
  static constexpr int WORK = D * NT * (SPLIT ? 2 : 1);
  static constexpr int MINB = WORK <= 128 ? 4 : WORK <= 256 ? 3 : 2;
  // Pages a warp takes in one step: two where the registers allow, for half the steps'
  // fixed cost (wait, vote, copy, loop) per page and twice the independent products.
  static constexpr int TP = NT == 1 && D <= 128 ? 2 : 1;
  static constexpr int NSTG = D == 256 ? 3 : D == 128 ? 5 : 8;
  static constexpr int DH = D / 2;       // dims joined in one pass through shared memory
  static constexpr int BUF_LD = DH + 4;  // padded row of a partial there
  static constexpr int OFF_BUF = WARPS * NSTG * REC;
  static constexpr int OFF_ML = OFF_BUF + WARPS * 8 * BUF_LD * 4;
  static constexpr int OFF_BAR = OFF_ML + WARPS * R * 8;
  static constexpr int OFF_MISC = OFF_BAR + WARPS * NSTG * 8;
  static constexpr int OFF_CUR = OFF_MISC + 64;  // the producers' cursors, off the registers
  static constexpr int SMEM = OFF_CUR + WARPS * 128;
};

template <typename T, int D, int NT, bool MOD>
__global__ void __launch_bounds__(THREADS, Cfg<T, D, NT>::MINB)
    attn_kernel(const __grid_constant__ Params P) {
  using C = Cfg<T, D, NT>;
  using MM = Mma<__half>;
  constexpr int R = C::R, NSTG = C::NSTG, REC = C::REC, TP = C::TP;
  constexpr int NW = D / 32;                   // code words per thread and row
  constexpr int VEC = NW < 4 ? NW : 4;         // of which one shared load brings VEC
  constexpr int NL = NW / VEC;
  constexpr int SP = C::SPLIT ? 2 : 1;
  auto lo4 = [](uint32_t w) { return operand<C::SPLIT, false>(w); };
  auto hi4 = [](uint32_t w) { return operand<C::SPLIT, true>(w); };
  extern __shared__ __align__(128) uint8_t smem[];
  uint64_t* bars = reinterpret_cast<uint64_t*>(smem + C::OFF_BAR);
  uint32_t* misc = reinterpret_cast<uint32_t*>(smem + C::OFF_MISC);
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const int g4 = lane >> 2, t4 = lane & 3;
  const int B = P.a.num_seqs;

  if (tid == 0) {
    for (int i = 0; i < WARPS * NSTG; ++i) mbar_init(&bars[i], 1);
    fence_barrier_init();
  }
  grid_launch_dependents();
  grid_dependency_wait();

  // ------------------------------------------ tiles of all sequences, and my range
  const int per = (B + THREADS - 1) / THREADS;
  const int s_lo = min(tid * per, B), s_hi = min(s_lo + per, B);
  uint32_t mine = 0;
  Geo first{};  // of sequence s_lo
  for (int s = s_lo; s < s_hi; ++s) {
    const Geo g = seq_geo<MOD>(P, s, R, blockIdx.x == 0);
    if (s == s_lo) first = g;
    mine += (uint32_t)(g.n * g.nrt * P.a.hkv);
  }
  uint32_t incl = mine;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const uint32_t v = __shfl_up_sync(0xffffffffu, incl, o);
    if (lane >= o) incl += v;
  }
  if (lane == 31) misc[warp] = incl;
  __syncthreads();
  uint32_t before = incl - mine, total = 0;
#pragma unroll
  for (int w = 0; w < WARPS; ++w) {
    if (w < warp) before += misc[w];
    total += misc[w];
  }
  if (blockIdx.x == 0) {
    uint32_t at = before;
    for (int s = s_lo; s < s_hi; ++s) {
      P.prefix[s] = (int)at;
      const Geo g = s == s_lo ? first : seq_geo<MOD>(P, s, R, false);
      at += (uint32_t)(g.n * g.nrt * P.a.hkv);
    }
    if (tid == 0) P.prefix[B] = (int)total;
  }
  if (total == 0) return;
  const Split S = make_split(total, gridDim.x, P.min_tiles);
  const uint32_t lo = S.bound(blockIdx.x), hi = S.bound(blockIdx.x + 1);
  if (lo >= hi) return;
  if (lo >= before && lo < before + mine) {  // one thread: the sequence that holds tile lo
    uint32_t at = before;
    int s = s_lo;
    for (; s + 1 < s_hi; ++s) {
      const Geo g = s == s_lo ? first : seq_geo<MOD>(P, s, R, false);
      const uint32_t t = (uint32_t)(g.n * g.nrt * P.a.hkv);
      if (lo < at + t) break;
      at += t;
    }
    misc[4] = at;
    misc[5] = (uint32_t)s;
  }
  __syncthreads();

  Cursor<R, MOD> cc;  // the consumer's; the producer's lies in shared memory
  cc.pos = lo;
  cc.base = misc[4];
  cc.s = (int)misc[5];
  cc.g = seq_geo<MOD>(P, cc.s, R, false);
  using Cur = Cursor<R, MOD>;
  static_assert(sizeof(Cur) <= 128, "cursor slot");
  Cur* pcs = reinterpret_cast<Cur*>(smem + C::OFF_CUR + warp * 128);
  {
    Cur pc = cc;
    pc.open(P, hi);
    pc.k = pc.k0 + TP * warp;
    if (lane == 0) *pcs = pc;
    __syncwarp();
  }
  const uint32_t ring = smem_u32(smem) + warp * NSTG * REC;
  uint64_t* bar = bars + warp * NSTG;
  const uint64_t pol = l2_evict_first_policy();
  const uint8_t* pool = static_cast<const uint8_t*>(P.a.kp);
  bool dead = false;  // a wait gave up: no more copies or products, barriers only
  int issued = 0, taken = 0, pstage = 0;
  // The producer's next records: lane j holds the address of this warp's j-th next page of
  // its piece, and fetches it itself; todo: lanes whose page is still to be fetched.
  const uint8_t* src = nullptr;
  uint32_t todo = 0;
  bool more = true;

  auto refill = [&]() {
    Cur pc = *pcs;
    while (todo == 0 && pc.valid) {
      if (pc.k >= pc.k1) {
        pc.open(P, hi);
        pc.k = pc.k0 + TP * warp;
        continue;
      }
      const int k = pc.k + (lane / TP) * (TP * WARPS) + lane % TP;
      bool want = k < pc.k1;
      if (want) {
        const int pg = pc.page(k);
        want = pc.live(pg);
        int id = want ? __ldg(P.a.tables + (int64_t)pc.s * P.a.table_stride + pg) : 0;
        if (id < 0 || id >= P.a.num_blocks) {
          set_err(P.a.err, MF_ERR_BLOCK_ID);
          id = 0;
        }
        src = pool + (int64_t)id * P.a.sb + (int64_t)pc.h * P.a.sh;
      }
      todo = __ballot_sync(0xffffffffu, want);
      pc.k += 32 * WARPS;
    }
    more = todo != 0;
    __syncwarp();
    if (lane == 0) *pcs = pc;
    __syncwarp();
  };
  // Fetches the next `want` (1 or 2) records, each by the lane that holds its address.
  auto issue = [&](int want) {
    while (want > 0) {
      if (todo == 0) {
        if (more) refill();
        if (todo == 0) return;
      }
      const uint32_t rest = todo & (todo - 1);
      const int l0 = __ffs(todo) - 1, l1 = want == 2 && rest ? __ffs(rest) - 1 : l0;
      const int next = pstage + 1 == NSTG ? 0 : pstage + 1;
      if (lane == l0 || lane == l1) {
        const int st = lane == l0 ? pstage : next;
        mbar_arrive_expect_tx(&bar[st], REC);
        bulk_load(ring + st * REC, src, REC, &bar[st], pol);
      }
      const bool two = l1 != l0;
      todo = two ? rest & (rest - 1) : rest;
      pstage = !two ? next : next + 1 == NSTG ? 0 : next + 1;
      issued += two ? 2 : 1;
      want -= two ? 2 : 1;
    }
  };

  bool primed = false;  // the ring's first fill goes out behind the first unit's q loads

  const float sl2 = P.a.scale * kLog2e;
  const float cap2 = P.a.mods.softcap * kLog2e, two_over = MOD ? 2.f / P.a.mods.softcap : 0.f;
  float* buf = reinterpret_cast<float*>(smem + C::OFF_BUF);
  float2* ml = reinterpret_cast<float2*>(smem + C::OFF_ML);
  int stage = 0;
  uint32_t phase = 0;

  for (cc.open(P, hi); cc.valid; cc.open(P, hi)) {
    const Geo& g = cc.g;
    // -------------------------------------------------------------- q of the unit
    uint32_t qb[NT][SP][NW][4];
    float qs[NT][2], cq;
    int qi[NT][2];
    float slope[NT][2];
    {
      const T* rowp[NT];
      bool have[NT];
#pragma unroll
      for (int nt = 0; nt < NT; ++nt) {
        const int rr = cc.rt * R + nt * 8 + g4;
        have[nt] = rr < g.q_len * P.G;
        rowp[nt] = static_cast<const T*>(P.a.q) +
                   (have[nt] ? (int64_t)map_row(P.a, g.q_start + div_g(P, rr)) * P.a.q_sr +
                                   (int64_t)(cc.h * P.G + mod_g(P, rr)) * P.a.q_sh
                             : 0);
#pragma unroll
        for (int j = 0; j < 2; ++j) {
          const int r2 = cc.rt * R + nt * 8 + 2 * t4 + j;
          qi[nt][j] = div_g(P, r2);
          slope[nt][j] = MOD && P.a.mods.slopes && r2 < g.q_len * P.G
                             ? P.a.mods.slopes[cc.h * P.G + mod_g(P, r2)] * kLog2e
                             : 0.f;
        }
      }
      constexpr int QV = sizeof(T) / 2;  // 16-byte loads for eight elements
      uint4 raw[NT][NW][QV];
#pragma unroll
      for (int nt = 0; nt < NT; ++nt)
#pragma unroll
        for (int i = 0; i < NW; ++i) {
          const int dim = (i / VEC) * 128 + t4 * (8 * VEC) + (i % VEC) * 8;
          const T* p = rowp[nt] + dim;
#pragma unroll
          for (int e = 0; e < QV; ++e) raw[nt][i][e] = make_uint4(0, 0, 0, 0);
          if (have[nt]) {
            if (P.vec) {
#pragma unroll
              for (int e = 0; e < QV; ++e)
                raw[nt][i][e] = __ldg(reinterpret_cast<const uint4*>(p) + e);
            } else {
              T v[8];
#pragma unroll
              for (int e = 0; e < 8; ++e) v[e] = p[e];
#pragma unroll
              for (int e = 0; e < QV; ++e) raw[nt][i][e] = reinterpret_cast<const uint4*>(v)[e];
            }
          }
        }
      if (!primed) {
        primed = true;
#pragma unroll 1
        for (int i = 0; i < NSTG; ++i) issue(1);
      }
      float top = 0.f;
#pragma unroll
      for (int nt = 0; nt < NT; ++nt) {
        float sum = 0.f;
#pragma unroll
        for (int i = 0; i < NW; ++i) {
          const T* v = reinterpret_cast<const T*>(raw[nt][i]);
#pragma unroll
          for (int e = 0; e < 8; ++e) {
            const float x = Elt<T>::to_f32(v[e]);
            sum += x;
            if (fabsf(x) <= 3.402823466e38f) top = fmaxf(top, fabsf(x));  // else its row only
          }
        }
        sum += __shfl_xor_sync(0xffffffffu, sum, 1);
        sum += __shfl_xor_sync(0xffffffffu, sum, 2);
#pragma unroll
        for (int j = 0; j < 2; ++j)
          qs[nt][j] = sl2 * __shfl_sync(0xffffffffu, sum, (2 * t4 + j) * 4);
      }
#pragma unroll
      for (int o = 1; o < 32; o <<= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, o));
      const int ex = (int)(__float_as_uint(top) >> 23);
      const float mul = __uint_as_float((uint32_t)min(max(268 - ex, 1), 240) << 23);
      cq = sl2 * C::UNIT / mul;
#pragma unroll
      for (int nt = 0; nt < NT; ++nt)
#pragma unroll
        for (int i = 0; i < NW; ++i) {
          const T* v = reinterpret_cast<const T*>(raw[nt][i]);
          float x[8];
#pragma unroll
          for (int e = 0; e < 8; ++e) x[e] = Elt<T>::to_f32(v[e]) * ((e & 1) ? mul * 0.0625f : mul);
#pragma unroll
          for (int sp = 0; sp < SP; ++sp) {
#pragma unroll
            for (int e = 0; e < 4; ++e) {  // (x0,x4) (x1,x5) (x2,x6) (x3,x7)
              const uint32_t w = MM::pack(x[e], x[e + 4]);
              qb[nt][sp][i][e] = w;
              if (SP == 2 && sp == 0) {
                const float2 f = __half22float2(*reinterpret_cast<const __half2*>(&w));
                x[e] -= f.x;
                x[e + 4] -= f.y;
              }
            }
          }
        }
    }
    float o[NT][D / 16][4], ones[NT][4];
    // mu: what scores are taken relative to (0 before any key is seen); up: how far one may
    // pass it (anything does, before).  sv_top: the largest scale that kinv serves.
    float up[NT][2], mu[NT][2], l[NT][2], ob[NT][2], kinv = 0.f, sv_top = -1.f;
#pragma unroll
    for (int nt = 0; nt < NT; ++nt) {
#pragma unroll
      for (int n = 0; n < D / 16; ++n) o[nt][n][0] = o[nt][n][1] = o[nt][n][2] = o[nt][n][3] = 0.f;
      ones[nt][0] = ones[nt][1] = ones[nt][2] = ones[nt][3] = 0.f;
      up[nt][0] = up[nt][1] = -INFINITY;
      mu[nt][0] = mu[nt][1] = 0.f;
      l[nt][0] = l[nt][1] = ob[nt][0] = ob[nt][1] = 0.f;
    }
    // Largest key every row sees from below, smallest every row sees from above.
    const int first_qi = div_g(P, cc.rt * R);
    const int hi_all = P.a.causal ? min(g.win0 + first_qi, g.kv - 1) : g.kv - 1;
    const int last_qi = div_g(P, min(cc.rt * R + R, g.q_len * P.G) - 1);
    const int lo_all = MOD && P.a.mods.window > 0 ? g.win0 + last_qi - P.a.mods.window + 1 : 0;

    for (int k = cc.k0 + TP * warp; k < cc.k1; k += TP * WARPS) {
      // The step's pages, live ones first; without a second one, its place re-reads the
      // first record as keys that no row sees.
      int kb[TP];
      constexpr int SPAN = C::SHIFT * WARPS;
      if (__builtin_expect((k & (SPAN - 1)) >= SPAN - TP * WARPS, 0) && kinv > 0.f) {
        // (unlikely: out of the way of the loop; at its end this cost 5 % instead of 2)
#pragma unroll
        for (int nt = 0; nt < NT; ++nt)
#pragma unroll
          for (int j = 0; j < 2; ++j) {
            float two = 0.f;  // twice the mean; sums of high nibbles are 16 times the values'
#pragma unroll
            for (int i = 0; i < D / 16; ++i) two += fmaf(o[nt][i][2 + j], 0.0625f, o[nt][i][j]);
#pragma unroll
            for (int x = 4; x < 32; x <<= 1) two += __shfl_xor_sync(0xffffffffu, two, x);
            two *= 2.f / D;
#pragma unroll
            for (int i = 0; i < D / 16; ++i) {
              o[nt][i][j] -= two;
              o[nt][i][2 + j] = fmaf(-16.f, two, o[nt][i][2 + j]);
            }
            if (g4 == 0)  // (ob is summed over the lanes of a row, ones is the same in each)
              ob[nt][j] += (two * C::UNIT - (C::CENTRE ? 8.f * ones[nt][j] : 0.f)) / kinv;
            ones[nt][j] = 0.f;
          }
      }
      int n = 0;
      if (!MOD && TP == 2) {  // live pages are the first ones
        kb[0] = k * PAGE;
        if (kb[0] > cc.hi_max) continue;
        const bool two = k + 1 < cc.k1 && kb[0] + PAGE <= cc.hi_max;
        kb[TP - 1] = two ? kb[0] + PAGE : 0x7fffff00;
        n = two ? 2 : 1;
      } else {
#pragma unroll
        for (int u = 0; u < TP; ++u) {
          kb[u] = 0x7fffff00;
          const int pg = cc.page(k + u);
          if (k + u < cc.k1 && cc.live(pg)) {
            if (TP == 2 && n == 0) kb[0] = pg * PAGE;
            else kb[u] = pg * PAGE;
            ++n;
          }
        }
        if (n == 0) continue;
      }
      const bool wrap = stage + 1 == NSTG;
      const int st1 = wrap ? 0 : stage + 1;
      const uint32_t ph1 = phase ^ (wrap ? 1u : 0u);
      uint32_t rec[TP];
      rec[0] = ring + stage * REC;
      if (TP == 2) rec[TP - 1] = n == 2 ? ring + st1 * REC : rec[0];
      bool here = mbar_try_wait(&bar[stage], phase);
      if (TP == 2 && n == 2) here = here && mbar_try_wait(&bar[st1], ph1);
      if (!__all_sync(0xffffffffu, here)) {
        if (!dead) {
          dead = !mbar_wait_bounded(&bar[stage], phase, WAIT_LIMIT);
          if (TP == 2 && n == 2 && !dead) dead = !mbar_wait_bounded(&bar[st1], ph1, WAIT_LIMIT);
        }
        dead = __any_sync(0xffffffffu, dead);
      }
      if (dead) continue;
      taken += n;
      stage = st1;
      phase = ph1;
      if (TP == 2 && n == 2 && ++stage == NSTG) {
        stage = 0;
        phase ^= 1u;
      }

      // ---------------------------------------------------------- S^T = K Q^T
      // At NT = 1 two accumulators halve the dependent chain.
      float sc[TP][NT][4], sd[TP][4];
#pragma unroll
      for (int u = 0; u < TP; ++u) {
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          sd[u][e] = 0.f;
#pragma unroll
          for (int nt = 0; nt < NT; ++nt) sc[u][nt][e] = 0.f;
        }
#pragma unroll
        for (int c = 0; c < NL; ++c) {
          uint32_t ka[VEC], kc[VEC];
          lds_words<VEC>(rec[u] + g4 * (D / 2) + c * 64 + t4 * (4 * VEC), ka);
          lds_words<VEC>(rec[u] + (g4 + 8) * (D / 2) + c * 64 + t4 * (4 * VEC), kc);
#pragma unroll
          for (int i = 0; i < VEC; ++i) {
            const uint32_t a0[4] = {lo4(ka[i]), lo4(kc[i]), hi4(ka[i]), hi4(kc[i])};
            const uint32_t ka8 = ka[i] >> 8, kc8 = kc[i] >> 8;
            const uint32_t a1[4] = {lo4(ka8), lo4(kc8), hi4(ka8), hi4(kc8)};
#pragma unroll
            for (int nt = 0; nt < NT; ++nt)
#pragma unroll
              for (int sp = 0; sp < SP; ++sp) {
                const uint32_t* q = qb[nt][sp][c * VEC + i];
                MM::run(sc[u][nt], a0, q[0], q[1]);
                MM::run(NT == 1 ? sd[u] : sc[u][nt], a1, q[2], q[3]);
              }
          }
        }
      }
      // ------------------------------------------------- scores in log2 units, less mu
      float sv[TP][2], bv[TP][2];  // V scale and base (of centred codes) of keys g4, g4 + 8
      bool need_mask = false;
#pragma unroll
      for (int u = 0; u < TP; ++u) {
        const uint32_t par = rec[u] + 16 * D + g4 * 4;
        float2 pk0 = lds_half2(par), pk1 = lds_half2(par + 32);
        float2 pv0 = lds_half2(par + 64), pv1 = lds_half2(par + 96);
        need_mask = need_mask || kb[u] + PAGE - 1 > hi_all ||
                    (MOD && kb[u] < lo_all && kb[u] + PAGE > g.pfx);
        if (kb[u] + PAGE > g.kv) {  // slots behind the last token hold anything
          if (kb[u] + g4 >= g.kv) pk0 = pv0 = make_float2(0.f, 0.f);
          if (kb[u] + g4 + 8 >= g.kv) pk1 = pv1 = make_float2(0.f, 0.f);
        }
        if (C::SPLIT) {  // codes were taken as n - 8
          pk0.y = fmaf(8.f, pk0.x, pk0.y);
          pk1.y = fmaf(8.f, pk1.x, pk1.y);
        }
        sv[u][0] = pv0.x;
        sv[u][1] = pv1.x;
        bv[u][0] = C::CENTRE || C::SPLIT ? fmaf(8.f, pv0.x, pv0.y) : pv0.y;
        bv[u][1] = C::CENTRE || C::SPLIT ? fmaf(8.f, pv1.x, pv1.y) : pv1.y;
        const float sk0 = pk0.x * cq, sk1 = pk1.x * cq;
#pragma unroll
        for (int nt = 0; nt < NT; ++nt)
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            const int j = e & 1;
            const float raw = NT == 1 ? sc[u][nt][e] + sd[u][e] : sc[u][nt][e];
            const float by = e < 2 ? pk0.y : pk1.y, sk = e < 2 ? sk0 : sk1;
            float x;
            if (MOD) {
              const int back = g.win0 + qi[nt][j] - (kb[u] + g4 + (e < 2 ? 0 : 8));
              x = fmaf(raw, sk, by * qs[nt][j]);
              if (P.a.mods.softcap > 0.f) x = softcap_log2(x, cap2, two_over);
              if (P.a.mods.slopes) x = fmaf(-slope[nt][j], (float)back, x);
              x -= mu[nt][j];
            } else {
              x = fmaf(raw, sk, fmaf(by, qs[nt][j], -mu[nt][j]));
            }
            sc[u][nt][e] = x;
          }
      }
      uint32_t vis = 0xffffffffu;  // bit (u * NT + nt) * 4 + e
      if (need_mask) {
        vis = 0;
#pragma unroll
        for (int u = 0; u < TP; ++u)
#pragma unroll
          for (int nt = 0; nt < NT; ++nt)
#pragma unroll
            for (int e = 0; e < 4; ++e) {
              const int key = kb[u] + g4 + (e < 2 ? 0 : 8);
              const int qpos = g.win0 + qi[nt][e & 1];
              bool see = !P.a.causal || key <= qpos;
              if (MOD && P.a.mods.window > 0) see = see && qpos - key < P.a.mods.window;
              if (MOD) see = see || key < g.pfx;
              see = see && key < g.kv;
              if (see) vis |= 1u << ((u * NT + nt) * 4 + e);
              else sc[u][nt][e] = -INFINITY;
            }
      }
      // ------------------------------------------------ running maximum, lazily
      float tm[NT][2], st = fmaxf(sv[0][0], sv[0][1]);
#pragma unroll
      for (int nt = 0; nt < NT; ++nt)
#pragma unroll
        for (int j = 0; j < 2; ++j) {
          tm[nt][j] = fmaxf(sc[0][nt][j], sc[0][nt][2 + j]);
          if (TP == 2) tm[nt][j] = fmax3f(tm[nt][j], sc[TP - 1][nt][j], sc[TP - 1][nt][2 + j]);
        }
      if (TP == 2) st = fmax3f(st, sv[TP - 1][0], sv[TP - 1][1]);
      bool raise = st > sv_top;
#pragma unroll
      for (int nt = 0; nt < NT; ++nt) raise = raise || tm[nt][0] > up[nt][0] || tm[nt][1] > up[nt][1];
      if (__any_sync(0xffffffffu, raise)) {
#pragma unroll
        for (int x = 4; x < 32; x <<= 1) st = fmaxf(st, __shfl_xor_sync(0xffffffffu, st, x));
        if (!(st <= 65504.f)) st = 0.f;  // a NaN or infinite scale is no size to go by
        float fv = 1.f;
        if (st > sv_top) {
          // 2^6 / 2^floor(log2 st): sv * kinv <= 2^7, with room for the last factor of two
          const int ex = (int)((__float_as_uint(st) >> 23) & 255u);
          const float next = __uint_as_float((uint32_t)min(max(260 - ex, 97), 160) << 23);
          fv = kinv == 0.f ? 0.f : next / kinv;
          kinv = next;
          sv_top = PV_TOP / next;
        }
#pragma unroll
        for (int nt = 0; nt < NT; ++nt)
#pragma unroll
          for (int j = 0; j < 2; ++j) {
            float t = tm[nt][j];
#pragma unroll
            for (int x = 4; x < 32; x <<= 1) t = fmaxf(t, __shfl_xor_sync(0xffffffffu, t, x));
            float al = 1.f;
            if (t > up[nt][j]) {  // t is relative to mu
              al = up[nt][j] == -INFINITY ? 0.f : fast_exp2(-t);
              mu[nt][j] += t;
              up[nt][j] = RAISE;
#pragma unroll
              for (int u = 0; u < TP; ++u) {
                sc[u][nt][j] -= t;
                sc[u][nt][2 + j] -= t;
              }
            }
            l[nt][j] *= al;
            ob[nt][j] *= al;
            const float f = al * fv;
#pragma unroll
            for (int n = 0; n < D / 16; ++n) {
              o[nt][n][j] *= f;
              o[nt][n][2 + j] *= f;
            }
            ones[nt][j] *= f;
          }
      }
      // -------------------------------------------------------------- P and sums
      uint32_t pb[TP][NT][SP][2];
#pragma unroll
      for (int u = 0; u < TP; ++u) {
        const float sv0 = sv[u][0] * kinv, sv1 = sv[u][1] * kinv;
#pragma unroll
        for (int nt = 0; nt < NT; ++nt) {
          float pp[4], pq[4];
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            const float p = fast_exp2(sc[u][nt][e]);
            l[nt][e & 1] += p;
            pq[e] = p * bv[u][e >> 1];
            pp[e] = p * (e < 2 ? sv0 : sv1);
          }
          if (need_mask) {  // p = 0 must not meet a NaN that its row does not see
#pragma unroll
            for (int e = 0; e < 4; ++e)
              if (!((vis >> ((u * NT + nt) * 4 + e)) & 1u)) pp[e] = pq[e] = 0.f;
          }
          ob[nt][0] += pq[0] + pq[2];
          ob[nt][1] += pq[1] + pq[3];
#pragma unroll
          for (int hf = 0; hf < 2; ++hf) {
            const uint32_t w = MM::pack(pp[2 * hf], pp[2 * hf + 1]);
            pb[u][nt][0][hf] = movm_trans(w);
            if (SP == 2) {
              const float2 f = __half22float2(*reinterpret_cast<const __half2*>(&w));
              pb[u][nt][SP - 1][hf] =
                  movm_trans(MM::pack(pp[2 * hf] - f.x, pp[2 * hf + 1] - f.y));
            }
          }
          if (C::CENTRE) {
            const uint32_t one[4] = {0x3C003C00u, 0x3C003C00u, 0x3C003C00u, 0x3C003C00u};
            MM::run(ones[nt], one, pb[u][nt][0][0], pb[u][nt][0][1]);
          }
        }
      }
      // ------------------------------------------------------- O^T += V^T P^T
#pragma unroll
      for (int u = 0; u < TP; ++u)
#pragma unroll
        for (int c = 0; c < NL; ++c) {
          uint32_t va[VEC], vb[VEC];
          const uint32_t at = rec[u] + 8 * D + c * 1024 + lane * (4 * VEC);
          lds_words<VEC>(at, va);
          lds_words<VEC>(at + 128 * VEC, vb);
#pragma unroll
          for (int i = 0; i < VEC; ++i) {
            const uint32_t a0[4] = {lo4(va[i]), hi4(va[i]), lo4(vb[i]), hi4(vb[i])};
            const uint32_t va8 = va[i] >> 8, vb8 = vb[i] >> 8;
            const uint32_t a1[4] = {lo4(va8), hi4(va8), lo4(vb8), hi4(vb8)};
#pragma unroll
            for (int nt = 0; nt < NT; ++nt)
#pragma unroll
              for (int sp = 0; sp < SP; ++sp) {
                MM::run(o[nt][2 * (c * VEC + i)], a0, pb[u][nt][sp][0], pb[u][nt][sp][1]);
                MM::run(o[nt][2 * (c * VEC + i) + 1], a1, pb[u][nt][sp][0], pb[u][nt][sp][1]);
              }
          }
        }
      __syncwarp();
      issue(n);
    }

    // --------------------------------------------------- join the four warps' parts
    const bool whole = cc.k0 == 0 && cc.k1 == g.n;
    float* slot = P.part + ((int64_t)blockIdx.x * 2 + (cc.k0 > 0 ? 0 : 1)) * P.part_floats;
#pragma unroll
    for (int nt = 0; nt < NT; ++nt)
#pragma unroll
      for (int j = 0; j < 2; ++j) {
#pragma unroll
        for (int x = 4; x < 32; x <<= 1) {
          l[nt][j] += __shfl_xor_sync(0xffffffffu, l[nt][j], x);
          ob[nt][j] += __shfl_xor_sync(0xffffffffu, ob[nt][j], x);
        }
        if (up[nt][j] == -INFINITY) mu[nt][j] = -INFINITY;  // no key was seen
        if (g4 == 0) ml[warp * R + nt * 8 + 2 * t4 + j] = make_float2(mu[nt][j], l[nt][j]);
      }
    __syncthreads();
    // One warp: each row's common maximum M and sum L, every warp's factor to M.
    for (int row = tid; row < R; row += THREADS) {
      float M = -INFINITY, L = 0.f;
#pragma unroll
      for (int w = 0; w < WARPS; ++w) M = fmaxf(M, ml[w * R + row].x);
#pragma unroll
      for (int w = 0; w < WARPS; ++w) {
        const float2 v = ml[w * R + row];
        const float f = v.x == -INFINITY ? 0.f : fast_exp2(v.x - M);
        L += v.x == -INFINITY ? v.y : v.y * f;  // (a row of NaN scores has no maximum)
        ml[w * R + row].x = f;
      }
      if (whole) {
        ml[row].y = L == 0.f ? 0.f : 1.f / L;
      } else {
        slot[R * D + row] = M;
        slot[R * D + R + row] = L;
      }
    }
    __syncthreads();
    const float inv_k = kinv > 0.f ? 1.f / kinv : 0.f;
#pragma unroll
    for (int nt = 0; nt < NT; ++nt)
#pragma unroll
      for (int half = 0; half < 2; ++half) {  // words [half * NW / 2, + NW / 2) of each thread
#pragma unroll
        for (int j = 0; j < 2; ++j) {
          const int row = 2 * t4 + j;
          const float f = ml[warp * R + nt * 8 + row].x;
          const float add = f * (ob[nt][j] - (C::CENTRE ? 8.f * ones[nt][j] * inv_k : 0.f));
          const float fo = f * C::UNIT * inv_k, fo16 = fo * 0.0625f;
          float* dst = buf + (warp * 8 + row) * C::BUF_LD + g4 * (NW * 2);
#pragma unroll
          for (int i = 0; i < NW / 2; ++i) {
            const float* x0 = o[nt][2 * (half * (NW / 2) + i)];
            const float* x1 = o[nt][2 * (half * (NW / 2) + i) + 1];
            *reinterpret_cast<float4*>(dst + i * 4) =
                make_float4(fmaf(x0[j], fo, add), fmaf(x0[2 + j], fo16, add),
                            fmaf(x1[j], fo, add), fmaf(x1[2 + j], fo16, add));
          }
        }
        __syncthreads();
        for (int idx = tid; idx < 8 * (C::DH / 4); idx += THREADS) {
          const int row = idx / (C::DH / 4), in = idx % (C::DH / 4);
          // thread group in / (NW / 2), its word half * NW / 2 + in % (NW / 2)
          const int wd = half * (NW / 2) + in % (NW / 2);
          const int col = (wd / VEC) * 128 + (in / (NW / 2)) * (4 * VEC) + (wd % VEC) * 4;
          const int rr = cc.rt * R + nt * 8 + row;
          if (rr >= g.q_len * P.G) continue;
          float4 a = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
          for (int w = 0; w < WARPS; ++w) {
            const float4 b =
                *reinterpret_cast<const float4*>(buf + (w * 8 + row) * C::BUF_LD + in * 4);
            a.x += b.x;
            a.y += b.y;
            a.z += b.z;
            a.w += b.w;
          }
          if (whole) {
            const float inv = ml[nt * 8 + row].y;
            T* dst = static_cast<T*>(P.a.out) +
                     (int64_t)map_row(P.a, g.q_start + div_g(P, rr)) * P.a.o_sr +
                     (int64_t)(cc.h * P.G + mod_g(P, rr)) * P.a.o_sh + col;
            alignas(16) T e[4] = {from_f32<T>(a.x * inv), from_f32<T>(a.y * inv), from_f32<T>(a.z * inv),
                      from_f32<T>(a.w * inv)};
            if (P.vec) {
              if constexpr (sizeof(T) == 2)
                *reinterpret_cast<uint2*>(dst) = *reinterpret_cast<uint2*>(e);
              else
                *reinterpret_cast<uint4*>(dst) = *reinterpret_cast<uint4*>(e);
            } else {
#pragma unroll
              for (int i = 0; i < 4; ++i) dst[i] = e[i];
            }
          } else {
            const int pr = nt * 8 + row;
            *reinterpret_cast<float4*>(slot + pr * D + col) = a;
          }
        }
        __syncthreads();
      }
  }
  if (dead) {  // copies in flight still target this CTA's shared memory
    if (lane == 0) set_err(P.a.err, MF_ERR_TIMEOUT);
    for (; taken < issued; ++taken) {
      mbar_wait_bounded(&bar[stage], phase, WAIT_LIMIT);
      if (++stage == NSTG) {
        stage = 0;
        phase ^= 1u;
      }
    }
  }
}

// Joins the partials of units that range borders cut (log-sum-exp identity), one CTA per
// unit, in range order; zeros for rows of sequences without any visible page.  Bound by
// latency: a thread owns one float4 of a row and loads a batch of parts at once.
constexpr int JOIN_THREADS = 256, JOIN_BATCH = 8;

template <typename T, int D, int NT, bool MOD>
__global__ void __launch_bounds__(JOIN_THREADS) join_kernel(const __grid_constant__ Params P,
                                                            int ranges) {
  constexpr int R = 8 * NT;
  grid_dependency_wait();
  const int s = blockIdx.y, u = blockIdx.x;
  const uint32_t total = (uint32_t)__ldcg(P.prefix + P.a.num_seqs);
  const uint32_t first = (uint32_t)__ldcg(P.prefix + s);
  const Geo g = seq_geo<MOD>(P, s, R, false);
  const int rt = P.RT == 1 ? 0 : u / P.a.hkv, h = u - rt * P.a.hkv;
  if (rt >= g.nrt) return;
  int c0 = 0, c1 = 0;
  if (g.n > 0) {
    const Split S = make_split(total, ranges, P.min_tiles);
    const uint32_t start = first + (uint32_t)u * g.n;
    c0 = S.owner(start);
    c1 = S.owner(start + g.n - 1);
    if (c0 == c1) return;  // written whole
  }
  for (int idx = threadIdx.x; idx < R * (D / 4); idx += JOIN_THREADS) {
    const int row = idx / (D / 4), col = (idx % (D / 4)) * 4;
    const int rr = rt * R + row;
    if (rr >= g.q_len * P.G) break;
    float4 a = make_float4(0.f, 0.f, 0.f, 0.f);
    float L = 0.f, M = -INFINITY;
    for (int c = c0; g.n > 0 && c <= c1; c += JOIN_BATCH) {
      float m[JOIN_BATCH], l[JOIN_BATCH];
      float4 b[JOIN_BATCH];
#pragma unroll
      for (int i = 0; i < JOIN_BATCH; ++i) {
        const int ci = min(c + i, c1);
        const float* sl = P.part + ((int64_t)ci * 2 + (ci == c0 ? 1 : 0)) * P.part_floats;
        m[i] = __ldcg(sl + R * D + row);
        l[i] = __ldcg(sl + R * D + R + row);
        b[i] = __ldcg(reinterpret_cast<const float4*>(sl + row * D + col));
      }
      float top = M;
#pragma unroll
      for (int i = 0; i < JOIN_BATCH; ++i) top = fmaxf(top, m[i]);
      const float f0 = M == -INFINITY ? 0.f : fast_exp2(M - top);
      L *= f0;
      a.x *= f0;
      a.y *= f0;
      a.z *= f0;
      a.w *= f0;
      M = top;
#pragma unroll
      for (int i = 0; i < JOIN_BATCH; ++i) {
        if (c + i > c1) break;
        const float f = m[i] == -INFINITY ? 0.f : fast_exp2(m[i] - top);
        L += m[i] == -INFINITY ? l[i] : l[i] * f;  // (a row of NaN scores has no maximum)
        a.x = fmaf(b[i].x, f, a.x);
        a.y = fmaf(b[i].y, f, a.y);
        a.z = fmaf(b[i].z, f, a.z);
        a.w = fmaf(b[i].w, f, a.w);
      }
    }
    const float inv = L == 0.f ? 0.f : 1.f / L;
    T* dst = static_cast<T*>(P.a.out) +
             (int64_t)map_row(P.a, g.q_start + div_g(P, rr)) * P.a.o_sr +
             (int64_t)(h * P.G + mod_g(P, rr)) * P.a.o_sh + col;
    alignas(16) T e[4] = {from_f32<T>(a.x * inv), from_f32<T>(a.y * inv),
                          from_f32<T>(a.z * inv), from_f32<T>(a.w * inv)};
    if (P.vec) {
      if constexpr (sizeof(T) == 2) *reinterpret_cast<uint2*>(dst) = *reinterpret_cast<uint2*>(e);
      else *reinterpret_cast<uint4*>(dst) = *reinterpret_cast<uint4*>(e);
    } else {
#pragma unroll
      for (int i = 0; i < 4; ++i) dst[i] = e[i];
    }
  }
}

}  // namespace q4a

// ------------------------------------------------------------------ host side

namespace {

// Which kernel takes a call's longest runs (the shortest, up to ROWS_CAP rows per kv head, stay
// with mma.sync).  Per 128 keys, mma.sync spends about 10 ns of the whole GPU on a 16-row tile
// of one head, and cuts long contexts over the SMs; the tcgen05 kernel 2.2 us of one SM on a
// 128-row tile, whole contexts at a time, so ragged batches wait for their longest (half as
// much again).  25 rows of 16 sequences, 8 heads: 64 us against 88.
constexpr int ROWS_CAP = 32;
bool chunks_win(int64_t rows, int64_t heads, int sms) {
  const int64_t waves = (heads * ((rows + 127) / 128) + sms - 1) / std::max(sms, 1);
  return rows > ROWS_CAP && heads * ((rows + 15) / 16) >= 340 * waves;
}

struct Plan {
  bool chunks, tiles;  // launch the tcgen05 kernel; launch the mma.sync kernel
  bool expand;         // the tcgen05 kernel reads an expanded copy (at ws + expand_at)
  size_t expand_at;
  Q4Scratch scratch;
  int nt, ranges;
  int64_t rt;
  size_t prefix_bytes, ws_bytes;
  int part_floats;
};

// Row tiles: 8 rows while a run has no more (decode), else 16.  A 32-row tile reads the
// cache half as often but spills and leaves 8 warps on an SM: 25 rows at D = 128 took 71 us
// with it and 64 us in two tiles of 16.  fp32's two-part q and P fit 16 rows at D = 64 only.
int row_tile(int64_t rows, int d, bool f32) { return rows <= 8 || (f32 && d > 64) ? 1 : 2; }

template <typename T_, int D_, int NT_, bool MOD_>
struct Kern {
  using C = q4a::Cfg<T_, D_, NT_>;
  static constexpr int smem = C::SMEM, per_sm = C::MINB;
  static constexpr auto attn = q4a::attn_kernel<T_, D_, NT_, MOD_>;
  static constexpr auto join = q4a::join_kernel<T_, D_, NT_, MOD_>;
};

template <typename T, bool MOD, typename F>
int with_tile(int d, int nt, F&& f) {
  constexpr bool f32 = sizeof(T) == 4;
  if (d == 64 && nt == 1) return f(Kern<T, 64, 1, MOD>{});
  if (d == 64 && nt == 2) return f(Kern<T, 64, 2, MOD>{});
  if (d == 128 && nt == 1) return f(Kern<T, 128, 1, MOD>{});
  if (d == 256 && nt == 1) return f(Kern<T, 256, 1, MOD>{});
  if constexpr (!f32) {
    if (d == 128 && nt == 2) return f(Kern<T, 128, 2, MOD>{});
    if (d == 256 && nt == 2) return f(Kern<T, 256, 2, MOD>{});
  }
  return fail(MF_EUNSUPPORTED, "q4 attention: no kernel for this head_dim and dtype");
}

template <typename F>
int with_kernel(mf_dtype dt, int d, int nt, bool mod, F&& f) {
  if (dt == MF_BF16)
    return mod ? with_tile<__nv_bfloat16, true>(d, nt, f) : with_tile<__nv_bfloat16, false>(d, nt, f);
  if (dt == MF_F16)
    return mod ? with_tile<__half, true>(d, nt, f) : with_tile<__half, false>(d, nt, f);
  return mod ? with_tile<float, true>(d, nt, f) : with_tile<float, false>(d, nt, f);
}

int to_q4_params(const mf_q4_attention_args* a, int32_t* err, q4a::Params& P) {
  if (!a || a->struct_size != sizeof(mf_q4_attention_args))
    return fail(MF_EINVAL, "q4 attention: mf_q4_attention_args size mismatch (ABI version)");
  if (a->num_seqs < 0 || a->total_q < 0 || a->max_q_len < 0 || a->table_stride < 0 ||
      a->table_width < 0 || a->table_width > 0x7fffffff / q4::BLOCK)
    return fail(MF_EINVAL, "q4 attention: negative size");
  if (a->num_q_heads <= 0 || a->num_kv_heads <= 0 || a->num_q_heads % a->num_kv_heads)
    return fail(MF_EINVAL, "q4 attention: query heads must be a positive multiple of kv heads");
  if (!q4::head_dim_ok(a->head_dim))
    return fail(MF_EUNSUPPORTED, "q4 attention: head_dim must be 64, 128 or 256");
  if (a->num_blocks <= 0) return fail(MF_EINVAL, "q4 attention: non-positive num_blocks");
  if (a->dtype != MF_F32 && a->dtype != MF_F16 && a->dtype != MF_BF16)
    return fail(MF_EINVAL, "q4 attention: unknown dtype");
  if (!a->cu_seqlens_q && a->q_per_seq <= 0)
    return fail(MF_EINVAL, "q4 attention: q_per_seq must be positive without cu_seqlens_q");
  if ((reinterpret_cast<uintptr_t>(a->pool) | (uintptr_t)a->pool_stride_block |
       (uintptr_t)a->pool_stride_head) & 15)
    return fail(MF_EINVAL, "q4 attention: pool base and strides must be multiples of 16 bytes");
  if (a->num_seqs > 65535) return fail(MF_EUNSUPPORTED, "q4 attention: more than 65535 sequences");
  if (a->num_seqs > 0 && a->total_q > 0 &&
      (!a->q || !a->out || !a->pool || (!a->block_tables && a->table_width > 0) || !a->kv_lens))
    return fail(MF_EINVAL, "q4 attention: null pointer");
  if (!softcap_ok(a->mods.softcap) || a->mods.window < 0)
    return fail(MF_EINVAL, "q4 attention: softcap must be 0 or from 1e-30 to 1e30, window not "
                           "negative");
  if (!a->cu_seqlens_q && a->total_q > 0 && (int64_t)a->num_seqs * a->q_per_seq > a->total_q)
    return fail(MF_EINVAL, "q4 attention: total_q below num_seqs * q_per_seq");
  if (!scale_ok(a->scale))
    return fail(MF_EINVAL, "q4 attention: scale must be from 1e-9 to 1e9");
  P = q4a::Params{};
  P.a.q = a->q;
  P.a.q_sr = a->q_stride_row;
  P.a.q_sh = a->q_stride_head;
  P.a.out = a->out;
  P.a.o_sr = a->out_stride_row;
  P.a.o_sh = a->out_stride_head;
  P.a.kp = a->pool;
  P.a.sb = a->pool_stride_block;
  P.a.sh = a->pool_stride_head;
  P.a.num_blocks = a->num_blocks;
  P.a.block_size = q4::BLOCK;
  P.a.tables = a->block_tables;
  P.a.table_stride = a->table_stride;
  P.width = a->table_width;
  P.a.cu_q = a->cu_seqlens_q;
  P.a.q_per_seq = a->q_per_seq;
  P.a.kv_lens = a->kv_lens;
  P.a.row_map = a->row_map;
  P.a.num_seqs = a->num_seqs;
  P.a.total_q = a->total_q;
  P.a.max_q_len = a->cu_seqlens_q ? a->max_q_len : a->q_per_seq;
  P.a.hq = a->num_q_heads;
  P.a.hkv = a->num_kv_heads;
  P.a.d = a->head_dim;
  P.a.scale = a->scale;
  P.a.causal = a->causal;
  P.a.err = err;
  P.a.mods = {a->mods.softcap, a->mods.alibi_slopes,
              bounded_window(a->mods.window, P.a.max_q_len), a->mods.prefix_lens};
  P.G = a->num_q_heads / a->num_kv_heads;
  P.g_mul = (uint32_t)(((1ull << 32) + P.G - 1) / P.G);
  if (P.G > 255 || (int64_t)P.a.max_q_len * P.G >= (1 << 24))
    return fail(MF_EUNSUPPORTED, "q4 attention: more than 255 query heads per kv head, or 2^24 "
                                 "rows of a run");
  const int64_t es = a->dtype == MF_F32 ? 4 : 2;
  P.vec = (((reinterpret_cast<uintptr_t>(a->q) | reinterpret_cast<uintptr_t>(a->out)) & 15) == 0 &&
           (a->q_stride_row * es) % 16 == 0 && (a->q_stride_head * es) % 16 == 0 &&
           (a->out_stride_row * es) % 16 == 0 && (a->out_stride_head * es) % 16 == 0);
  return MF_OK;
}

// expand: may long runs read an expanded copy of the cache (else they convert as they go)
Plan make_plan(q4a::Params& P, mf_dtype dt, int sms, bool expand = true) {
  Plan pl{};
  P.rows_cap = 0;
  int64_t rows = (int64_t)P.a.max_q_len * P.G;
  pl.chunks = P.width > 0 && chunks_win(rows, (int64_t)P.a.num_seqs * P.a.hkv, sms) && q4_prefill_serves(P.a, dt);
  pl.expand = expand && pl.chunks && q4_expand_plan(P.a, P.width, P.vec, dt, pl.scratch);
  pl.chunks = pl.chunks && (pl.expand || q4_converting_built());
  pl.tiles = !pl.chunks || P.a.cu_q;  // without offsets every run has max_q_len rows
  if (!pl.tiles) {
    if (pl.expand) pl.ws_bytes = pl.scratch.bytes;
    return pl;
  }
  if (pl.chunks) {
    P.rows_cap = ROWS_CAP;
    rows = std::min<int64_t>(rows, ROWS_CAP);
  }
  pl.nt = row_tile(rows, P.a.d, dt == MF_F32);
  pl.rt = (rows + 8 * pl.nt - 1) / (8 * pl.nt);
  P.RT = (int)pl.rt;
  // Two pages per warp at least: fewer would spend more on joining than on reading.
  P.min_tiles = 2 * q4a::WARPS;
  int per_sm = 1;
  with_kernel(dt, P.a.d, pl.nt, P.a.mods.any(), [&](auto kern) {
    per_sm = decltype(kern)::per_sm;
    return MF_OK;
  });
  const int64_t most = (int64_t)P.a.num_seqs * pl.rt * P.a.hkv * std::max(P.width, 1);
  pl.ranges = (int)std::min<int64_t>((int64_t)sms * per_sm,
                                     std::max<int64_t>((most + P.min_tiles - 1) / P.min_tiles, 1));
  pl.part_floats = 8 * pl.nt * (P.a.d + 2);
  pl.prefix_bytes = ((size_t)(P.a.num_seqs + 1) * 4 + 255) & ~(size_t)255;
  pl.ws_bytes = pl.prefix_bytes + (size_t)pl.ranges * 2 * pl.part_floats * sizeof(float);
  if (pl.expand) {
    pl.expand_at = (pl.ws_bytes + 255) & ~(size_t)255;
    pl.ws_bytes = pl.expand_at + pl.scratch.bytes;
  }
  return pl;
}

}  // namespace
}  // namespace mf

using namespace mf;

static size_t q4_workspace_bytes(const mf_q4_attention_args* args, int device, bool expand) {
  q4a::Params P;
  int sms = 0;
  if (to_q4_params(args, nullptr, P) != MF_OK || P.a.num_seqs == 0 || P.a.total_q == 0 ||
      cudaDeviceGetAttribute(&sms, cudaDevAttrMultiProcessorCount, device) != cudaSuccess)
    return 0;
  return make_plan(P, args->dtype, sms, expand).ws_bytes;
}

extern "C" size_t mf_q4_paged_attention_workspace_size(const mf_q4_attention_args* args,
                                                       int device) {
  return q4_workspace_bytes(args, device, true);
}

extern "C" size_t mf_q4_paged_attention_min_workspace_size(const mf_q4_attention_args* args,
                                                           int device) {
  return q4_workspace_bytes(args, device, false);
}

extern "C" int mf_q4_paged_attention(const mf_q4_attention_args* args, void* workspace,
                                     size_t workspace_bytes, int32_t* err_flag,
                                     mf_stream_t stream) {
  q4a::Params P;
  const int rc = to_q4_params(args, err_flag, P);
  if (rc != MF_OK) return rc;
  if (P.a.num_seqs == 0 || P.a.total_q == 0 || P.a.max_q_len == 0) return MF_OK;
  Plan pl = make_plan(P, args->dtype, current_sm_count());
  if (pl.expand && workspace_bytes < pl.ws_bytes)
    pl = make_plan(P, args->dtype, current_sm_count(), false);
  cudaStream_t s = reinterpret_cast<cudaStream_t>(stream);
  if (pl.tiles && (double)pl.rt * P.a.hkv * P.a.num_seqs * P.width >= 2147483648.0)
    return fail(MF_EUNSUPPORTED, "q4 attention: the tables could hold 2^31 or more (row tile, "
                                 "page) pairs");
  if (pl.ws_bytes > 0 && (!workspace || workspace_bytes < pl.ws_bytes ||
                          (reinterpret_cast<uintptr_t>(workspace) & 15)))
    return fail(MF_EWORKSPACE, "q4 attention: workspace missing, misaligned or smaller than "
                               "mf_q4_paged_attention_min_workspace_size()");
  P.prefix = static_cast<int32_t*>(workspace);
  if (pl.tiles) P.part = reinterpret_cast<float*>(static_cast<uint8_t*>(workspace) + pl.prefix_bytes);
  P.part_floats = pl.part_floats;
  if (pl.chunks) {
    const int rc2 =
        pl.expand ? launch_q4_expanded(P.a, P.width, P.rows_cap, pl.scratch,
                                       static_cast<uint8_t*>(workspace) + pl.expand_at, s)
                  : launch_q4_prefill(P.a, P.width, P.vec, P.rows_cap, s);
    if (rc2 != MF_OK || !pl.tiles) return rc2;
  }
  return with_kernel(
      args->dtype, P.a.d, pl.nt, P.a.mods.any(), [&](auto kern) -> int {
        using Kn = decltype(kern);
        static thread_local int ready = -1;  // the device this kernel was last set up on
        int dev = 0;
        cudaGetDevice(&dev);
        if (ready != dev) {
          const cudaError_t e = cudaFuncSetAttribute(
              Kn::attn, cudaFuncAttributeMaxDynamicSharedMemorySize, Kn::smem);
          if (e != cudaSuccess)
            return fail(MF_ECUDA, std::string("q4 attention: ") + cudaGetErrorString(e));
          ready = dev;
        }
        cudaLaunchAttribute attr[1];
        attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
        attr[0].val.programmaticStreamSerializationAllowed = 1;
        cudaLaunchConfig_t cfg = {};
        cfg.gridDim = dim3((unsigned)pl.ranges);
        cfg.blockDim = dim3(q4a::THREADS);
        cfg.dynamicSmemBytes = (size_t)Kn::smem;
        cfg.stream = s;
        cfg.attrs = attr;
        cfg.numAttrs = 1;
        cudaError_t e = cudaLaunchKernelEx(&cfg, Kn::attn, P);
        if (e == cudaSuccess) {
          cfg.gridDim = dim3((unsigned)(pl.rt * P.a.hkv), (unsigned)P.a.num_seqs);
          cfg.blockDim = dim3(q4a::JOIN_THREADS);
          cfg.dynamicSmemBytes = 0;
          e = cudaLaunchKernelEx(&cfg, Kn::join, P, pl.ranges);
        }
        if (e != cudaSuccess)
          return fail(MF_ECUDA, std::string("q4 attention: ") + cudaGetErrorString(e));
        return check_launch("q4 attention");
      });
}
