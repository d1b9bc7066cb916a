// Paged chunked-prefill attention on the sm_100a tensor cores (tcgen05 + TMEM).
//
// Persistent: one CTA per SM walks a list of work items, each one 128-row
// query tile of one sequence for one kv head.  The 128 rows are (query
// position, query head of the GQA group) pairs, so each K/V tile is loaded once
// for every query head sharing the kv head.
//
//   warps 0..4*WPQ-1  softmax and epilogue: warp w reads TMEM lanes 32 (w % 4) ..
//              (tile rows) and columns [CW (w / 4), CW (w / 4 + 1)) of S, P and O;
//              the WPQ warps of one lane quarter combine their partial row maxima
//              (and, at the end, row sums) through shared memory
//   next 2     TMA producer warps: Q (two buffers) and K, and V; per 128-key
//              tile 8 pages x 2 halves (4-D tiled loads from the pool, 128-byte
//              swizzled), one box per lane, into two-stage K and V rings
//   next warp  S issuer (one thread): S = Q K^T into one of two TMEM S buffers
//   last warp  P V issuer (one thread): O += P V with P read from one of two
//              TMEM P buffers
//
// tcgen05.mma issue returns only as the tensor pipe takes the instruction, so
// one thread issuing everything would leave the pipe idle whenever it waits
// (for a P, a K tile, a free buffer).  Two issuers, one per product, let each
// keep the pipe busy while the other waits.
//
// TMEM (512 columns): S_a S_b (128 fp32 each), P_a P_b (64 columns of packed
// 16-bit pairs each), O (128 fp32).  P does not alias S, so an S buffer is free
// again as soon as the softmax warps have loaded it: the S of a tile can be
// computed while the softmax of the previous tile runs.
//
// Each lane quarter has two softmax warps that take alternate key tiles, so one
// warp's TMEM load, row max and P store overlap the other's exponentials.  An
// item's epilogue (combining the two warps' row sums, normalising O, storing)
// is deferred past each warp's first tile of the next item, so the tensor pipe
// is not idle while O is read out.
//
// The online softmax keeps a per-row reference max (log2 units) and only
// rescales O (a TMEM read-modify-write) when a tile's max exceeds it by more
// than 2^8, so the exponentials stay <= 256 and the correction is rare after the
// first tiles.  Masking: key k is visible to row r iff k < kv_len and k <=
// kv_len - q_len + position(r) (causal) — the varlen rule of
// memforge_ml/kernels/varlen_attention.py:193-201.  Pages past the block table
// load as zeros (out-of-range TMA coordinates) and unwritten slots of the last
// page are zeroed in shared memory before the P V product.
//
// MOD instances apply score modifiers (mf_score.cuh) to S as it is read from TMEM.  Key
// tiles that no row of a query tile sees (between the prefix and the window) are left
// out, and so are the pages of a tile that lie behind the window.  The cap is a
// polynomial while a warp's scores stay below 3/4 of it (3.5 packed instructions per
// score, where the exponential and the reciprocal would add two SFU operations to the
// softmax's one), else softcap_large_log2.
//
// Every mbarrier wait is bounded; on expiry the CTA raises MF_ERR_TIMEOUT, drains
// its TMA loads and MMAs, frees its TMEM and returns.

#pragma once

#include "mf_attn.h"
#include "mf_q4.cuh"

namespace mf {
namespace pf {

constexpr int BM = 128;
constexpr int BN = 128;
constexpr int WPQ = 2;                  // softmax warps per TMEM lane quarter (tile parities)
constexpr int SM_WARPS = 4 * WPQ;       // softmax warps
constexpr int TILE_WARPS = 4;           // softmax warps working on one tile (one per quarter)
constexpr int CW = BN;                  // score columns per softmax warp (all of its tiles)
constexpr int TMA_WARP = SM_WARPS, V_WARP = SM_WARPS + 1, MMA_WARP = SM_WARPS + 2,
              PV_WARP = SM_WARPS + 3;
constexpr int THREADS = (SM_WARPS + 4) * 32;
// Q4: after the softmax warps the two issuers and the warp that loads records (and one
// idle), then four warps that bring Q and convert K and four that convert V.
constexpr int Q4_MMA_WARP = SM_WARPS, Q4_PV_WARP = SM_WARPS + 1, Q4_LOAD_WARP = SM_WARPS + 2,
              Q4_K_WARP = SM_WARPS + 4, Q4_V_WARP = SM_WARPS + 8;
constexpr int Q4_CW = 4;  // converter warps of each kind
constexpr int Q4_THREADS = (SM_WARPS + 4 + 2 * Q4_CW) * 32;
// Registers: 640 threads start with 96 each; 256 * 168 + 384 * 48 is the same sum (the
// plan checks that the kernel was built with 96).
constexpr int Q4_REGS_LAUNCH = 96, Q4_REGS_SOFTMAX = 168, Q4_REGS_REST = 48;
static_assert(Q4_THREADS * Q4_REGS_LAUNCH ==
                  SM_WARPS * 32 * Q4_REGS_SOFTMAX + (Q4_THREADS - SM_WARPS * 32) * Q4_REGS_REST,
              "register split");

static_assert(CW == 32 || CW == 64 || CW == 128, "softmax column split");
constexpr int D = 128;
constexpr int PAGE = q4::BLOCK;
constexpr int KS = 2;  // K and V ring stages
constexpr int MAX_SEQS = 4096;
constexpr uint32_t TMEM_COLS = 512;
constexpr uint64_t WAIT_LIMIT = 2000000000ull;
constexpr float RESCALE_THRESHOLD = 8.0f;  // log2 units

constexpr uint32_t TILE_BYTES = BN * D * 2;   // 32 KB: [half][128 rows][128 B]
constexpr uint32_t HALF_BYTES = BN * 128;     // 16 KB
constexpr uint32_t OFF_Q = 0;
constexpr int RAW = 3;  // Q4: ring of key tiles as records
constexpr uint32_t RAW_BYTES = (BN / PAGE) * q4::record_bytes(D);
// Q buffers: two, or with Q4 one, whose space the records take (the next item's Q is
// brought while the softmax of this one's last two tiles runs).
__host__ __device__ constexpr int q_buffers(bool q4) { return q4 ? 1 : 2; }
__host__ __device__ constexpr uint32_t off_k(bool q4) { return OFF_Q + q_buffers(q4) * TILE_BYTES; }
__host__ __device__ constexpr uint32_t off_v(bool q4) { return off_k(q4) + KS * TILE_BYTES; }
__host__ __device__ constexpr uint32_t off_raw() { return off_v(true) + KS * TILE_BYTES; }
__host__ __device__ constexpr uint32_t off_bar(bool q4) {
  return q4 ? off_raw() + RAW * RAW_BYTES : off_v(false) + KS * TILE_BYTES;
}

// mbarrier indices
// S_DONE[b] (the S of tile g completed, b = g & 1) also frees K ring stage
// g % KS, and PV_DONE[b] (the P V of tile g completed) also frees P buffer b and
// V ring stage g % KS: with two stages the indices coincide, so one commit
// serves both waiters.
static_assert(KS == 2, "ring stages double as S / P buffer indices");
constexpr int B_QFULL = 0, B_QEMPTY = 2, B_KFULL = 4, B_VFULL = B_KFULL + KS,
              B_SDONE = B_VFULL + KS, B_SFREE = B_SDONE + 2, B_PFULL = B_SFREE + 2,
              B_PVDONE = B_PFULL + 2,
              B_OFULL = B_PVDONE + 2, B_OFREE = B_OFULL + 1, B_IDLE = B_OFREE + 1,
              B_HAND = B_IDLE + 1, B_EXL = B_HAND + 8, B_RFULL = B_EXL + 4,
              B_REMPTY = B_RFULL + RAW;
__host__ __device__ constexpr uint32_t off_misc(bool q4) {  // TMEM base, abort flag
  return off_bar(q4) + (q4 ? B_REMPTY + RAW : B_RFULL) * 8;
}
// Row statistics passed between the two softmax warps of a lane quarter:
// m[2 parities][BM] (the reference max after a tile), then l[2 items][2
// parities][BM] and ms[2 items][2 parities][BM] (an item's partial row sums and
// the reference max they are scaled to).
__host__ __device__ constexpr uint32_t off_xch(bool q4) { return (off_misc(q4) + 16 + 15) & ~15u; }
// Work-list tables: prefix int[num_seqs + 1] (query tiles before the k-th
// sequence in longest-first order), order uint16[num_seqs] (that sequence), and
// NBK bucket counters of the counting sort.
constexpr int NBK = 256;

// TMEM column offsets
constexpr uint32_t COL_S = 0, COL_P = 256, COL_O = 384;

// Q4: a power of two per tile row that q was multiplied by (its inverse, in the softmax's
// units), for four items: its writers run at most two ahead of the softmax.
__host__ __device__ constexpr uint32_t off_qs() { return off_xch(true) + 10 * BM * 4; }
__host__ __device__ constexpr uint32_t off_prefix(bool q4) {
  return off_xch(q4) + 10 * BM * 4 + (q4 ? 4 * BM * 4 : 0u);
}
__host__ __device__ constexpr uint32_t off_order(int num_seqs, bool q4) {
  return off_prefix(q4) + (((uint32_t)(num_seqs + 1) * 4u + 15u) & ~15u);
}
__host__ __device__ constexpr uint32_t off_counts(int num_seqs, bool q4) {
  return off_order(num_seqs, q4) + (((uint32_t)num_seqs * 2u + 15u) & ~15u);
}
__host__ __device__ constexpr uint32_t smem_bytes(int num_seqs, bool q4 = false) {
  return off_counts(num_seqs, q4) + NBK * 4u;
}
constexpr int Q4_MAX_SEQS = 1024;
static_assert(smem_bytes(MAX_SEQS) + 1024 <= 227u * 1024u, "shared memory budget");
static_assert(smem_bytes(Q4_MAX_SEQS, true) + 1024 <= 227u * 1024u, "shared memory budget (Q4)");

// Sort key of a sequence: about 8 buckets per doubling of kv_len, longest first
// (bucket 0); sequences without work last.
MF_DEVINL int length_bucket(int kv_len, int tiles) {
  if (tiles == 0 || kv_len <= 0) return NBK - 1;
  const int e = 31 - __clz(kv_len);
  const int mant = e >= 3 ? (kv_len >> (e - 3)) & 7 : (kv_len << (3 - e)) & 7;
  return NBK - 2 - min(8 * e + mant, NBK - 2);
}

// Verify items (a window: one query tile per sequence in practice) sort by
// their exact key-tile count, so the snake deal pairs long and short items
// as closely as the counts allow; other items by length_bucket.
template <typename PP>
MF_DEVINL int sort_bucket(const PP& P, int kv_len, int q_len, int tiles) {
  if (!P.window || tiles == 0 || kv_len <= 0) return length_bucket(kv_len, tiles);
  const int nt = (kv_len - q_len + BN - 1) / BN + 1;
  return NBK - 2 - min(nt, NBK - 2);
}

// Work item handled by this CTA in its k-th step: items are dealt to the CTAs
// in a snake order (0..G-1, then G-1..0, ...), so that with the longest items
// first the CTAs that get the longest of one pass get the shortest of the next.
MF_DEVINL int snake_item(int k) {
  const int G = gridDim.x, c = blockIdx.x;
  return k * G + ((k & 1) ? G - 1 - c : c);
}

struct Params {
  AttnParams a;
  int G;
  int rows_cap;      // sequences with q_len * G <= rows_cap belong to the decode kernel
  float scale_log2;
  uint32_t in_fmt;   // 0 = f16, 1 = bf16
  int window;        // 1: the last q_len keys of each sequence come from the window buffers
  int width;         // Q4, EXP: entries of a block table's row
  int vec;           // Q4: q and out rows allow 16-byte accesses
  const float* qs;   // EXP: per (row, query head), what scales S to log2 units
  // softcap in log2 units, its inverse, 2 / softcap: divided on the host, where it costs the
  // tile loop no registers (689 against 713 us for 2 x 2048 rows, 6000..8192 keys, cap 30)
  float cap2, inv_cap2, two_over;

  // The scale and the cap of the call.
  void set_scores() {
    scale_log2 = a.scale * kLog2e;
    cap2 = a.mods.softcap * kLog2e;
    inv_cap2 = a.mods.softcap > 0.f ? 1.f / cap2 : 0.f;
    two_over = a.mods.softcap > 0.f ? 2.f / a.mods.softcap : 0.f;
  }
};

// Geometry of one work item (identical in every role).
struct Item {
  int s, h, q_start, q_len, kv_len, win_start, pos0, nt;
  int pool_len;  // keys read from the pool (the rest, with a window, from the window buffers)
  int pfx, pt, gap, lo;  // MOD: prefix keys and tiles, tiles left out after them, first
                         // key that row 0 of the tile sees through the window

  template <bool MOD>
  MF_DEVINL int tile(int j) const { return !MOD || j < pt ? j : j + gap; }
  template <bool MOD>
  MF_DEVINL bool page_live(int page) const {
    return !MOD || page * PAGE + PAGE - 1 >= lo || page * PAGE < pfx;
  }
};

// Query positions per tile: the tile's rows are (position, query head) pairs,
// floor(128 / G) positions x G heads (the rows past that are padding).
__host__ __device__ constexpr int positions_per_tile(int G) { return BM / G; }

MF_DEVINL int find_tile_seq(const int* prefix, int B, int t) {
  int lo = 0, hi = B;  // prefix[lo] <= t < prefix[hi]
  while (hi - lo > 1) {
    const int mid = (lo + hi) >> 1;
    if (prefix[mid] <= t) lo = mid; else hi = mid;
  }
  return lo;
}

// Items run longest first: sequences by decreasing kv_len, and within a
// sequence the last query tiles (which see the most keys) first.
template <bool MOD, bool Q4>  // Q4: of a 4-bit cache (in either form)
MF_DEVINL Item item_at(const Params& P, const int* prefix, const uint16_t* order, int B,
                       int it) {
  Item I;
  const int hkv = P.a.hkv;
  const int t = it / hkv;
  I.h = it % hkv;
  const int k = find_tile_seq(prefix, B, t);
  I.s = order[k];
  const int qt = prefix[k + 1] - 1 - t;
  seq_rows(P.a, I.s, I.q_start, I.q_len);
  I.kv_len = __ldg(P.a.kv_lens + I.s);
  if (Q4) I.q_len = min(I.q_len, P.a.max_q_len);
  I.win_start = I.kv_len - I.q_len;
  const int ppt = positions_per_tile(P.G);
  I.pos0 = qt * ppt;
  const int pos_last = min(I.q_len - 1, I.pos0 + ppt - 1);
  I.pfx = I.pt = I.gap = I.lo = 0;
  if constexpr (MOD || Q4) {
    const ScoreMods& md = P.a.mods;
    I.pool_len = Q4 ? min(I.kv_len, P.width * PAGE) : I.kv_len;
    if (MOD && md.prefix) I.pfx = min(max(__ldg(md.prefix + I.s), 0), I.pool_len);
    if (MOD && md.window > 0) I.lo = max(I.win_start + I.pos0 - md.window + 1, 0);
    I.pt = (I.pfx + BN - 1) / BN;
    const int end = P.a.causal ? min(I.win_start + pos_last + 1, I.pool_len) : I.pool_len;
    const int all = (max(max(end, I.pfx), 0) + BN - 1) / BN;
    I.gap = max(min(I.lo / BN, all) - I.pt, 0);
    I.nt = max(all - I.gap, 1);  // a tile without any key still writes its rows
    // Hidden from the compiler: knowing that the loop over key tiles runs at least once, it moves
    // the item's values into registers that the softmax needs (200 against 16 bytes of spills in
    // the EXP kernel; 787 against 665 us for four chunks of 300..2048 rows, 32/8 heads).
    asm("" : "+r"(I.nt));
  } else if (P.window) {
    // Pool tiles for positions < kv_len - q_len, then one tile holding the
    // window (q_len <= 16 keys) in its first rows.
    I.pool_len = I.win_start;
    I.nt = (I.pool_len + BN - 1) / BN + 1;
  } else {
    I.pool_len = I.kv_len;
    const int key_end = I.win_start + pos_last + 1;  // keys this tile can see
    I.nt = (key_end + BN - 1) / BN;
  }
  return I;
}

// tanh(y) / y as polynomials in y^2: least maximum of |tanh| error (Lawson's reweighted
// least squares), 4.9e-08 up to |y| = 1/4 and 1.9e-7 up to 3/4.
constexpr float CAP_MAX1 = 0.25f, CAP_MAX2 = 0.75f;
constexpr float CAP1[3] = {0.9999986329817142f, -0.3331570152146305f,
                           0.1276223146927044f};
constexpr float CAP2[5] = {0.9999972283095431f, -0.33323076454511924f, 0.1322609142435701f,
                           -0.04928044211128824f, 0.01231882752544035f};

// sv = capped scores in log2 units, of raw scores (times sl2: log2 units).  The polynomial's
// factors take in sl2 and the cap, so the short one is four packed operations a pair; the
// largest score of the warp's rows decides, and that its factors are finite: under a cap far
// below any score (1e-12, say) they are not, and a score of 0 would come out as NaN.
template <int N>
MF_DEVINL void cap_scores(const Params& P, float* sv, float sl2) {
  const float ky = fminf(sl2 * P.inv_cap2, 1e30f);
  float top[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
  for (int c = 0; c < N; c += 2)
    top[(c >> 1) & 3] = fmax3f(top[(c >> 1) & 3], fabsf(sv[c]), fabsf(sv[c + 1]));
  const float mx = fmaxf(fmaxf(top[0], top[1]), fmaxf(top[2], top[3])) * ky;
  const float k2 = ky * ky;
  const float f0 = CAP1[0] * sl2, f1 = CAP1[1] * sl2 * k2, f2 = CAP1[2] * sl2 * k2 * k2;
  if (!__any_sync(0xffffffffu, mx > CAP_MAX1 || f2 > 1e38f)) {
    const uint64_t c0 = f32x2(f0, f0), c1 = f32x2(f1, f1), c2 = f32x2(f2, f2);
#pragma unroll
    for (int c = 0; c < N; c += 2) {
      const uint64_t v = f32x2(sv[c], sv[c + 1]), u = f32x2_mul(v, v);
      f32x2_split(f32x2_mul(v, f32x2_fma(u, f32x2_fma(u, c2, c1), c0)), sv[c], sv[c + 1]);
    }
  } else if (__any_sync(0xffffffffu, mx > CAP_MAX2)) {
#pragma unroll
    for (int c = 0; c < N; ++c)  // exp(2 s / cap) = 2^(2 log2(e) s2 / cap2)
      sv[c] = softcap_large_log2(sv[c] * sl2, P.cap2, P.two_over);
  } else {
    const uint64_t k2 = f32x2(ky, ky), s2 = f32x2(P.cap2, P.cap2);
    const uint64_t c0 = f32x2(CAP2[0], CAP2[0]), c1 = f32x2(CAP2[1], CAP2[1]),
                   c2 = f32x2(CAP2[2], CAP2[2]), c3 = f32x2(CAP2[3], CAP2[3]),
                   c4 = f32x2(CAP2[4], CAP2[4]);
#pragma unroll
    for (int c = 0; c < N; c += 2) {
      const uint64_t y = f32x2_mul(f32x2(sv[c], sv[c + 1]), k2), u = f32x2_mul(y, y);
      uint64_t t = f32x2_fma(u, c4, c3);
      t = f32x2_fma(u, t, c2);
      t = f32x2_fma(u, t, c1);
      t = f32x2_fma(u, t, c0);
      f32x2_split(f32x2_mul(f32x2_mul(y, s2), t), sv[c], sv[c + 1]);
    }
  }
}

// ---------------------------------------------- Q4: operands from 4-bit records
// A word's codes as fp16 integers n: pairs (n0, n4), (n1, n5), (n2, n6), (n3, n7).  Under
// the exponent of 1024 the masks give 1024 + n and 1024 + 16 n, both exact.
MF_DEVINL uint32_t half2_fma(uint32_t a, uint32_t b, uint32_t c) {
  uint32_t r;
  asm("fma.rn.f16x2 %0, %1, %2, %3;" : "=r"(r) : "r"(a), "r"(b), "r"(c));
  return r;
}
MF_DEVINL void code_pairs(uint32_t w, uint32_t* p) {
  constexpr uint32_t K1024 = 0x64006400u, SIXTEENTH = 0x2C002C00u, M64 = 0xD400D400u;
#pragma unroll
  for (int i = 0; i < 2; ++i) {
    const uint32_t v = w >> (8 * i);
    asm("sub.rn.f16x2 %0, %1, %2;" : "=r"(p[2 * i]) : "r"((v & 0x000F000Fu) | K1024), "r"(K1024));
    p[2 * i + 1] = half2_fma((v & 0x00F000F0u) | K1024, SIXTEENTH, M64);
  }
}
MF_DEVINL uint32_t half2_max(uint32_t a, uint32_t b) {  // (a NaN is passed over)
  uint32_t r;
  asm("max.f16x2 %0, %1, %2;" : "=r"(r) : "r"(a), "r"(b));
  return r;
}
// Whether 15 * scale + base can pass fp16's largest number, of (scale, base) or the largest of
// several; such values are then held to that number.  Only a row that reaches it has them:
// scale's rounding up takes its largest code at most 120 past its largest value.
MF_DEVINL bool past_range(uint32_t params) {
  const float2 p = __half22float2(*reinterpret_cast<const __half2*>(&params));
  return fmaf(15.f, p.x, p.y) > 65504.f;
}
// A value row of NaN must not enter P V, where the weight 0 of a row that does not see it would
// make a NaN of it: the value becomes zeros and its key NaN instead, and the scores, which are
// masked row by row, carry it to the rows that see it.
MF_DEVINL bool nan_row(uint32_t params) {  // (scale, base) not both finite
  const uint32_t inf = 0x7C007C00u;
  return !__hblt2(__habs2(*reinterpret_cast<const __half2*>(&params)),
                  *reinterpret_cast<const __half2*>(&inf));
}
MF_DEVINL uint32_t key_params(uint32_t key, uint32_t value) {
  return nan_row(value) ? 0x7E007E00u : key;
}
MF_DEVINL uint32_t held(uint32_t v) {
  asm("min.NaN.f16x2 %0, %0, %1;" : "+r"(v) : "r"(0x7BFF7BFFu));
  return v;
}
MF_DEVINL void lds128(uint32_t addr, uint32_t* v) {
  asm volatile("ld.shared.v4.u32 {%0,%1,%2,%3}, [%4];"
               : "=r"(v[0]), "=r"(v[1]), "=r"(v[2]), "=r"(v[3])
               : "r"(addr)
               : "memory");
}
MF_DEVINL void sts128(uint32_t addr, uint32_t a, uint32_t b, uint32_t c, uint32_t d) {
  asm volatile("st.shared.v4.u32 [%0], {%1, %2, %3, %4};" ::"r"(addr), "r"(a), "r"(b), "r"(c),
               "r"(d)
               : "memory");
}
// 16-byte chunk c (0..15: dims 8c .. 8c+7) of row r of an operand tile.
MF_DEVINL uint32_t chunk_at(uint32_t tile, int r, int c) {
  return tile + (c >> 3) * HALF_BYTES + r * 128 + (((c & 7) ^ (r & 7)) << 4);
}

// The records of every key tile into the raw ring: lane l < 8 of one warp fetches page l with
// an untiled bulk copy.  Pages without a token, or behind every row's window, are not
// fetched; the converters never use their slots.
template <bool MOD>
MF_DEVINL void q4_load(const Params& P, const int* prefix, const uint16_t* order, int items,
                       uint32_t base, uint64_t* bar, volatile int* abort_flag, int lane) {
  constexpr int PAGES = BN / PAGE, REC = q4::record_bytes(D);
  const uint64_t pol = l2_evict_last_policy();  // the item's other row tiles read it again
  const uint8_t* pool = static_cast<const uint8_t*>(P.a.kp);
  const int nb = P.a.num_blocks;
  uint32_t g = 0, armed = 0;
  bool run = true;
  for (int k = 0; run && snake_item(k) < items; ++k) {
    const Item I = item_at<MOD, true>(P, prefix, order, P.a.num_seqs, snake_item(k));
    const int32_t* table = P.a.tables + (int64_t)I.s * P.a.table_stride;
    const int pages = (I.pool_len + PAGE - 1) / PAGE;
    const uint8_t* head = pool + (int64_t)I.h * P.a.sh;
    auto block_of = [&](int j) {  // of this lane's page, one tile ahead; -1: not fetched
      const int L = I.template tile<MOD>(j) * PAGES + lane;
      if (lane >= PAGES || L >= pages || !I.template page_live<MOD>(L)) return -1;
      const int id = __ldg(table + L);
      if (id >= 0 && id < nb) return id;
      set_err(P.a.err, MF_ERR_BLOCK_ID);
      return 0;
    };
    int nxt = block_of(0);
    for (int j = 0; j < I.nt; ++j, ++g) {
      const int blk = nxt, st = g % RAW;
      if (j + 1 < I.nt) nxt = block_of(j + 1);
      const uint32_t n = __popc(__ballot_sync(0xffffffffu, blk >= 0));
      bool fine = true;
      if (lane == 0) {
        if (g >= RAW && !mbar_wait_bounded(&bar[B_REMPTY + st], ((g / RAW) - 1) & 1, WAIT_LIMIT)) {
          set_err(P.a.err, MF_ERR_TIMEOUT);
          *abort_flag = 1;
        }
        fine = !*abort_flag;
        if (fine && n) mbar_arrive_expect_tx(&bar[B_RFULL + st], n * REC);
        if (fine && !n) mbar_arrive(&bar[B_RFULL + st]);
      }
      run = __shfl_sync(0xffffffffu, fine, 0);  // also orders expect_tx before the copies
      if (!run) break;
      armed = g + 1;
      if (blk >= 0)
        asm volatile(
            "cp.async.bulk.shared::cluster.global.mbarrier::complete_tx::bytes.L2::cache_hint "
            "[%0], [%1], %2, [%3], %4;" ::"r"(base + off_raw() + st * RAW_BYTES + lane * REC),
            "l"(head + (int64_t)blk * P.a.sb), "r"(REC), "r"(smem_u32(&bar[B_RFULL + st])), "l"(pol)
            : "memory");
    }
  }
  // No copy may still target shared memory at the exit.
  if (lane == 0)
    for (uint32_t k = armed > (uint32_t)RAW ? armed - RAW : 0u; k < armed; ++k)
      if (!mbar_wait_bounded(&bar[B_RFULL + k % RAW], (k / RAW) & 1, WAIT_LIMIT))
        set_err(P.a.err, MF_ERR_TIMEOUT);
}

// The Q tile of one item, by the K warps (ts: thread of the 128; 16 lanes a row, 16 rows a
// warp): rows in fp16, times the power of two that brings a row's largest element to
// [2^14, 2^15) (exact for bf16 and fp16 elements down to 2^-28 of it); its inverse goes to the
// softmax.  Rows without a query are zeros.  The rows are copied asynchronously to their places
// in the tile and converted there by the threads that copied them, in rolled loops: code that
// runs once an item comes from far in the instruction cache, so less of it is faster (unrolled
// over registers this took 10 us an item).
MF_DEVINL int q4_q_row(int it, int ts) { return (it * Q4_CW + (ts >> 5)) * 2 + ((ts & 31) >> 4); }

template <typename T>
MF_DEVINL void q4_stage_q(const Params& P, const Item& I, uint32_t tile, float* qs, int ts) {
  const int c = ts & 15;
  const int rows = positions_per_tile(P.G) * P.G;
  const uint32_t inv = 65536u / (uint32_t)P.G + 1u;  // r / G = r * inv >> 16 for r < 128
  const T* q = static_cast<const T*>(P.a.q) + c * 8;
#pragma unroll 1
  for (int it = 0; it < BM / (2 * Q4_CW); ++it) {
    const int r = q4_q_row(it, ts);
    const int in = (int)((uint32_t)r * inv >> 16), pos = I.pos0 + in;
    const uint32_t dst = chunk_at(tile, r, c);
    if (r < rows && pos < I.q_len) {
      const T* p = q + (int64_t)map_row(P.a, I.q_start + pos) * P.a.q_sr +
                   (int64_t)(I.h * P.G + (r - in * P.G)) * P.a.q_sh;
      if (P.vec) {
        asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(dst), "l"(p) : "memory");
      } else {
        const uint16_t* e = reinterpret_cast<const uint16_t*>(p);
        sts128(dst, e[0] | (uint32_t)e[1] << 16, e[2] | (uint32_t)e[3] << 16,
               e[4] | (uint32_t)e[5] << 16, e[6] | (uint32_t)e[7] << 16);
      }
    } else {
      sts128(dst, 0, 0, 0, 0);
    }
  }
  asm volatile("cp.async.wait_all;" ::: "memory");
#pragma unroll 1
  for (int it = 0; it < BM / (2 * Q4_CW); ++it) {
    const int r = q4_q_row(it, ts);
    const uint32_t dst = chunk_at(tile, r, c);
    uint32_t raw[4];
    lds128(dst, raw);
    const T* t = reinterpret_cast<const T*>(raw);
    float x[8];
#pragma unroll
    for (int e = 0; e < 8; ++e) x[e] = Elt<T>::to_f32(t[e]);
    // (a NaN is passed over; with an infinity the row's output is NaN whatever the factor)
    float top = fmaxf(fmax3f(fabsf(x[0]), fabsf(x[1]), fabsf(x[2])),
                      fmax3f(fabsf(x[3]), fabsf(x[4]), fmax3f(fabsf(x[5]), fabsf(x[6]), fabsf(x[7]))));
#pragma unroll
    for (int o = 1; o < 16; o <<= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, o));
    const int ex = (int)(__float_as_uint(top) >> 23);
    const float mul = __uint_as_float((uint32_t)min(max(268 - ex, 1), 240) << 23);
    if (c == 0) qs[r] = P.scale_log2 / mul;
#pragma unroll
    for (int e = 0; e < 8; ++e) x[e] *= mul;
    sts128(dst, Mma<__half>::pack(x[0], x[4]), Mma<__half>::pack(x[1], x[5]),
           Mma<__half>::pack(x[2], x[6]), Mma<__half>::pack(x[3], x[7]));
  }
}

// K or V of every tile, by four warps; ts: thread of the 128, which take the pages of a tile
// two at a time.  The K warps bring an item's Q after its first K tile.  Codes become
// n * scale + base in fp16 with one rounding: scale and base are multiples of 2^-24, so it is off
// by at most 2^-11 of the value, and subnormal values are exact.  They are stored as the swizzled
// tile the MMA reads.  Keys without a token (or behind every row's window) become zeros, whatever
// their slots hold.  K's dims stay in the order the masks give inside each group of eight
// (0 4 1 5 2 6 3 7); q is stored in the same order.
template <typename T, bool MOD, bool V>
MF_DEVINL void q4_stage(const Params& P, const int* prefix, const uint16_t* order, int items,
                        uint32_t base, float* qs, uint64_t* bar, volatile int* abort_flag,
                        int ts0) {
  constexpr int PAGES = BN / PAGE, REC = q4::record_bytes(D);
  constexpr int UN = 1;  // pages in flight; the loop stays rolled (see above)
  const int lane = ts0 & 31, ts = ts0 & 63, first = ts0 >> 6;
  const uint32_t ring = base + (V ? off_v(true) : off_k(true));
  uint64_t* fullb = &bar[V ? B_VFULL : B_KFULL];
  uint64_t* emptyb = &bar[V ? B_PVDONE : B_SDONE];
  // This thread's rows in a page: K one (dims 32 q .. +31), V two (dims 16 q .. +15).  Half the
  // lanes (up) take their two 8-byte halves in the other order, so that the chunks of one
  // store instruction fall on different banks.
  const int r0 = V ? (ts >> 5) * 8 + 2 * (ts & 3) : ts >> 2;
  const int q = V ? (ts & 31) >> 2 : ts & 3;
  const int up = V ? q & 1 : q >> 1;
  const uint32_t code_off = (V ? 8 * D : 0) + ts * 16 + up * 8;
  const uint32_t par_off = 16 * D + (V ? 64 : 0) + r0 * 4;
  // Stores of a page: K words 0 .. 3 (of this lane's order), V (half, token).
  uint32_t at[4];
#pragma unroll
  for (int c = 0; c < 4; ++c)
    at[c] = V ? chunk_at(0, r0 + (c & 1), q * 2 + ((c >> 1) ^ up))
              : chunk_at(0, r0, q * 4 + (c ^ (2 * up)));
  uint32_t g = 0;
  int ic = 0;
  for (int k = 0; snake_item(k) < items; ++k, ++ic) {
    const Item I = item_at<MOD, true>(P, prefix, order, P.a.num_seqs, snake_item(k));
    for (int j = 0; j < I.nt; ++j, ++g) {
      const int st = g % KS, rs = g % RAW;
      const int key0 = I.template tile<MOD>(j) * BN + r0;
      bool fine = mbar_wait_bounded(&bar[B_RFULL + rs], (g / RAW) & 1, WAIT_LIMIT);
      if (g >= KS) fine = fine && mbar_wait_bounded(&emptyb[st], ((g / KS) - 1) & 1, WAIT_LIMIT);
      if (!__all_sync(0xffffffffu, fine && !*abort_flag)) {
        if (!fine) set_err(P.a.err, MF_ERR_TIMEOUT);
        *abort_flag = 1;
        return;
      }
      const uint32_t tile = ring + st * TILE_BYTES + first * PAGE * 128;
      const uint32_t raw = base + off_raw() + rs * RAW_BYTES + first * REC;
      uint32_t most = 0xFC00FC00u;  // largest scale and base of this thread's rows
#pragma unroll 1
      for (int half = 0; half < PAGES / (2 * UN); ++half) {
        uint32_t w[UN][4], pr[UN][2];
#pragma unroll
        for (int u = 0; u < UN; ++u) {  // all loads before any arithmetic
          const uint32_t rec = raw + (half * UN + u) * 2 * REC;
          asm volatile("ld.shared.v2.u32 {%0,%1}, [%2];"
                       : "=r"(w[u][0]), "=r"(w[u][1])
                       : "r"(rec + code_off));
          asm volatile("ld.shared.v2.u32 {%0,%1}, [%2];"
                       : "=r"(w[u][2]), "=r"(w[u][3])
                       : "r"(rec + (code_off ^ 8)));
          if constexpr (V)
            asm volatile("ld.shared.v2.u32 {%0,%1}, [%2];"
                         : "=r"(pr[u][0]), "=r"(pr[u][1])
                         : "r"(rec + par_off));
          else {  // K's parameters and V's
            asm volatile("ld.shared.u32 %0, [%1];" : "=r"(pr[u][0]) : "r"(rec + par_off));
            asm volatile("ld.shared.u32 %0, [%1];" : "=r"(pr[u][1]) : "r"(rec + par_off + 64));
          }
        }
#pragma unroll
        for (int u = 0; u < UN; ++u) {
          const int i = (half * UN + u) * 2;  // page, but for `first`
          uint32_t sc[2], ba[2];
#pragma unroll
          for (int e = 0; e < (V ? 2 : 1); ++e) {
            const int key = key0 + (i + first) * PAGE + e;
            uint32_t v = V ? (nan_row(pr[u][e]) ? 0u : pr[u][e]) : key_params(pr[u][0], pr[u][1]);
            if (key >= I.pool_len || (MOD && key < I.lo && key >= I.pfx)) v = 0u;
            most = half2_max(most, v);
            sc[e] = __byte_perm(v, v, 0x1010);
            ba[e] = __byte_perm(v, v, 0x3232);
          }
          const uint32_t dst = tile + i * PAGE * 128;
          if constexpr (!V) {
#pragma unroll
            for (int c = 0; c < 4; ++c) {
              uint32_t p[4];
              code_pairs(w[u][c], p);
#pragma unroll
              for (int e = 0; e < 4; ++e) p[e] = half2_fma(p[e], sc[0], ba[0]);
              sts128(dst + at[c], p[0], p[1], p[2], p[3]);
            }
          } else {
            const uint32_t s2 = __byte_perm(sc[0], sc[1], 0x5410),
                           b2 = __byte_perm(ba[0], ba[1], 0x5410);
#pragma unroll
            for (int ch = 0; ch < 2; ++ch) {
              uint32_t p[8];
              code_pairs(w[u][2 * ch], p);  // (even, odd token) of dims 0 .. 3
              code_pairs(w[u][2 * ch + 1], p + 4);
#pragma unroll
              for (int e = 0; e < 8; ++e) p[e] = half2_fma(p[e], s2, b2);
              sts128(dst + at[2 * ch], __byte_perm(p[0], p[1], 0x5410),
                     __byte_perm(p[2], p[3], 0x5410), __byte_perm(p[4], p[5], 0x5410),
                     __byte_perm(p[6], p[7], 0x5410));
              sts128(dst + at[2 * ch + 1], __byte_perm(p[0], p[1], 0x7632),
                     __byte_perm(p[2], p[3], 0x7632), __byte_perm(p[4], p[5], 0x7632),
                     __byte_perm(p[6], p[7], 0x7632));
            }
          }
        }
      }
      // Values that may pass fp16's range, held to it apart from the loop: inside, a test and a
      // branch for every page cost the converters 6 to 9 % (16 sequences, 8 heads, four row tiles).
      if (past_range(most)) {
#pragma unroll 1
        for (int i = 0; i < PAGES; i += 2) {
#pragma unroll
          for (int c = 0; c < 4; ++c) {
            const uint32_t dst = tile + i * PAGE * 128 + at[c];
            uint32_t v[4];
            lds128(dst, v);
            sts128(dst, held(v[0]), held(v[1]), held(v[2]), held(v[3]));
          }
        }
      }
      fence_proxy_async_smem();
      __syncwarp();
      if (lane == 0) {
        mbar_arrive(&bar[B_REMPTY + rs]);
        mbar_arrive(&fullb[st]);
      }
      if constexpr (!V) {
        if (j == 0) {
          // The item's Q, once the previous item's last S is done: after the first K tile, which
          // only waited for a free stage.
          const bool free = ic == 0 || mbar_wait_bounded(&bar[B_QEMPTY], (ic - 1) & 1, WAIT_LIMIT);
          if (!__all_sync(0xffffffffu, free && !*abort_flag)) {
            if (!free) set_err(P.a.err, MF_ERR_TIMEOUT);
            *abort_flag = 1;
            return;
          }
          q4_stage_q<T>(P, I, base + OFF_Q, qs + (ic & 3) * BM, ts0);
          fence_proxy_async_smem();
          __syncwarp();
          if (lane == 0) mbar_arrive(&bar[B_QFULL]);
        }
      }
    }
  }
}

// The kernel: Q, K and V tiles by TMA from a 16-bit pool (the five tensor maps); with Q4
// converted by warps from a 4-bit pool (no maps); with EXP by TMA from a 4-bit pool that was
// expanded to fp16 beforehand (sequence s's page L at s * width + L, and q with it).  In the
// latter two keys, values and P are fp16.
template <typename T, bool MOD, bool Q4, bool EXP = false>
MF_DEVINL void prefill_body(const CUtensorMap* tmq, const CUtensorMap* tmk, const CUtensorMap* tmv,
                            const CUtensorMap* tmwk, const CUtensorMap* tmwv, const Params& P) {
  constexpr bool FOUR = Q4 || EXP;                              // of a 4-bit cache
  using PT = typename std::conditional<FOUR, __half, T>::type;  // type of P
  constexpr int NTHR = Q4 ? Q4_THREADS : THREADS;
  extern __shared__ uint8_t smem_raw[];
  const uint32_t raw_base = smem_u32(smem_raw);
  const uint32_t base = (raw_base + 1023u) & ~1023u;
  uint8_t* gbase = smem_raw + (base - raw_base);
  uint64_t* bar = reinterpret_cast<uint64_t*>(gbase + off_bar(Q4));
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(gbase + off_misc(Q4));
  volatile int* abort_flag = reinterpret_cast<volatile int*>(gbase + off_misc(Q4) + 4);
  int* prefix = reinterpret_cast<int*>(gbase + off_prefix(Q4));
  uint16_t* order = reinterpret_cast<uint16_t*>(gbase + off_order(P.a.num_seqs, Q4));
  int* counts = reinterpret_cast<int*>(gbase + off_counts(P.a.num_seqs, Q4));

  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  const int B = P.a.num_seqs;
  const int G = P.G;

  // ------------------------------------------------------------- set-up
  if (tid == 0) {
    for (int i = 0; i < 2; ++i) {
      mbar_init(&bar[B_QFULL + i], Q4 ? Q4_CW : 1);
      mbar_init(&bar[B_QEMPTY + i], 1);
      mbar_init(&bar[B_SDONE + i], 1);
      mbar_init(&bar[B_SFREE + i], TILE_WARPS);
      mbar_init(&bar[B_PFULL + i], TILE_WARPS);
      mbar_init(&bar[B_PVDONE + i], 1);
    }
    for (int st = 0; st < KS; ++st) {
      mbar_init(&bar[B_KFULL + st], Q4 ? Q4_CW : 1);
      mbar_init(&bar[B_VFULL + st], Q4 ? Q4_CW : 1);
    }
    if (Q4)
      for (int st = 0; st < RAW; ++st) {
        mbar_init(&bar[B_RFULL + st], 1);
        mbar_init(&bar[B_REMPTY + st], 2 * Q4_CW);
      }
    mbar_init(&bar[B_OFULL], 1);
    mbar_init(&bar[B_OFREE], SM_WARPS);  // every softmax warp reads its half of O
    mbar_init(&bar[B_IDLE], 2);  // one commit per issuer
    for (int i = 0; i < 8; ++i) mbar_init(&bar[B_HAND + i], 1);
    for (int q = 0; q < 4; ++q) mbar_init(&bar[B_EXL + q], WPQ);
    *abort_flag = 0;
    fence_barrier_init();
  }
  for (int i = tid; i < NBK; i += NTHR) counts[i] = 0;
  // Everything above overlaps the previous kernel (programmatic launch);
  // nothing in global memory is read before this point.
  grid_dependency_wait();
  if (warp == 0) {
    tmem_alloc(tmem_slot, TMEM_COLS);
    tmem_relinquish();
  }
  tc_fence_before();
  __syncthreads();
  // Query tiles per sequence (only runs longer than rows_cap rows are served
  // here) and a counting sort of the sequences by kv_len, longest first.  Every
  // CTA builds the same list, so the sort is stable (ties keep index order).
  for (int i = tid; i < B; i += NTHR) {
    int qs, ql;
    seq_rows(P.a, i, qs, ql);
    int tiles = 0;
    const int kvl = P.a.kv_lens[i];
    const bool mine = ql > 0 && (int64_t)ql * G > P.rows_cap;
    if (FOUR && mine) {
      if (ql > P.a.max_q_len || kvl < 0) set_err(P.a.err, MF_ERR_LENGTH);
      if ((kvl + (int64_t)PAGE - 1) / PAGE > P.width) set_err(P.a.err, MF_ERR_TABLE);
      ql = min(ql, P.a.max_q_len);
      const int ppt = positions_per_tile(G);
      tiles = (ql + ppt - 1) / ppt;
    } else if (mine) {
      if (MOD ? kvl < 0 : kvl < ql) {
        set_err(P.a.err, MF_ERR_LENGTH);
      } else if (((P.window ? kvl - ql : kvl) + PAGE - 1) / PAGE > P.a.table_stride) {
        set_err(P.a.err, MF_ERR_TABLE);
      } else {
        const int ppt = positions_per_tile(G);
        tiles = (ql + ppt - 1) / ppt;
      }
    }
    atomicAdd(&counts[sort_bucket(P, kvl, ql, tiles)], 1);
    prefix[i + 1] = tiles;
  }
  __syncthreads();
  if (warp == 0) {  // exclusive scan of the bucket counts
    int run = 0;
    for (int c0 = 0; c0 < NBK; c0 += 32) {
      int v = counts[c0 + lane];
      const int own = v;
#pragma unroll
      for (int o = 1; o < 32; o <<= 1) {
        const int n = __shfl_up_sync(0xffffffffu, v, o);
        if (lane >= o) v += n;
      }
      counts[c0 + lane] = run + v - own;
      run += __shfl_sync(0xffffffffu, v, 31);
    }
  }
  __syncthreads();
  if (warp == 0) {  // place the sequences 32 at a time, in index order
    for (int c0 = 0; c0 < B; c0 += 32) {
      const int i = c0 + lane;
      int qs_, ql_ = 0;
      if (i < B) seq_rows(P.a, i, qs_, ql_);
      const int b = i < B ? sort_bucket(P, P.a.kv_lens[i], ql_, prefix[i + 1]) : -1;
      const unsigned same = __match_any_sync(0xffffffffu, b);
      const int slot = b >= 0 ? counts[b] + __popc(same & ((1u << lane) - 1u)) : 0;
      __syncwarp();
      if (b >= 0) {
        order[slot] = (uint16_t)i;
        if (lane == __ffs(same) - 1) counts[b] += __popc(same);
      }
      __syncwarp();
    }
  }
  __syncthreads();
  // Tiles per sequence in sorted order (all read before any is overwritten),
  // then their prefix sums.
  {
    constexpr int NR = (MAX_SEQS + NTHR - 1) / NTHR;
    int tv[NR];
#pragma unroll
    for (int r = 0; r < NR; ++r) {
      const int k = r * NTHR + tid;
      tv[r] = k < B ? prefix[order[k] + 1] : 0;
    }
    __syncthreads();
#pragma unroll
    for (int r = 0; r < NR; ++r) {
      const int k = r * NTHR + tid;
      if (k < B) prefix[k + 1] = tv[r];
    }
  }
  __syncthreads();
  if (warp == 0) {
    int run = 0;
    if (lane == 0) prefix[0] = 0;
    for (int c0 = 0; c0 < B; c0 += 32) {
      const int i = c0 + lane;
      int v = (i < B) ? prefix[i + 1] : 0;
#pragma unroll
      for (int o = 1; o < 32; o <<= 1) {
        const int n = __shfl_up_sync(0xffffffffu, v, o);
        if (lane >= o) v += n;
      }
      if (i < B) prefix[i + 1] = run + v;
      run += __shfl_sync(0xffffffffu, v, 31);
    }
  }
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = *tmem_slot;
  const int items = prefix[B] * P.a.hkv;

  auto issue = [&]() {
    // ========================================================= MMA issuers
    if (lane == 0) {
      const bool is_pv = warp == (Q4 ? Q4_PV_WARP : PV_WARP);
      const uint32_t idesc_s = idesc_f16(BM, BN, P.in_fmt, false);
      const uint32_t idesc_o = idesc_f16(BM, D, P.in_fmt, true);
      const uint32_t tO = tmem + COL_O;
      bool ok = true;
      uint32_t g = 0;
      int ic = 0;
      for (int k = 0; ok && snake_item(k) < items; ++k, ++ic) {
        const Item I = item_at<MOD, FOUR>(P, prefix, order, B, snake_item(k));
        constexpr int NQ = q_buffers(Q4);
        const int qb = ic % NQ;
        if (!is_pv) ok = mbar_wait_bounded(&bar[B_QFULL + qb], (ic / NQ) & 1, WAIT_LIMIT);
        const uint32_t qbase = base + OFF_Q + qb * TILE_BYTES;
        for (int j = 0; ok && j < I.nt; ++j, ++g) {
          const int b2 = g & 1, st = g % KS;
          if (!is_pv) {
            // S_g = Q K_g^T once the softmax has loaded the S of tile g - 2.
            if (g >= 2)
              ok = ok && mbar_wait_bounded(&bar[B_SFREE + b2], ((g >> 1) - 1) & 1, WAIT_LIMIT);
            ok = ok && mbar_wait_bounded(&bar[B_KFULL + st], (g / KS) & 1, WAIT_LIMIT);
            if (!ok || *abort_flag) break;
            tc_fence_after();
            const uint32_t kb = base + off_k(Q4) + st * TILE_BYTES;
#pragma unroll
            for (int ks = 0; ks < D / 16; ++ks) {
              const uint32_t off = (ks >> 2) * HALF_BYTES + (ks & 3) * 32;
              umma_ss(tmem + COL_S + b2 * 128, sdesc_sw128(qbase + off, 16, 1024),
                      sdesc_sw128(kb + off, 16, 1024), idesc_s, ks > 0);
            }
            umma_commit(&bar[B_SDONE + b2]);
            if (j == I.nt - 1) umma_commit(&bar[B_QEMPTY + qb]);
          } else {
            // O += P_g V_g; the first P V of an item overwrites O, after the
            // previous epilogue has read it.
            ok = ok && mbar_wait_bounded(&bar[B_PFULL + b2], (g >> 1) & 1, WAIT_LIMIT);
            ok = ok && mbar_wait_bounded(&bar[B_VFULL + st], (g / KS) & 1, WAIT_LIMIT);
            if (j == 0 && ic > 0)
              ok = ok && mbar_wait_bounded(&bar[B_OFREE], (ic - 1) & 1, WAIT_LIMIT);
            if (!ok || *abort_flag) break;
            tc_fence_after();
            const uint32_t vb = base + off_v(Q4) + st * TILE_BYTES;
#pragma unroll
            for (int ks = 0; ks < BN / 16; ++ks)
              // P columns ks*8 .. (16 keys packed 2 per column); V rows ks*16 ..
              umma_ts(tO, tmem + COL_P + b2 * 64 + ks * 8,
                      sdesc_sw128(vb + ks * 16 * 128, HALF_BYTES, 1024), idesc_o,
                      (j == 0 && ks == 0) ? 0u : 1u);
            umma_commit(&bar[B_PVDONE + b2]);
            if (j == I.nt - 1) umma_commit(&bar[B_OFULL]);
          }
        }
      }
      if (!ok) {
        set_err(P.a.err, MF_ERR_TIMEOUT);
        *abort_flag = 1;
      }
      // Every MMA either thread issued has completed before TMEM can be freed.
      umma_commit(&bar[B_IDLE]);
      if (!mbar_wait_bounded(&bar[B_IDLE], 0, WAIT_LIMIT)) set_err(P.a.err, MF_ERR_TIMEOUT);
    }
  };
  auto softmax = [&]() {
    // ====================================== softmax (warps 0 .. SM_WARPS-1)
    // Two warps per TMEM lane quarter: the warp of parity par = warp / 4 takes
    // the tiles whose global index g has g % 2 == par (S buffer par, P buffer
    // par), so one warp's TMEM load, row max and P store overlap the other's
    // exponentials.  The online softmax is sequential only in its reference
    // max: a warp finishes its tile's row max, then takes the previous tile's
    // reference max from the other warp (mbox, B_HAND), decides its own,
    // publishes it, and only then computes the exponentials.  Each warp keeps
    // its own row sums, scaled to the reference max it last saw; at an item's
    // end the two partial sums are combined (l / ms boxes, B_EXL) and each
    // warp normalises and stores half of O's columns.
    const int quarter = warp & 3, par = warp >> 2;
    const int row = quarter * 32 + lane;  // TMEM lane == tile row
    const uint32_t lane_off = (uint32_t)(quarter * 32) << 16;
    const uint32_t tO = tmem + COL_O + lane_off;
    float* mbox = reinterpret_cast<float*>(gbase + off_xch(Q4));  // [2][BM]
    float* lbox = mbox + 2 * BM;                               // [2 items][2][BM]
    float* msbox = lbox + 4 * BM;                              // [2 items][2][BM]
    // Scores that were capped or biased are in log2 units already.
    const bool transformed = MOD && (P.a.mods.softcap > 0.f || P.a.mods.slopes);
    float sl2 = transformed ? 1.f : P.scale_log2;
    float raw_sl2 = P.scale_log2;  // of S itself; Q4: of this row's, which q was scaled for
    bool ok = true;
    // An item's epilogue runs after this warp's first tile of the next item
    // (or at the next item's end when it has none): by then the item's last
    // P V has completed and the other warp has finished the item too, so
    // neither the O wait nor the row-sum exchange stalls, and the next item's
    // first tiles run meanwhile.  Its first P V waits for O to be read.
    bool pend = false;
    int pend_ic = 0;
    bool pend_valid = false;
    T* pend_row = nullptr;
    float pend_l = 0.f, pend_m = -INFINITY;
    auto epilogue = [&]() -> bool {
      float* lb = lbox + (pend_ic & 1) * 2 * BM;
      float* mb = msbox + (pend_ic & 1) * 2 * BM;
      lb[par * BM + row] = pend_l;
      mb[par * BM + row] = pend_m;
      __syncwarp();
      if (lane == 0) mbar_arrive(&bar[B_EXL + quarter]);
      bool done = mbar_wait_bounded(&bar[B_EXL + quarter], pend_ic & 1, WAIT_LIMIT);
      const float l_oth = lb[(par ^ 1) * BM + row], m_oth = mb[(par ^ 1) * BM + row];
      const float m_fin = fmaxf(pend_m, m_oth);
      float l_tot = 0.f;
      if (pend_m != -INFINITY) l_tot += pend_l * fast_exp2(pend_m - m_fin);
      if (m_oth != -INFINITY) l_tot += l_oth * fast_exp2(m_oth - m_fin);
      done = done && !*abort_flag && mbar_wait_bounded(&bar[B_OFULL], pend_ic & 1, WAIT_LIMIT);
      done = __all_sync(0xffffffffu, done);
      if (!done) return false;
      tc_fence_after();
      uint32_t o[64];
      tmem_ld32(tO + par * 64, o);
      tmem_ld32(tO + par * 64 + 32, o + 32);
      tmem_wait_ld();
      tc_fence_before();
      __syncwarp();
      if (lane == 0) mbar_arrive(&bar[B_OFREE]);  // O may be overwritten
      if (pend_valid) {
        const float inv = FOUR ? (l_tot == 0.f ? 0.f : 1.f / l_tot) : l_tot > 0.f ? 1.f / l_tot : 0.f;
        if (Q4 && !P.vec) {  // (EXP takes calls with 16-byte rows only)
#pragma unroll
          for (int e = 0; e < 64; ++e) pend_row[e] = from_f32<T>(__uint_as_float(o[e]) * inv);
        } else
#pragma unroll
        for (int e = 0; e < 64; e += 8) {
          uint4 v;
          v.x = Mma<T>::pack(__uint_as_float(o[e]) * inv, __uint_as_float(o[e + 1]) * inv);
          v.y = Mma<T>::pack(__uint_as_float(o[e + 2]) * inv, __uint_as_float(o[e + 3]) * inv);
          v.z = Mma<T>::pack(__uint_as_float(o[e + 4]) * inv, __uint_as_float(o[e + 5]) * inv);
          v.w = Mma<T>::pack(__uint_as_float(o[e + 6]) * inv, __uint_as_float(o[e + 7]) * inv);
          *reinterpret_cast<uint4*>(pend_row + e) = v;
        }
      }
      pend = false;
      return true;
    };
    uint32_t g = 0;
    int ic = 0;
    for (int k = 0; ok && snake_item(k) < items; ++k, ++ic) {
      const Item I = item_at<MOD, FOUR>(P, prefix, order, B, snake_item(k));
      const int pos = I.pos0 + row / G;  // query position of this row within the sequence
      const int gg = row % G;
      const bool row_valid = row < positions_per_tile(G) * G && pos < I.q_len;
      // Last visible key: causal over the context; with a window, every pool key
      // and, in the window tile, window keys 0..pos.
      const int limit = !FOUR && !MOD && P.window ? I.pool_len - 1
                        : FOUR   ? min(P.a.causal ? I.win_start + pos : I.kv_len - 1, I.pool_len - 1)
                                 : min(I.win_start + pos, I.kv_len - 1);
      const int row_lo =
          MOD && P.a.mods.window > 0 ? I.win_start + pos - P.a.mods.window + 1 : 0;
      const float slope = MOD && P.a.mods.slopes ? P.a.mods.slopes[I.h * G + gg] * kLog2e : 0.f;
      const float item_sl2 =
          EXP && row_valid ? __ldg(P.qs + (int64_t)(I.q_start + pos) * P.a.hq + I.h * G + gg) : 0.f;
      float m_seen = -INFINITY;  // reference max l_own is scaled to
      float l_own = 0.f;
      for (int j = 0; j < I.nt; ++j, ++g) {
        if ((int)(g & 1) != par) continue;  // the other warp's tile
        if (!mbar_wait_bounded(&bar[B_SDONE + par], (g >> 1) & 1, WAIT_LIMIT)) ok = false;
        // Warp-uniform decision: tcgen05.ld/st below are warp-collective.
        if (__any_sync(0xffffffffu, !ok || *abort_flag != 0)) {
          ok = false;
          break;
        }
        tc_fence_after();
        float sv[CW];
#pragma unroll
        for (int c = 0; c < CW / 32; ++c)
          tmem_ld32(tmem + COL_S + par * 128 + lane_off + c * 32,
                    reinterpret_cast<uint32_t*>(sv + c * 32));
        if constexpr (EXP) {
          raw_sl2 = item_sl2;
          if (!transformed) sl2 = raw_sl2;
        } else if constexpr (Q4) {
          raw_sl2 = reinterpret_cast<const float*>(gbase + off_qs())[(ic & 3) * BM + row];
          if (!transformed) sl2 = raw_sl2;
        }
        tmem_wait_ld();
        tc_fence_before();
        __syncwarp();
        if (lane == 0) mbar_arrive(&bar[B_SFREE + par]);  // S buffer may be overwritten

        // Row max of the raw scores over the visible columns (c <= limit).
        const bool win_tile = !FOUR && !MOD && P.window && j == I.nt - 1;
        const int kbase = I.template tile<MOD>(j) * BN;
        const int lim = win_tile ? pos : limit - kbase;
        if constexpr (MOD) {
          if (P.a.mods.softcap > 0.f) cap_scores<CW>(P, sv, raw_sl2);
          if (P.a.mods.slopes) {
            const float up = P.a.mods.softcap > 0.f ? 1.f : raw_sl2;
            const uint64_t up2 = f32x2(up, up), two = f32x2(2.f * slope, 2.f * slope);
#pragma unroll
            for (int c0 = 0; c0 < CW; c0 += 16) {  // the bias steps by adds, anew every 16 keys
              const float at = slope * (float)(kbase + c0 - (I.win_start + pos));
              uint64_t b = f32x2(at, at + slope);
#pragma unroll
              for (int c = c0; c < c0 + 16; c += 2) {
                f32x2_split(f32x2_fma(f32x2(sv[c], sv[c + 1]), up2, b), sv[c], sv[c + 1]);
                b = f32x2_add(b, two);
              }
            }
          }
          const int lo_c = row_lo - kbase, pf_c = I.pfx - kbase;
          if (__any_sync(0xffffffffu, !(pf_c >= CW || (lim >= CW - 1 && lo_c <= 0)))) {
#pragma unroll
            for (int c = 0; c < CW; ++c)
              if (c >= pf_c && (c > lim || c < lo_c)) sv[c] = -INFINITY;
          }
        } else if (__any_sync(0xffffffffu, lim < CW - 1)) {
#pragma unroll
          for (int c = 0; c < CW; ++c)
            if (c > lim) sv[c] = -INFINITY;
        }
        float mx[8];
#pragma unroll
        for (int e = 0; e < 8; ++e) mx[e] = sv[e];
#pragma unroll
        for (int c = 8; c < CW; c += 2) mx[(c >> 1) & 7] = fmax3f(mx[(c >> 1) & 7], sv[c], sv[c + 1]);
        const float mraw = fmax3f(fmax3f(mx[0], mx[1], mx[2]), fmax3f(mx[3], mx[4], mx[5]),
                                  fmaxf(mx[6], mx[7]));
        // The previous tile's reference max (the other warp's), unless this
        // tile starts an item.
        float m_prev = -INFINITY;
        if (g > 0) {
          if (!mbar_wait_bounded(&bar[B_HAND + quarter * 2 + (par ^ 1)], ((g - 1) >> 1) & 1,
                                 WAIT_LIMIT))
            ok = false;
          if (j > 0) m_prev = mbox[(par ^ 1) * BM + row];
        }
        if (__any_sync(0xffffffffu, !ok)) {
          ok = false;
          break;
        }
        // l_own follows every rescale the other warp decided.
        if (m_prev != m_seen && m_seen != -INFINITY) l_own *= fast_exp2(m_seen - m_prev);
        // Lazy rescale: a row keeps its reference max unless this tile exceeds
        // it by more than 2^8 (log2 units).
        const float tmax = mraw * sl2;
        float m_ref = m_prev, f = 1.f;
        if (mraw != -INFINITY && (m_ref == -INFINITY || tmax > m_ref + RESCALE_THRESHOLD)) {
          if (m_ref != -INFINITY) f = fast_exp2(m_ref - tmax);
          m_ref = tmax;
        }
        l_own *= f;
        m_seen = m_ref;
        mbox[par * BM + row] = m_ref;
        __syncwarp();
        if (lane == 0) mbar_arrive(&bar[B_HAND + quarter * 2 + par]);
        // The P buffer is free once the P V product of two tiles ago completed.
        if (g >= 2 && !mbar_wait_bounded(&bar[B_PVDONE + par], ((g >> 1) - 1) & 1, WAIT_LIMIT))
          ok = false;
        if (__any_sync(0xffffffffu, !ok)) {
          ok = false;
          break;
        }
        tc_fence_after();
        // P = 2^(s * scale_log2 - m_ref), packed to 16-bit pairs and stored 32
        // columns at a time (the scores of a stored chunk are dead, so their
        // registers hold the next chunk's P); scaling and row sums as packed
        // fp32 pairs, the exponentials on the SFU.
        const float nmu = (m_ref == -INFINITY) ? 0.f : -m_ref;
        const uint64_t sl2x2 = f32x2(sl2, sl2), nmux2 = f32x2(nmu, nmu);
        uint64_t ps2[2] = {f32x2(0.f, 0.f), f32x2(0.f, 0.f)};
        const uint32_t tp = tmem + COL_P + par * 64 + lane_off;
#pragma unroll
        for (int ch = 0; ch < CW / 32; ++ch) {
          uint32_t pk[16];
#pragma unroll
          for (int c = 0; c < 16; ++c) {
            float x0, x1;
            const int col = ch * 32 + 2 * c;
            f32x2_split(f32x2_fma(f32x2(sv[col], sv[col + 1]), sl2x2, nmux2), x0, x1);
            const float p0 = fast_exp2(x0), p1 = fast_exp2(x1);
            ps2[c & 1] = f32x2_add(ps2[c & 1], f32x2(p0, p1));
            pk[c] = Mma<PT>::pack(p0, p1);
          }
          tmem_st16(tp + ch * 16, pk);
        }
        float ps_lo, ps_hi;
        f32x2_split(f32x2_add(ps2[0], ps2[1]), ps_lo, ps_hi);
        l_own += ps_lo + ps_hi;
        tmem_wait_st();
        if (j > 0 && __any_sync(0xffffffffu, f != 1.f)) {
          // O must include P_{g-1} V_{g-1} before it is rescaled, and the
          // rescale must land before this tile's P V (ordered by P-full below).
          // A pending epilogue goes first: P_{g-1} V_{g-1} may be this item's
          // first P V, which waits for the previous item's O to be read.
          if (pend && !epilogue()) ok = false;
          if (!mbar_wait_bounded(&bar[B_PVDONE + ((g - 1) & 1)], ((g - 1) >> 1) & 1, WAIT_LIMIT))
            ok = false;
          tc_fence_after();
#pragma unroll 1
          for (int c = 0; c < CW / 32; ++c) {
            uint32_t o[32];
            tmem_ld32(tO + c * 32, o);
            tmem_wait_ld();
#pragma unroll
            for (int e = 0; e < 32; ++e) o[e] = __float_as_uint(__uint_as_float(o[e]) * f);
            tmem_st32(tO + c * 32, o);
          }
          tmem_wait_st();
        }
        // Keys of this tile past the last one loaded: past the pool in the last
        // pool tile, past q_len in the window tile (whose other rows were never
        // written by this tile's loads).
        const int loaded = win_tile ? I.q_len : I.pool_len - kbase;
        // MOD: keys [dead0, dead1) lie behind every row's window.
        const int dead0 = MOD ? max(I.pfx - kbase, 0) : 0;
        const int dead1 = MOD ? min(I.lo - kbase, BN) : 0;
        if (!Q4 && quarter == 0 && ((!EXP && loaded < BN) || dead0 < dead1)) {
          // Zero the V rows of those keys (whole 128-byte rows of both halves)
          // so p = 0 adds nothing even where a slot holds NaN.  This warp's
          // P-full arrival orders it before P V.
          const int st = g % KS;
          if (!mbar_wait_bounded(&bar[B_VFULL + st], (g / KS) & 1, WAIT_LIMIT)) ok = false;
          const uint32_t vb = base + off_v(Q4) + st * TILE_BYTES;
          const int first = min(max(0, loaded), BN);
          for (int idx = lane; MOD && idx < (dead1 - dead0) * 16; idx += 32) {
            const int r = dead0 + idx / 16, c16 = idx % 16;
            const uint32_t a = vb + (c16 >> 3) * HALF_BYTES + r * 128 + (c16 & 7) * 16;
            asm volatile("st.shared.v4.u32 [%0], {%1, %1, %1, %1};" ::"r"(a), "r"(0u) : "memory");
          }
          for (int idx = lane; idx < (BN - first) * 16; idx += 32) {
            const int r = first + idx / 16, c16 = idx % 16;
            const uint32_t a = vb + (c16 >> 3) * HALF_BYTES + r * 128 + (c16 & 7) * 16;
            asm volatile("st.shared.v4.u32 [%0], {%1, %1, %1, %1};" ::"r"(a), "r"(0u) : "memory");
          }
          fence_proxy_async_smem();
        }
        tc_fence_before();
        __syncwarp();
        if (lane == 0) mbar_arrive(&bar[B_PFULL + par]);
        if (pend && !epilogue()) {
          ok = false;
          break;
        }
      }
      // Uniform: the epilogue below is warp-collective.
      if (__any_sync(0xffffffffu, !ok)) {
        ok = false;
        break;
      }
      if (pend && !epilogue()) {  // no tile of this item was this warp's
        ok = false;
        break;
      }
      pend = true;
      pend_ic = ic;
      pend_valid = row_valid;
      const int out_row = I.q_start + (row_valid ? pos : 0);
      pend_row = static_cast<T*>(P.a.out) +
                 (int64_t)(FOUR && row_valid ? map_row(P.a, out_row) : out_row) * P.a.o_sr +
                 (int64_t)(I.h * G + gg) * P.a.o_sh + par * 64;
      pend_l = l_own;
      pend_m = m_seen;
    }
    if (ok && pend && !epilogue()) ok = false;
    if (!ok) {
      if (lane == 0) set_err(P.a.err, MF_ERR_TIMEOUT);
      *abort_flag = 1;
    }
  };
  if constexpr (Q4) {
    if (warp >= SM_WARPS) {
      asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(Q4_REGS_REST));
      float* qs = reinterpret_cast<float*>(gbase + off_qs());
      if (warp >= Q4_V_WARP)
        q4_stage<T, MOD, true>(P, prefix, order, items, base, qs, bar, abort_flag,
                               tid - Q4_V_WARP * 32);
      else if (warp >= Q4_K_WARP)
        q4_stage<T, MOD, false>(P, prefix, order, items, base, qs, bar, abort_flag,
                                tid - Q4_K_WARP * 32);
      else if (warp == Q4_LOAD_WARP)
        q4_load<MOD>(P, prefix, order, items, base, bar, abort_flag, lane);
      else if (warp < Q4_LOAD_WARP)
        issue();
    } else {
      asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(Q4_REGS_SOFTMAX));
      softmax();
    }
  } else if (warp == TMA_WARP || warp == V_WARP) {
    // ======================================================= TMA producers
    // One warp loads Q and K, another V: the K ring frees at S completion and
    // the V ring only at P V completion, so K loads never queue behind V.  A
    // 128-key tile is 8 pages x 2 halves = 16 boxes: lane l < 16 loads the block
    // id of page l / 2 (one tile ahead) and issues the box of (page l / 2, half
    // l % 2), so a tile goes out as one warp instruction; lane 0 does the ring
    // waits and the transaction count, and broadcasts every decision.
    const bool is_v = warp == V_WARP;
    const uint32_t q_bytes = (uint32_t)(positions_per_tile(G) * G) * D * 2;  // both halves
    const CUtensorMap* wmap = is_v ? tmwv : tmwk;
    const uint64_t pol_once = l2_evict_first_policy();
    const uint64_t pol_keep = l2_evict_last_policy();
    if (lane == 0) {
      if (!is_v) {
        prefetch_tmap(tmq);
        prefetch_tmap(tmk);
      } else {
        prefetch_tmap(tmv);
      }
      if (P.window) prefetch_tmap(wmap);
    }
    const CUtensorMap* tmap = is_v ? tmv : tmk;
    const uint32_t ring = is_v ? off_v(Q4) : off_k(Q4);
    uint64_t* fullb = &bar[is_v ? B_VFULL : B_KFULL];
    uint64_t* emptyb = &bar[is_v ? B_PVDONE : B_SDONE];  // ring stage g % KS frees
    const int nb = EXP ? P.a.num_seqs * P.width : P.a.num_blocks;
    const bool boxer = lane < 2 * (BN / PAGE);
    const int my_pg = lane >> 1, my_half = lane & 1;
    uint32_t g = 0;      // tiles started (all items)
    uint32_t armed = 0;  // tiles whose loads were issued
    int ic = 0;          // items whose Q load was issued
    bool run = true;
    for (int k = 0; run && snake_item(k) < items; ++k) {
      run = __shfl_sync(0xffffffffu, *abort_flag == 0, 0);
      if (!run) break;
      const Item I = item_at<MOD, FOUR>(P, prefix, order, B, snake_item(k));
      if (!is_v) {
        const int qb = ic & 1;
        bool fine = true;
        if (lane == 0) {
          if (ic >= 2 &&
              !mbar_wait_bounded(&bar[B_QEMPTY + qb], ((ic >> 1) - 1) & 1, WAIT_LIMIT)) {
            set_err(P.a.err, MF_ERR_TIMEOUT);
            *abort_flag = 1;
            fine = false;
          } else {
            mbar_arrive_expect_tx(&bar[B_QFULL + qb], q_bytes);
            for (int half = 0; half < 2; ++half)
              tma_load_4d(gbase + OFF_Q + qb * TILE_BYTES + half * HALF_BYTES, tmq,
                          &bar[B_QFULL + qb], 0, I.h * G, half, I.q_start + I.pos0, pol_once);
          }
        }
        run = __shfl_sync(0xffffffffu, fine, 0);
        if (!run) break;
        ++ic;
      }
      const int pool_pages = (I.pool_len + PAGE - 1) / PAGE;
      const int32_t* table = P.a.tables + (int64_t)I.s * P.a.table_stride;
      // Block id of this lane's page, loaded one tile ahead.  Out-of-table
      // pages use an out-of-range coordinate: TMA fills zeros.
      auto block_of = [&](int page) {
        if (!boxer || page >= pool_pages || !I.template page_live<MOD>(page)) return -1;
        return EXP ? I.s * P.width + page : __ldg(table + page);
      };
      int nxt = block_of(I.template tile<MOD>(0) * (BN / PAGE) + my_pg);
      for (int j = 0; j < I.nt; ++j, ++g) {
        const int L = I.template tile<MOD>(j) * (BN / PAGE) + my_pg;
        int tok = nb * PAGE;
        if (boxer && L < pool_pages && I.template page_live<MOD>(L)) {
          if (nxt >= 0 && nxt < nb) tok = nxt * PAGE;
          else set_err(P.a.err, MF_ERR_BLOCK_ID);
        }
        if (j + 1 < I.nt) nxt = block_of(I.template tile<MOD>(j + 1) * (BN / PAGE) + my_pg);
        const int st = g % KS;
        // With a window, the last tile is the window: 16 rows of each half.
        const bool win_tile = P.window && j == I.nt - 1;
        bool fine = true;
        if (lane == 0) {
          if (g >= KS && !mbar_wait_bounded(&emptyb[st], ((g / KS) - 1) & 1, WAIT_LIMIT)) {
            set_err(P.a.err, MF_ERR_TIMEOUT);
            *abort_flag = 1;
            fine = false;
          } else if (*abort_flag) {
            fine = false;
          } else {
            mbar_arrive_expect_tx(&fullb[st], win_tile ? 2u * PAGE * 128u : TILE_BYTES);
          }
        }
        run = __shfl_sync(0xffffffffu, fine, 0);  // also orders expect_tx before the loads
        if (!run) break;
        armed = g + 1;
        uint8_t* dst = gbase + ring + st * TILE_BYTES + my_half * HALF_BYTES;
        if (win_tile) {
          if (lane < 2)
            tma_load_4d(dst, wmap, &fullb[st], 0, I.q_start, my_half, I.h, pol_once);
        } else if (boxer) {
          tma_load_4d(dst + my_pg * PAGE * 128, tmap, &fullb[st], 0, tok, my_half, I.h, pol_keep);
        }
      }
    }
    // Drain every armed load before the CTA can exit (the ring holds the last
    // KS tiles and the last two Q tiles in flight at most).
    if (lane == 0) {
      for (uint32_t k = armed > (uint32_t)KS ? armed - KS : 0u; k < armed; ++k)
        if (!mbar_wait_bounded(&fullb[k % KS], (k / KS) & 1, WAIT_LIMIT))
          set_err(P.a.err, MF_ERR_TIMEOUT);
      if (!is_v)
        for (int i = ic > 2 ? ic - 2 : 0; i < ic; ++i)
          if (!mbar_wait_bounded(&bar[B_QFULL + (i & 1)], (i >> 1) & 1, WAIT_LIMIT))
            set_err(P.a.err, MF_ERR_TIMEOUT);
    }
  } else if (warp == MMA_WARP || warp == PV_WARP) {
    issue();
  } else {
    softmax();
  }

  // ---------------------------------------------------------- teardown
  tc_fence_before();
  __syncthreads();
  if (warp == 0) {
    tc_fence_after();
    tmem_dealloc(tmem, TMEM_COLS);
  }
}

}  // namespace pf
}  // namespace mf
