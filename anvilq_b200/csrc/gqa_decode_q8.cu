// gqa_decode_q8.cu -- GQA decode attention over a paged cache held in 8 bits with a
// scale for each block of 16 tokens and kv head (kv_q8.cuh).
//
// Mathematics.  Query token i of sequence b (Q of them, at positions
// seqlens[b] - Q + i) sees the positions t up to its own:
//   out = sum_t softmax_t(q . kc_t ks_t * scale) vc_t vs_t
// with integer or e4m3 codes kc, vc and their blocks' scales ks, vs.  A query
// that sees nothing (an empty sequence, or a position below 0) gives zeros.
//
// What bounds it: the codes' bytes, read once (4 Hq/Hkv Q flops a byte).
//
// Work split.  A tile is 32 tokens of one kv head, two blocks: 4 KB of K codes and
// 4 KB of V codes at D = 128, in runs of 2 KB at least.  The rows of a tile's
// products are the Q * Hq/Hkv query rows of its kv head, in groups of 8 or 16
// (kRows); a pair is a (sequence, kv head, row group).  All pairs' tiles in a row --
// sequence, then pair, then tile -- are cut into equal stretches, one a warp, so that
// the device is evenly loaded whatever the lengths; the lengths are on the device,
// so every warp finds its stretch from them.  A pair inside one warp's stretch is
// finished by that warp.  The others' partial softmax states are merged in shared
// memory, and where a pair spans CTAs, by the CTA that arrives last at the pair's
// ticket, in CTA order (bit-reproducible).  plan_of has the rules.
//
// A warp streams its tiles through its own TMA ring, mbarrier by mbarrier.  The
// codes never return to memory as binary16: fragments of mma.m16n8k16 are formed
// in registers.
//   S^T = K Q^T: a lane's A fragment is chunks of 16 bytes of two tokens (the
//     contraction's order over d is free, so q is loaded in the same order).  An int8
//     code c enters as the binary16 subnormal (c + 128) 2^-24 -- a byte beside a zero
//     byte, no arithmetic -- and the accumulator starts at -128 2^-24 sum q.  An
//     e4m3 code is converted (exactly) by the cvt instruction.
//   O^T += V^T P^T: P^T's B fragment is the accumulator of S^T, packed and
//     transposed (movmatrix), so a lane holds the same query rows' scores, softmax
//     statistics and outputs.  V^T's fragments pair the bytes of two tokens.  Over a
//     long context the sum of p c is far smaller than the sum of p, so here an offset
//     would cost precision: int8 codes are made signed first,
//     (1024 + 128 + c) - 1152 in binary16.
//   (With S = Q K^T instead, eight rows as a 16-row operand, the empty half took as
//   many MMAs again and its zero registers a move each: 389 instructions a block of
//   16 tokens.)
// The tokens of a block are dealt to fragment rows in an order (token_of) that
// keeps both reads of the 128-byte-swizzled block free of bank conflicts.  Two
// blocks a step share the waits, votes and bookkeeping: one block a step took 480
// instructions a block and was bound by their issue, not by memory.
//
// Softmax: binary32, log2 domain, online.  The running reference m is not the
// maximum but stays within 12 of it (above: p <= 2^12; m is set 4 below a new
// maximum), so that most tiles neither reduce over lanes nor rescale; p then fits
// binary16 with more room below than the maximum itself would leave.  The V scale
// is folded into p relative to a running F, which likewise moves only when a
// block's scale leaves [F/8, 8F]: p vs/F <= 2^15.
//
// Fewer bits than binary32 are kept in two places, by choice.  p vs/F enters PV as
// binary16, 2^-11 of each p at most (the sum l takes p as it is): 32 bits would be two
// binary16 parts and PV's MMAs and fragments of P twice.  And an int8 score is summed beside
// its offset, which at most doubles the partial sums and so their binary32 roundings, for one
// subtraction a code less.  Against 64 bits outputs are off by 2.2e-4 to 3.0e-4 (root mean
// square, relative); 2.1e-4 is the binary16 output's own rounding.
#include <cuda.h>
#include <cudaTypedefs.h>

#include <algorithm>
#include <cmath>
#include <mutex>
#include <type_traits>

#include "kv_q8.cuh"

namespace anvilq {
namespace attn8 {

using q8::kBlock;
constexpr int kTile = 2 * kBlock;   // tokens of a step
constexpr int kMaxSms = 160;        // SMs that are used, one CTA each
constexpr int kMaxBatch = 65536;
constexpr unsigned long long kWaitLimitNs = 1000000000ull;

struct Divisor {     // x / d for 0 <= x < 2^17, 1 <= d < 2^15: the error of m is below d / 2^32
  int d;
  unsigned m;        // ceil(2^32 / d); 0 for d = 1
  __device__ __forceinline__ int quotient(int x) const { return m ? (int)__umulhi((unsigned)x, m) : x; }
};

struct Params {
  const __half* q;             // [B][Q][Hq][D]
  const float* k_scales;       // [num_pages][Hkv][page_tokens / 16]
  const float* v_scales;
  const uint32_t* page_table;  // [B][max_pages]
  const int* seqlens;          // [B]
  __half* out;                 // [B][Q][Hq][D]
  int* tickets;                // one a CTA, of the pair that goes on from it
  float* partials;             // [CTA][2] states: of the pair begun earlier, of the pair that goes on
  float* parked;               // [CTA][warp] states
  int* dev_err;
  int B, Q, Hq, Hkv, page_tokens, max_pages, num_pages;
  Divisor group, row_groups;   // query heads a kv head; row groups a (sequence, kv head)
  int wide;                    // pages hold whole tiles: one copy of 32 rows, not two of 16
  unsigned expire;             // ANVILQ_EXPIRE_WAITS: bits of the waits that give up at once
  float scale_log2;            // softmax scale * log2(e)
};

// RT: rows of a pair in eights
template <int D_, int RT_>
struct Shape {
  static constexpr int D = D_, RT = RT_;
  static constexpr int kRows = 8 * RT;
  static constexpr int kWarps = RT == 1 ? 12 : 8;              // one CTA an SM: 168 or 255 registers a thread
  static constexpr int kThreads = kWarps * 32;
  static_assert(kWarps <= 12, "Control has room for their parts");
  static constexpr int kTileBytes = kTile * D;                 // of K or V
  static constexpr int kStageBytes = 2 * kTileBytes;
  // 16 KB a warp: the copies of all warps in flight are several times what the
  // memory's latency needs; more of them only queue (half as much again ran 8 %
  // slower, the page table, scales and q waiting behind them)
  static constexpr int kStages = 16 * 1024 / kStageBytes;
  static constexpr int kRingBytes = kStages * kStageBytes;     // per warp
  static constexpr int kState = kRows * D;                     // floats of a state's o
  static constexpr int kSlots = 32;                            // tiles that are described ahead, two batches
  static constexpr int kStatOffset = kWarps * kRingBytes;      // (m, l) [warp][2][row]
  static constexpr int kMetaOffset = kStatOffset + kWarps * 2 * kRows * 8;
  static constexpr int kBarOffset = kMetaOffset + kWarps * kSlots * 48;
  static constexpr int kGroupOffset = kBarOffset + kWarps * kStages * 8;   // tiles of 32 sequences each
  static constexpr int kEnd = kGroupOffset + kMaxBatch / 32 * 4;
  static constexpr int kTotal = kEnd + 1024;                   // + slack to align the rings
  static constexpr int kPartial = kState + 2 * kRows;          // floats of a state in global memory
  static_assert((kStages & (kStages - 1)) == 0 && kStages <= 4,
                "a slot's old tile is used by the time it is named again");
  static_assert(kRingBytes >= kState * 4, "a state fits the idle ring");
  static_assert(kTotal + 4096 <= 227 * 1024, "one CTA an SM");
};

struct Meta {        // a tile: what its copies and its consumer need
  float ks[2], vs[2];            // its blocks' scales
  int tile, n;                   // tile of the pair, the pair's tiles
  int b, pair;                   // sequence, pair of the sequence
  int row[2];                    // blocks' first rows in the pools (as matrices of D-byte rows)
  uint32_t word[2];              // page-table words
};
static_assert(sizeof(Meta) == 48, "three 16-byte reads");

struct Part {        // a pair that a warp did not finish alone
  unsigned first;    // its first tile in the row of all tiles
  int n, b, pair;
};

// How the work is cut: a warp's stretch is 1 / kWarps of a CTA's tiles.
struct Plan {
  bool whole;        // a CTA takes a whole pair
  unsigned total;    // tiles in all
  unsigned chunk;    // else: tiles of a CTA
};

__device__ __forceinline__ uint32_t smem_u32(const void* p) {
  return static_cast<uint32_t>(__cvta_generic_to_shared(p));
}
__device__ __forceinline__ unsigned long long globaltimer() {
  unsigned long long t;
  asm volatile("mov.u64 %0, %%globaltimer;" : "=l"(t));
  return t;
}
__device__ __forceinline__ bool mbar_try_wait(uint32_t bar, uint32_t parity) {
  uint32_t done;
  asm volatile(
      "{\n .reg .pred p;\n mbarrier.try_wait.parity.shared::cta.b64 p, [%1], %2;\n selp.u32 %0, 1, 0, p;\n}"
      : "=r"(done)
      : "r"(bar), "r"(parity)
      : "memory");
  return done != 0;
}
// The warp's bounded wait: true when the phase completed, false after ~kWaitLimitNs.
__device__ __noinline__ bool warp_wait_long(uint32_t bar, uint32_t parity) {
  const unsigned long long t0 = globaltimer();
  for (uint32_t i = 0;; ++i) {
    if (__all_sync(0xffffffffu, mbar_try_wait(bar, parity))) return true;
    if ((i & 63u) == 63u && __any_sync(0xffffffffu, globaltimer() - t0 > kWaitLimitNs)) return false;
  }
}
__device__ __forceinline__ bool warp_wait(uint32_t bar, uint32_t parity) {
#pragma unroll 1
  for (int i = 0; i < 8; ++i)
    if (__all_sync(0xffffffffu, mbar_try_wait(bar, parity))) return true;
  return warp_wait_long(bar, parity);
}
__device__ __forceinline__ void copy4_async(uint32_t dst, const void* src) {
  asm volatile("cp.async.ca.shared.global [%0], [%1], 4;" ::"r"(dst), "l"(src) : "memory");
}
__device__ __forceinline__ void copy16_async(uint32_t dst, const void* src) {   // through L2 alone
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(dst), "l"(src) : "memory");
}
__device__ __forceinline__ void copies_done() { asm volatile("cp.async.wait_all;" ::: "memory"); }
__device__ __forceinline__ void tma_2d(uint32_t dst, const CUtensorMap* map, int c0, int c1, uint32_t bar) {
  asm volatile(
      "cp.async.bulk.tensor.2d.shared::cluster.global.tile.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3}], [%4];" ::"r"(
          dst),
      "l"(map), "r"(c0), "r"(c1), "r"(bar)
      : "memory");
}
// D(16x8, f32) += A(16x16, f16, row) * B(16x8, f16, col)
__device__ __forceinline__ void mma16816(float* c, uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0,
                                         uint32_t b1) {
  asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, "
      "{%0,%1,%2,%3};"
      : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
      : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}
__device__ __forceinline__ uint32_t pack_half2(float lo, float hi) {
  const __half2 h = __floats2half2_rn(lo, hi);
  return *reinterpret_cast<const uint32_t*>(&h);
}
// an 8x8 matrix of binary16 values (row lane / 4, columns 2 (lane % 4) and + 1), transposed
__device__ __forceinline__ uint32_t transpose8x8(uint32_t a) {
  uint32_t d;
  asm("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(d) : "r"(a));
  return d;
}
__device__ __forceinline__ float fast_exp2(float x) {   // 2^x, 2 units in the last place; 0 for -inf
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}
// four e4m3 codes as two pairs of binary16 values (exact)
__device__ __forceinline__ void e4m3x4_to_half4(uint32_t w, uint32_t& lo, uint32_t& hi) {
  asm("{\n .reg .b16 l, h;\n mov.b32 {l, h}, %2;\n cvt.rn.f16x2.e4m3x2 %0, l;\n cvt.rn.f16x2.e4m3x2 %1, h;\n}"
      : "=r"(lo), "=r"(hi)
      : "r"(w));
}
// The token of a block at row n (of 16) of S^T: within eights, even rows keep
// their place and odd ones are crossed, so that the two rows of a quarter-warp's
// K read differ in bit 2 and the four rows of its V read in bits 1 and 2 -- with
// the swizzle, 8 different 16-byte banks either way.
__device__ __forceinline__ int token_of(int n) { return (n & 8) | ((n & 1) ? ((n & 6) ^ 5) : (n & 7)); }

// A CTA a pair, where there are enough CTAs and no warp then has more than one tile
// more than with equal shares: it saves the merge across CTAs (tickets and a round
// trip through L2).  One sequence, 14/2 heads of 64: 150 tokens 6.7 us against 12.0,
// 500 tokens (a tile more) 9.0 against 10.7, but 1500 tokens (three more) 12.7 against
// 10.3; several pairs a CTA one after the other, 64 sequences of 256 tokens, 32/8 heads
// of 128, 25.7 against 19.2.  Equal shares otherwise: 32 sequences x 32768 tokens, 32/8
// heads of 128, 332 us; with the last sixth of the work dealt out in small chunks as
// CTAs finish 351 us (each chunk drains a CTA's pipeline), and two CTAs an SM instead
// of one larger 364 us.
template <int W>
__device__ __forceinline__ Plan plan_of(unsigned total, int longest, int all_pairs, int ctas) {
  Plan pl;
  pl.total = total;
  const unsigned even = max(1u, (total + ctas * W - 1) / (ctas * W));
  const unsigned rounds = (all_pairs + ctas - 1) / ctas;
  pl.whole = rounds == 1 && (longest + W - 1) / W <= even + 1;
  pl.chunk = even * W;
  return pl;
}

// tiles of a pair of sequence b; none for a length outside 0 .. capacity
__device__ __forceinline__ int tiles_of(const Params& p, int b) {
  const int n = p.seqlens[b];
  return n < 0 || n > p.page_tokens * p.max_pages ? 0 : (n + kTile - 1) / kTile;
}

constexpr int kMaxWarps = 12;
enum { kHas0 = 1, kEnds0 = 2, kParked0 = 4, kHas1 = 8 };
struct Control {     // in shared memory
  Part part[kMaxWarps][2];   // [0] a pair begun before the warp's stretch, [1] one that goes on after it
  int flags[kMaxWarps];      // kHas0 ...
  int longest[kMaxWarps];    // tiles of a pair that the warp has seen
  int last[2];
  uint2 open[2];             // first CTA and number of CTAs of a pair that spans several
  Plan plan;                 // out of the registers of the tile loop; every warp writes the same
};

// One warp's stretch: `count` tiles from tile `begin` of the row on, b and base a
// sequence no later than the first tile's and where its tiles start.  Pairs inside
// it are finished, the states of others left for merge_states.
template <int D, int TYPE, int RT>
__device__ __forceinline__ void run_stretch(const CUtensorMap& mk, const CUtensorMap& mv, const Params& p,
                                         unsigned char* smem, Control& ctl, unsigned begin, int count,
                                         int b_first, unsigned base_first) {
  using S = Shape<D, RT>;
  constexpr int KS = D / 16;        // k-steps of S, m-tiles of O^T
  constexpr int NC = D / 64;        // 16-byte K chunks of a lane
  constexpr int VW = D / 32;        // V words of a lane and token
  constexpr int W = S::kWarps;
  const int warp = threadIdx.x / 32, lane = threadIdx.x % 32;
  const int g = lane / 4, c = lane % 4;
  unsigned char* ring = smem + warp * S::kRingBytes;
  Meta* meta = reinterpret_cast<Meta*>(smem + S::kMetaOffset) + warp * S::kSlots;   // of tile j: slot j % kSlots
  const uint32_t bar0 = smem_u32(smem + S::kBarOffset) + warp * S::kStages * 8;
  const int pairs = p.Hkv * p.row_groups.d, Q = p.Q;
  const bool wide = p.wide;
  const int* seqlens = p.seqlens;
  const unsigned* group_tiles = reinterpret_cast<const unsigned*>(smem + S::kGroupOffset);   // of B > 32 sequences
  // the scores' scale in the log2 domain (int8: codes enter S as c 2^-24)
  const float scale = p.scale_log2 * (TYPE == q8::kInt8 ? 0x1p24f : 1.0f);
  bool ok = true;

  // ---- the tiles' slots, 16 at a time, a lane each block: first which tiles they
  // are (and the page-table word, on its way), later their rows and scales.  b: a
  // sequence no later than the first tile's, base: where its tiles start ----
  const int half = lane & 1;
  auto name_tiles = [&](int j0, int b, unsigned base) {
    const unsigned x = begin + min(j0 + lane / 2, count - 1);
    int n = tiles_of(p, b);
    while (x - base >= (unsigned)n * pairs && b + 1 < p.B) {
      base += (unsigned)n * pairs;
      // whole groups at a time where idle slots leave many without a tile (two sequences of
      // 8000 tokens, 4094 slots between them: 38 us; stepping over each slot 284)
      for (++b; b % 32 == 0 && b + 32 < p.B && x - base >= group_tiles[b / 32] * pairs; b += 32)
        base += group_tiles[b / 32] * pairs;
      n = tiles_of(p, b);
    }
    // the bounds below hold by themselves unless the lengths change under the kernel
    n = max(n, 1);
    const unsigned rel = x - base;
    const unsigned pair = min(rel / (unsigned)n, (unsigned)pairs - 1u), tile = min(rel - pair * n, (unsigned)n - 1u);
    // a tile without a second block has its first one twice
    unsigned t = tile * kTile + half * kBlock;
    if ((int)t >= p.seqlens[b]) t = tile * kTile;
    const unsigned logical = min(t / (unsigned)p.page_tokens, (unsigned)p.max_pages - 1u);
    Meta& md = meta[(j0 + lane / 2) & (S::kSlots - 1)];
    copy4_async(smem_u32(&md.word[half]), p.page_table + (size_t)b * p.max_pages + logical);
    md.row[half] = t % (unsigned)p.page_tokens;   // of its page, for now
    if (half == 0) *reinterpret_cast<int4*>(&md.tile) = make_int4(tile, n, b, pair);
  };
  auto find_tiles = [&](int j0) {   // after a barrier of the warp since name_tiles
    Meta& md = meta[(j0 + lane / 2) & (S::kSlots - 1)];
    copies_done();   // this lane's own
    const uint32_t word = md.word[half];
    unsigned page = word & 0x7FFFFFFFu;
    if (!(word >> 31) || page >= (unsigned)p.num_pages) {   // the copies then stay inside the pool
      atomicOr(p.dev_err, ANVILQ_DEV_ERR_PAGE);
      page = 0;
    }
    // rows of a pool fit an int
    const int row = (int)(page * p.Hkv + p.row_groups.quotient(md.pair)) * p.page_tokens + md.row[half];
    md.row[half] = row;
    copy4_async(smem_u32(&md.ks[half]), p.k_scales + row / kBlock);
    copy4_async(smem_u32(&md.vs[half]), p.v_scales + row / kBlock);
  };
  auto copy = [&](int j) {
    if (lane == 0) {
      const uint32_t st = j & (S::kStages - 1);
      const uint32_t bar = bar0 + 8 * st, dst = smem_u32(ring) + st * S::kStageBytes;
      const int2 row = *reinterpret_cast<const int2*>(meta[j & (S::kSlots - 1)].row);
      asm volatile("mbarrier.arrive.expect_tx.shared::cta.b64 _, [%0], %1;" ::"r"(bar), "r"(S::kStageBytes) : "memory");
      tma_2d(dst, &mk, 0, row.x, bar);
      tma_2d(dst + S::kTileBytes, &mv, 0, row.x, bar);
      if (!wide) {
        tma_2d(dst + S::kTileBytes / 2, &mk, 0, row.y, bar);
        tma_2d(dst + S::kTileBytes * 3 / 2, &mv, 0, row.y, bar);
      }
    }
  };

  // ---- the state of the current pair ----
  uint32_t qb[KS][RT][2];    // B fragments of Q^T: row 8 t + g
  // of rows 8 t + 2 c and + 1, as all that follows:
  float start[RT][2];        // where S^T's accumulators start (int8)
  float m[RT][2], l[RT][2];  // the softmax's reference; the lane's share of its sum
  float o[RT][KS][4];        // O^T: two dims, two rows
  float F = 1.0f, F_inv = 1.0f;
  int flags = 0;

  auto begin_pair = [&](const Meta& md) {   // its query rows, and an empty state
    const int kvh = p.row_groups.quotient(md.pair), r0 = (md.pair - kvh * p.row_groups.d) * S::kRows;
#pragma unroll
    for (int t = 0; t < RT; ++t) {
      const int r = r0 + 8 * t + g, i = p.group.quotient(r);
      const bool row = i < p.Q;
      const __half* src =
          p.q + (((size_t)md.b * p.Q + (row ? i : 0)) * p.Hq + kvh * p.group.d + r - i * p.group.d) * D + 16 * c;
#pragma unroll
      for (int h = 0; h < NC; ++h)
#pragma unroll
        for (int u = 0; u < 2; ++u) {
          uint4 w = make_uint4(0, 0, 0, 0);
          if (row) w = *reinterpret_cast<const uint4*>(src + 64 * h + 8 * u);
          qb[4 * h + 2 * u][t][0] = w.x;
          qb[4 * h + 2 * u][t][1] = w.y;
          qb[4 * h + 2 * u + 1][t][0] = w.z;
          qb[4 * h + 2 * u + 1][t][1] = w.w;
        }
      m[t][0] = m[t][1] = -1e30f;
      l[t][0] = l[t][1] = 0.0f;
#pragma unroll
      for (int mt = 0; mt < KS; ++mt) o[t][mt][0] = o[t][mt][1] = o[t][mt][2] = o[t][mt][3] = 0.0f;
    }
    F = F_inv = 1.0f;
  };
  int issued = 0, j = 0;
  if (count > 0) {
    name_tiles(0, b_first, base_first);
    __syncwarp();
    begin_pair(meta[0]);      // q's loads travel with the page-table words
    find_tiles(0);
    __syncwarp();
    const int ahead = min(S::kStages, count);
    for (; issued < ahead; ++issued) copy(issued);
    copies_done();
    __syncwarp();
  }

#pragma unroll 1
  for (; j < count; ++j) {
    const uint32_t st = j & (S::kStages - 1);
    const Meta& slot = meta[j & (S::kSlots - 1)];
    const struct { int tile, n; } md = {slot.tile, slot.n};
    const bool fresh = j == 0 || md.tile == 0;
    if (fresh && j > 0) begin_pair(slot);
    if ((p.expire && (p.expire >> ((blockIdx.x + warp + j) & 15) & 1u)) ||
        !warp_wait(bar0 + 8 * st, j / S::kStages & 1)) {   // no tile is used after this
      ok = false;
      if (lane == 0) atomicOr(p.dev_err, ANVILQ_DEV_ERR_TIMEOUT);
      break;
    }
    if (TYPE == q8::kInt8 && fresh) {
#pragma unroll
      for (int t = 0; t < RT; ++t) {
        float sum = 0.0f;
#pragma unroll
        for (int ks = 0; ks < KS; ++ks)
#pragma unroll
          for (int e = 0; e < 2; ++e) {
            const float2 f = __half22float2(*reinterpret_cast<const __half2*>(&qb[ks][t][e]));
            sum += f.x + f.y;
          }
        sum += __shfl_xor_sync(0xffffffffu, sum, 1);
        sum += __shfl_xor_sync(0xffffffffu, sum, 2);
        sum *= -0x1p-17f;   // -128 2^-24
        start[t][0] = __shfl_sync(0xffffffffu, sum, 8 * c);
        start[t][1] = __shfl_sync(0xffffffffu, sum, 8 * c + 4);
      }
    }

    const unsigned char* tile = ring + st * S::kStageBytes;
    float x[2][RT][4];   // scores of both blocks: tokens token_of(g), then + 8; two rows each
    bool edge[2];
    int len = 0;
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      const unsigned char* kt = tile + h * kBlock * D;
      const int t0 = md.tile * kTile + h * kBlock;
      // ---- S^T = K Q^T: tokens token_of(g) and + 8, rows 8 t + 2 c and + 1 ----
      float s[2][RT][4];   // two sums: an accumulator's next MMA waits for its last
#pragma unroll
      for (int t = 0; t < RT; ++t)
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          s[0][t][e] = TYPE == q8::kInt8 ? start[t][e & 1] : 0.0f;
          s[1][t][e] = 0.0f;
        }
      uint4 w[NC][2];
#pragma unroll
      for (int q = 0; q < NC; ++q)
#pragma unroll
        for (int z = 0; z < 2; ++z) {
          const int row = token_of(g) + 8 * z;
          const int at =
              D == 128 ? row * 128 + (((c + 4 * q) ^ (row & 7)) << 4) : row * 64 + ((c ^ ((row >> 1) & 3)) << 4);
          w[q][z] = *reinterpret_cast<const uint4*>(kt + at);
        }
#pragma unroll
      for (int q = 0; q < NC; ++q)
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          uint32_t a[2][2];   // [token][pair of dims]
#pragma unroll
          for (int z = 0; z < 2; ++z) {
            const uint4 k = w[q][z];
            const uint32_t v = e == 0 ? k.x : e == 1 ? k.y : e == 2 ? k.z : k.w;
            if (TYPE == q8::kInt8) {
              const uint32_t u = v ^ 0x80808080u;
              a[z][0] = __byte_perm(u, 0, 0x4140);
              a[z][1] = __byte_perm(u, 0, 0x4342);
            } else {
              e4m3x4_to_half4(v, a[z][0], a[z][1]);
            }
          }
#pragma unroll
          for (int t = 0; t < RT; ++t)
            mma16816(s[e & 1][t], a[0][0], a[1][0], a[0][1], a[1][1], qb[4 * q + e][t][0], qb[4 * q + e][t][1]);
        }

      const float ks = slot.ks[h] * scale;
#pragma unroll
      for (int t = 0; t < RT; ++t)
#pragma unroll
        for (int e = 0; e < 4; ++e) x[h][t][e] = (s[0][t][e] + s[1][t][e]) * ks;
      // some row may not see all of the block: length >= 32 (n - 1) + 1, row 0 sees Q - 1 less
      edge[h] = t0 + kBlock > kTile * (md.n - 1) + 2 - Q;
      if (edge[h]) {
        len = seqlens[slot.b];
        const int r0 = (slot.pair - p.row_groups.quotient(slot.pair) * p.row_groups.d) * S::kRows;
#pragma unroll
        for (int t = 0; t < RT; ++t)
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            const int sees = len - Q + 1 + p.group.quotient(r0 + 8 * t + 2 * c + (e & 1)) - t0;
            if (token_of(g) + 8 * (e >> 1) >= sees) x[h][t][e] = -INFINITY;
          }
      }
    }
    // ---- softmax: the reference for both blocks ----
    {
      float mx[RT][2];
      bool above = false;
#pragma unroll
      for (int t = 0; t < RT; ++t)
#pragma unroll
        for (int e = 0; e < 2; ++e) {
          mx[t][e] = fmaxf(fmaxf(x[0][t][e], x[0][t][2 + e]), fmaxf(x[1][t][e], x[1][t][2 + e]));
          above |= mx[t][e] > m[t][e] + 12.0f;
        }
      if (__any_sync(0xffffffffu, above)) {
#pragma unroll
        for (int t = 0; t < RT; ++t)
#pragma unroll
          for (int e = 0; e < 2; ++e) {
#pragma unroll
            for (int z = 4; z < 32; z <<= 1) mx[t][e] = fmaxf(mx[t][e], __shfl_xor_sync(0xffffffffu, mx[t][e], z));
            const float m_new = mx[t][e] > m[t][e] + 12.0f ? mx[t][e] - 4.0f : m[t][e];
            const float alpha = fast_exp2(m[t][e] - m_new);
            m[t][e] = m_new;
            l[t][e] *= alpha;
#pragma unroll
            for (int mt = 0; mt < KS; ++mt) {
              o[t][mt][e] *= alpha;
              o[t][mt][2 + e] *= alpha;
            }
          }
      }
    }
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      const unsigned char* vt = tile + S::kTileBytes + h * kBlock * D;
      const int t0 = md.tile * kTile + h * kBlock;
      const float vs = slot.vs[h];
      float rel = vs * F_inv;
      if ((rel > 8.0f || rel < 0.125f) && vs > 0.0f) {
        // values of scales below 2^-40 round to nothing in the binary16 result
        const float F_new = fmaxf(vs, 0x1p-40f);
        const float f = F * (F_inv = 1.0f / F_new);
        F = F_new;
        rel = vs * F_inv;
#pragma unroll
        for (int t = 0; t < RT; ++t)
#pragma unroll
          for (int mt = 0; mt < KS; ++mt)
#pragma unroll
            for (int e = 0; e < 4; ++e) o[t][mt][e] *= f;
      }
      uint32_t pb[RT][2];
#pragma unroll
      for (int t = 0; t < RT; ++t) {
#pragma unroll
        for (int e = 0; e < 4; ++e) x[h][t][e] = fast_exp2(x[h][t][e] - m[t][e & 1]);
        l[t][0] += x[h][t][0] + x[h][t][2];
        l[t][1] += x[h][t][1] + x[h][t][3];
        pb[t][0] = transpose8x8(pack_half2(x[h][t][0] * rel, x[h][t][1] * rel));
        pb[t][1] = transpose8x8(pack_half2(x[h][t][2] * rel, x[h][t][3] * rel));
      }

      // ---- O^T += V^T P^T ----
      uint32_t v[4][VW];
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        const int row = token_of(2 * c + (e & 1)) + 8 * (e >> 1);
        if (D == 128) {
          const uint4 k = *reinterpret_cast<const uint4*>(vt + row * 128 + ((g ^ (row & 7)) << 4));
          v[e][0] = k.x; v[e][1] = k.y; v[e][2 % VW] = k.z; v[e][3 % VW] = k.w;
        } else {
          const uint2 k =
              *reinterpret_cast<const uint2*>(vt + row * 64 + (((g >> 1) ^ ((row >> 1) & 3)) << 4) + 8 * (g & 1));
          v[e][0] = k.x; v[e][1] = k.y;
        }
        // rows behind the sequence may hold anything: an e4m3 NaN times p = 0 would be a NaN
        if (TYPE == q8::kE4m3 && edge[h] && t0 + row >= len) {
#pragma unroll
          for (int w = 0; w < VW; ++w) v[e][w] = 0u;
        }
      }
#pragma unroll
      for (int w = 0; w < VW; ++w)
#pragma unroll
        for (int u = 0; u < 2; ++u) {
          // dims 4 w + 2 u and + 1 of the lane's chunk: bytes of tokens (0, 1), then (2, 3)
          const uint32_t p01 = __byte_perm(v[0][w], v[1][w], u ? 0x7362 : 0x5140);
          const uint32_t p23 = __byte_perm(v[2][w], v[3][w], u ? 0x7362 : 0x5140);
          uint32_t a[4];
          if (TYPE == q8::kInt8) {
            const __half2 off = __floats2half2_rn(1152.0f, 1152.0f);
            const uint32_t s01 = p01 ^ 0x80808080u, s23 = p23 ^ 0x80808080u;
            a[0] = __byte_perm(s01, 0x64646464u, 0x4140);
            a[1] = __byte_perm(s01, 0x64646464u, 0x4342);
            a[2] = __byte_perm(s23, 0x64646464u, 0x4140);
            a[3] = __byte_perm(s23, 0x64646464u, 0x4342);
#pragma unroll
            for (int e = 0; e < 4; ++e) {
              const __half2 d = __hsub2(*reinterpret_cast<__half2*>(&a[e]), off);
              a[e] = *reinterpret_cast<const uint32_t*>(&d);
            }
          } else {
            e4m3x4_to_half4(p01, a[0], a[1]);
            e4m3x4_to_half4(p23, a[2], a[3]);
          }
#pragma unroll
          for (int t = 0; t < RT; ++t) mma16816(o[t][2 * w + u], a[0], a[1], a[2], a[3], pb[t][0], pb[t][1]);
        }
    }
    __syncwarp();
    // the stage is free again
    if (issued < count) {
      copy(issued);
      ++issued;
      // the next 16 tiles' slots, well before they are needed: at 8 the last of
      // these slots' old tiles have been used (kStages <= 4)
      if ((issued & 3) == 0) {
        const int at = issued & 15, upcoming = issued - at + 16;
        if (at == 8 && upcoming < count) {
          const Meta& last = meta[(upcoming - 1) & (S::kSlots - 1)];
          name_tiles(upcoming, last.b, begin + upcoming - 1 - (unsigned)last.pair * last.n - last.tile);
        }
        if (at == 12 && upcoming < count) find_tiles(upcoming);
        if (at == 0) copies_done();
        __syncwarp();
      }
    }

    // ---- the pair's last tile here ----
    const bool ends = md.tile == md.n - 1;
    if (ends || j == count - 1) {
#pragma unroll
      for (int t = 0; t < RT; ++t)
#pragma unroll
        for (int e = 0; e < 2; ++e)
#pragma unroll
          for (int z = 4; z < 32; z <<= 1) l[t][e] += __shfl_xor_sync(0xffffffffu, l[t][e], z);
      const bool from_start = j >= md.tile;   // the pair's first tile is in this stretch
      const int sb = slot.b, sp = slot.pair;
      if (from_start && ends) {
        const int kvh = p.row_groups.quotient(sp), r0 = (sp - kvh * p.row_groups.d) * S::kRows;
#pragma unroll
        for (int t = 0; t < RT; ++t) {
#pragma unroll
          for (int e = 0; e < 2; ++e) {
            const float f = l[t][e] == 0.0f ? 0.0f : F / l[t][e];
            const int r = r0 + 8 * t + 2 * c + e, i = p.group.quotient(r);
            if (i < p.Q) {
              __half* dst =
                  p.out + (((size_t)sb * p.Q + i) * p.Hq + kvh * p.group.d + r - i * p.group.d) * D + g * (D / 8);
#pragma unroll
              for (int q = 0; q < NC; ++q) {
                uint4 w;
                w.x = pack_half2(o[t][4 * q][e] * f, o[t][4 * q][2 + e] * f);
                w.y = pack_half2(o[t][4 * q + 1][e] * f, o[t][4 * q + 1][2 + e] * f);
                w.z = pack_half2(o[t][4 * q + 2][e] * f, o[t][4 * q + 2][2 + e] * f);
                w.w = pack_half2(o[t][4 * q + 3][e] * f, o[t][4 * q + 3][2 + e] * f);
                reinterpret_cast<uint4*>(dst)[q] = w;
              }
            }
          }
        }
      } else {
        // the state: in the ring where the stretch is over, else (a pair begun
        // earlier, the ring in use) in this warp's place in global memory
        const int which = from_start ? 1 : 0;
        const bool parked = j < count - 1;
        float* state = parked ? p.parked + ((size_t)blockIdx.x * W + warp) * S::kState : reinterpret_cast<float*>(ring);
        float2* stat = reinterpret_cast<float2*>(smem + S::kStatOffset) + (warp * 2 + which) * S::kRows;
        __syncwarp();
#pragma unroll
        for (int t = 0; t < RT; ++t) {
#pragma unroll
          for (int e = 0; e < 2; ++e) {
            if (g == 0) stat[8 * t + 2 * c + e] = make_float2(m[t][e], l[t][e]);
            float4* dst = reinterpret_cast<float4*>(state + (8 * t + 2 * c + e) * D + g * (D / 8));
#pragma unroll
            for (int q = 0; q < KS / 2; ++q)
              dst[q] = make_float4(o[t][2 * q][e] * F, o[t][2 * q][2 + e] * F, o[t][2 * q + 1][e] * F,
                                   o[t][2 * q + 1][2 + e] * F);
          }
        }
        flags |= which ? kHas1 : kHas0 | (ends ? kEnds0 : 0) | (parked ? kParked0 : 0);
        if (lane == 0) ctl.part[warp][which] = Part{begin + j - md.tile, md.n, sb, sp};
      }
    }
  }
  if (!ok) {
    // Copies in flight land before the shared memory is used for anything else.
    for (int i = j; i < issued; ++i)
      if (!warp_wait(bar0 + 8 * (i & (S::kStages - 1)), i / S::kStages & 1)) break;
    // The output is lost, but not the accounts: empty states stand for what is left of
    // the stretch, so that every pair has all of its members, every ticket all of its
    // arrivals, and the workspace's counters are zero after this call as after any other.
    copies_done();
    __syncwarp();
    const Meta at = meta[j & (S::kSlots - 1)];
    __syncwarp();
    name_tiles(count - 1, at.b, begin + j - (unsigned)at.pair * at.n - at.tile);
    copies_done();
    __syncwarp();
    const Meta end = meta[(count - 1) & (S::kSlots - 1)];
    float4* state = reinterpret_cast<float4*>(ring);
    for (int i = lane; i < S::kState / 4; i += 32) state[i] = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
    auto leave_empty = [&](int which, const Meta& md, int k) {   // of the pair of tile k
      float2* stat = reinterpret_cast<float2*>(smem + S::kStatOffset) + (warp * 2 + which) * S::kRows;
      if (lane < S::kRows) stat[lane] = make_float2(-1e30f, 0.0f);
      if (lane == 0) ctl.part[warp][which] = Part{begin + k - md.tile, md.n, md.b, md.pair};
    };
    if (at.tile > j) {                                    // begun earlier
      leave_empty(0, at, j);
      flags |= kHas0 | (at.n - at.tile <= count - j ? kEnds0 : 0);
    }
    if (end.tile < count && end.tile < end.n - 1) {       // begun here, goes on
      leave_empty(1, end, count - 1);
      flags |= kHas1;
    }
  }
  if (lane == 0) ctl.flags[warp] = flags;
}

// Merges what the warps left.  Its loops keep few values at a time: the tile loop
// lives within the same registers, and a merge that held a state's sums of all
// members in registers made it spill (1.6 times the time).
template <int D, int RT>
__device__ __forceinline__ void merge_states(const Params& p, unsigned char* smem, Control& ctl) {
  using S = Shape<D, RT>;
  constexpr int W = S::kWarps;
  constexpr int kVec = S::kRows * (D / 4);   // float4s of a state
  auto finish = [&](const Part& pt, int at, float4 acc, float lsum) {   // at: float4 of the state
    const int row = at / (D / 4);
    const int kvh = p.row_groups.quotient(pt.pair), r = (pt.pair - kvh * p.row_groups.d) * S::kRows + row;
    const int i = p.group.quotient(r);
    if (i >= p.Q) return;
    const float inv = lsum == 0.0f ? 0.0f : 1.0f / lsum;
    __half* dst =
        p.out + (((size_t)pt.b * p.Q + i) * p.Hq + kvh * p.group.d + r - i * p.group.d) * D + 4 * (at % (D / 4));
    *reinterpret_cast<uint2*>(dst) =
        make_uint2(pack_half2(acc.x * inv, acc.y * inv), pack_half2(acc.z * inv, acc.w * inv));
  };
  auto add_state = [](float M, float& lsum, float4& acc, float2 ml, float4 v) {   // M: at least ml.x
    const float f = fast_exp2(ml.x - M);
    lsum += f * ml.y;
    acc.x += f * v.x; acc.y += f * v.y; acc.z += f * v.z; acc.w += f * v.w;
  };
  // A chain: the states of one pair in consecutive warps.  It begins with a
  // pair begun earlier in warp 0, or with a warp's pair that goes on.
  const float2* stats = reinterpret_cast<const float2*>(smem + S::kStatOffset);
  // bit w: warp w's; of starts bit 0: slot 0 of warp 0, bit w + 1: slot 1 of w
  unsigned has0, ends0, parked0, starts;
  {
    const int lane = threadIdx.x % 32, fl = lane < W ? ctl.flags[lane] : 0;
    has0 = __ballot_sync(0xffffffffu, fl & kHas0);
    ends0 = __ballot_sync(0xffffffffu, fl & kEnds0);
    parked0 = __ballot_sync(0xffffffffu, fl & kParked0);
    starts = __ballot_sync(0xffffffffu, fl & kHas1) << 1 | (has0 & 1);
  }
  int open = 0;        // bit s: the pair of ctl.part[open warp][s] spans CTAs
  int open_warp1 = 0;  // (that of slot 0 is warp 0's)
  // Chains are merged one after the other by all warps, or when there are many, as
  // short sequences leave them, by a warp each, a thread then taking U = 4 float4s of
  // the state at a time: 256 sequences of 1 .. 200 tokens, 32/8 heads of 128, 28.9 us
  // against 31.9, but 16 of up to 4096, a few chains of several warps each, 28.2
  // against 26.4.
  auto merge_chain = [&](auto each, int w, int slot, int members, bool whole, int me, int threads) {
    constexpr int U = decltype(each)::value;
    float* out = p.partials + ((size_t)blockIdx.x * 2 + slot) * S::kPartial;
    const float2* stat = stats + (w * 2 + slot) * S::kRows;   // of members after the first: slot 0 of their warps
    static_assert(kVec % (32 * U) == 0, "whole steps of a warp");
#pragma unroll 1
    for (int at0 = me; at0 < kVec; at0 += U * threads) {
      float M[U], lsum[U];
      float4 acc[U];
#pragma unroll
      for (int u = 0; u < U; ++u) {
        M[u] = stat[(at0 + u * threads) / (D / 4)].x;
        lsum[u] = 0.0f;
        acc[u] = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
      }
#pragma unroll (U == 1 ? 2 : 1)
      for (int k = 1; k < members; ++k)
#pragma unroll
        for (int u = 0; u < U; ++u)
          M[u] = fmaxf(M[u], stats[(w + k) * 2 * S::kRows + (at0 + u * threads) / (D / 4)].x);
#pragma unroll (U == 1 ? 2 : 1)
      for (int k = 0; k < members; ++k) {
        const bool parked = (k || !slot) && (parked0 >> (w + k) & 1);
        const float4* state =
            parked ? reinterpret_cast<const float4*>(p.parked + ((size_t)blockIdx.x * W + w + k) * S::kState)
                   : reinterpret_cast<const float4*>(smem + (w + k) * S::kRingBytes);
#pragma unroll
        for (int u = 0; u < U; ++u) {
          const int at = at0 + u * threads, row = at / (D / 4);
          add_state(M[u], lsum[u], acc[u], k ? stats[(w + k) * 2 * S::kRows + row] : stat[row], state[at]);
        }
      }
#pragma unroll
      for (int u = 0; u < U; ++u) {
        const int at = at0 + u * threads, row = at / (D / 4);
        if (whole) {
          finish(ctl.part[w][1], at, acc[u], lsum[u]);
        } else {
          __stcg(reinterpret_cast<float4*>(out) + at, acc[u]);
          if (at % (D / 4) == 0) __stcg(reinterpret_cast<float2*>(out + S::kState) + row, make_float2(M[u], lsum[u]));
        }
      }
    }
  };
  const bool alone = __popc(starts) > W / 2;
  const int warp = threadIdx.x / 32;
#pragma unroll 1
  for (int c = 0; starts; starts &= starts - 1, ++c) {
    const int slot = (starts & 1) ? 0 : 1, w = max(__ffs(starts) - 2, 0);
    int members = 1;
    bool ended = slot == 0 && (ends0 & 1);
    while (!ended && (has0 >> (w + members) & 1)) {
      ended = ends0 >> (w + members) & 1;
      ++members;
    }
    const bool whole = slot == 1 && ended;
    if (!alone)
      merge_chain(std::integral_constant<int, 1>(), w, slot, members, whole, threadIdx.x, S::kThreads);
    else if (c == warp || c == warp + W)
      merge_chain(std::integral_constant<int, 4>(), w, slot, members, whole, threadIdx.x % 32, 32);
    if (!whole) {
      open |= 1 << slot;
      if (slot) open_warp1 = w;
    }
  }

  // ---- pairs that span CTAs: the last CTA to arrive merges, in CTA order ----
  __syncthreads();   // the partials are written (and the rings free again)
  if (!open) return;
  if (threadIdx.x < 2) {
    const int slot = threadIdx.x;
    bool last = false;
    if (open >> slot & 1) {
      const Part pt = ctl.part[slot ? open_warp1 : 0][slot];
      const unsigned c0 = pt.first / ctl.plan.chunk, c1 = (pt.first + pt.n - 1) / ctl.plan.chunk;
      int* ticket = p.tickets + c0;
      // releases the CTA's partials (through the barrier above) and acquires the others'
      int arrived;
      asm volatile("atom.acq_rel.gpu.global.add.s32 %0, [%1], 1;" : "=r"(arrived) : "l"(ticket) : "memory");
      last = arrived == (int)(c1 - c0);
      if (last) *ticket = 0;
      ctl.open[slot] = make_uint2(c0, c1 - c0 + 1);
    }
    ctl.last[slot] = last;
  }
  __syncthreads();
  // Both merges at once where there are two, each by half of the warps with half
  // of the rings: their time is latency.
  const int both = ctl.last[0] + ctl.last[1];
  if (!both) return;
  static_assert(W % 2 == 0, "two halves");
  const int threads = both == 2 ? S::kThreads / 2 : S::kThreads;
  const int slot = both == 2 ? (int)threadIdx.x / threads : ctl.last[1];
  const int me = both == 2 ? threadIdx.x % threads : threadIdx.x;
  unsigned char* room = smem + (both == 2 ? slot * (W / 2) * S::kRingBytes : 0);
  constexpr int kFitAll = W * S::kRingBytes / (S::kPartial * 4), kFitHalf = W / 2 * S::kRingBytes / (S::kPartial * 4);
  const int fit = both == 2 ? kFitHalf : kFitAll;                         // states that fit the room
  constexpr int kMine = (2 * kVec + S::kThreads - 1) / S::kThreads;       // float4s of a thread, at most
  auto sync = [&] { asm volatile("bar.sync %0, %1;" ::"r"(1 + slot), "r"(threads) : "memory"); };
  const unsigned c0 = ctl.open[slot].x;
  const int n = (int)ctl.open[slot].y;
  float M[kMine], lsum[kMine];
  float4 acc[kMine];
#pragma unroll
  for (int i = 0; i < kMine; ++i) {
    M[i] = -1e30f;
    lsum[i] = 0.0f;
    acc[i] = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
  }
#pragma unroll 1
  for (int k0 = 0; k0 < n; k0 += fit) {
    const int m = min(fit, n - k0);
    // the states of m CTAs, all on their way at once
#pragma unroll 1
    for (int k = 0; k < m; ++k) {
      // the first CTA's state is of a pair that goes on, the others' of one begun earlier
      const float* from = p.partials + ((size_t)(c0 + k0 + k) * 2 + (k0 + k == 0)) * S::kPartial;
#pragma unroll 2
      for (int at = me; at < S::kPartial / 4; at += threads)
        copy16_async(smem_u32(room) + (k * (S::kPartial / 4) + at) * 16, from + 4 * at);
    }
    copies_done();
    sync();
    const float* state = reinterpret_cast<const float*>(room);
#pragma unroll
    for (int i = 0; i < kMine; ++i) {
      const int at = me + i * threads, row = at / (D / 4);
      if (at >= kVec) break;
      float top = M[i];
#pragma unroll 4
      for (int k = 0; k < m; ++k) top = fmaxf(top, state[k * S::kPartial + S::kState + 2 * row]);
      const float old = fast_exp2(M[i] - top);
      M[i] = top;
      lsum[i] *= old;
      acc[i].x *= old; acc[i].y *= old; acc[i].z *= old; acc[i].w *= old;
#pragma unroll 4
      for (int k = 0; k < m; ++k)
        add_state(top, lsum[i], acc[i], reinterpret_cast<const float2*>(state + k * S::kPartial + S::kState)[row],
                  reinterpret_cast<const float4*>(state + k * S::kPartial)[at]);
    }
    if (k0 + fit < n) sync();   // the room is used again
  }
#pragma unroll
  for (int i = 0; i < kMine; ++i) {
    const int at = me + i * threads;
    if (at < kVec) finish(ctl.part[slot ? open_warp1 : 0][slot], at, acc[i], lsum[i]);
  }
}

template <int D, int TYPE, int RT>
__global__ void __launch_bounds__(Shape<D, RT>::kThreads, 1)
    gqa_decode_q8_kernel(const __grid_constant__ CUtensorMap mk, const __grid_constant__ CUtensorMap mv,
                         const __grid_constant__ Params p) {
  using S = Shape<D, RT>;
  constexpr int W = S::kWarps;
  extern __shared__ __align__(1024) unsigned char smem_raw[];
  __shared__ Control ctl;
  unsigned char* smem = smem_raw + ((1024u - (smem_u32(smem_raw) & 1023u)) & 1023u);
  const int warp = threadIdx.x / 32, lane = threadIdx.x % 32;
  const uint32_t bar0 = smem_u32(smem + S::kBarOffset) + warp * S::kStages * 8;
  if (lane == 0) {
    for (int s = 0; s < S::kStages; ++s)
      asm volatile("mbarrier.init.shared::cta.b64 [%0], 1;" ::"r"(bar0 + 8 * s) : "memory");
    asm volatile("prefetch.tensormap [%0];" ::"l"(&mk) : "memory");
    asm volatile("prefetch.tensormap [%0];" ::"l"(&mv) : "memory");
  }
  asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
  __syncwarp();
  asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
  asm volatile("griddepcontrol.wait;" ::: "memory");

  const int capacity = p.page_tokens * p.max_pages;   // <= 2^30
  // ---- the row of all tiles: its length, its longest pair ----
  // Up to 32 sequences every warp counts for itself (no barrier).  More: the warps
  // share the counting, 32 sequences a group.  (Every warp counting all:
  // 1024 sequences of 1 .. 64 tokens, 32/8 heads of 128, 40.0 us against 35.4.)
  const int pairs = p.Hkv * p.row_groups.d;   // of a sequence
  unsigned* group_tiles = reinterpret_cast<unsigned*>(smem + S::kGroupOffset);
  {
    const int groups = (p.B + 31) / 32;
    unsigned sum = 0;
    int longest = 0;
    if (groups == 1) {
      const int n = lane < p.B ? tiles_of(p, lane) : 0;
      sum = __reduce_add_sync(0xffffffffu, (unsigned)n);
      longest = __reduce_max_sync(0xffffffffu, n);
    } else {
#pragma unroll 4
      for (int i = warp; i < groups; i += W) {
        const int b = 32 * i + lane, n = b < p.B ? tiles_of(p, b) : 0;
        const unsigned tiles = __reduce_add_sync(0xffffffffu, (unsigned)n);
        if (lane == 0) group_tiles[i] = tiles;
        longest = max(longest, n);
      }
      longest = __reduce_max_sync(0xffffffffu, longest);
      if (lane == 0) ctl.longest[warp] = longest;
      __syncthreads();
      for (int i = lane; i < groups; i += 32) sum += group_tiles[i];
      sum = __reduce_add_sync(0xffffffffu, sum);
      longest = __reduce_max_sync(0xffffffffu, lane < W ? ctl.longest[lane] : 0);
    }
    const Plan plan = plan_of<W>(sum * pairs, longest, p.B * pairs, gridDim.x);
    if (lane == 0) ctl.plan = plan;
    __syncwarp();
  }
  // ---- this warp's stretch: `count` tiles from `begin` on ----
  unsigned begin = 0;
  int count = 0;
  int b_first = 0;           // the sequence of the first tile, and where its tiles start
  unsigned base_first = 0;
  if (ctl.plan.whole) {
    if (blockIdx.x < (unsigned)(p.B * pairs)) {
      b_first = blockIdx.x / pairs;
      const int n = tiles_of(p, b_first), share = (n + W - 1) / W;
      // any row's start will do: nothing refers to tiles of other sequences
      begin = (blockIdx.x - b_first * pairs) * n + warp * share;
      count = max(0, min(n - warp * share, share));
    }
  } else {
    const unsigned share = ctl.plan.chunk / W;
    begin = blockIdx.x * ctl.plan.chunk + warp * share;
    count = begin < ctl.plan.total ? (int)min(share, ctl.plan.total - begin) : 0;
    // of 32 runs of tiles, the next from base_first on, the one that holds `begin`
    // (moving base_first there); 32 where none does
    auto holds = [&](unsigned tiles) {
      unsigned incl = tiles;
#pragma unroll
      for (int o = 1; o < 32; o <<= 1) {
        const unsigned up = __shfl_up_sync(0xffffffffu, incl, o);
        if (lane >= o) incl += up;
      }
      const uint32_t past = __ballot_sync(0xffffffffu, base_first + incl > begin);
      const int l = past ? __ffs(past) - 1 : 32;
      base_first += __shfl_sync(0xffffffffu, past ? incl - tiles : incl, min(l, 31));
      return l;
    };
    if (count > 0) {   // some sequence holds it, as begin < total
      int group = 0;
      const int groups = (p.B + 31) / 32;
      for (int l = 32; groups > 1 && l == 32 && group < groups; group += l)
        l = holds(group + lane < groups ? group_tiles[group + lane] * pairs : 0);
      const int b = 32 * group + lane;
      b_first = 32 * group + holds(b < p.B ? tiles_of(p, b) * pairs : 0);
      b_first = min(b_first, p.B - 1);
    }
  }
  run_stretch<D, TYPE, RT>(mk, mv, p, smem, ctl, begin, count, b_first, base_first);
  __syncthreads();
  merge_states<D, RT>(p, smem, ctl);
  // empty sequences (and lengths that are none)
  for (int b0 = blockIdx.x; b0 < p.B; b0 += 32 * gridDim.x) {   // a lane each, 32 at a time
    const int b = b0 + lane * gridDim.x, len = b < p.B ? p.seqlens[b] : 1;
    if (warp == 0 && (len < 0 || len > capacity)) atomicOr(p.dev_err, ANVILQ_DEV_ERR_SEQLEN);
    for (uint32_t none = __ballot_sync(0xffffffffu, len < 1 || len > capacity); none; none &= none - 1) {
      uint4* o = reinterpret_cast<uint4*>(p.out + (size_t)(b0 + (__ffs(none) - 1) * gridDim.x) * p.Q * p.Hq * D);
      for (int i = threadIdx.x; i < p.Q * p.Hq * (D / 8); i += S::kThreads) o[i] = make_uint4(0, 0, 0, 0);
    }
  }
}

// ---------------------------------------------------------------------------
static bool a16(const void* p) { return (reinterpret_cast<uintptr_t>(p) & 15u) == 0; }

// A block's scale (at most 729, of a rotated binary16 65504) times the softmax scale times
// 2^24 log2(e) stays below binary32's largest value.
constexpr float kMaxScale = 0x1p64f;
constexpr int kMaxQueries = 64;   // query tokens of a sequence
static bool shape_ok(int B, int Q, int Hq, int Hkv, int D) {
  return B >= 1 && B < kMaxBatch && Q >= 1 && Q <= kMaxQueries && Hkv >= 1 && Hq >= Hkv && Hq % Hkv == 0 &&
         Hq <= 1024 && (D == 64 || D == 128);
}

constexpr int kMaxDevices = 64;
static int g_sms[kMaxDevices];
static std::once_flag g_once[kMaxDevices];
template <int D, int TYPE, int RT>
static void allow_smem() {
  cudaFuncSetAttribute(gqa_decode_q8_kernel<D, TYPE, RT>, cudaFuncAttributeMaxDynamicSharedMemorySize,
                       Shape<D, RT>::kTotal);
}
static int sm_count() {
  int dev = 0;
  if (cudaGetDevice(&dev) != cudaSuccess || dev < 0 || dev >= kMaxDevices) return 0;
  std::call_once(g_once[dev], [dev] {
    cudaDeviceGetAttribute(&g_sms[dev], cudaDevAttrMultiProcessorCount, dev);
    allow_smem<64, q8::kInt8, 1>();
    allow_smem<64, q8::kInt8, 2>();
    allow_smem<64, q8::kE4m3, 1>();
    allow_smem<64, q8::kE4m3, 2>();
    allow_smem<128, q8::kInt8, 1>();
    allow_smem<128, q8::kInt8, 2>();
    allow_smem<128, q8::kE4m3, 1>();
    allow_smem<128, q8::kE4m3, 2>();
    cudaGetLastError();
  });
  return g_sms[dev];
}

// 8 rows a pair where they suffice, else 16 (the MMA's row count): more rows
// would leave too few registers for enough warps
static int row_tiles(int Q, int Hq, int Hkv) { return Q * (Hq / Hkv) <= 8 ? 1 : 2; }
static int max_ctas(int sms) { return std::min(sms, kMaxSms); }
static size_t partial_floats(int rt, int D, int sms) { return (size_t)max_ctas(sms) * 2 * (8 * rt) * (D + 2); }
static size_t parked_floats(int rt, int D, int sms) {
  return (size_t)max_ctas(sms) * (rt == 1 ? Shape<64, 1>::kWarps : Shape<64, 2>::kWarps) * (8 * rt) * D;
}

static std::once_flag g_encode_once;
static PFN_cuTensorMapEncodeTiled_v12000 g_encode = nullptr;

// A pool's codes as a matrix of D-byte rows, swizzled over the row's length; one box
// is a tile where pages hold whole ones, else a block.
static bool pool_map(CUtensorMap* map, const void* codes, long long rows, int D, int box_rows) {
  std::call_once(g_encode_once, [] {
    void* fn = nullptr;
    cudaDriverEntryPointQueryResult q;
    if (cudaGetDriverEntryPoint("cuTensorMapEncodeTiled", &fn, cudaEnableDefault, &q) == cudaSuccess &&
        q == cudaDriverEntryPointSuccess)
      g_encode = reinterpret_cast<PFN_cuTensorMapEncodeTiled_v12000>(fn);
    cudaGetLastError();
  });
  if (!g_encode) return false;
  const cuuint64_t dims[2] = {(cuuint64_t)D, (cuuint64_t)rows};
  const cuuint64_t strides[1] = {(cuuint64_t)D};
  const cuuint32_t box[2] = {(cuuint32_t)D, (cuuint32_t)box_rows};
  const cuuint32_t estr[2] = {1, 1};
  return g_encode(map, CU_TENSOR_MAP_DATA_TYPE_UINT8, 2, const_cast<void*>(codes), dims, strides, box, estr,
                  CU_TENSOR_MAP_INTERLEAVE_NONE, D == 128 ? CU_TENSOR_MAP_SWIZZLE_128B : CU_TENSOR_MAP_SWIZZLE_64B,
                  CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}

template <int D, int TYPE, int RT>
static int launch(const CUtensorMap& mk, const CUtensorMap& mv, const Params& p, int ctas, unsigned flags,
                  cudaStream_t st) {
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(ctas);
  cfg.blockDim = dim3(Shape<D, RT>::kThreads);
  cfg.dynamicSmemBytes = Shape<D, RT>::kTotal;
  cfg.stream = st;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = attr;
  cfg.numAttrs = (flags & ANVILQ_GEMM_OVERLAP_PRIOR) ? 1 : 0;
  if (cudaLaunchKernelEx(&cfg, gqa_decode_q8_kernel<D, TYPE, RT>, mk, mv, p) != cudaSuccess) {
    cudaGetLastError();
    return ANVILQ_ECUDA;
  }
  return ANVILQ_OK;
}

}  // namespace attn8
}  // namespace anvilq

extern "C" {

size_t anvilq_gqa_decode_q8_workspace_size(int B, int Q, int Hq, int Hkv, int D) {
  using namespace anvilq::attn8;
  if (!shape_ok(B, Q, Hq, Hkv, D)) return 0;
  const int sms = sm_count();
  if (sms <= 0) return 0;
  const int rt = row_tiles(Q, Hq, Hkv);
  return ANVILQ_WORKSPACE_COUNTER_BYTES + (partial_floats(rt, D, sms) + parked_floats(rt, D, sms)) * sizeof(float);
}

int anvilq_gqa_decode_q8(const uint16_t* q, const void* k_codes, const void* v_codes, const float* k_scales,
                         const float* v_scales, int code_type, const uint32_t* page_table, const int32_t* seqlens,
                         uint16_t* out, int B, int Q, int Hq, int Hkv, int D, int page_tokens, int max_pages,
                         int num_pages, float scale, void* workspace, size_t workspace_bytes, int* dev_err,
                         unsigned flags, anvilq_stream_t stream) {
  using namespace anvilq;
  using namespace anvilq::attn8;
  if (!q || !k_codes || !v_codes || !k_scales || !v_scales || !page_table || !seqlens || !out || !dev_err)
    return ANVILQ_EINVAL;
  if (code_type != ANVILQ_KV_Q8_INT8 && code_type != ANVILQ_KV_Q8_E4M3) return ANVILQ_EINVAL;
  if (flags & ~(ANVILQ_GEMM_OVERLAP_PRIOR | ANVILQ_EXPIRE_WAITS(0xFFFF))) return ANVILQ_EINVAL;
  if (!std::isfinite(scale) || scale > kMaxScale) return ANVILQ_EINVAL;
  if (!shape_ok(B, Q, Hq, Hkv, D) || page_tokens < kBlock || page_tokens % kBlock || max_pages < 1 || num_pages < 1 ||
      (long long)page_tokens * max_pages > (1LL << 30))
    return ANVILQ_ESHAPE;
  const long long positions = (long long)num_pages * page_tokens;
  if (positions > 0x7FFFFFFFLL / Hkv) return ANVILQ_ESHAPE;   // a TMA coordinate is an int
  const long long rows = positions * Hkv;
  const int rt = row_tiles(Q, Hq, Hkv), warps = rt == 1 ? Shape<128, 1>::kWarps : Shape<128, 2>::kWarps;
  const int row_groups = (Q * (Hq / Hkv) + 8 * rt - 1) / (8 * rt);
  const double all_pairs = (double)B * Hkv * row_groups;
  const double tiles = all_pairs * ((double)max_pages * page_tokens / kTile + 1);   // that the table has room for
  if (tiles > (double)(1u << 31)) return ANVILQ_ESHAPE;   // they are counted in 32 bits
  if (!a16(q) || !a16(k_codes) || !a16(v_codes) || !a16(out) || !a16(workspace)) return ANVILQ_EALIGN;
  // out may be q: a pair's rows are written when all that read them have done so
  const size_t rows_bytes = (size_t)B * Q * Hq * D * 2, codes = (size_t)rows * D, scales = (size_t)rows / kBlock * 4;
  if ((out != q && q8::overlap(out, rows_bytes, q, rows_bytes)) || q8::overlap(out, rows_bytes, k_codes, codes) ||
      q8::overlap(out, rows_bytes, v_codes, codes) || q8::overlap(out, rows_bytes, k_scales, scales) ||
      q8::overlap(out, rows_bytes, v_scales, scales) ||
      (workspace && q8::overlap(out, rows_bytes, workspace, workspace_bytes)))
    return ANVILQ_EINVAL;
  const int sms = sm_count();
  if (sms <= 0) return ANVILQ_ECUDA;
  if (!workspace || workspace_bytes < anvilq_gqa_decode_q8_workspace_size(B, Q, Hq, Hkv, D)) return ANVILQ_EWORKSPACE;
  Params p{};
  p.q = reinterpret_cast<const __half*>(q);
  p.k_scales = k_scales;
  p.v_scales = v_scales;
  p.page_table = page_table;
  p.seqlens = seqlens;
  p.out = reinterpret_cast<__half*>(out);
  p.tickets = static_cast<int*>(workspace);
  p.partials = reinterpret_cast<float*>(static_cast<char*>(workspace) + ANVILQ_WORKSPACE_COUNTER_BYTES);
  p.parked = p.partials + partial_floats(rt, D, sms);
  p.dev_err = dev_err;
  p.B = B; p.Q = Q; p.Hq = Hq; p.Hkv = Hkv;
  auto divisor = [](int d) { return Divisor{d, d == 1 ? 0u : (unsigned)(((1ull << 32) + d - 1) / d)}; };
  p.group = divisor(Hq / Hkv);
  p.row_groups = divisor(row_groups);
  p.page_tokens = page_tokens; p.max_pages = max_pages; p.num_pages = num_pages;
  p.expire = flags >> 16;
  p.scale_log2 = (scale > 0.0f ? scale : 1.0f / std::sqrt((float)D)) * 1.4426950408889634f;
  // as many CTAs as the device holds, but no more than there can be work for: a pair
  // each, or a tile a warp
  const int ctas = (int)std::min((double)max_ctas(sms), std::max(all_pairs, std::ceil(tiles / warps)));
  CUtensorMap mk, mv;
  p.wide = page_tokens % kTile == 0;
  const int box = p.wide ? kTile : kBlock;
  if (!pool_map(&mk, k_codes, rows, D, box) || !pool_map(&mv, v_codes, rows, D, box)) return ANVILQ_EALIGN;
  cudaStream_t st = reinterpret_cast<cudaStream_t>(stream);
  const bool int8 = code_type == ANVILQ_KV_Q8_INT8;
  if (D == 64)
    return int8 ? (rt == 1 ? launch<64, q8::kInt8, 1>(mk, mv, p, ctas, flags, st)
                           : launch<64, q8::kInt8, 2>(mk, mv, p, ctas, flags, st))
                : (rt == 1 ? launch<64, q8::kE4m3, 1>(mk, mv, p, ctas, flags, st)
                           : launch<64, q8::kE4m3, 2>(mk, mv, p, ctas, flags, st));
  return int8 ? (rt == 1 ? launch<128, q8::kInt8, 1>(mk, mv, p, ctas, flags, st)
                         : launch<128, q8::kInt8, 2>(mk, mv, p, ctas, flags, st))
              : (rt == 1 ? launch<128, q8::kE4m3, 1>(mk, mv, p, ctas, flags, st)
                         : launch<128, q8::kE4m3, 2>(mk, mv, p, ctas, flags, st));
}

}  // extern "C"
