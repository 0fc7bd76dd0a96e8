// gqa_chunk.cu -- attention of many new tokens a sequence over a paged binary16
// cache: prompts in chunks, questions about long documents, batches that mix them
// with decode steps.  Fifth-generation tensor cores (tcgen05), softmax in registers.
//
// Mathematics.  Token t of sequence b is at position pos = seqlens[b] - n_b + (t -
// start_b) (its n_b new tokens are its last, in the cache already); query head h reads
// kv head h / g, g = Hq / Hkv, and
//   out = sum_{s <= pos} p_s v_s / sum p_s,   p_s = exp2(scale log2(e) q.k_s - m)
// with a running reference m of each row, 7 below the row's largest exponent when it is
// set, moved where p would pass 2^15: so it seldom moves and the sums are rescaled only then.
// Scores, sums and outputs are binary32; p enters the tensor cores as binary16, which they
// need as the operand beside binary16 values: half a step, 2^-11 of p, and below 2^-14
// 2^-25, which is 2^-32 of the row's largest or less.
//
// Tiles.  A pair of 128-row tiles holds 2 tpt tokens of one kv head's g query heads,
// tpt = 128 / g (row r: token r / g, head r % g; rows behind tpt g are padding), and
// walks over the keys up to its last token's position, 128 a step: S = Q K^T into TMEM,
// softmax by a warpgroup (a thread a row), P back into TMEM over S, O += P V.  Two
// tiles in turn keep the tensor cores at one's products while the other's softmax runs.
//
// Work split (stream-K).  All pairs' keys in a row, in the order (sequence, kv head,
// pair), with kSetup units more for a pair's beginning, are cut into equal stretches, one a
// CTA; a key tile is the CTA's in whose stretch it begins.  So lengths do not matter to the
// balance and few rows over a long axis are split over it.  A pair that
// several CTAs share leaves binary32 partial sums in the workspace; a second kernel,
// launched with the first's end overlapped, merges them in CTA order (bit-reproducible).
// A share of more than 128 key tiles is taken in segments, added up there by the CTA itself.
// Every CTA finds its stretch from the lengths on the device, by sums in closed form.
//
// Warp roles (16 warps, one CTA an SM):
//   0-3, 4-7   softmax of tile 0 and tile 1; they rescale its O where they must
//   8-11       store O, while the next pair's scores are under way
//   12, 13     TMA of Q and K, and of V (side by side: pages of 16 tokens take 16 copies
//              a tile); the latter zeroes V's rows behind a sequence's last token
//   14, 15     MMA of tile 0 and tile 1 (14 owns the TMEM); one thread of each issues
// K and V tiles share a ring: [half of 64 dims][128 keys][128 bytes], 128-byte swizzle.
// K is the K-major B operand of S, V the MN-major one of O.
//
// What bounds it: two tiles' step of 128 keys is 2048 cycles of the tensor cores and as
// many of the MUFU (an exponential a score), and takes 4100, as a tile's chain does: softmax
// 1830, its products and next scores 1400, hand-overs.  With D = 128 two S and two O fill the
// TMEM, so there is no second S to take the chain apart; with D = 64 a quarter of it is left,
// which this kernel does not use.  Measured, 32/8 heads of 128: 4096 tokens after 12288 in
// 890 us (1080 TFLOP/s of the causal products; 1001 us when run on end, under the power cap),
// 60 tokens after 60001 in 88 us with the merge (2.8 TB/s); 14/2 heads of 64: eight prompts of
// 117 to 2000 tokens after 133 to 1000 in 104 us (390 TFLOP/s), 13 tokens after 150 in 12 us: plan 3,
// first copies 3.5, two steps, merge.
#include <cuda.h>
#include <cuda_fp16.h>
#include <cuda_runtime.h>
#include <cudaTypedefs.h>
#include <stdint.h>

#include <algorithm>
#include <cmath>
#include <mutex>

#include "kv_q8.cuh"

namespace anvilq {
namespace chunk {

using q8::overlap;
using u64 = unsigned long long;
constexpr int kRows = 128;                 // of a tile: MMA M, a TMEM lane each
constexpr int kKeys = 128;                 // of a step
constexpr int kThreads = 512;
constexpr int kWarps = kThreads / 32;
constexpr int kStoreWarp = 8, kKWarp = 12, kVWarp = 13, kMmaWarp = 14;
// What a pair's beginning costs, in keys: queries, first scores, outputs.  (12 sequences of which
// six take a step, the others chunks up to 500: without it 149 us, with 128 keys 129, 192 123.)
constexpr int kSetup = 192;
constexpr int kLeast = 1;                  // key tiles' worth of units of a stretch, at least
constexpr int kMaxCtas = 148;
// Key tiles of a segment, at most.  The tensor cores add to binary32 by cutting off, up to 2^-23 of the sum at
// each 16 keys and always downwards: over 2^20 keys of equal weights 6.7e-3.  So after a segment the
// products begin anew, and its outputs are added to those before by rounded operations, when the products go
// on: 1e-4 at any length.  (4096 tokens after 61440, 32/8 heads: of 128 4.20 ms, 4.08 without, of 64 3.48 as without;
// with outputs added before the products go on 4.43 and 3.64.)
constexpr int kPiece = 128;
constexpr int kSlots = 3;                  // of partial sums a CTA
constexpr int kMaxBatch = 65536;
constexpr float kNone = -1e30f;            // a reference below every exponent
// How far (log2) the reference is below a row's largest when it is set, and may lag behind it later: the
// largest p is from 2^7 to 2^15, so that binary16 has normal numbers down to 2^-21 of it or less.
constexpr float kBelow = 7.0f, kSlack = 15.0f;
// An exponent is a product less the reference, rounded once, so of a row's largest it is half a step of
// the reference off: up to here it stays below 2^15.5, which binary16 takes.  From here on different scores are 16
// or more apart, so that only the largest count, and a power of two as the scale gives their exponents exactly.
constexpr float kLarge = 0x1p28f;
constexpr u64 kWaitLimitNs = 1000000000ull;
constexpr uint32_t kTmemCols = 512, kTmemO = 256;   // S of tile t at 128 t, O at 256 + 128 t

template <int D>
struct Cfg {
  static constexpr int kHalves = D / 64;
  static constexpr int kTileBytes = kKeys * D * 2;                 // a K, V or Q tile
  static constexpr int kStages = D == 128 ? 5 : 10;
  static constexpr int kOffQ = kStages * kTileBytes;
  static constexpr int kOffBar = kOffQ + 2 * kTileBytes;
  static constexpr int kBars = 2 * kStages + 2 * 9 + 1;
  static constexpr int kOffShared = (kOffBar + kBars * 8 + 15) / 16 * 16;
  static_assert(kMaxBatch / 32 * 8 <= kOffQ, "the groups' counts lie in the ring before its first copy");
};

struct Params {
  const __half* q;              // [T] tokens of Hq D, `q_stride` elements apart
  long long q_stride;
  const int* starts;            // [B + 1]
  const int* seqlens;           // [B]
  const uint32_t* page_table;   // [B][max_pages]
  __half* out;                  // [T][Hq][D]
  // [CTAs][kSlots][256 (D + 2)]: sums of a share that is not all of a pair, or not one segment; the first place is
  // for a stretch's first share where an earlier CTA's goes before it, the last for a segment's yet to be added
  float* partials;
  float2* fresh;                // [CTAs][256]: references and sums of a segment that others of its share came before
  struct Open* open;            // [CTAs]
  int* dev_err;
  float scale_log2, scale_large;   // the latter a power of two, 16 to 32 times the former
  int T, B, Hq, Hkv, group, tpt, page_tokens, max_pages, num_pages, box;
  int sectors;                  // out lies on 32 bytes, and with it every 16 dims of a row
};

// What the merge needs to know of a CTA's first pair.
struct Open {
  u64 begin, end;               // the units of its first and last key tile; the CTA's own begin at `at`
  u64 at, chunk;
  int token, tokens, head, mid; // first token, tokens left in the sequence from it on; mid: begun by an earlier CTA
};

// ---- PTX ------------------------------------------------------------------------
__device__ __forceinline__ uint32_t smem_u32(const void* p) { return static_cast<uint32_t>(__cvta_generic_to_shared(p)); }
__device__ __forceinline__ u64 globaltimer() {
  u64 t;
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
// Waits for the phase of `parity`; gives up after kWaitLimitNs, or once another role has.
__device__ __forceinline__ bool mbar_wait(uint32_t bar, uint32_t parity, volatile int* abort_flag) {
  if (mbar_try_wait(bar, parity)) return true;
  const u64 t0 = globaltimer();
  for (;;) {
    if (mbar_try_wait(bar, parity)) return true;
    if (*abort_flag || globaltimer() - t0 > kWaitLimitNs) return false;
  }
}
__device__ __forceinline__ void mbar_drain(uint32_t bar, uint32_t parity) {
  const u64 t0 = globaltimer();
  while (!mbar_try_wait(bar, parity))
    if (globaltimer() - t0 > kWaitLimitNs) return;
}
__device__ __forceinline__ void mbar_init(uint32_t bar, uint32_t count) {
  asm volatile("mbarrier.init.shared::cta.b64 [%0], %1;" ::"r"(bar), "r"(count) : "memory");
}
__device__ __forceinline__ void mbar_arrive(uint32_t bar) {
  asm volatile("mbarrier.arrive.shared::cta.b64 _, [%0];" ::"r"(bar) : "memory");
}
__device__ __forceinline__ bool elect_one() {
  uint32_t pred;
  asm volatile("{\n .reg .pred e;\n .reg .b32 r;\n elect.sync r|e, 0xffffffff;\n selp.u32 %0, 1, 0, e;\n}"
               : "=r"(pred));
  return pred != 0;
}
__device__ __forceinline__ void tma_2d(uint32_t dst, const CUtensorMap* map, int x, int y, uint32_t bar) {
  asm volatile(
      "cp.async.bulk.tensor.2d.shared::cluster.global.tile.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3}], "
      "[%4];" ::"r"(dst),
      "l"(map), "r"(x), "r"(y), "r"(bar)
      : "memory");
}
__device__ __forceinline__ void tma_3d(uint32_t dst, const CUtensorMap* map, int x, int y, int z, uint32_t bar) {
  asm volatile(
      "cp.async.bulk.tensor.3d.shared::cluster.global.tile.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3, %4}], "
      "[%5];" ::"r"(dst),
      "l"(map), "r"(x), "r"(y), "r"(z), "r"(bar)
      : "memory");
}
__device__ __forceinline__ void tc_fence_before() { asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory"); }
__device__ __forceinline__ void tc_fence_after() { asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory"); }
__device__ __forceinline__ void tc_commit(uint32_t bar) {
  asm volatile("tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [%0];" ::"r"(bar) : "memory");
}
// D[tmem] (+)= A[smem] B[smem]^T and D[tmem] (+)= A[tmem] B[smem]^T, binary16 operands
__device__ __forceinline__ void mma_ss(uint32_t d, u64 a, u64 b, uint32_t idesc, uint32_t accumulate) {
  asm volatile(
      "{\n .reg .pred p;\n setp.ne.b32 p, %4, 0;\n"
      " tcgen05.mma.cta_group::1.kind::f16 [%0], %1, %2, %3, p;\n}" ::"r"(d),
      "l"(a), "l"(b), "r"(idesc), "r"(accumulate)
      : "memory");
}
__device__ __forceinline__ void mma_ts(uint32_t d, uint32_t a, u64 b, uint32_t idesc, uint32_t accumulate) {
  asm volatile(
      "{\n .reg .pred p;\n setp.ne.b32 p, %4, 0;\n"
      " tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], %2, %3, p;\n}" ::"r"(d),
      "r"(a), "l"(b), "r"(idesc), "r"(accumulate)
      : "memory");
}
#define ANVILQ_R32(r)                                                                                              \
  r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]), "=r"(r[8]),           \
      "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15]), "=r"(r[16]),       \
      "=r"(r[17]), "=r"(r[18]), "=r"(r[19]), "=r"(r[20]), "=r"(r[21]), "=r"(r[22]), "=r"(r[23]), "=r"(r[24]),      \
      "=r"(r[25]), "=r"(r[26]), "=r"(r[27]), "=r"(r[28]), "=r"(r[29]), "=r"(r[30]), "=r"(r[31]
// 32 consecutive columns of the thread's lane; wait_ld() before the registers are used
__device__ __forceinline__ void tmem_ld32(uint32_t taddr, uint32_t* r) {
  asm volatile(
      "tcgen05.ld.sync.aligned.32x32b.x32.b32 {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16,%17,%18,"
      "%19,%20,%21,%22,%23,%24,%25,%26,%27,%28,%29,%30,%31}, [%32];"
      : "=r"(ANVILQ_R32(r))
      : "r"(taddr));
}
__device__ __forceinline__ void tmem_st32(uint32_t taddr, const uint32_t* v) {
  asm volatile(
      "tcgen05.st.sync.aligned.32x32b.x32.b32 [%0], {%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16,"
      "%17,%18,%19,%20,%21,%22,%23,%24,%25,%26,%27,%28,%29,%30,%31,%32};" ::"r"(taddr),
      "r"(v[0]), "r"(v[1]), "r"(v[2]), "r"(v[3]), "r"(v[4]), "r"(v[5]), "r"(v[6]), "r"(v[7]), "r"(v[8]),
      "r"(v[9]), "r"(v[10]), "r"(v[11]), "r"(v[12]), "r"(v[13]), "r"(v[14]), "r"(v[15]), "r"(v[16]),
      "r"(v[17]), "r"(v[18]), "r"(v[19]), "r"(v[20]), "r"(v[21]), "r"(v[22]), "r"(v[23]), "r"(v[24]),
      "r"(v[25]), "r"(v[26]), "r"(v[27]), "r"(v[28]), "r"(v[29]), "r"(v[30]), "r"(v[31])
      : "memory");
}
__device__ __forceinline__ void tmem_ld16(uint32_t taddr, uint32_t* r) {
  asm volatile(
      "tcgen05.ld.sync.aligned.32x32b.x16.b32 {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15}, [%16];"
      : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]),
        "=r"(r[8]), "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15])
      : "r"(taddr));
}
__device__ __forceinline__ void tmem_st16(uint32_t taddr, const uint32_t* v) {
  asm volatile(
      "tcgen05.st.sync.aligned.32x32b.x16.b32 [%0], {%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16};" ::"r"(
          taddr),
      "r"(v[0]), "r"(v[1]), "r"(v[2]), "r"(v[3]), "r"(v[4]), "r"(v[5]), "r"(v[6]), "r"(v[7]), "r"(v[8]),
      "r"(v[9]), "r"(v[10]), "r"(v[11]), "r"(v[12]), "r"(v[13]), "r"(v[14]), "r"(v[15])
      : "memory");
}
__device__ __forceinline__ void wait_ld() { asm volatile("tcgen05.wait::ld.sync.aligned;" ::: "memory"); }
__device__ __forceinline__ void wait_st() { asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory"); }
__device__ __forceinline__ float fast_exp2(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}

__device__ __forceinline__ float max3(float a, float b, float c) {
  float d;
  asm("max.f32 %0, %1, %2, %3;" : "=f"(d) : "f"(a), "f"(b), "f"(c));
  return d;
}
// two binary32 values at a time
__device__ __forceinline__ u64 pair(float a, float b) {
  u64 v;
  asm("mov.b64 %0, {%1, %2};" : "=l"(v) : "f"(a), "f"(b));
  return v;
}
__device__ __forceinline__ float2 unpair(u64 v) {
  float2 f;
  asm("mov.b64 {%0, %1}, %2;" : "=f"(f.x), "=f"(f.y) : "l"(v));
  return f;
}
__device__ __forceinline__ u64 fma2(u64 a, u64 b, u64 c) {
  u64 d;
  asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(d) : "l"(a), "l"(b), "l"(c));
  return d;
}
__device__ __forceinline__ u64 add2(u64 a, u64 b) {
  u64 d;
  asm("add.rn.f32x2 %0, %1, %2;" : "=l"(d) : "l"(a), "l"(b));
  return d;
}

// Shared-memory matrix descriptor: start, leading and stride byte offsets in 16-byte
// units, version 1, 128-byte swizzle.  K-major: stride between 8-row groups (leading
// unused).  MN-major: leading between blocks of 64 dims, stride between 8-key groups.
__device__ __forceinline__ u64 smem_desc(uint32_t addr, uint32_t lbo, uint32_t sbo) {
  return (u64)((addr >> 4) & 0x3FFFu) | ((u64)((lbo >> 4) & 0x3FFFu) << 16) | ((u64)((sbo >> 4) & 0x3FFFu) << 32) |
         (1ull << 46) | (2ull << 61);
}
// Instruction descriptor, kind::f16: binary32 accumulator, binary16 operands, M 128;
// bit 16: B is MN-major
__host__ __device__ constexpr uint32_t instr_desc(int n, bool b_mn_major) {
  return (1u << 4) | ((uint32_t)b_mn_major << 16) | ((uint32_t)(n >> 3) << 17) | ((uint32_t)(kRows >> 4) << 24);
}

// ---- the plan -----------------------------------------------------------------------

// A sequence's new tokens: rows [start, start + n) at positions before and on.
struct Seq {
  int start, n, before;
};
__device__ __forceinline__ Seq sequence(const Params& p, int b) {
  const int s0 = p.starts[b], s1 = p.starts[b + 1], len = p.seqlens[b];
  const long long n = (long long)s1 - s0;
  if (n <= 0) return Seq{0, 0, 0};
  if (s0 < 0 || s1 > p.T || n > len || len > (long long)p.page_tokens * p.max_pages) {
    atomicOr(p.dev_err, ANVILQ_DEV_ERR_SEQLEN);
    return Seq{0, 0, 0};
  }
  return Seq{s0, (int)n, len - (int)n};
}
__device__ __forceinline__ int pairs_of(const Params& p, const Seq& s) { return (s.n + 2 * p.tpt - 1) / (2 * p.tpt); }
// key tiles of the first `tokens` (> 0) new tokens
__device__ __forceinline__ int tiles_to(const Seq& s, int tokens) {
  return (s.before + min(tokens, s.n) + kKeys - 1) / kKeys;
}
// A pair's units are kSetup for its beginning, then its keys.  Those of a head's first i
// pairs, i < pairs_of: their keys are an arithmetic series.
__device__ __forceinline__ u64 units_before(const Params& p, const Seq& s, int i) {
  return (u64)i * (kSetup + s.before) + (u64)i * (i + 1) / 2 * (2 * p.tpt);
}
__device__ __forceinline__ u64 units_of(const Params& p, const Seq& s) {   // of a head
  return s.n ? units_before(p, s, pairs_of(p, s) - 1) + kSetup + s.before + s.n : 0;
}
// A key tile belongs to the stretch that its first key is in: of a pair's tiles, those whose
// first key lies below the pair's unit x.
__device__ __forceinline__ int tiles_below(int x) { return max(0, x - kSetup + kKeys - 1) / kKeys; }

// Where a stretch is: every role walks the same way.
struct Walk {
  Seq s;
  int b, h, i, x;   // pair i of head h of sequence b, x units into it
  int part;         // kOn, kMid of the segment that comes next
  u64 left;
};
// What a segment is of a pair: kOn, not the first of its stretch's share of it; kMid, that share is not
// the pair's first; kShared, another CTA has a share too; kOne, it is all of the pair.
enum { kOn = 1, kMid = 2, kShared = 4, kOne = 8 };
// Key tiles [j0, j1) of a pair, at most kPiece.
struct Segment {
  Seq s;
  int b, h, i, j0, j1, part;
  // tile t's part of them ends here, at j0 or before where it has none
  __device__ __forceinline__ int end(const Params& p, int t) const {
    const int first = (2 * i + t) * p.tpt;
    return first < s.n ? min(j1, tiles_to(s, first + p.tpt)) : j0;
  }
};
// The next segment that has a key tile; the whole warp calls it.  Both lie in shared
// memory, as the softmax needs the registers.
__device__ __forceinline__ bool next_segment(const Params& p, Walk& walk, Segment& seg) {
  __syncwarp();
  Walk w = walk;
  Segment g;
  g.j0 = g.j1 = 0;
  while (w.left && g.j1 <= g.j0) {
    g.s = w.s;
    g.b = w.b; g.h = w.h; g.i = w.i;
    const int nk = tiles_to(w.s, (w.i + 1) * 2 * p.tpt);
    int end = (int)min((u64)(kSetup + w.s.before + min((w.i + 1) * 2 * p.tpt, w.s.n)), w.x + w.left);
    const int to = tiles_below(end);
    g.j0 = min(nk, tiles_below(w.x));
    g.j1 = min(g.j0 + kPiece, to);
    if (!w.part && g.j0 > 0) w.part = kMid;
    g.part = w.part | (w.part & kMid || to < nk ? kShared : 0) | (g.j0 == 0 && g.j1 == nk ? kOne : 0);
    const bool on = g.j1 < to;   // the next segment begins there
    if (on) end = kSetup + g.j1 * kKeys;
    w.left -= end - w.x;
    w.x = on ? end : 0;
    w.part = on ? w.part | kOn : 0;
    if (w.left == 0 || on || ++w.i < pairs_of(p, w.s)) continue;
    w.i = 0;
    if (++w.h < p.Hkv) continue;
    w.h = 0;
    const int lane = threadIdx.x % 32;
    int b0 = w.b + 1;
    for (; b0 < p.B; b0 += 32) {   // the next sequence with new tokens
      const Seq s = b0 + lane < p.B ? sequence(p, b0 + lane) : Seq{0, 0, 0};
      const uint32_t some = __ballot_sync(0xffffffffu, s.n > 0);
      if (!some) continue;
      const int l = __ffs(some) - 1;
      w.b = b0 + l;
      w.s.start = __shfl_sync(0xffffffffu, s.start, l);
      w.s.n = __shfl_sync(0xffffffffu, s.n, l);
      w.s.before = __shfl_sync(0xffffffffu, s.before, l);
      break;
    }
    if (b0 >= p.B) w.left = 0;
  }
  __syncwarp();
  if (threadIdx.x % 32 == 0) {
    walk = w;
    seg = g;
  }
  __syncwarp();
  return g.j1 > g.j0;
}

__device__ __forceinline__ u64 warp_sum(u64 v) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
  return v;
}

struct Shared {
  Walk walk[kWarps];
  Segment seg[kWarps];
  float sums[2][kRows];
  uint32_t tmem;
  int turn;                  // 1: one of the tiles has its products and its next scores issued
  volatile int abort;
};

// The CTA's stretch, from the lengths: all threads; `groups` holds a number for every 32
// sequences.
__device__ __forceinline__ void plan(const Params& p, u64* groups, Shared& sh) {
  const int warp = threadIdx.x / 32, lane = threadIdx.x % 32, n = (p.B + 31) / 32;
  if (n > 1) {
    for (int i = warp; i < n; i += kWarps) {
      const int b = 32 * i + lane;
      const u64 units = warp_sum(b < p.B ? units_of(p, sequence(p, b)) * p.Hkv : 0);
      if (lane == 0) groups[i] = units;
    }
    __syncthreads();
  }
  if (warp == 0) {
    Seq s{0, 0, 0};          // of a group's sequences, the lane's
    u64 units = 0, total = 0;
    if (n == 1) {
      if (lane < p.B) s = sequence(p, lane);
      units = units_of(p, s);
      total = units * p.Hkv;
    } else {
      for (int i = lane; i < n; i += 32) total += groups[i];
    }
    total = warp_sum(total);
    const u64 chunk = max((total + gridDim.x - 1) / gridDim.x, (u64)(kLeast * kKeys));
    const u64 at = min(total, blockIdx.x * chunk);
    Walk w{};
    w.left = min(chunk, total - at);
    if (w.left) {
      u64 rest = at;   // units between the ones passed over and `at`
      // of 32 runs, the first that holds `rest`, which becomes its offset there; 32: none
      auto holds = [&](u64 run) {
        u64 incl = run;
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
          const u64 up = __shfl_up_sync(0xffffffffu, incl, o);
          if (lane >= o) incl += up;
        }
        const uint32_t past = __ballot_sync(0xffffffffu, incl > rest);
        const int l = past ? __ffs(past) - 1 : 32;
        rest -= __shfl_sync(0xffffffffu, past ? incl - run : incl, min(l, 31));
        return l;
      };
      int g = 0, l = 32;
      if (n > 1) {
        for (; l == 32 && g < n; g += l == 32 ? 32 : l) l = holds(g + lane < n ? groups[g + lane] : 0);
        const int b = 32 * g + lane;
        s = b < p.B ? sequence(p, b) : Seq{0, 0, 0};
        units = units_of(p, s);   // of a head
      }
      l = min(holds(units * p.Hkv), 31);
      w.b = 32 * g + l;
      w.s.start = __shfl_sync(0xffffffffu, s.start, l);
      w.s.n = __shfl_sync(0xffffffffu, s.n, l);
      w.s.before = __shfl_sync(0xffffffffu, s.before, l);
      units = __shfl_sync(0xffffffffu, units, l);
      w.h = p.Hkv == 1 ? 0 : (int)(rest / units);
      rest -= w.h * units;
      int lo = 0, span = pairs_of(p, w.s);   // the pair is one of [lo, lo + span)
      u64 before = 0;                        // units before pair lo
      while (span > 1) {
        const int step = (span + 31) / 32, i = lo + lane * step;
        const u64 mine = lane * step < span ? units_before(p, w.s, i) : rest + 1;
        const int k = 31 - __clz(__ballot_sync(0xffffffffu, mine <= rest));
        before = __shfl_sync(0xffffffffu, mine, k);
        lo += k * step;
        span = min(step, span - k * step);
      }
      w.i = lo;
      w.x = (int)(rest - before);
    }
    if (lane < kWarps) sh.walk[lane] = w;
    if (lane == 0) {
      // for the merge: the pair that the stretch begins in
      Open o{};
      if (w.left) {
        const int nk = tiles_to(w.s, (w.i + 1) * 2 * p.tpt), j0 = tiles_below(w.x);
        o.begin = at - w.x + kSetup;
        o.end = o.begin + (u64)(nk - 1) * kKeys;
        o.at = at;
        o.chunk = chunk;
        o.token = w.s.start + w.i * 2 * p.tpt;
        o.tokens = w.s.n - w.i * 2 * p.tpt;
        o.head = w.h;
        o.mid = j0 > 0 && j0 < nk;
      }
      p.open[blockIdx.x] = o;
    }
  }
  // the counts' place is the ring's, which asynchronous copies write next
  asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
  __syncthreads();
}

// ---- the kernel ----------------------------------------------------------------------

template <int D>
__global__ void __launch_bounds__(kThreads, 1)
    chunk_kernel(const __grid_constant__ CUtensorMap mq, const __grid_constant__ CUtensorMap mk,
                 const __grid_constant__ CUtensorMap mv, const __grid_constant__ Params p) {
  using C = Cfg<D>;
  extern __shared__ __align__(1024) unsigned char smem[];
  Shared& sh = *reinterpret_cast<Shared*>(smem + C::kOffShared);
  const uint32_t base = smem_u32(smem);
  const int warp = threadIdx.x / 32, lane = threadIdx.x % 32;
  const uint32_t bars = base + C::kOffBar;
  auto kv_full = [&](int s) { return bars + 8u * s; };
  auto kv_empty = [&](int s) { return bars + 8u * (C::kStages + s); };
  auto bar_of = [&](int kind, int t) { return bars + 8u * (2 * C::kStages + 2 * kind + t); };
  auto q_full = [&](int t) { return bar_of(0, t); };
  auto q_empty = [&](int t) { return bar_of(1, t); };
  auto s_full = [&](int t) { return bar_of(2, t); };
  auto p_full = [&](int t, int half) { return bar_of(3 + half, t); };   // 64 keys each
  auto pv_done = [&](int t) { return bar_of(5, t); };
  auto sums_full = [&](int t) { return bar_of(6, t); };
  auto o_empty = [&](int t) { return bar_of(7, t); };
  auto drained = [&](int t) { return bar_of(8, t); };
  const uint32_t landed = bar_of(9, 0);   // a V tile whose last rows are still to be zeroed
  if (threadIdx.x == 0) {
    for (int s = 0; s < C::kStages; ++s) {
      mbar_init(kv_full(s), 1);
      mbar_init(kv_empty(s), 2);
    }
    for (int t = 0; t < 2; ++t) {
      mbar_init(q_full(t), 1);
      mbar_init(q_empty(t), 1);
      mbar_init(s_full(t), 1);
      mbar_init(p_full(t, 0), 4);
      mbar_init(p_full(t, 1), 4);
      mbar_init(pv_done(t), 1);
      mbar_init(sums_full(t), 4);
      mbar_init(o_empty(t), 4);
      mbar_init(drained(t), 1);
    }
    mbar_init(landed, 1);
    sh.turn = 0;
    sh.abort = 0;
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    asm volatile("prefetch.tensormap [%0];" ::"l"(&mq) : "memory");
    asm volatile("prefetch.tensormap [%0];" ::"l"(&mk) : "memory");
    asm volatile("prefetch.tensormap [%0];" ::"l"(&mv) : "memory");
  }
  if (warp == kMmaWarp) {
    asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(&sh.tmem)),
                 "r"(kTmemCols)
                 : "memory");
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
    tc_fence_before();
  }
  asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
  asm volatile("griddepcontrol.wait;" ::: "memory");
  plan(p, reinterpret_cast<u64*>(smem), sh);   // ends with a barrier
  tc_fence_after();
  const uint32_t tmem = sh.tmem;
  Walk& w = sh.walk[warp];
  Segment& g = sh.seg[warp];
  auto fail = [&]() {
    sh.abort = 1;
    atomicOr(p.dev_err, ANVILQ_DEV_ERR_TIMEOUT);
  };
  auto wait = [&](uint32_t bar, uint32_t parity) {   // the whole warp; false: leave
    const bool ok = __all_sync(0xffffffffu, mbar_wait(bar, parity, &sh.abort));
    if (!ok && lane == 0) fail();
    return ok;
  };
  auto expect = [&](uint32_t bar, uint32_t bytes) {
    asm volatile("mbarrier.arrive.expect_tx.shared::cta.b64 _, [%0], %1;" ::"r"(bar), "r"(bytes) : "memory");
  };
  // `uses` of a tile: the segments that it has a part in

  if (warp >= kKWarp) {
    asm volatile("setmaxnreg.dec.sync.aligned.u32 72;");
    if (warp == kKWarp || warp == kVWarp) {
      // ------------------------------------------------------------------ Q, K and V
      const bool is_v = warp == kVWarp;
      const CUtensorMap* map = is_v ? &mv : &mk;
      const int boxes = kKeys / p.box, box_bytes = p.box * 128;
      const int my_box = lane % boxes, my_half = lane / boxes;   // at most 8 x 2 copies
      int stage = is_v ? 1 : 0;                                  // K and V tiles alternate in the ring
      uint32_t phase = 0, q_uses[2] = {0, 0}, tails = 0, issued = 0;   // issued: a bit a stage, its phase in the upper half
      bool ok = true;
      while (ok && next_segment(p, w, g)) {
        if (!is_v) {
          // Q: a box is tpt tokens of g heads.  Tokens behind the sequence's are other rows,
          // which are not stored, tokens behind the last zeros.
#pragma unroll
          for (int t = 0; t < 2; ++t) {
            if (!ok || g.end(p, t) <= g.j0) continue;
            ok = wait(q_empty(t), (q_uses[t]++ & 1) ^ 1);
            if (ok && lane == 0) {
              expect(q_full(t), C::kHalves * p.group * p.tpt * 128);
#pragma unroll
              for (int h = 0; h < C::kHalves; ++h)
                tma_3d(base + C::kOffQ + t * C::kTileBytes + h * (kRows * 128), &mq, h * 64, g.h * p.group,
                       g.s.start + (2 * g.i + t) * p.tpt, q_full(t));
            }
            __syncwarp();
          }
        }
        const int len = g.s.before + g.s.n;
        for (int j = g.j0; ok && j < g.j1; ++j) {
          // the lane's box: its page is looked up while the stage is waited for
          const int key = j * kKeys + my_box * p.box;
          const bool live = my_half < C::kHalves && key < len;
          int page = live ? q8::page_of(p.page_table, p.max_pages, p.num_pages, g.b, key / p.page_tokens) : 0;
          if (page < 0) {   // the output is not to be used
            atomicOr(p.dev_err, ANVILQ_DEV_ERR_PAGE);
            page = 0;
          }
          ok = wait(kv_empty(stage), phase ^ 1);
          if (!ok) break;
          // V's rows behind the sequence's last token may hold anything: times p = 0 they must be 0
          const int rows = len - j * kKeys;
          const bool tail = is_v && rows < kKeys;
          const uint32_t at = base + stage * C::kTileBytes, full = tail ? landed : kv_full(stage);
          const int copies = __popc(__ballot_sync(0xffffffffu, live));
          if (lane == 0) expect(full, copies * box_bytes);
          __syncwarp();
          if (live)
            tma_2d(at + my_half * (kKeys * 128) + my_box * box_bytes, map, g.h * D + my_half * 64,
                   page * p.page_tokens + key % p.page_tokens, full);
          __syncwarp();
          if (tail) {
            ok = wait(landed, tails++ & 1);
            if (!ok) break;
            for (int i = rows * 8 + lane; i < kKeys * 8; i += 32)
#pragma unroll
              for (int h = 0; h < C::kHalves; ++h)
                asm volatile("st.shared.v4.u32 [%0], {%1, %1, %1, %1};" ::"r"(at + h * (kKeys * 128) + i * 16), "r"(0)
                             : "memory");
            asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
            __syncwarp();
            if (lane == 0) mbar_arrive(kv_full(stage));
          }
          issued = (issued & ~(0x10001u << stage)) | ((1u | phase << 16) << stage);
          stage += 2;
          if (stage >= C::kStages) {
            stage -= C::kStages;
            phase ^= 1;
          }
        }
      }
      if (sh.abort && lane == 0) {   // let the copies in flight land before the CTA exits
        for (int s = 0; s < C::kStages; ++s)
          if (issued >> s & 1) mbar_drain(kv_full(s), issued >> (16 + s) & 1);
        if (is_v && tails) mbar_drain(landed, (tails - 1) & 1);
        for (int t = 0; t < 2; ++t)
          if (q_uses[t]) mbar_drain(q_full(t), (q_uses[t] - 1) & 1);
      }
    } else {
      // ------------------------------------------------------------------ MMA
      // A warp a tile issues its products, one thread of it (`leader`) the instructions: S = Q K^T
      // when a K tile is there, O += P V when its P and the V tile are.  The whole warp walks and
      // waits, so that descriptors are uniform values; with one thread alone each came from
      // its registers (4096 tokens after 12288, 32/8 heads: 950 us, so 907).  A tile's last
      // products and its next scores go together, one tile at a time (`turn`): so the tiles'
      // softmax run in turns, each beside the other's products.  Left alone, both ran at once
      // and both waited at once (955 us).
      const int t = warp - kMmaWarp;
      constexpr uint32_t idesc_s = instr_desc(kKeys, false), idesc_o = instr_desc(D, true);
      // low words of the descriptors (start, leading offset); the high one is all tiles'
      constexpr uint32_t kHigh = (uint32_t)(1024 >> 4) | (1u << 14) | (2u << 29);
      constexpr uint32_t kHalf = kKeys * 128 / 16, kTile = C::kTileBytes / 16;
      auto low = [](uint32_t at, uint32_t lbo) { return at >> 4 | (lbo >> 4) << 16; };
      const uint32_t q_low = low(base + C::kOffQ + t * C::kTileBytes, 16), k_low = low(base, 16),
                     v_low = low(base, kKeys * 128);
      auto desc = [](uint32_t lo) {
        u64 d;
        asm("mov.b64 %0, {%1, %2};" : "=l"(d) : "r"(lo), "r"(kHigh));
        return d;
      };
      const uint32_t s_at = tmem + t * kKeys, o_at = tmem + kTmemO + t * 128;
      int stage = 0;                           // the ring's next tile: K, V, K, V ...
      uint32_t phase = 0, steps = 0, uses = 0;
      bool ok = true;
      const bool leader = elect_one();
      auto next_stage = [&]() {
        if (++stage == C::kStages) {
          stage = 0;
          phase ^= 1;
        }
      };
      auto take_turn = [&]() {
        bool mine = !leader || atomicCAS(&sh.turn, 0, 1) == 0;
        if (!mine) {
          const u64 t0 = globaltimer();
          do {
            mine = atomicCAS(&sh.turn, 0, 1) == 0;
          } while (!mine && !sh.abort && globaltimer() - t0 <= kWaitLimitNs);
          if (!mine) fail();
        }
        return __all_sync(0xffffffffu, mine) != 0;
      };
      auto scores = [&](int ks) {              // S_t = Q_t K^T
        tc_fence_after();
        const uint32_t k = k_low + ks * kTile;
        if (leader) {
#pragma unroll
          for (int i = 0; i < D / 16; ++i)
            mma_ss(s_at, desc(q_low + (i / 4 * kHalf + i % 4 * 2)), desc(k + (i / 4 * kHalf + i % 4 * 2)), idesc_s, i > 0);
          tc_commit(s_full(t));
        }
      };
      // the tile's steps [j0, end) of a segment, none of them: passed over
      auto run = [&](int j0, int end, int j1) {
        if (end > j0) {
          if (!wait(kv_full(stage), phase) || !wait(q_full(t), uses & 1)) return false;
          if (steps && !wait(pv_done(t), (steps - 1) & 1)) return false;
          scores(stage);
          if (leader) {
            if (j0 + 1 == end) tc_commit(q_empty(t));
            tc_commit(kv_empty(stage));
          }
          next_stage();
          for (int j = j0; j < end; ++j, ++steps) {
            const int vs = stage;
            const bool more = j + 1 < end;
            if (!wait(kv_full(vs), phase)) return false;
            next_stage();
            const uint32_t v = v_low + vs * kTile;
            if (j == j0 && !wait(o_empty(t), (uses & 1) ^ 1)) return false;
            if (!wait(p_full(t, 0), steps & 1)) return false;
            tc_fence_after();
            if (leader)
#pragma unroll
              for (int i = 0; i < 4; ++i) mma_ts(o_at, s_at + i * 8, desc(v + i * 128), idesc_o, (j > j0 || i > 0) ? 1u : 0u);
            if (more && !wait(kv_full(stage), phase)) return false;
            if (!wait(p_full(t, 1), steps & 1) || !take_turn()) return false;
            tc_fence_after();
            if (leader) {
#pragma unroll
              for (int i = 4; i < 8; ++i) mma_ts(o_at, s_at + i * 8, desc(v + i * 128), idesc_o, 1u);
              tc_commit(pv_done(t));
            }
            if (more) {   // S goes where the products read P
              if (!wait(pv_done(t), steps & 1)) return false;
              scores(stage);
            }
            if (leader) {
              atomicExch(&sh.turn, 0);
              tc_commit(kv_empty(vs));
              if (more) tc_commit(kv_empty(stage));
              if (j + 2 == end) tc_commit(q_empty(t));
            }
            if (more) next_stage();
          }
          ++uses;
        }
        for (int i = 2 * (j1 - max(end, j0)); i > 0; --i) {
          if (!wait(kv_full(stage), phase)) return false;
          if (leader) mbar_arrive(kv_empty(stage));
          next_stage();
        }
        return true;
      };
      while (ok && next_segment(p, w, g))
        ok = run(__shfl_sync(0xffffffffu, g.j0, 0), __shfl_sync(0xffffffffu, g.end(p, t), 0),
                 __shfl_sync(0xffffffffu, g.j1, 0));
      if (sh.abort) {   // MMAs still running write TMEM
        if (leader) {
          tc_commit(drained(t));
          mbar_drain(drained(t), 0);
        }
        __syncwarp();
      }
    }
  } else if (warp >= kStoreWarp) {
    asm volatile("setmaxnreg.dec.sync.aligned.u32 72;");
    {
      // ------------------------------------------------------------------ stores
      const int row = warp % 4 * 32 + lane, of_token = row / p.group;
      auto leave = [&](int t) {   // tile t's outputs are out of TMEM
        tc_fence_before();
        __syncwarp();
        if (lane == 0) mbar_arrive(o_empty(t));
      };
      // A place's outputs [dims / 4][row] of tile t, and its states [row].
      auto start_of = [&](int i) { return p.partials + ((size_t)blockIdx.x * kSlots + i) * (2 * kRows * (D + 2)); };
      auto place = [&](int i, int t) { return reinterpret_cast<float4*>(start_of(i)) + t * kRows + row; };
      auto state_at = [&](int i, int t) {
        return reinterpret_cast<float2*>(start_of(i) + 2 * kRows * D) + t * kRows + row;
      };
      auto token_of = [&](int t) { return (2 * g.i + t) * p.tpt + of_token; };   // of the sequence's new ones
      auto is_token = [&](int t) { return of_token < p.tpt && token_of(t) < g.s.n; };
      auto out_at = [&](int t) {
        return p.out + ((long long)(g.s.start + token_of(t)) * p.Hq + g.h * p.group + row - of_token * p.group) * D;
      };
      // no other segment and no other CTA has more of the tile
      auto is_last = [&](int t) { return !(g.part & kShared) && tiles_to(g.s, (2 * g.i + t + 1) * p.tpt) <= g.j1; };
      unsigned phases = 0;   // of the next sums (bit t) and of the products (bit 2 + t) of tile t
      bool ok = true;
      while (ok && next_segment(p, w, g)) {
        const int own = g.part & kMid ? 0 : 1;   // the place of the share's sums
        const bool on = g.part & kOn;
#pragma unroll
        for (int t = 0; t < 2; ++t) {
          const int end = g.end(p, t);
          if (end <= g.j0) {
            // the merge reads both tiles'
            if ((g.part & (kShared | kOn)) == kShared) __stcg(state_at(own, t), make_float2(kNone, 0.0f));
            continue;
          }
          const bool mine = is_token(t), last = is_last(t);
          // the outputs of a segment that others came before go out of the way, to be added below
          float4* to = place(on ? kSlots - 1 : own, t);
          __half* out = out_at(t);
          phases ^= (unsigned)(end - g.j0 & 1) << (2 + t);
          ok = wait(sums_full(t), phases >> t & 1) && wait(pv_done(t), ~phases >> (2 + t) & 1);
          phases ^= 1u << t;
          if (!ok) break;
          tc_fence_after();
          if (on && mine) {
            const float2 then = __ldcg(state_at(own, t));
            const float2 now = __ldcg(p.fresh + (blockIdx.x * 2 + t) * kRows + row);
            const float top = fmaxf(then.x, now.x);
            float f_then = fast_exp2(then.x - top), f = fast_exp2(now.x - top);
            const float sum = then.y * f_then + now.y * f;
            if (last) {
              const float inv = sum == 0.0f ? 0.0f : 1.0f / sum;
              f_then *= inv;
              f *= inv;
            } else {
              __stcg(state_at(own, t), make_float2(top, sum));
            }
            __stcg(state_at(kSlots - 1, t), make_float2(f_then, f));   // factors of the outputs before, and of these
          }
          const float sum = sh.sums[t][row], inv = sum == 0.0f ? 0.0f : 1.0f / sum;   // (only scores of -inf: zeros)
#pragma unroll
          for (int c = 0; c < D; c += 32) {
            uint32_t o[32];
            tmem_ld32(tmem + kTmemO + t * 128 + ((uint32_t)(warp % 4 * 32) << 16) + c, o);
            wait_ld();
            if (c + 32 == D) leave(t);
            if (!mine) continue;
            if (last && !on) {
#pragma unroll
              for (int e = 0; e < 32; e += 16) {   // a sector at a time
                uint32_t v[8];
#pragma unroll
                for (int k = 0; k < 8; ++k) {
                  const __half2 h = __floats2half2_rn(__uint_as_float(o[e + 2 * k]) * inv,
                                                      __uint_as_float(o[e + 2 * k + 1]) * inv);
                  v[k] = *reinterpret_cast<const uint32_t*>(&h);
                }
                if (p.sectors) {
                  asm volatile("st.global.v8.b32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8};" ::"l"(out + c + e), "r"(v[0]),
                               "r"(v[1]), "r"(v[2]), "r"(v[3]), "r"(v[4]), "r"(v[5]), "r"(v[6]), "r"(v[7])
                               : "memory");
                } else {
                  *reinterpret_cast<uint4*>(out + c + e) = make_uint4(v[0], v[1], v[2], v[3]);
                  *reinterpret_cast<uint4*>(out + c + e + 8) = make_uint4(v[4], v[5], v[6], v[7]);
                }
              }
            } else {
#pragma unroll
              for (int e = 0; e < 32; e += 4)
                __stcg(to + (c + e) / 4 * (2 * kRows),
                       make_float4(__uint_as_float(o[e]), __uint_as_float(o[e + 1]), __uint_as_float(o[e + 2]),
                                   __uint_as_float(o[e + 3])));
            }
          }
        }
        if (!on || !ok) continue;
#pragma unroll 1
        for (int t = 0; t < 2; ++t) {   // added to the outputs before
          if (g.end(p, t) <= g.j0 || !is_token(t)) continue;
          const bool last = is_last(t);
          const float2 factor = __ldcg(state_at(kSlots - 1, t));
          float4* at = place(own, t);
          const float4* more = place(kSlots - 1, t);
          __half* out = out_at(t);
#pragma unroll 1
          for (int c = 0; c < D; c += 16) {
            float4 a[4], b[4];
#pragma unroll
            for (int k = 0; k < 4; ++k) {
              a[k] = __ldcg(at + (c / 4 + k) * (2 * kRows));
              b[k] = __ldcg(more + (c / 4 + k) * (2 * kRows));
            }
#pragma unroll
            for (int k = 0; k < 4; ++k) {
              a[k].x = a[k].x * factor.x + b[k].x * factor.y;
              a[k].y = a[k].y * factor.x + b[k].y * factor.y;
              a[k].z = a[k].z * factor.x + b[k].z * factor.y;
              a[k].w = a[k].w * factor.x + b[k].w * factor.y;
              if (!last) __stcg(at + (c / 4 + k) * (2 * kRows), a[k]);
            }
            if (!last) continue;
#pragma unroll
            for (int k = 0; k < 4; k += 2) {
              uint4 v;
              __half2* h = reinterpret_cast<__half2*>(&v);
#pragma unroll
              for (int e = 0; e < 2; ++e) {
                h[2 * e] = __floats2half2_rn(a[k + e].x, a[k + e].y);
                h[2 * e + 1] = __floats2half2_rn(a[k + e].z, a[k + e].w);
              }
              *reinterpret_cast<uint4*>(out + c + 4 * k) = v;
            }
          }
        }
      }
    }
  } else {
    // -------------------------------------------------------------------- softmax
    asm volatile("setmaxnreg.inc.sync.aligned.u32 184;");
    const int t = warp / 4, row = threadIdx.x % kRows;
    const uint32_t lanes = (uint32_t)(warp % 4 * 32) << 16;
    const uint32_t s_at = tmem + t * kKeys + lanes, o_at = tmem + kTmemO + t * 128 + lanes;
    unsigned phases = 0;   // of the next scores and (bit 1) of the outputs' place
    bool ok = true;
    while (ok && next_segment(p, w, g)) {
      const int end = g.end(p, t), j0 = g.j0;
      // the last position that the row sees (of a row that is none, some)
      const int pos = g.s.before + min((2 * g.i + t) * p.tpt + row / p.group, g.s.n - 1);
      float m = kNone, sum = 0.0f, scale = p.scale_log2;
      for (int j = j0; j < end; ++j, phases ^= 1) {
        ok = wait(s_full(t), phases & 1);
        if (!ok) break;
        tc_fence_after();
        float s[kKeys];
#pragma unroll
        for (int c = 0; c < kKeys; c += 32) tmem_ld32(s_at + c, reinterpret_cast<uint32_t*>(s) + c);
        wait_ld();
        const int visible = pos + 1 - j * kKeys;   // keys of the tile that the row sees
        if (__any_sync(0xffffffffu, visible < kKeys)) {
#pragma unroll
          for (int c = 0; c < kKeys; ++c) s[c] = c < visible ? s[c] : -INFINITY;
        }
        float tops[4] = {s[0], s[1], s[2], s[3]};
#pragma unroll
        for (int c = 4; c + 1 < kKeys; c += 2) tops[c / 2 % 4] = max3(tops[c / 2 % 4], s[c], s[c + 1]);
        const float top = fmaxf(max3(tops[0], tops[1], tops[2]), tops[3]), bound = top * scale;
        const bool moves = bound > __fadd_rd(m, kSlack);
        if (__any_sync(0xffffffffu, moves)) {
          const float other = fabsf(top * p.scale_log2) < kLarge ? p.scale_log2 : p.scale_large;
          scale = moves ? other : scale;
          const float now = moves ? top * scale - kBelow : m;
          const float f = fast_exp2(m - now);
          m = now;
          sum *= f;
          if (j > j0) {
            ok = wait(pv_done(t), ~phases & 1);
            if (!ok) break;
            tc_fence_after();
#pragma unroll
            for (int c = 0; c < D; c += 16) {
              uint32_t o[16];
              tmem_ld16(o_at + c, o);
              wait_ld();
#pragma unroll
              for (int e = 0; e < 16; ++e) o[e] = __float_as_uint(__uint_as_float(o[e]) * f);
              tmem_st16(o_at + c, o);
            }
          }
        }
        const u64 scale2 = pair(scale, scale), ref2 = pair(-m, -m);
        u64 part[2] = {0, 0};
#pragma unroll
        for (int c = 0; c < kKeys; c += 64) {
          uint32_t half[32];
#pragma unroll
          for (int e = 0; e < 32; ++e) {
            const float2 x = unpair(fma2(pair(s[c + 2 * e], s[c + 2 * e + 1]), scale2, ref2));
            const float a = fast_exp2(x.x), b = fast_exp2(x.y);
            part[e % 2] = add2(part[e % 2], pair(a, b));
            const __half2 h = __floats2half2_rn(a, b);
            half[e] = *reinterpret_cast<const uint32_t*>(&h);
          }
          tmem_st32(s_at + c / 2, half);
          wait_st();
          tc_fence_before();
          __syncwarp();
          if (lane == 0) mbar_arrive(p_full(t, c / 64));
        }
        const float2 both = unpair(add2(part[0], part[1]));
        sum += both.x + both.y;
      }
      if (!ok) break;
      if (end > j0) {
        ok = wait(o_empty(t), ~phases >> 1 & 1);   // the sums of the segment before are read
        phases ^= 2;
        sh.sums[t][row] = sum;
        if (!(g.part & kOne)) {   // for the merge, or the stores
          float* slot = p.partials + ((size_t)blockIdx.x * kSlots + (g.part & kMid ? 0 : 1)) * (2 * kRows * (D + 2));
          float2* to = reinterpret_cast<float2*>(slot + 2 * kRows * D);
          if (g.part & kOn) to = p.fresh + blockIdx.x * (2 * kRows);
          __stcg(to + t * kRows + row, make_float2(scale == p.scale_log2 ? m : m / scale * p.scale_log2, sum));
        }
        __syncwarp();
        if (lane == 0) mbar_arrive(sums_full(t));
      }
    }
  }
  __syncthreads();
  if (warp == kMmaWarp) {
    tc_fence_after();
    asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(kTmemCols) : "memory");
  }
}

// ---- the merge of pairs that several CTAs share ---------------------------------------

constexpr int kMergeThreads = 256;

// Resident blocks over (shared pair, 32 of its rows).  A thread has a row and 4 dims in
// D / 32 places of it, so that a warp reads whole lines; several CTAs' states and sums are
// on their way at once and merged as a softmax goes on.  The outputs are turned in shared
// memory into rows.
template <int D>
__global__ void __launch_bounds__(kMergeThreads) merge_kernel(const __grid_constant__ Params p, int ctas) {
  constexpr int kVec = D / 4, kMine = kVec / (kMergeThreads / 32), kSlices = 2 * kRows / 32, kAtOnce = 4;
  constexpr size_t kSlot = 2 * kRows * (D + 2);
  __shared__ int seconds[kMaxCtas];   // the CTAs that go on with a pair that the CTA before them began
  __shared__ int count[kMergeThreads / 32];
  __shared__ uint2 turned[32][kVec + 1];
  asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
  asm volatile("griddepcontrol.wait;" ::: "memory");
  static_assert(kMaxCtas <= kMergeThreads, "a CTA a thread");
  const int warp = threadIdx.x / 32, lane = threadIdx.x % 32;
  bool shared = false;
  if (threadIdx.x < ctas) {
    const Open& o = p.open[threadIdx.x];
    shared = o.mid && o.begin + o.chunk >= o.at;
  }
  const uint32_t some = __ballot_sync(0xffffffffu, shared);
  if (lane == 0) count[warp] = __popc(some);
  __syncthreads();
  int at = __popc(some & ((1u << lane) - 1)), pairs = 0;
#pragma unroll
  for (int w = 0; w < kMergeThreads / 32; ++w) {
    if (w < warp) at += count[w];
    pairs += count[w];
  }
  if (shared) seconds[at] = threadIdx.x;
  __syncthreads();
  for (int work = blockIdx.x; work < pairs * kSlices; work += gridDim.x) {
    const int second = seconds[work / kSlices], r0 = work % kSlices * 32, r = r0 + lane;
    const Open o = p.open[second];
    // token of a row in the pair, -1: none
    auto token_of = [&](int row) {
      const int of = row % kRows / p.group, token = row / kRows * p.tpt + of;
      return of < p.tpt && token < o.tokens ? token : -1;
    };
    const bool mine = token_of(r) >= 0;
    const int n = (int)(o.end / o.chunk) - second + 2;   // CTAs
    // the pair is the last of the CTA that began it, the first of the others
    const float* begin = p.partials + ((size_t)(second - 1) * kSlots + 1) * kSlot;
    const float* others = p.partials + (size_t)second * kSlots * kSlot;
    float m = kNone, sum = 0.0f;
    float4 acc[kMine];
#pragma unroll
    for (int i = 0; i < kMine; ++i) acc[i] = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
    for (int c0 = 0; c0 < n && mine; c0 += kAtOnce) {
      float2 state[kAtOnce];
      float4 v[kAtOnce][kMine];
#pragma unroll
      for (int k = 0; k < kAtOnce; ++k) {
        state[k] = make_float2(kNone, 0.0f);
        if (c0 + k < n) {
          const float* slot = c0 + k ? others + (size_t)(c0 + k - 1) * kSlots * kSlot : begin;
          state[k] = __ldcg(reinterpret_cast<const float2*>(slot + 2 * kRows * D) + r);
#pragma unroll
          for (int i = 0; i < kMine; ++i)
            v[k][i] = __ldcg(reinterpret_cast<const float4*>(slot) + (warp * kMine + i) * (2 * kRows) + r);
        }
      }
      float now = m;
#pragma unroll
      for (int k = 0; k < kAtOnce; ++k) now = fmaxf(now, state[k].x);
      const float f = fast_exp2(m - now);
      m = now;
      sum *= f;
#pragma unroll
      for (int i = 0; i < kMine; ++i) {
        acc[i].x *= f; acc[i].y *= f; acc[i].z *= f; acc[i].w *= f;
      }
#pragma unroll
      for (int k = 0; k < kAtOnce; ++k) {
        if (state[k].y == 0.0f) continue;   // the row saw nothing there, and there may be no sums either
        const float e = fast_exp2(state[k].x - now);
        sum += state[k].y * e;
#pragma unroll
        for (int i = 0; i < kMine; ++i) {
          acc[i].x += v[k][i].x * e;
          acc[i].y += v[k][i].y * e;
          acc[i].z += v[k][i].z * e;
          acc[i].w += v[k][i].w * e;
        }
      }
    }
    const float inv = sum == 0.0f ? 0.0f : 1.0f / sum;
#pragma unroll
    for (int i = 0; i < kMine; ++i) {
      uint2 w;
      __half2* h = reinterpret_cast<__half2*>(&w);
      h[0] = __floats2half2_rn(acc[i].x * inv, acc[i].y * inv);
      h[1] = __floats2half2_rn(acc[i].z * inv, acc[i].w * inv);
      turned[lane][warp * kMine + i] = w;
    }
    __syncthreads();
    for (int i = threadIdx.x; i < 32 * kVec; i += kMergeThreads) {
      const int row = r0 + i / kVec, token = token_of(row);
      if (token >= 0)
        reinterpret_cast<uint2*>(p.out + ((long long)(o.token + token) * p.Hq + o.head * p.group +
                                          row % kRows % p.group) * D)[i % kVec] = turned[i / kVec][i % kVec];
    }
    __syncthreads();
  }
}

// ---- host -----------------------------------------------------------------------------
static bool a16(const void* p) { return (reinterpret_cast<uintptr_t>(p) & 15u) == 0; }
// 128 products of two binary16 values, times it, stay far above kNone
constexpr float kMaxScale = 0x1p32f;

static bool shape_ok(int T, int B, int Hq, int Hkv, int D) {
  return T >= 0 && T <= (1 << 30) && B >= 1 && B < kMaxBatch && Hkv >= 1 && Hq >= Hkv && Hq % Hkv == 0 && Hq <= 1024 &&
         Hq / Hkv <= kRows && (D == 64 || D == 128);
}

template <int D>
constexpr int smem_bytes() {
  static_assert(Cfg<D>::kOffShared + sizeof(Shared) <= 227 * 1024, "shared memory per CTA");
  return Cfg<D>::kOffShared + sizeof(Shared);
}

constexpr int kMaxDevices = 64;
static int g_sms[kMaxDevices];
static std::once_flag g_once[kMaxDevices];
static int sm_count() {
  int dev = 0;
  if (cudaGetDevice(&dev) != cudaSuccess || dev < 0 || dev >= kMaxDevices) return 0;
  std::call_once(g_once[dev], [dev] {
    cudaDeviceGetAttribute(&g_sms[dev], cudaDevAttrMultiProcessorCount, dev);
    cudaFuncSetAttribute(chunk_kernel<64>, cudaFuncAttributeMaxDynamicSharedMemorySize, smem_bytes<64>());
    cudaFuncSetAttribute(chunk_kernel<128>, cudaFuncAttributeMaxDynamicSharedMemorySize, smem_bytes<128>());
    cudaGetLastError();
  });
  return g_sms[dev];
}

static std::once_flag g_encode_once;
static PFN_cuTensorMapEncodeTiled_v12000 g_encode = nullptr;

static bool encode(CUtensorMap* map, const void* base, int rank, const cuuint64_t* dims, const cuuint64_t* strides,
                   const cuuint32_t* box) {
  std::call_once(g_encode_once, [] {
    void* fn = nullptr;
    cudaDriverEntryPointQueryResult q;
    if (cudaGetDriverEntryPoint("cuTensorMapEncodeTiled", &fn, cudaEnableDefault, &q) == cudaSuccess &&
        q == cudaDriverEntryPointSuccess)
      g_encode = reinterpret_cast<PFN_cuTensorMapEncodeTiled_v12000>(fn);
    cudaGetLastError();
  });
  const cuuint32_t estr[3] = {1, 1, 1};
  return g_encode && g_encode(map, CU_TENSOR_MAP_DATA_TYPE_FLOAT16, rank, const_cast<void*>(base), dims, strides, box,
                              estr, CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B,
                              CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}
// A pool as a matrix of positions, each a row of all heads: a box is 64 dims of `box` of them.
static bool pool_map(CUtensorMap* map, const void* pool, long long rows, int width, int box) {
  const cuuint64_t dims[2] = {(cuuint64_t)width, (cuuint64_t)rows}, strides[1] = {(cuuint64_t)width * 2};
  const cuuint32_t boxes[2] = {64, (cuuint32_t)box};
  return encode(map, pool, 2, dims, strides, boxes);
}
// Queries: a box is 64 dims of a group's heads of a tile's tokens.
static bool query_map(CUtensorMap* map, const Params& p, int D) {
  const cuuint64_t dims[3] = {(cuuint64_t)D, (cuuint64_t)p.Hq, (cuuint64_t)p.T};
  const cuuint64_t strides[2] = {(cuuint64_t)D * 2, (cuuint64_t)p.q_stride * 2};
  const cuuint32_t boxes[3] = {64, (cuuint32_t)p.group, (cuuint32_t)p.tpt};
  return encode(map, p.q, 3, dims, strides, boxes);
}

template <int D>
static int launch(const CUtensorMap& mq, const CUtensorMap& mk, const CUtensorMap& mv, const Params& p, int ctas,
                  unsigned flags, cudaStream_t st) {
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(ctas);
  cfg.blockDim = dim3(kThreads);
  cfg.dynamicSmemBytes = smem_bytes<D>();
  cfg.stream = st;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = attr;
  cfg.numAttrs = (flags & ANVILQ_GEMM_OVERLAP_PRIOR) ? 1 : 0;
  if (cudaLaunchKernelEx(&cfg, chunk_kernel<D>, mq, mk, mv, p) != cudaSuccess) {
    cudaGetLastError();
    return ANVILQ_ECUDA;
  }
  if (ctas == 1) return ANVILQ_OK;   // nothing is shared
  cfg.gridDim = dim3(std::min(ctas * 8, kMaxCtas * 3));
  cfg.blockDim = dim3(kMergeThreads);
  cfg.dynamicSmemBytes = 0;
  cfg.numAttrs = 1;
  if (cudaLaunchKernelEx(&cfg, merge_kernel<D>, p, ctas) != cudaSuccess) {
    cudaGetLastError();
    return ANVILQ_ECUDA;
  }
  return ANVILQ_OK;
}

// CTAs of a call: one an SM, no more than there can be units.
static int ctas_for(int sms, int T, int B, int Hq, int Hkv, long long capacity) {
  const int tpt = kRows / (Hq / Hkv);
  const double pairs = ((double)T / (2 * tpt) + std::min(T, B)) * Hkv;
  return (int)std::max(1.0, std::min({(double)std::min(sms, kMaxCtas), pairs * (double)((capacity + kKeys - 1) / kKeys)}));
}
static size_t partial_bytes(int ctas, int D) { return (size_t)ctas * kSlots * 2 * kRows * (D + 2) * sizeof(float); }

}  // namespace chunk
}  // namespace anvilq

extern "C" {

size_t anvilq_gqa_chunk_paged_workspace_size(int T, int B, int Hq, int Hkv, int D, int page_tokens, int max_pages) {
  using namespace anvilq::chunk;
  if (!shape_ok(T, B, Hq, Hkv, D) || page_tokens < 16 || page_tokens % 16 || max_pages < 1 ||
      (long long)page_tokens * max_pages > (1LL << 30))
    return 0;
  const int sms = sm_count();
  if (sms <= 0) return 0;
  const int ctas = ctas_for(sms, T, B, Hq, Hkv, (long long)page_tokens * max_pages);
  return ANVILQ_WORKSPACE_COUNTER_BYTES + partial_bytes(ctas, D) + ctas * (2 * kRows * sizeof(float2) + sizeof(Open));
}

int anvilq_gqa_chunk_paged(const uint16_t* q, long long q_stride, const uint16_t* k_pool, const uint16_t* v_pool,
                           const uint32_t* page_table, const int32_t* seqlens, const int32_t* token_starts,
                           uint16_t* out, int T, int B, int Hq, int Hkv, int D, int page_tokens, int max_pages,
                           int num_pages, float scale, void* workspace, size_t workspace_bytes, int* dev_err,
                           unsigned flags, anvilq_stream_t stream) {
  using namespace anvilq;
  using namespace anvilq::chunk;
  if ((T != 0 && (!q || !out)) || !k_pool || !v_pool || !page_table || !seqlens || !token_starts || !dev_err)
    return ANVILQ_EINVAL;
  if (flags & ~(unsigned)ANVILQ_GEMM_OVERLAP_PRIOR) return ANVILQ_EINVAL;
  if (!std::isfinite(scale) || scale > kMaxScale) return ANVILQ_EINVAL;
  if (T < 0 || (T > 0 && q_stride < (long long)Hq * D)) return ANVILQ_EINVAL;
  if (!shape_ok(T, B, Hq, Hkv, D) || page_tokens < 16 || page_tokens % 16 || max_pages < 1 || num_pages < 1 ||
      (long long)page_tokens * max_pages > (1LL << 30))
    return ANVILQ_ESHAPE;
  const long long positions = (long long)num_pages * page_tokens;
  if (positions > 0x7FFFFFFFLL || (T > 0 && q_stride > 1LL << 38)) return ANVILQ_ESHAPE;   // of a tensor map
  if (!a16(q) || !a16(k_pool) || !a16(v_pool) || !a16(out) || !a16(workspace) || q_stride % 8) return ANVILQ_EALIGN;
  if (T == 0) return ANVILQ_OK;
  const size_t pool = (size_t)positions * Hkv * D * 2, rows = (size_t)T * Hq * D * 2;
  const size_t read = ((size_t)(T - 1) * q_stride + (size_t)Hq * D) * 2;
  // the outputs and the workspace are written while all else is still to be read
  const struct {
    const void* start;
    size_t bytes;
  } reads[] = {{q, read}, {k_pool, pool}, {v_pool, pool}, {page_table, (size_t)B * max_pages * 4},
               {seqlens, (size_t)B * 4}, {token_starts, (size_t)(B + 1) * 4}};
  const size_t scratch = workspace ? workspace_bytes : 0;
  for (const auto& r : reads)
    if (overlap(out, rows, r.start, r.bytes) || overlap(workspace, scratch, r.start, r.bytes)) return ANVILQ_EINVAL;
  if (overlap(out, rows, workspace, scratch)) return ANVILQ_EINVAL;
  const int sms = sm_count();
  if (sms <= 0) return ANVILQ_ECUDA;
  const size_t need = anvilq_gqa_chunk_paged_workspace_size(T, B, Hq, Hkv, D, page_tokens, max_pages);
  if (!workspace || workspace_bytes < need) return ANVILQ_EWORKSPACE;
  const int ctas = ctas_for(sms, T, B, Hq, Hkv, (long long)page_tokens * max_pages);
  Params p{};
  p.q = reinterpret_cast<const __half*>(q);
  p.q_stride = q_stride;
  p.starts = token_starts;
  p.seqlens = seqlens;
  p.page_table = page_table;
  p.out = reinterpret_cast<__half*>(out);
  char* at = static_cast<char*>(workspace) + ANVILQ_WORKSPACE_COUNTER_BYTES;
  p.partials = reinterpret_cast<float*>(at);
  p.fresh = reinterpret_cast<float2*>(at + partial_bytes(ctas, D));
  p.open = reinterpret_cast<Open*>(p.fresh + (size_t)ctas * 2 * kRows);
  p.dev_err = dev_err;
  p.scale_log2 = (scale > 0.0f ? scale : 1.0f / std::sqrt((float)D)) * 1.4426950408889634f;
  p.scale_large = std::ldexp(1.0f, std::ilogb(p.scale_log2) + 5);
  p.T = T; p.B = B; p.Hq = Hq; p.Hkv = Hkv;
  p.group = Hq / Hkv;
  p.tpt = kRows / p.group;
  p.page_tokens = page_tokens; p.max_pages = max_pages; p.num_pages = num_pages;
  // Stores of 32 bytes need addresses of their multiples, out need only lie on 16.  (12 mixed
  // sequences 127 us a call, by stores of 16 bytes 131; 4096 tokens after 12288 the same.)
  p.sectors = reinterpret_cast<uintptr_t>(out) % 32 == 0;
  p.box = 16;
  while (p.box < kKeys && page_tokens % (2 * p.box) == 0) p.box *= 2;
  CUtensorMap mq, mk, mv;
  if (!query_map(&mq, p, D) || !pool_map(&mk, k_pool, positions, Hkv * D, p.box) || !pool_map(&mv, v_pool, positions, Hkv * D, p.box))
    return ANVILQ_ECUDA;
  cudaStream_t st = reinterpret_cast<cudaStream_t>(stream);
  return D == 64 ? launch<64>(mq, mk, mv, p, ctas, flags, st) : launch<128>(mq, mk, mv, p, ctas, flags, st);
}

}  // extern "C"
