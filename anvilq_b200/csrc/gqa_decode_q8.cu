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
// Work split.  A tile is a block of 16 tokens of one kv head: 2 KB of K codes and
// 2 KB of V codes at D = 128, each one contiguous run, one TMA box.  The rows of a
// tile's products are the Q * Hq/Hkv query rows of its kv head, in groups of 8 or
// 16 (kRows); a pair is a (sequence, kv head, row group).  All pairs' tiles in a
// row -- sequence, then pair, then tile -- are cut into equal stretches, one a
// warp, so that the device is evenly loaded whatever the lengths; the table of
// lengths is on the device, so every warp finds its stretch from it.  A pair that
// lies inside one warp's stretch is finished by that warp.  The others' partial
// softmax states are merged in shared memory, and where a pair spans CTAs, by the
// CTA that arrives last at the pair's ticket, in CTA order (bit-reproducible).
//
// A warp streams its tiles through its own TMA ring, mbarrier by mbarrier.  The
// codes never return to memory as binary16: fragments of mma.m16n8k16 are formed
// in registers.
//   S = Q K^T: a lane's B fragment is a token's 16-byte chunks (the contraction's
//     order over d is free, so q is loaded in the same order).  An int8 code c
//     enters as the binary16 subnormal (c + 128) 2^-24 -- a byte beside a zero
//     byte, no arithmetic -- and the accumulator starts at -128 2^-24 sum q.  An
//     e4m3 code is converted (exactly) by the cvt instruction.
//   O^T += V^T P^T: the accumulator layout of S is the B fragment of P^T; V^T's
//     fragments pair the bytes of two tokens.  Over a long context the sum of p c
//     is far smaller than the sum of p, so here an offset would cost precision:
//     int8 codes are made signed first, (1024 + 128 + c) - 1152 in binary16.
// The tokens of a tile are dealt to fragment columns in an order (token_of) that
// keeps both reads of the 128-byte-swizzled tile free of bank conflicts.
//
// Softmax: binary32, log2 domain, online.  The running reference m is not the
// maximum but stays within 12 of it (above: p <= 2^12; m is set 4 below a new
// maximum), so that most tiles neither reduce over lanes nor rescale; p then fits
// binary16 with more room below than the maximum itself would leave.  The V scale
// is folded into p relative to a running F, which likewise moves only when a
// block's scale leaves [F/8, 8F]: p vs/F <= 2^15.
#include <cuda.h>
#include <cudaTypedefs.h>

#include <algorithm>
#include <cmath>
#include <mutex>

#include "kv_q8.cuh"

namespace anvilq {
namespace attn8 {

using q8::kBlock;
constexpr int kTile = kBlock;
constexpr unsigned long long kWaitLimitNs = 1000000000ull;

struct Params {
  const __half* q;             // [B][Q][Hq][D]
  const float* k_scales;       // [num_pages][Hkv][page_tokens / 16]
  const float* v_scales;
  const uint32_t* page_table;  // [B][max_pages]
  const int* seqlens;          // [B]
  __half* out;                 // [B][Q][Hq][D]
  int* tickets;                // one a CTA (of the pair that starts in it and ends in a later one)
  float* partials;             // [CTA][2] states: of the pair begun earlier, of the pair that goes on
  int* dev_err;
  int B, Q, Hq, Hkv, group, row_groups, page_tokens, max_pages, num_pages;
  float scale_log2;            // softmax scale * log2(e)
};

// RT: rows of a pair in eights
template <int D_, int RT_>
struct Shape {
  static constexpr int D = D_, RT = RT_;
  static constexpr int kRows = 8 * RT;
  static constexpr int kWarps = RT == 1 ? 8 : 4;
  static constexpr int kThreads = kWarps * 32;
  static constexpr int kCtas = RT == 1 ? 2 : 3;                // per SM
  static constexpr int kStages = D == 128 ? 2 : 4;
  static constexpr int kTileBytes = kTile * D;                 // of K or V
  static constexpr int kStageBytes = 2 * kTileBytes;
  static constexpr int kRingBytes = kStages * kStageBytes;     // per warp
  static constexpr int kState = kRows * D;                     // floats of a state's o
  // a warp's state of a pair begun earlier has its own room (the ring is in use
  // when it is stored); that of a pair that goes on takes the idle ring
  static constexpr int kStateOffset = kWarps * kRingBytes;
  static constexpr int kStatOffset = kStateOffset + kWarps * kState * 4;   // (m, l) [warp][2][row]
  static constexpr int kMetaOffset = kStatOffset + kWarps * 2 * kRows * 8;
  static constexpr int kBarOffset = kMetaOffset + kWarps * kStages * 32;
  static constexpr int kTotal = kBarOffset + kWarps * kStages * 8 + 1024;  // + slack to align the ring
  static constexpr int kPartial = kState + 2 * kRows;          // floats of a state in global memory
  static_assert(kRingBytes >= kState * 4, "a state fits the idle ring");
  static_assert(kCtas * (kTotal + 2048) <= 227 * 1024, "CTAs per SM");
};

struct Meta {        // what a tile's consumer needs beside the codes
  float ks, vs;      // scales
  int tile, n;       // tile of the pair, the pair's tiles
  int b, pair;       // sequence, pair of the sequence
  int pad[2];
};
static_assert(sizeof(Meta) == 32, "one 32-byte slot a stage");

struct Part {        // a warp's state of a pair that it did not finish alone
  long long first;   // the pair's first tile in the row of all tiles
  int n, b, pair;
  int valid, ends;   // ends: the pair's last tile is in it
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
// Bounded wait: true when the phase completed, false after ~kWaitLimitNs.
__device__ __forceinline__ bool mbar_wait_bounded(uint32_t bar, uint32_t parity) {
  if (mbar_try_wait(bar, parity)) return true;
  const unsigned long long t0 = globaltimer();
  for (uint32_t i = 0;; ++i) {
    if (mbar_try_wait(bar, parity)) return true;
    if ((i & 63u) == 63u && globaltimer() - t0 > kWaitLimitNs) return false;
  }
}
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
  asm volatile(
      "mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, "
      "{%0,%1,%2,%3};"
      : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
      : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}
__device__ __forceinline__ uint32_t pack_half2(float lo, float hi) {
  const __half2 h = __floats2half2_rn(lo, hi);
  return *reinterpret_cast<const uint32_t*>(&h);
}
__device__ __forceinline__ float fast_exp2(float x) {   // 2^x, 2 units in the last place; 0 for -inf
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}
__device__ __forceinline__ uint32_t e4m3x2_to_half2(uint32_t low16) {
  uint32_t h;
  asm("{\n .reg .b16 t;\n cvt.u16.u32 t, %1;\n cvt.rn.f16x2.e4m3x2 %0, t;\n}" : "=r"(h) : "r"(low16));
  return h;
}
// The token of a tile at column n (of 16) of S: within eights, even columns keep
// their place and odd ones are crossed, so that the two rows of a quarter-warp's
// K read differ in bit 2 and the four rows of its V read in bits 1 and 2 -- with
// the swizzle, 8 different 16-byte banks either way.
__device__ __forceinline__ int token_of(int n) { return (n & 8) | ((n & 1) ? ((n & 6) ^ 5) : (n & 7)); }

template <int D, int TYPE, int RT>
__global__ void __launch_bounds__(Shape<D, RT>::kThreads, Shape<D, RT>::kCtas)
    gqa_decode_q8_kernel(const __grid_constant__ CUtensorMap mk, const __grid_constant__ CUtensorMap mv,
                         const __grid_constant__ Params p) {
  using S = Shape<D, RT>;
  constexpr int KS = D / 16;        // k-steps of S, m-tiles of O^T
  constexpr int NC = D / 64;        // 16-byte K chunks of a lane
  constexpr int VW = D / 32;        // V words of a lane and token
  constexpr int W = S::kWarps;
  extern __shared__ __align__(1024) unsigned char smem_raw[];
  __shared__ Part s_part[W][2];
  __shared__ int s_last[2];
  unsigned char* smem = smem_raw + ((1024u - (smem_u32(smem_raw) & 1023u)) & 1023u);
  const int warp = threadIdx.x / 32, lane = threadIdx.x % 32;
  const int g = lane / 4, c = lane % 4;
  unsigned char* ring = smem + warp * S::kRingBytes;
  Meta* meta = reinterpret_cast<Meta*>(smem + S::kMetaOffset) + warp * S::kStages;
  const uint32_t bar0 = smem_u32(smem + S::kBarOffset) + warp * S::kStages * 8;
  if (lane == 0) {
    for (int s = 0; s < S::kStages; ++s)
      asm volatile("mbarrier.init.shared::cta.b64 [%0], 1;" ::"r"(bar0 + 8 * s) : "memory");
    s_part[warp][0].valid = s_part[warp][1].valid = 0;
    asm volatile("prefetch.tensormap [%0];" ::"l"(&mk) : "memory");
    asm volatile("prefetch.tensormap [%0];" ::"l"(&mv) : "memory");
  }
  asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
  __syncwarp();
  asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
  asm volatile("griddepcontrol.wait;" ::: "memory");

  const long long capacity = (long long)p.page_tokens * p.max_pages;
  auto tiles_of = [&](int b) {
    const int n = p.seqlens[b];
    return n < 0 || n > capacity ? 0 : (n + kTile - 1) / kTile;
  };
  // empty sequences (and lengths that are none) are this loop's
  for (int b = blockIdx.x; b < p.B; b += gridDim.x) {
    const int n = p.seqlens[b];
    if (n >= 1 && n <= capacity) continue;
    if (n != 0 && threadIdx.x == 0) atomicOr(p.dev_err, ANVILQ_DEV_ERR_SEQLEN);
    uint4* o = reinterpret_cast<uint4*>(p.out + (size_t)b * p.Q * p.Hq * D);
    for (int i = threadIdx.x; i < p.Q * p.Hq * (D / 8); i += S::kThreads) o[i] = make_uint4(0, 0, 0, 0);
  }

  // ---- this warp's stretch [begin, end) of all tiles ----
  const int pairs = p.Hkv * p.row_groups;   // of a sequence
  long long total = 0;
  for (int b = lane; b < p.B; b += 32) total += tiles_of(b);
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) total += __shfl_xor_sync(0xffffffffu, total, o);
  total *= pairs;
  const long long workers = (long long)gridDim.x * W;
  const long long chunk = max(1ll, (total + workers - 1) / workers);
  const long long begin = ((long long)blockIdx.x * W + warp) * chunk;
  const long long end = min(total, begin + chunk);
  const int count = (int)max(0ll, end - begin);   // chunk <= 2^30 tiles of 16 tokens
  // the sequence of the first tile, and where its tiles start
  int at_b = 0;
  long long at_base = 0;
  if (count > 0) {
    for (int b0 = 0;; b0 += 32) {
      const long long mine = b0 + lane < p.B ? (long long)tiles_of(b0 + lane) * pairs : 0;
      long long incl = mine;
#pragma unroll
      for (int o = 1; o < 32; o <<= 1) {
        const long long up = __shfl_up_sync(0xffffffffu, incl, o);
        if (lane >= o) incl += up;
      }
      const uint32_t past = __ballot_sync(0xffffffffu, at_base + incl > begin);
      if (past) {   // some sequence holds it, as begin < total
        const int l = __ffs(past) - 1;
        at_b = b0 + l;
        at_base += __shfl_sync(0xffffffffu, incl - mine, l);
        break;
      }
      at_base += __shfl_sync(0xffffffffu, incl, 31);
    }
  }

  // ---- producer: lane l of the warp prepares tile j0 + l of every 32 and issues it ----
  int pr_row = 0;          // row of the pools (as matrices of D-byte rows) of this lane's tile
  Meta pr_meta;
  auto prepare = [&](int j0) {
    const long long x = begin + min(j0 + lane, count - 1);
    int n = tiles_of(at_b);
    while (x >= at_base + (long long)n * pairs && at_b + 1 < p.B) {
      at_base += (long long)n * pairs;
      n = tiles_of(++at_b);
    }
    // the bounds below hold by themselves unless the lengths change under the kernel
    n = max(n, 1);
    const unsigned long long rel = (unsigned long long)(x - at_base);
    pr_meta.b = at_b;
    pr_meta.n = n;
    pr_meta.pair = min((int)(rel / (unsigned)n), pairs - 1);
    pr_meta.tile = (int)min(rel - (unsigned long long)pr_meta.pair * n, (unsigned long long)n - 1);
    const int t0 = pr_meta.tile * kTile;
    int page = q8::page_of(p.page_table, p.max_pages, p.num_pages, at_b, t0 / p.page_tokens);
    if (page < 0) {   // reported; the copies then stay inside the pool
      atomicOr(p.dev_err, ANVILQ_DEV_ERR_PAGE);
      page = 0;
    }
    const size_t run = (size_t)page * p.Hkv + pr_meta.pair / p.row_groups;
    const int row = t0 % p.page_tokens;
    pr_row = (int)(run * p.page_tokens + row);
    const size_t block = run * (p.page_tokens / kBlock) + row / kBlock;
    pr_meta.ks = p.k_scales[block];
    pr_meta.vs = p.v_scales[block];
    // the next 32 start where the last of these is
    at_b = __shfl_sync(0xffffffffu, at_b, 31);
    at_base = __shfl_sync(0xffffffffu, at_base, 31);
  };
  auto copy = [&](int j) {
    if (lane == j % 32) {
      const int st = j % S::kStages;
      const uint32_t bar = bar0 + 8 * st, dst = smem_u32(ring + st * S::kStageBytes);
      asm volatile("mbarrier.arrive.expect_tx.shared::cta.b64 _, [%0], %1;" ::"r"(bar), "r"(S::kStageBytes) : "memory");
      tma_2d(dst, &mk, 0, pr_row, bar);
      tma_2d(dst + S::kTileBytes, &mv, 0, pr_row, bar);
    }
  };
  auto note = [&](int j) {
    if (lane == j % 32) meta[j % S::kStages] = pr_meta;
  };
  int issued = 0;
  if (count > 0) {
    prepare(0);
    const int ahead = min(S::kStages, count);
    for (; issued < ahead; ++issued) copy(issued);
    for (int j = 0; j < ahead; ++j) note(j);   // after the copies: these wait for the scales
    __syncwarp();
  }

  // ---- the state of the current pair ----
  uint32_t qa[KS][2 * RT];   // A fragments: rows g (and g + 8)
  float start[RT];           // where S's accumulators start
  float m[RT], l[RT];
  float o[RT][KS][4];        // O^T: dims g.., rows 8 t + 2 c and + 1
  float F = 1.0f, F_inv = 1.0f, F_top = 1.0f;
  int len = 0, sees[RT];     // positions that row g (g + 8) sees
  bool from_start = false;   // the pair's first tile was in this stretch
  bool ok = true;

  for (int j = 0; j < count; ++j) {
    const int st = j % S::kStages;
    if (ok) {
      const bool landed = mbar_wait_bounded(bar0 + 8 * st, (j / S::kStages) & 1);
      if (!__all_sync(0xffffffffu, landed)) {   // no more tiles are used; the stretch is walked to its end
        ok = false;
        if (lane == 0) atomicOr(p.dev_err, ANVILQ_DEV_ERR_TIMEOUT);
      }
    }
    if (!ok) break;
    const Meta md = meta[st];
    const int t0 = md.tile * kTile;
    if (j == 0 || md.tile == 0) {
      // a new pair: its query rows, and an empty state
      from_start = md.tile == 0;
      len = p.seqlens[md.b];
      const int kvh = md.pair / p.row_groups, r0 = (md.pair % p.row_groups) * S::kRows;
#pragma unroll
      for (int t = 0; t < RT; ++t) {
        const int r = r0 + 8 * t + g, i = r / p.group;
        const bool row = i < p.Q;
        sees[t] = row ? len - p.Q + 1 + i : 0;
        const __half* src = p.q + (((size_t)md.b * p.Q + (row ? i : 0)) * p.Hq + kvh * p.group + r % p.group) * D + 16 * c;
        float sum = 0.0f;
#pragma unroll
        for (int h = 0; h < NC; ++h)
#pragma unroll
          for (int u = 0; u < 2; ++u) {
            uint4 w = make_uint4(0, 0, 0, 0);
            if (row) w = *reinterpret_cast<const uint4*>(src + 64 * h + 8 * u);
            qa[4 * h + 2 * u][t] = w.x;
            qa[4 * h + 2 * u][RT + t] = w.y;
            qa[4 * h + 2 * u + 1][t] = w.z;
            qa[4 * h + 2 * u + 1][RT + t] = w.w;
            if (TYPE == q8::kInt8) {
              const uint32_t v[4] = {w.x, w.y, w.z, w.w};
#pragma unroll
              for (int e = 0; e < 4; ++e) {
                const float2 f = __half22float2(*reinterpret_cast<const __half2*>(&v[e]));
                sum += f.x + f.y;
              }
            }
          }
        if (TYPE == q8::kInt8) {
          sum += __shfl_xor_sync(0xffffffffu, sum, 1);
          sum += __shfl_xor_sync(0xffffffffu, sum, 2);
        }
        start[t] = sum * -0x1p-17f;   // -128 2^-24
        m[t] = -1e30f;
        l[t] = 0.0f;
#pragma unroll
        for (int mt = 0; mt < KS; ++mt) o[t][mt][0] = o[t][mt][1] = o[t][mt][2] = o[t][mt][3] = 0.0f;
      }
      F = F_inv = F_top = 1.0f;
    }

    // ---- S = Q K^T: columns token_of(0..7) and token_of(8..15) ----
    const unsigned char* kt = ring + st * S::kStageBytes;
    const unsigned char* vt = kt + S::kTileBytes;
    float s[2][4];
#pragma unroll
    for (int nt = 0; nt < 2; ++nt) {
      s[nt][0] = s[nt][1] = TYPE == q8::kInt8 ? start[0] : 0.0f;
      s[nt][2] = s[nt][3] = TYPE == q8::kInt8 ? start[RT - 1] : 0.0f;
      const int row = token_of(8 * nt + g);
#pragma unroll
      for (int h = 0; h < NC; ++h) {
        const int at = D == 128 ? row * 128 + (((c + 4 * h) ^ (row & 7)) << 4) : row * 64 + ((c ^ ((row >> 1) & 3)) << 4);
        const uint4 w = *reinterpret_cast<const uint4*>(kt + at);
        const uint32_t v[4] = {w.x, w.y, w.z, w.w};
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          uint32_t b0, b1;
          if (TYPE == q8::kInt8) {
            const uint32_t u = v[e] ^ 0x80808080u;
            b0 = __byte_perm(u, 0, 0x4140);
            b1 = __byte_perm(u, 0, 0x4342);
          } else {
            b0 = e4m3x2_to_half2(v[e]);
            b1 = e4m3x2_to_half2(v[e] >> 16);
          }
          const uint32_t* a = qa[4 * h + e];
          if (RT == 1) mma16816(s[nt], a[0], 0u, a[1], 0u, b0, b1);
          else mma16816(s[nt], a[0], a[RT - 1], a[RT], a[2 * RT - 1], b0, b1);
        }
      }
    }

    // ---- softmax: rows g (c0, c1) and, with RT == 2, g + 8 (c2, c3) ----
    const float ks = md.ks * p.scale_log2 * (TYPE == q8::kInt8 ? 0x1p24f : 1.0f);
    float x[RT][4];
#pragma unroll
    for (int t = 0; t < RT; ++t)
#pragma unroll
      for (int e = 0; e < 4; ++e) x[t][e] = s[e >> 1][2 * t + (e & 1)] * ks;
    const bool edge = t0 + kTile > len - p.Q + 1;   // some row does not see all of the tile
    if (edge) {
#pragma unroll
      for (int t = 0; t < RT; ++t)
#pragma unroll
        for (int e = 0; e < 4; ++e)
          if (t0 + token_of(8 * (e >> 1) + 2 * c + (e & 1)) >= sees[t]) x[t][e] = -INFINITY;
    }
    float mx[RT];
    bool above = false;
#pragma unroll
    for (int t = 0; t < RT; ++t) {
      mx[t] = fmaxf(fmaxf(x[t][0], x[t][1]), fmaxf(x[t][2], x[t][3]));
      above |= mx[t] > m[t] + 12.0f;
    }
    if (__any_sync(0xffffffffu, above)) {
#pragma unroll
      for (int t = 0; t < RT; ++t) {
        mx[t] = fmaxf(mx[t], __shfl_xor_sync(0xffffffffu, mx[t], 1));
        mx[t] = fmaxf(mx[t], __shfl_xor_sync(0xffffffffu, mx[t], 2));
        const float m_new = mx[t] > m[t] + 12.0f ? mx[t] - 4.0f : m[t];
        const float alpha = fast_exp2(m[t] - m_new);
        m[t] = m_new;
        l[t] *= alpha;
        const float a0 = __shfl_sync(0xffffffffu, alpha, 8 * c), a1 = __shfl_sync(0xffffffffu, alpha, 8 * c + 4);
#pragma unroll
        for (int mt = 0; mt < KS; ++mt) {
          o[t][mt][0] *= a0;
          o[t][mt][1] *= a1;
          o[t][mt][2] *= a0;
          o[t][mt][3] *= a1;
        }
      }
    }
    float vs = md.vs * F_inv;
    if ((vs > 8.0f || vs < 0.125f) && md.vs > 0.0f) {
      // 2^-40 of the largest scale so far is below what the binary16 result can
      // show of it, and keeps o / F inside binary32
      F_top = fmaxf(F_top, md.vs);
      const float F_new = fmaxf(md.vs, F_top * 0x1p-40f);
      const float f = F * (F_inv = 1.0f / F_new);
      F = F_new;
      vs = md.vs * F_inv;
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
      float pr[4];
#pragma unroll
      for (int e = 0; e < 4; ++e) pr[e] = fast_exp2(x[t][e] - m[t]);
      l[t] += (pr[0] + pr[1]) + (pr[2] + pr[3]);
      pb[t][0] = pack_half2(pr[0] * vs, pr[1] * vs);
      pb[t][1] = pack_half2(pr[2] * vs, pr[3] * vs);
    }

    // ---- O^T += V^T P^T ----
    uint32_t v[4][VW];
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      const int row = token_of(8 * (e >> 1) + 2 * c + (e & 1));
      if (D == 128) {
        const uint4 w = *reinterpret_cast<const uint4*>(vt + row * 128 + ((g ^ (row & 7)) << 4));
        v[e][0] = w.x; v[e][1] = w.y; v[e][2 % VW] = w.z; v[e][3 % VW] = w.w;
      } else {
        const uint2 w = *reinterpret_cast<const uint2*>(vt + row * 64 + (((g >> 1) ^ ((row >> 1) & 3)) << 4) + 8 * (g & 1));
        v[e][0] = w.x; v[e][1] = w.y;
      }
      // rows behind the sequence may hold anything: an e4m3 NaN times p = 0 would be a NaN
      if (TYPE == q8::kE4m3 && edge && t0 + row >= len) {
#pragma unroll
        for (int w = 0; w < VW; ++w) v[e][w] = 0u;
      }
    }
    __syncwarp();
    // the stage is free again
    if (issued < count) {
      if (issued % 32 == 0) prepare(issued);
      copy(issued);
      note(issued);
      ++issued;
      __syncwarp();
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
            const __half2 h = __hsub2(*reinterpret_cast<__half2*>(&a[e]), off);
            a[e] = *reinterpret_cast<const uint32_t*>(&h);
          }
        } else {
          a[0] = e4m3x2_to_half2(p01);
          a[1] = e4m3x2_to_half2(p01 >> 16);
          a[2] = e4m3x2_to_half2(p23);
          a[3] = e4m3x2_to_half2(p23 >> 16);
        }
#pragma unroll
        for (int t = 0; t < RT; ++t) mma16816(o[t][2 * w + u], a[0], a[1], a[2], a[3], pb[t][0], pb[t][1]);
      }

    // ---- the pair's last tile here ----
    const bool ends = md.tile == md.n - 1;
    if (ends || j == count - 1) {
#pragma unroll
      for (int t = 0; t < RT; ++t) {
        l[t] += __shfl_xor_sync(0xffffffffu, l[t], 1);
        l[t] += __shfl_xor_sync(0xffffffffu, l[t], 2);
      }
      if (from_start && ends) {
        const int kvh = md.pair / p.row_groups, r0 = (md.pair % p.row_groups) * S::kRows;
#pragma unroll
        for (int t = 0; t < RT; ++t) {
          const float inv = l[t] == 0.0f ? 0.0f : F / l[t];
#pragma unroll
          for (int e = 0; e < 2; ++e) {
            const float f = __shfl_sync(0xffffffffu, inv, 8 * c + 4 * e);
            const int r = r0 + 8 * t + 2 * c + e, i = r / p.group;
            if (i < p.Q) {
              __half* dst = p.out + (((size_t)md.b * p.Q + i) * p.Hq + kvh * p.group + r % p.group) * D + g * (D / 8);
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
        const int slot = from_start ? 1 : 0;
        float* state = from_start ? reinterpret_cast<float*>(ring)
                                  : reinterpret_cast<float*>(smem + S::kStateOffset) + warp * S::kState;
        float2* stat = reinterpret_cast<float2*>(smem + S::kStatOffset) + (warp * 2 + slot) * S::kRows;
        __syncwarp();
#pragma unroll
        for (int t = 0; t < RT; ++t) {
          if (c == 0) stat[8 * t + g] = make_float2(m[t], l[t]);
#pragma unroll
          for (int e = 0; e < 2; ++e) {
            float4* dst = reinterpret_cast<float4*>(state + (8 * t + 2 * c + e) * D + g * (D / 8));
#pragma unroll
            for (int q = 0; q < KS / 2; ++q)
              dst[q] = make_float4(o[t][2 * q][e] * F, o[t][2 * q][2 + e] * F, o[t][2 * q + 1][e] * F,
                                   o[t][2 * q + 1][2 + e] * F);
          }
        }
        if (lane == 0) {
          const long long x = begin + j;
          s_part[warp][slot] = Part{x - md.tile, md.n, md.b, md.pair, 1, ends};
        }
      }
    }
  }
  if (!ok) {
    // copies in flight land before the shared memory is given up
    for (int j = max(0, issued - S::kStages); j < issued; ++j)
      if (j >= 0) mbar_wait_bounded(bar0 + 8 * (j % S::kStages), (j / S::kStages) & 1);
  }
  __syncthreads();

  // ---- merge what the warps left ----
  // A chain: the states of one pair in consecutive warps.  It begins with a
  // pair begun earlier in warp 0, or with a warp's pair that goes on.
  auto weights = [](float M, float mi) { return fast_exp2(mi - M); };
  auto finish = [&](const Part& pt, int row, int d4, float4 acc, float lsum) {
    const int kvh = pt.pair / p.row_groups, r = (pt.pair % p.row_groups) * S::kRows + row, i = r / p.group;
    if (i >= p.Q) return;
    const float inv = lsum == 0.0f ? 0.0f : 1.0f / lsum;
    __half* dst = p.out + (((size_t)pt.b * p.Q + i) * p.Hq + kvh * p.group + r % p.group) * D + 4 * d4;
    *reinterpret_cast<uint2*>(dst) =
        make_uint2(pack_half2(acc.x * inv, acc.y * inv), pack_half2(acc.z * inv, acc.w * inv));
  };
  const float2* stats = reinterpret_cast<const float2*>(smem + S::kStatOffset);
  Part open[2];                       // this CTA's share of pairs that span CTAs
  open[0].valid = open[1].valid = 0;
  for (int w = 0; w < W; ++w)
    for (int slot = w == 0 ? 0 : 1; slot < 2; ++slot) {
      const Part first = s_part[w][slot];
      if (!first.valid) continue;
      int members = 1;
      bool ended = first.ends != 0;
      while (!ended && w + members < W && s_part[w + members][0].valid) {
        ended = s_part[w + members][0].ends != 0;
        ++members;
      }
      const bool whole = slot == 1 && ended;
      float* out = p.partials + ((size_t)blockIdx.x * 2 + slot) * S::kPartial;
      for (int i = threadIdx.x; i < S::kRows * (D / 4); i += S::kThreads) {
        const int row = i / (D / 4), d4 = i % (D / 4);
        float M = -1e30f, lsum = 0.0f;
        for (int k = 0; k < members; ++k) M = fmaxf(M, stats[((w + k) * 2 + (k ? 0 : slot)) * S::kRows + row].x);
        float4 acc = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
        for (int k = 0; k < members; ++k) {
          const float2 ml = stats[((w + k) * 2 + (k ? 0 : slot)) * S::kRows + row];
          const float f = weights(M, ml.x);
          const float* state = k == 0 && slot == 1 ? reinterpret_cast<const float*>(smem + w * S::kRingBytes)
                                                   : reinterpret_cast<const float*>(smem + S::kStateOffset) + (w + k) * S::kState;
          const float4 v = *reinterpret_cast<const float4*>(state + row * D + 4 * d4);
          lsum += f * ml.y;
          acc.x += f * v.x; acc.y += f * v.y; acc.z += f * v.z; acc.w += f * v.w;
        }
        if (whole) {
          finish(first, row, d4, acc, lsum);
        } else {
          __stcg(reinterpret_cast<float4*>(out + row * D) + d4, acc);
          if (d4 == 0) __stcg(reinterpret_cast<float2*>(out + S::kState) + row, make_float2(M, lsum));
        }
      }
      if (!whole) open[slot] = first;
    }
  if (!open[0].valid && !open[1].valid) return;

  // ---- pairs that span CTAs: the last CTA to arrive merges, in CTA order ----
  const long long cta_tiles = chunk * W;
  int first_cta[2], ctas[2];
#pragma unroll
  for (int s = 0; s < 2; ++s) {
    first_cta[s] = s == 1 ? (int)blockIdx.x : open[0].valid ? (int)(open[0].first / cta_tiles) : 0;
    ctas[s] = open[s].valid ? (int)((open[s].first + open[s].n - 1) / cta_tiles) - first_cta[s] + 1 : 0;
  }
  __threadfence();
  __syncthreads();
  if (threadIdx.x < 2) {
    const int s = threadIdx.x;
    bool last = false;
    if (open[s].valid) {
      last = atomicAdd(p.tickets + first_cta[s], 1) == ctas[s] - 1;
      if (last) p.tickets[first_cta[s]] = 0;
    }
    s_last[s] = last;
  }
  __syncthreads();
  for (int s = 0; s < 2; ++s) {
    if (!s_last[s]) continue;
    __threadfence();
    // the first CTA's state is of a pair that goes on, the others' of one begun earlier
    auto state_of = [&](int k) { return p.partials + ((size_t)(first_cta[s] + k) * 2 + (k == 0)) * S::kPartial; };
    for (int i = threadIdx.x; i < S::kRows * (D / 4); i += S::kThreads) {
      const int row = i / (D / 4), d4 = i % (D / 4);
      float M = -1e30f, lsum = 0.0f;
      for (int k = 0; k < ctas[s]; ++k)
        M = fmaxf(M, __ldcg(reinterpret_cast<const float2*>(state_of(k) + S::kState) + row).x);
      float4 acc = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
#pragma unroll 4
      for (int k = 0; k < ctas[s]; ++k) {
        const float2 ml = __ldcg(reinterpret_cast<const float2*>(state_of(k) + S::kState) + row);
        const float4 v = __ldcg(reinterpret_cast<const float4*>(state_of(k) + row * D) + d4);
        const float f = weights(M, ml.x);
        lsum += f * ml.y;
        acc.x += f * v.x; acc.y += f * v.y; acc.z += f * v.z; acc.w += f * v.w;
      }
      finish(open[s], row, d4, acc, lsum);
    }
  }
}

// ---------------------------------------------------------------------------
static bool a16(const void* p) { return (reinterpret_cast<uintptr_t>(p) & 15u) == 0; }

constexpr int kMaxQueries = 64;   // query tokens of a sequence
static bool shape_ok(int B, int Q, int Hq, int Hkv, int D) {
  return B >= 1 && B <= 65535 && Q >= 1 && Q <= kMaxQueries && Hkv >= 1 && Hq >= Hkv && Hq % Hkv == 0 &&
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
static int max_ctas(int rt, int sms) { return sms * (rt == 1 ? Shape<128, 1>::kCtas : Shape<128, 2>::kCtas); }

static std::once_flag g_encode_once;
static PFN_cuTensorMapEncodeTiled_v12000 g_encode = nullptr;

// A pool's codes as a matrix of D-byte rows; one box = a tile's 16 rows, swizzled
// over the row's length.
static bool pool_map(CUtensorMap* map, const void* codes, long long rows, int D) {
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
  const cuuint32_t box[2] = {(cuuint32_t)D, (cuuint32_t)kTile};
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
  return ANVILQ_WORKSPACE_COUNTER_BYTES + (size_t)max_ctas(rt, sms) * 2 * (8 * rt) * (D + 2) * sizeof(float);
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
  if (flags & ~(unsigned)ANVILQ_GEMM_OVERLAP_PRIOR) return ANVILQ_EINVAL;
  if (!shape_ok(B, Q, Hq, Hkv, D) || page_tokens < kBlock || page_tokens % kBlock || max_pages < 1 || num_pages < 1 ||
      (long long)page_tokens * max_pages > (1LL << 30))
    return ANVILQ_ESHAPE;
  const long long rows = (long long)num_pages * page_tokens * Hkv;   // a TMA coordinate is an int
  if ((long long)num_pages * page_tokens > (1LL << 31) || rows > 0x7FFFFFFFLL) return ANVILQ_ESHAPE;
  if (!a16(q) || !a16(k_codes) || !a16(v_codes) || !a16(out) || !a16(workspace)) return ANVILQ_EALIGN;
  const int sms = sm_count();
  if (sms <= 0) return ANVILQ_ECUDA;
  if (!workspace || workspace_bytes < anvilq_gqa_decode_q8_workspace_size(B, Q, Hq, Hkv, D)) return ANVILQ_EWORKSPACE;
  const int rt = row_tiles(Q, Hq, Hkv), warps = rt == 1 ? Shape<128, 1>::kWarps : Shape<128, 2>::kWarps;
  Params p{};
  p.q = reinterpret_cast<const __half*>(q);
  p.k_scales = k_scales;
  p.v_scales = v_scales;
  p.page_table = page_table;
  p.seqlens = seqlens;
  p.out = reinterpret_cast<__half*>(out);
  p.tickets = static_cast<int*>(workspace);
  p.partials = reinterpret_cast<float*>(static_cast<char*>(workspace) + ANVILQ_WORKSPACE_COUNTER_BYTES);
  p.dev_err = dev_err;
  p.B = B; p.Q = Q; p.Hq = Hq; p.Hkv = Hkv;
  p.group = Hq / Hkv;
  p.row_groups = (Q * p.group + 8 * rt - 1) / (8 * rt);
  p.page_tokens = page_tokens; p.max_pages = max_pages; p.num_pages = num_pages;
  p.scale_log2 = (scale > 0.0f ? scale : 1.0f / std::sqrt((float)D)) * 1.4426950408889634f;
  // as many CTAs as the device holds, but no more warps than the table has room for tiles
  const double tiles = (double)B * Hkv * p.row_groups * max_pages * (page_tokens / kTile);
  const int ctas = (int)std::max(1.0, std::min((double)max_ctas(rt, sms), std::ceil(tiles / warps)));
  if (tiles / ((double)ctas * warps) > (double)(1 << 30)) return ANVILQ_ESHAPE;   // a warp counts its tiles in an int
  CUtensorMap mk, mv;
  if (!pool_map(&mk, k_codes, rows, D) || !pool_map(&mv, v_codes, rows, D)) return ANVILQ_EALIGN;
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
