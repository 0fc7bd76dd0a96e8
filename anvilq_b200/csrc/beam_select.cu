// beam_select.cu -- a beam search's step: the best N continuations of an item's K
// beams over the vocabulary, and the reordering of per-beam rows by their parents.
//
// Mathematics.  For a beam k with score S_k and logits l_kv,
//   lse_k = log sum_v exp(l_kv),   s_kv = S_k + (l_kv - lse_k),
//   rank  = s_kv / (length_k + 1)^alpha.
// An ended beam has one candidate, its own score with rank S_k / max(length_k, 1)^alpha,
// at its first place.  The N candidates of the largest ranks win, ties by the lowest
// place k V + v.
//
// Within a beam the order is that of the logits, which is exact; across beams it hangs
// on the lse.  The exponent of exp2((l - c) log2 e) is formed from a difference and a product
// in two parts, a thread's partial sums are short, and everything from a span's sum on is
// binary64.  The lse is off by at most
//   3 2^-22 (ex2.approx, of a logit to its thread's largest, that to the span's, that to the row's)
//   + 2^-23 d (their exponents' two roundings; d: the logits' mean distance to the row's largest,
//     weighted by their exponentials) + 32 2^-24 (a tile's additions of a thread)
//   + V / 4096 (2^-22 + 2 2^-24) (for each of a thread's tiles its addition, and the sum taken
//     to a new largest, if every tile has one),
// below 3e-6 + 2^-23 d + 4e-7 V / 4096.  Random logits' sums were 2e-8 off.  Candidates of
// different beams whose scores are closer than that may come in either order.
//
// What bounds it: the logits are read once (HBM), 13 instructions a fp16 logit, 27 a fp32 one
// in spans of 7 tiles a warp, whose beginning and end count.  A small call is bound by
// latency: load, threshold, merge.
//
// Work split.  A CTA takes a span of a beam's vocabulary (splits so that the device is
// full, splits_for), its warps tiles of 32 x 4 x 16 bytes in turn, without a barrier: a
// warp adds a tile up, and looks for candidates only where a 16-byte unit's largest beats
// the span's bar.  Where every warp has N / warps keys, there are N: the first tiles' lanes
// set it so, lists that fill raise it, for all warps of the CTA.  Of random logits few beat it (N log of the span over
// the tile in all).  The span's sum and N best go to the workspace, and the item's last
// CTA (by a ticket) merges them.
//
// Measured: 48 x 8 beams over 151936 fp16 logits, some masked, some beams ended, 60 us (1.9
// TB/s: a tile's dependent instructions at 21 warps an SM, issue slots 30 % busy; 8 us of a
// CTA's beginning and end); 100 x 5 over 32000 fp32 logits, N = 10, 35 us; one item's 4 beams
// over 151936 17 us with the reordering.  Rows off 16 bytes are loaded logit by logit: 48 x 8 over
// 50257 fp16 logits 40.5 us, over 50256 30.2; fp32 66 and 35.
#include <algorithm>
#include <climits>
#include <cmath>

#include "kv_q8.cuh"

namespace anvilq {
namespace beam {

using q8::overlap;
constexpr int kThreads = 256;
constexpr int kWarps = kThreads / 32;
constexpr int kMaxBeams = 64, kMaxBest = 128;   // K, N
constexpr int kMaxItems = 4096;
constexpr int kUnits = 4;                       // 16-byte units of a thread in a tile
constexpr int kKeys = 1536;                     // of the merge in shared memory, at most
constexpr int kWarpList = 192;                  // a warp's
constexpr int kPending = 160;                   // units a warp has put off, at most
constexpr int kMaxSplits = 64;
constexpr int kResident = 4;                    // CTAs an SM
constexpr float kLog2e = 1.44269504f, kLog2eLow = 1.92596299e-8f;   // log2 e in two parts

struct Params {
  const void* logits;        // [B K] rows of V, `stride` elements apart
  long long stride;
  const float* scores;       // [B][K]
  const int* lengths;        // [B][K], null: no length penalty, no lengths out
  const uint8_t* finished;   // [B][K], null: none
  const int* eos;            // [eos_count]
  int* tokens;               // [B][N]
  int* parents;
  float* new_scores;
  int* new_lengths;          // null where lengths is
  uint8_t* new_finished;
  int* tickets;              // [B]
  double* scales;            // [B][K]: the ranks' divisors
  double2* sums;             // [B][K][splits]: the largest logit, sum of exp(logit - it)
  unsigned long long* best;  // [B][K][splits][N]: keys, best first
  int* dev_err;
  float alpha;
  int B, K, V, N, splits, eos_count, pad;
};

__device__ __forceinline__ float fast_exp2(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}

// A logit and its place as one number that grows with the logit and, among equals,
// with smaller places; 0 is below every logit but those of -inf, which get 0 too.
__device__ __forceinline__ unsigned long long key_of(float v, int at) {
  const uint32_t u = __float_as_uint(v + 0.0f);   // -0 as +0
  const uint32_t order = (u >> 31) ? ~u : u | 0x80000000u;
  return v == -INFINITY ? 0 : ((unsigned long long)order << 32) | (0xFFFFFFFFu - (uint32_t)at);
}
__device__ __forceinline__ float logit_of(unsigned long long key) {
  const uint32_t order = (uint32_t)(key >> 32);
  return __uint_as_float((order >> 31) ? order & 0x7FFFFFFFu : ~order);
}
__device__ __forceinline__ int place_of(unsigned long long key) { return (int)(0xFFFFFFFFu - (uint32_t)key); }

// A beam that goes on or has ended; scores of NaN and +inf are reported and count as none.
__device__ __forceinline__ bool is_live(float score) { return score > -INFINITY && score < INFINITY; }

// A span's candidates: a list a warp, and what any of them has to beat.
struct List {
  unsigned long long key[kWarps][kWarpList];
  unsigned long long all[kWarps * kMaxBest];
  unsigned long long bar;   // at least N keys of the span are above it, or it is the N-th
  int pending[kWarps][kPending];   // units that may hold candidates
  uint32_t share[kWarps];   // the warp has its share of N keys, N / warps, of this order or above
  int count[kWarps];
};
// What a key has to be above: the bar, or what all warps have their shares of.
__device__ __forceinline__ unsigned long long bar_of(const List& s, int warps) {
  const int lane = threadIdx.x % 32;
  const uint32_t mine = lane < warps ? *reinterpret_cast<const volatile uint32_t*>(&s.share[lane]) : 0xFFFFFFFFu;
  const unsigned long long all = (unsigned long long)__reduce_min_sync(0xffffffffu, mine) << 32;
  const unsigned long long bar = *reinterpret_cast<const volatile unsigned long long*>(&s.bar);
  return all > bar ? all : bar;
}

// The n keys' best N, best first, in `to`: every thread of the group (thread `me` of
// `threads`) calls it, all keys differ.
__device__ __forceinline__ void best_of(const unsigned long long* key, int n, unsigned long long* to, int N, int me,
                                        int threads) {
  for (int i = me; i < n; i += threads) {
    const unsigned long long mine = key[i];
    int above = 0;
    for (int j = 0; j < n; ++j) above += key[j] > mine;
    if (above < N) to[above] = mine;
  }
}

// The lanes' values in descending order, by exchanges (Batcher's bitonic network).
__device__ __forceinline__ float sorted(float v) {
  const int lane = threadIdx.x % 32;
#pragma unroll
  for (int size = 2; size <= 32; size *= 2)
#pragma unroll
    for (int o = size / 2; o > 0; o /= 2) {
      const float other = __shfl_xor_sync(0xffffffffu, v, o);
      const bool larger = ((lane & o) == 0) == ((lane & size) == 0);   // this lane keeps the larger one
      v = larger ? fmaxf(v, other) : fminf(v, other);
    }
  return v;
}

// A binary64 number as one that compares alike; 0 stays free for "none".
__device__ __forceinline__ unsigned long long order_of(double r) {
  const unsigned long long u = (unsigned long long)__double_as_longlong(r + 0.0);   // -0 as +0
  return (u >> 63) ? ~u : u | 1ull << 63;
}
struct Merge {
  double score[kMaxBeams];
  double top[kMaxBeams];      // lse = top + log_sum: kept apart, as a logit minus top is exact however
  double log_sum[kMaxBeams];  // large both are
  double scale[kMaxBeams];    // the rank's divisor
  int ended[kMaxBeams];
  unsigned long long key[kKeys];    // the spans' lists, where they fit
  unsigned long long best[kKeys];   // [K][N]: the beams' lists, where they fit
  unsigned long long rank[kKeys];   // their ranks' orders
  int taken[kMaxBest];              // beam, candidate of it
};

// The largest of the lanes' numbers and the lowest lane that has it; -1 where all are 0.
__device__ __forceinline__ int largest_lane(unsigned long long v) {
  const uint32_t high = (uint32_t)(v >> 32), top = __reduce_max_sync(0xffffffffu, high);
  const uint32_t low = high == top ? (uint32_t)v : 0u, rest = __reduce_max_sync(0xffffffffu, low);
  const uint32_t who = __ballot_sync(0xffffffffu, high == top && low == rest);
  return top | rest ? __ffs(who) - 1 : -1;
}

// The largest, or NaN where one of them is (fmaxf would pass it over).
__device__ __forceinline__ float max_or_nan(float a, float b) {
  float d;
  asm("max.NaN.f32 %0, %1, %2;" : "=f"(d) : "f"(a), "f"(b));
  return d;
}
__device__ __forceinline__ float max_or_nan(float a, float b, float c) {
  float d;
  asm("max.NaN.f32 %0, %1, %2, %3;" : "=f"(d) : "f"(a), "f"(b), "f"(c));
  return d;
}
// two binary32 values at a time
using u64 = unsigned long long;
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
__device__ __forceinline__ u64 mul2(u64 a, u64 b) {
  u64 d;
  asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(d) : "l"(a), "l"(b));
  return d;
}
__device__ __forceinline__ u64 add2(u64 a, u64 b) {
  u64 d;
  asm("add.rn.f32x2 %0, %1, %2;" : "=l"(d) : "l"(a), "l"(b));
  return d;
}

__device__ __forceinline__ void widen(const uint4& w, float* v, __half) {
  const __half2* h = reinterpret_cast<const __half2*>(&w);
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const float2 f = __half22float2(h[i]);
    v[2 * i] = f.x;
    v[2 * i + 1] = f.y;
  }
}
__device__ __forceinline__ void widen(const uint4& w, float* v, float) {
  v[0] = __uint_as_float(w.x); v[1] = __uint_as_float(w.y);
  v[2] = __uint_as_float(w.z); v[3] = __uint_as_float(w.w);
}
// What seldom runs is kept out of the loops, whose instructions would not fit the
// instruction cache (beam batch 148 us with all of it unrolled in place).

// 16 bytes of a row, of which `n` values are in it (all where it holds a whole unit); the
// others are -inf.
template <typename T>
__device__ __noinline__ uint4 load_odd_unit(const T* p, int n) {
  uint4 w;
  uint32_t* o = &w.x;
#pragma unroll 1
  for (int i = 0; i < 4; ++i) {
    if (sizeof(T) == 4) {
      o[i] = i < n ? __ldg(reinterpret_cast<const uint32_t*>(p) + i) : 0xFF800000u;
    } else {
      const unsigned short* q = reinterpret_cast<const unsigned short*>(p);
      const uint32_t a = 2 * i < n ? __ldg(q + 2 * i) : 0xFC00u, b = 2 * i + 1 < n ? __ldg(q + 2 * i + 1) : 0xFC00u;
      o[i] = a | b << 16;
    }
  }
  return w;
}

// A warp's list cut to its N best, of which `share` are its share; returns their number.
__device__ __noinline__ int cut_list(List& s, int count, int N, int share) {
  const int warp = threadIdx.x / 32, lane = threadIdx.x % 32;
  unsigned long long *mine = s.key[warp], *room = s.all + warp * kMaxBest;
  __syncwarp();
  best_of(mine, count, room, N, lane, 32);
  __syncwarp();
  const int left = min(count, N);
  for (int i = lane; i < left; i += 32) mine[i] = room[i];
  if (lane == 0) {
    if (count >= N) atomicMax(&s.bar, room[N - 1]);
    if (count >= share) s.share[warp] = max(s.share[warp], (uint32_t)(room[share - 1] >> 32));
  }
  __syncwarp();
  return left;
}

// The candidates of a warp's pending units, appended to its list, whose new length is
// returned.  A lane takes a unit and reads it again.
template <typename T>
__device__ __noinline__ int scan_pending(List& s, const T* x, bool aligned, int pending, int V, int count, int N,
                                         int warps, int share) {
  constexpr int kVec = 16 / sizeof(T);
  const int warp = threadIdx.x / 32, lane = threadIdx.x % 32;
  unsigned long long* mine = s.key[warp];
  __syncwarp();
#pragma unroll 1
  for (int i = 0; i < pending; i += 32) {
    const bool some = i + lane < pending;
    const int at = some ? s.pending[warp][i + lane] * kVec : 0, n = some ? V - at : 0;
    const uint4 w = aligned && n >= kVec ? *reinterpret_cast<const uint4*>(x + at) : load_odd_unit(x + at, n);
    float v[kVec];
    widen(w, v, T());
    const unsigned long long bar = bar_of(s, warps);
#pragma unroll
    for (int e = 0; e < kVec; ++e) {
      const unsigned long long key = v[e] < INFINITY ? key_of(v[e], at + e) : 0;   // 0, of -inf too: none
      const uint32_t hits = __ballot_sync(0xffffffffu, key > bar);
      if (hits >> lane & 1) mine[count + __popc(hits & ((1u << lane) - 1))] = key;
      count += __popc(hits);
      if (count > kWarpList - 32) count = cut_list(s, count, N, share);
    }
  }
  __syncwarp();
  return count;
}

// The divisor of a beam's ranks, for the merge: a power in binary64 takes 2 us, here beside
// other threads' work.
__device__ __noinline__ void write_divisor(const Params& p, int row) {
  const int length = p.lengths ? max(p.lengths[row], 0) : 0;
  const double steps = p.finished && p.finished[row] ? (double)max(length, 1) : (double)length + 1.0;
  __stcg(p.scales + row, p.alpha == 0.0f ? 1.0 : p.alpha == 1.0f ? steps : pow(steps, (double)p.alpha));
  if (!(p.scores[row] < INFINITY)) atomicOr(p.dev_err, ANVILQ_DEV_ERR_NONFINITE);
}

template <typename T>
__device__ void span_pass(const Params& p, List& s, int row, int split) {
  constexpr int kVec = 16 / sizeof(T), kEach = kUnits * kVec;
  const int tid = threadIdx.x;
  const T* x = static_cast<const T*>(p.logits) + (long long)row * p.stride;
  // Units of kVec places, wherever the row starts: two equal rows give equal sums, so
  // that their candidates tie.
  const int units = (p.V + kVec - 1) / kVec;
  const bool aligned = reinterpret_cast<uintptr_t>(x) % 16 == 0;
  const int u0 = (int)((long long)units * split / p.splits), u1 = (int)((long long)units * (split + 1) / p.splits);
  const int warp = tid / 32, lane = tid % 32;
  // the warps that have a tile, and of each the keys that make N in all
  const int warps = min(kWarps, (u1 - u0 + 31) / 32), share = (p.N + warps - 1) / warps;
  if (tid == 0) s.bar = 0;
  if (tid < kWarps) s.share[tid] = 0;
  __syncthreads();
  int count = 0, pending = 0;         // of the warp's lists
  float c = -INFINITY, sum = 0.0f;    // sum of exp2(log2 e (l - c)), c the thread's largest
  bool odd = false;                   // a logit of +inf or NaN was left out
  bool begun = false;
  auto sync_warps = [&]() { asm volatile("bar.sync 1, %0;" ::"r"(32 * warps) : "memory"); };   // that have a tile
  const bool more = u1 - u0 > 3 * kThreads * kUnits;
  for (int t0 = u0 + warp * 32; t0 < u1; t0 += kThreads * kUnits) {
    float v[kEach], tops[kUnits];     // tops: of the units
    {
      uint4 raw[kUnits];
      const int end = t0 + (kUnits - 1) * kThreads + 32;   // of the tile's units
      if (aligned && end <= u1 && end <= p.V / kVec) {     // the same for all lanes
#pragma unroll
        for (int i = 0; i < kUnits; ++i)
          raw[i] = __ldcs(reinterpret_cast<const uint4*>(x) + (t0 + i * kThreads + lane));
      } else {
#pragma unroll
        for (int i = 0; i < kUnits; ++i) {
          const int u = t0 + i * kThreads + lane, n = u < u1 ? p.V - u * kVec : 0;
          raw[i] = load_odd_unit(x + (n > 0 ? u * kVec : 0), n);
        }
      }
#pragma unroll
      for (int i = 0; i < kUnits; ++i) widen(raw[i], v + i * kVec, T());
    }
    const float c_was = c, sum_was = sum;
    float top;
#pragma unroll 1
    for (bool again = false;; again = true) {
#pragma unroll
      for (int i = 0; i < kUnits; ++i) {
        float a = max_or_nan(v[i * kVec], v[i * kVec + 1]);
#pragma unroll
        for (int e = 2; e < kVec; e += 2) a = max_or_nan(a, v[i * kVec + e], v[i * kVec + e + 1]);
        tops[i] = a;
      }
      top = tops[0];
#pragma unroll
      for (int i = 1; i < kUnits; ++i) top = max_or_nan(top, tops[i]);
      // the tile's sum relative to the largest so far
      const float now = fmaxf(c, top);   // c where top is NaN: the tile is then taken again
      float part = 0.0f;
      if (now != -INFINITY) {
        if (now > c) {
          const float d = c - now;
          sum *= c == -INFINITY ? 0.0f : fast_exp2(fmaf(d, kLog2e, d * kLog2eLow));
          c = now;
        }
        const u64 minus = pair(-c, -c), high = pair(kLog2e, kLog2e), low = pair(kLog2eLow, kLog2eLow);
        u64 parts[2] = {0, 0};
#pragma unroll
        for (int i = 0; i < kEach; i += 2) {
          const u64 d = add2(pair(v[i], v[i + 1]), minus);
          const float2 e = unpair(fma2(d, high, mul2(d, low)));
          parts[i / 2 % 2] = add2(parts[i / 2 % 2], pair(fast_exp2(e.x), fast_exp2(e.y)));
        }
        const float2 a = unpair(add2(parts[0], parts[1]));
        part = a.x + a.y;
      }
      if ((part < INFINITY && top == top) || again) {
        sum += part;
        break;
      }
      // +inf (the sum is then no number) or NaN among them: they count as -inf, and are reported
      odd = true;
      c = c_was;
      sum = sum_was;
#pragma unroll
      for (int i = 0; i < kEach; ++i)
        if (!(v[i] < INFINITY)) v[i] = -INFINITY;
    }
    // ---- candidates ----
    const bool first = !begun;
    if (first) {
      // the lanes' largest bound the warp's share, and its N-th, from below
      const float order = sorted(top), a = __shfl_sync(0xffffffffu, order, share - 1),
                  b = __shfl_sync(0xffffffffu, order, min(p.N, 32) - 1);
      if (lane == 0) {
        if (share <= 32) s.share[warp] = (uint32_t)(key_of(a, 0) >> 32);   // else there are too few lanes to tell
        if (p.N <= 32 && b > -INFINITY) atomicMax(&s.bar, key_of(b, 0) & ~0xFFFFFFFFull);
      }
      sync_warps();
      begun = true;
    }
    const unsigned long long bar = bar_of(s, warps);
    const float least = bar ? logit_of(bar) : -INFINITY;
    if (!first && !__any_sync(0xffffffffu, top >= least && top > -INFINITY)) continue;
    // units that may hold candidates are put off: looking at each at once took 20 us of 67
#pragma unroll
    for (int i = 0; i < kUnits; ++i) {
      const bool hit = tops[i] >= least && tops[i] > -INFINITY;
      const uint32_t hits = __ballot_sync(0xffffffffu, hit);
      if (hit) s.pending[warp][pending + __popc(hits & ((1u << lane) - 1))] = t0 + i * kThreads + lane;
      pending += __popc(hits);
    }
    if (first || pending > kPending - 32 * kUnits) {
      count = scan_pending(s, x, aligned, pending, p.V, count, p.N, warps, share);
      if (!first && count > p.N) count = cut_list(s, count, p.N, share);   // it raises the bar
      pending = 0;
    }
    // The N-th of all that the first tiles gave: few later logits beat it, where the bar so
    // far lets through several a tile (48 x 8 beams 67 us without it).
    if (first && more) {
      if (count > p.N) count = cut_list(s, count, p.N, share);
      if (lane == 0) s.count[warp] = count;
      sync_warps();
      int total = 0, before = 0;
      for (int w = 0; w < warps; ++w) {
        if (w < warp) before += s.count[w];
        total += s.count[w];
      }
      for (int i = lane; i < count; i += 32) s.all[before + i] = s.key[warp][i];
      sync_warps();
      for (int i = tid; i < total; i += 32 * warps) {
        const unsigned long long key = s.all[i];
        int above = 0;
        for (int j = 0; j < total; ++j) above += s.all[j] > key;
        if (above == p.N - 1) atomicMax(&s.bar, key);
      }
      sync_warps();   // (the room is used again)
    }
  }
  if (pending) count = scan_pending(s, x, aligned, pending, p.V, count, p.N, warps, share);
  if (count > p.N) count = cut_list(s, count, p.N, share);
  if (lane == 0) s.count[warp] = count;
  // ---- the span's sum, in binary64 from the threads' on, and its N best ----
  __shared__ float tops[kWarps];
  __shared__ double parts[kWarps];
  float top = c;
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, o));
  if (lane == 0) tops[warp] = top;
  __syncthreads();
  top = tops[0];
  int total = 0, before = 0;
#pragma unroll
  for (int w = 0; w < kWarps; ++w) {
    top = fmaxf(top, tops[w]);
    if (w < warp) before += s.count[w];
    total += s.count[w];
  }
  double term = 0.0;
  if (c > -INFINITY) {
    const float d = c - top;
    term = (double)(sum * fast_exp2(fmaf(d, kLog2e, d * kLog2eLow)));
  }
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) term += __shfl_xor_sync(0xffffffffu, term, o);
  if (lane == 0) parts[warp] = term;
  if (odd) atomicOr(p.dev_err, ANVILQ_DEV_ERR_NONFINITE);
  for (int i = lane; i < count; i += 32) s.all[before + i] = s.key[warp][i];
  __syncthreads();
  const size_t at = (size_t)row * p.splits + split;
  if (tid == 0) {
    double all = 0.0;
    for (int w = 0; w < kWarps; ++w) all += parts[w];
    __stcg(p.sums + at, make_double2(top, all));
  }
  if (split == 0 && tid == kThreads - 1) write_divisor(p, row);
  for (int i = tid; i < total; i += kThreads) {   // ranked among all
    const unsigned long long key = s.all[i];
    int above = 0;
    for (int j = 0; j < total; ++j) above += s.all[j] > key;
    if (above < p.N) __stcg(p.best + at * p.N + above, key);
  }
  for (int i = total + tid; i < p.N; i += kThreads) __stcg(p.best + at * p.N + i, 0ull);
}

template <typename T>
__global__ void __launch_bounds__(kThreads, kResident) beam_kernel(const __grid_constant__ Params p) {
  extern __shared__ __align__(16) unsigned char room[];   // a List, then a Merge
  asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
  asm volatile("griddepcontrol.wait;" ::: "memory");
  const int tid = threadIdx.x, split = blockIdx.x, row = blockIdx.y, b = row / p.K;
  // a beam that is dead or ended has no logits to be read
  const bool live = is_live(p.scores[row]) && !(p.finished && p.finished[row]);
  if (!live && split == 0 && tid == kThreads - 1) write_divisor(p, row);
  if (live) span_pass<T>(p, *reinterpret_cast<List*>(room), row, split);
  // ---- the item's last CTA goes on ----
  __shared__ int last;
  __syncthreads();   // the thread that takes the ticket releases, and acquires, for all
  if (tid == 0) {
    int arrived;
    asm volatile("atom.acq_rel.gpu.global.add.s32 %0, [%1], 1;" : "=r"(arrived) : "l"(p.tickets + b) : "memory");
    last = arrived == p.K * p.splits - 1;
    if (last) p.tickets[b] = 0;
  }
  __syncthreads();
  if (!last) return;
  Merge& m = *reinterpret_cast<Merge*>(room);
  const int warp = tid / 32, lane = tid % 32;
  const int per = p.splits * p.N;                                    // keys of a beam
  const bool keys_fit = p.K * per <= kKeys, best_fit = p.K * p.N <= kKeys;
  unsigned long long* spans = p.best + (size_t)b * p.K * per;
  if (keys_fit)
    for (int i = tid; i < p.K * per; i += kThreads) m.key[i] = __ldcg(spans + i);
  __syncthreads();
  // ---- a beam a warp: its sum, and its N best, the heads of its spans' lists compared ----
  for (int k = warp; k < p.K; k += kWarps) {
    const int r = b * p.K + k;
    const float score = p.scores[r];
    const bool ended = p.finished && p.finished[r];
    unsigned long long* to = best_fit ? m.best + k * p.N : spans + (size_t)k * per;   // (in place: see below)
    if (lane == 0) {
      m.score[k] = score;
      m.scale[k] = __ldcg(p.scales + r);
      m.ended[k] = ended;
    }
    int found = 0;
    if (is_live(score) && ended) {
      if (lane == 0) to[0] = 1;   // any key will do
      found = 1;
    } else if (is_live(score)) {
      static_assert(kMaxSplits <= 64, "two spans a lane");
      const double2 none = make_double2(-INFINITY, 0.0);
      const double2* at = p.sums + (size_t)r * p.splits;
      const double2 one = lane < p.splits ? __ldcg(at + lane) : none;
      const double2 two = lane + 32 < p.splits ? __ldcg(at + lane + 32) : none;
      double top = fmax(one.x, two.x);
#pragma unroll
      for (int o = 16; o > 0; o >>= 1) top = fmax(top, __shfl_xor_sync(0xffffffffu, top, o));
      // (binary32 exponents of binary32 differences, as in a span)
      auto part = [&](double2 v) {
        const float d = (float)(v.x - top);
        return v.y > 0.0 ? v.y * (double)fast_exp2(fmaf(d, kLog2e, d * kLog2eLow)) : 0.0;
      };
      double all = part(one) + part(two);
#pragma unroll
      for (int o = 16; o > 0; o >>= 1) all += __shfl_xor_sync(0xffffffffu, all, o);
      if (lane == 0) {
        m.top[k] = top;           // of a beam without candidates: not used
        m.log_sum[k] = log(all);
      }
      auto key_at = [&](int span, int i) {
        if (span >= p.splits || i >= p.N) return 0ull;
        return keys_fit ? m.key[k * per + span * p.N + i] : __ldcg(spans + (size_t)k * per + span * p.N + i);
      };
      if (p.splits == 1) {
        if (best_fit)   // else it is there
          for (int i = lane; i < p.N; i += 32) to[i] = key_at(0, i);
        found = p.N;
      } else {
        // Keys differ, so a head is at one lane only.  The list grows in registers' place:
        // results go out behind the loop where they would overwrite lists still to be read.
        int i0 = 0, i1 = 0;
        unsigned long long h0 = key_at(lane, 0), h1 = key_at(lane + 32, 0), kept[kMaxBest / 32];
#pragma unroll
        for (int q = 0; q < kMaxBest / 32; ++q) kept[q] = 0;
        for (; found < p.N; ++found) {
          const unsigned long long mine = h0 > h1 ? h0 : h1;
          const int l = largest_lane(mine);
          if (l < 0) break;
          const unsigned long long best = __shfl_sync(0xffffffffu, mine, l);
#pragma unroll
          for (int q = 0; q < kMaxBest / 32; ++q)
            if (found == 32 * q + lane) kept[q] = best;
          if (lane == l) {
            if (h0 > h1) h0 = key_at(lane, ++i0);
            else h1 = key_at(lane + 32, ++i1);
          }
        }
        __syncwarp();
#pragma unroll
        for (int q = 0; q < kMaxBest / 32; ++q)
          if (32 * q + lane < found) to[32 * q + lane] = kept[q];
      }
    }
    __syncwarp();
    for (int i = found + lane; i < p.N; i += 32) to[i] = 0;
  }
  __syncthreads();
  // ---- ranks, and the N best of all ----
  auto key_of_beam = [&](int k, int i) {
    return best_fit ? m.best[k * p.N + i] : *reinterpret_cast<volatile unsigned long long*>(spans + (size_t)k * per + i);
  };
  auto score_of = [&](int k, unsigned long long key) {
    return m.ended[k] ? m.score[k] : m.score[k] + (((double)logit_of(key) - m.top[k]) - m.log_sum[k]);
  };
  auto order_at = [&](int k, int i) {   // 0: no candidate, or one of a rank that is none
    const unsigned long long key = key_of_beam(k, i);
    if (!key) return 0ull;
    const double rank = score_of(k, key) / m.scale[k];
    return rank > -INFINITY ? order_of(rank) : 0ull;
  };
  if (best_fit)
    for (int i = tid; i < p.K * p.N; i += kThreads) m.rank[i] = order_at(i / p.N, i % p.N);
  __syncthreads();
  __shared__ int chosen;
  if (warp == 0) {
    static_assert(kMaxBeams <= 64, "two beams a lane");
    // lane l has beams 2 l and 2 l + 1: of equal ranks the lowest lane's lower beam is first
    auto head = [&](int k, int i) {
      if (k >= p.K || i >= p.N) return 0ull;
      return best_fit ? m.rank[k * p.N + i] : order_at(k, i);
    };
    int i0 = 0, i1 = 0, n = 0;
    unsigned long long h0 = head(2 * lane, 0), h1 = head(2 * lane + 1, 0);
    for (; n < p.N; ++n) {
      const int l = largest_lane(h0 >= h1 ? h0 : h1);
      if (l < 0) break;
      if (lane == l) {
        if (h0 >= h1) {
          m.taken[n] = 2 * lane << 16 | i0;
          h0 = head(2 * lane, ++i0);
        } else {
          m.taken[n] = (2 * lane + 1) << 16 | i1;
          h1 = head(2 * lane + 1, ++i1);
        }
      }
    }
    if (lane == 0) chosen = n;
  }
  __syncthreads();
  for (int i = tid; i < p.N; i += kThreads) {
    const int at = b * p.N + i;
    if (i >= chosen) {
      p.tokens[at] = p.parents[at] = -1;
      p.new_scores[at] = -INFINITY;
      p.new_finished[at] = 1;
      if (p.new_lengths) p.new_lengths[at] = 0;
      continue;
    }
    const int k = m.taken[i] >> 16;
    const unsigned long long key = key_of_beam(k, m.taken[i] & 0xffff);
    const bool ended = m.ended[k];
    const int token = ended ? p.pad : place_of(key);
    bool over = ended;
    for (int e = 0; e < p.eos_count; ++e) over |= p.eos[e] == token;
    p.tokens[at] = token;
    p.parents[at] = k;
    p.new_scores[at] = (float)score_of(k, key);
    p.new_finished[at] = over;
    if (p.new_lengths) p.new_lengths[at] = ended ? max(p.lengths[b * p.K + k], 0) : min(max(p.lengths[b * p.K + k], 0), INT_MAX - 1) + 1;
  }
}

// ---- rows by their parents ---------------------------------------------------------

constexpr int kMaxStates = 32;
struct State {
  const char* in;
  char* out;
  long long row_bytes;
};
struct Reorder {
  const int* parents;   // [B][N]
  int* dev_err;
  int B, K, N, states;
  State state[kMaxStates];
};

template <typename W>
__device__ __forceinline__ void move_row(const char* from, char* to, long long bytes) {
  constexpr int kAhead = 4;
  const long long n = bytes / (long long)sizeof(W), step = (long long)gridDim.x * kThreads;
  for (long long i0 = (long long)blockIdx.x * kThreads + threadIdx.x; i0 < n; i0 += kAhead * step) {
    W w[kAhead];
#pragma unroll
    for (int a = 0; a < kAhead; ++a) {
      w[a] = W{};
      if (from && i0 + a * step < n) w[a] = reinterpret_cast<const W*>(from)[i0 + a * step];
    }
#pragma unroll
    for (int a = 0; a < kAhead; ++a)
      if (i0 + a * step < n) reinterpret_cast<W*>(to)[i0 + a * step] = w[a];
  }
}

__global__ void __launch_bounds__(kThreads) reorder_kernel(const __grid_constant__ Reorder p) {
  asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
  asm volatile("griddepcontrol.wait;" ::: "memory");
  const State& s = p.state[blockIdx.z];
  for (int row = blockIdx.y; row < p.B * p.N; row += gridDim.y) {
    int parent = p.parents[row];
    if (parent < -1 || parent >= p.K) {
      if (threadIdx.x == 0) atomicOr(p.dev_err, ANVILQ_DEV_ERR_SEQLEN);
      parent = -1;
    }
    const char* from = parent < 0 ? nullptr : s.in + ((long long)(row / p.N) * p.K + parent) * s.row_bytes;
    char* to = s.out + (long long)row * s.row_bytes;
    const uintptr_t all = reinterpret_cast<uintptr_t>(s.in) | reinterpret_cast<uintptr_t>(s.out) | s.row_bytes;
    if (all % 16 == 0) move_row<uint4>(from, to, s.row_bytes);
    else if (all % 4 == 0) move_row<uint32_t>(from, to, s.row_bytes);
    else move_row<uint8_t>(from, to, s.row_bytes);
  }
}

template <typename P>
static int launch(void (*kernel)(P), dim3 grid, size_t smem, cudaStream_t s, unsigned flags, const P& p) {
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = grid;
  cfg.blockDim = dim3(kThreads);
  cfg.dynamicSmemBytes = smem;
  cfg.stream = s;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = attr;
  cfg.numAttrs = (flags & ANVILQ_GEMM_OVERLAP_PRIOR) ? 1 : 0;
  if (cudaLaunchKernelEx(&cfg, kernel, p) != cudaSuccess) {
    cudaGetLastError();
    return ANVILQ_ECUDA;
  }
  return ANVILQ_OK;
}

static bool shape_ok(int B, int K, int V, int N) {
  return B >= 1 && B <= kMaxItems && K >= 1 && K <= kMaxBeams && N >= 1 && N <= kMaxBest && V >= 1 && V <= (1 << 30) &&
         B * K <= 65535;
}
// Spans of a row: the number of least cost, in waves of resident CTAs, of a span's logits
// and what it costs besides.  (8 us: as much as 60000 logits, so that a second wave seldom
// pays.  48 x 8 rows of 151936 fp16 logits as one span 58.6 us, as three 60.7; 64 rows as
// nine 22.9, as two 26.3.)
static int splits_for(int B, int K, int V) {
  const long long rows = (long long)B * K, resident = 148 * kResident;
  int best = 1;
  long long least = 0;
  for (int s = 1; s <= kMaxSplits && (s == 1 || V / s >= 2048); ++s) {
    const long long cost = (rows * s + resident - 1) / resident * (V / s + 60000);
    if (s == 1 || cost < least) {
      least = cost;
      best = s;
    }
  }
  return best;
}

}  // namespace beam
}  // namespace anvilq

extern "C" {

size_t anvilq_beam_select_workspace_size(int B, int K, int V, int N) {
  using namespace anvilq::beam;
  if (!shape_ok(B, K, V, N)) return 0;
  const size_t spans = (size_t)B * K * splits_for(B, K, V);
  return ANVILQ_WORKSPACE_COUNTER_BYTES + spans * (sizeof(double2) + (size_t)N * 8) + (size_t)B * K * sizeof(double);
}

int anvilq_beam_select(const void* logits, int logits_half, long long logits_stride, const float* scores,
                       const int32_t* lengths, float length_penalty, const uint8_t* finished, const int32_t* eos_ids,
                       int eos_count, int pad_id, int32_t* tokens, int32_t* parents, float* new_scores,
                       int32_t* new_lengths, uint8_t* new_finished, int B, int K, int V, int N, void* workspace,
                       size_t workspace_bytes, int* dev_err, unsigned flags, anvilq_stream_t stream) {
  using namespace anvilq;
  using namespace anvilq::beam;
  if (!logits || !scores || !tokens || !parents || !new_scores || !new_finished || !dev_err) return ANVILQ_EINVAL;
  if ((logits_half != 0 && logits_half != 1) || eos_count < 0 || (eos_count && !eos_ids)) return ANVILQ_EINVAL;
  if ((lengths == nullptr) != (new_lengths == nullptr) || (!lengths && length_penalty != 0.0f)) return ANVILQ_EINVAL;
  if (!(std::fabs(length_penalty) <= 16.0f)) return ANVILQ_EINVAL;
  if (flags & ~(unsigned)ANVILQ_GEMM_OVERLAP_PRIOR) return ANVILQ_EINVAL;
  if (!shape_ok(B, K, V, N) || eos_count > 1024) return ANVILQ_ESHAPE;
  if (logits_stride < V) return ANVILQ_EINVAL;
  const uintptr_t ints = reinterpret_cast<uintptr_t>(scores) | reinterpret_cast<uintptr_t>(lengths) |
                         reinterpret_cast<uintptr_t>(eos_ids) | reinterpret_cast<uintptr_t>(tokens) |
                         reinterpret_cast<uintptr_t>(parents) | reinterpret_cast<uintptr_t>(new_scores) |
                         reinterpret_cast<uintptr_t>(new_lengths);
  if (ints % 4 || reinterpret_cast<uintptr_t>(logits) % (logits_half ? 2 : 4) ||
      reinterpret_cast<uintptr_t>(workspace) % 16)
    return ANVILQ_EALIGN;
  // an item's results are written while other items are still to be read
  const size_t in = (size_t)B * K, out = (size_t)B * N;
  struct Span {
    const void* start;
    size_t bytes;
  };
  const Span reads[] = {{logits, ((in - 1) * (size_t)logits_stride + V) * (logits_half ? 2 : 4)}, {scores, in * 4},
                        {lengths, lengths ? in * 4 : 0}, {finished, finished ? in : 0}, {eos_ids, eos_count * 4u},
                        {workspace, workspace ? workspace_bytes : 0}};
  const Span writes[] = {{tokens, out * 4}, {parents, out * 4}, {new_scores, out * 4},
                         {new_lengths, new_lengths ? out * 4 : 0}, {new_finished, out}};
  for (int i = 0; i < 5; ++i) {
    for (const Span& r : reads)
      if (overlap(writes[i].start, writes[i].bytes, r.start, r.bytes)) return ANVILQ_EINVAL;
    for (int j = 0; j < i; ++j)
      if (overlap(writes[i].start, writes[i].bytes, writes[j].start, writes[j].bytes)) return ANVILQ_EINVAL;
    if (workspace && i < 4 && overlap(reads[i].start, reads[i].bytes, workspace, workspace_bytes)) return ANVILQ_EINVAL;
  }
  if (!workspace || workspace_bytes < anvilq_beam_select_workspace_size(B, K, V, N)) return ANVILQ_EWORKSPACE;
  Params p{};
  p.logits = logits;
  p.stride = logits_stride;
  p.scores = scores;
  p.lengths = lengths;
  p.finished = finished;
  p.eos = eos_ids;
  p.tokens = tokens;
  p.parents = parents;
  p.new_scores = new_scores;
  p.new_lengths = new_lengths;
  p.new_finished = new_finished;
  p.dev_err = dev_err;
  p.alpha = length_penalty;
  p.B = B; p.K = K; p.V = V; p.N = N;
  p.splits = splits_for(B, K, V);
  p.eos_count = eos_count;
  p.pad = pad_id;
  char* at = static_cast<char*>(workspace) + ANVILQ_WORKSPACE_COUNTER_BYTES;
  p.tickets = static_cast<int*>(workspace);
  p.sums = reinterpret_cast<double2*>(at);
  p.best = reinterpret_cast<unsigned long long*>(at + (size_t)B * K * p.splits * sizeof(double2));
  p.scales = reinterpret_cast<double*>(p.best + (size_t)B * K * p.splits * N);
  const size_t smem = std::max(sizeof(List), sizeof(Merge));
  const dim3 grid(p.splits, B * K);
  cudaStream_t st = reinterpret_cast<cudaStream_t>(stream);
  return logits_half ? launch(beam_kernel<__half>, grid, smem, st, flags, p)
                     : launch(beam_kernel<float>, grid, smem, st, flags, p);
}

int anvilq_beam_reorder(const anvilq_beam_state* states, int count, const int32_t* parents, int B, int K, int N,
                        int* dev_err, unsigned flags, anvilq_stream_t stream) {
  using namespace anvilq;
  using namespace anvilq::beam;
  if (!parents || !dev_err || count < 0 || (count && !states)) return ANVILQ_EINVAL;
  if (flags & ~(unsigned)ANVILQ_GEMM_OVERLAP_PRIOR) return ANVILQ_EINVAL;
  if (B < 1 || K < 1 || N < 1 || (long long)B * std::max(K, N) > (1 << 24)) return ANVILQ_ESHAPE;
  if (reinterpret_cast<uintptr_t>(parents) % 4) return ANVILQ_EALIGN;
  for (int i = 0; i < count; ++i) {
    const anvilq_beam_state& a = states[i];
    if (!a.in || !a.out || a.row_bytes < 1) return ANVILQ_EINVAL;
    if (a.row_bytes > (1LL << 40) / (B * (long long)std::max(K, N))) return ANVILQ_ESHAPE;
  }
  for (int i = 0; i < count; ++i) {
    const anvilq_beam_state& a = states[i];
    const size_t out = (size_t)B * N * a.row_bytes;
    if (overlap(a.out, out, parents, (size_t)B * N * 4)) return ANVILQ_EINVAL;
    for (int j = 0; j < count; ++j) {
      const anvilq_beam_state& o = states[j];
      if (overlap(a.out, out, o.in, (size_t)B * K * o.row_bytes) ||
          (j != i && overlap(a.out, out, o.out, (size_t)B * N * o.row_bytes)))
        return ANVILQ_EINVAL;
    }
  }
  for (int done = 0; done < count; done += kMaxStates) {
    Reorder p{};
    p.parents = parents;
    p.dev_err = dev_err;
    p.B = B; p.K = K; p.N = N;
    p.states = std::min(kMaxStates, count - done);
    long long widest = 0;
    for (int i = 0; i < p.states; ++i) {
      const anvilq_beam_state& a = states[done + i];
      p.state[i] = State{static_cast<const char*>(a.in), static_cast<char*>(a.out), a.row_bytes};
      widest = std::max<long long>(widest, a.row_bytes);
    }
    // CTAs of a row: 16 KB each, no more than fill the device
    const int rows = std::min(B * N, 65535);
    const long long fill = (148 * 8 + (long long)rows * p.states - 1) / ((long long)rows * p.states);
    const int ctas = (int)std::max<long long>(1, std::min<long long>((widest + 16383) / 16384, fill));
    if (const int rc = launch(reorder_kernel, dim3(ctas, rows, p.states), 0, reinterpret_cast<cudaStream_t>(stream),
                              done ? flags | ANVILQ_GEMM_OVERLAP_PRIOR : flags, p))
      return rc;
  }
  return ANVILQ_OK;
}

}  // extern "C"
