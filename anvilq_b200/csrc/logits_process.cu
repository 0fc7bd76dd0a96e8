// logits_process.cu -- penalties for repeated tokens, biases and grammar masks on
// a batch's logits, and the greedy choice.
//
// Mathematics, for row b and token v (binary32, each operation rounded):
//   seen   v occurs in history[b][0 .. history_lens[b])
//   count  its occurrences from prompt_lens[b] on (the generated part)
//   l = logits[b][v]
//   seen:       l = l > 0 ? l / repetition[b] : l * repetition[b]
//   count > 0:  l = (l - frequency[b] * count) - presence[b]
//   biased:     l = l + the last of v's entries in the row's bias list
//   not allowed by the row's mask: l = -inf
//   out[b][v] = l;  token[b] = the lowest v with the largest l > -inf, else -1.
//
// What bounds it: bytes -- each logit in and out once (the history, the lists and
// the mask's bits are small beside them).
//
// Work split: the vocabulary is cut into chunks of 256, dealt in turn to a row's
// CTAs (the tokens of a history crowd at one end of a vocabulary: with a contiguous
// span a CTA, the first one's took several rounds -- below -- while the others
// waited; 64 rows with 32768 tokens of history 141 us, dealt out 99 us).
// While its first logits travel a CTA marks its special tokens -- of the row's
// history and of its bias list -- in a bitmap, counts the marks up to each word, and
// so gives every one a place in short tables (occurrences, last bias index).  A dense
// pass then masks and writes all logits, taking the largest of the others; behind a
// barrier the special ones are computed from their tables, a thread each, and
// written over.  More special tokens than the tables hold take further rounds over
// the history.  (One pass that looks every token up took 55 instructions a logit,
// as nearly every warp has some lane with a penalty; tables as long as the
// vocabulary, stretch by stretch, spent their time in barriers.)  The choice is a
// maximum over orderable (value, index) keys, combined over a row's CTAs with an
// integer atomicMax, so its result does not depend on their order.
#include <algorithm>
#include <cmath>

#include <cuda_fp16.h>
#include <cuda_runtime.h>
#include <stdint.h>

#include "../../include/anvilq.h"

namespace anvilq {
namespace logits {

constexpr int kThreads = 256;
constexpr int kMaxRows = 4096;
constexpr int kTicketOffset = 32768;   // of the workspace's counters: 4096 keys, then 4096 tickets
static_assert(kTicketOffset >= kMaxRows * 8 && kTicketOffset + kMaxRows * 4 <= ANVILQ_WORKSPACE_COUNTER_BYTES,
              "keys and tickets lie in the counter region");

struct Params {
  const void* x;                 // fp32 or fp16 [B] rows of V, ld elements apart
  long long ld;
  float* out;                    // [B] rows of V, out_ld apart; may be x itself; or null
  long long out_ld;
  int32_t* token;                // [B] or null
  const int32_t* history;        // [B] rows of L
  long long history_ld;
  const int32_t* history_lens;   // [B]
  const int32_t* prompt_lens;    // [B] or null (0)
  const float* repetition;       // [B] or null, as the next two
  const float* presence;
  const float* frequency;
  const int32_t* bias_starts;    // [B + 1]
  const int32_t* bias_ids;
  const float* bias_values;
  const uint32_t* allowed;       // rows of words, allowed_ld apart
  long long allowed_ld;
  const int32_t* allowed_rows;   // [B] or null (b)
  unsigned long long* keys;
  int* tickets;
  int* dev_err;
  int V, L, bias_total, masks;
  unsigned magic, shift;         // chunk / CTAs of a row = umulhi(2 chunk, magic) >> shift
  int wide_out;                  // out's rows start on 16-byte boundaries
};

// ascending with the value, above that of -inf for every other number; -0 as +0
__device__ __forceinline__ unsigned orderable(float v) {
  const uint32_t b = __float_as_uint(v + 0.0f);
  return (b & 0x80000000u) ? ~b : (b | 0x80000000u);
}

constexpr int kPiece = 8;                      // logits of a thread at a time
constexpr int kAhead = 2;                      // pieces loaded ahead
constexpr int kAcross = kThreads * kPiece;
constexpr int kChunk = 32 * kPiece;            // logits of a warp at a time
constexpr int kMaxSpan = 32768;                // logits of a CTA
constexpr int kWords = kMaxSpan / 32;          // of the bitmap
constexpr int kTable = 2048;                   // special tokens of a round
constexpr int kIds = 8;                        // tokens of the history that a thread keeps
constexpr int kScan = 8;                       // further ones, loaded at a time
static_assert(kWords == 4 * kThreads && kMaxSpan <= 0x8000, "four words a thread; an `at` has 15 bits");

// eight consecutive logits, 16-byte aligned, as they are stored
template <typename T> struct Raw8;
template <> struct Raw8<float> {
  float4 a, b;
  __device__ __forceinline__ void load(const float* p) {
    a = reinterpret_cast<const float4*>(p)[0];
    b = reinterpret_cast<const float4*>(p)[1];
  }
  __device__ __forceinline__ void get(float* l) const {
    l[0] = a.x; l[1] = a.y; l[2] = a.z; l[3] = a.w;
    l[4] = b.x; l[5] = b.y; l[6] = b.z; l[7] = b.w;
  }
};
template <> struct Raw8<__half> {
  uint4 w;
  __device__ __forceinline__ void load(const __half* p) { w = *reinterpret_cast<const uint4*>(p); }
  __device__ __forceinline__ void get(float* l) const {
    const __half2* h = reinterpret_cast<const __half2*>(&w);
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const float2 f = __half22float2(h[i]);
      l[2 * i] = f.x;
      l[2 * i + 1] = f.y;
    }
  }
};
__device__ __forceinline__ float to_float(float v) { return v; }
__device__ __forceinline__ float to_float(__half v) { return __half2float(v); }

// WIDE: rows start on 16-byte boundaries; a thread's piece is 8 consecutive logits.
// Otherwise its 8 logits lie 32 apart, so that a warp's loads still are whole sectors.
// A CTA numbers the logits of its chunks, one after the other, by `at`.
template <typename T, bool WIDE>
__global__ void __launch_bounds__(kThreads, 4) logits_kernel(const __grid_constant__ Params p) {
  __shared__ uint32_t s_map[kWords];    // bit: a special token (at first: of the bias list)
  __shared__ uint32_t s_seen[kWords];   // bit: a token of the history
  __shared__ int s_rank[kWords];        // special tokens before the word's
  __shared__ int s_count[kTable];       // occurrences in the generated part
  __shared__ int s_entry[kTable];       // last index in the bias list, or -1
  __shared__ uint16_t s_token[kTable];  // its `at`; bit 15: of the history
  __shared__ int s_sum[kThreads / 32];
  __shared__ unsigned s_best[kThreads / 32];
  __shared__ int s_at;
  asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
  asm volatile("griddepcontrol.wait;" ::: "memory");
  const int b = blockIdx.y, lane = threadIdx.x % 32, warp = threadIdx.x / 32;
  const int nth = blockIdx.x, ctas = gridDim.x;
  const bool lead = blockIdx.x == 0 && threadIdx.x == 0;
  const T* x = static_cast<const T*>(p.x) + b * p.ld;
  constexpr int kApart = WIDE ? 1 : 32;                   // between a piece's logits
  const int first_at = WIDE ? threadIdx.x * kPiece : warp * kChunk + lane;
  const int first = (warp * ctas + nth) * kChunk + first_at % kChunk, across = kAcross * ctas;
  const uint32_t* allowed = nullptr;
  if (p.allowed) {
    const int row = p.allowed_rows ? p.allowed_rows[b] : b;   // negative: the row has no mask
    if (row >= p.masks) {
      if (lead) atomicOr(p.dev_err, ANVILQ_DEV_ERR_SEQLEN);
    } else if (row >= 0) {
      allowed = p.allowed + row * p.allowed_ld;
    }
  }
  Raw8<T> raw[kAhead];       // whole pieces, and their words of the mask
  uint32_t bits[kAhead];
  auto load = [&](int i, int v) {
    if (WIDE && v + kPiece <= p.V) raw[i].load(x + v);    // others are loaded when they are used
    if (WIDE && allowed && v < p.V) bits[i] = allowed[v / 32];
  };
#pragma unroll
  for (int i = 0; i < kAhead; ++i) load(i, first + i * across);

  // ---- the special tokens ----
  int hist = 0, prompt = 0, bias0 = 0, bias1 = 0, specials = 0;
  const int32_t* history = p.history + b * p.history_ld;
  constexpr int kNone = 0x7FFFFFFF;   // no token
  int ids[kIds];                      // then: their `at`, or -1
  auto at_of = [&](int id) {          // -1: in another CTA's chunks
    const unsigned chunk = (unsigned)id / kChunk, q = __umulhi(2 * chunk, p.magic) >> p.shift;
    return (unsigned)id < (unsigned)p.V && chunk - q * ctas == nth ? (int)(q * kChunk + (unsigned)id % kChunk) : -1;
  };
  const bool special = p.history || p.bias_starts;
  // the history from `from` on, kScan tokens of a thread on their way at a time (kNone
  // behind its end)
  auto scan = [&](int from, auto each) {
#pragma unroll 1
    for (int i = from + threadIdx.x; i < hist; i += kScan * kThreads) {
      int id[kScan];
#pragma unroll
      for (int k = 0; k < kScan; ++k) id[k] = i + k * kThreads < hist ? history[i + k * kThreads] : kNone;
      each(id, i);
    }
  };
  auto clear = [&] {
    for (int i = threadIdx.x; i < kTable; i += kThreads) {
      s_count[i] = 0;
      s_entry[i] = -1;
    }
  };
  if (special) {
#pragma unroll
    for (int k = 0; k < kIds; ++k) {
      const int i = threadIdx.x + k * kThreads;
      ids[k] = p.history && i < p.L ? history[i] : kNone;
    }
    if (p.history) {
      hist = p.history_lens[b];
      prompt = p.prompt_lens ? p.prompt_lens[b] : 0;
      if (hist < 0 || hist > p.L) {
        if (lead) atomicOr(p.dev_err, ANVILQ_DEV_ERR_SEQLEN);
        hist = max(0, min(hist, p.L));
      }
      prompt = max(0, min(prompt, hist));
    }
    if (p.bias_starts) {
      bias0 = p.bias_starts[b];
      bias1 = p.bias_starts[b + 1];
      if (bias0 < 0 || bias1 > p.bias_total || bias0 > bias1) {
        if (lead) atomicOr(p.dev_err, ANVILQ_DEV_ERR_SEQLEN);
        bias0 = bias1 = 0;
      }
    }
    for (int i = threadIdx.x; i < kWords; i += kThreads) s_map[i] = s_seen[i] = 0u;
    clear();
    __syncthreads();
    // an id outside the vocabulary is reported (by the row's first CTA) and ignored
    auto report = [&](int id) {
      if (nth == 0 && (unsigned)id >= (unsigned)p.V) atomicOr(p.dev_err, ANVILQ_DEV_ERR_TOKEN);
    };
    // (most tokens of a long history are marked already: reading first keeps their
    // lanes from queueing at one word)
    auto mark = [](uint32_t* map, int at) {
      if (at >= 0 && !(map[at / 32] >> (at % 32) & 1u)) atomicOr(map + at / 32, 1u << (at % 32));
    };
#pragma unroll
    for (int k = 0; k < kIds; ++k) {
      const bool live = (int)threadIdx.x + k * kThreads < hist;
      if (live) report(ids[k]);
      ids[k] = live ? at_of(ids[k]) : -1;
      mark(s_seen, ids[k]);
    }
    scan(kIds * kThreads, [&](const int* id, int i) {
#pragma unroll
      for (int k = 0; k < kScan; ++k) {
        if (i + k * kThreads < hist) report(id[k]);
        mark(s_seen, at_of(id[k]));
      }
    });
    for (int i = bias0 + threadIdx.x; i < bias1; i += kThreads) {
      report(p.bias_ids[i]);
      mark(s_map, at_of(p.bias_ids[i]));
    }
    __syncthreads();
    // Marks before each word, in the order of threads (a thread's words lie apart, so
    // that crowded neighbours are several threads'), its four words, its warp, the warps.
    int n[4], mine = 0;
#pragma unroll
    for (int k = 0; k < 4; ++k) {
      const int w = threadIdx.x + k * kThreads;
      n[k] = __popc(s_map[w] |= s_seen[w]);
      mine += n[k];
    }
    int upto = mine;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const int up = __shfl_up_sync(0xffffffffu, upto, o);
      if (lane >= o) upto += up;
    }
    if (lane == 31) s_sum[warp] = upto;
    __syncthreads();
    int before = upto - mine;
#pragma unroll
    for (int w = 0; w < kThreads / 32; ++w) {
      const int sum = s_sum[w];
      specials += sum;
      if (w < warp) before += sum;
    }
#pragma unroll
    for (int k = 0; k < 4; ++k) {
      s_rank[threadIdx.x + k * kThreads] = before;
      before += n[k];
    }
    __syncthreads();
  }
  // the special tokens from rank r0 on, as many as the tables hold: which they are,
  // and their occurrences
  auto tally = [&](int r0) {
    auto place = [&](int at) {   // in the tables, of a special token
      const int i = s_rank[at / 32] + __popc(s_map[at / 32] & ((1u << (at % 32)) - 1u)) - r0;
      return i >= 0 && i < kTable ? i : -1;
    };
    // Of a short history, all in registers, each token names itself; of a longer one
    // the bitmap's bits are walked, as then only its generated part is read again (by
    // later rounds all of that: the tokens in registers would cost the dense pass).
    const bool counts = p.presence || p.frequency, direct = r0 == 0 && hist <= kIds * kThreads;
    if (!direct) {
#pragma unroll
      for (int k = 0; k < 4; ++k) {
        const int w = threadIdx.x + k * kThreads;
        const uint32_t seen = s_seen[w];
        int i = s_rank[w] - r0;
        for (uint32_t m = s_map[w]; m; m &= m - 1, ++i) {
          const int bit = __ffs(m) - 1;
          if (i >= 0 && i < kTable) s_token[i] = (uint16_t)(w * 32 + bit | (seen >> bit & 1u) << 15);
        }
      }
    }
    if (r0 == 0)
#pragma unroll
      for (int k = 0; k < kIds; ++k) {
        const int i = ids[k] >= 0 ? place(ids[k]) : -1;
        if (i < 0) continue;
        if (direct) s_token[i] = (uint16_t)(ids[k] | 0x8000);
        if ((int)threadIdx.x + k * kThreads >= prompt) atomicAdd(s_count + i, 1);
      }
    if (counts)
      scan(max(prompt, r0 == 0 ? kIds * kThreads : 0), [&](const int* id, int) {
#pragma unroll
        for (int k = 0; k < kScan; ++k) {
          const int at = at_of(id[k]), i = at >= 0 ? place(at) : -1;
          if (i >= 0) atomicAdd(s_count + i, 1);
        }
      });
    for (int i = bias0 + threadIdx.x; i < bias1; i += kThreads) {
      const int at = at_of(p.bias_ids[i]), j = at >= 0 ? place(at) : -1;
      if (j < 0) continue;
      s_token[j] = (uint16_t)(at | (s_seen[at / 32] >> (at % 32) & 1u) << 15);
      atomicMax(s_entry + j, i);   // the last entry of an id
    }
  };
  if (threadIdx.x == 0) s_at = kNone;
  if (specials > 0) tally(0);

  // ---- dense: all logits masked and written, the largest of those that are not special ----
  const float rep = p.repetition ? p.repetition[b] : 1.0f;
  const float pres = p.presence ? p.presence[b] : 0.0f;
  const float freq = p.frequency ? p.frequency[b] : 0.0f;
  float* out = p.out ? p.out + b * p.out_ld : nullptr;
  float best = -INFINITY;
  int best_at = kNone;        // the lowest of equals
#pragma unroll 1
  for (int vb = first, at = first_at; vb < p.V; vb += kAhead * across) {
#pragma unroll
    for (int i = 0; i < kAhead; ++i) {
      const int v = vb + i * across;
      if (v >= p.V) break;
      const bool whole = v + (kPiece - 1) * kApart < p.V;
      float l[kPiece];
      uint32_t skip = 0u;     // bit e: special
      if (WIDE) {
        if (special) skip = s_map[at / 32] >> (at % 32) & 0xFFu;
        if (whole) {
          raw[i].get(l);
        } else {
#pragma unroll
          for (int e = 0; e < kPiece; ++e) l[e] = v + e < p.V ? to_float(x[v + e]) : -INFINITY;
        }
        if (allowed) {
          const uint32_t a = bits[i] >> (v % 32);
#pragma unroll
          for (int e = 0; e < kPiece; ++e)
            if (!(a >> e & 1u)) l[e] = -INFINITY;
        }
      } else {
#pragma unroll
        for (int e = 0; e < kPiece; ++e) {
          const int u = v + e * kApart;
          l[e] = -INFINITY;
          if (u < p.V) {
            l[e] = to_float(x[u]);
            if (special) skip |= (s_map[at / 32 + e] >> lane & 1u) << e;
            if (allowed && !(allowed[u / 32] >> (u % 32) & 1u)) l[e] = -INFINITY;
          }
        }
      }
      load(i, v + kAhead * across);
      at += kAcross;
      if (out) {
        if (WIDE && whole && p.wide_out) {
          reinterpret_cast<float4*>(out + v)[0] = make_float4(l[0], l[1], l[2], l[3]);
          reinterpret_cast<float4*>(out + v)[1] = make_float4(l[4], l[5], l[6], l[7]);
        } else {
#pragma unroll
          for (int e = 0; e < kPiece; ++e)
            if (v + e * kApart < p.V) out[v + e * kApart] = l[e];
        }
      }
      if (skip)
#pragma unroll
        for (int e = 0; e < kPiece; ++e)
          if (skip >> e & 1u) l[e] = -INFINITY;
      const float t01 = fmaxf(l[0], l[1]), t23 = fmaxf(l[2], l[3]), t45 = fmaxf(l[4], l[5]), t67 = fmaxf(l[6], l[7]);
      const float t03 = fmaxf(t01, t23), top = fmaxf(t03, fmaxf(t45, t67));
      if (top > best) {       // a thread's places ascend: an equal one later is not lower
        best = top;
        // the first that has it, by halves
        const bool e4 = t03 != top, e2 = (e4 ? t45 : t01) != top;
        const bool e1 = (e4 ? (e2 ? l[6] : l[4]) : (e2 ? l[2] : l[0])) != top;
        best_at = v + (4 * e4 + 2 * e2 + e1) * kApart;
      }
    }
  }

  // ---- the special tokens, over what the dense pass wrote ----
  // (Out may be the logits themselves: the dense pass then leaves an allowed one as
  // it is, and a masked one ends as -inf whatever it is computed from.)
#pragma unroll 1
  for (int r0 = 0; r0 < specials; r0 += kTable) {
    if (r0 > 0) {
      __syncthreads();
      clear();
      __syncthreads();
      tally(r0);
    }
    __syncthreads();
    for (int i = threadIdx.x; i < min(kTable, specials - r0); i += kThreads) {
      const int token = s_token[i], at = token & 0x7FFF, count = s_count[i], k = s_entry[i];
      const int v = (at / kChunk * ctas + nth) * kChunk + at % kChunk;
      float l = to_float(x[v]);
      if (token >> 15) l = l > 0.0f ? __fdiv_rn(l, rep) : __fmul_rn(l, rep);
      if (count) l = __fsub_rn(__fsub_rn(l, __fmul_rn(freq, (float)count)), pres);
      if (k >= 0) l = __fadd_rn(l, p.bias_values[k]);
      if (allowed && !(allowed[v / 32] >> (v % 32) & 1u)) l = -INFINITY;
      if (out) out[v] = l;
      if (l > best || (l == best && v < best_at && l > -INFINITY)) {
        best = l;
        best_at = v;
      }
    }
  }
  if (!p.token) return;
  // the CTA's best value, then the lowest index that has it
  const unsigned mine = orderable(best);
  const unsigned warp_best = __reduce_max_sync(0xffffffffu, mine);
  if (lane == 0) s_best[warp] = warp_best;
  __syncthreads();
  unsigned top = 0u;
#pragma unroll
  for (int w = 0; w < kThreads / 32; ++w) top = max(top, s_best[w]);
  if (mine == top && best > -INFINITY) atomicMin(&s_at, best_at);
  __syncthreads();
  if (threadIdx.x == 0) {
    if (s_at != kNone)
      atomicMax(p.keys + b, (unsigned long long)top << 32 | (unsigned long long)(0xFFFFFFFFu - (unsigned)s_at));
    __threadfence();
    if (atomicAdd(p.tickets + b, 1) == (int)gridDim.x - 1) {   // the row's last CTA
      __threadfence();
      const unsigned long long k = atomicExch(p.keys + b, 0ull);
      p.tickets[b] = 0;
      p.token[b] = k ? (int)(0xFFFFFFFFu - (uint32_t)(k & 0xFFFFFFFFull)) : -1;
    }
  }
}

// The CTAs of a row.  A CTA's time grows with its span, about 0.18 us for 1000 logits;
// the launch's with the CTAs in all, about 4 ns each, so the sum is least at
// sqrt(V / 20 B) CTAs a row.  8 rows of 32000: 16 CTAs a row 5.6 us, 4 6.5, 74 6.8; one
// row of 151936: 100 CTAs 5.3 us, 16 6.5; 297 as much as 74, but of two rows 7.7 against
// 5.8.  Where one wave (four an SM) holds a CTA a row at least, they stay within it: 64
// rows of 151936, 9 a row 20.5 us, 10 25.8.  (600 rows of 32000: 2 a row 40.2, 1 46.9.)
static int ctas_for(int B, int V) {
  constexpr int kWave = 4 * 148;
  const int chunks = (V + kChunk - 1) / kChunk;
  int ctas = std::max(1, (int)(std::sqrt(V / (20.0 * B)) + 0.5));
  if (B <= kWave) ctas = std::min(ctas, kWave / B);
  const int each = std::min(std::max(2, (chunks + ctas - 1) / ctas), kMaxSpan / kChunk);
  return (chunks + each - 1) / each;
}

// Whether out can be written while the logits are read: it is the logits, or no row
// of it touches one of theirs (rows of both may take turns in one buffer).
static bool apart(const void* logits, size_t each, long long stride, const float* out, long long out_stride, int B,
                  int V) {
  const uintptr_t x = reinterpret_cast<uintptr_t>(logits), y = reinterpret_cast<uintptr_t>(out);
  const size_t xs = (size_t)stride * each, ys = (size_t)out_stride * 4, xn = V * each, yn = (size_t)V * 4;
  if (x == y) return each == 4 && (B == 1 || xs == ys);
  if (x + (B - 1) * xs + xn <= y || y + (B - 1) * ys + yn <= x) return true;
  if (B == 1 || xs != ys) return false;
  const size_t d = y > x ? (y - x) % xs : (xs - (x - y) % xs) % xs;
  return d >= xn && xs - d >= yn;
}

static bool aligned(const void* p, size_t n) { return reinterpret_cast<uintptr_t>(p) % n == 0; }

}  // namespace logits
}  // namespace anvilq

extern "C" {

size_t anvilq_logits_process_workspace_size(int B, int V) {
  using namespace anvilq::logits;
  if (B < 1 || V < 1 || B > kMaxRows || V > (1 << 30)) return 0;
  return ANVILQ_WORKSPACE_COUNTER_BYTES;
}

int anvilq_logits_process(const void* logits, int logits_half, long long logits_stride, float* out,
                          long long out_stride, int32_t* token, int B, int V, const int32_t* history,
                          long long history_stride, const int32_t* history_lens, const int32_t* prompt_lens, int L,
                          const float* repetition, const float* presence, const float* frequency,
                          const int32_t* bias_starts, const int32_t* bias_ids, const float* bias_values,
                          int bias_total, const uint32_t* allowed, long long allowed_stride,
                          const int32_t* allowed_rows, int masks, void* workspace, size_t workspace_bytes,
                          int* dev_err, unsigned flags, anvilq_stream_t stream) {
  using namespace anvilq::logits;
  if (!logits || (!out && !token) || !dev_err) return ANVILQ_EINVAL;
  if (B < 1 || V < 1 || (logits_half != 0 && logits_half != 1)) return ANVILQ_EINVAL;
  if (flags & ~(unsigned)ANVILQ_GEMM_OVERLAP_PRIOR) return ANVILQ_EINVAL;
  if (logits_stride < V || (out && out_stride < V)) return ANVILQ_EINVAL;
  if (history ? (!history_lens || L < 0 || history_stride < L) : (repetition || presence || frequency))
    return ANVILQ_EINVAL;   // a penalty needs a history
  if (bias_starts && (bias_total < 0 || (bias_total > 0 && (!bias_ids || !bias_values)))) return ANVILQ_EINVAL;
  if (allowed && (masks < 1 || allowed_stride < (V + 31) / 32 || (!allowed_rows && masks < B))) return ANVILQ_EINVAL;
  if (out && !apart(logits, logits_half ? 2 : 4, logits_stride, out, out_stride, B, V)) return ANVILQ_EINVAL;
  if (B > kMaxRows || V > (1 << 30) || (history && L > (1 << 30)) || (bias_starts && bias_total > (1 << 30)))
    return ANVILQ_ESHAPE;
  if (token && (!workspace || workspace_bytes < ANVILQ_WORKSPACE_COUNTER_BYTES)) return ANVILQ_EWORKSPACE;
  if (token && !aligned(workspace, 16)) return ANVILQ_EALIGN;
  if (!aligned(logits, logits_half ? 2 : 4) || !aligned(out, 4)) return ANVILQ_EALIGN;
  Params p{};
  p.x = logits;
  p.ld = logits_stride;
  p.out = out;
  p.out_ld = out_stride;
  p.token = token;
  p.history = history;
  p.history_ld = history_stride;
  p.history_lens = history_lens;
  p.prompt_lens = prompt_lens;
  p.repetition = repetition;
  p.presence = presence;
  p.frequency = frequency;
  p.bias_starts = bias_starts;
  p.bias_ids = bias_ids;
  p.bias_values = bias_values;
  p.allowed = allowed;
  p.allowed_ld = allowed_stride;
  p.allowed_rows = allowed_rows;
  p.keys = static_cast<unsigned long long*>(workspace);
  p.tickets = token ? reinterpret_cast<int*>(static_cast<char*>(workspace) + kTicketOffset) : nullptr;
  p.dev_err = dev_err;
  p.V = V; p.L = L; p.bias_total = bias_total; p.masks = masks;
  const int ctas = ctas_for(B, V);
  // with shift = floor(log2 ctas) and magic = ceil(2^(31 + shift) / ctas) <= 2^31 the
  // quotient is exact below 2^30, and a chunk's number is below 2^24 even of a bad id
  while (ctas >> (p.shift + 1)) ++p.shift;
  p.magic = (unsigned)(((1ull << (31 + p.shift)) + ctas - 1) / ctas);
  const bool wide = aligned(logits, 16) && logits_stride % (logits_half ? 8 : 4) == 0;
  p.wide_out = out && aligned(out, 16) && out_stride % 4 == 0;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(ctas, B);
  cfg.blockDim = dim3(kThreads);
  cfg.stream = reinterpret_cast<cudaStream_t>(stream);
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = attr;
  cfg.numAttrs = (flags & ANVILQ_GEMM_OVERLAP_PRIOR) ? 1 : 0;
  const cudaError_t e = logits_half ? (wide ? cudaLaunchKernelEx(&cfg, logits_kernel<__half, true>, p)
                                            : cudaLaunchKernelEx(&cfg, logits_kernel<__half, false>, p))
                                    : (wide ? cudaLaunchKernelEx(&cfg, logits_kernel<float, true>, p)
                                            : cudaLaunchKernelEx(&cfg, logits_kernel<float, false>, p));
  if (e != cudaSuccess) {
    cudaGetLastError();
    return ANVILQ_ECUDA;
  }
  return ANVILQ_OK;
}

}  // extern "C"
