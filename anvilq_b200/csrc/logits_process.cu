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
// Work split: a CTA takes a span of the vocabulary of one row.  While its first
// logits travel it marks the span's special tokens -- of the row's history and of
// its bias list -- in a bitmap, counts the marks up to each word, and so gives every
// special token a place in short tables (occurrences, last bias index).  A dense
// pass then masks and writes all logits, taking the largest of the others; behind a
// barrier the special ones are computed from their tables, a thread each, and
// written over.  More special tokens than the tables hold take further rounds over
// the history.  (One pass that looks every token up took 55 instructions a logit,
// as nearly every warp has some lane with a penalty; tables as long as the
// vocabulary, stretch by stretch, spent their time in barriers.)  The choice is a
// maximum over orderable (value, index) keys, combined over a row's CTAs with an
// integer atomicMax, so its result does not depend on their order.
#include <algorithm>

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
  int V, L, bias_total, masks, span;
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
constexpr int kMaxSpan = 32768;
constexpr int kWords = kMaxSpan / 32;          // of the bitmap
constexpr int kTable = 2048;                   // special tokens of a round
constexpr int kIds = 8;                        // tokens of the history that a thread keeps
static_assert(kWords == 4 * kThreads && kMaxSpan <= 0x10000, "four words a thread; a place fits 16 bits");

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
// Otherwise its 8 logits lie kThreads apart, so that a warp's loads still are whole
// sectors.
template <typename T, bool WIDE>
__global__ void __launch_bounds__(kThreads, 4) logits_kernel(const __grid_constant__ Params p) {
  __shared__ uint32_t s_map[kWords];    // bit: a special token
  __shared__ int s_rank[kWords];        // special tokens before the word's
  __shared__ int s_count[kTable];       // occurrences in the generated part; bit 31: in the history at all
  __shared__ int s_entry[kTable];       // last index in the bias list, or -1
  __shared__ uint16_t s_token[kTable];
  __shared__ int s_sum[kThreads / 32];
  __shared__ unsigned s_best[kThreads / 32];
  __shared__ int s_at;
  asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
  asm volatile("griddepcontrol.wait;" ::: "memory");
  const int b = blockIdx.y, lane = threadIdx.x % 32, warp = threadIdx.x / 32;
  const int v0 = blockIdx.x * p.span, v1 = min(p.V, v0 + p.span);
  const bool lead = blockIdx.x == 0 && threadIdx.x == 0;
  const T* x = static_cast<const T*>(p.x) + b * p.ld;
  constexpr int kApart = WIDE ? 1 : kThreads;             // between a piece's logits
  const int first = v0 + (int)threadIdx.x * (WIDE ? kPiece : 1);
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
    if (WIDE && v + kPiece <= v1) raw[i].load(x + v);     // others are loaded when they are used
    if (WIDE && allowed && v < v1) bits[i] = allowed[v / 32];
  };
#pragma unroll
  for (int i = 0; i < kAhead; ++i) load(i, first + i * kAcross);

  // ---- the special tokens ----
  int hist = 0, prompt = 0, bias0 = 0, bias1 = 0, specials = 0;
  const int32_t* history = p.history + b * p.history_ld;
  constexpr int kNone = 0x7FFFFFFF;   // in no span
  int ids[kIds];
  const bool special = p.history || p.bias_starts;
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
    }
    if (p.bias_starts) {
      bias0 = p.bias_starts[b];
      bias1 = p.bias_starts[b + 1];
      if (bias0 < 0 || bias1 > p.bias_total || bias0 > bias1) {
        if (lead) atomicOr(p.dev_err, ANVILQ_DEV_ERR_SEQLEN);
        bias0 = bias1 = 0;
      }
    }
    for (int i = threadIdx.x; i < kWords; i += kThreads) s_map[i] = 0u;
    clear();
    __syncthreads();
    // an id outside the vocabulary is reported (by the row's first CTA) and ignored
    auto mark = [&](int id) {
      if (blockIdx.x == 0 && (unsigned)id >= (unsigned)p.V) atomicOr(p.dev_err, ANVILQ_DEV_ERR_TOKEN);
      if (id >= v0 && id < v1) atomicOr(s_map + (id - v0) / 32, 1u << ((id - v0) % 32));
    };
#pragma unroll
    for (int k = 0; k < kIds; ++k) {
      if ((int)threadIdx.x + k * kThreads < hist) mark(ids[k]);
      else ids[k] = kNone;
    }
    for (int i = kIds * kThreads + threadIdx.x; i < hist; i += kThreads) mark(history[i]);
    for (int i = bias0 + threadIdx.x; i < bias1; i += kThreads) mark(p.bias_ids[i]);
    __syncthreads();
    // marks before each word: a thread's four words, the warp's threads, the warps
    const uint4 mine = reinterpret_cast<const uint4*>(s_map)[threadIdx.x];
    const int n0 = __popc(mine.x), n1 = n0 + __popc(mine.y), n2 = n1 + __popc(mine.z), n3 = n2 + __popc(mine.w);
    int upto = n3;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const int up = __shfl_up_sync(0xffffffffu, upto, o);
      if (lane >= o) upto += up;
    }
    if (lane == 31) s_sum[warp] = upto;
    __syncthreads();
    int before = upto - n3;
#pragma unroll
    for (int w = 0; w < kThreads / 32; ++w) {
      const int n = s_sum[w];
      specials += n;
      if (w < warp) before += n;
    }
    reinterpret_cast<int4*>(s_rank)[threadIdx.x] = make_int4(before, before + n0, before + n1, before + n2);
    __syncthreads();
  }
  // the occurrences of the special tokens from rank r0 on, as many as the tables hold
  auto tally = [&](int r0) {
    auto place = [&](int id) {
      if (id < v0 || id >= v1) return -1;
      const int at = id - v0;
      const int i = s_rank[at / 32] + __popc(s_map[at / 32] & ((1u << (at % 32)) - 1u)) - r0;
      if (i < 0 || i >= kTable) return -1;
      s_token[i] = (uint16_t)at;
      return i;
    };
    auto occurs = [&](int at, int i) {
      if (at < 0) return;
      if (i >= prompt) atomicAdd(s_count + at, 1);
      else atomicOr(reinterpret_cast<unsigned*>(s_count + at), 0x80000000u);
    };
    if (r0 == 0)
#pragma unroll
      for (int k = 0; k < kIds; ++k) occurs(place(ids[k]), threadIdx.x + k * kThreads);
    // (later rounds read all of it again: its tokens in registers would cost the dense pass)
    for (int i = (r0 == 0 ? kIds * kThreads : 0) + threadIdx.x; i < hist; i += kThreads) occurs(place(history[i]), i);
    for (int i = bias0 + threadIdx.x; i < bias1; i += kThreads) {
      const int at = place(p.bias_ids[i]);
      if (at >= 0) atomicMax(s_entry + at, i);   // the last entry of an id
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
  for (int vb = first; vb < v1; vb += kAhead * kAcross) {
#pragma unroll
    for (int i = 0; i < kAhead; ++i) {
      const int v = vb + i * kAcross;
      if (v >= v1) break;
      const bool whole = v + (kPiece - 1) * kApart < v1;
      float l[kPiece];
      uint32_t skip = 0u;     // bit e: special
      if (WIDE) {
        if (special) skip = s_map[(v - v0) / 32] >> (v % 32) & 0xFFu;   // a span starts with a word
        if (whole) {
          raw[i].get(l);
        } else {
#pragma unroll
          for (int e = 0; e < kPiece; ++e) l[e] = v + e < v1 ? to_float(x[v + e]) : -INFINITY;
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
          if (u < v1) {
            l[e] = to_float(x[u]);
            if (special) skip |= (s_map[(u - v0) / 32] >> (u % 32) & 1u) << e;
            if (allowed && !(allowed[u / 32] >> (u % 32) & 1u)) l[e] = -INFINITY;
          }
        }
      }
      load(i, v + kAhead * kAcross);
      if (out) {
        if (WIDE && whole && p.wide_out) {
          reinterpret_cast<float4*>(out + v)[0] = make_float4(l[0], l[1], l[2], l[3]);
          reinterpret_cast<float4*>(out + v)[1] = make_float4(l[4], l[5], l[6], l[7]);
        } else {
#pragma unroll
          for (int e = 0; e < kPiece; ++e)
            if (v + e * kApart < v1) out[v + e * kApart] = l[e];
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
      const int v = v0 + s_token[i], said = s_count[i], k = s_entry[i];
      float l = to_float(x[v]);
      if (said) {
        l = l > 0.0f ? __fdiv_rn(l, rep) : __fmul_rn(l, rep);
        if (said & 0x7FFFFFFF) l = __fsub_rn(__fsub_rn(l, __fmul_rn(freq, (float)(said & 0x7FFFFFFF))), pres);
      }
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

// The span of a CTA: one wave of CTAs (four an SM) over the rows, each at least a
// few hundred logits and at most what the bitmap holds.
static int span_for(int B, int V) {
  const int ctas = std::max(1, 592 / B);
  const int span = ((V + ctas - 1) / ctas + 511) / 512 * 512;
  return std::min(span, kMaxSpan);
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
  if (B > kMaxRows || V > (1 << 30)) return ANVILQ_ESHAPE;
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
  p.span = span_for(B, V);
  const bool wide = aligned(logits, 16) && logits_stride % (logits_half ? 8 : 4) == 0;
  p.wide_out = out && aligned(out, 16) && out_stride % 4 == 0;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3((V + p.span - 1) / p.span, B);
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
