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
// Work split: a CTA takes some consecutive stretches of the vocabulary of one row.
// It keeps the row's history in registers (its first 2048 tokens; longer ones are
// read again) and for each stretch, while the stretch's logits travel, enters the
// tokens that lie in it -- of the history and of the bias list -- into tables in
// shared memory: occurrences, list indexes, a bitmap, and a list of the different
// tokens.  Then a dense pass masks and writes the logits outside the bitmap, and a
// sparse one computes the listed tokens, each by one thread, which cleans their
// cells.  (One pass that looks every token up took 55 instructions a logit: nearly
// every warp has some lane with a penalty.)  The choice is a maximum over orderable
// (value, index) keys, combined over a row's CTAs with an integer atomicMax, so
// its result does not depend on their order.
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
  int V, L, bias_total, masks, stretch, per_cta;
  int wide_out;                  // out's rows start on 16-byte boundaries
};

// ascending with the value, above that of -inf for every other number; -0 as +0
__device__ __forceinline__ unsigned orderable(float v) {
  const uint32_t b = __float_as_uint(v + 0.0f);
  return (b & 0x80000000u) ? ~b : (b | 0x80000000u);
}

constexpr int kPiece = 8;                                // logits of a thread at a time
constexpr int kPieces = 2;
constexpr int kMaxStretch = kThreads * kPiece * kPieces;

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

constexpr int kIds = 8;                                  // tokens of the history that a thread keeps

// WIDE: rows start on 16-byte boundaries; a thread's piece is 8 consecutive logits.
// Otherwise its 8 logits lie kThreads apart, so that a warp's loads still are whole
// sectors.
template <typename T, bool WIDE>
__global__ void __launch_bounds__(kThreads, 4) logits_kernel(const __grid_constant__ Params p) {
  extern __shared__ __align__(16) int tables[];
  __shared__ uint32_t s_map[2][kMaxStretch / 32];   // the listed tokens; of even and odd stretches
  __shared__ int s_listed[2];
  __shared__ unsigned s_best[kThreads / 32];
  __shared__ int s_at;
  asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
  asm volatile("griddepcontrol.wait;" ::: "memory");
  const int b = blockIdx.y;
  const int row_end = min((long long)p.V, ((long long)blockIdx.x + 1) * p.per_cta * p.stretch);
  int v0 = blockIdx.x * p.per_cta * p.stretch;
  const bool lead = blockIdx.x == 0 && threadIdx.x == 0;
  const T* x = static_cast<const T*>(p.x) + b * p.ld;
  constexpr int kAcross = kThreads * kPiece;
  constexpr int kApart = WIDE ? 1 : kThreads;             // between a piece's logits
  const int first = (int)threadIdx.x * (WIDE ? kPiece : 1);
  Raw8<T> raw[kPieces];       // whole pieces
  auto load = [&](int v0) {
    const int v1 = min(row_end, v0 + p.stretch);
#pragma unroll
    for (int i = 0; i < kPieces; ++i) {
      const int v = v0 + first + i * kAcross;
      if (WIDE && v + kPiece <= v1) raw[i].load(x + v);   // others are loaded when they are used
    }
  };
  load(v0);
  // ---- what the row brings ----
  const int32_t* history = p.history + b * p.history_ld;
  int ids[kIds];
  int hist = 0, prompt = 0, bias0 = 0, bias1 = 0;
  if (p.history) {
#pragma unroll
    for (int k = 0; k < kIds; ++k) {
      const int i = threadIdx.x + k * kThreads;
      ids[k] = i < p.L ? history[i] : -1;
    }
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
  const float rep = p.repetition ? p.repetition[b] : 1.0f;
  const float pres = p.presence ? p.presence[b] : 0.0f;
  const float freq = p.frequency ? p.frequency[b] : 0.0f;
  const uint32_t* allowed = nullptr;
  if (p.allowed) {
    const int row = p.allowed_rows ? p.allowed_rows[b] : b;   // negative: the row has no mask
    if (row >= p.masks) {
      if (lead) atomicOr(p.dev_err, ANVILQ_DEV_ERR_SEQLEN);
    } else if (row >= 0) {
      allowed = p.allowed + row * p.allowed_ld;
    }
  }
  float* out = p.out ? p.out + b * p.out_ld : nullptr;
  const bool special = p.history || p.bias_starts;
  int* count = tables;                                            // occurrences in the generated part
  int* entry = tables + (p.history ? p.stretch : 0);              // last index of the bias list, or -1
  uint16_t* listed = reinterpret_cast<uint16_t*>(entry + (p.bias_starts ? p.stretch : 0));
  static_assert(kMaxStretch <= 0x10000, "a place fits 16 bits");
  if (special) {
    if (p.history)
      for (int i = threadIdx.x; i < p.stretch / 4; i += kThreads) reinterpret_cast<int4*>(count)[i] = make_int4(0, 0, 0, 0);
    if (p.bias_starts)
      for (int i = threadIdx.x; i < p.stretch / 4; i += kThreads) reinterpret_cast<int4*>(entry)[i] = make_int4(-1, -1, -1, -1);
    for (int i = threadIdx.x; i < kMaxStretch / 32; i += kThreads) s_map[0][i] = s_map[1][i] = 0u;
    if (threadIdx.x < 2) s_listed[threadIdx.x] = 0;
  }
  if (threadIdx.x == 0) s_at = 0x7FFFFFFF;
  // an id outside the vocabulary is reported (by the row's first CTA) and ignored
  auto report = [&](int id) {
    if (blockIdx.x == 0 && (unsigned)id >= (unsigned)p.V) atomicOr(p.dev_err, ANVILQ_DEV_ERR_TOKEN);
  };
#pragma unroll
  for (int k = 0; k < kIds; ++k) {
    const int i = threadIdx.x + k * kThreads;
    if (p.history && i < hist) report(ids[k]);
    else ids[k] = -1;
  }
  for (int i = kIds * kThreads + threadIdx.x; i < hist; i += kThreads) report(history[i]);
  for (int i = bias0 + threadIdx.x; i < bias1; i += kThreads) report(p.bias_ids[i]);

  float best = -INFINITY;
  int best_at = 0x7FFFFFFF;   // the lowest of equals
  int parity = 0;
#pragma unroll 1
  for (; v0 < row_end; v0 += p.stretch, parity ^= 1) {
    const int v1 = min(row_end, v0 + p.stretch);
    uint32_t* map = s_map[parity];
    if (special) {
      __syncthreads();      // the tables are clean
      auto enter = [&](int at) {   // the first of a token's threads lists it
        const uint32_t bit = 1u << (at % 32);
        if (!(atomicOr(map + at / 32, bit) & bit)) listed[atomicAdd(&s_listed[parity], 1)] = (uint16_t)at;
      };
      auto occurs = [&](int id, int i) {
        if (id >= v0 && id < v1) {
          enter(id - v0);
          // bit 31: in the history at all
          if (i >= prompt) atomicAdd(count + (id - v0), 1);
          else atomicOr(reinterpret_cast<unsigned*>(count + (id - v0)), 0x80000000u);
        }
      };
      if (p.history) {
#pragma unroll
        for (int k = 0; k < kIds; ++k) occurs(ids[k], threadIdx.x + k * kThreads);
        for (int i = kIds * kThreads + threadIdx.x; i < hist; i += kThreads) occurs(history[i], i);
      }
      for (int i = bias0 + threadIdx.x; i < bias1; i += kThreads) {
        const int id = p.bias_ids[i];
        if (id >= v0 && id < v1) {
          enter(id - v0);
          atomicMax(entry + (id - v0), i);   // the last entry of an id
        }
      }
      __syncthreads();
    }

    // ---- dense: what is not listed ----
#pragma unroll
    for (int i = 0; i < kPieces; ++i) {
      const int v = v0 + first + i * kAcross, at = v - v0;
      if (v >= v1) break;
      const bool whole = v + (kPiece - 1) * kApart < v1;
      float l[kPiece];
      uint32_t skip = 0u;     // bit e: listed
      if (WIDE) {
        if (special) skip = map[at / 32] >> (at % 32) & 0xFFu;
        if (whole) {
          raw[i].get(l);
        } else {
#pragma unroll
          for (int e = 0; e < kPiece; ++e) l[e] = v + e < v1 ? to_float(x[v + e]) : -INFINITY;
        }
        if (allowed) {
          const uint32_t bits = allowed[v / 32] >> (v % 32);
#pragma unroll
          for (int e = 0; e < kPiece; ++e)
            if (!(bits >> e & 1u)) l[e] = -INFINITY;
        }
      } else {
#pragma unroll
        for (int e = 0; e < kPiece; ++e) {
          const int u = v + e * kApart;
          l[e] = -INFINITY;
          if (u < v1) {
            l[e] = to_float(x[u]);
            if (special) skip |= (map[(u - v0) / 32] >> ((u - v0) % 32) & 1u) << e;
            if (allowed && !(allowed[u / 32] >> (u % 32) & 1u)) l[e] = -INFINITY;
          }
        }
      }
      if (out) {
        if (WIDE && whole && p.wide_out && !skip) {
          reinterpret_cast<float4*>(out + v)[0] = make_float4(l[0], l[1], l[2], l[3]);
          reinterpret_cast<float4*>(out + v)[1] = make_float4(l[4], l[5], l[6], l[7]);
        } else {
#pragma unroll
          for (int e = 0; e < kPiece; ++e)
            if (v + e * kApart < v1 && !(skip >> e & 1u)) out[v + e * kApart] = l[e];
        }
      }
      if (skip)
#pragma unroll
        for (int e = 0; e < kPiece; ++e)
          if (skip >> e & 1u) l[e] = -INFINITY;
      const float top = fmaxf(fmaxf(fmaxf(l[0], l[1]), fmaxf(l[2], l[3])), fmaxf(fmaxf(l[4], l[5]), fmaxf(l[6], l[7])));
      if (top > best) {       // a thread's places ascend: an equal one later is not lower
        best = top;
#pragma unroll
        for (int e = kPiece - 1; e >= 0; --e)
          if (l[e] == top) best_at = v + e * kApart;
      }
    }
    load(v0 + p.stretch);     // nothing behind row_end

    // ---- sparse: the listed tokens ----
    if (special) {
      const int n = s_listed[parity];
      for (int i = threadIdx.x; i < n; i += kThreads) {
        const int at = listed[i], v = v0 + at;
        float l = to_float(x[v]);
        if (p.history) {
          const int said = count[at];
          count[at] = 0;
          if (said) {
            l = l > 0.0f ? __fdiv_rn(l, rep) : __fmul_rn(l, rep);
            if (said & 0x7FFFFFFF) l = __fsub_rn(__fsub_rn(l, __fmul_rn(freq, (float)(said & 0x7FFFFFFF))), pres);
          }
        }
        if (p.bias_starts) {
          const int k = entry[at];
          entry[at] = -1;
          if (k >= 0) l = __fadd_rn(l, p.bias_values[k]);
        }
        if (allowed && !(allowed[v / 32] >> (v % 32) & 1u)) l = -INFINITY;
        if (out) out[v] = l;
        if (l > best || (l == best && v < best_at && l > -INFINITY)) {
          best = l;
          best_at = v;
        }
      }
      // the other stretches' map and length, not used before the next barrier
      for (int i = threadIdx.x; i < kMaxStretch / 32; i += kThreads) s_map[parity ^ 1][i] = 0u;
      if (threadIdx.x == 0) s_listed[parity ^ 1] = 0;
    }
  }
  if (!p.token) return;
  // the CTA's best value, then the lowest index that has it
  const unsigned mine = orderable(best);
  const unsigned warp_best = __reduce_max_sync(0xffffffffu, mine);
  if (threadIdx.x % 32 == 0) s_best[threadIdx.x / 32] = warp_best;
  __syncthreads();
  unsigned top = 0u;
#pragma unroll
  for (int w = 0; w < kThreads / 32; ++w) top = max(top, s_best[w]);
  if (mine == top && best > -INFINITY) atomicMin(&s_at, best_at);
  __syncthreads();
  if (threadIdx.x == 0) {
    if (s_at != 0x7FFFFFFF)
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

// A CTA's stretches: short ones, one a CTA, until few rows fill the device; then
// as many a CTA as leave it full (four CTAs an SM), so that the history is read rarely.
static void cut(int B, int V, int* stretch, int* per_cta) {
  int s = kMaxStretch;
  while (s > 512 && (long long)B * ((V + s - 1) / s) < 296) s /= 2;
  const int n = (V + s - 1) / s, ctas = std::max(1, std::min(n, 592 / B));
  *stretch = s;
  *per_cta = (n + ctas - 1) / ctas;
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
  cut(B, V, &p.stretch, &p.per_cta);
  const size_t smem = history || bias_starts ? (size_t)p.stretch * (4 * ((history ? 1 : 0) + (bias_starts ? 1 : 0)) + 2) : 0;
  const bool wide = aligned(logits, 16) && logits_stride % (logits_half ? 8 : 4) == 0;
  p.wide_out = out && aligned(out, 16) && out_stride % 4 == 0;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3((V + p.stretch * p.per_cta - 1) / (p.stretch * p.per_cta), B);
  cfg.blockDim = dim3(kThreads);
  cfg.dynamicSmemBytes = smem;
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
