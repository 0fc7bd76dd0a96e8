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
// Work split: a CTA takes a stretch of the vocabulary of one row.  Its logits are
// loaded first; while they travel it scans the row's history and bias list for the
// tokens of its stretch, into tables in shared memory (occurrences; list index).
// The tables are cleared and read densely: a word a token each way costs less than
// a second scan of the history for the cells that matter.  One pass then applies
// everything.  The choice is a maximum over orderable (value, index) keys, combined
// over a row's CTAs with an integer atomicMax, so its result does not depend on
// their order.
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
  int V, L, bias_total, masks, stretch;
  int wide_out;                  // out's rows start on 16-byte boundaries
};

// larger value first, then the lower index; above 0 for v > -inf
__device__ __forceinline__ unsigned long long choice_key(float v, int index) {
  uint32_t b = __float_as_uint(v + 0.0f);   // -0 as +0
  b = (b & 0x80000000u) ? ~b : (b | 0x80000000u);
  return ((unsigned long long)b << 32) | (unsigned long long)(0xFFFFFFFFu - (uint32_t)index);
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

// WIDE: rows start on 16-byte boundaries; a thread's piece is 8 consecutive logits.
// Otherwise its 8 logits lie kThreads apart, so that a warp's loads still are whole
// sectors.
template <typename T, bool WIDE>
__global__ void __launch_bounds__(kThreads) logits_kernel(const __grid_constant__ Params p) {
  extern __shared__ __align__(16) int tables[];
  __shared__ unsigned long long s_best[kThreads / 32];
  asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
  asm volatile("griddepcontrol.wait;" ::: "memory");
  const int b = blockIdx.y;
  const int v0 = blockIdx.x * p.stretch, v1 = min(p.V, v0 + p.stretch);
  const bool lead = blockIdx.x == 0 && threadIdx.x == 0;
  const T* x = static_cast<const T*>(p.x) + b * p.ld;
  constexpr int kAcross = kThreads * kPiece;
  const int mine = v0 + (int)threadIdx.x * (WIDE ? kPiece : 1), apart = WIDE ? 1 : kThreads;   // of a piece's logits
  Raw8<T> raw[kPieces];
  float loose[kPieces][kPiece];
  // whole pieces only: the row's last logits may not fill one
  auto whole = [&](int i) { return WIDE && mine + i * kAcross + kPiece <= v1; };
#pragma unroll
  for (int i = 0; i < kPieces; ++i) {
    const int v = mine + i * kAcross;
    if (whole(i)) {
      raw[i].load(x + v);
    } else {
#pragma unroll
      for (int e = 0; e < kPiece; ++e)
        loose[i][e] = v + e * apart < v1 ? to_float(x[v + e * apart]) : -INFINITY;
    }
  }

  // ---- the tables: occurrences (top bit: only before the generated part), list indexes ----
  int* count = tables;
  int* entry = tables + (p.history ? p.stretch : 0);
  if (p.history || p.bias_starts) {
    if (p.history)
      for (int i = threadIdx.x; i < p.stretch / 4; i += kThreads) reinterpret_cast<int4*>(count)[i] = make_int4(0, 0, 0, 0);
    if (p.bias_starts)
      for (int i = threadIdx.x; i < p.stretch / 4; i += kThreads) reinterpret_cast<int4*>(entry)[i] = make_int4(-1, -1, -1, -1);
    int hist = 0, prompt = 0, bias0 = 0, bias1 = 0;
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
    __syncthreads();
    auto place = [&](int id) {   // in the stretch, or -1
      if ((unsigned)id >= (unsigned)p.V) {
        if (blockIdx.x == 0) atomicOr(p.dev_err, ANVILQ_DEV_ERR_TOKEN);
        return -1;
      }
      return id >= v0 && id < v1 ? id - v0 : -1;
    };
    const int32_t* history = p.history + b * p.history_ld;
#pragma unroll 4
    for (int i = threadIdx.x; i < hist; i += kThreads) {
      const int at = place(history[i]);
      if (at >= 0) {
        if (i >= prompt) atomicAdd(count + at, 1);
        else atomicOr(reinterpret_cast<unsigned*>(count + at), 0x80000000u);
      }
    }
    for (int i = bias0 + threadIdx.x; i < bias1; i += kThreads) {
      const int at = place(p.bias_ids[i]);
      if (at >= 0) atomicMax(entry + at, i);   // the last entry of an id
    }
    __syncthreads();
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
  float best = -INFINITY;   // the thread's logits come in ascending order: the first of equals stays
  int best_at = -1;
#pragma unroll
  for (int i = 0; i < kPieces; ++i) {
    const int v = mine + i * kAcross, at = v - v0;
    if (v >= v1) break;
    float l[kPiece];
    if (whole(i)) {
      raw[i].get(l);
    } else {
#pragma unroll
      for (int e = 0; e < kPiece; ++e) l[e] = loose[i][e];
    }
    if (p.history) {
      int n[kPiece];
      if (WIDE) {   // the stretch is a multiple of a piece
        *reinterpret_cast<int4*>(n) = *reinterpret_cast<const int4*>(count + at);
        *reinterpret_cast<int4*>(n + 4) = *reinterpret_cast<const int4*>(count + at + 4);
      } else {
#pragma unroll
        for (int e = 0; e < kPiece; ++e) n[e] = v + e * apart < v1 ? count[at + e * apart] : 0;
      }
#pragma unroll
      for (int e = 0; e < kPiece; ++e)
        if (n[e]) {
          l[e] = l[e] > 0.0f ? __fdiv_rn(l[e], rep) : __fmul_rn(l[e], rep);
          const int said = n[e] & 0x7FFFFFFF;
          if (said) l[e] = __fsub_rn(__fsub_rn(l[e], __fmul_rn(freq, (float)said)), pres);
        }
    }
    if (p.bias_starts) {
      int n[kPiece];
      if (WIDE) {
        *reinterpret_cast<int4*>(n) = *reinterpret_cast<const int4*>(entry + at);
        *reinterpret_cast<int4*>(n + 4) = *reinterpret_cast<const int4*>(entry + at + 4);
      } else {
#pragma unroll
        for (int e = 0; e < kPiece; ++e) n[e] = v + e * apart < v1 ? entry[at + e * apart] : -1;
      }
#pragma unroll
      for (int e = 0; e < kPiece; ++e)
        if (n[e] >= 0) l[e] = __fadd_rn(l[e], p.bias_values[n[e]]);
    }
    if (allowed) {
      const uint32_t bits = WIDE ? allowed[v / 32] >> (v % 32) : 0u;
#pragma unroll
      for (int e = 0; e < kPiece; ++e) {
        const int u = v + e * apart;
        if (WIDE ? !(bits >> e & 1u) : u < v1 && !(allowed[u / 32] >> (u % 32) & 1u)) l[e] = -INFINITY;
      }
    }
#pragma unroll
    for (int e = 0; e < kPiece; ++e)
      if (l[e] > best && v + e * apart < v1) {
        best = l[e];
        best_at = v + e * apart;
      }
    if (out) {
      if (whole(i) && p.wide_out) {
        reinterpret_cast<float4*>(out + v)[0] = make_float4(l[0], l[1], l[2], l[3]);
        reinterpret_cast<float4*>(out + v)[1] = make_float4(l[4], l[5], l[6], l[7]);
      } else {
#pragma unroll
        for (int e = 0; e < kPiece; ++e)
          if (v + e * apart < v1) out[v + e * apart] = l[e];
      }
    }
  }
  if (!p.token) return;
  unsigned long long key = best_at >= 0 ? choice_key(best, best_at) : 0ull;
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) {
    const unsigned long long other = __shfl_xor_sync(0xffffffffu, key, o);
    key = other > key ? other : key;
  }
  if (threadIdx.x % 32 == 0) s_best[threadIdx.x / 32] = key;
  __syncthreads();
  if (threadIdx.x == 0) {
    for (int w = 1; w < kThreads / 32; ++w) key = s_best[w] > key ? s_best[w] : key;
    if (key) atomicMax(p.keys + b, key);
    __threadfence();
    if (atomicAdd(p.tickets + b, 1) == (int)gridDim.x - 1) {   // the row's last CTA
      __threadfence();
      const unsigned long long k = atomicExch(p.keys + b, 0ull);
      p.tickets[b] = 0;
      p.token[b] = k ? (int)(0xFFFFFFFFu - (uint32_t)(k & 0xFFFFFFFFull)) : -1;
    }
  }
}

// The stretch of a CTA: few CTAs a row scan the history fewer times, many fill
// the device.
static int stretch_for(int B, int V) {
  int s = kMaxStretch;
  while (s > 512 && (long long)B * ((V + s - 1) / s) < 296) s /= 2;
  return s;
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
  p.stretch = stretch_for(B, V);
  const size_t smem = (size_t)p.stretch * 4 * ((history ? 1 : 0) + (bias_starts ? 1 : 0));
  const bool wide = aligned(logits, 16) && logits_stride % (logits_half ? 8 : 4) == 0;
  p.wide_out = out && aligned(out, 16) && out_stride % 4 == 0;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3((V + p.stretch - 1) / p.stretch, B);
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
