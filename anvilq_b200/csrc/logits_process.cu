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
// Work split: a CTA takes a stretch of the vocabulary of one row.  It scans the
// row's history and bias list for the tokens of its stretch: a bitmap in shared
// memory says which occur, and a table of the stretch's size holds the counts
// (or the list index), of which only occurring tokens' cells are ever set or
// read.  Then one pass over the logits applies everything; cells are looked up
// only where the bitmap has the token.  The choice is a maximum over orderable
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
  int V, L, bias_total, masks, stretch;
};

// larger value first, then the lower index; 0 for what is never chosen
__device__ __forceinline__ unsigned long long choice_key(float v, int index) {
  if (!(v > -INFINITY)) return 0ull;
  uint32_t b = __float_as_uint(v + 0.0f);   // -0 as +0
  b = (b & 0x80000000u) ? ~b : (b | 0x80000000u);
  return ((unsigned long long)b << 32) | (unsigned long long)(0xFFFFFFFFu - (uint32_t)index);
}

template <typename T> __device__ __forceinline__ float to_float(T v);
template <> __device__ __forceinline__ float to_float<float>(float v) { return v; }
template <> __device__ __forceinline__ float to_float<__half>(__half v) { return __half2float(v); }

// VEC: logits of a thread at a time (4, or 1 where rows are not aligned for it)
template <typename T, int VEC>
__global__ void __launch_bounds__(kThreads) logits_kernel(const __grid_constant__ Params p) {
  extern __shared__ __align__(16) uint32_t smem[];
  __shared__ unsigned long long s_best[kThreads / 32];
  asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
  asm volatile("griddepcontrol.wait;" ::: "memory");
  const int b = blockIdx.y;
  const int v0 = blockIdx.x * p.stretch, v1 = min(p.V, v0 + p.stretch);
  const int words = p.stretch / 32;
  uint32_t* seen = smem;                       // bitmaps of the stretch
  uint32_t* biased = smem + words;
  int* count = reinterpret_cast<int*>(smem + 2 * words);
  int* entry = count + p.stretch;              // present only with a bias list
  const bool lead = blockIdx.x == 0 && threadIdx.x == 0;

  int hist = 0, prompt = 0, bias0 = 0, bias1 = 0;
  const int32_t* history = nullptr;
  if (p.history) {
    hist = p.history_lens[b];
    if (hist < 0 || hist > p.L) {
      if (lead && p.dev_err) atomicOr(p.dev_err, ANVILQ_DEV_ERR_SEQLEN);
      hist = max(0, min(hist, p.L));
    }
    history = p.history + b * p.history_ld;
    prompt = p.prompt_lens ? p.prompt_lens[b] : 0;
  }
  if (p.bias_starts) {
    bias0 = p.bias_starts[b];
    bias1 = p.bias_starts[b + 1];
    if (bias0 < 0 || bias1 > p.bias_total || bias0 > bias1) {
      if (lead && p.dev_err) atomicOr(p.dev_err, ANVILQ_DEV_ERR_SEQLEN);
      bias0 = bias1 = 0;
    }
  }
  for (int i = threadIdx.x; i < 2 * words; i += kThreads) smem[i] = 0u;
  __syncthreads();
  // mark the occurring tokens and clear their cells ...
  auto mark = [&](int id, uint32_t* map, int* cells, int clear) {
    if ((unsigned)id >= (unsigned)p.V) {
      if (blockIdx.x == 0 && p.dev_err) atomicOr(p.dev_err, ANVILQ_DEV_ERR_TOKEN);
    } else if (id >= v0 && id < v1) {
      cells[id - v0] = clear;
      atomicOr(map + (id - v0) / 32, 1u << ((id - v0) % 32));
    }
  };
  for (int i = threadIdx.x; i < hist; i += kThreads) mark(history[i], seen, count, 0);
  for (int i = bias0 + threadIdx.x; i < bias1; i += kThreads) mark(p.bias_ids[i], biased, entry, -1);
  __syncthreads();
  // ... then count them, and take the last entry of each
  for (int i = max(prompt, 0) + threadIdx.x; i < hist; i += kThreads) {
    const int id = history[i];
    if (id >= v0 && id < v1) atomicAdd(count + (id - v0), 1);
  }
  for (int i = bias0 + threadIdx.x; i < bias1; i += kThreads) {
    const int id = p.bias_ids[i];
    if (id >= v0 && id < v1) atomicMax(entry + (id - v0), i);
  }
  __syncthreads();

  const float rep = p.repetition ? p.repetition[b] : 1.0f;
  const float pres = p.presence ? p.presence[b] : 0.0f;
  const float freq = p.frequency ? p.frequency[b] : 0.0f;
  const uint32_t* allowed = nullptr;
  if (p.allowed) {
    const int row = p.allowed_rows ? p.allowed_rows[b] : b;   // negative: the row has no mask
    if (row >= p.masks) {
      if (lead && p.dev_err) atomicOr(p.dev_err, ANVILQ_DEV_ERR_SEQLEN);
    } else if (row >= 0) {
      allowed = p.allowed + row * p.allowed_ld;
    }
  }
  const T* x = static_cast<const T*>(p.x) + b * p.ld;
  float* out = p.out ? p.out + b * p.out_ld : nullptr;
  unsigned long long best = 0ull;
  for (int v = v0 + VEC * threadIdx.x; v < v1; v += VEC * kThreads) {
    float l[VEC];
    if (VEC == 4 && v + 4 <= v1) {
      if (sizeof(T) == 4) {
        const float4 w = *reinterpret_cast<const float4*>(x + v);
        l[0] = w.x; l[1 % VEC] = w.y; l[2 % VEC] = w.z; l[3 % VEC] = w.w;
      } else {
        const uint2 w = *reinterpret_cast<const uint2*>(x + v);
        const float2 a = __half22float2(*reinterpret_cast<const __half2*>(&w.x));
        const float2 c = __half22float2(*reinterpret_cast<const __half2*>(&w.y));
        l[0] = a.x; l[1 % VEC] = a.y; l[2 % VEC] = c.x; l[3 % VEC] = c.y;
      }
    } else {
#pragma unroll
      for (int e = 0; e < VEC; ++e) l[e] = v + e < v1 ? to_float<T>(x[v + e]) : 0.0f;
    }
    const int at = v - v0;
    const uint32_t s = seen[at / 32] >> (at % 32), z = biased[at / 32] >> (at % 32);
    const uint32_t a = allowed ? allowed[v / 32] >> (v % 32) : 0xFFFFFFFFu;
#pragma unroll
    for (int e = 0; e < VEC; ++e) {
      if (s >> e & 1u) {
        l[e] = l[e] > 0.0f ? __fdiv_rn(l[e], rep) : __fmul_rn(l[e], rep);
        const int n = count[at + e];
        if (n > 0) l[e] = __fsub_rn(__fsub_rn(l[e], __fmul_rn(freq, (float)n)), pres);
      }
      if (z >> e & 1u) l[e] = __fadd_rn(l[e], p.bias_values[entry[at + e]]);
      if (!(a >> e & 1u)) l[e] = -INFINITY;
      if (v + e < v1) {
        const unsigned long long k = choice_key(l[e], v + e);
        best = k > best ? k : best;
      }
    }
    if (out) {
      if (VEC == 4 && v + 4 <= v1) {
        *reinterpret_cast<float4*>(out + v) = make_float4(l[0], l[1 % VEC], l[2 % VEC], l[3 % VEC]);
      } else {
#pragma unroll
        for (int e = 0; e < VEC; ++e)
          if (v + e < v1) out[v + e] = l[e];
      }
    }
  }
  if (!p.token) return;
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) {
    const unsigned long long other = __shfl_xor_sync(0xffffffffu, best, o);
    best = other > best ? other : best;
  }
  if (threadIdx.x % 32 == 0) s_best[threadIdx.x / 32] = best;
  __syncthreads();
  if (threadIdx.x == 0) {
    for (int w = 1; w < kThreads / 32; ++w) best = s_best[w] > best ? s_best[w] : best;
    if (best) atomicMax(p.keys + b, best);
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
  int s = 4096;
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
  const size_t smem = p.stretch / 32 * 8 + (size_t)p.stretch * 4 * (bias_starts ? 2 : 1);
  const bool wide = aligned(logits, logits_half ? 8 : 16) && logits_stride % 4 == 0 &&
                    (!out || (aligned(out, 16) && out_stride % 4 == 0));
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
  const cudaError_t e = logits_half ? (wide ? cudaLaunchKernelEx(&cfg, logits_kernel<__half, 4>, p)
                                            : cudaLaunchKernelEx(&cfg, logits_kernel<__half, 1>, p))
                                    : (wide ? cudaLaunchKernelEx(&cfg, logits_kernel<float, 4>, p)
                                            : cudaLaunchKernelEx(&cfg, logits_kernel<float, 1>, p));
  if (e != cudaSuccess) {
    cudaGetLastError();
    return ANVILQ_ECUDA;
  }
  return ANVILQ_OK;
}

}  // extern "C"
