// gqa_decode_q8.cu -- GQA decode attention over a paged cache held in 8 bits with a
// scale for each block of 16 tokens and kv head (kv_q8.cuh).
//
// Mathematics.  Query token i of sequence b (Q of them, at positions
// seqlens[b] - Q + i) sees the positions t up to its own:
//   out = sum_t softmax_t(q . kc_t ks_t * scale) vc_t vs_t
// with integer or e4m3 codes kc, vc and their blocks' scales ks, vs.  A query
// that sees nothing (an empty sequence, or a position below 0) gives zeros.
#include <cmath>

#include "kv_q8.cuh"

namespace anvilq {
namespace attn8 {

using q8::kBlock;
constexpr int kWarps = 8;

struct Params {
  const __half* q;             // [B][Q][Hq][D]
  const uint8_t* k;            // codes [num_pages][Hkv][page_tokens][D]
  const uint8_t* v;
  const float* k_scales;       // [num_pages][Hkv][page_tokens / 16]
  const float* v_scales;
  const uint32_t* page_table;  // [B][max_pages]
  const int* seqlens;          // [B]
  __half* out;                 // [B][Q][Hq][D]
  int* dev_err;
  int B, Q, Hq, Hkv, page_tokens, max_pages, num_pages;
  float scale_log2;            // softmax scale * log2(e)
};

// One CTA a (query token, query head); its warps take blocks of 16 tokens in turn.
template <int D, int TYPE>
__global__ void __launch_bounds__(kWarps * 32) simple_kernel(const __grid_constant__ Params p) {
  constexpr int E = D / 32;    // dims of a lane
  __shared__ float s_state[kWarps][D + 2];
  asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
  asm volatile("griddepcontrol.wait;" ::: "memory");
  const int warp = threadIdx.x / 32, lane = threadIdx.x % 32;
  const int head = blockIdx.x, i = blockIdx.y, b = blockIdx.z, kvh = head / (p.Hq / p.Hkv);
  int len = p.seqlens[b];
  if (len < 0 || len > (long long)p.page_tokens * p.max_pages) {
    if (threadIdx.x == 0) atomicOr(p.dev_err, ANVILQ_DEV_ERR_SEQLEN);
    len = 0;
  }
  const int sees = len - p.Q + 1 + i;
  const size_t at = (((size_t)b * p.Q + i) * p.Hq + head) * D;
  float q[E], o[E] = {}, m = -INFINITY, l = 0.0f;
  for (int e = 0; e < E; ++e) q[e] = __half2float(p.q[at + lane + 32 * e]);
  for (int t0 = warp * kBlock; t0 < sees; t0 += kWarps * kBlock) {
    const int page = q8::page_of(p.page_table, p.max_pages, p.num_pages, b, t0 / p.page_tokens);
    if (page < 0) {
      if (lane == 0) atomicOr(p.dev_err, ANVILQ_DEV_ERR_PAGE);
      break;
    }
    const size_t run = (size_t)page * p.Hkv + kvh;
    const size_t block = run * (p.page_tokens / kBlock) + t0 % p.page_tokens / kBlock;
    const float ks = p.k_scales[block] * p.scale_log2, vs = p.v_scales[block];
    const uint8_t* kr = p.k + block * kBlock * D;
    const uint8_t* vr = p.v + block * kBlock * D;
    for (int t = 0; t < min(kBlock, sees - t0); ++t) {
      float s = 0.0f, f[4];
      for (int e = 0; e < E; ++e) {
        q8::codes_to_float4<TYPE>(kr[t * D + lane + 32 * e], f);
        s = fmaf(q[e], f[0], s);
      }
      for (int w = 16; w > 0; w >>= 1) s += __shfl_xor_sync(0xffffffffu, s, w);
      s *= ks;
      const float m_new = fmaxf(m, s);
      const float old = m == -INFINITY ? 0.0f : exp2f(m - m_new), pr = exp2f(s - m_new);
      l = l * old + pr;
      m = m_new;
      for (int e = 0; e < E; ++e) {
        q8::codes_to_float4<TYPE>(vr[t * D + lane + 32 * e], f);
        o[e] = fmaf(o[e], old, pr * vs * f[0]);
      }
    }
  }
  for (int e = 0; e < E; ++e) s_state[warp][lane + 32 * e] = o[e];
  if (lane == 0) {
    s_state[warp][D] = m;
    s_state[warp][D + 1] = l;
  }
  __syncthreads();
  if (threadIdx.x < D) {
    float M = -INFINITY, L = 0.0f, acc = 0.0f;
    for (int w = 0; w < kWarps; ++w) M = fmaxf(M, s_state[w][D]);
    for (int w = 0; w < kWarps; ++w) {
      const float f = s_state[w][D] == -INFINITY ? 0.0f : exp2f(s_state[w][D] - M);
      L += f * s_state[w][D + 1];
      acc += f * s_state[w][threadIdx.x];
    }
    p.out[at + threadIdx.x] = __float2half_rn(L > 0.0f ? acc / L : 0.0f);
  }
}

static bool a16(const void* p) { return (reinterpret_cast<uintptr_t>(p) & 15u) == 0; }

constexpr int kMaxQueries = 64;   // query tokens of a sequence
static bool shape_ok(int B, int Q, int Hq, int Hkv, int D) {
  return B >= 1 && B <= 65535 && Q >= 1 && Q <= kMaxQueries && Hkv >= 1 && Hq >= Hkv && Hq % Hkv == 0 &&
         Hq <= 1024 && (D == 64 || D == 128);
}

}  // namespace attn8
}  // namespace anvilq

extern "C" {

size_t anvilq_gqa_decode_q8_workspace_size(int B, int Q, int Hq, int Hkv, int D) {
  using namespace anvilq::attn8;
  if (!shape_ok(B, Q, Hq, Hkv, D)) return 0;
  return ANVILQ_WORKSPACE_COUNTER_BYTES;
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
  if (!a16(q) || !a16(k_codes) || !a16(v_codes) || !a16(out)) return ANVILQ_EALIGN;
  if (!workspace || workspace_bytes < anvilq_gqa_decode_q8_workspace_size(B, Q, Hq, Hkv, D)) return ANVILQ_EWORKSPACE;
  if (!a16(workspace)) return ANVILQ_EALIGN;
  Params p{};
  p.q = reinterpret_cast<const __half*>(q);
  p.k = static_cast<const uint8_t*>(k_codes);
  p.v = static_cast<const uint8_t*>(v_codes);
  p.k_scales = k_scales;
  p.v_scales = v_scales;
  p.page_table = page_table;
  p.seqlens = seqlens;
  p.out = reinterpret_cast<__half*>(out);
  p.dev_err = dev_err;
  p.B = B; p.Q = Q; p.Hq = Hq; p.Hkv = Hkv;
  p.page_tokens = page_tokens; p.max_pages = max_pages; p.num_pages = num_pages;
  p.scale_log2 = (scale > 0.0f ? scale : 1.0f / std::sqrt((float)D)) * 1.4426950408889634f;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(Hq, Q, B);
  cfg.blockDim = dim3(kWarps * 32);
  cfg.stream = reinterpret_cast<cudaStream_t>(stream);
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = attr;
  cfg.numAttrs = (flags & ANVILQ_GEMM_OVERLAP_PRIOR) ? 1 : 0;
  const bool int8 = code_type == ANVILQ_KV_Q8_INT8;
  const cudaError_t e =
      D == 64 ? (int8 ? cudaLaunchKernelEx(&cfg, simple_kernel<64, q8::kInt8>, p)
                      : cudaLaunchKernelEx(&cfg, simple_kernel<64, q8::kE4m3>, p))
              : (int8 ? cudaLaunchKernelEx(&cfg, simple_kernel<128, q8::kInt8>, p)
                      : cudaLaunchKernelEx(&cfg, simple_kernel<128, q8::kE4m3>, p));
  if (e != cudaSuccess) {
    cudaGetLastError();
    return ANVILQ_ECUDA;
  }
  return ANVILQ_OK;
}

}  // extern "C"
