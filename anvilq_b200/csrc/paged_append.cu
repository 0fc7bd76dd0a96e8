// paged_append.cu -- appending the new tokens of a ragged batch to a paged KV
// cache, with the position rotation of q and k on the way: binary16 pages (the
// pools of anvilq_gqa_decode_paged) or 8-bit pages (kv_q8.cuh).
//
// Mathematics.  Row t of qkv is a new token of sequence b at position p.  With
// angle_i = fp32(p * theta^(-2i/D)) (binary64 product, as anvilq_rope_kv_append),
// every q and k head is rotated in split halves,
//   a' = a cos angle_i - b sin angle_i,  b' = b cos angle_i + a sin angle_i
// (a = x[i], b = x[i + D/2]; binary32, each operation rounded), q goes to q_out in
// binary16, k' and v to row p % page_tokens of page page_table[b][p / page_tokens].
// 8-bit pages: a block of 16 tokens and a head share a scale s,
//   s = max(s_kept, scale_for(largest |value| of the block's new rows)),
//   code = round(value * fp32(1 / s)),
// s_kept being the scale of rows already in the block (0 where the block starts
// with a new row).  Where s > s_kept the kept rows are re-coded,
//   code' = round(code * fp32(s_kept / s)).
// Values are coded from binary32, not from a binary16 rounding of them.
//
// What bounds it: bytes (2 B in, 2 or 1 B out for every element; a few binary32
// operations each), and for a decode step, one token a sequence, the latency of
// the chain search -> page-table word -> row -> store.
//
// Work split: an item is the run of new rows of one sequence inside one block of
// 16 positions (the unit of a scale; it never leaves a page), and a slice of the
// heads.  A CTA computes the item's cosines and sines once, into shared memory.
// For rows that are copied or rotated into binary16 a thread keeps one row and 8
// consecutive dims of both halves, their cosines and sines in registers, and goes
// from head to head, several heads' loads ahead (dealing rows to threads in the
// order of memory instead, cosines read from shared memory each time, took 1.9
// times the instructions and was bound by them).  A
// block that is coded needs its largest value first, so a warp takes all of a
// head's rows, keeps them as they came (binary16) and rotates them twice, which
// costs fewer registers than it saves time to keep them rotated; of a decode step's
// items, a row or two, it takes several heads at once.
#include <algorithm>
#include <cmath>
#include <iterator>

#include "kv_q8.cuh"

namespace anvilq {
namespace append {

using q8::kBlock;
using q8::overlap;
constexpr int kBinary16 = -1;   // the pool's type: binary16, q8::kInt8 or q8::kE4m3
constexpr int kThreads = 128;
constexpr int kWarps = kThreads / 32;
constexpr int kMaxPairs = 64;   // D <= 128

struct Freq {
  double inv[kMaxPairs];   // theta^(-2i/D), binary64, computed on the host
};

struct Params {
  const __half* qkv;            // [T] rows of (Hq + 2 Hkv) D, `stride` elements apart
  long long stride;
  const int* starts;            // [B + 1]
  const int* seqlens;           // [B], the new tokens counted
  const uint32_t* page_table;   // [B][max_pages]
  __half* q_out;                // [T][Hq][D]
  void* k;
  void* v;
  float* k_scales;
  float* v_scales;
  int* dev_err;
  int T, B, Hq, Hkv, page_tokens, max_pages, num_pages;
  int by_token;                 // how blockIdx.x names an item, see find_item
  int heads_per_cta;
};

// The item of a CTA: rows [row, row + count) of qkv, positions pos .. of sequence b.
struct Item {
  int b, row, pos, count;
};

// Two ways to number the items without a pass over the batch, the host taking
// the one with fewer numbers (a number without an item ends its CTA):
//   by token: number t names the item whose first row is t, if t is one;
//   by place: sequence b's items follow from starts[b] / 16 + 2 b on (its n rows
//             lie in at most n / 16 + 2 blocks, so the ranges are disjoint).
// The whole warp looks for the largest b with key(b) <= number, key non-decreasing:
// 32 probes a step, and with the last step's probes come every candidate's lengths.
__device__ __forceinline__ Item find_item(const Params& p, int number) {
  const int lane = threadIdx.x % 32;
  const Item none{0, 0, 0, 0};
  int lo = 0, span = p.B;
  while (span > 31) {
    const int step = (span + 31) / 32, at = lane * step;
    bool le = false;
    if (at < span) {
      const int s = p.starts[lo + at];
      le = (p.by_token ? s : s / kBlock + 2 * (lo + at)) <= number;
    }
    const uint32_t hit = __ballot_sync(0xffffffffu, le);
    const int k = hit ? 31 - __clz(hit) : 0;
    lo += k * step;
    span = min(step, span - k * step);
  }
  const int mine = lane <= span ? p.starts[lo + lane] : 0;   // span <= 31: the end of the last one too
  const int my_len = lane < span ? p.seqlens[lo + lane] : 0;
  const bool le = lane < span && (p.by_token ? mine : mine / kBlock + 2 * (lo + lane)) <= number;
  const uint32_t hit = __ballot_sync(0xffffffffu, le);
  const int k = hit ? 31 - __clz(hit) : 0, b = lo + k;
  const int s0 = __shfl_sync(0xffffffffu, mine, k), s1 = __shfl_sync(0xffffffffu, mine, k + 1);
  const int len = __shfl_sync(0xffffffffu, my_len, k);
  if (s1 <= s0) return none;
  const long long first = (long long)len - ((long long)s1 - s0);   // position of row s0
  if (s0 < 0 || s1 > p.T || first < 0 || len > (long long)p.page_tokens * p.max_pages) {
    if (threadIdx.x == 0) atomicOr(p.dev_err, ANVILQ_DEV_ERR_SEQLEN);
    return none;
  }
  const int p0 = (int)first;
  int pos;
  if (p.by_token) {
    if (number < s0 || number >= s1) return none;
    pos = p0 + (number - s0);
    if (number != s0 && pos % kBlock) return none;
  } else {
    const int nth = number - (s0 / kBlock + 2 * b);
    const int block = p0 / kBlock + nth;
    if (nth < 0 || block > (len - 1) / kBlock) return none;
    pos = max(p0, block * kBlock);
  }
  return Item{b, s0 + (pos - p0), pos, min(len, (pos / kBlock + 1) * kBlock) - pos};
}

__device__ __forceinline__ void unpack8(const uint4& w, float* v) {
  const __half2* h = reinterpret_cast<const __half2*>(&w);
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const float2 f = __half22float2(h[i]);
    v[2 * i] = f.x;
    v[2 * i + 1] = f.y;
  }
}
__device__ __forceinline__ uint4 pack8(const float* v) {
  uint4 w;
  __half2* h = reinterpret_cast<__half2*>(&w);
#pragma unroll
  for (int i = 0; i < 4; ++i) h[i] = __floats2half2_rn(v[2 * i], v[2 * i + 1]);
  return w;
}

__device__ __forceinline__ void load8(const float* src, float* v) {   // 16-byte aligned
  const float4 a = *reinterpret_cast<const float4*>(src), b = *reinterpret_cast<const float4*>(src + 4);
  v[0] = a.x; v[1] = a.y; v[2] = a.z; v[3] = a.w;
  v[4] = b.x; v[5] = b.y; v[6] = b.z; v[7] = b.w;
}
// 8 dims of both halves of a row, rotated: (a, b) -> (a cos - b sin, b cos + a sin)
__device__ __forceinline__ void rotate8(float* a, float* b, const float* co, const float* si) {
#pragma unroll
  for (int e = 0; e < 8; ++e) {
    const float u = a[e], v = b[e];
    a[e] = __fsub_rn(__fmul_rn(u, co[e]), __fmul_rn(v, si[e]));
    b[e] = __fadd_rn(__fmul_rn(v, co[e]), __fmul_rn(u, si[e]));
  }
}

// FEW: with a path for items of a row or two (run has the rule)
template <int D, int TYPE, bool FEW>
__global__ void __launch_bounds__(kThreads, TYPE == kBinary16 ? 8 : 5)
    append_kernel(const __grid_constant__ Params p, const __grid_constant__ Freq freq) {
  constexpr int kHalf = D / 2;
  constexpr int kLanes = D / 16;              // threads of a row: 8 dims of each half a thread
  __shared__ __align__(16) float s_cos[kBlock][kHalf];
  __shared__ __align__(16) float s_sin[kBlock][kHalf];
  asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
  asm volatile("griddepcontrol.wait;" ::: "memory");
  const Item it = find_item(p, blockIdx.x);
  if (it.count <= 0) return;   // the same for the whole CTA
  const int heads = p.Hq + 2 * p.Hkv;
  const int head0 = blockIdx.y * p.heads_per_cta, head1 = min(heads, head0 + p.heads_per_cta);
  // rows into binary16: q, and with binary16 pages k and v.  The threads of a head
  // are a power of two of rows; the other threads take other heads.
  const int end16 = TYPE == kBinary16 ? head1 : min(head1, p.Hq);
  const int log_rows = 32 - __clz(it.count - 1);   // 0 for one row
  const int d16 = 8 * (threadIdx.x % kLanes), r16 = (threadIdx.x / kLanes) & ((1 << log_rows) - 1);
  const int step = (kThreads / kLanes) >> log_rows;
  const __half* src16 = p.qkv + (size_t)(it.row + r16) * p.stride + d16;
  constexpr int kAhead = 3;   // heads a thread loads at a time
  uint4 lo[kAhead], hi[kAhead];
  auto load = [&](int h0) {
#pragma unroll
    for (int k = 0; k < kAhead; ++k)
      if (r16 < it.count && h0 + k * step < end16) {
        lo[k] = *reinterpret_cast<const uint4*>(src16 + (h0 + k * step) * D);
        hi[k] = *reinterpret_cast<const uint4*>(src16 + (h0 + k * step) * D + kHalf);
      }
  };
  int h0 = head0 + ((threadIdx.x / kLanes) >> log_rows);
  load(h0);   // the first heads' rows travel with the page-table word, while the cosines are computed

  const int page = q8::page_of(p.page_table, p.max_pages, p.num_pages, it.b, it.pos / p.page_tokens);
  for (int i = threadIdx.x; i < it.count * kHalf; i += kThreads) {
    const int r = i / kHalf, pair = i % kHalf;
    const float angle = (float)((double)(it.pos + r) * freq.inv[pair]);
    sincosf(angle, &s_sin[r][pair], &s_cos[r][pair]);
  }
  if (page < 0) {
    if (threadIdx.x == 0) atomicOr(p.dev_err, ANVILQ_DEV_ERR_PAGE);
    return;
  }
  __syncthreads();
  const int slot = it.pos % p.page_tokens;    // row of the page of the item's first token
  {
    float co[8], si[8];
    load8(s_cos[r16] + d16, co);   // of a row behind the item's: not used
    load8(s_sin[r16] + d16, si);
#pragma unroll 1
    for (; h0 < end16; h0 += kAhead * step) {
#pragma unroll
      for (int k = 0; k < kAhead; ++k) {
        const int head = h0 + k * step;
        if (r16 >= it.count || head >= end16) break;
        if (TYPE != kBinary16 || head < p.Hq + p.Hkv) {
          float a[8], b[8];
          unpack8(lo[k], a);
          unpack8(hi[k], b);
          rotate8(a, b, co, si);
          lo[k] = pack8(a);
          hi[k] = pack8(b);
        }
        __half* dst;
        if (TYPE != kBinary16 || head < p.Hq) {
          dst = p.q_out + ((size_t)(it.row + r16) * p.Hq + head) * D + d16;
        } else {
          const bool is_k = head < p.Hq + p.Hkv;
          dst = static_cast<__half*>(is_k ? p.k : p.v) +
                (((size_t)page * p.page_tokens + slot + r16) * p.Hkv + head - p.Hq - (is_k ? 0 : p.Hkv)) * D + d16;
        }
        *reinterpret_cast<uint4*>(dst) = lo[k];
        *reinterpret_cast<uint4*>(dst + kHalf) = hi[k];
      }
      load(h0 + kAhead * step);
    }
  }
  if (TYPE == kBinary16) return;

  // ---- blocks into codes ----
  constexpr int kCode = TYPE == q8::kE4m3 ? q8::kE4m3 : q8::kInt8;
  constexpr int kRows = 32 / kLanes;          // rows of a pass of a warp
  constexpr int kPasses = kBlock / kRows;
  const int warp = threadIdx.x / 32, lane = threadIdx.x % 32, r0 = lane / kLanes, d0 = 8 * (lane % kLanes);
  const int kept = it.pos % kBlock;           // rows of the block that were there before
  auto finite = [](float v) { return fabsf(v) <= 3.4028234664e38f ? v : 0.0f; };
  // the block's earlier codes in the lane's dims, rows first, first + step ..., times ratio
  auto recode = [&](uint8_t* rows, int first, int step, float ratio) {
#pragma unroll 1
    for (int r = first; r < kept; r += step) {
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        uint2* at = reinterpret_cast<uint2*>(rows + r * D + d0 + h * kHalf);
        uint2 w = *at;
        float v[8];
        q8::codes_to_float4<kCode>(w.x, v);
        q8::codes_to_float4<kCode>(w.y, v + 4);
#pragma unroll
        for (int e = 0; e < 8; ++e) v[e] *= ratio;
        *at = make_uint2(q8::float4_to_codes<kCode>(v), q8::float4_to_codes<kCode>(v + 4));
      }
    }
  };
  if (FEW && 2 * it.count <= kRows) {
    // A new token or two, as in a decode step: the lanes that share a pass's rows below
    // share heads here.
    const int row = r0 & ((1 << log_rows) - 1), heads_per_warp = kRows >> log_rows;
#pragma unroll 1
    for (int h0 = max(head0, p.Hq) + warp * heads_per_warp; h0 < head1; h0 += kWarps * heads_per_warp) {
      const int head = h0 + (r0 >> log_rows);
      const bool live = head < head1, mine = live && row < it.count, is_k = head < p.Hq + p.Hkv;
      const size_t run = (size_t)page * p.Hkv + head - p.Hq - (is_k ? 0 : p.Hkv);
      float* scale_at = (is_k ? p.k_scales : p.v_scales) + run * (p.page_tokens / kBlock) + slot / kBlock;
      uint8_t* rows = static_cast<uint8_t*>(is_k ? p.k : p.v) + (run * p.page_tokens + (slot - kept)) * D;
      uint4 a = make_uint4(0, 0, 0, 0), b = a;
      float s_kept = 0.0f;
      if (mine) {
        const __half* src = p.qkv + (size_t)(it.row + row) * p.stride + head * D + d0;
        a = *reinterpret_cast<const uint4*>(src);
        b = *reinterpret_cast<const uint4*>(src + kHalf);
      }
      if (live && kept) s_kept = *scale_at;
      float x[16];
      unpack8(a, x);
      unpack8(b, x + 8);
      if (is_k && mine) {
        float co[8], si[8];
        load8(s_cos[row] + d0, co);
        load8(s_sin[row] + d0, si);
        rotate8(x, x + 8, co, si);
      }
      float top = 0.0f, probe = 0.0f;   // probe: NaN after a value that is not finite
#pragma unroll
      for (int e = 0; e < 16; ++e) {
        top = fmaxf(top, fabsf(x[e]));
        probe = fmaf(x[e], 0.0f, probe);
      }
      if (__any_sync(0xffffffffu, probe != 0.0f)) {   // stored as 0, and reported
        if (lane == 0) atomicOr(p.dev_err, ANVILQ_DEV_ERR_NONFINITE);
        top = 0.0f;
#pragma unroll
        for (int e = 0; e < 16; ++e) {
          x[e] = finite(x[e]);
          top = fmaxf(top, fabsf(x[e]));
        }
      }
#pragma unroll
      for (int o = kRows * kLanes / 4; o > 0; o >>= 1)
        if (o < kLanes << log_rows) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, o));
      __syncwarp();   // every lane has read its head's scale, which one of them replaces
      if (live) {
        const float s = fmaxf(s_kept, q8::scale_for<kCode>(top));
        const float inv = s > 0.0f ? __fdiv_rn(1.0f, s) : 0.0f;
        if (kept && s > s_kept) recode(rows, row, 1 << log_rows, __fdiv_rn(s_kept, s));
#pragma unroll
        for (int e = 0; e < 16; ++e) x[e] *= inv;
        if (mine)
#pragma unroll
          for (int h = 0; h < 2; ++h)
            *reinterpret_cast<uint2*>(rows + (kept + row) * D + d0 + h * kHalf) =
                make_uint2(q8::float4_to_codes<kCode>(x + 8 * h), q8::float4_to_codes<kCode>(x + 8 * h + 4));
        if (row == 0 && d0 == 0) *scale_at = s;
      }
    }
    return;
  }
#pragma unroll 1
  for (int head = max(head0, p.Hq) + warp; head < head1; head += kWarps) {
    const bool is_k = head < p.Hq + p.Hkv;
    const int kvh = head - p.Hq - (is_k ? 0 : p.Hkv);
    uint4 raw[kPasses][2];
    const __half* src = p.qkv + (size_t)(it.row + r0) * p.stride + head * D + d0;
#pragma unroll
    for (int i = 0; i < kPasses; ++i) {
      raw[i][0] = raw[i][1] = make_uint4(0, 0, 0, 0);
      if (i * kRows + r0 < it.count) {
        raw[i][0] = *reinterpret_cast<const uint4*>(src + (size_t)i * kRows * p.stride);
        raw[i][1] = *reinterpret_cast<const uint4*>(src + (size_t)i * kRows * p.stride + kHalf);
      }
    }
    auto values = [&](int i, float* x) {   // of pass i
      unpack8(raw[i][0], x);
      unpack8(raw[i][1], x + 8);
      if (is_k && i * kRows + r0 < it.count) {
        float co[8], si[8];
        load8(s_cos[i * kRows + r0] + d0, co);
        load8(s_sin[i * kRows + r0] + d0, si);
        rotate8(x, x + 8, co, si);
      }
    };
    float top = 0.0f, probe = 0.0f;   // probe: NaN after a value that is not finite
#pragma unroll
    for (int i = 0; i < kPasses; ++i) {
      if (i * kRows >= it.count) break;
      float x[16];
      values(i, x);
#pragma unroll
      for (int e = 0; e < 16; ++e) {
        top = fmaxf(top, fabsf(x[e]));
        probe = fmaf(x[e], 0.0f, probe);
      }
    }
    // such a value has no code: it is stored as 0, and reported
    const bool odd = __any_sync(0xffffffffu, probe != 0.0f);
    if (odd) {
      if (lane == 0) atomicOr(p.dev_err, ANVILQ_DEV_ERR_NONFINITE);
      top = 0.0f;
#pragma unroll
      for (int i = 0; i < kPasses; ++i) {
        float x[16];
        values(i, x);
#pragma unroll
        for (int e = 0; e < 16; ++e) top = fmaxf(top, fabsf(finite(x[e])));
      }
    }
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, o));
    const size_t run = (size_t)page * p.Hkv + kvh;
    float* scale_at = (is_k ? p.k_scales : p.v_scales) + run * (p.page_tokens / kBlock) + slot / kBlock;
    uint8_t* rows = static_cast<uint8_t*>(is_k ? p.k : p.v) + (run * p.page_tokens + (slot - kept)) * D;
    const float s_kept = kept ? *scale_at : 0.0f;
    const float s = fmaxf(s_kept, q8::scale_for<kCode>(top));
    const float inv = s > 0.0f ? __fdiv_rn(1.0f, s) : 0.0f;
    if (kept && s > s_kept) recode(rows, r0, kRows, __fdiv_rn(s_kept, s));
#pragma unroll
    for (int i = 0; i < kPasses; ++i) {
      const int r = i * kRows + r0;
      if (i * kRows >= it.count) break;
      float x[16];
      values(i, x);
      if (odd)
#pragma unroll
        for (int e = 0; e < 16; ++e) x[e] = finite(x[e]);
#pragma unroll
      for (int e = 0; e < 16; ++e) x[e] *= inv;
      if (r < it.count)
#pragma unroll
        for (int h = 0; h < 2; ++h)
          *reinterpret_cast<uint2*>(rows + (kept + r) * D + d0 + h * kHalf) =
              make_uint2(q8::float4_to_codes<kCode>(x + 8 * h), q8::float4_to_codes<kCode>(x + 8 * h + 4));
    }
    __syncwarp();   // every lane has read the scale
    if (lane == 0) *scale_at = s;
  }
}

// values[page][head][token][:] = fp16(code * scale), K's pool then V's: a thread
// takes 8 codes of a row at a time, so that a warp stores whole sectors, eight such
// pieces on their way.
template <int TYPE>
__global__ void __launch_bounds__(256) values_kernel(const uint8_t* k, const uint8_t* v, const float* ks,
                                                     const float* vs, __half* ko, __half* vo, long long pieces,
                                                     int pieces_per_block) {
  asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
  asm volatile("griddepcontrol.wait;" ::: "memory");
  constexpr int kAhead = 8;
  const bool second = blockIdx.y != 0;
  const uint2* codes = reinterpret_cast<const uint2*>(second ? v : k);
  const float* scales = second ? vs : ks;
  uint4* out = reinterpret_cast<uint4*>(second ? vo : ko);
  for (long long i0 = (long long)blockIdx.x * (kAhead * 256) + threadIdx.x; i0 < pieces;
       i0 += (long long)gridDim.x * (kAhead * 256)) {
    uint2 w[kAhead];
    float s[kAhead];
#pragma unroll
    for (int a = 0; a < kAhead; ++a) {
      const long long c = i0 + 256 * a;
      if (c < pieces) {
        w[a] = __ldcs(codes + c);
        s[a] = scales[c / pieces_per_block];
      }
    }
#pragma unroll
    for (int a = 0; a < kAhead; ++a) {
      const long long c = i0 + 256 * a;
      if (c >= pieces) break;
      float f[8];
      q8::codes_to_float4<TYPE>(w[a].x, f);
      q8::codes_to_float4<TYPE>(w[a].y, f + 4);
#pragma unroll
      for (int e = 0; e < 8; ++e) f[e] *= s[a];
      out[c] = pack8(f);
    }
  }
}

static bool a16(const void* p) { return (reinterpret_cast<uintptr_t>(p) & 15u) == 0; }

template <typename... KArgs, typename... Args>
static int launch(void (*kernel)(KArgs...), dim3 grid, int threads, cudaStream_t s, unsigned flags, Args... args) {
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = grid;
  cfg.blockDim = dim3(threads);
  cfg.stream = s;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = attr;
  cfg.numAttrs = (flags & ANVILQ_GEMM_OVERLAP_PRIOR) ? 1 : 0;
  if (cudaLaunchKernelEx(&cfg, kernel, args...) != cudaSuccess) {
    cudaGetLastError();
    return ANVILQ_ECUDA;
  }
  return ANVILQ_OK;
}

struct Span {
  const void* start;
  size_t bytes;
};

// type: kBinary16 or an ANVILQ_KV_Q8_* code type (scales then given)
static int run(const uint16_t* qkv, long long stride, const int32_t* starts, const int32_t* seqlens,
               const uint32_t* page_table, uint16_t* q_out, void* k, void* v, float* k_scales, float* v_scales,
               int type, int T, int B, int Hq, int Hkv, int D, int page_tokens, int max_pages, int num_pages,
               float theta, int* dev_err, unsigned flags, cudaStream_t st) {
  if ((T != 0 && (!qkv || !q_out)) || !starts || !seqlens || !page_table || !k || !v || !dev_err) return ANVILQ_EINVAL;
  if (type != kBinary16 && (!k_scales || !v_scales)) return ANVILQ_EINVAL;
  if (flags & ~(unsigned)ANVILQ_GEMM_OVERLAP_PRIOR) return ANVILQ_EINVAL;
  if (T < 0 || B < 1 || Hq < 1 || Hkv < 1 || Hq % Hkv || !(theta > 0.0f) || !std::isfinite(theta))
    return ANVILQ_EINVAL;
  if (type != kBinary16 && type != q8::kInt8 && type != q8::kE4m3) return ANVILQ_EINVAL;
  if ((D != 64 && D != 128) || page_tokens < kBlock || page_tokens % kBlock || max_pages < 1 || num_pages < 1 ||
      (long long)page_tokens * max_pages > (1LL << 30) || B > (1 << 24) || Hq > (1 << 16) || T > (1 << 30))
    return ANVILQ_ESHAPE;
  const int heads = Hq + 2 * Hkv;
  if (stride < (long long)heads * D) return ANVILQ_EINVAL;
  const long long positions = (long long)num_pages * page_tokens;
  if (positions > (1LL << 40) / Hkv) return ANVILQ_ESHAPE;
  if (!a16(qkv) || !a16(q_out) || !a16(k) || !a16(v) || stride % 8) return ANVILQ_EALIGN;
  if (T == 0) return ANVILQ_OK;
  // an item's q is written while others' rows are still to be read, and every pool by
  // warps of its own
  const size_t pool = (size_t)positions * Hkv * D * (type == kBinary16 ? 2 : 1);
  const size_t scales = type == kBinary16 ? 0 : (size_t)positions / kBlock * Hkv * sizeof(float);
  const Span spans[] = {{qkv, ((size_t)(T - 1) * stride + (size_t)heads * D) * 2}, {q_out, (size_t)T * Hq * D * 2},
                        {k, pool}, {v, pool}, {k_scales, scales}, {v_scales, scales}};
  for (const Span& a : spans)
    for (const Span* b = &a + 1; b != std::end(spans); ++b)
      if (overlap(a.start, a.bytes, b->start, b->bytes)) return ANVILQ_EINVAL;
  Params p{};
  p.qkv = reinterpret_cast<const __half*>(qkv);
  p.stride = stride;
  p.starts = starts;
  p.seqlens = seqlens;
  p.page_table = page_table;
  p.q_out = reinterpret_cast<__half*>(q_out);
  p.k = k;
  p.v = v;
  p.k_scales = k_scales;
  p.v_scales = v_scales;
  p.dev_err = dev_err;
  p.T = T; p.B = B; p.Hq = Hq; p.Hkv = Hkv;
  p.page_tokens = page_tokens; p.max_pages = max_pages; p.num_pages = num_pages;
  const long long by_place = T / kBlock + 2LL * B;
  p.by_token = T <= by_place;
  const int items = (int)(p.by_token ? (long long)T : by_place);
  // Slices of the heads, more than 4 heads each, only until there are four CTAs an SM
  // (three with 8-bit pages, whose CTAs take more registers): every slice looks up
  // its tokens and computes their cosines again.  32/8 heads of 128, one slice and
  // two: 560 items into binary16 47.5 and 39.9 us, 350 items into 8 bits 32.0 and
  // 24.8, but 538 items into 8 bits 38.1 and 41.8.
  const long long enough = 148 * (type == kBinary16 ? 4 : 3);
  // (Items are counted as if every sequence had one more than its rows fill, since
  // the lengths are on the device.)
  const long long likely = std::min<long long>(items, T / kBlock + B);
  int slices = 1;
  while (slices * 8 < heads && likely * slices < enough) slices *= 2;
  p.heads_per_cta = (heads + slices - 1) / slices;
  // the frequencies of the thread's last theta and D (64 powers cost the host 3 us)
  thread_local Freq freq;
  thread_local float freq_theta = 0.0f;
  thread_local int freq_d = 0;
  if (theta != freq_theta || D != freq_d) {
    for (int i = 0; i < D / 2; ++i) freq.inv[i] = std::pow((double)theta, -2.0 * i / D);
    freq_theta = theta;
    freq_d = D;
  }
  const dim3 grid(items, (heads + p.heads_per_cta - 1) / p.heads_per_cta);
  auto go = [&](auto kernel) { return launch(kernel, grid, kThreads, st, flags, p, Freq(freq)); };
  // Up to two tokens a sequence on average: the kernel that gives a warp several heads
  // of an item of few rows.  32/32 heads of 128: 1024 sequences of one token 16.4 us
  // against 50.3, of two 30.2 against 58.  It takes 10 % longer where items are full (4096
  // tokens of one sequence 44.2 against 38.6), though those items go the same way in both.
  const bool few = T <= 2LL * B;
  if (type == kBinary16)
    return D == 64 ? go(append_kernel<64, kBinary16, false>) : go(append_kernel<128, kBinary16, false>);
  if (D == 64)
    return type == q8::kInt8 ? (few ? go(append_kernel<64, q8::kInt8, true>) : go(append_kernel<64, q8::kInt8, false>))
                             : (few ? go(append_kernel<64, q8::kE4m3, true>) : go(append_kernel<64, q8::kE4m3, false>));
  return type == q8::kInt8 ? (few ? go(append_kernel<128, q8::kInt8, true>) : go(append_kernel<128, q8::kInt8, false>))
                           : (few ? go(append_kernel<128, q8::kE4m3, true>) : go(append_kernel<128, q8::kE4m3, false>));
}

}  // namespace append
}  // namespace anvilq

extern "C" {

int anvilq_paged_kv_append(const uint16_t* qkv, long long qkv_stride, const int32_t* token_starts,
                           const int32_t* seqlens, const uint32_t* page_table, uint16_t* q_out, uint16_t* k_pool,
                           uint16_t* v_pool, int T, int B, int Hq, int Hkv, int D, int page_tokens, int max_pages,
                           int num_pages, float theta, int* dev_err, unsigned flags, anvilq_stream_t stream) {
  using namespace anvilq::append;
  return run(qkv, qkv_stride, token_starts, seqlens, page_table, q_out, k_pool, v_pool, nullptr, nullptr, kBinary16,
             T, B, Hq, Hkv, D, page_tokens, max_pages, num_pages, theta, dev_err, flags,
             reinterpret_cast<cudaStream_t>(stream));
}

int anvilq_paged_kv_append_q8(const uint16_t* qkv, long long qkv_stride, const int32_t* token_starts,
                              const int32_t* seqlens, const uint32_t* page_table, uint16_t* q_out, void* k_codes,
                              void* v_codes, float* k_scales, float* v_scales, int code_type, int T, int B, int Hq,
                              int Hkv, int D, int page_tokens, int max_pages, int num_pages, float theta,
                              int* dev_err, unsigned flags, anvilq_stream_t stream) {
  using namespace anvilq::append;
  if (code_type != ANVILQ_KV_Q8_INT8 && code_type != ANVILQ_KV_Q8_E4M3) return ANVILQ_EINVAL;
  return run(qkv, qkv_stride, token_starts, seqlens, page_table, q_out, k_codes, v_codes, k_scales, v_scales,
             code_type, T, B, Hq, Hkv, D, page_tokens, max_pages, num_pages, theta, dev_err, flags,
             reinterpret_cast<cudaStream_t>(stream));
}

int anvilq_kv_q8_values(const void* k_codes, const void* v_codes, const float* k_scales, const float* v_scales,
                        int code_type, uint16_t* k_out, uint16_t* v_out, int num_pages, int Hkv, int page_tokens,
                        int D, unsigned flags, anvilq_stream_t stream) {
  using namespace anvilq::append;
  if (!k_codes || !v_codes || !k_scales || !v_scales || !k_out || !v_out) return ANVILQ_EINVAL;
  if (code_type != ANVILQ_KV_Q8_INT8 && code_type != ANVILQ_KV_Q8_E4M3) return ANVILQ_EINVAL;
  if (flags & ~(unsigned)ANVILQ_GEMM_OVERLAP_PRIOR) return ANVILQ_EINVAL;
  if (num_pages < 1 || Hkv < 1) return ANVILQ_EINVAL;
  if ((D != 64 && D != 128) || page_tokens < kBlock || page_tokens % kBlock) return ANVILQ_ESHAPE;
  if (!a16(k_codes) || !a16(v_codes) || !a16(k_out) || !a16(v_out)) return ANVILQ_EALIGN;
  const long long rows = (long long)num_pages * page_tokens;
  if (rows > (1LL << 40) / Hkv) return ANVILQ_ESHAPE;
  const long long pieces = rows * Hkv * (D / 8);
  const size_t values = pieces * 16, codes = pieces * 8;
  if (overlap(k_out, values, v_out, values) || overlap(k_out, values, k_codes, codes) ||
      overlap(k_out, values, v_codes, codes) || overlap(v_out, values, k_codes, codes) ||
      overlap(v_out, values, v_codes, codes))
    return ANVILQ_EINVAL;
  const int blocks = (int)std::min<long long>((pieces + 2047) / 2048, 148 * 8);
  auto go = [&](auto kernel) {
    return launch(kernel, dim3(blocks, 2), 256, reinterpret_cast<cudaStream_t>(stream), flags,
                  static_cast<const uint8_t*>(k_codes), static_cast<const uint8_t*>(v_codes), k_scales, v_scales,
                  reinterpret_cast<__half*>(k_out), reinterpret_cast<__half*>(v_out), pieces, kBlock * D / 8);
  };
  return code_type == ANVILQ_KV_Q8_INT8 ? go(values_kernel<ANVILQ_KV_Q8_INT8>) : go(values_kernel<ANVILQ_KV_Q8_E4M3>);
}

}  // extern "C"
