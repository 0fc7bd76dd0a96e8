// kv_pages.cu -- the pages of a paged KV cache as things that sequences share: table
// rows forked (beams, prompts that several answers share), pages made writable
// (allocated, or copied when shared), released, compacted and copied.
//
// State.  refs[p] counts the table entries that name page p; 0: the page is free.
// A table entry is a uint32, bit 31 valid, bits 30:0 the page.  Nothing else is kept,
// so the calls compose in any order and a captured graph replays on whatever state
// it finds.
//
// Definitions.  Free pages are taken lowest first, entries ask in (row, index) order:
//   fork      out[n] = table[parent(n)];  refs += entries of out - entries of table
//   reserve   of row b, the entries of positions before[b] .. after[b]:  absent -> a new
//             page; named by other entries too -> a new page, the rows below before[b]
//             copied.  In order, so where all that name a page ask, the last keeps it.
//   release   entries from ceil(keep[b] / page_tokens) on are dropped
//   compact   with n pages in use, those at n and above go to the free ones below n,
//             in order; a shared page stays shared
//
// What bounds it: the copies, by HBM (a page of every layer's pools); without copies
// the latency of a few dependent passes over small arrays.
//
// Work split.  A fork is a CTA a row: entry copies, and for the row's own entries one
// atomic add of (children - 1), none for a row with one child.  Reserve and compact
// plan in ONE CTA: their ranks are prefix sums over at most some 10^5 words, where
// passes by several CTAs would each cost a launch or a grid barrier, more than the
// words' reading takes.  The copies are a second launch of resident CTAs over (moved
// page, pool, piece), overlapping the plan's end.
//
// Measured: 64 rows forked and made writable with 64 pools of 128 KB pages (252 MB read and
// written) 53 us: fork and plan 9, copies 40; 96 rows released and 48 pools of 8 KB pages
// compacted (278 MB) 64 us, copies 45, 0.95 of a plain copy's bandwidth; four beams' fork
// with 4 KB pages 11 us, three launches' latency.
#include <algorithm>
#include <climits>
#include <initializer_list>
#include <iterator>

#include "kv_q8.cuh"

namespace anvilq {
namespace pages {

using q8::overlap;
constexpr int kPlan = 1024;            // threads of a planning CTA
constexpr int kMaxRows = 16384;        // rows of a table: their first entries' numbers lie in shared memory
constexpr int kMaxPools = 128;         // pools of one copy launch (more: several)
constexpr int kCopyThreads = 256;
constexpr int kAhead = 8;              // loads of a thread on their way
constexpr uint32_t kValid = 1u << 31;

// A moved page: rows < 0 means the whole page.
struct Move {
  int src, dst, rows;
};

__device__ __forceinline__ void prologue() {
  asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
  asm volatile("griddepcontrol.wait;" ::: "memory");
}

// Exclusive prefix sum over the CTA's threads; `total` is the whole sum.
__device__ __forceinline__ int block_scan(int v, int& total) {
  __shared__ int sums[kPlan / 32];
  const int lane = threadIdx.x % 32, warp = threadIdx.x / 32;
  int incl = v;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const int up = __shfl_up_sync(0xffffffffu, incl, o);
    if (lane >= o) incl += up;
  }
  if (lane == 31) sums[warp] = incl;
  __syncthreads();
  if (warp == 0) {
    const int s = sums[lane];
    int t = s;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const int up = __shfl_up_sync(0xffffffffu, t, o);
      if (lane >= o) t += up;
    }
    sums[lane] = t;
  }
  __syncthreads();
  total = sums[kPlan / 32 - 1];
  const int before = warp ? sums[warp - 1] : 0;
  __syncthreads();   // the sums are used again
  return before + incl - v;
}

// ---- fork ---------------------------------------------------------------------

struct Fork {
  const uint32_t* table;   // [old_rows][max_pages]
  uint32_t* out;           // [new_rows][max_pages]
  int* refs;
  const int* parents;      // [new_rows]; of new row n: (n / per_new) * per_old + parents[n]
  int* dev_err;
  int old_rows, new_rows, per_old, per_new, max_pages, num_pages;
};

__global__ void __launch_bounds__(256) fork_kernel(const __grid_constant__ Fork p) {
  prologue();
  const int r = blockIdx.x;
  bool bad_page = false;
  if (r < p.new_rows) {
    int parent = p.parents[r];
    if (parent < -1 || parent >= p.per_old) {
      if (threadIdx.x == 0) atomicOr(p.dev_err, ANVILQ_DEV_ERR_SEQLEN);
      parent = -1;
    }
    const uint32_t* from = p.table + ((size_t)(r / p.per_new) * p.per_old + max(parent, 0)) * p.max_pages;
    uint32_t* to = p.out + (size_t)r * p.max_pages;
    for (int j = threadIdx.x; j < p.max_pages; j += blockDim.x) {
      uint32_t e = parent < 0 ? 0 : from[j];
      if ((e & kValid) && (e & ~kValid) >= (uint32_t)p.num_pages) {
        bad_page = true;
        e = 0;
      }
      to[j] = e;
    }
  }
  if (r < p.old_rows) {
    const int first = r / p.per_old * p.per_new, me = r % p.per_old;
    int children = 0;
    for (int n0 = 0; n0 < p.per_new; n0 += blockDim.x) {
      const int n = n0 + threadIdx.x;
      children += __syncthreads_count(n < p.per_new && p.parents[first + n] == me);
    }
    const int change = children - 1;
    if (change)
      for (int j = threadIdx.x; j < p.max_pages; j += blockDim.x) {
        const uint32_t e = p.table[(size_t)r * p.max_pages + j];
        if (!(e & kValid)) continue;
        if ((e & ~kValid) < (uint32_t)p.num_pages)
          atomicAdd(p.refs + (e & ~kValid), change);
        else
          bad_page = true;
      }
  }
  if (bad_page) atomicOr(p.dev_err, ANVILQ_DEV_ERR_PAGE);
}

// ---- reserve --------------------------------------------------------------------

// Of a page that entries of this call will write: its references, how many of them
// are such entries, and the last of those (by number).
struct Writers {
  int refs, count, last, unused;
};

struct Reserve {
  uint32_t* table;        // [rows][max_pages]
  int* refs;              // [num_pages]
  const int* before;      // [rows]
  const int* after;
  int* lacking;           // [1]: pages that were missing
  Writers* writers;       // [num_pages], scratch
  int* free_pages;        // [num_pages], scratch
  Move* moves;            // [rows], scratch
  int* move_count;        // [1], scratch
  int* dev_err;
  int rows, max_pages, num_pages, page_tokens;
};

__global__ void __launch_bounds__(kPlan) reserve_kernel(const __grid_constant__ Reserve p) {
  extern __shared__ int first[];   // [rows + 1]: the number of a row's first entry
  prologue();
  const int tid = threadIdx.x;
  // ---- the entries that will be written, numbered in order ----
  int entries = 0;
  for (int b0 = 0; b0 < p.rows; b0 += kPlan) {
    const int b = b0 + tid;
    int n = 0;
    if (b < p.rows) {
      const int lo = p.before[b], hi = p.after[b];
      if (lo < 0 || hi > (long long)p.page_tokens * p.max_pages)
        atomicOr(p.dev_err, ANVILQ_DEV_ERR_SEQLEN);
      else if (hi > lo)
        n = (hi - 1) / p.page_tokens - lo / p.page_tokens + 1;
    }
    int total;
    const int at = block_scan(n, total);
    if (b < p.rows) first[b] = entries + at;
    entries += total;
  }
  if (tid == 0) first[p.rows] = entries;
  __syncthreads();
  struct Entry {
    int b, j, page;   // page: -1 absent, -2 not an entry (or one out of range)
  };
  auto entry = [&](int e) {
    if (e >= entries) return Entry{0, 0, -2};
    int lo = 0, hi = p.rows;   // first[lo] <= e < first[hi]
    while (hi - lo > 1) {
      const int mid = (lo + hi) / 2;
      if (first[mid] <= e) lo = mid; else hi = mid;
    }
    Entry x{lo, p.before[lo] / p.page_tokens + (e - first[lo]), -1};
    const uint32_t w = p.table[(size_t)x.b * p.max_pages + x.j];
    if (w & kValid) x.page = (w & ~kValid) < (uint32_t)p.num_pages ? (int)(w & ~kValid) : -2;
    return x;
  };
  // ---- who writes which page ----
  for (int e = tid; e < entries; e += kPlan) {
    const Entry x = entry(e);
    const int refs = x.page >= 0 ? p.refs[x.page] : 0;
    if (x.page == -2 || (x.page >= 0 && refs < 1)) atomicOr(p.dev_err, ANVILQ_DEV_ERR_PAGE);
    if (x.page >= 0) p.writers[x.page] = Writers{refs, 0, -1, 0};   // the same by all
  }
  __syncthreads();
  for (int e = tid; e < entries; e += kPlan) {
    const Entry x = entry(e);
    if (x.page < 0) continue;
    atomicAdd(&p.writers[x.page].count, 1);
    atomicMax(&p.writers[x.page].last, e);
  }
  __syncthreads();
  // an entry that needs a new page, and whether it has one already
  auto needs = [&](const Entry& x, int e) {
    if (x.page < 0) return x.page == -1;
    const Writers w = p.writers[x.page];
    return w.refs > 1 && w.refs >= w.count && !(w.refs == w.count && w.last == e);   // (below: miscounted, passed over)
  };
  int wanted = 0;
  for (int e0 = 0; e0 < entries; e0 += kPlan) {
    const int e = e0 + tid;
    const Entry x = entry(e);
    if (x.page >= 0 && p.writers[x.page].refs < p.writers[x.page].count) atomicOr(p.dev_err, ANVILQ_DEV_ERR_PAGE);
    wanted += __syncthreads_count(needs(x, e));
  }
  // ---- that many of the free pages, the lowest ----
  int found = 0;
  constexpr int kEach = 16;   // pages of a thread at a time
  for (int p0 = 0; p0 < p.num_pages && found < wanted; p0 += kPlan * kEach) {
    int free = 0;   // a bit a page
#pragma unroll
    for (int i = 0; i < kEach; ++i) {
      const int page = p0 + tid * kEach + i;
      if (page < p.num_pages && p.refs[page] == 0) free |= 1 << i;
    }
    int total;
    int at = found + block_scan(__popc(free), total);
    for (; free && at < wanted; free &= free - 1) p.free_pages[at++] = p0 + tid * kEach + __ffs(free) - 1;
    found += total;
  }
  const bool enough = found >= wanted;
  if (tid == 0) {
    *p.lacking = enough ? 0 : wanted - found;
    if (!enough) {
      atomicOr(p.dev_err, ANVILQ_DEV_ERR_NOPAGE);
      *p.move_count = 0;
    }
  }
  if (!enough) return;   // nothing is changed
  __syncthreads();
  // ---- handed out ----
  int given = 0, moves = 0;
  for (int e0 = 0; e0 < entries; e0 += kPlan) {
    const int e = e0 + tid;
    const Entry x = entry(e);
    const bool need = needs(x, e);
    const int rows = need ? p.before[x.b] - x.j * p.page_tokens : 0;   // that were there before
    const bool move = need && x.page >= 0 && rows > 0;
    int total;
    const int at = block_scan((need ? 1 : 0) | (move ? 1 << 16 : 0), total);   // both fit: at most 1024 each
    if (need) {
      const int page = p.free_pages[given + (at & 0xffff)];
      p.table[(size_t)x.b * p.max_pages + x.j] = (uint32_t)page | kValid;
      p.refs[page] = 1;
      if (x.page >= 0) atomicSub(p.refs + x.page, 1);
      if (move) p.moves[moves + (at >> 16)] = Move{x.page, page, rows};
    }
    given += total & 0xffff;
    moves += total >> 16;
  }
  if (tid == 0) *p.move_count = moves;
}

// ---- release --------------------------------------------------------------------

struct Release {
  uint32_t* table;
  int* refs;
  const int* keep;
  int* dev_err;
  int max_pages, num_pages, page_tokens;
};

__global__ void __launch_bounds__(256) release_kernel(const __grid_constant__ Release p) {
  prologue();
  const int b = blockIdx.x, keep = p.keep[b];
  if (keep < 0) {
    if (threadIdx.x == 0) atomicOr(p.dev_err, ANVILQ_DEV_ERR_SEQLEN);
    return;
  }
  const int first = keep / p.page_tokens + (keep % p.page_tokens != 0);
  for (int j = first + threadIdx.x; j < p.max_pages; j += blockDim.x) {
    uint32_t* at = p.table + (size_t)b * p.max_pages + j;
    const uint32_t e = *at;
    if (!e) continue;
    *at = 0;
    if (!(e & kValid)) continue;
    const uint32_t page = e & ~kValid;
    bool bad = page >= (uint32_t)p.num_pages;
    if (!bad && atomicSub(p.refs + page, 1) <= 0) {   // more entries than the count says
      atomicAdd(p.refs + page, 1);
      bad = true;
    }
    if (bad) atomicOr(p.dev_err, ANVILQ_DEV_ERR_PAGE);
  }
}

// ---- compact --------------------------------------------------------------------

struct Compact {
  const uint32_t* table;
  uint32_t* out;
  const int* refs;
  int* out_refs;
  int* used;              // [1]: pages in use
  int* to;                // [num_pages], scratch: where a page goes
  Move* moves;            // [num_pages / 2 + 1], scratch
  int* move_count;
  int* dev_err;
  long long entries;
  int num_pages;
};

__global__ void __launch_bounds__(kPlan) compact_kernel(const __grid_constant__ Compact p) {
  prologue();
  const int tid = threadIdx.x;
  constexpr int kEach = 16;
  int n = 0;
  for (int p0 = 0; p0 < p.num_pages; p0 += kPlan * kEach) {
    int mine = 0;
#pragma unroll
    for (int i = 0; i < kEach; ++i) {
      const int page = p0 + i * kPlan + tid;
      mine += page < p.num_pages && p.refs[page] != 0;
    }
    int total;
    block_scan(mine, total);
    n += total;
  }
  // free pages below n and used ones from n on, each numbered; they are equally many,
  // and all the former come first
  int holes = 0, moved = 0;
  for (int p0 = 0; p0 < p.num_pages; p0 += kPlan * kEach) {
    uint32_t used = 0;
    int here = 0;
    for (int i = 0; i < kEach; ++i) {
      const int page = p0 + tid * kEach + i;
      if (page >= p.num_pages) break;
      const int r = p.refs[page];
      if (r) used |= 1u << i;
      if (page < n && !r) ++here;
      if (page >= n && r) here += 1 << 16;   // at most 16384 of each: both fit
    }
    int total;
    const int at = block_scan(here, total);
    int hole = holes + (at & 0xffff), move = moved + (at >> 16);
    for (int i = 0; i < kEach; ++i) {
      const int page = p0 + tid * kEach + i;
      if (page >= p.num_pages) break;
      if (page < n) {
        if (!(used >> i & 1)) p.moves[hole++].dst = page;
        p.to[page] = page;
      }
    }
    __syncthreads();
    for (int i = 0; i < kEach; ++i) {
      const int page = p0 + tid * kEach + i;
      if (page < n || page >= p.num_pages) continue;
      if (used >> i & 1) {
        const int dst = p.moves[move].dst;
        p.moves[move].src = page;
        p.moves[move].rows = -1;
        p.to[page] = dst;
        ++move;
      } else {
        p.to[page] = page;
      }
    }
    holes += total & 0xffff;
    moved += total >> 16;
  }
  __syncthreads();
  if (p.out_refs != p.refs)
    for (int page = tid; page < p.num_pages; page += kPlan) p.out_refs[page] = p.refs[page];
  __syncthreads();
  for (int k = tid; k < moved; k += kPlan) {
    p.out_refs[p.moves[k].dst] = p.refs[p.moves[k].src];
    p.out_refs[p.moves[k].src] = 0;
  }
  if (tid == 0) {
    *p.used = n;
    *p.move_count = moved;
  }
}

__global__ void __launch_bounds__(256) rename_kernel(const __grid_constant__ Compact p) {
  prologue();
  bool bad = false;
  for (long long i = (long long)blockIdx.x * blockDim.x + threadIdx.x; i < p.entries;
       i += (long long)gridDim.x * blockDim.x) {
    const uint32_t e = p.table[i], page = e & ~kValid;
    uint32_t now = e;
    if (e & kValid) {
      if (page < (uint32_t)p.num_pages) now = (uint32_t)p.to[page] | kValid;
      else bad = true;
    }
    p.out[i] = now;
  }
  if (bad) atomicOr(p.dev_err, ANVILQ_DEV_ERR_PAGE);
}

// ---- copies ---------------------------------------------------------------------

struct Pool {
  char* base;
  unsigned segments;       // runs of a page that each hold all tokens in order
  unsigned segment_bytes;
  unsigned unit_bytes;     // of the tokens that share a unit
  unsigned unit_tokens;
};
struct Copy {
  const Move* moves;       // or, null, the three lists
  const int* src;
  const int* dst;
  const int* rows;         // may be null: whole pages
  const int* count;        // may be null: `most`
  int* dev_err;
  int most, num_pages, pools;
  int stretches;   // of a page
  Pool pool[kMaxPools];
};

// Resident CTAs over stretches of a moved page of a pool, each a team's: a CTA of TEAM = 256
// threads takes 32 KB at a time, a warp 4 KB where pages are smaller, so that kAhead loads
// of every thread are on their way before their stores.  W: 16 bytes, or 4 where pools are
// not aligned to more.
template <typename W, int TEAM>
__global__ void __launch_bounds__(kCopyThreads) copy_kernel(const __grid_constant__ Copy p) {
  prologue();
  constexpr unsigned kStep = TEAM * sizeof(W), kRounds = 16 / sizeof(W);
  constexpr int kTeams = kCopyThreads / TEAM;
  const unsigned team = TEAM == kCopyThreads ? 0 : threadIdx.x / TEAM, me = threadIdx.x % TEAM;
  const int count = p.count ? min(max(*p.count, 0), p.most) : p.most;
  const long long units = (long long)count * p.pools * p.stretches;
  for (long long u = (long long)blockIdx.x * kTeams + team; u < units; u += (long long)gridDim.x * kTeams) {
    const int stretch = (int)(u % p.stretches);
    const int t = (int)(u / p.stretches);
    const int i = t / p.pools;
    const Pool& pool = p.pool[t % p.pools];
    const Move m = p.moves ? p.moves[i] : Move{p.src[i], p.dst[i], p.rows ? p.rows[i] : -1};
    if (m.src < 0 || m.dst < 0) continue;
    if (m.src >= p.num_pages || m.dst >= p.num_pages) {
      if (me == 0) atomicOr(p.dev_err, ANVILQ_DEV_ERR_PAGE);
      continue;
    }
    // of a segment of the page, what the move's rows take
    const unsigned live = m.rows < 0 ? pool.segment_bytes
                                     : (unsigned)min((unsigned long long)pool.segment_bytes,
                                                     (unsigned long long)(((unsigned)m.rows + pool.unit_tokens - 1) /
                                                                          pool.unit_tokens) * pool.unit_bytes);
    const unsigned page_bytes = pool.segments * pool.segment_bytes;   // below 2^31
    const char* from = pool.base + (size_t)m.src * page_bytes;
    char* to = pool.base + (size_t)m.dst * page_bytes;
#pragma unroll 1
    for (unsigned round = 0; round < kRounds; ++round) {
      const unsigned o0 = (stretch * kRounds + round) * (kAhead * kStep) + me * (unsigned)sizeof(W);
      W w[kAhead];
      bool on[kAhead];
#pragma unroll
      for (int a = 0; a < kAhead; ++a) {
        const unsigned o = o0 + a * kStep;
        on[a] = o < page_bytes && (pool.segments == 1 ? o : o % pool.segment_bytes) < live;
        if (on[a]) w[a] = *reinterpret_cast<const W*>(from + o);
      }
#pragma unroll
      for (int a = 0; a < kAhead; ++a)
        if (on[a]) *reinterpret_cast<W*>(to + o0 + a * kStep) = w[a];
    }
  }
}

template <typename P>
static int launch(void (*kernel)(P), int ctas, int threads, size_t smem, cudaStream_t s, bool overlaps, const P& p) {
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(ctas);
  cfg.blockDim = dim3(threads);
  cfg.dynamicSmemBytes = smem;
  cfg.stream = s;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = attr;
  cfg.numAttrs = overlaps ? 1 : 0;
  if (cudaLaunchKernelEx(&cfg, kernel, p) != cudaSuccess) {
    cudaGetLastError();
    return ANVILQ_ECUDA;
  }
  return ANVILQ_OK;
}

static bool aligned(const void* p, unsigned n) { return (reinterpret_cast<uintptr_t>(p) & (n - 1)) == 0; }

// ANVILQ_OK, or why the pools cannot be copied in.  Nothing that the call reads or
// writes besides (`other`, null or bytes 0 skipped) may lie in a pool.
struct Span {
  const void* start;
  size_t bytes;
};
static int check_pools(const anvilq_page_pool* pools, int n, int num_pages, int moves, int page_tokens,
                       std::initializer_list<Span> others) {
  if (n < 0 || (n && !pools)) return ANVILQ_EINVAL;
  if ((long long)std::min(n, kMaxPools) * moves > INT_MAX) return ANVILQ_ESHAPE;   // a copy launch's numbers of them
  for (int i = 0; i < n; ++i) {
    const anvilq_page_pool& a = pools[i];
    if (!a.base || a.segments < 1 || a.segment_bytes < 1 || a.unit_tokens < 1) return ANVILQ_EINVAL;
    if (page_tokens % a.unit_tokens || a.segment_bytes % (page_tokens / a.unit_tokens)) return ANVILQ_ESHAPE;
    const int unit = a.segment_bytes / (page_tokens / a.unit_tokens);
    if ((long long)a.segments * a.segment_bytes > INT_MAX) return ANVILQ_ESHAPE;
    if (!aligned(a.base, 4) || unit % 4) return ANVILQ_EALIGN;
    const size_t bytes = (size_t)num_pages * a.segments * a.segment_bytes;
    for (const Span& o : others)
      if (overlap(a.base, bytes, o.start, o.bytes)) return ANVILQ_EINVAL;
  }
  return ANVILQ_OK;
}

// The copies of `moves` (or of the lists) in all pools: those aligned to 16 bytes, then the
// others.
static int copy_all(Copy& c, const anvilq_page_pool* pools, int n, int page_tokens, bool overlaps, cudaStream_t st) {
  for (int odd = 0; odd < 2; ++odd) {
    for (int next = 0; next < n;) {
      size_t widest = 0;
      for (c.pools = 0; next < n && c.pools < kMaxPools; ++next) {
        const anvilq_page_pool& a = pools[next];
        const int unit = a.segment_bytes / (page_tokens / a.unit_tokens);
        if ((aligned(a.base, 16) && a.segment_bytes % 16 == 0 && unit % 16 == 0) == (bool)odd) continue;
        c.pool[c.pools++] = Pool{static_cast<char*>(a.base), (unsigned)a.segments, (unsigned)a.segment_bytes,
                                 (unsigned)unit, (unsigned)a.unit_tokens};
        widest = std::max(widest, (size_t)a.segments * a.segment_bytes);
      }
      if (!c.pools) continue;
      const bool small = widest < (size_t)kCopyThreads * kAhead * 16;
      const size_t stretch = (size_t)(small ? 32 : kCopyThreads) * kAhead * 16;
      c.stretches = (int)((widest + stretch - 1) / stretch);
      const double units = (double)c.most * c.pools * c.stretches;
      const int ctas = (int)std::min(std::max(small ? units / (kCopyThreads / 32) : units, 1.0), 148.0 * 6);
      auto go = [&](auto kernel) { return launch(kernel, ctas, kCopyThreads, 0, st, overlaps, c); };
      const int rc = odd ? (small ? go(copy_kernel<uint32_t, 32>) : go(copy_kernel<uint32_t, kCopyThreads>))
                         : (small ? go(copy_kernel<uint4, 32>) : go(copy_kernel<uint4, kCopyThreads>));
      if (rc) return rc;
      overlaps = true;   // the next one waits for this one's stores all the same
    }
  }
  return ANVILQ_OK;
}

static bool table_ok(int rows, int max_pages, int num_pages) {
  return rows >= 1 && max_pages >= 1 && num_pages >= 1 && rows <= kMaxRows && (long long)rows * max_pages <= INT_MAX / 2;
}
static size_t up16(size_t n) { return (n + 15) / 16 * 16; }

}  // namespace pages
}  // namespace anvilq

extern "C" {

int anvilq_pages_fork(const uint32_t* page_table, uint32_t* out, int32_t* refs, const int32_t* parents, int old_rows,
                      int new_rows, int groups, int max_pages, int num_pages, int* dev_err, unsigned flags,
                      anvilq_stream_t stream) {
  using namespace anvilq;
  using namespace anvilq::pages;
  if (!page_table || !out || !refs || !parents || !dev_err) return ANVILQ_EINVAL;
  if (flags & ~(unsigned)ANVILQ_GEMM_OVERLAP_PRIOR) return ANVILQ_EINVAL;
  if (!table_ok(old_rows, max_pages, num_pages) || !table_ok(new_rows, max_pages, num_pages)) return ANVILQ_ESHAPE;
  if (groups < 1 || old_rows % groups || new_rows % groups) return ANVILQ_EINVAL;
  if (!aligned(page_table, 4) || !aligned(out, 4) || !aligned(refs, 4) || !aligned(parents, 4)) return ANVILQ_EALIGN;
  const size_t in = (size_t)old_rows * max_pages * 4, to = (size_t)new_rows * max_pages * 4, r = (size_t)num_pages * 4;
  const size_t pa = (size_t)new_rows * 4;
  if (overlap(out, to, page_table, in) || overlap(out, to, refs, r) || overlap(out, to, parents, pa) ||
      overlap(refs, r, page_table, in) || overlap(refs, r, parents, pa))
    return ANVILQ_EINVAL;
  const Fork p{page_table, out, refs, parents, dev_err, old_rows, new_rows, old_rows / groups, new_rows / groups,
               max_pages, num_pages};
  return launch(fork_kernel, std::max(old_rows, new_rows), 256, 0, reinterpret_cast<cudaStream_t>(stream),
                (flags & ANVILQ_GEMM_OVERLAP_PRIOR) != 0, p);
}

size_t anvilq_pages_reserve_workspace_size(int rows, int num_pages) {
  using namespace anvilq::pages;
  if (!table_ok(rows, 1, num_pages)) return 0;
  return ANVILQ_WORKSPACE_COUNTER_BYTES + (size_t)num_pages * sizeof(Writers) + up16((size_t)num_pages * 4) +
         up16((size_t)rows * sizeof(Move)) + 16;
}

int anvilq_pages_reserve(uint32_t* page_table, int32_t* refs, const int32_t* before, const int32_t* after,
                         int32_t* lacking, const anvilq_page_pool* pools, int pool_count, int rows, int page_tokens,
                         int max_pages, int num_pages, void* workspace, size_t workspace_bytes, int* dev_err,
                         unsigned flags, anvilq_stream_t stream) {
  using namespace anvilq;
  using namespace anvilq::pages;
  if (!page_table || !refs || !before || !after || !lacking || !dev_err) return ANVILQ_EINVAL;
  if (flags & ~(unsigned)ANVILQ_GEMM_OVERLAP_PRIOR) return ANVILQ_EINVAL;
  if (!table_ok(rows, max_pages, num_pages) || page_tokens < 1 || (long long)page_tokens * max_pages > (1LL << 30))
    return ANVILQ_ESHAPE;
  if (!aligned(page_table, 4) || !aligned(refs, 4) || !aligned(before, 4) || !aligned(after, 4) ||
      !aligned(lacking, 4) || !aligned(workspace, 16))
    return ANVILQ_EALIGN;
  const Span spans[] = {{page_table, (size_t)rows * max_pages * 4}, {refs, (size_t)num_pages * 4}, {lacking, 4},
                        {before, (size_t)rows * 4}, {after, (size_t)rows * 4}, {workspace, workspace ? workspace_bytes : 0}};
  for (const Span& a : spans)
    for (const Span* b = &a + 1; b != std::end(spans); ++b)
      if (!(a.start == before && b->start == after) && overlap(a.start, a.bytes, b->start, b->bytes))
        return ANVILQ_EINVAL;
  if (const int rc = check_pools(pools, pool_count, num_pages, rows, page_tokens,
                                 {spans[0], spans[1], spans[2], spans[3], spans[4], spans[5]}))
    return rc;
  if (!workspace || workspace_bytes < anvilq_pages_reserve_workspace_size(rows, num_pages)) return ANVILQ_EWORKSPACE;
  char* at = static_cast<char*>(workspace) + ANVILQ_WORKSPACE_COUNTER_BYTES;
  Reserve p{page_table, refs, before, after, lacking, nullptr, nullptr, nullptr, nullptr, dev_err,
            rows, max_pages, num_pages, page_tokens};
  p.writers = reinterpret_cast<Writers*>(at);
  at += (size_t)num_pages * sizeof(Writers);
  p.free_pages = reinterpret_cast<int*>(at);
  at += up16((size_t)num_pages * 4);
  p.moves = reinterpret_cast<Move*>(at);
  at += up16((size_t)rows * sizeof(Move));
  p.move_count = reinterpret_cast<int*>(at);
  cudaStream_t st = reinterpret_cast<cudaStream_t>(stream);
  const size_t smem = (size_t)(rows + 1) * 4;
  if (smem > 40 * 1024 &&
      cudaFuncSetAttribute(reserve_kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, (kMaxRows + 1) * 4) != cudaSuccess) {
    cudaGetLastError();
    return ANVILQ_ECUDA;
  }
  if (const int rc = launch(reserve_kernel, 1, kPlan, smem, st, (flags & ANVILQ_GEMM_OVERLAP_PRIOR) != 0, p)) return rc;
  Copy c{};
  c.moves = p.moves;
  c.count = p.move_count;
  c.dev_err = dev_err;
  c.most = rows;
  c.num_pages = num_pages;
  return copy_all(c, pools, pool_count, page_tokens, true, st);
}

int anvilq_pages_release(uint32_t* page_table, int32_t* refs, const int32_t* keep, int rows, int page_tokens,
                         int max_pages, int num_pages, int* dev_err, unsigned flags, anvilq_stream_t stream) {
  using namespace anvilq;
  using namespace anvilq::pages;
  if (!page_table || !refs || !keep || !dev_err) return ANVILQ_EINVAL;
  if (flags & ~(unsigned)ANVILQ_GEMM_OVERLAP_PRIOR) return ANVILQ_EINVAL;
  if (!table_ok(rows, max_pages, num_pages) || page_tokens < 1) return ANVILQ_ESHAPE;
  if (!aligned(page_table, 4) || !aligned(refs, 4) || !aligned(keep, 4)) return ANVILQ_EALIGN;
  const size_t t = (size_t)rows * max_pages * 4, r = (size_t)num_pages * 4, k = (size_t)rows * 4;
  if (overlap(page_table, t, refs, r) || overlap(page_table, t, keep, k) || overlap(refs, r, keep, k))
    return ANVILQ_EINVAL;
  const Release p{page_table, refs, keep, dev_err, max_pages, num_pages, page_tokens};
  return launch(release_kernel, rows, 256, 0, reinterpret_cast<cudaStream_t>(stream),
                (flags & ANVILQ_GEMM_OVERLAP_PRIOR) != 0, p);
}

size_t anvilq_pages_compact_workspace_size(int num_pages) {
  using namespace anvilq::pages;
  if (num_pages < 1) return 0;
  return ANVILQ_WORKSPACE_COUNTER_BYTES + up16((size_t)num_pages * 4) +
         up16(((size_t)num_pages / 2 + 1) * sizeof(Move)) + 16;
}

int anvilq_pages_compact(const uint32_t* page_table, uint32_t* out, const int32_t* refs, int32_t* out_refs,
                         int32_t* used, const anvilq_page_pool* pools, int pool_count, int rows, int page_tokens,
                         int max_pages, int num_pages, void* workspace, size_t workspace_bytes, int* dev_err,
                         unsigned flags, anvilq_stream_t stream) {
  using namespace anvilq;
  using namespace anvilq::pages;
  if (!page_table || !out || !refs || !out_refs || !used || !dev_err) return ANVILQ_EINVAL;
  if (flags & ~(unsigned)ANVILQ_GEMM_OVERLAP_PRIOR) return ANVILQ_EINVAL;
  if (!table_ok(rows, max_pages, num_pages) || page_tokens < 1) return ANVILQ_ESHAPE;
  if (!aligned(page_table, 4) || !aligned(out, 4) || !aligned(refs, 4) || !aligned(out_refs, 4) || !aligned(used, 4) ||
      !aligned(workspace, 16))
    return ANVILQ_EALIGN;
  const size_t t = (size_t)rows * max_pages * 4, r = (size_t)num_pages * 4;
  const Span spans[] = {{page_table, t}, {out, out == page_table ? 0 : t}, {refs, r},
                        {out_refs, out_refs == refs ? 0 : r}, {used, 4}, {workspace, workspace ? workspace_bytes : 0}};
  for (const Span& a : spans)
    for (const Span* b = &a + 1; b != std::end(spans); ++b)
      if (overlap(a.start, a.bytes, b->start, b->bytes)) return ANVILQ_EINVAL;
  if (const int rc = check_pools(pools, pool_count, num_pages, num_pages / 2 + 1, page_tokens,
                                 {spans[0], spans[1], spans[2], spans[3], spans[4], spans[5]}))
    return rc;
  if (!workspace || workspace_bytes < anvilq_pages_compact_workspace_size(num_pages)) return ANVILQ_EWORKSPACE;
  char* at = static_cast<char*>(workspace) + ANVILQ_WORKSPACE_COUNTER_BYTES;
  Compact p{page_table, out, refs, out_refs, used, nullptr, nullptr, nullptr, dev_err, (long long)rows * max_pages,
            num_pages};
  p.to = reinterpret_cast<int*>(at);
  at += up16((size_t)num_pages * 4);
  p.moves = reinterpret_cast<Move*>(at);
  at += up16(((size_t)num_pages / 2 + 1) * sizeof(Move));
  p.move_count = reinterpret_cast<int*>(at);
  cudaStream_t st = reinterpret_cast<cudaStream_t>(stream);
  if (const int rc = launch(compact_kernel, 1, kPlan, 0, st, (flags & ANVILQ_GEMM_OVERLAP_PRIOR) != 0, p)) return rc;
  const int ctas = (int)std::min<long long>((p.entries + 255) / 256, 148 * 8);
  if (const int rc = launch(rename_kernel, ctas, 256, 0, st, true, p)) return rc;
  Copy c{};
  c.moves = p.moves;
  c.count = p.move_count;
  c.dev_err = dev_err;
  c.most = num_pages / 2 + 1;
  c.num_pages = num_pages;
  return copy_all(c, pools, pool_count, page_tokens, true, st);
}

int anvilq_pages_copy(const anvilq_page_pool* pools, int pool_count, const int32_t* src, const int32_t* dst,
                      const int32_t* rows, const int32_t* count, int most, int page_tokens, int num_pages,
                      int* dev_err, unsigned flags, anvilq_stream_t stream) {
  using namespace anvilq;
  using namespace anvilq::pages;
  if (most < 0 || (most && (!src || !dst)) || !dev_err) return ANVILQ_EINVAL;
  if (flags & ~(unsigned)ANVILQ_GEMM_OVERLAP_PRIOR) return ANVILQ_EINVAL;
  if (num_pages < 1 || page_tokens < 1) return ANVILQ_ESHAPE;
  if (!aligned(src, 4) || !aligned(dst, 4) || !aligned(rows, 4) || !aligned(count, 4)) return ANVILQ_EALIGN;
  const size_t list = (size_t)most * 4;
  if (const int rc = check_pools(pools, pool_count, num_pages, most, page_tokens,
                                 {{src, list}, {dst, list}, {rows, rows ? list : 0}, {count, count ? 4u : 0u}}))
    return rc;
  if (most == 0) return ANVILQ_OK;
  Copy c{};
  c.src = src;
  c.dst = dst;
  c.rows = rows;
  c.count = count;
  c.dev_err = dev_err;
  c.most = most;
  c.num_pages = num_pages;
  return copy_all(c, pools, pool_count, page_tokens, (flags & ANVILQ_GEMM_OVERLAP_PRIOR) != 0,
                  reinterpret_cast<cudaStream_t>(stream));
}

}  // extern "C"
