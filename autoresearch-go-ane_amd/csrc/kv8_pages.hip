// The tables of the 8-bit cache's pages: forking with copy on write, reserving
// and freeing (ane_kv8_fork), compacting (ane_kv8_compact) and copying
// (ane_kv8_copy); include/ane_serve.h says what each does.
//
// Everything is whole numbers, so results do not depend on the order in which
// blocks run: reference counts change by atomic additions, and the pages that
// are handed out are ranked (by sequence and position), as are the free ones
// (by id).
//
// What bounds it.  Copies: HBM, once pages fill it (compacting, 558 MB read and
// written, 105 us, 5.3 TB/s; 3700 pages in 8 layers, 490 MB, 98 us, 5.0 TB/s).
// Tables: chains of dependent accesses, and launches (a fork of 4 sequences 4.6 us
// for the table and 3.8 for its copies; of 384 sequences of up to 8000 tokens 3.6
// for the rows, 5.0 for the plan and 8.4 for the table and 63 MB of copies).
#include <algorithm>

#include "kv8.h"
#include "op_error.h"
#include "wave_ops.h"

namespace ane {

namespace {

constexpr int kMaxLayers = 32;  // of a launch
constexpr int kTh = 1024;       // threads of the blocks that rank
constexpr int kChunk = 4 * kTh; // pages such a block ranks at a time

// The layers' pages as the copies take them: k, v, exponents, and the bounds or
// null.
struct Layers {
  uint8_t *k[kMaxLayers], *v[kMaxLayers];
  int8_t *ke[kMaxLayers], *ve[kMaxLayers];
  int8_t *box[kMaxLayers], *unit[kMaxLayers];
};
struct Pool {
  int pages, pshift, NKV, dshift;  // page_tokens = 1 << pshift, head_dim = 1 << dshift
};

__device__ __forceinline__ int load_ref(const int* p) {
  return __hip_atomic_load(p, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
}

// A barrier behind which the block's atomics and stores to global memory so far
// have arrived.
__device__ __forceinline__ void settle() {
  asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
  __syncthreads();
}

// Of page `from` to page `to`, `sides` sides from side0 on (side 2 l is layer
// l's keys, 2 l + 1 its values), their first `units` units of 16 tokens, by a
// block of TH threads.  A unit of a head is 16 * head_dim bytes in a row on both
// sides.  Four loads a thread are under way at once: of one side, or of four
// where sides are small and come several to a block.  FAR: pages that the caches
// do not hold until somebody reads them go past them.
template <int TH, bool FAR>
__device__ __forceinline__ void copy_sides(const Pool& p, const Layers& x, const Layers& y, int side0, int sides,
                                           int from, int to, int units) {
  const int tid = threadIdx.x;
  const uint32_t whole = 1u << (p.pshift - 4 + p.dshift), used = (uint32_t)units << p.dshift;  // 16-byte words of a head
  const uint32_t n = p.NKV * used;
  const size_t at = (size_t)p.NKV * whole;
  const auto place = [&](uint32_t t) {
    const uint32_t h = used == whole ? 0 : t / used;
    return h * whole + (t - h * used);
  };
  const auto load = [](const u32x4* p) { return FAR ? __builtin_nontemporal_load(p) : *p; };
  const auto store = [](u32x4* p, u32x4 w) {
    if (FAR) __builtin_nontemporal_store(w, p);
    else *p = w;
  };
  constexpr int U = 4;
  if (sides == 1) {
    const int l = side0 >> 1;
    const u32x4* s = reinterpret_cast<const u32x4*>(side0 & 1 ? x.v[l] : x.k[l]) + from * at;
    u32x4* d = reinterpret_cast<u32x4*>(side0 & 1 ? y.v[l] : y.k[l]) + to * at;
    for (uint32_t t0 = tid; t0 < n; t0 += TH * U) {
      u32x4 w[U];
      uint32_t o[U];
#pragma unroll
      for (int u = 0; u < U; u++) {
        o[u] = place(min(t0 + u * TH, n - 1));
        w[u] = load(s + o[u]);
      }
#pragma unroll
      for (int u = 0; u < U; u++)
        if (t0 + u * TH < n) store(d + o[u], w[u]);
    }
  } else {
    for (int i = 0; i < sides; i += U) {
      const u32x4* s[U];
      u32x4* d[U];
#pragma unroll
      for (int u = 0; u < U; u++) {
        const int c = side0 + min(i + u, sides - 1), l = c >> 1;
        s[u] = reinterpret_cast<const u32x4*>(c & 1 ? x.v[l] : x.k[l]) + from * at;
        d[u] = reinterpret_cast<u32x4*>(c & 1 ? y.v[l] : y.k[l]) + to * at;
      }
      for (uint32_t t = tid; t < n; t += TH) {
        const uint32_t o = place(t);
        u32x4 w[U];
#pragma unroll
        for (int u = 0; u < U; u++) w[u] = load(s[u] + o);
#pragma unroll
        for (int u = 0; u < U; u++)
          if (i + u < sides) store(d[u] + o, w[u]);
      }
    }
  }
  const size_t ef = (size_t)from * p.NKV, et = (size_t)to * p.NKV;
  for (int c = side0; c < side0 + sides; c++) {
    const int l = c >> 1;
    const int8_t* se = c & 1 ? x.ve[l] : x.ke[l];
    int8_t* de = c & 1 ? y.ve[l] : y.ke[l];
    for (int h = tid; h < p.NKV; h += TH) de[et + h] = se[ef + h];
    if (!(c & 1) && x.box[l] && y.box[l]) {
      const int m = p.NKV << (p.dshift - 3);  // 16-byte words of a page's boxes
      const u32x4* sb = reinterpret_cast<const u32x4*>(x.box[l]) + (size_t)from * m;
      u32x4* db = reinterpret_cast<u32x4*>(y.box[l]) + (size_t)to * m;
      for (int t = tid; t < m; t += TH) db[t] = sb[t];
      for (int h = tid; h < p.NKV; h += TH) y.unit[l][et + h] = x.unit[l][ef + h];
    }
  }
}
// Copies of so many bytes go past the caches, which hold twice that no more
// (compacting, 372 MB read and written 75 us either way, 466 MB 94 past them and
// 101 through them, 279 MB 58 and 49).
constexpr int64_t kFar = 180 << 20;
__host__ __device__ __forceinline__ int64_t bytes_of(const Pool& p, int nlayers) {
  return (int64_t)2 * nlayers * (p.NKV << (p.pshift + p.dshift));
}

// The sides of an item (a page's copy in all layers of a launch) that a block
// takes, `group` at a time.
struct Sides {
  int item, first, count;
};
__device__ __forceinline__ Sides sides_of(uint32_t block, int nlayers, int group) {
  const int per = (2 * nlayers + group - 1) / group;
  Sides s;
  s.item = block / per;
  s.first = (block - s.item * per) * group;
  s.count = min(group, 2 * nlayers - s.first);
  return s;
}

__device__ __forceinline__ int units_of(const Pool& p, int tokens) {
  return (clampi(tokens, 0, 1 << p.pshift) + 15) >> 4;
}

// ---- fork ----------------------------------------------------------------------

// What becomes of a sequence: it holds st tokens and will hold `end`; its new
// pages have the ranks from `base` on, the first of them for a copy of page
// `src` (-1: none).
struct Next {
  int st, end, base, src;
};

struct ForkArgs {
  Pool p;
  int *table, *start, *refs, *missing;
  const int *parents, *news;
  int stride, width, nseq, new_tokens;
  int* mid;    // [nseq][width]: the parents' rows (unused where there are no parents)
  Next* next;  // [nseq]
  int* free;    // [pages]: free pages by rank
  int* found;   // how many of them there are, of those that are wanted
  int* want;    // of a large pool: how many are
  int* counts;  // and how many each chunk has
  int chunks;
};

// One block does the tables by itself where they are small: their entries are
// in LDS (8 rows of 31 a fork 7.8 us, with launches for the rows and the table
// 9.9; 32 of 59 9.1 and 9.8; but 64 of 59 11.9 and 10.8).
constexpr int kSmall = 2048;
bool small_table(int64_t nseq, int64_t width) { return nseq <= kTh && nseq * width <= kSmall; }

__device__ __forceinline__ int there(int id, int pages) { return (unsigned)id < (unsigned)pages ? id : -1; }
__device__ __forceinline__ int held_of(const ForkArgs& a, int i) {
  const int from = a.parents ? a.parents[i] : i;
  return (unsigned)from < (unsigned)a.nseq ? clampi(a.start[from], 0, a.width << a.p.pshift) : 0;
}
__device__ __forceinline__ int end_of(const ForkArgs& a, int i, int st) {
  return st + clampi(a.news ? a.news[i] : a.new_tokens, 0, (a.width << a.p.pshift) - st);
}
__device__ __forceinline__ int pages_for(const ForkArgs& a, int tokens) {
  return (tokens + (1 << a.p.pshift) - 1) >> a.p.pshift;
}
// whether tokens that come go to a page that holds some already
__device__ __forceinline__ bool goes_on(const ForkArgs& a, int st, int end) {
  return end > st && (st & ((1 << a.p.pshift) - 1));
}
__device__ __forceinline__ void recount(const ForkArgs& a, int old, int mid) {
  if (old == mid) return;
  if (old >= 0) atomicSub(a.refs + old, 1);
  if (mid >= 0) atomicAdd(a.refs + mid, 1);
}
// What entry j of a sequence's row becomes: a new page by its rank, which then
// has one holder, or what the parent has there.
__device__ __forceinline__ int entry_of(const ForkArgs& a, const Next& n, int j, int mid, int found, bool& fresh) {
  const int copies = n.src >= 0, held = pages_for(a, n.st);
  int rank = -1;
  if (copies && j == n.st >> a.p.pshift) rank = n.base;
  else if (j >= held && j < pages_for(a, n.end)) rank = n.base + copies + (j - held);
  fresh = rank >= 0;
  if (!fresh) return mid;
  const int id = rank < found ? a.free[rank] : -1;
  if (id >= 0) a.refs[id] = 1;
  return id;
}

// The parents' rows, cut to what they hold; reference counts follow.  A thread
// an entry.
__global__ __launch_bounds__(256) void rows_kernel(ForkArgs a) {
  const int blocks = (a.width + 255) / 256, i = blockIdx.x / blocks;
  const int j = (blockIdx.x - i * blocks) * 256 + threadIdx.x;
  if (j >= a.width) return;
  const int from = a.parents ? a.parents[i] : i;
  const bool holds = j < pages_for(a, held_of(a, i));
  int* mine = a.table + (size_t)i * a.stride + j;
  const int raw = *mine, old = there(raw, a.p.pages);
  const int mid = !holds ? -1 : from == i ? old : there(a.table[(size_t)from * a.stride + j], a.p.pages);
  recount(a, old, mid);
  if (a.parents) a.mid[(size_t)i * a.width + j] = mid;
  else if (raw != mid) *mine = mid;
}

// the sum over the threads before this one, and over all
__device__ __forceinline__ int block_scan(int x, int (&sums)[kTh / 64], int& total) {
  const int lane = threadIdx.x & 63, w = threadIdx.x >> 6;
  const int s = sum_up_to(x);
  __syncthreads();
  if (lane == 63) sums[w] = s;
  __syncthreads();
  const int y = sum_up_to(sums[lane % (kTh / 64)]);  // lane k: the waves up to k
  total = __builtin_amdgcn_readlane(y, kTh / 64 - 1);
  const int upto = __shfl(y, w, 64);
  return upto - __builtin_amdgcn_readlane(s, 63) + s - x;
}

// Sequences that write into a page they hold (`page`, of threads up to nseq <=
// kTh; below 0: none): whether this one copies it first.  Counts become those
// without the sequences that do.  The writers of a page meet in a table of
// twice as many places as there can be pages: a page's place is the first free
// one, or its own, from where its id's hash points on.
constexpr int kPlaces = 2 * kTh;
struct Writers {
  int page[kPlaces], count[kPlaces], lowest[kPlaces];
};
__device__ __forceinline__ bool copies_few(const ForkArgs& a, int page, Writers& t) {
  const int tid = threadIdx.x;
  const int held = page >= 0 ? load_ref(a.refs + page) : 0;  // behind a barrier after the rows' counts
  for (int k = tid; k < kPlaces; k += kTh) {
    t.page[k] = -1;
    t.count[k] = 0;
    t.lowest[k] = kTh;
  }
  __syncthreads();
  int at = 0;
  if (page >= 0) {
    at = (uint32_t)page * 2654435769u >> 21;  // 2^32 / golden ratio; 11 bits
    for (;;) {
      const int was = atomicCAS(&t.page[at], -1, page);
      if (was == -1 || was == page) break;
      at = (at + 1) % kPlaces;
    }
    atomicAdd(&t.count[at], 1);
    atomicMin(&t.lowest[at], tid);
  }
  __syncthreads();
  if (page < 0) return false;
  const int writers = t.count[at];
  const bool first = t.lowest[at] == tid;
  if (first)
    __hip_atomic_store(a.refs + page, held <= writers ? 1 : held - writers, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
  return !(first && held <= writers);
}

// The same of any number of sequences, whose pages stand in next[].base; those
// that copy have them in next[].src then.  A page whose count falls to 0 when
// its writers leave it is held by writers alone, and the lowest of them keeps
// it: the count holds its number, as a negative one, until it becomes 1 again.
__device__ __forceinline__ void copies_many(const ForkArgs& a) {
  constexpr int kMark = -(1 << 30);
  const int tid = threadIdx.x;
  for (int i = tid; i < a.nseq; i += kTh)
    if (const int p = a.next[i].base; p >= 0) atomicSub(a.refs + p, 1);
  settle();
  for (int i = tid; i < a.nseq; i += kTh)
    if (const int p = a.next[i].base; p >= 0 && load_ref(a.refs + p) <= 0) atomicMin(a.refs + p, kMark + i);
  settle();
  for (int i = tid; i < a.nseq; i += kTh) {
    const int p = a.next[i].base;
    if (p >= 0 && load_ref(a.refs + p) != kMark + i) a.next[i].src = p;
  }
  settle();
  for (int i = tid; i < a.nseq; i += kTh) {
    const Next n = a.next[i];
    if (n.base >= 0 && n.src < 0) __hip_atomic_store(a.refs + n.base, 1, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
  }
}

// The lowest `want` free pages, by rank; how many of them there are.
__device__ __forceinline__ int find_free(const ForkArgs& a, int want, int (&sums)[kTh / 64]) {
  int found = 0;
  const uint32_t pages = a.p.pages;
  for (uint32_t p0 = 0; p0 < pages && found < want; p0 += kChunk) {
    int is[4], n = 0;
#pragma unroll
    for (int u = 0; u < 4; u++) {
      const uint32_t p = p0 + threadIdx.x * 4 + u;
      is[u] = p < pages && load_ref(a.refs + min(p, pages - 1)) <= 0;
      n += is[u];
    }
    int all;
    int rank = found + block_scan(n, sums, all);
#pragma unroll
    for (int u = 0; u < 4; u++)
      if (is[u]) {
        if (rank < want) a.free[rank] = (int)(p0 + threadIdx.x * 4 + u);
        rank++;
      }
    found += all;
  }
  return min(found, want);
}

// One block: who copies, how many pages each sequence gets, and which are free.
// A block ranks all of them without another launch (384 sequences in 5.0 us,
// most of it waits for loads and atomics).  SMALL: also the rows before that, and
// the table behind it, in one launch in place of two.
// FIND: and the free pages; otherwise the launches behind it do.
template <bool SMALL, bool FIND>
__global__ __launch_bounds__(kTh) void plan_kernel(ForkArgs a) {
  __shared__ int sums[kTh / 64];
  __shared__ Writers writers;
  __shared__ int lost_all;
  __shared__ int mids[SMALL ? kSmall : 1], source[SMALL ? kTh : 1], holds[SMALL ? kTh : 1];
  __shared__ Next nexts[SMALL ? kTh : 1];
  constexpr int E = SMALL ? kSmall / kTh : 1;  // entries a thread
  const int tid = threadIdx.x;
  if (tid == 0) lost_all = 0;
  int raw[E];
  int st = 0, end = 0;
  if constexpr (SMALL) {
    if (tid < a.nseq) {
      source[tid] = a.parents ? a.parents[tid] : tid;
      st = held_of(a, tid);
      end = end_of(a, tid, st);
      holds[tid] = pages_for(a, st);
    }
    __syncthreads();
#pragma unroll
    for (int k = 0; k < E; k++) {
      const int e = k * kTh + tid;
      if (e >= a.nseq * a.width) break;
      const int i = e / a.width, j = e - i * a.width;
      raw[k] = a.table[(size_t)i * a.stride + j];
      mids[e] = j < holds[i] ? there(a.table[(size_t)source[i] * a.stride + j], a.p.pages) : -1;
      recount(a, there(raw[k], a.p.pages), mids[e]);
    }
    settle();
  }
  int want = 0, lost = 0;
  if (SMALL || a.nseq <= kTh) {
    int page = -2;  // -1: it is not there
    if (tid < a.nseq) {
      if (!SMALL) {
        st = held_of(a, tid);
        end = end_of(a, tid, st);
      }
      if (goes_on(a, st, end)) {
        const int j = st >> a.p.pshift;
        if (SMALL) page = mids[tid * a.width + j];
        else if (a.parents) page = a.mid[(size_t)tid * a.width + j];
        else page = there(a.table[(size_t)tid * a.stride + j], a.p.pages);
      }
    }
    lost = page == -1;
    const bool copies = copies_few(a, page, writers);
    const int before = block_scan(copies + pages_for(a, end) - pages_for(a, st), sums, want);
    if (tid < a.nseq) {
      const Next n = {st, end, before, copies ? page : -1};
      a.next[tid] = n;
      if (SMALL) nexts[tid] = n;
    }
  } else {
    for (int i = tid; i < a.nseq; i += kTh) {
      st = held_of(a, i);
      end = end_of(a, i, st);
      int page = -2;
      if (goes_on(a, st, end)) {
        const int j = st >> a.p.pshift;
        page = a.parents ? a.mid[(size_t)i * a.width + j] : there(a.table[(size_t)i * a.stride + j], a.p.pages);
        lost += page < 0;
      }
      a.next[i] = {st, end, page, -1};
    }
    copies_many(a);
    for (int i0 = 0; i0 < a.nseq; i0 += kTh) {
      const int i = i0 + tid;
      Next n = {0, 0, 0, -1};
      if (i < a.nseq) n = a.next[i];
      int all;
      n.base = want + block_scan((n.src >= 0) + pages_for(a, n.end) - pages_for(a, n.st), sums, all);
      if (i < a.nseq) a.next[i] = n;
      want += all;
    }
  }
  if (lost) atomicAdd(&lost_all, lost);
  settle();
  if constexpr (!FIND) {
    if (tid == 0) {
      *a.want = want;
      *a.missing = lost_all;
    }
    return;
  }
  const int found = find_free(a, want, sums);
  if (tid == 0) {
    *a.found = found;
    *a.missing = want - found + lost_all;
  }
  if constexpr (SMALL) {
    settle();  // the free pages are written
#pragma unroll
    for (int k = 0; k < E; k++) {
      const int e = k * kTh + tid;
      if (e >= a.nseq * a.width) break;
      const int i = e / a.width, j = e - i * a.width;
      bool fresh;
      const int id = entry_of(a, nexts[i], j, mids[e], found, fresh);
      if (id != raw[k]) a.table[(size_t)i * a.stride + j] = id;
    }
    if (tid < a.nseq) a.start[tid] = st;
  }
}

// The free (or held) pages of each chunk, a block a chunk.
__global__ __launch_bounds__(kTh) void count_kernel(const int* refs, int pages, bool held, int* counts) {
  __shared__ int sums[kTh / 64];
  int n = 0;
#pragma unroll
  for (int u = 0; u < 4; u++) {
    const int64_t p = (int64_t)blockIdx.x * kChunk + u * kTh + threadIdx.x;
    n += p < pages && (refs[p] > 0) == held;
  }
  int all;
  block_scan(n, sums, all);
  if (threadIdx.x == 0) counts[blockIdx.x] = all;
}

// What find_free does, of a large pool: a block a chunk, which adds up the counts
// of all.
__global__ __launch_bounds__(kTh) void list_kernel(ForkArgs a) {
  __shared__ int sums[kTh / 64];
  const int tid = threadIdx.x, want = *a.want;
  int n = 0, m = 0, all, before;
  for (int b = tid; b < a.chunks; b += kTh) {
    const int c = a.counts[b];
    n += c;
    m += b < (int)blockIdx.x ? c : 0;
  }
  block_scan(m, sums, before);
  if (blockIdx.x == 0) {
    block_scan(n, sums, all);
    if (tid == 0) {
      *a.found = min(all, want);
      *a.missing += want - min(all, want);
    }
  }
  if (before >= want) return;
  const int64_t p0 = (int64_t)blockIdx.x * kChunk + tid * 4;
  int is[4];
  n = 0;
#pragma unroll
  for (int u = 0; u < 4; u++) {
    is[u] = p0 + u < a.p.pages && a.refs[p0 + u] <= 0;
    n += is[u];
  }
  int rank = before + block_scan(n, sums, all);
#pragma unroll
  for (int u = 0; u < 4; u++)
    if (is[u]) {
      if (rank < want) a.free[rank] = (int)(p0 + u);
      rank++;
    }
}

// The tables' entries and starts, a thread an entry (table_blocks of them);
// behind those blocks the copies, blocks for each sequence.
__global__ __launch_bounds__(256) void finish_kernel(ForkArgs a, Layers x, int nlayers, int group, int table_blocks) {
  const int found = *a.found;
  if ((int)blockIdx.x < table_blocks) {
    const int blocks = (a.width + 255) / 256, i = blockIdx.x / blocks;
    const int j = (blockIdx.x - i * blocks) * 256 + threadIdx.x;
    if (j >= a.width) return;
    const Next n = a.next[i];
    bool fresh;
    const int id = entry_of(a, n, j, a.parents ? a.mid[(size_t)i * a.width + j] : -1, found, fresh);
    if (a.parents || fresh) a.table[(size_t)i * a.stride + j] = id;
    if (j == 0) a.start[i] = n.st;
    return;
  }
  const Sides s = sides_of(blockIdx.x - table_blocks, nlayers, group);
  const Next n = a.next[s.item];
  if (n.src < 0 || n.base >= found) return;
  copy_sides<256, false>(a.p, x, x, s.first, s.count, n.src, a.free[n.base],
                         units_of(a.p, n.st & ((1 << a.p.pshift) - 1)));
}

// ---- compact -------------------------------------------------------------------

struct CompactArgs {
  Pool p;
  int *table, *refs, *moved;
  int stride, width, nseq;
  int chunks;
  int* counts;          // [chunks]: pages held in each
  int* total;           // [1]: pages that go
  int* code;            // [pages]: where a page is then; -1 free; -2 - k: it is the k-th that goes
  int *holes, *movers;  // [pages / 2 + 1]
};

// Ranks: a block a chunk, which adds up the counts of all (of one chunk, its
// own).
__global__ __launch_bounds__(kTh) void rank_kernel(CompactArgs a) {
  __shared__ int sums[kTh / 64];
  const int tid = threadIdx.x;
  const int64_t p0 = (int64_t)blockIdx.x * kChunk + tid * 4;
  int is[4], n = 0, m = 0, held, before = 0, low;
#pragma unroll
  for (int u = 0; u < 4; u++) {
    is[u] = p0 + u < a.p.pages && a.refs[p0 + u] > 0;
    n += is[u];
  }
  int rank = block_scan(n, sums, held);  // pages held before the thread's
  if (a.chunks > 1) {
    n = 0;
    for (int b = tid; b < a.chunks; b += kTh) {
      const int c = a.counts[b];
      n += c;
      m += b < (int)blockIdx.x ? c : 0;
    }
    block_scan(n, sums, held);    // U: the pages held
    block_scan(m, sums, before);  // those before this chunk
    rank += before;
  }
  // those below U: whole chunks, and the one that U lies in
  const int cu = held / kChunk;
  n = 0;
  if (a.chunks > 1) {
    for (int b = tid; b < cu; b += kTh) n += a.counts[b];
    for (int p = cu * kChunk + tid; p < held; p += kTh) n += a.refs[p] > 0;
  } else {
#pragma unroll
    for (int u = 0; u < 4; u++) n += is[u] && p0 + u < held;
  }
  block_scan(n, sums, low);
  if (blockIdx.x == 0 && tid == 0) *a.total = held - low;
#pragma unroll
  for (int u = 0; u < 4; u++) {
    if (p0 + u >= a.p.pages) break;
    const int p = (int)p0 + u;
    int code = -1;
    if (is[u]) {
      code = p;
      if (p >= held) {
        const int k = rank - low;
        code = -2 - k;
        a.movers[k] = p;
      }
      rank++;
    } else if (p < held) {
      a.holes[p - rank] = p;
    }
    a.code[p] = code;
  }
}

__global__ __launch_bounds__(256) void move_kernel(CompactArgs a, Layers x, int nlayers, int group, int items, int book_blocks) {
  if ((int)blockIdx.x < book_blocks) {
    // a thread a page or an entry of the table
    const int64_t t = (int64_t)blockIdx.x * 256 + threadIdx.x;
    if (t < a.p.pages) {
      const int p = (int)t, c = a.code[p];
      int to = c;
      if (c <= -2) {
        to = a.holes[-2 - c];
        a.refs[to] = a.refs[p];
        a.refs[p] = 0;
      }
      a.moved[p] = to;
    } else if (t - a.p.pages < (int64_t)a.nseq * a.width) {
      const int64_t e = t - a.p.pages;
      const int i = (int)(e / a.width), j = (int)(e - (int64_t)i * a.width);
      int* at = a.table + (size_t)i * a.stride + j;
      const int id = *at;
      if ((unsigned)id < (unsigned)a.p.pages) {
        const int c = a.code[id];
        *at = c <= -2 ? a.holes[-2 - c] : c;
      }
    }
    return;
  }
  const Sides s = sides_of(blockIdx.x - book_blocks, nlayers, group);
  const int total = *a.total, units = 1 << (a.p.pshift - 4);
  if (total * bytes_of(a.p, nlayers) >= kFar) {
    for (int k = s.item; k < total; k += items)
      copy_sides<256, true>(a.p, x, x, s.first, s.count, a.movers[k], a.holes[k], units);
  } else {
    for (int k = s.item; k < total; k += items)
      copy_sides<256, false>(a.p, x, x, s.first, s.count, a.movers[k], a.holes[k], units);
  }
}

// ---- copy ----------------------------------------------------------------------

template <bool FAR>
__global__ __launch_bounds__(256) void copy_kernel(Pool p, int into_pages, Layers x, Layers y, int nlayers,
                                                   int group, const int* src, const int* dst, const int* tokens) {
  const Sides s = sides_of(blockIdx.x, nlayers, group);
  const int from = src[s.item], to = dst[s.item];
  if ((unsigned)from >= (unsigned)p.pages || (unsigned)to >= (unsigned)into_pages) return;
  const int units = tokens ? units_of(p, tokens[s.item]) : 1 << (p.pshift - 4);
  if (units > 0) copy_sides<256, FAR>(p, x, y, s.first, s.count, from, to, units);
}

// ---- host ----------------------------------------------------------------------

int check_pool(const char* op, const ane_kv8_pool* pool, bool refs, Pool* out) {
  if (!pool || !pool->layers || pool->nlayers < 1 || pool->nlayers > 1024)
    return op_fail(ANE_ERR_ARG, "storiesane %s: no pool, or %d layers, want 1..1024", op, pool ? pool->nlayers : 0);
  if (refs && !pool->refs) return op_fail(ANE_ERR_ARG, "storiesane %s: null refs", op);
  const ane_kv8_cache& c = pool->layers[0];
  for (int l = 0; l < pool->nlayers; l++) {
    const ane_kv8_cache& x = pool->layers[l];
    const int rc = kv8_cache_check(op, &x);
    if (rc) return rc;
    if (x.pages != c.pages || x.page_tokens != c.page_tokens || x.kv_heads != c.kv_heads || x.head_dim != c.head_dim ||
        x.device != c.device)
      return op_fail(ANE_ERR_ARG, "storiesane %s: layer %d differs from layer 0 in its sizes or its device", op, l);
    if (pool->bounds) {
      const ane_kv8_bounds& b = pool->bounds[l];
      if (!b.box != !b.unit || ((uintptr_t)b.box & 15))
        return op_fail(ANE_ERR_ARG, "storiesane %s: bounds of layer %d: box without unit, or not 16-byte aligned", op, l);
    }
  }
  *out = {c.pages, 0, c.kv_heads, c.head_dim == 64 ? 6 : 7};
  while (1 << out->pshift < c.page_tokens) out->pshift++;
  return ANE_OK;
}

// the layers from l0 on that a launch takes
int layers_of(const ane_kv8_pool& pool, int l0, Layers* x) {
  const int n = std::min(kMaxLayers, pool.nlayers - l0);
  for (int i = 0; i < n; i++) {
    const ane_kv8_cache& c = pool.layers[l0 + i];
    x->k[i] = (uint8_t*)c.k; x->v[i] = (uint8_t*)c.v; x->ke[i] = c.k_exp; x->ve[i] = c.v_exp;
    x->box[i] = pool.bounds ? pool.bounds[l0 + i].box : nullptr;
    x->unit[i] = pool.bounds ? pool.bounds[l0 + i].unit : nullptr;
  }
  return n;
}

// Sides a block copies: one where there are few, and of small pages as many as
// make 16 KB, which is what a block's threads load at a time (pages of 1 KB a side
// 30 us, one a block 66; of 4 KB 98 and 101; 64 KB for pages of 16 KB 126 and
// 112).
int group_of(const Pool& p, int64_t items, int nlayers) {
  const int side = p.NKV << (p.pshift + p.dshift);  // bytes
  int g = std::max(1, std::min(2 * nlayers, 16384 / side));
  while (g > 1 && items * ((2 * nlayers + g - 1) / g) < 2048) g /= 2;
  return g;
}
int blocks_of(int64_t items, int nlayers, int group) { return (int)(items * ((2 * nlayers + group - 1) / group)); }

int check_table(const char* op, const int* table, int stride, int width, int nseq, int pshift) {
  if (nseq < 0 || nseq > 65536) return op_fail(ANE_ERR_ARG, "storiesane %s: nseq=%d want 0..65536", op, nseq);
  if (nseq == 0) return ANE_OK;
  if (!table) return op_fail(ANE_ERR_ARG, "storiesane %s: null table", op);
  if (width < 1 || stride < width || ((int64_t)width << pshift) > 1 << 30)
    return op_fail(ANE_ERR_ARG, "storiesane %s: table_pages=%d (at least 1, at most its stride %d and %d tokens)", op,
                   width, stride, 1 << 30);
  if ((int64_t)nseq * width > 1 << 30)
    return op_fail(ANE_ERR_ARG, "storiesane %s: a table of %d x %d entries, want at most %d", op, nseq, width, 1 << 30);
  return ANE_OK;
}

int64_t up16(int64_t n) { return (n + 15) / 16 * 16; }

// Of larger pools the free pages are found by a block a chunk: 13 us a fork (32
// sequences of 8 pages) wherever they lie.  The block of the plan goes from chunk
// to chunk until it has enough: 6 us where they lie all over the pool, but where
// the lowest nine tenths are held 12 of 20,000 pages, 18 of 40,000, 37 of 100,000,
// 100 of 300,000.  The host does not know which, so the line is where the worst is
// equal.
constexpr int kLarge = 20480;

struct ForkPlan {
  int chunks;
  int64_t next, mid, free, counts, bytes;  // offsets; found and want come first
};
ForkPlan fork_plan(const Pool& p, int nseq, int width) {
  ForkPlan w;
  w.next = 16;
  w.mid = w.next + (int64_t)nseq * sizeof(Next);
  w.free = w.mid + up16((int64_t)nseq * width * 4);
  w.chunks = p.pages > kLarge ? (int)(((int64_t)p.pages + kChunk - 1) / kChunk) : 0;
  w.counts = w.free + up16((int64_t)p.pages * 4);
  w.bytes = w.counts + up16((int64_t)w.chunks * 4);
  return w;
}
struct CompactPlan {
  int chunks;
  int64_t counts, code, holes, movers, bytes;  // offsets; total comes first
};
CompactPlan compact_plan(const Pool& p) {
  CompactPlan w;
  w.chunks = (int)(((int64_t)p.pages + kChunk - 1) / kChunk);
  w.counts = 16;
  w.code = w.counts + up16((int64_t)w.chunks * 4);
  w.holes = w.code + up16((int64_t)p.pages * 4);
  w.movers = w.holes + up16(((int64_t)p.pages / 2 + 1) * 4);
  w.bytes = w.movers + up16(((int64_t)p.pages / 2 + 1) * 4);
  return w;
}

int check_ws(const char* op, const void* ws, int64_t given, int64_t need) {
  if (!ws || ((uintptr_t)ws & 15) || given < need)
    return op_fail(ANE_ERR_ARG, "storiesane %s: workspace of %lld bytes, want %lld, 16-byte aligned", op,
                   (long long)(ws ? given : 0), (long long)need);
  return ANE_OK;
}
int launched(const char* op) {
  const hipError_t h = hipGetLastError();
  return h == hipSuccess ? ANE_OK : op_fail(ANE_ERR_HIP, "storiesane %s: %s", op, hipGetErrorString(h));
}
int device_error(const char* op, int device, hipError_t h) {
  return op_fail(ANE_ERR_HIP, "storiesane %s: device %d: %s", op, device, hipGetErrorString(h));
}

}  // namespace

}  // namespace ane

using namespace ane;

extern "C" int64_t ane_kv8_fork_workspace(const ane_kv8_pool* pool, int32_t nseq, int32_t table_pages) {
  const char* op = "kv8 fork workspace";
  Pool p;
  int rc = check_pool(op, pool, false, &p);
  if (!rc) rc = check_table(op, &table_pages, table_pages, table_pages, nseq, p.pshift);
  return rc ? rc : fork_plan(p, nseq, table_pages).bytes;
}

extern "C" int ane_kv8_fork(const ane_kv8_pool* pool, const ane_kv8_fork_args* args, void* stream) {
  const char* op = "kv8 fork";
  ForkArgs a;
  int rc = check_pool(op, pool, true, &a.p);
  if (rc) return rc;
  if (!args) return op_fail(ANE_ERR_ARG, "storiesane %s: null arguments", op);
  const ane_kv8_fork_args& g = *args;
  rc = check_table(op, g.table, g.table_stride, g.table_pages, g.nseq, a.p.pshift);
  if (rc) return rc;
  if (!g.missing || (g.nseq > 0 && !g.start)) return op_fail(ANE_ERR_ARG, "storiesane %s: null buffer", op);
  if (!g.news && g.new_tokens < 0) return op_fail(ANE_ERR_ARG, "storiesane %s: new_tokens=%d", op, g.new_tokens);
  const Buffer buffers[] = {{"table", row_major(g.table, g.nseq, g.table_stride * 4ll, g.table_pages * 4ll), true},
                            {"start", flat(g.start, g.nseq * 4ll), true},
                            {"parents", flat(g.parents, g.nseq * 4ll), false},
                            {"news", flat(g.news, g.nseq * 4ll), false},
                            {"missing", flat(g.missing, 4), true},
                            {"refs", flat(pool->refs, a.p.pages * 4ll), true}};
  rc = check_apart(op, buffers, sizeof buffers / sizeof *buffers);
  if (rc) return rc;
  const ForkPlan w = fork_plan(a.p, g.nseq, g.table_pages);
  rc = check_ws(op, g.ws, g.ws_bytes, w.bytes);
  if (rc) return rc;
  const int device = pool->layers[0].device;
  DeviceScope dev(device);
  if (dev.status() != hipSuccess) return device_error(op, device, dev.status());
  a.table = g.table; a.start = g.start; a.refs = pool->refs; a.missing = g.missing;
  a.parents = g.parents; a.news = g.news;
  a.stride = g.table_stride; a.width = g.table_pages; a.nseq = g.nseq; a.new_tokens = g.new_tokens;
  char* ws = (char*)g.ws;
  a.found = (int*)ws;
  a.want = a.found + 1;
  a.counts = (int*)(ws + w.counts);
  a.chunks = w.chunks;
  a.next = (Next*)(ws + w.next);
  a.mid = (int*)(ws + w.mid);
  a.free = (int*)(ws + w.free);
  const hipStream_t st = (hipStream_t)stream;
  const int table_blocks = a.nseq * ((a.width + 255) / 256);
  const bool large = a.chunks > 0 && a.nseq > 0, small = !large && small_table(a.nseq, a.width);
  if (small) {
    hipLaunchKernelGGL((plan_kernel<true, true>), dim3(1), dim3(kTh), 0, st, a);
  } else {
    hipLaunchKernelGGL(rows_kernel, dim3(table_blocks), dim3(256), 0, st, a);
    hipLaunchKernelGGL((large ? plan_kernel<false, false> : plan_kernel<false, true>), dim3(1), dim3(kTh), 0, st, a);
  }
  if (large) {
    hipLaunchKernelGGL(count_kernel, dim3(a.chunks), dim3(kTh), 0, st, a.refs, a.p.pages, false, a.counts);
    hipLaunchKernelGGL(list_kernel, dim3(a.chunks), dim3(kTh), 0, st, a);
  }
  for (int l0 = 0; l0 < pool->nlayers && a.nseq > 0; l0 += kMaxLayers) {
    Layers x;
    const int n = layers_of(*pool, l0, &x);
    const int tb = l0 == 0 && !small ? table_blocks : 0;
    const int group = group_of(a.p, a.nseq, n);
    hipLaunchKernelGGL(finish_kernel, dim3(tb + blocks_of(a.nseq, n, group)), dim3(256), 0, st, a, x, n, group, tb);
  }
  return launched(op);
}

extern "C" int64_t ane_kv8_compact_workspace(const ane_kv8_pool* pool) {
  Pool p;
  const int rc = check_pool("kv8 compact workspace", pool, false, &p);
  return rc ? rc : compact_plan(p).bytes;
}

extern "C" int ane_kv8_compact(const ane_kv8_pool* pool, const ane_kv8_compact_args* args, void* stream) {
  const char* op = "kv8 compact";
  CompactArgs a;
  int rc = check_pool(op, pool, true, &a.p);
  if (rc) return rc;
  if (!args || !args->moved) return op_fail(ANE_ERR_ARG, "storiesane %s: null arguments", op);
  const ane_kv8_compact_args& g = *args;
  rc = check_table(op, g.table, g.table_stride, g.table_pages, g.nseq, a.p.pshift);
  if (rc) return rc;
  const Buffer buffers[] = {{"table", row_major(g.table, g.nseq, g.table_stride * 4ll, g.table_pages * 4ll), true},
                            {"moved", flat(g.moved, a.p.pages * 4ll), true},
                            {"refs", flat(pool->refs, a.p.pages * 4ll), true}};
  rc = check_apart(op, buffers, sizeof buffers / sizeof *buffers);
  if (rc) return rc;
  const CompactPlan w = compact_plan(a.p);
  rc = check_ws(op, g.ws, g.ws_bytes, w.bytes);
  if (rc) return rc;
  const int device = pool->layers[0].device;
  DeviceScope dev(device);
  if (dev.status() != hipSuccess) return device_error(op, device, dev.status());
  a.table = g.table; a.refs = pool->refs; a.moved = g.moved;
  a.stride = g.table_stride; a.width = g.nseq > 0 ? g.table_pages : 0; a.nseq = g.nseq;
  a.chunks = w.chunks;
  char* ws = (char*)g.ws;
  a.total = (int*)ws;
  a.counts = (int*)(ws + w.counts);
  a.code = (int*)(ws + w.code);
  a.holes = (int*)(ws + w.holes);
  a.movers = (int*)(ws + w.movers);
  const hipStream_t st = (hipStream_t)stream;
  if (a.chunks > 1) hipLaunchKernelGGL(count_kernel, dim3(a.chunks), dim3(kTh), 0, st, a.refs, a.p.pages, true, a.counts);
  hipLaunchKernelGGL(rank_kernel, dim3(a.chunks), dim3(kTh), 0, st, a);
  const int book = (int)(((int64_t)a.p.pages + (int64_t)a.nseq * a.width + 255) / 256);
  for (int l0 = 0; l0 < pool->nlayers; l0 += kMaxLayers) {
    Layers x;
    const int n = layers_of(*pool, l0, &x);
    const int bb = l0 == 0 ? book : 0;
    // pages at a time, as blocks go through them in turn: 1024 of sides from 16 KB on
    // (558 MB 110 us, 2048 118), 2048 of smaller ones (27 MB of 1 KB 20 us, 1024 23;
    // 76 MB of 2 KB 26.4 and 27.8; 4096 no faster)
    const int most = a.p.NKV << (a.p.pshift + a.p.dshift) < 16384 ? 2048 : 1024;
    const int items = std::min(std::max(a.p.pages / 2, 1), most);
    const int group = group_of(a.p, items, n);
    hipLaunchKernelGGL(move_kernel, dim3(bb + blocks_of(items, n, group)), dim3(256), 0, st, a, x, n, group, items, bb);
  }
  return launched(op);
}

extern "C" int ane_kv8_copy(const ane_kv8_pool* from, const ane_kv8_pool* into, const ane_kv8_copy_args* args,
                            void* stream) {
  const char* op = "kv8 copy";
  Pool p, q;
  int rc = check_pool(op, from, false, &p);
  if (!rc) rc = check_pool(op, into, false, &q);
  if (rc) return rc;
  if (from->nlayers != into->nlayers || p.pshift != q.pshift || p.NKV != q.NKV || p.dshift != q.dshift ||
      from->layers[0].device != into->layers[0].device)
    return op_fail(ANE_ERR_ARG, "storiesane %s: the pools differ in layers, page_tokens, kv_heads, head_dim or device", op);
  if (!args) return op_fail(ANE_ERR_ARG, "storiesane %s: null arguments", op);
  const ane_kv8_copy_args& g = *args;
  if (g.n < 0 || g.n > 1 << 24) return op_fail(ANE_ERR_ARG, "storiesane %s: n=%d want 0..%d", op, g.n, 1 << 24);
  if (g.n == 0) return ANE_OK;  // an empty tensor may have no address
  if (!g.src || !g.dst) return op_fail(ANE_ERR_ARG, "storiesane %s: null buffer", op);
  const int device = from->layers[0].device;
  DeviceScope dev(device);
  if (dev.status() != hipSuccess) return device_error(op, device, dev.status());
  const hipStream_t st = (hipStream_t)stream;
  for (int l0 = 0; l0 < from->nlayers; l0 += kMaxLayers) {
    Layers x, y;
    const int n = layers_of(*from, l0, &x);
    layers_of(*into, l0, &y);
    const int group = group_of(p, g.n, n);
    const bool far = g.n * bytes_of(p, n) >= kFar;
    const int most = (1 << 23) / blocks_of(1, n, group);  // pages of a launch, which has fewer than 2^32 threads
    for (int i = 0; i < g.n; i += most)
      hipLaunchKernelGGL(far ? copy_kernel<true> : copy_kernel<false>,
                         dim3(blocks_of(std::min(most, g.n - i), n, group)), dim3(256), 0, st, p, q.pages, x, y, n,
                         group, g.src + i, g.dst + i, g.tokens ? g.tokens + i : nullptr);
  }
  return launched(op);
}

extern "C" int ane_debug_kv8_copy_form(const ane_kv8_pool* pool, int32_t pages, int32_t* out) {
  const char* op = "debug kv8 copy form";
  Pool p;
  const int rc = check_pool(op, pool, false, &p);
  if (rc) return rc;
  if (!out || pages < 0 || pages > 1 << 24) return op_fail(ANE_ERR_ARG, "storiesane %s: null buffer, or pages=%d", op, pages);
  const int n = std::min(kMaxLayers, pool->nlayers);
  out[0] = pages * bytes_of(p, n) >= kFar;
  out[1] = group_of(p, pages, n);
  return ANE_OK;
}
