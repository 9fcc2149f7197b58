// The paged 8-bit key/value cache: index arithmetic and codes shared by the
// append and attention kernels (include/ane_serve.h has the layouts).
//
// Every index that comes from device memory (offsets, starts, page ids) is
// brought into range here, by functions that also run on the host, where
// ane_debug_kv8_item lets a test walk them without a GPU.
#pragma once
#include <math.h>

#include "../../include/ane_hip.h"
#include "../../include/ane_serve.h"
#include "hip_common.h"

namespace ane {

constexpr int kKvExpMin = -15, kKvExpMax = 8;
constexpr int kKvMaxGroup = 32;  // query heads per key/value head

// A batch of new tokens as the kernels take it.
struct Kv8Batch {
  const int* table;
  const int* start;
  const int* offsets;
  int table_stride, table_pages, nseq, rows;
  int pages, pshift, NKV;  // of the cache; page_tokens = 1 << pshift
};

__host__ __device__ __forceinline__ int clampi(int x, int lo, int hi) { return x < lo ? lo : x > hi ? hi : x; }

// Rows [row0, row0 + n) of sequence i, the first at position st; positions
// from the table's end on are cut off.
struct Kv8Seq {
  int row0, n, st;
};
__host__ __device__ __forceinline__ Kv8Seq kv8_seq(const Kv8Batch& b, int i) {
  Kv8Seq s;
  s.row0 = clampi(b.offsets[i], 0, b.rows);
  s.n = clampi(b.offsets[i + 1], s.row0, b.rows) - s.row0;
  const int cap = b.table_pages << b.pshift;  // at most 2^30, checked on the host
  s.st = clampi(b.start[i], 0, cap);
  s.n = s.n < cap - s.st ? s.n : cap - s.st;
  return s;
}
// The page's id, or -1 where the table names none of the pool.
__host__ __device__ __forceinline__ int kv8_page(const Kv8Batch& b, int i, int pg) {
  const int id = b.table[(size_t)i * b.table_stride + pg];
  return (unsigned)id < (unsigned)b.pages ? id : -1;
}

// Work items are numbered so that an item's sequence follows from offsets
// alone, without a pass that counts: sequence i has the items f(i) ..
// f(i + 1) - 1 with f(i) = floor((offsets[i] + i * slack) / width), which are
// at least floor((n + slack) / width) of them.  Tiles of w tokens: width = w,
// slack = w - 1 is the ceil(n / w) that n rows need (one each where every
// sequence has one new token and slack, so a decoding step has no empty
// items).  Pages that n rows can touch: floor((n + P - 2) / P) + 1, so width =
// P, slack = 2 P - 2.  Surplus items are empty.
struct Kv8Items {
  uint32_t width, slack;
};
__host__ __device__ __forceinline__ Kv8Items kv8_tiles(int w) { return {(uint32_t)w, (uint32_t)w - 1}; }
__host__ __device__ __forceinline__ Kv8Items kv8_pages(int page) { return {(uint32_t)page, 2 * (uint32_t)page - 2}; }
// rows <= 2^30 and nseq <= 65536 (kv8_check): 32 bits hold the sums
__host__ __device__ __forceinline__ uint32_t kv8_first(const Kv8Batch& b, Kv8Items t, int i) {
  return ((uint32_t)clampi(b.offsets[i], 0, b.rows) + (uint32_t)i * t.slack) / t.width;
}
inline uint32_t kv8_count(int nseq, int rows, Kv8Items t) {
  return ((uint32_t)rows + (uint32_t)nseq * t.slack) / t.width;
}

// The sequence of an item -- the largest i with f(i) <= item -- and its rows:
// 64 candidates a round, so up to 64 sequences take one load's latency, up to
// 4096 two.  In the last round each lane holds its own sequence's numbers, and
// the chosen lane's become scalars, without another load.  Offsets that do
// not rise lead to some i in [0, nseq), never outside.
struct Kv8Found {
  int i;
  Kv8Seq s;
  uint32_t first;  // f(i)
};
__host__ __device__ __forceinline__ Kv8Found kv8_find(const Kv8Batch& b, Kv8Items t, uint32_t item) {
  int lo = 0, span = b.nseq;
  while (span > 64) {
    const int step = (span + 63) >> 6;
    int below = 0;
#ifdef __HIP_DEVICE_COMPILE__
    const int lane = threadIdx.x & 63;
    below = __popcll(__ballot(lane * step < span && kv8_first(b, t, lo + lane * step) <= item));
#else
    for (int lane = 0; lane < 64; lane++)
      below += lane * step < span && kv8_first(b, t, lo + lane * step) <= item;
#endif
    const int c = below > 0 ? below - 1 : 0;
    const int rest = span - c * step;
    lo += c * step;
    span = step < rest ? step : rest;
  }
#ifdef __HIP_DEVICE_COMPILE__
  const int lane = threadIdx.x & 63;
  const int mine = lo + min(lane, span - 1);
  const Kv8Seq s = kv8_seq(b, mine);
  const uint32_t first = ((uint32_t)s.row0 + (uint32_t)mine * t.slack) / t.width;
  const int below = __popcll(__ballot(lane < span && first <= item));
  const int c = below > 0 ? below - 1 : 0;
  return {__builtin_amdgcn_readfirstlane(lo + c),
          {__builtin_amdgcn_readlane(s.row0, c), __builtin_amdgcn_readlane(s.n, c), __builtin_amdgcn_readlane(s.st, c)},
          (uint32_t)__builtin_amdgcn_readlane((int)first, c)};
#else
  int below = 0;
  for (int lane = 0; lane < span; lane++) below += kv8_first(b, t, lo + lane) <= item;
  const int i = lo + (below > 0 ? below - 1 : 0);
  return {i, kv8_seq(b, i), kv8_first(b, t, i)};
#endif
}

// What an item takes: tokens of sequence `seq` at positions pos .. pos + n - 1,
// in rows row .. row + n - 1 (n = 0: nothing).
struct Kv8Span {
  int seq, row, n, pos;
};
__host__ __device__ __forceinline__ Kv8Span kv8_cut(const Kv8Seq& s, int i, int64_t t0, int64_t t1) {
  if (t0 < s.st) t0 = s.st;
  if (t1 > (int64_t)s.st + s.n) t1 = (int64_t)s.st + s.n;
  if (t0 >= t1) return {i, 0, 0, 0};
  return {i, s.row0 + (int)(t0 - s.st), (int)(t1 - t0), (int)t0};
}
// the item-th tile of `w` tokens
__host__ __device__ __forceinline__ Kv8Span kv8_tile_span(const Kv8Batch& b, int w, uint32_t item) {
  const Kv8Found f = kv8_find(b, kv8_tiles(w), item);
  const int64_t k = (int64_t)item - f.first;
  if (k < 0) return {f.i, 0, 0, 0};
  return kv8_cut(f.s, f.i, f.s.st + k * w, f.s.st + (k + 1) * w);
}
// The same tiles with the longest contexts first, for at most 64 sequences:
// those of the sequence that ends last, its own last tile first, and so on.
// A lane holds a sequence and adds up the tiles of those before it.
__host__ __device__ __forceinline__ Kv8Span kv8_tile_longest(const Kv8Batch& b, int w, uint32_t item) {
#ifdef __HIP_DEVICE_COMPILE__
  const int lane = threadIdx.x & 63;
  Kv8Seq s = kv8_seq(b, min(lane, b.nseq - 1));
  if (lane >= b.nseq) s.n = 0;
  const int end = s.st + s.n;
  const uint32_t tiles = ((uint32_t)s.n + w - 1) / w;
  uint32_t first = 0;
  for (int j0 = 0; j0 < b.nseq; j0 += 4)  // four at a time: lanes past the last have no tiles
#pragma unroll
    for (int j = j0; j < j0 + 4; j++) {
      const int e = __builtin_amdgcn_readlane(end, j);
      first += e > end || (e == end && j < lane) ? (uint32_t)__builtin_amdgcn_readlane((int)tiles, j) : 0;
    }
  const uint64_t mine = __ballot(first <= item && item - first < tiles);
  if (mine == 0) return {0, 0, 0, 0};
  const int i = __ffsll((unsigned long long)mine) - 1;
  s = {__builtin_amdgcn_readlane(s.row0, i), __builtin_amdgcn_readlane(s.n, i), __builtin_amdgcn_readlane(s.st, i)};
  const uint32_t last = (uint32_t)__builtin_amdgcn_readlane((int)(first + tiles), i) - 1;
#else
  int i = 0;
  Kv8Seq s;
  uint32_t last = 0;
  for (;; i++) {
    if (i == b.nseq) return {0, 0, 0, 0};
    s = kv8_seq(b, i);
    const uint32_t tiles = ((uint32_t)s.n + w - 1) / w;
    uint32_t first = 0;
    for (int j = 0; j < b.nseq; j++) {
      const Kv8Seq o = kv8_seq(b, j);
      if (o.st + o.n > s.st + s.n || (o.st + o.n == s.st + s.n && j < i)) first += ((uint32_t)o.n + w - 1) / w;
    }
    last = first + tiles - 1;
    if (first <= item && item - first < tiles) break;
  }
#endif
  const int64_t k = last - item;
  return kv8_cut(s, i, s.st + k * w, s.st + (k + 1) * w);
}
// the rows of the item-th page that gets any (page pos >> pshift of the table)
__host__ __device__ __forceinline__ Kv8Span kv8_page_span(const Kv8Batch& b, uint32_t item) {
  const Kv8Found f = kv8_find(b, kv8_pages(1 << b.pshift), item);
  const int64_t k = (int64_t)item - f.first;
  if (k < 0) return {f.i, 0, 0, 0};
  const int64_t pg = (f.s.st >> b.pshift) + k;
  return kv8_cut(f.s, f.i, pg << b.pshift, (pg + 1) << b.pshift);
}

// The same with an item for every row: a page belongs to its first one, the
// others are empty.  Fewer items where sequences have a token each.
__host__ __device__ __forceinline__ Kv8Span kv8_row_page_span(const Kv8Batch& b, uint32_t item) {
  const Kv8Found f = kv8_find(b, kv8_tiles(1), item);
  const int64_t k = (int64_t)item - f.first, t = f.s.st + k, page = 1 << b.pshift;
  if (k < 0 || (k > 0 && (t & (page - 1)))) return {f.i, 0, 0, 0};
  return kv8_cut(f.s, f.i, t, (t | (page - 1)) + 1);
}

// e4m3 -> fp16 with the exponent applied, two codes of a dword at a time;
// exact, since every code * 2^e is an fp16 number.
typedef __fp16 fp16x2_t __attribute__((ext_vector_type(2)));
template <bool HI>
__device__ __forceinline__ half2v kv8_up(uint32_t codes, float scale) {
  return __builtin_bit_cast(half2v, __builtin_amdgcn_cvt_scalef32_pk_f16_fp8((int)codes, scale, HI));
}
__device__ __forceinline__ float kv8_scale(int e) { return __int_as_float((127 + e) << 23); }

// The smallest exponent in [-15, 8] at which amax <= 448 * 2^e (448 = 1.75 *
// 2^8); amax as the bits of a non-negative float.
__device__ __forceinline__ int kv8_exponent(uint32_t amax_bits) {
  const int e = (int)(amax_bits >> 23) - 127 - 8 + ((amax_bits & 0x7fffff) > 0x600000 ? 1 : 0);
  return clampi(e, kKvExpMin, kKvExpMax);
}

// Host: checks the cache of operator `op`; ANE_OK or ANE_ERR_ARG with the
// message set.
int kv8_cache_check(const char* op, const ane_kv8_cache* c);

// Host: checks the cache and the batch of operator `op` and fills the
// kernels' form; ANE_OK or ANE_ERR_ARG with the message set.
int kv8_check(const char* op, const ane_kv8_cache* c, const ane_kv8_batch* b, Kv8Batch* out);

// Rows q | k | v of the decoder's product as its fp32 sums [splits][kDecRows][n]
// (added, times row_scale if there is one).  A set *err: nothing is appended (a
// step then attends over what is there; its outputs are redone).
struct Kv8Sums {
  const float* part = nullptr;
  int splits = 0, n = 0;
  const float* row_scale = nullptr;
  const int* err = nullptr;
};
// ane_kv8_append; from: the rows come from there and not from q, k and v
// (head dimension 64).
int kv8_append(const ane_kv8_cache* cache, const ane_kv8_batch* batch, const ane_kv8_append_args* args,
               const Kv8Sums* from, void* stream);

// ane_kv8_attend; frag: out is the decoder's 64-row activation fragments
// (decode.h), its strides unused.
int kv8_attend(const ane_kv8_cache* cache, const ane_kv8_batch* batch, const ane_kv8_attend_args* args, bool frag,
               void* stream);

// Both for a step of at most one new token a sequence, in one launch where the
// contexts stay whole (q_out is then not written); the same bits.
int kv8_step(const ane_kv8_cache* cache, const ane_kv8_batch* batch, const ane_kv8_append_args* append,
             const Kv8Sums* from, const ane_kv8_attend_args* args, bool frag, void* stream);

// Whether fp16 rows of [rows][heads][dh] with these strides do not overlap
// (outputs; either order of the two outer dimensions).
inline bool kv8_apart(int64_t rows, int64_t row, int64_t heads, int64_t head, int64_t dh) {
  const int64_t r = rows > 1 ? row : 0, h = heads > 1 ? head : 0;
  return ((heads == 1 || h >= dh) && (rows == 1 || r >= (heads - 1) * h + dh)) ||
         ((rows == 1 || r >= dh) && (heads == 1 || h >= (rows - 1) * r + dh));
}

// A tensor of [rows][heads][width], for the question whether two of them share
// memory.  All in bytes.
struct Extent {
  uintptr_t at;
  int64_t rows, row, heads, head, width;
};
// Whether they do.  Rows that lie between another tensor's rows do not.  Exact,
// but for tensors that lie through each other in different orders and are
// large, which count as sharing.
bool share_memory(Extent a, Extent b);
inline Extent fp16_rows(const void* p, int64_t rows, int64_t row, int64_t heads, int64_t head, int64_t dh) {
  return {(uintptr_t)p, rows, row * 2, heads, head * 2, dh * 2};
}

// The buffers of a call, for the refusal of outputs that share memory with
// another one.  Two with the same `pair` (not 0) may be one and the same.
struct Buffer {
  const char* name;
  Extent at;
  bool out;
  int pair = 0;
};
inline Extent flat(const void* p, int64_t bytes) { return {(uintptr_t)p, 1, 0, 1, 0, bytes}; }
inline Extent row_major(const void* p, int64_t rows, int64_t row, int64_t width) {
  return {(uintptr_t)p, rows, row, 1, 0, width};
}
// ANE_OK, or ANE_ERR_ARG with the message set; null buffers share nothing.
int check_apart(const char* op, const Buffer* b, int n);

// Makes the cache's device current for a scope (launches go to the current
// device; the caller's choice comes back).
class DeviceScope {
 public:
  explicit DeviceScope(int device) {
    status_ = taken(hipGetDevice(&before_));
    if (status_ == hipSuccess && before_ != device) {
      status_ = taken(hipSetDevice(device));
      changed_ = status_ == hipSuccess;
    }
  }
  ~DeviceScope() {
    if (changed_) (void)hipSetDevice(before_);
  }
  DeviceScope(const DeviceScope&) = delete;
  DeviceScope& operator=(const DeviceScope&) = delete;
  hipError_t status() const { return status_; }

 private:
  int before_ = 0;
  bool changed_ = false;
  hipError_t status_ = hipSuccess;
};

}  // namespace ane
