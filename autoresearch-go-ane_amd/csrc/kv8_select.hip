// Which pages of a long context a query attends to: bounds on the keys of each
// page (ane_kv8_bound), and the choice of the pages whose bounds promise most
// (ane_kv8_select); formulas in include/ane_serve.h.
//
// A key k of a page lies in the box smallest..largest, so q . k is at most
// sum_d max(q_d largest_d, q_d smallest_d) = q+ . largest + q- . smallest: a
// product of 2 head_dim terms, and of whole numbers, as the boxes are and the
// queries become.  The matrix cores add it up exactly (MFMA i8 16x16x64, at
// most 256 * 127^2 < 2^24), and powers of two scale it exactly in fp32, so the
// choice does not depend on the order of any sum.
#include <algorithm>

#include "kv8.h"
#include "op_error.h"

namespace ane {

namespace {

typedef int intx4 __attribute__((ext_vector_type(4)));

constexpr int kUnitMin = -30;

// the smallest exponent from kUnitMin on at which amax <= 127 * 2^e; amax finite, >= 0
__device__ __forceinline__ int unit_of(float amax) {
  const uint32_t b = __float_as_uint(amax);  // 127 = 1.984375 * 2^6
  return max((int)(b >> 23) - 127 - 6 + ((b & 0x7fffff) > 0x7e0000 ? 1 : 0), kUnitMin);
}

// ---- bounds --------------------------------------------------------------------

struct BoundArgs {
  Kv8Batch b;
  const uint8_t* k;
  const int8_t* k_exp;
  int8_t *box, *unit;
};

__device__ __forceinline__ half2v min2(half2v a, half2v b) { return __builtin_elementwise_min(a, b); }
__device__ __forceinline__ half2v max2(half2v a, half2v b) { return __builtin_elementwise_max(a, b); }
__device__ __forceinline__ half2v shfl2(half2v x, int o) {
  return __builtin_bit_cast(half2v, __shfl_xor(__builtin_bit_cast(int, x), o, 64));
}

// A wave per page that got rows and key/value head.  A lane takes 16
// dimensions of every 64 / LR-th row; the codes' own values, which are fp16
// numbers, are compared, and the page's exponent comes in at the end.  A
// comparison with NaN takes the number.
template <int DH>
__global__ __launch_bounds__(64) void bound_kernel(BoundArgs a) {
  constexpr int LR = DH / 16, RP = 64 / LR;  // lanes of a row, rows of a pass
  const Kv8Batch& b = a.b;
  const int h = blockIdx.y;
  const Kv8Span span = kv8_page_span(b, blockIdx.x);
  if (span.n == 0) return;
  const int id = kv8_page(b, span.seq, span.pos >> b.pshift);
  if (id < 0) return;
  const int lane = threadIdx.x, sub = lane / LR, P = 1 << b.pshift;
  const int rows = (span.pos + span.n - 1 & (P - 1)) + 1;
  const size_t ph = (size_t)id * b.NKV + h;
  const uint8_t* p = a.k + (ph << b.pshift) * DH + lane % LR * 16;
  const half_t inf = (half_t)INFINITY;
  half2v lo[8], hi[8];
#pragma unroll
  for (int j = 0; j < 8; j++) {
    lo[j] = half2v{inf, inf};
    hi[j] = half2v{-inf, -inf};
  }
  for (int r = sub; r < rows; r += RP) {
    const u32x4 c = *reinterpret_cast<const u32x4*>(p + r * DH);
#pragma unroll
    for (int j = 0; j < 4; j++) {
      const half2v x = kv8_up<false>(c[j], 1.f), y = kv8_up<true>(c[j], 1.f);
      lo[2 * j] = min2(lo[2 * j], x);
      hi[2 * j] = max2(hi[2 * j], x);
      lo[2 * j + 1] = min2(lo[2 * j + 1], y);
      hi[2 * j + 1] = max2(hi[2 * j + 1], y);
    }
  }
  const float ks = kv8_scale(a.k_exp[ph]);
  float amax = 0.f;
  float l[16], u[16];
#pragma unroll
  for (int j = 0; j < 8; j++) {
#pragma unroll
    for (int o = 32; o >= LR; o >>= 1) {
      lo[j] = min2(lo[j], shfl2(lo[j], o));
      hi[j] = max2(hi[j], shfl2(hi[j], o));
    }
#pragma unroll
    for (int e = 0; e < 2; e++) {
      // no number: lo = inf, hi = -inf (or both NaN)
      const bool some = lo[j][e] <= hi[j][e];
      l[2 * j + e] = some ? (float)lo[j][e] * ks : 0.f;
      u[2 * j + e] = some ? (float)hi[j][e] * ks : 0.f;
      amax = fmaxf(amax, fmaxf(-l[2 * j + e], u[2 * j + e]));
    }
  }
#pragma unroll
  for (int o = 1; o < LR; o <<= 1) amax = fmaxf(amax, __shfl_xor(amax, o, 64));
  const int e = unit_of(amax);
  const float inv = kv8_scale(-e);
  if (sub == 0) {
    u32x4 x, y;
#pragma unroll
    for (int j = 0; j < 4; j++) {
      x[j] = y[j] = 0;
#pragma unroll
      for (int i = 0; i < 4; i++) {
        x[j] |= ((uint32_t)(int)ceilf(u[4 * j + i] * inv) & 0xff) << (8 * i);
        y[j] |= ((uint32_t)(int)floorf(l[4 * j + i] * inv) & 0xff) << (8 * i);
      }
    }
    u32x4* box = reinterpret_cast<u32x4*>(a.box + ph * 2 * DH);
    box[lane] = x;
    box[LR + lane] = y;
    if (lane == 0) a.unit[ph] = (int8_t)e;
  }
}

// ---- choice --------------------------------------------------------------------

struct SelectArgs {
  Kv8Batch b;
  const half_t* q;
  const int8_t *box, *unit;
  int* blocks;
  int64_t q_row, q_head;
  int G, count, first, recent;
};

// A page's place in the order of the choice: fp32 scores as whole numbers that
// rise with them.
constexpr uint32_t kNever = 0, kAlways = 0xffffffffu;
__device__ __forceinline__ uint32_t key_of(float x) {
  const uint32_t b = __float_as_uint(x);
  return b >> 31 ? ~b : b | 0x80000000u;
}

constexpr int kKeys = 4096;  // pages whose keys are held at a time

// NW waves a row and key/value head.  The keys of kKeys pages at a time lie in
// LDS: all of a context that is no longer, otherwise each pass over the keys
// computes them again.
template <int DH, int NT, int NW>
__global__ __launch_bounds__(64 * NW) void select_kernel(SelectArgs a) {
  constexpr int NM = DH / 32;  // products of 64 terms
  __shared__ uint32_t keys[kKeys];
  __shared__ int sums[2][NW];
  const Kv8Batch& b = a.b;
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6, col = lane & 15, g = lane >> 4;
  const int h = blockIdx.x % b.NKV;
  const Kv8Span span = kv8_tile_span(b, 1, blockIdx.x / b.NKV);
  if (span.n == 0) return;
  const int np = (span.pos >> b.pshift) + 1;  // pages of the context
  const int* trow = b.table + (size_t)span.seq * b.table_stride;

  // the queries, rows 16 t + col of the product: largest's factors, then smallest's
  intx4 z[NT][NM];
  float up[NT][4], off[NT][4];  // what the lane's rows of the result are scaled by; rows of no head: -inf
#pragma unroll
  for (int t = 0; t < NT; t++) {
    const int head = min(16 * t + col, a.G - 1);
    const half_t* p = a.q + (int64_t)span.row * a.q_row + (h * a.G + head) * a.q_head;
    // the lane's 16 dimensions of each 64; its row's other 48 lie with lanes col + 16 i
    float x[DH / 64][16];
    float amax = 0.f;
#pragma unroll
    for (int m = 0; m < DH / 64; m++)
#pragma unroll
      for (int v = 0; v < 2; v++) {
        const half8 y = ld_h8(p + 64 * m + 16 * g + 8 * v);
#pragma unroll
        for (int j = 0; j < 8; j++) {
          float w = (float)y[j];
          w = w == w ? fminf(fmaxf(w, -65504.f), 65504.f) : 0.f;
          x[m][8 * v + j] = w;
          amax = fmaxf(amax, fabsf(w));
        }
      }
    amax = fmaxf(amax, __shfl_xor(amax, 16, 64));
    amax = fmaxf(amax, __shfl_xor(amax, 32, 64));
    const int e = unit_of(amax);
    const float inv = kv8_scale(-e);
#pragma unroll
    for (int m = 0; m < DH / 64; m++)
#pragma unroll
      for (int j = 0; j < 4; j++) {
        uint32_t pos = 0, neg = 0;
#pragma unroll
        for (int i = 0; i < 4; i++) {
          const int w = (int)rintf(x[m][4 * j + i] * inv);
          pos |= ((uint32_t)max(w, 0) & 0xff) << (8 * i);
          neg |= ((uint32_t)min(w, 0) & 0xff) << (8 * i);
        }
        z[t][m][j] = (int)pos;
        z[t][DH / 64 + m][j] = (int)neg;
      }
#pragma unroll
    for (int j = 0; j < 4; j++) {
      const int row = 4 * g + j;
      const int er = __shfl(e, row, 64);
      up[t][j] = 16 * t + row < a.G ? kv8_scale(er) : 0.f;
      off[t][j] = 16 * t + row < a.G ? 0.f : -INFINITY;
    }
  }

  // keys of pages p0 .. p1 - 1 to LDS, 16 a wave at a time
  const auto fill = [&](int p0, int p1) {
    for (int c = p0 + wave * 16; c < p1; c += NW * 16) {
      const int page = c + col;
      const int id = page < np ? trow[page] : -1;
      const bool there = (unsigned)id < (unsigned)b.pages;
      const size_t ph = (size_t)(there ? id : 0) * b.NKV + h;
      const int8_t* box = a.box + ph * (2 * DH) + 16 * g;
      const int unit = a.unit[ph];
      intx4 w[NM];
#pragma unroll
      for (int m = 0; m < NM; m++) w[m] = *reinterpret_cast<const intx4*>(box + 64 * m);
      float best = -INFINITY;
#pragma unroll
      for (int t = 0; t < NT; t++) {
        intx4 s = {0, 0, 0, 0};
#pragma unroll
        for (int m = 0; m < NM; m++) s = __builtin_amdgcn_mfma_i32_16x16x64_i8(z[t][m], w[m], s, 0, 0, 0);
#pragma unroll
        for (int j = 0; j < 4; j++) best = fmaxf(best, __builtin_fmaf((float)s[j], up[t][j], off[t][j]));
      }
      best = fmaxf(best, __shfl_xor(best, 16, 64));
      best = fmaxf(best, __shfl_xor(best, 32, 64));
      if (g == 0 && page < p1) {
        uint32_t key = key_of(best * kv8_scale(max(unit, kUnitMin)));
        if (page < a.first || page >= np - a.recent) key = kAlways;
        keys[page - p0] = there ? key : kNever;
      }
    }
  };
  const bool once = np <= kKeys;
  // f(page, key, whether it is one) over the pages, in order, all threads at a time
  const auto each = [&](bool filled, auto f) {
    for (int p0 = 0; p0 < np; p0 += kKeys) {
      const int p1 = min(np, p0 + kKeys);
      if (!once || !filled) {
        __syncthreads();
        fill(p0, p1);
        __syncthreads();
      }
      for (int c = p0; c < p1; c += 64 * NW) f(c + tid, c + tid < p1 ? keys[c + tid - p0] : kNever, c + tid < p1);
    }
  };
  // the sum of x over the waves (x the same in a wave's lanes)
  int turn = 0;
  const auto total = [&](int x) {
    if (NW == 1) return x;
    if (lane == 0) sums[turn][wave] = x;
    __syncthreads();
    int s = 0;
#pragma unroll
    for (int w = 0; w < NW; w++) s += sums[turn][w];
    turn ^= 1;
    return s;
  };
  const auto count_from = [&](bool filled, uint32_t bar) {
    int n = 0;
    each(filled, [&](int, uint32_t key, bool is) { n += __popcll(__ballot(is && key >= bar)); });
    return total(n);
  };

  // The lowest key of the choice, from the top bit down: the largest bar that
  // `count` pages reach.  Where exactly that many do, it is found.
  uint32_t bar = 1;
  int reach = count_from(false, bar);
  if (reach > a.count) {
    bar = 0;
    for (uint32_t bit = 0x80000000u; bit; bit >>= 1) {
      const int n = count_from(true, bar | bit);
      if (n >= a.count) {
        bar |= bit;
        reach = n;
        if (n == a.count) break;
      }
    }
  }
  // pages above the bar, and as many at the bar, from the lowest, as are left
  int at_bar = 0x7fffffff;  // how many of those with the bar's own key
  if (reach > a.count) at_bar = a.count - (bar == kAlways ? 0 : count_from(true, bar + 1));
  int* out = a.blocks + ((size_t)span.row * b.NKV + h) * a.count;
  int taken = 0, equal = 0;  // before this stretch of pages
  each(true, [&](int page, uint32_t key, bool is) {
    const uint64_t eq = __ballot(is && key == bar);
    const uint64_t below = (1ull << lane) - 1;
    int eq_before = equal, n = __popcll(eq);
    if (NW > 1) {
      if (lane == 0) sums[turn][wave] = n;
      __syncthreads();
      n = 0;
#pragma unroll
      for (int w = 0; w < NW; w++) {
        eq_before += w < wave ? sums[turn][w] : 0;
        n += sums[turn][w];
      }
      turn ^= 1;
    }
    equal += n;
    const bool take = is && (key > bar || (key == bar && eq_before + __popcll(eq & below) < at_bar));
    const uint64_t tk = __ballot(take);
    int before = taken;
    n = __popcll(tk);
    if (NW > 1) {
      if (lane == 0) sums[turn][wave] = n;
      __syncthreads();
      n = 0;
#pragma unroll
      for (int w = 0; w < NW; w++) {
        before += w < wave ? sums[turn][w] : 0;
        n += sums[turn][w];
      }
      turn ^= 1;
    }
    taken += n;
    if (take) out[before + __popcll(tk & below)] = page;
  });
  for (int c = taken + tid; c < a.count; c += 64 * NW) out[c] = -1;
}

bool aligned16(const void* p) { return ((uintptr_t)p & 15) == 0; }

int check_bounds(const char* op, const ane_kv8_bounds* x) {
  if (!x || !x->box || !x->unit || !aligned16(x->box))
    return op_fail(ANE_ERR_ARG, "storiesane %s: null bounds, or box not 16-byte aligned", op);
  return ANE_OK;
}

int check_sizes(const char* op, const Kv8Batch& b, int heads, int count) {
  if (heads < 1 || heads % b.NKV || heads / b.NKV > kKvMaxGroup)
    return op_fail(ANE_ERR_ARG, "storiesane %s: heads=%d must be 1..%d times kv_heads=%d", op, heads, kKvMaxGroup,
                   b.NKV);
  if (count < 1 || count > 65536) return op_fail(ANE_ERR_ARG, "storiesane %s: count=%d want 1..65536", op, count);
  if ((int64_t)kv8_count(b.nseq, b.rows, kv8_tiles(1)) * b.NKV > 0x7fffffff)
    return op_fail(ANE_ERR_ARG, "storiesane %s: rows=%d are too many for one launch", op, b.rows);
  return ANE_OK;
}

template <int DH>
void launch(const SelectArgs& a, hipStream_t st) {
  const dim3 grid(kv8_count(a.b.nseq, a.b.rows, kv8_tiles(1)) * a.b.NKV);
  if (a.G <= 16) hipLaunchKernelGGL((select_kernel<DH, 1, 4>), grid, dim3(256), 0, st, a);
  else hipLaunchKernelGGL((select_kernel<DH, 2, 4>), grid, dim3(256), 0, st, a);
}

}  // namespace

}  // namespace ane

using namespace ane;

extern "C" int ane_kv8_bound(const ane_kv8_cache* cache, const ane_kv8_bounds* bounds, const ane_kv8_batch* batch,
                             void* stream) {
  const char* op = "kv8 bound";
  BoundArgs a;
  int rc = kv8_check(op, cache, batch, &a.b);
  if (!rc) rc = check_bounds(op, bounds);
  if (rc || a.b.nseq == 0 || a.b.rows == 0) return rc;
  DeviceScope dev(cache->device);
  if (dev.status() != hipSuccess)
    return op_fail(ANE_ERR_HIP, "storiesane %s: device %d: %s", op, cache->device, hipGetErrorString(dev.status()));
  a.k = (const uint8_t*)cache->k; a.k_exp = cache->k_exp; a.box = bounds->box; a.unit = bounds->unit;
  const dim3 grid(kv8_count(a.b.nseq, a.b.rows, kv8_pages(1 << a.b.pshift)), a.b.NKV);
  const hipStream_t st = (hipStream_t)stream;
  if (cache->head_dim == 64) hipLaunchKernelGGL(bound_kernel<64>, grid, dim3(64), 0, st, a);
  else hipLaunchKernelGGL(bound_kernel<128>, grid, dim3(64), 0, st, a);
  const hipError_t h = hipGetLastError();
  if (h != hipSuccess) return op_fail(ANE_ERR_HIP, "storiesane %s: %s", op, hipGetErrorString(h));
  return ANE_OK;
}

extern "C" int64_t ane_kv8_select_workspace(const ane_kv8_cache* cache, const ane_kv8_batch* batch, int32_t heads,
                                            int32_t count) {
  const char* op = "kv8 select workspace";
  Kv8Batch b;
  int rc = kv8_check(op, cache, batch, &b);
  if (!rc) rc = check_sizes(op, b, heads, count);
  return rc ? rc : 0;
}

extern "C" int ane_kv8_select(const ane_kv8_cache* cache, const ane_kv8_bounds* bounds, const ane_kv8_batch* batch,
                              const ane_kv8_select_args* args, void* stream) {
  const char* op = "kv8 select";
  SelectArgs a;
  int rc = kv8_check(op, cache, batch, &a.b);
  if (!rc) rc = check_bounds(op, bounds);
  if (rc) return rc;
  if (!args) return op_fail(ANE_ERR_ARG, "storiesane %s: null arguments", op);
  const ane_kv8_select_args& g = *args;
  rc = check_sizes(op, a.b, g.heads, g.count);
  if (rc) return rc;
  if (g.first < 0 || g.recent < 0 || (int64_t)g.first + g.recent > g.count)
    return op_fail(ANE_ERR_ARG, "storiesane %s: first=%d recent=%d want 0 or more, together at most count=%d", op,
                   g.first, g.recent, g.count);
  if (a.b.nseq == 0 || a.b.rows == 0) return ANE_OK;  // an empty tensor may have no address
  if (!g.q || !g.blocks) return op_fail(ANE_ERR_ARG, "storiesane %s: null buffer", op);
  if (g.q_row < 0 || g.q_row % 8 || g.q_head < 0 || g.q_head % 8 || !aligned16(g.q))
    return op_fail(ANE_ERR_ARG, "storiesane %s: strides %lld and %lld must be multiples of 8, q 16-byte aligned", op,
                   (long long)g.q_row, (long long)g.q_head);
  const Buffer buffers[] = {{"q", fp16_rows(g.q, a.b.rows, g.q_row, g.heads, g.q_head, cache->head_dim), false},
                            {"blocks", flat(g.blocks, (int64_t)a.b.rows * a.b.NKV * g.count * 4), true}};
  rc = check_apart(op, buffers, 2);
  if (rc) return rc;
  DeviceScope dev(cache->device);
  if (dev.status() != hipSuccess)
    return op_fail(ANE_ERR_HIP, "storiesane %s: device %d: %s", op, cache->device, hipGetErrorString(dev.status()));
  a.q = (const half_t*)g.q; a.box = bounds->box; a.unit = bounds->unit; a.blocks = g.blocks;
  a.q_row = g.q_row; a.q_head = g.q_head;
  a.G = g.heads / a.b.NKV; a.count = g.count; a.first = g.first; a.recent = g.recent;
  if (cache->head_dim == 64) launch<64>(a, (hipStream_t)stream);
  else launch<128>(a, (hipStream_t)stream);
  const hipError_t h = hipGetLastError();
  if (h != hipSuccess) return op_fail(ANE_ERR_HIP, "storiesane %s: %s", op, hipGetErrorString(h));
  return ANE_OK;
}
