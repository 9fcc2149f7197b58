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
#include "wave_ops.h"

namespace ane {

namespace {

typedef int intx4 __attribute__((ext_vector_type(4)));

// Units of bounds that an update has written are in between (keys are at most
// 448 * 2^8); of others they are taken so, and scores stay finite.
constexpr int kUnitMin = -30, kUnitMax = 40;

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
// over the lanes that are N apart, N = 4 or 8
template <int N, typename Op>
__device__ __forceinline__ half2v over_rows(half2v v, Op op) {
  if constexpr (N == 4) v = op(v, __builtin_bit_cast(half2v, row_ror<4>(__builtin_bit_cast(int, v))));
  v = op(v, __builtin_bit_cast(half2v, row_ror<8>(__builtin_bit_cast(int, v))));
  half2v w = v;
  swap16(v, w);
  v = op(v, w);
  w = v;
  swap32(v, w);
  return op(v, w);
}

// A wave per page that got rows and key/value head: launch and chain of
// offsets, page id and codes bound it (a token of one sequence 3.9 us, of 64 4.8,
// 841 rows of 5 chunks 4.7).  A lane takes 16
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
    lo[j] = over_rows<LR>(lo[j], [](half2v a, half2v b) { return min2(a, b); });
    hi[j] = over_rows<LR>(hi[j], [](half2v a, half2v b) { return max2(a, b); });
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
  int room;       // scores that LDS holds
  float* scores;  // [rows][NKV][table_pages], where the choice has a launch of its own
};

constexpr int kBins = 256;
constexpr int kHeld = 1024;  // pages of a token whose scores its waves hold in registers
constexpr int kFar = 32768;  // scores that LDS holds at most

// LDS accesses of a wave stay in order; this keeps the compiler to it.
__device__ __forceinline__ void in_order() {
  __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
  __builtin_amdgcn_wave_barrier();
}

// What the CW waves of a token choose with.
template <int CW>
struct Choice {
  int bins[kBins];
  __attribute__((aligned(16))) float few[64];
  int fews, sums[2][CW];
};

// The choice among scores that each(f) gives as f(page, score), a thread a page,
// in order (-inf behind the last), by CW waves: of one, without a barrier.
template <int CW, typename Each>
__device__ __forceinline__ void choose(Choice<CW>& c, const Each& each, int count, int* out) {
  constexpr int CT = 64 * CW;
  const int lane = threadIdx.x & 63, ct = threadIdx.x % CT;
  const int cw = __builtin_amdgcn_readfirstlane(ct >> 6);
  for (int i = ct; i < kBins; i += CT) c.bins[i] = 0;
  if (ct == 0) c.fews = 0;  // behind barriers before they count
  if constexpr (CW == 1) in_order();
  const auto meet = [] {
    if constexpr (CW > 1) __syncthreads();
    else in_order();
  };
  // over the waves, of values that are the same in a wave's lanes; and the sum
  // over those before
  int turn = 0;
  const auto over = [&](auto x, auto op) {
    if constexpr (CW > 1) {
      using T = decltype(x);
      if (lane == 0) c.sums[turn][cw] = __builtin_bit_cast(int, x);
      __syncthreads();
      x = over_lanes<CW>(__builtin_bit_cast(T, c.sums[turn][lane % CW]), op);
      turn ^= 1;
    }
    return x;
  };
  const auto ranked = [&](int x, int& before) {
    before = 0;
    if constexpr (CW > 1) {
      if (lane == 0) c.sums[turn][cw] = x;
      __syncthreads();
      const int y = c.sums[turn][lane % CW];
      turn ^= 1;
      x = 0;
#pragma unroll
      for (int w = 0; w < CW; w++) {
        const int k = __builtin_amdgcn_readlane(y, w);
        before += w < cw ? k : 0;
        x += k;
      }
    }
    return x;
  };
  const auto widest = [&](float x) { return over(over_lanes<64>(x, Max()), Max()); };
  const uint64_t below = (1ull << lane) - 1;
  int all = 0, always = 0;
  float hi = -INFINITY, lo = -INFINITY;  // of the scores in question; the lowest one negated until it is known
  each([&](int, float x) {
    all += __popcll(__ballot(x > -INFINITY));
    always += __popcll(__ballot(x == INFINITY));
    if (fabsf(x) < INFINITY) {
      hi = fmaxf(hi, x);
      lo = fmaxf(lo, -x);
    }
  });
  all = over(all, Sum());
  // what is taken: scores above the bar, and of those at the bar the first
  // `ties`, or all of them (-1)
  float bar = -INFINITY;
  int ties = 0;
  if (all > count) {
    always = over(always, Sum());
    int need = count - always, in = all - always;  // pages to be taken, of those in question
    bar = INFINITY;
    if (need > 0) {
      int bin = -1;
      float step = 0.f;
      const auto bin_of = [&](float x) {
        return x >= lo && x <= hi ? min((int)((x - lo) * step), kBins - 1) : -1;
      };
      if (in > 64) {
        hi = widest(hi);
        lo = -widest(lo);
        while (lo < hi) {
          step = (float)kBins / (hi - lo);
          each([&](int, float x) {
            const int k = bin_of(x);
            if (k >= 0) atomicAdd(&c.bins[k], 1);
          });
          meet();
          // pages in the bins above the lane's four, and in them
          int in_bin[4], sum = 0;
#pragma unroll
          for (int i = 0; i < 4; i++) {
            in_bin[i] = c.bins[kBins - 1 - (lane * 4 + i)];
            sum += in_bin[i];
          }
          int above = sum_up_to(sum) - sum, it = -1, left = 0, size = 0;
#pragma unroll
          for (int i = 0; i < 4; i++) {
            if (above < need && need <= above + in_bin[i]) {
              it = kBins - 1 - (lane * 4 + i);
              left = need - above;
              size = in_bin[i];
            }
            above += in_bin[i];
          }
          const int who = __ffsll((unsigned long long)__ballot(it >= 0)) - 1;
          bin = __builtin_amdgcn_readlane(it, who);
          need = __builtin_amdgcn_readlane(left, who);
          in = __builtin_amdgcn_readlane(size, who);
          if (in <= 64) break;
          float x1 = -INFINITY, x0 = -INFINITY;
          each([&](int, float x) {
            if (bin_of(x) == bin) {
              x1 = fmaxf(x1, x);
              x0 = fmaxf(x0, -x);
            }
          });
          hi = widest(x1);  // behind its barrier no wave reads the bins
          lo = -widest(x0);
          bin = -1;
          for (int i = ct; i < kBins; i += CT) c.bins[i] = 0;
          meet();
        }
      }
      if (in <= 64) {
        // the ones that are left, in any order
        int at = 0;
        each([&](int, float x) {
          const bool is = bin < 0 ? fabsf(x) < INFINITY : bin_of(x) == bin;
          const uint64_t who = __ballot(is);
          if (CW > 1 && who) {
            if (lane == 0) at = atomicAdd(&c.fews, __popcll(who));
            at = __builtin_amdgcn_readfirstlane(at);
          }
          if (is) c.few[at + __popcll(who & below)] = x;
          at += __popcll(who);
        });
        if (ct < 4 && in + ct < 64) c.few[in + ct] = -INFINITY;  // behind them, to whole words
        meet();
        const float x = c.few[min(lane, in - 1)];
        int above = 0, from = 0;
#pragma unroll 2
        for (int k = 0; k < in; k += 4) {
          const floatx4 y = *reinterpret_cast<const floatx4*>(c.few + k);
#pragma unroll
          for (int j = 0; j < 4; j++) {
            above += y[j] > x;
            from += y[j] >= x;
          }
        }
        const int who = __ffsll((unsigned long long)__ballot(lane < in && above < need && need <= from)) - 1;
        bar = __int_as_float(__builtin_amdgcn_readlane(__float_as_int(x), who));
        above = __builtin_amdgcn_readlane(above, who);
        from = __builtin_amdgcn_readlane(from, who);
        ties = need == from ? -1 : need - above;
      } else {  // all equal
        bar = lo;
        ties = need;
      }
    }
  }
  int taken = 0, equal = 0;  // before these 64 pages
  each([&](int page, float x) {
    bool take = x > bar || x == INFINITY || (ties < 0 && x == bar);
    int before;
    if (ties > 0) {
      const uint64_t eq = __ballot(x == bar);
      const int all_eq = ranked(__popcll(eq), before);
      take = take || (x == bar && equal + before + __popcll(eq & below) < ties);
      equal += all_eq;
    }
    const uint64_t tk = __ballot(take);
    const int all_tk = ranked(__popcll(tk), before);
    if (take) out[taken + before + __popcll(tk & below)] = page;
    taken += all_tk;
  });
  for (int i = taken + ct; i < count; i += CT) out[i] = -1;
}

// A block takes up to 4, 2 or 1 tokens of a sequence (whose query heads, up to 4,
// 8 or 16, or 32 with NT = 2, go into the 16 rows of a product) and a key/value
// head.
//
// First its NW waves score the context's pages for all the tokens: 64 pages a
// wave at a time, their ids with one load, their boxes in four products of 16.
// Row 4 g + j of a product is token j / (4 / TOK) and head g + 4 (j % (4 / TOK)),
// so that a token's heads are registers of a lane and rows of lanes.  Then each
// token is CW waves' own: one's, which needs no barrier, or where there is one
// token, all waves'.  Contexts that LDS does not hold are scored again, by those
// waves, in each pass over the scores.
//
// The choice.  The score of the last page to be taken is narrowed down by
// histograms between the lowest and the highest score in question, in steps of
// equal width (a step's number rises with the score whatever the rounding),
// until at most 64 pages are left, or ones that are all equal; then ranks are
// counted.  The bin that the last page lies in has neither all of them nor
// none, so every histogram leaves fewer.
//
// What bounds it: the chain of ids, boxes and scores, then the narrowing's steps,
// each an LDS round trip and a barrier (in a captured graph, 1 token of 20,000
// keys, 4 heads, 313 pages: 7.0 us; 64 tokens of 3500 to 24,000, 2 heads of 128,
// pages of 32: 12.1 us for 14 MB of boxes; 841 tokens of 4 heads in 5 chunks 9.8
// us).  Narrowing by halves, of bits or values, takes more such steps (21.6 us for
// the first with update and attention, by histograms 19.2).
//
// PART: a block leaves the scores of 64 NW pages of a token (and of those as many
// blocks on) to choose_kernel.
template <int DH, int NT, int TOK, int NW, int CW, bool PART>
__global__ __launch_bounds__(64 * NW) void select_kernel(SelectArgs a) {
  static_assert(!PART || TOK == 1);
  constexpr int NM = DH / 32;  // products of 64 terms
  constexpr int HJ = 4 / TOK;  // registers of a token
  static_assert(CW == 1 || CW == NW);
  constexpr int CH = NW / CW, CT = 64 * CW, R = kHeld / CT;
  extern __shared__ float scores[];  // [TOK][stride], room of them in all
  __shared__ Choice<CW> choices[PART ? 1 : CH];
  const Kv8Batch& b = a.b;
  const int tid = threadIdx.x, lane = tid & 63, col = lane & 15, g = lane >> 4;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int h = blockIdx.x % b.NKV;
  const Kv8Span span = kv8_tile_span(b, TOK, blockIdx.x / b.NKV);
  if (span.n == 0) return;
  const int np = ((span.pos + span.n - 1) >> b.pshift) + 1;  // pages of the last token's context
  const int* trow = b.table + (size_t)span.seq * b.table_stride;
  const auto id_of = [&](int page) {
    const int id = trow[min(page, np - 1)];
    return page < np && (unsigned)id < (unsigned)b.pages ? id : -1;
  };
  const int base = PART ? blockIdx.y * (64 * NW) : 0, on = 64 * NW * (PART ? gridDim.y : 1);
  if (base >= np) return;
  int id = id_of(base + tid);

  // the boxes of 64 neighbours (id: of the lane's page, or -1), and what the
  // lane's page's scores are scaled by (-1: it is not there)
  struct Boxes {
    intx4 w[4][NM];
    float scale;
  };
  const auto load = [&](int id) {
    Boxes x;
    const int unit = a.unit[(size_t)max(id, 0) * b.NKV + h];
#pragma unroll
    for (int c = 0; c < 4; c++) {
      const int i = __shfl(id, 16 * c + col, 64);
      const int8_t* box = a.box + ((size_t)max(i, 0) * b.NKV + h) * (2 * DH) + 16 * g;
#pragma unroll
      for (int m = 0; m < NM; m++) x.w[c][m] = *reinterpret_cast<const intx4*>(box + 64 * m);
    }
    x.scale = id < 0 ? -1.f : kv8_scale(clampi(unit, kUnitMin, kUnitMax));
    return x;
  };
  // the queries: largest's factors, then smallest's; on their way with the wave's
  // first boxes
  half8 qs[NT][DH / 64][2];
#pragma unroll
  for (int t = 0; t < NT; t++) {
    const int tok = min((col & 3) / HJ, span.n - 1), head = 16 * t + (col >> 2) + 4 * ((col & 3) % HJ);
    const half_t* p = a.q + (int64_t)(span.row + tok) * a.q_row + (h * a.G + min(head, a.G - 1)) * a.q_head;
#pragma unroll
    for (int m = 0; m < DH / 64; m++)
#pragma unroll
      for (int v = 0; v < 2; v++) qs[t][m][v] = ld_h8(p + 64 * m + 16 * g + 8 * v);
  }
  Boxes now = load(id);
  intx4 z[NT][NM];
  float up[NT][4], off[NT][4];  // what the lane's rows of the result are scaled by; rows of no head: -inf
#pragma unroll
  for (int t = 0; t < NT; t++) {
    // the lane's 16 dimensions of each 64; its row's other 48 lie with lanes col + 16 i
    float x[DH / 64][16];
    float amax = 0.f;
#pragma unroll
    for (int m = 0; m < DH / 64; m++)
#pragma unroll
      for (int v = 0; v < 2; v++) {
        const half8 y = qs[t][m][v];
#pragma unroll
        for (int j = 0; j < 8; j++) {
          float w = (float)y[j];
          w = w == w ? fminf(fmaxf(w, -65504.f), 65504.f) : 0.f;
          x[m][8 * v + j] = w;
          amax = fmaxf(amax, fabsf(w));
        }
      }
    float other = amax;  // the row's other dimensions lie in the other rows of lanes
    swap16(amax, other);
    amax = fmaxf(amax, other);
    other = amax;
    swap32(amax, other);
    amax = fmaxf(amax, other);
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
      const int er = __shfl(e, 4 * g + j, 64);
      const bool is = 16 * t + g + 4 * (j % HJ) < a.G;
      up[t][j] = is ? kv8_scale(er) : 0.f;
      off[t][j] = is ? 0.f : -INFINITY;
    }
  }

  // Scores before that scale: of the values i = c TOK + token, for 16 pages c
  // and a token, row g of the lanes ends with those of i = 4 k + g in v[k].
  struct Raw {
    float v[TOK];
  };
  const auto raw_of = [&](const Boxes& x) {
    float best[4 * TOK];
#pragma unroll
    for (int c = 0; c < 4; c++) {
#pragma unroll
      for (int i = 0; i < TOK; i++) best[c * TOK + i] = -INFINITY;
#pragma unroll
      for (int t = 0; t < NT; t++) {
        intx4 s = {0, 0, 0, 0};
#pragma unroll
        for (int m = 0; m < NM; m++) s = __builtin_amdgcn_mfma_i32_16x16x64_i8(z[t][m], x.w[c][m], s, 0, 0, 0);
#pragma unroll
        for (int j = 0; j < 4; j++) {
          float& y = best[c * TOK + j / HJ];
          y = fmaxf(y, __builtin_fmaf((float)s[j], up[t][j], off[t][j]));
        }
      }
    }
    Raw r;
#pragma unroll
    for (int k = 0; k < TOK; k++) {
      float* y = best + 4 * k;
      swap32(y[0], y[2]);
      swap32(y[1], y[3]);
      y[0] = fmaxf(y[0], y[2]);
      y[1] = fmaxf(y[1], y[3]);
      swap16(y[0], y[1]);
      r.v[k] = fmaxf(y[0], y[1]);
    }
    return r;
  };
  const auto pages_of = [&](int tok) { return ((span.pos + tok) >> b.pshift) + 1; };
  // a token's score of a page: inf where it is always taken, -inf where it never is
  const auto score = [&](float raw, float scale, int page, int n) {
    const float x = page < a.first || page >= n - a.recent ? INFINITY : raw * scale;
    return scale < 0.f || page >= n ? -INFINITY : x;
  };

  const int stride = (np + 63) & ~63;
  const bool near = PART || span.n * stride <= a.room;
  if (near) {
    // a wave's boxes are on their way while it works on those before
    for (int p = base + wave * 64; p < np; p += on) {
      Boxes then = now;
      if (p + on < np) then = load(id_of(p + on + lane));
      const Raw r = raw_of(now);
#pragma unroll
      for (int k = 0; k < TOK; k++) {
        const int i = 4 * k + g, at = i / TOK * 16 + col, tok = i % TOK;
        const float scale = __shfl(now.scale, at, 64);
        const float x = score(r.v[k], scale, p + at, pages_of(tok));
        if constexpr (PART) {
          if (p + at < np) a.scores[((size_t)span.row * b.NKV + h) * b.table_pages + p + at] = x;
        } else if (tok < span.n) {
          scores[tok * stride + p + at] = x;
        }
      }
      now = then;
    }
    if constexpr (PART) return;
    if constexpr (NW > 1) __syncthreads();
    else in_order();
  }

  const int ct = tid % CT, cw = wave % CW;
  for (int tok = wave / CW; tok < span.n; tok += CH) {
    const int n = pages_of(tok);
    const bool held = near && n <= kHeld;
    float mine[R];
    if (held) {
#pragma unroll
      for (int r = 0; r < R; r++) {
        mine[r] = -INFINITY;
        if (r * CT + cw * 64 < n) mine[r] = scores[tok * stride + r * CT + ct];
      }
    }
    // f(page, score) over the pages, in order, a thread a page (-inf behind the last)
    const auto each = [&](auto f) {
      if (held) {
#pragma unroll
        for (int r = 0; r < R; r++)
          if (r * CT < n) f(r * CT + ct, mine[r]);
      } else if (near) {
        for (int p = 0; p < n; p += CT)
          f(p + ct, p + cw * 64 < n ? scores[tok * stride + p + ct] : -INFINITY);
      } else {
        for (int p = 0; p < n; p += CT) {
          const Boxes x = load(id_of(p + ct));
          const Raw r = raw_of(x);
          const int i = g * TOK + tok;
          float y = 0.f;
#pragma unroll
          for (int k = 0; k < TOK; k++) {
            const float v = __shfl(r.v[k], (i & 3) * 16 + col, 64);
            y = k == i >> 2 ? v : y;
          }
          f(p + ct, score(y, x.scale, p + ct, n));
        }
      }
    };

    choose<CW>(choices[wave / CW], each, a.count, a.blocks + ((size_t)(span.row + tok) * b.NKV + h) * a.count);
  }
}

// The choice among scores that another launch left: a block a token and key/value
// head (4 of 2000 pages 10 us with the scores' launch, 5 of them this one's).
constexpr int kHeldFar = 16384;  // of them, those that registers hold; more are read in every pass
__global__ __launch_bounds__(512) void choose_kernel(SelectArgs a) {
  constexpr int CW = 8, CT = 64 * CW, R = kHeldFar / CT;
  __shared__ Choice<CW> c;
  const Kv8Batch& b = a.b;
  const int tid = threadIdx.x, h = blockIdx.x % b.NKV;
  const Kv8Span span = kv8_tile_span(b, 1, blockIdx.x / b.NKV);
  if (span.n == 0) return;
  const int n = (span.pos >> b.pshift) + 1;
  const size_t list = (size_t)span.row * b.NKV + h;
  const float* s = a.scores + list * b.table_pages;
  float mine[R];
#pragma unroll
  for (int r = 0; r < R; r++) {
    mine[r] = -INFINITY;
    if (r * CT < n && n <= kHeldFar) mine[r] = r * CT + tid < n ? s[r * CT + tid] : -INFINITY;
  }
  const auto each = [&](auto f) {
    if (n <= kHeldFar) {
#pragma unroll
      for (int r = 0; r < R; r++)
        if (r * CT < n) f(r * CT + tid, mine[r]);
    } else {
      for (int p = 0; p < n; p += CT) f(p + tid, p + tid < n ? s[p + tid] : -INFINITY);
    }
  };
  choose<CW>(c, each, a.count, a.blocks + list * a.count);
}

// of the workspace of a choice in parts
int64_t scores_bytes(const Kv8Batch& b) { return (int64_t)b.rows * b.NKV * b.table_pages * 4; }

bool aligned16(const void* p) { return ((uintptr_t)p & 15) == 0; }

int check_bounds(const char* op, const ane_kv8_bounds* x) {
  if (!x || !x->box || !x->unit || !aligned16(x->box))
    return op_fail(ANE_ERR_ARG, "storiesane %s: null bounds, or box not 16-byte aligned", op);
  return ANE_OK;
}

// How a batch's tokens are dealt to blocks: nt tiles of 16 query rows, tok tokens
// a block, its waves (which choose for a token together, or where it has several
// each for its own).
//
// Tokens of chunks share their context's boxes, 4 to a block (of up to 4 heads)
// or 2 (of up to 8), where there are more than 512 lists to make (800 of 3 heads
// and 250 pages 7.4 us, a token a block 8.7 to 15.5 by its waves; 2000 pages 27
// and 41; but 480 lists 26.6 and 25.2).  Otherwise a token has a block: of one
// wave up to 64 pages (256 lists of 60 pages 5.2 us, of four waves 5.6, of eight
// 6.1; 5600 13, 34 and 64), or 256 and 512 where there are more than 512 and 1024
// lists (800 of 120 pages 7.3 us, of four 8.7; 512 of 250 8.3 and 7.8; 1600 of 250
// 16.4 and 18.9); of four up to 512 pages (256 lists of 250 pages 6.4 us, eight
// 6.8); of eight beyond (900 pages 10.1 us, four 10.7; 2000 pages, 4 lists, 15.5
// and 17.9).
//
// Up to 128 lists of long contexts: the scores by two waves for every 128 pages,
// the choice behind a launch (4 lists of head dimension 64 and 1000 pages 9.0 us,
// in one launch 10.0; of 2000 10.1 and 15.5, 8000 16.4 and 44; of 750 9.1 and 9.0;
// head dimension 128, 8 of 500 9.5 and 9.8, 8000 18 and 73).  Of more than 32 they
// have to be twice as long (64 of 1500 11.7 and 13.9, of 1000 10.1 and 10.2; 128 of
// head dimension 128, 1500 18.5 and 21.0, of up to 750 13.4 and 12.4), and 256 gain
// nothing (of 2000 22.9 and 20.2).
struct Form {
  int nt, tok, waves;
  bool parts = false;
};
// pages of the longest context, as far as the host knows
int pages_of(const Kv8Batch& b, const ane_kv8_batch& batch) {
  const int cap = b.table_pages << b.pshift;
  return (((batch.max_len ? std::min(batch.max_len, cap) : cap) - 1) >> b.pshift) + 1;
}
Form form_of(const Kv8Batch& b, const ane_kv8_batch& batch, int dh, int G) {
  const int pages = pages_of(b, batch);
  const int most = batch.max_new ? batch.max_new : (batch.rows + batch.nseq - 1) / std::max(batch.nseq, 1);
  const int64_t lists = (int64_t)b.rows * b.NKV;
  const int nt = G <= 16 ? 1 : 2;
  if (most > 1 && lists > 512 && (G <= 4 || (G <= 8 && pages > 64))) return {nt, G <= 4 ? 4 : 2, 4};
  if (pages <= (lists > 1024 ? 512 : lists > 512 ? 256 : 64)) return {nt, 1, 1};
  if (lists <= 128 && (int64_t)pages * dh >= (lists <= 32 ? 65536 : 131072) && lists * b.table_pages <= 1 << 22)
    return {nt, 1, 2, true};
  return {nt, 1, pages <= 512 ? 4 : 8};
}

int check_sizes(const char* op, const Kv8Batch& b, const ane_kv8_batch& batch, int dh, int heads, int count) {
  if (heads < 1 || heads % b.NKV || heads / b.NKV > kKvMaxGroup)
    return op_fail(ANE_ERR_ARG, "storiesane %s: heads=%d must be 1..%d times kv_heads=%d", op, heads, kKvMaxGroup,
                   b.NKV);
  if (count < 1 || count > 65536) return op_fail(ANE_ERR_ARG, "storiesane %s: count=%d want 1..65536", op, count);
  const Form f = form_of(b, batch, dh, heads / b.NKV);
  if ((int64_t)kv8_count(b.nseq, b.rows, kv8_tiles(f.tok)) * b.NKV * 64 * f.waves > 0xffffffffll)  // threads
    return op_fail(ANE_ERR_ARG, "storiesane %s: rows=%d are too many for one launch", op, b.rows);
  return ANE_OK;
}

// scores that a block's LDS holds, of contexts as long as the host knows
int room_of(int tok, int pages) { return std::min(tok * ((pages + 63) & ~63), kFar); }

template <int DH, int NT>
void launch_parts(const SelectArgs& a, int pages, hipStream_t st) {
  const uint32_t lists = kv8_count(a.b.nseq, a.b.rows, kv8_tiles(1)) * a.b.NKV;
  // blocks for what the longest context may have, but no more than fill the card many times
  const uint32_t parts = std::min<uint32_t>((pages + 127) / 128, std::max(1u, 16384 / lists));
  hipLaunchKernelGGL((select_kernel<DH, NT, 1, 2, 1, true>), dim3(lists, parts), dim3(128), 0, st, a);
  hipLaunchKernelGGL(choose_kernel, dim3(lists), dim3(512), 0, st, a);
}

template <int DH, int NT, int TOK, int NW, int CW>
int launch_form(const char* op, SelectArgs a, int pages, hipStream_t st) {
  auto* const kernel = select_kernel<DH, NT, TOK, NW, CW, false>;
  a.room = room_of(TOK, pages);
  const int lds = a.room * 4;
  if (lds > 32768) {
    const hipError_t e = taken(hipFuncSetAttribute((const void*)kernel, hipFuncAttributeMaxDynamicSharedMemorySize, lds));
    if (e != hipSuccess) return op_fail(ANE_ERR_HIP, "storiesane %s: %s", op, hipGetErrorString(e));
  }
  const dim3 grid(kv8_count(a.b.nseq, a.b.rows, kv8_tiles(TOK)) * a.b.NKV);
  hipLaunchKernelGGL(kernel, grid, dim3(64 * NW), lds, st, a);
  return ANE_OK;
}

template <int DH, int NT>
int launch_token(const char* op, const SelectArgs& a, int pages, const Form& f, hipStream_t st) {
  if (f.waves == 1) return launch_form<DH, NT, 1, 1, 1>(op, a, pages, st);
  if (f.waves == 4) return launch_form<DH, NT, 1, 4, 4>(op, a, pages, st);
  return launch_form<DH, NT, 1, 8, 8>(op, a, pages, st);
}

template <int DH>
int launch(const char* op, const SelectArgs& a, const ane_kv8_batch& batch, hipStream_t st) {
  const int pages = pages_of(a.b, batch);
  const Form f = form_of(a.b, batch, DH, a.G);
  if (f.parts) {
    if (f.nt == 1) launch_parts<DH, 1>(a, pages, st);
    else launch_parts<DH, 2>(a, pages, st);
    return ANE_OK;
  }
  if (f.tok == 4) return launch_form<DH, 1, 4, 4, 1>(op, a, pages, st);
  if (f.tok == 2) return launch_form<DH, 1, 2, 4, 1>(op, a, pages, st);
  return f.nt == 1 ? launch_token<DH, 1>(op, a, pages, f, st) : launch_token<DH, 2>(op, a, pages, f, st);
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
  const dim3 grid(kv8_count(a.b.nseq, a.b.rows, kv8_pages(1 << a.b.pshift)), a.b.NKV);
  if (grid.x * 64ll > 0xffffffffll)  // threads
    return op_fail(ANE_ERR_ARG, "storiesane %s: rows=%d are too many for one launch", op, a.b.rows);
  DeviceScope dev(cache->device);
  if (dev.status() != hipSuccess)
    return op_fail(ANE_ERR_HIP, "storiesane %s: device %d: %s", op, cache->device, hipGetErrorString(dev.status()));
  a.k = (const uint8_t*)cache->k; a.k_exp = cache->k_exp; a.box = bounds->box; a.unit = bounds->unit;
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
  if (!rc) rc = check_sizes(op, b, *batch, cache->head_dim, heads, count);
  return rc ? rc : form_of(b, *batch, cache->head_dim, heads / b.NKV).parts ? scores_bytes(b) : 0;
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
  rc = check_sizes(op, a.b, *batch, cache->head_dim, g.heads, g.count);
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
  if (form_of(a.b, *batch, cache->head_dim, g.heads / a.b.NKV).parts &&
      (!g.ws || !aligned16(g.ws) || g.ws_bytes < scores_bytes(a.b)))
    return op_fail(ANE_ERR_ARG, "storiesane %s: workspace of %lld bytes, want %lld, 16-byte aligned", op,
                   (long long)(g.ws ? g.ws_bytes : 0), (long long)scores_bytes(a.b));
  DeviceScope dev(cache->device);
  if (dev.status() != hipSuccess)
    return op_fail(ANE_ERR_HIP, "storiesane %s: device %d: %s", op, cache->device, hipGetErrorString(dev.status()));
  a.q = (const half_t*)g.q; a.box = bounds->box; a.unit = bounds->unit; a.blocks = g.blocks;
  a.q_row = g.q_row; a.q_head = g.q_head;
  a.scores = (float*)g.ws;
  a.G = g.heads / a.b.NKV; a.count = g.count; a.first = g.first; a.recent = g.recent;
  rc = cache->head_dim == 64 ? launch<64>(op, a, *batch, (hipStream_t)stream)
                             : launch<128>(op, a, *batch, (hipStream_t)stream);
  if (rc) return rc;
  const hipError_t h = hipGetLastError();
  if (h != hipSuccess) return op_fail(ANE_ERR_HIP, "storiesane %s: %s", op, hipGetErrorString(h));
  return ANE_OK;
}

extern "C" int ane_debug_kv8_select_form(const ane_kv8_cache* cache, const ane_kv8_batch* batch, int32_t heads,
                                         int32_t* out) {
  const char* op = "debug kv8 select form";
  Kv8Batch b;
  int rc = kv8_check(op, cache, batch, &b);
  if (!rc) rc = check_sizes(op, b, *batch, cache->head_dim, heads, 1);
  if (rc) return rc;
  if (!out) return op_fail(ANE_ERR_ARG, "storiesane %s: null buffer", op);
  const Form f = form_of(b, *batch, cache->head_dim, heads / b.NKV);
  out[0] = f.nt;
  out[1] = f.tok;
  out[2] = f.waves;
  out[3] = f.parts;
  out[4] = f.parts ? 0 : room_of(f.tok, pages_of(b, *batch));
  return ANE_OK;
}
