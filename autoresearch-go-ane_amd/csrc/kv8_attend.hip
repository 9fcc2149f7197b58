// Attention over the paged 8-bit cache (ane_kv8_attend): prompts, chunks of
// prompts and single tokens.
//
// Mathematics: out = softmax(scale Q K^T) V per key/value head, in one pass
// over the keys with a running maximum and sum per row.  The rows of a tile
// are (token, query head of the group), so one reading of K and V serves the
// whole group.  Scores come transposed, S^T = K Q^T (MFMA 16x16x32, fp32
// sums): a lane then holds, for one row, keys 4 g + j of every 16, and that is
// what the second product's operand P^T takes, with V stored so that the same
// lane finds the same four keys of its dimensions side by side: neither P nor
// V moves between lanes or through LDS.  Codes become fp16 (exactly, page
// exponent applied) in the registers.
//
// A block is one tile and one key/value head (and one part of the keys where
// tiles are few); its waves take steps of 32 keys in turn and meet once
// at the end, in LDS.  There is no barrier in the loop.  A decoder's step has
// its append in the same launch (kv8_step).
//
// What bounds it.  Single tokens over long contexts: the cache's bytes (40
// sequences of up to 40,000 tokens, 2 heads of 128: 494 MB in 108 us, 4.6 TB/s,
// where a large copy has 5.1).  Single tokens over short contexts: the chain
// launch, offsets, page table, first loads, meeting (one sequence of 777 tokens
// 6.7 us, 64 of 1100 10.1, in a graph).  Prompts: the vector instructions around the
// products, about 150 for 32 keys and 48 rows where the products are 24 MFMAs,
// with the vector units 77 % busy (one of 8192 tokens, 12 heads of 64: 121 us,
// 850 TFLOP/s).
//
// Lists of pages (ane_kv8_attend_blocks) go the same ways, their keys numbered in
// the list's order.  Single tokens: the chain again, the list's loads before the
// page table's (in a captured graph, one row of 12 heads and 32 pages of 64 8.4
// us; 64 rows of 16 heads of 128 and 48 pages of 32 13.2 us, 47 MB).  Chunks: the
// vector instructions, so the tokens of a tile share what they name (5 chunks, 841
// rows of 12 heads, 24 pages of 64 each out of up to 190: 21.5 us, a tile a row
// 48).
#include <algorithm>
#include <type_traits>

#include "kv8_rows.h"
#include "op_error.h"

namespace ane {

namespace {

// Units of 16 keys in a wave's step.  Two: with four, single tokens are slower
// (64 of 1100 tokens 10.8 us, not 10.1) and larger tiles and head dimension 128
// do not fit (64 of 1500 81 us, not 34).
constexpr int NU = 2;
constexpr int kStep = 16 * NU;

struct AttendArgs {
  Kv8Batch b;
  const uint8_t *k, *v;
  const int8_t *k_exp, *v_exp;
  const half_t* q;
  half_t* out;
  int64_t q_row, q_head, out_row, out_head;
  int frag;     // out is the decoder's activation fragments (decode.h) instead
  int G;        // query heads per key/value head
  int tt;       // tokens per tile: tt * G <= rows of the tile
  int tiles;    // items
  int longest;  // tiles are numbered with the longest contexts first
  int nsplit;   // parts that the keys of a tile are cut into, at most
  int round;    // keys that a block takes at a time: parts are multiples of it
  float c;      // scale * log2(e)
  float* part;  // [tiles][NKV][nsplit][tt * G][DH]: a row's sums
  float2* ml;   // [tiles][NKV][nsplit][tt * G]: what they are relative to, and the sum of exponentials
};

// with the append of the rows' own keys and values, from a product's sums
struct StepArgs : AttendArgs {
  Kv8AppendArgs in;
};

// over the pages that are named for each row and key/value head (tt = 1)
struct ListArgs : AttendArgs {
  const int* blocks;  // [rows][NKV][count] places in the table
  int count;
};
// the same for tiles of several tokens, over the pages that any of them names
struct UnionArgs : ListArgs {
  int room;  // places that LDS has masks of
};
__device__ __forceinline__ const int* list_of(const ListArgs& a, int row, int h) {
  return a.blocks + ((size_t)row * a.b.NKV + h) * a.count;
}
// The list's keys, in its own order: those of its pages up to the last place
// that is one (at least a page, so that a row without any gets its zeros).
__device__ __forceinline__ int list_keys(const ListArgs& a, const int* list) {
  int c = (a.count - 1) & ~63;
  for (;; c -= 64) {
    const int at = c + (int)(threadIdx.x & 63);
    const uint64_t is = __ballot(at < a.count && (unsigned)list[min(at, a.count - 1)] < (unsigned)a.b.table_pages);
    if (is) return (c + 64 - __clzll((long long)is)) << a.b.pshift;
    if (c == 0) return 1 << a.b.pshift;
  }
}

// The pages that the tokens of a tile name: their places, and which tokens name
// each.  Rising places, each once; but where a token names one twice, or there
// are more places than LDS has masks of, all lists one behind the other.  The
// order does not depend on that of any atomics.
struct Named {
  int* place;      // [tt * count]
  uint16_t* mask;  // [tt * count]
};
extern __shared__ uint32_t union_lds[];  // masks of all places in halves of words, then the two above
__device__ __forceinline__ Named named_of(const UnionArgs& a) {
  int* place = reinterpret_cast<int*>(union_lds + (a.room + 1) / 2);
  return {place, reinterpret_cast<uint16_t*>(place + a.tt * a.count)};
}
template <int KW>
__device__ __forceinline__ int name_pages(const UnionArgs& a, const Kv8Span& span, int h, Named out) {
  __shared__ int twice, counts[KW];
  const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  // places behind the tile's last token have no key for it
  const int np = min(((span.pos + span.n - 1) >> a.b.pshift) + 1, a.b.table_pages), all = span.n * a.count;
  const auto place_of = [&](int e, int tok) {
    const int at = list_of(a, span.row + tok, h)[e - tok * a.count];
    return (unsigned)at < (unsigned)np ? at : -1;
  };
  bool apart = np > a.room;
  if (!apart) {
    for (int i = tid; i < (np + 1) / 2; i += 64 * KW) union_lds[i] = 0;
    if (tid == 0) twice = 0;
    __syncthreads();
    for (int e = tid; e < all; e += 64 * KW) {
      const int tok = e / a.count, at = place_of(e, tok);
      if (at >= 0) {
        const uint32_t bit = 1u << (tok + 16 * (at & 1));
        if (atomicOr(union_lds + (at >> 1), bit) & bit) twice = 1;
      }
    }
    __syncthreads();
    apart = twice;
  }
  if (apart) {
    for (int e = tid; e < all; e += 64 * KW) {
      const int tok = e / a.count;
      out.place[e] = place_of(e, tok);
      out.mask[e] = (uint16_t)(1 << tok);
    }
    __syncthreads();
    return all;
  }
  // a wave a run of places
  const int run = (np + 64 * KW - 1) / (64 * KW) * 64, p0 = wave * run, p1 = min(p0 + run, np);
  const auto mask_of = [&](int p) { return p < p1 ? union_lds[p >> 1] >> (16 * (p & 1)) & 0xffff : 0u; };
  int n = 0;
  for (int p = p0; p < p1; p += 64) n += __popcll(__ballot(mask_of(p + lane) != 0));
  if (lane == 0) counts[wave] = n;
  __syncthreads();
  int at = 0;
  n = 0;
#pragma unroll
  for (int w = 0; w < KW; w++) {
    at += w < wave ? counts[w] : 0;
    n += counts[w];
  }
  for (int p = p0; p < p1; p += 64) {
    const uint32_t mask = mask_of(p + lane);
    const uint64_t is = __ballot(mask != 0);
    if (mask) {
      const int i = at + __popcll(is & ((1ull << lane) - 1));
      out.place[i] = p + lane;
      out.mask[i] = (uint16_t)mask;
    }
    at += __popcll(is);
  }
  __syncthreads();
  return n;
}

// where dimension d of a row's query head goes
template <int DH>
__device__ __forceinline__ half_t* out_at(const AttendArgs& a, int row, int head, int d) {
  return a.out + (a.frag ? (int64_t)act_frag_off(row, head * DH + d) : row * a.out_row + head * a.out_head + d);
}

// the rows of a tile; the grid counts tiles down
__device__ __forceinline__ Kv8Span tile_span(const AttendArgs& a, int tile) {
  return a.longest ? kv8_tile_longest(a.b, a.tt, a.tiles - 1 - tile) : kv8_tile_span(a.b, a.tt, tile);
}

// The keys of a tile are cut into equal parts of whole rounds, at most nsplit.
__device__ __forceinline__ int part_keys(const AttendArgs& a, int keys) {
  const int n = (keys + a.nsplit - 1) / a.nsplit;
  return (n + a.round - 1) / a.round * a.round;
}

__device__ __forceinline__ float xor16_max(float x) {
  const auto r = __builtin_amdgcn_permlane16_swap(__float_as_uint(x), __float_as_uint(x), false, false);
  return fmaxf(__uint_as_float(r[0]), __uint_as_float(r[1]));
}
__device__ __forceinline__ float xor32_max(float x) {
  const auto r = __builtin_amdgcn_permlane32_swap(__float_as_uint(x), __float_as_uint(x), false, false);
  return fmaxf(__uint_as_float(r[0]), __uint_as_float(r[1]));
}
__device__ __forceinline__ half8 join(half2v a, half2v b, half2v c, half2v d) {
  half8 r;
  r[0] = a[0]; r[1] = a[1]; r[2] = b[0]; r[3] = b[1]; r[4] = c[0]; r[5] = c[1]; r[6] = d[0]; r[7] = d[1];
  return r;
}

// 0xff in every byte of w that is a NaN code
__device__ __forceinline__ uint32_t nan_bytes(uint32_t w) {
  return ((((w & 0x7f7f7f7fu) + 0x01010101u) & 0x80808080u) >> 7) * 0xffu;
}

// One step's K and V, NU units of 16 keys: raw codes, and of each unit's page
// the exponents (K in bits 0..7, V in 8..15) and whether it is there (bit 16).
// A page that is not there reads the pool's first, which exists but may hold
// anything; its scores are masked, its values cleared, and its exponents 0 (a
// scale made of a stray one, -128, is NaN and makes NaN of cleared values too).
// pos: of a list's pages, where the unit's tokens stand in the sequence; by:
// which of the tile's tokens name the page.
template <int DH>
struct Step {
  u32x4 k[NU][DH / 64], v[NU][DH / 64];
  int ex[NU], pos[NU], by[NU];
};
constexpr int kThere = 1 << 16;
__device__ __forceinline__ float k_scale(int ex) { return kv8_scale((int8_t)(ex & 0xff)); }
__device__ __forceinline__ float v_scale(int ex) { return kv8_scale((int8_t)(ex >> 8 & 0xff)); }

// Waves a SIMD is to hold: what the registers of a form leave.
constexpr int waves_per_simd(int DH, int NT) {
  return NT == 1 ? (DH == 64 ? 4 : 3) : DH == 64 ? (NT == 2 ? 4 : 3) : 2;
}

// NT: tiles of 16 rows; KW: waves that share a tile's keys; RW: tiles a block
// takes, each by a wave of its own (KW = 1: the waves have nothing to do with
// each other); ONE: a step's keys are of one page (pages of at least kStep
// tokens).  Args is StepArgs: the sequences have a token each, and the block
// first appends its key and value and rotates its queries.  ListArgs: the keys
// are those of a list of pages, numbered in its order.  UnionArgs: and each page
// is for some of the tile's tokens.
template <int DH, int NT, int KW, int RW, bool ONE, typename Args>
__global__ __launch_bounds__(64 * KW * RW, waves_per_simd(DH, NT)) void attend_kernel(Args a) {
  constexpr bool STEP = std::is_same_v<Args, StepArgs>;
  constexpr bool UNION = std::is_same_v<Args, UnionArgs>, LIST = UNION || std::is_same_v<Args, ListArgs>;
  static_assert(!STEP || (NT == 1 && KW == 4));
  static_assert(KW == 1 || RW == 1, "the waves of a block meet over one tile");
  constexpr int R = 16 * NT;    // rows of the tile
  constexpr int NM = DH / 32;   // MFMAs along the head dimension
  constexpr int ND = DH / 16;   // 16-dimension groups of the output
  // the waves meet over the output's dimensions in parts that leave LDS for
  // as many blocks as there are registers for
  constexpr int PASS = KW == 4 && R * DH > 2048 ? 2 : 1;
  constexpr int DP = DH / PASS;
  constexpr int LD = DP + 4;
  __shared__ __attribute__((aligned(16))) float lds_o[KW == 1 ? 1 : KW][KW == 1 ? 1 : R][LD];
  __shared__ float lds_m[KW][R], lds_l[KW][R];
  const Kv8Batch& b = a.b;
  const int tid = threadIdx.x, lane = tid & 63;
  const int wave = KW == 1 ? 0 : __builtin_amdgcn_readfirstlane(tid >> 6);
  const int col = lane & 15, g = lane >> 4;
  const int h = blockIdx.x % b.NKV;
  const int rest = blockIdx.x / b.NKV;
  const int sp = rest % a.nsplit;
  // the longest rows of a prompt first
  const int tile = a.tiles - 1 - rest / a.nsplit * RW - (RW > 1 ? __builtin_amdgcn_readfirstlane(tid >> 6) : 0);
  if (RW > 1 && tile < 0) return;
  const Kv8Span span = UNION || (NT > 1 && KW > 1) ? tile_span(a, tile) : kv8_tile_span(b, a.tt, tile);
  if (span.n == 0) return;
  const int rows = span.n * a.G;
  const int* list = nullptr;
  Named named = {};
  int npages = 0;
  int kend = span.pos + span.n;  // keys of the tile's last token
  if constexpr (UNION) {
    named = named_of(a);
    npages = name_pages<KW>(a, span, h, named);
    kend = max(npages, 1) << b.pshift;
  } else if constexpr (LIST) {
    list = list_of(a, span.row, h);
    kend = list_keys(a, list);
  }
  const int pk = part_keys(a, kend);
  const int k0 = sp * pk;
  if (k0 >= kend) return;
  const int k1 = min(kend, k0 + pk);

  constexpr int CPR = DH / 8;
  __shared__ half8 qs[STEP ? 16 * CPR : 1];  // the rotated queries
  if constexpr (STEP) {
    // one wave appends, three rotate; no other block touches the page and head,
    // and behind the barrier the block's waves see what was written
    __shared__ uint4 unit[DH];
    if (wave == 0) {
      if (!a.in.from.err || !*a.in.from.err) kv8_append_rows<DH, true>(a.in, span, h, unit);
    } else if (const int c = tid - 64; c < a.G * CPR) {
      const int d0 = c % CPR * 8;
      qs[c] = narrow8(rotate8(sums8(a.in.from, span.row, (h * a.G + c / CPR) * DH + d0),
                              turn_of<DH>(a.in.cos, a.in.sin, span.pos, d0)));
    }
    __syncthreads();
  }

  // 64 pages from wbase on, one per lane: where the head's rows begin, and
  // what Step says of the page.  wend: the first position behind them.
  const int* trow = b.table + (size_t)span.seq * b.table_stride;
  int wbase = 0, wexp = 0, wpos = 0, wby = 0;
  int wend = 0;
  uint32_t wlo = 0, whi = 0;
  auto window = [&](int pg) {
    wbase = pg;
    wend = (pg + 64) << b.pshift;  // a table covers at most 2^30 tokens
    const int p = pg + lane;
    int id = -1;
    if constexpr (LIST) {
      if (p << b.pshift < k1) {  // and so within the list
        int place;
        if constexpr (UNION) {
          place = npages ? named.place[p] : -1;
          wby = npages ? named.mask[p] : 0;
        } else {
          place = list[p];
        }
        if ((unsigned)place < (unsigned)b.table_pages) {
          id = trow[place];
          wpos = place << b.pshift;
        }
      }
      if ((unsigned)id >= (unsigned)b.pages) id = -1;
    } else if (p < b.table_pages && ((int64_t)p << b.pshift) < k1) {
      id = trow[p];
      if ((unsigned)id >= (unsigned)b.pages) id = -1;
    }
    const size_t e = (size_t)(id >= 0 ? id : 0) * b.NKV + h;
    const size_t at = e * ((size_t)DH << b.pshift);
    wlo = (uint32_t)at;
    whi = (uint32_t)(at >> 32);
    wexp = id >= 0 ? ((int)a.k_exp[e] & 0xff) | ((int)a.v_exp[e] & 0xff) << 8 | kThere : 0;
  };
  // The codes of the step at kb; `on` false: nothing is wanted of them (one
  // line is read).
  const uint32_t kl = col * DH + 16 * g, vl = lane * (DH / 4);
  auto fetch = [&](Step<DH>& s, int kb, bool on) {
    if (kb + kStep > wend) window(kb >> b.pshift);
    const uint32_t ko = on ? kl : 0, vo = on ? vl : 0;
    size_t at = 0;
#pragma unroll
    for (int u = 0; u < NU; u++) {
      const int ku = kb + 16 * u;
      if (u == 0 || !ONE) {
        const int w = (ku >> b.pshift) - wbase;
        at = (uint32_t)__builtin_amdgcn_readlane((int)wlo, w) |
             (size_t)(uint32_t)__builtin_amdgcn_readlane((int)whi, w) << 32;
        s.ex[u] = __builtin_amdgcn_readlane(wexp, w);
        at += (ku & ((1 << b.pshift) - 1)) * DH;
        if (LIST) s.pos[u] = __builtin_amdgcn_readlane(wpos, w) + (ku & ((1 << b.pshift) - 1));
        if (UNION) s.by[u] = __builtin_amdgcn_readlane(wby, w);
      } else {
        s.ex[u] = s.ex[0];
        at += 16 * DH;
        if (LIST) s.pos[u] = s.pos[0] + 16;
        if (UNION) s.by[u] = s.by[0];
      }
      const uint8_t *kp = a.k + at, *vp = a.v + at;
#pragma unroll
      for (int x = 0; x < DH / 64; x++) {
        s.k[u][x] = *reinterpret_cast<const u32x4*>(kp + ko + 64 * x);
        s.v[u][x] = *reinterpret_cast<const u32x4*>(vp + vo + 16 * x);
      }
    }
  };

  // Q: row r = 16 t + col, dimensions 64 (m / 2) + 16 g + 8 (m % 2) + j
  half8 q[NT][NM];
  int lim[NT];  // the last key of the lane's row
  int me[NT];   // its token's bit
#pragma unroll
  for (int t = 0; t < NT; t++) {
    const int r = min(16 * t + col, rows - 1);
    const int tok = r / a.G, hg = r - tok * a.G;
    lim[t] = span.pos + tok;
    me[t] = 1 << tok;
    const half_t* p = a.q + (span.row + tok) * a.q_row + (h * a.G + hg) * a.q_head + 16 * g;
#pragma unroll
    for (int m = 0; m < NM; m++)
      q[t][m] = STEP ? qs[r * CPR + 8 * (m >> 1) + 2 * g + (m & 1)] : ld_h8(p + 64 * (m >> 1) + 8 * (m & 1));
  }
  Step<DH> cur;
  int kb = k0 + wave * kStep;
  fetch(cur, kb, kb < k1);
  // waited for here, once (they were issued first), and not in every step
#pragma unroll
  for (int t = 0; t < NT; t++)
#pragma unroll
    for (int m = 0; m < NM; m++) asm volatile("" : "+v"(q[t][m]));

  // m: what the exponentials are relative to, the same in the four lanes of a
  // row: kBase below the row's largest score when it last moved.  It moves only
  // when a score passes it by kBase + kSlack, so that most steps neither join
  // the lanes' maxima nor touch the sums.  bar: how far a score may pass it;
  // -inf while the row has seen no key (m is then 0).
  // The weights are rounded to fp16 for the second product, the largest between
  // 2^kBase and 2^(kBase + kSlack), half of fp16's range: those down to 2^-21 of
  // it are normal numbers, off by at most 2^-11 of themselves (and divided by
  // the sum of the weights as rounded), smaller ones by 2^-32 of the largest, so
  // that a million keys behind one that takes most of the weight stay below the
  // output's own rounding.  A larger base would hold more of them, but moves
  // more often (prompt of 8192 tokens, base 7: 121 us, 8: 123, 9: 125, 11: 126).
  constexpr float kBase = 7.f, kSlack = 8.f;
  float m[NT], bar[NT];
  floatx4 o[ND][NT], l[NT];  // l: the sum of the row's weights, four times
#pragma unroll
  for (int t = 0; t < NT; t++) {
    m[t] = 0.f;
    bar[t] = -INFINITY;
    l[t] = floatx4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
    for (int d = 0; d < ND; d++) o[d][t] = floatx4{0.f, 0.f, 0.f, 0.f};
  }

  // where the unit's first token stands
  auto unit_pos = [&](const Step<DH>& s, int kb, int u) { return LIST ? s.pos[u] : kb + 16 * u; };
  // not 0: the step holds keys that some row does not attend to
  auto at_edge = [&](const Step<DH>& s, int kb) {
    int all = s.ex[0];
#pragma unroll
    for (int u = 1; u < (ONE ? 1 : NU); u++) all &= s.ex[u];
    int last = kb + kStep - 1;
    if (LIST) {
      last = s.pos[0] + 15;
#pragma unroll
      for (int u = 1; u < NU; u++) last = max(last, s.pos[u] + 15);
    }
    return max(last - span.pos, 0) | (~all & kThere);
  };

  half8 ones;
#pragma unroll
  for (int j = 0; j < 8; j++) ones[j] = (half_t)1.f;
  asm volatile("" : "+v"(ones));  // in vector registers: scalar ones are spilled and read back in every step
  uint32_t nan = 0;
  int careful = 0;
  auto step = [&](Step<DH>& s, int kb) {
    const int edge = at_edge(s, kb) | careful;
    floatx4 sc[NU][NT];
#pragma unroll
    for (int u = 0; u < NU; u++) {
      half8 kf[NM];
      const float ks = k_scale(s.ex[u]);
#pragma unroll
      for (int x = 0; x < NM; x++) {
        const uint32_t w0 = s.k[u][x >> 1][2 * (x & 1)], w1 = s.k[u][x >> 1][2 * (x & 1) + 1];
        kf[x] = join(kv8_up<false>(w0, ks), kv8_up<true>(w0, ks), kv8_up<false>(w1, ks), kv8_up<true>(w1, ks));
      }
#pragma unroll
      for (int t = 0; t < NT; t++) {
        floatx4 c = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int x = 0; x < NM; x++) c = __builtin_amdgcn_mfma_f32_16x16x32_f16(kf[x], q[t][x], c, 0, 0, 0);
        sc[u][t] = c;
      }
    }
    if (edge) {
#pragma unroll
      for (int u = 0; u < NU; u++)
#pragma unroll
        for (int t = 0; t < NT; t++)
#pragma unroll
          for (int j = 0; j < 4; j++)
            if (!(s.ex[u] & kThere) || unit_pos(s, kb, u) + 4 * g + j > lim[t]) sc[u][t][j] = -INFINITY;
    }
    if constexpr (UNION) {
#pragma unroll
      for (int u = 0; u < NU; u++)
#pragma unroll
        for (int t = 0; t < NT; t++) {
          const bool is = s.by[u] & me[t];
#pragma unroll
          for (int j = 0; j < 4; j++) sc[u][t][j] = is ? sc[u][t][j] : -INFINITY;
        }
    }
    float mx[NT];
    bool up = false;
#pragma unroll
    for (int t = 0; t < NT; t++) {
      mx[t] = -INFINITY;
#pragma unroll
      for (int u = 0; u < NU; u++)
#pragma unroll
        for (int j = 0; j < 4; j++) {
          sc[u][t][j] = __builtin_fmaf(sc[u][t][j], a.c, -m[t]);
          mx[t] = fmaxf(mx[t], sc[u][t][j]);
        }
      up |= mx[t] > bar[t];
    }
    if (__any(up)) {
#pragma unroll
      for (int t = 0; t < NT; t++) {
        const float top = xor32_max(xor16_max(mx[t]));
        if (top > bar[t]) {  // the same in the row's four lanes
          const float by = top - kBase;
          const float al = bar[t] == -INFINITY ? 0.f : __builtin_amdgcn_exp2f(-by);
          m[t] += by;
          bar[t] = kBase + kSlack;
#pragma unroll
          for (int u = 0; u < NU; u++)
#pragma unroll
            for (int j = 0; j < 4; j++) sc[u][t][j] -= by;
#pragma unroll
          for (int j = 0; j < 4; j++) l[t][j] *= al;
#pragma unroll
          for (int d = 0; d < ND; d++)
#pragma unroll
            for (int j = 0; j < 4; j++) o[d][t][j] *= al;
        }
      }
    }
    half8 pf[NU / 2][NT];
#pragma unroll
    for (int t = 0; t < NT; t++) {
#pragma unroll
      for (int u = 0; u < NU; u++)
#pragma unroll
        for (int j = 0; j < 4; j++) pf[u >> 1][t][4 * (u & 1) + j] = (half_t)__builtin_amdgcn_exp2f(sc[u][t][j]);
      // the weights' sums on the matrix cores, of the weights as rounded
#pragma unroll
      for (int y = 0; y < NU / 2; y++) l[t] = __builtin_amdgcn_mfma_f32_16x16x32_f16(ones, pf[y][t], l[t], 0, 0, 0);
    }
    // Values that no row of the tile attends to may be anything (rows not yet
    // written): cleared.  NaN among those that some row attends to and some
    // does not is taken out of the product, and put back behind the loop into
    // the rows that attend to it.
    if (edge) {
#pragma unroll
      for (int u = 0; u < NU; u++) {
        const int first = unit_pos(s, kb, u) + 4 * g;  // the lane's four keys
        const int n = s.ex[u] & kThere ? clampi((LIST ? span.pos + span.n : k1) - first, 0, 4) : 0;
        const uint32_t mine = n == 4 ? 0xffffffffu : (1u << (8 * n)) - 1;
#pragma unroll
        for (int x = 0; x < DH / 64; x++)
#pragma unroll
          for (int j = 0; j < 4; j++) {
            const uint32_t w = s.v[u][x][j] & mine, bad = nan_bytes(w);
            nan |= bad;
            s.v[u][x][j] = w & ~bad;
          }
      }
    }
#pragma unroll
    for (int y = 0; y < NU / 2; y++)
#pragma unroll
      for (int d = 0; d < ND; d++) {
        const float v0 = v_scale(s.ex[2 * y]), v1 = v_scale(s.ex[2 * y + 1]);
        const uint32_t w0 = s.v[2 * y][d >> 2][d & 3], w1 = s.v[2 * y + 1][d >> 2][d & 3];
        const half8 vf = join(kv8_up<false>(w0, v0), kv8_up<true>(w0, v0), kv8_up<false>(w1, v1), kv8_up<true>(w1, v1));
#pragma unroll
        for (int t = 0; t < NT; t++) o[d][t] = __builtin_amdgcn_mfma_f32_16x16x32_f16(vf, pf[y][t], o[d][t], 0, 0, 0);
      }
  };

  // One step on `now`, with the loads of the one behind it under way into
  // `then`; whether there is one.  Behind the last step they are of one line,
  // so that every path has the same loads outstanding and waits for no more
  // than it needs.
  auto turn = [&](Step<DH>& now, Step<DH>& then) {
    const int kn = kb + kStep * KW;
    fetch(then, kn < k1 ? kn : kb, kn < k1);
    step(now, kb);
    kb = kn;
    return kn < k1;
  };
  for (;;) {
    if (kb < k1) {
      Step<DH> nxt;
      while (turn(cur, nxt) && turn(nxt, cur)) {
      }
    }
    if constexpr (!UNION) break;
    // NaN among values that some row's page holds and another's does not: rare,
    // and all over again, with them taken out in every step
    if (careful) break;
    float sum = 0.f;
#pragma unroll
    for (int t = 0; t < NT; t++)
#pragma unroll
      for (int d = 0; d < ND; d++)
#pragma unroll
        for (int j = 0; j < 4; j++) sum = __builtin_fmaf(o[d][t][j], 0.f, sum);
    if (!__any(sum != sum)) break;
    careful = 1;
    nan = 0;
#pragma unroll
    for (int t = 0; t < NT; t++) {
      m[t] = 0.f;
      bar[t] = -INFINITY;
      l[t] = floatx4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
      for (int d = 0; d < ND; d++) o[d][t] = floatx4{0.f, 0.f, 0.f, 0.f};
    }
    wend = 0;
    kb = k0 + wave * kStep;
    fetch(cur, kb, kb < k1);
  }
  if (__any(nan != 0)) {
    // rare: how many NaN of each dimension a row attends to, as a product of
    // zeros and ones, over the steps that had them taken out
    wend = 0;
    for (kb = k0 + wave * kStep; kb < k1; kb += kStep * KW) {
      fetch(cur, kb, true);
      if (!at_edge(cur, kb) && !careful) continue;
#pragma unroll
      for (int y = 0; y < NU / 2; y++) {
        half8 sees[NT];
#pragma unroll
        for (int t = 0; t < NT; t++)
#pragma unroll
          for (int j = 0; j < 8; j++) {
            const int u = 2 * y + (j >> 2);
            sees[t][j] = (cur.ex[u] & kThere) && unit_pos(cur, kb, u) + 4 * g + (j & 3) <= lim[t] &&
                                 (!UNION || (cur.by[u] & me[t]))
                             ? (half_t)1.f
                             : (half_t)0.f;
          }
#pragma unroll
        for (int d = 0; d < ND; d++) {
          half8 isnan;
#pragma unroll
          for (int j = 0; j < 8; j++)
            isnan[j] = nan_bytes(cur.v[2 * y + (j >> 2)][d >> 2][d & 3]) >> (8 * (j & 3)) & 1 ? (half_t)1.f
                                                                                             : (half_t)0.f;
#pragma unroll
          for (int t = 0; t < NT; t++) {
            floatx4 n = {0.f, 0.f, 0.f, 0.f};
            n = __builtin_amdgcn_mfma_f32_16x16x32_f16(isnan, sees[t], n, 0, 0, 0);
#pragma unroll
            for (int j = 0; j < 4; j++)
              if (n[j] > 0.f) o[d][t][j] = NAN;
          }
        }
      }
    }
  }

  if constexpr (KW == 1) {  // the tile's only wave: lane (col, g) has 4 dimensions of 16 in row col
#pragma unroll
    for (int t = 0; t < NT; t++) {
      const int r = 16 * t + col;
      const float inv = l[t][0] == 0.f ? 0.f : 1.f / l[t][0];
      const int tok = r / a.G, hg = r - tok * a.G;
      if (r < rows) {
#pragma unroll
        for (int d = 0; d < ND; d++) {
          half4 z;
#pragma unroll
          for (int j = 0; j < 4; j++) z[j] = (half_t)(o[d][t][j] * inv);
          *reinterpret_cast<half4*>(out_at<DH>(a, span.row + tok, h * a.G + hg, 16 * d + 4 * g)) = z;
        }
      }
    }
    return;
  }
  // The waves meet: maximum over the waves, every wave's sums brought to it.
#pragma unroll
  for (int t = 0; t < NT; t++) {
    if (bar[t] == -INFINITY) m[t] = -INFINITY;  // no key
    if (g == 0) lds_m[wave][16 * t + col] = m[t];
  }
  __syncthreads();
#pragma unroll
  for (int t = 0; t < NT; t++) {
    const int r = 16 * t + col;
    float mm = lds_m[0][r];
#pragma unroll
    for (int w = 1; w < KW; w++) mm = fmaxf(mm, lds_m[w][r]);
    m[t] = __builtin_amdgcn_exp2f(m[t] - (mm == -INFINITY ? 0.f : mm));  // the wave's factor from here on
    if (g == 0) lds_l[wave][r] = l[t][0] * m[t];
  }
  const bool whole = pk >= kend;
  const size_t part = (((size_t)tile * b.NKV + h) * a.nsplit + sp) * ((size_t)a.tt * a.G);  // its first row
#pragma unroll
  for (int z = 0; z < PASS; z++) {
    if (z > 0) __syncthreads();
#pragma unroll
    for (int t = 0; t < NT; t++) {
      const int r = 16 * t + col;
      if (r < rows) {
#pragma unroll
        for (int d = 0; d < ND / PASS; d++)
          *reinterpret_cast<floatx4*>(&lds_o[wave][r][16 * d + 4 * g]) = o[z * (ND / PASS) + d][t] * m[t];
      }
    }
    __syncthreads();
    for (int c = tid; c < rows * (DP / 4); c += 64 * KW) {
      const int r = c / (DP / 4), d0 = c % (DP / 4) * 4, d = z * DP + d0;
      floatx4 x = *reinterpret_cast<const floatx4*>(&lds_o[0][r][d0]);
      float ls = lds_l[0][r];
#pragma unroll
      for (int w = 1; w < KW; w++) {
        x += *reinterpret_cast<const floatx4*>(&lds_o[w][r][d0]);
        ls += lds_l[w][r];
      }
      if (whole) {
        const float inv = ls == 0.f ? 0.f : 1.f / ls;
        const int tok = r / a.G, hg = r - tok * a.G;
        half4 y;
#pragma unroll
        for (int j = 0; j < 4; j++) y[j] = (half_t)(x[j] * inv);
        *reinterpret_cast<half4*>(out_at<DH>(a, span.row + tok, h * a.G + hg, d)) = y;
      } else {
        *reinterpret_cast<floatx4*>(a.part + (part + r) * DH + d) = x;
        if (d == 0) {
          float mm = lds_m[0][r];
#pragma unroll
          for (int w = 1; w < KW; w++) mm = fmaxf(mm, lds_m[w][r]);
          a.ml[part + r] = make_float2(mm, ls);
        }
      }
    }
  }
}

// Joins the parts of a tile's keys: a wave per row, lane s first taking part
// s's maximum and sum (at most kMaxSplit parts), then every lane DH / 64
// dimensions of all parts.
constexpr int kMaxSplit = 64;
template <int DH, typename Args>
__global__ __launch_bounds__(256) void join_kernel(Args a) {
  constexpr int W = DH / 64;
  const Kv8Batch& b = a.b;
  const int lane = threadIdx.x & 63;
  const int h = blockIdx.x % b.NKV, tile = blockIdx.x / b.NKV;
  const Kv8Span span = tile_span(a, tile);
  const int r = blockIdx.y * 4 + (threadIdx.x >> 6);
  if (r >= span.n * a.G) return;
  int kend = span.pos + span.n;
  if constexpr (std::is_same_v<Args, ListArgs>) kend = list_keys(a, list_of(a, span.row, h));
  const int pk = part_keys(a, kend);
  if (pk >= kend) return;  // one part: the output is written
  const int np = (kend + pk - 1) / pk;
  const size_t stride = (size_t)a.tt * a.G;  // rows of a part
  const size_t row = ((size_t)tile * b.NKV + h) * a.nsplit * stride + r;
  const float* part = a.part + row * DH;
  float m = -INFINITY, l = 0.f;
  if (lane < np) {
    const float2 p = a.ml[row + lane * stride];
    m = p.x;
    l = p.y;
  }
  const float mm = wave_max(m);
  const float al = __builtin_amdgcn_exp2f(m - (mm == -INFINITY ? 0.f : mm));
  l = wave_sum(l * al);
  float x[W] = {};
  constexpr int B = 8;  // parts whose loads are under way at once
  for (int s = 0; s < np; s += B) {
    float v[B][W];
#pragma unroll
    for (int u = 0; u < B; u++)
#pragma unroll
      for (int j = 0; j < W; j++) v[u][j] = part[min(s + u, np - 1) * stride * DH + lane + 64 * j];
#pragma unroll
    for (int u = 0; u < B; u++) {
      const float w = s + u < np ? __int_as_float(__builtin_amdgcn_readlane(__float_as_int(al), s + u)) : 0.f;
#pragma unroll
      for (int j = 0; j < W; j++)
        if (s + u < np) x[j] += v[u][j] * w;
    }
  }
  const float inv = l == 0.f ? 0.f : 1.f / l;
  const int tok = r / a.G, hg = r - tok * a.G;
#pragma unroll
  for (int j = 0; j < W; j++) *out_at<DH>(a, span.row + tok, h * a.G + hg, lane + 64 * j) = (half_t)(x[j] * inv);
}

struct Plan {
  int nt = 0, tt = 0, nsplit = 0, kw = 4, round = 0, longest = 0;
  uint32_t tiles = 0;
  int64_t bytes = 0;
  int room = 0;  // of UnionArgs
};

// count: pages of a row's list (0: the whole context)
int plan(const char* op, const Kv8Batch& b, const ane_kv8_batch& given, int DH, int heads, int count, Plan* p) {
  if (heads < 1 || heads % b.NKV || heads / b.NKV > kKvMaxGroup)
    return op_fail(ANE_ERR_ARG, "storiesane %s: heads=%d must be 1..%d times kv_heads=%d", op, heads, kKvMaxGroup,
                   b.NKV);
  const int G = heads / b.NKV;
  if (b.nseq == 0 || b.rows == 0) return ANE_OK;
  const int cap = b.table_pages << b.pshift;
  const int len = count ? count << b.pshift : given.max_len ? std::min(given.max_len, cap) : cap;
  // Tiles of 16 or 32 rows: the smallest that takes the longest sequence's rows
  // (the mean one's where that is not known), and at least a token's.  48 rows
  // use what a step converts a third better, in fewer and longer blocks: for
  // one sequence of 4096 keys or more (a prompt of 8192 tokens 123 us, in
  // tiles of 32 136; but one of 3000 29.5 and 27.9), and where they are 1536
  // blocks all the same (8 chunks of 2000 on 4,000 to 8,000 219 and 236; but
  // 20 of 50 to 150 on up to 9000 66 and 60, 32 of 10 to 128 on up to 4000 43
  // and 37); not where they would stay a fifth emptier, and not at head
  // dimension 128, whose registers end at 32 (two prompts of 2000 tokens 109
  // us, not 49).
  const int64_t most = (int64_t)G * (given.max_new ? std::min(given.max_new, b.rows) : (b.rows + b.nseq - 1) / b.nseq);
  p->nt = most <= 16 && G <= 16 ? 1 : 2;
  if (DH == 64 && most > 32 && 32 / G * 48 <= 48 / G * 38 &&
      ((b.nseq == 1 && len >= 4096) || (int64_t)kv8_count(b.nseq, b.rows, kv8_tiles(48 / G)) * b.NKV >= 1536))
    p->nt = 3;
  p->tt = 16 * p->nt / G;
  if (count) {  // a row is a tile
    p->nt = G <= 16 ? 1 : 2;
    p->tt = 1;
    // Chunks: tiles of several tokens (UnionArgs), which read and convert a page
    // once for all that name it.  They cost the joining of the lists, 3 us, and
    // blocks, so where there is enough to do (update, choice and attention, pages
    // named at random out of 125: 5 x 300 rows of 4 heads and 1536 keys 59 us, a
    // row a tile 100; 2 x 100 rows 22.9 and 27.2; 2 x 50 23.1 and 21.7; 4 x 200
    // of 256 keys 34 and 40, 4 x 50 24 and 20; head dimension 128, 4 x 100 of 2
    // heads 31 and 47, 4 x 30 30 and 24).  Of 5 to 8 heads, two or three tokens a
    // tile, from 1024 keys on (the attention of 5 x 200 rows of 8 heads and 1536 keys
    // 41 us, a row a tile 52; of head dimension 128 86 and 120; named out of 470
    // pages, which few tokens share, 2 x 100 rows 39 and 36; 31 x 38 rows of 640 keys
    // 42 and 39).
    const int pages = ((given.max_len ? std::min(given.max_len, cap) : cap) + (1 << b.pshift) - 1) >> b.pshift;
    const int most = given.max_new ? given.max_new : (b.rows + b.nseq - 1) / b.nseq;
    const int64_t lists = (int64_t)b.rows * b.NKV;
    if (G <= (len < 1024 ? 4 : 8) && most > 1 && pages <= 8192 && 16 / G * count <= 2048 && lists >= 640 &&
        lists * len * DH >= 48 << 20) {
      p->tt = 16 / G;
      p->room = pages;
    }
  }
  p->tiles = kv8_count(b.nseq, b.rows, kv8_tiles(p->tt));
  const int64_t blocks = (int64_t)p->tiles * b.NKV;
  // Waves that share a tile's keys: four, and in larger tiles each wave a tile
  // of its own, with nothing to meet over, where that leaves the GPU full long
  // enough to hide the longest (head dimension 64: 64 prompts of 256 23 us
  // against 41, 16 of 1024 42 against 50; but 4 of 512 11.9 against 9.8, one of
  // 2048 36 against 18; head dimension 128: 8 of 2048 206 against 248; but one
  // of 2048 46 against 37).
  const int wps = waves_per_simd(DH, p->nt);
  p->kw = p->nt > 1 && !count && 2 * blocks >= (int64_t)wps * len ? 1 : 4;
  // Lists of up to 2048 keys in up to 128 blocks: eight waves, and whole (with
  // update and choice of pages, 4 blocks of 1024 keys 17.5 us, with four waves
  // 18.1; of 2048 19.3, in parts 19.5; 64 blocks of 2048 20.3 and 21.4, 128 22.8
  // and 23.9; but 256 28.1 and 27.1, 4 of 4096 23.0 and 20.1, and at head
  // dimension 128 26.4 and 22.0).
  // Tiles of several tokens up to 320: eight (5 x 100 rows, 400 tiles 32.0 us,
  // with four 32.0; 3 x 100, 240 tiles 24.5 and 26.9; head dimension 128, 140
  // tiles 29.7 and 29.1).
  const bool eight = count && DH == 64 && p->nt == 1 && (p->room ? blocks <= 320 : blocks <= 128 && len <= 2048);
  if (eight) p->kw = 8;
  // Many short lists: a wave a tile, four to a block (1200 of 64 keys, 16 heads, 6.3
  // us, with four waves a tile 8.1; of 256 11.4 and 11.9, of 1024 29.8 and 28.4; 400
  // of 128 6.6 and 5.9; of 32 heads 1200 of 512 20.3 and 24.7).
  if (count && !p->room && blocks >= 768 && len <= 256 * p->nt) p->kw = 1;
  p->round = p->kw * kStep;
  // The longest contexts first, so that the last blocks to end are short ones:
  // chunks of prompts at the lengths they come in (8 of 100 to 400 on up to
  // 8000, three draws: 73, 101, 57 us against 100, 105, 60; 32 of 10 to 128 on
  // up to 4000 33 against 38).  Finding them costs each block 1.2 us at 64
  // sequences (64 of 16 to 100, head dimension 128: 138 against 129), so up to
  // 32, and not where a CU has no second block.  Tiles over lists likewise (update,
  // choice and attention, 5 chunks of 50 to 333 on up to 12,000 38.7 us, in the
  // batch's order 41.5; 6 on up to 30,000 54 and 56, of 10 to 200 44.0 and 43.9).
  p->longest = (count ? p->room > 0 : p->nt > 1 && p->kw == 4) && b.nseq > 1 && b.nseq <= 32 && blocks > 256;
  // Parts of the keys, where there are few blocks.  What parts cost is the
  // join's launch, 3 us, and their sums in fp32: for tiles of 32 and 48 rows a
  // block has to save more than it writes (1500 tokens of a prompt, 600 blocks:
  // whole 13 us, halves 28).  So those are cut up to a block a CU, in parts of
  // 512 keys at least (28 blocks of 2064 keys: whole 13.2 us, four parts 11.0;
  // of 664: 8.2, two 10.1), and further, as many as the CUs hold at once, only
  // into parts of 4096 (128 blocks of 16,500 keys: whole 87 us, halves 55,
  // four 45; 250 of 17,000 90, 78, 77).
  // Single tokens stay whole up to 1280 keys, 768 of head dimension 128 (4
  // blocks of 512 keys 5.3 us, in parts 7.3; of 1280 7.6 and 8.1; of 2048 9.7
  // and 7.6), and up to 32 for each block, 8192 at most, where there are 128
  // blocks (64 sequences of 4 heads and 4224 keys 25 us, in parts 30; of up to
  // 5000 21 and 23; 128 blocks of 10,000 36 and 23).  Beyond, up to 512 blocks,
  // in parts of 256 keys at least (4 blocks of 4096: 16 parts 8.0 us, 32 8.6)
  // and, ragged as they are, 2048 at most, so that one long context does not
  // outlast the rest (64 of 8 heads and up to 30,000 keys 206 us, whole 232;
  // 80 blocks of up to 40,000 108 us, of 4096 keys 113).
  int64_t ns = 1;
  if (eight || p->room) {
    ns = 1;
  } else if (p->nt == 1) {
    if (len > (blocks >= 128 ? std::min<int64_t>(32 * blocks, 8192) : DH == 64 ? 1280 : 768))
      ns = std::max<int64_t>(std::min<int64_t>((511 + blocks) / blocks, (len + 255) / 256), (len + 2047) / 2048);
  } else if (p->kw == 4) {
    ns = std::max<int64_t>(std::min<int64_t>(256 / blocks, len / 512),
                           std::min<int64_t>(256 * wps / blocks, len / 4096));
  }
  ns = std::min<int64_t>(ns, (len + p->round - 1) / p->round);
  ns = std::max<int64_t>(1, std::min<int64_t>(ns, kMaxSplit));
  p->nsplit = (int)ns;
  if (blocks * ns * 64 * p->kw > 0xffffffffll)  // threads (kw 1: a wave a tile)
    return op_fail(ANE_ERR_ARG, "storiesane %s: rows=%d nseq=%d are too many for one launch", op, b.rows, b.nseq);
  p->bytes = ns > 1 ? blocks * ns * p->tt * G * (DH + 2) * 4 : 0;
  return ANE_OK;
}

bool aligned16(const void* p) { return ((uintptr_t)p & 15) == 0; }

int check_count(const char* op, int count) {
  if (count < 1 || count > 65536) return op_fail(ANE_ERR_ARG, "storiesane %s: count=%d want 1..65536", op, count);
  return ANE_OK;
}

template <int DH, int NT, int KW, int RW, typename Args>
void launch_form(const Args& a, hipStream_t st, int lds = 0) {
  const dim3 grid(((uint32_t)a.tiles + RW - 1) / RW * a.b.NKV * a.nsplit), block(64 * KW * RW);
  if (kStep <= 1 << a.b.pshift)
    hipLaunchKernelGGL((attend_kernel<DH, NT, KW, RW, true, Args>), grid, block, lds, st, a);
  else
    hipLaunchKernelGGL((attend_kernel<DH, NT, KW, RW, false, Args>), grid, block, lds, st, a);
}

template <int DH>
void launch(const AttendArgs& a, const Plan& p, hipStream_t st) {
  if (p.nt == 1) launch_form<DH, 1, 4, 1>(a, st);
  else if (p.nt == 2 && p.kw == 4) launch_form<DH, 2, 4, 1>(a, st);
  else if (p.nt == 2) launch_form<DH, 2, 1, 4>(a, st);
  else if constexpr (DH == 64) {
    if (p.kw == 4) launch_form<DH, 3, 4, 1>(a, st);
    else launch_form<DH, 3, 1, 4>(a, st);
  }
  if (a.nsplit > 1)
    hipLaunchKernelGGL((join_kernel<DH, AttendArgs>), dim3((uint32_t)a.tiles * a.b.NKV, (a.tt * a.G + 3) / 4),
                       dim3(256), 0, st, a);
}

template <int DH>
void launch_list(const UnionArgs& a, const Plan& p, hipStream_t st) {
  const int lds = (a.room + 1) / 2 * 4 + a.tt * a.count * 6;
  if constexpr (DH == 64) {  // which alone has eight waves
    if (p.kw == 8 && p.room) return launch_form<DH, 1, 8, 1>(a, st, lds);
    if (p.kw == 8) launch_form<DH, 1, 8, 1, ListArgs>(a, st);
  }
  if (p.room) return launch_form<DH, 1, 4, 1>(a, st, lds);
  if (p.kw == 1 && p.nt == 1) launch_form<DH, 1, 1, 4, ListArgs>(a, st);
  else if (p.kw == 1) launch_form<DH, 2, 1, 4, ListArgs>(a, st);
  if (p.kw == 4 && p.nt == 1) launch_form<DH, 1, 4, 1, ListArgs>(a, st);
  else if (p.kw == 4) launch_form<DH, 2, 4, 1, ListArgs>(a, st);
  if (a.nsplit > 1)
    hipLaunchKernelGGL((join_kernel<DH, ListArgs>), dim3((uint32_t)a.tiles * a.b.NKV, (a.G + 3) / 4), dim3(256), 0, st,
                       a);
}

}  // namespace

}  // namespace ane

using namespace ane;

extern "C" int64_t ane_kv8_attend_workspace(const ane_kv8_cache* cache, const ane_kv8_batch* batch, int32_t heads) {
  const char* op = "kv8 attend workspace";
  Kv8Batch b;
  int rc = kv8_check(op, cache, batch, &b);
  if (rc) return rc;
  Plan p;
  rc = plan(op, b, *batch, cache->head_dim, heads, 0, &p);
  return rc ? rc : p.bytes;
}

extern "C" int64_t ane_kv8_attend_blocks_workspace(const ane_kv8_cache* cache, const ane_kv8_batch* batch,
                                                   int32_t heads, int32_t count) {
  const char* op = "kv8 attend workspace";
  Kv8Batch b;
  int rc = kv8_check(op, cache, batch, &b);
  if (!rc) rc = check_count(op, count);
  if (rc) return rc;
  Plan p;
  rc = plan(op, b, *batch, cache->head_dim, heads, count, &p);
  return rc ? rc : p.bytes;
}

extern "C" int ane_kv8_attend(const ane_kv8_cache* cache, const ane_kv8_batch* batch, const ane_kv8_attend_args* args,
                              void* stream) {
  return kv8_attend(cache, batch, args, false, stream);
}

namespace {

struct List {
  const int* blocks = nullptr;
  int count = 0;
};

// in: the append that the launch takes with it, where the plan lets it; list:
// the pages that the rows attend to, if not all
int attend(const ane_kv8_cache* cache, const ane_kv8_batch* batch, const ane_kv8_attend_args* args, bool frag,
           const Kv8AppendArgs* in, const List* list, void* stream) {
  const char* op = "kv8 attend";
  StepArgs step;
  AttendArgs& a = step;
  int rc = kv8_check(op, cache, batch, &a.b);
  if (!rc && list) rc = check_count(op, list->count);
  if (rc) return rc;
  if (!args) return op_fail(ANE_ERR_ARG, "storiesane %s: null arguments", op);
  if (a.b.nseq == 0 || a.b.rows == 0) return ANE_OK;  // an empty tensor may have no address
  if (!args->q || !args->out || (list && !list->blocks))
    return op_fail(ANE_ERR_ARG, "storiesane %s: null buffer", op);
  const ane_kv8_attend_args& g = *args;
  for (const int64_t s : {g.q_row, g.q_head, g.out_row, g.out_head})
    if (s < 0 || s % 8)
      return op_fail(ANE_ERR_ARG, "storiesane %s: stride %lld must be a multiple of 8", op, (long long)s);
  if (!aligned16(g.q) || !aligned16(g.out) || !aligned16(g.ws))
    return op_fail(ANE_ERR_ARG, "storiesane %s: buffers must be 16-byte aligned", op);
  const float c = g.scale * 1.44269504088896340736f;  // log2(e)
  if (!(g.scale > 0.f) || !std::isfinite(c))
    return op_fail(ANE_ERR_ARG, "storiesane %s: scale=%g must be positive and finite, times log2(e) too", op,
                   (double)g.scale);
  Plan p;
  rc = plan(op, a.b, *batch, cache->head_dim, g.heads, list ? list->count : 0, &p);
  if (rc) return rc;
  if (frag && a.b.rows > kDecRows)
    return op_fail(ANE_ERR_ARG, "storiesane %s: rows=%d of fragments, want at most %d", op, a.b.rows, kDecRows);
  if (!frag && !kv8_apart(a.b.rows, g.out_row, g.heads, g.out_head, cache->head_dim))
    return op_fail(ANE_ERR_ARG, "storiesane %s: rows of out overlap", op);
  const bool same = (const void*)g.q == g.out && g.q_row == g.out_row && g.q_head == g.out_head;
  if (!frag && !same && share_memory(fp16_rows(g.q, a.b.rows, g.q_row, g.heads, g.q_head, cache->head_dim),
                                     fp16_rows(g.out, a.b.rows, g.out_row, g.heads, g.out_head, cache->head_dim)))
    return op_fail(ANE_ERR_ARG, "storiesane %s: out overlaps q with other strides, or in part", op);
  if (list) {
    const Buffer buffers[] = {{"blocks", flat(list->blocks, (int64_t)a.b.rows * a.b.NKV * list->count * 4), false},
                              {"out", fp16_rows(g.out, a.b.rows, g.out_row, g.heads, g.out_head, cache->head_dim), true}};
    rc = check_apart(op, buffers, 2);
    if (rc) return rc;
  }
  if (p.bytes > 0 && (!g.ws || g.ws_bytes < p.bytes))
    return op_fail(ANE_ERR_ARG, "storiesane %s: workspace of %lld bytes, want %lld", op,
                   (long long)(g.ws ? g.ws_bytes : 0), (long long)p.bytes);
  DeviceScope dev(cache->device);
  if (dev.status() != hipSuccess)
    return op_fail(ANE_ERR_HIP, "storiesane %s: device %d: %s", op, cache->device, hipGetErrorString(dev.status()));
  a.k = (const uint8_t*)cache->k; a.v = (const uint8_t*)cache->v; a.k_exp = cache->k_exp; a.v_exp = cache->v_exp;
  a.q = (const half_t*)g.q; a.out = (half_t*)g.out;
  a.q_row = g.q_row; a.q_head = g.q_head; a.out_row = g.out_row; a.out_head = g.out_head;
  a.G = g.heads / a.b.NKV; a.tt = p.tt; a.tiles = (int)p.tiles; a.nsplit = p.nsplit; a.round = p.round;
  a.longest = p.longest;
  a.c = c;
  a.part = (float*)g.ws;
  a.ml = (float2*)(a.part + (size_t)p.tiles * a.b.NKV * p.nsplit * p.tt * a.G * cache->head_dim);
  a.frag = frag;
  if (in) {
    step.in = *in;
    launch_form<64, 1, 4, 1>(step, (hipStream_t)stream);
  } else if (list) {
    UnionArgs l;
    static_cast<AttendArgs&>(l) = a;
    l.blocks = list->blocks;
    l.count = list->count;
    l.room = p.room;
    if (cache->head_dim == 64) launch_list<64>(l, p, (hipStream_t)stream);
    else launch_list<128>(l, p, (hipStream_t)stream);
  } else if (cache->head_dim == 64) launch<64>(a, p, (hipStream_t)stream);
  else launch<128>(a, p, (hipStream_t)stream);
  const hipError_t h = hipGetLastError();
  if (h != hipSuccess) return op_fail(ANE_ERR_HIP, "storiesane %s: %s", op, hipGetErrorString(h));
  return ANE_OK;
}

}  // namespace

int ane::kv8_attend(const ane_kv8_cache* cache, const ane_kv8_batch* batch, const ane_kv8_attend_args* args, bool frag,
                    void* stream) {
  return attend(cache, batch, args, frag, nullptr, nullptr, stream);
}

extern "C" int ane_kv8_attend_blocks(const ane_kv8_cache* cache, const ane_kv8_batch* batch,
                                     const ane_kv8_attend_args* args, const int32_t* blocks, int32_t count,
                                     void* stream) {
  const List list = {blocks, count};
  return attend(cache, batch, args, false, nullptr, &list, stream);
}

int ane::kv8_step(const ane_kv8_cache* cache, const ane_kv8_batch* batch, const ane_kv8_append_args* append,
                  const Kv8Sums* from, const ane_kv8_attend_args* args, bool frag, void* stream) {
  Kv8AppendArgs in;
  int rc = kv8_append_check("kv8 append", cache, batch, append, from, &in);
  if (rc || in.b.nseq == 0 || in.b.rows == 0) return rc;
  Plan p;
  rc = plan("kv8 attend", in.b, *batch, cache->head_dim, append->heads, 0, &p);
  if (rc) return rc;
  // The decoder's step of 64 sequences and 1024 tokens, 12 layers: 0.504 ms in
  // one launch a layer, 0.534 in two; of 3 sequences 0.330 and 0.346.
  const bool one = from && batch->max_new == 1 && in.b.rows <= in.b.nseq && p.nt == 1 && p.nsplit == 1;
  if (one) return attend(cache, batch, args, frag, &in, nullptr, stream);
  rc = kv8_append(cache, batch, append, from, stream);
  return rc ? rc : attend(cache, batch, args, frag, nullptr, nullptr, stream);
}

extern "C" int ane_debug_kv8_attend_form(const ane_kv8_cache* cache, const ane_kv8_batch* batch, int32_t heads,
                                         int32_t count, int32_t* out) {
  const char* op = "debug kv8 attend form";
  Kv8Batch b;
  int rc = kv8_check(op, cache, batch, &b);
  if (!rc && count) rc = check_count(op, count);
  Plan p;
  if (!rc) rc = plan(op, b, *batch, cache->head_dim, heads, count, &p);
  if (rc) return rc;
  if (!out) return op_fail(ANE_ERR_ARG, "storiesane %s: null buffer", op);
  out[0] = p.nt;
  out[1] = p.tt;
  out[2] = p.kw;
  out[3] = p.nsplit;
  out[4] = p.longest;
  out[5] = p.room;
  return ANE_OK;
}
