// Beam search's step (ane_beam_select): the best continuations of a request's
// beams over beams and vocabulary, and the reordering of the beams' states;
// formulas in include/ane_serve.h.
//
// Two launches.  The first reads the logits once: a wave takes kSeg entries at
// a time and leaves each such segment's largest value, and the sum of the
// exponentials of all it took.  The second, a block per request, turns a
// segment's largest value into the key of the best candidate in it; of a
// request's W best candidates, every one lies in one of the W segments whose
// best are best (the best of W better segments are W better candidates), so
// that only W segments are read again and no launch sorts or keeps more.
//
// Keys are 64-bit sums of 32-bit logits and scores and of log sums.  In a log sum
// the exponentials, a lane's sums of up to 16 of them and the factors between
// parts are fp32, the sums of lanes and parts and the logarithm 64-bit (a 64-bit
// exponential takes a series where an fp32 one takes an instruction, and the
// first launch has one for every logit).  With half steps, 2^-24: 1 for x - max and 2 for the
// scaling by log2(e), each of the exponent, 2 for each of the two powers of two,
// 15 for the lane's sums; together at most (19 + 3 sum_v p_v (max - x_v)) 2^-24,
// p = softmax(x), which is 2e-6 for logits of normal distribution.  Measured:
// 5e-8, at most 1.2e-7 (256 rows of 60011, fp32 or fp16), 3.3e-7 (rows of 1000
// fp16).  The order of two beams' candidates is in doubt only where their keys
// differ by less, and of one beam's where 64 bits make them equal; equal ones go
// to the lower beam, then the lower token.
//
// What bounds it.  Much to read: the first launch, HBM (640 rows of 60011 fp16
// logits, 77 MB, in 18.6 us, 4.1 TB/s; 512 rows of 32000 fp32, 66 MB, in 13.2, 5.0
// TB/s) and then the second one's chain of accesses and barriers, 15.9 us for 16
// beams (of them 4 for histories of 2564 ids), 9.5 for 8.  Little: the two
// launches' chains (4 rows of 32000 fp32 logits 3.2 and 6.2 us, 64 rows 4.0 and
// 7.6).
#include <algorithm>

#include "kv8.h"
#include "op_error.h"
#include "wave_ops.h"

namespace ane {

namespace {

constexpr int kSeg = 256;       // entries of a segment
constexpr int kMaxBeams = 32;   // of a request
constexpr int kPer = 8;         // items a thread of the second launch holds
constexpr int kMaxParts = 128;  // of a row
constexpr int kWords = 1024;    // of 8 ids: the histories of a request that the second launch reads ahead
constexpr int kMoved = 8;       // words a thread of it moves
// It has 32 threads a beam, or more: enough for the segments of a beam, and for
// one segment.
static_assert(65536 / kSeg <= 32 * kPer && kSeg <= 32 * kPer, "");
// Ids of a history: places in it, and those that the last words and stretches
// reach to behind its end, are 32-bit numbers.
constexpr int kMaxHistory = 1 << 30;

// a wave's part of a row's log sum
struct Part {
  double sum;  // of exp(x - max)
  float max;
  int pad;
};

// where a row's history comes from (-1: nowhere), how long that is, and the
// token behind it (-1: none)
struct Move {
  int from, len, token;
};

struct BeamArgs {
  const void* logits;
  const float *scores, *weights;
  const uint8_t* finished;
  int *tokens, *parents;
  float* scores_out;
  uint8_t* finished_out;
  uint16_t* history;
  int* lengths;
  int64_t logits_row, history_row;
  int beams, vocab, eos, history_max;
  int segs, parts;     // of a row
  int words, stretch;  // of 8 ids: of a history; of one that a block moves at a time
  uint32_t words_magic, segs_magic;
  Move* moves;         // [rows], where histories have a launch of their own
  float* seg_max;   // [rows][segs]
  Part* part;       // [rows][parts]
};

typedef uint16_t ushort8u __attribute__((ext_vector_type(8), aligned(2)));

// ids c .. c + 7 of a history of n > c (behind the last: anything)
__device__ __forceinline__ ushort8u get_ids(const uint16_t* h, int c, int n) {
  if (c + 8 <= n) return *reinterpret_cast<const ushort8u*>(h + c);
  ushort8u v;
#pragma unroll
  for (int j = 0; j < 8; j++) v[j] = h[min(c + j, n - 1)];
  return v;
}
__device__ __forceinline__ void put_ids(uint16_t* h, int c, int n, ushort8u v) {
  if (c + 8 <= n) {
    *reinterpret_cast<ushort8u*>(h + c) = v;
  } else {
#pragma unroll
    for (int j = 0; j < 8; j++)
      if (c + j < n) h[c + j] = v[j];
  }
}
// t / n for t below 2^16; magic = ceil(2^32 / n)
__device__ __forceinline__ int quotient(int t, int n, uint32_t magic) { return n == 1 ? t : (int)__umulhi(t, magic); }

// a beam that has continuations: alive, and not finished
__device__ __forceinline__ bool proposes(const BeamArgs& a, int r) {
  return !(a.finished && a.finished[r]) && a.scores[r] > -INFINITY && (!a.weights || a.weights[r] > 0.f);
}

// A wave takes U loads of 64 N entries of a row, all under way at once: waves that
// take several such turns, the next one's loads under way, are no faster (33.3 to
// 39.0 us a step for 640 rows of 60011, one turn 32.0).  A lane whose N reach past the
// row's end takes the row's last N instead, and of those its own; rows of fewer
// than N are read one by one.
template <typename T, int U>
__global__ __launch_bounds__(256) void part_kernel(BeamArgs a) {
  constexpr int N = 16 / sizeof(T), LS = kSeg / N, SPW = 64 / LS;  // lanes of a segment, segments of a load
  typedef T Words __attribute__((ext_vector_type(N), aligned(sizeof(T))));
  const int lane = threadIdx.x & 63, r = blockIdx.y;
  const int p = blockIdx.x * 4 + __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  if (p >= a.parts) return;
  if (!proposes(a, r)) return;
  const T* row = static_cast<const T*>(a.logits) + r * a.logits_row;
  const int c0 = p * (U * 64 * N) + lane * N;
  Words w[U];
#pragma unroll
  for (int u = 0; u < U; u++) {
    const int c = min(c0 + u * 64 * N, a.vocab - N);
    if (a.vocab >= N) {
      w[u] = *reinterpret_cast<const Words*>(row + c);
    } else {
#pragma unroll
      for (int j = 0; j < N; j++) w[u][j] = row[min(j, a.vocab - 1)];
    }
  }
  Words none;  // -inf; the larger of it and NaN is it
#pragma unroll
  for (int j = 0; j < N; j++) none[j] = (T)-INFINITY;
#pragma unroll
  for (int u = 0; u < U; u++) w[u] = __builtin_elementwise_max(w[u], none);
  if ((p + 1) * (U * 64 * N) > a.vocab) {  // the row's last wave
#pragma unroll
    for (int u = 0; u < U; u++) {
      const int c = c0 + u * 64 * N, at = a.vocab >= N ? min(c, a.vocab - N) : 0;
#pragma unroll
      for (int j = 0; j < N; j++) w[u][j] = at + j >= c && at + j < a.vocab ? w[u][j] : (T)-INFINITY;
    }
  }
  float top[U];
  float m = -INFINITY;
#pragma unroll
  for (int u = 0; u < U; u++) {
    Words t = w[u];
#pragma unroll
    for (int n = N / 2; n > 0; n /= 2)  // of pairs while there are any
#pragma unroll
      for (int j = 0; j < n; j++) t[j] = __builtin_elementwise_max(t[j], t[j + n]);
    top[u] = over_lanes<32>((float)t[0], Max());
    const float both = fmaxf(top[u], xor32_f(top[u]));
    if (SPW == 1) top[u] = both;
    m = fmaxf(m, both);
  }
  // 2^((x - m) log2 e).  Of fp16 logits in one multiply-add, x log2 e less m
  // log2 e as rounded; the sum makes up for that rounding, d (below 0.003 for any
  // fp16 m), to its third power.  An infinite m makes NaN: a row without
  // candidates.
  constexpr float kLog2e = 1.44269504088896340736f;
  float s = 0.f;
  double more = 1.0;
  if (m > -INFINITY) {
    const float ml = m * kLog2e;
    if (sizeof(T) == 2) {
      const double d = (double)__builtin_fmaf(m, kLog2e, -ml) * 0.69314718055994531;
      more = 1.0 - d * (1.0 - 0.5 * d);
    }
#pragma unroll
    for (int u = 0; u < U; u++)
#pragma unroll
      for (int j = 0; j < N; j++) {
        const float x = (float)w[u][j];
        s += __builtin_amdgcn_exp2f(sizeof(T) == 2 ? __builtin_fmaf(x, kLog2e, -ml) : (x - m) * kLog2e);
      }
  }
  const double sum = sum_over_lanes((double)s) * more;
  float* seg = a.seg_max + (size_t)r * a.segs;
#pragma unroll
  for (int u = 0; u < U; u++) {
    const int k = (p * U + u) * SPW + lane / LS;
    if (lane % LS == 0 && k < a.segs) seg[k] = top[u];
  }
  if (lane == 0) a.part[(size_t)r * a.parts + p] = {sum, m, 0};
}

// An item that is chosen among: the larger key first, then the lower index.
// No two have the same index; those that are nothing have kNone and their place.
constexpr int kNone = 1 << 30;
struct Item {
  double key;
  int at;
  float x;  // the logit behind it
};
__device__ __forceinline__ bool before(double ak, int aa, double bk, int ba) {
  return (ak > bk) | ((ak == bk) & (aa < ba));
}

template <int TH>
struct Pick {
  static constexpr int kBeams = TH / 32, kGroups = TH / 16;
  static constexpr int kMost = kBeams * 16 * kPer;
  double key[kMost];  // those that may be among the best
  int at[kMost];
  float x[kMost];
  double gkey[kGroups];
  int gat[kGroups];
  int count[2];  // of the first pick and of the second
  double bar_key;
  int bar_at;
};

template <int N>
__device__ __forceinline__ void row_best(double& key, int& at) {
  const double k = row_ror<N>(key);
  const int i = row_ror<N>(at);
  const bool b = before(k, i, key, at);
  key = b ? k : key;
  at = b ? i : at;
}

// The `want` best of the block's items (`per` a thread, keys above -inf count),
// best(rank, item) called for each by one thread.
//
// The want-th best of the best items of groups of 16 threads is a bar that at
// least `want` items reach and few others do; ranks are counted among those, a
// wave an item, its lanes the others.  Where the groups were uneven and more
// than a wave's lanes reach the bar, they are dealt out again, one to each group
// in turn: at most the items of `want` groups, half of them, reach the next bar.
// BAR: a key that at least `want` items reach, if there are as many, is known, and
// `count` is 0; it does in place of the first bar where those that reach it have
// room.
template <int TH, bool BAR, typename F>
__device__ __forceinline__ void pick(Item (&x)[kPer], int per, int want, Pick<TH>& p, int& count, double known, F best) {
  constexpr int GR = Pick<TH>::kGroups;
  static_assert(2 * Pick<TH>::kBeams <= GR, "");
  const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  for (bool first = BAR;; first = false) {
    double key = known;
    int at = 0x7fffffff;  // behind every index
    if (!first) {
      key = x[0].key;
      at = x[0].at;
#pragma unroll
      for (int j = 1; j < kPer; j++) {
        if (j >= per) break;
        const bool b = before(x[j].key, x[j].at, key, at);
        key = b ? x[j].key : key;
        at = b ? x[j].at : at;
      }
      row_best<8>(key, at);
      row_best<4>(key, at);
      row_best<2>(key, at);
      row_best<1>(key, at);
      if ((tid & 15) == 0) {
        p.gkey[tid >> 4] = key;
        p.gat[tid >> 4] = at;
      }
      if (tid == 0) count = 0;
      __syncthreads();
      key = p.gkey[lane % GR];
      at = p.gat[lane % GR];
#pragma unroll
      for (int j = 0; j < 4; j++) {  // the groups have different items: one of them has this rank
        const int b = wave * 4 + j;
        const double bk = p.gkey[b];
        const int ba = p.gat[b];
        if (__popcll(__ballot(lane < GR && before(key, at, bk, ba))) == want - 1 && lane == 0) {
          p.bar_key = bk;
          p.bar_at = ba;
        }
      }
      __syncthreads();
      key = p.bar_key;
      at = p.bar_at;
    }
#pragma unroll
    for (int j = 0; j < kPer; j++) {
      if (j >= per) break;
      if ((x[j].key > -INFINITY) & !before(key, at, x[j].key, x[j].at)) {
        const int k = atomicAdd(&count, 1);
        if (first && k >= Pick<TH>::kMost) continue;
        p.key[k] = x[j].key;
        p.at[k] = x[j].at;
        p.x[k] = x[j].x;
      }
    }
    __syncthreads();
    const int n = count;
    if (n <= 64) {
      key = p.key[min(lane, n)];
      at = p.at[min(lane, n)];
      for (int b = wave; b < n; b += TH / 64) {
        const double bk = p.key[b];
        const int ba = p.at[b];
        const int rank = __popcll(__ballot(lane < n && before(key, at, bk, ba)));
        if (rank < want && lane == 0) best(rank, Item{bk, ba, p.x[b]});
      }
      break;
    }
    if (n <= Pick<TH>::kMost) {
      per = (n + TH - 1) / TH;
#pragma unroll
      for (int j = 0; j < kPer; j++) {
        if (j >= per) break;
        const int k = j * TH + (tid & 15) * GR + (tid >> 4);
        x[j] = {-INFINITY, kNone + k, 0.f};
        if (k < n) x[j] = {p.key[k], p.at[k], p.x[k]};
      }
    }
    __syncthreads();
  }
  __syncthreads();
}

// The natural logarithm of a positive number, to 1e-11: of m 2^e with m about 1,
// 2 atanh((m - 1) / (m + 1)) as its series.  The library's, to the last bit,
// takes three times the instructions, in all 16 waves.
__device__ __forceinline__ double log_of(double x) {
  int e = __builtin_amdgcn_frexp_exp(x);
  double m = __builtin_amdgcn_frexp_mant(x);  // 0.5 .. 1
  if (m < 0.70710678118654752) {
    m *= 2.0;
    e -= 1;
  }
  const double s = (m - 1.0) / (m + 1.0), q = s * s;  // q < 0.0295, whose 7th power over 15 is 1e-12
  double y = 1.0 / 13;
  y = __builtin_fma(y, q, 1.0 / 11);
  y = __builtin_fma(y, q, 1.0 / 9);
  y = __builtin_fma(y, q, 1.0 / 7);
  y = __builtin_fma(y, q, 1.0 / 5);
  y = __builtin_fma(y, q, 1.0 / 3);
  y = __builtin_fma(y, q, 1.0);
  return __builtin_fma((double)e, 0.69314718055994531, 2.0 * s * y);
}

// A block per request.  What bounds it is the chain of its memory accesses:
// everything that does not depend on a choice is on its way first.  Of 5.5 us for
// 4 beams of 32000 (16 of 60011: 13.3) the loads take 1.2 (1.3), log sums 0.8
// (1.9), segments' keys 0.2 (0.6), their choice 1.2 (2.0), candidates 0.7 (2.2),
// their choice 0.7 (1.5), outputs and histories 0.7 (3.8).
template <typename T, int TH>
__global__ __launch_bounds__(TH) void choose_kernel(BeamArgs a) {
  constexpr int NW = TH / 64, MB = Pick<TH>::kBeams;
  constexpr int BW = MB / NW, PL = kMaxParts / 64, HQ = kWords / TH;  // beams of a wave, parts and words of a lane
  __shared__ Pick<TH> pick_;
  __shared__ double bar;  // the key of the last of the best segments
  // a beam's s(v) = score + (x - lse); one that is finished has lse 0 and the
  // candidate x = 0, and one that proposes nothing has no number
  __shared__ double score[MB], lse[MB], weight[MB], score_of[MB];
  __shared__ int ended[MB], length[MB];
  __shared__ int seg_of[MB], parent[MB], token[MB];  // seg_of: beam << 16 | segment, -1: none
  __shared__ ushort8u hist[kWords];
  const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6), W = a.beams;
  const int row0 = blockIdx.x * W;
  const T* logits = static_cast<const T*>(a.logits);

  // segments: one a thread, dealt to the groups in turn, or 64 of a beam a wave's at
  // a time
  const int runs = (a.segs + 63) >> 6, dealt = (tid & 15) * Pick<TH>::kGroups + (tid >> 4);
  const bool few = W * a.segs <= TH;
  int per = few ? 1 : (W * runs + NW - 1) / NW;
  Item x[kPer];
#pragma unroll
  for (int j = 0; j < kPer; j++) {
    x[j] = {-INFINITY, kNone + j * TH + tid, -INFINITY};
    if (j >= per) continue;
    const int u = j * NW + wave, w = few ? quotient(dealt, a.segs, a.segs_magic) : u / runs;
    const int seg = few ? dealt - w * a.segs : (u - w * runs) * 64 + lane;
    x[j].x = a.seg_max[(size_t)(row0 + min(w, W - 1)) * a.segs + min(seg, a.segs - 1)];
    if (w < W && seg < a.segs) x[j].at = w << 16 | seg;
  }
  Part q[BW][PL];
  float sc[BW], wt[BW];
  int done[BW], len[BW];
#pragma unroll
  for (int i = 0; i < BW; i++) {
    const int w = min(wave + i * NW, W - 1), r = row0 + w;
    sc[i] = a.scores[r];
    wt[i] = a.weights ? a.weights[r] : 1.f;
    done[i] = a.finished ? a.finished[r] : 0;
    len[i] = a.lengths ? a.lengths[r] : 0;
#pragma unroll
    for (int k = 0; k < PL; k++) {
      q[i][k] = a.part[(size_t)r * a.parts + min(lane + 64 * k, a.parts - 1)];
      if (lane + 64 * k >= a.parts) q[i][k] = {0.0, -INFINITY, 0};
    }
  }
  ushort8u ids[HQ];
  const int words = a.lengths && !a.moves ? W * a.words : 0;
#pragma unroll
  for (int k = 0; k < HQ; k++) {
    const int t = k * TH + tid;
    if (t < words && words <= kWords) {
      const int w = quotient(t, a.words, a.words_magic);
      ids[k] = get_ids(a.history + (row0 + w) * a.history_row, (t - w * a.words) * 8, a.history_max);
    }
  }
  double sum = 0.0, top = 0.0;
#pragma unroll
  for (int i = 0; i < BW; i++) {
    float m = q[i][0].max;
#pragma unroll
    for (int k = 1; k < PL; k++) m = fmaxf(m, q[i][k].max);
    m = over_lanes<64>(m, Max());
    // Factors of the parts in fp32: off by what a part's own exponentials are.
    // An infinite maximum makes NaN, as it should.
    double s = 0.0;
#pragma unroll
    for (int k = 0; k < PL; k++) {
      const float f = __builtin_amdgcn_exp2f((q[i][k].max - m) * 1.44269504088896340736f);
      s += q[i][k].max > -INFINITY ? q[i][k].sum * f : 0.0;
    }
    s = sum_over_lanes(s);
    sum = lane == i ? s : sum;
    top = lane == i ? (double)m : top;
  }
  const double l = top + log_of(sum);
#pragma unroll
  for (int i = 0; i < BW; i++) {
    const int w = wave + i * NW;
    if (lane == i && w < W) {
      const bool live = sc[i] > -INFINITY && wt[i] > 0.f;
      score[w] = sc[i];
      weight[w] = wt[i];
      lse[w] = !live ? (double)NAN : done[i] ? 0.0 : l;
      ended[w] = done[i];
      length[w] = clampi(len[i], 0, a.history_max);
      seg_of[w] = -1;
      parent[w] = -1;
      token[w] = ANE_NO_TOKEN;
      score_of[w] = -INFINITY;
    }
  }
#pragma unroll
  for (int k = 0; k < HQ; k++)
    if (k * TH + tid < words && words <= kWords) hist[k * TH + tid] = ids[k];
  __syncthreads();
  const auto key_of = [&](int w, float x) {
    const double k = weight[w] * (score[w] + ((double)x - lse[w]));
    return k == k ? k : (double)-INFINITY;
  };

  // the best W segments
#pragma unroll
  for (int j = 0; j < kPer; j++) {
    if (j >= per) break;
    const int w = x[j].at < kNone ? x[j].at >> 16 : 0;
    if (ended[w]) x[j].x = (x[j].at & 0xffff) == 0 ? 0.f : -INFINITY;
    if (x[j].at < kNone) x[j].key = key_of(w, x[j].x);
  }
  if (tid == 0) {
    bar = -INFINITY;
    pick_.count[1] = 0;
  }
  pick<TH, false>(x, per, W, pick_, pick_.count[0], 0.0, [&](int rank, const Item& t) {
    seg_of[rank] = t.at;
    if (rank == W - 1) bar = t.key;
  });

  // the best W candidates in them, 64 of a segment a wave's at a time; an index
  // is the beam and the token
  per = (W * (kSeg / 64) + NW - 1) / NW;
  T y[kPer];
#pragma unroll
  for (int j = 0; j < kPer; j++) {  // all on their way
    x[j] = {-INFINITY, kNone + j * TH + tid, 0.f};
    if (j >= per) continue;
    const int u = j * NW + wave, k = u / (kSeg / 64), seg = __builtin_amdgcn_readfirstlane(seg_of[min(k, W - 1)]);
    const int w = max(seg, 0) >> 16, i = u % (kSeg / 64) * 64 + lane, v = (seg & 0xffff) * kSeg + i;
    y[j] = logits[(row0 + w) * a.logits_row + min(v, a.vocab - 1)];
    if (seg >= 0 && k < W) {
      if (ended[w]) x[j].at = i == 0 ? w << 16 | a.eos : x[j].at;
      else if (v < a.vocab) x[j].at = w << 16 | v;
    }
  }
#pragma unroll
  for (int j = 0; j < kPer; j++) {
    if (j >= per) break;
    if (x[j].at < kNone) {
      const int w = x[j].at >> 16;
      x[j].x = ended[w] ? 0.f : (float)y[j];
      x[j].key = key_of(w, x[j].x);
    }
  }
  pick<TH, true>(x, per, W, pick_, pick_.count[1], bar, [&](int rank, const Item& t) {
    const int w = t.at >> 16;
    parent[rank] = w;
    token[rank] = t.at & 0xffff;
    score_of[rank] = score[w] + ((double)t.x - lse[w]);
  });

  if (tid < W) {
    const int r = row0 + tid, w = parent[tid];
    a.tokens[r] = token[tid];
    a.parents[r] = w < 0 ? -1 : row0 + w;
    a.scores_out[r] = (float)score_of[tid];
    if (a.finished_out) a.finished_out[r] = w >= 0 && (ended[w] || token[tid] == a.eos);
  }
  if (!a.lengths) return;
  if (a.moves) {  // in a launch of their own
    if (tid < W) {
      const int r = row0 + tid, w = parent[tid], len = w < 0 ? 0 : length[w];
      const bool grows = w >= 0 && !ended[w] && len < a.history_max;
      a.moves[r] = {w < 0 ? -1 : row0 + w, len, grows ? token[tid] : -1};
      a.lengths[r] = len + grows;
    }
    return;
  }
  if (words > kWords) {
    // the ones that move: all are read before any is written
    ushort8u v[kMoved];
#pragma unroll
    for (int k = 0; k < kMoved; k++) {
      const int t = k * TH + tid, w = quotient(min(t, words - 1), a.words, a.words_magic), c = (t - w * a.words) * 8;
      const int from = parent[w];
      if (t < words && from >= 0 && from != w && c < length[from])
        v[k] = get_ids(a.history + (row0 + from) * a.history_row, c, length[from]);
    }
    __syncthreads();
#pragma unroll
    for (int k = 0; k < kMoved; k++) {
      const int t = k * TH + tid, w = quotient(min(t, words - 1), a.words, a.words_magic), c = (t - w * a.words) * 8;
      const int from = parent[w];
      if (t < words && from >= 0 && from != w) put_ids(a.history + (row0 + w) * a.history_row, c, length[from], v[k]);
    }
  }
  // the ones that are in LDS
#pragma unroll 1
  for (int t = tid; t < words && words <= kWords; t += TH) {
    const int w = quotient(t, a.words, a.words_magic), c = t - w * a.words, from = parent[w];
    if (from >= 0 && from != w) put_ids(a.history + (row0 + w) * a.history_row, c * 8, length[from], hist[from * a.words + c]);
  }
  if (tid < W) {
    const int r = row0 + tid, w = parent[tid];
    int len = w < 0 ? 0 : length[w];
    if (w >= 0 && !ended[w] && len < a.history_max) a.history[r * a.history_row + len++] = (uint16_t)token[tid];
    a.lengths[r] = len;
  }
}

// The histories, where they are long: a block takes a stretch of columns of a
// request's rows, all of which it reads before it writes any.
__global__ __launch_bounds__(256) void move_kernel(BeamArgs a) {
  __shared__ Move move[kMaxBeams];
  const int tid = threadIdx.x, W = a.beams, row0 = blockIdx.y * W, c0 = blockIdx.x * a.stretch;
  constexpr int Q = kWords / 256;
  if (tid < W) move[tid] = a.moves[row0 + tid];
  __syncthreads();
  ushort8u v[Q];
  int c[Q], to[Q];
#pragma unroll
  for (int q = 0; q < Q; q++) {
    const int t = q * 256 + tid, w = t / a.stretch;
    c[q] = (c0 + t - w * a.stretch) * 8;
    to[q] = -1;
    if (w < W && move[w].from >= 0 && move[w].from != row0 + w && c[q] < move[w].len) {
      to[q] = w;
      v[q] = get_ids(a.history + move[w].from * a.history_row, c[q], move[w].len);
    }
  }
  __syncthreads();
#pragma unroll
  for (int q = 0; q < Q; q++)
    if (to[q] >= 0) put_ids(a.history + (row0 + to[q]) * a.history_row, c[q], move[to[q]].len, v[q]);
  if (tid < W && move[tid].token >= 0 && move[tid].len / 8 >= c0 && move[tid].len / 8 < c0 + a.stretch)
    a.history[(row0 + tid) * a.history_row + move[tid].len] = (uint16_t)move[tid].token;
}

// Loads of a wave in the first launch.  Of fp32 logits four, where that leaves
// enough waves (512 rows of 32000: 20.3 us a step, with two 21.2; 272 rows 15.7
// and 15.9, 256 15.7 and 15.6, 64 10.9 and 10.8; 4100 rows of 2049 24.5 and 26.4);
// of fp16, which take as many instructions for half the bytes, two (640 rows of
// 60011: 33.1 us, with four 33.8; 512 of 32000 18.4 and 18.8).
int loads_of(int64_t rows, int vocab, bool half) { return !half && rows * (vocab / 512) >= 16384 ? 4 : 2; }

struct Plan {
  int loads, segs, parts;
  int64_t seg_bytes, move_bytes, bytes;
};
int plan(const char* op, int requests, int beams, int vocab, bool half, Plan* p) {
  if (requests < 0 || beams < 1 || beams > kMaxBeams || vocab < 1 || vocab > 65535 || (int64_t)requests * beams > 65535)
    return op_fail(ANE_ERR_ARG,
                   "storiesane %s: requests=%d beams=%d vocab=%d, want beams 1..%d, vocab 1..65535, at most 65535 rows",
                   op, requests, beams, vocab, kMaxBeams);
  const int64_t rows = (int64_t)requests * beams;
  p->loads = loads_of(rows, vocab, half);
  const int width = p->loads * 64 * (half ? 8 : 4);
  p->segs = (vocab + kSeg - 1) / kSeg;
  p->parts = (vocab + width - 1) / width;
  p->seg_bytes = (rows * p->segs * 4 + 15) / 16 * 16;
  p->move_bytes = (rows * (int64_t)sizeof(Move) + 15) / 16 * 16;
  p->bytes = p->seg_bytes + p->move_bytes + rows * p->parts * (int64_t)sizeof(Part);
  return ANE_OK;
}

uint32_t magic(int n) { return (uint32_t)(((1ull << 32) + n - 1) / n); }

// 512 threads for up to 8 beams, 1024 for more (4 beams of 32000, 16 requests, 10.9
// us a step, with 256 threads 12.3, with 1024 11.3; one request 9.0, 10.1 and 10.1;
// 2 of 2000, 64 requests, 9.5, 9.7 and 10.6; 8 of 60011, 8 requests, 15.3, 19.1 and
// 14.6; 8 of 32000, one request, 11.1, 13.7 and 11.0; 9 of 32000 12.6 with 512 and
// with 1024, 12 of 32000, 16 requests, 16.6 and 15.6, 16 of 60011, 40 requests, 38.1
// and 33.1).
int threads_of(int beams) { return beams <= 8 ? 512 : 1024; }
// Histories of up to 8 words a thread move in the second launch (40 requests of
// 16 beams and 2564 ids: 32.9 us a step, in a launch of their own 35.4; 16 of 4 and
// 4064 ids 11.9 and 13.6).
bool moves_apart(int beams, int words) { return (int64_t)beams * words > kMoved * threads_of(beams); }

template <typename T>
void launch_choose(const BeamArgs& a, int requests, hipStream_t st) {
  if (threads_of(a.beams) == 512) hipLaunchKernelGGL((choose_kernel<T, 512>), dim3(requests), dim3(512), 0, st, a);
  else hipLaunchKernelGGL((choose_kernel<T, 1024>), dim3(requests), dim3(1024), 0, st, a);
}

}  // namespace

}  // namespace ane

using namespace ane;

extern "C" int64_t ane_beam_select_workspace(int32_t requests, int32_t beams, int32_t vocab, int32_t half) {
  Plan p;
  const int rc = plan("beam select workspace", requests, beams, vocab, half != 0, &p);
  return rc ? rc : p.bytes;
}

extern "C" int ane_beam_select(const ane_beam_args* args, void* stream) {
  const char* op = "beam select";
  if (!args) return op_fail(ANE_ERR_ARG, "storiesane %s: null arguments", op);
  const ane_beam_args& g = *args;
  Plan p;
  int rc = plan(op, g.requests, g.beams, g.vocab, g.half != 0, &p);
  if (rc) return rc;
  if (g.requests == 0) return ANE_OK;  // an empty tensor may have no address
  if (!g.logits || !g.scores || !g.tokens || !g.parents || !g.scores_out)
    return op_fail(ANE_ERR_ARG, "storiesane %s: null buffer", op);
  if (!g.finished != !g.finished_out || (g.finished ? g.eos < 0 || g.eos >= g.vocab : g.eos != -1))
    return op_fail(ANE_ERR_ARG, "storiesane %s: finished, finished_out and eos=%d (of vocab=%d; -1: none) go together",
                   op, g.eos, g.vocab);
  if ((g.history && !g.lengths) || g.history_max < 0 || (g.history ? g.history_row < g.history_max : g.history_max > 0))
    return op_fail(ANE_ERR_ARG, "storiesane %s: history without lengths, or not of history_max=%d within its stride %lld",
                   op, g.history_max, (long long)g.history_row);
  if (g.history_max > kMaxHistory)
    return op_fail(ANE_ERR_ARG, "storiesane %s: history_max=%d want at most %d", op, g.history_max, kMaxHistory);
  if (g.logits_row < g.vocab)
    return op_fail(ANE_ERR_ARG, "storiesane %s: logits_row=%lld is shorter than vocab=%d", op, (long long)g.logits_row,
                   g.vocab);
  if (!g.ws || ((uintptr_t)g.ws & 15) || g.ws_bytes < p.bytes)
    return op_fail(ANE_ERR_ARG, "storiesane %s: workspace of %lld bytes, want %lld, 16-byte aligned", op,
                   (long long)(g.ws ? g.ws_bytes : 0), (long long)p.bytes);
  const int64_t rows = (int64_t)g.requests * g.beams;
  const int64_t size = g.half ? 2 : 4;
  const Buffer buffers[] = {{"logits", row_major(g.logits, rows, g.logits_row * size, g.vocab * size), false},
                            {"scores", flat(g.scores, rows * 4), false, 1},
                            {"weights", flat(g.weights, rows * 4), false},
                            {"finished", flat(g.finished, rows), false, 2},
                            {"tokens", flat(g.tokens, rows * 4), true},
                            {"parents", flat(g.parents, rows * 4), true},
                            {"scores_out", flat(g.scores_out, rows * 4), true, 1},
                            {"finished_out", flat(g.finished_out, rows), true, 2},
                            {"history", row_major(g.history, rows, g.history_row * 2, g.history_max * 2ll), true},
                            {"lengths", flat(g.lengths, rows * 4), true}};
  rc = check_apart(op, buffers, sizeof buffers / sizeof *buffers);
  if (rc) return rc;
  DeviceScope dev(g.device);
  if (dev.status() != hipSuccess)
    return op_fail(ANE_ERR_HIP, "storiesane %s: device %d: %s", op, g.device, hipGetErrorString(dev.status()));
  BeamArgs a;
  a.logits = g.logits; a.scores = g.scores; a.weights = g.weights; a.finished = g.finished;
  a.tokens = g.tokens; a.parents = g.parents; a.scores_out = g.scores_out; a.finished_out = g.finished_out;
  a.history = g.history; a.lengths = g.lengths; a.logits_row = g.logits_row; a.history_row = g.history_row;
  a.beams = g.beams; a.vocab = g.vocab; a.eos = g.eos; a.history_max = g.history_max;
  a.segs = p.segs; a.parts = p.parts;
  a.seg_max = (float*)g.ws;
  a.words = (g.history_max + 7) / 8;
  a.words_magic = a.words ? magic(a.words) : 0;
  a.segs_magic = magic(a.segs);
  a.stretch = kWords / g.beams;
  a.moves = moves_apart(g.beams, a.words) ? (Move*)((char*)g.ws + p.seg_bytes) : nullptr;
  a.part = (Part*)((char*)g.ws + p.seg_bytes + p.move_bytes);
  const hipStream_t st = (hipStream_t)stream;
  const dim3 grid((p.parts + 3) / 4, (uint32_t)rows);
  if (g.half) {
    hipLaunchKernelGGL((part_kernel<half_t, 2>), grid, dim3(256), 0, st, a);
    launch_choose<half_t>(a, g.requests, st);
  } else {
    if (p.loads == 4) hipLaunchKernelGGL((part_kernel<float, 4>), grid, dim3(256), 0, st, a);
    else hipLaunchKernelGGL((part_kernel<float, 2>), grid, dim3(256), 0, st, a);
    launch_choose<float>(a, g.requests, st);
  }
  if (a.moves)
    hipLaunchKernelGGL(move_kernel, dim3((a.words + a.stretch - 1) / a.stretch, g.requests), dim3(256), 0, st, a);
  const hipError_t h = hipGetLastError();
  if (h != hipSuccess) return op_fail(ANE_ERR_HIP, "storiesane %s: %s", op, hipGetErrorString(h));
  return ANE_OK;
}

extern "C" int ane_debug_beam_form(int32_t requests, int32_t beams, int32_t vocab, int32_t half, int32_t history_max,
                                   int32_t* out) {
  const char* op = "debug beam form";
  Plan p;
  const int rc = plan(op, requests, beams, vocab, half != 0, &p);
  if (rc) return rc;
  if (!out || history_max < 0 || history_max > kMaxHistory)
    return op_fail(ANE_ERR_ARG, "storiesane %s: null buffer, or history_max=%d", op, history_max);
  out[0] = p.loads;
  out[1] = threads_of(beams);
  out[2] = moves_apart(beams, (history_max + 7) / 8);
  return ANE_OK;
}
