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
// Keys are 64-bit sums of 32-bit logits and scores and of log sums whose
// exponentials are fp32 and whose additions are 64-bit: two candidates' order
// is in doubt only where they differ by 1e-8 or so; equal ones go to the lower
// beam, then the lower token.
#include <algorithm>

#include "kv8.h"
#include "op_error.h"

namespace ane {

namespace {

constexpr int kSeg = 256;       // entries of a segment
constexpr int kMaxBeams = 32;   // of a request
constexpr int kTh = 1024;       // threads of the second launch
constexpr int kPer = 8;         // items a thread of it holds
static_assert(kMaxBeams * (65536 / kSeg) <= kTh * kPer && kMaxBeams * kSeg <= kTh * kPer, "");

// a wave's part of a row's log sum
struct Part {
  double sum;  // of exp(x - max)
  float max;
  int pad;
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
  int segs, parts;  // of a row
  float* seg_max;   // [rows][segs]
  Part* part;       // [rows][parts]
};

typedef float float4u __attribute__((ext_vector_type(4), aligned(4)));
typedef _Float16 half8u __attribute__((ext_vector_type(8), aligned(2)));
typedef uint16_t ushort8u __attribute__((ext_vector_type(8), aligned(2)));

// a beam that has continuations: alive, and not finished
__device__ __forceinline__ bool proposes(const BeamArgs& a, int r) {
  return !(a.finished && a.finished[r]) && a.scores[r] > -INFINITY && (!a.weights || a.weights[r] > 0.f);
}

// N neighbours from entry c on, NaN and what lies behind the vocabulary as -inf
template <typename T, int N>
__device__ __forceinline__ void load_row(const T* row, int c, int vocab, float (&x)[N]) {
  if (c + N <= vocab) {
    if constexpr (sizeof(T) == 4) {
      const float4u v = *reinterpret_cast<const float4u*>(row + c);
#pragma unroll
      for (int j = 0; j < N; j++) x[j] = v[j];
    } else {
      const half8u v = *reinterpret_cast<const half8u*>(row + c);
#pragma unroll
      for (int j = 0; j < N; j++) x[j] = (float)v[j];
    }
  } else {
#pragma unroll
    for (int j = 0; j < N; j++) x[j] = c + j < vocab ? (float)row[c + j] : -INFINITY;
  }
#pragma unroll
  for (int j = 0; j < N; j++) x[j] = x[j] == x[j] ? x[j] : -INFINITY;
}

// A wave takes U loads of 64 N entries of a row.
template <typename T, int U>
__global__ __launch_bounds__(256) void part_kernel(BeamArgs a) {
  constexpr int N = 16 / sizeof(T), LS = kSeg / N, SPW = 64 / LS;  // lanes of a segment, segments of a load
  const int lane = threadIdx.x & 63, r = blockIdx.y;
  const int p = blockIdx.x * 4 + __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  if (p >= a.parts || !proposes(a, r)) return;
  const T* row = static_cast<const T*>(a.logits) + r * a.logits_row;
  const int c0 = p * (U * 64 * N) + lane * N;
  float x[U][N], top[U];
#pragma unroll
  for (int u = 0; u < U; u++) load_row<T, N>(row, c0 + u * 64 * N, a.vocab, x[u]);
  float m = -INFINITY;
#pragma unroll
  for (int u = 0; u < U; u++) {
    top[u] = x[u][0];
#pragma unroll
    for (int j = 1; j < N; j++) top[u] = fmaxf(top[u], x[u][j]);
#pragma unroll
    for (int o = LS / 2; o > 0; o >>= 1) top[u] = fmaxf(top[u], __shfl_xor(top[u], o, 64));
    m = fmaxf(m, top[u]);
  }
  if (SPW == 2) m = fmaxf(m, __shfl_xor(m, 32, 64));
  float s = 0.f;
  if (m > -INFINITY) {  // +inf: NaN, a row without candidates
#pragma unroll
    for (int u = 0; u < U; u++)
#pragma unroll
      for (int j = 0; j < N; j++) s += __builtin_amdgcn_exp2f((x[u][j] - m) * 1.44269504088896340736f);
  }
  const double sum = wave_sum_d((double)s);
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
};
__device__ __forceinline__ bool before(const Item& a, const Item& b) {
  return a.key > b.key || (a.key == b.key && a.at < b.at);
}

struct Pick {
  double key[kMaxBeams * 16 * kPer];  // those that may be among the best
  int at[kMaxBeams * 16 * kPer];
  double gkey[64];
  int gat[64], grank[64];
  int rank[64];
  int count;
  Item bar;
};

// The `want` best of the block's items (kPer a thread, n of them used, keys
// above -inf count), best(rank, item) called for each by some thread.
//
// The want-th best of 64 groups' best items is a bar that at least `want`
// items reach and few others do; ranks are counted among those.  At most the
// items of `want` groups reach it.
template <typename F>
__device__ __forceinline__ void pick(const Item (&x)[kPer], int per, int want, Pick& p, F best) {
  const int tid = threadIdx.x, lane = tid & 63;
  Item t = x[0];
#pragma unroll
  for (int j = 1; j < kPer; j++)
    if (j < per && before(x[j], t)) t = x[j];
#pragma unroll
  for (int o = 8; o > 0; o >>= 1) {
    const Item y = {__shfl_xor(t.key, o, 64), __shfl_xor(t.at, o, 64)};
    if (before(y, t)) t = y;
  }
  if ((tid & 15) == 0) {
    p.gkey[tid >> 4] = t.key;
    p.gat[tid >> 4] = t.at;
    p.grank[tid >> 4] = 0;
    p.rank[tid >> 4] = 0;
  }
  if (tid == 0) p.count = 0;
  __syncthreads();
  const Item mine = {p.gkey[lane], p.gat[lane]};
  int above = 0;
#pragma unroll
  for (int j = 0; j < 4; j++) {
    const int b = (tid >> 6) * 4 + j;
    above += before({p.gkey[b], p.gat[b]}, mine);
  }
  if (above) atomicAdd(&p.grank[lane], above);
  __syncthreads();
  if (tid < 64 && p.grank[tid] == want - 1) p.bar = mine;  // groups have different items: one has this rank
  __syncthreads();
  const Item bar = p.bar;
#pragma unroll
  for (int j = 0; j < kPer; j++)
    if (j < per && x[j].key > -INFINITY && !before(bar, x[j])) {
      const int k = atomicAdd(&p.count, 1);
      p.key[k] = x[j].key;
      p.at[k] = x[j].at;
    }
  __syncthreads();
  const int n = p.count;
  if (n <= 64) {
    if (lane < n) {
      const Item me = {p.key[lane], p.at[lane]};
      above = 0;
      for (int b = tid >> 6; b < n; b += kTh / 64) above += before({p.key[b], p.at[b]}, me);
      if (above) atomicAdd(&p.rank[lane], above);
    }
    __syncthreads();
    if (tid < n && p.rank[tid] < want) best(p.rank[tid], Item{p.key[tid], p.at[tid]});
  } else {
    for (int k = tid; k < n; k += kTh) {
      const Item me = {p.key[k], p.at[k]};
      above = 0;
      for (int b = 0; b < n && above < want; b++) above += before({p.key[b], p.at[b]}, me);
      if (above < want) best(above, me);
    }
  }
  __syncthreads();
}

// A block per request.
template <typename T>
__global__ __launch_bounds__(kTh) void choose_kernel(BeamArgs a) {
  __shared__ Pick pick_;
  __shared__ double score[kMaxBeams], lse[kMaxBeams], weight[kMaxBeams];
  __shared__ int state[kMaxBeams], length[kMaxBeams];  // 0: proposes nothing, 1: continuations, 2: itself
  __shared__ int seg_of[kMaxBeams], parent[kMaxBeams], token[kMaxBeams];
  __shared__ double score_of[kMaxBeams];
  const int tid = threadIdx.x, lane = tid & 63, W = a.beams;
  const int row0 = blockIdx.x * W;
  const T* logits = static_cast<const T*>(a.logits);
  for (int w = tid >> 6; w < W; w += kTh / 64) {
    const int r = row0 + w;
    const bool done = a.finished && a.finished[r];
    const float sc = a.scores[r], wt = a.weights ? a.weights[r] : 1.f;
    const bool live = sc > -INFINITY && wt > 0.f;
    double sum = 0.0;
    float m = -INFINITY;
    if (live && !done) {
      const Part* p = a.part + (size_t)r * a.parts;
      for (int k = lane; k < a.parts; k += 64) {
        const Part q = p[k];
        if (q.max > -INFINITY) {
          const float hi = fmaxf(m, q.max);
          // the larger one's factor is 1 (infinities: NaN, as they should be)
          sum = (m == hi ? sum : sum * exp((double)m - hi)) + (q.max == hi ? q.sum : q.sum * exp((double)q.max - hi));
          m = hi;
        }
      }
    }
    const float top = wave_max(m);
    sum = wave_sum_d(m > -INFINITY && m != top ? sum * exp((double)m - top) : sum);
    if (lane == 0) {
      score[w] = sc;
      weight[w] = wt;
      lse[w] = top + log(sum);
      state[w] = !live ? 0 : done ? 2 : 1;
      length[w] = a.lengths ? clampi(a.lengths[r], 0, a.history_max) : 0;
      seg_of[w] = -1;
      parent[w] = -1;
      token[w] = ANE_NO_TOKEN;
      score_of[w] = -INFINITY;
    }
  }
  __syncthreads();
  const auto score_at = [&](int w, float x) { return score[w] + ((double)x - lse[w]); };
  const auto key_of = [&](int w, double s) {
    const double k = s * weight[w];
    return k == k ? k : (double)-INFINITY;
  };

  // the best W segments
  Item x[kPer];
  int n = W * a.segs;
#pragma unroll
  for (int j = 0; j < kPer; j++) {
    const int t = j * kTh + tid;
    x[j] = {-INFINITY, kNone + t};
    if (t < n) {
      x[j].at = t;
      const int w = t / a.segs, g = t - w * a.segs;
      if (state[w] == 1) x[j].key = key_of(w, score_at(w, a.seg_max[(size_t)(row0 + w) * a.segs + g]));
      else if (state[w] == 2 && g == 0) x[j].key = key_of(w, score[w]);
    }
  }
  pick(x, (n + kTh - 1) / kTh, W, pick_, [&](int rank, const Item& t) { seg_of[rank] = t.at; });

  // the best W candidates in them
  n = W * kSeg;
#pragma unroll
  for (int j = 0; j < kPer; j++) {
    const int t = j * kTh + tid;
    x[j] = {-INFINITY, kNone + t};
    if (t < n && seg_of[t / kSeg] >= 0) {
      const int w = seg_of[t / kSeg] / a.segs, v = (seg_of[t / kSeg] - w * a.segs) * kSeg + t % kSeg;
      if (state[w] == 2) {
        if (t % kSeg == 0) x[j] = {key_of(w, score[w]), w * a.vocab + a.eos};
      } else if (v < a.vocab) {
        x[j].at = w * a.vocab + v;
        const float y = (float)logits[(row0 + w) * a.logits_row + v];
        if (y == y) x[j].key = key_of(w, score_at(w, y));
      }
    }
  }
  pick(x, (n + kTh - 1) / kTh, W, pick_, [&](int rank, const Item& t) {
    const int w = t.at / a.vocab, v = t.at - w * a.vocab;
    parent[rank] = w;
    token[rank] = v;
    score_of[rank] = state[w] == 2 ? score[w] : score_at(w, (float)logits[(row0 + w) * a.logits_row + v]);
  });

  if (tid < W) {
    const int r = row0 + tid, w = parent[tid];
    a.tokens[r] = token[tid];
    a.parents[r] = w < 0 ? -1 : row0 + w;
    a.scores_out[r] = (float)score_of[tid];
    if (a.finished_out) a.finished_out[r] = w >= 0 && (state[w] == 2 || token[tid] == a.eos);
  }
  if (!a.lengths) return;

  // The histories move with their beams: a stretch of columns at a time is read
  // by the block before any of it is written.
  int most = 0;
  for (int w = 0; w < W; w++) most = max(most, parent[w] >= 0 && parent[w] != w ? length[parent[w]] : 0);
  constexpr int Q = 4;
  const int wide = kTh * Q / W;  // stretches of 8 ids
  for (int c0 = 0; c0 * 8 < most; c0 += wide) {
    ushort8u v[Q];
    int c[Q], to[Q];
#pragma unroll
    for (int q = 0; q < Q; q++) {
      const int t = q * kTh + tid, w = t / wide;
      c[q] = (c0 + t - w * wide) * 8;
      to[q] = -1;
      if (w < W && parent[w] >= 0 && parent[w] != w && c[q] < length[parent[w]]) {
        to[q] = w;
        const uint16_t* h = a.history + (row0 + parent[w]) * a.history_row;
        if (c[q] + 8 <= length[parent[w]]) {
          v[q] = *reinterpret_cast<const ushort8u*>(h + c[q]);
        } else {
#pragma unroll
          for (int j = 0; j < 8; j++) v[q][j] = c[q] + j < length[parent[w]] ? h[c[q] + j] : 0;
        }
      }
    }
    __syncthreads();
#pragma unroll
    for (int q = 0; q < Q; q++)
      if (to[q] >= 0) {
        uint16_t* h = a.history + (row0 + to[q]) * a.history_row;
        const int len = length[parent[to[q]]];
        if (c[q] + 8 <= len) {
          *reinterpret_cast<ushort8u*>(h + c[q]) = v[q];
        } else {
#pragma unroll
          for (int j = 0; j < 8; j++)
            if (c[q] + j < len) h[c[q] + j] = v[q][j];
        }
      }
  }
  __syncthreads();
  if (tid < W) {
    const int r = row0 + tid, w = parent[tid];
    int len = w < 0 ? 0 : length[w];
    if (w >= 0 && state[w] == 1 && len < a.history_max) a.history[r * a.history_row + len++] = (uint16_t)token[tid];
    a.lengths[r] = len;
  }
}

// Loads of a wave in the first launch.
int loads_of(int64_t rows, int vocab, bool half) { return 2; }

struct Plan {
  int loads, segs, parts;
  int64_t seg_bytes, bytes;
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
  p->bytes = p->seg_bytes + rows * p->parts * (int64_t)sizeof(Part);
  return ANE_OK;
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
                            {"history", row_major(g.history, rows, g.history_row * 2, g.history_max * 2), true},
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
  a.part = (Part*)((char*)g.ws + p.seg_bytes);
  const hipStream_t st = (hipStream_t)stream;
  const dim3 grid((p.parts + 3) / 4, (uint32_t)rows);
  if (g.half) {
    hipLaunchKernelGGL((part_kernel<half_t, 2>), grid, dim3(256), 0, st, a);
    hipLaunchKernelGGL(choose_kernel<half_t>, dim3(g.requests), dim3(kTh), 0, st, a);
  } else {
    hipLaunchKernelGGL((part_kernel<float, 2>), grid, dim3(256), 0, st, a);
    hipLaunchKernelGGL(choose_kernel<float>, dim3(g.requests), dim3(kTh), 0, st, a);
  }
  const hipError_t h = hipGetLastError();
  if (h != hipSuccess) return op_fail(ANE_ERR_HIP, "storiesane %s: %s", op, hipGetErrorString(h));
  return ANE_OK;
}
