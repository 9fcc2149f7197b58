// Controls on logits and the greedy choice (ane_control_logits): penalties
// for repeated tokens, biases, masks; formulas in include/ane_serve.h.
//
// One pass over the logits: a block takes CH vocabulary entries of a row; its
// logits, mask words and biases are under way while it counts the row's
// history over them in LDS (whole-number atomics: the order does not matter).
// Where a row is several blocks', a second launch picks among their choices.
//
// What bounds it.  Many rows: bytes (400 rows of 60,011 with masks and up to
// 8000 ids: 199 MB in 53 us, 3.7 TB/s; without histories 45: each block of a
// row reads the row's history again.  A block per row, which reads it once,
// took 64).  Few rows: the chain of length, history, counts, choice and the
// second launch (one row of 32,000 7.1 us).
#include <algorithm>

#include "kv8.h"
#include "op_error.h"

namespace ane {

namespace {

constexpr uint32_t kInPrompt = 0x80000000u;  // in a token's count: it is in the prompt (below: how often in the output)

// rows and history need not be aligned beyond their elements
typedef float float4u __attribute__((ext_vector_type(4), aligned(4)));
typedef uint16_t ushort8u __attribute__((ext_vector_type(8), aligned(2)));

struct LogitsArgs {
  const float* logits;
  float* out;
  const uint16_t* history;
  const int *lengths, *prompts;
  const float *repetition, *frequency, *presence, *bias;
  const uint32_t* mask;
  int* tokens;
  float2* best;  // [rows][chunks]: value, index
  int64_t logits_row, out_row, history_row, bias_row, mask_row;
  int rows, vocab, history_max, chunks;
};

// the larger value, the lower index on ties
__device__ __forceinline__ void take(float& v, int& i, float ov, int oi) {
  if (ov > v || (ov == v && oi < i)) {
    v = ov;
    i = oi;
  }
}

// What a row is changed by.
struct Row {
  const float *x, *bias;
  const uint32_t* mask;
  const uint16_t* hist;
  float* out;
  float rep, freq, pres;
  int len, prompt;
};
__device__ __forceinline__ Row row_of(const LogitsArgs& a, int r) {
  Row w;
  w.x = a.logits + r * a.logits_row;
  w.bias = a.bias ? a.bias + r * a.bias_row : nullptr;
  w.mask = a.mask ? a.mask + r * a.mask_row : nullptr;
  w.out = a.out ? a.out + r * a.out_row : nullptr;
  w.hist = nullptr;
  w.rep = 1.f;
  w.freq = w.pres = 0.f;
  w.len = w.prompt = 0;
  if (a.history) {
    w.hist = a.history + r * a.history_row;
    w.len = clampi(a.lengths[r], 0, a.history_max);
    w.prompt = a.prompts ? clampi(a.prompts[r], 0, w.len) : 0;
    if (a.repetition) w.rep = a.repetition[r];
    if (a.frequency) w.freq = a.frequency[r];
    if (a.presence) w.pres = a.presence[r];
  }
  return w;
}

__device__ __forceinline__ float4u load4(const float* p, int c, int vocab) {
  if (c + 3 < vocab) return *reinterpret_cast<const float4u*>(p + c);
  float4u v = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
  for (int j = 0; j < 3; j++)
    if (c + j < vocab) v[j] = p[c + j];
  return v;
}

// The row's first ids, eight a thread, on their way before its length is known
// (they lie within history_max).
template <int TH>
__device__ __forceinline__ ushort8u first_ids(const LogitsArgs& a, const Row& w) {
  const int j = threadIdx.x * 8;
  ushort8u h;
#pragma unroll
  for (int u = 0; u < 8; u++) h[u] = 0xffff;
  if (!w.hist) return h;
  if (j + 7 < a.history_max) return *reinterpret_cast<const ushort8u*>(w.hist + j);
#pragma unroll
  for (int u = 0; u < 7; u++)
    if (j + u < a.history_max) h[u] = w.hist[j + u];
  return h;
}
// count(j, id) for the row's ids
template <int TH, typename F>
__device__ __forceinline__ void for_history(const Row& w, const ushort8u& first, F count) {
  int j = threadIdx.x * 8;
#pragma unroll
  for (int u = 0; u < 8; u++)
    if (j + u < w.len) count(j + u, first[u]);
  for (j += TH * 8; j < w.len; j += TH * 8) {
    if (j + 7 < w.len) {
      const ushort8u h = *reinterpret_cast<const ushort8u*>(w.hist + j);
#pragma unroll
      for (int u = 0; u < 8; u++) count(j + u, h[u]);
    } else {
      for (int u = 0; u < 7; u++)
        if (j + u < w.len) count(j + u, w.hist[j + u]);
    }
  }
}

// Four neighbours from entry c on: penalties by their counts, bias and mask,
// each step rounded; written, and the best kept.
__device__ __forceinline__ void change4(const Row& w, float4u x, const uint32_t (&n)[4], float4u bias, uint32_t word,
                                        int c, int vocab, float& best, int& at) {
#pragma clang fp contract(off)
#pragma unroll
  for (int j = 0; j < 4; j++) {
    float v = x[j];
    if (n[j] != 0) {
      v = v > 0.f ? v / w.rep : v * w.rep;
      const uint32_t o = n[j] & ~kInPrompt;
      if (o > 0) {
        v = v - w.freq * (float)o;
        v = v - w.pres;
      }
    }
    if (w.bias) v = v + bias[j];
    if (!(word >> ((c + j) & 31) & 1)) v = -INFINITY;
    x[j] = v;
    if (c + j < vocab && v > best) {
      best = v;
      at = c + j;
    }
  }
  if (w.out) {
    if (c + 3 < vocab) {
      *reinterpret_cast<float4u*>(w.out + c) = x;
    } else {
#pragma unroll
      for (int j = 0; j < 3; j++)
        if (c + j < vocab) w.out[c + j] = x[j];
    }
  }
}

// the block's best, in thread 0
template <int TH>
__device__ __forceinline__ void block_best(float& v, int& i) {
  __shared__ float sv[TH / 64];
  __shared__ int si[TH / 64];
#pragma unroll
  for (int o = 32; o > 0; o >>= 1) take(v, i, __shfl_xor(v, o, 64), __shfl_xor(i, o, 64));
  if ((threadIdx.x & 63) == 0) {
    sv[threadIdx.x >> 6] = v;
    si[threadIdx.x >> 6] = i;
  }
  __syncthreads();
  if (threadIdx.x == 0) {
#pragma unroll
    for (int k = 1; k < TH / 64; k++) take(v, i, sv[k], si[k]);
  }
}

// A block takes CH entries of a row.
template <int CH, int TH>
__global__ __launch_bounds__(TH) void part_kernel(LogitsArgs a) {
  constexpr int Q = CH / 4 / TH;
  static_assert(Q * 4 * TH == CH, "");
  extern __shared__ __attribute__((aligned(16))) uint32_t cnt[];
  const int tid = threadIdx.x, r = blockIdx.y, lo = blockIdx.x * CH;
  const Row w = row_of(a, r);
  const ushort8u ids = first_ids<TH>(a, w);
  float4u x[Q], bias[Q];
  uint32_t word[Q];
#pragma unroll
  for (int q = 0; q < Q; q++) {
    const int c = lo + (q * TH + tid) * 4;
    x[q] = load4(w.x, c, a.vocab);
    bias[q] = w.bias ? load4(w.bias, c, a.vocab) : float4u{0.f, 0.f, 0.f, 0.f};
    word[q] = w.mask && c < a.vocab ? w.mask[c >> 5] : 0xffffffffu;
  }
  if (w.hist) {
#pragma unroll
    for (int q = 0; q < Q; q++) reinterpret_cast<uint4*>(cnt)[q * TH + tid] = make_uint4(0, 0, 0, 0);
    __syncthreads();
    for_history<TH>(w, ids, [&](int j, uint16_t id) {
      const uint32_t v = (uint32_t)id - (uint32_t)lo;
      if (v < (uint32_t)CH) {
        if (j < w.prompt) atomicOr(&cnt[v], kInPrompt);
        else atomicAdd(&cnt[v], 1u);
      }
    });
    __syncthreads();
  }
  float best = -INFINITY;
  int at = ANE_NO_TOKEN;
#pragma unroll
  for (int q = 0; q < Q; q++) {
    uint32_t n[4] = {0, 0, 0, 0};
    if (w.hist) {
      const uint4 k = reinterpret_cast<const uint4*>(cnt)[q * TH + tid];
      n[0] = k.x; n[1] = k.y; n[2] = k.z; n[3] = k.w;
    }
    change4(w, x[q], n, bias[q], word[q], lo + (q * TH + tid) * 4, a.vocab, best, at);
  }
  if (!a.tokens) return;
  block_best<TH>(best, at);
  if (tid == 0) {
    if (gridDim.x == 1) a.tokens[r] = at;
    else a.best[(size_t)r * gridDim.x + blockIdx.x] = make_float2(best, __int_as_float(at));
  }
}

// A wave per row.
__global__ __launch_bounds__(256) void choose_kernel(LogitsArgs a) {
  const int r = blockIdx.x * 4 + (threadIdx.x >> 6);
  if (r >= a.rows) return;
  float v = -INFINITY;
  int i = ANE_NO_TOKEN;
  for (int c = threadIdx.x & 63; c < a.chunks; c += 64) {
    const float2 p = a.best[(size_t)r * a.chunks + c];
    take(v, i, p.x, __float_as_int(p.y));
  }
#pragma unroll
  for (int o = 32; o > 0; o >>= 1) take(v, i, __shfl_xor(v, o, 64), __shfl_xor(i, o, 64));
  if ((threadIdx.x & 63) == 0) a.tokens[r] = i;
}

// Entries a block takes of a row.  Few rows: small parts, for latency and for
// enough blocks (1 row of 32000: 7.1 us against 8.2 in parts of 8192; 64 rows
// 12.2 against 12.9).  Many rows: large ones, since every part reads the
// history again (400 rows of 60011 with 8000 ids 53 us against 62; 400 of 5000
// 9.8 against 12.2, with nothing left to choose among).  The two are equal at
// 128 rows of 32000.
int chunk_of(int rows) { return rows >= 128 ? 8192 : 2048; }
int chunks_of(int rows, int vocab) {
  const int c = chunk_of(rows);
  return (vocab + c - 1) / c;
}

template <int CH, int TH>
void launch_parts(const LogitsArgs& a, hipStream_t st) {
  const size_t lds = a.history ? (size_t)CH * 4 : 0;
  hipLaunchKernelGGL((part_kernel<CH, TH>), dim3(a.chunks, a.rows), dim3(TH), lds, st, a);
}

int check_sizes(const char* op, int rows, int vocab) {
  if (rows < 0 || rows > 65535 || vocab < 1 || vocab > 65535)
    return op_fail(ANE_ERR_ARG, "storiesane %s: rows=%d want 0..65535, vocab=%d want 1..65535", op, rows, vocab);
  return ANE_OK;
}

}  // namespace

}  // namespace ane

using namespace ane;

extern "C" int64_t ane_control_logits_workspace(int32_t rows, int32_t vocab) {
  const int rc = check_sizes("control logits workspace", rows, vocab);
  if (rc) return rc;
  const int c = chunks_of(rows, vocab);
  return c > 1 ? (int64_t)rows * c * 8 : 0;
}

extern "C" int ane_control_logits(const ane_logits_args* args, void* stream) {
  const char* op = "control logits";
  if (!args) return op_fail(ANE_ERR_ARG, "storiesane %s: null arguments", op);
  const ane_logits_args& g = *args;
  int rc = check_sizes(op, g.rows, g.vocab);
  if (rc) return rc;
  if (g.rows == 0) return ANE_OK;  // an empty tensor may have no address
  if (!g.logits) return op_fail(ANE_ERR_ARG, "storiesane %s: null buffer", op);
  if (!g.out && !g.tokens) return op_fail(ANE_ERR_ARG, "storiesane %s: neither out nor tokens", op);
  if (g.history_max < 0 || (g.history && (!g.lengths || g.history_row < g.history_max)) ||
      (!g.history && g.history_max > 0))
    return op_fail(ANE_ERR_ARG, "storiesane %s: history without lengths, or not of history_max=%d within its stride %lld",
                   op, g.history_max, (long long)g.history_row);
  if (!g.history && !g.lengths && (g.repetition || g.frequency || g.presence))
    return op_fail(ANE_ERR_ARG, "storiesane %s: penalties without a history", op);
  const int64_t words = (g.vocab + 31) / 32;
  if (g.logits_row < g.vocab || (g.out && g.out_row < g.vocab) || (g.bias && g.bias_row && g.bias_row < g.vocab) ||
      (g.mask && g.mask_row && g.mask_row < words))
    return op_fail(ANE_ERR_ARG, "storiesane %s: a row stride is shorter than its row (vocab=%d)", op, g.vocab);
  if (g.out == g.logits && g.out_row != g.logits_row)
    return op_fail(ANE_ERR_ARG, "storiesane %s: in place, but out_row=%lld and logits_row=%lld", op,
                   (long long)g.out_row, (long long)g.logits_row);
  if (g.out && g.out != g.logits &&
      share_memory({(uintptr_t)g.out, g.rows, g.out_row * 4, 1, 0, g.vocab * 4},
                   {(uintptr_t)g.logits, g.rows, g.logits_row * 4, 1, 0, g.vocab * 4}))
    return op_fail(ANE_ERR_ARG, "storiesane %s: out overlaps logits in part", op);
  LogitsArgs a;
  a.chunks = chunks_of(g.rows, g.vocab);
  const int64_t need = a.chunks > 1 && g.tokens ? (int64_t)g.rows * a.chunks * 8 : 0;
  if (((uintptr_t)g.ws & 15) || (need > 0 && (!g.ws || g.ws_bytes < need)))
    return op_fail(ANE_ERR_ARG, "storiesane %s: workspace of %lld bytes, want %lld, 16-byte aligned", op,
                   (long long)(g.ws ? g.ws_bytes : 0), (long long)need);
  DeviceScope dev(g.device);
  if (dev.status() != hipSuccess)
    return op_fail(ANE_ERR_HIP, "storiesane %s: device %d: %s", op, g.device, hipGetErrorString(dev.status()));
  const bool counted = g.history && g.history_max > 0 && (g.repetition || g.frequency || g.presence);
  a.logits = g.logits; a.out = g.out; a.history = counted ? g.history : nullptr; a.lengths = g.lengths;
  a.prompts = g.prompts; a.repetition = g.repetition; a.frequency = g.frequency; a.presence = g.presence;
  a.bias = g.bias; a.mask = g.mask; a.tokens = g.tokens; a.best = (float2*)g.ws;
  a.logits_row = g.logits_row; a.out_row = g.out_row; a.history_row = g.history_row; a.bias_row = g.bias_row;
  a.mask_row = g.mask_row; a.rows = g.rows; a.vocab = g.vocab; a.history_max = g.history_max;
  const hipStream_t st = (hipStream_t)stream;
  if (chunk_of(g.rows) == 8192) launch_parts<8192, 512>(a, st);
  else launch_parts<2048, 256>(a, st);
  if (g.tokens && a.chunks > 1) hipLaunchKernelGGL(choose_kernel, dim3((g.rows + 3) / 4), dim3(256), 0, st, a);
  const hipError_t h = hipGetLastError();
  if (h != hipSuccess) return op_fail(ANE_ERR_HIP, "storiesane %s: %s", op, hipGetErrorString(h));
  return ANE_OK;
}
