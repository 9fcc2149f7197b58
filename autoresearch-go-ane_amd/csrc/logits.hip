// Controls on logits and the greedy choice (ane_control_logits): penalties
// for repeated tokens, biases, masks; formulas in include/ane_serve.h.
//
// One pass over the logits: a block takes kChunk vocabulary entries of a row,
// counts the row's history over them in LDS (whole-number atomics: the order
// does not matter), then reads, changes and writes its logits and keeps the
// largest.  A second launch picks among a row's blocks.
#include <algorithm>

#include "kv8.h"
#include "op_error.h"

namespace ane {

namespace {

constexpr int kThreads = 256;
constexpr int kChunk = 4096;
constexpr uint32_t kInPrompt = 0x80000000u;

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

__device__ __forceinline__ void block_best(float& v, int& i) {
  __shared__ float sv[kThreads / 64];
  __shared__ int si[kThreads / 64];
#pragma unroll
  for (int o = 32; o > 0; o >>= 1) take(v, i, __shfl_xor(v, o, 64), __shfl_xor(i, o, 64));
  if ((threadIdx.x & 63) == 0) {
    sv[threadIdx.x >> 6] = v;
    si[threadIdx.x >> 6] = i;
  }
  __syncthreads();
#pragma unroll
  for (int w = 0; w < kThreads / 64; w++) take(v, i, sv[w], si[w]);
}

__global__ __launch_bounds__(kThreads) void control_kernel(LogitsArgs a) {
  __shared__ __attribute__((aligned(16))) uint32_t cnt[kChunk];
  const int tid = threadIdx.x;
  const int r = blockIdx.y, lo = blockIdx.x * kChunk, n = min(kChunk, a.vocab - lo);
  const bool counted = a.history != nullptr;
  float rep = 1.f, freq = 0.f, pres = 0.f;
  if (counted) {
    if (a.repetition) rep = a.repetition[r];
    if (a.frequency) freq = a.frequency[r];
    if (a.presence) pres = a.presence[r];
    for (int c = tid; c < kChunk / 4; c += kThreads) reinterpret_cast<uint4*>(cnt)[c] = make_uint4(0, 0, 0, 0);
    const int len = clampi(a.lengths[r], 0, a.history_max);
    const int prompt = a.prompts ? clampi(a.prompts[r], 0, len) : 0;
    __syncthreads();
    const uint16_t* hist = a.history + r * a.history_row;
    for (int j = tid; j < len; j += kThreads) {
      const uint32_t v = (uint32_t)hist[j] - (uint32_t)lo;
      if (v < (uint32_t)n) {
        if (j < prompt) atomicOr(&cnt[v], kInPrompt);
        else atomicAdd(&cnt[v], 1u);
      }
    }
    __syncthreads();
  }
  const float* x = a.logits + r * a.logits_row + lo;
  float best = -INFINITY;
  int at = ANE_NO_TOKEN;
  for (int c = tid; c < n; c += kThreads) {
#pragma clang fp contract(off)
    float y = x[c];
    const uint32_t w = counted ? cnt[c] : 0;
    if (w != 0) {
      y = y > 0.f ? y / rep : y * rep;
      const uint32_t o = w & ~kInPrompt;
      if (o > 0) {
        y = y - freq * (float)o;
        y = y - pres;
      }
    }
    const int v = lo + c;
    if (a.bias) y = y + a.bias[r * a.bias_row + v];
    if (a.mask && !(a.mask[r * a.mask_row + (v >> 5)] >> (v & 31) & 1)) y = -INFINITY;
    if (a.out) a.out[r * a.out_row + v] = y;
    if (y > best) {
      best = y;
      at = v;
    }
  }
  if (!a.tokens) return;
  block_best(best, at);
  if (tid == 0) {
    if (a.chunks == 1) a.tokens[r] = at;
    else a.best[(size_t)r * a.chunks + blockIdx.x] = make_float2(best, __int_as_float(at));
  }
}

__global__ __launch_bounds__(64) void choose_kernel(LogitsArgs a) {
  const int r = blockIdx.x;
  float v = -INFINITY;
  int i = ANE_NO_TOKEN;
  for (int c = threadIdx.x; c < a.chunks; c += 64) {
    const float2 p = a.best[(size_t)r * a.chunks + c];
    take(v, i, p.x, __float_as_int(p.y));
  }
#pragma unroll
  for (int o = 32; o > 0; o >>= 1) take(v, i, __shfl_xor(v, o, 64), __shfl_xor(i, o, 64));
  if (threadIdx.x == 0) a.tokens[r] = i;
}

int chunks_of(int vocab) { return (vocab + kChunk - 1) / kChunk; }

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
  const int c = chunks_of(vocab);
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
  LogitsArgs a;
  a.chunks = chunks_of(g.vocab);
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
  hipLaunchKernelGGL(control_kernel, dim3(a.chunks, g.rows), dim3(kThreads), 0, st, a);
  if (g.tokens && a.chunks > 1) hipLaunchKernelGGL(choose_kernel, dim3(g.rows), dim3(64), 0, st, a);
  const hipError_t h = hipGetLastError();
  if (h != hipSuccess) return op_fail(ANE_ERR_HIP, "storiesane %s: %s", op, hipGetErrorString(h));
  return ANE_OK;
}
