// What the kernels that append rows to the 8-bit cache share: the rotation, the
// codes, and the appending of few rows by one wave.
#ifndef ANE_KV8_ROWS_H
#define ANE_KV8_ROWS_H

#include "decode.h"
#include "kv8.h"

namespace ane {

struct Kv8AppendArgs {
  Kv8Batch b;
  uint8_t *k, *v;
  int8_t *k_exp, *v_exp;
  const half_t *xq, *xk, *xv;
  half_t* q_out;
  const float *cos, *sin;
  int64_t q_row, q_head, k_row, k_head, v_row, v_head, qo_row, qo_head;
  int heads;
  int by_row;    // append_few_kernel: items are rows, not pages
  Kv8Sums from;  // where the rows come from in the SUMS form, instead of xq, xk, xv
};

struct F8 {
  float x[8];
};

__device__ __forceinline__ F8 wide8(half8 h) {
  F8 f;
#pragma unroll
  for (int j = 0; j < 8; j++) f.x[j] = (float)h[j];
  return f;
}

// rounded to fp16 from fp32 as it stands: an instruction that multiplies, adds
// and rounds to fp16 at once would round some numbers the other way
__device__ __forceinline__ half8 narrow8(F8 f) {
  half8 h;
#pragma unroll
  for (int j = 0; j < 8; j++) {
    asm volatile("" : "+v"(f.x[j]));
    h[j] = (half_t)f.x[j];
  }
  return h;
}

// dimensions d0 .. d0 + 7 of row r, columns from `col` on, of a product's sums
// over its splits, rounded to fp16 as the rows are elsewhere
__device__ __forceinline__ half8 sums8(const Kv8Sums& p, int r, int col) {
  float4 lo = {0.f, 0.f, 0.f, 0.f}, hi = lo;
  const float* x = p.part + (size_t)r * p.n + col;
  for (int s = 0; s < p.splits; s++, x += (size_t)kDecRows * p.n) {
    const float4 u = *reinterpret_cast<const float4*>(x), v = *reinterpret_cast<const float4*>(x + 4);
    lo.x += u.x; lo.y += u.y; lo.z += u.z; lo.w += u.w;
    hi.x += v.x; hi.y += v.y; hi.z += v.z; hi.w += v.w;
  }
  const float w = p.row_scale ? p.row_scale[r] : 1.f;
  return narrow8({lo.x * w, lo.y * w, lo.z * w, lo.w * w, hi.x * w, hi.y * w, hi.z * w, hi.w * w});
}

// the cosines and sines of the four pairs of dimensions from d0 on
struct Turn {
  float4 c, s;
};
template <int DH>
__device__ __forceinline__ Turn turn_of(const float* cs, const float* sn, int pos, int d0) {
  return {*reinterpret_cast<const float4*>(cs + (size_t)pos * (DH / 2) + d0 / 2),
          *reinterpret_cast<const float4*>(sn + (size_t)pos * (DH / 2) + d0 / 2)};
}
// a product rounded, then a multiply-add: written out, for the same bits in
// every kernel
__device__ __forceinline__ F8 rotate8(half8 h, const Turn& w) {
  const F8 f = wide8(h);
  const float cc[4] = {w.c.x, w.c.y, w.c.z, w.c.w}, ss[4] = {w.s.x, w.s.y, w.s.z, w.s.w};
  F8 r;
#pragma unroll
  for (int j = 0; j < 4; j++) {
    r.x[2 * j] = __builtin_fmaf(f.x[2 * j], cc[j], -(f.x[2 * j + 1] * ss[j]));
    r.x[2 * j + 1] = __builtin_fmaf(f.x[2 * j + 1], cc[j], f.x[2 * j] * ss[j]);
  }
  return r;
}

// into +-65504, by comparisons: NaN stays
__device__ __forceinline__ void limit8(F8& f) {
#pragma unroll
  for (int j = 0; j < 8; j++) f.x[j] = f.x[j] > 65504.f ? 65504.f : f.x[j] < -65504.f ? -65504.f : f.x[j];
}

// largest magnitude as float bits, NaN counted as 0
__device__ __forceinline__ uint32_t amax8(const F8& f, uint32_t m) {
#pragma unroll
  for (int j = 0; j < 8; j++) {
    const uint32_t u = __float_as_uint(f.x[j]) & 0x7fffffffu;
    m = max(m, u > 0x7f800000u ? 0u : u);
  }
  return m;
}

// 4 codes of x * inv, inv a power of two; top: 240 at exponent 8, else 448
// (at which the exponent already holds every number)
__device__ __forceinline__ uint32_t codes4(const float* x, float inv, float top) {
  float y[4];
#pragma unroll
  for (int j = 0; j < 4; j++) {
    y[j] = x[j] * inv;
    y[j] = y[j] > top ? top : y[j] < -top ? -top : y[j];
  }
  int c = __builtin_amdgcn_cvt_pk_fp8_f32(y[0], y[1], 0, false);
  return (uint32_t)__builtin_amdgcn_cvt_pk_fp8_f32(y[2], y[3], c, true);
}

// 4 codes rounded again at a larger exponent
__device__ __forceinline__ uint32_t again4(uint32_t c, float down) {
  const auto lo = __builtin_amdgcn_cvt_pk_f32_fp8((int)c, false);
  const auto hi = __builtin_amdgcn_cvt_pk_f32_fp8((int)c, true);
  int r = __builtin_amdgcn_cvt_pk_fp8_f32(lo[0] * down, lo[1] * down, 0, false);
  return (uint32_t)__builtin_amdgcn_cvt_pk_fp8_f32(hi[0] * down, hi[1] * down, r, true);
}

// LDS accesses of a wave stay in order; this keeps the compiler to it
__device__ __forceinline__ void wave_order() {
  __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
  __builtin_amdgcn_wave_barrier();
}

// Rows span.row .. of one page and key/value head h, by one wave: 64 / CPR rows
// at a time, V a unit of 16 tokens at a time in `unit` (LDS).  Rows past the
// first pass are read again for their codes.  SUMS: the rows come from a
// product's sums.
template <int DH, bool SUMS>
__device__ __forceinline__ void kv8_append_rows(const Kv8AppendArgs& a, const Kv8Span& span, int h, uint4 (&unit)[DH]) {
  constexpr int CPR = DH / 8, G = 64 / CPR, T = DH / 16;
  const Kv8Batch& b = a.b;
  const int lane = threadIdx.x & 63, sub = lane / CPR, d0 = lane % CPR * 8;
  const int P = 1 << b.pshift;
  const int nr = span.n, row0 = span.row, t0 = span.pos;
  const int id = kv8_page(b, span.seq, t0 >> b.pshift);
  F8 fk, fv;
  auto rows = [&](int r) {  // the lane's part of row r
    r = min(r, nr - 1);     // rows past the last repeat it
    const half8 k = SUMS ? sums8(a.from, row0 + r, (a.heads + h) * DH + d0)
                         : ld_h8(a.xk + (row0 + r) * a.k_row + h * a.k_head + d0);
    const half8 v = SUMS ? sums8(a.from, row0 + r, (a.heads + b.NKV + h) * DH + d0)
                         : ld_h8(a.xv + (row0 + r) * a.v_row + h * a.v_head + d0);
    fk = rotate8(k, turn_of<DH>(a.cos, a.sin, t0 + r, d0));
    fv = wide8(v);
    limit8(fk);
    limit8(fv);
  };
  uint32_t mk = 0, mv = 0;
  for (int g = 0; g < nr; g += G) {
    rows(g + sub);
    mk = amax8(fk, mk);
    mv = amax8(fv, mv);
  }
  if (id < 0) return;
  const size_t ph = (size_t)id * b.NKV + h;
  uint8_t* kp = a.k + ph * P * DH;
  uint8_t* vp = a.v + ph * P * DH;
  const int r0 = t0 & (P - 1), r1 = r0 + nr;
  int ok = kKvExpMin, ov = kKvExpMin;
  if (r0 > 0) {
    ok = a.k_exp[ph];
    ov = a.v_exp[ph];
  }
  const int u0 = r0 >> 4, u1 = (r1 - 1) >> 4;
  uint4 was[DH / 64];  // the first unit
#pragma unroll
  for (int i = 0; i < DH / 64; i++) was[i] = reinterpret_cast<const uint4*>(vp)[u0 * DH + i * 64 + lane];
#pragma unroll
  for (int o = 32; o > 0; o >>= 1) {
    mk = max(mk, (uint32_t)__shfl_xor((int)mk, o, 64));
    mv = max(mv, (uint32_t)__shfl_xor((int)mv, o, 64));
  }
  const int ek = max(kv8_exponent(mk), ok), ev = max(kv8_exponent(mv), ov);
  if (lane == 0) {
    a.k_exp[ph] = (int8_t)ek;
    a.v_exp[ph] = (int8_t)ev;
  }
  const float ik = kv8_scale(-ek), iv = kv8_scale(-ev);
  const float tk = ek == kKvExpMax ? 240.f : 448.f, tv = ev == kKvExpMax ? 240.f : 448.f;

  // rows from before, rounded again where the exponent rose
  if (r0 > 0 && ek > ok) {
    const float down = kv8_scale(ok - ek);
    uint32_t* x = reinterpret_cast<uint32_t*>(kp);
    for (int c = lane; c < r0 * DH / 4; c += 64) x[c] = again4(x[c], down);
  }
  const bool up = r0 > 0 && ev > ov;
  const float down = kv8_scale(ov - ev);
  if (up) {  // whole units of them
    uint32_t* x = reinterpret_cast<uint32_t*>(vp);
    for (int c = lane; c < u0 * 4 * DH; c += 64) x[c] = again4(x[c], down);
  }
  for (int u = u0; u <= u1; u++) {
    const int s0 = max(r0, 16 * u), s1 = min(r1, 16 * u + 16);  // the new rows of this unit
#pragma unroll
    for (int i = 0; i < DH / 64; i++) {
      const int c = i * 64 + lane;
      uint4 x = was[i];
      if (up && u == u0) {
        const int n = clampi(r0 - (16 * u + 4 * c / DH * 4), 0, 4);  // of its four tokens, those from before
        const uint32_t mine = n == 4 ? 0xffffffffu : (1u << (8 * n)) - 1;
        x.x = (again4(x.x, down) & mine) | (x.x & ~mine);
        x.y = (again4(x.y, down) & mine) | (x.y & ~mine);
        x.z = (again4(x.z, down) & mine) | (x.z & ~mine);
        x.w = (again4(x.w, down) & mine) | (x.w & ~mine);
      }
      unit[c] = x;
      if (u < u1) was[i] = reinterpret_cast<const uint4*>(vp)[(u + 1) * DH + c];
    }
    wave_order();
    for (int g = (s0 - r0) / G * G; g < s1 - r0; g += G) {
      if (nr > G) rows(g + sub);
      const int s = r0 + g + sub;
      if (s < s0 || s >= s1) continue;
      *reinterpret_cast<uint2*>(kp + s * DH + d0) = make_uint2(codes4(fk.x, ik, tk), codes4(fk.x + 4, ik, tk));
      const uint32_t cv[2] = {codes4(fv.x, iv, tv), codes4(fv.x + 4, iv, tv)};
      uint8_t* y = reinterpret_cast<uint8_t*>(unit) + (s & 15) / 4 * 4 * DH + (s & 3);
#pragma unroll
      for (int j = 0; j < 8; j++) {
        const int d = d0 + j;
        y[((d & 15) * T + (d >> 4)) * 4] = (uint8_t)(cv[j / 4] >> (8 * (j & 3)));
      }
    }
    wave_order();
#pragma unroll
    for (int i = 0; i < DH / 64; i++) reinterpret_cast<uint4*>(vp)[u * DH + i * 64 + lane] = unit[i * 64 + lane];
    wave_order();
  }
}

// Host: checks an append of operator `op` and fills the kernels' form; nothing
// of it but the batch where there are no rows.
int kv8_append_check(const char* op, const ane_kv8_cache* cache, const ane_kv8_batch* batch,
                     const ane_kv8_append_args* args, const Kv8Sums* from, Kv8AppendArgs* into);

}  // namespace ane

#endif
