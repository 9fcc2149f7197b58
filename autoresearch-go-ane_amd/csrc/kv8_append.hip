// Append to the paged 8-bit cache, with the rotation on the way
// (ane_kv8_append), and the checks both cache operators share.
//
// Mathematics: include/ane_serve.h.  One block per (page that gets rows, kv
// head) holds its new keys and values in registers, rotates the keys, takes
// the largest magnitude of each side over the block, and writes codes; no
// other block touches that page and head, so a page's rows from before can be
// rounded again in place when its exponent rises.  V's codes go through LDS
// into the order of the cache.  Blocks behind the kv heads rotate the queries
// of the same rows, kQHeads heads each.
//
// What bounds it.  Prompts: bytes, each read and written once (24 ragged
// prompts, 18,000 tokens, 12 / 4 heads of 64: 100 MB in 22.8 us, 4.4 TB/s).
// Single tokens, which a wave per page and head takes: a chain of loads,
// offsets, page id, rows, old exponent and codes, each waiting for the one
// before (one token 4.3 us, 64 of them 4.5 in a graph); the rows and their
// angles are asked for while the page id is under way.
#include <algorithm>
#include <utility>

#include "kv8_rows.h"
#include "op_error.h"

namespace ane {

namespace {

constexpr int kQHeads = 4;

// NC * TH chunks of 8 dimensions are a page's.
template <int DH, int NC, int TH>
__global__ __launch_bounds__(TH) void append_kernel(Kv8AppendArgs a) {
  constexpr int CPR = DH / 8;  // chunks per row
  constexpr int T = DH / 16;
  __shared__ __attribute__((aligned(16))) uint8_t vbuf[NC * TH * 8];  // the page's V codes
  __shared__ uint32_t top[2][TH / 64];
  const Kv8Batch& b = a.b;
  const int tid = threadIdx.x;
  const int P = 1 << b.pshift;
  const Kv8Span span = kv8_page_span(b, blockIdx.x);
  if (span.n == 0) return;
  const int nr = span.n, row0 = span.row, t0 = span.pos;

  if ((int)blockIdx.y >= b.NKV) {  // query heads
    const int h0 = (blockIdx.y - b.NKV) * kQHeads;
    for (int c = tid; c < nr * CPR; c += TH) {
      const int r = c / CPR, d0 = c % CPR * 8;
      const Turn w = turn_of<DH>(a.cos, a.sin, t0 + r, d0);
      const half_t* x = a.xq + (row0 + r) * a.q_row + d0;
      half_t* y = a.q_out + (row0 + r) * a.qo_row + d0;
      half8 in[kQHeads];
#pragma unroll
      for (int k = 0; k < kQHeads; k++)
        if (h0 + k < a.heads) in[k] = ld_h8(x + (h0 + k) * a.q_head);
#pragma unroll
      for (int k = 0; k < kQHeads; k++)
        if (h0 + k < a.heads) st_h8(y + (h0 + k) * a.qo_head, narrow8(rotate8(in[k], w)));
    }
    return;
  }

  const int h = blockIdx.y;
  const half_t* xk = a.xk + row0 * a.k_row + h * a.k_head;
  const half_t* xv = a.xv + row0 * a.v_row + h * a.v_head;
  const int id = kv8_page(b, span.seq, t0 >> b.pshift);
  half8 hk[NC], hv[NC];
  Turn w[NC];
#pragma unroll
  for (int i = 0; i < NC; i++) {
    const int c = min(i * TH + tid, nr * CPR - 1), r = c / CPR, d0 = c % CPR * 8;
    hk[i] = ld_h8(xk + r * a.k_row + d0);
    hv[i] = ld_h8(xv + r * a.v_row + d0);
    w[i] = turn_of<DH>(a.cos, a.sin, t0 + r, d0);
  }
  if (id < 0) return;  // the same in the whole block
  const size_t ph = (size_t)id * b.NKV + h;
  uint8_t* kp = a.k + ph * P * DH;
  uint8_t* vp = a.v + ph * P * DH;
  const int r0 = t0 & (P - 1), r1 = r0 + nr;
  int ok = kKvExpMin, ov = kKvExpMin;
  if (r0 > 0) {
    ok = a.k_exp[ph];
    ov = a.v_exp[ph];
  }
  // V's units of 16 tokens that the new rows fill in part: their codes first
  const int u0 = r0 >> 4, u1 = (r1 - 1) >> 4;
  {
    const uint4* src = reinterpret_cast<const uint4*>(vp);
    uint4* dst = reinterpret_cast<uint4*>(vbuf);
    for (int c = tid; c < 2 * DH; c += TH) {
      const int u = c < DH ? u0 : u1, at = u * DH + (c & (DH - 1));
      const bool part = c < DH ? (r0 & 15) || (u0 == u1 && (r1 & 15)) : u1 > u0 && (r1 & 15);
      if (part) dst[at] = src[at];
    }
  }
  F8 fk[NC];
  uint32_t mk = 0, mv = 0;
#pragma unroll
  for (int i = 0; i < NC; i++) {
    fk[i] = rotate8(hk[i], w[i]);
    limit8(fk[i]);
    mk = amax8(fk[i], mk);  // chunks past the last row repeat it
    F8 f = wide8(hv[i]);
    limit8(f);
    mv = amax8(f, mv);
  }
#pragma unroll
  for (int o = 32; o > 0; o >>= 1) {
    mk = max(mk, (uint32_t)__shfl_xor((int)mk, o, 64));
    mv = max(mv, (uint32_t)__shfl_xor((int)mv, o, 64));
  }
  if ((tid & 63) == 0) {
    top[0][tid >> 6] = mk;
    top[1][tid >> 6] = mv;
  }
  __syncthreads();  // every thread has read the old exponents too
#pragma unroll
  for (int k = 0; k < TH / 64; k++) {
    mk = max(mk, top[0][k]);
    mv = max(mv, top[1][k]);
  }
  const int ek = max(kv8_exponent(mk), ok), ev = max(kv8_exponent(mv), ov);
  if (tid == 0) {
    a.k_exp[ph] = (int8_t)ek;
    a.v_exp[ph] = (int8_t)ev;
  }
  const float ik = kv8_scale(-ek), iv = kv8_scale(-ev);
  const float tk = ek == kKvExpMax ? 240.f : 448.f, tv = ev == kKvExpMax ? 240.f : 448.f;

  // rows from before, rounded again where the exponent rose
  if (r0 > 0 && ek > ok) {
    const float down = kv8_scale(ok - ek);
    uint32_t* x = reinterpret_cast<uint32_t*>(kp);
    for (int c = tid; c < r0 * DH / 4; c += TH) x[c] = again4(x[c], down);
  }
  if (r0 > 0 && ev > ov) {
    const float down = kv8_scale(ov - ev);
    uint32_t* x = reinterpret_cast<uint32_t*>(vp);
    for (int c = tid; c < u0 * 4 * DH; c += TH) x[c] = again4(x[c], down);  // whole units of them
    x = reinterpret_cast<uint32_t*>(vbuf);
    for (int c = u0 * 4 * DH + tid; c < (u0 + 1) * 4 * DH && (r0 & 15); c += TH) {
      const int n = clampi(r0 - (u0 * 16 + c % (4 * DH) / (16 * T) * 4), 0, 4);  // of the dword's four tokens
      const uint32_t mine = n == 4 ? 0xffffffffu : (1u << (8 * n)) - 1;
      x[c] = (again4(x[c], down) & mine) | (x[c] & ~mine);
    }
    __syncthreads();
  }
#pragma unroll
  for (int i = 0; i < NC; i++) {
    const int c = i * TH + tid;
    if (c >= nr * CPR) break;
    const int s = r0 + c / CPR, d0 = c % CPR * 8;
    *reinterpret_cast<uint2*>(kp + s * DH + d0) = make_uint2(codes4(fk[i].x, ik, tk), codes4(fk[i].x + 4, ik, tk));
    const F8 f = wide8(hv[i]);
    const uint32_t cv[2] = {codes4(f.x, iv, tv), codes4(f.x + 4, iv, tv)};
    uint8_t* y = vbuf + (s >> 4) * 16 * DH + (s & 15) / 4 * 4 * DH + (s & 3);
#pragma unroll
    for (int j = 0; j < 8; j++) {
      const int d = d0 + j;
      y[((d & 15) * T + (d >> 4)) * 4] = (uint8_t)(cv[j / 4] >> (8 * (j & 3)));
    }
  }
  __syncthreads();
  const uint4* src = reinterpret_cast<const uint4*>(vbuf);
  uint4* dst = reinterpret_cast<uint4*>(vp);
  for (int c = u0 * DH + tid; c < (u1 + 1) * DH; c += TH) dst[c] = src[c];
}

// The same for few new rows: a wave per page and head (kv8_rows.h), and one per
// 64 / CPR query heads.
template <int DH, bool SUMS>
__global__ __launch_bounds__(64) void append_few_kernel(Kv8AppendArgs a) {
  constexpr int CPR = DH / 8, G = 64 / CPR;
  __shared__ uint4 unit[DH];  // 16 tokens' V codes
  const Kv8Batch& b = a.b;
  const int lane = threadIdx.x, sub = lane / CPR, d0 = lane % CPR * 8;
  const Kv8Span span = a.by_row ? kv8_row_page_span(b, blockIdx.x) : kv8_page_span(b, blockIdx.x);
  if (span.n == 0) return;
  if (SUMS && a.from.err && *a.from.err) return;
  const int nr = span.n, row0 = span.row, t0 = span.pos;

  if ((int)blockIdx.y >= b.NKV) {  // query heads
    const int h = (blockIdx.y - b.NKV) * G + sub;
    if (h >= a.heads) return;
    for (int r = 0; r < nr; r++) {
      const Turn w = turn_of<DH>(a.cos, a.sin, t0 + r, d0);
      const half8 x = SUMS ? sums8(a.from, row0 + r, h * DH + d0)
                           : ld_h8(a.xq + (row0 + r) * a.q_row + h * a.q_head + d0);
      st_h8(a.q_out + (row0 + r) * a.qo_row + h * a.qo_head + d0, narrow8(rotate8(x, w)));
    }
    return;
  }

  kv8_append_rows<DH, SUMS>(a, span, blockIdx.y, unit);
}

template <int DH>
void launch(const Kv8AppendArgs& a, dim3 grid, hipStream_t st) {
  switch ((DH / 8) << a.b.pshift) {
    case 128: hipLaunchKernelGGL((append_kernel<DH, 1, 128>), grid, dim3(128), 0, st, a); break;
    case 256: hipLaunchKernelGGL((append_kernel<DH, 1, 256>), grid, dim3(256), 0, st, a); break;
    case 512: hipLaunchKernelGGL((append_kernel<DH, 2, 256>), grid, dim3(256), 0, st, a); break;
    case 1024: hipLaunchKernelGGL((append_kernel<DH, 4, 256>), grid, dim3(256), 0, st, a); break;
    case 2048: hipLaunchKernelGGL((append_kernel<DH, 4, 512>), grid, dim3(512), 0, st, a); break;
    default: hipLaunchKernelGGL((append_kernel<DH, 4, 1024>), grid, dim3(1024), 0, st, a); break;
  }
}

bool aligned16(const void* p) { return ((uintptr_t)p & 15) == 0; }

}  // namespace

namespace {

int64_t floor_div(int64_t x, int64_t y) { return x / y - (x % y < 0); }

// Whether any [i sa, i sa + wa), i < na, meets any [d + j sb, d + j sb + wb), j < nb.
bool meet(int64_t na, int64_t sa, int64_t wa, int64_t d, int64_t nb, int64_t sb, int64_t wb) {
  for (int64_t i = 0; i < (sa ? na : 1); i++) {
    const int64_t lo = i * sa - d - wb, hi = i * sa - d + wa;  // lo < j sb < hi
    if (sb == 0 ? lo < 0 && hi > 0
                : std::max<int64_t>(0, floor_div(lo, sb) + 1) <= std::min(nb - 1, -floor_div(-hi, sb) - 1))
      return true;
  }
  return false;
}

}  // namespace

bool share_memory(Extent a, Extent b) {
  for (Extent* e : {&a, &b}) {
    if (e->rows <= 0 || e->heads <= 0 || e->width <= 0) return false;
    if (e->rows == 1) e->row = 0;
    if (e->heads == 1) e->head = 0;
    if (e->head > e->row) {  // the longer stride outside
      std::swap(e->rows, e->heads);
      std::swap(e->row, e->head);
    }
  }
  const int64_t ea = (a.heads - 1) * a.head + a.width, eb = (b.heads - 1) * b.head + b.width;  // of a row
  const int64_t d = (int64_t)(b.at - a.at);
  if (d >= (a.rows - 1) * a.row + ea || -d >= (b.rows - 1) * b.row + eb) return false;
  int64_t left = 1 << 20;  // comparisons
  // rows j of b that reach over row i of a: lo < j b.row < hi; with equal strides they depend on j - i alone
  const bool same = a.row == b.row && a.row > 0;
  for (int64_t i = 0; i < (a.row && !same ? a.rows : 1); i++) {
    const int64_t lo = i * a.row - d - eb, hi = i * a.row - d + ea;
    int64_t j0 = same ? 1 - a.rows : 0, j1 = b.row ? b.rows - 1 : 0;
    if (b.row) {
      j0 = std::max(j0, floor_div(lo, b.row) + 1);
      j1 = std::min(j1, -floor_div(-hi, b.row) - 1);
    }
    for (int64_t j = j0; j <= j1; j++) {
      if ((left -= a.heads) < 0) return true;
      if (meet(a.heads, a.head, a.width, d + j * b.row - i * a.row, b.heads, b.head, b.width)) return true;
    }
    if (--left < 0) return true;
  }
  return false;
}

int kv8_check(const char* op, const ane_kv8_cache* c, const ane_kv8_batch* b, Kv8Batch* out) {
  if (!c || !b) return op_fail(ANE_ERR_ARG, "storiesane %s: no cache or batch", op);
  if (!c->k || !c->v || !c->k_exp || !c->v_exp) return op_fail(ANE_ERR_ARG, "storiesane %s: null cache buffer", op);
  if (!aligned16(c->k) || !aligned16(c->v))
    return op_fail(ANE_ERR_ARG, "storiesane %s: k and v must be 16-byte aligned", op);
  const int P = c->page_tokens;
  if (P < 16 || P > 256 || (P & (P - 1)))
    return op_fail(ANE_ERR_ARG, "storiesane %s: page_tokens=%d must be 16, 32, 64, 128 or 256", op, P);
  if (c->head_dim != 64 && c->head_dim != 128)
    return op_fail(ANE_ERR_ARG, "storiesane %s: head_dim=%d must be 64 or 128", op, c->head_dim);
  if (c->pages < 1 || c->kv_heads < 1 || c->kv_heads > 1024)
    return op_fail(ANE_ERR_ARG, "storiesane %s: pages=%d kv_heads=%d (pages at least 1, kv_heads 1..1024)", op,
                   c->pages, c->kv_heads);
  if (b->nseq < 0 || b->nseq > 65536 || b->rows < 0 || b->rows > (1 << 30))
    return op_fail(ANE_ERR_ARG, "storiesane %s: nseq=%d want 0..65536, rows=%d want 0..%d", op, b->nseq, b->rows,
                   1 << 30);
  if (b->nseq > 0 && (!b->table || !b->start || !b->offsets))
    return op_fail(ANE_ERR_ARG, "storiesane %s: null batch buffer", op);
  if (b->table_pages < 1 || b->table_stride < b->table_pages || (int64_t)b->table_pages * P > (1 << 30))
    return op_fail(ANE_ERR_ARG, "storiesane %s: table_pages=%d (at least 1, at most its stride %d and %d tokens)", op,
                   b->table_pages, b->table_stride, 1 << 30);
  if (b->max_len < 0 || b->max_new < 0)
    return op_fail(ANE_ERR_ARG, "storiesane %s: max_len=%d max_new=%d", op, b->max_len, b->max_new);
  int n = 0;
  while ((1 << n) < P) n++;
  *out = Kv8Batch{b->table, b->start, b->offsets, b->table_stride, b->table_pages, b->nseq, b->rows,
                  c->pages, n, c->kv_heads};
  return ANE_OK;
}

}  // namespace ane

using namespace ane;

extern "C" int ane_kv8_append(const ane_kv8_cache* cache, const ane_kv8_batch* batch, const ane_kv8_append_args* args,
                              void* stream) {
  return kv8_append(cache, batch, args, nullptr, stream);
}

int ane::kv8_append_check(const char* op, const ane_kv8_cache* cache, const ane_kv8_batch* batch,
                          const ane_kv8_append_args* args, const Kv8Sums* from, Kv8AppendArgs* into) {
  Kv8AppendArgs& a = *into;
  int rc = kv8_check(op, cache, batch, &a.b);
  if (rc) return rc;
  if (!args) return op_fail(ANE_ERR_ARG, "storiesane %s: null arguments", op);
  if (a.b.nseq == 0 || a.b.rows == 0) return ANE_OK;  // an empty tensor may have no address
  if (from && (cache->head_dim != 64 || a.b.rows > kDecRows || from->splits < 1 || from->n % 8 ||
               from->n < (args->heads + 2 * a.b.NKV) * 64))
    return op_fail(ANE_ERR_ARG, "storiesane %s: head_dim=%d rows=%d splits=%d n=%d of sums", op, cache->head_dim,
                   a.b.rows, from->splits, from->n);
  if ((!from && (!args->k || !args->v)) || !args->cos || !args->sin || args->heads < 0 ||
      (args->heads > 0 && ((!from && !args->q) || !args->q_out)))
    return op_fail(ANE_ERR_ARG, "storiesane %s: null buffer", op);
  const ane_kv8_append_args& g = *args;
  const int64_t strides[] = {g.k_row, g.k_head, g.v_row, g.v_head, g.q_row, g.q_head, g.q_out_row, g.q_out_head};
  for (int j = 0; j < (g.heads > 0 ? 8 : 4); j++)
    if (strides[j] < 0 || strides[j] % 8)
      return op_fail(ANE_ERR_ARG, "storiesane %s: stride %lld must be a multiple of 8", op, (long long)strides[j]);
  if (!aligned16(g.k) || !aligned16(g.v) || !aligned16(g.cos) || !aligned16(g.sin) ||
      (g.heads > 0 && (!aligned16(g.q) || !aligned16(g.q_out))))
    return op_fail(ANE_ERR_ARG, "storiesane %s: buffers must be 16-byte aligned", op);
  if (g.heads > 32768) return op_fail(ANE_ERR_ARG, "storiesane %s: heads=%d", op, g.heads);
  if (g.positions < a.b.table_pages << a.b.pshift)
    return op_fail(ANE_ERR_ARG, "storiesane %s: positions=%d must cover the table's %d", op, g.positions,
                   a.b.table_pages << a.b.pshift);
  if (g.heads > 0 && !kv8_apart(a.b.rows, g.q_out_row, g.heads, g.q_out_head, cache->head_dim))
    return op_fail(ANE_ERR_ARG, "storiesane %s: rows of q_out overlap", op);
  if (g.heads > 0 && g.q == g.q_out && (g.q_row != g.q_out_row || g.q_head != g.q_out_head))
    return op_fail(ANE_ERR_ARG, "storiesane %s: q_out is q with other strides", op);
  if (g.heads > 0 && !from) {
    const Extent out = fp16_rows(g.q_out, a.b.rows, g.q_out_row, g.heads, g.q_out_head, cache->head_dim);
    if ((g.q != g.q_out && share_memory(out, fp16_rows(g.q, a.b.rows, g.q_row, g.heads, g.q_head, cache->head_dim))) ||
        share_memory(out, fp16_rows(g.k, a.b.rows, g.k_row, a.b.NKV, g.k_head, cache->head_dim)) ||
        share_memory(out, fp16_rows(g.v, a.b.rows, g.v_row, a.b.NKV, g.v_head, cache->head_dim)))
      return op_fail(ANE_ERR_ARG, "storiesane %s: q_out overlaps q, k or v", op);
  }
  a.k = (uint8_t*)cache->k; a.v = (uint8_t*)cache->v; a.k_exp = cache->k_exp; a.v_exp = cache->v_exp;
  a.xq = (const half_t*)g.q; a.xk = (const half_t*)g.k; a.xv = (const half_t*)g.v; a.q_out = (half_t*)g.q_out;
  a.cos = g.cos; a.sin = g.sin;
  a.q_row = g.q_row; a.q_head = g.q_head; a.k_row = g.k_row; a.k_head = g.k_head; a.v_row = g.v_row;
  a.v_head = g.v_head; a.qo_row = g.q_out_row; a.qo_head = g.q_out_head;
  a.heads = g.heads;
  a.from = from ? *from : Kv8Sums{};
  a.by_row = 0;
  return ANE_OK;
}

int ane::kv8_append(const ane_kv8_cache* cache, const ane_kv8_batch* batch, const ane_kv8_append_args* args,
                    const Kv8Sums* from, void* stream) {
  const char* op = "kv8 append";
  Kv8AppendArgs a;
  const int rc = kv8_append_check(op, cache, batch, args, from, &a);
  if (rc || a.b.nseq == 0 || a.b.rows == 0) return rc;
  DeviceScope dev(cache->device);
  if (dev.status() != hipSuccess)
    return op_fail(ANE_ERR_HIP, "storiesane %s: device %d: %s", op, cache->device, hipGetErrorString(dev.status()));
  const int P = 1 << a.b.pshift;
  const uint32_t pages = kv8_count(a.b.nseq, a.b.rows, kv8_pages(P));
  const int each = batch->max_new ? std::min(batch->max_new, a.b.rows) : (a.b.rows + a.b.nseq - 1) / a.b.nseq;
  const hipStream_t st = (hipStream_t)stream;
  // A wave takes a page's new rows where they fit a pass of it (the longest
  // sequence's, or where that is not known the mean one's): 64 single tokens
  // 4.8 us against 5.9, 64 of 32 heads of 128 6.0 against 18, in pages of 256
  // 5.1 against 23; 64 sequences of 8 rows at head dimension 64 5.6 against
  // 6.1, but of 16 8.9 against 6.5, and of 8 at 128 9.4 against 7.7.
  const int per = 512 / cache->head_dim;  // rows of a pass, or query heads of a block
  if (from || each <= per) {
    a.by_row = (uint32_t)a.b.rows < pages;
    const dim3 grid(a.by_row ? a.b.rows : pages, a.b.NKV + (a.heads + per - 1) / per);
    if (from) hipLaunchKernelGGL((append_few_kernel<64, true>), grid, dim3(64), 0, st, a);
    else if (cache->head_dim == 64) hipLaunchKernelGGL((append_few_kernel<64, false>), grid, dim3(64), 0, st, a);
    else hipLaunchKernelGGL((append_few_kernel<128, false>), grid, dim3(64), 0, st, a);
  } else {
    const dim3 grid(pages, a.b.NKV + (a.heads + kQHeads - 1) / kQHeads);
    if (cache->head_dim == 64) launch<64>(a, grid, st);
    else launch<128>(a, grid, st);
  }
  const hipError_t h = hipGetLastError();
  if (h != hipSuccess) return op_fail(ANE_ERR_HIP, "storiesane %s: %s", op, hipGetErrorString(h));
  return ANE_OK;
}

extern "C" int ane_debug_share_memory(const int64_t* a, const int64_t* b) {
  return share_memory({(uintptr_t)a[0], a[1], a[2], a[3], a[4], a[5]}, {(uintptr_t)b[0], b[1], b[2], b[3], b[4], b[5]});
}

extern "C" int ane_debug_kv8_item(const ane_kv8_cache* cache, const ane_kv8_batch* batch, int32_t tile_tokens,
                                  int32_t pages, int64_t item, int32_t* out) {
  const char* op = "debug kv8 item";
  Kv8Batch b;
  int rc = kv8_check(op, cache, batch, &b);
  if (rc) return rc;
  if (!out || tile_tokens < 1 || tile_tokens > 64 || b.nseq < 1)
    return op_fail(ANE_ERR_ARG, "storiesane %s: tile_tokens=%d nseq=%d", op, tile_tokens, b.nseq);
  if (pages == 2 && b.nseq > 64)
    return op_fail(ANE_ERR_ARG, "storiesane %s: nseq=%d want at most 64", op, b.nseq);
  const bool tiles = pages == 0 || pages == 2;
  const Kv8Items items = tiles ? kv8_tiles(tile_tokens) : pages == 1 ? kv8_pages(1 << b.pshift) : kv8_tiles(1);
  const uint32_t n = kv8_count(b.nseq, b.rows, items);
  if (item < 0 || item >= (int64_t)n)
    return op_fail(ANE_ERR_ARG, "storiesane %s: item=%lld want below %u", op, (long long)item, n);
  const Kv8Span s = pages == 0   ? kv8_tile_span(b, tile_tokens, (uint32_t)item)
                    : pages == 1 ? kv8_page_span(b, (uint32_t)item)
                    : pages == 2 ? kv8_tile_longest(b, tile_tokens, (uint32_t)item)
                                 : kv8_row_page_span(b, (uint32_t)item);
  out[0] = s.seq;
  out[1] = s.row;
  out[2] = s.n;
  out[3] = s.pos;
  out[4] = !tiles && s.n > 0 ? kv8_page(b, s.seq, s.pos >> b.pshift) : -1;
  out[5] = (int)n;
  return ANE_OK;
}
