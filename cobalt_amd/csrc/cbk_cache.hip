// Writing keys and values into the 4-bit cache and reading them back.
//
// Per token, head and group of G channels, in float32:
//   x' = x clamped to +-CACHE_TOP;  m = fp16(min x');  s = fp16((max x' - m) * fp32(1/15))
//   c  = clamp(rint((x' - m) / s), 0, 15), 0 where s = 0;   held value: m + c s
// A NaN anywhere in a token's key or value of a head is held as a NaN in the minimum of all its key groups, and the value
// as zeros: a row of attention that sees the token gets a NaN score, and a row that does not multiplies a
// masked 0 with finite values.
//
// Both kernels only move data (2 B in, 0.5 + 4/G B out per number, or the other way round); D/8 lanes take a token's
// head, eight channels each: 16-byte loads of the dense side, one dword of codes.
#include "cbk_cache.h"

namespace cbk {

// The sequence row t belongs to, -1: none.  `lane` holds one of 64 offsets a turn; every lane of the wavefront takes part.
template <int TW>
__device__ inline void seqs_of(const DRows& r, const int (&t)[TW], int lane, int (&b)[TW]) {
#pragma unroll
  for (int i = 0; i < TW; ++i) b[i] = 0;
  if (!r.starts) {
#pragma unroll
    for (int i = 0; i < TW; ++i) b[i] = t[i] < r.tokens ? t[i] / r.per : -1;
    return;
  }
  for (int j = 0; j < r.seqs + 1; j += 64) {
    const int s = j + lane <= r.seqs ? r.starts[j + lane] : 0x7fffffff;
#pragma unroll
    for (int i = 0; i < TW; ++i) b[i] += __popcll(__ballot(s <= t[i]));
  }
#pragma unroll
  for (int i = 0; i < TW; ++i) {
    b[i] -= 1;                              // offsets at or before t, less one
    if (b[i] >= r.seqs) b[i] = -1;
  }
}

// Where a token of a head is held: its block and its place in the page; block -1: nowhere
__device__ inline int64_t place_of(const DCache& c, const DRows& r, int b, int t, int h, int& at) {
  at = 0;
  if (b < 0) return -1;
  const Seq s = seq_of(r, b);
  const int i = t - s.first;
  if (i < 0 || i >= s.n) return -1;
  const int pos = s.pos0 + i;
  if (pos < 0 || pos >= s.held) return -1;
  const int64_t p = page_of(c, r, b, pos);
  at = pos & (c.page - 1);
  return p < 0 ? -1 : p * c.heads + h;
}

template <int N> __device__ inline float group_min(float x) {
#pragma unroll
  for (int o = 1; o < N; o *= 2) x = fminf(x, __shfl_xor(x, o));
  return x;
}
template <int N> __device__ inline float group_max(float x) {
#pragma unroll
  for (int o = 1; o < N; o *= 2) x = fmaxf(x, __shfl_xor(x, o));
  return x;
}

// A float32 result that is rounded again: without the barrier the compiler takes one instruction that rounds the exact value to fp16.
__device__ inline float as_float32(float x) {
  asm("" : "+v"(x));
  return x;
}

template <int DT>
__device__ inline void unpack8(const v4u q, float (&x)[8]) {
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const uint16_t lo = (uint16_t)(q[i] & 0xffffu), hi = (uint16_t)(q[i] >> 16);
    x[2 * i] = DT == CBK_F16 ? h2f(lo) : bf2f(lo);
    x[2 * i + 1] = DT == CBK_F16 ? h2f(hi) : bf2f(hi);
  }
}

// Codes (one dword) and scale | minimum of eight channels whose group is GL lanes wide.  The quotient is the
// correctly rounded one: the product with the rounded reciprocal, corrected by its exact remainder.
template <int GL>
__device__ inline uint32_t quantise(const float (&x)[8], uint32_t& meta) {
  float lo = x[0], hi = x[0];
#pragma unroll
  for (int i = 1; i < 8; ++i) { lo = fminf(lo, x[i]); hi = fmaxf(hi, x[i]); }
  lo = group_min<GL>(lo);
  hi = group_max<GL>(hi);
  const uint16_t mb = f2h(lo);
  const float m = h2f(mb);
  const uint16_t sb = f2h(as_float32((hi - m) * (1.f / 15.f)));
  const float s = h2f(sb);
  meta = (uint32_t)sb | (uint32_t)mb << 16;
  const float r = s > 0.f ? 1.f / s : 0.f;
  uint32_t w = 0;
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    const float d = x[i] - m, q0 = d * r, q = fmaf(fmaf(-q0, s, d), r, q0);
    const uint32_t c = (uint32_t)fminf(fmaxf(rintf(q), 0.f), 15.f);
    w |= c << (4 * (i / 2 + 4 * (i & 1)));
  }
  return w;
}

template <int D, int GL, int DT>
__global__ __launch_bounds__(256) void cache_write_kernel(DCache c, DRows r, CacheIo io) {
  constexpr int L = D / 8, TW = 64 / L;                             // lanes a token's head, tokens a wavefront
  const int lane = threadIdx.x & 63, e = lane % L, k = lane / L;
  const int64_t wave = (int64_t)blockIdx.x * 4 + (threadIdx.x >> 6);
  const int h = (int)(wave % c.heads);
  const int64_t t0 = wave / c.heads * TW;
  if (t0 >= r.tokens) return;
  int t[TW], b[TW];
#pragma unroll
  for (int i = 0; i < TW; ++i) t[i] = (int)t0 + i;                  // (tokens stay below 2^30)
  seqs_of<TW>(r, t, lane, b);
  int bk = b[0];
#pragma unroll
  for (int i = 1; i < TW; ++i) bk = k == i ? b[i] : bk;
  const int tk = (int)t0 + k;
  int at;
  const int64_t blk = place_of(c, r, bk, tk, h, at);
  v4u qk = {}, qv = {};
  if (blk >= 0) {
    qk = *(const v4u*)((const uint16_t*)io.k + tk * io.kt + h * io.kh + e * 8);
    qv = *(const v4u*)((const uint16_t*)io.v + tk * io.vt + h * io.vh + e * 8);
  }
  float xk[8], xv[8];
  unpack8<DT>(qk, xk);
  unpack8<DT>(qv, xv);
  float nan = 0.f;
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    nan = (xk[i] != xk[i] || xv[i] != xv[i]) ? 1.f : nan;
    xk[i] = fminf(fmaxf(xk[i], -CACHE_TOP), CACHE_TOP);
    xv[i] = fminf(fmaxf(xv[i], -CACHE_TOP), CACHE_TOP);
  }
  const bool bad = group_max<L>(nan) > 0.f;
  uint32_t mk, mv, wk = quantise<GL>(xk, mk), wv = quantise<GL>(xv, mv);
  if (bad) { wk = wv = mv = 0; mk = 0x7e000000u; }
  if (blk < 0) return;
  const int64_t bytes = (int64_t)c.page * (D / 2);
  *(uint32_t*)(c.kc + blk * bytes + at * (D / 2) + key_dword<D>(e) * 4) = wk;
  *(uint32_t*)(c.vc + blk * bytes + (at >> 2) * (2 * D) + e * 16 + (at & 3) * 4) = wv;
  if (e % GL == 0) {
    const int64_t i = blk * ((int64_t)c.page * (D / (8 * GL))) + (e / GL) * c.page + at;
    c.km[i] = mk;
    c.vm[i] = mv;
  }
}

template <int DT>
__device__ inline void store8(void* p, int64_t i, const float (&x)[8]) {
  if (DT == CBK_F32) {
    *(float4*)((float*)p + i) = make_float4(x[0], x[1], x[2], x[3]);
    *(float4*)((float*)p + i + 4) = make_float4(x[4], x[5], x[6], x[7]);
  } else {
    v4u o;
#pragma unroll
    for (int j = 0; j < 4; ++j)
      o[j] = DT == CBK_F16 ? (uint32_t)f2h(as_float32(x[2 * j])) | (uint32_t)f2h(as_float32(x[2 * j + 1])) << 16
                           : (uint32_t)f2bf(x[2 * j]) | (uint32_t)f2bf(x[2 * j + 1]) << 16;
    *(v4u*)((uint16_t*)p + i) = o;
  }
}

__device__ inline void values_of(uint32_t w, uint32_t meta, bool nan, float (&x)[8]) {
  const float s = h2f((uint16_t)(meta & 0xffffu)), m = nan ? __builtin_nanf("") : h2f((uint16_t)(meta >> 16));
#pragma unroll
  for (int i = 0; i < 8; ++i) x[i] = fmaf((float)((w >> (4 * (i / 2 + 4 * (i & 1)))) & 15u), s, m);
}

// Rows that no page holds read as zero; rows behind the last sequence stay as they were.
template <int D, int DT>
__global__ __launch_bounds__(256) void cache_read_kernel(DCache c, DRows r, CacheIo io) {
  constexpr int L = D / 8, TW = 64 / L;
  const int lane = threadIdx.x & 63, e = lane % L, k = lane / L;
  const int64_t wave = (int64_t)blockIdx.x * 4 + (threadIdx.x >> 6);
  const int h = (int)(wave % c.heads);
  const int64_t t0 = wave / c.heads * TW;
  if (t0 >= r.tokens) return;
  int t[TW], b[TW];
#pragma unroll
  for (int i = 0; i < TW; ++i) t[i] = (int)t0 + i;
  seqs_of<TW>(r, t, lane, b);
  int bk = b[0];
#pragma unroll
  for (int i = 1; i < TW; ++i) bk = k == i ? b[i] : bk;
  const int tk = (int)t0 + k;
  if (bk < 0 || tk >= r.tokens) return;
  int at;
  const int64_t blk = place_of(c, r, bk, tk, h, at);
  uint32_t wk = 0, wv = 0, mk = 0, mv = 0;
  if (blk >= 0) {
    const int64_t bytes = (int64_t)c.page * (D / 2), i = blk * ((int64_t)c.page * c.groups) + (e * 8 / c.group) * c.page + at;
    wk = *(const uint32_t*)(c.kc + blk * bytes + at * (D / 2) + key_dword<D>(e) * 4);
    wv = *(const uint32_t*)(c.vc + blk * bytes + (at >> 2) * (2 * D) + e * 16 + (at & 3) * 4);
    mk = c.km[i];
    mv = c.vm[i];
  }
  const bool nan = (mk >> 16 & 0x7fffu) > 0x7c00u;
  float x[8];
  values_of(wk, mk, nan, x);
  store8<DT>(io.k, tk * io.kt + h * io.kh + e * 8, x);
  values_of(wv, mv, nan, x);
  store8<DT>(io.v, tk * io.vt + h * io.vh + e * 8, x);
}

static dim3 io_grid(const DCache& c, const DRows& r) {
  const int tw = 512 / c.dim;
  return dim3((unsigned)((((int64_t)r.tokens + tw - 1) / tw * c.heads + 3) / 4));
}

template <int D, int GL>
static void write2(const DCache& c, const DRows& r, const CacheIo& io, int dt, hipStream_t st) {
  if (dt == CBK_F16) hipLaunchKernelGGL((cache_write_kernel<D, GL, CBK_F16>), io_grid(c, r), dim3(256), 0, st, c, r, io);
  else hipLaunchKernelGGL((cache_write_kernel<D, GL, CBK_BF16T>), io_grid(c, r), dim3(256), 0, st, c, r, io);
}
template <int D>
static void write1(const DCache& c, const DRows& r, const CacheIo& io, int dt, hipStream_t st) {
  if (c.group == 32) write2<D, 4>(c, r, io, dt, st);
  else if (c.group == 64) write2<D, 8>(c, r, io, dt, st);
  else if constexpr (D >= 128) write2<D, 16>(c, r, io, dt, st);
}
int launch_cache_write(const DCache& c, const DRows& r, const CacheIo& io, int dt, hipStream_t st) {
  if (c.dim == 64) write1<64>(c, r, io, dt, st);
  else if (c.dim == 128) write1<128>(c, r, io, dt, st);
  else write1<256>(c, r, io, dt, st);
  return hipGetLastError() == hipSuccess ? CBK_OK : CBK_ERR_HIP;
}

template <int D>
static void read1(const DCache& c, const DRows& r, const CacheIo& io, int dt, hipStream_t st) {
  if (dt == CBK_F32) hipLaunchKernelGGL((cache_read_kernel<D, CBK_F32>), io_grid(c, r), dim3(256), 0, st, c, r, io);
  else if (dt == CBK_F16) hipLaunchKernelGGL((cache_read_kernel<D, CBK_F16>), io_grid(c, r), dim3(256), 0, st, c, r, io);
  else hipLaunchKernelGGL((cache_read_kernel<D, CBK_BF16T>), io_grid(c, r), dim3(256), 0, st, c, r, io);
}
int launch_cache_read(const DCache& c, const DRows& r, const CacheIo& io, int dt, hipStream_t st) {
  if (c.dim == 64) read1<64>(c, r, io, dt, st);
  else if (c.dim == 128) read1<128>(c, r, io, dt, st);
  else read1<256>(c, r, io, dt, st);
  return hipGetLastError() == hipSuccess ? CBK_OK : CBK_ERR_HIP;
}

}  // namespace cbk
