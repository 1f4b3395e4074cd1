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
// head, eight channels each: 16-byte loads of the dense side, one dword of codes.  What a wavefront has to look up before it
// knows an address (sequence, length, page) takes longer than its move, so in large calls a lane takes U rows one after the other with
// all their loads under way.  Bound by the bytes: 65536 tokens of 8 heads of 128 channels, bf16, groups of 64, written in 83 us (344 MB, 4.1 TB/s) and read
// back in 63 us (5.4); small calls by the launch (4 us).  The dense side goes past the caches, which the codes' halves of a line need.
#include "cbk_cache_io.h"

namespace cbk {

// U rows of a lane (t0 + k, t0 + TW + k, ...): the sequence of each, -1 for none, the page that holds its token, -1: none, and its place there
template <int U, int TW>
__device__ inline void places_of(const DCache& c, const DRows& r, int t0, int k, int lane, int (&b)[U], int (&page)[U], int (&at)[U]) {
  const int b0 = seq_at(r, t0, lane);
  Seq s{0, 0, 0, 0};
  const int bb = min(max(b0, 0), r.seqs - 1);
  s = seq_of(r, bb);
  const bool one = b0 >= 0 && b0 < r.seqs && t0 + U * TW <= s.first + s.n;     // all of the wavefront's rows are of one sequence
#pragma unroll
  for (int u = 0; u < U; ++u) {
    const int t = t0 + u * TW + k;
    b[u] = b0;
    Seq q = s;
    if (!one) {
      if (t >= r.tokens) {
        b[u] = -1;
      } else if (!r.starts) {
        b[u] = t / r.per;
      } else {
        while (b[u] < r.seqs && r.starts[b[u] + 1] <= t) ++b[u];    // (starts has seqs + 1 entries; -1: in front of the first)
        if (b[u] >= r.seqs) b[u] = -1;
      }
      q = seq_of(r, max(b[u], 0));
    }
    const int i = t - q.first, pos = q.pos0 + i;
    page[u] = -1;
    if (b[u] >= 0 && i >= 0 && i < q.n && pos >= 0 && pos < q.held) {
      const int e = r.table[(int64_t)b[u] * r.ld + (pos >> c.shift)];          // (held: within the table's columns)
      page[u] = e >= 0 && e < c.pages ? e : -1;
    }
    at[u] = pos & (c.page - 1);
  }
}

// Byte offsets of a page's part of head h
struct Blocks {
  uint32_t code_page, meta_page;
  uint64_t code_head, meta_head;
  __device__ Blocks(const DCache& c, int h, int dim)
      : code_page((uint32_t)c.heads * c.page * (dim / 2)), meta_page((uint32_t)c.heads * c.page * c.groups * 4),
        code_head((uint64_t)h * c.page * (dim / 2)), meta_head((uint64_t)h * c.page * c.groups * 4) {}
  __device__ uint64_t code(int page) const { return (uint64_t)(uint32_t)page * code_page + code_head; }
  __device__ uint64_t meta(int page) const { return (uint64_t)(uint32_t)page * meta_page + meta_head; }
};

// Codes (one dword) and scale | minimum of eight channels whose group is GL lanes wide.  The quotient (x - m) / s is the
// correctly rounded one: the product with a reciprocal that is good to a step or so, corrected by its exact remainder.  (What is left is
// off by 2^-46, and no quotient of a 24-bit by an 11-bit number lies that close to the middle between two floats.)
template <int GL>
__device__ inline uint32_t quantise(float (&x)[8], uint32_t& meta) {
#pragma unroll
  for (int i = 0; i < 8; ++i) x[i] = __builtin_amdgcn_fmed3f(x[i], -CACHE_TOP, CACHE_TOP);
  float lo = fminf(fminf(fminf(x[0], x[1]), fminf(x[2], x[3])), fminf(fminf(x[4], x[5]), fminf(x[6], x[7])));
  float hi = fmaxf(fmaxf(fmaxf(x[0], x[1]), fmaxf(x[2], x[3])), fmaxf(fmaxf(x[4], x[5]), fmaxf(x[6], x[7])));
  lo = over_lanes<GL>(lo, [](float a, float b) { return fminf(a, b); });
  hi = over_lanes<GL>(hi, [](float a, float b) { return fmaxf(a, b); });
  const uint16_t mb = f2h(lo);
  const float m = h2f(mb);
  const uint16_t sb = f2h(as_float32((hi - m) * (1.f / 15.f)));
  const float s = h2f(sb);
  meta = (uint32_t)sb | (uint32_t)mb << 16;
  float r = __builtin_amdgcn_rcpf(s);
  r = s > 0.f ? fmaf(fmaf(-s, r, 1.f), r, r) : 0.f;
  float even = 0.f, odd = 0.f;                                      // four codes each, as whole numbers below 2^16
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    const float d = x[i] - m, q0 = d * r, q = fmaf(fmaf(-q0, s, d), r, q0);
    const float code = rintf(__builtin_amdgcn_fmed3f(q, 0.f, 15.f)), place = (float)(1 << (4 * (i / 2)));
    if (i & 1) odd = fmaf(code, place, odd); else even = fmaf(code, place, even);
  }
  return (uint32_t)even | (uint32_t)odd << 16;
}

template <int D, int GL, int DT, int U>
__global__ __launch_bounds__(256, 8) void cache_write_kernel(DCache c, DRows r, CacheIo io) {
  constexpr int L = D / 8, TW = 64 / L;                             // lanes a token's head, tokens a wavefront at a time
  const int lane = threadIdx.x & 63, e = lane % L, k = lane / L;
  const int64_t wave = (int64_t)blockIdx.x * 4 + __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int h = (int)(wave % c.heads);
  const int64_t first = wave / c.heads * (TW * U);
  if (first >= r.tokens) return;
  const int t0 = (int)first;
  int b[U], at[U];
  int page[U];
  places_of<U, TW>(c, r, t0, k, lane, b, page, at);
  v4u qk[U], qv[U];
#pragma unroll
  for (int u = 0; u < U; ++u) {
    const int64_t t = t0 + u * TW + k;
    qk[u] = qv[u] = v4u{};
    if (page[u] >= 0) {
      qk[u] = __builtin_nontemporal_load((const v4u*)((const uint16_t*)io.k + t * io.kt + h * io.kh + e * 8));
      qv[u] = __builtin_nontemporal_load((const v4u*)((const uint16_t*)io.v + t * io.vt + h * io.vh + e * 8));
    }
  }
  const Blocks at_head(c, h, D);
#pragma unroll
  for (int u = 0; u < U; ++u) {
    float nan = any_nan<DT>(qk[u]) || any_nan<DT>(qv[u]) ? 1.f : 0.f;
    nan = over_lanes<(L < 16 ? L : 16)>(nan, [](float a, float b) { return fmaxf(a, b); });
    if (L > 16) nan = fmaxf(nan, __shfl_xor(nan, 16));
    float x[8];
    uint32_t mk, mv;
    unpack8<DT>(qk[u], x);
    uint32_t wk = quantise<GL>(x, mk);
    unpack8<DT>(qv[u], x);
    uint32_t wv = quantise<GL>(x, mv);
    if (nan > 0.f) { wk = wv = mv = 0; mk = 0x7e000000u; }
    if (page[u] >= 0) {
      const uint64_t code = at_head.code(page[u]), meta = at_head.meta(page[u]);
      *(uint32_t*)(c.kc + code + (uint32_t)(at[u] * (D / 2) + key_dword<D>(e) * 4)) = wk;
      *(uint32_t*)(c.vc + code + (uint32_t)((at[u] >> 2) * (2 * D) + e * 16 + (at[u] & 3) * 4)) = wv;
      if (e % GL == 0) {
        const uint32_t i = 4 * ((e / GL) * c.page + at[u]);
        *(uint32_t*)((uint8_t*)c.km + meta + i) = mk;
        *(uint32_t*)((uint8_t*)c.vm + meta + i) = mv;
      }
    }
  }
}

__device__ inline void values_of(uint32_t w, uint32_t meta, bool nan, float (&x)[8]) {
  const float s = h2f((uint16_t)(meta & 0xffffu)), m = nan ? __builtin_nanf("") : h2f((uint16_t)(meta >> 16));
#pragma unroll
  for (int i = 0; i < 8; ++i) x[i] = fmaf((float)((w >> (4 * (i / 2 + 4 * (i & 1)))) & 15u), s, m);
}

// Rows that no page holds read as zero; rows in front of the first sequence and behind the last stay as they were.
template <int D, int DT, int U>
__global__ __launch_bounds__(256) void cache_read_kernel(DCache c, DRows r, CacheIo io) {
  constexpr int L = D / 8, TW = 64 / L;
  const int lane = threadIdx.x & 63, e = lane % L, k = lane / L;
  const int64_t wave = (int64_t)blockIdx.x * 4 + __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int h = (int)(wave % c.heads);
  const int64_t first = wave / c.heads * (TW * U);
  if (first >= r.tokens) return;
  const int t0 = (int)first;
  int b[U], at[U];
  int page[U];
  places_of<U, TW>(c, r, t0, k, lane, b, page, at);
  uint32_t wk[U], wv[U], mk[U], mv[U];
  const Blocks at_head(c, h, D);
  const uint32_t group = (e * 8 / c.group) * c.page;
#pragma unroll
  for (int u = 0; u < U; ++u) {
    wk[u] = wv[u] = mk[u] = mv[u] = 0;
    if (page[u] >= 0) {
      const uint64_t code = at_head.code(page[u]), meta = at_head.meta(page[u]) + 4 * (group + at[u]);
      wk[u] = *(const uint32_t*)(c.kc + code + (uint32_t)(at[u] * (D / 2) + key_dword<D>(e) * 4));
      wv[u] = *(const uint32_t*)(c.vc + code + (uint32_t)((at[u] >> 2) * (2 * D) + e * 16 + (at[u] & 3) * 4));
      mk[u] = *(const uint32_t*)((const uint8_t*)c.km + meta);
      mv[u] = *(const uint32_t*)((const uint8_t*)c.vm + meta);
    }
  }
#pragma unroll
  for (int u = 0; u < U; ++u) {
    if (b[u] < 0) continue;
    const int64_t t = t0 + u * TW + k;
    const bool nan = (mk[u] >> 16 & 0x7fffu) > 0x7c00u;
    float x[8];
    values_of(wk[u], mk[u], nan, x);
    store8<DT>(io.k, t * io.kt + h * io.kh + e * 8, x);
    values_of(wv[u], mv[u], nan, x);
    store8<DT>(io.v, t * io.vt + h * io.vh + e * 8, x);
  }
}

// Rows a lane takes: four where wavefronts that take one would fill the chip more than four times over (65536 tokens of 8 heads of 128
// channels: written in 83 us, 93 with one row; read in 63, 71; 16384 tokens alike, 2048 tokens 4.9 with one row and 5.4, read 5.1 and 7.3)
constexpr int MANY = 4;                     // (to write: two, which a chip-wide call has enough wavefronts for)
static bool many_io(const DCache& c, const DRows& r) { return (int64_t)r.tokens * c.heads * c.dim >= (int64_t)MANY * 8192 * 512; }
static dim3 io_grid(const DCache& c, const DRows& r, int u) {
  const int tw = 512 / c.dim * u;
  return dim3((unsigned)((((int64_t)r.tokens + tw - 1) / tw * c.heads + 3) / 4));
}

template <int D, int GL, int DT>
static void write3(const DCache& c, const DRows& r, const CacheIo& io, hipStream_t st) {
  if (many_io(c, r)) hipLaunchKernelGGL((cache_write_kernel<D, GL, DT, 2>), io_grid(c, r, 2), dim3(256), 0, st, c, r, io);
  else hipLaunchKernelGGL((cache_write_kernel<D, GL, DT, 1>), io_grid(c, r, 1), dim3(256), 0, st, c, r, io);
}
template <int D, int GL>
static void write2(const DCache& c, const DRows& r, const CacheIo& io, int dt, hipStream_t st) {
  if (dt == CBK_F16) write3<D, GL, CBK_F16>(c, r, io, st);
  else write3<D, GL, CBK_BF16T>(c, r, io, st);
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

template <int D, int DT>
static void read2(const DCache& c, const DRows& r, const CacheIo& io, hipStream_t st) {
  if (many_io(c, r)) hipLaunchKernelGGL((cache_read_kernel<D, DT, MANY>), io_grid(c, r, MANY), dim3(256), 0, st, c, r, io);
  else hipLaunchKernelGGL((cache_read_kernel<D, DT, 1>), io_grid(c, r, 1), dim3(256), 0, st, c, r, io);
}
template <int D>
static void read1(const DCache& c, const DRows& r, const CacheIo& io, int dt, hipStream_t st) {
  if (dt == CBK_F32) read2<D, CBK_F32>(c, r, io, st);
  else if (dt == CBK_F16) read2<D, CBK_F16>(c, r, io, st);
  else read2<D, CBK_BF16T>(c, r, io, st);
}
int launch_cache_read(const DCache& c, const DRows& r, const CacheIo& io, int dt, hipStream_t st) {
  if (c.dim == 64) read1<64>(c, r, io, dt, st);
  else if (c.dim == 128) read1<128>(c, r, io, dt, st);
  else read1<256>(c, r, io, dt, st);
  return hipGetLastError() == hipSuccess ? CBK_OK : CBK_ERR_HIP;
}

}  // namespace cbk
