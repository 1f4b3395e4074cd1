// Writing keys and values into the 8-bit cache and reading them back.
//
// Per block of tokens and head, keys and values apart, in float32:
//   x' = x clamped to +-CACHE8_TOP;  need = the smallest power of two s >= 2^-15 with max |x'| of the call's tokens <= 448 s
//   s  = need if the block's first token is among them (the block begins anew), else the larger of need and the scale so far
//   c  = e4m3(x' / s), to nearest;  held value: c s, which fp16 and bf16 hold exactly
// and where s has grown, the codes of the block's other tokens are rounded once more, c = e4m3(c s_old / s): a move of the
// exponent, exact down to the smallest numbers.  A NaN anywhere in a token's key or value of a head is held as
// NaN in all of its key and as zeros in its value (cbk_cache8.h says why), and counts nothing for the scale.
//
// A block has one writer: a wavefront for each sixteen of its tokens, all of one workgroup, which agree on the largest
// magnitudes through LDS and keep the numbers in registers meanwhile.  Workgroups find their blocks by the rows of the call: a row
// begins one if it is its sequence's first or its token a block's first.  Small calls have a workgroup per row, those
// whose row begins none end at once; large ones have one per `block` rows and walk through what begins there.
//
// Both kernels only move data (2 B in and 1 B out per number, or the other way round) and are bound by the bytes: 28600 tokens of 8 heads of 128 channels, bf16,
// written in 35.6 us and read in 29.6 (4.9 and 5.9 TB/s; a large copy reaches 5.1); 32 single tokens, bound by a chain of look-ups (sequence, length, page, scale),
// in 4.4 and 4.8 us.
#include "cbk_cache_io.h"
#include "cbk_cache8.h"

namespace cbk {

typedef uint16_t v2s __attribute__((ext_vector_type(2)));

// Lanes of a wavefront over sixteen tokens: L lanes a token, CH channels each, TW quads of tokens at a time, Q of them one
// after the other; a lane has all four tokens of its quads.
template <int D>
struct Lanes8 {
  static constexpr int CH = D == 64 ? 4 : 8, L = D / CH, TW = 64 / L, Q = 4 / TW, W = CH / 4;
};

template <int CH>
struct Sixteens { uint32_t w[CH / 2]; };    // CH 16-bit numbers
template <int CH>
__device__ inline Sixteens<CH> load16(const void* p, int64_t i) {
  Sixteens<CH> x;
  if constexpr (CH == 8) {
    const v4u v = __builtin_nontemporal_load((const v4u*)((const uint16_t*)p + i));
    x.w[0] = v[0]; x.w[1] = v[1]; x.w[2] = v[2]; x.w[3] = v[3];
  } else {
    const v2u v = __builtin_nontemporal_load((const v2u*)((const uint16_t*)p + i));
    x.w[0] = v[0]; x.w[1] = v[1];
  }
  return x;
}
__device__ inline v2s magnitudes(uint32_t w) { return __builtin_bit_cast(v2s, w & 0x7fff7fffu); }
// The maxima over all lanes, without trips through LDS: neighbours, pairs, mirrored eights and sixteens, then quarters and halves
template <int CTRL>
__device__ inline v2s with_moved(v2s x) {
  const uint32_t y = __builtin_amdgcn_update_dpp(0, (int)__builtin_bit_cast(uint32_t, x), CTRL, 0xf, 0xf, false);
  return __builtin_elementwise_max(x, __builtin_bit_cast(v2s, y));
}
__device__ inline v2s across_lanes(v2s x) {
  x = with_moved<0xb1>(x);
  x = with_moved<0x4e>(x);
  x = with_moved<0x141>(x);
  x = with_moved<0x140>(x);
  uint32_t w = __builtin_bit_cast(uint32_t, x);
  const auto q = __builtin_amdgcn_permlane16_swap(w, w, false, false);
  x = __builtin_elementwise_max(__builtin_bit_cast(v2s, (uint32_t)q[0]), __builtin_bit_cast(v2s, (uint32_t)q[1]));
  w = __builtin_bit_cast(uint32_t, x);
  const auto h = __builtin_amdgcn_permlane32_swap(w, w, false, false);
  return __builtin_elementwise_max(__builtin_bit_cast(v2s, (uint32_t)h[0]), __builtin_bit_cast(v2s, (uint32_t)h[1]));
}
template <int DT>
__device__ inline float from16(uint16_t b) { return DT == CBK_F16 ? h2f(b) : bf2f(b); }

// Bytes of four dwords (a token's four channels each) by channel instead
__device__ inline void transpose4(uint32_t (&x)[4]) {
  const uint32_t a = __builtin_amdgcn_perm(x[1], x[0], 0x05010400u), b = __builtin_amdgcn_perm(x[1], x[0], 0x07030602u);
  const uint32_t c = __builtin_amdgcn_perm(x[3], x[2], 0x05010400u), d = __builtin_amdgcn_perm(x[3], x[2], 0x07030602u);
  x[0] = __builtin_amdgcn_perm(c, a, 0x05040100u);
  x[1] = __builtin_amdgcn_perm(c, a, 0x07060302u);
  x[2] = __builtin_amdgcn_perm(d, b, 0x05040100u);
  x[3] = __builtin_amdgcn_perm(d, b, 0x07060302u);
}

// The sequence that row t (the same in all lanes) belongs to or would: the last offset at or before it, found a 64th of the list a step
__device__ inline int sequence_of(const DRows& r, int t, int lane) {
  if (!r.starts) return t / r.per;
  int lo = 0;                                                       // the first offset that passes t is in [lo, lo + width]
  for (int width = r.seqs + 1; width > 0;) {
    const int step = (width + 63) / 64;
    const int64_t at = lo + (int64_t)(lane + 1) * step - 1;
    const uint64_t m = __ballot(at > r.seqs || r.starts[at] > t);
    lo += (m ? __ffsll((unsigned long long)m) - 1 : 64) * step;
    width = step - 1;
  }
  return min(lo, r.seqs + 1) - 1;
}

// What begins among rows [t, end): calls f(first row, rows, sequence, position of the first) for each run of one sequence's rows in
// one block of 2^shift tokens.  Uniform over the workgroup.
template <class F>
__device__ inline void runs_from(const DRows& r, int t, int end, int shift, int lane, bool may, F f) {
  // Up to 63 sequences: a lane has an offset and a length each, so that one load does not wait for the other (write and read, 16 sequences of 16 tokens 9.1 and
  // 9.8 -> 8.3 and 9.4 us, with the event; 16 of 4000 70.3 and 77.4 -> 68.0 and 76.7; a read of 87000 tokens of 16 heads 184 -> 189, so not there)
  const bool lanes = may && r.starts && r.seqs < 64;
  const int offset = lanes ? r.starts[min(lane, r.seqs)] : 0, length = lanes ? r.lens[min(lane, r.seqs - 1)] : 0;
  int b = lanes ? __popcll(__ballot(lane <= r.seqs && offset <= t)) - 1 : sequence_of(r, t, lane);
  while (t < end) {
    if (!r.starts) b = t / r.per;
    if (b >= r.seqs) return;
    const int at = max(b, 0);
    const Seq s = lanes ? seq_from(r, __builtin_amdgcn_readlane(offset, at), __builtin_amdgcn_readlane(offset, at + 1), __builtin_amdgcn_readlane(length, at))
                        : seq_of(r, at);
    if (b < 0 || t < s.first || t >= s.first + s.n) {               // in front of the first sequence, or behind this one
      if (r.starts && r.starts[b + 1] <= t) {                       // the next one's, or, where some are empty, a later one's
        ++b;
        if (b < r.seqs && r.starts[b + 1] <= t) b = max(b, sequence_of(r, t, lane));
      } else {
        ++t;
      }
      continue;
    }
    const int pos = s.pos0 + (t - s.first), in = pos & ((1 << shift) - 1), left = (1 << shift) - in;
    const int rows = min(left, s.first + s.n - t);
    if (t == s.first || in == 0) f(t, rows, b, pos);
    t += rows;
  }
}

template <int D, int DT, int NW>
__global__ __launch_bounds__(64 * (NW == 1 ? 4 : NW)) void cache8_write_kernel(DCache8 c, DRows r, CacheIo io, int chunk) {
  using T = Lanes8<D>;
  constexpr int CH = T::CH, Q = T::Q;
  __shared__ uint32_t top_sh[2][NW];
  const int lane = threadIdx.x & 63, e = lane % T::L, k = lane / T::L;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), part = NW == 1 ? 0 : wave;
  const int64_t item = NW == 1 ? (int64_t)blockIdx.x * 4 + wave : blockIdx.x;
  const int h = (int)(item % c.heads);
  const int64_t first = item / c.heads * chunk;
  if (first >= r.tokens) return;
  const Parts8 at(c, h, D);
  int turn = 0;
  runs_from(r, (int)first, min((int)first + chunk, r.tokens), c.block_shift, lane, true, [&](int t, int rows, int b, int pos) {
    const int from = pos & (16 * NW - 1);                           // the run is tokens [from, from + rows) of the block
    const uint32_t in = pos & (c.page - 1) & ~(16 * NW - 1);        // where the block begins in the page
    const bool anew = from == 0;
    // ---- the numbers, and the largest magnitudes
    Sixteens<CH> xk[Q][4], xv[Q][4];
    bool is[Q][4];
#pragma unroll
    for (int q = 0; q < Q; ++q)
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const int tok = 16 * part + 4 * (k + T::TW * q) + i;
        is[q][i] = tok >= from && tok < from + rows;
        xk[q][i] = xv[q][i] = Sixteens<CH>{};
        if (is[q][i]) {
          const int64_t row = t + (tok - from);
          xk[q][i] = load16<CH>(io.k, row * io.kt + h * io.kh + e * CH);
          xv[q][i] = load16<CH>(io.v, row * io.vt + h * io.vh + e * CH);
        }
      }
    const int page = pos < 0 ? -1 : page_of(c, r, b, pos);          // (looked up while the numbers are on their way)
    if (page < 0) return;                                           // (all of the run: a block is on one page)
    float2* const sc = c.sc + at.scale(page) + (in >> c.block_shift);
    const float2 was = *sc;
    v2s tk = {0, 0}, tv = {0, 0};
    uint32_t nan = 0;                                               // a bit a token
    constexpr uint16_t inf = DT == CBK_F16 ? 0x7c00 : 0x7f80;
#pragma unroll
    for (int q = 0; q < Q; ++q)
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        v2s mk = {0, 0}, mv = {0, 0};
#pragma unroll
        for (int j = 0; j < CH / 2; ++j) {
          mk = __builtin_elementwise_max(mk, magnitudes(xk[q][i].w[j]));
          mv = __builtin_elementwise_max(mv, magnitudes(xv[q][i].w[j]));
        }
        const v2s m = __builtin_elementwise_max(mk, mv);
        if (m.x > inf || m.y > inf) nan |= 1u << (4 * q + i);
        tk = __builtin_elementwise_max(tk, mk);
        tv = __builtin_elementwise_max(tv, mv);
      }
    if (__ballot(nan != 0)) {                                       // rare: tokens with a NaN out of the maxima, and marked in all their lanes
#pragma unroll
      for (int o = 1; o < T::L; o *= 2) nan |= __shfl_xor(nan, o);
      tk = tv = v2s{0, 0};
#pragma unroll
      for (int q = 0; q < Q; ++q)
#pragma unroll
        for (int i = 0; i < 4; ++i)
          if (!(nan >> (4 * q + i) & 1)) {
#pragma unroll
            for (int j = 0; j < CH / 2; ++j) {
              tk = __builtin_elementwise_max(tk, magnitudes(xk[q][i].w[j]));
              tv = __builtin_elementwise_max(tv, magnitudes(xv[q][i].w[j]));
            }
          }
    }
    v2s top = {tk.x > tk.y ? tk.x : tk.y, tv.x > tv.y ? tv.x : tv.y};
    top = across_lanes(top);
    if constexpr (NW > 1) {                                         // (two places in turn: a wavefront may be a run ahead)
      if (lane == 0) top_sh[turn][part] = __builtin_bit_cast(uint32_t, top);
      __syncthreads();
#pragma unroll
      for (int i = 0; i < NW; ++i) top = __builtin_elementwise_max(top, __builtin_bit_cast(v2s, top_sh[turn][i]));
      turn ^= 1;
    }
    // ---- scales
    const float nk = scale8(fminf(from16<DT>(top.x), CACHE8_TOP)), nv = scale8(fminf(from16<DT>(top.y), CACHE8_TOP));
    const float sk = anew ? nk : fmaxf(nk, was.x), sv = anew ? nv : fmaxf(nv, was.y);
    const bool grown_k = !anew && sk != was.x, grown_v = !anew && sv != was.y;
    const float rk = reciprocal8(sk), rv = reciprocal8(sv), fk = was.x * rk, fv = was.y * rv;
    if (part == 0 && lane == 0) *sc = make_float2(sk, sv);
    // ---- codes
    const uint64_t code = at.code(page);
#pragma unroll
    for (int q = 0; q < Q; ++q) {
      const int quad = 4 * part + k + T::TW * q;                    // of the block's tokens
      uint32_t* const vp = (uint32_t*)(c.vc + code + (uint32_t)((in + 4 * quad) * D + e * CH * 4));
      uint32_t vw[T::W][4];                                         // by token, then by channel
      uint32_t mine = 0;                                            // bytes of the quad's tokens that are written
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const bool bad = nan >> (4 * q + i) & 1;
        uint32_t* const kp = (uint32_t*)(c.kc + code + (uint32_t)((in + 4 * quad + i) * D + e * CH));
        uint32_t kw[T::W];
        if (__ballot(is[q][i]) == 0 && !grown_k) {                  // (single tokens: three of four)
#pragma unroll
          for (int w = 0; w < T::W; ++w) vw[w][i] = 0;
          continue;
        }
#pragma unroll
        for (int w = 0; w < T::W; ++w) {
          float x[4], y[4];
#pragma unroll
          for (int j = 0; j < 4; ++j) {
            const uint32_t a = xk[q][i].w[2 * w + j / 2], b = xv[q][i].w[2 * w + j / 2];
            x[j] = __builtin_amdgcn_fmed3f(from16<DT>((uint16_t)(j & 1 ? a >> 16 : a)), -CACHE8_TOP, CACHE8_TOP) * rk;
            y[j] = __builtin_amdgcn_fmed3f(from16<DT>((uint16_t)(j & 1 ? b >> 16 : b)), -CACHE8_TOP, CACHE8_TOP) * rv;
          }
          kw[w] = bad ? 0x7f7f7f7fu : codes8(x[0], x[1], x[2], x[3]);
          vw[w][i] = bad ? 0u : codes8(y[0], y[1], y[2], y[3]);
        }
        if (is[q][i]) {
          mine |= 0xffu << (8 * i);
        } else if (grown_k) {
#pragma unroll
          for (int w = 0; w < T::W; ++w) kw[w] = rescaled8(kp[w], fk);
        }
        if (is[q][i] || grown_k) {
          if constexpr (T::W == 2) *(v2u*)kp = v2u{kw[0], kw[1]};
          else *kp = kw[0];
        }
      }
      if (!mine && !grown_v) continue;
#pragma unroll
      for (int w = 0; w < T::W; ++w) {
        transpose4(vw[w]);
        v4u o = {vw[w][0], vw[w][1], vw[w][2], vw[w][3]};
        if (mine != 0xffffffffu) {                                  // the quad's other tokens stay, or follow the scale
          const v4u old = *(const v4u*)(vp + 4 * w);
#pragma unroll
          for (int j = 0; j < 4; ++j) o[j] = (o[j] & mine) | ((grown_v ? rescaled8(old[j], fv) : old[j]) & ~mine);
        }
        *(v4u*)(vp + 4 * w) = o;
      }
    }
  });
}

// Rows that no page holds read as zero; rows in front of the first sequence and behind the last stay as they were.
template <int D, int DT>
__global__ __launch_bounds__(256) void cache8_read_kernel(DCache8 c, DRows r, CacheIo io, int chunk) {
  using T = Lanes8<D>;
  constexpr int CH = T::CH, Q = T::Q;
  const int lane = threadIdx.x & 63, e = lane % T::L, k = lane / T::L;
  const int64_t item = (int64_t)blockIdx.x * 4 + __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int h = (int)(item % c.heads);
  const int64_t first = item / c.heads * chunk;
  if (first >= r.tokens) return;
  const Parts8 at(c, h, D);
  const bool few = (int64_t)r.tokens * c.heads < (int64_t)chunk << 15;   // wavefronts
  runs_from(r, (int)first, min((int)first + chunk, r.tokens), 4, lane, few, [&](int t, int rows, int b, int pos) {
    const int page = pos < 0 ? -1 : page_of(c, r, b, pos), from = pos & 15;
    const uint32_t in = pos & (c.page - 1) & ~15;
    const uint64_t code = page < 0 ? 0 : at.code(page);
    const float2 s = page < 0 ? make_float2(0.f, 0.f) : scales8(c, at.scale(page), in);
#pragma unroll
    for (int q = 0; q < Q; ++q) {
      const int quad = k + T::TW * q;
      uint32_t kw[4][T::W], vw[T::W][4];
#pragma unroll
      for (int w = 0; w < T::W; ++w)
#pragma unroll
        for (int i = 0; i < 4; ++i) kw[i][w] = vw[w][i] = 0;
      if (page >= 0 && 4 * quad < from + rows && 4 * quad + 4 > from) {
        const uint32_t* const vp = (const uint32_t*)(c.vc + code + (uint32_t)((in + 4 * quad) * D + e * CH * 4));
#pragma unroll
        for (int w = 0; w < T::W; ++w) {
          const v4u x = *(const v4u*)(vp + 4 * w);
#pragma unroll
          for (int j = 0; j < 4; ++j) vw[w][j] = x[j];
        }
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const uint32_t* const kp = (const uint32_t*)(c.kc + code + (uint32_t)((in + 4 * quad + i) * D + e * CH));
#pragma unroll
          for (int w = 0; w < T::W; ++w) kw[i][w] = kp[w];
        }
      }
#pragma unroll
      for (int w = 0; w < T::W; ++w) transpose4(vw[w]);             // (its own inverse)
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const int tok = 4 * quad + i;
        if (tok < from || tok >= from + rows) continue;
        const int64_t row = t + (tok - from);
        float x[CH], y[CH];
#pragma unroll
        for (int w = 0; w < T::W; ++w) {
          float a[4], v[4];
          floats8(kw[i][w], a);
          floats8(vw[w][i], v);
#pragma unroll
          for (int j = 0; j < 4; ++j) {
            x[4 * w + j] = a[j] * s.x;
            y[4 * w + j] = a[j] != a[j] ? a[j] : v[j] * s.y;
          }
        }
        auto put = [&](void* p, int64_t i, const float (&x)[CH]) {
          if constexpr (CH == 8) {
            store8<DT>(p, i, x);
          } else if constexpr (DT == CBK_F32) {
            *(float4*)((float*)p + i) = make_float4(x[0], x[1], x[2], x[3]);
          } else {
            v2u o;
#pragma unroll
            for (int j = 0; j < 2; ++j)
              o[j] = DT == CBK_F16 ? (uint32_t)f2h(x[2 * j]) | (uint32_t)f2h(x[2 * j + 1]) << 16
                                   : (uint32_t)f2bf(x[2 * j]) | (uint32_t)f2bf(x[2 * j + 1]) << 16;
            __builtin_nontemporal_store(o, (v2u*)((uint16_t*)p + i));
          }
        };
        put(io.k, row * io.kt + h * io.kh + e * CH, x);
        put(io.v, row * io.vt + h * io.vh + e * CH, y);
      }
    }
  });
}

// Rows a wavefront (or, in wide blocks, a workgroup) walks through: as many as leave 2048 wavefronts, but no more than a sequence has on average, or a block.
// Those that begin no block end at once, and cost their start; blocks that one wavefront meets one behind the other cost their loads each.  Write, read, 8
// heads of 128 channels, blocks of 16, us: 512 sequences' 4 tokens a row a wavefront 28 and 26, so 11.6 and 12.4, their single tokens 10.2 and 8.9 (16 rows
// a wavefront 52 and 42); a prompt of 16384 tokens a row a wavefront 173 and 160, 16 rows 24 and 27; 16 sequences' 48 tokens 14.7, so 9.6, 16 rows 8.4;
// 64 sequences' 8 tokens 11.6, so 9.6, 16 rows 17.6; 10 of 49 tokens in blocks of 256 28 with 256 rows a workgroup, so 9.8.  Not helped by it: few rows into
// wide blocks, a wavefront for each sixteen of which is started (256 sequences' 12 rows in blocks of 256, 128, 64 and 16: written in 34, 18, 11 and 6.5, read in 7).
static int chunk_of(const DCache8& c, const DRows& r, int block) {
  const int64_t waves = (int64_t)r.tokens * c.heads * (block / 16);
  if (waves >= (int64_t)1 << 25) return block;                      // (a launch has fewer than 2^32 threads)
  const int64_t each = r.seqs ? r.tokens / r.seqs : 1, most = each < block ? each : block, fit = (waves + 2047) / 2048;
  const int64_t n = fit < most ? fit : most;
  return n < 1 ? 1 : (int)n;
}

template <int D, int DT, int NW>
static void write3(const DCache8& c, const DRows& r, const CacheIo& io, hipStream_t st) {
  const int chunk = chunk_of(c, r, 16 * NW);
  const int64_t items = ((int64_t)r.tokens + chunk - 1) / chunk * c.heads;
  hipLaunchKernelGGL((cache8_write_kernel<D, DT, NW>), dim3((unsigned)(NW == 1 ? (items + 3) / 4 : items)), dim3(64 * (NW == 1 ? 4 : NW)), 0, st,
                     c, r, io, chunk);
}
template <int D, int DT>
static void write2(const DCache8& c, const DRows& r, const CacheIo& io, hipStream_t st) {
  switch (c.block_shift) {
    case 4: return write3<D, DT, 1>(c, r, io, st);
    case 5: return write3<D, DT, 2>(c, r, io, st);
    case 6: return write3<D, DT, 4>(c, r, io, st);
    case 7: return write3<D, DT, 8>(c, r, io, st);
    default: return write3<D, DT, 16>(c, r, io, st);
  }
}
template <int D>
static void write1(const DCache8& c, const DRows& r, const CacheIo& io, int dt, hipStream_t st) {
  if (dt == CBK_F16) write2<D, CBK_F16>(c, r, io, st);
  else write2<D, CBK_BF16T>(c, r, io, st);
}
int launch_cache8_write(const DCache8& c, const DRows& r, const CacheIo& io, int dt, hipStream_t st) {
  if (c.dim == 64) write1<64>(c, r, io, dt, st);
  else if (c.dim == 128) write1<128>(c, r, io, dt, st);
  else write1<256>(c, r, io, dt, st);
  return hipGetLastError() == hipSuccess ? CBK_OK : CBK_ERR_HIP;
}

template <int D, int DT>
static void read2(const DCache8& c, const DRows& r, const CacheIo& io, hipStream_t st) {
  const int chunk = chunk_of(c, r, 16);
  const int64_t items = ((int64_t)r.tokens + chunk - 1) / chunk * c.heads;
  hipLaunchKernelGGL((cache8_read_kernel<D, DT>), dim3((unsigned)((items + 3) / 4)), dim3(256), 0, st, c, r, io, chunk);
}
template <int D>
static void read1(const DCache8& c, const DRows& r, const CacheIo& io, int dt, hipStream_t st) {
  if (dt == CBK_F32) read2<D, CBK_F32>(c, r, io, st);
  else if (dt == CBK_F16) read2<D, CBK_F16>(c, r, io, st);
  else read2<D, CBK_BF16T>(c, r, io, st);
}
int launch_cache8_read(const DCache8& c, const DRows& r, const CacheIo& io, int dt, hipStream_t st) {
  if (c.dim == 64) read1<64>(c, r, io, dt, st);
  else if (c.dim == 128) read1<128>(c, r, io, dt, st);
  else read1<256>(c, r, io, dt, st);
  return hipGetLastError() == hipSuccess ? CBK_OK : CBK_ERR_HIP;
}

}  // namespace cbk
