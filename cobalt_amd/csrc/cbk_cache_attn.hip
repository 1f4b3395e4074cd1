// Attention over the 4-bit cache for few rows a sequence: single tokens, drafts, the ends of prompts.
//
//   o_i = sum_j p_ij v_j / sum_j p_ij,  p_ij = 2^(c q_i . k_j - M_i),  c = scale log2 e
//
// over the tokens j that row i sees, in one pass with running M and sum (float32; the products of p and v are
// of 16 bits each, see below).  The rows of a sequence that read one cache head (its tokens times the query heads on
// that head) are the columns of the matrix instructions, 16 at a time: S^T = K Q^T and O^T = V^T P^T.  In both the
// cache is the left operand and comes straight out of the loads: a lane holds eight channels of one token's key, or one
// channel of eight tokens' values.  The sums of S^T lie in the lanes that P^T wants them in when the tokens of a
// step are numbered 4h + r of the first and of the second 16, so nothing passes through LDS until a wavefront has done
// its share.
//
// Operands are fp16: a key or value m + c s is rounded once (2^-11; its scale and minimum are fp16 already), a bf16
// query row is brought to [1, 2) by a power of two and is then exact, and p is kept at 2^8 times its size against the
// running maximum, so that what an fp16 cannot hold lies 2^-32 below the largest.  The sum adds the rounded p.
//
// The tokens of all sequences and heads are one list of units of 128 tokens, cut into equal pieces, one a workgroup;
// what a workgroup has of a head it does not finish goes to the workspace with its maximum and sum, and a second
// launch joins the pieces.  Lengths are read on the device: the host knows none of them.
#include "cbk_cache.h"
#include "cbk_cache_attn.h"

namespace cbk {

constexpr int UNIT = 128;                   // tokens: 32 a wavefront
constexpr float FLOOR = -3.0e38f;           // running maximum before the first token: below every score that is one
constexpr float P_BITS = 8.f, P_SLACK = 6.f;   // p = 2^(t - M + P_BITS) with t <= M + P_SLACK: at most 2^14

struct Range { int units, head, skip; };    // units of a sequence; the first `head` from token 0, the others `skip` units on
__device__ inline Range range_of(const Seq& s, const AttnArgs& a) {
  Range g{0, 0, 0};
  if (s.n <= 0) return g;
  const int all = max((s.held + UNIT - 1) / UNIT, 1);
  if (a.window > 0) {
    const int lo = min(max(s.pos0 - a.window + 1, 0) / UNIT, all - 1);
    g.head = min((a.sinks + UNIT - 1) / UNIT, lo);
    g.skip = lo - g.head;
  }
  g.units = all - g.skip;
  return g;
}

// Sequences are walked in 256 parts, one a thread: total units of all, and where unit `want` lies
struct Cursor { int b; int64_t base; };     // sequence and its first unit
struct Walk {
  int64_t sums[256];
};
__device__ inline int64_t units_of(const DRows& r, const AttnArgs& a, int heads, int b, int rows) {
  const Seq s = seq_of(r, b);
  const int64_t tiles = ((int64_t)s.n * a.ratio + rows - 1) / rows;
  return tiles * heads * range_of(s, a).units;
}

__device__ inline float across_max(float x) {                       // over the four quarters of the wavefront
  x = fmaxf(x, __shfl_xor(x, 16));
  return fmaxf(x, __shfl_xor(x, 32));
}
__device__ inline float across_sum(float x) {
  x += __shfl_xor(x, 16);
  return x + __shfl_xor(x, 32);
}

// A product that stays one when something is added to it: the largest score less the maximum is 0 only if both were
// rounded alike, and where scores pass 2^24 nothing else keeps p in range.
__device__ inline float rounded_product(float a, float b) {
#pragma clang fp contract(off)
  return a * b;
}

template <int D>
struct Held {                               // a wavefront's 32 tokens: two sixteens
  uint32_t k[2][D / 32];
  uint32_t km[2][D > 128 ? D / 128 : 1];
  v4u v[2][D > 128 ? D / 128 : 1], vm[2][D > 128 ? D / 128 : 1];
};

template <int D, int NT>
__global__ __launch_bounds__(256) void cache_attn_kernel(DCache c, DRows r, AttnArgs a) {
  constexpr int R = 16 * NT, KS = D / 32, VU = D > 128 ? D / 128 : 1, TILES = D / 16;
  __shared__ float o_sh[4][R][D + 4];
  __shared__ float m_sh[4][R], l_sh[4][R];
  __shared__ int64_t walk[256];
  __shared__ int64_t found[4];
  const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int col = lane & 15, h4 = lane >> 4;

  // ---- this workgroup's piece of the list
  const int per = (r.seqs + 255) / 256;
  int64_t mine = 0;
  for (int i = 0; i < per; ++i) {
    const int b = tid * per + i;
    if (b < r.seqs) mine += units_of(r, a, c.heads, b, R);
  }
  walk[tid] = mine;
  __syncthreads();
  for (int o = 1; o < 256; o *= 2) {
    const int64_t x = tid >= o ? walk[tid - o] : 0;
    __syncthreads();
    walk[tid] += x;
    __syncthreads();
  }
  const int64_t total = walk[255];
  const int64_t pieces = min((int64_t)gridDim.x, (total + a.least - 1) / a.least);
  const int64_t w = blockIdx.x;
  AttnPiece* const desc = (AttnPiece*)a.ws + w;
  if (w >= pieces) {
    if (a.ws && tid == 0) desc->count = 0;
    return;
  }
  const int64_t begin = w * total / pieces, end = (w + 1) * total / pieces;
  if (walk[tid] - mine <= begin && begin < walk[tid]) {             // one thread
    int b = tid * per;
    int64_t base = walk[tid] - mine;
    for (;; ++b) {
      const int64_t u = units_of(r, a, c.heads, b, R);
      if (begin < base + u) break;
      base += u;
    }
    found[0] = b; found[1] = base;
  }
  __syncthreads();
  int b = __builtin_amdgcn_readfirstlane((int)found[0]);
  int64_t base = found[1], at = begin;
  int joined = 0;

  while (at < end) {
    // ---- one head's tile of rows and the units of it that are this workgroup's
    const Seq s = seq_of(r, b);
    const Range g = range_of(s, a);
    const int rows = s.n * a.ratio, tiles = (rows + R - 1) / R;
    const int64_t all = (int64_t)tiles * c.heads * g.units;
    if (at >= base + all) { base += all; ++b; continue; }
    const int64_t item = (at - base) / g.units;
    const int u0 = (int)((at - base) - item * g.units);
    const int u1 = (int)min((int64_t)g.units, u0 + (end - at));
    const int h = (int)(item / tiles), row0 = (int)(item % tiles) * R;
    const int valid = min(R, rows - row0);

    // ---- queries: fragments, positions and factors
    v8h q[NT][KS];
    float cs[NT];
    int pos[NT];
#pragma unroll
    for (int n = 0; n < NT; ++n) {
      const int row = row0 + 16 * n + col;
      const bool is = 16 * n + col < valid;
      const int tok = is ? row / a.ratio : 0, hq = h * a.ratio + (is ? row % a.ratio : 0);
      pos[n] = s.pos0 + (is ? tok : (row0 + valid - 1) / a.ratio);
      const uint16_t* qp = (const uint16_t*)a.q + (int64_t)(s.first + tok) * a.qt + (int64_t)hq * a.qh;
      float x[KS][8], top = 0.f;
#pragma unroll
      for (int k = 0; k < KS; ++k) {
        const int d = D >= 128 ? 128 * (k / 4) + 32 * h4 + 8 * (k % 4) : 16 * h4 + 8 * k;
        const v4u v = is ? *(const v4u*)(qp + d) : v4u{};
        if (a.bf) {
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            x[k][2 * i] = __uint_as_float(v[i] << 16);
            x[k][2 * i + 1] = __uint_as_float(v[i] & 0xffff0000u);
            top = fmaxf(top, fmaxf(fabsf(x[k][2 * i]), fabsf(x[k][2 * i + 1])));
          }
        } else {
          q[n][k] = __builtin_bit_cast(v8h, v);
        }
      }
      cs[n] = a.scale;
      if (a.bf) {
        top = across_max(top);
        int e = 0;
        if (top > 0.f && top < __builtin_inff()) e = max((int)(__float_as_uint(top) >> 23), 1) - 127;
        const float down = __uint_as_float((uint32_t)(127 - min(e, 126)) << 23);   // 2^-e, e = 127: 2^-126 leaves [2, 4)
        cs[n] = a.scale * __uint_as_float((uint32_t)(min(e, 126) + 127) << 23);
#pragma unroll
        for (int k = 0; k < KS; ++k)
#pragma unroll
          for (int i = 0; i < 8; ++i) q[n][k][i] = (_Float16)(x[k][i] * down);
      }
      cs[n] = fmaxf(cs[n], 1e-30f);         // (a smaller one has every score at 0; a masked one stays -inf)
    }
    const int pos_lo = s.pos0 + row0 / a.ratio, pos_hi = s.pos0 + (row0 + valid - 1) / a.ratio;

    v4f o[NT][TILES];
    float m[NT], l[NT];
#pragma unroll
    for (int n = 0; n < NT; ++n) {
      m[n] = FLOOR; l[n] = 0.f;
#pragma unroll
      for (int t = 0; t < TILES; ++t) o[n][t] = v4f{0.f, 0.f, 0.f, 0.f};
    }

    const int64_t kblk = (int64_t)c.page * (D / 2), mblk = (int64_t)c.page * c.groups;
    auto token_of = [&](int u) { return ((u < g.head ? u : u + g.skip) * 4 + wave) * 32; };
    auto pages_of = [&](int tok, int64_t (&pg)[2]) {
#pragma unroll
      for (int t = 0; t < 2; ++t) pg[t] = tok + 16 * t < s.held ? page_of(c, r, b, tok + 16 * t) : -1;
    };
    auto fetch = [&](int tok, const int64_t (&pg)[2], Held<D>& x) {
#pragma unroll
      for (int t = 0; t < 2; ++t) {
        const int in = (tok + 16 * t) & (c.page - 1);
        const int64_t blk = max(pg[t], (int64_t)0) * c.heads + h;
        const uint8_t* kp = c.kc + blk * kblk + (in + col) * (D / 2);
        const uint8_t* vp = c.vc + blk * kblk + ((in >> 2) + h4) * (2 * D);
        const uint32_t* kmp = c.km + blk * mblk + in + col;
        const uint32_t* vmp = c.vm + blk * mblk + in + 4 * h4;
        if constexpr (D == 64) {
          const uint2 d = *(const uint2*)(kp + h4 * 8);
          x.k[t][0] = d.x; x.k[t][1] = d.y;
          x.km[t][0] = kmp[(16 * h4 / c.group) * c.page];
          const int n = col & 7;
          x.v[t][0] = *(const v4u*)(vp + n * 16);
          x.vm[t][0] = *(const v4u*)(vmp + (8 * n / c.group) * c.page);
        } else {
#pragma unroll
          for (int i = 0; i < VU; ++i) {
            const v4u d = *(const v4u*)(kp + 64 * i + h4 * 16);
#pragma unroll
            for (int j = 0; j < 4; ++j) x.k[t][4 * i + j] = d[j];
            x.km[t][i] = kmp[((128 * i + 32 * h4) / c.group) * c.page];
            const int n = col + 16 * i;
            x.v[t][i] = *(const v4u*)(vp + n * 16);
            x.vm[t][i] = *(const v4u*)(vmp + (8 * n / c.group) * c.page);
          }
        }
      }
    };

    Held<D> next;
    int64_t pg[2], pg_next[2];
    pages_of(token_of(u0), pg);
    fetch(token_of(u0), pg, next);
    pages_of(token_of(min(u0 + 1, u1 - 1)), pg_next);
    for (int u = u0; u < u1; ++u) {
      Held<D> x = next;
      const int tok = token_of(u);
      const bool p0 = pg[0] >= 0, p1 = pg[1] >= 0;
      if (u + 1 < u1) {
        pg[0] = pg_next[0]; pg[1] = pg_next[1];
        fetch(token_of(u + 1), pg, next);
        pages_of(token_of(min(u + 2, u1 - 1)), pg_next);
      }
      if (tok >= s.held) continue;
      // every row sees all 32 tokens, and all of them are there
      const bool whole = p0 && p1 && tok + 32 <= s.held && tok + 31 <= pos_lo &&
                         (a.window <= 0 || tok > pos_hi - a.window || tok + 32 <= a.sinks);
      v4f sc[NT][2];
#pragma unroll
      for (int t = 0; t < 2; ++t) {
#pragma unroll
        for (int n = 0; n < NT; ++n) sc[n][t] = v4f{0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int k = 0; k < KS; ++k) {
          const v8h f = key_octet(x.k[t][k], x.km[t][k / 4]);
#pragma unroll
          for (int n = 0; n < NT; ++n) sc[n][t] = __builtin_amdgcn_mfma_f32_16x16x32_f16(f, q[n][k], sc[n][t], 0, 0, 0);
        }
      }
      if (!whole) {
#pragma unroll
        for (int t = 0; t < 2; ++t)
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            const int key = tok + 16 * t + 4 * h4 + i;
            const bool there = key < s.held && (t ? p1 : p0);
#pragma unroll
            for (int n = 0; n < NT; ++n) {
              const bool seen = there && key <= pos[n] && (a.window <= 0 || key > pos[n] - a.window || key < a.sinks);
              sc[n][t][i] = seen ? sc[n][t][i] : -__builtin_inff();
            }
            if (!there)
#pragma unroll
              for (int v = 0; v < VU; ++v) x.vm[t][v][i] = 0;       // whatever stands there: its value is 0
          }
      }
      v8h p[NT];
#pragma unroll
      for (int n = 0; n < NT; ++n) {
        float e[8], top;
#pragma unroll
        for (int i = 0; i < 8; ++i) e[i] = rounded_product(sc[n][i >> 2][i & 3], cs[n]);
        top = fmaxf(fmaxf(fmaxf(e[0], e[1]), fmaxf(e[2], e[3])), fmaxf(fmaxf(e[4], e[5]), fmaxf(e[6], e[7])));
        top = across_max(top);
        if (__ballot(top > m[n] + P_SLACK)) {                       // the maximum follows when p would leave its range
          const float up = fmaxf(m[n], top), f = __builtin_amdgcn_exp2f(m[n] - up);
          m[n] = up;
          l[n] *= f;
#pragma unroll
          for (int t = 0; t < TILES; ++t) o[n][t] *= f;
        }
        const float shift = P_BITS - m[n];
#pragma unroll
        for (int i = 0; i < 8; ++i) e[i] = __builtin_amdgcn_exp2f(e[i] + shift);
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const v2h ph = {(_Float16)e[2 * i], (_Float16)e[2 * i + 1]};
          l[n] = __builtin_amdgcn_fdot2(ph, v2h{(_Float16)1.f, (_Float16)1.f}, l[n], false);
          p[n][2 * i] = ph.x; p[n][2 * i + 1] = ph.y;
        }
      }
#pragma unroll
      for (int v = 0; v < VU; ++v) {
        v2h s2[4], m2[4];
        uint32_t wd[2][4];
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const uint32_t lo = x.vm[i >> 1][v][2 * (i & 1)], hi = x.vm[i >> 1][v][2 * (i & 1) + 1];
          s2[i] = __builtin_bit_cast(v2h, __builtin_amdgcn_perm(hi, lo, 0x05040100u));
          m2[i] = __builtin_bit_cast(v2h, __builtin_amdgcn_perm(hi, lo, 0x07060302u));
        }
#pragma unroll
        for (int t = 0; t < 2; ++t)
#pragma unroll
          for (int i = 0; i < 4; ++i) wd[t][i] = D == 64 ? x.v[t][0][i] >> (4 * (col >> 3)) : x.v[t][v][i];
#pragma unroll
        for (int by = 0; by < 4; ++by) {
          uint32_t pr[4];
#pragma unroll
          for (int i = 0; i < 4; ++i)
            pr[i] = __builtin_amdgcn_perm(wd[i >> 1][2 * (i & 1) + 1], wd[i >> 1][2 * (i & 1)], 0x0c040c00u + by * 0x00010001u);
          v8h f;
#pragma unroll
          for (int i = 0; i < 4; ++i) { const v2h y = code_pair<false>(pr[i], s2[i], m2[i]); f[2 * i] = y.x; f[2 * i + 1] = y.y; }
          const int t0 = D == 64 ? by : 2 * by * VU + v;
#pragma unroll
          for (int n = 0; n < NT; ++n) o[n][t0] = __builtin_amdgcn_mfma_f32_16x16x32_f16(f, p[n], o[n][t0], 0, 0, 0);
          if constexpr (D > 64) {
#pragma unroll
            for (int i = 0; i < 4; ++i) { const v2h y = code_pair<true>(pr[i], s2[i], m2[i]); f[2 * i] = y.x; f[2 * i + 1] = y.y; }
#pragma unroll
            for (int n = 0; n < NT; ++n) o[n][t0 + VU] = __builtin_amdgcn_mfma_f32_16x16x32_f16(f, p[n], o[n][t0 + VU], 0, 0, 0);
          }
        }
      }
    }

    // ---- the four wavefronts' parts together
    __syncthreads();                                                // (the reads of the last item)
#pragma unroll
    for (int n = 0; n < NT; ++n) {
      l[n] = across_sum(l[n]);
      if (h4 == 0) { m_sh[wave][16 * n + col] = m[n]; l_sh[wave][16 * n + col] = l[n]; }
#pragma unroll
      for (int t = 0; t < TILES; ++t)
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const int rw = 4 * h4 + i;                                // row of the tile: channel 8 n + that of the nibble
          const int nd = D == 64 ? rw & 7 : D == 128 ? rw : 16 * (t & 1) + rw;
          const int nib = D == 64 ? 2 * t + (rw >> 3) : D == 128 ? t : t >> 1;
          o_sh[wave][16 * n + col][8 * nd + (nib < 4 ? 2 * nib : 2 * nib - 7)] = o[n][t][i];
        }
    }
    __syncthreads();
    const bool direct = u0 == 0 && u1 == g.units;
    const int slot = at == begin ? 0 : 1;
    if (!direct && u0 == 0 && tid == 0) {                           // this workgroup begins the tile: it is joined from here
      // the last piece with a unit of it: pieces are cut at floor(i total / pieces)
      const int64_t last = base + (item + 1) * g.units - 1;
      int64_t e = last * pieces / total;
      while (e + 1 < pieces && (e + 1) * total / pieces <= last) ++e;
      while (e > w && e * total / pieces > last) --e;
      desc->first = s.first; desc->row0 = row0; desc->valid = valid; desc->head = h; desc->slot = slot;
      desc->count = (int)(e - w + 1);
    }
    if (!direct && u0 == 0) joined = 1;
    for (int x = tid; x < valid * (D / 4); x += 256) {
      const int row = x / (D / 4), d = 4 * (x % (D / 4));
      float top = m_sh[0][row];
#pragma unroll
      for (int i = 1; i < 4; ++i) top = fmaxf(top, m_sh[i][row]);
      float sum = 0.f, y[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const float f = __builtin_amdgcn_exp2f(m_sh[i][row] - top);
        sum += f * l_sh[i][row];
#pragma unroll
        for (int j = 0; j < 4; ++j) y[j] += f * o_sh[i][row][d + j];
      }
      if (direct) {
        const int gr = row0 + row;
        store_row4(a, s.first + gr / a.ratio, h * a.ratio + gr % a.ratio, d, y, sum);
      } else {
        float* const part = attn_part<D>(a.ws, gridDim.x, (w * 2 + slot) * R + row);
        *(float4*)(part + d) = make_float4(y[0], y[1], y[2], y[3]);
        if (d == 0) { part[D] = top; part[D + 1] = sum; }
      }
    }
    at += u1 - u0;
  }
  if (a.ws && !joined && tid == 0) desc->count = 0;
}

// One row of a tile that several workgroups have parts of: 256 threads, D/4 of them a part, a part after another.
template <int D, int R>
__global__ __launch_bounds__(256) void cache_attn_join_kernel(AttnArgs a, int grid) {
  constexpr int C = D / 4, P = 256 / C;
  __shared__ float sh[P][D + 4];
  const int64_t w = blockIdx.x;
  const AttnPiece e = ((const AttnPiece*)a.ws)[w];
  const int row = blockIdx.y, tid = threadIdx.x, d = 4 * (tid % C), p = tid / C;
  if (e.count == 0 || row >= e.valid) return;
  float top = FLOOR, sum = 0.f, y[4] = {0.f, 0.f, 0.f, 0.f};
  for (int i = p; i < e.count; i += P) {
    const float* const part = attn_part<D>(a.ws, grid, ((w + i) * 2 + (i ? 0 : e.slot)) * R + row);
    const float4 o = *(const float4*)(part + d);
    const float mm = part[D], ll = part[D + 1], up = fmaxf(top, mm);
    const float f = __builtin_amdgcn_exp2f(top - up), g = __builtin_amdgcn_exp2f(mm - up);
    top = up;
    sum = sum * f + ll * g;
    y[0] = y[0] * f + o.x * g; y[1] = y[1] * f + o.y * g; y[2] = y[2] * f + o.z * g; y[3] = y[3] * f + o.w * g;
  }
  *(float4*)&sh[p][d] = make_float4(y[0], y[1], y[2], y[3]);
  if (d == 0) { sh[p][D] = top; sh[p][D + 1] = sum; }
  __syncthreads();
  if (p) return;
#pragma unroll
  for (int i = 0; i < P; ++i) top = fmaxf(top, sh[i][D]);
  sum = 0.f;
  y[0] = y[1] = y[2] = y[3] = 0.f;
#pragma unroll
  for (int i = 0; i < P; ++i) {
    const float f = __builtin_amdgcn_exp2f(sh[i][D] - top);
    sum += f * sh[i][D + 1];
#pragma unroll
    for (int j = 0; j < 4; ++j) y[j] += f * sh[i][d + j];
  }
  const int gr = e.row0 + row;
  store_row4(a, e.first + gr / a.ratio, e.head * a.ratio + gr % a.ratio, d, y, sum);
}

// ------------------------------------------------------------------ launch
struct AttnPlan { int grid, least, rows; bool split; size_t bytes; };
static AttnPlan plan_attn(const DCache& c, const DRows& r, int ratio) {
  AttnPlan p;
  p.rows = 16;
  p.least = 1;
  // every tile of rows in units, if all sequences were as long as the table allows
  const int64_t tiles = ((int64_t)r.tokens * ratio / p.rows + r.seqs) * c.heads, units = r.cap > UNIT ? (r.cap + UNIT - 1) / UNIT : 1;
  const int64_t most = tiles * units;
  p.grid = (int)(most < 1024 ? most : 1024);
  p.split = units > 1;
  p.bytes = p.split ? attn_bytes(p.grid, p.rows, c.dim) : 0;
  return p;
}
size_t cache_attn_workspace(const DCache& c, const DRows& r, int ratio) { return plan_attn(c, r, ratio).bytes; }

template <int D>
static void attn1(const AttnPlan& p, const DCache& c, const DRows& r, const AttnArgs& a, hipStream_t st) {
  hipLaunchKernelGGL((cache_attn_kernel<D, 1>), dim3(p.grid), dim3(256), 0, st, c, r, a);
  if (p.split) hipLaunchKernelGGL((cache_attn_join_kernel<D, 16>), dim3(p.grid, 16), dim3(256), 0, st, a, p.grid);
}
int launch_cache_attn(const DCache& c, const DRows& r, AttnArgs a, size_t ws_bytes, hipStream_t st) {
  const AttnPlan p = plan_attn(c, r, a.ratio);
  if (p.bytes > ws_bytes || (p.bytes && !a.ws)) return CBK_ERR_WORKSPACE;
  if (!p.bytes) a.ws = nullptr;
  a.least = p.split ? p.least : 1;
  if (c.dim == 64) attn1<64>(p, c, r, a, st);
  else if (c.dim == 128) attn1<128>(p, c, r, a, st);
  else attn1<256>(p, c, r, a, st);
  return hipGetLastError() == hipSuccess ? CBK_OK : CBK_ERR_HIP;
}

}  // namespace cbk
