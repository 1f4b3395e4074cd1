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
// Scores are exact up to float32: the codes themselves are the operands, one product per group of channels, and its sum is
// multiplied by the token's scale; the minima, which are fp16 already, meet the sums of q over the groups in a product
// of their own.  (Keys rounded to fp16 put 5e-4 of error into an fp16 result, which itself rounds by 2e-4.)  Query rows are
// operands as they are (bf16 of ordinary size is exact in fp16), rows of very large or small numbers after division by a power of two.
// Values m + c s are rounded once to fp16 (2^-11).  p is kept at 2^7.5 times its size against the running maximum, so that what
// an fp16 cannot hold lies 2^-31 below the largest; for an fp16 result the rest p - fp16(p) is a second operand, for a
// bf16 one, whose own step is eight times as large, it is left out, and the sum adds the rounded p.
//
// The tokens of all sequences and heads are one list of units of 128 tokens, cut into equal pieces, one a workgroup;
// what a workgroup has of a head it does not finish goes to the workspace with its maximum and sum, and a second
// launch joins the pieces.  Lengths are read on the device: the host knows none of them.
//
// Bound by the bytes of the cache where histories are long (floor: a copy's 4.92 TB/s): 32 sequences of 8192 tokens, 128
// channels, groups of 64, bf16: 65 us, 4.6 TB/s; groups of 32 70 us, 4.8; 256 channels 62 us, 4.8, but with groups of 32 90 us, 3.7 (reads of eight
// groups' scales and queries from LDS); 64 channels 89 us, 3.4 (vector and scalar instructions a token, which do not halve with the
// channels).  126 k tokens in 32 ragged sequences: 42 + 5 us with the join; one sequence of 700 tokens 9 + 2.  About 8 us of a launch
// are the look-ups in front of the first load and the end of a tile.
#include "cbk_cache.h"
#include "cbk_cache_attn.h"

namespace cbk {

template <int D, int G>
struct Held {                               // a wavefront's 32 tokens: two sixteens
  uint32_t k[2][D / 32];
  uint32_t km[2][(D / G + 3) / 4];
  v4u v[2][D > 128 ? D / 128 : 1], vm[2][D > 128 ? D / 128 : 1];
};

template <int D, int G, bool BF>
__global__ __launch_bounds__(256, D == 256 ? 2 : D == 128 ? 3 : 4) void cache_attn_kernel(DCache c, DRows r, AttnArgs a) {
  constexpr int R = 16, KS = D / 32, GS = D / G, GU = (GS + 3) / 4, VU = D > 128 ? D / 128 : 1, TILES = D / 16;
  __shared__ float o_sh[4][R][D + 4];
  __shared__ float m_sh[4][R], l_sh[4][R];
  constexpr bool Q_LDS = G == 32 && D > 64;   // queries in LDS, not in registers, of which groups of 32 leave too few (32 sequences of 8192 tokens: 128 channels 80 -> 70 us, 256 channels 138 -> 90)
  __shared__ v8h q_sh[Q_LDS ? KS * 64 : 1];
  __shared__ v2u scale_sh[4][2][GS][4];       // a wavefront's own: scales of its 32 keys, by group, four in a piece
  const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int col = lane & 15, h4 = lane >> 4;

  // ---- this workgroup's piece of the list
  auto units = [&](int b) { return units_of(seq_of(r, b), a, c.heads, R); };
  const Index list(r.seqs, lane, units);
  const int64_t total = list.total, pieces = min((int64_t)gridDim.x, total);
  const int64_t w = blockIdx.x;
  AttnPiece* const desc = (AttnPiece*)a.ws + w;
  if (w >= pieces) {
    if (a.ws && tid == 0) desc->count = 0;
    return;
  }
  const Shares shares(total, pieces);
  const int64_t begin = shares.begin(w), end = shares.end(w);
  int64_t base;
  int b = list.find(begin, base, units);
  int64_t at = begin;
  int joined = 0;
  const Exponents ex = exponents();

  while (at < end) {
    // ---- one head's tile of rows and the units of it that are this workgroup's
    const Seq s = seq_of(r, b);
    const Range g = range_of(s, a);
    const int rows = s.n * a.ratio, tiles = (rows + R - 1) / R;
    const int weight = a.whole ? 1 : g.units + EXTRA;
    const int64_t all = (int64_t)tiles * c.heads * weight;
    if (at >= base + all) {
      base += all;
      if (++b == r.seqs) break;                                     // (there is a next one, unless lengths change under the call)
      continue;
    }
    const int64_t item = quotient(at - base, weight), start = base + item * weight;
    const int64_t until = min(end, start + weight);
    const int u0 = a.whole ? 0 : max((int)(at - start) - EXTRA, 0), u1 = a.whole ? g.units : (int)(until - start) - EXTRA;
    const bool is_first = at == begin;
    at = until;
    if (u1 <= u0) continue;                                         // nothing but what the tile counts for by itself
    const int h = (int)quotient(item, tiles), row0 = (int)(item - (int64_t)h * tiles) * R;
    const int valid = min(R, rows - row0);

    const int pos_lo = s.pos0 + row0 / a.ratio, pos_hi = s.pos0 + (row0 + valid - 1) / a.ratio;

    // where the cache head's part of page 0 is, and what a page takes; offsets of the lane from a sixteen's first token
    const uint32_t code_page = (uint32_t)c.heads * c.page * (D / 2), meta_page = (uint32_t)c.heads * c.page * (GS * 4);
    const int64_t code_head = (int64_t)h * c.page * (D / 2), meta_head = (int64_t)h * c.page * (GS * 4);
    const uint8_t *const kc = c.kc + code_head, *const vc = c.vc + code_head;
    const uint8_t *const km = (const uint8_t*)c.km + meta_head, *const vm = (const uint8_t*)c.vm + meta_head;
    const uint32_t k_at = col * (D / 2) + h4 * (D == 64 ? 8 : 16);
    const uint32_t v_at = h4 * (2 * D) + (D == 64 ? col & 7 : col) * 16;
    const uint32_t km_at = 4 * (min(h4, GS - 1) * c.page + col), vm_at = 4 * ((8 * (D == 64 ? col & 7 : col) / G) * c.page + 4 * h4);
    auto token_of = [&](int u) { return ((u < g.head ? u : u + g.skip) * 4 + wave) * 32; };
    // Pages of the two sixteens of a step.  Pages of 32 tokens and more hold both, so that one address serves them (2 to 4 % of the time at 64 and 128
    // channels)
    const bool one_page = c.page >= 32;
    auto pages_of = [&](int tok, int (&pg)[2]) {
      pg[0] = tok < s.held ? page_of(c, r, b, tok) : -1;
      pg[1] = one_page ? pg[0] : tok + 16 < s.held ? page_of(c, r, b, tok + 16) : -1;
    };
    Held<D, G> x;
    auto key_of = [&](int t, const uint8_t* kp, const uint8_t* mp) {
#pragma unroll
      for (int i = 0; i < GU; ++i) x.km[t][i] = *(const uint32_t*)(mp + (uint32_t)(i * 16) * c.page + km_at);
      if constexpr (D == 64) {
        const uint2 d = *(const uint2*)(kp + k_at);
        x.k[t][0] = d.x; x.k[t][1] = d.y;
      } else {
#pragma unroll
        for (int i = 0; i < VU; ++i) {
          const v4u d = *(const v4u*)(kp + 64 * i + k_at);
#pragma unroll
          for (int j = 0; j < 4; ++j) x.k[t][4 * i + j] = d[j];
        }
      }
    };
    auto value_of = [&](int t, const uint8_t* vp, const uint8_t* mp) {
#pragma unroll
      for (int i = 0; i < VU; ++i) {
        x.v[t][i] = *(const v4u*)(vp + 256 * i + v_at);
        x.vm[t][i] = *(const v4u*)(mp + (uint32_t)(i * (128 / G) * 4) * c.page + vm_at);
      }
    };
    auto fetch = [&](auto of, const uint8_t* codes, const uint8_t* metas, int tok, const int (&pg)[2]) {   // (a page that is not there: page 0, and masked)
      const uint32_t in = tok & (c.page - 1), page = max(pg[0], 0);
      const uint8_t *cp = codes + ((uint64_t)page * code_page + in * (D / 2)), *mp = metas + ((uint64_t)page * meta_page + in * 4);
      of(0, cp, mp);
      if (one_page) {
        of(1, cp + 16 * (D / 2), mp + 16 * 4);
      } else {
        const uint32_t in = (tok + 16) & (c.page - 1), page = max(pg[1], 0);
        of(1, codes + ((uint64_t)page * code_page + in * (D / 2)), metas + ((uint64_t)page * meta_page + in * 4));
      }
    };
    auto fetch_keys = [&](int tok, const int (&pg)[2]) { fetch(key_of, kc, km, tok, pg); };
    auto fetch_values = [&](int tok, const int (&pg)[2]) { fetch(value_of, vc, vm, tok, pg); };

    // keys of the next step are under way while this one's values are worked on, and the other way round
    int pg[2], pg_next[2];
    pages_of(token_of(u0), pg);
    fetch_keys(token_of(u0), pg);
    fetch_values(token_of(u0), pg);
    pages_of(token_of(min(u0 + 1, u1 - 1)), pg_next);

    // ---- queries: fragments, positions and factors
    v8h q[KS], qm;
    float cs;
    Sight sight;
    const int row = row0 + col;
    const bool is = col < valid;
    const int tok = is ? row / a.ratio : 0, hq = h * a.ratio + (is ? row % a.ratio : 0);
    sight = sight_of(s.pos0 + (is ? tok : (row0 + valid - 1) / a.ratio), s.held, a);
    const uint16_t* qp = (const uint16_t*)a.q + (int64_t)(s.first + tok) * a.qt + (int64_t)hq * a.qh;
    v4u raw[KS];
#pragma unroll
    for (int k = 0; k < KS; ++k) raw[k] = is ? *(const v4u*)(qp + 32 * k + 8 * h4) : v4u{};
    float top = 0.f, down;
#pragma unroll
    for (int k = 0; k < KS; ++k) top = bits_top(raw[k], BF, top);
    top = across_max(top);
    cs = a.scale * row_factor(top, down);
#pragma unroll
    for (int k = 0; k < KS; ++k)
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const uint32_t two = raw[k][i];
        const float x0 = BF ? __uint_as_float(two << 16) : h2f((uint16_t)two), x1 = BF ? __uint_as_float(two & 0xffff0000u) : h2f((uint16_t)(two >> 16));
        q[k][2 * i] = (_Float16)(x0 * down);
        q[k][2 * i + 1] = (_Float16)(x1 * down);
      }
    // sums of q over the groups: as two fp16 that meet the minima
#pragma unroll
    for (int i = 0; i < 8; ++i) qm[i] = (_Float16)0.f;
#pragma unroll
    for (int g = 0; g < GS; ++g) {
      float sum = 0.f;
#pragma unroll
      for (int k = g * (G / 32); k < (g + 1) * (G / 32); ++k)
#pragma unroll
        for (int i = 0; i < 8; ++i) sum += (float)q[k][i];
      sum = across_sum(sum);
      const _Float16 hi = (_Float16)sum;
      if (h4 == g % 4) { qm[2 * (g / 4)] = hi; qm[2 * (g / 4) + 1] = (_Float16)(sum - (float)hi); }
    }
    if constexpr (Q_LDS) {                                          // (the last item's are read: two barriers ago)
      if (wave == 0)
#pragma unroll
        for (int k = 0; k < KS; ++k) q_sh[k * 64 + lane] = q[k];
      __syncthreads();
    }
    cs = fminf(fmaxf(cs, 1e-30f), 0x1.fffffep127f);                 // (a smaller one has every score at 0, a larger one every difference past any weight; a masked one stays -inf)
    v4f o[TILES];
    float m, l;
    m = FLOOR; l = 0.f;
#pragma unroll
    for (int t = 0; t < TILES; ++t) o[t] = v4f{0.f, 0.f, 0.f, 0.f};

    for (int u = u0; u < u1; ++u) {
      const int tok = token_of(u), tok_next = token_of(min(u + 1, u1 - 1));
      if (tok >= s.held) break;                                     // (of the last unit: nothing follows)
      const bool p0 = pg[0] >= 0, p1 = pg[1] >= 0;
      // every row sees all 32 tokens, and all of them are there
      const bool whole = p0 && p1 && tok + 32 <= s.held && tok + 31 <= pos_lo &&
                         (a.window <= 0 || tok > pos_hi - a.window || tok + 32 <= a.sinks);
      v4f sc[2];
      uint16_t* const mine_sh = (uint16_t*)scale_sh[wave];
#pragma unroll
      for (int t = 0; t < 2; ++t)
#pragma unroll
        for (int i = 0; i < GU; ++i)
          if (4 * i + h4 < GS) mine_sh[(t * GS + 4 * i + h4) * 16 + col] = (uint16_t)x.km[t][i];
      __builtin_amdgcn_fence(__ATOMIC_RELEASE, "wavefront");
      __builtin_amdgcn_wave_barrier();
      __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "wavefront");
#pragma unroll
      for (int t = 0; t < 2; ++t) {
        v8h mins;
#pragma unroll
        for (int i = 0; i < 8; ++i) mins[i] = i < 2 * GU ? __builtin_bit_cast(v2h, x.km[t][i / 2 % GU]).y : (_Float16)0.f;
        sc[t] = __builtin_amdgcn_mfma_f32_16x16x32_f16(mins, qm, v4f{0.f, 0.f, 0.f, 0.f}, 0, 0, 0);
#pragma unroll
        for (int g = 0; g < GS; ++g) {
          v4f part;
          part = v4f{0.f, 0.f, 0.f, 0.f};
#pragma unroll
          for (int k = g * (G / 32); k < (g + 1) * (G / 32); ++k) {
            const v8h f = code_octet(x.k[t][k], ex);
            part = __builtin_amdgcn_mfma_f32_16x16x32_f16(f, Q_LDS ? q_sh[k * 64 + lane] : q[k], part, 0, 0, 0);
          }
          const v2u sm = scale_sh[wave][t][g][h4];
#pragma unroll
            for (int i = 0; i < 4; ++i) {
              const uint32_t two = sm[i >> 1];                      // (a bit cast of a vector's element reads its first)
              sc[t][i] = fmaf((float)__builtin_bit_cast(v2h, two)[i & 1], part[i], sc[t][i]);
            }
        }
        __builtin_amdgcn_sched_barrier(0);                          // (or the second sixteen's operands take registers early)
      }
      if (u + 1 < u1) fetch_keys(tok_next, pg_next);
      if (!whole) {
#pragma unroll
        for (int t = 0; t < 2; ++t)
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            const int key = tok + 16 * t + 4 * h4 + i;
            const bool there = key < s.held && (t ? p1 : p0);
            sc[t][i] = there && sees(sight, key) ? sc[t][i] : -__builtin_inff();
            if (!there)
#pragma unroll
              for (int v = 0; v < VU; ++v) x.vm[t][v][i] = 0;       // whatever stands there: its value is 0
          }
      }
      v8h p, rest;
      float e[8], top;
#pragma unroll
      for (int i = 0; i < 8; ++i) e[i] = rounded_product(sc[i >> 2][i & 3], cs);
      top = fmaxf(fmaxf(fmaxf(e[0], e[1]), fmaxf(e[2], e[3])), fmaxf(fmaxf(e[4], e[5]), fmaxf(e[6], e[7])));
      top = across_max(top);
      if (__ballot(top > m + P_SLACK)) {                       // the maximum follows when p would leave its range
        const float up = fmaxf(m, top), f = __builtin_amdgcn_exp2f(m - up);
        m = up;
        l *= f;
#pragma unroll
        for (int t = 0; t < TILES; ++t) o[t] *= f;
      }
      const float shift = P_BITS - m;
#pragma unroll
      for (int i = 0; i < 8; ++i) e[i] = __builtin_amdgcn_exp2f(e[i] + shift);
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const v2h ph = {(_Float16)e[2 * i], (_Float16)e[2 * i + 1]};
        l = __builtin_amdgcn_fdot2(ph, v2h{(_Float16)1.f, (_Float16)1.f}, l, false);
        p[2 * i] = ph.x; p[2 * i + 1] = ph.y;
        if constexpr (!BF) {
          const v2h pl = rest_of(ph, e[2 * i], e[2 * i + 1]);
          rest[2 * i] = pl.x; rest[2 * i + 1] = pl.y;
          l = __builtin_amdgcn_fdot2(pl, v2h{(_Float16)1.f, (_Float16)1.f}, l, false);
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
          __builtin_amdgcn_sched_barrier(0);
          uint32_t pr[4];
#pragma unroll
          for (int i = 0; i < 4; ++i)
            pr[i] = __builtin_amdgcn_perm(wd[i >> 1][2 * (i & 1) + 1], wd[i >> 1][2 * (i & 1)], 0x0c040c00u + by * 0x00010001u);
          v8h f;
#pragma unroll
          for (int i = 0; i < 4; ++i) { const v2h y = __builtin_elementwise_fma(codes_of<false>(pr[i], ex), s2[i], m2[i]); f[2 * i] = y.x; f[2 * i + 1] = y.y; }
          const int t0 = D == 64 ? by : 2 * by * VU + v;
          o[t0] = __builtin_amdgcn_mfma_f32_16x16x32_f16(f, p, o[t0], 0, 0, 0);
          if constexpr (!BF)
            o[t0] = __builtin_amdgcn_mfma_f32_16x16x32_f16(f, rest, o[t0], 0, 0, 0);
          if constexpr (D > 64) {
#pragma unroll
            for (int i = 0; i < 4; ++i) { const v2h y = __builtin_elementwise_fma(codes_of<true>(pr[i], ex), s2[i], m2[i]); f[2 * i] = y.x; f[2 * i + 1] = y.y; }
            o[t0 + VU] = __builtin_amdgcn_mfma_f32_16x16x32_f16(f, p, o[t0 + VU], 0, 0, 0);
            if constexpr (!BF)
              o[t0 + VU] = __builtin_amdgcn_mfma_f32_16x16x32_f16(f, rest, o[t0 + VU], 0, 0, 0);
          }
        }
      }
      if (u + 1 < u1) {
        fetch_values(tok_next, pg_next);
        pg[0] = pg_next[0]; pg[1] = pg_next[1];
        pages_of(token_of(min(u + 2, u1 - 1)), pg_next);
      }
    }

    // ---- the four wavefronts' parts together
    __syncthreads();                                                // (the reads of the last item)
    l = across_sum(l);
    if (h4 == 0) { m_sh[wave][col] = m; l_sh[wave][col] = l; }
#pragma unroll
    for (int t = 0; t < TILES; ++t)
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const int rw = 4 * h4 + i;                                // row of the tile: channel 8 n + that of the nibble
        const int nd = D == 64 ? rw & 7 : D == 128 ? rw : 16 * (t & 1) + rw;
        const int nib = D == 64 ? 2 * t + (rw >> 3) : D == 128 ? t : t >> 1;
        o_sh[wave][col][8 * nd + (nib < 4 ? 2 * nib : 2 * nib - 7)] = o[t][i];
      }
    __syncthreads();
    const bool direct = u0 == 0 && u1 == g.units;
    const int slot = is_first ? 0 : 1;
    if (!direct && u0 == 0 && tid == 0) {                           // this workgroup begins the tile: it is joined from here
      desc->first = s.first; desc->row0 = row0; desc->valid = valid; desc->head = h; desc->slot = slot;
      desc->count = (int)(shares.of(start + weight - 1) - w + 1);
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
  }
  if (a.ws && !joined && tid == 0) desc->count = 0;
}

// Every P-th part of a row from the p-th on: four channels of each, against the maximum so far.  U of them are loaded at a time, one behind the
// other they would each cost the way to memory (joins of 64 new tokens of 30000, 256 channels, 4 heads: 81 us, 4 at a time 44); none that is not there (the
// last one loaded in its place: 56, and the chunks below 18.9).
template <int D, int R, int P, int U>
__device__ inline void add_parts(const AttnArgs& a, int grid, int64_t w, const AttnPiece& e, int p, int row, int d, float& top, float& sum, float (&y)[4]) {
  for (int i0 = p; i0 < e.count; i0 += U * P) {
    float4 o[U];
    float2 ml[U];
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const int i = i0 + u * P;
      if (i < e.count) {
        const float* const x = attn_part<D>(a.ws, grid, ((w + i) * 2 + (i ? 0 : e.slot)) * R + row);
        o[u] = *(const float4*)(x + d);
        ml[u] = *(const float2*)(x + D);
      }
    }
#pragma unroll
    for (int u = 0; u < U; ++u)
      if (i0 + u * P < e.count) {
        const float up = fmaxf(top, ml[u].x), f = __builtin_amdgcn_exp2f(top - up), g = __builtin_amdgcn_exp2f(ml[u].x - up);
        top = up;
        sum = sum * f + ml[u].y * g;
        y[0] = y[0] * f + o[u].x * g; y[1] = y[1] * f + o[u].y * g; y[2] = y[2] * f + o[u].z * g; y[3] = y[3] * f + o[u].w * g;
      }
  }
}

// Rows of a tile that several workgroups have parts of.  Workgroup (x, y) takes row y of the tile that begins in workgroup x: D/4 threads a
// part, 4T/D parts side by side, there may be hundreds.  (x is turned by y: tiles often begin every so many workgroups, and workgroups go to
// the XCDs in turn.  512 rows in 16 parts each took one XCD 68 us.)  T: 256, or 1024 where tiles have 200 parts and more on average: one sequence of 120000
// tokens on one head of 256 channels, 8-bit cache, 35 against 57 us with the launch before it; four of 60000, 192 parts each, 37 against 33.
template <int D, int R, int T>
__global__ __launch_bounds__(T) void cache_attn_join_kernel(AttnArgs a, int grid) {
  constexpr int C = D / 4, P = T / C;
  __shared__ float sh[P][D + 4];
  const int64_t w = (blockIdx.x + blockIdx.y) % gridDim.x;
  const AttnPiece e = ((const AttnPiece*)a.ws)[w];
  const int tid = threadIdx.x, d = 4 * (tid % C), p = tid / C, row = blockIdx.y;
  if (e.count == 0 || row >= e.valid) return;
  float top = FLOOR, sum = 0.f, y[4] = {0.f, 0.f, 0.f, 0.f};
  add_parts<D, R, P, 4>(a, grid, w, e, p, row, d, top, sum, y);
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

// The same for tiles of 256 rows, most of them in two or three parts: a wavefront a row, 256/D parts side by side.
template <int D>
__global__ __launch_bounds__(256) void cache_prompt_join_kernel(AttnArgs a, int grid) {
  constexpr int C = D / 4, P = 64 / C, R = 256, SHARE = 16;
  const int64_t w = (blockIdx.x + blockIdx.y) % gridDim.x;
  const AttnPiece e = ((const AttnPiece*)a.ws)[w];
  if (e.count == 0) return;
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), d = 4 * (lane % C), p = lane / C;
  const int end = min(((int)blockIdx.y + 1) * SHARE, e.valid);
  for (int row = blockIdx.y * SHARE + wave; row < end; row += 4) {
    float top = FLOOR, sum = 0.f, y[4] = {0.f, 0.f, 0.f, 0.f};
    // One a thread where they all have room side by side: chunks of six sequences, 64 channels, 2 to 4 parts a tile, 16.0 against 17.2 us
    if (e.count <= P) add_parts<D, R, P, 1>(a, grid, w, e, p, row, d, top, sum, y);
    else add_parts<D, R, P, 4>(a, grid, w, e, p, row, d, top, sum, y);
#pragma unroll
    for (int by = C; by < 64; by *= 2) {
      const float up = fmaxf(top, __shfl_xor(top, by)), f = __builtin_amdgcn_exp2f(top - up);
      top = up;
      sum *= f;
      sum += __shfl_xor(sum, by);
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        y[j] *= f;
        y[j] += __shfl_xor(y[j], by);
      }
    }
    const int gr = e.row0 + row;
    if (p == 0) store_row4(a, e.first + gr / a.ratio, e.head * a.ratio + gr % a.ratio, d, y, sum);
  }
}

// ------------------------------------------------------------------ launch
// Every tile of 16 rows, at most; its units, if all sequences were as long as the table allows; the workgroups that run at once:
// four, three or two a CU, by the registers and the LDS they take.
struct Load { int64_t tiles, units; int chip; };
static Load load_of(const DCache& c, const DRows& r, int ratio) {
  return {((int64_t)r.tokens * ratio / 16 + r.seqs) * c.heads, r.cap > UNIT ? (r.cap + UNIT - 1) / UNIT : 1, 256 * (c.dim == 64 ? 4 : c.dim == 128 ? 3 : 2)};
}
struct AttnPlan { int grid; bool split; size_t bytes; };
static AttnPlan plan_attn(const DCache& c, const DRows& r, int ratio) {
  const Load w = load_of(c, r, ratio);
  AttnPlan p;
  // Tiles of few units stay in one piece, which saves the second launch: up to 4 units (300 tokens of one sequence 10.2 against 11.4 us,
  // 500 alike, 700 14.5 against 11.6), up to 8 where the tiles fill half the chip (64 sequences of 1000 tokens 24.4 against 32.5 us).
  p.split = w.units > 8 || (w.units > 4 && 2 * w.tiles < w.chip);
  const int64_t most = p.split ? w.tiles * (w.units + EXTRA) : w.tiles;
  p.grid = (int)(most < w.chip ? most : w.chip);
  p.bytes = p.split ? attn_bytes(p.grid, 16, c.dim) : 0;
  return p;
}
template <int D>
static void join1(const AttnArgs& a, int grid, int rows, bool wide, hipStream_t st) {
  if (rows == 16 && wide) hipLaunchKernelGGL((cache_attn_join_kernel<D, 16, 1024>), dim3(grid, 16), dim3(1024), 0, st, a, grid);
  else if (rows == 16) hipLaunchKernelGGL((cache_attn_join_kernel<D, 16, 256>), dim3(grid, 16), dim3(256), 0, st, a, grid);
  else if (rows == 32) hipLaunchKernelGGL((cache_attn_join_kernel<D, 32, 256>), dim3(grid, 32), dim3(256), 0, st, a, grid);
  else hipLaunchKernelGGL((cache_prompt_join_kernel<D>), dim3(grid, 16), dim3(256), 0, st, a, grid);
}
void launch_cache_join(int dim, const AttnArgs& a, int grid, int rows, hipStream_t st, bool wide) {
  if (dim == 64) join1<64>(a, grid, rows, wide, st);
  else if (dim == 128) join1<128>(a, grid, rows, wide, st);
  else join1<256>(a, grid, rows, wide, st);
}

// Which of the two kernels.  That of cbk_cache_prompt.hip takes tiles of 256 rows, filled or not, and wins from about 100 rows a sequence
// (128 channels, 8 cache heads, 16 sequences of 4096 tokens: 96 rows 85 against 89 us here, 256 rows 110 against 235; fp16 128 rows 146
// against 137, 256 rows 172 against 256), but only where there is work for the chip: it starts and joins more slowly (one sequence of 8192
// tokens: 256 rows 56 against 41 us here, 512 rows 59 against 66; of 1024 tokens: 1024 rows 56 against 23).
static bool many_rows(const DCache& c, const DRows& r, int ratio) {
  const int64_t rows = (int64_t)r.tokens * ratio;
  if (rows <= (int64_t)112 * r.seqs) return false;
  const Load w = load_of(c, r, ratio);
  return w.tiles * (w.units + EXTRA) > (int64_t)16 * w.chip;
}
size_t cache_attn_workspace(const DCache& c, const DRows& r, int ratio) {
  return many_rows(c, r, ratio) ? plan_prompt(c, r, ratio).bytes : plan_attn(c, r, ratio).bytes;
}

template <int D, int G>
static void attn2(const AttnPlan& p, const DCache& c, const DRows& r, const AttnArgs& a, hipStream_t st) {
  if (a.bf) hipLaunchKernelGGL((cache_attn_kernel<D, G, true>), dim3(p.grid), dim3(256), 0, st, c, r, a);
  else hipLaunchKernelGGL((cache_attn_kernel<D, G, false>), dim3(p.grid), dim3(256), 0, st, c, r, a);
}
template <int D>
static void attn1(const AttnPlan& p, const DCache& c, const DRows& r, const AttnArgs& a, hipStream_t st) {
  if (c.group == 32) attn2<D, 32>(p, c, r, a, st);
  else if (c.group == 64) attn2<D, 64>(p, c, r, a, st);
  else if constexpr (D > 64) attn2<D, 128>(p, c, r, a, st);
}
int launch_cache_attn(const DCache& c, const DRows& r, AttnArgs a, size_t ws_bytes, hipStream_t st) {
  const size_t need = cache_attn_workspace(c, r, a.ratio);
  if (need > ws_bytes || (need && !a.ws)) return CBK_ERR_WORKSPACE;
  if (!need) a.ws = nullptr;
  if (many_rows(c, r, a.ratio)) return launch_cache_prompt(plan_prompt(c, r, a.ratio), c, r, a, st);
  const AttnPlan p = plan_attn(c, r, a.ratio);
  a.whole = !p.split;
  if (c.dim == 64) attn1<64>(p, c, r, a, st);
  else if (c.dim == 128) attn1<128>(p, c, r, a, st);
  else attn1<256>(p, c, r, a, st);
  if (p.split) launch_cache_join(c.dim, a, p.grid, 16, st);
  return hipGetLastError() == hipSuccess ? CBK_OK : CBK_ERR_HIP;
}

}  // namespace cbk
