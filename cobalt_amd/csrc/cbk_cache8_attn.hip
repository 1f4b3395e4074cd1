// Attention over the 8-bit cache for few rows a sequence: single tokens, drafts, the ends of prompts.
//
//   o_i = sum_j p_ij v_j / sum_j p_ij,  p_ij = 2^(c q_i . k_j - M_i),  c = scale log2 e
//
// over the tokens j that row i sees, in one pass with running M and sum (float32; the products of p and v are
// of 16 bits each, see below).  The rows of a sequence that read one cache head (its tokens times the query heads on
// that head) are the columns of the matrix instructions, 16 at a time: S^T = K Q^T and O^T = V^T P^T.  In both the
// cache is the left operand and comes straight out of the loads: a lane holds 16 channels a load of one token's key, or four
// channels of four tokens' values.  The sums of S^T lie in the lanes that P^T wants them in when the tokens of a
// step are numbered 4h + r of the first and of the second 16, so nothing passes through LDS until a wavefront has done
// its share.
//
// Held values are fp16 numbers, so keys and values are exact as operands: one instruction widens two codes and multiplies them
// with their block's scale.  fp16 query rows are operands as they are; bf16 ones are rounded once to fp16, those whose largest number is below
// 2^-6 or from 2^15 on divided by a power of two first: exact down to 2^-17 and off by 2^-25 at most below it, of rows that are divided 2^-39 of the
// largest.  Scores are exact up to float32 but for that.  p is kept at 2^7.5 times its size against the running
// maximum, so that what an fp16 cannot hold lies 2^-31 below the largest; for an fp16 result the rest p - fp16(p) is a second operand, for a
// bf16 one, whose own step is eight times as large, it is left out, and the sum adds the rounded p.
//
// The tokens of all sequences and heads are one list of units of 128 tokens, cut into equal pieces, one a workgroup;
// what a workgroup has of a head it does not finish goes to the workspace with its maximum and sum, and a second
// launch joins the pieces.  Lengths are read on the device: the host knows none of them.
//
// Bound by the bytes of the cache where histories are long: two sequences, 269000 tokens (552 MB), 101 us and the join 5.5, 5.5 TB/s in the kernel; 32
// sequences, 115000 tokens (236 MB), 49 and 4.8, of which some 7 are the chain of look-ups before the first load and the joins in LDS at the end.  One token over
// 700 of history 7.2 us and 2.8, all of it that chain and the launches.
#include "cbk_cache8.h"
#include "cbk_cache_attn.h"
#include "cbk_cache8_attn.h"

namespace cbk {

template <int D>
struct Held8 {                              // a wavefront's 32 tokens: two sixteens
  v4u k[2][D / 64], v[2][D / 64];
  float2 s[2];                              // scales of their keys and values
};

// Workgroups of R rows a tile that run at once on a CU, by the registers and the LDS they take
template <int D, int R>
constexpr int RESIDENT = R == 16 ? (D == 256 ? 2 : D == 128 ? 3 : 4) : D == 128 ? 2 : 3;

// R rows a tile: one or two sixteens of columns, which share what is widened
template <int D, int R, bool BF>
__global__ __launch_bounds__(256, (RESIDENT<D, R>)) void cache8_attn_kernel(DCache8 c, DRows r, AttnArgs a) {
  constexpr int NC = R / 16, KS = D / 32, VU = D / 64, TILES = D / 16;
  __shared__ float o_sh[4][R][D + 4];
  __shared__ float m_sh[4][R], l_sh[4][R];
  const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int col = lane & 15, h4 = lane >> 4;

  // ---- this workgroup's piece of the list
  const bool lanes = r.seqs <= 64;                                  // each lane has a sequence, which saves the loads below
  const Seq mine = lanes ? seq_of(r, min(lane, r.seqs - 1)) : Seq{};
  auto units = [&](int b) { return units_of(lanes ? mine : seq_of(r, b), a, c.heads, R); };
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
  Seq s = lanes ? of_lane(mine, b) : seq_of(r, b);
  int64_t at = begin;
  int joined = 0;

  while (at < end) {
    // ---- one head's tile of rows and the units of it that are this workgroup's
    const Range g = range_of(s, a);
    const int rows = s.n * a.ratio, tiles = (rows + R - 1) / R;
    const int weight = a.whole ? 1 : g.units + EXTRA;
    const int64_t all = (int64_t)tiles * c.heads * weight;
    if (at >= base + all) {
      base += all;
      if (++b == r.seqs) break;                                     // (there is a next one, unless lengths change under the call)
      s = seq_of(r, b);
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

    const Parts8 part(c, h, D);
    const uint32_t k_at = col * D + h4 * 16, v_at = h4 * (4 * D) + col * 16;   // of the lane, from a sixteen's first token
    auto token_of = [&](int u) { return ((u < g.head ? u : u + g.skip) * 4 + wave) * 32; };
    // Pages of the two sixteens of a step.  Pages of 32 tokens and more hold both
    const bool one_page = c.page >= 32;
    auto pages_of = [&](int tok, int (&pg)[2]) {
      pg[0] = tok < s.held ? page_of(c, r, b, tok) : -1;
      pg[1] = one_page ? pg[0] : tok + 16 < s.held ? page_of(c, r, b, tok + 16) : -1;
    };
    Held8<D> x;
    // (a page that is not there: page 0, and masked)
    auto fetch_keys = [&](int tok, const int (&pg)[2]) {
#pragma unroll
      for (int t = 0; t < 2; ++t) {
        const uint32_t in = (tok + 16 * t) & (c.page - 1);
        const int page = max(pg[t], 0);
        const uint8_t* const p = c.kc + (part.code(page) + in * D) + k_at;
        x.s[t].x = scales8(c, part.scale(page), in).x;
#pragma unroll
        for (int j = 0; j < VU; ++j) x.k[t][j] = *(const v4u*)(p + 64 * j);
      }
    };
    auto fetch_values = [&](int tok, const int (&pg)[2]) {
#pragma unroll
      for (int t = 0; t < 2; ++t) {
        const uint32_t in = (tok + 16 * t) & (c.page - 1);
        const int page = max(pg[t], 0);
        const uint8_t* const p = c.vc + (part.code(page) + in * D) + v_at;
        x.s[t].y = scales8(c, part.scale(page), in).y;
#pragma unroll
        for (int j = 0; j < VU; ++j) x.v[t][j] = *(const v4u*)(p + 256 * j);
      }
    };

    // keys of the next step are under way while this one's values are worked on, and the other way round
    int pg[2], pg_next[2];
    pages_of(token_of(u0), pg);
    // ---- queries: loaded while the pages are looked up, made ready while the first codes are on their way
    v8h q[NC][KS];
    float cs[NC];
    Sight sight[NC];
    v4u raw[NC][KS];
#pragma unroll
    for (int n = 0; n < NC; ++n) {
      const int row = row0 + 16 * n + col;
      const bool is = 16 * n + col < valid;
      const int tok = is ? row / a.ratio : 0, hq = h * a.ratio + (is ? row % a.ratio : 0);
      sight[n] = sight_of(s.pos0 + (is ? tok : (row0 + valid - 1) / a.ratio), s.held, a);
      const uint16_t* qp = (const uint16_t*)a.q + (int64_t)(s.first + tok) * a.qt + (int64_t)hq * a.qh;
#pragma unroll
      for (int k = 0; k < KS; ++k) raw[n][k] = is ? *(const v4u*)(qp + 64 * (k >> 1) + 16 * h4 + 8 * (k & 1)) : v4u{};
    }
    fetch_keys(token_of(u0), pg);
    fetch_values(token_of(u0), pg);
    pages_of(token_of(min(u0 + 1, u1 - 1)), pg_next);
#pragma unroll
    for (int n = 0; n < NC; ++n) {
      float top = 0.f, down;
#pragma unroll
      for (int k = 0; k < KS; ++k) top = bits_top(raw[n][k], BF, top);
      top = across_max(top);
      cs[n] = a.scale * row_factor8<BF>(top, down);
#pragma unroll
      for (int k = 0; k < KS; ++k)
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const uint32_t two = raw[n][k][i];
          const float x0 = BF ? __uint_as_float(two << 16) : h2f((uint16_t)two), x1 = BF ? __uint_as_float(two & 0xffff0000u) : h2f((uint16_t)(two >> 16));
          q[n][k][2 * i] = (_Float16)(x0 * down);
          q[n][k][2 * i + 1] = (_Float16)(x1 * down);
        }
      cs[n] = fminf(fmaxf(cs[n], 1e-30f), 0x1.fffffep127f);         // (a smaller one has every score at 0, a larger one every difference past any weight; a masked one stays -inf)
    }
    v4f o[NC][TILES];
    float m[NC], l[NC];
#pragma unroll
    for (int n = 0; n < NC; ++n) {
      m[n] = FLOOR; l[n] = 0.f;
#pragma unroll
      for (int t = 0; t < TILES; ++t) o[n][t] = v4f{0.f, 0.f, 0.f, 0.f};
    }

    for (int u = u0; u < u1; ++u) {
      const int tok = token_of(u), tok_next = token_of(min(u + 1, u1 - 1));
      if (tok >= s.held) break;                                     // (of the last unit: nothing follows)
      const bool p0 = pg[0] >= 0, p1 = pg[1] >= 0;
      // every row sees all 32 tokens, and all of them are there
      const bool whole = p0 && p1 && tok + 32 <= s.held && tok + 31 <= pos_lo &&
                         (a.window <= 0 || tok > pos_hi - a.window || tok + 32 <= a.sinks);
      v4f sc[NC][2];
#pragma unroll
      for (int t = 0; t < 2; ++t) {
#pragma unroll
        for (int n = 0; n < NC; ++n) sc[n][t] = v4f{0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int k = 0; k < KS; ++k) {
          const v4u w4 = x.k[t][k >> 1];
          const v8h f = octet8(w4[2 * (k & 1)], w4[2 * (k & 1) + 1], x.s[t].x, x.s[t].x);
#pragma unroll
          for (int n = 0; n < NC; ++n) sc[n][t] = __builtin_amdgcn_mfma_f32_16x16x32_f16(f, q[n][k], sc[n][t], 0, 0, 0);
        }
      }
      if (u + 1 < u1) fetch_keys(tok_next, pg_next);
      if (!whole) {
#pragma unroll
        for (int t = 0; t < 2; ++t)
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            const int key = tok + 16 * t + 4 * h4 + i;
            const bool there = key < s.held && (t ? p1 : p0);
#pragma unroll
            for (int n = 0; n < NC; ++n) sc[n][t][i] = there && sees(sight[n], key) ? sc[n][t][i] : -__builtin_inff();
          }
#pragma unroll
        for (int t = 0; t < 2; ++t) {                               // whatever stands where no token is: its value is 0
          const uint32_t keep = bytes_below((t ? p1 : p0) ? s.held - (tok + 16 * t + 4 * h4) : 0);
#pragma unroll
          for (int v = 0; v < VU; ++v) x.v[t][v] &= keep;
        }
      }
      v8h p[NC], rest[NC];
#pragma unroll
      for (int n = 0; n < NC; ++n) {
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
          if constexpr (!BF) {
            const v2h pl = rest_of(ph, e[2 * i], e[2 * i + 1]);
            rest[n][2 * i] = pl.x; rest[n][2 * i + 1] = pl.y;
            l[n] = __builtin_amdgcn_fdot2(pl, v2h{(_Float16)1.f, (_Float16)1.f}, l[n], false);
          }
        }
      }
#pragma unroll
      for (int v = 0; v < VU; ++v)
#pragma unroll
        for (int i = 0; i < 4; ++i) {                               // channels 64 v + 4 n + i
          const v8h f = octet8(x.v[0][v][i], x.v[1][v][i], x.s[0].y, x.s[1].y);
#pragma unroll
          for (int n = 0; n < NC; ++n) {
            o[n][4 * v + i] = __builtin_amdgcn_mfma_f32_16x16x32_f16(f, p[n], o[n][4 * v + i], 0, 0, 0);
            if constexpr (!BF)
              o[n][4 * v + i] = __builtin_amdgcn_mfma_f32_16x16x32_f16(f, rest[n], o[n][4 * v + i], 0, 0, 0);
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
#pragma unroll
    for (int n = 0; n < NC; ++n) {
      l[n] = across_sum(l[n]);
      if (h4 == 0) { m_sh[wave][16 * n + col] = m[n]; l_sh[wave][16 * n + col] = l[n]; }
#pragma unroll
      for (int v = 0; v < VU; ++v)
#pragma unroll
        for (int i = 0; i < 4; ++i)                                 // row 4 h4 + i of four tiles: channels 64 v + 4 (4 h4 + i) ..
          *(v4f*)&o_sh[wave][16 * n + col][64 * v + 16 * h4 + 4 * i] = v4f{o[n][4 * v][i], o[n][4 * v + 1][i], o[n][4 * v + 2][i], o[n][4 * v + 3][i]};
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

// ------------------------------------------------------------------ launch
// Tokens that the rows of a sequence see: all that the table holds, if there is no window, else about the window, what is new, and the sinks
static int seen_of(const DRows& r, int window, int sinks) {
  if (window <= 0) return r.cap;
  const int64_t s = (int64_t)window + r.tokens / r.seqs + UNIT + ((int64_t)sinks + UNIT - 1) / UNIT * UNIT;
  return (int)(s < r.cap ? s : r.cap);
}
// Every tile of `rows` rows, at most; its units, if all sequences saw `seen` tokens; the workgroups that run at once.
struct Load8 { int64_t tiles, units; int rows, chip; };
static Load8 load_of(const DCache8& c, const DRows& r, int ratio, int seen) {
  const int64_t rows = (int64_t)r.tokens * ratio;
  Load8 w{(rows / 16 + r.seqs) * c.heads, seen > UNIT ? (seen + UNIT - 1) / UNIT : 1, 16,
          256 * (c.dim == 64 ? RESIDENT<64, 16> : c.dim == 128 ? RESIDENT<128, 16> : RESIDENT<256, 16>)};
  // Tiles of 32 rows read a head's tokens once where two of 16 would read them twice: from 17 rows a sequence, and eight units a workgroup, which else have
  // what they start and end with to win back (128 channels, 8 cache heads, 4 query heads on one: 16 sequences of 4000 tokens, 5 tokens 49 us
  // against 60, 8 tokens 52 against 62, 4 tokens 47 against 45; 2 of 100000, 8 tokens 91 against 140; one of 8000, 8 tokens 27 against 25).  256 channels have no
  // registers for it (one workgroup a CU: 43 against 38).
  if (c.dim < 256 && rows > (int64_t)16 * r.seqs && w.tiles * (w.units + EXTRA) > (int64_t)8 * w.chip)
    w = Load8{(rows / 32 + r.seqs) * c.heads, w.units, 32, 256 * (c.dim == 64 ? RESIDENT<64, 32> : RESIDENT<128, 32>)};
  return w;
}
struct Plan8 { int grid, rows; bool split, wide; size_t bytes; };
static Plan8 plan_few(const DCache8& c, const DRows& r, int ratio, int seen) {
  const Load8 w = load_of(c, r, ratio, seen);
  Plan8 p;
  p.rows = w.rows;
  // Tiles of few units stay in one piece, which saves the second launch, where there are enough of them: up to 8 units from a tile a CU, up to 16
  // where they about fill the chip (128 channels, 8 cache heads, single tokens; whole against cut: 1 sequence of 640 tokens 16.2 and 14.1 us, 32 of 640 17.9 and 23.4,
  // of 1024 22.4 and 26.5; 64 of 2048 54 and 64, of up to 2048 39 and 43; 32 of up to 2048 32 and 28; 256 of up to 2048 132 and 119).
  p.split = w.units > 16 || (w.units > 8 && (2 * w.tiles < w.chip || w.tiles > 2 * w.chip)) || (w.units > 4 && w.tiles < 256);
  const int64_t most = p.split ? w.tiles * (w.units + EXTRA) : w.tiles;
  p.grid = (int)(most < w.chip ? most : w.chip);
  p.bytes = p.split ? attn_bytes(p.grid, p.rows, c.dim) : 0;
  p.wide = p.grid > 200 * w.tiles;
  return p;
}

// What a call is to take, in us, by the launches (their start, and the join behind a cut), the tiles of rows, and the units that each reads.  Which kernel, and
// whether that for many rows cuts its tiles, is the least of three such times: a tile of 256 rows reads the cache a 16th as often as tiles of 16 and fills two
// thirds of the chip's rate for an ordinary product, but is one workgroup a CU, filled or not, and a cut leaves 256 rows of float32 in memory for each
// end.  Constants from 500 calls of 24 rows a sequence and more in all forms (1 to 64 sequences of 1 to 140000 tokens, 1 to 16 cache heads, windows),
// each in all three ways: the least of the three estimates is within 1.2 % of the fastest on the (geometric) mean and within 9 % for 95 of 100.  For instance
// (128 channels, bf16 unless said): 61 new of 85 tokens of 46 sequences, 4 cache heads x 4, 256 channels: few rows 104 us, whole 60, cut 103;
// 1 sequence of 37 new behind 132000, 8 x 4, fp16: 210, 5788, 251; 180 new of 75000, 16 x 16, 256 channels, window of 39: 115, 38, 91; the last 512 of 16384 tokens, 8 x 4:
// whole 469, cut 174; prompts of 3100 tokens, 8 x 2, fp16: whole 159, cut 124; of 4096, 8 x 4: whole 155, cut 190.
struct Choice8 { bool many; PromptPlan prompt; Plan8 few; size_t bytes; };
static Choice8 choose(const DCache8& c, const DRows& r, const AttnArgs& a, int window, int sinks) {
  const int seen = seen_of(r, window, sinks);
  const int64_t rows = (int64_t)r.tokens * a.ratio;
  Choice8 x{};
  x.few = plan_few(c, r, a.ratio, seen);
  x.bytes = x.few.bytes;
  if (rows <= (int64_t)16 * r.seqs || (rows / 256 + r.seqs) * c.heads >= (int64_t)1 << 23) return x;   // (a launch of workgroups of 512 has fewer than 2^32 threads)
  const Load8 w = load_of(c, r, a.ratio, seen);
  const double slow = c.dim == 256 ? 1.2 : 1., unit = 2 + 1.1 * w.units, filled = (double)w.tiles / w.chip;
  const double few = x.few.split ? (w.rows == 32 ? 16 : 14) + filled * (w.units + 2) * 2.5 * slow : 9 + fmax(unit, filled * unit * 2.2) * slow;
  // tokens that a tile of 256 rows sees, in tiles of its own, at most and on average
  const int keys = c.dim == 256 ? 64 : 128, least = r.cap < keys ? keys : r.cap;
  const double limit = window > 0 ? fmin(least, (double)window + 256 / a.ratio + sinks + keys) : least;
  const double mean = fmin(limit, fmax(least - 0.5 * r.tokens / r.seqs, 0.5 * least));
  const double longest = ceil(limit / keys), usual = ceil(mean / keys), tiles = (double)(rows / 256 + r.seqs) * c.heads / 256;
  const double step = c.dim == 64 ? (a.bf ? 2.2 : 3.6) : c.dim == 128 ? (a.bf ? 3.4 : 4.3) : a.bf ? 3.4 : 3.8;
  const double start = c.dim == 64 ? 6 : c.dim == 128 ? 9 : 12, join = c.dim == 64 ? 25 : c.dim == 128 ? 31 : 49;
  const double whole = 4 + fmax(start + longest * step, tiles * (start + usual * step)), cut = join + tiles * (usual + 2) * step;
  x.many = fmin(whole, cut) < few;
  if (x.many) {
    x.prompt = plan_prompt8(c, r, a.ratio, cut < whole);
    x.bytes = x.prompt.bytes;
  }
  return x;
}
size_t cache8_attn_workspace(const DCache8& c, const DRows& r, int ratio) {   // (of either type)
  AttnArgs a{};
  a.ratio = ratio;
  const size_t f16 = choose(c, r, a, 0, 0).bytes;
  a.bf = 1;
  const size_t bf16 = choose(c, r, a, 0, 0).bytes;
  return f16 > bf16 ? f16 : bf16;
}

template <int D, int R>
static void few(const Plan8& p, const DCache8& c, const DRows& r, const AttnArgs& a, hipStream_t st) {
  if (a.bf) hipLaunchKernelGGL((cache8_attn_kernel<D, R, true>), dim3(p.grid), dim3(256), 0, st, c, r, a);
  else hipLaunchKernelGGL((cache8_attn_kernel<D, R, false>), dim3(p.grid), dim3(256), 0, st, c, r, a);
}
template <int D>
static void few(const Plan8& p, const DCache8& c, const DRows& r, const AttnArgs& a, hipStream_t st) {
  if constexpr (D < 256)
    if (p.rows == 32) return few<D, 32>(p, c, r, a, st);
  few<D, 16>(p, c, r, a, st);
}
int launch_cache8_attn(const DCache8& c, const DRows& r, AttnArgs a, size_t ws_bytes, hipStream_t st) {
  const size_t need = cache8_attn_workspace(c, r, a.ratio);
  if (need > ws_bytes || (need && !a.ws)) return CBK_ERR_WORKSPACE;
  Choice8 x = choose(c, r, a, a.window, a.sinks);
  if (x.bytes > need) x = choose(c, r, a, 0, 0);                    // (the workspace is asked for without the window)
  if (!x.bytes) a.ws = nullptr;
  if (x.many) return launch_cache8_prompt(x.prompt, c, r, a, st);
  const Plan8 p = x.few;
  a.whole = !p.split;
  if (c.dim == 64) few<64>(p, c, r, a, st);
  else if (c.dim == 128) few<128>(p, c, r, a, st);
  else few<256>(p, c, r, a, st);
  if (p.split) launch_cache_join(c.dim, a, p.grid, p.rows, st, p.wide);
  return hipGetLastError() == hipSuccess ? CBK_OK : CBK_ERR_HIP;
}

}  // namespace cbk
