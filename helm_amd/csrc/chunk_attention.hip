// chunk_attention.hip — attention of a ragged batch of new tokens over a paged cache,
// with a sliding window and first tokens that stay visible.
//
// Sequence b has rows q_starts[b] .. q_starts[b + 1] - 1 of q, its n newest tokens; its
// t-th row stands at p = seq_lens[b] - n + t and sees key j where j <= p and (no window,
// or j > p - window, or j < sinks).  out = softmax(scale q . K^T) V over those keys.
//
// All lengths are on the device, so what a workgroup does is found on the device too (the
// plan, 1.4 us of a workgroup's start with up to 64 sequences; every wave reads all of them, 64 at a time,
// so it grows with their number: one token after 100 of 32 heads takes 33 us with 256 sequences, 70 with 512, 165
// with 1024): each sequence's rows (token, head of the kv head's group; token-major) are cut into
// row tiles, each tile's keys into the sequence's number of pieces, and workgroup x of a kv head takes the x-th (sequence, tile, piece).  Pieces are
// sized so that all of them find places on the chip at once, whatever the lengths are;
// sequences of one piece write their output, the others fp32 partials that a second kernel
// merges.  The grid and the workspace depend on bounds that the host knows (plan_of).  The kv
// head is the fastest-varying workgroup index: with 8 of them each XCD serves one, and its
// K/V stays in that XCD's L2.
//
// Two forms share the sequences by their number of rows:
//   few_body   up to 16 or 32 rows (decode, drafts): bound by streaming K and V once; the four
//              waves of a workgroup take key steps in turn.  16 items of up to 12000 tokens
//              under a window of 2048, 40 heads over 8 (117 MB): 24 us and 4.5 for the merge;
//              one item of 16384 under 4096 (17 MB): 7.3 and 4.5, a chain of round trips (kernel
//              arguments, lengths, table, K / V) on either side of one step
//   tile_body  more (prompts): bound by the matrix cores; the waves take rows and share K and V
//              through LDS.  4096 tokens after 12288, 40 heads over 8: 1075-1105 us, 1.09-1.12 PFLOP/s,
//              0.95-0.98 of what an 8192^3 fp16 product reaches on this card (1.15).  A workgroup's start and end
//              cost 8 us beside 1.9 a step of 64 keys (two workgroups a CU): prompts under a window of
//              1024, 18 steps a tile, run at 0.80 PFLOP/s
// A batch with sequences of both kinds runs them in one launch (both_attn_kernel).
// Both forms run S^T = K . Q^T and O^T += V^T . P^T on v_mfma_f32_16x16x32_f16 with the keys of the
// score tiles permuted so that each lane holds the probabilities of the 8 consecutive keys
// whose V^T it feeds to the second product, and an online softmax in the log2 domain whose
// maximum is raised only when it is passed by kLazy.
#include <algorithm>
#include <type_traits>

#include "helm_common.h"

namespace {

constexpr int kThreads = 256;
constexpr int kWaves = 4;
constexpr float kLazy = 8.f;            // lazy-rescale slack of the running maximum (log2)
// What a probability is carried times 2^: the largest, 2^(kLazy + kLift), stays in fp16's range, and a
// small one keeps 2^-11 of itself down to 2^-21 of the maximum's and 2^-32 of the maximum's below (at
// 2^0, 131072 keys of 2^-25 beside one of 1 would vanish, 0.4% of the weight).
constexpr float kLift = 7.f;
constexpr int kMaxPieces = 64;          // of a tile's keys

typedef _Float16 h8_t __attribute__((ext_vector_type(8)));
typedef float f4_t __attribute__((ext_vector_type(4)));
typedef __attribute__((address_space(3))) void lds_void_t;

// How one of the two kernels cuts the sequences it takes, and its partials: sums [Hkv][parts]
// [tile rows][D], not normalised, then [Hkv][parts][tile rows][2] running maximum and sum.
struct Form {
  int lo, hi;          // it takes sequences of lo < rows <= hi
  int tile, step;      // log2 of the rows of a tile, of the keys of a step
  int min_steps;       // least steps of a piece
  float per_piece;     // most pieces of a step
  int want;            // pieces of a kv head that fill the chip
  float per_want;      // 1 / want and a little, so that work * per_want is not below work / want
  int most_keys;       // that a tile can see
  int items;           // workgroups of a kv head that the grid has (0: not launched)
  int parts;           // partials of a kv head (0: no sequence can have two pieces)
  int cut_tiles;       // tiles of several pieces, at most
  float* part_o;
  float* part_ml;
};

struct ChunkArgs {
  const uint16_t* q;
  int64_t q_st, q_sh;                   // query element (t, h, d): t*q_st + h*q_sh + d
  uint16_t* out;
  int64_t o_st, o_sh;
  const uint16_t* k;
  int64_t k_ss, k_hs;
  const uint16_t* v;
  int64_t v_ss, v_hs, v_ds;
  int32_t num_slots;
  const int32_t* page_table;
  int64_t pt_stride;
  const int32_t* seq_lens;
  const int32_t* q_starts;              // null: one row per sequence
  int N, B, Hq, Hkv, G, P, max_pages, max_new;
  int window, sinks;                    // window 0: none
  uint32_t mul_g;                       // 2^32 / G + 1 (G = 1: 0)
  int covered;                          // tokens that the table has room for
  float qk_scale_log2;
  Form f[2];                            // few rows, many rows
};
constexpr int kFew = 0, kMany = 1;

// Token of a row (token, head): x / G as one high product, exact while x G < 2^32.
__device__ __forceinline__ int token_of(const ChunkArgs& a, int row) {
  return a.mul_g ? (int)__umulhi((uint32_t)row, a.mul_g) : row;
}

struct Seq {
  int start, n, rows, len;              // first row, new tokens, rows (token, head) to do, tokens
  int tiles, steps;                     // 0: not this form's
};

__device__ __forceinline__ Seq seq_of(const ChunkArgs& a, const Form& f, int i) {
  const int j = min(i, a.B - 1);
  int s0 = j, e = j + 1;
  const int len = a.seq_lens[j];
  if (a.q_starts) {
    s0 = a.q_starts[j];
    e = a.q_starts[j + 1];
  }
  Seq s;
  s.len = len;
  s.start = min(max(s0, 0), a.N);
  s.n = max(min(e, a.N) - s.start, 0);
  s.rows = min(s.n, a.max_new) * a.G;
  const bool mine = i < a.B && s.rows > f.lo && s.rows <= f.hi;
  s.tiles = mine ? (s.rows + (1 << f.tile) - 1) >> f.tile : 0;
  s.steps = mine ? max((min(max(len, 0), f.most_keys) + (1 << f.step) - 1) >> f.step, 1) : 0;
  return s;
}

struct Item {
  int seq, start, n, rows, len;         // the sequence: index, first row, new tokens, rows to do, tokens
  int tile, piece, pieces;
  int part;                             // partial of its tile's piece 0
};

template <int CTRL, int ROWS>
__device__ __forceinline__ float dpp_of(float v, float none) {
  return __int_as_float(__builtin_amdgcn_update_dpp(__float_as_int(none), __float_as_int(v), CTRL, ROWS, 0xF, false));
}
__device__ __forceinline__ float dpp_sum(float v) {      // of a wave, the same in all lanes
  v += dpp_of<0x111, 0xF>(v, 0.f);
  v += dpp_of<0x112, 0xF>(v, 0.f);
  v += dpp_of<0x114, 0xF>(v, 0.f);
  v += dpp_of<0x118, 0xF>(v, 0.f);
  v += dpp_of<0x142, 0xA>(v, 0.f);
  v += dpp_of<0x143, 0xC>(v, 0.f);
  return __int_as_float(__builtin_amdgcn_readlane(__float_as_int(v), 63));
}
__device__ __forceinline__ float dpp_max(float v) {
  v = fmaxf(v, dpp_of<0x111, 0xF>(v, v));
  v = fmaxf(v, dpp_of<0x112, 0xF>(v, v));
  v = fmaxf(v, dpp_of<0x114, 0xF>(v, v));
  v = fmaxf(v, dpp_of<0x118, 0xF>(v, v));
  v = fmaxf(v, dpp_of<0x142, 0xA>(v, v));
  v = fmaxf(v, dpp_of<0x143, 0xC>(v, v));
  return __int_as_float(__builtin_amdgcn_readlane(__float_as_int(v), 63));
}

// Pieces of a tile of so many steps: of m each at most, and of 1 / per_piece at least.
__device__ __forceinline__ int pieces_of(const Form& f, int steps, float inv_m) {
  const int most = min(max((int)((float)steps * f.per_piece), 1), kMaxPieces);
  return min(max((int)ceilf((float)steps * inv_m), 1), most);
}

// Most steps of a piece, 1 / m returned: with W the sum of tiles x steps of a kv head, the least m
// of W / want x 1, 1.25, 1.5, 2 whose pieces find places all at once (a second round of
// workgroups would cost as much as the first, and more pieces more partials); with more tiles than
// places only what is twice as long as the mean is cut.  So there are at most want + tiles items,
// and at most want in tiles of several pieces.
__device__ __forceinline__ float inv_steps(const ChunkArgs& a, const Form& f, const Seq& first) {
  const int lane = threadIdx.x & 63;
  float work = (float)first.tiles * (float)first.steps, tiles = (float)first.tiles;
  for (int i = 64; i < a.B; i += 64) {
    const Seq s = seq_of(a, f, i + lane);
    work += (float)s.tiles * (float)s.steps;
    tiles += (float)s.tiles;
  }
  const float mean = dpp_sum(work) * f.per_want;
  float m = 2.f * mean;
  if (m > (float)f.min_steps && dpp_sum(tiles) < (float)f.want) {
#pragma unroll 1
    for (float by = 1.f; by < 2.f; by += 0.25f) {
      const float inv = 1.f / fmaxf(mean * by, (float)f.min_steps);
      float n = (float)(first.tiles * pieces_of(f, first.steps, inv));
      for (int i = 64; i < a.B; i += 64) {
        const Seq s = seq_of(a, f, i + lane);
        n += (float)(s.tiles * pieces_of(f, s.steps, inv));
      }
      if (dpp_sum(n) <= (float)f.want) {
        m = mean * by;
        break;
      }
    }
  }
  return 1.f / fmaxf(m, (float)f.min_steps);
}

// The want-th (tile, piece) of a kv head, or with MERGE the want-th tile of more than one
// piece; false where there are fewer.  Every wave finds it by itself, a lane per sequence.
template <bool FEW, bool MERGE>
__device__ __forceinline__ bool find_item(const ChunkArgs& a, int want, Item& it) {
  const Form& f = a.f[FEW ? kFew : kMany];
  const int lane = threadIdx.x & 63;
  const Seq first = seq_of(a, f, lane);
  const float inv = inv_steps(a, f, first);
  uint32_t items = 0, parts = 0;        // of the sequences before
  for (int i0 = 0; i0 < a.B; i0 += 64) {
    const Seq s = i0 == 0 ? first : seq_of(a, f, i0 + lane);
    const int pieces = pieces_of(f, s.steps, inv);
    const uint32_t own_parts = pieces > 1 ? (uint32_t)(s.tiles * pieces) : 0u;
    const uint32_t mine = MERGE ? (pieces > 1 ? (uint32_t)s.tiles : 0u) : (uint32_t)(s.tiles * pieces);
    const uint32_t upto = items + wave_scan(mine), parts_upto = parts + wave_scan(own_parts);
    const uint64_t hit = __ballot(upto > (uint32_t)want);
    if (hit) {                          // the first sequence that reaches it
      const int l = __ffsll((unsigned long long)hit) - 1;
      it.seq = i0 + l;
      it.pieces = (int)lane_of((uint32_t)pieces, l);
      it.start = (int)lane_of((uint32_t)s.start, l);
      it.n = (int)lane_of((uint32_t)s.n, l);
      it.rows = (int)lane_of((uint32_t)s.rows, l);
      it.len = (int)lane_of((uint32_t)s.len, l);
      const int at = want - (int)(lane_of(upto, l) - lane_of(mine, l));
      const int per = MERGE ? 1 : it.pieces;
      const int t = (int)((uint32_t)at / (uint32_t)per);
      it.tile = (int)lane_of((uint32_t)s.tiles, l) - 1 - t;      // the tiles with the most keys first
      it.piece = at - t * per;
      it.part = (int)(lane_of(parts_upto, l) - lane_of(own_parts, l)) + it.tile * it.pieces;
      return true;
    }
    items = lane_of(upto, 63);
    parts = lane_of(parts_upto, 63);
  }
  return false;
}

// The keys that a tile's rows, at positions p0 .. p1, see, in steps: those of the sinks, then those
// of the window.  Step j covers the keys from at(j) * step on.
struct Steps {
  int sink, first, count;               // steps of the sinks; first step of the window; all
  int end;                              // the tile sees no key from end on
  // No row of the sequence sees a key in [sinks, open) or from close on: their V may be anything.
  // (V of other keys that a row does not see meets a probability of 0.)
  int open, close;
  __device__ __forceinline__ int at(int j) const { return j < sink ? j : first + j - sink; }
};
__device__ __forceinline__ Steps steps_of(const ChunkArgs& a, const Item& it, int p0, int p1, int step) {
  Steps s{0, 0, 0, 0, 0, 0};
  const int base = it.len - it.n;       // position of the sequence's first row
  const int all = min(it.len, a.covered);
  s.end = max(min(p1 + 1, all), 0);
  s.close = max(min(base + token_of(a, it.rows), all), 0);
  const int last = (s.end + step - 1) / step;
  s.count = last;
  if (a.window) {
    s.open = max(base - a.window + 1, 0);
    s.first = max(p0 - a.window + 1, 0) / step;
    s.sink = min((min(a.sinks, s.end) + step - 1) / step, s.first);
    s.count = s.sink + max(last - s.first, 0);
  }
  return s;
}

// the few-row kernel reads q and K and V once (non-temporal)
__device__ __forceinline__ h8_t ld_h8_nt(const uint16_t* p) {
  return __builtin_bit_cast(h8_t, __builtin_nontemporal_load(reinterpret_cast<const u32x4_t*>(p)));
}
__device__ __forceinline__ h8_t ld_h8(const uint16_t* p) {
  return __builtin_bit_cast(h8_t, *reinterpret_cast<const u32x4_t*>(p));
}

// Of eight keys from `key` on, in an operand's words: the bits of those that some row may see.
__device__ __forceinline__ u32x4_t seen_bits(const ChunkArgs& a, const Steps& s, int key, bool page_ok) {
  u32x4_t w;
#pragma unroll
  for (int q = 0; q < 4; ++q) {
    auto seen = [&](int k) { return page_ok & (k < s.close) & ((k >= s.open) | (k < a.sinks)); };
    w[q] = (seen(key + 2 * q) ? 0x0000ffffu : 0u) | (seen(key + 2 * q + 1) ? 0xffff0000u : 0u);
  }
  return w;
}

// ── few rows ─────────────────────────────────────────────────────────────────

// NC tiles of 16 rows.  Steps of 32 keys, one wave each, round robin; K's and V's registers
// are filled again as soon as they have been read (157 registers at NC = 1, 215 at 2: three and two
// workgroups a CU).  P is split into fp16 hi + lo parts (the matrix cores wait for memory anyway): at
// 2^kLift it enters the product to 2^-22 of itself, below 2^-21 of the maximum's to 2^-32 of that, where lo
// has no bits left.  Its sum is that of the fp32 values.
template <int D, int NC>
struct FewLds {
  float o[kWaves][16 * NC][D];
  float m[kWaves][16 * NC], l[kWaves][16 * NC];
};

template <int D, int P, int NC>
__device__ __forceinline__ void few_body(const ChunkArgs& a, int hk, int item, FewLds<D, NC>& lds) {
  constexpr int KT = D / 32;
  constexpr int DT = D / 16;
  constexpr int kStep = 32;
  auto& s_m = lds.m;
  auto& s_l = lds.l;
  auto& s_o = lds.o;
  const Form& f = a.f[kFew];

  const int tid = threadIdx.x;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int lane = tid & 63;
  const int col = lane & 15, grp = lane >> 4;
  Item it;
  if (!find_item<true, false>(a, item, it)) return;
  const int G = a.G;
  const int p0 = it.len - it.n, p1 = p0 + token_of(a, it.rows) - 1;      // (one tile a sequence)
  const Steps steps = steps_of(a, it, p0, p1, kStep);
  const int lo = (int)((int64_t)steps.count * it.piece / it.pieces);
  const int hi = (int)((int64_t)steps.count * (it.piece + 1) / it.pieces);
  const int mine = hi - lo > wave ? (hi - lo - 1 - wave) / kWaves + 1 : 0;
  const int32_t* ptab = a.page_table + (int64_t)it.seq * a.pt_stride;
  auto tok = [&](int i) { return steps.at(min(lo + wave + i * kWaves, hi - 1)) * kStep; };
  // slots of this lane's K rows (keys 8 (col / 4) + 4 t + col % 4 of a step) and V keys (8 grp ..)
  auto slot = [&](int key) {
    const int s = ptab[min(key / P, a.max_pages - 1)];
    return s >= 0 && s < a.num_slots ? s : -1;
  };
  int nk = -1, nv = -1;
  if (mine > 0) {
    nk = slot(tok(0) + (col >> 2) * 8);
    nv = slot(tok(0) + grp * 8);
  }
  const bool two = NC > 1 && it.rows > 16;
  int pos[NC];
  h8_t qb[NC][KT];
#pragma unroll
  for (int c = 0; c < NC; ++c) {
    const int row = min(c * 16 + col, it.rows - 1);
    const int t = token_of(a, row);
    pos[c] = p0 + t;
    const uint16_t* qp = a.q + (int64_t)(it.start + t) * a.q_st + (int64_t)(hk * G + row - t * G) * a.q_sh + grp * 8;
#pragma unroll
    for (int kk = 0; kk < KT; ++kk) qb[c][kk] = ld_h8(qp + kk * 32);
  }
  const uint16_t* kbase = a.k + (int64_t)hk * a.k_hs + grp * 8;
  const uint16_t* vbase = a.v + (int64_t)hk * a.v_hs + (int64_t)col * a.v_ds;
  h8_t kb[2][KT], vb[DT];
  auto load_k = [&](int s, int t0) {
    const uint16_t* kp = kbase + (int64_t)max(s, 0) * a.k_ss + ((t0 + (col >> 2) * 8) % P + (col & 3)) * D;
#pragma unroll
    for (int t = 0; t < 2; ++t)
#pragma unroll
      for (int kk = 0; kk < KT; ++kk) kb[t][kk] = ld_h8_nt(kp + t * 4 * D + kk * 32);
  };
  auto load_v = [&](int s, int t0) {
    const uint16_t* vp = vbase + (int64_t)max(s, 0) * a.v_ss + (t0 + grp * 8) % P;
#pragma unroll
    for (int d = 0; d < DT; ++d) vb[d] = ld_h8_nt(vp + (int64_t)d * 16 * a.v_ds);
  };

  float m_run[NC], l_run[NC];
  f4_t o[NC][DT];
#pragma unroll
  for (int c = 0; c < NC; ++c) {
    m_run[c] = -INFINITY;
    l_run[c] = 0.f;
#pragma unroll
    for (int d = 0; d < DT; ++d) o[c][d] = f4_t{0.f, 0.f, 0.f, 0.f};
  }
  bool ok = nv >= 0;
  if (mine > 0) {
    load_k(nk, tok(0));
    load_v(nv, tok(0));
    nk = slot(tok(1) + (col >> 2) * 8);
    nv = slot(tok(1) + grp * 8);
  }
  auto step = [&](int i, auto more) {
    constexpr bool kMore = decltype(more)::value;
    const int t0 = tok(i), tv = t0 + grp * 8;
    const bool whole = __all(ok) && t0 + kStep - 1 <= p0 && t0 + kStep <= steps.end &&
                       (!a.window || t0 > p1 - a.window || t0 + kStep <= a.sinks);
    float sv[NC][8];
#pragma unroll
    for (int c = 0; c < NC; ++c) {
      if (c && !two) break;
      f4_t s0 = {0.f, 0.f, 0.f, 0.f}, s1 = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
      for (int kk = 0; kk < KT; ++kk) {
        s0 = __builtin_amdgcn_mfma_f32_16x16x32_f16(kb[0][kk], qb[c][kk], s0, 0, 0, 0);
        s1 = __builtin_amdgcn_mfma_f32_16x16x32_f16(kb[1][kk], qb[c][kk], s1, 0, 0, 0);
      }
#pragma unroll
      for (int r = 0; r < 4; ++r) {
        sv[c][r] = s0[r];
        sv[c][4 + r] = s1[r];
      }
    }
    if constexpr (kMore) load_k(nk, tok(i + 1));
    if (!whole) {
      const u32x4_t bits = seen_bits(a, steps, tv, ok);
#pragma unroll
      for (int d = 0; d < DT; ++d) vb[d] = __builtin_bit_cast(h8_t, __builtin_bit_cast(u32x4_t, vb[d]) & bits);
    }
#pragma unroll
    for (int c = 0; c < NC; ++c) {
      if (c && !two) break;
      if (!whole) {
        const int top = ok ? min(pos[c], steps.end - 1) : -1;
        const int low = a.window ? pos[c] - a.window + 1 : 0;
#pragma unroll
        for (int j = 0; j < 8; ++j)
          sv[c][j] = (tv + j <= top) & ((tv + j >= low) | (tv + j < a.sinks)) ? sv[c][j] : -INFINITY;
      }
      const float mx = fmaxf(fmaxf(fmaxf(sv[c][0], sv[c][1]), fmaxf(sv[c][2], sv[c][3])),
                             fmaxf(fmaxf(sv[c][4], sv[c][5]), fmaxf(sv[c][6], sv[c][7]))) * a.qk_scale_log2;
      if (__ballot(mx > m_run[c] + kLazy)) {
        float m = fmaxf(mx, __shfl_xor(mx, 16, 64));
        m = fmaxf(m, __shfl_xor(m, 32, 64));
        const float m_new = fmaxf(m_run[c], m);
        const float alpha = __builtin_amdgcn_exp2f(m_run[c] - (m_new == -INFINITY ? 0.f : m_new));
        l_run[c] *= alpha;
#pragma unroll
        for (int d = 0; d < DT; ++d) o[c][d] *= alpha;
        m_run[c] = m_new;
      }
      const float ref = m_run[c] == -INFINITY ? 0.f : kLift - m_run[c];
      h8_t ph, pl;
      float sum = 0.f;
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        const float p = __builtin_amdgcn_exp2f(__builtin_fmaf(sv[c][j], a.qk_scale_log2, ref));
        sum += p;
        ph[j] = (_Float16)p;
        pl[j] = (_Float16)(p - (float)ph[j]);
      }
      l_run[c] += sum;
#pragma unroll
      for (int d = 0; d < DT; ++d) {
        o[c][d] = __builtin_amdgcn_mfma_f32_16x16x32_f16(vb[d], ph, o[c][d], 0, 0, 0);
        o[c][d] = __builtin_amdgcn_mfma_f32_16x16x32_f16(vb[d], pl, o[c][d], 0, 0, 0);
      }
    }
    if constexpr (kMore) {
      load_v(nv, tok(i + 1));
      ok = nv >= 0;
      nk = slot(tok(i + 2) + (col >> 2) * 8);
      nv = slot(tok(i + 2) + grp * 8);
    }
  };
  if (mine > 0) {
    for (int i = 0; i + 1 < mine; ++i) step(i, std::true_type{});
    step(mine - 1, std::false_type{});
  }

  // the lane groups' sums, then (through LDS) the waves
#pragma unroll
  for (int c = 0; c < NC; ++c) {
    float l = l_run[c];
    l += __shfl_xor(l, 16, 64);
    l += __shfl_xor(l, 32, 64);
#pragma unroll
    for (int d = 0; d < DT; ++d) *reinterpret_cast<f4_t*>(&s_o[wave][c * 16 + col][d * 16 + grp * 4]) = o[c][d];
    if (grp == 0) {
      s_m[wave][c * 16 + col] = m_run[c];
      s_l[wave][c * 16 + col] = l;
    }
  }
  __syncthreads();
  for (int idx = tid; idx < it.rows * (D / 4); idx += kThreads) {
    const int row = idx / (D / 4), d = (idx - row * (D / 4)) * 4;
    float m = s_m[0][row];
#pragma unroll
    for (int w = 1; w < kWaves; ++w) m = fmaxf(m, s_m[w][row]);
    const float ref = m == -INFINITY ? 0.f : m;
    float l = 0.f;
    f4_t n = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
    for (int w = 0; w < kWaves; ++w) {
      const float f = __builtin_amdgcn_exp2f(s_m[w][row] - ref);
      l = fmaf(f, s_l[w][row], l);
      const f4_t x = *reinterpret_cast<const f4_t*>(&s_o[w][row][d]);
#pragma unroll
      for (int e = 0; e < 4; ++e) n[e] = fmaf(f, x[e], n[e]);
    }
    if (it.pieces > 1) {
      const int64_t at = ((int64_t)hk * f.parts + it.part + it.piece) * (16 * NC) + row;
      *reinterpret_cast<f4_t*>(f.part_o + at * D + d) = n;
      if (d == 0) *reinterpret_cast<float2*>(f.part_ml + at * 2) = make_float2(m, l);
    } else {
      const float inv = l == 0.f ? 0.f : 1.f / l;       // (a row that sees nothing: zeros; NaN stays)
      const int t = token_of(a, row);
      *reinterpret_cast<uint2*>(a.out + (int64_t)(it.start + t) * a.o_st + (int64_t)(hk * G + row - t * G) * a.o_sh + d) =
          make_uint2(pack_h2(n[0] * inv, n[1] * inv), pack_h2(n[2] * inv, n[3] * inv));
    }
  }
}

// ── many rows ────────────────────────────────────────────────────────────────

constexpr int kNC = 2;                   // 16-row tiles of a wave
constexpr int kTile = kWaves * 16 * kNC; // rows of a workgroup
constexpr int kKeys = 64;                // keys of a step

// Workgroup barrier for the K / V stages: this wave's copies into LDS have landed and its
// LDS reads have returned (s_waitcnt vmcnt(0) lgkmcnt(0)), then s_barrier.
__device__ __forceinline__ void stage_barrier() {
  asm volatile("" ::: "memory");
  __builtin_amdgcn_s_waitcnt(0 | (7 << 4) | (0 << 8));
  __builtin_amdgcn_s_barrier();
  asm volatile("" ::: "memory");
}

// One wave's 1 KiB global -> LDS copy: lane l moves 16 bytes from base + off to LDS byte lds +
// 16 l.  Inline assembly, so that the compiler does not make a step's operand reads wait for
// the copies of the next one; the step's barrier waits.
#pragma clang diagnostic push
#pragma clang diagnostic ignored "-Winline-asm"   // m0 is named as clobbered on purpose
__device__ __forceinline__ void copy_to_lds(const uint16_t* base, uint32_t off, uint32_t lds) {
  const uint64_t p = (uint64_t)(uintptr_t)base;
  const uint64_t at = (uint64_t)(uint32_t)__builtin_amdgcn_readfirstlane((int)(uint32_t)p) |
                      (uint64_t)(uint32_t)__builtin_amdgcn_readfirstlane((int)(uint32_t)(p >> 32)) << 32;
  asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %1, %2"
               :
               : "s"(__builtin_amdgcn_readfirstlane(lds)), "v"(off), "s"(at)
               : "memory", "m0");
}
#pragma clang diagnostic pop

// XOR swizzle of K chunk columns: the 16 rows (col >> 2) * 8 + t * 4 + (col & 3) of an operand
// read have the swizzles col
template <int CPR>
__device__ __forceinline__ int kswz(int r) {
  return ((r & 3) | (((r >> 3) & 3) << 2)) & (CPR - 1);
}

// A wave takes kNC x 16 rows, a workgroup kTile.  Per step of 64 keys a wave runs 68 products a
// 1088 cycles of the matrix core at D = 128, and on the vector unit per score a multiply-add, half
// a maximum, an exponential and half a conversion; the two halves of a step share one check of
// the maximum, so that the second half's products can run beside the first half's softmax.
// What the step does not compute: page slots come by scalar loads a step ahead (a copy
// instruction reads one page), operand addresses are constants and one toggled stage bit, sums
// are products with ones.  (Steps of 32 keys with three workgroups a CU in 168 registers: long
// prompts 1% faster, mixed batches 4%, prompts under a window 5% and short ones 15% slower.)
template <int D>
struct TileLds {
  u32x4_t kv[2][2 * kKeys * D / 8];
};

// WIN: there is a window.
template <int D, int P, bool WIN>
__device__ __forceinline__ void tile_body(const ChunkArgs& a, int hk, int item, TileLds<D>& lds) {
  constexpr int NC = kNC;
  constexpr int KT = D / 32;
  constexpr int DT = D / 16;
  constexpr int CPR = D / 8;                        // 16-byte chunks of a K row
  constexpr int kKC = kKeys * CPR;                  // chunks of a stage's K, and of its V
  constexpr int kI = kKC / kThreads;                // copies of a thread for each
  constexpr int UPP = kKeys / P;                    // pages of a step
  constexpr uint32_t kStage = 2 * kKC * 16;         // bytes of a stage
  auto& s_kv = lds.kv;
  const Form& f = a.f[kMany];

  const int tid = threadIdx.x;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int lane = tid & 63;
  const int col = lane & 15, grp = lane >> 4;
  Item it;
  if (!find_item<false, false>(a, item, it)) return;
  const int r0 = it.tile * kTile, rw = r0 + wave * 16 * NC;       // first row of the tile, of this wave
  const int base = it.len - it.n;                                 // position of the sequence's first row
  const Steps steps = steps_of(a, it, base + token_of(a, r0), base + token_of(a, min(r0 + kTile, it.rows) - 1), kKeys);
  const int lo = (int)((int64_t)steps.count * it.piece / it.pieces);
  const int hi = (int)((int64_t)steps.count * (it.piece + 1) / it.pieces);
  // positions of this wave's rows (none: every key is behind its last one)
  const int pw0 = base + token_of(a, rw), pw1 = rw < it.rows ? base + token_of(a, min(rw + 16 * NC, it.rows) - 1) : -1;

  // The table is read through scalar loads: a step's slots are the same for all lanes
  typedef const __attribute__((address_space(4))) int32_t cint_t;
  cint_t* ptab = (cint_t*)(uintptr_t)(a.page_table + (int64_t)it.seq * a.pt_stride);
  int slot[UPP];                                    // of the step whose copies go out next
  auto look_up = [&](int j) {
    const int pg = steps.at(min(j, hi - 1)) * UPP;
#pragma unroll
    for (int u = 0; u < UPP; ++u) slot[u] = ptab[min(pg + u, a.max_pages - 1)];
  };
  if (lo < hi) look_up(lo);
  int pos[NC];
  h8_t qb[NC][KT];
#pragma unroll
  for (int c = 0; c < NC; ++c) {
    const int row = min(rw + c * 16 + col, it.rows - 1);
    const int t = token_of(a, row);
    pos[c] = base + t;
    const uint16_t* qp =
        a.q + (int64_t)(it.start + t) * a.q_st + (int64_t)(hk * a.G + row - t * a.G) * a.q_sh + grp * 8;
#pragma unroll
    for (int kk = 0; kk < KT; ++kk) qb[c][kk] = ld_h8(qp + kk * 32);
  }

  // bytes of this thread's chunks from their page's start
  uint32_t k_off[kI], v_off[kI];
#pragma unroll
  for (int i = 0; i < kI; ++i) {
    const int pc = i * kThreads + tid, row = pc / CPR;
    k_off[i] = (uint32_t)((row % P) * D + ((pc % CPR) ^ kswz<CPR>(row)) * 8) * 2;
    const int vi = i * kWaves + wave, kp = vi / (D / 32), dim = vi % (D / 32) * 32 + (lane & 31);
    v_off[i] = ((uint32_t)dim * (uint32_t)a.v_ds + (uint32_t)((kp * 16) % P + (lane >> 5) * 8)) * 2;
  }
  const uint16_t* kbase = a.k + (int64_t)hk * a.k_hs;
  const uint16_t* vbase = a.v + (int64_t)hk * a.v_hs;
  const uint32_t k_ss = (uint32_t)a.k_ss, v_ss = (uint32_t)a.v_ss;
  const uint32_t lds0 = (uint32_t)(uintptr_t)(lds_void_t*)&s_kv[0][0];
  // Copies of the looked-up step into the stage at LDS byte `to`; its invalid pages, one bit
  // each (they read slot 0).  Copy i of a wave is 1 KiB of K rows and 32 dims x 16 keys of V,
  // both of the step's 16 keys i (D = 128) or 2 i + wave / 2.
  auto issue = [&](uint32_t to) {
    uint32_t bad = 0;
    int s[UPP];
#pragma unroll
    for (int u = 0; u < UPP; ++u) {
      const bool ok = (uint32_t)slot[u] < (uint32_t)a.num_slots;
      s[u] = ok ? slot[u] : 0;
      bad |= ok ? 0u : 1u << u;
    }
#pragma unroll
    for (int i = 0; i < kI; ++i) {
      uint32_t x = (uint32_t)s[D == 128 ? i * 16 / P : i * 32 / P];
      if (D == 64 && P == 16) x = wave >> 1 ? (uint32_t)s[(2 * i + 1) % UPP] : x;
      copy_to_lds(kbase + (uint64_t)x * k_ss, k_off[i], to + (uint32_t)(i * kThreads + wave * 64) * 16);
      copy_to_lds(vbase + (uint64_t)x * v_ss, v_off[i], to + (uint32_t)(kKC + (i * kWaves + wave) * 64) * 16);
    }
    return bad;
  };

  // LDS bytes of this lane's operands in the stage that is read: K row (col >> 2) * 8 + (col &
  // 3), chunk (4 kk + grp) ^ col, and V key group grp, dim col
  uint32_t k_at[KT], v_at;
#pragma unroll
  for (int kk = 0; kk < KT; ++kk)
    k_at[kk] = (uint32_t)(((col >> 2) * 8 + (col & 3)) * CPR + ((kk * 4 + grp) ^ (col & (CPR - 1)))) * 16;
  v_at = (uint32_t)(kKC + (grp >> 1) * (D / 32) * 64 + (grp & 1) * 32 + col) * 16;
  auto lds_h8 = [&](uint32_t at) { return *reinterpret_cast<const h8_t*>(reinterpret_cast<const char*>(&s_kv[0][0]) + at); };

  // m_run: what a column's scores are relative to, kLift below the maximum it was last set to (0 until it
  // has met a key), thr: how far a score may pass it (a column that has met no key takes any)
  constexpr float kTop = kLazy + kLift;
  float m_run[NC], thr[NC];
  f4_t o[NC][DT], l_acc[NC];
#pragma unroll
  for (int c = 0; c < NC; ++c) {
    m_run[c] = 0.f;
    thr[c] = -3.4e38f;
    l_acc[c] = f4_t{0.f, 0.f, 0.f, 0.f};
#pragma unroll
    for (int d = 0; d < DT; ++d) o[c][d] = f4_t{0.f, 0.f, 0.f, 0.f};
  }
  h8_t ones;
#pragma unroll
  for (int j = 0; j < 8; ++j) ones[j] = (_Float16)1.f;

  uint32_t bad_next = 0, stage = 0;
  if (lo < hi) {
    bad_next = issue(lds0);
    look_up(lo + 1);
  }
  for (int j = lo; j < hi; ++j) {
    stage_barrier();                                // the step is in its stage; the other one is no longer read
    const uint32_t bad = bad_next, cur = stage;
    stage ^= kStage;
    if (j + 1 < hi) {
      bad_next = issue(lds0 + stage);
      look_up(j + 2);
    }
    const int key0 = steps.at(j) * kKeys;
    // V of keys that no row sees may hold anything: zero (uniform over the workgroup; the first
    // and last steps of a sequence)
    if (bad || key0 + kKeys > steps.close || (WIN && key0 < steps.open && key0 + kKeys > a.sinks)) {
#pragma unroll 1
      for (int i = 0; i < kI; ++i) {
        const int vi = i * kWaves + wave, key = vi / (D / 32) * 16 + (lane >> 5) * 8;
        u32x4_t* x = reinterpret_cast<u32x4_t*>(reinterpret_cast<char*>(&s_kv[0][0]) + cur) + kKC + vi * 64 + lane;
        *x &= seen_bits(a, steps, key0 + key, !((bad >> (key / P)) & 1));
      }
      lds_barrier();
    }
    // nothing of the step is visible to this wave's rows
    if (key0 > pw1 || (WIN && key0 + kKeys - 1 <= pw0 - a.window && key0 >= a.sinks)) continue;
    const bool whole = !bad && key0 + kKeys - 1 <= pw0 && key0 + kKeys <= steps.end &&
                       (!WIN || key0 > pw1 - a.window || key0 + kKeys <= a.sinks);

    // scores of keys key0 + 32 u + 8 grp + e
    float t[2][NC][8];
#pragma unroll
    for (int u = 0; u < 2; ++u) {
      h8_t kf[2][KT];
#pragma unroll
      for (int y = 0; y < 2; ++y)
#pragma unroll
        for (int kk = 0; kk < KT; ++kk) kf[y][kk] = lds_h8(cur + k_at[kk] + (uint32_t)(u * 32 + y * 4) * CPR * 16);
#pragma unroll
      for (int c = 0; c < NC; ++c) {
        f4_t s0 = {0.f, 0.f, 0.f, 0.f}, s1 = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int kk = 0; kk < KT; ++kk) {
          s0 = __builtin_amdgcn_mfma_f32_16x16x32_f16(kf[0][kk], qb[c][kk], s0, 0, 0, 0);
          s1 = __builtin_amdgcn_mfma_f32_16x16x32_f16(kf[1][kk], qb[c][kk], s1, 0, 0, 0);
        }
#pragma unroll
        for (int r = 0; r < 4; ++r) {
          t[u][c][r] = s0[r];
          t[u][c][4 + r] = s1[r];
        }
      }
    }
    if (!whole) {
#pragma unroll
      for (int u = 0; u < 2; ++u) {
        const int tv = key0 + u * 32 + grp * 8;
        const bool ok = !((bad >> ((u * 32 + grp * 8) / P)) & 1);
#pragma unroll
        for (int c = 0; c < NC; ++c) {
          // bit e: key tv + e is visible (v_bfe spreads it over a word, v_bfi picks)
          auto below = [](int x) { return (1u << min(max(x, 0), 8)) - 1u; };    // bits e < x
          uint32_t see = below(min(pos[c], steps.end - 1) - tv + 1);
          if (WIN) see &= ~below(pos[c] - a.window + 1 - tv) | below(a.sinks - tv);
          see = ok ? see : 0u;
#pragma unroll
          for (int e = 0; e < 8; ++e) {
            const uint32_t all = (uint32_t)__builtin_amdgcn_sbfe((int)see, e, 1);
            t[u][c][e] = __uint_as_float((__float_as_uint(t[u][c][e]) & all) | (0xff800000u & ~all));
          }
        }
      }
    }
    bool raise = false;
    float mx[NC];
#pragma unroll
    for (int c = 0; c < NC; ++c) {
      mx[c] = -INFINITY;
#pragma unroll
      for (int u = 0; u < 2; ++u)
#pragma unroll
        for (int e = 0; e < 8; ++e) {
          t[u][c][e] = __builtin_fmaf(t[u][c][e], a.qk_scale_log2, -m_run[c]);
          mx[c] = fmaxf(mx[c], t[u][c][e]);
        }
      raise |= mx[c] > thr[c];
    }
    if (__ballot(raise)) {
#pragma unroll
      for (int c = 0; c < NC; ++c) {
        float m = fmaxf(mx[c], __shfl_xor(mx[c], 16, 64));
        m = fmaxf(m, __shfl_xor(m, 32, 64));
        const bool up = m > thr[c];
        const float by = up ? m - kLift : 0.f;
        const float alpha = up ? (thr[c] == kTop ? __builtin_amdgcn_exp2f(-by) : 0.f) : 1.f;
        m_run[c] += by;
        thr[c] = up ? kTop : thr[c];
        l_acc[c] *= alpha;
#pragma unroll
        for (int d = 0; d < DT; ++d) o[c][d] *= alpha;
#pragma unroll
        for (int u = 0; u < 2; ++u)
#pragma unroll
          for (int e = 0; e < 8; ++e) t[u][c][e] -= by;
      }
    }
    // P enters the product rounded to fp16, and so do the sums (a product with ones): the
    // rounding of a probability then moves numerator and denominator alike, an output by 2^-11 sum p |v - o|
    // at most (random data: 2.9e-4 of the output's size from the exact one, its own rounding is 2.1e-4 of
    // that).  A second product of a low part, as few rows have, would be 32 more of a step's 68.
#pragma unroll
    for (int u = 0; u < 2; ++u) {
      h8_t ph[NC];
#pragma unroll
      for (int c = 0; c < NC; ++c)
#pragma unroll
        for (int e = 0; e < 8; ++e) ph[c][e] = (_Float16)__builtin_amdgcn_exp2f(t[u][c][e]);
#pragma unroll
      for (int c = 0; c < NC; ++c) l_acc[c] = __builtin_amdgcn_mfma_f32_16x16x32_f16(ones, ph[c], l_acc[c], 0, 0, 0);
#pragma unroll
      for (int d = 0; d < DT; ++d) {
        const h8_t vf = lds_h8(cur + v_at + (uint32_t)(u * 2 * (D / 32) * 64 + (d >> 1) * 64 + (d & 1) * 16) * 16);
#pragma unroll
        for (int c = 0; c < NC; ++c) o[c][d] = __builtin_amdgcn_mfma_f32_16x16x32_f16(vf, ph[c], o[c][d], 0, 0, 0);
      }
    }
    // The order of this block: the first half's probabilities, its products with the second half's
    // probabilities between them (two vector instructions and an operand read a product), the second
    // half's products.  chunk of 4096 after 12288, 40 heads 1099 -> 1066 us, the compiler's own order
    // before; raised wave priority around the products 1132-1170.
    __builtin_amdgcn_sched_group_barrier(0x100, 4, 0);      // operand reads
    __builtin_amdgcn_sched_group_barrier(0x002, 28, 0);     // vector instructions
#pragma unroll
    for (int i = 0; i < NC * (1 + DT); ++i) {
      __builtin_amdgcn_sched_group_barrier(0x008, 1, 0);    // a product
      __builtin_amdgcn_sched_group_barrier(0x002, 2, 0);
      __builtin_amdgcn_sched_group_barrier(0x100, 1, 0);
    }
#pragma unroll
    for (int i = 0; i < NC * (1 + DT); ++i) {
      __builtin_amdgcn_sched_group_barrier(0x008, 1, 0);
      __builtin_amdgcn_sched_group_barrier(0x100, 1, 0);
    }
  }

  // o[c][d][r] = O^T[dim d*16 + grp*4 + r][row col of tile c]
#pragma unroll
  for (int c = 0; c < NC; ++c) {
    const int row = rw + c * 16 + col;
    if (row >= it.rows) continue;
    const float l = l_acc[c][0];
    if (it.pieces > 1) {
      const int64_t at = ((int64_t)hk * f.parts + it.part + it.piece) * kTile + (row - r0);
      float* dst = f.part_o + at * D + grp * 4;
#pragma unroll
      for (int d = 0; d < DT; ++d) *reinterpret_cast<f4_t*>(dst + d * 16) = o[c][d];
      if (grp == 0) *reinterpret_cast<float2*>(f.part_ml + at * 2) = make_float2(thr[c] == kTop ? m_run[c] : -INFINITY, l);
    } else {
      const float inv = l == 0.f ? 0.f : 1.f / l;       // (a row that sees nothing: zeros; NaN stays)
      const int tt = pos[c] - base;
      uint16_t* dst = a.out + (int64_t)(it.start + tt) * a.o_st + (int64_t)(hk * a.G + row - tt * a.G) * a.o_sh + grp * 4;
#pragma unroll
      for (int d = 0; d < DT; ++d)
        *reinterpret_cast<uint2*>(dst + d * 16) = make_uint2(pack_h2(o[c][d][0] * inv, o[c][d][1] * inv),
                                                             pack_h2(o[c][d][2] * inv, o[c][d][3] * inv));
    }
  }
}

// ── the kernels ──────────────────────────────────────────────────────────────

template <int D, int P, int NC>
__global__ __launch_bounds__(kThreads, NC == 1 ? 3 : 2) void few_attn_kernel(ChunkArgs a) {
  __shared__ __attribute__((aligned(16))) FewLds<D, NC> lds;
  few_body<D, P, NC>(a, (int)(blockIdx.x % (unsigned)a.Hkv), (int)(blockIdx.x / (unsigned)a.Hkv), lds);
}
template <int D, int P, bool WIN>
__global__ __launch_bounds__(kThreads, 2) void tile_attn_kernel(ChunkArgs a) {
  __shared__ __attribute__((aligned(16))) TileLds<D> lds;
  tile_body<D, P, WIN>(a, (int)(blockIdx.x % (unsigned)a.Hkv), (int)(blockIdx.x / (unsigned)a.Hkv), lds);
}
// Both forms in one launch, the many rows' workgroups first: those of few rows wait for memory and
// fill the places that are left.  700 rows after 8000 beside 24 single rows, 40 heads: 190 us.  Before the
// products and exponentials were put in turn 204, in two launches 214, with the two kinds in turn 260.
template <int D, int P, bool WIN>
__global__ __launch_bounds__(kThreads, 2) void both_attn_kernel(ChunkArgs a) {
  __shared__ __attribute__((aligned(16))) union { FewLds<D, 1> few; TileLds<D> tile; } lds;
  const int hk = (int)(blockIdx.x % (unsigned)a.Hkv), x = (int)(blockIdx.x / (unsigned)a.Hkv);
  if (x < a.f[kMany].items) tile_body<D, P, WIN>(a, hk, x, lds.tile);
  else few_body<D, P, 1>(a, hk, x - a.f[kMany].items, lds.few);
}

// out = sum_p 2^(m_p - M) o_p / sum_p 2^(m_p - M) l_p over a tile's pieces.  Bound by latency (the
// plan, the maxima, the partials: 3.5-4.5 us, with nothing to merge too), beside many rows by
// reading their partials (30 MB: 13 us).  A workgroup takes R rows (grid.y of them a tile, the tiles of
// few rows first); its threads are 4 dims of a row each, and where those are fewer than 256, groups
// that take the pieces in turn.
template <int D, int R>
__global__ __launch_bounds__(kThreads) void chunk_merge_kernel(ChunkArgs a, int few_tiles) {
  constexpr int S = R * (D / 4);        // threads of a group
  constexpr int PG = S < kThreads ? kThreads / S : 1;
  constexpr int U = S < kThreads ? 1 : S / kThreads;     // (row, 4 dims) of a thread
  __shared__ float s_w[R][kMaxPieces], s_inv[R];
  __shared__ __attribute__((aligned(16))) f4_t s_n[PG][S];
  const int tid = threadIdx.x;
  const int hk = (int)(blockIdx.x % (unsigned)a.Hkv);
  int want = (int)(blockIdx.x / (unsigned)a.Hkv);
  const bool few = want < few_tiles;
  if (!few) want -= few_tiles;
  const Form& f = a.f[few ? kFew : kMany];
  Item it;
  if (!(few ? find_item<true, true>(a, want, it) : find_item<false, true>(a, want, it))) return;
  const int r0 = it.tile << f.tile, y0 = (int)blockIdx.y * R;
  const int rows = min(it.rows - r0, 1 << f.tile) - y0;       // of this workgroup and on
  if (rows <= 0) return;
  const int64_t base = ((int64_t)hk * f.parts + it.part) << f.tile;
  // lane p of a wave: piece p of a row
  for (int r = tid >> 6; r < min(rows, R); r += kWaves) {
    const int p = tid & 63;
    float2 x = make_float2(-INFINITY, 0.f);
    if (p < it.pieces)
      x = *reinterpret_cast<const float2*>(f.part_ml + (base + ((int64_t)p << f.tile) + y0 + r) * 2);
    const float m = dpp_max(x.x);
    const float w = m == -INFINITY ? 0.f : __builtin_amdgcn_exp2f(x.x - m);
    const float l = dpp_sum(w * x.y);
    s_w[r][p] = w;
    if (p == 0) s_inv[r] = l == 0.f ? 0.f : 1.f / l;    // (a row that sees nothing: zeros; NaN stays)
  }
  __syncthreads();
  const int pg = tid / S;
  // each thread's U rows together: their loads do not wait for one another
  const float* po[U];
  f4_t n[U];
  int at[U];
#pragma unroll
  for (int u = 0; u < U; ++u) {
    at[u] = tid % S + u * kThreads;
    po[u] = f.part_o + (base + y0 + min(at[u] / (D / 4), rows - 1)) * D + at[u] % (D / 4) * 4;
    n[u] = f4_t{0.f, 0.f, 0.f, 0.f};
  }
  const int64_t stride = (int64_t)D << f.tile;
  constexpr int L = 8 / U;              // pieces at a time
  for (int p0 = pg; p0 < it.pieces; p0 += L * PG) {
    f4_t y[L][U];
#pragma unroll
    for (int i = 0; i < L; ++i)
      if (p0 + i * PG < it.pieces) {
#pragma unroll
        for (int u = 0; u < U; ++u) y[i][u] = *reinterpret_cast<const f4_t*>(po[u] + (p0 + i * PG) * stride);
      }
#pragma unroll
    for (int i = 0; i < L; ++i)
      if (p0 + i * PG < it.pieces) {
#pragma unroll
        for (int u = 0; u < U; ++u) {
          const float w = s_w[min(at[u] / (D / 4), rows - 1)][p0 + i * PG];
#pragma unroll
          for (int e = 0; e < 4; ++e) n[u][e] = fmaf(w, y[i][u][e], n[u][e]);
        }
      }
  }
  if constexpr (PG > 1) {
    s_n[pg][at[0]] = n[0];
    __syncthreads();
    if (pg > 0) return;
#pragma unroll
    for (int g = 1; g < PG; ++g) n[0] += s_n[g][at[0]];
  }
#pragma unroll
  for (int u = 0; u < U; ++u) {
    const int r = at[u] / (D / 4), d = at[u] % (D / 4) * 4;
    if (r >= rows) break;
    const float inv = s_inv[r];
    const int row = r0 + y0 + r, t = token_of(a, row);
    *reinterpret_cast<uint2*>(a.out + (int64_t)(it.start + t) * a.o_st + (int64_t)(hk * a.G + row - t * a.G) * a.o_sh + d) =
        make_uint2(pack_h2(n[u][0] * inv, n[u][1] * inv), pack_h2(n[u][2] * inv, n[u][3] * inv));
  }
}

// ── host ─────────────────────────────────────────────────────────────────────

// How a call's sequences are shared between the two kernels and cut, from what the host knows.
struct Plan {
  Form f[2];
  int few_nc;                           // 16-row tiles of the few-row kernel
};

Form form_of(int lo, int hi, int tile, int step, int min_steps, float per_piece, int want, int64_t tiles,
             int64_t keys) {
  Form f{};
  f.lo = lo; f.hi = hi; f.tile = tile; f.step = step; f.min_steps = min_steps; f.want = want;
  f.per_want = 1.00002f / (float)want;
  f.per_piece = per_piece;
  f.most_keys = (int)keys;
  const int64_t steps = (keys + (1 << step) - 1) >> step;
  const bool cut = steps > min_steps && (float)steps * per_piece >= 2.f;
  f.items = (int)std::min<int64_t>(tiles + (cut ? want + 1 : 0), 1 << 28);
  f.parts = cut ? want + 2 : 0;         // (also where q_starts is no ascending list)
  f.cut_tiles = (int)std::min<int64_t>(f.parts / 2, tiles);
  return f;
}

Plan plan_of(int N, int B, int Hq, int Hkv, int P, int max_pages, int max_new, int window, int sinks) {
  Plan p{};
  const int G = Hq / Hkv;
  const int64_t most = (int64_t)std::min(max_new, N) * G;         // rows of a sequence
  const int seqs = std::min(B, N);
  const int few = G > 32 || (B == 1 && most > 32) ? 0 : most <= 16 ? 16 : most <= 32 || G > 16 ? 32 : 16;
  p.few_nc = few / 16;
  // keys that a tile of so many rows can see: its window begins at its first row's and ends at
  // its last row, both rounded to steps
  auto keys = [&](int rows, int step) {
    const int64_t all = (int64_t)max_pages * P;
    return window ? std::min<int64_t>(all, (int64_t)window + sinks + rows / G + 2 * step) : all;
  };
  const int want = std::max(1, 512 / Hkv);
  if (few) p.f[kFew] = form_of(0, few, few == 16 ? 4 : 5, 5, 4, 1.f, want, seqs, keys(few, 32));
  if (most > few)
    // a piece of fewer than 8 steps costs more in partials than it saves (700 rows after 100 of 40 heads in
    // two pieces of 7 steps 32.4 us, whole 26.2)
    p.f[kMany] = form_of(few, 1 << 30, 7, 6, 8, 0.125f, want, (int64_t)N * G / kTile + seqs, keys(kTile, kKeys));
  return p;
}
int64_t part_floats(const Form& f, int Hkv, int D) { return ((int64_t)Hkv * f.parts << f.tile) * (D + 2); }

template <int D, int P>
void launch(ChunkArgs a, const Plan& p, float* ws, hipStream_t s) {
  for (int w = 0; w < 2; ++w) {
    a.f[w] = p.f[w];
    a.f[w].part_o = ws;
    a.f[w].part_ml = ws + ((int64_t)a.Hkv * p.f[w].parts << p.f[w].tile) * D;
    ws += part_floats(p.f[w], a.Hkv, D);
  }
  const Form &few = p.f[kFew], &many = p.f[kMany];
  auto run = [&](auto kernel, int items) {
    hipLaunchKernelGGL(kernel, dim3((unsigned)items * (unsigned)a.Hkv), dim3(kThreads), 0, s, a);
  };
  if (many.items && few.items && p.few_nc == 1) {
    if (a.window) run(both_attn_kernel<D, P, true>, many.items + few.items);
    else run(both_attn_kernel<D, P, false>, many.items + few.items);
  } else if (many.items) {
    if (a.window) run(tile_attn_kernel<D, P, true>, many.items);
    else run(tile_attn_kernel<D, P, false>, many.items);
  }
  if (few.items && !(many.items && p.few_nc == 1)) {
    if (p.few_nc == 1) run(few_attn_kernel<D, P, 1>, few.items);
    else run(few_attn_kernel<D, P, 2>, few.items);
  }
  const int few_tiles = few.cut_tiles, tiles = few_tiles + many.cut_tiles;
  if (tiles == 0) return;
  if (many.parts)
    hipLaunchKernelGGL((chunk_merge_kernel<D, 32>), dim3((unsigned)tiles * (unsigned)a.Hkv, kTile / 32), dim3(kThreads), 0,
                       s, a, few_tiles);
  else
    hipLaunchKernelGGL((chunk_merge_kernel<D, 2>), dim3((unsigned)tiles * (unsigned)a.Hkv, (1 << few.tile) / 2),
                       dim3(kThreads), 0, s, a, few_tiles);
}

}  // namespace

extern "C" int64_t helm_chunk_attn_workspace_bytes(int N, int B, int Hq, int Hkv, int D, int P, int max_pages,
                                                   int max_new, int window, int sinks) {
  if (N < 1 || B < 1 || Hkv < 1 || Hq < Hkv || Hq % Hkv || D < 1 || P < 1 || max_pages < 1 || max_new < 1 ||
      window < 0 || sinks < 0)
    return 0;
  const Plan p = plan_of(N, B, Hq, Hkv, P, max_pages, max_new, window, sinks);
  return (part_floats(p.f[kFew], Hkv, D) + part_floats(p.f[kMany], Hkv, D)) * (int64_t)sizeof(float);
}

extern "C" int helm_chunk_attn(const void* q, int64_t q_stride_t, int64_t q_stride_h, const helm_kv_pool* pool,
                               const int32_t* page_table, int64_t pt_stride, const int32_t* seq_lens,
                               const int32_t* q_starts, int N, int B, int Hq, int Hkv, int D, int P, int max_pages,
                               int max_new, int window, int sinks, float scale, void* out, int64_t out_stride_t,
                               int64_t out_stride_h, void* workspace, int64_t workspace_bytes, void* stream) {
  const std::string f("helm_chunk_attn");
  HELM_CHECK_ARG(q && pool && pool->k && pool->v && page_table && seq_lens && out, f + ": null pointer");
  HELM_CHECK_ARG(N >= 1 && B >= 1 && Hq >= 1 && Hkv >= 1 && max_pages >= 1 && max_new >= 1,
                 f + ": sizes must be positive");
  HELM_CHECK_ARG(window >= 0 && sinks >= 0, f + ": window and sinks must not be negative");
  HELM_CHECK_ARG(q_starts || N == B, f + ": without q_starts there is one row per sequence");
  HELM_CHECK_ARG(Hq % Hkv == 0, f + ": Hq must be a multiple of Hkv");
  HELM_CHECK_ARG(scale > 0.f && scale * kLog2e < INFINITY, f + ": scale must be positive and finite");
  HELM_CHECK_SUPPORTED(D == 64 || D == 128, f + ": head_dim must be 64 or 128");
  HELM_CHECK_SUPPORTED(P == 16 || P == 32 || P == 64, f + ": page size must be 16, 32 or 64");
  HELM_CHECK_SUPPORTED((int64_t)N * (Hq / Hkv) < (1 << 30) && (int64_t)N * (Hq / Hkv) * (Hq / Hkv) < (1ll << 32) && Hq <= 65535,
                       f + ": too many rows or heads");
  HELM_CHECK_SUPPORTED((int64_t)max_pages * P <= (int64_t)1 << 30 && window <= 1 << 30 && sinks <= 1 << 30,
                       f + ": more than 2^30 keys");
  HELM_CHECK_ARG(B == 1 || pt_stride >= max_pages, f + ": page-table stride < max_pages");
  HELM_CHECK_ARG(pool->num_slots >= 1 && pool->k_head_stride >= (int64_t)P * D && pool->v_dim_stride >= P &&
                     pool->v_head_stride >= (int64_t)P,
                 f + ": pool strides too small for the page");
  HELM_CHECK_SUPPORTED(pool->v_dim_stride * D < (1ll << 30), f + ": V dim stride too large (in-page offsets are 32-bit)");
  HELM_CHECK_SUPPORTED(pool->k_slot_stride >= 0 && pool->k_slot_stride < (1ll << 32) && pool->v_slot_stride >= 0 &&
                           pool->v_slot_stride < (1ll << 32),
                       f + ": slot strides must be below 2^32 elements");
  HELM_CHECK_SUPPORTED(q_stride_t % 8 == 0 && q_stride_h % 8 == 0 && out_stride_t % 4 == 0 && out_stride_h % 4 == 0 &&
                           pool->k_slot_stride % 8 == 0 && pool->k_head_stride % 8 == 0 &&
                           pool->v_slot_stride % 8 == 0 && pool->v_head_stride % 8 == 0 && pool->v_dim_stride % 8 == 0,
                       f + ": strides must be multiples of 8 (q, pool) / 4 (out) elements");
  HELM_CHECK_SUPPORTED(helm::aligned16(q) && helm::aligned16(pool->k) && helm::aligned16(pool->v) &&
                           (reinterpret_cast<uintptr_t>(out) & 7u) == 0,
                       f + ": q and pools must be 16-byte aligned, out 8-byte aligned");
  const Plan p = plan_of(N, B, Hq, Hkv, P, max_pages, max_new, window, sinks);
  const int64_t need = helm_chunk_attn_workspace_bytes(N, B, Hq, Hkv, D, P, max_pages, max_new, window, sinks);
  HELM_CHECK_ARG(need == 0 || (workspace && helm::aligned16(workspace) && workspace_bytes >= need),
                 f + ": this call needs " + std::to_string(need) + " bytes of 16-byte aligned workspace");
  HELM_CHECK_SUPPORTED(((int64_t)p.f[kFew].items + p.f[kMany].items) * Hkv < (1ll << 31), f + ": too many workgroups");
  ChunkArgs a{};
  a.q = static_cast<const uint16_t*>(q); a.q_st = q_stride_t; a.q_sh = q_stride_h;
  a.out = static_cast<uint16_t*>(out); a.o_st = out_stride_t; a.o_sh = out_stride_h;
  a.k = static_cast<const uint16_t*>(pool->k); a.k_ss = pool->k_slot_stride; a.k_hs = pool->k_head_stride;
  a.v = static_cast<const uint16_t*>(pool->v);
  a.v_ss = pool->v_slot_stride; a.v_hs = pool->v_head_stride; a.v_ds = pool->v_dim_stride;
  a.num_slots = (int32_t)std::min<int64_t>(pool->num_slots, 0x7fffffff);   // (slots are int32)
  a.page_table = page_table; a.pt_stride = pt_stride; a.seq_lens = seq_lens; a.q_starts = q_starts;
  a.N = N; a.B = B; a.Hq = Hq; a.Hkv = Hkv; a.G = Hq / Hkv; a.P = P;
  a.mul_g = a.G > 1 ? (uint32_t)((1ull << 32) / (uint32_t)a.G + 1) : 0; a.max_pages = max_pages;
  a.max_new = std::min(max_new, N);
  a.window = window; a.sinks = window ? sinks : 0;
  a.covered = max_pages * P;
  a.qk_scale_log2 = scale * kLog2e;
  float* ws = static_cast<float*>(workspace);
  const hipStream_t s = static_cast<hipStream_t>(stream);
  auto by_page = [&](auto d_tag) {
    constexpr int Dc = decltype(d_tag)::value;
    if (P == 16) launch<Dc, 16>(a, p, ws, s);
    else if (P == 32) launch<Dc, 32>(a, p, ws, s);
    else launch<Dc, 64>(a, p, ws, s);
  };
  if (D == 64) by_page(std::integral_constant<int, 64>{});
  else by_page(std::integral_constant<int, 128>{});
  HELM_CHECK_LAUNCH("helm_chunk_attn launch");
  return HELM_OK;
}
