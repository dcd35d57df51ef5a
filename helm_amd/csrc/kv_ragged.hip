// kv_ragged.hip — a ragged batch's way into a paged cache (rotary positions and K/V writes),
// and pages moved inside a pool.
#include <algorithm>
#include <type_traits>

#include "helm_common.h"

namespace {

struct Pool {
  uint16_t* k;
  int64_t k_ss, k_hs;
  uint16_t* v;
  int64_t v_ss, v_hs, v_ds;
  int64_t num_slots;
};

struct RopeArgs {
  const uint16_t* qkv;
  int64_t qkv_st;
  const uint16_t* q_norm_w;
  const uint16_t* k_norm_w;
  float eps;
  const int32_t* page_table;
  int64_t pt_stride;
  const int32_t* seq_lens;
  const int32_t* q_starts;      // null: one row per sequence
  const int32_t* positions;     // null: the tokens' own
  const float* inv_freq;
  float rope_scale;
  uint16_t* q_out;
  Pool pool;
  int N, B, Hq, Hkv, P, max_pages, rot;
  bool inter;
};

// cos and sin of pos * inv_freq times scale, the angle reduced in 64 bits.
__device__ __forceinline__ float2 rope_factors(int pos, float inv_freq, float scale) {
  constexpr double kInvPi = 0.31830988618379067154;
  double t = (double)pos * (double)inv_freq * kInvPi;   // half turns
  t -= 2.0 * rint(0.5 * t);                             // [-1, 1]
  return make_float2(cospif((float)t) * scale, sinpif((float)t) * scale);
}

struct Place {
  int seq, pos, slot, off;      // seq -1: no sequence's row; slot -1: nowhere in the pool
};
// Where row `row` of sequence b goes (b = B or a row before the first sequence: nowhere).
__device__ __forceinline__ Place place_of(const RopeArgs& a, int row, int b) {
  Place p{-1, 0, -1, 0};
  if (b >= a.B) return p;
  int end = row + 1;
  if (a.q_starts) {
    if (row < a.q_starts[b]) return p;
    end = a.q_starts[b + 1];
  }
  p.seq = b;
  p.pos = a.seq_lens[b] - (end - row);
  if (p.pos >= 0 && p.pos / a.P < a.max_pages) {
    const int s = a.page_table[(int64_t)b * a.pt_stride + p.pos / a.P];
    if (s >= 0 && s < a.pool.num_slots) p.slot = s;
    p.off = p.pos % a.P;
  }
  return p;
}

// One wave per (row, head).  Bound by latency: the row's sequence (how many of q_starts[1 ..] are
// not above it, 64 at a time), its length, its slot, and then the write: 16 rows of 32 + 8 + 8 heads 3.2
// us.
template <int D>
__global__ __launch_bounds__(256) void rope_rows_kernel(RopeArgs a) {
  constexpr int J = D / 64;
  const int lane = threadIdx.x & 63;
  const int64_t item = (int64_t)blockIdx.x * 4 + (threadIdx.x >> 6);
  const int heads = a.Hq + 2 * a.Hkv;
  if (item >= (int64_t)a.N * heads) return;
  const int row = __builtin_amdgcn_readfirstlane((int)(item / heads));
  const int hh = __builtin_amdgcn_readfirstlane((int)(item - (int64_t)row * heads));
  const bool is_v = hh >= a.Hq + a.Hkv, is_q = hh < a.Hq;
  const uint16_t* src = a.qkv + (int64_t)row * a.qkv_st + (int64_t)hh * D;
  uint16_t raw[J];
#pragma unroll
  for (int j = 0; j < J; ++j) raw[j] = src[lane + 64 * j];
  // pair and angle of each of the lane's dims
  const int half = a.rot / 2;
  float w[J], freq[J];
  int other[J];
  bool turns[J];
  const uint16_t* nw = is_v ? nullptr : is_q ? a.q_norm_w : a.k_norm_w;
#pragma unroll
  for (int j = 0; j < J; ++j) {
    const int d = lane + 64 * j;
    turns[j] = !is_v && d < a.rot;
    other[j] = a.inter ? d ^ 1 : d < half ? d + half : d - half;
    freq[j] = turns[j] ? a.inv_freq[a.inter ? d >> 1 : d < half ? d : d - half] : 0.f;
    w[j] = nw ? h2f(nw[d]) : 1.f;
  }
  int b = row;
  if (a.q_starts) {
    b = 0;
    for (int i = 0; i < a.B; i += 64) b += __popcll(__ballot(i + lane < a.B && a.q_starts[min(i + lane, a.B - 1) + 1] <= row));
  }
  const Place p = place_of(a, row, b);
  if (p.seq < 0) return;
  if (is_v) {
    if (p.slot < 0) return;
    uint16_t* dst = a.pool.v + (int64_t)p.slot * a.pool.v_ss + (int64_t)(hh - a.Hq - a.Hkv) * a.pool.v_hs + p.off;
#pragma unroll
    for (int j = 0; j < J; ++j) dst[(int64_t)(lane + 64 * j) * a.pool.v_ds] = raw[j];
    return;
  }
  float x[J];
#pragma unroll
  for (int j = 0; j < J; ++j) x[j] = h2f(raw[j]);
  if (nw) {
    float ss = 0.f;
#pragma unroll
    for (int j = 0; j < J; ++j) ss = fmaf(x[j], x[j], ss);
    const float rstd = rsqrtf(wave_sum(ss) / (float)D + a.eps);
#pragma unroll
    for (int j = 0; j < J; ++j) x[j] = x[j] * rstd * w[j];
  }
  const int pos = a.positions ? a.positions[row] : p.pos;
  float y[J];
#pragma unroll
  for (int j = 0; j < J; ++j) {
    // the pair's other value, from lane other % 64 (its dim other / 64 of that lane)
    float partner = __shfl(x[0], other[j] & 63, 64);
    if constexpr (J == 2) {
      const float p1 = __shfl(x[1], other[j] & 63, 64);
      partner = other[j] >= 64 ? p1 : partner;
    }
    const int d = lane + 64 * j;
    const float2 cs = rope_factors(pos, freq[j], a.rope_scale);
    const bool first = a.inter ? !(d & 1) : d < half;
    y[j] = turns[j] ? fmaf(x[j], cs.x, (first ? -partner : partner) * cs.y) : x[j];
  }
  uint16_t* dst;
  if (is_q) {
    dst = a.q_out + ((int64_t)row * a.Hq + hh) * D;
  } else {
    if (p.slot < 0) return;
    dst = a.pool.k + (int64_t)p.slot * a.pool.k_ss + (int64_t)(hh - a.Hq) * a.pool.k_hs + p.off * D;
  }
#pragma unroll
  for (int j = 0; j < J; ++j) dst[lane + 64 * j] = f2h(y[j]);
}

// Sum over the LANES (8 or 16) neighbouring lanes of a row, in all of them.
template <int LANES>
__device__ __forceinline__ float row_sum(float v) {
  auto with = [&](auto ctrl) {
    v += __int_as_float(__builtin_amdgcn_update_dpp(0, __float_as_int(v), decltype(ctrl)::value, 0xF, 0xF, true));
  };
  with(std::integral_constant<int, 0xB1>{});     // quad_perm [1,0,3,2]
  with(std::integral_constant<int, 0x4E>{});     // quad_perm [2,3,0,1]
  with(std::integral_constant<int, 0x141>{});    // row_half_mirror
  if constexpr (LANES == 16) with(std::integral_constant<int, 0x140>{});   // row_mirror
  return v;
}

// The same for many rows.  Bound by moving qkv once: 3926 rows of 40 + 8 + 8 heads (112 MB) 22 us, with
// inputs in the last-level cache or without, and 22 at the rate of a large copy.  The form above spends its time on a sine, a
// cosine and a 64-bit reduction per element of every head and on a store per V element in a line of
// its own.  Here a workgroup takes 256 / (D / 8) tokens, D / 8 lanes a token, and
//   * of q and k PH heads one after another: a lane holds the same four pairs of each, so their
//     factors are made once and stay in registers and no value changes lanes.  Its 8 dims are two
//     groups of 4: at 4 l and r/2 + 4 l of the r rotated dims (r a multiple of 8), behind them, or
//     with interleaved pairs everywhere, 8 neighbours.
//   * of v kVH heads of 16 tokens that lie in one page from a multiple of 16 on (whatever rows they
//     are), turned through LDS: V pages are [D][P], and 32 bytes of a dim written by two workgroups
//     are two partial writes of two L2s (the rows' own blocks of 16, in 2-byte stores, take 1 us more)
// q, K and V are stored non-temporally: the 3926 rows 25 us warm and 32 cold with plain stores.  An
// attention over them right after takes about as much back at up to 4000 rows (append and attention of
// 4 x 256 rows after 200 39.6 -> 38.9 us, 4 x 1000 99 -> 101), but not at 8000 (16 x 500 after 300 203 -> 194).
constexpr int kVH = 8;
constexpr int kPad = 2;                  // halves between the tokens of a head's V in LDS

// The want-th block of 16 positions that holds new tokens: its sequence's first row and position,
// the positions [lo, hi) of it that are new, and the slot (-1: none); false where there are fewer.
struct VBlock {
  int row, slot, at, lo, hi;             // position p is row `row + p`; the block begins at `at`
};
__device__ __forceinline__ bool v_block(const RopeArgs& a, int want, VBlock& v) {
  const int lane = threadIdx.x & 63;
  uint32_t before = 0;
  for (int i0 = 0; i0 < a.B; i0 += 64) {
    const int i = min(i0 + lane, a.B - 1);
    int s0 = i, e = i + 1;
    const int len = a.seq_lens[i];
    if (a.q_starts) {
      s0 = a.q_starts[i];
      e = a.q_starts[i + 1];
    }
    const int first = len - (e - s0);    // position of row s0
    // (rows outside qkv and positions outside the table are none)
    const int lo = max(first + max(-s0, 0), 0), hi = (int)min((int64_t)(len - max(e - a.N, 0)), (int64_t)a.max_pages * a.P);
    const uint32_t n = i0 + lane < a.B && e > s0 && hi > lo ? (uint32_t)((hi - 1) / 16 - lo / 16 + 1) : 0u;
    const uint32_t upto = before + wave_scan(n);
    const uint64_t hit = __ballot(upto > (uint32_t)want);
    if (hit) {
      const int l = __ffsll((unsigned long long)hit) - 1;
      v.lo = (int)lane_of((uint32_t)lo, l);
      v.hi = (int)lane_of((uint32_t)hi, l);
      v.row = (int)lane_of((uint32_t)(s0 - first), l);
      v.at = (v.lo / 16 + want - (int)(lane_of(upto, l) - lane_of(n, l))) * 16;
      const int s = a.page_table[(int64_t)(i0 + l) * a.pt_stride + v.at / a.P];
      v.slot = s >= 0 && s < a.pool.num_slots ? s : -1;
      v.lo = max(v.lo, v.at);
      v.hi = min(v.hi, v.at + 16);
      return true;
    }
    before = lane_of(upto, 63);
  }
  return false;
}

template <int D>
__device__ __forceinline__ void v_tile(const RopeArgs& a, int block, int h0, uint16_t* s_v) {
  constexpr int RL = D / 8;              // lanes of a token
  constexpr int kIter = 16 * kVH * RL / 256;
  const int tid = threadIdx.x;
  VBlock v;
  if (!v_block(a, block, v) || v.slot < 0) return;
  const int nh = min(kVH, a.Hkv - h0);
  uint4 x[kIter];
#pragma unroll
  for (int i = 0; i < kIter; ++i) {
    const int c = i * 256 + tid, h = min(c / (16 * RL), nh - 1), p = min(max(v.at + c / RL % 16, v.lo), v.hi - 1);
    x[i] = ld_nt16(a.qkv + (int64_t)(v.row + p) * a.qkv_st + (int64_t)(a.Hq + a.Hkv + h0 + h) * D + c % RL * 8);
  }
#pragma unroll
  for (int i = 0; i < kIter; ++i) {
    const int c = i * 256 + tid;
    uint32_t* dst = reinterpret_cast<uint32_t*>(s_v + c / RL * (D + kPad) + c % RL * 8);
    dst[0] = x[i].x;
    dst[1] = x[i].y;
    dst[2] = x[i].z;
    dst[3] = x[i].w;
  }
  __syncthreads();
  uint16_t* base = a.pool.v + (int64_t)v.slot * a.pool.v_ss + (int64_t)h0 * a.pool.v_hs + v.at % a.P;
  // neighbouring lanes: the two halves of a dim's 16 tokens, then the next dim
  const int t0 = (tid & 1) * 8;
  const bool whole = v.lo <= v.at + t0 && v.hi >= v.at + t0 + 8;
#pragma unroll 2
  for (int i = tid >> 1; i < nh * D; i += 128) {
    const int h = i / D, d = i % D;
    const uint16_t* src = s_v + (h * 16 + t0) * (D + kPad) + d;
    uint16_t* dst = base + (int64_t)h * a.pool.v_hs + (int64_t)d * a.pool.v_ds + t0;
    uint16_t y[8];
#pragma unroll
    for (int e = 0; e < 8; ++e) y[e] = src[e * (D + kPad)];
    if (whole) {
      st_nt16(dst, make_uint4(y[0] | (uint32_t)y[1] << 16, y[2] | (uint32_t)y[3] << 16,
                              y[4] | (uint32_t)y[5] << 16, y[6] | (uint32_t)y[7] << 16));
    } else {
#pragma unroll
      for (int e = 0; e < 8; ++e)
        if (v.at + t0 + e >= v.lo && v.at + t0 + e < v.hi) dst[e] = y[e];
    }
  }
}

// The first v_items workgroups are those of v.
template <int D, int PH>
__global__ __launch_bounds__(256, 4) void rope_tile_kernel(RopeArgs a, int v_items, int qk_tiles) {
  constexpr int RL = D / 8;
  constexpr int PT = 256 / RL;           // tokens of a workgroup
  __shared__ int s_cnt[4][PT];
  __shared__ Place s_place[PT];
  __shared__ __attribute__((aligned(16))) uint16_t s_v[kVH * 16 * (D + kPad)];
  if ((int)blockIdx.x < v_items) {
    const int groups = (a.Hkv + kVH - 1) / kVH;
    v_tile<D>(a, (int)(blockIdx.x / (unsigned)groups), (int)(blockIdx.x % (unsigned)groups) * kVH, s_v);
    return;
  }
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
  const int li = tid % RL, lt = tid / RL;
  const int x = (int)blockIdx.x - v_items, group = x / qk_tiles;
  const int row0 = (x - group * qk_tiles) * PT, nt = min(PT, a.N - row0);
  const int h0 = group * PH, nh = min(PH, a.Hq + a.Hkv - h0);
  const int half = a.rot / 2;
  int dA = li * 8, dB = dA + 4;
  if (!a.inter && li < a.rot / 8) dA = li * 4, dB = half + li * 4;
  const uint16_t* src = a.qkv + (int64_t)(row0 + min(lt, nt - 1)) * a.qkv_st + (int64_t)h0 * D;
  constexpr int kAhead = PH < 8 ? PH : 8;  // heads on the way
  uint2 rA[kAhead], rB[kAhead];
  auto load = [&](int i, int h) {
    rA[i] = *reinterpret_cast<const uint2*>(src + (int64_t)min(h, nh - 1) * D + dA);
    rB[i] = *reinterpret_cast<const uint2*>(src + (int64_t)min(h, nh - 1) * D + dB);
  };
#pragma unroll
  for (int i = 0; i < kAhead; ++i) load(i, i);
  uint2 wq[2], wk[2];
  float freq[4];
  bool turn[4];                          // the lane's pairs 4 li + e: (dA + e, dB + e), or neighbours
#pragma unroll
  for (int e = 0; e < 4; ++e) {
    turn[e] = (a.inter || li < a.rot / 8) && li * 4 + e < half;
    freq[e] = turn[e] ? a.inv_freq[li * 4 + e] : 0.f;
  }
  if (a.q_norm_w) {
    wq[0] = *reinterpret_cast<const uint2*>(a.q_norm_w + dA);
    wq[1] = *reinterpret_cast<const uint2*>(a.q_norm_w + dB);
    wk[0] = *reinterpret_cast<const uint2*>(a.k_norm_w + dA);
    wk[1] = *reinterpret_cast<const uint2*>(a.k_norm_w + dB);
  }
  if (a.q_starts) {                      // how many sequences end at or before each row
    int cnt = 0;                         // lane t: of row0 + t
    for (int i0 = wave * 64; i0 < a.B; i0 += 256) {
      const int e = i0 + lane < a.B ? a.q_starts[i0 + lane + 1] : 0x7fffffff;
#pragma unroll 8
      for (int t = 0; t < PT; ++t) {
        const int c = __popcll(__ballot(e <= row0 + t));
        cnt += lane == t ? c : 0;
      }
    }
    if (lane < PT) s_cnt[wave][lane] = cnt;
    __syncthreads();
  }
  if (tid < PT) {
    const int row = row0 + tid;
    int b = row;
    if (a.q_starts) b = s_cnt[0][tid] + s_cnt[1][tid] + s_cnt[2][tid] + s_cnt[3][tid];
    Place p{-1, 0, -1, 0};
    if (tid < nt) {
      p = place_of(a, row, b);
      if (a.positions) p.pos = a.positions[row];
    }
    s_place[tid] = p;
  }
  __syncthreads();
  const Place p = s_place[lt];
  float2 cs[4];
#pragma unroll
  for (int e = 0; e < 4; ++e) cs[e] = rope_factors(p.pos, freq[e], a.rope_scale);
  uint16_t* kdst = a.pool.k + (int64_t)max(p.slot, 0) * a.pool.k_ss + p.off * D;
  uint16_t* qdst = a.q_out + (int64_t)(row0 + lt) * a.Hq * D;
#pragma unroll 1
  for (int h8 = 0; h8 < nh; h8 += kAhead) {
#pragma unroll
    for (int i = 0; i < kAhead; ++i) {
      const int h = h0 + h8 + i;
      const bool is_q = h < a.Hq;
      float x[8] = {lo_h(rA[i].x), hi_h(rA[i].x), lo_h(rA[i].y), hi_h(rA[i].y),
                    lo_h(rB[i].x), hi_h(rB[i].x), lo_h(rB[i].y), hi_h(rB[i].y)};
      if (h8 + kAhead < nh) load(i, h8 + kAhead + i);
      if (a.q_norm_w) {
        float ss = 0.f;
#pragma unroll
        for (int e = 0; e < 8; ++e) ss = fmaf(x[e], x[e], ss);
        const float rstd = rsqrtf(row_sum<RL>(ss) / (float)D + a.eps);
#pragma unroll
        for (int g = 0; g < 2; ++g) {
          const uint32_t w0 = is_q ? wq[g].x : wk[g].x, w1 = is_q ? wq[g].y : wk[g].y;
          x[4 * g] = x[4 * g] * rstd * lo_h(w0);
          x[4 * g + 1] = x[4 * g + 1] * rstd * hi_h(w0);
          x[4 * g + 2] = x[4 * g + 2] * rstd * lo_h(w1);
          x[4 * g + 3] = x[4 * g + 3] * rstd * hi_h(w1);
        }
      }
      float y[8];
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        const float u = a.inter ? x[2 * e] : x[e], v = a.inter ? x[2 * e + 1] : x[4 + e];
        const float yu = turn[e] ? fmaf(u, cs[e].x, -v * cs[e].y) : u, yv = turn[e] ? fmaf(v, cs[e].x, u * cs[e].y) : v;
        if (a.inter) {
          y[2 * e] = yu;
          y[2 * e + 1] = yv;
        } else {
          y[e] = yu;
          y[4 + e] = yv;
        }
      }
      const uint2 oA = make_uint2(pack_h2(y[0], y[1]), pack_h2(y[2], y[3]));
      const uint2 oB = make_uint2(pack_h2(y[4], y[5]), pack_h2(y[6], y[7]));
      if (lt >= nt || h8 + i >= nh) continue;
      if (is_q) {
        if (p.seq < 0) continue;
        st_nt8(qdst + h * D + dA, oA.x, oA.y);
        st_nt8(qdst + h * D + dB, oB.x, oB.y);
      } else if (p.slot >= 0) {
        st_nt8(kdst + (int64_t)(h - a.Hq) * a.pool.k_hs + dA, oA.x, oA.y);
        st_nt8(kdst + (int64_t)(h - a.Hq) * a.pool.k_hs + dB, oB.x, oB.y);
      }
    }
  }
}

// (row, head) rows from which the tile form is the faster one (us against the form above): 40 + 8 + 8 heads of
// 128 5600 rows 5.5 / 5.3, 6384 5.6 / 5.6, 8176 5.7 / 6.2; 16 + 1 + 1 of 128 5598 5.5 / 5.3, 6390 5.5 / 5.7; 16 + 8
// + 8 of 64 8160 5.7 / 5.1, 9600 5.8 / 5.7, 12000 5.8 / 6.4.  Half pairs of r dims that are no multiple of 8 stay
// in the form above at any size: 4000 rows of 40 + 8 + 8 heads 90 us at r = 26 or 36 and 99 at 100, where r = 32
// takes 27, 128 21 and interleaved pairs of any r 27.
constexpr int64_t tile_rows(int D) { return D == 128 ? 6000 : 9000; }

// ── pages moved inside a pool ────────────────────────────────────────────────

// A page's bytes in 16-byte chunks, E elements each: K [Hkv][P * D], V [Hkv][D][P] and for pages
// of codes both scales [Hkv][P] (fp16).
struct PageArgs {
  uint8_t* k;
  uint8_t* v;
  uint8_t* ks;
  uint8_t* vs;
  int64_t k_ss, k_hs, v_ss, v_hs, v_ds, s_ss;   // bytes
  int64_t num_slots;
  const int32_t* src;
  const int32_t* dst;
  int n, Hkv;
  int k_chunks, v_dim_chunks, v_chunks;         // of a head's K, of a dim's V, of a head's V
  int s_chunks;                                 // of a page's K scales (0: none)
  // fork
  const int32_t* table;
  int64_t t_stride;
  const int32_t* lens;
  const int32_t* parents;
  const int32_t* fresh;
  int32_t* table_out;
  int64_t o_stride;
  int32_t* lens_out;
  int B, cols, P;
};

__device__ __forceinline__ int page_chunks(const PageArgs& a) {
  return a.Hkv * (a.k_chunks + a.v_chunks) + 2 * a.s_chunks;
}
// Chunk c of page `slot`.
__device__ __forceinline__ uint8_t* chunk_at(const PageArgs& a, int64_t slot, int c) {
  const int nk = a.Hkv * a.k_chunks, nv = a.Hkv * a.v_chunks;
  if (c < nk) return a.k + slot * a.k_ss + (int64_t)(c / a.k_chunks) * a.k_hs + (int64_t)(c % a.k_chunks) * 16;
  c -= nk;
  if (c < nv) {
    const int h = c / a.v_chunks, r = c % a.v_chunks;
    return a.v + slot * a.v_ss + (int64_t)h * a.v_hs + (int64_t)(r / a.v_dim_chunks) * a.v_ds +
           (int64_t)(r % a.v_dim_chunks) * 16;
  }
  c -= nv;
  return (c < a.s_chunks ? a.ks : a.vs) + slot * a.s_ss + (int64_t)(c < a.s_chunks ? c : c - a.s_chunks) * 16;
}
// U chunks of a thread, all requested before the first is stored.
template <int U>
__device__ __forceinline__ void copy_part(const PageArgs& a, int64_t from, int64_t to, int part) {
  const int all = page_chunks(a);
  uint4 x[U];
#pragma unroll
  for (int u = 0; u < U; ++u) {
    const int c = (part * U + u) * 256 + threadIdx.x;
    if (c < all) x[u] = ld_nt16(chunk_at(a, from, c));
  }
#pragma unroll
  for (int u = 0; u < U; ++u) {
    const int c = (part * U + u) * 256 + threadIdx.x;
    if (c >= all) continue;
    if (U > 1) st_nt16(chunk_at(a, to, c), x[u]);
    else *reinterpret_cast<uint4*>(chunk_at(a, to, c)) = x[u];
  }
}

template <int U>
__global__ __launch_bounds__(256) void copy_pages_kernel(PageArgs a) {
  const int parts = (page_chunks(a) + 256 * U - 1) / (256 * U);
  const int i = blockIdx.x / parts, part = blockIdx.x - i * parts;
  const int64_t s = a.src[i], d = a.dst[i];
  if (s < 0 || s >= a.num_slots || d < 0 || d >= a.num_slots || s == d) return;
  copy_part<U>(a, s, d, part);
}

// Workgroup (child, part): part 0 writes the child's row and length, the others copy pieces of
// the page that it goes on in.
template <int U>
__global__ __launch_bounds__(256) void fork_pages_kernel(PageArgs a) {
  const int parts = (page_chunks(a) + 256 * U - 1) / (256 * U) + 1;
  const int i = blockIdx.x / parts, part = blockIdx.x - i * parts;
  const int p = a.parents[i], f = a.fresh[i];
  const bool some = p >= 0 && p < a.B;
  const int32_t* row = a.table + (int64_t)(some ? p : 0) * a.t_stride;
  const int len = some ? (int)min((int64_t)max(a.lens[p], 0), (int64_t)a.cols * a.P) : 0;
  const int full = len / a.P;
  if (part == 0) {
    for (int c = threadIdx.x; c < a.cols; c += 256) {
      const int x = some ? row[c] : -1;
      a.table_out[(int64_t)i * a.o_stride + c] = !some || f < 0 || c < full ? x : c == full ? f : -1;
    }
    if (threadIdx.x == 0) a.lens_out[i] = len;
    return;
  }
  if (!some || f < 0 || f >= a.num_slots || len % a.P == 0) return;
  const int64_t s = row[full];
  if (s < 0 || s >= a.num_slots || s == f) return;
  copy_part<U>(a, s, f, part - 1);
}

// Chunks of a thread: one while all its workgroups are in flight at once (5 pages of 64 KiB 2.4 us), four
// for more, stored non-temporally: 2048 pages with nothing in the last-level cache 55 us, with plain stores 58;
// where it holds both sides 53 against 45, but 512 pages 13.4 against 14.8.
template <typename Go>
void by_width(int64_t chunks, Go go) {
  if (chunks <= 256 * 1024) go(std::integral_constant<int, 1>{});
  else go(std::integral_constant<int, 4>{});
}

int check_pool(const helm_kv_pool* pool, int Hkv, int D, int P, const char* fn) {
  const std::string f(fn);
  HELM_CHECK_ARG(pool && pool->k && pool->v, f + ": null pool pointer");
  HELM_CHECK_ARG(Hkv >= 1, f + ": sizes must be positive");
  HELM_CHECK_SUPPORTED(D == 64 || D == 128, f + ": head_dim must be 64 or 128");
  HELM_CHECK_SUPPORTED(P == 16 || P == 32 || P == 64, f + ": page size must be 16, 32 or 64");
  HELM_CHECK_ARG(pool->num_slots >= 1 && pool->k_head_stride >= (int64_t)P * D && pool->v_dim_stride >= P &&
                     pool->v_head_stride >= P,
                 f + ": pool strides too small for the page");
  HELM_CHECK_SUPPORTED(pool->k_slot_stride % 8 == 0 && pool->k_head_stride % 8 == 0 && pool->v_slot_stride % 8 == 0 &&
                           pool->v_head_stride % 8 == 0 && pool->v_dim_stride % 8 == 0,
                       f + ": pool strides must be multiples of 8 elements");
  HELM_CHECK_SUPPORTED(helm::aligned16(pool->k) && helm::aligned16(pool->v), f + ": pools must be 16-byte aligned");
  return HELM_OK;
}

PageArgs pages_of(const helm_kv_pool* p, int Hkv, int D, int P) {
  PageArgs a{};
  a.k = static_cast<uint8_t*>(p->k); a.v = static_cast<uint8_t*>(p->v);
  a.k_ss = p->k_slot_stride * 2; a.k_hs = p->k_head_stride * 2;
  a.v_ss = p->v_slot_stride * 2; a.v_hs = p->v_head_stride * 2; a.v_ds = p->v_dim_stride * 2;
  a.num_slots = p->num_slots;
  a.Hkv = Hkv; a.P = P;
  a.k_chunks = P * D / 8; a.v_dim_chunks = P / 8; a.v_chunks = P * D / 8;
  return a;
}
PageArgs pages_of(const helm_kv_pool_q8* p, int Hkv, int D, int P) {
  PageArgs a{};
  a.k = static_cast<uint8_t*>(p->k); a.v = static_cast<uint8_t*>(p->v);
  a.ks = static_cast<uint8_t*>(p->k_scale); a.vs = static_cast<uint8_t*>(p->v_scale);
  a.k_ss = a.v_ss = p->slot_stride; a.k_hs = a.v_hs = (int64_t)P * D; a.v_ds = P;
  a.s_ss = p->scale_slot_stride * 2;
  a.num_slots = p->num_slots;
  a.Hkv = Hkv; a.P = P;
  a.k_chunks = P * D / 16; a.v_dim_chunks = P / 16; a.v_chunks = P * D / 16;
  a.s_chunks = Hkv * P / 8;
  return a;
}
int chunks_of(const PageArgs& a) { return a.Hkv * (a.k_chunks + a.v_chunks) + 2 * a.s_chunks; }

int copy_launch(PageArgs a, const int32_t* src, const int32_t* dst, int n, const char* fn, void* stream) {
  const std::string f(fn);
  HELM_CHECK_ARG(src && dst, f + ": null pointer");
  HELM_CHECK_ARG(n >= 1, f + ": sizes must be positive");
  const int64_t all = chunks_of(a);
  HELM_CHECK_SUPPORTED((int64_t)n * ((all + 255) / 256) < (1ll << 31), f + ": too many pages");
  a.src = src; a.dst = dst; a.n = n;
  by_width(all * n, [&](auto u) {
    constexpr int U = decltype(u)::value;
    hipLaunchKernelGGL((copy_pages_kernel<U>), dim3((unsigned)((all + 256 * U - 1) / (256 * U) * n)), dim3(256), 0,
                       static_cast<hipStream_t>(stream), a);
  });
  HELM_CHECK_LAUNCH(fn);
  return HELM_OK;
}

int fork_launch(PageArgs a, const int32_t* table, int64_t t_stride, const int32_t* lens, int B, const int32_t* parents,
                const int32_t* fresh, int32_t* table_out, int64_t o_stride, int32_t* lens_out, int n, int cols,
                const char* fn, void* stream) {
  const std::string f(fn);
  HELM_CHECK_ARG(table && lens && parents && fresh && table_out && lens_out, f + ": null pointer");
  HELM_CHECK_ARG(n >= 1 && B >= 1 && cols >= 1, f + ": sizes must be positive");
  HELM_CHECK_ARG((B == 1 || t_stride >= cols) && (n == 1 || o_stride >= cols), f + ": page-table stride < max_pages");
  HELM_CHECK_SUPPORTED((int64_t)cols * a.P <= (int64_t)1 << 30, f + ": page table covers too many tokens");
  const int64_t all = chunks_of(a);
  HELM_CHECK_SUPPORTED((int64_t)n * ((all + 255) / 256 + 1) < (1ll << 31), f + ": too many rows");
  a.table = table; a.t_stride = t_stride; a.lens = lens; a.B = B; a.parents = parents; a.fresh = fresh;
  a.table_out = table_out; a.o_stride = o_stride; a.lens_out = lens_out; a.n = n; a.cols = cols;
  by_width(all * n, [&](auto u) {
    constexpr int U = decltype(u)::value;
    hipLaunchKernelGGL((fork_pages_kernel<U>), dim3((unsigned)(((all + 256 * U - 1) / (256 * U) + 1) * n)), dim3(256),
                       0, static_cast<hipStream_t>(stream), a);
  });
  HELM_CHECK_LAUNCH(fn);
  return HELM_OK;
}

}  // namespace

extern "C" int helm_rope_append(const void* qkv, int64_t qkv_stride_t, const void* q_norm_w, const void* k_norm_w,
                                float eps, const int32_t* page_table, int64_t pt_stride, int max_pages,
                                const int32_t* seq_lens, const int32_t* q_starts, const int32_t* positions,
                                const float* inv_freq, int rotary_dim, int interleaved, float rope_scale, void* q_out,
                                const helm_kv_pool* pool, int N, int B, int Hq, int Hkv, int D, int P, void* stream) {
  const std::string f("helm_rope_append");
  HELM_CHECK_ARG(qkv && page_table && seq_lens && q_out && (inv_freq || rotary_dim == 0), f + ": null pointer");
  HELM_CHECK_ARG((q_norm_w == nullptr) == (k_norm_w == nullptr), f + ": both norm weights or neither");
  HELM_CHECK_ARG(N >= 1 && B >= 1 && Hq >= 1 && Hkv >= 1 && max_pages >= 0, f + ": sizes must be positive");
  HELM_CHECK_ARG(q_starts || N == B, f + ": without q_starts there is one row per sequence");
  if (const int rc = check_pool(pool, Hkv, D, P, "helm_rope_append")) return rc;
  HELM_CHECK_ARG(rotary_dim >= 0 && rotary_dim <= D && rotary_dim % 2 == 0, f + ": rotary_dim must be even and at most D");
  HELM_CHECK_ARG(B == 1 || pt_stride >= max_pages, f + ": page-table stride < max_pages");
  HELM_CHECK_ARG(qkv_stride_t >= (int64_t)(Hq + 2 * Hkv) * D || N == 1, f + ": rows of qkv overlap");
  HELM_CHECK_SUPPORTED(qkv_stride_t % 8 == 0 && helm::aligned16(qkv) && helm::aligned16(q_out) &&
                           helm::aligned16(q_norm_w) && helm::aligned16(k_norm_w),
                       f + ": qkv rows, norm weights and q_out must be 16-byte aligned");
  HELM_CHECK_SUPPORTED(Hq <= 65535 && Hkv <= 65535 && (int64_t)N * (Hq + 2 * Hkv) < (1ll << 31),
                       f + ": too many rows or heads");
  RopeArgs a{};
  a.qkv = static_cast<const uint16_t*>(qkv); a.qkv_st = qkv_stride_t;
  a.q_norm_w = static_cast<const uint16_t*>(q_norm_w); a.k_norm_w = static_cast<const uint16_t*>(k_norm_w);
  a.eps = eps;
  a.page_table = page_table; a.pt_stride = pt_stride; a.seq_lens = seq_lens; a.q_starts = q_starts;
  a.positions = positions; a.inv_freq = inv_freq; a.rope_scale = rope_scale;
  a.q_out = static_cast<uint16_t*>(q_out);
  a.pool = {static_cast<uint16_t*>(pool->k), pool->k_slot_stride, pool->k_head_stride,
            static_cast<uint16_t*>(pool->v), pool->v_slot_stride, pool->v_head_stride, pool->v_dim_stride,
            pool->num_slots};
  a.N = N; a.B = B; a.Hq = Hq; a.Hkv = Hkv; a.P = P; a.max_pages = max_pages; a.rot = rotary_dim;
  a.inter = interleaved != 0;
  const hipStream_t s = static_cast<hipStream_t>(stream);
  const int64_t rows = (int64_t)N * (Hq + 2 * Hkv);
  const bool tiles = rows >= tile_rows(D) && (a.inter || rotary_dim % 8 == 0);
  auto go = [&](auto d_tag) {
    constexpr int Dc = decltype(d_tag)::value;
    if (tiles) {
      constexpr int pt = 256 / (Dc / 8);
      const int qk_tiles = (N + pt - 1) / pt;
      // a sequence's n tokens lie in at most n / 16 + 2 blocks
      const int64_t v_items = ((int64_t)N / 16 + 2 * (int64_t)std::min(B, N)) * ((Hkv + kVH - 1) / kVH);
      auto run = [&](auto ph_tag) {
        constexpr int PH = decltype(ph_tag)::value;
        const int groups = (Hq + Hkv + PH - 1) / PH;
        hipLaunchKernelGGL((rope_tile_kernel<Dc, PH>), dim3((unsigned)(v_items + (int64_t)qk_tiles * groups)), dim3(256), 0,
                           s, a, (int)v_items, qk_tiles);
      };
      // Heads of a workgroup: 16 make the factors least often, but are a chain; fewer where the chip has
      // places left.  us with 4 / 8 / 16, 40 + 8 + 8 heads of 128: 300 rows (57 workgroups of 16) 6.5 / 8.4 / 11.5,
      // 1024 (192) 10.4 / 10.0 / 12.8, 2048 (384) 15.8 / 14.1 / 15.3, 3000 (564) 21.7 / 20.6 / 18.8
      const int64_t wide = (int64_t)qk_tiles * ((Hq + Hkv + 15) / 16);
      if (wide >= 512) run(std::integral_constant<int, 16>{});
      else if (wide >= 192) run(std::integral_constant<int, 8>{});
      else run(std::integral_constant<int, 4>{});
    } else {
      hipLaunchKernelGGL((rope_rows_kernel<Dc>), dim3((unsigned)((rows + 3) / 4)), dim3(256), 0, s, a);
    }
  };
  if (D == 64) go(std::integral_constant<int, 64>{});
  else go(std::integral_constant<int, 128>{});
  HELM_CHECK_LAUNCH("helm_rope_append launch");
  return HELM_OK;
}

extern "C" int helm_copy_pages(const helm_kv_pool* pool, const int32_t* src, const int32_t* dst, int n, int Hkv, int D,
                               int P, void* stream) {
  if (const int rc = check_pool(pool, Hkv, D, P, "helm_copy_pages")) return rc;
  return copy_launch(pages_of(pool, Hkv, D, P), src, dst, n, "helm_copy_pages", stream);
}

extern "C" int helm_copy_pages_q8(const helm_kv_pool_q8* pool, const int32_t* src, const int32_t* dst, int n, int Hkv,
                                  int D, int P, void* stream) {
  HELM_CHECK_ARG(Hkv >= 1, "helm_copy_pages_q8: sizes must be positive");
  if (const int rc = helm::check_q8_pool(pool, Hkv, D, P, "helm_copy_pages_q8")) return rc;
  return copy_launch(pages_of(pool, Hkv, D, P), src, dst, n, "helm_copy_pages_q8", stream);
}

extern "C" int helm_fork_pages(const helm_kv_pool* pool, const int32_t* page_table, int64_t pt_stride,
                               const int32_t* seq_lens, int B, const int32_t* parents, const int32_t* fresh,
                               int32_t* table_out, int64_t out_stride, int32_t* lens_out, int n, int max_pages, int Hkv,
                               int D, int P, void* stream) {
  if (const int rc = check_pool(pool, Hkv, D, P, "helm_fork_pages")) return rc;
  return fork_launch(pages_of(pool, Hkv, D, P), page_table, pt_stride, seq_lens, B, parents, fresh, table_out,
                     out_stride, lens_out, n, max_pages, "helm_fork_pages", stream);
}

extern "C" int helm_fork_pages_q8(const helm_kv_pool_q8* pool, const int32_t* page_table, int64_t pt_stride,
                                  const int32_t* seq_lens, int B, const int32_t* parents, const int32_t* fresh,
                                  int32_t* table_out, int64_t out_stride, int32_t* lens_out, int n, int max_pages,
                                  int Hkv, int D, int P, void* stream) {
  HELM_CHECK_ARG(Hkv >= 1, "helm_fork_pages_q8: sizes must be positive");
  if (const int rc = helm::check_q8_pool(pool, Hkv, D, P, "helm_fork_pages_q8")) return rc;
  return fork_launch(pages_of(pool, Hkv, D, P), page_table, pt_stride, seq_lens, B, parents, fresh, table_out,
                     out_stride, lens_out, n, max_pages, "helm_fork_pages_q8", stream);
}
