// paged_attention_q8.hip — paged GQA decode attention over K/V pages of 8-bit codes
// with one fp16 scale per token and kv head.
//
// out[b,h] = softmax(scale * q[b,h] . K_b^T) V_b with K = ck * sk, V = cv * sv.  A
// token's K scale multiplies its score and its V scale its probability, so both
// contractions run on the codes themselves.  Scores: int8 products on the matrix cores,
// K as it lies in memory, q in 24-bit fixed point relative to its head's largest value (three
// bytes, three exact integer products: off by 2^-24 of that value, as fp32 sums are).
// Output: V's codes turned into fp16 (exact), fp32 accumulation.
//
// Bound by streaming the pages once, with the vector ALU close behind: 16384 tokens of 8 heads, D
// 128, 34 MB, take 10 us and 2.2 for the merge, 16 items of up to 12000 35 and 4 (with nothing in them
// 21 together: 1024 workgroups in two rounds, whose first loads do not wait for a length).  One 256-thread
// workgroup per (split, kv head, item), its four waves taking 64-token steps round robin.
// Per step a wave computes
//   S[64 tok x 16 col] = K . Q^T         four 16 x 16 tiles
//   O^T[D x 16]       += V^T . P^T       D / 16 tiles
// Every load of codes is 16 bytes per lane: 16 dims of a token for K, the 16 tokens of a dim
// for V (V pages are stored [D][P]), which takes 64-token steps and this token order inside
// the score tiles: row 4 a + r of tile t is token 16 a + 4 t + r, so that lane group g ends
// with the scores of tokens 16 g .. 16 g + 15, whose V^T it feeds to the second product.
// The 16 columns hold GM >= G = Hq / Hkv query heads R = 16 / GM times over: column c + GM j
// keeps the scores of head c for the j-th R-th of every lane group's tokens only (the
// others' probabilities are 0 in it) and is an online softmax of its own, so no lane
// computes an exponential twice; the R columns of a head meet once, at the end.
// p * sv is split into fp16 hi + lo parts (fp32-level accuracy).  fp16 has too few
// exponents for any sv, so a column keeps the binary exponent e of the largest V scale it
// has met, as it keeps the largest score: the products run on p * sv * 2^(14 - e) and the
// sums are rescaled when e grows.
#include <algorithm>
#include <type_traits>

#include "helm_common.h"

namespace {

constexpr int kThreads = 256;
constexpr int kWaves = 4;
constexpr int kStep = 64;             // tokens per wave step
constexpr int kMaxSplitPages = 4096;  // page-table entries of one split staged in LDS
constexpr int kMinExp = -24;          // exponent of the smallest fp16 number
constexpr float kQUnits = 8323072.f;  // largest |q| of a head in units of its query operand: 127 * 65536
constexpr int kTopExp = 14;           // probabilities reach 2^(kTopExp + 1): below fp16's largest

typedef _Float16 h8_t __attribute__((ext_vector_type(8)));
typedef float f4_t __attribute__((ext_vector_type(4)));
typedef int i4_t __attribute__((ext_vector_type(4)));

__host__ __device__ inline int q8_table_steps(int max_pages, int P) {
  return (int)(((int64_t)max_pages * P + kStep - 1) / kStep);
}

struct Q8Args {
  const uint16_t* q;
  int64_t q_sb, q_sh;
  const uint8_t* k;
  const uint8_t* v;
  const uint16_t* ks;
  const uint16_t* vs;
  int64_t slot_stride, scale_slot_stride;   // elements of a slot's codes / scales
  int64_t num_slots;
  const int32_t* page_table;
  int64_t pt_stride;
  const int32_t* seq_lens;
  float* part_o;
  float* part_ml;
  uint16_t* out;                            // written here when there is one split
  int B, Hq, Hkv, max_pages, num_splits;
  float qk_scale_log2;
};

__device__ __forceinline__ uint4 ld16(const void* p) { return ld_nt16(p); }

// codes 8 h .. 8 h + 7 of a 16-byte piece as fp16 integers
__device__ __forceinline__ h8_t codes8(uint32_t a, uint32_t b) {
  h2_t d[4];
  i8x4_to_h2x2(a, d[0], d[1]);
  i8x4_to_h2x2(b, d[2], d[3]);
  return h8_t{d[0][0], d[0][1], d[1][0], d[1][1], d[2][0], d[2][1], d[3][0], d[3][1]};
}

// 2^x; results below fp32's normal range are 0 (a probability of 2^-126)
__device__ __forceinline__ float exp2_(float x) { return __builtin_amdgcn_exp2f(x); }
__device__ __forceinline__ float pow2(int e) { return __int_as_float((127 + e) << 23); }   // |e| < 127

// One step's codes and the 16 scales of lane group grp's tokens.
template <int D, int NT>
struct KBuf {
  uint4 k[4][D / 64];
  uint32_t s[NT / 2];       // scales of the lane's own NT tokens
};
template <int D, int NT>
struct VBuf {
  uint4 v[D / 16];
  uint32_t s[NT / 2];
};

// NT fp16 numbers (8, 16 or 32 bytes, aligned)
template <int NT>
__device__ __forceinline__ void ld_scales(uint32_t (&o)[NT / 2], const uint16_t* p) {
  if constexpr (NT == 4) {
    const uint2 v = *reinterpret_cast<const uint2*>(p);
    o[0] = v.x;
    o[1] = v.y;
  } else {
#pragma unroll
    for (int h = 0; h < NT / 8; ++h) {
      const uint4 v = *reinterpret_cast<const uint4*>(p + 8 * h);
      o[4 * h] = v.x;
      o[4 * h + 1] = v.y;
      o[4 * h + 2] = v.z;
      o[4 * h + 3] = v.w;
    }
  }
}

// v combined with that of the other lane groups of its column (lanes 16 and 32 apart)
__device__ __forceinline__ float grp_max(float v) {
  const auto a = __builtin_amdgcn_permlane16_swap(__float_as_uint(v), __float_as_uint(v), false, false);
  v = fmaxf(__uint_as_float(a[0]), __uint_as_float(a[1]));
  const auto b = __builtin_amdgcn_permlane32_swap(__float_as_uint(v), __float_as_uint(v), false, false);
  return fmaxf(__uint_as_float(b[0]), __uint_as_float(b[1]));
}
__device__ __forceinline__ uint32_t grp_max(uint32_t v) {
  const auto a = __builtin_amdgcn_permlane16_swap(v, v, false, false);
  v = max((uint32_t)a[0], (uint32_t)a[1]);
  const auto b = __builtin_amdgcn_permlane32_swap(v, v, false, false);
  return max((uint32_t)b[0], (uint32_t)b[1]);
}
// the value N lanes on in its row of 16
template <int N>
__device__ __forceinline__ float row_ror(float v) {
  return __int_as_float(__builtin_amdgcn_update_dpp(0, __float_as_int(v), 0x120 + N, 0xF, 0xF, true));
}

template <int D, int P, int GM>
__global__ __launch_bounds__(kThreads, 2) void paged_attn_q8_kernel(Q8Args a) {
  constexpr int KT = D / 64;
  constexpr int DT = D / 16;
  constexpr int UPP = kStep / P;        // page-table entries of a step
  constexpr int R = 16 / GM;            // columns per head
  constexpr int NT = 16 / R;            // tokens of a lane's column and group

  __shared__ int s_slot[kMaxSplitPages];
  __shared__ __attribute__((aligned(16))) int s_q[3][KT][64][4];   // Q^T operands by lane
  __shared__ float s_m[kWaves][GM], s_l[kWaves][GM];
  __shared__ __attribute__((aligned(16))) float s_o[kWaves][GM][D];

  const int tid = threadIdx.x;
  const int wave = tid >> 6;
  const int lane = tid & 63;
  const int col = lane & 15;
  const int grp = lane >> 4;
  const int head = col % GM, sub = col / GM;
  const int split = blockIdx.x;
  const int hk = blockIdx.y;
  const int b = blockIdx.z;
  const int G = a.Hq / a.Hkv;
  const int S = a.num_splits;

  // q first: loads return in order, and its arithmetic runs while K and V are on the way
  uint4 qw[KT][2];
  {
    const uint16_t* qp = a.q + (int64_t)b * a.q_sb + (int64_t)(hk * G + min(head, G - 1)) * a.q_sh + grp * 16;
#pragma unroll
    for (int kk = 0; kk < KT; ++kk)
#pragma unroll
      for (int h = 0; h < 2; ++h) qw[kk][h] = *reinterpret_cast<const uint4*>(qp + kk * 64 + h * 8);
  }
  const int seq = a.seq_lens[b];
  // The split's steps of the table (its reads do not wait for the length): split + j S
  const int max_steps = q8_table_steps(a.max_pages, P);
  const int n_local = max_steps > split ? (max_steps - 1 - split) / S + 1 : 0;
  const int p_cnt = n_local * UPP;
  const int p_last = max(p_cnt - 1, 0);
  const int32_t* ptab = a.page_table + (int64_t)b * a.pt_stride;
  // The slots of the wave's first step, straight from the table: its loads go out before the
  // staging and q's arithmetic (a wave without a step reads slot 0 and uses nothing of it)
  auto in_pool = [&](int slot) { return (slot >= 0 && slot < a.num_slots) ? slot : 0; };
  const int gk = col >> 2;                      // 16-token block of this lane's score-tile rows
  int first_k = -1, first_v = -1;
  if (n_local > wave) {
    const int pg = (split + wave * S) * UPP;
    first_k = ptab[min(pg + gk * 16 / P, a.max_pages - 1)];
    first_v = ptab[min(pg + grp * 16 / P, a.max_pages - 1)];
  }
  for (int i = tid; i < p_cnt; i += kThreads) {
    const int j = i / UPP;
    const int pg = (split + j * S) * UPP + (i - j * UPP);
    const int slot = pg < a.max_pages ? ptab[pg] : -1;
    s_slot[i] = (slot >= 0 && slot < a.num_slots) ? slot : -1;
  }
  // staged slot of 16-token block g of local step j
  auto entry = [&](int j, int g) { return min(j * UPP + g * 16 / P, p_last); };
  constexpr int64_t kPage = (int64_t)P * D;
  const int tok_in_page = (grp * 16) % P + sub * NT;   // of the lane's own tokens

  auto load_k = [&](KBuf<D, NT>& bf, int slot_k, int slot_s) {
    const uint8_t* kp = a.k + (int64_t)slot_k * a.slot_stride + hk * kPage +
                        ((gk * 16) % P + (col & 3)) * D + grp * 16;
#pragma unroll
    for (int t = 0; t < 4; ++t)
#pragma unroll
      for (int kk = 0; kk < KT; ++kk) bf.k[t][kk] = ld16(kp + t * 4 * D + kk * 64);
    ld_scales<NT>(bf.s, a.ks + (int64_t)slot_s * a.scale_slot_stride + hk * P + tok_in_page);
  };
  auto load_v = [&](VBuf<D, NT>& bf, int slot_v) {
    ld_scales<NT>(bf.s, a.vs + (int64_t)slot_v * a.scale_slot_stride + hk * P + tok_in_page);
    const uint8_t* vp = a.v + (int64_t)slot_v * a.slot_stride + hk * kPage + col * P + (grp * 16) % P;
#pragma unroll
    for (int d = 0; d < DT; ++d) bf.v[d] = ld16(vp + d * 16 * P);
  };
  KBuf<D, NT> kb;
  VBuf<D, NT> vb;
  load_k(kb, in_pool(first_k), in_pool(first_v));
  load_v(vb, in_pool(first_v));
  __builtin_amdgcn_sched_barrier(0);

  // Q^T operands: lane holds q[head][64 kk + 16 grp .. + 15] in units of qs, as three bytes
  // 65536 h + 256 m + l (columns of heads past G repeat the last and are never published).
  // v = 65536 h + 256 m + l with signed bytes: l is byte 0 of v, m byte 1 of v + 128, h byte
  // 2 of v + 128 + 32768.  Each wave makes its share of the 4 KT words, through LDS.
  float qs;
  {
    typedef uint16_t us2_t __attribute__((ext_vector_type(2)));
    us2_t big = {0, 0};
#pragma unroll
    for (int kk = 0; kk < KT; ++kk)
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        const uint32_t w[4] = {qw[kk][h].x, qw[kk][h].y, qw[kk][h].z, qw[kk][h].w};
#pragma unroll
        for (int d = 0; d < 4; ++d) big = __builtin_elementwise_max(big, __builtin_bit_cast(us2_t, w[d] & 0x7fff7fffu));
      }
    const uint32_t top = grp_max((uint32_t)max(big[0], big[1]));   // bits order like values
    const float amax = h2f((uint16_t)top);
    const bool finite = top < 0x7c00u;
    const float inv = finite && top ? kQUnits / amax : 0.f;
    // a q that is not finite makes every score of its head NaN
    qs = (finite ? amax / kQUnits : NAN) * a.qk_scale_log2;
#pragma unroll
    for (int i = 0; i < KT; ++i) {       // word n = wave + 4 i: elements 4 n .. 4 n + 3
      const int kk = i, d = wave;        // (n = 4 kk + d)
      const uint4 w0 = qw[kk][0], w1 = qw[kk][1];
      const uint32_t x0 = (d & 2) ? ((d & 1) ? w1.z : w1.x) : ((d & 1) ? w0.z : w0.x);
      const uint32_t x1 = (d & 2) ? ((d & 1) ? w1.w : w1.y) : ((d & 1) ? w0.w : w0.y);
      const float f[4] = {lo_h(x0), hi_h(x0), lo_h(x1), hi_h(x1)};
      uint32_t l = 0, m = 0, h = 0;
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        const int v = finite ? (int)rintf(f[e] * inv) : 0;
        l |= (uint32_t)(v & 255) << (8 * e);
        m |= (uint32_t)(((v + 128) >> 8) & 255) << (8 * e);
        h |= (uint32_t)(((v + 32896) >> 16) & 255) << (8 * e);
      }
      s_q[0][kk][lane][d] = (int)h;
      s_q[1][kk][lane][d] = (int)m;
      s_q[2][kk][lane][d] = (int)l;
    }
  }
  lds_barrier();   // s_slot, s_q; the first steps' loads stay in flight

  i4_t qb[3][KT];
#pragma unroll
  for (int l = 0; l < 3; ++l)
#pragma unroll
    for (int kk = 0; kk < KT; ++kk) qb[l][kk] = *reinterpret_cast<const i4_t*>(s_q[l][kk][lane]);

  const int64_t tokens = min((int64_t)max(seq, 0), (int64_t)a.max_pages * P);
  const int steps = (int)((tokens + kStep - 1) / kStep);
  const int nsteps = steps > split ? (steps - 1 - split) / S + 1 : 0;
  const int my_steps = nsteps > wave ? (nsteps - 1 - wave) / kWaves + 1 : 0;

  float m_run = -INFINITY, l_run = 0.f;       // of the column (m: same in every lane group)
  int e_run = kMinExp;                        // exponent of its largest V scale
  f4_t o[DT];
#pragma unroll
  for (int d = 0; d < DT; ++d) o[d] = f4_t{0.f, 0.f, 0.f, 0.f};

  // One step; K and V each have one buffer, refilled (more: there is a step after) as soon as
  // it has been read: K arrives during the softmax and V's product, V during the next scores.
  // (Two buffers each, loads two steps ahead, gained nothing: a lone wave takes 1.85 us a step
  // either way, its CU's rate of misses, and the longer start cost 2 us.)
  auto step = [&](int i, auto more) {
    constexpr bool kMore = decltype(more)::value;
    const int j = wave + kWaves * i, jn = j + kWaves;
    const int64_t tv = (int64_t)(split + j * S) * kStep + grp * 16 + sub * NT;
    const bool page_ok = s_slot[entry(j, grp)] >= 0;
    // this lane's NT tokens: the first nvalid are real
    const int nvalid = page_ok ? (int)max((int64_t)0, min((int64_t)NT, tokens - tv)) : 0;
    const bool whole = __all(nvalid == NT);     // no place without a token: nothing to mask
    int v[3][NT];                               // the lane's own tokens: tiles sub * NT / 4 on
#pragma unroll
    for (int t = 0; t < 4; ++t)
#pragma unroll
      for (int l = 0; l < 3; ++l) {
        i4_t c = {0, 0, 0, 0};
#pragma unroll
        for (int kk = 0; kk < KT; ++kk)
          c = __builtin_amdgcn_mfma_i32_16x16x64_i8(__builtin_bit_cast(i4_t, kb.k[t][kk]), qb[l][kk], c, 0, 0, 0);
#pragma unroll
        for (int r = 0; r < 4; ++r) {
          int& d = v[l][(t * 4 + r) % NT];
          d = t < NT / 4 || sub == t / (NT / 4) ? c[r] : d;
        }
      }
    float s[NT];
    float mx = -INFINITY;
#pragma unroll
    for (int e = 0; e < NT; ++e) {
      const float sk = (e & 1) ? hi_h(kb.s[e / 2]) : lo_h(kb.s[e / 2]);
      s[e] = fmaf((float)v[0][e], 65536.f, (float)((v[1][e] << 8) + v[2][e])) * (sk * qs);
    }
    if (!whole) {                               // codes and scales there may be any bits
#pragma unroll
      for (int e = 0; e < NT; ++e) s[e] = e < nvalid ? s[e] : -INFINITY;
    }
    if constexpr (kMore) {
      load_k(kb, max(s_slot[entry(jn, gk)], 0), max(s_slot[entry(jn, grp)], 0));
      __builtin_amdgcn_sched_barrier(0);
    }
#pragma unroll
    for (int e = 0; e < NT; ++e) mx = fmaxf(mx, s[e]);
    uint32_t vsw[NT / 2];
#pragma unroll
    for (int q = 0; q < NT / 2; ++q) vsw[q] = vb.s[q];
    if (!whole) {
#pragma unroll
      for (int q = 0; q < NT / 2; ++q)
        vsw[q] &= (2 * q < nvalid ? 0x0000ffffu : 0u) | (2 * q + 1 < nvalid ? 0xffff0000u : 0u);
    }
    typedef uint16_t us2_t __attribute__((ext_vector_type(2)));
    us2_t big = {0, 0};
#pragma unroll
    for (int q = 0; q < NT / 2; ++q)
      big = __builtin_elementwise_max(big, __builtin_bit_cast(us2_t, vsw[q] & 0x7fff7fffu));
    const uint32_t top = grp_max((uint32_t)max(big[0], big[1]));
    const int e_top = (int)(__float_as_uint(h2f((uint16_t)top)) >> 23) - 127;
    const int e_new = max(e_run, min(e_top, 15));
    const float m_new = fmaxf(m_run, grp_max(mx));
    const float ref = (m_new == -INFINITY) ? 0.f : m_new;   // exp2(-inf - ref) stays 0
    const float alpha = exp2_(m_run - ref);
    const float alpha_o = alpha * pow2(e_run - e_new);
    const float pscale = pow2(kTopExp - e_new);
    uint32_t hi[NT / 2], lo[NT / 2];
    float lsum = 0.f;
#pragma unroll
    for (int q = 0; q < NT / 2; ++q) {
      const float p0 = exp2_(s[2 * q] - ref), p1 = exp2_(s[2 * q + 1] - ref);
      lsum += p0 + p1;
      const float v0 = p0 * (lo_h(vsw[q]) * pscale), v1 = p1 * (hi_h(vsw[q]) * pscale);   // 0 where no token
      hi[q] = pack_h2(v0, v1);
      lo[q] = pack_h2(v0 - lo_h(hi[q]), v1 - hi_h(hi[q]));
    }
    l_run = l_run * alpha + lsum;
    m_run = m_new;
    e_run = e_new;
    // P^T operands: tokens 0-7 and 8-15 of the lane group, 0 but for the column's own
    h8_t ph[2], pl[2];
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      u32x4_t wh, wl;
#pragma unroll
      for (int q = 0; q < 4; ++q) {
        const int at = h * 4 + q;
        const bool own = R == 1 || sub == at / (NT / 2);
        wh[q] = own ? hi[at % (NT / 2)] : 0u;
        wl[q] = own ? lo[at % (NT / 2)] : 0u;
      }
      ph[h] = __builtin_bit_cast(h8_t, wh);
      pl[h] = __builtin_bit_cast(h8_t, wl);
    }
    if (__any(alpha_o != 1.0f)) {               // rare once the largest score has been met
#pragma unroll
      for (int d = 0; d < DT; ++d) o[d] *= alpha_o;
    }
#pragma unroll
    for (int d = 0; d < DT; ++d) {
      const h8_t v0 = codes8(vb.v[d].x, vb.v[d].y), v1 = codes8(vb.v[d].z, vb.v[d].w);
      o[d] = __builtin_amdgcn_mfma_f32_16x16x32_f16(v0, ph[0], o[d], 0, 0, 0);
      o[d] = __builtin_amdgcn_mfma_f32_16x16x32_f16(v1, ph[1], o[d], 0, 0, 0);
      o[d] = __builtin_amdgcn_mfma_f32_16x16x32_f16(v0, pl[0], o[d], 0, 0, 0);
      o[d] = __builtin_amdgcn_mfma_f32_16x16x32_f16(v1, pl[1], o[d], 0, 0, 0);
    }
    if constexpr (kMore) {
      load_v(vb, max(s_slot[entry(jn, grp)], 0));
      __builtin_amdgcn_sched_barrier(0);
    }
  };
  if (my_steps > 0) {
    for (int i = 0; i + 1 < my_steps; ++i) step(i, std::true_type{});
    step(my_steps - 1, std::false_type{});
  }

  // the lane groups' sums, then the R columns of a head, then (through LDS) the waves
  float l = l_run, unscale = pow2(e_run - kTopExp);
  l += __shfl_xor(l, 16, 64);
  l += __shfl_xor(l, 32, 64);
  if constexpr (R > 1) {
    float mh = m_run;
    if constexpr (R == 4) mh = fmaxf(mh, row_ror<4>(mh));
    mh = fmaxf(mh, row_ror<8>(mh));
    const float f = exp2_(m_run - (mh == -INFINITY ? 0.f : mh));
    unscale *= f;
    l *= f;
    if constexpr (R == 4) l += row_ror<4>(l);
    l += row_ror<8>(l);
    m_run = mh;
  }
#pragma unroll
  for (int d = 0; d < DT; ++d) {
    o[d] *= unscale;
#pragma unroll
    for (int r = 0; r < 4; ++r) {
      if constexpr (R == 4) o[d][r] += row_ror<4>(o[d][r]);
      if constexpr (R > 1) o[d][r] += row_ror<8>(o[d][r]);
    }
  }
  if (col < G) {
#pragma unroll
    for (int d = 0; d < DT; ++d)
      *reinterpret_cast<float4*>(&s_o[wave][col][d * 16 + grp * 4]) =
          make_float4(o[d][0], o[d][1], o[d][2], o[d][3]);
    if (grp == 0) {
      s_m[wave][col] = m_run;
      s_l[wave][col] = l;
    }
  }
  __syncthreads();

  for (int idx = tid; idx < G * (D / 4); idx += kThreads) {
    const int g = idx / (D / 4);
    const int d = (idx - g * (D / 4)) * 4;
    float mx = s_m[0][g];
#pragma unroll
    for (int w = 1; w < kWaves; ++w) mx = fmaxf(mx, s_m[w][g]);
    const float ref = (mx == -INFINITY) ? 0.f : mx;
    float num[4] = {0.f, 0.f, 0.f, 0.f}, den = 0.f;
#pragma unroll
    for (int w = 0; w < kWaves; ++w) {
      const float sc = exp2f(s_m[w][g] - ref);
      const float4 ow = *reinterpret_cast<const float4*>(&s_o[w][g][d]);
      num[0] = fmaf(sc, ow.x, num[0]);
      num[1] = fmaf(sc, ow.y, num[1]);
      num[2] = fmaf(sc, ow.z, num[2]);
      num[3] = fmaf(sc, ow.w, num[3]);
      den = fmaf(sc, s_l[w][g], den);
    }
    float4 r = make_float4(0.f, 0.f, 0.f, 0.f);
    // (a NaN sum stays one: only an empty split gives zeros)
    if (!(den <= 0.f)) {
      const float inv = 1.0f / den;
      r = make_float4(num[0] * inv, num[1] * inv, num[2] * inv, num[3] * inv);
    }
    const int64_t bh = (int64_t)b * a.Hq + hk * G + g;
    if (S == 1) {
      *reinterpret_cast<uint2*>(a.out + bh * D + d) = make_uint2(pack_h2(r.x, r.y), pack_h2(r.z, r.w));
    } else {
      const int64_t pidx = bh * S + split;
      *reinterpret_cast<float4*>(&a.part_o[pidx * D + d]) = r;
      if (d == 0) {
        // a NaN goes on in part_o: the merge leaves out splits whose sum is not positive
        a.part_ml[pidx * 2] = den == den ? mx : 0.0f;
        a.part_ml[pidx * 2 + 1] = den == den ? den : 1.0f;
      }
    }
  }
}

template <int D, int P>
void launch_q8(const Q8Args& a, int G, hipStream_t s) {
  const dim3 grid(a.num_splits, a.Hkv, a.B);
  if (G <= 4) hipLaunchKernelGGL((paged_attn_q8_kernel<D, P, 4>), grid, dim3(kThreads), 0, s, a);
  else if (G <= 8) hipLaunchKernelGGL((paged_attn_q8_kernel<D, P, 8>), grid, dim3(kThreads), 0, s, a);
  else hipLaunchKernelGGL((paged_attn_q8_kernel<D, P, 16>), grid, dim3(kThreads), 0, s, a);
}

// Splits of a call: the caller's, or by a rule; more where a split would have to stage more
// page-table entries than it can.  The rule, us with 1 / 2 / 4 / 8 / 16 / 32 / 64 splits:
//   * one split up to 1024 / D steps: a wave's two or three further steps cost less than the
//     merge (2.5 us and a launch).  2 x 300 tokens, D 128: 7.5 / 8.1 / 8.0; 4 x 700, D 64: 6.4 /
//     7.3 / 7.0 / 7.6; but 2000 tokens, D 128: 18.9 / 14.1 / 10.6 / 8.6 / 9.3
//   * else a workgroup per CU, at least a step per wave: 16384 tokens, 8 heads 120 / 65 / 37 / 22.5
//     / 15.7 / 13.0 / 15.8; 32768: .. / 24.8 / 18.9 / 22.6
//   * up to four times as many (to 32, past which the merge is slower) while a split keeps
//     11 steps: the CUs even out between long and short items.  16 items of up to 12000
//     tokens, 8 heads 95 / 57 / 44 / 42 / 49; 3 of 6000, 32 heads 31 / 21 / 19.0 / 18.2 / 19.4; but 8 of
//     4000, 8 heads 36 / 24 / 17.9 / 18.9 / 21.2
int q8_splits(int B, int Hkv, int D, int P, int max_pages, int want) {
  const int64_t steps = q8_table_steps(max_pages, P);
  const int64_t least = (steps + kMaxSplitPages / (kStep / P) - 1) / (kMaxSplitPages / (kStep / P));
  int64_t n = want;
  if (n < 1) {
    n = 1;
    if (steps * D > 1024) {
      n = std::max<int64_t>(1, std::min<int64_t>(256 / std::max<int64_t>(1, (int64_t)B * Hkv), steps / 4));
      for (int i = 0; i < 2 && 2 * n <= 32 && steps >= 11 * 2 * n; ++i) n *= 2;
    }
  }
  return (int)std::min<int64_t>(std::max(std::max<int64_t>(n, 1), least), 1 << 20);
}

}  // namespace

extern "C" int64_t helm_paged_attn_q8_workspace_bytes(int B, int Hq, int Hkv, int D, int P, int max_pages,
                                                      int num_splits) {
  if (B < 1 || Hq < 1 || Hkv < 1 || D < 1 || max_pages < 1 || (P != 16 && P != 32 && P != 64)) return 0;
  const int64_t n = q8_splits(B, Hkv, D, P, max_pages, num_splits);
  return n > 1 ? n * B * Hq * (D + 2) * (int64_t)sizeof(float) : 0;
}

extern "C" int helm_paged_decode_attn_q8(const void* q, int64_t q_stride_b, int64_t q_stride_h,
                                         const helm_kv_pool_q8* pool, const int32_t* page_table,
                                         int64_t pt_stride, const int32_t* seq_lens, void* out, int B, int Hq,
                                         int Hkv, int D, int P, int max_pages, float scale, int num_splits,
                                         void* workspace, int64_t workspace_bytes, void* stream) {
  const std::string f("helm_paged_decode_attn_q8");
  HELM_CHECK_ARG(q && page_table && seq_lens && out, f + ": null pointer");
  HELM_CHECK_ARG(B >= 1 && Hq >= 1 && Hkv >= 1 && max_pages >= 1 && num_splits >= 0, f + ": sizes must be positive");
  HELM_CHECK_ARG(Hq % Hkv == 0, f + ": Hq must be a multiple of Hkv");
  HELM_CHECK_SUPPORTED(Hq / Hkv <= 16, f + ": at most 16 query heads per kv head");
  HELM_CHECK_SUPPORTED(B <= 65535 && Hq <= 65535, f + ": at most 65535 items and heads");
  if (const int rc = helm::check_q8_pool(pool, Hkv, D, P, "helm_paged_decode_attn_q8")) return rc;
  HELM_CHECK_ARG(pt_stride >= max_pages, f + ": page-table stride < max_pages");
  HELM_CHECK_SUPPORTED((int64_t)max_pages * P <= (int64_t)1 << 30, f + ": page table covers too many tokens");
  HELM_CHECK_SUPPORTED(q_stride_h % 8 == 0 && q_stride_b % 8 == 0 && helm::aligned16(q),
                       f + ": q strides must be multiples of 8 and q 16-byte aligned");
  HELM_CHECK_SUPPORTED(reinterpret_cast<uintptr_t>(out) % 8 == 0, f + ": out must be 8-byte aligned");
  const int n = q8_splits(B, Hkv, D, P, max_pages, num_splits);
  const int64_t need = n > 1 ? (int64_t)n * B * Hq * (D + 2) * (int64_t)sizeof(float) : 0;
  HELM_CHECK_ARG(need == 0 || (workspace && helm::aligned16(workspace) && workspace_bytes >= need),
                 f + ": this shape needs " + std::to_string(need) + " bytes of 16-byte aligned workspace");
  Q8Args a{};
  a.q = static_cast<const uint16_t*>(q); a.q_sb = q_stride_b; a.q_sh = q_stride_h;
  a.k = static_cast<const uint8_t*>(pool->k); a.v = static_cast<const uint8_t*>(pool->v);
  a.ks = static_cast<const uint16_t*>(pool->k_scale); a.vs = static_cast<const uint16_t*>(pool->v_scale);
  a.slot_stride = pool->slot_stride; a.scale_slot_stride = pool->scale_slot_stride;
  a.num_slots = pool->num_slots;
  a.page_table = page_table; a.pt_stride = pt_stride; a.seq_lens = seq_lens;
  a.part_o = static_cast<float*>(workspace);
  a.part_ml = a.part_o + (n > 1 ? (int64_t)n * B * Hq * D : 0);
  a.out = static_cast<uint16_t*>(out);
  a.B = B; a.Hq = Hq; a.Hkv = Hkv; a.max_pages = max_pages; a.num_splits = n;
  a.qk_scale_log2 = scale * kLog2e;
  const hipStream_t s = static_cast<hipStream_t>(stream);
  const int G = Hq / Hkv;
  if (D == 64) {
    if (P == 16) launch_q8<64, 16>(a, G, s);
    else if (P == 32) launch_q8<64, 32>(a, G, s);
    else launch_q8<64, 64>(a, G, s);
  } else {
    if (P == 16) launch_q8<128, 16>(a, G, s);
    else if (P == 32) launch_q8<128, 32>(a, G, s);
    else launch_q8<128, 64>(a, G, s);
  }
  HELM_CHECK_LAUNCH("helm_paged_decode_attn_q8 launch");
  if (n == 1) return HELM_OK;
  return helm_paged_attn_reduce(a.part_o, a.part_ml, out, B, Hq, D, n, stream);
}
