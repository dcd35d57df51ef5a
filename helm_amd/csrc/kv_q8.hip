// kv_q8.hip — KV pages of 8-bit codes with one fp16 scale per token and kv head: the
// writes (plain, and with q / k norm and RoPE on the way) and the way back to fp16.
//
// Quantisation of a row x[D]: s = fp16(max |x| / 127), c = rne(x / s) in [-127, 127].
#include <type_traits>

#include "helm_common.h"

namespace helm {

int check_q8_pool(const helm_kv_pool_q8* pool, int Hkv, int D, int P, const char* fn) {
  const std::string f(fn);
  HELM_CHECK_ARG(pool && pool->k && pool->v && pool->k_scale && pool->v_scale, f + ": null pool pointer");
  HELM_CHECK_SUPPORTED(D == 64 || D == 128, f + ": head_dim must be 64 or 128");
  HELM_CHECK_SUPPORTED(P == 16 || P == 32 || P == 64, f + ": page size must be 16, 32 or 64");
  HELM_CHECK_ARG(pool->num_slots >= 1, f + ": num_slots must be positive");
  HELM_CHECK_ARG(pool->slot_stride >= (int64_t)Hkv * P * D && pool->scale_slot_stride >= (int64_t)Hkv * P,
                 f + ": pool strides too small for the page");
  HELM_CHECK_SUPPORTED(pool->slot_stride % 16 == 0 && pool->scale_slot_stride % 8 == 0,
                       f + ": slot strides must be multiples of 16 (codes) and 8 (scales)");
  HELM_CHECK_SUPPORTED(aligned16(pool->k) && aligned16(pool->v) && aligned16(pool->k_scale) &&
                           aligned16(pool->v_scale),
                       f + ": pool pointers must be 16-byte aligned");
  return HELM_OK;
}

}  // namespace helm

namespace {

struct Q8Pool {
  int8_t* k;
  int8_t* v;
  uint16_t* ks;
  uint16_t* vs;
  int64_t slot_stride, scale_slot_stride, num_slots;
};

Q8Pool pool_of(const helm_kv_pool_q8* p) {
  return {static_cast<int8_t*>(p->k), static_cast<int8_t*>(p->v), static_cast<uint16_t*>(p->k_scale),
          static_cast<uint16_t*>(p->v_scale), p->slot_stride, p->scale_slot_stride, p->num_slots};
}

// fp16 scale of a row whose largest magnitude is amax; NaN where the row holds one.
__device__ __forceinline__ uint16_t row_scale(float amax, bool nan) {
  return nan ? (uint16_t)0x7e00 : f2h(amax / 127.0f);
}
// x / s as x * r with r near 1 / s, and one step of its remainder: exact where the quotient
// has few bits (so the halves that round to even are), within an ulp elsewhere.
struct Scale {
  float s, r;
  bool ok;                              // above 0 and finite: otherwise every code is 0
};
__device__ __forceinline__ Scale scale_of(uint16_t bits) {
  Scale c;
  c.s = h2f(bits);
  c.ok = c.s > 0.f && c.s < INFINITY;
  const float r = __builtin_amdgcn_rcpf(c.ok ? c.s : 1.0f);
  c.r = fmaf(fmaf(-c.s, r, 1.0f), r, r);
  return c;
}
// The code is the low byte of the result: 1.5 * 2^23 + z rounds z to a whole number.
__device__ __forceinline__ uint32_t code_of(float x, const Scale& c) {
  const float q = x * c.r;
  const float z = fmaf(fmaf(-q, c.s, x), c.r, q);
  return __float_as_uint(__builtin_amdgcn_fmed3f(z, -127.f, 127.f) + 12582912.0f);
}

// One wave's row, lane holding dims lane + 64 j: scale and codes into the page.
template <int D>
__device__ __forceinline__ void store_row(const float (&x)[D / 64], int lane, bool is_v, const Q8Pool& p,
                                          int64_t slot, int hk, int off, int P) {
  constexpr int J = D / 64;
  float amax = 0.f;
  bool bad = false;
#pragma unroll
  for (int j = 0; j < J; ++j) {
    amax = fmaxf(amax, fabsf(x[j]));
    bad |= x[j] != x[j];
  }
  const uint16_t sh = row_scale(wave_max(amax), __any(bad));
  const Scale s = scale_of(sh);
#pragma unroll
  for (int j = 0; j < J; ++j) {
    const int d = lane + 64 * j;
    const int8_t c = s.ok ? (int8_t)code_of(x[j], s) : (int8_t)0;
    if (is_v) p.v[slot * p.slot_stride + ((int64_t)hk * D + d) * P + off] = c;
    else p.k[slot * p.slot_stride + ((int64_t)hk * P + off) * D + d] = c;
  }
  if (lane == 0) (is_v ? p.vs : p.ks)[slot * p.scale_slot_stride + (int64_t)hk * P + off] = sh;
}

// cos and sin of pos * inv_freq, the angle reduced in 64 bits.
__device__ __forceinline__ void rope_factors(int pos, float inv_freq, float& c, float& s) {
  constexpr double kInvPi = 0.31830988618379067154;
  double t = (double)pos * (double)inv_freq * kInvPi;   // half turns
  t -= 2.0 * rint(0.5 * t);                             // [-1, 1]
  c = cospif((float)t);
  s = sinpif((float)t);
}

// One wave per (token, head): q and k heads normed and rotated, q to q_out, k and v
// quantised into their page.  Latency-bound at a few tokens: 3.6 us for 1 to 32 tokens of 40 + 8 + 8
// heads of 128.
template <int D>
__global__ __launch_bounds__(256) void qk_norm_rope_append_q8_kernel(
    const uint16_t* __restrict__ qkv, int64_t qkv_sb, const uint16_t* __restrict__ q_norm_w,
    const uint16_t* __restrict__ k_norm_w, float eps, const int32_t* __restrict__ positions,
    const float* __restrict__ inv_freq, uint16_t* __restrict__ q_out, Q8Pool pool,
    const int32_t* __restrict__ slots, const int32_t* __restrict__ offsets, int64_t items, int Hq, int Hkv,
    int P) {
  constexpr int J = D / 64, HALF = D / 2;
  const int lane = threadIdx.x & 63;
  const int64_t item = (int64_t)blockIdx.x * 4 + (threadIdx.x >> 6);
  if (item >= items) return;
  const int heads = Hq + 2 * Hkv;
  const int64_t b = item / heads;
  const int hh = (int)(item - b * heads);
  const uint16_t* src = qkv + b * qkv_sb + (int64_t)hh * D;
  float x[J];
#pragma unroll
  for (int j = 0; j < J; ++j) x[j] = h2f(src[lane + 64 * j]);
  if (hh < Hq + Hkv) {
    const uint16_t* nw = hh < Hq ? q_norm_w : k_norm_w;
    if (nw != nullptr) {
      float ss = 0.f;
#pragma unroll
      for (int j = 0; j < J; ++j) ss = fmaf(x[j], x[j], ss);
      const float rstd = rsqrtf(wave_sum(ss) / (float)D + eps);
#pragma unroll
      for (int j = 0; j < J; ++j) x[j] = x[j] * rstd * h2f(nw[lane + 64 * j]);
    }
    float c, s, y[J];
    rope_factors(positions[b], inv_freq[lane % HALF], c, s);
#pragma unroll
    for (int j = 0; j < J; ++j) {
      float partner;
      if constexpr (J == 2) partner = x[1 - j];
      else partner = __shfl_xor(x[j], HALF, 64);
      const float rot = lane + 64 * j < HALF ? -partner : partner;
      y[j] = fmaf(x[j], c, rot * s);
    }
#pragma unroll
    for (int j = 0; j < J; ++j) x[j] = y[j];
    if (hh < Hq) {
#pragma unroll
      for (int j = 0; j < J; ++j) q_out[(b * Hq + hh) * D + lane + 64 * j] = f2h(x[j]);
      return;
    }
  }
  const int slot = slots[b], off = offsets[b];
  if (slot < 0 || slot >= pool.num_slots || off < 0 || off >= P) return;   // uniform per wave
  const bool is_v = hh >= Hq + Hkv;
  store_row<D>(x, lane, is_v, pool, slot, hh - Hq - (is_v ? Hkv : 0), off, P);
}

// The same for a prompt's tokens, and bit for bit (the sum of squares adds in the order of
// wave_sum over lanes d mod 64).  The floor is moving qkv once through HBM (53 MB for 2000
// tokens of 40 + 8 + 8 heads: 11 us at the card's copy rate; this takes 19, its vector
// instructions what is left).  The form above spends its time on a sine, a cosine and a 64-bit
// reduction per element of every head, and on a byte store per V element, each in a line of
// its own.  Here a workgroup takes 16 tokens x 8 heads:
//   * q / k heads: RoPE factors of the 16 tokens once into LDS; a lane holds 8 dims of a row
//     (16-byte loads and stores, D / 8 lanes a row), all rows of a wave requested before the
//     first is used
//   * v heads: 16 tokens of a head are quantised and transposed through LDS; four tokens of a
//     dim that lie next to each other in one page from a multiple of 4 on go out as one word
//     (all 16 at once where they fill an aligned run), the others byte by byte.
constexpr int kPT = 16;               // tokens of a workgroup
constexpr int kPH = 8;                // heads
constexpr int kPW = 8;                // waves
// (token, head) rows from which this is the faster form: D = 128, 14336 rows 7.8 us against 7.5,
// 20480 rows 8.2 against 8.9, 112000 rows (2000 tokens of 40 + 8 + 8) 19 against 38; D = 64, 1536
// rows 4.6 against 3.7, 8192 rows 4.7 against 5.5, 192000 rows 16 against 58.
constexpr int64_t prompt_rows(int D) { return D == 128 ? 16384 : 6144; }

template <int CTRL, int BANKS = 0xF>
__device__ __forceinline__ float dpp_f(float v, float old = 0.f) {
  return __int_as_float(__builtin_amdgcn_update_dpp(__float_as_int(old), __float_as_int(v), CTRL, 0xF, BANKS, BANKS == 0xF));
}
// the value four (eight) lanes on in its eight (sixteen)
__device__ __forceinline__ float xor4(float v) {
  return dpp_f<0x114, 0xA>(v, dpp_f<0x104, 0x5>(v));   // row_shl 4 to lanes 0-3, 8-11, row_shr 4 to the others
}
__device__ __forceinline__ float xor8(float v) { return dpp_f<0x128>(v); }   // row_ror 8

// Largest of the D / 8 lanes of a row (8 or 16 neighbours), in all of them.
template <int D>
__device__ __forceinline__ uint32_t row_max(uint32_t v) {
  auto with = [&](auto ctrl) {
    v = max(v, (uint32_t)__builtin_amdgcn_update_dpp(0, (int)v, decltype(ctrl)::value, 0xF, 0xF, true));
  };
  with(std::integral_constant<int, 0xB1>{});     // quad_perm [1,0,3,2]
  with(std::integral_constant<int, 0x4E>{});     // quad_perm [2,3,0,1]
  with(std::integral_constant<int, 0x141>{});    // row_half_mirror
  if constexpr (D == 128) with(std::integral_constant<int, 0x140>{});   // row_mirror
  return v;
}
// Sum of squares of a row of which lane l holds dims 8 l + e, in the order in which wave_sum
// adds lanes d mod 64 (each with dims d and d + 64): lane bits 5..3 (l's low three) first,
// then 2..0 (e's).  A step over two lanes leaves each of them half of the e's.
template <int D>
__device__ __forceinline__ float row_squares(const float (&x)[8], int l) {
  float a[4];
  if constexpr (D == 128) {             // lanes l < 8 take e 0..3, the others 4..7
    const bool hi = l & 8;
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      const float own = hi ? x[e + 4] : x[e], got = xor8(hi ? x[e] : x[e + 4]);
      const float lo = hi ? got : own, up = hi ? own : got;
      a[e] = fmaf(up, up, lo * lo);
    }
    const bool b2 = l & 4, b1 = l & 2;
    float c[2];
#pragma unroll
    for (int e = 0; e < 2; ++e) c[e] = (b2 ? a[e + 2] : a[e]) + xor4(b2 ? a[e] : a[e + 2]);
    float v = (b1 ? c[1] : c[0]) + dpp_f<0x4E>(b1 ? c[0] : c[1]);
    v += dpp_f<0xB1>(v);
    v += xor8(v);                       // e bits 2, 1, 0
    v += xor4(v);
    return v + dpp_f<0x4E>(v);
  } else {
    const bool b2 = l & 4, b1 = l & 2, b0 = l & 1;
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      const float lo = x[e] * x[e], up = x[e + 4] * x[e + 4];
      a[e] = (b2 ? up : lo) + xor4(b2 ? lo : up);
    }
    float c[2];
#pragma unroll
    for (int e = 0; e < 2; ++e) c[e] = (b1 ? a[e + 2] : a[e]) + dpp_f<0x4E>(b1 ? a[e] : a[e + 2]);
    float v = (b0 ? c[1] : c[0]) + dpp_f<0xB1>(b0 ? c[0] : c[1]);
    v += xor4(v);
    v += dpp_f<0x4E>(v);
    return v + dpp_f<0xB1>(v);
  }
}

template <int D>
__global__ __launch_bounds__(kPW * 64, 8) void qk_norm_rope_append_q8_prompt_kernel(
    const uint16_t* __restrict__ qkv, int64_t qkv_sb, const uint16_t* __restrict__ q_norm_w,
    const uint16_t* __restrict__ k_norm_w, float eps, const int32_t* __restrict__ positions,
    const float* __restrict__ inv_freq, uint16_t* __restrict__ q_out, Q8Pool pool,
    const int32_t* __restrict__ slots, const int32_t* __restrict__ offsets, int B, int Hq, int Hkv, int P) {
  constexpr int HALF = D / 2;
  constexpr int RL = D / 8;             // lanes of a row
  constexpr int RW = 64 / RL;           // rows of a wave at a time
  constexpr int kIter = kPT * kPH / (kPW * RW);   // rows of a lane, neighbouring tokens of one head
  __shared__ float2 s_cs[kPT][8][HALF / 8];   // dim 8 l + e at [e][l]: a row's lanes read neighbours
  __shared__ int s_slot[kPT], s_off[kPT], s_next;   // s_next: bit t is set where token t lies right behind t - 1
  // a dim's tokens, then 4 bytes: the dims of a row's lanes would lie in two banks without them
  __shared__ __attribute__((aligned(16))) int8_t s_v[kPH][D][kPT + 4];
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
  const int li = lane % RL, lr = lane / RL;
  const int b0 = blockIdx.x * kPT, nt = min(kPT, B - b0);
  const int groups_qk = (Hq + Hkv + kPH - 1) / kPH;
  const bool v_heads = (int)blockIdx.y >= groups_qk;
  const int h0 = v_heads ? (blockIdx.y - groups_qk) * kPH : blockIdx.y * kPH;   // of the group's kind
  const int nh = min(kPH, (v_heads ? Hkv : Hq + Hkv) - h0);

  const int t0 = (wave * RW + lr) % (kPT / kIter) * kIter, hi = (wave * RW + lr) / (kPT / kIter), h = h0 + hi;
  uint4 raw[kIter];
#pragma unroll
  for (int i = 0; i < kIter; ++i) {
    const int t = min(t0 + i, nt - 1);
    raw[i] = *reinterpret_cast<const uint4*>(
        qkv + (int64_t)(b0 + t) * qkv_sb + (int64_t)((v_heads ? Hq + Hkv : 0) + h0 + min(hi, nh - 1)) * D + li * 8);
  }
  if (tid < kPT) {
    const int t = min(tid, nt - 1);
    const int slot = slots[b0 + t], off = offsets[b0 + t];
    const bool ok = tid < nt && slot >= 0 && slot < pool.num_slots && off >= 0 && off < P;
    s_slot[tid] = ok ? slot : -1;
    s_off[tid] = off;
    const int pslot = __shfl_up(ok ? slot : -1, 1, 64), poff = __shfl_up(off, 1, 64);
    const uint64_t next = __ballot(ok && tid > 0 && pslot == slot && poff + 1 == off);
    if (tid == 0) s_next = (int)next;
  }
  uint4 qw{}, kw{};
  if (!v_heads) {
    if (q_norm_w != nullptr) {
      qw = *reinterpret_cast<const uint4*>(q_norm_w + li * 8);
      kw = *reinterpret_cast<const uint4*>(k_norm_w + li * 8);
    }
    for (int i = tid; i < kPT * HALF; i += kPW * 64) {
      const int t = i / HALF, e = i % HALF / (HALF / 8), l = i % (HALF / 8);
      float c, s;
      rope_factors(positions[b0 + min(t, nt - 1)], inv_freq[8 * l + e], c, s);
      s_cs[t][e][l] = make_float2(c, s);
    }
  }
  __syncthreads();

  const bool is_q = !v_heads && h < Hq;
  const int hk = v_heads ? h : h - Hq;
  uint32_t vt[8] = {};                  // V: bytes of a dim's tokens
#pragma unroll
  for (int i = 0; i < kIter; ++i) {
    const int t = t0 + i;
    const uint32_t rw[4] = {raw[i].x, raw[i].y, raw[i].z, raw[i].w};
    float x[8];
#pragma unroll
    for (int e = 0; e < 8; ++e) x[e] = (e & 1) ? hi_h(rw[e / 2]) : lo_h(rw[e / 2]);
    if (!v_heads) {
      if (q_norm_w != nullptr) {
        const float rstd = rsqrtf(row_squares<D>(x, li) / (float)D + eps);
        const uint4 w4 = is_q ? qw : kw;
        const uint32_t ww[4] = {w4.x, w4.y, w4.z, w4.w};
#pragma unroll
        for (int e = 0; e < 8; ++e) x[e] = x[e] * rstd * ((e & 1) ? hi_h(ww[e / 2]) : lo_h(ww[e / 2]));
      }
      float y[8];
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        const float partner = D == 128 ? xor8(x[e]) : xor4(x[e]);
        const float2 cs = s_cs[t][e][li % (HALF / 8)];
        y[e] = fmaf(x[e], cs.x, (li < RL / 2 ? -partner : partner) * cs.y);
      }
#pragma unroll
      for (int e = 0; e < 8; ++e) x[e] = y[e];
      if (is_q && t < nt && hi < nh)
        *reinterpret_cast<uint4*>(q_out + ((int64_t)(b0 + t) * Hq + h) * D + li * 8) =
            make_uint4(pack_h2(x[0], x[1]), pack_h2(x[2], x[3]), pack_h2(x[4], x[5]), pack_h2(x[6], x[7]));
      // (a wave's rows may be of either kind: no lane leaves ahead of the row operations)
      if (h0 + nh <= Hq) continue;      // q heads alone (the whole workgroup)
    }
    // magnitudes compare as their bits do, NaN above infinity
    uint32_t amax = 0;
#pragma unroll
    for (int e = 0; e < 8; ++e) amax = max(amax, __float_as_uint(x[e]) & 0x7fffffffu);
    amax = row_max<D>(amax);
    const uint16_t sh = row_scale(__uint_as_float(amax), amax > 0x7f800000u);
    const Scale s = scale_of(sh);
    uint32_t c[8];
#pragma unroll
    for (int e = 0; e < 8; ++e) c[e] = code_of(x[e], s) & 255u;
    const uint32_t keep = s.ok ? ~0u : 0u;
    const int slot = s_slot[t];
    if (!is_q && hi < nh && t < nt && slot >= 0) {
      if (li == 0) (v_heads ? pool.vs : pool.ks)[(int64_t)slot * pool.scale_slot_stride + (int64_t)hk * P + s_off[t]] = sh;
      if (!v_heads)
        *reinterpret_cast<uint2*>(pool.k + (int64_t)slot * pool.slot_stride + ((int64_t)hk * P + s_off[t]) * D + li * 8) =
            make_uint2((c[0] | c[1] << 8 | c[2] << 16 | c[3] << 24) & keep, (c[4] | c[5] << 8 | c[6] << 16 | c[7] << 24) & keep);
    }
#pragma unroll
    for (int e = 0; e < 8; ++e) vt[e] |= (c[e] & keep) << (8 * i);
  }
  if (v_heads) {
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      if constexpr (kIter == 4) *reinterpret_cast<uint32_t*>(&s_v[hi][li * 8 + e][t0]) = vt[e];
      else *reinterpret_cast<uint16_t*>(&s_v[hi][li * 8 + e][t0]) = (uint16_t)vt[e];
    }
  }
  if (!v_heads) return;                 // the whole workgroup
  __syncthreads();
  // word g: tokens 4 g - r .. 4 g - r + 3, in one aligned word of the page if they are neighbours
  const int next = __builtin_amdgcn_readfirstlane(s_next), off0 = __builtin_amdgcn_readfirstlane(s_off[0]), r = off0 & 3;
  const bool all = next == (1 << kPT) - 2 && off0 % 16 == 0;
  for (int i = tid; i < nh * D; i += kPW * 64) {
    const int hi = i / D, d = i - hi * D;
    const uint32_t* sv = reinterpret_cast<const uint32_t*>(s_v[hi][d]);
    const uint32_t w[6] = {0u, sv[0], sv[1], sv[2], sv[3], 0u};
    int8_t* dst = pool.v + ((int64_t)(h0 + hi) * D + d) * P;
    if (all) {
      *reinterpret_cast<uint4*>(dst + (int64_t)s_slot[0] * pool.slot_stride + off0) = make_uint4(w[1], w[2], w[3], w[4]);
      continue;
    }
#pragma unroll
    for (int g = 0; g <= kPT / 4; ++g) {
      const int t = 4 * g - r;
      const uint32_t word = r == 0 ? w[g + 1] : __builtin_amdgcn_alignbyte(w[g + 1], w[g], 4 - r);
      if (t >= 0 && t + 3 < kPT && (next >> (t + 1) & 7) == 7 && s_off[t] % 4 == 0) {
        *reinterpret_cast<uint32_t*>(dst + (int64_t)s_slot[t] * pool.slot_stride + s_off[t]) = word;
        continue;
      }
#pragma unroll
      for (int j = 0; j < 4; ++j)
        if (t + j >= 0 && t + j < kPT && s_slot[t + j] >= 0)
          dst[(int64_t)s_slot[t + j] * pool.slot_stride + s_off[t + j]] = (int8_t)(word >> (8 * j));
    }
  }
}

// One wave per (item, kv head, token, K or V).  Latency-bound at a token per item (4.0 us, 16
// items of 8 heads of 128); V's codes are a byte store each, P apart: 256 items of 16 tokens take
// 24 us, a copy of their bytes 11.
template <int D>
__global__ __launch_bounds__(256) void kv_append_q8_kernel(const uint16_t* __restrict__ k_new,
                                                           const uint16_t* __restrict__ v_new, Q8Pool pool,
                                                           const int32_t* __restrict__ slots,
                                                           const int32_t* __restrict__ offsets, int64_t rows,
                                                           int Hkv, int n_tok, int P) {
  constexpr int J = D / 64;
  const int lane = threadIdx.x & 63;
  const int64_t item = (int64_t)blockIdx.x * 4 + (threadIdx.x >> 6);
  if (item >= 2 * rows) return;
  const bool is_v = item >= rows;
  const int64_t row = is_v ? item - rows : item;       // (b, head, token)
  const int64_t bh = row / n_tok;
  const int t = (int)(row - bh * n_tok);
  const int64_t b = bh / Hkv;
  const int slot = slots[b];
  const int64_t off = (int64_t)offsets[b] + t;
  if (slot < 0 || slot >= pool.num_slots || off < 0 || off >= P) return;   // uniform per wave
  float x[J];
#pragma unroll
  for (int j = 0; j < J; ++j) x[j] = h2f((is_v ? v_new : k_new)[row * D + lane + 64 * j]);
  store_row<D>(x, lane, is_v, pool, slot, (int)(bh - b * Hkv), (int)off, P);
}

// One thread per 16 codes: of a K token's dims, or of a V dim's tokens.  Bound by HBM: 2048 pages
// of 8 heads, 16 tokens, D 128 (202 MB read and written) in 35 us, 5.8 TB/s; 16 pages in 4.5.
__global__ __launch_bounds__(256) void dequantize_pages_kernel(Q8Pool pool, const int32_t* __restrict__ pages,
                                                               int64_t pieces, int Hkv, int D, int P,
                                                               uint16_t* __restrict__ k_out,
                                                               uint16_t* __restrict__ v_out) {
  const int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x;
  if (i >= 2 * pieces) return;
  const bool is_v = i >= pieces;
  const int64_t piece = is_v ? i - pieces : i;
  const int per_page = Hkv * P * D / 16;
  const int64_t n = piece / per_page;
  const int e = (int)(piece - n * per_page) * 16;      // first element in the page
  const int slot = pages[n];
  uint32_t o[8] = {0u, 0u, 0u, 0u, 0u, 0u, 0u, 0u};
  if (slot >= 0 && slot < pool.num_slots) {
    const uint4 c = *reinterpret_cast<const uint4*>((is_v ? pool.v : pool.k) + slot * pool.slot_stride + e);
    const uint32_t cw[4] = {c.x, c.y, c.z, c.w};
    float s[16];
    if (is_v) {
      const int h = e / (P * D);
      const uint16_t* sp = pool.vs + slot * pool.scale_slot_stride + h * P + e % P;
#pragma unroll
      for (int j = 0; j < 2; ++j) {
        const uint4 sw = *reinterpret_cast<const uint4*>(sp + 8 * j);
        const uint32_t w[4] = {sw.x, sw.y, sw.z, sw.w};
#pragma unroll
        for (int q = 0; q < 4; ++q) {
          s[8 * j + 2 * q] = lo_h(w[q]);
          s[8 * j + 2 * q + 1] = hi_h(w[q]);
        }
      }
    } else {
      const float s1 = h2f(pool.ks[slot * pool.scale_slot_stride + e / D]);
#pragma unroll
      for (int j = 0; j < 16; ++j) s[j] = s1;
    }
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      const float a = (float)(int8_t)(cw[j / 2] >> ((j & 1) * 16)) * s[2 * j];
      const float b = (float)(int8_t)(cw[j / 2] >> ((j & 1) * 16 + 8)) * s[2 * j + 1];
      o[j] = pack_h2(a, b);
    }
  }
  uint4* dst = reinterpret_cast<uint4*>((is_v ? v_out : k_out) + piece * 16);
  dst[0] = make_uint4(o[0], o[1], o[2], o[3]);
  dst[1] = make_uint4(o[4], o[5], o[6], o[7]);
}

}  // namespace

extern "C" int helm_qk_norm_rope_append_q8(const void* qkv, int64_t qkv_stride_b, const void* q_norm_w,
                                           const void* k_norm_w, float eps, const int32_t* positions,
                                           const float* inv_freq, void* q_out, const helm_kv_pool_q8* pool,
                                           const int32_t* slots, const int32_t* offsets, int B, int Hq,
                                           int Hkv, int D, int P, void* stream) {
  const std::string f("helm_qk_norm_rope_append_q8");
  HELM_CHECK_ARG(qkv && positions && inv_freq && q_out && slots && offsets, f + ": null pointer");
  HELM_CHECK_ARG((q_norm_w == nullptr) == (k_norm_w == nullptr),
                 f + ": give both q / k norm weights or neither");
  HELM_CHECK_ARG(B >= 1 && Hq >= 1 && Hkv >= 1, f + ": sizes must be positive");
  HELM_CHECK_SUPPORTED(Hq <= (1 << 16) && Hkv <= (1 << 16), f + ": too many heads");
  if (const int rc = helm::check_q8_pool(pool, Hkv, D, P, f.c_str())) return rc;
  if (q_norm_w)
    HELM_CHECK_SUPPORTED(helm::aligned16(q_norm_w) && helm::aligned16(k_norm_w),
                         f + ": norm weights must be 16-byte aligned");
  HELM_CHECK_ARG(qkv_stride_b >= (int64_t)(Hq + 2 * Hkv) * D, f + ": qkv row stride too small");
  HELM_CHECK_SUPPORTED(qkv_stride_b % 8 == 0 && helm::aligned16(qkv) && helm::aligned16(q_out),
                       f + ": qkv rows and q_out must be 16-byte aligned");
  const int64_t items = (int64_t)B * (Hq + 2 * Hkv);
  HELM_CHECK_SUPPORTED(items <= (int64_t)1 << 25, f + ": too many tokens");
  const hipStream_t s = static_cast<hipStream_t>(stream);
  if (items >= prompt_rows(D)) {
    const dim3 grid((B + kPT - 1) / kPT, (Hq + Hkv + kPH - 1) / kPH + (Hkv + kPH - 1) / kPH);
    auto go = [&](auto kern) {
      hipLaunchKernelGGL(kern, grid, dim3(kPW * 64), 0, s, static_cast<const uint16_t*>(qkv), qkv_stride_b,
                         static_cast<const uint16_t*>(q_norm_w), static_cast<const uint16_t*>(k_norm_w), eps,
                         positions, inv_freq, static_cast<uint16_t*>(q_out), pool_of(pool), slots, offsets, B, Hq,
                         Hkv, P);
    };
    if (D == 64) go(qk_norm_rope_append_q8_prompt_kernel<64>);
    else go(qk_norm_rope_append_q8_prompt_kernel<128>);
    HELM_CHECK_LAUNCH("helm_qk_norm_rope_append_q8 launch");
    return HELM_OK;
  }
  const dim3 grid((unsigned)((items + 3) / 4));
  auto go = [&](auto kern) {
    hipLaunchKernelGGL(kern, grid, dim3(256), 0, s, static_cast<const uint16_t*>(qkv), qkv_stride_b,
                       static_cast<const uint16_t*>(q_norm_w), static_cast<const uint16_t*>(k_norm_w), eps,
                       positions, inv_freq, static_cast<uint16_t*>(q_out), pool_of(pool), slots, offsets, items,
                       Hq, Hkv, P);
  };
  if (D == 64) go(qk_norm_rope_append_q8_kernel<64>);
  else go(qk_norm_rope_append_q8_kernel<128>);
  HELM_CHECK_LAUNCH("helm_qk_norm_rope_append_q8 launch");
  return HELM_OK;
}

extern "C" int helm_kv_append_q8(const void* k_new, const void* v_new, const helm_kv_pool_q8* pool,
                                 const int32_t* slots, const int32_t* offsets, int B, int Hkv, int n_tok, int D,
                                 int P, void* stream) {
  const std::string f("helm_kv_append_q8");
  HELM_CHECK_ARG(k_new && v_new && slots && offsets, f + ": null pointer");
  HELM_CHECK_ARG(B >= 1 && Hkv >= 1 && n_tok >= 1, f + ": sizes must be positive");
  if (const int rc = helm::check_q8_pool(pool, Hkv, D, P, f.c_str())) return rc;
  HELM_CHECK_ARG(n_tok <= P, f + ": more new tokens than a page holds");
  const int64_t rows = (int64_t)B * Hkv * n_tok;
  HELM_CHECK_SUPPORTED(rows <= (int64_t)1 << 24, f + ": too many rows");
  const dim3 grid((unsigned)((2 * rows + 3) / 4));
  const hipStream_t s = static_cast<hipStream_t>(stream);
  auto go = [&](auto kern) {
    hipLaunchKernelGGL(kern, grid, dim3(256), 0, s, static_cast<const uint16_t*>(k_new),
                       static_cast<const uint16_t*>(v_new), pool_of(pool), slots, offsets, rows, Hkv, n_tok, P);
  };
  if (D == 64) go(kv_append_q8_kernel<64>);
  else go(kv_append_q8_kernel<128>);
  HELM_CHECK_LAUNCH("helm_kv_append_q8 launch");
  return HELM_OK;
}

extern "C" int helm_dequantize_pages(const helm_kv_pool_q8* pool, const int32_t* pages, int n, void* k_out,
                                     void* v_out, int Hkv, int D, int P, void* stream) {
  const std::string f("helm_dequantize_pages");
  HELM_CHECK_ARG(pages && k_out && v_out, f + ": null pointer");
  HELM_CHECK_ARG(n >= 1 && Hkv >= 1, f + ": sizes must be positive");
  if (const int rc = helm::check_q8_pool(pool, Hkv, D, P, f.c_str())) return rc;
  HELM_CHECK_SUPPORTED(helm::aligned16(k_out) && helm::aligned16(v_out), f + ": outputs must be 16-byte aligned");
  HELM_CHECK_SUPPORTED(Hkv <= (1 << 16), f + ": too many kv heads");
  const int64_t pieces = (int64_t)n * Hkv * P * D / 16;
  HELM_CHECK_SUPPORTED(pieces <= (int64_t)1 << 30, f + ": too many pages");
  hipLaunchKernelGGL(dequantize_pages_kernel, dim3((unsigned)((2 * pieces + 255) / 256)), dim3(256), 0,
                     static_cast<hipStream_t>(stream), pool_of(pool), pages, pieces, Hkv, D, P,
                     static_cast<uint16_t*>(k_out), static_cast<uint16_t*>(v_out));
  HELM_CHECK_LAUNCH("helm_dequantize_pages launch");
  return HELM_OK;
}
