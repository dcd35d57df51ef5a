// paged_attention_q8.hip — paged GQA decode attention over K/V pages of 8-bit codes
// with one fp16 scale per token and kv head.
//
// out[b,h] = softmax(scale * q[b,h] . K_b^T) V_b with K = ck * sk, V = cv * sv.  A
// token's K scale multiplies its score and its V scale its probability, so both
// contractions run on the exact integers: a code is turned into fp16 by a bias trick
// and multiplied on the matrix cores with fp32 accumulation.
//
// Bound by streaming the pages once.  One 256-thread workgroup per (split, kv head,
// item), its four waves taking 64-token steps round robin.  Per step a wave computes
//   S[64 tok x 16 col] = K . Q^T         four 16 x 16 tiles
//   O^T[D x 16]       += V^T . P^T       D / 16 tiles
// with the G = Hq / Hkv query heads of the kv head as columns.  Every load is 16 bytes
// per lane: 16 dims of a token for K, the 16 tokens of a dim for V (V pages are stored
// [D][P]), which takes 64-token steps and this token order inside the score tiles: row
// 4 a + r of tile t is token 16 a + 4 t + r, so that lane group g ends with the scores
// of tokens 16 g .. 16 g + 15, whose V^T it feeds to the second product.
// p * sv is split into fp16 hi + lo parts (fp32-level accuracy).  fp16 has too few
// exponents for any sv, so the wave keeps the binary exponent e of the largest V scale it
// has met, as it keeps the largest score: the products run on p * sv * 2^(14 - e) and the
// sums are rescaled when e grows.
#include "helm_common.h"

namespace {

constexpr int kThreads = 256;
constexpr int kWaves = 4;
constexpr int kStep = 64;             // tokens per wave step
constexpr int kMaxSplitPages = 4096;  // page-table entries of one split staged in LDS
constexpr int kMinExp = -24;          // exponent of the smallest fp16 number
constexpr int kTopExp = 14;           // probabilities reach 2^(kTopExp + 1): below fp16's largest

typedef _Float16 h8_t __attribute__((ext_vector_type(8)));
typedef float f4_t __attribute__((ext_vector_type(4)));

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

__device__ __forceinline__ float pow2(int e) { return __int_as_float((127 + e) << 23); }   // |e| < 127

template <int D>
struct StepBuf {
  uint4 k[4][D / 64];
  uint4 v[D / 16];
  uint4 ks[2], vs[2];     // the 16 scales of lane group grp's tokens
};

template <int D, int P, int GMAX>
__global__ __launch_bounds__(kThreads, 2) void paged_attn_q8_kernel(Q8Args a) {
  constexpr int KT = D / 64;
  constexpr int DT = D / 16;
  constexpr int UPP = kStep / P;        // page-table entries of a step

  __shared__ int s_slot[kMaxSplitPages];
  __shared__ float s_m[kWaves][GMAX], s_l[kWaves][GMAX];
  __shared__ __attribute__((aligned(16))) float s_o[kWaves][GMAX][D];

  const int tid = threadIdx.x;
  const int wave = tid >> 6;
  const int lane = tid & 63;
  const int col = lane & 15;
  const int grp = lane >> 4;
  const int split = blockIdx.x;
  const int hk = blockIdx.y;
  const int b = blockIdx.z;
  const int G = a.Hq / a.Hkv;
  const int S = a.num_splits;

  const int seq = max(a.seq_lens[b], 0);
  const int max_steps = q8_table_steps(a.max_pages, P);
  const int n_local = max_steps > split ? (max_steps - 1 - split) / S + 1 : 0;
  const int p_cnt = n_local * UPP;
  const int p_last = max(p_cnt - 1, 0);
  const int32_t* ptab = a.page_table + (int64_t)b * a.pt_stride;
  for (int i = tid; i < p_cnt; i += kThreads) {
    const int j = i / UPP;
    const int pg = (split + j * S) * UPP + (i - j * UPP);
    const int slot = pg < a.max_pages ? ptab[pg] : -1;
    s_slot[i] = (slot >= 0 && slot < a.num_slots) ? slot : -1;
  }
  // Q^T operands: lane holds q[head col][64 kk + 16 grp + 8 h, + 8]; columns past G
  // repeat the last head and are never published
  h8_t qb[KT][2];
  {
    const uint16_t* qp = a.q + (int64_t)b * a.q_sb + (int64_t)(hk * G + min(col, G - 1)) * a.q_sh + grp * 16;
#pragma unroll
    for (int kk = 0; kk < KT; ++kk)
#pragma unroll
      for (int h = 0; h < 2; ++h) qb[kk][h] = *reinterpret_cast<const h8_t*>(qp + kk * 64 + h * 8);
  }
  lds_barrier();

  const int64_t tokens = min((int64_t)seq, (int64_t)a.max_pages * P);
  const int live_steps = (int)((tokens + kStep - 1) / kStep);
  const int nsteps = live_steps > split ? (live_steps - 1 - split) / S + 1 : 0;
  const int my_steps = nsteps > wave ? (nsteps - 1 - wave) / kWaves + 1 : 0;

  // staged slot of 16-token block g of local step j, and the block's first token in its page
  auto entry = [&](int j, int g) { return min(j * UPP + g * 16 / P, p_last); };
  constexpr int64_t kPage = (int64_t)P * D;

  auto load = [&](StepBuf<D>& bf, int i) {
    const int j = wave + kWaves * i;
    const int gk = col >> 2;                    // block of this lane's score-tile rows
    const int slot_k = max(s_slot[entry(j, gk)], 0);
    const int slot_v = max(s_slot[entry(j, grp)], 0);
    const uint8_t* kp = a.k + (int64_t)slot_k * a.slot_stride + hk * kPage +
                        (int64_t)((gk * 16) % P + (col & 3)) * D + grp * 16;
#pragma unroll
    for (int t = 0; t < 4; ++t)
#pragma unroll
      for (int kk = 0; kk < KT; ++kk) bf.k[t][kk] = ld16(kp + t * 4 * D + kk * 64);
    const uint8_t* vp = a.v + (int64_t)slot_v * a.slot_stride + hk * kPage + (int64_t)col * P + (grp * 16) % P;
#pragma unroll
    for (int d = 0; d < DT; ++d) bf.v[d] = ld16(vp + d * 16 * P);
    const int64_t so = (int64_t)slot_v * a.scale_slot_stride + hk * P + (grp * 16) % P;
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      bf.ks[h] = *reinterpret_cast<const uint4*>(a.ks + so + h * 8);
      bf.vs[h] = *reinterpret_cast<const uint4*>(a.vs + so + h * 8);
    }
  };

  float m_run = -INFINITY, l_run = 0.f;
  int e_run = kMinExp;                        // exponent of the largest V scale (whole wave)
  f4_t o[DT];
#pragma unroll
  for (int d = 0; d < DT; ++d) o[d] = f4_t{0.f, 0.f, 0.f, 0.f};

  auto compute = [&](const StepBuf<D>& bf, int i) {
    const int j = wave + kWaves * i;
    const int64_t tv = (int64_t)(split + j * S) * kStep + grp * 16;
    const bool page_ok = s_slot[entry(j, grp)] >= 0;
    // this lane's 16 tokens: the first nvalid are real
    const int nvalid = page_ok ? (int)max((int64_t)0, min((int64_t)16, tokens - tv)) : 0;

    float s[16];
#pragma unroll
    for (int t = 0; t < 4; ++t) {
      f4_t c = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
      for (int kk = 0; kk < KT; ++kk) {
        c = __builtin_amdgcn_mfma_f32_16x16x32_f16(codes8(bf.k[t][kk].x, bf.k[t][kk].y), qb[kk][0], c, 0, 0, 0);
        c = __builtin_amdgcn_mfma_f32_16x16x32_f16(codes8(bf.k[t][kk].z, bf.k[t][kk].w), qb[kk][1], c, 0, 0, 0);
      }
#pragma unroll
      for (int r = 0; r < 4; ++r) s[t * 4 + r] = c[r];
    }
    const uint32_t ksw[8] = {bf.ks[0].x, bf.ks[0].y, bf.ks[0].z, bf.ks[0].w,
                             bf.ks[1].x, bf.ks[1].y, bf.ks[1].z, bf.ks[1].w};
    uint32_t vsw[8] = {bf.vs[0].x, bf.vs[0].y, bf.vs[0].z, bf.vs[0].w,
                       bf.vs[1].x, bf.vs[1].y, bf.vs[1].z, bf.vs[1].w};
    // scales of places that hold no token may be any bits
    if (!__all(nvalid == 16)) {
#pragma unroll
      for (int q = 0; q < 8; ++q)
        vsw[q] &= (2 * q < nvalid ? 0x0000ffffu : 0u) | (2 * q + 1 < nvalid ? 0xffff0000u : 0u);
    }
    typedef uint16_t us2_t __attribute__((ext_vector_type(2)));
    us2_t big = {0, 0};
#pragma unroll
    for (int q = 0; q < 8; ++q) big = __builtin_elementwise_max(big, __builtin_bit_cast(us2_t, vsw[q] & 0x7fff7fffu));
    int top = max((int)big[0], (int)big[1]);
    top = max(top, __shfl_xor(top, 16, 64));
    top = max(top, __shfl_xor(top, 32, 64));
    const int e_top = (int)(__float_as_uint(h2f((uint16_t)top)) >> 23) - 127;
    const int e_new = max(e_run, min(e_top, 15));
    float mx = -INFINITY;
#pragma unroll
    for (int e = 0; e < 16; ++e) {
      const float sk = (e & 1) ? hi_h(ksw[e / 2]) : lo_h(ksw[e / 2]);
      s[e] = e < nvalid ? s[e] * (sk * a.qk_scale_log2) : -INFINITY;
      mx = fmaxf(mx, s[e]);
    }
    mx = fmaxf(mx, __shfl_xor(mx, 16, 64));
    mx = fmaxf(mx, __shfl_xor(mx, 32, 64));
    const float m_new = fmaxf(m_run, mx);
    const float ref = (m_new == -INFINITY) ? 0.f : m_new;   // exp2(-inf - ref) stays 0
    const float alpha = exp2f(m_run - ref);
    const float alpha_o = alpha * pow2(e_run - e_new);
    const float pscale = pow2(kTopExp - e_new);
    h8_t phi[2], plo[2];
    float lsum = 0.f;
#pragma unroll
    for (int e = 0; e < 16; ++e) {
      const float sv = (e & 1) ? hi_h(vsw[e / 2]) : lo_h(vsw[e / 2]);
      const float p = exp2f(s[e] - ref);
      lsum += p;
      const float pv = p * (sv * pscale);   // 0 * 0 where there is no token
      const _Float16 h = (_Float16)pv;
      phi[e / 8][e % 8] = h;
      plo[e / 8][e % 8] = (_Float16)(pv - (float)h);
    }
    l_run = l_run * alpha + lsum;
    m_run = m_new;
    e_run = e_new;
#pragma unroll
    for (int d = 0; d < DT; ++d) {
      const h8_t v0 = codes8(bf.v[d].x, bf.v[d].y), v1 = codes8(bf.v[d].z, bf.v[d].w);
      o[d] *= alpha_o;
      o[d] = __builtin_amdgcn_mfma_f32_16x16x32_f16(v0, phi[0], o[d], 0, 0, 0);
      o[d] = __builtin_amdgcn_mfma_f32_16x16x32_f16(v1, phi[1], o[d], 0, 0, 0);
      o[d] = __builtin_amdgcn_mfma_f32_16x16x32_f16(v0, plo[0], o[d], 0, 0, 0);
      o[d] = __builtin_amdgcn_mfma_f32_16x16x32_f16(v1, plo[1], o[d], 0, 0, 0);
    }
  };

  StepBuf<D> bufA, bufB;
  if (my_steps > 0) load(bufA, 0);
  int i = 0;
  for (; i + 2 < my_steps; i += 2) {
    load(bufB, i + 1);
    compute(bufA, i);
    load(bufA, i + 2);
    compute(bufB, i + 1);
  }
  if (i + 1 < my_steps) {
    load(bufB, i + 1);
    compute(bufA, i);
    compute(bufB, i + 1);
  } else if (i < my_steps) {
    compute(bufA, i);
  }

  float l = l_run;
  l += __shfl_xor(l, 16, 64);
  l += __shfl_xor(l, 32, 64);
  if (col < G) {
    const float unscale = pow2(e_run - kTopExp);
#pragma unroll
    for (int d = 0; d < DT; ++d) {
      o[d] *= unscale;
      *reinterpret_cast<float4*>(&s_o[wave][col][d * 16 + grp * 4]) =
          make_float4(o[d][0], o[d][1], o[d][2], o[d][3]);
    }
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
        a.part_ml[pidx * 2] = mx;
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

}  // namespace

extern "C" int helm_paged_decode_attn_q8(const void* q, int64_t q_stride_b, int64_t q_stride_h,
                                         const helm_kv_pool_q8* pool, const int32_t* page_table,
                                         int64_t pt_stride, const int32_t* seq_lens, float* part_o,
                                         float* part_ml, void* out, int B, int Hq, int Hkv, int D, int P,
                                         int max_pages, int num_splits, float scale, void* stream) {
  const std::string f("helm_paged_decode_attn_q8");
  HELM_CHECK_ARG(q && page_table && seq_lens && out, f + ": null pointer");
  HELM_CHECK_ARG(B >= 1 && Hq >= 1 && Hkv >= 1 && max_pages >= 1 && num_splits >= 1,
                 f + ": sizes must be positive");
  HELM_CHECK_ARG(Hq % Hkv == 0, f + ": Hq must be a multiple of Hkv");
  HELM_CHECK_SUPPORTED(Hq / Hkv <= 16, f + ": at most 16 query heads per kv head");
  HELM_CHECK_SUPPORTED(B <= 65535 && Hkv <= 65535, f + ": at most 65535 items and kv heads");
  if (const int rc = helm::check_q8_pool(pool, Hkv, D, P, "helm_paged_decode_attn_q8")) return rc;
  HELM_CHECK_ARG(pt_stride >= max_pages, f + ": page-table stride < max_pages");
  HELM_CHECK_SUPPORTED((int64_t)max_pages * P <= (int64_t)1 << 30, f + ": page table covers too many tokens");
  HELM_CHECK_SUPPORTED((int64_t)(q8_table_steps(max_pages, P) + num_splits - 1) / num_splits * (kStep / P) <=
                           kMaxSplitPages,
                       f + ": more than " + std::to_string(kMaxSplitPages) + " pages per split (raise num_splits)");
  HELM_CHECK_SUPPORTED(q_stride_h % 8 == 0 && q_stride_b % 8 == 0 && helm::aligned16(q),
                       f + ": q strides must be multiples of 8 and q 16-byte aligned");
  HELM_CHECK_SUPPORTED(reinterpret_cast<uintptr_t>(out) % 8 == 0, f + ": out must be 8-byte aligned");
  if (num_splits > 1) {
    HELM_CHECK_ARG(part_o && part_ml, f + ": splits need part_o and part_ml");
    HELM_CHECK_SUPPORTED(helm::aligned16(part_o) && reinterpret_cast<uintptr_t>(part_ml) % 8 == 0,
                         f + ": part_o must be 16-byte and part_ml 8-byte aligned");
  }
  Q8Args a{};
  a.q = static_cast<const uint16_t*>(q); a.q_sb = q_stride_b; a.q_sh = q_stride_h;
  a.k = static_cast<const uint8_t*>(pool->k); a.v = static_cast<const uint8_t*>(pool->v);
  a.ks = static_cast<const uint16_t*>(pool->k_scale); a.vs = static_cast<const uint16_t*>(pool->v_scale);
  a.slot_stride = pool->slot_stride; a.scale_slot_stride = pool->scale_slot_stride;
  a.num_slots = pool->num_slots;
  a.page_table = page_table; a.pt_stride = pt_stride; a.seq_lens = seq_lens;
  a.part_o = part_o; a.part_ml = part_ml; a.out = static_cast<uint16_t*>(out);
  a.B = B; a.Hq = Hq; a.Hkv = Hkv; a.max_pages = max_pages; a.num_splits = num_splits;
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
  if (num_splits == 1) return HELM_OK;
  return helm_paged_attn_reduce(part_o, part_ml, out, B, Hq, D, num_splits, stream);
}
