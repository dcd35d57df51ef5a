// kv_q8.hip — KV pages of 8-bit codes with one fp16 scale per token and kv head: the
// writes (plain, and with q / k norm and RoPE on the way) and the way back to fp16.
//
// Quantisation of a row x[D]: s = fp16(max |x| / 127), c = rne(x / s) in [-127, 127].
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
// Code of x under scale s; 0 under a scale of 0 or one that is not finite.
__device__ __forceinline__ int8_t code_of(float x, float s) {
  if (!(s > 0.f && s < INFINITY)) return 0;
  return (int8_t)(int)rintf(fminf(fmaxf(x / s, -127.f), 127.f));
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
  const float s = h2f(sh);
#pragma unroll
  for (int j = 0; j < J; ++j) {
    const int d = lane + 64 * j;
    const int8_t c = code_of(x[j], s);
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
// quantised into their page.  Latency-bound at a few tokens.
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
      y[j] = x[j] * c + rot * s;
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

// One wave per (item, kv head, token, K or V).
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

// One thread per 16 codes: of a K token's dims, or of a V dim's tokens.
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
  if (const int rc = helm::check_q8_pool(pool, Hkv, D, P, f.c_str())) return rc;
  HELM_CHECK_ARG(qkv_stride_b >= (int64_t)(Hq + 2 * Hkv) * D, f + ": qkv row stride too small");
  HELM_CHECK_SUPPORTED(qkv_stride_b % 8 == 0 && helm::aligned16(qkv) && helm::aligned16(q_out),
                       f + ": qkv rows and q_out must be 16-byte aligned");
  const int64_t items = (int64_t)B * (Hq + 2 * Hkv);
  HELM_CHECK_SUPPORTED(items <= (int64_t)1 << 25, f + ": too many tokens");
  const dim3 grid((unsigned)((items + 3) / 4));
  const hipStream_t s = static_cast<hipStream_t>(stream);
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
