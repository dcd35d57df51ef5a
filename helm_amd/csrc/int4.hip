// int4.hip — linears with 4-bit weights and one scale per group of inputs.
//
// y[m,n] = fp16( sum_g s[n,g] * sum_{k in g} c[n,k] x[m,k]  (+ bias[n]) ), c in
// [-8, 7], s fp16, groups of 32, 64 or 128 inputs, fp32 accumulation.
//
// Weights are laid out once, in the matrix cores' operand order: tiles of 16
// outputs x 128 inputs (1 KiB), tile (nt, kt) at word (nt * KT + kt) * 256, lane l
// of a wave owning the 16 bytes at lane l: output 16 nt + l % 16, word t (0..3)
// holding inputs 128 kt + 32 t + 8 (l / 16) + 0..7.  So one coalesced 16-byte load
// per lane is the operand of four MFMAs and nothing is shuffled.  A word keeps the
// even inputs' codes (plus 8) in its low half and the odd ones' in its high half,
// input 2p / 2p + 1 at bit 4p of either, so two codes at a time become fp16 numbers.
// Scales follow the tiles: [NT][KT][128 / group][16] fp16.  N is padded to 16
// outputs and K to 128 inputs with codes of 0 and scales of 0.
#include <algorithm>
#include <type_traits>

#include "helm_common.h"

namespace {

typedef _Float16 h8_t __attribute__((ext_vector_type(8)));
typedef float f4_t __attribute__((ext_vector_type(4)));
typedef __attribute__((address_space(3))) void lds_void_t;

constexpr int kTileWords = 256;       // 32-bit words of a 16 x 128 tile

// The eight codes of a word as fp16 numbers b + u, exact: u in mantissa bits 2-5 of [256,
// 512) for inputs 0, 1, 4, 5, in bits 6-9 of [16, 32) for inputs 2, 3, 6, 7; two shifts and four
// and-ors.  The masks and exponents live in registers (as literals they take an and and an
// or, eight bytes each).
struct Unpack {
  uint32_t m0 = 0x003C003Cu, m1 = 0x03C003C0u, o0 = 0x5C005C00u, o1 = 0x4C004C00u;
  __device__ __forceinline__ Unpack() {
    asm("" : "+s"(m0), "+s"(m1), "+v"(o0), "+v"(o1));
  }
  __device__ __forceinline__ u32x4_t operator()(uint32_t w) const {
    const uint32_t l = w << 2, r = w >> 6;
    return u32x4_t{(l & m0) | o0, (l & m1) | o1, (r & m0) | o0, (r & m1) | o1};
  }
};

// Word of eight codes as fp16 (b + u - b - 8, exact).
__device__ __forceinline__ h8_t word_codes(const Unpack& unpack, uint32_t w) {
  const h2_t off0 = {(_Float16)-264.0f, (_Float16)-264.0f}, off1 = {(_Float16)-24.0f, (_Float16)-24.0f};
  const u32x4_t p = unpack(w);
  h8_t r;
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const h2_t v = __builtin_bit_cast(h2_t, (uint32_t)p[i]) + (i & 1 ? off1 : off0);
    r[2 * i] = v[0];
    r[2 * i + 1] = v[1];
  }
  return r;
}

template <int N>
__device__ __forceinline__ void wait_vm() {
  static_assert(N >= 0 && N < 64, "vmcnt range");
  asm volatile("" ::: "memory");
  __builtin_amdgcn_s_waitcnt((N & 15) | (7 << 4) | (15 << 8) | ((N >> 4) << 14));
  asm volatile("" ::: "memory");
}
__device__ __forceinline__ void wait_vm_n(int n) {      // n: a constant once inlined
  asm volatile("" ::: "memory");
  switch (n) {
    case 4: __builtin_amdgcn_s_waitcnt(4 | (7 << 4) | (15 << 8)); break;
    case 5: __builtin_amdgcn_s_waitcnt(5 | (7 << 4) | (15 << 8)); break;
    case 6: __builtin_amdgcn_s_waitcnt(6 | (7 << 4) | (15 << 8)); break;
    case 7: __builtin_amdgcn_s_waitcnt(7 | (7 << 4) | (15 << 8)); break;
    case 8: __builtin_amdgcn_s_waitcnt(8 | (7 << 4) | (15 << 8)); break;
    case 10: __builtin_amdgcn_s_waitcnt(10 | (7 << 4) | (15 << 8)); break;
    default: __builtin_amdgcn_s_waitcnt((7 << 4) | (15 << 8)); break;
  }
  asm volatile("" ::: "memory");
}
// One wave's global -> LDS copies: lane l moves 16 (4) bytes to LDS byte lds + 16 (4) l.  In
// assembly so that the compiler does not count them: it would wait for every copy in
// flight before each LDS read.  The kernels wait for them by number (wait_vm).
#pragma clang diagnostic push
#pragma clang diagnostic ignored "-Winline-asm"   // m0 is named as clobbered on purpose
__device__ __forceinline__ void copy_to_lds(const void* base, uint32_t off, uint32_t lds) {
  asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %1, %2"
               :
               : "s"(__builtin_amdgcn_readfirstlane(lds)), "v"(off), "s"(base)
               : "memory", "m0");
}
// the same of what is read once
__device__ __forceinline__ void copy_nt_to_lds(const void* base, uint32_t off, uint32_t lds) {
  asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %1, %2 nt"
               :
               : "s"(__builtin_amdgcn_readfirstlane(lds)), "v"(off), "s"(base)
               : "memory", "m0");
}
__device__ __forceinline__ void copy4_to_lds(const void* base, uint32_t off, uint32_t lds) {
  asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tglobal_load_lds_dword %1, %2"
               :
               : "s"(__builtin_amdgcn_readfirstlane(lds)), "v"(off), "s"(base)
               : "memory", "m0");
}
#pragma clang diagnostic pop

// a pointer that is the same in every lane, as a scalar
__device__ __forceinline__ const void* uniform(const void* p) {
  const uint64_t v = reinterpret_cast<uint64_t>(p);
  const uint32_t lo = __builtin_amdgcn_readfirstlane((uint32_t)v), hi = __builtin_amdgcn_readfirstlane((uint32_t)(v >> 32));
  return reinterpret_cast<const void*>((uint64_t)hi << 32 | lo);
}

// ---------------------------------------------------------------------------
// 1 to 32 tokens
// ---------------------------------------------------------------------------
// Bound by the weight stream, and by the instructions that unpack it: x^T operands of a
// wave's inputs stay in registers; a workgroup's 16 waves (four a SIMD: a wave alone takes 950
// cycles a tile, mostly latencies) split the inputs of a k slice (UW tiles each) and walk
// row tiles tb, tb + nb, ....  Weights go global -> LDS through a private ring of kDepth
// tiles per wave, and the scales of a row tile's share through another, waited for by count:
// 96 KB on the way per CU, and no register holds any (two or three row tiles in registers
// instead spilled, or kept less on the way: 4.2 TB/s; this streams 151936 x 4096, 321 MB, at
// 6.1).  Where the shares are uneven the barriers wait: 5120 inputs are two tiles for half of the waves
// and three for the others, and 34816 outputs nine row tiles for half of the workgroups and eight for
// the others, so 0.79 of the places hold a tile: 92 MB in 20 us, 4.6 TB/s.  A tile is read
// back as it lies, a 16-byte operand word group per lane.
// The products of up to 16 tokens run on b + u; the -sum((b + 8) x) that turns them into codes is the
// same for every output, so it is computed once per wave and group (an MFMA with a constant operand)
// and starts each accumulation.  Its partial sums are up to 300 sum |x| of the group, each rounded by
// 2^-24 of that.  (Codes for every product, four more instructions a word: 151936 x 4096 at one token
// 53 -> 61 us, 5120 -> 34816 20 -> 22.9.)  Infinite starts take a walk of their own.  A group's sum is scaled by its outputs' scales in fp32.  The waves' partial
// tiles meet in LDS, one barrier per row tile, and take turns at the epilogue.
// 17 to 32 tokens are two operands of each unpacked weight, here the codes themselves (two products share
// the four instructions): 12288 x 4096 at 24 tokens 13.0 us, where the tiled product
// takes 19 at 33.
constexpr int kGemvTokens = 32;
constexpr int kW = 16;
constexpr int kMaxTiles = 64;         // row tiles a workgroup may walk (staged biases)

struct Int4Args {
  const uint16_t* x;
  int64_t ldx;
  const uint32_t* w;
  const uint16_t* scale;
  const uint16_t* bias;
  uint16_t* y;
  int64_t ldy;
  float* part;                        // [S][M][np] partial sums (PART)
  int np;
  int M, N, K, NT, KT;
  int S;                              // k slices
};

// UW: tiles of a wave's k share.  GU: groups per tile (UW * GU <= 8: a row tile's scales are
// one copy).
// MB: blocks of 16 tokens.
template <int UW, int GU, bool PART, int MB>
__global__ __launch_bounds__(kW * 64) void int4_gemv_kernel(Int4Args a) {
  // tiles of a wave on the way, and row tiles whose scales are (256 bytes each): what the
  // partial tiles leave of LDS
  constexpr int kDepth = MB == 1 ? 6 : 4, kScSlots = kDepth + 1;
  __shared__ __attribute__((aligned(1024))) uint8_t s_w[kW][kDepth * 1024];
  __shared__ __attribute__((aligned(16))) uint8_t s_s[kW][kScSlots * 256];
  __shared__ __attribute__((aligned(16))) f4_t s_c[2][MB][kW][64];
  __shared__ uint16_t s_bias[PART ? 2 : kMaxTiles * 16];
  constexpr int TG = 4 / GU;          // MFMAs per group
  static_assert(UW * GU <= 8 && (kDepth + UW - 1) / UW + 1 <= kScSlots, "scale ring");

  const int tid = threadIdx.x;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int lane = tid & 63;
  const int col = lane & 15;
  const int grp = lane >> 4;
  const int M = a.M;

  const int sl = PART ? (int)blockIdx.x % a.S : 0;
  const int tb = PART ? (int)blockIdx.x / a.S : (int)blockIdx.x;
  const int nb = PART ? (int)gridDim.x / a.S : (int)gridDim.x;
  const int T = __builtin_amdgcn_readfirstlane((a.NT - 1 - tb) / nb + 1);   // nb <= NT: at least one
  const int sa = (int)((int64_t)sl * a.KT / a.S), sn = (int)((int64_t)(sl + 1) * a.KT / a.S) - sa;
  const int u0 = __builtin_amdgcn_readfirstlane(sa + wave * sn / kW);      // [u0, u1): at most UW tiles
  const int u1 = __builtin_amdgcn_readfirstlane(sa + (wave + 1) * sn / kW);
  const int own = u1 - u0;

  // Tile u of the wave's share in row tile t, with the row tile's scales ahead of tile 0.  Past
  // the share all lanes copy the same 16 bytes, so that the copies can be counted.  Addresses
  // are scalar: the vector ALU has the unpacking to do.
  const uint32_t lds_w = __builtin_amdgcn_readfirstlane((uint32_t)(uintptr_t)(lds_void_t*)&s_w[wave][0]);
  const uint32_t lds_s = __builtin_amdgcn_readfirstlane((uint32_t)(uintptr_t)(lds_void_t*)&s_s[wave][0]);
  const uint32_t soff = (uint32_t)min(lane * 4, max(own, 1) * GU * 32 - 4), woff = (uint32_t)lane * 16;
  const int64_t first = (int64_t)tb * a.KT + min(u0, a.KT - 1), stride = (int64_t)nb * a.KT;
  const uint8_t* wbase = static_cast<const uint8_t*>(uniform(a.w + first * kTileWords));
  const uint8_t* sbase = static_cast<const uint8_t*>(uniform(a.scale + first * (GU * 16)));
  uint32_t at_w = lds_w, at_s = lds_s;          // slots of the next copies
  auto issue = [&](int t, int u) {
    const int64_t tile = t * stride;
    if (u == 0) {
      copy4_to_lds(uniform(sbase + tile * (GU * 32)), soff, at_s);
      at_s = at_s + 256 == lds_s + kScSlots * 256 ? lds_s : at_s + 256;
    }
    copy_nt_to_lds(uniform(wbase + (tile + (u < own ? u : 0)) * 1024), u < own ? woff : 0u, at_w);
    at_w = at_w + 1024 == lds_w + kDepth * 1024 ? lds_w : at_w + 1024;
  };
  h8_t xr[MB][UW][4];
#pragma unroll
  for (int mb = 0; mb < MB; ++mb) {
    const uint16_t* xrow = a.x + (int64_t)min(mb * 16 + col, M - 1) * a.ldx;
#pragma unroll
    for (int u = 0; u < UW; ++u)
#pragma unroll
      for (int t = 0; t < 4; ++t)
        xr[mb][u][t] = *reinterpret_cast<const h8_t*>(xrow + min((u0 + u) * 128 + t * 32 + grp * 8, a.K - 8));
  }
  asm volatile("" ::: "memory");
  // the first row tile's share right behind x; x's wait covers both (ahead of x: 7.1 us instead
  // of 6.9 at 4096 x 4096 and 16 tokens, the same at one)
#pragma unroll
  for (int u = 0; u < UW; ++u) issue(0, u);

  // bias of the workgroup's outputs, one of each per thread
  uint16_t bs = 0;
  if constexpr (!PART) {
    const int64_t n = min((int64_t)(tb + (int64_t)(tid >> 4) * nb) * 16 + (tid & 15), (int64_t)a.N - 1);
    if (a.bias) bs = a.bias[n];
  }
  // x has arrived: from here on the ring fills while the prologue computes
#pragma unroll
  for (int mb = 0; mb < MB; ++mb)
#pragma unroll
    for (int u = 0; u < UW; ++u)
#pragma unroll
      for (int t = 0; t < 4; ++t) asm volatile("" : "+v"(xr[mb][u][t]));
  if constexpr (!PART) {
    static_assert(kMaxTiles * 16 == kW * 64, "one bias per thread");
    s_bias[tid] = bs;
  }
#pragma unroll
  for (int n = UW; n < kDepth; ++n)
    if (n / UW < T) issue(n / UW, n % UW);
#pragma unroll
  for (int mb = 0; mb < MB; ++mb)
#pragma unroll
    for (int u = 0; u < UW; ++u)
#pragma unroll
      for (int t = 0; t < 4; ++t)
        if (u >= own || (u0 + u) * 128 + t * 32 >= a.K) xr[mb][u][t] = h8_t{};
  // -sum((b + 8) x) of each group: every row of the product with a constant operand.  Where x holds an
  // infinity it is one too, or NaN, and the sum that starts with it NaN.
  float nbias[MB][UW][GU];
  bool inf = false;                     // of the lane's token
  if constexpr (MB == 1) {
    const _Float16 p = (_Float16)-264.0f, q = (_Float16)-24.0f;
    const h8_t c = {p, p, q, q, p, p, q, q};
#pragma unroll
    for (int u = 0; u < UW; ++u)
#pragma unroll
      for (int g = 0; g < GU; ++g) {
        f4_t s = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int t = 0; t < TG; ++t) s = __builtin_amdgcn_mfma_f32_16x16x32_f16(c, xr[0][u][g * TG + t], s, 0, 0, 0);
        nbias[0][u][g] = s[0];
        inf |= !(fabsf(s[0]) < INFINITY);
      }
  }
  const Unpack unpack;

  const uint8_t* pw = &s_w[wave][0];  // slots read next
  const uint8_t* ps = &s_s[wave][0];
  const int total = T * UW;
  // inf_c: some token's group starts with an infinity; such sums run on the codes themselves, all others as ever
  auto walk = [&](auto inf_c) {
    for (int t = 0; t < T; ++t) {
      f4_t acc[MB];
#pragma unroll
      for (int mb = 0; mb < MB; ++mb) acc[mb] = f4_t{0.f, 0.f, 0.f, 0.f};
#pragma unroll
      for (int u = 0; u < UW; ++u) {
        // tile landed: at most the kDepth - 1 later tiles' copies are on the way, and those of
        // the row tiles that begin among them (the stream's end, where fewer follow, waits for
        // all)
        constexpr auto later = [](int u_) {
          int n = kDepth - 1;
          for (int j = 1; j < kDepth; ++j) n += (u_ + j) % UW == 0;
          return n;
        };
        if (t * UW + u + kDepth <= total) wait_vm_n(later(u));
        else wait_vm<0>();
        uint4 w = *reinterpret_cast<const uint4*>(pw + lane * 16);
        uint2 sc[GU];
#pragma unroll
        for (int g = 0; g < GU; ++g) sc[g] = *reinterpret_cast<const uint2*>(ps + (u * GU + g) * 32 + grp * 8);
        pw = pw + 1024 == &s_w[wave][kDepth * 1024] ? &s_w[wave][0] : pw + 1024;
        // the slot is refilled once this wave's reads have returned
        asm volatile("s_waitcnt lgkmcnt(0)" : "+v"(w.x), "+v"(w.y), "+v"(w.z), "+v"(w.w) :: "memory");
#pragma unroll
        for (int g = 0; g < GU; ++g) asm volatile("" : "+v"(sc[g].x), "+v"(sc[g].y));
        if (t + (u + kDepth) / UW < T) issue(t + (u + kDepth) / UW, (u + kDepth) % UW);
        if (u >= own) continue;         // not this wave's (uniform)
        const uint32_t wd[4] = {w.x, w.y, w.z, w.w};
#pragma unroll
        for (int g = 0; g < GU; ++g) {
          h8_t wf[TG];
#pragma unroll
          for (int q = 0; q < TG; ++q)
            wf[q] = MB == 1 ? __builtin_bit_cast(h8_t, unpack(wd[g * TG + q])) : word_codes(unpack, wd[g * TG + q]);
#pragma unroll
          for (int mb = 0; mb < MB; ++mb) {
            float z = MB == 1 ? nbias[mb][u][g] : 0.f;
            if constexpr (MB == 1) asm("" : "+v"(z));   // (or four copies of each would be kept)
            f4_t c = {z, z, z, z};
#pragma unroll
            for (int q = 0; q < TG; ++q) c = __builtin_amdgcn_mfma_f32_16x16x32_f16(wf[q], xr[mb][u][g * TG + q], c, 0, 0, 0);
            if constexpr (decltype(inf_c)::value) {
              f4_t e = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
              for (int q = 0; q < TG; ++q)
                e = __builtin_amdgcn_mfma_f32_16x16x32_f16(word_codes(unpack, wd[g * TG + q]), xr[mb][u][g * TG + q], e, 0, 0, 0);
#pragma unroll
              for (int r = 0; r < 4; ++r) c[r] = fabsf(z) < INFINITY ? c[r] : e[r];
            }
            acc[mb][0] = fmaf(lo_h(sc[g].x), c[0], acc[mb][0]);
            acc[mb][1] = fmaf(hi_h(sc[g].x), c[1], acc[mb][1]);
            acc[mb][2] = fmaf(lo_h(sc[g].y), c[2], acc[mb][2]);
            acc[mb][3] = fmaf(hi_h(sc[g].y), c[3], acc[mb][3]);
          }
        }
      }
      ps = ps + 256 == &s_s[wave][kScSlots * 256] ? &s_s[wave][0] : ps + 256;
#pragma unroll
      for (int mb = 0; mb < MB; ++mb) s_c[t & 1][mb][wave][lane] = acc[mb];
      lds_barrier();      // buffer t & 1 is written again only after tile t + 1's barrier
#pragma unroll
      for (int mb = 0; mb < MB; ++mb) {
        if (wave != ((t * MB + mb) & (kW - 1))) continue;
        const f4_t(*sc)[64] = s_c[t & 1][mb];
        f4_t v = sc[0][lane];
#pragma unroll (UW * MB <= 2 ? 15 : 5)  // (as many reads on the way as registers are left: 57 -> 53 us at 151936 x 4096)
        for (int w = 1; w < kW; ++w) {
          const f4_t o = sc[w][lane];
#pragma unroll
          for (int r = 0; r < 4; ++r) v[r] += o[r];
        }
        const int n0 = (tb + t * nb) * 16 + grp * 4, m = mb * 16 + col;   // v[r]: output n0 + r of token m
        if (m < M && n0 < a.N) {
          if constexpr (PART) {
            *reinterpret_cast<f4_t*>(a.part + ((int64_t)sl * M + m) * a.np + n0) = v;
          } else {
            uint16_t* yp = a.y + (int64_t)m * a.ldy + n0;
#pragma unroll
            for (int r = 0; r < 4; ++r)
              if (n0 + r < a.N) yp[r] = f2h(v[r] + h2f(s_bias[t * 16 + grp * 4 + r]));
          }
        }
      }
    }
  };
  if constexpr (MB == 1) {
    if (__builtin_expect(__any(inf), 0)) return walk(std::true_type{});
  }
  walk(std::false_type{});
}

// Adds the S partial sums of four outputs of a token, and the bias.
__global__ __launch_bounds__(256) void int4_reduce_kernel(const float* __restrict__ part, int S, int np,
                                                          const uint16_t* __restrict__ bias,
                                                          uint16_t* __restrict__ y, int64_t ldy, int M, int N) {
  const int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x;
  const int nq = np / 4;
  if (i >= (int64_t)M * nq) return;
  const int m = (int)(i / nq), n = (int)(i - (int64_t)m * nq) * 4;
  f4_t v = {0.f, 0.f, 0.f, 0.f};
  for (int s = 0; s < S; s += 8) {      // eight loads on the way; past the last they repeat it
    f4_t o[8];
#pragma unroll
    for (int j = 0; j < 8; ++j) o[j] = *reinterpret_cast<const f4_t*>(part + ((int64_t)min(s + j, S - 1) * M + m) * np + n);
#pragma unroll
    for (int j = 0; j < 8; ++j)
#pragma unroll
      for (int r = 0; r < 4; ++r) v[r] += s + j < S ? o[j][r] : 0.f;
  }
#pragma unroll
  for (int r = 0; r < 4; ++r)
    if (n + r < N) y[(int64_t)m * ldy + n + r] = f2h(v[r] + (bias ? h2f(bias[n + r]) : 0.f));
}

// k slices of a GEMV, tiles per wave (at most what x^T leaves of 128 registers), workgroups per
// slice.  Every workgroup is on a CU from the start, so the longest one counts: its row tiles,
// the x that it reads, and where there are slices the partial sums' traffic and a second
// launch.  Fitted (us) to 1149 timed (shape, tokens, S), within 5% of each; what it picks is 1% off
// the fastest on average, 8% at most.  5120 x 17408 at 16 tokens: 20 us in 9 slices, 17.6 in 5, 18.4
// in 3; 4096 x 4096 at 1: 5.6 in one, 7.5 in 2.
constexpr int max_uw(int GU, int M) { return M > 16 ? (GU == 4 ? 1 : 2) : GU == 1 ? 4 : GU == 2 ? 3 : 2; }
struct GemvPlan {
  int S, uw, nb;
};
GemvPlan plan_gemv(int M, int NT, int KT, int GU) {
  GemvPlan best{1, 1, 1};
  double least = -1.0;
  for (int S = (KT + kW * max_uw(GU, M) - 1) / (kW * max_uw(GU, M)); S <= std::min(KT, 256); ++S) {
    GemvPlan p;
    p.S = S;
    p.uw = ((KT + S - 1) / S + kW - 1) / kW;
    p.nb = S > 1 ? std::min(NT, 256 / S) : std::max(std::min(NT, 256), (NT + kMaxTiles - 1) / kMaxTiles);
    const int rows = (NT + p.nb - 1) / p.nb;
    const double sums = (double)S * M * NT * 128.0, x = 0.006 * M * KT / S;
    const double c = M <= 16 ? rows * (0.45 + 0.32 * p.uw + 0.034 * p.uw * (GU - 1)) + 0.88 * p.uw + x + (S > 1 ? 2.8 + sums / 4.2e6 : 0.0)
                             : rows * (0.2 + 0.61 * p.uw + 0.08 * p.uw * (GU - 1)) + 0.54 * p.uw + x + (S > 1 ? 3.6 + sums / 5.4e6 : 0.0);
    if (least < 0.0 || c < least) {
      least = c;
      best = p;
    }
    if (S > 1 && p.uw == 1) break;
  }
  return best;
}

template <int UW, int GU, int MB>
void launch_gemv(const Int4Args& a, int nb, hipStream_t s) {
  if (a.S > 1) hipLaunchKernelGGL((int4_gemv_kernel<UW, GU, true, MB>), dim3(nb * a.S), dim3(kW * 64), 0, s, a);
  else hipLaunchKernelGGL((int4_gemv_kernel<UW, GU, false, MB>), dim3(nb), dim3(kW * 64), 0, s, a);
}
template <int GU>
void launch_gemv_uw(const GemvPlan& p, const Int4Args& a, hipStream_t s) {
  if (a.M > 16) {
    if constexpr (GU <= 2) {
      if (p.uw == 2) return launch_gemv<2, GU, 2>(a, p.nb, s);
    }
    return launch_gemv<1, GU, 2>(a, p.nb, s);
  }
  if (p.uw == 1) return launch_gemv<1, GU, 1>(a, p.nb, s);
  if constexpr (GU <= 2) {
    if (p.uw == 3) return launch_gemv<3, GU, 1>(a, p.nb, s);
  }
  if constexpr (GU == 1) {
    if (p.uw == 4) return launch_gemv<4, GU, 1>(a, p.nb, s);
  }
  launch_gemv<2, GU, 1>(a, p.nb, s);
}

// ---------------------------------------------------------------------------
// Prompts
// ---------------------------------------------------------------------------
// A 256-thread workgroup computes 16 RI rows x 128 outputs.  Wave (kh, side) owns the
// 64 outputs of its side over half kh of the inputs, so that every weight is unpacked
// by one wave only; the halves are added through LDS at the end.  A step is a tile of 128
// inputs: x goes global -> LDS (16-byte copies, XOR-swizzled, two stages), the weights straight into
// registers, both one step ahead.  A step begins by waiting for all of them: copies in assembly and
// loads that the compiler places cannot be told apart by number.
// The products run on the codes, exact in fp16, and the sums of 64 inputs (32 in groups of 32)
// are scaled in fp32: a fused multiply-add per accumulator, where weights of fp16(code * scale)
// would need none but be off by 2^-11 each, and infinite for scales above 8188.
constexpr int kGThreads = 256;
__device__ __forceinline__ int aswz(int r) { return r & 15; }         // 256-byte rows

__device__ __forceinline__ void lds_read_barrier() {
  asm volatile("s_waitcnt lgkmcnt(0)\n\ts_barrier" ::: "memory");
}

template <int RI, int GU, bool PART>
__global__ __launch_bounds__(kGThreads, RI <= 4 && (RI == 2 || GU < 4) ? 3 : 2) void int4_gemm_kernel(Int4Args a) {
  constexpr int TN = 4;
  constexpr int kStageBytes = 16 * RI * 256;
  constexpr int kCopies = kStageBytes / 1024 / 4;       // per wave and step
  constexpr int kRed = 4 * (RI / 2) * TN * 1024;
  __shared__ __attribute__((aligned(1024))) uint8_t smem[2 * kStageBytes > kRed ? 2 * kStageBytes : kRed];

  const int tid = threadIdx.x;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int lane = tid & 63;
  const int col = lane & 15;
  const int grp = lane >> 4;
  const int kh = wave >> 1, side = wave & 1;
  const int M = a.M, N = a.N, K = a.K;
  const int m0 = blockIdx.y * (16 * RI);
  const int nt0 = blockIdx.x * 8 + side * 4;
  // this workgroup's 128-input tiles
  const int kt0 = PART ? (int)((int64_t)a.KT * blockIdx.z / gridDim.z) : 0;
  const int kt1 = PART ? (int)((int64_t)a.KT * (blockIdx.z + 1) / gridDim.z) : a.KT;

  // 16-byte chunk g of row r of a tile lies in slot g ^ aswz(r).  Rows past M read the last row.
  const uint32_t lds0 = (uint32_t)(uintptr_t)(lds_void_t*)smem;
  const uint8_t* xbase = static_cast<const uint8_t*>(uniform(a.x + (int64_t)m0 * a.ldx));
  // slot c of the stage: its chunk's bytes from row m0, tile 0 (ldx is below 2^23)
  auto chunk = [&](int c) { return (c & 15) ^ aswz(c >> 4); };
  auto offset = [&](int c) { return (uint32_t)min(c >> 4, M - 1 - m0) * (uint32_t)(a.ldx * 2) + chunk(c) * 16; };
  uint32_t aoff[kCopies];
#pragma unroll
  for (int i = 0; i < kCopies; ++i) aoff[i] = offset((wave * kCopies + i) * 64 + lane);
  auto copy = [&](int kt, int stage) {
    const uint32_t base = lds0 + stage * kStageBytes + wave * kCopies * 1024;
    const uint8_t* xb = xbase + (int64_t)kt * 256;
    if ((kt + 1) * 128 <= K) {
#pragma unroll
      for (int i = 0; i < kCopies; ++i) copy_to_lds(xb, aoff[i], base + i * 1024);
      return;
    }
    // K ends inside the tile: zeros past it (against weights of 0 an infinity would give NaN)
    int c = wave * kCopies * 64 + lane;
    asm volatile("" : "+v"(c));         // (nothing of this is kept in registers around the loop)
#pragma unroll 1
    for (int i = 0; i < kCopies; ++i, c += 64) {
      if (kt * 128 + chunk(c) * 8 < K) copy_to_lds(xb, offset(c), base + i * 1024);
      else *reinterpret_cast<uint4*>(smem + stage * kStageBytes + c * 16) = uint4{};
    }
  };

  // a tile's weights of this wave: words 2 kh, 2 kh + 1 and their scales
  constexpr int SG = GU == 4 ? 2 : 1;   // scales per half tile
  typedef uint32_t u32x2_t __attribute__((ext_vector_type(2)));
  struct BBuf {
    u32x2_t w[TN];
    uint16_t s[TN][SG];
  };
  // (buffer loads: offsets of a tile are scalar)
  const int ntb = min(nt0, a.NT - 1), tiles = min(TN, a.NT - ntb) * a.KT;
  const auto wrsrc = __builtin_amdgcn_make_buffer_rsrc(const_cast<uint32_t*>(a.w + (int64_t)ntb * a.KT * kTileWords), 0,
                                                       tiles * 1024, 0x20000);
  const auto srsrc = __builtin_amdgcn_make_buffer_rsrc(const_cast<uint16_t*>(a.scale + (int64_t)ntb * a.KT * (GU * 16)), 0,
                                                       tiles * (GU * 32), 0x20000);
  const int wv = lane * 16 + kh * 8, sv = col * 2 + (GU == 4 ? 2 * kh : GU == 2 ? kh : 0) * 32;
  auto load = [&](BBuf& b, int kt) {
#pragma unroll
    for (int j = 0; j < TN; ++j) {
      const int tile = (min(nt0 + j, a.NT - 1) - ntb) * a.KT + kt;
      b.w[j] = __builtin_amdgcn_raw_buffer_load_b64(wrsrc, wv, tile * 1024, 0);
#pragma unroll
      for (int g = 0; g < SG; ++g) b.s[j][g] = __builtin_amdgcn_raw_buffer_load_b16(srsrc, sv + 32 * g, tile * (GU * 32), 0);
    }
  };

  f4_t acc[RI][TN];
#pragma unroll
  for (int i = 0; i < RI; ++i)
#pragma unroll
    for (int j = 0; j < TN; ++j) acc[i][j] = f4_t{0.f, 0.f, 0.f, 0.f};

  const Unpack unpack;
  // Tile kt from `stage` and b; the next one's requests go out as soon as their places are free:
  // every wave has read the other stage before it came to the barrier.
  BBuf b;
  auto tile = [&](int kt, int stage) {
    const uint8_t* As = smem + stage * kStageBytes;
    wait_vm<0>();
    lds_read_barrier();
    if (kt + 1 < kt1) copy(kt + 1, 1 - stage);
    h8_t bf[2][TN];
    float sc[SG][TN];
#pragma unroll
    for (int j = 0; j < TN; ++j) {
#pragma unroll
      for (int h = 0; h < 2; ++h) bf[h][j] = word_codes(unpack, b.w[j][h]);
#pragma unroll
      for (int g = 0; g < SG; ++g) sc[g][j] = h2f(b.s[j][g]);
    }
    __builtin_amdgcn_sched_barrier(0);
    if (kt + 1 < kt1) load(b, kt + 1);
    // Operands of row tile i + 1 are read, and the sums of the one before are scaled, beside the products
    // of i; a barrier of the schedule after each keeps no more than that in registers.
    auto rows = [&](int i, int h) {
      const int r = 16 * i + col;
      return *reinterpret_cast<const h8_t*>(As + r * 256 + (((8 * kh + 4 * h + grp) ^ aswz(r)) << 4));
    };
    constexpr bool kAhead = RI != 4;    // (three workgroups a CU leave no registers for it)
    h8_t af[2], nf[2];
    if (kAhead) {
      nf[0] = rows(0, 0);
      nf[1] = rows(0, 1);
    }
    f4_t last[TN];
    auto scaled = [&](int s) {          // sum s: row tile s / SG, scale s % SG
#pragma unroll
      for (int j = 0; j < TN; ++j)
#pragma unroll
        for (int q = 0; q < 4; ++q)
          acc[s / SG][j][q] = fmaf(sc[s % SG][j], last[j][q], acc[s / SG][j][q]);
    };
#pragma unroll
    for (int s = 0; s < RI * SG; ++s) {
      const int i = s / SG;
      if (s % SG == 0) {
        af[0] = kAhead ? nf[0] : rows(i, 0);
        af[1] = kAhead ? nf[1] : rows(i, 1);
      }
      if (kAhead && s % SG == 0 && i + 1 < RI) {
        nf[0] = rows(i + 1, 0);
        nf[1] = rows(i + 1, 1);
      }
      f4_t c[TN];
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        if (SG == 2 && h != s % 2) continue;
#pragma unroll
        for (int j = 0; j < TN; ++j)
          c[j] = __builtin_amdgcn_mfma_f32_16x16x32_f16(af[h], bf[h][j], SG == 2 || h == 0 ? f4_t{0.f, 0.f, 0.f, 0.f} : c[j], 0, 0, 0);
      }
      if (s > 0) scaled(s - 1);
#pragma unroll
      for (int j = 0; j < TN; ++j) last[j] = c[j];
      __builtin_amdgcn_sched_barrier(0);
    }
    scaled(RI * SG - 1);
  };

  copy(kt0, 0);
  load(b, kt0);
  for (int kt = kt0; kt < kt1; ++kt) tile(kt, (kt - kt0) & 1);

  // wave (kh, side) keeps half of the row tiles and hands the others to wave ^ 2
  __syncthreads();
  f4_t* red = reinterpret_cast<f4_t*>(smem);
  auto finish = [&](auto keep_c) {
    constexpr int H = RI / 2;
    constexpr int keep = decltype(keep_c)::value;
    constexpr int give = H - keep;
#pragma unroll
    for (int i = 0; i < H; ++i)
#pragma unroll
      for (int j = 0; j < TN; ++j) red[((wave * H + i) * TN + j) * 64 + lane] = acc[give + i][j];
    __syncthreads();
    const int partner = wave ^ 2;
#pragma unroll
    for (int j = 0; j < TN; ++j) {
      const int n = (nt0 + j) * 16 + col;
      if (n >= N) continue;
      const float bs = !PART && a.bias ? h2f(a.bias[n]) : 0.f;
#pragma unroll
      for (int i = 0; i < H; ++i) {
        const f4_t o = red[((partner * H + i) * TN + j) * 64 + lane];
#pragma unroll
        for (int r = 0; r < 4; ++r) {
          const int m = m0 + (keep + i) * 16 + grp * 4 + r;
          if (m >= M) continue;
          const float v = acc[keep + i][j][r] + o[r];
          if constexpr (PART) a.part[((int64_t)blockIdx.z * M + m) * a.np + n] = v;
          else a.y[(int64_t)m * a.ldy + n] = f2h(v + bs);
        }
      }
    }
  };
  if (kh == 0) finish(std::integral_constant<int, 0>{});
  else finish(std::integral_constant<int, RI / 2>{});
}

// Row tiles (16 RI rows) and k slices of a prompt, by the time of a slice's 128-input tiles: a
// CU's workgroups share its matrix and vector units (us per tile for each that it gets; groups of 32
// scale twice the sums), and a round of as many as its registers hold takes at least a wave's own
// latencies; slices add the partial sums' way out and back and a second launch.  Fitted to 2937 timed
// (shape, RI, S) of 33 to 2048 tokens, over half of them within 4% and 90% within 10%; what it picks
// is 1% off the fastest on average, 11% at most.  1500 x 4096 -> 12288 takes 166 us in tiles of 96 rows
// (exactly six workgroups a CU), 169 in 64 and 170 in 128; 512 x 5120 -> 17408 takes 119 us in tiles of 64
// and 130 in 96 or 128.
constexpr int gemm_workgroups(int ri, int GU) { return ri == 2 ? (GU < 4 ? 4 : 3) : ri == 4 && GU < 4 ? 3 : 2; }   // of a CU
struct GemmPlan {
  int ri, S;
};
GemmPlan plan_gemm(int M, int NT, int KT, int GU) {
  GemmPlan p{8, 1};
  double least = -1.0;
  for (int ri = 2; ri <= 8; ri += 2) {
    const int64_t tiles = (int64_t)((NT + 7) / 8) * ((M + 16 * ri - 1) / (16 * ri));
    const int64_t slots = 256 * gemm_workgroups(ri, GU);
    for (int S = 1; S <= std::min(KT, 16); ++S) {
      const int64_t w = tiles * S;
      const double shared = (double)((w + 255) / 256) * (0.157 + (GU < 4 ? 0.1 : 0.132) * ri);
      const double alone = (double)((w + slots - 1) / slots) * (0.294 + (GU < 4 ? 0.117 : 0.171) * ri);
      const double c = ((KT + S - 1) / S) * std::max(shared, alone) + (S > 1 ? 2.97 + (double)S * M * NT * 128.0 / 6.26e6 : 0.0);
      if (least < 0.0 || c < least) {
        least = c;
        p = {ri, S};
      }
    }
    if (16 * ri >= M) break;            // taller than the rows need
  }
  return p;
}

template <int RI, int GU>
void launch_gemm(const Int4Args& a, hipStream_t s) {
  const dim3 grid((a.NT + 7) / 8, (a.M + 16 * RI - 1) / (16 * RI), a.S);
  if (a.S > 1) hipLaunchKernelGGL((int4_gemm_kernel<RI, GU, true>), grid, dim3(kGThreads), 0, s, a);
  else hipLaunchKernelGGL((int4_gemm_kernel<RI, GU, false>), grid, dim3(kGThreads), 0, s, a);
}
template <int GU>
void launch_gemm_ri(int ri, const Int4Args& a, hipStream_t s) {
  if (ri == 2) launch_gemm<2, GU>(a, s);
  else if (ri == 4) launch_gemm<4, GU>(a, s);
  else if (ri == 6) launch_gemm<6, GU>(a, s);
  else launch_gemm<8, GU>(a, s);
}

}  // namespace

extern "C" int64_t helm_int4_linear_workspace_bytes(int M, int N, int K, int group_size) {
  if (M < 1 || N < 1 || K < 1 || N > (1 << 27) || K > (1 << 19)) return 0;
  if (group_size != 32 && group_size != 64 && group_size != 128) return 0;
  const int NT = (N + 15) / 16, KT = (K + 127) / 128;
  const int S = M <= kGemvTokens ? plan_gemv(M, NT, KT, 128 / group_size).S : plan_gemm(M, NT, KT, 128 / group_size).S;
  return S > 1 ? (int64_t)S * M * NT * 16 * (int64_t)sizeof(float) : 0;
}

extern "C" int helm_int4_linear_form(int M, int N, int K, int group_size, int32_t* form) {
  HELM_CHECK_ARG(form, "helm_int4_linear_form: null pointer");
  HELM_CHECK_ARG(M >= 1 && N >= 1 && K >= 1, "helm_int4_linear_form: M, N, K must be positive");
  HELM_CHECK_SUPPORTED(N <= (1 << 27) && K <= (1 << 19) && M <= (1 << 22), "helm_int4_linear_form: shape too large");
  HELM_CHECK_SUPPORTED((group_size == 32 || group_size == 64 || group_size == 128) && K % group_size == 0,
                       "helm_int4_linear_form: group size must be 32, 64 or 128 and divide K");
  const int NT = (N + 15) / 16, KT = (K + 127) / 128, GU = 128 / group_size;
  if (M <= kGemvTokens) {
    const GemvPlan p = plan_gemv(M, NT, KT, GU);
    form[0] = M > 16 ? 2 : 1;
    form[1] = p.uw;
    form[2] = p.S;
  } else {
    const GemmPlan p = plan_gemm(M, NT, KT, GU);
    form[0] = 0;
    form[1] = 16 * p.ri;
    form[2] = p.S;
  }
  return HELM_OK;
}

extern "C" int helm_int4_linear(const void* x, int64_t ldx, const void* qweight, const void* scale,
                                int group_size, const void* bias, void* y, int64_t ldy, int M, int N, int K,
                                void* workspace, int64_t workspace_bytes, void* stream) {
  HELM_CHECK_ARG(x && qweight && scale && y, "helm_int4_linear: null pointer");
  HELM_CHECK_ARG(M >= 1 && N >= 1 && K >= 1, "helm_int4_linear: M, N, K must be positive");
  HELM_CHECK_SUPPORTED(N <= (1 << 27) && K <= (1 << 19) && M <= (1 << 22), "helm_int4_linear: shape too large");
  HELM_CHECK_ARG(ldx >= K && ldy >= N, "helm_int4_linear: leading dimension too small");
  HELM_CHECK_SUPPORTED(group_size == 32 || group_size == 64 || group_size == 128,
                       "helm_int4_linear: group size must be 32, 64 or 128");
  HELM_CHECK_SUPPORTED(K % group_size == 0, "helm_int4_linear: K must be a multiple of the group size");
  HELM_CHECK_SUPPORTED(M == 1 || ldx <= (1 << 23), "helm_int4_linear: ldx above 2^23");
  HELM_CHECK_SUPPORTED(ldx % 8 == 0 && helm::aligned16(x) && helm::aligned16(qweight) && helm::aligned16(scale),
                       "helm_int4_linear: x rows, qweight and scale must be 16-byte aligned");
  Int4Args a{};
  a.x = static_cast<const uint16_t*>(x); a.ldx = ldx;
  a.w = static_cast<const uint32_t*>(qweight);
  a.scale = static_cast<const uint16_t*>(scale);
  a.bias = static_cast<const uint16_t*>(bias);
  a.y = static_cast<uint16_t*>(y); a.ldy = ldy;
  a.M = M; a.N = N; a.K = K;
  a.NT = (N + 15) / 16; a.KT = (K + 127) / 128; a.np = a.NT * 16;
  const int GU = 128 / group_size;
  const GemvPlan gp = M <= kGemvTokens ? plan_gemv(M, a.NT, a.KT, GU) : GemvPlan{};
  const GemmPlan mp = M <= kGemvTokens ? GemmPlan{} : plan_gemm(M, a.NT, a.KT, GU);
  a.S = M <= kGemvTokens ? gp.S : mp.S;
  const int64_t need = a.S > 1 ? (int64_t)a.S * M * a.np * (int64_t)sizeof(float) : 0;
  HELM_CHECK_ARG(need == 0 || (workspace && helm::aligned16(workspace) && workspace_bytes >= need),
                 "helm_int4_linear: this shape needs " + std::to_string(need) + " bytes of 16-byte aligned workspace");
  a.part = static_cast<float*>(workspace);
  const hipStream_t s = static_cast<hipStream_t>(stream);
  if (M <= kGemvTokens) {
    if (GU == 1) launch_gemv_uw<1>(gp, a, s);
    else if (GU == 2) launch_gemv_uw<2>(gp, a, s);
    else launch_gemv_uw<4>(gp, a, s);
  } else {
    HELM_CHECK_SUPPORTED((M + 16 * mp.ri - 1) / (16 * mp.ri) <= 65535, "helm_int4_linear: too many rows");
    if (GU == 1) launch_gemm_ri<1>(mp.ri, a, s);
    else if (GU == 2) launch_gemm_ri<2>(mp.ri, a, s);
    else launch_gemm_ri<4>(mp.ri, a, s);
  }
  HELM_CHECK_LAUNCH("helm_int4_linear launch");
  if (a.S > 1) {
    const int64_t n = (int64_t)M * (a.np / 4);
    hipLaunchKernelGGL(int4_reduce_kernel, dim3((unsigned)((n + 255) / 256)), dim3(256), 0, s, a.part, a.S, a.np,
                       a.bias, a.y, a.ldy, M, N);
    HELM_CHECK_LAUNCH("helm_int4_linear reduce launch");
  }
  return HELM_OK;
}
