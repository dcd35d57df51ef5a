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
// input 2p / 2p + 1 at bit 4p of either: one shift, mask and or give two fp16
// numbers 16 + u (u = c + 8 in the top mantissa bits of [16, 32)), exactly.
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

// Pair p of a word as two fp16 numbers 16 + u (exact).
template <int PAIR>
__device__ __forceinline__ uint32_t pair16(uint32_t w) {
  constexpr int sh = 6 - 4 * PAIR;
  const uint32_t v = sh >= 0 ? w << (sh >= 0 ? sh : 0) : w >> (sh < 0 ? -sh : 0);
  return (v & 0x03C003C0u) | 0x4C004C00u;
}
__device__ __forceinline__ h8_t word16(uint32_t w) {
  const u32x4_t r = {pair16<0>(w), pair16<1>(w), pair16<2>(w), pair16<3>(w)};
  return __builtin_bit_cast(h8_t, r);
}

// ---------------------------------------------------------------------------
// 1 to 16 tokens
// ---------------------------------------------------------------------------
// Bound by the weight stream.  x^T operands of a wave's inputs stay in registers;
// a workgroup's eight waves split the inputs of a k slice (UW tiles each) and walk
// row tiles tb, tb + nb, ..., the next row tile's weights requested before this
// one's products.  The products run on 16 + u; the -24 sum(x) that turns them into
// codes is the same for every output, so it is computed once per wave and group (an
// MFMA with a constant operand) and starts each accumulation.  It costs no accuracy:
// the sums are fp32 and 24 is 3 times the largest code.  A group's sum is scaled by
// its outputs' scales in fp32.
constexpr int kW = 8;
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

// UW: tiles of a wave's k share.  GU: groups per tile.
template <int UW, int GU, bool PART>
__global__ __launch_bounds__(kW * 64) void int4_gemv_kernel(Int4Args a) {
  __shared__ __attribute__((aligned(16))) f4_t s_c[2][kW][64];
  __shared__ float s_bias[PART ? 1 : kMaxTiles * 16];
  constexpr int TG = 4 / GU;          // MFMAs per group

  const int tid = threadIdx.x;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int lane = tid & 63;
  const int col = lane & 15;
  const int grp = lane >> 4;
  const int M = a.M;

  const int sl = PART ? (int)blockIdx.x % a.S : 0;
  const int tb = PART ? (int)blockIdx.x / a.S : (int)blockIdx.x;
  const int nb = PART ? (int)gridDim.x / a.S : (int)gridDim.x;
  const int T = tb < a.NT ? (a.NT - 1 - tb) / nb + 1 : 0;
  const int sa = (int)((int64_t)sl * a.KT / a.S), sn = (int)((int64_t)(sl + 1) * a.KT / a.S) - sa;
  const int u0 = sa + wave * sn / kW, u1 = sa + (wave + 1) * sn / kW;   // at most UW tiles

  struct Buf {
    uint4 w[UW];
    uint2 s[UW][GU];
  };
  // Row tile tb + t nb (clamped to the last one) of this wave's k share; tiles past the
  // share re-read its last one (their x operands are zero).
  auto load = [&](Buf& b, int t) {
    const int64_t row = (int64_t)min(tb + t * nb, a.NT - 1) * a.KT;
#pragma unroll
    for (int u = 0; u < UW; ++u) {
      const int64_t tile = row + min(min(u0 + u, max(u1 - 1, u0)), a.KT - 1);
      b.w[u] = ld_nt16(a.w + tile * kTileWords + lane * 4);
#pragma unroll
      for (int g = 0; g < GU; ++g)
        b.s[u][g] = *reinterpret_cast<const uint2*>(a.scale + (tile * GU + g) * 16 + grp * 4);
    }
  };
  Buf b0, b1;
  load(b0, 0);

  h8_t xr[UW][4];
  const uint16_t* xrow = a.x + (int64_t)min(col, M - 1) * a.ldx;
#pragma unroll
  for (int u = 0; u < UW; ++u)
#pragma unroll
    for (int t = 0; t < 4; ++t) {
      const int k = (u0 + u) * 128 + t * 32 + grp * 8;
      xr[u][t] = *reinterpret_cast<const h8_t*>(xrow + min(k, a.K - 8));
      if (u0 + u >= u1 || k >= a.K) xr[u][t] = h8_t{};
    }
  if constexpr (!PART) {
    for (int i = tid; i < T * 16; i += kW * 64) {
      const int n = min((tb + (i >> 4) * nb) * 16 + (i & 15), a.N - 1);
      s_bias[i] = a.bias ? h2f(a.bias[n]) : 0.f;
    }
  }
  // -24 * (sum of a group's x): every row of the product with a constant operand
  float nbias[UW][GU];
  {
    h8_t c;
#pragma unroll
    for (int e = 0; e < 8; ++e) c[e] = (_Float16)-24.0f;
#pragma unroll
    for (int u = 0; u < UW; ++u)
#pragma unroll
      for (int g = 0; g < GU; ++g) {
        f4_t s = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int t = 0; t < TG; ++t) s = __builtin_amdgcn_mfma_f32_16x16x32_f16(c, xr[u][g * TG + t], s, 0, 0, 0);
        nbias[u][g] = s[0];
      }
  }
  lds_barrier();

  auto tile = [&](const Buf& b, int t) {
    f4_t acc = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
    for (int u = 0; u < UW; ++u) {
      const uint32_t wd[4] = {b.w[u].x, b.w[u].y, b.w[u].z, b.w[u].w};
#pragma unroll
      for (int g = 0; g < GU; ++g) {
        const float z = nbias[u][g];
        f4_t c = {z, z, z, z};
#pragma unroll
        for (int q = 0; q < TG; ++q)
          c = __builtin_amdgcn_mfma_f32_16x16x32_f16(word16(wd[g * TG + q]), xr[u][g * TG + q], c, 0, 0, 0);
        acc[0] = fmaf(lo_h(b.s[u][g].x), c[0], acc[0]);
        acc[1] = fmaf(hi_h(b.s[u][g].x), c[1], acc[1]);
        acc[2] = fmaf(lo_h(b.s[u][g].y), c[2], acc[2]);
        acc[3] = fmaf(hi_h(b.s[u][g].y), c[3], acc[3]);
      }
    }
    f4_t (*sc)[64] = s_c[t & 1];
    sc[wave][lane] = acc;
    lds_barrier();      // buffer t & 1 is written again only after tile t + 1's barrier
    if (wave == (t & (kW - 1))) {
      f4_t v = sc[0][lane];
#pragma unroll
      for (int w = 1; w < kW; ++w) {
        const f4_t o = sc[w][lane];
#pragma unroll
        for (int r = 0; r < 4; ++r) v[r] += o[r];
      }
      const int n0 = (tb + t * nb) * 16 + grp * 4;   // v[r]: output n0 + r of token col
      if (col < M && n0 < a.N) {
        if constexpr (PART) {
          *reinterpret_cast<f4_t*>(a.part + ((int64_t)sl * M + col) * a.np + n0) = v;
        } else {
          uint16_t* yp = a.y + (int64_t)col * a.ldy + n0;
#pragma unroll
          for (int r = 0; r < 4; ++r)
            if (n0 + r < a.N) yp[r] = f2h(v[r] + s_bias[t * 16 + grp * 4 + r]);
        }
      }
    }
  };
  int t = 0;
  for (; t + 1 < T; t += 2) {
    load(b1, t + 1);
    tile(b0, t);
    if (t + 2 < T) load(b0, t + 2);
    tile(b1, t + 1);
  }
  if (t < T) tile(b0, t);
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
  for (int s = 0; s < S; ++s) {
    const f4_t o = *reinterpret_cast<const f4_t*>(part + ((int64_t)s * M + m) * np + n);
#pragma unroll
    for (int r = 0; r < 4; ++r) v[r] += o[r];
  }
#pragma unroll
  for (int r = 0; r < 4; ++r)
    if (n + r < N) y[(int64_t)m * ldy + n + r] = f2h(v[r] + (bias ? h2f(bias[n + r]) : 0.f));
}

// k slices and tiles per wave of a GEMV: the fewest slices of at most kMaxUw tiles per
// wave.
constexpr int kMaxUw = 6;
struct GemvPlan {
  int S, uw;
};
GemvPlan plan_gemv(int NT, int KT) {
  (void)NT;
  GemvPlan p;
  p.S = (KT + kW * kMaxUw - 1) / (kW * kMaxUw);
  const int sn = (KT + p.S - 1) / p.S;
  p.uw = (sn + kW - 1) / kW;
  return p;
}

template <int UW, int GU>
void launch_gemv(const Int4Args& a, hipStream_t s) {
  const int nb = std::max(std::min(a.NT, std::max(1, 256 / a.S)), (a.NT + kMaxTiles - 1) / kMaxTiles);
  if (a.S > 1) hipLaunchKernelGGL((int4_gemv_kernel<UW, GU, true>), dim3(nb * a.S), dim3(kW * 64), 0, s, a);
  else hipLaunchKernelGGL((int4_gemv_kernel<UW, GU, false>), dim3(nb), dim3(kW * 64), 0, s, a);
}
template <int GU>
void launch_gemv_uw(int uw, const Int4Args& a, hipStream_t s) {
  switch (uw) {
    case 1: return launch_gemv<1, GU>(a, s);
    case 2: return launch_gemv<2, GU>(a, s);
    case 3: return launch_gemv<3, GU>(a, s);
    case 4: return launch_gemv<4, GU>(a, s);
    case 5: return launch_gemv<5, GU>(a, s);
    default: return launch_gemv<6, GU>(a, s);
  }
}

// ---------------------------------------------------------------------------
// Prompts
// ---------------------------------------------------------------------------
// A 256-thread workgroup computes 16 RI rows x 128 outputs.  Wave (kh, side) owns the
// 64 outputs of its side over half kh of the inputs, so that every weight is turned
// into fp16 by one wave only; the halves are added through LDS at the end.  x goes
// global -> LDS (16-byte copies, XOR-swizzled, a ring of three 64-input steps), the
// weights straight into registers, a tile ahead.  A weight enters the products as
// fp16(code * scale), the number that Int4Weight.dequantize() gives rounded to fp16: one
// rounding of 2^-12 relative at most, and it spares a scaling of every accumulator
// per group.
constexpr int kGThreads = 256;
constexpr int kStages = 3;
__device__ __forceinline__ int aswz(int r) { return (r >> 1) & 7; }   // 128-byte rows

template <int N>
__device__ __forceinline__ void wait_vm() {
  static_assert(N >= 0 && N < 64, "vmcnt range");
  asm volatile("" ::: "memory");
  __builtin_amdgcn_s_waitcnt((N & 15) | (7 << 4) | (15 << 8) | ((N >> 4) << 14));
  asm volatile("" ::: "memory");
}
// One wave's 1 KiB global -> LDS copy: lane l moves 16 bytes from `src` to LDS byte
// lds + 16 l; waited for by the kernel itself.
#pragma clang diagnostic push
#pragma clang diagnostic ignored "-Winline-asm"   // m0 is named as clobbered on purpose
__device__ __forceinline__ void copy_to_lds(const void* src, uint32_t lds) {
  asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %1, off"
               :
               : "s"(__builtin_amdgcn_readfirstlane(lds)), "v"(src)
               : "memory", "m0");
}
#pragma clang diagnostic pop
__device__ __forceinline__ void lds_read_barrier() {
  asm volatile("s_waitcnt lgkmcnt(0)\n\ts_barrier" ::: "memory");
}

// Word of eight codes times a scale, each product rounded to fp16 once (16 + u - 24 is
// exact).
__device__ __forceinline__ h8_t word_scaled(uint32_t w, h2_t s) {
  const h2_t off = {(_Float16)-24.0f, (_Float16)-24.0f};
  const uint32_t p[4] = {pair16<0>(w), pair16<1>(w), pair16<2>(w), pair16<3>(w)};
  h8_t r;
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const h2_t v = (__builtin_bit_cast(h2_t, p[i]) + off) * s;
    r[2 * i] = v[0];
    r[2 * i + 1] = v[1];
  }
  return r;
}

template <int RI, int GU, bool PART>
__global__ __launch_bounds__(kGThreads, 2) void int4_gemm_kernel(Int4Args a) {
  constexpr int TN = 4;
  constexpr int kStageBytes = 16 * RI * 128;
  constexpr int kCopies = kStageBytes / 1024 / 4 > 0 ? kStageBytes / 1024 / 4 : 1;   // per wave and step
  constexpr int kRing = kStages * kStageBytes;
  constexpr int kRed = 4 * (RI / 2) * TN * 1024;
  __shared__ __attribute__((aligned(1024))) uint8_t smem[kRing > kRed ? kRing : kRed];

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
  const int nk = 2 * (kt1 - kt0);      // steps: two per tile

  // Step s of a tile holds inputs 32 s .. + 32 and 64 + 32 s .. + 32 of its 128 (chunks
  // 0-3 and 4-7 of a row: the two waves' halves), chunk g of row r in slot g ^ aswz(r).
  // Rows past M read the last row, inputs past K the row's last chunk (weights there are
  // zero).
  int64_t arow[kCopies];
  int akc[kCopies];
#pragma unroll
  for (int i = 0; i < kCopies; ++i) {
    const int c = (wave * kCopies + i) * 64 + lane;
    const int r = c >> 3;
    const int g = (c & 7) ^ aswz(r);
    arow[i] = (int64_t)min(m0 + r, M - 1) * a.ldx;
    akc[i] = (g >> 2) * 64 + (g & 3) * 8;
  }
  const uint32_t lds0 = (uint32_t)(uintptr_t)(lds_void_t*)smem;
  auto copy = [&](int kb) {
    const uint32_t base = lds0 + (kb % kStages) * kStageBytes;
    const int k0 = (kt0 + (kb >> 1)) * 128 + (kb & 1) * 32;
#pragma unroll
    for (int i = 0; i < kCopies; ++i)
      copy_to_lds(a.x + arow[i] + min(k0 + akc[i], K - 8), base + (wave * kCopies + i) * 1024);
  };

  // a tile's weights of this wave: words 2 kh, 2 kh + 1 and their scales
  constexpr int SG = GU == 4 ? 2 : 1;   // scales per half tile
  struct BBuf {
    uint2 w[TN];
    uint16_t s[TN][SG];
  };
  auto load = [&](BBuf& b, int kt) {
#pragma unroll
    for (int j = 0; j < TN; ++j) {
      const int64_t tile = (int64_t)min(nt0 + j, a.NT - 1) * a.KT + min(kt, kt1 - 1);
      b.w[j] = *reinterpret_cast<const uint2*>(a.w + tile * kTileWords + lane * 4 + 2 * kh);
#pragma unroll
      for (int g = 0; g < SG; ++g)
        b.s[j][g] = a.scale[(tile * GU + (GU == 4 ? 2 * kh + g : GU == 2 ? kh : 0)) * 16 + col];
    }
  };

  f4_t acc[RI][TN];
#pragma unroll
  for (int i = 0; i < RI; ++i)
#pragma unroll
    for (int j = 0; j < TN; ++j) acc[i][j] = f4_t{0.f, 0.f, 0.f, 0.f};

  auto step = [&](const BBuf& b, int kb, auto half_c) {
    constexpr int half = decltype(half_c)::value;
    if (kb + 1 < nk) wait_vm<kCopies>();
    else wait_vm<0>();
    lds_read_barrier();
    if (kb + 2 < nk) copy(kb + 2);
    const uint8_t* As = smem + (kb % kStages) * kStageBytes;
    h8_t af[RI];
#pragma unroll
    for (int i = 0; i < RI; ++i) {
      const int r = 16 * i + col;
      af[i] = *reinterpret_cast<const h8_t*>(As + r * 128 + (((4 * kh + grp) ^ aswz(r)) << 4));
    }
#pragma unroll
    for (int j = 0; j < TN; ++j) {
      const _Float16 s1 = __builtin_bit_cast(_Float16, b.s[j][SG == 2 ? half : 0]);
      const h8_t bf = word_scaled(half ? b.w[j].y : b.w[j].x, h2_t{s1, s1});
#pragma unroll
      for (int i = 0; i < RI; ++i)
        acc[i][j] = __builtin_amdgcn_mfma_f32_16x16x32_f16(af[i], bf, acc[i][j], 0, 0, 0);
    }
  };

  BBuf b0, b1;
  load(b0, kt0);
  copy(0);
  if (nk > 1) copy(1);
  int kt = kt0;
  for (; kt + 1 < kt1; kt += 2) {
    const int kb = 2 * (kt - kt0);
    load(b1, kt + 1);
    step(b0, kb, std::integral_constant<int, 0>{});
    step(b0, kb + 1, std::integral_constant<int, 1>{});
    load(b0, kt + 2);
    step(b1, kb + 2, std::integral_constant<int, 0>{});
    step(b1, kb + 3, std::integral_constant<int, 1>{});
  }
  if (kt < kt1) {
    const int kb = 2 * (kt - kt0);
    step(b0, kb, std::integral_constant<int, 0>{});
    step(b0, kb + 1, std::integral_constant<int, 1>{});
  }

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

// Row tiles and k slices of a prompt: tiles as tall as the rows need, k split until the
// workgroups fill two per CU.
struct GemmPlan {
  int ri, S;
};
GemmPlan plan_gemm(int M, int NT, int KT) {
  GemmPlan p;
  p.ri = M <= 32 ? 2 : M <= 64 ? 4 : 8;
  const int64_t tiles = (int64_t)((NT + 7) / 8) * ((M + 16 * p.ri - 1) / (16 * p.ri));
  p.S = (int)std::max<int64_t>(1, std::min<int64_t>(std::min<int64_t>(512 / std::max<int64_t>(tiles, 1), KT / 4), 16));
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
  else launch_gemm<8, GU>(a, s);
}

int slices(int M, int NT, int KT) { return M <= 16 ? plan_gemv(NT, KT).S : plan_gemm(M, NT, KT).S; }

}  // namespace

extern "C" int64_t helm_int4_linear_workspace_bytes(int M, int N, int K) {
  if (M < 1 || N < 1 || K < 1 || N > (1 << 30) || K > (1 << 30)) return 0;
  const int NT = (N + 15) / 16, KT = (K + 127) / 128;
  const int S = slices(M, NT, KT);
  return S > 1 ? (int64_t)S * M * NT * 16 * (int64_t)sizeof(float) : 0;
}

extern "C" int helm_int4_linear(const void* x, int64_t ldx, const void* qweight, const void* scale,
                                int group_size, const void* bias, void* y, int64_t ldy, int M, int N, int K,
                                void* workspace, int64_t workspace_bytes, void* stream) {
  HELM_CHECK_ARG(x && qweight && scale && y, "helm_int4_linear: null pointer");
  HELM_CHECK_ARG(M >= 1 && N >= 1 && K >= 1, "helm_int4_linear: M, N, K must be positive");
  HELM_CHECK_SUPPORTED(N <= (1 << 30) && K <= (1 << 30) && M <= (1 << 22), "helm_int4_linear: shape too large");
  HELM_CHECK_ARG(ldx >= K && ldy >= N, "helm_int4_linear: leading dimension too small");
  HELM_CHECK_SUPPORTED(group_size == 32 || group_size == 64 || group_size == 128,
                       "helm_int4_linear: group size must be 32, 64 or 128");
  HELM_CHECK_SUPPORTED(K % group_size == 0, "helm_int4_linear: K must be a multiple of the group size");
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
  a.S = slices(M, a.NT, a.KT);
  const int64_t need = helm_int4_linear_workspace_bytes(M, N, K);
  HELM_CHECK_ARG(need == 0 || (workspace && helm::aligned16(workspace) && workspace_bytes >= need),
                 "helm_int4_linear: this shape needs " + std::to_string(need) + " bytes of 16-byte aligned workspace");
  a.part = static_cast<float*>(workspace);
  const hipStream_t s = static_cast<hipStream_t>(stream);
  if (M <= 16) {
    const int uw = plan_gemv(a.NT, a.KT).uw;
    if (group_size == 128) launch_gemv_uw<1>(uw, a, s);
    else if (group_size == 64) launch_gemv_uw<2>(uw, a, s);
    else launch_gemv_uw<4>(uw, a, s);
  } else {
    const int ri = plan_gemm(M, a.NT, a.KT).ri;
    HELM_CHECK_SUPPORTED((M + 16 * ri - 1) / (16 * ri) <= 65535, "helm_int4_linear: too many rows");
    if (group_size == 128) launch_gemm_ri<1>(ri, a, s);
    else if (group_size == 64) launch_gemm_ri<2>(ri, a, s);
    else launch_gemm_ri<4>(ri, a, s);
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
