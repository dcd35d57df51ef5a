// sample.hip — one token per row drawn from fp16 logits with temperature, top-k, top-p
// and min-p, from given random numbers.
//
// w_i = 2^((x_i - max) log2(e) / t).  An fp16 logit has a 16-bit key that orders like
// its value (equal values, equal keys), so every filter is a border (key, how many of its
// equals stay): no sort, and ties go to the lowest index.  Keys fall into 64 chunks of
// 1024 neighbours.  Two kernels:
//   * slices: a workgroup per 4096 logits lists their keys by chunk, the largest first, and sums
//     count and weight of each chunk;
//   * pick: a workgroup per row finds the chunk that holds a border from those sums and
//     resolves the key inside it from the few logits of that chunk, then the slice that
//     holds the drawn token, then the token.
// Weights of a chunk are summed in 2^-44 fixed point relative to the slice's largest, those of
// the border's chunk that stay in 2^-50 of what the chunk's stay below: sums of integers do not
// depend on their order, so atomics leave the result the same from run to run.  All else is in 64
// bits: a token next to a border decides a whole number.
// Bound by latency: the logits are read once by as many CUs as there are slices; then a
// row has four dependent round trips to memory (sums, the border's chunk, the slice's
// borders, its logits) and a scan after each, and one more for u and for settings of its own, which are
// read where they are needed.  Scans run over DPP, and every wave repeats
// the small ones for itself instead of waiting at a barrier for another.  A row of 151936 with
// top-k 20 and top-p 0.8 takes 16.5 us (5 of them the slices); 16 rows without filters 19, with
// top-p alone 31.5 (every logit is listed, and the border's chunk holds a third of them); 64 rows of
// 50257 with min-p 21.
#include "helm_common.h"

namespace {

constexpr int kSlice = 4096;          // logits of a slice
constexpr int kST = 512;              // threads of a slice: 8 logits each
constexpr int kPT = 1024;             // threads of a row's pick: one per key of a chunk
constexpr int kPW = kPT / 64;
constexpr int kChunks = 64;
constexpr int kRep = 16;              // replicas of the slice's counters (fewer conflicts)
constexpr int kMaxSlices = 64;        // one per lane of a wave
constexpr int kOwn = kMaxSlices / kPW;   // slices of a wave of the pick
constexpr int kDeep = 4;              // list loads of a lane in flight, for each of its wave's slices
constexpr uint32_t kNegInf = 0x03FFu; // key of -inf
constexpr uint32_t kPosInf = 0xFC00u; // key of +inf
constexpr double kFix = 17592186044416.0;   // 2^44
constexpr uint32_t kNone = 0xFFFFFFFFu;

struct SliceSums {
  uint32_t greedy_key, greedy_idx;    // NaN as the largest value
  uint32_t max_key, max_idx;          // NaN as -inf; idx: first of the largest in the slice
  uint64_t mass[kChunks];             // 2^44 sum of w relative to the slice's largest
  uint16_t cnt[kChunks];
  uint16_t off[kChunks];              // first entry of the chunk in the slice's list
};

struct SampleArgs {
  const uint16_t* x;
  int64_t ldx;
  int M, N, S;
  const float* u;
  const float* temperature;
  const int32_t* top_k;
  const float* top_p;
  const float* min_p;
  float t, p, lo;
  int k;
  SliceSums* sums;                    // [M][S]
  uint16_t* list;                     // [M][S][kSlice]: keys, largest chunk first
  int64_t* out;
};

__device__ __forceinline__ uint32_t key_of(uint16_t b) {   // not for NaN
  if (b == 0x8000u) b = 0;                                  // -0 equals 0
  return b & 0x8000u ? (uint32_t)(uint16_t)~b : (uint32_t)b | 0x8000u;
}
__device__ __forceinline__ double value_of(uint32_t key) {
  return (double)h2f((uint16_t)(key & 0x8000u ? key & 0x7fffu : ~key));
}
// 2^y for y <= 0: 2^(n / 64) from a table of 64, the rest (at most 2^-7 ln 2) by its series to
// the fifth power; off by a few 2^-53.
__device__ __forceinline__ double exp2_neg(double y, const double* tab) {
  const double n = rint(y * 64.0);
  const double r = fma(n, -1.0 / 64.0, y) * 0.69314718055994530942;
  const double p = fma(fma(fma(fma(fma(r, 1.0 / 120, 1.0 / 24), r, 1.0 / 6), r, 0.5), r, 1.0), r, 1.0);
  const int i = (int)fmax(n, -131072.0);
  return ldexp(p * tab[i & 63], i >> 6);
}
__device__ __forceinline__ double pow2(int e) {             // |e| < 1023
  return __builtin_bit_cast(double, (unsigned long long)(1023 + e) << 52);
}
// weight of `key` against `top`, the largest; c = log2(e) / t
__device__ __forceinline__ double weight(uint32_t key, uint32_t top, double c, const double* tab) {
  const double w = exp2_neg(fmin((value_of(key) - value_of(top)) * c, 0.0), tab);
  return key == top ? 1.0 : key <= kNegInf || top == kPosInf ? 0.0 : w;
}
__device__ __forceinline__ bool is_nan16(uint16_t b) { return (b & 0x7fffu) > 0x7c00u; }
__device__ __forceinline__ float row_t(const SampleArgs& a, int m) { return a.temperature ? a.temperature[m] : a.t; }

// ---- wave operations over DPP (whole waves) ----
template <int CTRL, int ROWS>
__device__ __forceinline__ uint32_t dpp(uint32_t v) {       // 0 where the lane has no source
  return (uint32_t)__builtin_amdgcn_update_dpp(0, (int)v, CTRL, ROWS, 0xF, true);
}
template <int CTRL, int ROWS>
__device__ __forceinline__ unsigned long long dpp(unsigned long long b) {
  return (unsigned long long)dpp<CTRL, ROWS>((uint32_t)(b >> 32)) << 32 | dpp<CTRL, ROWS>((uint32_t)b);
}
template <int CTRL, int ROWS>
__device__ __forceinline__ double dpp(double v) {
  const uint64_t b = __builtin_bit_cast(uint64_t, v);
  return __builtin_bit_cast(double, (uint64_t)dpp<CTRL, ROWS>((uint32_t)(b >> 32)) << 32 | dpp<CTRL, ROWS>((uint32_t)b));
}
__device__ __forceinline__ uint32_t lane_of(uint32_t v, int lane) {
  return (uint32_t)__builtin_amdgcn_readlane((int)v, lane);
}
__device__ __forceinline__ unsigned long long lane_of(unsigned long long b, int lane) {
  return (unsigned long long)lane_of((uint32_t)(b >> 32), lane) << 32 | lane_of((uint32_t)b, lane);
}
__device__ __forceinline__ double lane_of(double v, int lane) {
  const uint64_t b = __builtin_bit_cast(uint64_t, v);
  return __builtin_bit_cast(double, (uint64_t)lane_of((uint32_t)(b >> 32), lane) << 32 | lane_of((uint32_t)b, lane));
}
template <typename T>
__device__ __forceinline__ T wave_scan(T v) {               // inclusive
  v += dpp<0x111, 0xF>(v);   // row_shr 1, 2, 4, 8
  v += dpp<0x112, 0xF>(v);
  v += dpp<0x114, 0xF>(v);
  v += dpp<0x118, 0xF>(v);
  v += dpp<0x142, 0xA>(v);   // row_bcast 15, 31
  v += dpp<0x143, 0xC>(v);
  return v;
}
template <typename T>
__device__ __forceinline__ T wave_total(T v) { return lane_of(wave_scan(v), 63); }
__device__ __forceinline__ uint32_t wave_max_u32(uint32_t v) {
  v = max(v, dpp<0x111, 0xF>(v));
  v = max(v, dpp<0x112, 0xF>(v));
  v = max(v, dpp<0x114, 0xF>(v));
  v = max(v, dpp<0x118, 0xF>(v));
  v = max(v, dpp<0x142, 0xA>(v));
  v = max(v, dpp<0x143, 0xC>(v));
  return lane_of(v, 63);
}

__global__ __launch_bounds__(kST) void sample_slice_kernel(SampleArgs a, bool vec) {
  __shared__ double s_tab[64];
  __shared__ uint32_t s_g[kST / 64], s_m[kST / 64];
  // [chunk][replica]: replicas of one counter in different banks
  __shared__ uint32_t s_cnt[kChunks * kRep];
  __shared__ unsigned long long s_mass[kChunks * kRep];
  __shared__ uint32_t s_n;
  __shared__ __attribute__((aligned(16))) uint16_t s_list[kSlice];
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
  const int sl = blockIdx.x, m = blockIdx.y;
  const int i0 = sl * kSlice + tid * 8;               // this thread's logits
  const uint16_t* xr = a.x + (int64_t)m * a.ldx;
  SliceSums* o = a.sums + (int64_t)m * a.S + sl;
  const float t = row_t(a, m);

  uint16_t b[8];
  if (vec && i0 + 8 <= a.N) {
    const uint4 q = *reinterpret_cast<const uint4*>(xr + i0);
    const uint32_t w[4] = {q.x, q.y, q.z, q.w};
#pragma unroll
    for (int e = 0; e < 8; ++e) b[e] = (uint16_t)(w[e / 2] >> (16 * (e & 1)));
  } else {
#pragma unroll
    for (int e = 0; e < 8; ++e) b[e] = xr[min(i0 + e, a.N - 1)];
  }
  if (tid < 64) s_tab[tid] = exp2(tid * (1.0 / 64.0));
  for (int i = tid; i < kRep * kChunks; i += kST) {
    s_cnt[i] = 0;
    s_mass[i] = 0;
  }
  uint32_t key[8], g = 0, mx = 0;
#pragma unroll
  for (int e = 0; e < 8; ++e) {
    const bool in = i0 + e < a.N, nan = is_nan16(b[e]);
    const uint32_t low = kSlice - 1 - (tid * 8 + e);  // first index wins among equals
    key[e] = nan ? kNegInf : key_of(b[e]);
    if (!in) key[e] = 0;
    g = max(g, in ? (nan ? 0xFFFFu : key[e]) << 16 | low : 0u);
    mx = max(mx, in ? key[e] << 16 | low : 0u);
  }
  g = wave_max_u32(g);
  mx = wave_max_u32(mx);
  if (lane == 0) {
    s_g[wave] = g;
    s_m[wave] = mx;
  }
  __syncthreads();
#pragma unroll
  for (int w = 0; w < kST / 64; ++w) {
    g = max(g, s_g[w]);
    mx = max(mx, s_m[w]);
  }
  if (tid == 0) {
    o->greedy_key = g >> 16;
    o->greedy_idx = sl * kSlice + (kSlice - 1 - (g & 0xFFFFu));
    o->max_key = mx >> 16;
    o->max_idx = sl * kSlice + (kSlice - 1 - (mx & 0xFFFFu));
  }
  if (!(t > 0.f)) return;                              // greedy row (uniform)

  const uint32_t top = mx >> 16;
  const double c = 1.4426950408889634074 / (double)t;
  const int k = a.top_k ? a.top_k[m] : a.k;
  const float p = a.top_p ? a.top_p[m] : a.p;
  const float lo = a.min_p ? a.min_p[m] : a.lo;
  if (k < 1 && !(p < 1.0f) && !(lo > 0.0f)) {
    // no filter: no border to look for, the slice's weight is all that is needed (it goes
    // to the largest chunk)
    unsigned long long own = 0;
#pragma unroll
    for (int e = 0; e < 8; ++e)
      if (key[e] > kNegInf) own += (unsigned long long)(weight(key[e], top, c, s_tab) * kFix + 0.5);
    atomicAdd(&s_mass[tid % (kChunks * kRep)], own);
    __syncthreads();
    if (wave == 0) {
      own = 0;
      for (int i = lane; i < kChunks * kRep; i += 64) own += s_mass[i];
      own = wave_total(own);
      o->mass[lane] = lane == kChunks - 1 ? own : 0;
      o->cnt[lane] = o->off[lane] = 0;
    }
    return;
  }
  // Logits that no filter can keep are left out of the list, and their weight with them
  // where no share of it is asked for:
  //   * top-k up to 64: what is below the wave's own k-th largest thread maximum has k larger
  //     logits in this wave alone
  //   * min-p without top-p: weights against the slice's largest are no smaller than against
  //     the row's (in fp32 with 2% of room; what it lets pass the border sorts out)
  uint32_t least = kNegInf + 1;                        // smallest key listed
  if (k >= 1 && k <= 64) {
    uint32_t tmax = 0;
#pragma unroll
    for (int e = 0; e < 8; ++e) tmax = max(tmax, key[e]);
    uint32_t kth = 0;                                  // largest key that k maxima reach
#pragma unroll
    for (int bit = 15; bit >= 0; --bit) {
      const uint32_t probe = kth | (1u << bit);
      if (__popcll(__ballot(tmax >= probe)) >= k) kth = probe;
    }
    least = max(least, kth);
  }
  if (!(p < 1.0f) && lo > 0.0f) {
    // the smallest key that comes near min-p: chunk, 16-key run, key
    const float c32 = (float)c, edge = (log2f(fminf(lo, 1.0f)) - 0.03f) * 1.001f;
    const float xt = (float)value_of(top);
    uint32_t base = 0;
#pragma unroll
    for (int st = 10; st >= -2; st -= 6) {             // every 1024th, every 16th, every key
      const uint32_t probe = min(base + ((uint32_t)lane << max(st, 0)), top);
      const float d = ((float)value_of(probe) - xt) * c32;
      const uint64_t ok = __ballot(probe > kNegInf && (probe == top || d >= edge));
      const int nth = ok ? __builtin_ctzll(ok) : 64;
      if (st > 0) base += (uint32_t)max(nth - 1, 0) << st;
      else least = max(least, min(base + (uint32_t)nth, top));
    }
  }
  const int rep = lane & (kRep - 1);
  uint32_t rank[8];
#pragma unroll
  for (int e = 0; e < 8; ++e) {
    if (key[e] < least) continue;                      // not listed
    rank[e] = atomicAdd(&s_cnt[(key[e] >> 10) * kRep + rep], 1u);
  }
  __syncthreads();
  if (wave == 0) {                                     // lane: chunk 63 - lane
    const int ch = kChunks - 1 - lane;
    uint32_t n = 0;
#pragma unroll
    for (int r = 0; r < kRep; ++r) n += s_cnt[ch * kRep + r];
    const uint32_t incl = wave_scan(n);
    uint32_t at = incl - n;
    o->cnt[ch] = (uint16_t)n;
    o->off[ch] = (uint16_t)at;
#pragma unroll
    for (int r = 0; r < kRep; ++r) {                   // counts become first places
      const uint32_t own = s_cnt[ch * kRep + r];
      s_cnt[ch * kRep + r] = at;
      at += own;
    }
    if (lane == 63) s_n = incl;                        // listed logits
  }
  __syncthreads();
#pragma unroll
  for (int e = 0; e < 8; ++e) {
    if (key[e] < least) continue;
    s_list[s_cnt[(key[e] >> 10) * kRep + rep] + rank[e]] = (uint16_t)key[e];
  }
  __syncthreads();
  // the list, and its weights: evaluated here, where every lane has a listed logit
  const int n = (int)s_n;
  uint16_t* list = a.list + ((int64_t)m * a.S + sl) * kSlice;
  for (int i = tid * 8; i < n; i += kST * 8)           // whole 16-byte pieces: the list has room
    *reinterpret_cast<uint4*>(list + i) = *reinterpret_cast<const uint4*>(&s_list[i]);
  for (int i = tid; i < n; i += kST) {
    const uint32_t ki = s_list[i];
    atomicAdd(&s_mass[(ki >> 10) * kRep + rep], (unsigned long long)(weight(ki, top, c, s_tab) * kFix + 0.5));
  }
  __syncthreads();
  // chunk tid / 8 by eight threads
  static_assert(kST == 8 * kChunks, "eight threads a chunk");
  unsigned long long ms = 0;
#pragma unroll
  for (int r = 0; r < kRep / 8; ++r) ms += s_mass[(tid >> 3) * kRep + (tid & 7) + 8 * r];
  ms += dpp<0x111, 0xF>(ms);                           // row_shr: the last of eight lanes sums them
  ms += dpp<0x112, 0xF>(ms);
  ms += dpp<0x114, 0xF>(ms);
  if ((tid & 7) == 7) o->mass[tid >> 3] = ms;
}

// Inclusive block scans over the kPT threads (all of them call it), one barrier each.  s_w:
// kPW + kPW entries, used in turns (`turn`), so a scan's reads are over before its half is
// written again.
template <typename T>
__device__ __forceinline__ T block_scan(T v, T (&s_w)[2][kPW], int turn) {
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  v = wave_scan(v);
  if (lane == 63) s_w[turn & 1][wave] = v;
  __syncthreads();
  T before = T(0);
#pragma unroll
  for (int w = 0; w < kPW; ++w)
    if (w < wave) before += s_w[turn & 1][w];
  return v + before;
}

__global__ __launch_bounds__(kPT) void sample_pick_kernel(SampleArgs a, bool vec) {
  __shared__ double s_tab[64];
  __shared__ double s_pm[kPW][kChunks];                // weight and count of the chunks, by wave
  __shared__ uint32_t s_pc[kPW][kChunks];
  __shared__ uint32_t s_hist[2][1024];                 // number of each key of a chunk
  __shared__ double s_wkey[1024];                      // weight of each key of the border's chunk
  __shared__ unsigned long long s_wfix[1024];          // the same in fixed point
  __shared__ double s_sm[kMaxSlices];                  // kept weight of a slice, without border ties
  __shared__ uint32_t s_tie[kMaxSlices];
  __shared__ double s_wd[2][kPW];
  __shared__ uint32_t s_wu[2][kPW];
  __shared__ uint32_t s_b[8];                          // [0..1] border of top-k, [2..3] of top-p, [4..5] the token
  __shared__ double s_left;                            // weight that top-k leaves
  const int tid = threadIdx.x, lane = tid & 63;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int m = blockIdx.x, S = a.S;
  const SliceSums* sums = a.sums + (int64_t)m * S;
  const float t = row_t(a, m);
  const bool greedy = !(t > 0.f);
  const int ch = kChunks - 1 - lane;                   // this lane's chunk

  // sums: lane = slice for the largest, lane = chunk for the wave's own slices
  uint32_t mk = 0, mi = kNone;
  if (lane < S) {
    mk = greedy ? sums[lane].greedy_key : sums[lane].max_key;
    mi = greedy ? sums[lane].greedy_idx : sums[lane].max_idx;
  }
  uint64_t raw[kOwn];
  uint32_t cnt[kOwn], off[kOwn];
#pragma unroll
  for (int i = 0; i < kOwn; ++i) {
    const int s = wave + kPW * i;
    const bool in = s < S && !greedy;                  // (a greedy row has no sums)
    raw[i] = in ? sums[s].mass[ch] : 0;
    cnt[i] = in ? sums[s].cnt[ch] : 0;
    off[i] = in ? sums[s].off[ch] : 0;
  }
  if (tid < 64) s_tab[tid] = exp2(tid * (1.0 / 64.0));
  s_hist[0][tid] = 0;
  s_hist[1][tid] = 0;
  if (tid < 8) s_b[tid] = (tid & 1) ? 0u : kNone;
  // the largest over slices, the first of equals
  const uint32_t top = wave_max_u32(mk);
  if (greedy || top <= kNegInf) {                      // nothing to draw from: the first index
    const uint64_t best = __ballot(mk == top);
    const uint32_t first = lane_of(mi, __builtin_ctzll(best));
    if (tid == 0) a.out[m] = greedy ? (int64_t)first : 0;
    return;
  }
  __syncthreads();
  const double c = 1.4426950408889634074 / (double)t;
  const double f = lane < S ? weight(mk, top, c, s_tab) : 0.0;   // of each slice's largest
  double mass[kOwn], pm = 0.0;
  uint32_t pc = 0;
#pragma unroll
  for (int i = 0; i < kOwn; ++i) {
    mass[i] = (double)raw[i] * (1.0 / kFix) * lane_of(f, (wave + kPW * i) & 63);
    pm += mass[i];
    pc += cnt[i];
  }
  s_pm[wave][lane] = pm;
  s_pc[wave][lane] = pc;
  __syncthreads();
  // every wave: count and weight of each chunk (lane), and of all chunks down to it
  double cm = 0.0;
  uint32_t cc = 0;
#pragma unroll
  for (int w = 0; w < kPW; ++w) {
    cm += s_pm[w][lane];
    cc += s_pc[w][lane];
  }
  const uint32_t icnt = wave_scan(cc);
  const double imass = wave_scan(cm);

  const uint16_t* list = a.list + (int64_t)m * S * kSlice;
  uint32_t el[kOwn];                                   // first 64 entries of chunk `held` in the wave's slices
  int held = -1, uses = 0, turn = 0;
  // f(i, key) of the entries past the first 64 of a chunk (lane cl) in the wave's slices, kOwn
  // kDeep loads at a time
  auto rest = [&](int cl, auto f) {
    int n[kOwn], last[kOwn], most = 0;
    const uint16_t* q[kOwn];
#pragma unroll
    for (int i = 0; i < kOwn; ++i) {
      n[i] = (int)lane_of(cnt[i], cl);
      q[i] = list + (int64_t)(wave + kPW * i) * kSlice + lane_of(off[i], cl);
      last[i] = max(n[i] - 1, 0);
      if (n[i] == 0) q[i] = list;                        // nothing is read but in range
      most = max(most, n[i]);
    }
    for (int j = 64 + lane; j - lane < most; j += 64 * kDeep) {
      uint32_t v[kOwn][kDeep];
#pragma unroll
      for (int i = 0; i < kOwn; ++i)
#pragma unroll
        for (int d = 0; d < kDeep; ++d) v[i][d] = q[i][min(j + 64 * d, last[i])];   // (clamped: no branch)
#pragma unroll
      for (int i = 0; i < kOwn; ++i)
#pragma unroll
        for (int d = 0; d < kDeep; ++d)
          if (j + 64 * d < n[i]) f(i, v[i][d]);
    }
  };
  // Number of this thread's key (1023 - tid of the chunk of lane cl), from the listed logits
  auto histogram = [&](int cl) {
    held = cl;
    uint32_t* hist = s_hist[uses++ & 1];
#pragma unroll
    for (int i = 0; i < kOwn; ++i) {
      const int n = (int)lane_of(cnt[i], cl);
      const uint16_t* p = list + (int64_t)(wave + kPW * i) * kSlice + lane_of(off[i], cl);
      el[i] = lane < n ? p[lane] : 0u;
    }
#pragma unroll
    for (int i = 0; i < kOwn; ++i) {
      const int n = (int)lane_of(cnt[i], cl);
      if (lane < n) atomicAdd(&hist[el[i] & 1023u], 1u);
    }
    rest(cl, [&](int, uint32_t key) { atomicAdd(&hist[key & 1023u], 1u); });
    __syncthreads();
    return hist[1023 - tid];
  };

  // Border: tokens with a larger key stay, and the first `bkeep` of the equal ones.
  uint32_t bkey = kNegInf, bkeep = 0;
  const int k = a.top_k ? a.top_k[m] : a.k;
  const float p = a.top_p ? a.top_p[m] : a.p;
  const float lo = a.min_p ? a.min_p[m] : a.lo;

  uint32_t mine = 0;                                   // of the held chunk: this key's tokens,
  double before_key = 0.0;                             // and the weight before them
  double total = lane_of(imass, 63);                   // weight left by top-k
  int kl = kChunks - 1;                                // lane of the chunk of the top-k border
  if (k >= 1 && (uint32_t)k <= lane_of(icnt, 63)) {   // (fewer: all there are, but for what min-p drops)
    kl = __builtin_ctzll(__ballot(icnt >= (uint32_t)k));
    const uint32_t n0 = kl ? lane_of(icnt, max(kl - 1, 0)) : 0u;
    const double m0 = kl ? lane_of(imass, max(kl - 1, 0)) : 0.0;
    mine = histogram(kl);
    const uint32_t key = (uint32_t)(kChunks - 1 - kl) << 10 | (uint32_t)(1023 - tid);
    const double w = mine ? weight(key, top, c, s_tab) : 0.0;
    s_wkey[1023 - tid] = w;
    const uint32_t incl = n0 + block_scan<uint32_t>(mine, s_wu, turn);
    const double v = (double)mine * w;
    before_key = m0 + (block_scan<double>(v, s_wd, turn) - v);
    ++turn;
    if (mine && incl - mine < (uint32_t)k && incl >= (uint32_t)k) {   // one thread
      const uint32_t keep = (uint32_t)k - (incl - mine);
      s_b[0] = key;
      s_b[1] = keep;
      s_left = before_key + (double)keep * w;
    }
    __syncthreads();
    bkey = s_b[0];
    bkeep = s_b[1];
    total = s_left;
    mine = key < bkey ? 0u : key == bkey ? min(mine, bkeep) : mine;
  }
  if (p < 1.0f) {
    const double target = (double)p * total;
    // the first chunk that reaches the target; the border's own ends with `total`
    const int pl = __builtin_ctzll(__ballot(lane == kl || (lane < kl && cc && imass >= target)));
    const double m0 = pl ? lane_of(imass, max(pl - 1, 0)) : 0.0;
    const uint32_t key = (uint32_t)(kChunks - 1 - pl) << 10 | (uint32_t)(1023 - tid);
    double w;
    if (pl != held) {
      mine = histogram(pl);
      w = mine ? weight(key, top, c, s_tab) : 0.0;
      s_wkey[1023 - tid] = w;
      const double v = (double)mine * w;
      // the weight before this key: exactly m0 for the chunk's first one
      before_key = m0 + (block_scan<double>(v, s_wd, turn++) - v);
    } else {
      w = s_wkey[1023 - tid];
    }
    // the border is the last key of the chunk before which less than the target lies
    // (the row's first always stays; a chunk's first does, as m0 is less)
    const bool in = mine && (before_key < target || key == top);
    const uint64_t ins = __ballot(in);                 // one atomic a wave: keys fall with the lane
    if (ins && lane == 63 - __builtin_clzll(ins)) atomicMin(&s_b[2], key);
    __syncthreads();
    if (in && key == s_b[2]) {
      const double need = w > 0.0 ? ceil((target - before_key) / w) : (double)mine;
      s_b[3] = (uint32_t)fmin(fmax(need, 1.0), (double)mine);
    }
    __syncthreads();
    if (s_b[2] != kNone) {
      bkey = s_b[2];
      bkeep = s_b[3];
    }
  }
  if (lo > 0.0f) {
    // the smallest key whose weight reaches min-p (every wave): chunk, 16-key run, key
    uint32_t base = 0;
#pragma unroll
    for (int st = 10; st >= 4; st -= 6) {              // every 1024th key, every 16th of a chunk
      const uint32_t key = base + ((uint32_t)lane << st);
      const uint64_t ok = __ballot(key > kNegInf && weight(min(key, top), top, c, s_tab) >= (double)lo);
      base += (uint32_t)max((ok ? __builtin_ctzll(ok) : 64) - 1, 0) << st;
    }
    // the border lies in the 16 keys after `base`, or is it
    const uint32_t key = base + (uint32_t)lane;
    const uint64_t ok = __ballot(key > kNegInf && weight(min(key, top), top, c, s_tab) >= (double)lo);
    const uint32_t mkey = ok ? base + (uint32_t)__builtin_ctzll(ok) : kNone;
    if (mkey > top) {                                  // min-p above 1: the first token alone
      bkey = top;
      bkeep = 1;
    } else if (mkey > bkey) {
      bkey = mkey;
      bkeep = kNone;
    }
  }

  bkey = (uint32_t)__builtin_amdgcn_readfirstlane((int)bkey);   // the same in every lane
  // kept weight of each slice: whole chunks above the border's, its own logit by logit
  const int bl = kChunks - 1 - (int)(bkey >> 10);
  // (a list's order within a chunk is that of atomics: sums in fixed point, 2^-50 of what the chunk's
  // weights stay below, do not depend on it; the largest of all is 1, so below 2^-900 they may be 0)
  const uint32_t ctop = min(bkey | 1023u, top);
  const float below = ((float)value_of(ctop) - (float)value_of(top)) * (float)c;
  const int wexp = ctop == top ? 1 : (int)ceilf(fmaxf(below, -900.f)) + 1;
  {
    const double w = held == bl ? s_wkey[1023 - tid] : weight((bkey & ~1023u) | (uint32_t)(1023 - tid), top, c, s_tab);
    // w 2^(50 - wexp) in the last places of a number from 2^52 on
    s_wfix[1023 - tid] = __builtin_bit_cast(unsigned long long, fma(w, pow2(50 - wexp), 4503599627370496.0)) -
                         __builtin_bit_cast(unsigned long long, 4503599627370496.0);
  }
#pragma unroll
  for (int i = 0; i < kOwn; ++i) {
    const int n = (int)lane_of(cnt[i], bl);
    if (held != bl) {
      const uint16_t* q = list + (int64_t)(wave + kPW * i) * kSlice + lane_of(off[i], bl);
      el[i] = lane < n ? q[lane] : 0u;
    }
  }
  __syncthreads();
  unsigned long long part[kOwn];                       // of the border's chunk
  uint32_t tie[kOwn];
  auto count = [&](int i, uint32_t key) {
    part[i] += key > bkey ? s_wfix[key & 1023u] : 0ull;
    tie[i] += key == bkey;
  };
#pragma unroll
  for (int i = 0; i < kOwn; ++i) {
    part[i] = 0;
    tie[i] = 0;
    if (lane < (int)lane_of(cnt[i], bl)) count(i, el[i]);
  }
  rest(bl, count);
#pragma unroll
  for (int i = 0; i < kOwn; ++i) {
    const int s = wave + kPW * i;
    if (s >= S) break;
    double sum = wave_total(lane < bl ? mass[i] : 0.0);
    uint32_t ties = 0;
    if (lane_of(cnt[i], bl) > 0) {                     // listed in the border's chunk
      sum += (double)wave_total(part[i]) * pow2(wexp - 50);
      ties = wave_total(tie[i]);
    }
    if (lane == 0) {
      s_sm[s] = sum;
      s_tie[s] = ties;
    }
  }
  __syncthreads();
  // every wave, lane = slice: the slice that holds the token
  const uint32_t st = lane < S ? s_tie[lane] : 0u;
  const uint32_t tie_before = wave_scan(st) - st;
  const uint32_t stay = tie_before >= bkeep ? 0u : min(st, bkeep - tie_before);
  const double sm = lane < S ? s_sm[lane] + (double)stay * weight(bkey, top, c, s_tab) : 0.0;
  const double incl = wave_scan(sm);
  const float u = a.u[m];
  const double target = (u > 0.f ? (u < 1.f ? (double)u : 1.0) : 0.0) * lane_of(incl, 63);
  const uint64_t some = __ballot(sm > 0.0), past = __ballot(sm > 0.0 && incl > target);
  // (u at its end, or rounding: the last slice with any weight)
  const int sl = past ? __builtin_ctzll(past) : 63 - __builtin_clzll(some | 1);
  const double base = lane_of(incl, sl) - lane_of(sm, sl);
  const uint32_t keep = lane_of(stay, sl), ties = lane_of(st, sl);

  // the slice's logits in index order, four per thread
  const uint16_t* xr = a.x + (int64_t)m * a.ldx;
  const int i0 = sl * kSlice + tid * 4;
  uint16_t b[4];
  if (vec && i0 + 4 <= a.N) {
    const uint2 q = *reinterpret_cast<const uint2*>(xr + i0);
    b[0] = (uint16_t)q.x; b[1] = (uint16_t)(q.x >> 16); b[2] = (uint16_t)q.y; b[3] = (uint16_t)(q.y >> 16);
  } else {
#pragma unroll
    for (int e = 0; e < 4; ++e) b[e] = i0 + e < a.N ? xr[i0 + e] : (uint16_t)0xFC00u;
  }
  uint32_t kk[4], eq = 0;
#pragma unroll
  for (int e = 0; e < 4; ++e) {
    kk[e] = is_nan16(b[e]) ? kNegInf : key_of(b[e]);
    eq += kk[e] == bkey;
  }
  uint32_t rank = 0;                                   // of the thread's first tie, where not all stay
  if (keep < ties) rank = block_scan<uint32_t>(eq, s_wu, turn) - eq;
  double w[4], own = 0.0;
#pragma unroll
  for (int e = 0; e < 4; ++e) {
    w[e] = 0.0;
    if (kk[e] > bkey || (kk[e] == bkey && rank < keep)) w[e] = weight(kk[e], top, c, s_tab);
    rank += keep < ties && kk[e] == bkey;
    own += w[e];
  }
  double cum = base + block_scan<double>(own, s_wd, turn) - own;
  uint32_t at = kNone, last = 0;                       // first token past the target, last with any weight
#pragma unroll
  for (int e = 0; e < 4; ++e) {
    cum += w[e];
    if (w[e] > 0.0) {
      if (cum > target) at = min(at, (uint32_t)(i0 + e));
      last = (uint32_t)(i0 + e);
    }
  }
  // one atomic a wave: indices rise with the lane
  const uint64_t hit = __ballot(at != kNone), any = __ballot(own > 0.0);
  if (hit && lane == __builtin_ctzll(hit)) atomicMin(&s_b[4], at);
  if (any && lane == 63 - __builtin_clzll(any)) atomicMax(&s_b[5], last);
  __syncthreads();
  if (tid == 0) a.out[m] = (int64_t)(s_b[4] != kNone ? s_b[4] : s_b[5]);
}

}  // namespace

extern "C" int64_t helm_sample_workspace_bytes(int M, int N) {
  if (M < 1 || N < 1) return 0;
  return (int64_t)M * ((N + (int64_t)kSlice - 1) / kSlice) * (int64_t)(sizeof(SliceSums) + kSlice * 2);
}

extern "C" int helm_sample(const void* x, int64_t ldx, int M, int N, const float* u, const float* temperature,
                           const int32_t* top_k, const float* top_p, const float* min_p, float t, int k, float p,
                           float lo, int64_t* out, void* workspace, int64_t workspace_bytes, void* stream) {
  HELM_CHECK_ARG(x && u && out, "helm_sample: null pointer");
  HELM_CHECK_ARG(M >= 1 && N >= 1 && ldx >= N, "helm_sample: bad sizes");
  HELM_CHECK_SUPPORTED(M <= 65535 && N <= kMaxSlices * kSlice, "helm_sample: at most 65535 rows of " +
                                                                   std::to_string(kMaxSlices * kSlice) + " logits");
  HELM_CHECK_ARG(workspace && helm::aligned16(workspace) && workspace_bytes >= helm_sample_workspace_bytes(M, N),
                 "helm_sample: workspace too small or not 16-byte aligned");
  SampleArgs a{};
  a.x = static_cast<const uint16_t*>(x); a.ldx = ldx; a.M = M; a.N = N; a.S = (N + kSlice - 1) / kSlice;
  a.u = u; a.temperature = temperature; a.top_k = top_k; a.top_p = top_p; a.min_p = min_p;
  a.t = t; a.k = k; a.p = p; a.lo = lo;
  static_assert(sizeof(SliceSums) % 16 == 0, "the lists follow 16-byte aligned");
  a.sums = static_cast<SliceSums*>(workspace);
  a.list = reinterpret_cast<uint16_t*>(a.sums + (int64_t)M * a.S);
  a.out = out;
  const bool vec = helm::aligned16(x) && ldx % 8 == 0;
  const hipStream_t s = static_cast<hipStream_t>(stream);
  hipLaunchKernelGGL(sample_slice_kernel, dim3(a.S, M), dim3(kST), 0, s, a, vec);
  HELM_CHECK_LAUNCH("helm_sample slice launch");
  hipLaunchKernelGGL(sample_pick_kernel, dim3(M), dim3(kPT), 0, s, a, vec);
  HELM_CHECK_LAUNCH("helm_sample pick launch");
  return HELM_OK;
}
