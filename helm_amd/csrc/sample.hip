// sample.hip — one token per row drawn from fp16 logits with temperature, top-k, top-p
// and min-p, from given random numbers.
//
// w_i = 2^((x_i - max) log2(e) / t).  An fp16 logit has a 16-bit key that orders like
// its value (equal values, equal keys), so every filter is a border (key, how many of its
// equals stay): no sort, and ties go to the lowest index.  Keys fall into 64 chunks of
// 1024 neighbours.  Two kernels:
//   * slices: a workgroup per 4096 logits groups them by chunk (key and index, largest
//     chunk first) and sums count and weight of each chunk;
//   * pick: a workgroup per row finds the chunk that holds a border from those sums and
//     resolves the key inside it from the few logits of that chunk, then the slice that
//     holds the drawn token, then the token.
// Weights of a chunk are summed in 2^-44 fixed point relative to the slice's largest:
// sums of integers do not depend on their order, so atomics leave the result the same
// from run to run.  All else is in 64 bits: a token next to a border decides a whole
// number.
// Bound by latency: one pass over the logits, then four dependent round trips.
#include "helm_common.h"

namespace {

constexpr int kSlice = 4096;          // logits of a slice
constexpr int kST = 512;              // threads of a slice: 8 logits each
constexpr int kPT = 1024;             // threads of a row's pick: one per key of a chunk
constexpr int kChunks = 64;
constexpr int kRep = 8;               // replicas of the slice's counters (fewer conflicts)
constexpr int kMaxSlices = 1024;
constexpr uint32_t kNegInf = 0x03FFu; // key of -inf
constexpr uint32_t kPosInf = 0xFC00u; // key of +inf
constexpr double kFix = 17592186044416.0;   // 2^44

struct SliceOut {
  uint32_t greedy_key, greedy_idx;    // NaN as the largest value
  uint32_t max_key, max_idx;          // NaN as -inf; idx: first of the largest in the slice
  uint64_t mass[kChunks];             // 2^44 sum of w relative to the slice's largest
  uint32_t cnt[kChunks];
  uint32_t off[kChunks];              // first entry of the chunk in `seg`
  uint32_t seg[kSlice];               // key << 16 | index in the slice, chunk by chunk
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
  SliceOut* ws;
  int64_t* out;
};

__device__ __forceinline__ uint32_t key_of(uint16_t b) {   // not for NaN
  if (b == 0x8000u) b = 0;                                  // -0 equals 0
  return b & 0x8000u ? (uint32_t)(uint16_t)~b : (uint32_t)b | 0x8000u;
}
__device__ __forceinline__ double value_of(uint32_t key) {
  return (double)h2f((uint16_t)(key & 0x8000u ? key & 0x7fffu : ~key));
}
// weight of `key` against `top`, the largest; c = log2(e) / t
__device__ __forceinline__ double weight(uint32_t key, uint32_t top, double c) {
  if (key == top) return 1.0;
  if (key <= kNegInf || top == kPosInf) return 0.0;
  return exp2((value_of(key) - value_of(top)) * c);
}
__device__ __forceinline__ bool is_nan16(uint16_t b) { return (b & 0x7fffu) > 0x7c00u; }

__device__ __forceinline__ uint32_t wave_max_u32(uint32_t v) {
#pragma unroll
  for (int o = 32; o >= 1; o >>= 1) v = max(v, (uint32_t)__shfl_xor((int)v, o, 64));
  return v;
}

__device__ __forceinline__ float row_t(const SampleArgs& a, int m) { return a.temperature ? a.temperature[m] : a.t; }

__global__ __launch_bounds__(kST) void sample_slice_kernel(SampleArgs a, bool vec) {
  __shared__ uint32_t s_g[kST / 64], s_m[kST / 64];
  __shared__ uint32_t s_cnt[kRep][kChunks];
  __shared__ unsigned long long s_mass[kRep][kChunks];
  __shared__ uint32_t s_off[kRep][kChunks];
  __shared__ __attribute__((aligned(16))) uint32_t s_seg[kSlice];
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
  const int sl = blockIdx.x, m = blockIdx.y;
  const int i0 = sl * kSlice + tid * 8;               // this thread's logits
  const uint16_t* xr = a.x + (int64_t)m * a.ldx;
  SliceOut* o = a.ws + (int64_t)m * a.S + sl;
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
  for (int i = tid; i < kRep * kChunks; i += kST) {
    (&s_cnt[0][0])[i] = 0;
    (&s_mass[0][0])[i] = 0;
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
  const int rep = lane & (kRep - 1);
#pragma unroll
  for (int e = 0; e < 8; ++e) {
    if (key[e] <= kNegInf) continue;                   // no weight: not listed
    const unsigned long long w = (unsigned long long)(weight(key[e], top, c) * kFix + 0.5);
    atomicAdd(&s_cnt[rep][key[e] >> 10], 1u);
    atomicAdd(&s_mass[rep][key[e] >> 10], w);
  }
  __syncthreads();
  if (wave == 0) {                                     // lane: chunk 63 - lane
    const int ch = kChunks - 1 - lane;
    uint32_t n = 0;
    unsigned long long ms = 0;
    for (int r = 0; r < kRep; ++r) {
      n += s_cnt[r][ch];
      ms += s_mass[r][ch];
    }
    uint32_t incl = n;
#pragma unroll
    for (int d = 1; d < 64; d <<= 1) {
      const uint32_t v = (uint32_t)__shfl_up((int)incl, d, 64);
      if (lane >= d) incl += v;
    }
    uint32_t at = incl - n;
    o->mass[ch] = ms;
    o->cnt[ch] = n;
    o->off[ch] = at;
    for (int r = 0; r < kRep; ++r) {
      s_off[r][ch] = at;
      at += s_cnt[r][ch];
    }
    if (lane == 63) s_g[0] = incl;                     // listed logits
  }
  __syncthreads();
#pragma unroll
  for (int e = 0; e < 8; ++e) {
    if (key[e] <= kNegInf) continue;
    s_seg[atomicAdd(&s_off[rep][key[e] >> 10], 1u)] = key[e] << 16 | (uint32_t)(tid * 8 + e);
  }
  __syncthreads();
  const int n = (int)s_g[0];
  for (int i = tid * 4; i < n; i += kST * 4)           // whole 16-byte pieces: seg has room
    *reinterpret_cast<uint4*>(&o->seg[i]) = *reinterpret_cast<const uint4*>(&s_seg[i]);
}

// Inclusive block scan over kPT threads (all of them call it); *total is the sum.
template <typename T>
__device__ __forceinline__ T block_scan(T v, T* s_w, T* total) {
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
#pragma unroll
  for (int d = 1; d < 64; d <<= 1) {
    const T u = __shfl_up(v, d, 64);
    if (lane >= d) v += u;
  }
  __syncthreads();                                     // s_w of an earlier scan has been read
  if (lane == 63) s_w[wave] = v;
  __syncthreads();
  T before = T(0), all = T(0);
#pragma unroll
  for (int w = 0; w < kPT / 64; ++w) {
    if (w < wave) before += s_w[w];
    all += s_w[w];
  }
  *total = all;
  return v + before;
}

__global__ __launch_bounds__(kPT) void sample_pick_kernel(SampleArgs a) {
  __shared__ double s_f[kMaxSlices];                   // weight of a slice's largest
  __shared__ double s_sm[kMaxSlices];                  // kept weight of a slice, without border ties
  __shared__ uint32_t s_tie[kMaxSlices];
  __shared__ double s_cmass[kChunks];
  __shared__ uint32_t s_ccnt[kChunks];
  __shared__ uint32_t s_hist[1024];
  __shared__ double s_wd[kPT / 64];
  __shared__ uint32_t s_wu[kPT / 64];
  __shared__ uint32_t s_key[4];                        // [0] top key, [1] its index, [2] / [3] a border found
  __shared__ double s_d[2];
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
  const int m = blockIdx.x, S = a.S;
  const SliceOut* ws = a.ws + (int64_t)m * S;
  const float t = row_t(a, m);
  const bool greedy = !(t > 0.f);

  // the largest over slices, the first of equals
  if (wave == 0) {
    uint32_t best = 0, idx = 0xFFFFFFFFu;
    for (int s = lane; s < S; s += 64) {
      const uint32_t k = greedy ? ws[s].greedy_key : ws[s].max_key;
      const uint32_t i = greedy ? ws[s].greedy_idx : ws[s].max_idx;
      if (k > best || (k == best && i < idx)) {
        best = k;
        idx = i;
      }
    }
#pragma unroll
    for (int d = 32; d >= 1; d >>= 1) {
      const uint32_t k = (uint32_t)__shfl_xor((int)best, d, 64), i = (uint32_t)__shfl_xor((int)idx, d, 64);
      if (k > best || (k == best && i < idx)) {
        best = k;
        idx = i;
      }
    }
    if (lane == 0) {
      s_key[0] = best;
      s_key[1] = idx;
    }
  }
  __syncthreads();
  const uint32_t top = s_key[0], first = s_key[1];
  if (greedy || top <= kNegInf) {                      // nothing to draw from: the first index
    if (tid == 0) a.out[m] = greedy ? (int64_t)first : 0;
    return;
  }

  const double c = 1.4426950408889634074 / (double)t;
  for (int s = tid; s < S; s += kPT) s_f[s] = weight(ws[s].max_key, top, c);
  __syncthreads();
  // count and weight of each chunk of the row (wave: four chunks, lanes over slices)
  for (int ch = wave; ch < kChunks; ch += kPT / 64) {
    uint32_t n = 0;
    double ms = 0.0;
    for (int s = lane; s < S; s += 64) {
      const uint32_t cn = ws[s].max_key > kNegInf ? ws[s].cnt[ch] : 0u;
      n += cn;
      if (cn) ms += (double)ws[s].mass[ch] * (1.0 / kFix) * s_f[s];
    }
#pragma unroll
    for (int d = 32; d >= 1; d >>= 1) {
      n += (uint32_t)__shfl_xor((int)n, d, 64);
      ms += __shfl_xor(ms, d, 64);
    }
    if (lane == 0) {
      s_ccnt[ch] = n;
      s_cmass[ch] = ms;
    }
  }
  __syncthreads();

  // Number of this thread's key in chunk ch (thread: key 1023 - tid of the chunk), from
  // the chunk's listed logits.
  auto histogram = [&](int ch) {
    s_hist[tid] = 0;
    __syncthreads();
    for (int s = wave; s < S; s += kPT / 64) {
      if (ws[s].max_key <= kNegInf) continue;
      const int n = (int)ws[s].cnt[ch];
      const uint32_t* seg = ws[s].seg + ws[s].off[ch];
      for (int i = lane; i < n; i += 64) atomicAdd(&s_hist[(seg[i] >> 16) & 1023u], 1u);
    }
    __syncthreads();
    return s_hist[1023 - tid];
  };

  // Border: tokens with a larger key stay, and the first `keep` of the equal ones.
  uint32_t bkey = kNegInf + 1, bkeep = 0xFFFFFFFFu;
  int held = -1;                                       // chunk whose counts `mine` holds
  uint32_t mine = 0;
  const int k = a.top_k ? a.top_k[m] : a.k;
  const float p = a.top_p ? a.top_p[m] : a.p;
  const float lo = a.min_p ? a.min_p[m] : a.lo;

  double total = 0.0;                                  // weight left by top-k
  uint32_t listed = 0;
  int kch = -1;                                        // chunk of the top-k border
  for (int ch = kChunks - 1; ch >= 0; --ch) {
    const uint32_t n = s_ccnt[ch];
    if (k >= 1 && kch < 0 && listed + n >= (uint32_t)k) {
      kch = ch;
      break;
    }
    listed += n;
    total += s_cmass[ch];
  }
  if (kch >= 0) {
    mine = histogram(kch);
    held = kch;
    const uint32_t key = (uint32_t)kch << 10 | (uint32_t)(1023 - tid);
    uint32_t all;
    const uint32_t incl = listed + block_scan<uint32_t>(mine, s_wu, &all);
    if (mine && incl - mine < (uint32_t)k && incl >= (uint32_t)k) {
      s_key[2] = key;
      s_key[3] = (uint32_t)k - (incl - mine);
    }
    // (the scan's barriers come after the writes of s_key by one thread)
    __syncthreads();
    bkey = s_key[2];
    bkeep = s_key[3];
    if (key < bkey) mine = 0;
    else if (key == bkey) mine = min(mine, bkeep);
    double part;
    block_scan<double>(mine ? (double)mine * weight(key, top, c) : 0.0, s_wd, &part);
    total += part;
  }
  if (p < 1.0f) {
    const double target = (double)p * total;
    double before = 0.0;
    int pch = -1;
    double next = 0.0;
    for (int ch = kChunks - 1; ch >= max(kch, 0); --ch) {
      if (!s_ccnt[ch]) continue;
      pch = ch;                                        // (the last one, should rounding leave none)
      before = next;
      next += ch == kch ? total - before : s_cmass[ch];
      if (next >= target) break;
    }
    if (pch != held) {
      mine = histogram(pch);
      held = pch;
    }
    const uint32_t key = (uint32_t)pch << 10 | (uint32_t)(1023 - tid);
    const double w = mine ? weight(key, top, c) : 0.0;
    const double v = (double)mine * w;
    double all;
    // the weight before this key: exactly `before` for the chunk's first one
    const double excl = before + (block_scan<double>(v, s_wd, &all) - v);
    // the border is the last key of the chunk before which less than the target lies
    // (the row's first always stays; a chunk's first does, as `before` is less)
    const bool in = mine && (excl < target || key == top);
    __syncthreads();
    if (tid == 0) s_key[2] = 0xFFFFFFFFu;
    __syncthreads();
    if (in) atomicMin(&s_key[2], key);
    __syncthreads();
    if (in && key == s_key[2]) {
      const double need = w > 0.0 ? ceil((target - excl) / w) : (double)mine;
      s_key[3] = (uint32_t)fmin(fmax(need, 1.0), (double)mine);
    }
    __syncthreads();
    bkey = s_key[2];
    bkeep = s_key[3];
  }
  if (lo > 0.0f) {
    // the smallest key whose weight reaches min-p: chunk, 16-key run, key
    __syncthreads();
    if (wave == 0) {
      uint32_t base = 0;
#pragma unroll
      for (int st = 10; st >= 4; st -= 6) {            // every 1024th key, every 16th of a chunk
        const uint32_t key = base + ((uint32_t)lane << st);
        const bool ok = key > kNegInf && weight(min(key, top), top, c) >= (double)lo;
        const uint64_t bal = __ballot(ok);
        const int nth = bal ? __builtin_ctzll(bal) : 64;
        base += (uint32_t)max(nth - 1, 0) << st;
      }
      // the border lies in the 16 keys after `base`, or is it
      const uint32_t key = base + (uint32_t)lane;
      const bool ok = key > kNegInf && weight(min(key, top), top, c) >= (double)lo;
      const uint64_t bal = __ballot(ok);
      if (lane == 0) s_key[2] = bal ? base + (uint32_t)__builtin_ctzll(bal) : top + 1;
    }
    __syncthreads();
    const uint32_t mk = s_key[2];
    if (mk > top) {                                    // min-p above 1: the first token alone
      bkey = top;
      bkeep = 1;
    } else if (mk > bkey) {
      bkey = mk;
      bkeep = 0xFFFFFFFFu;
    }
  }

  // kept weight of each slice: whole chunks above the border's, its own logit by logit
  const int bch = (int)(bkey >> 10);
  for (int s = wave; s < S; s += kPT / 64) {
    double ms = 0.0;
    uint32_t tie = 0;
    if (ws[s].max_key > kNegInf) {
      if (lane > bch && ws[s].cnt[lane]) ms = (double)ws[s].mass[lane] * (1.0 / kFix) * s_f[s];
      const int n = (int)ws[s].cnt[bch];
      const uint32_t* seg = ws[s].seg + ws[s].off[bch];
      for (int i = lane; i < n; i += 64) {
        const uint32_t key = seg[i] >> 16;
        if (key > bkey) ms += weight(key, top, c);
        tie += key == bkey;
      }
    }
#pragma unroll
    for (int d = 32; d >= 1; d >>= 1) {
      ms += __shfl_xor(ms, d, 64);
      tie += (uint32_t)__shfl_xor((int)tie, d, 64);
    }
    if (lane == 0) {
      s_sm[s] = ms;
      s_tie[s] = tie;
    }
  }
  __syncthreads();
  // S <= kPT: one slice per thread
  const double wb = weight(bkey, top, c);
  uint32_t ties_all;
  const uint32_t tie = tid < S ? s_tie[tid] : 0u;
  const uint32_t tie_before = block_scan<uint32_t>(tie, s_wu, &ties_all) - tie;
  const uint32_t stay = tie_before >= bkeep ? 0u : min(tie, bkeep - tie_before);
  const double mass = tid < S ? s_sm[tid] + (double)stay * wb : 0.0;
  double sum;
  const double incl = block_scan<double>(mass, s_wd, &sum);
  const float u = a.u[m];
  const double target = (u > 0.f ? (u < 1.f ? (double)u : 1.0) : 0.0) * sum;
  __syncthreads();
  if (tid == 0) {
    s_key[2] = 0xFFFFFFFFu;
    s_key[3] = 0;
  }
  __syncthreads();
  if (mass > 0.0) {
    if (incl > target) atomicMin(&s_key[2], (uint32_t)tid);
    atomicMax(&s_key[3], (uint32_t)tid);               // the last slice with any weight
  }
  __syncthreads();
  const int sl = (int)(s_key[2] != 0xFFFFFFFFu ? s_key[2] : s_key[3]);
  if (tid == sl) {
    s_d[0] = incl - mass;
    s_hist[0] = stay;
  }
  __syncthreads();
  const double base = s_d[0];
  const uint32_t keep = s_hist[0];

  // the slice's logits in index order, four per thread
  const uint16_t* xr = a.x + (int64_t)m * a.ldx;
  const int i0 = sl * kSlice + tid * 4;
  uint32_t kk[4], eq = 0;
#pragma unroll
  for (int e = 0; e < 4; ++e) {
    const uint16_t b = i0 + e < a.N ? xr[i0 + e] : (uint16_t)0xFC00u;
    kk[e] = is_nan16(b) ? kNegInf : key_of(b);
    eq += kk[e] == bkey;
  }
  uint32_t ignored;
  uint32_t rank = block_scan<uint32_t>(eq, s_wu, &ignored) - eq;
  double w[4], mine4 = 0.0;
#pragma unroll
  for (int e = 0; e < 4; ++e) {
    const bool in = kk[e] > bkey || (kk[e] == bkey && rank < keep);
    rank += kk[e] == bkey;
    w[e] = in ? weight(kk[e], top, c) : 0.0;
    mine4 += w[e];
  }
  double ignored_d;
  double cum = base + block_scan<double>(mine4, s_wd, &ignored_d) - mine4;
  __syncthreads();
  if (tid == 0) {
    s_key[2] = 0xFFFFFFFFu;
    s_key[3] = 0;
  }
  __syncthreads();
#pragma unroll
  for (int e = 0; e < 4; ++e) {
    cum += w[e];
    if (w[e] > 0.0) {
      if (cum > target) atomicMin(&s_key[2], (uint32_t)(i0 + e));
      atomicMax(&s_key[3], (uint32_t)(i0 + e));        // the last token with any weight
    }
  }
  __syncthreads();
  if (tid == 0) a.out[m] = (int64_t)(s_key[2] != 0xFFFFFFFFu ? s_key[2] : s_key[3]);
}

}  // namespace

extern "C" int64_t helm_sample_workspace_bytes(int M, int N) {
  if (M < 1 || N < 1) return 0;
  return (int64_t)M * ((N + (int64_t)kSlice - 1) / kSlice) * (int64_t)sizeof(SliceOut);
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
  a.ws = static_cast<SliceOut*>(workspace); a.out = out;
  const bool vec = helm::aligned16(x) && ldx % 8 == 0;
  const hipStream_t s = static_cast<hipStream_t>(stream);
  hipLaunchKernelGGL(sample_slice_kernel, dim3(a.S, M), dim3(kST), 0, s, a, vec);
  HELM_CHECK_LAUNCH("helm_sample slice launch");
  hipLaunchKernelGGL(sample_pick_kernel, dim3(M), dim3(kPT), 0, s, a);
  HELM_CHECK_LAUNCH("helm_sample pick launch");
  return HELM_OK;
}
