// The largest logits of a row, and sampling from a row of logits, on gfx950.
//
// Both rank a row's V logits x by (value falling, index rising); -0 equals +0
// and a NaN counts as -infinity.
//
// Top logits: the K first of that order, and the log-sum-exp of x_i / T over
// all others.
//
// Sampling at a temperature T: token j of the order has the whole-number weight
//   w_j = floor(2^42 exp((x_j - x_0) / T) + 1/2),
// so that every sum below is exact in 64 bits, whatever its order, and atomic
// additions cannot change a result (V <= 2^20 keeps a sum below 2^62).  Top-k
// keeps the first k tokens, top-p of these the shortest prefix with at least
// p of their weight, min-p of these the tokens with w_j >= min_p 2^42.  Each
// keeps a prefix of the order, so what is kept is told by its weight C alone,
// and the token drawn with the uniform number u is the first whose running sum
// passes floor(u C).  A row is never sorted: all that is needed is to find the
// token at a given running sum (or rank), "locating" it.
//
// The first tokens of the order come cheaply: the k-th largest of the threads'
// own maxima is a lower bound of the k-th largest logit that few other logits
// pass (T ln(1 / (1 - k/T)) of them for T threads and logits in no particular
// order); those that do are collected and ranked by counting, each against
// each.  That is all that the top logits and a small top-k need.  Without one,
// sampling adds up the weights of the whole row, and is done where the tokens
// so ranked hold what top-p asks for and the draw falls on one of them, as it
// does unless a distribution is rather flat.
//
// Locating, in general: a histogram of weights (or counts) over 2048 bins that
// are linear in (x_0 - x) / T up to the 43 ln 2 past which weights are zero; a
// prefix sum over it names the bin; the bin's tokens (about 50 for logits with
// a spread of a few nats) are collected and ranked by counting.  A bin with
// more than 1024 tokens is cut again by their bit patterns until it has fewer,
// or holds one value only, whose tokens rank by index.
//
// One workgroup per row.  The top logits hold the row in registers; sampling
// reads it again on every pass, from the caches, in loops that are not unrolled
// (with the fp64 exponentials in them they would not fit the instruction cache).

#include "kvm_rows.hpp"

namespace kvm {
namespace {

typedef unsigned long long u64;

constexpr int kBins = 2048;
constexpr int kCand = 1024;        // tokens that are ranked by counting
constexpr int kFirst = 128;        // tokens that sampling without a small top-k looks at first
constexpr int kMaxTop = 512;       // K of the top logits
constexpr double kUnit = 4398046511104.0;  // 2^42

// Bit patterns in the order of the values: larger float, larger key.
__device__ __forceinline__ uint32_t key_of(float x) {
  const uint32_t b = __float_as_uint(fmaxf(x, kNegInf) + 0.f);  // NaN -> -infinity, -0 -> +0
  return (b >> 31) ? ~b : b | 0x80000000u;
}
__device__ __forceinline__ float value_of(uint32_t key) {
  return __uint_as_float((key >> 31) ? key ^ 0x80000000u : ~key);
}
// The order of a row as one number: larger first.
__device__ __forceinline__ u64 rank_of(uint32_t key, int idx) { return u64(key) << 32 | (0xffffffffu - uint32_t(idx)); }
__device__ __forceinline__ int index_of(u64 rank) { return int(0xffffffffu - uint32_t(rank)); }
__device__ __forceinline__ uint32_t key_part(u64 rank) { return uint32_t(rank >> 32); }

// 2^42 2^(i / 256), rounded from the Taylor series of exp(i ln 2 / 256).
constexpr int kTable = 256;
struct Powers {
  double v[kTable];
  constexpr Powers() : v() {
    for (int i = 0; i < kTable; ++i) {
      const double f = double(i) * (0.6931471805599453 / kTable);
      double p = 1.0;
      for (int k = 24; k >= 1; --k) p = 1.0 + p * f / double(k);
      v[i] = p * kUnit;
    }
  }
};
__constant__ const Powers kPowers = Powers();

// Weights and bins of a row at one temperature.
struct Weights {
  float best;          // x_0
  double per;          // 256 log2(e) / T
  float bins_per;      // bins per unit of logit
  const double *table; // kPowers in LDS
  // 2^52 + floor(2^42 exp((x - best) / T) + 1/2) for a finite best: y = 256
  // log2 of the exponential is a whole number n and f, |f| <= 1/2; 2^(n/256) is
  // an entry of the table with its exponent moved, 2^(f/256) the Taylor series
  // to the fourth power (off by less than 2^-54), and adding 2^52 to the
  // product rounds it to a whole number in the low bits.  Weights below half a
  // unit, of -infinity and NaN are 0.  No contraction: a token's weight is the
  // same wherever it is computed.
  __device__ __forceinline__ double raised(float x) const {
#pragma clang fp contract(off)
    constexpr double kLn = 0.6931471805599453 / kTable;
    double y = (double(x) - double(best)) * per;
    y = fmax(y, -44.0 * kTable);
    const double shifted = y + 6755399441055744.0;  // 3 * 2^51: n in the low bits
    const double f = y - (shifted - 6755399441055744.0);
    const int n = int(__builtin_bit_cast(u64, shifted));
    double p = kLn * kLn * kLn * kLn / 24.0;
    p = __builtin_fma(p, f, kLn * kLn * kLn / 6.0);
    p = __builtin_fma(p, f, kLn * kLn / 2.0);
    p = __builtin_fma(p, f, kLn);
    p = __builtin_fma(p, f, 1.0);
    u64 e = __builtin_bit_cast(u64, table[n & (kTable - 1)]);
    e += u64(uint32_t(n & ~(kTable - 1)) << 12) << 32;  // the whole part of n / 256 into the exponent
    return __builtin_fma(__builtin_bit_cast(double, e), p, 4503599627370496.0);
  }
  __device__ __forceinline__ u64 operator()(float x) const {
    if (best == __builtin_inff()) return x == best ? u64(kUnit) : 0;  // infinities share
    return __builtin_bit_cast(u64, raised(x)) & 0xfffffffffffffull;
  }
  __device__ __forceinline__ float place(float x) const { return (x == best ? 0.f : best - x) * bins_per; }
  __device__ __forceinline__ int bin(float x) const {
    return int(fminf(fmaxf(place(x), 0.f), float(kBins - 1)));  // NaN (0 times infinity): 0
  }
  // Whether a token may have a weight: false only for weights of 0.
  __device__ __forceinline__ bool some(float x) const { return place(x) < float(kBins); }
};

struct Shared {
  u64 hist[kBins];
  u64 fine[kBins];
  u64 cand[kCand];
  u64 cw[kCand];
  u64 scan[17];
  float red[16];
  int ired[16];
  uint32_t kmin, kmax;
  int count, bin;
  u64 base;        // weight (or count) before the located bin
  u64 found;       // the located token (its rank_of)
  u64 found_end;   // running sum including it
  int above;       // of a bound: thread maxima before its bin
  double table[kTable];
};

template <int T>
__device__ __forceinline__ float block_max(float v, float *red) {
  v = wave_max(v);
  __syncthreads();
  if ((threadIdx.x & 63) == 0) red[threadIdx.x >> 6] = v;
  __syncthreads();
  return part_max<T / kWave>(red);
}
template <int T>
__device__ __forceinline__ int block_min(int v, int *red) {
#pragma unroll
  for (int o = 32; o >= 1; o >>= 1) v = min(v, __shfl_xor(v, o));
  __syncthreads();
  if ((threadIdx.x & 63) == 0) red[threadIdx.x >> 6] = v;
  __syncthreads();
#pragma unroll
  for (int w = 0; w < T / kWave; ++w) v = min(v, red[w]);
  return v;
}
template <int T>
__device__ __forceinline__ u64 block_add(u64 v, u64 *red) {
#pragma unroll
  for (int o = 32; o >= 1; o >>= 1) v += __shfl_xor(v, o);
  __syncthreads();
  if ((threadIdx.x & 63) == 0) red[threadIdx.x >> 6] = v;
  __syncthreads();
  v = 0;
#pragma unroll
  for (int w = 0; w < T / kWave; ++w) v += red[w];
  return v;
}
// Exclusive prefix sum over the workgroup's threads; *total its end.
template <int T>
__device__ __forceinline__ u64 block_scan(u64 v, u64 *red, u64 *total) {
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  u64 s = v;
#pragma unroll
  for (int o = 1; o < 64; o <<= 1) {
    const u64 up = __shfl_up(s, o);
    if (lane >= o) s += up;
  }
  __syncthreads();
  if (lane == 63) red[wave] = s;
  __syncthreads();
  u64 before = 0, all = 0;
#pragma unroll
  for (int w = 0; w < T / kWave; ++w) {
    if (w < wave) before += red[w];
    all += red[w];
  }
  *total = all;
  return before + s - v;
}

// Collects the values of a row with keys >= bound (in no particular order)
// and returns how many there are; the list holds the first kCand of them.
// TAKE: they leave the registers.
template <int T, bool TAKE, class R>
__device__ __forceinline__ int collect_above(R &x, uint32_t bound, Shared &sh) {
  constexpr int N = R::N;
  if (threadIdx.x == 0) sh.count = 0;
  __syncthreads();
  const float least = value_of(bound);
  auto chunk = [&](const float (&v)[N], int i0, int n) -> uint32_t {
    float m = v[0];
#pragma unroll
    for (int i = 1; i < N; ++i) m = fmaxf(m, v[i]);
    uint32_t bits = 0;
    if (!(m < least)) {  // nothing but NaN comes here too and is compared by key
#pragma unroll
      for (int i = 0; i < N; ++i) {
        const uint32_t k = key_of(v[i]);
        if (i < n && k >= bound) {
          bits |= 1u << i;
          const int at = atomicAdd(&sh.count, 1);
          if (at < kCand) sh.cand[at] = rank_of(k, i0 + i);
        }
      }
    }
    return bits;
  };
  if constexpr (TAKE)
    x.take(chunk);
  else
    x.each(chunk);
  __syncthreads();
  return sh.count;
}

// A lower bound of the k-th largest key of the row: one of the threads' maxima
// that k of them or a few more reach, from a histogram of the maxima over 256
// bins, twice.  Where fewer than k threads hold a number, -infinity's key.
template <int T>
__device__ __forceinline__ uint32_t bound_of(float thread_max, int k, Shared &sh) {
  constexpr int kCuts = 256;
  uint32_t *hist = reinterpret_cast<uint32_t *>(sh.fine);
  const int t = threadIdx.x;
  const uint32_t mine = key_of(thread_max), none = 0x007fffffu;  // -infinity's
  bool in = mine != none;
  int above = 0;
  uint32_t bound = none;
#pragma unroll 1
  for (int level = 0; level < 2; ++level) {
    __syncthreads();
    for (int i = t; i < kCuts; i += T) hist[i] = 0;
    if (t == 0) {
      sh.kmin = 0xffffffffu;
      sh.kmax = 0;
      sh.bin = -1;
    }
    __syncthreads();
    uint32_t lo = wave_min_u(in ? mine : 0xffffffffu), hi = wave_max_u(in ? mine : 0);
    if ((t & 63) == 0) {
      atomicMin(&sh.kmin, lo);
      atomicMax(&sh.kmax, hi);
    }
    __syncthreads();
    lo = sh.kmin;
    hi = sh.kmax;
    const float per = float(kCuts) / (float(hi - lo) + 1.f);
    const int cut = in ? min(int(float(hi - mine) * per), kCuts - 1) : kCuts;
    if (in) atomicAdd(&hist[cut], 1u);
    __syncthreads();
    if (t < kWave) {
      uint32_t q[kCuts / kWave], own = 0;
#pragma unroll
      for (int i = 0; i < kCuts / kWave; ++i) own += q[i] = hist[t * (kCuts / kWave) + i];
      uint32_t s = own;
#pragma unroll
      for (int o = 1; o < kWave; o <<= 1) {
        const uint32_t up = __shfl_up(s, o);
        if (t >= o) s += up;
      }
      s += above - own;
#pragma unroll
      for (int i = 0; i < kCuts / kWave; ++i) {
        if (int(s) < k && int(s + q[i]) >= k) {
          sh.bin = t * (kCuts / kWave) + i;
          sh.above = int(s);
          sh.count = int(s + q[i]);
        }
        s += q[i];
      }
    }
    __syncthreads();
    const int bin = sh.bin, reach = sh.count;
    if (bin < 0) return none;  // fewer than k numbers
    above = sh.above;
    // the smallest maximum of that bin
    const uint32_t least = wave_min_u(cut == bin ? mine : 0xffffffffu);
    if (t == 0) sh.kmin = 0xffffffffu;  // read by all before the last barrier
    __syncthreads();
    if ((t & 63) == 0) atomicMin(&sh.kmin, least);
    __syncthreads();
    bound = sh.kmin;
    if (reach <= k + k / 4 + 8) break;
    in = cut == bin;
  }
  return bound;
}

// f(i, token, rank) for the cnt tokens of the list, rank = how many of them
// come before it, once per token (by one lane).  A token is compared by as
// many lanes as there are to spare.
template <int T, class F>
__device__ __forceinline__ void ranked(int cnt, const Shared &sh, F &&f) {
  const int t = threadIdx.x;
  int lanes = 1;
  while (lanes < 16 && 2 * lanes * cnt <= T) lanes *= 2;
  const int part = t & (lanes - 1);
  for (int i0 = 0; i0 < cnt; i0 += T / lanes) {
    const int i = i0 + t / lanes;
    const u64 me = sh.cand[min(i, cnt - 1)];
    int r = 0;
#pragma unroll 4
    for (int j = part; j < cnt; j += lanes) r += sh.cand[j] > me;
    for (int o = lanes / 2; o >= 1; o >>= 1) r += __shfl_xor(r, o);
    if (part == 0 && i < cnt) f(i, me, r);
  }
}

// The token at running sum `target` (before <= target < before + its own) in
// the order of the row, of weights (COUNT: of ones).  hist: the quantity per
// bin of the row, which has been built; mine: this thread's exclusive prefix of
// it.  Writes sh.found and sh.found_end.  in(x) selects values with a positive
// quantity; every thread gets here.
template <int T, bool COUNT, class R, class In>
__device__ __forceinline__ void locate(const R &x, const Weights &wt, u64 target, u64 mine, Shared &sh, In &&in) {
  constexpr int N = R::N, PER = kBins / T;
  const int t = threadIdx.x;
  // the bin
  __syncthreads();
  {
    u64 s = mine;
#pragma unroll
    for (int i = 0; i < PER; ++i) {
      const u64 q = sh.hist[t * PER + i];
      if (target >= s && target < s + q) {
        sh.bin = t * PER + i;
        sh.base = s;
      }
      s += q;
    }
  }
  if (t == 0) {
    sh.count = 0;
    sh.kmin = 0xffffffffu;
    sh.kmax = 0;
  }
  __syncthreads();
  const int bin = sh.bin;
  u64 base = sh.base;
  uint32_t lo = 0, hi = 0xffffffffu;  // keys of the tokens in question
  bool first = true;
  uint32_t f_hi = 0, f_span = 0;
  int f_bin = 0;
  while (true) {
    // collect the tokens of the (sub-)bin, with their smallest and largest key
    uint32_t a = 0xffffffffu, b = 0;
    x.each([&](const float (&v)[N], int i0, int n) {
#pragma unroll
      for (int i = 0; i < N; ++i) {
        if (i < n) {
          if (wt.bin(v[i]) != bin) continue;
          const uint32_t k = key_of(v[i]);
          bool hit = k >= lo && k <= hi;
          if (hit && !first) hit = int(u64(f_hi - k) * kBins / (u64(f_span) + 1)) == f_bin;
          if (hit && in(v[i], i0 + i)) {
            a = min(a, k);
            b = max(b, k);
            const int at = atomicAdd(&sh.count, 1);
            if (at < kCand) sh.cand[at] = rank_of(k, i0 + i);
          }
        }
      }
    });
    if (a <= b) {
      atomicMin(&sh.kmin, a);
      atomicMax(&sh.kmax, b);
    }
    __syncthreads();
    const int cnt = sh.count;
    lo = sh.kmin;
    hi = sh.kmax;
    if (cnt <= kCand) {
      for (int i = t; i < cnt; i += T) sh.cw[i] = COUNT ? 1 : wt(value_of(key_part(sh.cand[i])));
      __syncthreads();
      int lanes = 1;
      while (lanes < 16 && 2 * lanes * cnt <= T) lanes *= 2;
      const int part = t & (lanes - 1);
      for (int i0 = 0; i0 < cnt; i0 += T / lanes) {
        const int i = min(i0 + t / lanes, cnt - 1);
        const u64 me = sh.cand[i];
        u64 before = 0;
#pragma unroll 4
        for (int j = part; j < cnt; j += lanes)
          if (sh.cand[j] > me) before += sh.cw[j];
        for (int o = lanes / 2; o >= 1; o >>= 1) before += __shfl_xor(before, o);
        before += base;
        if (target >= before && target < before + sh.cw[i]) {
          sh.found = me;
          sh.found_end = before + sh.cw[i];
        }
      }
      __syncthreads();
      return;
    }
    if (lo == hi) {
      // One value: the n-th of its tokens by index, found by bisection over the index.
      const u64 w = COUNT ? 1 : wt(value_of(lo));
      const u64 nth = (target - base) / w;
      int below = -1, upto = (1 << 20) - 1;  // at most nth tokens are <= below, more than nth are <= upto
      while (upto - below > 1) {
        const int mid = below + (upto - below) / 2;
        u64 c = 0;
        x.each([&](const float (&v)[N], int i0, int n) {
#pragma unroll
          for (int i = 0; i < N; ++i)
            if (i < n && i0 + i <= mid && key_of(v[i]) == lo && in(v[i], i0 + i)) ++c;
        });
        c = block_add<T>(c, sh.scan);
        if (c > nth)
          upto = mid;
        else
          below = mid;
      }
      if (t == 0) {
        sh.found = rank_of(lo, upto);
        sh.found_end = base + (nth + 1) * w;
      }
      __syncthreads();
      return;
    }
    // cut [lo, hi] into kBins by key, the largest keys first
    __syncthreads();
    for (int i = t; i < kBins; i += T) sh.fine[i] = 0;
    f_hi = hi;
    f_span = hi - lo;
    __syncthreads();
    x.each([&](const float (&v)[N], int i0, int n) {
#pragma unroll
      for (int i = 0; i < N; ++i) {
        if (i >= n || wt.bin(v[i]) != bin) continue;
        const uint32_t k = key_of(v[i]);
        if (k >= lo && k <= hi && in(v[i], i0 + i))
          atomicAdd(&sh.fine[int(u64(f_hi - k) * kBins / (u64(f_span) + 1))], COUNT ? 1 : wt(v[i]));
      }
    });
    __syncthreads();
    u64 own = 0, all;
#pragma unroll
    for (int i = 0; i < PER; ++i) own += sh.fine[t * PER + i];
    u64 s = base + block_scan<T>(own, sh.scan, &all);
#pragma unroll
    for (int i = 0; i < PER; ++i) {
      const u64 q = sh.fine[t * PER + i];
      if (target >= s && target < s + q) {
        sh.bin = t * PER + i;
        sh.base = s;
      }
      s += q;
    }
    if (t == 0) {
      sh.count = 0;
      sh.kmin = 0xffffffffu;
      sh.kmax = 0;
    }
    __syncthreads();
    f_bin = sh.bin;
    base = sh.base;
    first = false;
  }
}

// Histogram of a row's weights (COUNT: of ones) over the values that in()
// selects; returns this thread's exclusive prefix, *total the sum.  strong
// (optional): the sum of the weights >= least.
template <int T, bool COUNT, class R, class In>
__device__ __forceinline__ u64 build(const R &x, const Weights &wt, Shared &sh, u64 *total, double least, u64 *strong,
                                     In &&in) {
  constexpr int N = R::N, PER = kBins / T;
  const int t = threadIdx.x;
  __syncthreads();
  for (int i = t; i < kBins; i += T) sh.hist[i] = 0;
  __syncthreads();
  u64 big = 0;
  x.each([&](const float (&v)[N], int i0, int n) {
#pragma unroll
    for (int i = 0; i < N; ++i) {
      if (i < n && wt.some(v[i]) && in(v[i], i0 + i)) {
        const u64 w = COUNT ? 1 : wt(v[i]);
        if (w) atomicAdd(&sh.hist[wt.bin(v[i])], w);
        if (strong && double(w) >= least) big += w;
      }
    }
  });
  __syncthreads();
  if (strong) *strong = block_add<T>(big, sh.scan);
  u64 own = 0;
#pragma unroll
  for (int i = 0; i < PER; ++i) own += sh.hist[t * PER + i];
  return block_scan<T>(own, sh.scan, total);
}

// floor(u * c) for a uniform number, inside [0, c - 1] whatever u is.
__device__ __forceinline__ u64 target_of(float u, u64 c) {
  const double at = floor(double(u) * double(c));
  const u64 last = c - 1;
  if (!(at > 0.0)) return 0;
  return at >= double(last) ? last : u64(at);
}

template <int DT, int T>
__global__ __launch_bounds__(T) __attribute__((amdgpu_waves_per_eu(4))) void k_sample(kvm_sample_desc P) {
  using R = Row<DT, T, 0>;
  constexpr int N = R::N;
  __shared__ Shared sh;
  const int t = threadIdx.x, row = blockIdx.x;
  const int V = int(P.logits.vocab);
  R x;
  x.open(logits_row<DT>(P.logits, row), V);
  const float temp = P.temperature ? P.temperature[row] : float(P.temperature_all);
  float top_p = P.top_p ? P.top_p[row] : float(P.top_p_all);
  float min_p = P.min_p ? P.min_p[row] : float(P.min_p_all);
  top_p = top_p < 1.f ? top_p : 1.f;  // a NaN keeps everything
  min_p = min_p > 0.f ? min_p : 0.f;
  const int top_k = P.top_k ? P.top_k[row] : int(P.top_k_all);
  const float u = P.uniforms[row];
  if (t < kTable) sh.table[t] = kPowers.v[t];

  float mine = kNegInf;
  x.each([&](const float (&v)[N], int, int) {
#pragma unroll
    for (int i = 0; i < N; ++i) mine = fmaxf(mine, v[i]);
  });
  const float best = block_max<T>(mine, sh.red);
  auto answer = [&](int token, float logprob) {  // one thread
    P.tokens[row] = token;
    if (P.logprobs) P.logprobs[row] = logprob;
  };
  if (best == kNegInf) {  // nothing to draw from
    if (t == 0) answer(0, __builtin_nanf(""));
    return;
  }
  if (!(temp > 0.f) || top_k == 1) {  // the first token of the order
    int at = 0x7fffffff;
    x.each([&](const float (&v)[N], int i0, int n) {
#pragma unroll
      for (int i = N - 1; i >= 0; --i)
        if (i < n && v[i] == best) at = min(at, i0 + i);
    });
    at = block_min<T>(at, sh.ired);
    if (t == 0) answer(at, 0.f);
    return;
  }
  Weights wt;
  wt.best = best;
  wt.per = kTable * (1.4426950408889634 / double(temp));
  // 43 octaves of weight fill the bins
  wt.bins_per = float(fmin(double(kBins) / (43.0 * 0.6931471805599453 * double(temp)), 3e38));
  wt.table = sh.table;
  const double least = double(min_p) * kUnit;
  auto write = [&](u64 rank, u64 c) {  // one thread: the token and ln(w / C)
    const float xv = value_of(key_part(rank));
    const double d = xv == best ? 0.0 : (double(xv) - double(best)) / double(temp);
    answer(index_of(rank), float(d - log(double(c) / kUnit)));
  };

  // The first tokens of the order.
  const bool some = top_k > 0 && top_k < V;  // top-k drops tokens
  const bool few = some && top_k <= T / 2;
  const uint32_t bound = bound_of<T>(mine, few ? top_k : kFirst, sh);
  const int cnt = collect_above<T, false>(x, bound, sh);
  const bool covers = few || cnt == V;  // no token past the list is kept
  if (cnt <= kCand && (covers || !some)) {
    u64 *sorted = sh.hist, *weight = sh.hist + kCand;
    ranked<T>(cnt, sh, [&](int, u64 me, int r) {
      sorted[r] = me;
      weight[r] = wt(value_of(key_part(me)));
    });
    u64 z = 0, strong = 0;
    if (!covers) {  // the weight of the whole row
      u64 calls = 0;
      if (min_p > 0.f) {
        x.each([&](const float (&v)[N], int, int) {
#pragma unroll
          for (int i = 0; i < N; ++i) {
            const u64 w = wt(v[i]);
            z += w;
            if (double(w) >= least) strong += w;
          }
        });
        strong = block_add<T>(strong, sh.scan);
      } else if (best == __builtin_inff()) {
        x.each([&](const float (&v)[N], int, int) {
#pragma unroll
          for (int i = 0; i < N; ++i) z += v[i] == best ? u64(kUnit) : 0;
        });
      } else {
        // The bits of 2^52 + w are added up as they are; the constant part of
        // every term is taken off modulo 2^64.
        x.each([&](const float (&v)[N], int, int) {
          calls += N;
#pragma unroll
          for (int i = 0; i < N; ++i) z += __builtin_bit_cast(u64, wt.raised(v[i]));
        });
        z -= calls * (u64(0x433) << 52);
      }
      z = block_add<T>(z, sh.scan);
    }
    __syncthreads();
    bool done = true;
    if (t < kWave) {  // one wave finishes: consecutive tokens per lane, a prefix sum of their weights
      const int k = some ? min(top_k, cnt) : cnt, per = (k + kWave - 1) / kWave;
      const int first = min(t * per, k), last = min(first + per, k);
      u64 own = 0;
      for (int i = first; i < last; ++i) own += weight[i];
      u64 before = own;
#pragma unroll
      for (int o = 1; o < kWave; o <<= 1) {
        const u64 up = __shfl_up(before, o);
        if (t >= o) before += up;
      }
      const u64 sum = __shfl(before, kWave - 1);
      before -= own;
      if (covers) z = sum;
      const double end = double(top_p) * double(z);
      // What is kept of the list: each lane's last kept running sum, the largest of them.
      u64 c = 0, run = before;
      for (int i = first; i < last; ++i) {
        const u64 w = weight[i];
        if (i == 0 || (double(run) < end && double(w) >= least)) c = run + w;
        run += w;
      }
#pragma unroll
      for (int o = 32; o >= 1; o >>= 1) {
        const u64 other = __shfl_xor(c, o);
        c = other > c ? other : c;
      }
      if (!covers) {
        // Past the list: the weight of the row, unless top-p or min-p ends inside it.
        const bool p_in = top_p < 1.f && double(sum) >= end;
        const bool m_in = min_p > 0.f && strong < sum;
        if (!p_in && !m_in) {
          done = top_p >= 1.f;
          c = min_p > 0.f ? strong : z;
        }
      }
      const u64 at = target_of(u, c);
      done = done && at < sum;
      if (done) {
        run = before;
        for (int i = first; i < last; ++i) {
          const u64 w = weight[i];
          if (at >= run && at < run + w) write(sorted[i], c);
          run += w;
        }
      }
      if (t == 0) sh.count = done;
    }
    __syncthreads();
    if (sh.count) return;
  }
  auto all = [](float, int) { return true; };
  u64 limit = 0;  // the last token that top-k keeps (0: it keeps all)
  u64 z;
  if (some) {
    const u64 pre = build<T, true>(x, wt, sh, &z, 0.0, nullptr, all);
    if (u64(top_k) < z) {
      locate<T, true>(x, wt, u64(top_k) - 1, pre, sh, [&](float v, int) { return wt.some(v); });
      limit = sh.found;
    }
  }
  auto kept = [&](float v, int i) { return limit == 0 || rank_of(key_of(v), i) >= limit; };
  u64 strong = 0;
  const u64 pre = build<T, false>(x, wt, sh, &z, least, min_p > 0.f ? &strong : nullptr, kept);
  auto weighted = [&](float v, int i) { return wt.some(v) && kept(v, i) && wt(v) != 0; };
  u64 c = z;
#pragma unroll 1
  for (int step = top_p < 1.f ? 0 : 1; step < 2; ++step) {  // where top-p ends, then the draw
    u64 target;
    if (step == 0) {
      const double end = ceil(double(top_p) * double(z));
      target = end >= 1.0 ? u64(end) - 1 : 0;
    } else {
      if (min_p > 0.f && strong < c) c = strong;
      if (c < u64(kUnit)) c = u64(kUnit);  // the first token is always kept
      target = target_of(u, c);
    }
    locate<T, false>(x, wt, target, pre, sh, weighted);
    if (step == 0) c = sh.found_end;
  }
  if (t == 0) write(sh.found, c);
}

template <int DT, int T, int NV>
__global__ __launch_bounds__(T) __attribute__((amdgpu_waves_per_eu(4))) void k_top_logits(kvm_logits L, int K, float scale, void *values, int64_t *indices,
                                                  float *rest) {
  using R = Row<DT, T, NV>;
  using E = Elem<DT>;
  constexpr int N = R::N;
  __shared__ Shared sh;
  __shared__ u64 s_last, s_next;
  const int t = threadIdx.x, row = blockIdx.x;
  const int V = int(L.vocab);
  R x;
  x.open(logits_row<DT>(L, row), V);
  float mine = kNegInf;
  x.each([&](const float (&v)[N], int, int) {
#pragma unroll
    for (int i = 0; i < N; ++i) mine = fmaxf(mine, v[i]);
  });
  if (t == 0) s_next = 0;
  const uint32_t bound = bound_of<T>(mine, K, sh);
  int cnt = collect_above<T, (NV > 0)>(x, bound, sh);
  const bool many = cnt > kCand;
  Row<DT, T, 0> again;  // for rows that are not in registers, or no longer whole there
  if (NV == 0 || many) again.open(logits_row<DT>(L, row), V);
  u64 more_ties = 0;  // tokens of the K-th value behind it that are not in the list
  if (many) {
    // Many equal or clustered logits: the K-th token by rank, then exactly K are collected.
    Weights wt;  // one bin: the tokens are cut by their keys from the start
    wt.best = 0.f;
    wt.per = 0.0;
    wt.bins_per = 0.f;
    wt.table = sh.table;
    __syncthreads();
    for (int i = t; i < kBins; i += T) sh.hist[i] = i ? 0 : u64(V);
    locate<T, true>(again, wt, u64(K) - 1, t ? u64(V) : 0, sh, [](float, int) { return true; });
    const u64 last = sh.found;
    __syncthreads();
    if (t == 0) sh.count = 0;
    __syncthreads();
    u64 ties = 0;
    again.each([&](const float (&v)[N], int i0, int n) {
#pragma unroll
      for (int i = 0; i < N; ++i) {
        if (i < n) {
          const uint32_t k = key_of(v[i]);
          const u64 me = rank_of(k, i0 + i);
          if (me >= last) {
            const int at = atomicAdd(&sh.count, 1);
            if (at < kCand) sh.cand[at] = me;
          } else if (k == key_part(last)) {
            ++ties;
          }
        }
      }
    });
    __syncthreads();
    more_ties = block_add<T>(ties, sh.scan);
    cnt = K;
  }
  ranked<T>(cnt, sh, [&](int i, u64 me, int r) {
    sh.cw[i] = u64(r);
    if (r < K) {
      static_cast<typename E::raw *>(values)[int64_t(row) * K + r] = E::put(value_of(key_part(me)));
      indices[int64_t(row) * K + r] = index_of(me);
    }
    if (r == K - 1) s_last = me;
    if (r == K) s_next = me;
  });
  if (!rest) return;
  __syncthreads();
  const u64 last = s_last, next = s_next;
  // The largest of the others: behind the K-th in the list, or below the list's bound.
  float m = next ? value_of(key_part(next)) : kNegInf;
  float z = 0.f;
  double ref2;  // the sum's reference, in log2 units
  if (NV > 0 && !many) {
    if (!next) {
      x.each([&](const float (&v)[N], int, int) {
#pragma unroll
        for (int i = 0; i < N; ++i) m = fmaxf(m, v[i]);
      });
      m = block_max<T>(m, sh.red);
    }
    const float ref = m == kNegInf ? 0.f : m, scaled = ref * scale;
    if (fabsf(scaled) < 1e30f) {
      ref2 = double(scaled);
      auto term = [&](float v) { return __builtin_amdgcn_exp2f(__builtin_fmaf(v, scale, -scaled)); };
      x.each([&](const float (&v)[N], int, int) {
#pragma unroll
        for (int i = 0; i < N; ++i) z += term(fmaxf(v[i], kNegInf));
      });
      for (int i = t; i < cnt; i += T)
        if (sh.cw[i] >= u64(K)) z += term(value_of(key_part(sh.cand[i])));
    } else {  // logits near the type's lowest value: subtracted before they are scaled
      ref2 = double(ref) * scale;
      auto term = [&](float v) { return __builtin_amdgcn_exp2f((v - ref) * scale); };
      x.each([&](const float (&v)[N], int, int) {
#pragma unroll
        for (int i = 0; i < N; ++i) z += term(fmaxf(v[i], kNegInf));
      });
      for (int i = t; i < cnt; i += T)
        if (sh.cw[i] >= u64(K)) z += term(value_of(key_part(sh.cand[i])));
    }
  } else {
    const uint32_t kth = key_part(last);
    const float vk = value_of(kth);
    u64 in_list = 0;
    for (int i = t; i < cnt; i += T) in_list += sh.cand[i] < last && key_part(sh.cand[i]) == kth;
    const float ties = float(block_add<T>(in_list, sh.scan) + more_ties);
    if (!next && K < V) {
      again.each([&](const float (&v)[N], int, int) {
#pragma unroll
        for (int i = 0; i < N; ++i) m = fmaxf(m, v[i] < vk ? v[i] : kNegInf);
      });
      m = block_max<T>(m, sh.red);
      if (ties > 0.f) m = vk;
    }
    const float ref = m == kNegInf ? 0.f : m;
    ref2 = double(ref) * scale;
    again.each([&](const float (&v)[N], int, int) {
#pragma unroll
      for (int i = 0; i < N; ++i) z += __builtin_amdgcn_exp2f(v[i] < vk ? (v[i] - ref) * scale : kNegInf);
    });
    if (t == 0) z += ties;  // each of them is the reference itself: m = vk, exp = 1
  }
  z = wave_add(z);
  __syncthreads();
  if ((t & 63) == 0) sh.red[t >> 6] = z;
  __syncthreads();
  if (t < 16) {
    z = part_add<T / kWave>(sh.red);
    const double lse = m == kNegInf ? -__builtin_inf()
                       : m == __builtin_inff() ? __builtin_inf()
                                               : (ref2 + log2(double(z))) * 0.6931471805599453;
    if (t == 0) rest[row] = float(lse);
  }
}

struct TopLaunch {
  const kvm_logits &L;
  int K;
  float scale;
  void *values;
  int64_t *indices;
  float *rest;
  hipStream_t stream;
  template <int DT, int T, int NV>
  void run() {
    hipLaunchKernelGGL((k_top_logits<DT, T, NV>), dim3(unsigned(L.outer * L.inner)), dim3(T), 0, stream, L, K, scale,
                       values, indices, rest);
  }
};

}  // namespace

int64_t top_logits_max() { return kMaxTop; }

hipError_t launch_sample(const kvm_sample_desc &P, hipStream_t stream) {
  // Up to one row per compute unit: 1024 threads finish a row soonest; more
  // rows: workgroups of 512, two of which share a compute unit.
  const int64_t rows = P.logits.outer * P.logits.inner;
  const dim3 grid{unsigned(rows)};
#define KVM_SAMPLE(D)                                                                \
  if (rows <= 256)                                                                   \
    hipLaunchKernelGGL((k_sample<D, 1024>), grid, dim3(1024), 0, stream, P);         \
  else                                                                               \
    hipLaunchKernelGGL((k_sample<D, 512>), grid, dim3(512), 0, stream, P);
  if (P.logits.dtype == KVM_BF16) {
    KVM_SAMPLE(KVM_BF16)
  } else if (P.logits.dtype == KVM_F16) {
    KVM_SAMPLE(KVM_F16)
  } else {
    KVM_SAMPLE(KVM_F32)
  }
#undef KVM_SAMPLE
  return hipGetLastError();
}

hipError_t launch_top_logits(const kvm_logits &L, int64_t k, double temperature, void *values, int64_t *indices,
                             float *rest, hipStream_t stream) {
  TopLaunch l{L, int(k), float(1.4426950408889634 / temperature), values, indices, rest, stream};
  // At least twice as many threads as values: the bound from the threads' maxima then passes 1.4 K logits or fewer.
  with_row(L.vocab, L.dtype, 2 * k, l);
  return hipGetLastError();
}

}  // namespace kvm
