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
// sampling is done where the tokens so ranked hold what top-p asks for and the
// draw falls on one of them, as it does unless a distribution is rather flat.
// For top-p that takes the weight of the whole row only as closely as to tell
// which token it ends on: a sum in fp32 with its error bound, and the exact one
// where a token's edge falls within that bound or C is the weight of the row.
//
// Locating, in general: a histogram of weights (or counts) over 2048 bins that
// are linear in (x_0 - x) / T up to the 43 ln 2 past which weights are zero; a
// prefix sum over it names the bin; the bin's tokens (about 50 for logits with
// a spread of a few nats) are collected and ranked by counting.  A bin with
// more than 1024 tokens is cut again by their bit patterns until it has fewer,
// or holds one value only, whose tokens rank by index.
//
// One workgroup per row.  The top logits, and the first passes of sampling
// where there are more rows than compute units, hold it in registers; other
// passes read it again, from the caches, in loops (a pass over registers has
// its code once per chunk, which one workgroup alone would read from memory).
//
// Measured: the top 64 of 8192 rows of 50304 bf16 logits 0.25 ms, VALU 70 % busy
// (9 of 16 instructions per logit are the maximum's and the exponential's); 512
// rows of 65536 bf16 logits with min-p 23 us; one row of 50304 fp32 logits with
// top-p 16 us where the first list decides (22 with the exact weight of the row
// on one compute unit), 45 where it does not (the list 13, the histogram 16, the
// two searches 11 and 8).

#include <type_traits>

#include "kvm_rows.hpp"

namespace kvm {
namespace {

typedef unsigned long long u64;

constexpr int kBins = 2048;
constexpr int kCand = 1024;        // tokens that are ranked by counting
constexpr int kFirst = 128;        // tokens that sampling without a small top-k looks at first
constexpr int kMany = 4096;        // tokens of the list for a larger top-k
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
  int hit_chunks, hit_tokens;
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

// The chunks of a row that hold a value >= least, as collect_above lists them:
// packed in sh.hist, with the first token and the number of values in sh.cw.
struct Hits {
  int chunks;   // in the list
  float least;
  bool every;   // NaN and -infinity too
  // f(value, token, whether it is one of those >= least) for the list's values.
  template <int T, class E, class F>
  __device__ __forceinline__ void each(const Shared &sh, F &&f) const {
    for (int i = threadIdx.x; i < chunks * E::N; i += T) {
      const uint32_t tag = reinterpret_cast<const uint32_t *>(sh.cw)[i / E::N];
      const int e = i % E::N;
      if (e < int(tag >> 24)) {
        const float v = E::get(reinterpret_cast<const typename E::raw *>(sh.hist)[i]);
        f(v, int(tag & 0xffffff) + e, v >= least || every);
      }
    }
  }
};
constexpr int kHitChunks = 1024;

// Collects the tokens of a row with keys >= bound (in no particular order) and
// returns how many there are; the list holds the first kCand of them (more
// than kCand where their chunks do not fit either).  A pass over a row has its
// code once per chunk, so a chunk with such a token only goes to LDS; its
// tokens are looked at from there.  TAKE: those chunks leave the registers.
// also(v) is called on the way for the values of every chunk of a row that is
// read again, also(x) for a row in registers.
template <int T, bool TAKE, class R, int M, class F>
__device__ __forceinline__ int collect_above(R &x, const float (&most)[M], uint32_t bound, Shared &sh, Hits *hits,
                                             F &&also) {
  constexpr int N = R::N;
  uint4 *const chunks = reinterpret_cast<uint4 *>(sh.hist);
  uint32_t *const tags = reinterpret_cast<uint32_t *>(sh.cw);
  if (threadIdx.x == 0) sh.hit_chunks = sh.hit_tokens = 0;
  __syncthreads();
  const float least = value_of(bound);
  const bool every = least == kNegInf;
  auto list = [&](const float (&v)[N], int i0, int n) {
    const int at = atomicAdd(&sh.hit_chunks, 1);
    if (at < kHitChunks) {
      chunks[at] = R::E::pack(v);
      tags[at] = uint32_t(n) << 24 | uint32_t(i0);
    }
  };
  if constexpr (R::kResident) {
    x.template above<TAKE>(most, least, every, list);
    also(x);
  } else {
    auto above = [&](const float (&v)[N], bool there) {
      if (there) also(v);
      float m = v[0];
#pragma unroll
      for (int i = 1; i < N; ++i) m = fmaxf(m, v[i]);
      return m >= least || every;
    };
    x.where(above, list);
  }
  __syncthreads();
  *hits = {min(sh.hit_chunks, kHitChunks), least, every};
  if (sh.hit_chunks > kHitChunks) return kCand + 1;
  hits->template each<T, typename R::E>(sh, [&](float v, int idx, bool of_them) {
    if (of_them) {
      const int at = atomicAdd(&sh.hit_tokens, 1);
      if (at < kCand) sh.cand[at] = rank_of(key_of(v), idx);
    }
  });
  __syncthreads();
  return sh.hit_tokens;
}

// Inclusive prefix sum over a wave: shifts within rows of 16 lanes, then the
// rows' totals across (DPP row_shr, row_bcast).
template <int CTRL, int ROWS>
__device__ __forceinline__ uint32_t moved(uint32_t v) {
  return uint32_t(__builtin_amdgcn_update_dpp(0, int(v), CTRL, ROWS, 0xf, false));
}
__device__ __forceinline__ uint32_t wave_scan(uint32_t v) {
  v += moved<0x111, 0xf>(v);
  v += moved<0x112, 0xf>(v);
  v += moved<0x114, 0xf>(v);
  v += moved<0x118, 0xf>(v);
  v += moved<0x142, 0xa>(v);
  v += moved<0x143, 0xc>(v);
  return v;
}

// A lower bound of the k-th largest key of the row that k of the threads'
// maxima or a few more reach: the edge of a bin of a histogram of the maxima
// over 256 bins, cut once more where that bin is too full.  Where fewer than k
// threads hold a number, -infinity's key.
template <int T>
__device__ __forceinline__ uint32_t bound_of(float thread_max, int k, Shared &sh) {
  constexpr int kCuts = 256, PER = kCuts / kWave;
  uint32_t *hist = reinterpret_cast<uint32_t *>(sh.fine), *least = hist + kCuts, *most = least + 16;
  const int t = threadIdx.x;
  const uint32_t mine = key_of(thread_max), none = 0x007fffffu;  // -infinity's
  bool in = mine != none;
  int above = 0;
  uint32_t bound = none;
#pragma unroll 1
  for (int level = 0; level < 2; ++level) {
    if (level) __syncthreads();
    for (int i = t; i < kCuts; i += T) hist[i] = 0;
    uint32_t lo = wave_min_u(in ? mine : 0xffffffffu), hi = wave_max_u(in ? mine : 0);
    if ((t & 63) == 0) {
      least[t >> 6] = lo;
      most[t >> 6] = hi;
    }
    if (t == 0) sh.bin = -1;
    __syncthreads();
    const int l = t & 15;
    lo = l < T / kWave ? least[l] : 0xffffffffu;
    hi = l < T / kWave ? most[l] : 0;
    lo = wave_min_u(lo);
    hi = wave_max_u(hi);
    const float span = float(hi - lo) + 1.f, per = float(kCuts) / span;
    const int cut = in ? min(int(float(hi - mine) * per), kCuts - 1) : kCuts;
    if (in) atomicAdd(&hist[cut], 1u);
    __syncthreads();
    if (t < kWave) {
      uint32_t q[PER], own = 0;
#pragma unroll
      for (int i = 0; i < PER; ++i) own += q[i] = hist[t * PER + i];
      uint32_t s = above + wave_scan(own) - own;
#pragma unroll
      for (int i = 0; i < PER; ++i) {
        if (int(s) < k && int(s + q[i]) >= k) {
          sh.bin = t * PER + i;
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
    // The bin's lower edge: 2^-20 of the distance below where the fp32 cuts put it, to be on the safe side.
    const float below = float(bin + 1) * (span / float(kCuts)) * 1.000001f + 2.f;
    bound = below < float(hi - none) ? hi - uint32_t(below) : none;
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

// What is located: a rank among all tokens (one bin), a rank among the tokens
// that may have a weight, or a running sum of weights.
enum Quantity { kEvery, kCounted, kWeighed };

// The tokens of a chunk that lie in a bin, as bits.
template <Quantity Q, int N>
__device__ __forceinline__ uint32_t in_bin(const Weights &wt, const float (&v)[N], int n, int bin) {
  uint32_t bits = 0;
#pragma unroll
  for (int i = 0; i < N; ++i) {
    const float p = wt.place(v[i]);
    bits |= Q == kEvery || (p >= float(bin) && p < float(bin + 1)) ? 1u << i : 0u;
  }
  return bits & ((1u << n) - 1);
}

// The token at running sum `target` (before <= target < before + its own) in
// the order of the row.  hist: the quantity per bin, which has been built;
// mine: this thread's exclusive prefix of it; limit (kWeighed; 0: none): the
// last token that counts.  Writes sh.found and sh.found_end; every thread
// gets here.
template <int T, Quantity Q, class R>
__device__ __forceinline__ void locate(const R &x, const Weights &wt, u64 target, u64 mine, u64 limit, Shared &sh) {
  constexpr int N = R::N, PER = kBins / T;
  const int t = threadIdx.x;
  auto amount = [&](float v) -> u64 { return Q == kWeighed ? wt(v) : 1; };
  // Names the bin of `list` that holds the target; s: the sum before this thread's bins.
  auto choose = [&](const u64 *list, u64 s) {
#pragma unroll
    for (int i = 0; i < PER; ++i) {
      const u64 q = list[t * PER + i];
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
  };
  __syncthreads();
  choose(sh.hist, mine);
  const int bin = sh.bin;
  u64 base = sh.base;
  // The tokens in question: those of the bin with keys in [lo, hi] and, past
  // the first cut, in part f_part of kBins equal parts of [f_hi - f_span, f_hi].
  uint32_t lo = 0, hi = 0xffffffffu, f_hi = 0, f_span = 0;
  int f_part = -1;
  auto part_of = [&](uint32_t k) { return int(u64(f_hi - k) * kBins / (u64(f_span) + 1)); };
  // |x - mid| <= half for every value of the bin and few others, whatever the
  // rounding of either; where that says nothing (an edge is not finite) for all.
  const float width = 1.f / wt.bins_per;
  float mid = wt.best - (float(bin) + 0.5f) * width;
  float half = 0.501f * width + (fabsf(wt.best) + fabsf(mid)) * 0x1p-21f;
  if (!(half < __builtin_inff())) mid = 0.f, half = __builtin_inff();
  auto tokens = [&](auto &&f) {  // f(key, index, value) for each of them
    auto near = [&](const float (&v)[N], bool) {
      bool any = Q == kEvery;
#pragma unroll
      for (int i = 0; i < N; ++i) any = any | (fabsf(v[i] - mid) <= half);
      return any;
    };
    x.where(near, [&](const float (&v)[N], int i0, int n) {
      for (uint32_t bits = in_bin<Q, N>(wt, v, n, bin); bits; bits &= bits - 1) {
        const int e = __ffs(bits) - 1, idx = i0 + e;
        float xv = v[0];
#pragma unroll
        for (int i = 1; i < N; ++i) xv = e == i ? v[i] : xv;
        const uint32_t k = key_of(xv);
        if (k >= lo && k <= hi && (f_part < 0 || part_of(k) == f_part) && rank_of(k, idx) >= limit) f(k, idx, xv);
      }
    });
  };
#pragma unroll 1
  while (true) {
    // collect them, with their smallest and largest key
    uint32_t a = 0xffffffffu, b = 0;
    tokens([&](uint32_t k, int idx, float) {
      a = min(a, k);
      b = max(b, k);
      const int at = atomicAdd(&sh.count, 1);
      if (at < kCand) sh.cand[at] = rank_of(k, idx);
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
      for (int i = t; i < cnt; i += T) sh.cw[i] = amount(value_of(key_part(sh.cand[i])));
      __syncthreads();
      int lanes = 1;
      while (lanes < 16 && 2 * lanes * cnt <= T) lanes *= 2;
      const int part = t & (lanes - 1);
      for (int i0 = 0; i0 < cnt; i0 += T / lanes) {
        const int i = min(i0 + t / lanes, cnt - 1);
        const u64 me = sh.cand[i];
        u64 before = 0;
#pragma unroll 4
        for (int j = part; j < cnt; j += lanes) {
          const u64 w = sh.cw[j];
          before += sh.cand[j] > me ? w : 0;
        }
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
      const u64 w = max(amount(value_of(lo)), u64(1));
      const u64 nth = (target - base) / w;
      const int last = limit && key_part(limit) == lo ? index_of(limit) : 0x7fffffff;
      int below = -1, upto = int(kMaxVocab) - 1;  // at most nth tokens are <= below, more than nth are <= upto
#pragma unroll 1
      while (upto - below > 1) {
        const int mid = below + (upto - below) / 2;
        u64 c = 0;
        x.template each<1>([&](const float (&v)[N], int i0, int n) {
#pragma unroll
          for (int i = 0; i < N; ++i) c += i < n && i0 + i <= min(mid, last) && key_of(v[i]) == lo;
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
    // cut [lo, hi] into kBins parts, the largest keys first
    __syncthreads();
    for (int i = t; i < kBins; i += T) sh.fine[i] = 0;
    f_hi = hi;
    f_span = hi - lo;
    f_part = -1;
    __syncthreads();
    tokens([&](uint32_t k, int, float v) { atomicAdd(&sh.fine[part_of(k)], amount(v)); });
    __syncthreads();
    u64 own = 0, all;
#pragma unroll
    for (int i = 0; i < PER; ++i) own += sh.fine[t * PER + i];
    choose(sh.fine, base + block_scan<T>(own, sh.scan, &all));
    f_part = sh.bin;
    base = sh.base;
  }
}

// Histogram of a row's weights (kCounted: of ones) over the tokens down to
// limit (0: all); returns this thread's exclusive prefix, *total the sum.
// strong (optional): the sum of the weights >= least.
template <int T, Quantity Q, class R>
__device__ __forceinline__ u64 build(const R &x, const Weights &wt, u64 limit, Shared &sh, u64 *total, double least,
                                     u64 *strong) {
  constexpr int N = R::N, PER = kBins / T;
  const int t = threadIdx.x;
  __syncthreads();
  for (int i = t; i < kBins; i += T) sh.hist[i] = 0;
  __syncthreads();
  u64 big = 0;
  auto pass = [&](auto &&weight) {
    x.template each<1>([&](const float (&v)[N], int i0, int n) {
#pragma unroll
      for (int i = 0; i < N; ++i) {
        const u64 w = weight(v[i]);
        const float place = wt.place(v[i]);
        if (i < n && place < float(kBins) && (limit == 0 || rank_of(key_of(v[i]), i0 + i) >= limit)) {
          atomicAdd(&sh.hist[int(place)], w);
          if (Q == kWeighed && strong && double(w) >= least) big += w;
        }
      }
    });
  };
  if constexpr (Q == kCounted)
    pass([](float) { return u64(1); });
  else if (wt.best == __builtin_inff())
    pass([&](float v) { return u64(v == wt.best ? kUnit : 0.0); });
  else
    pass([&](float v) { return __builtin_bit_cast(u64, wt.raised(v)) & 0xfffffffffffffull; });
  __syncthreads();
  if (Q == kWeighed && strong) *strong = block_add<T>(big, sh.scan);
  u64 own = 0;
#pragma unroll
  for (int i = 0; i < PER; ++i) own += sh.hist[t * PER + i];
  return block_scan<T>(own, sh.scan, total);
}

// Tokens of a row in a list, as the functions above read a row.
template <int T>
struct Listed {
  static constexpr int N = 1;
  const u64 *list;
  int cnt;
  template <int BATCH, class F>
  __device__ __forceinline__ void each(F &&f) const {
#pragma unroll 1
    for (int i0 = 0; i0 < cnt; i0 += T) {
      const int i = i0 + threadIdx.x;
      const u64 token = list[min(i, cnt - 1)];
      const float v[1] = {value_of(key_part(token))};
      f(v, index_of(token), i < cnt ? 1 : 0);
    }
  }
  template <class W, class F>
  __device__ __forceinline__ void where(W &&, F &&f) const {
    each<1>(f);
  }
};

// Lists the first tokens of the order, `want` or somewhat more (all that may
// have a weight where there are fewer): a histogram of the chunks' maxima names
// a bin whose edge `want` of them reach; the tokens before that edge are
// collected.  Returns how many there are, kMany of them at most in the list.
template <int T, class R>
__device__ __forceinline__ int list_first(const R &x, const Weights &wt, int want, u64 *list, Shared &sh) {
  constexpr int N = R::N, PER = kBins / T;
  uint32_t *const hist = reinterpret_cast<uint32_t *>(sh.fine);
  const int t = threadIdx.x;
  __syncthreads();
  for (int i = t; i < kBins; i += T) hist[i] = 0;
  if (t == 0) {
    sh.bin = kBins - 1;
    sh.count = 0;
  }
  __syncthreads();
  x.template each<1>([&](const float (&v)[N], int, int) {
    float m = v[0];
#pragma unroll
    for (int i = 1; i < N; ++i) m = fmaxf(m, v[i]);
    if (wt.some(m)) atomicAdd(&hist[wt.bin(m)], 1u);
  });
  __syncthreads();
  uint32_t own = 0;
#pragma unroll
  for (int i = 0; i < PER; ++i) own += hist[t * PER + i];
  u64 all;
  int s = int(block_scan<T>(own, sh.scan, &all));
#pragma unroll
  for (int i = 0; i < PER; ++i) {
    const int q = int(hist[t * PER + i]);
    if (s < want && s + q >= want) sh.bin = t * PER + i;
    s += q;
  }
  __syncthreads();
  const float edge = float(sh.bin + 1);
  auto before = [&](const float (&v)[N], bool) {
    float m = v[0];
#pragma unroll
    for (int i = 1; i < N; ++i) m = fmaxf(m, v[i]);
    return wt.place(m) < edge;
  };
  x.where(before, [&](const float (&v)[N], int i0, int n) {
#pragma unroll
    for (int i = 0; i < N; ++i) {
      if (wt.place(v[i]) < edge && i < n) {
        const int at = atomicAdd(&sh.count, 1);
        if (at < kMany) list[at] = rank_of(key_of(v[i]), i0 + i);
      }
    }
  });
  __syncthreads();
  return sh.count;
}

// floor(u * c) for a uniform number, inside [0, c - 1] whatever u is.
__device__ __forceinline__ u64 target_of(float u, u64 c) {
  const double at = floor(double(u) * double(c));
  const u64 last = c - 1;
  if (!(at > 0.0)) return 0;
  return at >= double(last) ? last : u64(at);
}

template <int DT, int T, int NV>
__global__ __launch_bounds__(T) __attribute__((amdgpu_waves_per_eu(4))) void k_sample(kvm_sample_desc P) {
  using R = Row<DT, T, NV, true>;
  constexpr int N = R::N;
  __shared__ Shared sh;
  __shared__ u64 many[NV == 0 ? kMany : 1];
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

  float most[NV > 0 ? NV : 1];  // of the chunks
  float mine = kNegInf;
  if constexpr (NV > 0) {
    mine = x.maxima(most);
  } else {
    x.each([&](const float (&v)[N], int, int) {
#pragma unroll
      for (int i = 0; i < N; ++i) mine = fmaxf(mine, v[i]);
    });
  }
  const float best = block_max<T>(mine, sh.red);
  auto answer = [&](int token, float logprob) {  // one thread
    P.tokens[row] = token;
    if (P.logprobs) P.logprobs[row] = logprob;
  };
  Row<DT, T, 0> again;  // the passes after the first two read the row again
  again.open(logits_row<DT>(P.logits, row), V);
  if (best == kNegInf) {  // nothing to draw from
    if (t == 0) answer(0, __builtin_nanf(""));
    return;
  }
  if (!(temp > 0.f) || top_k == 1) {  // the first token of the order
    int at = 0x7fffffff;
    again.each([&](const float (&v)[N], int i0, int n) {
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
  // Whether min-p drops all tokens past the list, whose keys are below the bound.
  const bool m_in = min_p > 0.f && double(wt(value_of(bound))) < least;
  // Whether the row's weight matters: not where top-k or min-p alone says where the kept tokens end.
  const bool weighed = !some && !(m_in && top_p >= 1.f);
  // That weight in fp32, on the way: enough to tell where top-p ends unless
  // that falls on the edge of a token within its error.
  float about = 0.f;
  const float log2_per = 1.4426950408889634f / temp;
  auto terms = [&](const float (&v)[N]) {
#pragma unroll
    for (int i = 0; i < N; ++i) about += __builtin_amdgcn_exp2f((v[i] - best) * log2_per);
  };
  Hits hits;
  const int cnt = collect_above<T, false>(x, most, bound, sh, &hits, [&](const auto &part) {
    if constexpr (NV > 0) {
      if (weighed) part.each([&](const float (&v)[N], int, int) { terms(v); });
    } else {
      if (weighed) terms(part);
    }
  });
  const bool covers = few || cnt == V;  // no token past the list is kept
  if (cnt <= kCand && (covers || !some)) {
    u64 *sorted = sh.hist, *weight = sh.hist + kCand;
    ranked<T>(cnt, sh, [&](int, u64 me, int r) {
      sorted[r] = me;
      weight[r] = wt(value_of(key_part(me)));
    });
    about = wave_add(about);
    if ((t & 63) == 0) sh.red[t >> 6] = about;
    __syncthreads();
    enum { kDone, kWeigh, kLocate };
    // One wave finishes: consecutive tokens per lane, a prefix sum of their
    // weights.  The row's weight is within [z_lo, z_hi]; where they are equal, z
    // and strong (the weight of its tokens that min-p keeps) are exact.  Leaves in
    // sh.count whether the token was found, needs the exact weight, or lies past
    // the list.
    auto finish = [&](double z_lo, double z_hi, u64 z, u64 strong) {
      if (t < kWave) {
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
        if (covers) z_lo = z_hi = double(sum);
        const bool exact = z_lo == z_hi;
        const double end_lo = double(top_p) * z_lo, end_hi = double(top_p) * z_hi;
        // What is kept of the list: each lane's last kept running sum, the largest of them.
        u64 c = 0, run = before;
        bool edge = false;  // a token that top-p may keep or not
        for (int i = first; i < last; ++i) {
          const u64 w = weight[i];
          const double at = double(run);
          if (i == 0 || ((top_p >= 1.f || at < end_lo) && double(w) >= least)) c = run + w;
          edge = edge || (i > 0 && top_p < 1.f && at >= end_lo && at < end_hi);
          run += w;
        }
#pragma unroll
        for (int o = 32; o >= 1; o >>= 1) {
          const u64 other = __shfl_xor(c, o);
          c = other > c ? other : c;
        }
        int state = __ballot(edge) ? kWeigh : kDone;
        if (!covers && !m_in) {
          if (top_p >= 1.f) {  // past the list: the weight of the row, or of what min-p keeps of it
            c = min_p > 0.f ? strong : z;
            if (!exact) state = min_p <= 0.f && double(u) * z_lo > double(sum) ? kLocate : kWeigh;
          } else if (double(sum) < end_hi) {  // top-p may end past the list
            state = double(sum) < end_lo ? kLocate : kWeigh;
          }
        }
        if (!(z_lo <= z_hi)) state = kWeigh;  // NaN: infinities or NaN among the logits
        if (state == kDone) {
          const u64 at = target_of(u, c);
          if (at >= sum) state = kLocate;
          run = before;
          for (int i = first; i < last; ++i) {
            const u64 w = weight[i];
            if (at >= run && at < run + w) write(sorted[i], c);
            run += w;
          }
        }
        if (t == 0) sh.count = state;
      }
      __syncthreads();
      return sh.count;
    };
    // The fp32 sum is off by at most 2^-24 of it for every term a thread adds,
    // and 2^-17 for the exponentials' arguments (three roundings of at most 62
    // octaves); the weights' own roundings and the terms below their unit are
    // 2^-22 at most.  Both are taken with a margin, 2^-22 a term and 2^-16.
    const double sum32 = weighed ? double(part_add<T / kWave>(sh.red)) * kUnit : 0.0;
    const double off = sum32 * (double(V / T + 64) / 4194304.0);
    int state = finish(sum32 - off, sum32 + off, 0, 0);
    if (state == kWeigh) {
      u64 z = 0, strong = 0;
      if (best == __builtin_inff()) {
        again.template each<1>([&](const float (&v)[N], int, int) {
#pragma unroll
          for (int i = 0; i < N; ++i) z += v[i] == best ? u64(kUnit) : 0;
        });
      } else {
        // The bits of 2^52 + w are added up as they are; the constant part of
        // every term is taken off modulo 2^64.
        u64 calls = 0;
        again.template each<1>([&](const float (&v)[N], int, int) {
          calls += N;
#pragma unroll
          for (int i = 0; i < N; ++i) z += __builtin_bit_cast(u64, wt.raised(v[i]));
        });
        z -= calls * (u64(0x433) << 52);
      }
      if (min_p > 0.f && !m_in) {
        again.template each<1>([&](const float (&v)[N], int, int) {
#pragma unroll
          for (int i = 0; i < N; ++i) {
            const u64 w = wt(v[i]);
            strong += double(w) >= least ? w : 0;
          }
        });
        strong = block_add<T>(strong, sh.scan);
      }
      z = block_add<T>(z, sh.scan);
      state = finish(double(z), double(z), z, strong);
    }
    if (state == kDone) return;
  }
  // The draw, by locating, among the tokens of the row, or of a list that holds
  // all that top-k keeps.
  auto draw = [&](const auto &tokens) {
    u64 limit = 0, total;  // limit: the last token that top-k keeps (0: it keeps all)
    if (some) {
      const u64 pre = build<T, kCounted>(tokens, wt, 0, sh, &total, 0.0, nullptr);
      if (u64(top_k) < total) {
        locate<T, kCounted>(tokens, wt, u64(top_k) - 1, pre, 0, sh);
        limit = sh.found;
      }
    }
    u64 kept_strong = 0;
    const u64 pre = build<T, kWeighed>(tokens, wt, limit, sh, &total, least, min_p > 0.f ? &kept_strong : nullptr);
    u64 c = total;
#pragma unroll 1
    for (int step = top_p < 1.f ? 0 : 1; step < 2; ++step) {  // where top-p ends, then the draw
      u64 target;
      if (step == 0) {
        const double end = ceil(double(top_p) * double(c));
        target = end >= 1.0 ? u64(end) - 1 : 0;
      } else {
        if (min_p > 0.f && kept_strong < c) c = kept_strong;
        if (c < u64(kUnit)) c = u64(kUnit);  // the first token is always kept
        target = target_of(u, c);
      }
      locate<T, kWeighed>(tokens, wt, target, pre, limit, sh);
      if (step == 0) c = sh.found_end;
    }
    if (t == 0) write(sh.found, c);
  };
  if constexpr (NV == 0) {
    if (some && top_k <= kMany / 2) {
      const int listed = list_first<T>(again, wt, top_k, many, sh);
      if (listed <= kMany) {
        draw(Listed<T>{many, listed});
        return;
      }
    }
  }
  draw(again);
}

template <int DT, int T, int NV>
__global__ __launch_bounds__(T) __attribute__((amdgpu_waves_per_eu(4))) void k_top_logits(kvm_logits L, int K, float scale, void *values, int64_t *indices,
                                                  float *rest) {
  using R = Row<DT, T, NV, true>;
  using E = Elem<DT>;
  constexpr int N = R::N;
  __shared__ Shared sh;
  __shared__ u64 s_last, s_next, s_units;
  const int t = threadIdx.x, row = blockIdx.x;
  const int V = int(L.vocab);
  R x;
  x.open(logits_row<DT>(L, row), V);
  float most[NV > 0 ? NV : 1];  // of the chunks
  float mine = kNegInf;
  if constexpr (NV > 0) {
    mine = x.maxima(most);
  } else {
    x.each([&](const float (&v)[N], int, int) {
#pragma unroll
      for (int i = 0; i < N; ++i) mine = fmaxf(mine, v[i]);
    });
  }
  if (t == 0) s_next = s_units = 0;
  const uint32_t bound = bound_of<T>(mine, K, sh);
  Hits hits;
  int cnt = collect_above<T, (NV > 0)>(x, most, bound, sh, &hits, [](const auto &) {});
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
    locate<T, kEvery>(again, wt, u64(K) - 1, t ? u64(V) : 0, 0, sh);
    const u64 last = sh.found;
    __syncthreads();
    if (t == 0) sh.count = 0;
    __syncthreads();
    u64 ties = 0;
    again.template each<1>([&](const float (&v)[N], int i0, int n) {
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
  ranked<T>(cnt, sh, [&](int, u64 me, int r) {
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
  double ref2 = 0.0;  // the sum's reference, in log2 units
  bool done = false;
  if (NV > 0 && !many) {
    if (!next) {
      x.each([&](const float (&v)[N], int, int) {
#pragma unroll
        for (int i = 0; i < N; ++i) m = fmaxf(m, v[i]);
      });
      hits.template each<T, E>(sh, [&](float v, int, bool of_them) {
        if (!of_them) m = fmaxf(m, v);
      });
      m = block_max<T>(m, sh.red);
    }
    const float scaled = m == kNegInf ? 0.f : m * scale;
    if (fabsf(scaled) < 1e30f) {
      ref2 = double(scaled);
      auto term = [&](float v) { return __builtin_amdgcn_exp2f(__builtin_fmaf(v, scale, -scaled)); };
      // What left the registers but is not among the K: the rest of those chunks,
      // and of the list.  Both lists are in the order in which waves got there, so
      // these terms (at most 1) are added up as whole multiples of 2^-40.
      u64 units = 0;
      auto add = [&](float v) { units += u64(term(v) * 1099511627776.f); };
      hits.template each<T, E>(sh, [&](float v, int, bool of_them) {
        if (!of_them) add(fmaxf(v, kNegInf));
      });
      for (int i = t; i < cnt; i += T)
        if (sh.cand[i] < last) add(value_of(key_part(sh.cand[i])));
#pragma unroll
      for (int o = 32; o >= 1; o >>= 1) units += __shfl_xor(units, o);
      if ((t & 63) == 0) atomicAdd(&s_units, units);
      x.each([&](const float (&v)[N], int, int) {
#pragma unroll
        for (int i = 0; i < N; ++i) z += term(v[i]);
      });
      z = wave_add(z);
      __syncthreads();
      if ((t & 63) == 0) sh.red[t >> 6] = z;
      __syncthreads();
      z = part_add<T / kWave>(sh.red) + float(double(s_units) / 1099511627776.0);
      done = z == z;
    }
  }
  // Rows that are read again, too many equal logits, a NaN among them, or a
  // largest other that overflows when it is scaled before it is subtracted.
  if (!done) {
    if (NV > 0 && !many) again.open(logits_row<DT>(L, row), V);
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
    z = 0.f;
    again.each([&](const float (&v)[N], int, int) {
#pragma unroll
      for (int i = 0; i < N; ++i) z += __builtin_amdgcn_exp2f(v[i] < vk ? (v[i] - ref) * scale : kNegInf);
    });
    z = wave_add(z);
    __syncthreads();
    if ((t & 63) == 0) sh.red[t >> 6] = z;
    __syncthreads();
    z = ties + part_add<T / kWave>(sh.red);  // each of the ties is the reference itself: m = vk, exp = 1
  }
  if (t == 0) {
    const double lse = m == kNegInf ? -__builtin_inf()
                       : m == __builtin_inff() ? __builtin_inf()
                                               : (ref2 + log2(double(z))) * 0.6931471805599453;
    rest[row] = float(lse);
  }
}

struct SampleLaunch {
  const kvm_sample_desc &P;
  hipStream_t stream;
  template <int DT, int T, int NV>
  void run() {
    if constexpr (T >= 512)
      hipLaunchKernelGGL((k_sample<DT, T, NV>), dim3(unsigned(P.logits.outer * P.logits.inner)), dim3(T), 0, stream,
                         P);
  }
};

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
  // More rows than compute units: the rows stay in registers.  Fewer: a pass's
  // unrolled code would be read from memory by a workgroup that runs it once
  // (one row of 50304 when this was measured: 54 us, against 23 with the row read
  // again in loops).
  const int64_t rows = P.logits.outer * P.logits.inner;
  SampleLaunch l{P, stream};
  if (rows <= 256)
    with_row<false>(P.logits.vocab, P.logits.dtype, 1024, l);
  else
    with_row<true>(P.logits.vocab, P.logits.dtype, 512, l);
  return hipGetLastError();
}

hipError_t launch_top_logits(const kvm_logits &L, int64_t k, double temperature, void *values, int64_t *indices,
                             float *rest, hipStream_t stream) {
  TopLaunch l{L, int(k), float(1.4426950408889634 / temperature), values, indices, rest, stream};
  // At least twice as many threads as values: the bound from the threads' maxima then passes 1.4 K logits or fewer.
  with_row<true>(L.vocab, L.dtype, 2 * k, l);
  return hipGetLastError();
}

}  // namespace kvm
