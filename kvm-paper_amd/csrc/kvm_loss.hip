// Losses on a decoder's logits on gfx950: cross-entropy with hard labels, and
// distillation from a teacher's largest logits, each with its gradient.
//
// One row of V logits x, a label y, a teacher's K values t_k at tokens i_k and
// (optionally) the log-sum-exp R of the teacher's other logits, at the
// temperature T:
//   p   = softmax over (t_1/T, ..., t_K/T, R)   (R's entry is called r; without
//         R the softmax runs over the K values and r = 0)
//   q_k = the student's probability of token i_k at T, s that of all tokens
//         the teacher does not name, together
//   L   = (1 - a) T^2 [sum_k p_k ln(p_k / q_k) + r ln(r / s)]
//         + a [logsumexp(x) - x_y]
// and, with e_j = exp(x_j / T), Z = sum e over the row, Z_o = sum e over the
// tokens the teacher does not name, and P_j = sum of p_k with i_k = j:
//   dL/dx_j = (1 - a) T [e_j / Z - P_j - [j not named] r e_j / Z_o]
//           + a [softmax(x)_j - [j = y]].
// Both follow from d ln q_j / dx_i = ([i = j] - softmax_i) / T.  Z_o is summed
// directly, never as Z minus the named tokens, so a teacher and a student that
// both put nearly everything on the named tokens lose no digits.
//
// One workgroup per row.  The row is read once, into registers (16 chunks of
// 16 bytes per thread), and three passes run over the registers: maximum,
// sum of exponentials, gradient; a forward that needs a gradient therefore
// moves every logit once in and once out, and the backward has nothing left
// to do but a factor.  The teacher's tokens are marked in a bitmap in LDS (one
// bit per token, laid out as the chunks are: one LDS read per chunk) and hidden
// in the registers, so that the passes are those of a plain softmax; their
// gradient is written after the others' by the K threads that hold them.
//
// Sums and statistics are fp32, differences of logarithms of single tokens
// fp64 (they cancel where student and teacher agree).  The gradient is rounded
// once, to the type of the logits.
//
// Two workgroups of 512 threads share a compute unit (64 registers of a row,
// 128 in all): one loads while the other computes.  16384 rows of 50304 bf16
// logits, cross-entropy: 0.59 ms, 5.6 TB/s of reads and writes, the rate of a
// copy; VALU 57 % busy (14 instructions per logit).  8192 rows with 64 teacher
// values at T = 2 beside hard labels: 0.35 ms, VALU 82 % busy (25 per logit).

#include "kvm_rows.hpp"

namespace kvm {
namespace {

constexpr int kMaxTeacher = 1024;

// A value of one of the three types (teacher values: K per row).
__device__ __forceinline__ float load_any(const void *p, int64_t i, int dtype) {
  if (dtype == KVM_F32) return static_cast<const float *>(p)[i];
  const uint16_t b = static_cast<const uint16_t *>(p)[i];
  return dtype == KVM_BF16 ? Elem<KVM_BF16>::get(b) : Elem<KVM_F16>::get(b);
}

// A value that is the same in every lane, held once per wave.
__device__ __forceinline__ float uniform(float v) {
  return __builtin_bit_cast(float, __builtin_amdgcn_readfirstlane(__builtin_bit_cast(int, v)));
}
__device__ __forceinline__ double uniform(double v) {
  const uint64_t b = __builtin_bit_cast(uint64_t, v);
  const uint64_t lo = uint32_t(__builtin_amdgcn_readfirstlane(int(uint32_t(b))));
  const uint64_t hi = uint32_t(__builtin_amdgcn_readfirstlane(int(uint32_t(b >> 32))));
  return __builtin_bit_cast(double, hi << 32 | lo);
}

__device__ __forceinline__ float exp2_fast(float x) { return __builtin_amdgcn_exp2f(x); }

// log2(z) of a sum z >= 1 or so, off by about 2e-7 whatever its size: the
// fp32 logarithm and one Newton step on z 2^-l = 1.  -infinity for 0.
__device__ __forceinline__ double log2_fine(float z) {
  const float l = __log2f(z);
  const float fix = __builtin_fmaf(z, exp2_fast(-l), -1.f) * kLog2e;
  return z > 0.f ? double(l) + double(fix) : double(l);
}
// log2(2^a + 2^b) for doubles that may be -infinity.
__device__ __forceinline__ double log2_add(double a, double b) {
  const double m = fmax(a, b);
  if (m == -__builtin_inf()) return m;
  return m + log2_fine(exp2_fast(float(a - m)) + exp2_fast(float(b - m)));
}
// log2 of a sum s of 2^(v - ref): ref + log2(s), -infinity for an empty sum.
__device__ __forceinline__ double log2_of(double ref, float s) { return ref + log2_fine(s); }
// The reference of a sum of exponentials: the maximum, or 0 where there is
// none (every value -infinity), so that -infinity - reference stays -infinity.
__device__ __forceinline__ float reference(float m) { return m == kNegInf ? 0.f : m; }

template <int DT, int T, int NV, bool TEACHER>
__global__ __launch_bounds__(T) __attribute__((amdgpu_waves_per_eu(4))) void k_head_loss(kvm_head_loss_desc P, float every_row) {
  using R = Row<DT, T, NV>;
  using raw = typename R::raw;
  constexpr int N = R::N, W = T / kWave;
  extern __shared__ __align__(16) unsigned char dyn[];
  __shared__ float red_a[W][3], red_b[W][5], red_c[W];
  __shared__ int dup;
  const int t = threadIdx.x, lane = t & 63, wave = t >> 6;
  const int row = blockIdx.x;
  const int V = int(P.logits.vocab), K = int(P.k);
  float *const row_loss = P.row_loss;
  raw *grad = nullptr;
  if (P.grad) {
    const int o = row / int(P.logits.inner), i = row - o * int(P.logits.inner);
    grad = static_cast<raw *>(P.grad) + o * P.g_outer + i * P.g_inner;
  }
  // A gradient made again for an upstream gradient: rows for which it is one have theirs.
  const float up = P.upstream ? P.upstream[row * P.upstream_stride] : 1.f;
  if (P.upstream && up == 1.f) return;
  int64_t label = P.labels ? P.labels[row] : 0;
  const bool ignored = P.labels && label == P.ignore_index;
  // The teacher's first entries are asked for before the row: what depends on
  // them (the bitmap, the student's logits there) need not wait for the row.
  int64_t id_first = -1;
  float tv_first = kNegInf;
  if constexpr (TEACHER) {
    if (t < K) {
      id_first = P.t_indices[int64_t(row) * K + t];
      tv_first = load_any(P.t_values, int64_t(row) * K + t, int(P.t_dtype));
    }
  }
  R x;
  x.open(logits_row<DT>(P.logits, row), V);
  if (ignored) {  // uniform: no loss, a gradient of zeros
    if (t == 0) row_loss[row] = 0.f;
    if (grad)
      x.each([&](const float (&)[N], int i0, int n) {
        float z[N] = {};
        if (n == N)
          *reinterpret_cast<uint4 *>(grad + i0) = R::E::pack(z);
        else if (n == 1)
          grad[i0] = R::E::put(0.f);
      });
    return;
  }
  const float a = P.labels ? float(P.label_weight) : 0.f;  // weight of the hard labels
  float scale = (P.inv_count && P.labels ? *P.inv_count : every_row) * up;
  // A label outside the vocabulary (and not ignored) makes the row's loss and gradient NaN.
  const bool bad = P.labels && (label < 0 || label >= V);
  if (bad) {
    label = 0;
    scale = __builtin_nanf("");
  }
  const float tau = float(P.temperature);
  const float c = TEACHER ? kLog2e / tau : kLog2e;  // log2 units per logit at T
  const bool soft = TEACHER && a != 1.f;
  const bool hard = !TEACHER || a != 0.f;
  const bool two = TEACHER && hard && tau != 1.f;  // hard labels need a softmax of their own

  uint32_t *bits = nullptr;
  int *t_idx = nullptr;
  float *t_p = nullptr, *t_x = nullptr;
  if constexpr (TEACHER) {
    const int words = (V + 2 * N + 31) / 32;
    bits = reinterpret_cast<uint32_t *>(dyn);
    t_idx = reinterpret_cast<int *>(bits + (words + 3) / 4 * 4);
    t_p = reinterpret_cast<float *>(t_idx + K);
    t_x = t_p + K;
    for (int i = t; i < words; i += T) bits[i] = 0;
    if (t == 0) dup = 0;
    __syncthreads();
  }
  // ---- maxima: the teacher's values, the student's at the teacher's tokens, the student's others
  float m_t = kNegInf, m_x = kNegInf, m_o = kNegInf;
  if constexpr (TEACHER) {
    const raw *xr = logits_row<DT>(P.logits, row);
    for (int k = t; k < K; k += T) {
      const bool first = k == t;
      const int64_t id = first ? id_first : P.t_indices[int64_t(row) * K + k];
      const bool in = id >= 0 && id < V;  // anything else is padding
      float tv = first ? tv_first : load_any(P.t_values, int64_t(row) * K + k, int(P.t_dtype));
      float xv = R::E::get(xr[in ? id : 0]);
      if (!in) tv = xv = kNegInf;
      t_idx[k] = in ? int(id) : -1;
      t_p[k] = tv;
      t_x[k] = xv;
      m_t = fmaxf(m_t, tv);
      m_x = fmaxf(m_x, xv);
      if (in) {
        const int pos = x.shifted(int(id));
        const uint32_t bit = 1u << (pos & 31);
        if (atomicOr(&bits[pos >> 5], bit) & bit) dup = 1;
      }
    }
    __syncthreads();
  }
  // Bits of a chunk's tokens that the teacher names.  In registers those
  // tokens are hidden once; a row that is read again hides them on every pass.
  auto named = [&](int i0, int n) -> uint32_t {
    if (n == 0) return 0;
    const int pos = x.shifted(i0);
    return bits[pos >> 5] >> (pos & 31);
  };
  if constexpr (TEACHER) x.hide(named);
  auto others = [&](auto &&f) {
    x.each([&](const float (&v)[N], int i0, int n) {
      if constexpr (TEACHER && NV == 0) {
        const uint32_t nm = named(i0, n);
        float u[N];
#pragma unroll
        for (int i = 0; i < N; ++i) u[i] = nm >> i & 1 ? kNegInf : v[i];
        f(u, i0, n);
      } else {
        f(v, i0, n);
      }
    });
  };
  others([&](const float (&v)[N], int, int) {
#pragma unroll
    for (int i = 0; i < N; ++i) m_o = fmaxf(m_o, v[i]);
  });
  m_o = wave_max(m_o);
  if constexpr (TEACHER) {
    m_t = wave_max(m_t);
    m_x = wave_max(m_x);
  }
  if (lane == 0) {
    red_a[wave][0] = m_t;
    red_a[wave][1] = m_x;
    red_a[wave][2] = m_o;
  }
  __syncthreads();
  m_o = part_max<W>(&red_a[0][2], 3);
  if constexpr (TEACHER) {
    m_t = part_max<W>(&red_a[0][0], 3);
    m_x = part_max<W>(&red_a[0][1], 3);
  }
  const bool dups = TEACHER && dup;
  // ---- sums of exponentials.  Every logarithm below is relative to the
  // row's maximum m (the teacher's to its own, top2): logits are subtracted
  // before they are scaled and before they meet a logarithm, so that rows of
  // the type's lowest value neither overflow nor swallow it.
  const double m = uniform(reference(fmaxf(m_o, m_x)));
  m_o = uniform(reference(m_o));
  m_x = uniform(reference(m_x));
  const double rest2 = TEACHER && P.t_rest ? double(P.t_rest[row]) * 1.4426950408889634 : -__builtin_inf();
  double top2 = fmax(double(m_t) * c, rest2);
  if (top2 == -__builtin_inf()) top2 = 0.0;
  // The exponentials at T and, where hard labels need a softmax of their own,
  // at 1: one, or both, the second a power of the first for the usual whole T.
  // Each way has its own code, chosen once.
  enum Way { kOne, kBoth, kSquare, kFourth };
  const Way way = !two ? kOne : tau == 2.f ? kSquare : tau == 4.f ? kFourth : kBoth;
  auto chosen = [&](auto &&f) {
    if constexpr (TEACHER) {
      if (way == kBoth) return f(std::integral_constant<Way, kBoth>{});
      if (way == kSquare) return f(std::integral_constant<Way, kSquare>{});
      if (way == kFourth) return f(std::integral_constant<Way, kFourth>{});
    }
    return f(std::integral_constant<Way, kOne>{});
  };
  auto at_one = [&](auto w, float v, float e) -> float {  // exp(v - m_o) from e = exp((v - m_o) / T)
    if constexpr (decltype(w)::value == kBoth) return exp2_fast((v - m_o) * kLog2e);
    const float e2 = e * e;
    return decltype(w)::value == kSquare ? e2 : e2 * e2;
  };
  float z_o = 0.f, z_o1 = 0.f, z_t = 0.f, z_x = 0.f, z_x1 = 0.f;
  chosen([&](auto w) {
    others([&](const float (&v)[N], int, int) {
#pragma unroll
      for (int i = 0; i < N; ++i) {
        const float e = exp2_fast((v[i] - m_o) * c);
        z_o += e;
        if constexpr (decltype(w)::value != kOne) z_o1 += at_one(w, v[i], e);
      }
    });
  });
  // The lowest of the entries that name a token stands for it in the student's sums.
  auto first_of = [&](int k) -> bool {
    if (t_idx[k] < 0) return false;
    if (dups)
      for (int j = 0; j < k; ++j)
        if (t_idx[j] == t_idx[k]) return false;
    return true;
  };
  if constexpr (TEACHER) {
    for (int k = t; k < K; k += T) {
      z_t += exp2_fast(float(double(t_p[k]) * c - top2));
      if (first_of(k)) {
        z_x += exp2_fast((t_x[k] - m_x) * c);
        if (two) z_x1 += exp2_fast((t_x[k] - m_x) * kLog2e);
      }
    }
  }
  z_o = wave_add(z_o);
  if (two) z_o1 = wave_add(z_o1);
  if constexpr (TEACHER) {
    z_t = wave_add(z_t);
    z_x = wave_add(z_x);
    if (two) z_x1 = wave_add(z_x1);
  }
  if (lane == 0) {
    red_b[wave][0] = z_o;
    red_b[wave][1] = z_o1;
    red_b[wave][2] = z_t;
    red_b[wave][3] = z_x;
    red_b[wave][4] = z_x1;
  }
  __syncthreads();
  z_o = part_add<W>(&red_b[0][0], 5);
  if constexpr (TEACHER) {
    z_o1 = part_add<W>(&red_b[0][1], 5);
    z_t = part_add<W>(&red_b[0][2], 5);
    z_x = part_add<W>(&red_b[0][3], 5);
    z_x1 = part_add<W>(&red_b[0][4], 5);
  }
  // ---- logarithms of the row's sums (log2 units, relative to m)
  const double off_o = double(m_o) - m, off_x = double(m_x) - m;
  const double others2 = uniform(log2_of(off_o * c, z_o));  // log Z_o
  const double lse2 = uniform(TEACHER ? log2_add(others2, log2_of(off_x * c, z_x)) : others2);
  const double lse21 =
      two ? uniform(log2_add(log2_of(off_o * kLog2e, z_o1), log2_of(off_x * kLog2e, z_x1))) : lse2;
  // The teacher: its sum; its probability of the tokens it does not name; 1, or 0 for an empty teacher.
  double teach2 = 0.0;
  float r = 0.f, mass = 0.f;
  if constexpr (TEACHER) {
    z_t += exp2_fast(float(rest2 - top2));
    if (z_t != 0.f) {
      teach2 = uniform(log2_fine(z_t));
      mass = 1.f;
      r = uniform(rest2 == -__builtin_inf() ? 0.f : exp2_fast(float(rest2 - top2 - teach2)));
    }
  }
  // ---- loss
  float kl = 0.f;
  if constexpr (TEACHER) {
    for (int k = t; k < K; k += T) {
      const double lp = double(t_p[k]) * c - top2 - teach2;
      const float p = mass > 0.f && t_p[k] != kNegInf ? exp2_fast(float(lp)) : 0.f;
      t_p[k] = p;
      if (p != 0.f) kl += p * float(lp - ((double(t_x[k]) - m) * c - lse2));
    }
    kl = wave_add(kl);
    if (lane == 0) red_c[wave] = kl;
    __syncthreads();
  }
  if (t == 0) {
    double loss = 0.0;
    if (soft) {
      float s = 0.f;
      for (int w = 0; w < W; ++w) s += red_c[w];
      if (r != 0.f) s += r * float((rest2 - top2 - teach2) - (others2 - lse2));
      loss += double(1.f - a) * tau * tau * 0.6931471805599453 * s;
    }
    if (hard) {
      const float xy = R::E::get(logits_row<DT>(P.logits, row)[label]);
      loss += double(TEACHER ? a : 1.f) * 0.6931471805599453 * (lse21 - (double(xy) - m) * kLog2e);
    }
    row_loss[row] = bad ? __builtin_nanf("") : float(loss);
  }
  if (!grad) return;
  // ---- gradient: factors of the two exponentials, the tokens that are not named first
  const float w_soft = soft ? scale * (1.f - a) * tau : 0.f;
  const float w_hard = hard ? scale * (TEACHER ? a : 1.f) : 0.f;
  float f = 0.f, f1 = 0.f;
  if (soft) {
    f = mass * exp2_fast(float(off_o * c - lse2));
    if (r != 0.f && z_o > 0.f) f -= r / z_o;
    f *= w_soft;
  }
  if (hard) (two ? f1 : f) += w_hard * exp2_fast(float(off_o * (two ? kLog2e : c) - lse21));
  f = uniform(f);
  f1 = uniform(f1);
  auto other = [&](auto w, float v) -> float {
    const float e = exp2_fast((v - m_o) * c);
    float g = f * e;
    if constexpr (decltype(w)::value != kOne) g += f1 * at_one(w, v, e);
    return g;
  };
  chosen([&](auto w) {
    x.each([&](const float (&v)[N], int i0, int n) {
      float g[N];
#pragma unroll
      for (int i = 0; i < N; ++i) g[i] = other(w, v[i]);
      if (n == N)
        *reinterpret_cast<uint4 *>(grad + i0) = R::E::pack(g);
      else if (n == 1)
        grad[i0] = R::E::put(g[0]);
    });
  });
  __syncthreads();  // the tokens below are written over what the pass wrote there
  if constexpr (TEACHER) {
    for (int k = t; k < K; k += T) {
      const int id = t_idx[k];
      if (id < 0) continue;
      float p = t_p[k];
      if (dups) {  // every entry of a token writes the same value: the sum in the order of the entries
        p = 0.f;
        for (int j = 0; j < K; ++j)
          if (t_idx[j] == id) p += t_p[j];
      }
      float g = 0.f;
      if (soft) g += w_soft * (mass * exp2_fast(float((double(t_x[k]) - m) * c - lse2)) - p);
      if (hard) g += w_hard * (exp2_fast(float((double(t_x[k]) - m) * kLog2e - lse21)) - (id == label && !bad ? 1.f : 0.f));
      grad[id] = R::E::put(g);
    }
  }
  if (t == 0 && hard && !bad) {
    const int pos = x.shifted(int(label));
    const bool in_teacher = TEACHER && (bits[pos >> 5] >> (pos & 31) & 1);
    const float v = x.at(int(label));
    if (!in_teacher) grad[label] = R::E::put(chosen([&](auto w) { return other(w, v); }) - w_hard);
  }
}

// f(i) for i < n, 8 of a thread's indices at a time, so that their loads are
// in flight together (one workgroup of 1024 threads).
template <class F>
__device__ __forceinline__ void strided(int64_t n, F &&f) {
  int64_t i = threadIdx.x;
  for (; i + 7 * 1024 < n; i += 8 * 1024) {
#pragma unroll
    for (int k = 0; k < 8; ++k) f(i + k * 1024);
  }
  for (; i < n; i += 1024) f(i);
}

// One workgroup: counts the labels that are not ignored and writes
// 1 / max(count, 1).
__global__ __launch_bounds__(1024) void k_count_labels(const int64_t *labels, int64_t n, int64_t ignore, float *inv) {
  __shared__ int part[16];
  int s = 0;
  strided(n, [&](int64_t i) { s += labels[i] != ignore; });
#pragma unroll
  for (int o = 32; o >= 1; o >>= 1) s += __shfl_xor(s, o);
  if ((threadIdx.x & 63) == 0) part[threadIdx.x >> 6] = s;
  __syncthreads();
  if (threadIdx.x == 0) {
    int64_t c = 0;
    for (int w = 0; w < 16; ++w) c += part[w];
    *inv = 1.f / float(c > 0 ? c : 1);
  }
}

// One workgroup: out = factor * sum of n row losses (fp64 sums in a fixed
// order, rounded once).
__global__ __launch_bounds__(1024) void k_sum_losses(const float *loss, int64_t n, const float *factor,
                                                     float every_row, float *out) {
  __shared__ double part[16];
  double s = 0.0;
  strided(n, [&](int64_t i) { s += loss[i]; });
#pragma unroll
  for (int o = 32; o >= 1; o >>= 1) s += __shfl_xor(s, o);
  if ((threadIdx.x & 63) == 0) part[threadIdx.x >> 6] = s;
  __syncthreads();
  if (threadIdx.x == 0) {
    double c = 0.0;
    for (int w = 0; w < 16; ++w) c += part[w];
    *out = float(c * double(factor ? *factor : every_row));
  }
}

// Rows of a gradient times the upstream gradient, in place; rows whose factor
// is one are left as they are, so the usual loss.backward() reads only it.
template <int DT>
__global__ __launch_bounds__(256) void k_scale_rows(void *data, int64_t rows, int64_t inner, int64_t s_outer,
                                                    int64_t s_inner, int64_t V, const float *up, int64_t up_st) {
  using E = Elem<DT>;
  constexpr int N = E::N;
  for (int64_t r = blockIdx.x; r < rows; r += gridDim.x) {
    const float u = up[r * up_st];
    if (u == 1.f) {
      if (!up_st) return;
      continue;
    }
    typename E::raw *p = static_cast<typename E::raw *>(data) + (r / inner) * s_outer + (r % inner) * s_inner;
    const int mis = int((reinterpret_cast<uintptr_t>(p) & 15) / sizeof(*p));
    const int64_t head = mis ? (N - mis < V ? N - mis : V) : 0, nfull = (V - head) / N, tail = head + nfull * N;
    uint4 *q = reinterpret_cast<uint4 *>(p + head);
    for (int64_t i = threadIdx.x; i < nfull; i += 256) {
      float x[N];
      E::unpack(q[i], x);
#pragma unroll
      for (int e = 0; e < N; ++e) x[e] *= u;
      q[i] = E::pack(x);
    }
    const int64_t e = threadIdx.x < head ? int64_t(threadIdx.x) : tail + (int64_t(threadIdx.x) - head);
    if (e < V) {
      if (threadIdx.x < head || e >= tail) p[e] = E::put(E::get(p[e]) * u);
    }
  }
}

struct LossLaunch {
  const kvm_head_loss_desc &P;
  float every_row;
  hipStream_t stream;
  hipError_t err = hipSuccess;

  template <int DT, int T, int NV>
  void run() {
    const dim3 grid(unsigned(P.logits.outer * P.logits.inner));
    if (P.k == 0) {
      hipLaunchKernelGGL((k_head_loss<DT, T, NV, false>), grid, dim3(T), 0, stream, P, every_row);
    } else {
      const size_t words = size_t(P.logits.vocab + 2 * Elem<DT>::N + 31) / 32;
      const size_t lds = (words + 3) / 4 * 16 + size_t(P.k) * 12;
      if (lds > 64 * 1024) {
        err = hipFuncSetAttribute(reinterpret_cast<const void *>(&k_head_loss<DT, T, NV, true>),
                                  hipFuncAttributeMaxDynamicSharedMemorySize, int(lds));
        if (err != hipSuccess) return;
      }
      hipLaunchKernelGGL((k_head_loss<DT, T, NV, true>), grid, dim3(T), lds, stream, P, every_row);
    }
    err = hipGetLastError();
  }
};

}  // namespace

int64_t head_loss_max_teacher() { return kMaxTeacher; }

hipError_t launch_head_loss(const kvm_head_loss_desc &P, hipStream_t stream) {
  const int64_t rows = P.logits.outer * P.logits.inner;
  // A mean's factor: counted from the labels, or known.
  const float *counted = P.labels ? P.inv_count : nullptr;
  const float every_row = P.inv_count && !P.labels ? 1.f / float(rows) : 1.f;
  if (counted && !P.upstream)
    hipLaunchKernelGGL(k_count_labels, dim3(1), dim3(1024), 0, stream, P.labels, rows, P.ignore_index, P.inv_count);
  LossLaunch l{P, every_row, stream};
  with_row<true>(P.logits.vocab, P.logits.dtype, 256, l);
  if (l.err != hipSuccess) return l.err;
  if (P.loss)
    hipLaunchKernelGGL(k_sum_losses, dim3(1), dim3(1024), 0, stream, P.row_loss, rows, counted, every_row, P.loss);
  return hipGetLastError();
}

hipError_t launch_scale_rows(const kvm_logits &L, const float *up, int64_t up_st, hipStream_t stream) {
  const int64_t rows = L.outer * L.inner;
  const dim3 grid(unsigned(rows < 2048 ? rows : 2048));
  void *p = const_cast<void *>(L.data);
#define KVM_SCALE(D) \
  hipLaunchKernelGGL(k_scale_rows<D>, grid, dim3(256), 0, stream, p, rows, L.inner, L.s_outer, L.s_inner, L.vocab, up, up_st)
  if (L.dtype == KVM_BF16)
    KVM_SCALE(KVM_BF16);
  else if (L.dtype == KVM_F16)
    KVM_SCALE(KVM_F16);
  else
    KVM_SCALE(KVM_F32);
#undef KVM_SCALE
  return hipGetLastError();
}

}  // namespace kvm
