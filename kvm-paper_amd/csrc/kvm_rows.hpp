// Rows of logits held by one workgroup (gfx950, wave64): loading, passes over
// the values, and workgroup reductions.  Shared by the kernels that work on
// whole rows [vocab] of a decoder's logits (kvm_sample.hip, kvm_loss.hip).
//
// A row is cut into 16-byte chunks that are aligned in memory; chunk c belongs
// to thread c % T.  The up to N - 1 values before the first chunk and after the
// last one (odd vocabularies and views that start anywhere) are held one per
// lane of the first wave, so that no load touches memory outside the row.
#pragma once

#include <type_traits>

#include "kvm_device.hpp"
#include "kvm_internal.hpp"

namespace kvm {

constexpr float kLog2e = 1.4426950408889634f;
constexpr float kNegInf = -__builtin_inff();

// 16-byte chunks of the three value types <-> floats.
template <int DT>
struct Elem;
template <>
struct Elem<KVM_BF16> {
  using raw = uint16_t;
  static constexpr int N = 8;
  static __device__ __forceinline__ float get(raw b) { return bf2f(b); }
  static __device__ __forceinline__ raw put(float f) { return raw(f2bf(f)); }
  static __device__ __forceinline__ void unpack(const uint4 u, float (&x)[N]) { unpack8(u, x); }
  static __device__ __forceinline__ uint4 pack(const float (&x)[N]) { return pack8(x); }
};
template <>
struct Elem<KVM_F16> {
  using raw = uint16_t;
  typedef _Float16 h8 __attribute__((ext_vector_type(8)));
  static constexpr int N = 8;
  static __device__ __forceinline__ float get(raw b) { return float(__builtin_bit_cast(_Float16, b)); }
  static __device__ __forceinline__ raw put(float f) { return __builtin_bit_cast(raw, _Float16(f)); }
  static __device__ __forceinline__ void unpack(const uint4 u, float (&x)[N]) {
    const h8 h = __builtin_bit_cast(h8, u);
#pragma unroll
    for (int i = 0; i < N; ++i) x[i] = float(h[i]);
  }
  static __device__ __forceinline__ uint4 pack(const float (&x)[N]) {
    h8 h;
#pragma unroll
    for (int i = 0; i < N; ++i) h[i] = _Float16(x[i]);
    return __builtin_bit_cast(uint4, h);
  }
};
template <>
struct Elem<KVM_F32> {
  using raw = float;
  static constexpr int N = 4;
  static __device__ __forceinline__ float get(raw b) { return b; }
  static __device__ __forceinline__ raw put(float f) { return f; }
  static __device__ __forceinline__ void unpack(const uint4 u, float (&x)[N]) {
    x[0] = __uint_as_float(u.x);
    x[1] = __uint_as_float(u.y);
    x[2] = __uint_as_float(u.z);
    x[3] = __uint_as_float(u.w);
  }
  static __device__ __forceinline__ uint4 pack(const float (&x)[N]) {
    return make_uint4(__float_as_uint(x[0]), __float_as_uint(x[1]), __float_as_uint(x[2]), __float_as_uint(x[3]));
  }
};

// First value of row r of a logits descriptor.
template <int DT>
__device__ __forceinline__ const typename Elem<DT>::raw *logits_row(const kvm_logits &L, int r) {
  const int o = r / int(L.inner), i = r - o * int(L.inner);
  return static_cast<const typename Elem<DT>::raw *>(L.data) + o * L.s_outer + i * L.s_inner;
}

// Sum / maximum over a wave, the same value in every lane (fixed order).
__device__ __forceinline__ float lane_of(float v, int l) {
  return __builtin_bit_cast(float, __builtin_amdgcn_readlane(__builtin_bit_cast(int, v), l));
}
__device__ __forceinline__ float wave_add(float v) {
  v = group_sum<16>(v);
  return (lane_of(v, 0) + lane_of(v, 16)) + (lane_of(v, 32) + lane_of(v, 48));
}
__device__ __forceinline__ float wave_max(float v) {
  v = fmaxf(v, dpp<kDppRowRor8>(v));
  v = fmaxf(v, dpp<kDppRowRor4>(v));
  v = fmaxf(v, dpp<kDppQuadXor2>(v));
  v = fmaxf(v, dpp<kDppQuadXor1>(v));
  return fmaxf(fmaxf(lane_of(v, 0), lane_of(v, 16)), fmaxf(lane_of(v, 32), lane_of(v, 48)));
}

// Minimum / maximum of unsigned numbers over a wave, in every lane.
template <int CTRL>
__device__ __forceinline__ uint32_t dpp_u(uint32_t v) {
  return uint32_t(__builtin_amdgcn_update_dpp(0, int(v), CTRL, 0xf, 0xf, false));
}
__device__ __forceinline__ uint32_t lane_of(uint32_t v, int l) { return uint32_t(__builtin_amdgcn_readlane(int(v), l)); }
__device__ __forceinline__ uint32_t wave_min_u(uint32_t v) {
  v = min(v, dpp_u<kDppRowRor8>(v));
  v = min(v, dpp_u<kDppRowRor4>(v));
  v = min(v, dpp_u<kDppQuadXor2>(v));
  v = min(v, dpp_u<kDppQuadXor1>(v));
  return min(min(lane_of(v, 0), lane_of(v, 16)), min(lane_of(v, 32), lane_of(v, 48)));
}
__device__ __forceinline__ uint32_t wave_max_u(uint32_t v) { return ~wave_min_u(~v); }

// The same over the W <= 16 partial results of a workgroup's waves, part[0],
// part[stride], ...: one LDS read per lane, the same value in every lane.
template <int W>
__device__ __forceinline__ float part_add(const float *part, int stride = 1) {
  const int l = threadIdx.x & 15;
  return group_sum<16>(l < W ? part[l * stride] : 0.f);
}
template <int W>
__device__ __forceinline__ float part_max(const float *part, int stride = 1) {
  const int l = threadIdx.x & 15;
  float v = l < W ? part[l * stride] : kNegInf;
  v = fmaxf(v, dpp<kDppRowRor8>(v));
  v = fmaxf(v, dpp<kDppRowRor4>(v));
  v = fmaxf(v, dpp<kDppQuadXor2>(v));
  return fmaxf(v, dpp<kDppQuadXor1>(v));
}

// A row of V values in the registers of a workgroup of T threads, NV chunks
// per thread (NV = 0: read again on every pass; for rows that do not fit).
template <int DT, int T, int NV, bool FRESH = false>
struct Row {
  using E = Elem<DT>;
  using raw = typename E::raw;
  static constexpr int N = E::N;
  static constexpr bool kResident = NV > 0;

  uint4 v[NV > 0 ? NV : 1];
  const raw *first;  // of the row
  const uint4 *chunks;
  int head, nfull, edges;  // values before the first chunk, whole chunks, values outside them
  int edge_idx;            // this lane's value outside the chunks (-1: none)
  float edge;

  // Chunk j as it is in the registers.  FRESH: the compiler may not know that it
  // is the value of an earlier pass, where it would keep the floats unpacked
  // there, at two registers for every one that holds the row, and spill.
  __device__ __forceinline__ uint4 held(int j) const {
    uint4 u = v[j];
    if constexpr (FRESH) asm volatile("" : "+v"(u.x), "+v"(u.y), "+v"(u.z), "+v"(u.w));
    return u;
  }

  __device__ __forceinline__ uint4 fetch(int c) const {
    const uint4 u = chunks[min(c, nfull - 1)];
    return u;
  }
  static __device__ __forceinline__ uint4 empty() {
    float x[N];
#pragma unroll
    for (int i = 0; i < N; ++i) x[i] = kNegInf;
    return E::pack(x);
  }

  __device__ __forceinline__ void open(const raw *row, int V) {
    const int t = threadIdx.x;
    const int mis = int((reinterpret_cast<uintptr_t>(row) & 15) / sizeof(raw));
    first = row;
    head = mis ? min(N - mis, V) : 0;
    nfull = (V - head) / N;
    edges = V - nfull * N;
    chunks = reinterpret_cast<const uint4 *>(row + head);
    if constexpr (NV > 0) {
      if (nfull > 0) {
#pragma unroll
        for (int j = 0; j < NV; ++j) v[j] = fetch(j * T + t);
      }
#pragma unroll
      for (int j = 0; j < NV; ++j)
        if (j * T + t >= nfull) v[j] = empty();
    }
    edge_idx = t < head ? t : head + nfull * N + (t - head);
    if (t >= edges) edge_idx = -1;
    edge = edge_idx >= 0 ? E::get(row[edge_idx]) : kNegInf;
  }

  // Value idx of the row, from memory.
  __device__ __forceinline__ float at(int idx) const { return E::get(first[idx]); }

  // Position of value idx in an array that is laid out as the chunks are:
  // the first value of every chunk lies at a multiple of N.
  __device__ __forceinline__ int shifted(int idx) const { return idx + (head ? N - head : 0); }

  // Replaces the values that f(first, n) names (bit i: value first + i) by
  // -infinity, in the registers; rows that are read again keep them.
  template <class F>
  __device__ __forceinline__ void hide(F &&f) {
    const int t = threadIdx.x;
    if constexpr (NV > 0) {
#pragma unroll
      for (int j = 0; j < NV; ++j) {
        if (j * T < nfull) {
          const int c = j * T + t;
          const uint32_t bits = c < nfull ? f(head + c * N, N) : 0;
          if (bits & ((1u << N) - 1)) {
            float x[N];
            E::unpack(held(j), x);
#pragma unroll
            for (int i = 0; i < N; ++i) x[i] = bits >> i & 1 ? kNegInf : x[i];
            v[j] = E::pack(x);
          }
        }
      }
      if (edge_idx >= 0 && (f(edge_idx, 1) & 1)) edge = kNegInf;
    }
  }

  // The largest value of each of this thread's chunks, and of all it holds (a
  // NaN is passed over).
  __device__ __forceinline__ float maxima(float (&most)[NV > 0 ? NV : 1]) const {
    float m = edge;
#pragma unroll
    for (int j = 0; j < NV; ++j) {
      most[j] = kNegInf;
      if (j * T < nfull) {
        float x[N];
        E::unpack(held(j), x);
#pragma unroll
        for (int i = 0; i < N; ++i) most[j] = fmaxf(most[j], x[i]);
        m = fmaxf(m, most[j]);
      }
    }
    return m;
  }

  // f(x, first, n) for the chunks (and values outside them) whose maxima are
  // >= least, or for all of them.  TAKE: they become -infinity.
  template <bool TAKE, class F>
  __device__ __forceinline__ void above(const float (&most)[NV > 0 ? NV : 1], float least, bool all, F &&f) {
    const int t = threadIdx.x;
#pragma unroll
    for (int j = 0; j < NV; ++j) {
      const int c = j * T + t;
      if ((most[j] >= least || all) && c < nfull) {
        float x[N];
        E::unpack(held(j), x);
        f(x, head + c * N, N);
        if constexpr (TAKE) v[j] = empty();
      }
    }
    if (edge_idx >= 0 && (edge >= least || all)) {
      float x[N];
#pragma unroll
      for (int i = 0; i < N; ++i) x[i] = kNegInf;
      x[0] = edge;
      f(x, edge_idx, 1);
      if constexpr (TAKE) edge = kNegInf;
    }
  }

  // f(x, first, n): n values x[0..n) with indices first, first + 1, ...  n is
  // N, or 1 (a value outside the chunks), or 0 (none); the values past n are
  // -infinity.  Chunks that no lane of the workgroup has are skipped.  A row
  // that is read again is read BATCH chunks per thread at a time, one batch
  // ahead of f, whose code is there BATCH times.
  template <int BATCH = 4, class F>
  __device__ __forceinline__ void each(F &&f) const {
    const int t = threadIdx.x;
    if constexpr (NV > 0) {
#pragma unroll
      for (int j = 0; j < NV; ++j) {
        if (j * T < nfull) {
          float x[N];
          E::unpack(held(j), x);
          const int c = j * T + t;
          f(x, head + c * N, c < nfull ? N : 0);
        }
      }
    } else {
      uint4 next[BATCH];
      if (nfull > 0) {
#pragma unroll
        for (int i = 0; i < BATCH; ++i) next[i] = fetch(t + i * T);
      }
#pragma unroll 1
      for (int b = 0; b < nfull; b += T * BATCH) {  // chunks of the batch: b, b + 1, ...
        uint4 u[BATCH];
#pragma unroll
        for (int i = 0; i < BATCH; ++i) {
          u[i] = next[i];
          next[i] = fetch(b + T * (BATCH + i) + t);
        }
#pragma unroll
        for (int i = 0; i < BATCH; ++i) {
          const int c = b + i * T + t;
          if (b + i * T < nfull) {
            float x[N];
            E::unpack(c < nfull ? u[i] : empty(), x);
            f(x, head + c * N, c < nfull ? N : 0);
          }
        }
      }
    }
    if (edges && t < kWave) {
      float x[N];
#pragma unroll
      for (int i = 0; i < N; ++i) x[i] = kNegInf;
      x[0] = edge;
      f(x, edge_idx, edge_idx >= 0 ? 1 : 0);
    }
  }

  // f(x, first, n) as above for those with which(x, true), few of the row (x is
  // of no chunk, and the answer not used, where false is passed).  A row that is read again: a pass finds
  // them, 32 chunks per thread, and the lanes then take theirs side by side,
  // where one by one they would hold up the pass (locating a bin of 142 tokens
  // among 50257 fp32 logits, one workgroup: 7.0 us, so 4.4).
  template <class W, class F>
  __device__ __forceinline__ void where(W &&which, F &&f) const {
    static_assert(NV == 0, "rows in registers have above()");
    constexpr int BATCH = 4;
    const int t = threadIdx.x;
#pragma unroll 1
    for (int b0 = 0; b0 < nfull; b0 += 32 * T) {
      uint32_t found = 0;
      uint4 next[BATCH];
#pragma unroll
      for (int i = 0; i < BATCH; ++i) next[i] = fetch(b0 + t + i * T);
#pragma unroll 1
      for (int j = 0; j < 32 && b0 + j * T < nfull; j += BATCH) {
        uint4 u[BATCH];
#pragma unroll
        for (int i = 0; i < BATCH; ++i) {
          u[i] = next[i];
          next[i] = fetch(b0 + T * (j + BATCH + i) + t);
        }
#pragma unroll
        for (int i = 0; i < BATCH; ++i) {
          const bool there = b0 + (j + i) * T + t < nfull;
          float x[N];
          E::unpack(u[i], x);
          found |= which(x, there) && there ? 1u << (j + i) : 0u;
        }
      }
      while (found) {
        const int c = b0 + (__ffs(found) - 1) * T + t;
        found &= found - 1;
        float x[N];
        E::unpack(chunks[c], x);
        f(x, head + c * N, N);
      }
    }
    if (edge_idx >= 0) {
      float x[N];
#pragma unroll
      for (int i = 0; i < N; ++i) x[i] = kNegInf;
      x[0] = edge;
      if (which(x, true)) f(x, edge_idx, 1);
    }
  }
};

// What a launch takes for rows of a type and length: threads per workgroup,
// and whether the row stays in registers.  16 chunks per thread are 64
// registers, which leaves two workgroups of 512 threads (or one of 1024) per
// compute unit; longer rows are read again on every pass, from the caches.
constexpr int kRowChunks = 16;
inline int row_threads(int64_t vocab, int64_t dtype, int64_t at_least = 256) {
  const int64_t n = dtype == KVM_F32 ? 4 : 8;
  int64_t t = 256;
  while (t < 1024 && (t < at_least || t * kRowChunks * n < vocab)) t *= 2;
  return int(t);
}
inline bool row_resident(int64_t vocab, int64_t dtype) {
  return vocab <= int64_t(1024) * kRowChunks * (dtype == KVM_F32 ? 4 : 8);
}

// Calls f.run<DT, T, NV>() for a row's type and length; RESIDENT false: for a
// row that is read again whatever its length.
template <bool RESIDENT, class F>
void with_row(int64_t vocab, int64_t dtype, int64_t at_least, F &&f) {
  auto typed = [&](auto dt) {
    constexpr int DT = decltype(dt)::value;
    if constexpr (RESIDENT) {
      const int t = row_threads(vocab, dtype, at_least);
      if (row_resident(vocab, dtype)) {
        if (t == 256)
          f.template run<DT, 256, kRowChunks>();
        else if (t == 512)
          f.template run<DT, 512, kRowChunks>();
        else
          f.template run<DT, 1024, kRowChunks>();
        return;
      }
    }
    f.template run<DT, 1024, 0>();
  };
  if (dtype == KVM_BF16)
    typed(std::integral_constant<int, KVM_BF16>{});
  else if (dtype == KVM_F16)
    typed(std::integral_constant<int, KVM_F16>{});
  else
    typed(std::integral_constant<int, KVM_F32>{});
}

}  // namespace kvm
