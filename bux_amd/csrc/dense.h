// The dense products' epilogues, shared by every kernel that forms sums of x w: 8 consecutive
// columns of a row at a time, in float32, rounded once to the rows' type.
//
//   Forward   z = v + bias (kept as `product`, if asked for);  out = act(z) + residual, where a
//             gated act takes the columns as (up, gate) pairs and gives half as many
//   Backward  v is the gradient dh of the activation's output: dp = dh d act(product)
//   Partial   v as it is, to a split's own place in the workspace
//
// act runs in float32 on the sums themselves, before their rounding: `product` is rounded only
// to be kept, so that the outputs do not depend on whether it is.
#pragma once

#include <type_traits>

#include "glu.h"

namespace bux {
namespace {

typedef float f32x16 __attribute__((ext_vector_type(16)));

constexpr int NO_ACT = -1;  // Act::kind of a product without an activation

// 8 elements as they lie, at an element's alignment.
template <typename T>
struct Eight {
  struct __attribute__((packed, aligned(sizeof(T)))) Bytes {
    T at[8];
  };
  Bytes b;
  __device__ __forceinline__ float value(int j) const { return Elem<T>::value(b.at[j]); }
};
// The first `count` (8 or more: all) of 8 elements from p on, zeros for the rest.
template <typename T>
__device__ __forceinline__ Eight<T> load_eight(const T* p, int64_t count) {
  Eight<T> r{};
  if (count >= 8) {
    r.b = *reinterpret_cast<const typename Eight<T>::Bytes*>(p);
  } else {
#pragma unroll
    for (int j = 0; j < 8; ++j)
      if (j < count) r.b.at[j] = p[j];
  }
  return r;
}
template <typename T, int N = 8>
__device__ __forceinline__ void store_some(T* p, const float* v, int64_t count) {
  struct __attribute__((packed, aligned(sizeof(T)))) Some {
    T at[N];
  };
  Some s;
#pragma unroll
  for (int j = 0; j < N; ++j) s.at[j] = Elem<T>::make(v[j]);
  if (count >= N) {
    *reinterpret_cast<Some*>(p) = s;
  } else {
#pragma unroll
    for (int j = 0; j < N; ++j)
      if (j < count) p[j] = s.at[j];
  }
}

struct NoAct {};
// Calls f(Kind<kind, GATED>{}), or f(NoAct{}) for none: a branch that every lane takes alike.
template <bool GATED, typename F>
__device__ __forceinline__ void of_kind(int kind, F&& f) {
  switch (kind) {
    case BUX_SWISH: f(Kind<BUX_SWISH, GATED>{}); break;
    case BUX_QUICK_GELU: f(Kind<BUX_QUICK_GELU, GATED>{}); break;
    case BUX_RELU: f(Kind<BUX_RELU, GATED>{}); break;
    case BUX_RELU2: f(Kind<BUX_RELU2, GATED>{}); break;
    case BUX_GELU: f(Kind<BUX_GELU, GATED>{}); break;
    case BUX_GELU_TANH: f(Kind<BUX_GELU_TANH, GATED>{}); break;
    case BUX_SIGMOID: f(Kind<BUX_SIGMOID, GATED>{}); break;
    case BUX_TANH: f(Kind<BUX_TANH, GATED>{}); break;
    case BUX_SOFTPLUS: f(Kind<BUX_SOFTPLUS, GATED>{}); break;
    case BUX_SITU: f(Kind<BUX_SITU, GATED>{}); break;
    default:
      if constexpr (!GATED) f(NoAct{});
  }
}

// An epilogue E: In, what a row's 8 columns need beside their sums; load(row, col) of it;
// choose(f), which calls f with the activation's kind; store(kind, row, col, v, in).

template <typename T, bool GATED>
struct Forward {
  static constexpr bool F32 = sizeof(T) == 4;
  Act act;  // kind NO_ACT: none
  const T* bias;
  const T* residual;  // (a gated act has none)
  T* product;
  T* out;
  int64_t n;  // columns of the sums

  struct In {
    Eight<T> residual;
  };
  __device__ __forceinline__ In load(int64_t row, int64_t col) const {
    In in{};
    if (!GATED && residual) in.residual = load_eight(residual + row * n + col, n - col);
    return in;
  }
  template <typename F>
  __device__ __forceinline__ void choose(F&& f) const {
    of_kind<GATED>(act.kind, f);
  }
  template <typename K>
  __device__ __forceinline__ void store(K, int64_t row, int64_t col, const float v[8],
                                        const In& in) const {
    const int64_t count = n - col;
    float z[8];
#pragma unroll
    for (int j = 0; j < 8; ++j) z[j] = v[j];
    if (bias) {
      const Eight<T> b = load_eight(bias + col, count);
#pragma unroll
      for (int j = 0; j < 8; ++j) z[j] += b.value(j);
    }
    if (product) store_some<T>(product + row * n + col, z, count);
    if constexpr (GATED) {
      float h[4];
#pragma unroll
      for (int j = 0; j < 4; ++j) h[j] = glu_unit<K, F32>(act, z[2 * j], z[2 * j + 1], 1.0f);
      store_some<T, 4>(out + row * (n / 2) + col / 2, h, count / 2);
    } else {
      if constexpr (!std::is_same<K, NoAct>::value) {
#pragma unroll
        for (int j = 0; j < 8; ++j) z[j] = glu_unit<K, F32>(act, z[j], 0.0f, 1.0f);
      }
      if (residual) {
#pragma unroll
        for (int j = 0; j < 8; ++j) z[j] += in.residual.value(j);
      }
      store_some<T>(out + row * n + col, z, count);
    }
  }
};

template <typename T, bool GATED>
struct Backward {
  static constexpr bool F32 = sizeof(T) == 4;
  static constexpr int P = GATED ? 2 : 1;
  Act act;
  const T* product;  // [m, n, P]
  T* out;            // the same
  int64_t n;         // units

  struct In {
    Eight<T> p[P];
  };
  __device__ __forceinline__ In load(int64_t row, int64_t col) const {
    In in{};
#pragma unroll
    for (int i = 0; i < P; ++i)
      in.p[i] = load_eight(product + (row * n + col) * P + 8 * i, (n - col) * P - 8 * i);
    return in;
  }
  template <typename F>
  __device__ __forceinline__ void choose(F&& f) const {
    of_kind<GATED>(act.kind, f);
  }
  template <typename K>
  __device__ __forceinline__ void store(K, int64_t row, int64_t col, const float v[8],
                                        const In& in) const {
    float d[8 * P];
    if constexpr (std::is_same<K, NoAct>::value) {
#pragma unroll
      for (int j = 0; j < 8; ++j) d[j] = v[j];
    } else {
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        float du, dg, dw;
        const float up = in.p[j * P / 8].value(j * P % 8);
        const float gate = GATED ? in.p[j * P / 8].value(j * P % 8 + 1) : 0.0f;
        glu_unit_grad<K, F32>(act, up, gate, 1.0f, v[j], &du, &dg, &dw);
        d[j * P] = du;
        if (GATED) d[j * P + 1] = dg;
      }
    }
#pragma unroll
    for (int i = 0; i < P; ++i)
      store_some<T>(out + (row * n + col) * P + 8 * i, d + 8 * i, (n - col) * P - 8 * i);
  }
};

// The workspace's rows are whole 8s of columns, `pitch`.
struct Partial {
  float* out;
  int64_t pitch;
  struct In {};
  __device__ __forceinline__ In load(int64_t, int64_t) const { return In{}; }
  template <typename F>
  __device__ __forceinline__ void choose(F&& f) const {
    f(NoAct{});
  }
  template <typename K>
  __device__ __forceinline__ void store(K, int64_t row, int64_t col, const float v[8],
                                        const In&) const {
    float4* const p = reinterpret_cast<float4*>(out + row * pitch + col);
    p[0] = make_float4(v[0], v[1], v[2], v[3]);
    p[1] = make_float4(v[4], v[5], v[6], v[7]);
  }
};

// --- from MFMA sums to rows of 8 columns ---------------------------------------------------
//
// v_mfma_f32_32x32 of (B's block, A's block) leaves lane l with row l % 32 of A's and columns
// 8 g + 4 (l / 32) .. + 3 of B's in registers 4 g .. 4 g + 3. A wave turns 32 rows x 64 columns
// around through 8 KiB of LDS of its own: 256 bytes a row, 16-byte chunk c of row r at place
// c ^ (r % 16), so that the 16 lanes of a phase write 16 places; then lane l takes columns
// 8 (l % 8) of rows l / 8 + 8 it: whole lines of the output, 8 rows an instruction.

constexpr int UNIT_BYTES = 32 * 256;

__device__ __forceinline__ void wave_done_lds() {
  asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
  __builtin_amdgcn_wave_barrier();
}

__device__ __forceinline__ void put_unit(uint8_t* region, const f32x16& c0, const f32x16& c1) {
  const int lane = threadIdx.x & 63, r = lane & 31, h = lane >> 5;
  uint8_t* const mine = region + r * 256;
#pragma unroll
  for (int q = 0; q < 2; ++q) {
    const f32x16& a = q ? c1 : c0;
#pragma unroll
    for (int g = 0; g < 4; ++g)
      *reinterpret_cast<float4*>(mine + 16 * ((8 * q + 2 * g + h) ^ (r & 15))) =
          make_float4(a[4 * g], a[4 * g + 1], a[4 * g + 2], a[4 * g + 3]);
  }
}
__device__ __forceinline__ void get_row(const uint8_t* region, int it, float v[8]) {
  const int lane = threadIdx.x & 63, r = (lane >> 3) + 8 * it, c = 2 * (lane & 7);
  const float4 x = *reinterpret_cast<const float4*>(region + r * 256 + 16 * (c ^ (r & 15)));
  const float4 y = *reinterpret_cast<const float4*>(region + r * 256 + 16 * ((c + 1) ^ (r & 15)));
  v[0] = x.x; v[1] = x.y; v[2] = x.z; v[3] = x.w;
  v[4] = y.x; v[5] = y.y; v[6] = y.z; v[7] = y.w;
}

// A unit's 32 rows from row0 and 64 columns from col0 (those below m and n), put in `region`
// before, through `epi`.
template <typename Epi>
__device__ __forceinline__ void store_unit(const Epi& epi, const uint8_t* region, int64_t row0,
                                           int64_t col0, int64_t m, int64_t n) {
  const int lane = threadIdx.x & 63;
  const int64_t row = row0 + (lane >> 3), col = col0 + 8 * (lane & 7);
  typename Epi::In in[4];
#pragma unroll
  for (int it = 0; it < 4; ++it) {
    in[it] = typename Epi::In{};
    if (row + 8 * it < m && col < n) in[it] = epi.load(row + 8 * it, col);
  }
  epi.choose([&](auto kind) {
#pragma unroll
    for (int it = 0; it < 4; ++it) {
      float v[8];
      get_row(region, it, v);
      if (row + 8 * it < m && col < n) epi.store(kind, row + 8 * it, col, v, in[it]);
    }
  });
}

}  // namespace
}  // namespace bux
