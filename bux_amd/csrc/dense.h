// The dense products' epilogues, shared by every kernel that forms sums of x w: 8 consecutive
// columns of a row at a time, in float32, rounded once to the rows' type.
//
//   Forward   z = v + bias (kept as `product`, if asked for);  out = act(z) + residual, where a
//             gated act takes the columns as (up, gate) pairs and gives half as many
//   Backward  v is the gradient dh of the activation's output: dp = dh d act(product)
//             (bfloat16: from 24 bits of each value, where its low bytes were kept too)
//   Partial   v as it is, to a split's own place in the workspace
//
// act runs in float32 on the sums themselves, before their rounding: `product` is rounded only
// to be kept, so that the outputs do not depend on whether it is.
#pragma once

#include <type_traits>

#include "glu.h"

namespace bux {
namespace dense {

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
  if constexpr (sizeof(T) == 2) {
#pragma unroll
    for (int j = 0; j < N; j += 2) {
      const uint32_t w = pack_bf16x2(v[j], v[j + 1]);
      s.at[j] = static_cast<T>(w & 0xffffu);
      s.at[j + 1] = static_cast<T>(w >> 16);
    }
  } else {
#pragma unroll
    for (int j = 0; j < N; ++j) s.at[j] = Elem<T>::make(v[j]);
  }
  if (count >= N) {
    *reinterpret_cast<Some*>(p) = s;
  } else {
#pragma unroll
    for (int j = 0; j < N; ++j)
      if (j < count) p[j] = s.at[j];
  }
}

// --- a bfloat16 value's next 8 bits ---------------------------------------------------------
//
// z kept as bfloat16 alone would put a rounding of up to 2^-8 of it into the activation's gradient
// beside the one that d product takes to be multiplied: of a block's gradients to x and up sqrt 3
// rather than sqrt 2 of their outputs' own. A signed byte beside it, the difference of the float32's
// bits from the bfloat16's in units of 2^8, keeps 16 bits of mantissa, at half the bytes that float32
// would add. (A value that bfloat16 rounds to infinity comes back finite, but for the 128 next to
// float32's infinity; a NaN stays one.)

__device__ __forceinline__ uint32_t low_byte(float z, uint32_t high) {
  const int32_t off = static_cast<int32_t>(__float_as_uint(z)) - static_cast<int32_t>(high << 16);
  const int32_t b = (off + 128) >> 8;
  return static_cast<uint32_t>(b < -128 ? -128 : b > 127 ? 127 : b) & 0xffu;
}
// 8 values' low bytes, the first lowest; `high`: their bfloat16s, in pairs.
__device__ __forceinline__ uint64_t low_bytes(const float v[8], const uint32_t high[4]) {
  uint32_t w[2] = {0, 0};
#pragma unroll
  for (int j = 0; j < 8; ++j)
    w[j / 4] |= low_byte(v[j], j & 1 ? high[j / 2] >> 16 : high[j / 2] & 0xffffu) << (8 * (j % 4));
  return static_cast<uint64_t>(w[1]) << 32 | w[0];
}
__device__ __forceinline__ float with_low(float z, uint64_t low, int j) {
  const uint32_t w = static_cast<uint32_t>(j < 4 ? low : low >> 32);
  const int32_t b = static_cast<int32_t>(w << (24 - 8 * (j & 3))) >> 24;
  return __uint_as_float(__float_as_uint(z) + (static_cast<uint32_t>(b) << 8));
}
__device__ __forceinline__ uint64_t load_low(const uint8_t* p, int64_t count) {
  uint64_t v = 0;
  if (count >= 8) {
    __builtin_memcpy(&v, p, 8);
  } else {
#pragma unroll
    for (int j = 0; j < 8; ++j)
      if (j < count) v |= static_cast<uint64_t>(p[j]) << (8 * j);
  }
  return v;
}
__device__ __forceinline__ void store_low(uint8_t* p, uint64_t v, int64_t count) {
  if (count >= 8) {
    __builtin_memcpy(p, &v, 8);
  } else {
#pragma unroll
    for (int j = 0; j < 8; ++j)
      if (j < count) p[j] = static_cast<uint8_t>(v >> (8 * j));
  }
}

struct NoAct {};
// An activation's kind, and whether its up branch is neither clipped nor capped: known where it
// runs, so that the units a lane makes at once have no branches between them.
template <int KIND, bool GATED, bool BARE>
struct Choice {
  using K = Kind<KIND, GATED>;
  static __device__ __forceinline__ Act of(const Act& act) {
    Act a = act;
    if (BARE) a.clamped = a.capped = 0;
    return a;
  }
};
// Calls f(Choice<kind, GATED, ..>{}), or f(NoAct{}) for none: a branch that every lane takes alike.
template <bool GATED, bool BARE, typename F>
__device__ __forceinline__ void of_kind(int kind, F&& f) {
  switch (kind) {
    case BUX_SWISH: f(Choice<BUX_SWISH, GATED, BARE>{}); break;
    case BUX_QUICK_GELU: f(Choice<BUX_QUICK_GELU, GATED, BARE>{}); break;
    case BUX_RELU: f(Choice<BUX_RELU, GATED, BARE>{}); break;
    case BUX_RELU2: f(Choice<BUX_RELU2, GATED, BARE>{}); break;
    case BUX_GELU: f(Choice<BUX_GELU, GATED, BARE>{}); break;
    case BUX_GELU_TANH: f(Choice<BUX_GELU_TANH, GATED, BARE>{}); break;
    case BUX_SIGMOID: f(Choice<BUX_SIGMOID, GATED, BARE>{}); break;
    case BUX_TANH: f(Choice<BUX_TANH, GATED, BARE>{}); break;
    case BUX_SOFTPLUS: f(Choice<BUX_SOFTPLUS, GATED, BARE>{}); break;
    case BUX_SITU: f(Choice<BUX_SITU, GATED, BARE>{}); break;
    default:
      if constexpr (!GATED && BARE) f(NoAct{});
  }
}
template <bool GATED, typename F>
__device__ __forceinline__ void of_act(const Act& act, F&& f) {
  if (act.clamped || act.capped) of_kind<GATED, false>(act.kind, f);
  else of_kind<GATED, true>(act.kind, f);
}
template <typename C, bool F32>
__device__ __forceinline__ float unit_of(const Act& act, float up, float gate) {
  return glu_unit<typename C::K, F32>(C::of(act), up, gate, 1.0f);
}
template <typename C, bool F32>
__device__ __forceinline__ void unit_grad_of(const Act& act, float up, float gate, float dh,
                                             float* d_up, float* d_gate) {
  float dw;
  glu_unit_grad<typename C::K, F32>(C::of(act), up, gate, 1.0f, dh, d_up, d_gate, &dw);
}

// --- whole tiles ---------------------------------------------------------------------------
//
// A tile that lies inside outputs of whole, aligned 16 bytes moves its values at 32-bit offsets
// from its corner, without a check a chunk: a lane's own offset (row l / 8, columns 8 (l % 8) of a
// unit, below) and a scalar one. Where 8 columns are 32 bytes (HALVES) a lane takes columns 4 (l % 8)
// of the unit's two halves instead, so that 8 lanes store 128 bytes in a row. (Stores of every other
// 16 bytes, past the caches, took 184 of the 627 us of the gated block's gradient of 16384 x 8192
// units.) Stores are non-temporal: another kernel reads them, and they would
// push the operands out of L2.

typedef uint32_t words4 __attribute__((ext_vector_type(4)));
typedef uint32_t words2 __attribute__((ext_vector_type(2)));
constexpr int NON_TEMPORAL = 2;

struct Place {
  __amdgpu_buffer_rsrc_t rsrc;
  int32_t lane;   // bytes
  int32_t pitch;  // bytes a row
};
// `COLUMNS` elements to 8 columns of sums (8, 4 of a gated act's units, 16 of its pairs).
template <int COLUMNS>
__device__ __forceinline__ Place place_in(const uint16_t* p, int64_t row, int64_t col, int64_t n) {
  const int lane = threadIdx.x & 63;
  const int64_t ld = n * COLUMNS / 8;
  Place r;
  r.rsrc = __builtin_amdgcn_make_buffer_rsrc(
      const_cast<uint16_t*>(p) + row * ld + col * COLUMNS / 8, 0, 0x7fffffff, 0x00020000);
  r.pitch = static_cast<int32_t>(ld) * 2;
  r.lane = (lane >> 3) * r.pitch + (lane & 7) * (COLUMNS == 16 ? 16 : COLUMNS * 2);
  return r;
}
constexpr int HALF = 128;  // bytes from a lane's first 16 to its second, where COLUMNS is 16
// As many bytes, one an element, of COLUMNS (8 or 16) elements.
template <int COLUMNS>
__device__ __forceinline__ Place bytes_in(const uint8_t* p, int64_t row, int64_t col, int64_t n) {
  const int lane = threadIdx.x & 63;
  const int64_t ld = n * COLUMNS / 8;
  Place r;
  r.rsrc = __builtin_amdgcn_make_buffer_rsrc(
      const_cast<uint8_t*>(p) + row * ld + col * COLUMNS / 8, 0, 0x7fffffff, 0x00020000);
  r.pitch = static_cast<int32_t>(ld);
  r.lane = (lane >> 3) * r.pitch + (lane & 7) * 8;
  return r;
}
template <int COLUMNS>
__device__ __forceinline__ int32_t scalar_in(const Place& p, int row, int col) {
  return row * p.pitch + col * COLUMNS / 8 * 2;
}
__device__ __forceinline__ words4 packed8(const float* v) {
  return words4{pack_bf16x2(v[0], v[1]), pack_bf16x2(v[2], v[3]), pack_bf16x2(v[4], v[5]),
                pack_bf16x2(v[6], v[7])};
}
__device__ __forceinline__ float half_of(words4 w, int j) {
  const uint32_t x = w[j >> 1];
  return __uint_as_float(j & 1 ? x & 0xffff0000u : x << 16);
}
// Whether every row of `columns` bfloat16 from p on begins at 16 bytes.
__device__ __forceinline__ bool aligned16(const void* p, int64_t columns) {
  return reinterpret_cast<uintptr_t>(p) % 16 == 0 && columns % 8 == 0;
}

// An epilogue E: In, what a row's 8 columns need beside their sums; load(row, col) of it;
// choose(f), which calls f with the activation's kind; store(kind, row, col, v, in).

template <typename T, bool GATED>
struct Forward {
  static constexpr bool HALVES = false;
  static constexpr bool F32 = sizeof(T) == 4;
  Act act;  // kind NO_ACT: none
  const T* bias;
  const T* residual;  // (a gated act has none)
  T* product;
  uint8_t* low;  // product's low bytes (bfloat16)
  T* out;
  int64_t n;  // columns of the sums

  struct Tile {
    Place out, product, low, residual;
    words4 bias[2];  // of a wave's two units of 64 columns
  };
  struct Fast {
    words4 residual;
  };
  // Whether tiles inside the output take the path above.
  __device__ __forceinline__ bool aligned() const {
    return aligned16(out, GATED ? n / 2 : n) && n % 8 == 0 && n < (1 << 20) &&
           (product == nullptr || aligned16(product, n)) &&
           (low == nullptr || reinterpret_cast<uintptr_t>(low) % 8 == 0) &&
           (residual == nullptr || aligned16(residual, n)) &&
           (bias == nullptr || aligned16(bias, n));
  }
  __device__ __forceinline__ Tile tile(int64_t row, int64_t col) const {
    Tile t;
    t.out = place_in<GATED ? 4 : 8>(out, row, col, n);
    t.product = place_in<8>(product, row, col, n);
    t.low = bytes_in<8>(low, row, col, n);
    t.residual = place_in<8>(residual, row, col, n);
    const int c = 8 * (threadIdx.x & 7);
    if (bias) {
#pragma unroll
      for (int u = 0; u < 2; ++u)
        t.bias[u] = *reinterpret_cast<const words4*>(bias + col + 64 * u + c);
    }
    return t;
  }
  __device__ __forceinline__ Fast fast(const Tile& t, int row, int col) const {
    Fast f{};
    if (!GATED && residual)
      f.residual = __builtin_amdgcn_raw_buffer_load_b128(
          t.residual.rsrc, t.residual.lane, scalar_in<8>(t.residual, row, col), 0);
    return f;
  }
  template <typename K>
  __device__ __forceinline__ void store_fast(K, const Tile& t, int row, int col, float v[8],
                                             const Fast& f) const {
    if (bias) {
      const words4 b = col ? t.bias[1] : t.bias[0];
#pragma unroll
      for (int j = 0; j < 8; ++j) v[j] += half_of(b, j);
    }
    if (product) {
      const words4 z = packed8(v);
      __builtin_amdgcn_raw_buffer_store_b128(z, t.product.rsrc, t.product.lane,
                                             scalar_in<8>(t.product, row, col), NON_TEMPORAL);
      if (low) {
        const uint32_t high[4] = {z.x, z.y, z.z, z.w};
        __builtin_amdgcn_raw_buffer_store_b64(
            __builtin_bit_cast(words2, low_bytes(v, high)), t.low.rsrc, t.low.lane,
            row * t.low.pitch + col, NON_TEMPORAL);
      }
    }
    if constexpr (GATED) {
      float h[4];
#pragma unroll
      for (int j = 0; j < 4; ++j) h[j] = unit_of<K, F32>(act, v[2 * j], v[2 * j + 1]);
      __builtin_amdgcn_raw_buffer_store_b64(
          words2{pack_bf16x2(h[0], h[1]), pack_bf16x2(h[2], h[3])}, t.out.rsrc, t.out.lane,
          scalar_in<4>(t.out, row, col), NON_TEMPORAL);
    } else {
      if constexpr (!std::is_same<K, NoAct>::value) {
#pragma unroll
        for (int j = 0; j < 8; ++j) v[j] = unit_of<K, F32>(act, v[j], 0.0f);
      }
      if (residual) {
#pragma unroll
        for (int j = 0; j < 8; ++j) v[j] += half_of(f.residual, j);
      }
      __builtin_amdgcn_raw_buffer_store_b128(packed8(v), t.out.rsrc, t.out.lane,
                                             scalar_in<8>(t.out, row, col), NON_TEMPORAL);
    }
  }

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
    of_act<GATED>(act, f);
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
    if constexpr (!F32) {
      if (low) {
        uint32_t high[4];
#pragma unroll
        for (int j = 0; j < 4; ++j) high[j] = pack_bf16x2(z[2 * j], z[2 * j + 1]);
        store_low(low + row * n + col, low_bytes(z, high), count);
      }
    }
    if constexpr (GATED) {
      float h[4];
#pragma unroll
      for (int j = 0; j < 4; ++j) h[j] = unit_of<K, F32>(act, z[2 * j], z[2 * j + 1]);
      store_some<T, 4>(out + row * (n / 2) + col / 2, h, count / 2);
    } else {
      if constexpr (!std::is_same<K, NoAct>::value) {
#pragma unroll
        for (int j = 0; j < 8; ++j) z[j] = unit_of<K, F32>(act, z[j], 0.0f);
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
  static constexpr bool HALVES = GATED;
  Act act;
  const T* product;    // [m, n, P]
  const uint8_t* low;  // its low bytes (bfloat16), or NULL
  T* out;              // product's shape
  uint8_t* out_low;    // its low bytes (bfloat16), or NULL: what the biases' sums take
  int64_t n;         // units

  struct Tile {
    Place out, product, low, out_low;
  };
  struct Fast {
    words4 p[P];
    words2 low[P];
  };
  __device__ __forceinline__ bool aligned() const {
    return aligned16(out, n) && aligned16(product, n) && n < (1 << 20) &&
           (low == nullptr || reinterpret_cast<uintptr_t>(low) % 8 == 0) &&
           (out_low == nullptr || reinterpret_cast<uintptr_t>(out_low) % 8 == 0);
  }
  __device__ __forceinline__ Tile tile(int64_t row, int64_t col) const {
    return Tile{place_in<8 * P>(out, row, col, n), place_in<8 * P>(product, row, col, n),
                bytes_in<8 * P>(low, row, col, n), bytes_in<8 * P>(out_low, row, col, n)};
  }
  __device__ __forceinline__ Fast fast(const Tile& t, int row, int col) const {
    Fast f;
#pragma unroll
    for (int i = 0; i < P; ++i)
      f.p[i] = __builtin_amdgcn_raw_buffer_load_b128(
          t.product.rsrc, t.product.lane + HALF * i, scalar_in<8 * P>(t.product, row, col), 0);
    if (low) {
#pragma unroll
      for (int i = 0; i < P; ++i)
        f.low[i] = __builtin_amdgcn_raw_buffer_load_b64(t.low.rsrc, t.low.lane + HALF / 2 * i,
                                                        row * t.low.pitch + col * P, 0);
    }
    return f;
  }
  template <typename K>
  __device__ __forceinline__ void store_fast(K, const Tile& t, int row, int col, float v[8],
                                             const Fast& f) const {
    float d[8 * P];
    if constexpr (std::is_same<K, NoAct>::value) {
#pragma unroll
      for (int j = 0; j < 8; ++j) d[j] = v[j];
    } else {
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        float du, dg;
        float up = half_of(f.p[j * P / 8], j * P % 8);
        float gate = GATED ? half_of(f.p[j * P / 8], j * P % 8 + 1) : 0.0f;
        if (low) {
          const uint64_t b = __builtin_bit_cast(uint64_t, f.low[j * P / 8]);
          up = with_low(up, b, j * P % 8);
          if (GATED) gate = with_low(gate, b, j * P % 8 + 1);
        }
        unit_grad_of<K, F32>(act, up, gate, v[j], &du, &dg);
        d[j * P] = du;
        if (GATED) d[j * P + 1] = dg;
      }
    }
#pragma unroll
    for (int i = 0; i < P; ++i) {
      const words4 w = packed8(d + 8 * i);
      __builtin_amdgcn_raw_buffer_store_b128(w, t.out.rsrc, t.out.lane + HALF * i,
                                             scalar_in<8 * P>(t.out, row, col), NON_TEMPORAL);
      if (out_low) {
        const uint32_t high[4] = {w.x, w.y, w.z, w.w};
        __builtin_amdgcn_raw_buffer_store_b64(
            __builtin_bit_cast(words2, low_bytes(d + 8 * i, high)), t.out_low.rsrc,
            t.out_low.lane + HALF / 2 * i, row * t.out_low.pitch + col * P, NON_TEMPORAL);
      }
    }
  }

  struct In {
    Eight<T> p[P];
    uint64_t low[P];
  };
  __device__ __forceinline__ In load(int64_t row, int64_t col) const {
    In in{};
#pragma unroll
    for (int i = 0; i < P; ++i)
      in.p[i] = load_eight(product + (row * n + col) * P + 8 * i, (n - col) * P - 8 * i);
    if (!F32 && low) {
#pragma unroll
      for (int i = 0; i < P; ++i)
        in.low[i] = load_low(low + (row * n + col) * P + 8 * i, (n - col) * P - 8 * i);
    }
    return in;
  }
  template <typename F>
  __device__ __forceinline__ void choose(F&& f) const {
    of_act<GATED>(act, f);
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
        float du, dg;
        float up = in.p[j * P / 8].value(j * P % 8);
        float gate = GATED ? in.p[j * P / 8].value(j * P % 8 + 1) : 0.0f;
        if (!F32 && low) {
          up = with_low(up, in.low[j * P / 8], j * P % 8);
          if (GATED) gate = with_low(gate, in.low[j * P / 8], j * P % 8 + 1);
        }
        unit_grad_of<K, F32>(act, up, gate, v[j], &du, &dg);
        d[j * P] = du;
        if (GATED) d[j * P + 1] = dg;
      }
    }
#pragma unroll
    for (int i = 0; i < P; ++i) {
      const int64_t at = (row * n + col) * P + 8 * i, count = (n - col) * P - 8 * i;
      store_some<T>(out + at, d + 8 * i, count);
      if constexpr (!F32) {
        if (out_low) {
          uint32_t high[4];
#pragma unroll
          for (int j = 0; j < 4; ++j)
            high[j] = pack_bf16x2(d[8 * i + 2 * j], d[8 * i + 2 * j + 1]);
          store_low(out_low + at, low_bytes(d + 8 * i, high), count);
        }
      }
    }
  }
};

// The workspace's rows are whole 8s of columns, `pitch`.
struct Partial {
  static constexpr bool HALVES = true;
  float* out;
  int64_t pitch;
  struct Tile {
    Place out;
  };
  struct Fast {};
  __device__ __forceinline__ bool aligned() const { return pitch < (1 << 20); }
  __device__ __forceinline__ Tile tile(int64_t row, int64_t col) const {
    // (as pairs of 16 bits)
    return Tile{place_in<16>(reinterpret_cast<const uint16_t*>(out), row, col, pitch)};
  }
  __device__ __forceinline__ Fast fast(const Tile&, int, int) const { return Fast{}; }
  template <typename K>
  __device__ __forceinline__ void store_fast(K, const Tile& t, int row, int col, float v[8],
                                             const Fast&) const {
    const int32_t at = scalar_in<16>(t.out, row, col);
#pragma unroll
    for (int i = 0; i < 2; ++i)
      __builtin_amdgcn_raw_buffer_store_b128(
          words4{__float_as_uint(v[4 * i]), __float_as_uint(v[4 * i + 1]),
                 __float_as_uint(v[4 * i + 2]), __float_as_uint(v[4 * i + 3])},
          t.out.rsrc, t.out.lane + HALF * i, at, 0);
  }
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
// (HALVES: columns 4 (l % 8) and 32 + 4 (l % 8).)
template <bool HALVES = false>
__device__ __forceinline__ void get_row(const uint8_t* region, int it, float v[8]) {
  const int lane = threadIdx.x & 63, r = (lane >> 3) + 8 * it;
  const int c = HALVES ? lane & 7 : 2 * (lane & 7), d = HALVES ? c + 8 : c + 1;
  const float4 x = *reinterpret_cast<const float4*>(region + r * 256 + 16 * (c ^ (r & 15)));
  const float4 y = *reinterpret_cast<const float4*>(region + r * 256 + 16 * (d ^ (r & 15)));
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
  epi.choose([&](auto kind) {
#pragma unroll 1
    for (int it = 0; it < 4; ++it) {
      if (row + 8 * it >= m || col >= n) continue;
      const typename Epi::In in = epi.load(row + 8 * it, col);
      float v[8];
      get_row(region, it, v);
      epi.store(kind, row + 8 * it, col, v, in);
    }
  });
}

// --- the kernels' operands ------------------------------------------------------------------

// A(r, k) at p[r ld + k] (K-major) or p[k ld + r], r < rows.
template <typename T>
struct Mat {
  const T* p;
  int64_t ld, rows;
};

inline int64_t pitch_of(int64_t n) { return (n + 7) / 8 * 8; }

// Tile `id` of an output of row_tiles x col_tiles: bands of 8 row tiles, a band's columns one
// after another, so that neighbouring tiles share both operands' rows in an XCD's L2.
__device__ __forceinline__ void place_of(int32_t id, int32_t row_tiles, int32_t col_tiles,
                                         int32_t* row, int32_t* col) {
  const int32_t band = id / (8 * col_tiles), first = 8 * band;
  const int32_t high = row_tiles - first < 8 ? row_tiles - first : 8;
  const int32_t rest = id - first * col_tiles;
  *row = first + rest % high;
  *col = rest / high;
}

// The large tiles' kernel (dense_tiles.hip): whether it takes the operands, and its launch, K
// [0, k) in `splits` parts of `units` 64s.
bool large_takes(const Mat<uint16_t>& A, bool a_km, const Mat<uint16_t>& B, bool b_km, int64_t m,
                 int64_t n, int64_t k);
template <bool AKM, bool BKM, typename Epi>
int launch_large(const Mat<uint16_t>& A, const Mat<uint16_t>& B, int64_t m, int64_t n, int64_t k,
                 int64_t units, int64_t splits, const Epi& epi, hipStream_t s);


// The few rows' kernel (dense_few.hip): whether it takes the operands (x K-major), the parts that K
// is split into, and its launch.
bool few_takes(const Mat<uint16_t>& A, const Mat<uint16_t>& B, int64_t m, int64_t n, int64_t k);
int64_t few_splits(int64_t n, int64_t k);
template <bool BKM, typename Epi>
int launch_few(const Mat<uint16_t>& A, const Mat<uint16_t>& B, int64_t m, int64_t n, int64_t k,
               int64_t splits, const Epi& epi, hipStream_t s);

}  // namespace dense
}  // namespace bux
