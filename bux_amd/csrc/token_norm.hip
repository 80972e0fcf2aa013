// The tokens' norm before a layer (layers/norm.py:14-78), with the residual stream's addition:
//
//   u = x + residual (rounded to the rows' type, stored as `summed`), or x
//   v = u, or u g with scale_input
//   c = v - mean(v) (layernorm) or v (rmsnorm);  r = (mean(c^2) + eps)^(-1/2)
//   out = c r g + b  (g: scale, or 1 + scale; not with scale_input), rounded once
//
// and its backward, given dy and the gradient that reaches u past the norm (d_summed):
//
//   h = dy g (dy with scale_input);  dv = r (h - mean(h) - c r^2 mean(h c)), mean(h) for a
//   layernorm alone;  dx = dv + d_summed (dv g + d_summed with scale_input), rounded once
//   d_scale = sum over rows of dy c r (dv u with scale_input);  d_bias = sum of dy
//
// Everything between the loads and the stores is float32; the expert norm (norm.hip) rounds at
// every step as the reference's bfloat16 ops do, this op once, so its results are the nearer.
//
// Both are bound by HBM. A row is W waves', its values in registers, read once: each lane the
// 8 columns of C chunks. Rows of any width and alignment take the same loads, of 8 elements at
// an element's alignment. The backward's workgroups take rows in turn; each lane adds its
// columns' gradients in registers over all of them, the workgroup's waves meet in LDS, and
// params_kernel adds the workgroups' sums in a fixed order (4.6 us, a launch's latency).
//
// Forward, 16384 bfloat16 rows of 2048 with their residual: 44.6 us, 6.0 TB/s; one row of 7168 5.1
// us, its chain of loads and sums. Backward: 8192 bfloat16 rows of 2880 38 us and 16384 of 7168
// 141 us, 5.0 TB/s of the 6.2 that a hand-written copy reaches (the library's 5.1).

#include <type_traits>

#include "common.h"

namespace bux {
namespace {

constexpr int VEC = 8;
typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));
constexpr int MAX_CHUNKS = 3;
constexpr int64_t MAX_WIDTH = 8 * 64 * VEC * MAX_CHUNKS;  // 12288: 8 waves

// 8 elements at any element's alignment, as they lie.
template <typename T>
struct Raw8 {
  struct __attribute__((packed, aligned(sizeof(T)))) Bytes {
    T at[VEC];
  };
  Bytes b;
  __device__ __forceinline__ void load(const T* p) { b = *reinterpret_cast<const Bytes*>(p); }
  __device__ __forceinline__ float value(int j) const { return Elem<T>::value(b.at[j]); }
};

// A lane's part of a row of d columns (8 at least): those from c on, up to 8, none from d on.
// TAIL (d is no multiple of 8): the part that the row's end cuts short holds the row's last 8
// columns; those that the part before it has count 0 here. So every part is one load, and
// element j is the column base() + j.
template <bool TAIL>
struct Part {
  int c, d;
  __device__ __forceinline__ bool any() const { return c < d; }
  __device__ __forceinline__ int base() const { return TAIL && c + VEC > d ? d - VEC : c; }
  __device__ __forceinline__ bool has(int j) const { return c < d && (!TAIL || base() + j >= c); }
};
template <bool TAIL, typename T>
__device__ __forceinline__ Raw8<T> load_part(const T* row, Part<TAIL> p) {
  Raw8<T> r{};
  if (p.any()) {
    r.load(row + p.base());
    if (TAIL && p.base() < p.c) {
#pragma unroll
      for (int j = 0; j < VEC; ++j)
        if (!p.has(j)) r.b.at[j] = Elem<T>::make(0.0f);
    }
  }
  return r;
}
template <bool TAIL, typename T>
__device__ __forceinline__ void store_part(T* row, Part<TAIL> p, const float* v) {
  if (!p.any()) return;
  Raw8<T> r;
#pragma unroll
  for (int j = 0; j < VEC; ++j) r.b.at[j] = Elem<T>::make(v[j]);
  T* at = row + p.base();
  if (!TAIL || p.base() == p.c) {
    *reinterpret_cast<typename Raw8<T>::Bytes*>(at) = r.b;
  } else {
#pragma unroll
    for (int j = 0; j < VEC; ++j)
      if (p.has(j)) at[j] = r.b.at[j];
  }
}

// The sum over a row's W waves, to all of them. `red`: W floats of LDS for each sum in
// flight; a second call may not reuse the first's before the workgroup's next barrier.
template <int W>
__device__ __forceinline__ float row_sum(float v, float* red) {
#pragma unroll
  for (int s = 32; s >= 1; s >>= 1) v += __shfl_xor(v, s);
  if constexpr (W == 1) return v;
  const int wave = (threadIdx.x >> 6) % W;
  if ((threadIdx.x & 63) == 0) red[wave] = v;
  asm volatile("s_waitcnt lgkmcnt(0)\n\ts_barrier" ::: "memory");  // loads stay in flight
  float t = red[0];
#pragma unroll
  for (int w = 1; w < W; ++w) t += red[w];
  return t;
}

template <typename T>
struct Settings {
  bool centred, affine, scale_input, biased;
  float eps;
  float base;  // the gain is base + scale: 1 for a zero-centered one, and for none (scale 0)
  const T* scale;
  const T* bias;
};

template <bool TAIL, typename T>
__device__ __forceinline__ Raw8<T> load_scale(const Settings<T>& a, Part<TAIL> p) {
  return load_part(a.scale, Part<TAIL>{p.c, a.affine ? p.d : 0});
}

// Workgroups of max(4, W) waves; rows a workgroup holds at once: 4 / W, or 1.
template <int W>
constexpr int threads_of() { return 64 * (W > 4 ? W : 4); }

// Which of a workgroup's rows this wave works on, as a scalar, and its lane there.
template <int W>
__device__ __forceinline__ int sub_row() {
  return __builtin_amdgcn_readfirstlane(threadIdx.x / (64 * W));
}

template <typename T, int W, int C, bool TAIL>
__global__ __launch_bounds__(threads_of<W>()) void forward_kernel(
    const T* __restrict__ x, const T* __restrict__ residual, int64_t m, int d, Settings<T> a,
    T* __restrict__ summed, T* __restrict__ out, float2* __restrict__ stats) {
  constexpr int ROWS = threads_of<W>() / (64 * W);
  __shared__ float red[2][ROWS][W];
  const int sub = sub_row<W>(), lane = threadIdx.x % (64 * W);
  auto part = [&](int i) { return Part<TAIL>{(i * 64 * W + lane) * VEC, d}; };
  const int64_t r = static_cast<int64_t>(blockIdx.x) * ROWS + sub;
  const bool live = r < m;  // (a workgroup's barriers are for all of its rows)
  const int64_t row = live ? r : m - 1;
  const float n = static_cast<float>(d);
  float v[C][VEC];
  Raw8<T> xs[C], rs[C];
#pragma unroll
  for (int i = 0; i < C; ++i) {
    xs[i] = load_part(x + row * d, part(i));
    if (residual) rs[i] = load_part(residual + row * d, part(i));
  }
  float sum = 0.0f;
#pragma unroll
  for (int i = 0; i < C; ++i) {
#pragma unroll
    for (int j = 0; j < VEC; ++j) {
      v[i][j] = xs[i].value(j);
      if (residual) v[i][j] = Elem<T>::round(v[i][j] + rs[i].value(j));
    }
    if (summed && live) store_part(summed + row * d, part(i), v[i]);
    if (a.scale_input) {
      const Raw8<T> s = load_scale(a, part(i));
#pragma unroll
      for (int j = 0; j < VEC; ++j) v[i][j] *= a.base + s.value(j);
    }
#pragma unroll
    for (int j = 0; j < VEC; ++j) sum += v[i][j];  // columns past d hold 0
  }
  const float mean = a.centred ? row_sum<W>(sum, red[0][sub]) / n : 0.0f;
  float sq = 0.0f;
#pragma unroll
  for (int i = 0; i < C; ++i)
#pragma unroll
    for (int j = 0; j < VEC; ++j) {
      v[i][j] = part(i).has(j) ? v[i][j] - mean : 0.0f;
      sq += v[i][j] * v[i][j];
    }
  const float rstd = 1.0f / sqrtf(row_sum<W>(sq, red[1][sub]) / n + a.eps);
  if (!live) return;
  if (stats && lane == 0) stats[row] = make_float2(mean, rstd);
#pragma unroll
  for (int i = 0; i < C; ++i) {
    if (!part(i).any()) continue;
#pragma unroll
    for (int j = 0; j < VEC; ++j) v[i][j] *= rstd;
    if (a.affine && !a.scale_input) {
      const Raw8<T> s = load_scale(a, part(i));
#pragma unroll
      for (int j = 0; j < VEC; ++j) v[i][j] *= a.base + s.value(j);
    }
    if (a.biased) {
      const Raw8<T> b = load_part(a.bias, part(i));
#pragma unroll
      for (int j = 0; j < VEC; ++j) v[i][j] += b.value(j);
    }
    store_part(out + row * d, part(i), v[i]);
  }
}

// The backward's workgroups over m rows of W waves of C chunks: as many as the chip holds at
// once by their registers (4, 3 or 2 waves a SIMD; of 8 waves two a CU or one, so two), or a turn
// each where there are fewer rows. (16384 bfloat16 rows of 7168, before Ahead: 384 workgroups of
// 8 waves 200 us, 512 161; the next row's loads to registers ahead of this one's sums 189.)
constexpr int64_t MAX_BLOCKS = 1024;
constexpr int64_t SIMDS = 1024;  // 256 CUs of 4
// One workgroup where it has at most so many turns, whose sums are the gradients themselves: a
// launch less (4 bfloat16 rows of 512 5.1 us, so 3.0, 4 of 2880, two turns, 6.4 both; eager 15.8
// and 13.4). At four turns 16 rows of 1027 took 17.1 us and 9.8.
constexpr int64_t ALONE_TURNS = 2;
// Whole 256s of workgroups of so many turns at least, of 8 waves and of 4: with fewer turns their
// sums, two rows of float32 each, weigh beside the rows themselves (bfloat16 rows in us: 1000 of
// 7168 in 512 workgroups 33, in 256 23, 4000 55 and 47; 3001 of 1024 in 751 14.6, in 256 11.9, but
// 2000 of 2880, two rows a turn, 18.4 in 512 and 19.6 in 256).
constexpr int64_t SUMS_TURNS_8 = 16, SUMS_TURNS_4 = 3;
int64_t backward_blocks(int64_t m, int w, int c) {
  const int64_t a_simd = c == 1 || (c == 2 && w > 4) ? 4 : c == 2 ? 3 : 2;
  const int64_t most = a_simd * SIMDS / (w > 4 ? w : 4);
  const int64_t want = ceil_div(m, w > 4 ? 1 : 4 / w);
  if (want <= ALONE_TURNS) return 1;
  const int64_t in_turns = ceil_div(want, (w > 4 ? SUMS_TURNS_8 : SUMS_TURNS_4) * 256) * 256;
  const int64_t enough = in_turns < most ? in_turns : most;
  return want < enough ? want : enough;
}

// A lane's sums of its columns' gradients, from the workgroup's waves that hold the same
// columns (ROWS of them) added in LDS in their order, to partials[block][d].
template <int W, int C, int ROWS, bool TAIL>
__device__ __forceinline__ void store_sums(float (&s)[C][VEC], float* lds, int d, float* out) {
  const int sub = sub_row<W>(), lane = threadIdx.x % (64 * W);
  if constexpr (ROWS > 1) {
#pragma unroll 1
    for (int k = 1; k < ROWS; ++k) {
      __syncthreads();
      if (sub == k) {
#pragma unroll
        for (int i = 0; i < C; ++i)
#pragma unroll
          for (int j = 0; j < VEC; ++j) lds[(i * VEC + j) * 64 * W + lane] = s[i][j];
      }
      __syncthreads();
      if (sub == 0) {
#pragma unroll
        for (int i = 0; i < C; ++i)
#pragma unroll
          for (int j = 0; j < VEC; ++j) s[i][j] += lds[(i * VEC + j) * 64 * W + lane];
      }
    }
    if (sub != 0) return;
  }
#pragma unroll
  for (int i = 0; i < C; ++i) {
    const Part<TAIL> p{(i * 64 * W + lane) * VEC, d};
#pragma unroll
    for (int j = 0; j < VEC; ++j)
      if (p.has(j)) out[p.base() + j] = s[i][j];
  }
}

// Makes the compiler forget what it knows of a part, so that it computes from it again
// rather than keep what it computed (8 registers a part and value).
template <typename T>
__device__ __forceinline__ void forget(Raw8<T>& r) {
  typedef uint32_t Words __attribute__((ext_vector_type(sizeof(T) * VEC / 4)));
  Words w = __builtin_bit_cast(Words, r);
  asm volatile("" : "+v"(w));
  r = __builtin_bit_cast(Raw8<T>, w);
}

// A wave's operands of one row, 512 columns of each chunk of x, dy and d_summed, on their way
// through LDS: no registers, so that the next row's loads fly while this one's sums are made
// (to registers when their turn comes: 8192 rows of 2880 44 us, 16384 of 7168 161; so 38 and 141).
// 32-bit rows would leave a CU one workgroup of 8 waves, and rows of an odd width or alignment
// have no direct load.
template <int W, int C>
struct Ahead {
  uint4 at[3][C][W][64];
};

// BIASED: the bias's gradient too. INPUT: scale_input's. AHEAD: 16-bit rows of whole chunks at
// 16 bytes' alignment; their operands come through LDS, a row ahead. scale_sums, bias_sums:
// [blocks][d], NULL where the norm has none.
template <typename T, int W, int C, bool BIASED, bool INPUT, bool TAIL, bool AHEAD>
__global__ __launch_bounds__(threads_of<W>()) void backward_kernel(
    const T* __restrict__ dy, const T* __restrict__ x, const float2* __restrict__ stats,
    const T* __restrict__ d_summed, int64_t m, int d, Settings<T> a, T* __restrict__ dx,
    float* __restrict__ scale_sums, float* __restrict__ bias_sums) {
  static_assert(!AHEAD || (!TAIL && sizeof(T) == 2), "16-bit rows of whole chunks");
  constexpr int ROWS = threads_of<W>() / (64 * W);
  __shared__ float red[2][2][ROWS][W];
  __shared__ float sums[ROWS > 1 ? C * VEC * 64 * W : 1];
  __shared__ Ahead<W, C> ahead[AHEAD ? ROWS : 1];
  const int sub = sub_row<W>(), lane = threadIdx.x % (64 * W);
  auto part = [&](int i) { return Part<TAIL>{(i * 64 * W + lane) * VEC, d}; };
  const int64_t step = static_cast<int64_t>(gridDim.x) * ROWS;
  const float inv_n = 1.0f / static_cast<float>(d);
  Raw8<T> gain[C];
  float dg[C][VEC], db[C][VEC];
#pragma unroll
  for (int i = 0; i < C; ++i) {
    gain[i] = load_scale(a, part(i));
#pragma unroll
    for (int j = 0; j < VEC; ++j) dg[i][j] = db[i][j] = 0.0f;
  }
  // AHEAD: a row's loads, zeros past its end and for a row past the last
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x / 64 % W);
  const uint32_t lds = lds_at(&ahead[AHEAD ? sub : 0]) + wave * 1024;
  float2 next_st;
  auto fetch = [&](int64_t base) {
    const int64_t row = base + sub < m ? base + sub : m - 1;
    const int64_t bytes = base + sub < m ? d * 2 : 0;
    next_st = stats[row];
    const T* from[3] = {x, dy, d_summed};
#pragma unroll
    for (int k = 0; k < 3; ++k) {
      if (k == 2 && !d_summed) break;
      const i32x4 r = resource(from[k] + row * d, bytes);
#pragma unroll
      for (int i = 0; i < C; ++i)
        load_lds16_uniform(r, lds + (k * C + i) * W * 1024, part(i).c * 2, 0);
    }
  };
  int turn = 0;
  int64_t base = static_cast<int64_t>(blockIdx.x) * ROWS;
  if constexpr (AHEAD) {
#pragma unroll
    for (int i = 0; i < C; ++i) forget(gain[i]);  // in registers: no wait for it in the loop
    fetch(base);
    asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
  }
  for (; base < m; base += step, turn ^= 1) {
    // a row past the last: the last one's values (or zeros) with a gradient of 0, and nothing
    // stored
    const bool live = base + sub < m;
    const int64_t row = live ? base + sub : m - 1;
    Raw8<T> xs[C], gs[C], past[C];
    float2 st;
    if constexpr (AHEAD) {
      const Ahead<W, C>& mine = ahead[sub];
#pragma unroll
      for (int i = 0; i < C; ++i) {
        xs[i] = __builtin_bit_cast(Raw8<T>, mine.at[0][i][wave][threadIdx.x & 63]);
        gs[i] = __builtin_bit_cast(Raw8<T>, mine.at[1][i][wave][threadIdx.x & 63]);
      }
      if (d_summed) {
#pragma unroll
        for (int i = 0; i < C; ++i)
          past[i] = __builtin_bit_cast(Raw8<T>, mine.at[2][i][wave][threadIdx.x & 63]);
      }
      st = next_st;
      asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");  // read: the next row may land there
      if (base + step < m) fetch(base + step);
    } else {
#pragma unroll
      for (int i = 0; i < C; ++i) {
        xs[i] = load_part(x + row * d, part(i));
        gs[i] = load_part(dy + row * d, Part<TAIL>{part(i).c, live ? d : 0});
      }
      st = stats[row];
      if (d_summed) {
#pragma unroll
        for (int i = 0; i < C; ++i) past[i] = load_part(d_summed + row * d, part(i));
      }
    }
    const float mean = st.x, rstd = st.y;
    auto gain_at = [&](int i, int j) { return a.base + gain[i].value(j); };
    // the normalized value and the gradient to it; past d the gradient is 0
    auto normal = [&](int i, int j) {
      const float v = xs[i].value(j);
      return ((INPUT ? v * gain_at(i, j) : v) - mean) * rstd;
    };
    auto to_normal = [&](int i, int j) {
      return INPUT ? gs[i].value(j) : gs[i].value(j) * gain_at(i, j);
    };
    float s1 = 0.0f, s2 = 0.0f;
#pragma unroll
    for (int i = 0; i < C; ++i)
#pragma unroll
      for (int j = 0; j < VEC; ++j) {
        const float u = normal(i, j), h = to_normal(i, j);
        if (!INPUT) dg[i][j] += gs[i].value(j) * u;
        if (BIASED) db[i][j] += gs[i].value(j);
        s1 += h;
        s2 += h * u;
      }
    const float m1 = a.centred ? row_sum<W>(s1, red[turn][0][sub]) * inv_n : 0.0f;
    const float m2 = row_sum<W>(s2, red[turn][1][sub]) * inv_n;
    if (C == MAX_CHUNKS) {
#pragma unroll
      for (int i = 0; i < C; ++i) {
        forget(xs[i]);
        forget(gs[i]);
        forget(gain[i]);
      }
    }
    const auto to = __builtin_amdgcn_make_buffer_rsrc(dx + row * d, 0, live ? d * sizeof(T) : 0,
                                                      0x00020000);
#pragma unroll
    for (int i = 0; i < C; ++i) {
      float o[VEC];
#pragma unroll
      for (int j = 0; j < VEC; ++j) {
        float v = rstd * (to_normal(i, j) - m1 - normal(i, j) * m2);
        if (INPUT) {
          if (live) dg[i][j] += v * xs[i].value(j);  // x is 0 past d
          v *= gain_at(i, j);
        }
        if (d_summed) v += past[i].value(j);
        o[j] = v;
      }
      if constexpr (AHEAD) {
        // in every lane and turn, those past the row's end dropped: a count to wait by
        Raw8<T> r;
#pragma unroll
        for (int j = 0; j < VEC; ++j) r.b.at[j] = Elem<T>::make(o[j]);
        __builtin_amdgcn_raw_buffer_store_b128(__builtin_bit_cast(u32x4, r), to, part(i).c * 2, 0,
                                               0);
      } else {
        if (live) store_part(dx + row * d, part(i), o);
      }
    }
    // the next row's loads are in (memory operations end in order; this row's stores may not)
    if constexpr (AHEAD) asm volatile("s_waitcnt vmcnt(%0)" ::"n"(C) : "memory");
  }
  const int64_t at = static_cast<int64_t>(blockIdx.x) * d;
  if (a.affine) store_sums<W, C, ROWS, TAIL>(dg, sums, d, scale_sums + at);
  if (BIASED) store_sums<W, C, ROWS, TAIL>(db, sums, d, bias_sums + at);
}

// d_scale (blockIdx.y 0) and d_bias (1): the workgroups' sums of 64 columns, a wave every
// 16th of them in order, then the waves' in wave order.
constexpr int PARAM_THREADS = 1024;
__global__ __launch_bounds__(PARAM_THREADS) void params_kernel(const float* __restrict__ partials,
                                                               int64_t blocks, int64_t d,
                                                               float* __restrict__ d_scale,
                                                               float* __restrict__ d_bias) {
  constexpr int WAVES = PARAM_THREADS / 64;
  __shared__ float part[WAVES][64];
  float* out = blockIdx.y == 0 ? d_scale : d_bias;
  if (out == nullptr) return;
  const int wave = threadIdx.x >> 6, lane = threadIdx.x & 63;
  const int64_t c = static_cast<int64_t>(blockIdx.x) * 64 + lane;
  const float* from = partials + static_cast<int64_t>(blockIdx.y) * blocks * d;
  float s = 0.0f;
  if (c < d) {
#pragma unroll 8
    for (int64_t k = wave; k < blocks; k += WAVES) s += from[k * d + c];
  }
  part[wave][lane] = s;
  __syncthreads();
  if (wave != 0 || c >= d) return;
#pragma unroll
  for (int w = 1; w < WAVES; ++w) s += part[w][lane];
  out[c] = s;
}

// Calls f(W, C, TAIL) for rows of d columns: the fewest waves that hold them in at most 3
// chunks a lane (a fourth takes the backward past the 256 registers of two waves a SIMD).
template <typename F>
void with_shape(int64_t d, F&& f) {
  using std::integral_constant;
  auto chunks = [&](auto w) {
    const int64_t c = ceil_div(d, 64 * VEC * decltype(w)::value);
    auto go = [&](auto n) {
      if (d % VEC == 0) f(w, n, std::false_type{});
      else f(w, n, std::true_type{});
    };
    if constexpr (decltype(w)::value == 1) {
      if (c <= 1) return go(integral_constant<int, 1>{});
    }
    return c <= 2 ? go(integral_constant<int, 2>{}) : go(integral_constant<int, 3>{});
  };
  constexpr int64_t WAVE = 64 * VEC * MAX_CHUNKS;
  if (d <= WAVE) return chunks(integral_constant<int, 1>{});
  if (d <= 2 * WAVE) return chunks(integral_constant<int, 2>{});
  if (d <= 4 * WAVE) return chunks(integral_constant<int, 4>{});
  return chunks(integral_constant<int, 8>{});
}

bool aligned16(const void* p) { return reinterpret_cast<uintptr_t>(p) % 16 == 0; }

template <typename T>
int settings_of(const char* name, int64_t m, int64_t d, const bux_norm* norm, const T* scale,
                const T* bias, bool forward, Settings<T>* a) {
  BUX_CHECK(m >= 0 && m < (1LL << 31) && d >= VEC && d <= MAX_WIDTH,
            "%s: bad shape m=%lld d=%lld (d of %d to %lld)", name, (long long)m, (long long)d, VEC,
            (long long)MAX_WIDTH);
  // a launch holds fewer than 2^32 threads, and a row takes 64 of them at least
  BUX_CHECK(m * ceil_div(d, 64 * VEC * MAX_CHUNKS) < (1LL << 25),
            "%s: m=%lld rows of d=%lld are more than a launch holds", name, (long long)m,
            (long long)d);
  BUX_CHECK(norm != nullptr, "%s: NULL norm", name);
  BUX_CHECK(norm->kind == BUX_LAYERNORM || norm->kind == BUX_RMSNORM,
            "%s: kind %d is neither BUX_LAYERNORM nor BUX_RMSNORM", name, norm->kind);
  BUX_CHECK(norm->eps >= 0.0f, "%s: eps %g", name, norm->eps);
  BUX_CHECK(!norm->affine || scale, "%s: an affine norm needs its scale", name);
  BUX_CHECK(!forward || !norm->bias || bias, "%s: a biased norm needs its bias", name);
  const bool affine = norm->affine != 0;
  *a = Settings<T>{norm->kind == BUX_LAYERNORM, affine, affine && norm->scale_input != 0,
                   norm->bias != 0, norm->eps, affine && norm->zero_centered == 0 ? 0.0f : 1.0f,
                   scale, bias};
  return BUX_OK;
}

template <typename T>
int forward(const char* name, const T* x, const T* residual, int64_t m, int64_t d,
            const bux_norm* norm, const T* scale, const T* bias, T* summed, T* out, float* stats,
            void* stream) {
  Settings<T> a;
  if (int rc = settings_of(name, m, d, norm, scale, bias, true, &a)) return rc;
  BUX_CHECK((residual == nullptr) == (summed == nullptr),
            "%s: residual and summed come together", name);
  if (m == 0) return BUX_OK;
  BUX_CHECK(x && out, "%s: NULL buffer", name);
  with_shape(d, [&](auto w, auto c, auto tail) {
    constexpr int W = decltype(w)::value, C = decltype(c)::value;
    constexpr int ROWS = threads_of<W>() / (64 * W);
    hipLaunchKernelGGL((forward_kernel<T, W, C, decltype(tail)::value>),
                       dim3(static_cast<unsigned>(ceil_div(m, ROWS))), dim3(threads_of<W>()), 0,
                       as_stream(stream), x, residual, m, static_cast<int>(d), a, summed, out,
                       reinterpret_cast<float2*>(stats));
  });
  return launched("token norm forward_kernel");
}

// Two sums a workgroup and column, for the most workgroups that rows of any width have: so
// that the size never falls as m or d grows.
size_t backward_workspace(int64_t m, int64_t d) {
  if (m <= 0 || d <= 0) return 0;
  return static_cast<size_t>(2 * (m < MAX_BLOCKS ? m : MAX_BLOCKS) * d) * sizeof(float);
}

template <typename T>
int backward(const char* name, const T* dy, const T* x, const float* stats, const T* d_summed,
             int64_t m, int64_t d, const bux_norm* norm, const T* scale, T* dx, float* d_scale,
             float* d_bias, void* workspace, size_t workspace_bytes, void* stream) {
  Settings<T> a;
  if (int rc = settings_of<T>(name, m, d, norm, scale, nullptr, false, &a)) return rc;
  BUX_CHECK((!a.affine || d_scale) && (!a.biased || d_bias),
            "%s: NULL d_scale or d_bias for a norm that has them", name);
  const size_t need = backward_workspace(m, d);
  if (need > 0 && (workspace == nullptr || workspace_bytes < need))
    return fail(BUX_E_WORKSPACE, "%s: workspace of %zu bytes, %zu needed", name, workspace_bytes,
                need);
  BUX_CHECK(m == 0 || (dy && x && stats && dx), "%s: NULL buffer", name);
  hipStream_t s = as_stream(stream);
  float* const partials = static_cast<float*>(workspace);
  int64_t blocks = 0;
  if (m > 0) {
    with_shape(d, [&](auto w, auto c, auto tail) {
      constexpr int W = decltype(w)::value, C = decltype(c)::value;
      blocks = backward_blocks(m, W, C);
      auto with = [&](auto biased, auto input, auto ahead) {
        hipLaunchKernelGGL((backward_kernel<T, W, C, decltype(biased)::value,
                                            decltype(input)::value, decltype(tail)::value,
                                            decltype(ahead)::value>),
                           dim3(static_cast<unsigned>(blocks)), dim3(threads_of<W>()), 0, s, dy, x,
                           reinterpret_cast<const float2*>(stats), d_summed, m,
                           static_cast<int>(d), a, dx, blocks == 1 ? d_scale : partials,
                           blocks == 1 ? d_bias : partials + blocks * d);
      };
      auto go = [&](auto biased, auto input) {
        if constexpr (sizeof(T) == 2 && !decltype(tail)::value) {
          if (aligned16(dy) && aligned16(x) && aligned16(d_summed) && aligned16(dx))
            return with(biased, input, std::true_type{});
        }
        with(biased, input, std::false_type{});
      };
      if (a.scale_input) a.biased ? go(std::true_type{}, std::true_type{})
                                  : go(std::false_type{}, std::true_type{});
      else a.biased ? go(std::true_type{}, std::false_type{})
                    : go(std::false_type{}, std::false_type{});
    });
    if (int rc = launched("token norm backward_kernel")) return rc;
  }
  if (blocks == 1 || (!a.affine && !a.biased)) return BUX_OK;
  // with no rows, the sums are 0: a workspace of no partials
  hipLaunchKernelGGL(params_kernel, dim3(static_cast<unsigned>(ceil_div(d, 64)), a.biased ? 2 : 1),
                     dim3(PARAM_THREADS), 0, s, static_cast<const float*>(partials), blocks, d,
                     a.affine ? d_scale : nullptr, a.biased ? d_bias : nullptr);
  return launched("token norm params_kernel");
}

}  // namespace
}  // namespace bux

extern "C" int bux_norm_forward(const uint16_t* x, const uint16_t* residual, int64_t m, int64_t d,
                                const bux_norm* norm, const uint16_t* scale, const uint16_t* bias,
                                uint16_t* summed, uint16_t* out, float* stats, void* stream) {
  bux::clear_error();
  return bux::forward("bux_norm_forward", x, residual, m, d, norm, scale, bias, summed, out, stats,
                      stream);
}

extern "C" int bux_norm_forward_f32(const float* x, const float* residual, int64_t m, int64_t d,
                                    const bux_norm* norm, const float* scale, const float* bias,
                                    float* summed, float* out, float* stats, void* stream) {
  bux::clear_error();
  return bux::forward("bux_norm_forward_f32", x, residual, m, d, norm, scale, bias, summed, out,
                      stats, stream);
}

extern "C" size_t bux_norm_backward_workspace_size(int64_t m, int64_t d) {
  return bux::backward_workspace(m, d);
}

extern "C" int bux_norm_backward(const uint16_t* dy, const uint16_t* x, const float* stats,
                                 const uint16_t* d_summed, int64_t m, int64_t d,
                                 const bux_norm* norm, const uint16_t* scale, uint16_t* dx,
                                 float* d_scale, float* d_bias, void* workspace,
                                 size_t workspace_bytes, void* stream) {
  bux::clear_error();
  return bux::backward("bux_norm_backward", dy, x, stats, d_summed, m, d, norm, scale, dx, d_scale,
                       d_bias, workspace, workspace_bytes, stream);
}

extern "C" int bux_norm_backward_f32(const float* dy, const float* x, const float* stats,
                                     const float* d_summed, int64_t m, int64_t d,
                                     const bux_norm* norm, const float* scale, float* dx,
                                     float* d_scale, float* d_bias, void* workspace,
                                     size_t workspace_bytes, void* stream) {
  bux::clear_error();
  return bux::backward("bux_norm_backward_f32", dy, x, stats, d_summed, m, d, norm, scale, dx,
                       d_scale, d_bias, workspace, workspace_bytes, stream);
}
