// 8-bit integers with a scale a row: rows of tokens (by pick too), the activation's rows as
// they are computed, and the columns of the experts' kernels.
//
//   s = max |x| / 127,  q = the integer nearest 127 x / max |x|, the even one at a tie
//
// q is that of the exact quotient. In bfloat16, 127 / max |x| goes in two float32 parts, hi and
// lo, and x hi + (x lo) is the quotient rounded once (to 2^-29 of it): a quotient that is no tie
// lies 2^-17 from one at least (two products of 8-bit mantissas, over one), twice the rounding
// there, and a tie is a float32. In float32 the quotient's nearest integer n comes in float64
// and 127 x - n max |x|, exact there, moves it by one where it exceeds half of max |x|. A row of
// zeros has scale 0 and codes 0; one that holds an infinity or a NaN has that as its scale and
// codes of 0, so that its products are NaN.
//
// The codes are in the GEMM's tiled layout, [K / 64][rows][64] with K padded to whole 128s.
// Bound by HBM: a wave takes a row (narrow rows: 16 lanes each), in registers where it has at most
// 8192 columns (else read twice, the second time from L2); a workgroup's rows lie in one run of
// each K chunk. The activation of 131072 bfloat16 rows of 768 gated units: 131 us, 3.8 TB/s; of
// 65536 of 4096 290, 4.6 TB/s; of 4100, past those kept in registers and so computed twice, 430.

#include <type_traits>

#include "glu.h"

namespace bux {
namespace {

constexpr int THREADS = 256;
constexpr int64_t MAX_K = 131072;  // 127^2 K stays below 2^31
constexpr int64_t MAX_HEIGHT = (1LL << 26) - 4;

template <typename T>
struct Part {
  T at[8];
};

// The larger magnitude's bits of a part's 8 values: as unsigned integers, with infinities above
// every finite value and NaN above those.
__device__ __forceinline__ uint32_t top_of(const Part<uint16_t>& p) {
  const uint4 w = __builtin_bit_cast(uint4, p);
  uint32_t m = max_abs_pair(max_abs_pair(max_abs_pair(max_abs_pair(0u, w.x), w.y), w.z), w.w);
  return larger_half(m) << 16;  // as a float32's bits
}
__device__ __forceinline__ uint32_t top_of(const Part<float>& p) {
  uint32_t m = 0;
#pragma unroll
  for (int j = 0; j < 8; ++j) {
    const uint32_t b = __float_as_uint(p.at[j]) & 0x7fffffffu;
    m = b > m ? b : m;
  }
  return m;
}
// Over a row's L lanes.
template <int L>
__device__ __forceinline__ uint32_t row_top(uint32_t v) {
#pragma unroll
  for (int o = L / 2; o >= 1; o >>= 1) {
    const uint32_t u = __shfl_xor(v, o);
    v = u > v ? u : v;
  }
  return v;
}

// How a row whose largest magnitude is `top` turns into codes.
template <typename T>
struct Coder {
  float scale;
  float pre, hi, lo;    // bfloat16: the quotient is x pre hi + x pre lo
  double most, inverse;  // float32
  __device__ __forceinline__ explicit Coder(uint32_t top) {
    const float a = __uint_as_float(top);
    scale = a / 127.0f;
    const bool live = top > 0 && top < 0x7f800000u;
    if constexpr (std::is_same<T, uint16_t>::value) {
      // tiny rows first times 2^64, so that 127 / a stays finite; in others 1
      pre = live ? (a < 0x1p-100f ? 0x1p64f : 1.0f) : 0.0f;
      const float b = a * pre;
      hi = live ? 127.0f / b : 0.0f;
      lo = live ? __builtin_fmaf(-hi, b, 127.0f) / b : 0.0f;
    } else {
      most = live ? a : 0.0;
      inverse = live ? 127.0 / static_cast<double>(a) : 0.0;
    }
  }
  // The code of x in the low byte; 0 for every x of a row of zeros, infinities or NaN.
  __device__ __forceinline__ uint32_t code(float x) const {
    if constexpr (std::is_same<T, uint16_t>::value) {
#pragma clang fp contract(off)
      if (hi == 0.0f) return 0;
      const float v = x * pre;
      const float q = __builtin_fmaf(v, hi, v * lo);
      // adding 1.5 2^23 rounds to the nearest integer, the even one at a tie
      return __float_as_uint(q + 12582912.0f);
    } else {
      if (most == 0.0) return 0;
      const double v = x;
      double n = __builtin_rint(v * inverse);
      const double r = __builtin_fma(-n, most, 127.0 * v);  // exact
      if (2.0 * r > most) n += 1.0;
      else if (2.0 * r < -most) n -= 1.0;
      else if (__builtin_fabs(2.0 * r) == most) n = 2.0 * __builtin_rint(0.5 * (n + r / most));
      return static_cast<uint32_t>(static_cast<int32_t>(n));
    }
  }
  __device__ __forceinline__ uint2 codes(const Part<T>& p) const {
    uint32_t w[2] = {0, 0};
#pragma unroll
    for (int j = 0; j < 8; ++j)
      w[j / 4] |= (code(Elem<T>::value(p.at[j])) & 0xffu) << (8 * (j % 4));
    return make_uint2(w[0], w[1]);
  }
};

// --- rows ------------------------------------------------------------------------------

// Where a row's values come from: x[row], or x[index[row] / index_div] (a row of 0 where that
// lies outside x's `sources` rows).
enum class Load {
  WHOLE,  // columns a multiple of 8: a part a load (two of float32), at an element's alignment
  TAIL,   // 8 columns at least: the row's last part from its last 8 columns, moved into place (an
          // element at a time: 19276 bfloat16 rows of 990 39 us, so 13)
  NARROW  // fewer: an element at a time
};

// The part's values from place n (0 .. 7) on, zeros after them: 4, 2 and 1 places where n has
// those bits (a runtime index would put the part in scratch memory).
template <typename T>
__device__ __forceinline__ Part<T> from_place(const Part<T>& p, int n) {
  constexpr int WORDS = sizeof(Part<T>) / 4;
  typedef uint32_t Words __attribute__((ext_vector_type(WORDS)));
  Words w = __builtin_bit_cast(Words, p);
  auto move = [&](int by, bool wanted) {
#pragma unroll
    for (int j = 0; j < WORDS; ++j) {
      const uint32_t from = j + by < WORDS ? w[j + by] : 0u;
      w[j] = wanted ? from : w[j];
    }
  };
  if constexpr (sizeof(T) == 2) {
    move(2, n & 4);
    move(1, n & 2);
#pragma unroll
    for (int j = 0; j < WORDS; ++j) {
      const uint32_t next = j + 1 < WORDS ? w[j + 1] : 0u;
      w[j] = n & 1 ? (w[j] >> 16) | (next << 16) : w[j];
    }
  } else {
    move(4, n & 4);
    move(2, n & 2);
    move(1, n & 1);
  }
  return __builtin_bit_cast(Part<T>, w);
}

template <typename T, Load LOAD>
struct Rows {
  const T* x;
  const int32_t* index;
  int32_t index_div;
  int64_t sources, cols;
  struct Row {
    const T* at;  // NULL: a row of 0
  };
  __device__ __forceinline__ Row row(int64_t i) const {
    if (index == nullptr) return Row{x + i * cols};
    const int32_t pick = index[i];
    const int64_t src = pick < 0 ? -1 : pick / index_div;
    return Row{src >= 0 && src < sources ? x + src * cols : nullptr};
  }
  __device__ __forceinline__ Part<T> load(const Row& r, int64_t c) const {
    Part<T> p{};
    if (r.at == nullptr || c >= cols) return p;
    if constexpr (LOAD != Load::NARROW) {
      struct __attribute__((packed, aligned(sizeof(T)))) Any {
        Part<T> p;
      };
      const int64_t at = LOAD == Load::TAIL && c + 8 > cols ? cols - 8 : c;
      p = reinterpret_cast<const Any*>(r.at + at)->p;
      if (LOAD == Load::TAIL && at < c) p = from_place(p, static_cast<int>(c - at));
    } else {
#pragma unroll
      for (int j = 0; j < 8; ++j)
        if (c + j < cols) p.at[j] = r.at[c + j];
    }
    return p;
  }
};

// The activation's rows, each value rounded to the layer's type as bux_glu_forward rounds it.
template <typename K, typename T>
struct Units {
  const T* projected;
  const T* weights;
  int64_t cols;  // f, a multiple of 4
  Act act;
  struct Row {
    const T* at;
    float w;
  };
  __device__ __forceinline__ Row row(int64_t i) const {
    return Row{projected + i * cols * (K::gated ? 2 : 1), Elem<T>::value(weights[i])};
  }
  __device__ __forceinline__ Part<T> load(const Row& r, int64_t c) const {
    constexpr bool F32 = std::is_same<T, float>::value;
    struct __attribute__((packed, aligned(sizeof(T)))) Eight {
      Part<T> p;
    };
    struct __attribute__((packed, aligned(sizeof(T)))) Four {
      T at[4];
    };
    Part<T> p{};
#pragma unroll
    for (int half = 0; half < 2; ++half) {
      const int64_t u = c + 4 * half;
      if (u >= cols) continue;
      float v[8];
      if constexpr (K::gated) {
        const Part<T> in = reinterpret_cast<const Eight*>(r.at + 2 * u)->p;
#pragma unroll
        for (int j = 0; j < 8; ++j) v[j] = Elem<T>::value(in.at[j]);
      } else {
        const Four in = *reinterpret_cast<const Four*>(r.at + u);
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          v[2 * j] = Elem<T>::value(in.at[j]);
          v[2 * j + 1] = 0.0f;
        }
      }
#pragma unroll
      for (int j = 0; j < 4; ++j)
        p.at[4 * half + j] = Elem<T>::make(glu_unit<K, F32>(act, v[2 * j], v[2 * j + 1], r.w));
    }
    return p;
  }
};

// L lanes a row of the copy's `height`: rows from `rows` or *filled on are 0. C: the row's parts
// a lane keeps, or 0 to read them twice. PLAIN: the codes row after row, not tiled.
template <typename T, int L, int C, bool PLAIN, typename Source>
__global__ __launch_bounds__(THREADS) void rows_kernel(Source from, int64_t rows, int64_t height,
                                                       const int32_t* __restrict__ filled,
                                                       int64_t cols, int64_t k,
                                                       uint8_t* __restrict__ values,
                                                       float* __restrict__ scales) {
  constexpr int TURN = 8 * L;  // columns
  const int lane = threadIdx.x % L;
  int sub = threadIdx.x / L;
  if constexpr (L == 64) sub = __builtin_amdgcn_readfirstlane(sub);
  const int64_t i = static_cast<int64_t>(blockIdx.x) * (THREADS / L) + sub;
  if (i >= height) return;
  const int64_t live = filled && *filled < rows ? *filled : rows;
  uint8_t* const out = values + i * (PLAIN ? k : 64);
  auto put = [&](int64_t c, uint2 codes) {
    const int64_t at = PLAIN ? c : (c >> 6) * (height * 64) + (c & 63);
    if (c < k) *reinterpret_cast<uint2*>(out + at) = codes;
  };
  if (i >= live) {
    for (int64_t c = 8 * lane; c < k; c += TURN) put(c, make_uint2(0, 0));
    if (lane == 0) scales[i] = 0.0f;
    return;
  }
  const typename Source::Row row = from.row(i);
  if constexpr (C > 0) {
    Part<T> p[C];
#pragma unroll
    for (int j = 0; j < C; ++j) p[j] = from.load(row, TURN * j + 8 * lane);
    uint32_t top = 0;
#pragma unroll
    for (int j = 0; j < C; ++j) {
      const uint32_t t = top_of(p[j]);
      top = t > top ? t : top;
    }
    const Coder<T> coder(row_top<L>(top));
#pragma unroll
    for (int j = 0; j < C; ++j) put(TURN * j + 8 * lane, coder.codes(p[j]));
    if (lane == 0) scales[i] = coder.scale;
  } else {
    uint32_t top = 0;
    for (int64_t c = 8 * lane; c < cols; c += TURN) {
      const uint32_t t = top_of(from.load(row, c));
      top = t > top ? t : top;
    }
    const Coder<T> coder(row_top<L>(top));
    for (int64_t c = 8 * lane; c < k; c += TURN) put(c, coder.codes(from.load(row, c)));
    if (lane == 0) scales[i] = coder.scale;
  }
}

template <typename T, int L, int C, bool PLAIN = false, typename Source>
int launch_rows(const char* kernel, const Source& from, int64_t rows, int64_t height,
                const int32_t* filled, int64_t cols, uint8_t* values, float* scales,
                hipStream_t s) {
  const int64_t k = ceil_div(cols, 128) * 128;
  hipLaunchKernelGGL((rows_kernel<T, L, C, PLAIN, Source>),
                     dim3(static_cast<unsigned>(ceil_div(height, THREADS / L))), dim3(THREADS), 0,
                     s, from, rows, height, filled, cols, k, values, scales);
  return launched(kernel);
}

// Calls f(L, C) for rows of `cols` columns: narrow ones 4 a wave, whose chains of loads and
// exchanges overlap (99320 rows of 134 bfloat16 columns: a wave each 40 us, so 15; from 1024
// columns on 16 lanes are slower, 19276 float32 rows of 1024 26 us and 19).
template <typename F>
int with_lanes(int64_t cols, F&& f) {
  using std::integral_constant;
  if (cols <= 256) return f(integral_constant<int, 16>{}, integral_constant<int, 2>{});
  if (cols <= 512) return f(integral_constant<int, 16>{}, integral_constant<int, 4>{});
  if (cols <= 1024) return f(integral_constant<int, 64>{}, integral_constant<int, 2>{});
  if (cols <= 2048) return f(integral_constant<int, 64>{}, integral_constant<int, 4>{});
  if (cols <= 4096) return f(integral_constant<int, 64>{}, integral_constant<int, 8>{});
  if (cols <= 8192) return f(integral_constant<int, 64>{}, integral_constant<int, 16>{});
  return f(integral_constant<int, 64>{}, integral_constant<int, 0>{});
}

// Rows by index from tokens quantized once (codes (sources, k) row after row, and their scales).
// A workgroup moves 128 codes of 256 rows: loads of 64-byte runs, two a token's line, stores of 1
// KiB in one run. The workgroups go through all rows for one 128 of K after another, an XCD (a
// workgroup's id modulo 8) a contiguous share, so that those 128 bytes of every token stay in
// its L2 for all of the token's rows.
constexpr int GATHERED = 256;
typedef uint32_t Word4 __attribute__((ext_vector_type(4)));
__global__ __launch_bounds__(THREADS) void gather_kernel(
    const uint8_t* __restrict__ codes, const float* __restrict__ from_scales,
    const int32_t* __restrict__ index, int32_t index_div, int64_t sources, int64_t rows,
    int64_t height, const int32_t* __restrict__ filled, int64_t k, int64_t row_blocks,
    int64_t share, uint8_t* __restrict__ values, float* __restrict__ scales) {
  const int64_t item = (blockIdx.x % 8) * share + blockIdx.x / 8;
  const int64_t pair = item / row_blocks;
  if (pair >= k / 128) return;
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, piece = 16 * (lane & 3);
  const int64_t live = filled && *filled < rows ? *filled : rows;
  const int64_t i0 = item % row_blocks * GATHERED + wave * 64 + (lane >> 2);
  constexpr int U = 4;  // of 16 rows
  int64_t token[U];
#pragma unroll
  for (int u = 0; u < U; ++u) {
    const int64_t i = i0 + 16 * u;
    const int32_t pick = i < live ? index[i] : -1;
    token[u] = pick < 0 ? -1 : pick / index_div;
    if (token[u] >= sources) token[u] = -1;
  }
  uint4 v[U][2];
#pragma unroll
  for (int u = 0; u < U; ++u)
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      v[u][h] = make_uint4(0, 0, 0, 0);
      if (token[u] >= 0)
        v[u][h] = *reinterpret_cast<const uint4*>(codes + token[u] * k + pair * 128 + 64 * h + piece);
    }
#pragma unroll
  for (int u = 0; u < U; ++u) {
    const int64_t i = i0 + 16 * u;
    if (i >= height) continue;
#pragma unroll
    for (int h = 0; h < 2; ++h)
      __builtin_nontemporal_store(
          __builtin_bit_cast(Word4, v[u][h]),
          reinterpret_cast<Word4*>(values + (2 * pair + h) * (height * 64) + i * 64 + piece));
    if (pair == 0 && piece == 0) scales[i] = token[u] >= 0 ? from_scales[token[u]] : 0.0f;
  }
}

// --- the kernels' columns ------------------------------------------------------------------

// A workgroup 64 columns of a group's (k, n) matrix: each wave every 4th row of it, a lane a
// column; then 64 rows at a time through LDS, so that a lane writes 16 bytes of a column. Two passes
// over w, in loads of 2 bytes a lane: 128 bfloat16 kernels of 2048 x 1536 724 us, where their 1.2 GB
// take 195 at 6.2 TB/s, once as they are loaded.
constexpr int PITCH = 80;  // bytes of a column's 64 codes in LDS, 16-byte aligned
template <typename T>
__global__ __launch_bounds__(THREADS) void columns_kernel(const T* __restrict__ w, int64_t cols,
                                                          int64_t n, int64_t k,
                                                          uint8_t* __restrict__ values,
                                                          float* __restrict__ scales) {
  __shared__ uint32_t tops[THREADS / 64][64];
  __shared__ __align__(16) uint8_t tile[64 * PITCH];
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const int64_t col_blocks = (n + 63) / 64;
  const int64_t g = blockIdx.x / col_blocks, c = (blockIdx.x % col_blocks) * 64 + lane;
  const T* const from = w + g * cols * n + (c < n ? c : n - 1);
  uint32_t top = 0;
#pragma unroll 8
  for (int64_t r = wave; r < cols; r += 4) {
    const uint32_t b = __float_as_uint(Elem<T>::value(from[r * n])) & 0x7fffffffu;
    top = b > top ? b : top;
  }
  tops[wave][lane] = top;
  __syncthreads();
#pragma unroll
  for (int j = 0; j < THREADS / 64; ++j) top = tops[j][lane] > top ? tops[j][lane] : top;
  const Coder<T> coder(top);
  if (wave == 0 && c < n) scales[g * n + c] = coder.scale;
  uint8_t* const out = values + g * n * k;
  const int64_t c0 = c - lane;
  for (int64_t r0 = 0; r0 < k; r0 += 64) {
#pragma unroll
    for (int q = 0; q < 4; ++q) {  // this wave's 16 of the 64 rows, 4 a word
      uint32_t word = 0;
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const int64_t r = r0 + wave * 16 + q * 4 + j;
        const float x = r < cols ? Elem<T>::value(from[r * n]) : 0.0f;
        word |= (coder.code(x) & 0xffu) << (8 * j);
      }
      *reinterpret_cast<uint32_t*>(tile + lane * PITCH + wave * 16 + q * 4) = word;
    }
    __syncthreads();
    const int column = threadIdx.x >> 2, piece = threadIdx.x & 3;
    if (c0 + column < n)
      *reinterpret_cast<uint4*>(out + (r0 >> 6) * (n * 64) + (c0 + column) * 64 + piece * 16) =
          *reinterpret_cast<const uint4*>(tile + column * PITCH + piece * 16);
    __syncthreads();
  }
}

int check_copy(const char* name, int64_t rows, int64_t cols, int64_t height) {
  // a launch holds fewer than 2^32 threads, a row's 64 of them
  BUX_CHECK(rows >= 0 && height >= rows && height <= MAX_HEIGHT,
            "%s: bad shape rows=%lld height=%lld (at least the rows, up to %lld)", name,
            (long long)rows, (long long)height, (long long)MAX_HEIGHT);
  BUX_CHECK(cols > 0 && cols <= MAX_K, "%s: cols=%lld outside [1, %lld]", name, (long long)cols,
            (long long)MAX_K);
  return BUX_OK;
}

// The bytes of the tokens' own codes and scales, or 0 where rows are quantized one by one: few
// codes, whose second launch costs more than it saves, or not twice as many rows as tokens.
// us, each row quantized from its token and each token once (bfloat16; float32):
//   4096 tokens of 2048, 4 rows each   21  19;   30  23      1024 of 7168, 4   19  22;   49  31
//   16384 of 2048, 2                   38  39;   55  51      1024 of 7168, 8   34  27;   88  36
//   16384 of 2048, 8                  137  71;  192  83      16384 of 7168, 8 590 240; 1261 421
//   16384 of 512, 4                    21  22;   31  23      4096 of 512, 8    12  11;   19  14
//   12415 of 990, 8                    52  32;   88  37      12415 of 134, 8   15  15;   24  18
size_t gather_workspace(int64_t sources, int64_t rows, int64_t cols) {
  if (rows < 2 * sources || rows * cols < (1LL << 25)) return 0;
  return static_cast<size_t>(sources) * (ceil_div(cols, 128) * 128 + sizeof(float));
}

template <typename T>
int quantize(const char* name, const T* x, const int32_t* index, int32_t index_div,
             int64_t sources, int64_t rows, int64_t cols, int64_t height, const int32_t* filled,
             uint8_t* values, float* scales, void* workspace, size_t workspace_bytes,
             void* stream) {
  if (int rc = check_copy(name, rows, cols, height)) return rc;
  BUX_CHECK(index == nullptr || (index_div >= 1 && sources >= 0), "%s: index_div=%d sources=%lld",
            name, index_div, (long long)sources);
  if (height == 0) return BUX_OK;
  BUX_CHECK(values && scales && (rows == 0 || x || (index && sources == 0)), "%s: NULL buffer",
            name);
  hipStream_t s = as_stream(stream);
  const size_t need = index ? gather_workspace(sources, rows, cols) : 0;
  const bool gathered = need > 0;
  if (gathered && (workspace == nullptr || workspace_bytes < need))
    return fail(BUX_E_WORKSPACE, "%s: workspace of %zu bytes, %zu needed", name, workspace_bytes,
                need);
  const int64_t k = ceil_div(cols, 128) * 128;
  const int64_t row_blocks = ceil_div(height, GATHERED), share = ceil_div(row_blocks * (k / 128), 8);
  BUX_CHECK(!gathered || 8 * share * THREADS < (1LL << 32),
            "%s: height=%lld rows of cols=%lld are more than a launch holds", name,
            (long long)height, (long long)cols);
  BUX_CHECK(!gathered || reinterpret_cast<uintptr_t>(workspace) % 16 == 0,
            "%s: the workspace is 16-byte aligned", name);
  uint8_t* const codes = static_cast<uint8_t*>(workspace);
  float* const own = reinterpret_cast<float*>(codes + (gathered ? sources * k : 0));
  auto go = [&](auto lanes, auto c, auto load) {
    constexpr int L = decltype(lanes)::value, C = decltype(c)::value;
    const Rows<T, decltype(load)::value> from{x, gathered ? nullptr : index, index_div, sources,
                                              cols};
    if (gathered)  // every token, row after row
      return launch_rows<T, L, C, true>("int8 rows_kernel", from, sources, sources, nullptr, cols,
                                        codes, own, s);
    return launch_rows<T, L, C>("int8 rows_kernel", from, rows, height, filled, cols, values,
                                scales, s);
  };
  auto quantized = [&] {
    using std::integral_constant;
    if (cols < 8)
      return go(integral_constant<int, 16>{}, integral_constant<int, 0>{},
                integral_constant<Load, Load::NARROW>{});
    return with_lanes(cols, [&](auto lanes, auto c) {
      return cols % 8 == 0 ? go(lanes, c, integral_constant<Load, Load::WHOLE>{})
                           : go(lanes, c, integral_constant<Load, Load::TAIL>{});
    });
  };
  if (int rc = quantized(); rc != BUX_OK || !gathered) return rc;
  hipLaunchKernelGGL(gather_kernel, dim3(static_cast<unsigned>(8 * share)), dim3(THREADS), 0, s,
                     codes, own, index, index_div, sources, rows, height, filled, k, row_blocks,
                     share, values, scales);
  return launched("int8 gather_kernel");
}

template <typename T>
int quantize_units(const char* name, const T* projected, const T* weights, const int32_t* filled,
                   int64_t m, int64_t f, const bux_ffn* ffn, int64_t height, uint8_t* values,
                   float* scales, void* stream) {
  if (int rc = check_copy(name, m, f, height)) return rc;
  BUX_CHECK(f % 4 == 0, "%s: f=%lld is not a multiple of 4", name, (long long)f);
  Act act;
  if (int rc = act_of(name, ffn, &act)) return rc;
  if (height == 0) return BUX_OK;
  BUX_CHECK(values && scales && (m == 0 || (projected && weights)), "%s: NULL buffer", name);
  return with_kind(act, [&](auto kind) {
    const Units<decltype(kind), T> from{projected, weights, f, act};
    auto go = [&](auto c) {
      return launch_rows<T, 64, decltype(c)::value>("int8 units rows_kernel", from, m, height,
                                                    filled, f, values, scales, as_stream(stream));
    };
    if (f <= 1024) return go(std::integral_constant<int, 2>{});
    if (f <= 4096) return go(std::integral_constant<int, 8>{});
    return go(std::integral_constant<int, 0>{});
  });
}

template <typename T>
int quantize_columns(const char* name, const T* w, int64_t groups, int64_t k, int64_t n,
                     uint8_t* values, float* scales, void* stream) {
  BUX_CHECK(groups >= 0 && n > 0 && k > 0 && k <= MAX_K && groups * ceil_div(n, 64) < (1LL << 24),
            "%s: bad shape groups=%lld k=%lld n=%lld (k up to %lld)", name, (long long)groups,
            (long long)k, (long long)n, (long long)MAX_K);
  if (groups == 0) return BUX_OK;
  BUX_CHECK(w && values && scales, "%s: NULL buffer", name);
  hipLaunchKernelGGL((columns_kernel<T>), dim3(static_cast<unsigned>(groups * ceil_div(n, 64))),
                     dim3(THREADS), 0, as_stream(stream), w, k, n, ceil_div(k, 128) * 128, values,
                     scales);
  return launched("int8 columns_kernel");
}

}  // namespace
}  // namespace bux

extern "C" size_t bux_int8_quantize_workspace_size(int64_t sources, int64_t rows, int64_t cols) {
  return sources < 0 || rows < 0 || cols <= 0 ? 0 : bux::gather_workspace(sources, rows, cols);
}
extern "C" int bux_int8_quantize(const uint16_t* x, const int32_t* index, int32_t index_div,
                                 int64_t sources, int64_t rows, int64_t cols, int64_t height,
                                 const int32_t* filled, uint8_t* values, float* scales,
                                 void* workspace, size_t workspace_bytes, void* stream) {
  bux::clear_error();
  return bux::quantize("bux_int8_quantize", x, index, index_div, sources, rows, cols, height,
                       filled, values, scales, workspace, workspace_bytes, stream);
}
extern "C" int bux_int8_quantize_f32(const float* x, const int32_t* index, int32_t index_div,
                                     int64_t sources, int64_t rows, int64_t cols, int64_t height,
                                     const int32_t* filled, uint8_t* values, float* scales,
                                     void* workspace, size_t workspace_bytes, void* stream) {
  bux::clear_error();
  return bux::quantize("bux_int8_quantize_f32", x, index, index_div, sources, rows, cols, height,
                       filled, values, scales, workspace, workspace_bytes, stream);
}
extern "C" int bux_int8_glu(const uint16_t* projected, const uint16_t* weights,
                            const int32_t* filled, int64_t m, int64_t f, const bux_ffn* ffn,
                            int64_t height, uint8_t* values, float* scales, void* stream) {
  bux::clear_error();
  return bux::quantize_units("bux_int8_glu", projected, weights, filled, m, f, ffn, height, values,
                             scales, stream);
}
extern "C" int bux_int8_glu_f32(const float* projected, const float* weights,
                                const int32_t* filled, int64_t m, int64_t f, const bux_ffn* ffn,
                                int64_t height, uint8_t* values, float* scales, void* stream) {
  bux::clear_error();
  return bux::quantize_units("bux_int8_glu_f32", projected, weights, filled, m, f, ffn, height,
                             values, scales, stream);
}
extern "C" int bux_int8_quantize_columns(const uint16_t* w, int64_t groups, int64_t k, int64_t n,
                                         uint8_t* values, float* scales, void* stream) {
  bux::clear_error();
  return bux::quantize_columns("bux_int8_quantize_columns", w, groups, k, n, values, scales, stream);
}
extern "C" int bux_int8_quantize_columns_f32(const float* w, int64_t groups, int64_t k, int64_t n,
                                             uint8_t* values, float* scales, void* stream) {
  bux::clear_error();
  return bux::quantize_columns("bux_int8_quantize_columns_f32", w, groups, k, n, values, scales,
                               stream);
}
