// The 8-bit product for groups of few rows (a decode step, a short prompt): grouped_int8.hip's y
// to the bit, for calls whose time is reading the experts' kernels.
//
// A workgroup takes 16 or 32 rows by 64 columns, its 2 waves a half of K each (integer sums are
// exact, so that their order is free): v_mfma_i32_16x16x64_i8, whose lanes take of 16 rows' 64
// bytes of K, in the tiled layout one run of 1 KiB, 16 bytes each; operands straight from global
// memory to registers, P chunks of K at once and the next P behind them. The halves meet in LDS,
// where 16 threads a row add, scale and store.
//
// What bounds it is each CU's loads in flight, which waves and chunks carry. 128 kernels of K
// 2048, N 1536, in us for one wave a tile, two, four, and one with twice the chunks (64 rows on
// 43 of them; 320 on 100; 1608 on 118, the most 104): 31.5, 30.1, 31.6, 31.7; 59.9, 61.1, 66.3,
// 68.3; 89, 80, 94, 123: two, 5.2 TB/s. All of a tile's rows in one workgroup, in turn, was slower
// (crowded tiles last), and non-temporal loads of the kernels no faster.

#include "int8_direct.h"

#include "tiles.h"

namespace bux {
namespace {

typedef int v4i __attribute__((ext_vector_type(4)));

constexpr int COLS = 64;
constexpr int CB = COLS / 16;
constexpr int S = 2;             // waves a tile, each its part of K
constexpr int P = 2;             // chunks of 64 K loaded at once
constexpr int PITCH = COLS + 4;  // ints: rows 16 bytes past a multiple of the banks

template <typename T>
__device__ __forceinline__ void store4(T* at, const float (&v)[4]) {
  if constexpr (sizeof(T) == 2)
    *reinterpret_cast<uint2*>(at) = make_uint2(pack_bf16x2(v[0], v[1]), pack_bf16x2(v[2], v[3]));
  else
    *reinterpret_cast<float4*>(at) = make_float4(v[0], v[1], v[2], v[3]);
}

template <typename T, int R>
__device__ __forceinline__ void split_tile(const uint8_t* a, const float* a_scales,
                                           const uint8_t* b, const float* b_scales, int32_t a_rows,
                                           int32_t n, int32_t chunks, int64_t row0, int64_t end,
                                           int32_t col0, const T* bias, T* y, int32_t* lds) {
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int lane = threadIdx.x & 63;
  const int quarter = lane >> 4, r16 = lane & 15;
  const int64_t a_chunk = static_cast<int64_t>(a_rows) * 64, b_chunk = static_cast<int64_t>(n) * 64;
  uint32_t at_a[R], at_b[CB];  // rows past an operand's: its last one's again (a's count as 0)
#pragma unroll
  for (int i = 0; i < R; ++i) {
    const int64_t row = row0 + 16 * i + r16;
    at_a[i] = static_cast<uint32_t>(row < a_rows ? row : a_rows - 1) * 64 + 16 * quarter;
  }
#pragma unroll
  for (int j = 0; j < CB; ++j)
    at_b[j] = static_cast<uint32_t>(smaller(col0 + 16 * j + r16, n - 1)) * 64 + 16 * quarter;
  v4i acc[R][CB];
#pragma unroll
  for (int i = 0; i < R; ++i)
#pragma unroll
    for (int j = 0; j < CB; ++j) acc[i][j] = v4i{};
  struct Batch {
    v4i a[P][R], b[P][CB];
  };
  const int32_t lo = chunks * wave / S, hi = chunks * (wave + 1) / S;
  auto load = [&](Batch& s, int32_t c) {
#pragma unroll
    for (int u = 0; u < P; ++u) {
      if (c + u >= hi) break;
#pragma unroll
      for (int j = 0; j < CB; ++j)
        s.b[u][j] = *reinterpret_cast<const v4i*>(b + (c + u) * b_chunk + at_b[j]);
#pragma unroll
      for (int i = 0; i < R; ++i)
        s.a[u][i] = *reinterpret_cast<const v4i*>(a + (c + u) * a_chunk + at_a[i]);
    }
  };
  auto multiply = [&](const Batch& s, int32_t c) {
#pragma unroll
    for (int u = 0; u < P; ++u) {
      if (c + u >= hi) break;
#pragma unroll
      for (int i = 0; i < R; ++i)
#pragma unroll
        for (int j = 0; j < CB; ++j)
          acc[i][j] = __builtin_amdgcn_mfma_i32_16x16x64_i8(s.b[u][j], s.a[u][i], acc[i][j], 0, 0, 0);
    }
  };
  Batch one, two;
  if (lo < hi) load(one, lo);
  for (int32_t c = lo; c < hi; c += 2 * P) {
    if (c + P < hi) load(two, c + P);
    multiply(one, c);
    if (c + 2 * P < hi) load(one, c + 2 * P);
    if (c + P < hi) multiply(two, c + P);
  }
  // four columns' outputs: the sums times both scales, plus the bias, rounded once
  auto put = [&](int r, int c, v4i sum) {
#pragma clang fp contract(off)
    const int64_t row = row0 + r;
    const int32_t col = col0 + c;
    if (row >= end || col >= n) return;  // n is a multiple of 4
    // rows past the groups (no chunks), and those that the sizes put past a's: 0
    const bool held = chunks > 0 && row < a_rows;
    const float sa = held ? a_scales[row] : 0.0f;
    if (!held) sum = v4i{};
    float v[4];
#pragma unroll
    for (int q = 0; q < 4; ++q) {
      const float sb = chunks > 0 ? b_scales[col + q] : 0.0f;
      v[q] = static_cast<float>(sum[q]) * (sa * sb);
      if (bias != nullptr) v[q] += Elem<T>::value(bias[col + q]);
    }
    store4(y + row * n + col, v);
  };
  // lane l holds row l % 16 of a block, columns 4 (l / 16) .. + 3 of each 16
  int32_t* mine = lds + wave * (16 * R * PITCH);
#pragma unroll
  for (int i = 0; i < R; ++i)
#pragma unroll
    for (int j = 0; j < CB; ++j)
      *reinterpret_cast<v4i*>(mine + (16 * i + r16) * PITCH + 16 * j + 4 * quarter) = acc[i][j];
  __syncthreads();
  for (int at = threadIdx.x; at < 16 * R * (COLS / 4); at += 64 * S) {
    const int r = at >> 4, c = 4 * (at & 15);
    v4i sum{};
#pragma unroll
    for (int w = 0; w < S; ++w)
      sum += *reinterpret_cast<const v4i*>(lds + (w * 16 * R + r) * PITCH + c);
    put(r, c, sum);
  }
}

template <typename T>
__global__ __launch_bounds__(64 * S) __attribute__((amdgpu_waves_per_eu(3))) void rows_split_kernel(
    const uint8_t* __restrict__ a_values, const float* __restrict__ a_scales,
    const uint8_t* __restrict__ b_values, const float* __restrict__ b_scales, int32_t k,
    int32_t a_rows, int32_t n, int32_t groups, int32_t height, const int32_t* __restrict__ starts,
    const Tile* __restrict__ tiles, int32_t col_blocks, const T* __restrict__ bias,
    T* __restrict__ y) {
  __shared__ __align__(16) int32_t lds[S * 32 * PITCH];
  const int32_t id = blockIdx.x / col_blocks;
  // the record beside the list's header, not after it: a list's buffer holds every record
  const Tile t = tiles[id];
  const int32_t count = starts[groups + 1];
  if (!list_fits(starts, groups, a_rows, height) || id >= count) return;
  const int64_t row0 = t.lo + static_cast<int64_t>(blockIdx.y) * 32, end = smaller(t.hi, height);
  if (row0 >= end) return;
  const int32_t col0 = (blockIdx.x % col_blocks) * COLS;
  const bool live = t.group < groups;
  const int64_t group = live ? t.group : 0;
  const int32_t chunks = live ? k / 64 : 0;
  const uint8_t* const b = b_values + group * n * k;
  const T* const added = bias != nullptr && live ? bias + group * n : nullptr;
  if (end - row0 > 16)
    split_tile<T, 2>(a_values, a_scales, b, b_scales + group * n, a_rows, n, chunks, row0, end,
                     col0, added, y, lds);
  else
    split_tile<T, 1>(a_values, a_scales, b, b_scales + group * n, a_rows, n, chunks, row0, end,
                     col0, added, y, lds);
}

}  // namespace

// The line between the two kernels, by what the host knows: up to a block of 16 rows a group. On
// even loads rows_split_kernel gains there, less the more rows; past it rows_kernel does. Where
// rows crowd into few groups each 32 of a group read its kernel again, from L2: such a call
// loses to rows_kernel, but takes no longer than the same call with an even load, since m rows
// make at most m / 32 such reads and an even load at 16 rows a group twice as many from HBM.
// us, this and rows_kernel at 4, 8, 16, 32 rows a group on even loads; on Zipf(1.2) loads; at 16
// with all rows in a fifth of the groups:
//   128 of K 2048, N 1536  65  93   74  91    82   90   117   97;  61  88   70  89    90   99;   45  27
//   128 of K 768, N 2048   37  59   40  60    47   61    64   66;  35  48   43  60    51   65;   27  16
//   32 of K 2048, N 2048   27  33   29  33    31   33    37   33;  24  31   28  32    33   33;   14  25
//   8 of K 4096, N 7168    44  49   44  48    46   47    59   49;  44  48   45  48    49   49;   51  48
//   16 of K 6400, N 4096   67  72   68  73    83   77    99   82;  58  70   81  81    89   79;   32  60
//   256 of K 7168, N 4096 968 1184 1116 1301 1452 1448 2066 1501; 956 1110 1194 1292 1527 1476; 810 346
// (Its loads take a's last row for those past it, so there has to be one.)
bool int8_rows_direct(int64_t m, int32_t groups) {
  return m > 0 && m <= 16 * static_cast<int64_t>(groups);
}

int launch_int8_direct(const uint8_t* a_values, const float* a_scales, const uint8_t* b_values,
                       const float* b_scales, const void* list, int64_t slots, int32_t groups,
                       int64_t m, int64_t n, int64_t k, int64_t height, int out_dtype,
                       const void* bias, void* y, hipStream_t s) {
  const int64_t col_blocks = ceil_div(n, COLS);
  if (slots * col_blocks >= (1LL << 24))
    return fail(BUX_E_ARGUMENT, "bux_int8_grouped_rows_listed: too many tiles");
  const int64_t rows = m > height ? m : height;  // no tile holds more
  const dim3 grid(static_cast<unsigned>(slots * col_blocks),
                  static_cast<unsigned>(ceil_div(rows < BM ? rows : BM, 32)));
  auto go = [&](auto* out) {
    using T = std::remove_pointer_t<decltype(out)>;
    hipLaunchKernelGGL((rows_split_kernel<T>), grid, dim3(64 * S), 0, s, a_values, a_scales,
                       b_values, b_scales, static_cast<int32_t>(k), static_cast<int32_t>(m),
                       static_cast<int32_t>(n), groups, static_cast<int32_t>(height),
                       starts_in(list), tiles_in(list, groups), static_cast<int32_t>(col_blocks),
                       static_cast<const T*>(bias), out);
    return launched("int8 rows_split_kernel");
  };
  return out_dtype == BUX_BF16 ? go(static_cast<uint16_t*>(y)) : go(static_cast<float*>(y));
}

}  // namespace bux

// Which kernel a call takes, for tests alone (not in bux_amd.h: the line may move).
extern "C" int bux_int8_direct(int64_t m, int32_t groups) {
  return bux::int8_rows_direct(m, groups) ? 1 : 0;
}
