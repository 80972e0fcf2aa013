// Dense bfloat16 products of few rows (a decode step's): bound by w's bytes from HBM.
//
// A workgroup makes 64 columns, whole 128-byte lines of w's rows, over a part of K: 8 waves take
// its steps of 32 K in turn, each with v_mfma_f32_16x16x32_bf16 on its own ring of LDS, filled RING
// steps ahead by direct loads (no barrier in the loop), and their sums meet in LDS at the end, in
// order. K goes in as many parts as fill the chip; a second kernel (join_kernel) adds the parts'
// sums in order, with the epilogue. (16 columns over all of K, one launch, came to 1.9 TB/s: a
// request a 32-byte piece.)
//   w          [32 K rows][128 bytes], chunk c (16 bytes) of K row k at place c ^ 2 (k / 2 % 2) ^
//              4 (k / 8 % 2), read by ds_read_b64_tr_b16; w transposed: as x
//   x          blocks of [16 rows][64 bytes], chunk c of row r at place c ^ (r / 4 % 4)
// Rows past x's read 0; so do the steps past a part's end, which keep the loads in flight counted.

#include "dense.h"

namespace bux {
using namespace dense;
namespace {

typedef __bf16 v8bf __attribute__((ext_vector_type(8)));
typedef short v4s __attribute__((ext_vector_type(4)));
typedef float f32x4 __attribute__((ext_vector_type(4)));
typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));
typedef __attribute__((address_space(3))) v4s lds_v4s;
typedef __attribute__((address_space(3))) uint4 lds_u4;

constexpr int WAVES = 8;
constexpr int THREADS = 64 * WAVES;
constexpr int COLUMNS = 64;
constexpr int BLOCKS_N = COLUMNS / 16;
constexpr int STEP = 32;  // K

// How far ahead a wave loads: 8 rings fill most of a CU's 160 KiB.
template <int BLOCKS>
constexpr int RING = BLOCKS == 1 ? 4 : BLOCKS == 2 ? 3 : 2;

template <int N>
__device__ __forceinline__ void wait_loads() {
  asm volatile("s_waitcnt vmcnt(%0)" ::"n"(N) : "memory");
}

// BLOCKS: 16 rows of x each. Part `id / groups` of K: `part` steps of it.
template <bool BKM, int BLOCKS, typename Epi>
__global__ __launch_bounds__(THREADS) void few_kernel(const uint16_t* __restrict__ x,
                                                      const uint16_t* __restrict__ w, int32_t m,
                                                      int32_t n, int32_t k, int32_t groups,
                                                      int32_t part, int32_t count, Epi epi) {
  constexpr int R = RING<BLOCKS>;
  constexpr int LOADS = BLOCKS_N + BLOCKS;  // 1 KiB each, of a step
  constexpr int BYTES = LOADS * 1024;
  extern __shared__ __align__(16) uint8_t lds[];
  const int32_t per = (count + 7) / 8;
  const int32_t id = static_cast<int32_t>(blockIdx.x % 8) * per + static_cast<int32_t>(blockIdx.x / 8);
  if (static_cast<int32_t>(blockIdx.x / 8) >= per || id >= count) return;
  const int32_t split = id / groups, col = (id - split * groups) * COLUMNS;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), lane = threadIdx.x & 63;
  const uint32_t ring = lds_at(lds) + wave * (R * BYTES);
  const int32_t all = (k + STEP - 1) / STEP, first = split * part;
  const int32_t steps = all - first < part ? all - first : part;
  const int32_t mine = (steps + WAVES - 1) / WAVES;

  // x's and w transposed's loads: row l / 4 of a block, place l % 4; w's load j: K row 8 j + l / 8,
  // place l % 8
  const int chunk = (lane & 3) ^ ((lane >> 4) & 3);
  i32x4 ra = resource(x, static_cast<int64_t>(m) * k * 2);
  i32x4 rb = resource(w, static_cast<int64_t>(n) * k * 2);
  const int32_t va = (lane >> 2) * k * 2 + 16 * chunk;
  const int32_t vb = BKM ? (col + (lane >> 2)) * k * 2 : (lane >> 3) * n * 2 + col * 2;
  const int32_t in_row = BKM ? chunk : (lane & 7) ^ (2 * ((lane >> 4) & 1));
  const int32_t a_bytes = ra[2], b_bytes = rb[2];
  auto load = [&](int32_t i, int slot) {
    const int32_t t = i * WAVES + wave, s = first + t;
    ra[2] = t < steps ? a_bytes : 0;
    rb[2] = t < steps ? b_bytes : 0;
    const uint32_t at = ring + slot * BYTES;
#pragma unroll
    for (int j = 0; j < BLOCKS_N; ++j) {
      if constexpr (BKM)
        load_lds16(rb, at + j * 1024, vb + 16 * in_row, s * (STEP * 2) + j * 16 * k * 2);
      else  // rows 8 j ..: their k / 8 is j's
        load_lds16(rb, at + j * 1024, vb + 16 * (in_row ^ (4 * (j & 1))),
                           (s * STEP + 8 * j) * n * 2);
    }
#pragma unroll
    for (int b = 0; b < BLOCKS; ++b)
      load_lds16(ra, at + (BLOCKS_N + b) * 1024, va, s * (STEP * 2) + b * 16 * k * 2);
  };

  const int g = lane >> 4, r = lane & 15;
  const uint32_t km = r * 64 + 16 * (g ^ (r >> 2));  // K-major operands
  // w's block j, the first read: K rows 8 g + r / 4, columns 16 j + 4 (r % 4); the second 4 rows on
  uint32_t tr[BLOCKS_N];
#pragma unroll
  for (int j = 0; j < BLOCKS_N; ++j)
    tr[j] = (8 * g + (r >> 2)) * 128 +
            16 * ((2 * j + ((r >> 1) & 1)) ^ (2 * ((r >> 3) & 1)) ^ (4 * (g & 1))) + 8 * (r & 1);
  f32x4 acc[BLOCKS][BLOCKS_N];
#pragma unroll
  for (int b = 0; b < BLOCKS; ++b)
#pragma unroll
    for (int j = 0; j < BLOCKS_N; ++j) acc[b][j] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
  for (int i = 0; i < R; ++i) load(i, i);
  int slot = 0;
  for (int32_t i = 0; i < mine; ++i) {
    wait_loads<(R - 1) * LOADS>();
    const uint32_t at = ring + slot * BYTES;
    v8bf wv[BLOCKS_N], xv[BLOCKS];
#pragma unroll
    for (int j = 0; j < BLOCKS_N; ++j) {
      if constexpr (BKM) {
        wv[j] = __builtin_bit_cast(v8bf, *reinterpret_cast<const lds_u4*>(at + j * 1024 + km));
      } else {
        const v4s p = __builtin_amdgcn_ds_read_tr16_b64_v4i16(reinterpret_cast<lds_v4s*>(at + tr[j]));
        const v4s q =
            __builtin_amdgcn_ds_read_tr16_b64_v4i16(reinterpret_cast<lds_v4s*>(at + tr[j] + 512));
        wv[j] = __builtin_bit_cast(v8bf, __builtin_shufflevector(p, q, 0, 1, 2, 3, 4, 5, 6, 7));
      }
    }
#pragma unroll
    for (int b = 0; b < BLOCKS; ++b)
      xv[b] = __builtin_bit_cast(
          v8bf, *reinterpret_cast<const lds_u4*>(at + (BLOCKS_N + b) * 1024 + km));
    // the reads are done before the slot's next loads
    asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
    load(i + R, slot);
    const int32_t left = k - (first + i * WAVES + wave) * STEP;
    if (left < STEP) {  // K positions past k count 0 in both operands
      auto cut = [&](v8bf v) {
        u32x4 u = __builtin_bit_cast(u32x4, v);
#pragma unroll
        for (int d = 0; d < 4; ++d) {
          const int32_t at_k = 8 * g + 2 * d;
          u[d] &= (at_k < left ? 0xffffu : 0u) | (at_k + 1 < left ? 0xffff0000u : 0u);
        }
        return __builtin_bit_cast(v8bf, u);
      };
#pragma unroll
      for (int j = 0; j < BLOCKS_N; ++j) wv[j] = cut(wv[j]);
#pragma unroll
      for (int b = 0; b < BLOCKS; ++b) xv[b] = cut(xv[b]);
    }
#pragma unroll
    for (int b = 0; b < BLOCKS; ++b)
#pragma unroll
      for (int j = 0; j < BLOCKS_N; ++j)
        acc[b][j] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(wv[j], xv[b], acc[b][j], 0, 0, 0);
    slot = slot + 1 == R ? 0 : slot + 1;
  }
  // Every wave's loads have landed before the rings are reused. Lane l has row l % 16 of block b and
  // columns 4 (l / 16) .. + 3 of block j; a row's sums are 16 bytes more than its 64 columns apart.
  wait_loads<0>();
  __syncthreads();
  constexpr int PITCH = COLUMNS + 4;
  float* const sums = reinterpret_cast<float*>(lds);
#pragma unroll
  for (int b = 0; b < BLOCKS; ++b)
#pragma unroll
    for (int j = 0; j < BLOCKS_N; ++j)
      *reinterpret_cast<f32x4*>(sums + ((wave * BLOCKS + b) * 16 + r) * PITCH + 16 * j + 4 * g) =
          acc[b][j];
  __syncthreads();
  const int t = threadIdx.x;  // a row's 8 columns each
  const int32_t row = t >> 3, c = 8 * (t & 7);
  if (t >= BLOCKS * 128 || row >= m || col + c >= n) return;
  Epi mine_epi = epi;
  if constexpr (std::is_same<Epi, Partial>::value)
    mine_epi.out += static_cast<int64_t>(split) * m * epi.pitch;
  const typename Epi::In in = mine_epi.load(row, col + c);
  float v[8] = {};
#pragma unroll
  for (int u = 0; u < WAVES; ++u) {
    const float* const p = sums + (u * BLOCKS * 16 + row) * PITCH + c;
#pragma unroll
    for (int j = 0; j < 8; ++j) v[j] += p[j];
  }
  mine_epi.choose([&](auto kind) { mine_epi.store(kind, row, col + c, v, in); });
}

template <bool BKM, int BLOCKS, typename Epi>
int launch(const uint16_t* x, const uint16_t* w, int64_t m, int64_t n, int64_t k, int64_t splits,
           const Epi& epi, hipStream_t s) {
  constexpr int RINGS = WAVES * RING<BLOCKS> * (BLOCKS_N + BLOCKS) * 1024;
  constexpr int SUMS = WAVES * BLOCKS * 16 * (COLUMNS + 4) * 4;
  constexpr int BYTES = RINGS > SUMS ? RINGS : SUMS;
  static_assert(BYTES <= 160 * 1024, "a CU's LDS");
  const int64_t groups = ceil_div(n, COLUMNS), count = groups * splits;
  const int64_t part = ceil_div(ceil_div(k, STEP), splits);
  auto kernel = few_kernel<BKM, BLOCKS, Epi>;
  const hipError_t err = hipFuncSetAttribute(reinterpret_cast<const void*>(kernel),
                                             hipFuncAttributeMaxDynamicSharedMemorySize, BYTES);
  if (err != hipSuccess) return fail(BUX_E_LAUNCH, "dense few_kernel: %s", hipGetErrorString(err));
  hipLaunchKernelGGL(kernel, dim3(static_cast<unsigned>(8 * ceil_div(count, 8))), dim3(THREADS),
                     BYTES, s, x, w, static_cast<int32_t>(m), static_cast<int32_t>(n),
                     static_cast<int32_t>(k), static_cast<int32_t>(groups),
                     static_cast<int32_t>(part), static_cast<int32_t>(count), epi);
  return launched("dense few_kernel");
}

}  // namespace

namespace dense {

bool few_takes(const Mat<uint16_t>& A, const Mat<uint16_t>& B, int64_t m, int64_t n, int64_t k) {
  // direct loads of whole 16-byte chunks at 32-bit offsets, the columns and a ring of steps past
  // the operands' ends included
  const int64_t past = 8 * STEP * WAVES;
  return m <= 64 && A.ld == k && k % 8 == 0 && n % 8 == 0 &&
         reinterpret_cast<uintptr_t>(A.p) % 16 == 0 && reinterpret_cast<uintptr_t>(B.p) % 16 == 0 &&
         (n + COLUMNS) * (k + past) * 2 < (1LL << 31) && (m + 64) * (k + past) * 2 < (1LL << 31);
}

// Parts of K: a workgroup a CU, as long as a part has two steps a wave; one where the columns
// alone come to three quarters of that (a second kernel takes as long as they gain).
int64_t few_splits(int64_t n, int64_t k) {
  const int64_t groups = ceil_div(n, COLUMNS);
  if (groups >= 192) return 1;
  const int64_t most = ceil_div(k, STEP * WAVES * 2);
  int64_t s = 256 / groups;
  s = s < most ? s : most;
  // no part without steps
  const int64_t steps = ceil_div(k, STEP);
  return s < 1 ? 1 : ceil_div(steps, ceil_div(steps, s));
}

template <bool BKM, typename Epi>
int launch_few(const Mat<uint16_t>& A, const Mat<uint16_t>& B, int64_t m, int64_t n, int64_t k,
               int64_t splits, const Epi& epi, hipStream_t s) {
  if (m <= 16) return launch<BKM, 1>(A.p, B.p, m, n, k, splits, epi, s);
  if (m <= 32) return launch<BKM, 2>(A.p, B.p, m, n, k, splits, epi, s);
  if (m <= 48) return launch<BKM, 3>(A.p, B.p, m, n, k, splits, epi, s);
  return launch<BKM, 4>(A.p, B.p, m, n, k, splits, epi, s);
}

#define BUX_FEW(B, ...)                                                                        \
  template int launch_few<B, __VA_ARGS__>(const Mat<uint16_t>&, const Mat<uint16_t>&, int64_t, \
                                          int64_t, int64_t, int64_t, const __VA_ARGS__&, hipStream_t)
BUX_FEW(false, Forward<uint16_t, false>);
BUX_FEW(false, Forward<uint16_t, true>);
BUX_FEW(false, Partial);
BUX_FEW(true, Forward<uint16_t, false>);
BUX_FEW(true, Forward<uint16_t, true>);
BUX_FEW(true, Backward<uint16_t, false>);
BUX_FEW(true, Backward<uint16_t, true>);
BUX_FEW(true, Partial);

}  // namespace dense
}  // namespace bux
