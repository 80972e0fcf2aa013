// The grouped GEMMs' epilogue where a workgroup's 256 x 256 outputs lie in its 4 waves'
// accumulators (MFMAs of 32 x 32 with B's rows first): through one stage of LDS (S, at least
// STAGING bytes) to whole rows a store instruction, rows and columns past the tile's left out.
// What an accumulator becomes is a functor's: operator()(i, j, g) the bfloat16 pairs, f32(i, j,
// g) the floats, of block (i, j)'s register run g.
#pragma once

#include <type_traits>

#include "tiles.h"

namespace bux {
namespace {

// Output stores are non-temporal: the tile is written once and read by another kernel,
// and a whole round of tiles' outputs (4 MiB an XCD in bfloat16) passing through the
// XCD's 4 MiB L2 would evict the operands the other CUs are about to reuse.
typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));
typedef uint32_t u32x2 __attribute__((ext_vector_type(2)));
constexpr int NT = 2;  // a buffer store's cache policy: non-temporal
__device__ __forceinline__ void stream16(void* at, uint4 v) {
  __builtin_nontemporal_store(u32x4{v.x, v.y, v.z, v.w}, reinterpret_cast<u32x4*>(at));
}
__device__ __forceinline__ void stream8(void* at, uint32_t x, uint32_t y) {
  __builtin_nontemporal_store(u32x2{x, y}, reinterpret_cast<u32x2*>(at));
}

// float32 through the wave's region of the stage, 32 rows x 64 columns (a row's 256 bytes,
// rows 272 apart) at a time: read back 16 bytes a lane, 16 lanes a row, a store writes
// 4 whole rows of 256 bytes. (Straight from the accumulators a store instruction wrote
// 32 rows of 32 bytes: config 3's up wgrad into float32, 1.6 GB of outputs, took 1528 us,
// this way 575.) I, J: the wave's blocks of 32 rows and columns, its first row and column
// row0 and col0 of the tile; the rows [0, rows) and columns [0, cols) are stored (cols a
// multiple of 4).
template <int I, int J, typename Values, typename S>
__device__ void store_f32(const Values& values, float* tile, int32_t ld, int32_t rows, int32_t cols,
                          int32_t row0, int32_t col0, S& stage) {
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  constexpr int FP = 272;
  uint8_t* region = reinterpret_cast<uint8_t*>(&stage) + wave * 32 * FP;
  uint8_t* mine = region + (lane & 31) * FP + 16 * (lane >> 5);
  const int cc = lane & 15;
  const uint8_t* from = region + (lane >> 4) * FP + cc * 16;
  // a lane's first output, its others a scalar offset away: an address a row took 90
  // registers, which went to scratch memory (the contract above 609 us with them)
  float* const out = tile + (row0 + (lane >> 4)) * ld + col0 + 4 * cc;
  float4 bias[J / 2];
  if constexpr (Values::BIASED) {
#pragma unroll
    for (int jj = 0; jj < J; jj += 2) bias[jj / 2] = values.bias4(col0 + jj * 32 + 4 * cc, cols);
  }
#pragma unroll
  for (int i = 0; i < I; ++i)
#pragma unroll
    for (int jj = 0; jj < J; jj += 2) {
#pragma unroll
      for (int b = 0; b < 2; ++b)
#pragma unroll
        for (int g = 0; g < 4; ++g)
          *reinterpret_cast<float4*>(mine + b * 128 + g * 32) = values.f32(i, jj + b, g);
      asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
      __builtin_amdgcn_wave_barrier();
      uint4 v[8];
#pragma unroll
      for (int it = 0; it < 8; ++it) v[it] = *reinterpret_cast<const uint4*>(from + it * 4 * FP);
      if constexpr (Values::BIASED) {
        const float4& b = bias[jj / 2];
#pragma unroll
        for (int it = 0; it < 8; ++it)
          v[it] = make_uint4(__float_as_uint(__uint_as_float(v[it].x) + b.x),
                             __float_as_uint(__uint_as_float(v[it].y) + b.y),
                             __float_as_uint(__uint_as_float(v[it].z) + b.z),
                             __float_as_uint(__uint_as_float(v[it].w) + b.w));
      }
      const int32_t col = col0 + jj * 32 + 4 * cc;
      if (col < cols) {
#pragma unroll
        for (int it = 0; it < 8; ++it) {
          const int32_t row = row0 + i * 32 + it * 4 + (lane >> 4);
          if (row < rows) stream16(out + (i * 32 + it * 4) * ld + jj * 32, v[it]);
        }
      }
      asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
      __builtin_amdgcn_wave_barrier();
    }
}

// bfloat16 through one stage of LDS, in 4 rounds of 32 rows: each wave puts its block of
// 32 x 128 outputs in a region of its own (rows 272 bytes apart, 256 and a pad, so that
// the 16 lanes that read a row and rows 4 apart use different banks; the four regions
// fill the stage), reads it back 16 bytes a lane, 16 lanes a row, and stores 4 runs of
// 256 bytes an instruction. No other wave touches the region: no workgroup barrier.
// Every LDS address is a lane's base plus a constant.
constexpr int PITCH = 272;
constexpr int STAGING = 4 * 32 * PITCH;  // the bytes of a stage that the waves' regions take

// The accumulators of a 32 x 32 block as bfloat16 pairs: run g's columns 0-1 and 2-3
// (v_cvt_pk_bf16_f32: two floats to two bfloat16, nearest even).
__device__ __forceinline__ uint32_t bf16_pair(float lo, float hi) {
  typedef __bf16 bf16x2 __attribute__((ext_vector_type(2)));
  typedef float f32x2 __attribute__((ext_vector_type(2)));
  return __builtin_bit_cast(uint32_t, __builtin_convertvector((f32x2{lo, hi}), bf16x2));
}
struct FromAcc {
  static constexpr bool BIASED = false;
  const v16f (*acc)[4];
  __device__ __forceinline__ uint2 operator()(int i, int j, int g) const {
    const v16f& a = acc[i][j];
    return make_uint2(bf16_pair(a[4 * g], a[4 * g + 1]), bf16_pair(a[4 * g + 2], a[4 * g + 3]));
  }
  __device__ __forceinline__ float4 f32(int i, int j, int g) const {
    const v16f& a = acc[i][j];
    return make_float4(a[4 * g], a[4 * g + 1], a[4 * g + 2], a[4 * g + 3]);
  }
};

// `pairs(i, j, g)`: the bfloat16 pairs of block (i, j), register run g. With LO, only
// the rows from row_lo on are stored.
template <bool LO = false, typename Pairs, typename S>
__device__ void store_bf16(const Pairs& pairs, uint16_t* tile, int32_t ld, int32_t rows,
                           int32_t cols, S& stage, int32_t row_lo = 0) {
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const int wm = wave >> 1, wn = wave & 1;
  uint8_t* region = reinterpret_cast<uint8_t*>(&stage) + wave * 32 * PITCH;
  // Lane l writes row l % 32 of the block, its 4 columns of each 8 at byte 8 (l / 32).
  uint8_t* mine = region + (lane & 31) * PITCH + 8 * (lane >> 5);
  // ... and reads back chunk l % 16 (8 columns) of row l / 16 (of 4).
  const int cc = lane & 15;
  const uint8_t* from = region + (lane >> 4) * PITCH + cc * 16;
  const int32_t col = wn * 128 + 8 * cc;
  uint16_t* out = tile + (wm * 128 + (lane >> 4)) * ld + col;
  // A whole tile (the common case) stores without bounds checks, through a buffer
  // resource from its corner: the lane's offset, a scalar one a row of stores.
  const bool whole = rows >= BM && cols >= BN && (!LO || row_lo <= 0);
  const __amdgpu_buffer_rsrc_t rsrc =
      __builtin_amdgcn_make_buffer_rsrc(tile, 0, 0x7fffffff, 0x00020000);
  const int32_t lane_off = ((wm * 128 + (lane >> 4)) * ld + col) * 2;
#pragma unroll
  for (int i = 0; i < 4; ++i) {
#pragma unroll
    for (int j = 0; j < 4; ++j)
#pragma unroll
      for (int g = 0; g < 4; ++g) *reinterpret_cast<uint2*>(mine + (j * 4 + g) * 16) = pairs(i, j, g);
    asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
    __builtin_amdgcn_wave_barrier();
    // All 8 reads of the round go out before its first store.
    uint4 v[8];
#pragma unroll
    for (int it = 0; it < 8; ++it) v[it] = *reinterpret_cast<const uint4*>(from + it * 4 * PITCH);
    if (whole) {
#pragma unroll
      for (int it = 0; it < 8; ++it)
        __builtin_amdgcn_raw_buffer_store_b128(u32x4{v[it].x, v[it].y, v[it].z, v[it].w}, rsrc,
                                               lane_off, (i * 32 + it * 4) * ld * 2, NT);
    } else if (col < cols) {
#pragma unroll
      for (int it = 0; it < 8; ++it) {
        const int32_t row = wm * 128 + i * 32 + it * 4 + (lane >> 4);
        if (row < rows && (!LO || row >= row_lo)) {
          uint16_t* at = out + (i * 32 + it * 4) * ld;
          if (col + 8 <= cols) stream16(at, v[it]);
          else stream8(at, v[it].x, v[it].y);  // cols % 4 == 0
        }
      }
    }
    // The reads are done before the next round's writes.
    asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
    __builtin_amdgcn_wave_barrier();
  }
}

template <typename From, typename S>
__device__ __forceinline__ void store_tile(const From& from, uint16_t* tile, int32_t ld,
                                           int32_t rows, int32_t cols, S& stage) {
  store_bf16(from, tile, ld, rows, cols, stage);
}
template <typename From, typename S>
__device__ __forceinline__ void store_tile(const From& from, float* tile, int32_t ld,
                                           int32_t rows, int32_t cols, S& stage) {
  const int wave = threadIdx.x >> 6;
  store_f32<4, 4>(from, tile, ld, rows, cols, (wave >> 1) * 128, (wave & 1) * 128, stage);
}

// A half tile's outputs, each wave's 128 rows x 64 columns (columns 64 w on; accumulator
// blocks [i][0..1]). bfloat16 through the wave's region of the stage as store_bf16 does,
// read back 16 bytes a lane, 8 lanes a row, in 4 rounds of 32 rows.
template <typename From, typename S>
__device__ void store_tile_half(const From& pairs, uint16_t* tile, int32_t ld, int32_t rows,
                                int32_t cols, S& stage) {
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  uint8_t* region = reinterpret_cast<uint8_t*>(&stage) + wave * 32 * PITCH;
  uint8_t* mine = region + (lane & 31) * PITCH + 8 * (lane >> 5);
  const int cc = lane & 7;
  const uint8_t* from = region + (lane >> 3) * PITCH + cc * 16;
  const int32_t col = wave * 64 + 8 * cc;
  uint16_t* out = tile + (lane >> 3) * ld + col;
  const bool whole = rows >= BM / 2 && cols >= BN;
  const __amdgpu_buffer_rsrc_t rsrc =
      __builtin_amdgcn_make_buffer_rsrc(tile, 0, 0x7fffffff, 0x00020000);
  const int32_t lane_off = ((lane >> 3) * ld + col) * 2;
#pragma unroll
  for (int i = 0; i < 4; ++i) {
#pragma unroll
    for (int j = 0; j < 2; ++j)
#pragma unroll
      for (int g = 0; g < 4; ++g) *reinterpret_cast<uint2*>(mine + (j * 4 + g) * 16) = pairs(i, j, g);
    asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
    __builtin_amdgcn_wave_barrier();
    uint4 v[4];
#pragma unroll
    for (int it = 0; it < 4; ++it) v[it] = *reinterpret_cast<const uint4*>(from + it * 8 * PITCH);
    if (whole) {
#pragma unroll
      for (int it = 0; it < 4; ++it)
        __builtin_amdgcn_raw_buffer_store_b128(u32x4{v[it].x, v[it].y, v[it].z, v[it].w}, rsrc,
                                               lane_off, (i * 32 + it * 8) * ld * 2, NT);
    } else if (col < cols) {
#pragma unroll
      for (int it = 0; it < 4; ++it) {
        const int32_t row = i * 32 + it * 8 + (lane >> 3);
        if (row < rows) {
          uint16_t* at = out + (i * 32 + it * 8) * ld;
          if (col + 8 <= cols) stream16(at, v[it]);
          else stream8(at, v[it].x, v[it].y);  // cols % 4 == 0
        }
      }
    }
    asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
    __builtin_amdgcn_wave_barrier();
  }
}
// float32 as store_f32.
template <typename From, typename S>
__device__ void store_tile_half(const From& from, float* tile, int32_t ld, int32_t rows,
                                int32_t cols, S& stage) {
  const int wave = threadIdx.x >> 6;
  store_f32<4, 2>(from, tile, ld, rows, cols, 0, wave * 64, stage);
}

// bfloat16 of a tile that stores every row and column (PH: a half tile's 128 rows),
// through the wave's region of the stage as pairs of 32 x 32 accumulator blocks: a whole
// tile's wave holds 8 pairs (block row p / 2, its 64 columns from 64 (p % 2)), a half
// tile's 4 (block row p, the wave's 64 columns). Two buffers of 32 rows 136 bytes apart
// (128 bytes of a pair's row and 8 of pad: the 32 rows of a lane half start on distinct
// banks) fill the region; each lane writes its row's 4 runs of 4 columns of both blocks
// (8 bytes each), reads back 16 bytes of a row, 8 lanes a row (as two 8-byte reads: the
// rows are 8-byte aligned), and a store writes 8 whole rows of 128 bytes. Pair p + 1 is
// converted and written while pair p's reads are in flight, and pair p's stores go out
// after them: the wave's LDS operations run in order, so a read after a write sees it and
// a write after a read (into the buffer the pair before last used) leaves it alone.
constexpr int PAIR_PITCH = 136;
constexpr int PAIR_BUF = 32 * PAIR_PITCH;
static_assert(2 * PAIR_BUF == 32 * PITCH, "a wave's two pair buffers fill its region of the stage");

template <bool PH, typename From, typename S>
__device__ void store_pairs(const From& pairs, uint16_t* tile, int32_t ld, S& stage) {
  const int lane = threadIdx.x & 63;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  uint8_t* region = reinterpret_cast<uint8_t*>(&stage) + wave * 2 * PAIR_BUF;
  uint8_t* mine = region + (lane & 31) * PAIR_PITCH + 8 * (lane >> 5);
  const uint8_t* from = region + (lane >> 3) * PAIR_PITCH + (lane & 7) * 16;
  const __amdgpu_buffer_rsrc_t rsrc =
      __builtin_amdgcn_make_buffer_rsrc(tile, 0, 0x7fffffff, 0x00020000);
  const int32_t lane_off = ((lane >> 3) * ld + 8 * (lane & 7)) * 2;
  constexpr int M = PH ? 4 : 8;
  auto write = [&](int p) {
    const int i = PH ? p : p >> 1, j0 = PH ? 0 : (p & 1) * 2;
    uint8_t* at = mine + (p & 1) * PAIR_BUF;
#pragma unroll
    for (int jb = 0; jb < 2; ++jb)
#pragma unroll
      for (int g = 0; g < 4; ++g) *reinterpret_cast<uint2*>(at + jb * 64 + g * 16) = pairs(i, j0 + jb, g);
  };
  write(0);
#pragma unroll
  for (int p = 0; p < M; ++p) {
    const uint8_t* at = from + (p & 1) * PAIR_BUF;
    uint2 v[8];
#pragma unroll
    for (int it = 0; it < 4; ++it) {
      v[2 * it] = *reinterpret_cast<const uint2*>(at + it * 8 * PAIR_PITCH);
      v[2 * it + 1] = *reinterpret_cast<const uint2*>(at + it * 8 * PAIR_PITCH + 8);
    }
    if (p + 1 < M) write(p + 1);
    const int32_t row0 = PH ? p * 32 : (wave >> 1) * 128 + (p >> 1) * 32;
    const int32_t col0 = PH ? wave * 64 : (wave & 1) * 128 + (p & 1) * 64;
    const int32_t corner = (row0 * ld + col0) * 2;
#pragma unroll
    for (int it = 0; it < 4; ++it)
      __builtin_amdgcn_raw_buffer_store_b128(
          u32x4{v[2 * it].x, v[2 * it].y, v[2 * it + 1].x, v[2 * it + 1].y}, rsrc, lane_off,
          corner + it * 8 * ld * 2, NT);
  }
}

// The plain epilogue: the tile's rows [0, rows) and columns [0, cols) of a row-major
// output of pitch ld, from its corner.
template <typename T, typename From, typename S>
__device__ __forceinline__ void store_plain(const From& from, T* out, int32_t ld, const Job& j,
                                            S& stage) {
  if constexpr (std::is_same<T, uint16_t>::value) {
    if (j.cols >= BN && j.rows >= (j.half ? BM / 2 : BM)) {
      if (j.half) store_pairs<true>(from, out + j.corner, ld, stage);
      else store_pairs<false>(from, out + j.corner, ld, stage);
      return;
    }
  }
  if (j.half) store_tile_half(from, out + j.corner, ld, j.rows, j.cols, stage);
  else store_tile(from, out + j.corner, ld, j.rows, j.cols, stage);
}

// Whether these stores' 32-bit offsets from a tile's corner hold an output of `rows` rows of n:
// bytes of bfloat16 in a buffer resource, elements of float32 (half as many bits). Past that, rows
// of a tile were dropped, and from twice as many on written before the output.
inline bool stores_fit(int64_t rows, int64_t n) {
  return 2 * (rows < BM ? rows : BM) * n < (1LL << 31);
}

}  // namespace
}  // namespace bux
