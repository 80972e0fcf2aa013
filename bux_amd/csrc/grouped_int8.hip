// The experts' products in 8-bit integers: y[i] = s_a[i] s_b[g(i)] sum_k a[i][k] b[g(i)][k], for
// each group g's rows i; v_mfma_i32_32x32x32_i8, sums exact in 32-bit integers (K at most
// 131072), one rounding to the output's type after the scales (and the group's bias).
//
// The schedule is the MXFP8 GEMMs' (tiles.h, grouped_mx.hip): a tile list, a persistent grid,
// 256 x 256 outputs a workgroup in 4 waves, direct loads into a ring of 4 LDS stages; operands
// in the same tiled layout, codes [K / 64][rows][64]. A step is 64 of K, 32 MFMAs a wave: an
// 8-bit integer MFMA has the rate of an MXFP8 one. Both operands' scales are a float a row: a
// tile's go to LDS once, with its first step's codes, to one of two places that tiles take in
// turn, where the epilogue finds them. (A load of each beside every step's codes instead: 131072
// rows of K 2048, N 1536 510 us and 506, 8192 tokens of gpt-oss-120b's up product 860 and 842.)
//
// What bounds it: power on uniform codes (8192^3 in 536 us, 2050 TOPS, and with codes of 0 in 358),
// and the epilogue, which no MFMA hides: 131072 rows of K 2048, N 1536 in 128 even groups take 453,
// of K 128 114.
//
// MFMA lane layout (32 x 32 x 32): lane l holds row l % 32 of either operand, its half l / 32
// the 16 bytes of K 16 (l / 32) .. + 15; accumulators as the float MFMAs'.

#include "epilogue.h"
#include "int8_direct.h"
#include "tiles.h"

namespace bux {
namespace {

typedef int v4i __attribute__((ext_vector_type(4)));
typedef int v16i __attribute__((ext_vector_type(16)));

constexpr int BK = 64;  // bytes of K a step
constexpr int LOADS_A_STEP = 8;
constexpr int64_t MAX_K = 131072;

struct Operand {
  const uint8_t* values;
  const float* scales;  // [rows]
  int32_t k;            // bytes of K a row: whole 128s
  int32_t rows;
};

// One K step's codes of 256 rows of A and B, and to the bytes that the epilogue stages outputs in.
struct Stage {
  uint8_t a[BM * BK];
  uint8_t b[BN * BK];
  uint8_t gap[STAGING - BM * BK - BN * BK];
};
struct Scales {
  float a[BM];
  float b[BN];
  float added[BN];  // the columns' biases, written by the epilogue
};
struct Lds {
  Stage st[STAGES];
  Scales tile[2];
};
static_assert(sizeof(Lds) <= 160 * 1024, "the stages fit a CU's LDS");

// Which of the two places a tile's scales take rides above its first row's bits.
constexpr int32_t PLACE_BIT = 1 << 30;
constexpr int32_t ROW_MASK = PLACE_BIT - 1;

// Where a 64-byte LDS row's 16-byte chunk c sits: c ^ swizzle(row), so that 16 lanes that read
// one chunk of 16 consecutive rows hit every bank once.
__device__ __forceinline__ int swizzle(int row) { return (row >> 2) & 3; }

struct Loads {
  const uint8_t* values;
  i32x4 rv, rs;
  int32_t voff, soff;    // this lane's
  int32_t chunk_stride;  // a K chunk's bytes: rows x 64
  int32_t place;         // A's: of the tile's scales
};

__device__ __forceinline__ Loads loads_for(const Operand& op, int32_t placed_row) {
  const int32_t row0 = placed_row & ROW_MASK;
  const int w = threadIdx.x >> 6, l = threadIdx.x & 63;
  Loads ld;
  ld.values = op.values;
  ld.rv = resource(op.values, static_cast<int64_t>(op.k) * op.rows);
  ld.rs = resource(op.scales, static_cast<int64_t>(op.rows) * 4);
  const int r = w * 64 + (l >> 2);
  ld.voff = (row0 + r) * 64 + 16 * ((l & 3) ^ swizzle(r));
  ld.soff = (row0 + w * 64 + l) * 4;
  ld.chunk_stride = op.rows * 64;
  ld.place = placed_row >> 30;
  return ld;
}

// K chunk c's resource and scalar offset: wide operands (W: past 2 GiB) a chunk at a time.
template <bool W>
__device__ __forceinline__ i32x4 chunk_at(const Loads& l, int32_t c, int32_t& soff) {
  if constexpr (W) {
    soff = 0;
    return resource(l.values + static_cast<int64_t>(c) * l.chunk_stride, l.chunk_stride);
  } else {
    soff = c * l.chunk_stride;
    return l.rv;
  }
}

// Direct load Q (0 .. 7) of K step ks: a 16-row slice of A's (even Q) or B's (odd Q) rows of this
// wave. In a half tile (H) waves 2 and 3, whose rows of A do not exist, load their rows' scales
// again in their place, so that every wave issues 8.
__device__ __forceinline__ uint32_t scales_at(uint32_t lds0, int32_t place) {
  return lds0 + static_cast<uint32_t>(offsetof(Lds, tile) + place * sizeof(Scales));
}
template <int Q, bool H, bool W>
__device__ __forceinline__ void issue_one(const Loads& la, const Loads& lb, int32_t ks,
                                          uint32_t lds0, int st) {
  const uint32_t w = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const uint32_t at = lds0 + static_cast<uint32_t>(st * sizeof(Stage));
  constexpr int i = Q >> 1;
  const uint32_t slice = w * 4096 + i * 1024;
  int32_t so;
  if ((Q & 1) == 0 && H && w >= 2) {
    load_lds4(la.rs, scales_at(lds0, la.place) + offsetof(Scales, a) + w * 256, la.soff, 0);
  } else if ((Q & 1) == 0) {
    const i32x4 r = chunk_at<W>(la, ks, so);
    load_lds16(r, at + offsetof(Stage, a) + slice, la.voff, so + i * 1024);
  } else {
    const i32x4 r = chunk_at<W>(lb, ks, so);
    load_lds16(r, at + offsetof(Stage, b) + slice, lb.voff, so + i * 1024);
  }
}
template <int Q, bool H, bool W>
__device__ __forceinline__ void issue_from(const Loads& la, const Loads& lb, int32_t ks,
                                           uint32_t lds0, int st) {
  issue_one<Q, H, W>(la, lb, ks, lds0, st);
  if constexpr (Q + 1 < LOADS_A_STEP) issue_from<Q + 1, H, W>(la, lb, ks, lds0, st);
}

// A wave's operands of one step: 4 blocks of 32 rows of A and of B, K 0 .. 31 and 32 .. 63.
struct Frag {
  v4i a[4][2], b[4][2];
};
struct Lanes {
  int32_t a[2], b[2];  // byte offsets of block 0's two chunks
};
template <bool H>
__device__ __forceinline__ Lanes lanes_of() {
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const int half = lane >> 5, row = lane & 31, sw = swizzle(row);
  const int ra = (H ? 0 : (wave >> 1) * 128) + row;
  const int rb = (H ? wave * 64 : (wave & 1) * 128) + row;
  const int lo = (half ^ sw) << 4, hi = ((2 + half) ^ sw) << 4;
  return Lanes{{ra * BK + lo, ra * BK + hi}, {rb * BK + lo, rb * BK + hi}};
}
__device__ __forceinline__ void read_a(Frag& f, const Lds& lds, const Lanes& ln, int st, int p) {
#pragma unroll
  for (int h = 0; h < 2; ++h)
    f.a[p][h] = *reinterpret_cast<const v4i*>(lds.st[st].a + p * 2048 + ln.a[h]);
}
__device__ __forceinline__ void read_b(Frag& f, const Lds& lds, const Lanes& ln, int st, int p) {
#pragma unroll
  for (int h = 0; h < 2; ++h)
    f.b[p][h] = *reinterpret_cast<const v4i*>(lds.st[st].b + p * 2048 + ln.b[h]);
}

// The accumulators pass the shared pipeline as floats' registers; their bits are integers.
__device__ __forceinline__ void multiply(const v4i& b, const v4i& a, v16f& acc) {
  acc = __builtin_bit_cast(
      v16f, __builtin_amdgcn_mfma_i32_32x32x32_i8(b, a, __builtin_bit_cast(v16i, acc), 0, 0, 0));
}

// One step on `cur`, J blocks of B a block of A (4; in a half tile 2): each pair of MFMAs is
// followed by a slice of the memory work, LOAD's next loads and READ's operands of the next
// step in the order its MFMAs take them.
template <bool LOAD, bool READ, bool H, bool W>
__device__ __forceinline__ void step_of(const Frag& cur, Frag& nxt, const Loads& la,
                                        const Loads& lb, const Lds& lds, uint32_t lds0,
                                        const Lanes& ln, int32_t ks_load, int st_load, int st_next,
                                        v16f acc[4][4]) {
  constexpr int J = H ? 2 : 4;
#pragma unroll
  for (int q = 0; q < 4 * J; ++q) {
    const int i = q / J, j = q % J;
    multiply(cur.b[j][0], cur.a[i][0], acc[i][j]);
    multiply(cur.b[j][1], cur.a[i][1], acc[i][j]);
    __builtin_amdgcn_sched_barrier(0);
    if (LOAD) {
      switch (q) {
        case 0: issue_one<0, H, W>(la, lb, ks_load, lds0, st_load); break;
        case 1: issue_one<1, H, W>(la, lb, ks_load, lds0, st_load); break;
        case 2: issue_one<2, H, W>(la, lb, ks_load, lds0, st_load); break;
        case 3: issue_one<3, H, W>(la, lb, ks_load, lds0, st_load); break;
        case 4: issue_one<4, H, W>(la, lb, ks_load, lds0, st_load); break;
        case 5: issue_one<5, H, W>(la, lb, ks_load, lds0, st_load); break;
        case 6: issue_one<6, H, W>(la, lb, ks_load, lds0, st_load); break;
        case 7: issue_one<7, H, W>(la, lb, ks_load, lds0, st_load); break;
        default: break;
      }
    }
    if (READ) {
      if (q == 0) read_a(nxt, lds, ln, st_next, 0);
      if (q < J) read_b(nxt, lds, ln, st_next, q);
      if (q > 0 && j == 0) read_a(nxt, lds, ln, st_next, i);
    }
    __builtin_amdgcn_sched_barrier(0);
  }
}

// The format's part of the shared pipeline (run_tiles).
template <bool W>
struct Int8 {
  using Operand = bux::Operand;
  using Lds = bux::Lds;
  using Loads = bux::Loads;
  using Lanes = bux::Lanes;
  using Frag = bux::Frag;
  static constexpr bool HALVES = true;
  __device__ static __forceinline__ Loads loads_a(const Operand& a, int32_t row0) {
    return loads_for(a, row0);
  }
  __device__ static __forceinline__ Loads loads_b(const Operand& b, int32_t group, int32_t row0) {
    Operand own = b;
    own.values += static_cast<int64_t>(group) * b.rows * b.k;
    own.scales += static_cast<int64_t>(group) * b.rows;
    return loads_for(own, row0);
  }
  __device__ static __forceinline__ void issue(const Loads& la, const Loads& lb, int32_t ks,
                                               uint32_t lds0, int st, bool half) {
    // A tile's scales go ahead of its first step's codes (never in a step: those load from step 4
    // on). The waits count 8 loads a step: these two among later ones make them stricter.
    if (ks == 0) {
      const uint32_t w = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
      const uint32_t at = scales_at(lds0, la.place) + w * 256;
      load_lds4(la.rs, at + offsetof(Scales, a), la.soff, 0);
      load_lds4(lb.rs, at + offsetof(Scales, b), lb.soff, 0);
    }
    if (half) issue_from<0, true, W>(la, lb, ks, lds0, st);
    else issue_from<0, false, W>(la, lb, ks, lds0, st);
  }
  __device__ static __forceinline__ void wait_loads(int32_t steps) {
    if (steps >= 3) asm volatile("s_waitcnt vmcnt(24)" ::: "memory");
    else if (steps == 2) asm volatile("s_waitcnt vmcnt(16)" ::: "memory");
    else if (steps == 1) asm volatile("s_waitcnt vmcnt(8)" ::: "memory");
    else asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
  }
  template <bool H>
  __device__ static __forceinline__ Lanes lanes_of() { return bux::lanes_of<H>(); }
  template <bool H>
  __device__ static __forceinline__ void read_frag(Frag& f, const Lds& lds, const Lanes& ln, int st,
                                                   int32_t) {
#pragma unroll
    for (int p = 0; p < 4; ++p) {
      read_a(f, lds, ln, st, p);
      if (!H || p < 2) read_b(f, lds, ln, st, p);
    }
  }
  __device__ static __forceinline__ void mask_frag(Frag&, int32_t, int32_t, int32_t) {}
  template <bool LOAD, bool READ, bool H>
  __device__ static __forceinline__ void step(const Frag& cur, Frag& nxt, const Loads& la,
                                              const Loads& lb, const Lds& lds, uint32_t lds0,
                                              const Lanes& ln, int32_t ks_load, int st_load,
                                              int32_t, int st_next, v16f acc[4][4]) {
    step_of<LOAD, READ, H, W>(cur, nxt, la, lb, lds, lds0, ln, ks_load, st_load, st_next, acc);
  }
};

// The sums times both scales, plus the column's bias: a lane's row's scale a block of A in
// registers, its 4 columns' a run read from LDS where they are used (32 lanes one address; in
// registers they would take 64, and went to scratch memory).
template <bool BIASED_>
struct Scaled {
  static constexpr bool BIASED = false;  // store_f32's own addition is not used
  const v16f (*acc)[4];
  float row[4];
  const float* col;    // this lane's first column's scale, and the biases beside it
  const float* added;
  __device__ __forceinline__ float4 f32(int i, int j, int g) const {
#pragma clang fp contract(off)
    // The sums stay in accumulation registers up to here: moved out all at once, ahead of the
    // epilogue's forms, they pushed the lane's offsets to scratch memory.
    auto sum = [&](int q) {
      float v = acc[i][j][4 * g + q];
      asm volatile("" : "+a"(v));
      return static_cast<float>(__builtin_bit_cast(int, v));
    };
    const float4 s = *reinterpret_cast<const float4*>(col + 32 * j + 8 * g);
    float4 v = make_float4(sum(0) * (row[i] * s.x), sum(1) * (row[i] * s.y),
                           sum(2) * (row[i] * s.z), sum(3) * (row[i] * s.w));
    if constexpr (BIASED_) {
      const float4 b = *reinterpret_cast<const float4*>(added + 32 * j + 8 * g);
      v = make_float4(v.x + b.x, v.y + b.y, v.z + b.z, v.w + b.w);
    }
    return v;
  }
  __device__ __forceinline__ uint2 operator()(int i, int j, int g) const {
    const float4 v = f32(i, j, g);
    return make_uint2(bf16_pair(v.x, v.y), bf16_pair(v.z, v.w));
  }
};

// The rows GEMM's tiles, each with the place of its scales in turn.
struct PlacedTiles : RowsTiles<false, true> {
  mutable int32_t place = 0;
  __device__ explicit PlacedTiles(const RowsTiles<false, true>& list) : RowsTiles<false, true>(list) {}
  __device__ bool job(int32_t id, Job& j) const {
    if (!RowsTiles<false, true>::job(id, j)) return false;
    j.a_row0 |= place;
    place ^= PLACE_BIT;
    return true;
  }
};

template <typename T, bool BIASED>
struct Out {
  T* out;
  int32_t ld;
  const T* bias;  // (groups, ld)
  Scales* tiles;  // the two places
  __device__ __forceinline__ void store(const v16f acc[4][4], const Job& j, Stage& stage) const {
    // The thread's place, computed here: hoisted out of the tiles' loop, what depends on it
    // alone would be held through every K loop, and went to scratch memory.
    int thread = threadIdx.x;
    asm volatile("" : "+v"(thread));
    const int lane = thread & 63, wave = thread >> 6;
    const int row0 = (j.half ? 0 : (wave >> 1) * 128) + (lane & 31);
    const int col0 = (j.half ? wave * 64 : (wave & 1) * 128) + 4 * (lane >> 5);
    Scales& scales = tiles[j.a_row0 >> 30];
    if (j.n == 0) {  // rows past the groups: no step ran, so the scales are 0 here
      scales.b[thread] = 0.0f;
      barrier_lds();
    }
    if constexpr (BIASED) {
      const T* const row = bias + static_cast<int64_t>(j.group) * ld + j.b_row0;
      const int c = thread;
      scales.added[c] = j.n > 0 && c < j.cols ? Elem<T>::value(row[c]) : 0.0f;
      barrier_lds();
    }
    Scaled<BIASED> from;
    from.acc = acc;
    from.col = scales.b + col0;
    from.added = scales.added + col0;
#pragma unroll
    for (int i = 0; i < 4; ++i) from.row[i] = j.n > 0 ? scales.a[row0 + 32 * i] : 0.0f;
    store_plain(from, out, ld, j, stage);
  }
};

template <typename T, bool W, bool BIASED>
__global__ __launch_bounds__(THREADS) __attribute__((amdgpu_waves_per_eu(1, 1))) void rows_kernel(
    Operand A, Operand B, int32_t groups, int32_t n, int32_t height,
    const int32_t* __restrict__ starts, const Tile* __restrict__ tiles, int32_t col_tiles,
    const T* __restrict__ bias, T* __restrict__ y) {
  extern __shared__ __align__(16) uint8_t smem[];
  if (!list_fits(starts, groups, A.rows, height)) return;
  Lds& lds = *reinterpret_cast<Lds*>(smem);
  const PlacedTiles list(RowsTiles<false, true>{tiles, groups, n, height, col_tiles, A.k / BK, A.k});
  const int32_t count = starts[groups + 1] * col_tiles;
  run_tiles<Int8<W>>(list, count, A, B, lds, Out<T, BIASED>{y, n, bias, lds.tile});
}

// The loads' 32-bit offsets hold a K chunk's rows (a tile's reads past them included), and the
// rows' scales; an operand under 2 GiB goes by one resource.
constexpr int64_t MAX_ROWS = (1LL << 31) / BK - BM;
bool narrow(int64_t rows, int64_t k) { return (rows + BM) * k < (1LL << 31); }

template <typename T>
int launch_rows(const Operand& A, const Operand& B, int32_t groups, int64_t n, int64_t height,
                const void* list, int64_t slots, const void* bias, void* y, hipStream_t s) {
  const int64_t col_tiles = ceil_div(n, BN);
  BUX_CHECK(stores_fit(height, n), "bux_int8_grouped_rows_listed: n=%lld columns by height=%lld "
            "rows: a tile's outputs exceed 2 GiB", (long long)n, (long long)height);
  if (slots * col_tiles >= (1LL << 31))
    return fail(BUX_E_ARGUMENT, "bux_int8_grouped_rows_listed: too many tiles");
  unsigned blocks = 0;
  if (int rc = grid_for(slots * col_tiles, &blocks)) return rc;
  auto go = [&](auto kernel) {
    if (int rc = allow_lds(kernel, sizeof(Lds), "int8 rows_kernel")) return rc;
    hipLaunchKernelGGL(kernel, dim3(blocks), dim3(THREADS), sizeof(Lds), s, A, B, groups,
                       static_cast<int32_t>(n), static_cast<int32_t>(height), starts_in(list),
                       tiles_in(list, groups), static_cast<int32_t>(col_tiles),
                       static_cast<const T*>(bias), static_cast<T*>(y));
    return launched("int8 rows_kernel");
  };
  if (narrow(A.rows, A.k) && narrow(B.rows, B.k))
    return bias ? go(rows_kernel<T, false, true>) : go(rows_kernel<T, false, false>);
  return bias ? go(rows_kernel<T, true, true>) : go(rows_kernel<T, true, false>);
}

}  // namespace
}  // namespace bux

extern "C" int bux_int8_grouped_rows_listed(const uint8_t* a_values, const float* a_scales,
                                            const uint8_t* b_values, const float* b_scales,
                                            void* list, size_t list_bytes, int32_t groups,
                                            int64_t m, int64_t n, int64_t k, int64_t height,
                                            int out_dtype, const void* bias, void* y,
                                            void* stream) {
  using namespace bux;
  constexpr const char* name = "bux_int8_grouped_rows_listed";
  clear_error();
  BUX_CHECK(groups >= 1 && groups <= MAX_GROUPS, "%s: groups=%d outside [1, %d]", name, groups,
            MAX_GROUPS);
  BUX_CHECK(m >= 0 && n > 0 && height >= 0 && height < (1LL << 31),
            "%s: bad shape m=%lld n=%lld height=%lld", name, (long long)m, (long long)n,
            (long long)height);
  BUX_CHECK(k > 0 && k % 128 == 0 && k <= MAX_K,
            "%s: k=%lld is not a multiple of 128 (the tiled layout's padded K) up to %lld", name,
            (long long)k, (long long)MAX_K);
  BUX_CHECK(n % 4 == 0, "%s: n=%lld is not a multiple of 4", name, (long long)n);
  BUX_CHECK(m <= MAX_ROWS && n <= MAX_ROWS, "%s: an operand of %lld rows exceeds %lld", name,
            (long long)(m > n ? m : n), (long long)MAX_ROWS);
  BUX_CHECK(out_dtype == BUX_BF16 || out_dtype == BUX_F32, "%s: out_dtype=%d", name, out_dtype);
  BUX_CHECK(b_values && b_scales && (height == 0 || y) && (m == 0 || (a_values && a_scales)),
            "%s: NULL buffer", name);
  const int64_t slots = row_slots(groups, m, height);
  const size_t need = starts_bytes(groups) + static_cast<size_t>(slots) * sizeof(Tile);
  if (list == nullptr || list_bytes < need)
    return fail(BUX_E_WORKSPACE, "%s: list of %zu bytes, %zu needed", name, list_bytes, need);
  if (height == 0) return BUX_OK;
  hipStream_t s = as_stream(stream);
  if (int8_rows_direct(m, groups))
    return launch_int8_direct(a_values, a_scales, b_values, b_scales, list, slots, groups, m, n, k,
                              height, out_dtype, bias, y, s);
  const Operand A{a_values, a_scales, static_cast<int32_t>(k), static_cast<int32_t>(m)};
  const Operand B{b_values, b_scales, static_cast<int32_t>(k), static_cast<int32_t>(n)};
  return out_dtype == BUX_BF16 ? launch_rows<uint16_t>(A, B, groups, n, height, list, slots, bias, y, s)
                               : launch_rows<float>(A, B, groups, n, height, list, slots, bias, y, s);
}
