// Dense matrix products with their epilogues (dense.h), any shape and alignment, in bfloat16
// (v_mfma_f32_32x32x16_bf16) and float32 (v_mfma_f32_32x32x2_f32), float32 sums:
//
//   rows      y = epilogue(x w)     w [k, n], or [n, k] (transposed: x w^T)
//   contract  dw = x^T dy           x [m, k], dy [m, n]
//
// A workgroup of 4 waves makes 128 x 128 of the output, a wave 64 x 64 of it (in float32 also 128 x
// 64, which leave less of a narrow or an odd output to nothing), in steps of 128 bytes of K (64 bfloat16, 32 float32). A step's operands come into registers 16 bytes a load at
// an element's alignment, two steps ahead, then into one of two LDS stages of 32 KiB:
//   K-major (x; w transposed)   128 rows of 128 bytes, 16-byte chunk c of row r at place
//                               c ^ (r % 8), so that 16 lanes that read one chunk of 16 rows
//                               take every bank twice at most
//   MN-major (w; contract's)    K rows of 128 elements, chunk c of K row k at place c ^ 4 (k % 4)
//                               in bfloat16 (read by ds_read_b64_tr_b16, which transposes) and at
//                               c ^ 8 ((k / 8) % 2) in float32
// Rows past an operand's read its last row (no output takes them); K positions past k read 0 in
// both operands.
//
// Few tiles leave CUs idle: K is then split over workgroups, whose sums go to the workspace in
// float32 and are added in order, with the epilogue, by a second kernel.

#include "dense.h"

namespace bux {
using namespace dense;
namespace {

typedef __bf16 v8bf __attribute__((ext_vector_type(8)));
typedef short v4s __attribute__((ext_vector_type(4)));
typedef __attribute__((address_space(3))) v4s lds_v4s;

constexpr int THREADS = 256;
constexpr int TILE = 128;

template <typename T>
constexpr int BK = 128 / sizeof(T);
template <typename T>
constexpr int PER = 16 / sizeof(T);  // elements of a chunk

struct Chunk {
  uint32_t w[4];
};
template <typename T>
__device__ __forceinline__ Chunk load_chunk(const T* p) {
  struct __attribute__((packed, aligned(sizeof(T)))) Any {
    Chunk c;
  };
  return reinterpret_cast<const Any*>(p)->c;
}
// Its first `count` elements, zeros after them.
template <typename T>
__device__ __forceinline__ Chunk load_chunk(const T* p, int64_t count) {
  if (count >= PER<T>) return load_chunk(p);
  struct {
    T at[PER<T>];
  } e{};
#pragma unroll
  for (int j = 0; j < PER<T>; ++j)
    if (j < count) e.at[j] = p[j];
  return __builtin_bit_cast(Chunk, e);
}

// A thread's chunks of an operand's step, SIDE rows of it: K-major chunk i is of row 32 i + tid / 8 at K chunk
// tid % 8; MN-major of K row (256 i + tid) / (chunks a K row). K is `k` long in all.
template <typename T, bool KM, int SIDE>
struct Loader {
  static constexpr int ROW = KM ? 8 : SIDE / PER<T>;  // chunks a row, or a K row
  static constexpr int N = SIDE / 32;                 // chunks a thread
  const T* at[N];
  int64_t ld, left;  // MN-major: columns from this lane's on
  int64_t plain;     // steps that end at or before this K position load without a check
  __device__ __forceinline__ Loader(const Mat<T>& a, int64_t row0, int64_t k0, int64_t k,
                                    int64_t kend)
      : ld(a.ld) {
    const int tid = threadIdx.x, c = tid % ROW;
    left = a.rows - row0 - PER<T> * c;
    plain = kend;
    if (!KM && row0 + SIDE > a.rows) {
      // The tile reaches past the columns. A chunk that they cut reads on into the next K row (its
      // columns are no output's), which the last K row does not have; the lanes past them read the
      // row's last chunk.
      if (a.rows % PER<T> != 0 && kend == k) plain = k - 1;
      if (a.rows < PER<T>) plain = k0;
    }
    const int64_t col = left > 0 || a.rows < PER<T> ? row0 + PER<T> * c : a.rows - PER<T>;
#pragma unroll
    for (int i = 0; i < N; ++i) {
      const int s = i * (THREADS / ROW) + tid / ROW;
      if (KM) {
        const int64_t r = row0 + s;
        at[i] = a.p + (r < a.rows ? r : a.rows - 1) * ld + k0 + PER<T> * c;
      } else {
        at[i] = a.p + (k0 + s) * ld + col;
      }
    }
  }
  // The step at K position k (its first), K ending at kend; then on to the next.
  __device__ __forceinline__ void step(Chunk out[N], int64_t k, int64_t kend) {
    const int tid = threadIdx.x;
    if (k + BK<T> <= plain) {
#pragma unroll
      for (int i = 0; i < N; ++i) out[i] = load_chunk(at[i]);
    } else {
#pragma unroll
      for (int i = 0; i < N; ++i) {
        const int s = i * (THREADS / ROW) + tid / ROW;
        const int64_t count = KM ? kend - k - PER<T> * (tid % ROW) : k + s < kend ? left : 0;
        out[i] = load_chunk(at[i], count);
      }
    }
#pragma unroll
    for (int i = 0; i < N; ++i) at[i] += KM ? BK<T> : BK<T> * ld;
  }
};

template <typename T, bool KM, int SIDE>
__device__ __forceinline__ void put_step(uint8_t* lds, const Chunk c[SIDE / 32]) {
  constexpr int ROW = KM ? 8 : SIDE / PER<T>;
  const int tid = threadIdx.x, place = tid % ROW;
#pragma unroll
  for (int i = 0; i < SIDE / 32; ++i) {
    const int s = i * (THREADS / ROW) + tid / ROW;
    const int sw = KM ? (s & 7) : sizeof(T) == 2 ? 4 * (s & 3) : 8 * ((s >> 3) & 1);
    *reinterpret_cast<Chunk*>(lds + s * (16 * ROW) + 16 * (place ^ sw)) = c[i];
  }
}

// bfloat16: the operand of an MFMA over K 16 s .. + 15 of the step, rows base .. base + 31:
// lane l row base + l % 32, K 8 (l / 32) .. + 7 of those.
template <bool KM>
__device__ __forceinline__ v8bf read_bf16(const uint8_t* lds, int base, int s) {
  const int l = threadIdx.x & 63, h = l >> 5;
  if constexpr (KM) {
    const int r = base + (l & 31);
    return *reinterpret_cast<const v8bf*>(lds + r * 128 + 16 * ((2 * s + h) ^ (r & 7)));
  } else {
    const int q = l & 15, kq = q >> 2;
    const int k = 16 * s + 8 * h + kq, col = base + 16 * ((l >> 4) & 1) + 4 * (q & 3);
    const uint32_t at = static_cast<uint32_t>(reinterpret_cast<uintptr_t>(lds)) + k * 256 +
                        16 * ((col >> 3) ^ (4 * kq)) + 8 * ((col >> 2) & 1);
    const v4s x = __builtin_amdgcn_ds_read_tr16_b64_v4i16(reinterpret_cast<lds_v4s*>(at));
    const v4s y = __builtin_amdgcn_ds_read_tr16_b64_v4i16(reinterpret_cast<lds_v4s*>(at + 1024));
    return __builtin_bit_cast(v8bf, __builtin_shufflevector(x, y, 0, 1, 2, 3, 4, 5, 6, 7));
  }
}
// float32: 8 of them, for K 16 s + 8 (l / 32) + 0 .. 7.
template <bool KM, int SIDE>
__device__ __forceinline__ void read_f32(const uint8_t* lds, int base, int s, float v[8]) {
  const int l = threadIdx.x & 63, h = l >> 5, r = base + (l & 31);
  if constexpr (KM) {
    const int c = 4 * s + 2 * h;
    const float4 x = *reinterpret_cast<const float4*>(lds + r * 128 + 16 * (c ^ (r & 7)));
    const float4 y = *reinterpret_cast<const float4*>(lds + r * 128 + 16 * ((c + 1) ^ (r & 7)));
    v[0] = x.x; v[1] = x.y; v[2] = x.z; v[3] = x.w;
    v[4] = y.x; v[5] = y.y; v[6] = y.z; v[7] = y.w;
  } else {
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      const int k = 16 * s + 8 * h + j;
      v[j] = *reinterpret_cast<const float*>(lds + k * (4 * SIDE) + 16 * ((r >> 2) ^ (8 * h)) +
                                             4 * (r & 3));
    }
  }
}

// A wave's part of a step: P x Q blocks of 32 x 32 from row and col on.
template <typename T, bool AKM, bool BKM, int P, int Q, int SIDE_N>
__device__ __forceinline__ void multiply(const uint8_t* a, const uint8_t* b, int row, int col,
                                         f32x16 acc[P][Q]) {
  if constexpr (sizeof(T) == 2) {
#pragma unroll
    for (int s = 0; s < 4; ++s) {
      v8bf x[P], y[Q];
#pragma unroll
      for (int p = 0; p < P; ++p) x[p] = read_bf16<AKM>(a, row + p * 32, s);
#pragma unroll
      for (int q = 0; q < Q; ++q) y[q] = read_bf16<BKM>(b, col + q * 32, s);
#pragma unroll
      for (int p = 0; p < P; ++p)
#pragma unroll
        for (int q = 0; q < Q; ++q)
          acc[p][q] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(y[q], x[p], acc[p][q], 0, 0, 0);
    }
  } else {
#pragma unroll
    for (int s = 0; s < 2; ++s) {
      float x[P][8], y[Q][8];
#pragma unroll
      for (int p = 0; p < P; ++p) read_f32<AKM, TILE>(a, row + p * 32, s, x[p]);
#pragma unroll
      for (int q = 0; q < Q; ++q) read_f32<BKM, SIDE_N>(b, col + q * 32, s, y[q]);
#pragma unroll
      for (int j = 0; j < 8; ++j)
#pragma unroll
        for (int p = 0; p < P; ++p)
#pragma unroll
          for (int q = 0; q < Q; ++q)
            acc[p][q] = __builtin_amdgcn_mfma_f32_32x32x2f32(y[q][j], x[p][j], acc[p][q], 0, 0, 0);
    }
  }
}

// C[r][c] = sum over K of A(r, k) B(c, k), K [0, k) in `splits` parts of `part` each: with one
// part `epi` takes the sums, else `partial` (part i's m rows after those before it). Tiles of 128
// rows and SIDE_N columns, 128 (a wave 64 x 64) or 64 (a wave 32 x 64).
template <typename T, bool AKM, bool BKM, int SIDE_N, typename Epi>
__global__ __launch_bounds__(THREADS, SIDE_N == 64 ? 3 : 2) void tile_kernel(
    Mat<T> A, Mat<T> B, int64_t m, int64_t n, int64_t k, int64_t part, int64_t splits, Epi epi) {
  constexpr int P = SIDE_N / 64, Q = 2;
  constexpr int A_BYTES = TILE * 128, STAGE = A_BYTES + SIDE_N * 128;
  static_assert(2 * STAGE >= 4 * P * UNIT_BYTES, "the outputs' units fit");
  __shared__ __align__(16) uint8_t lds[2 * STAGE];
  const int64_t row_tiles = (m + TILE - 1) / TILE, col_tiles = (n + SIDE_N - 1) / SIDE_N;
  const int64_t tiles = row_tiles * col_tiles, count = tiles * splits;
  // an XCD (workgroup id % 8) takes a contiguous run
  const int64_t id = (blockIdx.x % 8) * ((count + 7) / 8) + blockIdx.x / 8;
  if (blockIdx.x / 8 >= (count + 7) / 8 || id >= count) return;
  const int64_t split = id / tiles;
  int32_t row_tile, col_tile;
  place_of(static_cast<int32_t>(id - split * tiles), static_cast<int32_t>(row_tiles),
           static_cast<int32_t>(col_tiles), &row_tile, &col_tile);
  const int64_t row = static_cast<int64_t>(row_tile) * TILE;
  const int64_t col = static_cast<int64_t>(col_tile) * SIDE_N;
  const int64_t k0 = split * part, kend = k0 + part < k ? k0 + part : k;
  const int wave = threadIdx.x >> 6;
  const int wrow = P == 2 ? 64 * (wave >> 1) : 32 * wave, wcol = P == 2 ? 64 * (wave & 1) : 0;
  f32x16 acc[P][Q];
#pragma unroll
  for (int p = 0; p < P; ++p)
#pragma unroll
    for (int q = 0; q < Q; ++q)
#pragma unroll
      for (int j = 0; j < 16; ++j) acc[p][q][j] = 0.0f;
  Loader<T, AKM, TILE> la(A, row, k0, k, kend);
  Loader<T, BKM, SIDE_N> lb(B, col, k0, k, kend);
  // Two steps' operands are on their way while a third is multiplied.
  struct Step {
    Chunk a[TILE / 32], b[SIDE_N / 32];
  };
  auto load = [&](Step& o, int64_t at) {
    if (at >= kend) return;
    la.step(o.a, at, kend);
    lb.step(o.b, at, kend);
  };
  auto turn = [&](Step& o, int64_t at, uint8_t* s) {
    put_step<T, AKM, TILE>(s, o.a);
    put_step<T, BKM, SIDE_N>(s + A_BYTES, o.b);
    // The last step's reads of the other stage are behind this barrier, so the next step's
    // writes may follow it.
    __syncthreads();
    load(o, at + 2 * BK<T>);
    multiply<T, AKM, BKM, P, Q, SIDE_N>(s, s + A_BYTES, wrow, wcol, acc);
  };
  Step even, odd;
  load(even, k0);
  load(odd, k0 + BK<T>);
  for (int64_t at = k0; at < kend; at += 2 * BK<T>) {
    turn(even, at, lds);
    if (at + BK<T> < kend) turn(odd, at + BK<T>, lds + STAGE);
  }
  __syncthreads();
  uint8_t* const region = lds + wave * (P * UNIT_BYTES);
#pragma unroll
  for (int p = 0; p < P; ++p) put_unit(region + p * UNIT_BYTES, acc[p][0], acc[p][1]);
  wave_done_lds();
  Epi mine = epi;
  if constexpr (std::is_same<Epi, Partial>::value) mine.out += split * m * epi.pitch;
#pragma unroll 1
  for (int u = 0; u < P; ++u)
    store_unit(mine, region + u * UNIT_BYTES, row + wrow + u * 32, col + wcol, m, n);
}

// The sums of the splits' parts, in order, through the epilogue: a thread 8 columns of a row.
template <typename Epi>
__global__ __launch_bounds__(THREADS) void join_kernel(const float* __restrict__ parts,
                                                       int64_t splits, int64_t m, int64_t n,
                                                       int64_t pitch, Epi epi) {
  const int64_t per = pitch / 8;
  const int64_t i = static_cast<int64_t>(blockIdx.x) * THREADS + threadIdx.x;
  if (i >= m * per) return;
  const int64_t row = i / per, col = 8 * (i - row * per);
  const typename Epi::In in = epi.load(row, col);
  float v[8] = {};
  const float* p = parts + row * pitch + col;
  for (int64_t s = 0; s < splits; ++s, p += m * pitch) {
    float w[8];
    Elem<float>::load8(p, w);
#pragma unroll
    for (int j = 0; j < 8; ++j) v[j] += w[j];
  }
  epi.choose([&](auto kind) { epi.store(kind, row, col, v, in); });
}

// Which kernel a product runs on, and the parts of K.
enum class Form { TILE, NARROW, LARGE, FEW };
struct Plan {
  Form form;
  int64_t splits;
};

// The tiles and the parts of K that take the fewest microseconds by a fit to measured times (300 x
// 512 x 512 up to 8192 x 7168 x 4096, within a quarter): a launch; a 256 x 256 tile's unit of 64 K
// takes a CU 1.2, a 128 x 128 tile's step 0.7 where it has the CU to itself and 1.15 beside another
// (float32: 2.7 and 4.1, its MFMAs), a float32 128 x 64 tile's step 1.2, or 1.15 for each on the CU; the
// parts' join is a launch and their sums written and read.
// (1024 x 4096 x 4096: large tiles in 4 parts 48.2 us, 128s 53.4; 2048^3: 128s 30.7, large ones 36.6 at
// best; 201 x 2880 x 5760: 128s in 4 parts 25.4, in one 36.7. float32: 128 x 64 takes 300 x 512 x 512 in
// 12.5 us, 128 x 128 at best 14.9, 3000 x 2000 x 700 83 and 94; 1001 x 1027 x 1443 47 and 46, 1 x 4096 x
// 4096 43 and 42.)
Plan cheapest(bool f32, bool large, int64_t m, int64_t n, int64_t k) {
  Plan best{Form::TILE, 1};
  double least = 1e30;
  for (const Form form : {Form::TILE, Form::NARROW, Form::LARGE}) {
    if (form == Form::LARGE && !large) continue;
    if (form == Form::NARROW && !f32) continue;
    const bool big = form == Form::LARGE, narrow = form == Form::NARROW;
    const int64_t tiles =
        ceil_div(m, big ? 256 : TILE) * ceil_div(n, big ? 256 : narrow ? TILE / 2 : TILE);
    const int64_t steps = ceil_div(k, !big && f32 ? 32 : 64);
    const double alone = f32 ? 2.7 : 0.7, beside = f32 ? 4.1 : 1.15;
    for (int64_t s = 1; s <= 32 && s <= (steps > 1 ? steps : 1) && (s == 1 || s * tiles <= 768);
         s += s < 4 ? 1 : s / 4) {
      // no part has no steps
      const int64_t each = ceil_div(steps, s), splits = s == 1 ? 1 : ceil_div(steps, each);
      const int64_t jobs = tiles * splits;
      const double part = static_cast<double>(each);
      double t = 5;
      if (big) {
        t += static_cast<double>((jobs + 255) >> 8) * (1.2 * part + 5);
      } else if (narrow) {
        const int64_t on = (jobs + 255) >> 8;  // a CU's
        t += on == 1 ? 1.2 * part + 2 : 1.15 * static_cast<double>(on) * part + 2 * ((on + 2) / 3);
      } else {
        const int64_t rest = jobs & 511;
        t += static_cast<double>(jobs >> 9) * (beside * part + 2);
        if (rest > 0) t += (rest > 256 ? beside : alone) * part + 2;
      }
      if (splits > 1) t += 2.5 + static_cast<double>(splits * m) * n * 8e-7;
      if (t < least) {
        least = t;
        best = Plan{form, splits};
      }
    }
  }
  return best;
}
// ... kept for the shapes that this thread asked for last: a call asks several times.
Plan plan_of(bool f32, bool large, bool few, int64_t m, int64_t n, int64_t k) {
  if (few) return Plan{Form::FEW, few_splits(n, k)};
  struct Entry {
    int64_t m, n, k;
    Plan plan;
  };
  static thread_local Entry kept[64] = {};
  const uint64_t at = (static_cast<uint64_t>(m) * 31 + static_cast<uint64_t>(n) * 7 +
                       static_cast<uint64_t>(k)) % 16;
  Entry& e = kept[at * 4 + (f32 ? 2 : 0) + (large ? 1 : 0)];
  if (e.m != m || e.n != n || e.k != k) e = Entry{m, n, k, cheapest(f32, large, m, n, k)};
  return e.plan;
}

// What any form may ask for: the operands' alignment decides between them, which is not known here.
size_t workspace_for(bool f32, int64_t m, int64_t n, int64_t k) {
  int64_t most = plan_of(f32, false, false, m, n, k).splits;
  if (!f32) {
    const int64_t large = plan_of(f32, true, false, m, n, k).splits;
    if (large > most) most = large;
    if (m <= 64 && few_splits(n, k) > most) most = few_splits(n, k);
  }
  return most == 1 ? 0 : static_cast<size_t>(most) * m * pitch_of(n) * sizeof(float);
}

// m, n > 0.
template <typename T, bool AKM, bool BKM, typename Epi>
int run(const char* name, const Mat<T>& A, const Mat<T>& B, int64_t m, int64_t n, int64_t k,
        const Epi& epi, void* workspace, size_t workspace_bytes, hipStream_t s) {
  const size_t need = workspace_for(sizeof(T) == 4, m, n, k);
  if (need > 0 && (workspace == nullptr || workspace_bytes < need))
    return fail(BUX_E_WORKSPACE, "%s: workspace of %zu bytes, %zu needed", name, workspace_bytes,
                need);
  BUX_CHECK(reinterpret_cast<uintptr_t>(workspace) % 16 == 0, "%s: unaligned workspace", name);
  bool large = false, few = false;
  if constexpr (sizeof(T) == 2) {
    large = large_takes(A, AKM, B, BKM, m, n, k);
    few = AKM && few_takes(A, B, m, n, k);
  }
  const Plan plan = plan_of(sizeof(T) == 4, large, few, m, n, k);
  const int64_t splits = plan.splits, pitch = pitch_of(n);
  auto launch = [&](const auto& e) {
    if constexpr (sizeof(T) == 2) {
      if constexpr (AKM) {
        if (plan.form == Form::FEW) return launch_few<BKM>(A, B, m, n, k, splits, e, s);
      }
      if (plan.form == Form::LARGE)
        return launch_large<AKM, BKM>(A, B, m, n, k, ceil_div(ceil_div(k, 64), splits), splits, e, s);
    }
    auto tiles = [&](auto side) {
      constexpr int SIDE_N = decltype(side)::value;
      const int64_t blocks = 8 * ceil_div(ceil_div(m, TILE) * ceil_div(n, SIDE_N) * splits, 8);
      if (blocks >= (1LL << 31)) return fail(BUX_E_ARGUMENT, "%s: too many tiles", name);
      const int64_t part = ceil_div(ceil_div(k, BK<T>), splits) * BK<T>;
      hipLaunchKernelGGL((tile_kernel<T, AKM, BKM, SIDE_N, std::decay_t<decltype(e)>>),
                         dim3(static_cast<unsigned>(blocks)), dim3(THREADS), 0, s, A, B, m, n, k,
                         part, splits, e);
      return launched("dense tile_kernel");
    };
    if constexpr (sizeof(T) == 4) {
      if (plan.form == Form::NARROW) return tiles(std::integral_constant<int, TILE / 2>{});
    }
    return tiles(std::integral_constant<int, TILE>{});
  };
  if (splits == 1) return launch(epi);
  float* const parts = static_cast<float*>(workspace);
  if (int rc = launch(Partial{parts, pitch})) return rc;
  const int64_t threads = m * (pitch / 8);
  BUX_CHECK(ceil_div(threads, THREADS) < (1LL << 31), "%s: too many rows", name);
  hipLaunchKernelGGL(join_kernel<Epi>, dim3(static_cast<unsigned>(ceil_div(threads, THREADS))),
                     dim3(THREADS), 0, s, parts, splits, m, n, pitch, epi);
  return launched("dense join_kernel");
}

constexpr int64_t MOST = 1LL << 31;

int check_shape(const char* name, int64_t m, int64_t n, int64_t k) {
  BUX_CHECK(m >= 0 && n > 0 && k > 0, "%s: bad shape m=%lld n=%lld k=%lld", name, (long long)m,
            (long long)n, (long long)k);
  BUX_CHECK(m < MOST && n < MOST && k < MOST, "%s: m=%lld n=%lld k=%lld: each below 2^31", name,
            (long long)m, (long long)n, (long long)k);
  return BUX_OK;
}

// ffn, or no activation where it is NULL.
int act_or_none(const char* name, const bux_ffn* ffn, Act* act) {
  if (ffn != nullptr) return act_of(name, ffn, act);
  *act = Act{NO_ACT, 0, 0, 0.0f, 0, 0.0f, 0.0f};
  return BUX_OK;
}

template <typename T>
int rows(const char* name, const T* x, const T* w, int transposed, int64_t m, int64_t n, int64_t k,
         const T* bias, const bux_ffn* ffn, const T* residual, T* product, uint8_t* low, T* out,
         void* workspace, size_t workspace_bytes, void* stream) {
  clear_error();
  if (int rc = check_shape(name, m, n, k)) return rc;
  Act act;
  if (int rc = act_or_none(name, ffn, &act)) return rc;
  BUX_CHECK(!act.gated || (n % 2 == 0 && residual == nullptr),
            "%s: a gated activation takes an even n (%lld) and no residual", name, (long long)n);
  BUX_CHECK(low == nullptr || product != nullptr, "%s: low bytes without the product", name);
  if (m == 0) return BUX_OK;
  BUX_CHECK(x && w && out, "%s: NULL buffer", name);
  hipStream_t s = as_stream(stream);
  const Mat<T> A{x, k, m}, B{w, transposed ? k : n, n};
  auto with = [&](auto epi) {
    return transposed ? run<T, true, true>(name, A, B, m, n, k, epi, workspace, workspace_bytes, s)
                      : run<T, true, false>(name, A, B, m, n, k, epi, workspace, workspace_bytes, s);
  };
  if (act.gated) return with(Forward<T, true>{act, bias, residual, product, low, out, n});
  return with(Forward<T, false>{act, bias, residual, product, low, out, n});
}

template <typename T>
int units_backward(const char* name, const T* dy, const T* down, int64_t m, int64_t f, int64_t d,
                   const T* product, const uint8_t* low, const bux_ffn* ffn, T* dp,
                   uint8_t* dp_low, void* workspace, size_t workspace_bytes, void* stream) {
  clear_error();
  if (int rc = check_shape(name, m, f, d)) return rc;
  Act act;
  if (int rc = act_of(name, ffn, &act)) return rc;
  if (m == 0) return BUX_OK;
  BUX_CHECK(dy && down && product && dp, "%s: NULL buffer", name);
  hipStream_t s = as_stream(stream);
  const Mat<T> A{dy, d, m}, B{down, d, f};
  if (act.gated)
    return run<T, true, true>(name, A, B, m, f, d, Backward<T, true>{act, product, low, dp, dp_low, f},
                              workspace, workspace_bytes, s);
  return run<T, true, true>(name, A, B, m, f, d, Backward<T, false>{act, product, low, dp, dp_low, f}, workspace,
                            workspace_bytes, s);
}

template <typename T>
int contract(const char* name, const T* x, const T* dy, int64_t m, int64_t k, int64_t n, T* dw,
             void* workspace, size_t workspace_bytes, void* stream) {
  clear_error();
  if (int rc = check_shape(name, m, n, k)) return rc;
  BUX_CHECK(dw && (m == 0 || (x && dy)), "%s: NULL buffer", name);
  const Act none{NO_ACT, 0, 0, 0.0f, 0, 0.0f, 0.0f};
  const Mat<T> A{x, k, k}, B{dy, n, n};
  return run<T, false, false>(name, A, B, k, n, m,
                              Forward<T, false>{none, nullptr, nullptr, nullptr, nullptr, dw, n}, workspace,
                              workspace_bytes, as_stream(stream));
}

// --- the activation's gradient alone, and sums over the rows ---------------------------------
//
// dz = dy act'(product) (dy itself without a product) and the column sums of it before its
// rounding. L lanes (a power of two) take a row's 8 L columns, 256 / L rows a workgroup; its
// sums over the rows that it takes in turn meet in LDS and, where there are more workgroups
// along the rows, are added in order by a second kernel.

constexpr int64_t MAX_RUNS = 256;  // workgroups along the rows

int lanes_of(int64_t n) {
  int l = 1;
  while (l < 64 && 8 * l < n) l *= 2;
  return l;
}
int64_t runs_of(int64_t m, int64_t n) {
  const int64_t rows = THREADS / lanes_of(n), strips = ceil_div(n, 8 * lanes_of(n));
  int64_t r = ceil_div(m, 4 * rows);  // 4 turns a workgroup at least
  const int64_t most = 2048 / strips > 1 ? 2048 / strips : 1;
  if (r > most) r = most;
  if (r > MAX_RUNS) r = MAX_RUNS;
  return r < 1 ? 1 : r;
}

template <typename T>
__global__ __launch_bounds__(THREADS) void slope_kernel(const T* __restrict__ dy,
                                                        const uint8_t* __restrict__ dy_low,
                                                        const T* __restrict__ product, Act act,
                                                        int64_t m, int64_t n, int lanes,
                                                        T* __restrict__ dz, T* __restrict__ sums,
                                                        float* __restrict__ parts) {
  __shared__ float red[THREADS][9];
  const int lane = threadIdx.x % lanes, sub = threadIdx.x / lanes, rows = THREADS / lanes;
  const int64_t col = (static_cast<int64_t>(blockIdx.x) * lanes + lane) * 8, count = n - col;
  float sum[8] = {};
  if (count > 0) {
    of_act<false>(act, [&](auto kind) {
      using K = decltype(kind);
      constexpr int TURN = 4;  // rows on their way at once
      constexpr bool PLAIN = std::is_same<K, NoAct>::value;
      const int64_t stride = static_cast<int64_t>(gridDim.y) * rows;
      for (int64_t r0 = static_cast<int64_t>(blockIdx.y) * rows + sub; r0 < m; r0 += TURN * stride) {
        Eight<T> g[TURN], z[TURN];
        uint64_t low[TURN];
#pragma unroll
        for (int i = 0; i < TURN; ++i) {
          const int64_t r = r0 + i * stride;
          g[i] = load_eight(dy + r * n + col, r < m ? count : 0);
          if (PLAIN && sizeof(T) == 2 && dy_low) low[i] = load_low(dy_low + r * n + col, r < m ? count : 0);
          if (!PLAIN) z[i] = load_eight(product + r * n + col, r < m ? count : 0);
        }
#pragma unroll
        for (int i = 0; i < TURN; ++i) {
          const int64_t r = r0 + i * stride;
          if (r >= m) break;
          float v[8];
          if constexpr (PLAIN) {
#pragma unroll
            for (int j = 0; j < 8; ++j) v[j] = g[i].value(j);
            if (sizeof(T) == 2 && dy_low) {
#pragma unroll
              for (int j = 0; j < 8; ++j) v[j] = with_low(v[j], low[i], j);
            }
          } else {
#pragma unroll
            for (int j = 0; j < 8; ++j) {
              float dg;
              unit_grad_of<K, sizeof(T) == 4>(act, z[i].value(j), 0.0f, g[i].value(j), &v[j], &dg);
            }
          }
          if (dz) store_some<T>(dz + r * n + col, v, count);
#pragma unroll
          for (int j = 0; j < 8; ++j) sum[j] += v[j];
        }
      }
    });
  }
  if (!sums) return;
#pragma unroll
  for (int j = 0; j < 8; ++j) red[threadIdx.x][j] = sum[j];
  __syncthreads();
  if (sub != 0 || count <= 0) return;
  for (int s = 1; s < rows; ++s)
#pragma unroll
    for (int j = 0; j < 8; ++j) sum[j] += red[s * lanes + lane][j];
  if (gridDim.y == 1) {
    store_some<T>(sums + col, sum, count);
  } else {
    float* const p = parts + blockIdx.y * n + col;
#pragma unroll
    for (int j = 0; j < 8; ++j)
      if (j < count) p[j] = sum[j];
  }
}

// 64 columns a workgroup: its 4 waves take the runs in turn, and their sums meet in order.
template <typename T>
__global__ __launch_bounds__(THREADS) void sums_kernel(const float* __restrict__ parts,
                                                       int64_t runs, int64_t n,
                                                       T* __restrict__ sums) {
  __shared__ float red[THREADS];
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const int64_t c = static_cast<int64_t>(blockIdx.x) * 64 + lane;
  float v = 0.0f;
  if (c < n) {
#pragma unroll 8
    for (int64_t r = wave; r < runs; r += THREADS / 64) v += parts[r * n + c];
  }
  red[threadIdx.x] = v;
  __syncthreads();
  if (wave != 0 || c >= n) return;
#pragma unroll
  for (int w = 1; w < THREADS / 64; ++w) v += red[64 * w + lane];
  sums[c] = Elem<T>::make(v);
}

template <typename T>
int slope(const char* name, const T* dy, const uint8_t* dy_low, const T* product, const bux_ffn* ffn, int64_t m, int64_t n,
          T* dz, T* sums, void* workspace, size_t workspace_bytes, void* stream) {
  clear_error();
  if (int rc = check_shape(name, m, n, 1)) return rc;
  Act act;
  if (int rc = act_or_none(name, ffn, &act)) return rc;
  BUX_CHECK(!act.gated, "%s: a gated activation", name);
  // (of no rows dy, product and dz are empty: their addresses may be NULL)
  BUX_CHECK(m == 0 || (ffn == nullptr) == (product == nullptr),
            "%s: an activation's gradient takes its product", name);
  BUX_CHECK(m == 0 || dz || sums, "%s: nothing asked for", name);
  BUX_CHECK(dy_low == nullptr || (ffn == nullptr && dz == nullptr),
            "%s: low bytes are for dy's own sums", name);
  BUX_CHECK(m == 0 || dy, "%s: NULL buffer", name);
  const int64_t runs = runs_of(m, n);
  const size_t need = sums && runs > 1 ? static_cast<size_t>(runs) * n * sizeof(float) : 0;
  if (need > 0 && (workspace == nullptr || workspace_bytes < need))
    return fail(BUX_E_WORKSPACE, "%s: workspace of %zu bytes, %zu needed", name, workspace_bytes,
                need);
  if (m == 0 && !sums) return BUX_OK;
  const int lanes = lanes_of(n);
  hipStream_t s = as_stream(stream);
  float* const parts = static_cast<float*>(workspace);
  hipLaunchKernelGGL(slope_kernel<T>, dim3(static_cast<unsigned>(ceil_div(n, 8 * lanes)),
                                           static_cast<unsigned>(runs)),
                     dim3(THREADS), 0, s, dy, dy_low, product, act, m, n, lanes, dz, sums, parts);
  if (int rc = launched("dense slope_kernel")) return rc;
  if (!sums || runs == 1) return BUX_OK;
  hipLaunchKernelGGL(sums_kernel<T>, dim3(static_cast<unsigned>(ceil_div(n, 64))),
                     dim3(THREADS), 0, s, parts, runs, n, sums);
  return launched("dense sums_kernel");
}

}  // namespace
}  // namespace bux

extern "C" size_t bux_dense_workspace_size(int64_t m, int64_t n, int64_t k) {
  using namespace bux;
  if (m <= 0 || n <= 0 || k <= 0) return 0;
  const size_t a = workspace_for(false, m, n, k), b = workspace_for(true, m, n, k);
  return a > b ? a : b;
}
extern "C" size_t bux_dense_slope_workspace_size(int64_t m, int64_t n) {
  using namespace bux;
  if (m <= 0 || n <= 0 || runs_of(m, n) == 1) return 0;
  return static_cast<size_t>(runs_of(m, n)) * n * sizeof(float);
}

extern "C" int bux_dense_rows(const uint16_t* x, const uint16_t* w, int transposed, int64_t m,
                              int64_t n, int64_t k, const uint16_t* bias, const bux_ffn* ffn,
                              const uint16_t* residual, uint16_t* product, uint8_t* product_low,
                              uint16_t* out, void* workspace, size_t workspace_bytes,
                              void* stream) {
  return bux::rows("bux_dense_rows", x, w, transposed, m, n, k, bias, ffn, residual, product,
                   product_low, out, workspace, workspace_bytes, stream);
}
extern "C" int bux_dense_rows_f32(const float* x, const float* w, int transposed, int64_t m,
                                  int64_t n, int64_t k, const float* bias, const bux_ffn* ffn,
                                  const float* residual, float* product, float* out,
                                  void* workspace, size_t workspace_bytes, void* stream) {
  return bux::rows<float>("bux_dense_rows_f32", x, w, transposed, m, n, k, bias, ffn, residual,
                          product, nullptr, out, workspace, workspace_bytes, stream);
}
extern "C" int bux_dense_units_backward(const uint16_t* dy, const uint16_t* down, int64_t m,
                                        int64_t f, int64_t d, const uint16_t* product,
                                        const uint8_t* product_low, const bux_ffn* ffn,
                                        uint16_t* dp, uint8_t* dp_low, void* workspace,
                                        size_t workspace_bytes, void* stream) {
  return bux::units_backward("bux_dense_units_backward", dy, down, m, f, d, product, product_low,
                             ffn, dp, dp_low, workspace, workspace_bytes, stream);
}
extern "C" int bux_dense_units_backward_f32(const float* dy, const float* down, int64_t m,
                                            int64_t f, int64_t d, const float* product,
                                            const bux_ffn* ffn, float* dp, void* workspace,
                                            size_t workspace_bytes, void* stream) {
  return bux::units_backward<float>("bux_dense_units_backward_f32", dy, down, m, f, d, product,
                                    nullptr, ffn, dp, nullptr, workspace, workspace_bytes, stream);
}
extern "C" int bux_dense_contract(const uint16_t* x, const uint16_t* dy, int64_t m, int64_t k,
                                  int64_t n, uint16_t* dw, void* workspace, size_t workspace_bytes,
                                  void* stream) {
  return bux::contract("bux_dense_contract", x, dy, m, k, n, dw, workspace, workspace_bytes, stream);
}
extern "C" int bux_dense_contract_f32(const float* x, const float* dy, int64_t m, int64_t k,
                                      int64_t n, float* dw, void* workspace,
                                      size_t workspace_bytes, void* stream) {
  return bux::contract("bux_dense_contract_f32", x, dy, m, k, n, dw, workspace, workspace_bytes,
                       stream);
}
extern "C" int bux_dense_slope(const uint16_t* dy, const uint8_t* dy_low, const uint16_t* product,
                               const bux_ffn* ffn, int64_t m, int64_t n, uint16_t* dz,
                               uint16_t* sums, void* workspace, size_t workspace_bytes,
                               void* stream) {
  return bux::slope("bux_dense_slope", dy, dy_low, product, ffn, m, n, dz, sums, workspace, workspace_bytes,
                    stream);
}
extern "C" int bux_dense_slope_f32(const float* dy, const float* product, const bux_ffn* ffn,
                                   int64_t m, int64_t n, float* dz, float* sums, void* workspace,
                                   size_t workspace_bytes, void* stream) {
  return bux::slope<float>("bux_dense_slope_f32", dy, nullptr, product, ffn, m, n, dz, sums, workspace,
                    workspace_bytes, stream);
}
