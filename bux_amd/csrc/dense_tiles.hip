// Dense bfloat16 products in 256 x 256 tiles: for outputs of enough tiles to fill the chip.
//
// A persistent grid, a workgroup of 4 waves a CU, each wave 128 x 128 of a tile as 8 x 8 MFMAs of
// 16 x 16 x 32 (256 accumulator registers). Operands come in units of 64 K, 32 KiB: 256 rows of
// 128 bytes (K-major) or 64 K rows of 512 bytes (MN-major), whole cache lines either way, by
// direct loads into a ring of 5 slots, the CU's 160 KiB. (Of K-major rows 64 bytes at a time,
// as the experts' kernels load them, each line comes through L1 twice: x w^T of 8192^3 ran at
// 1.24 PFLOP/s.)
//
// The units of all of a workgroup's tiles form one stream, A's and B's in turn. A pair of units is
// two steps of 64 MFMAs a wave; while one step's MFMAs run, the other operand registers take the
// next step's from LDS. Pair p's first step issues A's unit of pair p + 2, its second B's. The
// one barrier a pair stands between the steps: pair p + 1 is then whole, and every wave has read
// pair p, whose slots the next units take.
//
// K-major units: chunk c (16 bytes) of row r at place c ^ (r % 8): 8 lanes that read one chunk of
// 8 rows take 32 banks. MN-major: chunk c of K row k at c ^ 4 (k % 4) ^ 2 (k / 8 %
// 2), read by ds_read_b64_tr_b16 (32 lanes: 8 K rows x 32 bytes, on banks of their own).
//
// The epilogue (dense.h) goes through the last pair's two slots, while the next tile's first three
// units are in flight in the others. K positions past k are zeroed in both operands' registers.

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

constexpr int THREADS = 256;
constexpr int TILE = 256;
constexpr int UNIT_K = 64;
constexpr int SLOT = TILE * UNIT_K * 2;  // bytes
constexpr int SLOTS = 5;
constexpr int LOADS = SLOT / 1024 / 4;  // a wave's direct loads of a unit

// An operand's units of a tile: this lane's offset (of a wave's even and odd loads), the scalar
// bytes from one of a wave's loads to the next and from one unit to the next.
struct Loads {
  i32x4 rsrc;
  int32_t voff[2];
  int32_t slice, step;
};
struct Operand {
  const uint16_t* p;
  int64_t ld, rows, k;
};

template <bool KM>
__device__ __forceinline__ Loads loads_of(const Operand& o, int64_t row0) {
  const int w = threadIdx.x >> 6, l = threadIdx.x & 63;
  const int32_t ld = static_cast<int32_t>(o.ld);
  Loads r;
  r.slice = 8 * ld * 2;
  if (KM) {  // load i of wave w: rows 64 w + 8 i .. + 7
    const int64_t bytes = (o.rows - row0) * o.ld * 2;
    r.rsrc = resource(o.p + row0 * o.ld, bytes < 0x7fffffff ? bytes : 0x7fffffff);
    r.voff[0] = r.voff[1] = (64 * w + (l >> 3)) * ld * 2 + 16 * ((l & 7) ^ (l >> 3));
    r.step = UNIT_K * 2;
  } else {  // K rows 8 i + 2 w and + 1
    const int k = 2 * w + (l >> 5);
    r.rsrc = resource(o.p, o.k * o.ld * 2);
#pragma unroll
    for (int odd = 0; odd < 2; ++odd)
      r.voff[odd] = k * ld * 2 + static_cast<int32_t>(row0) * 2 +
                    16 * ((l & 31) ^ (4 * (k & 3)) ^ (2 * odd));
    r.step = UNIT_K * ld * 2;
  }
  return r;
}
// Where a wave's load 0 lands in a slot, and how much further each next one.
template <bool KM>
__device__ __forceinline__ uint32_t wave_at() {
  return __builtin_amdgcn_readfirstlane(threadIdx.x >> 6) * (KM ? 8192 : 1024);
}
template <bool KM>
constexpr int LOAD_AT = KM ? 1024 : 4096;

// Load I of a unit whose first load's place is `at` and whose bytes begin at `from`; as load_lds16
// (common.h), with one scalar instruction for the place.
template <bool KM, int I>
__device__ __forceinline__ void load_slice(const Loads& o, uint32_t at, int32_t from) {
  asm volatile("s_add_u32 m0, %0, %4\n\tbuffer_load_dwordx4 %1, %2, %3 offen lds"
               :: "s"(at), "v"(o.voff[I & 1]), "s"(o.rsrc), "s"(from + I * o.slice),
                  "n"(I * LOAD_AT<KM>)
               : "memory", "m0", "scc");
}
template <bool KM, int I = 0>
__device__ __forceinline__ void load_unit(const Loads& o, uint32_t at, int32_t from) {
  load_slice<KM, I>(o, at, from);
  if constexpr (I + 1 < LOADS) load_unit<KM, I + 1>(o, at, from);
}

// This lane's offsets in a slot of its MFMA operands, 16 rows x 32 K of them (row l % 16, K 8 (l /
// 16) .. + 7): K-major, of 32 K s (0, 1) of row block 0 (block p 2048 bytes further); MN-major, of
// the first read of block p (32 K s 16384 s bytes further, the second read 2048).
template <bool KM>
struct Lanes {
  static constexpr int N = KM ? 2 : 8;
  int32_t at[N];
  __device__ __forceinline__ explicit Lanes(int base) {
    const int l = threadIdx.x & 63, g = l >> 4;
    if (KM) {
      const int r = base + (l & 15);
#pragma unroll
      for (int s = 0; s < N; ++s) at[s] = r * 128 + 16 * ((4 * s + g) ^ (r & 7));
    } else {
      const int q = l & 15, kq = q >> 2, col = 4 * (q & 3);
#pragma unroll
      for (int p = 0; p < N; ++p)
        at[p] = (8 * g + kq) * 512 +
                16 * (base / 8 + ((2 * p) ^ (4 * kq) ^ (2 * (g & 1))) + (col >> 3)) +
                8 * ((col >> 2) & 1);
    }
  }
};
// The address of one of them in a slot, kept from being taken apart again: what follows is added by
// the read's own offset.
__device__ __forceinline__ uint32_t in_slot(uint32_t slot, int32_t at) {
  uint32_t r;
  asm("v_add_u32 %0, %1, %2" : "=v"(r) : "s"(slot), "v"(at));
  return r;
}

// A wave's operands of a step: 8 blocks of 16 rows of A and of B, 32 K.
struct Frag {
  v8bf a[8], b[8];
};
// The reads of step SUB of a pair in the slots a and b, 16 of them, in the order its MFMAs take
// them.
template <bool AKM, bool BKM, int SUB>
struct Reader {
  const Lanes<AKM>& la;
  const Lanes<BKM>& lb;
  uint32_t a, b, a0, b0;
  __device__ __forceinline__ Reader(const Lanes<AKM>& la, const Lanes<BKM>& lb, uint32_t a,
                                    uint32_t b)
      : la(la), lb(lb), a(a), b(b) {
    if (AKM) a0 = in_slot(a, la.at[SUB]);
    if (BKM) b0 = in_slot(b, lb.at[SUB]);
  }
  template <bool KM>
  static __device__ __forceinline__ v8bf block(const Lanes<KM>& o, uint32_t slot, uint32_t first,
                                               int p) {
    if constexpr (KM) {
      return __builtin_bit_cast(v8bf, *reinterpret_cast<const lds_u4*>(first + p * 2048));
    } else {
      const uint32_t at = in_slot(slot, o.at[p]) + SUB * 16384;
      const v4s x = __builtin_amdgcn_ds_read_tr16_b64_v4i16(reinterpret_cast<lds_v4s*>(at));
      const v4s y = __builtin_amdgcn_ds_read_tr16_b64_v4i16(reinterpret_cast<lds_v4s*>(at + 2048));
      return __builtin_bit_cast(v8bf, __builtin_shufflevector(x, y, 0, 1, 2, 3, 4, 5, 6, 7));
    }
  }
  __device__ __forceinline__ void read(Frag& f, int x) const {
    if (x == 0) f.a[0] = block<AKM>(la, a, a0, 0);
    else if (x <= 8) f.b[x - 1] = block<BKM>(lb, b, b0, x - 1);
    else f.a[x - 8] = block<AKM>(la, a, a0, x - 8);
  }
};

// Zeroes the elements of v whose K (k0 + e) is not below `end`.
__device__ __forceinline__ v8bf below(v8bf v, int32_t k0, int32_t end) {
  u32x4 u = __builtin_bit_cast(u32x4, v);
#pragma unroll
  for (int d = 0; d < 4; ++d) {
    const int32_t k = k0 + 2 * d;
    u[d] &= (k < end ? 0xffffu : 0u) | (k + 1 < end ? 0xffff0000u : 0u);
  }
  return __builtin_bit_cast(v8bf, u);
}
// ... of step SUB of a pair of which `left` K positions count.
template <int SUB>
__device__ __forceinline__ void mask(Frag& f, int32_t left) {
  const int g = (threadIdx.x & 63) >> 4;
#pragma unroll
  for (int p = 0; p < 8; ++p) {
    f.a[p] = below(f.a[p], 32 * SUB + 8 * g, left);
    f.b[p] = below(f.b[p], 32 * SUB + 8 * g, left);
    asm volatile("s_nop 1" : "+v"(f.a[p]), "+v"(f.b[p]));  // an MFMA reads them 2 waits later
  }
}

// acc += a b^T of blocks of 16 rows x 32 K. In assembly so that the sums stay in accumulator
// registers: of 64 blocks of the builtin's the compiler moves some in and out of others at every
// turn of the K loop. It sees no MFMA here and so inserts none of the waits that one needs: the
// callers do (`settled`).
__device__ __forceinline__ void multiply(const v8bf& a, const v8bf& b, f32x4& acc) {
  asm volatile("v_mfma_f32_16x16x32_bf16 %0, %1, %2, %0" : "+a"(acc) : "v"(a), "v"(b));
}
// Between the sums' last MFMA and what reads them (a 16-pass MFMA's result takes 19 waits, this one's
// fewer), or between what wrote them and their first (2).
__device__ __forceinline__ void settled(f32x4 acc[8][8]) {
  auto pin = [&] {
#pragma unroll
    for (int i = 0; i < 8; ++i)
#pragma unroll
      for (int j = 0; j < 8; ++j) asm volatile("" : "+a"(acc[i][j]));
  };
  pin();
  asm volatile("s_nop 15\n\ts_nop 15" ::: "memory");
  pin();
}

// Load I (0 .. 7) by a runtime constant.
template <bool KM>
__device__ __forceinline__ void load_one(const Loads& o, uint32_t at, int32_t from, int i) {
  switch (i) {
    case 0: load_slice<KM, 0>(o, at, from); break;
    case 1: load_slice<KM, 1>(o, at, from); break;
    case 2: load_slice<KM, 2>(o, at, from); break;
    case 3: load_slice<KM, 3>(o, at, from); break;
    case 4: load_slice<KM, 4>(o, at, from); break;
    case 5: load_slice<KM, 5>(o, at, from); break;
    case 6: load_slice<KM, 6>(o, at, from); break;
    default: load_slice<KM, 7>(o, at, from);
  }
}

// The 64 MFMAs of a step on `cur`; in the first half, with READ, the next step's operands into
// `nxt`, so that none is still on its way at the barrier; in the second, with LOAD, a unit's loads
// of a KM operand. One wave a SIMD issues all of it in order: what an MFMA's 16 cycles do not
// cover, it waits for, scalar instructions too.
template <bool KM, bool LOAD, bool READ, typename R>
__device__ __forceinline__ void step(const Frag& cur, Frag& nxt, const Loads& from, uint32_t at,
                                     int32_t bytes, const R& reader, f32x4 acc[8][8]) {
#pragma unroll
  for (int q = 0; q < 64; ++q) {
    const int i = q >> 3, j = q & 7;
    multiply(cur.b[j], cur.a[i], acc[i][j]);
    __builtin_amdgcn_sched_barrier(0);
    if (LOAD && q >= 32 && (q & 3) == 0) load_one<KM>(from, at, bytes, (q - 32) >> 2);
    if (READ && q < 32 && (q & 1) == 0) reader.read(nxt, q >> 1);
    __builtin_amdgcn_sched_barrier(0);
  }
}

// Waits until at most `units` units' loads of this wave are in flight. (Its stores count too: then
// it waits longer, never too little.)
template <int units>
__device__ __forceinline__ void wait_units() {
  static_assert(units == 1 || units == 2, "");
  if (units == 2) asm volatile("s_waitcnt vmcnt(16)" ::: "memory");
  else asm volatile("s_waitcnt vmcnt(8)" ::: "memory");
}
// This wave's LDS reads and writes are done, then the workgroup's barrier; loads stay in flight.
__device__ __forceinline__ void barrier_lds() {
  asm volatile("s_waitcnt lgkmcnt(0)\n\ts_barrier" ::: "memory");
}

// Two rows of 8 blocks of sums, 32 rows x 128 columns, as two units (dense.h): lane l has row l % 16
// of a block and columns 4 (l / 16) .. + 3.
__device__ __forceinline__ void put_blocks(uint8_t* r0, uint8_t* r1, const f32x4 lo[8],
                                           const f32x4 hi[8]) {
  const int lane = threadIdx.x & 63, r = lane & 15, g = lane >> 4;
#pragma unroll
  for (int j = 0; j < 8; ++j) {
    uint8_t* const at = (j < 4 ? r0 : r1) + r * 256 + 16 * ((4 * (j & 3) + g) ^ r);
    *reinterpret_cast<f32x4*>(at) = lo[j];
    *reinterpret_cast<f32x4*>(at + 16 * 256) = hi[j];
  }
}

// The i-th 32 rows of a wave's 128. (Without marks of their own around them the compiler makes one
// of the cases, its sums taken by an index from memory.)
__device__ __forceinline__ void put_rows(int i, uint8_t* r0, uint8_t* r1, const f32x4 (&acc)[8][8]) {
#define BUX_ROWS(I)                                     \
  asm volatile("; rows %0" ::"n"(I) : "memory");        \
  put_blocks(r0, r1, acc[2 * I], acc[2 * I + 1]);       \
  asm volatile("; rows %0 put" ::"n"(I) : "memory");    \
  break;
  switch (i) {
    case 0: BUX_ROWS(0)
    case 1: BUX_ROWS(1)
    case 2: BUX_ROWS(2)
    default: BUX_ROWS(3)
  }
#undef BUX_ROWS
  wave_done_lds();
}

struct Job {
  int32_t row, col;    // the tile's corner
  int32_t unit, n;     // its K: units from `unit` on
  int32_t split;
};

template <bool AKM, bool BKM, typename Epi>
__global__ __launch_bounds__(THREADS) __attribute__((amdgpu_waves_per_eu(1, 1))) void large_kernel(
    Operand A, Operand B, int32_t m, int32_t n, int32_t k, int32_t units, int32_t row_tiles,
    int32_t col_tiles, int32_t count, Epi epi) {
  extern __shared__ __align__(16) uint8_t lds[];
  const int wave = threadIdx.x >> 6;
  // XCD x (workgroup id % 8) takes a contiguous run of the tiles, its workgroups in turn
  const int32_t per = (count + 7) / 8, lo = static_cast<int32_t>(blockIdx.x % 8) * per;
  const int32_t end = lo + per < count ? lo + per : count;
  const int32_t stride = gridDim.x / 8, tiles = row_tiles * col_tiles;
  const int32_t all = (k + UNIT_K - 1) / UNIT_K;  // units of K
  int32_t id = lo + static_cast<int32_t>(blockIdx.x / 8);
  if (id >= end) return;
  auto job_of = [&](int32_t at) {
    Job j;
    j.split = at / tiles;
    place_of(at - j.split * tiles, row_tiles, col_tiles, &j.row, &j.col);
    j.row *= TILE;
    j.col *= TILE;
    j.unit = j.split * units;
    j.n = all - j.unit < units ? all - j.unit : units;
    return j;
  };
  const uint32_t lds0 = lds_at(lds);
  const Lanes<AKM> ra((wave >> 1) * 128);
  const Lanes<BKM> rb((wave & 1) * 128);
  Job job = job_of(id);
  Loads la = loads_of<AKM>(A, job.row), lb = loads_of<BKM>(B, job.col);
  const bool aligned = epi.aligned();
  int32_t base = 0;   // the slot of this tile's unit 0
  int32_t ahead = 0;  // this tile's stream's units issued before it began
  for (;;) {
    const bool more = id + stride < end;
    const Job next = more ? job_of(id + stride) : job;
    Loads na = loads_of<AKM>(A, next.row), nb = loads_of<BKM>(B, next.col);
    const int32_t pairs = job.n, then = more ? next.n : 0;
    // Past the last tile the loads read nothing (zeros land in a slot that nothing reads): a wave's
    // loads in flight are always whole units.
    if (!more) na.rsrc[2] = nb.rsrc[2] = 0;
    // Unit u of the stream from this tile's first on: even A's, odd B's, of this tile's pair u / 2
    // or of the next tile's.
    auto slot = [&](int32_t u) { return lds0 + static_cast<uint32_t>((base + u) % SLOTS) * SLOT; };
    auto pick = [&](const Loads& mine, const Loads& theirs, int32_t p, int32_t* bytes) {
      const bool here = p < pairs;
      Loads o = here ? mine : theirs;
      if (p >= pairs + then) o.rsrc[2] = 0;
      *bytes = (here ? job.unit + p : next.unit + p - pairs) * o.step;
      return o;
    };
    for (int32_t u = ahead; u < 4; ++u) {
      int32_t bytes;
      if (u & 1) {
        const Loads o = pick(lb, nb, u >> 1, &bytes);
        load_unit<BKM>(o, slot(u) + wave_at<BKM>(), bytes);
      } else {
        const Loads o = pick(la, na, u >> 1, &bytes);
        load_unit<AKM>(o, slot(u) + wave_at<AKM>(), bytes);
      }
    }
    f32x4 acc[8][8];
#pragma unroll
    for (int i = 0; i < 8; ++i)
#pragma unroll
      for (int j = 0; j < 8; ++j) acc[i][j] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
    settled(acc);
    // K positions of the last pair that count
    const int32_t left = k - (job.unit + pairs - 1) * UNIT_K;
    const bool cut = left < UNIT_K;
    // units 2 p .. 2 p + 4 of pair p
    uint32_t s0 = slot(0), s1 = slot(1), s2 = slot(2), s3 = slot(3), s4 = slot(4);
    Frag cur, nxt;
    if (ahead == 0) {  // (a later tile's units 0 and 1 landed before the last one's epilogue)
      wait_units<2>();
      barrier_lds();
    }
    {
      const Reader<AKM, BKM, 0> r(ra, rb, s0, s1);
#pragma unroll
      for (int x = 0; x < 16; ++x) r.read(cur, x);
    }
    int32_t at_a, at_b;  // the bytes of the units of pair p + 2
    Loads fa = pick(la, na, 2, &at_a), fb = pick(lb, nb, 2, &at_b);
    int32_t p = 0;
    for (; p + 1 < pairs; ++p) {
      if (p + 2 == pairs) {  // they are the next tile's
        fa = na;
        fb = nb;
        at_a = next.unit * na.step;
        at_b = next.unit * nb.step;
      }
      step<AKM, true, true>(cur, nxt, fa, s4 + wave_at<AKM>(), at_a,
                            Reader<AKM, BKM, 1>(ra, rb, s0, s1), acc);
      at_a += fa.step;
      wait_units<1>();
      barrier_lds();
      step<BKM, true, true>(nxt, cur, fb, s0 + wave_at<BKM>(), at_b,
                            Reader<AKM, BKM, 0>(ra, rb, s2, s3), acc);
      at_b += fb.step;
      const uint32_t t0 = s0, t1 = s1;
      s0 = s2; s1 = s3; s2 = s4; s3 = t0; s4 = t1;
    }
    // The last pair: B's unit of the next tile's second pair waits for the epilogue.
    {
      fa = pick(la, na, p + 2, &at_a);
      if (cut) mask<0>(cur, left);
      step<AKM, true, true>(cur, nxt, fa, s4 + wave_at<AKM>(), at_a,
                            Reader<AKM, BKM, 1>(ra, rb, s0, s1), acc);
      barrier_lds();
      if (cut) mask<1>(nxt, left);
      step<BKM, false, false>(nxt, cur, fb, 0, 0, Reader<AKM, BKM, 0>(ra, rb, s2, s3), acc);
    }
    settled(acc);
    // The next tile's units 0 and 1 have landed, so that its first step need not wait for the stores
    // that follow.
    wait_units<1>();
    // The last pair's slots are free (every wave has read them before the last barrier): 16 KiB of
    // them a wave for the outputs.
    uint8_t* const r0 = lds + (base + 2 * pairs - 2) % SLOTS * SLOT + wave * UNIT_BYTES;
    uint8_t* const r1 = lds + (base + 2 * pairs - 1) % SLOTS * SLOT + wave * UNIT_BYTES;
    Epi out = epi;
    if constexpr (std::is_same<Epi, Partial>::value)
      out.out += static_cast<int64_t>(job.split) * m * epi.pitch;
    const int32_t row = job.row + (wave >> 1) * 128, col = job.col + (wave & 1) * 128;
    if (aligned && row + 128 <= m && col + 128 <= n) {
      // What the next unit needs beside its sums is on its way while this one is made.
      const typename Epi::Tile t = out.tile(row, col);
      typename Epi::Fast now[4], then[4];
#pragma unroll
      for (int it = 0; it < 4; ++it) now[it] = out.fast(t, 8 * it, 0);
#pragma unroll 1
      for (int u = 0; u < 8; ++u) {
        const int r = 32 * (u >> 1), c = 64 * (u & 1);
        if (u < 7) {
#pragma unroll
          for (int it = 0; it < 4; ++it)
            then[it] = out.fast(t, 32 * ((u + 1) >> 1) + 8 * it, 64 * ((u + 1) & 1));
        }
        if ((u & 1) == 0) {
          wave_done_lds();  // the last rows are read
          put_rows(u >> 1, r0, r1, acc);
        }
        float v[4][8];
#pragma unroll
        for (int it = 0; it < 4; ++it) get_row<Epi::HALVES>(u & 1 ? r1 : r0, it, v[it]);
        out.choose([&](auto kind) {
#pragma unroll
          for (int it = 0; it < 4; ++it) out.store_fast(kind, t, r + 8 * it, c, v[it], now[it]);
        });
#pragma unroll
        for (int it = 0; it < 4; ++it) now[it] = then[it];
      }
    } else {
#pragma unroll 1
      for (int i = 0; i < 4; ++i) {
        put_rows(i, r0, r1, acc);
#pragma unroll 1
        for (int u = 0; u < 2; ++u)
          store_unit(out, u ? r1 : r0, row + 32 * i, col + 64 * u, m, n);
        wave_done_lds();
      }
    }
    if (!more) break;
    // Of the next tile's stream units 0 .. 2 are issued (of a tile of one pair 0 and 1: what
    // comes after it was not known).
    ahead = then == 1 ? 2 : 3;
    base = (base + 2 * pairs) % SLOTS;
    job = next;
    la = na;
    lb = nb;
    id += stride;
    barrier_lds();  // every wave is done with the slots that staged the outputs
  }
  // no load lands in LDS that is another workgroup's by then
  asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
}

// The tile kernel's compute units.
int compute_units(int64_t* cus) {
  int device = 0, n = 0;
  hipError_t err = hipGetDevice(&device);
  if (err == hipSuccess)
    err = hipDeviceGetAttribute(&n, hipDeviceAttributeMultiprocessorCount, device);
  if (err != hipSuccess)
    return fail(BUX_E_DEVICE, "the device's compute units: %s", hipGetErrorString(err));
  *cus = n >= 8 ? n / 8 * 8 : 8;
  return BUX_OK;
}

}  // namespace

namespace dense {

bool large_takes(const Mat<uint16_t>& A, bool a_km, const Mat<uint16_t>& B, bool b_km, int64_t m,
                 int64_t n, int64_t k) {
  // direct loads of whole 16-byte chunks, at 32-bit offsets from a tile's rows (K-major) or from
  // the operand (MN-major), a tile and a unit past its end included
  auto takes = [&](const Mat<uint16_t>& x, bool km) {
    const int64_t span = km ? (TILE + 8) * x.ld + k + UNIT_K : (k + 3 * UNIT_K) * x.ld + x.rows + TILE;
    return x.ld % 8 == 0 && reinterpret_cast<uintptr_t>(x.p) % 16 == 0 && 2 * span < (1LL << 31);
  };
  return takes(A, a_km) && takes(B, b_km) && k >= 1 && m < (1LL << 31) - TILE &&
         n < (1LL << 31) - TILE;
}

template <bool AKM, bool BKM, typename Epi>
int launch_large(const Mat<uint16_t>& A, const Mat<uint16_t>& B, int64_t m, int64_t n, int64_t k,
                 int64_t units, int64_t splits, const Epi& epi, hipStream_t s) {
  const int64_t row_tiles = ceil_div(m, TILE), col_tiles = ceil_div(n, TILE);
  const int64_t count = row_tiles * col_tiles * splits;
  if (count >= (1LL << 28)) return fail(BUX_E_ARGUMENT, "dense product: too many tiles");
  int64_t cus = 0;
  if (int rc = compute_units(&cus)) return rc;
  const int64_t want = 8 * ceil_div(count, 8);
  auto kernel = large_kernel<AKM, BKM, Epi>;
  const hipError_t err = hipFuncSetAttribute(reinterpret_cast<const void*>(kernel),
                                             hipFuncAttributeMaxDynamicSharedMemorySize, SLOTS * SLOT);
  if (err != hipSuccess) return fail(BUX_E_LAUNCH, "dense large_kernel: %s", hipGetErrorString(err));
  hipLaunchKernelGGL(kernel, dim3(static_cast<unsigned>(want < cus ? want : cus)), dim3(THREADS),
                     SLOTS * SLOT, s, Operand{A.p, A.ld, A.rows, k}, Operand{B.p, B.ld, B.rows, k},
                     static_cast<int32_t>(m), static_cast<int32_t>(n), static_cast<int32_t>(k),
                     static_cast<int32_t>(units), static_cast<int32_t>(row_tiles),
                     static_cast<int32_t>(col_tiles), static_cast<int32_t>(count), epi);
  return launched("dense large_kernel");
}

#define BUX_LARGE(A, B, ...)                                                                       \
  template int launch_large<A, B, __VA_ARGS__>(const Mat<uint16_t>&, const Mat<uint16_t>&, int64_t, \
                                               int64_t, int64_t, int64_t, int64_t,                 \
                                               const __VA_ARGS__&, hipStream_t)
BUX_LARGE(true, false, Forward<uint16_t, false>);
BUX_LARGE(true, false, Forward<uint16_t, true>);
BUX_LARGE(true, false, Partial);
BUX_LARGE(true, true, Forward<uint16_t, false>);
BUX_LARGE(true, true, Forward<uint16_t, true>);
BUX_LARGE(true, true, Backward<uint16_t, false>);
BUX_LARGE(true, true, Backward<uint16_t, true>);
BUX_LARGE(true, true, Partial);
BUX_LARGE(false, false, Forward<uint16_t, false>);
BUX_LARGE(false, false, Partial);

}  // namespace dense
}  // namespace bux
