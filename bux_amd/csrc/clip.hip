// The global norm of many gradients and their clipping by it.
//
//   norm = (sum over every tensor of g^2)^(1/2);  out = g min(1, max_norm / norm)
//
// The squares are added in float64: float32's would overflow above 1.8e19 and vanish below
// 1e-23, and a sum over 10^9 of them would lose its last digits. The tensors are cut into pieces
// of 32 KiB; a workgroup takes pieces in turn, each lane 16 bytes a load at an element's alignment,
// 8 of them on their way at once, and leaves one sum. The second kernel's workgroups each add all those sums, in order
// (8 KiB at most for every 64 tensors of the list, from L2), so that no atomics decide the order, and
// then scale their pieces, the last ones first: those are what the first kernel left in the Infinity
// Cache. Bound by HBM: 400 tensors of 2 MB take 527 us, 4.8 TB/s of the two reads and the write; small ones
// by their launches, two for every 64 tensors, 400 of 16 KiB 70 us.

#include "common.h"

namespace bux {
namespace {

constexpr int THREADS = 256;
constexpr int64_t PIECE_BYTES = 32768;
template <typename T>
constexpr int64_t PIECE = PIECE_BYTES / sizeof(T);
constexpr int ITEMS = 64;         // tensors a launch
constexpr int64_t GROUPS = 1024;  // workgroups a launch: 4 a CU

struct Item {
  const void* g;
  void* out;
  int64_t n;
  int64_t first;  // its first piece
};
// N: its items, for lists that hold fewer than ITEMS (a launch copies its arguments).
template <int N>
struct Table {
  Item item[N];
  uint64_t f32;  // which are float32
  int32_t count;
  int64_t pieces;
};

// Which item holds piece p: the last whose first is at most p.
template <typename Table>
__device__ __forceinline__ int item_of(const Table& t, int64_t p) {
  int lo = 0, hi = t.count;
  while (hi - lo > 1) {
    const int mid = (lo + hi) >> 1;
    if (t.item[mid].first <= p) lo = mid;
    else hi = mid;
  }
  return lo;
}

// 16 bytes at an element's alignment.
template <typename T>
struct __attribute__((packed, aligned(sizeof(T)))) Chunk {
  static constexpr int N = 16 / sizeof(T);
  T at[N];
};

// f(index, chunk) for this lane's chunks of the elements [lo, hi), a piece at most, then g(index,
// value) for the elements left.
template <typename T, typename F, typename G>
__device__ __forceinline__ void over(const T* p, int64_t lo, int64_t hi, F&& f, G&& g) {
  constexpr int N = Chunk<T>::N, TURN = N * THREADS, TURNS = PIECE<T> / TURN;
  if (hi - lo == PIECE<T>) {
    Chunk<T> e[TURNS];
#pragma unroll
    for (int i = 0; i < TURNS; ++i)
      e[i] = *reinterpret_cast<const Chunk<T>*>(p + lo + N * (i * THREADS + threadIdx.x));
#pragma unroll
    for (int i = 0; i < TURNS; ++i) f(lo + N * (i * THREADS + threadIdx.x), e[i]);
    return;
  }
  for (int64_t at = lo + N * threadIdx.x; at < hi; at += TURN) {
    if (at + N <= hi) {
      f(at, *reinterpret_cast<const Chunk<T>*>(p + at));
    } else {
      for (int64_t i = at; i < hi; ++i) g(i, p[i]);
    }
  }
}

template <typename T>
__device__ __forceinline__ double squares(const void* from, int64_t piece, int64_t n) {
  const T* const p = static_cast<const T*>(from);
  const int64_t lo = piece * PIECE<T>, hi = lo + PIECE<T> < n ? lo + PIECE<T> : n;
  double s = 0.0;
  auto add = [&](T x) {
    const double v = Elem<T>::value(x);
    s = __builtin_fma(v, v, s);
  };
  over(p, lo, hi,
       [&](int64_t, const Chunk<T>& e) {
#pragma unroll
         for (int j = 0; j < Chunk<T>::N; ++j) add(e.at[j]);
       },
       [&](int64_t, T x) { add(x); });
  return s;
}

typedef uint32_t Words __attribute__((ext_vector_type(4), aligned(2)));

// x factor, in float64: float32's factor would lose digits where max_norm / norm is under 2^-126, and
// a float32 gradient would be rounded twice. (bfloat16 goes through float32. 1.2 GB of bfloat16 take
// 645 us, 644 by a float32 factor; 0.8 GB of float32 417 and 425.)
template <typename T>
__device__ __forceinline__ T scaled(T x, double factor) {
  return Elem<T>::make(static_cast<float>(Elem<T>::value(x) * factor));
}

template <typename T>
__device__ __forceinline__ void scale(const void* from, void* to, int64_t piece, int64_t n,
                                      double factor) {
  const T* const p = static_cast<const T*>(from);
  T* const out = static_cast<T*>(to);
  const int64_t lo = piece * PIECE<T>, hi = lo + PIECE<T> < n ? lo + PIECE<T> : n;
  over(p, lo, hi,
       [&](int64_t at, const Chunk<T>& e) {
         // Stored past the caches: nothing here reads it again, and what the squares left is still
         // to be read.
         Chunk<T> r;
#pragma unroll
         for (int j = 0; j < Chunk<T>::N; ++j)
           r.at[j] = scaled<T>(e.at[j], factor);
         __builtin_nontemporal_store(__builtin_bit_cast(Words, r),
                                     reinterpret_cast<Words*>(out + at));
       },
       [&](int64_t at, T x) { out[at] = scaled<T>(x, factor); });
}

// The sum over a workgroup, to all of its lanes, in a fixed order.
__device__ __forceinline__ double group_sum(double v, double* red) {
#pragma unroll
  for (int s = 32; s >= 1; s >>= 1) v += __shfl_xor(v, s);
  if ((threadIdx.x & 63) == 0) red[threadIdx.x >> 6] = v;
  __syncthreads();
  double t = red[0];
#pragma unroll
  for (int w = 1; w < THREADS / 64; ++w) t += red[w];
  return t;
}

template <typename Table>
__global__ __launch_bounds__(THREADS) void squares_kernel(Table t, double* __restrict__ sums) {
  __shared__ double red[THREADS / 64];
  double s = 0.0;
  for (int64_t p = blockIdx.x; p < t.pieces; p += gridDim.x) {
    const int i = item_of(t, p);
    const Item& it = t.item[i];
    if ((t.f32 >> i) & 1) s += squares<float>(it.g, p - it.first, it.n);
    else s += squares<uint16_t>(it.g, p - it.first, it.n);
  }
  s = group_sum(s, red);
  if (threadIdx.x == 0) sums[blockIdx.x] = s;
}

// The square root of the `count` sums' sum.
__device__ __forceinline__ double norm_of(const double* sums, int64_t count, double* red) {
  double s = 0.0;
  for (int64_t i = threadIdx.x; i < count; i += THREADS) s += sums[i];
  return sqrt(group_sum(s, red));
}

__global__ __launch_bounds__(THREADS) void norm_kernel(const double* __restrict__ sums,
                                                       int64_t count, float* __restrict__ norm) {
  __shared__ double red[THREADS / 64];
  const double v = norm_of(sums, count, red);
  if (threadIdx.x == 0) *norm = static_cast<float>(v);
}

template <typename Table>
__global__ __launch_bounds__(THREADS) void scale_kernel(Table t, const double* __restrict__ sums,
                                                        int64_t count, float max_norm,
                                                        float* __restrict__ norm) {
  __shared__ double red[THREADS / 64];
  const double v = norm_of(sums, count, red);
  if (norm && blockIdx.x == 0 && threadIdx.x == 0) *norm = static_cast<float>(v);
  // a NaN norm makes every gradient NaN
  const double factor = v <= max_norm ? 1.0 : max_norm / v;
  for (int64_t q = blockIdx.x; q < t.pieces; q += gridDim.x) {
    const int64_t p = t.pieces - 1 - q;
    const int i = item_of(t, p);
    const Item& it = t.item[i];
    if ((t.f32 >> i) & 1) scale<float>(it.g, it.out, p - it.first, it.n, factor);
    else scale<uint16_t>(it.g, it.out, p - it.first, it.n, factor);
  }
}

// The launch's tensors from `at` on (empty ones left out); where the next launch's begin.
template <int N>
int32_t table_of(const bux_gradient* grads, int32_t count, int32_t at, Table<N>* t) {
  t->count = 0;
  t->pieces = 0;
  t->f32 = 0;
  for (; at < count && t->count < N; ++at) {
    const bux_gradient& g = grads[at];
    if (g.n == 0) continue;
    t->item[t->count] = Item{g.g, g.out, g.n, t->pieces};
    if (g.dtype == BUX_F32) t->f32 |= 1ull << t->count;
    t->pieces += ceil_div(g.n, PIECE_BYTES / (g.dtype == BUX_F32 ? 4 : 2));
    ++t->count;
  }
  return at;
}
template <int N>
unsigned groups_of(const Table<N>& t) {
  return static_cast<unsigned>(t.pieces < GROUPS ? t.pieces : GROUPS);
}

// N: a launch's tensors.
template <int N>
int clip(const bux_gradient* grads, int32_t count, bool clips, float max_norm, float* norm,
         double* sums, hipStream_t s) {
  Table<N> t;
  int64_t made = 0;
  for (int32_t at = 0; at < count;) {
    at = table_of(grads, count, at, &t);
    if (t.count == 0) break;
    hipLaunchKernelGGL(squares_kernel<Table<N>>, dim3(groups_of(t)), dim3(THREADS), 0, s, t,
                       sums + made);
    if (int rc = launched("squares_kernel")) return rc;
    made += groups_of(t);
  }
  if (!clips) {
    hipLaunchKernelGGL(norm_kernel, dim3(1), dim3(THREADS), 0, s, sums, made, norm);
    return launched("norm_kernel");
  }
  float* to = norm;
  for (int32_t at = 0; at < count;) {
    at = table_of(grads, count, at, &t);
    if (t.count == 0) break;
    hipLaunchKernelGGL(scale_kernel<Table<N>>, dim3(groups_of(t)), dim3(THREADS), 0, s, t, sums,
                       made, max_norm, to);
    if (int rc = launched("scale_kernel")) return rc;
    to = nullptr;
  }
  return BUX_OK;
}

}  // namespace
}  // namespace bux

extern "C" size_t bux_clip_workspace_size(int32_t count) {
  using namespace bux;
  return count <= 0 ? 0 : static_cast<size_t>(ceil_div(count, ITEMS)) * GROUPS * sizeof(double);
}

extern "C" int bux_clip(const bux_gradient* grads, int32_t count, float max_norm, float* norm,
                        void* workspace, size_t workspace_bytes, void* stream) {
  using namespace bux;
  const char* const name = "bux_clip";
  clear_error();
  BUX_CHECK(count >= 1 && grads, "%s: %d gradients", name, count);
  BUX_CHECK(norm, "%s: NULL norm", name);
  bool clips = false;
  for (int32_t i = 0; i < count; ++i) {
    const bux_gradient& g = grads[i];
    BUX_CHECK(g.n >= 0 && g.n < (1LL << 40), "%s: gradient %d has %lld elements", name, i,
              (long long)g.n);
    BUX_CHECK(g.dtype == BUX_BF16 || g.dtype == BUX_F32, "%s: gradient %d: dtype %d", name, i,
              g.dtype);
    BUX_CHECK(g.n == 0 || g.g, "%s: gradient %d is NULL", name, i);
    if (g.n > 0 && g.out) clips = true;
  }
  for (int32_t i = 0; i < count; ++i)
    BUX_CHECK(!clips || grads[i].n == 0 || grads[i].out, "%s: gradient %d has no output", name, i);
  BUX_CHECK(!clips || max_norm > 0.0f, "%s: max_norm %g", name, max_norm);
  const size_t need = bux_clip_workspace_size(count);
  if (workspace == nullptr || workspace_bytes < need)
    return fail(BUX_E_WORKSPACE, "%s: workspace of %zu bytes, %zu needed", name, workspace_bytes,
                need);
  BUX_CHECK(reinterpret_cast<uintptr_t>(workspace) % 8 == 0, "%s: unaligned workspace", name);
  double* const sums = static_cast<double*>(workspace);
  hipStream_t s = as_stream(stream);
  // (a list of empty tensors alone has the norm 0 and nothing to scale)
  // A launch copies its table, 2 KiB of 64 tensors, 256 bytes of 8, and one of few workgroups waits for
  // that: 1 tensor of 16 KiB takes 6.6 us in a table of 8, 7.7 in one of 64, 6 take 7.7 and 8.0, 8 as long in
  // either. A list of more takes more launches in 8s: 9 tensors 14.4 us, 7.8 in 64s; 64 tensors 61 and 9.2.
  return count <= 8 ? clip<8>(grads, count, clips, max_norm, norm, sums, s)
                    : clip<ITEMS>(grads, count, clips, max_norm, norm, sums, s);
}
