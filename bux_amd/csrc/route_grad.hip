// The router's backward: from the gradients of the picks' and the sinks' weights, and of what
// losses put on the scores and the logits, to the tokens, the router's kernel and its bias.
//
// With s the scores of the logits z (softmax over all of them, sigmoid or sqrt(softplus)), w
// the picks' scores, T = sum w + sum of the sinks' scores, and a = scaling (rounded to
// bfloat16, as the forward multiplies by it):
//
//   weights = a w / T, sinks = a s / T  (or without T, not normalized), so that
//   ds_i = (a g_i - D / T) / T at a pick or sink i of gradient g_i,  D = sum a g_i s_i;
//   ds  += d_scores;  a pick made twice adds twice
//   dz   = s (ds - sum ds s) | ds s (1 - s) | ds sigmoid(z) / (2 s);  dz += d_logits
//   G    = dz logit_scale  [t, n]
//   dx   = dz_in + G kernel^T,  d_kernel = x^T G,  d_bias = sum over the tokens of G
//
// (moe.py:249-270's transpose: the forward's roundings to bfloat16 pass the gradient as they
// are.) Four kernels: grads_kernel (a wave a token) writes G, in two bfloat16 parts, hi and
// the rest lo: G to 2^-17 at the rate of two bfloat16 MFMAs, where one part alone would put an
// error of a bfloat16 step's half (2^-9) into every product, as large as the outputs' rounding.
// dx_kernel multiplies it by the router's kernel, whose rows lie along n; kernel_grad_kernel
// contracts slices of the tokens, transposing on the way out of LDS; reduce_kernel adds the
// slices, and d_bias's partial sums, in a fixed order.
//
// Bound by HBM at a router's sizes: x read once, dx written once (and dz read); n is small.

#include <math.h>

#include <type_traits>

#include "common.h"

namespace bux {
namespace {

constexpr int THREADS = 256;  // 4 waves
constexpr int MAX_LOGITS = 1024;
constexpr int MAX_PICKS = 16;
constexpr int MAX_GRADS_BLOCKS = 512;

typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));
typedef float v16f __attribute__((ext_vector_type(16)));
typedef short v4s __attribute__((ext_vector_type(4)));
typedef __attribute__((address_space(3))) v4s lds_v4s;

struct Params {
  const uint16_t* x;
  const uint16_t* kernel;  // (d, npad) where n is no multiple of 32: the padded copy
  const int32_t* idx;
  const float* logits;
  const uint16_t* d_weights;
  const uint16_t* d_sinks;
  const float* d_scores;
  const float* d_logits;
  const uint16_t* dz;
  int64_t t, d;
  int32_t n, npad, scored, k, router;
  float logit_scale, factor;
  bool normalize;
  uint16_t* hi;  // G's parts [t, npad]
  uint16_t* lo;
  float* bias_partials;    // [grads blocks, npad], or NULL
  float* kernel_partials;  // [slices, d, npad]
  int32_t grads_blocks, slices;
  int64_t slice;  // tokens a slice, a multiple of 32
  uint16_t* dx;
  uint16_t* d_kernel;
  float* d_bias;
};

__device__ __forceinline__ float wave_sum(float v) {
#pragma unroll
  for (int o = 32; o >= 1; o >>= 1) v += __shfl_xor(v, o);
  return v;
}
__device__ __forceinline__ float wave_max(float v) {
#pragma unroll
  for (int o = 32; o >= 1; o >>= 1) v = fmaxf(v, __shfl_xor(v, o));
  return v;
}

__device__ __forceinline__ float softplus(float v) {
  return fmaxf(v, 0.0f) + log1pf(expf(-fabsf(v)));
}
// A logit's score off the softmax.
__device__ __forceinline__ float score_of(int router, float z) {
  return router == BUX_ROUTER_SIGMOID ? 1.0f / (1.0f + expf(-z)) : sqrtf(softplus(z));
}
// ... and its derivative, in forms that do not cancel for large |z|.
__device__ __forceinline__ float slope_of(int router, float z, float s) {
  const float e = expf(-fabsf(z)), p = 1.0f + e;
  if (router == BUX_ROUTER_SIGMOID) return e / (p * p);
  const float sigmoid = (z >= 0.0f ? 1.0f : e) / p;
  return s == 0.0f ? 0.0f : sigmoid / (2.0f * s);
}

// A wave a token, lane l the logits l, l + 64, ... (Q of them).
template <int Q>
__global__ __launch_bounds__(THREADS) void grads_kernel(Params p) {
  __shared__ float sums[THREADS / 64][Q * 64];
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), lane = threadIdx.x & 63;
  const int n = p.n, scored = p.scored, k = p.k;
  float bias[Q];
#pragma unroll
  for (int q = 0; q < Q; ++q) bias[q] = 0.0f;
  for (int64_t tok = static_cast<int64_t>(blockIdx.x) * 4 + wave; tok < p.t;
       tok += static_cast<int64_t>(gridDim.x) * 4) {
    const float* row = p.logits + tok * n;
    float z[Q], s[Q], ds[Q];
#pragma unroll
    for (int q = 0; q < Q; ++q) {
      const int i = lane + 64 * q;
      z[q] = i < n ? row[i] : -INFINITY;
    }
    // the picks, one a lane: those outside the scored experts count for nothing
    int32_t id = -1;
    float zp = 0.0f, g = 0.0f;
    if (lane < k) {
      id = p.idx[tok * k + lane];
      g = bf16_to_f32(p.d_weights[tok * k + lane]) * p.factor;
    }
    const bool ok = id >= 0 && id < scored;
    if (ok) zp = row[id];
    float w;
    if (p.router == BUX_ROUTER_SOFTMAX) {
      float m = z[0];
#pragma unroll
      for (int q = 1; q < Q; ++q) m = fmaxf(m, z[q]);
      m = wave_max(m);
      float sum = 0.0f;
#pragma unroll
      for (int q = 0; q < Q; ++q) {
        s[q] = expf(z[q] - m);
        sum += s[q];
      }
      const float all = wave_sum(sum);
#pragma unroll
      for (int q = 0; q < Q; ++q) s[q] /= all;
      w = expf(zp - m) / all;
    } else {
#pragma unroll
      for (int q = 0; q < Q; ++q) s[q] = lane + 64 * q < n ? score_of(p.router, z[q]) : 0.0f;
      w = score_of(p.router, zp);
    }
    if (!ok) w = g = 0.0f;
    float sink[Q];  // the sinks' gradients
#pragma unroll
    for (int q = 0; q < Q; ++q) {
      const int i = lane + 64 * q;
      sink[q] = p.d_sinks && i >= scored && i < n
                    ? bf16_to_f32(p.d_sinks[tok * (n - scored) + i - scored]) * p.factor : 0.0f;
    }
    float inv = 1.0f, shift = 0.0f;  // ds = (g - shift) inv
    if (p.normalize) {
      float total = w, dot = g * w;
#pragma unroll
      for (int q = 0; q < Q; ++q) {
        const int i = lane + 64 * q;
        if (i >= scored && i < n) {
          total += s[q];
          dot += sink[q] * s[q];
        }
      }
      total = wave_sum(total);
      dot = wave_sum(dot);
      inv = total == 0.0f ? 0.0f : 1.0f / total;
      shift = total == 0.0f ? 0.0f : dot / total;
    }
    const float dp = ok ? (g - shift) * inv : 0.0f;
#pragma unroll
    for (int q = 0; q < Q; ++q) {
      const int i = lane + 64 * q;
      ds[q] = i >= scored && i < n ? (sink[q] - shift) * inv : 0.0f;
      if (p.d_scores && i < scored) ds[q] += p.d_scores[tok * scored + i];
    }
    for (int j = 0; j < k; ++j) {
      const int32_t at = __builtin_amdgcn_readlane(id, j);
      const float v = __uint_as_float(__builtin_amdgcn_readlane(__float_as_uint(dp), j));
#pragma unroll
      for (int q = 0; q < Q; ++q)
        if (lane + 64 * q == at) ds[q] += v;
    }
    float inner = 0.0f;
    if (p.router == BUX_ROUTER_SOFTMAX) {
#pragma unroll
      for (int q = 0; q < Q; ++q) inner += ds[q] * s[q];
      inner = wave_sum(inner);
    }
#pragma unroll
    for (int q = 0; q < Q; ++q) {
      const int i = lane + 64 * q;
      float dl = 0.0f;
      if (i < n) {
        dl = p.router == BUX_ROUTER_SOFTMAX ? s[q] * (ds[q] - inner)
                                            : ds[q] * slope_of(p.router, z[q], s[q]);
        if (p.d_logits) dl += p.d_logits[tok * n + i];
        dl *= p.logit_scale;
      }
      bias[q] += dl;
      if (i < p.npad) {
        const uint16_t h = f32_to_bf16(dl);
        p.hi[tok * p.npad + i] = h;
        p.lo[tok * p.npad + i] = f32_to_bf16(dl - bf16_to_f32(h));
      }
    }
  }
  if (p.bias_partials == nullptr) return;
#pragma unroll
  for (int q = 0; q < Q; ++q) sums[wave][lane + 64 * q] = bias[q];
  __syncthreads();
  for (int i = threadIdx.x; i < p.npad; i += THREADS)
    p.bias_partials[static_cast<int64_t>(blockIdx.x) * p.npad + i] =
        (sums[0][i] + sums[1][i]) + (sums[2][i] + sums[3][i]);
}

// The router's kernel (d, n) with its rows padded by zeros to npad.
__global__ __launch_bounds__(THREADS) void pad_kernel(const uint16_t* __restrict__ kernel,
                                                      int64_t d, int32_t n, int32_t npad,
                                                      uint16_t* __restrict__ out) {
  const int64_t i = static_cast<int64_t>(blockIdx.x) * THREADS + threadIdx.x;
  if (i >= d * npad) return;
  const int64_t r = i / npad;
  const int32_t c = static_cast<int32_t>(i - r * npad);
  out[i] = c < n ? kernel[r * n + c] : 0;
}

__device__ __forceinline__ bf16x8 load8(const uint16_t* p) {
  return __builtin_bit_cast(bf16x8, *reinterpret_cast<const uint4*>(p));
}

// dx: a wave 32 RB tokens by 128 columns, K = npad in 16s, the operands from L2 straight to
// registers. MFMA with the kernel's rows first: lane l holds token l % 32, runs of 4 columns
// 8 g + 4 (l / 32) of each block. The results pass LDS (32 tokens at a time) so that 16 lanes
// store 256 bytes of a row, with dz added in float32 before the one rounding.
constexpr int COLS = 128;
constexpr int DX_PITCH = COLS + 4;  // floats: rows 16 bytes past a multiple of the banks
template <int RB>
__global__ __launch_bounds__(THREADS) void dx_kernel(Params p, uint32_t columns) {
  __shared__ __align__(16) float out[THREADS / 64][32 * DX_PITCH];
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), lane = threadIdx.x & 63;
  const int r = lane & 31, h = lane >> 5;
  const int64_t t0 = static_cast<int64_t>(blockIdx.x / columns) * (32 * RB);
  const int64_t c0 = (static_cast<int64_t>(blockIdx.x % columns) * 4 + wave) * COLS;
  if (c0 >= p.d) return;  // no barrier follows
  const uint16_t* ah[RB];
  const uint16_t* al[RB];
  const uint16_t* b[4];
#pragma unroll
  for (int i = 0; i < RB; ++i) {  // tokens and columns past the last: the last one's, not stored
    const int64_t tok = t0 + 32 * i + r < p.t ? t0 + 32 * i + r : p.t - 1;
    ah[i] = p.hi + tok * p.npad + 8 * h;
    al[i] = p.lo + tok * p.npad + 8 * h;
  }
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    const int64_t col = c0 + 32 * j + r < p.d ? c0 + 32 * j + r : p.d - 1;
    b[j] = p.kernel + col * p.npad + 8 * h;
  }
  v16f acc[RB][4];
#pragma unroll
  for (int i = 0; i < RB; ++i)
#pragma unroll
    for (int j = 0; j < 4; ++j) acc[i][j] = v16f{};
#pragma unroll 2
  for (int32_t e = 0; e < p.npad; e += 16) {
    bf16x8 hi[RB], lo[RB], w[4];
#pragma unroll
    for (int i = 0; i < RB; ++i) {
      hi[i] = load8(ah[i] + e);
      lo[i] = load8(al[i] + e);
    }
#pragma unroll
    for (int j = 0; j < 4; ++j) w[j] = load8(b[j] + e);
#pragma unroll
    for (int j = 0; j < 4; ++j)
#pragma unroll
      for (int i = 0; i < RB; ++i) {
        acc[i][j] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(w[j], hi[i], acc[i][j], 0, 0, 0);
        acc[i][j] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(w[j], lo[i], acc[i][j], 0, 0, 0);
      }
  }
  float* mine = out[wave];
#pragma unroll
  for (int i = 0; i < RB; ++i) {
#pragma unroll
    for (int j = 0; j < 4; ++j)
#pragma unroll
      for (int g = 0; g < 4; ++g)
        *reinterpret_cast<float4*>(mine + r * DX_PITCH + 32 * j + 8 * g + 4 * h) =
            make_float4(acc[i][j][4 * g], acc[i][j][4 * g + 1], acc[i][j][4 * g + 2],
                        acc[i][j][4 * g + 3]);
    // the wave's own region: its LDS operations run in order
    asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
    __builtin_amdgcn_wave_barrier();
    const int64_t col = c0 + 8 * (lane & 15);
#pragma unroll
    for (int it = 0; it < 8; ++it) {
      const int row = it * 4 + (lane >> 4);
      const int64_t tok = t0 + 32 * i + row;
      float v[8];
      Elem<float>::load8(mine + row * DX_PITCH + 8 * (lane & 15), v);
      if (tok >= p.t || col >= p.d) continue;
      if (p.dz) {
        float add[8];
        Elem<uint16_t>::load8(p.dz + tok * p.d + col, add);
#pragma unroll
        for (int e = 0; e < 8; ++e) v[e] += add[e];
      }
      Elem<uint16_t>::store8(p.dx + tok * p.d + col, v);
    }
    asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
    __builtin_amdgcn_wave_barrier();
  }
}

// d_kernel's partial sums: a workgroup 128 of d by 128 logits over a slice of the tokens, 32 a
// step, in two LDS stages filled through registers. x and G lie token-major, the contracted
// axis slow: a stage holds 32 tokens' 256 bytes, 16-byte chunk c of token k at place
// c ^ 4 (k % 4), and ds_read_b64_tr_b16 transposes on the way out (within each 16 lanes, lane
// j's 16-bit element e is element j % 4 of the 8 bytes that lane 4 e + j / 4 read).
constexpr int STEP = 32;
struct KStage {
  uint16_t x[STEP * COLS], hi[STEP * COLS], lo[STEP * COLS];
};

__device__ __forceinline__ bf16x8 read_tr(uint32_t at) {
  const v4s a = __builtin_amdgcn_ds_read_tr16_b64_v4i16(reinterpret_cast<lds_v4s*>(at));
  const v4s b = __builtin_amdgcn_ds_read_tr16_b64_v4i16(reinterpret_cast<lds_v4s*>(at + 4 * 256));
  return __builtin_bit_cast(bf16x8, __builtin_shufflevector(a, b, 0, 1, 2, 3, 4, 5, 6, 7));
}

__global__ __launch_bounds__(THREADS) void kernel_grad_kernel(Params p) {
  __shared__ __align__(16) KStage st[2];
  const int wave = threadIdx.x >> 6, lane = threadIdx.x & 63;
  const int64_t j0 = static_cast<int64_t>(blockIdx.x) * COLS;
  const int32_t e0 = blockIdx.y * COLS;
  const int64_t lo_t = blockIdx.z * p.slice;
  const int64_t hi_t = lo_t + p.slice < p.t ? lo_t + p.slice : p.t;
  const int steps = static_cast<int>((hi_t - lo_t + STEP - 1) / STEP);
  // this thread's two chunks of each operand's stage: tokens row and row + 16
  const int row = threadIdx.x >> 4, chunk = threadIdx.x & 15;
  const bool x_in = j0 + 8 * chunk < p.d, g_in = e0 + 8 * chunk < p.npad;
  uint4 xs[2], hs[2], ls[2];
  auto load = [&](int s) {
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      const int64_t tok = lo_t + static_cast<int64_t>(s) * STEP + row + 16 * i;
      const uint4 zero = make_uint4(0, 0, 0, 0);
      xs[i] = hs[i] = ls[i] = zero;
      if (tok < hi_t) {
        if (x_in) xs[i] = *reinterpret_cast<const uint4*>(p.x + tok * p.d + j0 + 8 * chunk);
        if (g_in) {
          hs[i] = *reinterpret_cast<const uint4*>(p.hi + tok * p.npad + e0 + 8 * chunk);
          ls[i] = *reinterpret_cast<const uint4*>(p.lo + tok * p.npad + e0 + 8 * chunk);
        }
      }
    }
  };
  auto put = [&](int b) {
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      const int k = row + 16 * i, at = k * COLS + 8 * (chunk ^ (4 * (k & 3)));
      *reinterpret_cast<uint4*>(st[b].x + at) = xs[i];
      *reinterpret_cast<uint4*>(st[b].hi + at) = hs[i];
      *reinterpret_cast<uint4*>(st[b].lo + at) = ls[i];
    }
  };
  // wave (a, b) of 2 x 2: 64 of d from 64 a, 64 logits from 64 b; block q of 32 columns
  const int s16 = lane & 15, kq = s16 >> 2;
  const int col = 16 * ((lane >> 4) & 1) + 4 * (s16 & 3);
  auto offset = [&](int block) {
    return (8 * (lane >> 5) + kq) * 256 + 16 * (4 * (block ^ kq) + (col >> 3)) +
           8 * ((col >> 2) & 1);
  };
  uint32_t xat[2], gat[2];
#pragma unroll
  for (int q = 0; q < 2; ++q) {
    xat[q] = offset(2 * (wave >> 1) + q);
    gat[q] = offset(2 * (wave & 1) + q);
  }
  const uint32_t lds0 = static_cast<uint32_t>(reinterpret_cast<uintptr_t>(&st[0]));
  v16f acc[2][2];
#pragma unroll
  for (int i = 0; i < 2; ++i)
#pragma unroll
    for (int j = 0; j < 2; ++j) acc[i][j] = v16f{};
  if (steps > 0) {
    load(0);
    put(0);
  }
  for (int s = 0; s < steps; ++s) {
    __syncthreads();
    if (s + 1 < steps) load(s + 1);
    const uint32_t at = lds0 + (s & 1) * sizeof(KStage);
#pragma unroll
    for (int half = 0; half < 2; ++half) {
      const uint32_t k16 = half * 16 * 256;
      bf16x8 xv[2], hv[2], lv[2];
#pragma unroll
      for (int q = 0; q < 2; ++q) {
        xv[q] = read_tr(at + offsetof(KStage, x) + k16 + xat[q]);
        hv[q] = read_tr(at + offsetof(KStage, hi) + k16 + gat[q]);
        lv[q] = read_tr(at + offsetof(KStage, lo) + k16 + gat[q]);
      }
#pragma unroll
      for (int i = 0; i < 2; ++i)
#pragma unroll
        for (int j = 0; j < 2; ++j) {
          acc[i][j] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(hv[j], xv[i], acc[i][j], 0, 0, 0);
          acc[i][j] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(lv[j], xv[i], acc[i][j], 0, 0, 0);
        }
    }
    if (s + 1 < steps) put((s + 1) & 1);
  }
  float* base = p.kernel_partials + static_cast<int64_t>(blockIdx.z) * p.d * p.npad;
#pragma unroll
  for (int i = 0; i < 2; ++i) {
    const int64_t j = j0 + 64 * (wave >> 1) + 32 * i + (lane & 31);
    if (j >= p.d) continue;
#pragma unroll
    for (int q = 0; q < 2; ++q)
#pragma unroll
      for (int g = 0; g < 4; ++g) {
        const int32_t e = e0 + 64 * (wave & 1) + 32 * q + 8 * g + 4 * (lane >> 5);
        if (e < p.npad)
          *reinterpret_cast<float4*>(base + j * p.npad + e) =
              make_float4(acc[i][q][4 * g], acc[i][q][4 * g + 1], acc[i][q][4 * g + 2],
                          acc[i][q][4 * g + 3]);
      }
  }
}

// d_kernel: the slices' sums in order, 4 logits a thread; d_bias: a block each 64 logits after
// those, its waves every 4th partial, then the waves' in order.
__global__ __launch_bounds__(THREADS) void reduce_kernel(Params p, int64_t kernel_blocks) {
  __shared__ float part[THREADS / 64][64];
  const int64_t size = p.d * p.npad;
  if (static_cast<int64_t>(blockIdx.x) < kernel_blocks) {
    const int64_t i = (static_cast<int64_t>(blockIdx.x) * THREADS + threadIdx.x) * 4;
    if (i >= size) return;
    float4 v = make_float4(0, 0, 0, 0);
#pragma unroll 4
    for (int32_t s = 0; s < p.slices; ++s) {
      const float4 a = *reinterpret_cast<const float4*>(p.kernel_partials + s * size + i);
      v.x += a.x;
      v.y += a.y;
      v.z += a.z;
      v.w += a.w;
    }
    const int64_t j = i / p.npad;
    const int32_t e = static_cast<int32_t>(i - j * p.npad);
    uint16_t* out = p.d_kernel + j * p.n + e;
    const float f[4] = {v.x, v.y, v.z, v.w};
    if (p.n % 4 == 0 && e < p.n) {
      *reinterpret_cast<uint2*>(out) = make_uint2(
          f32_to_bf16(f[0]) | (static_cast<uint32_t>(f32_to_bf16(f[1])) << 16),
          f32_to_bf16(f[2]) | (static_cast<uint32_t>(f32_to_bf16(f[3])) << 16));
    } else {
#pragma unroll
      for (int q = 0; q < 4; ++q)
        if (e + q < p.n) out[q] = f32_to_bf16(f[q]);
    }
    return;
  }
  const int wave = threadIdx.x >> 6, lane = threadIdx.x & 63;
  const int32_t e = static_cast<int32_t>(blockIdx.x - kernel_blocks) * 64 + lane;
  float s = 0.0f;
  if (e < p.n) {
#pragma unroll 4
    for (int32_t b = wave; b < p.grads_blocks; b += 4)
      s += p.bias_partials[static_cast<int64_t>(b) * p.npad + e];
  }
  part[wave][lane] = s;
  __syncthreads();
  if (wave == 0 && e < p.n)
    p.d_bias[e] = (part[0][lane] + part[1][lane]) + (part[2][lane] + part[3][lane]);
}

int32_t padded(int32_t n) { return static_cast<int32_t>(ceil_div(n, 32) * 32); }

// What a call of t tokens, d columns and n logits keeps in its workspace.
struct Plan {
  int32_t npad, grads_blocks, slices;
  int64_t slice;
  size_t parts, kernel, bias, partials, bytes;  // offsets, and the whole
};
Plan plan_of(int64_t t, int64_t d, int32_t n) {
  Plan w{};
  w.npad = padded(n);
  w.grads_blocks = static_cast<int32_t>(
      ceil_div(t, 4) < MAX_GRADS_BLOCKS ? ceil_div(t, 4) : MAX_GRADS_BLOCKS);
  // as many workgroups as two a CU, slices of 256 tokens at least
  const int64_t tiles = ceil_div(d, COLS) * ceil_div(w.npad, COLS);
  const int64_t most = 512 / tiles > 1 ? 512 / tiles : 1;
  const int64_t by_tokens = ceil_div(t > 0 ? t : 1, 256);
  const int64_t slices = most < by_tokens ? most : by_tokens;
  w.slice = ceil_div(ceil_div(t > 0 ? t : 1, slices), STEP) * STEP;
  w.slices = static_cast<int32_t>(ceil_div(t, w.slice));
  auto whole = [](size_t v) { return (v + 255) & ~static_cast<size_t>(255); };
  const size_t part = whole(static_cast<size_t>(t) * w.npad * sizeof(uint16_t));
  w.parts = 0;
  w.kernel = 2 * part;
  w.bias = w.kernel + (n % 32 == 0 ? 0 : whole(static_cast<size_t>(d) * w.npad * sizeof(uint16_t)));
  w.partials = w.bias + whole(static_cast<size_t>(w.grads_blocks) * w.npad * sizeof(float));
  w.bytes = w.partials + static_cast<size_t>(w.slices) * d * w.npad * sizeof(float);
  return w;
}

}  // namespace
}  // namespace bux

extern "C" size_t bux_route_backward_workspace_size(int64_t t, int64_t d, int32_t n_logits) {
  using namespace bux;
  if (t < 0 || d <= 0 || n_logits <= 0) return 0;
  return plan_of(t, d, n_logits).bytes;
}

extern "C" int bux_route_backward(const uint16_t* x, const uint16_t* kernel, int64_t t, int64_t d,
                                  int32_t n_logits, float logit_scale, int router, int32_t scored,
                                  const int32_t* idx, int32_t k, int normalize, float scaling,
                                  const float* logits, const uint16_t* d_weights,
                                  const uint16_t* d_sinks, const float* d_scores,
                                  const float* d_logits, const uint16_t* dz, uint16_t* dx,
                                  uint16_t* d_kernel, float* d_bias, void* workspace,
                                  size_t workspace_bytes, void* stream) {
  using namespace bux;
  clear_error();
  BUX_CHECK(t >= 0 && t < (1LL << 31) && d > 0 && d % 16 == 0 && d < (1LL << 31),
            "bux_route_backward: t=%lld d=%lld (d a positive multiple of 16)", (long long)t,
            (long long)d);
  BUX_CHECK(n_logits >= 1 && n_logits <= MAX_LOGITS,
            "bux_route_backward: n_logits=%d outside [1, %d]", n_logits, MAX_LOGITS);
  BUX_CHECK(scored >= 1 && scored <= n_logits, "bux_route_backward: scored=%d outside [1, %d]",
            scored, n_logits);
  BUX_CHECK(router == BUX_ROUTER_SOFTMAX || router == BUX_ROUTER_SIGMOID ||
                router == BUX_ROUTER_SQRTSOFTPLUS,
            "bux_route_backward: router=%d", router);
  BUX_CHECK(k >= 1 && k <= MAX_PICKS && k <= scored,
            "bux_route_backward: k=%d outside [1, min(%d, %d)]", k, MAX_PICKS, scored);
  BUX_CHECK(d_sinks == nullptr || n_logits > scored, "bux_route_backward: d_sinks without sinks");
  BUX_CHECK(kernel && d_kernel, "bux_route_backward: NULL kernel or d_kernel");
  BUX_CHECK(t == 0 || (x && idx && logits && d_weights && dx), "bux_route_backward: NULL buffer");
  const Plan w = plan_of(t, d, n_logits);
  // a launch holds fewer than 2^32 threads
  BUX_CHECK(ceil_div(t, 32) * ceil_div(d, 4 * COLS) < (1LL << 24) && d * w.npad < (1LL << 32),
            "bux_route_backward: t=%lld d=%lld n_logits=%d are more than a launch holds",
            (long long)t, (long long)d, n_logits);
  if (w.bytes > 0 && (workspace == nullptr || workspace_bytes < w.bytes))
    return fail(BUX_E_WORKSPACE, "bux_route_backward: workspace of %zu bytes, %zu needed",
                workspace_bytes, w.bytes);
  hipStream_t s = as_stream(stream);
  uint8_t* ws = static_cast<uint8_t*>(workspace);
  Params p{};
  p.x = x;
  p.kernel = kernel;
  p.idx = idx;
  p.logits = logits;
  p.d_weights = d_weights;
  p.d_sinks = d_sinks;
  p.d_scores = d_scores;
  p.d_logits = d_logits;
  p.dz = dz;
  p.t = t;
  p.d = d;
  p.n = n_logits;
  p.npad = w.npad;
  p.scored = scored;
  p.k = k;
  p.router = router;
  p.logit_scale = logit_scale;
  uint32_t bits;
  __builtin_memcpy(&bits, &scaling, sizeof(bits));
  if ((bits & 0x7fffffffu) <= 0x7f800000u) bits += 0x7fffu + ((bits >> 16) & 1u);
  bits &= 0xffff0000u;  // the scaling rounded to bfloat16, as the forward multiplies by it
  __builtin_memcpy(&p.factor, &bits, sizeof(bits));
  p.normalize = normalize != 0;
  p.hi = reinterpret_cast<uint16_t*>(ws + w.parts);
  p.lo = reinterpret_cast<uint16_t*>(ws + w.parts + w.kernel / 2);
  p.bias_partials = d_bias ? reinterpret_cast<float*>(ws + w.bias) : nullptr;
  p.kernel_partials = reinterpret_cast<float*>(ws + w.partials);
  p.grads_blocks = t > 0 ? w.grads_blocks : 0;
  p.slices = t > 0 ? w.slices : 0;
  p.slice = w.slice;
  p.dx = dx;
  p.d_kernel = d_kernel;
  p.d_bias = d_bias;
  if (t > 0) {
    auto grads = [&](auto q) {
      hipLaunchKernelGGL((grads_kernel<decltype(q)::value>), dim3(w.grads_blocks), dim3(THREADS), 0,
                         s, p);
    };
    if (p.npad <= 64) grads(std::integral_constant<int, 1>{});
    else if (p.npad <= 128) grads(std::integral_constant<int, 2>{});
    else if (p.npad <= 256) grads(std::integral_constant<int, 4>{});
    else if (p.npad <= 512) grads(std::integral_constant<int, 8>{});
    else grads(std::integral_constant<int, 16>{});
    if (int rc = launched("route grads_kernel")) return rc;
    if (n_logits % 32 != 0) {
      uint16_t* pad = reinterpret_cast<uint16_t*>(ws + w.kernel);
      hipLaunchKernelGGL(pad_kernel, dim3(static_cast<unsigned>(ceil_div(d * w.npad, THREADS))),
                         dim3(THREADS), 0, s, kernel, d, n_logits, w.npad, pad);
      if (int rc = launched("route pad_kernel")) return rc;
      p.kernel = pad;
    }
    const uint32_t columns = static_cast<uint32_t>(ceil_div(d, 4 * COLS));
    auto input = [&](auto rb) {
      constexpr int RB = decltype(rb)::value;
      hipLaunchKernelGGL((dx_kernel<RB>),
                         dim3(static_cast<unsigned>(columns * ceil_div(t, 32 * RB))), dim3(THREADS),
                         0, s, p, columns);
    };
    if (ceil_div(t, 64) * columns >= 256) input(std::integral_constant<int, 2>{});
    else input(std::integral_constant<int, 1>{});
    if (int rc = launched("route dx_kernel")) return rc;
    hipLaunchKernelGGL(kernel_grad_kernel,
                       dim3(static_cast<unsigned>(ceil_div(d, COLS)),
                            static_cast<unsigned>(ceil_div(w.npad, COLS)),
                            static_cast<unsigned>(w.slices)),
                       dim3(THREADS), 0, s, p);
    if (int rc = launched("route kernel_grad_kernel")) return rc;
  }
  const int64_t kernel_blocks = ceil_div(d * w.npad, 4 * THREADS);
  const int64_t bias_blocks = d_bias ? ceil_div(n_logits, 64) : 0;
  hipLaunchKernelGGL(reduce_kernel, dim3(static_cast<unsigned>(kernel_blocks + bias_blocks)),
                     dim3(THREADS), 0, s, p, kernel_blocks);
  return launched("route reduce_kernel");
}
