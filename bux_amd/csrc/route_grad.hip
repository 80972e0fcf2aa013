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
// are.) Three kernels: grads_kernel writes G, in three bfloat16 parts of 8 bits of its mantissa
// each, whose sum is G: its products are float32's, at the rate of three bfloat16 MFMAs (two
// parts would hold it to 2^-17 alone, which sums that cancel bring to the top). products_kernel
// multiplies it by the router's kernel, whose rows lie along n (dx_tile), and contracts slices of
// the tokens with it, transposing on the way out of LDS (kernel_grad_tile), and adds d_bias's partial
// sums. reduce_kernel adds the slices, where there are several. All in a fixed order.
//
// What bounds it: HBM for few logits (x read once, dx written once, dz read; G stays in L2), the
// MFMAs of G's three parts for many. us of the three: 500 tokens of 2048, 128 logits 6.1, 11.5, 4.0
// (a launch's latency each); 16384 with dz 9.4, 62, 5.0, where its 212 MB take 34 at 6.2 TB/s; 8192
// of 7168, 256 logits 16, 173 to 210 (the card's clock), 5.5, whose 180 GFLOP take 147 at a large
// matrix product's 1.22 PFLOP/s. With two parts the products took 9.7, 50.6 and 125 to 150.

#include <math.h>

#include <type_traits>

#include "common.h"

namespace bux {
namespace {

constexpr int THREADS = 256;  // 4 waves
constexpr int MAX_LOGITS = 1024;
constexpr int MAX_PICKS = 16;
constexpr int MAX_GRADS_BLOCKS = 1024;
constexpr int PARTS = 3;

typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));
typedef float v16f __attribute__((ext_vector_type(16)));
typedef short v4s __attribute__((ext_vector_type(4)));
typedef __attribute__((address_space(3))) v4s lds_v4s;

struct Params {
  const uint16_t* x;
  const uint16_t* kernel;  // (d, n)
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
  uint16_t* parts[PARTS];  // G's, in blocks (at_block), the first 8 bits' first
  uint16_t* blocks;  // the kernel, in blocks
  float* bias_partials;    // [grads blocks, npad], or NULL
  float* kernel_partials;  // [slices, d, npad]
  int32_t grads_blocks, slices;
  int64_t slice;  // tokens a slice, whole steps
  uint16_t* dx;
  uint16_t* d_kernel;
  float* d_bias;
};

// G and the router's kernel lie in blocks of 32 rows by 8 columns, a block's 32 x 16 bytes in one
// run and a row of blocks' one after another, padded with zeros to npad columns: a wave's load of
// an MFMA operand (lane l row l % 32, columns 8 (l / 32) .. + 7 of 16) is one run of 1 KiB. (From
// rows, 32 runs of 32 bytes: dx alone 68 us for 16384 tokens of 2048, 128 logits, so 43.) The element
// (r, c), c a multiple of 4:
__device__ __forceinline__ int64_t at_block(int64_t r, int32_t c, int32_t npad) {
  return ((r >> 5) * (npad >> 3) + (c >> 3)) * 256 + (r & 31) * 8 + (c & 7);
}

// Over the L lanes of a token.
template <int L>
__device__ __forceinline__ float lanes_sum(float v) {
#pragma unroll
  for (int o = 1; o < L; o <<= 1) v += __shfl_xor(v, o);
  return v;
}
template <int L>
__device__ __forceinline__ float lanes_max(float v) {
#pragma unroll
  for (int o = 1; o < L; o <<= 1) v = fmaxf(v, __shfl_xor(v, o));
  return v;
}

// A logit's score off the softmax and its derivative, in forms that do not cancel for large |z|:
// with e = exp(-|z|) and p = 1 / (1 + e), sigmoid(z) is p or e p, its derivative e p^2.
__device__ __forceinline__ void score_of(int router, float z, float* s, float* slope) {
  const float e = expf(-fabsf(z)), p = __builtin_amdgcn_rcpf(1.0f + e);
  const float sigmoid = z >= 0.0f ? p : e * p;
  if (router == BUX_ROUTER_SIGMOID) {
    *s = sigmoid;
    *slope = e * p * p;
  } else {
    *s = sqrtf(fmaxf(z, 0.0f) + log1pf(e));
    *slope = *s == 0.0f ? 0.0f : sigmoid / (2.0f * *s);
  }
}

// Columns i .. i + 3 of a row of n, `fill` past it.
__device__ __forceinline__ void load4(const float* row, int i, int n, float fill, float* v) {
  struct __attribute__((packed, aligned(4))) Four {
    float at[4];
  };
  if (i + 4 <= n) {
    const Four f = *reinterpret_cast<const Four*>(row + i);
#pragma unroll
    for (int j = 0; j < 4; ++j) v[j] = f.at[j];
  } else {
#pragma unroll
    for (int j = 0; j < 4; ++j) v[j] = i + j < n ? row[i + j] : fill;
  }
}

// The upper 8 bits of two mantissas as bfloat16 (cut off, so that no part overflows), the rest
// left in the values, exactly: after three parts 0.
__device__ __forceinline__ uint32_t next_part(float& a, float& b) {
  const uint32_t x = __float_as_uint(a), y = __float_as_uint(b) & 0xffff0000u;
  a -= __uint_as_float(x & 0xffff0000u);
  b -= __uint_as_float(y);
  return (x >> 16) | y;
}

// L lanes a token, lane l the logits 4 l + 4 L c .. + 3 for c < Q / 4, so that a wave's tokens
// share its chain of sums (a wave a token: 24.6 us for 16384 tokens of 128 logits). Bound by
// VALU work then: each logit's count among the picks, and the sum of their gradients, pass
// LDS, where the first of equal picks puts them (compared with every logit instead, 11 us).
template <int L, int Q>
__global__ __launch_bounds__(THREADS) void grads_kernel(Params p) {
  if (static_cast<int32_t>(blockIdx.x) >= p.grads_blocks) {  // the kernel into blocks, 4 columns a thread
    const int64_t i = (static_cast<int64_t>(blockIdx.x - p.grads_blocks) * THREADS + threadIdx.x) * 4;
    const int64_t r = i / p.npad;
    if (r >= p.d) return;
    const int32_t c = static_cast<int32_t>(i - r * p.npad);
    uint32_t v[4];
#pragma unroll
    for (int j = 0; j < 4; ++j) v[j] = c + j < p.n ? p.kernel[r * p.n + c + j] : 0;
    *reinterpret_cast<uint2*>(p.blocks + at_block(r, c, p.npad)) =
        make_uint2(v[0] | (v[1] << 16), v[2] | (v[3] << 16));
    return;
  }
  static_assert(L >= MAX_PICKS && Q % 4 == 0, "a lane a pick, whole fours of logits");
  constexpr int TOKENS = THREADS / L;
  __shared__ __align__(16) float counts[TOKENS][L * Q], grads[TOKENS][L * Q];
  const int lane = threadIdx.x % L, sub = threadIdx.x / L;
  const int first = (threadIdx.x & 63) - lane;  // the token's first lane of its wave
  const int n = p.n, scored = p.scored, k = p.k;
  auto column = [&](int q) { return (q / 4) * 4 * L + 4 * lane + q % 4; };
  float bias[Q];
#pragma unroll
  for (int q = 0; q < Q; ++q) bias[q] = 0.0f;
  // to whole blocks of 32 tokens: those past the last are zeros (their x counts as 0, but a NaN
  // beside it would not)
  const int64_t whole = (p.t + 31) / 32 * 32;
  for (int64_t base = static_cast<int64_t>(blockIdx.x) * TOKENS; base < whole;
       base += static_cast<int64_t>(p.grads_blocks) * TOKENS) {
    const bool live = base + sub < p.t;
    const int64_t tok = live ? base + sub : p.t - 1;
    const float* row = p.logits + tok * n;
    float z[Q], s[Q], ds[Q];
#pragma unroll
    for (int q = 0; q < Q; q += 4) load4(row, column(q), n, -INFINITY, z + q);
    // the picks, one a lane: those outside the scored experts count for nothing
    int32_t id = -1;
    float g = 0.0f;
    if (lane < k) {
      id = p.idx[tok * k + lane];
      g = bf16_to_f32(p.d_weights[tok * k + lane]) * p.factor;
      if (id >= scored || id < 0) id = -1 - lane;  // no other pick's
    }
    // the picks' counts and gradients by logit: of equal picks the first's lane puts all
    float count[Q], grad[Q];
#pragma unroll
    for (int q = 0; q < Q; q += 4) {
      *reinterpret_cast<float4*>(&counts[sub][column(q)]) = make_float4(0, 0, 0, 0);
      *reinterpret_cast<float4*>(&grads[sub][column(q)]) = make_float4(0, 0, 0, 0);
    }
    float times = 0.0f, sum_g = 0.0f;
    int before = k;
    for (int j = 0; j < k; ++j) {
      const int32_t other = __shfl(id, first + j);
      const float v = __shfl(g, first + j);
      if (other == id) {
        times += 1.0f;
        sum_g += v;
        before = j < before ? j : before;
      }
    }
    asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");  // a wave's own region
    __builtin_amdgcn_wave_barrier();
    if (lane < k && before == lane && id >= 0) {
      counts[sub][id] = times;
      grads[sub][id] = sum_g;
    }
    asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
    __builtin_amdgcn_wave_barrier();
#pragma unroll
    for (int q = 0; q < Q; q += 4) {
      const float4 c = *reinterpret_cast<const float4*>(&counts[sub][column(q)]);
      const float4 v = *reinterpret_cast<const float4*>(&grads[sub][column(q)]);
      count[q] = c.x; count[q + 1] = c.y; count[q + 2] = c.z; count[q + 3] = c.w;
      grad[q] = v.x; grad[q + 1] = v.y; grad[q + 2] = v.z; grad[q + 3] = v.w;
    }
    asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
    __builtin_amdgcn_wave_barrier();
    if (n > scored) {  // a sink counts once
#pragma unroll
      for (int q = 0; q < Q; ++q) {
        const int i = column(q);
        if (i < scored || i >= n) continue;
        count[q] = 1.0f;
        if (p.d_sinks) grad[q] = bf16_to_f32(p.d_sinks[tok * (n - scored) + i - scored]) * p.factor;
      }
    }
    float slope[Q];
    if (p.router == BUX_ROUTER_SOFTMAX) {
      float m = z[0];
#pragma unroll
      for (int q = 1; q < Q; ++q) m = fmaxf(m, z[q]);
      m = lanes_max<L>(m);
      float sum = 0.0f;
#pragma unroll
      for (int q = 0; q < Q; ++q) {
        s[q] = expf(z[q] - m);
        sum += s[q];
      }
      const float inv = 1.0f / lanes_sum<L>(sum);
#pragma unroll
      for (int q = 0; q < Q; ++q) slope[q] = s[q] *= inv;
    } else {
#pragma unroll
      for (int q = 0; q < Q; ++q) {
        score_of(p.router, z[q], &s[q], &slope[q]);
        if (column(q) >= n) s[q] = slope[q] = 0.0f;
      }
    }
    if (p.normalize) {
      // a pick's ds = (g T - D) / T^2, each product rounded, so that a single pick's, whose weight
      // is constant, is 0
#pragma clang fp contract(off)
      float total = 0.0f, dot = 0.0f;
#pragma unroll
      for (int q = 0; q < Q; ++q) {
        total += count[q] * s[q];
        dot += grad[q] * s[q];
      }
      total = lanes_sum<L>(total);
      dot = lanes_sum<L>(dot);
      const float inv = total >= __FLT_MIN__ ? 1.0f / total : 0.0f;  // (1 / total may be infinite)
#pragma unroll
      for (int q = 0; q < Q; ++q) ds[q] = (grad[q] * total - count[q] * dot) * inv * inv;
    } else {
#pragma unroll
      for (int q = 0; q < Q; ++q) ds[q] = grad[q];
    }
    if (p.d_scores) {
#pragma unroll
      for (int q = 0; q < Q; q += 4) {
        float v[4];
        load4(p.d_scores + tok * scored, column(q), scored, 0.0f, v);
#pragma unroll
        for (int j = 0; j < 4; ++j) ds[q + j] += v[j];
      }
    }
    float inner = 0.0f;
    if (p.router == BUX_ROUTER_SOFTMAX) {
#pragma unroll
      for (int q = 0; q < Q; ++q) inner += ds[q] * s[q];
      inner = lanes_sum<L>(inner);
    }
#pragma unroll
    for (int q = 0; q < Q; ++q) ds[q] = (ds[q] - inner) * slope[q];
    if (p.d_logits) {
#pragma unroll
      for (int q = 0; q < Q; q += 4) {
        float v[4];
        load4(p.d_logits + tok * n, column(q), n, 0.0f, v);
#pragma unroll
        for (int j = 0; j < 4; ++j) ds[q + j] += v[j];
      }
    }
#pragma unroll
    for (int q = 0; q < Q; q += 4) {
      float d[4];
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        d[j] = live && column(q + j) < n ? ds[q + j] * p.logit_scale : 0.0f;
        bias[q + j] += d[j];
      }
      if (column(q) < p.npad) {
        const int64_t at = at_block(base + sub, column(q), p.npad);
#pragma unroll
        for (int part = 0; part < PARTS; ++part)
          *reinterpret_cast<uint2*>(p.parts[part] + at) =
              make_uint2(next_part(d[0], d[1]), next_part(d[2], d[3]));
      }
    }
  }
  if (p.bias_partials == nullptr) return;
#pragma unroll
  for (int q = 0; q < Q; ++q) counts[sub][column(q)] = bias[q];
  __syncthreads();
  for (int i = threadIdx.x; i < p.npad; i += THREADS) {
    float s = counts[0][i];
#pragma unroll
    for (int j = 1; j < TOKENS; ++j) s += counts[j][i];
    p.bias_partials[static_cast<int64_t>(blockIdx.x) * p.npad + i] = s;
  }
}

__device__ __forceinline__ bf16x8 load8(const uint16_t* p) {
  return __builtin_bit_cast(bf16x8, *reinterpret_cast<const uint4*>(p));
}

// dx: a wave 32 RB tokens by 128 columns, K = npad in 16s, the operands from L2 straight to
// registers: the tokens' a step ahead, the kernel's blocks as the step's last product of each goes
// out (both a step ahead would leave two waves a SIMD). MFMA with the kernel's rows first: lane l holds token l % 32, runs of 4
// columns 8 g + 4 (l / 32) of each block. The results pass LDS (32 tokens by 64 columns at a
// time) so that 8 lanes store 128 bytes of a row, with dz added in float32 before the one
// rounding; dz's loads go out ahead of what they wait beside: the first 32 tokens' before the
// products, the next 32's before the first are stored.
constexpr int COLS = 128;
constexpr int DX_PITCH = COLS / 2 + 4;  // floats: rows 16 bytes past a multiple of the banks
constexpr size_t DX_BYTES = (THREADS / 64) * 32 * DX_PITCH * sizeof(float);
template <int RB>
__device__ __forceinline__ void dx_tile(const Params& p, uint32_t block, uint32_t columns,
                                        uint8_t* smem) {
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), lane = threadIdx.x & 63;
  const int r = lane & 31, h = lane >> 5;
  const int64_t t0 = static_cast<int64_t>(block / columns) * (32 * RB);
  const int64_t c0 = (static_cast<int64_t>(block % columns) * 4 + wave) * COLS;
  if (c0 >= p.d) return;  // no barrier follows
  // blocks past the last: the last one's, not stored
  const int64_t t_last = (p.t - 1) >> 5, c_last = (p.d - 1) >> 5;
  const int64_t stride = static_cast<int64_t>(p.npad) * 32;  // elements of a row of blocks
  const uint16_t* a[RB][PARTS];
  const uint16_t* b[4];
#pragma unroll
  for (int i = 0; i < RB; ++i) {
    const int64_t at = ((t0 >> 5) + i < t_last ? (t0 >> 5) + i : t_last) * stride;
#pragma unroll
    for (int part = 0; part < PARTS; ++part) a[i][part] = p.parts[part] + at;
  }
#pragma unroll
  for (int j = 0; j < 4; ++j)
    b[j] = p.blocks + ((c0 >> 5) + j < c_last ? (c0 >> 5) + j : c_last) * stride;
  // this lane's 8 columns of 8 rows of each 32 x 64
  const int srow = lane >> 3, scol = 8 * (lane & 7);
  uint4 add[2][4];
  auto load_dz = [&](int i) {
#pragma unroll
    for (int half = 0; half < 2; ++half)
#pragma unroll
      for (int it = 0; it < 4; ++it) {
        const int64_t tok = t0 + 32 * i + it * 8 + srow, col = c0 + 64 * half + scol;
        add[half][it] = make_uint4(0, 0, 0, 0);
        if (tok < p.t && col < p.d)
          add[half][it] = *reinterpret_cast<const uint4*>(p.dz + tok * p.d + col);
      }
  };
  if (p.dz) load_dz(0);
  v16f acc[RB][4];
#pragma unroll
  for (int i = 0; i < RB; ++i)
#pragma unroll
    for (int j = 0; j < 4; ++j) acc[i][j] = v16f{};
  struct Tokens {
    bf16x8 g[RB][PARTS];
  };
  bf16x8 w[4];
  auto load = [&](Tokens& s, int32_t e) {
#pragma unroll
    for (int i = 0; i < RB; ++i)
#pragma unroll
      for (int part = 0; part < PARTS; ++part) s.g[i][part] = load8(a[i][part] + e * 32 + lane * 8);
  };
  auto load_w = [&](int j, int32_t e) { w[j] = load8(b[j] + e * 32 + lane * 8); };  // two blocks of 8
  // a step: the next one's tokens, then each of the kernel's blocks as its last product is under way
  auto step = [&](const Tokens& now, Tokens& next, int32_t e, bool more) {
    if (more) load(next, e + 16);
    __builtin_amdgcn_sched_barrier(0);
#pragma unroll
    for (int j = 0; j < 4; ++j) {
#pragma unroll
      for (int part = 0; part < PARTS; ++part)
#pragma unroll
        for (int i = 0; i < RB; ++i)
          acc[i][j] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(w[j], now.g[i][part], acc[i][j], 0, 0, 0);
      __builtin_amdgcn_sched_barrier(0);
      if (more) load_w(j, e + 16);
      __builtin_amdgcn_sched_barrier(0);
    }
  };
  Tokens one, two;
  load(one, 0);
#pragma unroll
  for (int j = 0; j < 4; ++j) load_w(j, 0);
  for (int32_t e = 0; e < p.npad; e += 32) {  // npad is a multiple of 32
    step(one, two, e, true);
    step(two, one, e + 16, e + 32 < p.npad);
  }
  float* mine = reinterpret_cast<float*>(smem) + wave * 32 * DX_PITCH;
#pragma unroll
  for (int i = 0; i < RB; ++i) {
    uint4 now[2][4];
#pragma unroll
    for (int half = 0; half < 2; ++half)
#pragma unroll
      for (int it = 0; it < 4; ++it) now[half][it] = add[half][it];
    if (p.dz && i + 1 < RB) load_dz(i + 1);
#pragma unroll
    for (int half = 0; half < 2; ++half) {
#pragma unroll
      for (int j = 0; j < 2; ++j)
#pragma unroll
        for (int g = 0; g < 4; ++g) {
          const v16f& c = acc[i][2 * half + j];
          *reinterpret_cast<float4*>(mine + r * DX_PITCH + 32 * j + 8 * g + 4 * h) =
              make_float4(c[4 * g], c[4 * g + 1], c[4 * g + 2], c[4 * g + 3]);
        }
      // the wave's own region: its LDS operations run in order
      asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
      __builtin_amdgcn_wave_barrier();
      const int64_t col = c0 + 64 * half + scol;
#pragma unroll
      for (int it = 0; it < 4; ++it) {
        const int64_t tok = t0 + 32 * i + it * 8 + srow;
        float v[8];
        Elem<float>::load8(mine + (it * 8 + srow) * DX_PITCH + scol, v);
        if (p.dz) {
          const uint32_t w[4] = {now[half][it].x, now[half][it].y, now[half][it].z, now[half][it].w};
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            v[2 * e] += __uint_as_float(w[e] << 16);
            v[2 * e + 1] += __uint_as_float(w[e] & 0xffff0000u);
          }
        }
        if (tok < p.t && col < p.d)
          *reinterpret_cast<uint4*>(p.dx + tok * p.d + col) =
              make_uint4(pack_bf16x2(v[0], v[1]), pack_bf16x2(v[2], v[3]), pack_bf16x2(v[4], v[5]),
                         pack_bf16x2(v[6], v[7]));
      }
      asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
      __builtin_amdgcn_wave_barrier();
    }
  }
}

// d_kernel's partial sums: a workgroup 128 of d by 128 logits over a slice of the tokens, 16 a
// step, in a ring of LDS stages that direct loads fill RING - 1 steps ahead (48 KiB, so that three
// workgroups fit a CU: steps of 32 in two stages of 32 KiB 84 us eager for 16384 tokens of 2048, 128
// logits, so 79). A stage holds the step's operands as they lie in memory, x's tokens of 256
// bytes (16-byte chunk c of token k at place c ^ 4 (k % 4)) and G's half blocks, 16 of 16 tokens by
// one chunk (token k of chunk c at place k ^ 4 (c % 4)): a load is runs of 256 bytes, and the 16
// lanes of a read hit every bank once. ds_read_b64_tr_b16 transposes on the way out (within each
// 16 lanes, lane j's 16-bit element e is element j % 4 of the 8 bytes that lane 4 e + j / 4 read).
// Columns past d or npad read what follows them in memory, into sums that are not stored;
// tokens past the last read 0.
constexpr int STEP = 16;
constexpr int RING = 3;
struct KStage {
  uint16_t x[STEP * COLS], g[PARTS][STEP * COLS];
};

// 8 tokens of a lane's column: 4 and the 4 after them.
__device__ __forceinline__ bf16x8 read_tr(uint32_t at, uint32_t at4) {
  const v4s a = __builtin_amdgcn_ds_read_tr16_b64_v4i16(reinterpret_cast<lds_v4s*>(at));
  const v4s b = __builtin_amdgcn_ds_read_tr16_b64_v4i16(reinterpret_cast<lds_v4s*>(at4));
  return __builtin_bit_cast(bf16x8, __builtin_shufflevector(a, b, 0, 1, 2, 3, 4, 5, 6, 7));
}

constexpr size_t RING_BYTES = RING * sizeof(KStage);

// Four logits of row j of d_kernel.
__device__ __forceinline__ void store_kernel(const Params& p, int64_t j, int32_t e, float4 v) {
  uint16_t* const out = p.d_kernel + j * p.n + e;
  if ((p.n & 3) == 0 && (reinterpret_cast<uintptr_t>(out) & 7) == 0) {
    if (e < p.n)
      *reinterpret_cast<uint2*>(out) = make_uint2(pack_bf16x2(v.x, v.y), pack_bf16x2(v.z, v.w));
    return;
  }
  const float f[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
  for (int q = 0; q < 4; ++q)
    if (e + q < p.n) out[q] = f32_to_bf16(f[q]);
}

__device__ __forceinline__ void kernel_grad_tile(const Params& p, uint32_t block, uint8_t* smem) {
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), lane = threadIdx.x & 63;
  // the logits' tiles of one slice and columns beside each other, then the columns'
  const uint32_t e_tiles = (p.npad + COLS - 1) / COLS, j_tiles = (p.d + COLS - 1) / COLS;
  const int32_t e0 = block % e_tiles * COLS;
  const int64_t j0 = static_cast<int64_t>(block / e_tiles % j_tiles) * COLS;
  const int64_t slice = block / e_tiles / j_tiles;
  const int64_t lo_t = slice * p.slice;
  const int64_t hi_t = lo_t + p.slice < p.t ? lo_t + p.slice : p.t;
  const int steps = static_cast<int>((hi_t - lo_t + STEP - 1) / STEP);
  const uint32_t lds0 = lds_at(smem);
  // a wave's load of x: 4 tokens, lane l the l / 16th's chunk that belongs in place l % 16; of one
  // of G's parts: 4 chunks, lane l the l / 16th's token that belongs in place l % 16
  const int row = 4 * wave + (lane >> 4);
  const int chunk = (lane & 15) ^ (4 * ((lane >> 4) & 3));
  const int x_row = static_cast<int>(p.d) * 2, g_tokens = p.npad * 64;  // bytes of 32 tokens of G
  const int x_off = row * x_row + 16 * chunk;
  const int g_chunk = 4 * wave + (lane >> 4);
  const int g_off = g_chunk * 512 + ((lane & 15) ^ (4 * (g_chunk & 3))) * 16;
  auto issue = [&](int s) {
    const int64_t tok = lo_t + static_cast<int64_t>(s) * STEP;
    const uint32_t at = lds0 + (s % RING) * sizeof(KStage) + wave * 1024;
    const i32x4 xr = resource(p.x + tok * p.d + j0, ((p.t - tok) * p.d - j0) * 2);
    load_lds16_uniform(xr, at + offsetof(KStage, x), x_off, 0);
    // its 32 tokens' blocks from e0 on, and the step's tokens of them
    const int64_t g = (tok & ~static_cast<int64_t>(31)) * p.npad + static_cast<int64_t>(e0) * 32;
    const int in_block = static_cast<int>(tok & 31) * 16;
#pragma unroll
    for (int part = 0; part < PARTS; ++part) {
      const i32x4 gr = resource(p.parts[part] + g, g_tokens - e0 * 64);
      load_lds16_uniform(gr, at + offsetof(KStage, g) + part * sizeof(KStage::g[0]), g_off, in_block);
    }
  };
  // wave (a, b) of 2 x 2: 64 of d from 64 a, 64 logits from 64 b; block q of 32 columns
  const int s16 = lane & 15, kq = s16 >> 2;
  const int col = 16 * ((lane >> 4) & 1) + 4 * (s16 & 3);
  auto offset = [&](int block) {
    return (8 * (lane >> 5) + kq) * 256 + 16 * (4 * (block ^ kq) + (col >> 3)) +
           8 * ((col >> 2) & 1);
  };
  auto block_offset = [&](int block) {
    const int c = 4 * block + (col >> 3), k = 8 * (lane >> 5) + kq;
    return c * (16 * STEP) + (k ^ (4 * (c & 3))) * 16 + 8 * ((col >> 2) & 1);
  };
  uint32_t xat[2], gat[2];
#pragma unroll
  for (int q = 0; q < 2; ++q) {
    xat[q] = offset(2 * (wave >> 1) + q);
    gat[q] = block_offset(2 * (wave & 1) + q);
  }
  v16f acc[2][2];
#pragma unroll
  for (int i = 0; i < 2; ++i)
#pragma unroll
    for (int j = 0; j < 2; ++j) acc[i][j] = v16f{};
  for (int s = 0; s < RING - 1 && s < steps; ++s) issue(s);
  for (int s = 0; s < steps; ++s) {
    // this step's loads are in, those of the RING - 2 after it may not be
    if (s + RING - 2 < steps)
      asm volatile("s_waitcnt vmcnt(%0)" ::"n"((RING - 2) * (1 + PARTS)) : "memory");
    else
      asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
    // ... in every wave; and every wave has read the stage that the next loads take
    asm volatile("s_waitcnt lgkmcnt(0)\n\ts_barrier" ::: "memory");
    if (s + RING - 1 < steps) issue(s + RING - 1);
    const uint32_t at = lds0 + (s % RING) * sizeof(KStage);
    bf16x8 xv[2], gv[2][PARTS];
#pragma unroll
    for (int q = 0; q < 2; ++q) {
      const uint32_t x = at + offsetof(KStage, x) + xat[q];
      xv[q] = read_tr(x, x + 1024);  // 4 tokens on: 1 KiB of x, of G place ^ 4
#pragma unroll
      for (int part = 0; part < PARTS; ++part) {
        const uint32_t g = at + offsetof(KStage, g) + part * sizeof(KStage::g[0]);
        gv[q][part] = read_tr(g + gat[q], g + (gat[q] ^ 64));
      }
    }
#pragma unroll
    for (int part = 0; part < PARTS; ++part)
#pragma unroll
      for (int i = 0; i < 2; ++i)
#pragma unroll
        for (int j = 0; j < 2; ++j)
          acc[i][j] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(gv[j][part], xv[i], acc[i][j], 0, 0, 0);
  }
  float* base = p.kernel_partials + slice * p.d * p.npad;
  const bool last = p.slices == 1;  // nothing to add: the gradient itself
#pragma unroll
  for (int i = 0; i < 2; ++i) {
    const int64_t j = j0 + 64 * (wave >> 1) + 32 * i + (lane & 31);
    if (j >= p.d) continue;
#pragma unroll
    for (int q = 0; q < 2; ++q)
#pragma unroll
      for (int g = 0; g < 4; ++g) {
        const int32_t e = e0 + 64 * (wave & 1) + 32 * q + 8 * g + 4 * (lane >> 5);
        const float4 v = make_float4(acc[i][q][4 * g], acc[i][q][4 * g + 1], acc[i][q][4 * g + 2],
                                     acc[i][q][4 * g + 3]);
        if (last) store_kernel(p, j, e, v);
        else if (e < p.npad) *reinterpret_cast<float4*>(base + j * p.npad + e) = v;
      }
  }
}

// d_bias of 16 logits: 16 threads a logit, every 16th partial each, then their sums in order.
__device__ __forceinline__ void bias_tile(const Params& p, uint32_t block, float (*part)[16]) {
  const int row = threadIdx.x >> 4, lane = threadIdx.x & 15;
  const int32_t e = static_cast<int32_t>(block) * 16 + lane;
  float s = 0.0f;
  if (e < p.n) {
#pragma unroll 8
    for (int32_t b = row; b < p.grads_blocks; b += 16)
      s += p.bias_partials[static_cast<int64_t>(b) * p.npad + e];
  }
  part[row][lane] = s;
  __syncthreads();
  if (row != 0 || e >= p.n) return;
#pragma unroll
  for (int r = 1; r < 16; ++r) s += part[r][lane];
  p.d_bias[e] = s;
}

// Of `count` tiles, workgroup b's: an XCD (a workgroup's id modulo 8) takes a contiguous share, so
// that the tiles of the same tokens find G in its L2 (16384 tokens of 2048, 128 logits 67.1 us,
// so 62.0; the kernel's gradient of several tiles of logits loses by it: 8192 of 7168, 256 logits
// 176 us and 185, the best of 30 each). in_shares: workgroups for all of them.
__host__ __device__ __forceinline__ uint32_t in_shares(uint32_t count) { return (count + 7) / 8 * 8; }
__device__ __forceinline__ uint32_t shared(uint32_t b, uint32_t count) {
  return b % 8 * ((count + 7) / 8) + b / 8;
}

// Both products in one launch, so that either's loads fill the other's waits: the kernel's
// gradient's workgroups first, which take longer; and d_bias's.
template <int RB>
__global__ __launch_bounds__(THREADS, RB == 1 ? 3 : 2) void products_kernel(
    Params p, uint32_t kernel_blocks, uint32_t bias_blocks, uint32_t dx_blocks, uint32_t columns) {
  extern __shared__ __align__(16) uint8_t smem[];
  uint32_t block = blockIdx.x;
  const uint32_t grads = in_shares(kernel_blocks);
  if (block < grads) {
    if (p.npad <= COLS) block = shared(block, kernel_blocks);
    if (block < kernel_blocks) kernel_grad_tile(p, block, smem);
    return;
  }
  block -= grads;
  if (block < bias_blocks) return bias_tile(p, block, reinterpret_cast<float(*)[16]>(smem));
  block = shared(block - bias_blocks, dx_blocks);
  if (block < dx_blocks) dx_tile<RB>(p, block, columns, smem);
}

// d_kernel: the slices' sums in order, 4 logits a thread; and, with no tokens, d_bias.
__global__ __launch_bounds__(THREADS) void reduce_kernel(Params p, int64_t kernel_blocks) {
  __shared__ float part[16][16];
  const int64_t size = p.d * p.npad;
  if (static_cast<int64_t>(blockIdx.x) >= kernel_blocks)
    return bias_tile(p, blockIdx.x - static_cast<uint32_t>(kernel_blocks), part);
  const int64_t i = (static_cast<int64_t>(blockIdx.x) * THREADS + threadIdx.x) * 4;
  if (i >= size) return;
  float4 v = make_float4(0, 0, 0, 0);
#pragma unroll 8
  for (int32_t s = 0; s < p.slices; ++s) {
    const float4 a = *reinterpret_cast<const float4*>(p.kernel_partials + s * size + i);
    v.x += a.x;
    v.y += a.y;
    v.z += a.z;
    v.w += a.w;
  }
  const int64_t j = i / p.npad;
  store_kernel(p, j, static_cast<int32_t>(i - j * p.npad), v);
}

// The lanes grads_kernel gives a token.
int lanes_of(int32_t npad) { return npad <= 128 ? 16 : npad <= 256 ? 32 : 64; }

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
  const int64_t blocks = ceil_div(ceil_div(t, 32) * 32, THREADS / lanes_of(w.npad));
  w.grads_blocks = static_cast<int32_t>(blocks < MAX_GRADS_BLOCKS ? blocks : MAX_GRADS_BLOCKS);
  // a workgroup a CU for the kernel's gradient (two measured no faster beside dx's, and their
  // partial sums' addition 1.6 us slower), slices of 128 tokens at least (500 tokens of 2048, 128
  // logits, all three kernels: of 256 20.7 us, of 128 18.0, of 64 19.9)
  const int64_t tiles = ceil_div(d, COLS) * ceil_div(w.npad, COLS);
  const int64_t most = 256 / tiles > 1 ? 256 / tiles : 1;
  const int64_t by_tokens = ceil_div(t > 0 ? t : 1, 128);
  const int64_t slices = most < by_tokens ? most : by_tokens;
  w.slice = ceil_div(ceil_div(t > 0 ? t : 1, slices), STEP) * STEP;
  w.slices = static_cast<int32_t>(ceil_div(t, w.slice));
  auto whole = [](size_t v) { return (v + 255) & ~static_cast<size_t>(255); };
  const size_t part = static_cast<size_t>(ceil_div(t, 32) * 32) * w.npad * sizeof(uint16_t);
  w.parts = 0;
  w.kernel = PARTS * part;
  w.bias = w.kernel + static_cast<size_t>(ceil_div(d, 32) * 32) * w.npad * sizeof(uint16_t);
  w.partials = w.bias + whole(static_cast<size_t>(w.grads_blocks) * w.npad * sizeof(float));
  // for as many slices as asked for, though whole steps may fill fewer: so that the size never
  // falls as t grows
  w.bytes = w.partials + static_cast<size_t>(slices) * d * w.npad * sizeof(float);
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
  BUX_CHECK(t >= 0 && t < (1LL << 31) && d > 0 && d % 16 == 0 && d <= (1LL << 24),
            "bux_route_backward: t=%lld d=%lld (d a positive multiple of 16, up to 2^24)",
            (long long)t, (long long)d);
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
  auto aligned = [](const void* q) { return reinterpret_cast<uintptr_t>(q) % 16 == 0; };
  BUX_CHECK(aligned(x) && aligned(dz) && aligned(dx) && aligned(workspace),
            "bux_route_backward: x, dz, dx and the workspace are 16-byte aligned");
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
  for (int part = 0; part < PARTS; ++part)
    p.parts[part] = reinterpret_cast<uint16_t*>(ws + w.parts + part * (w.kernel / PARTS));
  p.blocks = reinterpret_cast<uint16_t*>(ws + w.kernel);
  p.bias_partials = d_bias ? reinterpret_cast<float*>(ws + w.bias) : nullptr;
  p.kernel_partials = reinterpret_cast<float*>(ws + w.partials);
  p.grads_blocks = t > 0 ? w.grads_blocks : 0;
  p.slices = t > 0 ? w.slices : 0;
  p.slice = w.slice;
  p.dx = dx;
  p.d_kernel = d_kernel;
  p.d_bias = d_bias;
  if (t > 0) {
    auto grads = [&](auto lanes, auto q) {
      hipLaunchKernelGGL((grads_kernel<decltype(lanes)::value, decltype(q)::value>),
                         dim3(static_cast<unsigned>(w.grads_blocks + ceil_div(d * w.npad, 4 * THREADS))),
                         dim3(THREADS), 0, s, p);
    };
    using std::integral_constant;
    if (p.npad <= 64) grads(integral_constant<int, 16>{}, integral_constant<int, 4>{});
    else if (p.npad <= 128) grads(integral_constant<int, 16>{}, integral_constant<int, 8>{});
    else if (p.npad <= 256) grads(integral_constant<int, 32>{}, integral_constant<int, 8>{});
    else if (p.npad <= 512) grads(integral_constant<int, 64>{}, integral_constant<int, 8>{});
    else grads(integral_constant<int, 64>{}, integral_constant<int, 16>{});
    if (int rc = launched("route grads_kernel")) return rc;
    const uint32_t columns = static_cast<uint32_t>(ceil_div(d, 4 * COLS));
    const uint32_t tiles =
        static_cast<uint32_t>(ceil_div(d, COLS) * ceil_div(w.npad, COLS) * w.slices);
    const uint32_t bias = d_bias ? static_cast<uint32_t>(ceil_div(n_logits, 16)) : 0;
    constexpr size_t LDS = RING_BYTES > DX_BYTES ? RING_BYTES : DX_BYTES;
    auto products = [&](auto rb) {
      constexpr int RB = decltype(rb)::value;
      const uint32_t dx_blocks = columns * static_cast<uint32_t>(ceil_div(t, 32 * RB));
      hipLaunchKernelGGL((products_kernel<RB>),
                         dim3(in_shares(tiles) + bias + in_shares(dx_blocks)), dim3(THREADS), LDS,
                         s, p, tiles, bias, dx_blocks, columns);
    };
    static_assert(LDS <= 64 * 1024, "a launch's LDS without an attribute");
    // 32 tokens a wave where its products are few, with three waves a SIMD to hide their loads; 64
    // where the kernel's loads for them count (16384 tokens, 2048 columns, 128 logits: 62.0 us and
    // 65.8; 8192, 7168, 256: 223 and 207) and there are workgroups to fill the chip
    if (w.npad > 128 && ceil_div(t, 64) * columns >= 256) products(integral_constant<int, 2>{});
    else products(integral_constant<int, 1>{});
    if (int rc = launched("route products_kernel"); rc != BUX_OK || w.slices == 1) return rc;
  }
  const int64_t kernel_blocks = ceil_div(d * w.npad, 4 * THREADS);
  const int64_t bias_blocks = d_bias && t == 0 ? ceil_div(n_logits, 16) : 0;
  hipLaunchKernelGGL(reduce_kernel, dim3(static_cast<unsigned>(kernel_blocks + bias_blocks)),
                     dim3(THREADS), 0, s, p, kernel_blocks);
  return launched("route reduce_kernel");
}
