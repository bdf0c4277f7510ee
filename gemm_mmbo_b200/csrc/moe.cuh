// A whole mixture-of-experts layer for a few tokens:
//
//   p(t, :) = softmax(router * x_t),  S(t) = the topk experts of largest p (equal ones: the lower index first)
//   g(t, e) = p(t, e)                 (or p(t, e) / sum of p over S(t))
//   y_t     = sum over e in S(t) of g(t, e) * down_e * (silu(gate_e * x_t) o (up_e * x_t))  +  beta * y_t
//
// with silu(v) = v / (1 + exp(-v)).  All sums, the softmax and the products in between are held in 32 bits.
#pragma once

#include "w4.cuh"

namespace mmbo {

struct MoeArgs {
  size_t tokens, d, f, experts, topk;
  int renorm;
  W4Format fmt;             // 4-bit experts; group 0: 16-bit ones
  const void *X, *router, *gate, *up, *down;
  size_t ldx, ldr, ldg, strideG, ldd, strideD;  // strides in elements, for packed experts in bytes
  float beta;
  void* Y;
  size_t ldy;
  int* ids;       // tokens x topk, expert numbers (workspace or the caller's)
  float* gates;   // tokens x topk
  float* hidden;  // tokens * topk x f
};

// Order of the scores as unsigned integers: larger score, larger key; -0 equals +0; NaN comes first.
__device__ __forceinline__ uint32_t moe_score_key(float v) {
  if (v != v) return 0xffffffffu;
  if (v == 0.f) v = 0.f;
  const uint32_t b = __float_as_uint(v);
  return (b & 0x80000000u) ? ~b : (b | 0x80000000u);
}

// Sum over k of row `p` times x, by one warp.
template <typename T>
__device__ __forceinline__ float row_dot(const T* __restrict__ p, const T* __restrict__ x, size_t k) {
  float acc = 0.f;
  for (size_t j = threadIdx.x & 31; j < k; j += 32) acc = fmaf(to_f32(p[j]), to_f32(x[j]), acc);
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) acc += __shfl_xor_sync(0xffffffffu, acc, o);
  return acc;
}

// One block per token: scores by one warp per expert, then the selection by the first warp.
template <typename T>
__global__ void moe_route_kernel(MoeArgs a) {
  extern __shared__ float scores[];
  const size_t t = blockIdx.x;
  const int lane = threadIdx.x & 31, warp = threadIdx.x / 32, warps = blockDim.x / 32;
  const T* x = static_cast<const T*>(a.X) + t * a.ldx;
  for (size_t e = warp; e < a.experts; e += warps) {
    const float v = row_dot(static_cast<const T*>(a.router) + e * a.ldr, x, a.d);
    if (lane == 0) scores[e] = v;
  }
  __syncthreads();
  if (warp != 0) return;
  float top = -INFINITY, sum = 0.f;
  for (size_t e = lane; e < a.experts; e += 32) top = fmaxf(top, scores[e]);
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, o));
  for (size_t e = lane; e < a.experts; e += 32) sum += expf(scores[e] - top);
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
  float chosen = 0.f;
  uint64_t last = ~0ull;  // (key, ~index) of the expert taken before
  for (size_t s = 0; s < a.topk; ++s) {
    uint64_t best = 0;
    for (size_t e = lane; e < a.experts; e += 32) {
      const uint64_t c = ((uint64_t)moe_score_key(scores[e]) << 32) | (0xffffffffu - (uint32_t)e);
      if (c < last && c > best) best = c;
    }
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) {
      const uint64_t c = __shfl_xor_sync(0xffffffffu, best, o);
      best = c > best ? c : best;
    }
    last = best;
    const uint32_t e = 0xffffffffu - (uint32_t)best;
    const float p = expf(scores[e] - top) / sum;
    chosen += p;
    if (lane == 0) {
      a.ids[t * a.topk + s] = (int)e;
      a.gates[t * a.topk + s] = p;
    }
  }
  __syncwarp();
  if (a.renorm)
    for (size_t s = lane; s < a.topk; s += 32) a.gates[t * a.topk + s] /= chosen;
}

template <typename T>
__device__ __forceinline__ float moe_row(const MoeArgs& a, const void* w, size_t ld, size_t stride, size_t e, size_t i,
                                         size_t k, const T* x) {
  if (a.fmt.group) return w4_row_dot(static_cast<const unsigned char*>(w) + e * stride, a.fmt, i, k, x);
  return row_dot(static_cast<const T*>(w) + e * stride + i * ld, x, k);
}

// One warp per (token and slot, row of the experts' hidden vector).
template <typename T>
__global__ void moe_up_simple_kernel(MoeArgs a) {
  const size_t i = (size_t)blockIdx.x * (blockDim.x / 32) + threadIdx.x / 32;
  if (i >= a.f) return;
  for (size_t pair = blockIdx.y; pair < a.tokens * a.topk; pair += gridDim.y) {
    const size_t e = a.ids[pair];
    const T* x = static_cast<const T*>(a.X) + pair / a.topk * a.ldx;
    const float g = moe_row(a, a.gate, a.ldg, a.strideG, e, i, a.d, x);
    const float u = moe_row(a, a.up, a.ldg, a.strideG, e, i, a.d, x);
    if ((threadIdx.x & 31) == 0) a.hidden[pair * a.f + i] = g / (1.f + expf(-g)) * u;
  }
}

// One warp per (token, row of the output).
template <typename T>
__global__ void moe_down_simple_kernel(MoeArgs a) {
  const size_t i = (size_t)blockIdx.x * (blockDim.x / 32) + threadIdx.x / 32;
  const int lane = threadIdx.x & 31;
  if (i >= a.d) return;
  for (size_t t = blockIdx.y; t < a.tokens; t += gridDim.y) {
    float y = 0.f;
    for (size_t s = 0; s < a.topk; ++s) {
      const size_t pair = t * a.topk + s, e = a.ids[pair];
      const float* h = a.hidden + pair * a.f;
      float acc = 0.f;
      for (size_t j = lane; j < a.f; j += 32) {
        float w;
        if (a.fmt.group) {
          const size_t tiles = w4_k_tiles(a.f);
          const unsigned char* in = static_cast<const unsigned char*>(a.down) + e * a.strideD +
                                    (i / kW4Rows * tiles + j / kW4Cols) * a.fmt.tile_bytes();
          const int row = (int)(i % kW4Rows), c = (int)(j % kW4Cols), g = c / a.fmt.group;
          const uint32_t word = *reinterpret_cast<const uint32_t*>(in + w4_piece(row, c % 32 / 8) + c / 32 * 4);
          const int el = c % 8, z = a.fmt.zeros ? in[a.fmt.zero_at(g, row)] : 8;
          w = (float)((int)((word >> (4 * w4_nibble(el))) & 15u) - z) *
              to_f32(*reinterpret_cast<const T*>(in + a.fmt.scale_at(g, row)));
        } else {
          w = to_f32(static_cast<const T*>(a.down)[e * a.strideD + i * a.ldd + j]);
        }
        acc = fmaf(w, h[j], acc);
      }
#pragma unroll
      for (int o = 16; o > 0; o >>= 1) acc += __shfl_xor_sync(0xffffffffu, acc, o);
      y = fmaf(a.gates[pair], acc, y);
    }
    if (lane == 0) {
      T* out = static_cast<T*>(a.Y) + t * a.ldy + i;
      *out = from_f32<T>(a.beta != 0.f ? fmaf(a.beta, to_f32(*out), y) : y);
    }
  }
}

}  // namespace mmbo
