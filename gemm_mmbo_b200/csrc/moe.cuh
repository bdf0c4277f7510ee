// A whole mixture-of-experts layer for a few tokens:
//
//   p(t, :) = softmax(router * x_t),  S(t) = the topk experts of largest p (equal ones: the lower index first)
//   g(t, e) = p(t, e)                 (or p(t, e) / sum of p over S(t))
//   y_t     = sum over e in S(t) of g(t, e) * down_e * (silu(gate_e * x_t) o (up_e * x_t))  +  beta * y_t
//
// with silu(v) = v / (1 + exp(-v)).  All sums, the softmax and the products in between are held in 32 bits.
//
// What bounds it: the bytes of the experts that the tokens choose.  Three kernels in one stream, each started while the
// one in front drains (programmatic dependent launch):
//   scores   one warp per (token, expert); also an aligned, zero-padded copy of the activations
//   up       every block repeats the selection for itself (a microsecond, cheaper than another kernel and its launch), then
//            works through its share of the units (expert, 16 rows of gate and up): sixteen warps split d
//   down     a block owns 16 rows of the output for all tokens, its warps split the list of (expert, part of f); the sums
//            of the experts meet in shared memory in a fixed order
// Weights go straight from memory to registers, in the order of the fragments of mma.sync.m16n8k16: a lane reads 16 bytes
// of a row and the same 16 bytes' worth of k of its token, so that nothing is staged, and a warp has its next 64 columns
// (4 or 8 KB) under way while it multiplies.  Tokens are the eight columns of the instruction; an expert with more
// tokens is taken in groups of eight, the later ones finding its weights in L2.
#pragma once

#include "w4_umma.cuh"

namespace mmbo {

constexpr int kMoeWarps = 16, kMoeThreads = kMoeWarps * 32;
constexpr int kMoeTokens = 64;  // of one pass; more are taken in several

struct MoeArgs {
  int tokens, d, f, experts, topk, renorm;
  W4Format fmt;  // 4-bit experts; group 0: 16-bit ones
  const void *X, *router, *gate, *up, *down;
  size_t ldx, ldr, ldg, strideG, ldd, strideD;  // strides in elements, for packed experts in bytes
  float beta;
  void* Y;
  size_t ldy;
  int* ids;      // tokens x topk, the caller's or null
  float* gates;  // tokens x topk, the caller's or null
  // workspace
  float* scores;    // tokens x experts
  void* x;          // tokens x d_pad: the activations, zero behind d
  void* hidden;     // pairs x f_pad: floats, or bfloat16 twice (the value and what its rounding left)
  uint32_t* peak;   // pairs: bits of the largest hidden magnitude
  int* plan;        // what `up` found out for `down`, see MoePlan
  int d_pad, f_pad; // multiples of 128
  int hidden_f32;
};

// The selection, sorted by expert: `order` holds the pairs (token * topk + slot) of expert 0's tokens, then expert 1's ..;
// the a-th expert with tokens is expert[a], its pairs order[start[a] .. start[a + 1]).
struct MoePlan {
  int* active;  // number of experts with tokens
  int* expert;
  int* start;
  int* order;
  float* gate;  // per pair
  __host__ __device__ static int words(int experts, int pairs) {
    const int a = experts < pairs ? experts : pairs;
    return 1 + a + a + 1 + 2 * pairs;
  }
  __device__ __forceinline__ MoePlan(int* at, int experts, int pairs) {
    const int a = min(experts, pairs);
    active = at;
    expert = at + 1;
    start = expert + a;
    order = start + a + 1;
    gate = reinterpret_cast<float*>(order + pairs);
  }
};

// Order of the scores as unsigned integers: larger score, larger key; -0 equals +0; NaN comes first.
__device__ __forceinline__ uint32_t moe_score_key(float v) {
  if (v != v) return 0xffffffffu;
  if (v == 0.f) v = 0.f;
  const uint32_t b = __float_as_uint(v);
  return (b & 0x80000000u) ? ~b : (b | 0x80000000u);
}

template <typename T>
__global__ void __launch_bounds__(256) moe_scores_kernel(const MoeArgs a) {
  griddep_launch_dependents();
  griddep_wait();
  const int t = blockIdx.y, e = blockIdx.x * 8 + threadIdx.x / 32, lane = threadIdx.x & 31;
  const T* x = static_cast<const T*>(a.X) + (size_t)t * a.ldx;
  if (blockIdx.x == 0) {
    T* copy = static_cast<T*>(a.x) + (size_t)t * a.d_pad;
    for (int j = threadIdx.x * 8; j < a.d_pad; j += 256 * 8) *reinterpret_cast<uint4*>(copy + j) = load8(x, a.d, j);
    for (int s = threadIdx.x; s < a.topk; s += 256) a.peak[t * a.topk + s] = 0;
    // hidden vectors behind f: floats, or two rows of bfloat16 (zero bytes either way)
    uint16_t* h = static_cast<uint16_t*>(a.hidden) + (size_t)t * a.topk * a.f_pad * 2;
    const int pad = a.f_pad - a.f, per = a.hidden_f32 ? 1 : 2, width = a.hidden_f32 ? 2 : 1;
    for (int i = threadIdx.x; i < a.topk * per * pad * width; i += 256) {
      const int row = i / (pad * width), at = i % (pad * width);
      h[(size_t)row * a.f_pad * width + a.f * width + at] = 0;
    }
  }
  if (e >= a.experts) return;
  const T* w = static_cast<const T*>(a.router) + (size_t)e * a.ldr;
  float sum = 0.f;
#pragma unroll 4
  for (int j = lane * 8; j < a.d; j += 256) {
    const uint4 u = load8(w, a.d, j), v = load8(x, a.d, j);
    const uint32_t uw[4] = {u.x, u.y, u.z, u.w}, vw[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const float2 p = widen2<T>(uw[i]), q = widen2<T>(vw[i]);
      sum = fmaf(p.x, q.x, sum);
      sum = fmaf(p.y, q.y, sum);
    }
  }
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
  if (lane == 0) a.scores[(size_t)t * a.experts + e] = sum;
}

// The topk experts of one token by one warp: ids and gates (shared memory).
__device__ __forceinline__ void moe_select(const MoeArgs& a, const float* scores, int* ids, float* gates) {
  const int lane = threadIdx.x & 31;
  float top = -INFINITY, sum = 0.f;
  for (int e = lane; e < a.experts; e += 32) top = fmaxf(top, scores[e]);
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, o));
  for (int e = lane; e < a.experts; e += 32) sum += expf(scores[e] - top);
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
  float chosen = 0.f;
  uint64_t last = ~0ull;  // (key, ~index) of the expert taken before
  for (int s = 0; s < a.topk; ++s) {
    uint64_t best = 0;
    for (int e = lane; e < a.experts; e += 32) {
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
      ids[s] = (int)e;
      gates[s] = p;
    }
  }
  __syncwarp();
  if (a.renorm)
    for (int s = lane; s < a.topk; s += 32) gates[s] /= chosen;
}

// ---------------------------------------------------------------- fragments -----------
template <typename T>
__device__ __forceinline__ void mma_16816(float (&c)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0,
                                          uint32_t b1);
template <>
__device__ __forceinline__ void mma_16816<__half>(float (&c)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3,
                                                  uint32_t b0, uint32_t b1) {
  mma_f16(c, a0, a1, a2, a3, b0, b1);
}
template <>
__device__ __forceinline__ void mma_16816<__nv_bfloat16>(float (&c)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3,
                                                         uint32_t b0, uint32_t b1) {
  asm("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
      : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
      : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}

// Sixteen rows of 16-bit weights, 64 columns at a time: lane 4 r + t holds columns 32 u + 8 t .. + 7 of rows r and r + 8.
// `rows` that exist; the others and what lies behind `k` are zero.
template <typename T>
struct Rows16 {
  static constexpr int kStep = 64;
  uint4 w[2][2];
  __device__ __forceinline__ void load(const T* base, size_t ld, int rows, int k, int step, bool vec) {
    const int lane = threadIdx.x & 31, r = lane >> 2, t = lane & 3;
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      const T* row = base + (size_t)(r + 8 * h) * ld;
      const bool have = r + 8 * h < rows;
#pragma unroll
      for (int u = 0; u < 2; ++u) {
        const int j = step * 64 + u * 32 + t * 8;
        if (vec) {
          w[h][u] = have && j < k ? __ldcs(reinterpret_cast<const uint4*>(row + j)) : make_uint4(0, 0, 0, 0);
        } else {
          w[h][u] = load8(row, have ? k : 0, j);
        }
      }
    }
  }
  // acc += weights * columns; b: this lane's 16 bytes of each 32 columns
  __device__ __forceinline__ void multiply(float (&acc)[4], const uint4 (&b)[2]) const {
#pragma unroll
    for (int u = 0; u < 2; ++u) {
      mma_16816<T>(acc, w[0][u].x, w[1][u].x, w[0][u].y, w[1][u].y, b[u].x, b[u].y);
      mma_16816<T>(acc, w[0][u].z, w[1][u].z, w[0][u].w, w[1][u].w, b[u].z, b[u].w);
    }
  }
};

// Sixteen rows of packed weights, a tile of 128 columns at a time; U: the 16-bit type the products are formed in, S: the
// scales'.
template <typename S, typename U>
struct Rows4 {
  static constexpr int kStep = 128;
  uint4 c[2];
  uint32_t scale[4], zero[4];  // rows r and r + 8, by group
  __device__ __forceinline__ void load(const unsigned char* tile, const W4Format& f) {
    const int lane = threadIdx.x & 31, r = lane >> 2, t = lane & 3, groups = f.groups();
    c[0] = __ldcs(reinterpret_cast<const uint4*>(tile + w4_piece(r, t)));
    c[1] = __ldcs(reinterpret_cast<const uint4*>(tile + w4_piece(r, t) + 512));
#pragma unroll
    for (int g = 0; g < 4; ++g)
      if (g < groups) {
        scale[g] = *reinterpret_cast<const uint32_t*>(tile + f.scale_at(g, r));
        zero[g] = f.zeros ? *reinterpret_cast<const uint16_t*>(tile + f.zero_at(g, r)) : 0x0808u;
      }
  }
  // acc += weights * (columns of every b[i])
  template <int N>
  __device__ __forceinline__ void multiply(float (&acc)[4], const uint4 (&b)[N][4], const W4Format& f) const {
    const uint32_t w0[4] = {c[0].x, c[0].y, c[0].z, c[0].w}, w1[4] = {c[1].x, c[1].y, c[1].z, c[1].w};
    const int per = f.group / 32;
    W4Unpacker<U> lo, hi;
    float part[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
    for (int u = 0; u < 4; ++u) {
      const int g = per == 4 ? 0 : per == 2 ? u >> 1 : u;
      const uint32_t z = g == 0 ? zero[0] : g == 1 ? zero[1] : g == 2 ? zero[2] : zero[3];
      lo.set_zero(z & 15u);
      hi.set_zero(z >> 8 & 15u);
      uint32_t p[4], q[4];
      lo.unpack(w0[u], p);
      hi.unpack(w1[u], q);
#pragma unroll
      for (int i = 0; i < N; ++i) {
        mma_16816<U>(part, p[0], q[0], p[1], q[1], b[i][u].x, b[i][u].y);
        mma_16816<U>(part, p[2], q[2], p[3], q[3], b[i][u].z, b[i][u].w);
      }
      if (u == 3 || per == 1 || (per == 2 && u == 1)) {  // the group is complete
        const float2 s = widen2<S>(g == 0 ? scale[0] : g == 1 ? scale[1] : g == 2 ? scale[2] : scale[3]);
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          acc[i] = fmaf(i < 2 ? s.x : s.y, part[i], acc[i]);
          part[i] = 0.f;
        }
      }
    }
  }
};

// The power of two that brings a vector whose largest magnitude has these bits below 2^15.
__device__ __forceinline__ float moe_scale(uint32_t peak) {
  const int up = 14 - ((int)max(peak >> 23, 1u) - 127);
  return __uint_as_float((uint32_t)(min(max(up, -100), 100) + 127) << 23);
}

// ---------------------------------------------------------------- up ------------------
// Shared memory of both kernels: the plan, then partial sums.
template <typename T, bool W4>
__global__ void __launch_bounds__(kMoeThreads, 1) moe_up_kernel(const MoeArgs a) {
  extern __shared__ __align__(16) unsigned char smem[];
  const int warp = threadIdx.x / 32, lane = threadIdx.x & 31, r = lane >> 2, t = lane & 3;
  const int pairs = a.tokens * a.topk;
  MoePlan plan(reinterpret_cast<int*>(smem), a.experts, pairs);
  int* ids = reinterpret_cast<int*>(smem) + MoePlan::words(a.experts, pairs);
  int* count = ids + pairs;  // experts
  float* sums = reinterpret_cast<float*>(smem + ((size_t)(MoePlan::words(a.experts, pairs) + pairs + a.experts) * 4 + 15) / 16 * 16);
  griddep_launch_dependents();
  griddep_wait();

  // the selection, by every block for itself
  for (int e = threadIdx.x; e < a.experts; e += kMoeThreads) count[e] = 0;
  for (int tok = warp; tok < a.tokens; tok += kMoeWarps)
    moe_select(a, a.scores + (size_t)tok * a.experts, ids + tok * a.topk, plan.gate + tok * a.topk);
  __syncthreads();
  for (int p = threadIdx.x; p < pairs; p += kMoeThreads) atomicAdd(&count[ids[p]], 1);
  __syncthreads();
  if (warp == 0) {  // experts with tokens, numbered in order, and where their pairs start
    int n = 0, at = 0;
    for (int e0 = 0; e0 < a.experts; e0 += 32) {
      const int e = e0 + lane, c = e < a.experts ? count[e] : 0;
      int before = c;
#pragma unroll
      for (int o = 1; o < 32; o <<= 1) {
        const int v = __shfl_up_sync(0xffffffffu, before, o);
        if (lane >= o) before += v;
      }
      const unsigned live = __ballot_sync(0xffffffffu, c > 0);
      if (c > 0) {
        const int i = n + __popc(live & ((1u << lane) - 1u));
        plan.expert[i] = e;
        plan.start[i] = at + before - c;
      }
      n += __popc(live);
      at += __shfl_sync(0xffffffffu, before, 31);
    }
    if (lane == 0) {
      *plan.active = n;
      plan.start[n] = at;
    }
  }
  __syncthreads();
  const int active = *plan.active;
  for (int i = threadIdx.x; i < active; i += kMoeThreads) {
    int at = plan.start[i];
    for (int p = 0; p < pairs; ++p)
      if (ids[p] == plan.expert[i]) plan.order[at++] = p;
  }
  __syncthreads();
  if (blockIdx.x == 0) {
    for (int i = threadIdx.x; i < MoePlan::words(a.experts, pairs); i += kMoeThreads) a.plan[i] = reinterpret_cast<int*>(smem)[i];
    for (int p = threadIdx.x; p < pairs; p += kMoeThreads) {
      if (a.ids) a.ids[p] = ids[p];
      if (a.gates) a.gates[p] = plan.gate[p];
    }
  }

  // units: expert, 16 rows, group of eight tokens
  const int blocks = (a.f + 15) / 16;
  int total = 0;
  for (int i = 0; i < active; ++i) total += blocks * ((plan.start[i + 1] - plan.start[i] + 7) / 8);
  const int begin = (int)((long long)total * blockIdx.x / gridDim.x), end = (int)((long long)total * (blockIdx.x + 1) / gridDim.x);
  struct Unit {
    int index, rows, group, groups, left;  // expert (of the active ones), row block, group of tokens; units left of the expert
  };
  Unit unit{0, 0, 0, 0, 0};
  {
    int at = 0;
    for (; unit.index < active; ++unit.index) {
      const int g = (plan.start[unit.index + 1] - plan.start[unit.index] + 7) / 8;
      if (begin < at + blocks * g) {
        unit.groups = g;
        unit.rows = (begin - at) / g;
        unit.group = (begin - at) % g;
        break;
      }
      at += blocks * g;
    }
  }
  auto advance = [&](Unit& u) {
    if (++u.group < u.groups) return;
    u.group = 0;
    if (++u.rows < blocks) return;
    u.rows = 0;
    if (++u.index < active) u.groups = (plan.start[u.index + 1] - plan.start[u.index] + 7) / 8;
  };

  using Stream = typename std::conditional<W4, Rows4<T, T>, Rows16<T>>::type;
  constexpr int kStep = Stream::kStep;
  const int steps = (a.d + kStep - 1) / kStep, s0 = steps * warp / kMoeWarps, s1 = steps * (warp + 1) / kMoeWarps;
  const bool vec = !W4 && a.ldg % 8 == 0 && a.strideG % 8 == 0 && a.d % 8 == 0 &&
                   ((reinterpret_cast<uintptr_t>(a.gate) | reinterpret_cast<uintptr_t>(a.up)) & 15u) == 0;
  const int k_tiles = (a.d + 127) / 128;
  auto load = [&](Stream& g, Stream& u, const Unit& at, int step) {
    const size_t e = plan.expert[at.index];
    if constexpr (W4) {
      const size_t off = e * a.strideG + ((size_t)at.rows * k_tiles + step) * a.fmt.tile_bytes();
      g.load(static_cast<const unsigned char*>(a.gate) + off, a.fmt);
      u.load(static_cast<const unsigned char*>(a.up) + off, a.fmt);
    } else {
      const size_t off = e * a.strideG + (size_t)at.rows * 16 * a.ldg;
      g.load(static_cast<const T*>(a.gate) + off, a.ldg, a.f - at.rows * 16, a.d, step, vec);
      u.load(static_cast<const T*>(a.up) + off, a.ldg, a.f - at.rows * 16, a.d, step, vec);
    }
  };
  // one step ahead, across units
  Stream gate[2], up[2];
  if (begin < end && s0 < s1) load(gate[0], up[0], unit, s0);
  int cur = 0;
  for (int n = begin; n < end; ++n) {
    Unit next = unit;
    advance(next);
    const int p0 = plan.start[unit.index] + unit.group * 8, cols = min(8, plan.start[unit.index + 1] - p0);
    const T* x = static_cast<const T*>(a.x) + (size_t)(plan.order[p0 + min(r, cols - 1)] / a.topk) * a.d_pad + t * 8;
    float accg[4] = {0.f, 0.f, 0.f, 0.f}, accu[4] = {0.f, 0.f, 0.f, 0.f};
    for (int s = s0; s < s1; ++s) {
      const bool more = s + 1 < s1;
      auto body = [&](Stream& g0, Stream& u0, Stream& g1, Stream& u1) {
        if (more) load(g1, u1, unit, s + 1);
        else if (n + 1 < end) load(g1, u1, next, s0);
        if constexpr (W4) {
          uint4 b[1][4];
#pragma unroll
          for (int q = 0; q < 4; ++q) b[0][q] = *reinterpret_cast<const uint4*>(x + s * 128 + q * 32);
          g0.multiply(accg, b, a.fmt);
          u0.multiply(accu, b, a.fmt);
        } else {
          uint4 b[2];
#pragma unroll
          for (int q = 0; q < 2; ++q) b[q] = *reinterpret_cast<const uint4*>(x + s * 64 + q * 32);
          g0.multiply(accg, b);
          u0.multiply(accu, b);
        }
      };
      if (cur == 0) body(gate[0], up[0], gate[1], up[1]);
      else body(gate[1], up[1], gate[0], up[0]);
      cur ^= 1;
    }
    // [warp][gate, up][column][row]
    float* mine = sums + ((n & 1) * kMoeWarps + warp) * 256;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const int at = (t * 2 + (i & 1)) * 16 + r + 8 * (i >> 1);
      mine[at] = accg[i];
      mine[128 + at] = accu[i];
    }
    __syncthreads();
    // finished by four warps, others' turn with every unit
    const int i = (int)((threadIdx.x + 384 * (n & 3)) & (kMoeThreads - 1));
    if (i < cols * 16) {
      const float* p = sums + (n & 1) * kMoeWarps * 256 + i;
      float g = 0.f, u = 0.f;
#pragma unroll
      for (int w = 0; w < kMoeWarps; ++w) {
        g += p[w * 256];
        u += p[w * 256 + 128];
      }
      const int row = unit.rows * 16 + (i & 15), pair = plan.order[p0 + i / 16];
      const float h = row < a.f ? g / (1.f + expf(-g)) * u : 0.f;
      if (W4 || !std::is_same<T, __half>::value) {
        __nv_bfloat16* out = static_cast<__nv_bfloat16*>(a.hidden) + (size_t)pair * 2 * a.f_pad + row;
        const __nv_bfloat16 v = __float2bfloat16_rn(h);
        out[0] = v;
        out[a.f_pad] = __float2bfloat16_rn(isfinite(h) ? h - __bfloat162float(v) : 0.f);
      } else {
        static_cast<float*>(a.hidden)[(size_t)pair * a.f_pad + row] = h;
        uint32_t top = __float_as_uint(fabsf(h));  // sixteen lanes hold the rows of a pair
        const unsigned lanes = 0xffffu << (lane & 16);
#pragma unroll
        for (int o = 1; o < 16; o <<= 1) top = max(top, __shfl_xor_sync(lanes, top, o));
        if ((lane & 15) == 0) atomicMax(&a.peak[pair], top);
      }
    }
    unit = next;
  }
}

// ---------------------------------------------------------------- down ----------------
template <typename T, bool W4>
__global__ void __launch_bounds__(kMoeThreads, 1) moe_down_kernel(const MoeArgs a) {
  extern __shared__ __align__(16) unsigned char smem[];
  const int warp = threadIdx.x / 32, lane = threadIdx.x & 31, r = lane >> 2, t = lane & 3;
  const int pairs = a.tokens * a.topk, words = MoePlan::words(a.experts, pairs);
  MoePlan plan(reinterpret_cast<int*>(smem), a.experts, pairs);
  float* sums = reinterpret_cast<float*>(smem + ((size_t)words * 4 + 15) / 16 * 16);  // [warp][token][row]
  griddep_launch_dependents();
  griddep_wait();
  for (int i = threadIdx.x; i < words; i += kMoeThreads) reinterpret_cast<int*>(smem)[i] = a.plan[i];
  __syncthreads();
  const int active = *plan.active;

  using U = typename std::conditional<W4, __nv_bfloat16, T>::type;  // type of the products
  using Stream = typename std::conditional<W4, Rows4<T, U>, Rows16<T>>::type;
  constexpr int kStep = Stream::kStep;
  constexpr bool kScaled = !W4 && std::is_same<T, __half>::value;  // hidden vectors as floats, scaled here into half precision
  const int steps = (a.f + kStep - 1) / kStep, k_tiles = (a.f + 127) / 128;
  int total = 0;
  for (int i = 0; i < active; ++i) total += (plan.start[i + 1] - plan.start[i] + 7) / 8;
  const long long all = (long long)total * steps;
  const long long w0 = all * warp / kMoeWarps, w1 = all * (warp + 1) / kMoeWarps;
  const bool vec = !W4 && a.ldd % 8 == 0 && a.strideD % 8 == 0 && a.f % 8 == 0 &&
                   (reinterpret_cast<uintptr_t>(a.down) & 15u) == 0;
  struct Place {
    int index, group, groups, step;
  };
  Place first{0, 0, 0, 0};
  {
    long long at = 0;
    for (; first.index < active; ++first.index) {
      first.groups = (plan.start[first.index + 1] - plan.start[first.index] + 7) / 8;
      if (w0 < at + (long long)first.groups * steps) {
        first.group = (int)((w0 - at) / steps);
        first.step = (int)((w0 - at) % steps);
        break;
      }
      at += (long long)first.groups * steps;
    }
  }
  auto advance = [&](Place& p) {
    if (++p.step < steps) return;
    p.step = 0;
    if (++p.group < p.groups) return;
    p.group = 0;
    if (++p.index < active) p.groups = (plan.start[p.index + 1] - plan.start[p.index] + 7) / 8;
  };
  auto load = [&](Stream& s, int rows, const Place& p) {
    const size_t e = plan.expert[p.index];
    if constexpr (W4)
      s.load(static_cast<const unsigned char*>(a.down) + e * a.strideD + ((size_t)rows * k_tiles + p.step) * a.fmt.tile_bytes(),
             a.fmt);
    else
      s.load(static_cast<const T*>(a.down) + e * a.strideD + (size_t)rows * 16 * a.ldd, a.ldd, a.d - rows * 16, a.f, p.step, vec);
  };

  const int row_blocks = (a.d + 15) / 16;
  for (int rows = blockIdx.x; rows < row_blocks; rows += gridDim.x) {
    for (int i = threadIdx.x; i < kMoeWarps * a.tokens * 16; i += kMoeThreads) sums[i] = 0.f;
    __syncthreads();
    Place place = first;
    Stream w[2];
    if (w0 < w1) load(w[0], rows, place);
    int cur = 0;
    float acc[4] = {0.f, 0.f, 0.f, 0.f};
    for (long long n = w0; n < w1; ++n) {
      Place next = place;
      advance(next);
      const int p0 = plan.start[place.index] + place.group * 8, cols = min(8, plan.start[place.index + 1] - p0);
      const int pair = plan.order[p0 + min(r, cols - 1)];
      auto body = [&](Stream& now, Stream& then) {
        if (n + 1 < w1) load(then, rows, next);
        if constexpr (W4) {
          const __nv_bfloat16* h = static_cast<const __nv_bfloat16*>(a.hidden) + (size_t)pair * 2 * a.f_pad + place.step * 128 + t * 8;
          uint4 b[2][4];
#pragma unroll
          for (int i = 0; i < 2; ++i)
#pragma unroll
            for (int q = 0; q < 4; ++q) b[i][q] = *reinterpret_cast<const uint4*>(h + (size_t)i * a.f_pad + q * 32);
          now.multiply(acc, b, a.fmt);
        } else if constexpr (!kScaled) {
          const T* h = static_cast<const T*>(a.hidden) + (size_t)pair * 2 * a.f_pad + place.step * 64 + t * 8;
#pragma unroll
          for (int i = 0; i < 2; ++i) {
            uint4 b[2];
#pragma unroll
            for (int q = 0; q < 2; ++q) b[q] = *reinterpret_cast<const uint4*>(h + (size_t)i * a.f_pad + q * 32);
            now.multiply(acc, b);
          }
        } else {
          const float* h = static_cast<const float*>(a.hidden) + (size_t)pair * a.f_pad + place.step * 64 + t * 8;
          const float up = moe_scale(a.peak[pair]);
          uint4 hi[2], lo[2];
#pragma unroll
          for (int q = 0; q < 2; ++q) {
            const float4 u = *reinterpret_cast<const float4*>(h + q * 32), v = *reinterpret_cast<const float4*>(h + q * 32 + 4);
            const float e[8] = {u.x * up, u.y * up, u.z * up, u.w * up, v.x * up, v.y * up, v.z * up, v.w * up};
            uint32_t* ph = &hi[q].x;
            uint32_t* pl = &lo[q].x;
#pragma unroll
            for (int i = 0; i < 4; ++i) {
              const __half2 c = __floats2half2_rn(e[2 * i], e[2 * i + 1]);
              const float2 back = __half22float2(c);
              const __half2 d = __floats2half2_rn(e[2 * i] - back.x, e[2 * i + 1] - back.y);
              ph[i] = *reinterpret_cast<const uint32_t*>(&c);
              pl[i] = *reinterpret_cast<const uint32_t*>(&d);
            }
          }
          now.multiply(acc, hi);
          now.multiply(acc, lo);
        }
      };
      if (cur == 0) body(w[0], w[1]);
      else body(w[1], w[0]);
      cur ^= 1;
      if (next.step == 0 || n + 1 == w1) {  // the expert's tokens are finished (as far as this warp goes)
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const int col = t * 2 + (i & 1);
          if (col < cols) {
            const int p = plan.order[p0 + col];
            float v = acc[i];
            if (kScaled) v /= moe_scale(a.peak[p]);
            sums[(warp * a.tokens + p / a.topk) * 16 + r + 8 * (i >> 1)] += plan.gate[p] * v;
          }
          acc[i] = 0.f;
        }
        __syncwarp();
      }
      place = next;
    }
    __syncthreads();
    for (int i = threadIdx.x; i < a.tokens * 16; i += kMoeThreads) {
      float v = 0.f;
#pragma unroll
      for (int w2 = 0; w2 < kMoeWarps; ++w2) v += sums[w2 * a.tokens * 16 + i];
      const int row = rows * 16 + (i & 15);
      if (row < a.d) {
        T* y = static_cast<T*>(a.Y) + (size_t)(i / 16) * a.ldy + row;
        *y = from_f32<T>(a.beta != 0.f ? fmaf(a.beta, to_f32(*y), v) : v);
      }
    }
    __syncthreads();
  }
}

}  // namespace mmbo
