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
//   scores   one warp per (token, expert); also an aligned, zero-padded copy of the activations (for 4-bit experts in half
//            precision with the groups' sums, as w4_tile_mma wants them)
//   up       every block repeats the selection for itself (a microsecond, cheaper than another kernel and its launch), then
//            teams of 4, 8 or 16 warps work through their shares of the units (expert, 16 rows of gate and up) and split d
//   down     a block owns 16 rows of the output for all tokens, its warps split the list of (expert, part of f); the sums
//            of the experts meet in shared memory in a fixed order
// Each warp has a ring in shared memory that its lanes fill with 16-byte asynchronous copies of weights, every lane with
// the pieces that it will itself read as fragments of mma.sync.m16n8k16, so the ring needs no barrier and the copies in
// flight no registers; the columns come straight from L2, the same 16 bytes' worth of k of a lane's token, asked for
// before the wait for the weights.  (Weights loaded straight to registers one step ahead left 64 KB in flight an SM at
// best: 255 us for the batch of 48 tokens in `up`, 2.9 TB/s.)  Tokens are the eight columns of the instruction; an expert with more tokens is taken in groups of
// eight, the later ones finding its weights in L2.
#pragma once

#include "w4_umma.cuh"

namespace mmbo {

constexpr int kMoeWarps = 16, kMoeThreads = kMoeWarps * 32;
// Tokens of one pass (more are taken in several): what the plan and the sums of `down` leave room for in shared memory.
__host__ __device__ constexpr int moe_pass_tokens(int topk) { return 512 / topk < 64 ? 512 / topk : 64; }

struct MoeArgs {
  int tokens, d, f, experts, topk, renorm;
  W4Format fmt;  // 4-bit experts; group 0: 16-bit ones
  const void *X, *router, *gate, *up, *down;
  size_t ldx, ldr, ldg, strideG, ldd, strideD;  // strides in elements, for packed experts in bytes
  float beta;
  int team_log2;  // warps of a team of `up`
  void* Y;
  size_t ldy;
  int* ids;      // tokens x topk, the caller's or null
  float* gates;  // tokens x topk, the caller's or null
  // workspace
  float* scores;    // tokens x experts
  void* x;          // tokens x d_pad: the activations, zero behind d (4-bit experts: in half precision, scaled)
  float* x_sums;    // 4-bit experts: tokens x (d_pad / group) sums of these, in units of 2^20
  float2* x_undo;   // 4-bit experts: two factors a token that undo its scale and the unit of 2^20
  void* hidden;     // pairs x 2 x f_pad, zero behind f: hidden vectors as a 16-bit value and what its rounding left, see MoeHidden
  int* plan;        // what `up` found out for `down`, see MoePlan
  int d_pad, f_pad; // multiples of 128
};

// The selection, sorted by expert: `order` holds the pairs (token * topk + slot, and the token again in the upper half: a
// division saved wherever a column is looked up) of expert 0's tokens, then expert 1's ..;
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
  __shared__ uint32_t peak;
  griddep_launch_dependents();
  if (threadIdx.x == 0) peak = 0;
  __syncthreads();
  griddep_wait();
  const int t = blockIdx.y, lane = threadIdx.x & 31;
  const T* x = static_cast<const T*>(a.X) + (size_t)t * a.ldx;
  if (blockIdx.x == gridDim.x - 1) {  // the last block of a token prepares the workspace instead
    uint16_t* h = static_cast<uint16_t*>(a.hidden) + (size_t)t * a.topk * a.f_pad * 2;
    const int pad = a.f_pad - a.f;
    for (int i = threadIdx.x; i < a.topk * 2 * pad; i += 256) h[(size_t)(i / pad) * a.f_pad + a.f + i % pad] = 0;
    if (!a.fmt.group) {
      T* copy = static_cast<T*>(a.x) + (size_t)t * a.d_pad;
      for (int j = threadIdx.x * 8; j < a.d_pad; j += 256 * 8) *reinterpret_cast<uint4*>(copy + j) = load8(x, a.d, j);
      return;
    }
    float f1 = 1.f, f2 = 1.f;
    if (!std::is_same<T, __half>::value) {
      // exponent of the largest magnitude (below the normal range: the smallest normal one), 2^(14 - e) as a product
      uint32_t top = 0;
      for (int j = threadIdx.x * 8; j < a.d; j += 256 * 8) {
        const uint4 v = load8(x, a.d, j);
        const uint32_t w[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
        for (int i = 0; i < 4; ++i) top = max(top, max(w[i] << 16 & 0x7fffffffu, w[i] & 0x7fff0000u));
      }
      top = __reduce_max_sync(0xffffffffu, top);
      if (lane == 0) atomicMax(&peak, top);
      __syncthreads();
      const int up = 14 - ((int)max(peak >> 23, 1u) - 127), up1 = min(max(up, -100), 100), up2 = up - up1;
      f1 = __uint_as_float((uint32_t)(up1 + 127) << 23);
      f2 = __uint_as_float((uint32_t)(up2 + 127) << 23);
      if (threadIdx.x == 0)
        a.x_undo[t] = peak < 0x7f800000u ? make_float2(__uint_as_float((uint32_t)(127 - up1) << 23),
                                                       __uint_as_float((uint32_t)(127 - up2 + 20) << 23))
                                         : make_float2(__int_as_float(0x7fc00000), 0.f);
    } else if (threadIdx.x == 0) {
      a.x_undo[t] = make_float2(1.f, 0x1p20f);
    }
    __half* copy = static_cast<__half*>(a.x) + (size_t)t * a.d_pad;
    const int lanes = a.fmt.group / 8;  // neighbouring threads that hold a group
    for (int j0 = 0; j0 < a.d_pad; j0 += 256 * 8) {
      const int j = j0 + threadIdx.x * 8;
      const uint4 v = load8(x, a.d, j);
      const uint32_t w[4] = {v.x, v.y, v.z, v.w};
      uint32_t out[4];
      float sum = 0.f;
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const float2 e = widen2<T>(w[i]);
        const __half2 c = __floats2half2_rn(e.x * f1 * f2, e.y * f1 * f2);
        out[i] = *reinterpret_cast<const uint32_t*>(&c);
        const float2 back = __half22float2(c);
        sum += back.x + back.y;
      }
      for (int o = 1; o < lanes; o <<= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
      if (j < a.d_pad) {
        *reinterpret_cast<uint4*>(copy + j) = make_uint4(out[0], out[1], out[2], out[3]);
        if (threadIdx.x % lanes == 0) a.x_sums[(size_t)t * (a.d_pad / a.fmt.group) + j / a.fmt.group] = sum * 0x1p-20f;
      }
    }
    return;
  }
  const int e = blockIdx.x * 8 + threadIdx.x / 32;
  if (e >= a.experts) return;
  const T* w = static_cast<const T*>(a.router) + (size_t)e * a.ldr;
  float sum = 0.f;
  auto dot = [&](const uint4& u, const uint4& v) {
    const uint32_t uw[4] = {u.x, u.y, u.z, u.w}, vw[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const float2 p = widen2<T>(uw[i]), q = widen2<T>(vw[i]);
      sum = fmaf(p.x, q.x, sum);
      sum = fmaf(p.y, q.y, sum);
    }
  };
  if (a.d % 8 == 0 && ((reinterpret_cast<uintptr_t>(w) | reinterpret_cast<uintptr_t>(x)) & 15u) == 0) {
    for (int j = lane * 8; j < a.d; j += 8 * 256) {  // eight pieces of each under way at a time
      uint4 u[8], v[8];
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        const bool have = j + i * 256 < a.d;
        u[i] = have ? *reinterpret_cast<const uint4*>(w + j + i * 256) : make_uint4(0, 0, 0, 0);
        v[i] = have ? *reinterpret_cast<const uint4*>(x + j + i * 256) : make_uint4(0, 0, 0, 0);
      }
#pragma unroll
      for (int i = 0; i < 8; ++i) dot(u[i], v[i]);
    }
  } else {
    for (int j = lane * 8; j < a.d; j += 256) dot(load8(w, a.d, j), load8(x, a.d, j));
  }
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
  if (lane == 0) a.scores[(size_t)t * a.experts + e] = sum;
}

// The topk experts of one token by one warp: ids and gates (shared memory); `scores`: room for the experts' scores in
// shared memory (read once from memory: each of the topk rounds would wait for it again).
__device__ __forceinline__ void moe_select(const MoeArgs& a, const float* from, float* scores, int* ids, float* gates) {
  const int lane = threadIdx.x & 31;
  for (int e = lane; e < a.experts; e += 32) scores[e] = from[e];
  __syncwarp();
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

// ---------------------------------------------------------------- rings ---------------
// 16 bytes to shared memory, in the background; zeros where `have` is false.
__device__ __forceinline__ void copy16(uint32_t dst, const void* src, bool have) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst), "l"(src), "r"(have ? 16 : 0) : "memory");
}
__device__ __forceinline__ void copy16(uint32_t dst, const void* src) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(dst), "l"(src) : "memory");
}
__device__ __forceinline__ void copies_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
// Waits until at most N of the groups committed are under way.
template <int N>
__device__ __forceinline__ void copies_wait() {
  asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory");
}
__device__ __forceinline__ void sts128(uint32_t addr, const uint4& v) {
  asm volatile("st.shared.v4.u32 [%0], {%1, %2, %3, %4};" ::"r"(addr), "r"(v.x), "r"(v.y), "r"(v.z), "r"(v.w) : "memory");
}

// Feeds a ring with sixteen rows of 16-bit weights, 32 C columns at a time: piece (h, u) of a lane, columns 32 u + 8 t ..
// + 7 of row r + 8 h, goes to (h C + u) * 512 + lane * 16.  Rows that do not exist and columns behind k come as zeros.
template <typename T, int C>
struct RowsFeed {
  const T *lo, *hi;  // this lane's place in rows r and r + 8
  int j, k;          // its column; a row's length
  bool have_lo, have_hi, vec, plain;  // plain: everything is there and aligned
  __device__ __forceinline__ void start(const T* base, size_t ld, int rows, int k_, int step, bool vec_) {
    const int lane = threadIdx.x & 31, r = lane >> 2;
    have_lo = r < rows;
    have_hi = r + 8 < rows;
    j = step * 32 * C + (lane & 3) * 8;
    k = k_;
    vec = vec_;
    plain = vec && rows >= 16 && k % (32 * C) == 0;
    lo = base + (have_lo ? r * ld : 0) + j;
    hi = base + (have_hi ? (r + 8) * ld : 0) + j;
  }
  __device__ __forceinline__ void fetch(uint32_t to) {
    to += (threadIdx.x & 31) * 16;
    if (plain) {
#pragma unroll
      for (int u = 0; u < C; ++u) {
        copy16(to + u * 512, lo + 32 * u);
        copy16(to + (C + u) * 512, hi + 32 * u);
      }
    } else {
#pragma unroll 1
      for (int u = 0; u < C; ++u) {
        const bool in = j + 32 * u < k;
        if (vec) {
          copy16(to + u * 512, in ? lo + 32 * u : lo - j, in && have_lo);
          copy16(to + (C + u) * 512, in ? hi + 32 * u : hi - j, in && have_hi);
        } else {
          sts128(to + u * 512, load8(lo - j, have_lo ? k : 0, j + 32 * u));
          sts128(to + (C + u) * 512, load8(hi - j, have_hi ? k : 0, j + 32 * u));
        }
      }
      j += 32 * C;
    }
    lo += 32 * C;
    hi += 32 * C;
  }
};
// acc += those weights * columns; b: this lane's 16 bytes of each 32 columns
template <typename T, int C>
__device__ __forceinline__ void rows16_multiply(uint32_t from, float (&acc)[4], const uint4 (&b)[C]) {
  const uint32_t at = from + (threadIdx.x & 31) * 16;
#pragma unroll
  for (int u = 0; u < C; ++u) {
    const uint4 lo = lds128(at + u * 512), hi = lds128(at + (C + u) * 512);
    mma_16816<T>(acc, lo.x, hi.x, lo.y, hi.y, b[u].x, b[u].y);
    mma_16816<T>(acc, lo.z, hi.z, lo.w, hi.w, b[u].z, b[u].w);
  }
}

// The same with packed tiles, in their own layout: two pieces of codes a lane, scales and zero points by the lanes from
// `first` on.  (Others read what a lane copied: __syncwarp() behind the wait.)
struct TileFeed {
  const unsigned char *codes, *scales;
  uint32_t piece, scale_piece, bytes;
  bool has_scale;
  __device__ __forceinline__ void start(const unsigned char* tile, uint32_t tile_bytes, int first) {
    const int lane = threadIdx.x & 31, i = lane - first;
    bytes = tile_bytes;
    piece = w4_piece(lane >> 2, lane & 3);
    has_scale = i >= 0 && i * 16 < (int)tile_bytes - kW4Codes;
    scale_piece = kW4Codes + (has_scale ? i * 16 : 0);
    codes = tile + piece;
    scales = tile + scale_piece;
  }
  __device__ __forceinline__ void fetch(uint32_t to) {
    copy16(to + piece, codes);
    copy16(to + piece + 512, codes + 512);
    if (has_scale) copy16(to + scale_piece, scales);
    codes += bytes;
    scales += bytes;
  }
};
// acc += a packed tile * two bfloat16 columns' worth (a value and its remainder, by quarters).  Codes become exact integers:
// for w4_tile_mma a hidden vector would first have to be brought to half precision.
template <typename T, int QG>
__device__ __forceinline__ void tile_multiply_bf16(uint32_t tile, const uint4 (&b)[2][4], bool zeros, float (&acc)[4]) {
  using L = W4Tile<QG, true>;
  const int lane = threadIdx.x & 31, r = lane >> 2;
  const uint32_t codes = tile + w4_piece(r, lane & 3);
  const uint4 c0 = lds128(codes), c1 = lds128(codes + 512);
  const uint32_t w0[4] = {c0.x, c0.y, c0.z, c0.w}, w1[4] = {c1.x, c1.y, c1.z, c1.w};
  W4Unpacker<__nv_bfloat16> lo, hi;
#pragma unroll
  for (int g = 0; g < L::kGroups; ++g) {
    const uint32_t z = zeros ? lds16(tile + L::kZeros + g * 16 + r * 2) : 0x0808u;
    lo.set_zero(z & 15u);
    hi.set_zero(z >> 8 & 15u);
    float part[2][4] = {{0.f, 0.f, 0.f, 0.f}, {0.f, 0.f, 0.f, 0.f}};
#pragma unroll
    for (int qq = 0; qq < QG; ++qq) {
      const int q = g * QG + qq;
      uint32_t p[4], s[4];
      lo.unpack(w0[q], p);
      hi.unpack(w1[q], s);
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        mma_16816<__nv_bfloat16>(part[i], p[0], s[0], p[1], s[1], b[i][q].x, b[i][q].y);
        mma_16816<__nv_bfloat16>(part[i], p[2], s[2], p[3], s[3], b[i][q].z, b[i][q].w);
      }
    }
    const float2 s = widen2<T>(lds32(tile + L::kScales + g * 32 + r * 4));
#pragma unroll
    for (int i = 0; i < 4; ++i) acc[i] = fmaf(i < 2 ? s.x : s.y, part[0][i] + part[1][i], acc[i]);
  }
}
constexpr uint32_t kTileRoom = kW4Codes + 4 * 48;  // of a tile in a ring, whatever its groups

// Hidden vectors as products take them: a 16-bit value and what its rounding left, so that 16 bits and more survive.
// bfloat16 has the range of a float.  Half precision holds h / 64 and 2^11 times the remainder: magnitudes up to 4.19e6,
// steps of 2^-30 near zero (results in half precision have steps of 2^-24).
template <typename U>
struct MoeHidden;
template <>
struct MoeHidden<__nv_bfloat16> {
  static constexpr float kScale = 1.f, kRest = 1.f;
};
template <>
struct MoeHidden<__half> {
  static constexpr float kScale = 0x1p-6f, kRest = 0x1p11f;
};

// ---------------------------------------------------------------- up ------------------
// QG: quarters of a group of packed weights, 0: 16-bit weights.
template <int QG>
struct MoeUpShape {
  static constexpr int kStep = QG ? 128 : 64;  // columns: whole 128-byte lines of 16-bit rows
  static constexpr uint32_t kSlot = QG ? kTileRoom : 2048;  // gate and up take turns
  static constexpr int kSlots = QG ? 8 : 5;
};
constexpr size_t kMoeUpSums = (size_t)2 * kMoeWarps * 256 * 4;

template <typename T, int QG>
__global__ void __launch_bounds__(kMoeThreads, 1) moe_up_kernel(const MoeArgs a) {
  using S = MoeUpShape<QG>;
  constexpr bool W4 = QG > 0;
  extern __shared__ __align__(128) unsigned char smem[];
  const int warp = threadIdx.x / 32, lane = threadIdx.x & 31, r = lane >> 2, t = lane & 3;
  const int pairs = a.tokens * a.topk;
  // shared memory: rings | partial sums (before that: scores) | plan | ids | count
  const uint32_t ring = smem_u32(smem) + warp * S::kSlots * S::kSlot;
  float* sums = reinterpret_cast<float*>(smem + kMoeWarps * S::kSlots * S::kSlot);
  int* at_plan = reinterpret_cast<int*>(sums) + kMoeUpSums / 4;
  MoePlan plan(at_plan, a.experts, pairs);
  int* ids = at_plan + MoePlan::words(a.experts, pairs);
  int* count = ids + pairs;  // experts
  griddep_launch_dependents();
  for (int e = threadIdx.x; e < a.experts; e += kMoeThreads) count[e] = 0;
  griddep_wait();

  // the selection, by every block for itself
  const int selecting = min(kMoeWarps, (int)(kMoeUpSums / 4) / a.experts);  // warps that have room for a token's scores
  for (int tok = warp; warp < selecting && tok < a.tokens; tok += selecting)
    moe_select(a, a.scores + (size_t)tok * a.experts, sums + warp * a.experts, ids + tok * a.topk, plan.gate + tok * a.topk);
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
      if (ids[p] == plan.expert[i]) plan.order[at++] = p | (p / a.topk) << 16;
  }
  __syncthreads();
  if (blockIdx.x == 0) {
    for (int i = threadIdx.x; i < MoePlan::words(a.experts, pairs); i += kMoeThreads) a.plan[i] = at_plan[i];
    for (int p = threadIdx.x; p < pairs; p += kMoeThreads) {
      if (a.ids) a.ids[p] = ids[p];
      if (a.gates) a.gates[p] = plan.gate[p];
    }
  }

  // units: expert, 16 rows, group of eight tokens; a team of warps shares a unit and cuts d
  const int WK = 1 << a.team_log2, wk = warp & (WK - 1), team = warp >> a.team_log2, teams = kMoeWarps >> a.team_log2;
  const int blocks = (a.f + 15) / 16;
  int total = 0;
  for (int i = 0; i < active; ++i) total += blocks * ((plan.start[i + 1] - plan.start[i] + 7) / 8);
  const long long share = (long long)gridDim.x * teams, mine = (long long)blockIdx.x * teams + team;
  const int begin = (int)(total * mine / share), end = (int)(total * (mine + 1) / share);
  struct Unit {
    int index, rows, group, groups;  // expert (of the active ones), row block, group of tokens
  };
  Unit unit{0, 0, 0, 0};
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

  const int steps = (a.d + S::kStep - 1) / S::kStep, s0 = steps * wk >> a.team_log2, s1 = steps * (wk + 1) >> a.team_log2;
  const bool vec = !W4 && a.ldg % 8 == 0 && a.strideG % 8 == 0 && a.d % 8 == 0 &&
                   ((reinterpret_cast<uintptr_t>(a.gate) | reinterpret_cast<uintptr_t>(a.up)) & 15u) == 0;
  const uint32_t tile_bytes = W4 ? a.fmt.tile_bytes() : 0;
  // the copies run ahead of the products, through the same order
  using Feed = typename std::conditional<W4, TileFeed, RowsFeed<T, 2>>::type;
  Feed gate, up;
  Unit ahead = unit;
  int ahead_n = s0 < s1 ? begin : end, ahead_left = s1 - s0;
  uint32_t ahead_at = ring;
  auto start = [&]() {
    if (ahead_n >= end) return;
    const size_t e = plan.expert[ahead.index];
    if constexpr (W4) {
      const size_t off = e * a.strideG + ((size_t)ahead.rows * steps + s0) * tile_bytes;
      gate.start(static_cast<const unsigned char*>(a.gate) + off, tile_bytes, 0);
      up.start(static_cast<const unsigned char*>(a.up) + off, tile_bytes, 0);
    } else {
      const size_t off = e * a.strideG + (size_t)ahead.rows * 16 * a.ldg;
      gate.start(static_cast<const T*>(a.gate) + off, a.ldg, a.f - ahead.rows * 16, a.d, s0, vec);
      up.start(static_cast<const T*>(a.up) + off, a.ldg, a.f - ahead.rows * 16, a.d, s0, vec);
    }
  };
  int turn = 0;  // gate's or up's
  auto fetch = [&]() {
    if (ahead_n < end) {
      if (turn == 0) gate.fetch(ahead_at);
      else up.fetch(ahead_at);
      ahead_at += S::kSlot;
      if (ahead_at == ring + S::kSlots * S::kSlot) ahead_at = ring;
      turn ^= 1;
      if (turn == 0 && --ahead_left == 0) {
        ahead_left = s1 - s0;
        if (++ahead_n < end) advance(ahead);
        start();
      }
    }
    copies_commit();
  };
  start();
  for (int i = 0; i + 1 < S::kSlots; ++i) fetch();

  uint32_t from = ring;
  for (int n = begin; n < end; ++n) {
    const int p0 = plan.start[unit.index] + unit.group * 8, cols = min(8, plan.start[unit.index + 1] - p0);
    // columns past the last token repeat it; their sums are not used
    const uint16_t* x = static_cast<const uint16_t*>(a.x) + (size_t)(plan.order[p0 + min(r, cols - 1)] >> 16) * a.d_pad +
                        s0 * S::kStep + t * 8;
    const float *sums0 = nullptr, *sums1 = nullptr;
    if constexpr (W4) {
      const int per = a.d_pad / (32 * QG), at = s0 * (4 / QG);
      sums0 = a.x_sums + (size_t)(plan.order[p0 + min(2 * t, cols - 1)] >> 16) * per + at;
      sums1 = a.x_sums + (size_t)(plan.order[p0 + min(2 * t + 1, cols - 1)] >> 16) * per + at;
    }
    float accg[4] = {0.f, 0.f, 0.f, 0.f}, accu[4] = {0.f, 0.f, 0.f, 0.f};
    for (int s = s0; s < s1; ++s) {
      constexpr int kQuarters = S::kStep / 32;
      uint4 b[kQuarters];
#pragma unroll
      for (int q = 0; q < kQuarters; ++q) b[q] = *reinterpret_cast<const uint4*>(x + q * 32);
      x += S::kStep;
      float2 xs[W4 ? 4 / (QG ? QG : 1) : 1];
      if constexpr (W4) {
#pragma unroll
        for (int g = 0; g < 4 / QG; ++g) xs[g] = make_float2(*sums0++, *sums1++);
      }
#pragma unroll
      for (int half = 0; half < 2; ++half) {
        __syncwarp();
        fetch();
        copies_wait<S::kSlots - 1>();
        if constexpr (W4) {
          __syncwarp();
          w4_tile_mma<T, QG>(from, [&](int q) { return b[q]; }, [&](int g) { return xs[g]; }, a.fmt.zeros, half ? accu : accg);
        } else {
          rows16_multiply<T, 2>(from, half ? accu : accg, b);
        }
        from += S::kSlot;
        if (from == ring + S::kSlots * S::kSlot) from = ring;
      }
    }
    // [turn][warp][gate, up][column][row]
    float* ours = sums + ((n & 1) * kMoeWarps + (team << a.team_log2)) * 256;
    float* mine_sums = ours + wk * 256;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const int at = (t * 2 + (i & 1)) * 16 + r + 8 * (i >> 1);
      mine_sums[at] = accg[i];
      mine_sums[128 + at] = accu[i];
    }
    asm volatile("bar.sync %0, %1;" ::"r"(1 + team), "r"(WK * 32) : "memory");
    // finished by four warps, with larger teams others' turn with every unit
    const int i = (wk * 32 + lane + 384 * (n & 3)) & (WK * 32 - 1);
    if (i < cols * 16) {
      const float* p = ours + i;
      float g = 0.f, u = 0.f;
      for (int w = 0; w < WK; w += 4) {
#pragma unroll
        for (int v = 0; v < 4; ++v) {
          g += p[(w + v) * 256];
          u += p[(w + v) * 256 + 128];
        }
      }
      const int row = unit.rows * 16 + (i & 15), entry = plan.order[p0 + i / 16], pair = entry & 0xffff;
      if (W4) {
        const float2 undo = a.x_undo[entry >> 16];
        g *= undo.x * undo.y;
        u *= undo.x * undo.y;
      }
      const float h = row < a.f ? g / (1.f + expf(-g)) * u : 0.f;
      using U = typename std::conditional<W4, __nv_bfloat16, T>::type;  // type of the products with down
      U* out = static_cast<U*>(a.hidden) + (size_t)pair * 2 * a.f_pad + row;
      const float scaled = h * MoeHidden<U>::kScale;
      const U v = from_f32<U>(scaled);
      const float rest = (scaled - to_f32(v)) * MoeHidden<U>::kRest;
      out[0] = v;
      out[a.f_pad] = from_f32<U>(isfinite(rest) ? rest : 0.f);
    }
    if (n + 1 < end) advance(unit);
  }
  asm volatile("cp.async.wait_all;" ::: "memory");
}

// ---------------------------------------------------------------- down ----------------
template <int QG>
struct MoeDownShape {
  static constexpr int kStep = QG ? 128 : 64;
  static constexpr uint32_t kSlot = QG ? kTileRoom : 2048;
  static constexpr int kSlots = QG ? 6 : 4;
};

template <typename T, int QG>
__global__ void __launch_bounds__(kMoeThreads, 1) moe_down_kernel(const MoeArgs a) {
  using S = MoeDownShape<QG>;
  constexpr bool W4 = QG > 0;
  using U = typename std::conditional<W4, __nv_bfloat16, T>::type;  // type of the products
  extern __shared__ __align__(128) unsigned char smem[];
  const int warp = threadIdx.x / 32, lane = threadIdx.x & 31, r = lane >> 2, t = lane & 3;
  const int pairs = a.tokens * a.topk, words = MoePlan::words(a.experts, pairs);
  const uint32_t ring = smem_u32(smem) + warp * S::kSlots * S::kSlot;
  float* sums = reinterpret_cast<float*>(smem + kMoeWarps * S::kSlots * S::kSlot);  // [warp][token][row]
  int* at_plan = reinterpret_cast<int*>(sums + kMoeWarps * a.tokens * 16);
  MoePlan plan(at_plan, a.experts, pairs);
  griddep_launch_dependents();
  griddep_wait();
  for (int i = threadIdx.x; i < words; i += kMoeThreads) at_plan[i] = a.plan[i];
  for (int i = threadIdx.x; i < kMoeWarps * a.tokens * 16; i += kMoeThreads) sums[i] = 0.f;
  __syncthreads();
  const int active = *plan.active;

  const int steps = (a.f + S::kStep - 1) / S::kStep;
  int total = 0;
  for (int i = 0; i < active; ++i) total += (plan.start[i + 1] - plan.start[i] + 7) / 8;
  const long long all = (long long)total * steps;
  const int row_blocks = (a.d + 15) / 16;
  const long long w0 = all * warp / kMoeWarps, w1 = all * (warp + 1) / kMoeWarps;
  const bool vec = !W4 && a.ldd % 8 == 0 && a.strideD % 8 == 0 && a.f % 8 == 0 &&
                   (reinterpret_cast<uintptr_t>(a.down) & 15u) == 0;
  const uint32_t tile_bytes = W4 ? a.fmt.tile_bytes() : 0;
  // a run: what of this warp's part belongs to one expert and group of tokens
  struct Run {
    int index, group, groups, step;
  };
  Run first{0, 0, 0, 0};
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
  auto advance = [&](Run& p) {
    p.step = 0;
    if (++p.group < p.groups) return;
    p.group = 0;
    if (++p.index < active) p.groups = (plan.start[p.index + 1] - plan.start[p.index] + 7) / 8;
  };
  // the copies run ahead of the products, through the same order, on into the next row block
  using Feed = typename std::conditional<W4, TileFeed, RowsFeed<T, 2>>::type;
  Feed feed;
  Run ahead = first;
  int ahead_rows = w0 < w1 ? blockIdx.x : row_blocks, ahead_left = 0;
  long long ahead_n = w0;
  uint32_t ahead_at = ring;
  auto start = [&]() {
    if (ahead_rows >= row_blocks) return;
    const size_t e = plan.expert[ahead.index];
    ahead_left = (int)min((long long)(steps - ahead.step), w1 - ahead_n);
    if constexpr (W4)
      feed.start(static_cast<const unsigned char*>(a.down) + e * a.strideD + ((size_t)ahead_rows * steps + ahead.step) * tile_bytes,
                 tile_bytes, 0);
    else
      feed.start(static_cast<const T*>(a.down) + e * a.strideD + (size_t)ahead_rows * 16 * a.ldd, a.ldd, a.d - ahead_rows * 16,
                 a.f, ahead.step, vec);
    ahead_n += ahead_left;
  };
  auto fetch = [&]() {
    if (ahead_rows < row_blocks) {
      feed.fetch(ahead_at);
      ahead_at += S::kSlot;
      if (ahead_at == ring + S::kSlots * S::kSlot) ahead_at = ring;
      if (--ahead_left == 0) {
        if (ahead_n == w1) {
          ahead_n = w0;
          ahead = first;
          ahead_rows += gridDim.x;
        } else {
          advance(ahead);
        }
        start();
      }
    }
    copies_commit();
  };
  start();
  for (int i = 0; i + 1 < S::kSlots; ++i) fetch();

  uint32_t from = ring;
  for (int rows = blockIdx.x; rows < row_blocks; rows += gridDim.x) {
    Run run = first;
    for (long long n = w0; n < w1; advance(run)) {
      const int p0 = plan.start[run.index] + run.group * 8, cols = min(8, plan.start[run.index + 1] - p0);
      const int length = (int)min((long long)(steps - run.step), w1 - n);
      n += length;
      const uint16_t* h = static_cast<const uint16_t*>(a.hidden) + (size_t)(plan.order[p0 + min(r, cols - 1)] & 0xffff) * 2 * a.f_pad +
                          run.step * S::kStep + t * 8;
      float acc[4] = {0.f, 0.f, 0.f, 0.f}, rest[4] = {0.f, 0.f, 0.f, 0.f};
      constexpr int kQuarters = S::kStep / 32;
      uint4 b[2][kQuarters], ahead_b[2][kQuarters];
      auto columns = [&](uint4(&to)[2][kQuarters]) {
#pragma unroll
        for (int q = 0; q < kQuarters; ++q) {
          to[0][q] = *reinterpret_cast<const uint4*>(h + q * 32);
          to[1][q] = *reinterpret_cast<const uint4*>(h + a.f_pad + q * 32);
        }
        h += S::kStep;
      };
      if (!W4) columns(ahead_b);
      for (int i = 0; i < length; ++i) {
        // 16-bit weights: the columns of the next step, too (packed ones leave no registers for it)
        if (W4) {
          columns(b);
        } else {
#pragma unroll
          for (int q = 0; q < kQuarters; ++q) {
            b[0][q] = ahead_b[0][q];
            b[1][q] = ahead_b[1][q];
          }
          if (i + 1 < length) columns(ahead_b);
        }
        __syncwarp();
        fetch();
        copies_wait<S::kSlots - 1>();
        if constexpr (W4) {
          __syncwarp();
          tile_multiply_bf16<T, QG>(from, b, a.fmt.zeros, acc);
        } else {
          rows16_multiply<T, 2>(from, acc, b[0]);
          rows16_multiply<T, 2>(from, rest, b[1]);
        }
        from += S::kSlot;
        if (from == ring + S::kSlots * S::kSlot) from = ring;
      }
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const int col = t * 2 + (i & 1);
        if (col < cols) {
          const int entry = plan.order[p0 + col];
          const float v = (acc[i] + rest[i] * (1.f / MoeHidden<U>::kRest)) * (1.f / MoeHidden<U>::kScale);
          sums[(warp * a.tokens + (entry >> 16)) * 16 + r + 8 * (i >> 1)] += plan.gate[entry & 0xffff] * v;
        }
      }
      __syncwarp();
    }
    __syncthreads();
    for (int i = threadIdx.x; i < a.tokens * 16; i += kMoeThreads) {
      float v = 0.f;
#pragma unroll
      for (int w = 0; w < kMoeWarps; ++w) {
        float* p = sums + w * a.tokens * 16 + i;
        v += *p;
        *p = 0.f;
      }
      const int row = rows * 16 + (i & 15);
      if (row < a.d) {
        T* y = static_cast<T*>(a.Y) + (size_t)(i / 16) * a.ldy + row;
        *y = from_f32<T>(a.beta != 0.f ? fmaf(a.beta, to_f32(*y), v) : v);
      }
    }
    __syncthreads();
  }
  asm volatile("cp.async.wait_all;" ::: "memory");
}

}  // namespace mmbo
