// A whole mixture-of-experts layer for a few tokens:
//
//   p(t, :) = softmax(router * x_t),  S(t) = the topk experts of largest p (equal ones: the lower index first)
//   g(t, e) = p(t, e)                 (or p(t, e) / sum of p over S(t))
//   y_t     = sum over e in S(t) of g(t, e) * down_e * (silu(gate_e * x_t) o (up_e * x_t))  +  beta * y_t
//
// with silu(v) = v / (1 + exp(-v)).  Scores, softmax, gates and all sums are held in 32 bits; a hidden value in a pair of 16-bit
// numbers, see MoeHidden.
//
// What bounds it: the bytes of the experts that the tokens choose, and for one token the chain of three kernels.  They run in
// one stream, each launched while the one in front drains (programmatic dependent launch).  That hides the launch and what a block
// sets up, no more: a block of `down` has no room beside one of `up` on an SM, so it asks for its first weights when all of
// `up` has finished.
//   scores   one warp per (token, expert); also an aligned, zero-padded copy of the activations
//   up       every block repeats the selection for itself (one to eight microseconds, cheaper than another kernel and its
//            launch), then its share of the units (expert, 16 rows of gate and up, group of up to eight tokens)
//   down     a block owns 16 rows of the output for all tokens, its warps split the list of (expert, part of f); the sums
//            of the experts meet in shared memory in a fixed order
// Weights come through rings in shared memory that bulk copies fill, by warps that do nothing else (16-bit weights) or by the
// warps that multiply them (packed ones, whose copies are few and long); the columns, fragments of mma.sync.m16n8k16 (the same
// 16 bytes' worth of k of a lane's token), come straight from L2.  Tokens are the eight columns of the instruction; an expert
// with more tokens is taken in groups of eight, the later ones finding its weights in L2.
//
// Measured (whole layer, B200): 48 tokens, 8 of 64 fp16 experts, 2048 to 1408: 228 to 242 us, up 131 us (740 MB, 5.6 TB/s), down 100 us
// (371 MB on 128 of 148 SMs; 76 us without its arithmetic); one token, 6 of 64 bf16 experts of that size: 35 us, of which
// scores 8, up 22, down 13 one by one; 8 tokens, 4 of 32 packed experts, 4096 to 1800: 84 to 93 us (by the experts that the tokens
// choose), up 50 us and down 46 us (3.6 and 2.1 TB/s: instructions, about 150 a tile in up and 215 in down).  Asking for packed
// experts' columns a tile ahead made both slower (97 us where 89 were taken): the added instructions cost more than the wait.
// More than a pass's tokens read the experts again: 64 tokens 260 us, 128 tokens 522, 256 tokens 1056 (8 of 64 fp16).
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
  void* x;          // tokens x d_pad: the activations, zero behind d
  void* hidden;     // pairs x 2 x f_pad, zero behind f: hidden vectors as a 16-bit value and what its rounding left, see MoeHidden
  int* plan;        // what `up` found out for `down`, see MoePlan
  int d_pad, f_pad; // multiples of 128
};

// The selection, sorted by expert: `order` holds the pairs (token * topk + slot, and the token again in the upper half: a
// division saved wherever a column is looked up) of expert 0's tokens, then expert 1's ..;
// the a-th expert with tokens is expert[a], its pairs order[start[a] .. start[a + 1]), in groups of eight, the first of which
// is number base[a].
struct MoePlan {
  int* active;  // number of experts with tokens
  int* expert;
  int* start;
  int* base;
  int* order;
  float* gate;  // per pair
  __host__ __device__ static int words(int experts, int pairs) {
    const int a = experts < pairs ? experts : pairs;
    return 1 + a + 2 * (a + 1) + 2 * pairs;
  }
  __device__ __forceinline__ MoePlan(int* at, int experts, int pairs) {
    const int a = min(experts, pairs);
    active = at;
    expert = at + 1;
    start = expert + a;
    base = start + a + 1;
    order = base + a + 1;
    gate = reinterpret_cast<float*>(order + pairs);
  }
};

// Order of the scores as unsigned integers: larger score, larger key; -0 equals +0.
__device__ __forceinline__ uint32_t moe_score_key(float v) {
  if (v == 0.f) v = 0.f;
  const uint32_t b = __float_as_uint(v);
  return (b & 0x80000000u) ? ~b : (b | 0x80000000u);
}

template <typename T>
__global__ void __launch_bounds__(256) moe_scores_kernel(const MoeArgs a) {
  griddep_launch_dependents();
  griddep_wait();
  const int t = blockIdx.y, lane = threadIdx.x & 31;
  const T* x = static_cast<const T*>(a.X) + (size_t)t * a.ldx;
  if (blockIdx.x == gridDim.x - 1) {  // the last block of a token prepares the workspace instead
    uint16_t* h = static_cast<uint16_t*>(a.hidden) + (size_t)t * a.topk * a.f_pad * 2;
    const int pad = a.f_pad - a.f;
    for (int i = threadIdx.x; i < a.topk * 2 * pad; i += 256) h[(size_t)(i / pad) * a.f_pad + a.f + i % pad] = 0;
    T* copy = static_cast<T*>(a.x) + (size_t)t * a.d_pad;
    for (int j = threadIdx.x * 8; j < a.d_pad; j += 256 * 8) *reinterpret_cast<uint4*>(copy + j) = load8(x, a.d, j);
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
  // A NaN or +inf among the scores, or nothing but -inf: every p is a NaN, so all are equal.
  const bool lost = sum != sum;
  uint32_t last_key = 0xffffffffu;
  int last = -1;  // the expert taken before
  for (int s = 0; s < a.topk; ++s) {
    uint32_t key = 0;
    int best = 0;
    for (int e = lane; e < a.experts; e += 32) {
      const uint32_t k = lost ? 1u : moe_score_key(scores[e]);
      if ((k < last_key || (k == last_key && e > last)) && k > key) {
        key = k;
        best = e;
      }
    }
    last_key = __reduce_max_sync(0xffffffffu, key);
    last = (int)__reduce_min_sync(0xffffffffu, key == last_key ? (uint32_t)best : 0xffffffffu);
    if (lane == 0) ids[s] = last;
  }
  __syncwarp();
  const float p = lane < a.topk ? expf(scores[ids[lane]] - top) / sum : 0.f;
  float chosen = p;
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) chosen += __shfl_xor_sync(0xffffffffu, chosen, o);
  if (lane < a.topk) gates[lane] = a.renorm ? p / chosen : p;
}

// ---------------------------------------------------------------- hidden vectors ------
// Hidden vectors as products take them: a 16-bit value and what its rounding left, so that 16 bits and more survive.
// bfloat16 has the range of a float: off by 2^-17 of the value at most.  Half precision holds h / 64 and 2^11 times the
// remainder: off by 2^-22 of the value, near zero by 2^-30 (results in half precision have steps of 2^-24), up to magnitudes of
// 4.19e6.  32 bits would take a third product, or one in a type that the weights do not have.
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

// The selection and its plan, by every block for itself; `scores`: kMoeUpSums bytes of shared memory.  All threads of
// the block take part (the first kMoeWarps warps in the selection).
constexpr size_t kMoeUpSums = (size_t)2 * kMoeWarps * 256 * 4;
template <typename A>
__device__ __forceinline__ void moe_make_plan(const A& a, MoePlan& plan, int* ids, int* count, float* scores) {
  const int warp = threadIdx.x / 32, lane = threadIdx.x & 31, pairs = a.tokens * a.topk;
  const int selecting = min(kMoeWarps, (int)(kMoeUpSums / 4) / a.experts);  // warps that have room for a token's scores
  for (int e = threadIdx.x; e < a.experts; e += blockDim.x) count[e] = 0;
  for (int tok = warp; warp < selecting && tok < a.tokens; tok += selecting)
    moe_select(a, a.scores + (size_t)tok * a.experts, scores + warp * a.experts, ids + tok * a.topk, plan.gate + tok * a.topk);
  __syncthreads();
  for (int p = threadIdx.x; p < pairs; p += blockDim.x) atomicAdd(&count[ids[p]], 1);
  __syncthreads();
  if (warp == 0) {  // experts with tokens, numbered in order, and where their pairs start
    int n = 0, at = 0, groups = 0;
    for (int e0 = 0; e0 < a.experts; e0 += 32) {
      const int e = e0 + lane, c = e < a.experts ? count[e] : 0;
      int before = c, before_groups = (c + 7) / 8;
#pragma unroll
      for (int o = 1; o < 32; o <<= 1) {
        const int v = __shfl_up_sync(0xffffffffu, before, o), w = __shfl_up_sync(0xffffffffu, before_groups, o);
        if (lane >= o) {
          before += v;
          before_groups += w;
        }
      }
      const unsigned live = __ballot_sync(0xffffffffu, c > 0);
      if (c > 0) {
        const int i = n + __popc(live & ((1u << lane) - 1u));
        plan.expert[i] = e;
        plan.start[i] = at + before - c;
        plan.base[i] = groups + before_groups - (c + 7) / 8;
      }
      n += __popc(live);
      at += __shfl_sync(0xffffffffu, before, 31);
      groups += __shfl_sync(0xffffffffu, before_groups, 31);
    }
    if (lane == 0) {
      *plan.active = n;
      plan.start[n] = at;
      plan.base[n] = groups;
    }
  }
  __syncthreads();
  const int active = *plan.active;
  for (int i = warp; i < active; i += blockDim.x / 32) {
    const int e = plan.expert[i];
    int at = plan.start[i];
    for (int p0 = 0; p0 < pairs; p0 += 32) {
      const int p = p0 + lane;
      const bool its = p < pairs && ids[p] == e;
      const unsigned which = __ballot_sync(0xffffffffu, its);
      if (its) plan.order[at + __popc(which & ((1u << lane) - 1u))] = p | (p / a.topk) << 16;
      at += __popc(which);
    }
  }
  __syncthreads();
  if (blockIdx.x == 0) {
    for (int i = threadIdx.x; i < MoePlan::words(a.experts, pairs); i += blockDim.x) a.plan[i] = plan.active[i];
    for (int p = threadIdx.x; p < pairs; p += blockDim.x) {
      if (a.ids) a.ids[p] = ids[p];
      if (a.gates) a.gates[p] = plan.gate[p];
    }
  }
}

// The units of `up`, in order: experts with tokens, row blocks of the hidden vector, groups of eight tokens.
struct MoeUnit {
  int index, rows, group, groups;
  __device__ __forceinline__ static int total(const MoePlan& plan, int blocks) { return blocks * plan.base[*plan.active]; }
  __device__ __forceinline__ void find(const MoePlan& plan, int blocks, int number) {
    int lo = 0, hi = *plan.active;  // blocks * base[lo] <= number
    while (hi - lo > 1) {
      const int mid = (lo + hi) / 2;
      (blocks * plan.base[mid] <= number ? lo : hi) = mid;
    }
    index = lo;
    groups = plan.base[lo + 1] - plan.base[lo];
    rows = (number - blocks * plan.base[lo]) / groups;
    group = (number - blocks * plan.base[lo]) % groups;
  }
  __device__ __forceinline__ void advance(const MoePlan& plan, int blocks) {
    if (++group < groups) return;
    group = 0;
    if (++rows < blocks) return;
    rows = 0;
    if (++index < *plan.active) groups = plan.base[index + 1] - plan.base[index];
  }
};

// A hidden value into the workspace, as the products with `down` take it.
template <typename U>
__device__ __forceinline__ void moe_store_hidden(const MoeArgs& a, int pair, int row, float g, float u) {
  const float h = row < a.f ? g / (1.f + expf(-g)) * u : 0.f;
  U* out = static_cast<U*>(a.hidden) + (size_t)pair * 2 * a.f_pad + row;
  const float scaled = h * MoeHidden<U>::kScale;
  const U v = from_f32<U>(scaled);
  const float rest = (scaled - to_f32(v)) * MoeHidden<U>::kRest;
  out[0] = v;
  out[a.f_pad] = from_f32<U>(isfinite(rest) ? rest : 0.f);
}

// ---------------------------------------------------------------- up ------------------
// Joins a unit's sums, [warp][gate, up][column][row] of `warps` warps at `sums`, `unit` times too small, and stores the hidden
// values; thread i of those that share the unit.
template <typename U>
__device__ __forceinline__ void moe_finish_unit(const MoeArgs& a, const float* sums, int warps, int i, int cols, int rows,
                                                const int* order, float unit) {
  if (i >= cols * 16) return;
  float g = 0.f, u = 0.f;
  for (int w = 0; w < warps; w += 4) {
#pragma unroll
    for (int v = 0; v < 4; ++v) {
      g += sums[(w + v) * 256 + i];
      u += sums[(w + v) * 256 + 128 + i];
    }
  }
  moe_store_hidden<U>(a, order[i / 16] & 0xffff, rows * 16 + (i & 15), g * unit, u * unit);
}
__device__ __forceinline__ void moe_keep_sums(float* to, const float (&gate)[4], const float (&up)[4]) {
  const int lane = threadIdx.x & 31, r = lane >> 2, t = lane & 3;
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const int at = (t * 2 + (i & 1)) * 16 + r + 8 * (i >> 1);
    to[at] = gate[i];
    to[128 + at] = up[i];
  }
}

// 16-bit weights.  A stage holds 512 columns of 16 rows of gate and of up, each row one copy of 1 KB (a warp's own copies of
// 64 or 128 bytes a row left DRAM at 3.9 TB/s).  Teams of four warps take the stages in turn: with all sixteen in step on
// every stage the columns' way from L2 was the bound (390 us instead of 241 for 48 tokens, 8 of 64 experts each, 2048 to
// 1408).  Rows lie 64 bytes out of step: conflict-free 16-byte reads.
constexpr int kMoeChunk = 512, kMoeTeam = 4;
constexpr uint32_t kMoeRowBytes = kMoeChunk * 2 + 64;
// Multiples of the teams: a team always waits at the same barriers, phase after phase (one that skipped phases could take an
// older one for its own).
constexpr int kMoeUpStages = 4, kMoeDownStages = 8;
static_assert(kMoeUpStages % (kMoeWarps / kMoeTeam) == 0 && kMoeDownStages % (kMoeWarps / kMoeTeam) == 0, "");
// Feeding warps, each for a part of the rows of a stage: a copy costs the warp that issues it some 30 clocks.
constexpr int kMoeFeeders = 4, kMoeFed16Threads = kMoeThreads + kMoeFeeders * 32;

// One warp's copies of `rows` rows into a stage.  One elected lane issues them: 100 clocks a copy with one row to a lane.
template <typename T>
__device__ __forceinline__ void moe_bring_rows(uint32_t to, const T* src, size_t ld, int rows, uint32_t bytes, uint32_t bar) {
  if (elect_one()) {
    mbar_expect_tx(bar, rows * bytes);
#pragma unroll 4
    for (int i = 0; i < rows; ++i) bulk_load(to + i * kMoeRowBytes, src + i * ld, bytes, bar);
  }
  __syncwarp();
}

// A lane's quarters of a stage, f(which of the team's four, its first column): all of them, without a branch, when the stage
// is whole.
template <typename F>
__device__ __forceinline__ void moe_quarters(int member, int columns, F f) {
  if (columns >= kMoeChunk) {
#pragma unroll
    for (int i = 0; i < 4; ++i) f(i, (i * kMoeTeam + member) * 32, std::true_type());
  } else {
#pragma unroll
    for (int i = 0; i < 4; ++i)
      if ((i * kMoeTeam + member) * 32 < columns) f(i, (i * kMoeTeam + member) * 32, std::false_type());
  }
}
// Sixteen bytes of a lane's row in a stage; zeros where the row ends before them.
template <bool WHOLE>
__device__ __forceinline__ uint4 moe_piece(uint32_t stage, int row, int column, int columns) {
  return WHOLE || column < columns ? lds128(stage + row * kMoeRowBytes + column * 2) : make_uint4(0, 0, 0, 0);
}

// FED: rows that bulk copies can address; others are read by the multiplying warps themselves, four times as slow (48 tokens, 8 of
// 64 fp16 experts: 230 us at 2048 to 1408, 960 at 2047 to 1407).
template <typename T, bool FED>
__global__ void __launch_bounds__(kMoeFed16Threads, 1) moe_up16_kernel(const MoeArgs a) {
  extern __shared__ __align__(128) unsigned char smem[];
  __shared__ __align__(8) unsigned long long full[kMoeUpStages], empty[kMoeUpStages], sums_full[2], sums_free[2];
  __shared__ uint32_t abort_flag;
  constexpr uint32_t kStage = 32 * kMoeRowBytes;
  const int warp = threadIdx.x / 32, lane = threadIdx.x & 31, r = lane >> 2, t = lane & 3;
  const int pairs = a.tokens * a.topk;
  // shared memory: stages | partial sums (before that: scores) | plan | ids | count
  const uint32_t ring = smem_u32(smem);
  float* sums = reinterpret_cast<float*>(smem + kMoeUpStages * kStage);
  int* at_plan = reinterpret_cast<int*>(sums) + kMoeUpSums / 4;
  MoePlan plan(at_plan, a.experts, pairs);
  int* ids = at_plan + MoePlan::words(a.experts, pairs);
  if (threadIdx.x == 0) {
    abort_flag = 0;
    for (int i = 0; i < kMoeUpStages; ++i) {
      mbar_init(smem_u32(&full[i]), kMoeFeeders);
      mbar_init(smem_u32(&empty[i]), kMoeTeam);
    }
    for (int i = 0; i < 2; ++i) {
      mbar_init(smem_u32(&sums_full[i]), kMoeWarps);
      mbar_init(smem_u32(&sums_free[i]), kMoeTeam);
    }
  }
  fence_mbar_init();
  griddep_launch_dependents();
  griddep_wait();
  moe_make_plan(a, plan, ids, ids + pairs, sums);

  const int blocks = (a.f + 15) / 16, total = MoeUnit::total(plan, blocks);
  const int begin = (int)((long long)total * blockIdx.x / gridDim.x), end = (int)((long long)total * (blockIdx.x + 1) / gridDim.x);
  MoeUnit unit;
  unit.find(plan, blocks, begin);
  const int chunks = (a.d + kMoeChunk - 1) / kMoeChunk, units = end - begin;
  constexpr int kTeams = kMoeWarps / kMoeTeam;
  bool ok = true;
  int count = 0;  // of stages
  if (warp >= kMoeWarps) {
    constexpr int kRows = 32 / kMoeFeeders;
    const int first = (warp - kMoeWarps) * kRows;  // of the stage's rows, those that this warp brings
    for (int n = 0; FED && ok && n < units; ++n) {
      const int row = unit.rows * 16 + (first & 15), have = min(kRows, max(a.f - row, 0));
      const T* src = static_cast<const T*>(first < 16 ? a.gate : a.up) + plan.expert[unit.index] * a.strideG + (size_t)row * a.ldg;
      for (int c = 0; c < a.d; c += kMoeChunk, ++count) {
        const int stage = count % kMoeUpStages;
        ok = mbar_wait_together(smem_u32(&empty[stage]), (count / kMoeUpStages & 1) ^ 1u, &abort_flag, kFaultWaitEmpty, 0x4d00u);
        if (!ok) break;
        moe_bring_rows(ring + stage * kStage + first * kMoeRowBytes, src + c, a.ldg, have, min(kMoeChunk, a.d - c) * 2,
                       smem_u32(&full[stage]));
      }
      unit.advance(plan, blocks);
    }
  } else {
    const int team = warp / kMoeTeam, member = warp % kMoeTeam;
    // A lane's columns of a stage, asked for a turn ahead; columns past the last token repeat it, their sums are not used.
    uint4 b[4];
    MoeUnit ahead = unit;
    int ahead_n = -1;
    const T* x = nullptr;
    auto ask = [&](int at) {
      if (at >= units * chunks) return;
      const bool moved = at >= (ahead_n + 1) * chunks;
      while (at >= (ahead_n + 1) * chunks)
        if (++ahead_n > 0) ahead.advance(plan, blocks);
      if (moved) {
        const int p0 = plan.start[ahead.index] + ahead.group * 8, cols = min(8, plan.start[ahead.index + 1] - p0);
        x = static_cast<const T*>(a.x) + (size_t)(plan.order[p0 + min(r, cols - 1)] >> 16) * a.d_pad + t * 8;
      }
      const int c = (at - ahead_n * chunks) * kMoeChunk;
      moe_quarters(member, a.d - c, [&](int i, int j, auto) { b[i] = *reinterpret_cast<const uint4*>(x + c + j); });
    };
    ask(count = team);
    for (int n = 0; n < units; ++n) {
      const int p0 = plan.start[unit.index] + unit.group * 8, cols = min(8, plan.start[unit.index + 1] - p0);
      float gate[4] = {0.f, 0.f, 0.f, 0.f}, up[4] = {0.f, 0.f, 0.f, 0.f};
      for (; count < (n + 1) * chunks; count += kTeams) {
        const int stage = count % kMoeUpStages, c = (count - n * chunks) * kMoeChunk, columns = min(kMoeChunk, a.d - c);
        if (FED && ok)
          ok = mbar_wait_together(smem_u32(&full[stage]), count / kMoeUpStages & 1, &abort_flag, kFaultWaitFull, 0x4d01u);
        const uint32_t at = ring + stage * kStage;
        const size_t off = plan.expert[unit.index] * a.strideG + (size_t)(unit.rows * 16 + r) * a.ldg;
        const int lo = unit.rows * 16 + r < a.f ? a.d : 0, hi = unit.rows * 16 + r + 8 < a.f ? a.d : 0;
        moe_quarters(member, columns, [&](int i, int j, auto whole) {
          uint4 g0, g1, u0, u1;
          if (FED) {
            constexpr bool kWhole = decltype(whole)::value;
            g0 = moe_piece<kWhole>(at, r, j + t * 8, columns);
            g1 = moe_piece<kWhole>(at, r + 8, j + t * 8, columns);
            u0 = moe_piece<kWhole>(at, r + 16, j + t * 8, columns);
            u1 = moe_piece<kWhole>(at, r + 24, j + t * 8, columns);
          } else {
            g0 = load8(static_cast<const T*>(a.gate) + off, lo, c + j + t * 8);
            g1 = load8(static_cast<const T*>(a.gate) + off + 8 * a.ldg, hi, c + j + t * 8);
            u0 = load8(static_cast<const T*>(a.up) + off, lo, c + j + t * 8);
            u1 = load8(static_cast<const T*>(a.up) + off + 8 * a.ldg, hi, c + j + t * 8);
          }
          mma_16816<T>(gate, g0.x, g1.x, g0.y, g1.y, b[i].x, b[i].y);
          mma_16816<T>(up, u0.x, u1.x, u0.y, u1.y, b[i].x, b[i].y);
          mma_16816<T>(gate, g0.z, g1.z, g0.w, g1.w, b[i].z, b[i].w);
          mma_16816<T>(up, u0.z, u1.z, u0.w, u1.w, b[i].z, b[i].w);
        });
        __syncwarp();
        if (FED && lane == 0) mbar_arrive(smem_u32(&empty[stage]));
        ask(count + kTeams);
      }
      // the team that had the unit's last stage finishes it
      const uint32_t which = n & 1, parity = n >> 1 & 1;
      float* ours = sums + which * kMoeWarps * 256;
      if (ok) ok = mbar_wait_together(smem_u32(&sums_free[which]), parity ^ 1u, &abort_flag, kFaultWaitEmpty, 0x4d02u);
      moe_keep_sums(ours + warp * 256, gate, up);
      __syncwarp();
      if (lane == 0) mbar_arrive(smem_u32(&sums_full[which]));
      if (((n + 1) * chunks - 1) % kTeams == team) {
        if (ok) ok = mbar_wait_together(smem_u32(&sums_full[which]), parity, &abort_flag, kFaultWaitFull, 0x4d03u);
        moe_finish_unit<T>(a, ours, kMoeWarps, member * 32 + lane, cols, unit.rows, plan.order + p0, 1.f);
        __syncwarp();
        if (lane == 0) mbar_arrive(smem_u32(&sums_free[which]));
      }
      unit.advance(plan, blocks);
    }
  }
  if (!ok) {  // a wait ran out: give the copies still in flight time to land
    const uint64_t since = global_timer_ns();
    while (global_timer_ns() - since < MMBO_DRAIN_LIMIT_NS) __nanosleep(1000);
  }
}

// Packed weights.  Every warp fills a ring of its own: a slot holds up to kMoeTiles consecutive tiles of gate and as many of
// up.  Teams of warps share units and cut d.
constexpr int kMoeTiles = 2, kMoeSlots = 2;

template <typename T, int QG>
__global__ void __launch_bounds__(kMoeThreads, 1) moe_up4_kernel(const MoeArgs a) {
  extern __shared__ __align__(128) unsigned char smem[];
  __shared__ __align__(8) unsigned long long full_bars[kMoeWarps * kMoeSlots];
  __shared__ uint32_t abort_flag;
  const int warp = threadIdx.x / 32, lane = threadIdx.x & 31, r = lane >> 2, t = lane & 3;
  const int pairs = a.tokens * a.topk;
  const uint32_t tile_bytes = a.fmt.tile_bytes(), half = kMoeTiles * tile_bytes, slot_bytes = 2 * half;
  // shared memory: rings | partial sums (before that: scores) | plan | ids | count
  float* sums = reinterpret_cast<float*>(smem + kMoeWarps * kMoeSlots * slot_bytes);
  int* at_plan = reinterpret_cast<int*>(sums) + kMoeUpSums / 4;
  MoePlan plan(at_plan, a.experts, pairs);
  int* ids = at_plan + MoePlan::words(a.experts, pairs);
  if (threadIdx.x == 0) abort_flag = 0;
  if (threadIdx.x < kMoeWarps * kMoeSlots) mbar_init(smem_u32(&full_bars[threadIdx.x]), 1);
  fence_mbar_init();
  griddep_launch_dependents();
  griddep_wait();
  moe_make_plan(a, plan, ids, ids + pairs, sums);

  const int WK = 1 << a.team_log2, wk = warp & (WK - 1), team = warp >> a.team_log2, teams = kMoeWarps >> a.team_log2;
  const int blocks = (a.f + 15) / 16, total = MoeUnit::total(plan, blocks);
  const long long share = (long long)gridDim.x * teams, mine = (long long)blockIdx.x * teams + team;
  const int begin = (int)(total * mine / share), end = (int)(total * (mine + 1) / share);
  MoeUnit unit;
  unit.find(plan, blocks, begin);
  const int steps = (a.d + 127) / 128, s0 = steps * wk >> a.team_log2, s1 = steps * (wk + 1) >> a.team_log2;
  const uint32_t full = smem_u32(&full_bars[warp * kMoeSlots]), ring = smem_u32(smem) + warp * kMoeSlots * slot_bytes;
  // what the ring is filled with next
  MoeUnit ahead = unit;
  int units_left = s0 < s1 ? end - begin : 0, at_step = s0;
  const unsigned char *from_gate = nullptr, *from_up = nullptr;
  auto fill = [&](int slot) {
    if (units_left <= 0) return;
    if (at_step == s0) {
      const size_t off = plan.expert[ahead.index] * a.strideG + ((size_t)ahead.rows * steps + s0) * tile_bytes;
      from_gate = static_cast<const unsigned char*>(a.gate) + off;
      from_up = static_cast<const unsigned char*>(a.up) + off;
    }
    const uint32_t bytes = min(kMoeTiles, s1 - at_step) * tile_bytes;
    if (elect_one()) {
      const uint32_t bar = full + slot * 8, to = ring + slot * slot_bytes;
      mbar_expect_tx(bar, 2 * bytes);
      bulk_load(to, from_gate, bytes, bar);
      bulk_load(to + half, from_up, bytes, bar);
    }
    __syncwarp();
    from_gate += bytes;
    from_up += bytes;
    if ((at_step += kMoeTiles) >= s1) {
      at_step = s0;
      --units_left;
      ahead.advance(plan, blocks);
    }
  };
  for (int i = 0; i < kMoeSlots; ++i) fill(i);
  bool ok = true;
  int slot = 0;
  uint32_t phase = 0;
  for (int n = begin; n < end; ++n) {
    const int p0 = plan.start[unit.index] + unit.group * 8, cols = min(8, plan.start[unit.index + 1] - p0);
    // columns past the last token repeat it; their sums are not used
    const T* x = static_cast<const T*>(a.x) + (size_t)(plan.order[p0 + min(r, cols - 1)] >> 16) * a.d_pad + s0 * 128 + t * 8;
    float gate[4] = {0.f, 0.f, 0.f, 0.f}, up[4] = {0.f, 0.f, 0.f, 0.f};
    for (int s = s0; s < s1; s += kMoeTiles) {
      const int cnt = min(kMoeTiles, s1 - s);
      uint32_t at = ring + slot * slot_bytes;
      for (int i = 0; i < cnt; ++i) {
        uint4 b[4];
#pragma unroll
        for (int q = 0; q < 4; ++q) b[q] = *reinterpret_cast<const uint4*>(x + q * 32);
        x += 128;
        if (i == 0 && ok) ok = mbar_wait_together(full + slot * 8, phase, &abort_flag, kFaultWaitFull, 0x4d10u + warp);
        w4_tile_mma<T, T, QG>(at, [&](int, int q) { return b[q]; }, a.fmt.zeros, gate);
        w4_tile_mma<T, T, QG>(at + half, [&](int, int q) { return b[q]; }, a.fmt.zeros, up);
        at += tile_bytes;
      }
      __syncwarp();
      fill(slot);
      if (++slot == kMoeSlots) {
        slot = 0;
        phase ^= 1u;
      }
    }
    float* ours = sums + ((n & 1) * kMoeWarps + (team << a.team_log2)) * 256;
    moe_keep_sums(ours + wk * 256, gate, up);
    __syncwarp();
    asm volatile("bar.sync %0, %1;" ::"r"(2 + team), "r"(WK * 32) : "memory");
    moe_finish_unit<__nv_bfloat16>(a, ours, WK, (wk * 32 + lane + 384 * (n & 3)) & (WK * 32 - 1), cols, unit.rows,
                                   plan.order + p0, W4Operand<T>::kUnit);
    unit.advance(plan, blocks);
  }
  if (!ok) {  // a wait ran out: give the copies still in flight time to land
    const uint64_t since = global_timer_ns();
    while (global_timer_ns() - since < MMBO_DRAIN_LIMIT_NS) __nanosleep(1000);
  }
}

// ---------------------------------------------------------------- down ----------------
// Adds an expert's products with the tokens of a group, times their gates and `unit`, to this warp's sums, [token][row].
template <typename U>
__device__ __forceinline__ void moe_add_products(const MoePlan& plan, float* sums, const int* order, int cols, const float (&acc)[4],
                                                 const float (&rest)[4], float unit) {
  const int lane = threadIdx.x & 31, r = lane >> 2, t = lane & 3;
  float v[4], *to[4];
#pragma unroll
  for (int i = 0; i < 4; ++i) {  // all read before one is written: a lane's four are different ones
    const int entry = order[min(t * 2 + (i & 1), cols - 1)];
    to[i] = sums + (entry >> 16) * 16 + r + 8 * (i >> 1);
    v[i] = fmaf(plan.gate[entry & 0xffff] * unit, acc[i] + rest[i] * (1.f / MoeHidden<U>::kRest), *to[i]);
  }
#pragma unroll
  for (int i = 0; i < 4; ++i)
    if (t * 2 + (i & 1) < cols) *to[i] = v[i];
  __syncwarp();
}
// Joins the warps' sums, stores 16 rows of the output and clears the sums; by the multiplying warps.
template <typename T>
__device__ __forceinline__ void moe_store_rows(const MoeArgs& a, float* sums, int rows) {
  workers_sync();
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
  workers_sync();
}

// 16-bit weights: stages of 512 columns of the block's 16 rows, expert after expert; teams of four warps take
// them in turn.
template <typename T, bool FED>
__global__ void __launch_bounds__(kMoeFed16Threads, 1) moe_down16_kernel(const MoeArgs a) {
  extern __shared__ __align__(128) unsigned char smem[];
  __shared__ __align__(8) unsigned long long full[kMoeDownStages], empty[kMoeDownStages];
  __shared__ uint32_t abort_flag;
  constexpr uint32_t kStage = 16 * kMoeRowBytes;
  const int warp = threadIdx.x / 32, lane = threadIdx.x & 31, r = lane >> 2, t = lane & 3;
  const int pairs = a.tokens * a.topk, words = MoePlan::words(a.experts, pairs);
  const uint32_t ring = smem_u32(smem);
  float* sums = reinterpret_cast<float*>(smem + kMoeDownStages * kStage);  // [warp][token][row]
  int* at_plan = reinterpret_cast<int*>(sums + kMoeWarps * a.tokens * 16);
  MoePlan plan(at_plan, a.experts, pairs);
  if (threadIdx.x == 0) {
    abort_flag = 0;
    for (int i = 0; i < kMoeDownStages; ++i) {
      mbar_init(smem_u32(&full[i]), kMoeFeeders);
      mbar_init(smem_u32(&empty[i]), kMoeTeam);
    }
  }
  fence_mbar_init();
  for (int i = threadIdx.x; i < kMoeWarps * a.tokens * 16; i += kMoeFed16Threads) sums[i] = 0.f;
  griddep_launch_dependents();
  griddep_wait();
  for (int i = threadIdx.x; i < words; i += kMoeFed16Threads) at_plan[i] = a.plan[i];
  __syncthreads();

  const int active = *plan.active, row_blocks = (a.d + 15) / 16;
  const int chunks = (a.f + kMoeChunk - 1) / kMoeChunk, row_stages = MoeUnit::total(plan, chunks);
  constexpr int kTeams = kMoeWarps / kMoeTeam;
  bool ok = true;
  int count = 0;  // of stages
  if (warp >= kMoeWarps) {
    constexpr int kRows = 16 / kMoeFeeders;
    const int first = (warp - kMoeWarps) * kRows;  // of the stage's rows, those that this warp brings
    for (int rows = blockIdx.x; FED && ok && rows < row_blocks; rows += gridDim.x) {
      const int row = rows * 16 + first, have = min(kRows, max(a.d - row, 0));
      for (int i = 0; ok && i < active; ++i) {
        const T* src = static_cast<const T*>(a.down) + plan.expert[i] * a.strideD + (size_t)row * a.ldd;
        for (int g = plan.base[i]; ok && g < plan.base[i + 1]; ++g)
          for (int c = 0; c < a.f; c += kMoeChunk, ++count) {
            const int stage = count % kMoeDownStages;
            ok = mbar_wait_together(smem_u32(&empty[stage]), (count / kMoeDownStages & 1) ^ 1u, &abort_flag, kFaultWaitEmpty,
                                    0x4d20u);
            if (!ok) break;
            moe_bring_rows(ring + stage * kStage + first * kMoeRowBytes, src + c, a.ldd, have, min(kMoeChunk, a.f - c) * 2,
                           smem_u32(&full[stage]));
          }
      }
    }
  } else {
    const int team = warp / kMoeTeam, member = warp % kMoeTeam;
    float* ours = sums + warp * a.tokens * 16;
    // The stage that is next, as expert, pairs and piece of f; a lane's columns of it are asked for a turn ahead.
    int e = 0, p0 = plan.start[0], c = 0;
    uint4 b[4][2];
    auto move = [&](int by) {
      for (c += by; c >= chunks;) {
        c -= chunks;
        if ((p0 += 8) < plan.start[e + 1]) continue;
        if (++e == active) e = 0;
        p0 = plan.start[e];
      }
    };
    auto ask = [&] {
      // columns past the last token repeat it; their sums are not used
      const T* h = static_cast<const T*>(a.hidden) +
                   (size_t)(plan.order[min(p0 + r, plan.start[e + 1] - 1)] & 0xffff) * 2 * a.f_pad + t * 8;
      h += c * kMoeChunk;
      moe_quarters(member, a.f - c * kMoeChunk, [&](int i, int j, auto) {
        b[i][0] = *reinterpret_cast<const uint4*>(h + j);
        b[i][1] = *reinterpret_cast<const uint4*>(h + a.f_pad + j);
      });
    };
    move(count = team);
    ask();
    for (int rows = blockIdx.x, until = row_stages; rows < row_blocks; rows += gridDim.x, until += row_stages) {
      for (; count < until; count += kTeams) {
        const int stage = count % kMoeDownStages, columns = min(kMoeChunk, a.f - c * kMoeChunk);
        const int cols = min(8, plan.start[e + 1] - p0);
        const T* w = static_cast<const T*>(a.down) + plan.expert[e] * a.strideD + (size_t)(rows * 16 + r) * a.ldd + c * kMoeChunk;
        const int lo = rows * 16 + r < a.d ? columns : 0, hi = rows * 16 + r + 8 < a.d ? columns : 0;
        const int* order = plan.order + p0;
        float acc[4] = {0.f, 0.f, 0.f, 0.f}, rest[4] = {0.f, 0.f, 0.f, 0.f};
        if (FED && ok)
          ok = mbar_wait_together(smem_u32(&full[stage]), count / kMoeDownStages & 1, &abort_flag, kFaultWaitFull, 0x4d21u);
        const uint32_t at = ring + stage * kStage;
        moe_quarters(member, columns, [&](int i, int j, auto whole) {
          uint4 w0, w1;
          if (FED) {
            constexpr bool kWhole = decltype(whole)::value;
            w0 = moe_piece<kWhole>(at, r, j + t * 8, columns);
            w1 = moe_piece<kWhole>(at, r + 8, j + t * 8, columns);
          } else {
            w0 = load8(w, lo, j + t * 8);
            w1 = load8(w + 8 * a.ldd, hi, j + t * 8);
          }
          mma_16816<T>(acc, w0.x, w1.x, w0.y, w1.y, b[i][0].x, b[i][0].y);
          mma_16816<T>(rest, w0.x, w1.x, w0.y, w1.y, b[i][1].x, b[i][1].y);
          mma_16816<T>(acc, w0.z, w1.z, w0.w, w1.w, b[i][0].z, b[i][0].w);
          mma_16816<T>(rest, w0.z, w1.z, w0.w, w1.w, b[i][1].z, b[i][1].w);
        });
        __syncwarp();
        if (FED && lane == 0) mbar_arrive(smem_u32(&empty[stage]));
        move(kTeams);
        ask();
        moe_add_products<T>(plan, ours, order, cols, acc, rest, 1.f / MoeHidden<T>::kScale);
      }
      moe_store_rows<T>(a, sums, rows);
    }
  }
  if (!ok) {  // a wait ran out: give the copies still in flight time to land
    const uint64_t since = global_timer_ns();
    while (global_timer_ns() - since < MMBO_DRAIN_LIMIT_NS) __nanosleep(1000);
  }
}

// Packed weights: the warps cut the list of (expert, group of tokens, tile) into equal parts and fill rings
// of their own.
constexpr int kMoeDownTiles = 3;

template <typename T, int QG>
__global__ void __launch_bounds__(kMoeThreads, 1) moe_down4_kernel(const MoeArgs a) {
  extern __shared__ __align__(128) unsigned char smem[];
  __shared__ __align__(8) unsigned long long full_bars[kMoeWarps * kMoeSlots];
  __shared__ uint32_t abort_flag;
  const int warp = threadIdx.x / 32, lane = threadIdx.x & 31, r = lane >> 2, t = lane & 3;
  const int pairs = a.tokens * a.topk, words = MoePlan::words(a.experts, pairs);
  const uint32_t tile_bytes = a.fmt.tile_bytes(), slot_bytes = kMoeDownTiles * tile_bytes;
  float* sums = reinterpret_cast<float*>(smem + kMoeWarps * kMoeSlots * slot_bytes);  // [warp][token][row]
  int* at_plan = reinterpret_cast<int*>(sums + kMoeWarps * a.tokens * 16);
  MoePlan plan(at_plan, a.experts, pairs);
  if (threadIdx.x == 0) abort_flag = 0;
  if (threadIdx.x < kMoeWarps * kMoeSlots) mbar_init(smem_u32(&full_bars[threadIdx.x]), 1);
  fence_mbar_init();
  for (int i = threadIdx.x; i < kMoeWarps * a.tokens * 16; i += kMoeThreads) sums[i] = 0.f;
  griddep_launch_dependents();
  griddep_wait();
  for (int i = threadIdx.x; i < words; i += kMoeThreads) at_plan[i] = a.plan[i];
  __syncthreads();

  const int steps = (a.f + 127) / 128, row_blocks = (a.d + 15) / 16;
  const long long all = (long long)MoeUnit::total(plan, 1) * steps;
  const long long w0 = all * warp / kMoeWarps, w1 = all * (warp + 1) / kMoeWarps;
  // a run: what of a warp's part belongs to one expert and group of tokens
  MoeUnit first;
  first.find(plan, 1, (int)(w0 / steps));
  const int first_step = (int)(w0 % steps);
  const uint32_t full = smem_u32(&full_bars[warp * kMoeSlots]), ring = smem_u32(smem) + warp * kMoeSlots * slot_bytes;
  // what the ring is filled with next
  MoeUnit ahead = first;
  int at_rows = blockIdx.x, at_step = first_step;
  long long at = w0;
  auto fill = [&](int slot) {
    if (at_rows >= row_blocks || w0 == w1) return;
    const int cnt = (int)min((long long)min(kMoeDownTiles, steps - at_step), w1 - at);
    const uint32_t bytes = cnt * tile_bytes;
    const unsigned char* src = static_cast<const unsigned char*>(a.down) + plan.expert[ahead.index] * a.strideD +
                               ((size_t)at_rows * steps + at_step) * tile_bytes;
    if (elect_one()) {
      mbar_expect_tx(full + slot * 8, bytes);
      bulk_load(ring + slot * slot_bytes, src, bytes, full + slot * 8);
    }
    __syncwarp();
    at += cnt;
    if ((at_step += cnt) == steps) {
      at_step = 0;
      ahead.advance(plan, 1);
    }
    if (at == w1) {
      at = w0;
      at_step = first_step;
      ahead = first;
      at_rows += gridDim.x;
    }
  };
  for (int i = 0; i < kMoeSlots; ++i) fill(i);
  bool ok = true;
  int slot = 0;
  uint32_t phase = 0;
  float* ours = sums + warp * a.tokens * 16;
  for (int rows = blockIdx.x; rows < row_blocks; rows += gridDim.x) {
    MoeUnit run = first;
    int step = first_step;
    for (long long n = w0; n < w1; run.advance(plan, 1), step = 0) {
      const int length = (int)min((long long)(steps - step), w1 - n);
      n += length;
      const int p0 = plan.start[run.index] + run.group * 8, cols = min(8, plan.start[run.index + 1] - p0);
      const __nv_bfloat16* h = static_cast<const __nv_bfloat16*>(a.hidden) +
                               (size_t)(plan.order[p0 + min(r, cols - 1)] & 0xffff) * 2 * a.f_pad + step * 128 + t * 8;
      float acc[4] = {0.f, 0.f, 0.f, 0.f};
      const float none[4] = {0.f, 0.f, 0.f, 0.f};
      for (int s = 0; s < length; s += kMoeDownTiles) {
        const int cnt = min(kMoeDownTiles, length - s);
        uint32_t tile = ring + slot * slot_bytes;
        for (int i = 0; i < cnt; ++i) {
          uint4 b[2][4];
#pragma unroll
          for (int q = 0; q < 4; ++q) {
            b[0][q] = *reinterpret_cast<const uint4*>(h + q * 32);
            b[1][q] = *reinterpret_cast<const uint4*>(h + a.f_pad + q * 32);
          }
          h += 128;
          if (i == 0 && ok) ok = mbar_wait_together(full + slot * 8, phase, &abort_flag, kFaultWaitFull, 0x4d30u + warp);
          w4_tile_mma<__nv_bfloat16, T, QG, 2>(tile, [&](int i, int q) { return b[i][q]; }, a.fmt.zeros, acc);
          tile += tile_bytes;
        }
        __syncwarp();
        fill(slot);
        if (++slot == kMoeSlots) {
          slot = 0;
          phase ^= 1u;
        }
      }
      moe_add_products<__nv_bfloat16>(plan, ours, plan.order + p0, cols, acc, none, W4Operand<__nv_bfloat16>::kUnit);
    }
    moe_store_rows<T>(a, sums, rows);
  }
  if (!ok) {  // a wait ran out: give the copies still in flight time to land
    const uint64_t since = global_timer_ns();
    while (global_timer_ns() - since < MMBO_DRAIN_LIMIT_NS) __nanosleep(1000);
  }
}

}  // namespace mmbo
