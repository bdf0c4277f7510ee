// Host side of the 4-bit and mixture-of-experts entry points: checks, launch shapes, launches.  Included by
// mmbo_api.cu behind its own definitions, whose lock, launch counter and device queries it uses.
#pragma once

#include "moe.cuh"
#include "w4.cuh"
#include "w4_gemv.cuh"
#include "w4_umma.cuh"

namespace mmbo {

static bool aligned_to(const void* p, uintptr_t a) { return (reinterpret_cast<uintptr_t>(p) & (a - 1)) == 0; }

static int check_w4(int dtype, size_t m, size_t k, int group, int zeros) {
  if (dtype != MMBO_DTYPE_F16 && dtype != MMBO_DTYPE_BF16) return MMBO_ERR_BAD_DTYPE;
  if (m > 0x7fffffffull || k > 0x7fffffffull) return MMBO_ERR_BAD_DIM;
  if (group != 32 && group != 64 && group != 128) return MMBO_ERR_BAD_GROUP;
  if (zeros != 0 && zeros != 1) return MMBO_ERR_BAD_GROUP;
  return MMBO_OK;
}

static size_t w4_total_bytes(size_t m, size_t k, const W4Format& f) {
  return w4_row_blocks(m) * w4_k_tiles(k) * f.tile_bytes();
}

// One warp per tile, eight to a block.
static int w4_tile_grid(size_t m, size_t k, unsigned* grid) {
  const size_t blocks = (w4_row_blocks(m) * w4_k_tiles(k) + 7) / 8;
  if (blocks > 0x1fffffffull) return MMBO_ERR_TOO_LARGE;  // tiles are counted in 32 bits
  *grid = (unsigned)blocks;
  return MMBO_OK;
}

// Lets a kernel use `bytes` of dynamic shared memory, once per device.
template <typename K>
static int allow_smem(K kernel, size_t bytes, bool (&done)[kMaxDevices]) {
  const int dev = current_device();
  if (dev < 0 || dev >= kMaxDevices) return MMBO_ERR_TOO_LARGE;
  if (done[dev]) return MMBO_OK;
  const cudaError_t e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)bytes);
  done[dev] = e == cudaSuccess;
  return (int)e;
}

constexpr size_t kGemvSmem = 227 * 1024 - 4096;  // of an SM's shared memory, less the kernel's static part

// Clusters of 1 << log2 blocks that run at once with one block per SM: fewer than SMs / blocks, since the blocks of a
// cluster share a group of SMs whose number is no multiple of theirs.
static int g_cluster_slots[kMaxDevices][3];

static int cluster_slots(int log2) {
  const int dev = current_device();
  if (log2 == 0 || dev < 0 || dev >= kMaxDevices) return sm_count() >> log2;
  int& known = g_cluster_slots[dev][log2];
  if (known == 0) {
    static bool prepared[kMaxDevices];
    auto kernel = w4_gemv_kernel<__half, 4, false>;
    int fit = 0;
    if (allow_smem(kernel, kGemvSmem, prepared) == MMBO_OK) {
      cudaLaunchConfig_t cfg = {};
      cfg.gridDim = dim3(1u << log2);
      cfg.blockDim = dim3(kGemvThreads);
      cfg.dynamicSmemBytes = kGemvSmem;
      cudaLaunchAttribute attr[1];
      attr[0].id = cudaLaunchAttributeClusterDimension;
      attr[0].val.clusterDim.x = 1u << log2;
      attr[0].val.clusterDim.y = attr[0].val.clusterDim.z = 1;
      cfg.attrs = attr;
      cfg.numAttrs = 1;
      if (cudaOccupancyMaxActiveClusters(&fit, kernel, &cfg) != cudaSuccess) fit = 0;
    }
    cudaGetLastError();
    if (fit <= 0) fit = (sm_count() >> log2) * 7 / 8;
    known = fit < (sm_count() >> log2) ? fit : sm_count() >> log2;
  }
  return known;
}

// Launch with clusters of 1 << log2 blocks and programmatic stream serialization.
template <typename K, typename... Args>
static int launch_clustered(K kernel, unsigned grid, unsigned threads, size_t smem, int log2, cudaStream_t st, Args... args) {
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(grid);
  cfg.blockDim = dim3(threads);
  cfg.dynamicSmemBytes = smem;
  cfg.stream = st;
  cudaLaunchAttribute attr[2];
  int n = 0;
  if (log2) {
    attr[n].id = cudaLaunchAttributeClusterDimension;
    attr[n].val.clusterDim.x = 1u << log2;
    attr[n].val.clusterDim.y = attr[n].val.clusterDim.z = 1;
    ++n;
  }
  if (settings().pdl) {
    attr[n].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[n].val.programmaticStreamSerializationAllowed = 1;
    ++n;
  }
  cfg.attrs = attr;
  cfg.numAttrs = n;
  const cudaError_t e = cudaLaunchKernelEx(&cfg, kernel, args...);
  MMBO_COUNT_LAUNCH();
  return (int)e;
}

// How w4_gemv_kernel cuts a problem: the cheapest of all (warps along k, blocks along k), by a sum of what was measured
// (B200, us): 0.022 a tile of the busiest SM, 0.3 a slot of a warp's ring, 0.05 a KB of activations staged, 1.8 / 2.5 to join
// clusters of two / four, 1 a batch of row groups.  8192 x 28672, one column: 29.2 us with the chosen 16 x 2, 30.8 with
// 16 x 1, 52 with 1 x 2; 4096 x 4096: 5.5 with 8 x 1, 8.1 with 8 x 2 (times of a call in a graph).
static bool plan_gemv(GemvArgs& a, uint32_t tile_bytes, const int (&clusters)[3], size_t* smem) {
  const size_t k_tiles = w4_k_tiles(a.k), blocks = w4_row_blocks(a.m);
  double best = 1e30;
  for (int wk_log2 = 0; wk_log2 <= 4; ++wk_log2)
    for (int split_log2 = 0; split_log2 <= 2; ++split_log2) {
      const size_t wk = (size_t)1 << wk_log2, split = (size_t)1 << split_log2, wm = kGemvWarps / wk;
      if (split > 1 && k_tiles < split) continue;
      const size_t groups = (blocks + wm - 1) >> (4 - wk_log2), span = (k_tiles + split - 1) >> split_log2;
      const size_t part = (span + wk - 1) >> wk_log2;
      const size_t cl = groups < (size_t)clusters[split_log2] ? groups : (size_t)clusters[split_log2];
      const size_t rounds = (groups + cl - 1) / cl;
      const int slot_tiles = part < 4 ? (int)(part ? part : 1) : 4;
      const double staged = (double)a.n * span * 0.25;
      double cost = rounds * wm * span * 0.022 + rounds * ((part + slot_tiles - 1) / slot_tiles) * 0.3 + staged * 0.05 +
                    (split == 1 ? 0.0 : split == 2 ? 1.8 : 2.5);
      if (cost >= best) continue;
      const size_t ring = (size_t)kGemvWarps * 2 * slot_tiles * tile_bytes;
      const size_t one = gemv_sums_bytes((int)wk, (int)split, a.n, 1);
      if (ring + one + gemv_x_bytes(a.n, 1) > kGemvSmem) continue;
      size_t x_tiles = (kGemvSmem - ring - one - a.n * 64) / (a.n * 256);
      if (x_tiles > span) x_tiles = span ? span : 1;
      if (x_tiles == 0) continue;
      const size_t x = gemv_x_bytes(a.n, x_tiles);
      size_t batch = (kGemvSmem - ring - x) / one;
      if (batch > rounds) batch = rounds;
      if (batch == 0 || (split > 1 && batch < rounds)) continue;
      const size_t batches = (rounds + batch - 1) / batch;
      cost += (x_tiles < span ? (batches - 1) * staged * 0.05 : 0.0) + (batches - 1) * 1.0;
      if (cost < best) {
        best = cost;
        a.wk_log2 = wk_log2;
        a.split_log2 = split_log2;
        a.slots = 2;
        a.slot_tiles = slot_tiles;
        a.x_tiles = (int)x_tiles;
        a.batch = (int)batch;
        a.clusters = (int)cl;
        *smem = ring + x + gemv_sums_bytes((int)wk, (int)split, a.n, (int)batch);
      }
    }
  return best < 1e30;
}

template <typename T, int QG, bool ZEROS>
static int launch_w4_gemv(GemvArgs a, cudaStream_t st) {
  auto kernel = w4_gemv_kernel<T, QG, ZEROS>;
  static bool prepared[kMaxDevices];
  int rc = allow_smem(kernel, kGemvSmem, prepared);
  if (rc) return rc;
  const int clusters[3] = {cluster_slots(0), cluster_slots(1), cluster_slots(2)};
  size_t smem = 0;
  if (!plan_gemv(a, W4Tile<QG, ZEROS>::kBytes, clusters, &smem)) return MMBO_ERR_TOO_LARGE;
  return launch_clustered(kernel, (unsigned)a.clusters << a.split_log2, kGemvThreads, smem, a.split_log2, st, a);
}

template <typename T>
static int dispatch_w4_gemv(const GemvArgs& a, W4Format f, cudaStream_t st) {
  switch (f.group * 2 + f.zeros) {
    case 64: return launch_w4_gemv<T, 1, false>(a, st);
    case 65: return launch_w4_gemv<T, 1, true>(a, st);
    case 128: return launch_w4_gemv<T, 2, false>(a, st);
    case 129: return launch_w4_gemv<T, 2, true>(a, st);
    case 256: return launch_w4_gemv<T, 4, false>(a, st);
    default: return launch_w4_gemv<T, 4, true>(a, st);
  }
}

// Tile width and blocks along k of w4_umma_kernel: the smallest number of cycles of the busiest SM, counted as rounds of
// tiles x k-tiles x the cycles of one (measured: 500, 620, 900 with 32, 64, 128 columns; 700, 1100 where the unpacking
// warps have to bring the activations, not worth it with 128) and what joining a cluster costs.
static void plan_umma(size_t m, size_t n, size_t k, bool x_tma, int* nt, int* split_log2) {
  const size_t row_tiles = (m + 127) / 128, k_tiles = w4_k_tiles(k);
  double best = 1e30;
  for (int w = 32; w <= (x_tma ? 128 : 64); w *= 2)
    for (int log2 = 0; log2 <= (w <= 64 ? 2 : 0); ++log2) {
      const size_t tiles = row_tiles * ((n + w - 1) / w), slots = (size_t)cluster_slots(log2);
      if (log2 && (tiles > slots || k_tiles < ((size_t)1 << log2))) continue;
      const size_t rounds = (tiles + slots - 1) / slots, span = (k_tiles + ((size_t)1 << log2) - 1) >> log2;
      const double tile = w == 32 ? (x_tma ? 500.0 : 700.0) : w == 64 ? (x_tma ? 620.0 : 1100.0) : 900.0;
      const double cost = (double)rounds * span * tile + (double)rounds * w * 10 +
                          (log2 == 0 ? 0.0 : log2 == 1 ? 2500.0 : 3500.0);
      if (cost < best) {
        best = cost;
        *nt = w;
        *split_log2 = log2;
      }
    }
}

// Packed tiles as 64-bit words: word of a tile, k-tile, row block; one load takes a k-tile of eight row blocks.  (With a row
// block's tiles as one axis the coordinate of a word would pass 2^31 for k above 1.8e9.)
static int make_tile_map(CUtensorMap* map, const unsigned char* packed, uint32_t tile_bytes, size_t k_tiles, size_t row_blocks) {
  EncodeTiledFn enc = encode_fn();
  if (!enc) return MMBO_ERR_NO_DRIVER_ENTRY;
  const cuuint64_t dims[3] = {tile_bytes / 8, k_tiles, row_blocks};
  const cuuint64_t strides[2] = {tile_bytes, k_tiles * tile_bytes};
  const cuuint32_t box[3] = {tile_bytes / 8, 1, 8}, steps[3] = {1, 1, 1};
  const CUresult r = enc(map, CU_TENSOR_MAP_DATA_TYPE_INT64, 3, const_cast<unsigned char*>(packed), dims, strides, box, steps,
                         CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_NONE, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
                         CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
  return r == CUDA_SUCCESS ? MMBO_OK : MMBO_ERR_TENSOR_MAP;
}

template <typename T, int NT, int QG, bool ZEROS>
static int launch_w4_umma(UmmaArgs a, cudaStream_t st) {
  using S = UmmaShape<NT>;
  auto kernel = w4_umma_kernel<T, NT, QG, ZEROS>;
  static bool prepared[kMaxDevices];
  int rc = allow_smem(kernel, kGemvSmem, prepared);
  if (rc) return rc;
  constexpr uint32_t kTile = W4Tile<QG, ZEROS>::kBytes;
  const size_t stage = S::kXBytes + umma_code_bytes(kTile), fixed = 1024 + (a.split_log2 ? NT * 512 : 0);
  static_assert(S::kUnpackSets == 1 || (kGemvSmem - 1024 - NT * 512) / (S::kXBytes + umma_code_bytes(kTile)) >=
                                           S::kUnpackSets + kUmmaASlots, "");  // see the unpackers
  a.stages = (int)((kGemvSmem - fixed) / stage);
  if (a.stages > kUmmaMaxStages) a.stages = kUmmaMaxStages;
  a.col_tiles = (int)((a.n + NT - 1) / NT);
  const size_t tiles = (a.m + 127) / 128 * (size_t)a.col_tiles;
  if (tiles > 0x3fffffffull) return MMBO_ERR_TOO_LARGE;
  a.tiles = (int)tiles;
  CUtensorMap w_map, map;
  memset(&w_map, 0, sizeof w_map);
  memset(&map, 0, sizeof map);
  if (a.k > 0 && (rc = make_tile_map(&w_map, a.packed, kTile, w4_k_tiles(a.k), w4_row_blocks(a.m)))) return rc;
  if (a.x_tma &&
      (rc = make_map(&map, std::is_same<T, __half>::value ? CU_TENSOR_MAP_DATA_TYPE_FLOAT16 : CU_TENSOR_MAP_DATA_TYPE_BFLOAT16,
                     2, a.B, a.k, a.n, a.ldb, 64, NT)))
    return rc;
  const unsigned blocks = a.split_log2 ? (unsigned)a.tiles << a.split_log2
                                       : (unsigned)(a.tiles < sm_count() ? a.tiles : sm_count());
  return launch_clustered(kernel, blocks, S::kThreads, a.stages * stage + fixed, a.split_log2, st, a, w_map, map);
}

template <typename T, int NT>
static int dispatch_w4_umma(const UmmaArgs& a, W4Format f, cudaStream_t st) {
  switch (f.group * 2 + f.zeros) {
    case 64: return launch_w4_umma<T, NT, 1, false>(a, st);
    case 65: return launch_w4_umma<T, NT, 1, true>(a, st);
    case 128: return launch_w4_umma<T, NT, 2, false>(a, st);
    case 129: return launch_w4_umma<T, NT, 2, true>(a, st);
    case 256: return launch_w4_umma<T, NT, 4, false>(a, st);
    default: return launch_w4_umma<T, NT, 4, true>(a, st);
  }
}

template <typename T>
static int run_w4_gemm(size_t m, size_t n, size_t k, float alpha, const void* packed, W4Format f, const void* B,
                       size_t ldb, float beta, void* C, size_t ldc, cudaStream_t st) {
  const unsigned char* w = static_cast<const unsigned char*>(packed);
  if (n <= 8) return dispatch_w4_gemv<T>(GemvArgs{m, n, k, ldb, ldc, alpha, beta, w, B, C}, f, st);
  int nt = 0, split_log2 = 0;
  const bool x_tma = k > 0 && ldb % 8 == 0 && aligned16(B);
  plan_umma(m, n, k, x_tma, &nt, &split_log2);
  const UmmaArgs a{m, n, k, ldb, ldc, alpha, beta, w, B, C, split_log2, x_tma};
  if (nt == 32) return dispatch_w4_umma<T, 32>(a, f, st);
  if (nt == 64) return dispatch_w4_umma<T, 64>(a, f, st);
  return dispatch_w4_umma<T, 128>(a, f, st);
}

// Workspace of the expert layer, for one pass.
struct MoeWorkspace {
  size_t scores, x, hidden, plan, total;
};
static MoeWorkspace moe_workspace(size_t tokens, size_t d, size_t f, size_t experts, size_t topk) {
  if (tokens > (size_t)moe_pass_tokens((int)topk)) tokens = moe_pass_tokens((int)topk);
  const size_t pairs = tokens * topk;
  MoeWorkspace w;
  w.scores = 0;
  w.x = w.scores + align_up(tokens * experts * 4, 256);
  w.hidden = w.x + align_up(tokens * align_up(d, 128) * 2, 256);
  w.plan = w.hidden + align_up(pairs * align_up(f, 128) * 4, 256);
  w.total = w.plan + align_up((size_t)MoePlan::words((int)experts, (int)pairs) * 4, 256);
  return w;
}

static int check_moe_sizes(int dtype, size_t tokens, size_t d, size_t f, size_t experts, size_t topk) {
  if (dtype != MMBO_DTYPE_F16 && dtype != MMBO_DTYPE_BF16) return MMBO_ERR_BAD_DTYPE;
  if (tokens > MMBO_MOE_MAX_TOKENS || experts == 0 || experts > MMBO_MOE_MAX_EXPERTS || topk == 0 || topk > experts ||
      topk > MMBO_MOE_MAX_TOPK || d == 0 || f == 0 || d > MMBO_MOE_MAX_WIDTH || f > MMBO_MOE_MAX_WIDTH)
    return MMBO_ERR_BAD_DIM;
  return MMBO_OK;
}

// QG: quarters of a group of packed weights, 0: 16-bit weights.
template <typename T, int QG>
static int launch_moe(const MoeArgs& args, cudaStream_t st) {
  MoeArgs a = args;
  const size_t pairs = (size_t)a.tokens * a.topk, words = MoePlan::words(a.experts, (int)pairs);
  const size_t up_rest = kMoeUpSums + (words + pairs + a.experts) * 4;
  const size_t down_rest = (size_t)kMoeWarps * a.tokens * 16 * 4 + words * 4;
  const size_t rows = (a.d + 15) / 16, down_blocks = rows < (size_t)sm_count() ? rows : (size_t)sm_count();
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3((unsigned)((a.experts + 7) / 8 + 1), (unsigned)a.tokens);
  cfg.blockDim = dim3(256);
  cfg.stream = st;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = attr;
  cfg.numAttrs = settings().pdl ? 1 : 0;
  static bool up_ready[2][kMaxDevices], down_ready[2][kMaxDevices];
  int rc;
  if constexpr (QG == 0) {
    const bool up_fed = a.ldg % 8 == 0 && a.strideG % 8 == 0 && a.d % 8 == 0 && aligned16(a.gate) && aligned16(a.up);
    const bool down_fed = a.ldd % 8 == 0 && a.strideD % 8 == 0 && a.f % 8 == 0 && aligned16(a.down);
    auto up = up_fed ? moe_up16_kernel<T, true> : moe_up16_kernel<T, false>;
    auto down = down_fed ? moe_down16_kernel<T, true> : moe_down16_kernel<T, false>;
    if ((rc = allow_smem(up, kGemvSmem, up_ready[up_fed])) || (rc = allow_smem(down, kGemvSmem, down_ready[down_fed]))) return rc;
    const size_t up_smem = kMoeUpStages * (size_t)(32 * kMoeRowBytes) + up_rest;
    const size_t down_smem = kMoeDownStages * (size_t)(16 * kMoeRowBytes) + down_rest;
    const cudaError_t e = cudaLaunchKernelEx(&cfg, moe_scores_kernel<T>, a);
    MMBO_COUNT_LAUNCH();
    if (e != cudaSuccess) return (int)e;
    if ((rc = launch_clustered(up, (unsigned)sm_count(), kMoeFed16Threads, up_smem, 0, st, a)))
      return rc;
    return launch_clustered(down, (unsigned)down_blocks, kMoeFed16Threads, down_smem, 0, st, a);
  } else {
    auto up = moe_up4_kernel<T, QG>;
    auto down = moe_down4_kernel<T, QG>;
    if ((rc = allow_smem(up, kGemvSmem, up_ready[0])) || (rc = allow_smem(down, kGemvSmem, down_ready[0]))) return rc;
    // Teams of `up`: small ones (fewer sums to join, fewer barriers) as long as most of them have a unit.  8 tokens, 4 of 32
    // experts, 4096 to 1800 (some 2200 units): 83 us with teams of four, 90 with sixteen; 1 token, 2 experts, 2048 to 1408 (176
    // units): 14.7 with four, 14.4 with eight, 15.1 with sixteen (the rule's).
    const size_t experts = pairs < (size_t)a.experts ? pairs : (size_t)a.experts, units = experts * ((a.f + 15) / 16);
    a.team_log2 = 4;
    while (a.team_log2 > 2 && units >= (size_t)sm_count() * (kMoeWarps >> (a.team_log2 - 1)) * 3 / 4) --a.team_log2;
    const size_t tile = a.fmt.tile_bytes();
    const cudaError_t e = cudaLaunchKernelEx(&cfg, moe_scores_kernel<T>, a);
    MMBO_COUNT_LAUNCH();
    if (e != cudaSuccess) return (int)e;
    if ((rc = launch_clustered(up, (unsigned)sm_count(), kMoeThreads, kMoeWarps * kMoeSlots * 2 * kMoeTiles * tile + up_rest, 0, st,
                               a)))
      return rc;
    return launch_clustered(down, (unsigned)down_blocks, kMoeThreads, kMoeWarps * kMoeSlots * kMoeDownTiles * tile + down_rest, 0,
                            st, a);
  }
}

template <typename T>
static int run_moe(const MoeArgs& a, cudaStream_t st) {
  switch (a.fmt.group) {
    case 0: return launch_moe<T, 0>(a, st);
    case 32: return launch_moe<T, 1>(a, st);
    case 64: return launch_moe<T, 2>(a, st);
    default: return launch_moe<T, 4>(a, st);
  }
}

}  // namespace mmbo

// f(a zero of the type, quarters of a group, whether there are zero points, whether the rows are aligned), all as types.
template <typename F>
static void for_w4_kind(int dtype, int group, int zeros, bool aligned, F f) {
  auto with_aligned = [&](auto zero, auto quarters, auto has_zeros) {
    if (aligned) f(zero, quarters, has_zeros, std::true_type());
    else f(zero, quarters, has_zeros, std::false_type());
  };
  auto with_group = [&](auto zero, auto has_zeros) {
    if (group == 32) with_aligned(zero, std::integral_constant<int, 1>(), has_zeros);
    else if (group == 64) with_aligned(zero, std::integral_constant<int, 2>(), has_zeros);
    else with_aligned(zero, std::integral_constant<int, 4>(), has_zeros);
  };
  auto with_zeros = [&](auto zero) {
    if (zeros) with_group(zero, std::true_type());
    else with_group(zero, std::false_type());
  };
  if (dtype == MMBO_DTYPE_F16) with_zeros(__half());
  else with_zeros(__nv_bfloat16());
}

extern "C" {

int mmbo_w4_bytes(size_t m, size_t k, int group, int zeros, size_t* bytes) {
  int rc = check_w4(MMBO_DTYPE_F16, m, k, group, zeros);
  if (rc) return rc;
  if (!bytes) return MMBO_ERR_NULL_POINTER;
  *bytes = w4_total_bytes(m, k, W4Format{group, zeros});
  return MMBO_OK;
}

int mmbo_w4_quantize(int dtype, size_t m, size_t k, int group, int zeros, const void* W, size_t ldw, void* packed,
                     void* stream) {
  MMBO_API_LOCK();
  int rc = check_w4(dtype, m, k, group, zeros);
  if (rc) return rc;
  if (m == 0 || k == 0) return MMBO_OK;
  if (!W || !packed) return MMBO_ERR_NULL_POINTER;
  if (ldw < k) return MMBO_ERR_BAD_LDA;
  if (!aligned_to(W, 2) || !aligned_to(packed, 16)) return MMBO_ERR_MISALIGNED;
  unsigned grid = 0;
  if ((rc = w4_tile_grid(m, k, &grid))) return rc;
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  for_w4_kind(dtype, group, zeros, ldw % 8 == 0 && aligned16(W), [&](auto zero, auto quarters, auto has_zeros, auto aligned) {
    using T = decltype(zero);
    w4_quantize_kernel<T, decltype(quarters)::value, decltype(has_zeros)::value, decltype(aligned)::value>
        <<<grid, 256, 0, st>>>(m, k, static_cast<const T*>(W), ldw, static_cast<unsigned char*>(packed));
  });
  MMBO_COUNT_LAUNCH();
  return (int)cudaGetLastError();
}

int mmbo_w4_pack(int dtype, size_t m, size_t k, int group, const unsigned char* codes, size_t ldcodes,
                 const void* scales, size_t ldscales, const unsigned char* zeroPoints, size_t ldzeros, void* packed,
                 void* stream) {
  MMBO_API_LOCK();
  const int zeros = zeroPoints != nullptr;
  int rc = check_w4(dtype, m, k, group, zeros);
  if (rc) return rc;
  if (m == 0 || k == 0) return MMBO_OK;
  if (!codes || !scales || !packed) return MMBO_ERR_NULL_POINTER;
  const size_t groups = (k + group - 1) / group;
  if (ldcodes < (k + 1) / 2) return MMBO_ERR_BAD_LDA;
  if (ldscales < groups || (zeros && ldzeros < groups)) return MMBO_ERR_BAD_LDB;
  if (!aligned_to(scales, 2) || !aligned_to(packed, 16)) return MMBO_ERR_MISALIGNED;
  unsigned grid = 0;
  if ((rc = w4_tile_grid(m, k, &grid))) return rc;
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  const W4Format f{group, zeros};
  unsigned char* out = static_cast<unsigned char*>(packed);
  if (dtype == MMBO_DTYPE_F16)
    w4_pack_kernel<__half><<<grid, 256, 0, st>>>(m, k, f, codes, ldcodes, static_cast<const __half*>(scales), ldscales,
                                                 zeroPoints, ldzeros, out);
  else
    w4_pack_kernel<__nv_bfloat16><<<grid, 256, 0, st>>>(m, k, f, codes, ldcodes,
                                                        static_cast<const __nv_bfloat16*>(scales), ldscales,
                                                        zeroPoints, ldzeros, out);
  MMBO_COUNT_LAUNCH();
  return (int)cudaGetLastError();
}

int mmbo_w4_unpack(int dtype, size_t m, size_t k, int group, int zeros, const void* packed, void* W, size_t ldw,
                   void* stream) {
  MMBO_API_LOCK();
  int rc = check_w4(dtype, m, k, group, zeros);
  if (rc) return rc;
  if (m == 0 || k == 0) return MMBO_OK;
  if (!W || !packed) return MMBO_ERR_NULL_POINTER;
  if (ldw < k) return MMBO_ERR_BAD_LDA;
  if (!aligned_to(W, 2) || !aligned_to(packed, 16)) return MMBO_ERR_MISALIGNED;
  unsigned grid = 0;
  if ((rc = w4_tile_grid(m, k, &grid))) return rc;
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  for_w4_kind(dtype, group, zeros, ldw % 8 == 0 && aligned16(W), [&](auto zero, auto quarters, auto has_zeros, auto aligned) {
    using T = decltype(zero);
    w4_unpack_kernel<T, decltype(quarters)::value, decltype(has_zeros)::value, decltype(aligned)::value>
        <<<grid, 256, 0, st>>>(m, k, static_cast<const unsigned char*>(packed), static_cast<T*>(W), ldw);
  });
  MMBO_COUNT_LAUNCH();
  return (int)cudaGetLastError();
}

int mmbo_gemm_w4(int dtype, size_t m, size_t n, size_t k, const float* alpha, const void* packed, int group, int zeros,
                 const void* B, size_t ldb, const float* beta, void* C, size_t ldc, void* stream) {
  MMBO_API_LOCK();
  int rc = check_w4(dtype, m, k, group, zeros);
  if (rc) return rc;
  if (n > 0x7fffffffull) return MMBO_ERR_BAD_DIM;
  if (!alpha || !beta) return MMBO_ERR_NULL_POINTER;
  if (m == 0 || n == 0) return MMBO_OK;
  if (!C || (k && (!packed || !B))) return MMBO_ERR_NULL_POINTER;
  if (k && (ldb < k || ldb > 0x7fffffffull)) return MMBO_ERR_BAD_LDB;
  if (ldc < m || ldc > 0x7fffffffull) return MMBO_ERR_BAD_LDC;
  if (!aligned_to(C, 2) || (k && (!aligned_to(B, 2) || !aligned_to(packed, 16)))) return MMBO_ERR_MISALIGNED;
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  const W4Format f{group, zeros};
  if (dtype == MMBO_DTYPE_F16) return run_w4_gemm<__half>(m, n, k, *alpha, packed, f, B, ldb, *beta, C, ldc, st);
  return run_w4_gemm<__nv_bfloat16>(m, n, k, *alpha, packed, f, B, ldb, *beta, C, ldc, st);
}

int mmbo_moe_workspace_bytes(int dtype, size_t tokens, size_t d, size_t f, size_t experts, size_t topk, size_t* bytes) {
  int rc = check_moe_sizes(dtype, tokens, d, f, experts, topk);
  if (rc) return rc;
  if (!bytes) return MMBO_ERR_NULL_POINTER;
  *bytes = moe_workspace(tokens, d, f, experts, topk).total;
  return MMBO_OK;
}

int mmbo_moe(int dtype, size_t tokens, size_t d, size_t f, size_t experts, size_t topk, int renorm, int group, int zeros,
             const void* X, size_t ldx, const void* router, size_t ldr, const void* gate, const void* up, size_t ldg,
             size_t strideG, const void* down, size_t ldd, size_t strideD, const float* beta, void* Y, size_t ldy,
             int* ids, float* gates, void* workspace, size_t workspaceBytes, void* stream) {
  MMBO_API_LOCK();
  int rc = check_moe_sizes(dtype, tokens, d, f, experts, topk);
  if (rc) return rc;
  if (renorm != 0 && renorm != 1) return MMBO_ERR_BAD_DIM;
  if (group != 0 && (rc = check_w4(dtype, d, f, group, zeros))) return rc;
  if (group == 0 && zeros != 0) return MMBO_ERR_BAD_GROUP;
  if (!beta) return MMBO_ERR_NULL_POINTER;
  if (tokens == 0) return MMBO_OK;
  if (!X || !router || !gate || !up || !down || !Y || !workspace) return MMBO_ERR_NULL_POINTER;
  if (ldx < d || ldx > 0x7fffffffull) return MMBO_ERR_BAD_LDB;
  if (ldy < d || ldy > 0x7fffffffull) return MMBO_ERR_BAD_LDC;
  if (ldr < d || ldr > 0x7fffffffull) return MMBO_ERR_BAD_LDA;
  const W4Format fmt{group, zeros};
  if (group == 0) {
    if (ldg < d || ldd < f || ldg > 0x7fffffffull || ldd > 0x7fffffffull) return MMBO_ERR_BAD_LDA;
    if (experts > 1 && (strideG < (f - 1) * ldg + d || strideD < (d - 1) * ldd + f)) return MMBO_ERR_BAD_LDA;
    if (!aligned_to(gate, 2) || !aligned_to(up, 2) || !aligned_to(down, 2)) return MMBO_ERR_MISALIGNED;
  } else {
    if (experts > 1 && (strideG < w4_total_bytes(f, d, fmt) || strideD < w4_total_bytes(d, f, fmt)))
      return MMBO_ERR_BAD_LDA;
    if (!aligned_to(gate, 16) || !aligned_to(up, 16) || !aligned_to(down, 16)) return MMBO_ERR_MISALIGNED;
    if (experts > 1 && (strideG % 16 != 0 || strideD % 16 != 0)) return MMBO_ERR_MISALIGNED;
  }
  if (!aligned_to(X, 2) || !aligned_to(router, 2) || !aligned_to(Y, 2) || !aligned_to(ids, 4) ||
      !aligned_to(gates, 4) || !aligned_to(workspace, 256))
    return MMBO_ERR_MISALIGNED;
  const MoeWorkspace ws = moe_workspace(tokens, d, f, experts, topk);
  if (workspaceBytes < ws.total) return MMBO_ERR_WORKSPACE;
  char* base = static_cast<char*>(workspace);
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  const size_t pass = moe_pass_tokens((int)topk);
  for (size_t t0 = 0; t0 < tokens; t0 += pass) {
    const size_t n = tokens - t0 < pass ? tokens - t0 : pass;
    MoeArgs a{};
    a.tokens = (int)n;
    a.d = (int)d;
    a.f = (int)f;
    a.experts = (int)experts;
    a.topk = (int)topk;
    a.renorm = renorm;
    a.fmt = fmt;
    a.X = static_cast<const char*>(X) + t0 * ldx * 2;
    a.router = router;
    a.gate = gate;
    a.up = up;
    a.down = down;
    a.ldx = ldx;
    a.ldr = ldr;
    a.ldg = ldg;
    a.strideG = strideG;
    a.ldd = ldd;
    a.strideD = strideD;
    a.beta = *beta;
    a.Y = static_cast<char*>(Y) + t0 * ldy * 2;
    a.ldy = ldy;
    a.ids = ids ? ids + t0 * topk : nullptr;
    a.gates = gates ? gates + t0 * topk : nullptr;
    a.scores = reinterpret_cast<float*>(base + ws.scores);
    a.x = base + ws.x;
    a.hidden = base + ws.hidden;
    a.plan = reinterpret_cast<int*>(base + ws.plan);
    a.d_pad = (int)align_up(d, 128);
    a.f_pad = (int)align_up(f, 128);
    rc = dtype == MMBO_DTYPE_F16 ? run_moe<__half>(a, st) : run_moe<__nv_bfloat16>(a, st);
    if (rc) return rc;
  }
  return MMBO_OK;
}

}  // extern "C"
