// Packed 4-bit weights times many columns of activations, on the fifth-generation tensor cores.
//
// A block computes 128 rows x NT columns.  The weights never exist in 16 bits outside tensor memory:
//   warp 0      feeds: TMA loads of the packed tiles (8 row blocks in one) and of the activations (128 x NT) into a ring
//   warp 1      issues the products: A (the unpacked weights) from tensor memory, B (the activations) from shared memory
//   unpackers   (4 or 8 warps) turn codes into exact integers q - z (bfloat16: times 2^-11, see W4Operand) in the activations'
//               type and write them to tensor memory, thread = row; where the activations are not aligned for TMA they bring
//               those, too
//   drainers    (4 or 8 warps) take each group's sums out of tensor memory, multiply by the group's scale and add them to
//               the tile's sums in fp32 registers: the scales never meet a 16-bit rounding
// Bounds: with few columns the codes' bytes (a 128 x 128 tile is 8.4 KB, 365 cycles of an SM's share of the memory); with
// many the tensor pipe (a tile times 128 columns is 512 cycles) beside the unpacking (16 words a thread and tile, 9 to 11
// instructions each) and shared memory (activations are written and read once a tile: 512 cycles at 128 columns).
// A from tensor memory rather than from shared memory: its 32 KB a tile would have to be written and read there too.
#pragma once

#include "w4_gemv.cuh"

namespace mmbo {

// 32 lanes x 32 consecutive 32-bit columns of tensor memory, thread t of the warp writing lane (base lane + t).
__device__ __forceinline__ void tmem_st_32x32(uint32_t taddr, const uint32_t (&r)[32]) {
  asm volatile(
      "tcgen05.st.sync.aligned.32x32b.x32.b32 [%0], "
      "{%1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15, %16, "
      "%17, %18, %19, %20, %21, %22, %23, %24, %25, %26, %27, %28, %29, %30, %31, %32};" ::"r"(taddr),
      "r"(r[0]), "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7]), "r"(r[8]), "r"(r[9]),
      "r"(r[10]), "r"(r[11]), "r"(r[12]), "r"(r[13]), "r"(r[14]), "r"(r[15]), "r"(r[16]), "r"(r[17]), "r"(r[18]),
      "r"(r[19]), "r"(r[20]), "r"(r[21]), "r"(r[22]), "r"(r[23]), "r"(r[24]), "r"(r[25]), "r"(r[26]), "r"(r[27]),
      "r"(r[28]), "r"(r[29]), "r"(r[30]), "r"(r[31])
      : "memory");
}
__device__ __forceinline__ void tmem_st_wait() { asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory"); }

// D[tmem] (+)= A[tmem] * B[smem desc]; issued by one thread.
__device__ __forceinline__ void umma_ts_f16(uint32_t tmem_d, uint32_t tmem_a, uint64_t desc_b, uint32_t idesc,
                                            uint32_t accumulate) {
  asm volatile(
      "{\n\t"
      ".reg .pred p;\n\t"
      "setp.ne.b32 p, %4, 0;\n\t"
      "tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], %2, %3, p;\n\t"
      "}\n" ::"r"(tmem_d),
      "r"(tmem_a), "l"(desc_b), "r"(idesc), "r"(accumulate)
      : "memory");
}

// Wait by a whole warp with one answer for all of it.
__device__ __forceinline__ bool mbar_wait_together(uint32_t bar, uint32_t parity, volatile uint32_t* abort_flag,
                                                   unsigned int fault_code, unsigned int detail) {
  return __all_sync(0xffffffffu, mbar_wait_asleep(bar, parity, abort_flag, fault_code, detail));
}

struct UmmaArgs {
  size_t m, n, k, ldb, ldc;
  float alpha, beta;
  const unsigned char* packed;
  const void* B;
  void* C;
  int split_log2;  // blocks of a cluster, which cut k (then every cluster has one tile)
  int x_tma;       // the activations are aligned for TMA
  int stages;
  int tiles, col_tiles;
};

// NT: columns of a tile (32, 64 or 128).
template <int NT>
struct UmmaShape {
  static constexpr int kUnpackSets = NT <= 64 ? 2 : 1;   // sets of four unpacking warps, taking tiles in turn
  static constexpr int kDrainers = NT <= 64 ? 4 : 8;     // warps; beyond four they share the columns
  static constexpr int kThreads = (4 + 4 * kUnpackSets + kDrainers) * 32;
  static constexpr int kDrainCols = NT * 4 / kDrainers;  // of a draining warp
  static constexpr int kSums = 256 / NT > 4 ? 4 : 256 / NT;  // group sums in tensor memory at a time
  static constexpr int kXBytes = NT * 256;               // activations of a k-tile
};
constexpr int kUmmaMaxStages = 10;
constexpr int kUmmaASlots = 4;  // unpacked tiles in tensor memory, 64 columns each
// Packed tiles of a stage, in the order of the row blocks; TMA wants its destination on a 128-byte boundary.
__host__ __device__ constexpr uint32_t umma_code_bytes(uint32_t tile_bytes) { return (8 * tile_bytes + 127) / 128 * 128; }

template <typename T, int NT, int QG, bool ZEROS>
__global__ void __launch_bounds__(UmmaShape<NT>::kThreads, 1)
    w4_umma_kernel(const UmmaArgs a, const __grid_constant__ CUtensorMap w_map, const __grid_constant__ CUtensorMap x_map) {
  using S = UmmaShape<NT>;
  using L = W4Tile<QG, ZEROS>;
  constexpr uint32_t TILE = L::kBytes, CODES = umma_code_bytes(TILE);
  constexpr int G = 4 / QG;
  extern __shared__ unsigned char smem_raw[];
  __shared__ __align__(8) unsigned long long full_bars[kUmmaMaxStages], empty_bars[kUmmaMaxStages];
  __shared__ __align__(8) unsigned long long a_full[kUmmaASlots], a_empty[kUmmaASlots], d_full[S::kSums], d_empty[S::kSums];
  __shared__ uint32_t abort_flag, tmem_slot;
  const int warp = __shfl_sync(0xffffffffu, (int)threadIdx.x / 32, 0), lane = threadIdx.x & 31;
  const int split = 1 << a.split_log2, rank = blockIdx.x & (split - 1);
  const int k_tiles = (int)w4_k_tiles(a.k), row_blocks = (int)w4_row_blocks(a.m);
  const int t0 = (int)(((long long)k_tiles * rank) >> a.split_log2);
  const int span = (int)(((long long)k_tiles * (rank + 1)) >> a.split_log2) - t0;
  const int first = blockIdx.x >> a.split_log2, step = gridDim.x >> a.split_log2;
  const uint32_t smem = (smem_u32(smem_raw) + 1023u) & ~1023u;
  const uint32_t codes_at = smem + a.stages * S::kXBytes;
  float* received = reinterpret_cast<float*>(smem_raw + (codes_at + a.stages * CODES - smem_u32(smem_raw)));

  if (threadIdx.x == 0) {
    abort_flag = 0;
    for (int s = 0; s < a.stages; ++s) {
      mbar_init(smem_u32(&full_bars[s]), 1);
      mbar_init(smem_u32(&empty_bars[s]), 5);  // four unpackers and the products
    }
    for (int i = 0; i < kUmmaASlots; ++i) {
      mbar_init(smem_u32(&a_full[i]), 4);
      mbar_init(smem_u32(&a_empty[i]), 1);
    }
    for (int i = 0; i < S::kSums; ++i) {
      mbar_init(smem_u32(&d_full[i]), 1);
      mbar_init(smem_u32(&d_empty[i]), S::kDrainers);
    }
  }
  fence_mbar_init();
  if (warp == 1) {
    tmem_alloc<1>(smem_u32(&tmem_slot), 512);
    tmem_relinquish<1>();
  }
  if (warp == 0 && first < a.tiles) {  // the first tiles, brought into L2 while the kernel in front finishes
    const int block = first / a.col_tiles * 8 + (lane & 7), cnt = min(span, a.stages);
    if (lane < 8 && block < row_blocks && cnt > 0)
      bulk_prefetch(a.packed + ((size_t)block * k_tiles + t0) * TILE, cnt * TILE);
    if (lane == 8 && span > 0) prefetch_tensormap(&w_map);  // (no map where k is 0)
    if (lane == 9 && a.x_tma) prefetch_tensormap(&x_map);
  }
  tcgen05_fence_before();
  __syncthreads();
  tcgen05_fence_after();
  const uint32_t tmem = __shfl_sync(0xffffffffu, tmem_slot, 0);
  const uint32_t a_cols = tmem + 256;  // group sums in columns 0 .. 255, four tiles of weights in 256 .. 511
  if (split > 1) cluster_arrive();
  griddep_launch_dependents();
  griddep_wait();

  bool ok = true;
  if (warp == 0) {
    // ---- feeder (one elected lane, for the same reason as below)
    int stage = 0;
    uint32_t phase = 0;
    for (int tile = first; ok && tile < a.tiles; tile += step) {
      const int row_tile = tile / a.col_tiles, col0 = (tile - row_tile * a.col_tiles) * NT;
      for (int i = 0; ok && i < span; ++i) {
        ok = mbar_wait_together(smem_u32(&empty_bars[stage]), phase ^ 1u, &abort_flag, kFaultWaitEmpty, 0x4c00u + stage);
        if (!ok) break;
        if (elect_one()) {
          const uint32_t bar = smem_u32(&full_bars[stage]), x = smem + stage * S::kXBytes;
          mbar_expect_tx(bar, 8 * TILE + (a.x_tma ? S::kXBytes : 0));
          tma_load_3d(codes_at + stage * CODES, &w_map, bar, 0, t0 + i, row_tile * 8);
          if (a.x_tma) {
            tma_load_2d(x, &x_map, bar, (t0 + i) * kW4Cols, col0);
            tma_load_2d(x + NT * 128, &x_map, bar, (t0 + i) * kW4Cols + 64, col0);
          }
        }
        __syncwarp();
        if (++stage == a.stages) {
          stage = 0;
          phase ^= 1u;
        }
      }
    }
  } else if (warp == 1) {
    // ---- products.  The whole warp walks the loop and one elected lane issues: what the instructions take (uniform
    // registers) then comes from uniform arithmetic; under `if (lane == 0)` each cost 100 cycles to get ready.
    constexpr uint32_t idesc = make_idesc(std::is_same<T, __half>::value ? 0u : 1u, 0u, 0u, 128u, (uint32_t)NT);
    int stage = 0;
    uint32_t phase = 0, sums = 0, done = 0;
    for (int tile = first; ok && tile < a.tiles; tile += step)
      for (int i = 0; ok && i < span; ++i, ++done) {
        const uint32_t slot = done % kUmmaASlots, slot_phase = done / kUmmaASlots & 1u;
        // one answer of the barrier unit takes 60 cycles: ask all three before looking at any
        const uint32_t d0 = sums % S::kSums;
        const bool ready = mbar_try_wait(smem_u32(&a_full[slot]), slot_phase) & mbar_try_wait(smem_u32(&full_bars[stage]), phase) &
                           mbar_try_wait(smem_u32(&d_empty[d0]), ((sums / S::kSums) & 1u) ^ 1u);
        bool asked = __all_sync(0xffffffffu, ready);
        if (!asked)
          ok = mbar_wait_together(smem_u32(&a_full[slot]), slot_phase, &abort_flag, kFaultWaitFull, 0x4c10u) &&
               mbar_wait_together(smem_u32(&full_bars[stage]), phase, &abort_flag, kFaultWaitFull, 0x4c11u);
        if (!ok) break;
        const uint64_t desc = make_smem_desc_sw128(smem + stage * S::kXBytes, 16u, 1024u);
#pragma unroll
        for (int g = 0; g < G; ++g, ++sums) {
          const uint32_t d = sums % S::kSums;
          if (!(g == 0 && asked))
            ok = mbar_wait_together(smem_u32(&d_empty[d]), ((sums / S::kSums) & 1u) ^ 1u, &abort_flag, kFaultWaitTmemEmpty,
                                    0x4c12u);
          if (!ok) break;
          tcgen05_fence_after();
          if (elect_one()) {
#pragma unroll
            for (int j = 0; j < 2 * QG; ++j) {
              const int step16 = g * 2 * QG + j;  // of the tile's eight steps of 16; four to a 64-column half
              umma_ts_f16(tmem + d * NT, a_cols + slot * 64 + step16 * 8,
                          desc + (((step16 >> 2) * (NT * 128) + (step16 & 3) * 32) >> 4), idesc, j > 0);
            }
            umma_commit(smem_u32(&d_full[d]));
            if (g == G - 1) {
              umma_commit(smem_u32(&a_empty[slot]));
              umma_commit(smem_u32(&empty_bars[stage]));
            }
          }
          __syncwarp();
        }
        if (!ok) break;
        if (++stage == a.stages) {
          stage = 0;
          phase ^= 1u;
        }
      }
  } else if (warp >= 4 && warp < 4 + 4 * S::kUnpackSets) {
    // ---- unpackers: thread = row of the tile.  A set skips phases of the ring's barriers, those of the other set's tiles.  It
    // cannot take an older phase for its own: tile i - kUnpackSets had its place in tensor memory only after the products of
    // the tile kUmmaASlots before it, so what was loaded up to there is complete, and the ring has that many stages or more.
    const int set = (warp - 4) / 4, row = (warp & 3) * 32 + lane, r = row & 15;
    const uint32_t lane_base = (uint32_t)((warp & 3) * 32) << 16;
    int stage = set % a.stages;
    uint32_t phase = (uint32_t)(set / a.stages) & 1u;
    const int total = first < a.tiles ? ((a.tiles - first + step - 1) / step) * span : 0;
    for (int i = set; ok && i < total; i += S::kUnpackSets) {
      const uint32_t slot = (uint32_t)i % kUmmaASlots;
      ok = mbar_wait_together(smem_u32(&full_bars[stage]), phase, &abort_flag, kFaultWaitFull, 0x4c30u) &&
           mbar_wait_together(smem_u32(&a_empty[slot]), ((uint32_t)i / kUmmaASlots & 1u) ^ 1u, &abort_flag, kFaultWaitEmpty, 0x4c31u);
      if (!ok) break;
      tcgen05_fence_after();
      const uint32_t block = codes_at + stage * CODES + (row >> 4) * TILE;
      uint4 c[4];
#pragma unroll
      for (int t = 0; t < 4; ++t) c[t] = lds128(block + w4_piece(r, t));
      uint32_t z[G];
#pragma unroll
      for (int g = 0; g < G; ++g) {
        z[g] = 8u;
        if (ZEROS) asm volatile("ld.shared.u8 %0, [%1];" : "=r"(z[g]) : "r"(block + L::kZeros + g * 16 + W4Format::slot(r)));
      }
      W4Operand<T> un;
#pragma unroll
      for (int half = 0; half < 2; ++half) {
        uint32_t w[32];
#pragma unroll
        for (int uu = 0; uu < 2; ++uu) {
          const int u = half * 2 + uu;
          un.set_zero(z[u / QG] & 15u);
#pragma unroll
          for (int t = 0; t < 4; ++t)
            un.unpack(u == 0 ? c[t].x : u == 1 ? c[t].y : u == 2 ? c[t].z : c[t].w, &w[uu * 16 + t * 4]);
        }
        tmem_st_32x32(a_cols + slot * 64 + half * 32 + lane_base, w);
      }
      if (!a.x_tma) {
        // 16-byte chunks of 128 elements of a column, four under way at a time
        const int tile = first + i / span * step, col0 = tile % a.col_tiles * NT;
        unsigned char* xs = smem_raw + (smem + stage * S::kXBytes - smem_u32(smem_raw));
#pragma unroll 1
        for (int p0 = (warp & 3) * 32 + lane; p0 < NT * 16; p0 += 512) {
          Load8 l[4];
#pragma unroll
          for (int b = 0; b < 4; ++b) {
            const int p = p0 + b * 128;
            const size_t col = (size_t)col0 + (p >> 4);
            l[b].issue(static_cast<const T*>(a.B) + col * a.ldb, col < a.n ? (long long)a.k : 0,
                       (long long)(t0 + i % span) * kW4Cols + (p & 15) * 8);
          }
#pragma unroll
          for (int b = 0; b < 4; ++b) {
            const int p = p0 + b * 128, row_x = p >> 4, chunk = p & 15;
            const size_t col = (size_t)col0 + row_x;
            *reinterpret_cast<uint4*>(xs + (chunk >> 3) * (NT * 128) + row_x * 128 + (((chunk & 7) ^ (row_x & 7)) << 4)) =
                l[b].finish(static_cast<const T*>(a.B) + col * a.ldb, col < a.n ? (long long)a.k : 0,
                            (long long)(t0 + i % span) * kW4Cols + chunk * 8);
          }
        }
        fence_proxy_async_smem();
      }
      tmem_st_wait();
      tcgen05_fence_before();
      __syncwarp();
      if (lane == 0) {
        mbar_arrive(smem_u32(&a_full[slot]));
        mbar_arrive(smem_u32(&empty_bars[stage]));
      }
      stage += S::kUnpackSets;
      while (stage >= a.stages) {
        stage -= a.stages;
        phase ^= 1u;
      }
    }
  } else if (warp >= 4) {
    // ---- drainers: thread = row of the tile
    const int part = (warp - 4 - 4 * S::kUnpackSets) / 4, row = (warp & 3) * 32 + lane, r = row & 15;
    const uint32_t lane_base = (uint32_t)((warp & 3) * 32) << 16;
    uint32_t sums = 0;
    for (int tile = first; tile < a.tiles; tile += step) {
      const int row_tile = tile / a.col_tiles, col0 = (tile - row_tile * a.col_tiles) * NT + part * S::kDrainCols;
      const int block = row_tile * 8 + (row >> 4);
      const unsigned char* scales = a.packed + ((size_t)min(block, row_blocks - 1) * k_tiles + t0) * TILE + L::kScales +
                                    W4Format::slot(r) * 2;
      float acc[S::kDrainCols];
#pragma unroll
      for (int j = 0; j < S::kDrainCols; ++j) acc[j] = 0.f;
      T next[G];
#pragma unroll
      for (int g = 0; g < G; ++g) next[g] = span > 0 ? *reinterpret_cast<const T*>(scales + g * 32) : from_f32<T>(0.f);
      for (int i = 0; ok && i < span; ++i) {
        T now[G];
#pragma unroll
        for (int g = 0; g < G; ++g) now[g] = next[g];
        scales += TILE;
        if (i + 1 < span) {
#pragma unroll
          for (int g = 0; g < G; ++g) next[g] = *reinterpret_cast<const T*>(scales + g * 32);
        }
#pragma unroll
        for (int g = 0; g < G; ++g, ++sums) {
          const uint32_t d = sums % S::kSums;
          if (ok) ok = mbar_wait_together(smem_u32(&d_full[d]), (sums / S::kSums) & 1u, &abort_flag, kFaultWaitTmemFull, 0x4c40u);
          if (!ok) break;
          tcgen05_fence_after();
          const float s = to_f32(now[g]);
#pragma unroll
          for (int c = 0; c < S::kDrainCols; c += 32) {
            uint32_t v[32];
            tmem_ld_32x32(tmem + d * NT + part * S::kDrainCols + c + lane_base, v);
            tmem_ld_wait();
            if (c + 32 == S::kDrainCols) {
              tcgen05_fence_before();
              __syncwarp();
              if (lane == 0) mbar_arrive(smem_u32(&d_empty[d]));
            }
#pragma unroll
            for (int j = 0; j < 32; ++j) acc[c + j] = fmaf(s, __uint_as_float(v[j]), acc[c + j]);
          }
        }
      }
      const size_t grow = (size_t)row_tile * 128 + row;
      auto store = [&](int col, float v) {
        if (grow < a.m && (size_t)col < a.n) {
          T* c = static_cast<T*>(a.C) + (size_t)col * a.ldc + grow;
          v = v * a.alpha * W4Operand<T>::kUnit;
          *c = from_f32<T>(a.beta != 0.f ? fmaf(a.beta, to_f32(*c), v) : v);
        }
      };
      if (split == 1) {
#pragma unroll
        for (int j = 0; j < S::kDrainCols; ++j) store(col0 + j, acc[j]);
      } else if (S::kDrainers == 4) {
        // every block finishes NT / split of the columns, in the order of the parts of k
        const int share = NT >> a.split_log2;
        cluster_wait();  // all blocks of the cluster are running
        const uint32_t to = smem_u32(received) + (rank * share * 128 + row) * 4;
        const int share_log2 = (NT == 32 ? 5 : 6) - a.split_log2;
#pragma unroll
        for (int j = 0; j < S::kDrainCols; ++j) cluster_store(to + (j & (share - 1)) * 512, j >> share_log2, acc[j]);
        cluster_arrive();
        cluster_wait();
        for (int j = 0; j < share; ++j) {
          float v = received[(size_t)j * 128 + row];
          for (int s = 1; s < split; ++s) v += received[((size_t)s * share + j) * 128 + row];
          store(col0 + rank * share + j, v);
        }
      }
    }
  }
  if (split > 1 && warp < 4 + 4 * S::kUnpackSets) {
    cluster_wait();
    cluster_arrive();
    cluster_wait();
  }
  if (!ok) {  // a wait ran out: give copies and products still in flight time to land
    const uint64_t since = global_timer_ns();
    while (global_timer_ns() - since < MMBO_DRAIN_LIMIT_NS) __nanosleep(1000);
  }
  tcgen05_fence_before();
  __syncthreads();
  tcgen05_fence_after();
  if (warp == 1) tmem_dealloc<1>(tmem, 512);
}

}  // namespace mmbo
