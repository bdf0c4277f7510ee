// Packed 4-bit weights times up to 8 columns of activations.
//
// What bounds it: the codes, read once (0.53 bytes a weight); for small matrices the latency of one trip to memory.  8192 x 28672,
// one column, fp16: 29.7 us a call (121 MB, 4.1 TB/s; 140 warp instructions a tile at 2.0 a cycle).
//   - Every multiplying warp has a ring of tiles in shared memory, which a lane of the feeding warp fills with bulk
//     copies: the copies in flight cost no registers and no instructions of the warps that multiply.  (With each warp
//     filling its own ring the copies' issue cost 500 cycles a slot: 32 us at 8192 x 28672, one column, where the fed rings took
//     27; both with zero points taken off the sums, two us faster than off the codes.)
//   - One block per SM, persistent over its row blocks, so the rings run on from one to the next.
//   - The activations of the block's share of k sit in shared memory, staged once.
//   - Each warp keeps its partial sums of every row block in shared memory; they are joined at the end, over the warps
//     that split k within a block and over the blocks of a cluster (distributed shared memory), in a fixed order: the
//     same bits every time, and no scratch memory.
//   - Before it waits for the kernel in front of it the feeding warp asks L2 for its first tiles.
// The products run on mma.sync.m16n8k16: with at most 8 columns its rate is ample (a tile takes 8 instructions of 8
// cycles, on four schedulers, in the 45 cycles its bytes take), and its fragments come straight from the packed order
// without a trip through tensor memory.  (With 16 columns the kernel of w4_umma.cuh is ahead at 8192 x 8192, 17 us against 23;
// with 8 this one is, 13.3 against 16.9 for 9.  Over few rows this one stays ahead for longer, since it spreads a row block over
// up to 64 warps: 1024 x 8192 takes 5.8 us with 8 columns and 9.3 with 9.)
#pragma once

#include <type_traits>

#include "ptx.cuh"
#include "w4.cuh"

namespace mmbo {


// c (16 x 8) = a (16 x 16) * b (16 x 8) + c (or + 0), fp32 sums, operands of type T.
template <typename T>
__device__ __forceinline__ void mma_16816(float (&c)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0,
                                          uint32_t b1) {
  if constexpr (std::is_same<T, __half>::value)
    asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
        : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
        : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
  else
    asm("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
        : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
        : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}
template <typename T>
__device__ __forceinline__ void mma_16816_from_zero(float (&c)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3,
                                                    uint32_t b0, uint32_t b1) {
  if constexpr (std::is_same<T, __half>::value)
    asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%10, %10, %10, %10};"
        : "=f"(c[0]), "=f"(c[1]), "=f"(c[2]), "=f"(c[3])
        : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1), "f"(0.f));
  else
    asm("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%10, %10, %10, %10};"
        : "=f"(c[0]), "=f"(c[1]), "=f"(c[2]), "=f"(c[3])
        : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1), "f"(0.f));
}

__device__ __forceinline__ uint4 lds128(uint32_t addr) {
  uint4 v;
  asm volatile("ld.shared.v4.u32 {%0, %1, %2, %3}, [%4];" : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w) : "r"(addr));
  return v;
}
__device__ __forceinline__ uint32_t lds32(uint32_t addr) {
  uint32_t v;
  asm volatile("ld.shared.u32 %0, [%1];" : "=r"(v) : "r"(addr));
  return v;
}
__device__ __forceinline__ uint32_t lds16(uint32_t addr) {
  uint16_t v;
  asm volatile("ld.shared.u16 %0, [%1];" : "=h"(v) : "r"(addr));
  return v;
}
// acc += the products of a tile with 128 rows of 8 columns, PARTS of them added (a vector kept as a value and its remainder):
// column(i, q) is this lane's 16 bytes of quarter q of its column in part i.  U: type of the columns, T: of the scales.  Sums
// are W4Operand<U>::kUnit times too small.
//
// Every code becomes the exact difference q - z before it is multiplied, so that an error is measured by the terms
// |q - z| |x| of the formula: a large activation at a weight of zero drops out.  (Taking z times the sum of x off a group's
// sum of q x saves four of nine instructions a word, but leaves that activation's rounding behind.)
template <typename U, typename T, int QG, int PARTS = 1, typename Columns>
__device__ __forceinline__ void w4_tile_mma(uint32_t tile, Columns column, bool zeros, float (&acc)[4]) {
  using L = W4Tile<QG, true>;  // (where there are zero points does not depend on whether there are)
  const int lane = threadIdx.x & 31, r = lane >> 2;
  const uint32_t codes = tile + w4_piece(r, lane & 3);
  const uint4 c0 = lds128(codes), c1 = lds128(codes + 512);  // rows r and r + 8
  const uint32_t w0[4] = {c0.x, c0.y, c0.z, c0.w}, w1[4] = {c1.x, c1.y, c1.z, c1.w};
  W4Operand<U> lo, hi;
#pragma unroll
  for (int g = 0; g < L::kGroups; ++g) {
    const uint32_t z = zeros ? lds16(tile + L::kZeros + g * 16 + r * 2) : 0x0808u;
    lo.set_zero(z & 15u);
    hi.set_zero(z >> 8 & 15u);
    float part[PARTS][4];
#pragma unroll
    for (int qq = 0; qq < QG; ++qq) {
      const int q = g * QG + qq;
      uint32_t p[4], s[4];
      lo.unpack(w0[q], p);
      hi.unpack(w1[q], s);
#pragma unroll
      for (int i = 0; i < PARTS; ++i) {
        const uint4 b = column(i, q);
        if (qq == 0) mma_16816_from_zero<U>(part[i], p[0], s[0], p[1], s[1], b.x, b.y);
        else mma_16816<U>(part[i], p[0], s[0], p[1], s[1], b.x, b.y);
        mma_16816<U>(part[i], p[2], s[2], p[3], s[3], b.z, b.w);
      }
    }
    const float2 s = widen2<T>(lds32(tile + L::kScales + g * 32 + r * 4));
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      float sum = part[0][i];
#pragma unroll
      for (int j = 1; j < PARTS; ++j) sum += part[j][i];
      acc[i] = fmaf(i < 2 ? s.x : s.y, sum, acc[i]);
    }
  }
}

constexpr int kGemvWarps = 16;                       // that multiply
constexpr int kGemvThreads = (kGemvWarps + 1) * 32;  // and one that feeds them
constexpr int kGemvMaxSlots = 4;
// Barrier of the multiplying warps.  Loops in front of it may have split a warp, which has to arrive as one.
__device__ __forceinline__ void workers_sync() {
  __syncwarp();
  asm volatile("bar.sync 1, %0;" ::"n"(kGemvWarps * 32) : "memory");
}

// Untiled bulk copy, completion on an mbarrier of this CTA (addresses and size multiples of 16 bytes), and the request
// to have the bytes brought into L2.
__device__ __forceinline__ void bulk_load(uint32_t dst, const void* src, uint32_t bytes, uint32_t bar) {
  asm volatile("cp.async.bulk.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1], %2, [%3];" ::"r"(dst),
               "l"(src), "r"(bytes), "r"(bar)
               : "memory");
}
__device__ __forceinline__ void bulk_prefetch(const void* src, uint32_t bytes) {
  asm volatile("cp.async.bulk.prefetch.L2.global [%0], %1;" ::"l"(src), "r"(bytes) : "memory");
}

// Bounded wait that sleeps in the barrier unit instead of polling: the polls of waiting warps would cost the working ones
// issue slots.  A first try without a time to sleep: where the phase has passed already, the sleeping form takes 300
// cycles to say so.  Then 200 tries of at most 10 ms each.
__device__ __forceinline__ bool mbar_wait_asleep(uint32_t bar, uint32_t parity, volatile uint32_t* abort_flag,
                                                 unsigned int fault_code, unsigned int detail) {
  if (mbar_try_wait(bar, parity)) return true;
#pragma unroll 1
  for (int i = 0; i < 200; ++i) {
    uint32_t done;
    asm volatile(
        "{\n\t"
        ".reg .pred p;\n\t"
        "mbarrier.try_wait.parity.shared::cta.b64 p, [%1], %2, %3;\n\t"
        "selp.u32 %0, 1, 0, p;\n\t"
        "}\n"
        : "=r"(done)
        : "r"(bar), "r"(parity), "r"(10000000u)
        : "memory");
    if (done) return true;
    if (*abort_flag) return false;
  }
  report_fault(fault_code, detail);
  *abort_flag = 1u;
  return false;
}

// Cluster barrier in its two halves, which a warp passes as one, and a store to the same place in another block's shared
// memory.
__device__ __forceinline__ void cluster_arrive() {
  __syncwarp();
  asm volatile("barrier.cluster.arrive.release.aligned;" ::: "memory");
}
__device__ __forceinline__ void cluster_wait() {
  __syncwarp();
  asm volatile("barrier.cluster.wait.acquire.aligned;" ::: "memory");
}
__device__ __forceinline__ void cluster_store(uint32_t addr, uint32_t rank, float v) {
  asm volatile("st.shared::cluster.f32 [%0], %1;" ::"r"(mapa_shared(addr, rank)), "f"(v) : "memory");
}

// How the work is cut.  The multiplying warps are WM x WK: warp w takes the rows of row block w / WK and the (w % WK)-th
// part of the block's k-tiles.  `split` blocks of a cluster share one set of rows and cut k; a cluster works through row
// groups of WM row blocks: cluster_id, cluster_id + clusters, ...
struct GemvArgs {
  size_t m, n, k, ldb, ldc;
  float alpha, beta;
  const unsigned char* packed;
  const void* B;
  void* C;
  int wk_log2;     // warps that cut k
  int split_log2;  // blocks of a cluster
  int slots;       // slots of a warp's ring
  int slot_tiles;  // consecutive k-tiles in a slot
  int x_tiles;     // k-tiles of activations in shared memory at a time
  int batch;       // row groups whose partial sums are kept before they are joined and stored (split > 1: all)
  int clusters;
};

// Staged columns.
__host__ __device__ inline size_t gemv_x_bytes(size_t n, size_t tiles) { return n * (tiles * 256 + 64); }
// Partial sums of a batch of row groups, and the room for what the other blocks of a cluster hand over.
__host__ __device__ inline size_t gemv_sums_bytes(int wk, int split, size_t n, int batch) {
  const size_t out = (size_t)batch * (kGemvWarps / wk) * kW4Rows * n;
  return (out * wk + (split > 1 ? out : 0)) * 4;
}

template <typename T, int QG, bool ZEROS>
__global__ void __launch_bounds__(kGemvThreads, 1) w4_gemv_kernel(const GemvArgs a) {
  constexpr uint32_t TILE = W4Tile<QG, ZEROS>::kBytes;
  constexpr int kWorkers = kGemvWarps * 32;
  extern __shared__ __align__(128) unsigned char smem[];
  __shared__ __align__(8) unsigned long long full_bars[kGemvWarps * kGemvMaxSlots], empty_bars[kGemvWarps * kGemvMaxSlots];
  __shared__ __align__(8) unsigned long long x_bar;
  __shared__ uint32_t abort_flag;
  const int split = 1 << a.split_log2, rank = blockIdx.x & (split - 1), first = blockIdx.x >> a.split_log2;
  const int warp = threadIdx.x / 32, lane = threadIdx.x & 31, r = lane >> 2, t = lane & 3;
  const int WK = 1 << a.wk_log2, WM = kGemvWarps >> a.wk_log2;
  const int k_tiles = (int)w4_k_tiles(a.k), row_blocks = (int)w4_row_blocks(a.m), n = (int)a.n;
  const int t0 = (int)(((long long)k_tiles * rank) >> a.split_log2);
  const int span = (int)(((long long)k_tiles * (rank + 1)) >> a.split_log2) - t0;
  const int groups = (row_blocks + WM - 1) / WM;
  const int mine = first < groups ? (groups - first + a.clusters - 1) / a.clusters : 0;  // row groups of this cluster

  // shared memory: rings | activations | partial sums | sums from the cluster
  const uint32_t slot_bytes = a.slot_tiles * TILE;
  unsigned char* xs = smem + (size_t)kGemvWarps * a.slots * slot_bytes;
  const uint32_t x_stride = a.x_tiles * 256 + 64;  // columns 64 bytes out of step: conflict-free 16-byte reads
  float* sums = reinterpret_cast<float*>(xs + (size_t)n * x_stride);
  float* received = sums + (size_t)a.batch * kGemvWarps * kW4Rows * n;

  if (threadIdx.x == 0) {
    abort_flag = 0;
    mbar_init(smem_u32(&x_bar), 1);
  }
  if (threadIdx.x < kGemvWarps * kGemvMaxSlots) {
    mbar_init(smem_u32(&full_bars[threadIdx.x]), 1);
    mbar_init(smem_u32(&empty_bars[threadIdx.x]), 1);
  }
  fence_mbar_init();

  // A warp's part of the tiles of a chunk, and its weights for a row group.
  auto part_of = [&](int chunk, int which) {
    return chunk + (int)(((long long)min(a.x_tiles, span - chunk) * which) >> a.wk_log2);
  };
  auto weights_of = [&](int g, int wm, int tile) {
    return a.packed + ((size_t)((first + g * a.clusters) * WM + wm) * k_tiles + t0 + tile) * TILE;
  };
  // Lane w of the last warp serves warp w.
  const int serves = warp == kGemvWarps ? min(lane, kGemvWarps - 1) : warp, wk = serves & (WK - 1), wm = serves >> a.wk_log2;
  if (warp == kGemvWarps && lane < kGemvWarps && mine > 0 && first * WM + wm < row_blocks) {
    const int begin = part_of(0, wk), cnt = min(part_of(0, wk + 1) - begin, a.slots * a.slot_tiles);
    if (cnt > 0) bulk_prefetch(weights_of(0, wm, begin), cnt * TILE);
  }
  __syncthreads();
  if (split > 1) cluster_arrive();
  griddep_launch_dependents();
  griddep_wait();

  // Activations of a chunk of k: requested before the weights, so that they do not queue behind them.
  const bool x_bulk = a.ldb % 8 == 0 && (reinterpret_cast<uintptr_t>(a.B) & 15u) == 0;
  uint32_t x_phase = 0;
  auto request_x = [&](int chunk0) {
    const size_t k0 = (size_t)(t0 + chunk0) * kW4Cols;
    const int pieces = min(span - chunk0, a.x_tiles) * 16;  // of 16 bytes in a column
    const int whole = x_bulk ? (int)min((size_t)pieces, (a.k - min(a.k, k0)) / 8) : 0;
    if (x_bulk && threadIdx.x == 0) {
      mbar_expect_tx(smem_u32(&x_bar), n * whole * 16);
      for (int col = 0; col < n && whole > 0; ++col)
        bulk_load(smem_u32(xs) + col * x_stride, static_cast<const T*>(a.B) + col * a.ldb + k0, whole * 16, smem_u32(&x_bar));
    }
    // what bulk copies cannot bring: four pieces of a thread under way at a time
    int col = whole < pieces ? 0 : n, piece = whole + threadIdx.x;
    while (col < n) {
      Load8 load[4];
      int cols[4], at[4];
#pragma unroll
      for (int i = 0; i < 4; ++i, piece += kWorkers) {
        while (piece >= pieces && col < n) {
          piece -= pieces - whole;
          ++col;
        }
        cols[i] = col;
        at[i] = piece;
        if (col < n) load[i].issue(static_cast<const T*>(a.B) + col * a.ldb, (long long)a.k, (long long)k0 + piece * 8);
      }
#pragma unroll
      for (int i = 0; i < 4; ++i)
        if (cols[i] < n)
          *reinterpret_cast<uint4*>(xs + cols[i] * x_stride + at[i] * 16) =
              load[i].finish(static_cast<const T*>(a.B) + cols[i] * a.ldb, (long long)a.k, (long long)k0 + at[i] * 8);
    }
  };
  if (warp < kGemvWarps) request_x(0);

  const uint32_t full0 = smem_u32(&full_bars[serves * kGemvMaxSlots]), empty0 = smem_u32(&empty_bars[serves * kGemvMaxSlots]);
  const uint32_t ring_at = smem_u32(smem) + serves * a.slots * slot_bytes;
  int slot = 0;
  uint32_t phase = 0;
  if (warp == kGemvWarps) {
    // For each batch of row groups, for each chunk of k, for each row group: the served warp's part of the chunk in
    // pieces of slot_tiles.  This warp takes no part in the barriers of the others.
    uint32_t idle = 0;  // tries of the present wait
    bool more = lane < kGemvWarps;
    for (int batch0 = 0; more && batch0 < mine; batch0 += a.batch) {
      for (int chunk0 = 0; more && chunk0 < span; chunk0 += a.x_tiles) {
        const int begin = part_of(chunk0, wk), end = part_of(chunk0, wk + 1);
        for (int g = batch0; more && g < min(mine, batch0 + a.batch); ++g) {
          const bool have = (first + g * a.clusters) * WM + wm < row_blocks;
          const unsigned char* src = weights_of(g, wm, begin);
          for (int tile = begin; tile < end;) {
            if (!mbar_try_wait(empty0 + slot * 8, phase ^ 1u)) {
              more = !*(volatile uint32_t*)&abort_flag && ++idle <= (1u << 24);
              if (!more) break;  // the others report
              continue;
            }
            idle = 0;
            const int cnt = min(a.slot_tiles, end - tile);
            mbar_expect_tx(full0 + slot * 8, have ? cnt * TILE : 0);
            if (have) bulk_load(ring_at + slot * slot_bytes, src, cnt * TILE, full0 + slot * 8);
            src += cnt * TILE;
            tile += cnt;
            if (++slot == a.slots) {
              slot = 0;
              phase ^= 1u;
            }
          }
        }
      }
    }
    __syncwarp();
    if (split > 1) cluster_wait();
    return;
  }

  bool ok = true;
  // columns past n repeat the last one; their sums are not stored
  const uint32_t x_lane = smem_u32(xs) + min(r, n - 1) * x_stride + t * 16;
  for (int batch0 = 0; batch0 < mine; batch0 += a.batch) {
    const int batch_end = min(mine, batch0 + a.batch);
    for (int chunk0 = 0; chunk0 < span || chunk0 == 0; chunk0 += a.x_tiles) {
      if (span > a.x_tiles || batch0 == 0) {
        if (batch0 + chunk0 > 0) {
          fence_proxy_async_smem();  // bulk copies will overwrite what plain stores left
          workers_sync();
          request_x(chunk0);
        }
        if (x_bulk && ok) ok = mbar_wait_asleep(smem_u32(&x_bar), x_phase, &abort_flag, kFaultWaitCLoad, 0x4b10u);
        x_phase ^= 1u;
        workers_sync();
      }
      const int w0 = part_of(chunk0, wk), w1 = part_of(chunk0, wk + 1);
      for (int g = batch0; g < batch_end; ++g) {
        float acc[4] = {0.f, 0.f, 0.f, 0.f};
        for (int tile = w0; tile < w1; tile += a.slot_tiles) {
          if (ok) ok = mbar_wait_asleep(full0 + slot * 8, phase, &abort_flag, kFaultWaitFull, 0x4b00u + warp);
          const int cnt = min(a.slot_tiles, w1 - tile);
          uint32_t at = ring_at + slot * slot_bytes, x = x_lane + (tile - chunk0) * 256;
#pragma unroll 2
          for (int i = 0; i < cnt; ++i) {
            w4_tile_mma<T, T, QG>(at, [&](int, int q) { return lds128(x + q * 64); }, ZEROS, acc);
            at += TILE;
            x += 256;
          }
          __syncwarp();
          if (lane == 0) mbar_arrive(empty0 + slot * 8);
          if (++slot == a.slots) {
            slot = 0;
            phase ^= 1u;
          }
        }
        // [row group][warp][column][row]
        float* out = sums + (size_t)(((g - batch0) * kGemvWarps + warp) * n) * kW4Rows;
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const int col = t * 2 + (i & 1), row = r + 8 * (i >> 1);
          if (col < n) {
            float* o = out + col * kW4Rows + row;
            *o = chunk0 == 0 ? acc[i] : *o + acc[i];
          }
        }
      }
    }

    // Join the partial sums and store: over the warps that share rows, then over the cluster.  An output is named by its
    // unit (row group, row block, column) and row; every block of a cluster finishes 16 / split of the rows, the others
    // hand it their sums through its shared memory.
    workers_sync();
    const int units = (batch_end - batch0) * WM * n;
    auto warp_sum = [&](int group_block, int col, int row) {  // group_block: row group * WM + row block
      const float* p = sums + ((size_t)(group_block << a.wk_log2) * n + col) * kW4Rows + row;
      float v = p[0];
      for (int w = 1; w < WK; ++w) v += p[(size_t)w * n * kW4Rows];
      return v;
    };
    auto store = [&](int group_block, int col, int row, float v) {
      const int g = group_block >> (4 - a.wk_log2), b = group_block & (WM - 1);
      const size_t grow = ((size_t)(first + (batch0 + g) * a.clusters) * WM + b) * kW4Rows + row;
      if (grow >= a.m) return;
      T* c = static_cast<T*>(a.C) + col * a.ldc + grow;
      v = v * a.alpha * W4Operand<T>::kUnit;
      *c = from_f32<T>(a.beta != 0.f ? fmaf(a.beta, to_f32(*c), v) : v);
    };
    // thread i: row i % 16 of the units i / 16, i / 16 + 32, ...; unit = group_block * n + column, kept without divisions
    const int row = threadIdx.x & 15;
    int col = threadIdx.x >> 4, gb = 0;
    auto settle = [&]() {
      while (col >= n) {
        col -= n;
        ++gb;
      }
    };
    settle();
    if (split == 1) {
      for (int u = threadIdx.x >> 4; u < units; u += kWorkers / 16, col += kWorkers / 16, settle())
        store(gb, col, row, warp_sum(gb, col, row));
      if (batch_end < mine) workers_sync();
    } else {
      const int share = kW4Rows >> a.split_log2, owner = row >> (4 - a.split_log2);  // rows of an owner
      cluster_wait();  // all blocks of the cluster are running
      for (int u = threadIdx.x >> 4; u < units; u += kWorkers / 16, col += kWorkers / 16, settle())
        cluster_store(smem_u32(received + ((size_t)u * split + rank) * share + (row & (share - 1))), owner,
                      warp_sum(gb, col, row));
      cluster_arrive();
      cluster_wait();
      const int per = kWorkers >> (4 - a.split_log2);  // units of a round
      gb = 0;
      col = threadIdx.x >> (4 - a.split_log2);
      settle();
      for (int u = threadIdx.x >> (4 - a.split_log2); u < units; u += per, col += per, settle()) {
        const float* p = received + (size_t)u * split * share + (threadIdx.x & (share - 1));
        float v = p[0];
        for (int s = 1; s < split; ++s) v += p[s * share];
        store(gb, col, rank * share + (threadIdx.x & (share - 1)), v);
      }
    }
  }
  if (!ok) {  // a wait ran out: give the copies still in flight time to land before the block's memory goes
    const uint64_t since = global_timer_ns();
    while (global_timer_ns() - since < MMBO_DRAIN_LIMIT_NS) __nanosleep(1000);
  }
}

}  // namespace mmbo
