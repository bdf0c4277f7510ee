// 4-bit weights with group scales: the packed format, the kernels that write and read it, and the product of a packed
// matrix with columns of 16-bit activations.
//
//   W(i, j) = (q(i, j) - z(i, g)) * s(i, g),   g = j / group,   q and z in 0..15   (z = 8 where no zero points are kept)
//   C = alpha * W * B + beta * C               W is m x k, B is k x n, C is m x n, column-major
//
// Packed format.  Rows are taken in blocks of 16 and columns in tiles of 128; the tiles of one row block follow one
// another, so that whoever walks along k reads one contiguous stream.  A tile is
//     1024 bytes of codes          row r (0..15) at 64 r; within a row, 16 bytes for each of four "lanes" t, holding one
//                                  32-bit word for each quarter u of the tile: the columns 32 u + 8 t .. + 7.  Lane t's
//                                  piece lies at place t ^ (r / 2 % 4), so that both ways of reading a tile from shared
//                                  memory, four lanes a row and one lane a row, touch every bank once
//     (128 / group) x 16 scales    in the activations' type, group by group, rows in the order 0, 8, 1, 9, .. 7, 15
//     (128 / group) x 16 bytes     zero points in the same order, where the matrix has them
// In a word, columns 0 .. 7 sit in nibbles 0, 4, 2, 6, 1, 5, 3, 7: with v = w >> 8, the registers w & 0x000f000f,
// v & 0x000f000f, w & 0x00f000f0 and v & 0x00f000f0 hold the pairs (0, 1), (2, 3), (4, 5), (6, 7), one code in each half,
// ready to be read as two 16-bit floats.  With this order the four words of
// a lane are the four pairs of k-steps a 16-row matrix instruction wants from that lane, one 16-byte load serves a
// whole tile row, no k-step spans two groups (groups are 32, 64 or 128 wide), and the scales of the two rows r and
// r + 8 whose sums a lane holds come with one load.
// Rows past m and columns past k hold the code of weight zero.
#pragma once

#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_runtime.h>
#include <stdint.h>

#include "ref_kernels.cuh"

namespace mmbo {

constexpr int kW4Rows = 16;    // rows of a block
constexpr int kW4Cols = 128;   // columns of a tile
constexpr int kW4Codes = 1024; // bytes of codes in a tile

struct W4Format {
  int group, zeros;
  __host__ __device__ int groups() const { return kW4Cols / group; }
  __host__ __device__ uint32_t tile_bytes() const { return kW4Codes + groups() * (kW4Rows * 2 + (zeros ? kW4Rows : 0)); }
  // places of the scale and the zero point of row r, group g within a tile
  __host__ __device__ uint32_t scale_at(int g, int r) const { return kW4Codes + (g * kW4Rows + slot(r)) * 2; }
  __host__ __device__ uint32_t zero_at(int g, int r) const { return kW4Codes + groups() * kW4Rows * 2 + g * kW4Rows + slot(r); }
  __host__ __device__ static int slot(int r) { return 2 * (r & 7) + (r >> 3); }
};
__host__ __device__ constexpr int w4_piece(int r, int t) { return r * 64 + (t ^ ((r >> 1) & 3)) * 16; }  // lane t of row r
__host__ __device__ constexpr int w4_nibble(int column) {  // of one of a word's eight columns
  return (column >> 2) + 2 * ((column >> 1) & 1) + 4 * (column & 1);
}
__host__ __device__ inline size_t w4_row_blocks(size_t m) { return (m + kW4Rows - 1) / kW4Rows; }
__host__ __device__ inline size_t w4_k_tiles(size_t k) { return (k + kW4Cols - 1) / kW4Cols; }

// ---------------------------------------------------------------- 16-bit types --------
template <>
__device__ __forceinline__ float to_f32<__nv_bfloat16>(__nv_bfloat16 v) { return __bfloat162float(v); }
template <>
__device__ __forceinline__ __nv_bfloat16 from_f32<__nv_bfloat16>(float v) { return __float2bfloat16_rn(v); }

// Elements at .. at + 7 of an array of `len`, zero behind its end, as they lie in memory; the array starts on any 2-byte
// boundary.  Off the 16-byte boundaries two aligned loads are shifted together (eight loads of two bytes took four times
// as long); nothing outside the array is read.  In two steps, so that several can be under way at a time.
struct Load8 {
  uint4 u, v;
  int off;    // bytes past the boundary
  bool fast;
  template <typename T>
  __device__ __forceinline__ void issue(const T* array, long long len, long long at) {
    const uintptr_t p = reinterpret_cast<uintptr_t>(array + at);
    off = (int)(p & 15u);
    fast = 2 * at >= off && at + (off ? 16 - off / 2 : 8) <= len;
    if (fast) {
      const uint4* q = reinterpret_cast<const uint4*>(p & ~(uintptr_t)15);
      u = q[0];
      if (off) v = q[1];
    }
  }
  template <typename T>
  __device__ __forceinline__ uint4 finish(const T* array, long long len, long long at) const {
    if (fast) {
      if (off == 0) return u;
      const bool two = off & 8, one = off & 4;
      const uint32_t w0 = two ? u.z : u.x, w1 = two ? u.w : u.y, w2 = two ? v.x : u.z, w3 = two ? v.y : u.w,
                     w4 = two ? v.z : v.x, w5 = two ? v.w : v.y;
      const uint32_t a0 = one ? w1 : w0, a1 = one ? w2 : w1, a2 = one ? w3 : w2, a3 = one ? w4 : w3, a4 = one ? w5 : w4;
      const int bits = (off & 2) * 8;
      return make_uint4(__funnelshift_r(a0, a1, bits), __funnelshift_r(a1, a2, bits), __funnelshift_r(a2, a3, bits),
                        __funnelshift_r(a3, a4, bits));
    }
    __align__(16) T e[8];
#pragma unroll
    for (int i = 0; i < 8; ++i) e[i] = at + i < len ? array[at + i] : from_f32<T>(0.f);
    return *reinterpret_cast<const uint4*>(e);
  }
};
template <typename T>
__device__ __forceinline__ uint4 load8(const T* array, long long len, long long at) {
  Load8 l;
  l.issue(array, len, at);
  return l.finish(array, len, at);
}

// ---------------------------------------------------------------- writing the format --
// One warp per tile; lane 4 r + t (r 0..7, t 0..3) owns rows r and r + 8 of the block and, in each quarter u, the
// columns 32 u + 8 t .. + 7: its eight words are two 16-byte stores, and the loads of four lanes are 64 contiguous
// bytes of a row.  One pass, so bound by bytes: 2 m k in, m k / 2 out.
//
// Symmetric: s = max|w| / 7 rounded to the weights' type, z = 8.  With zero points: lo = min(w, 0), hi = max(w, 0),
// s = (hi - lo) / 15 rounded to the weights' type, z = rint(-lo / s).  q = rint(w / s) + z, held to 0..15; ties to
// even.  A group whose scale rounds to zero becomes zeros; one with an infinity or a NaN becomes NaN (its scale is).
template <typename T>
__global__ void w4_quantize_kernel(size_t m, size_t k, W4Format f, const T* __restrict__ W, size_t ldw,
                                   unsigned char* __restrict__ packed) {
  const size_t tiles = w4_k_tiles(k);
  const size_t unit = (size_t)blockIdx.x * (blockDim.x / 32) + threadIdx.x / 32;
  if (unit >= w4_row_blocks(m) * tiles) return;
  const size_t block = unit / tiles, tile = unit % tiles;
  const int lane = threadIdx.x & 31, r = lane >> 2, t = lane & 3;
  unsigned char* out = packed + unit * f.tile_bytes();
  const int per = f.group / 32;  // quarters in a group
#pragma unroll
  for (int half = 0; half < 2; ++half) {
    const int row = r + 8 * half;
    const size_t i = block * kW4Rows + row;
    __align__(16) T w[4][8];
#pragma unroll
    for (int u = 0; u < 4; ++u)
      *reinterpret_cast<uint4*>(w[u]) =
          load8(W + i * ldw, i < m ? (long long)k : 0, (long long)(tile * kW4Cols + 32 * u + 8 * t));
    float lo[4], hi[4];
    bool bad[4];
#pragma unroll
    for (int u = 0; u < 4; ++u) {
      lo[u] = hi[u] = 0.f;
      bad[u] = false;
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        const float v = to_f32(w[u][e]);
        lo[u] = fminf(lo[u], v);
        hi[u] = fmaxf(hi[u], v);
        bad[u] |= !(fabsf(v) <= 3.4e38f);
      }
    }
#pragma unroll
    for (int u = 0; u < 4; ++u) {
#pragma unroll
      for (int x = 1; x <= 2; x <<= 1) {
        lo[u] = fminf(lo[u], __shfl_xor_sync(0xffffffffu, lo[u], x));
        hi[u] = fmaxf(hi[u], __shfl_xor_sync(0xffffffffu, hi[u], x));
        bad[u] |= __shfl_xor_sync(0xffffffffu, (int)bad[u], x) != 0;
      }
    }
    uint32_t word[4];
#pragma unroll
    for (int u = 0; u < 4; ++u) {
      const int first = u / per * per;
      float l = lo[u], h = hi[u];
      bool b = bad[u];
#pragma unroll
      for (int v = 0; v < 4; ++v)
        if (v >= first && v < first + per) {
          l = fminf(l, lo[v]);
          h = fmaxf(h, hi[v]);
          b |= bad[v];
        }
      // halves first: the span of two bfloat16 values may pass the largest float
      const float wide = f.zeros ? (0.5f * h - 0.5f * l) / 7.5f : fmaxf(-l, h) / 7.f;
      float s = to_f32(from_f32<T>(wide));
      if (b || !(s <= 3.4e38f)) s = __int_as_float(0x7fc00000);
      const bool live = s > 0.f;
      const float z = f.zeros ? (live ? fminf(fmaxf(rintf(-l / s), 0.f), 15.f) : 0.f) : 8.f;
      word[u] = 0;
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        const float q = live ? fminf(fmaxf(rintf(to_f32(w[u][e]) / s) + z, 0.f), 15.f) : z;
        word[u] |= (uint32_t)q << (4 * w4_nibble(e));
      }
      if (t == 0 && u % per == 0) {
        const int g = u / per;
        *reinterpret_cast<T*>(out + f.scale_at(g, row)) = from_f32<T>(s);
        if (f.zeros) out[f.zero_at(g, row)] = (unsigned char)z;
      }
    }
    *reinterpret_cast<uint4*>(out + w4_piece(row, t)) = make_uint4(word[0], word[1], word[2], word[3]);
  }
}

// Codes, scales and zero points that exist already (a quantised checkpoint), put into the packed order.
// codes: two a byte, the even column in the low half, rows `ldcodes` bytes apart; scales and zero points row by row.
template <typename T>
__global__ void w4_pack_kernel(size_t m, size_t k, W4Format f, const unsigned char* __restrict__ codes, size_t ldcodes,
                               const T* __restrict__ scales, size_t lds, const unsigned char* __restrict__ zps,
                               size_t ldz, unsigned char* __restrict__ packed) {
  const size_t tiles = w4_k_tiles(k);
  const size_t unit = (size_t)blockIdx.x * (blockDim.x / 32) + threadIdx.x / 32;
  if (unit >= w4_row_blocks(m) * tiles) return;
  const size_t block = unit / tiles, tile = unit % tiles;
  const int lane = threadIdx.x & 31, r = lane >> 2, t = lane & 3;
  unsigned char* out = packed + unit * f.tile_bytes();
  const size_t total_groups = (k + f.group - 1) / f.group;
  const int per = f.group / 32;
#pragma unroll
  for (int half = 0; half < 2; ++half) {
    const int row = r + 8 * half;
    const size_t i = block * kW4Rows + row;
    uint32_t word[4];
#pragma unroll
    for (int u = 0; u < 4; ++u) {
      const size_t j0 = tile * kW4Cols + 32 * u + 8 * t;
      const size_t g = (tile * kW4Cols + 32 * u) / f.group;
      const bool have = i < m && g < total_groups;
      const uint32_t z = f.zeros ? (have ? (uint32_t)(zps[i * ldz + g] & 15) : 0u) : 8u;
      word[u] = 0;
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        const size_t j = j0 + e;
        uint32_t q = z;
        if (i < m && j < k) {
          const uint32_t byte = codes[i * ldcodes + j / 2];
          q = (j & 1) ? byte >> 4 : byte & 15u;
        }
        word[u] |= q << (4 * w4_nibble(e));
      }
      if (t == 0 && u % per == 0) {
        const int gt = u / per;
        *reinterpret_cast<T*>(out + f.scale_at(gt, row)) = have ? scales[i * lds + g] : from_f32<T>(0.f);
        if (f.zeros) out[f.zero_at(gt, row)] = (unsigned char)z;
      }
    }
    *reinterpret_cast<uint4*>(out + w4_piece(row, t)) = make_uint4(word[0], word[1], word[2], word[3]);
  }
}

// The weights that a packed matrix stands for, rounded to the 16-bit type (the product of a 4-bit difference and a
// 16-bit scale has up to 15 bits): the mirror of w4_quantize_kernel.
template <typename T>
__global__ void w4_unpack_kernel(size_t m, size_t k, W4Format f, const unsigned char* __restrict__ packed,
                                 T* __restrict__ W, size_t ldw) {
  const size_t tiles = w4_k_tiles(k);
  const size_t unit = (size_t)blockIdx.x * (blockDim.x / 32) + threadIdx.x / 32;
  if (unit >= w4_row_blocks(m) * tiles) return;
  const size_t block = unit / tiles, tile = unit % tiles;
  const int lane = threadIdx.x & 31, r = lane >> 2, t = lane & 3;
  const unsigned char* in = packed + unit * f.tile_bytes();
  const bool vec = ldw % 8 == 0 && (reinterpret_cast<uintptr_t>(W) & 15u) == 0;
  const int per = f.group / 32;
#pragma unroll
  for (int half = 0; half < 2; ++half) {
    const int row = r + 8 * half;
    const size_t i = block * kW4Rows + row;
    if (i >= m) continue;
    const uint4 c = __ldg(reinterpret_cast<const uint4*>(in + w4_piece(row, t)));
    const uint32_t word[4] = {c.x, c.y, c.z, c.w};
#pragma unroll
    for (int u = 0; u < 4; ++u) {
      const size_t j = tile * kW4Cols + 32 * u + 8 * t;
      if (j >= k) continue;
      const int g = u / per;
      const float s = to_f32(*reinterpret_cast<const T*>(in + f.scale_at(g, row)));
      const int z = f.zeros ? in[f.zero_at(g, row)] : 8;
      T v[8];
#pragma unroll
      for (int e = 0; e < 8; ++e)
        v[e] = from_f32<T>((float)((int)((word[u] >> (4 * w4_nibble(e))) & 15u) - z) * s);
      T* dst = W + i * ldw + j;
      if (vec && j + 8 <= k) {
        *reinterpret_cast<uint4*>(dst) = *reinterpret_cast<const uint4*>(v);
      } else {
#pragma unroll
        for (int e = 0; e < 8; ++e)
          if (j + e < k) dst[e] = v[e];
      }
    }
  }
}

}  // namespace mmbo
