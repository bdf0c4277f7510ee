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

// Two 16-bit floats (as stored, low half first) widened.
template <typename T>
__device__ __forceinline__ float2 widen2(uint32_t v);
template <>
__device__ __forceinline__ float2 widen2<__half>(uint32_t v) { return __half22float2(*reinterpret_cast<__half2*>(&v)); }
template <>
__device__ __forceinline__ float2 widen2<__nv_bfloat16>(uint32_t v) {
  return make_float2(__uint_as_float(v << 16), __uint_as_float(v & 0xffff0000u));
}

// Bytes off .. off + 15 of u and v, off even and below 16.
__device__ __forceinline__ uint4 bytes_from(const uint4& u, const uint4& v, int off) {
  const bool two = off & 8, one = off & 4;
  const uint32_t w0 = two ? u.z : u.x, w1 = two ? u.w : u.y, w2 = two ? v.x : u.z, w3 = two ? v.y : u.w, w4 = two ? v.z : v.x,
                 w5 = two ? v.w : v.y;
  const uint32_t a0 = one ? w1 : w0, a1 = one ? w2 : w1, a2 = one ? w3 : w2, a3 = one ? w4 : w3, a4 = one ? w5 : w4;
  const int bits = (off & 2) * 8;
  return make_uint4(__funnelshift_r(a0, a1, bits), __funnelshift_r(a1, a2, bits), __funnelshift_r(a2, a3, bits),
                    __funnelshift_r(a3, a4, bits));
}

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
      return bytes_from(u, v, off);
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

// ---------------------------------------------------------------- codes ---------------
// Tile layout known at compile time.
template <int QG, bool ZEROS>
struct W4Tile {
  static constexpr int kGroups = 4 / QG;  // QG: quarters of 32 columns in a group
  static constexpr int kScales = kW4Codes, kZeros = kW4Codes + kGroups * kW4Rows * 2;
  static constexpr int kBytes = kZeros + (ZEROS ? kGroups * kW4Rows : 0);
};

constexpr uint32_t kLowCodes = 0x000f000fu, kHighCodes = 0x00f000f0u;
// Eight codes of a word as four registers of two 16-bit floats with the zero point subtracted, all exact.
//   half precision: 0x6400 | q is 1024 + q and 0x6400 | 16 q is 1024 + 16 q, of which a fused multiply-add makes q - z
//   bfloat16: 0x4300 | q is 128 + q (the 16 q form would spill into the exponent)
template <typename T>
struct W4Unpacker;
// (x & mask) | with in one instruction.
__device__ __forceinline__ uint32_t and_or(uint32_t x, uint32_t mask, uint32_t with) {
  uint32_t r;
  asm("lop3.b32 %0, %1, %2, %3, 0xea;" : "=r"(r) : "r"(x), "r"(mask), "r"(with));
  return r;
}
// A constant the compiler keeps in a register: as an immediate beside the mask it would need a second instruction.
__device__ __forceinline__ uint32_t in_register(uint32_t c) {
  asm volatile("" : "+r"(c));
  return c;
}
template <>
struct W4Unpacker<__half> {
  uint32_t bias, z1, z16;
  __device__ __forceinline__ W4Unpacker() : bias(in_register(0x64006400u)) {}
  __device__ __forceinline__ void set_zero(uint32_t z) {
    z1 = (0x6400u | z) * 0x10001u;
    z16 = (0xd400u | (z << 4)) * 0x10001u;  // -(64 + z)
  }
  __device__ __forceinline__ static __half2 h2(uint32_t x) { return *reinterpret_cast<__half2*>(&x); }
  __device__ __forceinline__ static uint32_t u32(__half2 x) { return *reinterpret_cast<uint32_t*>(&x); }
  __device__ __forceinline__ void unpack(uint32_t w, uint32_t* a) const {
    const uint32_t v = w >> 8;
    const __half2 c16 = __half2half2(__ushort_as_half(0x2c00));  // 1 / 16
    a[0] = u32(__hsub2(h2(and_or(w, kLowCodes, bias)), h2(z1)));
    a[1] = u32(__hsub2(h2(and_or(v, kLowCodes, bias)), h2(z1)));
    a[2] = u32(__hfma2(h2(and_or(w, kHighCodes, bias)), c16, h2(z16)));
    a[3] = u32(__hfma2(h2(and_or(v, kHighCodes, bias)), c16, h2(z16)));
  }
};
// DOWN: bfloat16 codes come times 2^-DOWN, by another exponent in the same constants.
template <int DOWN = 0>
struct W4UnpackerBf16 {
  static constexpr uint32_t kBias = 0x4300u - (DOWN << 7);
  uint32_t bias, z1;
  __device__ __forceinline__ W4UnpackerBf16() : bias(in_register(kBias * 0x10001u)) {}
  __device__ __forceinline__ void set_zero(uint32_t z) { z1 = (kBias | z) * 0x10001u; }
  __device__ __forceinline__ uint32_t one(uint32_t w) const {
    uint32_t x = and_or(w, kLowCodes, bias);
    const __nv_bfloat162 d = __hsub2(*reinterpret_cast<__nv_bfloat162*>(&x), *reinterpret_cast<const __nv_bfloat162*>(&z1));
    return *reinterpret_cast<const uint32_t*>(&d);
  }
  __device__ __forceinline__ void unpack(uint32_t w, uint32_t* a) const {
    a[0] = one(w);
    a[1] = one(w >> 8);
    a[2] = one(w >> 4);
    a[3] = one(w >> 12);
  }
};
template <>
struct W4Unpacker<__nv_bfloat16> : W4UnpackerBf16<> {};

// Codes as the products take them, kUnit times too small.  A group's sum of bfloat16 activations could pass the largest float
// where the scale would bring it back: up to 128 products with differences up to 15, so below 2^11 times the largest
// activation.  With differences times 2^-11 it cannot; results get the factor back at the end.  What that costs: results
// below 2^-115 are held to steps of 2^-138 (bfloat16's are 2^-133).
template <typename T>
struct W4Operand : W4Unpacker<T> {
  static constexpr float kUnit = 1.f;
};
template <>
struct W4Operand<__nv_bfloat16> : W4UnpackerBf16<11> {
  static constexpr float kUnit = 0x1p11f;
};

// ---------------------------------------------------------------- writing the format --
// One warp per tile; lane 4 r + t (r 0..7, t 0..3) owns rows r and r + 8 of the block and, in each quarter u, the
// columns 32 u + 8 t .. + 7: its eight words are two 16-byte stores, and the loads of four lanes are 64 contiguous
// bytes of a row.  One pass, so bound by bytes: 2 m k in, m k / 2 out.
//
// Symmetric: s = max|w| / 7 rounded to the weights' type, z = 8.  With zero points: lo = min(w, 0), hi = max(w, 0),
// s = (hi - lo) / 15 rounded to the weights' type, z = rint(-lo / s).  q = rint(w / s) + z, held to 0..15; ties to
// even.  A group whose scale rounds to zero becomes zeros; one with an infinity or a NaN becomes NaN (its scale is).
//
// rint(w / s) without a division per element (a division bound the kernel: 53 us instead of 21 for a round trip of
// 4096 x 4096): w * (1 / s) is within 2^-18 of w / s, and one fused multiply-add rounds it to a multiple of 2^-14.  With
// significands of 11 bits at most w / s is either a tie, n + 1/2, which that rounding restores, or at least 2^-13 away from
// one, which it keeps on its side (all pairs of significands were compared with the quotient).  A second
// addition rounds to an integer, ties to even.
// A group's scale, too, is computed by one of its four lanes instead of all (ragged 11001 x 8200 in groups of 32 with zero
// points: 83 us before, 54 us after).
constexpr float kSnap = 768.f;             // adding it leaves multiples of 2^-14
constexpr float kToInteger = 12582144.f;   // 1.5 * 2^23 - kSnap: adding it then leaves integers, in the low bits
constexpr uint32_t kIntegerBits = 0x4b400000u;
template <typename T>
struct W4Pair {
  using type = __half2;
};
template <>
struct W4Pair<__nv_bfloat16> {
  using type = __nv_bfloat162;
};

// ALIGNED: every row of W starts on a 16-byte boundary.
template <typename T, int QG, bool ZEROS, bool ALIGNED>
__global__ void __launch_bounds__(256) w4_quantize_kernel(size_t m, size_t k, const T* __restrict__ W, size_t ldw,
                                                          unsigned char* __restrict__ packed) {
  using L = W4Tile<QG, ZEROS>;
  using Pair = typename W4Pair<T>::type;
  const unsigned tiles = (unsigned)w4_k_tiles(k), unit = blockIdx.x * 8 + threadIdx.x / 32;
  const unsigned block = unit / tiles, tile = unit % tiles;
  if (block >= w4_row_blocks(m)) return;
  const int lane = threadIdx.x & 31, r = lane >> 2, t = lane & 3;
  unsigned char* out = packed + (size_t)unit * L::kBytes;
  const size_t j0 = (size_t)tile * kW4Cols + 8 * t;
  // Tiles inside the rows need no checks of their columns: one 16-byte load of eight columns, or two off the boundaries.
  const bool whole = (size_t)(tile + 1) * kW4Cols + (ALIGNED ? 0 : 8) <= k && (ALIGNED || tile > 0);
  auto lesser = [](uint32_t x, uint32_t y) {
    const Pair p = __hmin2_nan(*reinterpret_cast<const Pair*>(&x), *reinterpret_cast<const Pair*>(&y));
    return *reinterpret_cast<const uint32_t*>(&p);
  };
  uint4 w[2][4];
#pragma unroll
  for (int half = 0; half < 2; ++half) {
    const size_t i = (size_t)block * kW4Rows + r + 8 * half;
    const T* row = W + i * ldw;
    const int off = (int)(reinterpret_cast<uintptr_t>(row) & 15u);
    const uint4* at = reinterpret_cast<const uint4*>(reinterpret_cast<uintptr_t>(row + j0) & ~(uintptr_t)15);
#pragma unroll
    for (int u = 0; u < 4; ++u) {
      if (whole)
        w[half][u] = i >= m ? make_uint4(0, 0, 0, 0) : ALIGNED ? at[4 * u] : bytes_from(at[4 * u], at[4 * u + 1], off);
      else
        w[half][u] = load8(row, i < m ? (long long)k : 0, (long long)(j0 + 32 * u));
    }
  }
#pragma unroll
  for (int half = 0; half < 2; ++half) {
    const int row = r + 8 * half;
    // (lo, -hi) of each quarter, a NaN stays; then of quarter t over the four lanes of the row, then of t's group
    uint32_t ends[4];
#pragma unroll
    for (int u = 0; u < 4; ++u) {
      const uint32_t e[4] = {w[half][u].x, w[half][u].y, w[half][u].z, w[half][u].w}, none = 0;
      Pair lo = *reinterpret_cast<const Pair*>(&none), hi = lo;
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        lo = __hmin2_nan(lo, *reinterpret_cast<const Pair*>(&e[i]));
        hi = __hmax2_nan(hi, *reinterpret_cast<const Pair*>(&e[i]));
      }
      const uint32_t lows = *reinterpret_cast<const uint32_t*>(&lo), highs = *reinterpret_cast<const uint32_t*>(&hi) ^ 0x80008000u;
      ends[u] = lesser(__byte_perm(lows, highs, 0x5410), __byte_perm(lows, highs, 0x7632));
    }
#pragma unroll
    for (int u = 0; u < 4; u += 2) {
      const uint32_t other = __shfl_xor_sync(0xffffffffu, t & 1 ? ends[u] : ends[u + 1], 1);
      ends[u] = lesser(t & 1 ? ends[u + 1] : ends[u], other);
    }
    ends[0] = lesser(t & 2 ? ends[2] : ends[0], __shfl_xor_sync(0xffffffffu, t & 2 ? ends[0] : ends[2], 2));
#pragma unroll
    for (int x = 1; x < QG; x <<= 1) ends[0] = lesser(ends[0], __shfl_xor_sync(0xffffffffu, ends[0], x));
    const float2 range = widen2<T>(ends[0]);
    const float l = range.x, h = -range.y;
    // halves first: the span of two bfloat16 values may pass the largest float
    float span = 0.5f * h - 0.5f * l;
    if (ZEROS && std::is_same<T, __half>::value) {
      // Two half-precision ends may need 27 bits together (bfloat16 ones that do are too far apart to matter).  Rounded to nearest, a
      // span beside 15 times a tie of the scale became that tie; rounded to the odd neighbour it stays beside it, and so does the
      // quotient.
      const float part = span - 0.5f * h, lost = (0.5f * h - (span - part)) + (-0.5f * l - part);
      const uint32_t bits = __float_as_uint(span);
      if (lost != 0.f && (bits & 1u) == 0) span = __uint_as_float(lost > 0.f ? bits + 1 : bits - 1);
    }
    const float wide = ZEROS ? span / 7.5f : fmaxf(-l, h) / 7.f;
    float s = to_f32(from_f32<T>(wide));
    if (!(s <= 3.4e38f)) s = __int_as_float(0x7fc00000);
    // A group's multiplier; -s for a scale whose reciprocal might overflow (bfloat16 only): these divide.
    const float by = !(s > 0.f) ? 0.f : std::is_same<T, __nv_bfloat16>::value && s < 0x1p-100f ? -s : __frcp_rn(s);
    int zero = 8;
    if (ZEROS) {
      const float y = by < 0.f ? -l / s + kSnap : fmaf(-l, by, kSnap);
      zero = s > 0.f ? (int)(__float_as_uint(fminf(y, kSnap + 15.f) + kToInteger) - kIntegerBits) : 0;
    }
    if (t % QG == 0) {
      const int at = t / QG * kW4Rows + W4Format::slot(row);
      *reinterpret_cast<T*>(out + L::kScales + at * 2) = from_f32<T>(s);
      if (ZEROS) out[L::kZeros + at] = (unsigned char)zero;
    }
    uint32_t word[4];
#pragma unroll
    for (int g = 0; g < L::kGroups; ++g) {
      const float times = __shfl_sync(0xffffffffu, by, (lane & ~3) | g * QG);
      const int z = ZEROS ? __shfl_sync(0xffffffffu, zero, (lane & ~3) | g * QG) : 8;
      const float least = kSnap - (float)z, most = kSnap + (float)(15 - z);
      const uint32_t shift = (uint32_t)z * 0x11111111u - kIntegerBits * 0x11111111u;
#pragma unroll
      for (int u = g * QG; u < (g + 1) * QG; ++u) {
        const uint32_t e[4] = {w[half][u].x, w[half][u].y, w[half][u].z, w[half][u].w};
        float y[8];
        uint32_t bits[8], all = 0;
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const float2 p = widen2<T>(e[i]);
          y[2 * i] = fmaf(p.x, times, kSnap);
          y[2 * i + 1] = fmaf(p.y, times, kSnap);
        }
        if (std::is_same<T, __nv_bfloat16>::value && times < 0.f) {
#pragma unroll
          for (int i = 0; i < 8; ++i) {
            const float2 p = widen2<T>(e[i / 2]);
            y[i] = (i & 1 ? p.y : p.x) / -times + kSnap;
          }
        }
#pragma unroll
        for (int i = 0; i < 8; ++i)  // (a group of NaN: code 0)
          bits[i] = __float_as_uint(fminf(fmaxf(y[i], least), most) + kToInteger);
#pragma unroll
        for (int n = 7; n >= 0; --n) all = all * 16u + bits[w4_nibble(n)];  // nibble n holds column w4_nibble(n)
        word[u] = all + shift;
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
template <typename T, int QG, bool ZEROS, bool ALIGNED>
__global__ void __launch_bounds__(256) w4_unpack_kernel(size_t m, size_t k, const unsigned char* __restrict__ packed,
                                                        T* __restrict__ W, size_t ldw) {
  using L = W4Tile<QG, ZEROS>;
  using Pair = typename W4Pair<T>::type;
  const unsigned tiles = (unsigned)w4_k_tiles(k), unit = blockIdx.x * 8 + threadIdx.x / 32;
  const unsigned block = unit / tiles, tile = unit % tiles;
  if (block >= w4_row_blocks(m)) return;
  const int lane = threadIdx.x & 31, r = lane >> 2, t = lane & 3;
  const unsigned char* in = packed + (size_t)unit * L::kBytes;
  const bool whole = (size_t)(tile + 1) * kW4Cols <= k;
  W4Unpacker<T> unpacker;
#pragma unroll
  for (int half = 0; half < 2; ++half) {
    const int row = r + 8 * half;
    const size_t i = (size_t)block * kW4Rows + row;
    const uint4 c = __ldg(reinterpret_cast<const uint4*>(in + w4_piece(row, t)));
    const uint32_t word[4] = {c.x, c.y, c.z, c.w};
    uint4 v[4];
#pragma unroll
    for (int u = 0; u < 4; ++u) {
      const int g = u / QG;
      const uint32_t scale = *reinterpret_cast<const uint16_t*>(in + L::kScales + (g * kW4Rows + W4Format::slot(row)) * 2);
      const uint32_t scales = scale * 0x10001u;
      unpacker.set_zero(ZEROS ? in[L::kZeros + g * kW4Rows + W4Format::slot(row)] : 8u);
      uint32_t e[4];
      unpacker.unpack(word[u], e);
#pragma unroll
      for (int x = 0; x < 4; ++x) {
        const Pair p = __hmul2(*reinterpret_cast<const Pair*>(&e[x]), *reinterpret_cast<const Pair*>(&scales));
        e[x] = *reinterpret_cast<const uint32_t*>(&p);
      }
      v[u] = make_uint4(e[0], e[1], e[2], e[3]);
    }
    T* dst = W + i * ldw + (size_t)tile * kW4Cols + 8 * t;
    const int off = (int)(reinterpret_cast<uintptr_t>(dst) & 15u);
    if (whole && ALIGNED) {
      if (i < m) {
#pragma unroll
        for (int u = 0; u < 4; ++u) *reinterpret_cast<uint4*>(dst + 32 * u) = v[u];
      }
    } else if (whole) {
      // Off the 16-byte boundaries every piece between two of them is the end of one lane's eight columns and the start of the
      // next one's; the row's first and last columns go singly (all of them singly: 382 us instead of 128 for a round
      // trip of 3938 x 19374 with rows four bytes off).
      uint4 last = make_uint4(0, 0, 0, 0);
#pragma unroll
      for (int u = 0; u < 4; ++u) {
        const int from = (lane & ~3) | ((t + 3) & 3);
        const uint4 turned = make_uint4(__shfl_sync(0xffffffffu, v[u].x, from), __shfl_sync(0xffffffffu, v[u].y, from),
                                        __shfl_sync(0xffffffffu, v[u].z, from), __shfl_sync(0xffffffffu, v[u].w, from));
        const uint4 before = t ? turned : last;
        last = turned;
        if (i >= m) continue;
        T* at = dst + 32 * u;
        if (off == 0)
          *reinterpret_cast<uint4*>(at) = v[u];
        else if (u + t > 0)
          *reinterpret_cast<uint4*>(reinterpret_cast<uintptr_t>(at) - off) = bytes_from(before, v[u], 16 - off);
      }
      if (off && i < m && (t == 0 || t == 3)) {
        const uint4 ends = make_uint4(t ? v[3].x : v[0].x, t ? v[3].y : v[0].y, t ? v[3].z : v[0].z, t ? v[3].w : v[0].w);
        const T* from = reinterpret_cast<const T*>(&ends);
        T* at = dst + (t ? 96 : 0);
#pragma unroll
        for (int e = 0; e < 8; ++e)
          if (t ? e >= 8 - off / 2 : e < 8 - off / 2) at[e] = from[e];
      }
    } else if (i < m) {
#pragma unroll
      for (int u = 0; u < 4; ++u) {
        const T* from = reinterpret_cast<const T*>(&v[u]);
        const size_t j = (size_t)tile * kW4Cols + 32 * u + 8 * t;
#pragma unroll
        for (int e = 0; e < 8; ++e)
          if (j + e < k) dst[32 * u + e] = from[e];
      }
    }
  }
}

}  // namespace mmbo
