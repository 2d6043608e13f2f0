// Streaming products of weights with a few rows of activations on the
// warp-level tensor instructions: the part that the 4-bit linear and the
// mixture-of-experts kernels share.
//
// A step with few rows is bound by the bytes of its weights, so the weights
// are the 16 rows of an m16n8k16 product and eight activation rows its
// columns: each weight goes from memory to registers once, and is used for
// every row.  (tcgen05 needs its operands in shared memory and at least 64
// rows of a tile filled; here the weights would pass through shared memory
// only to meet a tile that is nearly empty.)  The reduction index may be
// permuted freely as long as both operands agree, so a lane's fragment is
// whatever consecutive bytes wide loads of a row bring: checkpoints'
// row-major layouts are read as they are, and the activations are laid out
// once in the order in which the lanes use them.
//
// A "unit" is the piece of a row that the four lanes of a fragment row hold
// at a time, 16 bytes a lane in one load: 32 bf16, 64 e4m3 or 128 4-bit codes.
// (A load costs L1 a cycle for each of its eight rows whatever its width, so
// narrower ones would cap the rate.)  A warp works in quads of units, the next
// quad on its way in registers while one is consumed, across the ends of
// tiles; rows are padded to whole quads with activations that are zero, so the
// loop over quads has no branches.  (Rings in shared memory, filled by TMA
// boxes or asynchronous copies, came to 3.7 TB/s where this comes to 5.2, with
// 4-bit weights [129281, 4096] and 8 rows: each unit then starts with a wait and
// a read that nothing overlaps.)  What is on its way needs lines of L1, so a CTA
// takes no more shared memory than it must: with 64 KB more for further columns
// the expert layer's time rose from 192 to 268 us.
//
// A product may only sum over one group of codes; with groups of 64 or 32 the
// four lanes exchange words first.  Sums are held in 32 bits; group and block
// scales multiply the 32-bit sums of their own groups.  The 4-bit scales and zero
// points of a warp's share of a tile come into shared memory a tile ahead, in
// runs along the rows: loaded unit by unit they cost L1 more cycles than the
// codes.
//
// No code is converted.  The smallest floats of a 16-bit type are evenly
// spaced: bits 0..7 of a bf16 (0..10 of an fp16) with nothing above them are
// the number times 2^-133 (2^-24), across the end of the subnormals.  So a
// word of 4-bit codes, masked, is two codes as exact floats, and those four
// bits higher are 16 times theirs: five bit operations for eight codes.  e4m3
// moved into the low exponent and high mantissa bits of a bf16 is its value
// times 2^-120, the subnormals with it.  bf16 activations are scaled by 2^80
// when they are laid out, so that the products keep clear of both ends of the
// 32-bit range, and the powers of two leave with the finished sum.  From 2^48 on
// an activation becomes infinite that way, and so does, or NaN, what its row
// gives; below 2^-73 terms lose bits.  (Columns laid out again without the
// scaling where it overflows were right, but cost ordinary ones 3 to 6 %.)  An
// e4m3 NaN comes out as 480, so the stream tells its source of tiles that have one.
//
// Zero points come off the group's sum: s (sum q x - z sum x), with sum x
// known once per column and group, where taking z from every code costs half
// as much again as the extraction.
#pragma once

#include <cuda_fp16.h>

#include <type_traits>

#include "hca_common.cuh"

namespace hca {

enum WFormat : int { kWBf16 = 0, kWFp8 = 1, kW4G32 = 2, kW4G64 = 3, kW4G128 = 4 };

template <int F>
struct WTraits {
  static constexpr bool kIs4 = F >= kW4G32;
  static constexpr int kUnitK = F == kWBf16 ? 32 : F == kWFp8 ? 64 : 128;
  static constexpr int kSub = F == kW4G32 ? 4 : F == kW4G64 ? 2 : 1;  // groups of a unit
  static constexpr int kPieces = kUnitK / 32;    // 16-byte activation pieces of a lane and column
  static constexpr int kGroupK = kUnitK / kSub;  // reduction length of a group
  __host__ __device__ static constexpr int64_t row_bytes(int64_t k) {
    return F == kWBf16 ? 2 * k : F == kWFp8 ? k : k / 2;
  }
  // units that a warp has on its way: with two blocks of columns and 4-bit
  // codes four and the sums would not fit a thread's 128 registers (8 % slower)
  static constexpr int step(int blocks) { return kIs4 && blocks > 1 ? 2 : 4; }
  // units of rows of k, in whole quads
  __host__ __device__ static constexpr int units(int k) { return (k + 4 * kUnitK - 1) / (4 * kUnitK) * 4; }
};

template <typename T>
struct MmaType;
template <>
struct MmaType<__nv_bfloat16> {
  static __device__ __forceinline__ void mma(float (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3,
                                             uint32_t b0, uint32_t b1) {
    asm("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};\n"
        : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
        : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
  }
  static __device__ __forceinline__ uint32_t pack(float lo, float hi) {
    __nv_bfloat162 v = __floats2bfloat162_rn(lo, hi);
    return *reinterpret_cast<uint32_t*>(&v);
  }
  static __device__ __forceinline__ float2 unpack(uint32_t v) {
    return make_float2(__uint_as_float(v << 16), __uint_as_float(v & 0xffff0000u));
  }
  // both halves times a power of two, exactly
  static __device__ __forceinline__ uint32_t times(uint32_t v, float f) {
    const __nv_bfloat162 r = __hmul2(*reinterpret_cast<__nv_bfloat162*>(&v), __float2bfloat162_rn(f));
    return *reinterpret_cast<const uint32_t*>(&r);
  }
  static __device__ __forceinline__ float to_float(uint16_t v) { return bf16_bits_to_float(v); }
  static __device__ __forceinline__ __nv_bfloat16 from_float(float v) { return __float2bfloat16_rn(v); }
};
template <>
struct MmaType<__half> {
  static __device__ __forceinline__ void mma(float (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3,
                                             uint32_t b0, uint32_t b1) {
    asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};\n"
        : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
        : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
  }
  static __device__ __forceinline__ uint32_t pack(float lo, float hi) {
    __half2 v = __floats2half2_rn(lo, hi);
    return *reinterpret_cast<uint32_t*>(&v);
  }
  static __device__ __forceinline__ float2 unpack(uint32_t v) { return __half22float2(*reinterpret_cast<__half2*>(&v)); }
  static __device__ __forceinline__ float to_float(uint16_t v) { return __half2float(__ushort_as_half(v)); }
  static __device__ __forceinline__ __half from_float(float v) { return __float2half_rn(v); }
};

// Powers of two on the way: x is laid out times kX, group sums of x are kept
// times kSum, and the finished sums take kOut.
template <int F, typename T>
struct Scaling {
  static constexpr bool kHalf = sizeof(T) == 2 && !std::is_same<T, __nv_bfloat16>::value;
  static_assert(!kHalf || WTraits<F>::kIs4, "fp16 goes with 4-bit weights only");
  static constexpr float kX = F == kWBf16 || kHalf ? 1.0f : 0x1p80f;
  static constexpr float kXOdd = WTraits<F>::kIs4 ? kX / 16 : kX;
  // fp16 activations have no room for that: sums of the odd codes are held apart
  static constexpr bool kApart = kHalf;
  static constexpr float kSum = kHalf ? 0x1p-24f : 0x1p-53f;
  static constexpr float kOut = F == kWBf16 ? 1.0f : kHalf ? 0x1p24f : F == kWFp8 ? 0x1p40f : 0x1p53f;
};

// The words of a unit by group: on return lane c of the four holds words of
// group i alone in w[i * 4 / kSub ..].  With groups of 32 that is a transpose
// of the four lanes' words, with groups of 64 an exchange of two.
template <int F>
__device__ __forceinline__ void by_group(uint32_t (&w)[4]) {
  const int c = threadIdx.x & 3;
  if constexpr (F == kW4G64) {
    const bool up = c & 2;
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      const uint32_t v = __shfl_xor_sync(0xffffffffu, up ? w[i] : w[i + 2], 2);
      if (up) w[i] = v; else w[i + 2] = v;
    }
  } else if constexpr (F == kW4G32) {
    const bool b0 = c & 1, b1 = c & 2;
#pragma unroll
    for (int i = 0; i < 4; i += 2) {
      const uint32_t v = __shfl_xor_sync(0xffffffffu, b0 ? w[i] : w[i + 1], 1);
      if (b0) w[i] = v; else w[i + 1] = v;
    }
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      const uint32_t v = __shfl_xor_sync(0xffffffffu, b1 ? w[i] : w[i + 2], 2);
      if (b1) w[i] = v; else w[i + 2] = v;
    }
  }
}

// Place of the 16-byte piece that holds column col's activations k .. k + 7
// (k a multiple of 8) among the pieces of a block of columns: the pieces of a
// unit follow each other, each 4 kWidth lanes wide.  The lanes of a piece are
// swapped around by `piece_swap`, so that eight threads that lay out
// consecutive activations write to eight different bank groups.
// (A single column has no lanes to swap.)
template <int F, int kWidth>
__device__ __forceinline__ int piece_swap(int u, int j) {
  return kWidth == 1 ? 0 : F == kWBf16 ? 4 * (u & 1) : F == kW4G128 ? 2 * j : 4 * (j & 1);
}
template <int F, int kWidth, int kParts>
__device__ __forceinline__ int piece_index(int k, int col, int part) {
  using W = WTraits<F>;
  const int u = k / W::kUnitK, r = k % W::kUnitK;
  int c, j;
  if constexpr (F == kWBf16) c = r / 8, j = 0;
  else if constexpr (F == kWFp8) c = r / 16, j = r / 8 % 2;
  else if constexpr (F == kW4G128) c = r / 32, j = r / 8 % 4;
  else if constexpr (F == kW4G64) c = r / 32 % 2 + r / 16 % 2 * 2, j = r / 64 * 2 + r / 8 % 2;
  else c = r / 8 % 4, j = r / 32;
  return ((u * W::kPieces + j) * kParts + part) * kWidth * 4 + ((col * 4 + c) ^ piece_swap<F, kWidth>(u, j));
}

// Eight consecutive activations in a piece's order, that in which weights come
// out of a word together: codes 0,4 2,6 1,5 3,7 and e4m3 0,2 1,3 of each four.
// The odd codes come out 16 times as large, which bf16 activations make up for.
template <int F, typename T>
__device__ __forceinline__ uint4 piece_order(uint4 v) {
  using M = MmaType<T>;
  using S = Scaling<F, T>;
  if constexpr (WTraits<F>::kIs4)
    v = make_uint4(__byte_perm(v.x, v.z, 0x5410), __byte_perm(v.y, v.w, 0x5410), __byte_perm(v.x, v.z, 0x7632),
                   __byte_perm(v.y, v.w, 0x7632));
  if constexpr (F == kWFp8)
    v = make_uint4(__byte_perm(v.x, v.y, 0x5410), __byte_perm(v.x, v.y, 0x7632), __byte_perm(v.z, v.w, 0x5410),
                   __byte_perm(v.z, v.w, 0x7632));
  if constexpr (S::kX != 1.0f)
    v = make_uint4(M::times(v.x, S::kX), M::times(v.y, S::kX), M::times(v.z, S::kXOdd), M::times(v.w, S::kXOdd));
  return v;
}

// The warps that share a tile: warp `index` of `warps`, group `id` of the
// block.  They take the tile's quads of units in even runs.
struct TileGroup {
  int warps, index, id;

  __device__ __forceinline__ explicit TileGroup(int warps_)
      : warps(warps_), index((threadIdx.x >> 5) % warps_), id((threadIdx.x >> 5) / warps_) {}
  __device__ __forceinline__ int first_unit(int units) const { return units / 4 * index / warps * 4; }
  __device__ __forceinline__ int end_unit(int units) const { return units / 4 * (index + 1) / warps * 4; }
  __device__ __forceinline__ int threads() const { return warps * 32; }
  __device__ __forceinline__ int thread() const { return index * 32 + (threadIdx.x & 31); }

  // Waits for the whole group; barriers 1..15 are the groups'.
  __device__ __forceinline__ void sync() const {
    if (warps == 1) __syncwarp();
    else asm volatile("bar.sync %0, %1;\n" ::"r"(1 + id), "r"(warps * 32) : "memory");
  }
};

// Where a tile row's scales and zero points are (4-bit only): the addresses of
// the row's first, and the ends of the whole arrays.
struct WScales {
  const uint8_t *scale, *scale_end;
  const uint8_t *zero, *zero_end;  // null: 8 everywhere
};
// Whether rows of `groups` scales start on 16 bytes and their zero points on 8.
__device__ __forceinline__ bool scales_wide(const void* scale, const void* zero, int groups) {
  return ((reinterpret_cast<uintptr_t>(scale) | 2 * reinterpret_cast<uintptr_t>(zero) | 2 * groups) & 15) == 0;
}

// Scales and zero points of a warp's share of a tile, in shared memory, two
// tiles in turn.  If every row's share begins and ends on 16 bytes (wide), it
// is copied in pieces of 16 (zero points 8); else whole words around it are,
// and it starts 0..3 bytes into the first.  The former depends on the arrays'
// first bytes, on the groups of a whole row of theirs and on the share's ends.
template <int F>
struct ScaleTile {
  using W = WTraits<F>;
  uint8_t* base;  // this warp's: [2][16 rows][scales, zero points]
  int pitch, zero_at;
  bool wide;

  // bytes of a row: n scales and n zero points, each with room for words'
  // edges; an odd number of 16 bytes, so that eight rows start in different banks
  __host__ __device__ static int zero_offset(int n) { return (2 * n + 4 + 15) / 16 * 16; }
  __host__ __device__ static int row_pitch(int n, bool zeros) {
    return ((zero_offset(n) + (zeros ? n + 8 : 0) + 15) / 16 | 1) * 16;
  }
  // most groups of a warp's share
  __host__ __device__ static int share(int units, int warps) { return (units / 4 + warps - 1) / warps * 4 * W::kSub; }
  __host__ __device__ static int64_t bytes(int units, bool zeros, int group_warps, int block_warps) {
    return W::kIs4 ? 32ll * block_warps * row_pitch(share(units, group_warps), zeros) : 0;
  }

  __device__ __forceinline__ void init(uint8_t* smem, int units, bool zeros, int warps, bool rows_wide, int g0, int g1) {
    const int n = share(units, warps);
    zero_at = zero_offset(n), pitch = row_pitch(n, zeros);
    base = smem + (threadIdx.x >> 5) * 32 * pitch;
    wide = rows_wide && ((g0 | g1 | n) & 7) == 0;
  }
  __device__ __forceinline__ uint8_t* row(int i, int r) const { return base + ((i & 1) * 16 + r) * pitch; }
  // Starts the copy of groups [g0, g1) of the lane's row of tile `i`: lanes l
  // and l + 16 row l.
  __device__ __forceinline__ void fetch(int i, const WScales& from, int g0, int g1) const {
    const int lane = threadIdx.x & 31, half = lane >> 4;
    const uint32_t to = static_cast<uint32_t>(__cvta_generic_to_shared(row(i, lane & 15)));
    if (wide) {
#pragma unroll 1
      for (int g = g0 + 8 * half; g < g1; g += 16) {
        asm volatile("cp.async.cg.shared.global [%0], [%1], 16;\n" ::"r"(to + 2 * (g - g0)), "l"(from.scale + 2 * g) : "memory");
        if (from.zero != nullptr)
          asm volatile("cp.async.ca.shared.global [%0], [%1], 8;\n" ::"r"(to + zero_at + g - g0), "l"(from.zero + g) : "memory");
      }
    } else {
      copy(to, from.scale + 2 * g0, from.scale + 2 * g1, from.scale_end, half);
      if (from.zero != nullptr) copy(to + zero_at, from.zero + g0, from.zero + g1, from.zero_end, half);
    }
  }
  static __device__ __forceinline__ void copy(uint32_t to, const uint8_t* from, const uint8_t* until, const uint8_t* end, int first) {
    const uint8_t* p = reinterpret_cast<const uint8_t*>(reinterpret_cast<uintptr_t>(from) & ~uintptr_t{3}) + 4 * first;
    to += 4 * first;
#pragma unroll 1
    for (; p < until; p += 8, to += 8) {
      const int n = static_cast<int>(min(static_cast<int64_t>(4), static_cast<int64_t>(end - p)));  // not past the array
      asm volatile("cp.async.ca.shared.global [%0], [%1], 4, %2;\n" ::"r"(to), "l"(p), "r"(n) : "memory");
    }
  }
};

// Activations of NB blocks of columns in shared memory, in piece order, with
// their group sums.  A block has 8 columns, of which kWidth are stored.  With
// two parts an activation is the sum of two numbers, the second what rounding
// the first left: a second product with the same weights adds it.
template <int F, typename T, int NB, int kWidth, int kParts = 1>
struct XTile {
  using W = WTraits<F>;
  uint4* pieces;  // [NB][units][kPieces][kParts][kWidth][4]
  float* sums;    // [NB][units][kSub][8], 4-bit only
  int units;

  static constexpr int kUnitPieces = W::kPieces * kParts * kWidth * 4;
  static constexpr int kColumns = NB * kWidth;
  // Group sums of x by the tensor instructions once it is laid out, which costs
  // the same for one column as for eight, or by adding on the way: 16 rows of
  // 4096 10.0 us for 10.6, but one 7.5 for 7.1.
  static constexpr bool kSumProducts = W::kIs4 && kWidth == 8;

  __host__ __device__ static int64_t bytes(int units) {
    return NB * static_cast<int64_t>(units) * (kUnitPieces * 16 + (W::kIs4 ? W::kSub * 32 : 0));
  }

  __device__ __forceinline__ XTile(uint8_t* smem, int units_) : units(units_) {
    pieces = reinterpret_cast<uint4*>(smem);
    sums = reinterpret_cast<float*>(smem + static_cast<int64_t>(NB) * units * kUnitPieces * 16);
  }

  // All threads of the block; row(col) is column col's row of k values (and
  // behind them the k second parts) or null (zeros, as in the columns after
  // `columns`).  Ends with a block barrier.
  template <typename Row>
  __device__ __forceinline__ void stage(int k, int columns, int live, Row row) {
    const int padded = units * W::kUnitK;
    // several columns' loads under way at a time
    constexpr int kAhead = kWidth * kParts > 8 ? 8 / kParts : kWidth;
#pragma unroll 1
    for (int c0 = 0; c0 < live * kWidth; c0 += kAhead) {
      const T* p[kAhead];
#pragma unroll
      for (int n = 0; n < kAhead; ++n) p[n] = c0 + n < columns ? row(c0 + n) : nullptr;
      const int block = c0 / kWidth, col0 = c0 % kWidth;
      uint4* to = pieces + block * units * kUnitPieces;
#pragma unroll 1
      for (int i = threadIdx.x * 8; i < padded; i += blockDim.x * 8) {
        uint4 v[kAhead][kParts];
#pragma unroll
        for (int n = 0; n < kAhead; ++n)
#pragma unroll
          for (int part = 0; part < kParts; ++part)
            v[n][part] = p[n] != nullptr && i < k ? *reinterpret_cast<const uint4*>(p[n] + part * k + i) : make_uint4(0, 0, 0, 0);
#pragma unroll
        for (int n = 0; n < kAhead; ++n) {
          if constexpr (W::kIs4 && !kSumProducts) {
            // the group's threads are neighbours (padded is whole warps)
            float sum = 0.0f;
#pragma unroll
            for (int part = 0; part < kParts; ++part) {
              const uint4 w = v[n][part];
              const float2 a = MmaType<T>::unpack(w.x), b = MmaType<T>::unpack(w.y), c = MmaType<T>::unpack(w.z),
                           d = MmaType<T>::unpack(w.w);
              sum += ((a.x + a.y) + (b.x + b.y)) + ((c.x + c.y) + (d.x + d.y));
            }
#pragma unroll
            for (int o = W::kGroupK / 16; o > 0; o >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
            if (i % W::kGroupK == 0) sums[(block * units * W::kSub + i / W::kGroupK) * 8 + col0 + n] = sum * Scaling<F, T>::kSum;
          }
#pragma unroll
          for (int part = 0; part < kParts; ++part)
            to[piece_index<F, kWidth, kParts>(i, col0 + n, part)] = piece_order<F, T>(v[n][part]);
        }
      }
    }
    __syncthreads();
    if constexpr (kSumProducts) {
      // group sums as products with rows of the code 1, scaled as codes are
      constexpr uint32_t kOne = 0x00010001u, kOneOdd = Scaling<F, T>::kApart ? kOne : 16 * kOne;
      const int lane = threadIdx.x & 31, warps = blockDim.x >> 5;
#pragma unroll 1
      for (int i = threadIdx.x >> 5; i < live * units; i += warps) {
#pragma unroll
        for (int j = 0; j < W::kSub; ++j) {
          float sum[4] = {};
#pragma unroll
          for (int q = j * W::kPieces / W::kSub; q < (j + 1) * W::kPieces / W::kSub; ++q) {
#pragma unroll
            for (int part = 0; part < kParts; ++part) {
              const uint4 x = piece(pieces + i * kUnitPieces, i % units, q, part);
              MmaType<T>::mma(sum, kOne, kOne, kOne, kOne, x.x, x.y);
              MmaType<T>::mma(sum, kOneOdd, kOneOdd, kOneOdd, kOneOdd, x.z, x.w);
            }
          }
          if (lane < 4) *reinterpret_cast<float2*>(sums + (i * W::kSub + j) * 8 + 2 * lane) = make_float2(sum[0], sum[1]);
        }
      }
      __syncthreads();
    }
  }

  // The lane's piece j of unit u, whose pieces start at `at`.
  __device__ __forceinline__ uint4 piece(const uint4* at, int u, int j, int part) const {
    const int lane = threadIdx.x & 31;
    const uint4* p = at + (j * kParts + part) * kWidth * 4 + (lane ^ piece_swap<F, kWidth>(u, j));
    if (kWidth == 8) return *p;
    return lane < kWidth * 4 ? *p : make_uint4(0, 0, 0, 0);
  }

  // acc[b] += the step's rows times the columns of block b < NBL, over unit u.
  // w: the lane's shares of fragment rows lane / 4 and lane / 4 + 8;
  // scales(i, s, z) gives these rows' scale and zero point of the unit's group i.
  template <int NBL, typename Scales>
  __device__ __forceinline__ void consume(float (&acc)[NB][4], uint32_t (&w)[2][4], int u, Scales scales) const {
    using M = MmaType<T>;
    constexpr bool kApart = Scaling<F, T>::kApart;
    const int lane = threadIdx.x & 31;
    const uint4* at = pieces + u * kUnitPieces;
    if constexpr (F == kWBf16) {
#pragma unroll
      for (int b = 0; b < NBL; ++b) {
#pragma unroll
        for (int p = 0; p < kParts; ++p) {
          const uint4 x = piece(at + b * units * kUnitPieces, u, 0, p);
          M::mma(acc[b], w[0][0], w[1][0], w[0][1], w[1][1], x.x, x.y);
          M::mma(acc[b], w[0][2], w[1][2], w[0][3], w[1][3], x.z, x.w);
        }
      }
    } else {
      if constexpr (W::kIs4) {
        by_group<F>(w[0]);
        by_group<F>(w[1]);
      }
#pragma unroll
      for (int i = 0; i < W::kSub; ++i) {
        float part[NBL][4] = {}, odd[NBL][4] = {};
#pragma unroll
        for (int q = 0; q < W::kPieces / W::kSub; ++q) {
          const int j = i * (W::kPieces / W::kSub) + q;
          uint32_t a[2][4];
#pragma unroll
          for (int r = 0; r < 2; ++r) {
            if constexpr (W::kIs4) {
              const uint32_t lo = w[r][j], v = lo >> 8;
              a[r][0] = lo & 0x000f000fu;
              a[r][1] = v & 0x000f000fu;
              a[r][2] = lo & 0x00f000f0u;
              a[r][3] = v & 0x00f000f0u;
            } else {
#pragma unroll
              for (int n = 0; n < 2; ++n) {
                const uint32_t v = w[r][2 * j + n];
                a[r][2 * n] = ((v << 4) & 0x07f007f0u) | ((v << 8) & 0x80008000u);
                a[r][2 * n + 1] = ((v >> 4) & 0x07f007f0u) | (v & 0x80008000u);
              }
            }
          }
#pragma unroll
          for (int b = 0; b < NBL; ++b) {
#pragma unroll
            for (int p = 0; p < kParts; ++p) {
              const uint4 x = piece(at + b * units * kUnitPieces, u, j, p);
              M::mma(part[b], a[0][0], a[1][0], a[0][1], a[1][1], x.x, x.y);
              M::mma(kApart ? odd[b] : part[b], a[0][2], a[1][2], a[0][3], a[1][3], x.z, x.w);
            }
          }
        }
        float s[2], z[2];
        scales(i, s, z);
#pragma unroll
        for (int b = 0; b < NBL; ++b) {
#pragma unroll
          for (int n = 0; n < 4; ++n)
            if (kApart) part[b][n] = fmaf(odd[b][n], 1.0f / 16, part[b][n]);
          if constexpr (W::kIs4) {
            const float2 x = *reinterpret_cast<const float2*>(sums + ((b * units + u) * W::kSub + i) * 8 + 2 * (lane & 3));
#pragma unroll
            for (int r = 0; r < 2; ++r) {
              part[b][2 * r] = fmaf(-z[r], x.x, part[b][2 * r]);
              part[b][2 * r + 1] = fmaf(-z[r], x.y, part[b][2 * r + 1]);
            }
          }
#pragma unroll
          for (int n = 0; n < 4; ++n) acc[b][n] = fmaf(s[n >> 1], part[b][n], acc[b][n]);
        }
      }
    }
  }
};

// Sums of a tile's warps in shared memory: [2][block warps][NB][16 rows][8
// columns], the two halves in turn.  A half is written again two tiles later,
// after the group's barrier of the tile between.
template <int NB>
struct TileSums {
  float* base;
  int half = 0;

  __device__ __forceinline__ explicit TileSums(void* smem) : base(static_cast<float*>(smem)) {}
  __host__ __device__ static constexpr int bytes(int warps) { return 2 * warps * NB * 512; }

  // Leaves this warp's sums, clears them and waits for the group's.
  __device__ __forceinline__ const float* join(float (&acc)[NB][4], const TileGroup& g) {
    const int lane = threadIdx.x & 31, warps = blockDim.x >> 5;
    float* mine = base + (half * warps + (threadIdx.x >> 5)) * NB * 128 + (lane >> 2) * 8 + 2 * (lane & 3);
#pragma unroll
    for (int b = 0; b < NB; ++b)
#pragma unroll
      for (int r = 0; r < 2; ++r) {
        *reinterpret_cast<float2*>(mine + b * 128 + r * 64) = make_float2(acc[b][2 * r], acc[b][2 * r + 1]);
        acc[b][2 * r] = acc[b][2 * r + 1] = 0.0f;
      }
    g.sync();
    const float* sums = base + (half * warps + g.id * g.warps) * NB * 128;
    half ^= 1;
    return sums;
  }
  // The group's sum of a row and column, in warp order.
  static __device__ __forceinline__ float sum(const float* sums, const TileGroup& g, int row, int block, int col) {
    float v = 0.0f;
#pragma unroll 4
    for (int w = 0; w < g.warps; ++w) v += sums[w * NB * 128 + block * 128 + row * 8 + col];
    return v;
  }
};

// Weights are read once: past L1, a few units ahead into L2.
__device__ __forceinline__ void load_weights(uint32_t (&w)[4], const uint8_t* p) {
  asm volatile("ld.global.nc.L1::no_allocate.L2::256B.v4.u32 {%0,%1,%2,%3}, [%4];\n"
               : "=r"(w[0]), "=r"(w[1]), "=r"(w[2]), "=r"(w[3])
               : "l"(p));
}

// Brings the first `bytes` (a multiple of 16) from p on into L2.
__device__ __forceinline__ void prefetch_weights(const uint8_t* p, int64_t bytes) {
  asm volatile("cp.async.bulk.prefetch.L2.global [%0], %1;\n" ::"l"(p), "r"(static_cast<uint32_t>(bytes)) : "memory");
}

// The lane's two rows of a tile (fragment rows lane / 4 and lane / 4 + 8), from
// 16 (lane % 4) bytes on.
struct TileRows {
  const uint8_t* data[2];
  const float* scale[2];  // e4m3: of the row's blocks
};

// A warp's share of a run of tiles.  `source` knows the tiles: source.rows(i)
// are the lane's rows of the group's i-th tile, source.scales(i, row) tells
// where the scales of a row of it are and source.here the same for the tile now
// consumed, source.zeros whether there are zero points and source.rows_wide
// what scales_wide says of the arrays (4-bit only).  Each is
// asked for the tiles in order.  source.met_nan() hears of e4m3 NaN, which count
// as 480 otherwise.  finish(i, sums) may move xt to the next tile's
// columns.
template <int F, typename T, int kStep>
struct TileStream {
  using W = WTraits<F>;
  struct Unit {
    uint32_t w[2][4];
    float s[2];  // e4m3
  } quad[kStep];
  TileRows at;  // of the tile whose units are loaded next
  ScaleTile<F> sc;
  int k, u0, u1, count, g0, g1;

  // Units u .. u + 3.  What lies past the end of a row reads as its last bytes
  // again; the activations there are zeros.
  template <bool kWhole>
  __device__ __forceinline__ void load(const TileRows& from, int u) {
    const int last = static_cast<int>(W::row_bytes(k)) - 16 * (1 + (static_cast<int>(threadIdx.x) & 3));
#pragma unroll
    for (int d = 0; d < kStep; ++d) load_unit<kWhole>(quad[d], from, u, d, last);
  }
  template <bool kWhole>
  __device__ __forceinline__ void load_unit(Unit& to, const TileRows& from, int u, int d, int last) const {
    const int off = kWhole ? u * 64 : min((u + d) * 64, last);
#pragma unroll
    for (int r = 0; r < 2; ++r) {
      load_weights(to.w[r], from.data[r] + off + (kWhole ? d * 64 : 0));
      if (F == kWFp8) to.s[r] = __ldg(from.scale[r] + (kWhole ? (u + d) / 2 : min((u + d) / 2, (k - 1) / 128)));  // blocks of 128
    }
  }
  template <typename Source>
  __device__ __forceinline__ void fetch_scales(int i, Source& source) const {
    if constexpr (W::kIs4) {
      if (i < count) sc.fetch(i, source.scales(i, threadIdx.x & 15), g0, g1);
      asm volatile("cp.async.commit_group;\n" ::: "memory");
    }
  }
  // Starts the loads of `count` tiles of rows of k, this warp's share of each;
  // `smem` is for the scales, of ScaleTile::bytes(units, ...) at most.  Runs
  // that no block barrier parts have to name the same `scale_units`, those of
  // the longest: the warps' areas lie by it, and one warp may be a run ahead.
  template <typename Source>
  __device__ __forceinline__ void start(int k_, const TileGroup& g, int count_, uint8_t* smem, Source& source, int scale_units) {
    const int units = W::units(k_);
    k = k_, u0 = g.first_unit(units), u1 = g.end_unit(units), count = count_;
    if (count > 0) {
      at = source.rows(0);
      load<false>(at, u0);
    }
    if constexpr (W::kIs4) {
      g0 = min(u0 * W::kSub, k / W::kGroupK), g1 = min(u1 * W::kSub, k / W::kGroupK);
      sc.init(smem, scale_units, source.zeros(), g.warps, source.rows_wide(), g0, g1);
      __syncwarp();  // the last run's scales have been read
      fetch_scales(0, source);
      fetch_scales(1, source);
    }
  }
  // Consumes them; finish(i, sums) for each tile, in order.
  template <int NBL, typename X, typename Sums, int NB, typename Source, typename Finish>
  __device__ __forceinline__ void run(X& xt, const TileGroup& g, Sums& ts, float (&acc)[NB][4], Source& source, Finish finish) {
    if (k % (4 * W::kUnitK) == 0) run_tiles<NBL, true>(xt, g, ts, acc, source, finish);
    else run_tiles<NBL, false>(xt, g, ts, acc, source, finish);
  }
  template <int NBL, bool kWhole, typename X, typename Sums, int NB, typename Source, typename Finish>
  __device__ __forceinline__ void run_tiles(X& xt, const TileGroup& g, Sums& ts, float (&acc)[NB][4], Source& source, Finish finish) {
    const bool zeros = W::kIs4 && source.zeros();
    const int last = static_cast<int>(W::row_bytes(k)) - 16 * (1 + (static_cast<int>(threadIdx.x) & 3));
#pragma unroll 1
    for (int i = 0; i < count; ++i) {
      const uint8_t *srow[2], *zrow[2];  // of the lane's rows, at group 0
      if constexpr (W::kIs4) {
        asm volatile("cp.async.wait_group 1;\n" ::: "memory");  // all but the next tile's
        __syncwarp();
#pragma unroll
        for (int r = 0; r < 2; ++r) {
          const int row = ((threadIdx.x & 31) >> 2) + 8 * r;
          srow[r] = sc.row(i, row) - 2 * g0;
          zrow[r] = sc.row(i, row) + sc.zero_at - g0;
          if (!sc.wide) {
            const WScales from = source.here(i, row);
            srow[r] += reinterpret_cast<uintptr_t>(from.scale + 2 * g0) & 3;
            zrow[r] += reinterpret_cast<uintptr_t>(from.zero + g0) & 3;
          }
        }
      }
      uint32_t nans = 0;
#pragma unroll 1
      for (int u = u0; u < u1; u += kStep) {
        // the quad after this one: the tile's next, or the next tile's first
        // (after the last tile its own first again, which nothing reads)
        const bool ends = u + kStep >= u1;
        if (ends && i + 1 < count) at = source.rows(i + 1);
        const int next = ends ? u0 : u + kStep;
#pragma unroll
        for (int d = 0; d < kStep; ++d) {
          xt.template consume<NBL>(acc, quad[d].w, u + d, [&](int j, float (&s)[2], float (&z)[2]) {
            if constexpr (W::kIs4) {
              const int n = (u + d) * W::kSub + j;
              const bool in = kWhole || n < g1;  // no group: x is zero there
#pragma unroll
              for (int r = 0; r < 2; ++r) {
                s[r] = in ? MmaType<T>::to_float(*reinterpret_cast<const uint16_t*>(srow[r] + 2 * n)) : 0.0f;
                z[r] = zeros ? static_cast<float>(zrow[r][n]) : 8.0f;
              }
            } else {
              s[0] = quad[d].s[0], s[1] = quad[d].s[1];
            }
          });
          if constexpr (F == kWFp8) {
            // Adding 1 to a byte turns its bit 7 over if the others are ones, an
            // e4m3 NaN's; what 0xff carries into the next is of the same tile.
            // (116 -> 122 us for the e4m3 layer with 8 tokens; putting a NaN into
            // the product on the spot 125.)
#pragma unroll
            for (int n = 0; n < 8; ++n) nans |= quad[d].w[n >> 2][n & 3] ^ (quad[d].w[n >> 2][n & 3] + 0x01010101u);
          }
          load_unit<kWhole>(quad[d], at, next, d, last);
        }
      }
      if constexpr (W::kIs4) {
        __syncwarp();  // this tile's scales have been read
        fetch_scales(i + 2, source);
      }
      if constexpr (F == kWFp8)
        if (nans & 0x80808080u) source.met_nan();
      finish(i, ts.join(acc, g));
    }
  }
};

}  // namespace hca
