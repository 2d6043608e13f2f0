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
// at a time: 32 bf16, 64 e4m3 (16 bytes a lane in one load) or 128 4-bit
// codes (16 bytes a lane; one load, or two or four for groups of 64 and 32,
// so that each load stays inside a group).  Sums are held in 32 bits; group
// and block scales multiply the 32-bit sums of their own groups.
//
// No code is converted.  The smallest floats of a 16-bit type are evenly
// spaced: bits 0..7 of a bf16 (0..10 of an fp16) with nothing above them are
// the number times 2^-133 (2^-24), across the end of the subnormals.  So a
// word of 4-bit codes, masked, is two codes as exact floats, and those four
// bits higher are 16 times theirs: five bit operations for eight codes, and
// the sums of the two kinds meet as a + b / 16.  e4m3 moved into the low
// exponent and high mantissa bits of a bf16 is its value times 2^-120, the
// subnormals with it.  bf16 activations are scaled by 2^80 when they are laid
// out, so that the products keep clear of both ends of the 32-bit range for
// |x| from 2^-73 to 2^47, and the powers of two leave with the finished sum.
// An e4m3 NaN would count as 480; an infinite x makes its row NaN.
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
  // loads of a row for a unit, each inside one group
  static constexpr int kSub = F == kW4G32 ? 4 : F == kW4G64 ? 2 : 1;
  static constexpr int kWords = 4 / kSub;              // 32-bit words of a load and lane
  static constexpr int kPieces = kUnitK / 32;          // 16-byte activation pieces of a lane and column
  static constexpr int kGroupK = kUnitK / kSub;        // reduction length of a load
  static constexpr int kLaneK = kGroupK / 4;           // and of a lane's share of it
  __host__ __device__ static constexpr int64_t row_bytes(int64_t k) {
    return F == kWBf16 ? 2 * k : F == kWFp8 ? k : k / 2;
  }
  __host__ __device__ static constexpr int units(int k) { return (k + kUnitK - 1) / kUnitK; }
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
  static constexpr float kSum = kHalf ? 0x1p-24f : 0x1p-53f;
  static constexpr float kOut = F == kWBf16 ? 1.0f : kHalf ? 0x1p24f : F == kWFp8 ? 0x1p40f : 0x1p53f;
};

// Weights are read once: past L1.
template <int kWords>
__device__ __forceinline__ void load_words(uint32_t* w, const uint8_t* p) {
  if constexpr (kWords == 4) {
    asm volatile("ld.global.nc.L1::no_allocate.L2::256B.v4.u32 {%0,%1,%2,%3}, [%4];\n"
                 : "=r"(w[0]), "=r"(w[1]), "=r"(w[2]), "=r"(w[3])
                 : "l"(p));
  } else if constexpr (kWords == 2) {
    asm volatile("ld.global.nc.L1::no_allocate.L2::256B.v2.u32 {%0,%1}, [%2];\n" : "=r"(w[0]), "=r"(w[1]) : "l"(p));
  } else {
    // 16 bytes of a row at a time: the other half of the sector is the next load's
    asm volatile("ld.global.nc.L2::256B.u32 %0, [%1];\n" : "=r"(w[0]) : "l"(p));
  }
}

// A unit of two rows on its way from memory.
template <int F>
struct WStep {
  static constexpr int kScales = F == kWBf16 ? 0 : WTraits<F>::kSub;
  uint32_t w[2][4];
  uint32_t s[2][kScales > 0 ? kScales : 1];  // bits of the scales
  uint32_t z[2][WTraits<F>::kIs4 ? kScales : 1];
};

// A lane's two rows of a tile (fragment rows lane / 4 and lane / 4 + 8), read
// unit after unit.  Lanes whose share of a row's last unit lies past its end
// read its last bytes again; the activations there are zeros.
template <int F>
struct WCursor {
  using W = WTraits<F>;
  const uint8_t* data[2];
  const void* scale[2];    // 4-bit: 16-bit scales of the row's groups; e4m3: fp32 scales of its blocks
  const uint8_t* zero[2];  // zero points of the row's groups, or null
  int unit;

  // kRagged: k may end inside a unit (never for bf16 and groups of 128)
  static constexpr bool kRagged = F == kWFp8 || F == kW4G32 || F == kW4G64;

  // data[] of lane c starts c * 4 kWords bytes into the row
  __device__ __forceinline__ void load(WStep<F>& st, int k) {
    constexpr int kBytes = static_cast<int>(W::row_bytes(W::kUnitK));
#pragma unroll
    for (int i = 0; i < W::kSub; ++i) {
      int off = unit * kBytes + i * 16 * W::kWords;
      if (kRagged) off = min(off, static_cast<int>(W::row_bytes(k)) - 4 * W::kWords * (1 + (static_cast<int>(threadIdx.x) & 3)));
#pragma unroll
      for (int r = 0; r < 2; ++r) load_words<W::kWords>(&st.w[r][i * W::kWords], data[r] + off);
    }
    if constexpr (W::kIs4) {
#pragma unroll
      for (int i = 0; i < W::kSub; ++i) {
        int g = unit * W::kSub + i;
        if (kRagged) g = min(g, k / W::kGroupK - 1);
#pragma unroll
        for (int r = 0; r < 2; ++r) {
          st.s[r][i] = __ldg(static_cast<const uint16_t*>(scale[r]) + g);
          st.z[r][i] = 8;
          if (zero[r] != nullptr) st.z[r][i] = __ldg(zero[r] + g);
        }
      }
    } else if constexpr (F == kWFp8) {
#pragma unroll
      for (int r = 0; r < 2; ++r)
        st.s[r][0] = __float_as_uint(__ldg(static_cast<const float*>(scale[r]) + unit / 2));  // blocks of 128
    }
    ++unit;
  }
};

// Place of the 16-byte piece that holds column col's activations k .. k + 7
// (k a multiple of 8) among the pieces of a block of columns: the pieces of a
// unit follow each other, each 4 kWidth lanes wide.
template <int F, int kWidth>
__device__ __forceinline__ int piece_index(int k, int col) {
  using W = WTraits<F>;
  const int u = k / W::kUnitK, i = k % W::kUnitK / W::kGroupK, c = k % W::kGroupK / W::kLaneK;
  const int j = i * (W::kLaneK / 8) + k % W::kLaneK / 8;
  return ((u * W::kPieces + j) * kWidth + col) * 4 + c;
}

// Eight consecutive activations in a piece's order, that in which weights come
// out of a word together: codes 0,4 2,6 1,5 3,7 and e4m3 0,2 1,3 of each four.
template <int F, typename T>
__device__ __forceinline__ uint4 piece_order(uint4 v) {
  using M = MmaType<T>;
  constexpr float kX = Scaling<F, T>::kX;
  if constexpr (kX != 1.0f) {
    const float2 a = M::unpack(v.x), b = M::unpack(v.y), c = M::unpack(v.z), d = M::unpack(v.w);
    v = make_uint4(M::pack(a.x * kX, a.y * kX), M::pack(b.x * kX, b.y * kX), M::pack(c.x * kX, c.y * kX),
                   M::pack(d.x * kX, d.y * kX));
  }
  if constexpr (WTraits<F>::kIs4)
    return make_uint4(__byte_perm(v.x, v.z, 0x5410), __byte_perm(v.y, v.w, 0x5410), __byte_perm(v.x, v.z, 0x7632),
                      __byte_perm(v.y, v.w, 0x7632));
  if constexpr (F == kWFp8)
    return make_uint4(__byte_perm(v.x, v.y, 0x5410), __byte_perm(v.x, v.y, 0x7632), __byte_perm(v.z, v.w, 0x5410),
                      __byte_perm(v.z, v.w, 0x7632));
  return v;
}

// Activations of NB blocks of columns in shared memory, in piece order, with
// their group sums.  A block has 8 columns, of which kWidth are stored.
template <int F, typename T, int NB, int kWidth>
struct XTile {
  using W = WTraits<F>;
  uint4* pieces;  // [NB][units][kPieces][kWidth][4]
  float* sums;    // [NB][units][kSub][8], 4-bit only
  int units;

  static constexpr int kUnitPieces = W::kPieces * kWidth * 4;
  static constexpr int kColumns = NB * kWidth;

  __host__ __device__ static int64_t bytes(int units) {
    return NB * static_cast<int64_t>(units) * (kUnitPieces * 16 + (W::kIs4 ? W::kSub * 32 : 0));
  }

  __device__ __forceinline__ XTile(uint8_t* smem, int units_) : units(units_) {
    pieces = reinterpret_cast<uint4*>(smem);
    sums = reinterpret_cast<float*>(smem + static_cast<int64_t>(NB) * units * kUnitPieces * 16);
  }

  // All threads of the block; row(col) is column col's row of k values or
  // null (zeros, as in the columns after `columns`).  Ends with a block barrier.
  template <typename Row>
  __device__ __forceinline__ void stage(int k, int columns, int live, Row row) {
    const int padded = units * W::kUnitK;
    // several columns' loads under way at a time
    constexpr int kAhead = kWidth < 4 ? kWidth : 4;
    for (int c0 = 0; c0 < live * kWidth; c0 += kAhead) {
      const T* p[kAhead];
#pragma unroll
      for (int n = 0; n < kAhead; ++n) p[n] = c0 + n < columns ? row(c0 + n) : nullptr;
      uint4* to = pieces + c0 / kWidth * units * kUnitPieces;
      for (int i = threadIdx.x * 8; i < padded; i += blockDim.x * 8) {
        uint4 v[kAhead];
#pragma unroll
        for (int n = 0; n < kAhead; ++n)
          v[n] = p[n] != nullptr && i < k ? *reinterpret_cast<const uint4*>(p[n] + i) : make_uint4(0, 0, 0, 0);
#pragma unroll
        for (int n = 0; n < kAhead; ++n)
          to[piece_index<F, kWidth>(i, (c0 + n) % kWidth)] = piece_order<F, T>(v[n]);
      }
    }
    __syncthreads();
    if constexpr (W::kIs4) {
      const int lane = threadIdx.x & 31;
      const int groups = live * units * W::kSub;
      for (int g = threadIdx.x >> 5; g < groups; g += blockDim.x >> 5) {
        constexpr int kEach = W::kPieces / W::kSub;
        float v = 0.0f;
        if (lane < kWidth * 4) {
#pragma unroll
          for (int q = 0; q < kEach; ++q) {
            const uint4 x = pieces[(g * kEach + q) * kWidth * 4 + lane];
            const float2 a = MmaType<T>::unpack(x.x), b = MmaType<T>::unpack(x.y), c = MmaType<T>::unpack(x.z),
                         d = MmaType<T>::unpack(x.w);
            v += ((a.x + a.y) + (b.x + b.y)) + ((c.x + c.y) + (d.x + d.y));
          }
        }
        v += __shfl_xor_sync(0xffffffffu, v, 1);
        v += __shfl_xor_sync(0xffffffffu, v, 2);
        using S = Scaling<F, T>;
        v = v * S::kSum * (1.0f / S::kX);
        if ((lane & 3) == 0) sums[g * 8 + (lane >> 2)] = v;
      }
      __syncthreads();
    }
  }

  // acc[b] += the step's rows times the columns of block b < NBL, over unit u.
  template <int NBL>
  __device__ __forceinline__ void consume(float (&acc)[NB][4], const WStep<F>& st, int u) const {
    using M = MmaType<T>;
    const int lane = threadIdx.x & 31;
    const uint4* at = pieces + u * kUnitPieces + lane;
    auto piece = [&](int b, int j) -> uint4 {
      const uint4* p = at + b * units * kUnitPieces + j * kWidth * 4;
      if (kWidth == 8) return *p;
      return lane < kWidth * 4 ? *p : make_uint4(0, 0, 0, 0);
    };
    if constexpr (F == kWBf16) {
#pragma unroll
      for (int b = 0; b < NBL; ++b) {
        const uint4 x = piece(b, 0);
        M::mma(acc[b], st.w[0][0], st.w[1][0], st.w[0][1], st.w[1][1], x.x, x.y);
        M::mma(acc[b], st.w[0][2], st.w[1][2], st.w[0][3], st.w[1][3], x.z, x.w);
      }
    } else {
#pragma unroll
      for (int i = 0; i < W::kSub; ++i) {
        float part[NBL][4] = {}, high[NBL][4] = {};
#pragma unroll
        for (int q = 0; q < W::kPieces / W::kSub; ++q) {
          const int j = i * (W::kPieces / W::kSub) + q;
          uint32_t a[2][4];
#pragma unroll
          for (int r = 0; r < 2; ++r) {
            if constexpr (W::kIs4) {
              const uint32_t w = st.w[r][j], v = w >> 8;
              a[r][0] = w & 0x000f000fu;
              a[r][1] = v & 0x000f000fu;
              a[r][2] = w & 0x00f000f0u;
              a[r][3] = v & 0x00f000f0u;
            } else {
#pragma unroll
              for (int n = 0; n < 2; ++n) {
                const uint32_t w = st.w[r][2 * j + n];
                a[r][2 * n] = ((w << 4) & 0x07f007f0u) | ((w << 8) & 0x80008000u);
                a[r][2 * n + 1] = ((w >> 4) & 0x07f007f0u) | (w & 0x80008000u);
              }
            }
          }
#pragma unroll
          for (int b = 0; b < NBL; ++b) {
            const uint4 x = piece(b, j);
            M::mma(part[b], a[0][0], a[1][0], a[0][1], a[1][1], x.x, x.y);
            M::mma(high[b], a[0][2], a[1][2], a[0][3], a[1][3], x.z, x.w);
          }
        }
        float s[2];
#pragma unroll
        for (int r = 0; r < 2; ++r)
          s[r] = W::kIs4 ? M::to_float(static_cast<uint16_t>(st.s[r][i])) : __uint_as_float(st.s[r][i]);
#pragma unroll
        for (int b = 0; b < NBL; ++b) {
#pragma unroll
          for (int n = 0; n < 4; ++n) part[b][n] = W::kIs4 ? fmaf(high[b][n], 1.0f / 16, part[b][n]) : part[b][n] + high[b][n];
          if constexpr (W::kIs4) {
            const float2 x = *reinterpret_cast<const float2*>(sums + ((b * units + u) * W::kSub + i) * 8 + 2 * (lane & 3));
#pragma unroll
            for (int r = 0; r < 2; ++r) {
              const float z = -static_cast<float>(st.z[r][i]);
              part[b][2 * r] = fmaf(z, x.x, part[b][2 * r]);
              part[b][2 * r + 1] = fmaf(z, x.y, part[b][2 * r + 1]);
            }
          }
#pragma unroll
          for (int n = 0; n < 4; ++n) acc[b][n] = fmaf(s[n >> 1], part[b][n], acc[b][n]);
        }
      }
    }
  }
};

// The warps that share a tile: warp `index` of `warps`, group `id` of the
// block.  They take the tile's units in even runs and add their sums here.
struct TileGroup {
  int warps, index, id;

  __device__ __forceinline__ explicit TileGroup(int warps_)
      : warps(warps_), index((threadIdx.x >> 5) % warps_), id((threadIdx.x >> 5) / warps_) {}
  __device__ __forceinline__ int first_unit(int units) const { return units * index / warps; }
  __device__ __forceinline__ int end_unit(int units) const { return units * (index + 1) / warps; }
  __device__ __forceinline__ int threads() const { return warps * 32; }
  __device__ __forceinline__ int thread() const { return index * 32 + (threadIdx.x & 31); }

  // Waits for the whole group; barriers 1..15 are the groups'.
  __device__ __forceinline__ void sync() const {
    if (warps == 1) __syncwarp();
    else asm volatile("bar.sync %0, %1;\n" ::"r"(1 + id), "r"(warps * 32) : "memory");
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

// Units of a run of tiles on their way: kDepth of them, across the ends of
// tiles.  rows(cur, i) points the cursor at the rows of the group's i-th tile.
template <int F>
struct TileRing {
  // groups of 32 bring eight scales and zero points a unit
  static constexpr int kDepth = F == kW4G32 ? 3 : 4;
  WStep<F> st[kDepth];
  WCursor<F> cur;
  int k, u0, u1, next, count;

  template <typename Rows>
  __device__ __forceinline__ void load(WStep<F>& s, Rows& rows) {
    if (next >= count) return;
    cur.load(s, k);
    if (cur.unit == u1) {
      ++next;
      if (next < count) rows(cur, next);
      cur.unit = u0;
    }
  }
  // Starts the loads of `count` tiles of rows of k, this warp's share of each.
  template <typename Rows>
  __device__ __forceinline__ void start(int k_, const TileGroup& g, int count_, Rows rows) {
    const int units = WTraits<F>::units(k_);
    k = k_, u0 = g.first_unit(units), u1 = g.end_unit(units), next = 0, count = count_;
    cur.unit = u0;
    if (count > 0) rows(cur, 0);
#pragma unroll
    for (int d = 0; d < kDepth; ++d) load(st[d], rows);
  }
  // Consumes them; finish(i, sums) for each tile, in order.
  template <int NBL, typename X, typename Sums, int NB, typename Rows, typename Finish>
  __device__ __forceinline__ void run(const X& xt, const TileGroup& g, Sums& ts, float (&acc)[NB][4], Rows rows, Finish finish) {
    int u = u0, i = 0;
    while (i < count) {
#pragma unroll
      for (int d = 0; d < kDepth; ++d) {
        xt.template consume<NBL>(acc, st[d], u);
        load(st[d], rows);
        if (++u < u1) continue;
        finish(i, ts.join(acc, g));
        u = u0;
        if (++i >= count) break;
      }
    }
  }
};

}  // namespace hca
