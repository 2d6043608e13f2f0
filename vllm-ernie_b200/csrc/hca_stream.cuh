// Streaming products of weights with a few rows of activations on the
// warp-level tensor instructions: the part that the 4-bit linear and the
// mixture-of-experts kernels share.
//
// A step with few rows is bound by the bytes of its weights, so the weights
// are the 16 rows of an m16n8k16 product and up to eight activation rows its
// 8 columns: each weight goes from memory to registers once, and is used for
// every row.  (tcgen05 needs its operands in shared memory and at least 64
// rows of a tile filled; here the weights would pass through shared memory
// only to meet a tile that is nearly empty.)  The reduction index may be
// permuted freely as long as both operands agree, so a lane's fragment is
// whatever consecutive bytes one wide load of a row brings: no ldmatrix, no
// repacked weights, and checkpoints' row-major layouts are read as they are.
//
// A "unit" is the piece of a row that the four lanes of a fragment row load at
// once: 32 bf16, 64 e4m3, or one group of 4-bit codes.  Products of 4-bit
// codes (q - z, whole numbers) and of e4m3 values are exact in bf16/fp16;
// sums are held in 32 bits, and group or block scales multiply the 32-bit
// sums of their own groups.
#pragma once

#include <cuda_fp16.h>

#include "hca_common.cuh"

namespace hca {

enum WFormat : int { kWBf16 = 0, kWFp8 = 1, kW4G32 = 2, kW4G64 = 3, kW4G128 = 4 };

template <int F>
struct WTraits {
  static constexpr bool kIs4 = F >= kW4G32;
  // 32-bit words of one row that a lane loads for a unit
  static constexpr int kWords = F == kW4G32 ? 1 : F == kW4G64 ? 2 : 4;
  // reduction length of a unit, and of one lane's share of it
  static constexpr int kLaneK = F == kWBf16 ? 8 : F == kWFp8 ? 16 : 8 * kWords;
  static constexpr int kUnitK = 4 * kLaneK;
  // units loaded together: 2 rows x kBatch loads per lane in flight, twice
  static constexpr int kBatch = F == kW4G32 ? 8 : 4;
  // bytes of a row of `k` weights
  __host__ __device__ static constexpr int64_t row_bytes(int64_t k) {
    return F == kWBf16 ? 2 * k : F == kWFp8 ? k : k / 2;
  }
};

template <typename T>
struct MmaType;
template <>
struct MmaType<__nv_bfloat16> {
  static __device__ __forceinline__ void mma(float (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3,
                                             uint32_t b0, uint32_t b1) {
    asm volatile(
        "mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};\n"
        : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
        : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
  }
  // 128.0: its ulp is 1, so or-ing a 4-bit code into the mantissa adds it
  static constexpr uint32_t kMagic = 0x43004300u;
  static constexpr float kMagicValue = 128.0f;
  static __device__ __forceinline__ uint32_t pack(float lo, float hi) {
    __nv_bfloat162 v = __floats2bfloat162_rn(lo, hi);
    return *reinterpret_cast<uint32_t*>(&v);
  }
  static __device__ __forceinline__ uint32_t sub(uint32_t a, uint32_t b) {
    __nv_bfloat162 v = __hsub2(*reinterpret_cast<__nv_bfloat162*>(&a), *reinterpret_cast<__nv_bfloat162*>(&b));
    return *reinterpret_cast<uint32_t*>(&v);
  }
  static __device__ __forceinline__ float to_float(__nv_bfloat16 v) { return __bfloat162float(v); }
  static __device__ __forceinline__ __nv_bfloat16 from_float(float v) { return __float2bfloat16_rn(v); }
};
template <>
struct MmaType<__half> {
  static __device__ __forceinline__ void mma(float (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3,
                                             uint32_t b0, uint32_t b1) {
    asm volatile(
        "mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};\n"
        : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
        : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
  }
  static constexpr uint32_t kMagic = 0x64006400u;  // 1024.0, ulp 1
  static constexpr float kMagicValue = 1024.0f;
  static __device__ __forceinline__ uint32_t pack(float lo, float hi) {
    __half2 v = __floats2half2_rn(lo, hi);
    return *reinterpret_cast<uint32_t*>(&v);
  }
  static __device__ __forceinline__ uint32_t sub(uint32_t a, uint32_t b) {
    __half2 v = __hsub2(*reinterpret_cast<__half2*>(&a), *reinterpret_cast<__half2*>(&b));
    return *reinterpret_cast<uint32_t*>(&v);
  }
  static __device__ __forceinline__ float to_float(__half v) { return __half2float(v); }
  static __device__ __forceinline__ __half from_float(float v) { return __float2half_rn(v); }
};

// Weights are read once: past L1, so that it keeps the activations.
template <int kWords>
__device__ __forceinline__ void load_words(uint32_t (&w)[kWords], const uint8_t* p) {
  if constexpr (kWords == 4) {
    asm volatile("ld.global.nc.L1::no_allocate.v4.u32 {%0,%1,%2,%3}, [%4];\n"
                 : "=r"(w[0]), "=r"(w[1]), "=r"(w[2]), "=r"(w[3])
                 : "l"(p));
  } else if constexpr (kWords == 2) {
    asm volatile("ld.global.nc.L1::no_allocate.v2.u32 {%0,%1}, [%2];\n" : "=r"(w[0]), "=r"(w[1]) : "l"(p));
  } else {
    // 16 bytes of a row at a time: the other half of the sector is the next load's
    asm volatile("ld.global.nc.u32 %0, [%1];\n" : "=r"(w[0]) : "l"(p));
  }
}

// Four e4m3 bytes to two 16-bit pairs (exact: e4m3 fits both types).
template <typename T>
__device__ __forceinline__ void unpack_fp8(uint32_t w, uint32_t& p0, uint32_t& p1) {
  const float2 a = e4m3x2_to_float2(static_cast<uint16_t>(w));
  const float2 b = e4m3x2_to_float2(static_cast<uint16_t>(w >> 16));
  p0 = MmaType<T>::pack(a.x, a.y);
  p1 = MmaType<T>::pack(b.x, b.y);
}

// Eight 4-bit codes to four pairs (codes 0,4 | 1,5 | 2,6 | 3,7), each code
// minus the zero point: or-ed into the mantissa of 128 (1024), then 128 + z
// (1024 + z) is subtracted; both steps are exact.
template <typename T>
__device__ __forceinline__ void unpack_w4(uint32_t w, uint32_t offset, uint32_t (&p)[4]) {
#pragma unroll
  for (int i = 0; i < 4; ++i)
    p[i] = MmaType<T>::sub(((w >> (4 * i)) & 0x000f000fu) | MmaType<T>::kMagic, offset);
}

// The two weight rows of a lane (fragment rows lane / 4 and lane / 4 + 8).
template <typename T>
struct WRows {
  const uint8_t* data[2];
  // 4-bit: scales (and zero points, or null) of the row's groups; e4m3: fp32
  // scales of the row's blocks
  const void* scale[2];
  const uint8_t* zero[2];
};

// acc[b] += rows . x^T for units [begin, end) of rows of k weights.  x_off[b]
// is the element offset of column b * 8 + lane / 4 in x, negative where the
// column is empty; blocks from `live` on are skipped.  Lanes past the end of a
// row (e4m3 units of a row that ends inside) take zeros.
template <int F, typename T, int NB>
__device__ __forceinline__ void stream_rows(float (&acc)[NB][4], const WRows<T>& rows, const T* x,
                                            const int64_t (&x_off)[NB], int live, int k, int begin, int end) {
  using W = WTraits<F>;
  constexpr int kB = W::kBatch;
  const int c = threadIdx.x & 3;
  const uint8_t* p0 = rows.data[0] + c * W::row_bytes(W::kLaneK);
  const uint8_t* p1 = rows.data[1] + c * W::row_bytes(W::kLaneK);
  constexpr int kStep = static_cast<int>(W::row_bytes(W::kUnitK));

  uint32_t cur[kB][2][W::kWords], nxt[kB][2][W::kWords];
  auto load = [&](uint32_t (&buf)[kB][2][W::kWords], int u0) {
#pragma unroll
    for (int i = 0; i < kB; ++i) {
      const int u = u0 + i;
      if (u < end && (W::kIs4 || u * W::kUnitK + c * W::kLaneK < k)) {
        load_words<W::kWords>(buf[i][0], p0 + static_cast<int64_t>(u) * kStep);
        load_words<W::kWords>(buf[i][1], p1 + static_cast<int64_t>(u) * kStep);
      } else {
#pragma unroll
        for (int j = 0; j < W::kWords; ++j) buf[i][0][j] = buf[i][1][j] = 0;
      }
    }
  };
  load(cur, begin);
  for (int u0 = begin; u0 < end; u0 += kB) {
    load(nxt, u0 + kB);
#pragma unroll
    for (int i = 0; i < kB; ++i) {
      const int u = u0 + i;
      if (u >= end) break;
      const int k0 = u * W::kUnitK + c * W::kLaneK;
      const bool in = k0 < k;
      float s0 = 1.0f, s1 = 1.0f;
      uint32_t off0 = 0, off1 = 0;
      if constexpr (W::kIs4) {
        s0 = MmaType<T>::to_float(reinterpret_cast<const T*>(rows.scale[0])[u]);
        s1 = MmaType<T>::to_float(reinterpret_cast<const T*>(rows.scale[1])[u]);
        float z0 = 8.0f, z1 = 8.0f;
        if (rows.zero[0] != nullptr) {
          z0 = rows.zero[0][u];
          z1 = rows.zero[1][u];
        }
        off0 = MmaType<T>::pack(MmaType<T>::kMagicValue + z0, MmaType<T>::kMagicValue + z0);
        off1 = MmaType<T>::pack(MmaType<T>::kMagicValue + z1, MmaType<T>::kMagicValue + z1);
      } else if constexpr (F == kWFp8) {
        const int b = u * W::kUnitK / 128;
        s0 = reinterpret_cast<const float*>(rows.scale[0])[b];
        s1 = reinterpret_cast<const float*>(rows.scale[1])[b];
      }
      float part[NB][4] = {};
      // eight (4-bit, bf16) or four (e4m3) activations of a column at a time
      constexpr int kPieces = W::kLaneK / 8;
#pragma unroll
      for (int j = 0; j < kPieces; ++j) {
        uint32_t a0[4], a1[4];
        if constexpr (F == kWBf16) {
#pragma unroll
          for (int q = 0; q < 4; ++q) a0[q] = cur[i][0][q], a1[q] = cur[i][1][q];
        } else if constexpr (F == kWFp8) {
          unpack_fp8<T>(cur[i][0][2 * j], a0[0], a0[1]);
          unpack_fp8<T>(cur[i][0][2 * j + 1], a0[2], a0[3]);
          unpack_fp8<T>(cur[i][1][2 * j], a1[0], a1[1]);
          unpack_fp8<T>(cur[i][1][2 * j + 1], a1[2], a1[3]);
        } else {
          unpack_w4<T>(cur[i][0][j], off0, a0);
          unpack_w4<T>(cur[i][1][j], off1, a1);
        }
#pragma unroll
        for (int b = 0; b < NB; ++b) {
          if (b < live) {
            uint4 v = make_uint4(0, 0, 0, 0);
            if (in && x_off[b] >= 0) v = *reinterpret_cast<const uint4*>(x + x_off[b] + k0 + 8 * j);
            float(&d)[4] = F == kWBf16 ? acc[b] : part[b];
            if constexpr (W::kIs4) {
              MmaType<T>::mma(d, a0[0], a1[0], a0[1], a1[1], __byte_perm(v.x, v.z, 0x5410),
                              __byte_perm(v.x, v.z, 0x7632));
              MmaType<T>::mma(d, a0[2], a1[2], a0[3], a1[3], __byte_perm(v.y, v.w, 0x5410),
                              __byte_perm(v.y, v.w, 0x7632));
            } else {
              MmaType<T>::mma(d, a0[0], a1[0], a0[1], a1[1], v.x, v.y);
              MmaType<T>::mma(d, a0[2], a1[2], a0[3], a1[3], v.z, v.w);
            }
          }
        }
      }
      if constexpr (F != kWBf16) {
#pragma unroll
        for (int b = 0; b < NB; ++b) {
          acc[b][0] += s0 * part[b][0];
          acc[b][1] += s0 * part[b][1];
          acc[b][2] += s1 * part[b][2];
          acc[b][3] += s1 * part[b][3];
        }
      }
    }
#pragma unroll
    for (int i = 0; i < kB; ++i)
#pragma unroll
      for (int r = 0; r < 2; ++r)
#pragma unroll
        for (int j = 0; j < W::kWords; ++j) cur[i][r][j] = nxt[i][r][j];
  }
}

}  // namespace hca
