// The 8-bit block format and the device helpers that its kernels share.
//
// A Block8 of R rows and C columns holds
//   codes   [Cp / 128][R][128] bytes, Cp = C up to a multiple of 128: OCP
//           e4m3, the padding columns zero.  A panel of 128 columns is one
//           piece of memory, because products walk along the columns: the
//           128 bytes that they want of each of 256 rows are 32 KB in a row
//           here, and 256 far apart lines in a row-major matrix, which cost
//           them up to a fifth of their rate
//   scales  [ceil(Cp / 512)][Rp][4] bytes, Rp = R up to a multiple of 256:
//           byte j of dword (q, r) is the e8m0 scale E of row r's block
//           4q + j, worth 2^(E - 127)
// so that value = code * 2^(E - 127).  E is the smallest number >= 1 with
// max|x| <= 448 * 2^(E - 127) over the block's finite values; infinities and
// NaN become the NaN code (e4m3 has no infinity).  Powers of two because
// then scaling rounds nothing, codes differ between blockings only where
// they fall into e4m3's subnormals, and the matrix instruction applies the
// scale by itself.  One dword holds four blocks because a lane of the matrix
// product needs one scale a row and K step: one 4-byte load serves 512 K.
#pragma once
#include <hip/hip_runtime.h>
#include <cstdint>

namespace b8 {

using u32x2 = __attribute__((ext_vector_type(2))) uint32_t;
using u32x4 = __attribute__((ext_vector_type(4))) uint32_t;
using f32x4 = __attribute__((ext_vector_type(4))) float;
using f32x2 = __attribute__((ext_vector_type(2))) float;

// ------------------------------------------------ element types, 8 a lane
struct Bf16 {
  using raw = uint16_t;
  static __device__ __forceinline__ float to_f(raw v) {
    return __builtin_bit_cast(float, (uint32_t)v << 16);
  }
  static __device__ __forceinline__ raw from_f(float f) {
    return __builtin_bit_cast(raw, (__bf16)f);  // v_cvt_pk_bf16_f32, RNE
  }
};
struct Fp16 {
  using raw = uint16_t;
  static __device__ __forceinline__ float to_f(raw v) {
    return (float)__builtin_bit_cast(_Float16, v);
  }
  static __device__ __forceinline__ raw from_f(float f) {
    return __builtin_bit_cast(raw, (_Float16)f);
  }
};
struct Fp32 {
  using raw = float;
  static __device__ __forceinline__ float to_f(raw v) { return v; }
  static __device__ __forceinline__ raw from_f(float f) { return f; }
};

// How a kernel reads and writes plain rows.  kVec: the host has checked that
// the columns, the row strides and the bases allow 16-byte accesses, so a
// group of 8 lies inside the row or outside as a whole.  kOdd: accesses are
// aligned to a value only, and a group that reaches past the row's end goes
// value by value.  kStream: kVec, and the caches do not keep the line.
enum { kOdd, kVec, kStream };

// Loads columns [c, c + 8) of a row; columns from C on read as zero.
struct Eight {
  u32x4 a, b;  // 16-bit types use a only
};

// 16 bytes from p or to p, which is aligned as VEC says
template <int VEC>
__device__ __forceinline__ u32x4 load16(const void* p) {
  if constexpr (VEC == kOdd) {
    u32x4 v;
    __builtin_memcpy(&v, p, 16);
    return v;
  } else if constexpr (VEC == kVec) {
    return *(const u32x4*)p;
  } else {
    return __builtin_nontemporal_load((const u32x4*)p);
  }
}
template <int VEC>
__device__ __forceinline__ void store16(void* p, u32x4 v) {
  if constexpr (VEC == kOdd)
    __builtin_memcpy(p, &v, 16);
  else if constexpr (VEC == kVec)
    *(u32x4*)p = v;
  else
    __builtin_nontemporal_store(v, (u32x4*)p);
}

template <class T, int VEC>
__device__ __forceinline__ Eight load8_raw(const typename T::raw* row, int c,
                                           int C) {
  Eight e{{0, 0, 0, 0}, {0, 0, 0, 0}};
  if (VEC ? c < C : c + 8 <= C) {
    e.a = load16<VEC>(row + c);
    if constexpr (sizeof(typename T::raw) == 4)
      e.b = load16<VEC>(row + c + 4);
  } else if (!VEC && c < C) {
    // no branch a value: each would wait for its load alone
    typename T::raw v[8];
#pragma unroll
    for (int i = 0; i < 8; ++i) v[i] = row[c + i < C ? c + i : C - 1];
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      if constexpr (sizeof(typename T::raw) == 2)
        e.a[i >> 1] |= (c + i < C ? (uint32_t)v[i] : 0u) << (16 * (i & 1));
      else
        (i < 4 ? e.a : e.b)[i & 3] =
            c + i < C ? __builtin_bit_cast(uint32_t, (float)v[i]) : 0u;
    }
  }
  return e;
}

template <class T>
__device__ __forceinline__ void widen(const Eight& e, float (&v)[8]) {
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    if constexpr (sizeof(typename T::raw) == 2) {
      v[i] = T::to_f((uint16_t)(e.a[i >> 1] >> (16 * (i & 1))));
    } else {
      const uint32_t bits = i < 4 ? e.a[i & 3] : e.b[i & 3];
      v[i] = __builtin_bit_cast(float, bits);
    }
  }
}

template <class T, int VEC>
__device__ __forceinline__ void load8(const typename T::raw* row, int c,
                                      int C, float (&v)[8]) {
  widen<T>(load8_raw<T, VEC>(row, c, C), v);
}

template <class T, int VEC>
__device__ __forceinline__ void store8(typename T::raw* row, int c, int C,
                                       const float (&v)[8]) {
  if (VEC ? c < C : c + 8 <= C) {
    if constexpr (sizeof(typename T::raw) == 2) {
      u32x4 d;
#pragma unroll
      for (int i = 0; i < 4; ++i)
        d[i] = (uint32_t)T::from_f(v[2 * i]) |
               (uint32_t)T::from_f(v[2 * i + 1]) << 16;
      store16<VEC>(row + c, d);
    } else {
      u32x4 lo, hi;
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        lo[i] = __builtin_bit_cast(uint32_t, v[i]);
        hi[i] = __builtin_bit_cast(uint32_t, v[i + 4]);
      }
      store16<VEC>(row + c, lo);
      store16<VEC>(row + c + 4, hi);
    }
  } else if constexpr (!VEC) {
#pragma unroll
    for (int i = 0; i < 8; ++i)
      if (c + i < C) row[c + i] = T::from_f(v[i]);
  }
}

// ------------------------------------------------------------- the format
// bits of |x|, 0 for infinities and NaN: what a block's maximum runs over
__device__ __forceinline__ uint32_t finite_bits(float x) {
  const uint32_t a = __builtin_bit_cast(uint32_t, x) & 0x7fffffffu;
  return a < 0x7f800000u ? a : 0u;
}

// E from the bits of the block's maximum: 448 = 1.75 * 2^8
__device__ __forceinline__ uint32_t scale_of(uint32_t top) {
  const int e = (int)(top >> 23) - 8 + ((top & 0x7fffffu) > 0x600000u);
  return (uint32_t)(e < 1 ? 1 : e);
}
__device__ __forceinline__ float scale_value(uint32_t E) {
  return __builtin_bit_cast(float, E << 23);
}
__device__ __forceinline__ float scale_inverse(uint32_t E) {
  return __builtin_bit_cast(float, (254u - E) << 23);
}

// four scaled values to codes; v_cvt_pk_fp8_f32 rounds to nearest even
__device__ __forceinline__ uint32_t encode4(float a, float b, float c,
                                            float d) {
  int r = __builtin_amdgcn_cvt_pk_fp8_f32(a, b, 0, false);
  return (uint32_t)__builtin_amdgcn_cvt_pk_fp8_f32(c, d, r, true);
}
__device__ __forceinline__ u32x2 encode8(const float (&v)[8], float inv) {
  return u32x2{encode4(v[0] * inv, v[1] * inv, v[2] * inv, v[3] * inv),
               encode4(v[4] * inv, v[5] * inv, v[6] * inv, v[7] * inv)};
}
__device__ __forceinline__ void decode8(u32x2 c, float scale, float (&v)[8]) {
#pragma unroll
  for (int i = 0; i < 2; ++i) {
    const f32x2 lo = __builtin_amdgcn_cvt_pk_f32_fp8((int)c[i], false);
    const f32x2 hi = __builtin_amdgcn_cvt_pk_f32_fp8((int)c[i], true);
    v[4 * i] = lo[0] * scale;
    v[4 * i + 1] = lo[1] * scale;
    v[4 * i + 2] = hi[0] * scale;
    v[4 * i + 3] = hi[1] * scale;
  }
}

// the maximum over each row of 16 lanes, in every lane (rotations by DPP)
template <int N>
__device__ __forceinline__ uint32_t ror(uint32_t x) {
  return (uint32_t)__builtin_amdgcn_update_dpp(0, (int)x, 0x120 + N, 0xf,
                                               0xf, true);
}
__device__ __forceinline__ uint32_t max16(uint32_t x) {
  x = max(x, ror<8>(x));
  x = max(x, ror<4>(x));
  x = max(x, ror<2>(x));
  return max(x, ror<1>(x));
}

// the maximum over lanes l, l ^ 16, l ^ 32 and l ^ 48, in all of them
__device__ __forceinline__ uint32_t max_rows(uint32_t x) {
  const auto a = __builtin_amdgcn_permlane16_swap(x, x, false, false);
  x = max(a[0], a[1]);
  const auto b = __builtin_amdgcn_permlane32_swap(x, x, false, false);
  return max(b[0], b[1]);
}

// A wave holds 512 columns of one row, 8 a lane, so 16 lanes hold a block:
// their scales, gathered into the dword (q, row) of the format.
__device__ __forceinline__ uint32_t gather_scales(uint32_t E) {
  return (uint32_t)__builtin_amdgcn_readlane((int)E, 0) |
         (uint32_t)__builtin_amdgcn_readlane((int)E, 16) << 8 |
         (uint32_t)__builtin_amdgcn_readlane((int)E, 32) << 16 |
         (uint32_t)__builtin_amdgcn_readlane((int)E, 48) << 24;
}

__device__ __forceinline__ uint32_t block_top(const float (&v)[8]) {
  uint32_t m = 0;
#pragma unroll
  for (int i = 0; i < 8; ++i) m = max(m, finite_bits(v[i]));
  return max16(m);
}

// where the codes of columns c .. of a row are
__device__ __forceinline__ uint8_t* code_at(uint8_t* codes, long long R,
                                            long long row, int c) {
  return codes + ((c >> 7) * R + row) * 128 + (c & 127);
}
__device__ __forceinline__ const uint8_t* code_at(const uint8_t* codes,
                                                  long long R, long long row,
                                                  int c) {
  return codes + ((c >> 7) * R + row) * 128 + (c & 127);
}

// packs a wave's 512 columns of one row and stores them
__device__ __forceinline__ void pack512(const float (&v)[8], int lane, int c,
                                        int Cp, uint8_t* codes, long long R,
                                        long long row, uint32_t* scale_at) {
  const uint32_t E = scale_of(block_top(v));
  const u32x2 code = encode8(v, scale_inverse(E));
  if (c < Cp) *(u32x2*)code_at(codes, R, row, c) = code;
  const uint32_t four = gather_scales(E);
  if (lane == 0) *scale_at = four;
}

}  // namespace b8
