// Matrix product of two matrices in the 8-bit block format.
//
//   Y[m][n] = sum_k X[m][k] W[n][k]
//
// Both operands are packed along k in blocks of 128, which is the K of one
// v_mfma_scale_f32_16x16x128_f8f6f4: one instruction eats one block of 16
// rows of each and multiplies by the two e8m0 scales itself, so the scales
// cost no vector instruction.  A lane of that instruction holds 32 of the
// 128 values of one row and that row's scale; which 32 does not matter as
// long as both operands agree, since a row's scale holds for all 128.
//
// The weights are the instruction's first operand: a lane then ends with
// four neighbouring columns of one row of Y, one 8-byte store.
#include <hip/hip_runtime.h>

#include "block8.h"
#include "block8_api.h"

namespace b8 {

using i32x8 = __attribute__((ext_vector_type(8))) int;
using i32x4 = __attribute__((ext_vector_type(4))) int;

#define B8_GLOBAL(p) ((const __attribute__((address_space(1))) uint32_t*)(p))
#define B8_LDS(p) ((__attribute__((address_space(3))) uint32_t*)(p))

// A row of a K step is 128 bytes, eight 16-byte chunks, laid at chunk ^
// (row / 2 % 8): the 16 rows of a fragment then cover all 64 banks.
__device__ __forceinline__ int swizzled(int row, int chunk) {
  return row * 128 + ((chunk ^ (row >> 1 & 7)) << 4);
}

__device__ __forceinline__ i32x8 fragment(const char* tile, int row, int g) {
  const i32x4 lo = *(const i32x4*)(tile + swizzled(row, 2 * g));
  const i32x4 hi = *(const i32x4*)(tile + swizzled(row, 2 * g + 1));
  return __builtin_shufflevector(lo, hi, 0, 1, 2, 3, 4, 5, 6, 7);
}

// The compiler counts too few wait states between a matrix instruction and
// a vector read of its result where the two are in different basic blocks;
// the loop's accumulators pass through this before the epilogue reads them.
template <int N>
__device__ __forceinline__ void settle(f32x4 (&acc)[N]) {
  asm volatile("s_nop 15\n\ts_nop 15" ::: "memory");
#pragma unroll
  for (int i = 0; i < N; ++i) asm volatile("" : "+v"(acc[i]));
}

// writes columns [n, n + 4) of row m; n counts rows of w
__device__ __forceinline__ void store4(const GemmArgs& a, int m, int n,
                                       f32x4 v) {
  int p = 0;
#pragma unroll
  for (int k = 1; k < kMaxParts; ++k)
    if (k < a.parts && n >= a.first[k]) p = k;
  // selects, not an indexed load from the argument block
  void* out = a.out[0];
  int first = a.first[0], count = a.count[0];
#pragma unroll
  for (int k = 1; k < kMaxParts; ++k)
    if (p == k) out = a.out[k], first = a.first[k], count = a.count[k];
  const int c = n - first;
  const long long at = (long long)m * count + c;
  if (c + 3 < count && (count & 3) == 0) {
    if (a.f32) {
      *(f32x4*)((float*)out + at) = v;
    } else {
      *(u32x2*)((uint16_t*)out + at) =
          u32x2{Bf16::from_f(v[0]) | (uint32_t)Bf16::from_f(v[1]) << 16,
                Bf16::from_f(v[2]) | (uint32_t)Bf16::from_f(v[3]) << 16};
    }
    return;
  }
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    if (c + i >= count) break;
    if (a.f32)
      ((float*)out)[at + i] = v[i];
    else
      ((uint16_t*)out)[at + i] = Bf16::from_f(v[i]);
  }
}

// BM rows of x by BN rows of w; WM x WN waves.  Both tiles of a K step and,
// every fourth step, the scale dwords of all rows go straight to LDS
// (global_load_lds); two buffers, the next step's loads issued before this
// step's products and drained by the barrier after them.
template <int BM, int BN, int WM, int WN>
__global__ __launch_bounds__(WM* WN * 64) void gemm_tile(GemmArgs a,
                                                         int tiles_n) {
  constexpr int kWaves = WM * WN, FM = BM / WM / 16, FN = BN / WN / 16;
  constexpr int kTile = (BM + BN) * 128;
  __shared__ __align__(16) char lds[2 * kTile + 2 * (BM + BN) * 4];
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const int r = lane & 15, g = lane >> 4;
  const int m0 = blockIdx.x / tiles_n * BM, n0 = blockIdx.x % tiles_n * BN;
  const int wm = wave / WN * (BM / WM), wn = wave % WN * (BN / WN);

  // a wave's load covers 8 rows; rows past the end read the last one, their
  // products are never stored
  constexpr int kLoads = (BM + BN) / 8 / kWaves;
  const uint8_t* src[kLoads];
#pragma unroll
  for (int i = 0; i < kLoads; ++i) {
    const int row = (i * kWaves + wave) * 8 + (lane >> 3);
    const int chunk = (lane & 7) ^ (row >> 1 & 7);
    if (row < BM) {
      const int m = min(m0 + row, a.M - 1);
      src[i] = a.x + m * a.ldx + chunk * 16;
    } else {
      const int n = min(n0 + row - BM, a.N - 1);
      src[i] = a.w + n * a.ldw + chunk * 16;
    }
  }
  auto stage = [&](int kt) {
    char* buf = lds + (kt & 1) * kTile;
#pragma unroll
    for (int i = 0; i < kLoads; ++i)
      __builtin_amdgcn_global_load_lds(
          B8_GLOBAL(src[i] + (long long)kt * 128),
          B8_LDS(buf + (i * kWaves + wave) * 1024), 16, 0, 0);
    if ((kt & 3) == 0) {
      char* sc = lds + 2 * kTile + (kt >> 2 & 1) * (BM + BN) * 4;
#pragma unroll
      for (int i = 0; i < (BM + BN) / 64; i += kWaves) {
        if (i + wave < (BM + BN) / 64) {
          const int row = (i + wave) * 64;
          const uint32_t* s =
              row < BM ? a.xs + (kt >> 2) * a.xsp + m0 + row
                       : a.ws + (kt >> 2) * a.wsp + n0 + row - BM;
          __builtin_amdgcn_global_load_lds(B8_GLOBAL(s + lane),
                                           B8_LDS(sc + row * 4), 4, 0, 0);
        }
      }
    }
  };

  f32x4 acc[FM * FN];
#pragma unroll
  for (int i = 0; i < FM * FN; ++i) acc[i] = f32x4{0.f, 0.f, 0.f, 0.f};

  stage(0);
  __syncthreads();
  for (int kt = 0; kt < a.KT; ++kt) {
    if (kt + 1 < a.KT) stage(kt + 1);
    const char* xt = lds + (kt & 1) * kTile;
    const char* wt = xt + BM * 128;
    const uint32_t* sc =
        (const uint32_t*)(lds + 2 * kTile + (kt >> 2 & 1) * (BM + BN) * 4);
    const int shift = 8 * (kt & 3);
    i32x8 wf[FN];
    int wsc[FN];
#pragma unroll
    for (int j = 0; j < FN; ++j) {
      wf[j] = fragment(wt, wn + j * 16 + r, g);
      wsc[j] = (int)(sc[BM + wn + j * 16 + r] >> shift);
    }
#pragma unroll
    for (int i = 0; i < FM; ++i) {
      const i32x8 xf = fragment(xt, wm + i * 16 + r, g);
      const int xsc = (int)(sc[wm + i * 16 + r] >> shift);
#pragma unroll
      for (int j = 0; j < FN; ++j)
        acc[i * FN + j] = __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(
            wf[j], xf, acc[i * FN + j], 0, 0, 0, wsc[j], 0, xsc);
    }
    __syncthreads();
  }
  settle(acc);

#pragma unroll
  for (int i = 0; i < FM; ++i) {
    const int m = m0 + wm + i * 16 + r;
    if (m < a.M) {
#pragma unroll
      for (int j = 0; j < FN; ++j)
        store4(a, m, n0 + wn + j * 16 + 4 * g, acc[i * FN + j]);
    }
  }
}

}  // namespace b8

extern "C" void launch_b8_gemm(const b8::GemmArgs* args, hipStream_t st) {
  const b8::GemmArgs a = *args;
  const int tn = (a.N + 127) / 128;
  const unsigned blocks = (unsigned)((a.M + 127) / 128) * tn;
  b8::launch(b8::gemm_tile<128, 128, 2, 2>, blocks, 256, st, a, tn);
}
