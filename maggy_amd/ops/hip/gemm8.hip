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

// where a wave's columns go: they lie inside one of the outputs, as both
// start at multiples of 128 rows of w
struct Out {
  void* p;
  int c0, count, f32;
};
__device__ __forceinline__ Out out_of(const GemmArgs& a, int n) {
  Out o{a.out[0], n - a.first[0], a.count[0], a.f32};
#pragma unroll
  for (int k = 1; k < kMaxParts; ++k)
    if (k < a.parts && n >= a.first[k])
      o.p = a.out[k], o.c0 = n - a.first[k], o.count = a.count[k];
  return o;
}

// columns [c, c + 4) of row m
__device__ __forceinline__ void store4(const Out& o, int m, int c, f32x4 v) {
  const long long at = (long long)m * o.count + c;
  if ((o.count & 3) == 0) {
    if (c >= o.count) return;
    if (o.f32)
      *(f32x4*)((float*)o.p + at) = v;
    else
      *(u32x2*)((uint16_t*)o.p + at) =
          u32x2{Bf16::from_f(v[0]) | (uint32_t)Bf16::from_f(v[1]) << 16,
                Bf16::from_f(v[2]) | (uint32_t)Bf16::from_f(v[3]) << 16};
    return;
  }
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    if (c + i >= o.count) break;
    if (o.f32)
      ((float*)o.p)[at + i] = v[i];
    else
      ((uint16_t*)o.p)[at + i] = Bf16::from_f(v[i]);
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
  const int lane = threadIdx.x & 63;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
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

  const Out o = out_of(a, n0 + wn);
#pragma unroll
  for (int i = 0; i < FM; ++i) {
    const int m = m0 + wm + i * 16 + r;
    if (m < a.M) {
#pragma unroll
      for (int j = 0; j < FN; ++j)
        store4(o, m, o.c0 + j * 16 + 4 * g, acc[i * FN + j]);
    }
  }
}

// ------------------------------------------------------------ large tiles
// 256 x 256 by four waves, each 128 x 128 as 4 x 4 of 32x32x64.  A wave
// reads (128 + 128) bytes of LDS a unit of K for 128 x 128 products; eight
// waves of 128 x 64 would read 1.5 times as much, which with the writes is
// all that LDS can do.  One wave a SIMD, so the overlap is inside the wave:
// the fragments of the next half step are read while this half's products
// run, and one barrier a K step serves both uses of a buffer:
//
//   half 0: products of (kt, 0)    reads (kt, 1) from buffer kt
//   barrier: buffer kt is read by all, the loads of kt + 1 have landed
//   half 1: products of (kt, 1)    reads (kt + 1, 0) from buffer kt + 1
//                                  loads kt + 2 into buffer kt
//
// so a load has two half steps (2048 cycles of matrix work) to land.
using f32x16 = __attribute__((ext_vector_type(16))) float;

struct Half {
  i32x8 x[4], w[4];
};

__global__ __launch_bounds__(256, 1) void gemm_large(GemmArgs a, int tiles_m,
                                                     int tiles_n, int group) {
  constexpr int kTile = 512 * 128, kScales = 512 * 4;
  __shared__ __align__(16) char lds[2 * kTile + 2 * kScales];
  const int lane = threadIdx.x & 63;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);

  // tiles in order of a band of `group` tile rows, column by column; each of
  // the 8 XCDs takes a contiguous run of that order, so that the tiles in
  // its L2 at one time are a compact block
  const int tiles = tiles_m * tiles_n;
  int t = blockIdx.x;
  {
    const int q = tiles / 8, r = tiles % 8, xcd = t % 8, idx = t / 8;
    t = (xcd < r ? xcd * (q + 1) : r * (q + 1) + (xcd - r) * q) + idx;
  }
  const int band = t / (group * tiles_n), in_band = t % (group * tiles_n);
  const int rows = min(group, tiles_m - band * group);
  // divisions are done in vector registers; buffer descriptors need scalars
  const int m0 = __builtin_amdgcn_readfirstlane(
      (band * group + in_band % rows) * 256);
  const int n0 = __builtin_amdgcn_readfirstlane(in_band / rows * 256);
  const int wm = (wave >> 1) * 128, wn = (wave & 1) * 128;

  // loads by buffer descriptors: rows past the end read as zero
  const auto rx = __builtin_amdgcn_make_buffer_rsrc(
      (void*)(a.x + (long long)m0 * a.ldx), 0,
      (int)(min(256, a.M - m0) * a.ldx), 0x00020000);
  const auto rw = __builtin_amdgcn_make_buffer_rsrc(
      (void*)(a.w + (long long)n0 * a.ldw), 0,
      (int)(min(256, a.N - n0) * a.ldw), 0x00020000);
  const int lrow = wave * 8 + (lane >> 3);
  const int lchunk = ((lane & 7) ^ (lrow >> 1 & 7)) * 16;
  const int vx = lrow * (int)a.ldx + lchunk;
  const int vw = lrow * (int)a.ldw + lchunk;

  // scales of quad q: piece 0 those of x, 1 those of w
  const int Q = (a.KT + 3) >> 2;
  auto load_scales = [&](int q, int piece) {
    char* sc = lds + 2 * kTile + (q & 1) * kScales + piece * 1024;
    const int at = min(q, Q - 1);
    const uint32_t* src = piece ? a.ws + at * a.wsp + n0
                                : a.xs + at * a.xsp + m0;
    __builtin_amdgcn_global_load_lds(B8_GLOBAL(src + wave * 64 + lane),
                                     B8_LDS(sc + wave * 256), 4, 0, 0);
  };
  // the n-th of a step's 16 loads a wave: 8 rows of x, then of w
  auto load = [&](int step, int n) {
    char* to = lds + (step & 1) * kTile + (n * 32 + wave * 8) * 128;
    const int kt = min(step, a.KT - 1), row = n % 8 * 32;
    if (n < 8)
      __builtin_amdgcn_raw_ptr_buffer_load_lds(
          rx, B8_LDS(to), 16, vx, row * (int)a.ldx + kt * 128, 0, 0);
    else
      __builtin_amdgcn_raw_ptr_buffer_load_lds(
          rw, B8_LDS(to), 16, vw, row * (int)a.ldw + kt * 128, 0, 0);
  };

  // fragment (row = lane % 32, 32 bytes at half * 64 + lane / 32 * 32), in
  // the order that the products want them
  const int frow = lane & 31, fg = lane >> 5;
  auto read = [&](Half& f, int kt, int half, int n) {
    // n / 2: x0 w0 w1 w2 w3 x1 x2 x3
    const int k = n / 2, c = 4 * half + 2 * fg + n % 2;
    const bool of_w = k >= 1 && k < 5;
    const int row = of_w ? 256 + wn + (k - 1) * 32
                         : wm + (k ? k - 4 : 0) * 32;
    const i32x4 v = *(const i32x4*)(lds + (kt & 1) * kTile +
                                    swizzled(row + frow, c));
    i32x8& to = of_w ? f.w[k - 1] : f.x[k ? k - 4 : 0];
#pragma unroll
    for (int i = 0; i < 4; ++i) to[n % 2 * 4 + i] = v[i];
  };
  uint32_t quad_x[4], quad_w[4];  // the scales of four K steps
  auto read_scales = [&](int kt) {
    const uint32_t* sc =
        (const uint32_t*)(lds + 2 * kTile + (kt >> 2 & 1) * kScales);
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      quad_x[i] = sc[wm + i * 32 + frow];
      quad_w[i] = sc[256 + wn + i * 32 + frow];
    }
  };

  f32x16 acc[16];
#pragma unroll
  for (int i = 0; i < 16; ++i)
#pragma unroll
    for (int j = 0; j < 16; ++j) acc[i][j] = 0.f;
  auto product = [&](const Half& f, const int (&sx)[4], const int (&sw)[4],
                     int n) {
    acc[n] = __builtin_amdgcn_mfma_scale_f32_32x32x64_f8f6f4(
        f.w[n % 4], f.x[n / 4], acc[n], 0, 0, 0, sw[n % 4], 0, sx[n / 4]);
  };
  auto meet = [&] {
    asm volatile("s_waitcnt vmcnt(0) lgkmcnt(0)" ::: "memory");
    __builtin_amdgcn_s_barrier();
    asm volatile("" ::: "memory");
  };

  // Past the last step the loads repeat it and the reads find what is
  // there; nothing uses either.  The alternative, a peeled tail, made the
  // compiler copy all accumulators.
  load_scales(0, 0);
  load_scales(0, 1);
#pragma unroll
  for (int n = 0; n < 16; ++n) load(0, n);
#pragma unroll
  for (int n = 0; n < 16; ++n) load(1, n);
  meet();
  Half f0, f1;
#pragma unroll
  for (int n = 0; n < 16; ++n) read(f0, 0, 0, n);
  read_scales(0);
  // the fence after each product keeps the order written here
  for (int kt = 0; kt < a.KT; ++kt) {
    int sx[4], sw[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      sx[i] = (int)(quad_x[i] >> (8 * (kt & 3)));
      sw[i] = (int)(quad_w[i] >> (8 * (kt & 3)));
    }
#pragma unroll
    for (int n = 0; n < 16; ++n) {
      product(f0, sx, sw, n);
      if (n < 8) read(f1, kt, 1, 2 * n), read(f1, kt, 1, 2 * n + 1);
      __builtin_amdgcn_sched_barrier(0);
    }
    meet();
#pragma unroll
    for (int n = 0; n < 16; ++n) {
      product(f1, sx, sw, n);
      load(kt + 2, n);
      if (n < 8) read(f0, kt + 1, 0, 2 * n), read(f0, kt + 1, 0, 2 * n + 1);
      if (n == 8) read_scales(kt + 1);
      // one piece of the next quad a step (each comes twice); its buffer
      // was last read before this step's barrier
      if (n == 15) load_scales((kt + 1 >> 2) + 1, kt + 1 & 1);
      __builtin_amdgcn_sched_barrier(0);
    }
  }
  meet();

  // lane: row m = lane % 32 of its fragment, columns (r / 4) * 8 +
  // lane / 32 * 4 + r % 4
  const Out o = out_of(a, n0 + wn);
  if (o.f32 || (o.count & 7)) {
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const int m = m0 + wm + i * 32 + frow;
      if (m < a.M) {
#pragma unroll
        for (int j = 0; j < 4; ++j)
#pragma unroll
          for (int r = 0; r < 4; ++r) {
            const f32x16& v = acc[i * 4 + j];
            store4(o, m, o.c0 + j * 32 + r * 8 + fg * 4,
                   f32x4{v[4 * r], v[4 * r + 1], v[4 * r + 2],
                         v[4 * r + 3]});
          }
      }
    }
    return;
  }
  // through LDS, 32 KB a wave, so that 16 lanes store 256 bytes of one row:
  // straight from the accumulators a store would touch 16 bytes of 32 rows.
  // 16-byte chunk c of row m lies at c ^ (m % 16)
  char* mine = lds + wave * 32768;
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const int m = i * 32 + frow;
#pragma unroll
    for (int j = 0; j < 4; ++j)
#pragma unroll
      for (int r = 0; r < 4; ++r) {
        const f32x16& v = acc[i * 4 + j];
        *(u32x2*)(mine + m * 256 + ((j * 4 + r ^ m & 15) << 4) + fg * 8) =
            u32x2{Bf16::from_f(v[4 * r]) |
                      (uint32_t)Bf16::from_f(v[4 * r + 1]) << 16,
                  Bf16::from_f(v[4 * r + 2]) |
                      (uint32_t)Bf16::from_f(v[4 * r + 3]) << 16};
      }
  }
  asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
  const int c = lane & 15;
  if (o.c0 + c * 8 >= o.count) return;
  uint16_t* out = (uint16_t*)o.p + o.c0 + c * 8;
#pragma unroll 8
  for (int k = 0; k < 32; ++k) {
    const int row = k * 4 + (lane >> 4), m = m0 + wm + row;
    const u32x4 v = *(const u32x4*)(mine + row * 256 + ((c ^ row & 15) << 4));
    if (m < a.M) *(u32x4*)(out + (long long)m * o.count) = v;
  }
}

// -------------------------------------------------------------- few rows
// Up to 64 rows of x: the time is that of reading w once.  A workgroup takes
// 16 rows of w; its waves share K by quads of four K steps (512 bytes of a
// row, read by every lane's 16-byte loads straight into the operand), and
// their sums meet in LDS, added in the order of the waves.  With FUSED, for
// up to 16 rows of bf16, x is packed on the way: each lane needs 32
// neighbouring values a step, which four lanes share a scale for, so the
// codes are those of pack_rows and a launch is saved.
struct RowsArgs {
  GemmArgs g;
  const uint16_t* x;  // FUSED: bf16, rows of ldx elements, K columns
  long long ldx;
  int K;
};

using u16x2 = __attribute__((ext_vector_type(2))) uint16_t;

__device__ __forceinline__ u16x2 halves(uint32_t v) {
  return __builtin_bit_cast(u16x2, v);
}

// 32 values of one lane to codes; lanes l, l ^ 16, l ^ 32, l ^ 48 hold one
// block
__device__ __forceinline__ i32x8 pack_step(const u32x4 (&v)[4], int* scale) {
  u16x2 m = {0, 0};
#pragma unroll
  for (int i = 0; i < 16; ++i)
    m = __builtin_elementwise_max(m,
                                  halves(v[i / 4][i % 4] & 0x7fff7fffu));
  uint32_t top = max(m[0], m[1]);
  if (__builtin_expect(__any(top >= 0x7f80u), 0)) {
    top = 0;  // some are not finite: the maximum over the others
#pragma unroll
    for (int i = 0; i < 32; ++i) {
      const uint32_t a = v[i / 8][i / 2 % 4] >> (16 * (i & 1)) & 0x7fffu;
      if (a < 0x7f80u) top = max(top, a);
    }
  }
  top = max(top, (uint32_t)__shfl_xor((int)top, 16));
  top = max(top, (uint32_t)__shfl_xor((int)top, 32));
  const uint32_t E = scale_of(top << 16);
  *scale = (int)E;
  i32x8 code;
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    using bf16x2 = __attribute__((ext_vector_type(2))) __bf16;
    using i16x2 = __attribute__((ext_vector_type(2))) short;
    // copies: a bit cast of a vector's element would read its first one
    const uint32_t lo = v[i / 2][i % 2 * 2], hi = v[i / 2][i % 2 * 2 + 1];
    const float by = scale_value(E);
    i16x2 c = {0, 0};
    c = __builtin_amdgcn_cvt_scalef32_pk_fp8_bf16(
        c, __builtin_bit_cast(bf16x2, lo), by, false);
    c = __builtin_amdgcn_cvt_scalef32_pk_fp8_bf16(
        c, __builtin_bit_cast(bf16x2, hi), by, true);
    code[i] = __builtin_bit_cast(int, c);
  }
  return code;
}

template <int FM, int WAVES, bool FUSED>
__global__ __launch_bounds__(WAVES * 64) void gemm_rows(RowsArgs ra) {
  const GemmArgs& a = ra.g;
  __shared__ f32x4 sums[WAVES][FM][64];
  const int lane = threadIdx.x & 63;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int r = lane & 15, g = lane >> 4;
  const int n0 = blockIdx.x * 16;
  const int n = min(n0 + r, a.N - 1);
  const uint8_t* w = a.w + n * a.ldw + g * 32;
  const uint32_t* ws = a.ws + n;

  f32x4 acc[FM];
#pragma unroll
  for (int i = 0; i < FM; ++i) acc[i] = f32x4{0.f, 0.f, 0.f, 0.f};
  const int Q = (a.KT + 3) >> 2;
  for (int q = wave; q < Q; q += WAVES) {
    i32x4 wv[4][2];
    i32x8 xv[4][FM];
    u32x4 raw[FUSED ? 4 : 1][4];
    uint32_t xs[FM];
    const uint32_t wsc = ws[q * a.wsp];
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const int kt = min(4 * q + j, a.KT - 1);
      const i32x4* p = (const i32x4*)(w + (long long)kt * 128);
      wv[j][0] = p[0];
      wv[j][1] = p[1];
    }
    if constexpr (FUSED) {
#pragma unroll
      for (int j = 0; j < 4; ++j)
#pragma unroll
        for (int c = 0; c < 4; ++c) {
          const int k = (4 * q + j) * 128 + g * 32 + c * 8;
          raw[j][c] = r < a.M && k < ra.K
                          ? *(const u32x4*)(ra.x + r * ra.ldx + k)
                          : u32x4{0, 0, 0, 0};
        }
    } else {
#pragma unroll
      for (int i = 0; i < FM; ++i) {
        const int m = min(i * 16 + r, a.M - 1);
        xs[i] = a.xs[q * a.xsp + m];
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          const int kt = min(4 * q + j, a.KT - 1);
          const i32x4* p =
              (const i32x4*)(a.x + m * a.ldx + (long long)kt * 128 + g * 32);
          // past the end w repeats its last block, against zeros; the
          // scales there are not written, see below
          const i32x8 zero = {0, 0, 0, 0, 0, 0, 0, 0};
          xv[j][i] = 4 * q + j < a.KT
                         ? __builtin_shufflevector(p[0], p[1], 0, 1, 2, 3, 4,
                                                   5, 6, 7)
                         : zero;
        }
      }
    }
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const bool inside = 4 * q + j < a.KT;
      const int sw = inside ? (int)(wsc >> (8 * j)) : 1;
      const i32x8 wf =
          __builtin_shufflevector(wv[j][0], wv[j][1], 0, 1, 2, 3, 4, 5, 6, 7);
#pragma unroll
      for (int i = 0; i < FM; ++i) {
        int sx;
        i32x8 xf;
        if constexpr (FUSED) {
          xf = pack_step(raw[j], &sx);
        } else {
          xf = xv[j][i];
          sx = inside ? (int)(xs[i] >> (8 * j)) : 1;
        }
        acc[i] = __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(
            wf, xf, acc[i], 0, 0, 0, sw, 0, sx);
      }
    }
  }
#pragma unroll
  for (int i = 0; i < FM; ++i) sums[wave][i][lane] = acc[i];
  __syncthreads();
  if (wave >= FM) return;
  f32x4 v = sums[0][wave][lane];
#pragma unroll
  for (int k = 1; k < WAVES; ++k) v += sums[k][wave][lane];
  const int m = wave * 16 + r;
  if (m < a.M) {
    const Out o = out_of(a, n0);
    store4(o, m, o.c0 + 4 * g, v);
  }
}

template <int FM, bool FUSED>
static void rows_run(const RowsArgs& ra, hipStream_t st) {
  const int blocks = (ra.g.N + 15) / 16, Q = (ra.g.KT + 3) / 4;
  if (Q <= 4)
    launch(gemm_rows<FM, 4, FUSED>, blocks, 256, st, ra);
  else if (Q <= 8 || FM == 4)  // 16 waves have no registers for four
    launch(gemm_rows<FM, 8, FUSED>, blocks, 512, st, ra);
  else if constexpr (FM < 4)
    launch(gemm_rows<FM, 16, FUSED>, blocks, 1024, st, ra);
}

}  // namespace b8

using namespace b8;

extern "C" void launch_b8_gemm(const GemmArgs* args, hipStream_t st) {
  const GemmArgs a = *args;
  if (a.M <= 64) {
    const RowsArgs ra{a, nullptr, 0, 0};
    if (a.M <= 16)
      rows_run<1, false>(ra, st);
    else if (a.M <= 32)
      rows_run<2, false>(ra, st);
    else
      rows_run<4, false>(ra, st);
    return;
  }
  const int tm = (a.M + 255) / 256, tn = (a.N + 255) / 256;
  if ((long long)tm * tn >= 192) {
    launch(gemm_large, (long long)tm * tn, 256, st, a, tm, tn, 4);
    return;
  }
  const int t128 = (a.N + 127) / 128;
  launch(gemm_tile<128, 128, 2, 2>, (long long)((a.M + 127) / 128) * t128,
         256, st, a, t128);
}

// x in bf16, at most 16 rows of K columns, K and ldx multiples of 8, packed
// on the way; the codes of x in args are not read
extern "C" void launch_b8_gemm_bf16(const GemmArgs* args, const void* x,
                                    long long ldx, int K, hipStream_t st) {
  rows_run<1, true>(RowsArgs{*args, (const uint16_t*)x, ldx, K}, st);
}
