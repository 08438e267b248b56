// Packing to the 8-bit block format and the operators that keep their
// inputs in it: silu(g) * u and RMSNorm.  All are bound by memory: one pass
// over the data, 8 values a lane in one 16-byte load, no value read twice.
// A large copy reaches 4.9 TB/s on the same card.
//
// A block's code is x 2^-t rounded to nearest even, t the smallest exponent
// with max|x| <= 448 2^t: the scale is a power of two, so that scaling
// rounds nothing and the matrix unit can undo it.
#include <hip/hip_runtime.h>

#include "block8.h"
#include "block8_api.h"

namespace b8 {

constexpr int kThreads = 256;

// one wave's unit of work: 512 columns (one scale dword) of one row
struct Unit {
  long long row;
  int q;
};
__device__ __forceinline__ Unit unit_of(long long u, int Q) {
  const long long row = u / Q;
  return {row, (int)(u - row * Q)};
}

// ------------------------------------------------------------ pack, unpack
// A wave packs 512 columns of a row, four blocks of 16 lanes, so the maximum
// takes four DPP steps and the four scales leave as one dword.  24576 x 4096
// in bf16: packed in 53 us (5.7 TB/s), read back in 46 (6.5 TB/s, the codes
// partly from the last cache).
template <class T, int VEC>
__global__ __launch_bounds__(kThreads) void pack_rows(
    const typename T::raw* __restrict__ x, long long ldx, long long R, int C,
    uint8_t* __restrict__ codes, int Cp, uint32_t* __restrict__ scales,
    long long Rp, int Q) {
  const int lane = threadIdx.x & 63;
  const long long waves = (long long)gridDim.x * (kThreads / 64);
  const long long units = R * Q;
  for (long long u = (long long)blockIdx.x * (kThreads / 64) +
                     (threadIdx.x >> 6);
       u < units; u += waves) {
    const Unit at = unit_of(u, Q);
    const int c = at.q * 512 + lane * 8;
    float v[8];
    load8<T, VEC>(x + at.row * ldx, c, C, v);
    pack512(v, lane, c, Cp, codes, R, at.row,
            scales + at.q * Rp + at.row);
  }
}

template <class T, int VEC>
__global__ __launch_bounds__(kThreads) void unpack_rows(
    const uint8_t* __restrict__ codes, int Cp,
    const uint32_t* __restrict__ scales, long long Rp, int Q, long long R,
    int C, typename T::raw* __restrict__ out, float most) {
  const int lane = threadIdx.x & 63;
  const long long waves = (long long)gridDim.x * (kThreads / 64);
  const long long units = R * Q;
  for (long long u = (long long)blockIdx.x * (kThreads / 64) +
                     (threadIdx.x >> 6);
       u < units; u += waves) {
    const Unit at = unit_of(u, Q);
    const int c = at.q * 512 + lane * 8;
    if (c >= Cp) continue;
    const uint32_t E =
        scales[at.q * Rp + at.row] >> (8 * (lane >> 4)) & 255u;
    float v[8];
    decode8(*(const u32x2*)code_at(codes, R, at.row, c), scale_value(E), v);
    // a value next to the type's largest may have been rounded up past it
#pragma unroll
    for (int i = 0; i < 8; ++i)
      v[i] = v[i] > most ? most : v[i] < -most ? -most : v[i];
    store8<T, VEC>(out + at.row * C, c, C, v);
  }
}

// --------------------------------------------- 128 x 128 tiles, transposed
// Reads a 128 x 128 tile once and writes its codes by rows (blocks along the
// columns), by columns (the transpose, blocks along the rows) or both.  With
// ONE_SCALE the whole tile shares one scale, so that both orders stand for
// the same values.  FROM8 reads a packed matrix instead of plain numbers.
//
// 512 threads: thread (cg, rg) = (t % 16, t / 16) holds 8 columns of 4
// neighbouring rows, so that four rows of one column make one dword of the
// transposed codes, and 16 lanes (one DPP row) hold a whole row of the tile.
// Every line of the outputs is written whole.  What a pass packs is one
// launch: 24576 x 4096 with 14336 x 4096 weights by rows 84 us (5.7 TB/s);
// for its gradients, 24576 x 14336 both ways, the weights' columns and the
// kept input's, 332 us (5.4 TB/s); 357 before the plain rows passed by the
// caches, 377 with a load at a time a thread.
struct TileSpace {
  // the transposed codes: dword d of row c lies at d ^ (c / 8 % 8) * 4, so
  // that 16-byte reads take 8 lanes a row without a bank conflict, and the
  // columns that a wave writes at once, 8 apart, at most two by two
  uint32_t turned[128 * 32];
  static __device__ __forceinline__ int at(int c, int d) {
    return c * 32 + (d ^ (c >> 3 & 7) << 2);
  }
  uint32_t tops[8][128];
  uint32_t scales[128];
};

template <class T, bool FROM8, bool ONE_SCALE, bool ROWS, bool COLS>
__device__ __forceinline__ void pack_tile(const TileJob& a, TileSpace& space,
                                          int tile) {
  uint32_t(&tops)[8][128] = space.tops;
  uint32_t* turned = space.turned;
  const int t = threadIdx.x, cg = t & 15, rg = t >> 4, wave = t >> 6;
  const int tiles_c = (a.C + 127) / 128;
  const long long tr = tile / tiles_c;
  const int tc = tile % tiles_c;
  const long long r0 = tr * 128 + rg * 4;
  const int c0 = tc * 128 + cg * 8;

  // all four rows' loads under way at once; rows past the end repeat the
  // last one and count as zeros
  float v[4][8];
  if constexpr (FROM8) {
    u32x2 code[4];
    uint32_t E[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const long long r = min(r0 + i, a.R - 1ll);
      E[i] = ((const uint8_t*)a.xs)[4 * ((tc >> 2) * a.xsp + r) + (tc & 3)];
      code[i] = *(const u32x2*)code_at((const uint8_t*)a.x, a.ldx, r, c0);
    }
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      if (r0 + i >= a.R) code[i] = u32x2{0, 0};
      decode8(code[i], scale_value(E[i]), v[i]);
    }
  } else {
    Eight e[4];
    const auto* x = (const typename T::raw*)a.x;
    if (a.vec == kStream) {
#pragma unroll
      for (int i = 0; i < 4; ++i)
        e[i] = load8_raw<T, kStream>(x + min(r0 + i, a.R - 1ll) * a.ldx, c0,
                                     a.C);
    } else if (a.vec == kVec) {
#pragma unroll
      for (int i = 0; i < 4; ++i)
        e[i] = load8_raw<T, kVec>(x + min(r0 + i, a.R - 1ll) * a.ldx, c0,
                                  a.C);
    } else {
#pragma unroll
      for (int i = 0; i < 4; ++i)
        e[i] = load8_raw<T, kOdd>(x + min(r0 + i, a.R - 1ll) * a.ldx, c0,
                                   a.C);
    }
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      if (r0 + i >= a.R) e[i] = Eight{{0, 0, 0, 0}, {0, 0, 0, 0}};
      widen<T>(e[i], v[i]);
    }
  }

  uint32_t tile_E = 0;
  if constexpr (ONE_SCALE) {
    uint32_t m = 0;
#pragma unroll
    for (int i = 0; i < 4; ++i)
#pragma unroll
      for (int j = 0; j < 8; ++j) m = max(m, finite_bits(v[i][j]));
    m = max_rows(max16(m));
    if ((t & 63) == 0) tops[wave][0] = m;
    __syncthreads();
#pragma unroll
    for (int w = 0; w < 8; ++w) m = max(m, tops[w][0]);
    tile_E = scale_of(m);
  }

  if constexpr (ROWS) {
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const long long r = r0 + i;
      const uint32_t E = ONE_SCALE ? tile_E : scale_of(block_top(v[i]));
      const u32x2 code = encode8(v[i], scale_inverse(E));
      if (r < a.R) {
        const long long b = a.row_c0 / 128 + tc;
        *(u32x2*)(a.row_codes + (b * a.row_n + a.row_r0 + r) * 128 + cg * 8) =
            code;
        if (cg == 0)
          a.row_scales[4 * ((b >> 2) * a.row_sp + a.row_r0 + r) + (b & 3)] =
              (uint8_t)E;
      }
    }
  }

  if constexpr (COLS) {
    const long long b = a.col_c0 / 128 + tr;
    uint32_t E[8];
    if constexpr (ONE_SCALE) {
#pragma unroll
      for (int j = 0; j < 8; ++j) E[j] = tile_E;
    } else {
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        uint32_t m = 0;
#pragma unroll
        for (int i = 0; i < 4; ++i) m = max(m, finite_bits(v[i][j]));
        m = max_rows(m);
        if ((t & 63) < 16) tops[wave][cg * 8 + j] = m;
      }
      __syncthreads();
    }
    if (t < 128) {
      uint32_t mine = tile_E;
      if constexpr (!ONE_SCALE) {
        uint32_t top = 0;
#pragma unroll
        for (int w = 0; w < 8; ++w) top = max(top, tops[w][t]);
        space.scales[t] = mine = scale_of(top);
      }
      a.col_scales[4 * ((b >> 2) * a.col_sp + a.col_r0 + tc * 128 + t) +
                   (b & 3)] = (uint8_t)mine;
    }
    if constexpr (!ONE_SCALE) {
      __syncthreads();
#pragma unroll
      for (int j = 0; j < 8; ++j) E[j] = space.scales[cg * 8 + j];
    }
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      const float s = scale_inverse(E[j]);
      turned[TileSpace::at(cg * 8 + j, rg)] =
          encode4(v[0][j] * s, v[1][j] * s, v[2][j] * s, v[3][j] * s);
    }
    __syncthreads();
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      const int c = h * 64 + (t >> 3), k = (t & 7) * 4;
      *(u32x4*)(a.col_codes +
                (b * a.col_n + a.col_r0 + tc * 128 + c) * 128 + k * 4) =
          *(const u32x4*)(turned + TileSpace::at(c, k));
    }
  }
}

__global__ __launch_bounds__(512) void pack_tiles(TileJobs jobs) {
  __shared__ __align__(16) TileSpace space;
  int j = 0;
  while (j + 1 < jobs.count && (int)blockIdx.x >= jobs.job[j + 1].first_block)
    ++j;
  const TileJob& a = jobs.job[j];
  const int tile = (int)blockIdx.x - a.first_block;
  switch (a.kind) {
    case kTileBoth:
      return pack_tile<Bf16, false, false, true, true>(a, space, tile);
    case kTileCols:
      return pack_tile<Bf16, false, false, false, true>(a, space, tile);
    case kTileRows:
      return pack_tile<Bf16, false, false, true, false>(a, space, tile);
    case kTileOneRows:
      if (a.dtype)
        return pack_tile<Fp32, false, true, true, false>(a, space, tile);
      return pack_tile<Bf16, false, true, true, false>(a, space, tile);
    case kTileOneCols:
      if (a.dtype)
        return pack_tile<Fp32, false, true, false, true>(a, space, tile);
      return pack_tile<Bf16, false, true, false, true>(a, space, tile);
    case kTileFrom8:
      return pack_tile<Fp32, true, false, false, true>(a, space, tile);
  }
}

// ------------------------------------------------------------ silu(g) * u
// h = g s u with s = 1 / (1 + exp(-g)); the backward pass uses the 8-bit g~
// and u~:  dg = dh u~ s (1 + g~ (1 - s)),  du = dh g~ s.
// 24576 x 14336 in bf16: 560 us forward (5.0 TB/s), 622 backward (4.5 TB/s),
// which still writes back what the forward pass left in the last cache.
template <class T>
__device__ __forceinline__ float sigmoid(float g) {
  if constexpr (sizeof(typename T::raw) == 4)
    return 1.f / (1.f + expf(-g));
  else
    // The product of g and log2(e) is rounded before the exponential: off by
    // less than (1.2 |g| + 6) 2^-24 of itself, 2^-17 at the most, where a half
    // step of the 16-bit types is 2^-9 and 2^-12.  Below g = -88.7 the
    // exponential is infinite and the result 0, as in the branch above.
    return __builtin_amdgcn_rcpf(1.f + __expf(-g));
}

template <class T, int VEC>
__global__ __launch_bounds__(kThreads) void swiglu_fwd(
    const typename T::raw* __restrict__ g, long long ldg,
    const typename T::raw* __restrict__ u, long long ldu, long long R, int C,
    typename T::raw* __restrict__ h, uint8_t* __restrict__ gc,
    uint8_t* __restrict__ uc, int Cp, uint32_t* __restrict__ gs,
    uint32_t* __restrict__ us, long long Rp, int Q) {
  const int lane = threadIdx.x & 63;
  const long long waves = (long long)gridDim.x * (kThreads / 64);
  const long long units = R * Q;
  for (long long n = (long long)blockIdx.x * (kThreads / 64) +
                     (threadIdx.x >> 6);
       n < units; n += waves) {
    const Unit at = unit_of(n, Q);
    const int c = at.q * 512 + lane * 8;
    float a[8], b[8], o[8];
    load8<T, VEC>(g + at.row * ldg, c, C, a);
    load8<T, VEC>(u + at.row * ldu, c, C, b);
#pragma unroll
    for (int i = 0; i < 8; ++i) o[i] = a[i] * sigmoid<T>(a[i]) * b[i];
    store8<T, VEC>(h + at.row * C, c, C, o);
    if (gc) {
      const long long s = at.q * Rp + at.row;
      pack512(a, lane, c, Cp, gc, R, at.row, gs + s);
      pack512(b, lane, c, Cp, uc, R, at.row, us + s);
    }
  }
}

template <class T, int VEC>
__global__ __launch_bounds__(kThreads) void swiglu_bwd(
    const typename T::raw* __restrict__ dh, long long ldh,
    const uint8_t* __restrict__ gc, const uint8_t* __restrict__ uc, int Cp,
    const uint32_t* __restrict__ gs, const uint32_t* __restrict__ us,
    long long Rp, int Q, long long R, int C,
    typename T::raw* __restrict__ dg, typename T::raw* __restrict__ du) {
  const int lane = threadIdx.x & 63;
  const long long waves = (long long)gridDim.x * (kThreads / 64);
  const long long units = R * Q;
  for (long long n = (long long)blockIdx.x * (kThreads / 64) +
                     (threadIdx.x >> 6);
       n < units; n += waves) {
    const Unit at = unit_of(n, Q);
    const int c = at.q * 512 + lane * 8;
    if (c >= Cp) continue;
    const long long s = at.q * Rp + at.row;
    const int shift = 8 * (lane >> 4);
    float a[8], b[8], d[8];
    load8<T, VEC>(dh + at.row * ldh, c, C, d);
    decode8(*(const u32x2*)code_at(gc, R, at.row, c),
            scale_value(gs[s] >> shift & 255u), a);
    decode8(*(const u32x2*)code_at(uc, R, at.row, c),
            scale_value(us[s] >> shift & 255u), b);
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      const float sg = sigmoid<T>(a[i]);
      b[i] = d[i] * b[i] * sg * (1.f + a[i] * (1.f - sg));
      a[i] = d[i] * a[i] * sg;
    }
    store8<T, VEC>(dg + at.row * C, c, C, b);
    store8<T, VEC>(du + at.row * C, c, C, a);
  }
}

// ---------------------------------------------------------------- RMSNorm
// y = x inv w, inv = (mean x^2 + eps)^(-1/2), kept in fp32 from the exact x;
// the backward pass uses n = x~ inv of the 8-bit x~:
//   dx = inv (dy w - n mean(dy w n)),  dw = sum over rows of dy n.
// A row belongs to WPR waves (1 up to 2048 columns, else 4), each lane
// keeping its 8 * NI values in registers between the sum and the use: four
// waves share a row where one would need more registers than let others hide
// its loads.  24576 x 4096 in bf16: 96 us forward (5.2 TB/s), 100 backward
// (5.0 TB/s) and 6 for the fold; both passes 282 before the backward loaded
// the next row ahead.
__device__ __forceinline__ float wave_sum(float x) {
#pragma unroll
  for (int m = 32; m; m >>= 1) x += __shfl_xor(x, m);
  return x;
}

template <int WPR>
__device__ __forceinline__ float row_sum(float x, float (*part)[4],
                                         int parity) {
  x = wave_sum(x);
  if constexpr (WPR == 1) return x;
  // two buffers in turn: one barrier a row is enough
  if ((threadIdx.x & 63) == 0) part[parity][threadIdx.x >> 6] = x;
  __syncthreads();
  return part[parity][0] + part[parity][1] + part[parity][2] +
         part[parity][3];
}

template <class T, int VEC, int WPR, int NI>
__global__ __launch_bounds__(kThreads) void rms_fwd(
    const typename T::raw* __restrict__ x, long long ldx,
    const float* __restrict__ w, long long R, int C, float eps,
    typename T::raw* __restrict__ y, float* __restrict__ inv_rms,
    uint8_t* __restrict__ codes, int Cp, uint32_t* __restrict__ scales,
    long long Rp) {
  __shared__ float part[2][4];
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const int q0 = WPR == 1 ? 0 : wave;
  const long long step = (long long)gridDim.x * (4 / WPR);
  int parity = 0;
  for (long long r = (long long)blockIdx.x * (4 / WPR) +
                     (WPR == 1 ? wave : 0);
       r < R; r += step, parity ^= 1) {
    float v[NI][8], sum = 0.f;
#pragma unroll
    for (int i = 0; i < NI; ++i)
      load8<T, VEC>(x + r * ldx, (q0 + i * WPR) * 512 + lane * 8, C, v[i]);
#pragma unroll
    for (int i = 0; i < NI; ++i)
#pragma unroll
      for (int j = 0; j < 8; ++j) sum += v[i][j] * v[i][j];
    sum = row_sum<WPR>(sum, part, parity);
    const float inv = 1.f / sqrtf(sum / C + eps);
    if (inv_rms && lane == 0 && q0 == 0) inv_rms[r] = inv;
#pragma unroll
    for (int i = 0; i < NI; ++i) {
      const int q = q0 + i * WPR, c = q * 512 + lane * 8;
      if (q * 512 >= Cp) continue;  // the same for the whole wave
      if (codes)
        pack512(v[i], lane, c, Cp, codes, R, r, scales + q * Rp + r);
      float g[8];
      load8<Fp32, VEC ? kVec : kOdd>(w, c, C, g);
#pragma unroll
      for (int j = 0; j < 8; ++j) g[j] *= v[i][j] * inv;
      store8<T, VEC>(y + r * C, c, C, g);
    }
  }
}

// dw: every wave adds up its rows in registers and writes one row of
// partials; the fold sums them in a fixed order, so results repeat.
template <class T, int VEC, int WPR, int NI>
__global__ __launch_bounds__(kThreads, NI <= 2 ? 4 : NI <= 4 ? 2 : 1) void
rms_bwd(
    const typename T::raw* __restrict__ dy, long long ldy,
    const uint8_t* __restrict__ codes, int Cp,
    const uint32_t* __restrict__ scales, long long Rp,
    const float* __restrict__ w, const float* __restrict__ inv_rms,
    long long R, int C, typename T::raw* __restrict__ dx,
    float* __restrict__ partials) {
  __shared__ float part[2][4];
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const int q0 = WPR == 1 ? 0 : wave;
  const long long first =
      (long long)blockIdx.x * (4 / WPR) + (WPR == 1 ? wave : 0);
  const long long step = (long long)gridDim.x * (4 / WPR);
  float g[NI][8], dw[NI][8];
#pragma unroll
  for (int i = 0; i < NI; ++i) {
    load8<Fp32, VEC ? kVec : kOdd>(w, (q0 + i * WPR) * 512 + lane * 8, C, g[i]);
#pragma unroll
    for (int j = 0; j < 8; ++j) dw[i][j] = 0.f;
  }
  // the next row's loads are under way while this row is summed; 8 * 8
  // values a lane leave no registers for that
  constexpr bool kAhead = NI <= 4;
  struct Row {
    Eight d[NI];
    u32x2 code[NI];
    uint32_t E[NI];
    float inv;
  };
  auto load_row = [&](long long r, Row& row) {
    row.inv = inv_rms[r];
#pragma unroll
    for (int i = 0; i < NI; ++i) {
      const int q = q0 + i * WPR, c = q * 512 + lane * 8;
      row.d[i] = load8_raw<T, VEC>(dy + r * ldy, c, C);
      row.code[i] = u32x2{0, 0};
      row.E[i] = 1;
      if (c < Cp) {
        row.code[i] = *(const u32x2*)code_at(codes, R, r, c);
        row.E[i] = scales[q * Rp + r] >> (8 * (lane >> 4)) & 255u;
      }
    }
  };
  Row ahead;
  if (kAhead && first < R) load_row(first, ahead);
  int parity = 0;
  for (long long r = first; r < R; r += step, parity ^= 1) {
    float n[NI][8], d[NI][8], sum = 0.f;
    if (!kAhead) load_row(r, ahead);
    const float inv = ahead.inv;
#pragma unroll
    for (int i = 0; i < NI; ++i) {
      widen<T>(ahead.d[i], d[i]);
      decode8(ahead.code[i], scale_value(ahead.E[i]), n[i]);
    }
    if (kAhead) load_row(r + step < R ? r + step : r, ahead);
#pragma unroll
    for (int i = 0; i < NI; ++i)
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        n[i][j] *= inv;
        dw[i][j] += d[i][j] * n[i][j];
        d[i][j] *= g[i][j];
        sum += d[i][j] * n[i][j];
      }
    const float mean = row_sum<WPR>(sum, part, parity) / C;
    if (dx) {
#pragma unroll
      for (int i = 0; i < NI; ++i) {
#pragma unroll
        for (int j = 0; j < 8; ++j) d[i][j] = inv * (d[i][j] - n[i][j] * mean);
        store8<T, VEC>(dx + r * C, (q0 + i * WPR) * 512 + lane * 8, C, d[i]);
      }
    }
  }
  if (!partials) return;
  const long long row = WPR == 1 ? first : blockIdx.x;
#pragma unroll
  for (int i = 0; i < NI; ++i) {
    const int c = (q0 + i * WPR) * 512 + lane * 8;
    store8<Fp32, VEC ? kVec : kOdd>(partials + row * C, c, C, dw[i]);
  }
}

// out[c] = sum over rows of partials[row][c]: 64 columns a workgroup, 16
// waves each adding every 16th row, joined in order
__global__ __launch_bounds__(1024) void fold_rows(
    const float* __restrict__ partials, int P, int C,
    float* __restrict__ out) {
  __shared__ float part[16][64];
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const int c = blockIdx.x * 64 + lane;
  float s = 0.f;
  if (c < C) {
#pragma unroll 8
    for (int p = wave; p < P; p += 16) s += partials[(long long)p * C + c];
  }
  part[wave][lane] = s;
  __syncthreads();
  if (wave == 0 && c < C) {
    s = part[0][lane];
#pragma unroll
    for (int k = 1; k < 16; ++k) s += part[k][lane];
    out[c] = s;
  }
}

// ---------------------------------------------------------------- launches
static inline int unit_blocks(long long R, int Q) {
  const long long want = (R * Q + 3) / 4;
  return (int)(want < 8192 ? want : 8192);
}

// dtype: 0 bf16, 1 fp16, 2 fp32; vec: kOdd, kVec or kStream
#define B8_VEC(vec, ...)                                              \
  if (vec == kStream) { constexpr int V = kStream; return __VA_ARGS__; } \
  if (vec == kVec) { constexpr int V = kVec; return __VA_ARGS__; }    \
  constexpr int V = kOdd;                                             \
  return __VA_ARGS__
#define B8_TYPED(dtype, vec, ...)                                     \
  [&]() -> hipError_t {                                               \
    if (dtype == 0) { using T = Bf16; B8_VEC(vec, __VA_ARGS__); }     \
    if (dtype == 1) { using T = Fp16; B8_VEC(vec, __VA_ARGS__); }     \
    using T = Fp32;                                                   \
    B8_VEC(vec, __VA_ARGS__);                                         \
  }()

// for results of n values
static inline int stores_of(int vec, int dtype, long long n) {
  if (!vec) return kOdd;
  return n * (dtype == 2 ? 4 : 2) >= kStreamResult ? kStream : kVec;
}

template <class T, int V, int WPR, int NI>
static hipError_t rms_fwd_run(int blocks, hipStream_t st, const void* x,
                        long long ldx, const float* w, long long R, int C,
                        float eps, void* y, float* inv, uint8_t* codes,
                        int Cp, uint32_t* scales, long long Rp) {
  return launch(rms_fwd<T, V, WPR, NI>, blocks, kThreads, 0, st,
      (const typename T::raw*)x, ldx, w, R, C, eps, (typename T::raw*)y, inv,
      codes, Cp, scales, Rp);
}

template <class T, int V, int WPR, int NI>
static hipError_t rms_bwd_run(int blocks, hipStream_t st, const void* dy,
                        long long ldy, const uint8_t* codes, int Cp,
                        const uint32_t* scales, long long Rp, const float* w,
                        const float* inv, long long R, int C, void* dx,
                        float* partials) {
  return launch(rms_bwd<T, V, WPR, NI>, blocks, kThreads, 0, st,
      (const typename T::raw*)dy, ldy, codes, Cp, scales, Rp, w, inv, R, C,
      (typename T::raw*)dx, partials);
}

// rows of up to 16384 columns: the caller refuses longer ones
#define B8_ROWS(RUN, C, ...)                                   \
  (C <= 512    ? RUN<T, V, 1, 1>(__VA_ARGS__)                  \
   : C <= 1024 ? RUN<T, V, 1, 2>(__VA_ARGS__)                  \
   : C <= 2048 ? RUN<T, V, 1, 4>(__VA_ARGS__)                  \
   : C <= 4096 ? RUN<T, V, 4, 2>(__VA_ARGS__)                  \
   : C <= 8192 ? RUN<T, V, 4, 4>(__VA_ARGS__)                  \
               : RUN<T, V, 4, 8>(__VA_ARGS__))

}  // namespace b8

using namespace b8;

extern "C" hipError_t launch_b8_pack(int dtype, int vec, const void* x,
                               long long ldx, long long R, int C,
                               uint8_t* codes, int Cp, uint32_t* scales,
                               long long Rp, hipStream_t st) {
  const int Q = (Cp + 511) / 512;
  return B8_TYPED(dtype, vec,
           (launch(pack_rows<T, V ? kVec : kOdd>, unit_blocks(R, Q), kThreads,
               0, st, (const T::raw*)x, ldx, R, C, codes, Cp, scales, Rp, Q)));
}

extern "C" hipError_t launch_b8_unpack(int dtype, int vec, const uint8_t* codes,
                                 int Cp, const uint32_t* scales,
                                 long long Rp, long long R, int C, void* out,
                                 hipStream_t st) {
  const int Q = (Cp + 511) / 512;
  const float most =
      dtype == 0 ? 0x1.fep127f : dtype == 1 ? 65504.f : 0x1.fffffep127f;
  vec = stores_of(vec, dtype, R * C);
  return B8_TYPED(dtype, vec,
           (launch(unpack_rows<T, V>, unit_blocks(R, Q), kThreads, 0, st,
               codes, Cp, scales, Rp, Q, R, C, (T::raw*)out, most)));
}

extern "C" long long b8_tile_blocks(TileJobs* jobs) {
  long long blocks = 0;
  for (int j = 0; j < jobs->count; ++j) {
    TileJob& a = jobs->job[j];
    a.first_block = (int)blocks;
    if (a.vec && (a.dtype ? 4ll : 2ll) * a.R * a.C >= kStreamOnce)
      a.vec = kStream;
    blocks += (a.R + 127ll) / 128 * ((a.C + 127ll) / 128);
    // a launch has fewer than 2^32 threads
    if (blocks >= 1ll << 23) return -1;
  }
  return blocks;
}
extern "C" hipError_t launch_b8_tiles(const TileJobs* jobs, long long blocks,
                                      hipStream_t st) {
  return launch(pack_tiles, blocks, 512, 0, st, *jobs);
}

extern "C" hipError_t launch_b8_swiglu_fwd(int dtype, int vec, const void* g,
                                     long long ldg, const void* u,
                                     long long ldu, long long R, int C,
                                     void* h, uint8_t* gc, uint8_t* uc,
                                     int Cp, uint32_t* gs, uint32_t* us,
                                     long long Rp, hipStream_t st) {
  vec = stores_of(vec, dtype, R * C);
  const int Q = (Cp + 511) / 512;
  return B8_TYPED(dtype, vec,
           (launch(swiglu_fwd<T, V>, unit_blocks(R, Q), kThreads, 0, st,
               (const T::raw*)g, ldg, (const T::raw*)u, ldu, R, C,
               (T::raw*)h, gc, uc, Cp, gs, us, Rp, Q)));
}

extern "C" hipError_t launch_b8_swiglu_bwd(int dtype, int vec, const void* dh,
                                     long long ldh, const uint8_t* gc,
                                     const uint8_t* uc, int Cp,
                                     const uint32_t* gs, const uint32_t* us,
                                     long long Rp, long long R, int C,
                                     void* dg, void* du, hipStream_t st) {
  vec = stores_of(vec, dtype, 2 * R * C);
  const int Q = (Cp + 511) / 512;
  return B8_TYPED(dtype, vec,
           (launch(swiglu_bwd<T, V>, unit_blocks(R, Q), kThreads, 0, st,
               (const T::raw*)dh, ldh, gc, uc, Cp, gs, us, Rp, Q, R, C,
               (T::raw*)dg, (T::raw*)du)));
}

extern "C" hipError_t launch_b8_rms_fwd(int dtype, int vec, const void* x,
                                  long long ldx, const float* w, long long R,
                                  int C, float eps, void* y, float* inv,
                                  uint8_t* codes, int Cp, uint32_t* scales,
                                  long long Rp, hipStream_t st) {
  vec = stores_of(vec, dtype, R * C);
  const long long groups = C <= 2048 ? (R + 3) / 4 : R;
  const int blocks = (int)(groups < 8192 ? groups : 8192);
  return B8_TYPED(dtype, vec,
           B8_ROWS(rms_fwd_run, C, blocks, st, x, ldx, w, R, C, eps, y, inv,
                   codes, Cp, scales, Rp));
}

// the workgroups of the backward pass, and the rows of partials they write
extern "C" int b8_rms_bwd_blocks(long long R, int C) {
  const long long groups = C <= 2048 ? (R + 3) / 4 : R;
  // as many as the registers let run at once: 4 a CU where a lane holds up
  // to 2 * 8 values, else 2
  const int most = C <= 1024 || (C > 2048 && C <= 4096) ? 1024 : 512;
  return (int)(groups < most ? groups : most);
}
extern "C" int b8_rms_bwd_partials(long long R, int C) {
  return b8_rms_bwd_blocks(R, C) * (C <= 2048 ? 4 : 1);
}

extern "C" hipError_t launch_b8_rms_bwd(int dtype, int vec, const void* dy,
                                  long long ldy, const uint8_t* codes,
                                  int Cp, const uint32_t* scales,
                                  long long Rp, const float* w,
                                  const float* inv, long long R, int C,
                                  void* dx, float* partials, float* dw,
                                  hipStream_t st) {
  vec = stores_of(vec, dtype, R * C);
  const int blocks = b8_rms_bwd_blocks(R, C);
  const hipError_t e = B8_TYPED(dtype, vec,
           B8_ROWS(rms_bwd_run, C, blocks, st, dy, ldy, codes, Cp, scales,
                   Rp, w, inv, R, C, dx, partials));
  if (e != hipSuccess || !partials) return e;
  return launch(fold_rows, (C + 63) / 64, 1024, 0, st, partials,
                b8_rms_bwd_partials(R, C), C, dw);
}
