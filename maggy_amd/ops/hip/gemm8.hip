// Matrix product of two matrices in the 8-bit block format.
//
//   Y[m][n] = sum_k X[m][k] W[n][k]
//           = sum over blocks b of 2^(sx[m][b] + sw[n][b])
//             * sum over k in b of x~[m][k] w~[n][k]
//
// Both operands are packed along k in blocks of 128 with one power-of-two
// scale each.  v_mfma_scale_f32_16x16x128_f8f6f4 eats one block of 16 rows
// of each operand, _32x32x64_ half a block of 32, and both multiply by the
// two e8m0 scales themselves, so the scales cost no vector instruction and
// no rounding.  A lane holds 32 values of one row and that row's scale;
// which 32 of the block does not matter as long as both operands agree,
// since a row's scale holds for all 128.
//
// The accumulators are fp32, but the unit aligns before it adds: of each 8
// products that a lane's neighbouring values make, bits below 2^-13 of the
// largest one are cut (measured alike for all shapes of the instruction;
// 1.4e-5 of the result's rms on normal numbers).  That is about a hundredth
// of a rounding to bfloat16, the results' type; fp32 comes out for the
// gradients of fp32 weights only, and is no more exact than that.
//
// The weights are the instruction's first operand: a lane then ends with
// four neighbouring columns of one row of Y, one 8-byte store.
#include <hip/hip_runtime.h>
#include <type_traits>

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

// where a wave's results go: its rows and columns lie inside one of the
// outputs, as both start at multiples of 128 rows of w, or of x
struct Out {
  char* p;  // of row 0, column 0
  int c0, count, rows, f32;
};
__device__ __forceinline__ Out out_of(const GemmArgs& a, int m, int n) {
  const int at = a.by_rows ? m : n;
  Out o{(char*)a.out[0], 0, a.count[0], 0, a.f32};
  int first = 0;
#pragma unroll
  for (int k = 1; k < kMaxParts; ++k)
    if (k < a.parts && at >= a.first[k])
      o.p = (char*)a.out[k], first = a.first[k], o.count = a.count[k];
  if (a.by_rows) {
    o.p -= (long long)first * a.width * (a.f32 ? 4 : 2);
    o.rows = first + o.count;
    o.count = a.width;
    o.c0 = n;
  } else {
    o.rows = a.M;
    o.c0 = n - first;
  }
  return o;
}

// columns [c, c + 4) of row m; an odd row is aligned to a value only, which
// these stores may be
__device__ __forceinline__ void store4(const Out& o, int m, int c, f32x4 v) {
  const long long at = (long long)m * o.count + c;
  if (c + 4 <= o.count) {
    if (o.f32) {
      __builtin_memcpy((float*)o.p + at, &v, 16);
    } else {
      const u32x2 d{Bf16::from_f(v[0]) | (uint32_t)Bf16::from_f(v[1]) << 16,
                    Bf16::from_f(v[2]) | (uint32_t)Bf16::from_f(v[3]) << 16};
      __builtin_memcpy((uint16_t*)o.p + at, &d, 8);
    }
    return;
  }
#pragma unroll
  for (int i = 0; i < 3; ++i) {
    if (c + i >= o.count) break;
    if (o.f32)
      ((float*)o.p)[at + i] = v[i];
    else
      ((uint16_t*)o.p)[at + i] = Bf16::from_f(v[i]);
  }
}

// ------------------------------------------------------------ tiles in LDS
// Four waves, 2 x 2, each FX x FW products of 32x32x64 (one is half a block
// of K; both halves take the same scale).  One workgroup a CU, so the
// overlap is inside the wave: the fragments of the next half step are read
// while this half's products run, and one barrier a K step serves both uses
// of a buffer:
//
//   half 0: products of (kt, 0)    reads (kt, 1) from buffer kt
//   barrier: buffer kt is read by all, the loads of kt + 1 have landed
//   half 1: products of (kt, 1)    reads (kt + 1, 0) from buffer kt + 1
//                                  loads kt + NBUF into buffer kt
//
// Every wave issues the same number of loads a step, so that the barrier
// waits for the oldest step's only and leaves NBUF - 2 steps in flight.
//
// 4 x 4 is for large products: a wave reads 128 + 128 bytes of LDS a unit of
// K for 128 x 128 products; eight waves of 128 x 64 would read 1.5 times as
// much, which with the writes is all that LDS can do.  The smaller tiles
// have more workgroups and more steps in flight, for products too small to
// fill the card with 256 x 256.
//
// Measured for Y of 24576 x 14336, K 4096: 1100 to 1160 us (2.5 to 2.6
// PFLOP/s) on warm cards; 24576 x 4096, K 14336: 1010 to 1060;
// 14336 x 4096, K 24576 with its split last round: 1050 to 1070.  What
// bounds them is power: the matrix units are busy 72, 80 and 79 % of the
// cycles at a clock that falls from 2.4 to 1.64 GHz, and the products alone,
// without any load, take 840 us of the 1010.  Of the LDS cycles 5, 1.5 and
// 0.8 % are bank conflicts (all in the epilogue).  Two tries that lost:
// workgroups that stay and load their next tile's first steps early (1144 us
// to 1119), results stored straight from registers after swaps between lanes
// (1150 to 1144, and 137 to 131 for K 2048).
using f32x16 = __attribute__((ext_vector_type(16))) float;

// The work of one launch: `full` tiles as a whole, then each of the others
// `splits` times with a share of K, whose sums go to partials.  Tiles come
// in order of bands of four tile rows, column by column; each of the 8 XCDs
// takes a contiguous run of that order, so that the tiles in its L2 at one
// time are a compact block.
struct TileWork {
  int tiles_m, tiles_n, full, splits;
  int items;  // full + (tiles - full) * splits
  float* partials;
};

__device__ __forceinline__ int xcd_run(int i, int n) {
  const int q = n / 8, r = n % 8, xcd = i % 8, idx = i / 8;
  return (xcd < r ? xcd * (q + 1) : r * (q + 1) + (xcd - r) * q) + idx;
}

struct Item {
  int m0, n0, q0, q1;  // q: quads of K steps; scale dwords stay whole
  int partial;         // index of its partial sums, -1 for a whole tile
};
template <int BM, int BN>
__device__ __forceinline__ Item item_of(const TileWork& work, int quads,
                                        int i) {
  constexpr int kBand = 4;
  Item it{0, 0, 0, quads, -1};
  int t;
  if (i < work.full) {
    t = xcd_run(i, work.full);
  } else {
    const int rest = work.tiles_m * work.tiles_n - work.full;
    const int k = (i - work.full) % rest, split = (i - work.full) / rest;
    t = work.full + xcd_run(k, rest);
    if (work.splits > 1) {
      it.q0 = (int)((long long)quads * split / work.splits);
      it.q1 = (int)((long long)quads * (split + 1) / work.splits);
      it.partial = (t - work.full) * work.splits + split;
    }
  }
  const int band = t / (kBand * work.tiles_n);
  const int in_band = t % (kBand * work.tiles_n);
  const int rows = min(kBand, work.tiles_m - band * kBand);
  it.m0 = (band * kBand + in_band % rows) * BM;
  it.n0 = in_band / rows * BN;
  // divisions are done in vector registers; buffer descriptors need scalars
  it.m0 = __builtin_amdgcn_readfirstlane(it.m0);
  it.n0 = __builtin_amdgcn_readfirstlane(it.n0);
  it.q0 = __builtin_amdgcn_readfirstlane(it.q0);
  it.q1 = __builtin_amdgcn_readfirstlane(it.q1);
  it.partial = __builtin_amdgcn_readfirstlane(it.partial);
  return it;
}

template <int FX, int FW, int NBUF>
__global__ __launch_bounds__(256, 1) void gemm_tile(GemmArgs a,
                                                    TileWork work) {
  constexpr int BM = 64 * FX, BN = 64 * FW, kRows = BM + BN;
  constexpr int kTile = kRows * 128, kScales = kRows * 4;
  constexpr int kRing = NBUF <= 2 ? 2 : 4;     // quads of scales
  constexpr int kProducts = FX * FW;           // a half step
  constexpr int kReads = 2 * (FX + FW);        // 16 bytes a lane
  constexpr int kLoads = kRows / 32;           // tile loads a step and wave
  constexpr int kInFlight = (NBUF - 2) * (kLoads + 2);
  static_assert(kInFlight < 64 && 4 * kRing >= NBUF + 6);
  __shared__ __align__(16) char lds[NBUF * kTile + kRing * kScales];
  const int lane = threadIdx.x & 63;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);

  const int quads = (a.KT + 3) >> 2;
  const Item it = item_of<BM, BN>(work, quads, blockIdx.x);
  const int m0 = it.m0, n0 = it.n0, q0 = it.q0, q1 = it.q1;
  const int wm = (wave >> 1) * (BM / 2), wn = (wave & 1) * (BN / 2);

  const int KT = min(4 * q1, a.KT) - 4 * q0;

  // Loads by buffer descriptors: rows past the end read as zero (the range
  // check counts the whole offset, and what fails it arrives in LDS as
  // zeros), and all that changes from step to step is a base address a
  // matrix.  Scalar arithmetic between the products would hold them up: a
  // lone wave issues one instruction in about four cycles.
  const uint8_t* px = a.x + (4 * q0 * a.xn + m0) * 128;
  const uint8_t* pw = a.w + (4 * q0 * a.wn + n0) * 128;
  const long long x_step = a.xn * 128, w_step = a.wn * 128;
  const int x_bytes = min(BM, a.M - m0) * 128;
  const int w_bytes = min(BN, a.N - n0) * 128;
  const auto rxs = __builtin_amdgcn_make_buffer_rsrc(
      (void*)(a.xs + q0 * a.xsp + m0), 0,
      (int)((quads - q0) * a.xsp - m0) * 4, 0x00020000);
  const auto rws = __builtin_amdgcn_make_buffer_rsrc(
      (void*)(a.ws + q0 * a.wsp + n0), 0,
      (int)((quads - q0) * a.wsp - n0) * 4, 0x00020000);
  const int lrow = wave * 8 + (lane >> 3);
  const int at = lrow * 128 + ((lane & 7) ^ (lrow >> 1 & 7)) * 16;
  // the n-th of a step's loads: 32 rows of x, then of w
  auto load = [&](int step, int n) {
    char* to = lds + step % NBUF * kTile + (n * 32 + wave * 8) * 128;
    if (n < BM / 32)
      __builtin_amdgcn_raw_ptr_buffer_load_lds(
          __builtin_amdgcn_make_buffer_rsrc((void*)px, 0, x_bytes,
                                            0x00020000),
          B8_LDS(to), 16, at, n * 4096, 0, 0);
    else
      __builtin_amdgcn_raw_ptr_buffer_load_lds(
          __builtin_amdgcn_make_buffer_rsrc((void*)pw, 0, w_bytes,
                                            0x00020000),
          B8_LDS(to), 16, at, (n - BM / 32) * 4096, 0, 0);
  };
  auto advance = [&](int step) {
    px += step + 1 < KT ? x_step : 0;
    pw += step + 1 < KT ? w_step : 0;
  };
  // two loads of scales a step and wave, those of quad (step + 3) / 4: its
  // four steps bring it four times, all before the first of them is read
  const int sx_at = wave % (BM / 64) * 64, sw_at = wave % (BN / 64) * 64;
  auto load_scales = [&](int q) {
    char* to = lds + NBUF * kTile + q % kRing * kScales;
    const int at = min(q, q1 - q0 - 1);
    __builtin_amdgcn_raw_ptr_buffer_load_lds(
        rxs, B8_LDS(to + sx_at * 4), 4, (sx_at + lane) * 4,
        at * (int)a.xsp * 4, 0, 0);
    __builtin_amdgcn_raw_ptr_buffer_load_lds(
        rws, B8_LDS(to + (BM + sw_at) * 4), 4, (sw_at + lane) * 4,
        at * (int)a.wsp * 4, 0, 0);
  };

  // fragment (row = lane % 32, 32 bytes at half * 64 + lane / 32 * 32), in
  // the order that the products want them: x0 w0 .. x1 ..
  struct Half {
    i32x8 x[FX], w[FW];
  };
  const int frow = lane & 31, fg = lane >> 5;
  auto read = [&](Half& f, int kt, int half, int n) {
    const int k = n / 2, c = 4 * half + 2 * fg + n % 2;
    const bool of_w = k >= 1 && k <= FW;
    const int row = of_w ? BM + wn + (k - 1) * 32
                         : wm + (k ? k - FW : 0) * 32;
    const i32x4 v = *(const i32x4*)(lds + kt % NBUF * kTile +
                                    swizzled(row + frow, c));
    i32x8& to = of_w ? f.w[k - 1] : f.x[k ? k - FW : 0];
#pragma unroll
    for (int i = 0; i < 4; ++i) to[n % 2 * 4 + i] = v[i];
  };
  uint32_t quad_x[FX], quad_w[FW];  // the scales of four K steps
  auto read_scales = [&](int kt) {
    const uint32_t* sc = (const uint32_t*)(lds + NBUF * kTile +
                                           (kt >> 2) % kRing * kScales);
#pragma unroll
    for (int i = 0; i < FX; ++i) quad_x[i] = sc[wm + i * 32 + frow];
#pragma unroll
    for (int j = 0; j < FW; ++j) quad_w[j] = sc[BM + wn + j * 32 + frow];
  };

  f32x16 acc[kProducts];
#pragma unroll
  for (int i = 0; i < kProducts; ++i)
#pragma unroll
    for (int j = 0; j < 16; ++j) acc[i][j] = 0.f;
  auto product = [&](const Half& f, const int (&sx)[FX], const int (&sw)[FW],
                     int n) {
    acc[n] = __builtin_amdgcn_mfma_scale_f32_32x32x64_f8f6f4(
        f.w[n % FW], f.x[n / FW], acc[n], 0, 0, 0, sw[n % FW], 0,
        sx[n / FW]);
  };
  auto meet = [&] {
    asm volatile("s_waitcnt vmcnt(%0) lgkmcnt(0)" ::"n"(kInFlight)
                 : "memory");
    __builtin_amdgcn_s_barrier();
    asm volatile("" ::: "memory");
  };

  // Past the last step the loads repeat it and the reads find what is
  // there; nothing uses either.  The alternative, a peeled tail, made the
  // compiler copy all accumulators.
#pragma unroll
  for (int step = 0; step < NBUF; ++step) {
    load_scales((step + 3) >> 2);
#pragma unroll
    for (int n = 0; n < kLoads; ++n) load(step, n);
    advance(step);
  }
  asm volatile("s_waitcnt vmcnt(%0)" ::"n"((NBUF - 1) * (kLoads + 2))
               : "memory");
  __builtin_amdgcn_s_barrier();
  asm volatile("" ::: "memory");
  Half f0, f1;
#pragma unroll
  for (int n = 0; n < kReads; ++n) read(f0, 0, 0, n);
  read_scales(0);
  // the reads are done early in the half, the loads spread over it
  constexpr int kReadsEach =
      kProducts >= 4 ? 2 : (kReads + kProducts - 1) / kProducts;
  constexpr int kLoadsEach = (kLoads + kProducts - 1) / kProducts;
  static_assert(kReadsEach * kProducts >= kReads);
  // the fence after each product keeps the order written here: loads in a
  // burst would fill the memory unit's queue and hold up the products
  for (int kt = 0; kt < KT; ++kt) {
    int sx[FX], sw[FW];
#pragma unroll
    for (int i = 0; i < FX; ++i) sx[i] = (int)(quad_x[i] >> (8 * (kt & 3)));
#pragma unroll
    for (int j = 0; j < FW; ++j) sw[j] = (int)(quad_w[j] >> (8 * (kt & 3)));
#pragma unroll
    for (int n = 0; n < kProducts; ++n) {
      product(f0, sx, sw, n);
#pragma unroll
      for (int k = n * kReadsEach; k < (n + 1) * kReadsEach; ++k)
        if (k < kReads) read(f1, kt, 1, k);
      __builtin_amdgcn_sched_barrier(0);
    }
    meet();
#pragma unroll
    for (int n = 0; n < kProducts; ++n) {
      product(f1, sx, sw, n);
      if (n == 0) load_scales((kt + NBUF + 3) >> 2);
#pragma unroll
      for (int k = n * kLoadsEach; k < (n + 1) * kLoadsEach; ++k)
        if (k < kLoads) load(kt + NBUF, k);
#pragma unroll
      for (int k = n * kReadsEach; k < (n + 1) * kReadsEach; ++k)
        if (k < kReads) read(f0, kt + 1, 0, k);
      if (n == kProducts / 2) read_scales(kt + 1);
      if (n == kProducts - 1) advance(kt + NBUF);
      __builtin_amdgcn_sched_barrier(0);
    }
  }
  asm volatile("s_waitcnt vmcnt(0) lgkmcnt(0)" ::: "memory");
  __builtin_amdgcn_s_barrier();
  asm volatile("" ::: "memory");

  // lane: row m = lane % 32 of its fragment, columns (r / 4) * 8 +
  // lane / 32 * 4 + r % 4
  if (it.partial >= 0) {
    // in the order of the registers; join_splits knows it
    f32x4* p = (f32x4*)work.partials +
               ((long long)it.partial * 4 + wave) * kProducts * 256 + lane;
#pragma unroll
    for (int i = 0; i < kProducts; ++i)
#pragma unroll
      for (int r = 0; r < 4; ++r)
        p[(i * 4 + r) * 64] = f32x4{acc[i][4 * r], acc[i][4 * r + 1],
                                    acc[i][4 * r + 2], acc[i][4 * r + 3]};
    return;
  }
  const Out o = out_of(a, m0 + wm, n0 + wn);
  // straight from the accumulators: dW of 14336 x 4096, K 24576, takes 27 us
  // more than in bf16, and 117 MB more to write are 24
  if (o.f32) {
#pragma unroll
    for (int i = 0; i < FX; ++i) {
      const int m = m0 + wm + i * 32 + frow;
      if (m < o.rows) {
#pragma unroll
        for (int j = 0; j < FW; ++j)
#pragma unroll
          for (int r = 0; r < 4; ++r) {
            const f32x16& v = acc[i * FW + j];
            store4(o, m, o.c0 + j * 32 + r * 8 + fg * 4,
                   f32x4{v[4 * r], v[4 * r + 1], v[4 * r + 2],
                         v[4 * r + 3]});
          }
      }
    }
    return;
  }
  // through LDS, so that a row's lanes store whole lines: straight from the
  // accumulators a store would touch 16 bytes of 32 rows.  16-byte chunk c
  // of row m lies at c ^ m % kChunks
  constexpr int kChunks = FW * 4, kRowBytes = FW * 64;
  char* mine = lds + wave * (FX * 32 * kRowBytes);
#pragma unroll
  for (int i = 0; i < FX; ++i) {
    const int m = i * 32 + frow;
#pragma unroll
    for (int j = 0; j < FW; ++j)
#pragma unroll
      for (int r = 0; r < 4; ++r) {
        const f32x16& v = acc[i * FW + j];
        *(u32x2*)(mine + m * kRowBytes +
                  (((j * 4 + r) ^ m % kChunks) << 4) + fg * 8) =
            u32x2{Bf16::from_f(v[4 * r]) |
                      (uint32_t)Bf16::from_f(v[4 * r + 1]) << 16,
                  Bf16::from_f(v[4 * r + 2]) |
                      (uint32_t)Bf16::from_f(v[4 * r + 3]) << 16};
      }
  }
  asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
  const int c = lane % kChunks;
  const int left = o.count - (o.c0 + c * 8);
  if (left <= 0) return;
  uint16_t* out = (uint16_t*)o.p + o.c0 + c * 8;
  constexpr int kRowsEach = 64 / kChunks;
  using Pair __attribute__((aligned(2))) = u32x4;
  auto write = [&](auto stream) {
#pragma unroll 8
    for (int k = 0; k < FX * 32 / kRowsEach; ++k) {
      const int row = k * kRowsEach + lane / kChunks, m = m0 + wm + row;
      const u32x4 v = *(const u32x4*)(mine + row * kRowBytes +
                                      ((c ^ row % kChunks) << 4));
      if (m >= o.rows) continue;
      uint16_t* to = out + (long long)m * o.count;
      if (left >= 8) {
        if constexpr (stream)
          __builtin_nontemporal_store(v, (Pair*)to);
        else
          *(Pair*)to = v;
      } else {
#pragma unroll
        for (int i = 0; i < 7; ++i)
          if (i < left) to[i] = (uint16_t)(v[i / 2] >> (16 * (i & 1)));
      }
    }
  };
  // two loops: stores of one loop's two branches would become one store
  if (a.stream)
    write(std::true_type());
  else
    write(std::false_type());
}

// the sums of a split tile, in the order of the splits, to the outputs: 4
// values a thread, a wave's fragment and register group a workgroup
template <int FX, int FW>
__global__ __launch_bounds__(256) void join_splits(GemmArgs a,
                                                   TileWork work) {
  constexpr int BM = 64 * FX, BN = 64 * FW, kProducts = FX * FW;
  const int lane = threadIdx.x & 63, r = threadIdx.x >> 6;
  const int frag = blockIdx.x % kProducts;
  const int wave = blockIdx.x / kProducts % 4;
  const int k = blockIdx.x / (kProducts * 4);
  const Item it = item_of<BM, BN>(work, (a.KT + 3) >> 2, work.full + k);
  const f32x4* p = (const f32x4*)work.partials +
                   (((long long)it.partial * 4 + wave) * kProducts + frag) *
                       256 +
                   r * 64 + lane;
  f32x4 v = p[0];
  for (int s = 1; s < work.splits; ++s)
    v += p[(long long)s * 4 * kProducts * 256];
  const int wm = (wave >> 1) * (BM / 2), wn = (wave & 1) * (BN / 2);
  const int m = it.m0 + wm + frag / FW * 32 + (lane & 31);
  const Out o = out_of(a, it.m0 + wm, it.n0 + wn);
  if (m < o.rows)
    store4(o, m, o.c0 + frag % FW * 32 + r * 8 + (lane >> 5) * 4, v);
}

// ------------------------------------------------------- K over the waves
// Small products, few rows among them: what counts is how soon all of w and
// x is under way.  A workgroup takes 16 FM rows of x by 16 FN rows of w; its
// waves share K, a step at a time, and load their operands straight from
// global memory: within a workgroup nothing is read twice, so LDS would save
// nothing, and there is no barrier before the sums meet in LDS, added in the
// order of the waves.  With FUSED, for up to 32 rows of bf16, x is packed on
// the way: each lane needs 32 neighbouring values a step, which four lanes
// share a scale for, so the codes are those of pack_rows and a launch is
// saved.  Bound by the read of w: a call of 8 x 14336, K 4096 takes 13.5 us
// (4.4 TB/s of 59 MB) on one weight, which the last cache holds, and 15.1
// (3.9 TB/s) on weights in turn that come from memory, as a decoded token's
// do; 1 x 2048, K 2048 3.8 and 4.7, all of it latency.
struct SplitArgs {
  GemmArgs g;
  const uint16_t* x;  // FUSED: bf16, rows of ldx elements, K columns
  long long ldx;
  int K, tiles_n;
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
  top = max_rows(top);
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

template <int FM, int FN, int WAVES, bool FUSED>
__global__ __launch_bounds__(WAVES * 64) void gemm_split(SplitArgs sa) {
  const GemmArgs& a = sa.g;
  extern __shared__ f32x4 sums[];  // [WAVES][FM * FN][64]
  const int lane = threadIdx.x & 63;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int r = lane & 15, g = lane >> 4;
  const int m0 = (int)(blockIdx.x / sa.tiles_n) * 16 * FM;
  const int n0 = (int)(blockIdx.x % sa.tiles_n) * 16 * FN;
  // rows past the end repeat the last one and are not stored
  const uint8_t* w[FN];
  const uint32_t* ws[FN];
#pragma unroll
  for (int j = 0; j < FN; ++j) {
    const int n = min(n0 + j * 16 + r, a.N - 1);
    w[j] = a.w + n * 128ll + g * 32;
    ws[j] = a.ws + n;
  }
  const uint8_t* x[FM];
  const uint32_t* xs[FM];
  if constexpr (!FUSED) {
#pragma unroll
    for (int i = 0; i < FM; ++i) {
      const int m = min(m0 + i * 16 + r, a.M - 1);
      x[i] = a.x + m * 128ll + g * 32;
      xs[i] = a.xs + m;
    }
  }

  f32x4 acc[FM * FN];
#pragma unroll
  for (int i = 0; i < FM * FN; ++i) acc[i] = f32x4{0.f, 0.f, 0.f, 0.f};
  for (int kt = wave; kt < a.KT; kt += WAVES) {
    i32x4 wv[FN][2], xv[FM][2];
    u32x4 raw[FM][4];
    uint32_t wq[FN], xq[FM];
#pragma unroll
    for (int j = 0; j < FN; ++j) {
      wq[j] = ws[j][(kt >> 2) * a.wsp];
      const i32x4* p = (const i32x4*)(w[j] + kt * a.wn * 128);
      wv[j][0] = p[0];
      wv[j][1] = p[1];
    }
    if constexpr (FUSED) {
#pragma unroll
      for (int i = 0; i < FM; ++i)
#pragma unroll
        for (int c = 0; c < 4; ++c) {
          const int k = kt * 128 + g * 32 + c * 8, m = i * 16 + r;
          raw[i][c] = m < a.M && k < sa.K
                          ? *(const u32x4*)(sa.x + m * sa.ldx + k)
                          : u32x4{0, 0, 0, 0};
        }
    } else {
#pragma unroll
      for (int i = 0; i < FM; ++i) {
        xq[i] = xs[i][(kt >> 2) * a.xsp];
        const i32x4* p = (const i32x4*)(x[i] + kt * a.xn * 128);
        xv[i][0] = p[0];
        xv[i][1] = p[1];
      }
    }
    const int shift = 8 * (kt & 3);
#pragma unroll
    for (int i = 0; i < FM; ++i) {
      int sx;
      i32x8 xf;
      if constexpr (FUSED) {
        xf = pack_step(raw[i], &sx);
      } else {
        xf = __builtin_shufflevector(xv[i][0], xv[i][1], 0, 1, 2, 3, 4, 5, 6,
                                     7);
        sx = (int)(xq[i] >> shift);
      }
#pragma unroll
      for (int j = 0; j < FN; ++j)
        acc[i * FN + j] = __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(
            __builtin_shufflevector(wv[j][0], wv[j][1], 0, 1, 2, 3, 4, 5, 6,
                                    7),
            xf, acc[i * FN + j], 0, 0, 0, (int)(wq[j] >> shift), 0, sx);
    }
  }
#pragma unroll
  for (int i = 0; i < FM * FN; ++i)
    sums[(wave * FM * FN + i) * 64 + lane] = acc[i];
  __syncthreads();
#pragma unroll
  for (int f = 0; f < FM * FN; f += WAVES) {
    if (f + wave >= FM * FN) return;
    const int i = (f + wave) / FN, j = (f + wave) % FN;
    f32x4 v = sums[(f + wave) * 64 + lane];
#pragma unroll
    for (int k = 1; k < WAVES; ++k)
      v += sums[(k * FM * FN + f + wave) * 64 + lane];
    const int m = m0 + i * 16 + r;
    const Out o = out_of(a, m0, n0 + j * 16);
    if (m < o.rows) store4(o, m, o.c0 + 4 * g, v);
  }
}

template <int FM, int FN, int WAVES, bool FUSED>
static hipError_t split_run(SplitArgs sa, hipStream_t st) {
  constexpr int kLds = WAVES * FM * FN * 64 * 16;
  const auto kernel = gemm_split<FM, FN, WAVES, FUSED>;
  sa.tiles_n = (sa.g.N + 16 * FN - 1) / (16 * FN);
  const long long tiles_m = (sa.g.M + 16 * FM - 1) / (16 * FM);
  return launch(kernel, tiles_m * sa.tiles_n, WAVES * 64, kLds, st, sa);
}

// --------------------------------------------------------------- the choice
// Which kernel, and K split how often: the one with the least predicted
// time.  A tile takes fixed + steps * step us, where a step is slower when
// the whole card computes (its power limit); one workgroup fits a CU, so
// more than 256 tiles go in rounds.  K is split for the tiles of the last,
// partly filled round only.  Measured in us (gfx950, K steps of 128, one
// workgroup .. 256; a launch's first round takes about 2 us more):
//
//   tile       fixed   step alone   step on a full card
//   256 x 256    9.0      0.93          1.37
//   128 x 256    5.5      0.62          0.85
//   128 x 128    3.7      0.36          0.48
//    64 x  64    2.0      0.29          0.33
//
// Joining the splits costs a launch, about 2.5 us, and their traffic at about
// 5 TB/s.  gemm_split takes 0.6 + 0.16 steps us for each 256 workgroups.
// Over 220 products of up to 24576 x 14336 the choice is within 1 % of the
// best on average.  All of it was measured on operands that the caches hold
// as far as they fit, the model's figures too.  Measured either way (M x N,
// K), in us:
//   24576 x 4096, 14336: 1014 by 256 x 256 and 1500 by 128 x 128
//   4096 x 2048, 16384: 135 by 256 x 256, 117 with K split in two, 116 by
//     128 x 256, 133 by 128 x 128
//   2048 x 2048, 2048: 25, 17, 12.5 by 128 x 128, 29 by 64 x 64
//   1001 x 777, 1111: 18.5, 12.5, 8.6, 6.5 by 64 x 64
//   128 x 4096, 14336: 48 by 128 x 128, 20 in four splits
//   710 x 229, 176: 4.3 by 64 x 64, 3.4 by gemm_split
constexpr int kCUs = 256;

struct Plan {
  int kind;  // 0 256 x 256, 1 128 x 256, 2 128 x 128, 3 64 x 64, 4 gemm_split
  TileWork work;
  long long workspace;
};

static Plan plan_of(const GemmArgs& a) {
  static const struct {
    int bm, bn;
    float fixed, alone, full;
  } kinds[] = {{256, 256, 9.0f, 0.93f, 1.37f},
               {128, 256, 5.5f, 0.62f, 0.85f},
               {128, 128, 3.7f, 0.36f, 0.48f},
               {64, 64, 2.0f, 0.29f, 0.33f}};
  const int quads = (a.KT + 3) / 4;
  Plan best{};
  best.kind = -1;
  float least = 0.f;
  for (int k = 0; k < 4; ++k) {
    const auto& kind = kinds[k];
    const int tm = (a.M + kind.bm - 1) / kind.bm;
    const int tn = (a.N + kind.bn - 1) / kind.bn;
    const long long tiles = (long long)tm * tn;
    const long long rest = tiles % kCUs;
    const long long rounds = tiles / kCUs;
    for (int splits = 1; splits <= 8; splits *= 2) {
      if (splits > 1 && (quads < 2 * splits || rest == 0)) break;
      const long long last = rest * splits;  // workgroups of the last round
      const float steps =
          splits > 1 ? 4.f * ((quads + splits - 1) / splits) : a.KT;
      float us = 2.f + rounds * (kind.fixed + a.KT * kind.full);
      us += last / kCUs * (kind.fixed + steps * kind.full);
      if (last % kCUs)
        us += kind.fixed + steps * (kind.alone + (kind.full - kind.alone) *
                                               (last % kCUs) / kCUs);
      if (splits > 1)
        us += 2.5f + (4.f * splits + 2.f) * rest * kind.bm * kind.bn / 5e6f;
      if (least == 0.f || us < least) {
        least = us;
        const long long full = splits > 1 ? tiles - rest : tiles;
        const long long items = full + (tiles - full) * splits;
        if (items >= 1ll << 24) continue;  // a launch has < 2^32 threads
        best.kind = k;
        best.work = TileWork{tm, tn, (int)full, splits, (int)items, nullptr};
        best.workspace =
            splits > 1 ? 4ll * splits * rest * kind.bm * kind.bn : 0;
      }
    }
  }
  // 32 rows of x by 16 of w a workgroup, its waves sharing K
  const long long groups = (a.M + 31) / 32 * ((a.N + 15) / 16);
  const float us = 2.f + (groups + kCUs - 1) / kCUs * (0.6f + 0.16f * a.KT);
  if (groups < 1 << 22 && (us < least || best.kind < 0)) best = Plan{4};
  return best;
}

template <int FX, int FW, int NBUF>
static hipError_t tile_run(const GemmArgs& a, const Plan& p,
                           hipStream_t st) {
  const hipError_t e =
      launch(gemm_tile<FX, FW, NBUF>, p.work.items, 256, 0, st, a, p.work);
  const long long rest =
      (long long)p.work.tiles_m * p.work.tiles_n - p.work.full;
  if (e != hipSuccess || !rest) return e;
  return launch(join_splits<FX, FW>, rest * 4 * FX * FW, 256, 0, st, a,
                p.work);
}

}  // namespace b8

using namespace b8;

extern "C" long long b8_gemm_workspace(const GemmArgs* args) {
  const Plan p = plan_of(*args);
  return p.kind < 0 ? -1 : p.workspace;
}

extern "C" hipError_t launch_b8_gemm(const GemmArgs* args, float* workspace,
                                     hipStream_t st) {
  const GemmArgs a = *args;
  Plan p = plan_of(a);
  p.work.partials = workspace;
  if (p.kind == 0)
    return tile_run<4, 4, 2>(a, p, st);
  if (p.kind == 1)
    return tile_run<2, 4, 3>(a, p, st);
  if (p.kind == 2)
    return tile_run<2, 2, 4>(a, p, st);
  if (p.kind == 3)
    return tile_run<1, 1, 8>(a, p, st);
  return split_run<2, 1, 16, false>(SplitArgs{a}, st);
}

// Whether x in bf16 is packed on the way: up to 16 rows always, up to 32 where
// few workgroups repeat the packing.  A call with a launch for packing and
// without, in us, on weights in turn that come from memory: 24 rows (N x K)
// 2048 x 2048 8.0 and 7.6, 8192 x 2048 10.6 and 9.3, 8192 x 512 6.8 and 5.2;
// but 4096 x 4096 10.6 and 12.0, 14336 x 4096 17.1 and 27.6.  8 rows
// 4096 x 4096 9.5 and 8.4, 8192 x 4096 15.7 and 10.3, 14336 x 4096 16.6 and
// 15.2; where K is long 16 rows lose: 4096 x 4096 9.9 and 9.8, 4096 x 14336
// 21.1 and 26.7.
extern "C" bool b8_packs_on_the_way(const GemmArgs* args) {
  // a launch has fewer than 2^32 threads, 16 a row of w
  return args->M <= 16 ? args->N < 1 << 28
                       : args->M <= 32 && args->N <= 8192 && args->KT <= 16;
}

// x in rows of K columns, K and ldx multiples of 8; the codes of x in args
// are not read.  A workgroup takes 16 columns of y for each FN: more share
// the packing of x, fewer are more workgroups.  A call with 1, 2 and 4 in us,
// on one weight, which the last cache holds / on weights in turn from memory:
//   1 x 2048, K 2048     3.8,  4.6,  6.7 /  4.7,  5.6,  7.7
//   8 x 4096, K 4096     6.7,  8.1, 11.9 /  8.4,  9.7, 13.5
//   8 x 6144, K 4096    11.4,  8.2, 12.0 / 14.0, 10.0, 13.7
//   16 x 8192, K 2048    8.4,  6.1,  7.9 / 10.8,  8.1,  9.8
//   8 x 14336, K 4096   23.4, 16.0, 13.7 / 25.7, 18.3, 15.2
//   24 x 4096, K 2048    6.5,  7.4       /  7.8,  8.9
//   24 x 8192, K 2048   11.3,  7.5       / 13.2,  9.3
// 1 is best up to 256 workgroups (4096 columns), one a CU, 2 up to 512 (8192).
// The limits here lie halfway to the next such width, so that just below them
// a narrower kernel runs than the best: 1 at 6144 columns.
extern "C" hipError_t launch_b8_gemm_bf16(const GemmArgs* args, const void* x,
                                          long long ldx, int K,
                                          hipStream_t st) {
  const SplitArgs sa{*args, (const uint16_t*)x, ldx, K};
  if (args->M > 16)
    return args->N <= 4096 ? split_run<2, 1, 16, true>(sa, st)
                           : split_run<2, 2, 16, true>(sa, st);
  if (args->N <= 6144) return split_run<1, 1, 16, true>(sa, st);
  if (args->N <= 12288) return split_run<1, 2, 16, true>(sa, st);
  return split_run<1, 4, 16, true>(sa, st);
}
