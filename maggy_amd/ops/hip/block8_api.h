// What the launchers of block8.hip and gemm8.hip take; plain C++, shared
// with the bindings.
#pragma once
#include <hip/hip_runtime.h>
#include <cstdint>
#include <tuple>

namespace b8 {

// From these sizes on plain rows pass by the caches, so that these keep the
// packed operands, which every tile of a product reads again: results that
// the next kernel may want, and what is read once or wanted much later
// (operands to pack, gradients of weights).  Measured in us, streamed and
// not: linear8 24576x4096 -> 14336 trained 3480 and 3637, 4096x2048 -> 2 x
// 8192 427 and 471; 24576 x 4096 normed, with gradients, 198 and 216, packed
// and read back 100 and 125.  Small results are better found in a cache: a
// feed-forward of 64 rows takes 57.9 with all streamed and 57.5 with none.
// Codes always stay: a feed-forward of 512 rows 128, with codes streamed 132.
constexpr long long kStreamResult = 64 << 20, kStreamOnce = 32 << 20;

// What is packed of a matrix by 128 x 128 tiles (block8.hip): its rows, its
// columns (the transpose) or both, by blocks of their own or by one scale a
// tile, from plain numbers or from a packed matrix
enum TileKind {
  kTileBoth,
  kTileCols,
  kTileRows,
  kTileOneRows,
  kTileOneCols,
  kTileFrom8,  // columns of a packed matrix
};
struct TileJob {
  TileKind kind;
  int dtype, vec;       // 0 bf16, 2 fp32; whether 16-byte loads may be used
                        // (the launcher decides on how)
  int first_block;      // of the launch; a workgroup packs a tile
  const void* x;        // plain numbers, or codes
  const uint32_t* xs;   // codes: their scales
  long long ldx;        // elements a row (codes: rows of the packed matrix)
  long long xsp;        // codes: padded rows of xs
  int R, C;
  // outputs are packed matrices of row_n, col_n rows (scales row_sp, col_sp)
  uint8_t* row_codes;   // value (r, c) is at row row_r0 + r, column
  uint8_t* row_scales;  // row_c0 + c; the offsets are multiples of 128
  long long row_n, row_sp, row_c0, row_r0;
  uint8_t* col_codes;   // transposed: at row col_r0 + c, column col_c0 + r
  uint8_t* col_scales;
  long long col_n, col_sp, col_r0, col_c0;
};

// Y[m][n] = sum_k X[m][k] W[n][k], X and W packed along k (gemm8.hip).
// The rows of W are up to four matrices, each padded to a multiple of 128
// rows; each has a contiguous output of its own.  Or the rows of X are, where
// X is the gradients of several outputs and Y those of their weights.
constexpr int kMaxParts = 4;
// all packing that one call of linear8 needs is one launch
constexpr int kMaxJobs = 2 * kMaxParts + 1;
struct TileJobs {
  TileJob job[kMaxJobs];
  int count;
};
struct GemmArgs {
  const uint8_t* x;
  const uint32_t* xs;
  long long xn, xsp;  // rows of the codes, padded rows of the scales
  const uint8_t* w;
  const uint32_t* ws;
  long long wn, wsp;
  int M, N;  // rows of x and of w that take part
  int KT;    // K steps of 128
  void* out[kMaxParts];
  int first[kMaxParts];  // first row of w, or of x
  int count[kMaxParts];  // columns of the output, or rows
  int parts;
  int by_rows;  // the parts are rows of x
  int width;    // then: columns of every output
  int f32;  // outputs are fp32, else bf16
  int stream;  // outputs in bf16 pass by the caches
};

#ifdef __HIPCC__
// Arguments are converted to what the kernel takes.  The status is this
// launch's own, not one that an earlier call left.
template <class... P, class... A>
static inline hipError_t launch(void (*kernel)(P...), long long blocks,
                                int threads, int lds, hipStream_t st,
                                A... args) {
  std::tuple<P...> values(static_cast<P>(args)...);
  const hipError_t e = std::apply(
      [&](P&... v) {
        void* at[] = {(void*)&v...};
        return hipLaunchKernel((const void*)kernel, dim3((unsigned)blocks),
                               dim3(threads), at, lds, st);
      },
      values);
  if (e != hipSuccess) (void)hipGetLastError();  // it is reported here
  return e;
}
#endif

}  // namespace b8

// every launch returns its status
extern "C" {
hipError_t launch_b8_pack(int dtype, int vec, const void* x, long long ldx,
                    long long R, int C, uint8_t* codes, int Cp,
                    uint32_t* scales, long long Rp, hipStream_t st);
hipError_t launch_b8_unpack(int dtype, int vec, const uint8_t* codes, int Cp,
                      const uint32_t* scales, long long Rp, long long R,
                      int C, void* out, hipStream_t st);
// sets the jobs' first blocks; returns how many there are, -1 if too many
long long b8_tile_blocks(b8::TileJobs* jobs);
hipError_t launch_b8_tiles(const b8::TileJobs* jobs, long long blocks,
                           hipStream_t st);
hipError_t launch_b8_swiglu_fwd(int dtype, int vec, const void* g, long long ldg,
                          const void* u, long long ldu, long long R, int C,
                          void* h, uint8_t* gc, uint8_t* uc, int Cp,
                          uint32_t* gs, uint32_t* us, long long Rp,
                          hipStream_t st);
hipError_t launch_b8_swiglu_bwd(int dtype, int vec, const void* dh, long long ldh,
                          const uint8_t* gc, const uint8_t* uc, int Cp,
                          const uint32_t* gs, const uint32_t* us,
                          long long Rp, long long R, int C, void* dg,
                          void* du, hipStream_t st);
hipError_t launch_b8_rms_fwd(int dtype, int vec, const void* x, long long ldx,
                       const float* w, long long R, int C, float eps, void* y,
                       float* inv, uint8_t* codes, int Cp, uint32_t* scales,
                       long long Rp, hipStream_t st);
int b8_rms_bwd_partials(long long R, int C);
hipError_t launch_b8_rms_bwd(int dtype, int vec, const void* dy, long long ldy,
                       const uint8_t* codes, int Cp, const uint32_t* scales,
                       long long Rp, const float* w, const float* inv,
                       long long R, int C, void* dx, float* partials,
                       float* dw, hipStream_t st);
// bytes of workspace that the product wants (-1: too large a product for a
// launch), and the product
long long b8_gemm_workspace(const b8::GemmArgs* args);
hipError_t launch_b8_gemm(const b8::GemmArgs* args, float* workspace,
                    hipStream_t st);
// the same with x in bf16, packed on the way, if that is the better choice
bool b8_packs_on_the_way(const b8::GemmArgs* args);
hipError_t launch_b8_gemm_bf16(const b8::GemmArgs* args, const void* x,
                         long long ldx, int K, hipStream_t st);
}
