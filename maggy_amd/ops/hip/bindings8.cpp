// pybind11 bindings of the 8-bit block operators (block8.hip, gemm8.hip).
//
// Everything that the kernels assume is checked here: device, type, shape,
// and the strides and alignment that choose the 16-byte loads.  Matrices
// come with any row stride; the last axis is made contiguous if it is not.
// Outputs and workspaces come from torch's allocator, on the tensors' own
// device and the current stream of that device.
#include <torch/extension.h>
#include <ATen/cuda/CUDAContext.h>
#include <c10/cuda/CUDAGuard.h>
#include <torch/csrc/autograd/functions/accumulate_grad.h>

#include "block8_api.h"

namespace {

using torch::Tensor;
using c10::cuda::CUDAGuard;

int64_t up(int64_t n, int64_t to) { return (n + to - 1) / to * to; }

hipStream_t stream_of(const Tensor& t) {
  return at::cuda::getCurrentCUDAStream(t.get_device()).stream();
}

// outputs come uninitialised: a launch that was refused must not pass
void launched(const char* name, hipError_t e) {
  TORCH_CHECK(e == hipSuccess, name, ": the GPU refused the launch: ",
              hipGetErrorString(e));
}

int type_of(const Tensor& t, const char* name) {
  if (t.scalar_type() == torch::kBFloat16) return 0;
  if (t.scalar_type() == torch::kFloat16) return 1;
  TORCH_CHECK(t.scalar_type() == torch::kFloat32, name,
              " must be bfloat16, float16 or float32, got ", t.scalar_type());
  return 2;
}

// a 2-D matrix on the GPU whose columns are contiguous
Tensor matrix(const Tensor& t, const char* name) {
  if (t.is_neg()) return matrix(t.resolve_neg(), name);
  TORCH_CHECK(t.is_cuda(), name, " must be a GPU tensor");
  TORCH_CHECK(t.dim() == 2, name, " must be 2-D, got ", t.dim(), "-D");
  type_of(t, name);
  TORCH_CHECK(t.size(1) >= 1, name, " has no columns");
  TORCH_CHECK(t.size(0) < (int64_t)1 << 31 && t.size(1) < (int64_t)1 << 30,
              name, " is too large");
  if (t.size(1) > 1 && t.stride(1) != 1) return t.contiguous();
  return t;
}

// whether rows of t can be read in groups of 8 by 16-byte loads
bool vec8(const Tensor& t) {
  return t.size(1) % 8 == 0 && (t.size(0) <= 1 || t.stride(0) % 8 == 0) &&
         (uintptr_t)t.data_ptr() % 16 == 0;
}

// rows of one element or none may carry any stride
int64_t ld(const Tensor& t) { return t.size(0) > 1 ? t.stride(0) : 0; }

void same_device(const Tensor& a, const Tensor& b, const char* name) {
  TORCH_CHECK(a.device() == b.device(), name, " is on ", b.device(),
              ", expected ", a.device());
}

struct Packed {
  Tensor codes, scales;  // [Cp / 128][rows][128], [Q][Rp][4]
  uint8_t* c() const { return codes.data_ptr<uint8_t>(); }
  uint32_t* s() const { return (uint32_t*)scales.data_ptr<uint8_t>(); }
  int64_t rows() const { return codes.size(1); }
  int64_t Cp() const { return codes.size(0) * 128; }
  int64_t Rp() const { return scales.size(1); }
};

Packed new_packed(int64_t rows, int64_t C, const Tensor& like) {
  const auto o = like.options().dtype(torch::kUInt8).requires_grad(false);
  const int64_t Cp = up(C, 128);
  return {torch::empty({Cp / 128, rows, 128}, o),
          torch::empty({(Cp + 511) / 512, up(rows, 256), 4}, o)};
}

Packed packed(const Tensor& codes, const Tensor& scales, const char* name) {
  TORCH_CHECK(codes.is_cuda() && codes.scalar_type() == torch::kUInt8 &&
                  codes.dim() == 3 && codes.is_contiguous() &&
                  codes.size(0) >= 1 && codes.size(2) == 128,
              name, ": codes must be contiguous uint8 [n][rows][128]");
  TORCH_CHECK(scales.scalar_type() == torch::kUInt8 && scales.dim() == 3 &&
                  scales.is_contiguous() &&
                  scales.size(0) == (codes.size(0) + 3) / 4 &&
                  scales.size(1) == up(codes.size(1), 256) &&
                  scales.size(2) == 4,
              name, ": scales do not fit the codes");
  same_device(codes, scales, name);
  return {codes, scales};
}

Packed pack_rows(const Tensor& x) {
  Packed p = new_packed(x.size(0), x.size(1), x);
  if (x.size(0))
    launched("pack8",
             launch_b8_pack(type_of(x, "x"), vec8(x), x.data_ptr(), ld(x),
                            x.size(0), (int)x.size(1), p.c(), (int)p.Cp(),
                            p.s(), p.Rp(), stream_of(x)));
  return p;
}

std::vector<Tensor> pack8(Tensor x) {
  x = matrix(x, "x");
  const CUDAGuard guard(x.device());
  const Packed p = pack_rows(x);
  return {p.codes, p.scales};
}

Tensor unpack8(Tensor codes, Tensor scales, int64_t C,
               torch::ScalarType dtype) {
  const Packed p = packed(codes, scales, "unpack8");
  TORCH_CHECK(C >= 1 && up(C, 128) == p.Cp(), "unpack8: ", C,
              " columns do not fit the codes");
  const CUDAGuard guard(codes.device());
  const int64_t R = p.rows();
  Tensor out = torch::empty({R, C}, codes.options().dtype(dtype));
  if (R)
    launched("unpack8",
             launch_b8_unpack(type_of(out, "out"), C % 8 == 0, p.c(),
                              (int)p.Cp(), p.s(), p.Rp(), R, (int)C,
                              out.data_ptr(), stream_of(codes)));
  return out;
}

// A packed matrix in memory that a tensor somewhere owns
struct Mat8 {
  uint8_t* c = nullptr;
  uint32_t* s = nullptr;
  int64_t rows = 0, Cp = 0, Rp = 0;
  int64_t code_bytes() const { return up(rows * Cp, 256); }
  int64_t scale_bytes() const { return up((Cp + 511) / 512 * Rp * 4, 256); }
};
Mat8 mat8(const Packed& p) {
  return {p.c(), p.s(), p.rows(), p.Cp(), p.Rp()};
}

// Packed matrices, and a run of floats, in one tensor: the temporaries of a
// call, or what is kept for its backward pass, which lays them out again.
struct Arena {
  std::vector<Mat8*> mats;
  float* floats = nullptr;
  int64_t n_floats = 0;

  void want(Mat8* m, int64_t rows, int64_t C) {
    *m = Mat8{nullptr, nullptr, rows, up(C, 128), up(rows, 256)};
    mats.push_back(m);
  }
  int64_t bytes() const {
    int64_t n = 4 * n_floats;
    for (const Mat8* m : mats) n += m->code_bytes() + m->scale_bytes();
    return n;
  }
  void lay_out(const Tensor& space, const char* name) {
    TORCH_CHECK(space.is_cuda() && space.is_contiguous() &&
                    space.scalar_type() == torch::kUInt8 &&
                    space.numel() == bytes(),
                name, ": the gradient does not fit what was kept");
    uint8_t* at = space.data_ptr<uint8_t>();
    for (Mat8* m : mats) {
      m->c = at;
      m->s = (uint32_t*)(at + m->code_bytes());
      at += m->code_bytes() + m->scale_bytes();
    }
    floats = (float*)at;
  }
  Tensor take(const Tensor& like) {
    Tensor space = torch::empty(
        {bytes()}, like.options().dtype(torch::kUInt8).requires_grad(false));
    lay_out(space, "");
    return space;
  }
};

// ------------------------------------------------------------------ swiglu
// h, then with keep what the backward pass reads
std::vector<Tensor> swiglu8_fwd(Tensor g, Tensor u, bool keep) {
  g = matrix(g, "g");
  u = matrix(u, "u");
  TORCH_CHECK(g.sizes() == u.sizes() && g.scalar_type() == u.scalar_type(),
              "swiglu8: g and u must agree in shape and type");
  same_device(g, u, "u");
  const CUDAGuard guard(g.device());
  const int64_t R = g.size(0), C = g.size(1);
  std::vector<Tensor> out{torch::empty({R, C},
                                       g.options().requires_grad(false))};
  Mat8 mg, mu;
  if (keep) {
    Arena arena;
    arena.want(&mg, R, C);
    arena.want(&mu, R, C);
    out.push_back(arena.take(g));
  }
  if (R)
    launched("swiglu8",
             launch_b8_swiglu_fwd(type_of(g, "g"), vec8(g) && vec8(u),
                                  g.data_ptr(), ld(g), u.data_ptr(), ld(u), R,
                                  (int)C, out[0].data_ptr(), mg.c, mu.c,
                                  (int)up(C, 128), mg.s, mu.s, mg.Rp,
                                  stream_of(g)));
  return out;
}

std::vector<Tensor> swiglu8_bwd(Tensor dh, const Tensor& kept) {
  dh = matrix(dh, "dh");
  const int64_t R = dh.size(0), C = dh.size(1);
  Mat8 g, u;
  Arena arena;
  arena.want(&g, R, C);
  arena.want(&u, R, C);
  arena.lay_out(kept, "swiglu8");
  same_device(dh, kept, "g");
  const CUDAGuard guard(dh.device());
  const auto o = dh.options().requires_grad(false);
  Tensor dg = torch::empty({R, C}, o), du = torch::empty({R, C}, o);
  if (R)
    launched("swiglu8",
             launch_b8_swiglu_bwd(type_of(dh, "dh"), vec8(dh), dh.data_ptr(),
                                  ld(dh), g.c, u.c, (int)g.Cp, g.s, u.s, g.Rp,
                                  R, (int)C, dg.data_ptr(), du.data_ptr(),
                                  stream_of(dh)));
  return {dg, du};
}

// ----------------------------------------------------------------- RMSNorm
constexpr int64_t kRmsMost = 16384;  // columns that rms_fwd/rms_bwd hold

void check_rms_weight(const Tensor& x, const Tensor& w) {
  TORCH_CHECK(w.dim() == 1 && w.size(0) == x.size(1) && w.is_contiguous() &&
                  w.scalar_type() == torch::kFloat32,
              "rms_norm8: weight must be contiguous float32 [", x.size(1),
              "]");
  same_device(x, w, "weight");
}

// y, then with keep what the backward pass reads: x and a float a row
std::vector<Tensor> rms8_fwd(Tensor x, Tensor w, double eps, bool keep) {
  x = matrix(x, "x");
  const int64_t R = x.size(0), C = x.size(1);
  TORCH_CHECK(C <= kRmsMost, "rms_norm8: at most ", kRmsMost,
              " columns, got ", C);
  check_rms_weight(x, w);
  const CUDAGuard guard(x.device());
  std::vector<Tensor> out{torch::empty({R, C},
                                       x.options().requires_grad(false))};
  Mat8 m;
  Arena arena;
  if (keep) {
    arena.want(&m, R, C);
    arena.n_floats = R;
    out.push_back(arena.take(x));
  }
  if (R)
    launched("rms_norm8",
             launch_b8_rms_fwd(type_of(x, "x"),
                               vec8(x) && (uintptr_t)w.data_ptr() % 16 == 0,
                               x.data_ptr(), ld(x), w.data_ptr<float>(), R,
                               (int)C, (float)eps, out[0].data_ptr(),
                               arena.floats, m.c, (int)up(C, 128), m.s, m.Rp,
                               stream_of(x)));
  return out;
}

std::vector<c10::optional<Tensor>> rms8_bwd(Tensor dy, const Tensor& kept,
                                            const Tensor& w, bool need_dx,
                                            bool need_dw) {
  dy = matrix(dy, "dy");
  const int64_t R = dy.size(0), C = dy.size(1);
  Mat8 x;
  Arena arena;
  arena.want(&x, R, C);
  arena.n_floats = R;
  arena.lay_out(kept, "rms_norm8");
  check_rms_weight(dy, w);
  same_device(dy, kept, "x");
  const CUDAGuard guard(dy.device());
  const auto f32 = dy.options().dtype(torch::kFloat32).requires_grad(false);
  c10::optional<Tensor> dx, dw;
  Tensor partials;
  if (need_dx)
    dx = torch::empty({R, C}, dy.options().requires_grad(false));
  if (need_dw) {
    if (R == 0) {
      dw = torch::zeros({C}, f32);
    } else {
      dw = torch::empty({C}, f32);
      partials = torch::empty({b8_rms_bwd_partials(R, (int)C), C}, f32);
    }
  }
  if (R && (need_dx || need_dw))
    launched("rms_norm8",
             launch_b8_rms_bwd(type_of(dy, "dy"),
                               vec8(dy) && (uintptr_t)w.data_ptr() % 16 == 0,
                               dy.data_ptr(), ld(dy), x.c, (int)x.Cp, x.s,
                               x.Rp, w.data_ptr<float>(), arena.floats, R,
                               (int)C, dx ? dx->data_ptr() : nullptr,
                               need_dw ? partials.data_ptr<float>() : nullptr,
                               need_dw ? dw->data_ptr<float>() : nullptr,
                               stream_of(dy)));
  return {dx, dw};
}

// ----------------------------------------------------------------- linear8
// the first row of each weight when they are stacked, and the total
std::vector<int64_t> firsts(const std::vector<int64_t>& counts) {
  std::vector<int64_t> f{0};
  for (int64_t n : counts) f.push_back(f.back() + up(n, 128));
  return f;
}

void check_counts(const std::vector<int64_t>& counts) {
  TORCH_CHECK(counts.size() >= 1 && counts.size() <= b8::kMaxParts,
              "linear8 takes 1 to ", b8::kMaxParts, " weights, got ",
              counts.size());
}

// The packing that a call needs, in one launch.  A job's outputs start at
// (row_r0, row_c0) of rows and at (col_r0, col_c0) of cols.
struct Jobs {
  b8::TileJobs jobs{};

  b8::TileJob& add(b8::TileKind kind, const Mat8* rows, int64_t row_r0,
                   int64_t row_c0, const Mat8* cols, int64_t col_r0,
                   int64_t col_c0) {
    const bool by_rows = kind == b8::kTileBoth || kind == b8::kTileRows ||
                         kind == b8::kTileOneRows;
    TORCH_CHECK(by_rows == (rows != nullptr) &&
                    (kind == b8::kTileBoth || !by_rows) == (cols != nullptr),
                "linear8: outputs do not match the job");
    TORCH_CHECK(jobs.count < b8::kMaxJobs, "linear8: too many matrices");
    b8::TileJob& a = jobs.job[jobs.count++];
    a.kind = kind;
    if (rows) {
      a.row_codes = rows->c;
      a.row_scales = (uint8_t*)rows->s;
      a.row_n = rows->rows;
      a.row_sp = rows->Rp;
      a.row_r0 = row_r0;
      a.row_c0 = row_c0;
    }
    if (cols) {
      a.col_codes = cols->c;
      a.col_scales = (uint8_t*)cols->s;
      a.col_n = cols->rows;
      a.col_sp = cols->Rp;
      a.col_r0 = col_r0;
      a.col_c0 = col_c0;
    }
    return a;
  }
  void plain(const Tensor& t, b8::TileJob& a) {
    a.x = t.data_ptr();
    a.ldx = ld(t);
    a.R = (int)t.size(0);
    a.C = (int)t.size(1);
    a.dtype = type_of(t, "matrix");
    a.vec = vec8(t);
    const bool weight =
        a.kind == b8::kTileOneRows || a.kind == b8::kTileOneCols;
    TORCH_CHECK(a.dtype == 0 || (weight && a.dtype == 2),
                "linear8: no packing of ", t.scalar_type());
  }
  void packed(const Mat8& m, b8::TileJob& a) {
    a.x = m.c;
    a.xs = m.s;
    a.ldx = m.rows;
    a.xsp = m.Rp;
    a.R = (int)m.rows;
    a.C = (int)m.Cp;
  }
  void run(hipStream_t st) {
    const long long blocks = b8_tile_blocks(&jobs);
    TORCH_CHECK(blocks >= 0, "linear8: matrix is too large");
    if (blocks) launched("linear8", launch_b8_tiles(&jobs, blocks, st));
  }
};

// the weights' rows one below the other
void stack_weights(Jobs& jobs, const std::vector<Tensor>& ws,
                   const std::vector<int64_t>& first, const Mat8& to) {
  for (size_t i = 0; i < ws.size(); ++i)
    jobs.plain(ws[i], jobs.add(b8::kTileOneRows, &to, first[i], 0, nullptr, 0,
                               0));
}

std::vector<Tensor> weights_of(const std::vector<Tensor>& weights,
                               std::vector<int64_t>* counts) {
  std::vector<Tensor> ws;
  for (const Tensor& w : weights) {
    ws.push_back(matrix(w, "weight"));
    TORCH_CHECK(w.size(0) >= 1, "weight has no rows");
    TORCH_CHECK(w.size(1) == weights[0].size(1) &&
                    w.scalar_type() == weights[0].scalar_type(),
                "linear8: weights must agree in columns and type");
    TORCH_CHECK(w.scalar_type() != torch::kFloat16,
                "linear8: weights must be bfloat16 or float32");
    same_device(weights[0], w, "weight");
    counts->push_back(w.size(0));
  }
  check_counts(*counts);
  return ws;
}

// the product of packed w with x, packed (M rows) or, for a few rows, plain
// bf16 that the kernel packs on the way; like: a tensor of their device.  The
// outputs are the parts of w that counts tells, or with width > 0 those of x,
// of width columns each.
b8::GemmArgs gemm_args(const Mat8& w, int64_t M,
                       const std::vector<int64_t>& counts, int64_t width,
                       torch::ScalarType dtype, const Tensor& like,
                       std::vector<Tensor>* out) {
  const auto first = firsts(counts);
  const int64_t N = width ? w.rows : std::min(first.back(), w.rows);
  TORCH_CHECK(width <= w.rows && (!width || M == first[counts.size() - 1] +
                                                    counts.back()),
              "linear8: outputs do not match the product");
  TORCH_CHECK(M < (int64_t)1 << 30 && first.back() < (int64_t)1 << 30 &&
                  N < (int64_t)1 << 30,
              "linear8: too many rows");
  // the kernel reaches a matrix's scales by 32-bit offsets
  const int64_t quads = (w.Cp + 511) / 512;
  TORCH_CHECK(quads * w.Rp * 4 < (int64_t)1 << 31 &&
                  quads * up(M, 256) * 4 < (int64_t)1 << 31,
              "linear8: matrix is too large");
  b8::GemmArgs a{};
  a.w = w.c;
  a.ws = w.s;
  a.wn = w.rows;
  a.wsp = w.Rp;
  a.M = (int)M;
  a.N = (int)N;
  a.KT = (int)(w.Cp / 128);
  a.parts = (int)counts.size();
  a.by_rows = width > 0;
  a.width = (int)width;
  a.f32 = dtype == torch::kFloat32;
  const auto o = like.options().dtype(dtype).requires_grad(false);
  for (size_t i = 0; i < counts.size(); ++i) {
    out->push_back(width ? torch::empty({counts[i], width}, o)
                         : torch::empty({M, counts[i]}, o));
    a.out[i] = (*out)[i].data_ptr();
    a.first[i] = (int)first[i];
    a.count[i] = (int)counts[i];
  }
  return a;
}

// width: the outputs are parts of x (gemm_args), gradients that are wanted
// later; otherwise the next kernels are going to read them
std::vector<Tensor> product(const Mat8& x, const Mat8& w, int64_t M,
                            const std::vector<int64_t>& counts,
                            torch::ScalarType dtype, const Tensor& like,
                            int64_t width = 0) {
  TORCH_CHECK(x.Cp == w.Cp && M <= x.rows, "linear8: columns do not match");
  std::vector<Tensor> out;
  b8::GemmArgs a = gemm_args(w, M, counts, width, dtype, like, &out);
  a.x = x.c;
  a.xs = x.s;
  a.xn = x.rows;
  a.xsp = x.Rp;
  a.stream = 2 * M * a.N >= (width ? b8::kStreamOnce : b8::kStreamResult);
  if (M) {
    const long long bytes = b8_gemm_workspace(&a);
    TORCH_CHECK(bytes >= 0, "linear8: matrix is too large");
    Tensor space;
    if (bytes)
      space = torch::empty({bytes}, like.options()
                                        .dtype(torch::kUInt8)
                                        .requires_grad(false));
    launched("linear8",
             launch_b8_gemm(&a, bytes ? (float*)space.data_ptr() : nullptr,
                            stream_of(like)));
  }
  return out;
}

void check_bf16(const Tensor& x) {
  TORCH_CHECK(x.scalar_type() == torch::kBFloat16,
              "linear8 runs in bfloat16 on the GPU, got ", x.scalar_type());
}

// the stacked weights by their rows
std::vector<Tensor> pack8_weights(std::vector<Tensor> weights) {
  std::vector<int64_t> counts;
  const auto ws = weights_of(weights, &counts);
  const CUDAGuard guard(ws[0].device());
  const auto first = firsts(counts);
  const Packed p = new_packed(first.back(), ws[0].size(1), ws[0]);
  Jobs jobs;
  stack_weights(jobs, ws, first, mat8(p));
  jobs.run(stream_of(ws[0]));
  return {p.codes, p.scales};
}

// outputs, then with keep the packed x
std::vector<Tensor> linear8_fwd(Tensor x, std::vector<Tensor> weights,
                                bool keep) {
  check_bf16(x);
  x = matrix(x, "x");
  std::vector<int64_t> counts;
  const auto ws = weights_of(weights, &counts);
  TORCH_CHECK(ws[0].size(1) == x.size(1), "linear8: x has ", x.size(1),
              " columns, the weights ", ws[0].size(1));
  same_device(x, ws[0], "weight");
  const CUDAGuard guard(x.device());
  const auto first = firsts(counts);
  Mat8 held, w;
  Arena kept, arena;
  (keep ? kept : arena).want(&held, x.size(0), x.size(1));
  arena.want(&w, first.back(), x.size(1));
  Tensor kept_space;
  if (keep) kept_space = kept.take(x);
  const Tensor space = arena.take(x);
  Jobs jobs;
  if (x.size(0))
    jobs.plain(x, jobs.add(b8::kTileRows, &held, 0, 0, nullptr, 0, 0));
  stack_weights(jobs, ws, first, w);
  jobs.run(stream_of(x));
  auto out = product(held, w, x.size(0), counts, torch::kBFloat16, x);
  if (keep) out.push_back(kept_space);
  return out;
}

std::vector<Tensor> linear8_packed(Tensor x, Tensor wcodes, Tensor wscales,
                                   std::vector<int64_t> counts, int64_t K) {
  check_bf16(x);
  x = matrix(x, "x");
  check_counts(counts);
  const Packed w = packed(wcodes, wscales, "linear8");
  TORCH_CHECK(firsts(counts).back() == w.rows() &&
                  up(K, 128) == w.Cp(),
              "linear8: the packed weights do not have these shapes");
  TORCH_CHECK(x.size(1) == K, "linear8: x has ", x.size(1),
              " columns, the weights ", K);
  same_device(x, wcodes, "weight");
  const CUDAGuard guard(x.device());
  const int64_t M = x.size(0);
  // packed weights are shared between streams: their memory is not to be
  // used again before this call's kernels have read it
  for (const Tensor* t : {&wcodes, &wscales})
    c10::cuda::CUDACachingAllocator::recordStream(
        t->storage().data_ptr(), at::cuda::getCurrentCUDAStream());
  if (M >= 1 && vec8(x)) {
    b8::GemmArgs a{};
    a.M = (int)std::min(M, (int64_t)1 << 30);
    a.N = (int)std::min(w.rows(), (int64_t)1 << 30);
    a.KT = (int)(w.Cp() / 128);
    if (b8_packs_on_the_way(&a)) {
      std::vector<Tensor> out;
      a = gemm_args(mat8(w), M, counts, 0, torch::kBFloat16, x, &out);
      launched("linear8",
               launch_b8_gemm_bf16(&a, x.data_ptr(), ld(x), (int)K,
                                   stream_of(x)));
      return out;
    }
  }
  return product(mat8(pack_rows(x)), mat8(w), M, counts, torch::kBFloat16, x);
}

// dx and one dw a weight; dx empty or no dw where they are not asked for
std::vector<Tensor> linear8_bwd(std::vector<Tensor> dys, const Tensor& kept,
                                std::vector<Tensor> weights, bool need_dx,
                                bool need_dw) {
  std::vector<int64_t> counts;
  const auto ws = weights_of(weights, &counts);
  TORCH_CHECK(dys.size() == ws.size(), "linear8: one gradient an output");
  const auto first = firsts(counts);
  const int64_t K = ws[0].size(1), M = dys[0].size(0), N = first.back();
  for (size_t i = 0; i < dys.size(); ++i) {
    check_bf16(dys[i]);
    dys[i] = matrix(dys[i], "dy");
    TORCH_CHECK(dys[i].size(0) == M && dys[i].size(1) == counts[i],
                "linear8: gradient ", i, " has the wrong shape");
    same_device(ws[0], dys[i], "dy");
  }
  const CUDAGuard guard(ws[0].device());
  const auto o = ws[0].options().requires_grad(false);
  std::vector<Tensor> out(1);
  if (M == 0) {
    if (need_dx) out[0] = torch::empty({0, K}, dys[0].options());
    if (need_dw)
      for (int64_t n : counts) out.push_back(torch::zeros({n, K}, o));
    return out;
  }
  // dY by rows for dX and by columns for dW; W^T [K][N], each weight's
  // columns side by side; x^T from the codes that were kept
  Mat8 rows, cols, wt, xt, x;
  Arena arena;
  if (need_dx) {
    arena.want(&rows, M, N);
    arena.want(&wt, up(K, 128), N);
  }
  if (need_dw) {
    TORCH_CHECK(kept.defined(), "linear8: nothing was kept of x");
    Arena before;
    before.want(&x, M, K);
    before.lay_out(kept, "linear8");
    same_device(ws[0], kept, "x");
    arena.want(&cols, N, M);
    arena.want(&xt, x.Cp, M);
  }
  if (!need_dx && !need_dw) return out;
  const Tensor space = arena.take(ws[0]);
  Jobs jobs;
  for (size_t i = 0; i < dys.size(); ++i)
    jobs.plain(dys[i],
               jobs.add(need_dx && need_dw ? b8::kTileBoth
                        : need_dx          ? b8::kTileRows
                                           : b8::kTileCols,
                        need_dx ? &rows : nullptr, 0, first[i],
                        need_dw ? &cols : nullptr, first[i], 0));
  if (need_dx)
    for (size_t i = 0; i < ws.size(); ++i)
      jobs.plain(ws[i], jobs.add(b8::kTileOneCols, nullptr, 0, 0, &wt, 0,
                                 first[i]));
  if (need_dw)
    jobs.packed(x, jobs.add(b8::kTileFrom8, nullptr, 0, 0, &xt, 0, 0));
  jobs.run(stream_of(ws[0]));
  if (need_dx)
    out[0] = product(rows, wt, M, {K}, torch::kBFloat16, ws[0])[0];
  if (need_dw) {
    // all weights' dW in one product, a tensor each
    for (Tensor& dw : product(cols, xt, first[counts.size() - 1] +
                                            counts.back(),
                              counts, ws[0].scalar_type(), ws[0], K))
      out.push_back(std::move(dw));
  }
  return out;
}

// ---------------------------------------------------------------- autograd
// The graph's nodes are C++ too: a Python node costs tens of microseconds a
// pass, more than the kernels of a small batch.
using torch::autograd::AutogradContext;
using torch::autograd::variable_list;

// [..., C] as a matrix, and back
Tensor as_rows(const Tensor& t) {
  return t.dim() == 2 ? t : t.reshape({-1, t.size(-1)});
}
Tensor as_shape(const Tensor& rows, at::IntArrayRef lead) {
  if (lead.size() == 1) return rows;
  auto shape = lead.vec();
  shape.push_back(rows.size(1));
  return rows.view(shape);
}

bool wants_grad(std::initializer_list<const Tensor*> ts) {
  if (!at::GradMode::is_enabled()) return false;
  for (const Tensor* t : ts)
    if (t->requires_grad()) return true;
  return false;
}

// a tangent would be lost without a word
void no_forward_mode(const char* name, at::ArrayRef<Tensor> ts) {
  for (const Tensor& t : ts)
    TORCH_CHECK(!t.defined() || !t._fw_grad(0).defined(), name,
                " has no forward-mode derivative");
}

void no_second_derivative(const char* name) {
  TORCH_CHECK(!at::GradMode::is_enabled(), name,
              " has no second derivative: backward cannot create a graph");
}

// A leaf whose eager graph lives accumulates on that graph's stream.  If that
// is the default stream, capturing this pass would end in the runtime: no
// capture can wait for it.  Between the leaf and this node there may be views
// and conversions, a call's own (leading axes, a norm's weight in bf16) among
// them: whatever has one input.
void no_eager_leaves(const char* name) {
  if (at::cuda::currentStreamCaptureStatusMayInitCtx() ==
      c10::cuda::CaptureStatus::None)
    return;
  const auto node = torch::autograd::get_current_node();
  if (!node) return;
  for (const auto& edge : node->next_edges()) {
    torch::autograd::Node* at = edge.function.get();
    while (at && at->next_edges().size() == 1)
      at = at->next_edge(0).function.get();
    if (!dynamic_cast<torch::autograd::AccumulateGrad*>(at)) continue;
    const auto stream = at->stream();
    TORCH_CHECK(!stream || stream->id() != 0, name,
                ": a backward pass cannot be captured while an eager graph "
                "of the same leaf, made on the default stream, lives");
  }
}

struct SwiGLU8 : torch::autograd::Function<SwiGLU8> {
  static Tensor forward(AutogradContext* ctx, Tensor g, Tensor u) {
    auto out = swiglu8_fwd(g, u, true);
    ctx->save_for_backward({out[1]});
    return out[0];
  }
  static variable_list backward(AutogradContext* ctx, variable_list dh) {
    no_second_derivative("swiglu8");
    no_eager_leaves("swiglu8");
    const auto k = ctx->get_saved_variables();
    return swiglu8_bwd(dh[0], k[0]);
  }
};

Tensor swiglu8(Tensor g, Tensor u) {
  no_forward_mode("swiglu8", {g, u});
  const auto lead = g.sizes().slice(0, g.dim() - 1).vec();
  g = as_rows(g);
  u = as_rows(u);
  return as_shape(wants_grad({&g, &u}) ? SwiGLU8::apply(g, u)
                                       : swiglu8_fwd(g, u, false)[0],
                  lead);
}

struct RMSNorm8 : torch::autograd::Function<RMSNorm8> {
  static Tensor forward(AutogradContext* ctx, Tensor x, Tensor w,
                        double eps) {
    auto out = rms8_fwd(x, w, eps, true);
    ctx->save_for_backward({out[1], w});
    return out[0];
  }
  static variable_list backward(AutogradContext* ctx, variable_list dy) {
    no_second_derivative("rms_norm8");
    no_eager_leaves("rms_norm8");
    const auto k = ctx->get_saved_variables();
    auto d = rms8_bwd(dy[0], k[0], k[1], ctx->needs_input_grad(0),
                      ctx->needs_input_grad(1));
    return {d[0].value_or(Tensor()), d[1].value_or(Tensor()), Tensor()};
  }
};

Tensor rms_norm8(Tensor x, Tensor w, double eps) {
  no_forward_mode("rms_norm8", {x, w});
  const auto lead = x.sizes().slice(0, x.dim() - 1).vec();
  x = as_rows(x);
  w = w.resolve_neg();
  return as_shape(wants_grad({&x, &w}) ? RMSNorm8::apply(x, w, eps)
                                       : rms8_fwd(x, w, eps, false)[0],
                  lead);
}

static_assert(b8::kMaxParts == 4);
struct Linear8 : torch::autograd::Function<Linear8> {
  using Maybe = c10::optional<Tensor>;
  static variable_list forward(AutogradContext* ctx, Tensor x, Tensor w0,
                               Maybe w1, Maybe w2, Maybe w3) {
    variable_list weights{w0};
    for (const Maybe& w : {w1, w2, w3})
      if (w) weights.push_back(*w);
    // dX does not read x
    bool dw = false;
    for (const Tensor& w : weights) dw = dw || w.requires_grad();
    auto out = linear8_fwd(x, weights, dw);
    variable_list kept(weights);
    kept.push_back(dw ? out[weights.size()] : Tensor());
    ctx->save_for_backward(kept);
    out.resize(weights.size());
    return out;
  }
  static variable_list backward(AutogradContext* ctx, variable_list dys) {
    no_second_derivative("linear8");
    no_eager_leaves("linear8");
    auto kept = ctx->get_saved_variables();
    const size_t n = kept.size() - 1;
    const Tensor x = kept[n];
    kept.resize(n);
    bool need_dw = false;
    for (size_t i = 0; i < n; ++i)
      need_dw = need_dw || ctx->needs_input_grad(1 + i);
    auto d = linear8_bwd(dys, x, kept, ctx->needs_input_grad(0), need_dw);
    d.resize(1 + b8::kMaxParts);
    for (size_t i = 0; i < n; ++i)
      if (!ctx->needs_input_grad(1 + i)) d[1 + i] = Tensor();
    return d;
  }
};

std::vector<Tensor> linear8(Tensor x, std::vector<Tensor> weights) {
  no_forward_mode("linear8", x);
  no_forward_mode("linear8", weights);
  const auto lead = x.sizes().slice(0, x.dim() - 1).vec();
  x = as_rows(x);
  bool grad = wants_grad({&x});
  for (const Tensor& w : weights) grad = grad || wants_grad({&w});
  std::vector<Tensor> out;
  if (grad) {
    check_counts(std::vector<int64_t>(weights.size()));
    const auto at = [&](size_t i) {
      return i < weights.size() ? Linear8::Maybe(weights[i]) : c10::nullopt;
    };
    out = Linear8::apply(x, weights[0], at(1), at(2), at(3));
  } else {
    out = linear8_fwd(x, weights, false);
  }
  for (Tensor& y : out) y = as_shape(y, lead);
  return out;
}

std::vector<Tensor> linear8_on_packed(Tensor x, Tensor codes, Tensor scales,
                                      std::vector<int64_t> counts,
                                      int64_t K) {
  no_forward_mode("linear8", x);
  const auto lead = x.sizes().slice(0, x.dim() - 1).vec();
  auto out = linear8_packed(as_rows(x), codes, scales, counts, K);
  for (Tensor& y : out) y = as_shape(y, lead);
  return out;
}

}  // namespace

void bind_block8(pybind11::module_& m) {
  using release = pybind11::call_guard<pybind11::gil_scoped_release>;
  m.def("pack8", &pack8, "matrix -> 8-bit block codes and scales",
        release());
  m.def("unpack8", &unpack8, "8-bit block codes and scales -> matrix",
        release());
  m.def("swiglu8", &swiglu8, "silu(g)*u, differentiable, g and u kept in 8 "
        "bits", release());
  m.def("rms_norm8", &rms_norm8, "RMSNorm, differentiable, x kept in 8 bits",
        release());
  m.def("pack8_weights", &pack8_weights, "stacked weights in 8 bits",
        release());
  m.def("linear8", &linear8, "x @ W^T of 8-bit operands, differentiable",
        release());
  m.def("linear8_packed", &linear8_on_packed, "x @ W^T on packed weights",
        release());
}
