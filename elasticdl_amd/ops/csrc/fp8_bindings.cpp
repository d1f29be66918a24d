// Bindings of the 8-bit dense layers (fp8_kernels.hip): argument checks,
// outputs and workspaces. A layer's forward and its backward are one call
// each, so that small layers do not pay for Python between the launches.

#include <torch/extension.h>

#include <c10/core/DeviceGuard.h>
#include <c10/hip/HIPStream.h>

#include <cstdint>
#include <limits>

#include "fp8_kernels.h"

extern "C" {
int edl_fp8_quantize(const edl_fp8_quant*, hipStream_t);
int edl_fp8_column_sums(const float*, int64_t, int64_t, void*, int,
                        hipStream_t);
int edl_fp8_gemm_splits(const edl_fp8_gemm*);
int edl_fp8_gemm_run(const edl_fp8_gemm*, hipStream_t);
int edl_fp8_few_rows(const edl_fp8_gemm*, const void*, int64_t, int, int, int,
                     hipStream_t);
}

namespace {

using torch::Tensor;
using OptTensor = c10::optional<Tensor>;

constexpr int64_t kFewRows = 16;

int64_t round_up(int64_t n, int64_t to) { return (n + to - 1) / to * to; }

hipStream_t stream_of(const Tensor& t) {
  return c10::hip::getCurrentHIPStream(t.device().index()).stream();
}

void launched(int rc, const char* what) {
  TORCH_CHECK(rc == 0, what, ": kernel launch failed with HIP error ", rc);
}

int type_code(torch::ScalarType t, const char* name) {
  switch (t) {
    case torch::kFloat32: return EDL_T_F32;
    case torch::kBFloat16: return EDL_T_BF16;
    case torch::kFloat16: return EDL_T_F16;
    default:
      TORCH_CHECK(false, name, " must be float32, bfloat16 or float16, not ",
                  t);
  }
}

bool aligned(const Tensor& t, int64_t row_stride) {
  return reinterpret_cast<uintptr_t>(t.data_ptr()) % 16 == 0 &&
         row_stride * t.element_size() % 16 == 0;
}

void check_matrix(const Tensor& t, const char* name) {
  TORCH_CHECK(t.is_cuda(), name, " must be on a GPU");
  TORCH_CHECK(t.dim() == 2, name, " must have two dimensions, not ", t.dim());
  // 2^24 columns: a tile's 256 rows of bytes stay within a 32-bit offset
  TORCH_CHECK(t.size(1) >= 1 && t.size(1) < (1 << 24) - 128, name,
              " must have between 1 and 2^24 - 129 columns, not ", t.size(1));
  TORCH_CHECK(t.size(0) < std::numeric_limits<int32_t>::max() - 256, name,
              " has too many rows: ", t.size(0));
}

// rows may be strided, neighbours in a row may not
Tensor row_major(const Tensor& t) {
  return t.size(1) == 1 || t.stride(1) == 1 ? t : t.contiguous();
}

Tensor new_bytes(const Tensor& like, int64_t r, int64_t c) {
  return torch::empty({r, c}, like.options()
                                  .dtype(torch::kUInt8)
                                  .requires_grad(false)
                                  .memory_format(c10::nullopt));
}

// [R, C] contracted over C: bytes and scales
struct Blocks {
  Tensor q, s;
};
Blocks new_blocks(const Tensor& like, int64_t r, int64_t c) {
  const int64_t cp = round_up(c, EDL_FP8_BLOCK);
  return {new_bytes(like, r, cp),
          new_bytes(like, cp / EDL_FP8_BLOCK, round_up(r, 256))};
}
void into_rows(edl_fp8_quant& a, const Blocks& b) {
  a.rows = b.q.data_ptr<uint8_t>();
  a.rows_scale = b.s.data_ptr<uint8_t>();
  a.rows_ld = b.q.size(1);
  a.rows_rp = b.s.size(1);
}
void into_cols(edl_fp8_quant& a, const Blocks& b) {
  a.cols = b.q.data_ptr<uint8_t>();
  a.cols_scale = b.s.data_ptr<uint8_t>();
  a.cols_ld = b.q.size(1);
  a.cols_rp = b.s.size(1);
}

edl_fp8_quant quant_of(const Tensor& x, const char* name) {
  edl_fp8_quant a = {};
  a.x = x.data_ptr();
  a.ld = x.size(0) > 1 ? x.stride(0) : x.size(1);
  a.R = x.size(0);
  a.C = x.size(1);
  a.type = type_code(x.scalar_type(), name);
  a.wide = aligned(x, a.ld);
  const int64_t tiles = round_up(a.R, EDL_FP8_BLOCK) / EDL_FP8_BLOCK *
                        (round_up(a.C, EDL_FP8_BLOCK) / EDL_FP8_BLOCK);
  TORCH_CHECK(tiles < std::numeric_limits<int32_t>::max(), name,
              " is too large");
  return a;
}

void check_blocks(const Tensor& q, const Tensor& s, int64_t rows,
                  int64_t contracted, const Tensor& with, const char* name) {
  TORCH_CHECK(q.is_cuda() && s.is_cuda() && q.device() == with.device() &&
                  s.device() == with.device(),
              name, " must be on ", with.device());
  TORCH_CHECK(q.scalar_type() == torch::kUInt8 &&
                  s.scalar_type() == torch::kUInt8 && q.is_contiguous() &&
                  s.is_contiguous() && q.dim() == 2 && s.dim() == 2,
              name, " must be bytes and scales of a quantised matrix");
  TORCH_CHECK(
      q.size(0) == rows && q.size(1) == round_up(contracted, EDL_FP8_BLOCK) &&
          s.size(0) == q.size(1) / EDL_FP8_BLOCK &&
          s.size(1) == round_up(rows, 256),
      name, " does not match: expected ", rows, " x ", contracted);
}

void check_bias(const OptTensor& bias, int64_t n, const Tensor& x) {
  if (!bias.has_value()) return;
  TORCH_CHECK(bias->device() == x.device(), "bias must be on ", x.device());
  TORCH_CHECK(bias->dim() == 1 && bias->size(0) == n && bias->is_contiguous(),
              "bias must be contiguous with ", n, " values");
  type_code(bias->scalar_type(), "bias");
}

// c [M, N] = act(a b^T + bias)
Tensor multiply(const Tensor& a, const Tensor& as, int64_t M, const Tensor& b,
                const Tensor& bs, int64_t N, const OptTensor& bias, int act,
                torch::ScalarType type, Tensor* mask) {
  Tensor c = torch::empty(
      {M, N}, a.options().dtype(type).requires_grad(false));
  edl_fp8_gemm g = {};
  g.a = a.data_ptr<uint8_t>();
  g.sa = as.data_ptr<uint8_t>();
  g.b = b.data_ptr<uint8_t>();
  g.sb = bs.data_ptr<uint8_t>();
  g.M = M;
  g.N = N;
  g.ld = a.size(1);
  g.a_rp = as.size(1);
  g.b_rp = bs.size(1);
  if (bias.has_value()) {
    g.bias = bias->data_ptr();
    g.bias_type = type_code(bias->scalar_type(), "bias");
  }
  g.act = act;
  g.c = c.data_ptr();
  g.c_type = type_code(type, "output");
  g.c_wide = aligned(c, N);
  if (mask) {
    *mask = new_bytes(a, M, round_up(N, 16) / 8);
    g.mask = mask->data_ptr<uint8_t>();
    g.mask_ld = mask->size(1);
  }
  g.splits = edl_fp8_gemm_splits(&g);
  g.part_ld = round_up(N, 16);
  Tensor part;
  if (g.splits > 1) {
    part = torch::empty({g.splits, M, g.part_ld},
                        a.options().dtype(torch::kFloat32));
    g.part = part.data_ptr<float>();
  }
  launched(edl_fp8_gemm_run(&g, stream_of(a)), "fp8 product");
  return c;
}

// (bytes, scales, bytes of the transpose, its scales); the latter two where
// `cols`. Blocks lie along each form's rows, or are 128 x 128 where `tile`.
std::vector<OptTensor> fp8_quantize(Tensor x, bool tile, bool rows,
                                    bool cols) {
  check_matrix(x, "x");
  TORCH_CHECK(x.size(0) < (1 << 24) - 128 || !cols,
              "x has too many rows to be transposed: ", x.size(0));
  TORCH_CHECK(rows || cols, "nothing asked for");
  c10::DeviceGuard guard(x.device());
  x = row_major(x);
  edl_fp8_quant a = quant_of(x, "x");
  a.tile = tile;
  std::vector<OptTensor> out(4);
  Blocks r, c;
  if (rows) {
    r = new_blocks(x, a.R, a.C);
    into_rows(a, r);
    out[0] = r.q;
    out[1] = r.s;
  }
  if (cols) {
    c = new_blocks(x, a.C, a.R);
    into_cols(a, c);
    out[2] = c.q;
    out[3] = c.s;
  }
  if (a.R > 0) launched(edl_fp8_quantize(&a, stream_of(x)), "fp8 quantise");
  return out;
}

void check_act(int64_t act) {
  TORCH_CHECK(act >= EDL_ACT_NONE && act <= EDL_ACT_SIGMOID,
              "unknown activation ", act);
}

// y = act(x w^T + bias) from x as it is; and what a backward pass multiplies
// from: x^T in 8 bits and its scales (keep_x), relu's bits (keep_mask).
std::vector<OptTensor> fp8_dense_fwd(Tensor x, Tensor wq, Tensor ws, int64_t n,
                                     OptTensor bias, int64_t act, bool keep_x,
                                     bool keep_mask) {
  check_matrix(x, "x");
  check_act(act);
  const int64_t m = x.size(0), k = x.size(1);
  TORCH_CHECK(m < (1 << 24) - 128 || !keep_x,
              "x has too many rows to be kept for a backward pass: ", m);
  check_blocks(wq, ws, n, k, x, "weight");
  check_bias(bias, n, x);
  c10::DeviceGuard guard(x.device());
  x = row_major(x);
  std::vector<OptTensor> out(4);
  const bool bits = keep_mask && act == EDL_ACT_RELU;
  if (m == 0) {
    out[0] = torch::empty({0, n}, x.options().requires_grad(false));
    if (keep_x) {
      Blocks c = new_blocks(x, k, 0);
      out[1] = c.q;
      out[2] = c.s;
    }
    if (bits) out[3] = new_bytes(x, 0, round_up(n, 16) / 8);
    return out;
  }
  edl_fp8_quant a = quant_of(x, "x");
  if (m <= kFewRows && !keep_x && !bits) {
    Tensor y = torch::empty({m, n}, x.options().requires_grad(false));
    edl_fp8_gemm g = {};
    g.b = wq.data_ptr<uint8_t>();
    g.sb = ws.data_ptr<uint8_t>();
    g.M = m;
    g.N = n;
    g.ld = wq.size(1);
    g.b_rp = ws.size(1);
    if (bias.has_value()) {
      g.bias = bias->data_ptr();
      g.bias_type = type_code(bias->scalar_type(), "bias");
    }
    g.act = (int)act;
    g.c = y.data_ptr();
    g.c_type = a.type;
    launched(edl_fp8_few_rows(&g, a.x, a.ld, (int)k, a.type, a.wide,
                              stream_of(x)),
             "fp8 product");
    out[0] = y;
    return out;
  }
  Blocks r = new_blocks(x, m, k);
  into_rows(a, r);
  if (keep_x) {
    Blocks c = new_blocks(x, k, m);
    into_cols(a, c);
    out[1] = c.q;
    out[2] = c.s;
  }
  launched(edl_fp8_quantize(&a, stream_of(x)), "fp8 quantise");
  Tensor mask;
  out[0] = multiply(r.q, r.s, m, wq, ws, n, bias, (int)act, x.scalar_type(),
                    bits ? &mask : nullptr);
  if (bits) out[3] = mask;
  return out;
}

// (dx, dw, db); each where it is asked for. wtq, wts: the weight transposed.
std::vector<OptTensor> fp8_dense_bwd(Tensor dy, int64_t act, OptTensor mask,
                                     OptTensor y, OptTensor wtq,
                                     OptTensor wts, OptTensor xtq,
                                     OptTensor xts, int64_t k, bool need_dx,
                                     bool need_dw, bool need_db,
                                     py::object dw_type, py::object db_type) {
  check_matrix(dy, "gradient");
  check_act(act);
  const int64_t m = dy.size(0), n = dy.size(1);
  TORCH_CHECK(m < (1 << 24) - 128, "gradient has too many rows: ", m);
  c10::DeviceGuard guard(dy.device());
  dy = row_major(dy);
  const auto wt = need_dw ? torch::python::detail::py_object_to_dtype(dw_type)
                          : torch::kFloat32;
  const auto bt = need_db ? torch::python::detail::py_object_to_dtype(db_type)
                          : torch::kFloat32;
  std::vector<OptTensor> out(3);
  auto opts = dy.options().requires_grad(false);
  if (m == 0) {
    if (need_dx) out[0] = torch::empty({0, k}, opts);
    if (need_dw) out[1] = torch::zeros({n, k}, opts.dtype(wt));
    if (need_db) out[2] = torch::zeros({n}, opts.dtype(bt));
    return out;
  }
  edl_fp8_quant a = quant_of(dy, "gradient");
  a.deriv = true;
  a.act = (int)act;
  if (act == EDL_ACT_RELU) {
    TORCH_CHECK(mask.has_value() && mask->device() == dy.device() &&
                    mask->scalar_type() == torch::kUInt8 &&
                    mask->is_contiguous() && mask->dim() == 2 &&
                    mask->size(0) == m &&
                    mask->size(1) == round_up(n, 16) / 8,
                "relu's bits do not match the gradient");
    a.mask = mask->data_ptr<uint8_t>();
    a.mask_ld = mask->size(1);
  } else if (act == EDL_ACT_SIGMOID) {
    TORCH_CHECK(y.has_value() && y->device() == dy.device() &&
                    y->scalar_type() == dy.scalar_type() && y->dim() == 2 &&
                    y->size(0) == m && y->size(1) == n && y->is_contiguous(),
                "the kept output does not match the gradient");
    a.y = y->data_ptr();
    a.y_ld = n;
    a.y_wide = aligned(*y, n);
  }
  Blocks r, c;
  if (need_dx) {
    TORCH_CHECK(wtq.has_value() && wts.has_value(), "no transposed weight");
    check_blocks(*wtq, *wts, k, n, dy, "transposed weight");
    r = new_blocks(dy, m, n);
    into_rows(a, r);
  }
  if (need_dw) {
    TORCH_CHECK(xtq.has_value() && xts.has_value(), "no kept input");
    check_blocks(*xtq, *xts, k, m, dy, "kept input");
    c = new_blocks(dy, n, m);
    into_cols(a, c);
  }
  Tensor sums;
  const int64_t tiles = round_up(m, EDL_FP8_BLOCK) / EDL_FP8_BLOCK;
  if (need_db) {
    sums = torch::empty({tiles, n}, opts.dtype(torch::kFloat32));
    a.sums = sums.data_ptr<float>();
  }
  if (!need_dx && !need_dw && !need_db) return out;
  launched(edl_fp8_quantize(&a, stream_of(dy)), "fp8 quantise");
  if (need_db) {
    Tensor db = torch::empty({n}, opts.dtype(bt));
    launched(edl_fp8_column_sums(sums.data_ptr<float>(), tiles, n,
                                 db.data_ptr(), type_code(bt, "bias"),
                                 stream_of(dy)),
             "column sums");
    out[2] = db;
  }
  if (need_dx)
    out[0] = multiply(r.q, r.s, m, *wtq, *wts, k, c10::nullopt, EDL_ACT_NONE,
                      dy.scalar_type(), nullptr);
  if (need_dw)
    out[1] = multiply(c.q, c.s, n, *xtq, *xts, k, c10::nullopt, EDL_ACT_NONE,
                      wt, nullptr);
  return out;
}

}  // namespace

void edl_bind_fp8(py::module& m) {
  m.def("fp8_quantize", &fp8_quantize);
  m.def("fp8_dense_fwd", &fp8_dense_fwd);
  m.def("fp8_dense_bwd", &fp8_dense_bwd);
}
