// Bindings of the 8-bit dense layers (fp8_kernels.hip): argument checks,
// outputs, workspaces, and the layer's autograd function. It is written here
// and not in Python because a small layer's launches take less time than
// Python's autograd does between them (a 4096 x 624 x 400 training step: 158
// us so, 94 us of it on the GPU).

#include <torch/extension.h>
#include <torch/csrc/autograd/functions/basic_ops.h>

#include <c10/core/DeviceGuard.h>
#include <c10/hip/HIPStream.h>

#include <cstdint>
#include <limits>

#include "fp8_kernels.h"

extern "C" {
int edl_fp8_quantize(const edl_fp8_quant*, hipStream_t);
int edl_fp8_quantize_pair(const edl_fp8_quant*, const edl_fp8_quant*,
                          hipStream_t);
void edl_fp8_gemm_plan(edl_fp8_gemm*, int, int);
int edl_fp8_gemm_run(edl_fp8_finish*, int, hipStream_t);
int edl_fp8_few_rows(const edl_fp8_gemm*, const void*, int64_t, int, int, int,
                     hipStream_t);
}

namespace {

using torch::Tensor;
using OptTensor = c10::optional<Tensor>;

// rows that take one launch, and the outputs from which on it would have 2^32
// threads, 64 to each
constexpr int64_t kFewRows = 16, kFewOutputs = 1 << 26;

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

// what stands for a tensor (a traced call's, a subclass's) has no memory, and
// a kernel would read from address 0
void check_memory(const Tensor& t, const char* name) {
  TORCH_CHECK(t.numel() == 0 || t.data_ptr() != nullptr, name,
              " has no memory of its own");
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

// [R, C] contracted over C: where its bytes and scales lie, and their sizes
struct Blocks {
  uint8_t *q = nullptr, *s = nullptr;
  int64_t rows = 0, ld = 0, rp = 0;
};
Blocks blocks_of(int64_t r, int64_t c) {
  Blocks b;
  b.rows = r;
  b.ld = round_up(c, EDL_FP8_BLOCK);
  b.rp = round_up(r, 256);
  return b;
}
Blocks blocks_in(const Tensor& q, const Tensor& s) {
  Blocks b;
  b.q = q.data_ptr<uint8_t>();
  b.s = s.data_ptr<uint8_t>();
  b.rows = q.size(0);
  b.ld = q.size(1);
  b.rp = s.size(1);
  return b;
}

// Several pieces in one allocation, each on a border of 256 bytes: a tensor
// apiece would cost a small layer more than its launches.
class Pieces {
 public:
  void add(Blocks* b) {
    b->q = at(b->rows * b->ld);
    b->s = at(b->ld / EDL_FP8_BLOCK * b->rp);
    blocks_.push_back(b);
  }
  template <typename T>
  void add(T** p, int64_t n) {
    *p = reinterpret_cast<T*>(at(n * (int64_t)sizeof(T)));
    others_.push_back(reinterpret_cast<uint8_t**>(p));
  }
  // places what was added; once
  Tensor place(const Tensor& like) {
    Tensor t = new_bytes(like, 1, size_);
    place_in(t);
    return t;
  }
  void place_in(const Tensor& t) {
    TORCH_CHECK(t.numel() == size_, "kept bytes do not match");
    uint8_t* base = t.data_ptr<uint8_t>();
    for (Blocks* b : blocks_) {
      b->q = base + (intptr_t)b->q;
      b->s = base + (intptr_t)b->s;
    }
    for (uint8_t** p : others_) *p = base + (intptr_t)*p;
  }

 private:
  uint8_t* at(int64_t bytes) {  // an offset, until it is placed
    const int64_t a = size_;
    size_ += round_up(bytes, 256);
    return reinterpret_cast<uint8_t*>((intptr_t)a);
  }
  int64_t size_ = 0;
  c10::SmallVector<Blocks*, 4> blocks_;
  c10::SmallVector<uint8_t**, 4> others_;
};

void into_rows(edl_fp8_quant& a, const Blocks& b) {
  a.rows = b.q;
  a.rows_scale = b.s;
  a.rows_ld = b.ld;
  a.rows_rp = b.rp;
}
void into_cols(edl_fp8_quant& a, const Blocks& b) {
  a.cols = b.q;
  a.cols_scale = b.s;
  a.cols_ld = b.ld;
  a.cols_rp = b.rp;
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
  TORCH_CHECK(reinterpret_cast<uintptr_t>(q.data_ptr()) % 16 == 0 &&
                  reinterpret_cast<uintptr_t>(s.data_ptr()) % 16 == 0,
              name, " must lie on a border of 16 bytes");
}

// c = a b^T; returns c, of `type`
Tensor product_of(edl_fp8_gemm& g, const Blocks& a, const Blocks& b,
                  const Tensor& like, torch::ScalarType type) {
  Tensor c = torch::empty({a.rows, b.rows},
                          like.options().dtype(type).requires_grad(false));
  g.a = a.q;
  g.sa = a.s;
  g.b = b.q;
  g.sb = b.s;
  g.M = a.rows;
  g.N = b.rows;
  g.ld = a.ld;
  g.a_rp = a.rp;
  g.b_rp = b.rp;
  g.act = EDL_ACT_NONE;
  g.c = c.data_ptr();
  g.c_type = type_code(type, "output");
  g.c_wide = aligned(c, b.rows);
  g.wide = g.c_type == EDL_T_F32;
  return c;
}
void bias_into(edl_fp8_gemm& g, const Tensor& bias) {
  if (!bias.defined()) return;
  g.bias = bias.data_ptr();
  g.bias_type = type_code(bias.scalar_type(), "bias");
}
// decides the tiles and splits of f's n products and adds their workspace
void plan_into(edl_fp8_finish& f, int n, Pieces& pieces) {
  edl_fp8_gemm_plan(f.g, n, f.out != nullptr);
  for (int i = 0; i < n; ++i) {
    f.g[i].part_ld = round_up(f.g[i].N, 16);
    if (f.g[i].splits > 1)
      pieces.add(&f.g[i].part, f.g[i].splits * f.g[i].M * f.g[i].part_ld);
  }
}

// (bytes, scales, bytes of the transpose, its scales); the latter two where
// `cols`. Blocks lie along each form's rows, or are 128 x 128 where `tile`.
std::vector<OptTensor> fp8_quantize(Tensor x, bool tile, bool rows,
                                    bool cols) {
  check_matrix(x, "x");
  TORCH_CHECK(x.size(0) < (1 << 24) - 128 || !cols,
              "x has too many rows to be transposed: ", x.size(0));
  TORCH_CHECK(rows || cols, "nothing asked for");
  check_memory(x, "x");
  c10::DeviceGuard guard(x.device());
  x = row_major(x);
  edl_fp8_quant a = quant_of(x, "x");
  a.tile = tile;
  std::vector<OptTensor> out(4);
  auto add = [&](int at, int64_t r, int64_t c) {
    Blocks b = blocks_of(r, c);
    Tensor q = new_bytes(x, r, b.ld);
    Tensor s = new_bytes(x, b.ld / EDL_FP8_BLOCK, b.rp);
    out[at] = q;
    out[at + 1] = s;
    return blocks_in(q, s);
  };
  if (rows) into_rows(a, add(0, a.R, a.C));
  if (cols) into_cols(a, add(2, a.C, a.R));
  if (a.R > 0) launched(edl_fp8_quantize(&a, stream_of(x)), "fp8 quantise");
  return out;
}

// --------------------------------- layer ----------------------------------
// The checks that a user meets; the messages' wording is Python's, where the
// CPU path makes the same ones.
void check_type(const Tensor& t, const char* name) {
  const auto d = t.scalar_type();
  TORCH_CHECK_TYPE(d == torch::kFloat32 || d == torch::kBFloat16 ||
                       d == torch::kFloat16,
                   name, " must be float32, bfloat16 or float16, not ", d);
}
void check_layer(const Tensor& x, int64_t n, int64_t k, c10::Device w_device,
                 const Tensor& bias) {
  check_type(x, "x");
  TORCH_CHECK_VALUE(x.dim() >= 1 && x.size(-1) == k, "x is ", x.sizes(),
                    ", and the weight takes ", k);
  TORCH_CHECK_VALUE(w_device == x.device(), "x is on ", x.device(),
                    ", and the weight on ", w_device);
  TORCH_CHECK_VALUE(n > 0, "the weight has no rows");
  check_memory(x, "x");
  if (!bias.defined()) return;
  TORCH_CHECK_VALUE(bias.dim() == 1 && bias.size(0) == n, "bias is ",
                    bias.sizes(), ", not (", n, ")");
  check_type(bias, "bias");
  TORCH_CHECK_VALUE(bias.device() == x.device(), "x is on ", x.device(),
                    ", and the bias on ", bias.device());
  check_memory(bias, "bias");
}
Tensor rows_of(const Tensor& x) {
  return row_major(x.dim() == 2 ? x : x.reshape({-1, x.size(-1)}));
}
Tensor shaped_like(const Tensor& y, const Tensor& x) {
  if (x.dim() == 2) return y;
  auto shape = x.sizes().vec();
  shape.back() = y.size(1);
  return y.reshape(shape);
}

class Fp8Dense : public torch::autograd::Function<Fp8Dense> {
 public:
  // x [m, k], w [n, k]; grad: whether the caller's gradients are on
  static Tensor forward(torch::autograd::AutogradContext* ctx, Tensor x,
                        Tensor w, const OptTensor& bias_, int64_t act,
                        bool grad) {
    const bool has_bias = bias_.has_value() && bias_->defined();
    const bool need_x = grad && x.requires_grad();
    const bool need_w = grad && w.requires_grad();
    const bool need_b = grad && has_bias && bias_->requires_grad();
    const int64_t m = x.size(0), k = x.size(1), n = w.size(0);
    check_matrix(x, "x");
    check_matrix(w, "w");
    // w^T, and x^T and dz^T for w's gradient, have their rows as columns
    TORCH_CHECK(n < (1 << 24) - 128 && (m < (1 << 24) - 128 || !need_w),
                "too many rows to be transposed: x has ", m, ", w ", n);
    c10::DeviceGuard guard(x.device());
    x = row_major(x);
    w = row_major(w);
    Tensor bias = has_bias ? bias_->contiguous() : Tensor();

    // kept for the backward pass: w^T, x^T and relu's bits
    const bool bits = act == EDL_ACT_RELU && (need_x || need_w || need_b);
    const bool few = m <= kFewRows && !need_w && !bits;
    Pieces kept, passing;
    Blocks wr = blocks_of(n, k), xr = blocks_of(m, k);
    Blocks wc = blocks_of(k, n), xc = blocks_of(k, m);
    uint8_t* mask = nullptr;
    if (need_x) kept.add(&wc);
    if (need_w) kept.add(&xc);
    if (bits) kept.add(&mask, m * mask_row(n));
    passing.add(&wr);
    if (!few) passing.add(&xr);
    edl_fp8_finish f = {};
    Tensor y = product_of(f.g[0], xr, wr, x, x.scalar_type());
    f.g[0].act = (int)act;
    bias_into(f.g[0], bias);
    f.g[0].mask_ld = mask_row(n);
    f.g[0].wide |= bits;
    if (!few && m > 0) plan_into(f, 1, passing);
    Tensor held;
    if (need_x || need_w || bits) held = kept.place(x);
    const Tensor space = passing.place(x);
    f.g[0].a = xr.q;
    f.g[0].sa = xr.s;
    f.g[0].b = wr.q;
    f.g[0].sb = wr.s;
    f.g[0].mask = mask;

    edl_fp8_quant qw = quant_of(w, "w"), qx = quant_of(x, "x");
    qw.tile = true;
    into_rows(qw, wr);
    if (need_x) into_cols(qw, wc);
    if (!few) into_rows(qx, xr);
    if (need_w) into_cols(qx, xc);
    if (few || m == 0) {
      launched(edl_fp8_quantize(&qw, stream_of(x)), "fp8 quantise");
      if (m > 0) few_rows(x, qx, f.g[0]);
    } else {
      launched(edl_fp8_quantize_pair(&qx, &qw, stream_of(x)), "fp8 quantise");
      launched(edl_fp8_gemm_run(&f, 1, stream_of(x)), "fp8 product");
    }
    if (need_x || need_w || need_b) {
      ctx->saved_data["act"] = act;
      ctx->saved_data["k"] = k;
      ctx->saved_data["w"] = (int64_t)w.scalar_type();
      ctx->saved_data["b"] =
          has_bias ? (int64_t)bias.scalar_type() : (int64_t)-1;
      ctx->saved_data["need"] =
          (int64_t)(need_x | need_w << 1 | need_b << 2);
      ctx->save_for_backward({held, act == EDL_ACT_SIGMOID ? y : Tensor()});
    }
    return y;
  }

  // one launch for the gradients' rounding, one or two for the products, and
  // one for what is split and the bias
  static torch::autograd::variable_list backward(
      torch::autograd::AutogradContext* ctx,
      torch::autograd::variable_list grads) {
    const auto saved = ctx->get_saved_variables();
    const int64_t need = ctx->saved_data["need"].toInt();
    const int64_t act = ctx->saved_data["act"].toInt();
    const int64_t k = ctx->saved_data["k"].toInt();
    const auto wt = (torch::ScalarType)ctx->saved_data["w"].toInt();
    const int64_t b_type = ctx->saved_data["b"].toInt();
    torch::autograd::variable_list out(5);
    if (!grads[0].defined()) return out;
    check_memory(grads[0], "gradient");
    {
      at::NoGradGuard none;
      run(saved[0], saved[1], need, grads[0],
          (need & 1) && ctx->needs_input_grad(0),
          (need & 2) && ctx->needs_input_grad(1),
          b_type >= 0 && (need & 4) && ctx->needs_input_grad(2), act, k, wt,
          (torch::ScalarType)(b_type < 0 ? 0 : b_type), out);
    }
    if (at::GradMode::is_enabled()) {  // create_graph: fails where it is used
      torch::autograd::variable_list held;
      for (auto& t : out)
        if (t.defined()) held.push_back(t.detach().requires_grad_(true));
      auto fail = std::make_shared<torch::autograd::DelayedError>(
          "fp8_dense has no second derivative", (int64_t)held.size());
      held = (*fail)(std::move(held));
      size_t i = 0;
      for (auto& t : out)
        if (t.defined()) t = held[i++];
    }
    return out;
  }

  // g: the weight, the result, bias and act
  static void few_rows(const Tensor& x, const edl_fp8_quant& a,
                       const edl_fp8_gemm& g) {
    launched(edl_fp8_few_rows(&g, a.x, a.ld, (int)a.C, a.type, a.wide,
                              stream_of(x)),
             "fp8 product");
  }
  static int64_t mask_row(int64_t n) { return round_up(n, 16) / 8; }

 private:
  static void run(const Tensor& held, const Tensor& y, int64_t had, Tensor dy,
                  bool need_x, bool need_w, bool need_b, int64_t act,
                  int64_t k, torch::ScalarType wt, torch::ScalarType bt,
                  torch::autograd::variable_list& out) {
    c10::DeviceGuard guard(dy.device());
    dy = row_major(dy);
    const int64_t m = dy.size(0), n = dy.size(1);
    const auto opts = dy.options().requires_grad(false);
    if (m == 0) {
      if (need_x) out[0] = torch::empty({0, k}, opts);
      if (need_w) out[1] = torch::zeros({n, k}, opts.dtype(wt));
      if (need_b) out[2] = torch::zeros({n}, opts.dtype(bt));
      return;
    }
    if (!need_x && !need_w && !need_b) return;
    edl_fp8_quant a = quant_of(dy, "gradient");
    a.deriv = true;
    a.act = (int)act;
    Pieces kept, passing;  // kept: laid out as by forward
    Blocks wc = blocks_of(k, n), xc = blocks_of(k, m);
    uint8_t* mask = nullptr;
    if (had & 1) kept.add(&wc);
    if (had & 2) kept.add(&xc);
    if (act == EDL_ACT_RELU) kept.add(&mask, m * mask_row(n));
    if (held.defined()) kept.place_in(held);
    a.mask = mask;
    a.mask_ld = mask_row(n);
    if (act == EDL_ACT_SIGMOID) {
      a.y = y.data_ptr();
      a.y_ld = n;
      a.y_wide = aligned(y, n);
    }
    Blocks r = blocks_of(m, n), c = blocks_of(n, m);
    edl_fp8_finish f = {};
    int products = 0, of_x = -1, of_w = -1;
    if (need_x) {
      passing.add(&r);
      of_x = products++;
      out[0] = product_of(f.g[of_x], r, wc, dy, dy.scalar_type());
    }
    if (need_w) {
      passing.add(&c);
      of_w = products++;
      out[1] = product_of(f.g[of_w], c, xc, dy, wt);
    }
    float* sums = nullptr;
    if (need_b) {
      f.tiles = round_up(m, EDL_FP8_BLOCK) / EDL_FP8_BLOCK;
      f.C = n;
      passing.add(&sums, f.tiles * n);
      out[2] = torch::empty({n}, opts.dtype(bt));
      f.out = out[2].data_ptr();
      f.out_type = type_code(bt, "bias");
    }
    plan_into(f, products, passing);
    const Tensor space = passing.place(dy);
    f.sums = a.sums = sums;
    if (need_x) {
      f.g[of_x].a = r.q;
      f.g[of_x].sa = r.s;
      into_rows(a, r);
    }
    if (need_w) {
      f.g[of_w].a = c.q;
      f.g[of_w].sa = c.s;
      into_cols(a, c);
    }
    launched(edl_fp8_quantize(&a, stream_of(dy)), "fp8 quantise");
    launched(edl_fp8_gemm_run(&f, products, stream_of(dy)), "fp8 product");
  }
};

// act(x w^T + bias), with gradients for x, w and bias
Tensor fp8_dense(const Tensor& x, const Tensor& w, const OptTensor& bias_,
                 int64_t act) {
  const Tensor bias = bias_.has_value() ? *bias_ : Tensor();
  TORCH_CHECK_VALUE(w.dim() == 2, "w must have two dimensions, not ",
                    w.dim());
  check_type(w, "w");
  TORCH_CHECK_VALUE(w.size(1) > 0, "w has no columns");
  check_memory(w, "w");
  check_layer(x, w.size(0), w.size(1), w.device(), bias);
  return shaped_like(
      Fp8Dense::apply(rows_of(x), w, bias_, act, at::GradMode::is_enabled()),
      x);
}

// the same with a weight that was laid out before; no gradients
Tensor fp8_dense_frozen(const Tensor& x, const Tensor& wq, const Tensor& ws,
                        int64_t k, const OptTensor& bias_, int64_t act) {
  Tensor bias = bias_.has_value() ? *bias_ : Tensor();
  const int64_t n = wq.size(0);
  check_layer(x, n, k, wq.device(), bias);
  check_memory(wq, "weight");
  check_memory(ws, "weight");
  TORCH_CHECK(!at::GradMode::is_enabled() ||
                  !(x.requires_grad() ||
                    (bias.defined() && bias.requires_grad())),
              "a weight from quantize_fp8_weight has no backward pass: call "
              "under torch.no_grad(), or pass the weight as a tensor");
  at::NoGradGuard none;
  c10::DeviceGuard guard(x.device());
  const Tensor x2 = rows_of(x);
  check_matrix(x2, "x");
  check_blocks(wq, ws, n, k, x, "weight");
  if (bias.defined()) bias = bias.contiguous();
  const int64_t m = x2.size(0);
  const Blocks w = blocks_in(wq, ws);
  Blocks r = blocks_of(m, k);
  edl_fp8_finish f = {};
  const Tensor y = product_of(f.g[0], r, w, x2, x2.scalar_type());
  f.g[0].act = (int)act;
  bias_into(f.g[0], bias);
  if (m > 0) {
    edl_fp8_quant a = quant_of(x2, "x");
    if (m <= kFewRows && n < kFewOutputs) {
      Fp8Dense::few_rows(x2, a, f.g[0]);
    } else {
      Pieces passing;
      passing.add(&r);
      plan_into(f, 1, passing);
      const Tensor space = passing.place(x2);
      f.g[0].a = r.q;
      f.g[0].sa = r.s;
      into_rows(a, r);
      launched(edl_fp8_quantize(&a, stream_of(x2)), "fp8 quantise");
      launched(edl_fp8_gemm_run(&f, 1, stream_of(x2)), "fp8 product");
    }
  }
  return shaped_like(y, x);
}

}  // namespace

void edl_bind_fp8(py::module& m) {
  m.def("fp8_quantize", &fp8_quantize);
  m.def("fp8_dense", &fp8_dense, py::call_guard<py::gil_scoped_release>());
  m.def("fp8_dense_frozen", &fp8_dense_frozen,
        py::call_guard<py::gil_scoped_release>());
}
