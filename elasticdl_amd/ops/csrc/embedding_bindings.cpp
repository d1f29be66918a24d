// Bindings of the embedding lookup and its gradient (embedding_kernels.hip):
// argument checks, outputs, workspaces, and the lookup's autograd function.

#include <torch/extension.h>
#include <torch/csrc/autograd/functions/basic_ops.h>

#include <c10/core/DeviceGuard.h>
#include <c10/hip/HIPGraphsC10Utils.h>
#include <c10/hip/HIPStream.h>

#include <algorithm>
#include <cstdint>
#include <exception>
#include <limits>

#include "embedding_kernels.h"

extern "C" {
int edl_lookup(const edl_bag*, hipStream_t);
int edl_lookup_weight_grad(const edl_bag*, hipStream_t);
int edl_segment_sums(const edl_segments*, hipStream_t);
int edl_sort_rows(const void*, int, int64_t, int64_t, uint32_t* const*,
                  uint32_t* const*, uint32_t*, uint32_t*, void*, int64_t,
                  hipStream_t);
int edl_segment_chunk(int64_t, int, int);
int64_t edl_sort_counts(int64_t);
int edl_sort_rows_small(const void*, int, int64_t, int64_t, uint32_t*,
                        uint32_t*, uint32_t*, uint32_t*, uint32_t*, void*,
                        int64_t, hipStream_t);
int edl_sort_ids_small(const int64_t*, int64_t, uint32_t*, uint32_t*, int64_t*,
                       uint32_t*, uint32_t*, int64_t*, uint32_t*,
                       hipStream_t);
int edl_ids_range(const int64_t*, int64_t, int64_t*, hipStream_t);
int edl_sort_ids32_first(const int64_t*, int, int64_t, uint32_t* const*,
                         uint32_t* const*, uint32_t*, uint32_t*, hipStream_t);
int edl_sort_ids32_rest(int, int, int64_t, uint32_t* const*, uint32_t* const*,
                        uint32_t*, uint32_t*, hipStream_t);
int edl_sort_ids64(const int64_t*, int64_t, uint64_t* const*,
                   uint32_t* const*, uint32_t*, uint32_t*, hipStream_t);
int edl_unique32(const uint32_t*, int64_t, uint32_t*, uint32_t*, int64_t,
                 uint32_t*, int64_t*, hipStream_t);
int edl_unique64(const uint64_t*, int64_t, uint32_t*, uint32_t*, uint32_t*,
                 int64_t*, hipStream_t);
}

namespace {

using torch::Tensor;
using OptTensor = c10::optional<Tensor>;

// positions, and rows of a table, are 32-bit; a tile's worth is left free
constexpr int64_t kMost = std::numeric_limits<int32_t>::max() - EDL_SORT_TILE;

hipStream_t stream_of(const Tensor& t) {
  return c10::hip::getCurrentHIPStream(t.device().index()).stream();
}

// one event for each thread and device, kept: making one costs as much as it
// saves
hipEvent_t event_of(int device) {
  constexpr int kDevices = 64;
  static thread_local hipEvent_t events[kDevices] = {};
  TORCH_CHECK(device >= 0 && device < kDevices, "device ", device);
  if (!events[device])
    TORCH_CHECK(hipEventCreateWithFlags(&events[device],
                                        hipEventDisableTiming) == hipSuccess,
                "event");
  return events[device];
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

// the largest load of neighbours, up to 16 bytes, that every row allows
int vec_of(const Tensor& t, int64_t d, int64_t row_stride) {
  const int64_t size = t.element_size();
  const uintptr_t at = reinterpret_cast<uintptr_t>(t.data_ptr());
  for (int64_t v = 16 / size; v > 1; v /= 2)
    if (d % v == 0 && row_stride % v == 0 && at % (v * size) == 0)
      return (int)v;
  return 1;
}

Tensor words(const Tensor& like, std::vector<int64_t> shape,
             torch::ScalarType type = torch::kInt32) {
  return torch::empty(shape,
                      like.options().dtype(type).requires_grad(false));
}
uint32_t* u32(const Tensor& t) {
  return reinterpret_cast<uint32_t*>(t.data_ptr<int32_t>());
}

// several pieces of a workspace in one allocation, on borders of 256 bytes
class Pieces {
 public:
  template <typename T>
  void add(T** p, int64_t n) {
    *p = reinterpret_cast<T*>((intptr_t)size_);
    size_ += (n * (int64_t)sizeof(T) + 255) / 256 * 256;
    all_.push_back(reinterpret_cast<uint8_t**>(p));
  }
  Tensor place(const Tensor& like) {
    Tensor t = words(like, {size_}, torch::kUInt8);
    uint8_t* base = t.data_ptr<uint8_t>();
    for (uint8_t** p : all_) *p = base + (intptr_t)*p;
    return t;
  }

 private:
  int64_t size_ = 0;
  c10::SmallVector<uint8_t**, 12> all_;
};

edl_bag bag_of(const Tensor& ids, const OptTensor& weights, int64_t combiner,
               double scale) {
  TORCH_CHECK(ids.is_cuda(), "ids must be on a GPU");
  TORCH_CHECK(ids.scalar_type() == torch::kInt64 ||
                  ids.scalar_type() == torch::kInt32,
              "ids must be int64 or int32, not ", ids.scalar_type());
  TORCH_CHECK(ids.is_contiguous(), "ids must be contiguous");
  TORCH_CHECK(ids.numel() < kMost, "too many ids: ", ids.numel());
  TORCH_CHECK(combiner >= -1 && combiner <= EDL_BAG_SQRTN,
              "unknown combiner ", combiner);
  TORCH_CHECK(combiner < 0 || ids.dim() == 2,
              "ids of bags must be [bags, length]");
  edl_bag a = {};
  a.ids = ids.data_ptr();
  a.ids64 = ids.scalar_type() == torch::kInt64;
  a.B = combiner < 0 ? ids.numel() : ids.size(0);
  a.L = combiner < 0 ? 1 : (int)ids.size(1);
  a.combiner = combiner < 0 ? EDL_BAG_SUM : (int)combiner;
  a.scale = (float)scale;
  if (weights.has_value()) {
    TORCH_CHECK(combiner >= 0, "weights need a combiner");
    TORCH_CHECK(weights->device() == ids.device() &&
                    weights->sizes() == ids.sizes() &&
                    weights->is_contiguous(),
                "weights must be contiguous and of the ids' shape and device");
    a.weights = weights->data_ptr();
    a.w_type = type_code(weights->scalar_type(), "weights");
  }
  return a;
}

void table_into(edl_bag& a, const Tensor& table, const Tensor& ids) {
  TORCH_CHECK(table.is_cuda() && table.device() == ids.device(),
              "table must be on the ids' device");
  TORCH_CHECK(table.dim() == 2 && table.size(0) >= 1 && table.size(1) >= 1 &&
                  table.size(0) < kMost && table.size(1) < (1 << 20),
              "table must be [rows, dim] with between 1 and 2^31 - 4097 rows "
              "and fewer than 2^20 columns");
  TORCH_CHECK(table.size(1) == 1 || table.stride(1) == 1,
              "neighbours in a row of the table must be adjacent");
  a.table = table.data_ptr();
  a.V = table.size(0);
  a.D = (int)table.size(1);
  a.ld = table.stride(0);
  a.type = type_code(table.scalar_type(), "table");
  a.vec = vec_of(table, a.D, a.ld);
}

void segments_into(edl_segments& s, Pieces& pieces) {
  s.chunk = edl_segment_chunk(s.N, s.D, s.vec);
  const int64_t chunks = (s.N + s.chunk - 1) / s.chunk;
  pieces.add(&s.part, chunks * 2 * s.D);
  pieces.add(&s.head, chunks);
  pieces.add(&s.tail, chunks);
}

struct SortSpace {
  uint32_t *k[2] = {}, *p[2] = {}, *count = nullptr, *total = nullptr;
  SortSpace(Pieces& pieces, int64_t n) {
    for (int i = 0; i < 2; ++i) {
      pieces.add(&k[i], n);
      pieces.add(&p[i], n);
    }
    pieces.add(&count, edl_sort_counts(n));
    pieces.add(&total, EDL_SORT_BINS);
  }
};

struct SmallSpace {  // of a small sort
  uint32_t *keys = nullptr, *pos = nullptr, *starts = nullptr,
           *runs = nullptr, *rows = nullptr;
  int64_t* info = nullptr;
  SmallSpace(Pieces& pieces, int64_t n, bool with_rows) {
    pieces.add(&keys, n);
    pieces.add(&pos, n);
    pieces.add(&starts, n);
    pieces.add(&runs, 1);
    pieces.add(&info, 2);
    if (with_rows) pieces.add(&rows, n);
  }
  void into(edl_segments& s) const {
    s.pos = pos;
    s.starts = starts;
    s.runs = runs;
    s.rows = rows;
  }
};

class Lookup : public torch::autograd::Function<Lookup> {
 public:
  // grad: whether the caller's gradients are on
  static Tensor forward(torch::autograd::AutogradContext* ctx, Tensor table,
                        const OptTensor& weights_, Tensor ids,
                        int64_t combiner, double scale, bool grad) {
    const bool need_t = grad && table.requires_grad();
    const bool need_w =
        grad && weights_.has_value() && weights_->requires_grad();
    c10::DeviceGuard guard(ids.device());
    const OptTensor weights =
        weights_.has_value() ? OptTensor(weights_->contiguous()) : OptTensor();
    ids = ids.contiguous();
    edl_bag a = bag_of(ids, weights, combiner, scale);
    table_into(a, table, ids);
    Tensor out =
        torch::empty({a.B, a.D}, table.options().requires_grad(false));
    a.out = out.data_ptr();
    Tensor coef;  // each bag's factor, for the backward pass
    if (combiner >= 0 && (need_t || need_w)) {
      coef = words(ids, {a.B}, torch::kFloat32);
      a.coef = coef.data_ptr<float>();
    }
    if (a.B > 0) launched(edl_lookup(&a, stream_of(ids)), "embedding lookup");
    if (need_t || need_w) {
      ctx->saved_data["rows"] = a.V;
      ctx->saved_data["combiner"] = combiner;
      ctx->saved_data["scale"] = scale;
      ctx->saved_data["need"] = (int64_t)(need_t | need_w << 1);
      ctx->save_for_backward({ids, need_w ? table : Tensor(),
                              weights.has_value() ? *weights : Tensor(),
                              coef});
    }
    return out;
  }

  static torch::autograd::variable_list backward(
      torch::autograd::AutogradContext* ctx,
      torch::autograd::variable_list grads) {
    const auto saved = ctx->get_saved_variables();
    const int64_t need = ctx->saved_data["need"].toInt();
    torch::autograd::variable_list out(6);
    if (!grads[0].defined()) return out;
    check_memory(grads[0], "gradient");
    {
      at::NoGradGuard none;
      run(grads[0].contiguous(), saved[0], saved[1], saved[2], saved[3],
          ctx->saved_data["rows"].toInt(), ctx->saved_data["combiner"].toInt(),
          ctx->saved_data["scale"].toDouble(),
          (need & 1) && ctx->needs_input_grad(0),
          (need & 2) && ctx->needs_input_grad(1), out);
    }
    if (at::GradMode::is_enabled()) {  // create_graph: fails where it is used
      torch::autograd::variable_list held;
      for (auto& t : out)
        if (t.defined()) held.push_back(t.detach().requires_grad_(true));
      auto fail = std::make_shared<torch::autograd::DelayedError>(
          "embedding_lookup has no second derivative", (int64_t)held.size());
      held = (*fail)(std::move(held));
      size_t i = 0;
      for (auto& t : out)
        if (t.defined()) t = held[i++];
    }
    return out;
  }

 private:
  // the table's dense gradient [rows, D] of dy's type, the weights' [B, L]
  static void run(const Tensor& dy, const Tensor& ids, const Tensor& table,
                  const Tensor& weights, const Tensor& coef, int64_t rows,
                  int64_t combiner, double scale, bool need_t, bool need_w,
                  torch::autograd::variable_list& out) {
    c10::DeviceGuard guard(ids.device());
    edl_bag a = bag_of(ids, weights.defined() ? OptTensor(weights) : OptTensor(),
                       combiner, scale);
    if (coef.defined()) a.coef = coef.data_ptr<float>();
    const int64_t n = ids.numel(), d = dy.size(1);
    const auto opts = dy.options().requires_grad(false);
    if (need_w) {
      table_into(a, table, ids);
      const int v = vec_of(dy, d, d);
      if (v < a.vec) a.vec = v;
      a.dy = dy.data_ptr();
      Tensor dw = torch::empty(ids.sizes(), opts.dtype(torch::kFloat32));
      a.dw = dw.data_ptr<float>();
      if (n > 0)
        launched(edl_lookup_weight_grad(&a, stream_of(ids)),
                 "weights' gradient");
      out[1] = dw.to(weights.scalar_type());
    }
    if (!need_t) return;
    if (n == 0) {
      out[0] = torch::zeros({rows, d}, opts);
      return;
    }
    Tensor dt = torch::empty({rows, d}, opts);  // the sort fills it with zeros
    const int64_t bytes = dt.numel() * dt.element_size();
    out[0] = dt;
    edl_segments s = {};
    s.N = n;
    s.limit = (uint32_t)rows;
    s.src = dy.data_ptr();
    s.D = (int)d;
    s.type = type_code(dy.scalar_type(), "gradient");
    s.vec = vec_of(dy, d, d);
    s.L = a.L;
    s.scale = a.scale;
    s.coef = a.coef;
    s.weights = a.weights;
    s.w_type = a.w_type;
    s.out = dt.data_ptr();
    Pieces pieces;
    if (n <= EDL_SORT_SMALL) {
      SmallSpace small(pieces, n, true);
      const Tensor space = pieces.place(ids);
      launched(edl_sort_rows_small(a.ids, a.ids64, rows, n, small.keys,
                                   small.pos, small.starts, small.runs, small.rows,
                                   dt.data_ptr(), bytes, stream_of(ids)),
               "sort of ids");
      small.into(s);
      launched(edl_segment_sums(&s, stream_of(ids)), "embedding gradient");
      return;
    }
    SortSpace sort(pieces, n);
    segments_into(s, pieces);
    const Tensor space = pieces.place(ids);
    const int at =
        edl_sort_rows(a.ids, a.ids64, rows, n, sort.k, sort.p, sort.count,
                      sort.total, dt.data_ptr(), bytes, stream_of(ids));
    launched(at < 0 ? -1 - at : 0, "sort of ids");
    s.keys = sort.k[at];
    s.pos = sort.p[at];
    launched(edl_segment_sums(&s, stream_of(ids)), "embedding gradient");
  }
};

void check_type(const Tensor& t, const char* name) {
  const auto d = t.scalar_type();
  TORCH_CHECK_TYPE(d == torch::kFloat32 || d == torch::kBFloat16 ||
                       d == torch::kFloat16,
                   name, " must be float32, bfloat16 or float16, not ", d);
}

// the checks that a user meets are worded as on the CPU, in Python
Tensor embedding_lookup(const Tensor& table_, const Tensor& ids,
                        const OptTensor& weights, int64_t combiner,
                        double scale) {
  Tensor table = table_;
  TORCH_CHECK_VALUE(
      table.dim() == 2 && table.size(0) > 0 && table.size(1) > 0, "table is ",
      table.sizes(), ", not [rows, dim]");
  check_type(table, "table");
  TORCH_CHECK_TYPE(ids.scalar_type() == torch::kInt64 ||
                       ids.scalar_type() == torch::kInt32,
                   "ids must be int64 or int32, not ", ids.scalar_type());
  TORCH_CHECK_VALUE(ids.device() == table.device(), "ids are on ",
                    ids.device(), ", and the table on ", table.device());
  TORCH_CHECK_VALUE(combiner < 0 || ids.dim() == 2,
                    "ids of bags must be [bags, length], not ", ids.sizes());
  if (weights.has_value()) {
    TORCH_CHECK_VALUE(combiner >= 0, "weights need a combiner");
    TORCH_CHECK_VALUE(weights->sizes() == ids.sizes() &&
                          weights->device() == ids.device(),
                      "weights must have the ids' shape and device");
    check_type(*weights, "weights");
    check_memory(*weights, "weights");
  }
  check_memory(table, "table");
  check_memory(ids, "ids");
  if (table.size(1) > 1 && table.stride(1) != 1) table = table.contiguous();
  Tensor out = Lookup::apply(table, weights, ids, combiner, scale,
                             at::GradMode::is_enabled());
  if (combiner >= 0 || ids.dim() == 1) return out;
  auto shape = ids.sizes().vec();
  shape.push_back(table.size(1));
  return out.view(shape);
}

// (rows summed by id, the ids in order)
std::vector<Tensor> coalesce_rows(Tensor values, Tensor ids) {
  TORCH_CHECK(values.is_cuda() && ids.device() == values.device(),
              "values and ids must be on the same GPU");
  TORCH_CHECK(ids.scalar_type() == torch::kInt64 && ids.is_contiguous() &&
                  ids.dim() == 1,
              "ids must be contiguous int64 of one dimension");
  TORCH_CHECK(values.dim() == 2 && values.size(0) == ids.size(0) &&
                  values.is_contiguous() && values.size(1) < (1 << 20),
              "values must be contiguous [ids, dim]");
  const int64_t n = ids.size(0), d = values.size(1);
  TORCH_CHECK(n < kMost, "too many ids: ", n);
  check_memory(values, "values");
  check_memory(ids, "ids");
  c10::DeviceGuard guard(ids.device());
  TORCH_CHECK(c10::hip::currentStreamCaptureStatusMayInitCtx() ==
                  c10::hip::CaptureStatus::None,
              "coalesce_rows reads back how many ids there are and cannot be "
              "captured into a graph");
  auto opts = values.options().requires_grad(false);
  const int type = type_code(values.scalar_type(), "values");
  if (n == 0) return {torch::empty({0, d}, opts), torch::empty_like(ids)};
  const hipStream_t st = stream_of(ids);
  Tensor unique = torch::empty_like(ids);
  int64_t* ids_out = unique.data_ptr<int64_t>();
  const int64_t* id = ids.data_ptr<int64_t>();
  // what the host reads, in memory that the kernels write to directly: how
  // many ids, and their smallest and largest by parts
  const Tensor host =
      torch::empty({1 + 2 * EDL_RANGE_PARTS},
                   torch::TensorOptions().dtype(torch::kInt64).pinned_memory(
                       true));
  uint32_t* found_at = reinterpret_cast<uint32_t*>(host.data_ptr<int64_t>());
  int64_t* range = host.data_ptr<int64_t>() + 1;
  // an error on the way does not give that memory back while kernels that
  // were launched may write to it
  struct Settled {
    hipStream_t st;
    int thrown = std::uncaught_exceptions();
    ~Settled() {
      if (std::uncaught_exceptions() > thrown) (void)hipStreamSynchronize(st);
    }
  } settled{st};
  const hipEvent_t known = event_of(ids.device().index());
  const auto mark = [&] {
    TORCH_CHECK(hipEventRecord(known, st) == hipSuccess, "event record");
  };
  const auto wait = [&] {  // for what was launched before the mark
    TORCH_CHECK(hipEventSynchronize(known) == hipSuccess, "event wait");
  };
  edl_segments s = {};
  s.N = n;
  s.D = (int)d;
  s.vec = vec_of(values, d, d);
  s.src = values.data_ptr();
  s.type = type;
  s.L = 1;
  s.scale = 1.f;
  s.limit = (uint32_t)n;
  // small results are summed into room for n rows before the host knows how
  // many there are, which takes it longer than the sums take (20 thousand rows
  // of 16 columns 57 us, 62 where it waits first; 400 thousand, 73 and 80).
  // The limit is for memory: the result keeps the room
  const bool early = n * d * values.element_size() <= (4 << 20);
  Tensor rows;
  const auto sum_into = [&](int64_t most) {
    rows = torch::empty({most, d}, opts);
    s.out = rows.data_ptr();
    if (d > 0) launched(edl_segment_sums(&s, st), "sums of rows");
  };
  int64_t found = -1;
  if (n <= EDL_SORT_SMALL) {
    Pieces pieces;
    SmallSpace small(pieces, n, false);
    const Tensor space = pieces.place(ids);
    launched(edl_sort_ids_small(id, n, small.keys, small.pos, small.info,
                                small.starts, small.runs, ids_out, found_at,
                                st),
             "sort of ids");
    mark();
    small.into(s);
    if (early) sum_into(n);
    wait();
    found = found_at[0];
    if (!early) sum_into(found);
    return {rows.narrow(0, 0, found), unique.narrow(0, 0, found)};
  }
  uint32_t* place = nullptr;
  Pieces pieces;
  pieces.add(&place, n);
  SortSpace sort(pieces, n);
  if (d > 0) segments_into(s, pieces);
  const Tensor space = pieces.place(ids);
  s.keys = place;
  Tensor wide;  // 64-bit keys
  {
    constexpr int kFirst = 9;
    launched(edl_ids_range(id, n, range, st), "range of ids");
    mark();
    launched(edl_sort_ids32_first(id, kFirst, n, sort.k, sort.p, sort.count,
                                  sort.total, st),
             "sort of ids");
    wait();
    int64_t low = range[0], high = range[1];
    for (int i = 1; i < EDL_RANGE_PARTS; ++i) {
      low = std::min(low, range[2 * i]);
      high = std::max(high, range[2 * i + 1]);
    }
    const uint64_t differ = (uint64_t)low ^ (uint64_t)high;
    if (differ >> 32 == 0) {
      int bits = 1;
      while (bits < 32 && (differ >> bits) != 0) ++bits;
      const int at = edl_sort_ids32_rest(kFirst, bits, n, sort.k, sort.p,
                                         sort.count, sort.total, st);
      launched(at < 0 ? -1 - at : 0, "sort of ids");
      s.pos = sort.p[at];
      launched(edl_unique32(sort.k[at], n, sort.count, found_at,
                            low & ~(int64_t)0xffffffff, place, ids_out, st),
               "unique ids");
    } else {
      wide = words(ids, {2, n}, torch::kInt64);
      uint64_t* k[2];
      k[0] = reinterpret_cast<uint64_t*>(wide.data_ptr<int64_t>());
      k[1] = k[0] + n;
      const int at = edl_sort_ids64(id, n, k, sort.p, sort.count, sort.total,
                                    st);
      launched(at < 0 ? -1 - at : 0, "sort of ids");
      s.pos = sort.p[at];
      launched(edl_unique64(k[at], n, sort.count, found_at, place, ids_out,
                            st),
               "unique ids");
    }
    mark();
    if (early) sum_into(n);
    wait();
    found = found_at[0];
    if (!early) sum_into(found);
  }
  return {rows.narrow(0, 0, found), unique.narrow(0, 0, found)};
}

}  // namespace

void edl_bind_embedding(py::module& m) {
  m.def("embedding_lookup", &embedding_lookup,
        py::call_guard<py::gil_scoped_release>());
  m.def("coalesce_rows", &coalesce_rows,
        py::call_guard<py::gil_scoped_release>());
}
