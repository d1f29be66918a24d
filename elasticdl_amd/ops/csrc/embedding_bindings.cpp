// Bindings of the embedding lookup and its gradient (embedding_kernels.hip):
// argument checks, outputs and workspaces.

#include <torch/extension.h>

#include <c10/core/DeviceGuard.h>
#include <c10/hip/HIPStream.h>

#include <cstdint>
#include <limits>

#include "embedding_kernels.h"

extern "C" {
int edl_lookup(const edl_bag*, hipStream_t);
int edl_lookup_weight_grad(const edl_bag*, hipStream_t);
int edl_segment_sums(const edl_segments*, hipStream_t);
int edl_sort_rows(const void*, int, int64_t, int64_t, uint32_t* const*,
                  uint32_t* const*, uint32_t*, uint32_t*, hipStream_t);
int edl_sort_ids_small(const int64_t*, int64_t, uint32_t*, uint32_t*, int64_t*,
                       uint32_t*, hipStream_t);
int edl_ids_range(const int64_t*, int64_t, int64_t*, hipStream_t);
int edl_sort_ids32(const int64_t*, int64_t, int, int64_t, uint32_t* const*,
                   uint32_t* const*, uint32_t*, uint32_t*, hipStream_t);
int edl_sort_ids64(const int64_t*, int64_t, uint64_t* const*,
                   uint32_t* const*, uint32_t*, uint32_t*, hipStream_t);
int edl_unique32(const uint32_t*, int64_t, uint32_t*, uint32_t*, int64_t,
                 const int64_t*, uint32_t*, int64_t*, hipStream_t);
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

// (rows or pooled rows [.., D], each bag's factor where it is asked for)
std::vector<OptTensor> embedding_fwd(Tensor table, Tensor ids,
                                     OptTensor weights, int64_t combiner,
                                     double scale, bool want_coef) {
  c10::DeviceGuard guard(ids.device());
  edl_bag a = bag_of(ids, weights, combiner, scale);
  table_into(a, table, ids);
  TORCH_CHECK(a.B * ((int64_t)a.D + 64) / 256 <
                  std::numeric_limits<int32_t>::max(),
              "the result is too large");
  std::vector<OptTensor> out(2);
  Tensor y = torch::empty({a.B, a.D}, table.options().requires_grad(false));
  out[0] = y;
  a.out = y.data_ptr();
  if (want_coef) {
    Tensor c = torch::empty({a.B}, y.options().dtype(torch::kFloat32));
    a.coef = c.data_ptr<float>();
    out[1] = c;
  }
  if (a.B > 0) launched(edl_lookup(&a, stream_of(ids)), "embedding lookup");
  return out;
}

void segment_sums(edl_segments& s, const Tensor& like) {
  const int64_t chunks = (s.N + EDL_SEG_CHUNK - 1) / EDL_SEG_CHUNK;
  Tensor part = words(like, {chunks * 2, s.D}, torch::kFloat32);
  Tensor marks = words(like, {chunks * 3 + 1});
  s.part = part.data_ptr<float>();
  s.head = u32(marks);
  s.tail = s.head + chunks;
  s.list = s.tail + chunks;
  s.listed = s.list + chunks;
  launched(edl_segment_sums(&s, stream_of(like)), "embedding gradient");
}

struct SortSpace {
  Tensor keys, pos, counts;
  uint32_t *k[2], *p[2], *count, *total;
  SortSpace(const Tensor& like, int64_t n, bool with_keys = true) {
    const int64_t tiles = (n + EDL_SORT_TILE - 1) / EDL_SORT_TILE;
    if (with_keys) {
      keys = words(like, {2, n});
      k[0] = u32(keys);
      k[1] = k[0] + n;
    }
    pos = words(like, {2, n});
    p[0] = u32(pos);
    p[1] = p[0] + n;
    counts = words(like, {(tiles + 1) * EDL_SORT_BINS});
    count = u32(counts);
    total = count + tiles * EDL_SORT_BINS;
  }
};

// (the table's dense gradient [rows, D] of dy's type, the weights' [B, L] in
// float32); each where it is asked for
std::vector<OptTensor> embedding_bwd(Tensor dy, Tensor ids, OptTensor table,
                                     OptTensor weights, OptTensor coef,
                                     int64_t rows, int64_t combiner,
                                     double scale, bool need_table,
                                     bool need_weights) {
  c10::DeviceGuard guard(ids.device());
  edl_bag a = bag_of(ids, weights, combiner, scale);
  TORCH_CHECK(dy.device() == ids.device() && dy.dim() == 2 &&
                  dy.size(0) == a.B && dy.is_contiguous(),
              "gradient does not match the ids");
  TORCH_CHECK(rows >= 1 && rows < kMost, "too many rows: ", rows);
  if (coef.has_value()) {
    TORCH_CHECK(coef->device() == ids.device() &&
                    coef->scalar_type() == torch::kFloat32 &&
                    coef->numel() == a.B && coef->is_contiguous(),
                "factors do not match the ids");
    a.coef = coef->data_ptr<float>();
  }
  TORCH_CHECK(combiner < 0 || coef.has_value(), "no factors of the bags");
  std::vector<OptTensor> out(2);
  const int64_t n = ids.numel(), d = dy.size(1);
  auto opts = dy.options().requires_grad(false);
  if (need_weights) {
    TORCH_CHECK(table.has_value() && weights.has_value(),
                "no table or weights");
    table_into(a, *table, ids);
    TORCH_CHECK(a.D == d && table->scalar_type() == dy.scalar_type(),
                "gradient does not match the table");
    const int v = vec_of(dy, d, d);
    if (v < a.vec) a.vec = v;
    a.dy = dy.data_ptr();
    Tensor dw = torch::empty(ids.sizes(), opts.dtype(torch::kFloat32));
    a.dw = dw.data_ptr<float>();
    if (n > 0)
      launched(edl_lookup_weight_grad(&a, stream_of(ids)), "weights' gradient");
    out[1] = dw;
  }
  if (need_table) {
    Tensor dt = torch::zeros({rows, d}, opts);
    if (n > 0) {
      SortSpace sort(ids, n);
      const int at =
          edl_sort_rows(a.ids, a.ids64, rows, n, sort.k, sort.p, sort.count,
                        sort.total, stream_of(ids));
      launched(at < 0 ? -1 - at : 0, "sort of ids");
      edl_segments s = {};
      s.keys = sort.k[at];
      s.pos = sort.p[at];
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
      segment_sums(s, ids);
    }
    out[0] = dt;
  }
  return out;
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
  c10::DeviceGuard guard(ids.device());
  auto opts = values.options().requires_grad(false);
  const int type = type_code(values.scalar_type(), "values");
  if (n == 0) return {torch::empty({0, d}, opts), torch::empty_like(ids)};
  const hipStream_t st = stream_of(ids);
  Tensor place = words(ids, {n});
  Tensor unique = torch::empty_like(ids);
  SortSpace sort(ids, n);
  const int64_t* id = ids.data_ptr<int64_t>();
  uint32_t* pos = nullptr;
  int64_t found = -1;
  if (n <= EDL_SORT_SMALL) {
    Tensor low = words(ids, {1}, torch::kInt64);
    Tensor meta = words(ids, {2});  // how many; whether they lie too far apart
    launched(edl_sort_ids_small(id, n, sort.k[0], sort.p[0],
                                low.data_ptr<int64_t>(), u32(meta) + 1, st),
             "sort of ids");
    launched(edl_unique32(sort.k[0], n, sort.count, u32(meta), 0,
                          low.data_ptr<int64_t>(), u32(place),
                          unique.data_ptr<int64_t>(), st),
             "unique ids");
    Tensor host = meta.cpu();
    if (host.data_ptr<int32_t>()[1] == 0) {
      found = host.data_ptr<int32_t>()[0];
      pos = sort.p[0];
    }
  }
  if (found < 0) {
    Tensor range = words(ids, {2}, torch::kInt64);
    launched(edl_ids_range(id, n, range.data_ptr<int64_t>(), st),
             "range of ids");
    Tensor host = range.cpu();
    const int64_t low = host.data_ptr<int64_t>()[0];
    const uint64_t span = (uint64_t)host.data_ptr<int64_t>()[1] - (uint64_t)low;
    Tensor many = words(ids, {1});
    if (span >> 32 == 0) {
      int bits = 1;
      while (bits < 32 && (span >> bits) != 0) ++bits;
      const int at = edl_sort_ids32(id, low, bits, n, sort.k, sort.p,
                                    sort.count, sort.total, st);
      launched(at < 0 ? -1 - at : 0, "sort of ids");
      pos = sort.p[at];
      launched(edl_unique32(sort.k[at], n, sort.count, u32(many), low, nullptr,
                            u32(place), unique.data_ptr<int64_t>(), st),
               "unique ids");
    } else {
      Tensor wide = words(ids, {2, n}, torch::kInt64);
      uint64_t* k[2];
      k[0] = reinterpret_cast<uint64_t*>(wide.data_ptr<int64_t>());
      k[1] = k[0] + n;
      const int at = edl_sort_ids64(id, n, k, sort.p, sort.count, sort.total,
                                    st);
      launched(at < 0 ? -1 - at : 0, "sort of ids");
      pos = sort.p[at];
      launched(edl_unique64(k[at], n, sort.count, u32(many), u32(place),
                            unique.data_ptr<int64_t>(), st),
               "unique ids");
    }
    found = many.item<int32_t>();
  }
  Tensor rows = torch::empty({found, d}, opts);
  if (d > 0) {
    edl_segments s = {};
    s.keys = u32(place);
    s.pos = pos;
    s.N = n;
    s.limit = (uint32_t)found;
    s.src = values.data_ptr();
    s.D = (int)d;
    s.type = type;
    s.vec = vec_of(values, d, d);
    s.L = 1;
    s.scale = 1.f;
    s.out = rows.data_ptr();
    segment_sums(s, ids);
  }
  return {rows, unique.narrow(0, 0, found)};
}

}  // namespace

void edl_bind_embedding(py::module& m) {
  m.def("embedding_fwd", &embedding_fwd);
  m.def("embedding_bwd", &embedding_bwd);
  m.def("coalesce_rows", &coalesce_rows);
}
