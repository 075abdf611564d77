// TORCH_LIBRARY(bf, ...) operators over the C ABI (include/budgetformer_hip.h):
// the hot path's entry points as PyTorch operators taking and returning
// at::Tensor, launched on the current HIP stream of the inputs' device. Outputs
// and scratch come from PyTorch's caching allocator (a failed allocation raises
// torch.OutOfMemoryError), argument errors raise ValueError or
// NotImplementedError, HIP errors RuntimeError, as the ctypes bindings do.
// Host code only: every kernel is in libbudgetformer_hip.so.
//
// The attention index (bf_attn_index) travels as 16 optional tensors and 10
// integers, in the order of kIndexTensors and make_index below
// (budgetformer_amd.hip_ops.AttentionIndex.op_args builds them).
#include <ATen/ATen.h>
#include <ATen/MemoryOverlap.h>
#include <c10/core/DeviceGuard.h>
#include <c10/hip/HIPStream.h>
#include <torch/csrc/autograd/custom_function.h>
#include <torch/csrc/autograd/functions/basic_ops.h>
#include <torch/library.h>

#include <algorithm>
#include <string>

#include "budgetformer_hip.h"

namespace {

void check_rc(int rc, const char* what) {
  if (rc == BF_OK) return;
  const std::string msg = bf_last_error();
  TORCH_CHECK_VALUE(rc != BF_ERR_INVALID, what, ": ", msg);
  TORCH_CHECK_NOT_IMPLEMENTED(rc != BF_ERR_UNSUPPORTED, what, ": ", msg);
  TORCH_CHECK(false, what, ": ", msg);
}

void* stream_of(const at::Tensor& t) {
  return c10::hip::getCurrentHIPStream(t.device().index()).stream();
}

void require(const at::Tensor& t, const char* name, at::ScalarType st, const at::Device& dev) {
  TORCH_CHECK_VALUE(t.defined(), name, " is undefined");
  TORCH_CHECK_VALUE(t.device() == dev, name, " is on ", t.device(), ", expected ", dev);
  TORCH_CHECK_VALUE(t.scalar_type() == st, name, " must be ", st, " (got ", t.scalar_type(), ")");
  TORCH_CHECK_VALUE(t.is_contiguous(), name, " must be contiguous");
}

template <typename P>
P* opt_ptr(const std::optional<at::Tensor>& t, const char* name, at::ScalarType st, const at::Device& dev) {
  if (!t.has_value() || !t->defined()) return nullptr;
  require(*t, name, st, dev);
  return static_cast<P*>(t->data_ptr());
}

at::Tensor scratch_bytes(size_t bytes, const at::Device& dev) {
  return at::empty({int64_t(std::max<size_t>(bytes, 1))}, at::TensorOptions().dtype(at::kByte).device(dev));
}

// ---------------------------------------------------------------- attention index
constexpr const char* kIndexTensors[16] = {"qptr",       "kv",         "kptr",         "kq",
                                           "ks",         "q_nitems",   "q_item_off",   "q_item_row",
                                           "q_heavy_rows", "k_nitems", "k_item_off",   "k_item_row",
                                           "k_heavy_rows", "k_order",  "k_spans",      "plan_counts"};
// The 10 integers, in order: n_q, n_kv, nnz, chunk, item, q_items, q_heavy, k_items, k_heavy, token_column.

bf_attn_index make_index(const c10::List<std::optional<at::Tensor>>& t, at::IntArrayRef n, const at::Device& dev) {
  TORCH_CHECK_VALUE(t.size() == 16, "attention index: 16 tensors expected (got ", t.size(), ")");
  TORCH_CHECK_VALUE(n.size() == 10, "attention index: 10 sizes expected (got ", n.size(), ")");
  auto get = [&](int i, at::ScalarType st) -> const void* {
    const std::optional<at::Tensor> o = t.get(i);
    return opt_ptr<const void>(o, kIndexTensors[i], st, dev);
  };
  bf_attn_index x{};
  x.n_q = n[0];
  x.n_kv = n[1];
  x.nnz = n[2];
  x.chunk = int32_t(n[3]);
  x.item = int32_t(n[4]);
  x.q_items = int32_t(n[5]);
  x.q_heavy = int32_t(n[6]);
  x.k_items = int32_t(n[7]);
  x.k_heavy = int32_t(n[8]);
  x.token_column = int32_t(n[9]);
  x.qptr = static_cast<const int64_t*>(get(0, at::kLong));
  x.kv = static_cast<const int32_t*>(get(1, at::kInt));
  x.kptr = static_cast<const int64_t*>(get(2, at::kLong));
  x.kq = static_cast<const int32_t*>(get(3, at::kInt));
  x.ks = static_cast<const int32_t*>(get(4, at::kInt));
  x.q_nitems = static_cast<const int32_t*>(get(5, at::kInt));
  x.q_item_off = static_cast<const int32_t*>(get(6, at::kInt));
  x.q_item_row = static_cast<const int32_t*>(get(7, at::kInt));
  x.q_heavy_rows = static_cast<const int32_t*>(get(8, at::kInt));
  x.k_nitems = static_cast<const int32_t*>(get(9, at::kInt));
  x.k_item_off = static_cast<const int32_t*>(get(10, at::kInt));
  x.k_item_row = static_cast<const int32_t*>(get(11, at::kInt));
  x.k_heavy_rows = static_cast<const int32_t*>(get(12, at::kInt));
  x.k_order = static_cast<const int32_t*>(get(13, at::kInt));
  x.k_spans = static_cast<const uint64_t*>(get(14, at::kLong));
  x.plan_counts = static_cast<const int32_t*>(get(15, at::kInt));
  return x;
}

int32_t dtype_code(const at::Tensor& q) {
  if (q.scalar_type() == at::kFloat) return BF_DTYPE_F32;
  if (q.scalar_type() == at::kHalf) return BF_DTYPE_F16;
  TORCH_CHECK_VALUE(q.scalar_type() == at::kBFloat16,
                    "attention supports float32, bfloat16 and float16 activations (got ", q.scalar_type(), ")");
  return BF_DTYPE_BF16;
}

void check_qkv(const at::Tensor& q, const at::Tensor& k, const at::Tensor& v, const bf_attn_index& idx) {
  const at::Device dev = q.device();
  for (const auto* p : {&q, &k, &v}) {
    require(*p, p == &q ? "q" : p == &k ? "k" : "v", q.scalar_type(), dev);
    TORCH_CHECK_VALUE(p->dim() == 3, "q, k, v must be [rows, heads, head_dim]");
  }
  TORCH_CHECK_VALUE(k.sizes() == v.sizes() && q.size(1) == k.size(1) && q.size(2) == k.size(2), "q ", q.sizes(),
                    ", k ", k.sizes(), ", v ", v.sizes(), " disagree");
  TORCH_CHECK_VALUE(q.size(0) == idx.n_q && k.size(0) == idx.n_kv, "q rows ", q.size(0), " / kv rows ", k.size(0),
                    " do not match the index (", idx.n_q, ", ", idx.n_kv, ")");
}

const float* edge_tensor(const std::optional<at::Tensor>& t, const char* name, const bf_attn_index& idx, int64_t H,
                         const at::Device& dev) {
  const float* p = opt_ptr<const float>(t, name, at::kFloat, dev);
  if (p) TORCH_CHECK_VALUE(t->dim() == 2 && t->size(0) == idx.nnz && t->size(1) == H, name, " must be [", idx.nnz,
                           ", ", H, "] (got ", t->sizes(), ")");
  return p;
}

bf_attn_dropout make_dropout(double rate, int64_t seed, int64_t offset) {
  TORCH_CHECK_VALUE(rate >= 0.0 && rate <= 1.0, "dropout rate ", rate, " outside [0, 1]");
  return bf_attn_dropout{float(rate), uint64_t(seed), uint64_t(offset), nullptr};
}

// Entries the index's kv array holds room for (its capacity; nnz when sized exactly): the keep mask's
// rows, known without reading the entry count back.
int64_t kv_capacity(const c10::List<std::optional<at::Tensor>>& index) {
  const std::optional<at::Tensor> kv = index.get(1);
  return kv.has_value() ? kv->numel() : 0;
}

// Forward (bf_attn_fwd): (out [n_q, H, hn] in q's dtype, Z [n_q, H] float32, keep). With keep_mask and a
// dropout, keep is the mask of the bits drawn, uint8 [kv capacity, ceil(H / 8)], for the backward; else
// empty.
std::tuple<at::Tensor, at::Tensor, at::Tensor> sparse_attn_fwd(
    const at::Tensor& q, const at::Tensor& k, const at::Tensor& v, const c10::List<std::optional<at::Tensor>>& index,
    at::IntArrayRef sizes, const std::optional<at::Tensor>& bias, const std::optional<at::Tensor>& factor,
    double dropout_rate, int64_t dropout_seed, int64_t dropout_offset, double score_clamp, bool keep_mask) {
  TORCH_CHECK_VALUE(q.is_cuda(), "q must be a device tensor (got ", q.device(), ")");
  const c10::DeviceGuard guard(q.device());
  const at::Device dev = q.device();
  const bf_attn_index idx = make_index(index, sizes, dev);
  check_qkv(q, k, v, idx);
  const int64_t H = q.size(1), hn = q.size(2);
  const float* b = edge_tensor(bias, "bias", idx, H, dev);
  const float* f = edge_tensor(factor, "factor", idx, H, dev);
  bf_attn_dropout drop = make_dropout(dropout_rate, dropout_seed, dropout_offset);
  // the kernels read the mask by aligned dwords: its storage is rounded up to a multiple of 4 bytes
  const int64_t kb = (H + 7) / 8, rows = keep_mask && dropout_rate > 0.0 ? kv_capacity(index) : 0;
  at::Tensor keep =
      at::empty({(rows * kb + 3) / 4 * 4}, q.options().dtype(at::kByte)).narrow(0, 0, rows * kb).view({rows, kb});
  if (keep.numel()) drop.keep = keep.data_ptr<uint8_t>();
  at::Tensor out = at::empty_like(q);
  at::Tensor Z = at::empty({idx.n_q, H}, q.options().dtype(at::kFloat));
  const int64_t parts = bf_attn_partials_floats(&idx, int32_t(H), int32_t(hn));
  at::Tensor partials = at::empty({std::max<int64_t>(parts, 1)}, q.options().dtype(at::kFloat));
  check_rc(bf_attn_fwd(&idx, dtype_code(q), int32_t(H), int32_t(hn), float(score_clamp), q.data_ptr(), k.data_ptr(),
                       v.data_ptr(), b, f,
                       dropout_rate > 0.0 ? &drop : nullptr, out.data_ptr(), Z.data_ptr<float>(),
                       partials.data_ptr<float>(), stream_of(q)),
           "bf::sparse_attn_fwd");
  return {out, Z, keep};
}

// Backward (bf_attn_bwd): (dq, dk, dv, dbias); dbias is [nnz, H] float32 with need_dbias, else empty.
std::tuple<at::Tensor, at::Tensor, at::Tensor, at::Tensor> sparse_attn_bwd(
    const at::Tensor& q, const at::Tensor& k, const at::Tensor& v, const c10::List<std::optional<at::Tensor>>& index,
    at::IntArrayRef sizes, const at::Tensor& Z, const at::Tensor& dout, const std::optional<at::Tensor>& bias,
    const std::optional<at::Tensor>& factor, bool need_dbias, double dropout_rate, int64_t dropout_seed,
    int64_t dropout_offset, double score_clamp, const std::optional<at::Tensor>& keep) {
  TORCH_CHECK_VALUE(q.is_cuda(), "q must be a device tensor (got ", q.device(), ")");
  const c10::DeviceGuard guard(q.device());
  const at::Device dev = q.device();
  const bf_attn_index idx = make_index(index, sizes, dev);
  check_qkv(q, k, v, idx);
  const int64_t H = q.size(1), hn = q.size(2);
  require(dout, "dout", q.scalar_type(), dev);
  require(Z, "Z", at::kFloat, dev);
  TORCH_CHECK_VALUE(dout.sizes() == q.sizes() && Z.dim() == 2 && Z.size(0) == q.size(0) && Z.size(1) == H, "dout ",
                    dout.sizes(), " / Z ", Z.sizes(), " do not match q ", q.sizes());
  const float* b = edge_tensor(bias, "bias", idx, H, dev);
  const float* f = edge_tensor(factor, "factor", idx, H, dev);
  bf_attn_dropout drop = make_dropout(dropout_rate, dropout_seed, dropout_offset);
  if (keep.has_value() && keep->numel() && dropout_rate > 0.0) {
    // the forward's mask of this index, dropout and head count (a [kv capacity, ceil(H / 8)] byte tensor)
    drop.keep = opt_ptr<uint8_t>(keep, "keep", at::kByte, dev);
    TORCH_CHECK_VALUE(keep->dim() == 2 && keep->size(0) >= kv_capacity(index) && keep->size(1) == (H + 7) / 8 &&
                          keep->storage_offset() % 4 == 0 &&
                          int64_t(keep->storage().nbytes()) >= keep->storage_offset() + (keep->numel() + 3) / 4 * 4,
                      "keep must be the forward's [", kv_capacity(index), ", ", (H + 7) / 8, "] mask (got ",
                      keep->sizes(), ")");
  }
  at::Tensor dq = at::empty_like(q), dk = at::empty_like(k), dv = at::empty_like(v);
  at::Tensor dbias = need_dbias ? at::empty({idx.nnz, H}, q.options().dtype(at::kFloat))
                                : at::empty({0}, q.options().dtype(at::kFloat));
  at::Tensor rowstat = at::empty({idx.n_q, H, 2}, q.options().dtype(at::kFloat));
  const int64_t parts = bf_attn_partials_floats(&idx, int32_t(H), int32_t(hn));
  at::Tensor partials = at::empty({std::max<int64_t>(parts, 1)}, q.options().dtype(at::kFloat));
  check_rc(bf_attn_bwd(&idx, dtype_code(q), int32_t(H), int32_t(hn), float(score_clamp), q.data_ptr(), k.data_ptr(),
                       v.data_ptr(), b, f,
                       dropout_rate > 0.0 ? &drop : nullptr, Z.data_ptr<float>(), dout.data_ptr(), dq.data_ptr(),
                       dk.data_ptr(), dv.data_ptr(), need_dbias ? dbias.data_ptr<float>() : nullptr,
                       rowstat.data_ptr<float>(), partials.data_ptr<float>(), stream_of(q)),
           "bf::sparse_attn_bwd");
  return {dq, dk, dv, dbias};
}

// Typed-edge (Exphormer) attention: type_mod = E, float32 [2, H, hn]; the index's ids carry the types.
const float* type_mod_ptr(const at::Tensor& mod, int64_t H, int64_t hn, const at::Device& dev) {
  require(mod, "type_mod", at::kFloat, dev);
  TORCH_CHECK_VALUE(mod.numel() == 2 * H * hn && mod.size(0) == 2, "type_mod must be [2, ", H, ", ", hn, "] (got ",
                    mod.sizes(), ")");
  return mod.data_ptr<float>();
}

// Forward (bf_attn_fwd_typed): (out [n_q, H, hn] in q's dtype, Z [n_q, H] float32).
std::tuple<at::Tensor, at::Tensor> sparse_attn_fwd_typed(const at::Tensor& q, const at::Tensor& k,
                                                         const at::Tensor& v,
                                                         const c10::List<std::optional<at::Tensor>>& index,
                                                         at::IntArrayRef sizes, const at::Tensor& type_mod) {
  TORCH_CHECK_VALUE(q.is_cuda(), "q must be a device tensor (got ", q.device(), ")");
  const c10::DeviceGuard guard(q.device());
  const at::Device dev = q.device();
  const bf_attn_index idx = make_index(index, sizes, dev);
  check_qkv(q, k, v, idx);
  const int64_t H = q.size(1), hn = q.size(2);
  const float* mod = type_mod_ptr(type_mod, H, hn, dev);
  at::Tensor out = at::empty_like(q);
  at::Tensor Z = at::empty({idx.n_q, H}, q.options().dtype(at::kFloat));
  check_rc(bf_attn_fwd_typed(&idx, dtype_code(q), int32_t(H), int32_t(hn), q.data_ptr(), k.data_ptr(), v.data_ptr(),
                             mod, out.data_ptr(), Z.data_ptr<float>(), stream_of(q)),
           "bf::sparse_attn_fwd_typed");
  return {out, Z};
}

// Backward (bf_attn_bwd_typed): (dq, dk, dv, dtype_mod [2, H, hn] float32).
std::tuple<at::Tensor, at::Tensor, at::Tensor, at::Tensor> sparse_attn_bwd_typed(
    const at::Tensor& q, const at::Tensor& k, const at::Tensor& v, const c10::List<std::optional<at::Tensor>>& index,
    at::IntArrayRef sizes, const at::Tensor& type_mod, const at::Tensor& Z, const at::Tensor& dout) {
  TORCH_CHECK_VALUE(q.is_cuda(), "q must be a device tensor (got ", q.device(), ")");
  const c10::DeviceGuard guard(q.device());
  const at::Device dev = q.device();
  const bf_attn_index idx = make_index(index, sizes, dev);
  check_qkv(q, k, v, idx);
  const int64_t H = q.size(1), hn = q.size(2);
  const float* mod = type_mod_ptr(type_mod, H, hn, dev);
  require(dout, "dout", q.scalar_type(), dev);
  require(Z, "Z", at::kFloat, dev);
  TORCH_CHECK_VALUE(dout.sizes() == q.sizes() && Z.dim() == 2 && Z.size(0) == q.size(0) && Z.size(1) == H, "dout ",
                    dout.sizes(), " / Z ", Z.sizes(), " do not match q ", q.sizes());
  at::Tensor dq = at::empty_like(q), dk = at::empty_like(k), dv = at::empty_like(v);
  at::Tensor dmod = at::empty({2, H, hn}, q.options().dtype(at::kFloat));
  at::Tensor rowstat = at::empty({idx.n_q, H, 2}, q.options().dtype(at::kFloat));
  const int64_t parts = bf_attn_typed_partials_floats(&idx, dtype_code(q), int32_t(H), int32_t(hn));
  at::Tensor partials = at::empty({std::max<int64_t>(parts, 1)}, q.options().dtype(at::kFloat));
  check_rc(bf_attn_bwd_typed(&idx, dtype_code(q), int32_t(H), int32_t(hn), q.data_ptr(), k.data_ptr(), v.data_ptr(),
                             mod, Z.data_ptr<float>(), dout.data_ptr(), dq.data_ptr(), dk.data_ptr(), dv.data_ptr(),
                             dmod.data_ptr<float>(), rowstat.data_ptr<float>(), partials.data_ptr<float>(),
                             stream_of(q)),
           "bf::sparse_attn_bwd_typed");
  return {dq, dk, dv, dmod};
}

// ---------------------------------------------------------------- edge construction
// Walks (bf_random_walk): int64 [n_q * P, L + 1], walk q*P + p starting at query q_lo + q.
at::Tensor rw_walk(const at::Tensor& rowptr, const at::Tensor& col, int64_t q_lo, int64_t n_q, int64_t walks_per_node,
                   int64_t walk_length, int64_t philox_seed, int64_t philox_offset, const std::optional<at::Tensor>& u) {
  const c10::DeviceGuard guard(rowptr.device());
  const at::Device dev = rowptr.device();
  require(rowptr, "rowptr", at::kLong, dev);
  require(col, "col", at::kInt, dev);
  const float* up = opt_ptr<const float>(u, "u", at::kFloat, dev);
  if (up) TORCH_CHECK_VALUE(u->numel() == n_q * walks_per_node * walk_length, "u must be [", n_q * walks_per_node,
                            ", ", walk_length, "]");
  TORCH_CHECK_VALUE(n_q >= 0 && walks_per_node >= 1 && walk_length >= 0, "rw_walk: bad sizes");
  at::Tensor walks = at::empty({n_q * walks_per_node, walk_length + 1}, rowptr.options());
  check_rc(bf_random_walk(rowptr.data_ptr<int64_t>(), col.data_ptr<int32_t>(), rowptr.numel() - 1, q_lo, n_q,
                          int32_t(walks_per_node), int32_t(walk_length), up, uint64_t(philox_seed),
                          uint64_t(philox_offset), walks.data_ptr<int64_t>(), stream_of(rowptr)),
           "bf::rw_walk");
  return walks;
}

// Budgeted table (bf_build_edge_table): (table int32 [n_q, k_real + k_rw], row_len int32 [n_q]).
std::tuple<at::Tensor, at::Tensor> build_edge_table(
    const at::Tensor& rowptr, const at::Tensor& col, const std::optional<at::Tensor>& walk_rec,
    const at::Tensor& in_ptr, const at::Tensor& in_src, int64_t q_lo, int64_t n_q, int64_t walks_per_node,
    int64_t walk_length, int64_t k_real, int64_t k_rw, int64_t edge_seed, const std::optional<at::Tensor>& u,
    int64_t philox_seed, int64_t philox_offset, const std::optional<at::Tensor>& hubs, int64_t hub_threshold,
    const std::optional<at::Tensor>& heavy, int64_t light_max) {
  const c10::DeviceGuard guard(rowptr.device());
  const at::Device dev = rowptr.device();
  require(rowptr, "rowptr", at::kLong, dev);
  require(col, "col", at::kInt, dev);
  require(in_ptr, "in_ptr", at::kLong, dev);
  require(in_src, "in_src", at::kInt, dev);
  const void* rec = opt_ptr<const void>(walk_rec, "walk_rec", at::kInt, dev);
  if (rec) TORCH_CHECK_VALUE(walk_rec->numel() == 4 * col.numel(), "walk_rec must be [", col.numel(), ", 4]");
  const float* up = opt_ptr<const float>(u, "u", at::kFloat, dev);
  if (up) TORCH_CHECK_VALUE(u->numel() == n_q * walks_per_node * walk_length, "u must be [", n_q * walks_per_node,
                            ", ", walk_length, "]");
  const int32_t* hp = opt_ptr<const int32_t>(hubs, "hubs", at::kInt, dev);
  const int32_t* vp = opt_ptr<const int32_t>(heavy, "heavy", at::kInt, dev);
  const int64_t n_hubs = hp ? hubs->numel() : 0, n_heavy = vp ? heavy->numel() : 0;
  // with light_max >= 0 the light kernel leaves rows above it to the heavy list: it must be given (it may be empty)
  TORCH_CHECK_VALUE(light_max < 0 || (heavy.has_value() && heavy->defined()), "light_max >= 0 needs the heavy-query list");
  const int64_t width = std::max<int64_t>(k_real, 0) + std::max<int64_t>(k_rw, 0);
  at::Tensor table = at::empty({n_q, width}, in_src.options());
  at::Tensor row_len = at::empty({n_q}, in_src.options());
  size_t ws_bytes = 0;
  check_rc(bf_build_edge_table_workspace_size(n_q, int32_t(std::max<int64_t>(k_rw, 0)), n_hubs,
                                              int32_t(std::max<int64_t>(k_real, 0)), &ws_bytes),
           "bf::build_edge_table");
  at::Tensor ws = scratch_bytes(ws_bytes, dev);
  check_rc(bf_build_edge_table(rowptr.data_ptr<int64_t>(), col.data_ptr<int32_t>(), rec, in_ptr.data_ptr<int64_t>(),
                               in_src.data_ptr<int32_t>(), rowptr.numel() - 1, col.numel(), q_lo, n_q,
                               int32_t(walks_per_node), int32_t(walk_length), int32_t(k_real), int32_t(k_rw),
                               edge_seed, up, uint64_t(philox_seed), uint64_t(philox_offset), hp, n_hubs,
                               hub_threshold, vp, n_heavy, light_max, table.data_ptr<int32_t>(),
                               row_len.data_ptr<int32_t>(), ws.data_ptr(), size_t(ws.numel()), stream_of(rowptr)),
           "bf::build_edge_table");
  return {table, row_len};
}

// Query-major table -> attention CSR (bf_table_csr_ptr + bf_table_to_csr): (qptr int64 [n_q + 1], kv int32 [nnz]).
// token_row as in the C ABI (< 0: no token row); reads nnz to the host once. With id_limit >= 0 the table is
// validated on the device first (bf_check_table: row lengths in [0, width], ids in [0, id_limit)).
std::tuple<at::Tensor, at::Tensor> table_to_csr(const at::Tensor& table, const at::Tensor& row_len, bool global_token,
                                                int64_t token_row, int64_t id_limit) {
  const c10::DeviceGuard guard(table.device());
  const at::Device dev = table.device();
  require(table, "table", at::kInt, dev);
  require(row_len, "row_len", at::kInt, dev);
  TORCH_CHECK_VALUE(table.dim() == 2 && row_len.dim() == 1 && row_len.size(0) == table.size(0),
                    "table must be [n, width] and row_len [n]");
  const int64_t n_rows = table.size(0);
  if (id_limit >= 0) {
    at::Tensor bad = at::empty({2}, table.options().dtype(at::kLong));
    check_rc(bf_check_table(table.data_ptr<int32_t>(), row_len.data_ptr<int32_t>(), n_rows, int32_t(table.size(1)),
                            id_limit, nullptr, bad.data_ptr(), 16, stream_of(table)),
             "bf::table_to_csr");
  }
  const int64_t lead = (global_token && token_row >= 0) ? 1 : 0;
  const int64_t n_q = n_rows + lead;
  size_t ws_bytes = 0;
  check_rc(bf_scan_workspace_size(n_q, &ws_bytes), "bf::table_to_csr");
  at::Tensor ws = scratch_bytes(ws_bytes, dev);
  at::Tensor qptr = at::empty({n_q + 1}, table.options().dtype(at::kLong));
  int64_t nnz = 0;
  void* st = stream_of(table);
  check_rc(bf_table_csr_ptr(row_len.data_ptr<int32_t>(), n_rows, global_token ? 1 : 0, token_row,
                            qptr.data_ptr<int64_t>(), &nnz, ws.data_ptr(), size_t(ws.numel()), st),
           "bf::table_to_csr");
  at::Tensor kv = at::empty({nnz}, table.options());
  check_rc(bf_table_to_csr(table.data_ptr<int32_t>(), row_len.data_ptr<int32_t>(), n_rows, int32_t(table.size(1)),
                           global_token ? 1 : 0, token_row, qptr.data_ptr<int64_t>(), kv.data_ptr<int32_t>(), nullptr,
                           0, 0, st),
           "bf::table_to_csr");
  return {qptr, kv};
}

// Key-major view of an attention CSR (bf_reverse_index): (kptr int64 [n_kv + 1], kq int32 [nnz], ks int32 [nnz]:
// each entry's query and its slot in the query's row), entries of a key in CSR order.
std::tuple<at::Tensor, at::Tensor, at::Tensor> transpose_table(const at::Tensor& qptr, const at::Tensor& kv,
                                                               int64_t n_kv) {
  const c10::DeviceGuard guard(qptr.device());
  const at::Device dev = qptr.device();
  require(qptr, "qptr", at::kLong, dev);
  require(kv, "kv", at::kInt, dev);
  const int64_t nnz = kv.numel();
  size_t ws_bytes = 0;
  check_rc(bf_reverse_index_workspace_size(nnz, n_kv, &ws_bytes), "bf::transpose_table");
  at::Tensor ws = scratch_bytes(ws_bytes, dev);
  at::Tensor kptr = at::empty({n_kv + 1}, qptr.options());
  at::Tensor kq = at::empty({nnz}, kv.options()), ks = at::empty({nnz}, kv.options());
  check_rc(bf_reverse_index(qptr.data_ptr<int64_t>(), kv.data_ptr<int32_t>(), qptr.numel() - 1, n_kv, nnz,
                            kptr.data_ptr<int64_t>(), kq.data_ptr<int32_t>(), ks.data_ptr<int32_t>(), ws.data_ptr(),
                            size_t(ws.numel()), stream_of(qptr)),
           "bf::transpose_table");
  return {kptr, kq, ks};
}

// ---------------------------------------------------------------- index builds
// An index's build is a row of short launches: at small graphs the host's calls are what it costs. Each side of the
// index is one operator, so that its launches and allocations follow each other without Python between them
// (4096 nodes, B=16: a training step with its table and index build 456 -> 385 us).

// A split plan's arrays in one buffer: (nitems [n_rows], item_off [n_rows], item_row [items], heavy_rows [rows]).
struct PlanArrays {
  int64_t item_cap, heavy_cap;
  at::Tensor nitems, item_off, item_row, heavy_rows;
  PlanArrays(int64_t n_rows, int64_t nnz, int64_t threshold, int64_t item, const at::TensorOptions& opt)
      : item_cap(bf_split_item_capacity(nnz, threshold, item)), heavy_cap(bf_split_row_capacity(nnz, threshold)) {
    const int64_t r = std::max<int64_t>(n_rows, 1), i = std::max<int64_t>(item_cap, 1);
    const at::Tensor buf = at::empty({2 * r + i + std::max<int64_t>(heavy_cap, 1)}, opt);
    nitems = buf.narrow(0, 0, r);
    item_off = buf.narrow(0, r, r);
    item_row = buf.narrow(0, 2 * r, i);
    heavy_rows = buf.narrow(0, 2 * r + i, std::max<int64_t>(heavy_cap, 1));
  }
};

// `n` entries of storage for at least one (an empty array still has an address).
at::Tensor entries_of(int64_t n, const at::TensorOptions& opt) {
  at::Tensor t = at::empty({std::max<int64_t>(n, 1)}, opt);
  return n > 0 ? t : t.narrow(0, 0, 0);
}

// The query side of a table's index at its capacity `nnz` (every row full), nothing read back: bf_table_csr_ptr,
// bf_split_plan_first_row and bf_table_to_csr. Returns (qptr, kv, sort keys, nitems, item_off, item_row, heavy_rows).
// plan_items: items of the token row, the only row that may be split; counts: int32, its first two are written.
std::vector<at::Tensor> table_index(const at::Tensor& table, const at::Tensor& row_len, bool global_token,
                                    int64_t token_row, int64_t nnz, int64_t n_keys, int64_t q_bits, int64_t slot_bits,
                                    int64_t plan_items, int64_t chunk, int64_t item, const at::Tensor& counts) {
  const c10::DeviceGuard guard(table.device());
  const at::Device dev = table.device();
  require(table, "table", at::kInt, dev);
  require(row_len, "row_len", at::kInt, dev);
  require(counts, "counts", at::kInt, dev);
  TORCH_CHECK_VALUE(table.dim() == 2 && row_len.numel() >= table.size(0), "table must be [n, width] and row_len [n]");
  const int64_t n_rows = table.size(0), width = table.size(1);
  const int64_t tr = global_token ? std::max<int64_t>(token_row, -1) : -1;
  const int64_t n_q = n_rows + (tr >= 0 ? 1 : 0);
  TORCH_CHECK_VALUE(counts.numel() >= 2, "counts must hold two numbers");
  TORCH_CHECK_VALUE(nnz >= n_rows * width + (global_token ? n_rows : 0) + std::max<int64_t>(tr, 0) &&
                        n_keys >= n_rows * width,
                    "nnz and n_keys must be the table's capacity");
  const at::TensorOptions i32 = table.options(), i64 = i32.dtype(at::kLong);
  void* st = stream_of(table);
  const char* op = "bf::table_index";

  size_t ws_bytes = 0;
  check_rc(bf_scan_workspace_size(n_q, &ws_bytes), op);
  const at::Tensor ws = scratch_bytes(ws_bytes, dev);
  at::Tensor qptr = at::empty({n_q + 1}, i64);
  check_rc(bf_table_csr_ptr(row_len.data_ptr<int32_t>(), n_rows, global_token ? 1 : 0, tr, qptr.data_ptr<int64_t>(),
                            nullptr, ws.data_ptr(), size_t(ws.numel()), st),
           op);
  PlanArrays p(n_q, nnz, chunk, item, i32);
  check_rc(bf_split_plan_first_row(n_q, plan_items, p.nitems.data_ptr<int32_t>(), p.item_off.data_ptr<int32_t>(),
                                   p.item_row.data_ptr<int32_t>(), p.item_cap, p.heavy_rows.data_ptr<int32_t>(),
                                   p.heavy_cap, counts.data_ptr<int32_t>(), st),
           op);
  at::Tensor kv = entries_of(nnz, i32), keys = entries_of(n_keys, i64);
  check_rc(bf_table_to_csr(table.data_ptr<int32_t>(), row_len.data_ptr<int32_t>(), n_rows, int32_t(width),
                           global_token ? 1 : 0, tr, qptr.data_ptr<int64_t>(), static_cast<int32_t*>(kv.data_ptr()),
                           static_cast<uint64_t*>(keys.data_ptr()), int32_t(q_bits), int32_t(slot_bits), st),
           op);
  return {qptr, kv, keys, p.nitems, p.item_off, p.item_row, p.heavy_rows};
}

// The key side from the query side's sort keys: bf_reverse_index_packed and bf_row_order_and_plan. Returns (kptr, kq,
// sorted keys, order, spans, nitems, item_off, item_row, heavy_rows) and, with `entries`, ks.
std::vector<at::Tensor> reverse_index_and_plan(const at::Tensor& keys, const at::Tensor& qptr, int64_t nnz,
                                               int64_t n_kv, int64_t q_bits, int64_t slot_bits, bool global_token,
                                               int64_t token_row, bool entries, int64_t chunk, int64_t item,
                                               const at::Tensor& counts) {
  const c10::DeviceGuard guard(qptr.device());
  const at::Device dev = qptr.device();
  require(keys, "keys", at::kLong, dev);
  require(qptr, "qptr", at::kLong, dev);
  require(counts, "counts", at::kInt, dev);
  const int64_t n_q = qptr.numel() - 1;
  const int64_t own = global_token ? n_q - (token_row >= 0 ? 1 : 0) + std::max<int64_t>(token_row, 0) : 0;
  TORCH_CHECK_VALUE(counts.numel() >= 2, "counts must hold two numbers");
  TORCH_CHECK_VALUE(n_q >= 0 && n_kv >= 0 && nnz == keys.numel() + own, "nnz must be the keys and the token's entries");
  const at::TensorOptions i64 = qptr.options(), i32 = counts.options();
  void* st = stream_of(qptr);
  const char* op = "bf::reverse_index_and_plan";

  size_t ws_bytes = 0;
  check_rc(bf_reverse_index_packed_workspace_size(nnz, &ws_bytes), op);
  at::Tensor ws = scratch_bytes(ws_bytes, dev);
  at::Tensor sorted = entries_of(keys.numel(), i64), kptr = at::empty({n_kv + 1}, i64), kq = entries_of(nnz, i32), ks;
  if (entries) ks = entries_of(nnz, i32);
  check_rc(bf_reverse_index_packed(static_cast<const uint64_t*>(keys.data_ptr()), qptr.data_ptr<int64_t>(), nnz,
                                   n_q, n_kv, int32_t(q_bits), int32_t(slot_bits), global_token ? 1 : 0, token_row,
                                   static_cast<uint64_t*>(sorted.data_ptr()), kptr.data_ptr<int64_t>(),
                                   static_cast<int32_t*>(kq.data_ptr()),
                                   entries ? static_cast<int32_t*>(ks.data_ptr()) : nullptr, ws.data_ptr(),
                                   size_t(ws.numel()), st),
           op);
  ws.reset();                                 // the sort's scratch is free for what follows
  const int64_t r = std::max<int64_t>(n_kv, 1);
  PlanArrays p(n_kv, nnz, chunk, item, i32);
  check_rc(bf_row_order_and_plan_workspace_size(n_kv, p.heavy_cap, &ws_bytes), op);
  ws = scratch_bytes(ws_bytes, dev);
  at::Tensor order = at::empty({r}, i32), spans = at::empty({r}, i64);
  check_rc(bf_row_order_and_plan(kptr.data_ptr<int64_t>(), n_kv, chunk, item, order.data_ptr<int32_t>(),
                                 static_cast<uint64_t*>(spans.data_ptr()), p.nitems.data_ptr<int32_t>(),
                                 p.item_off.data_ptr<int32_t>(), p.item_row.data_ptr<int32_t>(), p.item_cap,
                                 p.heavy_rows.data_ptr<int32_t>(), p.heavy_cap, counts.data_ptr<int32_t>(),
                                 ws.data_ptr(), size_t(ws.numel()), st),
           op);
  std::vector<at::Tensor> out{kptr, kq, sorted, order, spans, p.nitems, p.item_off, p.item_row, p.heavy_rows};
  if (entries) out.push_back(ks);
  return out;
}

// ---------------------------------------------------------------- operators over packed sequences
// What each row sees (bf_packed_spans): (row_span int32 [n_q, 2], key_span int32 [n_k, 2], positions int32 [n_q]).
std::tuple<at::Tensor, at::Tensor, at::Tensor> packed_spans(const at::Tensor& q_offsets, const at::Tensor& k_offsets,
                                                            int64_t n_q, int64_t n_k, bool causal) {
  const c10::DeviceGuard guard(q_offsets.device());
  const at::Device dev = q_offsets.device();
  require(q_offsets, "q_offsets", at::kInt, dev);
  require(k_offsets, "k_offsets", at::kInt, dev);
  TORCH_CHECK_VALUE(q_offsets.dim() == 1 && q_offsets.sizes() == k_offsets.sizes() && q_offsets.numel() >= 1,
                    "offsets must be [n_seq + 1] each (got ", q_offsets.sizes(), " and ", k_offsets.sizes(), ")");
  TORCH_CHECK_VALUE(n_q >= 0 && n_k >= 0, "packed_spans: bad sizes");
  at::Tensor row_span = at::empty({n_q, 2}, q_offsets.options()), key_span = at::empty({n_k, 2}, q_offsets.options());
  at::Tensor positions = at::empty({n_q}, q_offsets.options());
  check_rc(bf_packed_spans(q_offsets.data_ptr<int32_t>(), k_offsets.data_ptr<int32_t>(), q_offsets.numel() - 1, n_q, n_k,
                           causal ? 1 : 0, row_span.data_ptr<int32_t>(), key_span.data_ptr<int32_t>(),
                           positions.data_ptr<int32_t>(), stream_of(q_offsets)),
           "bf::packed_spans");
  return {row_span, key_span, positions};
}

// A [rows, heads, dim] tensor as the kernels read it: a contiguous last dimension, rows and heads at whole 16-byte steps.
// Views that are so (slices of a fused projection, heads expanded) are taken as they are, others are copied.
at::Tensor as_rows(const at::Tensor& t, const char* name) {
  TORCH_CHECK_VALUE(t.dim() == 3, name, " must be [rows, heads, head_dim] (got ", t.sizes(), ")");
  const int64_t per = 16 / t.element_size();
  bool fits = reinterpret_cast<uintptr_t>(t.data_ptr()) % 16 == 0 && (t.size(2) <= 1 || t.stride(2) == 1);
  for (int d = 0; d < 2; ++d) fits = fits && (t.size(d) <= 1 || t.stride(d) % per == 0);
  return fits ? t : t.clone(at::MemoryFormat::Contiguous);
}

// A contiguous tensor at a 16-byte aligned address.
at::Tensor as_dense(const at::Tensor& t) {
  return t.is_contiguous() && reinterpret_cast<uintptr_t>(t.data_ptr()) % 16 == 0 ? t : t.clone(at::MemoryFormat::Contiguous);
}

// A [rows, heads, dim] tensor with a contiguous last dimension; its strides of a row and of a head in values. Strides of
// dimensions of one entry do not matter and are given as 0.
void require_heads(const at::Tensor& t, const char* name, at::ScalarType st, const at::Device& dev, int64_t (&stride)[2]) {
  TORCH_CHECK_VALUE(t.device() == dev, name, " is on ", t.device(), ", expected ", dev);
  TORCH_CHECK_VALUE(t.scalar_type() == st, name, " must be ", st, " (got ", t.scalar_type(), ")");
  TORCH_CHECK_VALUE(t.dim() == 3, name, " must be [rows, heads, head_dim] (got ", t.sizes(), ")");
  TORCH_CHECK_VALUE(t.stride(2) == 1 || t.size(2) <= 1, name, " must be contiguous along the head (strides ", t.strides(),
                    ")");
  stride[0] = t.size(0) > 1 ? t.stride(0) : 0;
  stride[1] = t.size(1) > 1 ? t.stride(1) : 0;
}

void require_span(const at::Tensor& t, const char* name, int64_t n, const at::Device& dev) {
  require(t, name, at::kInt, dev);
  TORCH_CHECK_VALUE(t.dim() == 2 && t.size(0) == n && t.size(1) == 2, name, " must be [", n, ", 2] (got ", t.sizes(), ")");
}

bf_packed_attn packed_args(const at::Tensor& q, const at::Tensor& k, const at::Tensor& v, const at::Tensor& row_span,
                           double scale, int64_t longest) {
  const at::Device dev = q.device();
  bf_packed_attn p{};
  p.dtype = dtype_code(q);
  require_heads(q, "q", q.scalar_type(), dev, p.q_stride);
  require_heads(k, "k", q.scalar_type(), dev, p.k_stride);
  require_heads(v, "v", q.scalar_type(), dev, p.v_stride);
  TORCH_CHECK_VALUE(k.sizes() == v.sizes() && q.size(2) == k.size(2), "q ", q.sizes(), ", k ", k.sizes(), ", v ", v.sizes(),
                    " disagree");
  TORCH_CHECK_VALUE(q.size(1) < (int64_t(1) << 31) && k.size(1) < (int64_t(1) << 31) && q.size(2) < (int64_t(1) << 31),
                    "too many heads");
  p.n_q = q.size(0), p.n_k = k.size(0);
  p.heads_q = int32_t(q.size(1)), p.heads_k = int32_t(k.size(1)), p.head_dim = int32_t(q.size(2));
  require_span(row_span, "row_span", p.n_q, dev);
  p.row_span = row_span.data_ptr<int32_t>();
  p.scale = float(scale);
  p.longest = int32_t(std::min<int64_t>(std::max<int64_t>(longest, 0), INT32_MAX));
  return p;
}

// A learned bias by buckets of the relative position: table float32 [heads_q, buckets], map int32 [2 reach + 1], the rows' positions.
struct BiasIn {
  at::Tensor table, map, positions;
};

bf_packed_bias bias_args(const BiasIn& b, const bf_packed_attn& p, const at::Device& dev) {
  bf_packed_bias r{};
  require(b.table, "bias", at::kFloat, dev);
  TORCH_CHECK_VALUE(b.table.dim() == 2 && b.table.size(0) == p.heads_q && b.table.size(1) < (int64_t(1) << 30), "bias must be [", p.heads_q,
                    ", buckets] (got ", b.table.sizes(), ")");
  require(b.map, "map", at::kInt, dev);
  TORCH_CHECK_VALUE(b.map.dim() == 1 && b.map.size(0) % 2 == 1 && b.map.size(0) < (int64_t(1) << 30), "map must be [2 reach + 1] (got ",
                    b.map.sizes(), ")");
  require(b.positions, "positions", at::kInt, dev);
  TORCH_CHECK_VALUE(b.positions.dim() == 1 && b.positions.size(0) == p.n_q, "positions must be [", p.n_q, "] (got ", b.positions.sizes(), ")");
  r.table = b.table.data_ptr<float>(), r.map = b.map.data_ptr<int32_t>(), r.positions = b.positions.data_ptr<int32_t>();
  r.buckets = int32_t(b.table.size(1)), r.reach = int32_t(b.map.size(0) / 2);
  return r;
}

// Forward (bf_packed_attn_fwd, bf_packed_attn_bias_fwd): (out [n_q, heads_q, head_dim], lse float32 [n_q, heads_q], in log2,
// rest). With `train`, rest is what the backward reads beside out (empty where it needs nothing).
std::tuple<at::Tensor, at::Tensor, at::Tensor> attn_fwd(const at::Tensor& q_in, const at::Tensor& k_in, const at::Tensor& v_in,
                                                        const at::Tensor& row_span, double scale, int64_t longest, bool train,
                                                        const BiasIn* bias_in) {
  TORCH_CHECK_VALUE(q_in.is_cuda(), "q must be a device tensor (got ", q_in.device(), ")");
  const c10::DeviceGuard guard(q_in.device());
  const at::Tensor q = as_rows(q_in, "q");
  const at::Tensor k = as_rows(k_in, "k");
  const at::Tensor v = as_rows(v_in, "v");
  const bf_packed_attn p = packed_args(q, k, v, row_span, scale, longest);
  at::Tensor out = at::empty(q.sizes(), q.options().memory_format(at::MemoryFormat::Contiguous));
  at::Tensor lse = at::empty({q.size(0), q.size(1)}, q.options().dtype(at::kFloat));
  bf_packed_bias bias{};
  if (bias_in) bias = bias_args(*bias_in, p, q.device());
  const int64_t floats = bias_in ? bf_packed_attn_bias_fwd_floats(&p, &bias) : bf_packed_attn_fwd_floats(&p);
  const bool keeps = train && (bias_in ? bf_packed_attn_bias_rest(&p, &bias) : bf_packed_attn_rest(&p));
  at::Tensor scratch, rest = keeps ? at::empty_like(out) : at::empty({0}, out.options());
  if (floats > 0) scratch = at::empty({floats}, lse.options());
  void* rp = keeps ? rest.data_ptr() : nullptr;
  float* sp = floats > 0 ? scratch.data_ptr<float>() : nullptr;
  if (bias_in)
    check_rc(bf_packed_attn_bias_fwd(&p, &bias, q.data_ptr(), k.data_ptr(), v.data_ptr(), out.data_ptr(), rp, lse.data_ptr<float>(), sp,
                                     stream_of(q)),
             "bf::packed_attn_bias_fwd");
  else
    check_rc(bf_packed_attn_fwd(&p, q.data_ptr(), k.data_ptr(), v.data_ptr(), out.data_ptr(), rp, lse.data_ptr<float>(), sp, stream_of(q)),
             "bf::packed_attn_fwd");
  return {out, lse, rest};
}

std::tuple<at::Tensor, at::Tensor, at::Tensor> packed_attn_fwd(const at::Tensor& q, const at::Tensor& k, const at::Tensor& v,
                                                               const at::Tensor& row_span, double scale, int64_t longest, bool train) {
  return attn_fwd(q, k, v, row_span, scale, longest, train, nullptr);
}

std::tuple<at::Tensor, at::Tensor, at::Tensor> packed_attn_bias_fwd(const at::Tensor& q, const at::Tensor& k, const at::Tensor& v,
                                                                    const at::Tensor& bias, const at::Tensor& map,
                                                                    const at::Tensor& positions, const at::Tensor& row_span, double scale,
                                                                    int64_t longest, bool train) {
  const BiasIn b{bias, map, positions};
  return attn_fwd(q, k, v, row_span, scale, longest, train, &b);
}

// Backward (bf_packed_attn_bwd, bf_packed_attn_bias_bwd): (dq, dk, dv, dbias or undefined), contiguous.
std::tuple<at::Tensor, at::Tensor, at::Tensor, at::Tensor> attn_bwd(const at::Tensor& q_in, const at::Tensor& k_in, const at::Tensor& v_in,
                                                                    const at::Tensor& row_span, const at::Tensor& key_span,
                                                                    const at::Tensor& out, const at::Tensor& lse,
                                                                    const at::Tensor& dout_in, double scale, int64_t longest,
                                                                    const std::optional<at::Tensor>& rest, const BiasIn* bias_in) {
  TORCH_CHECK_VALUE(q_in.is_cuda(), "q must be a device tensor (got ", q_in.device(), ")");
  const c10::DeviceGuard guard(q_in.device());
  const at::Tensor q = as_rows(q_in, "q");
  const at::Tensor k = as_rows(k_in, "k");
  const at::Tensor v = as_rows(v_in, "v");
  const at::Tensor dout = as_dense(dout_in);
  const at::Device dev = q.device();
  bf_packed_attn p = packed_args(q, k, v, row_span, scale, longest);
  require_span(key_span, "key_span", p.n_k, dev);
  p.key_span = key_span.data_ptr<int32_t>();
  require(out, "out", q.scalar_type(), dev);
  require(dout, "dout", q.scalar_type(), dev);
  require(lse, "lse", at::kFloat, dev);
  TORCH_CHECK_VALUE(out.sizes() == q.sizes() && dout.sizes() == q.sizes() && lse.numel() == q.size(0) * q.size(1), "out ",
                    out.sizes(), ", dout ", dout.sizes(), " or lse ", lse.sizes(), " do not match q ", q.sizes());
  const void* rp = nullptr;
  if (rest.has_value() && rest->defined() && rest->numel() > 0) {
    require(*rest, "rest", q.scalar_type(), dev);
    TORCH_CHECK_VALUE(rest->sizes() == q.sizes(), "rest ", rest->sizes(), " does not match q ", q.sizes());
    rp = rest->data_ptr();
  }
  const auto plain = q.options().memory_format(at::MemoryFormat::Contiguous);
  at::Tensor dq = at::empty(q.sizes(), plain), dk = at::empty(k.sizes(), plain), dv = at::empty(v.sizes(), plain);
  at::Tensor delta = at::empty_like(lse), scratch, dbias;
  bf_packed_bias bias{};
  if (bias_in) {
    bias = bias_args(*bias_in, p, dev);
    dbias = at::empty_like(bias_in->table);
  }
  const int64_t floats = bias_in ? bf_packed_attn_bias_bwd_floats(&p, &bias) : bf_packed_attn_bwd_floats(&p);
  if (floats > 0) scratch = at::empty({floats}, lse.options());
  float* sp = floats > 0 ? scratch.data_ptr<float>() : nullptr;
  if (bias_in)
    check_rc(bf_packed_attn_bias_bwd(&p, &bias, q.data_ptr(), k.data_ptr(), v.data_ptr(), out.data_ptr(), rp, lse.data_ptr<float>(),
                                     dout.data_ptr(), dq.data_ptr(), dk.data_ptr(), dv.data_ptr(), dbias.data_ptr<float>(),
                                     delta.data_ptr<float>(), sp, stream_of(q)),
             "bf::packed_attn_bias_bwd");
  else
    check_rc(bf_packed_attn_bwd(&p, q.data_ptr(), k.data_ptr(), v.data_ptr(), out.data_ptr(), rp, lse.data_ptr<float>(), dout.data_ptr(),
                                dq.data_ptr(), dk.data_ptr(), dv.data_ptr(), delta.data_ptr<float>(), sp, stream_of(q)),
             "bf::packed_attn_bwd");
  return {dq, dk, dv, dbias};
}

std::tuple<at::Tensor, at::Tensor, at::Tensor> packed_attn_bwd(const at::Tensor& q, const at::Tensor& k, const at::Tensor& v,
                                                               const at::Tensor& row_span, const at::Tensor& key_span,
                                                               const at::Tensor& out, const at::Tensor& lse, const at::Tensor& dout,
                                                               double scale, int64_t longest, const std::optional<at::Tensor>& rest) {
  auto [dq, dk, dv, dbias] = attn_bwd(q, k, v, row_span, key_span, out, lse, dout, scale, longest, rest, nullptr);
  return {dq, dk, dv};
}

std::tuple<at::Tensor, at::Tensor, at::Tensor, at::Tensor> packed_attn_bias_bwd(
    const at::Tensor& q, const at::Tensor& k, const at::Tensor& v, const at::Tensor& bias, const at::Tensor& map,
    const at::Tensor& positions, const at::Tensor& row_span, const at::Tensor& key_span, const at::Tensor& out, const at::Tensor& lse,
    const at::Tensor& dout, double scale, int64_t longest, const std::optional<at::Tensor>& rest) {
  const BiasIn b{bias, map, positions};
  return attn_bwd(q, k, v, row_span, key_span, out, lse, dout, scale, longest, rest, &b);
}

// Rotary positions (bf_rotary) of x and, if given, y: new contiguous tensors.
std::tuple<at::Tensor, at::Tensor> rotary(const at::Tensor& x_in, const std::optional<at::Tensor>& y_in, const at::Tensor& positions,
                                          const at::Tensor& turns, double amplitude, bool interleaved, bool inverse) {
  TORCH_CHECK_VALUE(x_in.is_cuda(), "x must be a device tensor (got ", x_in.device(), ")");
  const c10::DeviceGuard guard(x_in.device());
  const auto along = [](const at::Tensor& t) {       // contiguous along the head; other strides are taken as they are
    return t.dim() != 3 || t.size(2) <= 1 || t.stride(2) == 1 ? t : t.clone(at::MemoryFormat::Contiguous);
  };
  const at::Tensor x = along(x_in);
  std::optional<at::Tensor> y;
  if (y_in.has_value() && y_in->defined()) y = along(*y_in);
  const at::Device dev = x.device();
  const bool two = y.has_value() && y->defined();
  int64_t xs[2], ys[2] = {0, 0};
  require_heads(x, "x", x.scalar_type(), dev, xs);
  if (two) {
    require_heads(*y, "y", x.scalar_type(), dev, ys);
    TORCH_CHECK_VALUE(y->size(0) == x.size(0) && y->size(2) == x.size(2), "x ", x.sizes(), " and y ", y->sizes(), " disagree");
  }
  TORCH_CHECK_VALUE(positions.scalar_type() == at::kInt || positions.scalar_type() == at::kLong,
                    "positions must be int32 or int64 (got ", positions.scalar_type(), ")");
  require(positions, "positions", positions.scalar_type(), dev);
  TORCH_CHECK_VALUE(positions.dim() == 1 && positions.size(0) == x.size(0), "positions must be [", x.size(0), "] (got ",
                    positions.sizes(), ")");
  require(turns, "turns", at::kDouble, dev);
  TORCH_CHECK_VALUE(turns.dim() == 1, "turns must be [rot / 2]");
  for (int64_t n : {x.size(1), x.size(2), two ? y->size(1) : 0, turns.size(0)})
    TORCH_CHECK_VALUE(n < (int64_t(1) << 30), "rotary: bad sizes");
  const auto plain = x.options().memory_format(at::MemoryFormat::Contiguous);
  at::Tensor ox = at::empty(x.sizes(), plain), oy = two ? at::empty(y->sizes(), plain) : at::empty({0}, plain);
  const int32_t code = dtype_code(x);
  // a y of no heads is no y
  const bool y_heads = two && y->size(1) > 0;
  check_rc(bf_rotary(x.data_ptr(), y_heads ? y->data_ptr() : nullptr, x.size(0), int32_t(x.size(1)),
                     y_heads ? int32_t(y->size(1)) : 0, int32_t(x.size(2)), int32_t(2 * turns.size(0)), code, xs, ys,
                     positions.data_ptr(), positions.scalar_type() == at::kLong, turns.data_ptr<double>(), float(amplitude),
                     interleaved ? 1 : 0, inverse ? 1 : 0, ox.data_ptr(), y_heads ? oy.data_ptr() : nullptr, stream_of(x)),
           "bf::rotary");
  return {ox, oy};
}

bf_linear_attn linear_args(const at::Tensor& q, const at::Tensor& k, const at::Tensor& v, const at::Tensor& log_decay,
                           const at::Tensor& row_span, const at::Tensor& key_span, const at::Tensor& offsets, double scale,
                           int64_t longest, const std::optional<at::Tensor>& init_state) {
  const at::Device dev = q.device();
  bf_linear_attn p{};
  p.dtype = dtype_code(q);
  require_heads(q, "q", q.scalar_type(), dev, p.q_stride);
  require_heads(k, "k", q.scalar_type(), dev, p.k_stride);
  require_heads(v, "v", q.scalar_type(), dev, p.v_stride);
  TORCH_CHECK_VALUE(q.sizes() == k.sizes() && v.size(0) == q.size(0) && v.size(1) == q.size(1), "q ", q.sizes(), ", k ",
                    k.sizes(), ", v ", v.sizes(), " disagree");
  TORCH_CHECK_VALUE(q.size(1) < (int64_t(1) << 30) && q.size(2) < (int64_t(1) << 30) && v.size(2) < (int64_t(1) << 30),
                    "linear_attn: bad sizes");
  const int64_t T = q.size(0), H = q.size(1), dk = q.size(2), dv = v.size(2);
  require(log_decay, "log_decay", at::kFloat, dev);
  TORCH_CHECK_VALUE(log_decay.dim() == 1 && log_decay.size(0) == H, "log_decay must be [", H, "] (got ", log_decay.sizes(), ")");
  require_span(row_span, "row_span", T, dev);
  require_span(key_span, "key_span", T, dev);
  require(offsets, "offsets", at::kInt, dev);
  TORCH_CHECK_VALUE(offsets.dim() == 1 && offsets.numel() >= 1, "offsets must be [n_seq + 1]");
  p.n = T, p.n_seq = offsets.numel() - 1, p.heads = int32_t(H), p.dim_k = int32_t(dk), p.dim_v = int32_t(dv);
  p.row_span = row_span.data_ptr<int32_t>(), p.key_span = key_span.data_ptr<int32_t>();
  p.offsets = offsets.data_ptr<int32_t>(), p.log_decay = log_decay.data_ptr<float>();
  p.scale = float(scale);
  p.longest = int32_t(std::min<int64_t>(std::max<int64_t>(longest, 0), INT32_MAX));
  if (init_state.has_value() && init_state->defined()) {
    require(*init_state, "init_state", at::kFloat, dev);
    TORCH_CHECK_VALUE(init_state->sizes() == at::IntArrayRef({p.n_seq, H, dk, dv}), "init_state must be [", p.n_seq, ", ", H,
                      ", ", dk, ", ", dv, "] (got ", init_state->sizes(), ")");
    p.init = init_state->data_ptr<float>();
  }
  return p;
}

// Forward (bf_linear_attn_fwd): (out, final state float32 [n_seq, heads, dim_k, dim_v], or empty without return_state).
std::tuple<at::Tensor, at::Tensor> linear_attn_fwd(const at::Tensor& q_in, const at::Tensor& k_in, const at::Tensor& v_in,
                                                   const at::Tensor& log_decay, const at::Tensor& row_span,
                                                   const at::Tensor& key_span, const at::Tensor& offsets, double scale,
                                                   int64_t longest, const std::optional<at::Tensor>& init_state,
                                                   bool return_state) {
  TORCH_CHECK_VALUE(q_in.is_cuda(), "q must be a device tensor (got ", q_in.device(), ")");
  const c10::DeviceGuard guard(q_in.device());
  const at::Tensor q = as_rows(q_in, "q");
  const at::Tensor k = as_rows(k_in, "k");
  const at::Tensor v = as_rows(v_in, "v");
  bf_linear_attn p = linear_args(q, k, v, log_decay, row_span, key_span, offsets, scale, longest, init_state);
  at::Tensor out = at::empty(v.sizes(), v.options().memory_format(at::MemoryFormat::Contiguous)), scratch;
  at::Tensor state = return_state ? at::empty({p.n_seq, p.heads, p.dim_k, p.dim_v}, log_decay.options())
                                  : at::empty({0}, log_decay.options());
  if (return_state) p.final_state = state.data_ptr<float>();
  const int64_t floats = bf_linear_attn_fwd_floats(&p);
  if (floats > 0) scratch = at::empty({floats}, log_decay.options());
  check_rc(bf_linear_attn_fwd(&p, q.data_ptr(), k.data_ptr(), v.data_ptr(), out.data_ptr(),
                              floats > 0 ? scratch.data_ptr<float>() : nullptr, stream_of(q)),
           "bf::linear_attn_fwd");
  return {out, state};
}

// Backward (bf_linear_attn_bwd): (dq, dk, dv), contiguous.
std::tuple<at::Tensor, at::Tensor, at::Tensor> linear_attn_bwd(const at::Tensor& q_in, const at::Tensor& k_in, const at::Tensor& v_in,
                                                               const at::Tensor& log_decay, const at::Tensor& row_span,
                                                               const at::Tensor& key_span, const at::Tensor& offsets,
                                                               const at::Tensor& dout_in, double scale, int64_t longest,
                                                               const std::optional<at::Tensor>& init_state) {
  TORCH_CHECK_VALUE(q_in.is_cuda(), "q must be a device tensor (got ", q_in.device(), ")");
  const c10::DeviceGuard guard(q_in.device());
  const at::Tensor q = as_rows(q_in, "q");
  const at::Tensor k = as_rows(k_in, "k");
  const at::Tensor v = as_rows(v_in, "v");
  const at::Tensor dout = as_dense(dout_in);
  const bf_linear_attn p = linear_args(q, k, v, log_decay, row_span, key_span, offsets, scale, longest, init_state);
  require(dout, "dout", q.scalar_type(), q.device());
  TORCH_CHECK_VALUE(dout.sizes() == v.sizes(), "dout ", dout.sizes(), " does not match v ", v.sizes());
  const auto plain = q.options().memory_format(at::MemoryFormat::Contiguous);
  at::Tensor dq = at::empty(q.sizes(), plain), dk = at::empty(k.sizes(), plain), dv = at::empty(v.sizes(), plain), scratch;
  const int64_t floats = bf_linear_attn_bwd_floats(&p);
  if (floats > 0) scratch = at::empty({floats}, log_decay.options());
  check_rc(bf_linear_attn_bwd(&p, q.data_ptr(), k.data_ptr(), v.data_ptr(), dout.data_ptr(), dq.data_ptr(), dk.data_ptr(),
                              dv.data_ptr(), floats > 0 ? scratch.data_ptr<float>() : nullptr, stream_of(q)),
           "bf::linear_attn_bwd");
  return {dq, dk, dv};
}

// The kernels know no forward-mode derivatives: a dual tensor is refused, not taken as a plain one.
void refuse_tangents(std::initializer_list<const at::Tensor*> ts, const char* name) {
  for (const at::Tensor* t : ts)
    TORCH_CHECK_NOT_IMPLEMENTED(!t->defined() || !t->_fw_grad(/*level=*/0).defined(), name,
                                " has no forward-mode derivatives (an input is a dual tensor)");
}

// One token of each sequence (bf_linear_attn_step): (out, new state); out_state: where the new state goes (state itself
// updates it in place), else a new tensor.
std::tuple<at::Tensor, at::Tensor> linear_attn_step(const at::Tensor& q, const at::Tensor& k, const at::Tensor& v,
                                                    const at::Tensor& log_decay, const at::Tensor& state, double scale,
                                                    const std::optional<at::Tensor>& out_state) {
  TORCH_CHECK_VALUE(q.is_cuda(), "q must be a device tensor (got ", q.device(), ")");
  const at::Tensor into = out_state.value_or(at::Tensor());
  refuse_tangents({&q, &k, &v, &log_decay, &state, &into}, "linear_attention_step");
  const c10::DeviceGuard guard(q.device());
  const at::Device dev = q.device();
  const int32_t code = dtype_code(q);
  require(q, "q", q.scalar_type(), dev);
  require(k, "k", q.scalar_type(), dev);
  require(v, "v", q.scalar_type(), dev);
  TORCH_CHECK_VALUE(q.dim() == 3 && k.sizes() == q.sizes() && v.dim() == 3 && v.size(0) == q.size(0) && v.size(1) == q.size(1),
                    "q ", q.sizes(), ", k ", k.sizes(), ", v ", v.sizes(), " must be [sequences, heads, head_dim]");
  const int64_t n = q.size(0), H = q.size(1), dk = q.size(2), dv = v.size(2);
  TORCH_CHECK_VALUE(H < (int64_t(1) << 30) && dk < (int64_t(1) << 30) && dv < (int64_t(1) << 30), "linear_attn_step: bad sizes");
  require(log_decay, "log_decay", at::kFloat, dev);
  TORCH_CHECK_VALUE(log_decay.dim() == 1 && log_decay.size(0) == H, "log_decay must be [", H, "] (got ", log_decay.sizes(), ")");
  const bool given = out_state.has_value() && out_state->defined();
  for (const at::Tensor* s : {&state, given ? &*out_state : &state}) {
    require(*s, s == &state ? "state" : "out_state", at::kFloat, dev);
    TORCH_CHECK_VALUE(s->dim() == 4 && s->size(0) == n && s->size(1) == H && s->size(2) == dk && s->size(3) == dv,
                      "a state must be [", n, ", ", H, ", ", dk, ", ", dv, "] (got ", s->sizes(), ")");
  }
  at::Tensor out = at::empty_like(v), next = given ? *out_state : at::empty_like(state);
  if (n == 0) return {out, next};
  if (given) {
    const auto apart = at::MemOverlapStatus::No, same = at::MemOverlapStatus::Full, states = at::get_overlap_status(next, state);
    TORCH_CHECK_VALUE(states == apart || states == same, "out_state overlaps state and is not state itself");
    for (const at::Tensor* t : {&q, &k, &v, &log_decay})
      TORCH_CHECK_VALUE(at::get_overlap_status(next, *t) == apart, "out_state overlaps an input");
    next.unsafeGetTensorImpl()->bump_version();          // a gradient that kept the old state is refused, not wrong
  }
  check_rc(bf_linear_attn_step(q.data_ptr(), k.data_ptr(), v.data_ptr(), log_decay.data_ptr<float>(), state.data_ptr<float>(), n,
                               int32_t(H), int32_t(dk), int32_t(dv), code, float(scale), out.data_ptr(),
                               next.data_ptr<float>(), stream_of(q)),
           "bf::linear_attn_step");
  return {out, next};
}

// The gated delta rule's arguments: q, k [n, heads_k, dim_k], v [n, heads, dim_v], log_gate and beta [n, heads].
bf_gated_delta delta_args(const at::Tensor& q, const at::Tensor& k, const at::Tensor& v, const at::Tensor& log_gate,
                          const at::Tensor& beta, double scale) {
  const at::Device dev = q.device();
  bf_gated_delta p{};
  p.dtype = dtype_code(q);
  require_heads(q, "q", q.scalar_type(), dev, p.q_stride);
  require_heads(k, "k", q.scalar_type(), dev, p.k_stride);
  require_heads(v, "v", q.scalar_type(), dev, p.v_stride);
  TORCH_CHECK_VALUE(q.sizes() == k.sizes() && v.size(0) == q.size(0), "q ", q.sizes(), ", k ", k.sizes(), ", v ", v.sizes(), " disagree");
  TORCH_CHECK_VALUE(q.size(1) < (int64_t(1) << 30) && v.size(1) < (int64_t(1) << 30) && q.size(2) < (int64_t(1) << 30) &&
                        v.size(2) < (int64_t(1) << 30), "gated_delta: bad sizes");
  for (const at::Tensor* t : {&log_gate, &beta}) {
    require(*t, t == &beta ? "beta" : "log_gate", at::kFloat, dev);
    TORCH_CHECK_VALUE(t->dim() == 2 && t->size(0) == v.size(0) && t->size(1) == v.size(1), t == &beta ? "beta" : "log_gate", " must be [",
                      v.size(0), ", ", v.size(1), "] (got ", t->sizes(), ")");
  }
  p.n = q.size(0), p.heads_k = int32_t(q.size(1)), p.heads = int32_t(v.size(1)), p.dim_k = int32_t(q.size(2)), p.dim_v = int32_t(v.size(2));
  p.log_gate = log_gate.data_ptr<float>(), p.beta = beta.data_ptr<float>();
  p.scale = float(scale);
  return p;
}

void delta_sequences(bf_gated_delta& p, const at::Tensor& offsets, int64_t longest, const std::optional<at::Tensor>& init_state,
                     const at::Device& dev) {
  require(offsets, "offsets", at::kInt, dev);
  TORCH_CHECK_VALUE(offsets.dim() == 1 && offsets.numel() >= 1, "offsets must be [n_seq + 1]");
  p.offsets = offsets.data_ptr<int32_t>(), p.n_seq = offsets.numel() - 1;
  p.longest = int32_t(std::min<int64_t>(std::max<int64_t>(longest, 0), INT32_MAX));
  if (init_state.has_value() && init_state->defined()) {
    require(*init_state, "init_state", at::kFloat, dev);
    TORCH_CHECK_VALUE(init_state->sizes() == at::IntArrayRef({p.n_seq, p.heads, p.dim_k, p.dim_v}), "init_state must be [", p.n_seq, ", ",
                      p.heads, ", ", p.dim_k, ", ", p.dim_v, "] (got ", init_state->sizes(), ")");
    p.init = init_state->data_ptr<float>();
  }
}

// Forward (bf_gated_delta_fwd): (out, final state or empty without return_state, kept or empty without train).
std::tuple<at::Tensor, at::Tensor, at::Tensor> gated_delta_fwd(const at::Tensor& q_in, const at::Tensor& k_in, const at::Tensor& v_in,
                                                               const at::Tensor& log_gate, const at::Tensor& beta,
                                                               const at::Tensor& offsets, double scale, int64_t longest,
                                                               const std::optional<at::Tensor>& init_in, bool return_state,
                                                               bool train) {
  TORCH_CHECK_VALUE(q_in.is_cuda(), "q must be a device tensor (got ", q_in.device(), ")");
  const c10::DeviceGuard guard(q_in.device());
  const at::Tensor q = as_rows(q_in, "q");
  const at::Tensor k = as_rows(k_in, "k");
  const at::Tensor v = as_rows(v_in, "v");
  std::optional<at::Tensor> init;
  if (init_in.has_value() && init_in->defined()) init = as_dense(*init_in);
  bf_gated_delta p = delta_args(q, k, v, log_gate, beta, scale);
  delta_sequences(p, offsets, longest, init, q.device());
  at::Tensor out = at::empty(v.sizes(), v.options().memory_format(at::MemoryFormat::Contiguous)), scratch;
  at::Tensor state = return_state ? at::empty({p.n_seq, p.heads, p.dim_k, p.dim_v}, log_gate.options()) : at::empty({0}, log_gate.options());
  if (return_state) p.final_state = state.data_ptr<float>();
  const int64_t floats = bf_gated_delta_fwd_floats(&p, train ? 1 : 0), keeps = train && floats >= 0 ? bf_gated_delta_kept_floats(&p) : 0;
  at::Tensor kept = at::empty({std::max<int64_t>(keeps, 0)}, log_gate.options());
  if (floats > 0) scratch = at::empty({floats}, log_gate.options());
  check_rc(bf_gated_delta_fwd(&p, q.data_ptr(), k.data_ptr(), v.data_ptr(), out.data_ptr(), keeps > 0 ? kept.data_ptr<float>() : nullptr,
                              floats > 0 ? scratch.data_ptr<float>() : nullptr, stream_of(q)),
           "bf::gated_delta_fwd");
  return {out, state, kept};
}

// Backward (bf_gated_delta_bwd): (dq, dk, dv, dlog_gate, dbeta), contiguous.
std::tuple<at::Tensor, at::Tensor, at::Tensor, at::Tensor, at::Tensor> gated_delta_bwd(
    const at::Tensor& q_in, const at::Tensor& k_in, const at::Tensor& v_in, const at::Tensor& log_gate, const at::Tensor& beta,
    const at::Tensor& offsets, const at::Tensor& kept, const at::Tensor& dout_in, double scale, int64_t longest,
    const std::optional<at::Tensor>& init_in) {
  TORCH_CHECK_VALUE(q_in.is_cuda(), "q must be a device tensor (got ", q_in.device(), ")");
  const c10::DeviceGuard guard(q_in.device());
  const at::Tensor q = as_rows(q_in, "q");
  const at::Tensor k = as_rows(k_in, "k");
  const at::Tensor v = as_rows(v_in, "v");
  const at::Tensor dout = as_dense(dout_in);
  std::optional<at::Tensor> init;
  if (init_in.has_value() && init_in->defined()) init = as_dense(*init_in);
  bf_gated_delta p = delta_args(q, k, v, log_gate, beta, scale);
  delta_sequences(p, offsets, longest, init, q.device());
  require(dout, "dout", q.scalar_type(), q.device());
  TORCH_CHECK_VALUE(dout.sizes() == v.sizes(), "dout ", dout.sizes(), " does not match v ", v.sizes());
  require(kept, "kept", at::kFloat, q.device());
  TORCH_CHECK_VALUE(kept.numel() == bf_gated_delta_kept_floats(&p), "kept has ", kept.numel(), " values, expected ",
                    bf_gated_delta_kept_floats(&p));
  const auto plain = q.options().memory_format(at::MemoryFormat::Contiguous);
  at::Tensor dq = at::empty(q.sizes(), plain), dk = at::empty(k.sizes(), plain), dv = at::empty(v.sizes(), plain), scratch;
  at::Tensor dgate = at::empty_like(log_gate), dbeta = at::empty_like(beta);
  const int64_t floats = bf_gated_delta_bwd_floats(&p);
  if (floats > 0) scratch = at::empty({floats}, log_gate.options());
  check_rc(bf_gated_delta_bwd(&p, q.data_ptr(), k.data_ptr(), v.data_ptr(), dout.data_ptr(), kept.data_ptr<float>(), dq.data_ptr(),
                              dk.data_ptr(), dv.data_ptr(), dgate.data_ptr<float>(), dbeta.data_ptr<float>(),
                              floats > 0 ? scratch.data_ptr<float>() : nullptr, stream_of(q)),
           "bf::gated_delta_bwd");
  return {dq, dk, dv, dgate, dbeta};
}

// Whether the memory between two tensors' first and last values meets (strides are not negative).
bool ranges_meet(const at::Tensor& x, const at::Tensor& y) {
  const auto range = [](const at::Tensor& t) {
    uintptr_t values = 1;
    for (int64_t d = 0; d < t.dim(); ++d) values += uintptr_t(t.size(d) - 1) * uintptr_t(t.stride(d));
    const uintptr_t from = reinterpret_cast<uintptr_t>(t.data_ptr());
    return std::make_pair(from, from + values * t.element_size());
  };
  if (x.numel() == 0 || y.numel() == 0) return false;
  const auto a = range(x), b = range(y);
  return a.first < b.second && b.first < a.second;
}

// One token of each sequence (bf_gated_delta_step): (out, new state); out_state as in linear_attn_step.
std::tuple<at::Tensor, at::Tensor> gated_delta_step(const at::Tensor& q_in, const at::Tensor& k_in, const at::Tensor& v_in,
                                                    const at::Tensor& log_gate, const at::Tensor& beta, const at::Tensor& state,
                                                    double scale, const std::optional<at::Tensor>& out_state) {
  TORCH_CHECK_VALUE(q_in.is_cuda(), "q must be a device tensor (got ", q_in.device(), ")");
  const at::Tensor into = out_state.value_or(at::Tensor());
  refuse_tangents({&q_in, &k_in, &v_in, &log_gate, &beta, &state, &into}, "gated_delta_step");
  const c10::DeviceGuard guard(q_in.device());
  const auto along = [](const at::Tensor& t) { return t.dim() != 3 || t.size(2) <= 1 || t.stride(2) == 1 ? t : t.contiguous(); };
  const at::Tensor q = along(q_in), k = along(k_in), v = along(v_in);
  bf_gated_delta p = delta_args(q, k, v, log_gate, beta, scale);
  const bool given = out_state.has_value() && out_state->defined();
  for (const at::Tensor* s : {&state, given ? &*out_state : &state}) {
    require(*s, s == &state ? "state" : "out_state", at::kFloat, q.device());
    TORCH_CHECK_VALUE(s->sizes() == at::IntArrayRef({p.n, p.heads, p.dim_k, p.dim_v}), "a state must be [", p.n, ", ", p.heads, ", ", p.dim_k,
                      ", ", p.dim_v, "] (got ", s->sizes(), ")");
  }
  at::Tensor out = at::empty(v.sizes(), v.options().memory_format(at::MemoryFormat::Contiguous)), next = given ? *out_state : at::empty_like(state);
  if (given) {
    const auto apart = at::MemOverlapStatus::No, same = at::MemOverlapStatus::Full, states = at::get_overlap_status(next, state);
    TORCH_CHECK_VALUE(p.n == 0 || states == apart || states == same, "out_state overlaps state and is not state itself");
    for (const at::Tensor* t : {&q, &k, &v, &log_gate, &beta})
      TORCH_CHECK_VALUE(!ranges_meet(next, *t), "out_state overlaps an input");
    next.unsafeGetTensorImpl()->bump_version();          // a gradient that kept the old state is refused, not wrong
  }
  p.init = state.data_ptr<float>(), p.final_state = next.data_ptr<float>();
  check_rc(bf_gated_delta_step(&p, q.data_ptr(), k.data_ptr(), v.data_ptr(), out.data_ptr(), stream_of(q)), "bf::gated_delta_step");
  return {out, next};
}

// ---------------------------------------------------------------- gradients of the operators over packed sequences
// Formed here and not in Python: a small call's time is its host work (forward and backward of 64 tokens: 48, 42 and 43 us
// with Python functions, 41, 35 and 36 us so, for the three operators).
using torch::autograd::AutogradContext;
using torch::autograd::variable_list;

bool trains(std::initializer_list<const at::Tensor*> ts) {
  if (!at::GradMode::is_enabled()) return false;
  for (const at::Tensor* t : ts)
    if (t->defined() && t->requires_grad()) return true;
  return false;
}

// Gradients that raise if they are differentiated again.
variable_list once(variable_list grads) {
  if (!at::GradMode::is_enabled()) return grads;
  variable_list given;
  for (at::Tensor& g : grads)
    if (g.defined()) given.push_back(g.detach().set_requires_grad(true));
  const auto error = std::make_shared<torch::autograd::DelayedError>(
      "trying to differentiate twice a function that was marked with once_differentiable", int64_t(given.size()));
  variable_list out = (*error)(std::move(given));
  size_t at = 0;
  for (at::Tensor& g : grads)
    if (g.defined()) g = out[at++];
  return grads;
}

struct PackedAttention : torch::autograd::Function<PackedAttention> {
  static variable_list forward(AutogradContext* ctx, const at::Tensor& q, const at::Tensor& k, const at::Tensor& v,
                               const at::Tensor& row_span, const at::Tensor& key_span, double scale, int64_t longest) {
    at::AutoDispatchBelowADInplaceOrView below;
    auto [out, lse, rest] = packed_attn_fwd(q, k, v, row_span, scale, longest, true);
    ctx->save_for_backward({q, k, v, out, lse, rest, row_span, key_span});
    ctx->saved_data["scale"] = scale;
    ctx->saved_data["longest"] = longest;
    ctx->mark_non_differentiable({lse});
    ctx->set_materialize_grads(false);
    return {out, lse};
  }
  static variable_list backward(AutogradContext* ctx, const variable_list& grads) {
    variable_list out(7);
    if (!grads[0].defined()) return out;
    const variable_list s = ctx->get_saved_variables();
    {
      at::AutoDispatchBelowADInplaceOrView below;
      std::tie(out[0], out[1], out[2]) =
          packed_attn_bwd(s[0], s[1], s[2], s[6], s[7], s[3], s[4], grads[0], ctx->saved_data["scale"].toDouble(),
                          ctx->saved_data["longest"].toInt(), s[5]);
    }
    return once(std::move(out));
  }
};

// packed_attn_fwd's out and lse, with gradients.
std::tuple<at::Tensor, at::Tensor> packed_attention(const at::Tensor& q, const at::Tensor& k, const at::Tensor& v,
                                                    const at::Tensor& row_span, const at::Tensor& key_span, double scale,
                                                    int64_t longest) {
  refuse_tangents({&q, &k, &v}, "packed_attention");
  if (trains({&q, &k, &v})) {
    variable_list r = PackedAttention::apply(q, k, v, row_span, key_span, scale, longest);
    return {r[0], r[1]};
  }
  at::AutoDispatchBelowADInplaceOrView below;
  auto [out, lse, rest] = packed_attn_fwd(q, k, v, row_span, scale, longest, false);
  return {out, lse};
}

struct PackedBiasAttention : torch::autograd::Function<PackedBiasAttention> {
  static variable_list forward(AutogradContext* ctx, const at::Tensor& q, const at::Tensor& k, const at::Tensor& v,
                               const at::Tensor& bias, const at::Tensor& map, const at::Tensor& positions, const at::Tensor& row_span,
                               const at::Tensor& key_span, double scale, int64_t longest) {
    at::AutoDispatchBelowADInplaceOrView below;
    auto [out, lse, rest] = packed_attn_bias_fwd(q, k, v, bias, map, positions, row_span, scale, longest, true);
    ctx->save_for_backward({q, k, v, bias, map, positions, row_span, key_span, out, lse, rest});
    ctx->saved_data["scale"] = scale;
    ctx->saved_data["longest"] = longest;
    ctx->mark_non_differentiable({lse});
    ctx->set_materialize_grads(false);
    return {out, lse};
  }
  static variable_list backward(AutogradContext* ctx, const variable_list& grads) {
    variable_list out(10);
    if (!grads[0].defined()) return out;
    const variable_list s = ctx->get_saved_variables();
    {
      at::AutoDispatchBelowADInplaceOrView below;
      std::tie(out[0], out[1], out[2], out[3]) =
          packed_attn_bias_bwd(s[0], s[1], s[2], s[3], s[4], s[5], s[6], s[7], s[8], s[9], grads[0], ctx->saved_data["scale"].toDouble(),
                               ctx->saved_data["longest"].toInt(), s[10]);
    }
    return once(std::move(out));
  }
};

// packed_attn_bias_fwd's out and lse, with gradients for q, k, v and the bias.
std::tuple<at::Tensor, at::Tensor> packed_bias_attention(const at::Tensor& q, const at::Tensor& k, const at::Tensor& v,
                                                         const at::Tensor& bias, const at::Tensor& map, const at::Tensor& positions,
                                                         const at::Tensor& row_span, const at::Tensor& key_span, double scale,
                                                         int64_t longest) {
  refuse_tangents({&q, &k, &v, &bias}, "packed_attention");
  if (trains({&q, &k, &v, &bias})) {
    variable_list r = PackedBiasAttention::apply(q, k, v, bias, map, positions, row_span, key_span, scale, longest);
    return {r[0], r[1]};
  }
  at::AutoDispatchBelowADInplaceOrView below;
  auto [out, lse, rest] = packed_attn_bias_fwd(q, k, v, bias, map, positions, row_span, scale, longest, false);
  return {out, lse};
}

struct Rotary : torch::autograd::Function<Rotary> {
  static variable_list forward(AutogradContext* ctx, const at::Tensor& x, const std::optional<at::Tensor>& y,
                               const at::Tensor& positions, const at::Tensor& turns, double amplitude, bool interleaved) {
    at::AutoDispatchBelowADInplaceOrView below;
    auto [ox, oy] = rotary(x, y, positions, turns, amplitude, interleaved, false);
    ctx->save_for_backward({positions, turns});
    ctx->saved_data["amplitude"] = amplitude;
    ctx->saved_data["interleaved"] = interleaved;
    ctx->set_materialize_grads(false);
    if (!y.has_value()) ctx->mark_non_differentiable({oy});
    return {ox, oy};
  }
  static variable_list backward(AutogradContext* ctx, const variable_list& grads) {
    variable_list out(6);
    const at::Tensor &dx = grads[0], &dy = grads[1];
    if (!dx.defined() && !dy.defined()) return out;
    const variable_list s = ctx->get_saved_variables();
    {
      at::AutoDispatchBelowADInplaceOrView below;
      const bool both = dx.defined() && dy.defined();
      auto [a, b] = rotary(dx.defined() ? dx : dy, both ? std::optional<at::Tensor>(dy) : std::nullopt, s[0], s[1],
                           ctx->saved_data["amplitude"].toDouble(), ctx->saved_data["interleaved"].toBool(), true);
      if (dx.defined()) out[0] = a;
      if (dy.defined()) out[1] = both ? b : a;
    }
    return once(std::move(out));
  }
};

// rotary of x and y (undefined: none), with gradients.
std::tuple<at::Tensor, at::Tensor> rotary_embedding(const at::Tensor& x, const std::optional<at::Tensor>& y,
                                                    const at::Tensor& positions, const at::Tensor& turns, double amplitude,
                                                    bool interleaved) {
  const at::Tensor second = y.has_value() ? *y : at::Tensor();
  refuse_tangents({&x, &second}, "rotary_embedding");
  if (trains({&x, &second})) {
    variable_list r = Rotary::apply(x, second.defined() ? std::optional<at::Tensor>(second) : std::nullopt, positions, turns, amplitude, interleaved);
    return {r[0], r[1]};
  }
  at::AutoDispatchBelowADInplaceOrView below;
  return rotary(x, y, positions, turns, amplitude, interleaved, false);
}

struct LinearAttention : torch::autograd::Function<LinearAttention> {
  static variable_list forward(AutogradContext* ctx, const at::Tensor& q, const at::Tensor& k, const at::Tensor& v,
                               const at::Tensor& log_decay, const at::Tensor& row_span, const at::Tensor& key_span,
                               const at::Tensor& offsets, double scale, int64_t longest,
                               const std::optional<at::Tensor>& init_state, bool return_state) {
    at::AutoDispatchBelowADInplaceOrView below;
    auto [out, state] = linear_attn_fwd(q, k, v, log_decay, row_span, key_span, offsets, scale, longest, init_state, return_state);
    ctx->save_for_backward({q, k, v, log_decay, row_span, key_span, offsets, init_state.value_or(at::Tensor())});
    ctx->saved_data["scale"] = scale;
    ctx->saved_data["longest"] = longest;
    ctx->mark_non_differentiable({state});
    ctx->set_materialize_grads(false);
    return {out, state};
  }
  static variable_list backward(AutogradContext* ctx, const variable_list& grads) {
    variable_list out(11);
    if (!grads[0].defined()) return out;
    const variable_list s = ctx->get_saved_variables();
    {
      at::AutoDispatchBelowADInplaceOrView below;
      std::tie(out[0], out[1], out[2]) =
          linear_attn_bwd(s[0], s[1], s[2], s[3], s[4], s[5], s[6], grads[0], ctx->saved_data["scale"].toDouble(),
                          ctx->saved_data["longest"].toInt(), s[7].defined() ? std::optional<at::Tensor>(s[7]) : std::nullopt);
    }
    return once(std::move(out));
  }
};

// linear_attn_fwd, with gradients for q, k and v.
std::tuple<at::Tensor, at::Tensor> linear_attention(const at::Tensor& q, const at::Tensor& k, const at::Tensor& v,
                                                    const at::Tensor& log_decay, const at::Tensor& row_span,
                                                    const at::Tensor& key_span, const at::Tensor& offsets, double scale,
                                                    int64_t longest, const std::optional<at::Tensor>& init_state,
                                                    bool return_state) {
  const at::Tensor init = init_state.value_or(at::Tensor());
  refuse_tangents({&q, &k, &v, &log_decay, &init}, "linear_attention");
  if (trains({&q, &k, &v})) {
    variable_list r =
        LinearAttention::apply(q, k, v, log_decay, row_span, key_span, offsets, scale, longest, init_state, return_state);
    return {r[0], r[1]};
  }
  at::AutoDispatchBelowADInplaceOrView below;
  return linear_attn_fwd(q, k, v, log_decay, row_span, key_span, offsets, scale, longest, init_state, return_state);
}

struct GatedDelta : torch::autograd::Function<GatedDelta> {
  static variable_list forward(AutogradContext* ctx, const at::Tensor& q, const at::Tensor& k, const at::Tensor& v,
                               const at::Tensor& log_gate, const at::Tensor& beta, const at::Tensor& offsets, double scale,
                               int64_t longest, const std::optional<at::Tensor>& init_state, bool return_state) {
    at::AutoDispatchBelowADInplaceOrView below;
    auto [out, state, kept] = gated_delta_fwd(q, k, v, log_gate, beta, offsets, scale, longest, init_state, return_state, true);
    ctx->save_for_backward({q, k, v, log_gate, beta, offsets, kept, init_state.value_or(at::Tensor())});
    ctx->saved_data["scale"] = scale;
    ctx->saved_data["longest"] = longest;
    ctx->mark_non_differentiable({state});
    ctx->set_materialize_grads(false);
    return {out, state};
  }
  static variable_list backward(AutogradContext* ctx, const variable_list& grads) {
    variable_list out(10);
    if (!grads[0].defined()) return out;
    const variable_list s = ctx->get_saved_variables();
    {
      at::AutoDispatchBelowADInplaceOrView below;
      std::tie(out[0], out[1], out[2], out[3], out[4]) =
          gated_delta_bwd(s[0], s[1], s[2], s[3], s[4], s[5], s[6], grads[0], ctx->saved_data["scale"].toDouble(),
                          ctx->saved_data["longest"].toInt(), s[7].defined() ? std::optional<at::Tensor>(s[7]) : std::nullopt);
    }
    return once(std::move(out));
  }
};

// gated_delta_fwd, with gradients for q, k, v, log_gate and beta.
std::tuple<at::Tensor, at::Tensor> gated_delta_rule(const at::Tensor& q, const at::Tensor& k, const at::Tensor& v,
                                                    const at::Tensor& log_gate, const at::Tensor& beta, const at::Tensor& offsets,
                                                    double scale, int64_t longest, const std::optional<at::Tensor>& init_state,
                                                    bool return_state) {
  const at::Tensor init = init_state.value_or(at::Tensor());
  refuse_tangents({&q, &k, &v, &log_gate, &beta, &init}, "gated_delta_rule");
  if (trains({&q, &k, &v, &log_gate, &beta})) {
    variable_list r = GatedDelta::apply(q, k, v, log_gate, beta, offsets, scale, longest, init_state, return_state);
    return {r[0], r[1]};
  }
  at::AutoDispatchBelowADInplaceOrView below;
  auto [out, state, kept] = gated_delta_fwd(q, k, v, log_gate, beta, offsets, scale, longest, init_state, return_state, false);
  return {out, state};
}

}  // namespace

TORCH_LIBRARY(bf, m) {
  m.def("sparse_attn_fwd(Tensor q, Tensor k, Tensor v, Tensor?[] index, int[] sizes, Tensor? bias=None, "
        "Tensor? factor=None, float dropout_rate=0.0, int dropout_seed=0, int dropout_offset=0, "
        "float score_clamp=5.0, bool keep_mask=False) -> (Tensor, Tensor, Tensor)");
  m.def("sparse_attn_bwd(Tensor q, Tensor k, Tensor v, Tensor?[] index, int[] sizes, Tensor Z, Tensor dout, "
        "Tensor? bias=None, Tensor? factor=None, bool need_dbias=False, float dropout_rate=0.0, int dropout_seed=0, "
        "int dropout_offset=0, float score_clamp=5.0, Tensor? keep=None) -> (Tensor, Tensor, Tensor, Tensor)");
  m.def("sparse_attn_fwd_typed(Tensor q, Tensor k, Tensor v, Tensor?[] index, int[] sizes, Tensor type_mod) "
        "-> (Tensor, Tensor)");
  m.def("sparse_attn_bwd_typed(Tensor q, Tensor k, Tensor v, Tensor?[] index, int[] sizes, Tensor type_mod, "
        "Tensor Z, Tensor dout) -> (Tensor, Tensor, Tensor, Tensor)");
  m.def("rw_walk(Tensor rowptr, Tensor col, int q_lo, int n_q, int walks_per_node, int walk_length, "
        "int philox_seed=0, int philox_offset=0, Tensor? u=None) -> Tensor");
  m.def("build_edge_table(Tensor rowptr, Tensor col, Tensor? walk_rec, Tensor in_ptr, Tensor in_src, int q_lo, "
        "int n_q, int walks_per_node, int walk_length, int k_real, int k_rw, int edge_seed, Tensor? u=None, "
        "int philox_seed=0, int philox_offset=0, Tensor? hubs=None, int hub_threshold=1024, Tensor? heavy=None, "
        "int light_max=-1) -> (Tensor, Tensor)");
  m.def("table_to_csr(Tensor table, Tensor row_len, bool global_token=False, int token_row=-1, int id_limit=-1) "
        "-> (Tensor, Tensor)");
  m.def("transpose_table(Tensor qptr, Tensor kv, int n_kv) -> (Tensor, Tensor, Tensor)");
  m.def("table_index(Tensor table, Tensor row_len, bool global_token, int token_row, int nnz, int n_keys, int q_bits, "
        "int slot_bits, int plan_items, int chunk, int item, Tensor(a!) counts) -> Tensor[]");
  m.def("reverse_index_and_plan(Tensor keys, Tensor qptr, int nnz, int n_kv, int q_bits, int slot_bits, "
        "bool global_token, int token_row, bool entries, int chunk, int item, Tensor(a!) counts) -> Tensor[]");
  m.def("packed_spans(Tensor q_offsets, Tensor k_offsets, int n_q, int n_k, bool causal) -> (Tensor, Tensor, Tensor)");
  m.def("packed_attn_fwd(Tensor q, Tensor k, Tensor v, Tensor row_span, float scale, int longest=0, "
        "bool train=False) -> (Tensor, Tensor, Tensor)");
  m.def("packed_attn_bwd(Tensor q, Tensor k, Tensor v, Tensor row_span, Tensor key_span, Tensor out, Tensor lse, "
        "Tensor dout, float scale, int longest=0, Tensor? rest=None) -> (Tensor, Tensor, Tensor)");
  m.def("packed_attn_bias_fwd(Tensor q, Tensor k, Tensor v, Tensor bias, Tensor map, Tensor positions, Tensor row_span, float scale, "
        "int longest=0, bool train=False) -> (Tensor, Tensor, Tensor)");
  m.def("packed_attn_bias_bwd(Tensor q, Tensor k, Tensor v, Tensor bias, Tensor map, Tensor positions, Tensor row_span, Tensor key_span, "
        "Tensor out, Tensor lse, Tensor dout, float scale, int longest=0, Tensor? rest=None) -> (Tensor, Tensor, Tensor, Tensor)");
  m.def("packed_bias_attention(Tensor q, Tensor k, Tensor v, Tensor bias, Tensor map, Tensor positions, Tensor row_span, "
        "Tensor key_span, float scale, int longest=0) -> (Tensor, Tensor)");
  m.def("rotary(Tensor x, Tensor? y, Tensor positions, Tensor turns, float amplitude=1.0, bool interleaved=False, "
        "bool inverse=False) -> (Tensor, Tensor)");
  m.def("linear_attn_fwd(Tensor q, Tensor k, Tensor v, Tensor log_decay, Tensor row_span, Tensor key_span, Tensor offsets, "
        "float scale, int longest=0, Tensor? init_state=None, bool return_state=False) -> (Tensor, Tensor)");
  m.def("linear_attn_bwd(Tensor q, Tensor k, Tensor v, Tensor log_decay, Tensor row_span, Tensor key_span, Tensor offsets, "
        "Tensor dout, float scale, int longest=0, Tensor? init_state=None) -> (Tensor, Tensor, Tensor)");
  // the same with gradients (packed_attn_bwd, rotary with inverse, linear_attn_bwd)
  m.def("packed_attention(Tensor q, Tensor k, Tensor v, Tensor row_span, Tensor key_span, float scale, int longest=0) "
        "-> (Tensor, Tensor)");
  m.def("rotary_embedding(Tensor x, Tensor? y, Tensor positions, Tensor turns, float amplitude=1.0, bool interleaved=False) "
        "-> (Tensor, Tensor)");
  m.def("linear_attention(Tensor q, Tensor k, Tensor v, Tensor log_decay, Tensor row_span, Tensor key_span, Tensor offsets, "
        "float scale, int longest=0, Tensor? init_state=None, bool return_state=False) -> (Tensor, Tensor)");
  m.def("gated_delta_fwd(Tensor q, Tensor k, Tensor v, Tensor log_gate, Tensor beta, Tensor offsets, float scale, int longest=0, "
        "Tensor? init_state=None, bool return_state=False, bool train=False) -> (Tensor, Tensor, Tensor)");
  m.def("gated_delta_bwd(Tensor q, Tensor k, Tensor v, Tensor log_gate, Tensor beta, Tensor offsets, Tensor kept, Tensor dout, "
        "float scale, int longest=0, Tensor? init_state=None) -> (Tensor, Tensor, Tensor, Tensor, Tensor)");
  m.def("gated_delta_rule(Tensor q, Tensor k, Tensor v, Tensor log_gate, Tensor beta, Tensor offsets, float scale, int longest=0, "
        "Tensor? init_state=None, bool return_state=False) -> (Tensor, Tensor)");
  m.def("gated_delta_step(Tensor q, Tensor k, Tensor v, Tensor log_gate, Tensor beta, Tensor state, float scale, "
        "Tensor(a!)? out_state=None) -> (Tensor, Tensor)");
  m.def("linear_attn_step(Tensor q, Tensor k, Tensor v, Tensor log_decay, Tensor state, float scale, "
        "Tensor(a!)? out_state=None) -> (Tensor, Tensor)");
}

TORCH_LIBRARY_IMPL(bf, CUDA, m) {
  m.impl("sparse_attn_fwd", &sparse_attn_fwd);
  m.impl("sparse_attn_bwd", &sparse_attn_bwd);
  m.impl("sparse_attn_fwd_typed", &sparse_attn_fwd_typed);
  m.impl("sparse_attn_bwd_typed", &sparse_attn_bwd_typed);
  m.impl("rw_walk", &rw_walk);
  m.impl("build_edge_table", &build_edge_table);
  m.impl("table_to_csr", &table_to_csr);
  m.impl("transpose_table", &transpose_table);
  m.impl("table_index", &table_index);
  m.impl("reverse_index_and_plan", &reverse_index_and_plan);
  m.impl("packed_spans", &packed_spans);
  m.impl("packed_attn_fwd", &packed_attn_fwd);
  m.impl("packed_attn_bwd", &packed_attn_bwd);
  m.impl("packed_attn_bias_fwd", &packed_attn_bias_fwd);
  m.impl("packed_attn_bias_bwd", &packed_attn_bias_bwd);
  m.impl("rotary", &rotary);
  m.impl("linear_attn_fwd", &linear_attn_fwd);
  m.impl("linear_attn_bwd", &linear_attn_bwd);
  m.impl("linear_attn_step", &linear_attn_step);
  m.impl("packed_attention", &packed_attention);
  m.impl("packed_bias_attention", &packed_bias_attention);
  m.impl("rotary_embedding", &rotary_embedding);
  m.impl("linear_attention", &linear_attention);
  m.impl("gated_delta_fwd", &gated_delta_fwd);
  m.impl("gated_delta_bwd", &gated_delta_bwd);
  m.impl("gated_delta_step", &gated_delta_step);
  m.impl("gated_delta_rule", &gated_delta_rule);
}

TORCH_LIBRARY_IMPL(bf, AutogradCUDA, m) {
  m.impl("packed_attention", &packed_attention);
  m.impl("packed_bias_attention", &packed_bias_attention);
  m.impl("rotary_embedding", &rotary_embedding);
  m.impl("linear_attention", &linear_attention);
  m.impl("gated_delta_rule", &gated_delta_rule);
}
