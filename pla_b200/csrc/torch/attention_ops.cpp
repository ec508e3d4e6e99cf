// Host layer of the full-attention operators (block tables, rotary positions with norm and cache write, paged decode):
// tensor contracts checked with TORCH_CHECK (-> RuntimeError), outputs and scratch from torch's allocator, one C-ABI
// call on the current stream of the tensors' device. No synchronisation, no D2H.
#include <ATen/cuda/EmptyTensor.h>

#include <cmath>
#include <limits>
#include <tuple>

#include "ops_common.h"
#include "overlap.h"
#include "pla_b200_attention.h"

namespace pla_ops {
namespace {

constexpr int64_t MAX_I32 = std::numeric_limits<int32_t>::max();

// Uninitialised tensor straight from the CUDA allocator: at::empty takes about 1.2 us a call through the dispatcher, which is a
// tenth of a decode step's small ops each.
at::Tensor fresh(at::IntArrayRef size, at::ScalarType dtype, const at::Device& device) {
  return at::detail::empty_cuda(size, dtype, device, std::nullopt);
}

// The kernels take scalars as 32-bit numbers.
bool finite32(double x) { return std::isfinite(static_cast<float>(x)); }

void check_on(const at::Tensor& t, const at::Device& device, const char* name) {
  TORCH_CHECK(t.device() == device, name, " must be on ", device, ", got ", t.device());
}

void check_i32_vector(const at::Tensor& t, int64_t n, const at::Device& device, const char* name) {
  check_on(t, device, name);
  TORCH_CHECK(t.scalar_type() == at::kInt && t.dim() == 1 && t.is_contiguous(), name, " must be a contiguous 1-D int32 tensor");
  TORCH_CHECK(t.size(0) == n, name, " must have ", n, " entries, got ", t.size(0));
}

// 1-D int32 or int64 vector with any stride.
pla_b200_index index_view(const at::Tensor& t, int64_t n, const at::Device& device, const char* name) {
  check_on(t, device, name);
  TORCH_CHECK((t.scalar_type() == at::kInt || t.scalar_type() == at::kLong) && t.dim() == 1, name,
              " must be a 1-D int32 or int64 tensor");
  TORCH_CHECK(t.size(0) == n, name, " must have ", n, " entries, got ", t.size(0));
  return {t.data_ptr(), t.scalar_type() == at::kLong ? 1 : 0, t.stride(0)};
}

int32_t* status_ptr(const std::optional<at::Tensor>& status, const at::Device& device) {
  if (!status.has_value() || !status->defined()) return nullptr;
  check_on(*status, device, "status");
  TORCH_CHECK(status->scalar_type() == at::kInt && status->numel() >= 1, "status must be an int32 tensor of one entry");
  return status->data_ptr<int32_t>();
}

// [tokens, heads, D] view with contiguous channels.
void check_rows(const at::Tensor& t, const at::Device& device, const char* name) {
  check_on(t, device, name);
  TORCH_CHECK(t.dim() == 3, name, " must have shape [tokens, heads, dim]");
  TORCH_CHECK(t.stride(2) == 1 || t.size(2) <= 1 || t.numel() == 0, name, " channels must be contiguous");
  TORCH_CHECK(t.scalar_type() == at::kBFloat16 || t.scalar_type() == at::kHalf, name, " must be bf16 or fp16");
}

// Stride that the kernel may use: axes of extent 1 report whatever the view's history left there.
int64_t step(const at::Tensor& t, int64_t dim) { return t.size(dim) <= 1 ? 0 : t.stride(dim); }

struct CacheView {
  pla_b200_page_strides k, v;
  int64_t blocks, block_size;
};

CacheView cache_view(const at::Tensor& k, const at::Tensor& v, int64_t heads, int64_t D, at::ScalarType dtype, const at::Device& device) {
  for (const at::Tensor* t : {&k, &v}) {
    check_on(*t, device, "k_cache and v_cache");
    TORCH_CHECK(t->dim() == 4, "k_cache and v_cache must have shape [blocks, block_size, kv heads, dim]");
    TORCH_CHECK(t->scalar_type() == dtype, "k_cache and v_cache must have q's dtype");
    TORCH_CHECK(t->size(2) == heads && t->size(3) == D, "k_cache and v_cache must have ", heads, " heads of size ", D, ", got ",
                t->size(2), " of size ", t->size(3));
    TORCH_CHECK(t->stride(3) == 1 || t->numel() == 0, "k_cache and v_cache channels must be contiguous");
  }
  TORCH_CHECK(k.sizes() == v.sizes(), "k_cache and v_cache must have the same shape");
  TORCH_CHECK(k.size(1) > 0 && k.size(1) <= MAX_I32, "the block size must be positive");
  return {{step(k, 0), step(k, 1), step(k, 2)}, {step(v, 0), step(v, 1), step(v, 2)}, k.size(0), k.size(1)};
}

// ---------------------------------------------------------------------------------------------- block tables
std::tuple<at::Tensor, at::Tensor, at::Tensor, at::Tensor> build_block_tables(
    at::Tensor block_table, const at::Tensor& context_lens, const at::Tensor& query_start_loc, const at::Tensor& free_blocks,
    int64_t block_size, int64_t num_tokens, const std::optional<at::Tensor>& free_start, const std::optional<at::Tensor>& status) {
  check_cuda(block_table, "block_table");
  const at::Device device = block_table.device();
  TORCH_CHECK(block_table.scalar_type() == at::kInt && block_table.dim() == 2, "block_table must be a 2-D int32 tensor");
  const int64_t N = block_table.size(0), C = block_table.size(1);
  TORCH_CHECK(C <= 1 || block_table.stride(1) == 1, "block_table columns must be contiguous");
  TORCH_CHECK(N <= 1 || C == 0 || block_table.stride(0) >= C, "block_table rows must not overlap");
  check_i32_vector(context_lens, N, device, "context_lens");
  check_i32_vector(query_start_loc, N + 1, device, "query_start_loc");
  check_i32_vector(free_blocks, free_blocks.dim() == 1 ? free_blocks.size(0) : 0, device, "free_blocks");
  if (free_start.has_value()) check_i32_vector(*free_start, 1, device, "free_start");
  Arguments args;
  args.read(context_lens);
  args.read(query_start_loc);
  args.read(free_blocks);
  args.read(free_start);
  args.write(block_table, "block_table");
  TORCH_CHECK(block_size > 0 && block_size <= MAX_I32, "block_size must be positive");
  TORCH_CHECK(num_tokens >= 0, "num_tokens must not be negative");
  TORCH_CHECK(num_tokens < MAX_I32 / 2 && N < MAX_I32 / 2 && C < MAX_I32 && free_blocks.size(0) <= MAX_I32, "block tables: too many entries");
  c10::cuda::CUDAGuard guard(device);
  at::Tensor slots = fresh({num_tokens}, at::kLong, device), positions = fresh({num_tokens}, at::kLong, device);
  at::Tensor seq_lens = fresh({N}, at::kInt, device), free_next = fresh({1}, at::kInt, device);
  pla_b200_block_tables_args g{};
  g.block_table = block_table.data_ptr<int32_t>();
  g.table_row_stride = N <= 1 ? C : block_table.stride(0);
  g.context_lens = context_lens.data_ptr<int32_t>();
  g.query_start_loc = query_start_loc.data_ptr<int32_t>();
  g.free_blocks = free_blocks.data_ptr<int32_t>();
  g.free_start = i32_ptr(free_start, "free_start");
  g.slot_mapping = slots.data_ptr<int64_t>();
  g.positions = positions.data_ptr<int64_t>();
  g.seq_lens = seq_lens.data_ptr<int32_t>();
  g.free_next = free_next.data_ptr<int32_t>();
  g.N = static_cast<int32_t>(N);
  g.tokens = static_cast<int32_t>(num_tokens);
  g.columns = static_cast<int32_t>(C);
  g.free_count = static_cast<int32_t>(free_blocks.size(0));
  g.block_size = static_cast<int32_t>(block_size);
  g.status = status_ptr(status, device);
  if (sanity_check()) {
    const std::string bad = sanity_offsets(query_start_loc, num_tokens, 0);
    TORCH_CHECK(bad.empty(), "build_block_tables: sanity check: ", bad);
  }
  if (!bypass_exec()) check_abi(pla_b200_block_tables(&g, stream_of(block_table)), "build_block_tables");
  return {slots, positions, seq_lens, free_next};
}

// ---------------------------------------------------------------------------------------------- rotary
const void* norm_weight(const std::optional<at::Tensor>& w, int64_t D, const at::Device& device, const char* name, int32_t* dtype) {
  if (!w.has_value() || !w->defined()) return nullptr;
  check_on(*w, device, name);
  TORCH_CHECK(w->dim() == 1 && w->size(0) == D && w->is_contiguous(), name, " must be contiguous [", D, "]");
  *dtype = dtype_tag(*w, name);
  return w->data_ptr();
}

at::Tensor out_rows(const std::optional<at::Tensor>& out, const at::Tensor& like, const char* name) {
  if (!out.has_value() || !out->defined()) return fresh(like.sizes(), like.scalar_type(), like.device());
  check_rows(*out, like.device(), name);
  TORCH_CHECK(out->sizes() == like.sizes() && out->scalar_type() == like.scalar_type(), name, " must match its input in shape and dtype");
  return *out;
}

std::tuple<at::Tensor, at::Tensor> rotary(
    const at::Tensor& q, const std::optional<at::Tensor>& k, const std::optional<at::Tensor>& v,
    const std::optional<at::Tensor>& q_weight, const std::optional<at::Tensor>& k_weight, const at::Tensor& positions,
    const at::Tensor& inv_freq, const std::optional<at::Tensor>& k_cache, const std::optional<at::Tensor>& v_cache,
    const std::optional<at::Tensor>& slot_mapping, double eps, double factor, bool interleaved, bool unit_offset,
    const std::optional<at::Tensor>& out_q, const std::optional<at::Tensor>& out_k, const std::optional<at::Tensor>& status, const char* op) {
  check_cuda(q, "q");
  const at::Device device = q.device();
  check_rows(q, device, "q");
  const int64_t T = q.size(0), Hq = q.size(1), D = q.size(2);
  TORCH_CHECK(D > 0 && D % 8 == 0 && D <= 256, "the head size must be a multiple of 8, at most 256, got ", D);
  TORCH_CHECK(T <= MAX_I32 && Hq < 65536, "rotary: too many tokens or heads");
  pla_b200_rotary_args g{};
  if (k.has_value()) {
    check_rows(*k, device, "k");
    TORCH_CHECK(k->size(0) == T && k->size(2) == D && k->scalar_type() == q.scalar_type(), "k must match q in tokens, head size and dtype");
    TORCH_CHECK(k->size(1) < 65536, "rotary: too many heads");
    g.k = k->data_ptr();
    g.k_tok_stride = step(*k, 0);
    g.k_head_stride = step(*k, 1);
    g.Hk = static_cast<int32_t>(k->size(1));
  }
  check_on(inv_freq, device, "inv_freq");
  TORCH_CHECK(inv_freq.scalar_type() == at::kDouble && inv_freq.dim() == 1 && inv_freq.is_contiguous(),
              "inv_freq must be a contiguous 1-D float64 tensor (rotary_frequencies makes it)");
  TORCH_CHECK(2 * inv_freq.size(0) <= D, "the rotated part (2 * inv_freq entries) must be at most the head size");
  TORCH_CHECK(finite32(eps) && eps >= 0.0 && (eps == 0.0 || static_cast<float>(eps) > 0.0f) && finite32(factor),
              "eps must be finite and non-negative, factor finite, both as 32-bit numbers");
  g.positions = index_view(positions, T, device, "positions");
  g.inv_freq = inv_freq.data_ptr<double>();
  g.q_weight = norm_weight(q_weight, D, device, "q_weight", &g.q_weight_dtype);
  g.k_weight = norm_weight(k_weight, D, device, "k_weight", &g.k_weight_dtype);
  g.status = status_ptr(status, device);
  const bool cached = k_cache.has_value();
  if (cached) {
    TORCH_CHECK(k.has_value() && v.has_value() && v_cache.has_value() && slot_mapping.has_value(),
                "a cache needs k, v, k_cache, v_cache and slot_mapping");
    check_rows(*v, device, "v");
    TORCH_CHECK(v->sizes() == k->sizes() && v->scalar_type() == q.scalar_type(), "v must match k in shape and dtype");
    const CacheView c = cache_view(*k_cache, *v_cache, k->size(1), D, q.scalar_type(), device);
    g.v = v->data_ptr();
    g.v_tok_stride = step(*v, 0);
    g.v_head_stride = step(*v, 1);
    g.k_cache = k_cache->data_ptr();
    g.v_cache = v_cache->data_ptr();
    g.k_strides = c.k;
    g.v_strides = c.v;
    g.num_blocks = c.blocks;
    g.block_size = static_cast<int32_t>(c.block_size);
    g.slots = index_view(*slot_mapping, T, device, "slot_mapping");
    if (sanity_check()) {
      const std::string bad = sanity_slots(*slot_mapping, c.blocks * c.block_size);
      TORCH_CHECK(bad.empty(), "qk_norm_rotary_cache: sanity check: ", bad);
    }
    if (c.blocks == 0) TORCH_CHECK(T == 0, "the cache has no blocks");
  }
  c10::cuda::CUDAGuard guard(device);
  at::Tensor qo = out_rows(out_q, q, "out_q"), ko;
  if (k.has_value() && !cached) ko = out_rows(out_k, *k, "out_k");
  if (cached || out_q.has_value() || out_k.has_value()) {
    Arguments args;
    args.read(v);
    args.read(q_weight);
    args.read(k_weight);
    args.read(positions);
    args.read(inv_freq);
    args.read(slot_mapping);
    const int q_in = args.read(q), k_in = args.read(k);
    if (out_q.has_value()) args.write(qo, "out_q", q_in);
    if (out_k.has_value() && ko.defined()) args.write(ko, "out_k", k_in);
    if (cached) {
      args.write(*k_cache, "k_cache");
      args.write(*v_cache, "v_cache");
    }
  }
  g.q = q.data_ptr();
  g.q_tok_stride = step(q, 0);
  g.q_head_stride = step(q, 1);
  g.q_out = qo.data_ptr();
  g.qo_tok_stride = step(qo, 0);
  g.qo_head_stride = step(qo, 1);
  if (ko.defined()) {
    g.k_out = ko.data_ptr();
    g.ko_tok_stride = step(ko, 0);
    g.ko_head_stride = step(ko, 1);
  }
  g.T = static_cast<int32_t>(T);
  g.Hq = static_cast<int32_t>(Hq);
  g.D = static_cast<int32_t>(D);
  g.R = static_cast<int32_t>(2 * inv_freq.size(0));
  g.interleaved = interleaved;
  g.unit_offset = unit_offset;
  g.act_dtype = dtype_tag(q, "q");
  g.factor = static_cast<float>(factor);
  g.eps = static_cast<float>(eps);
  if (!bypass_exec()) check_abi(pla_b200_rotary(&g, stream_of(q)), op);
  return {qo, ko};
}

// One operator per use: an argument costs about a tenth of a microsecond on its way through the dispatcher.
std::tuple<at::Tensor, at::Tensor> apply_rotary(const at::Tensor& q, const std::optional<at::Tensor>& k, const at::Tensor& positions,
                                                const at::Tensor& inv_freq, double factor, bool interleaved,
                                                const std::optional<at::Tensor>& out_q, const std::optional<at::Tensor>& out_k) {
  return rotary(q, k, std::nullopt, std::nullopt, std::nullopt, positions, inv_freq, std::nullopt, std::nullopt, std::nullopt, 0.0, factor,
                interleaved, false, out_q, out_k, std::nullopt, "apply_rotary");
}

std::tuple<at::Tensor, at::Tensor> qk_norm_rotary(const at::Tensor& q, const std::optional<at::Tensor>& k,
                                                  const std::optional<at::Tensor>& q_weight, const std::optional<at::Tensor>& k_weight,
                                                  const at::Tensor& positions, const at::Tensor& inv_freq, double eps, double factor,
                                                  bool interleaved, bool unit_offset, const std::optional<at::Tensor>& out_q,
                                                  const std::optional<at::Tensor>& out_k) {
  return rotary(q, k, std::nullopt, q_weight, k_weight, positions, inv_freq, std::nullopt, std::nullopt, std::nullopt, eps, factor,
                interleaved, unit_offset, out_q, out_k, std::nullopt, "qk_norm_rotary");
}

at::Tensor qk_norm_rotary_cache(const at::Tensor& q, const at::Tensor& k, const at::Tensor& v, const std::optional<at::Tensor>& q_weight,
                                const std::optional<at::Tensor>& k_weight, const at::Tensor& positions, const at::Tensor& inv_freq,
                                const at::Tensor& k_cache, const at::Tensor& v_cache, const at::Tensor& slot_mapping, double eps, double factor,
                                bool interleaved, bool unit_offset, const std::optional<at::Tensor>& out_q,
                                const std::optional<at::Tensor>& status) {
  return std::get<0>(rotary(q, k, v, q_weight, k_weight, positions, inv_freq, k_cache, v_cache, slot_mapping, eps, factor, interleaved,
                            unit_offset, out_q, std::nullopt, status, "qk_norm_rotary_cache"));
}

// ---------------------------------------------------------------------------------------------- paged decode
std::tuple<at::Tensor, at::Tensor> paged_attention_decode(const at::Tensor& q, const at::Tensor& k_cache, const at::Tensor& v_cache,
                                                          const at::Tensor& block_table, const at::Tensor& seq_lens,
                                                          std::optional<double> scale, bool return_lse,
                                                          const std::optional<at::Tensor>& out, const std::optional<at::Tensor>& status) {
  check_cuda(q, "q");
  const at::Device device = q.device();
  TORCH_CHECK(q.dim() == 3, "q must have shape [requests, heads, dim]");
  check_rows(q, device, "q");
  const int64_t B = q.size(0), Hq = q.size(1), D = q.size(2);
  TORCH_CHECK(k_cache.dim() == 4, "k_cache and v_cache must have shape [blocks, block_size, kv heads, dim]");
  const int64_t Hk = k_cache.size(2);
  TORCH_CHECK(Hq > 0 && Hk > 0 && Hq % Hk == 0, "the query heads must be a positive multiple of the key/value heads, got ", Hq, " and ", Hk);
  TORCH_CHECK(D == 64 || D == 96 || D == 128 || D == 192 || D == 256, "the head size must be 64, 96, 128, 192 or 256, got ", D);
  TORCH_CHECK(B <= MAX_I32 && Hq < 65536 && B * Hq <= MAX_I32, "paged decode: too many rows");
  const CacheView c = cache_view(k_cache, v_cache, Hk, D, q.scalar_type(), device);
  check_on(block_table, device, "block_table");
  TORCH_CHECK(block_table.scalar_type() == at::kInt && block_table.dim() == 2 && block_table.size(0) == B,
              "block_table must be int32 with one row per request");
  TORCH_CHECK(block_table.size(1) <= 1 || block_table.stride(1) == 1, "block_table columns must be contiguous");
  TORCH_CHECK(block_table.size(1) <= MAX_I32, "block_table has too many columns");
  check_i32_vector(seq_lens, B, device, "seq_lens");
  TORCH_CHECK(!scale.has_value() || finite32(*scale), "scale must be finite as a 32-bit number");
  c10::cuda::CUDAGuard guard(device);
  at::Tensor o = out.has_value() ? *out : fresh({B, Hq, D}, q.scalar_type(), device);
  if (out.has_value()) {
    check_on(o, device, "out");
    TORCH_CHECK(o.is_contiguous() && o.sizes() == q.sizes() && o.scalar_type() == q.scalar_type(), "out must be contiguous with q's shape and dtype");
    Arguments args;
    args.read(k_cache);
    args.read(v_cache);
    args.read(block_table);
    args.read(seq_lens);
    args.write(o, "out", args.read(q));
  }
  at::Tensor lse;
  if (return_lse) lse = fresh({B, Hq}, at::kFloat, device);
  pla_b200_paged_decode_args g{};
  g.q = q.data_ptr();
  g.q_row_stride = step(q, 0);
  g.q_head_stride = step(q, 1);
  g.k_cache = k_cache.data_ptr();
  g.v_cache = v_cache.data_ptr();
  g.k_strides = c.k;
  g.v_strides = c.v;
  g.block_table = block_table.data_ptr<int32_t>();
  g.table_row_stride = step(block_table, 0);
  g.seq_lens = seq_lens.data_ptr<int32_t>();
  g.out = o.data_ptr();
  g.lse = return_lse ? lse.data_ptr<float>() : nullptr;
  g.num_blocks = c.blocks;
  g.block_size = static_cast<int32_t>(c.block_size);
  g.columns = static_cast<int32_t>(block_table.size(1));
  g.B = static_cast<int32_t>(B);
  g.Hq = static_cast<int32_t>(Hq);
  g.Hk = static_cast<int32_t>(Hk);
  g.D = static_cast<int32_t>(D);
  g.act_dtype = dtype_tag(q, "q");
  g.scale = static_cast<float>(scale.has_value() ? *scale : 1.0 / std::sqrt(static_cast<double>(D)));
  g.status = status_ptr(status, device);
  if (sanity_check()) {
    const at::Tensor lens = seq_lens.to(at::kCPU), table = block_table.to(at::kCPU).contiguous();
    const int32_t *n = lens.data_ptr<int32_t>(), *p = table.data_ptr<int32_t>();
    for (int64_t b = 0; b < B; ++b) {
      TORCH_CHECK(n[b] >= 0 && n[b] <= table.size(1) * c.block_size, "paged_attention_decode: sanity check: length ", n[b], " of request ", b,
                  " is negative or past its block-table row");
      for (int64_t j = 0; j * c.block_size < n[b]; ++j)
        TORCH_CHECK(p[b * table.size(1) + j] >= 0 && p[b * table.size(1) + j] < c.blocks, "paged_attention_decode: sanity check: page ",
                    p[b * table.size(1) + j], " of request ", b, " is outside the pool of ", c.blocks);
    }
  }
  const int64_t bytes = pla_b200_paged_decode_workspace_bytes(&g);
  TORCH_CHECK(bytes >= 0, "paged_attention_decode: ", pla_b200_last_error());
  at::Tensor workspace;
  if (bytes > 0) {
    workspace = fresh({bytes}, at::kByte, device);
    g.workspace = workspace.data_ptr();
    g.workspace_bytes = bytes;
  }
  if (!bypass_exec()) check_abi(pla_b200_paged_decode(&g, stream_of(q)), "paged_attention_decode");
  return {o, lse};
}

}  // namespace
}  // namespace pla_ops

TORCH_LIBRARY_FRAGMENT(pla_b200, m) {
  m.def(
      "build_block_tables(Tensor(a!) block_table, Tensor context_lens, Tensor query_start_loc, Tensor free_blocks, int block_size, "
      "int num_tokens, Tensor? free_start=None, Tensor(b!)? status=None) -> (Tensor, Tensor, Tensor, Tensor)",
      &pla_ops::build_block_tables);
  m.def(
      "apply_rotary(Tensor q, Tensor? k, Tensor positions, Tensor inv_freq, float factor, bool interleaved, Tensor(a!)? out_q=None, "
      "Tensor(b!)? out_k=None) -> (Tensor, Tensor)",
      &pla_ops::apply_rotary);
  m.def(
      "qk_norm_rotary(Tensor q, Tensor? k, Tensor? q_weight, Tensor? k_weight, Tensor positions, Tensor inv_freq, float eps, float factor, "
      "bool interleaved, bool unit_offset, Tensor(a!)? out_q=None, Tensor(b!)? out_k=None) -> (Tensor, Tensor)",
      &pla_ops::qk_norm_rotary);
  m.def(
      "qk_norm_rotary_cache(Tensor q, Tensor k, Tensor v, Tensor? q_weight, Tensor? k_weight, Tensor positions, Tensor inv_freq, "
      "Tensor(a!) k_cache, Tensor(b!) v_cache, Tensor slot_mapping, float eps, float factor, bool interleaved, bool unit_offset, "
      "Tensor(c!)? out_q=None, Tensor(d!)? status=None) -> Tensor",
      &pla_ops::qk_norm_rotary_cache);
  m.def(
      "paged_attention_decode(Tensor q, Tensor k_cache, Tensor v_cache, Tensor block_table, Tensor seq_lens, float? scale, bool return_lse, "
      "Tensor(a!)? out=None, Tensor(b!)? status=None) -> (Tensor, Tensor)",
      &pla_ops::paged_attention_decode);
}
