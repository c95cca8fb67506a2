// Thin PyTorch extension `deepseekrpc_cuda` over the C ABI of libdsr_b200.so.
//
// The four reference ops keep the names, argument order, return convention and
// TORCH_CHECK validation of native/bindings.cpp:20-26 / native/operations.cu:180-243
// (with the bounds widened to the DeepSeek-V3.2/V4 geometry); abi_version() is 2.
// New entry points expose the paged decode path.  Outputs are allocated with
// the caching allocator on the input's device; work runs on the current stream.
#include <ATen/cuda/CUDAContext.h>
#include <ATen/cuda/EmptyTensor.h>
#include <c10/cuda/CUDAGuard.h>
#include <torch/extension.h>

#include <algorithm>
#include <utility>
#include <vector>

#include "dsr_b200.h"

namespace {

void check(const at::Tensor& t, at::ScalarType dtype, const at::Tensor& anchor) {
  TORCH_CHECK(t.is_cuda() && t.device() == anchor.device(), "all inputs require the same CUDA device");
  TORCH_CHECK(t.scalar_type() == dtype && t.is_contiguous(), "input dtype/contiguity mismatch");
}

void check_cache(const at::Tensor& value, const at::Tensor& anchor) {
  TORCH_CHECK(value.scalar_type() == at::kBFloat16, "cache storage must be unquantized BF16");
  check(value, value.scalar_type(), anchor);
}

void ok(int rc) { TORCH_CHECK(rc == DSR_OK, dsr_last_error()); }

void* current_stream() { return at::cuda::getCurrentCUDAStream().stream(); }

const uint16_t* bf16(const at::Tensor& t) { return reinterpret_cast<const uint16_t*>(t.data_ptr()); }
uint16_t* bf16_mut(at::Tensor& t) { return reinterpret_cast<uint16_t*>(t.data_ptr()); }

at::Tensor status_like(const at::Tensor& anchor) {
  return at::zeros({1}, anchor.options().dtype(at::kInt));
}

}  // namespace

// ---------------------------------------------------------------- reference ops

std::vector<at::Tensor> ds_sparse_attention(at::Tensor q, at::Tensor window, at::Tensor source,
                                            at::Tensor indices, at::Tensor sink, double scale) {
  check(q, at::kFloat, q);
  check_cache(window, q);
  check_cache(source, q);
  check(indices, at::kInt, q);
  check(sink, at::kFloat, q);
  TORCH_CHECK(q.dim() == 3 && q.size(0) > 0 && q.size(0) <= 65536 && q.size(1) > 0 && q.size(1) <= 128,
              "invalid bounded query shape");
  const auto width = q.size(2);
  TORCH_CHECK(width > 0 && width <= 576 && window.dim() == 2 && source.dim() == 2 &&
                  window.size(1) == width && source.size(1) == width && window.size(0) <= 65536,
              "KV dimensions/capacity differ from bounded query");
  TORCH_CHECK(indices.dim() == 2 && indices.size(0) == q.size(0) && indices.size(1) <= 65536 &&
                  sink.dim() == 1 && sink.size(0) == q.size(1),
              "invalid sparse indices/sink shape");
  TORCH_CHECK(std::isfinite(static_cast<float>(scale)) && static_cast<float>(scale) > 0.0f,
              "invalid attention scale");
  const c10::cuda::CUDAGuard guard(q.device());
  auto out = at::empty_like(q);
  auto error = status_like(q);
  ok(dsr_sparse_attention(q.data_ptr<float>(), bf16(window), bf16(source), indices.data_ptr<int32_t>(),
                          sink.data_ptr<float>(), out.data_ptr<float>(), error.data_ptr<int32_t>(),
                          q.size(0), q.size(1), width, window.size(0), source.size(0),
                          indices.size(1), static_cast<float>(scale), current_stream()));
  return {out, error};
}

std::vector<at::Tensor> ds_index_scores(at::Tensor q, at::Tensor keys, at::Tensor weights,
                                        at::Tensor indices, at::Tensor visible) {
  check(q, at::kFloat, q);
  check_cache(keys, q);
  check(weights, at::kFloat, q);
  check(indices, at::kInt, q);
  check(visible, at::kInt, q);
  TORCH_CHECK(q.dim() == 3 && q.size(0) > 0 && q.size(0) <= 65536 && q.size(1) > 0 && q.size(1) <= 64 &&
                  q.size(2) == 128 && keys.dim() == 2 && keys.size(1) == 128,
              "invalid index query/key shape");
  TORCH_CHECK(weights.dim() == 2 && weights.size(0) == q.size(0) && weights.size(1) == q.size(1) &&
                  visible.dim() == 1 && visible.size(0) == q.size(0) && indices.dim() == 2 &&
                  indices.size(0) == q.size(0) && indices.size(1) > 0,
              "invalid bounded index tile");
  const c10::cuda::CUDAGuard guard(q.device());
  auto out = at::empty(indices.sizes(), q.options());
  auto error = status_like(q);
  ok(dsr_index_scores(q.data_ptr<float>(), bf16(keys), weights.data_ptr<float>(),
                      indices.data_ptr<int32_t>(), visible.data_ptr<int32_t>(), out.data_ptr<float>(),
                      error.data_ptr<int32_t>(), q.size(0), q.size(1), indices.size(1), keys.size(0),
                      current_stream()));
  return {out, error};
}

std::vector<at::Tensor> ds_engram_decode(at::Tensor encoded) {
  check(encoded, at::kByte, encoded);
  TORCH_CHECK(encoded.dim() == 2 && encoded.size(0) > 0 && encoded.size(0) <= 1024 && encoded.size(1) == 264,
              "encoded Engram rows must be bounded [rows,264] uint8");
  const c10::cuda::CUDAGuard guard(encoded.device());
  auto out = at::empty({encoded.size(0), 256}, encoded.options().dtype(at::kBFloat16));
  auto error = status_like(encoded);
  ok(dsr_engram_decode(encoded.data_ptr<uint8_t>(), bf16_mut(out), error.data_ptr<int32_t>(),
                       encoded.size(0), current_stream()));
  return {out, error};
}

at::Tensor ds_scatter_slots(at::Tensor pool, at::Tensor generations, at::Tensor slots,
                            at::Tensor expected_generations, at::Tensor values) {
  check_cache(pool, pool);
  check(generations, at::kLong, pool);
  check(slots, at::kInt, pool);
  check(expected_generations, at::kLong, pool);
  check_cache(values, pool);
  TORCH_CHECK(pool.dim() == 2 && pool.size(1) > 0 && pool.size(1) <= 576 && generations.dim() == 1 &&
                  generations.size(0) == pool.size(0),
              "invalid cache/generation pool");
  TORCH_CHECK(slots.dim() == 1 && slots.size(0) > 0 && slots.size(0) <= 4096 &&
                  expected_generations.dim() == 1 && expected_generations.size(0) == slots.size(0) &&
                  values.dim() == 2 && values.size(0) == slots.size(0) && values.size(1) == pool.size(1),
              "invalid cache update rows");
  const c10::cuda::CUDAGuard guard(pool.device());
  auto error = status_like(pool);
  ok(dsr_scatter_slots(bf16_mut(pool), generations.data_ptr<int64_t>(), slots.data_ptr<int32_t>(),
                       expected_generations.data_ptr<int64_t>(), bf16(values), error.data_ptr<int32_t>(),
                       slots.size(0), pool.size(1), pool.size(0), current_stream()));
  return error;
}

// ---------------------------------------------------------------- new entry points

std::vector<at::Tensor> ds_topk_select(at::Tensor scores, at::Tensor lengths, int64_t k,
                                       c10::optional<at::Tensor> ids, int64_t id_base,
                                       bool return_scores) {
  check(scores, at::kFloat, scores);
  check(lengths, at::kInt, scores);
  TORCH_CHECK(scores.dim() == 2 && lengths.dim() == 1 && lengths.size(0) == scores.size(0),
              "topk_select: scores [rows, n] and lengths [rows] expected");
  if (ids) {
    check(*ids, at::kInt, scores);
    TORCH_CHECK(ids->sizes() == scores.sizes(), "topk_select: ids must match scores");
  }
  const c10::cuda::CUDAGuard guard(scores.device());
  auto out = at::empty({scores.size(0), k}, scores.options().dtype(at::kInt));
  at::Tensor out_scores = return_scores ? at::empty({scores.size(0), k}, scores.options()) : at::Tensor();
  auto error = status_like(scores);
  const size_t ws_bytes = dsr_topk_workspace_bytes(scores.size(0), scores.size(1));
  auto ws = at::zeros({int64_t(ws_bytes)}, scores.options().dtype(at::kByte));
  ok(dsr_topk_select(scores.data_ptr<float>(), ids ? ids->data_ptr<int32_t>() : nullptr,
                     lengths.data_ptr<int32_t>(), out.data_ptr<int32_t>(),
                     return_scores ? out_scores.data_ptr<float>() : nullptr, error.data_ptr<int32_t>(),
                     scores.size(0), scores.size(1), k, id_base, ws.data_ptr(), ws_bytes,
                     current_stream()));
  if (return_scores) return {out, error, out_scores};
  return {out, error};
}

std::vector<at::Tensor> ds_indexer_decode(at::Tensor q, at::Tensor weights, at::Tensor index_pool,
                                          at::Tensor block_table, at::Tensor visible,
                                          int64_t score_stride) {
  check(q, at::kFloat, q);
  check(weights, at::kFloat, q);
  check_cache(index_pool, q);
  check(block_table, at::kInt, q);
  check(visible, at::kInt, q);
  TORCH_CHECK(q.dim() == 3 && q.size(2) == 128 && weights.dim() == 2 && weights.size(0) == q.size(0) &&
                  weights.size(1) == q.size(1),
              "indexer_decode: q [batch, heads, 128] and weights [batch, heads] expected");
  TORCH_CHECK(index_pool.dim() == 2 && index_pool.size(1) == 128 && index_pool.size(0) % 64 == 0,
              "indexer_decode: index_pool [blocks*64, 128] expected");
  TORCH_CHECK(block_table.dim() == 2 && block_table.size(0) == q.size(0) && visible.dim() == 1 &&
                  visible.size(0) == q.size(0),
              "indexer_decode: block_table [batch, blocks] and visible [batch] expected");
  const c10::cuda::CUDAGuard guard(q.device());
  auto scores = at::empty({q.size(0), score_stride}, q.options());
  auto error = status_like(q);
  ok(dsr_indexer_decode(q.data_ptr<float>(), weights.data_ptr<float>(), bf16(index_pool),
                        index_pool.size(0) / 64, block_table.data_ptr<int32_t>(), block_table.size(1),
                        visible.data_ptr<int32_t>(), scores.data_ptr<float>(), score_stride,
                        error.data_ptr<int32_t>(), q.size(0), q.size(1), current_stream()));
  return {scores, error};
}

std::vector<at::Tensor> ds_sparse_mla_decode(at::Tensor q, at::Tensor kv_pool, at::Tensor block_table,
                                             at::Tensor visible, at::Tensor topk, at::Tensor swa,
                                             at::Tensor swa_len, at::Tensor sink, double scale) {
  check(q, at::kFloat, q);
  check_cache(kv_pool, q);
  check(block_table, at::kInt, q);
  check(visible, at::kInt, q);
  check(topk, at::kInt, q);
  check_cache(swa, q);
  check(swa_len, at::kInt, q);
  check(sink, at::kFloat, q);
  const int64_t batch = q.size(0), heads = q.size(1);
  TORCH_CHECK(q.dim() == 3 && q.size(2) == DSR_KV_DIM, "sparse_mla_decode: q [batch, heads, 576] expected");
  TORCH_CHECK(kv_pool.dim() == 2 && kv_pool.size(1) == DSR_KV_DIM && kv_pool.size(0) % 64 == 0,
              "sparse_mla_decode: kv_pool [blocks*64, 576] expected");
  TORCH_CHECK(block_table.dim() == 2 && block_table.size(0) == batch && topk.dim() == 2 &&
                  topk.size(0) == batch && visible.size(0) == batch && swa_len.size(0) == batch &&
                  swa.dim() == 3 && swa.size(0) == batch && swa.size(1) == DSR_SWA_ROWS &&
                  swa.size(2) == DSR_KV_DIM && sink.dim() == 1 && sink.size(0) == heads,
              "sparse_mla_decode: inconsistent shapes");
  const c10::cuda::CUDAGuard guard(q.device());
  const int64_t k = topk.size(1);
  auto out = at::empty({batch, heads, DSR_V_DIM}, q.options());
  const size_t ws_bytes = dsr_mla_workspace_bytes(batch, heads, k);
  auto ws = at::empty({int64_t(ws_bytes)}, q.options().dtype(at::kByte));
  auto error = status_like(q);
  ok(dsr_sparse_mla_decode(q.data_ptr<float>(), bf16(kv_pool), kv_pool.size(0) / 64,
                           block_table.data_ptr<int32_t>(), block_table.size(1),
                           visible.data_ptr<int32_t>(), topk.data_ptr<int32_t>(), k, bf16(swa),
                           swa_len.data_ptr<int32_t>(), sink.data_ptr<float>(), static_cast<float>(scale),
                           out.data_ptr<float>(), ws.data_ptr(), ws_bytes, error.data_ptr<int32_t>(),
                           batch, heads, current_stream()));
  return {out, error};
}

at::Tensor ds_append_kv_index(at::Tensor kv_pool, at::Tensor index_pool, at::Tensor generations,
                              at::Tensor block_table, at::Tensor seq, at::Tensor positions,
                              at::Tensor expected, at::Tensor kv_values, at::Tensor index_values,
                              c10::optional<at::Tensor> swa) {
  check_cache(kv_pool, kv_pool);
  check_cache(index_pool, kv_pool);
  check(generations, at::kLong, kv_pool);
  check(block_table, at::kInt, kv_pool);
  check(seq, at::kInt, kv_pool);
  check(positions, at::kInt, kv_pool);
  check(expected, at::kLong, kv_pool);
  check_cache(kv_values, kv_pool);
  check_cache(index_values, kv_pool);
  const int64_t n = seq.size(0);
  TORCH_CHECK(kv_pool.dim() == 2 && kv_pool.size(1) == DSR_KV_DIM && index_pool.dim() == 2 &&
                  index_pool.size(1) == DSR_INDEX_DIM && kv_pool.size(0) == index_pool.size(0) &&
                  kv_pool.size(0) % 64 == 0 && generations.dim() == 1 &&
                  generations.size(0) == kv_pool.size(0),
              "append_kv_index: pools [blocks*64, 576/128] and generations [blocks*64] expected");
  TORCH_CHECK(block_table.dim() == 2 && positions.size(0) == n && expected.size(0) == n &&
                  kv_values.dim() == 2 && kv_values.size(0) == n && kv_values.size(1) == DSR_KV_DIM &&
                  index_values.dim() == 2 && index_values.size(0) == n &&
                  index_values.size(1) == DSR_INDEX_DIM,
              "append_kv_index: inconsistent row shapes");
  if (swa) {
    check_cache(*swa, kv_pool);
    TORCH_CHECK(swa->dim() == 3 && swa->size(0) == block_table.size(0) && swa->size(1) == DSR_SWA_ROWS &&
                    swa->size(2) == DSR_KV_DIM,
                "append_kv_index: swa [sequences, 128, 576] expected");
  }
  const c10::cuda::CUDAGuard guard(kv_pool.device());
  auto error = status_like(kv_pool);
  ok(dsr_append_kv_index(bf16_mut(kv_pool), bf16_mut(index_pool), generations.data_ptr<int64_t>(),
                         kv_pool.size(0) / 64, block_table.data_ptr<int32_t>(), block_table.size(0),
                         block_table.size(1), seq.data_ptr<int32_t>(), positions.data_ptr<int32_t>(),
                         expected.data_ptr<int64_t>(), bf16(kv_values), bf16(index_values),
                         swa ? bf16_mut(*swa) : nullptr, error.data_ptr<int32_t>(), n,
                         current_stream()));
  return error;
}

std::vector<at::Tensor> ds_lse_combine(at::Tensor part_o, at::Tensor part_m, at::Tensor part_l,
                                       c10::optional<at::Tensor> sink) {
  check(part_o, at::kFloat, part_o);
  check(part_m, at::kFloat, part_o);
  check(part_l, at::kFloat, part_o);
  TORCH_CHECK(part_o.dim() == 4 && part_m.dim() == 3 && part_l.sizes() == part_m.sizes() &&
                  part_o.size(0) == part_m.size(0) && part_o.size(1) == part_m.size(1) &&
                  part_o.size(2) == part_m.size(2),
              "lse_combine: part_o [batch, parts, heads, dv], part_m/part_l [batch, parts, heads]");
  const int64_t batch = part_o.size(0), parts = part_o.size(1), heads = part_o.size(2), dv = part_o.size(3);
  const c10::cuda::CUDAGuard guard(part_o.device());
  auto out = at::empty({batch, heads, dv}, part_o.options());
  auto error = status_like(part_o);
  if (sink) {
    check(*sink, at::kFloat, part_o);
    TORCH_CHECK(sink->dim() == 1 && sink->size(0) == heads, "lse_combine: sink [heads] expected");
    ok(dsr_lse_combine(part_o.data_ptr<float>(), part_m.data_ptr<float>(), part_l.data_ptr<float>(),
                       parts, sink->data_ptr<float>(), out.data_ptr<float>(), nullptr, nullptr,
                       error.data_ptr<int32_t>(), batch, heads, dv, current_stream()));
    return {out, error};
  }
  auto m = at::empty({batch, heads}, part_o.options());
  auto l = at::empty({batch, heads}, part_o.options());
  ok(dsr_lse_combine(part_o.data_ptr<float>(), part_m.data_ptr<float>(), part_l.data_ptr<float>(), parts,
                     nullptr, out.data_ptr<float>(), m.data_ptr<float>(), l.data_ptr<float>(),
                     error.data_ptr<int32_t>(), batch, heads, dv, current_stream()));
  return {out, m, l, error};
}

std::vector<at::Tensor> ds_decode_step(at::Tensor idx_q, at::Tensor idx_w, at::Tensor index_pool,
                                       at::Tensor q, at::Tensor kv_pool, at::Tensor block_table,
                                       at::Tensor visible, int64_t max_visible, int64_t k, at::Tensor swa,
                                       at::Tensor swa_len, at::Tensor sink, double scale,
                                       bool return_scores) {
  check(idx_q, at::kFloat, q);
  check(idx_w, at::kFloat, q);
  check_cache(index_pool, q);
  check(q, at::kFloat, q);
  check_cache(kv_pool, q);
  check(block_table, at::kInt, q);
  check(visible, at::kInt, q);
  check_cache(swa, q);
  check(swa_len, at::kInt, q);
  check(sink, at::kFloat, q);
  const int64_t batch = q.size(0), heads = q.size(1);
  TORCH_CHECK(idx_q.dim() == 3 && idx_q.size(0) == batch && idx_q.size(2) == 128 && idx_w.dim() == 2 &&
                  idx_w.size(0) == batch && idx_w.size(1) == idx_q.size(1),
              "decode_step: idx_q [batch, idx_heads, 128], idx_w [batch, idx_heads] expected");
  TORCH_CHECK(q.dim() == 3 && q.size(2) == DSR_KV_DIM && kv_pool.size(1) == DSR_KV_DIM &&
                  index_pool.size(1) == DSR_INDEX_DIM && kv_pool.size(0) == index_pool.size(0) &&
                  kv_pool.size(0) % 64 == 0,
              "decode_step: pool geometry mismatch");
  TORCH_CHECK(block_table.dim() == 2 && block_table.size(0) == batch && visible.size(0) == batch &&
                  swa.dim() == 3 && swa.size(0) == batch && swa_len.size(0) == batch &&
                  sink.size(0) == heads,
              "decode_step: inconsistent batch shapes");
  const c10::cuda::CUDAGuard guard(q.device());
  auto out = at::empty({batch, heads, DSR_V_DIM}, q.options());
  auto topk = at::empty({batch, k}, q.options().dtype(at::kInt));
  const int64_t stride = (max_visible + 63) / 64 * 64;
  at::Tensor scores = return_scores ? at::empty({batch, stride}, q.options()) : at::Tensor();
  const size_t ws_bytes = dsr_decode_workspace_bytes(batch, max_visible, heads, k);
  auto ws = at::zeros({int64_t(ws_bytes)}, q.options().dtype(at::kByte));
  auto error = status_like(q);
  ok(dsr_decode_step(idx_q.data_ptr<float>(), idx_w.data_ptr<float>(), idx_q.size(1), bf16(index_pool),
                     q.data_ptr<float>(), bf16(kv_pool), heads, kv_pool.size(0) / 64,
                     block_table.data_ptr<int32_t>(), block_table.size(1), visible.data_ptr<int32_t>(),
                     max_visible, k, bf16(swa), swa_len.data_ptr<int32_t>(), sink.data_ptr<float>(),
                     static_cast<float>(scale), out.data_ptr<float>(), topk.data_ptr<int32_t>(),
                     return_scores ? scores.data_ptr<float>() : nullptr, ws.data_ptr(), ws_bytes,
                     error.data_ptr<int32_t>(), batch, current_stream()));
  if (return_scores) return {out, topk, error, scores};
  return {out, topk, error};
}

// ---- ring-offset pools (the reference's DeviceRowPool layout): rings i64[batch, 3]
void check_ring(const at::Tensor& ring, int64_t batch, const at::Tensor& anchor, const char* what) {
  check(ring, at::kLong, anchor);
  TORCH_CHECK(ring.dim() == 2 && ring.size(0) == batch && ring.size(1) == 3, what,
              ": ring descriptors [batch, 3] = (first row, slots, offset) expected");
}

std::vector<at::Tensor> ds_indexer_decode_ring(at::Tensor q, at::Tensor weights, at::Tensor index_pool,
                                               at::Tensor ring, at::Tensor visible, int64_t score_stride) {
  check(q, at::kFloat, q);
  check(weights, at::kFloat, q);
  check_cache(index_pool, q);
  check(visible, at::kInt, q);
  TORCH_CHECK(q.dim() == 3 && q.size(2) == 128 && weights.dim() == 2 && weights.size(0) == q.size(0) &&
                  weights.size(1) == q.size(1) && index_pool.dim() == 2 && index_pool.size(1) == 128 &&
                  visible.dim() == 1 && visible.size(0) == q.size(0),
              "indexer_decode_ring: q [batch, heads, 128], weights [batch, heads], index_pool [rows, 128], "
              "visible [batch] expected");
  check_ring(ring, q.size(0), q, "indexer_decode_ring");
  const c10::cuda::CUDAGuard guard(q.device());
  auto scores = at::empty({q.size(0), score_stride}, q.options());
  auto error = status_like(q);
  ok(dsr_indexer_decode_ring(q.data_ptr<float>(), weights.data_ptr<float>(), bf16(index_pool),
                             index_pool.size(0), ring.data_ptr<int64_t>(), visible.data_ptr<int32_t>(),
                             scores.data_ptr<float>(), score_stride, error.data_ptr<int32_t>(), q.size(0),
                             q.size(1), current_stream()));
  return {scores, error};
}

std::vector<at::Tensor> ds_sparse_mla_decode_ring(at::Tensor q, at::Tensor kv_pool, at::Tensor kv_ring,
                                                  at::Tensor visible, at::Tensor topk, at::Tensor swa_pool,
                                                  at::Tensor swa_ring, at::Tensor swa_len, at::Tensor sink,
                                                  double scale) {
  check(q, at::kFloat, q);
  check_cache(kv_pool, q);
  check(visible, at::kInt, q);
  check(topk, at::kInt, q);
  check_cache(swa_pool, q);
  check(swa_len, at::kInt, q);
  check(sink, at::kFloat, q);
  const int64_t batch = q.size(0), heads = q.size(1);
  TORCH_CHECK(q.dim() == 3 && q.size(2) == DSR_KV_DIM && kv_pool.dim() == 2 && kv_pool.size(1) == DSR_KV_DIM &&
                  swa_pool.dim() == 2 && swa_pool.size(1) == DSR_KV_DIM && topk.dim() == 2 &&
                  topk.size(0) == batch && visible.size(0) == batch && swa_len.size(0) == batch &&
                  sink.dim() == 1 && sink.size(0) == heads,
              "sparse_mla_decode_ring: inconsistent shapes");
  check_ring(kv_ring, batch, q, "sparse_mla_decode_ring (KV pool)");
  check_ring(swa_ring, batch, q, "sparse_mla_decode_ring (SWA pool)");
  const c10::cuda::CUDAGuard guard(q.device());
  const int64_t k = topk.size(1);
  auto out = at::empty({batch, heads, DSR_V_DIM}, q.options());
  const size_t ws_bytes = dsr_mla_workspace_bytes(batch, heads, k);
  auto ws = at::empty({int64_t(ws_bytes)}, q.options().dtype(at::kByte));
  auto error = status_like(q);
  ok(dsr_sparse_mla_decode_ring(q.data_ptr<float>(), bf16(kv_pool), kv_pool.size(0), kv_ring.data_ptr<int64_t>(),
                                visible.data_ptr<int32_t>(), topk.data_ptr<int32_t>(), k, bf16(swa_pool),
                                swa_pool.size(0), swa_ring.data_ptr<int64_t>(), swa_len.data_ptr<int32_t>(),
                                sink.data_ptr<float>(), static_cast<float>(scale), out.data_ptr<float>(),
                                ws.data_ptr(), ws_bytes, error.data_ptr<int32_t>(), batch, heads,
                                current_stream()));
  return {out, error};
}

std::vector<at::Tensor> ds_decode_step_ring(at::Tensor idx_q, at::Tensor idx_w, at::Tensor index_pool,
                                            at::Tensor index_ring, at::Tensor q, at::Tensor kv_pool,
                                            at::Tensor kv_ring, at::Tensor visible, int64_t max_visible, int64_t k,
                                            at::Tensor swa_pool, at::Tensor swa_ring, at::Tensor swa_len,
                                            at::Tensor sink, double scale, bool return_scores) {
  check(idx_q, at::kFloat, q);
  check(idx_w, at::kFloat, q);
  check_cache(index_pool, q);
  check(q, at::kFloat, q);
  check_cache(kv_pool, q);
  check(visible, at::kInt, q);
  check_cache(swa_pool, q);
  check(swa_len, at::kInt, q);
  check(sink, at::kFloat, q);
  const int64_t batch = q.size(0), heads = q.size(1);
  TORCH_CHECK(idx_q.dim() == 3 && idx_q.size(0) == batch && idx_q.size(2) == 128 && idx_w.dim() == 2 &&
                  idx_w.size(0) == batch && idx_w.size(1) == idx_q.size(1),
              "decode_step_ring: idx_q [batch, idx_heads, 128], idx_w [batch, idx_heads] expected");
  TORCH_CHECK(q.dim() == 3 && q.size(2) == DSR_KV_DIM && kv_pool.dim() == 2 && kv_pool.size(1) == DSR_KV_DIM &&
                  index_pool.dim() == 2 && index_pool.size(1) == DSR_INDEX_DIM && swa_pool.dim() == 2 &&
                  swa_pool.size(1) == DSR_KV_DIM,
              "decode_step_ring: pool geometry mismatch");
  TORCH_CHECK(visible.size(0) == batch && swa_len.size(0) == batch && sink.size(0) == heads,
              "decode_step_ring: inconsistent batch shapes");
  check_ring(index_ring, batch, q, "decode_step_ring (index pool)");
  check_ring(kv_ring, batch, q, "decode_step_ring (KV pool)");
  check_ring(swa_ring, batch, q, "decode_step_ring (SWA pool)");
  const c10::cuda::CUDAGuard guard(q.device());
  auto out = at::empty({batch, heads, DSR_V_DIM}, q.options());
  auto topk = at::empty({batch, k}, q.options().dtype(at::kInt));
  const int64_t stride = (max_visible + 63) / 64 * 64;
  at::Tensor scores = return_scores ? at::empty({batch, stride}, q.options()) : at::Tensor();
  const size_t ws_bytes = dsr_decode_workspace_bytes(batch, max_visible, heads, k);
  auto ws = at::zeros({int64_t(ws_bytes)}, q.options().dtype(at::kByte));
  auto error = status_like(q);
  ok(dsr_decode_step_ring(idx_q.data_ptr<float>(), idx_w.data_ptr<float>(), idx_q.size(1), bf16(index_pool),
                          index_pool.size(0), index_ring.data_ptr<int64_t>(), q.data_ptr<float>(), bf16(kv_pool),
                          kv_pool.size(0), kv_ring.data_ptr<int64_t>(), heads, visible.data_ptr<int32_t>(),
                          max_visible, k, bf16(swa_pool), swa_pool.size(0), swa_ring.data_ptr<int64_t>(),
                          swa_len.data_ptr<int32_t>(), sink.data_ptr<float>(), static_cast<float>(scale),
                          out.data_ptr<float>(), topk.data_ptr<int32_t>(),
                          return_scores ? scores.data_ptr<float>() : nullptr, ws.data_ptr(), ws_bytes,
                          error.data_ptr<int32_t>(), batch, current_stream()));
  if (return_scores) return {out, topk, error, scores};
  return {out, topk, error};
}

at::Tensor ds_append_kv_index_ring(at::Tensor kv_pool, at::Tensor kv_ring, at::Tensor kv_generations,
                                   at::Tensor kv_expected, at::Tensor index_pool, at::Tensor index_ring,
                                   at::Tensor index_generations, at::Tensor index_expected, at::Tensor seq,
                                   at::Tensor positions, at::Tensor kv_values, at::Tensor index_values) {
  check_cache(kv_pool, kv_pool);
  check_cache(index_pool, kv_pool);
  check(kv_generations, at::kLong, kv_pool);
  check(index_generations, at::kLong, kv_pool);
  check(kv_expected, at::kLong, kv_pool);
  check(index_expected, at::kLong, kv_pool);
  check(seq, at::kInt, kv_pool);
  check(positions, at::kInt, kv_pool);
  check_cache(kv_values, kv_pool);
  check_cache(index_values, kv_pool);
  const int64_t n = seq.size(0), sequences = kv_ring.size(0);
  TORCH_CHECK(kv_pool.dim() == 2 && kv_pool.size(1) == DSR_KV_DIM && index_pool.dim() == 2 &&
                  index_pool.size(1) == DSR_INDEX_DIM && kv_generations.dim() == 1 &&
                  kv_generations.size(0) == kv_pool.size(0) && index_generations.dim() == 1 &&
                  index_generations.size(0) == index_pool.size(0),
              "append_kv_index_ring: pools [rows, 576/128] with generations [rows] expected");
  TORCH_CHECK(positions.size(0) == n && kv_expected.size(0) == n && index_expected.size(0) == n &&
                  kv_values.dim() == 2 && kv_values.size(0) == n && kv_values.size(1) == DSR_KV_DIM &&
                  index_values.dim() == 2 && index_values.size(0) == n && index_values.size(1) == DSR_INDEX_DIM,
              "append_kv_index_ring: inconsistent row shapes");
  check_ring(kv_ring, sequences, kv_pool, "append_kv_index_ring (KV pool)");
  check_ring(index_ring, sequences, kv_pool, "append_kv_index_ring (index pool)");
  const c10::cuda::CUDAGuard guard(kv_pool.device());
  auto error = status_like(kv_pool);
  ok(dsr_append_kv_index_ring(bf16_mut(kv_pool), kv_pool.size(0), kv_ring.data_ptr<int64_t>(),
                              kv_generations.data_ptr<int64_t>(), kv_expected.data_ptr<int64_t>(),
                              bf16_mut(index_pool), index_pool.size(0), index_ring.data_ptr<int64_t>(),
                              index_generations.data_ptr<int64_t>(), index_expected.data_ptr<int64_t>(), sequences,
                              seq.data_ptr<int32_t>(), positions.data_ptr<int32_t>(), bf16(kv_values),
                              bf16(index_values), error.data_ptr<int32_t>(), n, current_stream()));
  return error;
}

// ---- around the decode path.  `status`: a status word that the caller keeps (zeroed
// once, first error wins); without it the call makes a fresh one.
at::Tensor status_or(const c10::optional<at::Tensor>& status, const at::Tensor& anchor) {
  if (!status) return status_like(anchor);
  check(*status, at::kInt, anchor);
  TORCH_CHECK(status->numel() == 1, "status must hold one int32");
  return *status;
}

int element_type(const at::Tensor& t, const char* what) {
  TORCH_CHECK(t.scalar_type() == at::kBFloat16 || t.scalar_type() == at::kFloat, what, ": BF16 or FP32 expected");
  return t.scalar_type() == at::kFloat ? DSR_F32 : DSR_BF16;
}

// A tensor of the caller's that is written through its pointer: autograd would take what was
// there before for its value, so one with a history (or a leaf) is refused, as torch refuses
// it, and one that autograd may have saved is marked as changed.
void overwrite(const at::Tensor& t, const char* what) {
  TORCH_CHECK(!(at::GradMode::is_enabled() && t.requires_grad()), what,
              ": the output requires a gradient, which this call does not track");
  if (!t.is_inference()) t.unsafeGetTensorImpl()->bump_version();
}

// An uninitialised tensor without the dispatcher's round trip (a small call is made of these).
at::Tensor fresh(at::IntArrayRef sizes, at::ScalarType dtype, const at::Tensor& anchor) {
  return at::detail::empty_cuda(sizes, dtype, anchor.device(), c10::nullopt);
}

void check_vector(const at::Tensor& t, at::ScalarType dtype, int64_t n, const at::Tensor& anchor, const char* what) {
  check(t, dtype, anchor);
  TORCH_CHECK(t.dim() == 1 && t.size(0) == n, what);
}

std::vector<at::Tensor> ds_paged_plan(at::Tensor lengths, at::Tensor new_tokens, at::Tensor held,
                                      at::Tensor block_table, at::Tensor free_ring, at::Tensor ring_state,
                                      int64_t tokens, c10::optional<at::Tensor> status,
                                      c10::optional<at::Tensor> shares) {
  check(lengths, at::kInt, lengths);
  const int64_t batch = lengths.numel();
  const char* shapes =
      "paged_plan: lengths, new_tokens, held [batch], block_table [batch, blocks], free_ring [pool blocks] and "
      "ring_state [4] expected";
  check_vector(lengths, at::kInt, batch, lengths, shapes);
  check_vector(new_tokens, at::kInt, batch, lengths, shapes);
  check_vector(held, at::kInt, batch, lengths, shapes);
  check(block_table, at::kInt, lengths);
  TORCH_CHECK(block_table.dim() == 2 && block_table.size(0) == batch, shapes);
  check_vector(free_ring, at::kInt, free_ring.numel(), lengths, shapes);
  check_vector(ring_state, at::kInt, 4, lengths, shapes);
  if (shares) check_vector(*shares, at::kInt, free_ring.numel(), lengths, "paged_plan: shares [pool blocks] expected");
  TORCH_CHECK(tokens >= 0 && tokens < (int64_t(1) << 31), "paged_plan: invalid token count");
  const c10::cuda::CUDAGuard guard(lengths.device());
  auto error = status_or(status, lengths);
  // one allocation for the five outputs, each from a 16-byte boundary
  const auto rounded = [](int64_t n) { return (n + 3) / 4 * 4; };
  const at::Tensor store = fresh({3 * rounded(tokens) + rounded(batch + 1) + rounded(batch)}, at::kInt, lengths);
  int64_t used = 0;
  const auto part = [&](int64_t n) {
    auto t = at::detail::make_tensor<c10::TensorImpl>(c10::Storage(store.storage()), store.key_set(), store.dtype());
    t.unsafeGetTensorImpl()->set_storage_offset(used);
    t.unsafeGetTensorImpl()->set_sizes_contiguous({n});
    used += rounded(n);
    return t;
  };
  auto seq = part(tokens), positions = part(tokens), slots = part(tokens), cu = part(batch + 1), visible = part(batch);
  const auto call = [&](auto plan, auto... extra) {
    return plan(lengths.data_ptr<int32_t>(), new_tokens.data_ptr<int32_t>(), held.data_ptr<int32_t>(),
                block_table.data_ptr<int32_t>(), block_table.size(1), free_ring.data_ptr<int32_t>(),
                ring_state.data_ptr<int32_t>(), extra..., free_ring.size(0), seq.data_ptr<int32_t>(),
                positions.data_ptr<int32_t>(), slots.data_ptr<int32_t>(), tokens, cu.data_ptr<int32_t>(),
                visible.data_ptr<int32_t>(), error.data_ptr<int32_t>(), batch, current_stream());
  };
  ok(shares ? call(dsr_paged_plan_shared, shares->data_ptr<int32_t>()) : call(dsr_paged_plan));
  return {seq, positions, slots, cu, visible, error};
}

// ---- blocks that several requests map
// The five tables of a paged cache: their shapes, and what they are called with.
struct PageTables {
  at::Tensor held, table, ring, state, shares;
  int64_t batch, stride, blocks;
  PageTables(const at::Tensor& held_, const at::Tensor& table_, const at::Tensor& ring_, const at::Tensor& state_,
             const at::Tensor& shares_)
      : held(held_), table(table_), ring(ring_), state(state_), shares(shares_) {
    const char* shapes =
        "held [batch], block_table [batch, blocks], free_ring [pool blocks], ring_state [4] and shares [pool blocks] "
        "expected";
    check_vector(held, at::kInt, held.numel(), held, shapes);
    check(table, at::kInt, held);
    batch = held.numel();
    TORCH_CHECK(table.dim() == 2 && table.size(0) == batch, shapes);
    check_vector(ring, at::kInt, ring.numel(), held, shapes);
    check_vector(state, at::kInt, 4, held, shapes);
    check_vector(shares, at::kInt, ring.numel(), held, shapes);
    stride = table.size(1), blocks = ring.numel();
  }
};

// moves [n, 4] and count [1], and a call's scratch, of one allocation.
struct MoveList {
  at::Tensor moves, count;
  void* scratch;
  size_t scratch_bytes;
};
MoveList move_list(int64_t n, const at::Tensor& anchor, size_t scratch_bytes = 0) {
  const int64_t used = (4 * n + 4 + 63) / 64 * 64;  // 256 bytes
  const at::Tensor store = fresh({used + int64_t(scratch_bytes + 3) / 4}, at::kInt, anchor);
  const auto part = [&](int64_t offset, at::IntArrayRef sizes) {
    auto t = at::detail::make_tensor<c10::TensorImpl>(c10::Storage(store.storage()), store.key_set(), store.dtype());
    t.unsafeGetTensorImpl()->set_storage_offset(offset);
    t.unsafeGetTensorImpl()->set_sizes_contiguous(sizes);
    return t;
  };
  return {part(4, {n, 4}), part(0, {1}), store.data_ptr<int32_t>() + used, scratch_bytes};
}

std::vector<at::Tensor> ds_paged_fork(at::Tensor parent, at::Tensor lengths, at::Tensor held, at::Tensor block_table,
                                      at::Tensor free_ring, at::Tensor ring_state, at::Tensor shares,
                                      c10::optional<at::Tensor> status) {
  PageTables t(held, block_table, free_ring, ring_state, shares);
  check_vector(parent, at::kInt, t.batch, held, "paged_fork: parent [batch] expected");
  check_vector(lengths, at::kInt, t.batch, held, "paged_fork: lengths [batch] expected");
  const c10::cuda::CUDAGuard guard(held.device());
  auto error = status_or(status, held);
  const MoveList list = move_list(t.batch, held);
  ok(dsr_paged_fork(parent.data_ptr<int32_t>(), lengths.data_ptr<int32_t>(), held.data_ptr<int32_t>(),
                    block_table.data_ptr<int32_t>(), t.stride, free_ring.data_ptr<int32_t>(),
                    ring_state.data_ptr<int32_t>(), shares.data_ptr<int32_t>(), t.blocks, list.moves.data_ptr<int32_t>(),
                    list.count.data_ptr<int32_t>(), error.data_ptr<int32_t>(), t.batch, current_stream()));
  return {list.moves, list.count, error};
}

std::vector<at::Tensor> ds_paged_release(at::Tensor lengths, at::Tensor held, at::Tensor block_table,
                                         at::Tensor free_ring, at::Tensor ring_state, at::Tensor shares,
                                         c10::optional<at::Tensor> status) {
  PageTables t(held, block_table, free_ring, ring_state, shares);
  check_vector(lengths, at::kInt, t.batch, held, "paged_release: lengths [batch] expected");
  const c10::cuda::CUDAGuard guard(held.device());
  auto error = status_or(status, held);
  const MoveList list = move_list(t.batch, held, dsr_paged_release_workspace_bytes(t.batch, t.blocks));
  ok(dsr_paged_release(lengths.data_ptr<int32_t>(), held.data_ptr<int32_t>(), block_table.data_ptr<int32_t>(),
                       t.stride, free_ring.data_ptr<int32_t>(), ring_state.data_ptr<int32_t>(),
                       shares.data_ptr<int32_t>(), t.blocks, list.moves.data_ptr<int32_t>(), list.count.data_ptr<int32_t>(),
                       list.scratch, list.scratch_bytes, error.data_ptr<int32_t>(), t.batch, current_stream()));
  return {list.moves, list.count, error};
}

std::vector<at::Tensor> ds_paged_compact(at::Tensor held, at::Tensor block_table, at::Tensor free_ring,
                                         at::Tensor ring_state, at::Tensor shares, c10::optional<at::Tensor> status) {
  PageTables t(held, block_table, free_ring, ring_state, shares);
  const c10::cuda::CUDAGuard guard(held.device());
  auto error = status_or(status, held);
  const MoveList list =
      move_list(std::max<int64_t>(t.blocks / 2, 1), held, dsr_paged_compact_workspace_bytes(t.blocks));
  ok(dsr_paged_compact(held.data_ptr<int32_t>(), block_table.data_ptr<int32_t>(), t.stride,
                       free_ring.data_ptr<int32_t>(), ring_state.data_ptr<int32_t>(), shares.data_ptr<int32_t>(),
                       t.blocks, list.moves.data_ptr<int32_t>(), list.count.data_ptr<int32_t>(), list.scratch, list.scratch_bytes,
                       error.data_ptr<int32_t>(), t.batch, current_stream()));
  return {list.moves, list.count, error};
}

at::Tensor ds_paged_copy(std::vector<at::Tensor> pools, std::vector<at::Tensor> generations, at::Tensor moves,
                         at::Tensor count, c10::optional<at::Tensor> status) {
  check(moves, at::kInt, moves);
  TORCH_CHECK(moves.dim() == 2 && moves.size(1) == 4, "paged_copy: moves [n, 4] expected");
  check_vector(count, at::kInt, 1, moves, "paged_copy: count [1] expected");
  const c10::cuda::CUDAGuard guard(moves.device());
  auto error = status_or(status, moves);
  if (pools.empty() && generations.empty()) return error;
  const int64_t rows = (pools.empty() ? generations : pools)[0].size(0);
  for (const at::Tensor& p : pools) {
    check(p, p.scalar_type(), moves);
    TORCH_CHECK(p.dim() == 2 && p.size(0) == rows, "paged_copy: pools [rows, width] of as many rows expected");
    const int64_t bytes = p.size(1) * p.element_size();  // before the first of several launches
    TORCH_CHECK(bytes > 0 && bytes <= 65536 && bytes % 16 == 0 && reinterpret_cast<uintptr_t>(p.data_ptr()) % 16 == 0,
                "paged_copy: 16-byte aligned rows of 16 to 65536 bytes expected");
  }
  for (const at::Tensor& g : generations)
    check_vector(g, at::kLong, rows, moves, "paged_copy: generations [rows] of the pools' rows expected");
  constexpr size_t most = 64;  // of a launch, whose own check is of its generations
  std::vector<const int64_t*> all;
  for (const at::Tensor& g : generations) all.push_back(g.data_ptr<int64_t>());
  std::sort(all.begin(), all.end());
  TORCH_CHECK(std::adjacent_find(all.begin(), all.end(), [&](auto a, auto b) { return b - a < rows; }) == all.end(),
              "paged_copy: the same generations twice");
  for (const at::Tensor& p : pools) overwrite(p, "paged_copy");
  for (size_t i = 0; i < std::max(pools.size(), generations.size()); i += most) {
    std::vector<void*> data;
    std::vector<int64_t> bytes;
    std::vector<int64_t*> gens;
    for (size_t j = i; j < std::min(i + most, pools.size()); ++j)
      data.push_back(pools[j].data_ptr()), bytes.push_back(pools[j].size(1) * pools[j].element_size());
    for (size_t j = i; j < std::min(i + most, generations.size()); ++j) gens.push_back(generations[j].data_ptr<int64_t>());
    ok(dsr_paged_copy(data.data(), bytes.data(), int64_t(data.size()), gens.data(), int64_t(gens.size()), rows,
                      moves.data_ptr<int32_t>(), count.data_ptr<int32_t>(), moves.size(0), error.data_ptr<int32_t>(),
                      current_stream()));
  }
  return error;
}

at::Tensor ds_rope(std::vector<at::Tensor> x, std::vector<at::Tensor> out, at::Tensor positions,
                   at::Tensor frequencies, std::vector<int64_t> offsets, std::vector<bool> interleaved, double mscale,
                   bool inverse, c10::optional<at::Tensor> status) {
  check(positions, at::kInt, positions);
  check(frequencies, at::kDouble, positions);
  TORCH_CHECK(positions.dim() == 1 && frequencies.dim() == 1, "rope: positions [tokens] and frequencies [pairs] expected");
  TORCH_CHECK(!x.empty() && x.size() <= 4 && out.size() == x.size() && offsets.size() == x.size() &&
                  interleaved.size() == x.size(),
              "rope: 1 to 4 tensors, each with its output, offset and layout, expected");
  const int64_t tokens = positions.size(0);
  const c10::cuda::CUDAGuard guard(positions.device());
  auto error = status_or(status, positions);
  if (tokens == 0) return error;
  dsr_rope_tensor desc[4] = {};
  for (size_t i = 0; i < x.size(); ++i) {
    const at::Tensor &a = x[i], &b = out[i];
    TORCH_CHECK(a.is_cuda() && a.device() == positions.device() && b.is_cuda() && b.device() == positions.device(),
                "all inputs require the same CUDA device");
    TORCH_CHECK((a.dim() == 2 || a.dim() == 3) && a.size(0) == tokens && a.sizes() == b.sizes() &&
                    a.scalar_type() == b.scalar_type(),
                "rope: x and out [tokens, width] or [tokens, heads, width] of one type expected");
    TORCH_CHECK(a.numel() > 0 && (a.size(-1) == 1 || (a.stride(-1) == 1 && b.stride(-1) == 1)),
                "rope: the columns of x and out must be contiguous");
    const bool heads = a.dim() == 3;
    desc[i].x = a.data_ptr();
    desc[i].out = b.data_ptr();
    desc[i].x_token = a.stride(0);
    desc[i].out_token = b.stride(0);
    desc[i].x_head = heads ? a.stride(1) : 0;
    desc[i].out_head = heads ? b.stride(1) : 0;
    TORCH_CHECK(a.size(-1) <= 65536 && (!heads || a.size(1) <= 65536) && offsets[i] >= 0 && offsets[i] <= a.size(-1),
                "rope: invalid heads, width or offset");
    desc[i].heads = heads ? int32_t(a.size(1)) : 1;
    desc[i].width = int32_t(a.size(-1));
    desc[i].offset = int32_t(offsets[i]);
    desc[i].interleaved = interleaved[i];
    desc[i].dtype = element_type(a, "rope");
  }
  for (const at::Tensor& b : out) overwrite(b, "rope");
  ok(dsr_rope(desc, int64_t(x.size()), positions.data_ptr<int32_t>(), frequencies.data_ptr<double>(),
              frequencies.size(0), static_cast<float>(mscale), inverse, error.data_ptr<int32_t>(), tokens,
              current_stream()));
  return error;
}

std::vector<at::Tensor> ds_tree_mla_decode(at::Tensor q, at::Tensor kv_pool, at::Tensor block_table,
                                           at::Tensor context, at::Tensor cu_nodes, at::Tensor tree_mask,
                                           int64_t max_nodes, double scale, c10::optional<at::Tensor> sink,
                                           bool return_lse, c10::optional<at::Tensor> out,
                                           c10::optional<at::Tensor> status) {
  const int dtype = element_type(q, "tree_mla_decode");
  check(q, q.scalar_type(), q);
  check_cache(kv_pool, q);
  check(block_table, at::kInt, q);
  TORCH_CHECK(q.dim() == 3 && q.size(0) > 0 && q.size(2) == DSR_KV_DIM,
              "tree_mla_decode: q [nodes, heads, 576] expected");
  const int64_t nodes = q.size(0), heads = q.size(1), batch = context.numel();
  const char* shapes =
      "tree_mla_decode: context [batch], cu_nodes [batch + 1], tree_mask [nodes], block_table [batch, blocks], "
      "kv_pool [blocks*64, 576] and sink [heads] expected";
  check_vector(context, at::kInt, batch, q, shapes);
  check_vector(cu_nodes, at::kInt, batch + 1, q, shapes);
  check_vector(tree_mask, at::kLong, nodes, q, shapes);
  TORCH_CHECK(block_table.dim() == 2 && block_table.size(0) == batch && kv_pool.dim() == 2 &&
                  kv_pool.size(1) == DSR_KV_DIM && kv_pool.size(0) % DSR_BLOCK_TOKENS == 0,
              shapes);
  if (sink) check_vector(*sink, at::kFloat, heads, q, shapes);
  const c10::cuda::CUDAGuard guard(q.device());
  auto error = status_or(status, q);
  at::Tensor result;
  if (out) {
    result = *out;
    element_type(result, "tree_mla_decode");
    check(result, result.scalar_type(), q);
    TORCH_CHECK(result.dim() == 3 && result.size(0) == nodes && result.size(1) == heads &&
                    result.size(2) == DSR_V_DIM,
                "tree_mla_decode: out [nodes, heads, 512] expected");
    overwrite(result, "tree_mla_decode");
  } else {
    result = fresh({nodes, heads, DSR_V_DIM}, q.scalar_type(), q);
  }
  // what this call allocates has no row that nobody wrote; the caller's rows stay
  const int unused = out ? 0 : DSR_ZERO_UNUSED;
  at::Tensor lse;
  if (return_lse) lse = out ? at::full({nodes, heads}, -INFINITY, q.options().dtype(at::kFloat)) : fresh({nodes, heads}, at::kFloat, q);
  const size_t ws_bytes = dsr_tree_mla_workspace_bytes(batch, heads, max_nodes);
  auto ws = fresh({int64_t(ws_bytes)}, at::kByte, q);
  ok(dsr_tree_mla_decode(q.data_ptr(), dtype, bf16(kv_pool), kv_pool.size(0) / DSR_BLOCK_TOKENS,
                         block_table.data_ptr<int32_t>(), block_table.size(1), context.data_ptr<int32_t>(),
                         cu_nodes.data_ptr<int32_t>(), tree_mask.data_ptr<int64_t>(), max_nodes,
                         sink ? sink->data_ptr<float>() : nullptr, static_cast<float>(scale), result.data_ptr(),
                         element_type(result, "tree_mla_decode") | unused, return_lse ? lse.data_ptr<float>() : nullptr,
                         ws.data_ptr(), ws_bytes, error.data_ptr<int32_t>(), batch, nodes, heads, current_stream()));
  if (return_lse) return {result, error, lse};
  return {result, error};
}

std::vector<at::Tensor> ds_prefix_mla_decode(at::Tensor q, at::Tensor kv_pool, at::Tensor block_table,
                                             at::Tensor context, at::Tensor cu_nodes, at::Tensor tree_mask,
                                             int64_t max_nodes, at::Tensor prefix, at::Tensor holder, double scale,
                                             c10::optional<at::Tensor> sink, bool return_lse,
                                             c10::optional<at::Tensor> out, c10::optional<at::Tensor> status) {
  const int dtype = element_type(q, "prefix_mla_decode");
  check(q, q.scalar_type(), q);
  check_cache(kv_pool, q);
  check(block_table, at::kInt, q);
  TORCH_CHECK(q.dim() == 3 && q.size(0) > 0 && q.size(2) == DSR_KV_DIM,
              "prefix_mla_decode: q [nodes, heads, 576] expected");
  const int64_t nodes = q.size(0), heads = q.size(1), batch = context.numel();
  const char* shapes =
      "prefix_mla_decode: context, prefix, holder [batch], cu_nodes [batch + 1], tree_mask [nodes], block_table "
      "[batch or more, blocks], kv_pool [blocks*64, 576] and sink [heads] expected";
  check_vector(context, at::kInt, batch, q, shapes);
  check_vector(prefix, at::kInt, batch, q, shapes);
  check_vector(holder, at::kInt, batch, q, shapes);
  check_vector(cu_nodes, at::kInt, batch + 1, q, shapes);
  check_vector(tree_mask, at::kLong, nodes, q, shapes);
  TORCH_CHECK(block_table.dim() == 2 && block_table.size(0) >= batch && kv_pool.dim() == 2 &&
                  kv_pool.size(1) == DSR_KV_DIM && kv_pool.size(0) % DSR_BLOCK_TOKENS == 0,
              shapes);
  if (sink) check_vector(*sink, at::kFloat, heads, q, shapes);
  const c10::cuda::CUDAGuard guard(q.device());
  auto error = status_or(status, q);
  at::Tensor result;
  if (out) {
    result = *out;
    element_type(result, "prefix_mla_decode");
    check(result, result.scalar_type(), q);
    TORCH_CHECK(result.dim() == 3 && result.size(0) == nodes && result.size(1) == heads &&
                    result.size(2) == DSR_V_DIM,
                "prefix_mla_decode: out [nodes, heads, 512] expected");
    overwrite(result, "prefix_mla_decode");
  } else {
    result = fresh({nodes, heads, DSR_V_DIM}, q.scalar_type(), q);
  }
  const int unused = out ? 0 : DSR_ZERO_UNUSED;  // as in tree_mla_decode
  at::Tensor lse;
  if (return_lse && out) lse = at::full({nodes, heads}, -INFINITY, q.options().dtype(at::kFloat));
  else if (return_lse) lse = fresh({nodes, heads}, at::kFloat, q);
  const size_t ws_bytes = dsr_prefix_mla_workspace_bytes(batch, nodes, heads);
  auto ws = fresh({int64_t(ws_bytes)}, at::kByte, q);
  ok(dsr_prefix_mla_decode(q.data_ptr(), dtype, bf16(kv_pool), kv_pool.size(0) / DSR_BLOCK_TOKENS,
                           block_table.data_ptr<int32_t>(), block_table.size(0), block_table.size(1),
                           context.data_ptr<int32_t>(), cu_nodes.data_ptr<int32_t>(), tree_mask.data_ptr<int64_t>(),
                           max_nodes, prefix.data_ptr<int32_t>(), holder.data_ptr<int32_t>(),
                           sink ? sink->data_ptr<float>() : nullptr, static_cast<float>(scale), result.data_ptr(),
                           element_type(result, "prefix_mla_decode") | unused,
                           return_lse ? lse.data_ptr<float>() : nullptr, ws.data_ptr(), ws_bytes,
                           error.data_ptr<int32_t>(), batch, nodes, heads, current_stream()));
  if (return_lse) return {result, error, lse};
  return {result, error};
}

std::vector<at::Tensor> ds_sample_logits(at::Tensor logits, at::Tensor temperature, at::Tensor top_k,
                                         at::Tensor top_p, at::Tensor min_p, at::Tensor uniform,
                                         c10::optional<at::Tensor> status) {
  TORCH_CHECK(logits.is_cuda(), "all inputs require the same CUDA device");
  const int dtype = element_type(logits, "sample_logits");
  TORCH_CHECK(logits.dim() == 2 && logits.size(0) > 0 && logits.size(1) > 0 &&
                  (logits.size(1) == 1 || logits.stride(1) == 1),
              "sample_logits: logits [rows, vocab] with contiguous columns expected");
  const int64_t rows = logits.size(0);
  const char* shapes = "sample_logits: temperature, top_k, top_p, min_p and uniform [rows] expected";
  check_vector(temperature, at::kFloat, rows, logits, shapes);
  check_vector(top_k, at::kInt, rows, logits, shapes);
  check_vector(top_p, at::kFloat, rows, logits, shapes);
  check_vector(min_p, at::kFloat, rows, logits, shapes);
  check_vector(uniform, at::kFloat, rows, logits, shapes);
  const c10::cuda::CUDAGuard guard(logits.device());
  auto error = status_or(status, logits);
  auto tokens = fresh({rows}, at::kInt, logits), chances = fresh({rows}, at::kFloat, logits);
  ok(dsr_sample(logits.data_ptr(), dtype, logits.stride(0), logits.size(1), temperature.data_ptr<float>(),
                top_k.data_ptr<int32_t>(), top_p.data_ptr<float>(), min_p.data_ptr<float>(),
                uniform.data_ptr<float>(), tokens.data_ptr<int32_t>(), chances.data_ptr<float>(),
                error.data_ptr<int32_t>(), rows, current_stream()));
  return {tokens, chances, error};
}

PYBIND11_MODULE(TORCH_EXTENSION_NAME, m) {
  m.def("sparse_attention", &ds_sparse_attention);
  m.def("index_scores", &ds_index_scores);
  m.def("engram_decode", &ds_engram_decode);
  m.def("scatter_slots", &ds_scatter_slots);
  m.def("abi_version", [] { return dsr_abi_version(); });
  m.def("topk_select", &ds_topk_select, py::arg("scores"), py::arg("lengths"), py::arg("k"),
        py::arg("ids") = py::none(), py::arg("id_base") = 0, py::arg("return_scores") = false);
  m.def("indexer_decode", &ds_indexer_decode);
  m.def("sparse_mla_decode", &ds_sparse_mla_decode);
  m.def("append_kv_index", &ds_append_kv_index, py::arg("kv_pool"), py::arg("index_pool"),
        py::arg("generations"), py::arg("block_table"), py::arg("seq"), py::arg("positions"),
        py::arg("expected"), py::arg("kv_values"), py::arg("index_values"), py::arg("swa") = py::none());
  m.def("lse_combine", &ds_lse_combine, py::arg("part_o"), py::arg("part_m"), py::arg("part_l"),
        py::arg("sink") = py::none());
  m.def("decode_step", &ds_decode_step, py::arg("idx_q"), py::arg("idx_w"), py::arg("index_pool"),
        py::arg("q"), py::arg("kv_pool"), py::arg("block_table"), py::arg("visible"),
        py::arg("max_visible"), py::arg("k"), py::arg("swa"), py::arg("swa_len"), py::arg("sink"),
        py::arg("scale"), py::arg("return_scores") = false);
  m.def("indexer_decode_ring", &ds_indexer_decode_ring, py::arg("q"), py::arg("weights"), py::arg("index_pool"),
        py::arg("ring"), py::arg("visible"), py::arg("score_stride"));
  m.def("sparse_mla_decode_ring", &ds_sparse_mla_decode_ring, py::arg("q"), py::arg("kv_pool"),
        py::arg("kv_ring"), py::arg("visible"), py::arg("topk"), py::arg("swa_pool"), py::arg("swa_ring"),
        py::arg("swa_len"), py::arg("sink"), py::arg("scale"));
  m.def("decode_step_ring", &ds_decode_step_ring, py::arg("idx_q"), py::arg("idx_w"), py::arg("index_pool"),
        py::arg("index_ring"), py::arg("q"), py::arg("kv_pool"), py::arg("kv_ring"), py::arg("visible"),
        py::arg("max_visible"), py::arg("k"), py::arg("swa_pool"), py::arg("swa_ring"), py::arg("swa_len"),
        py::arg("sink"), py::arg("scale"), py::arg("return_scores") = false);
  m.def("append_kv_index_ring", &ds_append_kv_index_ring, py::arg("kv_pool"), py::arg("kv_ring"),
        py::arg("kv_generations"), py::arg("kv_expected"), py::arg("index_pool"), py::arg("index_ring"),
        py::arg("index_generations"), py::arg("index_expected"), py::arg("seq"), py::arg("positions"),
        py::arg("kv_values"), py::arg("index_values"));
  m.def("paged_plan", &ds_paged_plan, py::arg("lengths"), py::arg("new_tokens"), py::arg("held"),
        py::arg("block_table"), py::arg("free_ring"), py::arg("ring_state"), py::arg("tokens"),
        py::arg("status") = py::none(), py::arg("shares") = py::none());
  m.def("paged_fork", &ds_paged_fork, py::arg("parent"), py::arg("lengths"), py::arg("held"),
        py::arg("block_table"), py::arg("free_ring"), py::arg("ring_state"), py::arg("shares"),
        py::arg("status") = py::none());
  m.def("paged_release", &ds_paged_release, py::arg("lengths"), py::arg("held"), py::arg("block_table"),
        py::arg("free_ring"), py::arg("ring_state"), py::arg("shares"), py::arg("status") = py::none());
  m.def("paged_compact", &ds_paged_compact, py::arg("held"), py::arg("block_table"), py::arg("free_ring"),
        py::arg("ring_state"), py::arg("shares"), py::arg("status") = py::none());
  m.def("paged_copy", &ds_paged_copy, py::arg("pools"), py::arg("generations"), py::arg("moves"), py::arg("count"),
        py::arg("status") = py::none());
  m.def("rope", &ds_rope, py::arg("x"), py::arg("out"), py::arg("positions"), py::arg("frequencies"),
        py::arg("offsets"), py::arg("interleaved"), py::arg("mscale") = 1.0, py::arg("inverse") = false,
        py::arg("status") = py::none());
  m.def("tree_mla_decode", &ds_tree_mla_decode, py::arg("q"), py::arg("kv_pool"), py::arg("block_table"),
        py::arg("context"), py::arg("cu_nodes"), py::arg("tree_mask"), py::arg("max_nodes"), py::arg("scale"),
        py::arg("sink") = py::none(), py::arg("return_lse") = false, py::arg("out") = py::none(),
        py::arg("status") = py::none());
  m.def("prefix_mla_decode", &ds_prefix_mla_decode, py::arg("q"), py::arg("kv_pool"), py::arg("block_table"),
        py::arg("context"), py::arg("cu_nodes"), py::arg("tree_mask"), py::arg("max_nodes"), py::arg("prefix"),
        py::arg("holder"), py::arg("scale"), py::arg("sink") = py::none(), py::arg("return_lse") = false,
        py::arg("out") = py::none(), py::arg("status") = py::none());
  m.def("sample_logits", &ds_sample_logits, py::arg("logits"), py::arg("temperature"), py::arg("top_k"),
        py::arg("top_p"), py::arg("min_p"), py::arg("uniform"), py::arg("status") = py::none());
}
