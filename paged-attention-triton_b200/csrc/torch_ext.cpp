// torch_ext.cpp -- thin PyTorch extension over the C ABI (include/pa_decode.h).
//
// One Python call = argument checks, output allocation from the caching
// allocator, a workspace-size query and one pa_decode launch on the current
// CUDA stream, all in C++ (the equivalent Python/ctypes path costs ~15 us per
// call). The launcher itself lives in libpa_decode.so; this module only maps
// at::Tensor arguments onto pa_decode_params.
//
// Reference interface: paged_attention(Q, K_Cache, V_Cache, Block_Table,
// seq_len, block_size, num_splits) (paged_attention/torch_kernel.py:71-73).
#include <torch/extension.h>
#include <c10/core/AutogradState.h>
#include <c10/cuda/CUDAStream.h>
#include <c10/cuda/CUDAGuard.h>
#include <c10/cuda/CUDAGraphsC10Utils.h>

#include <cmath>
#include <tuple>
#include <vector>

#include "pa_decode.h"

namespace {

void check(bool cond, const char* msg) { TORCH_CHECK_VALUE(cond, "paged_attention: ", msg); }

int dtype_code(const at::Tensor& t) {
  if (t.scalar_type() == at::kHalf) return PA_F16;
  if (t.scalar_type() == at::kBFloat16) return PA_BF16;
  TORCH_CHECK_VALUE(false, "paged_attention: unsupported dtype ", t.scalar_type(),
                    " (fp16 or bf16)");
  return -1;
}

// Forward-mode tangents would be dropped: such inputs are refused, as gradients are.
bool has_tangent(const at::Tensor& t) {
  return c10::AutogradState::get_tls_state().get_fw_grad_mode() && t._fw_grad(0).defined();
}

// Queries whose rows start on 16 bytes, one element apart: the tensor itself or a copy
// (clone, as contiguous() hands back a tensor whose address, or the stride of a dimension
// of one, is the trouble).
at::Tensor aligned_rows(const at::Tensor& q) {
  if (q.stride(2) == 1 && q.stride(0) % 8 == 0 && q.stride(1) % 8 == 0 &&
      reinterpret_cast<uintptr_t>(q.data_ptr()) % 16 == 0)
    return q;
  return q.clone(at::MemoryFormat::Contiguous);
}

// Returns (status, tensors): status 0 and [out[, lse][, o_partial, lse_partial]]
// on success; when the workspace is too small nothing is launched and the
// result is (-1, []) with the needed sizes in the last two fields.
std::tuple<int64_t, std::vector<at::Tensor>, int64_t, int64_t> window_decode(
    const at::Tensor& q, const at::Tensor& k, const at::Tensor& v, const at::Tensor& bt,
    const c10::optional<at::Tensor>& seq_lens, int64_t seq_len, int64_t block_size,
    int64_t num_splits, double scale, bool return_lse, bool return_partials,
    const at::Tensor& ws_buffer, const at::Tensor& ws_counters, const at::Tensor& ws_status,
    int64_t kernel_variant, const c10::optional<at::Tensor>& out_opt, int64_t window,
    int64_t num_sinks) {
  check(q.is_cuda() && k.is_cuda() && v.is_cuda() && bt.is_cuda(),
        "Q, K_Cache, V_Cache and Block_Table must be CUDA tensors");
  check(q.dim() == 3, "Q must be [B, H, D]");
  check(k.dim() == 4 && v.sizes() == k.sizes(),
        "K_Cache and V_Cache must both be [num_blocks, block_size, Hkv, D]");
  const int dt = dtype_code(q);
  check(k.scalar_type() == q.scalar_type() && v.scalar_type() == q.scalar_type(),
        "Q, K_Cache and V_Cache must share one dtype");
  check(bt.scalar_type() == at::kInt && bt.dim() == 2,
        "Block_Table must be an int32 [B, max_blocks] tensor");
  const auto dev = q.device();
  check(k.device() == dev && v.device() == dev && bt.device() == dev,
        "tensors on different devices");
  const int64_t batch = q.size(0), heads = q.size(1), dim = q.size(2);
  const int64_t nblocks = k.size(0), bs = k.size(1), kv_heads = k.size(2);
  check(k.size(3) == dim, "head_dim of Q and the caches differ");
  check(dim == 32 || dim == 64 || dim == 128 || dim == 256,
        "head_dim must be 32, 64, 128 or 256");
  check(block_size == bs, "block_size differs from the cache's block dimension");
  check(bs >= 1, "block_size must be positive");
  check(kv_heads > 0 && heads % kv_heads == 0, "Hq must be a multiple of Hkv");
  check(bt.size(0) == batch, "Block_Table rows != batch");
  check(q.stride(2) == 1 && k.stride(3) == 1 && v.stride(3) == 1 && bt.stride(1) == 1,
        "last dimensions must be contiguous");
  const int64_t max_blocks = bt.size(1);

  c10::cuda::CUDAGuard guard(dev);
  const at::Tensor Q = aligned_rows(q);
  at::Tensor lens;
  if (seq_lens.has_value()) {
    lens = *seq_lens;
    check(lens.numel() == batch, "seq_lens must have B entries");
    if (lens.device() != dev || lens.scalar_type() != at::kInt || !lens.is_contiguous())
      lens = lens.to(dev, at::kInt).contiguous();
  } else {
    check(seq_len >= 0 && seq_len <= max_blocks * bs, "seq_len exceeds the Block_Table capacity");
  }
  check(num_splits >= 0, "num_splits must be >= 0");
  // window 0: every cached token is visible
  check(window >= 0 && window <= INT32_MAX && num_sinks >= 0 && num_sinks <= INT32_MAX,
        "window must be at least 1 and num_sinks at least 0");
  check(window > 0 || num_sinks == 0, "num_sinks goes with a window");
  TORCH_CHECK(window == 0 || !(has_tangent(q) || has_tangent(k) || has_tangent(v)),
              "PagedAttentionV2 is inference-only.");
  check(window == 0 || (num_splits == 0 && !return_partials),
        "a window goes with the default schedule (no num_splits, no return_partials)");
  int64_t ns = num_splits;
  if (return_partials && ns == 0) {
    const int64_t s = seq_lens.has_value() ? max_blocks * bs : seq_len;
    ns = pa_num_splits_heuristic(static_cast<int32_t>(batch), static_cast<int32_t>(heads),
                                 static_cast<int32_t>(s), static_cast<int32_t>(bs),
                                 pa_device_sm_count());
  }

  const auto opts = Q.options();
  at::Tensor out = out_opt.has_value() ? *out_opt : at::empty({batch, heads, dim}, opts);
  // (pinned host memory is the device's too; a peer's is the caller's to make reachable)
  check(out.device() == dev || out.is_pinned() || (window == 0 && out.is_cuda()),
        "out must be on Q's device");
  check(out.sizes() == Q.sizes() && out.scalar_type() == Q.scalar_type() && out.stride(2) == 1,
        "out must match Q's shape and dtype");
  check(ws_status.device() == dev, "the workspace is on another device");
  const auto f32 = opts.dtype(at::kFloat);
  at::Tensor lse, o_part, lse_part;
  if (return_lse) lse = at::empty({batch, heads}, f32);
  if (return_partials) {
    o_part = at::empty({batch, heads, ns, dim}, f32);
    lse_part = at::empty({batch, heads, ns}, f32);
  }

  pa_decode_params p{};
  p.q = Q.data_ptr();
  p.q_stride_b = Q.stride(0);
  p.q_stride_h = Q.stride(1);
  p.k_cache = k.data_ptr();
  p.k_stride_block = k.stride(0);
  p.k_stride_slot = k.stride(1);
  p.k_stride_head = k.stride(2);
  p.v_cache = v.data_ptr();
  p.v_stride_block = v.stride(0);
  p.v_stride_slot = v.stride(1);
  p.v_stride_head = v.stride(2);
  p.block_table = bt.data_ptr<int32_t>();
  p.bt_stride_b = bt.stride(0);
  p.max_blocks = static_cast<int32_t>(max_blocks);
  p.seq_lens = seq_lens.has_value() ? lens.data_ptr<int32_t>() : nullptr;
  p.seq_len = seq_lens.has_value() ? 0 : static_cast<int32_t>(seq_len);
  p.batch = static_cast<int32_t>(batch);
  p.num_heads = static_cast<int32_t>(heads);
  p.num_kv_heads = static_cast<int32_t>(kv_heads);
  p.head_dim = static_cast<int32_t>(dim);
  p.block_size = static_cast<int32_t>(bs);
  p.num_blocks = static_cast<int32_t>(nblocks);
  p.num_splits = static_cast<int32_t>(ns);
  p.scale = static_cast<float>(scale > 0 ? scale : 1.0 / std::sqrt(static_cast<double>(dim)));
  p.dtype = dt;
  p.out = out.data_ptr();
  p.out_stride_b = out.stride(0);
  p.out_stride_h = out.stride(1);
  p.lse = return_lse ? lse.data_ptr<float>() : nullptr;
  p.o_partial = return_partials ? o_part.data_ptr<float>() : nullptr;
  p.lse_partial = return_partials ? lse_part.data_ptr<float>() : nullptr;
  p.kernel_variant = static_cast<int32_t>(kernel_variant);

  size_t ws_bytes = 0, n_counters = 0;
  const auto win = static_cast<int32_t>(window), sinks = static_cast<int32_t>(num_sinks);
  pa_status_t rc = window ? pa_window_decode_workspace(&p, win, sinks, &ws_bytes, &n_counters)
                          : pa_decode_workspace(&p, &ws_bytes, &n_counters);
  TORCH_CHECK(rc == PA_OK, "pa_decode_workspace failed: ", pa_status_string(rc));
  if (ws_bytes > static_cast<size_t>(ws_buffer.numel()) ||
      n_counters > static_cast<size_t>(ws_counters.numel())) {
    return {-1, {}, static_cast<int64_t>(ws_bytes), static_cast<int64_t>(n_counters)};
  }
  p.workspace = ws_buffer.numel() ? ws_buffer.data_ptr() : nullptr;
  p.workspace_bytes = static_cast<size_t>(ws_buffer.numel());
  p.counters = ws_counters.data_ptr<int32_t>();
  p.counter_count = static_cast<size_t>(ws_counters.numel());
  p.status = reinterpret_cast<uint32_t*>(ws_status.data_ptr<int32_t>());

  const cudaStream_t stream = c10::cuda::getCurrentCUDAStream(dev.index()).stream();
  rc = window ? pa_window_decode(&p, win, sinks, stream) : pa_decode(&p, stream);
  TORCH_CHECK(rc == PA_OK, "pa_decode failed: ", pa_status_string(rc));

  std::vector<at::Tensor> res{out};
  if (return_lse) res.push_back(lse);
  if (return_partials) {
    res.push_back(o_part);
    res.push_back(lse_part);
  }
  return {0, std::move(res), 0, 0};
}

// The full-length step: its argument list, and with it the cost of a call, is the
// shorter one.
std::tuple<int64_t, std::vector<at::Tensor>, int64_t, int64_t> decode(
    const at::Tensor& q, const at::Tensor& k, const at::Tensor& v, const at::Tensor& bt,
    const c10::optional<at::Tensor>& seq_lens, int64_t seq_len, int64_t block_size,
    int64_t num_splits, double scale, bool return_lse, bool return_partials,
    const at::Tensor& ws_buffer, const at::Tensor& ws_counters, const at::Tensor& ws_status,
    int64_t kernel_variant, const c10::optional<at::Tensor>& out_opt) {
  return window_decode(q, k, v, bt, seq_lens, seq_len, block_size, num_splits, scale, return_lse,
                       return_partials, ws_buffer, ws_counters, ws_status, kernel_variant, out_opt,
                       0, 0);
}

// Prompt attention (prompt.py): (status, [out[, lse]], bytes); status -1: the
// workspace is too small for `bytes`, and nothing was launched.
std::tuple<int64_t, std::vector<at::Tensor>, int64_t> prompt(
    const at::Tensor& q, const at::Tensor& k, const at::Tensor& v, const at::Tensor& bt,
    const at::Tensor& query_starts, const at::Tensor& seq_lens, int64_t block_size, double scale,
    bool return_lse, const at::Tensor& ws_buffer, const at::Tensor& ws_status,
    const c10::optional<at::Tensor>& out_opt, int64_t window, int64_t num_sinks,
    int64_t num_splits) {
  const auto dev = q.device();
  for (const at::Tensor* t : {&q, &k, &v, &bt, &query_starts, &seq_lens})
    check(t->is_cuda() && t->device() == dev, "all tensors must be on one CUDA device");
  check(q.dim() == 3, "Q must be [T, H, D]");
  check(k.dim() == 4 && v.sizes() == k.sizes(),
        "K_Cache and V_Cache must both be [num_blocks, block_size, Hkv, D]");
  const int dt = dtype_code(q);
  check(k.scalar_type() == q.scalar_type() && v.scalar_type() == q.scalar_type(),
        "Q, K_Cache and V_Cache must share one dtype");
  check(bt.scalar_type() == at::kInt && bt.dim() == 2,
        "Block_Table must be an int32 [B, max_blocks] tensor");
  const int64_t batch = bt.size(0), tokens = q.size(0), heads = q.size(1), dim = q.size(2);
  check(k.size(3) == dim, "head_dim of Q and the caches differ");
  check(dim == 32 || dim == 64 || dim == 128 || dim == 256,
        "head_dim must be 32, 64, 128 or 256");
  check(block_size == k.size(1) && block_size >= 1,
        "block_size differs from the cache's block dimension");
  check(k.size(2) > 0 && heads > 0 && heads % k.size(2) == 0, "Hq must be a multiple of Hkv");
  for (const at::Tensor* t : {&query_starts, &seq_lens})
    check(t->scalar_type() == at::kInt && t->dim() == 1 && t->is_contiguous(),
          "query_starts and seq_lens must be contiguous int32 tensors");
  check(query_starts.size(0) == batch + 1, "query_starts must have B + 1 entries");
  check(seq_lens.size(0) == batch, "seq_lens must have B entries");
  check(k.stride(3) == 1 && v.stride(3) == 1 && (bt.size(1) <= 1 || bt.stride(1) == 1),
        "last dimensions must be contiguous");
  check(tokens <= INT32_MAX && batch < INT32_MAX && bt.size(1) <= INT32_MAX, "sizes beyond int32");
  TORCH_CHECK(!(has_tangent(q) || has_tangent(k) || has_tangent(v)),
              "paged_prompt_attention is inference-only.");

  c10::cuda::CUDAGuard guard(dev);
  const at::Tensor Q = aligned_rows(q);
  at::Tensor out = out_opt.has_value() ? *out_opt : at::empty({tokens, heads, dim}, Q.options());
  check(out.device() == dev && out.sizes() == Q.sizes() && out.scalar_type() == Q.scalar_type() &&
            out.stride(2) == 1,
        "out must match Q's shape, dtype and device");
  check(ws_status.device() == dev, "the workspace is on another device");
  at::Tensor lse;
  if (return_lse) lse = at::empty({tokens, heads}, Q.options().dtype(at::kFloat));

  pa_prompt_params p{};
  p.q = Q.data_ptr();
  p.q_stride_t = Q.stride(0);
  p.q_stride_h = Q.stride(1);
  p.k_cache = k.data_ptr();
  p.k_stride_block = k.stride(0);
  p.k_stride_slot = k.stride(1);
  p.k_stride_head = k.stride(2);
  p.v_cache = v.data_ptr();
  p.v_stride_block = v.stride(0);
  p.v_stride_slot = v.stride(1);
  p.v_stride_head = v.stride(2);
  p.block_table = bt.data_ptr<int32_t>();
  p.bt_stride_b = bt.stride(0);
  p.max_blocks = static_cast<int32_t>(bt.size(1));
  p.query_starts = query_starts.data_ptr<int32_t>();
  p.seq_lens = seq_lens.data_ptr<int32_t>();
  p.num_tokens = static_cast<int32_t>(tokens);
  p.batch = static_cast<int32_t>(batch);
  p.num_heads = static_cast<int32_t>(heads);
  p.num_kv_heads = static_cast<int32_t>(k.size(2));
  p.head_dim = static_cast<int32_t>(dim);
  p.block_size = static_cast<int32_t>(block_size);
  p.num_blocks = static_cast<int32_t>(k.size(0));
  p.window = static_cast<int32_t>(window);
  p.num_sinks = static_cast<int32_t>(num_sinks);
  p.scale = static_cast<float>(scale > 0 ? scale : 1.0 / std::sqrt(static_cast<double>(dim)));
  p.dtype = dt;
  p.out = out.data_ptr();
  p.out_stride_t = out.stride(0);
  p.out_stride_h = out.stride(1);
  p.lse = return_lse ? lse.data_ptr<float>() : nullptr;
  p.num_splits = static_cast<int32_t>(num_splits);
  size_t bytes = 0;
  pa_status_t rc = pa_prompt_workspace(&p, &bytes);
  TORCH_CHECK(rc == PA_OK, "pa_prompt_workspace failed: ", pa_status_string(rc));
  if (bytes > static_cast<size_t>(ws_buffer.numel())) return {-1, {}, static_cast<int64_t>(bytes)};
  p.workspace = bytes ? ws_buffer.data_ptr() : nullptr;
  p.workspace_bytes = bytes;
  p.status = reinterpret_cast<uint32_t*>(ws_status.data_ptr<int32_t>());
  rc = pa_prompt(&p, c10::cuda::getCurrentCUDAStream(dev.index()).stream());
  TORCH_CHECK(rc == PA_OK, "pa_prompt failed: ", pa_status_string(rc));
  std::vector<at::Tensor> res{out};
  if (return_lse) res.push_back(lse);
  return {0, std::move(res), 0};
}

// Writes key/value rows [T, Hkv, D] into the paged caches at slot_mapping[t]
// (negative: skipped) through pa_cache_append.
void cache_append(const at::Tensor& key, const at::Tensor& value, const at::Tensor& k_cache,
                  const at::Tensor& v_cache, const at::Tensor& slot_mapping,
                  const c10::optional<at::Tensor>& status) {
  check(key.is_cuda() && value.is_cuda() && k_cache.is_cuda() && v_cache.is_cuda() &&
            slot_mapping.is_cuda(),
        "cache_append: all tensors must be CUDA tensors");
  check(key.dim() == 3 && value.sizes() == key.sizes(), "key and value must be [T, Hkv, D]");
  check(k_cache.dim() == 4 && v_cache.sizes() == k_cache.sizes(),
        "caches must be [num_blocks, block_size, Hkv, D]");
  check(key.size(1) == k_cache.size(2) && key.size(2) == k_cache.size(3),
        "key rows and cache rows differ in Hkv or D");
  const int dt = dtype_code(key);
  check(value.scalar_type() == key.scalar_type() && k_cache.scalar_type() == key.scalar_type() &&
            v_cache.scalar_type() == key.scalar_type(),
        "key, value and caches must share one dtype");
  check(slot_mapping.scalar_type() == at::kLong && slot_mapping.dim() == 1 &&
            slot_mapping.size(0) == key.size(0) && slot_mapping.is_contiguous(),
        "slot_mapping must be a contiguous int64 [T] tensor");
  check(key.stride(2) == 1 && value.stride(2) == 1 && k_cache.stride(3) == 1 &&
            v_cache.stride(3) == 1,
        "head_dim must be contiguous");
  c10::cuda::CUDAGuard guard(key.device());
  pa_append_params a{};
  a.key = key.data_ptr();
  a.key_stride_t = key.stride(0);
  a.key_stride_h = key.stride(1);
  a.value = value.data_ptr();
  a.value_stride_t = value.stride(0);
  a.value_stride_h = value.stride(1);
  a.k_cache = k_cache.data_ptr();
  a.k_stride_block = k_cache.stride(0);
  a.k_stride_slot = k_cache.stride(1);
  a.k_stride_head = k_cache.stride(2);
  a.v_cache = v_cache.data_ptr();
  a.v_stride_block = v_cache.stride(0);
  a.v_stride_slot = v_cache.stride(1);
  a.v_stride_head = v_cache.stride(2);
  a.slot_mapping = slot_mapping.data_ptr<int64_t>();
  a.num_tokens = static_cast<int32_t>(key.size(0));
  a.num_kv_heads = static_cast<int32_t>(key.size(1));
  a.head_dim = static_cast<int32_t>(key.size(2));
  a.block_size = static_cast<int32_t>(k_cache.size(1));
  a.num_blocks = static_cast<int32_t>(k_cache.size(0));
  a.dtype = dt;
  a.status = status.has_value() ? reinterpret_cast<uint32_t*>(status->data_ptr<int32_t>())
                                : nullptr;
  const pa_status_t rc =
      pa_cache_append(&a, c10::cuda::getCurrentCUDAStream(key.device().index()).stream());
  TORCH_CHECK(rc == PA_OK, "pa_cache_append failed: ", pa_status_string(rc));
}

// A pool of pages (page_pool.py): the caches, the counts and free bits, and the
// scratch of its calls.
class PagePool {
 public:
  PagePool(std::vector<at::Tensor> k, std::vector<at::Tensor> v, int64_t num_blocks,
           int64_t block_size, const at::Device& device)
      : k_(std::move(k)), v_(std::move(v)), device_(device) {
    check(k_.size() == v_.size(), "k_caches and v_caches differ in number");
    check(device.is_cuda(), "the pool's caches must be CUDA tensors");
    pool_.num_layers = static_cast<int32_t>(k_.size());
    pool_.num_kv_heads = 1;
    pool_.head_dim = 8;
    std::vector<int64_t> ptrs;
    for (size_t l = 0; l < k_.size(); ++l) {
      for (const at::Tensor* t : {&k_[l], &v_[l]}) {
        check(t->is_cuda() && t->device() == device, "caches on different devices");
        dtype_code(*t);
        check(t->scalar_type() == k_[0].scalar_type(), "caches must share one dtype");
        check(t->dim() == 4 && t->sizes() == k_[0].sizes(),
              "caches must all be [num_blocks, block_size, Hkv, D]");
        check(t->stride(3) == 1, "head_dim must be contiguous");
        check(reinterpret_cast<uintptr_t>(t->data_ptr()) % 16 == 0 && t->stride(0) % 8 == 0 &&
                  t->stride(1) % 8 == 0 && t->stride(2) % 8 == 0,
              "caches must be 16-byte aligned, with strides that are multiples of 8");
        const at::Tensor& first = (t == &k_[l]) ? k_[0] : v_[0];
        check(t->strides() == first.strides(), "the layers' caches must have the same strides");
        ptrs.push_back(reinterpret_cast<int64_t>(t->data_ptr()));
      }
    }
    if (!k_.empty()) {
      check(k_[0].size(0) == num_blocks && k_[0].size(1) == block_size,
            "num_blocks or block_size differs from the caches'");
      check(k_[0].size(3) % 8 == 0, "head_dim must be a multiple of 8");
      pool_.num_kv_heads = static_cast<int32_t>(k_[0].size(2));
      pool_.head_dim = static_cast<int32_t>(k_[0].size(3));
      pool_.k_stride_block = k_[0].stride(0);
      pool_.k_stride_slot = k_[0].stride(1);
      pool_.k_stride_head = k_[0].stride(2);
      pool_.v_stride_block = v_[0].stride(0);
      pool_.v_stride_slot = v_[0].stride(1);
      pool_.v_stride_head = v_[0].stride(2);
    }
    check(num_blocks > 0 && num_blocks <= (1 << 29) && block_size > 0 && block_size <= (1 << 20),
          "num_blocks or block_size out of range");
    pool_.num_blocks = static_cast<int32_t>(num_blocks);
    pool_.block_size = static_cast<int32_t>(block_size);
    c10::cuda::CUDAGuard guard(device);
    const auto i32 = at::TensorOptions().dtype(at::kInt).device(device);
    const int64_t words = (num_blocks + 31) / 32;
    state_ = at::zeros({num_blocks + words}, i32);
    refs_ = state_.narrow(0, 0, num_blocks);
    words_ = state_.narrow(0, num_blocks, words);
    status_ = at::zeros({1}, i32);
    ptrs_ = at::tensor(ptrs, at::TensorOptions().dtype(at::kLong)).to(device);
    pool_.caches = k_.empty() ? nullptr : reinterpret_cast<void* const*>(ptrs_.data_ptr());
    pool_.refs = refs_.data_ptr<int32_t>();
    pool_.free_words = reinterpret_cast<uint32_t*>(words_.data_ptr<int32_t>());
    pool_.status = reinterpret_cast<uint32_t*>(status_.data_ptr<int32_t>());
    ensure(1024, 1024);
    // all pages free
    done(pa_pages_adopt(&pool_, nullptr, 0, 0, 0, nullptr, stream()), "pa_pages_adopt");
  }

  // Returns the call's own status word.
  at::Tensor adopt(const at::Tensor& bt, const at::Tensor& lens) {
    table(bt);
    rows(lens, bt, "seq_lens");
    c10::cuda::CUDAGuard guard(device_);
    ensure(bt.size(0), 0);
    at::Tensor word = at::zeros({1}, state_.options());
    pa_page_pool q = pool_;
    q.status = reinterpret_cast<uint32_t*>(word.data_ptr<int32_t>());
    done(pa_pages_adopt(&q, bt.data_ptr<int32_t>(), bt.stride(0), n(bt, 0), n(bt, 1),
                        lens.data_ptr<int32_t>(), stream()),
         "pa_pages_adopt");
    return word;
  }

  void resize(const at::Tensor& bt, const at::Tensor& lens, const at::Tensor& new_lens,
              int64_t window, int64_t num_sinks) {
    table(bt);
    rows(lens, bt, "seq_lens");
    rows(new_lens, bt, "new_lens");
    c10::cuda::CUDAGuard guard(device_);
    ensure(bt.size(0), 0);
    done(pa_pages_resize(&pool_, bt.data_ptr<int32_t>(), bt.stride(0), n(bt, 0), n(bt, 1),
                         lens.data_ptr<int32_t>(), new_lens.data_ptr<int32_t>(),
                         static_cast<int32_t>(window), static_cast<int32_t>(num_sinks), stream()),
         "pa_pages_resize");
  }

  void fork(const at::Tensor& bt, const at::Tensor& lens, const at::Tensor& parents,
            const at::Tensor& children) {
    table(bt);
    rows(lens, bt, "seq_lens");
    for (const at::Tensor* t : {&parents, &children})
      check(t->device() == device_ && t->scalar_type() == at::kInt && t->dim() == 1 &&
                t->is_contiguous() && t->size(0) == parents.size(0),
            "parents and children must be contiguous int32 [n] tensors on the pool's device");
    c10::cuda::CUDAGuard guard(device_);
    ensure(bt.size(0), parents.size(0));
    done(pa_pages_fork(&pool_, bt.data_ptr<int32_t>(), bt.stride(0), n(bt, 0), n(bt, 1),
                       lens.data_ptr<int32_t>(), parents.data_ptr<int32_t>(),
                       children.data_ptr<int32_t>(), n(parents, 0), stream()),
         "pa_pages_fork");
  }

  at::Tensor compact(const at::Tensor& bt) {
    table(bt);
    c10::cuda::CUDAGuard guard(device_);
    ensure(bt.size(0), 0);
    at::Tensor live = at::empty({1}, state_.options());
    done(pa_pages_compact(&pool_, bt.data_ptr<int32_t>(), bt.stride(0), n(bt, 0), n(bt, 1),
                          live.data_ptr<int32_t>(), stream()),
         "pa_pages_compact");
    return live;
  }

  at::Tensor state_, refs_, words_, status_;

 private:
  static int32_t n(const at::Tensor& t, int d) { return static_cast<int32_t>(t.size(d)); }
  void table(const at::Tensor& bt) const {
    check(bt.device() == device_ && bt.scalar_type() == at::kInt && bt.dim() == 2 &&
              (bt.size(1) <= 1 || bt.stride(1) == 1) &&
              (bt.size(0) <= 1 || bt.stride(0) >= bt.size(1)),
          "Block_Table must be an int32 [rows, max_blocks] tensor on the pool's device, its rows "
          "apart and contiguous");
    check(bt.size(0) <= INT32_MAX && bt.size(1) <= INT32_MAX / 2, "Block_Table is too large");
  }
  void rows(const at::Tensor& t, const at::Tensor& bt, const char* name) const {
    TORCH_CHECK_VALUE(t.device() == device_ && t.scalar_type() == at::kInt && t.dim() == 1 &&
                          t.is_contiguous() && t.size(0) == bt.size(0),
                      "paged_attention: ", name,
                      " must be a contiguous int32 [rows] tensor on the pool's device");
  }
  cudaStream_t stream() const {
    return c10::cuda::getCurrentCUDAStream(device_.index()).stream();
  }
  void done(pa_status_t rc, const char* what) const {
    TORCH_CHECK(rc == PA_OK, what, " failed: ", pa_status_string(rc));
  }
  // Scratch for tables of `r` rows and forks of `p` pairs. It grows outside
  // capture only: a graph that is replayed keeps the address it was captured with.
  void ensure(int64_t r, int64_t p) {
    size_t ints = 0;
    done(pa_pages_scratch(&pool_, static_cast<int32_t>(r), static_cast<int32_t>(p), &ints),
         "pa_pages_scratch");
    if (ints <= pool_.scratch_ints) return;
    TORCH_CHECK(c10::cuda::currentStreamCaptureStatusMayInitCtx() == c10::cuda::CaptureStatus::None,
                "paged_attention: the pool's scratch has to grow for this table; make one call with "
                "it before capturing");
    scratch_.push_back(at::zeros({static_cast<int64_t>(ints)}, state_.options()));
    pool_.scratch = scratch_.back().data_ptr<int32_t>();
    pool_.scratch_ints = ints;
  }

  std::vector<at::Tensor> k_, v_;
  at::Device device_;
  at::Tensor ptrs_;
  std::vector<at::Tensor> scratch_;   // earlier ones stay: captured graphs may hold them
  pa_page_pool pool_{};
};

}  // namespace

PYBIND11_MODULE(_pa_ext, m) {
  m.def("cache_append", &cache_append, "write K/V rows into the paged caches by slot");
  m.doc() = "PyTorch binding of the sm_100a paged-attention decode C ABI";
  py::class_<PagePool>(m, "PagePool")
      .def(py::init<std::vector<at::Tensor>, std::vector<at::Tensor>, int64_t, int64_t,
                    const at::Device&>())
      .def("adopt", &PagePool::adopt)
      .def("resize", &PagePool::resize)
      .def("fork", &PagePool::fork)
      .def("compact", &PagePool::compact)
      .def_readonly("state", &PagePool::state_)
      .def_readonly("refs", &PagePool::refs_)
      .def_readonly("free_words", &PagePool::words_)
      .def_readonly("status", &PagePool::status_);
  m.def("prompt", &prompt, "prompt attention over paged caches (see prompt.py)");
  m.def("window_decode", &window_decode, "a decode step under a sliding window");
  m.def("decode", &decode, "one paged-attention decode step (see torch_kernel.py)");
}
