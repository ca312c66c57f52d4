// Torch-facing binding of the C ABI, the counterpart of UniQL's csrc/linear/quant_linear.cpp:6-25 (which binds
// w4a16o16_gemm with pybind) and csrc/embedding/quant_embedding.cpp.  The drop-in modules call these functions from
// their forward: shape checks, output allocation, scratch and the C-ABI call cost a few microseconds here instead of the
// tens of microseconds the same steps cost in Python over ctypes.  Nothing is computed in this file; every function ends
// in a call of libuniql_b200.so with raw pointers and the current stream.

#include <torch/extension.h>

#include <ATen/cuda/CUDAContext.h>
#include <ATen/cuda/EmptyTensor.h>
#include <c10/cuda/CUDAGuard.h>

#include <mutex>
#include <optional>
#include <unordered_map>
#include <vector>

#include "uniql_b200.h"

namespace {

constexpr int kMaxDevices = 64;

struct DeviceState {
  at::Tensor status;                                          // int32[1]
  std::unordered_map<uintptr_t, at::Tensor> scratch;          // per stream; counter region stays zero between launches
};

std::mutex g_mu;
DeviceState g_state[kMaxDevices];

at::Tensor status_tensor(int64_t device) {
  TORCH_CHECK(device >= 0 && device < kMaxDevices, "device index out of range");
  std::lock_guard<std::mutex> lk(g_mu);
  auto& st = g_state[device];
  if (!st.status.defined())
    st.status = at::zeros({1}, at::TensorOptions().dtype(at::kInt).device(at::Device(at::kCUDA, (c10::DeviceIndex)device)));
  return st.status;
}

// The caller holds a device guard for `device`.
at::Tensor scratch_for(int device, cudaStream_t stream, size_t need) {
  std::lock_guard<std::mutex> lk(g_mu);
  auto& slot = g_state[device].scratch[(uintptr_t)stream];
  if (!slot.defined() || (size_t)slot.numel() < need) {
    size_t size = need < ((size_t)1 << 20) ? ((size_t)1 << 20) : need;
    size = (size + ((size_t)1 << 20) - 1) >> 20 << 20;
    slot = at::zeros({(int64_t)size}, at::TensorOptions().dtype(at::kByte).device(at::Device(at::kCUDA, (c10::DeviceIndex)device)));
  }
  return slot;
}

// Scratch of a call that a graph may replay at any time, on any stream, beside eager calls and other graphs: memory of the graph's
// own while the stream is captured (its counter region cleared by a captured memset), the stream's scratch otherwise.
at::Tensor own_scratch(int device, cudaStream_t stream, size_t need) {
  cudaStreamCaptureStatus status = cudaStreamCaptureStatusNone;
  if (cudaStreamIsCapturing(stream, &status) != cudaSuccess) (void)cudaGetLastError();
  if (status == cudaStreamCaptureStatusNone) return scratch_for(device, stream, need);
  at::Tensor t = at::empty({(int64_t)need}, at::TensorOptions().dtype(at::kByte).device(at::Device(at::kCUDA, (c10::DeviceIndex)device)));
  TORCH_CHECK(cudaMemsetAsync(t.data_ptr(), 0, UNIQL_SCRATCH_COUNTER_BYTES, stream) == cudaSuccess, "clearing captured scratch failed");
  return t;
}

// Scratch requirement of the last few shapes (a decode loop repeats a handful of them).
struct NeedKey {
  int64_t v[8];
  bool operator==(const NeedKey& o) const {
    for (int i = 0; i < 8; ++i)
      if (v[i] != o.v[i]) return false;
    return true;
  }
};
template <typename F>
size_t cached_need(const NeedKey& key, F&& compute) {
  static thread_local std::vector<std::pair<NeedKey, size_t>> cache;
  for (const auto& e : cache)
    if (e.first == key) return e.second;
  const size_t need = compute();
  if (cache.size() >= 64) cache.clear();
  cache.emplace_back(key, need);
  return need;
}

void check_code(int code, const char* what) {
  if (code == UNIQL_OK) return;
  if (code == UNIQL_ECUDA)
    TORCH_CHECK(false, what, " failed: ", uniql_strerror(code), " (cudaError ", uniql_last_cuda_error(), ")");
  TORCH_CHECK(false, what, " failed: ", uniql_strerror(code));
}

void check_layer(const at::Tensor& weight, const at::Tensor& scale, const std::optional<at::Tensor>& bias,
                 int64_t n_out, int64_t* k_out, int64_t* n_store) {
  TORCH_CHECK(weight.is_cuda() && scale.is_cuda(), "weight and scale must be CUDA tensors (uniql_b200 has no CPU path)");
  TORCH_CHECK(weight.scalar_type() == at::kInt && scale.scalar_type() == at::kHalf, "weight must be int32 and scale float16");
  TORCH_CHECK(weight.dim() == 2 && scale.dim() == 2 && weight.is_contiguous() && scale.is_contiguous(),
              "weight and scale must be contiguous 2-D tensors");
  const int64_t k = weight.size(0) * 16, n = weight.size(1) / 2;
  TORCH_CHECK(scale.size(1) == n, "scale width does not match the packed weight");
  TORCH_CHECK(scale.size(0) * 128 == k, "only group size 128 is supported");
  TORCH_CHECK(n_out >= 1 && n_out <= n, "out_features exceeds the packed width");
  if (bias.has_value() && bias->defined())
    TORCH_CHECK(bias->is_cuda() && bias->scalar_type() == at::kHalf && bias->numel() >= n_out && bias->is_contiguous(),
                "bias must be a contiguous float16 CUDA tensor with at least out_features elements");
  *k_out = k;
  *n_store = n;
}

// x [..., in_features] -> fp16 [rows, k] with unit column stride, 16-byte aligned rows
at::Tensor rows_of(const at::Tensor& x, int64_t pad_in, int64_t k) {
  TORCH_CHECK(x.is_cuda() && x.scalar_type() == at::kHalf && x.dim() >= 1, "x must be a float16 CUDA tensor");
  at::Tensor x2 = x.dim() == 2 ? x : x.reshape({-1, x.size(-1)});
  if (pad_in > 0) x2 = at::constant_pad_nd(x2, {0, pad_in}, 0);
  TORCH_CHECK(x2.size(1) == k, "size_k mismatch: x has ", x2.size(1), " columns, packed weight covers ", k);
  if (x2.stride(1) != 1 || (x2.size(0) > 1 && x2.stride(0) % 8 != 0) || ((uintptr_t)x2.data_ptr()) % 16 != 0)
    x2 = x2.clone(at::MemoryFormat::Contiguous);
  return x2;
}

std::vector<int64_t> out_shape(const at::Tensor& x, int64_t n_out) {
  std::vector<int64_t> shape(x.sizes().begin(), x.sizes().end());
  shape.back() = n_out;
  return shape;
}

// W4A16B16O16Linear.forward (quantize/quant_linear_layers.py:91-116): y = x W^T (+ bias), padded input columns added
// here, padded output columns and the bias handled by the kernel epilogue; `hadamard` applies the online transform of
// size k to the rows first (the Hadamard module in front of down_proj / out_proj).
at::Tensor linear(const at::Tensor& x, const at::Tensor& weight, const at::Tensor& scale,
                  const std::optional<at::Tensor>& bias, int64_t n_out, int64_t pad_in, bool hadamard) {
  int64_t k = 0, n = 0;
  check_layer(weight, scale, bias, n_out, &k, &n);
  const at::Tensor x2 = rows_of(x, pad_in, k);
  const int64_t m = x2.size(0);
  const c10::cuda::CUDAGuard guard(x2.device());
  const int dev = x2.device().index();
  at::Tensor out = at::empty(out_shape(x, n_out), x2.options());
  if (m == 0) return out;
  cudaStream_t stream = at::cuda::getCurrentCUDAStream(dev).stream();
  const int64_t had = hadamard ? k : 0;
  const size_t need = cached_need(NeedKey{{0, m, n, k, had, 0, 0, 0}}, [&] { return uniql_w4a16_scratch_bytes(m, n, k, had); });
  at::Tensor scratch = scratch_for(dev, stream, need);
  at::Tensor status = status_tensor(dev);
  const void* bias_ptr = (bias.has_value() && bias->defined()) ? bias->data_ptr() : nullptr;
  const int code = uniql_w4a16_linear(x2.data_ptr(), m > 1 ? x2.stride(0) : k, weight.data_ptr(), scale.data_ptr(), bias_ptr,
                                      out.data_ptr(), n_out, m, n, n_out, k, 128, had, scratch.data_ptr(),
                                      (size_t)scratch.numel(), (int*)status.data_ptr(), stream);
  check_code(code, "uniql_w4a16_linear");
  return out;
}

// One decode launch for projections that read the same activations (uniql_w4a16_linear_group): q/k/v, gate+up with
// act_fn(gate) * up (modeling/llama/llama_qblocks.py:48-51, :104-106), or one projection with the block's residual.
// Returns one tensor per projection (one tensor for the SwiGLU epilogue).  Up to 16 rows; 17..128 rows for plain
// outputs (one launch of the operand-swapped tensor-core kernel over all projections).
std::vector<at::Tensor> linear_group(const at::Tensor& x, const std::vector<at::Tensor>& weights,
                                     const std::vector<at::Tensor>& scales,
                                     const std::vector<std::optional<at::Tensor>>& biases,
                                     const std::vector<int64_t>& n_outs, int64_t epilogue,
                                     const std::optional<at::Tensor>& residual, int64_t pad_in, bool hadamard) {
  const int np = (int)weights.size();
  TORCH_CHECK(np >= 1 && np <= UNIQL_MAX_PROJ, "one launch takes 1 to ", UNIQL_MAX_PROJ, " projections");
  TORCH_CHECK((int)scales.size() == np && (int)biases.size() == np && (int)n_outs.size() == np,
              "weights, scales, biases and out_features must have one entry per projection");
  TORCH_CHECK(epilogue == UNIQL_EPILOGUE_NONE || epilogue == UNIQL_EPILOGUE_SWIGLU, "unknown epilogue");
  int64_t k = 0, ns[UNIQL_MAX_PROJ];
  for (int i = 0; i < np; ++i) {
    int64_t ki = 0;
    check_layer(weights[i], scales[i], biases[i], n_outs[i], &ki, &ns[i]);
    TORCH_CHECK(i == 0 || ki == k, "projections of one launch must share in_features");
    k = ki;
  }
  const at::Tensor x2 = rows_of(x, pad_in, k);
  const int64_t m = x2.size(0);
  TORCH_CHECK(m >= 1 && m <= 128, "grouped launches take 1 to 128 rows");
  TORCH_CHECK(m <= 16 || (epilogue == UNIQL_EPILOGUE_NONE && !hadamard && !(residual.has_value() && residual->defined())),
              "above 16 rows a grouped launch has plain outputs only");
  const c10::cuda::CUDAGuard guard(x2.device());
  const int dev = x2.device().index();
  const int nout = epilogue == UNIQL_EPILOGUE_SWIGLU ? 1 : np;
  std::vector<at::Tensor> outs;
  outs.reserve(nout);
  for (int i = 0; i < nout; ++i) outs.push_back(at::empty(out_shape(x, n_outs[i]), x2.options()));
  uniql_w4a16_proj proj[UNIQL_MAX_PROJ];
  for (int i = 0; i < np; ++i) {
    const at::Tensor& d = outs[i < nout ? i : nout - 1];
    proj[i].B = weights[i].data_ptr();
    proj[i].s = scales[i].data_ptr();
    proj[i].bias = (biases[i].has_value() && biases[i]->defined()) ? biases[i]->data_ptr() : nullptr;
    proj[i].D = d.data_ptr();
    proj[i].ldd = n_outs[i < nout ? i : nout - 1];
    proj[i].n = ns[i];
    proj[i].n_out = n_outs[i];
  }
  const void* res_ptr = nullptr;
  int64_t ldr = 0;
  at::Tensor res2;
  if (residual.has_value() && residual->defined()) {
    TORCH_CHECK(residual->is_cuda() && residual->scalar_type() == at::kHalf, "residual must be a float16 CUDA tensor");
    res2 = residual->dim() == 2 ? *residual : residual->reshape({-1, residual->size(-1)});
    if (res2.stride(1) != 1) res2 = res2.contiguous();
    TORCH_CHECK(res2.size(0) == m && res2.size(1) == n_outs[0], "residual must have the shape of the output");
    res_ptr = res2.data_ptr();
    ldr = res2.stride(0);
  }
  cudaStream_t stream = at::cuda::getCurrentCUDAStream(dev).stream();
  const int64_t had = hadamard ? k : 0;
  const size_t need = cached_need(
      NeedKey{{1 + epilogue + 2 * (had != 0), m, k, ns[0], np > 1 ? ns[1] : 0, np > 2 ? ns[2] : 0, np > 3 ? ns[3] : 0, np}},
      [&] { return uniql_w4a16_group_scratch_bytes(m, k, ns, np, (int)epilogue, had); });
  at::Tensor scratch = scratch_for(dev, stream, need);
  at::Tensor status = status_tensor(dev);
  const int code = uniql_w4a16_linear_group(x2.data_ptr(), m > 1 ? x2.stride(0) : k, m, k, proj, np, (int)epilogue, res_ptr,
                                            ldr, had, nullptr, 0, scratch.data_ptr(), (size_t)scratch.numel(),
                                            (int*)status.data_ptr(), stream);
  check_code(code, "uniql_w4a16_linear_group");
  return outs;
}

// W4O16Embedding.forward (quantize/quant_embedding_layers.py:49-51).
at::Tensor embedding(const at::Tensor& ids, const at::Tensor& weight, const at::Tensor& scales) {
  TORCH_CHECK(ids.is_cuda() && weight.is_cuda() && scales.is_cuda(), "input, weight and scale must be CUDA tensors");
  TORCH_CHECK(weight.dim() == 2 && weight.scalar_type() == at::kInt, "weight must be a 2-D int32 tensor");
  TORCH_CHECK(scales.dim() == 1 && scales.scalar_type() == at::kHalf && scales.numel() == weight.size(0),
              "scale must be a 1-D float16 tensor with one entry per table row");
  TORCH_CHECK((ids.dim() == 1 || ids.dim() == 2) && ids.scalar_type() == at::kLong, "input must be a 1-D or 2-D int64 tensor");
  const at::Tensor ids_c = ids.contiguous(), w = weight.contiguous(), s = scales.contiguous();
  const int64_t vocab = w.size(0), dim = w.size(1) * 8;
  std::vector<int64_t> shape(ids.sizes().begin(), ids.sizes().end());
  shape.push_back(dim);
  const c10::cuda::CUDAGuard guard(ids.device());
  const int dev = ids.device().index();
  at::Tensor out = at::empty(shape, at::TensorOptions().dtype(at::kHalf).device(ids.device()));
  at::Tensor status = status_tensor(dev);
  const int code = uniql_w4_embedding((const int64_t*)ids_c.data_ptr(), ids_c.numel(), w.data_ptr(), s.data_ptr(), out.data_ptr(), vocab, dim,
                                      (int*)status.data_ptr(), at::cuda::getCurrentCUDAStream(dev).stream());
  check_code(code, "uniql_w4_embedding");
  return out;
}

// act_fn(gate) * up between the launches of an MLP at more than 16 rows (uniql_silu_mul): one pass, PyTorch's roundings.
at::Tensor silu_mul(const at::Tensor& gate, const at::Tensor& up) {
  TORCH_CHECK(gate.is_cuda() && up.is_cuda() && gate.scalar_type() == at::kHalf && up.scalar_type() == at::kHalf,
              "gate and up must be float16 CUDA tensors");
  TORCH_CHECK(gate.sizes() == up.sizes() && gate.dim() >= 1, "gate and up must have the same shape");
  const int64_t cols = gate.size(-1);
  at::Tensor g2 = gate.reshape({-1, cols}), u2 = up.reshape({-1, cols});
  if (g2.stride(1) != 1 || g2.stride(0) % 8 || ((uintptr_t)g2.data_ptr()) % 16) g2 = g2.contiguous();
  if (u2.stride(1) != 1 || u2.stride(0) % 8 || ((uintptr_t)u2.data_ptr()) % 16) u2 = u2.contiguous();
  const c10::cuda::CUDAGuard guard(gate.device());
  at::Tensor out = at::empty(gate.sizes(), gate.options());
  const int code = uniql_silu_mul(g2.data_ptr(), g2.stride(0), u2.data_ptr(), u2.stride(0), out.data_ptr(), cols, g2.size(0),
                                  cols, at::cuda::getCurrentCUDAStream(gate.device().index()).stream());
  check_code(code, "uniql_silu_mul");
  return out;
}

// Hadamard.forward / had_transform (quantize/hadamard_helpers.py:18-48): y = H x * scale along the last axis.
at::Tensor hadamard(const at::Tensor& x, double scale) {
  TORCH_CHECK(x.is_cuda(), "x must be a CUDA tensor (uniql_b200 has no CPU path)");
  int dtype = 0;
  if (x.scalar_type() == at::kHalf) dtype = UNIQL_F16;
  else if (x.scalar_type() == at::kBFloat16) dtype = UNIQL_BF16;
  else if (x.scalar_type() == at::kFloat) dtype = UNIQL_F32;
  else TORCH_CHECK(false, "unsupported dtype");
  const at::Tensor xc = x.contiguous();
  const int64_t dim = xc.dim() ? xc.size(-1) : 0;
  const int64_t rows = dim ? xc.numel() / dim : 0;
  const c10::cuda::CUDAGuard guard(x.device());
  at::Tensor y = at::empty_like(xc);
  const int code = uniql_hadamard(xc.data_ptr(), y.data_ptr(), rows, dim, (float)scale, dtype,
                                  at::cuda::getCurrentCUDAStream(x.device().index()).stream());
  check_code(code, "uniql_hadamard");
  return y;
}

// ---- attention around the paged 4-bit KV cache (include/uniql_b200.h): types, devices and shapes are checked here, sizes and
// alignment by the C ABI.
int kv_dtype(const at::Tensor& t, const char* name) {
  if (t.scalar_type() == at::kHalf) return UNIQL_F16;
  TORCH_CHECK(t.scalar_type() == at::kBFloat16, name, " must be float16 or bfloat16");
  return UNIQL_BF16;
}

void check_ints(const at::Tensor& t, const at::Tensor& like, int64_t dim, const char* name) {
  TORCH_CHECK(t.is_cuda() && t.scalar_type() == at::kInt && t.dim() == dim, name, " must be a ", dim, "-D int32 CUDA tensor");
  TORCH_CHECK(t.device() == like.device(), name, " is on another device");
  TORCH_CHECK(t.size(-1) <= 1 || t.stride(-1) == 1, name, " must have unit stride in its last dimension");
}

// rows [tokens, heads, channels] that a kernel reads with 16-byte loads: unit channel stride, the other strides multiples of 8
at::Tensor head_rows(const at::Tensor& x) {
  const bool ok = x.stride(2) == 1 && (x.size(0) <= 1 || (x.stride(0) > 0 && x.stride(0) % 8 == 0)) &&
                  (x.size(1) <= 1 || (x.stride(1) > 0 && x.stride(1) % 8 == 0)) && ((uintptr_t)x.data_ptr()) % 16 == 0;
  return ok ? x : x.clone(at::MemoryFormat::Contiguous);
}
int64_t stride_of(const at::Tensor& x, int64_t dim) {          // of a dimension with one entry: anything valid
  return x.size(dim) > 1 ? x.stride(dim) : (dim == 0 ? x.size(1) * x.size(2) : x.size(2));
}

// A new tensor, straight from the allocator: half of what at::empty costs through the dispatcher.
at::Tensor new_tensor(at::IntArrayRef sizes, at::ScalarType type, at::Device device) {
  return at::Tensor(at::detail::empty_cuda(sizes, type, device, std::nullopt));
}

struct CacheView {
  int64_t pages, heads, page, dp;
};
CacheView check_cache(const at::Tensor& codes, const at::Tensor& scales) {
  TORCH_CHECK(codes.is_cuda() && scales.is_cuda(), "codes and scales must be CUDA tensors (uniql_b200 has no CPU path)");
  TORCH_CHECK(codes.scalar_type() == at::kInt && scales.scalar_type() == at::kHalf, "codes must be int32 and scales float16");
  TORCH_CHECK(codes.dim() == 5 && codes.size(1) == 2 && codes.is_contiguous(),
              "codes must be a contiguous [pages, 2, kv_heads, page_size, words] tensor");
  TORCH_CHECK(scales.dim() == 5 && scales.is_contiguous() && scales.size(0) == codes.size(0) && scales.size(1) == 2 &&
                  scales.size(2) == codes.size(2) && scales.size(3) == codes.size(3) && scales.size(4) == 2,
              "scales must be a contiguous [pages, 2, kv_heads, page_size, 2] tensor of the same cache");
  TORCH_CHECK(scales.device() == codes.device(), "codes and scales must be on one device");
  return {codes.size(0), codes.size(2), codes.size(3), codes.size(4) * 8};
}

// A 1-D tensor over part of a byte buffer: several results of one call share an allocation, which costs a microsecond.
at::Tensor part_of(const at::Tensor& bytes, int64_t offset, int64_t n, at::ScalarType type) {
  auto dtype = c10::scalarTypeToTypeMeta(type);
  at::Tensor t = at::detail::make_tensor<c10::TensorImpl>(c10::Storage(bytes.storage()), bytes.key_set(), dtype);
  auto* impl = t.unsafeGetTensorImpl();
  impl->set_storage_offset(offset / (int64_t)dtype.itemsize());
  impl->set_sizes_contiguous({n});
  return t;
}

std::vector<at::Tensor> kv_page_plan(const at::Tensor& lens, const at::Tensor& new_lens, const at::Tensor& block_table,
                                     const at::Tensor& free_pages, const at::Tensor& free_count, int64_t page_size,
                                     int64_t total_new, bool in_place, bool whole) {
  check_ints(lens, lens, 1, "lens");
  check_ints(new_lens, lens, 1, "new_lens");
  check_ints(block_table, lens, 2, "block_table");
  check_ints(free_pages, lens, 1, "free_pages");
  check_ints(free_count, lens, 1, "free_count");
  const int64_t batch = lens.size(0), width = block_table.size(1);
  TORCH_CHECK(new_lens.size(0) == batch && block_table.size(0) == batch, "lens, new_lens and block_table must have one row per request");
  TORCH_CHECK(free_count.size(0) == 1, "free_count must have one entry");
  TORCH_CHECK(batch <= 1 || block_table.stride(0) >= width, "rows of block_table must not overlap");
  TORCH_CHECK(total_new >= 0, "total_new must not be negative");
  const c10::cuda::CUDAGuard guard(lens.device());
  const int dev = lens.device().index();
  const int64_t longs = 16 * total_new, ints = 4 * (batch + 1);
  at::Tensor buf = new_tensor({longs + (whole ? 4 : 2) * ints + 4}, at::kByte, lens.device());
  at::Tensor slots = part_of(buf, 0, total_new, at::kLong), positions = part_of(buf, 8 * total_new, total_new, at::kLong);
  at::Tensor cu = part_of(buf, longs, batch + 1, at::kInt);
  at::Tensor lens_out = in_place ? lens : part_of(buf, longs + ints, batch, at::kInt);
  at::Tensor count_out = in_place ? free_count : part_of(buf, longs + 2 * ints, 1, at::kInt);
  at::Tensor status = status_tensor(dev);
  auto plan = [&](auto fn, auto... keys) {
    return fn((const int32_t*)lens.data_ptr(), (const int32_t*)new_lens.data_ptr(), batch, (int32_t*)block_table.data_ptr(),
              batch > 1 ? block_table.stride(0) : width, width, (const int32_t*)free_pages.data_ptr(), free_pages.size(0),
              (const int32_t*)free_count.data_ptr(), page_size, total_new, (int64_t*)slots.data_ptr(),
              (int64_t*)positions.data_ptr(), (int32_t*)cu.data_ptr(), (int32_t*)lens_out.data_ptr(),
              (int32_t*)count_out.data_ptr(), keys..., (int*)status.data_ptr(), at::cuda::getCurrentCUDAStream(dev).stream());
  };
  if (!whole) {
    check_code(plan(uniql_kv_page_plan), "uniql_kv_page_plan");
    return {slots, positions, cu, lens_out, count_out};
  }
  at::Tensor key_lens = part_of(buf, longs + 2 * ints + 4, batch, at::kInt), cu_keys = part_of(buf, longs + 3 * ints + 4, batch + 1, at::kInt);
  check_code(plan(uniql_kv_step_plan, (int32_t*)key_lens.data_ptr(), (int32_t*)cu_keys.data_ptr()), "uniql_kv_step_plan");
  return {slots, positions, cu, lens_out, count_out, key_lens, cu_keys};
}

void kv4_append(const at::Tensor& k, const at::Tensor& v, const at::Tensor& slots, const at::Tensor& codes, const at::Tensor& scales) {
  const CacheView cv = check_cache(codes, scales);
  TORCH_CHECK(k.is_cuda() && v.is_cuda() && k.dim() == 3 && v.dim() == 3, "k and v must be [tokens, kv_heads, channels] CUDA tensors");
  const int dtype = kv_dtype(k, "k");
  TORCH_CHECK(v.scalar_type() == k.scalar_type(), "k and v must have the same type");
  TORCH_CHECK(k.size(0) == v.size(0) && k.size(1) == cv.heads && v.size(1) == cv.heads, "k and v must have one row per token and kv head of the cache");
  TORCH_CHECK(slots.is_cuda() && slots.scalar_type() == at::kLong && slots.dim() == 1 && slots.size(0) == k.size(0),
              "slots must be an int64 CUDA tensor with one entry per token");
  TORCH_CHECK(k.device() == codes.device() && v.device() == codes.device() && slots.device() == codes.device(),
              "k, v, slots and the cache must be on one device");
  const c10::cuda::CUDAGuard guard(codes.device());
  const int dev = codes.device().index();
  const at::Tensor k3 = head_rows(k), v3 = head_rows(v), sl = slots.contiguous();
  at::Tensor status = status_tensor(dev);
  const int code = uniql_kv4_append(k3.data_ptr(), stride_of(k3, 0), stride_of(k3, 1), v3.data_ptr(), stride_of(v3, 0),
                                    stride_of(v3, 1), dtype, k3.size(0), cv.heads, k3.size(2), v3.size(2),
                                    (const int64_t*)sl.data_ptr(), codes.data_ptr(), scales.data_ptr(), cv.pages, cv.page, cv.dp,
                                    (int*)status.data_ptr(), at::cuda::getCurrentCUDAStream(dev).stream());
  check_code(code, "uniql_kv4_append");
}

std::vector<at::Tensor> kv4_gather(const at::Tensor& codes, const at::Tensor& scales, const at::Tensor& block_table,
                                   const at::Tensor& cu, int64_t total, int64_t dk, int64_t dv, bool bf16,
                                   const std::optional<at::Tensor>& starts) {
  const CacheView cv = check_cache(codes, scales);
  check_ints(block_table, codes, 2, "block_table");
  check_ints(cu, codes, 1, "cu");
  const int64_t batch = block_table.size(0), width = block_table.size(1);
  TORCH_CHECK(cu.size(0) == batch + 1, "cu must have one entry more than block_table has rows");
  TORCH_CHECK(batch <= 1 || block_table.stride(0) >= width, "rows of block_table must not overlap");
  const bool has_starts = starts.has_value() && starts->defined();
  if (has_starts) {
    check_ints(*starts, codes, 1, "starts");
    TORCH_CHECK(starts->size(0) == batch, "starts must have one entry per request");
  }
  TORCH_CHECK(total >= 0 && dk > 0 && dv > 0, "total, head_dim_k and head_dim_v must not be negative");
  const c10::cuda::CUDAGuard guard(codes.device());
  const int dev = codes.device().index();
  const auto type = bf16 ? at::kBFloat16 : at::kHalf;
  at::Tensor k = new_tensor({total, cv.heads, dk}, type, codes.device()), v = new_tensor({total, cv.heads, dv}, type, codes.device());
  at::Tensor status = status_tensor(dev);
  const int code = uniql_kv4_gather(codes.data_ptr(), scales.data_ptr(), cv.pages, cv.page, cv.dp, cv.heads,
                                    (const int32_t*)block_table.data_ptr(), batch > 1 ? block_table.stride(0) : width, width, batch,
                                    has_starts ? (const int32_t*)starts->data_ptr() : nullptr, (const int32_t*)cu.data_ptr(), total,
                                    dk, dv, bf16 ? UNIQL_BF16 : UNIQL_F16, k.data_ptr(), v.data_ptr(), (int*)status.data_ptr(),
                                    at::cuda::getCurrentCUDAStream(dev).stream());
  check_code(code, "uniql_kv4_gather");
  return {k, v};
}

at::Tensor kv4_attention(const at::Tensor& q, const at::Tensor& codes, const at::Tensor& scales, const at::Tensor& block_table,
                         const at::Tensor& lens, int64_t dv, double softmax_scale) {
  const CacheView cv = check_cache(codes, scales);
  TORCH_CHECK(q.is_cuda() && q.dim() == 3, "q must be a [batch, heads, channels] CUDA tensor");
  const int dtype = kv_dtype(q, "q");
  check_ints(block_table, codes, 2, "block_table");
  check_ints(lens, codes, 1, "lens");
  const int64_t batch = q.size(0), width = block_table.size(1);
  TORCH_CHECK(block_table.size(0) == batch && lens.size(0) == batch, "q, block_table and lens must have one row per request");
  TORCH_CHECK(batch <= 1 || block_table.stride(0) >= width, "rows of block_table must not overlap");
  TORCH_CHECK(q.device() == codes.device(), "q and the cache must be on one device");
  TORCH_CHECK(dv > 0 && q.size(1) > 0 && q.size(2) > 0, "q and head_dim_v must not be empty");
  TORCH_CHECK(cv.heads > 0 && q.size(1) % cv.heads == 0, "the query heads must be a multiple of the cache's kv heads");
  const c10::cuda::CUDAGuard guard(q.device());
  const int dev = q.device().index();
  const at::Tensor q3 = q.stride(2) == 1 || q.size(2) == 1 ? q : q.contiguous();
  at::Tensor out = new_tensor({batch, q.size(1), dv}, q.scalar_type(), q.device());
  if (batch == 0) return out;
  cudaStream_t stream = at::cuda::getCurrentCUDAStream(dev).stream();
  const size_t need = uniql_kv4_attention_scratch_bytes(batch, q.size(1), cv.heads, cv.dp);
  at::Tensor scratch = own_scratch(dev, stream, need);
  at::Tensor status = status_tensor(dev);
  const int code = uniql_kv4_attention(q3.data_ptr(), q3.stride(0), q3.stride(1), codes.data_ptr(), scales.data_ptr(), cv.pages,
                                       cv.page, cv.dp, (const int32_t*)block_table.data_ptr(),
                                       batch > 1 ? block_table.stride(0) : width, width, (const int32_t*)lens.data_ptr(), batch,
                                       q.size(1), cv.heads, q.size(2), dv, (float)softmax_scale, dtype, out.data_ptr(),
                                       scratch.data_ptr(), (size_t)scratch.numel(), (int*)status.data_ptr(), stream);
  check_code(code, "uniql_kv4_attention");
  return out;
}

at::Tensor prompt_attention(const at::Tensor& q, const at::Tensor& k, const at::Tensor& v, const at::Tensor& cu_q,
                            const std::optional<at::Tensor>& cu_k, bool causal, double softmax_scale) {
  TORCH_CHECK(q.is_cuda() && k.is_cuda() && v.is_cuda() && q.dim() == 3 && k.dim() == 3 && v.dim() == 3,
              "q, k and v must be [tokens, heads, channels] CUDA tensors");
  const int dtype = kv_dtype(q, "q");
  TORCH_CHECK(k.scalar_type() == q.scalar_type() && v.scalar_type() == q.scalar_type(), "q, k and v must have the same type");
  TORCH_CHECK(k.device() == q.device() && v.device() == q.device(), "q, k and v must be on one device");
  TORCH_CHECK(k.size(0) == v.size(0) && k.size(1) == v.size(1) && k.size(2) == q.size(2), "k and v must have the same tokens and heads, q and k the same channels");
  TORCH_CHECK(k.size(1) > 0 && q.size(1) > 0 && q.size(1) % k.size(1) == 0, "the query heads must be a multiple of the kv heads");
  TORCH_CHECK(q.size(2) > 0 && v.size(2) > 0, "q, k and v must have channels");
  check_ints(cu_q, q, 1, "cu_q");
  const at::Tensor ck = cu_k.has_value() && cu_k->defined() ? *cu_k : cu_q;
  check_ints(ck, q, 1, "cu_k");
  TORCH_CHECK(cu_q.size(0) >= 1 && ck.size(0) == cu_q.size(0), "cu_q and cu_k must have one entry more than there are requests");
  const c10::cuda::CUDAGuard guard(q.device());
  const int dev = q.device().index();
  const at::Tensor q3 = head_rows(q), k3 = head_rows(k), v3 = head_rows(v);
  at::Tensor out = new_tensor({q.size(0), q.size(1), v.size(2)}, q.scalar_type(), q.device());
  at::Tensor status = status_tensor(dev);
  const int code = uniql_prompt_attention(q3.data_ptr(), stride_of(q3, 0), stride_of(q3, 1), k3.data_ptr(), stride_of(k3, 0),
                                          stride_of(k3, 1), v3.data_ptr(), stride_of(v3, 0), stride_of(v3, 1),
                                          (const int32_t*)cu_q.data_ptr(), (const int32_t*)ck.data_ptr(), cu_q.size(0) - 1,
                                          q.size(0), k.size(0), q.size(1), k.size(1), q.size(2), v.size(2), (float)softmax_scale,
                                          causal ? 1 : 0, dtype, out.data_ptr(), (int*)status.data_ptr(),
                                          at::cuda::getCurrentCUDAStream(dev).stream());
  check_code(code, "uniql_prompt_attention");
  return out;
}

}  // namespace

PYBIND11_MODULE(TORCH_EXTENSION_NAME, m) {
  m.doc() = "uniql_b200: torch binding of the C ABI (libuniql_b200.so)";
  m.def("abi_version", []() { return uniql_abi_version(); });
  m.def("status_tensor", &status_tensor, "int32[1] diagnostics word of a device");
  m.def("linear", &linear, "W4A16 linear forward");
  m.def("linear_group", &linear_group, "grouped W4A16 decode launch");
  m.def("embedding", &embedding, "4-bit embedding gather");
  m.def("hadamard", &hadamard, "Hadamard transform along the last axis");
  m.def("silu_mul", &silu_mul, "silu(gate) * up in one pass");
  m.def("kv_page_plan", &kv_page_plan, "block tables, slots and positions of a step's new tokens");
  m.def("kv4_append", &kv4_append, "quantise K/V rows into a paged 4-bit cache");
  m.def("kv4_gather", &kv4_gather, "rows of a token range of a paged 4-bit cache");
  m.def("kv4_attention", &kv4_attention, "one query token per request over a paged 4-bit cache");
  m.def("prompt_attention", &prompt_attention, "causal attention of packed prompts");
}
