// Penalties, biases and grammar masks on the logits of the next token, one pass over them.
//
//   x = logits[b, v]
//   v among the row's tokens:                x = x > 0 ? x / repetition[b] : x * repetition[b]
//   c > 0 of the generated tokens are v:     x = x - frequency[b] * c - presence[b]
//   x = x + the row's biases for v
//   v not allowed:                           x = -inf
//
// in fp32.  A block owns a slice of one row's vocabulary: it counts the row's tokens that fall into
// its slice in shared memory (whole numbers, so the order of the atomics does not matter), adds the
// biases there in their order (one warp; equal ids of one step by their first lane, so that sums do
// not depend on scheduling), and then reads its logits once and writes them once.  The history is
// read by every block of a row, from L2 after the first.
#include <ATen/cuda/CUDAContext.h>
#include <c10/cuda/CUDAGuard.h>
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <torch/extension.h>

namespace {

constexpr int kThreads = 256;
constexpr int kSlice = 4096;
constexpr uint32_t kSeen = 0x80000000u;  // the token is in the row's history; the rest counts generated ones

template <typename T>
struct LogitsParams {
  const T* logits;
  int64_t ld;
  float* out;
  int rows, vocab;
  const int *tokens, *token_lens, *prompt_lens;
  int64_t tokens_ld;
  int tokens_width;
  const float *repetition, *presence, *frequency;
  const int *bias_offsets, *bias_ids;
  const float* bias_values;
  int bias_count;
  const int* allowed;
  int64_t allowed_ld;
};

__device__ __forceinline__ float to_float(float x) { return x; }
__device__ __forceinline__ float to_float(__half x) { return __half2float(x); }
__device__ __forceinline__ float to_float(__nv_bfloat16 x) { return __bfloat162float(x); }

template <typename T>
__global__ void __launch_bounds__(kThreads) process_logits_kernel(const LogitsParams<T> p) {
  __shared__ uint32_t counts[kSlice];
  __shared__ float bias[kSlice];
  const int row = blockIdx.y, v0 = blockIdx.x * kSlice, here = min(kSlice, p.vocab - v0);
  const bool with_tokens = p.tokens != nullptr;
  int b0 = 0, b1 = 0;
  if (p.bias_offsets != nullptr) {
    b0 = max(p.bias_offsets[row], 0);
    b1 = min(p.bias_offsets[row + 1], p.bias_count);
  }
  const bool with_bias = b1 > b0;
  if (with_tokens)
    for (int i = threadIdx.x; i < kSlice; i += kThreads) counts[i] = 0;
  if (with_bias)
    for (int i = threadIdx.x; i < kSlice; i += kThreads) bias[i] = 0.f;
  __syncthreads();
  if (with_tokens) {
    const int n = min(p.token_lens != nullptr ? p.token_lens[row] : p.tokens_width, p.tokens_width);
    const int prompt = p.prompt_lens != nullptr ? p.prompt_lens[row] : 0;
    const int* ids = p.tokens + row * p.tokens_ld;
    for (int i = threadIdx.x; i < n; i += kThreads) {
      const int at = ids[i] - v0;
      if (at < 0 || at >= here) continue;
      if (i >= prompt) atomicAdd(&counts[at], 1u);
      atomicOr(&counts[at], kSeen);
    }
  }
  if (with_bias && threadIdx.x < 32) {
    const int lane = threadIdx.x;
    for (int base = b0; base < b1; base += 32) {
      const int i = base + lane;
      int at = -1;
      float value = 0.f;
      if (i < b1) {
        at = p.bias_ids[i] - v0;
        if (at < 0 || at >= here) at = -1;
        else value = p.bias_values[i];
      }
      if (__any_sync(0xffffffffu, at >= 0)) {
        const uint32_t same = __match_any_sync(0xffffffffu, at);
        const bool first = (__ffs(same) - 1) == lane;
        // the sum of equal ids, lowest lane first
        float sum = first && at >= 0 ? bias[at] : 0.f;
        for (int l = 0; l < 32; ++l) {
          const float x = __shfl_sync(0xffffffffu, value, l);
          if (same >> l & 1) sum += x;
        }
        if (first && at >= 0) bias[at] = sum;
        __syncwarp();
      }
    }
  }
  __syncthreads();
  const float rep = p.repetition != nullptr ? p.repetition[row] : 1.f;
  const float freq = p.frequency != nullptr ? p.frequency[row] : 0.f;
  const float pres = p.presence != nullptr ? p.presence[row] : 0.f;
  const T* x = p.logits + row * p.ld + v0;
  float* y = p.out + (int64_t)row * p.vocab + v0;
  const uint32_t* allowed = p.allowed != nullptr ? reinterpret_cast<const uint32_t*>(p.allowed) + row * p.allowed_ld : nullptr;
  auto one = [&](float v, int i) {
    if (with_tokens) {
      const uint32_t c = counts[i];
      if (c != 0) {
        v = v > 0.f ? v / rep : v * rep;
        const uint32_t made = c & ~kSeen;
        if (made != 0) v = v - freq * (float)made - pres;
      }
    }
    if (with_bias) v += bias[i];
    if (allowed != nullptr && !(allowed[(v0 + i) >> 5] >> ((v0 + i) & 31) & 1)) v = -INFINITY;
    return v;
  };
  constexpr int N = 16 / sizeof(T);  // values of one 16-byte load
  const bool aligned = (reinterpret_cast<uintptr_t>(x) | reinterpret_cast<uintptr_t>(y)) % 16 == 0;
  int done = 0;
  if (aligned) {
    done = here / N * N;
    for (int i = threadIdx.x * N; i < done; i += kThreads * N) {
      const uint4 w = *reinterpret_cast<const uint4*>(x + i);
      const T* e = reinterpret_cast<const T*>(&w);
      float v[N];
#pragma unroll
      for (int u = 0; u < N; ++u) v[u] = one(to_float(e[u]), i + u);
#pragma unroll
      for (int u = 0; u < N; u += 4) *reinterpret_cast<float4*>(y + i + u) = make_float4(v[u], v[u + 1], v[u + 2], v[u + 3]);
    }
  }
  for (int i = done + threadIdx.x; i < here; i += kThreads) y[i] = one(to_float(x[i]), i);
}

template <typename T>
void launch(LogitsParams<T>& p, const at::Tensor& logits) {
  p.logits = reinterpret_cast<const T*>(logits.data_ptr());
  const dim3 grid((unsigned)((p.vocab + kSlice - 1) / kSlice), (unsigned)p.rows);
  process_logits_kernel<T><<<grid, kThreads, 0, at::cuda::getCurrentCUDAStream()>>>(p);
  C10_CUDA_KERNEL_LAUNCH_CHECK();
}

const at::Tensor* given(const c10::optional<at::Tensor>& t) { return t.has_value() ? &*t : nullptr; }

}  // namespace

at::Tensor process_logits(at::Tensor logits, c10::optional<at::Tensor> tokens, c10::optional<at::Tensor> token_lens,
                          c10::optional<at::Tensor> prompt_lens, c10::optional<at::Tensor> repetition,
                          c10::optional<at::Tensor> presence, c10::optional<at::Tensor> frequency,
                          c10::optional<at::Tensor> bias_offsets, c10::optional<at::Tensor> bias_ids,
                          c10::optional<at::Tensor> bias_values, c10::optional<at::Tensor> allowed,
                          c10::optional<at::Tensor> out) {
  TORCH_CHECK_VALUE(logits.is_cuda() && logits.dim() == 2 && (logits.stride(1) == 1 || logits.size(1) <= 1),
                    "logits must be [rows, vocab] on the GPU with contiguous rows");
  const auto type = logits.scalar_type();
  TORCH_CHECK_VALUE(type == at::kBFloat16 || type == at::kHalf || type == at::kFloat,
                    "logits must be bfloat16, float16 or float32");
  const at::Device dev = logits.device();
  const int64_t rows = logits.size(0), vocab = logits.size(1);
  TORCH_CHECK_VALUE(rows < 65536 && vocab < (int64_t(1) << 31) - kSlice, "too many rows or too large a vocabulary");
  auto per_row = [&](const at::Tensor* t, const char* name, at::ScalarType want, int64_t size) {
    if (t == nullptr) return;
    TORCH_CHECK_VALUE(t->device() == dev && t->scalar_type() == want && t->dim() == 1 && t->size(0) == size && t->is_contiguous(),
                      name, " must be a contiguous ", want, " tensor of ", size, " on ", dev);
  };
  per_row(given(token_lens), "token_lens", at::kInt, rows);
  per_row(given(prompt_lens), "prompt_lens", at::kInt, rows);
  per_row(given(repetition), "repetition", at::kFloat, rows);
  per_row(given(presence), "presence", at::kFloat, rows);
  per_row(given(frequency), "frequency", at::kFloat, rows);
  per_row(given(bias_offsets), "the bias offsets", at::kInt, rows + 1);
  if (tokens.has_value()) {
    TORCH_CHECK_VALUE(tokens->device() == dev && tokens->scalar_type() == at::kInt && tokens->dim() == 2 &&
                          tokens->size(0) == rows && (tokens->stride(1) == 1 || tokens->size(1) <= 1) &&
                          tokens->size(1) < (int64_t(1) << 31) - kThreads,
                      "tokens must be int32 [rows, history] on ", dev, " with contiguous rows");
  } else {
    TORCH_CHECK_VALUE(!token_lens.has_value() && !prompt_lens.has_value() && !repetition.has_value() &&
                          !presence.has_value() && !frequency.has_value(),
                      "lengths and penalties need tokens");
  }
  TORCH_CHECK_VALUE(bias_offsets.has_value() == bias_ids.has_value() && bias_ids.has_value() == bias_values.has_value(),
                    "bias is (offsets, ids, values)");
  if (bias_ids.has_value()) {
    TORCH_CHECK_VALUE(bias_ids->size(0) < (int64_t(1) << 31) - 64, "too many biases");
    per_row(given(bias_ids), "the bias ids", at::kInt, bias_ids->numel());
    per_row(given(bias_values), "the bias values", at::kFloat, bias_ids->numel());
  }
  if (allowed.has_value()) {
    TORCH_CHECK_VALUE(allowed->device() == dev && allowed->scalar_type() == at::kInt && allowed->dim() == 2 &&
                          allowed->size(0) == rows && allowed->size(1) == (vocab + 31) / 32 &&
                          (allowed->stride(1) == 1 || allowed->size(1) <= 1),
                      "allowed must be int32 [rows, ceil(vocab / 32)] on ", dev, " with contiguous rows");
  }
  c10::cuda::CUDAGuard guard(dev);
  at::Tensor y;
  if (out.has_value()) {
    TORCH_CHECK_VALUE(out->device() == dev && out->scalar_type() == at::kFloat && out->is_contiguous() &&
                          out->sizes() == logits.sizes(),
                      "out must be contiguous float32 of the logits' shape on ", dev);
    TORCH_CHECK_VALUE(out->data_ptr() != logits.data_ptr() || (type == at::kFloat && logits.is_contiguous()),
                      "out may be the logits only where they are contiguous float32");
    y = *out;
  } else {
    y = at::empty({rows, vocab}, logits.options().dtype(at::kFloat));
  }
  if (rows == 0 || vocab == 0) return y;
  auto fill = [&](auto& p) {
    p.ld = logits.stride(0);
    p.out = y.data_ptr<float>();
    p.rows = (int)rows, p.vocab = (int)vocab;
    if (tokens.has_value()) {
      p.tokens = tokens->data_ptr<int>();
      p.tokens_ld = tokens->stride(0);
      p.tokens_width = (int)tokens->size(1);
    }
    auto ints = [](const c10::optional<at::Tensor>& t) { return t.has_value() ? t->data_ptr<int>() : nullptr; };
    auto floats = [](const c10::optional<at::Tensor>& t) { return t.has_value() ? t->data_ptr<float>() : nullptr; };
    p.token_lens = ints(token_lens), p.prompt_lens = ints(prompt_lens);
    p.repetition = floats(repetition), p.presence = floats(presence), p.frequency = floats(frequency);
    p.bias_offsets = ints(bias_offsets), p.bias_ids = ints(bias_ids), p.bias_values = floats(bias_values);
    p.bias_count = bias_ids.has_value() ? (int)bias_ids->numel() : 0;
    p.allowed = ints(allowed);
    p.allowed_ld = allowed.has_value() ? allowed->stride(0) : 0;
  };
  if (type == at::kBFloat16) {
    LogitsParams<__nv_bfloat16> p{};
    fill(p);
    launch(p, logits);
  } else if (type == at::kHalf) {
    LogitsParams<__half> p{};
    fill(p);
    launch(p, logits);
  } else {
    LogitsParams<float> p{};
    fill(p);
    launch(p, logits);
  }
  return y;
}
