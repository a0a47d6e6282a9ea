// The serving operators' entry points: checks of the tensors, workspaces, launches on the current stream.
// Device code and layouts: serving.h.
#include <ATen/cuda/CUDAContext.h>
#include <c10/cuda/CUDAGraphsC10Utils.h>
#include <c10/cuda/CUDAGuard.h>
#include <torch/extension.h>

#include <algorithm>
#include <map>
#include <mutex>
#include <tuple>

#include "serving.h"
#include "tma.cuh"

using namespace mimir;

namespace {

#define SERVING_CHECK(cond, ...) TORCH_CHECK_VALUE(cond, __VA_ARGS__)

int* status_word(const at::Device& dev) {
  static int* words[64] = {nullptr};
  const int i = dev.index();
  if (words[i] == nullptr) {
    c10::cuda::CUDAGuard guard(dev);
    void* ptr = nullptr;
    C10_CUDA_CHECK(cache_status_address(&ptr));
    words[i] = static_cast<int*>(ptr);
  }
  return words[i];
}

void check_int32(const at::Tensor& t, const char* name, int64_t dim, const at::Device& dev) {
  SERVING_CHECK(t.device() == dev && t.scalar_type() == at::kInt && t.dim() == dim && t.is_contiguous(), name,
                " must be a contiguous int32 tensor of ", dim, " dimension(s) on ", dev);
}

void check_page_size(int64_t page) {
  SERVING_CHECK(page >= 16 && page <= 256 && (page & (page - 1)) == 0, "page_size must be 16, 32, 64, 128 or 256, not ",
                page);
}

// `lead`: dimensions before the page's (0, or 1 for a layer dimension).
void check_pool(const at::Tensor& pages, const at::Tensor& scales, int64_t lead) {
  SERVING_CHECK(pages.is_cuda() && pages.scalar_type() == at::kFloat8_e4m3fn && pages.is_contiguous() &&
                    pages.dim() == 5 + lead,
                "pages must be a contiguous float8_e4m3fn CUDA tensor of ", 5 + lead, " dimensions");
  SERVING_CHECK(pages.size(lead + 1) == 2 && pages.size(lead + 4) == kCacheDim && pages.size(lead + 2) >= 1,
                "pages must be [pages, 2, kv_heads, page_size, 128]");
  check_page_size(pages.size(lead + 3));
  SERVING_CHECK(reinterpret_cast<uintptr_t>(pages.data_ptr()) % 16 == 0, "pages must start on a 16-byte boundary");
  bool fits = scales.device() == pages.device() && scales.scalar_type() == at::kFloat && scales.is_contiguous() &&
              scales.dim() == 4 + lead && scales.size(lead + 3) == pages.size(lead + 3) / kCacheBlock;
  for (int64_t i = 0; fits && i < lead + 3; ++i) fits = scales.size(i) == pages.size(i);
  SERVING_CHECK(fits, "scales must be a contiguous float32 tensor [pages, 2, kv_heads, page_size / 16] beside the pages");
  SERVING_CHECK(pages.size(lead) * 2 * pages.size(lead + 2) < (int64_t(1) << 31), "the pool has too many pages");
}

void check_batch(const at::Tensor& table, const at::Tensor& lens, const at::Tensor& seqs, const at::Tensor& cu_new,
                 const at::Device& dev) {
  check_int32(table, "page_table", 2, dev);
  check_int32(lens, "seq_lens", 1, dev);
  check_int32(seqs, "seqs", 1, dev);
  check_int32(cu_new, "cu_new", 1, dev);
  SERVING_CHECK(lens.size(0) == table.size(0), "seq_lens needs one length for each row of page_table");
  SERVING_CHECK(cu_new.size(0) == seqs.size(0) + 1, "cu_new needs one more entry than seqs");
}

// Rows [T, heads, 128] of 16-bit values whose last dimension is contiguous and 16-byte aligned.
void check_rows(const at::Tensor& x, const char* name, const at::Device& dev) {
  SERVING_CHECK(x.device() == dev && x.dim() == 3 && x.size(2) == kCacheDim && x.stride(2) == 1, name,
                " must be [tokens, heads, 128] on ", dev, " with contiguous heads");
  SERVING_CHECK(x.scalar_type() == at::kBFloat16 || x.scalar_type() == at::kHalf, name, " must be bfloat16 or float16");
  SERVING_CHECK(reinterpret_cast<uintptr_t>(x.data_ptr()) % 16 == 0 && x.stride(0) % 8 == 0 && x.stride(1) % 8 == 0, name,
                " must start on a 16-byte boundary in every head");
}

Book book_of(const at::Tensor& table, const at::Tensor& lens, const at::Tensor& refs, int64_t page) {
  SERVING_CHECK(table.is_cuda(), "page_table must be a CUDA tensor");
  check_int32(table, "page_table", 2, table.device());
  check_int32(lens, "seq_lens", 1, table.device());
  check_int32(refs, "ref_counts", 1, table.device());
  SERVING_CHECK(lens.size(0) == table.size(0), "seq_lens needs one length for each row of page_table");
  SERVING_CHECK(refs.size(0) < (int64_t(1) << 30), "the pool has too many pages");
  check_page_size(page);
  return Book{table.data_ptr<int>(), lens.data_ptr<int>(), refs.data_ptr<int>(), (int)table.size(0), (int)table.size(1),
              (int)refs.size(0), (int)page, status_word(table.device())};
}

CopyParams copy_of(const at::Tensor& pages, const at::Tensor& scales, const at::Tensor& out_pages,
                   const at::Tensor& out_scales) {
  CopyParams p{};
  p.pages = static_cast<const uint8_t*>(pages.data_ptr());
  p.out_pages = static_cast<uint8_t*>(out_pages.data_ptr());
  p.scales = scales.data_ptr<float>();
  p.out_scales = out_scales.data_ptr<float>();
  p.npages = pages.size(1);
  p.out_npages = out_pages.size(1);
  p.page_bytes = pages.size(2) * pages.size(3) * pages.size(4) * pages.size(5);
  p.scale_floats = (int)(p.page_bytes / kCacheDim / kCacheBlock);
  p.layers = (int)pages.size(0);
  p.status = status_word(pages.device());
  return p;
}

// Keys and values as rows of 128 bytes: [pages * 2 * kv_heads][page_size][128], boxes of `keys` rows.
CUtensorMap pages_map(const at::Tensor& pages, int64_t keys) {
  const int64_t rows = pages.size(3), heads = pages.size(0) * 2 * pages.size(2);
  bind_device_context();
  CUtensorMap map;
  cuuint64_t dims[3] = {(cuuint64_t)kCacheDim, (cuuint64_t)rows, (cuuint64_t)heads};
  cuuint64_t strides[2] = {(cuuint64_t)kCacheDim, (cuuint64_t)(rows * kCacheDim)};
  cuuint32_t box[3] = {(cuuint32_t)kCacheDim, (cuuint32_t)std::min<int64_t>(rows, keys), 1};
  cuuint32_t estr[3] = {1, 1, 1};
  CUresult r = tensor_map_encoder()(&map, CU_TENSOR_MAP_DATA_TYPE_UINT8, 3, pages.data_ptr(), dims, strides, box, estr,
                                    CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B,
                                    CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
  TORCH_CHECK(r == CUDA_SUCCESS, "cuTensorMapEncodeTiled (pages) failed with code ", (int)r);
  return map;
}

// Query rows [tokens, H, 128]: boxes of 128 / group tokens, the heads of a group, 64 dimensions.
CUtensorMap queries_map(const at::Tensor& q, int64_t group) {
  bind_device_context();
  CUtensorMap map;
  cuuint64_t dims[3] = {(cuuint64_t)kCacheDim, (cuuint64_t)q.size(1), (cuuint64_t)q.size(0)};
  cuuint64_t strides[2] = {(cuuint64_t)(q.stride(1) * 2), (cuuint64_t)(q.stride(0) * 2)};
  cuuint32_t box[3] = {64, (cuuint32_t)group, (cuuint32_t)(128 / group)};
  cuuint32_t estr[3] = {1, 1, 1};
  const auto type = q.scalar_type() == at::kBFloat16 ? CU_TENSOR_MAP_DATA_TYPE_BFLOAT16 : CU_TENSOR_MAP_DATA_TYPE_FLOAT16;
  CUresult r = tensor_map_encoder()(&map, type, 3, q.data_ptr(), dims, strides, box, estr, CU_TENSOR_MAP_INTERLEAVE_NONE,
                                    CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
                                    CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
  TORCH_CHECK(r == CUDA_SUCCESS, "cuTensorMapEncodeTiled (queries) failed with code ", (int)r);
  return map;
}

// Counters that are zero before and after every call, and room for partial sums (7.4 MB).  Both are kept per stream,
// whose calls follow one another.  A graph may run beside the stream that it was captured on: it has counters of
// its own (per stream of the capture, cleared at its first call), and its partial sums come from its pool.
// Its counters do not: they outlive it, and would hold a whole segment of that pool.
struct AttentionParts {
  float2 ml[kAttentionBlocks][2][kAttentionRows];
  float sums[kAttentionBlocks][2][kAttentionRows][kCacheDim];
};

struct AttentionWork {
  at::Tensor arrived, parts;
};

AttentionWork attention_work(const at::Device& dev, cudaStream_t stream) {
  cudaStreamCaptureStatus capturing = cudaStreamCaptureStatusNone;
  unsigned long long capture = 0;
  C10_CUDA_CHECK(cudaStreamGetCaptureInfo(stream, &capturing, &capture));
  if (capturing == cudaStreamCaptureStatusNone) capture = 0;  // captures count from one
  const auto bytes = at::TensorOptions().device(dev).dtype(at::kByte);
  static std::mutex mutex;
  // Never freed: the tensors may outlive the context, and nothing tells when a graph is gone (2 KB each).
  static auto* kept = new std::map<std::tuple<int, cudaStream_t, unsigned long long>, AttentionWork>;
  std::lock_guard<std::mutex> lock(mutex);
  AttentionWork& work = (*kept)[{dev.index(), stream, capture}];
  if (!work.arrived.defined()) {
    {
      c10::cuda::CUDAStreamCaptureModeGuard relaxed(cudaStreamCaptureModeRelaxed);
      // Memory asked for on a stream that is not captured is the common pool's; always the same stream, since
      // every stream has segments of its own.
      static std::map<int, c10::cuda::CUDAStream> others;
      c10::cuda::OptionalCUDAStreamGuard other;
      if (capture != 0) {
        auto it = others.find(dev.index());
        if (it == others.end()) it = others.emplace(dev.index(), c10::cuda::getStreamFromPool(false, dev.index())).first;
        other.reset_stream(it->second);
      }
      work.arrived = at::empty({kAttentionBlocks * (int64_t)sizeof(int)}, bytes);
    }
    C10_CUDA_CHECK(cudaMemsetAsync(work.arrived.data_ptr(), 0, kAttentionBlocks * sizeof(int), stream));
    if (capture == 0) work.parts = at::empty({(int64_t)sizeof(AttentionParts)}, bytes);
  }
  if (capture == 0) return work;
  return {work.arrived, at::empty({(int64_t)sizeof(AttentionParts)}, bytes)};
}

const at::Tensor* given(const c10::optional<at::Tensor>& t) { return t.has_value() ? &*t : nullptr; }

}  // namespace

// The first status code of a cache kernel since the last read (0: none).
int64_t cache_status(int64_t device) {
  c10::cuda::CUDAGuard guard(static_cast<c10::DeviceIndex>(device));
  int* word = status_word(at::Device(at::kCUDA, static_cast<c10::DeviceIndex>(device)));
  int host = 0;
  C10_CUDA_CHECK(cudaStreamSynchronize(at::cuda::getCurrentCUDAStream()));  // this stream's kernels have reported
  C10_CUDA_CHECK(cudaMemcpy(&host, word, sizeof(int), cudaMemcpyDeviceToHost));
  if (host) C10_CUDA_CHECK(cudaMemset(word, 0, sizeof(int)));
  return host;
}

at::Tensor cache_append(at::Tensor q, at::Tensor k, at::Tensor v, at::Tensor cos, at::Tensor sin, at::Tensor pages,
                        at::Tensor scales, at::Tensor table, at::Tensor lens, at::Tensor seqs, at::Tensor cu_new) {
  check_pool(pages, scales, 0);
  const at::Device dev = pages.device();
  check_rows(q, "q", dev);
  check_rows(k, "k", dev);
  check_rows(v, "v", dev);
  check_batch(table, lens, seqs, cu_new, dev);
  SERVING_CHECK(q.scalar_type() == k.scalar_type() && q.scalar_type() == v.scalar_type(), "q, k and v must have one type");
  SERVING_CHECK(k.size(1) == pages.size(2) && v.size(1) == pages.size(2), "k and v must have the pages' ", pages.size(2),
              " heads");
  SERVING_CHECK(k.size(0) == q.size(0) && v.size(0) == q.size(0), "q, k and v must have as many tokens");
  SERVING_CHECK(q.size(1) >= 1 && q.size(1) % k.size(1) == 0, "query heads ", q.size(1),
              " must be divisible by key/value heads ", k.size(1));
  for (const at::Tensor* t : {&cos, &sin})
    SERVING_CHECK(t->device() == dev && t->scalar_type() == at::kFloat && t->dim() == 2 && t->size(1) == kCacheDim &&
                    t->is_contiguous() && reinterpret_cast<uintptr_t>(t->data_ptr()) % 16 == 0,
                "cos and sin must be contiguous float32 tables [positions, 128]");
  SERVING_CHECK(cos.size(0) == sin.size(0), "cos and sin must have as many positions");
  SERVING_CHECK(q.size(0) < (int64_t(1) << 31) - 64 && k.size(1) < 65536, "too many tokens or heads");
  c10::cuda::CUDAGuard guard(dev);
  at::Tensor out = at::empty({q.size(0), q.size(1), kCacheDim}, q.options());
  if (q.size(0) == 0) return out;
  AppendParams p{};
  p.q = q.data_ptr(), p.k = k.data_ptr(), p.v = v.data_ptr();
  p.q_tok = q.stride(0), p.q_head = q.stride(1);
  p.k_tok = k.stride(0), p.k_head = k.stride(1);
  p.v_tok = v.stride(0), p.v_head = v.stride(1);
  p.q_out = out.data_ptr();
  p.cos = cos.data_ptr<float>(), p.sin = sin.data_ptr<float>();
  p.positions = cos.size(0);
  p.pages = static_cast<uint8_t*>(pages.data_ptr());
  p.scales = scales.data_ptr<float>();
  p.npages = pages.size(0);
  p.table = table.data_ptr<int>(), p.lens = lens.data_ptr<int>();
  p.seqs = seqs.data_ptr<int>(), p.cu = cu_new.data_ptr<int>();
  p.slots = (int)table.size(0), p.width = (int)table.size(1), p.n = (int)seqs.size(0);
  p.tokens = (int)q.size(0), p.H = (int)q.size(1), p.KV = (int)k.size(1), p.page = (int)pages.size(3);
  p.status = status_word(dev);
  C10_CUDA_CHECK(launch_cache_append(p, q.scalar_type() == at::kBFloat16, at::cuda::getCurrentCUDAStream()));
  return out;
}

at::Tensor cache_reserve(at::Tensor table, at::Tensor lens, at::Tensor refs, at::Tensor seqs, at::Tensor counts,
                         int64_t page) {
  const Book b = book_of(table, lens, refs, page);
  check_int32(seqs, "seqs", 1, table.device());
  check_int32(counts, "counts", 1, table.device());
  const int64_t n = seqs.size(0);
  SERVING_CHECK(counts.size(0) == n, "counts needs one entry for each of seqs");
  SERVING_CHECK(n <= kBookBatch, "at most ", kBookBatch, " sequences a call");
  c10::cuda::CUDAGuard guard(table.device());
  // [missing | free pages found]
  const int64_t most = std::min<int64_t>(n * table.size(1), refs.size(0));
  at::Tensor work = at::empty({1 + std::max<int64_t>(most, 1)}, refs.options());
  int* w = work.data_ptr<int>();
  C10_CUDA_CHECK(launch_cache_reserve(b, seqs.data_ptr<int>(), counts.data_ptr<int>(), (int)n, w + 1, w,
                                      at::cuda::getCurrentCUDAStream()));
  return work.narrow(0, 0, 1);
}

void cache_free(at::Tensor table, at::Tensor lens, at::Tensor refs, at::Tensor seqs) {
  const Book b = book_of(table, lens, refs, kCacheBlock);
  check_int32(seqs, "seqs", 1, table.device());
  if (seqs.size(0) == 0) return;
  c10::cuda::CUDAGuard guard(table.device());
  C10_CUDA_CHECK(launch_cache_free(b, seqs.data_ptr<int>(), (int)seqs.size(0), at::cuda::getCurrentCUDAStream()));
}

at::Tensor cache_fork(at::Tensor pages, at::Tensor scales, at::Tensor table, at::Tensor lens, at::Tensor refs,
                      at::Tensor src, at::Tensor dst) {
  check_pool(pages, scales, 1);
  const Book b = book_of(table, lens, refs, pages.size(4));
  SERVING_CHECK(table.device() == pages.device(), "page_table and pages must be on one device");
  check_int32(src, "src", 1, table.device());
  check_int32(dst, "dst", 1, table.device());
  SERVING_CHECK(refs.size(0) == pages.size(1), "ref_counts needs one count for each page");
  const int64_t n = src.size(0);
  SERVING_CHECK(dst.size(0) == n, "src and dst must have as many slots");
  SERVING_CHECK(n <= kBookBatch, "at most ", kBookBatch, " sequences a call");
  c10::cuda::CUDAGuard guard(table.device());
  at::Tensor work = at::empty({1 + 3 * std::max<int64_t>(n, 1)}, refs.options());  // missing | from | to | found
  int* w = work.data_ptr<int>();
  auto stream = at::cuda::getCurrentCUDAStream();
  C10_CUDA_CHECK(launch_cache_fork(b, src.data_ptr<int>(), dst.data_ptr<int>(), (int)n, w + 1, w + 1 + n, w + 1 + 2 * n, w,
                                   stream));
  CopyParams p = copy_of(pages, scales, pages, scales);
  p.n = (int)n;
  p.from = w + 1;
  p.to = w + 1 + n;
  p.missing = w;
  C10_CUDA_CHECK(launch_cache_copy(p, stream));
  return work.narrow(0, 0, 1);
}

void cache_copy(at::Tensor pages, at::Tensor scales, at::Tensor src, at::Tensor dst) {
  check_pool(pages, scales, 1);
  check_int32(src, "src", 1, pages.device());
  check_int32(dst, "dst", 1, pages.device());
  SERVING_CHECK(src.size(0) == dst.size(0), "src and dst must have as many pages");
  SERVING_CHECK(src.size(0) < (int64_t(1) << 31), "too many pages");
  c10::cuda::CUDAGuard guard(pages.device());
  CopyParams p = copy_of(pages, scales, pages, scales);
  p.n = (int)src.size(0);
  p.from = src.data_ptr<int>();
  p.to = dst.data_ptr<int>();
  C10_CUDA_CHECK(launch_cache_copy(p, at::cuda::getCurrentCUDAStream()));
}

// out_*: another pool (its table the shape of `table`), or the same tensors for a move in place.
at::Tensor cache_compact(at::Tensor pages, at::Tensor scales, at::Tensor table, at::Tensor refs, at::Tensor out_pages,
                         at::Tensor out_scales, at::Tensor out_table, at::Tensor out_refs) {
  check_pool(pages, scales, 1);
  check_pool(out_pages, out_scales, 1);
  const at::Device dev = pages.device();
  check_int32(table, "page_table", 2, dev);
  check_int32(refs, "ref_counts", 1, dev);
  check_int32(out_table, "the new page_table", 2, dev);
  check_int32(out_refs, "the new ref_counts", 1, dev);
  SERVING_CHECK(out_pages.device() == dev, "both pools must be on one device");
  SERVING_CHECK(out_table.sizes() == table.sizes(), "the new page_table must have the shape of the old one");
  SERVING_CHECK(refs.size(0) == pages.size(1) && out_refs.size(0) == out_pages.size(1),
                "ref_counts needs one count for each page");
  SERVING_CHECK(refs.size(0) < (int64_t(1) << 30) && out_refs.size(0) < (int64_t(1) << 30), "the pool has too many pages");
  for (int64_t i : {0, 2, 3, 4, 5})
    SERVING_CHECK(pages.size(i) == out_pages.size(i), "the new pool must differ in its number of pages only");
  const bool in_place = pages.data_ptr() == out_pages.data_ptr();
  SERVING_CHECK(in_place == (table.data_ptr() == out_table.data_ptr()) && in_place == (refs.data_ptr() == out_refs.data_ptr()) &&
                    in_place == (scales.data_ptr() == out_scales.data_ptr()) &&
                    (!in_place || pages.size(1) == out_pages.size(1)),
                "compact into a pool of its own, or in place throughout");
  c10::cuda::CUDAGuard guard(dev);
  const int np = (int)refs.size(0);
  const int64_t span = std::max(np, 1);
  at::Tensor work = at::empty({1 + 3 * span}, refs.options());  // missing | to | holes | the old counts
  int* w = work.data_ptr<int>();
  auto stream = at::cuda::getCurrentCUDAStream();
  C10_CUDA_CHECK(launch_cache_plan(refs.data_ptr<int>(), np, out_refs.data_ptr<int>(), (int)out_refs.size(0), w + 1 + span, w + 1,
                                   w + 1 + 2 * span, w, stream));
  CopyParams p = copy_of(pages, scales, out_pages, out_scales);
  p.n = np;
  p.to = w + 1;
  p.missing = w;
  p.table = table.data_ptr<int>();
  p.out_table = out_table.data_ptr<int>();
  p.entries = table.numel();
  C10_CUDA_CHECK(launch_cache_copy(p, stream));
  return work.narrow(0, 0, 1);
}

// kernel: 0 chooses; 1 is the kernel that splits the keys, 2 the one for prompts.
at::Tensor cache_attention(at::Tensor q, at::Tensor pages, at::Tensor scales, at::Tensor table, at::Tensor lens,
                           at::Tensor seqs, at::Tensor cu_new, c10::optional<at::Tensor> prefix_lens,
                           double softmax_scale, int64_t max_new, int64_t kernel) {
  check_pool(pages, scales, 0);
  const at::Device dev = pages.device();
  check_rows(q, "q", dev);
  check_batch(table, lens, seqs, cu_new, dev);
  const int64_t H = q.size(1), KV = pages.size(2);
  SERVING_CHECK(H >= 1 && H % KV == 0, "query heads ", H, " must be divisible by key/value heads ", KV);
  SERVING_CHECK(q.size(0) * (H / KV) < (int64_t(1) << 31) - 64, "too many query rows");
  SERVING_CHECK(table.size(1) * pages.size(3) < (int64_t(1) << 31) - 4096, "sequences of 2^31 tokens or more");
  if (prefix_lens.has_value()) {
    check_int32(*prefix_lens, "prefix_lens", 1, dev);
    SERVING_CHECK(prefix_lens->size(0) == seqs.size(0), "prefix_lens needs one length for each of seqs");
  }
  c10::cuda::CUDAGuard guard(dev);
  at::Tensor out = at::empty({q.size(0), H, kCacheDim}, q.options());
  const int64_t n = seqs.size(0);
  if (q.size(0) == 0) return out;
  if (n == 0 || pages.size(0) == 0) return out.zero_();
  AttentionParams p{};
  p.q = q.data_ptr();
  p.q_tok = q.stride(0), p.q_head = q.stride(1);
  p.out = out.data_ptr();
  p.scales = scales.data_ptr<float>();
  p.table = table.data_ptr<int>(), p.lens = lens.data_ptr<int>();
  p.slots = (int)table.size(0), p.width = (int)table.size(1), p.tokens = (int)q.size(0);
  p.H = (int)H, p.KV = (int)KV, p.group = (int)(H / KV);
  p.page = (int)pages.size(3), p.page_shift = __builtin_ctz(p.page), p.npages = (int)pages.size(0);
  p.scale_log2 = (float)(softmax_scale * 1.4426950408889634);
  p.status = status_word(dev);
  auto stream = at::cuda::getCurrentCUDAStream();
  const bool bf16 = q.scalar_type() == at::kBFloat16;
  // (q strides of zero, a broadcast, are not for a tensor map)
  const bool can = p.group <= 64 && p.scale_log2 > 0.f && q.stride(0) > 0 && q.stride(1) > 0;
  SERVING_CHECK(kernel != 2 || can, "the prompt kernel cannot take these arguments");
  // Both kernels' times grow with the keys alike.  The one that splits them takes 4.2 ns for 16 rows and 64
  // keys on the whole GPU, the prompt kernel 1.05 us for the 256 rows of each of 148 blocks.  Measured on both
  // sides of the line (split / prompt): 4096 keys, 4 key/value heads, 16 heads, one sequence, 128 new tokens
  // 60 / 83 us, 256 88 / 84; 16 sequences, 8 new 61 / 65, 16 90 / 65; 64 sequences, 4 new 100 / 135, 8 165 / 136;
  // 16 and 16 heads, 16 sequences, 16 new 100 / 134, 32 166 / 134.
  const int64_t row_tiles = KV * std::max<int64_t>(n, (q.size(0) * p.group + 15) / 16);
  const int64_t per = p.group <= 64 ? 2 * (128 / p.group) : 1;
  const int64_t blocks = KV * std::max<int64_t>(n, (q.size(0) + per - 1) / per);
  if (kernel == 2 || (kernel == 0 && can && row_tiles >= 250 * ((blocks + 147) / 148))) {
    const CUtensorMap map_q = queries_map(q, p.group), map_pages = pages_map(pages, kPromptKeys);
    for (int64_t base = 0; base < n; base += kAttentionSeqs) {
      p.n = (int)std::min<int64_t>(kAttentionSeqs, n - base);
      p.seqs = seqs.data_ptr<int>() + base;
      p.cu = cu_new.data_ptr<int>() + base;
      p.prefix = prefix_lens.has_value() ? prefix_lens->data_ptr<int>() + base : nullptr;
      p.first_batch = base == 0;
      p.last_batch = base + p.n == n;
      C10_CUDA_CHECK(launch_cache_prompt(map_q, map_pages, p, bf16, stream));
    }
    return out;
  }
  const CUtensorMap map = pages_map(pages, kAttentionKeys);
  const AttentionWork work = attention_work(dev, stream);
  auto* parts = static_cast<AttentionParts*>(work.parts.data_ptr());
  p.arrived = static_cast<int*>(work.arrived.data_ptr());
  p.parts = &parts->sums[0][0][0][0];
  p.part_ml = &parts->ml[0][0][0];
  // Tiles of 8 rows are faster where they hold a sequence's rows, and right where they do not.
  const bool full = max_new < 1 || max_new * p.group > 8;
  const int64_t tile = full ? kAttentionRows : 8;
  const int64_t tiles = KV * std::max<int64_t>(n, (q.size(0) * p.group + tile - 1) / tile);
  for (int64_t base = 0; base < n; base += kAttentionSeqs) {
    p.n = (int)std::min<int64_t>(kAttentionSeqs, n - base);
    p.seqs = seqs.data_ptr<int>() + base;
    p.cu = cu_new.data_ptr<int>() + base;
    p.prefix = prefix_lens.has_value() ? prefix_lens->data_ptr<int>() + base : nullptr;
    p.join_cost = 4.f * (float)tiles * (float)p.n / (float)n;
    p.first_batch = base == 0;
    p.last_batch = base + p.n == n;
    // no more blocks than units: at most this many
    const int64_t segments = std::min<int64_t>(q.size(0), p.n) + q.size(0) * p.group / tile + 1;
    const int64_t most = segments * KV * (((int64_t)p.width * p.page + kAttentionKeys - 1) / kAttentionKeys + 1 + kAttentionEnds);
    const int grid = (int)std::min<int64_t>(kAttentionBlocks, std::max<int64_t>(most, 1));
    C10_CUDA_CHECK(launch_cache_attention(map, p, bf16, full, grid, stream));
  }
  return out;
}

at::Tensor process_logits(at::Tensor logits, c10::optional<at::Tensor> tokens, c10::optional<at::Tensor> token_lens,
                          c10::optional<at::Tensor> prompt_lens, c10::optional<at::Tensor> repetition,
                          c10::optional<at::Tensor> presence, c10::optional<at::Tensor> frequency,
                          c10::optional<at::Tensor> bias_offsets, c10::optional<at::Tensor> bias_ids,
                          c10::optional<at::Tensor> bias_values, c10::optional<at::Tensor> allowed,
                          c10::optional<at::Tensor> out) {
  SERVING_CHECK(logits.is_cuda() && logits.dim() == 2 && (logits.stride(1) == 1 || logits.size(1) <= 1),
                    "logits must be [rows, vocab] on the GPU with contiguous rows");
  const auto type = logits.scalar_type();
  SERVING_CHECK(type == at::kBFloat16 || type == at::kHalf || type == at::kFloat,
                    "logits must be bfloat16, float16 or float32");
  const at::Device dev = logits.device();
  const int64_t rows = logits.size(0), vocab = logits.size(1);
  SERVING_CHECK(rows < 65536 && vocab < (int64_t(1) << 31) - 8192, "too many rows or too large a vocabulary");
  auto per_row = [&](const at::Tensor* t, const char* name, at::ScalarType want, int64_t size) {
    if (t == nullptr) return;
    SERVING_CHECK(t->device() == dev && t->scalar_type() == want && t->dim() == 1 && t->size(0) == size && t->is_contiguous(),
                      name, " must be a contiguous ", want, " tensor of ", size, " on ", dev);
  };
  per_row(given(token_lens), "token_lens", at::kInt, rows);
  per_row(given(prompt_lens), "prompt_lens", at::kInt, rows);
  per_row(given(repetition), "repetition", at::kFloat, rows);
  per_row(given(presence), "presence", at::kFloat, rows);
  per_row(given(frequency), "frequency", at::kFloat, rows);
  per_row(given(bias_offsets), "the bias offsets", at::kInt, rows + 1);
  if (tokens.has_value()) {
    SERVING_CHECK(tokens->device() == dev && tokens->scalar_type() == at::kInt && tokens->dim() == 2 &&
                          tokens->size(0) == rows && (tokens->stride(1) == 1 || tokens->size(1) <= 1) &&
                          tokens->size(1) < (int64_t(1) << 21),
                      "tokens must be int32 [rows, history < 2^21] on ", dev, " with contiguous rows");
  } else {
    SERVING_CHECK(!token_lens.has_value() && !prompt_lens.has_value() && !repetition.has_value() &&
                          !presence.has_value() && !frequency.has_value(),
                      "lengths and penalties need tokens");
  }
  SERVING_CHECK(bias_offsets.has_value() == bias_ids.has_value() && bias_ids.has_value() == bias_values.has_value(),
                    "bias is (offsets, ids, values)");
  if (bias_ids.has_value()) {
    SERVING_CHECK(bias_ids->dim() == 1 && bias_ids->size(0) < (int64_t(1) << 31) - 1024, "too many biases");
    per_row(given(bias_ids), "the bias ids", at::kInt, bias_ids->numel());
    per_row(given(bias_values), "the bias values", at::kFloat, bias_ids->numel());
  }
  if (allowed.has_value()) {
    SERVING_CHECK(allowed->device() == dev && allowed->scalar_type() == at::kInt && allowed->dim() == 2 &&
                          allowed->size(0) == rows && allowed->size(1) == (vocab + 31) / 32 &&
                          (allowed->stride(1) == 1 || allowed->size(1) <= 1),
                      "allowed must be int32 [rows, ceil(vocab / 32)] on ", dev, " with contiguous rows");
  }
  c10::cuda::CUDAGuard guard(dev);
  at::Tensor y;
  if (out.has_value()) {
    SERVING_CHECK(out->device() == dev && out->scalar_type() == at::kFloat && out->is_contiguous() &&
                          out->sizes() == logits.sizes(),
                      "out must be contiguous float32 of the logits' shape on ", dev);
    const char* a = static_cast<const char*>(logits.data_ptr());
    const char* b = static_cast<const char*>(out->data_ptr());
    const bool apart = rows == 0 || vocab == 0 || b + out->nbytes() <= a ||
                       a + ((rows - 1) * logits.stride(0) + vocab) * logits.element_size() <= b;
    SERVING_CHECK(apart || (a == b && type == at::kFloat && logits.is_contiguous()),
                      "out may be the logits only where they are contiguous float32, and else shares no memory with them");
    y = *out;
  } else {
    y = at::empty({rows, vocab}, logits.options().dtype(at::kFloat));
  }
  if (rows == 0 || vocab == 0) return y;
  auto ints = [](const c10::optional<at::Tensor>& t) { return t.has_value() ? t->data_ptr<int>() : nullptr; };
  auto floats = [](const c10::optional<at::Tensor>& t) { return t.has_value() ? t->data_ptr<float>() : nullptr; };
  LogitsParams p{};
  p.logits = logits.data_ptr();
  p.ld = logits.stride(0);
  p.out = y.data_ptr<float>();
  p.rows = (int)rows, p.vocab = (int)vocab;
  p.tokens = ints(tokens);
  p.tokens_ld = tokens.has_value() ? tokens->stride(0) : 0;
  p.tokens_width = tokens.has_value() ? (int)tokens->size(1) : 0;
  p.token_lens = ints(token_lens), p.prompt_lens = ints(prompt_lens);
  p.repetition = floats(repetition), p.presence = floats(presence), p.frequency = floats(frequency);
  p.bias_offsets = ints(bias_offsets), p.bias_ids = ints(bias_ids), p.bias_values = floats(bias_values);
  p.bias_count = bias_ids.has_value() ? (int)bias_ids->numel() : 0;
  p.allowed = ints(allowed);
  p.allowed_ld = allowed.has_value() ? allowed->stride(0) : 0;
  C10_CUDA_CHECK(launch_process_logits(
      p, type == at::kFloat ? kLogitsFloat : type == at::kHalf ? kLogitsHalf : kLogitsBFloat16, at::cuda::getCurrentCUDAStream()));
  return y;
}
