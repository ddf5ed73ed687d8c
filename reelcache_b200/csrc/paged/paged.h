// What the paged-cache kernels share: the checked views of pages and block tables, and their status codes.
#pragma once

#include <ATen/ATen.h>
#include <ATen/Context.h>
#include <ATen/cuda/EmptyTensor.h>
#include <c10/core/impl/TorchDispatchModeTLS.h>

#include "../common/host.h"

namespace rc {

// The paged kernels report into the second word of the device's status words: a table entry that is out of range, or a
// page-table call that was refused, leaves everything in bounds and consistent, so it must not stop the waits of later
// kernels, which watch the first word.
constexpr int kPagedWord = 1;
constexpr int kPageExhausted = 0x401;
constexpr int kPageRefused = 0x402;
constexpr int kPageRange = 0x403;
constexpr int kPageRows = 0x404;

namespace paged {

constexpr int kPlanThreads = 1024;  // of the one-block kernels that plan

// Every kernel here is launched as a programmatic dependent of what runs before it on the stream: its launch and its setup
// overlap that kernel's end. after_earlier() comes before its first access to global memory and waits until everything
// before it on the stream is complete and visible; let_later() allows the next such kernel to be set up.
// A grid is thus alive while kernels before it still write, so its inputs must not go through the non-coherent path, which
// is for what nobody writes in a grid's lifetime: no __ldg and no __restrict__ on anything that another kernel makes
// (rows, positions, tables, lengths, plans).
#ifdef __CUDACC__
__device__ __forceinline__ void after_earlier() { asm volatile("griddepcontrol.wait;" ::: "memory"); }
__device__ __forceinline__ void let_later() { asm volatile("griddepcontrol.launch_dependents;" ::: "memory"); }

// Exclusive prefix sum over the block and its total (kPlanThreads threads, all of them).
__device__ __forceinline__ int block_scan(int value, int* warp_sums, int* total) {
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  int x = value;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const int y = __shfl_up_sync(0xffffffffu, x, o);
    if (lane >= o) x += y;
  }
  __syncthreads();  // warp_sums of a previous call has been read
  if (lane == 31) warp_sums[warp] = x;
  __syncthreads();
  if (warp == 0) {
    int w = warp_sums[lane];
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const int y = __shfl_up_sync(0xffffffffu, w, o);
      if (lane >= o) w += y;
    }
    warp_sums[lane] = w;
  }
  __syncthreads();
  *total = warp_sums[31];
  return x - value + (warp > 0 ? warp_sums[warp - 1] : 0);
}

// `cluster` CTAs to a cluster (0: no clusters).
template <typename... Params, typename... Args>
void launch(void (*kernel)(Params...), dim3 grid, int threads, int smem, int cluster, cudaStream_t stream, const Args&... args) {
  cudaLaunchConfig_t config{};
  config.gridDim = grid;
  config.blockDim = dim3(threads);
  config.dynamicSmemBytes = smem;
  config.stream = stream;
  cudaLaunchAttribute attributes[2] = {};
  attributes[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attributes[0].val.programmaticStreamSerializationAllowed = 1;
  attributes[1].id = cudaLaunchAttributeClusterDimension;
  attributes[1].val.clusterDim.x = cluster;
  attributes[1].val.clusterDim.y = 1;
  attributes[1].val.clusterDim.z = 1;
  config.attrs = attributes;
  config.numAttrs = cluster > 0 ? 2 : 1;
  RC_CUDA(cudaLaunchKernelEx(&config, kernel, static_cast<Params>(args)...));
}
#endif

// Division by a number below 2^24 of numbers below 2^31 as a product (an integer division takes some hundred cycles, of which a
// chain of small steps has few to spare).
struct Divider {
  uint32_t magic, shift;
  int by;
  static Divider of(int by) {
    uint32_t bits = 0;
    while ((int64_t{1} << bits) < by) ++bits;
    return {static_cast<uint32_t>(((uint64_t{1} << (31 + bits)) + by - 1) / by), 31 + bits, by};
  }
#ifdef __CUDACC__
  __device__ __forceinline__ int over(int n) const { return static_cast<int>((static_cast<uint64_t>(static_cast<uint32_t>(n)) * magic) >> shift); }
  __device__ __forceinline__ int up(int n) const { return over(n) + (n > over(n) * by); }  // rounded up
#endif
};

// A new tensor on `like`'s device, without the dispatcher (half a microsecond of a call's five) where nobody asks for it: a
// dispatch mode sees allocations, and deterministic algorithms fill new memory.
inline at::Tensor new_tensor(at::IntArrayRef sizes, const at::Tensor& like, at::ScalarType type) {
  const at::TensorOptions options = like.options().dtype(type);
  const at::Context& context = at::globalContext();
  if (c10::impl::TorchDispatchModeTLS::any_modes_set() ||
      (context.deterministicAlgorithms() && context.deterministicFillUninitializedMemory()))
    return at::empty(sizes, options);
  return at::detail::empty_cuda(sizes, options);
}

struct Pages {  // [pages, page_size, kv_heads, head_dim], strides in elements
  int count, size;
  int64_t page_stride, token_stride, head_stride;
};

struct Table {
  const int* table;    // [seqs, width], `row` elements apart, or [seqs, kv_heads, width]
  const int* kv_lens;  // [seqs]
  const int* cu_q;     // [seqs + 1]
  int seqs, width;
  int64_t row;         // elements from one sequence's row to the next
  int64_t head;        // and from one KV head's to the next (0: the heads share it)
};

inline Pages check_pages(const at::Tensor& t, int64_t heads, int64_t head_dim, const char* name) {
  const std::string who(name);
  RC_CHECK(t.dim() == 4 && t.size(2) == heads && t.size(3) == head_dim && t.stride(3) == 1,
           who + " must be [pages, page_size, kv_heads, head_dim] with unit inner stride");
  RC_CHECK(t.size(0) >= 1 && t.size(0) < (1ll << 31) && t.size(1) >= 8 && t.size(1) % 8 == 0 && t.size(1) <= 65536,
           who + ": the page size must be a multiple of 8 tokens, at most 65536");
  RC_CHECK(t.stride(0) % 8 == 0 && t.stride(1) % 8 == 0 && t.stride(2) % 8 == 0 &&
               reinterpret_cast<uintptr_t>(t.data_ptr()) % 16 == 0,
           who + " must have 16-byte aligned strides and base");
  return {static_cast<int>(t.size(0)), static_cast<int>(t.size(1)), t.stride(0), t.stride(1), t.stride(2)};
}

// kv_heads: of a call that takes a table for each KV head too (0: of one that does not).
inline Table check_table(const at::Tensor& table, const at::Tensor& kv_lens, const at::Tensor& cu_q,
                         const at::Device& device, int64_t kv_heads = 0) {
  const at::Tensor* all[3] = {&table, &kv_lens, &cu_q};
  for (const at::Tensor* t : all)
    RC_CHECK(t->device() == device && t->scalar_type() == at::kInt && (t == &table || t->is_contiguous()),
             "block_table, kv_lens and cu_q must be contiguous int32 tensors on the device of q (rows of the table may be "
             "strided)");
  const bool each = kv_heads > 0 && table.dim() == 3 && table.size(1) == kv_heads && table.stride(1) >= 0;
  const int64_t last = table.dim() - 1;
  RC_CHECK((table.dim() == 2 || each) && (table.stride(last) == 1 || table.size(last) <= 1) && table.stride(0) >= 0 && kv_lens.dim() == 1 &&
               cu_q.dim() == 1 && kv_lens.size(0) == table.size(0) && cu_q.size(0) == table.size(0) + 1,
           kv_heads > 0 ? "block_table is [seqs, width] or [seqs, kv_heads, width], kv_lens [seqs], cu_q [seqs + 1]"
                        : "block_table is [seqs, width], kv_lens [seqs], cu_q [seqs + 1]");
  RC_CHECK(table.size(0) < (1 << 20) && table.size(last) < (1ll << 31), "too many sequences or pages per sequence");
  return {table.data_ptr<int>(), kv_lens.data_ptr<int>(), cu_q.data_ptr<int>(), static_cast<int>(table.size(0)),
          static_cast<int>(table.size(last)), table.stride(0), each ? table.stride(1) : 0};
}

}  // namespace paged
}  // namespace rc
