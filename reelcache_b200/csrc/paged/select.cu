// Sparse attention's choice over a paged cache, for sm_100a: means of the keys of blocks, and the blocks that each block of
// queries attends to.
//
// A block is `block` consecutive positions of a sequence (a divisor of the page size, so that it lies in one page); its mean is
// kept with its page, so sequences that share pages share means. Means are sums in FP64 divided once: the order of the sum does
// not show, whichever tokens came in which call.
//
// The score of a block for the queries of a KV head's group is max over the heads h of (sum over the tokens of the query block
// of q_h) . mean. Blocks at the border of the choice differ by little, so it is computed in FP64, where the order of a sum
// moves it by 2^-50 of its size: the choice is that of the exact scores, the same for every batch and form of the kernel.
// Equal scores go to the lower block.
//
// One CTA, or a cluster of them that splits the blocks, for every (query block, KV head): pooled queries in shared memory,
// scores as 64-bit keys that sort like them in the shared memory of the cluster's first CTA, which finds the keep-th largest
// by digits of eight bits (a histogram each, until a digit's candidates are all taken) and writes the chosen blocks in order.
//
// What bounds it: the latency of a chain of small steps for few sequences, reading the means for many.
#include <ATen/ATen.h>
#include <ATen/MemoryOverlap.h>
#include <c10/cuda/CUDAGuard.h>
#include <c10/cuda/CUDAStream.h>

#include <algorithm>
#include <string>
#include <tuple>
#include <type_traits>

#include "attend.cuh"
#include "packed.h"

namespace rc {
namespace paged {

// -- means ------------------------------------------------------------------------------------------------------------

constexpr int kMeanThreads = 128;

struct Means {
  Args a;                // table, lengths, pages; tokens, max_q_len
  const uint8_t* keys;   // rows of 16-bit numbers, or codes
  int64_t page_stride, token_stride, head_stride;  // bytes
  const uint8_t* scales;  // packed pages, or null
  int64_t scale_page, scale_head;
  char* means;           // [pages, page_size / block, kv_heads, D]: strides in bytes
  int64_t mean_page, mean_block, mean_head;
  int block;
};

__device__ __forceinline__ void add_eight(double (&sum)[8], const uint4& u, __nv_bfloat16) {
  const uint32_t w[4] = {u.x, u.y, u.z, u.w};
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    sum[2 * i] += static_cast<double>(__uint_as_float(w[i] << 16));
    sum[2 * i + 1] += static_cast<double>(__uint_as_float(w[i] & 0xffff0000u));
  }
}
__device__ __forceinline__ void add_eight(double (&sum)[8], const uint4& u, __half) {
  const uint32_t w[4] = {u.x, u.y, u.z, u.w};
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const float2 f = __half22float2(*reinterpret_cast<const __half2*>(&w[i]));
    sum[2 * i] += static_cast<double>(f.x);
    sum[2 * i + 1] += static_cast<double>(f.y);
  }
}

template <typename T>
__device__ __forceinline__ uint4 eight_of(const double (&x)[8]) {
  uint32_t w[4];
#pragma unroll
  for (int i = 0; i < 4; ++i) w[i] = pack2<T>(static_cast<float>(x[2 * i]), static_cast<float>(x[2 * i + 1]));
  return make_uint4(w[0], w[1], w[2], w[3]);
}

// Block (touched block, sequence, KV head): a thread sums eight channels of every (128 / lanes of a row)-th token.
template <typename T, int D, bool kPacked>
__global__ void __launch_bounds__(kMeanThreads) means_kernel(const __grid_constant__ Means p) {
  constexpr int kLanes = D / 8, kRowsAtOnce = kMeanThreads / kLanes;
  __shared__ double part[kRowsAtOnce][kLanes][8];
  let_later();
  after_earlier();
  const Args& a = p.a;
  const int s = blockIdx.y, head = blockIdx.z;
  if (blockIdx.x == 0 && head == 0 && threadIdx.x == 0) report_rows(a, s);
  int q_first;
  const int q_len = min(new_tokens(a, s, &q_first), a.max_q_len), kv_len = held_keys(a, s);
  if (q_len <= 0 || kv_len == 0) return;
  const int b = max(kv_len - q_len, 0) / p.block + blockIdx.x;
  const int64_t from = static_cast<int64_t>(b) * p.block;
  if (from >= kv_len) return;
  const int rows = static_cast<int>(min(static_cast<int64_t>(p.block), kv_len - from));
  const int slot = static_cast<int>(from / a.tiling.page), row0 = static_cast<int>(from - static_cast<int64_t>(slot) * a.tiling.page);
  const int page = a.table[s * a.table_row + slot];
  if (page < 0 || page >= a.pages) {
    if (threadIdx.x == 0 && head == 0 && a.status != nullptr) atomicCAS(a.status + kPagedWord, 0, kPageRange);
    return;
  }
  const int vec = threadIdx.x % kLanes, group = threadIdx.x / kLanes;
  const uint8_t* src = p.keys + page * p.page_stride + head * p.head_stride + vec * (kPacked ? 8 : 16);
  const uint8_t* scales = kPacked ? p.scales + page * p.scale_page + head * p.scale_head : nullptr;
  double sum[8] = {};
#pragma unroll 4
  for (int r = group; r < rows; r += kRowsAtOnce) {
    const uint8_t* at = src + (row0 + r) * p.token_stride;
    if (kPacked) {
      const uint2 codes = *reinterpret_cast<const uint2*>(at);
      const float scale = scale_value(scales[row0 + r]);
      const uint32_t w[4] = {codes_to_half2(codes.x), upper_codes_to_half2(codes.x), codes_to_half2(codes.y), upper_codes_to_half2(codes.y)};
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const float2 f = __half22float2(*reinterpret_cast<const __half2*>(&w[i]));
        sum[2 * i] += static_cast<double>(f.x * scale);
        sum[2 * i + 1] += static_cast<double>(f.y * scale);
      }
    } else {
      add_eight(sum, *reinterpret_cast<const uint4*>(at), T());
    }
  }
#pragma unroll
  for (int e = 0; e < 8; ++e) part[group][vec][e] = sum[e];
  __syncthreads();
  if (group != 0) return;
  for (int g = 1; g < kRowsAtOnce; ++g)
#pragma unroll
    for (int e = 0; e < 8; ++e) sum[e] += part[g][vec][e];
#pragma unroll
  for (int e = 0; e < 8; ++e) sum[e] /= static_cast<double>(rows);
  char* dst = p.means + page * p.mean_page + (row0 / p.block) * p.mean_block + head * p.mean_head + vec * 16;
  *reinterpret_cast<uint4*>(dst) = eight_of<T>(sum);
}

// -- the choice -------------------------------------------------------------------------------------------------------

constexpr int kSelectThreads = 256;
constexpr int kSelectWarps = kSelectThreads / 32;
constexpr int kMostBlocks = 24576;  // whose keys fit one CTA's shared memory

struct Select {
  Args a;              // q, table, lengths, heads; causal; tokens, max_q_len
  const char* means;
  int64_t mean_page, mean_block, mean_head;
  int block, per_page, keep, query_block, sinks, recent;
  int items, width;
  int* table;          // [items, kv_heads, width]
  int* kv_lens;        // [items]
  int* cu_q;           // [items + 1]
  int cluster;
};

// A number that sorts like the score (both zeros alike).
__device__ __forceinline__ uint64_t key_of(double score) {
  const uint64_t bits = static_cast<uint64_t>(__double_as_longlong(score + 0.0));
  return (bits >> 63) != 0 ? ~bits : bits | 0x8000000000000000ull;
}

__device__ __forceinline__ void store_cluster_u64(uint32_t addr, uint64_t v) {
  asm volatile("st.shared::cluster.u64 [%0], %1;" ::"r"(addr), "l"(v) : "memory");
}

// Exclusive prefix sum over the block's threads and its total.
__device__ __forceinline__ int select_scan(int value, int* sums, int* total) {
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  int x = value;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const int y = __shfl_up_sync(0xffffffffu, x, o);
    if (lane >= o) x += y;
  }
  __syncthreads();  // sums of a previous call have been read
  if (lane == 31) sums[warp] = x;
  __syncthreads();
  int before = x - value, all = 0;
#pragma unroll
  for (int w = 0; w < kSelectWarps; ++w) {
    if (w < warp) before += sums[w];
    all += sums[w];
  }
  *total = all;
  return before;
}

template <typename T, int D>
__global__ void __launch_bounds__(kSelectThreads, 2) select_kernel(const __grid_constant__ Select p) {
  constexpr int kLanes = D / 8;          // lanes of a block's mean
  constexpr int kAtOnce = 32 / kLanes;   // blocks of a warp
  constexpr int kDepth = 4;              // of those in flight
  extern __shared__ __align__(16) uint8_t smem[];
  __shared__ int found[4];               // sequence, its first item, item's new tokens, items in all
  __shared__ int sums[kSelectWarps];
  __shared__ int histogram[256];
  __shared__ int digit[2];               // the digit of the keep-th largest key, how many of it are still to be taken
  const Args& a = p.a;
  const int index = static_cast<int>(blockIdx.x) / p.cluster, rank = static_cast<int>(blockIdx.x) - index * p.cluster;
  const int item = index / a.kv_heads, head = index - item * a.kv_heads;
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  double* pooled = reinterpret_cast<double*>(smem);                             // [group][D]
  uint64_t* keys = reinterpret_cast<uint64_t*>(smem + static_cast<size_t>(a.group) * D * 8);  // [blocks]
  let_later();
  after_earlier();

  // the item's sequence: items are counted sequence by sequence
  int items = 0;
  if (threadIdx.x == 0) found[0] = -1;
  for (int base = 0; base < a.seqs; base += kSelectThreads) {
    const int s = base + static_cast<int>(threadIdx.x);
    int n = 0, q_first = 0, q_len = 0;
    if (s < a.seqs) {
      q_len = min(new_tokens(a, s, &q_first), a.max_q_len);
      n = (q_len + p.query_block - 1) / p.query_block;
      if (index == 0 && rank == 0) report_rows(a, s);
    }
    int total;
    const int before = items + select_scan(n, sums, &total);
    if (item >= before && item < before + n) {
      found[0] = s;
      found[1] = before;
      found[2] = q_len;
    }
    items += total;
    if (item < items && index > 0) break;  // (the same for all threads; the first CTA looks at every sequence)
  }
  __syncthreads();
  const int s = found[0];
  const bool writes = rank == 0 && head == 0 && threadIdx.x == 0;
  int* out = p.table + (static_cast<int64_t>(item) * a.kv_heads + head) * p.width;
  if (s < 0) {  // fewer query blocks than there is room for: the whole cluster
    if (rank == 0)
      for (int i = threadIdx.x; i < p.width; i += kSelectThreads) out[i] = -1;
    if (writes) {
      p.kv_lens[item] = 0;
      p.cu_q[item] = min(max(a.cu_q[a.seqs], 0), a.tokens);
      if (item == p.items - 1) p.cu_q[p.items] = min(max(a.cu_q[a.seqs], 0), a.tokens);
    }
    return;
  }
  const int start = (item - found[1]) * p.query_block, q_len = found[2], count = min(p.query_block, q_len - start);
  const int kv_len = held_keys(a, s), q_first = a.cu_q[s];
  const int end = a.causal ? max(0, min(kv_len, kv_len - q_len + start + count)) : kv_len;
  const int blocks = (end + p.block - 1) / p.block;
  const int64_t near = max(static_cast<int64_t>(0), static_cast<int64_t>(kv_len) - q_len + (a.causal ? start : 0) - p.recent);
  const int high = min(blocks, static_cast<int>(near / p.block)), low = min(high, (p.sinks - 1) / p.block + (p.sinks > 0));
  const int candidates = high - low, keep = min(p.keep, candidates);
  const int chosen = low + keep + blocks - high;
  if (writes) {
    p.kv_lens[item] = chosen > 0 ? (chosen - 1) * p.block + end - (blocks - 1) * p.block : 0;
    p.cu_q[item] = q_first + start;
    if (item == p.items - 1) p.cu_q[p.items] = q_first + start + count;
  }
  const int* table = a.table + s * a.table_row;
  const bool scored = keep > 0 && keep < candidates;  // else there is nothing to choose

  if (scored) {
    // pooled queries: a thread sums eight channels of a head over a part of the tokens; the parts meet where the keys will be
    double* parts = reinterpret_cast<double*>(keys);
    const int vecs = a.group * kLanes, splits = max(1, min(kSelectThreads / vecs, count));
    for (int i = threadIdx.x; i < vecs * splits; i += kSelectThreads) {
      const int split = i / vecs, v = i - split * vecs, h = v / kLanes, vec = v - h * kLanes;
      double sum[8] = {};
      const T* src = static_cast<const T*>(a.q) + static_cast<int64_t>(q_first + start) * a.q_token + (head * a.group + h) * a.q_head + vec * 8;
#pragma unroll 4
      for (int t = split; t < count; t += splits) add_eight(sum, *reinterpret_cast<const uint4*>(src + t * a.q_token), T());
      double* to = splits == 1 ? pooled + v * 8 : parts + i * 8;
#pragma unroll
      for (int e = 0; e < 8; ++e) to[e] = sum[e];
    }
    __syncthreads();
    if (splits > 1) {
      for (int i = threadIdx.x; i < vecs * 8; i += kSelectThreads) {
        double sum = 0.0;
        for (int k = 0; k < splits; ++k) sum += parts[k * vecs * 8 + i];
        pooled[i] = sum;
      }
    }
    if (p.cluster > 1) cluster_sync_all();  // (the first CTA's parts have been read: others may write their keys there)
    else __syncthreads();

    // scores of this CTA's part of the candidates
    const int vec = lane % kLanes, sub = lane / kLanes;
    const uint32_t keys_at = cluster_addr(keys, 0);
    const int from = static_cast<int>(static_cast<int64_t>(candidates) * rank / p.cluster);
    const int to = static_cast<int>(static_cast<int64_t>(candidates) * (rank + 1) / p.cluster);
    for (int c0 = from + warp * kAtOnce * kDepth; c0 < to; c0 += kSelectWarps * kAtOnce * kDepth) {
      uint4 mean[kDepth];
      int page[kDepth];
#pragma unroll
      for (int d = 0; d < kDepth; ++d) {
        const int b = low + c0 + d * kAtOnce + sub;
        page[d] = c0 + d * kAtOnce + sub < to ? table[b / p.per_page] : -1;
      }
#pragma unroll
      for (int d = 0; d < kDepth; ++d) {
        const int b = low + c0 + d * kAtOnce + sub;
        mean[d] = make_uint4(0, 0, 0, 0);
        if (page[d] >= 0 && page[d] < a.pages)
          mean[d] = *reinterpret_cast<const uint4*>(p.means + page[d] * p.mean_page + (b % p.per_page) * p.mean_block + head * p.mean_head + vec * 16);
      }
#pragma unroll
      for (int d = 0; d < kDepth; ++d) {
        double x[8] = {};
        add_eight(x, mean[d], T());
        double best = -INFINITY;
        for (int h = 0; h < a.group; ++h) {
          const double* q = pooled + h * D + vec * 8;
          double dot = 0.0;
#pragma unroll
          for (int e = 0; e < 8; ++e) dot = fma(q[e], x[e], dot);
#pragma unroll
          for (int o = kLanes / 2; o > 0; o >>= 1) dot += __shfl_xor_sync(0xffffffffu, dot, o);
          best = fmax(best, dot);  // (NaN counts for nothing)
        }
        const int c = c0 + d * kAtOnce + sub;
        if (vec == 0 && c < to) store_cluster_u64(keys_at + c * 8, key_of(best));
      }
    }
  }
  if (p.cluster > 1) cluster_sync_all();
  else __syncthreads();
  if (rank != 0) return;

  // the keep-th largest key, digit by digit from the top: `prefix` so far, `rest` of it still to be taken
  uint64_t prefix = 0;
  int shift = 64, rest = keep;
  if (scored) {
    while (shift > 0) {
      for (int i = threadIdx.x; i < 256; i += kSelectThreads) histogram[i] = 0;
      __syncthreads();
      for (int c = threadIdx.x; c < candidates; c += kSelectThreads) {
        const uint64_t key = keys[c];
        if (shift == 64 || (key >> shift) == prefix) atomicAdd(&histogram[(key >> (shift - 8)) & 255], 1);
      }
      __syncthreads();
      // thread i looks at digit 255 - i
      const int mine = histogram[255 - threadIdx.x];
      int total;
      const int above = select_scan(mine, sums, &total);
      if (above < rest && above + mine >= rest) {
        digit[0] = 255 - static_cast<int>(threadIdx.x);
        digit[1] = above;
      }
      __syncthreads();
      const int d = digit[0];
      rest -= digit[1];
      prefix = (prefix << 8) | static_cast<uint64_t>(d);
      shift -= 8;
      if (histogram[d] == rest) break;  // all of them
      __syncthreads();
    }
  }
  // blocks in order: the first ones, the chosen, the last ones
  auto write = [&](int at, int b) {
    const int page = table[b / p.per_page];
    out[at] = page >= 0 && page < a.pages ? page * p.per_page + b % p.per_page : -1;
  };
  for (int i = threadIdx.x; i < low; i += kSelectThreads) write(i, i);
  for (int i = threadIdx.x; i < blocks - high; i += kSelectThreads) write(low + keep + i, high + i);
  for (int i = chosen + static_cast<int>(threadIdx.x); i < p.width; i += kSelectThreads) out[i] = -1;
  if (!scored) {
    if (keep > 0)
      for (int i = threadIdx.x; i < candidates; i += kSelectThreads) write(low + i, low + i);
    return;
  }
  int before = 0, equal = 0;  // taken and equal ones so far
  for (int c0 = 0; c0 < candidates && before < keep; c0 += kSelectThreads) {
    const int c = c0 + static_cast<int>(threadIdx.x);
    const uint64_t top = c < candidates ? (shift == 64 ? 0 : keys[c] >> shift) : 0;
    const bool is_above = c < candidates && top > prefix, is_equal = c < candidates && top == prefix;
    int total_equal, total;
    const int rank_equal = equal + select_scan(is_equal, sums, &total_equal);
    const bool take = is_above || (is_equal && rank_equal < rest);
    const int at = before + select_scan(take, sums, &total);
    if (take) write(low + at, low + c);
    equal += total_equal;
    before += total;
  }
}

template <typename T, int D>
void means_launch(const Means& p, int touched, cudaStream_t stream) {
  const dim3 grid(static_cast<unsigned>(touched), static_cast<unsigned>(p.a.seqs), static_cast<unsigned>(p.a.kv_heads));
  if (p.scales != nullptr) launch(means_kernel<T, D, true>, grid, kMeanThreads, 0, 0, stream, p);
  else launch(means_kernel<T, D, false>, grid, kMeanThreads, 0, 0, stream, p);
}

template <typename T, int D>
void select_launch(const Select& p, int smem, cudaStream_t stream, int device) {
  static int configured[64] = {};
  int& have = configured[device & 63];
  if (smem > have) {
    RC_CUDA(cudaFuncSetAttribute(select_kernel<T, D>, cudaFuncAttributeMaxDynamicSharedMemorySize, smem));
    have = smem;
  }
  launch(select_kernel<T, D>, dim3(static_cast<unsigned>(static_cast<int64_t>(p.items) * p.a.kv_heads * p.cluster)), kSelectThreads, smem,
         p.cluster > 1 ? p.cluster : 0, stream, p);
}

// Checks means [pages, page_size / block, kv_heads, D] of one layer; returns the blocks of a page.
int64_t check_means(const at::Tensor& means, int64_t kv_heads, int64_t head_dim, at::ScalarType type, const at::Device& device) {
  RC_CHECK(means.device() == device && means.scalar_type() == type && means.dim() == 4 && means.size(1) >= 1 && means.size(2) == kv_heads &&
               means.size(3) == head_dim && means.stride(3) == 1 && means.size(0) < (1ll << 31),
           "means must be [pages, page_size / block, kv_heads, head_dim] with unit inner stride, of the rows' type (bf16 or fp16 for packed "
           "pages) and on their device");
  RC_CHECK(means.stride(0) % 8 == 0 && means.stride(1) % 8 == 0 && means.stride(2) % 8 == 0 && reinterpret_cast<uintptr_t>(means.data_ptr()) % 16 == 0,
           "means must have 16-byte aligned strides and base");
  return means.size(1);
}

}  // namespace paged

// Means of the blocks that hold the last new tokens of every sequence, over the tokens that they hold.
void paged_block_means(const at::Tensor& k_pages, const c10::optional<at::Tensor>& k_scales, const at::Tensor& means, const at::Tensor& table,
                       const at::Tensor& kv_lens, const at::Tensor& cu_q, int64_t max_q_len, const c10::optional<at::Tensor>& status) {
  check_cuda_tensor(k_pages, "k_pages");
  refuse_gradients({&k_pages, &means}, "block_means");
  refuse_tangents({&k_pages, &means}, "block_means");
  const at::ScalarType type = means.scalar_type();
  RC_CHECK(type == at::kBFloat16 || type == at::kHalf, "means are bf16 or fp16");
  RC_CHECK(k_pages.dim() == 4 && (k_pages.size(3) == 64 || k_pages.size(3) == 128), "pages must have a head_dim of 64 or 128");
  c10::cuda::CUDAGuard guard(k_pages.device());
  const int64_t heads = k_pages.size(2), d = k_pages.size(3);
  RC_CHECK(heads >= 1 && heads < 65536, "too many KV heads for one launch");
  paged::Means p{};
  const int64_t per_page = paged::check_means(means, heads, d, type, k_pages.device());
  at::assert_no_internal_overlap(means);
  if (k_scales.has_value()) {
    const paged::Packed k = paged::check_packed(k_pages, *k_scales, heads, d, k_pages.device(), "k_pages");
    p.page_stride = k.page_stride;
    p.token_stride = k.token_stride;
    p.head_stride = k.head_stride;
    p.scales = k.scales;
    p.scale_page = k.scale_page;
    p.scale_head = k.scale_head;
  } else {
    RC_CHECK(k_pages.scalar_type() == type, "means must have the type of the pages");
    const paged::Pages k = paged::check_pages(k_pages, heads, d, "k_pages");
    p.page_stride = k.page_stride * 2;
    p.token_stride = k.token_stride * 2;
    p.head_stride = k.head_stride * 2;
  }
  RC_CHECK(means.size(0) == k_pages.size(0) && k_pages.size(1) % per_page == 0 && (k_pages.size(1) / per_page) % 8 == 0,
           "means must be [pages, page_size / block, kv_heads, head_dim] with a block that is a multiple of 8 tokens");
  const paged::Table t = paged::check_table(table, kv_lens, cu_q, k_pages.device());
  RC_CHECK(max_q_len >= 1 && max_q_len < (1ll << 24), "max_q_len must be positive");
  RC_CHECK(t.seqs < 65536, "too many sequences for one launch");
  p.keys = static_cast<const uint8_t*>(k_pages.data_ptr());
  p.means = static_cast<char*>(means.data_ptr());
  p.mean_page = means.stride(0) * 2;
  p.mean_block = means.stride(1) * 2;
  p.mean_head = means.stride(2) * 2;
  p.block = static_cast<int>(k_pages.size(1) / per_page);
  paged::Args& a = p.a;
  a.table = t.table;
  a.kv_lens = t.kv_lens;
  a.cu_q = t.cu_q;
  a.seqs = t.seqs;
  a.width = t.width;
  a.table_row = t.row;
  a.pages = static_cast<int>(k_pages.size(0));
  a.kv_heads = static_cast<int>(heads);
  a.tokens = 0x7fffffff;
  a.max_q_len = static_cast<int>(max_q_len);
  a.tiling.page = static_cast<int>(k_pages.size(1));
  a.status = status_ptr(status);
  if (a.seqs == 0) return;
  const int64_t held = (static_cast<int64_t>(a.width) * a.tiling.page + p.block - 1) / p.block;
  const int touched = static_cast<int>(std::min<int64_t>(held, (max_q_len + p.block - 2) / p.block + 1));
  if (touched == 0) return;
  cudaStream_t stream = c10::cuda::getCurrentCUDAStream(k_pages.get_device()).stream();
  if (type == at::kHalf) d == 128 ? paged::means_launch<__half, 128>(p, touched, stream) : paged::means_launch<__half, 64>(p, touched, stream);
  else d == 128 ? paged::means_launch<__nv_bfloat16, 128>(p, touched, stream) : paged::means_launch<__nv_bfloat16, 64>(p, touched, stream);
  written(means);
}

// For every query block (`query_block` consecutive new tokens of a sequence) and KV head the blocks that it attends to, as a
// batch for attention over pages of `block` tokens: block table [items, kv_heads, width], kv_lens [items], cu_q [items + 1].
std::tuple<at::Tensor, at::Tensor, at::Tensor> paged_select_blocks(const at::Tensor& q, const at::Tensor& means, const at::Tensor& table,
                                                                   const at::Tensor& kv_lens, const at::Tensor& cu_q, int64_t block, int64_t keep,
                                                                   int64_t query_block, int64_t max_q_len, bool causal, int64_t sinks,
                                                                   int64_t recent, const c10::optional<at::Tensor>& status) {
  check_cuda_tensor(q, "q");
  refuse_gradients({&q, &means}, "the choice of blocks");
  refuse_tangents({&q, &means}, "the choice of blocks");
  const at::ScalarType type = q.scalar_type();
  RC_CHECK(type == at::kBFloat16 || type == at::kHalf, "the choice of blocks takes bf16 or fp16");
  RC_CHECK(q.dim() == 3 && (q.size(2) == 64 || q.size(2) == 128), "q must be [tokens, heads, head_dim] with head_dim 64 or 128");
  RC_CHECK(q.size(0) < (1ll << 31), "too many tokens for one launch");
  RC_CHECK(q.numel() == 0 || (q.stride(2) == 1 && q.stride(0) % 8 == 0 && q.stride(1) % 8 == 0 && reinterpret_cast<uintptr_t>(q.data_ptr()) % 16 == 0),
           "rows must have unit inner stride and 16-byte aligned strides and base");
  RC_CHECK(means.dim() == 4 && means.size(2) >= 1 && q.size(1) >= means.size(2) && q.size(1) % means.size(2) == 0,
           "heads must be a multiple of the KV heads");
  c10::cuda::CUDAGuard guard(q.device());
  const int64_t kv_heads = means.size(2), per_page = paged::check_means(means, kv_heads, q.size(2), type, q.device());
  const paged::Table t = paged::check_table(table, kv_lens, cu_q, q.device());
  RC_CHECK(block >= 8 && block % 8 == 0 && block * per_page <= 65536, "block must be a multiple of 8 tokens, and its pages at most 65536");
  RC_CHECK(keep >= 0 && keep < (1 << 24) && sinks >= 0 && sinks < (1ll << 31) && recent >= 0 && recent < (1ll << 31), "keep, sinks and recent must not be negative");
  RC_CHECK(query_block >= 1 && query_block < (1ll << 24) && max_q_len >= 1 && max_q_len < (1ll << 24), "query_block and max_q_len must be positive");
  const int64_t tokens = q.size(0), seqs = t.seqs, held = static_cast<int64_t>(t.width) * per_page;
  RC_CHECK(held <= paged::kMostBlocks, "a block table of " + std::to_string(held) + " blocks is wider than the choice can hold (" +
                                           std::to_string(paged::kMostBlocks) + "): take larger blocks");
  const int64_t longest = std::min(max_q_len, std::max<int64_t>(tokens, 1));
  int64_t items = query_block == 1 ? tokens : tokens / query_block + seqs;
  items = std::min(items, seqs * ((longest + query_block - 1) / query_block));
  const int64_t span = (causal ? std::min(query_block, longest) : longest) + recent;
  const int64_t width = std::min(held, (sinks + block - 1) / block + keep + (span + block - 2) / block + 1);
  const at::TensorOptions ints = q.options().dtype(at::kInt);
  at::Tensor out = at::empty({items, kv_heads, width}, ints), lens = at::empty({items}, ints), cu = at::empty({items + 1}, ints);
  if (items == 0) {
    cu.zero_();
    return {out, lens, cu};
  }
  RC_CHECK(items < (1 << 20) && items * kv_heads * 8 < (1ll << 31), "too many query blocks for one launch");
  paged::Select p{};
  paged::Args& a = p.a;
  a.q = q.data_ptr();
  a.q_token = q.stride(0);
  a.q_head = q.stride(1);
  a.table = t.table;
  a.kv_lens = t.kv_lens;
  a.cu_q = t.cu_q;
  a.seqs = t.seqs;
  a.width = t.width;
  a.table_row = t.row;
  a.pages = static_cast<int>(means.size(0));
  a.heads = static_cast<int>(q.size(1));
  a.kv_heads = static_cast<int>(kv_heads);
  a.group = a.heads / a.kv_heads;
  a.causal = causal;
  a.tokens = static_cast<int>(tokens);
  a.max_q_len = static_cast<int>(max_q_len);
  a.tiling.page = static_cast<int>(block * per_page);
  a.status = status_ptr(status);
  p.means = static_cast<const char*>(means.data_ptr());
  p.mean_page = means.stride(0) * 2;
  p.mean_block = means.stride(1) * 2;
  p.mean_head = means.stride(2) * 2;
  p.block = static_cast<int>(block);
  p.per_page = static_cast<int>(per_page);
  p.keep = static_cast<int>(keep);
  p.query_block = static_cast<int>(query_block);
  p.sinks = static_cast<int>(sinks);
  p.recent = static_cast<int>(recent);
  p.items = static_cast<int>(items);
  p.width = static_cast<int>(width);
  p.table = out.data_ptr<int>();
  p.kv_lens = lens.data_ptr<int>();
  p.cu_q = cu.data_ptr<int>();
  const int device = q.get_device();
  // CTAs of an item and KV head: as many as leave every SM one, and each enough blocks to be worth the cluster's meeting
  p.cluster = 1;
  while (p.cluster < 8 && items * kv_heads * p.cluster * 2 <= sm_count(device) && held >= 128 * p.cluster) p.cluster *= 2;
  const int64_t smem = static_cast<int64_t>(a.group) * q.size(2) * 8 + std::max<int64_t>(held, paged::kSelectThreads * 8) * 8;
  RC_CHECK(smem <= 220 * 1024, "too many heads in a group, or blocks in the table, for the choice of blocks");
  cudaStream_t stream = c10::cuda::getCurrentCUDAStream(device).stream();
  const int bytes = static_cast<int>(smem);
  if (type == at::kHalf) q.size(2) == 128 ? paged::select_launch<__half, 128>(p, bytes, stream, device) : paged::select_launch<__half, 64>(p, bytes, stream, device);
  else q.size(2) == 128 ? paged::select_launch<__nv_bfloat16, 128>(p, bytes, stream, device) : paged::select_launch<__nv_bfloat16, 64>(p, bytes, stream, device);
  return {out, lens, cu};
}

}  // namespace rc
