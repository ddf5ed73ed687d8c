// Sparse attention's choice over a paged cache, for sm_100a: means of the keys of blocks, and the blocks that each block of
// queries attends to.
//
// A block is `block` consecutive positions of a sequence (a divisor of the page size, so that it lies in one page); its mean is
// kept with its page, so sequences that share pages share means. Means are sums in FP64 divided once: the order of the sum does
// not show, whichever tokens came in which call.
//
// The score of a block for the queries of a KV head's group is max over the heads h of (sum over the tokens of the query block
// of q_h) . mean. Blocks at the border of the choice differ by little, so the choice is that of scores in FP64, where the order
// of a sum moves them by 2^-50 of their size: the same for every batch and form of the kernel. Equal scores go to the lower
// block. Few blocks need FP64. Scores come from the tensor core first, the pooled query (summed in FP32) as three 16-bit
// numbers that add up to it, a single token as itself. What they may be off by is summed next to them, as one more product:
// with x the pooled query, y the sum of the tokens' magnitudes and m the mean, 2^-18.5 sum |x| |m| for the products (16 channels at a
// time, a sum of 16 terms cut at 2^-23 of the largest: 2^-19; those added in FP32: 2^-21; the small numbers' with them 2^-22) and n
// 2^-24 sum y |m| for the FP32 sums of n terms one after the other. With T the keep-th largest score and E the largest bound, blocks above T + 2 E
// are chosen and blocks below T - 2 E are not; only where there is more than one way to choose from those between are they
// computed again, in FP64 (in a call of 128 query blocks and heads for a few of them).
//
// One CTA, or a cluster of them that splits the blocks, for every (query block, KV head): scores go to the shared memory of the
// cluster's first CTA, which finds the keep-th largest (a histogram between the smallest and the largest, then the bucket
// that holds it; digit by digit where that bucket holds many) and writes the chosen blocks in order.
//
// What bounds it: the latency of a chain of small steps for few sequences (a CTA with 64 candidates takes 10,000 cycles: looking up the
// sequence 1,100, the queries and means 1,400, products 1,900, the keep-th largest 2,200 are the longest), reading the means
// for many (an SM's share through L2 at 64 bytes a cycle). Measured (us): one token over 1,024 blocks and 8 KV heads 8.5; 40
// tokens over up to 512 blocks 15; 77 query blocks of 32 tokens over up to 500 blocks 30. In FP64 throughout: 27, 100 and 159.
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

constexpr int kMeanThreads = 256;

struct Means {
  Args a;                // table, lengths, pages; tokens, max_q_len
  const uint8_t* keys;   // rows of 16-bit numbers, or codes
  int64_t page_stride, token_stride, head_stride;  // bytes
  const uint8_t* scales;  // packed pages, or null
  int64_t scale_page, scale_head;
  char* means;           // [pages, page_size / block, kv_heads, D]: strides in bytes
  int64_t mean_page, mean_block, mean_head;
  Divider block, per_page;
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

__device__ __forceinline__ __nv_bfloat16 rounded(float x, __nv_bfloat16) { return __float2bfloat16_rn(x); }
__device__ __forceinline__ __half rounded(float x, __half) { return __float2half_rn(x); }

// Block (touched block, sequence, KV head): a thread sums eight channels of every (256 / lanes of a row)-th token.
template <typename T, int D, bool kPacked>
__global__ void __launch_bounds__(kMeanThreads) means_kernel(const __grid_constant__ Means p) {
  constexpr int kLanes = D / 8, kRowsAtOnce = kMeanThreads / kLanes;
  __shared__ double part[kMeanThreads / 32][D];
  let_later();
  after_earlier();
  const Args& a = p.a;
  const int s = blockIdx.y, head = blockIdx.z;
  if (blockIdx.x == 0 && head == 0 && threadIdx.x == 0) report_rows(a, s);
  int q_first;
  const int q_len = min(new_tokens(a, s, &q_first), a.max_q_len), kv_len = held_keys(a, s);
  if (q_len <= 0 || kv_len == 0) return;
  const int b = p.block.over(max(kv_len - q_len, 0)) + blockIdx.x;
  if (b >= p.block.up(kv_len)) return;
  const int rows = min(p.block.by, kv_len - b * p.block.by), slot = p.per_page.over(b), part_of = b - slot * p.per_page.by;
  const int row0 = part_of * p.block.by, page = a.table[s * a.table_row + slot];
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
  // the rows that a warp holds meet by shuffles, then the warps, a thread to each channel
#pragma unroll
  for (int o = kLanes; o < 32; o <<= 1)
#pragma unroll
    for (int e = 0; e < 8; ++e) sum[e] += __shfl_xor_sync(0xffffffffu, sum[e], o);
  if ((threadIdx.x & 31) < kLanes) {
#pragma unroll
    for (int e = 0; e < 8; ++e) part[threadIdx.x >> 5][vec * 8 + e] = sum[e];
  }
  __syncthreads();
  const int c = threadIdx.x;
  if (c >= D) return;
  double all = 0.0;
#pragma unroll
  for (int w = 0; w < kMeanThreads / 32; ++w) all += part[w][c];
  char* dst = p.means + page * p.mean_page + part_of * p.mean_block + head * p.mean_head;
  reinterpret_cast<T*>(dst)[c] = rounded(static_cast<float>(all / static_cast<double>(rows)), T());
}

// -- the choice -------------------------------------------------------------------------------------------------------

constexpr int kSelectThreads = 256;
constexpr int kSelectWarps = kSelectThreads / 32;
constexpr int kMostBlocks = 12288;  // of a table: what a thread marks of its candidates is two words
constexpr int kSelectBytes = 224 * 1024;  // of shared memory: 16 a block of the table, and 16 D + 260 a head of the group, about
constexpr float kProductError = 0x1.6p-19f;
constexpr int kBuckets = 256;       // one for each thread
constexpr int kPieces = 3;          // 16-bit numbers that add up to a pooled query; a fourth row holds what bounds its errors

struct Select {
  Args a;              // q, table, lengths, heads; causal; tokens, max_q_len
  const char* means;
  int64_t mean_page, mean_block, mean_head;
  Divider block, per_page, query_block, kv_heads;
  int keep, sinks, recent;
  int items, width;
  int* table;          // [items, kv_heads, width]
  int* kv_lens;        // [items]
  int* cu_q;           // [items + 1]
  int cluster, log_cluster;
};

// Shared memory of a CTA: pooled queries in FP64 [group][D] (for the border; at first the sums of a lone part), their pieces as
// the products' operand, scales of those, scores [blocks], the list of the blocks that are computed again, their keys in 64 bits.
template <int D>
struct SelectShape {
  static constexpr int piece_row = D * 2 + 64;  // bytes: rows 64 bytes apart in the banks
  int tiles;                                    // groups of eight heads
  int pieces_off, scale_off, score_off, list_off, exact_off, bytes;
  __host__ __device__ SelectShape(int group, int blocks) {
    tiles = (group + 7) / 8;
    pieces_off = group * D * 8;
    scale_off = pieces_off + tiles * 8 * (kPieces + 1) * piece_row;
    score_off = (scale_off + tiles * 8 * 4 + 15) / 16 * 16;
    list_off = score_off + (blocks + 3) / 4 * 16;
    exact_off = list_off + (blocks + 3) / 4 * 16;
    const int room = kSelectThreads * 64;  // where the parts of the pooled queries meet first
    const int most = exact_off + blocks * 8;
    bytes = most > score_off + room ? most : score_off + room;
  }
};

// Numbers that sort like scores (both zeros alike).
__device__ __forceinline__ uint64_t key_of(double score) {
  const uint64_t bits = static_cast<uint64_t>(__double_as_longlong(score + 0.0));
  return (bits >> 63) != 0 ? ~bits : bits | 0x8000000000000000ull;
}
__device__ __forceinline__ uint32_t key_of(float score) {
  const uint32_t bits = __float_as_uint(score + 0.0f);
  return (bits >> 31) != 0 ? ~bits : bits | 0x80000000u;
}

__device__ __forceinline__ void store_cluster(uint32_t addr, float v) {
  asm volatile("st.shared::cluster.f32 [%0], %1;" ::"r"(addr), "f"(v) : "memory");
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

// The `rest`-th largest of n keys, digit by digit from the top: its upper bits `prefix` above `shift` (0: all of it), and how many of
// the keys with that prefix are among the `rest` largest (`rest` comes out as that number).
template <typename Key, typename Get>
__device__ __forceinline__ void nth_largest(Get get, int n, Key& prefix, int& shift, int& rest, int* histogram, int* digit, int* sums) {
  constexpr int kBits = sizeof(Key) * 8;
  prefix = 0;
  shift = kBits;
  while (shift > 0) {
    histogram[threadIdx.x] = 0;
    __syncthreads();
    for (int c = threadIdx.x; c < n; c += kSelectThreads) {
      const Key key = get(c);
      if (shift == kBits || (key >> shift) == prefix) atomicAdd(&histogram[static_cast<int>((key >> (shift - 8)) & 255)], 1);
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
    prefix = (prefix << 8) | static_cast<Key>(d);
    shift -= 8;
    if (histogram[d] == rest) break;  // all of them
    __syncthreads();
  }
  __syncthreads();
}

// The keep-th largest of n scores between bottom and top (histogram: zeros). `list` takes a few of their places.
__device__ __forceinline__ float keep_th(const float* scores, int n, int keep, float top, float bottom, int* histogram, int* sums, int* digit,
                                         int* list) {
  if (top == bottom) return top;
  const int lane = threadIdx.x & 31;
  const float step = static_cast<float>(kBuckets) / (top - bottom);
  if (step > 0.0f && step < INFINITY && fabsf(bottom) < INFINITY) {  // (else: bounds that are no numbers, or a range that FP32 cannot cut)
    const auto bucket_of = [&](float x) { return min(kBuckets - 1, static_cast<int>((x - bottom) * step)); };  // grows with x
    if (threadIdx.x == 0) digit[2] = 0;
    for (int c = threadIdx.x; c < n; c += kSelectThreads) atomicAdd(&histogram[bucket_of(scores[c])], 1);
    __syncthreads();
    // every warp by itself: a lane sums eight buckets from the top
    constexpr int kPer = kBuckets / 32;
    int counts[kPer], sum = 0;
#pragma unroll
    for (int i = 0; i < kPer; ++i) sum += counts[i] = histogram[kBuckets - 1 - (lane * kPer + i)];
    int above = sum;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const int y = __shfl_up_sync(0xffffffffu, above, o);
      if (lane >= o) above += y;
    }
    above -= sum;
    int bucket = -1, members = 0, rest = 0;
#pragma unroll
    for (int i = 0; i < kPer; ++i) {
      if (above < keep && above + counts[i] >= keep) {
        bucket = kBuckets - 1 - (lane * kPer + i);
        members = counts[i];
        rest = keep - above;
      }
      above += counts[i];
    }
    const int holder = __ffs(__ballot_sync(0xffffffffu, bucket >= 0)) - 1;
    bucket = __shfl_sync(0xffffffffu, bucket, holder);
    members = __shfl_sync(0xffffffffu, members, holder);
    rest = __shfl_sync(0xffffffffu, rest, holder);
    if (members <= 32) {
      for (int c = threadIdx.x; c < n; c += kSelectThreads)
        if (bucket_of(scores[c]) == bucket) list[atomicAdd(&digit[2], 1)] = c;
      __syncthreads();
      // every warp by itself: a member's place among them (of equal ones each counts the others that come before it in the list)
      const float x = lane < members ? scores[list[lane]] : -INFINITY;
      int place = 0;
      for (int i = 0; i < members; ++i) {
        const float other = __shfl_sync(0xffffffffu, x, i);
        place += other > x || (other == x && i < lane);
      }
      const uint32_t who = __ballot_sync(0xffffffffu, lane < members && place == rest - 1);
      return __shfl_sync(0xffffffffu, x, __ffs(who) - 1);  // (the list is written again only after further barriers)
    }
  }
  uint32_t prefix;
  int shift, rest = keep;
  __syncthreads();
  nth_largest<uint32_t>([&](int c) { return key_of(scores[c]); }, n, prefix, shift, rest, histogram, digit, sums);
  // its digits end where all that share them are among the keep largest: the smallest of those
  const uint32_t border = shift == 0 ? prefix : prefix << shift;
  float least = INFINITY;
  for (int c = threadIdx.x; c < n; c += kSelectThreads)
    if (key_of(scores[c]) >= border) least = fminf(least, scores[c]);
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) least = fminf(least, __shfl_xor_sync(0xffffffffu, least, o));
  if (lane == 0) histogram[threadIdx.x >> 5] = __float_as_int(least);
  __syncthreads();
#pragma unroll
  for (int w = 0; w < kSelectWarps; ++w) least = fminf(least, __int_as_float(histogram[w]));
  __syncthreads();
  return least;
}

struct Operand {
  uint32_t x[4];
};

__device__ __forceinline__ float value_of(__nv_bfloat16 x) { return __bfloat162float(x); }
__device__ __forceinline__ float value_of(__half x) { return __half2float(x); }

// The 16-bit number nearest to x (bits), and x without it.
__device__ __forceinline__ uint32_t nearest(float& x, __nv_bfloat16) {
  const __nv_bfloat16 v = __float2bfloat16_rn(x);
  x -= __bfloat162float(v);
  return *reinterpret_cast<const uint16_t*>(&v);
}
__device__ __forceinline__ uint32_t nearest(float& x, __half) {
  const __half v = __float2half_rn(x);
  x -= __half2float(v);
  return *reinterpret_cast<const uint16_t*>(&v);
}

__device__ __forceinline__ void add_eight(float (&sum)[8], float (&size)[8], const uint4& u, __nv_bfloat16) {
  const uint32_t w[4] = {u.x, u.y, u.z, u.w};
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const float lo = __uint_as_float(w[i] << 16), hi = __uint_as_float(w[i] & 0xffff0000u);
    sum[2 * i] += lo;
    sum[2 * i + 1] += hi;
    size[2 * i] += fabsf(lo);
    size[2 * i + 1] += fabsf(hi);
  }
}
__device__ __forceinline__ void add_eight(float (&sum)[8], float (&size)[8], const uint4& u, __half) {
  const uint32_t w[4] = {u.x, u.y, u.z, u.w};
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const float2 f = __half22float2(*reinterpret_cast<const __half2*>(&w[i]));
    sum[2 * i] += f.x;
    sum[2 * i + 1] += f.y;
    size[2 * i] += fabsf(f.x);
    size[2 * i + 1] += fabsf(f.y);
  }
}

// Bits of a thread's candidates (words by constant index, so that they stay in registers).
template <int kWords>
__device__ __forceinline__ void mark(uint32_t (&words)[kWords], int i, bool set) {
#pragma unroll
  for (int w = 0; w < kWords; ++w)
    if (set && i >> 5 == w) words[w] |= 1u << (i & 31);
}
template <int kWords>
__device__ __forceinline__ bool marked(const uint32_t (&words)[kWords], int i) {
  uint32_t word = 0;
#pragma unroll
  for (int w = 0; w < kWords; ++w)
    if (i >> 5 == w) word = words[w];
  return (word >> (i & 31)) & 1;
}

template <typename T, int D>
__global__ void __launch_bounds__(kSelectThreads, 3) select_kernel(const __grid_constant__ Select p) {
  constexpr int kLanes = D / 8;  // vectors of eight channels
  extern __shared__ __align__(16) uint8_t smem[];
  __shared__ int found[5];  // sequence, its first item, its new tokens, the first of them, its keys
  __shared__ int sums[kSelectWarps];
  __shared__ int histogram[kBuckets];
  __shared__ int digit[3];
  __shared__ float bounds[3 * 8 * kSelectWarps];  // of every warp of the cluster: largest error, largest and smallest score
  const Args& a = p.a;
  const int index = static_cast<int>(blockIdx.x) >> p.log_cluster, rank = static_cast<int>(blockIdx.x) & (p.cluster - 1);
  const int item = p.kv_heads.over(index), head = index - item * a.kv_heads;
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const SelectShape<D> shape(a.group, a.width * p.per_page.by);
  double* pooled = reinterpret_cast<double*>(smem);  // (for the border)
  uint8_t* pieces = smem + shape.pieces_off;
  float* scales = reinterpret_cast<float*>(smem + shape.scale_off);  // [heads of the group, up to eights]
  float* scores = reinterpret_cast<float*>(smem + shape.score_off);
  int* list = reinterpret_cast<int*>(smem + shape.list_off);
  uint64_t* exact = reinterpret_cast<uint64_t*>(smem + shape.exact_off);
  let_later();
  after_earlier();

  // the item's sequence: items are counted sequence by sequence
  int items = 0;
  if (threadIdx.x == 0) found[0] = -1;
  for (int base = 0; base < a.seqs; base += kSelectThreads) {
    const int s = base + static_cast<int>(threadIdx.x);
    int n = 0, q_first = 0, q_len = 0, kv_len = 0;
    if (s < a.seqs) {
      q_len = min(new_tokens(a, s, &q_first), a.max_q_len);
      kv_len = held_keys(a, s);
      n = q_len > 0 ? p.query_block.up(q_len) : 0;
      if (index == 0 && rank == 0) report_rows(a, s);
    }
    int total;
    const int before = items + select_scan(n, sums, &total);
    if (item >= before && item < before + n) {
      found[0] = s;
      found[1] = before;
      found[2] = q_len;
      found[3] = q_first;
      found[4] = kv_len;
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
      const int end = min(max(a.cu_q[a.seqs], 0), a.tokens);
      p.kv_lens[item] = 0;
      p.cu_q[item] = end;
      if (item == p.items - 1) p.cu_q[p.items] = end;
    }
    return;
  }
  const int start = (item - found[1]) * p.query_block.by, q_len = found[2], count = min(p.query_block.by, q_len - start);
  const int q_first = found[3], kv_len = found[4];
  const int end = a.causal ? max(0, kv_len - q_len + start + count) : kv_len;
  const int blocks = p.block.up(end);
  const int near = static_cast<int>(max(static_cast<int64_t>(0), static_cast<int64_t>(kv_len) - q_len + (a.causal ? start : 0) - p.recent));
  const int high = min(blocks, p.block.over(near)), low = min(high, p.block.up(p.sinks));
  const int candidates = high - low, keep = min(p.keep, candidates);
  const int chosen = low + keep + blocks - high;
  if (writes) {
    p.kv_lens[item] = chosen > 0 ? (chosen - blocks) * p.block.by + end : 0;
    p.cu_q[item] = q_first + start;
    if (item == p.items - 1) p.cu_q[p.items] = q_first + start + count;
  }
  const int* table = a.table + s * a.table_row;
  const bool scored = keep > 0 && keep < candidates;  // else there is nothing to choose
  const int used = count == 1 ? 1 : kPieces;          // (a single token is its own first piece)
  const auto mean_at = [&](int b, int page) {
    return p.means + page * p.mean_page + (b - p.per_page.over(b) * p.per_page.by) * p.mean_block + head * p.mean_head;
  };

  // blocks in order: the first ones, the chosen, the last ones; what is not chosen is written while the rest waits for its loads
  const auto write = [&](int at, int b) {
    const int slot = p.per_page.over(b), page = table[slot];
    out[at] = page >= 0 && page < a.pages ? (page - slot) * p.per_page.by + b : -1;
  };
  if (rank == p.cluster - 1) {
    const int last = blocks - high;
    for (int i = kSelectThreads - 1 - static_cast<int>(threadIdx.x); i < p.width - keep; i += kSelectThreads) {
      if (i < low + last) write(i < low ? i : i + keep, i < low ? i : high + i - low);
      else out[i + keep] = -1;
    }
  }
  if (scored) {
    // This CTA's part of the candidates, sixteen to a warp: rows r0 and r0 + 8 of the operand, channels 32 j + 8 quad and on (any
    // order of channels gives the same sum), heads 2 quad and 2 quad + 1 of the result. The first ones are asked for before the queries.
    const int r0 = lane >> 2, quad = lane & 3;
    const int sixteens = (candidates + 15) / 16;
    const int from = ((sixteens * rank) >> p.log_cluster) * 16, to = min(candidates, ((sixteens * (rank + 1)) >> p.log_cluster) * 16);
    int page[2];
    uint4 mean[2][D / 32];
    const auto look_up = [&](int c0) {
#pragma unroll
      for (int i = 0; i < 2; ++i) page[i] = c0 + r0 + 8 * i < to ? table[p.per_page.over(low + c0 + r0 + 8 * i)] : -1;
    };
    const auto load = [&](int c0) {
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        const bool there = page[i] >= 0 && page[i] < a.pages;
        const char* src = there ? mean_at(low + c0 + r0 + 8 * i, page[i]) + quad * 16 : nullptr;
#pragma unroll
        for (int j = 0; j < D / 32; ++j) mean[i][j] = there ? *reinterpret_cast<const uint4*>(src + j * 64) : make_uint4(0, 0, 0, 0);
      }
    };
    look_up(from + warp * 16);

    // pooled queries: a thread sums eight channels of a head over a part of the tokens
    const int vecs = a.group * kLanes, splits = max(1, min(kSelectThreads / vecs, count));
    float2* parts = reinterpret_cast<float2*>(splits == 1 ? smem : smem + shape.score_off);  // [splits][head][channel]: sum, magnitudes
    for (int i = threadIdx.x; i < vecs * splits; i += kSelectThreads) {
      const int split = i / vecs, v = i - split * vecs, h = v / kLanes, vec = v - h * kLanes;
      const T* src = static_cast<const T*>(a.q) + static_cast<int64_t>(q_first + start) * a.q_token + (head * a.group + h) * a.q_head + vec * 8;
      if (used == 1) {
        const uint4 x = *reinterpret_cast<const uint4*>(src);
        uint8_t* to_piece = pieces + h * (kPieces + 1) * SelectShape<D>::piece_row + vec * 16;
        *reinterpret_cast<uint4*>(to_piece) = x;
        *reinterpret_cast<uint4*>(to_piece + kPieces * SelectShape<D>::piece_row) =
            make_uint4(x.x & 0x7fff7fffu, x.y & 0x7fff7fffu, x.z & 0x7fff7fffu, x.w & 0x7fff7fffu);
        if (vec == 0) scales[h] = 1.0f;
      } else {
        float sum[8] = {}, size[8] = {};
#pragma unroll 4
        for (int t = split; t < count; t += splits) add_eight(sum, size, *reinterpret_cast<const uint4*>(src + t * a.q_token), T());
#pragma unroll
        for (int e = 0; e < 8; e += 2)
          *reinterpret_cast<float4*>(parts + i * 8 + e) = make_float4(sum[e], size[e], sum[e + 1], size[e + 1]);
      }
    }
    load(from + warp * 16);
    if (used > 1) {
      __syncthreads();
      // their pieces, a warp a head; fp16's are of a multiple by a power of two that brings the bounds' largest between 2^13 and
      // 2^14: what the last piece cannot hold is below 2^-25, with 128 means of 2^16 at most 0.25
      const float steps = static_cast<float>(count / splits + 1 + splits) * (0x1p-24f / kProductError);  // of the sums in FP32, over that of the products
      for (int h = warp; h < a.group; h += kSelectWarps) {
        constexpr int kPer = D / 32;
        float x[kPer], y[kPer], top = 0.0f;
#pragma unroll
        for (int e = 0; e < kPer; ++e) {
          float2 f = make_float2(0.0f, 0.0f);
          for (int k = 0; k < splits; ++k) {
            const float2 add = parts[k * vecs * 8 + h * D + lane * kPer + e];
            f.x += add.x;
            f.y += add.y;
          }
          x[e] = f.x;
          y[e] = fmaf(f.y, steps, fabsf(f.x)) * 1.01f;  // (and its own rounding to 16 bits)
          top = fmaxf(top, y[e]);
        }
        float down = 1.0f;
        if (std::is_same<T, __half>::value) {
          const int power = max(static_cast<int>(__reduce_max_sync(0xffffffffu, __float_as_uint(top)) >> 23) - 127, -100);
          const float up = __uint_as_float(static_cast<uint32_t>(127 + 13 - power) << 23);
          down = __uint_as_float(static_cast<uint32_t>(min(127 - 13 + power, 254)) << 23);
#pragma unroll
          for (int e = 0; e < kPer; ++e) {
            x[e] *= up;
            y[e] *= up;
          }
        }
        if (lane == 0) scales[h] = down;
#pragma unroll
        for (int k = 0; k <= kPieces; ++k)
#pragma unroll
          for (int e = 0; e < kPer; e += 2) {
            const uint32_t lower = nearest(k < kPieces ? x[e] : y[e], T()), upper = nearest(k < kPieces ? x[e + 1] : y[e + 1], T());
            *reinterpret_cast<uint32_t*>(pieces + (h * (kPieces + 1) + k) * SelectShape<D>::piece_row + (lane * kPer + e) * 2) = lower | upper << 16;
          }
      }
    }
    for (int i = threadIdx.x; i < kBuckets; i += kSelectThreads) histogram[i] = 0;
    if (p.cluster > 1) cluster_sync_all();  // (the first CTA's parts have been read: others may write their scores there)
    else __syncthreads();

    const uint32_t scores_at = cluster_addr(scores, 0);
    float most = 0.0f, top = -INFINITY, bottom = INFINITY;
    for (int c0 = from + warp * 16; c0 < to; c0 += kSelectWarps * 16) {
      look_up(c0 + kSelectWarps * 16);
      float best[2] = {-INFINITY, -INFINITY};
      for (int tile = 0; tile < shape.tiles; ++tile) {
        const uint8_t* piece = pieces + ((tile * 8 + r0) * (kPieces + 1)) * SelectShape<D>::piece_row + quad * 16;
        // the products of 16 channels by themselves, added in FP32: a sum over all of them would be cut at each step
        float sc[4] = {}, size[4] = {};
        for (int k = used - 1; k > 0; --k) {
#pragma unroll
          for (int j = 0; j < D / 32; ++j) {
            const uint4 b = *reinterpret_cast<const uint4*>(piece + k * SelectShape<D>::piece_row + j * 64);
            mma_16816(sc, Operand{mean[0][j].x, mean[1][j].x, mean[0][j].y, mean[1][j].y}.x, b.x, b.y, T());
            mma_16816(sc, Operand{mean[0][j].z, mean[1][j].z, mean[0][j].w, mean[1][j].w}.x, b.z, b.w, T());
          }
        }
#pragma unroll
        for (int j = 0; j < D / 32; ++j) {
          constexpr uint32_t kSize = 0x7fff7fffu;
          const uint4 b = *reinterpret_cast<const uint4*>(piece + j * 64), y = *reinterpret_cast<const uint4*>(piece + kPieces * SelectShape<D>::piece_row + j * 64);
          float one[4] = {}, two[4] = {};
          mma_16816(one, Operand{mean[0][j].x, mean[1][j].x, mean[0][j].y, mean[1][j].y}.x, b.x, b.y, T());
          mma_16816(two, Operand{mean[0][j].z, mean[1][j].z, mean[0][j].w, mean[1][j].w}.x, b.z, b.w, T());
          mma_16816(size, Operand{mean[0][j].x & kSize, mean[1][j].x & kSize, mean[0][j].y & kSize, mean[1][j].y & kSize}.x, y.x, y.y, T());
          mma_16816(size, Operand{mean[0][j].z & kSize, mean[1][j].z & kSize, mean[0][j].w & kSize, mean[1][j].w & kSize}.x, y.z, y.w, T());
#pragma unroll
          for (int e = 0; e < 4; ++e) sc[e] += one[e] + two[e];
        }
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          const int h = tile * 8 + 2 * quad + (e & 1);
          if (h >= a.group) continue;
          const float x = sc[e] * scales[h];
          best[e >> 1] = fmaxf(best[e >> 1], x);
          // (a bound or score that is no number makes every block one that is computed again)
          const float bound = fmaf(size[e], kProductError * 1.02f, std::is_same<T, __half>::value && used > 1 ? 0.25f : 0.0f) * scales[h];
          most = bound < INFINITY && fabsf(x) < INFINITY ? fmaxf(most, bound) : INFINITY;
        }
      }
      load(c0 + kSelectWarps * 16);
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        best[i] = fmaxf(best[i], __shfl_xor_sync(0xffffffffu, best[i], 1));
        best[i] = fmaxf(best[i], __shfl_xor_sync(0xffffffffu, best[i], 2));
        const int c = c0 + r0 + 8 * i;
        if (c < to) {
          top = fmaxf(top, best[i]);
          bottom = fminf(bottom, best[i]);
          if (quad == 0) store_cluster(scores_at + c * 4, best[i]);
        }
      }
    }
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) {
      most = fmaxf(most, __shfl_xor_sync(0xffffffffu, most, o));
      top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, o));
      bottom = fminf(bottom, __shfl_xor_sync(0xffffffffu, bottom, o));
    }
    if (lane == 0) {
      const uint32_t at = cluster_addr(&bounds[3 * (rank * kSelectWarps + warp)], 0);
      store_cluster(at, most);
      store_cluster(at + 4, top);
      store_cluster(at + 8, bottom);
    }
  }
  if (p.cluster > 1) cluster_sync_all();
  else __syncthreads();
  if (rank != 0) return;

  if (!scored) {
    for (int i = threadIdx.x; i < keep; i += kSelectThreads) write(low + i, low + i);
    return;
  }
  float spread = 0.0f, top = -INFINITY, bottom = INFINITY;  // 2 E, and the scores' range
  for (int i = lane; i < p.cluster * kSelectWarps; i += 32) {
    spread = fmaxf(spread, 2.0f * bounds[3 * i]);
    top = fmaxf(top, bounds[3 * i + 1]);
    bottom = fminf(bottom, bounds[3 * i + 2]);
  }
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) {
    spread = fmaxf(spread, __shfl_xor_sync(0xffffffffu, spread, o));
    top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, o));
    bottom = fminf(bottom, __shfl_xor_sync(0xffffffffu, bottom, o));
  }
  const float least = keep_th(scores, candidates, keep, top, bottom, histogram, sums, digit, list);
  const float sure = least + spread, out_of = least - spread;

  // a thread looks at `per` neighbouring candidates, so that one prefix sum puts what it finds in order
  const int per = (candidates + kSelectThreads - 1) / kSelectThreads;
  const int mine = min(candidates, static_cast<int>(threadIdx.x) * per), past = min(candidates, mine + per);
  int counts = 0;  // those above, and times 2^16 those between
  for (int c = mine; c < past; ++c) counts += scores[c] > sure ? 1 : scores[c] < out_of ? 0 : 1 << 16;
  int total;
  const int before = select_scan(counts, sums, &total);
  const int above = total & 0xffff, doubtful = total >> 16;
  int at = (before & 0xffff) + (before >> 16);
  if (doubtful <= keep - above) {
    for (int c = mine; c < past; ++c)
      if (!(scores[c] < out_of)) write(low + at++, low + c);
    return;
  }

  // ---------------- the border in FP64 ----------------
  {
    int place = before >> 16;
    for (int c = mine; c < past; ++c)
      if (!(scores[c] > sure) && !(scores[c] < out_of)) list[place++] = c;
  }
  // pooled queries in FP64: a warp takes every eighth group of tokens, a lane eight channels; the warps meet where the pieces were
  double* meet = reinterpret_cast<double*>(pieces);  // [warps][D]
  for (int h = 0; h < a.group; ++h) {
    double sum[8] = {};
    const int vec = lane % kLanes;
    const T* src = static_cast<const T*>(a.q) + static_cast<int64_t>(q_first + start) * a.q_token + (head * a.group + h) * a.q_head + vec * 8;
#pragma unroll 4
    for (int t = warp * (32 / kLanes) + lane / kLanes; t < count; t += kSelectWarps * (32 / kLanes))
      add_eight(sum, *reinterpret_cast<const uint4*>(src + t * a.q_token), T());
#pragma unroll
    for (int o = kLanes; o < 32; o <<= 1)
#pragma unroll
      for (int e = 0; e < 8; ++e) sum[e] += __shfl_xor_sync(0xffffffffu, sum[e], o);
    __syncthreads();  // the last head's have been read
    if (lane < kLanes)
#pragma unroll
      for (int e = 0; e < 8; ++e) meet[warp * D + vec * 8 + e] = sum[e];
    __syncthreads();
    for (int i = threadIdx.x; i < D; i += kSelectThreads) {
      double all = 0.0;
      for (int w = 0; w < min(kSelectWarps, count); ++w) all += meet[w * D + i];
      pooled[h * D + i] = all;
    }
  }
  __syncthreads();
  for (int i = warp; i < doubtful; i += kSelectWarps) {
    const int b = low + list[i], page = table[p.per_page.over(b)];
    constexpr int kPer = D / 32;
    double x[kPer] = {};
    if (page >= 0 && page < a.pages) {
      const T* src = reinterpret_cast<const T*>(mean_at(b, page)) + lane * kPer;
#pragma unroll
      for (int e = 0; e < kPer; ++e) x[e] = static_cast<double>(value_of(src[e]));
    }
    double best = -INFINITY;
    for (int h = 0; h < a.group; ++h) {
      double dot = 0.0;
#pragma unroll
      for (int e = 0; e < kPer; ++e) dot = fma(pooled[h * D + lane * kPer + e], x[e], dot);
#pragma unroll
      for (int o = 16; o > 0; o >>= 1) dot += __shfl_xor_sync(0xffffffffu, dot, o);
      best = fmax(best, dot);  // (NaN counts for nothing)
    }
    if (lane == 0) exact[i] = key_of(best);
  }
  __syncthreads();
  int rest = keep - above, number = 0;
  uint32_t taken[(kMostBlocks / kSelectThreads + 31) / 32] = {};  // of this thread's candidates
  int place = before >> 16;
  if (doubtful <= 32) {
    // every warp by itself: a member's place among them, equal ones in their order
    const uint64_t key = lane < doubtful ? exact[lane] : 0;
    int rank_of = 0;
    for (int i = 0; i < doubtful; ++i) {
      const uint64_t other = __shfl_sync(0xffffffffu, key, i);
      rank_of += other > key || (other == key && i < lane);
    }
    const uint32_t best = __ballot_sync(0xffffffffu, lane < doubtful && rank_of < rest);
    for (int c = mine; c < past; ++c) {
      bool take = scores[c] > sure;
      if (!take && !(scores[c] < out_of)) take = (best >> place++) & 1;
      mark(taken, c - mine, take);
      number += take;
    }
  } else {
    uint64_t prefix;
    int shift, equals = 0;
    nth_largest<uint64_t>([&](int i) { return exact[i]; }, doubtful, prefix, shift, rest, histogram, digit, sums);
    // those above the rest-th largest, and of its equals the first `rest`
    for (int c = mine; c < past; ++c)
      if (!(scores[c] > sure) && !(scores[c] < out_of)) equals += (exact[place++] >> shift) == prefix;
    int equal = select_scan(equals, sums, &total);
    place = before >> 16;
    for (int c = mine; c < past; ++c) {
      bool take = scores[c] > sure;
      if (!take && !(scores[c] < out_of)) {
        const uint64_t digits = exact[place++] >> shift;
        take = digits > prefix || (digits == prefix && equal++ < rest);
      }
      mark(taken, c - mine, take);
      number += take;
    }
  }
  at = select_scan(number, sums, &total);
  for (int c = mine; c < past; ++c)
    if (marked(taken, c - mine)) write(low + at++, low + c);
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
  if (k_scales.has_value()) {
    refuse_gradients({&*k_scales}, "block_means");
    refuse_tangents({&*k_scales}, "block_means");
  }
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
  p.block = paged::Divider::of(static_cast<int>(k_pages.size(1) / per_page));
  p.per_page = paged::Divider::of(static_cast<int>(per_page));
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
  const int64_t held = static_cast<int64_t>(a.width) * per_page;
  const int touched = static_cast<int>(std::min<int64_t>(held, (max_q_len + p.block.by - 2) / p.block.by + 1));
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
  // one allocation for the three of them
  at::Tensor room = paged::new_tensor({items * (kv_heads * width + 2) + 1}, q, at::kInt);
  const auto part = [&](int64_t offset, at::IntArrayRef sizes) {
    at::Tensor t = at::detail::make_tensor<c10::TensorImpl>(c10::Storage(room.storage()), room.key_set(), room.dtype());
    t.unsafeGetTensorImpl()->set_storage_offset(offset);
    t.unsafeGetTensorImpl()->set_sizes_contiguous(sizes);
    return t;
  };
  at::Tensor out = part(0, {items, kv_heads, width}), lens = part(items * kv_heads * width, {items}),
             cu = part(items * (kv_heads * width + 1), {items + 1});
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
  p.block = paged::Divider::of(static_cast<int>(block));
  p.per_page = paged::Divider::of(static_cast<int>(per_page));
  p.query_block = paged::Divider::of(static_cast<int>(query_block));
  p.kv_heads = paged::Divider::of(static_cast<int>(kv_heads));
  p.keep = static_cast<int>(keep);
  p.sinks = static_cast<int>(sinks);
  p.recent = static_cast<int>(recent);
  p.items = static_cast<int>(items);
  p.width = static_cast<int>(width);
  p.table = out.data_ptr<int>();
  p.kv_lens = lens.data_ptr<int>();
  p.cu_q = cu.data_ptr<int>();
  const int device = q.get_device();
  RC_CHECK(a.group <= 256, "too many heads in a group for the choice of blocks");  // (more never fit, and their bytes could wrap)
  const int smem = q.size(2) == 128 ? paged::SelectShape<128>(a.group, static_cast<int>(held)).bytes : paged::SelectShape<64>(a.group, static_cast<int>(held)).bytes;
  RC_CHECK(smem <= paged::kSelectBytes, "a group of " + std::to_string(a.group) + " heads with a block table of " + std::to_string(held) + " blocks needs " +
                                            std::to_string(smem) + " bytes of shared memory for the choice of blocks, of which there are " +
                                            std::to_string(paged::kSelectBytes) + ": take larger blocks, or fewer heads at a time");
  // CTAs of an item and KV head: as many as find room at once (up to three on an SM), with 128 blocks each
  const int resident = std::max(1, std::min(3, paged::kSelectBytes / smem));
  p.cluster = 1;
  while (p.cluster < 8 && items * kv_heads * p.cluster * 2 <= static_cast<int64_t>(resident) * sm_count(device) && held > 128 * p.cluster) {
    p.cluster *= 2;
    ++p.log_cluster;
  }
  cudaStream_t stream = c10::cuda::getCurrentCUDAStream(device).stream();
  if (type == at::kHalf) q.size(2) == 128 ? paged::select_launch<__half, 128>(p, smem, stream, device) : paged::select_launch<__half, 64>(p, smem, stream, device);
  else q.size(2) == 128 ? paged::select_launch<__nv_bfloat16, 128>(p, smem, stream, device) : paged::select_launch<__nv_bfloat16, 64>(p, smem, stream, device);
  return {out, lens, cu};
}

}  // namespace rc
