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
// block. Few blocks need FP64: scores come from the tensor core first (the pooled query as the sum of three 16-bit numbers, one for
// single tokens), together with the sum of their products' magnitudes, which bounds their error (2^-15 of it: 24 steps at most, each a sum
// of 17 terms cut at 2^-24 of the largest). With T the keep-th largest and E the largest bound, blocks above T + 2 E are chosen and blocks below T - 2 E are not;
// only the blocks between, where there is more than one way to choose from them, are computed again.
//
// One CTA, or a cluster of them that splits the blocks, for every (query block, KV head): scores as 32-bit keys that sort
// like them in the shared memory of the cluster's first CTA, which finds the keep-th largest by digits of eight bits (a
// histogram each, until a digit's candidates are all taken) and writes the chosen blocks in order.
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
constexpr int kMostBlocks = 12288;  // whose keys fit one CTA's shared memory
constexpr int kPieces = 3;          // 16-bit numbers that add up to a pooled query

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

// Shared memory of a CTA: pooled queries in FP64 [group][D], their pieces as the products' operand, scales of those, then the
// keys [blocks] (64 bits), of whose room the first half holds the 32-bit scores and the second half the list of blocks that
// are computed again... in that order: scores, list, exact keys.
template <int D>
struct SelectShape {
  static constexpr int piece_row = D * 2 + 64;  // bytes: rows 64 bytes apart in the banks
  int tiles;                                    // groups of eight heads
  int pieces_off, scale_off, score_off, list_off, exact_off, bytes;
  __host__ __device__ SelectShape(int group, int blocks) {
    tiles = (group + 7) / 8;
    pieces_off = group * D * 8;
    scale_off = pieces_off + tiles * 8 * kPieces * piece_row;
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
    for (int i = threadIdx.x; i < 256; i += kSelectThreads) histogram[i] = 0;
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

__device__ __forceinline__ void mma_means(float (&d)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1, __nv_bfloat16) {
  asm volatile(
      "mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
      : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
      : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
__device__ __forceinline__ void mma_means(float (&d)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1, __half) {
  asm volatile(
      "mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
      : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
      : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}

// The 16-bit number nearest to x (bits), and what it stands for.
__device__ __forceinline__ uint32_t nearest(double x, double* stands, __nv_bfloat16) {
  const __nv_bfloat16 v = __float2bfloat16_rn(static_cast<float>(x));
  *stands = static_cast<double>(__bfloat162float(v));
  return *reinterpret_cast<const uint16_t*>(&v);
}
__device__ __forceinline__ uint32_t nearest(double x, double* stands, __half) {
  const __half v = __float2half_rn(static_cast<float>(x));
  *stands = static_cast<double>(__half2float(v));
  return *reinterpret_cast<const uint16_t*>(&v);
}

template <typename T, int D>
__global__ void __launch_bounds__(kSelectThreads, 2) select_kernel(const __grid_constant__ Select p) {
  constexpr int kLanes = D / 8;  // vectors of eight channels
  extern __shared__ __align__(16) uint8_t smem[];
  __shared__ int found[4];  // sequence, its first item, its new tokens
  __shared__ int sums[kSelectWarps];
  __shared__ int histogram[256];
  __shared__ int digit[2];
  __shared__ float bounds[8 * kSelectWarps];  // of every warp of the cluster
  const Args& a = p.a;
  const int index = static_cast<int>(blockIdx.x) / p.cluster, rank = static_cast<int>(blockIdx.x) - index * p.cluster;
  const int item = index / a.kv_heads, head = index - item * a.kv_heads;
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const SelectShape<D> shape(a.group, a.width * p.per_page);
  double* pooled = reinterpret_cast<double*>(smem);
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
      const int end = min(max(a.cu_q[a.seqs], 0), a.tokens);
      p.kv_lens[item] = 0;
      p.cu_q[item] = end;
      if (item == p.items - 1) p.cu_q[p.items] = end;
    }
    return;
  }
  const int start = (item - found[1]) * p.query_block, q_len = found[2], count = min(p.query_block, q_len - start);
  const int kv_len = held_keys(a, s), q_first = a.cu_q[s];
  const int end = a.causal ? max(0, kv_len - q_len + start + count) : kv_len;
  const int blocks = (end + p.block - 1) / p.block;
  const int64_t near = max(static_cast<int64_t>(0), static_cast<int64_t>(kv_len) - q_len + (a.causal ? start : 0) - p.recent);
  const int high = min(blocks, static_cast<int>(near / p.block)), low = min(high, p.sinks / p.block + (p.sinks % p.block > 0));
  const int candidates = high - low, keep = min(p.keep, candidates);
  const int chosen = low + keep + blocks - high;
  if (writes) {
    p.kv_lens[item] = chosen > 0 ? (chosen - 1) * p.block + end - (blocks - 1) * p.block : 0;
    p.cu_q[item] = q_first + start;
    if (item == p.items - 1) p.cu_q[p.items] = q_first + start + count;
  }
  const int* table = a.table + s * a.table_row;
  const bool scored = keep > 0 && keep < candidates;  // else there is nothing to choose
  const int used = count == 1 ? 1 : kPieces;          // (a single token is its own first piece)
  const auto mean_at = [&](int b, int page) {
    return p.means + page * p.mean_page + (b % p.per_page) * p.mean_block + head * p.mean_head;
  };

  if (scored) {
    // pooled queries: a thread sums eight channels of a head over a part of the tokens; the parts meet where the scores will be
    double* parts = reinterpret_cast<double*>(scores);
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
      __syncthreads();
    }
    // their pieces, a warp a head; fp16's are of a multiple by a power of two whose largest magnitude lies between 2^13 and 2^14: what
    // the last piece cannot hold is below 2^-25, with 128 means of 2^16 at most 0.25
    for (int h = warp; h < shape.tiles * 8; h += kSelectWarps) {
      constexpr int kPer = D / 32;
      double x[kPer];
      float top = 0.0f;
#pragma unroll
      for (int e = 0; e < kPer; ++e) {
        x[e] = h < a.group ? pooled[h * D + lane * kPer + e] : 0.0;
        top = fmaxf(top, fabsf(static_cast<float>(x[e])));
      }
      float down = 1.0f;
      if (std::is_same<T, __half>::value && used > 1) {
        const int power = max(static_cast<int>(__reduce_max_sync(0xffffffffu, __float_as_uint(top)) >> 23) - 127, -100);
        const double up = __longlong_as_double(static_cast<long long>(1023 + 13 - power) << 52);
        down = __uint_as_float(static_cast<uint32_t>(min(127 - 13 + power, 254)) << 23);
#pragma unroll
        for (int e = 0; e < kPer; ++e) x[e] *= up;
      }
      if (lane == 0) scales[h] = down;
#pragma unroll
      for (int k = 0; k < kPieces; ++k)
#pragma unroll
        for (int e = 0; e < kPer; e += 2) {
          double stands[2];
          const uint32_t lower = nearest(x[e], &stands[0], T()), upper = nearest(x[e + 1], &stands[1], T());
          *reinterpret_cast<uint32_t*>(pieces + (h * kPieces + k) * SelectShape<D>::piece_row + (lane * kPer + e) * 2) = lower | upper << 16;
          x[e] -= stands[0];
          x[e + 1] -= stands[1];
        }
    }
    if (p.cluster > 1) cluster_sync_all();  // (the first CTA's parts have been read: others may write their scores there)
    else __syncthreads();

    // scores of this CTA's part of the candidates, sixteen to a warp: rows r0 and r0 + 8 of the operand, channels 32 j + 8 quad
    // and on (any order of channels gives the same sum), heads 2 quad and 2 quad + 1 of the result
    const int r0 = lane >> 2, quad = lane & 3;
    const uint32_t scores_at = cluster_addr(scores, 0);
    const int sixteens = (candidates + 15) / 16;
    const int from = static_cast<int>(static_cast<int64_t>(sixteens) * rank / p.cluster) * 16;
    const int to = min(candidates, static_cast<int>(static_cast<int64_t>(sixteens) * (rank + 1) / p.cluster) * 16);
    float most = 0.0f;
    const auto page_of = [&](int c) { return c < to ? table[(low + c) / p.per_page] : -1; };
    int page[2] = {page_of(from + warp * 16 + r0), page_of(from + warp * 16 + r0 + 8)};
    for (int c0 = from + warp * 16; c0 < to; c0 += kSelectWarps * 16) {
      uint4 mean[2][D / 32];
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        const bool there = page[i] >= 0 && page[i] < a.pages;
        const char* src = there ? mean_at(low + c0 + r0 + 8 * i, page[i]) + quad * 16 : nullptr;
#pragma unroll
        for (int j = 0; j < D / 32; ++j) mean[i][j] = there ? *reinterpret_cast<const uint4*>(src + j * 64) : make_uint4(0, 0, 0, 0);
        page[i] = page_of(c0 + kSelectWarps * 16 + r0 + 8 * i);
      }
      float best[2] = {-INFINITY, -INFINITY};
      for (int tile = 0; tile < shape.tiles; ++tile) {
        const uint8_t* piece = pieces + ((tile * 8 + r0) * kPieces) * SelectShape<D>::piece_row + quad * 16;
        float sc[4] = {}, size[4] = {};
#pragma unroll
        for (int j = 0; j < D / 32; ++j) {
          const uint32_t m0[4] = {mean[0][j].x, mean[0][j].y, mean[0][j].z, mean[0][j].w};
          const uint32_t m1[4] = {mean[1][j].x, mean[1][j].y, mean[1][j].z, mean[1][j].w};
          for (int k = 0; k < used; ++k) {
            const uint4 b = *reinterpret_cast<const uint4*>(piece + k * SelectShape<D>::piece_row + j * 64);
            const uint32_t q[4] = {b.x, b.y, b.z, b.w};
#pragma unroll
            for (int h = 0; h < 4; h += 2) {
              const uint32_t x[4] = {m0[h], m1[h], m0[h + 1], m1[h + 1]};
              mma_means(sc, x, q[h], q[h + 1], T());
              if (k > 0) continue;
              const uint32_t y[4] = {x[0] & 0x7fff7fffu, x[1] & 0x7fff7fffu, x[2] & 0x7fff7fffu, x[3] & 0x7fff7fffu};
              mma_means(size, y, q[h] & 0x7fff7fffu, q[h + 1] & 0x7fff7fffu, T());
            }
          }
        }
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          const int h = tile * 8 + 2 * quad + (e & 1);
          if (h >= a.group) continue;
          const float x = sc[e] * scales[h];
          best[e >> 1] = fmaxf(best[e >> 1], x);
          // (a bound or score that is no number makes every block one that is computed again)
          const float bound = fmaf(size[e], 0x1p-15f, std::is_same<T, __half>::value && used > 1 ? 0.25f : 0.0f) * scales[h];
          most = bound < INFINITY && fabsf(x) < INFINITY ? fmaxf(most, bound) : INFINITY;
        }
      }
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        best[i] = fmaxf(best[i], __shfl_xor_sync(0xffffffffu, best[i], 1));
        best[i] = fmaxf(best[i], __shfl_xor_sync(0xffffffffu, best[i], 2));
        const int c = c0 + r0 + 8 * i;
        if (quad == 0 && c < to) store_cluster(scores_at + c * 4, best[i]);
      }
    }
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) most = fmaxf(most, __shfl_xor_sync(0xffffffffu, most, o));
    if (lane == 0) store_cluster(cluster_addr(&bounds[rank * kSelectWarps + warp], 0), most);
  }
  if (p.cluster > 1) cluster_sync_all();
  else __syncthreads();
  if (rank != 0) return;

  // blocks in order: the first ones, the chosen, the last ones
  const auto write = [&](int at, int b) {
    const int page = table[b / p.per_page];
    out[at] = page >= 0 && page < a.pages ? page * p.per_page + b % p.per_page : -1;
  };
  for (int i = threadIdx.x; i < low; i += kSelectThreads) write(i, i);
  for (int i = threadIdx.x; i < blocks - high; i += kSelectThreads) write(low + keep + i, high + i);
  for (int i = chosen + static_cast<int>(threadIdx.x); i < p.width; i += kSelectThreads) out[i] = -1;
  if (!scored) {
    for (int i = threadIdx.x; i < keep; i += kSelectThreads) write(low + i, low + i);
    return;
  }
  float spread = 0.0f;  // 2 E
  for (int i = 0; i < p.cluster * kSelectWarps; ++i) spread = fmaxf(spread, 2.0f * bounds[i]);

  // T: the smallest score that has the keep-th largest's digits
  uint32_t prefix;
  int shift, rest = keep;
  nth_largest<uint32_t>([&](int c) { return key_of(scores[c]); }, candidates, prefix, shift, rest, histogram, digit, sums);
  const uint32_t border_key = shift == 0 ? prefix : prefix << shift;
  // (its digits end where all that share them are taken: the smallest of those is T)
  float least = INFINITY;
  for (int c = threadIdx.x; c < candidates; c += kSelectThreads)
    if (key_of(scores[c]) >= border_key) least = fminf(least, scores[c]);
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) least = fminf(least, __shfl_xor_sync(0xffffffffu, least, o));
  if (lane == 0) bounds[warp] = least;
  __syncthreads();
#pragma unroll
  for (int w = 0; w < kSelectWarps; ++w) least = fminf(least, bounds[w]);
  const float sure = least + spread, out_of = least - spread;

  // the blocks between, in order
  int doubtful = 0, above = 0;
  for (int c0 = 0; c0 < candidates; c0 += kSelectThreads) {
    const int c = c0 + static_cast<int>(threadIdx.x);
    const bool in = c < candidates && scores[c] > sure, between = c < candidates && !in && !(scores[c] < out_of);
    int total;
    const int packed = select_scan((in ? 1 << 16 : 0) | (between ? 1 : 0), sums, &total);
    if (between) list[doubtful + (packed & 0xffff)] = c;
    doubtful += total & 0xffff;
    above += total >> 16;
  }
  __syncthreads();
  rest = keep - above;
  uint64_t prefix64 = 0;
  int shift64 = 64;
  if (doubtful > rest) {
    for (int i = warp; i < doubtful; i += kSelectWarps) {
      const int b = low + list[i], at = table[b / p.per_page];
      constexpr int kPer = D / 32;
      double x[kPer] = {};
      if (at >= 0 && at < a.pages) {
        const char* src = mean_at(b, at) + lane * kPer * 2;
#pragma unroll
        for (int e = 0; e < kPer; ++e) {
          if (std::is_same<T, __half>::value) x[e] = static_cast<double>(__half2float(*reinterpret_cast<const __half*>(src + 2 * e)));
          else x[e] = static_cast<double>(__bfloat162float(*reinterpret_cast<const __nv_bfloat16*>(src + 2 * e)));
        }
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
    nth_largest<uint64_t>([&](int i) { return exact[i]; }, doubtful, prefix64, shift64, rest, histogram, digit, sums);
  }
  // in the order of the blocks: those above, and of the ones between those that have been found, of equal ones the first `rest`
  int before = 0, equal = 0, seen = 0;
  for (int c0 = 0; c0 < candidates && before < keep; c0 += kSelectThreads) {
    const int c = c0 + static_cast<int>(threadIdx.x);
    const bool in = c < candidates && scores[c] > sure, between = c < candidates && !in && !(scores[c] < out_of);
    bool take = in || between;
    int total;
    if (doubtful > keep - above) {
      const int at = seen + select_scan(between, sums, &total);
      seen += total;
      const uint64_t top = between ? exact[at] >> shift64 : 0;
      const bool same = between && top == prefix64;
      const int place = equal + select_scan(same, sums, &total);
      equal += total;
      take = in || (between && top > prefix64) || (same && place < rest);
    }
    const int at = before + select_scan(take, sums, &total);
    if (take) write(low + at, low + c);
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
  while (p.cluster < 8 && items * kv_heads * p.cluster * 2 <= sm_count(device) && held >= 256 * p.cluster) p.cluster *= 2;
  RC_CHECK(a.group <= 128, "too many heads in a group for the choice of blocks");
  const int smem = q.size(2) == 128 ? paged::SelectShape<128>(a.group, static_cast<int>(held)).bytes : paged::SelectShape<64>(a.group, static_cast<int>(held)).bytes;
  RC_CHECK(smem <= 224 * 1024, "too many heads in a group, or blocks in the table, for the choice of blocks: take larger blocks");
  cudaStream_t stream = c10::cuda::getCurrentCUDAStream(device).stream();
  if (type == at::kHalf) q.size(2) == 128 ? paged::select_launch<__half, 128>(p, smem, stream, device) : paged::select_launch<__half, 64>(p, smem, stream, device);
  else q.size(2) == 128 ? paged::select_launch<__nv_bfloat16, 128>(p, smem, stream, device) : paged::select_launch<__nv_bfloat16, 64>(p, smem, stream, device);
  return {out, lens, cu};
}

}  // namespace rc
