// What the paged-attention kernels share: how keys are cut into tiles, which keys a query sees, and the argument block.
#pragma once

#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include "../common/sm100.cuh"
#include "paged.h"

namespace rc {
namespace paged {

constexpr float kLog2e = 1.4426950408889634f;
constexpr float kLn2 = 0.6931471805599453f;

// Tile t holds the positions [t * rows, (t + 1) * rows) of a sequence. Where they lie in one page, one TMA box of `rows`
// token rows (and 64 channels) fetches them; else boxes of `step` rows do, the largest power of two that divides the page
// size (a multiple of 8, so each box starts on a swizzle atom), which never cross a page's end.
struct Tiling {
  int page;  // page size
  int step;  // rows of a narrow box

  static Tiling of(int page, int rows) {
    const int two = page & -page;
    return {page, two < rows ? two : rows};
  }
};

struct Args {
  const void* q;  // [tokens, heads, D]
  int64_t q_token, q_head;
  void* out;
  int64_t out_token, out_head;
  int out_sectors;  // every row of out begins on 32 bytes
  float* lse;  // [tokens, heads] or null
  const int* table;
  const int* kv_lens;
  const int* cu_q;
  int seqs, width, pages;
  int64_t table_row;  // elements from one sequence's row of the table to the next
  int64_t table_head;  // and from one KV head's to the next (0: the heads share it)
  int heads, kv_heads, group;
  int causal, window, sinks;  // window 0: no window
  int tokens, max_q_len;
  float scale_log2;  // scale * log2(e)
  Tiling tiling;
  int* status;
};

// New tokens of a sequence (returned) and where they begin.
__device__ __forceinline__ int new_tokens(const Args& a, int s, int* q_first) {
  *q_first = a.cu_q[s];
  return *q_first < 0 ? 0 : max(0, min(a.cu_q[s + 1], a.tokens) - *q_first);
}

// Reports a sequence with more new tokens than max_q_len, or with rows that q does not have: what the kernels do not reach
// of them has no result. For one thread per sequence, off the path that the work waits for (in every SeqWork it took 0.25 us
// of a single token's 8.8).
__device__ __forceinline__ void report_rows(const Args& a, int s) {
  const int first = a.cu_q[s], end = a.cu_q[s + 1];
  if ((first < 0 || end < first || end > a.tokens || end - first > a.max_q_len) && a.status != nullptr)
    atomicCAS(a.status + kPagedWord, 0, kPageRows);
}

// Keys of a sequence: as many as kv_lens says and its row of the table can name (a longer length is reported).
__device__ __forceinline__ int held_keys(const Args& a, int s) {
  const int64_t most = static_cast<int64_t>(a.width) * a.tiling.page;
  const int n = max(0, a.kv_lens[s]);
  if (n <= most) return n;
  if (a.status != nullptr) atomicCAS(a.status + kPagedWord, 0, kPageRange);
  return static_cast<int>(most);
}

// The keys that queries see. A query whose last key is at `last` sees [max(0, last - window + 1), last] and the sinks
// [0, sinks) below it; `last` is the query's own position (causal) or the sequence's end.
struct Sight {
  int length;      // keys of the sequence
  int first_last;  // `last` of the first query
  int window, sinks, causal;

  __device__ __forceinline__ Sight(const Args& a, int kv_len, int q_len)
      : length(kv_len), first_last(a.causal ? kv_len - q_len : kv_len - 1), window(a.window), sinks(a.sinks), causal(a.causal) {}
  __device__ __forceinline__ int last(int query) const { return causal ? first_last + query : first_last; }
  // (`last` may be far below 0, where last - window would wrap)
  __device__ __forceinline__ int low(int last) const { return window > 0 && last >= window ? last - window + 1 : 0; }
};

// The tiles that the queries [first, end) of a sequence visit: [0, sink_end) and [window_begin, window_end).
template <int kTile>
struct TileRange {
  int sink_end, window_begin, window_end;
  __device__ __forceinline__ TileRange(const Sight& s, int first, int end) {
    const int top = s.last(end - 1);
    if (top < 0) {  // no query sees a key
      sink_end = window_begin = window_end = 0;
      return;
    }
    const int low = min(s.low(s.last(first)), top);
    window_begin = low / kTile;
    window_end = top / kTile + 1;
    sink_end = s.sinks > 0 ? min(window_begin, min(s.sinks - 1, top) / kTile + 1) : 0;
  }
  __device__ __forceinline__ int count() const { return sink_end + window_end - window_begin; }
  __device__ __forceinline__ int tile(int i) const { return i < sink_end ? i : window_begin + i - sink_end; }
};

// The boxes that fetch one tile's rows of K or V: `count` of them (one per lane), `rows` rows each. Positions past the
// sequence's end are not fetched (but for the rest of a box).
template <int kTile>
struct Boxes {
  int count, rows;
  __device__ __forceinline__ Boxes(const Tiling& t, int first, int kv_len) {
    const int there = min(kTile, kv_len - first);
    if (there <= 0) {
      count = rows = 0;
    } else if (t.step == kTile || first % t.page + kTile <= t.page) {
      count = 1;
      rows = kTile;
    } else {
      rows = t.step;
      count = (there + rows - 1) / rows;
    }
  }
  // page and row in it of the box that `lane` fetches; a page outside the pool comes out as -1 (it reads as zeros)
  __device__ __forceinline__ int page(const int* table, int pages, const Tiling& t, int first, int lane, int* row, int* status) const {
    const int at = first + lane * rows, block = at / t.page;
    *row = at - block * t.page;
    int page = table[block];
    if (page < 0 || page >= pages) {
      page = -1;
      if (status != nullptr) atomicCAS(status + kPagedWord, 0, kPageRange);
    }
    return page;
  }
};

__device__ __forceinline__ float exp2_approx(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}

// A row's maximum `top` and its sum of exp2(x - base_of(top)), and what follows from them. No key seen: -inf and 0, which
// give zeros and a log-sum-exp of -inf. A score of +inf leaves the sum at +inf (so base_of is 0 there too), one of NaN at
// NaN: log_sum passes both on, and the output, whose P holds them, is NaN. fade is what a sum or output that was taken
// relative to `before` is worth relative to `top` (infinite maxima that agree are worth 1, not exp2(inf - inf)).
__device__ __forceinline__ float base_of(float top) { return fabsf(top) == INFINITY ? 0.0f : top; }
__device__ __forceinline__ float fade(float before, float top) { return before == top ? 1.0f : exp2_approx(before - top); }
__device__ __forceinline__ float inverse(float sum) { return sum == 0.0f ? 0.0f : 1.0f / sum; }
__device__ __forceinline__ float log_sum(float top, float sum) {
  return sum == 0.0f ? -INFINITY : (base_of(top) + log2f(sum)) * kLn2;
}

// 4-D tile load of one page's rows: channels from c, token rows from `row`, one head, one page. A page number outside
// the map reads zeros.
__device__ __forceinline__ void load_page_box(void* dst, const CUtensorMap* map, uint64_t* bar, int c, int row, int head,
                                              int page) {
  asm volatile(
      "cp.async.bulk.tensor.4d.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1, {%3, %4, %5, %6}], [%2];" ::
          "r"(smem_u32(dst)),
      "l"(reinterpret_cast<uint64_t>(map)), "r"(smem_u32(bar)), "r"(c), "r"(row), "r"(head), "r"(page)
      : "memory");
}

// Distributed shared memory: values of another CTA of the cluster (addresses from cluster_addr).
__device__ __forceinline__ uint32_t cluster_addr_of(uint32_t addr, int rank) {
  uint32_t out;
  asm("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(out) : "r"(addr), "r"(rank));
  return out;
}
__device__ __forceinline__ float2 load_cluster_2(uint32_t addr) {
  float2 v;
  asm volatile("ld.shared::cluster.v2.f32 {%0, %1}, [%2];" : "=f"(v.x), "=f"(v.y) : "r"(addr) : "memory");
  return v;
}
__device__ __forceinline__ float4 load_cluster_4(uint32_t addr) {
  float4 v;
  asm volatile("ld.shared::cluster.v4.f32 {%0, %1, %2, %3}, [%4];"
               : "=f"(v.x), "=f"(v.y), "=f"(v.z), "=f"(v.w)
               : "r"(addr)
               : "memory");
  return v;
}

// d += a b, of 16 x 16 and 16 x 8 numbers.
__device__ __forceinline__ void mma_16816(float (&d)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1, __nv_bfloat16) {
  asm volatile(
      "mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
      : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
      : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
__device__ __forceinline__ void mma_16816(float (&d)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1, __half) {
  asm volatile(
      "mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
      : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
      : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}

template <typename T>
__device__ __forceinline__ uint32_t pack2(float lo, float hi);
template <>
__device__ __forceinline__ uint32_t pack2<__nv_bfloat16>(float lo, float hi) { return pack_bf16x2(lo, hi); }
template <>
__device__ __forceinline__ uint32_t pack2<__half>(float lo, float hi) { return pack_f16x2(lo, hi); }

// Tensor map of [pages, page_size, heads, D] with boxes of 64 channels x `box` rows of one head and page.
inline CUtensorMap page_map(const at::Tensor& t, int box) {
  CUtensorMap map;
  const cuuint64_t dims[4] = {static_cast<cuuint64_t>(t.size(3)), static_cast<cuuint64_t>(t.size(1)),
                              static_cast<cuuint64_t>(t.size(2)), static_cast<cuuint64_t>(t.size(0))};
  const cuuint64_t strides[3] = {static_cast<cuuint64_t>(t.stride(1)) * 2, static_cast<cuuint64_t>(t.stride(2)) * 2,
                                 static_cast<cuuint64_t>(t.stride(0)) * 2};
  const cuuint32_t boxes[4] = {64, static_cast<cuuint32_t>(box), 1, 1};
  const cuuint32_t ones[4] = {1, 1, 1, 1};
  const CUresult res = encode_tiled_fn()(
      &map, t.scalar_type() == at::kHalf ? CU_TENSOR_MAP_DATA_TYPE_FLOAT16 : CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, 4,
      t.data_ptr(), dims, strides, boxes, ones, CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B,
      CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
  RC_CHECK(res == CUDA_SUCCESS, "cuTensorMapEncodeTiled (pages) failed (code " + std::to_string(static_cast<int>(res)) + ")");
  return map;
}

struct PageMaps {
  CUtensorMap k_wide, v_wide, k_step, v_step;
};

inline PageMaps page_maps(const at::Tensor& k, const at::Tensor& v, const Tiling& t, int rows,
                          CUtensorMap (*map_of)(const at::Tensor&, int) = page_map) {
  PageMaps maps;
  // a box may not be larger than the page it is cut from: without whole tiles in a page the wide maps are not used
  const bool wide = t.page >= rows, step = t.step < rows;
  if (wide) {
    maps.k_wide = map_of(k, rows);
    maps.v_wide = map_of(v, rows);
  }
  if (step) {
    maps.k_step = map_of(k, t.step);
    maps.v_step = map_of(v, t.step);
  }
  if (!wide) {
    maps.k_wide = maps.k_step;
    maps.v_wide = maps.v_step;
  }
  if (!step) {
    maps.k_step = maps.k_wide;
    maps.v_step = maps.v_wide;
  }
  return maps;
}

}  // namespace paged
}  // namespace rc
