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

// A tile holds consecutive positions of one sequence, at most `rows` of them, in at most one TMA box per page. Pages
// smaller than a tile: `per_tile` whole pages (page size a multiple of 8, so each lands on a swizzle atom). Larger
// pages: `per_page` boxes of `box` rows each; the last box of a page may reach past its end, where TMA fills zeros.
struct Tiling {
  int page;      // page size
  int box;       // rows of one TMA box
  int per_page;  // tiles of one page (1 where pages are smaller than a tile)
  int per_tile;  // pages of one tile (1 where tiles are smaller than a page)

  static Tiling of(int page, int rows) {
    Tiling t{page, page, 1, 1};
    if (page > rows) {
      t.per_page = (page + rows - 1) / rows;
      t.box = ((page + t.per_page - 1) / t.per_page + 7) / 8 * 8;
      t.per_page = (page + t.box - 1) / t.box;
    } else {
      t.per_tile = rows / page;
    }
    return t;
  }

  __device__ __forceinline__ int tile_of(int position) const {
    if (per_page > 1) {
      const int p = position / page;
      return p * per_page + (position - p * page) / box;
    }
    return position / (page * per_tile);
  }
  // first position of a tile, its first page's block in the table, its first row in that page
  __device__ __forceinline__ int first(int tile, int* block, int* row) const {
    if (per_page > 1) {
      *block = tile / per_page;
      *row = (tile - *block * per_page) * box;
      return *block * page + *row;
    }
    *block = tile * per_tile;
    *row = 0;
    return *block * page;
  }
  __device__ __forceinline__ int first(int tile) const {
    int block, row;
    return first(tile, &block, &row);
  }
  // positions of a tile that exist in its pages
  __device__ __forceinline__ int count(int row) const { return per_page > 1 ? min(box, page - row) : page * per_tile; }
};

struct Args {
  const void* q;  // [tokens, heads, D]
  int64_t q_token, q_head;
  void* out;
  int64_t out_token, out_head;
  float* lse;  // [tokens, heads] or null
  const int* table;
  const int* kv_lens;
  const int* cu_q;
  int seqs, width, pages;
  int heads, kv_heads, group;
  int causal, window, sinks;  // window 0: no window
  int tokens;
  float scale_log2;  // scale * log2(e)
  Tiling tiling;
  int* status;
};

// The keys that queries see. A query whose last key is at `last` sees [max(0, last - window + 1), last] and the sinks
// [0, sinks) below it; `last` is the query's own position (causal) or the sequence's end.
struct Sight {
  int length;      // keys of the sequence
  int first_last;  // `last` of the first query
  int window, sinks, causal;

  __device__ __forceinline__ Sight(const Args& a, int kv_len, int q_len)
      : length(kv_len), first_last(a.causal ? kv_len - q_len : kv_len - 1), window(a.window), sinks(a.sinks), causal(a.causal) {}
  __device__ __forceinline__ int last(int query) const { return causal ? first_last + query : first_last; }
  __device__ __forceinline__ int low(int last) const { return window > 0 ? max(0, last - window + 1) : 0; }
};

// The tiles that the queries [first, end) of a sequence visit: [0, sink_end) and [window_begin, window_end).
struct TileRange {
  int sink_end, window_begin, window_end;
  __device__ __forceinline__ TileRange(const Tiling& t, const Sight& s, int first, int end) {
    const int top = s.last(end - 1);
    if (top < 0) {  // no query sees a key
      sink_end = window_begin = window_end = 0;
      return;
    }
    const int low = min(s.low(s.last(first)), top);
    window_begin = t.tile_of(low);
    window_end = t.tile_of(top) + 1;
    sink_end = s.sinks > 0 ? min(window_begin, t.tile_of(min(s.sinks - 1, top)) + 1) : 0;
  }
  __device__ __forceinline__ int count() const { return sink_end + window_end - window_begin; }
  __device__ __forceinline__ int tile(int i) const { return i < sink_end ? i : window_begin + i - sink_end; }
};

__device__ __forceinline__ float exp2_approx(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
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

}  // namespace paged
}  // namespace rc
