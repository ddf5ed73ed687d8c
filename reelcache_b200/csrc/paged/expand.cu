// Pages in 8 bits as pages in 16 bits, for attention of many query rows over them, for sm_100a.
//
// Many rows (chunks, prompts) are bound by the tensor core and the exponentials, which have no issue slots left for turning
// codes into numbers once for every 256 rows; doing it once for each page of the call costs 5 bytes of traffic a number (1 read, 2 written, 2
// read) next to hundreds of operations. Only pages that the call's queries see are expanded, each once however many sequences
// and heads name it: a first kernel gives them places in the order in which it meets them (the place of a page depends on
// timing, what is in it does not), a second one expands them and writes the table of places. Room is taken before it is known which
// those are: for as many pages as the table has entries, of which a window and its sinks leave a part, or as the pool has pages.
// Measured: 4,680 tokens over 23,400 keys of 12 heads 667 us, 661 over 16-bit pages.
#include <ATen/ATen.h>
#include <c10/cuda/CUDAGuard.h>
#include <c10/cuda/CUDAStream.h>

#include <algorithm>
#include <string>

#include "attend.cuh"
#include "packed.h"

namespace rc {
namespace paged {

constexpr int kExpandThreads = 256;
constexpr int kExpandItems = 4;   // vectors of sixteen channels of a thread
constexpr int kTileKeys = 128;    // of the attention that reads the places: what it touches of a window's edge,
constexpr int kTileRows = 256;    // and rows of an item of it: some may be of tokens beyond max_q_len

struct Expand {
  Args a;
  int table_heads;  // 1: the heads share a table
  int* place;       // [pages]: place of a page, -1 for none
  int* count;       // places so far, less one
  int* list;        // [places]: page of each place
  int* table;       // [seqs, table_heads, width]: places
  int places;
  int reach;        // new tokens of a sequence that the attention takes, at most
  Packed pages[2];
  const uint8_t* codes[2];
  char* out[2];     // [places, page_size, kv_heads, head_dim]
  int vecs;         // of a head
};

__global__ void __launch_bounds__(kExpandThreads) place_kernel(const __grid_constant__ Expand p) {
  let_later();
  after_earlier();
  const Args& a = p.a;
  const int64_t cells = static_cast<int64_t>(a.seqs) * p.table_heads * a.width;
  for (int64_t c = static_cast<int64_t>(blockIdx.x) * kExpandThreads + threadIdx.x; c < cells; c += static_cast<int64_t>(gridDim.x) * kExpandThreads) {
    const int64_t row = c / a.width;
    const int block = static_cast<int>(c - row * a.width), s = static_cast<int>(row / p.table_heads), head = static_cast<int>(row - static_cast<int64_t>(s) * p.table_heads);
    int q_first;
    const int q_len = new_tokens(a, s, &q_first), kv_len = held_keys(a, s);
    const int64_t from = static_cast<int64_t>(block) * a.tiling.page;
    if (q_len == 0 || from >= kv_len) continue;
    const Sight sight(a, kv_len, q_len);
    const int low = sight.low(sight.last(0)) / kTileKeys * kTileKeys, top = sight.last(min(q_len, p.reach) - 1);
    if (top < 0) continue;
    const int64_t sinks = (static_cast<int64_t>(a.sinks) + kTileKeys - 1) / kTileKeys * kTileKeys;
    const int64_t end = (static_cast<int64_t>(top) / kTileKeys + 1) * kTileKeys;
    if ((from + a.tiling.page <= low || from >= end) && from >= sinks) continue;
    const int page = a.table[s * a.table_row + head * a.table_head + block];
    if (page < 0 || page >= a.pages || atomicCAS(p.place + page, -1, -2) != -1) continue;
    const int at = atomicAdd(p.count, 1) + 1;
    if (at >= p.places) continue;  // (more than the room was reckoned for: never)
    p.list[at] = page;
    p.place[page] = at;
  }
}

template <typename T>
__global__ void __launch_bounds__(kExpandThreads) expand_kernel(const __grid_constant__ Expand p) {
  let_later();
  after_earlier();
  const Args& a = p.a;
  const int64_t cells = static_cast<int64_t>(a.seqs) * p.table_heads * a.width, step = static_cast<int64_t>(gridDim.x) * kExpandThreads;
  for (int64_t c = static_cast<int64_t>(blockIdx.x) * kExpandThreads + threadIdx.x; c < cells; c += step) {
    const int64_t row = c / a.width;
    const int64_t s = row / p.table_heads, head = row - s * p.table_heads;
    const int page = a.table[s * a.table_row + head * a.table_head + c - row * a.width];
    // (a page that nothing taken sees has no place: any does, since what reads it has no result)
    p.table[c] = page >= 0 && page < a.pages ? max(p.place[page], 0) : -1;
  }
  const int places = min(p.places, *p.count + 1);
  const int per_token = a.kv_heads * p.vecs, per_page = a.tiling.page * per_token;
  const int parts = (per_page + kExpandThreads * kExpandItems - 1) / (kExpandThreads * kExpandItems);
  const int64_t items = static_cast<int64_t>(places) * 2 * parts;
  for (int64_t item = blockIdx.x; item < items; item += gridDim.x) {
    const int at = static_cast<int>(item / (2 * parts)), rest = static_cast<int>(item - static_cast<int64_t>(at) * 2 * parts);
    const int which = rest / parts, first = (rest - which * parts) * kExpandThreads * kExpandItems + threadIdx.x;
    const Packed& pages = which ? p.pages[1] : p.pages[0];
    const int64_t page = p.list[at];
    const uint8_t* from = (which ? p.codes[1] : p.codes[0]) + page * pages.page_stride;
    const uint8_t* scales = pages.scales + page * pages.scale_page;
    uint4 codes[kExpandItems];
    int scale[kExpandItems];
#pragma unroll
    for (int i = 0; i < kExpandItems; ++i) {
      const int v = first + i * kExpandThreads;
      if (v >= per_page) continue;
      const int row = v / per_token, part = v - row * per_token, head = part / p.vecs;
      codes[i] = *reinterpret_cast<const uint4*>(from + row * pages.token_stride + head * pages.head_stride + (part - head * p.vecs) * 16);
      scale[i] = scales[head * pages.scale_head + row];
    }
    char* to = (which ? p.out[1] : p.out[0]) + static_cast<int64_t>(at) * per_page * 32;
#pragma unroll
    for (int i = 0; i < kExpandItems; ++i) {
      const int v = first + i * kExpandThreads;
      if (v >= per_page) continue;
      store_values<T>(to + static_cast<int64_t>(v) * 32, codes[i], scale_value(scale[i]));
    }
  }
}

// The pages that the call sees in 16 bits (of like's type), in new tensors, and `a` changed to name them.
void expand_pages(Args& a, const at::Tensor& k_codes, const at::Tensor& v_codes, const Packed& k, const Packed& v, at::Tensor& k_pages,
                  at::Tensor& v_pages, at::Tensor& workspace, const at::Tensor& like, cudaStream_t stream) {
  Expand p{};
  p.a = a;
  p.table_heads = a.table_head != 0 ? a.kv_heads : 1;
  const int64_t cells = static_cast<int64_t>(a.seqs) * p.table_heads * a.width;
  RC_CHECK(cells < (1ll << 31), "too many sequences and blocks for packed pages");
  const int64_t rows = static_cast<int64_t>(std::min(a.max_q_len, a.tokens)) * a.group;
  p.reach = static_cast<int>(((rows + kTileRows - 1) / kTileRows * kTileRows + a.group - 1) / a.group);
  int64_t seen = a.width;  // pages of a table's row that the queries see, at most: those of the sinks' tiles, and of the window's
  if (a.window > 0) {
    const auto pages_of = [&](int64_t keys) { return (keys + a.tiling.page - 2) / a.tiling.page + 1; };
    seen = std::min(seen, (a.sinks > 0 ? pages_of(static_cast<int64_t>(a.sinks) + kTileKeys) : 0) +
                              pages_of(static_cast<int64_t>(a.window) + p.reach + 2 * kTileKeys));
  }
  p.places = static_cast<int>(std::min<int64_t>(a.pages, std::max<int64_t>(seen * a.seqs * p.table_heads, 1)));
  const int64_t d = like.size(2), per_page = static_cast<int64_t>(a.tiling.page) * a.kv_heads * (d / 16);
  RC_CHECK(per_page < (1ll << 30), "a packed page is too large");
  k_pages = at::empty({p.places, a.tiling.page, a.kv_heads, d}, like.options());
  v_pages = at::empty({p.places, a.tiling.page, a.kv_heads, d}, like.options());
  workspace = at::empty({1 + static_cast<int64_t>(a.pages) + p.places + cells}, like.options().dtype(at::kInt));
  p.count = workspace.data_ptr<int>();
  p.place = p.count + 1;
  p.list = p.place + a.pages;
  p.table = p.list + p.places;
  p.pages[0] = k;
  p.pages[1] = v;
  p.codes[0] = static_cast<const uint8_t*>(k_codes.data_ptr());
  p.codes[1] = static_cast<const uint8_t*>(v_codes.data_ptr());
  p.out[0] = static_cast<char*>(k_pages.data_ptr());
  p.out[1] = static_cast<char*>(v_pages.data_ptr());
  p.vecs = static_cast<int>(d / 16);
  const int sms = sm_count(like.get_device());
  RC_CUDA(cudaMemsetAsync(p.count, 0xff, sizeof(int) * (1 + static_cast<size_t>(a.pages)), stream));
  const int64_t blocks = std::max<int64_t>(1, (cells + kExpandThreads - 1) / kExpandThreads);
  launch(place_kernel, dim3(static_cast<unsigned>(std::min<int64_t>(blocks, sms * 8))), kExpandThreads, 0, 0, stream, p);
  const int64_t parts = (per_page + kExpandThreads * kExpandItems - 1) / (kExpandThreads * kExpandItems);
  const dim3 grid(static_cast<unsigned>(std::min<int64_t>(std::max<int64_t>(p.places * 2 * parts, blocks), sms * 8)));
  launch(like.scalar_type() == at::kHalf ? expand_kernel<__half> : expand_kernel<__nv_bfloat16>, grid, kExpandThreads, 0, 0, stream, p);
  a.table = p.table;
  a.table_row = static_cast<int64_t>(p.table_heads) * a.width;
  a.table_head = p.table_heads > 1 || a.table_head != 0 ? a.width : 0;
  a.pages = p.places;
}

}  // namespace paged
}  // namespace rc
