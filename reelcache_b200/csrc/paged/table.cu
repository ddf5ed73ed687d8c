// Page-table operators of the paged KV cache, all on the device (no read-back, so they can be captured in a graph).
//
// State: refcount[pages] (0: free), lens[seqs] (tokens held), table[seqs, width] (page of each block, -1: none). Every
// operator is a function of the state alone: free pages are taken lowest first, in the order of the call's sequences.
//
//   allocate  sequences grow to new lengths: their missing blocks take free pages
//   fork      a child takes the first `at` tokens of a parent: whole pages are shared (refcount + 1), the rows of a
//             partly filled last page are copied to a page of the child's own, so a page that may still be written
//             belongs to one sequence
//   release   a sequence gives its pages back
//   compact   with n pages in use, those at n and above move to the free ones below n (i-th to i-th); tables follow
//   copy      given pages (or their first rows) to given others
// What lies beside the pages (scales of packed ones, means of blocks) moves with them, whole pages of it.
//
// allocate, fork and compact start with a plan by one block of 1,024 threads: prefix sums over the call's sequences and
// over refcount, which it reads only as far as it finds what it needs. A call that cannot be served (too few free pages,
// a sequence out of range or named twice, a table row too short, a child that still holds pages) is refused whole: the
// plan writes nothing but the status word (a release skips sequences out of range, and gives back once what is named
// twice). Tables, counts and data are then moved by one launch over all SMs, which
// reads the plan from device memory. The plan is latency (4 to 6 us); the move is a copy, bound by HBM (measured: 0.5 GB of
// pages moved together in 152 us, 6.3 TB/s read and written).
#include <ATen/ATen.h>
#include <c10/cuda/CUDAGuard.h>
#include <c10/cuda/CUDAStream.h>

#include <algorithm>
#include <string>
#include <vector>

#include "../common/host.h"
#include "paged.h"

namespace rc {
namespace pagetable {

using paged::block_scan;
using paged::kPlanThreads;

constexpr int kMoveThreads = 256;
constexpr int kMoveVecs = 8;                                  // 16-byte vectors per thread and work item
constexpr int kMoveBytes = kMoveThreads * kMoveVecs * 16;     // 32 KB of a page and plane
constexpr int kMaxCall = 1 << 16;  // sequences of one call

struct State {
  int* refcount;
  int* lens;
  int* table;
  int pages, seqs, width, page;
};

// Plan words: [0] moves (or -1: refused), then per move source, target and rows.
struct Plan {
  int* count;
  int* source;
  int* target;
  int* rows;
};

__device__ __forceinline__ void refuse(int* status, int code) {
  if (status != nullptr) atomicCAS(status + kPagedWord, 0, code);
}

// Lists the first `wanted` free pages, lowest first, into `list`; returns how many there are (at most `wanted`).
__device__ int list_free(const State& s, int wanted, int* list, int* warp_sums) {
  int found = 0;
  for (int base = 0; base < s.pages && found < wanted; base += kPlanThreads * 4) {
    const int i0 = base + static_cast<int>(threadIdx.x) * 4;
    int flags = 0, mine = 0;
#pragma unroll
    for (int e = 0; e < 4; ++e)
      if (i0 + e < s.pages && s.refcount[i0 + e] == 0) {
        flags |= 1 << e;
        ++mine;
      }
    int total;
    int rank = found + block_scan(mine, warp_sums, &total);
#pragma unroll
    for (int e = 0; e < 4; ++e)
      if ((flags >> e) & 1) {
        if (rank < wanted) list[rank] = i0 + e;
        ++rank;
      }
    found += total;
  }
  __syncthreads();  // the list is read by other threads
  return min(found, wanted);
}

// Whether a sequence is named twice: `seen` holds one word per sequence, which the first to name it takes.
__device__ __forceinline__ bool take(int* seen, int seq) { return atomicExch(seen + seq, 1) == 0; }

// scratch: list[pages] | offsets[n + 1] | seen[seqs]
__global__ void __launch_bounds__(kPlanThreads) allocate_kernel(State s, const int* seqs, const int* lens, int n,
                                                                int* list, int* offsets, int* seen, int* status) {
  paged::let_later();
  paged::after_earlier();
  __shared__ int warp_sums[32];
  __shared__ int bad;
  if (threadIdx.x == 0) bad = 0;
  for (int i = threadIdx.x; i < s.seqs; i += kPlanThreads) seen[i] = 0;
  __syncthreads();
  int need = 0;
  for (int base = 0; base < n; base += kPlanThreads) {
    const int i = base + threadIdx.x;
    int mine = 0;
    if (i < n) {
      const int seq = seqs[i], len = lens[i];
      const bool known = seq >= 0 && seq < s.seqs;
      if (!known || !take(seen, seq) || len < s.lens[seq] || (len - 1) / s.page + (len > 0) > s.width) {
        bad = 1;
      } else {
        const int old = s.lens[seq];
        mine = min((len > 0 ? (len - 1) / s.page + 1 : 0) - (old > 0 ? (old - 1) / s.page + 1 : 0), s.pages + 1);
      }
    }
    int total;
    const int before = block_scan(mine, warp_sums, &total);
    if (i < n) offsets[i] = need + before;
    need = min(need + total, 1 << 29);  // more than any pool: refused below
  }
  if (threadIdx.x == 0) offsets[n] = need;
  __syncthreads();
  if (bad) {
    if (threadIdx.x == 0) refuse(status, kPageRefused);
    return;
  }
  if (need > s.pages || list_free(s, need, list, warp_sums) < need) {
    if (threadIdx.x == 0) refuse(status, kPageExhausted);
    return;
  }
  for (int r = threadIdx.x; r < need; r += kPlanThreads) {
    int lo = 0, hi = n - 1;  // the last i with offsets[i] <= r
    while (lo < hi) {
      const int mid = (lo + hi + 1) >> 1;
      if (offsets[mid] <= r) lo = mid;
      else hi = mid - 1;
    }
    const int seq = seqs[lo], old = s.lens[seq];
    const int block = (old > 0 ? (old - 1) / s.page + 1 : 0) + r - offsets[lo];
    s.table[static_cast<int64_t>(seq) * s.width + block] = list[r];
    s.refcount[list[r]] = 1;
  }
  __syncthreads();  // every old length has been read
  for (int i = threadIdx.x; i < n; i += kPlanThreads) s.lens[seqs[i]] = lens[i];
}

// Plans a fork: move i copies the partial tail of fork i (rows 0: there is none).
__global__ void __launch_bounds__(kPlanThreads) fork_plan_kernel(State s, const int* parents, const int* children,
                                                                 const int* at, int n, int* list, int* seen, Plan plan,
                                                                 int* status) {
  paged::let_later();
  paged::after_earlier();
  __shared__ int warp_sums[32];
  __shared__ int bad;
  if (threadIdx.x == 0) bad = 0;
  for (int i = threadIdx.x; i < s.seqs; i += kPlanThreads) seen[i] = 0;
  __syncthreads();
  int need = 0;
  for (int base = 0; base < n; base += kPlanThreads) {
    const int i = base + threadIdx.x;
    int mine = 0;
    if (i < n) {
      const int parent = parents[i], child = children[i], len = at[i];
      if (parent < 0 || parent >= s.seqs || child < 0 || child >= s.seqs || len < 0 || len > s.lens[parent] ||
          s.lens[child] != 0 || !take(seen, child) || (len + s.page - 1) / s.page > s.width) {
        bad = 1;
      } else {
        mine = len % s.page > 0;
        plan.rows[i] = len % s.page;
        plan.source[i] = mine ? s.table[static_cast<int64_t>(parent) * s.width + len / s.page] : 0;
      }
    }
    int total;
    const int before = block_scan(mine, warp_sums, &total);
    if (i < n) plan.target[i] = need + before;  // its place in the list of free pages
    need += total;
  }
  __syncthreads();
  // a child of this call is no parent of it: it is empty, so only forks of length 0 could name it
  if (bad || need > s.pages || list_free(s, need, list, warp_sums) < need) {
    if (threadIdx.x == 0) {
      refuse(status, bad ? kPageRefused : kPageExhausted);
      *plan.count = -1;
    }
    return;
  }
  for (int i = threadIdx.x; i < n; i += kPlanThreads)
    plan.target[i] = plan.rows[i] > 0 ? list[plan.target[i]] : -1;
  if (threadIdx.x == 0) *plan.count = n;
}

__global__ void __launch_bounds__(kPlanThreads) compact_plan_kernel(State s, int* place, Plan plan, int* in_use) {
  paged::let_later();
  paged::after_earlier();
  __shared__ int warp_sums[32];
  int live = 0;
  for (int base = 0; base < s.pages; base += kPlanThreads * 4) {
    const int i0 = base + static_cast<int>(threadIdx.x) * 4;
    int mine = 0;
#pragma unroll
    for (int e = 0; e < 4; ++e) mine += i0 + e < s.pages && s.refcount[i0 + e] != 0;
    int total;
    block_scan(mine, warp_sums, &total);
    live += total;
  }
  // holes below `live` and pages in use at or above it: equally many, in order
  int holes = 0, movers = 0;
  for (int base = 0; base < s.pages; base += kPlanThreads * 4) {
    const int i0 = base + static_cast<int>(threadIdx.x) * 4;
    int flags = 0, hole = 0, mover = 0;
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      const int i = i0 + e;
      if (i >= s.pages) continue;
      const bool used = s.refcount[i] != 0;
      if (i < live && !used) {
        flags |= 1 << e;
        ++hole;
      } else if (i >= live && used) {
        flags |= 1 << e;
        ++mover;
      }
    }
    int total_h, total_m;
    int rh = holes + block_scan(hole, warp_sums, &total_h);
    int rm = movers + block_scan(mover, warp_sums, &total_m);
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      if (!((flags >> e) & 1)) continue;
      const int i = i0 + e;
      if (i < live) {
        plan.target[rh++] = i;
      } else {
        plan.source[rm++] = i;
      }
    }
    holes += total_h;
    movers += total_m;
  }
  __syncthreads();
  for (int m = threadIdx.x; m < movers; m += kPlanThreads) place[plan.source[m]] = plan.target[m];
  if (threadIdx.x == 0) {
    *plan.count = movers;
    if (in_use != nullptr) *in_use = live;
  }
}

struct Storage {  // planes x pages, each page `page_bytes` contiguous bytes of `page` rows
  char* base;
  int64_t plane_stride, page_stride;
  int planes;
  int64_t page_bytes;
  int row_bytes;
};

// The copies of a plan: items of (move, plane, 32 KB part), spread over the grid. rows == nullptr: whole pages. The next
// item's entries of the plan are asked for before this one's stores, which the compiler must take for stores to the plan.
__device__ __forceinline__ void move_pages(const Storage& st, int moves, int pages, const int* source, const int* target,
                                           const int* rows, int* status) {
  const int parts = static_cast<int>((st.page_bytes + kMoveBytes - 1) / kMoveBytes);
  const int64_t items = static_cast<int64_t>(moves) * st.planes * parts;
  int src = 0, dst = 0;
  int64_t bytes = 0;
  auto look_up = [&](int64_t item) {
    if (item >= items) return;
    const int move = static_cast<int>(item / parts / st.planes);
    src = source[move];
    dst = target[move];
    bytes = rows == nullptr ? st.page_bytes : static_cast<int64_t>(rows[move]) * st.row_bytes;
  };
  look_up(blockIdx.x);
  for (int64_t item = blockIdx.x; item < items; item += gridDim.x) {
    const int plane = static_cast<int>(item / parts % st.planes);
    const int64_t at = item % parts * kMoveBytes + threadIdx.x * 16, there = bytes;
    bool ok = there > 0;
    if (ok && (src < 0 || src >= pages || dst < 0 || dst >= pages || there > st.page_bytes)) {
      if (threadIdx.x == 0 && !(src == -1 && dst == -1)) refuse(status, kPageRange);
      ok = false;
    }
    const char* from = st.base + plane * st.plane_stride + src * st.page_stride;
    char* to = st.base + plane * st.plane_stride + dst * st.page_stride;
    uint4 v[kMoveVecs];
#pragma unroll
    for (int e = 0; e < kMoveVecs; ++e) {
      const int64_t o = at + e * (kMoveThreads * 16);
      if (ok && o < there) v[e] = *reinterpret_cast<const uint4*>(from + o);
    }
    look_up(item + gridDim.x);
#pragma unroll
    for (int e = 0; e < kMoveVecs; ++e) {
      const int64_t o = at + e * (kMoveThreads * 16);
      if (ok && o < there) *reinterpret_cast<uint4*>(to + o) = v[e];
    }
  }
}

// Tensors beside the storage, [planes, pages, ...], of which whole pages move: in words of 8 bytes, small next to the pages.
struct Side {
  char* base;
  int64_t plane_stride, page_stride;
  int planes, words;
};
constexpr int kMostSides = 2;
struct Sides {
  Side at[kMostSides];
  int count;
};

__device__ __forceinline__ void move_sides(const Sides& sides, int moves, int pages, const int* source, const int* target, const int* rows) {
  for (int i = 0; i < sides.count; ++i) {
    const Side& side = sides.at[i];
    const int64_t each = static_cast<int64_t>(side.planes) * side.words, items = moves * each;
    for (int64_t item = static_cast<int64_t>(blockIdx.x) * kMoveThreads + threadIdx.x; item < items; item += static_cast<int64_t>(gridDim.x) * kMoveThreads) {
      const int move = static_cast<int>(item / each);
      const int64_t rest = item - move * each, plane = rest / side.words, word = rest - plane * side.words;
      if (rows != nullptr && rows[move] == 0) continue;
      const int src = source[move], dst = target[move];
      if (src < 0 || src >= pages || dst < 0 || dst >= pages) continue;  // (reported with the pages)
      char* base = side.base + plane * side.plane_stride + word * 8;
      *reinterpret_cast<uint2*>(base + dst * side.page_stride) = *reinterpret_cast<const uint2*>(base + src * side.page_stride);
    }
  }
}

__global__ void __launch_bounds__(kMoveThreads) copy_kernel(Storage st, int pages, const int* source, const int* target,
                                                            const int* rows, int moves, int* status) {
  paged::let_later();
  paged::after_earlier();
  move_pages(st, moves, pages, source, target, rows, status);
}

// kSides: whether anything lies beside the pages (the copies of the pages alone keep their registers).
template <bool kSides>
__global__ void __launch_bounds__(kMoveThreads) fork_kernel(State s, Storage st, Sides sides, const int* parents, const int* children,
                                                            const int* at, int n, Plan plan, int* status) {
  paged::let_later();
  paged::after_earlier();
  if (*plan.count < 0) return;
  const int64_t cells = static_cast<int64_t>(n) * s.width;
  for (int64_t c = static_cast<int64_t>(blockIdx.x) * kMoveThreads + threadIdx.x; c < cells;
       c += static_cast<int64_t>(gridDim.x) * kMoveThreads) {
    const int i = static_cast<int>(c / s.width), block = static_cast<int>(c - static_cast<int64_t>(i) * s.width);
    const int len = at[i], full = len / s.page, child = children[i];
    int page = -1;
    if (block < full) {
      page = s.table[static_cast<int64_t>(parents[i]) * s.width + block];
      if (page >= 0 && page < s.pages) atomicAdd(s.refcount + page, 1);
    } else if (block == full && plan.rows[i] > 0) {
      page = plan.target[i];
      s.refcount[page] = 1;
    }
    s.table[static_cast<int64_t>(child) * s.width + block] = page;
    if (block == 0) s.lens[child] = len;
  }
  move_pages(st, n, s.pages, plan.source, plan.target, plan.rows, status);
  if (kSides) move_sides(sides, n, s.pages, plan.source, plan.target, plan.rows);
}

template <bool kSides>
__global__ void __launch_bounds__(kMoveThreads) compact_kernel(State s, Storage st, Sides sides, const int* place, const int* in_use, Plan plan,
                                                               int* status) {
  paged::let_later();
  paged::after_earlier();
  const int moves = *plan.count, live = *in_use;
  const int64_t cells = static_cast<int64_t>(s.seqs) * s.width;
  const int64_t step = static_cast<int64_t>(gridDim.x) * kMoveThreads;
  const int64_t first = static_cast<int64_t>(blockIdx.x) * kMoveThreads + threadIdx.x;
  for (int64_t c = first; c < cells; c += step) {
    const int page = s.table[c];
    if (page >= live && page < s.pages) s.table[c] = place[page];
  }
  for (int64_t m = first; m < moves; m += step) {
    s.refcount[plan.target[m]] = s.refcount[plan.source[m]];
    s.refcount[plan.source[m]] = 0;
  }
  move_pages(st, moves, s.pages, plan.source, plan.target, nullptr, status);
  if (kSides) move_sides(sides, moves, s.pages, plan.source, plan.target, nullptr);
}

__global__ void __launch_bounds__(kMoveThreads) release_kernel(State s, const int* seqs, int n, int* status) {
  paged::let_later();
  paged::after_earlier();
  const int64_t cells = static_cast<int64_t>(n) * s.width;
  for (int64_t c = static_cast<int64_t>(blockIdx.x) * kMoveThreads + threadIdx.x; c < cells;
       c += static_cast<int64_t>(gridDim.x) * kMoveThreads) {
    const int i = static_cast<int>(c / s.width), block = static_cast<int>(c - static_cast<int64_t>(i) * s.width);
    const int seq = seqs[i];
    if (seq < 0 || seq >= s.seqs) {
      if (block == 0) refuse(status, kPageRefused);
      continue;
    }
    // the exchange makes a sequence that is named twice give its pages back once
    const int page = atomicExch(s.table + static_cast<int64_t>(seq) * s.width + block, -1);
    if (page >= 0 && page < s.pages) atomicSub(s.refcount + page, 1);
    if (block == 0) s.lens[seq] = 0;
  }
}

// state: refcount[pages] | lens[seqs] | table[seqs, width]
State check_state(at::Tensor& state, int64_t pages, int64_t seqs, int64_t page_size) {
  RC_CHECK(state.is_cuda() && state.scalar_type() == at::kInt && state.dim() == 1 && state.is_contiguous(),
           "a page table's state must be a contiguous int32 CUDA vector");
  // (below 2^20 pages the 1,024 needs that one prefix sum adds up stay below 2^31)
  RC_CHECK(pages >= 1 && pages < (1 << 20) && seqs >= 1 && seqs < (1 << 20), "the page table is empty or too large");
  const int64_t cells = state.numel() - pages - seqs, width = cells / seqs;
  RC_CHECK(cells > 0 && cells % seqs == 0 && width < (1 << 28), "a page table's state is pages + seqs + seqs * width entries");
  RC_CHECK(page_size >= 8 && page_size % 8 == 0 && page_size <= 65536,
           "the page size must be a multiple of 8 tokens, at most 65536");
  int* p = state.data_ptr<int>();
  return {p, p + pages, p + pages + seqs, static_cast<int>(pages), static_cast<int>(seqs), static_cast<int>(width),
          static_cast<int>(page_size)};
}

const int* check_list(const at::Tensor& t, const at::Device& device, int64_t n, const char* name) {
  RC_CHECK(t.device() == device && t.scalar_type() == at::kInt && t.dim() == 1 && t.is_contiguous() && t.size(0) == n &&
               n < kMaxCall,
           std::string(name) + " must be a contiguous int32 vector on the page table's device, one entry per sequence "
                               "of the call (fewer than 65536)");
  return t.data_ptr<int>();
}

// storage [planes, pages, page_size, ...]: pages whole and contiguous, planes and pages anywhere.
Storage check_storage(at::Tensor& t, int64_t pages, int64_t page_size, const at::Device& device) {
  refuse_gradients({&t}, "moving pages");
  RC_CHECK(t.device() == device && t.dim() >= 3 && t.size(1) == pages && t.size(2) == page_size,
           "storage must be [planes, pages, page_size, ...] on the page table's device");
  const int64_t size = t.element_size();
  int64_t inner = 1;
  bool dense = true;
  for (int64_t d = t.dim() - 1; d >= 2; --d) {
    dense = dense && (t.stride(d) == inner || t.size(d) == 1);
    inner *= t.size(d);
  }
  const int64_t row = inner / page_size * size;
  RC_CHECK(dense && t.numel() > 0, "a page of the storage must be contiguous");
  RC_CHECK(row % 16 == 0 && (t.stride(0) * size) % 16 == 0 && (t.stride(1) * size) % 16 == 0 &&
               reinterpret_cast<uintptr_t>(t.data_ptr()) % 16 == 0 && row < (1 << 30) && t.size(0) < (1 << 24),
           "the storage's token rows must be 16-byte multiples");
  RC_CHECK((pages == 1 || t.stride(1) >= inner) && (t.size(0) == 1 || t.stride(0) >= inner),
           "the storage's pages overlap");
  return {static_cast<char*>(t.data_ptr()), t.stride(0) * size, t.stride(1) * size, static_cast<int>(t.size(0)),
          inner * size, static_cast<int>(row)};
}

// sides: [planes, pages, ...], pages whole, contiguous and of 8-byte words, planes anywhere.
Sides check_sides(const std::vector<at::Tensor>& tensors, int64_t pages, const at::Device& device) {
  RC_CHECK(tensors.size() <= kMostSides, "at most " + std::to_string(kMostSides) + " tensors beside the storage");
  Sides sides{};
  for (const at::Tensor& t : tensors) {
    refuse_gradients({&t}, "moving pages");
    RC_CHECK(t.device() == device && t.dim() >= 2 && t.size(1) == pages && t.numel() > 0,
             "a tensor beside the storage must be [planes, pages, ...] on the page table's device");
    const int64_t size = t.element_size();
    int64_t inner = 1;
    bool dense = true;
    for (int64_t d = t.dim() - 1; d >= 2; --d) {
      dense = dense && (t.stride(d) == inner || t.size(d) == 1);
      inner *= t.size(d);
    }
    RC_CHECK(dense && (inner * size) % 8 == 0 && inner * size < (1ll << 31) && reinterpret_cast<uintptr_t>(t.data_ptr()) % 8 == 0 &&
                 (t.stride(0) * size) % 8 == 0 && (t.stride(1) * size) % 8 == 0 && (pages == 1 || t.stride(1) >= inner) &&
                 (t.size(0) == 1 || t.stride(0) >= inner) && t.size(0) < (1 << 24),
             "pages of a tensor beside the storage must be contiguous, apart and multiples of 8 bytes");
    sides.at[sides.count++] = {static_cast<char*>(t.data_ptr()), t.stride(0) * size, t.stride(1) * size, static_cast<int>(t.size(0)),
                               static_cast<int>(inner * size / 8)};
  }
  return sides;
}

int move_grid(int device) { return sm_count(device) * 8; }

}  // namespace pagetable

using pagetable::State;

void pages_allocate(at::Tensor& state, int64_t pages, int64_t seqs_held, int64_t page_size, const at::Tensor& seqs,
                    const at::Tensor& new_lens, const c10::optional<at::Tensor>& status) {
  const State s = pagetable::check_state(state, pages, seqs_held, page_size);
  const int64_t n = seqs.numel();
  const int* ids = pagetable::check_list(seqs, state.device(), n, "seqs");
  const int* to = pagetable::check_list(new_lens, state.device(), n, "lens");
  if (n == 0) return;
  c10::cuda::CUDAGuard guard(state.device());
  cudaStream_t stream = c10::cuda::getCurrentCUDAStream(state.get_device()).stream();
  at::Tensor scratch = at::empty({s.pages + n + 1 + s.seqs}, state.options());
  int* list = scratch.data_ptr<int>();
  paged::launch(pagetable::allocate_kernel, dim3(1), pagetable::kPlanThreads, 0, 0, stream, s, ids, to, static_cast<int>(n), list,
                                                                       list + s.pages, list + s.pages + n + 1,
                                                                       status_ptr(status));
  written(state);
}

void pages_fork(at::Tensor& state, int64_t pages, int64_t seqs_held, int64_t page_size, const at::Tensor& parents,
                const at::Tensor& children, const at::Tensor& at_lens, at::Tensor& storage,
                const c10::optional<at::Tensor>& status, const std::vector<at::Tensor>& sides) {
  const State s = pagetable::check_state(state, pages, seqs_held, page_size);
  const int64_t n = parents.numel();
  const int* from = pagetable::check_list(parents, state.device(), n, "parents");
  const int* to = pagetable::check_list(children, state.device(), n, "children");
  const int* len = pagetable::check_list(at_lens, state.device(), n, "lens");
  const pagetable::Storage st = pagetable::check_storage(storage, s.pages, page_size, state.device());
  const pagetable::Sides beside = pagetable::check_sides(sides, s.pages, state.device());
  if (n == 0) return;
  c10::cuda::CUDAGuard guard(state.device());
  cudaStream_t stream = c10::cuda::getCurrentCUDAStream(state.get_device()).stream();
  at::Tensor scratch = at::empty({1 + 3 * n + s.pages + s.seqs}, state.options());
  int* p = scratch.data_ptr<int>();
  const pagetable::Plan plan{p, p + 1, p + 1 + n, p + 1 + 2 * n};
  int* list = p + 1 + 3 * n;
  paged::launch(pagetable::fork_plan_kernel, dim3(1), pagetable::kPlanThreads, 0, 0, stream, s, from, to, len, static_cast<int>(n), list,
                                                                        list + s.pages, plan, status_ptr(status));
  paged::launch(beside.count > 0 ? pagetable::fork_kernel<true> : pagetable::fork_kernel<false>, dim3(pagetable::move_grid(state.get_device())), pagetable::kMoveThreads, 0, 0, stream,
      s, st, beside, from, to, len, static_cast<int>(n), plan, status_ptr(status));
  written(state);
  written(storage);
  for (const at::Tensor& t : sides) written(t);
}

void pages_release(at::Tensor& state, int64_t pages, int64_t seqs_held, int64_t page_size, const at::Tensor& seqs,
                   const c10::optional<at::Tensor>& status) {
  const State s = pagetable::check_state(state, pages, seqs_held, page_size);
  const int64_t n = seqs.numel();
  const int* ids = pagetable::check_list(seqs, state.device(), n, "seqs");
  if (n == 0) return;
  c10::cuda::CUDAGuard guard(state.device());
  cudaStream_t stream = c10::cuda::getCurrentCUDAStream(state.get_device()).stream();
  const int64_t blocks = (n * s.width + pagetable::kMoveThreads - 1) / pagetable::kMoveThreads;
  const int grid = static_cast<int>(std::min<int64_t>(blocks, pagetable::move_grid(state.get_device())));
  paged::launch(pagetable::release_kernel, dim3(grid), pagetable::kMoveThreads, 0, 0, stream, s, ids, static_cast<int>(n), status_ptr(status));
  written(state);
}

// Returns an int32 tensor of one entry: the pages in use, which after the call are pages 0 .. in_use.
at::Tensor pages_compact(at::Tensor& state, int64_t pages, int64_t seqs_held, int64_t page_size, at::Tensor& storage,
                         const c10::optional<at::Tensor>& status, const std::vector<at::Tensor>& sides) {
  const State s = pagetable::check_state(state, pages, seqs_held, page_size);
  const pagetable::Storage st = pagetable::check_storage(storage, s.pages, page_size, state.device());
  const pagetable::Sides beside = pagetable::check_sides(sides, s.pages, state.device());
  c10::cuda::CUDAGuard guard(state.device());
  cudaStream_t stream = c10::cuda::getCurrentCUDAStream(state.get_device()).stream();
  at::Tensor scratch = at::empty({1 + 3 * s.pages}, state.options());
  at::Tensor in_use = at::empty({1}, state.options());
  int* p = scratch.data_ptr<int>();
  const pagetable::Plan plan{p, p + 1, p + 1 + s.pages, nullptr};
  int* place = p + 1 + 2 * static_cast<int64_t>(s.pages);
  paged::launch(pagetable::compact_plan_kernel, dim3(1), pagetable::kPlanThreads, 0, 0, stream, s, place, plan, in_use.data_ptr<int>());
  paged::launch(beside.count > 0 ? pagetable::compact_kernel<true> : pagetable::compact_kernel<false>, dim3(pagetable::move_grid(state.get_device())), pagetable::kMoveThreads, 0, 0, stream,
      s, st, beside, place, in_use.data_ptr<int>(), plan, status_ptr(status));
  written(state);
  written(storage);
  for (const at::Tensor& t : sides) written(t);
  return in_use;
}

// Pages source[i] -> target[i] in every plane, all of them or their first rows[i] rows; entries of -1 and -1 are skipped.
void pages_copy(at::Tensor& storage, const at::Tensor& source, const at::Tensor& target,
                const c10::optional<at::Tensor>& rows, const c10::optional<at::Tensor>& status) {
  RC_CHECK(storage.is_cuda() && storage.dim() >= 3, "storage must be a CUDA tensor [planes, pages, page_size, ...]");
  const pagetable::Storage st =
      pagetable::check_storage(storage, storage.size(1), storage.size(2), storage.device());
  const int64_t n = source.numel();
  const int* from = pagetable::check_list(source, storage.device(), n, "source");
  const int* to = pagetable::check_list(target, storage.device(), n, "target");
  const int* part = rows.has_value() ? pagetable::check_list(*rows, storage.device(), n, "rows") : nullptr;
  if (n == 0) return;
  c10::cuda::CUDAGuard guard(storage.device());
  cudaStream_t stream = c10::cuda::getCurrentCUDAStream(storage.get_device()).stream();
  paged::launch(pagetable::copy_kernel, dim3(pagetable::move_grid(storage.get_device())), pagetable::kMoveThreads, 0, 0, stream,
      st, static_cast<int>(storage.size(1)), from, to, part, static_cast<int>(n), status_ptr(status));
  written(storage);
}

}  // namespace rc
