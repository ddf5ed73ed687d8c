// Attention of many query rows (chunks, prompts) over a paged cache on tcgen05, for sm_100a: out = softmax(scale Q K^T) V
// with Q, K, V in bf16 or fp16, head_dim 64 or 128, scores, statistics and outputs accumulated in FP32.
//
// What bounds it: the tensor core and the exponentials. A tile of 128 rows x 128 keys (head_dim 128) is 8.4 MFLOP, 1,024
// cycles of an SM's tcgen05 rate, and 16,384 exponentials, 1,024 cycles of its 16 a cycle, so the two have to run at the
// same time. Measured: 3,700 cycles for a pair of tiles over a whole launch, the tensor pipe busy for 56 % of them
// (counters, 2,340 tokens over 23,400 keys); 4,680 tokens over 23,400 keys of 12 heads 594 us in runs of three calls (1,130
// TFLOP/s) and 656 us in one of seconds (1,025), where the card's power limit binds too (993 W, 1.64 GHz): what saves energy
// is what helps then (exponentials by a polynomial on the FMA pipe cost 2 to 5 %; items out of step with each other 15 to
// 20 %).
//
// A CTA works on 256 rows as two tiles of 128 that share every K and V block. Rows are (query, head of the group),
// query-major, so grouped heads share the loads of their KV head. 384 threads:
//   warps 0-3, 4-7  softmax of tile 0, 1: a thread owns a row (TMEM lane). S comes from TMEM, the running maximum moves
//                   only when it grows by more than 8 (log2; then the row of O is rescaled in TMEM), P goes back to TMEM
//                   over S, where the P V product reads it as its A operand, in two halves of 64 keys: the product over
//                   the first runs during the exponentials of the second.
//   warps 8, 9      TMA: K blocks into a ring of 3, V blocks into a ring of 2. One box per page (or part of it).
//   warp 10         one thread issues the products, in the order O_0 += P_0 V', S_0 = Q_0 K, O_1 += P_1 V', S_1 = Q_1 K
//                   (V' of the block before), without a break between one item and the next.
//   warp 11         gathers the rows of Q with cp.async into the swizzled layout (any group size and strides).
// V is read as it lies in the pages (keys x channels: an MN-major B operand), no transposed copy exists.
// TMEM: S_g at column 128 g (P_g in its first 64), O_g at 256 + 128 g.
//
// Twin form, up to 128 rows: both tiles hold the same rows, tile 0 takes the even blocks of keys and tile 1 the odd ones,
// so that twice the keys are in flight; the tiles are joined at the end through shared memory. 16 sessions x 16 tokens over
// 4,096 keys (32 / 8 heads): 49 us, 67.8 us with the second tile idle, 89.9 us on mma.sync.
//
// Work: an item is 256 (twin: 128) rows of one sequence and KV head with the tiles that they see.
//   direct   a cluster of 1 to 16 CTAs per item, each with an even part of its tiles; they join through distributed shared
//            memory. One launch, no workspace: for work that a wave or two holds.
//   planned  a plan kernel lists the items on the device (the lengths never leave it) and deals them out: whole rounds of
//            one item per SM as long as no SM gets more than its share of all tiles, so that neighbours read the same keys
//            at the same time; then the rest, cut like one line so that every SM ends with its share. An item that is cut
//            leaves FP32 parts, which a third kernel joins in order. Plan, cut items and join cost about 25 us.
//
// Every wait is bounded (2 s): on expiry a status is recorded, the roles stop, the products in flight are drained and TMEM
// is freed.
#include <ATen/ATen.h>
#include <c10/cuda/CUDAGuard.h>
#include <c10/cuda/CUDAStream.h>

#include <algorithm>
#include <string>
#include <type_traits>

#include "attend.cuh"

namespace rc {
namespace paged {

constexpr int kTile = 128;      // keys of a block, rows of a tile
constexpr int kItemRows = 256;  // rows of an item: two tiles
constexpr int kChunkThreads = 384;
constexpr int kKStages = 3;
// Register split (setmaxnreg): the launch holds kLaunchRegs a thread (checked on the host); the third warpgroup gives up
// registers for the softmax warpgroups, which hold a row of 128 scores. Spilled at that cap (bytes stored and read, 128
// channels): planned form 8 and 56, direct 36 and 184, twin 40 and 240.
constexpr int kLaunchRegs = 168;
constexpr int kSoftmaxRegs = 208;
constexpr int kRoleRegs = 88;
static_assert(2 * kSoftmaxRegs + kRoleRegs == 3 * kLaunchRegs, "register split must equal the launch's registers");
constexpr float kRescale = 8.0f;  // log2 units

template <int D, bool kTwin>
struct ChunkShape {
  static constexpr int q_tiles = kTwin ? 1 : 2;
  static constexpr int v_stages = kTwin ? 3 : 2;
  static constexpr int rows = q_tiles * kTile;  // of an item
  static constexpr int boxes = D / 64;
  static constexpr int box_bytes = kTile * 128;
  static constexpr int tile_bytes = boxes * box_bytes;
  static constexpr int q_off = 0;
  static constexpr int k_off = q_off + q_tiles * tile_bytes;
  static constexpr int v_off = k_off + kKStages * tile_bytes;
  static constexpr int bar_off = v_off + v_stages * tile_bytes;
  static constexpr int bytes = bar_off + 256 + 1024;  // + barriers, alignment slack
  static constexpr int ml_off = kItemRows * D * 4;    // at the end, clustered: rows of FP32 from 0, then maxima and sums
  static constexpr int scratch_off = ml_off + kItemRows * 8;  // weights of a share's rows and parts, places of its rows
  static_assert(scratch_off + kItemRows * 4 + kItemRows * 8 <= bar_off, "the rows fit where the operands were");
  static_assert(bytes <= 227 * 1024, "shared memory of one CTA");
};

struct Item {  // 32 bytes
  int seq, head, row_tile, tiles;
  int q_first, q_len, kv_len, start;  // start: its place in the line (items that are not dealt out whole)
};

struct Plan {
  int* head;   // [0] items, [1] whole rounds
  int* cut;    // [ctas + 1]: the line's cuts
  int* first;  // [ctas]: the item in which each CTA's part of the line begins
  int* base;   // [seqs]: first item of each sequence
  Item* items;
};

struct Chunk {
  Args a;
  Plan plan;
  float* part_o;   // [2 * ctas, 256, D]
  float* part_ml;  // [2 * ctas, 256, 2]
  int ctas;
  int cluster;     // CTAs of an item (the direct form)
  int row_tiles;   // of a sequence and KV head, at most
  int most_items;  // room for items
};

// New tokens of a sequence (returned), where they begin and how many keys it has.
__device__ __forceinline__ int sequence(const Args& a, int s, int* q_first, int* kv_len) {
  *kv_len = held_keys(a, s);
  return new_tokens(a, s, q_first);
}

// Queries of a row tile of a sequence: [first, end).
struct RowQueries {
  int first, end;
  __device__ __forceinline__ RowQueries(const Args& a, int row_tile, int q_len, int item_rows = kItemRows) {
    first = row_tile * item_rows / a.group;
    end = min(q_len, (row_tile * item_rows + item_rows - 1) / a.group + 1);
  }
};

__device__ __forceinline__ int tiles_of(const Args& a, const Item& item, const RowQueries& rows) {
  return max(1, TileRange<kTile>(Sight(a, item.kv_len, item.q_len), rows.first, rows.end).count());
}

__global__ void __launch_bounds__(kPlanThreads) chunk_plan_kernel(const __grid_constant__ Chunk p) {
  __shared__ int warp_sums[32];
  let_later();
  after_earlier();
  const Args& a = p.a;
  const Plan& plan = p.plan;
  auto row_tiles = [&](int q_len) {
    return static_cast<int>(min(static_cast<int64_t>(p.row_tiles), (static_cast<int64_t>(q_len) * a.group + kItemRows - 1) / kItemRows));
  };
  int items = 0;
  for (int s0 = 0; s0 < a.seqs; s0 += kPlanThreads) {
    const int s = s0 + threadIdx.x;
    int n = 0, q_first, kv_len;
    if (s < a.seqs) {
      n = row_tiles(sequence(a, s, &q_first, &kv_len)) * a.kv_heads;
      report_rows(a, s);
    }
    int total;
    const int before = block_scan(n, warp_sums, &total);
    if (s < a.seqs) plan.base[s] = items + before;
    items += total;
  }
  items = min(items, p.most_items);  // cu_q that runs backwards could name rows more than once
  __syncthreads();
  int sum = 0;
  for (int i = threadIdx.x; i < items; i += kPlanThreads) {
    int lo = 0, hi = a.seqs - 1;
    while (lo < hi) {
      const int mid = (lo + hi + 1) >> 1;
      if (plan.base[mid] <= i) lo = mid;
      else hi = mid - 1;
    }
    Item item;
    item.seq = lo;
    item.q_len = sequence(a, lo, &item.q_first, &item.kv_len);
    const int n = row_tiles(item.q_len), local = i - plan.base[lo];
    item.head = local / n;
    item.row_tile = n - 1 - (local - item.head * n);  // the rows that see most come first
    const RowQueries rows(a, item.row_tile, item.q_len);
    item.tiles = tiles_of(a, item, rows);
    item.start = 0;
    plan.items[i] = item;
    sum += item.tiles;
  }
  int all;
  block_scan(sum, warp_sums, &all);
  const int share = (all + p.ctas - 1) / p.ctas;
  // whole rounds: 3 % above the share is less than cutting the last items costs
  const int limit = share + share / 32;
  const int c = threadIdx.x;
  int whole = 0, rounds = 0;
  for (;;) {
    const int at = rounds * p.ctas;
    if (at + p.ctas > items) break;
    const int next = c < p.ctas ? whole + plan.items[at + c].tiles : 0;
    if (!__syncthreads_and(next <= limit)) break;
    whole = next;
    ++rounds;
  }
  const int from = rounds * p.ctas;
  int line = 0;
  for (int i0 = from; i0 < items; i0 += kPlanThreads) {
    const int i = i0 + threadIdx.x;
    const int n = i < items ? plan.items[i].tiles : 0;
    int total;
    const int before = block_scan(n, warp_sums, &total);
    if (i < items) plan.items[i].start = line + before;
    line += total;
  }
  __syncthreads();
  int wanted_all;
  const int before = block_scan(c < p.ctas ? max(0, share - whole) : 0, warp_sums, &wanted_all);
  // if whole rounds went over the share, the last CTA takes what is left
  if (c <= p.ctas) {
    const int cut = c == p.ctas ? line : min(line, before);
    plan.cut[c] = cut;
    if (c < p.ctas) {
      int lo = from, hi = items - 1;
      while (lo < hi) {
        const int mid = (lo + hi + 1) >> 1;
        if (plan.items[mid].start <= cut) lo = mid;
        else hi = mid - 1;
      }
      plan.first[c] = lo;
    }
  }
  if (c == 0) {
    plan.head[0] = items;
    plan.head[1] = rounds;
  }
}

// What the plan deals to a CTA: its whole rounds, then its part [begin, end) of the line.
struct Share {
  int rounds, items, first, begin, end;
  Share() = default;
  __device__ __forceinline__ Share(const Chunk& p, int cta)
      : rounds(p.plan.head[1]), items(p.plan.head[0]), first(p.plan.first[cta]), begin(p.plan.cut[cta]), end(p.plan.cut[cta + 1]) {}
};

// A CTA's n-th piece of work. Direct form: the only one, rank `rank` of `cluster` of the item that the block index names.
struct Segment {
  Item item;
  int t0, t1;
  bool starts, ends;  // holds the item's first, last tile

  __device__ __forceinline__ bool load(const Chunk& p, const Share& share, int cta, int n) {
    const bool whole = n < share.rounds;
    const int i = whole ? n * p.ctas + cta : share.first + n - share.rounds;
    if (!whole && (share.begin >= share.end || i >= share.items)) return false;
    const int4* src = reinterpret_cast<const int4*>(p.plan.items + i);
    const int4 x = src[0], y = src[1];
    item = {x.x, x.y, x.z, x.w, y.x, y.y, y.z, y.w};
    if (!whole && item.start >= share.end) return false;
    t0 = whole ? 0 : max(0, share.begin - item.start);
    t1 = whole ? item.tiles : min(item.tiles, share.end - item.start);
    starts = t0 == 0;
    ends = t1 == item.tiles;
    return t0 < t1;
  }

  __device__ __forceinline__ bool direct(const Chunk& p, int block, int item_rows) {
    const int index = block / p.cluster, rank = block - index * p.cluster, each = p.a.kv_heads * p.row_tiles;
    item.seq = index / each;
    item.head = (index - item.seq * each) / p.row_tiles;
    item.row_tile = p.row_tiles - 1 - index % p.row_tiles;  // the rows that see most come first
    item.q_len = sequence(p.a, item.seq, &item.q_first, &item.kv_len);
    item.start = 0;
    if (static_cast<int64_t>(item.row_tile) * item_rows >= static_cast<int64_t>(item.q_len) * p.a.group) return false;
    item.tiles = tiles_of(p.a, item, RowQueries(p.a, item.row_tile, item.q_len, item_rows));
    t0 = item.tiles * rank / p.cluster;
    t1 = item.tiles * (rank + 1) / p.cluster;
    starts = t0 == 0;
    ends = t1 == item.tiles;
    return true;
  }
};

// -- two FP32 numbers at a time ---------------------------------------------------------------------------------------

__device__ __forceinline__ uint64_t pair(float x, float y) {
  uint64_t r;
  asm("mov.b64 %0, {%1, %2};" : "=l"(r) : "f"(x), "f"(y));
  return r;
}
__device__ __forceinline__ void unpair(uint64_t v, float& x, float& y) {
  asm("mov.b64 {%0, %1}, %2;" : "=f"(x), "=f"(y) : "l"(v));
}
__device__ __forceinline__ uint64_t fma2(uint64_t a, uint64_t b, uint64_t c) {
  uint64_t r;
  asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(r) : "l"(a), "l"(b), "l"(c));
  return r;
}
__device__ __forceinline__ uint64_t add2(uint64_t a, uint64_t b) {
  uint64_t r;
  asm("add.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b));
  return r;
}
__device__ __forceinline__ float max3(float a, float b, float c) {
  float r;
  asm("max.f32 %0, %1, %2, %3;" : "=f"(r) : "f"(a), "f"(b), "f"(c));
  return r;
}

// Exponentials of half a row: 64 raw scores become 32 pairs of P; their sum is added to `sum`. kMax: the maximum of the
// whole row (this half and `other`) is found on the way, two steps of it after every pair.
template <typename T, bool kMax>
__device__ __forceinline__ void softmax_half(const uint32_t (&r)[64], const uint32_t (&other)[64], float scale_log2, float neg_m,
                                             uint32_t (&pk)[32], float& sum, float& top) {
  const uint64_t scale2 = pair(scale_log2, scale_log2), m2 = pair(neg_m, neg_m);
  uint64_t sums[2] = {0, 0};
  float m[4] = {-INFINITY, -INFINITY, -INFINITY, -INFINITY};
#pragma unroll
  for (int c = 0; c < 32; ++c) {
    float p0, p1;
    unpair(fma2(pair(__uint_as_float(r[2 * c]), __uint_as_float(r[2 * c + 1])), scale2, m2), p0, p1);
    p0 = exp2_approx(p0);
    p1 = exp2_approx(p1);
    if (kMax) {
      m[c & 1] = max3(m[c & 1], __uint_as_float(r[2 * c]), __uint_as_float(r[2 * c + 1]));
      m[2 + (c & 1)] = max3(m[2 + (c & 1)], __uint_as_float(other[2 * c]), __uint_as_float(other[2 * c + 1]));
    }
    sums[c & 1] = add2(sums[c & 1], pair(p0, p1));
    pk[c] = pack2<T>(p0, p1);
  }
  float a, b;
  unpair(add2(sums[0], sums[1]), a, b);
  sum += a + b;
  if (kMax) top = fmaxf(max3(m[0], m[1], m[2]), m[3]);
}

__device__ __forceinline__ float row_max(const uint32_t (&r)[2][64]) {
  float m[8];
#pragma unroll
  for (int k = 0; k < 8; ++k) m[k] = fmaxf(__uint_as_float(r[0][k]), __uint_as_float(r[1][k]));
#pragma unroll
  for (int c = 8; c < 64; c += 8)
#pragma unroll
    for (int k = 0; k < 8; ++k) m[k] = max3(m[k], __uint_as_float(r[0][c + k]), __uint_as_float(r[1][c + k]));
  return max3(max3(m[0], m[1], m[2]), max3(m[3], m[4], m[5]), fmaxf(m[6], m[7]));
}

// Bits [0, n) of a word.
__device__ __forceinline__ uint32_t low_bits(int n) { return n <= 0 ? 0u : n >= 32 ? 0xffffffffu : (1u << n) - 1u; }

// Scores outside [from, high) and [0, sink) of the tile become minus infinity: 32 columns at a time as bits of a word, and
// not at all where no row of the warp has one. kHalf: 0 or 1.
template <int kHalf>
__device__ __forceinline__ void mask_half(uint32_t (&r)[64], int from, int high, int sink) {
#pragma unroll
  for (int w = 0; w < 2; ++w) {
    const int first = 64 * kHalf + 32 * w;
    const uint32_t seen = low_bits(high - first) & (~low_bits(from - first) | low_bits(sink - first));
    if (__all_sync(0xffffffffu, seen == 0xffffffffu)) continue;
#pragma unroll
    for (int e = 0; e < 32; ++e)
      if ((seen & (1u << e)) == 0) r[32 * w + e] = __float_as_uint(-INFINITY);
  }
}

// A whole sector in one store: a thread writes its own row, so narrower stores would each touch a sector of their own.
__device__ __forceinline__ void store_32_bytes(void* dst, const uint32_t* v) {
  asm volatile("st.global.v8.b32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8};" ::"l"(dst), "r"(v[0]), "r"(v[1]), "r"(v[2]),
               "r"(v[3]), "r"(v[4]), "r"(v[5]), "r"(v[6]), "r"(v[7])
               : "memory");
}

// One thread of a converged warp (elect.sync: the compiler then knows that what it issues is uniform).
__device__ __forceinline__ bool elect_one() {
  uint32_t one;
  asm volatile(
      "{\n\t.reg .pred p;\n\t"
      "elect.sync _|p, 0xffffffff;\n\t"
      "selp.u32 %0, 1, 0, p;\n\t}"
      : "=r"(one));
  return one != 0;
}

// Shared-memory descriptor of an MN-major operand in the 128-byte swizzle: blocks of 64 channels x 8 keys (1,024 bytes),
// `block_bytes` between the blocks of 64 channels (leading offset), 1,024 bytes between groups of 8 keys (stride offset).
__device__ __forceinline__ uint64_t sw128_mnmajor_desc(uint32_t smem_addr, uint32_t block_bytes) {
  uint64_t desc = 0;
  desc |= static_cast<uint64_t>((smem_addr >> 4) & 0x3FFFu);
  desc |= static_cast<uint64_t>((block_bytes >> 4) & 0x3FFFu) << 16;
  desc |= static_cast<uint64_t>(1024u >> 4) << 32;
  desc |= static_cast<uint64_t>(1u) << 46;
  desc |= static_cast<uint64_t>(2u) << 61;
  return desc;
}

// The clustered end: the rows that the CTAs of a cluster hold in shared memory (row-major FP32, 16-byte chunks turned by
// the row, maxima and sums at ml_off) become the item's output, each CTA an even share of the rows. A thread per row and
// part finds the part's weight and where the row goes (scratch_off: weights, then places); then a warp or half per row adds
// the parts, a vector of four channels a lane, kRows rows and kParts parts of it in flight, the first of them asked for
// before the weights are (remote shared memory takes most of a microsecond; more than eight vectors spill, and a spilled
// load waits). 256 threads; `cluster` is a power of two up to 16. Weights found again for each vector took 10 us of a 45 us
// call of clusters of two; so, 3 us.
template <typename T, int D, int kRows, int kParts>
__device__ __forceinline__ void join_cluster(const Args& a, const Item& item, uint8_t* smem, int ml_off, int scratch_off,
                                             int item_rows, int rank, int cluster) {
  constexpr int kLanes = D / 4, kStep = 8 * (32 / kLanes);
  const int packed0 = item.row_tile * item_rows;
  const int rows = static_cast<int>(min(static_cast<int64_t>(item_rows), static_cast<int64_t>(item.q_len) * a.group - packed0));
  const int share = (rows + cluster - 1) / cluster, first = rank * share, count = min(share, rows - first), last = max(count, 1) - 1;
  float* weights = reinterpret_cast<float*>(smem + scratch_off);                     // [share][cluster]
  int64_t* places = reinterpret_cast<int64_t*>(smem + scratch_off + kItemRows * 4);  // [share]

  const int chunk = threadIdx.x % kLanes;
  float4 x[kRows][kParts];
  const auto load = [&](int r0, int c0) {
#pragma unroll
    for (int i = 0; i < kRows; ++i) {
      const int row = first + min(r0 + i * kStep, last);
      const uint32_t at = smem_u32(smem) + (row * kLanes + (chunk ^ (row & 15))) * 16;
#pragma unroll
      for (int j = 0; j < kParts; ++j) x[i][j] = load_cluster_4(cluster_addr_of(at, c0 + j));
    }
  };
  int r0 = threadIdx.x / kLanes, c0 = 0;
  {
    const int at = threadIdx.x / cluster, part = threadIdx.x % cluster, row = first + min(at, last);
    const float2 ml = load_cluster_2(cluster_addr(reinterpret_cast<const float2*>(smem + ml_off) + row, part));
    load(r0, c0);
    float top = ml.x;
    for (int i = cluster >> 1; i > 0; i >>= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, i));
    const float weight = exp2_approx(ml.x - base_of(top));
    float sum = weight * ml.y;
    for (int i = cluster >> 1; i > 0; i >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, i);
    // (-1: no key seen there, nor, perhaps, anything written)
    weights[threadIdx.x] = ml.x == -INFINITY && ml.y == 0.0f ? -1.0f : weight / sum;
    if (part == 0 && at < count) {
      const int query = (packed0 + row) / a.group, h = item.head * a.group + packed0 + row - query * a.group;
      const int64_t token = item.q_first + query;
      places[at] = token * a.out_token + h * a.out_head;
      if (a.lse != nullptr) a.lse[token * a.heads + h] = log_sum(top, sum);
    }
  }
  asm volatile("bar.sync 3, 256;" ::: "memory");
  float4 acc[kRows] = {};
  while (r0 < count) {
#pragma unroll
    for (int i = 0; i < kRows; ++i)
#pragma unroll
      for (int j = 0; j < kParts; ++j) {
        const float w = weights[min(r0 + i * kStep, last) * cluster + c0 + j];
        if (w < 0.0f) continue;
        acc[i].x = fmaf(w, x[i][j].x, acc[i].x);
        acc[i].y = fmaf(w, x[i][j].y, acc[i].y);
        acc[i].z = fmaf(w, x[i][j].z, acc[i].z);
        acc[i].w = fmaf(w, x[i][j].w, acc[i].w);
      }
    c0 += kParts;
    if (c0 == cluster) {
#pragma unroll
      for (int i = 0; i < kRows; ++i) {
        if (r0 + i * kStep < count)
          *reinterpret_cast<uint2*>(static_cast<T*>(a.out) + places[r0 + i * kStep] + chunk * 4) =
              make_uint2(pack2<T>(acc[i].x, acc[i].y), pack2<T>(acc[i].z, acc[i].w));
        acc[i] = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
      }
      c0 = 0;
      r0 += kRows * kStep;
    }
    if (r0 < count) load(r0, c0);
  }
}

template <typename T, int D, bool kDirect, bool kTwin>
__global__ void __launch_bounds__(kChunkThreads, 1)
    chunk_kernel(const __grid_constant__ PageMaps maps, const __grid_constant__ Chunk p) {
  using Shape = ChunkShape<D, kTwin>;
  static_assert(kDirect || !kTwin, "twin items are dealt out whole");
  extern __shared__ __align__(1024) uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  uint64_t* q_full = reinterpret_cast<uint64_t*>(smem + Shape::bar_off);
  uint64_t* q_empty = q_full + 1;
  uint64_t* k_full = q_empty + 1;         // [kKStages]
  uint64_t* k_empty = k_full + kKStages;  // [kKStages]
  uint64_t* v_full = k_empty + kKStages;  // [v_stages]
  uint64_t* v_empty = v_full + Shape::v_stages;
  uint64_t* s_full = v_empty + Shape::v_stages;  // [2] per tile
  uint64_t* p_full = s_full + 2;          // [4] per tile and half of the keys
  uint64_t* o_done = p_full + 4;          // [2]
  uint64_t* v_raw = o_done + 2;
  uint64_t* drained = v_raw + 1;
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(drained + 1);
  const Args& a = p.a;
  int* status = a.status;
  const int warp = __shfl_sync(0xffffffffu, threadIdx.x >> 5, 0), lane = threadIdx.x & 31;
  const int cta = blockIdx.x;
  Segment seg;

  let_later();
  if (threadIdx.x == 0) {
    mbar_init(q_full, 32);
    mbar_init(q_empty, 1);
    for (int b = 0; b < kKStages; ++b) {
      mbar_init(&k_full[b], 1);
      mbar_init(&k_empty[b], 1);
    }
    for (int b = 0; b < Shape::v_stages; ++b) {
      mbar_init(&v_full[b], 1);
      mbar_init(&v_empty[b], 1);
    }
    for (int g = 0; g < 2; ++g) {
      mbar_init(&s_full[g], 1);
      mbar_init(&p_full[2 * g], 4);
      mbar_init(&p_full[2 * g + 1], 4);
      mbar_init(&o_done[g], 1);
    }
    mbar_init(v_raw, 1);
    mbar_init(drained, 1);
    fence_barrier_init();
  }
  if (warp == 8 && lane == 0) {
    tma_prefetch_desc(&maps.k_wide);
    tma_prefetch_desc(&maps.v_wide);
  }
  after_earlier();
  if (kDirect && !seg.direct(p, cta, Shape::rows)) {  // the whole cluster
    if (threadIdx.x == 0 && seg.item.row_tile == 0) report_rows(a, seg.item.seq);
    return;
  }
  if (warp == 10) tmem_alloc(tmem_slot, 512);
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem_base = *tmem_slot;
  Share share{};
  if (!kDirect) share = Share(p, cta);
  auto next = [&](int n) { return kDirect ? n == 0 && seg.t0 < seg.t1 : seg.load(p, share, cta, n); };
  if (warp >= 8) {
    asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(kRoleRegs));
    if (warp < 10) {
      // ---------------- TMA: warp 8 streams K, warp 9 streams V ----------------
      const bool is_k = warp == 8;
      const int stages = is_k ? kKStages : Shape::v_stages;
      uint64_t* full = is_k ? k_full : v_full;
      uint64_t* empty = is_k ? k_empty : v_empty;
      uint8_t* ring = smem + (is_k ? Shape::k_off : Shape::v_off);
      const CUtensorMap* wide = is_k ? &maps.k_wide : &maps.v_wide;
      const CUtensorMap* step = is_k ? &maps.k_step : &maps.v_step;
      int stage = 0;
      uint32_t phase = 1, raw_phase = 0;
      bool ok = true;
      for (int n = 0; ok && next(n); ++n) {
        const RowQueries rows(a, seg.item.row_tile, seg.item.q_len, Shape::rows);
        const Sight sight(a, seg.item.kv_len, seg.item.q_len);
        const TileRange<kTile> range(sight, rows.first, rows.end);
        const int low = sight.low(sight.last(rows.first)), top = min(sight.last(rows.end - 1), seg.item.kv_len - 1);
        const int* table = a.table + seg.item.seq * a.table_row;
        for (int t = seg.t0; t < seg.t1; ++t) {
          const int first = range.tile(t) * kTile;
          const Boxes<kTile> boxes(a.tiling, first, seg.item.kv_len);
          int row = 0, page = -1;
          if (lane < boxes.count) page = boxes.page(table, a.pages, a.tiling, first, lane, &row, status);
          // rows of V that no query of the item sees become zeros (0 * NaN is NaN): this warp does it between the copy
          // and the products, so the block's bytes are counted on a barrier of its own
          const int from = low - first, high = top + 1 - first, sink = a.sinks - first;
          const bool clean = !is_k && (high < kTile || (from > 0 && sink < kTile));
          uint64_t* bar = clean ? v_raw : &full[stage];
          ok = __all_sync(0xffffffffu, mbar_wait_park(&empty[stage], phase, status, kTimeoutProducer));
          if (!ok) break;
          if (lane == 0) {
            if (boxes.count > 0) mbar_arrive_expect_tx(bar, boxes.count * boxes.rows * 128 * Shape::boxes);
            else mbar_arrive(bar);
          }
          __syncwarp();
          uint8_t* tile = ring + stage * Shape::tile_bytes;
          if (lane < boxes.count) {
            const CUtensorMap* map = boxes.rows == kTile ? wide : step;
#pragma unroll
            for (int b = 0; b < Shape::boxes; ++b)
              load_page_box(tile + lane * boxes.rows * 128 + b * Shape::box_bytes, map, bar, b * 64, row, seg.item.head, page);
          }
          if (clean) {
            ok = __all_sync(0xffffffffu, mbar_wait_park(v_raw, raw_phase, status, kTimeoutProducer));
            if (!ok) break;
            raw_phase ^= 1;
            for (int i = lane; i < kTile * Shape::boxes * 8; i += 32) {
              const int r = i / (Shape::boxes * 8), c = i % (Shape::boxes * 8);
              if (r >= high || (r < from && r >= sink))
                *reinterpret_cast<uint4*>(tile + (c >> 3) * Shape::box_bytes + r * 128 + (c & 7) * 16) = make_uint4(0, 0, 0, 0);
            }
            fence_proxy_async_smem();
            __syncwarp();
            if (lane == 0) mbar_arrive(&full[stage]);
          }
          if (++stage == stages) {
            stage = 0;
            phase ^= 1;
          }
        }
      }
    } else if (warp == 11) {
      // ---------------- Q rows: each lane finds where a few rows lie, then four lanes fetch a row 64 bytes at a time ------
      const int quarter = lane & 3, sub = lane >> 2;
      if (kDirect && lane == 0 && seg.item.row_tile == 0) report_rows(a, seg.item.seq);
      bool ok = true;
      for (int n = 0; ok && next(n); ++n) {
        constexpr int kPlaces = Shape::rows / 32;
        const int packed0 = seg.item.row_tile * Shape::rows;
        const T* place[kPlaces];
#pragma unroll
        for (int i = 0; i < kPlaces; ++i) {
          const int packed = packed0 + 32 * i + lane, query = packed / a.group;
          const int h = seg.item.head * a.group + packed - query * a.group;
          place[i] = query < seg.item.q_len
                         ? static_cast<const T*>(a.q) + static_cast<int64_t>(seg.item.q_first + query) * a.q_token + h * a.q_head
                         : nullptr;
        }
        if (n > 0) ok = __all_sync(0xffffffffu, mbar_wait_park(q_empty, (n - 1) & 1, status, kTimeoutGather));
        if (!ok) break;
#pragma unroll
        for (int i = 0; i < kPlaces; ++i) {
#pragma unroll
          for (int j = 0; j < 4; ++j) {
            const int r = 32 * i + 8 * j + sub;
            const uint64_t src = __shfl_sync(0xffffffffu, reinterpret_cast<uint64_t>(place[i]), 8 * j + sub);
            const int bytes = src != 0 ? 16 : 0;  // rows past the sequence are zeros
            const uint64_t from = src != 0 ? src + quarter * 16 : reinterpret_cast<uint64_t>(a.q);
            const uint32_t row = smem_u32(smem + Shape::q_off + (r >> 7) * Shape::tile_bytes) + (r & 127) * 128;
#pragma unroll
            for (int c = 0; c < D / 32; ++c) {
              const uint32_t dst = row + (c >> 1) * Shape::box_bytes + ((((c & 1) * 4 + quarter) ^ (r & 7)) << 4);
              asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst), "l"(bytes ? from + c * 64 : from), "r"(bytes)
                           : "memory");
            }
          }
        }
        asm volatile("cp.async.wait_all;" ::: "memory");
        fence_proxy_async_smem();
        mbar_arrive(q_full);
      }
    } else {
      // ---------------- products ----------------
      // One thread issues everything; per block it has 32 instructions to get out, so descriptors are built once per
      // operand tile and stepped by constants (the start address is in units of 16 bytes and never carries).
      if (elect_one()) {
        constexpr uint32_t kFormat = std::is_same<T, __nv_bfloat16>::value ? 1u : 0u;
        constexpr uint32_t idesc_s = make_idesc_f16(kTile, kTile, kFormat);
        constexpr uint32_t idesc_o = make_idesc_f16(kTile, D, kFormat) | (1u << 16);  // B is MN-major
        const uint64_t q_desc = sw128_kmajor_desc(smem_u32(smem + Shape::q_off));
        const uint64_t k_desc = sw128_kmajor_desc(smem_u32(smem + Shape::k_off));
        const uint64_t v_desc = sw128_mnmajor_desc(smem_u32(smem + Shape::v_off), Shape::box_bytes);
        bool ok = true;
        int it = 0;  // blocks so far
        int k_stage = 0, v_stage = 0;
        uint32_t k_phase = 0, v_phase = 0;
        bool was_first = false, was_last = false;  // the block before: whether it begins, ends its segment
        int last_block[2] = {0, 0};                // twin: each tile's last block
        auto issue_s = [&](int g) {
          if (!ok) return;
          const uint64_t ka = k_desc + k_stage * (Shape::tile_bytes >> 4), qg = q_desc + (kTwin ? 0 : g) * (Shape::tile_bytes >> 4);
#pragma unroll
          for (int kk = 0; kk < D / 16; ++kk) {
            constexpr uint32_t kBox = Shape::box_bytes >> 4;
            mma_f16(tmem_base + g * kTile, qg + (kk >> 2) * kBox + 2 * (kk & 3), ka + (kk >> 2) * kBox + 2 * (kk & 3), idesc_s,
                    kk > 0 ? 1u : 0u);
          }
          mma_commit(&s_full[g]);
        };
        auto issue_pv = [&](int g) {  // the block before, each half of its keys as soon as its P is there
          const uint64_t va = v_desc + v_stage * (Shape::tile_bytes >> 4);
#pragma unroll
          for (int half = 0; half < 2; ++half) {
            if (ok) ok = mbar_wait_park(&p_full[2 * g + half], (it - 1) & 1, status, kTimeoutMma);
            if (!ok) return;
            tc_fence_after();
#pragma unroll
            for (int kk = 4 * half; kk < 4 * half + 4; ++kk)
              mma_f16_ts(tmem_base + 256 + g * kTile, tmem_base + g * kTile + kk * 8, va + kk * (16 * 128 >> 4), idesc_o,
                         kk > 0 || !was_first ? 1u : 0u);
          }
          if (kTwin ? it - 1 == last_block[g] : was_last) mma_commit(&o_done[g]);
        };
        auto done_v = [&]() {
          if (ok) mma_commit(&v_empty[v_stage]);
          if (++v_stage == Shape::v_stages) {
            v_stage = 0;
            v_phase ^= 1;
          }
        };
        auto take_k = [&]() {
          if (ok) ok = mbar_wait_park(&k_full[k_stage], k_phase, status, kTimeoutMma);
          tc_fence_after();
        };
        auto done_k = [&]() {
          if (ok) mma_commit(&k_empty[k_stage]);
          if (++k_stage == kKStages) {
            k_stage = 0;
            k_phase ^= 1;
          }
        };
        auto take_v = [&]() {
          if (ok) ok = mbar_wait_park(&v_full[v_stage], v_phase, status, kTimeoutMma);
        };
        if (kTwin && next(0)) {
          // tile 0 takes the even blocks, tile 1 the odd ones, with the same rows: twice the keys in flight for few rows
          const int n = seg.t1 - seg.t0;
          last_block[0] = (n + 1) / 2 - 1;
          last_block[1] = n / 2 - 1;
          ok = mbar_wait_park(q_full, 0, status, kTimeoutMma);
          for (; it <= last_block[0] && ok; ++it) {
            was_first = it == 1;
            take_k();
            if (it > 0) {
              take_v();
              issue_pv(0);
              done_v();
            }
            issue_s(0);
            done_k();
            if (it > 0) {
              take_v();
              issue_pv(1);
              done_v();
            }
            if (it <= last_block[1]) {
              take_k();
              issue_s(1);
              done_k();
            }
          }
          was_first = it == 1;
          take_v();
          issue_pv(0);
          done_v();
          if (it - 1 <= last_block[1]) {
            take_v();
            issue_pv(1);
            done_v();
          }
          it = 0;  // nothing is left to do
        }
        for (int n = 0; !kTwin && ok && next(n); ++n) {
          for (int t = seg.t0; t < seg.t1 && ok; ++t) {
            // everything that can be waited for ahead of P is
            take_k();
            if (it > 0) {
              take_v();
              issue_pv(0);
            }
            if (ok && t == seg.t0) ok = mbar_wait_park(q_full, n & 1, status, kTimeoutMma);
            tc_fence_after();
            issue_s(0);
            if (it > 0) {
              issue_pv(1);
              done_v();
            }
            issue_s(1);
            done_k();
            if (ok && t + 1 == seg.t1) mma_commit(q_empty);
            ++it;
            was_first = t == seg.t0;
            was_last = t + 1 == seg.t1;
          }
        }
        if (it > 0) {
          take_v();
          issue_pv(0);
          issue_pv(1);
          done_v();
        }
        mma_commit(drained);
        (void)mbar_wait_park(drained, 0, nullptr, 0);
      }
      __syncwarp();
    }
  } else {
    // ---------------- softmax: warpgroup g owns tile g ----------------
    asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(kSoftmaxRegs));
    const int g = warp >> 2, quarter = warp & 3;
    const int row = quarter * 32 + lane;
    const uint32_t lanes = static_cast<uint32_t>(quarter * 32) << 16;
    const uint32_t s_col = tmem_base + g * kTile + lanes;
    const uint32_t o_col = tmem_base + 256 + g * kTile + lanes;
    bool ok = true;
    int it = 0;
    bool more = next(0);
    for (int n = 0; ok && more; ++n) {
      const int packed = seg.item.row_tile * Shape::rows + (kTwin ? 0 : g * kTile) + row;
      const int query = packed / a.group;
      const Sight sight(a, seg.item.kv_len, seg.item.q_len);
      const RowQueries rows(a, seg.item.row_tile, seg.item.q_len, Shape::rows);
      const TileRange<kTile> range(sight, rows.first, rows.end);
      const int last = min(sight.last(min(query, seg.item.q_len - 1)), seg.item.kv_len - 1);
      const int low = sight.low(last);
      float m_run = -INFINITY, l_run = 0.0f;  // of scale * log2(e) * s
      for (int t = seg.t0 + (kTwin ? g : 0); t < seg.t1 && ok; t += kTwin ? 2 : 1, ++it) {
        uint32_t r[2][64], pk[32];
        ok = __all_sync(0xffffffffu, mbar_wait_park(&s_full[g], it & 1, status, kTimeoutEpilogue));
        if (!ok) break;
        tc_fence_after();
        tmem_ld_32x32b_x64(s_col, r[0]);
        tmem_ld_32x32b_x64(s_col + 64, r[1]);
        tmem_wait_ld();
        const int first = range.tile(t) * kTile;
        const int high = last + 1 - first, from = low - first, sink = a.sinks - first;  // sees [from, high), [0, sink)
        const bool whole = __all_sync(0xffffffffu, high >= kTile && (from <= 0 || sink >= kTile));
        if (!whole) {
          mask_half<0>(r[0], from, high, sink);
          mask_half<1>(r[1], from, high, sink);
        }
        // The exponentials start with the maximum so far, and this block's is found next to them (they leave issue slots
        // for it). Only where it has grown by more than kRescale are they done again.
        if (t < seg.t0 + (kTwin ? 2 : 1)) m_run = row_max(r) * a.scale_log2;
        float neg_m = -base_of(m_run);
        float sum = 0.0f, mx;
        softmax_half<T, true>(r[0], r[1], a.scale_log2, neg_m, pk, sum, mx);
        mx *= a.scale_log2;
        const bool need = mx > m_run + kRescale;
        if (__any_sync(0xffffffffu, need)) {
          // O_g holds the blocks before this one: their products were issued before this block's S
          const float alpha = need ? exp2_approx(m_run - mx) : 1.0f;
#pragma unroll
          for (int c = 0; c < D; c += 16) {
            uint32_t o[16];
            tmem_ld_32x32b_x16(o_col + c, o);
            tmem_wait_ld();
#pragma unroll
            for (int e = 0; e < 16; ++e) o[e] = __float_as_uint(__uint_as_float(o[e]) * alpha);
            tmem_st_32x32b_x16(o_col + c, o);
          }
          l_run *= alpha;
          if (need) m_run = mx;
          neg_m = -base_of(m_run);
          tmem_ld_32x32b_x64(s_col, r[0]);
          tmem_wait_ld();
          if (!whole) mask_half<0>(r[0], from, high, sink);
          sum = 0.0f;
          softmax_half<T, false>(r[0], r[1], a.scale_log2, neg_m, pk, sum, mx);
        }
        tmem_st_32x32b_x32(s_col, pk);
        tmem_wait_st();
        tc_fence_before();
        __syncwarp();
        if (lane == 0) mbar_arrive(&p_full[2 * g]);
        softmax_half<T, false>(r[1], r[0], a.scale_log2, neg_m, pk, sum, mx);
        l_run += sum;
        tmem_st_32x32b_x32(s_col + 32, pk);
        tmem_wait_st();
        tc_fence_before();
        __syncwarp();
        if (lane == 0) mbar_arrive(&p_full[2 * g + 1]);
      }
      // the next piece of work is looked up before the stores of this one fill the memory pipe
      Segment after = seg;
      more = kDirect ? false : after.load(p, share, cta, n + 1);
      const bool none = kTwin && seg.t0 + g >= seg.t1;  // a twin without blocks
      if (ok && !none) ok = __all_sync(0xffffffffu, mbar_wait_park(&o_done[g], n & 1, status, kTimeoutEpilogue));
      if (kDirect && (kTwin || p.cluster > 1)) {
        if (ok && (!kTwin || seg.t0 + 1 - g < seg.t1))
          ok = __all_sync(0xffffffffu, mbar_wait_park(&o_done[1 - g], 0, status, kTimeoutEpilogue));
        tc_fence_after();
      }
      // Every product is done in those forms, so the operands' memory takes rows: 16-byte chunks turned against bank
      // conflicts, a row's maximum and sum behind them.
      float4* rows_at = reinterpret_cast<float4*>(smem) + (g * kTile + row) * (D / 4);
      float2* ml_at = reinterpret_cast<float2*>(smem + Shape::ml_off) + g * kTile + row;
      float keep = 1.0f, add = 0.0f;  // twin: weights of this tile's row and the other's
      if (kTwin) {
        if (g == 1) {
#pragma unroll
          for (int c0 = 0; c0 < D; c0 += 32) {
            uint32_t o[32];
            tmem_ld_32x32b_x32(o_col + c0, o);
            tmem_wait_ld();
#pragma unroll
            for (int c = 0; c < 32; c += 4)
              rows_at[((c0 + c) / 4) ^ (row & 15)] = make_float4(__uint_as_float(o[c]), __uint_as_float(o[c + 1]),
                                                                  __uint_as_float(o[c + 2]), __uint_as_float(o[c + 3]));
          }
          *ml_at = make_float2(m_run, l_run);
        }
        asm volatile("bar.sync 1, 256;" ::: "memory");
        if (g == 1) break;
        const float2 ml = ml_at[kTile];
        const float top = fmaxf(m_run, ml.x), use = base_of(top);
        keep = exp2_approx(m_run - use);
        add = ml.x == -INFINITY ? 0.0f : exp2_approx(ml.x - use);
        l_run = l_run * keep + add * ml.y;
        m_run = top;
      }
      // (twin) the row's columns from c0 joined with the other tile's
      auto join = [&](uint32_t (&o)[32], int c0) {
        if (!kTwin || add == 0.0f) return;
        const float4* other = rows_at + kTile * (D / 4);
#pragma unroll
        for (int c = 0; c < 32; c += 4) {
          const float4 x = other[((c0 + c) / 4) ^ (row & 15)];
          o[c] = __float_as_uint(fmaf(add, x.x, keep * __uint_as_float(o[c])));
          o[c + 1] = __float_as_uint(fmaf(add, x.y, keep * __uint_as_float(o[c + 1])));
          o[c + 2] = __float_as_uint(fmaf(add, x.z, keep * __uint_as_float(o[c + 2])));
          o[c + 3] = __float_as_uint(fmaf(add, x.w, keep * __uint_as_float(o[c + 3])));
        }
      };
      if (kDirect && p.cluster > 1) {
#pragma unroll
        for (int c0 = 0; c0 < D; c0 += 32) {
          uint32_t o[32];
          tmem_ld_32x32b_x32(o_col + c0, o);
          tmem_wait_ld();
          join(o, c0);
#pragma unroll
          for (int c = 0; c < 32; c += 4)
            rows_at[((c0 + c) / 4) ^ (row & 15)] = make_float4(__uint_as_float(o[c]), __uint_as_float(o[c + 1]),
                                                                __uint_as_float(o[c + 2]), __uint_as_float(o[c + 3]));
        }
        *ml_at = make_float2(m_run, l_run);
      } else if (ok) {
        tc_fence_after();
        const bool valid = query < seg.item.q_len, whole = seg.starts && seg.ends;
        const float inv = whole ? inverse(l_run) : 1.0f;
        const int64_t token = seg.item.q_first + query;
        const int h = seg.item.head * a.group + packed - query * a.group;
        const int64_t slot = (2 * static_cast<int64_t>(cta) + (seg.starts ? 1 : 0)) * kItemRows + g * kTile + row;
#pragma unroll
        for (int c0 = 0; c0 < D; c0 += 32) {
          uint32_t o[32];
          tmem_ld_32x32b_x32(o_col + c0, o);
          tmem_wait_ld();
          join(o, c0);
          if (valid && whole) {
            T* dst = static_cast<T*>(a.out) + token * a.out_token + h * a.out_head + c0;
            uint32_t w[16];
#pragma unroll
            for (int e = 0; e < 16; ++e) w[e] = pack2<T>(__uint_as_float(o[2 * e]) * inv, __uint_as_float(o[2 * e + 1]) * inv);
            if (a.out_sectors) {
              store_32_bytes(dst, w);
              store_32_bytes(dst + 16, w + 8);
            } else {
#pragma unroll
              for (int c = 0; c < 16; c += 4)
                *reinterpret_cast<uint4*>(dst + 2 * c) = make_uint4(w[c], w[c + 1], w[c + 2], w[c + 3]);
            }
          } else if (valid) {
            float* dst = p.part_o + slot * D + c0;
#pragma unroll
            for (int c = 0; c < 32; c += 8) store_32_bytes(dst + c, o + c);
          }
          __syncwarp();
        }
        tc_fence_before();  // the next item's products overwrite O after this warp's next arrival
        if (valid && whole && a.lse != nullptr)
          a.lse[token * a.heads + h] = log_sum(m_run, l_run);
        if (valid && !whole) *reinterpret_cast<float2*>(p.part_ml + slot * 2) = make_float2(m_run, l_run);
      }
      seg = after;
    }
  }

  if (kDirect && p.cluster > 1) {
    // CTAs without tiles have nothing to give; every CTA joins a part of the item's rows over all of them, in order.
    if (seg.t0 == seg.t1 && threadIdx.x < kItemRows)
      reinterpret_cast<float2*>(smem + Shape::ml_off)[threadIdx.x] = make_float2(-INFINITY, 0.0f);
    cluster_sync_all();
    if (threadIdx.x < kItemRows) {
      const int rank = cta % p.cluster;
      if (p.cluster >= 8) join_cluster<T, D, 1, 8>(a, seg.item, smem, Shape::ml_off, Shape::scratch_off, Shape::rows, rank, p.cluster);
      else if (p.cluster >= 4) join_cluster<T, D, 2, 4>(a, seg.item, smem, Shape::ml_off, Shape::scratch_off, Shape::rows, rank, p.cluster);
      else join_cluster<T, D, 4, 2>(a, seg.item, smem, Shape::ml_off, Shape::scratch_off, Shape::rows, rank, p.cluster);
    }
    cluster_sync_all();  // the others have read this CTA's rows
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  if (warp == 10) tmem_dealloc(tmem_base, 512);
}

// Joins the parts of items that were cut. Block (x, c): rows 8 x .. of the item that begins in CTA c's part of the line
// and goes on in the next one's. One warp per row.
template <typename T, int D>
__global__ void __launch_bounds__(256) chunk_join_kernel(const __grid_constant__ Chunk p) {
  constexpr int kPer = D / 32;
  let_later();
  after_earlier();
  const Args& a = p.a;
  const int c0 = blockIdx.y;
  const int cut = p.plan.cut[c0 + 1];
  if (cut >= p.plan.cut[p.ctas]) return;
  const Item item = p.plan.items[p.plan.first[c0 + 1]];
  if (item.start >= cut || item.start < p.plan.cut[c0]) return;
  const int row = blockIdx.x * 8 + (threadIdx.x >> 5), lane = threadIdx.x & 31;
  const int packed = item.row_tile * kItemRows + row, query = packed / a.group;
  if (query >= item.q_len) return;
  const int end = item.start + item.tiles;
  auto slot_of = [&](int c) { return (2 * static_cast<int64_t>(c) + (c == c0)) * kItemRows + row; };
  // parts: c0's and those of the CTAs after it whose part of the line is not empty and begins before the item's end; 32
  // CTAs at a time, a lane to each one's maximum and sum
  float top = -INFINITY, acc[kPer], sum = 0.0f;
#pragma unroll
  for (int e = 0; e < kPer; ++e) acc[e] = 0.0f;
  for (int cb = c0; cb < p.ctas; cb += 32) {
    const int c = cb + lane;
    const int from = c < p.ctas ? p.plan.cut[c] : end, to = c < p.ctas ? p.plan.cut[c + 1] : end;
    const bool part = c == c0 || (from < to && from < end);
    float2 ml = make_float2(-INFINITY, 0.0f);
    if (part) ml = *reinterpret_cast<const float2*>(p.part_ml + slot_of(c) * 2);
    float mx = ml.x;
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, o));
    mx = fmaxf(mx, top);
    const float old = fade(top, mx), wt = exp2_approx(ml.x - base_of(mx));
    top = mx;
    float add = wt * ml.y;
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) add += __shfl_xor_sync(0xffffffffu, add, o);
    sum = fmaf(sum, old, add);
#pragma unroll
    for (int e = 0; e < kPer; ++e) acc[e] *= old;
    const uint32_t parts = __ballot_sync(0xffffffffu, part);
    for (int i0 = 0; i0 < 32 && (parts >> i0) != 0; i0 += 8) {
      float2 x[8][kPer / 2];
#pragma unroll
      for (int i = 0; i < 8; ++i)
#pragma unroll
        for (int e = 0; e < kPer / 2; ++e)
          x[i][e] = (parts >> (i0 + i)) & 1 ? *reinterpret_cast<const float2*>(p.part_o + slot_of(cb + i0 + i) * D + lane * kPer + 2 * e)
                                            : make_float2(0.0f, 0.0f);
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        const float w = __shfl_sync(0xffffffffu, wt, i0 + i);
#pragma unroll
        for (int e = 0; e < kPer / 2; ++e) {
          acc[2 * e] = fmaf(w, x[i][e].x, acc[2 * e]);
          acc[2 * e + 1] = fmaf(w, x[i][e].y, acc[2 * e + 1]);
        }
      }
    }
    if (__shfl_sync(0xffffffffu, to, 31) >= end) break;
  }
  const float inv = inverse(sum);
  const int64_t token = item.q_first + query;
  const int h = item.head * a.group + packed - query * a.group;
  T* dst = static_cast<T*>(a.out) + token * a.out_token + h * a.out_head + lane * kPer;
#pragma unroll
  for (int e = 0; e < kPer; e += 2) *reinterpret_cast<uint32_t*>(dst + e) = pack2<T>(acc[e] * inv, acc[e + 1] * inv);
  if (a.lse != nullptr && lane == 0) a.lse[token * a.heads + h] = log_sum(top, sum);
}

template <typename T, int D, bool kDirect, bool kTwin>
void chunk_configure(int device) {
  static bool known[64] = {};
  bool& configured = known[device & 63];
  if (configured) return;
  RC_CUDA(cudaFuncSetAttribute(chunk_kernel<T, D, kDirect, kTwin>, cudaFuncAttributeMaxDynamicSharedMemorySize, ChunkShape<D, kTwin>::bytes));
  if (kDirect) RC_CUDA(cudaFuncSetAttribute(chunk_kernel<T, D, kDirect, kTwin>, cudaFuncAttributeNonPortableClusterSizeAllowed, 1));
  cudaFuncAttributes attr;  // the register split assumes exactly kLaunchRegs a thread
  RC_CUDA(cudaFuncGetAttributes(&attr, chunk_kernel<T, D, kDirect, kTwin>));
  RC_CHECK(attr.numRegs == kLaunchRegs, "paged attention compiled to " + std::to_string(attr.numRegs) +
                                            " registers a thread; its register split needs " + std::to_string(kLaunchRegs));
  configured = true;
}

// Clusters of `size` CTAs that the device holds at a time.
template <typename T, int D>
int clusters_at_once(int size, int device) {
  static int known[64][5] = {};
  int index = 0;
  while ((1 << index) < size) ++index;
  int& count = known[device & 63][index];
  if (count == 0) {
    cudaLaunchConfig_t config{};
    config.gridDim = dim3(size);
    config.blockDim = dim3(kChunkThreads);
    config.dynamicSmemBytes = ChunkShape<D, false>::bytes;
    cudaLaunchAttribute attribute{};
    attribute.id = cudaLaunchAttributeClusterDimension;
    attribute.val.clusterDim.x = size;
    attribute.val.clusterDim.y = 1;
    attribute.val.clusterDim.z = 1;
    config.attrs = &attribute;
    config.numAttrs = 1;
    int n = 0;
    if (cudaOccupancyMaxActiveClusters(&n, chunk_kernel<T, D, true, false>, &config) != cudaSuccess) {
      (void)cudaGetLastError();
      n = 0;
    }
    count = n > 0 ? n : -1;
  }
  return count;
}

// CTAs of an item in the direct form, or 0 for the planned form, by estimated time in tile pairs (about 1.8 us each):
// direct, every item takes its tiles over its cluster, in as many rounds as its clusters need, and each round has its start
// and end to pay: about 3.5 tiles alone, 6 in a cluster, which joins. A block of the grid without an item (its row tile lies
// past its sequence's rows: one long sequence among short ones) keeps an SM for up to 2.4 us, half of it next to other work:
// 0.6. Planned, all SMs share all tiles, but the plan, the join and the cut items cost about 16. Measured with 1, 2, 4 and 8
// CTAs and planned (us): 16 items of 63 tiles 117, 65, 40, 52 and 40; 54 of 27: 55, 38, 50, 80 and 52; 32 of 63: 118, 66, 42,
// 78 and 57; 84 of 49: 97, 108, 105, 150 and 87; 16 of 8: 21, 18, 15, 25 and 25. 16 sequences with one of 4,000 new tokens
// (141 items, 1,859 empty blocks) 107 directly and 84 planned. Over 655 shapes, batches of unequal sequences among them, the
// choice costs 2.6 % on average (3.9 % without the empty blocks).
template <typename T, int D>
int direct_cluster(int64_t items, int64_t empty, int64_t tiles, bool uneven, int device) {
  const int sms = sm_count(device);
  double best = static_cast<double>(items) * tiles / sms * (uneven ? 0.75 : 1.0) + 16.0;
  int cluster = 0;
  for (int c = 1; c <= 16; c *= 2) {
    const int64_t slots = clusters_at_once<T, D>(c, device);
    if (slots <= 0) continue;
    const double t = static_cast<double>((items + slots - 1) / slots) * (static_cast<double>((tiles + c - 1) / c) + (c > 1 ? 6.0 : 3.5)) +
                     0.6 * static_cast<double>(empty * c) / sms;
    if (t < best) {
      best = t;
      cluster = c;
    }
  }
  return cluster;
}

// The form that a call takes, and its size: row tiles of a sequence and KV head (at most), items of the direct grid and of
// the plan (at most).
struct ChunkForm {
  int64_t row_tiles, grid_items, most_items;
  int cluster;  // 0: planned
  bool twin;
};

template <typename T, int D>
ChunkForm chunk_form(const Args& a, int max_q_len, int device) {
  ChunkForm form{};
  form.row_tiles = (static_cast<int64_t>(max_q_len) * a.group + kItemRows - 1) / kItemRows;
  form.grid_items = static_cast<int64_t>(a.seqs) * form.row_tiles * a.kv_heads;
  form.most_items =
      std::min<int64_t>(form.grid_items, (static_cast<int64_t>(a.tokens) * a.group / kItemRows + a.seqs) * a.kv_heads);
  // tiles of an item, at most: the table's width, or what a window leaves of it
  int64_t keys = static_cast<int64_t>(a.width) * a.tiling.page;
  if (a.window > 0) keys = std::min<int64_t>(keys, static_cast<int64_t>(a.window) + a.sinks + kItemRows / a.group + 2 * kTile);
  const int64_t tiles = (keys + kTile - 1) / kTile;
  form.twin = static_cast<int64_t>(max_q_len) * a.group <= kTile;
  chunk_configure<T, D, true, false>(device);
  form.cluster = direct_cluster<T, D>(form.most_items, form.grid_items - form.most_items, form.twin ? (tiles + 1) / 2 : tiles,
                                      a.causal && form.row_tiles > 1, device);
  return form;
}

template <typename T, int D>
void chunk_launch(const Args& args, const at::Tensor& k_pages, const at::Tensor& v_pages, int max_q_len,
                  const at::Tensor& like, cudaStream_t stream, int device) {
  using Shape = ChunkShape<D, false>;
  const ChunkForm form = chunk_form<T, D>(args, max_q_len, device);
  const int64_t most_items = form.most_items;
  RC_CHECK(most_items < (1ll << 26), "too many rows for one launch");
  Chunk p{};
  p.a = args;
  p.a.tiling = Tiling::of(args.tiling.page, kTile);
  p.row_tiles = static_cast<int>(form.row_tiles);
  p.most_items = static_cast<int>(most_items);
  p.ctas = sm_count(device);
  p.cluster = form.cluster;
  const PageMaps maps = page_maps(k_pages, v_pages, p.a.tiling, kTile);
  if (p.cluster > 0) {
    const int64_t blocks = form.grid_items * p.cluster;
    RC_CHECK(blocks < (1ll << 31), "too many sequences and rows for one launch");
    const dim3 grid(static_cast<unsigned>(blocks));
    if (form.twin) {
      chunk_configure<T, D, true, true>(device);
      launch(chunk_kernel<T, D, true, true>, grid, kChunkThreads, ChunkShape<D, true>::bytes, p.cluster, stream, maps, p);
    } else {
      launch(chunk_kernel<T, D, true, false>, grid, kChunkThreads, Shape::bytes, p.cluster, stream, maps, p);
    }
    return;
  }
  chunk_configure<T, D, false, false>(device);
  RC_CHECK(p.ctas < kPlanThreads, "more SMs than the plan's threads");
  const int64_t o_floats = 2ll * p.ctas * kItemRows * D, ml_floats = 2ll * p.ctas * kItemRows * 2;
  const int64_t ints = most_items * 8 + 4 + 2ll * (p.ctas + 1) + args.seqs;
  at::Tensor workspace = at::empty({o_floats + ml_floats + ints}, like.options().dtype(at::kFloat));
  p.part_o = workspace.data_ptr<float>();
  p.part_ml = p.part_o + o_floats;
  p.plan.items = reinterpret_cast<Item*>(p.part_ml + ml_floats);
  p.plan.head = reinterpret_cast<int*>(p.plan.items + most_items);
  p.plan.cut = p.plan.head + 4;
  p.plan.first = p.plan.cut + p.ctas + 1;
  p.plan.base = p.plan.first + p.ctas + 1;
  launch(chunk_plan_kernel, dim3(1), kPlanThreads, 0, 0, stream, p);
  launch(chunk_kernel<T, D, false, false>, dim3(p.ctas), kChunkThreads, Shape::bytes, 0, stream, maps, p);
  launch(chunk_join_kernel<T, D>, dim3(kItemRows / 8, p.ctas - 1), 256, 0, 0, stream, p);
}

void attend_chunk(const Args& a, int head_dim, bool half, const at::Tensor& k_pages, const at::Tensor& v_pages,
                  int max_q_len, const at::Tensor& like, cudaStream_t stream, int device) {
  if (head_dim == 128)
    half ? chunk_launch<__half, 128>(a, k_pages, v_pages, max_q_len, like, stream, device)
         : chunk_launch<__nv_bfloat16, 128>(a, k_pages, v_pages, max_q_len, like, stream, device);
  else
    half ? chunk_launch<__half, 64>(a, k_pages, v_pages, max_q_len, like, stream, device)
         : chunk_launch<__nv_bfloat16, 64>(a, k_pages, v_pages, max_q_len, like, stream, device);
}

std::string chunk_form_name(const Args& a, int head_dim, int max_q_len, int device) {
  const ChunkForm form = head_dim == 128 ? chunk_form<__nv_bfloat16, 128>(a, max_q_len, device)
                                         : chunk_form<__nv_bfloat16, 64>(a, max_q_len, device);
  if (form.cluster == 0) return "planned";
  return (form.twin ? "twin " : "direct ") + std::to_string(form.cluster);
}

}  // namespace paged
}  // namespace rc
