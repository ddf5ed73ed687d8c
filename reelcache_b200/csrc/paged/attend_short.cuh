// What the kernels for few query rows share (pages in 16 bits and in 8 bits): the line of work, and how parts of an item are
// joined, inside a CTA, over a cluster, and over the CTAs of the line.
#pragma once

#include <algorithm>

#include "attend.cuh"

namespace rc {
namespace paged {

constexpr int kShortTile = 64;       // keys of a tile
constexpr int kRows = 16;            // rows: new tokens x heads of a group, at most
constexpr int kGroups = 4;           // consumer warps, each with 16 keys of a tile
constexpr int kShortThreads = 160;   // four consumer warps, one producer warp
constexpr int kShortCtasPerSm = 2;
constexpr int kShortLeast = 2;       // tiles of a share, at least: every part costs a pass through the workspace

// The workspace's line of work, written by CTA 0 of the first kernel for the second.
struct Line {
  int* share;   // [1]
  int* first;   // [seqs]: first place of each sequence's items in the line
  int* tiles;   // [seqs]: tiles of each of its items
};

struct Short {
  Args a;
  Line line;
  float* part_o;   // [2 * CTAs, 16, D]
  float* part_ml;  // [2 * CTAs, 16, 2]
  int cluster;     // CTAs of a cluster (the clustered form)
  int rows;        // of an item: those of a sequence and KV head, or a slice of them
  int slices;      // slices of a sequence's rows (others than they hold have no result)
  int par;         // KV heads that the line's CTAs take side by side (a divisor of their number): of them and their
                   // slices: CTA (par slices) i + j takes share i of the j-th, j = slice par + head
};

__device__ __forceinline__ void ldmatrix_x4(uint32_t (&r)[4], uint32_t addr) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0, %1, %2, %3}, [%4];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
               : "r"(addr)
               : "memory");
}
__device__ __forceinline__ void ldmatrix_x4_trans(uint32_t (&r)[4], uint32_t addr) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0, %1, %2, %3}, [%4];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
               : "r"(addr)
               : "memory");
}

__device__ __forceinline__ void consumers_sync() { asm volatile("bar.sync 1, 128;" ::: "memory"); }

// New tokens and tiles of one sequence (of each of its KV heads).
struct SeqWork {
  int q_first, q_len, kv_len, tiles;
  __device__ __forceinline__ SeqWork(const Args& a, int s) {
    q_len = new_tokens(a, s, &q_first);
    kv_len = held_keys(a, s);
    tiles = 0;
    if (q_len > 0) tiles = max(1, TileRange<kShortTile>(Sight(a, kv_len, q_len), 0, q_len).count());
  }
};

// The line of work: total, this CTA's share (work[0], work[1]), and the sequence (work[2]) and its first place (work[3]) in which
// it begins. For the four consumer warps; work[4 ..] takes their sums.
__device__ __forceinline__ void place_share(const Short& p, int* work) {
  const Args& a = p.a;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, heads = a.kv_heads / p.par;
  // Thread i counts the tiles of sequences [i per, i per + per); their prefix sums place the share.
  const int per = (a.seqs + 127) / 128, s0 = static_cast<int>(threadIdx.x) * per;
  int mine = 0;
#pragma unroll 4
  for (int i = 0; i < per; ++i) {
    if (s0 + i < a.seqs) {
      const SeqWork w(a, s0 + i);
      mine += w.tiles * heads;
    }
  }
  int x = mine;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const int y = __shfl_up_sync(0xffffffffu, x, o);
    if (lane >= o) x += y;
  }
  if (lane == 31) work[4 + warp] = x;
  consumers_sync();
  int before = x - mine, total = 0;
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const int n = work[4 + i];
    if (i < warp) before += n;
    total += n;
  }
  const int sides = p.par * p.slices, ctas = static_cast<int>(gridDim.x) / sides, index = static_cast<int>(blockIdx.x) / sides;
  const int share = max(min(kShortLeast, total), (total + ctas - 1) / ctas);
  const int begin = min(total, index * share), end = min(total, begin + share);
  if (threadIdx.x == 0) {
    work[0] = begin;
    work[1] = end;
    if (blockIdx.x == 0) *p.line.share = share;
  }
  const bool here = begin < end && begin >= before && begin < before + mine;
  if (here || blockIdx.x == 0) {
    for (int i = 0; i < per && s0 + i < a.seqs; ++i) {
      const SeqWork w(a, s0 + i);
      const int n = w.tiles * heads;
      if (here && begin >= before && begin < before + n) {
        work[2] = s0 + i;
        work[3] = before;
      }
      if (blockIdx.x == 0) {
        p.line.first[s0 + i] = before;
        p.line.tiles[s0 + i] = w.tiles;
      }
      before += n;
    }
  }
}

// Joins the warps of a CTA, which split the keys, into warp 0: every lane's rows r0 and r0 + 8 of o (FP32, relative to m), m and
// l. join_buf: 24 * D floats.
template <int D>
__device__ __forceinline__ void join_warps(float (&o)[D / 8][4], float (&m)[2], float (&l)[2], float* join_ml, uint8_t* join_buf,
                                           int rows_here) {
  const int kg = threadIdx.x >> 5, lane = threadIdx.x & 31, r0 = lane >> 2;
#pragma unroll
  for (int i = 0; i < 2; ++i) {
    l[i] += __shfl_xor_sync(0xffffffffu, l[i], 1);
    l[i] += __shfl_xor_sync(0xffffffffu, l[i], 2);
  }
  // Warps that split the keys join theirs into key group 0, one after the other through shared memory. The same lane
  // of every warp holds the same rows and columns, so the buffer is laid out by lane.
  if ((lane & 3) == 0) {
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      join_ml[(kg * kRows + r0 + 8 * i) * 2] = m[i];
      join_ml[(kg * kRows + r0 + 8 * i) * 2 + 1] = l[i];
    }
  }
  consumers_sync();
  float w_o[2];
#pragma unroll
  for (int i = 0; i < 2; ++i) {
    float top = -INFINITY, total = 0.0f;
    float gm[kGroups];
#pragma unroll
    for (int g = 0; g < kGroups; ++g) {
      gm[g] = join_ml[(g * kRows + r0 + 8 * i) * 2];
      top = fmaxf(top, gm[g]);
    }
    const float use = base_of(top);
#pragma unroll
    for (int g = 0; g < kGroups; ++g)
      total = fmaf(join_ml[(g * kRows + r0 + 8 * i) * 2 + 1], exp2_approx(gm[g] - use), total);
    w_o[i] = exp2_approx(m[i] - use);
    m[i] = top;
    l[i] = total;
  }
#pragma unroll
  for (int i = 0; i < D / 8; ++i) {
    o[i][0] *= w_o[0];
    o[i][1] *= w_o[0];
    o[i][2] *= w_o[1];
    o[i][3] *= w_o[1];
  }
  if (rows_here <= 8) {
    // only the first 8 rows hold anything: all warps at once
    float2* buf = reinterpret_cast<float2*>(join_buf) + lane;
    if (kg > 0) {
#pragma unroll
      for (int i = 0; i < D / 8; ++i) buf[((kg - 1) * (D / 8) + i) * 32] = make_float2(o[i][0], o[i][1]);
    }
    consumers_sync();
    if (kg == 0) {
#pragma unroll
      for (int g = 0; g < kGroups - 1; ++g)
#pragma unroll
        for (int i = 0; i < D / 8; ++i) {
          const float2 x = buf[(g * (D / 8) + i) * 32];
          o[i][0] += x.x;
          o[i][1] += x.y;
        }
    }
    consumers_sync();
  } else {
    float4* buf = reinterpret_cast<float4*>(join_buf) + lane;
#pragma unroll
    for (int g = 1; g < kGroups; ++g) {
      if (kg == g) {
#pragma unroll
        for (int i = 0; i < D / 8; ++i) buf[i * 32] = make_float4(o[i][0], o[i][1], o[i][2], o[i][3]);
      }
      consumers_sync();
      if (kg == 0) {
#pragma unroll
        for (int i = 0; i < D / 8; ++i) {
          const float4 x = buf[i * 32];
          o[i][0] += x.x;
          o[i][1] += x.y;
          o[i][2] += x.z;
          o[i][3] += x.w;
        }
      }
      consumers_sync();
    }
  }
}

// Joins a part of the channels of an item's rows over the CTAs of a cluster, in order, through distributed shared memory: `res`
// [kRows][D] FP32, `res_ml` [kRows][maximum, sum] of each CTA. For 128 threads; the cluster has to meet once more before `res`
// may be written again.
template <typename T, int D>
__device__ __forceinline__ void join_few_cluster(const Short& p, const SeqWork& w, int head, int row0, int rows_here, const float* res,
                                                 const float* res_ml, bool ok) {
  const Args& a = p.a;
  const int rank = static_cast<int>(blockIdx.x) % p.cluster;
  const int vecs = D / 4 / p.cluster;  // float4 of a row that this CTA joins
  const int rows = min(p.rows, rows_here);
  for (int v = static_cast<int>(threadIdx.x); v < rows * vecs; v += 128) {
    const int row = v / vecs, col = (rank * vecs + v - row * vecs) * 4;
    float top = -INFINITY, sum = 0.0f;
    float4 acc = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
    for (int first = 0; first < p.cluster; first += 8) {  // eight CTAs' values at a time
      float2 ml[8];
      float4 x[8];
#pragma unroll
      for (int c = 0; c < 8; ++c) {
        if (first + c >= p.cluster) {
          ml[c] = make_float2(-INFINITY, 0.0f);
          x[c] = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
          continue;
        }
        ml[c] = load_cluster_2(cluster_addr(res_ml + row * 2, first + c));
        x[c] = load_cluster_4(cluster_addr(res + row * D + col, first + c));
      }
      float mx = top;
#pragma unroll
      for (int c = 0; c < 8; ++c) mx = fmaxf(mx, ml[c].x);
      const float use = base_of(mx), old = fade(top, mx);
      top = mx;
      sum *= old;
      acc.x *= old, acc.y *= old, acc.z *= old, acc.w *= old;
#pragma unroll
      for (int c = 0; c < 8; ++c) {
        const float wt = exp2_approx(ml[c].x - use);
        sum = fmaf(wt, ml[c].y, sum);
        acc.x = fmaf(wt, x[c].x, acc.x);
        acc.y = fmaf(wt, x[c].y, acc.y);
        acc.z = fmaf(wt, x[c].z, acc.z);
        acc.w = fmaf(wt, x[c].w, acc.w);
      }
    }
    const float inv = inverse(sum);
    const int query = (row0 + row) / a.group, h = head * a.group + row0 + row - query * a.group;
    const int64_t token = w.q_first + query;
    T* dst = static_cast<T*>(a.out) + token * a.out_token + h * a.out_head + col;
    if (ok) *reinterpret_cast<uint2*>(dst) = make_uint2(pack2<T>(acc.x * inv, acc.y * inv), pack2<T>(acc.z * inv, acc.w * inv));
    if (ok && a.lse != nullptr && col == 0) a.lse[token * a.heads + h] = log_sum(top, sum);
  }
}

// Joins the parts of items that more than one CTA worked on. One warp per row; the parts are those of the CTAs whose
// shares the item's tiles lie in, in order.
template <typename T, int D>
__global__ void __launch_bounds__(128) short_join_kernel(const __grid_constant__ Short p) {
  constexpr int kPer = D / 32;
  const Args& a = p.a;
  const int lane = threadIdx.x & 31;
  const int quads = kRows / 4;
  const int row = (blockIdx.x % quads) * 4 + (threadIdx.x >> 5);
  const int index = blockIdx.x / quads, item = index / p.slices, slice = index - item * p.slices, s = item / a.kv_heads, head = item - s * a.kv_heads;
  let_later();
  after_earlier();
  if (row == 0 && head == 0 && slice == 0 && lane == 0) report_rows(a, s);
  const SeqWork w(a, s);
  const int packed = slice * p.rows + row, query = packed / a.group;
  if (query >= w.q_len || row >= p.rows) return;
  const int share = *p.line.share;
  const int place = head / p.par, side = slice * p.par + head - place * p.par;
  const int begin = p.line.first[s] + place * w.tiles, end = begin + w.tiles;
  const int c0 = begin / share, c1 = (end - 1) / share;
  if (c0 == c1) return;
  const auto slot_of = [&](int c) { return (2 * (static_cast<int64_t>(c) * p.par * p.slices + side) + (c == c0)) * kRows + row; };
  // 32 parts at a time, a lane to each one's maximum and sum
  float top = -INFINITY, acc[kPer], sum = 0.0f;
#pragma unroll
  for (int e = 0; e < kPer; ++e) acc[e] = 0.0f;
  for (int cb = c0; cb <= c1; cb += 32) {
    const int n = min(32, c1 - cb + 1);
    float2 ml = make_float2(-INFINITY, 0.0f);
    if (lane < n) ml = *reinterpret_cast<const float2*>(p.part_ml + slot_of(cb + lane) * 2);
    float mx = ml.x;
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, o));
    mx = fmaxf(mx, top);
    const float old = fade(top, mx), wt = exp2_approx(ml.x - base_of(mx));
    top = mx;
    float part = wt * ml.y;
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) part += __shfl_xor_sync(0xffffffffu, part, o);
    sum = fmaf(sum, old, part);
#pragma unroll
    for (int e = 0; e < kPer; ++e) acc[e] *= old;
#pragma unroll 8
    for (int i = 0; i < n; ++i) {
      const float weight = __shfl_sync(0xffffffffu, wt, i);
      const int64_t at = slot_of(cb + i);
#pragma unroll
      for (int e = 0; e < kPer; e += 2) {
        const float2 x = *reinterpret_cast<const float2*>(p.part_o + at * D + lane * kPer + e);
        acc[e] = fmaf(weight, x.x, acc[e]);
        acc[e + 1] = fmaf(weight, x.y, acc[e + 1]);
      }
    }
  }
  const float inv = inverse(sum);
  const int64_t token = w.q_first + query;
  const int h = head * a.group + packed - query * a.group;
  T* dst = static_cast<T*>(a.out) + token * a.out_token + h * a.out_head + lane * kPer;
#pragma unroll
  for (int e = 0; e < kPer; e += 2) *reinterpret_cast<uint32_t*>(dst + e) = pack2<T>(acc[e] * inv, acc[e + 1] * inv);
  if (a.lse != nullptr && lane == 0) a.lse[token * a.heads + h] = log_sum(top, sum);
}

// Clusters of `size` CTAs of a form that run at the same time, or -1 where none does. A form names its clustered kernel, its
// CTAs on an SM and shared memory, the bytes of a tile of K (or V) and the boxes of 128 bytes or less that a row of it takes.
template <typename Form>
int short_clusters_at_once(int size, int device) {
  static int known[64][5] = {};
  int slot = 0;
  while ((1 << slot) < size) ++slot;
  int& count = known[device & 63][slot];
  if (count == 0) {
    cudaLaunchConfig_t config{};
    config.gridDim = dim3(static_cast<unsigned>(size));
    config.blockDim = dim3(kShortThreads);
    config.dynamicSmemBytes = Form::bytes;
    cudaLaunchAttribute attribute{};
    attribute.id = cudaLaunchAttributeClusterDimension;
    attribute.val.clusterDim.x = size;
    attribute.val.clusterDim.y = 1;
    attribute.val.clusterDim.z = 1;
    config.attrs = &attribute;
    config.numAttrs = 1;
    int n = 0;
    if (cudaOccupancyMaxActiveClusters(&n, Form::clustered(), &config) != cudaSuccess) {
      (void)cudaGetLastError();
      n = 0;
    }
    count = n > 0 ? n : -1;
  }
  return count;
}

// CTAs of an item in the clustered form, or 0 for the line, by estimated time in us. Clusters run in rounds of about 5 and
// the tiles of a CTA: 0.6 and 0.045 for every box that fetches one (pages of 16, 128 channels: 16 boxes, 1.3), or what HBM
// takes for all CTAs' tiles where that is more. The line takes 10, 0.2 for every part of an item (they are joined one after
// the other) and HBM's time for an even share of all tiles, of which a ragged batch may have fewer than its table has room
// for (so 0.75 of them). Measured clustered and as a line (8 KV heads, pages of 16): 1 session of 2,048 keys 8.1 and 13.4,
// of 65,536 keys 97 and 60; 2 of 2,048 keys 11.0 (clusters of 8; of 16, in two rounds, 15.3) and 13.8, of 16,384 keys 51
// and 35; 16 of 512 keys 11.4 and 13.8.
template <typename Form>
int short_cluster(int64_t items, int64_t tiles, int step, bool several, int device) {
  const double hbm = 2.0 * Form::tile_bytes / 6.5e6;  // us of a tile, for one CTA alone
  const double box = 0.6 + 0.045 * (2 * Form::boxes * kShortTile / step);
  const double slots = Form::ctas * sm_count(device), share = std::max<double>(kShortLeast, items * tiles / slots);
  double best = 10.0 + 0.2 * std::min<double>(tiles / kShortLeast, slots / items) + hbm * slots * (several ? 0.75 : 1.0) * share;
  int cluster = 0;
  for (int c = 2; c <= 16; c *= 2) {
    const int64_t at_once = short_clusters_at_once<Form>(c, device);
    if (at_once <= 0) continue;
    const double tile = std::max(box, hbm * c * std::min<int64_t>(items, at_once));
    const double t = static_cast<double>((items + at_once - 1) / at_once) * (5.0 + tile * static_cast<double>((tiles + c - 1) / c));
    if (t < best - (cluster > 0 ? 0.5 : 0.0)) {  // (larger clusters find room less easily: only where they gain something)
      best = t;
      cluster = c;
    }
  }
  return cluster;
}

inline int64_t short_tiles(const Args& a) { return (static_cast<int64_t>(a.width) * a.tiling.page + kShortTile - 1) / kShortTile; }

}  // namespace paged
}  // namespace rc
