// Attention of few query rows (single tokens, drafts) over a paged cache, for sm_100a.
//
// What bounds it: reading K and V once. A tile of 64 keys is 32 KB (head_dim 128) and needs 128 m16n8k16 products for
// 16 query rows (64 for S, 64 for P V), which keep the tensor pipe busy for a sixth of the time that the bytes take
// (counters: 17 %), so the products run on mma.sync from registers and the design is about keeping bytes in flight: one
// producer warp streams K and V tiles with TMA (one box per page and 64 channels, 128-byte swizzle) through a ring of
// stages, two CTAs per SM (168 registers a thread; the line form with 128 channels spills 12 bytes).
//
// Rows: the heads of a group share K and V, so a row is (query, head of the group), query-major, 16 rows at most. The four
// consumer warps take 16 keys of each tile: every warp runs its own online softmax (maximum, sum and output in FP32
// registers) and meets the others only when a sequence and head is finished.
//
// Work, shared out: all tiles of all (sequence, KV head) in one line, cut into equal shares, one per CTA, so ragged batches
// and a single long sequence fill all SMs alike, and the host needs no lengths. A CTA whose share holds only a part of an
// item leaves (output, maximum, sum) in FP32 in the workspace; a second kernel joins the parts in order of the CTAs (no
// atomics: results do not depend on timing).
// Work, clustered (few sequences): a cluster of up to 16 CTAs per sequence and head, joined through distributed shared
// memory; no scan of the lengths, no workspace, no second launch.
//
// Measured: 48 sessions of up to 16,384 keys (32 / 8 heads, 1.67 GB) 259 us, 6.45 TB/s; one session over 2,048 keys
// 8.1 us clustered, 13.4 us as a line (launches back to back).
#include <ATen/ATen.h>
#include <c10/cuda/CUDAGuard.h>
#include <c10/cuda/CUDAStream.h>

#include <algorithm>
#include <string>

#include "attend.cuh"

namespace rc {
namespace paged {

constexpr int kShortTile = 64;       // keys of a tile
constexpr int kRows = 16;            // rows: new tokens x heads of a group, at most
constexpr int kGroups = 4;           // consumer warps, each with 16 keys of a tile
constexpr int kShortThreads = 160;   // four consumer warps, one producer warp
constexpr int kShortCtasPerSm = 2;
constexpr int kShortLeast = 2;       // tiles of a share, at least: every part costs a pass through the workspace

template <int D>
struct ShortShape {
  static constexpr int boxes = D / 64;
  static constexpr int box_bytes = kShortTile * 128;            // 64 keys x 64 channels
  static constexpr int tile_bytes = boxes * box_bytes;          // one of K, V
  static constexpr int stages = D == 128 ? 3 : 6;
  static constexpr int join_off = stages * 2 * tile_bytes;      // FP32 rows: warps joining their keys
  static constexpr int join_bytes = 24 * D * 4;                 // three warps' lower 8 rows, or one warp's 16
  static constexpr int bar_off = join_off + join_bytes;
  static constexpr int bytes = bar_off + 1024 + 1024;           // + alignment slack
  static_assert((bytes + 1024) * kShortCtasPerSm <= 228 * 1024, "two CTAs per SM");
};

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
};

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

template <typename T, int D, bool kCluster>
__global__ void __launch_bounds__(kShortThreads, kShortCtasPerSm)
    short_kernel(const __grid_constant__ PageMaps maps, const __grid_constant__ Short p) {
  using Shape = ShortShape<D>;
  constexpr int kKeys = kShortTile / kGroups;  // keys of a warp
  constexpr int kN = kKeys / 8;                // its n-tiles of S
  extern __shared__ __align__(1024) uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  uint64_t* full = reinterpret_cast<uint64_t*>(smem + Shape::bar_off);
  uint64_t* empty = full + Shape::stages;
  float* join_ml = reinterpret_cast<float*>(empty + Shape::stages);  // [key groups][rows][maximum, sum]: 64 rows in all
  int* work = reinterpret_cast<int*>(join_ml + 128);                 // begin, end, sequence, its first place; warps' sums
  const Args& a = p.a;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;

  let_later();
  if (threadIdx.x == 0) {
    for (int s = 0; s < Shape::stages; ++s) {
      mbar_init(&full[s], 1);
      mbar_init(&empty[s], 4);
    }
    fence_barrier_init();
  }
  if (warp == 4) {
    tma_prefetch_desc(&maps.k_wide);
    tma_prefetch_desc(&maps.v_wide);
  }
  after_earlier();
  if (kCluster) {
    // A cluster per sequence and KV head: this CTA's tiles are its rank's part of the item's, and the line is the item.
    __syncthreads();
  } else if (warp < 4) {
    // The line of work: total, this CTA's share, and where it begins.
    // Thread i counts the tiles of sequences [i per, i per + per); their prefix sums place the share.
    const int per = (a.seqs + 127) / 128, s0 = static_cast<int>(threadIdx.x) * per;
    int mine = 0;
#pragma unroll 4
    for (int i = 0; i < per; ++i) {
      if (s0 + i < a.seqs) {
        const SeqWork w(a, s0 + i);
        mine += w.tiles * a.kv_heads;
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
    const int ctas = static_cast<int>(gridDim.x);
    const int share = max(min(kShortLeast, total), (total + ctas - 1) / ctas);
    const int begin = min(total, static_cast<int>(blockIdx.x) * share), end = min(total, begin + share);
    if (threadIdx.x == 0) {
      work[0] = begin;
      work[1] = end;
      if (blockIdx.x == 0) *p.line.share = share;
    }
    const bool here = begin < end && begin >= before && begin < before + mine;
    if (here || blockIdx.x == 0) {
      for (int i = 0; i < per && s0 + i < a.seqs; ++i) {
        const SeqWork w(a, s0 + i);
        const int n = w.tiles * a.kv_heads;
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
  int s, base, begin, end;
  if (kCluster) {
    const int item = static_cast<int>(blockIdx.x) / p.cluster, rank = static_cast<int>(blockIdx.x) - item * p.cluster;
    s = item / a.kv_heads;
    const SeqWork w(a, s);
    if (w.tiles == 0) {  // no new tokens: the whole cluster
      if (threadIdx.x == 0) report_rows(a, s);
      return;
    }
    base = (s * a.kv_heads - item) * w.tiles;  // the item's tiles are places 0 ..
    begin = w.tiles * rank / p.cluster;
    end = w.tiles * (rank + 1) / p.cluster;
  } else {
    __syncthreads();
    begin = work[0];
    end = work[1];
    if (begin >= end) return;
    s = work[2];
    base = work[3];
  }

  int stage = 0;
  uint32_t phase = 0;
  if (warp == 4) {
    // ---------------- producer ----------------
    bool ok = true;
    for (int at = begin; ok && at < end;) {
      const SeqWork w(a, s);
      const int n = w.tiles * a.kv_heads;
      if (at >= base + n) {
        base += n;
        ++s;
        continue;
      }
      const int head = (at - base) / w.tiles, t0 = (at - base) - head * w.tiles;
      const int t1 = min(w.tiles, t0 + end - at);
      const TileRange<kShortTile> range(Sight(a, w.kv_len, w.q_len), 0, w.q_len);
      for (int t = t0; t < t1; ++t) {
        const int first = range.tile(t) * kShortTile;
        const Boxes<kShortTile> boxes(a.tiling, first, w.kv_len);
        ok = __all_sync(0xffffffffu, mbar_wait(&empty[stage], phase ^ 1, a.status, kTimeoutProducer));
        if (!ok) break;
        if (lane == 0) {
          if (boxes.count > 0) mbar_arrive_expect_tx(&full[stage], boxes.count * boxes.rows * 128 * Shape::boxes * 2);
          else mbar_arrive(&full[stage]);
        }
        __syncwarp();
        if (lane < boxes.count) {
          int row;
          const int page = boxes.page(a.table + s * a.table_row, a.pages, a.tiling, first, lane, &row, a.status);
          const bool wide = boxes.rows == kShortTile;
          const CUtensorMap* km = wide ? &maps.k_wide : &maps.k_step;
          const CUtensorMap* vm = wide ? &maps.v_wide : &maps.v_step;
          uint8_t* k = smem + stage * 2 * Shape::tile_bytes + lane * boxes.rows * 128;
          uint8_t* v = k + Shape::tile_bytes;
#pragma unroll
          for (int b = 0; b < Shape::boxes; ++b) load_page_box(k + b * Shape::box_bytes, km, &full[stage], b * 64, row, head, page);
#pragma unroll
          for (int b = 0; b < Shape::boxes; ++b) load_page_box(v + b * Shape::box_bytes, vm, &full[stage], b * 64, row, head, page);
        }
        if (++stage == Shape::stages) {
          stage = 0;
          phase ^= 1;
        }
      }
      at += t1 - t0;
    }
    if (kCluster) {
      if (lane == 0) report_rows(a, s);
      cluster_sync_all();
      cluster_sync_all();
    }
    return;
  }

  // ---------------- consumers ----------------
  const int kg = warp;  // its keys
  const int r0 = lane >> 2, c0 = (lane & 3) * 2;
  bool ok = true;
  for (int at = begin; kCluster || at < end;) {  // a cluster's CTA goes round once, also without tiles
    const SeqWork w(a, s);
    const int n = w.tiles * a.kv_heads;
    if (!kCluster && at >= base + n) {
      base += n;
      ++s;
      continue;
    }
    const int head = kCluster ? static_cast<int>(blockIdx.x) / p.cluster - s * a.kv_heads : (at - base) / w.tiles;
    const int t0 = kCluster ? begin : (at - base) - head * w.tiles;
    const int t1 = kCluster ? end : min(w.tiles, t0 + end - at);
    const Sight sight(a, w.kv_len, w.q_len);
    const TileRange<kShortTile> range(sight, 0, w.q_len);

    // this thread's two rows
    int row_q[2], row_h[2], last[2], low[2];
    bool valid[2];
    uint32_t q[D / 16][4];
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      const int row = r0 + i * 8;
      row_q[i] = row / a.group;
      row_h[i] = head * a.group + row - row_q[i] * a.group;
      valid[i] = row_q[i] < w.q_len;
      last[i] = sight.last(min(row_q[i], w.q_len - 1));
      low[i] = sight.low(last[i]);
      const T* src = static_cast<const T*>(a.q) + static_cast<int64_t>(w.q_first + row_q[i]) * a.q_token + row_h[i] * a.q_head + c0;
#pragma unroll
      for (int k = 0; k < D / 16; ++k) {
        q[k][i] = valid[i] ? *reinterpret_cast<const uint32_t*>(src + k * 16) : 0u;
        q[k][i + 2] = valid[i] ? *reinterpret_cast<const uint32_t*>(src + k * 16 + 8) : 0u;
      }
    }
    const int rows_here = w.q_len * a.group;  // or fewer: kRows
    // bounds over the queries, for tiles that need no mask
    const int all_last = sight.last(0), all_low = sight.low(sight.last(w.q_len - 1));
    const int any_low = sight.low(all_last);

    float o[D / 8][4];
#pragma unroll
    for (int i = 0; i < D / 8; ++i)
#pragma unroll
      for (int e = 0; e < 4; ++e) o[i][e] = 0.0f;
    float m[2] = {-INFINITY, -INFINITY}, l[2] = {0.0f, 0.0f};

    for (int t = t0; t < t1; ++t) {
      const int first = range.tile(t) * kShortTile;
      if (ok) ok = __all_sync(0xffffffffu, mbar_wait(&full[stage], phase, a.status, kTimeoutEpilogue));
      if (ok) {
        const uint32_t kb = smem_u32(smem + stage * 2 * Shape::tile_bytes);
        const uint32_t vb = kb + Shape::tile_bytes;
        float sc[kN][4];
#pragma unroll
        for (int j = 0; j < kN; ++j)
#pragma unroll
          for (int e = 0; e < 4; ++e) sc[j][e] = 0.0f;
        // S = Q K^T: matrices (keys 0-7, d 0-7), (keys 0-7, d 8-15), (keys 8-15, d 0-7), (keys 8-15, d 8-15)
#pragma unroll
        for (int k = 0; k < D / 16; ++k) {
#pragma unroll
          for (int j = 0; j < kN / 2; ++j) {
            const int key = kg * kKeys + j * 16 + (lane & 7) + ((lane >> 4) << 3);
            const int chunk = (k & 3) * 2 + ((lane >> 3) & 1);
            uint32_t b[4];
            ldmatrix_x4(b, kb + (k >> 2) * Shape::box_bytes + key * 128 + ((chunk ^ (key & 7)) << 4));
            mma_16816(sc[2 * j], q[k], b[0], b[1], T());
            mma_16816(sc[2 * j + 1], q[k], b[2], b[3], T());
          }
        }
        const bool whole = first + kShortTile - 1 <= all_last &&
                           (first >= all_low || first + kShortTile <= a.sinks);
        if (!whole) {
#pragma unroll
          for (int j = 0; j < kN; ++j)
#pragma unroll
            for (int e = 0; e < 4; ++e) {
              const int r = kg * kKeys + j * 8 + c0 + (e & 1);
              const int at_key = first + r;
              const int i = e >> 1;
              if (!(at_key <= last[i] && at_key < w.kv_len && (at_key >= low[i] || at_key < a.sinks)))
                sc[j][e] = -INFINITY;
            }
        }
        float alpha[2];
#pragma unroll
        for (int i = 0; i < 2; ++i) {
          float mx = -INFINITY;
#pragma unroll
          for (int j = 0; j < kN; ++j) mx = fmaxf(mx, fmaxf(sc[j][2 * i], sc[j][2 * i + 1]));
          mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 1));
          mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 2));
          const float top = fmaxf(m[i], mx * a.scale_log2);
          const float use = base_of(top);
          alpha[i] = fade(m[i], top);
          m[i] = top;
          float sum = 0.0f;
#pragma unroll
          for (int j = 0; j < kN; ++j)
#pragma unroll
            for (int e = 0; e < 2; ++e) {
              const float x = exp2_approx(fmaf(sc[j][2 * i + e], a.scale_log2, -use));
              sc[j][2 * i + e] = x;
              sum += x;
            }
          l[i] = l[i] * alpha[i] + sum;
        }
        if (__any_sync(0xffffffffu, alpha[0] != 1.0f || alpha[1] != 1.0f)) {
#pragma unroll
          for (int i = 0; i < D / 8; ++i) {
            o[i][0] *= alpha[0];
            o[i][1] *= alpha[0];
            o[i][2] *= alpha[1];
            o[i][3] *= alpha[1];
          }
        }
        // O += P V: matrices (keys 0-7, d 0-7), (keys 8-15, d 0-7), (keys 0-7, d 8-15), (keys 8-15, d 8-15). Rows of V
        // that no query sees (past the sequence, before the window, never loaded) are taken as zeros whatever they
        // hold: 0 * NaN is NaN.
#pragma unroll
        for (int k = 0; k < kKeys / 16; ++k) {
          const uint32_t pa[4] = {pack2<T>(sc[2 * k][0], sc[2 * k][1]), pack2<T>(sc[2 * k][2], sc[2 * k][3]),
                                  pack2<T>(sc[2 * k + 1][0], sc[2 * k + 1][1]), pack2<T>(sc[2 * k + 1][2], sc[2 * k + 1][3])};
          uint32_t keep[2] = {0xffffffffu, 0xffffffffu};
          if (!whole) {
#pragma unroll
            for (int h = 0; h < 2; ++h) {
              keep[h] = 0;
#pragma unroll
              for (int e = 0; e < 2; ++e) {
                const int r = kg * kKeys + k * 16 + h * 8 + c0 + e;
                if (first + r < w.kv_len && (first + r >= any_low || first + r < a.sinks)) keep[h] |= 0xffffu << (16 * e);
              }
            }
          }
#pragma unroll
          for (int d = 0; d < D / 16; ++d) {
            const int key = kg * kKeys + k * 16 + (lane & 7) + (((lane >> 3) & 1) << 3);
            const int chunk = (d & 3) * 2 + (lane >> 4);
            uint32_t b[4];
            ldmatrix_x4_trans(b, vb + (d >> 2) * Shape::box_bytes + key * 128 + ((chunk ^ (key & 7)) << 4));
            mma_16816(o[2 * d], pa, b[0] & keep[0], b[1] & keep[1], T());
            mma_16816(o[2 * d + 1], pa, b[2] & keep[0], b[3] & keep[1], T());
          }
        }
        __syncwarp();
        if (lane == 0) mbar_arrive(&empty[stage]);
      }
      if (++stage == Shape::stages) {
        stage = 0;
        phase ^= 1;
      }
    }
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
      float2* buf = reinterpret_cast<float2*>(smem + Shape::join_off) + lane;
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
      float4* buf = reinterpret_cast<float4*>(smem + Shape::join_off) + lane;
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
    if (kCluster) {
      // The CTAs of the cluster put rows, maxima and sums into their stages (every tile has been consumed), then each
      // joins a part of the channels over all of them, in order, through distributed shared memory.
      float* res = reinterpret_cast<float*>(smem);  // [kRows][D]
      float* res_ml = res + kRows * D;              // [kRows][2]
      consumers_sync();
      if (kg == 0) {
#pragma unroll
        for (int i = 0; i < 2; ++i) {
          const int row = r0 + 8 * i;
#pragma unroll
          for (int d = 0; d < D / 8; ++d) *reinterpret_cast<float2*>(res + row * D + d * 8 + c0) = make_float2(o[d][2 * i], o[d][2 * i + 1]);
          if ((lane & 3) == 0) *reinterpret_cast<float2*>(res_ml + row * 2) = make_float2(m[i], l[i]);
        }
      }
      cluster_sync_all();
      const int rank = static_cast<int>(blockIdx.x) % p.cluster;
      const int vecs = D / 4 / p.cluster;  // float4 of a row that this CTA joins
      const int rows = min(kRows, rows_here);
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
        const int query = row / a.group, h = head * a.group + row - query * a.group;
        const int64_t token = w.q_first + query;
        T* dst = static_cast<T*>(a.out) + token * a.out_token + h * a.out_head + col;
        if (ok) *reinterpret_cast<uint2*>(dst) = make_uint2(pack2<T>(acc.x * inv, acc.y * inv), pack2<T>(acc.z * inv, acc.w * inv));
        if (ok && a.lse != nullptr && col == 0) a.lse[token * a.heads + h] = log_sum(top, sum);
      }
      cluster_sync_all();  // the others have read this CTA's rows
      return;
    }
    if (kg == 0 && ok) {
      const int item_first = base + head * w.tiles;
      const bool starts = item_first >= begin, ends = item_first + w.tiles <= end;
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        if (!valid[i]) continue;
        const int64_t token = w.q_first + row_q[i];
        if (starts && ends) {
          const float inv = inverse(l[i]);
          T* dst = static_cast<T*>(a.out) + token * a.out_token + row_h[i] * a.out_head + c0;
#pragma unroll
          for (int d = 0; d < D / 8; ++d)
            *reinterpret_cast<uint32_t*>(dst + d * 8) = pack2<T>(o[d][2 * i] * inv, o[d][2 * i + 1] * inv);
          if (a.lse != nullptr && (lane & 3) == 0)
            a.lse[token * a.heads + row_h[i]] = log_sum(m[i], l[i]);
        } else {
          const int64_t slot = (2 * static_cast<int64_t>(blockIdx.x) + (starts ? 1 : 0)) * kRows + r0 + 8 * i;
          float* dst = p.part_o + slot * D + c0;
#pragma unroll
          for (int d = 0; d < D / 8; ++d) *reinterpret_cast<float2*>(dst + d * 8) = make_float2(o[d][2 * i], o[d][2 * i + 1]);
          if ((lane & 3) == 0) *reinterpret_cast<float2*>(p.part_ml + slot * 2) = make_float2(m[i], l[i]);
        }
      }
    }
    at += t1 - t0;
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
  const int item = blockIdx.x / quads, s = item / a.kv_heads, head = item - s * a.kv_heads;
  let_later();
  after_earlier();
  if (row == 0 && head == 0 && lane == 0) report_rows(a, s);
  const SeqWork w(a, s);
  const int query = row / a.group;
  if (query >= w.q_len) return;
  const int share = *p.line.share;
  const int begin = p.line.first[s] + head * w.tiles, end = begin + w.tiles;
  const int c0 = begin / share, c1 = (end - 1) / share;
  if (c0 == c1) return;
  // 32 parts at a time, a lane to each one's maximum and sum
  float top = -INFINITY, acc[kPer], sum = 0.0f;
#pragma unroll
  for (int e = 0; e < kPer; ++e) acc[e] = 0.0f;
  for (int cb = c0; cb <= c1; cb += 32) {
    const int n = min(32, c1 - cb + 1);
    const int64_t first_slot = (2 * static_cast<int64_t>(cb) + (cb == c0)) * kRows + row;
    const int64_t slot = (2 * static_cast<int64_t>(cb + lane) + (cb + lane == c0)) * kRows + row;
    float2 ml = make_float2(-INFINITY, 0.0f);
    if (lane < n) ml = *reinterpret_cast<const float2*>(p.part_ml + slot * 2);
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
      const int64_t at = i == 0 ? first_slot : 2 * static_cast<int64_t>(cb + i) * kRows + row;
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
  const int h = head * a.group + row - query * a.group;
  T* dst = static_cast<T*>(a.out) + token * a.out_token + h * a.out_head + lane * kPer;
#pragma unroll
  for (int e = 0; e < kPer; e += 2) *reinterpret_cast<uint32_t*>(dst + e) = pack2<T>(acc[e] * inv, acc[e + 1] * inv);
  if (a.lse != nullptr && lane == 0) a.lse[token * a.heads + h] = log_sum(top, sum);
}

// Clusters of `size` CTAs that run at the same time, or -1 where none does.
template <typename T, int D>
int short_clusters_at_once(int size, int device) {
  static int known[64][5] = {};
  int slot = 0;
  while ((1 << slot) < size) ++slot;
  int& count = known[device & 63][slot];
  if (count == 0) {
    cudaLaunchConfig_t config{};
    config.gridDim = dim3(static_cast<unsigned>(size));
    config.blockDim = dim3(kShortThreads);
    config.dynamicSmemBytes = ShortShape<D>::bytes;
    cudaLaunchAttribute attribute{};
    attribute.id = cudaLaunchAttributeClusterDimension;
    attribute.val.clusterDim.x = size;
    attribute.val.clusterDim.y = 1;
    attribute.val.clusterDim.z = 1;
    config.attrs = &attribute;
    config.numAttrs = 1;
    int n = 0;
    if (cudaOccupancyMaxActiveClusters(&n, short_kernel<T, D, true>, &config) != cudaSuccess) {
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
template <typename T, int D>
int short_cluster(int64_t items, int64_t tiles, int step, bool several, int device) {
  const double hbm = 2.0 * ShortShape<D>::tile_bytes / 6.5e6;  // us of a tile, for one CTA alone
  const double box = 0.6 + 0.045 * (2 * ShortShape<D>::boxes * kShortTile / step);
  const double slots = kShortCtasPerSm * sm_count(device), share = std::max<double>(kShortLeast, items * tiles / slots);
  double best = 10.0 + 0.2 * std::min<double>(tiles / kShortLeast, slots / items) + hbm * slots * (several ? 0.75 : 1.0) * share;
  int cluster = 0;
  for (int c = 2; c <= 16; c *= 2) {
    const int64_t at_once = short_clusters_at_once<T, D>(c, device);
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

template <typename T, int D>
void short_configure(int device) {
  using Shape = ShortShape<D>;
  static bool known[64] = {};
  bool& configured = known[device & 63];
  if (!configured) {
    RC_CUDA(cudaFuncSetAttribute(short_kernel<T, D, false>, cudaFuncAttributeMaxDynamicSharedMemorySize, Shape::bytes));
    RC_CUDA(cudaFuncSetAttribute(short_kernel<T, D, true>, cudaFuncAttributeMaxDynamicSharedMemorySize, Shape::bytes));
    RC_CUDA(cudaFuncSetAttribute(short_kernel<T, D, true>, cudaFuncAttributeNonPortableClusterSizeAllowed, 1));
    configured = true;
  }
}

int64_t short_tiles(const Args& a) { return (static_cast<int64_t>(a.width) * a.tiling.page + kShortTile - 1) / kShortTile; }

// CTAs of a cluster, or 0 for the line.
template <typename T, int D>
int short_form(const Args& a, int device) {
  short_configure<T, D>(device);
  return short_cluster<T, D>(static_cast<int64_t>(a.seqs) * a.kv_heads, short_tiles(a), Tiling::of(a.tiling.page, kShortTile).step,
                             a.seqs > 1, device);
}

template <typename T, int D>
void short_launch(Args a, const at::Tensor& k_pages, const at::Tensor& v_pages, const at::Tensor& like, cudaStream_t stream,
                  int device) {
  using Shape = ShortShape<D>;
  static_assert(kRows * (D + 2) * 4 <= Shape::stages * 2 * Shape::tile_bytes, "a CTA's rows fit its stages");
  Short p{};
  p.a = a;
  p.a.tiling = Tiling::of(a.tiling.page, kShortTile);
  const PageMaps maps = page_maps(k_pages, v_pages, p.a.tiling, kShortTile);
  const int64_t items = static_cast<int64_t>(a.seqs) * a.kv_heads, slots = sm_count(device) * kShortCtasPerSm;
  p.cluster = short_form<T, D>(a, device);
  if (p.cluster > 0) {
    launch(short_kernel<T, D, true>, dim3(static_cast<unsigned>(items * p.cluster)), kShortThreads, Shape::bytes, p.cluster,
           stream, maps, p);
    return;
  }
  const int ctas = static_cast<int>(std::min<int64_t>(slots, items * (short_tiles(a) + 1)));
  RC_CHECK(items * (kRows / 4) < (1ll << 31), "too many sequences and rows for one launch");
  const int64_t floats = 2ll * ctas * kRows * (D + 2), ints = 1 + 2ll * a.seqs;
  at::Tensor workspace = at::empty({floats + ints}, like.options().dtype(at::kFloat));
  p.part_o = workspace.data_ptr<float>();
  p.part_ml = p.part_o + 2ll * ctas * kRows * D;
  int* line = reinterpret_cast<int*>(p.part_o + floats);
  p.line = {line, line + 1, line + 1 + a.seqs};
  launch(short_kernel<T, D, false>, dim3(ctas), kShortThreads, Shape::bytes, 0, stream, maps, p);
  launch(short_join_kernel<T, D>, dim3(static_cast<unsigned>(items * (kRows / 4))), 128, 0, 0, stream, p);
}

void attend_short(const Args& a, int head_dim, bool half, const at::Tensor& k_pages, const at::Tensor& v_pages,
                  int, const at::Tensor& like, cudaStream_t stream, int device) {
  if (head_dim == 128)
    half ? short_launch<__half, 128>(a, k_pages, v_pages, like, stream, device)
         : short_launch<__nv_bfloat16, 128>(a, k_pages, v_pages, like, stream, device);
  else
    half ? short_launch<__half, 64>(a, k_pages, v_pages, like, stream, device)
         : short_launch<__nv_bfloat16, 64>(a, k_pages, v_pages, like, stream, device);
}

std::string short_form_name(const Args& a, int head_dim, int device) {
  const int cluster = head_dim == 128 ? short_form<__nv_bfloat16, 128>(a, device) : short_form<__nv_bfloat16, 64>(a, device);
  return cluster > 0 ? "few rows, cluster " + std::to_string(cluster) : "few rows, line";
}

}  // namespace paged
}  // namespace rc
