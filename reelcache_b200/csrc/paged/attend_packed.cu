// Attention of few query rows (single tokens, drafts) over pages in 8 bits (packed.h), for sm_100a.
//
// What bounds it: reading the codes once, half the bytes of a 16-bit cache in the same time per product, so the frame of
// attend_short.cu is kept (a producer warp streams tiles of 64 keys with TMA, four consumer warps with 16 keys each on
// mma.sync, work in a line or in clusters) and what comes between the bytes and the products is kept short.
//
// Products are transposed: S^T = K Q^T and O^T = V^T P^T have keys and channels in the 16 rows of the instruction and the queries in its 8
// columns, so that up to 8 rows (a single token's group of heads) take one instruction where Q K^T would take two, half empty.
// P^T comes out of S^T's layout by a transposition of 8 x 8 numbers (movmatrix).
//
// Codes become fp16 in registers, exactly, two by one conversion; the products are fp16 whatever the rows' type. Q is brought
// to fp16 by a power of two for each row that puts its largest magnitude between 2^6 and 2^7: exact for what is at least 2^-20
// of that, off by at most 2^-31 of it below. Scales multiply neither codes nor channels: K's multiply the scores (FP32), V's
// the probabilities, as addends of their exponents: weight = 2^(score + log2 scale - unit). A row's unit follows the largest
// score + log2 scale that the row sees (not the largest scale, which may belong to a key of no weight), so that this key's weight
// lies between 2^7 and 2^15 of fp16's range. Weights are rounded to fp16 for the product: by half a step of 2^-10 of their size, or,
// below 2^-14, by 2^-25, which is 2^-32 of the largest weight; their sum, of the probabilities alone, is FP32. Maximum and unit move
// rarely, after one vote: the maximum when a score is more than 2^8 above it, the unit when a weight is above 2^15.
//
// Fragments without shuffles: ldmatrix hands a lane four consecutive channels of a key, taken as the pairs (2 t, 2 t + 1) and (2 t +
// 8, 2 t + 9) of the product's inner index: any order of channels gives the same sum, and Q is read in that order. Of V,
// transposed, a lane gets two neighbouring channels of two keys, which two byte permutations (over two registers) part into
// the rows r and r + 8 of the product: a lane's outputs are two consecutive channels.
//
// More than 16 rows are slices of 16, each an item of its own next to the others of its head.
//
// Measured: 48 sessions of up to 16,384 keys (32 / 8 heads, 0.84 GB) 161 to 168 us, 5.0 to 5.2 TB/s (282 with the queries in the
// rows of the product; 232 with spinning waits and copies that prefetch 256 bytes, of which a head's rows have 128; 163 head after
// head instead of side by side); three CTAs on an SM and four are alike. One session over 2,048 keys 8 us clustered, a call 9.
#include <ATen/ATen.h>
#include <c10/cuda/CUDAGuard.h>
#include <c10/cuda/CUDAStream.h>

#include <string>
#include <type_traits>

#include "attend_short.cuh"
#include "packed.h"

namespace rc {
namespace paged {

// kN: groups of eight rows. One group leaves registers for three CTAs on an SM.
template <int D, int kN>
struct PackedShape {
  static constexpr int ctas = kN == 1 ? 3 : 2;       // of an SM
  static constexpr int tile_bytes = kShortTile * D;  // one of K, V: 64 keys
  static constexpr int stages = (D == 128 ? 1 : 2) * (kN == 1 ? 3 : 6);
  static constexpr int scale_off = stages * 2 * tile_bytes;  // [stages][K, V][64]
  static constexpr int join_off = scale_off + stages * 2 * kShortTile;
  static constexpr int join_bytes = 24 * D * 4;
  static constexpr int bar_off = join_off + join_bytes;
  static constexpr int bytes = bar_off + 1024 + 1024;  // + alignment slack
  static_assert((bytes + 1024) * ctas <= 228 * 1024, "the CTAs of an SM");
  static_assert(kRows * (D + 2) * 4 <= stages * 2 * tile_bytes, "a CTA's rows fit its stages");
};

struct PackedShort {
  Short s;
  const uint8_t* k_scales;  // [kv_heads, pages, page_size]
  const uint8_t* v_scales;
  int64_t k_scale_page, k_scale_head, v_scale_page, v_scale_head;
};

// Place of 16-byte chunk c of row r of a tile as TMA's swizzle lays it out (rows of 128 or 64 bytes).
template <int D>
__device__ __forceinline__ uint32_t chunk_at(int r, int c) {
  return D == 128 ? r * 128 + ((c ^ (r & 7)) << 4) : r * 64 + ((c ^ ((r >> 1) & 3)) << 4);
}

// log2 of a scale byte.
__device__ __forceinline__ float scale_log2(int byte) { return byte == kNanScale ? __uint_as_float(0x7fffffffu) : static_cast<float>(byte - 127); }

__device__ __forceinline__ int load_byte(uint32_t shared) {
  uint32_t v;
  asm volatile("ld.shared.u8 %0, [%1];" : "=r"(v) : "r"(shared) : "memory");
  return static_cast<int>(v);
}

__device__ __forceinline__ uint32_t transpose_8x8(uint32_t v) {
  uint32_t out;
  asm volatile("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(out) : "r"(v));
  return out;
}

constexpr float kFewRescale = 8.0f;  // log2 of how far a score may be above the maximum
constexpr float kUnitTop = 7.0f;     // log2 of the largest weight when the unit moves,
constexpr float kUnitRoom = 15.0f;   // and of what it may grow to before the unit moves again

template <typename T>
__device__ __forceinline__ float2 two_of(uint32_t v);
template <>
__device__ __forceinline__ float2 two_of<__nv_bfloat16>(uint32_t v) {
  return make_float2(__uint_as_float(v << 16), __uint_as_float(v & 0xffff0000u));
}
template <>
__device__ __forceinline__ float2 two_of<__half>(uint32_t v) { return __half22float2(*reinterpret_cast<const __half2*>(&v)); }

template <typename T, int D, bool kCluster, int kN>
__global__ void __launch_bounds__(kShortThreads, PackedShape<D, kN>::ctas)
    packed_short_kernel(const __grid_constant__ PageMaps maps, const __grid_constant__ PackedShort ps) {
  using Shape = PackedShape<D, kN>;
  constexpr int kKeys = kShortTile / kGroups;  // keys of a warp
  static_assert(kKeys == 16, "a warp's keys are one inner step of P V");
  extern __shared__ __align__(1024) uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  uint8_t* scales = smem + Shape::scale_off;
  uint64_t* full = reinterpret_cast<uint64_t*>(smem + Shape::bar_off);
  uint64_t* empty = full + Shape::stages;
  float* join_ml = reinterpret_cast<float*>(empty + Shape::stages);  // [key groups][rows][maximum, sum]: 64 rows in all
  int* work = reinterpret_cast<int*>(join_ml + 128);                 // begin, end, sequence, its first place; warps' sums
  const Short& p = ps.s;
  const Args& a = p.a;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;

  let_later();
  if (threadIdx.x == 0) {
    for (int s = 0; s < Shape::stages; ++s) {
      mbar_init(&full[s], 33);  // the boxes' bytes, and every producer lane's scales
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
    __syncthreads();
  } else if (warp < 4) {
    place_share(p, work);
  }
  // which of the heads, and slice of rows, that are taken side by side
  const int sides = p.par * p.slices, beside = static_cast<int>(blockIdx.x) % sides;
  const int slice = kCluster ? static_cast<int>(blockIdx.x) / p.cluster % p.slices : beside / p.par, side = kCluster ? 0 : beside - slice * p.par;
  const int row0 = slice * 8 * kN;
  int s, base, begin, end;
  if (kCluster) {
    const int index = static_cast<int>(blockIdx.x) / p.cluster, rank = static_cast<int>(blockIdx.x) - index * p.cluster, item = index / p.slices;
    s = item / a.kv_heads;
    const SeqWork w(a, s);
    if (row0 >= w.q_len * a.group) {  // no rows: the whole cluster
      if (threadIdx.x == 0 && slice == 0) report_rows(a, s);
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
      const int n = w.tiles * (a.kv_heads / p.par);
      if (at >= base + n) {
        base += n;
        ++s;
        continue;
      }
      const int place = (at - base) / w.tiles, t0 = (at - base) - place * w.tiles, head = place * p.par + side;
      const int t1 = min(w.tiles, t0 + end - at);
      if (row0 >= w.q_len * a.group) {  // a slice without rows
        at += t1 - t0;
        continue;
      }
      const TileRange<kShortTile> range(Sight(a, w.kv_len, w.q_len), 0, w.q_len);
      const int* table = a.table + s * a.table_row + head * a.table_head;
      // lanes 0-7 bring the scales of K, 8-15 those of V, eight keys each (eight never cross a page's end)
      const int part = lane & 7;
      const uint8_t* scale_base = lane < 8 ? ps.k_scales + head * ps.k_scale_head : ps.v_scales + head * ps.v_scale_head;
      const int64_t scale_page = lane < 8 ? ps.k_scale_page : ps.v_scale_page;
      for (int t = t0; t < t1; ++t) {
        const int first = range.tile(t) * kShortTile;
        const Boxes<kShortTile> boxes(a.tiling, first, w.kv_len);
        int row = 0, page = -1;
        if (lane < boxes.count) page = boxes.page(table, a.pages, a.tiling, first, lane, &row, a.status);
        const uint8_t* from = nullptr;
        if (lane < 16 && first + part * 8 < w.kv_len) {
          const int key = first + part * 8, block = key / a.tiling.page, held = table[block];
          if (held >= 0 && held < a.pages) from = scale_base + held * scale_page + (key - block * a.tiling.page);
        }
        ok = __all_sync(0xffffffffu, mbar_wait_park(&empty[stage], phase ^ 1, a.status, kTimeoutProducer));
        if (!ok) break;
        if (lane == 0) {
          if (boxes.count > 0) mbar_arrive_expect_tx(&full[stage], boxes.count * boxes.rows * D * 2);
          else mbar_arrive(&full[stage]);
        }
        __syncwarp();
        if (lane < boxes.count) {
          const bool wide = boxes.rows == kShortTile;
          uint8_t* k = smem + stage * 2 * Shape::tile_bytes + lane * boxes.rows * D;
          load_page_box(k, wide ? &maps.k_wide : &maps.k_step, &full[stage], 0, row, head, page);
          load_page_box(k + Shape::tile_bytes, wide ? &maps.v_wide : &maps.v_step, &full[stage], 0, row, head, page);
        }
        if (lane < 16) {
          // (a page outside of the pool reads as zeros: a source of no bytes leaves the scale at 0, and its codes are 0)
          const uint32_t dst = smem_u32(scales + stage * 2 * kShortTile + lane * 8);
          asm volatile("cp.async.ca.shared.global [%0], [%1], 8, %2;" ::"r"(dst), "l"(from != nullptr ? from : ps.k_scales),
                       "r"(from != nullptr ? 8 : 0)
                       : "memory");
        }
        asm volatile("cp.async.mbarrier.arrive.noinc.shared::cta.b64 [%0];" ::"r"(smem_u32(&full[stage])) : "memory");
        if (++stage == Shape::stages) {
          stage = 0;
          phase ^= 1;
        }
      }
      at += t1 - t0;
    }
    asm volatile("cp.async.wait_all;" ::: "memory");
    if (kCluster) {
      if (lane == 0 && slice == 0) report_rows(a, s);
      cluster_sync_all();
      cluster_sync_all();
    }
    return;
  }

  // ---------------- consumers ----------------
  const int kg = warp;  // its keys
  const int r0 = lane >> 2, quad = lane & 3;
  // place of this lane's operand rows for ldmatrix: keys 0-7 and 8-15 of the warp's, of chunks 0 and 1; chunks c and c + 1 lie at
  // that ^ 16 c (tiles begin on 1,024 bytes, and the swizzle turns the same bits)
  const uint32_t operand = smem_u32(smem) + chunk_at<D>(kg * kKeys + (lane & 15), lane >> 4);
  bool ok = true;
  for (int at = begin; kCluster || at < end;) {  // a cluster's CTA goes round once, also without tiles
    const SeqWork w(a, s);
    const int n = w.tiles * (a.kv_heads / p.par);
    if (!kCluster && at >= base + n) {
      base += n;
      ++s;
      continue;
    }
    const int place = kCluster ? static_cast<int>(blockIdx.x) / p.cluster / p.slices - s * a.kv_heads : (at - base) / w.tiles;
    const int t0 = kCluster ? begin : (at - base) - place * w.tiles, head = place * p.par + side;
    const int t1 = kCluster ? end : min(w.tiles, t0 + end - at);
    if (row0 >= w.q_len * a.group) {  // a slice without rows
      at += t1 - t0;
      continue;
    }
    const Sight sight(a, w.kv_len, w.q_len);
    const TileRange<kShortTile> range(sight, 0, w.q_len);

    // Q as the right operand: row r0 of each group of eight, channels 16 c + 4 quad + 0 .. 3
    uint32_t q[kN][D / 16][2];
    float row_scale[kN][2];  // of the raw scores of rows 2 quad, 2 quad + 1, with log2(e)
    int last[kN][2], low[kN][2];
#pragma unroll
    for (int g = 0; g < kN; ++g) {
      const int row = row0 + g * 8 + r0, query = row / a.group, h = head * a.group + row - query * a.group;
      const bool valid = query < w.q_len;
      const T* src = static_cast<const T*>(a.q) + static_cast<int64_t>(w.q_first + query) * a.q_token + h * a.q_head + quad * 4;
      float top = 0.0f;
#pragma unroll
      for (int c = 0; c < D / 16; ++c) {
        const uint2 x = valid ? *reinterpret_cast<const uint2*>(src + c * 16) : make_uint2(0u, 0u);
        q[g][c][0] = x.x;
        q[g][c][1] = x.y;
      }
#pragma unroll
      for (int c = 0; c < D / 16; ++c)
#pragma unroll
        for (int i = 0; i < 2; ++i) {
          const float2 f = two_of<T>(q[g][c][i]);
          top = fmaxf(top, fmaxf(fabsf(f.x), fabsf(f.y)));
        }
      top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 1));
      top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 2));
      // 2^(6 - e) for a largest magnitude of 2^e and above (e within what leaves both factors numbers)
      const int e = max(static_cast<int>(__float_as_uint(top) >> 23) - 127, -120);
      const float up = __uint_as_float(static_cast<uint32_t>(127 + 6 - e) << 23);
      const float scale = a.scale_log2 * __uint_as_float(static_cast<uint32_t>(127 - 6 + e) << 23);
#pragma unroll
      for (int c = 0; c < D / 16; ++c)
#pragma unroll
        for (int i = 0; i < 2; ++i) {
          const float2 f = two_of<T>(q[g][c][i]);
          q[g][c][i] = pack_f16x2(f.x * up, f.y * up);
        }
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        row_scale[g][i] = __shfl_sync(0xffffffffu, scale, (2 * quad + i) * 4);
        last[g][i] = sight.last(min((row0 + g * 8 + 2 * quad + i) / a.group, w.q_len - 1));
        low[g][i] = sight.low(last[g][i]);
      }
    }
    const int rows_here = w.q_len * a.group - row0;  // or fewer: 8 kN
    // bounds over the queries, for tiles that need no mask
    const int all_last = sight.last(0), all_low = sight.low(sight.last(w.q_len - 1));
    const int any_low = sight.low(all_last);

    float o[kN][D / 16][4];  // channels 16 c + 2 r0 of rows 2 quad, 2 quad + 1, and the channels after them
#pragma unroll
    for (int g = 0; g < kN; ++g)
#pragma unroll
      for (int c = 0; c < D / 16; ++c)
#pragma unroll
        for (int e = 0; e < 4; ++e) o[g][c][e] = 0.0f;
    float m[kN][2], l[kN][2];  // a maximum that no score is more than 2^8 above; this lane's part of the sum
#pragma unroll
    for (int g = 0; g < kN; ++g) {
      m[g][0] = m[g][1] = -INFINITY;
      l[g][0] = l[g][1] = 0.0f;
    }
    float unit[kN][2];  // o is in units of 2^unit
#pragma unroll
    for (int g = 0; g < kN; ++g) unit[g][0] = unit[g][1] = -INFINITY;

    for (int t = t0; t < t1; ++t) {
      const int first = range.tile(t) * kShortTile;
      if (ok) ok = __all_sync(0xffffffffu, mbar_wait_park(&full[stage], phase, a.status, kTimeoutEpilogue));
      if (ok) {
        const uint32_t k_at = operand + stage * 2 * Shape::tile_bytes, v_at = k_at + Shape::tile_bytes;
        // scales of this lane's keys r0, r0 + 8 of the warp's
        const uint32_t scale_at = smem_u32(scales) + stage * 2 * kShortTile + kg * kKeys + r0;
        const int k_scale[2] = {load_byte(scale_at), load_byte(scale_at + 8)};
        int v_scale[2] = {load_byte(scale_at + kShortTile), load_byte(scale_at + kShortTile + 8)};
        float sc[kN][4];  // keys r0, r0 + 8 (pairs) of rows 2 quad, 2 quad + 1
#pragma unroll
        for (int g = 0; g < kN; ++g)
#pragma unroll
          for (int e = 0; e < 4; ++e) sc[g][e] = 0.0f;
#pragma unroll
        for (int c = 0; c < D / 16; c += 2) {
          uint32_t b[4];  // keys 0-7 and 8-15 of chunk c, and of chunk c + 1
          ldmatrix_x4(b, k_at ^ (c << 4));
#pragma unroll
          for (int i = 0; i < 2; ++i) {
            const uint32_t k4[4] = {codes_to_half2(b[2 * i]), codes_to_half2(b[2 * i + 1]), upper_codes_to_half2(b[2 * i]),
                                    upper_codes_to_half2(b[2 * i + 1])};
#pragma unroll
            for (int g = 0; g < kN; ++g) mma_16816(sc[g], k4, q[g][c + i][0], q[g][c + i][1], __half());
          }
        }
        const float factor[2] = {scale_value(k_scale[0]), scale_value(k_scale[1])};
#pragma unroll
        for (int g = 0; g < kN; ++g)
#pragma unroll
          for (int e = 0; e < 4; ++e) sc[g][e] *= factor[e >> 1] * row_scale[g][e & 1];
        const bool whole = first + kShortTile - 1 <= all_last && (first >= all_low || first + kShortTile <= a.sinks);
        uint32_t keep[2] = {0xffffffffu, 0xffffffffu};  // (of V's operand: keys 2 quad, 2 quad + 1 and those 8 on)
        if (!whole) {
          // a key that no query sees counts for nothing: neither its scales (never read, perhaps) nor its codes
#pragma unroll
          for (int i = 0; i < 2; ++i) {
            const int key = first + kg * kKeys + r0 + 8 * i;
            if (!(key < w.kv_len && (key >= any_low || key < a.sinks))) v_scale[i] = 0;
#pragma unroll
            for (int g = 0; g < kN; ++g)
#pragma unroll
              for (int e = 0; e < 2; ++e)
                if (!(key <= last[g][e] && key < w.kv_len && (key >= low[g][e] || key < a.sinks))) sc[g][2 * i + e] = -INFINITY;
            keep[i] = 0;
#pragma unroll
            for (int e = 0; e < 2; ++e) {
              const int of = first + kg * kKeys + 2 * quad + e + 8 * i;
              if (of < w.kv_len && (of >= any_low || of < a.sinks)) keep[i] |= 0xffffu << (16 * e);
            }
          }
        }
        const float v_log[2] = {scale_log2(v_scale[0]), scale_log2(v_scale[1])};
        bool grows = false;
#pragma unroll
        for (int g = 0; g < kN; ++g)
#pragma unroll
          for (int e = 0; e < 2; ++e)
            grows = grows || fmaxf(sc[g][e], sc[g][2 + e]) > m[g][e] + kFewRescale ||
                    fmaxf(sc[g][e] + v_log[0], sc[g][2 + e] + v_log[1]) > unit[g][e] + kUnitRoom;
        if (__any_sync(0xffffffffu, grows)) {
#pragma unroll
          for (int g = 0; g < kN; ++g)
#pragma unroll
            for (int e = 0; e < 2; ++e) {
              float top = fmaxf(sc[g][e], sc[g][2 + e]), high = fmaxf(sc[g][e] + v_log[0], sc[g][2 + e] + v_log[1]);
#pragma unroll
              for (int x = 4; x < 32; x <<= 1) {
                top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, x));
                high = fmaxf(high, __shfl_xor_sync(0xffffffffu, high, x));
              }
              top = fmaxf(top, m[g][e]);
              high = fmaxf(high - kUnitTop, unit[g][e]);
              l[g][e] *= fade(m[g][e], top);
              m[g][e] = top;
              const float faded = fade(unit[g][e], high);
              unit[g][e] = high;
#pragma unroll
              for (int c = 0; c < D / 16; ++c) {
                o[g][c][e] *= faded;
                o[g][c][2 + e] *= faded;
              }
            }
        }
        // the probabilities for their sum, and the weights in fp16 as the right operand
        uint32_t pb[kN][2];
#pragma unroll
        for (int g = 0; g < kN; ++g) {
          const float use[2] = {base_of(m[g][0]), base_of(m[g][1])}, in[2] = {base_of(unit[g][0]), base_of(unit[g][1])};
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            l[g][e & 1] += exp2_approx(sc[g][e] - use[e & 1]);
            sc[g][e] = exp2_approx(sc[g][e] + (v_log[e >> 1] - in[e & 1]));
          }
          pb[g][0] = transpose_8x8(pack_f16x2(sc[g][0], sc[g][1]));
          pb[g][1] = transpose_8x8(pack_f16x2(sc[g][2], sc[g][3]));
        }
        // codes of keys that no query sees are taken as zeros whatever they are: 0 * NaN is NaN
#pragma unroll
        for (int c = 0; c < D / 16; c += 2) {
          uint32_t b[4];
          ldmatrix_x4_trans(b, v_at ^ (c << 4));
#pragma unroll
          for (int i = 0; i < 2; ++i) {
            const uint32_t lower = b[2 * i] & keep[0], upper = b[2 * i + 1] & keep[1];
            const uint32_t even = __byte_perm(lower, upper, 0x6420), odd = __byte_perm(lower, upper, 0x7531);
            const uint32_t v4[4] = {codes_to_half2(even), codes_to_half2(odd), upper_codes_to_half2(even), upper_codes_to_half2(odd)};
#pragma unroll
            for (int g = 0; g < kN; ++g) mma_16816(o[g][c + i], v4, pb[g][0], pb[g][1], __half());
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

    // Warps that split the keys join theirs into key group 0 through shared memory. The same lane of every warp holds the same
    // rows and channels, so the buffer is laid out by lane. Maxima become ones that no score is above.
#pragma unroll
    for (int g = 0; g < kN; ++g)
#pragma unroll
      for (int e = 0; e < 2; ++e) {
        m[g][e] += kFewRescale;
        l[g][e] *= exp2f(-kFewRescale);
#pragma unroll
        for (int x = 4; x < 32; x <<= 1) l[g][e] += __shfl_xor_sync(0xffffffffu, l[g][e], x);
        if (r0 == 0) *reinterpret_cast<float2*>(join_ml + (kg * kRows + g * 8 + 2 * quad + e) * 2) = make_float2(m[g][e], l[g][e]);
      }
    consumers_sync();
#pragma unroll
    for (int g = 0; g < kN; ++g)
#pragma unroll
      for (int e = 0; e < 2; ++e) {
        float2 ml[kGroups];
        float top = -INFINITY, total = 0.0f;
#pragma unroll
        for (int k = 0; k < kGroups; ++k) {
          ml[k] = *reinterpret_cast<const float2*>(join_ml + (k * kRows + g * 8 + 2 * quad + e) * 2);
          top = fmaxf(top, ml[k].x);
        }
        const float use = base_of(top);
#pragma unroll
        for (int k = 0; k < kGroups; ++k) total = fmaf(ml[k].y, exp2_approx(ml[k].x - use), total);
        const float root = exp2_approx(0.5f * (unit[g][e] - use));  // (its square may be below FP32's range where o times it is not)
        m[g][e] = top;
        l[g][e] = total;
#pragma unroll
        for (int c = 0; c < D / 16; ++c) {
          o[g][c][e] = o[g][c][e] * root * root;
          o[g][c][2 + e] = o[g][c][2 + e] * root * root;
        }
      }
#pragma unroll
    for (int g = 0; g < kN; ++g) {
      float4* buf = reinterpret_cast<float4*>(smem + Shape::join_off) + lane;
      if (kg > 0) {
#pragma unroll
        for (int c = 0; c < D / 16; ++c) buf[((kg - 1) * (D / 16) + c) * 32] = make_float4(o[g][c][0], o[g][c][1], o[g][c][2], o[g][c][3]);
      }
      consumers_sync();
      if (kg == 0) {
#pragma unroll
        for (int k = 0; k < kGroups - 1; ++k)
#pragma unroll
          for (int c = 0; c < D / 16; ++c) {
            const float4 x = buf[(k * (D / 16) + c) * 32];
            o[g][c][0] += x.x;
            o[g][c][1] += x.y;
            o[g][c][2] += x.z;
            o[g][c][3] += x.w;
          }
      }
      consumers_sync();
    }
    if (kCluster) {
      float* res = reinterpret_cast<float*>(smem);  // [kRows][D]: every tile has been consumed
      float* res_ml = res + kRows * D;              // [kRows][2]
      if (kg == 0) {
#pragma unroll
        for (int g = 0; g < kN; ++g)
#pragma unroll
          for (int e = 0; e < 2; ++e) {
            const int row = g * 8 + 2 * quad + e;
#pragma unroll
            for (int c = 0; c < D / 16; ++c) *reinterpret_cast<float2*>(res + row * D + c * 16 + 2 * r0) = make_float2(o[g][c][e], o[g][c][2 + e]);
            if (r0 == 0) *reinterpret_cast<float2*>(res_ml + row * 2) = make_float2(m[g][e], l[g][e]);
          }
      }
      cluster_sync_all();
      join_few_cluster<T, D>(p, w, head, row0, rows_here, res, res_ml, ok);
      cluster_sync_all();  // the others have read this CTA's rows
      return;
    }
    if (kg == 0 && ok) {
      const int item_first = base + place * w.tiles;
      const bool starts = item_first >= begin, ends = item_first + w.tiles <= end;
#pragma unroll
      for (int g = 0; g < kN; ++g)
#pragma unroll
        for (int e = 0; e < 2; ++e) {
          const int row = g * 8 + 2 * quad + e, packed = row0 + row, query = packed / a.group, h = head * a.group + packed - query * a.group;
          if (query >= w.q_len) continue;
          const int64_t token = w.q_first + query;
          if (starts && ends) {
            const float inv = inverse(l[g][e]);
            T* dst = static_cast<T*>(a.out) + token * a.out_token + h * a.out_head + 2 * r0;
#pragma unroll
            for (int c = 0; c < D / 16; ++c) *reinterpret_cast<uint32_t*>(dst + c * 16) = pack2<T>(o[g][c][e] * inv, o[g][c][2 + e] * inv);
            if (a.lse != nullptr && r0 == 0) a.lse[token * a.heads + h] = log_sum(m[g][e], l[g][e]);
          } else {
            const int64_t slot = (2 * static_cast<int64_t>(blockIdx.x) + (starts ? 1 : 0)) * kRows + row;
#pragma unroll
            for (int c = 0; c < D / 16; ++c) *reinterpret_cast<float2*>(p.part_o + slot * D + c * 16 + 2 * r0) = make_float2(o[g][c][e], o[g][c][2 + e]);
            if (r0 == 0) *reinterpret_cast<float2*>(p.part_ml + slot * 2) = make_float2(m[g][e], l[g][e]);
          }
        }
    }
    at += t1 - t0;
  }
}

template <typename T, int D, int kN>
struct PackedForm {
  static constexpr int ctas = PackedShape<D, kN>::ctas, bytes = PackedShape<D, kN>::bytes, tile_bytes = PackedShape<D, kN>::tile_bytes, boxes = 1;
  static constexpr auto clustered() { return packed_short_kernel<T, D, true, kN>; }
};

template <typename T, int D, int kN>
void packed_configure(int device) {
  static bool known[64] = {};
  bool& configured = known[device & 63];
  if (configured) return;
  RC_CUDA(cudaFuncSetAttribute(packed_short_kernel<T, D, false, kN>, cudaFuncAttributeMaxDynamicSharedMemorySize, PackedShape<D, kN>::bytes));
  RC_CUDA(cudaFuncSetAttribute(packed_short_kernel<T, D, true, kN>, cudaFuncAttributeMaxDynamicSharedMemorySize, PackedShape<D, kN>::bytes));
  RC_CUDA(cudaFuncSetAttribute(packed_short_kernel<T, D, true, kN>, cudaFuncAttributeNonPortableClusterSizeAllowed, 1));
  configured = true;
}

// Tensor map of codes [pages, page_size, heads, D] with boxes of D channels x `box` rows of one head and page.
CUtensorMap code_map(const at::Tensor& t, int box) {
  CUtensorMap map;
  const cuuint64_t d = static_cast<cuuint64_t>(t.size(3));
  const cuuint64_t dims[4] = {d, static_cast<cuuint64_t>(t.size(1)), static_cast<cuuint64_t>(t.size(2)), static_cast<cuuint64_t>(t.size(0))};
  const auto stride = [&](int64_t i) { return static_cast<cuuint64_t>(t.size(i) == 1 ? 16 : t.stride(i)); };  // (of one place: any)
  const cuuint64_t strides[3] = {stride(1), stride(2), stride(0)};
  const cuuint32_t boxes[4] = {static_cast<cuuint32_t>(d), static_cast<cuuint32_t>(box), 1, 1};
  const cuuint32_t ones[4] = {1, 1, 1, 1};
  const CUresult res = encode_tiled_fn()(&map, CU_TENSOR_MAP_DATA_TYPE_UINT8, 4, t.data_ptr(), dims, strides, boxes, ones,
                                         CU_TENSOR_MAP_INTERLEAVE_NONE, d == 128 ? CU_TENSOR_MAP_SWIZZLE_128B : CU_TENSOR_MAP_SWIZZLE_64B,
                                         CU_TENSOR_MAP_L2_PROMOTION_L2_128B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
  RC_CHECK(res == CUDA_SUCCESS, "cuTensorMapEncodeTiled (codes) failed (code " + std::to_string(static_cast<int>(res)) + ")");
  return map;
}

// CTAs of an item's cluster, or 0 for the line.
template <typename T, int D, int kN>
int packed_cluster(const Args& a, int slices, int device) {
  return short_cluster<PackedForm<T, D, kN>>(static_cast<int64_t>(a.seqs) * a.kv_heads * slices, short_tiles(a),
                                             Tiling::of(a.tiling.page, kShortTile).step, a.seqs > 1 && a.table_head == 0, device);
}

template <typename T, int D, int kN>
void packed_launch(const Args& a, int slices, const at::Tensor& k_codes, const at::Tensor& v_codes, const Packed& k, const Packed& v,
                   const at::Tensor& like, cudaStream_t stream, int device) {
  using Shape = PackedShape<D, kN>;
  PackedShort ps{};
  Short& p = ps.s;
  p.a = a;
  p.a.tiling = Tiling::of(a.tiling.page, kShortTile);
  ps.k_scales = k.scales;
  ps.v_scales = v.scales;
  ps.k_scale_page = k.scale_page;
  ps.k_scale_head = k.scale_head;
  ps.v_scale_page = v.scale_page;
  ps.v_scale_head = v.scale_head;
  const PageMaps maps = page_maps(k_codes, v_codes, p.a.tiling, kShortTile, code_map);
  packed_configure<T, D, kN>(device);
  const int64_t items = static_cast<int64_t>(a.seqs) * a.kv_heads * slices, slots = sm_count(device) * Shape::ctas;
  p.par = 1;
  p.rows = 8 * kN;
  p.slices = slices;
  p.cluster = packed_cluster<T, D, kN>(a, slices, device);
  if (p.cluster > 0) {
    launch(packed_short_kernel<T, D, true, kN>, dim3(static_cast<unsigned>(items * p.cluster)), kShortThreads, Shape::bytes, p.cluster,
           stream, maps, ps);
    return;
  }
  // The line's CTAs take the KV heads side by side: the rows of neighbouring heads lie next to each other, and 128 bytes here
  // and there are too little for HBM (48 sessions of up to 16,384 keys: 163 us head after head).
  for (p.par = std::min(a.kv_heads, 32); a.kv_heads % p.par != 0;) --p.par;
  while (p.par > 1 && p.par * slices > slots)  // (few SMs)
    for (--p.par; a.kv_heads % p.par != 0;) --p.par;
  const int sides = p.par * slices, ctas = static_cast<int>(std::min<int64_t>(slots / sides, items / sides * (short_tiles(a) + 1))) * sides;
  RC_CHECK(items * (kRows / 4) < (1ll << 31), "too many sequences and rows for one launch");
  const int64_t floats = 2ll * ctas * kRows * (D + 2), ints = 1 + 2ll * a.seqs;
  at::Tensor workspace = new_tensor({floats + ints}, like, at::kFloat);
  p.part_o = workspace.data_ptr<float>();
  p.part_ml = p.part_o + 2ll * ctas * kRows * D;
  int* line = reinterpret_cast<int*>(p.part_o + floats);
  p.line = {line, line + 1, line + 1 + a.seqs};
  launch(packed_short_kernel<T, D, false, kN>, dim3(ctas), kShortThreads, Shape::bytes, 0, stream, maps, ps);
  launch(short_join_kernel<T, D>, dim3(static_cast<unsigned>(items * (kRows / 4))), 128, 0, 0, stream, p);
}

int packed_slices(int rows) { return (rows + 15) / 16; }

template <typename T, int D>
void packed_rows(const Args& a, int max_q_len, const at::Tensor& k_codes, const at::Tensor& v_codes, const Packed& k, const Packed& v,
                 const at::Tensor& like, cudaStream_t stream, int device) {
  const int rows = max_q_len * a.group;
  rows <= 8 ? packed_launch<T, D, 1>(a, 1, k_codes, v_codes, k, v, like, stream, device)
            : packed_launch<T, D, 2>(a, packed_slices(rows), k_codes, v_codes, k, v, like, stream, device);
}

void attend_packed_short(const Args& a, int head_dim, bool half, const at::Tensor& k_codes, const at::Tensor& v_codes, const Packed& k,
                         const Packed& v, int max_q_len, const at::Tensor& like, cudaStream_t stream, int device) {
  if (head_dim == 128)
    half ? packed_rows<__half, 128>(a, max_q_len, k_codes, v_codes, k, v, like, stream, device)
         : packed_rows<__nv_bfloat16, 128>(a, max_q_len, k_codes, v_codes, k, v, like, stream, device);
  else
    half ? packed_rows<__half, 64>(a, max_q_len, k_codes, v_codes, k, v, like, stream, device)
         : packed_rows<__nv_bfloat16, 64>(a, max_q_len, k_codes, v_codes, k, v, like, stream, device);
}

template <int D, int kN>
int packed_form(const Args& a, int slices, int device) {
  packed_configure<__nv_bfloat16, D, kN>(device);
  return packed_cluster<__nv_bfloat16, D, kN>(a, slices, device);
}

std::string packed_form_name(const Args& a, int head_dim, int max_q_len, int device) {
  const int rows = max_q_len * a.group, slices = packed_slices(rows);
  const int cluster = head_dim == 128 ? (rows <= 8 ? packed_form<128, 1>(a, 1, device) : packed_form<128, 2>(a, slices, device))
                                      : (rows <= 8 ? packed_form<64, 1>(a, 1, device) : packed_form<64, 2>(a, slices, device));
  return (slices > 1 ? std::to_string(slices) + " slices, " : std::string("few rows, ")) +
         (cluster > 0 ? "cluster " + std::to_string(cluster) : "line");
}

}  // namespace paged
}  // namespace rc
