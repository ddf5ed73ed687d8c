// Attention of few query rows (single tokens, drafts) over pages in 8 bits (packed.h), for sm_100a.
//
// What bounds it: reading the codes once, half the bytes of a 16-bit cache in the same time per product, so the design of
// attend_short.cu is kept (a producer warp streams tiles of 64 keys with TMA, four consumer warps with 16 keys each on
// mma.sync, work in a line or in clusters) and what comes between the bytes and the products is kept short:
//
// Codes become fp16 in registers, exactly, two by one conversion; the products are fp16 whatever the rows' type. Q is brought
// to fp16 by a power of two for each row that puts its largest magnitude between 2^6 and 2^7: exact for what is at least 2^-20
// of that, off by at most 2^-31 of it below. Scales multiply neither codes nor channels: K's multiply the scores (FP32),
// V's multiply the probabilities, which are rounded to fp16 for the product (half a step of 2^-11; their sum is not): a warp
// keeps the largest exponent of V's scales that it has seen as the unit of its output, so that no product overflows, and
// rescales the output when it grows, as with the maximum of the scores.
//
// Fragments without shuffles: a row of K lies as 16 bytes a chunk; ldmatrix hands a lane four consecutive channels of a key,
// taken as its pairs (2 t, 2 t + 1) and (2 t + 8, 2 t + 9) of the product's inner index: any order of channels gives the same sum,
// and Q is read in that order. Of V, transposed, a lane gets two neighbouring channels of two keys, which two byte
// permutations (over two registers) part into the even and the odd channel's product; a lane's outputs are then four
// consecutive channels.
#include <ATen/ATen.h>
#include <c10/cuda/CUDAGuard.h>
#include <c10/cuda/CUDAStream.h>

#include <string>
#include <type_traits>

#include "attend_short.cuh"
#include "packed.h"

namespace rc {
namespace paged {

template <int D>
struct PackedShape {
  static constexpr int tile_bytes = kShortTile * D;  // one of K, V: 64 keys
  static constexpr int stages = D == 128 ? 6 : 10;
  static constexpr int scale_off = stages * 2 * tile_bytes;  // [stages][K, V][64]
  static constexpr int join_off = scale_off + stages * 2 * kShortTile;
  static constexpr int join_bytes = 24 * D * 4;
  static constexpr int bar_off = join_off + join_bytes;
  static constexpr int bytes = bar_off + 1024 + 1024;  // + alignment slack
  static_assert((bytes + 1024) * kShortCtasPerSm <= 228 * 1024, "two CTAs per SM");
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

// 2^(e - base) of a scale byte as the factor of a probability; e above base never comes.
__device__ __forceinline__ float relative_scale(int e, int base) {
  const int d = 127 + e - base;
  return e == kNanScale ? __uint_as_float(0x7fffffffu) : d <= 0 ? 0.0f : __uint_as_float(static_cast<uint32_t>(d) << 23);
}

template <typename T>
__device__ __forceinline__ float2 two_of(uint32_t v);
template <>
__device__ __forceinline__ float2 two_of<__nv_bfloat16>(uint32_t v) {
  return make_float2(__uint_as_float(v << 16), __uint_as_float(v & 0xffff0000u));
}
template <>
__device__ __forceinline__ float2 two_of<__half>(uint32_t v) { return __half22float2(*reinterpret_cast<const __half2*>(&v)); }

template <typename T, int D, bool kCluster>
__global__ void __launch_bounds__(kShortThreads, kShortCtasPerSm)
    packed_short_kernel(const __grid_constant__ PageMaps maps, const __grid_constant__ PackedShort ps) {
  using Shape = PackedShape<D>;
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
        ok = __all_sync(0xffffffffu, mbar_wait(&empty[stage], phase ^ 1, a.status, kTimeoutProducer));
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
      if (lane == 0) report_rows(a, s);
      cluster_sync_all();
      cluster_sync_all();
    }
    return;
  }

  // ---------------- consumers ----------------
  const int kg = warp;  // its keys
  const int r0 = lane >> 2, quad = lane & 3, c0 = quad * 2;
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

    // this thread's two rows, channels 16 j + 4 quad + 0 .. 3
    int row_q[2], row_h[2], last[2], low[2];
    bool valid[2];
    float row_scale[2];  // of a raw score, with log2(e)
    uint32_t q[D / 16][4];
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      const int row = r0 + i * 8;
      row_q[i] = row / a.group;
      row_h[i] = head * a.group + row - row_q[i] * a.group;
      valid[i] = row_q[i] < w.q_len;
      last[i] = sight.last(min(row_q[i], w.q_len - 1));
      low[i] = sight.low(last[i]);
      const T* src = static_cast<const T*>(a.q) + static_cast<int64_t>(w.q_first + row_q[i]) * a.q_token + row_h[i] * a.q_head + quad * 4;
#pragma unroll
      for (int j = 0; j < D / 16; ++j) {
        const uint2 x = valid[i] ? *reinterpret_cast<const uint2*>(src + j * 16) : make_uint2(0u, 0u);
        q[j][i] = x.x;
        q[j][i + 2] = x.y;
      }
      float top = 0.0f;
#pragma unroll
      for (int j = 0; j < D / 16; ++j)
#pragma unroll
        for (int h = 0; h < 2; ++h) {
          const float2 f = two_of<T>(q[j][i + 2 * h]);
          top = fmaxf(top, fmaxf(fabsf(f.x), fabsf(f.y)));
        }
      top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 1));
      top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 2));
      // 2^(6 - e) for a largest magnitude of 2^e and above (e within what leaves both factors numbers)
      const int e = max(static_cast<int>(__float_as_uint(top) >> 23) - 127, -120);
      const float up = __uint_as_float(static_cast<uint32_t>(127 + 6 - e) << 23);
      row_scale[i] = a.scale_log2 * __uint_as_float(static_cast<uint32_t>(127 - 6 + e) << 23);
#pragma unroll
      for (int j = 0; j < D / 16; ++j)
#pragma unroll
        for (int h = 0; h < 2; ++h) {
          const float2 f = two_of<T>(q[j][i + 2 * h]);
          q[j][i + 2 * h] = pack_f16x2(f.x * up, f.y * up);
        }
    }
    const int rows_here = w.q_len * a.group;  // or fewer: kRows
    // bounds over the queries, for tiles that need no mask
    const int all_last = sight.last(0), all_low = sight.low(sight.last(w.q_len - 1));
    const int any_low = sight.low(all_last);

    float o[D / 8][4];  // products: 2 j the even channels of chunk j, 2 j + 1 the odd ones
#pragma unroll
    for (int i = 0; i < D / 8; ++i)
#pragma unroll
      for (int e = 0; e < 4; ++e) o[i][e] = 0.0f;
    float m[2] = {-INFINITY, -INFINITY}, l[2] = {0.0f, 0.0f};
    int unit = 1;  // o is in units of 2^(unit - 127): the largest scale of V so far

    for (int t = t0; t < t1; ++t) {
      const int first = range.tile(t) * kShortTile;
      if (ok) ok = __all_sync(0xffffffffu, mbar_wait(&full[stage], phase, a.status, kTimeoutEpilogue));
      if (ok) {
        const uint32_t kb = smem_u32(smem + stage * 2 * Shape::tile_bytes);
        const uint32_t vb = kb + Shape::tile_bytes;
        // scales of this lane's keys: c0, c0 + 1, c0 + 8, c0 + 9 of the warp's
        const uint8_t* ks = scales + stage * 2 * kShortTile + kg * kKeys + c0;
        const uint32_t k2[2] = {*reinterpret_cast<const uint16_t*>(ks), *reinterpret_cast<const uint16_t*>(ks + 8)};
        const uint32_t v2[2] = {*reinterpret_cast<const uint16_t*>(ks + kShortTile), *reinterpret_cast<const uint16_t*>(ks + kShortTile + 8)};
        float sc[2][4];
#pragma unroll
        for (int j = 0; j < 2; ++j)
#pragma unroll
          for (int e = 0; e < 4; ++e) sc[j][e] = 0.0f;
        // S = Q K^T: matrices (keys 0-7, chunk 2 c), (keys 0-7, 2 c + 1), (keys 8-15, 2 c), (keys 8-15, 2 c + 1)
#pragma unroll
        for (int c = 0; c < D / 32; ++c) {
          uint32_t b[4];
          ldmatrix_x4(b, kb + chunk_at<D>(kg * kKeys + (lane & 7) + ((lane >> 4) << 3), c * 2 + ((lane >> 3) & 1)));
#pragma unroll
          for (int e = 0; e < 4; ++e)
            mma_16816(sc[e >> 1], q[2 * c + (e & 1)], codes_to_half2(b[e]), upper_codes_to_half2(b[e]), __half());
        }
        const bool whole = first + kShortTile - 1 <= all_last && (first >= all_low || first + kShortTile <= a.sinks);
        // a key that no query sees counts for nothing: neither its scales (never read, perhaps) nor its codes
        bool seen[2][2] = {{true, true}, {true, true}};
#pragma unroll
        for (int j = 0; j < 2; ++j)
#pragma unroll
          for (int e = 0; e < 2; ++e) {
            const int key = first + kg * kKeys + j * 8 + c0 + e;
            if (!whole) seen[j][e] = key < w.kv_len && (key >= any_low || key < a.sinks);
            const float factor = scale_value((k2[j] >> (8 * e)) & 0xff);
#pragma unroll
            for (int i = 0; i < 2; ++i) {
              float& x = sc[j][2 * i + e];
              x *= factor;
              if (!whole && !(key <= last[i] && key < w.kv_len && (key >= low[i] || key < a.sinks))) x = -INFINITY;
            }
          }
        int above = 0;
#pragma unroll
        for (int j = 0; j < 2; ++j)
#pragma unroll
          for (int e = 0; e < 2; ++e) {
            const int byte = (v2[j] >> (8 * e)) & 0xff;
            if (seen[j][e] && byte != kNanScale) above = max(above, byte);
          }
        const int before = unit;
        unit = max(unit, __reduce_max_sync(0xffffffffu, above));
        const float grown = relative_scale(before, unit);
        float alpha[2];
#pragma unroll
        for (int i = 0; i < 2; ++i) {
          float mx = fmaxf(fmaxf(sc[0][2 * i], sc[0][2 * i + 1]), fmaxf(sc[1][2 * i], sc[1][2 * i + 1]));
          mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 1));
          mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 2));
          const float top = fmaxf(m[i], mx * row_scale[i]);
          const float use = base_of(top);
          const float faded = fade(m[i], top);
          m[i] = top;
          float sum = 0.0f;
#pragma unroll
          for (int j = 0; j < 2; ++j)
#pragma unroll
            for (int e = 0; e < 2; ++e) {
              const float x = exp2_approx(fmaf(sc[j][2 * i + e], row_scale[i], -use));
              sc[j][2 * i + e] = x;
              sum += x;
            }
          l[i] = l[i] * faded + sum;
          alpha[i] = faded * grown;
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
        uint32_t keep[2] = {0xffffffffu, 0xffffffffu};
#pragma unroll
        for (int j = 0; j < 2; ++j) {
#pragma unroll
          for (int e = 0; e < 2; ++e) {
            const float factor = seen[j][e] ? relative_scale((v2[j] >> (8 * e)) & 0xff, unit) : 0.0f;
            sc[j][e] *= factor;
            sc[j][2 + e] *= factor;
          }
          if (!whole) keep[j] = (seen[j][0] ? 0xffffu : 0u) | (seen[j][1] ? 0xffff0000u : 0u);
        }
        const uint32_t pa[4] = {pack_f16x2(sc[0][0], sc[0][1]), pack_f16x2(sc[0][2], sc[0][3]), pack_f16x2(sc[1][0], sc[1][1]),
                                pack_f16x2(sc[1][2], sc[1][3])};
        // O += P V: matrices (keys 0-7, chunk 2 c), (keys 8-15, 2 c), (keys 0-7, 2 c + 1), (keys 8-15, 2 c + 1); codes of keys
        // that no query sees are taken as zeros whatever they are: 0 * NaN is NaN
#pragma unroll
        for (int c = 0; c < D / 32; ++c) {
          uint32_t b[4];
          ldmatrix_x4_trans(b, vb + chunk_at<D>(kg * kKeys + (lane & 7) + (((lane >> 3) & 1) << 3), c * 2 + (lane >> 4)));
#pragma unroll
          for (int h = 0; h < 2; ++h) {
            const uint32_t lower = b[2 * h] & keep[0], upper = b[2 * h + 1] & keep[1];
            const uint32_t even = __byte_perm(lower, upper, 0x6420), odd = __byte_perm(lower, upper, 0x7531);
            mma_16816(o[4 * c + 2 * h], pa, codes_to_half2(even), upper_codes_to_half2(even), __half());
            mma_16816(o[4 * c + 2 * h + 1], pa, codes_to_half2(odd), upper_codes_to_half2(odd), __half());
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
    const float in_units = scale_value(unit);
#pragma unroll
    for (int i = 0; i < D / 8; ++i)
#pragma unroll
      for (int e = 0; e < 4; ++e) o[i][e] *= in_units;
    join_warps<D>(o, m, l, join_ml, smem + Shape::join_off, rows_here);
    // four consecutive channels of row i of chunk j
    auto four = [&](int i, int j) { return make_float4(o[2 * j][2 * i], o[2 * j + 1][2 * i], o[2 * j][2 * i + 1], o[2 * j + 1][2 * i + 1]); };
    if (kCluster) {
      float* res = reinterpret_cast<float*>(smem);  // [kRows][D]: every tile has been consumed
      float* res_ml = res + kRows * D;              // [kRows][2]
      consumers_sync();
      if (kg == 0) {
#pragma unroll
        for (int i = 0; i < 2; ++i) {
          const int row = r0 + 8 * i;
#pragma unroll
          for (int j = 0; j < D / 16; ++j) *reinterpret_cast<float4*>(res + row * D + j * 16 + quad * 4) = four(i, j);
          if (quad == 0) *reinterpret_cast<float2*>(res_ml + row * 2) = make_float2(m[i], l[i]);
        }
      }
      cluster_sync_all();
      join_few_cluster<T, D>(p, w, head, rows_here, res, res_ml, ok);
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
          T* dst = static_cast<T*>(a.out) + token * a.out_token + row_h[i] * a.out_head + quad * 4;
#pragma unroll
          for (int j = 0; j < D / 16; ++j) {
            const float4 x = four(i, j);
            *reinterpret_cast<uint2*>(dst + j * 16) = make_uint2(pack2<T>(x.x * inv, x.y * inv), pack2<T>(x.z * inv, x.w * inv));
          }
          if (a.lse != nullptr && quad == 0) a.lse[token * a.heads + row_h[i]] = log_sum(m[i], l[i]);
        } else {
          const int64_t slot = (2 * static_cast<int64_t>(blockIdx.x) + (starts ? 1 : 0)) * kRows + r0 + 8 * i;
#pragma unroll
          for (int j = 0; j < D / 16; ++j) *reinterpret_cast<float4*>(p.part_o + slot * D + j * 16 + quad * 4) = four(i, j);
          if (quad == 0) *reinterpret_cast<float2*>(p.part_ml + slot * 2) = make_float2(m[i], l[i]);
        }
      }
    }
    at += t1 - t0;
  }
}

template <typename T, int D>
struct PackedForm {
  static constexpr int bytes = PackedShape<D>::bytes, tile_bytes = PackedShape<D>::tile_bytes, boxes = 1;
  static constexpr auto clustered() { return packed_short_kernel<T, D, true>; }
};

template <typename T, int D>
void packed_configure(int device) {
  static bool known[64] = {};
  bool& configured = known[device & 63];
  if (configured) return;
  RC_CUDA(cudaFuncSetAttribute(packed_short_kernel<T, D, false>, cudaFuncAttributeMaxDynamicSharedMemorySize, PackedShape<D>::bytes));
  RC_CUDA(cudaFuncSetAttribute(packed_short_kernel<T, D, true>, cudaFuncAttributeMaxDynamicSharedMemorySize, PackedShape<D>::bytes));
  RC_CUDA(cudaFuncSetAttribute(packed_short_kernel<T, D, true>, cudaFuncAttributeNonPortableClusterSizeAllowed, 1));
  configured = true;
}

// Tensor map of codes [pages, page_size, heads, D] with boxes of D channels x `box` rows of one head and page.
CUtensorMap code_map(const at::Tensor& t, int box) {
  CUtensorMap map;
  const cuuint64_t d = static_cast<cuuint64_t>(t.size(3));
  const cuuint64_t dims[4] = {d, static_cast<cuuint64_t>(t.size(1)), static_cast<cuuint64_t>(t.size(2)), static_cast<cuuint64_t>(t.size(0))};
  const cuuint64_t strides[3] = {static_cast<cuuint64_t>(t.stride(1)), static_cast<cuuint64_t>(t.stride(2)), static_cast<cuuint64_t>(t.stride(0))};
  const cuuint32_t boxes[4] = {static_cast<cuuint32_t>(d), static_cast<cuuint32_t>(box), 1, 1};
  const cuuint32_t ones[4] = {1, 1, 1, 1};
  const CUresult res = encode_tiled_fn()(&map, CU_TENSOR_MAP_DATA_TYPE_UINT8, 4, t.data_ptr(), dims, strides, boxes, ones,
                                         CU_TENSOR_MAP_INTERLEAVE_NONE, d == 128 ? CU_TENSOR_MAP_SWIZZLE_128B : CU_TENSOR_MAP_SWIZZLE_64B,
                                         CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
  RC_CHECK(res == CUDA_SUCCESS, "cuTensorMapEncodeTiled (codes) failed (code " + std::to_string(static_cast<int>(res)) + ")");
  return map;
}

template <typename T, int D>
void packed_launch(const Args& a, const at::Tensor& k_codes, const at::Tensor& v_codes, const Packed& k, const Packed& v,
                   const at::Tensor& like, cudaStream_t stream, int device) {
  using Shape = PackedShape<D>;
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
  packed_configure<T, D>(device);
  const int64_t items = static_cast<int64_t>(a.seqs) * a.kv_heads, slots = sm_count(device) * kShortCtasPerSm;
  p.cluster = short_cluster<PackedForm<T, D>>(items, short_tiles(a), p.a.tiling.step, a.seqs > 1, device);
  if (p.cluster > 0) {
    launch(packed_short_kernel<T, D, true>, dim3(static_cast<unsigned>(items * p.cluster)), kShortThreads, Shape::bytes, p.cluster,
           stream, maps, ps);
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
  launch(packed_short_kernel<T, D, false>, dim3(ctas), kShortThreads, Shape::bytes, 0, stream, maps, ps);
  launch(short_join_kernel<T, D>, dim3(static_cast<unsigned>(items * (kRows / 4))), 128, 0, 0, stream, p);
}

void attend_packed_short(const Args& a, int head_dim, bool half, const at::Tensor& k_codes, const at::Tensor& v_codes, const Packed& k,
                         const Packed& v, const at::Tensor& like, cudaStream_t stream, int device) {
  if (head_dim == 128)
    half ? packed_launch<__half, 128>(a, k_codes, v_codes, k, v, like, stream, device)
         : packed_launch<__nv_bfloat16, 128>(a, k_codes, v_codes, k, v, like, stream, device);
  else
    half ? packed_launch<__half, 64>(a, k_codes, v_codes, k, v, like, stream, device)
         : packed_launch<__nv_bfloat16, 64>(a, k_codes, v_codes, k, v, like, stream, device);
}

}  // namespace paged
}  // namespace rc
