// What the rotation kernels share (rows on their own, into pages of a 16-bit or an 8-bit cache): vectors, the argument block,
// a token's sines, its place in the pages.
#pragma once

#include <ATen/ATen.h>
#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include <algorithm>

#include "../common/host.h"
#include "paged.h"
#include "rope_plan.h"

namespace rc {
namespace rotary {

constexpr int kThreads = 256;

template <typename T>
struct Vec;  // one 16-byte vector of T as floats

template <>
struct Vec<__nv_bfloat16> {
  static constexpr int n = 8;
  static __device__ __forceinline__ void unpack(const uint4& u, float* f) {
    const uint32_t w[4] = {u.x, u.y, u.z, u.w};
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      f[2 * i] = __uint_as_float(w[i] << 16);
      f[2 * i + 1] = __uint_as_float(w[i] & 0xffff0000u);
    }
  }
  static __device__ __forceinline__ uint4 pack(const float* f) {
    uint32_t w[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      __nv_bfloat162 v = __floats2bfloat162_rn(f[2 * i], f[2 * i + 1]);
      w[i] = *reinterpret_cast<uint32_t*>(&v);
    }
    return make_uint4(w[0], w[1], w[2], w[3]);
  }
};

template <>
struct Vec<__half> {
  static constexpr int n = 8;
  static __device__ __forceinline__ void unpack(const uint4& u, float* f) {
    const uint32_t w[4] = {u.x, u.y, u.z, u.w};
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const float2 v = __half22float2(*reinterpret_cast<const __half2*>(&w[i]));
      f[2 * i] = v.x;
      f[2 * i + 1] = v.y;
    }
  }
  static __device__ __forceinline__ uint4 pack(const float* f) {
    uint32_t w[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      __half2 v = __floats2half2_rn(f[2 * i], f[2 * i + 1]);
      w[i] = *reinterpret_cast<uint32_t*>(&v);
    }
    return make_uint4(w[0], w[1], w[2], w[3]);
  }
};

template <>
struct Vec<float> {
  static constexpr int n = 4;
  static __device__ __forceinline__ void unpack(const uint4& u, float* f) {
    f[0] = __uint_as_float(u.x);
    f[1] = __uint_as_float(u.y);
    f[2] = __uint_as_float(u.z);
    f[3] = __uint_as_float(u.w);
  }
  static __device__ __forceinline__ uint4 pack(const float* f) {
    return make_uint4(__float_as_uint(f[0]), __float_as_uint(f[1]), __float_as_uint(f[2]), __float_as_uint(f[3]));
  }
};

struct Rows {  // one tensor [tokens, heads, head_dim]: byte strides
  const char* src;
  char* dst;
  int64_t src_token, src_head, dst_token, dst_head;
  int heads;
  int per;     // heads of a thread
  int groups;  // threads that share a token and vector
};

struct Args {
  Rows q, k, v;            // v only where pages are written (heads == 0 otherwise)
  const void* positions;   // [tokens, axes], int32 or float32
  int position_float;
  int axes;
  int ends[4];             // first pair after each axis's section
  const float* turns;      // [2, pairs]: hi, lo
  const double* exact;     // [pairs]: the same in FP64
  float sign;              // -1 turns back
  int tokens, pairs;
  // the paged form: k and v rows go to page table[seq][at / page], row at % page
  const int* table;
  const int* kv_lens;
  const int* cu_q;
  int seqs, table_width, page, pages;
  int64_t table_row;
  int64_t page_k, page_v;  // page strides in bytes (dst_token / dst_head are strides inside a page)
  int* status;
};

constexpr float kFar = 16777216.0f;  // 2^24: from here on FP32 does not hold every whole number

// The fraction of a turn of pair j at a token's position, in FP64.
__device__ __forceinline__ double turn_part(const Args& a, int token, int j) {
  const int axis = j < a.ends[0] ? 0 : j < a.ends[1] ? 1 : j < a.ends[2] ? 2 : 3;
  const int64_t at = static_cast<int64_t>(token) * a.axes + axis;
  const double p = a.position_float ? static_cast<double>(static_cast<const float*>(a.positions)[at])
                                    : static_cast<double>(static_cast<const int*>(a.positions)[at]);
  const double t = __ldg(a.exact + j), n = p * t;
  return (n - rint(n)) + fma(p, t, -n);
}
__device__ __forceinline__ float far_part(const Args& a, int token, int j) { return static_cast<float>(turn_part(a, token, j)); }

// Sines of the kPairs pairs of a token that begin at vec * kPairs (sn times a.sign): within a few ULP (kFine), or from the special
// function unit (within 2^-21).
template <bool kFine, int kPairs>
__device__ __forceinline__ void sines(const Args& a, int token, int vec, float (&cs)[kPairs], float (&sn)[kPairs]) {
  float p[4];
  bool far = false;
#pragma unroll
  for (int x = 0; x < 4; ++x) {
    p[x] = 0.0f;
    if (x < a.axes) {
      const int64_t at = static_cast<int64_t>(token) * a.axes + x;
      p[x] = a.position_float ? static_cast<const float*>(a.positions)[at]
                              : static_cast<float>(static_cast<const int*>(a.positions)[at]);
      far = far || fabsf(p[x]) >= kFar;
    }
  }
#pragma unroll
  for (int e0 = 0; e0 < kPairs; e0 += 2) {
    const int j0 = vec * kPairs + e0;
    // (the table is written once, long before: the one input that no kernel writes)
    const float2 hi2 = __ldg(reinterpret_cast<const float2*>(a.turns + j0));
    const float2 lo2 = __ldg(reinterpret_cast<const float2*>(a.turns + a.pairs + j0));
#pragma unroll
    for (int e = 0; e < 2; ++e) {
      const int j = j0 + e;
      const float pos = j < a.ends[0] ? p[0] : j < a.ends[1] ? p[1] : j < a.ends[2] ? p[2] : p[3];
      const float hi = e ? hi2.y : hi2.x, lo = e ? lo2.y : lo2.x;
      float part = fmaf(pos, lo, fmaf(pos, hi, -rintf(pos * hi)));
      if (far) part = far_part(a, token, j);
      if (kFine) {
        sincospif(2.0f * part, &sn[e0 + e], &cs[e0 + e]);
      } else {
        __sincosf(6.283185307179586f * part, &sn[e0 + e], &cs[e0 + e]);
      }
      sn[e0 + e] *= a.sign;
    }
  }
}

// Turns one vector of neighbours (x), or the vectors x and y half a head apart.
template <bool kHalves, int kVec, int kPairs>
__device__ __forceinline__ void turn(float (&x)[kVec], float (&y)[kVec], const float (&cs)[kPairs], const float (&sn)[kPairs]) {
  if (kHalves) {
#pragma unroll
    for (int e = 0; e < kVec; ++e) {
      const float u = x[e] * cs[e % kPairs] - y[e] * sn[e % kPairs];
      y[e] = x[e] * sn[e % kPairs] + y[e] * cs[e % kPairs];
      x[e] = u;
    }
  } else {
#pragma unroll
    for (int e = 0; e < kVec / 2; ++e) {
      const float u = x[2 * e] * cs[e] - x[2 * e + 1] * sn[e];
      x[2 * e + 1] = x[2 * e] * sn[e] + x[2 * e + 1] * cs[e];
      x[2 * e] = u;
    }
  }
}

// Page of a new token and its row there; false for tokens that no sequence has and for pages outside of the pool (which the
// thread with `tells` reports).
__device__ __forceinline__ bool place(const Args& a, int token, bool tells, int* page, int* row) {
  int lo = 0, hi = a.seqs - 1;  // the last sequence that starts at or before the token
  while (lo < hi) {
    const int mid = (lo + hi + 1) >> 1;
    if (a.cu_q[mid] <= token) lo = mid;
    else hi = mid - 1;
  }
  const int begin = a.cu_q[lo], end = a.cu_q[lo + 1];
  if (token < begin || token >= end) return false;  // tokens past the last sequence belong to none
  const int at = a.kv_lens[lo] - end + token;
  const int slot = at >= 0 ? at / a.page : -1;
  *page = slot >= 0 && slot < a.table_width ? a.table[lo * a.table_row + slot] : -1;
  *row = at - slot * a.page;
  if (*page >= 0 && *page < a.pages) return true;
  if (tells && a.status != nullptr) atomicCAS(a.status + kPagedWord, 0, kPageRange);
  return false;
}

// How the heads of a tensor are spread over threads: as many to a thread as leave every SM a full set of threads, and then
// evenly. `rows`: threads of a head (tokens x vectors). Returns the most heads of a thread.
inline int spread_heads(Args& a, int64_t rows, int sms) {
  const int heads = a.q.heads + a.k.heads + a.v.heads;
  const int most = static_cast<int>(std::max<int64_t>(1, std::min<int64_t>(64, rows * heads / (static_cast<int64_t>(sms) * 2048))));
  int widest = 1;
  for (Rows* r : {&a.q, &a.k, &a.v}) {
    r->groups = (r->heads + most - 1) / most;
    r->per = r->groups > 0 ? (r->heads + r->groups - 1) / r->groups : 1;
    widest = std::max(widest, r->per);
  }
  return widest;
}

// The rotation's part of the arguments, checked: positions [tokens, axes].
inline void set_rotation(Args& a, const at::Tensor& positions, const RopePlan& plan, int64_t tokens, int64_t head_dim,
                  const at::Device& device) {
  const int axes = static_cast<int>(plan.sections.size());
  RC_CHECK(head_dim == 2 * plan.pairs, "the rotation is for another head_dim");
  RC_CHECK(plan.turns.device() == device, "the rotation's table is on another device");
  a.pairs = static_cast<int>(plan.pairs);
  int end = 0;
  for (int i = 0; i < 4; ++i) {
    if (i < axes) end += static_cast<int>(plan.sections[i]);
    a.ends[i] = end;
  }
  RC_CHECK(positions.device() == device && positions.dim() == 2 && positions.size(0) == tokens &&
               positions.size(1) == axes && positions.is_contiguous() &&
               (positions.scalar_type() == at::kInt || positions.scalar_type() == at::kFloat),
           "positions must be a contiguous int32 or float32 [tokens, axes] tensor on the same device");
  a.positions = positions.data_ptr();
  a.position_float = positions.scalar_type() == at::kFloat;
  a.axes = axes;
  a.turns = plan.turns.data_ptr<float>();
  a.exact = plan.exact.data_ptr<double>();
  a.tokens = static_cast<int>(tokens);
}

inline bool vector_rows(const at::Tensor& t) {
  const int64_t size = t.element_size();
  return t.dim() == 3 && t.stride(2) == 1 && (t.stride(0) * size) % 16 == 0 && (t.stride(1) * size) % 16 == 0 &&
         reinterpret_cast<uintptr_t>(t.data_ptr()) % 16 == 0;
}

}  // namespace rotary
}  // namespace rc
