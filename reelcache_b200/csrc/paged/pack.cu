// Rows into pages of an 8-bit cache, quantised on the way (with the rotation of q and k, or as they are), and out again, for
// sm_100a. The format is in packed.h.
//
// Into pages: the lanes that hold a row's vectors find its largest magnitude with shuffles (as integers, so that infinities and
// NaN come out on top), and the scale's exponent follows from its bits: m * 2^e with m from 1 to 2 needs k = e - 8, or e - 7
// where m > 1.75 (448 = 1.75 * 2^8). The product with 2^-k is exact, so a code is rounded once, from the rotated row in FP32.
// Layout of threads as in the rotation: a thread owns a vector of eight channels (two, half a head apart) of a token for as
// many heads as leave every SM full, so that its sines are computed once.
//
// What bounds it: memory (3 bytes a number of k and v, 4 of q), and the chain of a row: load, turn, maximum over the row's lanes,
// codes. Three chunks of 4,680 tokens and 12 heads 46.1 us, 4.7 TB/s (41.2 with sines of FP32 alone); 25.8 us without q and the
// rotation (129 MB, 5.0 TB/s).
//
// Out of pages: a block looks up where its rows lie, then every thread turns vectors of sixteen codes into 32 bytes, a whole
// sector in one store (16-byte stores: 42 us where these take 36.4, five chunks of 12 heads, 216 MB).
#include <ATen/ATen.h>
#include <ATen/MemoryOverlap.h>
#include <c10/cuda/CUDAGuard.h>
#include <c10/cuda/CUDAStream.h>

#include "packed.h"
#include "rotary.cuh"

namespace rc {
namespace pack {

using rotary::kThreads;
using rotary::Rows;
using rotary::Vec;

struct Exponents {  // range of the scales' exponents: code * 2^k is a number of the 16-bit type
  int low, high;
};

Exponents exponents_of(at::ScalarType type) { return type == at::kHalf ? Exponents{-15, 7} : Exponents{-124, 119}; }

struct Args {
  rotary::Args a;
  uint8_t* k_scales;
  uint8_t* v_scales;
  int64_t k_scale_page, k_scale_head, v_scale_page, v_scale_head;
  Exponents range;
};

// max(top, |a|, |b|), NaN if one of them is.
__device__ __forceinline__ float top_of(float top, float a, float b) {
  float r;
  asm("max.NaN.f32 %0, %1, %2, %3;" : "=f"(r) : "f"(top), "f"(fabsf(a)), "f"(fabsf(b)));
  return r;
}

__device__ __forceinline__ uint2 codes_of_vec(const float (&x)[8], float inverse, bool finite) {
  if (!finite) return make_uint2(0x7f7f7f7fu, 0x7f7f7f7fu);
  return make_uint2(paged::codes_of(x[0] * inverse, x[1] * inverse) | paged::codes_of(x[2] * inverse, x[3] * inverse) << 16,
                    paged::codes_of(x[4] * inverse, x[5] * inverse) | paged::codes_of(x[6] * inverse, x[7] * inverse) << 16);
}

// kTurn: 0 rows as they are, 1 pairs are neighbours, 2 half a head apart.
// (Blocks on an SM, two heads a round, three chunks of 4,680 tokens and 36 heads: neighbours 46.3 us with four, 48.5 with five; half
// a head apart 49.2 with two, 58.8 with three; one head after the other 10 us more.)
template <typename T, int kTurn, int kHeads>
__global__ void __launch_bounds__(kThreads, kTurn == 2 ? 2 : kTurn == 1 ? 4 : 5) pack_kernel(const __grid_constant__ Args p) {
  paged::let_later();
  paged::after_earlier();
  constexpr bool kHalves = kTurn == 2;
  constexpr int kPairs = kHalves ? 8 : 4, kParts = kHalves ? 2 : 1;
  const rotary::Args& a = p.a;
  const int per_row = a.pairs / kPairs;  // lanes of a row: 4, 8 or 16
  const int log_row = 31 - __clz(per_row);
  const int local = threadIdx.x >> log_row, vec = threadIdx.x & (per_row - 1), tokens = kThreads >> log_row;
  const int64_t token64 = static_cast<int64_t>(blockIdx.x) * tokens + local;
  const int token = static_cast<int>(min(token64, static_cast<int64_t>(a.tokens)));
  const int y = blockIdx.y;
  const bool is_q = y < a.q.groups, is_k = !is_q && y < a.q.groups + a.k.groups;
  const Rows& r = is_q ? a.q : is_k ? a.k : a.v;
  const int first = (is_q ? y : is_k ? y - a.q.groups : y - a.q.groups - a.k.groups) * r.per;
  const int heads = min(r.heads - first, r.per);
  bool active = token < a.tokens;
  const int part_bytes = a.pairs * 2;  // from the first half of a head to the second
  const char* src = r.src + token * r.src_token + first * r.src_head + vec * 16;

  uint4 raw[kHeads][kParts];
  auto load = [&](int i, int head) {  // the next head's vectors
#pragma unroll
    for (int s = 0; s < kParts; ++s) {
      raw[i][s] = make_uint4(0, 0, 0, 0);
      if (active && head < heads) raw[i][s] = *reinterpret_cast<const uint4*>(src + s * part_bytes);
    }
    src += r.src_head;
  };
#pragma unroll
  for (int i = 0; i < kHeads; ++i) load(i, i);

  char* dst = r.dst + first * r.dst_head;
  uint8_t* scale = nullptr;
  int64_t scale_head = 0;
  if (is_q) {
    dst += token * r.dst_token + vec * 16;
  } else {
    int page, row;
    if (active && rotary::place(a, token, vec == 0, &page, &row)) {
      dst += page * (is_k ? a.page_k : a.page_v) + row * r.dst_token + vec * 8;
      scale_head = is_k ? p.k_scale_head : p.v_scale_head;
      scale = (is_k ? p.k_scales : p.v_scales) + page * (is_k ? p.k_scale_page : p.v_scale_page) + row + first * scale_head;
    } else {
      active = false;
    }
  }

  // A code that falls to its neighbour is 2^-3 off, so k is turned nearer than FP32's sines allow: by sines of FP64 as the sums of
  // two numbers, computed once for all of the thread's heads. What is left are two roundings, 2^-24 each (14 to
  // 22 of 21.6 million codes are not the exact rotation's).
  float cs[kPairs] = {}, sn[kPairs] = {}, cs_low[kPairs] = {}, sn_low[kPairs] = {};
  const bool turned = kTurn != 0 && (is_q || is_k);
  if (turned && active && is_q) rotary::sines<false>(a, token, vec, cs, sn);
  if (turned && active && is_k) {
#pragma unroll 1
    for (int e = 0; e < kPairs; ++e) {
      double s, c;
      sincospi(2.0 * rotary::turn_part(a, token, vec * kPairs + e), &s, &c);
#pragma unroll
      for (int i = 0; i < kPairs; ++i)
        if (i == e) {
          cs[i] = static_cast<float>(c);
          sn[i] = static_cast<float>(s);
          cs_low[i] = static_cast<float>(c - static_cast<double>(cs[i]));
          sn_low[i] = static_cast<float>(s - static_cast<double>(sn[i]));
        }
    }
  }

  // a round of heads at a time, step by step, so that their chains run next to each other
  for (int done = 0; done < heads; done += kHeads) {
    float x[kHeads][8], y2[kHeads][8];
    uint32_t top[kHeads];
#pragma unroll
    for (int i = 0; i < kHeads; ++i) {
      Vec<T>::unpack(raw[i][0], x[i]);
      if (kHalves) Vec<T>::unpack(raw[i][kParts - 1], y2[i]);
      if (turned && is_q) {  // (as beside 16-bit pages: products with low parts of 0 would turn infinities into NaN)
        rotary::turn<kHalves>(x[i], y2[i], cs, sn);
      } else if (turned) {
#pragma unroll
        for (int e = 0; e < kPairs; ++e) {
          float& p = x[i][kHalves ? e : 2 * e];
          float& q = kHalves ? y2[i][e] : x[i][2 * e + 1];
          const float u = fmaf(p, cs[e], fmaf(-q, sn[e], fmaf(p, cs_low[e], -q * sn_low[e])));
          q = fmaf(p, sn[e], fmaf(q, cs[e], fmaf(p, sn_low[e], q * cs_low[e])));
          p = u;
        }
      }
      float most = 0.0f;
#pragma unroll
      for (int e = 0; e < 8; e += 2) {
        most = top_of(most, x[i][e], x[i][e + 1]);
        if (kHalves) most = top_of(most, y2[i][e], y2[i][e + 1]);
      }
      top[i] = __float_as_uint(most);
      load(i, done + kHeads + i);  // before the stores, which the compiler must take for ones to the same memory
    }
    if (!is_q) {
      for (int o = per_row >> 1; o > 0; o >>= 1)
#pragma unroll
        for (int i = 0; i < kHeads; ++i) top[i] = max(top[i], __shfl_xor_sync(0xffffffffu, top[i], o));
    }
#pragma unroll
    for (int i = 0; i < kHeads; ++i) {
      const bool here = active && done + i < heads;
      char* to = dst;
      dst += r.dst_head;
      if (is_q) {
        if (here) *reinterpret_cast<uint4*>(to) = Vec<T>::pack(x[i]);
        if (here && kHalves) *reinterpret_cast<uint4*>(to + part_bytes) = Vec<T>::pack(y2[i]);
        continue;
      }
      const bool finite = top[i] < 0x7f800000u;
      const int power = min(max(static_cast<int>(top[i] >> 23) - 127 - 8 + ((top[i] & 0x7fffffu) > 0x600000u), p.range.low), p.range.high);
      const float inverse = __uint_as_float(static_cast<uint32_t>(127 - power) << 23);
      if (here) *reinterpret_cast<uint2*>(to) = codes_of_vec(x[i], inverse, finite);
      if (here && kHalves) *reinterpret_cast<uint2*>(to + a.pairs) = codes_of_vec(y2[i], inverse, finite);
      if (here && vec == 0) *scale = static_cast<uint8_t>(finite ? power + 127 : paged::kNanScale);
      scale += scale_head;
    }
  }
}

template <typename T, int kTurn>
void pack_launch(Args p, cudaStream_t stream, int sms) {
  const int per_row = p.a.pairs / (kTurn == 2 ? 8 : 4);
  const int64_t rows = static_cast<int64_t>(p.a.tokens) * per_row;
  const int widest = rotary::spread_heads(p.a, rows, sms);
  const int64_t blocks = (rows + kThreads - 1) / kThreads;
  const int groups = p.a.q.groups + p.a.k.groups + p.a.v.groups;
  RC_CHECK(blocks < (1ll << 31) && groups < 65536, "too many tokens or heads for one launch");
  const dim3 grid(static_cast<unsigned>(blocks), groups);
  paged::launch(widest == 1 ? pack_kernel<T, kTurn, 1> : pack_kernel<T, kTurn, 2>, grid, kThreads, 0, 0, stream, p);
}

template <int kTurn>
void pack_dispatch(const Args& p, bool half, cudaStream_t stream, int sms) {
  half ? pack_launch<__half, kTurn>(p, stream, sms) : pack_launch<__nv_bfloat16, kTurn>(p, stream, sms);
}

// k and v, checked, and where they go; everything but q and the rotation.
void set_rows(Args& p, const at::Tensor& k, const at::Tensor& v, const at::Tensor& k_codes, const at::Tensor& k_scales,
              const at::Tensor& v_codes, const at::Tensor& v_scales, const at::Tensor& table, const at::Tensor& kv_lens,
              const at::Tensor& cu_q, const c10::optional<at::Tensor>& status) {
  check_cuda_tensor(k, "k");
  const at::ScalarType type = k.scalar_type();
  RC_CHECK(type == at::kBFloat16 || type == at::kHalf, "rows for a packed cache are bf16 or fp16");
  RC_CHECK(k.dim() == 3 && v.sizes() == k.sizes() && (k.size(2) == 64 || k.size(2) == 128),
           "k and v are [tokens, kv_heads, head_dim] with head_dim 64 or 128");
  RC_CHECK(v.scalar_type() == type && v.device() == k.device(), "k and v must agree on type and device");
  RC_CHECK((k.numel() == 0 || rotary::vector_rows(k)) && (v.numel() == 0 || rotary::vector_rows(v)),
           "rows must have unit inner stride and 16-byte aligned strides and base");
  RC_CHECK(k.size(0) < (1ll << 31), "too many tokens for one launch");
  const paged::Table t = paged::check_table(table, kv_lens, cu_q, k.device());
  const paged::Packed kp = paged::check_packed(k_codes, k_scales, k.size(1), k.size(2), k.device(), "k_pages");
  const paged::Packed vp = paged::check_packed(v_codes, v_scales, k.size(1), k.size(2), k.device(), "v_pages");
  RC_CHECK(kp.count == vp.count && kp.size == vp.size, "k_pages and v_pages must have the same pages");
  RC_CHECK(k_codes.data_ptr() != v_codes.data_ptr() && k_scales.data_ptr() != v_scales.data_ptr(), "k_pages and v_pages must be different pages");
  for (const at::Tensor* w : {&k_codes, &k_scales, &v_codes, &v_scales}) at::assert_no_internal_overlap(*w);
  p.range = exponents_of(type);
  p.k_scales = const_cast<uint8_t*>(kp.scales);
  p.v_scales = const_cast<uint8_t*>(vp.scales);
  p.k_scale_page = kp.scale_page;
  p.k_scale_head = kp.scale_head;
  p.v_scale_page = vp.scale_page;
  p.v_scale_head = vp.scale_head;
  rotary::Args& a = p.a;
  a.tokens = static_cast<int>(k.size(0));
  a.pairs = static_cast<int>(k.size(2) / 2);
  a.k = {static_cast<const char*>(k.data_ptr()), static_cast<char*>(k_codes.data_ptr()), k.stride(0) * 2, k.stride(1) * 2,
         kp.token_stride, kp.head_stride, static_cast<int>(k.size(1))};
  a.v = {static_cast<const char*>(v.data_ptr()), static_cast<char*>(v_codes.data_ptr()), v.stride(0) * 2, v.stride(1) * 2,
         vp.token_stride, vp.head_stride, static_cast<int>(v.size(1))};
  a.table = t.table;
  a.kv_lens = t.kv_lens;
  a.cu_q = t.cu_q;
  a.seqs = t.seqs;
  a.table_width = t.width;
  a.table_row = t.row;
  a.page = kp.size;
  a.pages = kp.count;
  a.page_k = kp.page_stride;
  a.page_v = vp.page_stride;
  a.status = status_ptr(status);
  if (t.seqs == 0) a.k.heads = a.v.heads = 0;  // k and v belong to no sequence
}

void written_pages(const at::Tensor& k_codes, const at::Tensor& k_scales, const at::Tensor& v_codes, const at::Tensor& v_scales) {
  for (const at::Tensor* w : {&k_codes, &k_scales, &v_codes, &v_scales}) written(*w);
}

// -- out of pages -----------------------------------------------------------------------------------------------------

struct Read {
  paged::Packed pages[2];  // K, V
  const uint8_t* codes[2];
  char* out[2];            // [rows, kv_heads, head_dim]
  const int* table;
  int64_t table_row;
  const int* starts;       // [seqs + 1]
  int seqs, width, heads, rows;
  int tokens;              // of a block
  int log_vecs;            // vectors of sixteen channels of a head
  paged::Divider heads_by;
  int* status;
};

constexpr int kReadVectors = 512;  // of a block, about
constexpr int kReadTokens = 256;    // of a block, at most

// A block reads K or V of some consecutive rows: first a thread for each finds its place, then all fetch vectors of sixteen
// channels (many small blocks: deeper loops at fewer blocks were slower).
template <typename T>
__global__ void __launch_bounds__(kThreads) read_kernel(const __grid_constant__ Read p) {
  __shared__ int64_t code_at[kReadTokens], scale_at[kReadTokens];  // (-1: reads as zeros, -2: a row of no sequence)
  paged::let_later();
  paged::after_earlier();
  const int which = blockIdx.y;
  const paged::Packed& pages = which ? p.pages[1] : p.pages[0];
  const uint8_t* base = which ? p.codes[1] : p.codes[0];
  const int token0 = static_cast<int>(blockIdx.x) * p.tokens, tokens = min(p.tokens, p.rows - token0);
  if (static_cast<int>(threadIdx.x) < tokens) {
    const int token = token0 + static_cast<int>(threadIdx.x);
    int seq = 0, hi = p.seqs - 1;  // the last sequence that starts at or before the token
    while (seq < hi) {
      const int mid = (seq + hi + 1) >> 1;
      if (p.starts[mid] <= token) seq = mid;
      else hi = mid - 1;
    }
    const int begin = p.starts[seq], end = p.starts[seq + 1];
    int64_t code = -2, scale = 0;
    if (token >= begin && token < end) {
      const int pos = token - begin, slot = pos / pages.size, row = pos - slot * pages.size;
      const int page = slot < p.width ? p.table[seq * p.table_row + slot] : -1;
      if (page >= 0 && page < pages.count) {
        code = page * pages.page_stride + row * pages.token_stride;
        scale = page * pages.scale_page + row;
      } else {
        code = -1;
        if (p.status != nullptr) atomicCAS(p.status + kPagedWord, 0, kPageRange);
      }
    }
    code_at[threadIdx.x] = code;
    scale_at[threadIdx.x] = scale;
  }
  __syncthreads();
  uint4* out = reinterpret_cast<uint4*>(which ? p.out[1] : p.out[0]) + static_cast<int64_t>(token0) * p.heads * 2 * (1 << p.log_vecs);
  const int vectors = (tokens * p.heads) << p.log_vecs;
  constexpr int kDepth = 2;
  for (int v0 = threadIdx.x; v0 < vectors; v0 += kThreads * kDepth) {
    uint4 codes[kDepth];
    int scale[kDepth];
#pragma unroll
    for (int i = 0; i < kDepth; ++i) {
      const int v = v0 + i * kThreads, row = v >> p.log_vecs, vec = v - (row << p.log_vecs);
      scale[i] = -1;
      if (v >= vectors) continue;
      const int token = p.heads_by.over(row), head = row - token * p.heads;
      const int64_t at = code_at[token];
      codes[i] = make_uint4(0, 0, 0, 0);
      if (at >= 0) {
        codes[i] = *reinterpret_cast<const uint4*>(base + at + head * pages.head_stride + vec * 16);
        scale[i] = pages.scales[scale_at[token] + head * pages.scale_head];
      } else if (at == -1) {
        scale[i] = 127;
      }
    }
#pragma unroll
    for (int i = 0; i < kDepth; ++i) {
      if (scale[i] < 0) continue;
      paged::store_values<T>(out + 2 * (v0 + i * kThreads), codes[i], paged::scale_value(scale[i]));
    }
  }
}

}  // namespace pack

// Rotation of q (returned; into `out` if it is given); k rotated and v as it is, quantised, into their pages.
at::Tensor packed_append(const at::Tensor& q, const at::Tensor& k, const at::Tensor& v, const at::Tensor& positions,
                         const RopePlan& plan, const at::Tensor& k_codes, const at::Tensor& k_scales, const at::Tensor& v_codes,
                         const at::Tensor& v_scales, const at::Tensor& table, const at::Tensor& kv_lens, const at::Tensor& cu_q,
                         const c10::optional<at::Tensor>& out, const c10::optional<at::Tensor>& status) {
  check_cuda_tensor(q, "q");
  refuse_gradients({&q, &k, &v, &positions, &k_codes, &k_scales, &v_codes, &v_scales}, "append");
  if (out.has_value()) refuse_gradients({&*out}, "append");
  refuse_tangents({&q, &k, &v, &positions, &k_codes, &k_scales, &v_codes, &v_scales}, "append");
  c10::cuda::CUDAGuard guard(q.device());
  pack::Args p{};
  pack::set_rows(p, k, v, k_codes, k_scales, v_codes, v_scales, table, kv_lens, cu_q, status);
  RC_CHECK(q.dim() == 3 && q.size(0) == k.size(0) && q.size(2) == k.size(2) && q.scalar_type() == k.scalar_type() && q.device() == k.device(),
           "q is [tokens, heads, head_dim], k and v [tokens, kv_heads, head_dim], of one type and device");
  at::Tensor q_out = out.has_value() ? *out : paged::new_tensor(q.sizes(), q, q.scalar_type());
  RC_CHECK(q_out.sizes() == q.sizes() && q_out.scalar_type() == q.scalar_type() && q_out.device() == q.device(), "out must match q");
  RC_CHECK((q.numel() == 0 || rotary::vector_rows(q)) && (q.numel() == 0 || rotary::vector_rows(q_out)),
           "rows must have unit inner stride and 16-byte aligned strides and base");
  at::assert_no_internal_overlap(q_out);
  at::assert_no_partial_overlap(q_out, q);
  rotary::set_rotation(p.a, positions, plan, q.size(0), q.size(2), q.device());
  p.a.sign = 1.0f;
  p.a.q = {static_cast<const char*>(q.data_ptr()), static_cast<char*>(q_out.data_ptr()), q.stride(0) * 2, q.stride(1) * 2,
           q_out.stride(0) * 2, q_out.stride(1) * 2, static_cast<int>(q.size(1))};
  const int device = q.get_device();
  if (p.a.tokens > 0 && p.a.q.heads + p.a.k.heads > 0)
    (plan.halves ? pack::pack_dispatch<2> : pack::pack_dispatch<1>)(p, q.scalar_type() == at::kHalf, c10::cuda::getCurrentCUDAStream(device).stream(),
                                                                  sm_count(device));
  if (out.has_value()) written(*out);
  if (p.a.seqs > 0) pack::written_pages(k_codes, k_scales, v_codes, v_scales);
  return q_out;
}

// k and v as they are, quantised, into their pages.
void packed_store(const at::Tensor& k, const at::Tensor& v, const at::Tensor& k_codes, const at::Tensor& k_scales,
                  const at::Tensor& v_codes, const at::Tensor& v_scales, const at::Tensor& table, const at::Tensor& kv_lens,
                  const at::Tensor& cu_q, const c10::optional<at::Tensor>& status) {
  check_cuda_tensor(k, "k");
  refuse_gradients({&k, &v, &k_codes, &k_scales, &v_codes, &v_scales}, "store");
  refuse_tangents({&k, &v, &k_codes, &k_scales, &v_codes, &v_scales}, "store");
  c10::cuda::CUDAGuard guard(k.device());
  pack::Args p{};
  pack::set_rows(p, k, v, k_codes, k_scales, v_codes, v_scales, table, kv_lens, cu_q, status);
  if (p.a.tokens == 0 || p.a.k.heads == 0) return;
  const int device = k.get_device();
  pack::pack_dispatch<0>(p, k.scalar_type() == at::kHalf, c10::cuda::getCurrentCUDAStream(device).stream(), sm_count(device));
  pack::written_pages(k_codes, k_scales, v_codes, v_scales);
}

// The first starts[s + 1] - starts[s] tokens of every sequence s as rows starts[s] .. of two new tensors [rows, kv_heads, head_dim].
std::pair<at::Tensor, at::Tensor> packed_read(const at::Tensor& k_codes, const at::Tensor& k_scales, const at::Tensor& v_codes,
                                              const at::Tensor& v_scales, const at::Tensor& table, const at::Tensor& starts,
                                              int64_t rows, at::ScalarType type, const c10::optional<at::Tensor>& status) {
  check_cuda_tensor(k_codes, "k_pages");
  refuse_gradients({&k_codes, &k_scales, &v_codes, &v_scales}, "read");
  refuse_tangents({&k_codes, &k_scales, &v_codes, &v_scales}, "read");
  RC_CHECK(type == at::kBFloat16 || type == at::kHalf, "packed pages are read as bf16 or fp16");
  RC_CHECK(k_codes.dim() == 4 && (k_codes.size(3) == 64 || k_codes.size(3) == 128), "packed pages have a head_dim of 64 or 128");
  c10::cuda::CUDAGuard guard(k_codes.device());
  pack::Read p{};
  const int64_t heads = k_codes.size(2), d = k_codes.size(3);
  p.pages[0] = paged::check_packed(k_codes, k_scales, heads, d, k_codes.device(), "k_pages");
  p.pages[1] = paged::check_packed(v_codes, v_scales, heads, d, k_codes.device(), "v_pages");
  RC_CHECK(p.pages[0].count == p.pages[1].count && p.pages[0].size == p.pages[1].size, "k_pages and v_pages must have the same pages");
  RC_CHECK(table.device() == k_codes.device() && table.scalar_type() == at::kInt && table.dim() == 2 &&
               (table.stride(1) == 1 || table.size(1) <= 1) && table.stride(0) >= 0 && table.size(0) < (1 << 20) && table.size(1) < (1ll << 31),
           "block_table must be an int32 [seqs, width] tensor on the device of the pages (rows may be strided)");
  RC_CHECK(starts.device() == k_codes.device() && starts.scalar_type() == at::kInt && starts.is_contiguous() && starts.dim() == 1 &&
               starts.size(0) == table.size(0) + 1,
           "starts must be a contiguous int32 [seqs + 1] tensor on the device of the pages");
  RC_CHECK(rows >= 0 && rows < (1ll << 31), "too many rows");
  at::Tensor out[2];
  for (int i = 0; i < 2; ++i) out[i] = paged::new_tensor({rows, heads, d}, k_codes, type);
  if (rows == 0 || heads == 0 || table.size(0) == 0) return {out[0], out[1]};
  p.codes[0] = static_cast<const uint8_t*>(k_codes.data_ptr());
  p.codes[1] = static_cast<const uint8_t*>(v_codes.data_ptr());
  p.out[0] = static_cast<char*>(out[0].data_ptr());
  p.out[1] = static_cast<char*>(out[1].data_ptr());
  p.table = table.data_ptr<int>();
  p.table_row = table.stride(0);
  p.starts = starts.data_ptr<int>();
  p.seqs = static_cast<int>(table.size(0));
  p.width = static_cast<int>(table.size(1));
  p.heads = static_cast<int>(heads);
  p.log_vecs = d == 128 ? 3 : 2;
  p.rows = static_cast<int>(rows);
  RC_CHECK(heads < (1 << 20), "too many KV heads");
  p.heads_by = paged::Divider::of(static_cast<int>(heads));
  p.tokens = static_cast<int>(std::min<int64_t>(pack::kReadTokens, std::max<int64_t>(1, pack::kReadVectors / (heads * (d / 16)))));
  p.status = status_ptr(status);
  const int64_t blocks = (rows + p.tokens - 1) / p.tokens;
  paged::launch(type == at::kHalf ? pack::read_kernel<__half> : pack::read_kernel<__nv_bfloat16>, dim3(static_cast<unsigned>(blocks), 2),
                pack::kThreads, 0, 0, c10::cuda::getCurrentCUDAStream(k_codes.get_device()).stream(), p);
  return {out[0], out[1]};
}

}  // namespace rc
