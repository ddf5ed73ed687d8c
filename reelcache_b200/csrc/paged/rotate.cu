// Rotary positions with several axes (frame, row, column, ...) for sm_100a, on their own (forward and gradient) and
// on the way into a paged KV cache.
//
// Pair j of a head belongs to one axis a(j) and turns by phi_j = p[token][a(j)] * w_j:
//   (x_j, y_j) -> (x_j cos phi - y_j sin phi, x_j sin phi + y_j cos phi),
// the gradient is the rotation by -phi. Pairs are neighbours (2j, 2j + 1) or half a head apart (j, j + pairs).
//
// The angle is kept in turns: w_j / (2 pi) comes as the sum of two FP32 numbers hi + lo, n = rint(p hi), and
// fma(p, hi, -n) + p lo is the fraction of a turn, exact to an ULP of 0.5 however many turns p makes (p w in radians
// would lose one bit for each doubling of p). sincospi takes it from there. That holds for |p| < 2^24, which FP32 counts
// exactly; a token with a position beyond takes the fraction in FP64 (off by 2^-25 of a turn at 2^31) from w_j / (2 pi) in
// FP64: a branch that other tokens pass by.
//
// What bounds it: memory, one read and one write of q, k (and v); next, the sines. So a thread owns one 16-byte vector
// position of a token (4 or 8 pairs), computes their sines once and applies them to as many heads of one tensor as leave
// every SM full; the loads of the first heads are issued before the sines are computed. A warp access covers whole heads
// (256 bytes each). A block works on one tensor, so nothing of it branches: v takes no sines, q no pages. The fused form
// writes k and v through the block table, so the rotated keys never exist outside the cache.
//
// 16-bit types take sin and cos from the special function unit (off by at most 2^-21, a thousandth of what rounding to
// fp16 loses), fp32 takes sincospi.
// Measured: q and k of 14,400 tokens x 64 heads of 128 (472 MB moved) 75 us, 6.3 TB/s; three chunks of 4,680 tokens
// x 36 heads into pages 42.2 us, 6.1 TB/s (47 us with each store before the loads of the next heads, 51 us with one head group of q, k and v mixed per thread, 81 us with two heads
// a thread).
#include <ATen/ATen.h>
#include <ATen/MemoryOverlap.h>
#include <c10/cuda/CUDAGuard.h>
#include <c10/cuda/CUDAStream.h>

#include "rotary.cuh"

namespace rc {
namespace rotary {

// kHalves: pairs (j, j + pairs), a thread holds one vector of each half; else neighbours in one vector.
template <typename T, bool kHalves, bool kPaged, int kHeads>
__global__ void __launch_bounds__(kThreads) rotate_kernel(const __grid_constant__ Args a) {
  paged::let_later();
  paged::after_earlier();
  constexpr int kVec = Vec<T>::n;
  constexpr int kPairs = kHalves ? kVec : kVec / 2;  // pairs a thread turns
  constexpr int kParts = kHalves ? 2 : 1;            // vectors a thread holds per head
  const int per_row = a.pairs / kPairs;
  const int64_t index = static_cast<int64_t>(blockIdx.x) * kThreads + threadIdx.x;
  const int token = static_cast<int>(index / per_row);
  const int vec = static_cast<int>(index - static_cast<int64_t>(token) * per_row);
  if (token >= a.tokens) return;
  const int y = blockIdx.y;
  const bool is_q = y < a.q.groups, is_k = !is_q && y < a.q.groups + a.k.groups;
  const Rows& r = is_q ? a.q : is_k ? a.k : a.v;
  const int first = (is_q ? y : is_k ? y - a.q.groups : y - a.q.groups - a.k.groups) * r.per;
  const int count = min(r.heads - first, r.per);
  const int part_bytes = a.pairs * static_cast<int>(sizeof(T));  // from the first half of a head to the second
  const char* src = r.src + token * r.src_token + first * r.src_head + vec * 16;

  uint4 raw[kHeads][kParts];
  auto load = [&](int i, int head) {
    if (head < count) {
#pragma unroll
      for (int s = 0; s < kParts; ++s) raw[i][s] = *reinterpret_cast<const uint4*>(src + head * r.src_head + s * part_bytes);
    }
  };
#pragma unroll
  for (int i = 0; i < kHeads; ++i) load(i, i);

  char* dst = r.dst + first * r.dst_head + vec * 16;
  if (!kPaged || is_q) {
    dst += token * r.dst_token;
  } else {
    int page, row;
    if (!place(a, token, vec == 0, &page, &row)) return;
    dst += page * (is_k ? a.page_k : a.page_v) + row * r.dst_token;
  }

  float cs[kPairs], sn[kPairs];
  if (!kPaged || is_q || is_k) sines<sizeof(T) == 4>(a, token, vec, cs, sn);

  for (int done = 0; done < count; done += kHeads) {
#pragma unroll
    for (int i = 0; i < kHeads; ++i) {
      if (done + i >= count) continue;
      uint4 out[kParts];
#pragma unroll
      for (int s = 0; s < kParts; ++s) out[s] = raw[i][s];
      if (!kPaged || is_q || is_k) {
        float x[kVec], y2[kVec];
        Vec<T>::unpack(out[0], x);
        if (kHalves) Vec<T>::unpack(out[kParts - 1], y2);
        turn<kHalves>(x, y2, cs, sn);
        out[0] = Vec<T>::pack(x);
        if (kHalves) out[kParts - 1] = Vec<T>::pack(y2);
      }
      load(i, done + kHeads + i);  // before the store, which the compiler must take for one to the same memory
#pragma unroll
      for (int s = 0; s < kParts; ++s) *reinterpret_cast<uint4*>(dst + (done + i) * r.dst_head + s * part_bytes) = out[s];
    }
  }
}

template <typename T, bool kHalves, bool kPaged>
void launch(Args a, cudaStream_t stream, int sms) {
  const int per_row = a.pairs / (kHalves ? Vec<T>::n : Vec<T>::n / 2);
  const int64_t rows = static_cast<int64_t>(a.tokens) * per_row;
  const int widest = spread_heads(a, rows, sms);
  const int64_t blocks = (rows + kThreads - 1) / kThreads;
  const int groups = a.q.groups + a.k.groups + a.v.groups;
  RC_CHECK(blocks < (1ll << 31) && groups < 65536, "too many tokens or heads for one launch");
  const dim3 grid(static_cast<unsigned>(blocks), groups);
  // loads in flight: 4 heads at a time (halves hold two vectors of each)
  if (widest == 1) paged::launch(rotate_kernel<T, kHalves, kPaged, 1>, grid, kThreads, 0, 0, stream, a);
  else if (widest == 2) paged::launch(rotate_kernel<T, kHalves, kPaged, 2>, grid, kThreads, 0, 0, stream, a);
  else paged::launch(rotate_kernel<T, kHalves, kPaged, kHalves ? 4 : 8>, grid, kThreads, 0, 0, stream, a);
}

template <bool kPaged>
void dispatch(const Args& a, at::ScalarType type, bool halves, cudaStream_t stream, int sms) {
  if (type == at::kBFloat16) {
    halves ? launch<__nv_bfloat16, true, kPaged>(a, stream, sms) : launch<__nv_bfloat16, false, kPaged>(a, stream, sms);
  } else if (type == at::kHalf) {
    halves ? launch<__half, true, kPaged>(a, stream, sms) : launch<__half, false, kPaged>(a, stream, sms);
  } else if constexpr (!kPaged) {
    halves ? launch<float, true, false>(a, stream, sms) : launch<float, false, false>(a, stream, sms);
  }
}

}  // namespace rotary

bool rotary_rows_ok(const at::Tensor& t) { return t.numel() == 0 || rotary::vector_rows(t); }

// out = rotation of x by sign * phi, for up to two tensors [tokens, heads, head_dim] in one launch (either may be
// undefined, not both).
void rotate_launch(const at::Tensor& q, at::Tensor& q_out, const at::Tensor& k, at::Tensor& k_out,
                   const at::Tensor& positions, const RopePlan& plan, double sign) {
  const at::Tensor& any = q.defined() ? q : k;
  RC_CHECK(any.defined() && any.is_cuda() && any.dim() == 3, "rotate takes CUDA tensors [tokens, heads, head_dim]");
  rotary::Args a{};
  const int64_t head_dim = any.size(2);
  RC_CHECK(any.size(0) < (1ll << 31), "too many tokens for one launch");
  const int tokens = static_cast<int>(any.size(0));
  const at::ScalarType type = any.scalar_type();
  RC_CHECK(type == at::kBFloat16 || type == at::kHalf || type == at::kFloat, "rotate takes bf16, fp16 or fp32");
  rotary::set_rotation(a, positions, plan, tokens, head_dim, any.device());
  const at::Tensor* in[2] = {&q, &k};
  at::Tensor* out[2] = {&q_out, &k_out};
  rotary::Rows* rows[2] = {&a.q, &a.k};
  for (int i = 0; i < 2; ++i) {
    if (!in[i]->defined()) continue;
    const int64_t size = in[i]->element_size();
    RC_CHECK(in[i]->scalar_type() == type && in[i]->device() == any.device() && in[i]->dim() == 3 &&
                 in[i]->size(0) == tokens && in[i]->size(2) == head_dim,
             "q and k must agree on type, device, tokens and head_dim");
    RC_CHECK(out[i]->scalar_type() == type && out[i]->device() == any.device() && out[i]->sizes() == in[i]->sizes(),
             "an output must match its input");
    RC_CHECK(rotary_rows_ok(*in[i]) && rotary_rows_ok(*out[i]),
             "rows must have unit inner stride and 16-byte aligned strides and base");
    *rows[i] = {static_cast<const char*>(in[i]->data_ptr()), static_cast<char*>(out[i]->data_ptr()),
                in[i]->stride(0) * size, in[i]->stride(1) * size, out[i]->stride(0) * size, out[i]->stride(1) * size,
                static_cast<int>(in[i]->size(1))};
  }
  a.sign = static_cast<float>(sign);
  if (tokens == 0 || a.q.heads + a.k.heads == 0) return;
  c10::cuda::CUDAGuard guard(any.device());
  rotary::dispatch<false>(a, type, plan.halves, c10::cuda::getCurrentCUDAStream(any.get_device()).stream(),
                          sm_count(any.get_device()));
}

// Rotation of q (returned; into `out` if it is given); k rotated and v as it is into their pages: token i of sequence s
// goes to position kv_lens[s] - (cu_q[s + 1] - cu_q[s]) + i of the sequence.
at::Tensor paged_append(const at::Tensor& q, const at::Tensor& k, const at::Tensor& v, const at::Tensor& positions,
                        const RopePlan& plan, at::Tensor& k_pages, at::Tensor& v_pages, const at::Tensor& table,
                        const at::Tensor& kv_lens, const at::Tensor& cu_q, const c10::optional<at::Tensor>& out,
                        const c10::optional<at::Tensor>& status) {
  check_cuda_tensor(q, "q");
  refuse_gradients({&q, &k, &v, &positions, &k_pages, &v_pages}, "append");
  if (out.has_value()) refuse_gradients({&*out}, "append");
  refuse_tangents({&q, &k, &v, &positions, &k_pages, &v_pages}, "append");
  const at::ScalarType type = q.scalar_type();
  RC_CHECK(type == at::kBFloat16 || type == at::kHalf, "a paged cache holds bf16 or fp16");
  c10::cuda::CUDAGuard guard(q.device());
  at::Tensor q_out = out.has_value() ? *out : at::empty(q.sizes(), q.options());
  RC_CHECK(q.dim() == 3 && k.dim() == 3 && v.sizes() == k.sizes() && k.size(0) == q.size(0) && k.size(2) == q.size(2) &&
               q_out.sizes() == q.sizes(),
           "q is [tokens, heads, head_dim], k and v [tokens, kv_heads, head_dim]");
  RC_CHECK(q.size(0) < (1ll << 31), "too many tokens for one launch");
  const at::Tensor* all[6] = {&q, &k, &v, &q_out, &k_pages, &v_pages};
  for (const at::Tensor* t : all)
    RC_CHECK(t->scalar_type() == type && t->device() == q.device(), "q, k, v and the pages must agree on type and device");
  for (int i = 0; i < 4; ++i)
    RC_CHECK(rotary_rows_ok(*all[i]), "rows must have unit inner stride and 16-byte aligned strides and base");
  // what threads of one launch write must not lie on top of itself (q may be turned in place)
  for (const at::Tensor* t : {static_cast<const at::Tensor*>(&q_out), static_cast<const at::Tensor*>(&k_pages), static_cast<const at::Tensor*>(&v_pages)})
    at::assert_no_internal_overlap(*t);
  RC_CHECK(k_pages.data_ptr() != v_pages.data_ptr(), "k_pages and v_pages must be different pages");
  at::assert_no_partial_overlap(q_out, q);
  const paged::Table t = paged::check_table(table, kv_lens, cu_q, q.device());
  const paged::Pages kp = paged::check_pages(k_pages, k.size(1), k.size(2), "k_pages");
  const paged::Pages vp = paged::check_pages(v_pages, k.size(1), k.size(2), "v_pages");
  RC_CHECK(kp.count == vp.count && kp.size == vp.size, "k_pages and v_pages must have the same pages");
  rotary::Args a{};
  const int tokens = static_cast<int>(q.size(0));
  rotary::set_rotation(a, positions, plan, tokens, q.size(2), q.device());
  a.sign = 1.0f;
  a.q = {static_cast<const char*>(q.data_ptr()), static_cast<char*>(q_out.data_ptr()), q.stride(0) * 2, q.stride(1) * 2,
         q_out.stride(0) * 2, q_out.stride(1) * 2, static_cast<int>(q.size(1))};
  a.k = {static_cast<const char*>(k.data_ptr()), static_cast<char*>(k_pages.data_ptr()), k.stride(0) * 2, k.stride(1) * 2,
         kp.token_stride * 2, kp.head_stride * 2, static_cast<int>(k.size(1))};
  a.v = {static_cast<const char*>(v.data_ptr()), static_cast<char*>(v_pages.data_ptr()), v.stride(0) * 2, v.stride(1) * 2,
         vp.token_stride * 2, vp.head_stride * 2, static_cast<int>(v.size(1))};
  a.table = t.table;
  a.kv_lens = t.kv_lens;
  a.cu_q = t.cu_q;
  a.seqs = t.seqs;
  a.table_width = t.width;
  a.table_row = t.row;
  a.page = kp.size;
  a.pages = kp.count;
  a.page_k = kp.page_stride * 2;
  a.page_v = vp.page_stride * 2;
  a.status = status_ptr(status);
  if (t.seqs == 0) a.k.heads = a.v.heads = 0;  // q alone: k and v belong to no sequence
  if (tokens > 0 && a.q.heads + a.k.heads > 0)
    rotary::dispatch<true>(a, type, plan.halves, c10::cuda::getCurrentCUDAStream(q.get_device()).stream(), sm_count(q.get_device()));
  if (out.has_value()) written(*out);
  if (t.seqs > 0) {
    written(k_pages);
    written(v_pages);
  }
  return q_out;
}

}  // namespace rc
