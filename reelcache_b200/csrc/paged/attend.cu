// Entry point of attention over a paged KV cache: checks, and the choice between the two kernels.
//
// Few query rows (new tokens x heads of a group) cannot fill the 128-row products of tcgen05, and reading K and V bounds
// them anyway: they take the streaming kernel of attend_short.cu (attend_packed.cu over codes). More rows take attend_chunk.cu.
#include <ATen/ATen.h>
#include <ATen/MemoryOverlap.h>
#include <c10/cuda/CUDAGuard.h>
#include <c10/cuda/CUDAStream.h>

#include <algorithm>
#include <cmath>
#include <string>
#include <utility>

#include "attend.cuh"
#include "packed.h"

namespace rc {
namespace paged {

constexpr int kShortRows = 16;
// Packed pages: slices of 16 rows side by side, which read the same codes through L2, while that is less than expanding them first
// (16 sessions over 4,096 keys, 32 / 8 heads, pages of 64: 32 rows 81 us, 48 rows 116, expanded 127). One number for all
// calls: slices cost conversions for every session and key, expansion for every page that differs; for 64 sessions over 1,024
// keys of pages of 16 48 rows take 158 and 64, expanded, 167, for one over 32,768 keys 81 and 101.
constexpr int kPackedRows = 48;

void attend_short(const Args& a, int head_dim, bool half, const at::Tensor& k_pages, const at::Tensor& v_pages,
                  int max_q_len, const at::Tensor& like, cudaStream_t stream, int device);
void attend_chunk(const Args& a, int head_dim, bool half, const at::Tensor& k_pages, const at::Tensor& v_pages,
                  int max_q_len, const at::Tensor& like, cudaStream_t stream, int device);
void attend_packed_short(const Args& a, int head_dim, bool half, const at::Tensor& k_codes, const at::Tensor& v_codes, const Packed& k,
                         const Packed& v, int max_q_len, const at::Tensor& like, cudaStream_t stream, int device);
void expand_pages(Args& a, const at::Tensor& k_codes, const at::Tensor& v_codes, const Packed& k, const Packed& v, at::Tensor& k_pages,
                  at::Tensor& v_pages, at::Tensor& workspace, const at::Tensor& like, cudaStream_t stream);
std::string short_form_name(const Args& a, int head_dim, int device);
std::string chunk_form_name(const Args& a, int head_dim, int max_q_len, int device);
std::string packed_form_name(const Args& a, int head_dim, int max_q_len, int device);

}  // namespace paged

// The form that a call of these sizes takes on `device`: "few rows, cluster N", "few rows, line", "twin N", "direct N" (N CTAs
// to a cluster), "planned"; with a table for each KV head (`tables`) also "twin 1, then M items in N"; over packed pages few rows may be
// in "S slices, ...", and more rows are "expanded, " and a form of theirs.
std::string paged_attention_form(int64_t device, int64_t tokens, int64_t heads, int64_t kv_heads, int64_t head_dim, int64_t seqs,
                                 int64_t width, int64_t page_size, int64_t max_q_len, bool causal, int64_t window, int64_t sinks, bool packed,
                                 bool tables) {
  RC_CHECK((head_dim == 64 || head_dim == 128) && tokens > 0 && kv_heads > 0 && heads % kv_heads == 0 && seqs > 0 && max_q_len > 0,
           "no such call of paged attention");
  c10::cuda::CUDAGuard guard(static_cast<c10::DeviceIndex>(device));
  paged::Args a{};
  a.tokens = static_cast<int>(tokens);
  a.heads = static_cast<int>(heads);
  a.kv_heads = static_cast<int>(kv_heads);
  a.group = a.heads / a.kv_heads;
  a.seqs = static_cast<int>(seqs);
  a.width = static_cast<int>(width);
  a.tiling.page = static_cast<int>(page_size);
  a.causal = causal;
  a.window = static_cast<int>(window);
  a.sinks = window > 0 ? static_cast<int>(sinks) : 0;
  a.table_head = tables ? std::max(a.width, 1) : 0;
  const int most = static_cast<int>(std::min(max_q_len, tokens)), d = static_cast<int>(head_dim), at = static_cast<int>(device);
  const bool few = static_cast<int64_t>(most) * a.group <= (packed ? paged::kPackedRows : paged::kShortRows);
  if (few) return packed ? paged::packed_form_name(a, d, most, at) : paged::short_form_name(a, d, at);
  return (packed ? "expanded, " : "") + paged::chunk_form_name(a, d, most, at);
}

// out = softmax over the visible keys of scale * q k^T, times v, for the new tokens of every sequence; lse its natural
// log-sum-exp. The pages are of q's type, or e4m3 codes with scales. max_q_len bounds every sequence's new tokens (more are reported); rows of q that no sequence names are left
// alone.
std::pair<at::Tensor, c10::optional<at::Tensor>> paged_attention(
    const at::Tensor& q, const at::Tensor& k_pages, const at::Tensor& v_pages, const at::Tensor& table,
    const at::Tensor& kv_lens, const at::Tensor& cu_q, int64_t max_q_len, bool causal, int64_t window, int64_t sinks,
    c10::optional<double> scale_given, bool want_lse, const c10::optional<at::Tensor>& out_given,
    const c10::optional<at::Tensor>& status, const c10::optional<at::Tensor>& k_scales, const c10::optional<at::Tensor>& v_scales) {
  check_cuda_tensor(q, "q");
  refuse_gradients({&q, &k_pages, &v_pages}, "attention over pages");
  if (out_given.has_value()) refuse_gradients({&*out_given}, "attention over pages");
  refuse_tangents({&q, &k_pages, &v_pages}, "attention over pages");
  for (const c10::optional<at::Tensor>* scales : {&k_scales, &v_scales}) {
    if (!scales->has_value()) continue;
    refuse_gradients({&**scales}, "attention over pages");
    refuse_tangents({&**scales}, "attention over pages");
  }
  const at::ScalarType type = q.scalar_type();
  RC_CHECK(type == at::kBFloat16 || type == at::kHalf, "paged attention takes bf16 or fp16");
  RC_CHECK(q.dim() == 3 && (q.size(2) == 64 || q.size(2) == 128), "q must be [tokens, heads, head_dim] with head_dim 64 or 128");
  RC_CHECK(q.size(0) < (1ll << 31), "too many tokens for one launch");
  c10::cuda::CUDAGuard guard(q.device());
  const double scale = scale_given.has_value() ? *scale_given : 1.0 / std::sqrt(static_cast<double>(q.size(2)));
  const at::Tensor out = out_given.has_value() ? *out_given : paged::new_tensor(q.sizes(), q, type);
  RC_CHECK(out.sizes() == q.sizes() && out.scalar_type() == type && out.device() == q.device(), "out must match q");
  at::assert_no_internal_overlap(out);
  at::assert_no_partial_overlap(out, q);
  const at::Tensor* rows[2] = {&q, &out};
  for (const at::Tensor* t : rows)
    RC_CHECK(t->numel() == 0 || (t->stride(2) == 1 && t->stride(0) % 8 == 0 && t->stride(1) % 8 == 0 &&
                                 reinterpret_cast<uintptr_t>(t->data_ptr()) % 16 == 0),
             "rows must have unit inner stride and 16-byte aligned strides and base");
  const bool packed = k_scales.has_value();
  RC_CHECK(packed == v_scales.has_value(), "both or neither of k_pages and v_pages must be packed");
  RC_CHECK(k_pages.dim() == 4 && (packed || (k_pages.device() == q.device() && v_pages.device() == q.device() &&
                                            k_pages.scalar_type() == type && v_pages.scalar_type() == type)),
           "the pages must have the type and device of q");
  const int64_t kv_heads = k_pages.size(2);
  RC_CHECK(kv_heads >= 1 && q.size(1) % kv_heads == 0 && q.size(1) >= kv_heads, "heads must be a multiple of the KV heads");
  paged::Packed k8{}, v8{};
  int pages, page_size;
  if (packed) {
    k8 = paged::check_packed(k_pages, *k_scales, kv_heads, q.size(2), q.device(), "k_pages");
    v8 = paged::check_packed(v_pages, *v_scales, kv_heads, q.size(2), q.device(), "v_pages");
    RC_CHECK(k8.count == v8.count && k8.size == v8.size, "k_pages and v_pages must have the same pages");
    pages = k8.count;
    page_size = k8.size;
  } else {
    const paged::Pages kp = paged::check_pages(k_pages, kv_heads, q.size(2), "k_pages");
    const paged::Pages vp = paged::check_pages(v_pages, kv_heads, q.size(2), "v_pages");
    RC_CHECK(kp.count == vp.count && kp.size == vp.size, "k_pages and v_pages must have the same pages");
    pages = kp.count;
    page_size = kp.size;
  }
  const paged::Table t = paged::check_table(table, kv_lens, cu_q, q.device(), kv_heads);
  RC_CHECK(window >= 0 && sinks >= 0 && window < (1ll << 31) && sinks < (1ll << 31), "window and sinks must not be negative");
  RC_CHECK(scale > 0.0, "scale must be positive");
  RC_CHECK(max_q_len >= 1 && max_q_len < (1ll << 24), "max_q_len must be positive");
  paged::Args a{};
  a.q = q.data_ptr();
  a.q_token = q.stride(0);
  a.q_head = q.stride(1);
  a.out = out.data_ptr();
  a.out_token = out.stride(0);
  a.out_head = out.stride(1);
  a.out_sectors = out.stride(0) % 16 == 0 && out.stride(1) % 16 == 0 && reinterpret_cast<uintptr_t>(out.data_ptr()) % 32 == 0;
  c10::optional<at::Tensor> lse;
  if (want_lse) {
    lse = paged::new_tensor({q.size(0), q.size(1)}, q, at::kFloat);
    a.lse = lse->data_ptr<float>();
  }
  a.table = t.table;
  a.kv_lens = t.kv_lens;
  a.cu_q = t.cu_q;
  a.seqs = t.seqs;
  a.width = t.width;
  a.table_row = t.row;
  a.table_head = t.head;
  a.pages = pages;
  a.heads = static_cast<int>(q.size(1));
  a.kv_heads = static_cast<int>(kv_heads);
  a.group = a.heads / a.kv_heads;
  a.causal = causal;
  a.window = static_cast<int>(window);
  a.sinks = window > 0 ? static_cast<int>(sinks) : 0;
  a.tokens = static_cast<int>(q.size(0));
  a.max_q_len = static_cast<int>(max_q_len);
  a.scale_log2 = static_cast<float>(scale * 1.4426950408889634);
  a.tiling.page = page_size;
  a.status = status_ptr(status);
  if (a.tokens == 0 || a.seqs == 0) return {out, lse};
  const int device = q.get_device();
  cudaStream_t stream = c10::cuda::getCurrentCUDAStream(device).stream();
  const int most = static_cast<int>(std::min<int64_t>(max_q_len, a.tokens));
  const bool few = static_cast<int64_t>(most) * a.group <= (packed ? paged::kPackedRows : paged::kShortRows);
  const int d = static_cast<int>(q.size(2));
  if (packed && few) {
    paged::attend_packed_short(a, d, type == at::kHalf, k_pages, v_pages, k8, v8, most, q, stream, device);
  } else if (packed) {
    at::Tensor k16, v16, workspace;
    paged::expand_pages(a, k_pages, v_pages, k8, v8, k16, v16, workspace, q, stream);
    paged::attend_chunk(a, d, type == at::kHalf, k16, v16, most, q, stream, device);
  } else {
    (few ? paged::attend_short : paged::attend_chunk)(a, d, type == at::kHalf, k_pages, v_pages, most, q, stream, device);
  }
  if (out_given.has_value()) written(out);
  return {out, lse};
}

}  // namespace rc
