// A multi-axis rotation as the kernels take it: the pairs' turns per position on one device, how the pairs are split
// over the axes, and the pairs' layout. Made once per rotation and device, passed by handle.
#pragma once

#include <ATen/ATen.h>

#include <vector>

#include "../common/host.h"

namespace rc {

struct RopePlan {
  RopePlan(const at::Tensor& turns_, const at::Tensor& exact_, const std::vector<int64_t>& sections_, bool halves_)
      : turns(turns_), exact(exact_), sections(sections_), halves(halves_) {
    pairs = 0;
    for (int64_t n : sections) pairs += n;
    RC_CHECK(!sections.empty() && sections.size() <= 4, "rotary positions have one to four axes");
    RC_CHECK(pairs % 8 == 0 && pairs > 0 && pairs <= 128, "head_dim must be a multiple of 16, at most 256");
    RC_CHECK(turns.is_cuda() && turns.scalar_type() == at::kFloat && turns.is_contiguous() && turns.numel() == 2 * pairs,
             "the rotation's table must be a contiguous CUDA float32 [2, head_dim / 2]");
    RC_CHECK(exact.device() == turns.device() && exact.scalar_type() == at::kDouble && exact.is_contiguous() && exact.numel() == pairs,
             "the rotation's exact table must be a contiguous float64 [head_dim / 2] on the table's device");
  }
  at::Tensor turns;  // turns of a pair per position, [2, pairs]: high and low part
  at::Tensor exact;  // [pairs]: the same in FP64, for positions beyond 2^24
  std::vector<int64_t> sections;
  bool halves;
  int64_t pairs;
};

}  // namespace rc
