// Pages in 8 bits: a row (one token's channels of one KV head) is head_dim e4m3 codes and one e8m0 scale, x = code * 2^k.
//
// k is the smallest integer with max|x| <= 448 * 2^k, clamped so that every code * 2^k is exactly a number of the 16-bit type
// that the row came in: reading back rounds nothing, and attention over packed pages is attention over those numbers. (e4m3
// keeps four significant bits wherever the scale lies, so scales finer than powers of two would not be nearer.) A row with a
// value that is not finite has the scale NaN and reads as NaN.
//
// Codes [pages, page_size, kv_heads, head_dim]: as pages in 16 bits. Scales [kv_heads, pages, page_size]: those of a head's
// consecutive tokens lie side by side, and cutting pages into smaller ones is a view of them.
#pragma once

#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include <type_traits>

#include "paged.h"

namespace rc {
namespace paged {

struct Packed {  // strides in bytes
  int count, size;
  int64_t page_stride, token_stride, head_stride;
  const uint8_t* scales;
  int64_t scale_page, scale_head;
};

inline Packed check_packed(const at::Tensor& codes, const at::Tensor& scales, int64_t heads, int64_t head_dim, const at::Device& device,
                           const char* name) {
  const std::string who(name);
  RC_CHECK(codes.scalar_type() == at::kFloat8_e4m3fn && scales.scalar_type() == at::ScalarType::Float8_e8m0fnu,
           who + ": packed pages are float8_e4m3fn codes and float8_e8m0fnu scales");
  RC_CHECK(codes.device() == device && scales.device() == device, who + " must be on the device of the rows");
  RC_CHECK(codes.dim() == 4 && codes.size(2) == heads && codes.size(3) == head_dim && codes.stride(3) == 1,
           who + ": codes must be [pages, page_size, kv_heads, head_dim] with unit inner stride");
  RC_CHECK(codes.size(0) >= 1 && codes.size(0) < (1ll << 31) && codes.size(1) >= 8 && codes.size(1) % 8 == 0 && codes.size(1) <= 65536,
           who + ": the page size must be a multiple of 8 tokens, at most 65536");
  RC_CHECK(scales.dim() == 3 && scales.size(0) == heads && scales.size(1) == codes.size(0) && scales.size(2) == codes.size(1) &&
               scales.stride(2) == 1,
           who + ": scales must be [kv_heads, pages, page_size] with unit inner stride");
  // (a dimension of one has any stride: nothing is at its other places)
  const auto stride = [](const at::Tensor& t, int64_t d, int64_t own) { return t.size(d) == 1 ? own : t.stride(d); };
  const Packed p{static_cast<int>(codes.size(0)), static_cast<int>(codes.size(1)), stride(codes, 0, 16), stride(codes, 1, 16),
                 stride(codes, 2, 16), static_cast<const uint8_t*>(scales.data_ptr()), stride(scales, 1, 8), stride(scales, 0, 8)};
  RC_CHECK(p.page_stride >= 0 && p.page_stride % 16 == 0 && p.token_stride >= 0 && p.token_stride % 16 == 0 && p.head_stride >= 0 &&
               p.head_stride % 16 == 0 && reinterpret_cast<uintptr_t>(codes.data_ptr()) % 16 == 0,
           who + ": codes must have 16-byte aligned strides and base");
  RC_CHECK(p.scale_page >= 0 && p.scale_page % 8 == 0 && p.scale_head >= 0 && p.scale_head % 8 == 0 &&
               reinterpret_cast<uintptr_t>(p.scales) % 8 == 0,
           who + ": scales must have 8-byte aligned strides and base");
  return p;
}

constexpr int kNanScale = 255;

#ifdef __CUDACC__
// 2^k of a scale byte (k + 127; 255: NaN).
__device__ __forceinline__ float scale_value(int byte) {
  return __uint_as_float(byte == kNanScale ? 0x7fffffffu : byte == 0 ? 0x00400000u : static_cast<uint32_t>(byte) << 23);
}

// Two e4m3 codes (the lower 16 bits) as fp16, exactly; a code of NaN is NaN.
__device__ __forceinline__ uint32_t codes_to_half2(uint32_t codes) {
  uint32_t out;
  asm("{\n\t.reg .b16 c;\n\tcvt.u16.u32 c, %1;\n\tcvt.rn.f16x2.e4m3x2 %0, c;\n\t}" : "=r"(out) : "r"(codes));
  return out;
}
__device__ __forceinline__ uint32_t upper_codes_to_half2(uint32_t codes) {
  uint32_t out;
  asm("{\n\t.reg .b16 l, h;\n\tmov.b32 {l, h}, %1;\n\tcvt.rn.f16x2.e4m3x2 %0, h;\n\t}" : "=r"(out) : "r"(codes));
  return out;
}

// Two numbers as e4m3 codes, to the nearest, ties to even; `lo` in the lower byte.
__device__ __forceinline__ uint32_t codes_of(float lo, float hi) {
  uint32_t out;
  asm("{\n\t.reg .b16 c;\n\tcvt.rn.satfinite.e4m3x2.f32 c, %2, %1;\n\tcvt.u32.u16 %0, c;\n\t}" : "=r"(out) : "f"(lo), "f"(hi));
  return out;
}

// Sixteen codes times a scale as 16-bit numbers, exactly, to 32 aligned bytes (a whole sector in one store).
template <typename T>
__device__ __forceinline__ void store_values(void* dst, const uint4& codes, float scale) {
  const uint32_t w[4] = {codes.x, codes.y, codes.z, codes.w};
  uint32_t out[8];
#pragma unroll
  for (int i = 0; i < 4; ++i) {
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      const uint32_t two = h ? upper_codes_to_half2(w[i]) : codes_to_half2(w[i]);
      const float2 f = __half22float2(*reinterpret_cast<const __half2*>(&two));
      if (std::is_same<T, __half>::value) {
        const __half2 v = __floats2half2_rn(f.x * scale, f.y * scale);
        out[2 * i + h] = *reinterpret_cast<const uint32_t*>(&v);
      } else {
        const __nv_bfloat162 v = __floats2bfloat162_rn(f.x * scale, f.y * scale);
        out[2 * i + h] = *reinterpret_cast<const uint32_t*>(&v);
      }
    }
  }
  asm volatile("st.global.v8.b32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8};" ::"l"(dst), "r"(out[0]), "r"(out[1]), "r"(out[2]), "r"(out[3]),
               "r"(out[4]), "r"(out[5]), "r"(out[6]), "r"(out[7])
               : "memory");
}
#endif

}  // namespace paged
}  // namespace rc
