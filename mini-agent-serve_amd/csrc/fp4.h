// fp4.h - the 4-bit KV cache's number format (OCP microscaling fp4) on gfx950.
//
// A head's row of head_dim elements is cut into blocks of 32. A block is 32 e2m1 codes (sign, two exponent
// bits, one mantissa bit: 0, 1/2, 1, 3/2, 2, 3, 4, 6), two a byte with the even element in the low half, and
// one power of two 2^(s - 127), s a byte (e8m0; 255 stands for NaN). The power is the smallest of at least
// 2^-127 under which the block's largest element lies below 7: the codes' largest value is 6 and their step
// there 2, so nothing is cut off by more than half a step (taking the exponent of the largest element alone would
// cut elements of up to 8 to 6).
#pragma once

#include "device.h"

namespace mas {

constexpr int kFp4Block = 32;      // elements that share a power of two
constexpr int kFp4MinPage = 16;    // slots per page, at least: a 16-position MFMA tile lies in one page

// A cache of one layer. Strides in bytes; the slots of a block's powers are adjacent and its blocks page_size
// bytes apart, so that 16 consecutive positions' powers are 16 consecutive bytes.
struct Fp4Cache {
  uint8_t* k;
  uint8_t* v;
  int64_t page_stride, entry_stride, head_stride;
  uint8_t* k_scale;
  uint8_t* v_scale;
  int64_t scale_page_stride, scale_head_stride;
  int64_t num_pages, page_size;
};

// MAS_OK for a cache that the fp4 kernels address: pages of a power of two of at least 16 slots, codes in
// 16-byte and powers in 4-byte steps.
inline int check_fp4_cache(const Fp4Cache& c) {
  if (c.num_pages < 0 || c.page_size <= 0) return MAS_ERR_INVALID_VALUE;
  if (c.page_size < kFp4MinPage || (c.page_size & (c.page_size - 1)) != 0) return MAS_ERR_UNSUPPORTED;
  if (c.num_pages > 0 && (c.k == nullptr || c.v == nullptr || c.k_scale == nullptr || c.v_scale == nullptr))
    return MAS_ERR_INVALID_VALUE;
  const auto aligned4 = [](const void* p) { return (reinterpret_cast<uintptr_t>(p) & 3u) == 0; };
  const bool ok = aligned16(c.k) && aligned16(c.v) && c.page_stride % 16 == 0 && c.entry_stride % 16 == 0 &&
                  c.head_stride % 16 == 0 && aligned4(c.k_scale) && aligned4(c.v_scale) &&
                  c.scale_page_stride % 4 == 0 && c.scale_head_stride % 4 == 0;
  return ok ? MAS_OK : MAS_ERR_MISALIGNED;
}

// The power byte of a block whose largest magnitude has these bf16 bits. bf16 and e8m0 share the exponent's
// bias; adding a quarter of the significand's unit carries into the exponent where the significand is 7/4 or
// more. A NaN or an infinity makes the block NaN.
__device__ __forceinline__ uint32_t fp4_power(uint32_t max_bits) {
  const int s = static_cast<int>((max_bits + 0x20u) >> 7) - 2;
  return max_bits >= 0x7f80u ? 255u : static_cast<uint32_t>(s > 0 ? s : 0);
}

// Eight bf16 (four words) divided by 2^(power - 127) and rounded to the nearest code, ties to the even one:
// eight codes, element i in nibble i. v_cvt_scalef32_pk_fp4_bf16 takes the exponent field of its fp32 scale
// (exact for every bf16 and power, checked on MI355X for all bf16 against powers 0, 100, 127 and 200).
__device__ __forceinline__ uint32_t fp4x8_encode(u32x4 w, uint32_t power) {
  const float scale = __uint_as_float(power << 23);
  uint32_t c = 0;
  c = __builtin_amdgcn_cvt_scalef32_pk_fp4_bf16(c, __builtin_bit_cast(bf16x2, static_cast<uint32_t>(w[0])), scale, 0);
  c = __builtin_amdgcn_cvt_scalef32_pk_fp4_bf16(c, __builtin_bit_cast(bf16x2, static_cast<uint32_t>(w[1])), scale, 1);
  c = __builtin_amdgcn_cvt_scalef32_pk_fp4_bf16(c, __builtin_bit_cast(bf16x2, static_cast<uint32_t>(w[2])), scale, 2);
  c = __builtin_amdgcn_cvt_scalef32_pk_fp4_bf16(c, __builtin_bit_cast(bf16x2, static_cast<uint32_t>(w[3])), scale, 3);
  return c;
}

// The two codes of byte kByte of `c` times 2^(exponent field of `scale` - 127), as a bf16 pair: exact (an e2m1
// value has two significant bits; subnormal bf16 results are kept), NaN for a field of 255. Sign and
// mantissa bits of `scale` do not matter, so the power byte needs no masking, only a shift to bits 23..30.
template <int kByte>
__device__ __forceinline__ uint32_t fp4x2_decode(uint32_t c, float scale) {
  return __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(c, scale, kByte));
}
__device__ __forceinline__ u32x4 fp4x8_decode(uint32_t c, float scale) {
  return u32x4{fp4x2_decode<0>(c, scale), fp4x2_decode<1>(c, scale), fp4x2_decode<2>(c, scale),
               fp4x2_decode<3>(c, scale)};
}

}  // namespace mas
