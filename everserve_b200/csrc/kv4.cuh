// The paged K/V cache held in 4 bits: its format, shared by the kernels that write, read and attend
// over it.
//
// One layer is uint8 [num_blocks, kv_heads, record]. A group is 64 channels, or the whole head, of
// one row (one token's K or V of one kv head); with mn and mx its smallest and largest value,
//   scale = bf16((mx - mn) / 15), zero = bf16(mn), code = clamp(rint((x - zero) / scale), 0, 15),
// and the value held is scale * code + zero. Codes are chosen against the rounded pair, so a value is held within
// half a scale, or, in a group that lies far from zero against its range, within what rounding the pair moves
// the group's ends by: 2^-8 (|mn| + mx - mn). A group holding a value that is not finite, or whose range passes
// fp32's largest number, reads as NaN. The attention kernels take values and queries below 2^90.
//
// The record of a (block, kv head) with block size BS, head dim D and NG = D / group:
//   K codes [BS][D / 2] | V codes [BS][D / 2] | K (scale, zero) [BS][NG][2] | V (scale, zero) [BS][NG][2]
// A row is D / 8 words of 8 channels. In a word, channel i sits at bit 4 * (i / 2) + 16 * (i % 2), so
// masking a word with 0x000F000F << 4 j leaves two neighbouring channels in the halves of a register.
// At head dim 128 word p of a row holds channels 8 * (p / 2 + 8 * (p % 2)) and up: the two words of
// an 8-byte piece belong to the two halves (the two groups of 64) of the head. At 64 words are in order.
#pragma once

#include <cuda_fp16.h>

#include <type_traits>

#include "common.cuh"
#include "ptx.cuh"

namespace es {
namespace kv4 {

template <int D, int NG, int BS>
struct Rec {
  static constexpr int kRow = D / 2;               // bytes of a row's codes
  static constexpr int kMeta = 4 * NG;             // bytes of a row's (scale, zero) pairs
  static constexpr int kV = BS * kRow;             // offset of the V codes
  static constexpr int kKMeta = 2 * BS * kRow;     // of the K pairs
  static constexpr int kVMeta = kKMeta + BS * kMeta;
  static constexpr int kBytes = kVMeta + BS * kMeta;
};

// (scale, zero) of a packed pair: bf16 scale in the low half, bf16 zero in the high half
ES_DEVICE float pair_scale(uint32_t p) { return __uint_as_float(p << 16); }
ES_DEVICE float pair_zero(uint32_t p) { return __uint_as_float(p & 0xFFFF0000u); }

// 2^x by the hardware's approximation (2^-22 relative); 0 below 2^-126
ES_DEVICE float ex2(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}

// Calls f with a cache's (head dim, groups, block size) as integral constants; refuses others.
template <typename F>
cudaError_t pick(int d, int groups, int bs, F&& f) {
  using std::integral_constant;
  auto sized = [&](auto dd, auto ng) -> cudaError_t {
    if (bs == 16) return f(dd, ng, integral_constant<int, 16>{});
    if (bs == 32) return f(dd, ng, integral_constant<int, 32>{});
    return cudaErrorInvalidValue;
  };
  if (d == 128 && groups == 2) return sized(integral_constant<int, 128>{}, integral_constant<int, 2>{});
  if (d == 128 && groups == 1) return sized(integral_constant<int, 128>{}, integral_constant<int, 1>{});
  if (d == 64 && groups == 1) return sized(integral_constant<int, 64>{}, integral_constant<int, 1>{});
  return cudaErrorInvalidValue;
}

}  // namespace kv4
}  // namespace es
