// Byte format of a KV cache held in 4 bits, head_dim 128 (the same format for any head_dim: ops/kv4.py).
//
// 16 tokens of one page and KV head are a unit of 1152 contiguous bytes: 16 rows of codes (64 bytes: channel 2i in the
// low nibble of byte i), then 16 rows of parameters (bf16 s0, c0, s1, c1). Eight channels are one 32-bit word; even
// words form group 0, odd words group 1; a channel stands for c_g + s_g * (code - 8).
//
// Values from codes: (word >> 4j) & 0x000f000f | 0x43004300 is the bf16 pair {128 + n_j, 128 + n_(j+4)} (bf16 holds the
// integers up to 256 exactly), one LOP3 per two channels and no table. Minus 136 it is n - 8, exact.
#pragma once

#include <cuda_bf16.h>
#include <stdint.h>

namespace xv {
namespace kv4 {

constexpr int kD = 128;
constexpr int kUnit = 16;                                  // tokens
constexpr int kCodeRow = kD / 2;                           // bytes of codes of one token
constexpr int kParRow = 8;                                 // bytes of parameters of one token
constexpr int kRow = kCodeRow + kParRow;
constexpr int kParBase = kUnit * kCodeRow;                 // offset of a unit's parameters
constexpr int kUnitBytes = kUnit * kRow;                   // 1152
constexpr uint32_t kMagic = 0x43004300u;                   // bf16 {128, 128}

// Byte offset of the unit that holds token `r` of page `blk` for KV head `h`.
__device__ __forceinline__ size_t unit_offset(int blk, int h, int hkv, int block_size, int r) {
  return ((static_cast<size_t>(blk) * hkv + h) * (block_size / kUnit) + r / kUnit) * kUnitBytes;
}

// bf16 pair {128 + nibble j of the low half, 128 + the same of the high half}, shift = 4j. The and-or is spelled as the
// one LOP3 it is: from C operators the compiler makes two.
__device__ __forceinline__ uint32_t biased(uint32_t w, int shift) {
  uint32_t r;
  asm("lop3.b32 %0, %1, %2, %3, 0xEA;" : "=r"(r) : "r"(w >> shift), "r"(0x000f000fu), "r"(kMagic));
  return r;
}

// {n - 8, n - 8} from biased(): exact.
__device__ __forceinline__ uint32_t centred(uint32_t b) {
  const uint32_t bias = 0x43084308u;                       // bf16 {136, 136}
  const __nv_bfloat162 v = __hsub2(*reinterpret_cast<const __nv_bfloat162*>(&b), *reinterpret_cast<const __nv_bfloat162*>(&bias));
  return *reinterpret_cast<const uint32_t*>(&v);
}

// Scale and centre of a parameter word {s, c}.
__device__ __forceinline__ float par_s(uint32_t w) { return __uint_as_float(w << 16); }
__device__ __forceinline__ float par_c(uint32_t w) { return __uint_as_float(w & 0xffff0000u); }

}  // namespace kv4
}  // namespace xv
