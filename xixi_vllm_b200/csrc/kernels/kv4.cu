// Writing and reading a KV cache held in 4 bits (format: common/kv4.cuh).
//
//   kv4_write_kernel - per-head RMSNorm of q and k, NeoX RoPE, q written in bf16, k and v rounded to bf16 (what a bf16
//                      cache would hold) and quantised into their slots. One warp per (token, head).
//   kv4_read_kernel  - the bf16 values of a list of slots.
//
// Quantising is a choice between 16 levels, so K is normalised and rotated in 64 bits from the fp32 row: a value next
// to a border between two levels then falls the same way wherever the row is computed (sixteen products a lane, for the
// K heads only).

#include <cuda_bf16.h>
#include <cuda_runtime.h>

#include "../common/kv4.cuh"
#include "../common/launch.cuh"
#include "../common/ptx.cuh"
#include "xv_cuda.h"

namespace {

using namespace xv;

constexpr int kIdWrite = 8, kIdRead = 9;       // kernel ids in the status word

__device__ __forceinline__ float round_bf16(float x) { return __bfloat162float(__float2bfloat16(x)); }

__device__ __forceinline__ double warp_sum_d(double v) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
  return v;
}

// Stores one row: lane l holds channels 2l, 2l+1 (lo) and 64 + 2l, 64 + 2l + 1 (hi), all four in group (l >> 2) & 1.
// ops/kv4.py fixes the arithmetic; the explicit _rn forms keep it under the library's fast-math flags.
__device__ __forceinline__ void store_row(uint8_t* unit, int r, int lane, float lo0, float lo1, float hi0, float hi1) {
  float mx = fmaxf(fmaxf(lo0, lo1), fmaxf(hi0, hi1)), mn = fminf(fminf(lo0, lo1), fminf(hi0, hi1));
  const bool fine = fabsf(lo0) <= 3.3895314e38f && fabsf(lo1) <= 3.3895314e38f && fabsf(hi0) <= 3.3895314e38f &&
                    fabsf(hi1) <= 3.3895314e38f;              // the largest bf16; false for NaN
#pragma unroll
  for (int o = 1; o <= 16; o <<= 1) {
    if (o == 4) continue;                                     // lane bit 2 is the group
    mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, o));
    mn = fminf(mn, __shfl_xor_sync(0xffffffffu, mn, o));
  }
  const uint32_t not_fine = __ballot_sync(0xffffffffu, !fine);
  const bool bad = (not_fine & ((lane & 4) ? 0xf0f0f0f0u : 0x0f0f0f0fu)) != 0;
  float s = round_bf16(__fdiv_rn(__fsub_rn(0.5f * mx, 0.5f * mn), 7.5f));
  if (s < 1.17549435e-38f) s = 0.f;
  const float c = round_bf16(__fadd_rn(__fadd_rn(0.5f * mx, 0.5f * mn), 0.5f * s));
  auto code = [&](float x) -> uint32_t {
    if (bad || s == 0.f) return 8u;
    const float n = rintf(__fdiv_rn(__fsub_rn(x, c), s)) + 8.f;
    return static_cast<uint32_t>(fminf(fmaxf(n, 0.f), 15.f));
  };
  uint8_t* codes = unit + r * kv4::kCodeRow;
  codes[lane] = static_cast<uint8_t>(code(lo0) | code(lo1) << 4);
  codes[32 + lane] = static_cast<uint8_t>(code(hi0) | code(hi1) << 4);
  if ((lane & 27) == 0) {                                     // lanes 0 and 4: one parameter word per group
    uint32_t w = 0x7fff7fffu;
    if (!bad) w = pack_bf16(s, c);
    *reinterpret_cast<uint32_t*>(unit + kv4::kParBase + r * kv4::kParRow + lane) = w;
  }
}

__global__ void __launch_bounds__(256)
kv4_write_kernel(const __nv_bfloat16* __restrict__ qkv, const float* __restrict__ partials, int splits,
                 long long split_stride, const __nv_bfloat16* __restrict__ q_w, const __nv_bfloat16* __restrict__ k_w,
                 float eps, const float* __restrict__ cos_sin, int max_pos, const int* __restrict__ positions,
                 const int* __restrict__ slots, __nv_bfloat16* __restrict__ q_out, uint8_t* __restrict__ k_cache,
                 uint8_t* __restrict__ v_cache, int tokens, int hq, int hkv, int block_size, int num_slots, int* status) {
  grid_dep_launch();
  grid_dep_wait();
  constexpr int D = kv4::kD, HALF = D / 2;
  const int heads = hq + 2 * hkv;
  const long long gw = (static_cast<long long>(blockIdx.x) * blockDim.x + threadIdx.x) >> 5;
  const int lane = threadIdx.x & 31;
  if (gw >= static_cast<long long>(tokens) * heads) return;
  const int t = static_cast<int>(gw / heads);
  const int h = static_cast<int>(gw - static_cast<long long>(t) * heads);
  int slot = -1;
  if (h >= hq) {
    slot = slots[t];
    if (slot >= num_slots) {
      if (lane == 0) report_status(status, kIdWrite, kBadIndex);
      slot = -1;
    }
    if (slot < 0) return;                                     // warp-uniform
  }
  const size_t off = static_cast<size_t>(t) * heads * D + static_cast<size_t>(h) * D;

  float lo0, lo1, hi0, hi1;
  if (partials != nullptr) {
    lo0 = lo1 = hi0 = hi1 = 0.f;
    for (int s = 0; s < splits; ++s) {
      const float2 a = *reinterpret_cast<const float2*>(partials + s * split_stride + off + lane * 2);
      const float2 b = *reinterpret_cast<const float2*>(partials + s * split_stride + off + HALF + lane * 2);
      lo0 += a.x; lo1 += a.y; hi0 += b.x; hi1 += b.y;
    }
    // same rounding point as the bf16 GEMM output would have had
    lo0 = round_bf16(lo0); lo1 = round_bf16(lo1); hi0 = round_bf16(hi0); hi1 = round_bf16(hi1);
  } else {
    const float2 a = __bfloat1622float2(*reinterpret_cast<const __nv_bfloat162*>(qkv + off + lane * 2));
    const float2 b = __bfloat1622float2(*reinterpret_cast<const __nv_bfloat162*>(qkv + off + HALF + lane * 2));
    lo0 = a.x; lo1 = a.y; hi0 = b.x; hi1 = b.y;
  }
  if (h >= hq + hkv) {
    store_row(v_cache + kv4::unit_offset(slot / block_size, h - hq - hkv, hkv, block_size, slot % block_size),
              slot % block_size % kv4::kUnit, lane, lo0, lo1, hi0, hi1);
    return;
  }
  int pos = positions[t];
  if (pos < 0 || pos >= max_pos) {
    if (lane == 0) report_status(status, kIdWrite, kBadIndex);
    pos = 0;
  }
  const float2 cs = *reinterpret_cast<const float2*>(cos_sin + static_cast<size_t>(pos) * D + lane * 2);
  const float2 sn = *reinterpret_cast<const float2*>(cos_sin + static_cast<size_t>(pos) * D + HALF + lane * 2);
  const __nv_bfloat16* w = h < hq ? q_w : k_w;
  const float2 wl = __bfloat1622float2(*reinterpret_cast<const __nv_bfloat162*>(w + lane * 2));
  const float2 wh = __bfloat1622float2(*reinterpret_cast<const __nv_bfloat162*>(w + HALF + lane * 2));
  if (h < hq) {
    const float ss = warp_sum(lo0 * lo0 + lo1 * lo1 + hi0 * hi0 + hi1 * hi1);
    const float inv = rsqrtf(ss / static_cast<float>(D) + eps);
    const float a0 = lo0 * inv * wl.x, a1 = lo1 * inv * wl.y, b0 = hi0 * inv * wh.x, b1 = hi1 * inv * wh.y;
    __nv_bfloat16* dst = q_out + static_cast<size_t>(t) * hq * D + static_cast<size_t>(h) * D;
    *reinterpret_cast<uint32_t*>(dst + lane * 2) = pack_bf16(a0 * cs.x - b0 * sn.x, a1 * cs.y - b1 * sn.y);
    *reinterpret_cast<uint32_t*>(dst + HALF + lane * 2) = pack_bf16(b0 * cs.x + a0 * sn.x, b1 * cs.y + a1 * sn.y);
    return;
  }
  const double l0 = lo0, l1 = lo1, h0 = hi0, h1 = hi1;
  const double ms = warp_sum_d(l0 * l0 + l1 * l1 + h0 * h0 + h1 * h1) * (1.0 / D) + static_cast<double>(eps);
  double inv = rsqrtf(static_cast<float>(ms));                // one Newton step doubles its 22 bits
  inv = inv + 0.5 * inv * (1.0 - ms * inv * inv);
  const double a0 = l0 * inv * wl.x, a1 = l1 * inv * wl.y, b0 = h0 * inv * wh.x, b1 = h1 * inv * wh.y;
  store_row(k_cache + kv4::unit_offset(slot / block_size, h - hq, hkv, block_size, slot % block_size),
            slot % block_size % kv4::kUnit, lane, round_bf16(static_cast<float>(a0 * cs.x - b0 * sn.x)),
            round_bf16(static_cast<float>(a1 * cs.y - b1 * sn.y)), round_bf16(static_cast<float>(b0 * cs.x + a0 * sn.x)),
            round_bf16(static_cast<float>(b1 * cs.y + a1 * sn.y)));
}

// Sixteen lanes per (token, head): lane i turns word i (8 channels) of K and of V into 16 bytes of bf16.
__global__ void __launch_bounds__(256)
kv4_read_kernel(const uint8_t* __restrict__ k_cache, const uint8_t* __restrict__ v_cache, const int* __restrict__ slots,
                __nv_bfloat16* __restrict__ k_out, __nv_bfloat16* __restrict__ v_out, long long rows, int hkv,
                int block_size, int num_slots, int* status) {
  grid_dep_launch();
  grid_dep_wait();
  const long long idx = static_cast<long long>(blockIdx.x) * blockDim.x + threadIdx.x;
  const long long row = idx >> 4;
  const int i = static_cast<int>(idx & 15);
  if (row >= rows) return;
  const int t = static_cast<int>(row / hkv), h = static_cast<int>(row - static_cast<long long>(t) * hkv);
  int slot = slots[t];
  if (slot >= num_slots) {
    if (i == 0) report_status(status, kIdRead, kBadIndex);
    slot = -1;
  }
  const size_t dst = static_cast<size_t>(row) * kv4::kD + i * 8;
  if (slot < 0) {
    *reinterpret_cast<uint4*>(k_out + dst) = make_uint4(0, 0, 0, 0);
    *reinterpret_cast<uint4*>(v_out + dst) = make_uint4(0, 0, 0, 0);
    return;
  }
  const int r = slot % block_size;
  const size_t unit = kv4::unit_offset(slot / block_size, h, hkv, block_size, r);
  const size_t co = unit + (r % kv4::kUnit) * kv4::kCodeRow + i * 4;
  const size_t po = unit + kv4::kParBase + (r % kv4::kUnit) * kv4::kParRow + (i & 1) * 4;
#pragma unroll
  for (int kv = 0; kv < 2; ++kv) {
    const uint8_t* cache = kv ? v_cache : k_cache;
    const uint32_t w = *reinterpret_cast<const uint32_t*>(cache + co), p = *reinterpret_cast<const uint32_t*>(cache + po);
    const float s = kv4::par_s(p), c = kv4::par_c(p);
    uint32_t o[4];
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const float n0 = static_cast<float>(static_cast<int>((w >> (8 * j)) & 15u) - 8);
      const float n1 = static_cast<float>(static_cast<int>((w >> (8 * j + 4)) & 15u) - 8);
      o[j] = pack_bf16(fmaf(s, n0, c), fmaf(s, n1, c));
    }
    *reinterpret_cast<uint4*>((kv ? v_out : k_out) + dst) = make_uint4(o[0], o[1], o[2], o[3]);
  }
}

inline int launch_ok() { return cudaGetLastError() == cudaSuccess ? 0 : XV_ERR_LAUNCH; }
inline bool misaligned(const void* p, uintptr_t a) { return (reinterpret_cast<uintptr_t>(p) & (a - 1)) != 0; }

int check_cache(int hkv, int d, int block_size, int num_blocks) {
  if (d != kv4::kD) return XV_ERR_UNSUPPORTED;
  if (hkv <= 0 || block_size <= 0 || block_size % kv4::kUnit || num_blocks <= 0) return XV_ERR_SHAPE;
  if (static_cast<long long>(num_blocks) * block_size > 0x7fffffffLL) return XV_ERR_SHAPE;   // slots are 32-bit
  return 0;
}

}  // namespace

extern "C" {

int xv_kv4_write(const void* qkv, const float* partials, int splits, long long split_stride, const void* q_w,
                 const void* k_w, float eps, const float* cos_sin, int max_pos, const int* positions, const int* slots,
                 void* q_out, void* k_cache, void* v_cache, int tokens, int hq, int hkv, int d, int block_size,
                 int num_blocks, int* status, cudaStream_t stream) {
  if (tokens <= 0) return 0;
  if (int rc = check_cache(hkv, d, block_size, num_blocks)) return rc;
  if (hq < 0 || max_pos <= 0 || (!qkv && !partials)) return XV_ERR_SHAPE;
  if (misaligned(qkv, 16) || misaligned(partials, 16) || misaligned(q_w, 4) || misaligned(k_w, 4) ||
      misaligned(cos_sin, 8) || misaligned(q_out, 16) || misaligned(k_cache, 16) || misaligned(v_cache, 16))
    return XV_ERR_ALIGN;
  const long long blocks = (static_cast<long long>(tokens) * (hq + 2 * hkv) + 7) / 8;
  if (blocks > 0x7fffffffLL) return XV_ERR_SHAPE;
  launch_pdl(kv4_write_kernel, dim3(static_cast<unsigned>(blocks)), dim3(256), 0, stream,
             static_cast<const __nv_bfloat16*>(qkv), partials, splits, split_stride, static_cast<const __nv_bfloat16*>(q_w),
             static_cast<const __nv_bfloat16*>(k_w), eps, cos_sin, max_pos, positions, slots,
             static_cast<__nv_bfloat16*>(q_out), static_cast<uint8_t*>(k_cache), static_cast<uint8_t*>(v_cache), tokens, hq,
             hkv, block_size, num_blocks * block_size, status);
  return launch_ok();
}

int xv_kv4_read(const void* k_cache, const void* v_cache, const int* slots, void* k_out, void* v_out, int tokens, int hkv,
                int d, int block_size, int num_blocks, int* status, cudaStream_t stream) {
  if (tokens <= 0) return 0;
  if (int rc = check_cache(hkv, d, block_size, num_blocks)) return rc;
  if (misaligned(k_cache, 16) || misaligned(v_cache, 16) || misaligned(k_out, 16) || misaligned(v_out, 16))
    return XV_ERR_ALIGN;
  const long long rows = static_cast<long long>(tokens) * hkv, blocks = (rows + 15) / 16;
  if (blocks > 0x7fffffffLL) return XV_ERR_SHAPE;
  launch_pdl(kv4_read_kernel, dim3(static_cast<unsigned>(blocks)), dim3(256), 0, stream,
             static_cast<const uint8_t*>(k_cache), static_cast<const uint8_t*>(v_cache), slots,
             static_cast<__nv_bfloat16*>(k_out), static_cast<__nv_bfloat16*>(v_out), rows, hkv, block_size,
             num_blocks * block_size, status);
  return launch_ok();
}

}  // extern "C"
