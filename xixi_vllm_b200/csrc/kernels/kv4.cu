// Writing and reading a KV cache held in 4 bits (format: common/kv4.cuh).
//
//   kv4_write_kernel - per-head RMSNorm of q and k, NeoX RoPE, q written in bf16, k and v rounded to bf16 (what a bf16
//                      cache would hold) and quantised into their slots. Half a warp per head, two heads of one kind at
//                      a time; a lane holds four channels and their four rotary partners. A warp takes up to eight such
//                      pairs, all of them on their way through shared memory at once (cp.async).
//   kv4_read_kernel  - the bf16 values of a list of slots. A warp per token.
//
// Both should be bound by memory: the writer moves (hq + 2 hkv) 256 + hq 256 + hkv 144 bytes a token, the reader
// hkv 2 (72 + 256). The writer is as much bound by its instructions (3600 a token of 32 + 2 x 8 heads, 66% of the issue
// slots): 8192 tokens 42 us (4.2 TB/s; with one pair sent for ahead in registers 48.5), 997 of 40 + 2 x 8 7.1 us; from four
// split-K planes 32 tokens 2.9 us. The reader: 32768 tokens of 8 heads 30.2 us in a stream (5.7 TB/s) and 34.8 with L2
// flushed; 26.2 in a graph, where the 38 MB that it reads stay in L2.
//
// Quantising is a choice between 16 levels, so K is normalised and rotated in 64 bits from the fp32 row: a value next
// to a border between two levels then falls the same way wherever the row is computed (five double operations a channel and
// their conversions, for the K heads only).

#include <cuda_bf16.h>
#include <cuda_runtime.h>

#include <algorithm>
#include <cfloat>
#include <type_traits>

#include "../common/kv4.cuh"
#include "../common/launch.cuh"
#include "../common/ptx.cuh"
#include "xv_cuda.h"

namespace {

using namespace xv;

constexpr int kIdWrite = 8, kIdRead = 9;       // kernel ids in the status word

__device__ __forceinline__ float round_bf16(float x) { return __bfloat162float(__float2bfloat16(x)); }

__device__ __forceinline__ float lo_f(uint32_t w) { return __uint_as_float(w << 16); }
__device__ __forceinline__ float hi_f(uint32_t w) { return __uint_as_float(w & 0xffff0000u); }
// Conversions and products that keep subnormal numbers, which the library's fast-math flags take for 0.
__device__ __forceinline__ double widen(float x) {
  double d;
  asm("cvt.f64.f32 %0, %1;" : "=d"(d) : "f"(x));
  return d;
}
__device__ __forceinline__ float narrow(double x) {
  float f;
  asm("cvt.rn.f32.f64 %0, %1;" : "=f"(f) : "d"(x));
  return f;
}
__device__ __forceinline__ float mul_whole(float a, float b) {
  float d;
  asm("mul.rn.f32 %0, %1, %2;" : "=f"(d) : "f"(a), "f"(b));
  return d;
}
__device__ __forceinline__ float max_whole(float a, float b) {
  float d;
  asm("max.f32 %0, %1, %2;" : "=f"(d) : "f"(a), "f"(b));
  return d;
}
__device__ __forceinline__ float min_whole(float a, float b) {
  float d;
  asm("min.f32 %0, %1, %2;" : "=f"(d) : "f"(a), "f"(b));
  return d;
}
// Sum over the 16 lanes of half a warp.
template <typename T>
__device__ __forceinline__ T half_sum(T v) {
#pragma unroll
  for (int o = 1; o <= 8; o <<= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
  return v;
}

// a / b rounded correctly, from the correctly rounded 1 / b: one step of the remainder on the product (P. Markstein,
// IBM J. Res. Dev. 34, 1990). The remainder must not underflow: a is 2^-102 at least.
__device__ __forceinline__ float quotient(float a, float b, float r_b) {
  const float q = __fmul_rn(a, r_b);
  return __fmaf_rn(__fmaf_rn(-q, b, a), r_b, q);
}

// Half a warp holds a head's row: lane c (0..15) channels 4c .. 4c + 3 in x[0..3] and 64 + 4c .. in x[4..7], so that rotary
// partners meet in a lane and all eight channels are of group (c >> 1) & 1.
//
// Stores one row of bf16 values. ops/kv4.py fixes the arithmetic; the explicit _rn forms keep it under the library's
// fast-math flags. A code is the quotient (x - centre) / step rounded to even, and ties are common (both are bf16), so
// the quotient has to be the correctly rounded one.
__device__ __forceinline__ void store_row(uint8_t* unit, int r, int c, unsigned half_mask, float (&x)[8], bool there) {
  float mx = max_whole(max_whole(max_whole(x[0], x[1]), max_whole(x[2], x[3])), max_whole(max_whole(x[4], x[5]), max_whole(x[6], x[7])));
  float mn = min_whole(min_whole(min_whole(x[0], x[1]), min_whole(x[2], x[3])), min_whole(min_whole(x[4], x[5]), min_whole(x[6], x[7])));
  float odd = 0.f;                                            // NaN if any value is NaN or infinite
#pragma unroll
  for (int i = 0; i < 8; ++i) odd = __fmaf_rn(x[i], 0.f, odd);
#pragma unroll
  for (int o = 1; o <= 8; o <<= 1) {
    if (o == 2) continue;                                     // lane bit 1 is the group
    mx = max_whole(mx, __shfl_xor_sync(0xffffffffu, mx, o));
    mn = min_whole(mn, __shfl_xor_sync(0xffffffffu, mn, o));
  }
  const uint32_t not_fine = __ballot_sync(0xffffffffu, !(odd == 0.f));
  const bool bad = (not_fine & half_mask & ((c & 2) ? 0xccccccccu : 0x33333333u)) != 0;
  // Groups below 2^-64 are taken at 2^64 of their size, where nothing underflows; step and centre come back rounded as they
  // would have been (a centre may be subnormal).
  const bool small = fmaxf(fabsf(mx), fabsf(mn)) < 0x1p-64f;
  const float up = small ? 0x1p64f : 1.f, down = small ? 0x1p-64f : 1.f;
  if (__any_sync(0xffffffffu, small)) {
    mx = mul_whole(mx, up);
    mn = mul_whole(mn, up);
#pragma unroll
    for (int i = 0; i < 8; ++i) x[i] = mul_whole(x[i], up);
  }
  float s = round_bf16(mul_whole(quotient(__fsub_rn(0.5f * mx, 0.5f * mn), 7.5f, 1.f / 7.5f), down));
  if (s < 1.17549435e-38f) s = 0.f;
  const float step = s * up;
  const float cen = round_bf16(mul_whole(__fadd_rn(__fadd_rn(0.5f * mx, 0.5f * mn), 0.5f * step), down)), mid = mul_whole(cen, up);
  // 1 / s is rounded correctly too: the step leaves an error of 2^-42, and no reciprocal of an 8-bit s is within 2^-33 of a tie.
  const float r0 = __fdividef(1.f, step);
  const float r_s = s > 0.f ? __fmaf_rn(__fmaf_rn(-step, r0, 1.f), r0, r0) : 0.f;
  // 1.5 2^23 + 8: adding it rounds to an integer, even on ties, and leaves code = integer + 8 in the low bits.
  constexpr float kRound = 12582920.f;
  constexpr uint32_t kBits = 0x4B400000u;                     // of 1.5 2^23
  uint32_t code[2] = {0u, 0u};
#pragma unroll
  for (int i = 7; i >= 0; --i) {
    const float t = quotient(__fsub_rn(x[i], mid), step, r_s);
    const float m = __fadd_rn(fminf(fmaxf(t, -8.f), 7.f), kRound);
    code[i >> 2] = code[i >> 2] * 16u + __float_as_uint(m);   // the constant part of four of them comes off at the end
  }
  code[0] -= kBits * 0x1111u;
  code[1] -= kBits * 0x1111u;
  if (bad || s == 0.f) code[0] = code[1] = 0x8888u;
  if (there) {
    uint8_t* row = unit + r * kv4::kCodeRow + c * 2;
    *reinterpret_cast<uint16_t*>(row) = static_cast<uint16_t>(code[0]);
    *reinterpret_cast<uint16_t*>(row + 32) = static_cast<uint16_t>(code[1]);
    if ((c & 13) == 0)                                        // lanes 0 and 2: one parameter word per group
      *reinterpret_cast<uint32_t*>(unit + kv4::kParBase + r * kv4::kParRow + c * 2) = bad ? 0x7fff7fffu : pack_bf16(s, cen);
  }
}

// Warps of a block of the writer, at 64 registers, for 32 warps an SM. A block holds its place until its last warp ends:
// 8192 rows (32 + 2 x 8 heads), written and read back, took 62.7 us with eight warps to a block, 59.6 with two and 57.5
// with one; 28 warps an SM 59.6, 24 63.4, 40 (which spill) 76.
constexpr int kWriteWarps = 1;
constexpr int kMaxPairs = 8;                  // of heads that a warp takes

// What a launch writes and where.
struct WriteParams {
  const __nv_bfloat16* qkv;
  const float* planes;
  const __nv_bfloat16* q_w;
  const __nv_bfloat16* k_w;
  const float* cos_sin;
  const int* positions;
  const int* slots;
  __nv_bfloat16* q_out;
  uint8_t* k_cache;
  uint8_t* v_cache;
  int* status;
  long long split_stride;
  double eps;
  int splits, max_pos, tokens, hq, hkv, block_size, num_slots;
  int per_warp, kv_per_warp;         // pairs of heads a warp takes: of Q, of K and V
  int q_tasks, tasks;                // warps per token: for Q, and in all
};

template <bool PLANES>
__global__ void __launch_bounds__(kWriteWarps * 32, 32 / kWriteWarps) kv4_write_kernel(const WriteParams p) {
  grid_dep_launch();
  grid_dep_wait();
  constexpr int D = kv4::kD, HALF = D / 2;
  const int warp = blockIdx.x * kWriteWarps + (threadIdx.x >> 5);
  // K's and V's warps first: they take longest.
  const int kv_tasks = p.tasks - p.q_tasks, kv_warps = p.tokens * kv_tasks;
  const bool is_q = warp >= kv_warps;
  const int of = is_q ? p.q_tasks : kv_tasks, at_kind = is_q ? warp - kv_warps : warp;
  const int t = at_kind / of, task = at_kind - t * of;
  if (t >= p.tokens) return;
  const int lane = threadIdx.x & 31, c = lane & 15, half = lane >> 4;
  const size_t row0 = static_cast<size_t>(t) * (p.hq + 2 * p.hkv) * D;
  // bf16 rows come through shared memory, all of a warp's pairs in flight at once: slot i holds its pair i, a head per half.
  __shared__ uint4 rows[kWriteWarps][kMaxPairs][32];
  uint4(&mine)[kMaxPairs][32] = rows[threadIdx.x >> 5];
  auto send = [&](int i, int h) {
    if constexpr (!PLANES) cp_async16(&mine[i][lane], p.qkv + row0 + static_cast<size_t>(h) * D + 8 * c);
  };

  auto arrive = [&]() {
    if constexpr (!PLANES) {
      cp_async_commit();
      cp_async_wait<0>();
      __syncwarp();
    }
  };

  // x[0..3] and x[4..7] of head h, the i-th pair of the warp
  auto load = [&](int i, int h, uint2& a, uint2& b) {
    if constexpr (PLANES) {
      const size_t off = row0 + static_cast<size_t>(h) * D + 4 * c;
      float4 u = make_float4(0.f, 0.f, 0.f, 0.f), v = u;
      for (int s = 0; s < p.splits; ++s) {
        const float4 e = *reinterpret_cast<const float4*>(p.planes + s * p.split_stride + off);
        const float4 f = *reinterpret_cast<const float4*>(p.planes + s * p.split_stride + off + HALF);
        u.x += e.x; u.y += e.y; u.z += e.z; u.w += e.w;
        v.x += f.x; v.y += f.y; v.z += f.z; v.w += f.w;
      }
      a = make_uint2(pack_bf16(u.x, u.y), pack_bf16(u.z, u.w));      // as the bf16 GEMM output would have been
      b = make_uint2(pack_bf16(v.x, v.y), pack_bf16(v.z, v.w));
    } else {
      const uint2* at = reinterpret_cast<const uint2*>(&mine[i][16 * half]);
      a = at[c];
      b = at[16 + c];
    }
  };
  auto unpack = [](const uint2& a, const uint2& b, float (&x)[8]) {
    x[0] = lo_f(a.x); x[1] = hi_f(a.x); x[2] = lo_f(a.y); x[3] = hi_f(a.y);
    x[4] = lo_f(b.x); x[5] = hi_f(b.x); x[6] = lo_f(b.y); x[7] = hi_f(b.y);
  };
  // The lane's four rotary pairs: cos, sin, and the two norm weights.
  float cs[4], sn[4], w[8];
  auto rotary = [&](const __nv_bfloat16* nw) {
    int pos = p.positions[t];
    if (pos < 0 || pos >= p.max_pos) {
      if (lane == 0) report_status(p.status, kIdWrite, kBadIndex);
      pos = 0;
    }
    const float* at = p.cos_sin + static_cast<size_t>(pos) * D + 4 * c;
    const float4 a = __ldg(reinterpret_cast<const float4*>(at)), b = __ldg(reinterpret_cast<const float4*>(at + HALF));
    cs[0] = a.x; cs[1] = a.y; cs[2] = a.z; cs[3] = a.w;
    sn[0] = b.x; sn[1] = b.y; sn[2] = b.z; sn[3] = b.w;
    unpack(__ldg(reinterpret_cast<const uint2*>(nw + 4 * c)), __ldg(reinterpret_cast<const uint2*>(nw + HALF + 4 * c)), w);
  };

  if (is_q) {
    // ---- Q: heads 2 i + half; a missing second head repeats the first and stores nothing ----
    const int first = task * p.per_warp, last = min(first + p.per_warp, (p.hq + 1) / 2);
    auto head_of = [&](int pair) { return min(2 * pair + half, p.hq - 1); };
#pragma unroll 2
    for (int i = first; i < last; ++i) send(i - first, head_of(i));
    rotary(p.q_w);
    uint64_t p1[2], p2[2], p3[2], p4[2];                      // w1 cos, -w2 sin, w2 cos, w1 sin, two channels each
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      p1[i] = pack_f32x2(w[2 * i] * cs[2 * i], w[2 * i + 1] * cs[2 * i + 1]);
      p2[i] = pack_f32x2(-w[4 + 2 * i] * sn[2 * i], -w[5 + 2 * i] * sn[2 * i + 1]);
      p3[i] = pack_f32x2(w[4 + 2 * i] * cs[2 * i], w[5 + 2 * i] * cs[2 * i + 1]);
      p4[i] = pack_f32x2(w[2 * i] * sn[2 * i], w[2 * i + 1] * sn[2 * i + 1]);
    }
    arrive();
    for (int i = first; i < last; ++i) {
      const int h = 2 * i + half;
      uint2 a, b;
      load(i - first, head_of(i), a, b);
      float x[8];
      unpack(a, b, x);
      uint64_t x1[2], x2[2], ss2 = 0ull;
#pragma unroll
      for (int k = 0; k < 2; ++k) {
        x1[k] = pack_f32x2(x[2 * k], x[2 * k + 1]);
        x2[k] = pack_f32x2(x[4 + 2 * k], x[5 + 2 * k]);
        ss2 = fma_f32x2(x2[k], x2[k], fma_f32x2(x1[k], x1[k], ss2));
      }
      float sa, sb;
      unpack_f32x2(ss2, sa, sb);
      const float inv = rsqrtf(half_sum(sa + sb) / static_cast<float>(D) + static_cast<float>(p.eps));
      const uint64_t inv2 = pack_f32x2(inv, inv);
      float o[8];
#pragma unroll
      for (int k = 0; k < 2; ++k) {
        unpack_f32x2(mul_f32x2(fma_f32x2(x2[k], p2[k], mul_f32x2(x1[k], p1[k])), inv2), o[2 * k], o[2 * k + 1]);
        unpack_f32x2(mul_f32x2(fma_f32x2(x1[k], p4[k], mul_f32x2(x2[k], p3[k])), inv2), o[4 + 2 * k], o[5 + 2 * k]);
      }
      if (h < p.hq) {
        __nv_bfloat16* dst = p.q_out + (static_cast<size_t>(t) * p.hq + h) * D + 4 * c;
        *reinterpret_cast<uint2*>(dst) = make_uint2(pack_bf16(o[0], o[1]), pack_bf16(o[2], o[3]));
        *reinterpret_cast<uint2*>(dst + HALF) = make_uint2(pack_bf16(o[4], o[5]), pack_bf16(o[6], o[7]));
      }
    }
    return;
  }

  // ---- K and V ----
  const int slot = p.slots[t];
  if (slot >= p.num_slots && lane == 0) report_status(p.status, kIdWrite, kBadIndex);
  if (slot < 0 || slot >= p.num_slots) return;
  const int kv_pairs = (p.hkv + 1) / 2;
  const int first = task * p.kv_per_warp, last = min(first + p.kv_per_warp, 2 * kv_pairs);
  const int place = slot % p.block_size;
  const size_t unit0 = kv4::unit_offset(slot / p.block_size, 0, p.hkv, p.block_size, place);
  const size_t head_bytes = static_cast<size_t>(p.block_size / kv4::kUnit) * kv4::kUnitBytes;
  const unsigned half_mask = half ? 0xffff0000u : 0x0000ffffu;
  auto head_of = [&](int pair) { return min(2 * (pair < kv_pairs ? pair : pair - kv_pairs) + half, p.hkv - 1); };
  auto source = [&](int pair) { return p.hq + (pair < kv_pairs ? 0 : p.hkv) + head_of(pair); };
#pragma unroll 2
  for (int i = first; i < last; ++i) send(i - first, source(i));
  bool small_w = false;
  if (first < kv_pairs) {
    rotary(p.k_w);
    float least = FLT_MAX;
#pragma unroll
    for (int k = 0; k < 8; ++k) least = fminf(least, fabsf(w[k]));
    small_w = __any_sync(0xffffffffu, least < 0x1p-40f);
  }
  arrive();
  for (int pair = first; pair < last; ++pair) {
    uint2 a, b;
    load(pair - first, source(pair), a, b);
    const bool is_k = pair < kv_pairs;
    const int h = head_of(pair);
    const bool there = 2 * (is_k ? pair : pair - kv_pairs) + half < p.hkv;
    float x[8];
    unpack(a, b, x);
    if (is_k) {
      double ss = 0.0;
#pragma unroll
      for (int k = 0; k < 8; ++k) ss += widen(x[k]) * widen(x[k]);
      ss = half_sum(ss);
      double ms = ss * (1.0 / D) + p.eps;
      if (ms > 1e38) {                                        // beyond fp32: the row at 2^-100 of its size
        ms *= 0x1p-200;
#pragma unroll
        for (int k = 0; k < 8; ++k) x[k] *= 0x1p-100f;
      } else if (ms < 1e-30) {                                // below it (without an eps): the row at 2^100 of its size
        ms *= 0x1p200;
#pragma unroll
        for (int k = 0; k < 8; ++k) x[k] = mul_whole(x[k], 0x1p100f);
      }
      const float about = rsqrtf(static_cast<float>(ms));     // one Newton step doubles its 22 bits; 0 for an infinite row
      double inv = about;
      if (about > 0.f) inv += 0.5 * inv * (1.0 - ms * inv * inv);
      float k8[8];
      auto rotate = [&](int k, double u, double v) {
        const double cd = cs[k], sd = sn[k];
        k8[k] = round_bf16(narrow((u * cd - v * sd) * inv));
        k8[4 + k] = round_bf16(narrow((v * cd + u * sd) * inv));
      };
      if (small_w || __any_sync(0xffffffffu, ss < 0x1p-120)) {       // products that may leave fp32
#pragma unroll
        for (int k = 0; k < 4; ++k) rotate(k, widen(x[k]) * widen(w[k]), widen(x[4 + k]) * widen(w[4 + k]));
      } else {                                                // value times weight is exact in fp32: 8 + 8 bits
#pragma unroll
        for (int k = 0; k < 4; ++k) rotate(k, x[k] * w[k], x[4 + k] * w[4 + k]);
      }
      store_row(p.k_cache + unit0 + h * head_bytes, place % kv4::kUnit, c, half_mask, k8, there);
    } else {
      store_row(p.v_cache + unit0 + h * head_bytes, place % kv4::kUnit, c, half_mask, x, there);
    }
  }
}

// Eight channels of one word as bf16: c + s (n - 8), rounded once.
__device__ __forceinline__ uint4 dequant8(uint32_t w, uint32_t par) {
  const uint32_t s2 = __byte_perm(par, par, 0x1010), c2 = __byte_perm(par, par, 0x3232);
  const __nv_bfloat162 s = *reinterpret_cast<const __nv_bfloat162*>(&s2), c = *reinterpret_cast<const __nv_bfloat162*>(&c2);
  uint32_t v[4];
#pragma unroll
  for (int j = 0; j < 4; ++j) {                               // channels j and j + 4
    const uint32_t n = kv4::centred(kv4::biased(w, 4 * j));
    const __nv_bfloat162 r = __hfma2(*reinterpret_cast<const __nv_bfloat162*>(&n), s, c);
    v[j] = *reinterpret_cast<const uint32_t*>(&r);
  }
  return make_uint4(__byte_perm(v[0], v[1], 0x5410), __byte_perm(v[2], v[3], 0x5410), __byte_perm(v[0], v[1], 0x7632),
                    __byte_perm(v[2], v[3], 0x7632));
}

// A warp per token: one half reads K's heads, the other V's; lane c turns word c (8 channels) into 16 bytes of bf16.
__global__ void __launch_bounds__(256)
kv4_read_kernel(const uint8_t* __restrict__ k_cache, const uint8_t* __restrict__ v_cache, const int* __restrict__ slots,
                __nv_bfloat16* __restrict__ k_out, __nv_bfloat16* __restrict__ v_out, int tokens, int hkv, int block_size,
                int num_slots, int* status) {
  grid_dep_launch();
  grid_dep_wait();
  const int t = blockIdx.x * 8 + (threadIdx.x >> 5);
  if (t >= tokens) return;
  const int lane = threadIdx.x & 31, c = lane & 15;
  const int slot = slots[t];
  uint4* dst = reinterpret_cast<uint4*>((lane < 16 ? k_out : v_out) + static_cast<size_t>(t) * hkv * kv4::kD) + c;
  if (slot < 0 || slot >= num_slots) {
    if (slot >= 0 && lane == 0) report_status(status, kIdRead, kBadIndex);
    for (int h = 0; h < hkv; ++h) dst[h * 16] = make_uint4(0u, 0u, 0u, 0u);
    return;
  }
  const int place = slot % block_size;
  const uint8_t* unit = (lane < 16 ? k_cache : v_cache) + kv4::unit_offset(slot / block_size, 0, hkv, block_size, place);
  const uint8_t* code = unit + (place % kv4::kUnit) * kv4::kCodeRow + c * 4;
  const uint8_t* par = unit + kv4::kParBase + (place % kv4::kUnit) * kv4::kParRow + (c & 1) * 4;
  const size_t head_bytes = static_cast<size_t>(block_size / kv4::kUnit) * kv4::kUnitBytes;
  // Eight rows' reads in flight, then four, then one. The values leave L2 first: nothing here reads them again. 32768 tokens of
  // 8 heads in a graph take 26.1 us; with plain stores 29.7, with four rows in flight 26.9, with both 32.0.
  int h = 0;
  auto rows = [&](auto n) {
    constexpr int N = decltype(n)::value;
    for (; h + N <= hkv; h += N) {
      uint32_t w[N], q[N];
#pragma unroll
      for (int i = 0; i < N; ++i) {
        w[i] = __ldg(reinterpret_cast<const uint32_t*>(code + (h + i) * head_bytes));
        q[i] = __ldg(reinterpret_cast<const uint32_t*>(par + (h + i) * head_bytes));
      }
#pragma unroll
      for (int i = 0; i < N; ++i) __stcs(dst + (h + i) * 16, dequant8(w[i], q[i]));
    }
  };
  rows(std::integral_constant<int, 8>{});
  rows(std::integral_constant<int, 4>{});
  rows(std::integral_constant<int, 1>{});
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
                 const void* k_w, double eps, const float* cos_sin, int max_pos, const int* positions, const int* slots,
                 void* q_out, void* k_cache, void* v_cache, int tokens, int hq, int hkv, int d, int block_size,
                 int num_blocks, int num_sms, int* status, cudaStream_t stream) {
  if (tokens <= 0) return 0;
  if (int rc = check_cache(hkv, d, block_size, num_blocks)) return rc;
  if (hq < 0 || max_pos <= 0 || num_sms <= 0 || (!qkv && !partials)) return XV_ERR_SHAPE;
  if (misaligned(qkv, 16) || misaligned(partials, 16) || misaligned(q_w, 16) || misaligned(k_w, 16) ||
      misaligned(cos_sin, 16) || misaligned(q_out, 16) || misaligned(k_cache, 16) || misaligned(v_cache, 16))
    return XV_ERR_ALIGN;
  // Pairs of heads per warp: one while that leaves a warp slot for each (short steps are latency), up to eight where it
  // saves making the token's rotary factors again. Below that cap the launch is about one wave, whose end is K's and V's
  // warps (a pair of K takes twice a pair of Q): they get half as many. 997 rows (40 + 2 x 8 heads) 8.0 -> 7.1 us, but
  // 8192 rows (32 + 2 x 8) at the cap 41.5 -> 42.6.
  const int q_pairs = (hq + 1) / 2, kv_pairs = 2 * ((hkv + 1) / 2);
  WriteParams p;
  const long long pairs = static_cast<long long>(tokens) * (q_pairs + kv_pairs), wave = static_cast<long long>(num_sms) * 32;
  p.per_warp = static_cast<int>(std::max(1ll, std::min<long long>(kMaxPairs, pairs / wave)));
  p.q_tasks = (q_pairs + p.per_warp - 1) / p.per_warp;
  p.kv_per_warp = p.per_warp == kMaxPairs ? kMaxPairs : (p.per_warp + 1) / 2;
  p.tasks = p.q_tasks + (kv_pairs + p.kv_per_warp - 1) / p.kv_per_warp;
  const long long blocks = (static_cast<long long>(tokens) * p.tasks + kWriteWarps - 1) / kWriteWarps;
  if (blocks > 0x0fffffffLL) return XV_ERR_SHAPE;
  p.qkv = static_cast<const __nv_bfloat16*>(qkv);
  p.planes = partials;
  p.q_w = static_cast<const __nv_bfloat16*>(q_w);
  p.k_w = static_cast<const __nv_bfloat16*>(k_w);
  p.cos_sin = cos_sin;
  p.positions = positions;
  p.slots = slots;
  p.q_out = static_cast<__nv_bfloat16*>(q_out);
  p.k_cache = static_cast<uint8_t*>(k_cache);
  p.v_cache = static_cast<uint8_t*>(v_cache);
  p.status = status;
  p.split_stride = split_stride;
  p.eps = eps;
  p.splits = splits; p.max_pos = max_pos; p.tokens = tokens; p.hq = hq; p.hkv = hkv; p.block_size = block_size;
  p.num_slots = num_blocks * block_size;
  launch_pdl(partials ? kv4_write_kernel<true> : kv4_write_kernel<false>, dim3(static_cast<unsigned>(blocks)), dim3(kWriteWarps * 32), 0, stream, p);
  return launch_ok();
}

int xv_kv4_read(const void* k_cache, const void* v_cache, const int* slots, void* k_out, void* v_out, int tokens, int hkv,
                int d, int block_size, int num_blocks, int* status, cudaStream_t stream) {
  if (tokens <= 0) return 0;
  if (int rc = check_cache(hkv, d, block_size, num_blocks)) return rc;
  if (misaligned(k_cache, 16) || misaligned(v_cache, 16) || misaligned(k_out, 16) || misaligned(v_out, 16))
    return XV_ERR_ALIGN;
  launch_pdl(kv4_read_kernel, dim3((static_cast<unsigned>(tokens) + 7) / 8), dim3(256), 0, stream,
             static_cast<const uint8_t*>(k_cache), static_cast<const uint8_t*>(v_cache), slots,
             static_cast<__nv_bfloat16*>(k_out), static_cast<__nv_bfloat16*>(v_out), tokens, hkv, block_size,
             num_blocks * block_size, status);
  return launch_ok();
}

}  // extern "C"
