// Paged GQA attention of single query rows over a KV cache held in 4 bits (format: common/kv4.cuh), head_dim 128.
//
//   kv4_decode_kernel  - one query row per sequence; a cluster of CTAs, one per KV split, owns (sequence, KV head). Each
//                        warp streams its own 16-token units through a ring of shared-memory slots (five 16-byte
//                        cp.async a lane for K and V of a unit; no block-wide barrier in the loop). Tokens are the M rows
//                        of both products and the group's query heads (up to 8, or 16 as two column tiles) the N
//                        columns, so one MMA covers 16 x 16 cache values:
//                          S^T[token, head] = s_g * (n Q^T) + (c_g - 8 s_g) * sum(Q)   per channel group g
//                          O^T[channel, head] = n^T (s_g P) - 8 sum(s_g P) + c_g^T P
//                        The MMAs are fp16 and see the codes as the subnormals that the nibbles are where they stand,
//                        n 2^-24 and n 2^-20, so a code of K costs an AND (and every second byte a shift). Scales and
//                        centres stay in fp32; the scale of V is folded into P before its one rounding to fp16.
//                        The tensor pipe aligns its sums by a subnormal's nominal exponent, -14: with n 2^-24 a sum of V
//                        loses what is below 2^-14 of the largest P s, which shows where 8 - 8 should leave 0 (an output
//                        of 5e-4 was off by 3e-5). So V's even codes are moved to n 2^-20 as well, a shift each (256 sequences
//                        131 -> 137 us); K's stay (a score loses 1e-5 of max |q| s; both moved: 143).
//                        K's lanes own 16-byte pieces of a row, V's lanes pair two tokens with PRMT, so codes go from
//                        shared memory to MMA operands in registers. Warps are merged through shared memory, splits
//                        through the cluster's distributed shared memory: one launch, no workspace.
//   kv4_share_kernel   - the same arithmetic for large or ragged batches: all units dealt to the warps in equal runs,
//   kv4_join_kernel      partial results of pairs that span runs joined by a second kernel.
// Prompt chunks: attn_prefill_kv4_sm100.cu.
//
// What bounds it: instructions, not memory: 275 of them for the 2304 bytes of 16 tokens of a head (some 20 more for groups of
// more than four query heads; up to four have columns for both channel groups: 256 sequences 137 -> 129 us, 32 11.7 -> 11.4),
// 104 of which take the codes apart. 96 sequences of 2048 tokens, 32 / 8 heads: 58% of the issue slots, 52% of the ALU, 30%
// of the tensor pipe, 4.2 TB/s. 256 sequences of 256-4096 tokens 147 us in a stream (4.4 TB/s), 139 with L2 flushed, 129 in
// a graph, whose passes find part of the cache in L2; one of 40960 (64 / 8 heads) 22.1 us in a stream, 27.7 with L2 flushed
// (1.7 TB/s). Groups of 16 heads: 32 sequences of 128-1280 18.2 us (128 / 8 heads), 256 215. On the way:
// codes as bf16 integers with shifts and a subtraction 333 instructions and 153 us, a unit at a time 424 and 189, bulk copies
// in place of cp.async 241. 128 registers, for four CTAs an SM, spill: 149 us. Small batches are a chain of dependent
// reads (length and page, codes), about 2500 cycles before the first product.

#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_runtime.h>
#include <math_constants.h>

#include <algorithm>
#include <atomic>
#include <cmath>
#include <type_traits>

#include "../common/kv4.cuh"
#include "../common/launch.cuh"
#include "../common/ptx.cuh"
#include "xv_cuda.h"

namespace {

using namespace xv;

constexpr int kD = kv4::kD;
constexpr int kIdDecode = 10;
constexpr double kLog2e = 1.4426950408889634;

struct Params {
  const __nv_bfloat16* q;
  const uint8_t* k_cache;
  const uint8_t* v_cache;
  const int* block_tables;
  const int* kv_lens;
  __nv_bfloat16* out;
  int* status;
  int hq, hkv, block_size, max_blocks, num_blocks, splits;
  int max_tokens;                        // that a block table can name; 32-bit sums of a unit more must not wrap
  float scale, sign;                     // of a score, times log2 e: sign * scale * 2^scale_exp, scale in 1/4 .. 1/2
  int scale_exp;
};

// Cached tokens of a sequence, never more than its block table can name.
__device__ __forceinline__ int kv_len_of(const Params& p, int b) {
  const int n = p.kv_lens[b];
  if (n > p.max_tokens) {
    report_status(p.status, kIdDecode, kBadIndex);
    return p.max_tokens;
  }
  return n < 0 ? 0 : n;
}

__device__ __forceinline__ uint32_t movmatrix_trans(uint32_t a) {
  uint32_t d;
  asm volatile("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(d) : "r"(a));
  return d;
}

// Token of row r (0..7) of an 8-row group of the MMAs. V's lanes read the tokens of rows 2t and 2t + 1: with this order
// their four 64-byte rows start on alternating halves of the 128-byte bank line (two-way conflicts, not four-way).
__device__ __forceinline__ int token_of_row(int r) { return ((r >> 1) ^ (r & 1)) + 4 * (r & 1); }

__device__ __forceinline__ float ld_cluster_f32(uint32_t addr) {
  float v;
  asm volatile("ld.shared::cluster.f32 %0, [%1];" : "=f"(v) : "r"(addr) : "memory");
  return v;
}

__device__ __forceinline__ void cp_async16_u32(uint32_t dst, const void* src, uint64_t policy) {
  asm volatile("cp.async.cg.shared.global.L2::cache_hint [%0], [%1], 16, %2;" ::"r"(dst), "l"(src), "l"(policy) : "memory");
}

constexpr int kStages = 3;               // ring slots of a warp (four measure the same)
constexpr int kPair = 2;                 // units per slot: two independent chains of work per iteration of a warp
constexpr int kUnitSlot = 2 * kv4::kUnitBytes;
constexpr int kSlot = kPair * kUnitSlot;
constexpr float kNoMax = -3.0e38f;       // finite, so that "nothing seen yet" needs no case of its own
constexpr float kLazy = 8.f;             // log2 units a running maximum may lag behind
constexpr uint32_t kLow = 0x000f000fu, kHigh = 0x00f000f0u;      // nibbles as fp16: n 2^-24, n 2^-20 (subnormals)
constexpr uint32_t kMinus8 = 0xC800C800u;                        // fp16 -8

constexpr int decode_smem(int warps) { return warps * kStages * kSlot; }

// Four channels of an output row from unnormalised sums; a row that saw nothing is zero.
__device__ __forceinline__ void store_out(__nv_bfloat16* dst, const float4& v, float l) {
  const float inv = l == 0.f ? 0.f : 1.f / l;
  *reinterpret_cast<uint2*>(dst) = make_uint2(pack_bf16(v.x * inv, v.y * inv), pack_bf16(v.z * inv, v.w * inv));
}

// D = A B on bf16: the centres' share of a score.
__device__ __forceinline__ void mma_bf16(float (&d)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
  asm(
      "mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, "
      "{%10, %10, %10, %10};"
      : "=f"(d[0]), "=f"(d[1]), "=f"(d[2]), "=f"(d[3])
      : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1), "f"(0.f));
}

// D = A B on fp16, and D += A B. Unlike ptx.cuh's forms not volatile: the two units of a slot may be interleaved.
__device__ __forceinline__ void mma_first(float (&d)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
  asm(
      "mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, "
      "{%10, %10, %10, %10};"
      : "=f"(d[0]), "=f"(d[1]), "=f"(d[2]), "=f"(d[3])
      : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1), "f"(0.f));
}
__device__ __forceinline__ void mma_more(float (&d)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
  asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, "
      "{%0, %1, %2, %3};"
      : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
      : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}

__device__ __forceinline__ uint32_t pack_f16(float lo, float hi) {
  const __half2 v = __floats2half2_rn(lo, hi);
  return *reinterpret_cast<const uint32_t*>(&v);
}
__device__ __forceinline__ float power_of_two(int e) { return __int_as_float((e + 127) << 23); }       // e in -126 .. 127

// The group's queries as B operands. NT: column tiles of 8 query heads. TWIN (up to four heads): column n + 4 is head n
// again, columns 0-3 hold its channels of group 0 and zeros, columns 4-7 those of group 1.
template <int NT, bool TWIN>
struct Query {
  static_assert(!TWIN || NT == 1);
  // MMA (word w, half hf) of lane (g, t) multiplies channels 32 t + 8 w + 2 hf + {0, 4, 1, 5}. Q is held in fp16, every head
  // scaled by a power of two that takes its largest value to 2^14 .. 2^15 (exact down to 2^-28 of it); the odd channels meet
  // codes that are 16 times too large and carry another 1 / 16.
  uint32_t f[NT][4][2][2];
  // The centres' share of a score, sum over groups of c_g Qs_g - 8 s_g Qs_g with Qs_g the group's sum of Q, is one more
  // MMA: its A operand is the parameter words as stored, its B operand {-8 Qs_g, Qs_g} as three bf16 terms (24 bits).
  uint32_t c[NT][2];
  // What the MMAs and K's parameters make of a score, times power, is the score in log2 units. power joins the head's power of
  // two, the codes' 2^-24 and the exponent of the softmax's scale, whose mantissa is in lift, by which K's steps and the
  // centres' operand are multiplied. A power of two, so that x power - m power is 0 for the largest x however large the scores
  // are. It stays in 2^-100 .. 2^120: where a head's would be larger (queries from 2^107 on at ordinary scales) lift takes the
  // rest for all heads of the group, where it would be smaller the head's Q is scaled down. For heads 2t, 2t + 1 of each tile.
  float power[NT][2], lift;

  uint32_t raw[NT][16];
  // Sends for Q. `row`: sequence * hq + first query head of the group.
  __device__ __forceinline__ void fetch(const Params& p, size_t row, int G, int g, int t) {
#pragma unroll
    for (int nt = 0; nt < NT; ++nt) {
      const int head = TWIN ? g & 3 : nt * 8 + g;
      const uint4* src = reinterpret_cast<const uint4*>(p.q + (row + head) * kD + 32 * t);
#pragma unroll
      for (int w = 0; w < 4; ++w) {
        const uint4 r = head < G ? __ldg(src + w) : make_uint4(0, 0, 0, 0);
        raw[nt][4 * w] = r.x; raw[nt][4 * w + 1] = r.y; raw[nt][4 * w + 2] = r.z; raw[nt][4 * w + 3] = r.w;
      }
    }
  }
  // Makes the operands of what fetch() brought.
  __device__ __forceinline__ void convert(const Params& p, int g, int t) {
    int e[NT];
#pragma unroll
    for (int nt = 0; nt < NT; ++nt) {
      uint32_t top = 0;
#pragma unroll
      for (int i = 0; i < 16; ++i) top = __vmaxu2(top, raw[nt][i] & 0x7fff7fffu);
      uint32_t most = max(top >> 16, top & 0xffffu);
      if (most >= 0x7f80u) {                               // infinities and NaN do not choose a power
        most = 0;
#pragma unroll
        for (int i = 0; i < 16; ++i) {
          const uint32_t lo = raw[nt][i] & 0x7fffu, hi = (raw[nt][i] >> 16) & 0x7fffu;
          most = max(most, max(lo < 0x7f80u ? lo : 0u, hi < 0x7f80u ? hi : 0u));
        }
      }
      most = max(most, __shfl_xor_sync(0xffffffffu, most, 1));
      most = max(most, __shfl_xor_sync(0xffffffffu, most, 2));
      e[nt] = max(static_cast<int>(most >> 7) - 127 - 14, -120);
    }
    const int top_e = __reduce_max_sync(0xffffffffu, NT == 2 ? max(e[0], e[NT - 1]) : e[0]), rest = p.scale_exp + 24;
    const int over = min(max(top_e + rest - 120, 0), 120);
    lift = p.scale * power_of_two(over);
#pragma unroll
    for (int nt = 0; nt < NT; ++nt) {
      e[nt] = max(e[nt], over - rest - 100);
#pragma unroll
      for (int hd = 0; hd < 2; ++hd)                       // a lane's scores are those of heads 2t + hd, whose rows lanes g = 2t + hd have
        power[nt][hd] = power_of_two(min(__shfl_sync(0xffffffffu, e[nt], 8 * t + 4 * hd) + rest - over, 127));
    }
#pragma unroll
    for (int nt = 0; nt < NT; ++nt) {
      const float by = power_of_two(-e[nt]) * p.sign;
      float sum[2] = {0.f, 0.f};
#pragma unroll
      for (int w = 0; w < 4; ++w) {
        float x[8];
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          x[2 * i] = __uint_as_float(raw[nt][4 * w + i] << 16) * by;
          x[2 * i + 1] = __uint_as_float(raw[nt][4 * w + i] & 0xffff0000u) * by;
          sum[w & 1] += x[2 * i] + x[2 * i + 1];
        }
#pragma unroll
        for (int hf = 0; hf < 2; ++hf) {
          f[nt][w][hf][0] = pack_f16(x[2 * hf], x[2 * hf + 4]);
          f[nt][w][hf][1] = pack_f16(x[2 * hf + 1] * 0.0625f, x[2 * hf + 5] * 0.0625f);
          if (TWIN && (w & 1) != (g >> 2)) f[nt][w][hf][0] = f[nt][w][hf][1] = 0u;
        }
      }
#pragma unroll
      for (int gr = 0; gr < 2; ++gr) {
        sum[gr] += __shfl_xor_sync(0xffffffffu, sum[gr], 1);
        sum[gr] += __shfl_xor_sync(0xffffffffu, sum[gr], 2);
      }
      // Lane (g, t) holds K rows 2t, 2t + 1 of B (first register) and 2t + 8, 2t + 9 (second): group t & 1; the first
      // term for t < 2, the second for t >= 2, the third in the second register for t < 2.
      const float qs = ((t & 1) ? sum[1] : sum[0]) * 5.9604644775390625e-08f * lift, bs = -8.f * qs;      // 2^-24
      const float q1 = __bfloat162float(__float2bfloat16(qs)), b1 = __bfloat162float(__float2bfloat16(bs));
      const float q2 = __bfloat162float(__float2bfloat16(qs - q1)), b2 = __bfloat162float(__float2bfloat16(bs - b1));
      c[nt][0] = t < 2 ? pack_bf16(b1, q1) : pack_bf16(b2, q2);
      c[nt][1] = t < 2 ? pack_bf16(bs - b1 - b2, qs - q1 - q2) : 0u;
      if (TWIN && g >= 4) c[nt][0] = c[nt][1] = 0u;        // both groups' centres count once
    }
  }
};

// Running state of the softmax over the tokens a warp has seen.
// How V's steps and P are scaled on their way to fp16. A step is multiplied by vs, one power of two for a warp, to 2^-6 .. 2^-1;
// saturation leaves that alone and makes NaN 0. (With more than four heads both groups' offsets are one accumulator, where a
// NaN of one would reach the other; the centre of such a group is NaN as well and stays in its channels.) P is multiplied by
// 2^k: 2^8, or where steps are far apart each head's own, so that the largest P s of what it gives weight is 4 .. 8: a token that
// a head gives none does not decide how the others are held. Both cancel at the end.
struct Scaling {
  float vs = 0.f, most = 0.f;            // no step yet; steps above `most` need a look: with a P of 2^8 they might leave fp16

  // To a larger step; returns what sums of P * s are to be multiplied by.
  __device__ __forceinline__ float fit(float step) {
    if (step == 0.f || (vs != 0.f && step * vs <= 0.5f)) return 1.f;
    const float now = power_of_two(-min(max((__float_as_int(step) >> 23) - 127 + 6, -112), 126));
    const float back = vs == 0.f ? 1.f : now / vs;
    vs = now;
    return back;
  }
  // Whether a slot is more than ordinary: `low`, this lane's smallest step that is not 0, is far below the slot's largest, the
  // steps so far are, or P is not at 2^8.
  static __device__ __forceinline__ bool apart(float low, float step, float back, bool other_k) {
    return __any_sync(0xffffffffu, low * 1024.f < step || back < 0.00390625f || other_k);
  }
  // A head's k for a slot whose largest P s and P |c| are given, where the sums so far are multiplied by `shrunk`. Beyond scores
  // of 2^20 rounding would take its part of it.
  __device__ __forceinline__ float next_k(float k, float shrunk, float ps, float pc, float score) const {
    auto ilog = [](float x) { return static_cast<float>((__float_as_int(x) >> 23) - 127); };
    float to = fminf(k - log2f(shrunk), 90.f);             // what they leave room for
    if (ps > 0.f) to = fminf(to, 2.f - ilog(ps * vs));
    if (pc > 0.f) to = fminf(to, 100.f - ilog(pc));        // the centres' sums stay in fp32
    if (fabsf(score) > 1048576.f) to = fminf(to, 8.f);
    return fmaxf(floorf(to), 0.f);
  }
  __device__ __forceinline__ void limit(float most_k) {
    if (vs != 0.f) most = exp2f(fminf(-1.f, 7.f - most_k)) / vs;
  }
  __device__ __forceinline__ float back() const { return vs == 0.f ? 0.f : 1.f / vs; }
};
// |s| and |c| of a parameter word; its step as a candidate for the smallest that is not 0.
__device__ __forceinline__ float low_s(uint32_t w) { return (w & 0x7fffu) == 0u ? CUDART_INF_F : fabsf(kv4::par_s(w)); }
__device__ __forceinline__ float abs_s(uint32_t w) { return fabsf(kv4::par_s(w)); }
__device__ __forceinline__ float abs_c(uint32_t w) { return fabsf(kv4::par_c(w)); }

template <int NT>
struct Softmax {
  float o[NT][2][4][4];            // [group][MMA]: rows g, g + 8 = channels 16 g + 8 group + 2 i + {0, 1}; heads 2t, 2t+1
  float cen[NT][2][2];             // sum of P * centre, this lane's tokens
  float off[NT][4];                // sum of -8 P * s, rounded as it is in o: group 0 (heads 2t, 2t + 1), group 1
  float m[NT][2], l[NT][2];        // running maximum of the products (may lag), sum of P of this lane's tokens
  float k[NT][2];
  Scaling v;

  __device__ __forceinline__ void clear() {
    v = Scaling();
#pragma unroll
    for (int nt = 0; nt < NT; ++nt) {
      k[nt][0] = k[nt][1] = 8.f;
#pragma unroll
      for (int gr = 0; gr < 2; ++gr) {
#pragma unroll
        for (int i = 0; i < 4; ++i) o[nt][gr][i][0] = o[nt][gr][i][1] = o[nt][gr][i][2] = o[nt][gr][i][3] = 0.f;
        cen[nt][gr][0] = cen[nt][gr][1] = 0.f;
      }
      off[nt][0] = off[nt][1] = off[nt][2] = off[nt][3] = 0.f;
      m[nt][0] = m[nt][1] = kNoMax;
      l[nt][0] = l[nt][1] = 0.f;
    }
  }

  // One slot of kPair units, of which the first `mine` tokens count. lane_k .. lane_v1: this lane's places in the slot.
  __device__ __forceinline__ void add(const Query<NT, false>& q, const uint8_t* lane_k, const uint8_t* lane_p, const uint8_t* lane_v0,
                                      const uint8_t* lane_v1, int mine, int tok, int t) {
    float x[kPair][NT][4];               // (row g: heads 2t, 2t + 1), (row g + 8: the same)
#pragma unroll
    for (int u = 0; u < kPair; ++u) {
      const uint4 k0 = *reinterpret_cast<const uint4*>(lane_k + u * kUnitSlot);
      const uint4 k1 = *reinterpret_cast<const uint4*>(lane_k + u * kUnitSlot + 8 * 64);
      const uint2 kp0 = *reinterpret_cast<const uint2*>(lane_p + u * kUnitSlot);
      const uint2 kp1 = *reinterpret_cast<const uint2*>(lane_p + u * kUnitSlot + 64);
      const uint32_t ka[4] = {k0.x, k0.y, k0.z, k0.w}, kb[4] = {k1.x, k1.y, k1.z, k1.w};
      const uint32_t w0 = *reinterpret_cast<const uint32_t*>(lane_p + u * kUnitSlot + (t & 1) * 4);
      const uint32_t w1 = *reinterpret_cast<const uint32_t*>(lane_p + u * kUnitSlot + (t & 1) * 4 + 64);
      const uint32_t ac[4] = {w0, w1, w0, w1};
      float s[NT][2][4], sc[NT][4];
#pragma unroll
      for (int nt = 0; nt < NT; ++nt) mma_bf16(sc[nt], ac, q.c[nt][0], q.c[nt][1]);
#pragma unroll
      for (int w = 0; w < 4; ++w)
#pragma unroll
        for (int hf = 0; hf < 2; ++hf) {
          const uint32_t wa = ka[w] >> (8 * hf), wb = kb[w] >> (8 * hf);
          const uint32_t a[4] = {wa & kLow, wb & kLow, wa & kHigh, wb & kHigh};
#pragma unroll
          for (int nt = 0; nt < NT; ++nt) {
            if (w < 2 && hf == 0) mma_first(s[nt][w], a, q.f[nt][w][hf][0], q.f[nt][w][hf][1]);
            else mma_more(s[nt][w & 1], a, q.f[nt][w][hf][0], q.f[nt][w][hf][1]);
          }
        }
      const float ks[2][2] = {{kv4::par_s(kp0.x) * q.lift, kv4::par_s(kp0.y) * q.lift},
                              {kv4::par_s(kp1.x) * q.lift, kv4::par_s(kp1.y) * q.lift}};
#pragma unroll
      for (int nt = 0; nt < NT; ++nt)
#pragma unroll
        for (int e = 0; e < 4; ++e) x[u][nt][e] = fmaf(ks[e >> 1][0], s[nt][0][e], fmaf(ks[e >> 1][1], s[nt][1][e], sc[nt][e]));
    }
    const bool ragged = mine < 16 * kPair;               // warp-uniform
    if (ragged) {
#pragma unroll
      for (int u = 0; u < kPair; ++u)
#pragma unroll
        for (int nt = 0; nt < NT; ++nt) {
          if (16 * u + tok >= mine) x[u][nt][0] = x[u][nt][1] = -CUDART_INF_F;
          if (16 * u + tok + 8 >= mine) x[u][nt][2] = x[u][nt][3] = -CUDART_INF_F;
        }
    }
    uint2 vp[kPair][2];                  // V's parameters of this lane's tokens
    float s_most = 0.f;
#pragma unroll
    for (int u = 0; u < kPair; ++u) {
      vp[u][0] = *reinterpret_cast<const uint2*>(lane_p + u * kUnitSlot + kv4::kUnitBytes);
      vp[u][1] = *reinterpret_cast<const uint2*>(lane_p + u * kUnitSlot + kv4::kUnitBytes + 64);
      if (ragged) {                      // P is 0 there, and whatever parameters an earlier owner of the page left (NaN
        if (16 * u + tok >= mine) vp[u][0] = make_uint2(0u, 0u);     // among them) must not reach the sums; codes are
        if (16 * u + tok + 8 >= mine) vp[u][1] = make_uint2(0u, 0u); // always finite
      }
#pragma unroll
      for (int r = 0; r < 2; ++r) s_most = fmaxf(s_most, fmaxf(fabsf(kv4::par_s(vp[u][r].x)), fabsf(kv4::par_s(vp[u][r].y))));
    }
    bool grow = s_most > v.most;
    float mx[NT][2];
#pragma unroll
    for (int nt = 0; nt < NT; ++nt)
#pragma unroll
      for (int hd = 0; hd < 2; ++hd) {
        mx[nt][hd] = fmaxf(fmaxf(x[0][nt][hd], x[0][nt][2 + hd]), fmaxf(x[1][nt][hd], x[1][nt][2 + hd]));
        grow |= (mx[nt][hd] - m[nt][hd]) * q.power[nt][hd] > kLazy;
      }
    if (__any_sync(0xffffffffu, grow)) {
      s_most = fmaxf(s_most, __shfl_xor_sync(0xffffffffu, s_most, 4));
      s_most = fmaxf(s_most, __shfl_xor_sync(0xffffffffu, s_most, 8));
      s_most = fmaxf(s_most, __shfl_xor_sync(0xffffffffu, s_most, 16));
      const float back = v.fit(s_most);
      float low = CUDART_INF_F, shrunk[NT][2];
      bool other_k = false;
#pragma unroll
      for (int u = 0; u < kPair; ++u)
#pragma unroll
        for (int r = 0; r < 2; ++r) low = fminf(low, fminf(low_s(vp[u][r].x), low_s(vp[u][r].y)));
#pragma unroll
      for (int nt = 0; nt < NT; ++nt) other_k |= k[nt][0] != 8.f || k[nt][1] != 8.f;
      const bool apart = Scaling::apart(low, s_most, back, other_k);
#pragma unroll
      for (int nt = 0; nt < NT; ++nt)
#pragma unroll
        for (int hd = 0; hd < 2; ++hd) {
          float mn = fmaxf(m[nt][hd], mx[nt][hd]);
          mn = fmaxf(mn, __shfl_xor_sync(0xffffffffu, mn, 4));
          mn = fmaxf(mn, __shfl_xor_sync(0xffffffffu, mn, 8));
          mn = fmaxf(mn, __shfl_xor_sync(0xffffffffu, mn, 16));
          const float cr = exp2f((m[nt][hd] - mn) * q.power[nt][hd]);
          m[nt][hd] = mn;
          shrunk[nt][hd] = cr * back;
          l[nt][hd] *= cr;
#pragma unroll
          for (int gr = 0; gr < 2; ++gr) {
            cen[nt][gr][hd] *= cr;
            off[nt][2 * gr + hd] *= cr * back;
#pragma unroll
            for (int j = 0; j < 4; ++j) {
              o[nt][gr][j][hd] *= cr * back;
              o[nt][gr][j][2 + hd] *= cr * back;
            }
          }
        }
      float most_k = 8.f;
      if (__builtin_expect(apart, false)) {
        most_k = 0.f;
#pragma unroll
        for (int nt = 0; nt < NT; ++nt)
#pragma unroll
          for (int hd = 0; hd < 2; ++hd) {
            float ps = 0.f, pc = 0.f;
#pragma unroll
            for (int u = 0; u < kPair; ++u)
#pragma unroll
              for (int r = 0; r < 2; ++r) {
                const float pr = exp2f((x[u][nt][2 * r + hd] - m[nt][hd]) * q.power[nt][hd]);
                ps = fmaxf(ps, pr * fmaxf(abs_s(vp[u][r].x), abs_s(vp[u][r].y)));
                pc = fmaxf(pc, pr * fmaxf(abs_c(vp[u][r].x), abs_c(vp[u][r].y)));
              }
#pragma unroll
            for (int d = 4; d <= 16; d <<= 1) {
              ps = fmaxf(ps, __shfl_xor_sync(0xffffffffu, ps, d));
              pc = fmaxf(pc, __shfl_xor_sync(0xffffffffu, pc, d));
            }
            const float to = v.next_k(k[nt][hd], shrunk[nt][hd], ps, pc, m[nt][hd] * q.power[nt][hd]), up = exp2f(to - k[nt][hd]);
            k[nt][hd] = to;
            most_k = fmaxf(most_k, to);
            l[nt][hd] *= up;
#pragma unroll
            for (int gr = 0; gr < 2; ++gr) {
              cen[nt][gr][hd] *= up;
              off[nt][2 * gr + hd] *= up;
#pragma unroll
              for (int j = 0; j < 4; ++j) {
                o[nt][gr][j][hd] *= up;
                o[nt][gr][j][2 + hd] *= up;
              }
            }
          }
      }
      v.limit(most_k);
    }
#pragma unroll
    for (int u = 0; u < kPair; ++u) {
      uint2 vw[4];                       // tokens of rows 2t, 2t + 1, then the same 8 further
      vw[0] = *reinterpret_cast<const uint2*>(lane_v0 + u * kUnitSlot);
      vw[1] = *reinterpret_cast<const uint2*>(lane_v1 + u * kUnitSlot);
      vw[2] = *reinterpret_cast<const uint2*>(lane_v0 + u * kUnitSlot + 8 * 64);
      vw[3] = *reinterpret_cast<const uint2*>(lane_v1 + u * kUnitSlot + 8 * 64);
      float vsc[2][2], vce[2][2];        // [group][token g, g + 8]: s (scaled) and c
#pragma unroll
      for (int r = 0; r < 2; ++r)
#pragma unroll
        for (int gr = 0; gr < 2; ++gr) {
          const uint32_t w = gr ? vp[u][r].y : vp[u][r].x;
          vsc[gr][r] = __saturatef(kv4::par_s(w) * v.vs);
          vce[gr][r] = kv4::par_c(w);
        }
      uint32_t pf[NT][2][2];             // P * s_g as the B operand of the second product
#pragma unroll
      for (int nt = 0; nt < NT; ++nt) {
        float pr[4];
#pragma unroll
        for (int e = 0; e < 4; ++e) pr[e] = exp2f(fmaf(x[u][nt][e], q.power[nt][e & 1], fmaf(-m[nt][e & 1], q.power[nt][e & 1], k[nt][e & 1])));
        l[nt][0] += pr[0] + pr[2];
        l[nt][1] += pr[1] + pr[3];
#pragma unroll
        for (int gr = 0; gr < 2; ++gr) {
          pf[nt][gr][0] = movmatrix_trans(pack_f16(pr[0] * vsc[gr][0], pr[1] * vsc[gr][0]));
          pf[nt][gr][1] = movmatrix_trans(pack_f16(pr[2] * vsc[gr][1], pr[3] * vsc[gr][1]));
          cen[nt][gr][0] = fmaf(pr[0], vce[gr][0], fmaf(pr[2], vce[gr][1], cen[nt][gr][0]));
          cen[nt][gr][1] = fmaf(pr[1], vce[gr][0], fmaf(pr[3], vce[gr][1], cen[nt][gr][1]));
        }
      }
#pragma unroll
      for (int gr = 0; gr < 2; ++gr) {
        const uint32_t w0 = gr ? vw[0].y : vw[0].x, w1 = gr ? vw[1].y : vw[1].x, w2 = gr ? vw[2].y : vw[2].x,
                       w3 = gr ? vw[3].y : vw[3].x;
        const uint32_t a8[4] = {gr ? 0u : kMinus8, gr ? kMinus8 : 0u, gr ? 0u : kMinus8, gr ? kMinus8 : 0u};
#pragma unroll
        for (int nt = 0; nt < NT; ++nt) mma_more(off[nt], a8, pf[nt][gr][0], pf[nt][gr][1]);
#pragma unroll
        for (int i = 0; i < 4; ++i) {                  // byte of the word: channels 2 i, 2 i + 1
          const uint32_t u0 = __byte_perm(w0, w1, 0x4400 + 0x1111 * i), u1 = __byte_perm(w2, w3, 0x4400 + 0x1111 * i);
          const uint32_t a[4] = {(u0 << 4) & kHigh, u0 & kHigh, (u1 << 4) & kHigh, u1 & kHigh};
#pragma unroll
          for (int nt = 0; nt < NT; ++nt) mma_more(o[nt][gr][i], a, pf[nt][gr][0], pf[nt][gr][1]);
        }
      }
    }
  }

  // Sums over the lanes of equal t; the centres join the outputs, the maximum turns to log2 units. Then every lane holds, for
  // its two heads, 16 channels.
  __device__ __forceinline__ void finish(const Query<NT, false>& q) {
    const float back = v.back();
#pragma unroll
    for (int nt = 0; nt < NT; ++nt)
#pragma unroll
      for (int hd = 0; hd < 2; ++hd) {
        const float down = exp2f(-k[nt][hd]);
        l[nt][hd] *= down;
        cen[nt][0][hd] *= down;
        cen[nt][1][hd] *= down;
#pragma unroll
        for (int x = 4; x <= 16; x <<= 1) {
          l[nt][hd] += __shfl_xor_sync(0xffffffffu, l[nt][hd], x);
          cen[nt][0][hd] += __shfl_xor_sync(0xffffffffu, cen[nt][0][hd], x);
          cen[nt][1][hd] += __shfl_xor_sync(0xffffffffu, cen[nt][1][hd], x);
        }
#pragma unroll
        for (int gr = 0; gr < 2; ++gr)
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            o[nt][gr][i][hd] = fmaf(fmaf(o[nt][gr][i][hd], 1048576.f, off[nt][2 * gr + hd]) * down, back, cen[nt][gr][hd]);      // n 2^-20
            o[nt][gr][i][2 + hd] = fmaf(fmaf(o[nt][gr][i][2 + hd], 1048576.f, off[nt][2 * gr + hd]) * down, back, cen[nt][gr][hd]);
          }
        m[nt][hd] = m[nt][hd] == kNoMax ? kNoMax : m[nt][hd] * q.power[nt][hd];
      }
  }
  // After finish(), f(head, first of four channels, their sums, m, l) for what this lane (g, t) holds.
  template <typename F>
  __device__ __forceinline__ void each(int g, int t, F f) const {
#pragma unroll
    for (int nt = 0; nt < NT; ++nt)
#pragma unroll
      for (int hd = 0; hd < 2; ++hd)
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          const float(&a)[4] = o[nt][j >> 1][2 * (j & 1)], (&b)[4] = o[nt][j >> 1][2 * (j & 1) + 1];
          f(nt * 8 + 2 * t + hd, 16 * g + 4 * j, make_float4(a[hd], a[2 + hd], b[hd], b[2 + hd]), m[nt][hd], l[nt][hd]);
        }
  }
};

// The same for up to four heads on the columns of Query<1, true>: a lane has one group (t >> 1) of heads 2 (t & 1) + {0, 1}, so
// parameters, products with them and the operands of the second MMA are half as many; scores are the sum over lane pairs.
struct TwinSoftmax {
  float o[2][4][4];                // as Softmax::o; valid where [group] is the lane's own
  float cen[2], off[4];            // of the lane's group
  float m[2], l[2];
  float k[2];
  Scaling v;

  __device__ __forceinline__ void clear() {
    v = Scaling();
    k[0] = k[1] = 8.f;
#pragma unroll
    for (int gr = 0; gr < 2; ++gr)
#pragma unroll
      for (int i = 0; i < 4; ++i) o[gr][i][0] = o[gr][i][1] = o[gr][i][2] = o[gr][i][3] = 0.f;
    cen[0] = cen[1] = 0.f;
    off[0] = off[1] = off[2] = off[3] = 0.f;
    m[0] = m[1] = kNoMax;
    l[0] = l[1] = 0.f;
  }

  __device__ __forceinline__ void add(const Query<1, true>& q, const uint8_t* lane_k, const uint8_t* lane_p, const uint8_t* lane_v0,
                                      const uint8_t* lane_v1, int mine, int tok, int t) {
    const uint8_t* lane_s = lane_p + (t >> 1) * 4;       // the lane's group's parameters
    const uint8_t* lane_c = lane_p + (t & 1) * 4;        // those that the centres' MMA takes from it
    float x[kPair][4];
#pragma unroll
    for (int u = 0; u < kPair; ++u) {
      const uint4 k0 = *reinterpret_cast<const uint4*>(lane_k + u * kUnitSlot);
      const uint4 k1 = *reinterpret_cast<const uint4*>(lane_k + u * kUnitSlot + 8 * 64);
      const uint32_t s0 = *reinterpret_cast<const uint32_t*>(lane_s + u * kUnitSlot);
      const uint32_t s1 = *reinterpret_cast<const uint32_t*>(lane_s + u * kUnitSlot + 64);
      const uint32_t w0 = *reinterpret_cast<const uint32_t*>(lane_c + u * kUnitSlot);
      const uint32_t w1 = *reinterpret_cast<const uint32_t*>(lane_c + u * kUnitSlot + 64);
      const uint32_t ka[4] = {k0.x, k0.y, k0.z, k0.w}, kb[4] = {k1.x, k1.y, k1.z, k1.w};
      const uint32_t ac[4] = {w0, w1, w0, w1};
      float s[4], sc[4];
      mma_bf16(sc, ac, q.c[0][0], q.c[0][1]);
#pragma unroll
      for (int w = 0; w < 4; ++w)
#pragma unroll
        for (int hf = 0; hf < 2; ++hf) {
          const uint32_t wa = ka[w] >> (8 * hf), wb = kb[w] >> (8 * hf);
          const uint32_t a[4] = {wa & kLow, wb & kLow, wa & kHigh, wb & kHigh};
          if (w == 0 && hf == 0) mma_first(s, a, q.f[0][w][hf][0], q.f[0][w][hf][1]);
          else mma_more(s, a, q.f[0][w][hf][0], q.f[0][w][hf][1]);
        }
      const float ks[2] = {kv4::par_s(s0) * q.lift, kv4::par_s(s1) * q.lift};
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        x[u][e] = fmaf(ks[e >> 1], s[e], sc[e]);
        x[u][e] += __shfl_xor_sync(0xffffffffu, x[u][e], 2);
      }
    }
    const bool ragged = mine < 16 * kPair;               // warp-uniform
    uint32_t vp[kPair][2];                               // V's parameters of this lane's tokens and group
    float s_most = 0.f;
#pragma unroll
    for (int u = 0; u < kPair; ++u) {
      vp[u][0] = *reinterpret_cast<const uint32_t*>(lane_s + u * kUnitSlot + kv4::kUnitBytes);
      vp[u][1] = *reinterpret_cast<const uint32_t*>(lane_s + u * kUnitSlot + kv4::kUnitBytes + 64);
      if (ragged) {                                      // as in Softmax
        if (16 * u + tok >= mine) {
          x[u][0] = x[u][1] = -CUDART_INF_F;
          vp[u][0] = 0u;
        }
        if (16 * u + tok + 8 >= mine) {
          x[u][2] = x[u][3] = -CUDART_INF_F;
          vp[u][1] = 0u;
        }
      }
#pragma unroll
      for (int r = 0; r < 2; ++r) s_most = fmaxf(s_most, fabsf(kv4::par_s(vp[u][r])));
    }
    bool grow = s_most > v.most;
    float mx[2];
#pragma unroll
    for (int hd = 0; hd < 2; ++hd) {
      mx[hd] = fmaxf(fmaxf(x[0][hd], x[0][2 + hd]), fmaxf(x[1][hd], x[1][2 + hd]));
      grow |= (mx[hd] - m[hd]) * q.power[0][hd] > kLazy;
    }
    if (__any_sync(0xffffffffu, grow)) {
#pragma unroll
      for (int d = 2; d <= 16; d <<= 1) s_most = fmaxf(s_most, __shfl_xor_sync(0xffffffffu, s_most, d));
      const float back = v.fit(s_most);
      float shrunk[2];
      const float low = fminf(fminf(low_s(vp[0][0]), low_s(vp[0][1])), fminf(low_s(vp[1][0]), low_s(vp[1][1])));
      const bool apart = Scaling::apart(low, s_most, back, k[0] != 8.f || k[1] != 8.f);
#pragma unroll
      for (int hd = 0; hd < 2; ++hd) {
        float mn = fmaxf(m[hd], mx[hd]);
        mn = fmaxf(mn, __shfl_xor_sync(0xffffffffu, mn, 4));
        mn = fmaxf(mn, __shfl_xor_sync(0xffffffffu, mn, 8));
        mn = fmaxf(mn, __shfl_xor_sync(0xffffffffu, mn, 16));
        const float cr = exp2f((m[hd] - mn) * q.power[0][hd]);
        m[hd] = mn;
        shrunk[hd] = cr * back;
        l[hd] *= cr;
        cen[hd] *= cr;
        off[hd] *= cr * back;
#pragma unroll
        for (int gr = 0; gr < 2; ++gr)
#pragma unroll
          for (int j = 0; j < 4; ++j) {
            o[gr][j][hd] *= cr * back;
            o[gr][j][2 + hd] *= cr * back;
          }
      }
      float most_k = 8.f;
      if (__builtin_expect(apart, false)) {
        most_k = 0.f;
#pragma unroll
        for (int hd = 0; hd < 2; ++hd) {
          float ps = 0.f, pc = 0.f;
#pragma unroll
          for (int u = 0; u < kPair; ++u)
#pragma unroll
            for (int r = 0; r < 2; ++r) {
              const float pr = exp2f((x[u][2 * r + hd] - m[hd]) * q.power[0][hd]);
              ps = fmaxf(ps, pr * abs_s(vp[u][r]));
              pc = fmaxf(pc, pr * abs_c(vp[u][r]));
            }
#pragma unroll
          for (int d = 2; d <= 16; d <<= 1) {              // the two groups of a head are of one k: their lanes share l
            ps = fmaxf(ps, __shfl_xor_sync(0xffffffffu, ps, d));
            pc = fmaxf(pc, __shfl_xor_sync(0xffffffffu, pc, d));
          }
          const float to = v.next_k(k[hd], shrunk[hd], ps, pc, m[hd] * q.power[0][hd]), up = exp2f(to - k[hd]);
          k[hd] = to;
          most_k = fmaxf(most_k, to);
          l[hd] *= up;
          cen[hd] *= up;
          off[hd] *= up;
#pragma unroll
          for (int gr = 0; gr < 2; ++gr)
#pragma unroll
            for (int j = 0; j < 4; ++j) {
              o[gr][j][hd] *= up;
              o[gr][j][2 + hd] *= up;
            }
        }
      }
      v.limit(most_k);
    }
#pragma unroll
    for (int u = 0; u < kPair; ++u) {
      uint2 vw[4];                                       // tokens of rows 2t, 2t + 1, then the same 8 further
      vw[0] = *reinterpret_cast<const uint2*>(lane_v0 + u * kUnitSlot);
      vw[1] = *reinterpret_cast<const uint2*>(lane_v1 + u * kUnitSlot);
      vw[2] = *reinterpret_cast<const uint2*>(lane_v0 + u * kUnitSlot + 8 * 64);
      vw[3] = *reinterpret_cast<const uint2*>(lane_v1 + u * kUnitSlot + 8 * 64);
      float pr[4];
#pragma unroll
      for (int e = 0; e < 4; ++e) pr[e] = exp2f(fmaf(x[u][e], q.power[0][e & 1], fmaf(-m[e & 1], q.power[0][e & 1], k[e & 1])));
      l[0] += pr[0] + pr[2];
      l[1] += pr[1] + pr[3];
      const float v0 = kv4::par_s(vp[u][0]) * v.vs, v1 = kv4::par_s(vp[u][1]) * v.vs;
      const float c0 = kv4::par_c(vp[u][0]), c1 = kv4::par_c(vp[u][1]);
      const uint32_t p0 = movmatrix_trans(pack_f16(pr[0] * v0, pr[1] * v0)), p1 = movmatrix_trans(pack_f16(pr[2] * v1, pr[3] * v1));
      cen[0] = fmaf(pr[0], c0, fmaf(pr[2], c1, cen[0]));
      cen[1] = fmaf(pr[1], c0, fmaf(pr[3], c1, cen[1]));
      const uint32_t a8[4] = {kMinus8, kMinus8, kMinus8, kMinus8};
      mma_more(off, a8, p0, p1);
#pragma unroll
      for (int gr = 0; gr < 2; ++gr) {
        const uint32_t w0 = gr ? vw[0].y : vw[0].x, w1 = gr ? vw[1].y : vw[1].x, w2 = gr ? vw[2].y : vw[2].x,
                       w3 = gr ? vw[3].y : vw[3].x;
#pragma unroll
        for (int i = 0; i < 4; ++i) {                    // byte of the word: channels 2 i, 2 i + 1
          const uint32_t u0 = __byte_perm(w0, w1, 0x4400 + 0x1111 * i), u1 = __byte_perm(w2, w3, 0x4400 + 0x1111 * i);
          const uint32_t a[4] = {(u0 << 4) & kHigh, u0 & kHigh, (u1 << 4) & kHigh, u1 & kHigh};
          mma_more(o[gr][i], a, p0, p1);
        }
      }
    }
  }

  __device__ __forceinline__ void finish(const Query<1, true>& q) {
    const float back = v.back();
#pragma unroll
    for (int hd = 0; hd < 2; ++hd) {
      const float down = exp2f(-k[hd]);
      l[hd] *= down;
      cen[hd] *= down;
#pragma unroll
      for (int x = 4; x <= 16; x <<= 1) {
        l[hd] += __shfl_xor_sync(0xffffffffu, l[hd], x);
        cen[hd] += __shfl_xor_sync(0xffffffffu, cen[hd], x);
      }
#pragma unroll
      for (int gr = 0; gr < 2; ++gr)
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          o[gr][i][hd] = fmaf(fmaf(o[gr][i][hd], 1048576.f, off[hd]) * down, back, cen[hd]);             // n 2^-20
          o[gr][i][2 + hd] = fmaf(fmaf(o[gr][i][2 + hd], 1048576.f, off[hd]) * down, back, cen[hd]);
        }
      m[hd] = m[hd] == kNoMax ? kNoMax : m[hd] * q.power[0][hd];
    }
  }
  template <typename F>
  __device__ __forceinline__ void each(int g, int t, F f) const {
    const bool second = t >= 2;
#pragma unroll
    for (int hd = 0; hd < 2; ++hd)
#pragma unroll
      for (int j = 0; j < 2; ++j) {
        auto own = [&](int i, int e) { return second ? o[1][i][e] : o[0][i][e]; };
        f(2 * (t & 1) + hd, 16 * g + 8 * (t >> 1) + 4 * j,
          make_float4(own(2 * j, hd), own(2 * j, 2 + hd), own(2 * j + 1, hd), own(2 * j + 1, 2 + hd)), m[hd], l[hd]);
      }
  }
};
template <int NT, bool TWIN>
using SoftmaxOf = std::conditional_t<TWIN, TwinSoftmax, Softmax<NT>>;

// A warp's ring of slots in shared memory and the walk over units of one (sequence, KV head) that fills it. Slot k takes the
// units first + k stride and the next one, below `end`. A unit in a slot: K's 1152 bytes, then V's; five cp.async of 16 bytes
// a lane (K's codes, V's codes, both parameter blocks by half a warp). Pages are looked up 32 units at a time, one batch
// ahead of use; a lane turns its entry into the unit's number in the cache.
struct Ring {
  uint32_t dst, slot, p_to;
  int lane;
  const uint8_t *k_src, *v_src, *p_src;      // this lane's 16 bytes of K's codes, V's codes and the parameters in unit 0
  const int* table;
  int first, stride, end, k, slots, upp, hkv, h;
  uint32_t units, units_next;
  uint64_t policy;                           // read once, codes and parameters leave L2 first: 256 sequences of 256-4096
                                             // tokens 129.3 -> 127.6 us, 141.3 -> 137.5 in an L2 full of written lines

  __device__ __forceinline__ void init(const Params& p, uint8_t* ring, int lane_) {
    lane = lane_;
    upp = p.block_size / kv4::kUnit;
    hkv = p.hkv;
    dst = smem_u32(ring) + lane * 16;
    p_to = kv4::kParBase + (lane < 8 ? 0 : kv4::kUnitBytes - 128);
    k_src = p.k_cache + lane * 16;
    v_src = p.v_cache + lane * 16;
    p_src = (lane < 8 ? k_src : v_src - 128) + kv4::kParBase;
    slot = 0;
    k = slots = 0;
    policy = l2_policy_evict_first();
  }
  // The walk, but for its end; sends for the first entries, which end() checks.
  __device__ __forceinline__ int begin(const Params& p, int b, int h_, int first_, int stride_) {
    h = h_;
    first = first_;
    stride = stride_;
    table = p.block_tables + static_cast<size_t>(b) * p.max_blocks;
    return entry(p, 0);
  }
  __device__ __forceinline__ int unit_of(int slot0) const { return first + (slot0 + (lane >> 1)) * stride + (lane & 1); }
  __device__ __forceinline__ int entry(const Params& p, int slot0) const {
    return __ldg(table + min(unit_of(slot0) / upp, p.max_blocks - 1));
  }
  __device__ __forceinline__ uint32_t number(const Params& p, int slot0, int blk) const {
    const int unit = unit_of(slot0);
    if (static_cast<unsigned>(blk) >= static_cast<unsigned>(p.num_blocks)) {
      if (unit < end) report_status(p.status, kIdDecode, kBadIndex);     // entries behind the sequence may be anything
      blk = 0;
    }
    return (static_cast<uint32_t>(blk) * hkv + h) * upp + unit % upp;
  }
  __device__ __forceinline__ void until(const Params& p, int end_, int entry0) {
    end = end_;
    k = 0;
    slots = first < end ? (end - first + stride - 1) / stride : 0;
    units = number(p, 0, entry0);
    if (slots > 16) units_next = number(p, 16, entry(p, 16));
  }
  // The next slot, if there is one; one commit group per call, empty ones included.
  __device__ __forceinline__ void issue(const Params& p) {
    if (k < slots) {
      const int unit0 = first + k * stride;
#pragma unroll
      for (int u = 0; u < kPair; ++u) {
        const uint64_t at = static_cast<uint64_t>(__shfl_sync(0xffffffffu, units, (2 * k + u) & 31)) * kv4::kUnitBytes;
        const uint32_t to = dst + slot * kSlot + u * kUnitSlot;
        if (unit0 + u < end) {
          cp_async16_u32(to, k_src + at, policy);
          cp_async16_u32(to + 512, k_src + at + 512, policy);
          cp_async16_u32(to + kv4::kUnitBytes, v_src + at, policy);
          cp_async16_u32(to + kv4::kUnitBytes + 512, v_src + at + 512, policy);
          if (lane < 16) cp_async16_u32(to + p_to, p_src + at, policy);
        }
      }
      if ((++k & 15) == 0) {
        units = units_next;
        if (k + 16 < slots) units_next = number(p, k + 16, entry(p, k + 16));
      }
    }
    cp_async_commit();
    slot = slot == kStages - 1 ? 0 : slot + 1;
  }
};
static_assert(kPair == 2, "a lookup of 32 lanes serves 16 slots");

// A cluster of CTAs, one per KV split, per (sequence, KV head). NT, TWIN: as in Query; W: warps.
template <int NT, int W, bool TWIN>
__global__ void __launch_bounds__(W * 32, NT == 1 ? 12 / W : 8 / W) kv4_decode_kernel(const Params p) {
  extern __shared__ __align__(128) uint8_t smem[];
  __shared__ float sm_m[W][8 * NT], sm_l[W][8 * NT];
  __shared__ float part_m[8 * NT], part_l[8 * NT];       // this CTA's result, read by the cluster (part_o: in the ring)
  grid_dep_launch();
  const int split = blockIdx.x, h = blockIdx.y, b = blockIdx.z;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int g = lane >> 2, t = lane & 3;
  const int G = p.hq / p.hkv;
  uint8_t* ring_mem = smem + warp * kStages * kSlot;
  grid_dep_wait();
  Query<NT, TWIN> q;
  q.fetch(p, static_cast<size_t>(b) * p.hq + h * G, G, g, t);      // first: everything else hangs on two more reads
  // Slots are dealt to the warps in turn: which pages a warp reads first does not hang on the length.
  const int first = (split * W + warp) * kPair, stride = p.splits * W * kPair;
  Ring ring;
  ring.init(p, ring_mem, lane);
  const int entry0 = ring.begin(p, b, h, first, stride);
  const int kv_len = kv_len_of(p, b);
  ring.until(p, (kv_len + 15) / 16, entry0);
#pragma unroll
  for (int i = 0; i < kStages - 1; ++i) ring.issue(p);
  q.convert(p, g, t);
  SoftmaxOf<NT, TWIN> st;
  st.clear();

  const int tok = token_of_row(g);
  const uint8_t* at = ring_mem;
  int mine = kv_len - first * 16;                        // tokens from the slot's first on
  for (; mine > 0; mine -= 16 * stride) {
    cp_async_wait<kStages - 2>();
    __syncwarp();                        // everyone's part of the slot has landed, and everyone has read the slot filled next
    ring.issue(p);
    st.add(q, at + tok * 64 + t * 16, at + kv4::kParBase + tok * 8, at + kv4::kUnitBytes + token_of_row(2 * t) * 64 + g * 8,
           at + kv4::kUnitBytes + token_of_row(2 * t + 1) * 64 + g * 8, mine, tok, t);
    at = at == ring_mem + (kStages - 1) * kSlot ? ring_mem : at + kSlot;
  }
  cp_async_wait<0>();

  // The warps meet in the (now idle) ring.
  st.finish(q);
  __syncthreads();
  float* sm_o = reinterpret_cast<float*>(smem);                    // [warp][8 NT][128]
  float* part_o = sm_o + W * 8 * NT * kD;                          // [8 NT][128]
  static_assert((W + 1) * 8 * NT * kD * 4 <= decode_smem(W));
  st.each(g, t, [&](int head, int channel, const float4& v, float m, float l) {
    if (head >= G) return;
    *reinterpret_cast<float4*>(&sm_o[(warp * 8 * NT + head) * kD + channel]) = v;
    if (channel == 0) {
      sm_m[warp][head] = m;
      sm_l[warp][head] = l;
    }
  });
  __syncthreads();
  // Four channels a thread. Sums stay unnormalised until the last join.
  for (int idx = threadIdx.x; idx < G * (kD / 4); idx += blockDim.x) {
    const int r = idx / (kD / 4), d = (idx % (kD / 4)) * 4;
    float M = kNoMax;
#pragma unroll
    for (int w = 0; w < W; ++w) M = fmaxf(M, sm_m[w][r]);
    float L = 0.f;
    float4 acc = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
    for (int w = 0; w < W; ++w) {
      const float f = exp2f(sm_m[w][r] - M);
      const float4 v = *reinterpret_cast<const float4*>(&sm_o[(w * 8 * NT + r) * kD + d]);
      L += sm_l[w][r] * f;
      acc.x += v.x * f; acc.y += v.y * f; acc.z += v.z * f; acc.w += v.w * f;
    }
    if (p.splits == 1) {
      store_out(p.out + (static_cast<size_t>(b) * p.hq + h * G + r) * kD + d, acc, L);
    } else {
      *reinterpret_cast<float4*>(part_o + r * kD + d) = acc;
      if (d == 0) {
        part_m[r] = M;
        part_l[r] = L;
      }
    }
  }
  if (p.splits == 1) return;
  // The cluster's CTAs hold one split each: every CTA joins a share of the (head, channel) outputs.
  cluster_sync_all();
  const uint32_t so = smem_u32(part_o), sm = smem_u32(part_m), sl = smem_u32(part_l);
  for (int idx = split * blockDim.x + threadIdx.x; idx < G * kD; idx += blockDim.x * p.splits) {
    const int r = idx / kD;
    float M = kNoMax;
    for (int c = 0; c < p.splits; ++c) M = fmaxf(M, ld_cluster_f32(map_to_cta(sm + r * 4, c)));
    float L = 0.f, acc = 0.f;
    for (int c = 0; c < p.splits; ++c) {
      const float f = exp2f(ld_cluster_f32(map_to_cta(sm + r * 4, c)) - M);
      L += ld_cluster_f32(map_to_cta(sl + r * 4, c)) * f;
      acc += ld_cluster_f32(map_to_cta(so + idx * 4, c)) * f;
    }
    p.out[(static_cast<size_t>(b) * p.hq + h * G) * kD + idx] = __float2bfloat16(L == 0.f ? 0.f : acc / L);
  }
  cluster_sync_all();                // nobody leaves while its shared memory is being read
}

// ---- even shares ----
// All units of the batch, in the order (sequence, KV head, unit), are dealt to the launch's warps in equal runs, so that
// ragged lengths leave no tail. A run crosses from one (sequence, head) pair to the next; a pair that lies in one run is
// finished there, the others leave one partial result per run for kv4_join_kernel. Runs and pairs are numbered in the
// same order, so the partial of (run w, pair x) has the slot w + x and a pair's slots are consecutive.
struct Shares {
  float* o;         // [slot][8 NT][128]
  float* ml;        // [slot][8 NT][2]: running maximum (log2 units), sum
  int* begin;       // [seq + 1]: units of one head before the sequence; then the units per run
};
constexpr int kShareWarps = 4, kMinRun = 4;

template <int NT, bool TWIN>
__global__ void __launch_bounds__(kShareWarps * 32, NT == 1 ? 3 : 2) kv4_share_kernel(const Params p, const Shares ws, int num_seqs) {
  extern __shared__ __align__(128) uint8_t smem[];
  constexpr int T = kShareWarps * 32;
  __shared__ int sums[T + 1];
  grid_dep_launch();
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int g = lane >> 2, t = lane & 3;
  const int G = p.hq / p.hkv;
  uint8_t* ring_mem = smem + warp * kStages * kSlot;
  grid_dep_wait();
  // Every CTA counts the units: a thread a run of sequences, then a scan over the threads.
  const int chunk = (num_seqs + T - 1) / T;
  const int c0 = min(static_cast<int>(threadIdx.x) * chunk, num_seqs), c1 = min(c0 + chunk, num_seqs);
  int mine_units = 0;
  for (int b = c0; b < c1; ++b) mine_units += (kv_len_of(p, b) + 15) / 16;
  int incl = mine_units;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const int v = __shfl_up_sync(0xffffffffu, incl, o);
    if (lane >= o) incl += v;
  }
  if (lane == 31) sums[warp] = incl;
  __syncthreads();
  int before = 0, total = 0;
#pragma unroll
  for (int w = 0; w < kShareWarps; ++w) {
    if (w < warp) before += sums[w];
    total += sums[w];
  }
  __syncthreads();
  sums[threadIdx.x + 1] = before + incl;
  if (threadIdx.x == 0) sums[0] = 0;
  const int runs = gridDim.x * kShareWarps;
  const int all = total * p.hkv;
  const int per = max((all + runs - 1) / runs, kMinRun);
  if (blockIdx.x == 0) {                       // for the joining kernel
    int at = before + incl - mine_units;
    for (int b = c0; b < c1; ++b) {
      ws.begin[b] = at;
      at += (kv_len_of(p, b) + 15) / 16;
    }
    if (threadIdx.x == 0) {
      ws.begin[num_seqs] = total;
      ws.begin[num_seqs + 1] = per;
    }
  }
  __syncthreads();
  const int run = blockIdx.x * kShareWarps + warp;
  const long long from = static_cast<long long>(run) * per;
  if (from >= all) return;
  int todo = min(per, all - static_cast<int>(from));      // units of this run still to be consumed

  // The sequence that holds the first one: the thread chunk by bisection, then one by one.
  int b, units, kv_len, h, first;
  {
    const int u = static_cast<int>(from / p.hkv);          // of one head
    int lo = 0, hi = T;
    while (hi - lo > 1) {
      const int mid = (lo + hi) >> 1;
      if (sums[mid] <= u) lo = mid; else hi = mid;
    }
    int at = sums[lo];
    b = lo * chunk;
    for (;; ++b) {
      kv_len = kv_len_of(p, b);
      units = (kv_len + 15) / 16;
      if (u < at + units) break;
      at += units;
    }
    const int rest = static_cast<int>(from - static_cast<long long>(at) * p.hkv);
    h = rest / units;
    first = rest - h * units;
  }

  Ring ring;
  ring.init(p, ring_mem, lane);
  const int tok = token_of_row(g);
  const uint8_t* at = ring_mem;
  // The fetching side runs kStages - 1 slots ahead and may already be in the next pair.
  int f_b = b, f_h = h, f_units = units, f_todo = todo;
  auto fetch_pair = [&](int start) {
    const int n = min(f_units - start, f_todo);
    f_todo -= n;
    const int entry0 = ring.begin(p, f_b, f_h, start, kPair);
    ring.until(p, start + n, entry0);
  };
  auto fetch = [&]() {
    if (ring.k == ring.slots && f_todo > 0) {
      if (++f_h == p.hkv) {
        f_h = 0;
        do f_units = (kv_len_of(p, ++f_b) + 15) / 16;
        while (f_units == 0);
      }
      fetch_pair(0);
    }
    ring.issue(p);
  };
  fetch_pair(first);
  ring.issue(p);
#pragma unroll
  for (int i = 1; i < kStages - 1; ++i) fetch();

  for (;;) {
    const int n = min(units - first, todo);
    Query<NT, TWIN> q;
    q.fetch(p, static_cast<size_t>(b) * p.hq + h * G, G, g, t);
    q.convert(p, g, t);
    SoftmaxOf<NT, TWIN> st;
    st.clear();
    int mine = min(kv_len - first * 16, n * 16);
    for (int i = 0; i < n; i += kPair, mine -= 16 * kPair) {
      cp_async_wait<kStages - 2>();
      __syncwarp();
      fetch();
      st.add(q, at + tok * 64 + t * 16, at + kv4::kParBase + tok * 8, at + kv4::kUnitBytes + token_of_row(2 * t) * 64 + g * 8,
             at + kv4::kUnitBytes + token_of_row(2 * t + 1) * 64 + g * 8, mine, tok, t);
      at = at == ring_mem + (kStages - 1) * kSlot ? ring_mem : at + kSlot;
    }
    st.finish(q);
    const bool whole = n == units;
    const int pair = b * p.hkv + h;
    const size_t slot = static_cast<size_t>(run) + pair;
    st.each(g, t, [&](int head, int channel, const float4& v, float m, float l) {
      if (head >= G) return;
      if (whole) {
        store_out(p.out + (static_cast<size_t>(pair) * G + head) * kD + channel, v, l);
      } else {
        *reinterpret_cast<float4*>(ws.o + (slot * 8 * NT + head) * kD + channel) = v;
        if (channel == 0) *reinterpret_cast<float2*>(ws.ml + (slot * 8 * NT + head) * 2) = make_float2(m, l);
      }
    });
    todo -= n;
    if (todo == 0) break;
    first = 0;
    if (++h == p.hkv) {
      h = 0;
      do {
        kv_len = kv_len_of(p, ++b);
        units = (kv_len + 15) / 16;
      } while (units == 0);
    }
  }
  cp_async_wait<0>();
}

// Joins the partial results of the pairs that several runs share, and clears the rows of empty sequences. R warps per
// (pair, query head) take the partials in turn, BATCH at a time (the kernel is a chain of L2 round trips); a lane holds
// four channels. A row's warps are one CTA; with one warp a row, four rows are.
template <int R, int BATCH>
__global__ void __launch_bounds__(R == 1 ? 128 : R * 32) kv4_join_kernel(const Params p, const Shares ws, int num_seqs, int rows) {
  grid_dep_launch();
  grid_dep_wait();
  __shared__ float4 sm_o[R][32];
  __shared__ float sm_m[R], sm_l[R];
  const int G = p.hq / p.hkv;
  const int warp = R == 1 ? 0 : threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int row = R == 1 ? blockIdx.x * 4 + (threadIdx.x >> 5) : blockIdx.x;      // sequence * hq + query head
  if (row >= num_seqs * p.hq) return;
  const int pair = row / G, head = row - pair * G;
  const int b = pair / p.hkv, h = pair - b * p.hkv;
  const int before = ws.begin[b], units = ws.begin[b + 1] - before, per = ws.begin[num_seqs + 1];
  __nv_bfloat16* dst = p.out + static_cast<size_t>(row) * kD + lane * 4;
  if (units == 0) {
    if (warp == 0) *reinterpret_cast<uint2*>(dst) = make_uint2(0u, 0u);
    return;
  }
  const long long from = static_cast<long long>(before) * p.hkv + static_cast<long long>(h) * units;
  const int run0 = static_cast<int>(from / per), run1 = static_cast<int>((from + units - 1) / per);
  if (run0 == run1) return;                    // written by its run
  float M = kNoMax, L = 0.f;
  float4 acc = make_float4(0.f, 0.f, 0.f, 0.f);
  for (int r = run0 + warp; r <= run1; r += BATCH * R) {
    float2 ml[BATCH];
    float4 v[BATCH];
    float mn = M;
#pragma unroll
    for (int i = 0; i < BATCH; ++i) {
      const bool there = r + i * R <= run1;
      const size_t slot = (static_cast<size_t>(r + i * R) + pair) * rows + head;
      ml[i] = there ? *reinterpret_cast<const float2*>(ws.ml + slot * 2) : make_float2(kNoMax, 0.f);
      v[i] = there ? *reinterpret_cast<const float4*>(ws.o + slot * kD + lane * 4) : make_float4(0.f, 0.f, 0.f, 0.f);
    }
#pragma unroll
    for (int i = 0; i < BATCH; ++i) mn = fmaxf(mn, ml[i].x);
    const float f0 = exp2f(M - mn);
    M = mn;
    L *= f0;
    acc.x *= f0; acc.y *= f0; acc.z *= f0; acc.w *= f0;
#pragma unroll
    for (int i = 0; i < BATCH; ++i) {
      const float f = exp2f(ml[i].x - mn);
      L += ml[i].y * f;
      acc.x += v[i].x * f; acc.y += v[i].y * f; acc.z += v[i].z * f; acc.w += v[i].w * f;
    }
  }
  if constexpr (R > 1) {
    sm_o[warp][lane] = acc;
    if (lane == 0) {
      sm_m[warp] = M;
      sm_l[warp] = L;
    }
    __syncthreads();
    if (warp != 0) return;
    M = kNoMax;
    L = 0.f;
    acc = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
    for (int w = 0; w < R; ++w) M = fmaxf(M, sm_m[w]);
#pragma unroll
    for (int w = 0; w < R; ++w) {
      const float f = exp2f(sm_m[w] - M);
      const float4 v = sm_o[w][lane];
      L += sm_l[w] * f;
      acc.x += v.x * f; acc.y += v.y * f; acc.z += v.z * f; acc.w += v.w * f;
    }
  }
  store_out(dst, acc, L);
}

int fill(Params& p, const void* q, const void* k_cache, const void* v_cache, const int* block_tables, const int* kv_lens,
         void* out, int hq, int hkv, int d, int block_size, int max_blocks, int num_blocks, float scale, int* status) {
  if (d != kD) return XV_ERR_UNSUPPORTED;
  if (hkv <= 0 || hq <= 0 || hq % hkv || block_size <= 0 || block_size % kv4::kUnit || max_blocks <= 0 || num_blocks <= 0)
    return XV_ERR_SHAPE;
  if ((reinterpret_cast<uintptr_t>(q) | reinterpret_cast<uintptr_t>(k_cache) | reinterpret_cast<uintptr_t>(v_cache) |
       reinterpret_cast<uintptr_t>(out)) & 15)
    return XV_ERR_ALIGN;
  p = Params{};
  p.q = static_cast<const __nv_bfloat16*>(q);
  p.k_cache = static_cast<const uint8_t*>(k_cache);
  p.v_cache = static_cast<const uint8_t*>(v_cache);
  p.block_tables = block_tables;
  p.kv_lens = kv_lens;
  p.out = static_cast<__nv_bfloat16*>(out);
  p.hq = hq; p.hkv = hkv; p.block_size = block_size; p.max_blocks = max_blocks; p.num_blocks = num_blocks;
  p.max_tokens = static_cast<int>(std::min(static_cast<long long>(max_blocks) * block_size, 0x7ffffff0ll));
  // The scale's sign is Q's, so the running maxima need not know it; a scale of 0 is a Q of 0.
  const double s = scale == 0.f ? 1.0 : std::abs(static_cast<double>(scale)) * kLog2e;
  p.scale = static_cast<float>(0.5 * std::frexp(s, &p.scale_exp));      // below 1: K's largest steps stay in fp32
  p.scale_exp += 1;
  p.sign = scale == 0.f ? 0.f : scale < 0.f ? -1.f : 1.f;
  p.status = status;
  return 0;
}

// Shared memory above 48 KiB is opted into once per device.
int allow_decode_kernels() {
  static std::atomic<bool> done[64];
  int dev = 0;
  if (cudaGetDevice(&dev) != cudaSuccess || dev < 0 || dev >= 64) return XV_ERR_LAUNCH;
  if (done[dev].load(std::memory_order_acquire)) return 0;
  const auto at = cudaFuncAttributeMaxDynamicSharedMemorySize;
  if (cudaFuncSetAttribute(kv4_decode_kernel<1, 4, true>, at, decode_smem(4)) != cudaSuccess ||
      cudaFuncSetAttribute(kv4_decode_kernel<1, 4, false>, at, decode_smem(4)) != cudaSuccess ||
      cudaFuncSetAttribute(kv4_decode_kernel<2, 4, false>, at, decode_smem(4)) != cudaSuccess ||
      cudaFuncSetAttribute(kv4_share_kernel<1, true>, at, decode_smem(kShareWarps)) != cudaSuccess ||
      cudaFuncSetAttribute(kv4_share_kernel<1, false>, at, decode_smem(kShareWarps)) != cudaSuccess ||
      cudaFuncSetAttribute(kv4_share_kernel<2, false>, at, decode_smem(kShareWarps)) != cudaSuccess)
    return XV_ERR_LAUNCH;
  done[dev].store(true, std::memory_order_release);
  return 0;
}
int share_ctas(int num_sms, int nt) { return num_sms * (nt == 1 ? 3 : 2); }

inline int launch_ok() { return cudaGetLastError() == cudaSuccess ? 0 : XV_ERR_LAUNCH; }

}  // namespace

extern "C" {

// How a decode launch divides its work, from launch-shape constants only (never from sequence lengths), so that a captured
// graph keeps its shape: 1, 2, 4 or 8 CTAs (one cluster) per (sequence, KV head) as long as they are one wave of three an
// SM and get 128 tokens each, or 0 for even shares. Device times, clusters of 1 / 2 / 4 / 8 against shares:
//   8 pairs of 2000 tokens 13.2 / 9.7 / 6.4 / 5.3 against 9.6 us, of 40960 228 / 118 / 62 / 33 against 19.7
//   72 pairs of up to 3001 18.7 / 13.2 / 10.7 / 13.1 against 15.8, 256 of up to 1280 11.4 / 15.0 / 17.0 / 29.9 against 14.8
// Two CTAs repay their join from about 1280 tokens on (8 pairs of 300 4.2 / 5.4 / 4.2, 128 of up to 1200 8.5 / 8.9).
// Shares pay where a CTA could get more than 2048 tokens (a tail that they do not have), until so many pairs wait for a place
// that the tail no longer counts: pairs of up to 4096, 320 of them 32.3 (one CTA each) against 27.5, 768 67.0 against
// 61.4, 1024 80.6 against 78.5, 1600 109.0 against 112.1, 2048 135.6 against 138.2.
int xv_kv4_decode_splits(int num_seqs, int hkv, int num_sms, int max_tokens_per_seq) {
  const long long pairs = static_cast<long long>(num_seqs) * hkv;
  int s = 1;
  while (s < 8 && pairs * 2 * s <= 3 * num_sms && max_tokens_per_seq / (2 * s) >= 128) s *= 2;
  if (s == 2 && max_tokens_per_seq < 1280) s = 1;
  return max_tokens_per_seq / s > 2048 && pairs < 4 * 3 * num_sms ? 0 : s;
}

long long xv_kv4_decode_workspace_bytes(int num_seqs, int hq, int hkv, int splits, int num_sms) {
  if (splits > 0) return 0;
  const int nt = hq / hkv > 8 ? 2 : 1;
  const long long slots = static_cast<long long>(share_ctas(num_sms, nt)) * kShareWarps + static_cast<long long>(num_seqs) * hkv;
  return slots * 8 * nt * (kD + 2) * 4 + (static_cast<long long>(num_seqs) + 2) * 4;
}

int xv_kv4_decode(const void* q, const void* k_cache, const void* v_cache, const int* block_tables, const int* kv_lens,
                  void* out, int num_seqs, int hq, int hkv, int d, int block_size, int max_blocks, int num_blocks,
                  float scale, int splits, int num_sms, void* workspace, long long workspace_bytes, int* status,
                  cudaStream_t stream) {
  if (num_seqs <= 0) return 0;
  Params p;
  if (int rc = fill(p, q, k_cache, v_cache, block_tables, kv_lens, out, hq, hkv, d, block_size, max_blocks, num_blocks,
                    scale, status))
    return rc;
  if (hq / hkv > 16 || hkv > 65535 || num_seqs > 65535 || splits < 0 || splits > 8) return XV_ERR_SHAPE;
  if (static_cast<long long>(num_blocks) * hkv * (block_size / kv4::kUnit) > 0xffffffffLL) return XV_ERR_SHAPE;     // units: 32-bit numbers
  if (int rc = allow_decode_kernels()) return rc;
  p.splits = splits;
  const int nt = hq / hkv > 8 ? 2 : 1;
  const bool twin = hq / hkv <= 4;             // half the columns would be idle
  if (splits > 0) {
    launch_pdl_cluster(twin ? kv4_decode_kernel<1, 4, true> : nt == 1 ? kv4_decode_kernel<1, 4, false> : kv4_decode_kernel<2, 4, false>, dim3(splits, hkv, num_seqs), dim3(4 * 32),
                       decode_smem(4), stream, splits, p);
    return launch_ok();
  }
  const long long units = static_cast<long long>(max_blocks) * (block_size / kv4::kUnit);
  if (units * num_seqs * hkv > 0x7fffffffLL || static_cast<long long>(num_seqs) * hq > 0x7fffffffLL) return XV_ERR_SHAPE;
  if (!workspace || workspace_bytes < xv_kv4_decode_workspace_bytes(num_seqs, hq, hkv, 0, num_sms)) return XV_ERR_WORKSPACE;
  if (reinterpret_cast<uintptr_t>(workspace) & 15) return XV_ERR_ALIGN;
  const int ctas = share_ctas(num_sms, nt);
  Shares ws;
  ws.o = static_cast<float*>(workspace);
  const size_t slots = static_cast<size_t>(ctas) * kShareWarps + static_cast<size_t>(num_seqs) * hkv;
  ws.ml = ws.o + slots * 8 * nt * kD;
  ws.begin = reinterpret_cast<int*>(ws.ml + slots * 8 * nt * 2);
  launch_pdl(twin ? kv4_share_kernel<1, true> : nt == 1 ? kv4_share_kernel<1, false> : kv4_share_kernel<2, false>, dim3(ctas), dim3(kShareWarps * 32), decode_smem(kShareWarps),
             stream, p, ws, num_seqs);
  if (int rc = launch_ok()) return rc;
  // Warps per row by the partials that a pair may have, its share of the runs. Both kernels with 16 / 4 / 1 warps a row:
  // 8 pairs (223 partials) 19.7 / 30.3 / 69.6 us, 32 (56) 27.3 / 29.7 / 40.6, 72 (25) 28.5 / 28.5 / 33.9, 160 (12)
  // 54.6 / 49.9 / 52.5, 256 (7) 54.1 / 47.5 / 48.2, 512 (4) 81.3 / 69.2 / 68.1, 2048 (1) 187.9 / 144.7 / 138.2.
  const int partials = ctas * kShareWarps / (num_seqs * hkv) + 1;
  const unsigned rows = static_cast<unsigned>(num_seqs) * hq;
  if (partials > 24) launch_pdl(kv4_join_kernel<16, 8>, dim3(rows), dim3(512), 0, stream, p, ws, num_seqs, 8 * nt);
  else if (partials > 4) launch_pdl(kv4_join_kernel<4, 4>, dim3(rows), dim3(128), 0, stream, p, ws, num_seqs, 8 * nt);
  else launch_pdl(kv4_join_kernel<1, 4>, dim3((rows + 3) / 4), dim3(128), 0, stream, p, ws, num_seqs, 8 * nt);
  return launch_ok();
}

}  // extern "C"
