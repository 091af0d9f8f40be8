// Paged causal attention of query chunks over a 4-bit KV cache (format: common/kv4.cuh) on the 5th-generation tensor
// cores. head_dim 128, page sizes that are multiples of 16, up to 16 query heads per KV head.
//
// The query heads of a KV group are packed into the rows of one tile: lane r of a unit is query row r / G, head r % G, so
// a CTA (two units, 256 lanes) reads and dequantises each K/V tile of 128 tokens once for the whole group. Warps:
//   0-3 / 4-7 - softmax of unit 0 / 1 (thread = lane): S row from tensor memory, causal mask, running maximum (lazy: the
//               output is rescaled in place only when it grows by more than 2^8), P back to tensor memory in fp16, where
//               the second MMA reads it as its A operand.
//   8-11      - dequantisers (thread = token of the tile): 64 bytes of codes and 8 of parameters of K and of V from global
//               memory, one tile ahead in registers, to fp16 rows in the 128-byte-swizzled shared-memory rings.
//   12, 13    - one MMA issuer thread per unit: O += P V as soon as P is written, then the next S = Q K^T.
//   14, 15    - fill up the warpgroup.
// Registers move from the issuers' and dequantisers' warpgroups to the softmax ones (setmaxnreg: 2 x 176 + 104 + 56 = 4 x 128).
//
// What bounds it: the chain of one unit, S -> softmax -> P -> O += P V -> next S, about 4100 cycles a tile of 128 tokens, of
// which 1590 are the exponentials (1024 of MUFU), 840 S's way through tensor memory and the maximum, 1030 the two MMAs and
// the rest hand-over; the other unit's exponentials lie in between. Both units' MMAs are 2050 of it. Beside them the
// dequantisers' loop takes as long when all SMs are busy. (Stamps of an earlier step, 261 us; powers for every row, and for
// tokens where they are far apart, took it to 271.) 4 x 2048 rows behind 512 tokens, 32 query heads: 280 us in a stream, 271 in
// a graph, 737 and 760 TFLOP/s; 737 us if every tile is one whose tokens have powers of their own. On the way: Q loaded by the
// lanes that convert it 285; then, at 273 with these registers, 277 with 2 x 184 + 96 + 48, 286 with 2 x 192 + 80 + 48, 287
// with 2 x 168 + 112 + 64.
//
// fp16 operands, not bf16: a dequantised value c + s (n - 8) has more than bf16's 8 bits, and its rounding (2^-12 instead
// of 2^-9) would otherwise be the largest error of the result. Their range is kept by powers of two: a row of Q is scaled
// by its largest element, a tile of K or V by an exponent that its dequantisers choose from the tile's parameters (and
// keep while it fits); the scores undo Q's and K's, and V's is carried with the output accumulator, row by row. In a tile
// with tokens 2^12 (to 2^20) below its largest every token has its own exponent, so that a large one that a row does not see, or
// gives no weight, costs the row nothing of the others; softmax takes such tiles by a slower way of its own.
// Inside a word the channels are stored in the order 0 4 1 5 2 6 3 7, which is how the nibbles unpack: Q follows it, and
// the output undoes it for V.
//
// Rows that do not see a token never meet its values: its score is replaced by -inf, P is 0 there, and a group of V whose
// parameters are not finite is stored as 0. The first token of each group that had such is kept; the rows that see it
// become NaN in that group's channels at the end.
// Every wait is bounded; one that runs out records a status code, the CTA stops issuing work, frees its tensor memory and
// returns.

#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_runtime.h>
#include <math_constants.h>

#include <algorithm>
#include <atomic>
#include <climits>
#include <cmath>
#include <cstdint>

#include "../common/kv4.cuh"
#include "../common/launch.cuh"
#include "../common/ptx.cuh"
#include "xv_cuda.h"

namespace {

using namespace xv;

constexpr int kD = kv4::kD;
constexpr int kBM = 128, kBN = 128;               // lanes of a unit, tokens of a tile
constexpr int kHalf = kBN * 128;                  // bytes of 64 channels of a tile
constexpr int kTileBytes = 2 * kHalf;             // 32 KiB
constexpr int kNK = 3, kNV = 2;                   // ring slots
constexpr int kBarBytes = 512;                    // barriers and small arrays
constexpr int kPowerBytes = 4 * 2 * kBN;          // [4 tiles][K, V][token]: powers of tokens
constexpr int kSmem = (2 + kNK + kNV) * kTileBytes + 1024 + kBarBytes + kPowerBytes;
constexpr uint32_t kTmemCols = 512, kTmemUnit = 256, kTmemO = 128;       // all of it, so it begins at address 0
constexpr int kId = 12;
constexpr double kLog2e = 1.4426950408889634;
constexpr float kLazy = 8.f;                      // log2 units
constexpr float kNoMax = -3.0e38f;

struct Params {
  const __nv_bfloat16* q;
  const uint8_t* k_cache;
  const uint8_t* v_cache;
  const int* block_tables;
  const int* cu_q;
  const int* kv_lens;
  __nv_bfloat16* out;
  int* status;
  float* ws_o;                                    // [CTA][split][256 lanes][128] unnormalised outputs, when splits > 1
  float* ws_ml;                                   // [CTA][split][256 lanes][2]: maximum (log2 units), sum
  int seq_begin, num_seqs, max_q_len, clear_to, hq, hkv, block_size, max_blocks, num_blocks, total_rows, splits;
  float scale, sign;                              // of a score, times log2 e: sign * scale * 2^scale_exp, scale in 1 .. 2
  int scale_exp;
  int G, rpu, by_g;                               // heads to a KV head, rows of a unit; 65536 / G + 1: lane / G is a product
  uint32_t inv_splits;                            // 2^32 / splits + 1, or 0 for one split
  // n / splits; exact for n splits < 2^32.
  __device__ __forceinline__ int by_splits(int n) const { return inv_splits ? __umulhi(n, inv_splits) : n; }
};

// Whether a chunk's rows are rows of Q behind the decode rows, and no more than the launch has CTAs for.
__device__ __forceinline__ bool rows_fine(const Params& p, int q_begin, int q_end) {
  return q_begin >= p.seq_begin && q_end >= q_begin && q_end <= p.total_rows && q_end - q_begin <= p.max_q_len;
}
// Clears 16-byte pieces of output rows: `pieces` from piece `at` on of each row in [from, to), by `workers` threads.
__device__ __forceinline__ void clear_rows(const Params& p, int from, int to, int at, int pieces, size_t worker, size_t workers) {
  const size_t row = static_cast<size_t>(p.hq) * (kD / 8), all = from < to ? static_cast<size_t>(to - from) * pieces : 0;
  for (size_t i = worker; i < all; i += workers)
    reinterpret_cast<uint4*>(p.out)[(from + i / pieces) * row + at + i % pieces] = make_uint4(0u, 0u, 0u, 0u);
}

struct alignas(16) TileScale {                    // of one tile: K and V are stored divided by 2^k and 2^v
  int k, v, own, unused;                          // own: each token has its own k and v
};

__device__ __forceinline__ uint32_t pack_f16(float lo, float hi) {
  const __half2 v = __floats2half2_rn(lo, hi);
  return *reinterpret_cast<const uint32_t*>(&v);
}
__device__ __forceinline__ uint64_t add_f32x2(uint64_t a, uint64_t b) {
  uint64_t d;
  asm("add.rn.f32x2 %0, %1, %2;" : "=l"(d) : "l"(a), "l"(b));
  return d;
}
__device__ __forceinline__ float pow2(int e) { return __int_as_float((127 + e) << 23); }
__device__ __forceinline__ uint32_t idesc_f16(int m, int n) {
  return (1u << 4) | static_cast<uint32_t>(n >> 3) << 17 | static_cast<uint32_t>(m >> 4) << 24;
}
template <int N>
__device__ __forceinline__ void set_regs_up() { asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(N)); }
template <int N>
__device__ __forceinline__ void set_regs_down() { asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(N)); }

// Address of 16-byte chunk c (0..15: one word of channels) of a row: `row_at` is the row's start with its swizzle (row & 7)
// in the chunk bits.
__device__ __forceinline__ uint32_t row_start(uint32_t tile, int row) {
  return tile + static_cast<uint32_t>(row * 128 + ((row & 7) << 4));
}
__device__ __forceinline__ uint32_t chunk_at(uint32_t row_at, int c) {
  return (row_at ^ static_cast<uint32_t>((c & 7) << 4)) + (c >> 3) * kHalf;
}
__device__ __forceinline__ void st_shared_v4(uint32_t addr, uint32_t a, uint32_t b, uint32_t c, uint32_t d) {
  asm volatile("st.shared.v4.b32 [%0], {%1, %2, %3, %4};" ::"r"(addr), "r"(a), "r"(b), "r"(c), "r"(d) : "memory");
}

__device__ __forceinline__ uint4 ld_shared_v4(uint32_t addr) {
  uint4 v;
  asm volatile("ld.shared.v4.b32 {%0, %1, %2, %3}, [%4];" : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w) : "r"(addr) : "memory");
  return v;
}
// A contiguous run of bytes (a multiple of 16) from global to this CTA's shared memory, counted in bytes on `bar`.
__device__ __forceinline__ void bulk_load(void* dst, const void* src, uint32_t bytes, uint64_t* bar) {
  asm volatile("cp.async.bulk.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1], %2, [%3];" ::"r"(smem_u32(dst)),
               "l"(src), "r"(bytes), "r"(smem_u32(bar))
               : "memory");
}

// Two channels of a word, nibbles j and j + 4, as n - 8 in fp16 (exact): even j as 1024 + n, odd j as 1024 + 16 n.
__device__ __forceinline__ __half2 centred_f16(uint32_t w, bool odd) {
  uint32_t r;
  if (odd) {
    asm("lop3.b32 %0, %1, %2, %3, 0xEA;" : "=r"(r) : "r"(w), "r"(0x00f000f0u), "r"(0x64006400u));
    return __hfma2(*reinterpret_cast<const __half2*>(&r), __floats2half2_rn(0.0625f, 0.0625f), __floats2half2_rn(-72.f, -72.f));
  }
  asm("lop3.b32 %0, %1, %2, %3, 0xEA;" : "=r"(r) : "r"(w), "r"(0x000f000fu), "r"(0x64006400u));
  return __hsub2(*reinterpret_cast<const __half2*>(&r), __floats2half2_rn(1032.f, 1032.f));
}

// a b and a b + c where a or c may be subnormal, which the library's fast-math flags take for 0: the centre of a group that
// is small throughout (its step is never subnormal).
__device__ __forceinline__ float mul_whole(float a, float b) {
  float d;
  asm("mul.rn.f32 %0, %1, %2;" : "=f"(d) : "f"(a), "f"(b));
  return d;
}
__device__ __forceinline__ float fma_whole(float a, float b, float c) {
  float d;
  asm("fma.rn.f32 %0, %1, %2, %3;" : "=f"(d) : "f"(a), "f"(b), "f"(c));
  return d;
}

// A group's parameters as fp16 pairs, the tile's power of two taken out.
struct Pair {
  __half2 s, c;
  __device__ __forceinline__ Pair(uint32_t w, float f)
      : s(__float2half2_rn(kv4::par_s(w) * f)), c(__float2half2_rn(mul_whole(kv4::par_c(w), f))) {}
};

// 16 of a row's 64 code bytes as fp16 c + s (n - 8) into chunks c0 .. c0 + 3: words of even index belong to group 0.
__device__ __forceinline__ void put_words(uint32_t row_at, int c0, const uint4& codes, const Pair& g0, const Pair& g1) {
  const uint32_t w[4] = {codes.x, codes.y, codes.z, codes.w};
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const Pair& g = (i & 1) ? g1 : g0;
    const uint32_t hi = w[i] >> 8;
    uint32_t v[4];
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const __half2 x = __hfma2(centred_f16(j < 2 ? w[i] : hi, j & 1), g.s, g.c);
      v[j] = *reinterpret_cast<const uint32_t*>(&x);
    }
    st_shared_v4(chunk_at(row_at, c0 + i), v[0], v[1], v[2], v[3]);
  }
}

// What a lane of the softmax keeps of its row between tiles.
struct RowState {
  float m, l;                                     // running maximum in log2 units (it may lag), sum of P
  // S scale - m leaves what rounding took from m, 2^-24 of it: of scores of 2^30 more than an exponential may see. Rows whose
  // maximum is beyond 2^24 leave the scale's mantissa out, so that the product with a power of two is exact. Their weights
  // are those of the largest score and of its equals, whatever the mantissa: others as near are within S's own rounding.
  float mantissa;
  // O is in units of 2^unit_v, the current tile's power, but within 2^60 of 2^most_v: no change of units takes it out of fp32.
  // 2^most_v is the largest that a tile's weights and V may have added (|O| < 2^54 2^most_v: 2^31 tokens, P up to 2^8, V up to
  // 2^15). P of a tile in other units than the row's is scaled; next to what O holds, or it itself, that tile is nothing.
  float most_v;
  int unit_v;

  static __device__ __forceinline__ bool is_huge(float x) { return fabsf(x) > 16777216.f && x != kNoMax; }
  // To a new maximum; returns the exponent (0 or below) of what all sums are to be multiplied by.
  __device__ __forceinline__ float raise(const Params& p, float top, float unit, float m_new) {
    const float want = is_huge(m_new) ? 1.f : p.scale;
    if (want != mantissa) {
      m *= want / mantissa;
      mantissa = want;
      m_new = fmaxf(m, top * (mantissa * unit));
    }
    const float grown = m - m_new;
    l *= exp2f(grown);
    m = m_new;
    return grown;
  }
  // To a tile of V in units of 2^tile_v with weights of at most 2^weight; returns what O is to be multiplied by.
  __device__ __forceinline__ float turn(float grown, int tile_v, float weight) {
    most_v = fmaxf(fmaxf(most_v + grown, static_cast<float>(tile_v) + fminf(weight, 0.f)), -200.f);
    const int mid = static_cast<int>(most_v), to = max(mid - 60, min(mid + 60, tile_v));
    const float alpha = exp2f(grown + static_cast<float>(unit_v - to));
    unit_v = to;
    return alpha;
  }
};

__device__ __forceinline__ void rescale(uint32_t taddr, float alpha) {
  const uint64_t alpha2 = pack_f32x2(alpha, alpha);
#pragma unroll 1
  for (int ch = 0; ch < kD / 16; ++ch) {
    uint32_t o[16];
    tmem_ld16(taddr + kTmemO + ch * 16, o);
    tmem_ld_wait();
#pragma unroll
    for (int i = 0; i < 16; i += 2) {
      float lo, hi;
      unpack_f32x2(mul_f32x2(pack_f32x2(__uint_as_float(o[i]), __uint_as_float(o[i + 1])), alpha2), lo, hi);
      o[i] = __float_as_uint(lo);
      o[i + 1] = __float_as_uint(hi);
    }
    tmem_st16(taddr + kTmemO + ch * 16, o);
  }
  tmem_st_wait();
}

// The softmax of a tile whose tokens have powers of their own (own: K's, then V's), of which the row sees the first `seen`: three
// walks over S, 32 columns at a time: the maximum; the largest of weight times V's power, which is the row's unit; P, each
// token's scaled to that unit. False: a wait ran out.
__device__ __forceinline__ bool apart_tile(const Params& p, RowState& st, const int8_t* own, int seen,
                                           int row_exp, uint32_t taddr, int u, int j, uint64_t* o_done, uint64_t* xu_done,
                                           uint64_t* p_ready) {
  uint32_t x[32];
  auto load = [&](int c) {                        // scores in log2 units but for the scale's mantissa
    tmem_ld32(taddr + c * 32, x);
    tmem_ld_wait();
    tmem_ld_fence_regs(x);
#pragma unroll
    for (int i = 0; i < 32; ++i) {
      const float unit = pow2(max(-126, min(126, row_exp + own[c * 32 + i])));
      x[i] = c * 32 + i < seen ? __float_as_uint(__uint_as_float(x[i]) * unit) : 0xff800000u;
    }
  };
  float top = __uint_as_float(0xff800000u);
#pragma unroll 1
  for (int c = 0; c < 4; ++c) {
    load(c);
#pragma unroll
    for (int i = 0; i < 32; ++i) top = fmaxf(top, __uint_as_float(x[i]));
  }
  if (j > 0) {
    if (!__all_sync(0xffffffffu, mbar_wait(&o_done[u], (j - 1) & 1))) return false;
    tc_fence_after_sync();
  }
  const float grown = st.raise(p, top, 1.f, fmaxf(st.m, top * st.mantissa)), scale = st.mantissa;
  float most = -120.f;
#pragma unroll 1
  for (int c = 0; c < 4; ++c) {
    load(c);
#pragma unroll
    for (int i = 0; i < 32; ++i)
      most = fmaxf(most, fmaf(__uint_as_float(x[i]), scale, -st.m) + static_cast<float>(own[kBN + c * 32 + i]));
  }
  const float alpha = st.turn(grown, static_cast<int>(ceilf(fminf(most, 120.f))), 0.f);
  if (j > 0) rescale(taddr, alpha);
  if ((u == 1 || j > 0) && !__all_sync(0xffffffffu, u == 1 ? mbar_wait(&xu_done[0], j & 1) : mbar_wait(&xu_done[1], (j - 1) & 1)))
    return false;
#pragma unroll 1
  for (int c = 0; c < 4; ++c) {
    load(c);
    uint32_t packed[16];
#pragma unroll
    for (int i = 0; i < 32; i += 2) {
      float of[2];
#pragma unroll
      for (int k = 0; k < 2; ++k) {
        const float y = fmaf(__uint_as_float(x[i + k]), scale, -st.m);
        st.l += exp2f(y);
        of[k] = exp2f(y + static_cast<float>(own[kBN + c * 32 + i + k] - st.unit_v));
      }
      packed[i >> 1] = pack_f16(of[0], of[1]);
    }
    tmem_st16(taddr + c * 16, packed);            // over scores that have been read
  }
  mbar_arrive(&xu_done[u]);
  tmem_st_wait();
  tc_fence_before_sync();
  mbar_arrive(&p_ready[u]);
  return true;
}

__global__ void __launch_bounds__(512, 1) kv4_prefill_tc_kernel(const Params p) {
  extern __shared__ __align__(1024) uint8_t smem_raw[];
  const uint32_t pad = (1024u - (smem_u32(smem_raw) & 1023u)) & 1023u;
  uint8_t* smem = smem_raw + pad;
  uint8_t* q_s = smem;                                       // [2 units]
  uint8_t* k_ring = q_s + 2 * kTileBytes;
  uint8_t* v_ring = k_ring + kNK * kTileBytes;
  uint64_t* bars = reinterpret_cast<uint64_t*>(v_ring + kNV * kTileBytes);
  uint64_t* q_full = bars;                                   // [2]
  uint64_t* k_full = q_full + 2;                             // [kNK]
  uint64_t* v_full = k_full + kNK;
  uint64_t* k_empty = v_full + kNV;
  uint64_t* v_empty = k_empty + kNK;
  uint64_t* s_full = v_empty + kNV;                          // [2] S written by the MMA
  uint64_t* p_ready = s_full + 2;                            // [2] P written (and O rescaled)
  uint64_t* o_done = p_ready + 2;                            // [2]
  uint64_t* xu_done = o_done + 2;                            // [2] a unit's exponentials of the tile are over
  uint64_t* q_raw = xu_done + 2;                             // [2] a unit's rows as they are in memory
  TileScale* scales = reinterpret_cast<TileScale*>(q_raw + 2);           // [8], by tile
  uint32_t* red = reinterpret_cast<uint32_t*>(scales + 8);   // [2][12]
  int* first_bad = reinterpret_cast<int*>(red + 24);         // [2 groups of V]: the first token whose values are not finite
  uint32_t* tmem_slot = red + 26;
  volatile int* again = reinterpret_cast<volatile int*>(red + 28);       // [4 warps]
  int8_t* powers = reinterpret_cast<int8_t*>(bars) + kBarBytes;          // slot: tile & 3; no tile is more than three ahead
  volatile int* abort_flag = reinterpret_cast<volatile int*>(tmem_slot + 1);
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int wg = warp >> 2;

  // Before the wait for the launch before: the barriers, under what is left of launch latency (the trigger that would let blocks
  // start earlier is compiled out, ptx.cuh). Tensor memory comes after it: that launch may want all of it.
  grid_dep_launch();
  if (threadIdx.x == 0) {
    for (int u = 0; u < 2; ++u) {
      mbar_init(&q_full[u], 128);
      mbar_init(&s_full[u], 1);
      mbar_init(&p_ready[u], 128);
      mbar_init(&o_done[u], 1);
      mbar_init(&xu_done[u], 128);
      mbar_init(&q_raw[u], 1);
    }
    for (int s = 0; s < kNK; ++s) {
      mbar_init(&k_full[s], 128);
      mbar_init(&k_empty[s], 2);
    }
    for (int s = 0; s < kNV; ++s) {
      mbar_init(&v_full[s], 128);
      mbar_init(&v_empty[s], 2);
    }
    *abort_flag = 0;
    first_bad[0] = first_bad[1] = INT_MAX;
    mbar_fence_init();
  }
  __syncthreads();
  grid_dep_wait();

  const int z = p.by_splits(blockIdx.z), split = blockIdx.z - z * p.splits, b = p.seq_begin + z, hk = blockIdx.y;
  const int q_begin = p.cu_q[b], q_end = p.cu_q[b + 1];
  int kv_len = max(p.kv_lens[b], 0);
  {                                                          // rows of no chunk: behind the last, by all; before the first
    const int last = p.seq_begin + p.num_seqs, from = max(max(p.cu_q[last - 1], p.cu_q[last]), p.seq_begin);
    const size_t block = (static_cast<size_t>(blockIdx.z) * gridDim.y + blockIdx.y) * gridDim.x + blockIdx.x;
    if (from < p.clear_to)
      clear_rows(p, from, p.clear_to, 0, p.hq * (kD / 8), block * blockDim.x + threadIdx.x,
                 static_cast<size_t>(gridDim.x) * gridDim.y * gridDim.z * blockDim.x);
    if (blockIdx.x == 0 && blockIdx.y == 0 && blockIdx.z == 0)
      clear_rows(p, p.seq_begin, min(q_begin, p.total_rows), 0, p.hq * (kD / 8), threadIdx.x, blockDim.x);
  }
  const int q_len = q_end - q_begin;
  if (!rows_fine(p, q_begin, q_end)) {
    if (threadIdx.x == 0) report_status(p.status, kId, kBadIndex);
    const int pieces = p.G * (kD / 8);
    if (split == 0)
      clear_rows(p, max(q_begin, p.seq_begin), min(q_end, p.total_rows), hk * pieces, pieces,
                 blockIdx.x * blockDim.x + threadIdx.x, gridDim.x * blockDim.x);
    return;
  }
  const int G = p.G, rpu = p.rpu;                            // heads of a KV head; query rows of a unit
  const int row0 = (static_cast<int>(gridDim.x) - 1 - static_cast<int>(blockIdx.x)) * 2 * rpu;     // long ones first
  if (row0 >= q_len) return;
  const long long most = min(static_cast<long long>(p.max_blocks) * p.block_size, 0x7fffff00ll);   // a tile more stays 32-bit
  if (kv_len > most) {
    if (threadIdx.x == 0) report_status(p.status, kId, kBadIndex);
    kv_len = static_cast<int>(most);
  }
  const int pos0 = kv_len - q_len;                           // position of query row 0; rows before position 0 see nothing
  const int rows_here = min(2 * rpu, q_len - row0);
  const int n_kv = max(0, min(kv_len, pos0 + row0 + rows_here));
  // This CTA's run of tiles.
  const int all_tiles = (n_kv + kBN - 1) / kBN, per_split = p.by_splits(all_tiles + p.splits - 1);
  const int tile0 = min(split * per_split, all_tiles), n_tiles = min(per_split, all_tiles - tile0);
  auto rows_of = [&](int u) { return max(0, min(rpu, q_len - row0 - u * rpu)); };

  if (wg == 2) {
    // ---------------- dequantisers ----------------
    set_regs_down<104>();
    const int row = threadIdx.x & 127;
    const int upp = p.block_size / kv4::kUnit;
    const int* table = p.block_tables + static_cast<size_t>(b) * p.max_blocks;
    // This thread's row, tile by tile: page and place in it follow from the tile before. Pages past the last one are
    // replaced by it; whatever row that reads does not count. A page's number is read two tiles ahead of its bytes' use.
    const int last_page = (max(n_kv, 1) - 1) / p.block_size;
    const int page_step = kBN / p.block_size, place_step = kBN % p.block_size;
    int page = (tile0 * kBN + row) / p.block_size, place = tile0 * kBN + row - page * p.block_size, place_next = 0, entry = 0;
    auto look = [&]() { entry = __ldg(table + min(page, last_page)); place_next = place; };
    auto step = [&]() {
      page += page_step;
      place += place_step;
      if (place >= p.block_size) {
        place -= p.block_size;
        ++page;
      }
    };
    const uint8_t *code = nullptr, *par = nullptr;           // in K's cache; V's is v_off further
    const ptrdiff_t v_off = p.v_cache - p.k_cache;
    auto resolve = [&]() {                                   // addresses from the entry that look() read
      if (static_cast<unsigned>(entry) >= static_cast<unsigned>(p.num_blocks)) {
        report_status(p.status, kId, kBadIndex);
        entry = 0;
      }
      const size_t unit = ((static_cast<size_t>(entry) * p.hkv + hk) * upp + (place_next >> 4)) * kv4::kUnitBytes;
      code = p.k_cache + unit + (place_next & 15) * kv4::kCodeRow;
      par = p.k_cache + unit + kv4::kParBase + (place_next & 15) * kv4::kParRow;
    };
    auto load_codes = [&](uint4 (&c)[4], const uint8_t* at) {
#pragma unroll
      for (int i = 0; i < 4; ++i) c[i] = __ldg(reinterpret_cast<const uint4*>(at) + i);
    };
    uint4 kc[4], vc[4];
    uint2 kp, vp, kp_next = make_uint2(0u, 0u), vp_next = make_uint2(0u, 0u);
    auto finite = [](uint32_t w) { return (w & 0x7f80u) != 0x7f80u && (w & 0x7f800000u) != 0x7f800000u; };
    // Largest possible magnitude of a token's values; 0 for K that is not finite.
    auto bound = [](uint2 w) {
      return max(__float_as_uint(fma_whole(8.f, kv4::par_s(w.x & 0x7fffu), kv4::par_c(w.x & 0x7fff0000u))),
                 __float_as_uint(fma_whole(8.f, kv4::par_s(w.y & 0x7fffu), kv4::par_c(w.y & 0x7fff0000u))));
    };
    auto bound_k = [&](uint2 w) { return finite(w.x) && finite(w.y) ? bound(w) : 0u; };
    // A token below 2^-5 in the tile's units (and not 0): its smaller channels would lose bits to fp16's subnormals, and P of
    // large tokens that it leaves little of to their own. `least`: that as a float's bits.
    auto least_of = [](int e) { return static_cast<uint32_t>(max(e + 127 - 5, 0)) << 23; };
    auto small = [](uint32_t bits, uint32_t least) { return bits - 1u < least; };
    int ek = -10, ev = -10;                                  // what magnitudes of 2 to 8 would choose
    uint32_t least_k = least_of(ek), least_v = least_k;
    // What counts of tile j's parameters (values of V that are not finite are noted and count as 0), and the tile's largest
    // possible magnitudes, left in `red` for everyone.
    auto admit = [&](int j, bool ok) {
      if ((tile0 + j) * kBN + row >= n_kv) kp = vp = make_uint2(0u, 0u);
      if (!finite(vp.x)) {
        atomicMin(first_bad, (tile0 + j) * kBN + row);
        vp.x = 0u;
      }
      if (!finite(vp.y)) {
        atomicMin(first_bad + 1, (tile0 + j) * kBN + row);
        vp.y = 0u;
      }
      const uint32_t kb = bound_k(kp), vb = bound(vp);
      const uint32_t kw = __reduce_max_sync(0xffffffffu, kb), vw = __reduce_max_sync(0xffffffffu, vb);
      const bool far = __any_sync(0xffffffffu, small(kb, least_k) || small(vb, least_v));
      if (lane == 0) {
        uint32_t* at = red + (j & 1) * 12 + (warp & 3);
        at[0] = kw;
        at[4] = vw;
        at[8] = (ok ? 0u : 1u) | (far ? 2u : 0u);
      }
    };
    // Largest magnitude of a stored tile: 2^12 .. 2^13 when an exponent is chosen (where tokens are below 2^-5, each
    // has its own), kept while it stays in 2^7 .. 2^15.
    auto choose = [](int e, uint32_t bits) {
      const int top = static_cast<int>(bits >> 23) - 127;
      if (bits != 0 && (top - e > 14 || top - e < 7)) e = top - 12;
      return max(-120, min(120, e));
    };
    auto own_power = [](uint32_t bits, int none) { return bits == 0u ? none : max(-120, static_cast<int>(bits >> 23) - 127 - 12); };
    // A wait that runs out is only noted: the four warps leave together, at the barrier of the next tile.
    bool ok = true;
    if (n_tiles > 0) {
      look();
      resolve();
      kp = __ldg(reinterpret_cast<const uint2*>(par));
      vp = __ldg(reinterpret_cast<const uint2*>(par + v_off));
      load_codes(kc, code);
      load_codes(vc, code + v_off);
      step();
      look();
      admit(0, true);
    }
    for (int j = 0; j < n_tiles; ++j) {
      named_barrier(1, 128);
      const uint4* seen = reinterpret_cast<const uint4*>(red + (j & 1) * 12);       // of the four warps: K, V, gave up
      const uint4 k4 = seen[0], v4 = seen[1], out = seen[2];
      const uint32_t flags = out.x | out.y | out.z | out.w;
      if (flags & 1u) break;
      bool own = flags & 2u;
      const int ek_new = choose(ek, max(max(k4.x, k4.y), max(k4.z, k4.w)));
      const int ev_new = choose(ev, max(max(v4.x, v4.y), max(v4.z, v4.w)));
      if (ek_new != ek || ev_new != ev) {                    // alike in the four warps: look again, in the new units
        ek = ek_new;
        ev = ev_new;
        least_k = least_of(ek);
        least_v = least_of(ev);
        const bool far = __any_sync(0xffffffffu, small(bound_k(kp), least_k) || small(bound(vp), least_v));
        if (lane == 0) again[warp & 3] = far;
        named_barrier(1, 128);
        own = again[0] | again[1] | again[2] | again[3];
      }
      if (row == 0) {
        TileScale sc;
        sc.k = ek;
        sc.v = ev;
        sc.own = own;
        sc.unused = 0;
        scales[j & 7] = sc;
      }
      const bool more = j + 1 < n_tiles;
      if (more) {                                            // the next tile's parameters now, its codes as registers become free
        resolve();
        kp_next = __ldg(reinterpret_cast<const uint2*>(par));
        vp_next = __ldg(reinterpret_cast<const uint2*>(par + v_off));
        step();
        look();
      }
      const int ks = j % kNK, vs = j % kNV;
      const uint2 vp_now = vp;
      int token_k = ek, token_v = ev;
      if (own) {                                             // here: both before S can be ready
        token_k = own_power(bound_k(kp), ek);
        token_v = own_power(bound(vp), -120);
        powers[(j & 3) * 2 * kBN + row] = static_cast<int8_t>(token_k);
        powers[(j & 3) * 2 * kBN + kBN + row] = static_cast<int8_t>(token_v);
      }
      if (j == 1 || j == 2) ok = ok && __all_sync(0xffffffffu, mbar_wait(&q_full[j - 1], 0));    // Q's rows lie in these slots
      ok = ok && __all_sync(0xffffffffu, mbar_wait(&k_empty[ks], ((j / kNK) & 1) ^ 1) && *abort_flag == 0);
      if (ok) {
        const float f = pow2(-token_k);
        const Pair g0(kp.x, f), g1(kp.y, f);
        const uint32_t at = row_start(smem_u32(k_ring) + ks * kTileBytes, row);
#pragma unroll
        for (int i = 0; i < 4; ++i) put_words(at, 4 * i, kc[i], g0, g1);
        fence_proxy_async_smem();
        mbar_arrive(&k_full[ks]);
      }
      if (more) {                                            // here, so that its reductions end under V's conversion
        load_codes(kc, code);
        kp = kp_next;
        vp = vp_next;
        admit(j + 1, ok);
      }
      ok = ok && __all_sync(0xffffffffu, mbar_wait(&v_empty[vs], ((j / kNV) & 1) ^ 1) && *abort_flag == 0);
      if (ok) {
        const float f = pow2(-token_v);
        const Pair g0(vp_now.x, f), g1(vp_now.y, f);
        const uint32_t at = row_start(smem_u32(v_ring) + vs * kTileBytes, row);
#pragma unroll
        for (int i = 0; i < 4; ++i) put_words(at, 4 * i, vc[i], g0, g1);
        fence_proxy_async_smem();
        mbar_arrive(&v_full[vs]);
      }
      if (more) load_codes(vc, code + v_off);
    }
    if (!ok && lane == 0) {
      report_status(p.status, kId, kWaitEmptyTimeout);
      *abort_flag = 1;
    }
  } else if (wg == 3) {
    // ---------------- MMA issuers: one warp per unit, one elected lane issues ----------------
    // The whole warp walks the loop, so that descriptors stay in uniform registers: a lone lane took about 120 cycles an
    // MMA, twice what the MMA itself takes.
    set_regs_down<56>();
    const int role = __shfl_sync(0xffffffffu, warp, 0) - 12;             // 0, 1: MMA issuers
    if (role < 2) {
      if (role == 0) {
        tmem_alloc(tmem_slot, kTmemCols);
        tmem_relinquish();
      }
      tc_fence_before_sync();
      named_barrier(2, 64);
      tc_fence_after_sync();
    }
    if (role < 2 && n_tiles > 0) {
      const int u = role;
      const uint32_t idesc_s = idesc_f16(kBM, kBN), idesc_o = idesc_f16(kBM, kD) | (1u << 16);
      const uint64_t q_desc = umma_desc_sw128(smem_u32(q_s) + u * kTileBytes);
      const uint64_t k_desc0 = umma_desc_sw128(smem_u32(k_ring)), v_desc0 = umma_desc_sw128_mn(smem_u32(v_ring), kHalf, 1024);
      const uint32_t s_tmem = u * kTmemUnit, o_tmem = s_tmem + kTmemO;
      bool ok = *tmem_slot == 0 && mbar_wait(&q_full[u], 0);
      int reason = kWaitFullTimeout;
      int ks = 0, vs = 0;                                     // ring slots and their phases
      uint32_t kph = 0, vph = 0;
      auto issue_s = [&]() -> bool {
        if (!mbar_wait(&k_full[ks], kph)) return false;
        tc_fence_after_sync();
        if (elect_one()) {
          const uint64_t k_desc = k_desc0 + static_cast<uint64_t>(ks * (kTileBytes >> 4));
#pragma unroll
          for (int i = 0; i < kD / 16; ++i) {
            const uint64_t off = ((i >> 2) * kHalf + (i & 3) * 32) >> 4;
            umma_bf16(s_tmem, q_desc + off, k_desc + off, idesc_s, i > 0);
          }
          umma_commit(&s_full[u]);
          umma_commit(&k_empty[ks]);
        }
        __syncwarp();
        if (++ks == kNK) {
          ks = 0;
          kph ^= 1;
        }
        return true;
      };
      ok = ok && issue_s();
      for (int j = 0; ok && j < n_tiles; ++j) {
        if (!mbar_wait(&p_ready[u], j & 1)) { ok = false; reason = kWaitAccumTimeout; break; }
        if (!mbar_wait(&v_full[vs], vph)) { ok = false; break; }
        tc_fence_after_sync();
        if (elect_one()) {
          const uint64_t v_desc = v_desc0 + static_cast<uint64_t>(vs * (kTileBytes >> 4));
#pragma unroll
          for (int i = 0; i < kBN / 16; ++i)
            umma_bf16_a_tmem(o_tmem, s_tmem + i * 8, v_desc + i * (2048 >> 4), idesc_o, (j > 0 || i > 0) ? 1u : 0u);
          umma_commit(&o_done[u]);
          umma_commit(&v_empty[vs]);
        }
        __syncwarp();
        if (++vs == kNV) {
          vs = 0;
          vph ^= 1;
        }
        if (j + 1 < n_tiles && !issue_s()) ok = false;
      }
      if (lane == 0 && (!ok || *abort_flag)) {
        if (!ok) report_status(p.status, kId, reason);
        *abort_flag = 1;
      }
    }
  } else {
    // ---------------- softmax and output: thread r of unit u is query row r / G, head r % G ----------------
    set_regs_up<176>();
    const int u = wg, r = threadIdx.x & 127;
    const int by_g = p.by_g, row = row0 + u * rpu + ((r * by_g) >> 16);
    const int pos = pos0 + min(row, q_len - 1);              // lanes without a row follow the last one
    // Q: a power of two per row (and head) takes its largest element to 2^14 .. 2^15 of fp16, which is exact down to 2^-31 of
    // it; the scale's sign is Q's, and a scale of 0 a Q of 0. A unit's rows of all its heads are contiguous in memory row by
    // row; bulk copies bring them into a K slot that is free until tile 1 + u. All four warps send their share: a copy takes
    // its warp 67 cycles (one warp for all of them 2160; loads by the lanes that convert 3500). Sixteen lanes convert a row,
    // two rows at a time.
    int q_exp = 0;
    {
      const uint32_t bytes = static_cast<uint32_t>(G) * kD * 2;
      const int rows = rows_of(u);
      if (r == 0) mbar_expect_tx(&q_raw[u], rows * bytes);
      const __nv_bfloat16* src = p.q + (static_cast<size_t>(q_begin + row0 + u * rpu) * p.hq + hk * G) * kD;
      for (int i = (warp & 3) + 4 * lane; i < rows; i += 128)
        bulk_load(k_ring + (1 + u) * kTileBytes + i * bytes, src + static_cast<size_t>(i) * p.hq * kD, bytes, &q_raw[u]);
      __syncwarp();
    }
    bool ok = __all_sync(0xffffffffu, mbar_wait(&q_raw[u], 0));
    if (!ok) mbar_wait(&q_raw[u], 0);                        // the copies must not outlive the CTA
    if (ok) {
      const int c = lane & 15, first = (warp & 3) * 32 + (lane >> 4), lanes = rows_of(u) * G;
      const uint32_t raw = smem_u32(k_ring) + (1 + u) * kTileBytes + c * 16;
      uint4 v[16];
#pragma unroll
      for (int i = 0; i < 16; ++i)
        v[i] = first + 2 * i < lanes ? ld_shared_v4(raw + (first + 2 * i) * 256) : make_uint4(0u, 0u, 0u, 0u);
      // Largest magnitude of each row, rows i and i + 8 in one word; then sixteen lanes' words in steps that halve what a lane
      // keeps, so that lanes 2k and 2k + 1 of a half warp end with rows k and k + 8.
      auto top_of = [](const uint4& r) {
        const uint32_t a = __vmaxu2(r.x & 0x7fff7fffu, r.y & 0x7fff7fffu), b = __vmaxu2(r.z & 0x7fff7fffu, r.w & 0x7fff7fffu);
        const uint32_t two = __vmaxu2(a, b);
        return max(two >> 16, two & 0xffffu);
      };
      uint32_t tops[8], any = 0u;
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        tops[i] = top_of(v[i]) | top_of(v[i + 8]) << 16;
        any = __vmaxu2(any, tops[i]);
      }
      // Infinities and NaN do not choose a power, and are NaN: a row of scores that are all -inf has no softmax.
      if (__any_sync(0xffffffffu, __vmaxu2(any, 0x7f7f7f7fu) != 0x7f7f7f7fu)) {
#pragma unroll
        for (int i = 0; i < 16; ++i) {
          uint32_t w[4] = {v[i].x, v[i].y, v[i].z, v[i].w};
          uint32_t most = 0u;
#pragma unroll
          for (int k = 0; k < 4; ++k) {
            const uint32_t lo = w[k] & 0x7fffu, hi = (w[k] >> 16) & 0x7fffu;
            most = max(most, max(lo < 0x7f80u ? lo : 0u, hi < 0x7f80u ? hi : 0u));
            w[k] |= (lo < 0x7f80u ? 0u : 0x7fffu) | (hi < 0x7f80u ? 0u : 0x7fff0000u);
          }
          v[i] = make_uint4(w[0], w[1], w[2], w[3]);
          tops[i & 7] = i < 8 ? most : tops[i & 7] | most << 16;
        }
      }
#pragma unroll
      for (int step = 8, n = 4; step >= 2; step >>= 1, n >>= 1)
#pragma unroll
        for (int i = 0; i < n; ++i) {
          const bool up = lane & step;
          const uint32_t other = __shfl_xor_sync(0xffffffffu, up ? tops[i] : tops[i + n], step);
          tops[i] = __vmaxu2(up ? tops[i + n] : tops[i], other);
        }
      tops[0] = __vmaxu2(tops[0], __shfl_xor_sync(0xffffffffu, tops[0], 1));
      // This thread's row is number 2 i + half of its warp: i = lane / 2, half = lane & 1.
      const uint32_t word = __shfl_sync(0xffffffffu, tops[0], 16 * (lane & 1) + 2 * ((lane >> 1) & 7));
      q_exp = max(-120, static_cast<int>((lane < 16 ? word & 0xffffu : word >> 16) >> 7) - 127 - 14);
      const float f_own = p.sign * pow2(-q_exp);
#pragma unroll
      for (int i = 0; i < 16; ++i) {
        const uint32_t w[4] = {v[i].x, v[i].y, v[i].z, v[i].w};         // channels 0 1, 2 3, 4 5, 6 7 of the word
        const float f = __shfl_sync(0xffffffffu, f_own, 2 * i + (lane >> 4));
        float x[8];
#pragma unroll
        for (int k = 0; k < 4; ++k) {
          x[2 * k] = __uint_as_float(w[k] << 16) * f;
          x[2 * k + 1] = __uint_as_float(w[k] & 0xffff0000u) * f;
        }
        st_shared_v4(chunk_at(row_start(smem_u32(q_s) + u * kTileBytes, first + 2 * i), c), pack_f16(x[0], x[4]), pack_f16(x[1], x[5]),
                     pack_f16(x[2], x[6]), pack_f16(x[3], x[7]));
      }
      fence_proxy_async_smem();
      mbar_arrive(&q_full[u]);
    }
    const int row_exp = p.scale_exp + q_exp;
    const uint32_t taddr = u * kTmemUnit + (static_cast<uint32_t>((warp & 3) * 32) << 16);
    RowState st{kNoMax, 0.f, p.scale, 0.f, 0};
    int j = 0;
    // The tiles whose tokens have powers of their own are outside the loop of the others: inside it they cost those 1.5%.
    for (;; ++j) {
      for (; ok && j < n_tiles; ++j) {
        ok = __all_sync(0xffffffffu, mbar_wait(&s_full[u], j & 1) && *abort_flag == 0);
        if (!ok) break;
        tc_fence_after_sync();
        const TileScale ts = scales[j & 7];
        const int k0 = (tile0 + j) * kBN;
        // |S| is below 2^37: what a scale below 2^-100 makes of it is nothing. Never 0: it meets -inf.
        const float unit = pow2(max(-100, min(126, row_exp + ts.k)));
        uint32_t sr[4][32];                                    // the score row: 128 fp32
        tmem_ld32(taddr, sr[0]);
        if (ts.own) break;                                   // handled below
        const bool diagonal = k0 + kBN - 1 > pos;
        float mx[4];
#pragma unroll
        for (int c = 0; c < 4; ++c) {                          // the maximum of one quarter while the next is on its way
          tmem_ld_wait();
          tmem_ld_fence_regs(sr[c]);
          if (c < 3) tmem_ld32(taddr + (c + 1) * 32, sr[c + 1]);
          if (diagonal) {
#pragma unroll
            for (int i = 0; i < 32; ++i)
              if (k0 + c * 32 + i > pos) sr[c][i] = 0xff800000u;       // -inf
          }
          float a[10];
#pragma unroll
          for (int i = 0; i < 10; ++i)
            a[i] = fmax3(__uint_as_float(sr[c][3 * i]), __uint_as_float(sr[c][3 * i + 1]), __uint_as_float(sr[c][3 * i + 2]));
          mx[c] = fmax3(fmax3(fmax3(a[0], a[1], a[2]), fmax3(a[3], a[4], a[5]), fmax3(a[6], a[7], a[8])),
                        fmax3(a[9], __uint_as_float(sr[c][30]), __uint_as_float(sr[c][31])), -INFINITY);
        }
        float scale = st.mantissa * unit;
        const float top = fmax3(fmaxf(mx[0], mx[1]), mx[2], mx[3]);
        const float mt = fmaxf(top * scale, kNoMax);
        if (j == 0) {
          st.m = mt;
          if (RowState::is_huge(st.m)) {
            st.mantissa = 1.f;
            scale = unit;
            st.m = top * scale;
          }
          st.unit_v = ts.v;
          st.most_v = static_cast<float>(ts.v);
        } else {
          const bool need = mt > st.m + kLazy || ts.v != st.unit_v;
          if (__any_sync(0xffffffffu, need)) {
            ok = __all_sync(0xffffffffu, mbar_wait(&o_done[u], (j - 1) & 1));
            if (!ok) break;
            tc_fence_after_sync();
            const float grown = st.raise(p, top, unit, need ? fmaxf(st.m, mt) : st.m);
            scale = st.mantissa * unit;
            rescale(taddr, st.turn(grown, ts.v, top * scale - st.m));
          }
        }
        // The units take turns on the MUFU pipe, so that one's exponentials run under the rest of the other's chain.
        if (u == 1 || j > 0) {
          ok = __all_sync(0xffffffffu, u == 1 ? mbar_wait(&xu_done[0], j & 1) : mbar_wait(&xu_done[1], (j - 1) & 1));
          if (!ok) break;
        }
        const int below = max(-60, min(100, ts.v - st.unit_v));    // 0 but for tiles far from most_v
        const float less = static_cast<float>(below);
        const uint64_t scale2 = pack_f32x2(scale, scale), negm2 = pack_f32x2(-st.m + less, -st.m + less);
        uint64_t sums[2] = {0ull, 0ull};
#pragma unroll
        for (int c = 0; c < 4; ++c) {
          uint32_t packed[16];
#pragma unroll
          for (int i = 0; i < 32; i += 2) {
            float x0, x1;
            unpack_f32x2(fma_f32x2(pack_f32x2(__uint_as_float(sr[c][i]), __uint_as_float(sr[c][i + 1])), scale2, negm2), x0, x1);
            const float p0 = exp2f(x0), p1 = exp2f(x1);
            sums[(i >> 1) & 1] = add_f32x2(sums[(i >> 1) & 1], pack_f32x2(p0, p1));
            packed[i >> 1] = pack_f16(p0, p1);
          }
          tmem_st16(taddr + c * 16, packed);
        }
        {
          float a, c;
          unpack_f32x2(add_f32x2(sums[0], sums[1]), a, c);
          st.l += (a + c) * pow2(-below);
        }
        mbar_arrive(&xu_done[u]);
        tmem_st_wait();
        tc_fence_before_sync();
        mbar_arrive(&p_ready[u]);
      }
      if (!ok || j == n_tiles) break;
      tmem_ld_wait();
      ok = apart_tile(p, st, powers + (j & 3) * 2 * kBN, min(kBN, pos - (tile0 + j) * kBN + 1), row_exp, taddr, u, j, o_done, xu_done,
                      p_ready);
    }
    if (ok && n_tiles > 0) ok = __all_sync(0xffffffffu, mbar_wait(&o_done[u], (n_tiles - 1) & 1) && *abort_flag == 0);
    if (ok && p.splits > 1) {
      tc_fence_after_sync();
      const size_t slot = (((static_cast<size_t>(z) * gridDim.y + hk) * gridDim.x + blockIdx.x) * p.splits + split) *
                              (2 * kBM) + u * kBM + r;
      *reinterpret_cast<float2*>(p.ws_ml + slot * 2) = make_float2(st.mantissa == p.scale ? st.m : st.m * p.scale, st.l);
      const float vf0 = pos >= first_bad[0] ? CUDART_NAN_F : pow2(st.unit_v);
      const float vf1 = pos >= first_bad[1] ? CUDART_NAN_F : pow2(st.unit_v);
      // Through the unit's Q tile (all its MMAs are over) half the channels at a time, so that the writes are whole lines. A
      // split without tiles leaves no output, only m = kNoMax, l = 0.
      const uint32_t tile = smem_u32(q_s) + u * kTileBytes;
      const size_t slot0 = slot - r;
#pragma unroll 1
      for (int half = 0; half < 2 && n_tiles > 0; ++half) {
        uint32_t o[2][32];
        tmem_ld32(taddr + kTmemO + half * 64, o[0]);
        tmem_ld32(taddr + kTmemO + half * 64 + 32, o[1]);
        tmem_ld_wait();
        tmem_ld_fence_regs(o[0]);
        tmem_ld_fence_regs(o[1]);
#pragma unroll
        for (int ch = 0; ch < 2; ++ch) {
#pragma unroll
          for (int w = 0; w < 4; ++w) {                      // words of channels 0 4 1 5 2 6 3 7
            auto x = [&](int i) { return __float_as_uint(__uint_as_float(o[ch][8 * w + i]) * ((w & 1) ? vf1 : vf0)); };
            const int k = ch * 8 + 2 * w;
            st_shared_v4(tile + r * 256 + ((k ^ (r & 15)) << 4), x(0), x(2), x(4), x(6));
            st_shared_v4(tile + r * 256 + (((k + 1) ^ (r & 15)) << 4), x(1), x(3), x(5), x(7));
          }
        }
        __syncwarp();
        const int c = lane & 15;
        uint4 v[16];
#pragma unroll
        for (int i = 0; i < 16; ++i) {
          const int at = (warp & 3) * 32 + 2 * i + (lane >> 4);
          v[i] = ld_shared_v4(tile + at * 256 + ((c ^ (at & 15)) << 4));
        }
#pragma unroll
        for (int i = 0; i < 16; ++i)
          *(reinterpret_cast<uint4*>(p.ws_o + (slot0 + (warp & 3) * 32 + 2 * i + (lane >> 4)) * kD + half * 64) + c) = v[i];
        __syncwarp();
      }
    } else if (ok) {
      tc_fence_after_sync();
      const float vf0 = pos >= first_bad[0] ? CUDART_NAN_F : pow2(st.unit_v);
      const float vf1 = pos >= first_bad[1] ? CUDART_NAN_F : pow2(st.unit_v);
      const float inv = st.l == 0.f ? 0.f : 1.f / st.l;            // times 2^unit_v it may leave fp32: small values, many tokens
      // Rows leave through the unit's Q tile (all its MMAs are over), so that the writes are whole lines.
      const uint32_t at = row_start(smem_u32(q_s) + u * kTileBytes, r);
      uint32_t o[4][32];
      if (n_tiles > 0) {
#pragma unroll
        for (int ch = 0; ch < 4; ++ch) tmem_ld32(taddr + kTmemO + ch * 32, o[ch]);
        tmem_ld_wait();
#pragma unroll
        for (int ch = 0; ch < 4; ++ch) tmem_ld_fence_regs(o[ch]);
      } else {
#pragma unroll
        for (int i = 0; i < 128; ++i) o[i >> 5][i & 31] = 0u;
      }
#pragma unroll
      for (int ch = 0; ch < 4; ++ch) {
#pragma unroll
        for (int w = 0; w < 4; ++w) {                        // words of channels 0 4 1 5 2 6 3 7
          auto x = [&](int i) { return st.l == 0.f ? 0.f : __uint_as_float(o[ch][8 * w + i]) * inv * ((w & 1) ? vf1 : vf0); };
          st_shared_v4(chunk_at(at, 4 * ch + w), pack_bf16(x(0), x(2)), pack_bf16(x(4), x(6)), pack_bf16(x(1), x(3)),
                       pack_bf16(x(5), x(7)));
        }
      }
      __syncwarp();
      const int c = lane & 15;
#pragma unroll 1
      for (int i0 = 0; i0 < 16; i0 += 8) {                   // eight reads, then eight writes: the compiler keeps their order
        uint4 v[8];
#pragma unroll
        for (int i = 0; i < 8; ++i)
          v[i] = ld_shared_v4(chunk_at(row_start(smem_u32(q_s) + u * kTileBytes, (warp & 3) * 32 + 2 * (i0 + i) + (lane >> 4)), c));
#pragma unroll
        for (int i = 0; i < 8; ++i) {
          const int qr_ = (warp & 3) * 32 + 2 * (i0 + i) + (lane >> 4), rr = (qr_ * by_g) >> 16, hh = qr_ - rr * G;
          const int qrow = row0 + u * rpu + rr;
          if (rr < rpu && qrow < q_len)
            *(reinterpret_cast<uint4*>(p.out + (static_cast<size_t>(q_begin + qrow) * p.hq + hk * G + hh) * kD) + c) = v[i];
        }
      }
    } else if (lane == 0) {
      report_status(p.status, kId, kWaitAccumTimeout);
      *abort_flag = 1;
    }
  }

  tc_fence_before_sync();
  __syncthreads();
  if (warp == 12) {
    tc_fence_after_sync();
    tmem_dealloc(*tmem_slot, kTmemCols);
  }
}

// Joins the splits: a warp a lane (query row, head) of the launch above, four channels a thread.
constexpr int kJoinWarps = 8;
__global__ void __launch_bounds__(kJoinWarps * 32) kv4_prefill_join_kernel(const Params p, int blocks) {
  grid_dep_launch();
  grid_dep_wait();
  const int b = p.seq_begin + blockIdx.z, hk = blockIdx.y;
  const int q_begin = p.cu_q[b], q_len = p.cu_q[b + 1] - q_begin;
  if (!rows_fine(p, q_begin, p.cu_q[b + 1])) return;
  const int G = p.hq / p.hkv, rpu = kBM / G;
  const int i = blockIdx.x * kJoinWarps + (threadIdx.x >> 5), lane = threadIdx.x & 31;
  const int block = i / (2 * kBM), u = (i / kBM) & 1, r = i % kBM;
  const int row = (blocks - 1 - block) * 2 * rpu + u * rpu + r / G;
  if (r >= rpu * G || row >= q_len) return;
  const size_t slot = ((static_cast<size_t>(blockIdx.z) * gridDim.y + hk) * blocks + block) * p.splits * (2 * kBM) + i % (2 * kBM);
  constexpr int kBatch = 8;                                  // splits in flight: the kernel is a chain of L2 round trips
  float M = kNoMax, L = 0.f;
  float4 acc = make_float4(0.f, 0.f, 0.f, 0.f);
  for (int s0 = 0; s0 < p.splits; s0 += kBatch) {
    float2 ml[kBatch];
    float4 v[kBatch];
    float mn = M;
#pragma unroll
    for (int i = 0; i < kBatch; ++i) {
      const size_t at = slot + static_cast<size_t>(s0 + i) * (2 * kBM);
      const bool there = s0 + i < p.splits;
      ml[i] = there ? *reinterpret_cast<const float2*>(p.ws_ml + at * 2) : make_float2(kNoMax, 0.f);
      v[i] = there ? *reinterpret_cast<const float4*>(p.ws_o + at * kD + lane * 4) : make_float4(0.f, 0.f, 0.f, 0.f);
    }
#pragma unroll
    for (int i = 0; i < kBatch; ++i) mn = fmaxf(mn, ml[i].x);
    const float f0 = exp2f(M - mn);
    M = mn;
    L *= f0;
    acc.x *= f0; acc.y *= f0; acc.z *= f0; acc.w *= f0;
#pragma unroll
    for (int i = 0; i < kBatch; ++i) {
      if (ml[i].x == kNoMax && ml[i].y == 0.f) continue;     // saw nothing, and may have written nothing
      const float f = exp2f(ml[i].x - M);
      L += ml[i].y * f;
      acc.x += v[i].x * f; acc.y += v[i].y * f; acc.z += v[i].z * f; acc.w += v[i].w * f;
    }
  }
  const float inv = L == 0.f ? 0.f : 1.f / L;
  *reinterpret_cast<uint2*>(p.out + (static_cast<size_t>(q_begin + row) * p.hq + hk * G + r % G) * kD + lane * 4) =
      make_uint2(pack_bf16(acc.x * inv, acc.y * inv), pack_bf16(acc.z * inv, acc.w * inv));
}

int blocks_of(int max_q_len, int hq, int hkv) {
  const int rows = 2 * (kBM / (hq / hkv));
  return std::max(1, static_cast<int>((max_q_len + rows - 1ll) / rows));          // one to clear rows even where all chunks are empty
}

}  // namespace

extern "C" {

// Splits of the KV range, from launch-shape constants: as many as leave every CTA an SM, but no shorter than a tile, and only
// from four tiles on. Device times: 8 CTAs of 1 tile 10.0 us whole, 12.6 in two; of 5 tiles 18.3 whole, 13.4 in five; of
// 13 35.0 whole, 15.0 in 13 or more; 24 of 13 35.4 whole, 19.0 in six, 27.0 in eight (more than the SMs); 40 of 3 14.1 whole,
// 16.6 in three; 80 of 26 63.1 whole, 79.4 in two, 63.2 in three.
int xv_kv4_prefill_splits(int num_seqs, int max_q_len, int hq, int hkv, int max_tokens_per_seq, int num_sms) {
  if (num_seqs <= 0 || max_q_len <= 0 || hkv <= 0 || hq < hkv || hq / hkv > 16) return 1;
  const long long ctas = static_cast<long long>(num_seqs) * hkv * blocks_of(max_q_len, hq, hkv);
  const long long by_sms = num_sms / ctas, by_len = (max_tokens_per_seq + kBN - 1ll) / kBN;
  return by_len < 4 ? 1 : static_cast<int>(std::max(1ll, std::min({by_sms, by_len, 16ll})));
}

long long xv_kv4_prefill_workspace_bytes(int num_seqs, int max_q_len, int hq, int hkv, int splits) {
  if (splits <= 1 || hkv <= 0 || hq < hkv || hq / hkv > 16) return 0;
  return static_cast<long long>(num_seqs) * hkv * blocks_of(max_q_len, hq, hkv) * splits * (2 * kBM) * (kD + 2) * 4;
}

int xv_kv4_prefill(const void* q, const void* k_cache, const void* v_cache, const int* block_tables, const int* cu_q,
                   const int* kv_lens, void* out, int seq_begin, int num_seqs, int max_q_len, int total_rows, int clear_to, int hq, int hkv,
                   int d, int block_size, int max_blocks, int num_blocks, float scale, int splits, void* workspace,
                   long long workspace_bytes, int* status, cudaStream_t stream) {
  if (num_seqs <= 0) return 0;
  if (d != kD) return XV_ERR_UNSUPPORTED;
  if (hkv <= 0 || hq <= 0 || hq % hkv || hq / hkv > 16 || block_size <= 0 || block_size % kv4::kUnit || max_blocks <= 0 ||
      num_blocks <= 0 || hkv > 65535 || splits < 1 || max_q_len < 0 || clear_to > total_rows || static_cast<long long>(num_seqs) * splits > 65535)
    return XV_ERR_SHAPE;
  if (splits > 1 && (!workspace || workspace_bytes < xv_kv4_prefill_workspace_bytes(num_seqs, max_q_len, hq, hkv, splits)))
    return XV_ERR_WORKSPACE;
  if (reinterpret_cast<uintptr_t>(workspace) & 15) return XV_ERR_ALIGN;
  if ((reinterpret_cast<uintptr_t>(q) | reinterpret_cast<uintptr_t>(k_cache) | reinterpret_cast<uintptr_t>(v_cache) |
       reinterpret_cast<uintptr_t>(out)) & 15)
    return XV_ERR_ALIGN;
  static std::atomic<bool> done[64];
  int dev = 0;
  if (cudaGetDevice(&dev) != cudaSuccess || dev < 0 || dev >= 64) return XV_ERR_LAUNCH;
  if (!done[dev].load(std::memory_order_acquire)) {
    if (cudaFuncSetAttribute(kv4_prefill_tc_kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, kSmem) != cudaSuccess)
      return XV_ERR_LAUNCH;
    done[dev].store(true, std::memory_order_release);
  }
  Params p;
  p.q = static_cast<const __nv_bfloat16*>(q);
  p.k_cache = static_cast<const uint8_t*>(k_cache);
  p.v_cache = static_cast<const uint8_t*>(v_cache);
  p.block_tables = block_tables;
  p.cu_q = cu_q;
  p.kv_lens = kv_lens;
  p.out = static_cast<__nv_bfloat16*>(out);
  p.status = status;
  p.seq_begin = seq_begin; p.num_seqs = num_seqs; p.max_q_len = max_q_len; p.clear_to = clear_to;
  p.hq = hq; p.hkv = hkv; p.block_size = block_size; p.max_blocks = max_blocks;
  p.num_blocks = num_blocks; p.total_rows = total_rows;
  const double s = scale == 0.f ? 1.0 : std::abs(static_cast<double>(scale)) * kLog2e;
  p.scale = static_cast<float>(2.0 * std::frexp(s, &p.scale_exp));
  p.scale_exp -= 1;
  p.sign = scale == 0.f ? 0.f : scale < 0.f ? -1.f : 1.f;
  const int blocks = blocks_of(max_q_len, hq, hkv);
  p.splits = splits;
  p.G = hq / hkv;
  p.rpu = kBM / p.G;
  p.by_g = 65536 / p.G + 1;                       // exact for 128 lanes and G up to 16
  p.inv_splits = splits > 1 ? static_cast<uint32_t>((1ull << 32) / splits) + 1 : 0u;
  p.ws_o = static_cast<float*>(workspace);
  p.ws_ml = splits > 1 ? p.ws_o + static_cast<size_t>(num_seqs) * hkv * blocks * splits * (2 * kBM) * kD : nullptr;
  launch_pdl(kv4_prefill_tc_kernel, dim3(blocks, hkv, num_seqs * splits), dim3(512), kSmem, stream, p);
  if (cudaGetLastError() != cudaSuccess) return XV_ERR_LAUNCH;
  if (splits > 1) {
    launch_pdl(kv4_prefill_join_kernel, dim3(blocks * (2 * kBM / kJoinWarps), hkv, num_seqs), dim3(kJoinWarps * 32), 0, stream, p,
               blocks);
    if (cudaGetLastError() != cudaSuccess) return XV_ERR_LAUNCH;
  }
  return 0;
}

}  // extern "C"
