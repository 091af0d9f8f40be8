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
// Registers move from the issuers' and dequantisers' warpgroups to the softmax ones (setmaxnreg: 2 x 184 + 96 + 48 = 4 x 128).
//
// fp16 operands, not bf16: a dequantised value c + s (n - 8) has more than bf16's 8 bits, and its rounding (2^-12 instead
// of 2^-9) would otherwise be the largest error of the result. Their range is kept by powers of two: a row of Q is scaled
// by its largest element, a tile of K or V by an exponent that its dequantisers choose from the tile's parameters (and
// keep while it fits); the scores undo Q's and K's, and V's is carried with the output accumulator.
// Inside a word the channels are stored in the order 0 4 1 5 2 6 3 7, which is how the nibbles unpack: Q follows it, and
// the output undoes it for V.
//
// Rows that do not see a token never meet its values: its score is replaced by -inf, P is 0 there, and V of a token whose
// parameters are not finite is stored as 0 with its K made NaN, so that exactly the rows that see it become NaN.
// Every wait is bounded; one that runs out records a status code, the CTA stops issuing work, frees its tensor memory and
// returns.

#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_runtime.h>

#include <atomic>
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
constexpr int kBarBytes = 512;
constexpr int kSmem = (2 + kNK + kNV) * kTileBytes + 1024 + kBarBytes;
constexpr uint32_t kTmemCols = 512, kTmemUnit = 256, kTmemO = 128;
constexpr int kId = 12;
constexpr float kLog2e = 1.4426950408889634f;
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
  int seq_begin, hq, hkv, block_size, max_blocks, num_blocks, total_rows;
  float scale_log2;
};

struct alignas(16) TileScale {                    // of one tile: K and V are stored divided by k and v
  float k, v, v_inv, unused;
};

__device__ __forceinline__ uint32_t pack_f16(float lo, float hi) {
  const __half2 v = __floats2half2_rn(lo, hi);
  return *reinterpret_cast<const uint32_t*>(&v);
}
__device__ __forceinline__ float pow2(int e) { return __int_as_float((127 + e) << 23); }
__device__ __forceinline__ uint32_t idesc_f16(int m, int n) {
  return (1u << 4) | static_cast<uint32_t>(n >> 3) << 17 | static_cast<uint32_t>(m >> 4) << 24;
}
template <int N>
__device__ __forceinline__ void set_regs_up() { asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(N)); }
template <int N>
__device__ __forceinline__ void set_regs_down() { asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(N)); }

// Byte offset of 16-byte chunk c (0..15: one word of channels) of row r in a tile.
__device__ __forceinline__ uint32_t chunk_at(int r, int c) {
  return static_cast<uint32_t>((c >> 3) * kHalf + r * 128 + (((c & 7) ^ (r & 7)) << 4));
}
__device__ __forceinline__ void st_shared_v4(uint32_t addr, uint32_t a, uint32_t b, uint32_t c, uint32_t d) {
  asm volatile("st.shared.v4.b32 [%0], {%1, %2, %3, %4};" ::"r"(addr), "r"(a), "r"(b), "r"(c), "r"(d) : "memory");
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

// 32 of a row's 64 code bytes as fp16 c + s (n - 8) into chunks 4 c0 .. : words of even index belong to group 0.
__device__ __forceinline__ void put_words(uint32_t tile, int row, int c0, const uint4& codes, __half2 s0, __half2 o0,
                                          __half2 s1, __half2 o1) {
  const uint32_t w[4] = {codes.x, codes.y, codes.z, codes.w};
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const __half2 s = (i & 1) ? s1 : s0, o = (i & 1) ? o1 : o0;
    const uint32_t hi = w[i] >> 8;
    uint32_t v[4];
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const __half2 x = __hfma2(centred_f16(j < 2 ? w[i] : hi, j & 1), s, o);
      v[j] = *reinterpret_cast<const uint32_t*>(&x);
    }
    st_shared_v4(tile + chunk_at(row, c0 + i), v[0], v[1], v[2], v[3]);
  }
}

__global__ void __launch_bounds__(512, 1) kv4_prefill_tc_kernel(const Params p) {
  extern __shared__ __align__(1024) uint8_t smem_raw[];
  grid_dep_launch();
  grid_dep_wait();
  const int b = p.seq_begin + blockIdx.z, hk = blockIdx.y;
  const int q_begin = p.cu_q[b];
  const int q_len = p.cu_q[b + 1] - q_begin;
  if (q_begin < 0 || q_len < 0 || q_len > p.total_rows - q_begin) {
    if (threadIdx.x == 0) report_status(p.status, kId, kBadIndex);
    return;
  }
  const int G = p.hq / p.hkv;
  const int rpu = kBM / G;                                   // query rows of a unit
  const int row0 = (static_cast<int>(gridDim.x) - 1 - static_cast<int>(blockIdx.x)) * 2 * rpu;     // long ones first
  if (row0 >= q_len) return;
  int kv_len = max(p.kv_lens[b], 0);
  const long long most = static_cast<long long>(p.max_blocks) * p.block_size;
  if (kv_len > most) {
    if (threadIdx.x == 0) report_status(p.status, kId, kBadIndex);
    kv_len = static_cast<int>(most);
  }
  const int pos0 = kv_len - q_len;                           // position of query row 0; rows before position 0 see nothing
  const int rows_here = min(2 * rpu, q_len - row0);
  const int n_kv = max(0, min(kv_len, pos0 + row0 + rows_here));
  const int n_tiles = (n_kv + kBN - 1) / kBN;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int wg = warp >> 2;

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
  TileScale* scales = reinterpret_cast<TileScale*>(xu_done + 2);         // [8], by tile (20 barriers before it: 16-byte aligned)
  uint32_t* red = reinterpret_cast<uint32_t*>(scales + 8);   // [2][12]
  uint32_t* tmem_slot = red + 24;
  volatile int* abort_flag = reinterpret_cast<volatile int*>(tmem_slot + 1);

  if (threadIdx.x == 0) {
    for (int u = 0; u < 2; ++u) {
      mbar_init(&q_full[u], 128);
      mbar_init(&s_full[u], 1);
      mbar_init(&p_ready[u], 128);
      mbar_init(&o_done[u], 1);
      mbar_init(&xu_done[u], 128);
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
    mbar_fence_init();
  }
  if (warp == 12) {
    tmem_alloc(tmem_slot, kTmemCols);
    tmem_relinquish();
  }
  tc_fence_before_sync();
  __syncthreads();
  tc_fence_after_sync();
  const uint32_t tmem_base = *tmem_slot;

  if (wg == 2) {
    // ---------------- dequantisers ----------------
    set_regs_down<96>();
    const int row = threadIdx.x & 127;
    const int upp = p.block_size / kv4::kUnit;
    const int* table = p.block_tables + static_cast<size_t>(b) * p.max_blocks;
    // This thread's row of tile j: offsets of its codes and parameters (a row past the end reads the last token's).
    auto place = [&](int j, size_t* code, size_t* par) {
      const int tok = min(j * kBN + row, n_kv - 1);
      const int page = tok / p.block_size, r = tok - page * p.block_size;
      int blk = __ldg(table + page);
      if (static_cast<unsigned>(blk) >= static_cast<unsigned>(p.num_blocks)) {
        report_status(p.status, kId, kBadIndex);
        blk = 0;
      }
      const size_t unit = ((static_cast<size_t>(blk) * p.hkv + hk) * upp + r / kv4::kUnit) * kv4::kUnitBytes;
      *code = unit + (r % kv4::kUnit) * kv4::kCodeRow;
      *par = unit + kv4::kParBase + (r % kv4::kUnit) * kv4::kParRow;
    };
    size_t code = 0, par = 0;
    uint4 kc[4], vc[4];
    uint2 kp = make_uint2(0, 0), vp = make_uint2(0, 0), kp_next, vp_next;
    auto load_codes = [&](uint4 (&c)[4], const uint8_t* cache) {
#pragma unroll
      for (int i = 0; i < 4; ++i) c[i] = __ldg(reinterpret_cast<const uint4*>(cache + code) + i);
    };
    if (n_tiles > 0) {
      place(0, &code, &par);
      kp = __ldg(reinterpret_cast<const uint2*>(p.k_cache + par));
      vp = __ldg(reinterpret_cast<const uint2*>(p.v_cache + par));
      load_codes(kc, p.k_cache);
      load_codes(vc, p.v_cache);
      place(min(1, n_tiles - 1), &code, &par);
    }
    int ek = 0, ev = 0;
    // A wait that runs out is only noted: the four warps leave together, at the barrier of the next tile.
    bool ok = true;
    for (int j = 0; j < n_tiles; ++j) {
      // The next tile's parameters now, its codes as the registers of this tile's become free.
      kp_next = __ldg(reinterpret_cast<const uint2*>(p.k_cache + par));
      vp_next = __ldg(reinterpret_cast<const uint2*>(p.v_cache + par));
      if (j * kBN + row >= n_kv) kp = vp = make_uint2(0u, 0u);
      // exponent bits all ones: not finite
      auto finite = [](uint32_t w) { return (w & 0x7f80u) != 0x7f80u && (w & 0x7f800000u) != 0x7f800000u; };
      if (!finite(vp.x) || !finite(vp.y)) {
        vp = make_uint2(0u, 0u);
        kp = make_uint2(0x7fff7fffu, 0x7fff7fffu);
      }
      const float ks0 = kv4::par_s(kp.x), kc0 = kv4::par_c(kp.x), ks1 = kv4::par_s(kp.y), kc1 = kv4::par_c(kp.y);
      const float vs0 = kv4::par_s(vp.x), vc0 = kv4::par_c(vp.x), vs1 = kv4::par_s(vp.y), vc1 = kv4::par_c(vp.y);
      const bool k_fine = finite(kp.x) && finite(kp.y);
      const float kb = k_fine ? fmaxf(fabsf(kc0) + 8.f * fabsf(ks0), fabsf(kc1) + 8.f * fabsf(ks1)) : 0.f;
      const float vb = fmaxf(fabsf(vc0) + 8.f * fabsf(vs0), fabsf(vc1) + 8.f * fabsf(vs1));
      const uint32_t kw = __reduce_max_sync(0xffffffffu, __float_as_uint(kb));
      const uint32_t vw = __reduce_max_sync(0xffffffffu, __float_as_uint(vb));
      uint32_t* slot_red = red + (j & 1) * 12;
      if (lane == 0) {
        slot_red[warp & 3] = kw;
        slot_red[4 + (warp & 3)] = vw;
        slot_red[8 + (warp & 3)] = ok ? 0u : 1u;
      }
      named_barrier(1, 128);
      if ((slot_red[8] | slot_red[9] | slot_red[10] | slot_red[11]) != 0u) break;
      const uint32_t kbits = max(max(slot_red[0], slot_red[1]), max(slot_red[2], slot_red[3]));
      const uint32_t vbits = max(max(slot_red[4], slot_red[5]), max(slot_red[6], slot_red[7]));
      // Largest magnitude of the stored tile: 8 .. 16 when an exponent is chosen, kept while it stays in 2^-4 .. 2^15.
      auto choose = [](int e, uint32_t bits) {
        const int top = static_cast<int>(bits >> 23) - 127;
        if (bits != 0 && (top - e > 14 || top - e < -4)) e = top - 3;
        return max(-100, min(100, e));
      };
      ek = choose(ek, kbits);
      ev = choose(ev, vbits);
      if (row == 0) {
        TileScale sc;
        sc.k = pow2(ek);
        sc.v = pow2(ev);
        sc.v_inv = pow2(-ev);
        sc.unused = 0.f;
        scales[j & 7] = sc;
      }
      const int ks = j % kNK, vs = j % kNV;
      ok = __all_sync(0xffffffffu, mbar_wait(&k_empty[ks], ((j / kNK) & 1) ^ 1) && *abort_flag == 0);
      if (ok) {
        const float f = pow2(-ek);
        const __half2 s0 = __float2half2_rn(ks0 * f), o0 = __float2half2_rn(kc0 * f), s1 = __float2half2_rn(ks1 * f),
                      o1 = __float2half2_rn(kc1 * f);
        const uint32_t tile = smem_u32(k_ring) + ks * kTileBytes;
#pragma unroll
        for (int i = 0; i < 4; ++i) put_words(tile, row, 4 * i, kc[i], s0, o0, s1, o1);
        fence_proxy_async_smem();
        mbar_arrive(&k_full[ks]);
      }
      if (j + 1 < n_tiles) load_codes(kc, p.k_cache);
      ok = ok && __all_sync(0xffffffffu, mbar_wait(&v_empty[vs], ((j / kNV) & 1) ^ 1) && *abort_flag == 0);
      if (ok) {
        const float f = pow2(-ev);
        const __half2 s0 = __float2half2_rn(vs0 * f), o0 = __float2half2_rn(vc0 * f), s1 = __float2half2_rn(vs1 * f),
                      o1 = __float2half2_rn(vc1 * f);
        const uint32_t tile = smem_u32(v_ring) + vs * kTileBytes;
#pragma unroll
        for (int i = 0; i < 4; ++i) put_words(tile, row, 4 * i, vc[i], s0, o0, s1, o1);
        fence_proxy_async_smem();
        mbar_arrive(&v_full[vs]);
      }
      if (j + 1 < n_tiles) {
        load_codes(vc, p.v_cache);
        kp = kp_next;
        vp = vp_next;
        place(min(j + 2, n_tiles - 1), &code, &par);
      }
    }
    if (!ok && lane == 0) {
      report_status(p.status, kId, kWaitEmptyTimeout);
      *abort_flag = 1;
    }
  } else if (wg == 3) {
    // ---------------- MMA issuers: one thread per unit ----------------
    set_regs_down<48>();
    const int u = warp - 12;
    if (u < 2 && lane == 0 && n_tiles > 0) {
      const uint32_t idesc_s = idesc_f16(kBM, kBN), idesc_o = idesc_f16(kBM, kD) | (1u << 16);
      const uint32_t q_addr = smem_u32(q_s) + u * kTileBytes;
      const uint32_t k_addr0 = smem_u32(k_ring), v_addr0 = smem_u32(v_ring);
      const uint32_t s_tmem = tmem_base + u * kTmemUnit, o_tmem = s_tmem + kTmemO;
      bool ok = mbar_wait(&q_full[u], 0);
      int reason = kWaitFullTimeout;
      auto issue_s = [&](int j) -> bool {
        const int slot = j % kNK;
        if (!mbar_wait(&k_full[slot], (j / kNK) & 1)) return false;
        tc_fence_after_sync();
        const uint32_t k_addr = k_addr0 + slot * kTileBytes;
#pragma unroll
        for (int ks = 0; ks < kD / 16; ++ks)
          umma_bf16(s_tmem, umma_desc_sw128(q_addr + (ks >> 2) * kHalf + (ks & 3) * 32),
                    umma_desc_sw128(k_addr + (ks >> 2) * kHalf + (ks & 3) * 32), idesc_s, ks > 0);
        umma_commit(&s_full[u]);
        umma_commit(&k_empty[slot]);
        return true;
      };
      if (ok) ok = issue_s(0);
      for (int j = 0; ok && j < n_tiles; ++j) {
        if (!mbar_wait(&p_ready[u], j & 1)) { ok = false; reason = kWaitAccumTimeout; break; }
        const int slot = j % kNV;
        if (!mbar_wait(&v_full[slot], (j / kNV) & 1)) { ok = false; break; }
        tc_fence_after_sync();
        const uint32_t v_addr = v_addr0 + slot * kTileBytes;
#pragma unroll
        for (int ks = 0; ks < kBN / 16; ++ks)
          umma_bf16_a_tmem(o_tmem, s_tmem + ks * 8, umma_desc_sw128_mn(v_addr + ks * 2048, kHalf, 1024), idesc_o,
                           (j > 0 || ks > 0) ? 1u : 0u);
        umma_commit(&o_done[u]);
        umma_commit(&v_empty[slot]);
        if (j + 1 < n_tiles && !issue_s(j + 1)) ok = false;
      }
      if (!ok || *abort_flag) {
        if (!ok) report_status(p.status, kId, reason);
        *abort_flag = 1;
      }
    }
  } else {
    // ---------------- softmax and output: thread r of unit u is query row r / G, head r % G ----------------
    set_regs_up<184>();
    const int u = wg, r = threadIdx.x & 127;
    const int qr = r / G, hd = r - qr * G;
    const int row = row0 + u * rpu + qr;
    const bool live = qr < rpu && row < q_len;
    const int pos = pos0 + min(row, q_len - 1);              // lanes without a row follow the last one
    // Q: a power of two per row keeps it in fp16's range; a negative scale is its sign.
    float row_scale;
    {
      const uint4* src = reinterpret_cast<const uint4*>(
          p.q + (static_cast<size_t>(q_begin + (live ? row : row0)) * p.hq + hk * G + (live ? hd : 0)) * kD);
      uint4 v[16];
      uint32_t top = 0;
#pragma unroll
      for (int c = 0; c < 16; ++c) {
        v[c] = __ldg(src + c);
        const uint32_t w[4] = {v[c].x, v[c].y, v[c].z, v[c].w};
#pragma unroll
        for (int i = 0; i < 4; ++i) top = max(top, max(w[i] & 0x7fffu, (w[i] >> 16) & 0x7fffu));
      }
      const int e = max(-100, min(100, static_cast<int>(top >> 7) - 127));
      const float f = p.scale_log2 < 0.f ? -pow2(-e) : pow2(-e);
      row_scale = fmaxf(fabsf(p.scale_log2), 1e-30f) * pow2(e);
      const uint32_t tile = smem_u32(q_s) + u * kTileBytes;
#pragma unroll
      for (int c = 0; c < 16; ++c) {
        const uint32_t w[4] = {v[c].x, v[c].y, v[c].z, v[c].w};   // channels 0 1, 2 3, 4 5, 6 7 of the word
        float x[8];
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          x[2 * i] = __uint_as_float(w[i] << 16) * f;
          x[2 * i + 1] = __uint_as_float(w[i] & 0xffff0000u) * f;
        }
        st_shared_v4(tile + chunk_at(r, c), pack_f16(x[0], x[4]), pack_f16(x[1], x[5]), pack_f16(x[2], x[6]),
                     pack_f16(x[3], x[7]));
      }
      fence_proxy_async_smem();
      mbar_arrive(&q_full[u]);
    }
    const uint32_t taddr = tmem_base + u * kTmemUnit + (static_cast<uint32_t>((warp & 3) * 32) << 16);
    float m = kNoMax, l = 0.f, vf = 1.f;
    bool ok = true;
    for (int j = 0; j < n_tiles; ++j) {
      ok = __all_sync(0xffffffffu, mbar_wait(&s_full[u], j & 1) && *abort_flag == 0);
      if (!ok) break;
      tc_fence_after_sync();
      uint32_t sr[8][16];                                    // the score row: 128 fp32
#pragma unroll
      for (int c = 0; c < 8; ++c) tmem_ld16(taddr + c * 16, sr[c]);
      const TileScale ts = scales[j & 7];
      tmem_ld_wait();
      const int k0 = j * kBN;
      if (k0 + kBN - 1 > pos) {
#pragma unroll
        for (int c = 0; c < 8; ++c)
#pragma unroll
          for (int i = 0; i < 16; ++i)
            if (k0 + c * 16 + i > pos) sr[c][i] = 0xff800000u;       // -inf
      }
      float mx[8];
#pragma unroll
      for (int c = 0; c < 8; ++c) {
        const float a0 = fmax3(__uint_as_float(sr[c][0]), __uint_as_float(sr[c][1]), __uint_as_float(sr[c][2]));
        const float a1 = fmax3(__uint_as_float(sr[c][3]), __uint_as_float(sr[c][4]), __uint_as_float(sr[c][5]));
        const float a2 = fmax3(__uint_as_float(sr[c][6]), __uint_as_float(sr[c][7]), __uint_as_float(sr[c][8]));
        const float a3 = fmax3(__uint_as_float(sr[c][9]), __uint_as_float(sr[c][10]), __uint_as_float(sr[c][11]));
        const float a4 = fmax3(__uint_as_float(sr[c][12]), __uint_as_float(sr[c][13]), __uint_as_float(sr[c][14]));
        mx[c] = fmax3(fmax3(a0, a1, a2), fmax3(a3, a4, __uint_as_float(sr[c][15])), -INFINITY);
      }
      const float scale = row_scale * ts.k;
      const float mt = fmaxf(fmax3(fmax3(mx[0], mx[1], mx[2]), fmax3(mx[3], mx[4], mx[5]), fmaxf(mx[6], mx[7])) * scale, kNoMax);
      if (j == 0) {
        m = mt;
        vf = ts.v;
      } else {
        const bool need = mt > m + kLazy || ts.v != vf;
        if (__any_sync(0xffffffffu, need)) {
          ok = __all_sync(0xffffffffu, mbar_wait(&o_done[u], (j - 1) & 1));
          if (!ok) break;
          tc_fence_after_sync();
          const float m_new = need ? fmaxf(m, mt) : m;
          const float down = exp2f(m - m_new);
          l *= down;
          m = m_new;
          const float alpha = down * (vf * ts.v_inv);
          vf = ts.v;
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
      }
      // The units take turns on the MUFU pipe, so that one's exponentials run under the rest of the other's chain.
      if (u == 1 || j > 0) {
        ok = __all_sync(0xffffffffu, u == 1 ? mbar_wait(&xu_done[0], j & 1) : mbar_wait(&xu_done[1], (j - 1) & 1));
        if (!ok) break;
      }
      const uint64_t scale2 = pack_f32x2(scale, scale), negm2 = pack_f32x2(-m, -m);
      float sums[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
      for (int c = 0; c < 8; c += 2) {
        uint32_t packed[16];
#pragma unroll
        for (int h = 0; h < 2; ++h)
#pragma unroll
          for (int i = 0; i < 16; i += 2) {
            float x0, x1;
            unpack_f32x2(fma_f32x2(pack_f32x2(__uint_as_float(sr[c + h][i]), __uint_as_float(sr[c + h][i + 1])), scale2, negm2),
                         x0, x1);
            const float p0 = exp2f(x0), p1 = exp2f(x1);
            sums[(i >> 1) & 3] += p0 + p1;
            packed[h * 8 + (i >> 1)] = pack_f16(p0, p1);
          }
        tmem_st16(taddr + (c >> 1) * 16, packed);
      }
      l += (sums[0] + sums[1]) + (sums[2] + sums[3]);
      mbar_arrive(&xu_done[u]);
      tmem_st_wait();
      tc_fence_before_sync();
      mbar_arrive(&p_ready[u]);
    }
    if (ok && n_tiles > 0) ok = __all_sync(0xffffffffu, mbar_wait(&o_done[u], (n_tiles - 1) & 1) && *abort_flag == 0);
    if (ok) {
      tc_fence_after_sync();
      const float inv = l == 0.f ? 0.f : vf / l;
      __nv_bfloat16* dst = p.out + (static_cast<size_t>(q_begin + (live ? row : 0)) * p.hq + hk * G + hd) * kD;
#pragma unroll 1
      for (int ch = 0; ch < kD / 16; ++ch) {
        uint32_t o[16];
        if (n_tiles > 0) {
          tmem_ld16(taddr + kTmemO + ch * 16, o);
          tmem_ld_wait();
        } else {
#pragma unroll
          for (int i = 0; i < 16; ++i) o[i] = 0u;
        }
        if (live) {
#pragma unroll
          for (int w = 0; w < 2; ++w) {                      // words of channels 0 4 1 5 2 6 3 7
            auto at = [&](int i) { return l == 0.f ? 0.f : __uint_as_float(o[8 * w + i]) * inv; };
            *reinterpret_cast<uint4*>(dst + ch * 16 + 8 * w) = make_uint4(
                pack_bf16(at(0), at(2)), pack_bf16(at(4), at(6)), pack_bf16(at(1), at(3)), pack_bf16(at(5), at(7)));
          }
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
    tmem_dealloc(tmem_base, kTmemCols);
  }
}

}  // namespace

extern "C" {

int xv_kv4_prefill_tc(const void* q, const void* k_cache, const void* v_cache, const int* block_tables, const int* cu_q,
                      const int* kv_lens, void* out, int seq_begin, int num_seqs, int max_q_len, int total_rows, int hq,
                      int hkv, int d, int block_size, int max_blocks, int num_blocks, float scale, int* status,
                      cudaStream_t stream) {
  if (num_seqs <= 0 || max_q_len <= 0) return 0;
  if (d != kD) return XV_ERR_UNSUPPORTED;
  if (hkv <= 0 || hq <= 0 || hq % hkv || hq / hkv > 16 || block_size <= 0 || block_size % kv4::kUnit || max_blocks <= 0 ||
      num_blocks <= 0 || hkv > 65535 || num_seqs > 65535)
    return XV_ERR_SHAPE;
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
  p.seq_begin = seq_begin; p.hq = hq; p.hkv = hkv; p.block_size = block_size; p.max_blocks = max_blocks;
  p.num_blocks = num_blocks; p.total_rows = total_rows;
  p.scale_log2 = scale * kLog2e;
  const int rows = 2 * (kBM / (hq / hkv));
  launch_pdl(kv4_prefill_tc_kernel, dim3((max_q_len + rows - 1) / rows, hkv, num_seqs), dim3(512), kSmem, stream, p);
  return cudaGetLastError() == cudaSuccess ? 0 : XV_ERR_LAUNCH;
}

}  // extern "C"
