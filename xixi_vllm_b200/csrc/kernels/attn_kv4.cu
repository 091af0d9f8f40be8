// Paged causal GQA attention over a KV cache held in 4 bits (format: common/kv4.cuh), head_dim 128.
//
//   kv4_decode_kernel  - one query row per sequence; a CTA owns (sequence, KV head, KV split), its 4 warps take 16-token
//                        units in turn. Tokens are the M rows of both products and the group's query heads (up to 8, or
//                        16 as two column tiles) the N columns, so one MMA covers 16 x 16 cache values:
//                          S^T[token, head] = s_g * (n Q^T) + c_g * sum(Q)   per channel group g
//                          O^T[channel, head] = (n - 8)^T (s_g P) + c_g^T P
//                        The MMAs see the codes as exact bf16 integers; scales and centres stay in fp32 (the scale of V
//                        is folded into P before its one rounding to bf16). Codes go from global memory to MMA operands
//                        in registers: K's lanes own 16-byte pieces of a row, V's lanes pair two tokens with PRMT.
//   kv4_combine_kernel - joins the splits.
//   kv4_prefill_kernel - packed query chunks: 64 query rows of one head per CTA, KV tiles of 64 tokens dequantised to
//                        bf16 in shared memory.

#include <cuda_bf16.h>
#include <cuda_runtime.h>
#include <math_constants.h>

#include "../common/kv4.cuh"
#include "../common/launch.cuh"
#include "../common/ptx.cuh"
#include "xv_cuda.h"

namespace {

using namespace xv;

constexpr int kD = kv4::kD;
constexpr int kIdDecode = 10, kIdPrefill = 11;
constexpr float kLog2e = 1.4426950408889634f;
constexpr int kDecWarps = 4;

struct Params {
  const __nv_bfloat16* q;
  const uint8_t* k_cache;
  const uint8_t* v_cache;
  const int* block_tables;
  const int* cu_q;
  const int* kv_lens;
  __nv_bfloat16* out;
  float* ws_o;      // [seq, hq, split, 128]
  float* ws_lse;    // [seq, hq, split]
  int* status;
  int hq, hkv, block_size, max_blocks, num_blocks, splits, seq_begin, total_rows;
  float scale_log2;
};

// Page of a block-table entry; an entry outside the cache is recorded and replaced by page 0.
__device__ __forceinline__ int page_of(const Params& p, int b, int entry, int id) {
  int blk = __ldg(p.block_tables + static_cast<size_t>(b) * p.max_blocks + entry);
  if (static_cast<unsigned>(blk) >= static_cast<unsigned>(p.num_blocks)) {
    report_status(p.status, id, kBadIndex);
    blk = 0;
  }
  return blk;
}

// Cached tokens of a sequence, never more than its block table can name.
__device__ __forceinline__ int kv_len_of(const Params& p, int b, int id) {
  const int n = p.kv_lens[b];
  const long long most = static_cast<long long>(p.max_blocks) * p.block_size;
  if (n > most) {
    if (threadIdx.x == 0) report_status(p.status, id, kBadIndex);
    return static_cast<int>(most);
  }
  return n < 0 ? 0 : n;
}

__device__ __forceinline__ uint32_t movmatrix_trans(uint32_t a) {
  uint32_t d;
  asm volatile("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(d) : "r"(a));
  return d;
}

// NT: column tiles of 8 query heads.
template <int NT>
__global__ void __launch_bounds__(kDecWarps * 32) kv4_decode_kernel(const Params p) {
  grid_dep_launch();
  grid_dep_wait();
  __shared__ float sm_o[kDecWarps][8 * NT][kD];
  __shared__ float sm_m[kDecWarps][8 * NT], sm_l[kDecWarps][8 * NT];
  const int split = blockIdx.x, h = blockIdx.y, b = blockIdx.z;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int g = lane >> 2, t = lane & 3;
  const int G = p.hq / p.hkv;
  const int kv_len = kv_len_of(p, b, kIdDecode);
  const int tiles = (kv_len + 15) / 16;
  const int per = (tiles + p.splits - 1) / p.splits;
  const int tile1 = min((split + 1) * per, tiles);
  const int units_per_page = p.block_size / kv4::kUnit;

  // Q as the B operand: MMA (word w, half hf) of lane (g, t) multiplies channels 32 t + 8 w + 2 hf + {0, 4, 1, 5}.
  uint32_t qf[NT][4][2][2];
  float qs[NT][2][2];      // sum of Q over each group for heads 2t, 2t + 1 of the tile
#pragma unroll
  for (int nt = 0; nt < NT; ++nt) {
    const int head = nt * 8 + g;
    uint4 raw[4];
    const uint4* src = reinterpret_cast<const uint4*>(p.q + (static_cast<size_t>(b) * p.hq + h * G + head) * kD + 32 * t);
    float sum[2] = {0.f, 0.f};
#pragma unroll
    for (int w = 0; w < 4; ++w) {
      raw[w] = head < G ? __ldg(src + w) : make_uint4(0, 0, 0, 0);
      const uint32_t r[4] = {raw[w].x, raw[w].y, raw[w].z, raw[w].w};
#pragma unroll
      for (int hf = 0; hf < 2; ++hf) {
        qf[nt][w][hf][0] = __byte_perm(r[hf], r[hf + 2], 0x5410);     // channels 2 hf, 2 hf + 4
        qf[nt][w][hf][1] = __byte_perm(r[hf], r[hf + 2], 0x7632);     // channels 2 hf + 1, 2 hf + 5
      }
#pragma unroll
      for (int i = 0; i < 4; ++i) sum[w & 1] += __uint_as_float(r[i] << 16) + __uint_as_float(r[i] & 0xffff0000u);
    }
#pragma unroll
    for (int gr = 0; gr < 2; ++gr) {
      sum[gr] += __shfl_xor_sync(0xffffffffu, sum[gr], 1);
      sum[gr] += __shfl_xor_sync(0xffffffffu, sum[gr], 2);
      qs[nt][gr][0] = __shfl_sync(0xffffffffu, sum[gr], (2 * t) * 4);
      qs[nt][gr][1] = __shfl_sync(0xffffffffu, sum[gr], (2 * t + 1) * 4);
    }
  }

  float o[NT][2][4][4];            // [group][MMA]: rows g, g + 8 = channels 16 g + 8 group + 2 i + {0, 1}; heads 2t, 2t+1
  float cen[NT][2][2];             // sum of P * centre, this lane's tokens
  float m[NT][2], l[NT][2];
#pragma unroll
  for (int nt = 0; nt < NT; ++nt) {
#pragma unroll
    for (int gr = 0; gr < 2; ++gr) {
#pragma unroll
      for (int i = 0; i < 4; ++i) o[nt][gr][i][0] = o[nt][gr][i][1] = o[nt][gr][i][2] = o[nt][gr][i][3] = 0.f;
      cen[nt][gr][0] = cen[nt][gr][1] = 0.f;
    }
    m[nt][0] = m[nt][1] = -CUDART_INF_F;
    l[nt][0] = l[nt][1] = 0.f;
  }

  for (int tile = split * per + warp; tile < tile1; tile += kDecWarps) {
    const int blk = page_of(p, b, tile / units_per_page, kIdDecode);
    const size_t unit = (static_cast<size_t>(blk) * p.hkv + h) * units_per_page * kv4::kUnitBytes +
                        static_cast<size_t>(tile % units_per_page) * kv4::kUnitBytes;
    const uint8_t* ku = p.k_cache + unit;
    const uint8_t* vu = p.v_cache + unit;
    const uint4 k0 = __ldg(reinterpret_cast<const uint4*>(ku + g * 64 + t * 16));
    const uint4 k1 = __ldg(reinterpret_cast<const uint4*>(ku + (g + 8) * 64 + t * 16));
    const uint2 kp0 = __ldg(reinterpret_cast<const uint2*>(ku + kv4::kParBase + g * 8));
    const uint2 kp1 = __ldg(reinterpret_cast<const uint2*>(ku + kv4::kParBase + (g + 8) * 8));
    uint2 vp0 = __ldg(reinterpret_cast<const uint2*>(vu + kv4::kParBase + g * 8));
    uint2 vp1 = __ldg(reinterpret_cast<const uint2*>(vu + kv4::kParBase + (g + 8) * 8));
    uint2 vw[4];
#pragma unroll
    for (int i = 0; i < 4; ++i)      // tokens 2t, 2t + 1, 2t + 8, 2t + 9
      vw[i] = __ldg(reinterpret_cast<const uint2*>(vu + (2 * t + (i & 1) + 8 * (i >> 1)) * 64 + g * 8));

    const uint32_t ka[4] = {k0.x, k0.y, k0.z, k0.w}, kb[4] = {k1.x, k1.y, k1.z, k1.w};
    const bool in0 = tile * 16 + g < kv_len, in1 = tile * 16 + g + 8 < kv_len;
    if (!in0) vp0 = make_uint2(0u, 0u);      // rows past the end: P is 0 and whatever parameters an earlier owner of the
    if (!in1) vp1 = make_uint2(0u, 0u);      // page left (NaN among them) must not reach the sums; codes are always finite
    const uint32_t kpar[2][2] = {{kp0.x, kp1.x}, {kp0.y, kp1.y}}, vpar[2][2] = {{vp0.x, vp1.x}, {vp0.y, vp1.y}};
    uint32_t pf[NT][2][2];           // P * s_g as the B operand of the second product
#pragma unroll
    for (int nt = 0; nt < NT; ++nt) {
      float s[2][4] = {{0.f, 0.f, 0.f, 0.f}, {0.f, 0.f, 0.f, 0.f}};
#pragma unroll
      for (int w = 0; w < 4; ++w)
#pragma unroll
        for (int hf = 0; hf < 2; ++hf) {
          const uint32_t a[4] = {kv4::biased(ka[w], 8 * hf), kv4::biased(kb[w], 8 * hf), kv4::biased(ka[w], 8 * hf + 4),
                                 kv4::biased(kb[w], 8 * hf + 4)};
          mma_bf16_16816(s[w & 1], a, qf[nt][w][hf][0], qf[nt][w][hf][1]);
        }
      float x[4];                    // (token g: heads 2t, 2t+1), (token g + 8: the same)
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        const int row = e >> 1, hd = e & 1;
        const float s0 = kv4::par_s(kpar[0][row]), s1 = kv4::par_s(kpar[1][row]);
        const float c0 = kv4::par_c(kpar[0][row]) - kv4::kBias * s0, c1 = kv4::par_c(kpar[1][row]) - kv4::kBias * s1;
        x[e] = (s0 * s[0][e] + c0 * qs[nt][0][hd]) + (s1 * s[1][e] + c1 * qs[nt][1][hd]);
        x[e] = (row ? in1 : in0) ? x[e] * p.scale_log2 : -CUDART_INF_F;
      }
#pragma unroll
      for (int hd = 0; hd < 2; ++hd) {
        float mx = fmaxf(x[hd], x[2 + hd]);
        mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 4));
        mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 8));
        mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 16));
        const float mn = fmaxf(m[nt][hd], mx), base = mn == -CUDART_INF_F ? 0.f : mn;
        const float cr = exp2f(m[nt][hd] - base);
        m[nt][hd] = mn;
        l[nt][hd] *= cr;
#pragma unroll
        for (int gr = 0; gr < 2; ++gr) {
          cen[nt][gr][hd] *= cr;
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            o[nt][gr][i][hd] *= cr;
            o[nt][gr][i][2 + hd] *= cr;
          }
        }
        x[hd] = exp2f(x[hd] - base);
        x[2 + hd] = exp2f(x[2 + hd] - base);
        l[nt][hd] += x[hd] + x[2 + hd];
      }
#pragma unroll
      for (int gr = 0; gr < 2; ++gr) {
        const float s0 = kv4::par_s(vpar[gr][0]), s1 = kv4::par_s(vpar[gr][1]);
        pf[nt][gr][0] = movmatrix_trans(pack_bf16(x[0] * s0, x[1] * s0));
        pf[nt][gr][1] = movmatrix_trans(pack_bf16(x[2] * s1, x[3] * s1));
        const float c0 = kv4::par_c(vpar[gr][0]), c1 = kv4::par_c(vpar[gr][1]);
        cen[nt][gr][0] += x[0] * c0 + x[2] * c1;
        cen[nt][gr][1] += x[1] * c0 + x[3] * c1;
      }
    }
#pragma unroll
    for (int gr = 0; gr < 2; ++gr) {
      const uint32_t w0 = gr ? vw[0].y : vw[0].x, w1 = gr ? vw[1].y : vw[1].x, w2 = gr ? vw[2].y : vw[2].x,
                     w3 = gr ? vw[3].y : vw[3].x;
#pragma unroll
      for (int hl = 0; hl < 2; ++hl) {               // low / high half of the word: channels 0-3 / 4-7
        const uint32_t sel = hl ? 0x7632 : 0x5410;
        const uint32_t u0 = __byte_perm(w0, w1, sel), u1 = __byte_perm(w2, w3, sel);
#pragma unroll
        for (int i = 0; i < 2; ++i) {
          const uint32_t a[4] = {kv4::centred(kv4::biased(u0, 8 * i)), kv4::centred(kv4::biased(u0, 8 * i + 4)),
                                 kv4::centred(kv4::biased(u1, 8 * i)), kv4::centred(kv4::biased(u1, 8 * i + 4))};
#pragma unroll
          for (int nt = 0; nt < NT; ++nt) mma_bf16_16816(o[nt][gr][hl * 2 + i], a, pf[nt][gr][0], pf[nt][gr][1]);
        }
      }
    }
  }

  // Sums over the token lanes, then the warps through shared memory.
#pragma unroll
  for (int nt = 0; nt < NT; ++nt)
#pragma unroll
    for (int hd = 0; hd < 2; ++hd) {
#pragma unroll
      for (int x = 4; x <= 16; x <<= 1) {
        l[nt][hd] += __shfl_xor_sync(0xffffffffu, l[nt][hd], x);
        cen[nt][0][hd] += __shfl_xor_sync(0xffffffffu, cen[nt][0][hd], x);
        cen[nt][1][hd] += __shfl_xor_sync(0xffffffffu, cen[nt][1][hd], x);
      }
      const int head = nt * 8 + 2 * t + hd;
#pragma unroll
      for (int gr = 0; gr < 2; ++gr)
#pragma unroll
        for (int i = 0; i < 4; ++i)
          *reinterpret_cast<float2*>(&sm_o[warp][head][16 * g + 8 * gr + 2 * i]) =
              make_float2(o[nt][gr][i][hd] + cen[nt][gr][hd], o[nt][gr][i][2 + hd] + cen[nt][gr][hd]);
      if (g == 0) {
        sm_m[warp][head] = m[nt][hd];
        sm_l[warp][head] = l[nt][hd];
      }
    }
  __syncthreads();
  for (int idx = threadIdx.x; idx < G * kD; idx += blockDim.x) {
    const int r = idx / kD, d = idx - r * kD;
    float M = -CUDART_INF_F;
#pragma unroll
    for (int w = 0; w < kDecWarps; ++w) M = fmaxf(M, sm_m[w][r]);
    const float base = M == -CUDART_INF_F ? 0.f : M;     // nothing seen, or nothing but NaN: sums decide
    float L = 0.f, acc = 0.f;
#pragma unroll
    for (int w = 0; w < kDecWarps; ++w) {
      const float sc = exp2f(sm_m[w][r] - base);
      L += sm_l[w][r] * sc;
      acc += sm_o[w][r][d] * sc;
    }
    const float val = L == 0.f ? 0.f : acc / L;
    const size_t row = static_cast<size_t>(b) * p.hq + h * G + r;
    if (p.splits == 1) {
      p.out[row * kD + d] = __float2bfloat16(val);
    } else {
      p.ws_o[(row * p.splits + split) * kD + d] = val;
      if (d == 0) p.ws_lse[row * p.splits + split] = L == 0.f ? -CUDART_INF_F : base + log2f(L);
    }
  }
}

// out[seq, head, :] = sum_s w_s * O_s with w_s = 2^(lse_s - max) / sum; a row that no split saw anything of is zero.
__global__ void kv4_combine_kernel(const float* __restrict__ ws_o, const float* __restrict__ ws_lse,
                                   __nv_bfloat16* __restrict__ out, int splits) {
  grid_dep_launch();
  grid_dep_wait();
  const size_t row = blockIdx.x;      // seq * hq + head
  const int d = threadIdx.x;
  float M = -CUDART_INF_F;
  for (int s = 0; s < splits; ++s) M = fmaxf(M, ws_lse[row * splits + s]);
  float L = 0.f, acc = 0.f;
  for (int s = 0; s < splits; ++s) {
    const float e = ws_lse[row * splits + s];
    const float w = e == -CUDART_INF_F ? 0.f : exp2f(e - (M == -CUDART_INF_F ? 0.f : M));   // NaN stays NaN
    L += w;
    acc += w * ws_o[(row * splits + s) * kD + d];
  }
  out[row * kD + d] = __float2bfloat16(L == 0.f ? 0.f : acc / L);
}

// ------------------------------------------------------------------------------------------
// Prompt chunks
// ------------------------------------------------------------------------------------------
constexpr int kPfM = 64, kPfN = 64, kPfWarps = 4, kRowBytes = kD * 2;
constexpr int kPfTile = kPfN * kRowBytes;                       // 16 KiB
constexpr int kPfSmem = kPfM * kRowBytes + 2 * kPfTile;         // Q, K, V: 48 KiB

// Byte offset of 16-byte chunk c of row r inside a swizzled tile with 256-byte rows.
__device__ __forceinline__ uint32_t swz(int r, int c) { return static_cast<uint32_t>(r * kRowBytes + ((c ^ (r & 7)) << 4)); }

// Eight channels of one word as bf16: c + s * (n - 8), rounded once.
__device__ __forceinline__ uint4 dequant8(uint32_t w, uint32_t par) {
  const uint32_t s2 = __byte_perm(par, par, 0x1010), c2 = __byte_perm(par, par, 0x3232);
  const __nv_bfloat162 s = *reinterpret_cast<const __nv_bfloat162*>(&s2), c = *reinterpret_cast<const __nv_bfloat162*>(&c2);
  uint32_t v[4];
#pragma unroll
  for (int j = 0; j < 4; ++j) {                                  // channels j and j + 4
    const uint32_t n = kv4::centred(kv4::biased(w, 4 * j));
    const __nv_bfloat162 r = __hfma2(*reinterpret_cast<const __nv_bfloat162*>(&n), s, c);
    v[j] = *reinterpret_cast<const uint32_t*>(&r);
  }
  return make_uint4(__byte_perm(v[0], v[1], 0x5410), __byte_perm(v[2], v[3], 0x5410), __byte_perm(v[0], v[1], 0x7632),
                    __byte_perm(v[2], v[3], 0x7632));
}

__global__ void __launch_bounds__(kPfWarps * 32) kv4_prefill_kernel(const Params p) {
  grid_dep_launch();
  grid_dep_wait();
  extern __shared__ __align__(128) uint8_t smem[];
  const int head = blockIdx.y, b = p.seq_begin + blockIdx.z;
  const int q_begin = p.cu_q[b];
  int q_len = p.cu_q[b + 1] - q_begin;
  const int row0 = blockIdx.x * kPfM;
  if (q_begin < 0 || q_len < 0 || q_len > p.total_rows - q_begin) {
    if (threadIdx.x == 0) report_status(p.status, kIdPrefill, kBadIndex);
    return;
  }
  if (row0 >= q_len) return;
  const int kv_len = kv_len_of(p, b, kIdPrefill);
  const int pos0 = kv_len - q_len;                    // absolute position of query row 0 (negative rows see nothing)
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int g = lane >> 2, t = lane & 3;
  const int hk = head / (p.hq / p.hkv);
  const int rows_here = min(kPfM, q_len - row0);
  const int n_kv = max(0, min(kv_len, pos0 + row0 + rows_here));
  const int n_tiles = (n_kv + kPfN - 1) / kPfN;
  const int units_per_page = p.block_size / kv4::kUnit;

  uint8_t* sq = smem;
  uint8_t* sk = smem + kPfM * kRowBytes;
  uint8_t* sv = sk + kPfTile;
  {
    const size_t ld = static_cast<size_t>(p.hq) * kD;
    const __nv_bfloat16* qb = p.q + (static_cast<size_t>(q_begin) + row0) * ld + static_cast<size_t>(head) * kD;
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      const int c = threadIdx.x + 128 * j, r = c >> 4, ch = c & 15;
      const bool ok = r < rows_here;
      cp_async16_zfill(sq + swz(r, ch), qb + (ok ? static_cast<size_t>(r) * ld + ch * 8 : 0), ok);
    }
    cp_async_commit();
  }
  // Thread i of a tile: codes of row i / 2, 32 of its 64 bytes, of K and of V.
  const int lr = threadIdx.x >> 1, lh = threadIdx.x & 1;
  uint4 kc[2], vc[2];
  uint2 kp, vp;
  auto fetch = [&](int j) {
    const int tok = j * kPfN + lr;
    kp = vp = make_uint2(0u, 0u);
    kc[0] = kc[1] = vc[0] = vc[1] = make_uint4(0u, 0u, 0u, 0u);
    if (tok < n_kv) {
      const int blk = page_of(p, b, tok / p.block_size, kIdPrefill);
      const int r = tok % p.block_size;
      const size_t unit = (static_cast<size_t>(blk) * p.hkv + hk) * units_per_page * kv4::kUnitBytes +
                          static_cast<size_t>(r / kv4::kUnit) * kv4::kUnitBytes;
      const size_t co = unit + (r % kv4::kUnit) * kv4::kCodeRow + lh * 32;
      const size_t po = unit + kv4::kParBase + (r % kv4::kUnit) * kv4::kParRow;
      kc[0] = __ldg(reinterpret_cast<const uint4*>(p.k_cache + co));
      kc[1] = __ldg(reinterpret_cast<const uint4*>(p.k_cache + co + 16));
      vc[0] = __ldg(reinterpret_cast<const uint4*>(p.v_cache + co));
      vc[1] = __ldg(reinterpret_cast<const uint4*>(p.v_cache + co + 16));
      kp = __ldg(reinterpret_cast<const uint2*>(p.k_cache + po));
      vp = __ldg(reinterpret_cast<const uint2*>(p.v_cache + po));
    }
  };
  auto put = [&](uint8_t* tile, const uint4 (&c)[2], uint2 par) {
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      const uint32_t w[4] = {c[i].x, c[i].y, c[i].z, c[i].w};
#pragma unroll
      for (int k = 0; k < 4; ++k)
        *reinterpret_cast<uint4*>(tile + swz(lr, lh * 8 + i * 4 + k)) = dequant8(w[k], (k & 1) ? par.y : par.x);
    }
  };
  fetch(0);

  float o[16][4];
#pragma unroll
  for (int i = 0; i < 16; ++i) o[i][0] = o[i][1] = o[i][2] = o[i][3] = 0.f;
  float m0 = -CUDART_INF_F, m1 = -CUDART_INF_F, l0 = 0.f, l1 = 0.f;
  uint32_t qf[8][4];
  const int my_pos0 = pos0 + row0 + warp * 16 + g;     // position of row g; row g + 8 is + 8
  cp_async_wait<0>();
  __syncthreads();
  {
    const int mi = lane >> 3;
    const int r = warp * 16 + ((mi & 1) << 3) + (lane & 7);
#pragma unroll
    for (int kk = 0; kk < 8; ++kk) ldmatrix_x4(qf[kk], smem_u32(sq) + swz(r, 2 * kk + (mi >> 1)));
  }

  for (int j = 0; j < n_tiles; ++j) {
    put(sk, kc, kp);
    put(sv, vc, vp);
    if (j + 1 < n_tiles) fetch(j + 1);
    __syncthreads();
    const uint32_t kb = smem_u32(sk), vb = smem_u32(sv);
    const int tile_k0 = j * kPfN;
    if (tile_k0 <= my_pos0 - g + 15) {                 // warp-uniform: some row of the warp sees this tile
      float s[8][4];
#pragma unroll
      for (int i = 0; i < 8; ++i) s[i][0] = s[i][1] = s[i][2] = s[i][3] = 0.f;
      {
        const int mi = lane >> 3;
        const int r = ((mi >> 1) << 3) + (lane & 7);
#pragma unroll
        for (int kk = 0; kk < 8; ++kk)
#pragma unroll
          for (int jp = 0; jp < 4; ++jp) {
            uint32_t kf[4];
            ldmatrix_x4(kf, kb + swz(jp * 16 + r, 2 * kk + (mi & 1)));
            mma_bf16_16816(s[2 * jp], qf[kk], kf[0], kf[1]);
            mma_bf16_16816(s[2 * jp + 1], qf[kk], kf[2], kf[3]);
          }
      }
      float mx0 = -CUDART_INF_F, mx1 = -CUDART_INF_F;
#pragma unroll
      for (int nt = 0; nt < 8; ++nt)
#pragma unroll
        for (int e = 0; e < 2; ++e) {
          const int key = tile_k0 + nt * 8 + 2 * t + e;
          const bool in = key < n_kv;
          s[nt][e] = (in && key <= my_pos0) ? s[nt][e] * p.scale_log2 : -CUDART_INF_F;
          s[nt][2 + e] = (in && key <= my_pos0 + 8) ? s[nt][2 + e] * p.scale_log2 : -CUDART_INF_F;
          mx0 = fmaxf(mx0, s[nt][e]);
          mx1 = fmaxf(mx1, s[nt][2 + e]);
        }
      mx0 = fmaxf(mx0, __shfl_xor_sync(0xffffffffu, mx0, 1));
      mx0 = fmaxf(mx0, __shfl_xor_sync(0xffffffffu, mx0, 2));
      mx1 = fmaxf(mx1, __shfl_xor_sync(0xffffffffu, mx1, 1));
      mx1 = fmaxf(mx1, __shfl_xor_sync(0xffffffffu, mx1, 2));
      const float mn0 = fmaxf(m0, mx0), mn1 = fmaxf(m1, mx1);
      const float base0 = mn0 == -CUDART_INF_F ? 0.f : mn0, base1 = mn1 == -CUDART_INF_F ? 0.f : mn1;
      const float cr0 = exp2f(m0 - base0), cr1 = exp2f(m1 - base1);
      m0 = mn0;
      m1 = mn1;
      float ps0 = 0.f, ps1 = 0.f;
#pragma unroll
      for (int nt = 0; nt < 8; ++nt) {
        s[nt][0] = exp2f(s[nt][0] - base0);
        s[nt][1] = exp2f(s[nt][1] - base0);
        s[nt][2] = exp2f(s[nt][2] - base1);
        s[nt][3] = exp2f(s[nt][3] - base1);
        ps0 += s[nt][0] + s[nt][1];
        ps1 += s[nt][2] + s[nt][3];
      }
      l0 = l0 * cr0 + ps0;
      l1 = l1 * cr1 + ps1;
#pragma unroll
      for (int i = 0; i < 16; ++i) {
        o[i][0] *= cr0; o[i][1] *= cr0; o[i][2] *= cr1; o[i][3] *= cr1;
      }
      {
        const int mi = lane >> 3;
        const int r = ((mi & 1) << 3) + (lane & 7);
#pragma unroll
        for (int ks = 0; ks < 4; ++ks) {
          const uint32_t pf[4] = {pack_bf16(s[2 * ks][0], s[2 * ks][1]), pack_bf16(s[2 * ks][2], s[2 * ks][3]),
                                  pack_bf16(s[2 * ks + 1][0], s[2 * ks + 1][1]), pack_bf16(s[2 * ks + 1][2], s[2 * ks + 1][3])};
#pragma unroll
          for (int jd = 0; jd < 8; ++jd) {
            uint32_t vf[4];
            ldmatrix_x4_trans(vf, vb + swz(ks * 16 + r, 2 * jd + (mi >> 1)));
            mma_bf16_16816(o[2 * jd], pf, vf[0], vf[1]);
            mma_bf16_16816(o[2 * jd + 1], pf, vf[2], vf[3]);
          }
        }
      }
    }
    __syncthreads();    // everyone is done with the tile before the next one overwrites it
  }

  l0 += __shfl_xor_sync(0xffffffffu, l0, 1);
  l0 += __shfl_xor_sync(0xffffffffu, l0, 2);
  l1 += __shfl_xor_sync(0xffffffffu, l1, 1);
  l1 += __shfl_xor_sync(0xffffffffu, l1, 2);
  const float inv0 = l0 == 0.f ? 0.f : 1.f / l0, inv1 = l1 == 0.f ? 0.f : 1.f / l1;
  const int r0 = row0 + warp * 16 + g, r1 = r0 + 8;
  const size_t ld = static_cast<size_t>(p.hq) * kD;
  __nv_bfloat16* ob = p.out + static_cast<size_t>(q_begin) * ld + static_cast<size_t>(head) * kD;
#pragma unroll
  for (int nt = 0; nt < 16; ++nt) {
    const int d0 = nt * 8 + 2 * t;
    if (r0 < q_len)
      *reinterpret_cast<uint32_t*>(ob + static_cast<size_t>(r0) * ld + d0) = pack_bf16(o[nt][0] * inv0, o[nt][1] * inv0);
    if (r1 < q_len)
      *reinterpret_cast<uint32_t*>(ob + static_cast<size_t>(r1) * ld + d0) = pack_bf16(o[nt][2] * inv1, o[nt][3] * inv1);
  }
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
  p.scale_log2 = scale * kLog2e;
  p.status = status;
  return 0;
}

inline int launch_ok() { return cudaGetLastError() == cudaSuccess ? 0 : XV_ERR_LAUNCH; }

}  // namespace

extern "C" {

// KV splits so that a small batch still fills the GPU; from launch-shape constants only (never from sequence lengths),
// so a captured graph keeps its shape.
int xv_kv4_decode_splits(int num_seqs, int hkv, int num_sms, int max_tokens_per_seq) {
  const int ctas = max(1, num_seqs * hkv);
  const int want = (4 * num_sms + ctas - 1) / ctas, by_len = max(1, max_tokens_per_seq / 256);
  return max(1, min(min(want, by_len), 64));
}

long long xv_kv4_decode_workspace_bytes(int num_seqs, int hq, int splits) {
  return splits <= 1 ? 0 : static_cast<long long>(num_seqs) * hq * splits * (kD + 1) * 4;
}

int xv_kv4_decode(const void* q, const void* k_cache, const void* v_cache, const int* block_tables, const int* kv_lens,
                  void* out, int num_seqs, int hq, int hkv, int d, int block_size, int max_blocks, int num_blocks,
                  float scale, int splits, void* workspace, long long workspace_bytes, int* status, cudaStream_t stream) {
  if (num_seqs <= 0) return 0;
  Params p;
  if (int rc = fill(p, q, k_cache, v_cache, block_tables, kv_lens, out, hq, hkv, d, block_size, max_blocks, num_blocks,
                    scale, status))
    return rc;
  if (hq / hkv > 16 || hkv > 65535 || num_seqs > 65535 || splits < 1) return XV_ERR_SHAPE;
  if (xv_kv4_decode_workspace_bytes(num_seqs, hq, splits) > workspace_bytes) return XV_ERR_WORKSPACE;
  p.splits = splits;
  p.ws_o = static_cast<float*>(workspace);
  p.ws_lse = splits > 1 ? p.ws_o + static_cast<size_t>(num_seqs) * hq * splits * kD : nullptr;
  const dim3 grid(splits, hkv, num_seqs);
  launch_pdl(hq / hkv <= 8 ? kv4_decode_kernel<1> : kv4_decode_kernel<2>, grid, dim3(kDecWarps * 32), 0, stream, p);
  if (int rc = launch_ok()) return rc;
  if (splits > 1) {
    launch_pdl(kv4_combine_kernel, dim3(num_seqs * hq), dim3(kD), 0, stream, p.ws_o, p.ws_lse, p.out, splits);
    return launch_ok();
  }
  return 0;
}

int xv_kv4_prefill(const void* q, const void* k_cache, const void* v_cache, const int* block_tables, const int* cu_q,
                   const int* kv_lens, void* out, int seq_begin, int num_seqs, int max_q_len, int total_rows, int hq,
                   int hkv, int d, int block_size, int max_blocks, int num_blocks, float scale, int* status,
                   cudaStream_t stream) {
  if (num_seqs <= 0 || max_q_len <= 0) return 0;
  Params p;
  if (int rc = fill(p, q, k_cache, v_cache, block_tables, kv_lens, out, hq, hkv, d, block_size, max_blocks, num_blocks,
                    scale, status))
    return rc;
  if (hq > 65535 || num_seqs > 65535) return XV_ERR_SHAPE;
  p.cu_q = cu_q;
  p.seq_begin = seq_begin;
  p.total_rows = total_rows;
  launch_pdl(kv4_prefill_kernel, dim3((max_q_len + kPfM - 1) / kPfM, hq, num_seqs), dim3(kPfWarps * 32), kPfSmem, stream, p);
  return launch_ok();
}

}  // extern "C"
