// A block's residual update, RMS norm and modulation as one step:
//
//   stream = bf16(x + gate_b * y)                                   (no gate: x + y)
//   h      = stream * rstd * (1 + w) * (1 + sc_b) + sh_b            rstd = (mean_k stream^2 + eps)^-1/2
//
//   residual_quant   h rotated by blocks of 128 and quantised to int8 with one scale per token (sampling:
//                    what the next quantised Linear reads); h itself never reaches memory
//   residual_fwd     dense bf16 h and rstd (training)
//   residual_bwd     with n = stream * rstd, g = dh * (1 + w)(1 + sc_b):
//                      d = dstream + rstd * (g - n * mean_k(g * n)),   dx = d,   dy = gate_b * d
//                    and, where asked for, the sums over a sample's rows  D = sum d*y,  S = sum dh*n,  H = sum dh:
//                      dgate_b = D,  dsc_b = S (1 + w),  dsh_b = H,  dw = sum_b S (1 + sc_b)
//
// Everything between the loads and the stores is fp32; the stream is rounded to bf16 once, where it is
// kept, and the norm reads the rounded values, so that the backward sees the same numbers.  b = row /
// rows_per_batch.  They move 7, 8 and 10 (12 with the sums) bytes per element; the forward and the backward without sums
// are held by HBM, the others by what follows.  A row is worked on by one CTA (its two reductions are CTA-wide); a CTA takes
// consecutive rows of one sample, so that the sample's vectors are read from L2 once per CTA and not once per row, and there
// are exactly as many CTAs as the SMs hold at once.  The quantising kernel is held to 96 registers (up to 16 bytes of a
// thread spill), so that three CTAs of 192 threads fit (at 124, two did, in 1.5 waves): that, with the shift and gate left
// as bf16 and the rotation's factor folded into the row scale, took it from 237 to 181 us.
// Measured on a B200 (copy bandwidth 6.55 TB/s), 16896 rows of 6144, gate and modulation:
//   quantising  137 us = 5.3 TB/s (0.81)      forward  138 us = 6.0 TB/s (0.92)
//   backward    187 us = 5.55 TB/s (0.85)     with every sum  280 us = 4.45 TB/s (0.68)
// (the chain of the two single kernels, cold: quantising 440 us, forward 248, forward and backward 630 against 336 here).
// The quantising kernel executes 22 instructions per element, 4 warps to an SM quarter, and issues in 49 % of the cycles;
// the largest stall is on shuffles and shared memory (the sample's vectors).  The backward with sums keeps them in shared
// memory above 4096 columns: one CTA of 12 warps per SM at 128 registers, 53 % of the shared-memory rate, 39 % issue, most
// of the stalls on shared memory; HBM waits for it.
#include <atomic>

#include "k2q_common.cuh"
#include "rows_math.cuh"

namespace k2q {
namespace {

constexpr int kMaxWarps = 16;

__device__ __forceinline__ void unpack8(const uint4& r, float* v) {
  const uint32_t w[4] = {r.x, r.y, r.z, r.w};
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    v[2 * i] = __uint_as_float(w[i] << 16);
    v[2 * i + 1] = __uint_as_float(w[i] & 0xFFFF0000u);
  }
}
__device__ __forceinline__ uint4 pack8(const float* v) {
  return make_uint4(pack_bf16x2(v[0], v[1]), pack_bf16x2(v[2], v[3]), pack_bf16x2(v[4], v[5]), pack_bf16x2(v[6], v[7]));
}
__device__ __forceinline__ void load8f(const float* p, float* v) {
  const float4 a = __ldg(reinterpret_cast<const float4*>(p));
  const float4 b = __ldg(reinterpret_cast<const float4*>(p) + 1);
  v[0] = a.x; v[1] = a.y; v[2] = a.z; v[3] = a.w; v[4] = b.x; v[5] = b.y; v[6] = b.z; v[7] = b.w;
}
// Rows that another thread block may overwrite in place later: coherent loads, not kept in L1.
__device__ __forceinline__ uint4 load_row16(const __nv_bfloat16* p) { return __ldcs(reinterpret_cast<const uint4*>(p)); }
__device__ __forceinline__ uint4 load_vec16(const __nv_bfloat16* p) { return __ldg(reinterpret_cast<const uint4*>(p)); }

// maximum that keeps a NaN: a row with one gets a NaN scale, not small codes
__device__ __forceinline__ float max_nan(float a, float b) {
  float d;
  asm("max.NaN.f32 %0, %1, %2;" : "=f"(d) : "f"(a), "f"(b));
  return d;
}

__device__ __forceinline__ float max_abs3(float a, float b, float c) {
  float d;
  asm("max.NaN.abs.f32 %0, %1, %2, %3;" : "=f"(d) : "f"(a), "f"(b), "f"(c));
  return d;
}

// Sum / maximum over the CTA, the same value in every thread, in a fixed order.  One barrier: successive
// calls of a kernel alternate between two slots, so a slot is written again only behind the barrier of
// the call in between, which every reader of the slot has passed.
template <bool MAX>
__device__ __forceinline__ float cta_reduce(float v, float* slot, int warps) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) {
    const float other = __shfl_xor_sync(0xffffffffu, v, o);
    v = MAX ? max_nan(v, other) : v + other;
  }
  if ((threadIdx.x & 31) == 0) slot[threadIdx.x >> 5] = v;
  __syncthreads();
  float t = slot[0];
  for (int w = 1; w < warps; ++w) t = MAX ? max_nan(t, slot[w]) : t + slot[w];
  return t;
}

struct ResParams {
  const __nv_bfloat16* x; int64_t ldx;
  const __nv_bfloat16* y; int64_t ldy;
  const __nv_bfloat16* gate;                 // [B, K] or NULL
  const float* normw;                        // [K]
  const __nv_bfloat16* mscale;               // [B, K] or NULL
  const __nv_bfloat16* mshift;               // [B, K] or NULL
  int64_t M; int K;
  int64_t rows_per_batch; float eps;
  __nv_bfloat16* stream; int64_t lds;        // forward: written; backward: read
  int8_t* xq; float* sx;                     // quantising form
  __nv_bfloat16* h; int64_t ldh; float* rstd;
  // backward
  const __nv_bfloat16* dstream; int64_t ldds;   // or NULL
  const __nv_bfloat16* dh; int64_t lddh;        // or NULL
  __nv_bfloat16* dx; int64_t lddx;              // or NULL
  __nv_bfloat16* dy; int64_t lddy;              // or NULL
  float* part;                                  // [B, chunks, 3, K] partial sums D, S, H, or NULL
  int chunks;                                   // CTAs per sample
};

// h of 8 consecutive elements from the kept stream
__device__ __forceinline__ void norm_mod8(const ResParams& p, int64_t b, int k0, float rstd, float* v) {
  float w[8];
  load8f(p.normw + k0, w);
#pragma unroll
  for (int e = 0; e < 8; ++e) v[e] = v[e] * rstd * (1.0f + w[e]);
  if (p.mscale != nullptr) {
    float s[8];
    unpack8(load_vec16(p.mscale + b * p.K + k0), s);
#pragma unroll
    for (int e = 0; e < 8; ++e) v[e] *= 1.0f + s[e];
  }
  if (p.mshift != nullptr) {
    float s[8];
    unpack8(load_vec16(p.mshift + b * p.K + k0), s);
#pragma unroll
    for (int e = 0; e < 8; ++e) v[e] += s[e];
  }
}

// ---- sampling: rotated int8 codes -------------------------------------------------------------
// A CTA works through consecutive rows of one sample.  Its vectors are combined once, in shared memory:
//   f = (1 + w)(1 + sc) in fp32,  sh and the gate in bf16 (the rotation's normalisation enters the scale alone),
// so that a row costs one packed bf16 multiply-add per two elements for the stream and one packed fp32 one for h.  In
// odd 128-blocks f's 16-byte pieces are swapped pairwise (the bf16 vectors' four apart), so that the eight lanes of a read
// phase, which span two blocks, meet all banks.  Four
// neighbouring lanes hold a 128-block.  Lane q of the four owns the 8-element chunks q, q + 4, q + 8, q + 12 of the
// block: a warp's 16-byte accesses then cover whole 64-byte pieces, and nothing has to be staged through shared memory.
// The next row is requested before the current one is worked on.
//
// The rotation's seven butterfly stages: h = 1, 2, 4 and 32, 64 lie inside a thread, h = 8 and 16 between lanes.  A lane
// would have to fetch all 32 of its partner's values for each of the latter.  Instead, after stage 32, lane bit 0 and
// the chunk's low bit change places: of each butterfly's two results the lane keeps the one whose index bit 5 is its
// own lane bit and sends the other, 16 values; stage 8 then lies inside the thread.  Likewise 64 and 16 with the
// other bits.  In the end lane q holds the 32 consecutive elements from 32 q on.  The differences of stage 8 (16) come out
// negated in lanes with bit 0 (1) set; the caller undoes it: rotated_sign().
__device__ __forceinline__ float rotated_sign(int chunk, int q) { return __popc(chunk & q) & 1 ? -1.0f : 1.0f; }

__device__ __forceinline__ void fwht128_chunks(uint64_t (&p)[16], int q) {
  const uint64_t neg2 = pack_f32x2(-1.0f, -1.0f);
#pragma unroll
  for (int i = 0; i < 16; ++i) {
    float a, b;
    unpack_f32x2(p[i], a, b);
    p[i] = pack_f32x2(__fadd_rn(a, b), __fsub_rn(a, b));
  }
#pragma unroll
  for (int h = 1; h < 4; h <<= 1) {
#pragma unroll
    for (int i = 0; i < 16; ++i) {
      if ((i & h) == 0) {
        const uint64_t a = p[i], b = p[i + h];
        p[i] = add_f32x2(a, b);
        p[i + h] = fma_f32x2(b, neg2, a);
      }
    }
  }
#pragma unroll
  for (int h = 4; h < 16; h <<= 1) {                     // 32 and 8, then 64 and 16
    const float sgn = (q & (h >> 2)) ? -1.0f : 1.0f;
    const uint64_t sgn2 = pack_f32x2(sgn, sgn), nsgn2 = pack_f32x2(-sgn, -sgn);
#pragma unroll
    for (int i = 0; i < 16; ++i) {
      if ((i & h) == 0) {
        const uint64_t keep = fma_f32x2(p[i + h], sgn2, p[i]), send = fma_f32x2(p[i + h], nsgn2, p[i]);
        float a, b;
        unpack_f32x2(send, a, b);
        p[i] = keep;
        p[i + h] = pack_f32x2(__shfl_xor_sync(0xffffffffu, a, h >> 2), __shfl_xor_sync(0xffffffffu, b, h >> 2));
      }
    }
#pragma unroll
    for (int i = 0; i < 16; ++i) {
      if ((i & h) == 0) {
        const uint64_t keep = p[i], got = p[i + h];
        p[i] = add_f32x2(keep, got);
        p[i + h] = fma_f32x2(got, neg2, keep);
      }
    }
  }
}

// bf16 pairs, each half rounded once (the product of two bf16 values is not rounded on its own)
__device__ __forceinline__ uint32_t fma_bf16x2(uint32_t a, uint32_t b, uint32_t c) {
  uint32_t d;
  asm("fma.rn.bf16x2 %0, %1, %2, %3;" : "=r"(d) : "r"(a), "r"(b), "r"(c));
  return d;
}
__device__ __forceinline__ uint64_t widen2(uint32_t w) { return pack_f32x2(w << 16, w & 0xFFFF0000u); }



struct RowChunks { uint4 x[4], y[4]; };

// rows [r0, r1) of sample b that CTA blockIdx.x = b * chunks + chunk works on
__device__ __forceinline__ void cta_rows(const ResParams& p, int64_t& b, int64_t& r0, int64_t& r1) {
  b = blockIdx.x / p.chunks;
  const int chunk = blockIdx.x - static_cast<int>(b) * p.chunks;
  r0 = b * p.rows_per_batch + p.rows_per_batch * chunk / p.chunks;
  r1 = b * p.rows_per_batch + p.rows_per_batch * (chunk + 1) / p.chunks;
}

template <bool GATE, bool SHIFT>
__global__ void __maxnreg__(96) residual_quant_kernel(const ResParams p) {
  extern __shared__ __align__(16) float vec[];                 // f [K] | sh [K] bf16 (SHIFT) | gate [K] bf16 (GATE)
  __shared__ float red[2][kMaxWarps];
  uint32_t* s_s = reinterpret_cast<uint32_t*>(vec + p.K);
  uint32_t* s_g = s_s + (SHIFT ? p.K / 2 : 0);
  const int warps = blockDim.x >> 5;
  const int q = threadIdx.x & 3;
  const int blk = threadIdx.x >> 2;                            // 128-block of the row
  const bool own = blk < (p.K >> 7);
  const int k00 = blk * 128 + q * 8;                           // first chunk; the others 32 elements apart
  int64_t b, r0, r1;
  cta_rows(p, b, r0, r1);
  pdl_wait();

  auto fetch = [&](int64_t row, RowChunks& c) {
    if (own) {
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        c.x[j] = load_row16(p.x + row * p.ldx + k00 + 32 * j);
        c.y[j] = load_row16(p.y + row * p.ldy + k00 + 32 * j);
      }
    } else {
#pragma unroll
      for (int j = 0; j < 4; ++j) c.x[j] = c.y[j] = make_uint4(0u, 0u, 0u, 0u);
    }
  };
  RowChunks next;
  fetch(r0, next);
  for (int c = threadIdx.x; c < (p.K >> 3); c += blockDim.x) {
    const int k = 8 * c;
    float f[8];
    load8f(p.normw + k, f);
#pragma unroll
    for (int e = 0; e < 8; ++e) f[e] += 1.0f;
    if (p.mscale != nullptr) {
      float s[8];
      unpack8(load_vec16(p.mscale + b * p.K + k), s);
#pragma unroll
      for (int e = 0; e < 8; ++e) f[e] *= 1.0f + s[e];
    }
    const int swap = (k >> 7) & 1, lo = k + 4 * swap, hi = k + 4 * (swap ^ 1);
    *reinterpret_cast<float4*>(vec + lo) = make_float4(f[0], f[1], f[2], f[3]);
    *reinterpret_cast<float4*>(vec + hi) = make_float4(f[4], f[5], f[6], f[7]);
    const int at = (k ^ (32 * swap)) >> 1;
    if (SHIFT) *reinterpret_cast<uint4*>(s_s + at) = load_vec16(p.mshift + b * p.K + k);
    if (GATE) *reinterpret_cast<uint4*>(s_g + at) = load_vec16(p.gate + b * p.K + k);
  }
  __syncthreads();

  const float inv_k = 1.0f / static_cast<float>(p.K);
  const int lo = k00 + 4 * (blk & 1), hi = k00 + 4 * ((blk & 1) ^ 1);
  for (int64_t row = r0; row < r1; ++row) {
    uint64_t v[16];
    uint64_t ss2[2] = {0ull, 0ull};
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      uint4 s = next.x[j];
      const uint4 y = next.y[j];
      uint4 g = make_uint4(0x3F803F80u, 0x3F803F80u, 0x3F803F80u, 0x3F803F80u);   // one
      if (GATE && own) g = *reinterpret_cast<const uint4*>(s_g + ((k00 + 32 * (j ^ (blk & 1))) >> 1));
      s.x = fma_bf16x2(g.x, y.x, s.x); s.y = fma_bf16x2(g.y, y.y, s.y);
      s.z = fma_bf16x2(g.z, y.z, s.z); s.w = fma_bf16x2(g.w, y.w, s.w);
      if (own) *reinterpret_cast<uint4*>(p.stream + row * p.lds + k00 + 32 * j) = s;
      v[4 * j] = widen2(s.x); v[4 * j + 1] = widen2(s.y); v[4 * j + 2] = widen2(s.z); v[4 * j + 3] = widen2(s.w);
#pragma unroll
      for (int e = 0; e < 4; ++e) ss2[e & 1] = fma_f32x2(v[4 * j + e], v[4 * j + e], ss2[e & 1]);
    }
    if (row + 1 < r1) fetch(row + 1, next);
    float a0, a1, a2, a3;
    unpack_f32x2(ss2[0], a0, a1);
    unpack_f32x2(ss2[1], a2, a3);
    const float rstd = rsqrtf(cta_reduce<false>((a0 + a1) + (a2 + a3), red[0], warps) * inv_k + p.eps);
    const uint64_t rstd2 = pack_f32x2(rstd, rstd);
    if (own) {
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const ulonglong2 f0 = *reinterpret_cast<const ulonglong2*>(vec + lo + 32 * j), f1 = *reinterpret_cast<const ulonglong2*>(vec + hi + 32 * j);
        const uint64_t f[4] = {f0.x, f0.y, f1.x, f1.y};
        if (SHIFT) {
          const uint4 sv = *reinterpret_cast<const uint4*>(s_s + ((k00 + 32 * (j ^ (blk & 1))) >> 1));
          const uint64_t s[4] = {widen2(sv.x), widen2(sv.y), widen2(sv.z), widen2(sv.w)};
#pragma unroll
          for (int e = 0; e < 4; ++e) v[4 * j + e] = fma_f32x2(mul_f32x2(v[4 * j + e], rstd2), f[e], s[e]);
        } else {
#pragma unroll
          for (int e = 0; e < 4; ++e) v[4 * j + e] = mul_f32x2(mul_f32x2(v[4 * j + e], rstd2), f[e]);
        }
      }
    }
    fwht128_chunks(v, q);
    float m0 = 0.f, m1 = 0.f;
#pragma unroll
    for (int i = 0; i < 16; ++i) {
      float a, c;
      unpack_f32x2(v[i], a, c);
      if (i & 1) m1 = max_abs3(m1, a, c);
      else m0 = max_abs3(m0, a, c);
    }
    // the scale of the normalised rotation; codes straight from the values without its factor
    const float s = __fdiv_rn(max_nan(cta_reduce<true>(max_nan(m0, m1), red[1], warps) * kHadNorm, 1e-8f), 127.0f);
    const float inv = __fdividef(kHadNorm, s);
    // v / s + 1.5 * 2^23 carries the rounded code in its low byte
    const uint64_t magic2 = pack_f32x2(kRoundMagic, kRoundMagic);
    uint32_t words[8];
#pragma unroll
    for (int w = 0; w < 8; ++w) {
      const float signed_inv = inv * rotated_sign(w >> 1, q);
      const uint64_t inv2 = pack_f32x2(signed_inv, signed_inv);
      float c0, c1, c2, c3;
      unpack_f32x2(fma_f32x2(v[2 * w], inv2, magic2), c0, c1);
      unpack_f32x2(fma_f32x2(v[2 * w + 1], inv2, magic2), c2, c3);
      words[w] = prmt_b(prmt_b(__float_as_uint(c0), __float_as_uint(c1), 0x0040u), prmt_b(__float_as_uint(c2), __float_as_uint(c3), 0x0040u), 0x5410u);
    }
    if (own) {
      uint4* out = reinterpret_cast<uint4*>(p.xq + row * p.K + blk * 128 + q * 32);
      out[0] = make_uint4(words[0], words[1], words[2], words[3]);
      out[1] = make_uint4(words[4], words[5], words[6], words[7]);
    }
    if (threadIdx.x == 0) p.sx[row] = s;
  }
}

// ---- training: dense output and its backward ------------------------------------------------------
// Both: a CTA works through consecutive rows of one sample, a thread owns the same columns in all of them; the next row
// is requested before the current one is worked on, and the sample's vectors stay in registers, combined.
template <int VPT>
__global__ void __launch_bounds__(512) residual_fwd_kernel(const ResParams p) {
  __shared__ float red[2][kMaxWarps];
  const int warps = blockDim.x >> 5, nvec = p.K >> 3;
  int64_t b, r0, r1;
  cta_rows(p, b, r0, r1);
  pdl_wait();
  uint4 nx[VPT], ny[VPT];
  auto fetch = [&](int64_t row) {
#pragma unroll
    for (int i = 0; i < VPT; ++i) {
      const int c = threadIdx.x + i * blockDim.x;
      if (c < nvec) {
        nx[i] = load_row16(p.x + row * p.ldx + 8 * c);
        ny[i] = load_row16(p.y + row * p.ldy + 8 * c);
      }
    }
  };
  fetch(r0);
  int it = 0;
  for (int64_t row = r0; row < r1; ++row, it ^= 1) {
    uint4 sv[VPT];
    uint64_t ss2 = 0ull;
#pragma unroll
    for (int i = 0; i < VPT; ++i) {
      const int c = threadIdx.x + i * blockDim.x;
      if (c < nvec) {
        uint4 g = make_uint4(0x3F803F80u, 0x3F803F80u, 0x3F803F80u, 0x3F803F80u);   // one
        if (p.gate != nullptr) g = load_vec16(p.gate + b * p.K + 8 * c);
        uint4 s = nx[i];
        s.x = fma_bf16x2(g.x, ny[i].x, s.x); s.y = fma_bf16x2(g.y, ny[i].y, s.y);
        s.z = fma_bf16x2(g.z, ny[i].z, s.z); s.w = fma_bf16x2(g.w, ny[i].w, s.w);
        reinterpret_cast<uint4*>(p.stream + row * p.lds)[c] = s;
        sv[i] = s;
        const uint64_t v[4] = {widen2(s.x), widen2(s.y), widen2(s.z), widen2(s.w)};
#pragma unroll
        for (int e = 0; e < 4; ++e) ss2 = fma_f32x2(v[e], v[e], ss2);
      }
    }
    float ss, ss_odd;
    unpack_f32x2(ss2, ss, ss_odd);
    ss += ss_odd;
    if (row + 1 < r1) fetch(row + 1);
    const float rstd = rsqrtf(cta_reduce<false>(ss, red[it], warps) / static_cast<float>(p.K) + p.eps);
    if (threadIdx.x == 0) p.rstd[row] = rstd;
#pragma unroll
    for (int i = 0; i < VPT; ++i) {
      const int c = threadIdx.x + i * blockDim.x;
      if (c < nvec) {
        float v[8];
        unpack8(sv[i], v);
        norm_mod8(p, b, 8 * c, rstd, v);
        reinterpret_cast<uint4*>(p.h + row * p.ldh)[c] = pack8(v);
      }
    }
  }
}

// SUMS: each CTA adds up its rows' terms of D, S and H, in registers (one vector per thread) or in its shared memory
// (several: 96 sums would not fit beside the rows), and leaves them in its own slice of the workspace.
// Up to two vectors per thread the next row is requested before the current one is worked on, and the sample's
// (1 + w)(1 + sc) stays in registers; beyond, registers hold one row and the vectors are read again (L2).
template <int VPT, bool SUMS>
__global__ void __maxnreg__(VPT == 1 ? (SUMS ? 96 : 64) : VPT == 2 && !SUMS ? 96 : 128) residual_bwd_kernel(const ResParams p) {
  constexpr bool PRE = VPT <= 2, SHARED = SUMS && VPT > 1;
  constexpr int Y = SUMS ? VPT : 1, W = PRE ? VPT : 1, A = SUMS && !SHARED ? 1 : 0;
  extern __shared__ __align__(16) float sums[];                // SHARED: D [K], S [K], H [K]
  __shared__ float red[2][kMaxWarps];
  const int warps = blockDim.x >> 5, nvec = p.K >> 3;
  int64_t b, r0, r1;
  cta_rows(p, b, r0, r1);
  pdl_wait();
  const bool has_h = p.dh != nullptr, has_s = p.dstream != nullptr, sum_d = SUMS && p.y != nullptr;
  uint64_t acc[A ? 3 : 1][4] = {};
  uint4 n_ds[VPT], n_dh[VPT], n_st[VPT], n_y[Y];
  float n_rstd = 0.f;
#pragma unroll
  for (int i = 0; i < VPT; ++i) n_ds[i] = n_dh[i] = n_st[i] = make_uint4(0u, 0u, 0u, 0u);
#pragma unroll
  for (int i = 0; i < Y; ++i) n_y[i] = make_uint4(0u, 0u, 0u, 0u);
  auto fetch = [&](int64_t row) {
    if (has_h) n_rstd = __ldg(p.rstd + row);
#pragma unroll
    for (int i = 0; i < VPT; ++i) {
      const int c = threadIdx.x + i * blockDim.x;
      if (c < nvec) {
        if (has_h) {
          n_dh[i] = __ldcs(reinterpret_cast<const uint4*>(p.dh + row * p.lddh) + c);
          n_st[i] = __ldcs(reinterpret_cast<const uint4*>(p.stream + row * p.lds) + c);
        }
        if (has_s) n_ds[i] = __ldcs(reinterpret_cast<const uint4*>(p.dstream + row * p.ldds) + c);
        if (sum_d) n_y[SUMS ? i : 0] = __ldcs(reinterpret_cast<const uint4*>(p.y + row * p.ldy) + c);
      }
    }
  };
  auto weights = [&](int c, uint64_t* w) {
    float f[8];
    load8f(p.normw + 8 * c, f);
#pragma unroll
    for (int e = 0; e < 8; ++e) f[e] += 1.0f;
    if (p.mscale != nullptr) {
      float s[8];
      unpack8(load_vec16(p.mscale + b * p.K + 8 * c), s);
#pragma unroll
      for (int e = 0; e < 8; ++e) f[e] *= 1.0f + s[e];
    }
#pragma unroll
    for (int e = 0; e < 4; ++e) w[e] = pack_f32x2(f[2 * e], f[2 * e + 1]);
  };
  fetch(r0);                                                   // chunks <= rows_per_batch: there is a row
  uint64_t w_keep[W][4];
#pragma unroll
  for (int i = 0; i < VPT; ++i) {
    const int c = threadIdx.x + i * blockDim.x;
    if (c < nvec) {
      if (PRE) weights(c, w_keep[PRE ? i : 0]);
      if (SHARED) {
#pragma unroll
        for (int j = 0; j < 3; ++j) {
          *reinterpret_cast<float4*>(sums + j * p.K + 8 * c) = make_float4(0.f, 0.f, 0.f, 0.f);
          *reinterpret_cast<float4*>(sums + j * p.K + 8 * c + 4) = make_float4(0.f, 0.f, 0.f, 0.f);
        }
      }
    }
  }
  // sum j of this thread's columns 8c .. += v * u, or + v
  auto add = [&](int j, int c, const uint64_t* v, const uint64_t* u) {
    if (A) {
#pragma unroll
      for (int e = 0; e < 4; ++e) acc[A ? j : 0][e] = u != nullptr ? fma_f32x2(v[e], u[e], acc[A ? j : 0][e]) : add_f32x2(acc[A ? j : 0][e], v[e]);
    } else {
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        ulonglong2* at = reinterpret_cast<ulonglong2*>(sums + j * p.K + 8 * c + 4 * h);
        ulonglong2 s = *at;
        s.x = u != nullptr ? fma_f32x2(v[2 * h], u[2 * h], s.x) : add_f32x2(s.x, v[2 * h]);
        s.y = u != nullptr ? fma_f32x2(v[2 * h + 1], u[2 * h + 1], s.y) : add_f32x2(s.y, v[2 * h + 1]);
        *at = s;
      }
    }
  };
  auto widen8 = [](const uint4& r, uint64_t* v) { v[0] = widen2(r.x); v[1] = widen2(r.y); v[2] = widen2(r.z); v[3] = widen2(r.w); };
  auto narrow8 = [](const uint64_t* v) {
    float f[8];
#pragma unroll
    for (int e = 0; e < 4; ++e) unpack_f32x2(v[e], f[2 * e], f[2 * e + 1]);
    return pack8(f);
  };
  const float inv_k = 1.0f / static_cast<float>(p.K);
  int it = 0;
  for (int64_t row = r0; row < r1; ++row, it ^= 1) {
    if (!PRE && row > r0) fetch(row);
    uint4 c_ds[VPT], c_dh[VPT], c_st[VPT], c_y[Y];
    const float rstd = n_rstd;
    const uint64_t rstd2 = pack_f32x2(rstd, rstd);
    uint64_t dot2 = 0ull;
#pragma unroll
    for (int i = 0; i < VPT; ++i) {
      const int c = threadIdx.x + i * blockDim.x;
      c_ds[i] = n_ds[i]; c_dh[i] = n_dh[i]; c_st[i] = n_st[i];
      if (SUMS) c_y[SUMS ? i : 0] = n_y[SUMS ? i : 0];
      if (c < nvec) {
        uint64_t g[4], n[4], w[4];
        widen8(c_dh[i], g);
        widen8(c_st[i], n);
        if (!PRE) weights(c, w);
#pragma unroll
        for (int e = 0; e < 4; ++e) n[e] = mul_f32x2(n[e], rstd2);
        if (SUMS) {
          add(1, c, g, n);
          add(2, c, g, nullptr);
        }
#pragma unroll
        for (int e = 0; e < 4; ++e) dot2 = fma_f32x2(mul_f32x2(g[e], PRE ? w_keep[PRE ? i : 0][e] : w[e]), n[e], dot2);
      }
    }
    if (PRE && row + 1 < r1) fetch(row + 1);
    float dot = 0.f;
    if (has_h) {
      float d0, d1;
      unpack_f32x2(dot2, d0, d1);
      dot = cta_reduce<false>(d0 + d1, red[it], warps) * inv_k;
    }
    const float back = -rstd * dot;                            // n is stream * rstd: n * dot = stream * (rstd dot)
    const uint64_t back2 = pack_f32x2(back, back);
#pragma unroll
    for (int i = 0; i < VPT; ++i) {
      const int c = threadIdx.x + i * blockDim.x;
      if (c < nvec) {
        uint64_t d[4];
        widen8(c_ds[i], d);
        if (has_h) {
          uint64_t g[4], s[4], w[4];
          widen8(c_dh[i], g);
          widen8(c_st[i], s);
          if (!PRE) weights(c, w);
#pragma unroll
          for (int e = 0; e < 4; ++e)
            d[e] = fma_f32x2(fma_f32x2(s[e], back2, mul_f32x2(g[e], PRE ? w_keep[PRE ? i : 0][e] : w[e])), rstd2, d[e]);
        }
        if (p.dx != nullptr) __stcs(reinterpret_cast<uint4*>(p.dx + row * p.lddx) + c, narrow8(d));
        if (sum_d) {
          uint64_t y[4];
          widen8(c_y[SUMS ? i : 0], y);
          add(0, c, d, y);
        }
        if (p.dy != nullptr) {
          if (p.gate != nullptr) {
            uint64_t gt[4];
            widen8(load_vec16(p.gate + b * p.K + 8 * c), gt);
#pragma unroll
            for (int e = 0; e < 4; ++e) d[e] = mul_f32x2(d[e], gt[e]);
          }
          __stcs(reinterpret_cast<uint4*>(p.dy + row * p.lddy) + c, narrow8(d));
        }
      }
    }
  }
  if (SUMS) {
    float* part = p.part + static_cast<int64_t>(blockIdx.x) * 3 * p.K;
#pragma unroll
    for (int i = 0; i < VPT; ++i) {
      const int c = threadIdx.x + i * blockDim.x;
      if (c < nvec) {
#pragma unroll
        for (int j = 0; j < 3; ++j)
#pragma unroll
          for (int h = 0; h < 2; ++h)
            *reinterpret_cast<ulonglong2*>(part + j * p.K + 8 * c + 4 * h) =
                SHARED ? *reinterpret_cast<const ulonglong2*>(sums + j * p.K + 8 * c + 4 * h)
                       : make_ulonglong2(acc[A ? j : 0][2 * h], acc[A ? j : 0][2 * h + 1]);
      }
    }
  }
}

struct SumParams {
  const float* part; int chunks; int64_t B; int K;
  const float* normw; const __nv_bfloat16* mscale;
  __nv_bfloat16* dgate; __nv_bfloat16* dmscale; __nv_bfloat16* dmshift;   // [B, K] or NULL
  float* dnorm;                                                           // [K] or NULL
  float* share;                                                           // [B, K]: a sample's part of dnorm (B > 1)
};

// 32 columns of one sample per CTA; sixteen groups of threads take every sixteenth chunk, and their sums are added in
// group order: the result does not depend on how the CTAs before were scheduled.
constexpr int kSumGroups = 16;
__global__ void __launch_bounds__(32 * kSumGroups) residual_sums_kernel(const SumParams p) {
  __shared__ float s[kSumGroups][3][32];
  const int col = threadIdx.x & 31, grp = threadIdx.x >> 5;
  const int k = blockIdx.x * 32 + col;
  const bool ok = k < p.K;
  pdl_wait();
  for (int64_t b = blockIdx.y; b < p.B; b += gridDim.y) {
    float a[3] = {0.f, 0.f, 0.f};
    if (ok) {
#pragma unroll 4
      for (int c = grp; c < p.chunks; c += kSumGroups) {
        const float* src = p.part + ((b * p.chunks + c) * 3) * p.K + k;
        a[0] += src[0];
        a[1] += src[p.K];
        a[2] += src[2 * static_cast<int64_t>(p.K)];
      }
    }
#pragma unroll
    for (int j = 0; j < 3; ++j) s[grp][j][col] = a[j];
    __syncthreads();
    if (grp == 0 && ok) {
#pragma unroll
      for (int j = 0; j < 3; ++j) {
        a[j] = s[0][j][col];
#pragma unroll
        for (int g = 1; g < kSumGroups; ++g) a[j] += s[g][j][col];
      }
      const int64_t at = b * p.K + k;
      if (p.dgate != nullptr) p.dgate[at] = __float2bfloat16_rn(a[0]);
      if (p.dmscale != nullptr) p.dmscale[at] = __float2bfloat16_rn(a[1] * (1.0f + p.normw[k]));
      if (p.dmshift != nullptr) p.dmshift[at] = __float2bfloat16_rn(a[2]);
      if (p.dnorm != nullptr) {
        const float d = p.mscale != nullptr ? a[1] * (1.0f + __bfloat162float(p.mscale[at])) : a[1];
        if (p.B == 1) p.dnorm[k] = d;
        else p.share[at] = d;
      }
    }
    __syncthreads();                           // the sums have been read before the next sample's are written
  }
}

__global__ void __launch_bounds__(128) residual_dnorm_kernel(const SumParams p) {
  const int k = blockIdx.x * 128 + threadIdx.x;
  pdl_wait();
  if (k >= p.K) return;
  float d = 0.f;
#pragma unroll 8
  for (int64_t b = 0; b < p.B; ++b) d += p.share[b * p.K + k];
  p.dnorm[k] = d;
}

// ---- host side ------------------------------------------------------------------------------------
bool off16(const void* ptr) { return (reinterpret_cast<uintptr_t>(ptr) & 15u) != 0; }
bool bad_rows(const void* ptr, int64_t ld, int64_t K) { return off16(ptr) || ld < K || (ld & 7) != 0; }

int check_common(const char* name, const ResParams& p, int64_t K, int unit) {
  if (p.M < 0 || K <= 0 || K > 16384 || K % unit != 0)
    return fail(K2Q_EINVAL, "%s: bad shape M=%lld K=%lld (K a multiple of %d up to 16384)", name, (long long)p.M, (long long)K, unit);
  if (p.rows_per_batch <= 0 || p.M % p.rows_per_batch != 0)
    return fail(K2Q_EINVAL, "%s: rows_per_batch %lld does not divide M=%lld", name, (long long)p.rows_per_batch, (long long)p.M);
  if (!p.normw || off16(p.normw) || off16(p.gate) || off16(p.mscale) || off16(p.mshift))
    return fail(K2Q_EINVAL, "%s: norm weight (non-NULL), gate and modulation vectors must be 16-byte aligned", name);
  return K2Q_OK;
}

// CTAs per sample: enough for `ctas_per_sm` on every SM over all samples, at most one per row
int chunks_for(int64_t B, int64_t rows_per_batch, int ctas_per_sm) {
  const int sms = sm_count() > 0 ? sm_count() : 148;
  int64_t c = (static_cast<int64_t>(sms) * ctas_per_sm + B - 1) / B;
  if (c > rows_per_batch) c = rows_per_batch;
  return static_cast<int>(c < 1 ? 1 : c);
}
using Kernel = void (*)(ResParams);
// Shared memory limits are a kernel's, not a launch's: always the largest that it can need, so that a host thread never
// lowers the limit between another one's setting it and launching.
constexpr int kQuantSmem = 16384 * 8, kBwdSmem = 16384 * 12;
// CTAs of a kernel that share an SM, asked of the runtime once per kernel (`slot`) and number of warps; `smem` belongs to
// the widest row of that number of warps, so that the grid does not depend on which row came first
int ctas_per_sm(Kernel kern, int slot, int threads, int smem, int limit) {
  static std::atomic<int> known[16][17];
  std::atomic<int>& k = known[slot][threads / 32];
  int n = k.load(std::memory_order_relaxed);
  if (n == 0) {
    if (cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, limit) != cudaSuccess ||
        cudaOccupancyMaxActiveBlocksPerMultiprocessor(&n, kern, threads, static_cast<size_t>(smem)) != cudaSuccess || n < 1) {
      cudaGetLastError();
      return 1;
    }
    k.store(n, std::memory_order_relaxed);
  }
  return n;
}

// threads per CTA and 16-byte vectors per thread of the dense kernels
void dense_shape(int64_t K, int* threads, int* vpt) {
  const int nvec = static_cast<int>(K / 8);
  *vpt = (nvec + 511) / 512;
  *threads = ((nvec + *vpt - 1) / *vpt + 31) / 32 * 32;
}

const Kernel kQuant[4] = {residual_quant_kernel<false, false>, residual_quant_kernel<false, true>, residual_quant_kernel<true, false>,
                          residual_quant_kernel<true, true>};
const Kernel kFwd[4] = {residual_fwd_kernel<1>, residual_fwd_kernel<2>, residual_fwd_kernel<3>, residual_fwd_kernel<4>};
const Kernel kBwd[8] = {residual_bwd_kernel<1, false>, residual_bwd_kernel<1, true>, residual_bwd_kernel<2, false>,
                        residual_bwd_kernel<2, true>,  residual_bwd_kernel<3, false>, residual_bwd_kernel<3, true>,
                        residual_bwd_kernel<4, false>, residual_bwd_kernel<4, true>};

struct BwdShape { int threads, slot, smem, chunks; };
BwdShape bwd_shape(int64_t B, int64_t rows_per_batch, int64_t K, bool sums) {
  BwdShape s{};
  int vpt;
  dense_shape(K, &s.threads, &vpt);
  s.slot = (vpt - 1) * 2 + (sums ? 1 : 0);
  s.smem = sums && vpt > 1 ? static_cast<int>(K) * 12 : 0;
  const int widest = s.smem > 0 ? s.threads * vpt * 8 * 12 : 0;
  s.chunks = chunks_for(B, rows_per_batch, ctas_per_sm(kBwd[s.slot], s.slot, s.threads, widest, s.smem > 0 ? kBwdSmem : 0));
  return s;
}

}  // namespace
}  // namespace k2q

using namespace k2q;

extern "C" {

int k2q_residual_norm_quant(const void* x_bf16, int64_t ldx, const void* y_bf16, int64_t ldy, const void* gate_bf16,
                            const float* norm_scale, const void* mod_scale_bf16, const void* mod_shift_bf16,
                            int64_t rows_per_batch, int64_t M, int64_t K, float eps, void* stream_bf16, int64_t lds,
                            int8_t* xq, float* sx, void* stream) {
  const char* name = "k2q_residual_norm_quant";
  if (int rc = check_device_arch()) return rc;
  ResParams p{};
  p.x = static_cast<const __nv_bfloat16*>(x_bf16); p.ldx = ldx;
  p.y = static_cast<const __nv_bfloat16*>(y_bf16); p.ldy = ldy;
  p.gate = static_cast<const __nv_bfloat16*>(gate_bf16); p.normw = norm_scale;
  p.mscale = static_cast<const __nv_bfloat16*>(mod_scale_bf16); p.mshift = static_cast<const __nv_bfloat16*>(mod_shift_bf16);
  p.M = M; p.K = static_cast<int>(K); p.rows_per_batch = rows_per_batch; p.eps = eps;
  p.stream = static_cast<__nv_bfloat16*>(stream_bf16); p.lds = lds; p.xq = xq; p.sx = sx;
  if (int rc = check_common(name, p, K, 128)) return rc;
  if (M == 0) return K2Q_OK;
  if (!p.gate && !p.mscale && !p.mshift) p.rows_per_batch = rows_per_batch = M;    // nothing tells the samples apart
  if (!p.x || !p.y || !p.stream || !xq || !sx) return fail(K2Q_EINVAL, "%s: NULL operand", name);
  if (bad_rows(p.x, ldx, K) || bad_rows(p.y, ldy, K) || bad_rows(p.stream, lds, K) || off16(xq))
    return fail(K2Q_EINVAL, "%s: rows must be 16-byte aligned with a leading dimension >= K", name);
  const int threads = (static_cast<int>(K / 32) + 31) / 32 * 32;
  const int64_t B = M / rows_per_batch;
  const int per_k = 4 + (p.mshift ? 2 : 0) + (p.gate ? 2 : 0), vec_bytes = static_cast<int>(K) * per_k;
  const int slot = (p.gate ? 2 : 0) + (p.mshift ? 1 : 0);
  p.chunks = chunks_for(B, rows_per_batch, ctas_per_sm(kQuant[slot], 12 + slot, threads, threads * 32 * per_k, kQuantSmem));
  if (B * p.chunks > 0x7fffffffLL) return fail(K2Q_EINVAL, "%s: too many samples (%lld)", name, (long long)B);
  if (int rc = check_cuda(cudaFuncSetAttribute(kQuant[slot], cudaFuncAttributeMaxDynamicSharedMemorySize, kQuantSmem),
                          "cudaFuncSetAttribute(residual_quant)"))
    return rc;
  return launch_overlapped(kQuant[slot], static_cast<unsigned>(B * p.chunks), static_cast<unsigned>(threads), static_cast<size_t>(vec_bytes),
                           static_cast<cudaStream_t>(stream), 1, "residual_quant launch", p);
}

int k2q_residual_norm_fwd(const void* x_bf16, int64_t ldx, const void* y_bf16, int64_t ldy, const void* gate_bf16,
                          const float* norm_scale, const void* mod_scale_bf16, const void* mod_shift_bf16,
                          int64_t rows_per_batch, int64_t M, int64_t K, float eps, void* stream_bf16, int64_t lds,
                          void* h_bf16, int64_t ldh, float* rstd, void* stream) {
  const char* name = "k2q_residual_norm_fwd";
  if (int rc = check_device_arch()) return rc;
  ResParams p{};
  p.x = static_cast<const __nv_bfloat16*>(x_bf16); p.ldx = ldx;
  p.y = static_cast<const __nv_bfloat16*>(y_bf16); p.ldy = ldy;
  p.gate = static_cast<const __nv_bfloat16*>(gate_bf16); p.normw = norm_scale;
  p.mscale = static_cast<const __nv_bfloat16*>(mod_scale_bf16); p.mshift = static_cast<const __nv_bfloat16*>(mod_shift_bf16);
  p.M = M; p.K = static_cast<int>(K); p.rows_per_batch = rows_per_batch; p.eps = eps;
  p.stream = static_cast<__nv_bfloat16*>(stream_bf16); p.lds = lds;
  p.h = static_cast<__nv_bfloat16*>(h_bf16); p.ldh = ldh; p.rstd = rstd;
  if (int rc = check_common(name, p, K, 8)) return rc;
  if (M == 0) return K2Q_OK;
  if (!p.gate && !p.mscale && !p.mshift) p.rows_per_batch = rows_per_batch = M;    // nothing tells the samples apart
  if (!p.x || !p.y || !p.stream || !p.h || !rstd) return fail(K2Q_EINVAL, "%s: NULL operand", name);
  if (bad_rows(p.x, ldx, K) || bad_rows(p.y, ldy, K) || bad_rows(p.stream, lds, K) || bad_rows(p.h, ldh, K))
    return fail(K2Q_EINVAL, "%s: rows must be 16-byte aligned with a leading dimension >= K", name);
  int threads, vpt;
  dense_shape(K, &threads, &vpt);
  const int64_t B = M / rows_per_batch;
  p.chunks = chunks_for(B, rows_per_batch, ctas_per_sm(kFwd[vpt - 1], 8 + vpt - 1, threads, 0, 0));
  if (B * p.chunks > 0x7fffffffLL) return fail(K2Q_EINVAL, "%s: too many samples (%lld)", name, (long long)B);
  return launch_overlapped(kFwd[vpt - 1], static_cast<unsigned>(B * p.chunks), static_cast<unsigned>(threads), 0,
                           static_cast<cudaStream_t>(stream), 1, "residual_fwd launch", p);
}

int64_t k2q_residual_norm_bwd_workspace_bytes(int64_t rows_per_batch, int64_t M, int64_t K) {
  if (rows_per_batch <= 0 || M <= 0 || K <= 0 || K > 16384) return 0;
  const int64_t B = M / rows_per_batch;
  return (B * bwd_shape(B, rows_per_batch, K, true).chunks * 3 + (B > 1 ? B : 0)) * K * static_cast<int64_t>(sizeof(float));
}

int k2q_residual_norm_bwd(const void* dstream_bf16, int64_t ldds, const void* dh_bf16, int64_t lddh,
                          const void* stream_bf16, int64_t lds, const float* rstd, const void* y_bf16, int64_t ldy,
                          const void* gate_bf16, const float* norm_scale, const void* mod_scale_bf16,
                          int64_t rows_per_batch, int64_t M, int64_t K, void* dx_bf16, int64_t lddx, void* dy_bf16,
                          int64_t lddy, void* dgate_bf16, void* dmod_scale_bf16, void* dmod_shift_bf16, float* dnorm,
                          void* ws, int64_t ws_bytes, void* stream) {
  const char* name = "k2q_residual_norm_bwd";
  if (int rc = check_device_arch()) return rc;
  ResParams p{};
  p.dstream = static_cast<const __nv_bfloat16*>(dstream_bf16); p.ldds = ldds;
  p.dh = static_cast<const __nv_bfloat16*>(dh_bf16); p.lddh = lddh;
  p.stream = static_cast<__nv_bfloat16*>(const_cast<void*>(stream_bf16)); p.lds = lds;
  p.rstd = const_cast<float*>(rstd);
  p.y = static_cast<const __nv_bfloat16*>(y_bf16); p.ldy = ldy;
  p.gate = static_cast<const __nv_bfloat16*>(gate_bf16); p.normw = norm_scale;
  p.mscale = static_cast<const __nv_bfloat16*>(mod_scale_bf16);
  p.M = M; p.K = static_cast<int>(K); p.rows_per_batch = rows_per_batch;
  p.dx = static_cast<__nv_bfloat16*>(dx_bf16); p.lddx = lddx;
  p.dy = static_cast<__nv_bfloat16*>(dy_bf16); p.lddy = lddy;
  if (int rc = check_common(name, p, K, 8)) return rc;
  if (M == 0) return K2Q_OK;
  if (!p.stream || !rstd) return fail(K2Q_EINVAL, "%s: NULL operand", name);
  if (bad_rows(p.stream, lds, K) || (p.dstream && bad_rows(p.dstream, ldds, K)) || (p.dh && bad_rows(p.dh, lddh, K)) ||
      (p.y && bad_rows(p.y, ldy, K)) || (p.dx && bad_rows(p.dx, lddx, K)) || (p.dy && bad_rows(p.dy, lddy, K)))
    return fail(K2Q_EINVAL, "%s: rows must be 16-byte aligned with a leading dimension >= K", name);
  if (!p.gate && !p.mscale && !dmod_scale_bf16 && !dmod_shift_bf16) p.rows_per_batch = rows_per_batch = M;
  if (dgate_bf16 && (!p.gate || !p.y)) return fail(K2Q_EINVAL, "%s: the gate's gradient needs gate and y", name);
  const int64_t B = M / rows_per_batch;
  const bool sums = dgate_bf16 || dmod_scale_bf16 || dmod_shift_bf16 || dnorm;
  const BwdShape shape = bwd_shape(B, rows_per_batch, K, sums);
  p.chunks = shape.chunks;
  if (!dgate_bf16) p.y = nullptr;
  if (sums) {
    if (!ws || off16(ws) || ws_bytes < k2q_residual_norm_bwd_workspace_bytes(rows_per_batch, M, K))
      return fail(K2Q_EINVAL, "%s: workspace too small or not 16-byte aligned", name);
    p.part = static_cast<float*>(ws);
  }
  if (B * p.chunks > 0x7fffffffLL) return fail(K2Q_EINVAL, "%s: too many samples (%lld)", name, (long long)B);
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  if (shape.smem > 0) {
    if (int rc = check_cuda(cudaFuncSetAttribute(kBwd[shape.slot], cudaFuncAttributeMaxDynamicSharedMemorySize, kBwdSmem),
                            "cudaFuncSetAttribute(residual_bwd)"))
      return rc;
  }
  if (int rc = launch_overlapped(kBwd[shape.slot], static_cast<unsigned>(B * p.chunks), static_cast<unsigned>(shape.threads),
                                 static_cast<size_t>(shape.smem), s, 1, "residual_bwd launch", p))
    return rc;
  if (!sums) return K2Q_OK;
  SumParams q{};
  q.part = p.part; q.chunks = p.chunks; q.B = B; q.K = p.K; q.normw = norm_scale; q.mscale = p.mscale;
  q.dgate = static_cast<__nv_bfloat16*>(dgate_bf16); q.dmscale = static_cast<__nv_bfloat16*>(dmod_scale_bf16);
  q.dmshift = static_cast<__nv_bfloat16*>(dmod_shift_bf16); q.dnorm = dnorm;
  q.share = p.part + B * p.chunks * 3 * static_cast<int64_t>(p.K);
  cudaLaunchConfig_t cfg{};
  cfg.gridDim = dim3(static_cast<unsigned>((p.K + 31) / 32), static_cast<unsigned>(B < 65535 ? B : 65535));
  cfg.blockDim = dim3(32 * kSumGroups);
  cfg.stream = s;
  cudaLaunchAttribute attr{};
  attr.id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr.val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = &attr;
  cfg.numAttrs = overlapped_launch_allowed(s) ? 1 : 0;
  if (int rc = check_cuda(cudaLaunchKernelEx(&cfg, residual_sums_kernel, q), "residual_sums launch")) return rc;
  if (!dnorm || B == 1) return K2Q_OK;
  return launch_overlapped(residual_dnorm_kernel, static_cast<unsigned>((p.K + 127) / 128), 128u, 0, s, 1, "residual_dnorm launch", q);
}

}  // extern "C"
