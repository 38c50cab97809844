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
// rows_per_batch.  All three are bound by HBM: 7, 8 and 8 (10 with the sums) bytes per element.
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

// Sum / maximum over the CTA, the same value in every thread, in a fixed order.  One barrier: successive
// calls of a kernel alternate between two slots, so a slot is written again only behind the barrier of
// the call in between, which every reader of the slot has passed.
template <bool MAX>
__device__ __forceinline__ float cta_reduce(float v, float* slot, int warps) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) {
    const float other = __shfl_xor_sync(0xffffffffu, v, o);
    v = MAX ? fmaxf(v, other) : v + other;
  }
  if ((threadIdx.x & 31) == 0) slot[threadIdx.x >> 5] = v;
  __syncthreads();
  float t = slot[0];
  for (int w = 1; w < warps; ++w) t = MAX ? fmaxf(t, slot[w]) : t + slot[w];
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
  float* part; int chunks;                      // [B, chunks, 3, K] partial sums D, S, H, or NULL
};

// stream of 8 consecutive elements; rounded product and rounded sum, as the two fp32 operations it is
__device__ __forceinline__ uint4 residual8(const ResParams& p, int64_t row, int64_t b, int k0) {
  float x[8], y[8];
  unpack8(load_row16(p.x + row * p.ldx + k0), x);
  unpack8(load_row16(p.y + row * p.ldy + k0), y);
  if (p.gate != nullptr) {
    float g[8];
    unpack8(load_vec16(p.gate + b * p.K + k0), g);
#pragma unroll
    for (int e = 0; e < 8; ++e) y[e] = __fmul_rn(g[e], y[e]);
  }
#pragma unroll
  for (int e = 0; e < 8; ++e) x[e] = __fadd_rn(x[e], y[e]);
  return pack8(x);
}

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
// One CTA per row, four neighbouring lanes per 128-block.  Lane q of the four owns the 8-element chunks
// q, q + 4, q + 8, q + 12 of the block: a warp's 16-byte accesses then cover whole 64-byte pieces (32-byte
// pieces of the codes), and no staging through shared memory is needed.  Of the rotation's seven
// butterfly stages, h = 1, 2, 4 and 32, 64 lie inside a thread, h = 8 and 16 between lanes.
__device__ __forceinline__ void fwht128_chunks(float (&v)[32], int q) {
#pragma unroll
  for (int h = 1; h < 8; h <<= 1) {
#pragma unroll
    for (int i = 0; i < 32; ++i) {
      if ((i & h) == 0) {
        const float a = v[i], b = v[i + h];
        v[i] = __fadd_rn(a, b);
        v[i + h] = __fsub_rn(a, b);
      }
    }
  }
#pragma unroll
  for (int j = 0; j < 2; ++j) {
    const float sgn = ((q >> j) & 1) ? -1.0f : 1.0f;     // lower lane a + b, upper lane a - b
#pragma unroll
    for (int i = 0; i < 32; ++i) {
      const float o = __shfl_xor_sync(0xffffffffu, v[i], 1 << j);
      v[i] = __fmaf_rn(v[i], sgn, o);
    }
  }
#pragma unroll
  for (int h = 8; h < 32; h <<= 1) {
#pragma unroll
    for (int i = 0; i < 32; ++i) {
      if ((i & h) == 0) {
        const float a = v[i], b = v[i + h];
        v[i] = __fadd_rn(a, b);
        v[i + h] = __fsub_rn(a, b);
      }
    }
  }
#pragma unroll
  for (int i = 0; i < 32; ++i) v[i] *= kHadNorm;
}

__global__ void __launch_bounds__(512) residual_quant_kernel(const ResParams p) {
  __shared__ float red[2][kMaxWarps];
  const int warps = blockDim.x >> 5;
  const int q = threadIdx.x & 3;
  const int blk = threadIdx.x >> 2;                       // 128-block of the row
  const bool own = blk < (p.K >> 7);
  for (int64_t row = blockIdx.x; row < p.M; row += gridDim.x) {
    const int64_t b = row / p.rows_per_batch;
    float v[32];
    float ss = 0.f;
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const int k0 = blk * 128 + (q + 4 * j) * 8;
      if (own) {
        const uint4 s = residual8(p, row, b, k0);
        *reinterpret_cast<uint4*>(p.stream + row * p.lds + k0) = s;
        unpack8(s, v + 8 * j);
      } else {
#pragma unroll
        for (int e = 0; e < 8; ++e) v[8 * j + e] = 0.f;
      }
    }
#pragma unroll
    for (int i = 0; i < 32; ++i) ss = fmaf(v[i], v[i], ss);
    const float rstd = rsqrtf(cta_reduce<false>(ss, red[0], warps) / static_cast<float>(p.K) + p.eps);
    if (own) {
#pragma unroll
      for (int j = 0; j < 4; ++j) norm_mod8(p, b, blk * 128 + (q + 4 * j) * 8, rstd, v + 8 * j);
    }
    fwht128_chunks(v, q);
    float amax = 0.f;
#pragma unroll
    for (int i = 0; i < 32; ++i) amax = fmaxf(amax, fabsf(v[i]));
    amax = cta_reduce<true>(amax, red[1], warps);
    const float s = __fdiv_rn(fmaxf(amax, 1e-8f), 127.0f);
    const float inv = __frcp_rn(s);
    uint32_t words[8];
    quant_row32_i8(v, s, inv, words);
    if (own) {
#pragma unroll
      for (int j = 0; j < 4; ++j)
        *reinterpret_cast<uint2*>(p.xq + row * p.K + blk * 128 + (q + 4 * j) * 8) = make_uint2(words[2 * j], words[2 * j + 1]);
    }
    if (threadIdx.x == 0) p.sx[row] = s;
  }
}

// ---- training: dense output and its backward ------------------------------------------------------
template <int VPT>
__global__ void __launch_bounds__(512) residual_fwd_kernel(const ResParams p) {
  __shared__ float red[2][kMaxWarps];
  const int warps = blockDim.x >> 5, nvec = p.K >> 3;
  int it = 0;
  for (int64_t row = blockIdx.x; row < p.M; row += gridDim.x, it ^= 1) {
    const int64_t b = row / p.rows_per_batch;
    float v[VPT][8];
    float ss = 0.f;
#pragma unroll
    for (int i = 0; i < VPT; ++i) {
      const int c = threadIdx.x + i * blockDim.x;
      if (c < nvec) {
        const uint4 s = residual8(p, row, b, 8 * c);
        reinterpret_cast<uint4*>(p.stream + row * p.lds)[c] = s;
        unpack8(s, v[i]);
#pragma unroll
        for (int e = 0; e < 8; ++e) ss = fmaf(v[i][e], v[i][e], ss);
      }
    }
    const float rstd = rsqrtf(cta_reduce<false>(ss, red[it], warps) / static_cast<float>(p.K) + p.eps);
    if (threadIdx.x == 0) p.rstd[row] = rstd;
#pragma unroll
    for (int i = 0; i < VPT; ++i) {
      const int c = threadIdx.x + i * blockDim.x;
      if (c < nvec) {
        norm_mod8(p, b, 8 * c, rstd, v[i]);
        reinterpret_cast<uint4*>(p.h + row * p.ldh)[c] = pack8(v[i]);
      }
    }
  }
}

// A CTA works through consecutive rows of ONE sample and a thread owns the same columns in all of them, so
// the sums over rows stay in registers; each CTA leaves its partial sums in its own slice of the workspace.
template <int VPT, bool SUMS>
__global__ void __launch_bounds__(512) residual_bwd_kernel(const ResParams p) {
  __shared__ float red[2][kMaxWarps];
  const int warps = blockDim.x >> 5, nvec = p.K >> 3;
  const int64_t b = blockIdx.x / p.chunks;
  const int chunk = blockIdx.x - static_cast<int>(b) * p.chunks;
  const int64_t r0 = b * p.rows_per_batch + p.rows_per_batch * chunk / p.chunks;
  const int64_t r1 = b * p.rows_per_batch + p.rows_per_batch * (chunk + 1) / p.chunks;
  float aD[SUMS ? VPT : 1][8] = {}, aS[SUMS ? VPT : 1][8] = {}, aH[SUMS ? VPT : 1][8] = {};
  int it = 0;
  for (int64_t row = r0; row < r1; ++row, it ^= 1) {
    float n[VPT][8], g[VPT][8];
    float dot = 0.f, rstd = 0.f;
    if (p.dh != nullptr) {
      rstd = p.rstd[row];
#pragma unroll
      for (int i = 0; i < VPT; ++i) {
        const int c = threadIdx.x + i * blockDim.x;
        if (c < nvec) {
          float w[8];
          unpack8(load_vec16(p.dh + row * p.lddh + 8 * c), g[i]);
          unpack8(load_vec16(p.stream + row * p.lds + 8 * c), n[i]);
          load8f(p.normw + 8 * c, w);
#pragma unroll
          for (int e = 0; e < 8; ++e) w[e] += 1.0f;
          if (p.mscale != nullptr) {
            float s[8];
            unpack8(load_vec16(p.mscale + b * p.K + 8 * c), s);
#pragma unroll
            for (int e = 0; e < 8; ++e) w[e] *= 1.0f + s[e];
          }
#pragma unroll
          for (int e = 0; e < 8; ++e) {
            n[i][e] *= rstd;
            if (SUMS) {
              aS[i][e] = fmaf(g[i][e], n[i][e], aS[i][e]);
              aH[i][e] += g[i][e];
            }
            g[i][e] *= w[e];
            dot = fmaf(g[i][e], n[i][e], dot);
          }
        }
      }
      dot = cta_reduce<false>(dot, red[it], warps) / static_cast<float>(p.K);
    }
#pragma unroll
    for (int i = 0; i < VPT; ++i) {
      const int c = threadIdx.x + i * blockDim.x;
      if (c < nvec) {
        float d[8];
        if (p.dstream != nullptr) unpack8(load_vec16(p.dstream + row * p.ldds + 8 * c), d);
        else {
#pragma unroll
          for (int e = 0; e < 8; ++e) d[e] = 0.f;
        }
        if (p.dh != nullptr) {
#pragma unroll
          for (int e = 0; e < 8; ++e) d[e] += rstd * (g[i][e] - n[i][e] * dot);
        }
        if (p.dx != nullptr) reinterpret_cast<uint4*>(p.dx + row * p.lddx)[c] = pack8(d);
        if (SUMS && p.gate != nullptr && p.y != nullptr) {
          float y[8];
          unpack8(load_vec16(p.y + row * p.ldy + 8 * c), y);
#pragma unroll
          for (int e = 0; e < 8; ++e) aD[i][e] = fmaf(d[e], y[e], aD[i][e]);
        }
        if (p.dy != nullptr) {
          if (p.gate != nullptr) {
            float gt[8];
            unpack8(load_vec16(p.gate + b * p.K + 8 * c), gt);
#pragma unroll
            for (int e = 0; e < 8; ++e) d[e] *= gt[e];
          }
          reinterpret_cast<uint4*>(p.dy + row * p.lddy)[c] = pack8(d);
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
        for (int e = 0; e < 8; e += 4) {
          *reinterpret_cast<float4*>(part + 8 * c + e) = make_float4(aD[i][e], aD[i][e + 1], aD[i][e + 2], aD[i][e + 3]);
          *reinterpret_cast<float4*>(part + p.K + 8 * c + e) = make_float4(aS[i][e], aS[i][e + 1], aS[i][e + 2], aS[i][e + 3]);
          *reinterpret_cast<float4*>(part + 2 * p.K + 8 * c + e) = make_float4(aH[i][e], aH[i][e + 1], aH[i][e + 2], aH[i][e + 3]);
        }
      }
    }
  }
}

struct SumParams {
  const float* part; int chunks; int64_t B; int K;
  const float* normw; const __nv_bfloat16* mscale;
  __nv_bfloat16* dgate; __nv_bfloat16* dmscale; __nv_bfloat16* dmshift;   // [B, K] or NULL
  float* dnorm;                                                           // [K] or NULL
};

// 32 columns per CTA; eight groups of threads take every eighth chunk of a sample, and their sums are added
// in group order: the result does not depend on how the CTAs before were scheduled.
__global__ void __launch_bounds__(256) residual_sums_kernel(const SumParams p) {
  __shared__ float s[8][3][32];
  const int col = threadIdx.x & 31, grp = threadIdx.x >> 5;
  const int k = blockIdx.x * 32 + col;
  const bool ok = k < p.K;
  float dn = 0.f;
  for (int64_t b = 0; b < p.B; ++b) {
    float a[3] = {0.f, 0.f, 0.f};
    if (ok) {
      for (int c = grp; c < p.chunks; c += 8) {
        const float* src = p.part + ((b * p.chunks + c) * 3) * p.K + k;
        a[0] += src[0];
        a[1] += src[p.K];
        a[2] += src[2 * static_cast<int64_t>(p.K)];
      }
    }
    __syncthreads();                        // the previous sample's sums have been read
#pragma unroll
    for (int j = 0; j < 3; ++j) s[grp][j][col] = a[j];
    __syncthreads();
    if (grp == 0 && ok) {
#pragma unroll
      for (int j = 0; j < 3; ++j) {
        a[j] = s[0][j][col];
        for (int g = 1; g < 8; ++g) a[j] += s[g][j][col];
      }
      if (p.dgate != nullptr) p.dgate[b * p.K + k] = __float2bfloat16_rn(a[0]);
      if (p.dmscale != nullptr) p.dmscale[b * p.K + k] = __float2bfloat16_rn(a[1] * (1.0f + p.normw[k]));
      if (p.dmshift != nullptr) p.dmshift[b * p.K + k] = __float2bfloat16_rn(a[2]);
      dn += p.mscale != nullptr ? a[1] * (1.0f + __bfloat162float(p.mscale[b * p.K + k])) : a[1];
    }
  }
  if (grp == 0 && ok && p.dnorm != nullptr) p.dnorm[k] = dn;
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

int grid_rows(int64_t rows, int ctas_per_sm) {
  const int sms = sm_count() > 0 ? sm_count() : 148;
  const int64_t most = static_cast<int64_t>(sms) * ctas_per_sm;
  return static_cast<int>(rows < most ? rows : most);
}

// threads per CTA and 16-byte vectors per thread of the dense kernels
void dense_shape(int64_t K, int* threads, int* vpt) {
  const int nvec = static_cast<int>(K / 8);
  *vpt = (nvec + 511) / 512;
  *threads = ((nvec + *vpt - 1) / *vpt + 31) / 32 * 32;
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
  if (!p.x || !p.y || !p.stream || !xq || !sx) return fail(K2Q_EINVAL, "%s: NULL operand", name);
  if (bad_rows(p.x, ldx, K) || bad_rows(p.y, ldy, K) || bad_rows(p.stream, lds, K) || off16(xq))
    return fail(K2Q_EINVAL, "%s: rows must be 16-byte aligned with a leading dimension >= K", name);
  const int threads = (static_cast<int>(K / 32) + 31) / 32 * 32;
  residual_quant_kernel<<<grid_rows(M, 32), threads, 0, static_cast<cudaStream_t>(stream)>>>(p);
  return check_cuda(cudaGetLastError(), "residual_quant launch");
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
  if (!p.x || !p.y || !p.stream || !p.h || !rstd) return fail(K2Q_EINVAL, "%s: NULL operand", name);
  if (bad_rows(p.x, ldx, K) || bad_rows(p.y, ldy, K) || bad_rows(p.stream, lds, K) || bad_rows(p.h, ldh, K))
    return fail(K2Q_EINVAL, "%s: rows must be 16-byte aligned with a leading dimension >= K", name);
  int threads, vpt;
  dense_shape(K, &threads, &vpt);
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  const int grid = grid_rows(M, 32);
  switch (vpt) {
    case 1: residual_fwd_kernel<1><<<grid, threads, 0, s>>>(p); break;
    case 2: residual_fwd_kernel<2><<<grid, threads, 0, s>>>(p); break;
    case 3: residual_fwd_kernel<3><<<grid, threads, 0, s>>>(p); break;
    default: residual_fwd_kernel<4><<<grid, threads, 0, s>>>(p); break;
  }
  return check_cuda(cudaGetLastError(), "residual_fwd launch");
}

static int bwd_chunks(int64_t B, int64_t rows_per_batch) {
  const int sms = sm_count() > 0 ? sm_count() : 148;
  int64_t c = (2LL * sms + B - 1) / B;
  if (c > rows_per_batch) c = rows_per_batch;
  return static_cast<int>(c < 1 ? 1 : c);
}

int64_t k2q_residual_norm_bwd_workspace_bytes(int64_t rows_per_batch, int64_t M, int64_t K) {
  if (rows_per_batch <= 0 || M <= 0 || K <= 0) return 0;
  const int64_t B = M / rows_per_batch;
  return B * bwd_chunks(B, rows_per_batch) * 3 * K * static_cast<int64_t>(sizeof(float));
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
  if (dgate_bf16 && (!p.gate || !p.y)) return fail(K2Q_EINVAL, "%s: the gate's gradient needs gate and y", name);
  const int64_t B = M / rows_per_batch;
  const bool sums = dgate_bf16 || dmod_scale_bf16 || dmod_shift_bf16 || dnorm;
  p.chunks = bwd_chunks(B, rows_per_batch);
  if (!dgate_bf16) p.y = nullptr;
  if (sums) {
    if (!ws || off16(ws) || ws_bytes < k2q_residual_norm_bwd_workspace_bytes(rows_per_batch, M, K))
      return fail(K2Q_EINVAL, "%s: workspace too small or not 16-byte aligned", name);
    p.part = static_cast<float*>(ws);
  }
  if (B * p.chunks > 0x7fffffffLL) return fail(K2Q_EINVAL, "%s: too many samples (%lld)", name, (long long)B);
  int threads, vpt;
  dense_shape(K, &threads, &vpt);
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  const unsigned grid = static_cast<unsigned>(B * p.chunks);
  switch (vpt * 2 + (sums ? 1 : 0)) {
    case 2: residual_bwd_kernel<1, false><<<grid, threads, 0, s>>>(p); break;
    case 3: residual_bwd_kernel<1, true><<<grid, threads, 0, s>>>(p); break;
    case 4: residual_bwd_kernel<2, false><<<grid, threads, 0, s>>>(p); break;
    case 5: residual_bwd_kernel<2, true><<<grid, threads, 0, s>>>(p); break;
    case 6: residual_bwd_kernel<3, false><<<grid, threads, 0, s>>>(p); break;
    case 7: residual_bwd_kernel<3, true><<<grid, threads, 0, s>>>(p); break;
    case 8: residual_bwd_kernel<4, false><<<grid, threads, 0, s>>>(p); break;
    default: residual_bwd_kernel<4, true><<<grid, threads, 0, s>>>(p); break;
  }
  if (int rc = check_cuda(cudaGetLastError(), "residual_bwd launch")) return rc;
  if (!sums) return K2Q_OK;
  SumParams q{};
  q.part = p.part; q.chunks = p.chunks; q.B = B; q.K = p.K; q.normw = norm_scale; q.mscale = p.mscale;
  q.dgate = static_cast<__nv_bfloat16*>(dgate_bf16); q.dmscale = static_cast<__nv_bfloat16*>(dmod_scale_bf16);
  q.dmshift = static_cast<__nv_bfloat16*>(dmod_shift_bf16); q.dnorm = dnorm;
  residual_sums_kernel<<<(p.K + 31) / 32, 256, 0, s>>>(q);
  return check_cuda(cudaGetLastError(), "residual_sums launch");
}

}  // extern "C"
