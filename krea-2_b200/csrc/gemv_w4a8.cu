// Products of a few token rows with a 4-bit base (group scales), M <= 32:
//
//   run = 0;  for g = 0 .. K/128-1:  run = fma(float(sum_{k in g} xq[m,k] q4[n,k]), sw4[n,g], run)
//   y[m,n] = bf16( act(run * sx[m] + bias[n]) + sum_j u[m,j] (lora_scale Bm[n,j]) )
//
// The group sums are exact integers and the scales enter in ascending order of the groups, one fused
// multiply-add each: the operations of the large W4A8 product on every element, so both give the same bits.
// Bound by reading the codes once: N*K/2 bytes.
#include "k2q_common.cuh"

namespace k2q {
namespace {

constexpr int kMaxRows = 32;
constexpr int kWarps = 4;

struct GemvParams {
  int M, N, K;
  const int8_t* xq; const uint8_t* wq; const __nv_bfloat16* sw;
  const float* sx; const float* bias; const float* u; const float* Bm;
  int64_t ldu, ldb; int rank; float lora_scale; int act;
  __nv_bfloat16* y; int64_t ldy;
};

// the activation of the large product: hardware tanh, |error| < 6e-4, below the bf16 step of the output
__device__ __forceinline__ float gelu_tanh_hw(float v) {
  const float z = v * fmaf(0.0356774081f, v * v, 0.7978845608f);
  float th;
  asm("tanh.approx.f32 %0, %1;" : "=f"(th) : "f"(z));
  const float hv = 0.5f * v;
  return fmaf(hv, th, hv);
}

__device__ __forceinline__ void finish(const GemvParams& p, int m, int n, float run) {
  float v = __fadd_rn(__fmul_rn(run, p.sx != nullptr ? __ldg(p.sx + m) : 1.0f), p.bias != nullptr ? __ldg(p.bias + n) : 0.0f);
  if (p.act == K2Q_ACT_GELU_TANH) v = gelu_tanh_hw(v);
  if (p.rank > 0) {
    float d = 0.f;
    for (int j = 0; j < p.rank; ++j)
      d = fmaf(__ldg(p.u + m * p.ldu + j), p.lora_scale * __ldg(p.Bm + n * p.ldb + j), d);
    v += d;
  }
  p.y[m * p.ldy + n] = __float2bfloat16_rn(v);
}

// One warp per output channel; a lane holds four codes of the group, the group sums are added over the
// warp, and lane m keeps the running value of token m.
__global__ void __launch_bounds__(kWarps * 32) gemv_kernel(const GemvParams p) {
  const int lane = threadIdx.x & 31;
  const int n = blockIdx.x * kWarps + (threadIdx.x >> 5);
  if (n >= p.N) return;
  const int groups = p.K >> 7;
  float run = 0.f;
  for (int g = 0; g < groups; ++g) {
    const uint32_t c = __ldg(reinterpret_cast<const uint16_t*>(p.wq + static_cast<int64_t>(n) * (p.K >> 1) + g * 64) + lane);
    // codes k0, k1, k2, k3 as the high nibbles of four bytes: 16 times their value
    const int w = static_cast<int>(((c << 4) & 0xF0u) | ((c & 0xF0u) << 8) | ((c & 0x0F00u) << 12) | ((c & 0xF000u) << 16));
    const float s = __bfloat162float(p.sw[static_cast<int64_t>(n) * groups + g]) * 0.0625f;
    for (int m = 0; m < p.M; ++m) {
      const int x = __ldg(reinterpret_cast<const int*>(p.xq + static_cast<int64_t>(m) * p.K + g * 128) + lane);
      const int acc = __reduce_add_sync(0xffffffffu, __dp4a(x, w, 0));
      if (lane == m) run = fmaf(static_cast<float>(acc), s, run);
    }
  }
  if (lane < p.M) finish(p, lane, n, run);
}

}  // namespace
}  // namespace k2q

using namespace k2q;

extern "C" int k2q_gemv_w4a8(const int8_t* xq, const uint8_t* wq4, const void* sw4_bf16, int64_t M, int64_t N, int64_t K,
                             const k2q_epilogue* ep, void* y_bf16, int64_t ldy, void* stream) {
  const char* name = "k2q_gemv_w4a8";
  if (int rc = check_device_arch()) return rc;
  if (M < 0 || M > kMaxRows || N <= 0 || K <= 0 || N > 0x7fffff00LL || K > 0x7fffff00LL)
    return fail(K2Q_EINVAL, "%s: bad shape M=%lld N=%lld K=%lld (at most %d rows)", name, (long long)M, (long long)N,
                (long long)K, kMaxRows);
  if (K % 128 != 0) return fail(K2Q_EINVAL, "%s: K=%lld is not a multiple of 128", name, (long long)K);
  if (N % 16 != 0) return fail(K2Q_EINVAL, "%s: N=%lld is not a multiple of 16", name, (long long)N);
  if (M == 0) return K2Q_OK;
  if (!xq || !wq4 || !sw4_bf16 || !y_bf16) return fail(K2Q_EINVAL, "%s: NULL operand", name);
  if ((reinterpret_cast<uintptr_t>(xq) | reinterpret_cast<uintptr_t>(wq4)) & 15u)
    return fail(K2Q_EINVAL, "%s: codes must be 16-byte aligned", name);
  if (ldy < N) return fail(K2Q_EINVAL, "%s: ldy < N", name);
  k2q_epilogue e{};
  if (ep) e = *ep;
  if (e.rank < 0 || e.rank > 32) return fail(K2Q_EINVAL, "%s: LoRA rank %d not in [0,32]", name, e.rank);
  if ((e.u == nullptr) != (e.Bm == nullptr) || ((e.u != nullptr) != (e.rank > 0)))
    return fail(K2Q_EINVAL, "%s: u, Bm and rank must be given together", name);
  if (e.rank > 0 && (e.ldu < e.rank || e.ldb < e.rank)) return fail(K2Q_EINVAL, "%s: ldu/ldb smaller than rank", name);
  if (e.act != K2Q_ACT_NONE && e.act != K2Q_ACT_GELU_TANH) return fail(K2Q_EINVAL, "%s: unknown activation %d", name, e.act);
  GemvParams p{};
  p.M = (int)M; p.N = (int)N; p.K = (int)K;
  p.xq = xq; p.wq = wq4; p.sw = static_cast<const __nv_bfloat16*>(sw4_bf16);
  p.sx = e.sx; p.bias = e.bias; p.u = e.u; p.Bm = e.Bm; p.ldu = e.ldu; p.ldb = e.ldb; p.rank = e.rank;
  p.lora_scale = e.lora_scale; p.act = e.act;
  p.y = static_cast<__nv_bfloat16*>(y_bf16); p.ldy = ldy;
  gemv_kernel<<<(p.N + kWarps - 1) / kWarps, kWarps * 32, 0, static_cast<cudaStream_t>(stream)>>>(p);
  return check_cuda(cudaGetLastError(), "gemv_w4a8 launch");
}
