// Momentum, orthogonalised update and parameter step of a set of matrices (the adapters' A [r, K] and
// B [N, r]) that lie end to end in flat fp32 buffers.  Per matrix, with S the short and L the long side:
//
//   m' = beta m + (1 - beta) g        u = beta m' + (1 - beta) g  (or m')       X0 = u / (||u||_F + eps),  S x L
//   X_{k+1} = (a I + b G_k + c G_k^2) X_k,   G_k = X_k X_k^T                    (Newton-Schulz, `steps` times)
//   p' = p (1 - lr wd) - lr scale X_steps
//
// Every factor Q_k = a I + b G_k + c G_k^2 is a polynomial of G_0, so all of them commute, and
//   X_steps = (Q_{steps-1} ... Q_0) X_0,    G_{k+1} = Q_k G_k Q_k :
// the iteration runs on S x S matrices alone and the data is touched twice, once for G_0 and once to be
// multiplied by the product.  Three kernels:
//   gram    m' and the partial Gram matrices of pieces of the long side
//   poly    partials added, normalised, iterated; leaves P = (Q ... Q_0) / (||u||_F + eps)
//   apply   P u and the parameter step
// The S x S iteration is in 64 bits: P's entries reach a^steps, so what G_0 loses to rounding comes back up to
// that much larger in the weak directions.  G_0's products are fp32, 32 columns are added in fp32 and
// the sums of those in 64 bits.  All sums run in a fixed order.
#include "k2q_common.cuh"

namespace k2q {
namespace {

constexpr int kMaxShort = 64;
constexpr int kThreads = 256;
constexpr int kSub = 32;                       // columns per sub-tile
constexpr double kA = 3.4445, kB = -4.7750, kC = 2.0315;

struct Mat {            // one entry of the device table
  int64_t off;          // first element in the flat buffers
  int64_t gram;         // first float of its partial Gram matrices in the workspace
  int64_t poly;         // first float of P
  int32_t s, tall;      // short side; tall: stored [L, S]
  int64_t l;            // long side
  int32_t tile0, tiles;
};
static_assert(sizeof(Mat) == 48, "table layout");
struct Tile { int32_t mat; int32_t pad; int64_t first; };   // columns [first, first + piece)

struct StepParams {
  const Mat* mats; const Tile* tiles; int64_t piece;
  float* p; float* g; float* m; float* out;
  float* ws;
  float lr, beta, wd, eps, max_norm;
  const float* normsq;
  int nesterov, steps, scale_mode, zero_grad;
};

__device__ __forceinline__ float clip_factor(const StepParams& a) {
  if (a.normsq == nullptr || !(a.max_norm > 0.f)) return 1.0f;
  return fminf(1.0f, a.max_norm / (sqrtf(__ldg(a.normsq)) + 1e-6f));
}
__device__ __forceinline__ int64_t address(const Mat& t, int i, int64_t l) { return t.off + (t.tall ? l * t.s + i : i * t.l + l); }

__global__ void __launch_bounds__(kThreads) gram_kernel(const StepParams a) {
  __shared__ float u[kMaxShort][kSub + 1];
  const Tile tile = a.tiles[blockIdx.x];
  const Mat t = a.mats[tile.mat];
  const float clip = clip_factor(a);
  const int64_t last = min(t.l, tile.first + a.piece);
  double acc[kMaxShort * kMaxShort / kThreads] = {};
  for (int64_t c0 = tile.first; c0 < last; c0 += kSub) {
    const int w = static_cast<int>(min(static_cast<int64_t>(kSub), last - c0));
    for (int e = threadIdx.x; e < t.s * kSub; e += kThreads) {
      const int i = t.tall ? e % t.s : e / kSub, l = t.tall ? e / t.s : e % kSub;
      float v = 0.f;
      if (l < w) {
        const int64_t at = address(t, i, c0 + l);
        v = a.g[at] * clip;
        if (a.m != nullptr) {
          const float m = a.beta * a.m[at] + (1.0f - a.beta) * v;
          a.m[at] = m;
          v = a.nesterov ? a.beta * m + (1.0f - a.beta) * v : m;
        }
      }
      u[i][l] = v;
    }
    __syncthreads();
    for (int k = 0, e = threadIdx.x; e < t.s * t.s; e += kThreads, ++k) {
      const int i = e / t.s, j = e % t.s;
      float s = 0.f;
      for (int l = 0; l < kSub; ++l) s = fmaf(u[i][l], u[j][l], s);
      acc[k] += s;
    }
    __syncthreads();
  }
  float* part = a.ws + t.gram + static_cast<int64_t>(blockIdx.x - t.tile0) * t.s * t.s;
  for (int k = 0, e = threadIdx.x; e < t.s * t.s; e += kThreads, ++k) part[e] = static_cast<float>(acc[k]);
}

__device__ void matmul(double* d, const double* x, const double* y, int s) {
  for (int e = threadIdx.x; e < s * s; e += kThreads) {
    const int i = e / s, j = e % s;
    double v = 0.0;
    for (int k = 0; k < s; ++k) v = fma(x[i * s + k], y[k * s + j], v);
    d[e] = v;
  }
  __syncthreads();
}

__global__ void __launch_bounds__(kThreads) poly_kernel(const StepParams a) {
  extern __shared__ double sh[];
  const Mat t = a.mats[blockIdx.x];
  const int s = t.s, n = s * s;
  double *g = sh, *q = sh + n, *x = sh + 2 * n, *y = sh + 3 * n;
  __shared__ double inv;
  for (int e = threadIdx.x; e < n; e += kThreads) {
    double v = 0.0;
    for (int k = 0; k < t.tiles; ++k) v += a.ws[t.gram + static_cast<int64_t>(k) * n + e];
    g[e] = v;
    x[e] = e % (s + 1) == 0 ? 1.0 : 0.0;
  }
  __syncthreads();
  if (threadIdx.x == 0) {
    double tr = 0.0;
    for (int i = 0; i < s; ++i) tr += g[i * s + i];
    inv = 1.0 / (sqrt(tr) + static_cast<double>(a.eps));
  }
  __syncthreads();
  for (int e = threadIdx.x; e < n; e += kThreads) g[e] *= inv * inv;
  __syncthreads();
  for (int it = 0; it < a.steps; ++it) {
    matmul(q, g, g, s);
    for (int e = threadIdx.x; e < n; e += kThreads) q[e] = (e % (s + 1) == 0 ? kA : 0.0) + kB * g[e] + kC * q[e];
    __syncthreads();
    matmul(y, q, x, s);
    double* o = x; x = y; y = o;
    if (it + 1 < a.steps) {
      matmul(y, q, g, s);
      matmul(g, q, y, s);
    }
  }
  for (int e = threadIdx.x; e < n; e += kThreads) a.ws[t.poly + e] = static_cast<float>(x[e] * inv);
}

__global__ void __launch_bounds__(kThreads) apply_kernel(const StepParams a) {
  __shared__ float u[kMaxShort][kSub + 1];
  __shared__ float pm[kMaxShort * kMaxShort];
  const Tile tile = a.tiles[blockIdx.x];
  const Mat t = a.mats[tile.mat];
  const float clip = clip_factor(a);
  const int64_t last = min(t.l, tile.first + a.piece);
  const float rows = t.tall ? t.l : t.s, cols = t.tall ? t.s : t.l;
  const float step = a.lr * (a.scale_mode == 0 ? 0.2f * sqrtf(fmaxf(rows, cols)) : sqrtf(fmaxf(1.0f, rows / cols)));
  const float keep = 1.0f - a.lr * a.wd;
  for (int e = threadIdx.x; e < t.s * t.s; e += kThreads) pm[e] = a.ws[t.poly + e];
  for (int64_t c0 = tile.first; c0 < last; c0 += kSub) {
    const int w = static_cast<int>(min(static_cast<int64_t>(kSub), last - c0));
    __syncthreads();
    for (int e = threadIdx.x; e < t.s * kSub; e += kThreads) {
      const int i = t.tall ? e % t.s : e / kSub, l = t.tall ? e / t.s : e % kSub;
      if (l < w) {
        const int64_t at = address(t, i, c0 + l);
        float v;
        if (a.m == nullptr) v = a.g[at] * clip;
        else v = a.nesterov ? a.beta * a.m[at] + (1.0f - a.beta) * (a.g[at] * clip) : a.m[at];
        u[i][l] = v;
        if (a.zero_grad) a.g[at] = 0.f;
      }
    }
    __syncthreads();
    for (int e = threadIdx.x; e < t.s * kSub; e += kThreads) {
      const int i = t.tall ? e % t.s : e / kSub, l = t.tall ? e / t.s : e % kSub;
      if (l < w) {
        float o = 0.f;
        for (int j = 0; j < t.s; ++j) o = fmaf(pm[i * t.s + j], u[j][l], o);
        const int64_t at = address(t, i, c0 + l);
        if (a.out != nullptr) a.out[at] = o;
        else a.p[at] = a.p[at] * keep - step * o;
      }
    }
  }
}

// ---- host side ---------------------------------------------------------------------------------
int make_plan(const char* name, const int64_t* rows, const int64_t* cols, int64_t count, k2q_matrices* out) {
  if (!rows || !cols || !out || count <= 0 || count > 0x7fffff) return fail(K2Q_EINVAL, "%s: bad arguments", name);
  k2q_matrices pl{};
  pl.count = count;
  for (int64_t i = 0; i < count; ++i) {
    const int64_t s = rows[i] < cols[i] ? rows[i] : cols[i], l = rows[i] < cols[i] ? cols[i] : rows[i];
    if (s < 1 || s > kMaxShort || l > 0x7fffff00LL)
      return fail(K2Q_EINVAL, "%s: matrix %lld is %lld x %lld; the short side must be 1 to %d", name, (long long)i,
                  (long long)rows[i], (long long)cols[i], kMaxShort);
    pl.total += s * l;
    if (s > pl.max_short) pl.max_short = static_cast<int32_t>(s);
  }
  // pieces of the long side: as long as they may be while every SM still gets four of them
  const int64_t wanted = 4 * 148;
  for (pl.piece = 2048; pl.piece > 128; pl.piece /= 2) {
    int64_t n = 0;
    for (int64_t i = 0; i < count; ++i) n += ((rows[i] < cols[i] ? cols[i] : rows[i]) + pl.piece - 1) / pl.piece;
    if (n >= wanted) break;
  }
  int64_t floats = 0;
  for (int64_t i = 0; i < count; ++i) {
    const int64_t s = rows[i] < cols[i] ? rows[i] : cols[i], l = rows[i] < cols[i] ? cols[i] : rows[i];
    const int64_t n = (l + pl.piece - 1) / pl.piece;
    pl.tiles += n;
    floats += (n + 1) * s * s;
  }
  if (pl.tiles > 0x7fffffffLL) return fail(K2Q_EINVAL, "%s: too many pieces", name);
  pl.workspace_bytes = floats * 4;
  pl.table_bytes = count * static_cast<int64_t>(sizeof(Mat)) + pl.tiles * static_cast<int64_t>(sizeof(Tile));
  *out = pl;
  return K2Q_OK;
}

bool off16(const void* ptr) { return (reinterpret_cast<uintptr_t>(ptr) & 15u) != 0; }

int run_steps(const char* name, const k2q_matrices* pl, const void* table, StepParams a, void* ws, int64_t ws_bytes, cudaStream_t s) {
  if (int rc = check_device_arch()) return rc;
  if (!pl || !table || off16(table) || pl->count <= 0) return fail(K2Q_EINVAL, "%s: no matrix table", name);
  if (!ws || off16(ws) || ws_bytes < pl->workspace_bytes) return fail(K2Q_EINVAL, "%s: workspace too small", name);
  if (a.steps < 0 || a.steps > 10) return fail(K2Q_EINVAL, "%s: steps %d not in [0,10]", name, a.steps);
  a.mats = static_cast<const Mat*>(table);
  a.tiles = reinterpret_cast<const Tile*>(a.mats + pl->count);
  a.piece = pl->piece;
  a.ws = static_cast<float*>(ws);
  const int poly_smem = 4 * pl->max_short * pl->max_short * 8;
  if (int rc = check_cuda(cudaFuncSetAttribute(poly_kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, poly_smem),
                          "cudaFuncSetAttribute(poly)"))
    return rc;
  const unsigned tiles = static_cast<unsigned>(pl->tiles);
  gram_kernel<<<tiles, kThreads, 0, s>>>(a);
  poly_kernel<<<static_cast<unsigned>(pl->count), kThreads, poly_smem, s>>>(a);
  apply_kernel<<<tiles, kThreads, 0, s>>>(a);
  return check_cuda(cudaGetLastError(), name);
}

}  // namespace
}  // namespace k2q

using namespace k2q;

extern "C" {

int k2q_matrices_plan(const int64_t* rows, const int64_t* cols, int64_t count, k2q_matrices* plan) {
  return make_plan("k2q_matrices_plan", rows, cols, count, plan);
}

int k2q_matrices_table(const int64_t* rows, const int64_t* cols, int64_t count, void* table_host, int64_t table_bytes) {
  k2q_matrices pl{};
  if (int rc = make_plan("k2q_matrices_table", rows, cols, count, &pl)) return rc;
  if (!table_host || table_bytes < pl.table_bytes) return fail(K2Q_EINVAL, "k2q_matrices_table: table too small");
  Mat* mats = static_cast<Mat*>(table_host);
  Tile* tiles = reinterpret_cast<Tile*>(mats + count);
  int64_t off = 0, floats = 0, nt = 0;
  for (int64_t i = 0; i < count; ++i) {
    Mat m{};
    m.tall = rows[i] > cols[i];
    m.s = static_cast<int32_t>(m.tall ? cols[i] : rows[i]);
    m.l = m.tall ? rows[i] : cols[i];
    m.off = off;
    m.tile0 = static_cast<int32_t>(nt);
    m.tiles = static_cast<int32_t>((m.l + pl.piece - 1) / pl.piece);
    m.gram = floats;
    floats += static_cast<int64_t>(m.tiles) * m.s * m.s;
    m.poly = floats;
    floats += static_cast<int64_t>(m.s) * m.s;
    off += m.s * m.l;
    mats[i] = m;
    for (int k = 0; k < m.tiles; ++k) tiles[nt++] = Tile{static_cast<int32_t>(i), 0, k * pl.piece};
  }
  return K2Q_OK;
}

int k2q_orthogonal_step(float* p, float* g, float* m, const k2q_matrices* plan, const void* table, float lr, float beta,
                        int nesterov, float weight_decay, int scale_mode, int steps, float eps, float max_norm,
                        const float* normsq_dev, int zero_grad, void* ws, int64_t ws_bytes, void* stream) {
  if (!p || !g || !m) return fail(K2Q_EINVAL, "k2q_orthogonal_step: NULL operand");
  if (scale_mode != 0 && scale_mode != 1) return fail(K2Q_EINVAL, "k2q_orthogonal_step: unknown scale mode %d", scale_mode);
  StepParams a{};
  a.p = p; a.g = g; a.m = m; a.lr = lr; a.beta = beta; a.nesterov = nesterov; a.wd = weight_decay; a.scale_mode = scale_mode;
  a.steps = steps; a.eps = eps; a.max_norm = max_norm; a.normsq = normsq_dev; a.zero_grad = zero_grad;
  return run_steps("k2q_orthogonal_step", plan, table, a, ws, ws_bytes, static_cast<cudaStream_t>(stream));
}

int k2q_orthogonalize(const float* u, float* out, const k2q_matrices* plan, const void* table, int steps, float eps, void* ws,
                      int64_t ws_bytes, void* stream) {
  if (!u || !out) return fail(K2Q_EINVAL, "k2q_orthogonalize: NULL operand");
  StepParams a{};
  a.g = const_cast<float*>(u); a.out = out; a.steps = steps; a.eps = eps;
  return run_steps("k2q_orthogonalize", plan, table, a, ws, ws_bytes, static_cast<cudaStream_t>(stream));
}

}  // extern "C"
