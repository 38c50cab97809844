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
//   gram    m' and the partial Gram matrices of pieces of the long side       12 B and S/2 FMA per element
//   poly    partials added, normalised, iterated; leaves P = (Q ... Q_0) / (||u||_F + eps)
//   apply   P u and the parameter step                                        16 B and S FMA per element
// gram and apply are bound by HBM up to S = 32 and by the fp32 pipe beyond.  Both keep a sub-block of 2048 elements in
// shared memory as it lies in memory, work on 4 x 4 register tiles with 16-byte shared reads (rows interleaved
// over the tiles and a row pitch that is an odd number of 16-byte pieces, so that eight lanes meet eight
// different pieces), and have the next sub-block in registers meanwhile.
// The S x S iteration is in 64 bits: P's entries reach a^steps, so what G_0 loses to rounding comes back up to
// that much larger in the weak directions.  G_0's products are summed in fp32 by each thread over its share of a piece
// (a few hundred terms), over threads in fp32, over pieces in 64 bits.  All sums run in a fixed order.
#include "k2q_common.cuh"

namespace k2q {
namespace {

constexpr int kMaxShort = 64;
constexpr int kThreads = 256;
constexpr int kVecs = 2;                       // 16-byte pieces of a sub-block per thread
constexpr double kA = 3.4445, kB = -4.7750, kC = 2.0315;

struct Mat {            // one entry of the device table
  int64_t off;          // first element in the flat buffers
  int64_t gram;         // first float of its partial Gram matrices in the workspace
  int64_t poly;         // first float of P [S4][S4]
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
  int aligned;          // the buffers' bases are 16-byte aligned
};

__host__ __device__ constexpr int up4(int s) { return (s + 3) & ~3; }
// 4 x 4 tiles of the upper triangle of a Gram matrix
__host__ __device__ constexpr int pairs_of(int s) { return (up4(s) / 4) * (up4(s) / 4 + 1) / 2; }
// positions of the long side per sub-block: 2048 elements, at least 32, a power of two
__host__ __device__ constexpr int block_of(int s) { return s <= 4 ? 512 : s <= 8 ? 256 : s <= 16 ? 128 : s <= 32 ? 64 : 32; }

__device__ __forceinline__ float clip_factor(const StepParams& a) {
  if (a.normsq == nullptr || !(a.max_norm > 0.f)) return 1.0f;
  return fminf(1.0f, a.max_norm / (sqrtf(__ldg(a.normsq)) + 1e-6f));
}

// A matrix as a CTA sees it: the sub-block is rows x width elements as stored (wide: S x block, tall: block x S).
struct Place {
  int s, s4, tall, block, width, pitch;
  int64_t row_stride, step;                    // elements from row to row, from sub-block to sub-block
  bool vec;                                    // 16-byte accesses fit
  __device__ __forceinline__ Place(const Mat& t, int aligned) {
    s = t.s; s4 = up4(s); tall = t.tall; block = block_of(s);
    width = tall ? s4 : block;
    pitch = ((width >> 2) & 1) ? width : width + 4;
    row_stride = tall ? s : t.l;
    step = tall ? static_cast<int64_t>(block) * s : block;
    vec = aligned && (t.off & 3) == 0 && ((tall ? static_cast<int64_t>(s) : t.l) & 3) == 0;
  }
};

__device__ __forceinline__ float4 ld4(const float* p) { return *reinterpret_cast<const float4*>(p); }

// The thread's share of a sub-block in registers: kVecs pieces of four elements (element e of piece k).
struct Share {
  int64_t at[kVecs];    // offset of the piece in the matrix, sub-block 0
  int sm[kVecs];        // place in shared memory
  int lrel[kVecs];      // its (first) position along the long side within the sub-block
  bool ok[kVecs];       // inside the sub-block
  __device__ __forceinline__ Share(const Place& pl) {
    const int per_row = pl.width >> 2, rows = pl.tall ? pl.block : pl.s;
#pragma unroll
    for (int k = 0; k < kVecs; ++k) {
      const int e = threadIdx.x + k * kThreads, r = e / per_row, c = (e - r * per_row) * 4;
      ok[k] = r < rows;
      at[k] = r * pl.row_stride + c;
      sm[k] = r * pl.pitch + c;
      lrel[k] = pl.tall ? r : c;
    }
  }
};

// Elements of a piece that exist: 4, or fewer at the end of a row or of the long side.
__device__ __forceinline__ int piece_len(const Place& pl, const Share& sh, int k, int left) {
  if (!sh.ok[k]) return 0;
  if (pl.tall) return sh.lrel[k] < left ? min(4, pl.s - (sh.sm[k] - (sh.lrel[k] * pl.pitch))) : 0;
  return max(0, min(4, left - sh.lrel[k]));
}
__device__ __forceinline__ float4 load_piece(const float* base, int n, bool vec) {
  if (vec && n == 4) return ld4(base);
  float4 v = make_float4(0.f, 0.f, 0.f, 0.f);
  if (n > 0) v.x = base[0];
  if (n > 1) v.y = base[1];
  if (n > 2) v.z = base[2];
  if (n > 3) v.w = base[3];
  return v;
}
__device__ __forceinline__ void store_piece(float* base, const float4& v, int n, bool vec) {
  if (vec && n == 4) {
    *reinterpret_cast<float4*>(base) = v;
    return;
  }
  if (n > 0) base[0] = v.x;
  if (n > 1) base[1] = v.y;
  if (n > 2) base[2] = v.z;
  if (n > 3) base[3] = v.w;
}
// m' (in place) and u of four elements
__device__ __forceinline__ float4 momentum4(const StepParams& a, float4 g, float4& m, float clip) {
  const float b = a.beta, c = 1.0f - a.beta;
  g.x *= clip; g.y *= clip; g.z *= clip; g.w *= clip;
  m.x = b * m.x + c * g.x; m.y = b * m.y + c * g.y; m.z = b * m.z + c * g.z; m.w = b * m.w + c * g.w;
  if (!a.nesterov) return m;
  return make_float4(b * m.x + c * g.x, b * m.y + c * g.y, b * m.z + c * g.z, b * m.w + c * g.w);
}
// u from g and the m' that is already stored
__device__ __forceinline__ float4 update4(const StepParams& a, const float4& g, const float4& m, float clip) {
  if (!a.nesterov) return m;
  const float b = a.beta, c = 1.0f - a.beta;
  return make_float4(b * m.x + c * (g.x * clip), b * m.y + c * (g.y * clip), b * m.z + c * (g.z * clip), b * m.w + c * (g.w * clip));
}

__host__ __device__ constexpr int sub_floats(int s, bool tall) {
  const int w = tall ? up4(s) : block_of(s), p = ((w >> 2) & 1) ? w : w + 4;
  return p * (tall ? block_of(s) : up4(s));
}
constexpr int max_sub_floats() {
  int best = 0;
  for (int s = 1; s <= kMaxShort; ++s) {
    if (sub_floats(s, false) > best) best = sub_floats(s, false);
    if (sub_floats(s, true) > best) best = sub_floats(s, true);
  }
  return best;
}
constexpr int kMaxSub = max_sub_floats();

__global__ void __launch_bounds__(kThreads) gram_kernel(const StepParams a) {
  __shared__ __align__(16) float u[kMaxSub > kThreads * 16 ? kMaxSub : kThreads * 16];
  const Tile tile = a.tiles[blockIdx.x];
  const Mat t = a.mats[tile.mat];
  const Place pl(t, a.aligned);
  const Share sh(pl);
  const float clip = clip_factor(a);
  const int64_t last = min(t.l, tile.first + a.piece);
  const int nt = pl.s4 >> 2, pairs = pairs_of(t.s), kgroups = kThreads / pairs;
  // this thread's tile (ti <= tj) and share of the positions
  const int kg = threadIdx.x / pairs;
  int ti = 0, tj = threadIdx.x - kg * pairs;
  while (tj >= nt - ti) { tj -= nt - ti; ++ti; }
  tj += ti;
  const bool works = kg < kgroups;
  float acc[4][4] = {};

  const int64_t origin = t.off + (t.tall ? tile.first * t.s : tile.first);
  float4 rg[kVecs], rm[kVecs];
  int rn[kVecs];
  int64_t base = origin;
  auto fetch = [&](int64_t c0) {
    const int left = static_cast<int>(min(static_cast<int64_t>(pl.block), last - c0));
#pragma unroll
    for (int k = 0; k < kVecs; ++k) {
      rn[k] = piece_len(pl, sh, k, left);
      rg[k] = load_piece(a.g + base + sh.at[k], rn[k], pl.vec);
      if (a.m != nullptr) rm[k] = load_piece(a.m + base + sh.at[k], rn[k], pl.vec);
    }
  };
  // rows of the padding (wide: S .. S4) stay zero
  for (int e = threadIdx.x; e < (pl.tall ? 0 : (pl.s4 - pl.s) * pl.pitch); e += kThreads) u[pl.s * pl.pitch + e] = 0.f;
  fetch(tile.first);
  for (int64_t c0 = tile.first; c0 < last; c0 += pl.block) {
#pragma unroll
    for (int k = 0; k < kVecs; ++k) {
      float4 v = rg[k];
      if (a.m != nullptr) {
        v = momentum4(a, rg[k], rm[k], clip);
        store_piece(a.m + base + sh.at[k], rm[k], rn[k], pl.vec);
        if (rn[k] < 4) {                       // positions that do not exist count as zero
          if (rn[k] < 1) v.x = 0.f;
          if (rn[k] < 2) v.y = 0.f;
          if (rn[k] < 3) v.z = 0.f;
          v.w = 0.f;
        }
      }
      if (sh.ok[k]) *reinterpret_cast<float4*>(u + sh.sm[k]) = v;
    }
    base += pl.step;
    __syncthreads();
    if (c0 + pl.block < last) fetch(c0 + pl.block);
    if (works) {
      if (pl.tall) {
        for (int l = kg; l < pl.block; l += kgroups) {
          const float4 x = ld4(u + l * pl.pitch + 4 * ti), y = ld4(u + l * pl.pitch + 4 * tj);
          const float xv[4] = {x.x, x.y, x.z, x.w}, yv[4] = {y.x, y.y, y.z, y.w};
#pragma unroll
          for (int i = 0; i < 4; ++i)
#pragma unroll
            for (int j = 0; j < 4; ++j) acc[i][j] = fmaf(xv[i], yv[j], acc[i][j]);
        }
      } else {
        for (int l = 4 * kg; l < pl.block; l += 4 * kgroups) {
          float4 x[4], y[4];
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            x[i] = ld4(u + (ti + i * nt) * pl.pitch + l);
            y[i] = ld4(u + (tj + i * nt) * pl.pitch + l);
          }
#pragma unroll
          for (int i = 0; i < 4; ++i)
#pragma unroll
            for (int j = 0; j < 4; ++j)
              acc[i][j] = fmaf(x[i].w, y[j].w, fmaf(x[i].z, y[j].z, fmaf(x[i].y, y[j].y, fmaf(x[i].x, y[j].x, acc[i][j]))));
        }
      }
    }
    __syncthreads();
  }
  // the shares of the positions, added in order
  if (works) {
#pragma unroll
    for (int i = 0; i < 4; ++i)
#pragma unroll
      for (int j = 0; j < 4; ++j) u[(kg * 16 + i * 4 + j) * pairs + (threadIdx.x - kg * pairs)] = acc[i][j];
  }
  __syncthreads();
  float* part = a.ws + t.gram + static_cast<int64_t>(blockIdx.x - t.tile0) * pairs * 16;
  for (int e = threadIdx.x; e < pairs * 16; e += kThreads) {
    float v = u[e];
    for (int k = 1; k < kgroups; ++k) v += u[k * pairs * 16 + e];
    part[e] = v;
  }
}

// d = x y for S4 x S4 matrices (padding rows and columns are zero), 4 x 2 register tiles
__device__ __forceinline__ void matmul(double* d, const double* x, const double* y, int s4) {
  const int across = s4 >> 1, tiles = (s4 >> 2) * across;
  for (int e = threadIdx.x; e < tiles; e += kThreads) {
    const int i = e / across * 4, j = (e - e / across * across) * 2;
    double v[4][2] = {};
    for (int k = 0; k < s4; ++k) {
      const double2 b = *reinterpret_cast<const double2*>(y + k * s4 + j);
#pragma unroll
      for (int r = 0; r < 4; ++r) {
        const double c = x[(i + r) * s4 + k];
        v[r][0] = fma(c, b.x, v[r][0]);
        v[r][1] = fma(c, b.y, v[r][1]);
      }
    }
#pragma unroll
    for (int r = 0; r < 4; ++r) *reinterpret_cast<double2*>(d + (i + r) * s4 + j) = make_double2(v[r][0], v[r][1]);
  }
  __syncthreads();
}

__global__ void __launch_bounds__(kThreads) poly_kernel(const StepParams a) {
  extern __shared__ __align__(16) double sh[];
  __shared__ double inv;
  const Mat t = a.mats[blockIdx.x];
  const int s4 = up4(t.s), n = s4 * s4, nt = s4 >> 2, pairs = pairs_of(t.s);
  double *g = sh, *q = sh + n, *x = sh + 2 * n, *y = sh + 3 * n;
  for (int e = threadIdx.x; e < pairs * 16; e += kThreads) {
    double v = 0.0;
    const float* part = a.ws + t.gram + e;
#pragma unroll 8
    for (int k = 0; k < t.tiles; ++k) v += part[static_cast<int64_t>(k) * pairs * 16];
    const int in = e / pairs;
    int ti = 0, tj = e - in * pairs;
    while (tj >= nt - ti) { tj -= nt - ti; ++ti; }
    tj += ti;
    // rows of a tile: neighbours where the matrix is tall, every nt-th where it is wide
    const int i = t.tall ? 4 * ti + (in >> 2) : ti + (in >> 2) * nt, j = t.tall ? 4 * tj + (in & 3) : tj + (in & 3) * nt;
    g[i * s4 + j] = v;
    g[j * s4 + i] = v;
  }
  __syncthreads();
  if (threadIdx.x < 32) {
    double tr = 0.0;
    for (int i = threadIdx.x; i < s4; i += 32) tr += g[i * s4 + i];
    for (int o = 16; o > 0; o >>= 1) tr += __shfl_xor_sync(0xffffffffu, tr, o);
    if (threadIdx.x == 0) inv = 1.0 / (sqrt(tr) + static_cast<double>(a.eps));
  }
  __syncthreads();
  const double f = inv;
  for (int e = threadIdx.x; e < n; e += kThreads) {
    const bool diag = e / s4 == e % s4 && e / s4 < t.s;
    g[e] *= f * f;
    if (a.steps == 0) x[e] = diag ? 1.0 : 0.0;
  }
  __syncthreads();
  for (int it = 0; it < a.steps; ++it) {
    double* dst = it == 0 ? x : q;             // the first factor is the product so far
    matmul(dst, g, g, s4);
    for (int e = threadIdx.x; e < n; e += kThreads) {
      const bool diag = e / s4 == e % s4 && e / s4 < t.s;
      dst[e] = (diag ? kA : 0.0) + kB * g[e] + kC * dst[e];
    }
    __syncthreads();
    if (it > 0) {
      matmul(y, q, x, s4);
      double* o = x; x = y; y = o;
    }
    if (it + 1 < a.steps) {
      const double* f1 = it == 0 ? x : q;
      matmul(y, f1, g, s4);
      matmul(g, f1, y, s4);
    }
  }
  for (int e = threadIdx.x; e < n; e += kThreads) a.ws[t.poly + e] = static_cast<float>(x[e] * f);
}

__global__ void __launch_bounds__(kThreads) apply_kernel(const StepParams a) {
  extern __shared__ __align__(16) float smem[];
  const Tile tile = a.tiles[blockIdx.x];
  const Mat t = a.mats[tile.mat];
  const Place pl(t, a.aligned);
  const Share sh(pl);
  const float clip = clip_factor(a);
  const int64_t last = min(t.l, tile.first + a.piece);
  const float rows = t.tall ? t.l : t.s, cols = t.tall ? t.s : t.l;
  const float step = a.lr * (a.scale_mode == 0 ? 0.2f * sqrtf(fmaxf(rows, cols)) : sqrtf(fmaxf(1.0f, rows / cols)));
  const float keep = 1.0f - a.lr * a.wd;
  float* u = smem;                                             // sub-block, replaced by its product
  float* pm = smem + kMaxSub;                         // P [S4][pp]
  const int pp = ((pl.s4 >> 2) & 1) ? pl.s4 : pl.s4 + 4;
  for (int e = threadIdx.x; e < pl.s4 * pl.s4; e += kThreads) pm[e / pl.s4 * pp + e % pl.s4] = a.ws[t.poly + e];
  for (int e = threadIdx.x; e < (pl.tall ? 0 : (pl.s4 - pl.s) * pl.pitch); e += kThreads) u[pl.s * pl.pitch + e] = 0.f;

  // out = A B with A's rows (wide: P, tall: the sub-block) interleaved over the tiles, B's columns neighbours
  const float *am = pl.tall ? u : pm, *bm = pl.tall ? pm : u;
  const int ap = pl.tall ? pl.pitch : pp, bp = pl.tall ? pp : pl.pitch;
  const int out_rows = pl.tall ? pl.block : pl.s4, rt = out_rows >> 2, ct = pl.width >> 2;
  const int tiles = rt * ct;                                   // 2048 / 16: half of the threads multiply

  float4 rg[kVecs], rm[kVecs], rp[kVecs];
  int rn[kVecs];
  int64_t base = t.off + (t.tall ? tile.first * t.s : tile.first);
  auto fetch = [&](int64_t c0) {
    const int left = static_cast<int>(min(static_cast<int64_t>(pl.block), last - c0));
#pragma unroll
    for (int k = 0; k < kVecs; ++k) {
      rn[k] = piece_len(pl, sh, k, left);
      if (a.m == nullptr || a.nesterov) rg[k] = load_piece(a.g + base + sh.at[k], rn[k], pl.vec);
      if (a.m != nullptr) rm[k] = load_piece(a.m + base + sh.at[k], rn[k], pl.vec);
      if (a.out == nullptr) rp[k] = load_piece(a.p + base + sh.at[k], rn[k], pl.vec);
    }
  };
  fetch(tile.first);
  for (int64_t c0 = tile.first; c0 < last; c0 += pl.block) {
    float4 cur_p[kVecs];
    int cur_n[kVecs];
    const int64_t cur = base;
    __syncthreads();
#pragma unroll
    for (int k = 0; k < kVecs; ++k) {
      if (sh.ok[k]) *reinterpret_cast<float4*>(u + sh.sm[k]) = a.m == nullptr ? rg[k] : update4(a, rg[k], rm[k], clip);
      cur_p[k] = rp[k];
      cur_n[k] = rn[k];
    }
    __syncthreads();
    base += pl.step;
    if (c0 + pl.block < last) fetch(c0 + pl.block);
    float acc[4][4];
    int ri = 0, ci = 0;
    const bool works = static_cast<int>(threadIdx.x) < tiles;
    if (works) {
      ri = threadIdx.x / ct;
      ci = (threadIdx.x - ri * ct) * 4;
#pragma unroll
      for (int i = 0; i < 4; ++i)
#pragma unroll
        for (int j = 0; j < 4; ++j) acc[i][j] = 0.f;
      for (int k = 0; k < pl.s4; k += 4) {
        float4 x[4], y[4];
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          x[i] = ld4(am + (ri + i * rt) * ap + k);
          y[i] = ld4(bm + (k + i) * bp + ci);
        }
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const float xv[4] = {x[i].x, x[i].y, x[i].z, x[i].w};
#pragma unroll
          for (int kk = 0; kk < 4; ++kk) {
            acc[i][0] = fmaf(xv[kk], y[kk].x, acc[i][0]);
            acc[i][1] = fmaf(xv[kk], y[kk].y, acc[i][1]);
            acc[i][2] = fmaf(xv[kk], y[kk].z, acc[i][2]);
            acc[i][3] = fmaf(xv[kk], y[kk].w, acc[i][3]);
          }
        }
      }
    }
    __syncthreads();
    if (works) {
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const int r = ri + i * rt;
        if (pl.tall || r < pl.s) *reinterpret_cast<float4*>(u + r * pl.pitch + ci) = make_float4(acc[i][0], acc[i][1], acc[i][2], acc[i][3]);
      }
    }
    __syncthreads();
#pragma unroll
    for (int k = 0; k < kVecs; ++k) {
      if (!sh.ok[k]) continue;
      float4 o = ld4(u + sh.sm[k]);
      if (a.out != nullptr) {
        store_piece(a.out + cur + sh.at[k], o, cur_n[k], pl.vec);
      } else {
        const float4 p0 = cur_p[k];
        o.x = p0.x * keep - step * o.x; o.y = p0.y * keep - step * o.y;
        o.z = p0.z * keep - step * o.z; o.w = p0.w * keep - step * o.w;
        store_piece(a.p + cur + sh.at[k], o, cur_n[k], pl.vec);
        if (a.zero_grad) store_piece(a.g + cur + sh.at[k], make_float4(0.f, 0.f, 0.f, 0.f), cur_n[k], pl.vec);
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
  // pieces of the long side: as long as they may be while the largest GPUs' SMs still get four of them each
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
    const int32_t s32 = static_cast<int32_t>(s);
    floats += n * pairs_of(s32) * 16 + up4(s32) * up4(s32);
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
  a.aligned = !off16(a.p) && !off16(a.g) && !off16(a.m) && !off16(a.out);
  const int s4 = up4(pl->max_short);
  const int poly_smem = 4 * s4 * s4 * 8, apply_smem = (kMaxSub + s4 * (s4 + 4)) * 4;
  if (int rc = check_cuda(cudaFuncSetAttribute(poly_kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, poly_smem),
                          "cudaFuncSetAttribute(poly)"))
    return rc;
  const unsigned tiles = static_cast<unsigned>(pl->tiles);
  gram_kernel<<<tiles, kThreads, 0, s>>>(a);
  poly_kernel<<<static_cast<unsigned>(pl->count), kThreads, poly_smem, s>>>(a);
  apply_kernel<<<tiles, kThreads, apply_smem, s>>>(a);
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
    floats += static_cast<int64_t>(m.tiles) * pairs_of(m.s) * 16;
    m.poly = floats;
    floats += up4(m.s) * up4(m.s);
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
