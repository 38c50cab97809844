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
// Neither saturates one unit (figures below): shared memory is the busiest.  Both work on sub-blocks of 4096 elements in
// shared memory with 4 x 4 register tiles and packed fp32 pairs: a pair holds two neighbouring positions of the
// CONTRACTED index, so no operand has to be broadcast and one instruction does two multiply-adds.  Where that index
// is the contiguous one in memory (gram of a wide matrix, apply of a tall one) the sub-block stays as it is
// ("natural"), otherwise neighbouring rows are interleaved on the way in ("paired").  The next sub-block travels
// meanwhile by asynchronous copies into a raw area where every thread reads back only what it copied itself.
// The S x S iteration is in 64 bits, on the fp64 tensor instructions (8 x 8 tiles of the upper triangle): P's entries reach
// a^steps, so what G_0 loses to rounding comes back up to that much larger in the weak directions.  G_0's products are summed
// in fp32 by each thread over its share of a piece (10 terms of each sub-block at rank 32, 32 at rank 64, of the up to 32
// sub-blocks of a piece: 1024 at most), over threads in fp32, over pieces in 64 bits.  All sums run in a fixed order.
// Relative error of X_5 against 64 bits on gradients with one strong direction: 0.7e-6 with one sub-block to a piece (rank
// 57), 3e-6 with 7 to 13 (rank 32, 64), 5e-6 with 30 (rank 64); the iteration on the data itself in fp32 has 1e-6.
// Measured on a B200 (copy bandwidth 6.55 TB/s), 224 adapter matrices, 58.7 M elements:
//   rank 32   353 us in all (launched one by one: gram 139, poly 25, apply 200).  20 B per element, which a single pass
//             could not do without, would take 179 us, the 28 B of two passes 251
//   rank 16   144 us for 22 M elements (67 at 20 B each)      rank 64, half the matrices, 58.7 M elements   568 us
// Counters of gram / apply at rank 32: shared-memory wavefronts 71 / 65 % of the pipe's, issue 59 / 54 %, DRAM 58 / 55 %, fp32
// pipe 38 / 37 %, at 22 / 15 warps per SM: shared memory is the busiest and no unit is full.  Taking apply's pieces
// backwards, to find the last of gram's in L2, saved 5 % of its reads and 0.4 % of the time, and is not done.  At rank 64:
// 73 / 71 %, issue 50 / 53 %, DRAM 36 / 37 %, fp32 pipe 42 / 46 %; gram waits most at its barriers.  The iteration takes
// 52 us there, on one SM per matrix.  apply spills 8 bytes of a thread at 128 registers.
#include "k2q_common.cuh"

namespace k2q {
namespace {

constexpr int kMaxShort = 64;
constexpr int kThreads = 256;
constexpr int kUnits = 2;                      // two rows by four columns of a sub-block, per thread
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
struct Tile { int32_t mat; int32_t pad; int64_t first; };   // positions of the long side from `first` on

struct StepParams {
  const Mat* mats; const Tile* tiles; int64_t piece;   // sub-blocks per piece
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
// positions of the long side per sub-block: up to 4096 elements, a power of two
__host__ __device__ constexpr int block_of(int s) { return s <= 4 ? 1024 : s <= 8 ? 512 : s <= 16 ? 256 : s <= 32 ? 128 : 64; }
__host__ __device__ constexpr int odd_pitch(int w) { return ((w >> 2) & 1) ? w : w + 4; }

__device__ __forceinline__ float clip_factor(const StepParams& a) {
  if (a.normsq == nullptr || !(a.max_norm > 0.f)) return 1.0f;
  return fminf(1.0f, a.max_norm / (sqrtf(__ldg(a.normsq)) + 1e-6f));
}

// A matrix as a CTA sees it: the sub-block is rows x width elements as stored (wide: S4 x block, tall: block x S4).
// In shared memory
//   natural   row r at r * pitch; the pitch is an odd number of 16-byte pieces, so that eight lanes on eight rows meet
//             eight different pieces
//   paired    rows 2r and 2r + 1 together at r * 2 * width: element pairs of columns 4c, 4c + 1 at 4c, those of columns
//             4c + 2, 4c + 3 at width + 4c
struct Place {
  int s, s4, tall, block, width, rows, pitch;
  int64_t row_stride, step;                    // elements from row to row, from sub-block to sub-block
  bool vec;                                    // 16-byte accesses fit
  // orientation and block come in as constants: the kernels' bodies are compiled for each
  __device__ __forceinline__ Place(const Mat& t, int aligned, bool tall_, int block_) {
    s = t.s; s4 = up4(s); tall = tall_; block = block_;
    width = tall ? s4 : block;
    rows = tall ? block : s4;
    pitch = odd_pitch(width);
    row_stride = tall ? s : t.l;
    step = tall ? static_cast<int64_t>(block) * s : block;
    vec = aligned && (t.off & 3) == 0 && ((tall ? static_cast<int64_t>(s) : t.l) & 3) == 0;
  }
  // elements of the four at (row, col .. col + 3) that exist, `left` positions of the long side remaining
  __device__ __forceinline__ int len(int row, int col, int left) const {
    const bool in = tall ? row < left : row < s;
    return in ? max(0, min(4, (tall ? s : left) - col)) : 0;
  }
};

__device__ __forceinline__ float4 ld4(const float* p) { return *reinterpret_cast<const float4*>(p); }
__device__ __forceinline__ ulonglong2 ldp(const float* p) { return *reinterpret_cast<const ulonglong2*>(p); }

// Requests four elements at base (n of them exist, the others become zero) into 16 bytes of shared memory.
__device__ __forceinline__ void copy_piece(uint32_t dst, const float* base, int n, bool vec) {
  if (vec) {
    cp_async16(dst, base, n == 4 ? 16u : 0u);
  } else {
#pragma unroll
    for (int e = 0; e < 4; ++e)
      asm volatile("cp.async.ca.shared.global [%0], [%1], 4, %2;" ::"r"(dst + 4 * e), "l"(e < n ? base + e : base), "r"(e < n ? 4 : 0) : "memory");
  }
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

// The thread's share of a sub-block: kUnits times the same four columns of two neighbouring rows.
// Piece k of it is row row[k / 2] + k % 2.
struct Share {
  int row[kUnits], col[kUnits];
  int64_t at[kUnits];                          // offset of piece 2k; piece 2k + 1 is one row further
  bool ok[kUnits];
  bool full[2 * kUnits];                       // the piece exists whole in a sub-block that is whole (16-byte accesses)
  __device__ __forceinline__ Share(const Place& pl) {
    const int per_row = pl.width >> 2;
#pragma unroll
    for (int k = 0; k < kUnits; ++k) {
      const int e = threadIdx.x + k * kThreads, r = e / per_row;
      row[k] = 2 * r;
      col[k] = (e - r * per_row) * 4;
      ok[k] = 2 * r < pl.rows;
      at[k] = row[k] * pl.row_stride + col[k];
      full[2 * k] = ok[k] && pl.len(row[k], col[k], pl.block) == 4;
      full[2 * k + 1] = ok[k] && pl.len(row[k] + 1, col[k], pl.block) == 4;
    }
  }
  __device__ __forceinline__ void store_natural(float* u, const Place& pl, int k, const float4& a, const float4& b) const {
    if (!ok[k]) return;
    *reinterpret_cast<float4*>(u + row[k] * pl.pitch + col[k]) = a;
    *reinterpret_cast<float4*>(u + (row[k] + 1) * pl.pitch + col[k]) = b;
  }
  __device__ __forceinline__ void store_paired(float* u, const Place& pl, int k, const float4& a, const float4& b) const {
    if (!ok[k]) return;
    float* at = u + row[k] * pl.width + col[k];
    *reinterpret_cast<float4*>(at) = make_float4(a.x, b.x, a.y, b.y);
    *reinterpret_cast<float4*>(at + pl.width) = make_float4(a.z, b.z, a.w, b.w);
  }
};
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

constexpr int max_sub_floats() {
  int best = 0;
  for (int s = 1; s <= kMaxShort; ++s) {
    const int wide = up4(s) * odd_pitch(block_of(s)), tall = block_of(s) * odd_pitch(up4(s));
    if (wide > best) best = wide;
    if (tall > best) best = tall;
  }
  return best;
}
constexpr int kMaxSub = max_sub_floats();
static_assert(kThreads * 16 <= kMaxSub, "the gram kernel adds its threads' shares in the sub-block's place");

constexpr int kRaw = 2 * kUnits * kThreads * 16;               // bytes of one buffer's raw sub-block
constexpr int kGramSmem = 2 * kRaw + kMaxSub * 4;

template <bool TALL, int BLOCK>
__device__ __forceinline__ void gram_body(const StepParams& a, const Tile& tile, const Mat& t, float* smem) {
  float* u = smem;
  float* raw = smem + kMaxSub + threadIdx.x * 4;               // piece k of this thread: g at k, m at 2 * kUnits + k
  const uint32_t raw_u32 = smem_u32(raw);
  const Place pl(t, a.aligned, TALL, BLOCK);
  const Share sh(pl);
  const float clip = clip_factor(a);
  const int64_t last = min(t.l, tile.first + a.piece * BLOCK);
  const int nt = pl.s4 >> 2, pairs = pairs_of(t.s), kgroups = kThreads / pairs;
  // this thread's tile (ti <= tj) and share of the positions
  const int kg = threadIdx.x / pairs, mine = threadIdx.x - kg * pairs;
  int ti = 0, tj = mine;
  while (tj >= nt - ti) { tj -= nt - ti; ++ti; }
  tj += ti;
  const bool works = kg < kgroups;
  uint64_t acc[4][4] = {};                     // sums over the even and over the odd positions

  int64_t base = t.off + (t.tall ? tile.first * t.s : tile.first);
  const bool has_m = a.m != nullptr;
  auto fetch = [&](int64_t at, int left) {
    if (pl.vec && left == pl.block) {          // whole sub-block: what exists was settled beforehand
#pragma unroll
      for (int k = 0; k < 2 * kUnits; ++k) {
        const int64_t o = at + sh.at[k >> 1] + (k & 1) * pl.row_stride;
        if (sh.full[k]) {
          cp_async16(raw_u32 + k * (kThreads * 16), a.g + o, 16);
          if (has_m) cp_async16(raw_u32 + kRaw + k * (kThreads * 16), a.m + o, 16);
        }
      }
    } else {
#pragma unroll 1
      for (int k = 0; k < 2 * kUnits; ++k) {
        const int row = 2 * ((threadIdx.x + (k >> 1) * kThreads) / (pl.width >> 2)) + (k & 1);
        const int col = (threadIdx.x + (k >> 1) * kThreads) % (pl.width >> 2) * 4;
        const int n = row < pl.rows ? pl.len(row, col, left) : 0;
        const int64_t o = n > 0 ? at + row * pl.row_stride + col : 0;
        copy_piece(raw_u32 + k * (kThreads * 16), a.g + o, n, pl.vec);
        if (has_m) copy_piece(raw_u32 + kRaw + k * (kThreads * 16), a.m + o, n, pl.vec);
      }
    }
    cp_async_commit();
  };
  auto left_of = [&](int64_t c0) { return static_cast<int>(min(static_cast<int64_t>(pl.block), last - c0)); };
#pragma unroll
  for (int k = 0; k < 4 * kUnits; ++k) *reinterpret_cast<float4*>(raw + k * (kThreads * 4)) = make_float4(0.f, 0.f, 0.f, 0.f);
  fetch(base, left_of(tile.first));
  for (int64_t c0 = tile.first; c0 < last; c0 += pl.block) {
    const int left = left_of(c0);
    const bool whole = pl.vec && left == pl.block;
    cp_async_wait<0>();
#pragma unroll
    for (int k = 0; k < kUnits; ++k) {
      float4 v[2];
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        v[h] = ld4(raw + (2 * k + h) * (kThreads * 4));
        if (has_m) {
          float4 m = ld4(raw + (2 * kUnits + 2 * k + h) * (kThreads * 4));
          v[h] = momentum4(a, v[h], m, clip);
          float* out = a.m + base + sh.at[k] + h * pl.row_stride;
          if (whole) {
            if (sh.full[2 * k + h]) *reinterpret_cast<float4*>(out) = m;
            else v[h] = make_float4(0.f, 0.f, 0.f, 0.f);
          } else {
            const int n = sh.ok[k] ? pl.len(sh.row[k] + h, sh.col[k], left) : 0;
            store_piece(out, m, n, pl.vec);
            if (n < 4) {                       // positions that do not exist count as zero, whatever the clip factor is
              if (n < 1) v[h].x = 0.f;
              if (n < 2) v[h].y = 0.f;
              if (n < 3) v[h].z = 0.f;
              v[h].w = 0.f;
            }
          }
        }
      }
      if (pl.tall) sh.store_paired(u, pl, k, v[0], v[1]);
      else sh.store_natural(u, pl, k, v[0], v[1]);
    }
    base += pl.step;
    __syncthreads();
    if (c0 + pl.block < last) fetch(base, left_of(c0 + pl.block));
    if (works) {
      if (pl.tall) {
        const float *xp = u + 4 * ti, *yp = u + 4 * tj;
#pragma unroll 2
        for (int l = kg; l < pl.block / 2; l += kgroups) {
          const float *xr = xp + l * 2 * pl.width, *yr = yp + l * 2 * pl.width;
          const ulonglong2 x0 = ldp(xr), x1 = ldp(xr + pl.width), y0 = ldp(yr), y1 = ldp(yr + pl.width);
          const uint64_t x[4] = {x0.x, x0.y, x1.x, x1.y}, y[4] = {y0.x, y0.y, y1.x, y1.y};
#pragma unroll
          for (int i = 0; i < 4; ++i)
#pragma unroll
            for (int j = 0; j < 4; ++j) acc[i][j] = fma_f32x2(x[i], y[j], acc[i][j]);
        }
      } else {
        const float *xp = u + ti * pl.pitch, *yp = u + tj * pl.pitch;
        const int hop = nt * pl.pitch;
        for (int l = 4 * kg; l < pl.block; l += 4 * kgroups) {
          ulonglong2 y[4];
#pragma unroll
          for (int j = 0; j < 4; ++j) y[j] = ldp(yp + j * hop + l);
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            const ulonglong2 x = ldp(xp + i * hop + l);
#pragma unroll
            for (int j = 0; j < 4; ++j) acc[i][j] = fma_f32x2(x.y, y[j].y, fma_f32x2(x.x, y[j].x, acc[i][j]));
          }
        }
      }
    }
    __syncthreads();
  }
  pdl_launch_dependents();                     // the next kernel's blocks may line up; they wait for this one's end
  // the shares of the positions, added in order
  if (works) {
#pragma unroll
    for (int i = 0; i < 4; ++i)
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        float lo, hi;
        unpack_f32x2(acc[i][j], lo, hi);
        u[(kg * 16 + i * 4 + j) * pairs + mine] = lo + hi;
      }
  }
  __syncthreads();
  float* part = a.ws + t.gram + static_cast<int64_t>(blockIdx.x - t.tile0) * pairs * 16;
  for (int e = threadIdx.x; e < pairs * 16; e += kThreads) {
    float v = u[e];
    for (int k = 1; k < kgroups; ++k) v += u[k * pairs * 16 + e];
    part[e] = v;
  }
}

#define K2Q_BY_SHAPE(body)                                              \
  if (t.tall) {                                                         \
    switch (block_of(t.s)) {                                            \
      case 1024: body<true, 1024>(a, tile, t, smem); break;             \
      case 512: body<true, 512>(a, tile, t, smem); break;               \
      case 256: body<true, 256>(a, tile, t, smem); break;               \
      case 128: body<true, 128>(a, tile, t, smem); break;               \
      default: body<true, 64>(a, tile, t, smem); break;                 \
    }                                                                   \
  } else {                                                              \
    switch (block_of(t.s)) {                                            \
      case 1024: body<false, 1024>(a, tile, t, smem); break;            \
      case 512: body<false, 512>(a, tile, t, smem); break;              \
      case 256: body<false, 256>(a, tile, t, smem); break;              \
      case 128: body<false, 128>(a, tile, t, smem); break;              \
      default: body<false, 64>(a, tile, t, smem); break;                \
    }                                                                   \
  }

__global__ void __launch_bounds__(kThreads, 3) gram_kernel(const StepParams a) {
  extern __shared__ __align__(16) float smem[];
  pdl_wait();
  const Tile tile = a.tiles[blockIdx.x];
  const Mat t = a.mats[tile.mat];
  K2Q_BY_SHAPE(gram_body)
}

// S x S matrices of the iteration in shared memory: S8 rows, the padding zero; the pitch lets the 32 lanes of a
// fragment read (8 rows, 4 neighbours each) meet all banks.
__host__ __device__ constexpr int up8(int s) { return (s + 7) & ~7; }
__host__ __device__ constexpr int pitch64(int s) { return ((s + 15) & ~15) + 4; }

// A warp's 8 x 8 tiles of the upper triangle (it takes every WARPS-th), as element offsets in the shared matrices.  Eight
// warps and two tiles each cover S = 32 and leave room for three matrices on an SM; beyond, 16 warps shorten the chain.
template <int WARPS, int TILES>
struct PolyTiles {
  int n, pitch;
  int xa[TILES], yb[TILES], ij[TILES], ji[TILES];
  bool up0[TILES], up1[TILES];       // this lane's two entries lie on or above the diagonal
  bool diag0[TILES], diag1[TILES];
  __device__ __forceinline__ PolyTiles(int s) {
    const int n8 = up8(s) >> 3, lane = threadIdx.x & 31, r = lane >> 2, q = lane & 3, pairs = n8 * (n8 + 1) / 2;
    pitch = pitch64(s);
    n = 0;
#pragma unroll
    for (int k = 0; k < TILES; ++k) {
      int ti = 0, tj = (threadIdx.x >> 5) + k * WARPS;
      if (tj < pairs) n = k + 1;
      else tj = 0;
      while (tj >= n8 - ti) { tj -= n8 - ti; ++ti; }
      tj += ti;
      const int i = 8 * ti + r, j = 8 * tj + 2 * q;
      xa[k] = i * pitch + q;
      yb[k] = (8 * tj + r) * pitch + q;
      ij[k] = i * pitch + j;
      ji[k] = j * pitch + i;
      up0[k] = i <= j;
      up1[k] = i <= j + 1;
      diag0[k] = i == j && i < s;
      diag1[k] = i == j + 1 && i < s;
    }
  }
};

// For two commuting symmetric matrices: d = x y, or with FACTOR d = a I + b y + c x y; computed on the upper triangle and
// mirrored.  x y is symmetric up to rounding in 64 bits, so y's columns may be read as its rows.
template <bool FACTOR, int WARPS, int TILES>
__device__ __forceinline__ void poly_step(double* d, const double* x, const double* y, const PolyTiles<WARPS, TILES>& t, int s8) {
#pragma unroll
  for (int k = 0; k < TILES; ++k) {
    if (k >= t.n) break;
    double c[2][2] = {};
    const double *xa = x + t.xa[k], *yb = y + t.yb[k];
#pragma unroll 4
    for (int l = 0; l < s8; l += 8)
#pragma unroll
      for (int h = 0; h < 2; ++h)
        asm("mma.sync.aligned.m8n8k4.row.col.f64.f64.f64.f64 {%0,%1}, {%2}, {%3}, {%0,%1};"
            : "+d"(c[h][0]), "+d"(c[h][1])
            : "d"(xa[l + 4 * h]), "d"(yb[l + 4 * h]));
    double c0 = c[0][0] + c[1][0], c1 = c[0][1] + c[1][1];
    if (FACTOR) {
      const double2 y2 = *reinterpret_cast<const double2*>(y + t.ij[k]);
      c0 = kC * c0 + kB * y2.x + (t.diag0[k] ? kA : 0.0);
      c1 = kC * c1 + kB * y2.y + (t.diag1[k] ? kA : 0.0);
    }
    if (t.up0[k]) d[t.ij[k]] = d[t.ji[k]] = c0;                // one writer per entry, in diagonal tiles too
    if (t.up1[k]) d[t.ij[k] + 1] = d[t.ji[k] + t.pitch] = c1;
  }
  __syncthreads();
}

template <int WARPS, int TILES>
__global__ void __launch_bounds__(WARPS * 32) poly_kernel(const StepParams a) {
  constexpr int kPolyThreads = WARPS * 32;
  extern __shared__ __align__(16) double sh[];
  __shared__ double inv;
  pdl_wait();
  const Mat t = a.mats[blockIdx.x];
  const int s4 = up4(t.s), s8 = up8(t.s), nt = s4 >> 2, pairs = pairs_of(t.s), pitch = pitch64(t.s), n = s8 * pitch;
  double *g = sh, *q = sh + n, *x = sh + 2 * n, *y = sh + 3 * n;
  const PolyTiles<WARPS, TILES> tiles(t.s);
  for (int e = threadIdx.x; e < n; e += kPolyThreads) {
    g[e] = 0.0;
    if (a.steps == 0) x[e] = e / pitch == e % pitch ? 1.0 : 0.0;
  }
  __syncthreads();
  for (int e = threadIdx.x; e < pairs * 16; e += kPolyThreads) {
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
    g[i * pitch + j] = v;
    g[j * pitch + i] = v;
  }
  __syncthreads();
  if (threadIdx.x < 32) {
    double tr = 0.0;
    for (int i = threadIdx.x; i < t.s; i += 32) tr += g[i * pitch + i];
    for (int o = 16; o > 0; o >>= 1) tr += __shfl_xor_sync(0xffffffffu, tr, o);
    if (threadIdx.x == 0) {
      // u of norm zero (squares below 1e-30^2 are zero in fp32 too): any factor serves that P keeps finite in fp32
      const double norm = sqrt(tr) + static_cast<double>(a.eps);
      inv = norm < 1e-30 ? 1e30 : 1.0 / norm;
    }
  }
  __syncthreads();
  const double f = inv;
  for (int e = threadIdx.x; e < n; e += kPolyThreads) g[e] *= f * f;
  __syncthreads();
  pdl_launch_dependents();
  for (int it = 0; it < a.steps; ++it) {
    double* factor = it == 0 ? x : q;          // the first factor is the product so far
    poly_step<true>(factor, g, g, tiles, s8);
    if (it > 0) {
      poly_step<false>(y, q, x, tiles, s8);
      double* o = x; x = y; y = o;
    }
    if (it + 1 < a.steps) {
      const double* f1 = it == 0 ? x : q;
      poly_step<false>(y, f1, g, tiles, s8);
      poly_step<false>(g, f1, y, tiles, s8);
    }
  }
  for (int e = threadIdx.x; e < s4 * s4; e += kPolyThreads) a.ws[t.poly + e] = static_cast<float>(x[e / s4 * pitch + e % s4] * f);
}

template <bool TALL, int BLOCK>
__device__ __forceinline__ void apply_body(const StepParams& a, const Tile& tile, const Mat& t, float* smem) {
  const Place pl(t, a.aligned, TALL, BLOCK);
  const Share sh(pl);
  const float clip = clip_factor(a);
  const int64_t last = min(t.l, tile.first + a.piece * BLOCK);
  const float rows = t.tall ? t.l : t.s, cols = t.tall ? t.s : t.l;
  const float step = a.lr * (a.scale_mode == 0 ? 0.2f * sqrtf(fmaxf(rows, cols)) : sqrtf(fmaxf(1.0f, rows / cols)));
  const float keep = 1.0f - a.lr * a.wd;
  float* u = smem;
  float* pm = smem + kMaxSub;                                  // P: natural where the matrix is wide, paired where it is tall
  const int pp = odd_pitch(pl.s4);
  for (int e = threadIdx.x; e < pl.s4 * pl.s4; e += kThreads) {
    const int r = e / pl.s4, c = e - r * pl.s4;
    const int at = pl.tall ? (r >> 1) * 2 * pl.s4 + ((c >> 1) & 1) * pl.s4 + (c & ~3) + (c & 1) * 2 + (r & 1) : r * pp + c;
    pm[at] = a.ws[t.poly + e];
  }
  // out = A B: A (wide: P, tall: the sub-block) natural, its rows interleaved over the tiles; B paired
  const float *am = pl.tall ? u : pm, *bm = pl.tall ? pm : u;
  const int ap = pl.tall ? pl.pitch : pp, bw = pl.tall ? pl.s4 : pl.width;
  const int rt = pl.rows >> 2, ct = pl.width >> 2;             // up to 256 tiles of 4 x 4
  // wide: eight threads side by side on a row, so that a warp's reads of B are four times one 128-byte line and not
  // four whole rows of it (tall: B is P, with at most 16 tiles to a row)
  const int strip = TALL ? ct : 8, in_strip = threadIdx.x % (rt * strip);
  const int ri = in_strip / strip, ci = (threadIdx.x / (rt * strip) * strip + in_strip % strip) * 4;
  const bool works = ci < pl.width;

  // raw pieces of this thread: g, m as the shares say, p where its results go
  float* raw = pm + up4(kMaxShort) * odd_pitch(up4(kMaxShort)) + threadIdx.x * 4;
  const uint32_t raw_u32 = smem_u32(raw);
  int64_t base = t.off + (t.tall ? tile.first * t.s : tile.first);
  const bool want_g = a.m == nullptr || a.nesterov;
  auto left_of = [&](int64_t c0) { return static_cast<int>(min(static_cast<int64_t>(pl.block), last - c0)); };
  const bool has_m = a.m != nullptr, to_p = a.out == nullptr;
  auto fetch = [&](int64_t at, int left) {
    if (pl.vec && left == pl.block) {
#pragma unroll
      for (int k = 0; k < 2 * kUnits; ++k) {
        const int64_t o = at + sh.at[k >> 1] + (k & 1) * pl.row_stride;
        if (sh.full[k]) {
          if (want_g) cp_async16(raw_u32 + k * (kThreads * 16), a.g + o, 16);
          if (has_m) cp_async16(raw_u32 + kRaw + k * (kThreads * 16), a.m + o, 16);
        }
      }
    } else {
#pragma unroll 1
      for (int k = 0; k < 2 * kUnits; ++k) {
        const int row = 2 * ((threadIdx.x + (k >> 1) * kThreads) / (pl.width >> 2)) + (k & 1);
        const int col = (threadIdx.x + (k >> 1) * kThreads) % (pl.width >> 2) * 4;
        const int n = row < pl.rows ? pl.len(row, col, left) : 0;
        const int64_t o = n > 0 ? at + row * pl.row_stride + col : 0;
        if (want_g) copy_piece(raw_u32 + k * (kThreads * 16), a.g + o, n, pl.vec);
        if (has_m) copy_piece(raw_u32 + kRaw + k * (kThreads * 16), a.m + o, n, pl.vec);
      }
    }
    cp_async_commit();
  };
  const int64_t out_at = ri * pl.row_stride + ci, out_hop = rt * pl.row_stride;
  auto fetch_p = [&](int64_t at, int left) {
    if (to_p && works) {
      if (pl.vec && left == pl.block) {
#pragma unroll
        for (int i = 0; i < 4; ++i)
          if (pl.tall || ri + i * rt < pl.s) cp_async16(raw_u32 + 2 * kRaw + i * (kThreads * 16), a.p + at + out_at + i * out_hop, 16);
      } else {
#pragma unroll 1
        for (int i = 0; i < 4; ++i) {
          const int n = pl.len(ri + i * rt, ci, left);
          copy_piece(raw_u32 + 2 * kRaw + i * (kThreads * 16), a.p + (n > 0 ? at + out_at + i * out_hop : 0), n, pl.vec);
        }
      }
    }
    cp_async_commit();
  };
#pragma unroll
  for (int k = 0; k < 4 * kUnits; ++k) *reinterpret_cast<float4*>(raw + k * (kThreads * 4)) = make_float4(0.f, 0.f, 0.f, 0.f);
  fetch(base, left_of(tile.first));
  fetch_p(base, left_of(tile.first));
  for (int64_t c0 = tile.first; c0 < last; c0 += pl.block) {
    const int64_t cur = base;
    const int left = left_of(c0);
    const bool whole = pl.vec && left == pl.block;
    cp_async_wait<1>();                                        // g and m; p is still on its way
    __syncthreads();                                           // the sub-block before has been read (and P is in place)
#pragma unroll
    for (int k = 0; k < kUnits; ++k) {
      float4 v[2];
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        const float4 g4 = want_g ? ld4(raw + (2 * k + h) * (kThreads * 4)) : make_float4(0.f, 0.f, 0.f, 0.f);
        v[h] = !has_m ? g4 : update4(a, g4, ld4(raw + (2 * kUnits + 2 * k + h) * (kThreads * 4)), clip);
      }
      if (pl.tall) sh.store_natural(u, pl, k, v[0], v[1]);
      else sh.store_paired(u, pl, k, v[0], v[1]);
    }
    __syncthreads();
    base += pl.step;
    const int next = c0 + pl.block < last ? left_of(c0 + pl.block) : 0;
    fetch(base, next);                                         // nothing exists past the end: no copy leaves
    if (works) {
    uint64_t acc[4][4] = {};
    const float *ax = am + ri * ap, *by = bm + ci;
    const int hop = rt * ap;
    for (int k = 0; k < pl.s4; k += 4) {
      const float* b0 = by + k * bw;
      const ulonglong2 y00 = ldp(b0), y01 = ldp(b0 + bw), y10 = ldp(b0 + 2 * bw), y11 = ldp(b0 + 3 * bw);
      const uint64_t ya[4] = {y00.x, y00.y, y01.x, y01.y}, yb[4] = {y10.x, y10.y, y11.x, y11.y};
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const ulonglong2 x = ldp(ax + i * hop + k);
#pragma unroll
        for (int j = 0; j < 4; ++j) acc[i][j] = fma_f32x2(x.y, yb[j], fma_f32x2(x.x, ya[j], acc[i][j]));
      }
    }
    cp_async_wait<1>();                                        // p; the next g and m are on their way
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      float o[4];
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        float lo, hi;
        unpack_f32x2(acc[i][j], lo, hi);
        o[j] = lo + hi;
      }
      const int64_t at = cur + out_at + i * out_hop;
      float4 v = make_float4(o[0], o[1], o[2], o[3]);
      if (to_p) {
        const float4 p0 = ld4(raw + (4 * kUnits + i) * (kThreads * 4));
        v = make_float4(p0.x * keep - step * o[0], p0.y * keep - step * o[1], p0.z * keep - step * o[2], p0.w * keep - step * o[3]);
      }
      float* out = (to_p ? a.p : a.out) + at;
      // the gradients are zeroed by the CTA that alone reads them, after it has
      if (whole) {
        if (pl.tall || ri + i * rt < pl.s) {
          *reinterpret_cast<float4*>(out) = v;
          if (a.zero_grad) *reinterpret_cast<float4*>(a.g + at) = make_float4(0.f, 0.f, 0.f, 0.f);
        }
      } else {
        const int n = pl.len(ri + i * rt, ci, left);
        store_piece(out, v, n, pl.vec);
        if (a.zero_grad) store_piece(a.g + at, make_float4(0.f, 0.f, 0.f, 0.f), n, pl.vec);
      }
    }
    }
    fetch_p(base, next);
  }
}

__global__ void __launch_bounds__(kThreads, 2) apply_kernel(const StepParams a) {
  extern __shared__ __align__(16) float smem[];
  pdl_wait();
  const Tile tile = a.tiles[blockIdx.x];
  const Mat t = a.mats[tile.mat];
  K2Q_BY_SHAPE(apply_body)
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
  // Sub-blocks per CTA: what fills whole waves best, two CTAs per SM in apply and three in gram, each with about 0.7
  // sub-blocks' worth of start.  Measured on 58.7 M elements at rank 32: 16 per CTA (3.03 and 2.02 waves) 368 us, 8 (6.05
  // and 4.04) 357, 10 (4.92 and 3.28, what this picks) 353.  The plan depends on the shapes alone, so the SM count is
  // the B200's.
  auto tiles_with = [&](int64_t per) {
    int64_t n = 0;
    for (int64_t i = 0; i < count; ++i) {
      const int64_t s = rows[i] < cols[i] ? rows[i] : cols[i], l = rows[i] < cols[i] ? cols[i] : rows[i];
      const int64_t len = per * block_of(static_cast<int>(s));
      n += (l + len - 1) / len;
    }
    return n;
  };
  double best = 0.0;
  for (int64_t per = 1; per <= 32; ++per) {
    const int64_t n = tiles_with(per);
    const double waves = static_cast<double>((n + 2 * 148 - 1) / (2 * 148) + (n + 3 * 148 - 1) / (3 * 148)), cost = waves * (per + 0.7);
    if (per == 1 || cost < best) {
      best = cost;
      pl.piece = per;
    }
  }
  int64_t floats = 0;
  for (int64_t i = 0; i < count; ++i) {
    const int64_t s = rows[i] < cols[i] ? rows[i] : cols[i], l = rows[i] < cols[i] ? cols[i] : rows[i];
    const int64_t len = pl.piece * block_of(static_cast<int>(s)), n = (l + len - 1) / len;
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
  if (!(a.eps >= 0.f) || a.eps > 3.4e38f) return fail(K2Q_EINVAL, "%s: eps must be a finite number, not negative", name);
  if (a.steps < 0 || a.steps > 10) return fail(K2Q_EINVAL, "%s: steps %d not in [0,10]", name, a.steps);
  a.mats = static_cast<const Mat*>(table);
  a.tiles = reinterpret_cast<const Tile*>(a.mats + pl->count);
  a.piece = pl->piece;
  a.ws = static_cast<float*>(ws);
  a.aligned = !off16(a.p) && !off16(a.g) && !off16(a.m) && !off16(a.out);
  const int s4 = up4(pl->max_short);
  const int poly_smem = 4 * up8(pl->max_short) * pitch64(pl->max_short) * 8;
  const int poly_widest = pl->max_short <= 32 ? 32 : kMaxShort;      // the limit is the kernel's: launches of other threads share it
  const int poly_limit = 4 * up8(poly_widest) * pitch64(poly_widest) * 8;
  const int apply_smem = (kMaxSub + up4(kMaxShort) * odd_pitch(up4(kMaxShort))) * 4 + 3 * kRaw;
  if (int rc = check_cuda(cudaFuncSetAttribute(gram_kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, kGramSmem),
                          "cudaFuncSetAttribute(gram)"))
    return rc;
  auto poly = pl->max_short <= 32 ? poly_kernel<8, 2> : poly_kernel<16, 3>;
  if (int rc = check_cuda(cudaFuncSetAttribute(poly, cudaFuncAttributeMaxDynamicSharedMemorySize, poly_limit),
                          "cudaFuncSetAttribute(poly)"))
    return rc;
  if (int rc = check_cuda(cudaFuncSetAttribute(apply_kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, apply_smem),
                          "cudaFuncSetAttribute(apply)"))
    return rc;
  const unsigned tiles = static_cast<unsigned>(pl->tiles);
  if (int rc = launch_overlapped(gram_kernel, tiles, kThreads, kGramSmem, s, 1, name, a)) return rc;
  if (int rc = launch_overlapped(poly, static_cast<unsigned>(pl->count), pl->max_short <= 32 ? 256u : 512u, poly_smem, s, 1, name, a)) return rc;
  return launch_overlapped(apply_kernel, tiles, kThreads, apply_smem, s, 1, name, a);
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
    const int64_t len = pl.piece * block_of(m.s);
    m.tiles = static_cast<int32_t>((m.l + len - 1) / len);
    m.gram = floats;
    floats += static_cast<int64_t>(m.tiles) * pairs_of(m.s) * 16;
    m.poly = floats;
    floats += up4(m.s) * up4(m.s);
    off += m.s * m.l;
    mats[i] = m;
    for (int k = 0; k < m.tiles; ++k) tiles[nt++] = Tile{static_cast<int32_t>(i), 0, k * len};
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
