// Products of a few token rows with a 4-bit base (group scales), M <= 32:
//
//   run = 0;  for g = 0 .. K/128-1:  run = fma(float(sum_{k in g} xq[m,k] q4[n,k]), sw4[n,g], run)
//   y[m,n] = bf16( act(run * sx[m] + bias[n]) + sum_j u[m,j] (lora_scale Bm[n,j]) )
//
// The group sums are exact integers and the scales enter in ascending order of the groups, one fused
// multiply-add each: the operations of the large W4A8 product on every element, so both give the same bits.
// Cannot do with less than reading the codes once, N*K/2 bytes, and is bound by that for wide products and up to eight rows.
//
// A warp owns 8 or 16 channels and folds its groups in registers.  A group of eight channels is four m16n8k32 int8 MMAs
// per 16 tokens, the tokens as rows (dp4a reaches a quarter of their rate, and needs the codes as bytes as well).  The
// order of k inside a group is free as long as both operands agree, so a lane simply takes 16
// consecutive bytes of a channel (32 codes): the low nibbles of a word, shifted up, and its high nibbles are two
// operand registers holding 16 times the codes, and the tokens' bytes are dealt out to match (even and odd
// bytes of eight).
//   - The codes travel by 16-byte asynchronous copies into a ring of shared memory; a lane reads back
//     only what it copied itself, so the ring needs no barrier and stays full whatever the arithmetic does.
//   - The tokens and the scales are staged in shared memory beforehand.  Plain loads of them inside the loop return
//     in order behind the codes' misses in the L1 pipe and cost each group a trip to DRAM (measured: 520 ns a
//     group); copies of them in the ring, several lanes from one address, were slower still (53 us against 24 to 31 at 16
//     rows, 6144 channels, K = 16384).  Two warps set aside to bring the tokens chunk by chunk took 46 us there, 29 without
//     them (the MMA order changed between the two as well).
// One CTA per SM, so that the tokens are staged once per SM.  With few channels per SM, several warps share eight
// channels and pass the running values on in block order (ring kernel below).
// Measured on a B200 (codes from DRAM): 36864 x 6144 23.0 / 25.2 / 27.0 us at 1 / 8 / 16 rows (reading the codes and scales
// at the copy bandwidth: 17.8), 6144 x 6144 7.9 / 9.2 / 11.8 (3.0), 6144 x 16384 14.8 / 19.2 / 27.3 (7.9), 6144 x 256
// 3.0 / 3.4 / 3.8 (0.1).  With 13 rows of K = 16384 the ring kernel runs 12 warps per SM, issues in 46 % of the cycles
// and reads DRAM at 23 % of its peak: instruction latency and shared memory, not the codes.
#include "k2q_common.cuh"

namespace k2q {
namespace {

constexpr int kMaxRows = 32;
constexpr int kMaxK = 131072;         // the scales of 16 channels stay in shared memory: K / 4 bytes

struct GemvParams {
  int M, N, K;
  const int8_t* xq; const uint8_t* wq; const __nv_bfloat16* sw;
  const float* sx; const float* bias; const float* u; const float* Bm;
  int64_t ldu, ldb; int rank; float lora_scale; int act;
  __nv_bfloat16* y; int64_t ldy;
  int warps;                          // warps per CTA that multiply
  int ks;                             // warps that share eight channels (ring kernel; `warps` then counts teams)
  int chunk;                          // groups of the tokens staged at a time
};

__device__ __forceinline__ void finish(const GemvParams& p, int m, int n, float run) {
  float v = __fadd_rn(__fmul_rn(run, p.sx != nullptr ? __ldg(p.sx + m) : 1.0f), p.bias != nullptr ? __ldg(p.bias + n) : 0.0f);
  if (p.act == K2Q_ACT_GELU_TANH) v = gelu_tanh(v);
  if (p.rank > 0) {
    float d = 0.f;
    for (int j = 0; j < p.rank; ++j)
      d = fmaf(__ldg(p.u + m * p.ldu + j), p.lora_scale * __ldg(p.Bm + n * p.ldb + j), d);
    v += d;
  }
  p.y[m * p.ldy + n] = __float2bfloat16_rn(v);
}

__device__ __forceinline__ void mma_s8_16832(int (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0,
                                             uint32_t b1) {
  asm("mma.sync.aligned.m16n8k32.row.col.s32.s8.s8.s32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
               : "+r"(d[0]), "+r"(d[1]), "+r"(d[2]), "+r"(d[3])
               : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}
__device__ __forceinline__ uint32_t pick(uint32_t a, uint32_t b, uint32_t sel) {
  uint32_t r;
  asm("prmt.b32 %0, %1, %2, %3;" : "=r"(r) : "r"(a), "r"(b), "r"(sel));
  return r;
}

__device__ __forceinline__ uint4 lds16(uint32_t addr) {
  uint4 v;
  asm volatile("ld.shared.v4.u32 {%0,%1,%2,%3}, [%4];" : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w) : "r"(addr) : "memory");
  return v;
}

constexpr int kMaxWarps = 16;
// named barriers (0 is __syncthreads)
__device__ __forceinline__ void bar_sync(int id, int threads) { asm volatile("bar.sync %0, %1;" ::"r"(id), "r"(threads) : "memory"); }
__device__ __forceinline__ void bar_arrive(int id, int threads) { asm volatile("bar.arrive %0, %1;" ::"r"(id), "r"(threads) : "memory"); }
constexpr int kSmemMax = 232448;      // also every kernel's limit, whatever the launch needs: launches of other threads share it

// Groups [g0, g0 + chunk) of every token into shared memory, the even and the odd bytes of every eight apart.  A
// token's row there is chunk * 128 + 16 bytes long: the eight lanes of a 16-byte read phase (two tokens, four
// quarters of a group) meet 32 different banks.
__device__ __forceinline__ void request_tokens(const GemvParams& p, uint32_t xs, int g0) {
  const int n = min(p.chunk, (p.K >> 7) - g0) * 8, row = p.chunk * 128 + 16;      // n 16-byte pieces per token
  const int8_t* src = p.xq + g0 * 128LL;
  for (int e = threadIdx.x, m = e / n, c = e - m * n; m < p.M;) {
    cp_async16(xs + m * row + c * 16, src + static_cast<int64_t>(m) * p.K + c * 16, 16);
    for (c += blockDim.x; c >= n; c -= n) ++m;
  }
}
// after this thread's copies have arrived
__device__ __forceinline__ void deal_tokens(const GemvParams& p, uint8_t* xs, int g0) {
  const int n = min(p.chunk, (p.K >> 7) - g0) * 8, row = p.chunk * 128 + 16;
  for (int e = threadIdx.x, m = e / n, c = e - m * n; m < p.M;) {
    uint4* at = reinterpret_cast<uint4*>(xs + m * row + c * 16);
    const uint4 v = *at;
    *at = make_uint4(pick(v.x, v.y, 0x6420u), pick(v.x, v.y, 0x7531u), pick(v.z, v.w, 0x6420u), pick(v.z, v.w, 0x7531u));
    for (c += blockDim.x; c >= n; c -= n) ++m;
  }
}

// 16 times the sums of GP groups: entry = this lane's codes, xg = the tokens at the first group, acc[h][t][c][0..1] token
// 16 t + r, channels 8 c + 2 q, + 1, acc[..][2..3] token 16 t + r + 8.
template <int MH, int CT, int GP>
__device__ __forceinline__ void group_sums(uint32_t entry, const uint8_t* xg, const int (&xoff)[MH], int (&acc)[GP][(MH + 1) / 2][CT][4]) {
  constexpr int MT = (MH + 1) / 2;
  uint4 wv[GP][CT];
#pragma unroll
  for (int h = 0; h < GP; ++h)
#pragma unroll
    for (int c = 0; c < CT; ++c) wv[h][c] = lds16(entry + (h * CT + c) * 512);
#pragma unroll
  for (int h = 0; h < GP; ++h)
#pragma unroll
    for (int t = 0; t < MT; ++t)
#pragma unroll
      for (int c = 0; c < CT; ++c) acc[h][t][c][0] = acc[h][t][c][1] = acc[h][t][c][2] = acc[h][t][c][3] = 0;
  // the groups side by side, so that neighbouring MMAs do not wait for one another
#pragma unroll
  for (int jj = 0; jj < 2; ++jj) {                         // 64 of a group's codes: two words of each lane
    uint4 x[GP][2 * MT];
#pragma unroll
    for (int h = 0; h < GP; ++h)
#pragma unroll
      for (int t = 0; t < 2 * MT; ++t)
        x[h][t] = t < MH ? *reinterpret_cast<const uint4*>(xg + h * 128 + xoff[t < MH ? t : 0] + jj * 16) : make_uint4(0, 0, 0, 0);
#pragma unroll
    for (int j = 0; j < 2; ++j) {
#pragma unroll
      for (int h = 0; h < GP; ++h) {
#pragma unroll
        for (int c = 0; c < CT; ++c) {
          const uint4 v = wv[h][c];
          const uint32_t word = jj ? (j ? v.w : v.z) : (j ? v.y : v.x);
          const uint32_t b0 = (word << 4) & 0xF0F0F0F0u, b1 = word & 0xF0F0F0F0u;
#pragma unroll
          for (int t = 0; t < MT; ++t)
            mma_s8_16832(acc[h][t][c], j ? x[h][2 * t].z : x[h][2 * t].x, j ? x[h][2 * t + 1].z : x[h][2 * t + 1].x,
                         j ? x[h][2 * t].w : x[h][2 * t].y, j ? x[h][2 * t + 1].w : x[h][2 * t + 1].y, b0, b1);
        }
      }
    }
  }
}

// MH halves of eight tokens, CT tiles of eight channels per warp, RING entries of GP groups.
template <int MH, int CT, int GP, int RING>
__global__ void __launch_bounds__(kMaxWarps * 32, 1) gemv_kernel(const GemvParams p) {
  constexpr int MT = (MH + 1) / 2;                             // tiles of 16 tokens
  constexpr uint32_t kEntry = CT * GP * 512;
  extern __shared__ __align__(16) uint8_t smem[];
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, r = lane >> 2, q = lane & 3, warps = p.warps;
  const int groups = p.K >> 7;
  const int n0 = (blockIdx.x * warps + warp) * (8 * CT);
  const bool live = warp < warps && n0 < p.N;                  // the other warps only help to stage the tokens
  // shared memory: rings | scales [channel][group] | tokens
  const uint32_t ring = smem_u32(smem) + warp * (RING * kEntry) + lane * 16;
  uint8_t* scales = smem + warps * RING * kEntry;
  uint8_t* xs = scales + warps * groups * (16 * CT);
  pdl_wait();
  request_tokens(p, smem_u32(xs), 0);
  {
    const int first = blockIdx.x * warps * (8 * CT), n = min(warps * 8 * CT, p.N - first) * groups / 8;
    const __nv_bfloat16* s = p.sw + static_cast<int64_t>(first) * groups;     // one contiguous block
    for (int c = threadIdx.x; c < n; c += blockDim.x) cp_async16(smem_u32(scales) + c * 16, s + c * 8, 16);
  }
  cp_async_commit();

  const int64_t row_bytes = p.K >> 1;
  const uint8_t* src = p.wq + (n0 + r) * row_bytes + q * 16;   // this lane's 16 bytes of channel r in the next group
  int todo = live ? groups : 0;                                // groups still to request
  uint32_t in = 0, out = 0;                                    // ring slots of the next request and the next entry
  auto request = [&]() {
#pragma unroll
    for (int h = 0; h < GP; ++h) {
      if (todo > h) {
#pragma unroll
        for (int c = 0; c < CT; ++c) cp_async16(ring + in + (h * CT + c) * 512, src + h * 64 + c * 8 * row_bytes, 16);
      }
    }
    todo -= GP;
    src += GP * 64;
    in = in == (RING - 1) * kEntry ? 0u : in + kEntry;
    cp_async_commit();
  };
#pragma unroll
  for (int i = 0; i < RING - 1; ++i) request();
  cp_async_wait<RING - 1>();
  deal_tokens(p, xs, 0);
  __syncthreads();

  int xoff[MH];                                                // this lane's place in the tokens
#pragma unroll
  for (int t = 0; t < MH; ++t) {
    const int tok = t * 8 + r;                                 // rows past M: any row, the result is not kept
    xoff[t] = (tok < p.M ? tok : p.M - 1) * (p.chunk * 128 + 16) + q * 32;
  }
  float run[MT][CT][4] = {};
  const __nv_bfloat16* sg = reinterpret_cast<const __nv_bfloat16*>(scales) + (warp * 8 * CT + 2 * q) * groups;
  for (int g0 = 0; g0 < groups; g0 += p.chunk) {
    if (g0 > 0) {                                              // the whole CTA: the next tokens
      __syncthreads();
      request_tokens(p, smem_u32(xs), g0);
      cp_async_commit();
      cp_async_wait<0>();
      deal_tokens(p, xs, g0);
      __syncthreads();
    }
    if (!live) continue;
    const int n = min(groups - g0, p.chunk);
    const uint8_t* xg = xs;
    for (int g = 0; g < n; g += GP, xg += GP * 128) {
      cp_async_wait<RING - 2>();
      int acc[GP][MT][CT][4];
      group_sums<MH, CT, GP>(ring + out, xg, xoff, acc);
      out = out == (RING - 1) * kEntry ? 0u : out + kEntry;
      request();
#pragma unroll
      for (int h = 0; h < GP; ++h) {
        if (g + h < n) {
#pragma unroll
          for (int c = 0; c < CT; ++c) {
            // the group sums hold 16 times the codes' product
            const float s0 = __bfloat162float(sg[c * 8 * groups]) * 0.0625f, s1 = __bfloat162float(sg[(c * 8 + 1) * groups]) * 0.0625f;
#pragma unroll
            for (int t = 0; t < MT; ++t) {
              run[t][c][0] = fmaf(static_cast<float>(acc[h][t][c][0]), s0, run[t][c][0]);
              run[t][c][1] = fmaf(static_cast<float>(acc[h][t][c][1]), s1, run[t][c][1]);
              if (2 * t + 1 < MH) {
                run[t][c][2] = fmaf(static_cast<float>(acc[h][t][c][2]), s0, run[t][c][2]);
                run[t][c][3] = fmaf(static_cast<float>(acc[h][t][c][3]), s1, run[t][c][3]);
              }
            }
          }
          ++sg;
        }
      }
    }
  }
  if (!live) return;
#pragma unroll
  for (int t = 0; t < MT; ++t)
#pragma unroll
    for (int c = 0; c < CT; ++c)
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        const int m = t * 16 + r + 8 * (e >> 1), n = n0 + c * 8 + 2 * q + (e & 1);
        if (m < p.M) finish(p, m, n, run[t][c][e]);
      }
}

// Few channels per SM: p.ks warps share eight channels.  They take blocks of G groups in turn, keep a block's sums in
// registers, and pass the running values on in block order: warp j folds its block when they arrive from warp j - 1, and
// hands them to warp j + 1 (the last to the first, for the next round), through a slot in shared memory and a named
// barrier of the two warps.  A block's arithmetic takes many times the fold, so that nobody waits in the steady state.  A
// slot or barrier is used again only after the values have gone round once, hence after its reader.
template <int MH, int RING>
__global__ void __launch_bounds__(kMaxWarps * 32, 1) gemv_ring_kernel(const GemvParams p) {
  constexpr int MT = (MH + 1) / 2, GP = 4, G = 8, IT = G / GP, V = MH == 1 ? 2 : 4;   // V values per lane and token tile
  constexpr uint32_t kEntry = GP * 512;
  extern __shared__ __align__(16) uint8_t smem[];
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, r = lane >> 2, q = lane & 3;
  const int groups = p.K >> 7, blocks = (groups + G - 1) / G, ks = p.ks;
  const int team = warp / ks, j = warp - team * ks, n0 = (blockIdx.x * p.warps + team) * 8;
  const bool live = team < p.warps && n0 < p.N;                // the other warps only help to stage the tokens
  // shared memory: rings | scales [channel][group] | slots | tokens
  const uint32_t ring = smem_u32(smem) + warp * (RING * kEntry) + lane * 16;
  uint8_t* scales = smem + p.warps * ks * RING * kEntry;
  float* slots = reinterpret_cast<float*>(scales + p.warps * groups * 16);
  uint8_t* xs = reinterpret_cast<uint8_t*>(slots + p.warps * ks * MT * V * 32);
  pdl_wait();
  request_tokens(p, smem_u32(xs), 0);
  {
    const int first = blockIdx.x * p.warps * 8, n = min(p.warps * 8, p.N - first) * groups / 8;
    const __nv_bfloat16* s = p.sw + static_cast<int64_t>(first) * groups;     // one contiguous block
    for (int c = threadIdx.x; c < n; c += blockDim.x) cp_async16(smem_u32(scales) + c * 16, s + c * 8, 16);
  }
  cp_async_commit();
  const int64_t row_bytes = p.K >> 1;
  const uint8_t* src = p.wq + (n0 + r) * row_bytes + static_cast<int64_t>(j) * G * 64 + q * 16;
  int next = live ? j * G : groups;                            // group of the next request; past the end: nothing left
  uint32_t in = 0, out = 0;
  auto request = [&]() {
#pragma unroll
    for (int h = 0; h < GP; ++h)
      if (next + h < groups) cp_async16(ring + in + h * 512, src + h * 64, 16);
    next += GP;
    src += GP * 64;
    if ((next & (G - 1)) == 0) {                               // the warp's block is requested: on to its next one
      next += (ks - 1) * G;
      src += static_cast<int64_t>(ks - 1) * G * 64;
    }
    in = in == (RING - 1) * kEntry ? 0u : in + kEntry;
    cp_async_commit();
  };
#pragma unroll
  for (int i = 0; i < RING - 1; ++i) request();
  cp_async_wait<RING - 1>();
  deal_tokens(p, xs, 0);
  __syncthreads();
  int xoff[MH];                                                // this lane's place in the tokens
#pragma unroll
  for (int t = 0; t < MH; ++t) {
    const int tok = t * 8 + r;                                 // rows past M: any row, the result is not kept
    xoff[t] = (tok < p.M ? tok : p.M - 1) * (p.chunk * 128 + 16) + q * 32;
  }
  const __nv_bfloat16* sc = reinterpret_cast<const __nv_bfloat16*>(scales) + (team * 8 + 2 * q) * groups;
  const int rounds = (blocks + ks - 1) / ks;
  const int prev = j == 0 ? ks - 1 : j - 1;
  float run[MT][V] = {};
  int g0 = 0;                                                  // first group of the staged tokens
  for (int rd = 0; rd < rounds; ++rd) {
    if (rd * ks * G >= g0 + p.chunk) {                         // the chunk is a multiple of a round
      g0 += p.chunk;
      __syncthreads();
      request_tokens(p, smem_u32(xs), g0);
      cp_async_commit();
      cp_async_wait<0>();
      deal_tokens(p, xs, g0);
      __syncthreads();
    }
    const int blk = rd * ks + j, b0 = blk * G;
    if (!live || blk >= blocks) continue;
    float sum[IT][GP][MT][V];
#pragma unroll
    for (int i = 0; i < IT; ++i) {
      cp_async_wait<RING - 2>();
      int acc[GP][MT][1][4];
      group_sums<MH, 1, GP>(ring + out, xs + (b0 + i * GP - g0) * 128, xoff, acc);
      out = out == (RING - 1) * kEntry ? 0u : out + kEntry;
      request();
#pragma unroll
      for (int h = 0; h < GP; ++h)
#pragma unroll
        for (int t = 0; t < MT; ++t)
#pragma unroll
          for (int v = 0; v < V; ++v) sum[i][h][t][v] = static_cast<float>(acc[h][t][0][v]);
    }
    if (blk > 0) {
      bar_sync(1 + team * ks + prev, 64);
#pragma unroll
      for (int t = 0; t < MT; ++t)
#pragma unroll
        for (int v = 0; v < V; ++v) run[t][v] = slots[((team * ks + prev) * MT * V + t * V + v) * 32 + lane];
    }
#pragma unroll
    for (int i = 0; i < IT; ++i)
#pragma unroll
      for (int h = 0; h < GP; ++h) {
        const int g = b0 + i * GP + h;
        if (g < groups) {
          // the group sums hold 16 times the codes' product
          const float s0 = __bfloat162float(sc[g]) * 0.0625f, s1 = __bfloat162float(sc[groups + g]) * 0.0625f;
#pragma unroll
          for (int t = 0; t < MT; ++t)
#pragma unroll
            for (int v = 0; v < V; ++v) run[t][v] = fmaf(sum[i][h][t][v], (v & 1) ? s1 : s0, run[t][v]);
        }
      }
    if (blk + 1 < blocks) {
#pragma unroll
      for (int t = 0; t < MT; ++t)
#pragma unroll
        for (int v = 0; v < V; ++v) slots[(warp * MT * V + t * V + v) * 32 + lane] = run[t][v];
      bar_arrive(1 + warp, 64);
    } else {
#pragma unroll
      for (int t = 0; t < MT; ++t)
#pragma unroll
        for (int v = 0; v < V; ++v) {
          const int m = t * 16 + r + 8 * (v >> 1), n = n0 + 2 * q + (v & 1);
          if (m < p.M) finish(p, m, n, run[t][v]);
        }
    }
  }
}

// groups of the tokens that fit beside `ks` warps per team, in whole rounds
template <int MH, int RING>
int ring_chunk(const GemvParams& p, int teams, int ks, int* fixed) {
  constexpr int MT = (MH + 1) / 2, G = 8, V = MH == 1 ? 2 : 4;
  *fixed = teams * ks * (RING * 2048 + MT * V * 32 * 4) + teams * (p.K >> 7) * 16;
  return *fixed >= kSmemMax ? 0 : ((kSmemMax - *fixed) / p.M - 16) / 128 / (G * ks) * (G * ks);
}

template <int MH, int RING>
int launch_ring(GemvParams p, int teams, int ks, cudaStream_t stream) {
  constexpr int G = 8;
  const int groups = p.K >> 7, warps = teams * ks;
  int fixed = 0;
  const int chunk = ring_chunk<MH, RING>(p, teams, ks, &fixed);
  const int all_groups = (groups + G * ks - 1) / (G * ks) * (G * ks);
  p.chunk = chunk < all_groups ? chunk : all_groups;
  p.warps = teams;
  p.ks = ks;
  const int smem = fixed + p.M * (p.chunk * 128 + 16);
  auto kern = gemv_ring_kernel<MH, RING>;
  if (int rc = check_cuda(cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, kSmemMax),
                          "cudaFuncSetAttribute(gemv_w4a8)"))
    return rc;
  const int tiles = p.N / 8, all = warps > 8 ? warps : 8;      // eight warps at least stage the tokens
  return launch_overlapped(kern, static_cast<unsigned>((tiles + teams - 1) / teams), static_cast<unsigned>(all * 32),
                           static_cast<size_t>(smem), stream, 1, "gemv_w4a8 launch", p);
}

template <int MH, int CT, int GP, int RING>
int launch_one(GemvParams p, int warps, cudaStream_t stream) {
  const int tiles = p.N / (8 * CT), groups = p.K >> 7;
  const int fixed = warps * (RING * CT * GP * 512 + groups * 16 * CT);
  const int chunk = ((kSmemMax - fixed) / p.M - 16) / 128 / GP * GP;
  if (fixed >= kSmemMax || chunk < GP) return fail(K2Q_EINVAL, "k2q_gemv_w4a8: no room for the tokens (M=%d, K=%d)", p.M, p.K);
  p.chunk = chunk < groups ? chunk : (groups + GP - 1) / GP * GP;
  const int smem = fixed + p.M * (p.chunk * 128 + 16);
  auto kern = gemv_kernel<MH, CT, GP, RING>;
  if (int rc = check_cuda(cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, kSmemMax),
                          "cudaFuncSetAttribute(gemv_w4a8)"))
    return rc;
  p.warps = warps;
  const int all = warps > 8 ? warps : 8;                       // eight warps at least stage the tokens
  return launch_overlapped(kern, static_cast<unsigned>((tiles + warps - 1) / warps), static_cast<unsigned>(all * 32),
                           static_cast<size_t>(smem), stream, 1, "gemv_w4a8 launch", p);
}

// One CTA per SM, as many warps as it takes to cover the channels at once (16 at most); where eight tiles of 16
// channels and more fall to an SM, a warp takes 16, so that two of its channels share each read of the tokens.
template <int MH>
int launch_gemv(const GemvParams& p, cudaStream_t stream) {
  const int sms = sm_count() > 0 ? sm_count() : 148, groups = p.K >> 7;
  const int ct = p.N / 16 >= sms * 8 ? 2 : 1;
  const int tiles = p.N / (8 * ct);
  int warps = (tiles + sms - 1) / sms;
  if (warps > kMaxWarps) warps = kMaxWarps;
  const int room = 64 * 1024 / (groups * 16 * ct);             // the scales stay in shared memory
  if (warps > room) warps = room;
  // few channels: the contraction is split among 15 warps at most (a named barrier each)
  int ks = 15 / warps;
  const int blocks = (groups + 7) / 8;
  if (ks > blocks) ks = blocks;
  if constexpr (MH <= 2) {
    int fixed;
    while (ks >= 2 && ring_chunk<MH, 4>(p, warps, ks, &fixed) == 0) --ks;
    if (ct == 1 && ks >= 2) return launch_ring<MH, 4>(p, warps, ks, stream);
  }
  if (ct == 2) return launch_one<MH, 2, 2, MH == 1 ? 4 : 3>(p, warps, stream);
  return warps <= 8 ? launch_one<MH, 1, 4, 6>(p, warps, stream) : launch_one<MH, 1, 4, 4>(p, warps, stream);
}

}  // namespace
}  // namespace k2q

using namespace k2q;

extern "C" int k2q_gemv_w4a8(const int8_t* xq, const uint8_t* wq4, const void* sw4_bf16, int64_t M, int64_t N, int64_t K,
                             const k2q_epilogue* ep, void* y_bf16, int64_t ldy, void* stream) {
  const char* name = "k2q_gemv_w4a8";
  if (int rc = check_device_arch()) return rc;
  if (M < 0 || M > kMaxRows || N <= 0 || K <= 0 || N > 0x7fffff00LL || K > kMaxK)
    return fail(K2Q_EINVAL, "%s: bad shape M=%lld N=%lld K=%lld (at most %d rows, K <= %d)", name, (long long)M, (long long)N,
                (long long)K, kMaxRows, kMaxK);
  if (K % 128 != 0) return fail(K2Q_EINVAL, "%s: K=%lld is not a multiple of 128", name, (long long)K);
  if (N % 16 != 0) return fail(K2Q_EINVAL, "%s: N=%lld is not a multiple of 16", name, (long long)N);
  if (M == 0) return K2Q_OK;
  if (!xq || !wq4 || !sw4_bf16 || !y_bf16) return fail(K2Q_EINVAL, "%s: NULL operand", name);
  if ((reinterpret_cast<uintptr_t>(xq) | reinterpret_cast<uintptr_t>(wq4) | reinterpret_cast<uintptr_t>(sw4_bf16)) & 15u)
    return fail(K2Q_EINVAL, "%s: codes and group scales must be 16-byte aligned", name);
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
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  if (M <= 8) return launch_gemv<1>(p, s);
  if (M <= 16) return launch_gemv<2>(p, s);
  return launch_gemv<4>(p, s);
}
