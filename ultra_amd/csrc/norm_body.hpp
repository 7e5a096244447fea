// Kernels of the stand-alone layer normalisation (norm.hip).
#pragma once
#include "storage.hpp"

#include <type_traits>

namespace ultr {

constexpr int kNThreads = 256;
constexpr int kGradThreads = 512;  // one workgroup a CU: 8 waves with up to 256 registers each

// Sums over the TPR threads that share a row (a power of two: part of a wave, a wave, or whole waves of one workgroup); all
// of them get the totals.  K values at once; red: K floats per wave of the workgroup.  The exchange ends without a barrier, so
// the next one must use another `red`, and the one after that may use this again.
template <int TPR, int K>
__device__ __forceinline__ void row_sums(float (&v)[K], float* red) {
#pragma unroll
  for (int k = 0; k < K; ++k) v[k] = group_sum<(TPR < 64 ? TPR : 64)>(v[k]);
  if (TPR > 64) {
    const int wave = threadIdx.x >> 6, first = wave & ~(TPR / 64 - 1);
    if ((threadIdx.x & 63) == 0) {
#pragma unroll
      for (int k = 0; k < K; ++k) red[wave * K + k] = v[k];
    }
    lds_barrier();
#pragma unroll
    for (int k = 0; k < K; ++k) {
      v[k] = 0.f;
#pragma unroll
      for (int w = 0; w < TPR / 64; ++w) v[k] += red[(first + w) * K + k];
    }
  }
}

// The same for the forward pass, whose K are many: one lane takes one wave's sum, the lanes of a DPP row (16) add them up, in
// 32 or 64 bits (A).  A lane that reads every wave's sums by itself holds 16 K of them in registers.
template <int CTRL>
__device__ __forceinline__ double dpp_f64(double v) {
  return __hiloint2double(__builtin_amdgcn_update_dpp(0, __double2hiint(v), CTRL, 0xF, 0xF, true),
                          __builtin_amdgcn_update_dpp(0, __double2loint(v), CTRL, 0xF, 0xF, true));
}
template <int WIDTH>
__device__ __forceinline__ double group_sum(double v) {
  static_assert(WIDTH <= 16, "one DPP row");
  if (WIDTH > 1) v += dpp_f64<0xB1>(v);   // quad_perm [1,0,3,2]
  if (WIDTH > 2) v += dpp_f64<0x4E>(v);   // quad_perm [2,3,0,1]
  if (WIDTH > 4) v += dpp_f64<0x141>(v);  // row_half_mirror (quads already uniform)
  if (WIDTH > 8) v += dpp_f64<0x140>(v);  // row_mirror
  return v;
}
template <int TPR, typename A, int K>
__device__ __forceinline__ void row_totals(float (&v)[K], A (&total)[K], float* red) {
#pragma unroll
  for (int k = 0; k < K; ++k) v[k] = group_sum<(TPR < 64 ? TPR : 64)>(v[k]);
  constexpr int W = TPR > 64 ? TPR / 64 : 1;
  if (W > 1) {
    const int wave = threadIdx.x >> 6, mine = (wave & ~(W - 1)) + (threadIdx.x & (W - 1));
    if ((threadIdx.x & 63) == 0) {
#pragma unroll
      for (int k = 0; k < K; ++k) red[wave * K + k] = v[k];
    }
    lds_barrier();
#pragma unroll
    for (int k = 0; k < K; ++k) v[k] = red[mine * K + k];
  }
#pragma unroll
  for (int k = 0; k < K; ++k) total[k] = group_sum<W>((A)v[k]);
}

// Where a thread's C pieces of V elements lie in a row of N.  With TAIL (N no multiple of V, N >= V) the last piece is moved
// back to end with the row; its first skip[] elements belong to the piece before it as well: they are left out of sums, and
// both pieces store the same values for them.  skip >= V: no piece.
template <int TPR, int C, int V, bool TAIL>
struct Pieces {
  int at[C], skip[C];
  __device__ __forceinline__ Pieces(int lane, int N) {
#pragma unroll
    for (int c = 0; c < C; ++c) {
      const int i = (c * TPR + lane) * V;
      at[c] = TAIL ? min(i, N - V) : i;
      skip[c] = TAIL ? i - at[c] : (i < N ? 0 : V);
    }
  }
  __device__ __forceinline__ bool any(int c) const { return skip[c] < V; }
  __device__ __forceinline__ float counted(int c, int j, float v) const { return !TAIL || j >= skip[c] ? v : 0.f; }
};

// Forward.  HBM-bound: one read and one write of the matrix.  TPR threads hold R whole rows in registers, so the mean, the
// variance about it and the output need one pass over memory.  R = 2: the weights, which come out of the caches once per
// row otherwise, serve two rows (fp16 rows of 5003 with fp32 weights, 30010 of them: 124 us against 160; they still move as
// many bytes of weights out of the caches as of the matrix).  Narrow rows ask for their weights along with the row (40960 x
// 136 fp32: 8.8 us against 9.9); in a workgroup of several waves the other workgroups cover that latency and the registers
// are worth more (two rows at a time, early against late: the 30010 rows in the kernel alone 126 us and 113, 16384 x 4096 bf16
// 48.6 and 47.4; fp32 is within 2.5 % either way, 8192 x 4096 47.5 and 48.6, 4096 x 8192 49.9 and 50.7).
//
// The mean is mean[r] + low[r]: an error of a fraction of the row's OFFSET would be the whole variance of a row that hardly
// varies (a constant row of 1e6, 5003 entries, came out as 0.9).  That costs 0 to 2 % over one fp32 sum, up to 5 % in
// one-wave rows that the caches hold (40960 x 136 fp32 9.8 us against 9.3, 16969 x 1052 fp16 19.6 against 18.8).
//   fp32    mean is the fp32 sum's; the second sums give low = sum(x - mean) / N and the variance sum((x - mean)^2) / N - low^2.
//   16 bit  an fp32 sum is exact for entries of similar size (up to a factor of 4 for 2048 of them with 11 bits or 8192 with 8),
//           and where they are not their spread is large against its roundings; longer rows meet in 64 bits from wave to wave.  So
//           low is what the sum's quotient has beyond fp32 and needs no second sum.
// Sums run in units of 2^kSumShift, so that no sum of finite entries overflows.
//
// x - mean must mean the same everywhere: the product that makes the mean is not to be fused into it.
__device__ __forceinline__ float rounded_product(float a, float b) {
#pragma clang fp contract(off)
  return a * b;
}
template <typename T>
constexpr int kSumShift = sizeof(T) == 4 ? 17 : 13;
template <typename T, typename W, int TPR, int C, int V, bool TAIL, int R>
__global__ void __launch_bounds__(TPR < 256 ? 256 : TPR)
    layer_norm_kernel(const T* x, long long ldx, const W* gamma, const W* beta, long long M, int N, double inv_n, float eps,
                      T* y, long long ldy, float* stats) {
  constexpr int NT = TPR < 256 ? 256 : TPR;
  constexpr bool EARLY = TPR <= 128, WIDE = sizeof(T) == 4;
  constexpr bool EXACT32 = TPR * C * V <= (std::is_same<T, f16_t>::value ? 2048 : 8192);
  typedef typename Piece<T, V>::type PT;
  typedef typename Piece<W, V>::type PW;
  __shared__ float red[2][2 * R * NT / 64];
  const int lane = threadIdx.x % TPR;
  const long long row0 = ((long long)blockIdx.x * (NT / TPR) + threadIdx.x / TPR) * R;
  const Pieces<TPR, C, V, TAIL> pc(lane, N);
  PT raw[R][C];
  PW g[C], b[C];
#pragma unroll
  for (int r = 0; r < R; ++r) {
    const T* xr = x + min(row0 + r, M - 1) * ldx;
#pragma unroll
    for (int c = 0; c < C; ++c)
      if (pc.any(c)) raw[r][c] = *reinterpret_cast<const PT*>(xr + pc.at[c]);
  }
  auto weights = [&](int c) {
    if (gamma) g[c] = *reinterpret_cast<const PW*>(gamma + pc.at[c]);
    if (beta) b[c] = *reinterpret_cast<const PW*>(beta + pc.at[c]);
  };
  if (EARLY) {
#pragma unroll
    for (int c = 0; c < C; ++c)
      if (pc.any(c)) weights(c);
  }
  constexpr int units = 1 << kSumShift<T>;
  float mean[R], low[R], rstd[R];
#pragma unroll
  for (int r = 0; r < R; ++r) {
    mean[r] = 0.f;
#pragma unroll
    for (int c = 0; c < C; ++c) {
      if (!pc.any(c)) continue;
#pragma unroll
      for (int j = 0; j < V; ++j) mean[r] = fmaf(1.f / units, pc.counted(c, j, to_f32(raw[r][c][j])), mean[r]);
    }
  }
  if constexpr (WIDE) {
    row_totals<TPR>(mean, mean, red[0]);
#pragma unroll
    for (int r = 0; r < R; ++r) mean[r] = rounded_product(mean[r], (float)(inv_n * units));
  } else if constexpr (EXACT32) {
    const double scale = inv_n * units;
    const float high = (float)scale, rest = (float)(scale - (double)high);
    float total[R];
    row_totals<TPR>(mean, total, red[0]);
#pragma unroll
    for (int r = 0; r < R; ++r) {
      mean[r] = rounded_product(total[r], high);
      low[r] = fmaf(total[r], rest, fmaf(total[r], high, -mean[r]));
    }
  } else {
    double total[R];
    row_totals<TPR>(mean, total, red[0]);
#pragma unroll
    for (int r = 0; r < R; ++r) {
      total[r] *= inv_n * units;
      mean[r] = (float)total[r];
      low[r] = (float)(total[r] - (double)mean[r]);
    }
  }
  float sums[WIDE ? 2 * R : R];  // of the squares, and of the deviations themselves
#pragma unroll
  for (int r = 0; r < R; ++r) {
    sums[r] = 0.f;
    if constexpr (WIDE) sums[R + r] = 0.f;
#pragma unroll
    for (int c = 0; c < C; ++c) {
      if (!pc.any(c)) continue;
#pragma unroll
      for (int j = 0; j < V; ++j) {
        const float d = to_f32(raw[r][c][j]) - mean[r], dc = pc.counted(c, j, d);
        sums[r] = fmaf(d, dc, sums[r]);
        if constexpr (WIDE) sums[R + r] += dc;
      }
    }
  }
  row_totals<TPR>(sums, sums, red[1]);
#pragma unroll
  for (int r = 0; r < R; ++r) {
    if constexpr (WIDE) low[r] = sums[R + r] * (float)inv_n;
    const float var = fmaf(-low[r], low[r], sums[r] * (float)inv_n);
    rstd[r] = 1.f / sqrtf((var < 0.f ? 0.f : var) + eps);  // NaN stays
  }
#pragma unroll
  for (int c = 0; c < C; ++c) {
    if (!pc.any(c)) continue;
    if (!EARLY) weights(c);
#pragma unroll
    for (int r = 0; r < R; ++r) {
      if (row0 + r >= M) break;
      float v[V];
#pragma unroll
      for (int j = 0; j < V; ++j) {
        v[j] = fmaf(to_f32(raw[r][c][j]) - mean[r], rstd[r], -low[r] * rstd[r]);
        if (gamma) v[j] *= to_f32(g[c][j]);
        if (beta) v[j] += to_f32(b[c][j]);
      }
      store_piece<V>(y + (row0 + r) * ldy + pc.at[c], v);
    }
  }
#pragma unroll
  for (int r = 0; r < R; ++r)
    if (lane == 0 && stats && row0 + r < M) *reinterpret_cast<float2*>(stats + 2 * (row0 + r)) = make_float2(mean[r] + low[r], rstd[r]);
}

// Backward, rows that a workgroup holds.  HBM-bound: two reads and one write of the matrix.  A workgroup walks over the rows,
// kGradThreads / TPR at a time, with the next ones on their way while these are worked on; a thread keeps its columns' share
// of d_gamma and d_beta in registers over the whole walk.  What the row groups of a workgroup hold meets in LDS at the end
// and leaves as one partial row.  16 elements a thread and 512 threads: 16384 rows of 4096 bf16 74 us = 5.4 TB/s; with 1024
// threads the registers spill (102 us), without the prefetch 8192 rows of 8192 take 100 us against 81.  Nothing needs x and
// dy after this, so they do not stay in the caches (40960 rows of 512 fp32: 45 us, 50 with plain loads) -- but for odd
// widths, whose pieces share cache lines with their neighbours.
template <typename T, typename W, int TPR, int C, int V, bool TAIL>
__global__ void __launch_bounds__(kGradThreads)
    layer_norm_grad_kernel(const T* dy, long long lddy, const T* x, long long ldx, const float* stats, const W* gamma,
                           long long M, int N, float inv_n, T* dx, long long lddx, float* ws) {
  constexpr int NT = kGradThreads, RG = NT / TPR;
  typedef typename Piece<T, V>::type PT;
  __shared__ float red[2][2 * NT / 64];
  __shared__ __align__(16) float cols[NT * C * V];
  const int lane = threadIdx.x % TPR, group = threadIdx.x / TPR;
  const Pieces<TPR, C, V, TAIL> pc(lane, N);
  float g_w[C][V], acc_g[C][V], acc_b[C][V];
#pragma unroll
  for (int c = 0; c < C; ++c) {
#pragma unroll
    for (int j = 0; j < V; ++j) {
      g_w[c][j] = 1.f;
      acc_g[c][j] = acc_b[c][j] = 0.f;
    }
    if (gamma && pc.any(c)) load_piece<V>(gamma + pc.at[c], g_w[c]);
  }
  const long long step = (long long)gridDim.x * RG;
  long long row = (long long)blockIdx.x * RG + group;
  PT nx[C], nd[C];
  float2 nst;
  auto fetch = [&](long long r) {
    r = min(r, M - 1);
    nst = *reinterpret_cast<const float2*>(stats + 2 * r);
#pragma unroll
    for (int c = 0; c < C; ++c)
      if (pc.any(c)) {
        const PT *px = reinterpret_cast<const PT*>(x + r * ldx + pc.at[c]), *pd = reinterpret_cast<const PT*>(dy + r * lddy + pc.at[c]);
        nx[c] = TAIL ? *px : __builtin_nontemporal_load(px);
        nd[c] = TAIL ? *pd : __builtin_nontemporal_load(pd);
      }
  };
  fetch(row);
  int odd = 0;
  for (long long first = (long long)blockIdx.x * RG; first < M; first += step, row += step, odd ^= 1) {
    PT px[C], pd[C];
    const float mean = nst.x, rstd = nst.y;
#pragma unroll
    for (int c = 0; c < C; ++c) {
      px[c] = nx[c];
      pd[c] = nd[c];
    }
    if (first + step < M) fetch(row + step);
    const bool live = row < M;
    float s[2] = {0.f, 0.f};
    float xh[C][V], gr[C][V];
#pragma unroll
    for (int c = 0; c < C; ++c) {
      if (!pc.any(c)) continue;
#pragma unroll
      for (int j = 0; j < V; ++j) {
        const float d = to_f32(pd[c][j]);
        xh[c][j] = (to_f32(px[c][j]) - mean) * rstd;
        gr[c][j] = d * g_w[c][j];
        const float gc = pc.counted(c, j, gr[c][j]);
        s[0] += gc;
        s[1] = fmaf(gc, xh[c][j], s[1]);
        if (live) {
          acc_g[c][j] = fmaf(d, xh[c][j], acc_g[c][j]);
          acc_b[c][j] += d;
        }
      }
    }
    if (dx) {
      row_sums<TPR>(s, red[odd]);
      const float a = s[0] * inv_n, b = s[1] * inv_n;
      if (live) {
#pragma unroll
        for (int c = 0; c < C; ++c) {
          if (!pc.any(c)) continue;
          float v[V];
#pragma unroll
          for (int j = 0; j < V; ++j) v[j] = rstd * (gr[c][j] - fmaf(xh[c][j], b, a));
          store_piece<V>(dx + row * lddx + pc.at[c], v);
        }
      }
    }
  }
  if (!ws) return;
#pragma unroll
  for (int which = 0; which < 2; ++which) {
    __syncthreads();
#pragma unroll
    for (int c = 0; c < C; ++c)
#pragma unroll
      for (int j = 0; j < V; ++j) cols[group * (TPR * C * V) + (c * TPR + lane) * V + j] = which ? acc_b[c][j] : acc_g[c][j];
    __syncthreads();
    float* part = ws + ((long long)blockIdx.x * 2 + which) * N;
    for (int i = threadIdx.x; i < TPR * C * V; i += NT) {
      const int piece = i / V * V, at = TAIL ? min(piece, N - V) : piece;
      const int col = at + i % V;
      if (col < piece || col >= N) continue;  // an element of the piece before, or none
      float sum = 0.f;
#pragma unroll
      for (int k = 0; k < RG; ++k) sum += cols[k * (TPR * C * V) + i];
      part[col] = sum;
    }
  }
}

// Backward of few rows, in one launch and without a workspace: d_gamma and d_beta need the statistics, not dx, so the last
// workgroups of the grid form dx, whole rows in registers, while the first ones sum columns.  Everything is read twice,
// mostly out of a cache the second time; the pass above writes and re-reads partial rows instead, and takes a second launch.
// 100 rows of 4096 bf16: 5.5 us, 9.0 the other way; 512 rows: 9.7 and 11.8; beyond, narrow rows lose by it (1000 rows of 136
// fp32: 12.4 and 6.5) and rows of more than 8192 gain up to about 1024 (777 rows of 12345 bf16: 22 us, 29 in column tiles).
// What bounds it there is not the memory: the workgroups that form dx, alone, take 20.2 us of the 777 x 12345 case, those that
// sum columns 20.9 alone, and their second reading mostly comes from the last-level cache.  A workgroup loads a row, sums and
// stores with nothing on its way meanwhile, and two of them fit a CU (97 to 101 registers): 512 rows at a time, so that 777 rows
// are two turns (the dx half alone: 512 rows 12.5 us, 777 rows 20.2, 1000 rows 22.1).
//
// Columns: the threads of a workgroup as `rt` row threads times NT / rt threads of V columns each (8 at least: 128 bytes).
template <typename T, typename W, int V, bool TAIL, int NT>
__device__ __forceinline__ void few_columns(int block, int rt, const T* dy, long long lddy, const T* x, long long ldx,
                                            const float* stats, int M, int N, W* d_gamma, W* d_beta, float* lds) {
  const int across = NT / rt, lane = threadIdx.x & (across - 1), rl = threadIdx.x / across;
  const int i = (block * across + lane) * V, at = TAIL ? min(i, N - V) : i;
  float acc[2 * V];
#pragma unroll
  for (int j = 0; j < 2 * V; ++j) acc[j] = 0.f;
  if (i < N) {
#pragma unroll 4
    for (int m = rl; m < M; m += rt) {
      const float2 st = *reinterpret_cast<const float2*>(stats + 2 * m);
      float vx[V], vd[V];
      load_piece<V>(x + m * ldx + at, vx);
      load_piece<V>(dy + m * lddy + at, vd);
#pragma unroll
      for (int j = 0; j < V; ++j) {
        acc[j] = fmaf(vd[j], (vx[j] - st.x) * st.y, acc[j]);
        acc[V + j] += vd[j];
      }
    }
  }
  // row threads that share a wave, then the waves that share columns
  for (int d = across; d < 64; d <<= 1) {
#pragma unroll
    for (int j = 0; j < 2 * V; ++j) acc[j] += __shfl_xor(acc[j], d);
  }
  const int per_wave = across < 64 ? across : 64;       // threads of a wave that hold different columns
  const int waves = across < 64 ? NT / 64 : NT / across;  // waves that hold the same ones
  if (waves > 1) {
    const int first = across < 64 ? 0 : (threadIdx.x / 64) % (across / 64), mine = across < 64 ? threadIdx.x / 64 : rl;
    const int slot = first * 64 + (threadIdx.x & 63);
    if ((threadIdx.x & 63) < per_wave) {
#pragma unroll
      for (int j = 0; j < 2 * V; ++j) lds[(mine * 2 * V + j) * across + slot] = acc[j];
    }
    __syncthreads();
    if (mine > 0 || (threadIdx.x & 63) >= per_wave) return;
    for (int w = 1; w < waves; ++w) {
#pragma unroll
      for (int j = 0; j < 2 * V; ++j) acc[j] += lds[(w * 2 * V + j) * across + slot];
    }
  } else if ((threadIdx.x & 63) >= per_wave) {
    return;
  }
  if (i >= N) return;
#pragma unroll
  for (int j = 0; j < V; ++j) {
    if (TAIL && at + j < i) continue;  // the piece before holds it
    if (d_gamma) d_gamma[at + j] = from_f32<W>(acc[j]);
    if (d_beta) d_beta[at + j] = from_f32<W>(acc[V + j]);
  }
}

template <typename T, typename W, int TPR, int C, int V, bool TAIL>
__global__ void __launch_bounds__(TPR < kGradThreads ? kGradThreads : TPR)
    layer_norm_grad_few_kernel(int col_blocks, int rt, const T* dy, long long lddy, const T* x, long long ldx, const float* stats,
                               const W* gamma, int M, int N, float inv_n, T* dx, long long lddx, W* d_gamma, W* d_beta) {
  constexpr int NT = TPR < kGradThreads ? kGradThreads : TPR, RG = NT / TPR;
  typedef typename Piece<T, V>::type PT;
  __shared__ float lds[NT * 2 * V];
  if ((int)blockIdx.x < col_blocks)
    return few_columns<T, W, V, TAIL, NT>(blockIdx.x, rt, dy, lddy, x, ldx, stats, M, N, d_gamma, d_beta, lds);
  const int lane = threadIdx.x % TPR, row = ((int)blockIdx.x - col_blocks) * RG + threadIdx.x / TPR;
  const Pieces<TPR, C, V, TAIL> pc(lane, N);
  const bool live = row < M;
  const long long r = live ? row : M - 1;
  const float2 st = *reinterpret_cast<const float2*>(stats + 2 * r);
  PT px[C], pd[C];
#pragma unroll
  for (int c = 0; c < C; ++c) {
    if (!pc.any(c)) continue;
    px[c] = *reinterpret_cast<const PT*>(x + r * ldx + pc.at[c]);
    pd[c] = *reinterpret_cast<const PT*>(dy + r * lddy + pc.at[c]);
  }
  auto normed = [&](int c, float (&xh)[V], float (&gr)[V]) {
    float g[V];
    if (gamma) load_piece<V>(gamma + pc.at[c], g);
#pragma unroll
    for (int j = 0; j < V; ++j) {
      xh[j] = (to_f32(px[c][j]) - st.x) * st.y;
      gr[j] = to_f32(pd[c][j]);
      if (gamma) gr[j] *= g[j];
    }
  };
  // 512 threads have registers for what the sums were made of; 1024 form it again (777 rows of 12345 bf16: 24 us, 27)
  constexpr bool KEEP = NT == kGradThreads;
  float xh[KEEP ? C : 1][V], gr[KEEP ? C : 1][V], s[2] = {0.f, 0.f};
#pragma unroll
  for (int c = 0; c < C; ++c) {
    if (!pc.any(c)) continue;
    const int k = KEEP ? c : 0;
    normed(c, xh[k], gr[k]);
#pragma unroll
    for (int j = 0; j < V; ++j) {
      const float gc = pc.counted(c, j, gr[k][j]);
      s[0] += gc;
      s[1] = fmaf(gc, xh[k][j], s[1]);
    }
  }
  row_sums<TPR>(s, lds);
  if (!live) return;
  const float a = s[0] * inv_n, b = s[1] * inv_n;
#pragma unroll
  for (int c = 0; c < C; ++c) {
    if (!pc.any(c)) continue;
    const int k = KEEP ? c : 0;
    if (!KEEP) normed(c, xh[k], gr[k]);
    float v[V];
#pragma unroll
    for (int j = 0; j < V; ++j) v[j] = st.y * (gr[k][j] - fmaf(xh[k][j], b, a));
    store_piece<V>(dx + r * lddx + pc.at[c], v);
  }
}

// Backward, rows wider than that: the two sums of every row first, then a pass in which a workgroup owns a column tile and
// a slice of the rows.  Reads the matrices twice; nothing but the two sums crosses threads.  The slice is the fastest index
// of that pass's grid and a multiple of 8, so that (workgroups go to the 8 XCDs in turn) an XCD meets the rows whose sums
// it formed, the last ones first: its L2 may still hold them (whole call; first ones first; one slice more, no multiple of 8:
// 2048 x 32768 bf16 131 us, 136, 133; 4096 x 16384 fp32 283, 294, 290; 512 x 65536 fp32 138, 154, 138; 3000 x 20001
// bf16 158, 166, but 144).
template <typename T, typename W, int V, bool TAIL, int NT>
__global__ void __launch_bounds__(NT)
    layer_norm_row_sums_kernel(const T* dy, long long lddy, const T* x, long long ldx, const float* stats, const W* gamma,
                               long long M, int N, float inv_n, float2* sums) {
  __shared__ float red[2][2 * NT / 64];
  int odd = 0;
  for (long long m = blockIdx.x; m < M; m += gridDim.x, odd ^= 1) {
    const float2 st = *reinterpret_cast<const float2*>(stats + 2 * m);
    float s[2] = {0.f, 0.f};
#pragma unroll 4
    for (int i = threadIdx.x * V; i < N; i += NT * V) {
      const int at = TAIL ? min(i, N - V) : i;
      float vx[V], vd[V], g[V];
      load_piece<V>(x + m * ldx + at, vx);
      load_piece<V>(dy + m * lddy + at, vd);
      if (gamma) load_piece<V>(gamma + at, g);
#pragma unroll
      for (int j = 0; j < V; ++j) {
        const float gr = !TAIL || at + j >= i ? (gamma ? vd[j] * g[j] : vd[j]) : 0.f;
        s[0] += gr;
        s[1] = fmaf(gr, (vx[j] - st.x) * st.y, s[1]);
      }
    }
    row_sums<NT>(s, red[odd]);
    if (threadIdx.x == 0) sums[m] = make_float2(s[0] * inv_n, s[1] * inv_n);
  }
}
template <typename T, typename W, int V, bool TAIL>
__global__ void __launch_bounds__(kNThreads)
    layer_norm_wide_grad_kernel(const T* dy, long long lddy, const T* x, long long ldx, const float* stats, const W* gamma,
                                const float2* sums, long long M, int N, T* dx, long long lddx, float* ws, W* d_gamma, W* d_beta) {
  const int i = (blockIdx.y * kNThreads + threadIdx.x) * V;
  if (i >= N) return;
  const int at = TAIL ? min(i, N - V) : i;
  float g[V], acc_g[V], acc_b[V];
#pragma unroll
  for (int j = 0; j < V; ++j) {
    g[j] = 1.f;
    acc_g[j] = acc_b[j] = 0.f;
  }
  if (gamma) load_piece<V>(gamma + at, g);
#pragma unroll 2
  for (long long m = blockIdx.x + (M - 1 - blockIdx.x) / gridDim.x * gridDim.x; m >= 0; m -= gridDim.x) {
    const float2 st = *reinterpret_cast<const float2*>(stats + 2 * m);
    float vx[V], vd[V];
    load_piece<V>(x + m * ldx + at, vx);
    load_piece<V>(dy + m * lddy + at, vd);
    const float2 ab = dx ? sums[m] : make_float2(0.f, 0.f);
#pragma unroll
    for (int j = 0; j < V; ++j) {
      const float xh = (vx[j] - st.x) * st.y;
      acc_g[j] = fmaf(vd[j], xh, acc_g[j]);
      acc_b[j] += vd[j];
      vx[j] = st.y * (vd[j] * g[j] - fmaf(xh, ab.y, ab.x));
    }
    if (dx) store_piece<V>(dx + m * lddx + at, vx);
  }
  if (ws) {
    float* part = ws + (long long)blockIdx.x * 2 * N + at;
    store_piece<V>(part, acc_g);
    store_piece<V>(part + N, acc_b);
  } else {  // one slice
    if (d_gamma) store_piece<V>(d_gamma + at, acc_g);
    if (d_beta) store_piece<V>(d_beta + at, acc_b);
  }
}

// Sums the partial rows [P][2][N]: 32 columns a workgroup, K threads a column, fixed order.
template <typename W, int K>
__global__ void __launch_bounds__(32 * K) layer_norm_dw_sum_kernel(const float* ws, int P, int N, W* d_gamma, W* d_beta) {
  __shared__ float part[K][33];
  const int c = threadIdx.x & 31, k = threadIdx.x >> 5;
  const int col = blockIdx.x * 32 + c;
  float s = 0.f;
  if (col < 2 * N) {
#pragma unroll 8
    for (int p = k; p < P; p += K) s += ws[(long long)p * 2 * N + col];
  }
  part[k][c] = s;
  __syncthreads();
  if (k > 0 || col >= 2 * N) return;
  s = 0.f;
#pragma unroll
  for (int q = 0; q < K; ++q) s += part[q][c];
  if (col < N) {
    if (d_gamma) d_gamma[col] = from_f32<W>(s);
  } else if (d_beta) {
    d_beta[col - N] = from_f32<W>(s);
  }
}

}  // namespace ultr
