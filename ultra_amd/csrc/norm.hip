// Layer normalisation of the rows of a tensor, forward and backward, as operators of their own.
// Reference: NORM_FUNC_DIC of base_ranking_model.py:67-70, applied at DNN.py:78-81.
//   forward   mu = sum x / N ; v = sum (x - mu)^2 / N ; r = 1 / sqrt(v + eps) ; y = (x - mu) r gamma + beta
//   backward  xh = (x - mu) r ; g = dy gamma ; dx = r (g - sum g / N - xh sum(g xh) / N)
//             d_gamma = sum_m dy xh ; d_beta = sum_m dy
#include "storage.hpp"

#include <algorithm>
#include <type_traits>

namespace ultr {

constexpr int kNThreads = 256;
constexpr int kNMaxSlices = 64;

template <typename T, typename W>
__global__ void __launch_bounds__(kNThreads) layer_norm_kernel(const T* x, long long ldx, const W* gamma, const W* beta,
                                                               long long M, int N, float eps, T* y, long long ldy,
                                                               float* stats) {
  __shared__ float red[kNThreads / 64];
  for (long long m = blockIdx.x; m < M; m += gridDim.x) {
    const T* xr = x + m * ldx;
    T* yr = y + m * ldy;
    float s[1] = {0.f};
    for (int i = threadIdx.x; i < N; i += kNThreads) s[0] += to_f32(xr[i]);
    block_sum<1>(s, red);
    const float mean = s[0] / N;
    s[0] = 0.f;
    for (int i = threadIdx.x; i < N; i += kNThreads) {
      const float d = to_f32(xr[i]) - mean;
      s[0] = fmaf(d, d, s[0]);
    }
    block_sum<1>(s, red);
    const float rstd = 1.f / sqrtf(s[0] / N + eps);
    for (int i = threadIdx.x; i < N; i += kNThreads)
      yr[i] = from_f32<T>(fmaf((to_f32(xr[i]) - mean) * rstd, gamma ? to_f32(gamma[i]) : 1.f, beta ? to_f32(beta[i]) : 0.f));
    if (threadIdx.x == 0 && stats) {
      stats[2 * m] = mean;
      stats[2 * m + 1] = rstd;
    }
  }
}

template <typename T, typename W>
__global__ void __launch_bounds__(kNThreads) layer_norm_dx_kernel(const T* dy, long long lddy, const T* x, long long ldx,
                                                                  const float* stats, const W* gamma, long long M, int N,
                                                                  T* dx, long long lddx) {
  __shared__ float red[2 * kNThreads / 64];
  for (long long m = blockIdx.x; m < M; m += gridDim.x) {
    const T* xr = x + m * ldx;
    const T* dr = dy + m * lddy;
    const float mean = stats[2 * m], rstd = stats[2 * m + 1];
    float s[2] = {0.f, 0.f};
    for (int i = threadIdx.x; i < N; i += kNThreads) {
      const float g = to_f32(dr[i]) * (gamma ? to_f32(gamma[i]) : 1.f);
      s[0] += g;
      s[1] = fmaf(g, (to_f32(xr[i]) - mean) * rstd, s[1]);
    }
    block_sum<2>(s, red);
    const float a = s[0] / N, b = s[1] / N;
    for (int i = threadIdx.x; i < N; i += kNThreads) {
      const float g = to_f32(dr[i]) * (gamma ? to_f32(gamma[i]) : 1.f);
      dx[m * lddx + i] = from_f32<T>(rstd * (g - a - (to_f32(xr[i]) - mean) * rstd * b));
    }
  }
}

// Column sums of one slice of rows: ws[slice][0][N] of dy * xh, ws[slice][1][N] of dy.
template <typename T>
__global__ void __launch_bounds__(kNThreads) layer_norm_dw_kernel(const T* dy, long long lddy, const T* x, long long ldx,
                                                                  const float* stats, long long M, int N, float* ws) {
  const int i = blockIdx.x * kNThreads + threadIdx.x;
  if (i >= N) return;
  float dg = 0.f, db = 0.f;
  for (long long m = blockIdx.y; m < M; m += gridDim.y) {
    const float d = to_f32(dy[m * lddy + i]);
    dg = fmaf(d, (to_f32(x[m * ldx + i]) - stats[2 * m]) * stats[2 * m + 1], dg);
    db += d;
  }
  float* w = ws + (long long)blockIdx.y * 2 * N;
  w[i] = dg;
  w[N + i] = db;
}
template <typename W>
__global__ void __launch_bounds__(kNThreads) layer_norm_dw_sum_kernel(const float* ws, int slices, int N, W* d_gamma, W* d_beta) {
  const int i = blockIdx.x * kNThreads + threadIdx.x;
  if (i >= N) return;
  float dg = 0.f, db = 0.f;
  for (int s = 0; s < slices; ++s) {
    dg += ws[(long long)s * 2 * N + i];
    db += ws[(long long)s * 2 * N + N + i];
  }
  if (d_gamma) d_gamma[i] = from_f32<W>(dg);
  if (d_beta) d_beta[i] = from_f32<W>(db);
}

static int slices_of(long long M) { return (int)std::min<long long>(M, kNMaxSlices); }

// Calls fn with null pointers of the storage types: fn(T*, W*).
template <typename F>
static int with_types(int x_dtype, int w_dtype, F&& fn) {
  if (x_dtype == ULTR_DTYPE_F32) return fn((float*)nullptr, (float*)nullptr);
  if (x_dtype == ULTR_DTYPE_BF16)
    return w_dtype == ULTR_DTYPE_F32 ? fn((bf16_t*)nullptr, (float*)nullptr) : fn((bf16_t*)nullptr, (bf16_t*)nullptr);
  return w_dtype == ULTR_DTYPE_F32 ? fn((f16_t*)nullptr, (float*)nullptr) : fn((f16_t*)nullptr, (f16_t*)nullptr);
}

static int check_norm(const char* who, long long M, int N, int x_dtype, int w_dtype) {
  ULTR_REQUIRE(M >= 0 && N > 0, ULTR_EINVAL, "%s: bad sizes M=%lld N=%d", who, M, N);
  ULTR_REQUIRE(N <= ULTR_MAX_NORM_WIDTH && M <= (1ll << 40), ULTR_ELIMIT, "%s: M=%lld N=%d too large", who, M, N);
  ULTR_REQUIRE(known_dtype(x_dtype) && (w_dtype == ULTR_DTYPE_F32 || w_dtype == x_dtype), ULTR_EINVAL,
               "%s: x_dtype=%d w_dtype=%d", who, x_dtype, w_dtype);
  return ULTR_OK;
}
// A matrix argument of M rows: present, aligned to its elements, rows that do not run into each other.
static int check_rows(const char* who, const char* name, const void* p, long long ld, long long M, int N, int dtype) {
  ULTR_REQUIRE(M == 0 || p, ULTR_EINVAL, "%s: null %s", who, name);
  ULTR_REQUIRE((M <= 1 || ld >= N) && ld <= (1ll << 40), ULTR_EINVAL, "%s: rows of %s are %lld elements apart, N=%d", who, name, ld, N);
  ULTR_REQUIRE(((uintptr_t)p & (dtype_bytes(dtype) - 1)) == 0, ULTR_EINVAL, "%s: %s is not aligned to its element type", who, name);
  return ULTR_OK;
}
static bool rows_overlap(const void* a, long long lda, const void* b, long long ldb, long long M, int N, int dtype) {
  if (M == 0 || !a || !b) return false;
  const int e = dtype_bytes(dtype);
  const uintptr_t pa = (uintptr_t)a, pb = (uintptr_t)b;
  const uintptr_t ea = pa + ((uintptr_t)(M - 1) * lda + N) * e, eb = pb + ((uintptr_t)(M - 1) * ldb + N) * e;
  return pa < eb && pb < ea;
}

}  // namespace ultr

using namespace ultr;

extern "C" int ultr_layer_norm_forward(const void* x, long long ldx, const void* gamma, const void* beta, long long M, int N,
                                       float eps, int x_dtype, int w_dtype, void* y, long long ldy, float* stats,
                                       void* stream) {
  const char* who = "ultr_layer_norm_forward";
  int rc = check_norm(who, M, N, x_dtype, w_dtype);
  if (!rc) rc = check_rows(who, "x", x, ldx, M, N, x_dtype);
  if (!rc) rc = check_rows(who, "y", y, ldy, M, N, x_dtype);
  if (rc) return rc;
  ULTR_REQUIRE(eps > 0.f, ULTR_EINVAL, "%s: eps=%g", who, (double)eps);
  ULTR_REQUIRE((((uintptr_t)gamma | (uintptr_t)beta) & (dtype_bytes(w_dtype) - 1)) == 0 && ((uintptr_t)stats & 7) == 0, ULTR_EINVAL,
               "%s: gamma, beta or stats not aligned", who);
  ULTR_REQUIRE((x == y && (ldx == ldy || M <= 1)) || !rows_overlap(x, ldx, y, ldy, M, N, x_dtype), ULTR_EINVAL,
               "%s: y overlaps x without being x", who);
  if (M == 0) return ULTR_OK;
  const unsigned grid = (unsigned)std::min<long long>(M, 65536);
  {
    ProfScope prof_("layer_norm_kernel", as_stream(stream));
    with_types(x_dtype, w_dtype, [&](auto* t, auto* w) {
      using T = std::remove_pointer_t<decltype(t)>;
      using W = std::remove_pointer_t<decltype(w)>;
      hipLaunchKernelGGL((layer_norm_kernel<T, W>), dim3(grid), dim3(kNThreads), 0, as_stream(stream), (const T*)x, ldx,
                         (const W*)gamma, (const W*)beta, M, N, eps, (T*)y, ldy, stats);
      return 0;
    });
  }
  return check_launch("layer_norm_kernel");
}

extern "C" long long ultr_layer_norm_workspace_bytes(long long M, int N) {
  if (check_norm("ultr_layer_norm_workspace_bytes", M, N, ULTR_DTYPE_F32, ULTR_DTYPE_F32) != ULTR_OK) return -1;
  return (long long)slices_of(M) * 2 * N * (long long)sizeof(float);
}

extern "C" int ultr_layer_norm_backward(const void* dy, long long lddy, const void* x, long long ldx, const float* stats,
                                        const void* gamma, long long M, int N, int x_dtype, int w_dtype, void* dx,
                                        long long lddx, void* d_gamma, void* d_beta, void* ws, void* stream) {
  const char* who = "ultr_layer_norm_backward";
  int rc = check_norm(who, M, N, x_dtype, w_dtype);
  if (!rc) rc = check_rows(who, "dy", dy, lddy, M, N, x_dtype);
  if (!rc) rc = check_rows(who, "x", x, ldx, M, N, x_dtype);
  if (!rc && dx) rc = check_rows(who, "dx", dx, lddx, M, N, x_dtype);
  if (rc) return rc;
  ULTR_REQUIRE(dx || d_gamma || d_beta, ULTR_EINVAL, "%s: nothing to compute", who);
  ULTR_REQUIRE(M == 0 || stats, ULTR_EINVAL, "%s: null stats", who);
  ULTR_REQUIRE((((uintptr_t)gamma | (uintptr_t)d_gamma | (uintptr_t)d_beta) & (dtype_bytes(w_dtype) - 1)) == 0 &&
                   ((uintptr_t)stats & 7) == 0 && ((uintptr_t)ws & 15) == 0,
               ULTR_EINVAL, "%s: gamma, d_gamma, d_beta, stats or ws not aligned", who);
  ULTR_REQUIRE(!rows_overlap(dx, lddx, x, ldx, M, N, x_dtype) && !rows_overlap(dx, lddx, dy, lddy, M, N, x_dtype), ULTR_EINVAL,
               "%s: dx overlaps x or dy", who);
  const bool dw = d_gamma || d_beta;
  ULTR_REQUIRE(!dw || ws || ultr_layer_norm_workspace_bytes(M, N) == 0, ULTR_EINVAL, "%s: workspace required", who);
  hipStream_t s = as_stream(stream);
  return with_types(x_dtype, w_dtype, [&](auto* t, auto* w) {
    using T = std::remove_pointer_t<decltype(t)>;
    using W = std::remove_pointer_t<decltype(w)>;
    if (dx && M > 0) {
      {
        ProfScope prof_("layer_norm_dx_kernel", s);
        hipLaunchKernelGGL((layer_norm_dx_kernel<T, W>), dim3((unsigned)std::min<long long>(M, 65536)), dim3(kNThreads), 0, s,
                           (const T*)dy, lddy, (const T*)x, ldx, stats, (const W*)gamma, M, N, (T*)dx, lddx);
      }
      const int rc2 = check_launch("layer_norm_dx_kernel");
      if (rc2) return rc2;
    }
    if (!dw) return ULTR_OK;
    const int slices = slices_of(M);
    const unsigned gx = (unsigned)cdiv(N, kNThreads);
    if (M > 0) {
      {
        ProfScope prof_("layer_norm_dw_kernel", s);
        hipLaunchKernelGGL((layer_norm_dw_kernel<T>), dim3(gx, slices), dim3(kNThreads), 0, s, (const T*)dy, lddy, (const T*)x,
                           ldx, stats, M, N, (float*)ws);
      }
      const int rc2 = check_launch("layer_norm_dw_kernel");
      if (rc2) return rc2;
    }
    {
      ProfScope prof_("layer_norm_dw_sum_kernel", s);
      hipLaunchKernelGGL((layer_norm_dw_sum_kernel<W>), dim3(gx), dim3(kNThreads), 0, s, (const float*)ws, slices, N,
                         (W*)d_gamma, (W*)d_beta);
    }
    return check_launch("layer_norm_dw_sum_kernel");
  });
}
