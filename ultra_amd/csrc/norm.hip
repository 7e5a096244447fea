// Layer normalisation of the rows of a tensor, forward and backward, as operators of their own.
// Reference: NORM_FUNC_DIC of base_ranking_model.py:67-70, applied at DNN.py:78-81.
//   forward   mu = sum x / N ; v = sum (x - mu)^2 / N ; r = 1 / sqrt(v + eps) ; y = (x - mu) r gamma + beta
//   backward  xh = (x - mu) r ; g = dy gamma ; dx = r (g - sum g / N - xh sum(g xh) / N)
//             d_gamma = sum_m dy xh ; d_beta = sum_m dy
#include "norm_body.hpp"

#include <algorithm>
#include <type_traits>

namespace ultr {

// ---- which threads hold a row ------------------------------------------------------------------------------------------
template <int TPR_, int C_, int V_>
struct Shape {
  static constexpr int TPR = TPR_, C = C_, V = V_;
};
// The first of the shapes that holds N entries.
template <typename... S, typename F>
static void first_shape(int N, F&& fn, S... shapes) {
  (void)((N <= S::TPR * S::C * S::V ? (fn(shapes), true) : false) || ...);
}
// Forward: two 16-byte pieces a thread until a workgroup is full, then more (fp32: one or four lose 2 to 10 %).  16-bit rows
// that fill twice the threads with one piece each take those (16384 rows of 4096 bf16, fp32 weights: 49.4 us, 51.6 with two
// pieces); where many threads would be idle they do not (16969 rows of 1052 fp16: 21.7 us, 18.4 with two pieces; 1592 of 2048
// threads' worth: 15.2 and 13.6).  Rows shorter than one piece: element by element.
template <typename T, typename F>
static void forward_shape(int N, F&& fn) {
  if constexpr (sizeof(T) == 4) {
    if (N < 4) return fn(Shape<4, 1, 1>{});
    first_shape(N, fn, Shape<4, 1, 4>{}, Shape<8, 2, 4>{}, Shape<16, 2, 4>{}, Shape<32, 2, 4>{}, Shape<64, 2, 4>{}, Shape<128, 2, 4>{},
                Shape<256, 2, 4>{}, Shape<512, 2, 4>{}, Shape<1024, 2, 4>{}, Shape<1024, 4, 4>{}, Shape<1024, 8, 4>{},
                Shape<1024, 16, 4>{});
  } else {
    if (N < 8) return fn(Shape<8, 1, 1>{});
    int held = 32;  // entries that a power of two of threads holds with one piece each
    while (held < N) held *= 2;
    if (held <= 4096 && 8 * N >= 7 * held)
      first_shape(N, fn, Shape<4, 1, 8>{}, Shape<8, 1, 8>{}, Shape<16, 1, 8>{}, Shape<32, 1, 8>{}, Shape<64, 1, 8>{}, Shape<128, 1, 8>{},
                  Shape<256, 1, 8>{}, Shape<512, 1, 8>{});
    else
      first_shape(N, fn, Shape<4, 1, 8>{}, Shape<4, 2, 8>{}, Shape<8, 2, 8>{}, Shape<16, 2, 8>{}, Shape<32, 2, 8>{}, Shape<64, 2, 8>{},
                  Shape<128, 2, 8>{}, Shape<256, 2, 8>{}, Shape<512, 2, 8>{}, Shape<1024, 2, 8>{}, Shape<1024, 4, 8>{},
                  Shape<1024, 8, 8>{});
  }
}
// Backward: 16 elements a thread, up to the 512 threads of a workgroup; 16-bit rows then 32 (4096 rows of 16384 bf16: 87 us,
// 129 in column tiles; 1500 rows: 44 and 54), though that spills 5 to 7 of 256 registers; fp32 rows would spill what they
// prefetch, and rows that are only held for a moment (FEW) what fits.
constexpr int kGradWidth = 16 * kGradThreads;
constexpr int kHeldWidth16 = 2 * kGradWidth;
constexpr int kFewWidth32 = 32768;  // 16-bit types: every width
template <typename T, bool FEW, typename F>
static void grad_shape(int N, F&& fn) {
  if constexpr (sizeof(T) == 4) {
    if (N < 4) return fn(Shape<4, 1, 1>{});
    if constexpr (FEW)
      if (N > kGradWidth) return first_shape(N, fn, Shape<512, 8, 4>{}, Shape<1024, 8, 4>{});
    first_shape(N, fn, Shape<4, 1, 4>{}, Shape<4, 4, 4>{}, Shape<8, 4, 4>{}, Shape<16, 4, 4>{}, Shape<32, 4, 4>{}, Shape<64, 4, 4>{},
                Shape<128, 4, 4>{}, Shape<256, 4, 4>{}, Shape<512, 4, 4>{});
  } else {
    if (N < 8) return fn(Shape<8, 1, 1>{});
    if constexpr (FEW)
      if (N > kHeldWidth16) return first_shape(N, fn, Shape<1024, 4, 8>{}, Shape<1024, 8, 8>{});
    if (N > kGradWidth) return fn(Shape<512, 4, 8>{});
    first_shape(N, fn, Shape<4, 1, 8>{}, Shape<4, 2, 8>{}, Shape<8, 2, 8>{}, Shape<16, 2, 8>{}, Shape<32, 2, 8>{}, Shape<64, 2, 8>{},
                Shape<128, 2, 8>{}, Shape<256, 2, 8>{}, Shape<512, 2, 8>{});
  }
}

// Which of the three backward passes: few rows in one launch; rows that a workgroup holds; wider ones.
enum GradPass { kFew, kHeld, kWide };
static GradPass grad_pass(long long M, int N, int x_dtype) {
  if (N <= kGradWidth) return M <= 512 ? kFew : kHeld;
  if (M <= 1024 && (x_dtype != ULTR_DTYPE_F32 || N <= kFewWidth32)) return kFew;
  return x_dtype != ULTR_DTYPE_F32 && N <= kHeldWidth16 ? kHeld : kWide;
}
// Row groups' workgroups of the held pass = its partial rows.  One per CU; half of them while each would get fewer than 3
// turns (the partial rows cost more than the idle CUs: 1000 rows of 4096 bf16 14.3 us with 128, 15.4 with 256; 3000 rows
// 25.4 and 22.1).
static int held_blocks(long long M, int rg) {
  const long long turns = cdiv(M, rg);
  return (int)std::min<long long>(turns, turns < 3 * 256 ? 128 : 256);
}
// Row slices of the wide pass: about 512 workgroups, at least 4 rows each; a multiple of 8 (see the kernel) unless that few.
static int wide_slices(long long M, int N, int x_dtype) {
  const int tiles = (int)cdiv(N, kNThreads * (x_dtype == ULTR_DTYPE_F32 ? 4 : 8));
  const long long s = std::min<long long>((512 / tiles + 7) / 8 * 8, M / 4);
  return (int)(s < 8 ? std::max<long long>(s, 1) : s / 8 * 8);
}
// Column threads of a workgroup in the few-rows pass: 8 of them (128 bytes of a row), more for wide rows so that about 128
// workgroups sum columns (512 rows of 32768 fp32: 56 us with 128, 67 with 512).
static int few_across(int N, int threads, int V) {
  int a = 8;
  while (N > kGradWidth && a < threads && (long long)a * a * 2 * 128 * 128 < ((long long)N / V) * (N / V)) a *= 2;
  return a;
}
static int partial_rows(long long M, int N, int x_dtype) {
  const GradPass p = grad_pass(M, N, x_dtype);
  if (p == kWide) return wide_slices(M, N, x_dtype);
  int parts = 0;
  auto set = [&](auto s) { parts = held_blocks(M, kGradThreads / decltype(s)::TPR); };
  if (p == kHeld) x_dtype == ULTR_DTYPE_F32 ? grad_shape<float, false>(N, set) : grad_shape<bf16_t, false>(N, set);
  return parts;
}

// One grid holds fewer than 2^32 threads: longer matrices go in slabs of whole workgroups.
constexpr long long kSlabBlocks = 1ll << 21;

// Calls fn with null pointers of the storage types: fn(T*, W*).
template <typename F>
static int with_types(int x_dtype, int w_dtype, F&& fn) {
  if (x_dtype == ULTR_DTYPE_F32) return fn((float*)nullptr, (float*)nullptr);
  if (x_dtype == ULTR_DTYPE_BF16)
    return w_dtype == ULTR_DTYPE_F32 ? fn((bf16_t*)nullptr, (float*)nullptr) : fn((bf16_t*)nullptr, (bf16_t*)nullptr);
  return w_dtype == ULTR_DTYPE_F32 ? fn((f16_t*)nullptr, (float*)nullptr) : fn((f16_t*)nullptr, (f16_t*)nullptr);
}

template <typename W>
static int launch_dw_sum(const float* part, int parts, int N, W* d_gamma, W* d_beta, hipStream_t s) {
  {
    ProfScope prof_("layer_norm_dw_sum_kernel", s);
    const unsigned grid = (unsigned)cdiv(2 * N, 32);
    if (parts > 64)
      hipLaunchKernelGGL((layer_norm_dw_sum_kernel<W, 32>), dim3(grid), dim3(1024), 0, s, part, parts, N, d_gamma, d_beta);
    else
      hipLaunchKernelGGL((layer_norm_dw_sum_kernel<W, 8>), dim3(grid), dim3(256), 0, s, part, parts, N, d_gamma, d_beta);
  }
  return check_launch("layer_norm_dw_sum_kernel");
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
// Memory of an argument: rows of `width` bytes, `pitch` bytes apart.
struct Extent {
  uint64_t at, end, pitch, width;
  bool one;  // row
};
static Extent vector(const void* p, long long bytes) {
  const uint64_t at = (uint64_t)(uintptr_t)p;
  return {at, p ? at + bytes : 0, 0, (uint64_t)bytes, true};  // a null pointer: nothing
}
static Extent matrix(const void* p, long long ld, long long M, int N, int dtype) {
  Extent v = vector(p, M == 0 ? 0 : (long long)N * dtype_bytes(dtype));
  if (!p || M <= 1) return v;
  v.one = false;
  v.pitch = (uint64_t)ld * dtype_bytes(dtype);
  uint64_t more;
  if (__builtin_mul_overflow((uint64_t)(M - 1), v.pitch, &more) || __builtin_add_overflow(v.end, more, &v.end)) v.end = UINT64_MAX;
  return v;
}
// Whether the two have a byte in common.  Rows that lie between each other's (columns of one table) do not; of matrices with
// different pitches nothing but their ends is looked at.
static bool touch(const Extent& a, const Extent& b) {
  if (b.at >= a.end || a.at >= b.end) return false;
  const Extent &f = a.at <= b.at ? a : b, &s = a.at <= b.at ? b : a;  // the first and the second to begin
  if (f.one || (!s.one && f.pitch != s.pitch)) return true;
  const uint64_t in = (s.at - f.at) % f.pitch;  // the second begins this far behind a row of the first
  return in < f.width || (s.at - in + f.pitch < f.end && in + s.width > f.pitch);
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
  const Extent mx = matrix(x, ldx, M, N, x_dtype), my = matrix(y, ldy, M, N, x_dtype);
  ULTR_REQUIRE((x == y && (ldx == ldy || M <= 1)) || !touch(mx, my), ULTR_EINVAL, "%s: y overlaps x without being x", who);
  const Extent weights[] = {vector(gamma, (long long)N * dtype_bytes(w_dtype)), vector(beta, (long long)N * dtype_bytes(w_dtype))};
  const Extent ms = vector(stats, M * 8);
  bool shared = touch(ms, mx) || touch(ms, my);
  for (const Extent& w : weights) shared = shared || touch(w, my) || touch(w, ms);
  ULTR_REQUIRE(!shared, ULTR_EINVAL, "%s: y or stats overlaps another argument", who);
  if (M == 0) return ULTR_OK;
  hipStream_t s = as_stream(stream);
  const double inv_n = 1.0 / N;
  with_types(x_dtype, w_dtype, [&](auto* t, auto* w) {
    using T = std::remove_pointer_t<decltype(t)>;
    using W = std::remove_pointer_t<decltype(w)>;
    forward_shape<T>(N, [&](auto shape) {
      using S = decltype(shape);
      constexpr int NT = S::TPR < 256 ? 256 : S::TPR;
      auto go = [&](auto tail, auto r) {
        constexpr int R = decltype(r)::value;
        constexpr long long rows = (long long)R * (NT / S::TPR);
        for (long long m = 0; m < M; m += kSlabBlocks * rows) {
          const long long n = std::min(M - m, kSlabBlocks * rows);
          ProfScope prof_("layer_norm_kernel", s);
          hipLaunchKernelGGL((layer_norm_kernel<T, W, S::TPR, S::C, S::V, decltype(tail)::value, R>), dim3((unsigned)cdiv(n, rows)),
                             dim3(NT), 0, s, (const T*)x + m * ldx, ldx, (const W*)gamma, (const W*)beta, n, N, inv_n, eps,
                             (T*)y + m * ldy, ldy, stats ? stats + 2 * m : nullptr);
        }
      };
      // two rows a thread group once there are rows enough to fill the chip that way, and registers for both: it is for
      // matrices beyond the caches with weights as wide (one row against two: 16384 x 4096 bf16 56.3 us and 49, with fp32
      // weights 60.8 and 50.4; 30010 x 5003 fp16 160 and 124; 3001 x 5003 15.9 and 15.2; 2048 x 4096 fp32 13.0 and
      // 12.1).  Those that the caches hold and narrow rows are within 10 % either way (4096 x 4096 bf16 14.6 and
      // 15.5; 40960 x 512 fp32 30.6 and 31.2; 16969 x 1052 fp16 18.0 and 19.0; 40960 x 700 fp32 42.8 and 42.0).
      constexpr bool pair = S::C * S::V * sizeof(T) <= 64;
      auto rows = [&](auto tail) {
        if constexpr (pair) {
          if (M >= 2048) return go(tail, std::integral_constant<int, 2>{});
        }
        go(tail, std::integral_constant<int, 1>{});
      };
      if (S::V > 1 && N % S::V) rows(std::integral_constant<bool, (S::V > 1)>{});
      else rows(std::false_type{});
    });
    return 0;
  });
  return check_launch("layer_norm_kernel");
}

// Row sums of the wide pass | partial rows of d_gamma and d_beta.
static long long sums_bytes(long long M, int N, int x_dtype) {
  return grad_pass(M, N, x_dtype) == kWide ? (M * 8 + 15) / 16 * 16 : 0;
}
extern "C" long long ultr_layer_norm_workspace_bytes(long long M, int N) {
  if (check_norm("ultr_layer_norm_workspace_bytes", M, N, ULTR_DTYPE_F32, ULTR_DTYPE_F32) != ULTR_OK) return -1;
  if (M == 0) return 0;
  long long most = 0;  // the types share one size
  for (int d : {ULTR_DTYPE_F32, ULTR_DTYPE_BF16}) {
    const long long p = partial_rows(M, N, d);
    most = std::max(most, sums_bytes(M, N, d) + (p > 1 ? p * 2 * N * (long long)sizeof(float) : 0));
  }
  return most;
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
  const bool dw = d_gamma || d_beta;
  const long long ws_bytes = !dw && N <= kGradWidth ? 0 : ultr_layer_norm_workspace_bytes(M, N);
  ULTR_REQUIRE(ws || ws_bytes == 0, ULTR_EINVAL, "%s: workspace required", who);
  {
    const long long w = (long long)N * dtype_bytes(w_dtype);
    const Extent in[] = {matrix(x, ldx, M, N, x_dtype), matrix(dy, lddy, M, N, x_dtype), vector(stats, M * 8), vector(gamma, w)};
    const Extent out[] = {matrix(dx, lddx, M, N, x_dtype), vector(d_gamma, w), vector(d_beta, w), vector(ws, ws_bytes)};
    static const char* const in_name[] = {"x", "dy", "stats", "gamma"};
    static const char* const out_name[] = {"dx", "d_gamma", "d_beta", "ws"};
    for (int o = 0; o < 4; ++o) {
      for (int i = 0; i < 4; ++i)
        ULTR_REQUIRE(!touch(out[o], in[i]), ULTR_EINVAL, "%s: %s overlaps %s", who, out_name[o], in_name[i]);
      for (int i = 0; i < o; ++i)
        ULTR_REQUIRE(!touch(out[o], out[i]), ULTR_EINVAL, "%s: %s overlaps %s", who, out_name[o], out_name[i]);
    }
  }
  hipStream_t s = as_stream(stream);
  const float inv_n = 1.f / (float)N;
  return with_types(x_dtype, w_dtype, [&](auto* t, auto* w) {
    using T = std::remove_pointer_t<decltype(t)>;
    using W = std::remove_pointer_t<decltype(w)>;
    if (M == 0 && !dw) return ULTR_OK;
    if (M == 0) return launch_dw_sum(nullptr, 0, N, (W*)d_gamma, (W*)d_beta, s);
    const GradPass pass = grad_pass(M, N, x_dtype);
    const int parts = partial_rows(M, N, x_dtype);
    float* part = dw && parts > 1 ? (float*)((char*)ws + sums_bytes(M, N, x_dtype)) : nullptr;
    if (pass == kFew) {
      grad_shape<T, true>(N, [&](auto shape) {
        using S = decltype(shape);
        constexpr int NT = S::TPR < kGradThreads ? kGradThreads : S::TPR, RG = NT / S::TPR;
        int rt = NT / few_across(N, NT, S::V);
        while (rt > 1 && rt / 2 >= M) rt /= 2;
        const int cols = dw ? (int)cdiv(N, NT / rt * S::V) : 0, rows = dx ? (int)cdiv(M, RG) : 0;
        auto go = [&](auto tail) {
          ProfScope prof_("layer_norm_grad_few_kernel", s);
          hipLaunchKernelGGL((layer_norm_grad_few_kernel<T, W, S::TPR, S::C, S::V, decltype(tail)::value>), dim3(cols + rows),
                             dim3(NT), 0, s, cols, rt, (const T*)dy, lddy, (const T*)x, ldx, stats, (const W*)gamma, (int)M, N,
                             inv_n, (T*)dx, lddx, (W*)d_gamma, (W*)d_beta);
        };
        if (S::V > 1 && N % S::V) go(std::integral_constant<bool, (S::V > 1)>{});
        else go(std::false_type{});
      });
    } else if (pass == kHeld) {
      grad_shape<T, false>(N, [&](auto shape) {
        using S = decltype(shape);
        auto go = [&](auto tail) {
          ProfScope prof_("layer_norm_grad_kernel", s);
          hipLaunchKernelGGL((layer_norm_grad_kernel<T, W, S::TPR, S::C, S::V, decltype(tail)::value>), dim3(parts),
                             dim3(kGradThreads), 0, s, (const T*)dy, lddy, (const T*)x, ldx, stats, (const W*)gamma, M, N, inv_n,
                             (T*)dx, lddx, part);
        };
        if (S::V > 1 && N % S::V) go(std::integral_constant<bool, (S::V > 1)>{});
        else go(std::false_type{});
      });
    } else {
      constexpr int V = 16 / sizeof(T);
      float2* sums = (float2*)ws;
      auto go = [&](auto tail) {
        constexpr bool TAIL = decltype(tail)::value;
        auto row_sums_of = [&](auto threads) {
          constexpr int NT = decltype(threads)::value;
          ProfScope prof_("layer_norm_row_sums_kernel", s);
          hipLaunchKernelGGL((layer_norm_row_sums_kernel<T, W, V, TAIL, NT>), dim3((unsigned)std::min<long long>(M, 2048)), dim3(NT),
                             0, s, (const T*)dy, lddy, (const T*)x, ldx, stats, (const W*)gamma, M, N, inv_n, sums);
        };
        // 16-bit rows that come here: small workgroups, more rows at a time (whole call, 256 threads against 1024: 3000 x
        // 20001 bf16 158 us and 169, 8192 x 20000 fp16 324 and 334, 2048 x 32768 bf16 131 and 134, though 1100 x 65536
        // 163 and 151).  fp32 rows that give 1024 threads three pieces each: all of them (4096 x 16384 283 us and 273,
        // 2000 x 12345 110 and 104.5, 1100 x 32768 165 and 150, 8 x 65536 33.6 and 17.8; 1100 x 9000 41.8 and 42.7).
        if (dx) {
          if (sizeof(T) == 2 || N < 3 * 1024 * V) row_sums_of(std::integral_constant<int, 256>{});
          else row_sums_of(std::integral_constant<int, sizeof(T) == 2 ? 256 : 1024>{});
        }
        ProfScope prof_("layer_norm_wide_grad_kernel", s);
        hipLaunchKernelGGL((layer_norm_wide_grad_kernel<T, W, V, TAIL>), dim3(parts, (unsigned)cdiv(N, kNThreads * V)),
                           dim3(kNThreads), 0, s, (const T*)dy, lddy, (const T*)x, ldx, stats, (const W*)gamma, sums, M, N, (T*)dx,
                           lddx, part, part ? nullptr : (W*)d_gamma, part ? nullptr : (W*)d_beta);
      };
      if (N % V) go(std::true_type{});
      else go(std::false_type{});
    }
    const int rc2 = check_launch("layer_norm_grad_kernel");
    return rc2 || !part ? rc2 : launch_dw_sum(part, parts, N, (W*)d_gamma, (W*)d_beta, s);
  });
}
