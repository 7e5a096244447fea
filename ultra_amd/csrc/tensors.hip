// Global norm, clipping and the optimiser update over a list of separate tensors.
// Reference: the clip by the global norm and the optimiser step over the variable list, dla.py:237-255, ipw_rank.py:155-165.
//   e = scale * g (+ l2 * theta) ; norm = sqrt(sum e^2) ; f = clip / max(norm, clip) ; out = f e, or
//   acc += (f e)^2, theta -= lr f e / sqrt(acc).
// The norm is needed before the first output: two passes over the gradients, one launch each.
#include "storage.hpp"

#include <algorithm>
#include <new>
#include <type_traits>
#include <vector>

namespace ultr {

constexpr int kTThreads = 256;
constexpr int kChunk = 4096;       // elements of one tensor that one workgroup takes at a time
// Workgroups of a pass, and partial sums of a norm.  Between 1024 and 2048 of them the times differ by 1 to 4 % (1000 ragged
// tensors, 2101 chunks: 15.2 us with 1024, 14.8 with 1536, 15.6 with 2048; clip of 553 M bf16 560, 539, 543; update of 151
// M 567, 565, 564; small lists alike).
constexpr int kTMaxBlocks = 1536;
// The last-level cache.  A second pass that moves more than this sends its data past the caches (NT): nothing of it would be there
// when something reads it again.  One that moves less leaves its outputs there, and its inputs may lie there already.  One
// list again and again, NT against plain: clip of fp32 224 MB 54.8 us and 53.3, 256 MB 61.9 and 61.8, 288 MB 69.8 and
// 72.6, 384 MB 92 and 101; of bf16 320 MB 75.6 and 80.6; update 200 MB 43.0 and 43.9, 320 MB 65.3 and 66.2, 480 MB 95 and
// 100.  (Three lists in turn, whose data the caches do not hold, gain from 128 MB on: 32.4 us and 38.0.)  60000 tensors of ten
// elements, 5 MB: 88 us and 78.
// A first pass over more gradients than this does the same, but for the last gradients of that size, with which the second pass
// begins (clip of 553 M bf16: 542 us, 625 without both; update of 151 M: 564 us, 666 without both; the last 128 MB or 512
// MB instead of 256 lose 0 to 4 %).
constexpr long long kCacheBytes = 256ll << 20;

struct ChunkRec {  // what one chunk needs: its tensor's pointers, moved to its first element
  const void* grad;
  void* out;
  float* param;
  float* accum;
  void* copy;
  int n;
  short grad_dtype, copy_dtype;
};
static_assert(sizeof(ChunkRec) == 48, "read as 12 words");

// Table: partial sums of the norm | the scale | a record per chunk.  One dependent load from a workgroup's number to its data;
// 48 bytes for the 8 KB or more that a full chunk moves.
constexpr long long kPartialBytes = kTMaxBlocks * sizeof(double);
constexpr long long kHeadBytes = kPartialBytes + 16;
static long long table_bytes_of(long long n_chunks) { return kHeadBytes + n_chunks * (long long)sizeof(ChunkRec); }

struct ListView {
  double* partials;
  float* scale;  // what the first pass made of denom: the second one may be overwriting that memory
  const ChunkRec* chunks;
  long long n_chunks;
  long long keep_from;  // the chunks from here on hold the last kCacheBytes of the gradients
};

constexpr int kFillTensors = 48;  // tensors per fill launch: they travel as kernel arguments (3 KB)
struct FillArgs {
  UltrTensor t[kFillTensors];
  long long first_chunk[kFillTensors];
};
__global__ void __launch_bounds__(kTThreads) tensors_fill_kernel(FillArgs a, ChunkRec* chunks) {
  const UltrTensor t = a.t[blockIdx.x];
  const int g = t.grad_dtype == ULTR_DTYPE_F32 ? 4 : 2, cp = t.copy_dtype == ULTR_DTYPE_F32 ? 4 : 2;
  for (long long c = (long long)blockIdx.y * blockDim.x + threadIdx.x; c * kChunk < t.n; c += (long long)gridDim.y * blockDim.x) {
    const long long i = c * kChunk;
    ChunkRec r;
    r.grad = (const char*)t.grad + i * g;
    r.out = t.out ? (char*)t.out + i * g : nullptr;
    r.param = t.param ? t.param + i : nullptr;
    r.accum = t.accum ? t.accum + i : nullptr;
    r.copy = t.copy ? (char*)t.copy + i * cp : nullptr;
    r.n = (int)min(t.n - i, (long long)kChunk);
    r.grad_dtype = (short)t.grad_dtype;
    r.copy_dtype = (short)t.copy_dtype;
    chunks[a.first_chunk[blockIdx.x] + c] = r;
  }
}

// Sum of one double per thread over the workgroup, fixed order; valid in every thread.  Once per kernel (red is not reused).
__device__ __forceinline__ double block_sum_f64(double v, double* red) {
#pragma unroll
  for (int m = 32; m >= 1; m >>= 1) v += __shfl_xor(v, m);
  if ((threadIdx.x & 63) == 0) red[threadIdx.x >> 6] = v;
  lds_barrier();
  double s = 0.0;
#pragma unroll
  for (int w = 0; w < kTThreads / 64; ++w) s += red[w];
  return s;
}

// A chunk as a workgroup walks it, in pieces of V elements: all of a thread's pieces are loaded before the first is stored
// (memory that may be the same for all the compiler knows keeps its order), in chunks that are not full too.  What is left
// beyond whole pieces goes element by element to the last threads, whose wave has the least else to do there.
// fn(at, ok, pieces, width): handle the pieces k of `width` elements at at(k) for which ok(k).
template <int V, typename F>
__device__ __forceinline__ void walk_chunk(int n, F&& fn) {
  constexpr std::integral_constant<int, kChunk / (V * kTThreads)> pieces{};
  constexpr std::integral_constant<int, V> width{};
  auto at = [&](int k) { return (k * kTThreads + (int)threadIdx.x) * V; };
  if (n == kChunk) {
    fn(at, [](int) { return true; }, pieces, width);
  } else {
    fn(at, [&](int k) { return at(k) + V <= n; }, pieces, width);
    const int rest = n % V, j = kTThreads - 1 - (int)threadIdx.x;
    if (j < rest) fn([&](int) { return n - rest + j; }, [](int) { return true; }, std::integral_constant<int, 1>{}, std::integral_constant<int, 1>{});
  }
}

__device__ __forceinline__ float scale_of(const float* denom, float scale_const) {
  return denom ? scale_const / denom[0] : scale_const;
}

// f of the header's formulas; the norm is the correctly rounded square root of a 64-bit sum.
__device__ __forceinline__ float clip_factor(double sumsq, float clip_norm, float* norm) {
  const double n = sqrt(sumsq);
  *norm = (float)n;
  if (clip_norm <= 0.f) return 1.f;
  if (!isfinite(*norm)) return __int_as_float(0x7fc00000);
  return n > (double)clip_norm ? (float)((double)clip_norm / n) : 1.f;
}

// fn(T*) for a storage type; it is the same for a whole chunk, so this is a scalar branch.
template <typename F>
__device__ __forceinline__ void with_type(int dtype, F&& fn) {
  if (dtype == ULTR_DTYPE_F32) fn((float*)nullptr);
  else if (dtype == ULTR_DTYPE_BF16) fn((bf16_t*)nullptr);
  else fn((f16_t*)nullptr);
}

// A record read by the whole wave: the same for every lane, kept in scalar registers.
__device__ __forceinline__ ChunkRec record_of(const ChunkRec* p) {
  union {
    ChunkRec r;
    unsigned w[12];
  } u;
  const uint4* q = reinterpret_cast<const uint4*>(p);
#pragma unroll
  for (int i = 0; i < 3; ++i) {
    const uint4 v = q[i];
    u.w[4 * i] = __builtin_amdgcn_readfirstlane(v.x);
    u.w[4 * i + 1] = __builtin_amdgcn_readfirstlane(v.y);
    u.w[4 * i + 2] = __builtin_amdgcn_readfirstlane(v.z);
    u.w[4 * i + 3] = __builtin_amdgcn_readfirstlane(v.w);
  }
  return u.r;
}

// The chunks of one workgroup, every gridDim.x-th one.  With `down` the last of them first: the pass that reads the gradients
// a second time starts with what the first one read last, and an XCD (workgroups go to the 8 XCDs in turn) meets its own
// chunks again.
template <typename F>
__device__ __forceinline__ void for_chunks(const ChunkRec* chunks, long long n_chunks, bool down, F&& fn) {
  long long c = blockIdx.x;
  if (c >= n_chunks) return;
  const long long step = down ? -(long long)gridDim.x : (long long)gridDim.x;
  if (down) c += (n_chunks - 1 - c) / gridDim.x * gridDim.x;
  ChunkRec r = record_of(chunks + c);
  while (true) {
    fn(r);
    c += step;
    if (c < 0 || c >= n_chunks) return;
    r = record_of(chunks + c);
  }
}

// First pass.  HBM-bound: one read of the gradients (and of the parameters with l2).  Squares are summed in 64 bits: fp32
// squares of a gradient of 1e-25 vanish and those of 1e25 overflow; the conversion and the 64-bit fma run at rates that
// leave the memory the bound.
template <bool NT>
__device__ __forceinline__ void add_squares(const ChunkRec& r, float sc, float l2, double& acc) {
  with_type(r.grad_dtype, [&](auto* t) {
    using T = std::remove_pointer_t<decltype(t)>;
    const T* g = static_cast<const T*>(r.grad);
    walk_chunk<16 / sizeof(T)>(r.n, [&](auto at, auto ok, auto pieces, auto width) {
      constexpr int K = decltype(pieces)::value, V = decltype(width)::value;
      float e[K][V];
#pragma unroll
      for (int k = 0; k < K; ++k)
        if (ok(k)) load_piece<V, NT>(g + at(k), e[k]);
#pragma unroll
      for (int k = 0; k < K; ++k) {
        if (!ok(k)) continue;
        float p[V] = {};
        if (l2 != 0.f) load_piece<V>(r.param + at(k), p);
#pragma unroll
        for (int j = 0; j < V; ++j) {
          const float v = fmaf(l2, p[j], e[k][j] * sc);
          acc += (double)v * (double)v;
        }
      }
    });
  });
}
template <bool STREAM>
__global__ void __launch_bounds__(kTThreads) tensors_sumsq_kernel(ListView l, const float* denom, float scale_const, float l2) {
  __shared__ double red[kTThreads / 64];
  const float sc = scale_of(denom, scale_const);
  double acc = 0.0;
  // whole turns of the grid, so that a chunk belongs to the same workgroup in both passes
  const long long past = STREAM ? l.keep_from / gridDim.x * gridDim.x : 0;
  if (STREAM) for_chunks(l.chunks, past, false, [&](const ChunkRec& r) { add_squares<true>(r, sc, l2, acc); });
  for_chunks(l.chunks + past, l.n_chunks - past, false, [&](const ChunkRec& r) { add_squares<false>(r, sc, l2, acc); });
  acc = block_sum_f64(acc, red);
  if (threadIdx.x == 0) {
    l.partials[blockIdx.x] = acc;
    if (blockIdx.x == 0) *l.scale = sc;
  }
}

__device__ __forceinline__ double partials_sum(const double* partials, int n, double* red) {
  double v = 0.0;
  for (int i = threadIdx.x; i < n; i += kTThreads) v += partials[i];
  return block_sum_f64(v, red);
}

__global__ void __launch_bounds__(kTThreads) tensors_norm_kernel(const double* partials, int n_partials, float* out_norm) {
  __shared__ double red[kTThreads / 64];
  const double s = partials_sum(partials, n_partials, red);
  if (threadIdx.x == 0) out_norm[0] = (float)sqrt(s);
}

template <bool STREAM>
__global__ void __launch_bounds__(kTThreads) tensors_clip_kernel(ListView l, int n_partials, float clip_norm,
                                                                 float* out_norm) {
  __shared__ double red[kTThreads / 64];
  const float sc = *l.scale;
  float f = 1.f;
  bool pending = true;
  auto factor = [&] {  // the norm, once, with the first chunk's elements on their way; every thread comes here
    if (!pending) return;
    pending = false;
    float norm;
    f = clip_factor(partials_sum(l.partials, n_partials, red), clip_norm, &norm);
    if (blockIdx.x == 0 && threadIdx.x == 0 && out_norm) out_norm[0] = norm;
  };
  for_chunks(l.chunks, l.n_chunks, true, [&](const ChunkRec& r) {
    with_type(r.grad_dtype, [&](auto* t) {
      using T = std::remove_pointer_t<decltype(t)>;
      const T* g = static_cast<const T*>(r.grad);
      T* o = static_cast<T*>(r.out);
      walk_chunk<16 / sizeof(T)>(r.n, [&](auto at, auto ok, auto pieces, auto width) {
        constexpr int K = decltype(pieces)::value, V = decltype(width)::value;
        float e[K][V];
#pragma unroll
        for (int k = 0; k < K; ++k)
          if (ok(k)) load_piece<V, STREAM>(g + at(k), e[k]);
        factor();
#pragma unroll
        for (int k = 0; k < K; ++k) {
          if (!ok(k)) continue;
#pragma unroll
          for (int j = 0; j < V; ++j) e[k][j] = e[k][j] * sc * f;
          store_piece<V, STREAM>(o + at(k), e[k]);
        }
      });
    });
  });
}

// Second pass of the update.  HBM-bound: reads gradient, parameter and accumulator, writes the last two and the copy.
template <bool STREAM>
__global__ void __launch_bounds__(kTThreads) tensors_update_kernel(ListView l, int n_partials, bool scaled,
                                                                   float scale_const, float l2, float clip_norm, float lr,
                                                                   int strategy, float* out_norm) {
  __shared__ double red[kTThreads / 64];
  const float sc = scaled ? *l.scale : scale_const;
  float f = 1.f;
  bool pending = n_partials > 0;
  auto factor = [&] {  // as above
    if (!pending) return;
    pending = false;
    float norm;
    f = clip_factor(partials_sum(l.partials, n_partials, red), clip_norm, &norm);
    if (blockIdx.x == 0 && threadIdx.x == 0 && out_norm) out_norm[0] = norm;
  };
  const bool ada = strategy == ULTR_OPT_ADAGRAD;
  for_chunks(l.chunks, l.n_chunks, true, [&](const ChunkRec& r) {
    with_type(r.grad_dtype, [&](auto* gt) {
      using T = std::remove_pointer_t<decltype(gt)>;
      const T* g = static_cast<const T*>(r.grad);
      walk_chunk<4>(r.n, [&](auto at, auto ok, auto pieces, auto width) {
        constexpr int K = decltype(pieces)::value, V = decltype(width)::value;
        float e[K][V], t[K][V], a[K][V];
#pragma unroll
        for (int k = 0; k < K; ++k) {
          if (!ok(k)) continue;
          load_piece<V, STREAM>(g + at(k), e[k]);
          load_piece<V, STREAM>(r.param + at(k), t[k]);
          if (ada) load_piece<V, STREAM>(r.accum + at(k), a[k]);
        }
        factor();
#pragma unroll
        for (int k = 0; k < K; ++k) {
          if (!ok(k)) continue;
#pragma unroll
          for (int j = 0; j < V; ++j) {
            const float v = fmaf(l2, t[k][j], e[k][j] * sc) * f;
            if (ada) {
              a[k][j] = fmaf(v, v, a[k][j]);
              t[k][j] -= lr * v / sqrtf(a[k][j]);
            } else {
              t[k][j] -= lr * v;
            }
          }
          store_piece<V, STREAM>(r.param + at(k), t[k]);
          if (ada) store_piece<V, STREAM>(r.accum + at(k), a[k]);
        }
        if (r.copy) {
          with_type(r.copy_dtype, [&](auto* ct) {
            using C = std::remove_pointer_t<decltype(ct)>;
#pragma unroll
            for (int k = 0; k < K; ++k)
              if (ok(k)) store_piece<V, STREAM>(static_cast<C*>(r.copy) + at(k), t[k]);
          });
        }
      });
    });
  });
}

// ---- host ------------------------------------------------------------------------------------
static int check_list(const char* who, const UltrTensor* t, int n, long long* n_chunks) {
  ULTR_REQUIRE(n >= 0 && (n == 0 || t), ULTR_EINVAL, "%s: bad list (n_tensors=%d)", who, n);
  long long chunks = 0;
  for (int i = 0; i < n; ++i) {
    const UltrTensor& a = t[i];
    ULTR_REQUIRE(a.n >= 0, ULTR_EINVAL, "%s: tensor %d has n=%lld", who, i, a.n);
    ULTR_REQUIRE(known_dtype(a.grad_dtype), ULTR_EINVAL, "%s: tensor %d has grad_dtype=%d", who, i, a.grad_dtype);
    if (a.n == 0) continue;
    ULTR_REQUIRE(a.n <= (1ll << 40), ULTR_ELIMIT, "%s: tensor %d has n=%lld", who, i, a.n);
    ULTR_REQUIRE(a.grad, ULTR_EINVAL, "%s: tensor %d has no gradient", who, i);
    ULTR_REQUIRE(!a.copy || (a.param && known_dtype(a.copy_dtype)), ULTR_EINVAL, "%s: tensor %d: a copy needs a parameter and a known dtype (copy_dtype=%d)",
                 who, i, a.copy_dtype);
    const int g = dtype_bytes(a.grad_dtype) - 1, c = a.copy ? dtype_bytes(a.copy_dtype) - 1 : 0;
    ULTR_REQUIRE((((uintptr_t)a.grad | (uintptr_t)a.out) & g) == 0 && (((uintptr_t)a.param | (uintptr_t)a.accum) & 3) == 0 &&
                     ((uintptr_t)a.copy & c) == 0,
                 ULTR_EINVAL, "%s: tensor %d is not aligned to its element type", who, i);
    chunks += (a.n + kChunk - 1) / kChunk;
  }
  ULTR_REQUIRE(chunks < (1ll << 31), ULTR_ELIMIT, "%s: too many elements in the list", who);
  *n_chunks = chunks;
  return ULTR_OK;
}

// Memory that a call writes must belong to one role of one tensor: two workgroups would race on it otherwise.
static int check_overlap(const char* who, const UltrTensor* t, int n) {
  struct Range {
    uintptr_t b, e;
    int tensor;
    bool written;
  };
  std::vector<Range> v;
  v.reserve(5 * (size_t)n);
  for (int i = 0; i < n; ++i) {
    const UltrTensor& a = t[i];
    if (a.n == 0) continue;
    auto add = [&](const void* p, int bytes, bool written) {
      if (p) v.push_back(Range{(uintptr_t)p, (uintptr_t)p + (uintptr_t)a.n * bytes, i, written});
    };
    const int g = dtype_bytes(a.grad_dtype);
    if (a.out != a.grad) add(a.grad, g, false);  // in place: the output stands for both
    add(a.out, g, true);
    add(a.param, 4, true);
    add(a.accum, 4, true);
    add(a.copy, a.copy ? dtype_bytes(a.copy_dtype) : 0, true);
  }
  std::sort(v.begin(), v.end(), [](const Range& x, const Range& y) { return x.b < y.b; });
  uintptr_t end_any = 0, end_written = 0;  // furthest end among the ranges that start before this one
  for (const Range& r : v) {
    ULTR_REQUIRE(r.b >= (r.written ? end_any : end_written), ULTR_EINVAL,
                 "%s: memory of tensor %d overlaps memory that the list writes", who, r.tensor);
    end_any = std::max(end_any, r.e);
    if (r.written) end_written = std::max(end_written, r.e);
  }
  return ULTR_OK;
}

// The first chunk of those, counted from the end of the list, that hold kCacheBytes of gradients.
static long long keep_from(const UltrTensor* t, int n, long long n_chunks) {
  long long left = kCacheBytes, chunk = n_chunks;
  for (int i = n - 1; i >= 0; --i) {
    const long long each = (long long)kChunk * dtype_bytes(t[i].grad_dtype), count = cdiv(t[i].n, kChunk);
    if (count * each > left) return chunk - left / each;
    left -= t[i].n * dtype_bytes(t[i].grad_dtype);
    chunk -= count;
  }
  return 0;
}

static int check_plan(const char* who, const UltrTensorPlan* p, int need, float clip_norm) {
  ULTR_REQUIRE(clip_norm == clip_norm, ULTR_EINVAL, "%s: clip_norm is not a number", who);
  ULTR_REQUIRE(p && p->table && p->n_chunks >= 0 && p->n_tensors >= 0 && p->keep_from >= 0 && p->keep_from <= p->n_chunks, ULTR_EINVAL,
               "%s: bad plan", who);
  ULTR_REQUIRE((p->has & need) == need, ULTR_EINVAL, "%s: the list lacks%s%s%s", who, (need & ~p->has & 1) ? " out" : "",
               (need & ~p->has & 2) ? " param" : "", (need & ~p->has & 4) ? " accum" : "");
  return ULTR_OK;
}
static ListView view_of(const UltrTensorPlan* p) {
  char* b = static_cast<char*>(p->table);
  return ListView{reinterpret_cast<double*>(b), reinterpret_cast<float*>(b + kPartialBytes), reinterpret_cast<const ChunkRec*>(b + kHeadBytes), p->n_chunks, p->keep_from};
}
static int pass_blocks(long long n_chunks) { return (int)std::min<long long>(n_chunks, kTMaxBlocks); }

static int launch_sumsq_blocks(const ListView& l, int nb, const float* denom, float scale_const, float l2, hipStream_t s) {
  {
    ProfScope prof_("tensors_sumsq_kernel", s);
    hipLaunchKernelGGL(l.keep_from > 0 ? tensors_sumsq_kernel<true> : tensors_sumsq_kernel<false>, dim3(nb), dim3(kTThreads), 0, s, l, denom, scale_const, l2);
  }
  return check_launch("tensors_sumsq_kernel");
}
// First pass: partial sums and the scale into the table.  Returns their number (0 for a list without elements) or an error.
static int launch_sumsq(const ListView& l, const float* denom, float scale_const, float l2, hipStream_t s) {
  const int nb = pass_blocks(l.n_chunks);
  if (nb == 0) return 0;
  const int rc = launch_sumsq_blocks(l, nb, denom, scale_const, l2, s);
  return rc ? rc : nb;
}
// The scale alone, for an update that forms no norm: the first pass over no chunk at all.
static int launch_scale(ListView l, const float* denom, float scale_const, hipStream_t s) {
  l.n_chunks = l.keep_from = 0;
  return launch_sumsq_blocks(l, 1, denom, scale_const, 0.f, s);
}
static int launch_norm(const ListView& l, int n_partials, float* out_norm, hipStream_t s) {
  {
    ProfScope prof_("tensors_norm_kernel", s);
    hipLaunchKernelGGL(tensors_norm_kernel, dim3(1), dim3(kTThreads), 0, s, l.partials, n_partials, out_norm);
  }
  return check_launch("tensors_norm_kernel");
}

}  // namespace ultr

using namespace ultr;

extern "C" long long ultr_tensors_table_bytes(const UltrTensor* tensors_h, int n_tensors) {
  long long chunks = 0;
  if (check_list("ultr_tensors_table_bytes", tensors_h, n_tensors, &chunks) != ULTR_OK) return -1;
  return table_bytes_of(chunks);
}

extern "C" int ultr_tensors_plan(const UltrTensor* tensors_h, int n_tensors, void* table, long long table_bytes,
                                 UltrTensorPlan* plan_h, void* stream) {
  const char* who = "ultr_tensors_plan";
  ULTR_REQUIRE(plan_h && table, ULTR_EINVAL, "%s: null pointer", who);
  ULTR_REQUIRE(((uintptr_t)table & 15) == 0, ULTR_EINVAL, "%s: table must be 16-byte aligned", who);
  long long chunks = 0;
  int rc = check_list(who, tensors_h, n_tensors, &chunks);
  if (rc) return rc;
  ULTR_REQUIRE(table_bytes >= table_bytes_of(chunks), ULTR_EINVAL, "%s: table of %lld bytes, %lld needed", who, table_bytes,
               table_bytes_of(chunks));
  try {
    rc = check_overlap(who, tensors_h, n_tensors);
  } catch (const std::bad_alloc&) {
    set_error("%s: out of host memory", who);
    return ULTR_ELIMIT;
  }
  if (rc) return rc;
  int has = 7;
  ChunkRec* recs = reinterpret_cast<ChunkRec*>(static_cast<char*>(table) + kHeadBytes);
  long long chunk = 0;
  for (int t0 = 0; t0 < n_tensors; t0 += kFillTensors) {
    FillArgs a{};
    const int count = std::min(kFillTensors, n_tensors - t0);
    long long most = 0;
    for (int k = 0; k < count; ++k) {
      const UltrTensor& u = a.t[k] = tensors_h[t0 + k];
      a.first_chunk[k] = chunk;
      const long long c = cdiv(u.n, kChunk);
      chunk += c;
      most = std::max(most, c);
      if (u.n > 0) has &= (u.out ? 1 : 0) | (u.param ? 2 : 0) | (u.accum ? 4 : 0);
    }
    if (most == 0) continue;
    {
      ProfScope prof_("tensors_fill_kernel", as_stream(stream));
      hipLaunchKernelGGL(tensors_fill_kernel, dim3(count, (unsigned)std::min<long long>(cdiv(most, kTThreads), 64)), dim3(kTThreads),
                         0, as_stream(stream), a, recs);
    }
    rc = check_launch("tensors_fill_kernel");
    if (rc) return rc;
  }
  *plan_h = UltrTensorPlan{table, chunks, n_tensors, has, keep_from(tensors_h, n_tensors, chunks), 0, 0};
  for (int i = 0; i < n_tensors; ++i) {
    const UltrTensor& t = tensors_h[i];
    const long long g = dtype_bytes(t.grad_dtype);
    plan_h->clip_bytes += t.n * 2 * g;
    plan_h->update_bytes += t.n * (g + 8 + (t.accum ? 8 : 0) + (t.copy ? dtype_bytes(t.copy_dtype) : 0));
  }
  return ULTR_OK;
}

extern "C" int ultr_global_norm(const UltrTensorPlan* plan_h, const float* denom, float scale_const, float* out_norm,
                                void* stream) {
  int rc = check_plan("ultr_global_norm", plan_h, 0, 0.f);
  if (rc) return rc;
  ULTR_REQUIRE(out_norm, ULTR_EINVAL, "ultr_global_norm: null out_norm");
  const ListView l = view_of(plan_h);
  const int nb = launch_sumsq(l, denom, scale_const, 0.f, as_stream(stream));
  return nb < 0 ? nb : launch_norm(l, nb, out_norm, as_stream(stream));
}

extern "C" int ultr_clip_by_global_norm(const UltrTensorPlan* plan_h, const float* denom, float scale_const, float clip_norm,
                                        float* out_norm, void* stream) {
  int rc = check_plan("ultr_clip_by_global_norm", plan_h, 1, clip_norm);
  if (rc) return rc;
  const ListView l = view_of(plan_h);
  hipStream_t s = as_stream(stream);
  const int nb = launch_sumsq(l, denom, scale_const, 0.f, s);
  if (nb < 0) return nb;
  if (nb == 0) return out_norm ? launch_norm(l, 0, out_norm, s) : ULTR_OK;
  {
    ProfScope prof_("tensors_clip_kernel", s);
    hipLaunchKernelGGL(plan_h->clip_bytes > kCacheBytes ? tensors_clip_kernel<true> : tensors_clip_kernel<false>, dim3(nb), dim3(kTThreads), 0, s, l, nb, clip_norm, out_norm);
  }
  return check_launch("tensors_clip_kernel");
}

extern "C" int ultr_clip_adagrad_tensors(const UltrTensorPlan* plan_h, const float* denom, float scale_const, float l2,
                                         float clip_norm, float lr, int strategy, float* out_norm, void* stream) {
  const char* who = "ultr_clip_adagrad_tensors";
  ULTR_REQUIRE(strategy == ULTR_OPT_ADAGRAD || strategy == ULTR_OPT_SGD, ULTR_EINVAL, "%s: grad_strategy=%d", who, strategy);
  int rc = check_plan(who, plan_h, strategy == ULTR_OPT_ADAGRAD ? 6 : 2, clip_norm);
  if (rc) return rc;
  const ListView l = view_of(plan_h);
  hipStream_t s = as_stream(stream);
  int np = 0;
  if (clip_norm > 0.f || out_norm) {
    np = launch_sumsq(l, denom, scale_const, l2, s);
    if (np < 0) return np;
  }
  const int nb = pass_blocks(l.n_chunks);
  if (nb == 0) return out_norm ? launch_norm(l, 0, out_norm, s) : ULTR_OK;
  if (np == 0 && denom) {
    rc = launch_scale(l, denom, scale_const, s);
    if (rc) return rc;
  }
  {
    ProfScope prof_("tensors_update_kernel", s);
    hipLaunchKernelGGL(plan_h->update_bytes > kCacheBytes ? tensors_update_kernel<true> : tensors_update_kernel<false>, dim3(nb), dim3(kTThreads), 0, s, l, np, np > 0 || denom, scale_const, l2, clip_norm, lr,
                       strategy, out_norm);
  }
  return check_launch("tensors_update_kernel");
}
