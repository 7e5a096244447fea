// Global norm, clipping and the optimiser update over a list of separate tensors.
// Reference: tf.clip_by_global_norm + apply_gradients over the variable list, dla.py:237-255, ipw_rank.py:155-165.
//   e = scale * g (+ l2 * theta) ; norm = sqrt(sum e^2) ; f = clip / max(norm, clip) ; out = f e, or
//   acc += (f e)^2, theta -= lr f e / sqrt(acc).
// The norm is needed before the first output: two passes over the gradients, one launch each.
#include "storage.hpp"

#include <algorithm>
#include <new>
#include <vector>

namespace ultr {

constexpr int kTThreads = 256;
constexpr int kChunk = 4096;       // elements of one tensor that one workgroup takes at a time
constexpr int kTMaxBlocks = 2048;  // workgroups of a pass, and partial sums of a norm

struct TensorRec {  // UltrTensor as the kernels read it
  const void* grad;
  void* out;
  float* param;
  float* accum;
  void* copy;
  long long n;
  int grad_dtype, copy_dtype;
};
static_assert(sizeof(TensorRec) == sizeof(UltrTensor), "the table holds the caller's records");

// Table: records | chunk map (tensor, chunk within it) | partial sums of the norm.
struct TableLayout {
  long long map, partials, bytes;
};
static TableLayout table_layout(int n_tensors, long long n_chunks) {
  TableLayout t;
  t.map = (long long)n_tensors * sizeof(TensorRec);
  t.partials = (t.map + n_chunks * (long long)sizeof(uint2) + 15) / 16 * 16;
  t.bytes = t.partials + kTMaxBlocks * (long long)sizeof(double);
  return t;
}

struct ListView {
  const TensorRec* recs;
  const uint2* map;
  double* partials;
  long long n_chunks;
};

constexpr int kFillTensors = 48;  // records per fill launch: they travel as kernel arguments (3.5 KB)
struct FillArgs {
  TensorRec rec[kFillTensors];
  long long first_chunk[kFillTensors];
  int first_tensor, count;
};
__global__ void __launch_bounds__(kTThreads) tensors_fill_kernel(FillArgs a, TensorRec* recs, uint2* map) {
  for (int t = blockIdx.x; t < a.count; t += gridDim.x) {
    if (threadIdx.x == 0 && blockIdx.y == 0) recs[a.first_tensor + t] = a.rec[t];
    const long long chunks = (a.rec[t].n + kChunk - 1) / kChunk;
    for (long long c = (long long)blockIdx.y * blockDim.x + threadIdx.x; c < chunks; c += (long long)gridDim.y * blockDim.x)
      map[a.first_chunk[t] + c] = make_uint2((unsigned)(a.first_tensor + t), (unsigned)c);
  }
}

// Sum of one double per thread over the workgroup, fixed order; valid in every thread.
__device__ __forceinline__ double block_sum_f64(double v, double* red) {
#pragma unroll
  for (int m = 32; m >= 1; m >>= 1) v += __shfl_xor(v, m);
  __syncthreads();
  if ((threadIdx.x & 63) == 0) red[threadIdx.x >> 6] = v;
  __syncthreads();
  double s = 0.0;
  for (int w = 0; w < (int)(blockDim.x >> 6); ++w) s += red[w];
  return s;
}

__device__ __forceinline__ float load_elem(const void* p, int dtype, long long i) {
  if (dtype == ULTR_DTYPE_F32) return static_cast<const float*>(p)[i];
  if (dtype == ULTR_DTYPE_BF16) return to_f32(static_cast<const bf16_t*>(p)[i]);
  return to_f32(static_cast<const f16_t*>(p)[i]);
}
__device__ __forceinline__ void store_elem(void* p, int dtype, long long i, float v) {
  if (dtype == ULTR_DTYPE_F32) static_cast<float*>(p)[i] = v;
  else if (dtype == ULTR_DTYPE_BF16) static_cast<bf16_t*>(p)[i] = from_f32<bf16_t>(v);
  else static_cast<f16_t*>(p)[i] = from_f32<f16_t>(v);
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

__global__ void __launch_bounds__(kTThreads) tensors_sumsq_kernel(ListView l, const float* denom, float scale_const, float l2) {
  __shared__ double red[kTThreads / 64];
  const float sc = scale_of(denom, scale_const);
  double acc = 0.0;
  for (long long c = blockIdx.x; c < l.n_chunks; c += gridDim.x) {
    const uint2 m = l.map[c];
    const TensorRec& r = l.recs[m.x];
    const long long first = (long long)m.y * kChunk, last = min(first + kChunk, r.n);
    for (long long i = first + threadIdx.x; i < last; i += kTThreads) {
      float e = load_elem(r.grad, r.grad_dtype, i) * sc;
      if (l2 != 0.f) e = fmaf(l2, r.param[i], e);
      acc += (double)e * (double)e;
    }
  }
  acc = block_sum_f64(acc, red);
  if (threadIdx.x == 0) l.partials[blockIdx.x] = acc;
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

__global__ void __launch_bounds__(kTThreads) tensors_clip_kernel(ListView l, int n_partials, const float* denom,
                                                                 float scale_const, float clip_norm, float* out_norm) {
  __shared__ double red[kTThreads / 64];
  const float sc = scale_of(denom, scale_const);
  float norm;
  const float f = clip_factor(partials_sum(l.partials, n_partials, red), clip_norm, &norm);
  if (blockIdx.x == 0 && threadIdx.x == 0 && out_norm) out_norm[0] = norm;
  for (long long c = blockIdx.x; c < l.n_chunks; c += gridDim.x) {
    const uint2 m = l.map[c];
    const TensorRec& r = l.recs[m.x];
    const long long first = (long long)m.y * kChunk, last = min(first + kChunk, r.n);
    for (long long i = first + threadIdx.x; i < last; i += kTThreads)
      store_elem(r.out, r.grad_dtype, i, load_elem(r.grad, r.grad_dtype, i) * sc * f);
  }
}

__global__ void __launch_bounds__(kTThreads) tensors_update_kernel(ListView l, int n_partials, const float* denom,
                                                                   float scale_const, float l2, float clip_norm, float lr,
                                                                   int strategy, float* out_norm) {
  __shared__ double red[kTThreads / 64];
  const float sc = scale_of(denom, scale_const);
  float f = 1.f;
  if (n_partials > 0) {
    float norm;
    f = clip_factor(partials_sum(l.partials, n_partials, red), clip_norm, &norm);
    if (blockIdx.x == 0 && threadIdx.x == 0 && out_norm) out_norm[0] = norm;
  }
  for (long long c = blockIdx.x; c < l.n_chunks; c += gridDim.x) {
    const uint2 m = l.map[c];
    const TensorRec& r = l.recs[m.x];
    const long long first = (long long)m.y * kChunk, last = min(first + kChunk, r.n);
    for (long long i = first + threadIdx.x; i < last; i += kTThreads) {
      float t = r.param[i];
      const float e = fmaf(l2, t, load_elem(r.grad, r.grad_dtype, i) * sc) * f;
      if (strategy == ULTR_OPT_ADAGRAD) {
        const float a = fmaf(e, e, r.accum[i]);
        r.accum[i] = a;
        t -= lr * e / sqrtf(a);
      } else {
        t -= lr * e;
      }
      r.param[i] = t;
      if (r.copy) store_elem(r.copy, r.copy_dtype, i, t);
    }
  }
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

static int check_plan(const char* who, const UltrTensorPlan* p, int need) {
  ULTR_REQUIRE(p && p->table && p->n_chunks >= 0 && p->n_tensors >= 0, ULTR_EINVAL, "%s: bad plan", who);
  ULTR_REQUIRE((p->has & need) == need, ULTR_EINVAL, "%s: the list lacks%s%s%s", who, (need & ~p->has & 1) ? " out" : "",
               (need & ~p->has & 2) ? " param" : "", (need & ~p->has & 4) ? " accum" : "");
  return ULTR_OK;
}
static ListView view_of(const UltrTensorPlan* p) {
  const TableLayout t = table_layout(p->n_tensors, p->n_chunks);
  char* b = static_cast<char*>(p->table);
  return ListView{reinterpret_cast<TensorRec*>(b), reinterpret_cast<uint2*>(b + t.map), reinterpret_cast<double*>(b + t.partials), p->n_chunks};
}
static int pass_blocks(long long n_chunks) { return (int)std::min<long long>(n_chunks, kTMaxBlocks); }

// First pass: partial sums into the table.  Returns their number (0 for a list without elements) or an error.
static int launch_sumsq(const ListView& l, const float* denom, float scale_const, float l2, hipStream_t s) {
  const int nb = pass_blocks(l.n_chunks);
  if (nb == 0) return 0;
  {
    ProfScope prof_("tensors_sumsq_kernel", s);
    hipLaunchKernelGGL(tensors_sumsq_kernel, dim3(nb), dim3(kTThreads), 0, s, l, denom, scale_const, l2);
  }
  const int rc = check_launch("tensors_sumsq_kernel");
  return rc ? rc : nb;
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
  return table_layout(n_tensors, chunks).bytes;
}

extern "C" int ultr_tensors_plan(const UltrTensor* tensors_h, int n_tensors, void* table, long long table_bytes,
                                 UltrTensorPlan* plan_h, void* stream) {
  const char* who = "ultr_tensors_plan";
  ULTR_REQUIRE(plan_h && table, ULTR_EINVAL, "%s: null pointer", who);
  ULTR_REQUIRE(((uintptr_t)table & 15) == 0, ULTR_EINVAL, "%s: table must be 16-byte aligned", who);
  long long chunks = 0;
  int rc = check_list(who, tensors_h, n_tensors, &chunks);
  if (rc) return rc;
  const TableLayout lay = table_layout(n_tensors, chunks);
  ULTR_REQUIRE(table_bytes >= lay.bytes, ULTR_EINVAL, "%s: table of %lld bytes, %lld needed", who, table_bytes, lay.bytes);
  try {
    rc = check_overlap(who, tensors_h, n_tensors);
  } catch (const std::bad_alloc&) {
    set_error("%s: out of host memory", who);
    return ULTR_ELIMIT;
  }
  if (rc) return rc;
  int has = 7;
  char* base = static_cast<char*>(table);
  long long chunk = 0;
  for (int t0 = 0; t0 < n_tensors; t0 += kFillTensors) {
    FillArgs a{};
    a.first_tensor = t0;
    a.count = std::min(kFillTensors, n_tensors - t0);
    long long most = 1;
    for (int k = 0; k < a.count; ++k) {
      const UltrTensor& u = tensors_h[t0 + k];
      a.rec[k] = TensorRec{u.grad, u.out, u.param, u.accum, u.copy, u.n, u.grad_dtype, u.copy_dtype};
      a.first_chunk[k] = chunk;
      const long long c = (u.n + kChunk - 1) / kChunk;
      chunk += c;
      most = std::max(most, c);
      if (u.n > 0) has &= (u.out ? 1 : 0) | (u.param ? 2 : 0) | (u.accum ? 4 : 0);
    }
    const int gy = (int)std::min<long long>(cdiv(most, kTThreads), 64);
    {
      ProfScope prof_("tensors_fill_kernel", as_stream(stream));
      hipLaunchKernelGGL(tensors_fill_kernel, dim3(a.count, gy), dim3(kTThreads), 0, as_stream(stream), a,
                         reinterpret_cast<TensorRec*>(base), reinterpret_cast<uint2*>(base + lay.map));
    }
    rc = check_launch("tensors_fill_kernel");
    if (rc) return rc;
  }
  *plan_h = UltrTensorPlan{table, chunks, n_tensors, has};
  return ULTR_OK;
}

extern "C" int ultr_global_norm(const UltrTensorPlan* plan_h, const float* denom, float scale_const, float* out_norm,
                                void* stream) {
  int rc = check_plan("ultr_global_norm", plan_h, 0);
  if (rc) return rc;
  ULTR_REQUIRE(out_norm, ULTR_EINVAL, "ultr_global_norm: null out_norm");
  const ListView l = view_of(plan_h);
  const int nb = launch_sumsq(l, denom, scale_const, 0.f, as_stream(stream));
  return nb < 0 ? nb : launch_norm(l, nb, out_norm, as_stream(stream));
}

extern "C" int ultr_clip_by_global_norm(const UltrTensorPlan* plan_h, const float* denom, float scale_const, float clip_norm,
                                        float* out_norm, void* stream) {
  int rc = check_plan("ultr_clip_by_global_norm", plan_h, 1);
  if (rc) return rc;
  const ListView l = view_of(plan_h);
  hipStream_t s = as_stream(stream);
  const int nb = launch_sumsq(l, denom, scale_const, 0.f, s);
  if (nb < 0) return nb;
  if (nb == 0) return out_norm ? launch_norm(l, 0, out_norm, s) : ULTR_OK;
  {
    ProfScope prof_("tensors_clip_kernel", s);
    hipLaunchKernelGGL(tensors_clip_kernel, dim3(nb), dim3(kTThreads), 0, s, l, nb, denom, scale_const, clip_norm, out_norm);
  }
  return check_launch("tensors_clip_kernel");
}

extern "C" int ultr_clip_adagrad_tensors(const UltrTensorPlan* plan_h, const float* denom, float scale_const, float l2,
                                         float clip_norm, float lr, int strategy, float* out_norm, void* stream) {
  const char* who = "ultr_clip_adagrad_tensors";
  ULTR_REQUIRE(strategy == ULTR_OPT_ADAGRAD || strategy == ULTR_OPT_SGD, ULTR_EINVAL, "%s: grad_strategy=%d", who, strategy);
  int rc = check_plan(who, plan_h, strategy == ULTR_OPT_ADAGRAD ? 6 : 2);
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
  {
    ProfScope prof_("tensors_update_kernel", s);
    hipLaunchKernelGGL(tensors_update_kernel, dim3(nb), dim3(kTThreads), 0, s, l, np, denom, scale_const, l2, clip_norm, lr,
                       strategy, out_norm);
  }
  return check_launch("tensors_update_kernel");
}
