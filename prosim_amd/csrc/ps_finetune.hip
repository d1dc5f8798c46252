// Operators of closed-loop fine-tuning: log-probability of a drawn choice, clipped policy loss with a KL term, pairwise preference loss,
// gradient clipping by the global norm (C ABI: include/prosim_hip.h, "Fine-tuning operators").  gfx950 only.
//
// All of them move bytes: ~10 operations per element against 2 - 8 B of HBM traffic, so what is designed for is one pass over the data.
// Statistics (sums of exponentials, log-probabilities, squares, losses) are held in 64 bits; only elements and stored results are narrower.
// No atomics: every sum has an order that depends on sizes alone, so equal inputs return equal bits.
#include "prosim_hip.h"

#include <hip/hip_runtime.h>

#include <cmath>
#include <tuple>
#include <type_traits>
#include <utility>

#include "ps_internal.h"

namespace {

using ps::set_error;

// ---- element types ---------------------------------------------------------------------------------------------------------
typedef _Float16 f16;
typedef __bf16 bf16;
template <typename T> __device__ __forceinline__ float to_f32(T v) { return (float)v; }
template <typename T> __device__ __forceinline__ T from_f32(float v) { return (T)v; }   // (round to nearest even, once per stored element)

// e^d for d <= 0.  fp32 elements take the library's expf (their results keep 24 bits); 16-bit elements v_exp_f32 on d * log2(e): the
// product's rounding is |d| 2^-24 relative, weighted by e^d <= 1, far under the 2^-9 / 2^-12 of the element's own type.
template <typename T> __device__ __forceinline__ float exp_of(float d) { return __builtin_amdgcn_exp2f(d * 1.44269504088896340736f); }
template <> __device__ __forceinline__ float exp_of<float>(float d) { return expf(d); }

// ---- block reductions (fixed order) ----------------------------------------------------------------------------------------
__device__ __forceinline__ double wave_sum(double v) {
  for (int o = 32; o; o >>= 1) v += __shfl_xor(v, o);
  return v;
}
__device__ __forceinline__ float wave_max(float v) {
  for (int o = 32; o; o >>= 1) v = fmaxf(v, __shfl_xor(v, o));
  return v;
}
// sum over the block, the same value in every thread; `s` holds one double per wave and may be reused after the call
template <int THREADS> __device__ __forceinline__ double block_sum(double v, double* s) {
  v = wave_sum(v);
  __syncthreads();
  if ((threadIdx.x & 63) == 0) s[threadIdx.x >> 6] = v;
  __syncthreads();
  double t = 0.0;
  for (int i = 0; i < THREADS / 64; ++i) t += s[i];
  return t;
}
template <int THREADS> __device__ __forceinline__ float block_max(float v, float* s) {
  v = wave_max(v);
  __syncthreads();
  if ((threadIdx.x & 63) == 0) s[threadIdx.x >> 6] = v;
  __syncthreads();
  float t = s[0];
  for (int i = 1; i < THREADS / 64; ++i) t = fmaxf(t, s[i]);
  return t;
}

// ---- rows of decisions -----------------------------------------------------------------------------------------------------
struct Rows {
  const void* x;          // [rows][stride], the first k of a row are its logits
  int64_t rows, k, stride;
  const void* choice;     // int32 or int64 per row
  const uint8_t* mask;    // per row, or NULL
  int choice64;
};
__device__ __forceinline__ int64_t choice_of(const Rows& r, int64_t i) {
  return r.choice64 ? ((const int64_t*)r.choice)[i] : (int64_t)((const int32_t*)r.choice)[i];
}

struct Policy {
  const float *old_logp, *advantage, *ref_logp;
  double lo, hi, beta, scale;     // clipping range [lo, hi] of the ratio
  const int64_t* count;           // valid rows (device), or NULL: all of them
  int mean;
};

// what one row contributes: filled by every thread that needs it from the row's statistics
struct RowLoss { double loss, kl, clip, d_logp; };
__device__ __forceinline__ RowLoss row_loss(const Policy& p, int64_t i, double logp) {
  RowLoss o;
  const double adv = p.advantage[i], r = exp(logp - (double)p.old_logp[i]);
  // (comparisons written so that a NaN ratio or advantage stays NaN: fmin / fmax would drop it)
  const double rc = r < p.lo ? p.lo : (r > p.hi ? p.hi : r);
  const double s1 = r * adv, s2 = rc * adv;
  const bool clipped = s2 < s1;
  o.loss = clipped ? -s2 : -s1;
  o.d_logp = clipped ? 0.0 : -s1;
  o.clip = clipped ? 1.0 : 0.0;
  o.kl = 0.0;
  if (p.ref_logp) {
    const double d = (double)p.ref_logp[i] - logp, em1 = expm1(d);
    o.kl = em1 - d;
    if (p.beta != 0.0) {
      o.loss += p.beta * o.kl;
      o.d_logp -= p.beta * em1;
    }
  }
  return o;
}
// scale / n of the loss: n = valid rows for the mean (an empty mask divides by 1: the sums are zero then), 1 for the sum
__device__ __forceinline__ double row_weight(const Policy& p, int64_t rows) {
  const int64_t n = p.mean ? (p.count ? *p.count : rows) : 1;
  return p.scale / (double)(n > 0 ? n : 1);
}

constexpr int LOGP = 0, POLICY = 1;
constexpr int kRowThreads = 256;
constexpr int kMaxGrid = 2048;        // row blocks of a launch (8 per CU); rows are dealt out in turn

// One block per row: maximum, sum of exponentials, then (GRAD) the gradient -- three passes over the row.
template <typename T, int MODE, bool GRAD>
__global__ void __launch_bounds__(kRowThreads) k_rows(Rows r, Policy p, float* logp_out, float2* stat, float* coef_out, T* dx, double* part) {
  __shared__ double sd[kRowThreads / 64];
  __shared__ float sf[kRowThreads / 64];
  double loss = 0.0, kl = 0.0, clip = 0.0;
  for (int64_t i = blockIdx.x; i < r.rows; i += gridDim.x) {
    const T* x = (const T*)r.x + i * r.stride;
    if (r.mask && !r.mask[i]) {     // (uniform over the block) a masked row is not read: its logits may hold anything
      if (threadIdx.x == 0) {
        logp_out[i] = 0.0f;
        if (stat) stat[i] = make_float2(0.0f, 0.0f);
        if (MODE == POLICY && coef_out) coef_out[i] = 0.0f;
      }
      if (GRAD)
        for (int64_t j = threadIdx.x; j < r.k; j += kRowThreads) dx[i * r.k + j] = from_f32<T>(0.0f);
      continue;
    }
    float m = -INFINITY;
    for (int64_t j = threadIdx.x; j < r.k; j += kRowThreads) m = fmaxf(m, to_f32(x[j]));
    m = block_max<kRowThreads>(m, sf);
    double s = 0.0;
    for (int64_t j = threadIdx.x; j < r.k; j += kRowThreads) s += (double)exp_of<T>(to_f32(x[j]) - m);
    s = block_sum<kRowThreads>(s, sd);
    const int64_t c = choice_of(r, i);
    const bool ok = c >= 0 && c < r.k;
    const double logp = ok ? ((double)to_f32(x[ok ? c : 0]) - (double)m) - log(s) : (double)NAN;
    const float inv = ok ? (float)(1.0 / s) : NAN;      // (a choice outside the row makes its gradient NaN too)
    if (threadIdx.x == 0) {
      logp_out[i] = (float)logp;
      if (stat) stat[i] = make_float2(m, inv);
    }
    if (MODE == POLICY) {
      const RowLoss o = row_loss(p, i, logp);
      const float coef = (float)(o.d_logp * row_weight(p, r.rows));
      if (threadIdx.x == 0) {
        loss += o.loss;
        kl += o.kl;
        clip += o.clip;
        if (coef_out) coef_out[i] = coef;
      }
      if (GRAD)
        for (int64_t j = threadIdx.x; j < r.k; j += kRowThreads)
          dx[i * r.k + j] = from_f32<T>(coef * ((j == c ? 1.0f : 0.0f) - exp_of<T>(to_f32(x[j]) - m) * inv));
    }
  }
  if (MODE == POLICY && threadIdx.x == 0) {
    part[blockIdx.x * 3 + 0] = loss;
    part[blockIdx.x * 3 + 1] = kl;
    part[blockIdx.x * 3 + 2] = clip;
  }
}

// dx = gain * coef (one-hot - p) from the stored statistics (m, 1 / s).  skip_one: dx already holds the result for gain 1.
template <typename T>
__global__ void __launch_bounds__(kRowThreads) k_rows_grad(Rows r, const float* coef_in, const float2* stat, const float* gain, int skip_one, T* dx) {
  const float g = gain ? *gain : 1.0f;
  if (skip_one && g == 1.0f) return;
  for (int64_t i = blockIdx.x; i < r.rows; i += gridDim.x) {
    const T* x = (const T*)r.x + i * r.stride;
    const float coef = r.mask && !r.mask[i] ? 0.0f : coef_in[i] * g;
    const float2 st = stat[i];
    const int64_t c = choice_of(r, i);
    for (int64_t j = threadIdx.x; j < r.k; j += kRowThreads)
      dx[i * r.k + j] = from_f32<T>(coef == 0.0f ? 0.0f : coef * ((j == c ? 1.0f : 0.0f) - exp_of<T>(to_f32(x[j]) - st.x) * st.y));
  }
}

__global__ void __launch_bounds__(1024) k_count(const uint8_t* mask, int64_t n, int64_t* out) {
  __shared__ double sd[16];
  int64_t c = 0;
  for (int64_t i = threadIdx.x; i < n; i += 1024) c += mask[i] != 0;
  const double t = block_sum<1024>((double)c, sd);     // (counts below 2^53 are exact)
  if (threadIdx.x == 0) *out = (int64_t)t;
}

// loss, mean kl, clipped share from the blocks' partial sums
__global__ void __launch_bounds__(256) k_policy_finish(Policy p, int64_t rows, const double* part, int blocks, float* loss, float* kl, float* clip_frac) {
  __shared__ double sd[4];
  double v[3] = {0.0, 0.0, 0.0};
  for (int b = threadIdx.x; b < blocks; b += 256)
    for (int q = 0; q < 3; ++q) v[q] += part[b * 3 + q];
  for (int q = 0; q < 3; ++q) v[q] = block_sum<256>(v[q], sd);
  if (threadIdx.x == 0) {
    const int64_t n = p.count ? *p.count : rows;
    const double inv = 1.0 / (double)(n > 0 ? n : 1);
    *loss = (float)(v[0] * row_weight(p, rows));
    *kl = (float)(v[1] * inv);
    *clip_frac = (float)(v[2] * inv);
  }
}

// ---- preference pairs ------------------------------------------------------------------------------------------------------
struct Side { const float *logp, *ref; const uint8_t* mask; int64_t steps; };
__device__ __forceinline__ double side_sum(const Side& s, int64_t p) {
  double v = 0.0;
  for (int64_t t = threadIdx.x; t < s.steps; t += 256) {
    const int64_t j = p * s.steps + t;
    if (s.mask && !s.mask[j]) continue;
    v += (double)s.logp[j] - (s.ref ? (double)s.ref[j] : 0.0);
  }
  return v;
}
__global__ void __launch_bounds__(256) k_pairs(Side w, Side l, int64_t pairs, double beta, double eps, double scale, float* margin, float* coef, double* part) {
  __shared__ double sd[4];
  double loss = 0.0;
  for (int64_t p = blockIdx.x; p < pairs; p += gridDim.x) {
    const double h = block_sum<256>(side_sum(w, p) - side_sum(l, p), sd);
    if (threadIdx.x == 0) {
      const double z = beta * h, e = exp(-fabs(z)), lp = log1p(e);
      const double neg = (z < 0.0 ? -z : 0.0) + lp, pos = (z > 0.0 ? z : 0.0) + lp;      // -ln sigmoid(z), -ln sigmoid(-z)
      const double down = z >= 0.0 ? e / (1.0 + e) : 1.0 / (1.0 + e), up = z >= 0.0 ? 1.0 / (1.0 + e) : e / (1.0 + e);   // sigmoid(-z), sigmoid(z)
      margin[p] = (float)z;
      coef[p] = (float)(scale * beta * (eps * up - (1.0 - eps) * down));
      loss += z != z ? z : (1.0 - eps) * neg + eps * pos;
    }
  }
  if (threadIdx.x == 0) part[blockIdx.x] = loss;
}
__global__ void __launch_bounds__(256) k_pairs_finish(const double* part, int blocks, double scale, float* out) {
  __shared__ double sd[4];
  double v = 0.0;
  for (int b = threadIdx.x; b < blocks; b += 256) v += part[b];
  v = block_sum<256>(v, sd);
  if (threadIdx.x == 0) *out = (float)(v * scale);
}
__global__ void __launch_bounds__(256) k_pairs_grad(const float* coef, const float* gain, const uint8_t* mask, int64_t pairs, int64_t steps, float sign, float* out) {
  const float g = sign * *gain;
  for (int64_t j = blockIdx.x * 256 + threadIdx.x; j < pairs * steps; j += (int64_t)gridDim.x * 256)
    out[j] = mask && !mask[j] ? 0.0f : coef[j / steps] * g;
}

// ---- gradient lists --------------------------------------------------------------------------------------------------------
constexpr int kClipSlots = 240;          // tensors of a launch: the table travels in the kernel's arguments (under 4 KB), no copy to wait for
constexpr int64_t kClipChunk = 32768;    // elements of a block
struct ClipTable {
  void* ptr[kClipSlots];
  uint32_t numel[kClipSlots];
  int32_t first[kClipSlots];             // first block of the tensor
  int n, block0;                         // block0: index of the launch's first block among the partial sums
};
__device__ __forceinline__ int clip_slot(const ClipTable& t, int b) {
  int lo = 0, hi = t.n - 1;
  while (lo < hi) {
    const int mid = (lo + hi + 1) >> 1;
    if (t.first[mid] <= b) lo = mid; else hi = mid - 1;
  }
  return lo;
}
template <typename T> __global__ void __launch_bounds__(256) k_clip_norm(ClipTable t, double* part) {
  __shared__ double sd[4];
  const int s = clip_slot(t, blockIdx.x);
  const int64_t a = (int64_t)(blockIdx.x - t.first[s]) * kClipChunk, e = min(a + kClipChunk, (int64_t)t.numel[s]);
  const T* g = (const T*)t.ptr[s];
  double v = 0.0;
  for (int64_t j = a + threadIdx.x; j < e; j += 256) {
    const double d = (double)to_f32(g[j]);
    v += d * d;
  }
  v = block_sum<256>(v, sd);
  if (threadIdx.x == 0) part[t.block0 + blockIdx.x] = v;
}
__global__ void __launch_bounds__(1024) k_clip_finish(const double* part, int64_t blocks, double max_norm, double eps, float* norm, float* coef) {
  __shared__ double sd[16];
  double v = 0.0;
  for (int64_t b = threadIdx.x; b < blocks; b += 1024) v += part[b];
  v = block_sum<1024>(v, sd);
  if (threadIdx.x == 0) {
    const double n = sqrt(v), c = isinf(max_norm) ? 1.0 : max_norm / (n + eps);
    *norm = (float)n;
    *coef = c >= 1.0 ? 1.0f : (float)c;       // (a NaN norm makes NaN gradients)
  }
}
template <typename T> __global__ void __launch_bounds__(256) k_clip_scale(ClipTable t, const float* coef) {
  const float c = *coef;
  if (c == 1.0f) return;
  const int s = clip_slot(t, blockIdx.x);
  const int64_t a = (int64_t)(blockIdx.x - t.first[s]) * kClipChunk, e = min(a + kClipChunk, (int64_t)t.numel[s]);
  T* g = (T*)t.ptr[s];
  for (int64_t j = a + threadIdx.x; j < e; j += 256) g[j] = from_f32<T>(to_f32(g[j]) * c);
}

// ---- host side -------------------------------------------------------------------------------------------------------------
// The launches of one entry: the first error ends it and is the entry's result (hipLaunchKernel's own return value -- hipGetLastError would
// also report, and clear, what an earlier call of somebody else's left).
struct Launches {
  hipStream_t stream;
  hipError_t err = hipSuccess;
  template <typename... P, size_t... I> void go(void (*k)(P...), int grid, int threads, std::tuple<P...> args, std::index_sequence<I...>) {
    void* ptr[] = {(void*)&std::get<I>(args)...};
    if (err == hipSuccess) err = hipLaunchKernel((const void*)k, dim3(grid), dim3(threads), ptr, 0, stream);
  }
  template <typename... P, typename... A> void operator()(void (*k)(P...), int grid, int threads, A... a) {
    go(k, grid, threads, std::tuple<P...>(a...), std::index_sequence_for<P...>{});
  }
  int result(const char* what) const { return err == hipSuccess ? PS_OK : set_error(PS_E_HIP, "%s: %s", what, hipGetErrorString(err)); }
};
int row_grid(int64_t rows) { return (int)(rows < kMaxGrid ? rows : kMaxGrid); }

int check_rows(const ps_decisions* d, const char* what, Rows* r) {
  if (!d) return set_error(PS_E_ARG, "%s: no decisions", what);
  if (d->rows < 0 || d->choices < 1 || d->choices > (1LL << 31) - 1 || d->rows > (1LL << 40)) return set_error(PS_E_ARG, "%s: rows must be >= 0 and choices in [1, 2^31)", what);
  if (d->row_stride < d->choices && d->rows > 1) return set_error(PS_E_ARG, "%s: row_stride < choices", what);
  if (d->dtype != PS_F32 && d->dtype != PS_BF16 && d->dtype != PS_F16) return set_error(PS_E_ARG, "%s: unknown element type", what);
  if (d->choice_bits != 32 && d->choice_bits != 64) return set_error(PS_E_ARG, "%s: choice_bits must be 32 or 64", what);
  if (d->rows && (!d->logits || !d->choice)) return set_error(PS_E_ARG, "%s: NULL logits or choice", what);
  *r = Rows{d->logits, d->rows, d->choices, d->row_stride, d->choice, d->mask, d->choice_bits == 64};
  return PS_OK;
}

template <typename F> int by_type(int dtype, F f) {
  return dtype == PS_F32 ? f((float*)nullptr) : dtype == PS_BF16 ? f((bf16*)nullptr) : f((f16*)nullptr);
}

struct LossSpace { int64_t* count; double* part; };
constexpr int64_t kLossSpace = 8 + 24 * (int64_t)kMaxGrid;
}  // namespace

extern "C" int64_t ps_policy_loss_workspace(const ps_decisions*) { return kLossSpace; }

extern "C" int ps_choice_logp(const ps_decisions* d, float* logp, float* stat, void* stream) {
  Rows r;
  if (int e = check_rows(d, "ps_choice_logp", &r)) return e;
  if (!r.rows) return PS_OK;
  if (!logp) return set_error(PS_E_ARG, "ps_choice_logp: NULL logp");
  Launches run{(hipStream_t)stream};
  by_type(d->dtype, [&](auto* t) {
    typedef std::remove_pointer_t<decltype(t)> T;
    run(k_rows<T, LOGP, false>, row_grid(r.rows), kRowThreads, r, Policy{}, logp, (float2*)stat, nullptr, nullptr, nullptr);
    return 0;
  });
  return run.result("ps_choice_logp");
}

extern "C" int ps_choice_grad(const ps_decisions* d, const float* coef, const float* stat, const float* gain, int32_t skip_if_one, void* grad, void* stream) {
  Rows r;
  if (int e = check_rows(d, "ps_choice_grad", &r)) return e;
  if (!r.rows) return PS_OK;
  if (!coef || !stat || !grad) return set_error(PS_E_ARG, "ps_choice_grad: NULL coef, stat or grad");
  Launches run{(hipStream_t)stream};
  by_type(d->dtype, [&](auto* t) {
    typedef std::remove_pointer_t<decltype(t)> T;
    run(k_rows_grad<T>, row_grid(r.rows), kRowThreads, r, coef, (const float2*)stat, gain, skip_if_one, (T*)grad);
    return 0;
  });
  return run.result("ps_choice_grad");
}

extern "C" int ps_policy_loss(const ps_decisions* d, const ps_policy_terms* q, float* loss, float* kl, float* clip_frac, float* logp, float* stat,
                              float* coef, void* grad, void* workspace, int64_t workspace_bytes, void* stream) {
  Rows r;
  if (int e = check_rows(d, "ps_policy_loss", &r)) return e;
  if (!q || !loss || !kl || !clip_frac || (r.rows && (!q->old_logp || !q->advantage || !logp))) return set_error(PS_E_ARG, "ps_policy_loss: NULL terms, loss, kl, clip_frac, old_logp, advantage or logp");
  if (!(q->clip_low >= 0.0 && q->clip_low <= 1.0) || !(q->clip_high >= 0.0)) return set_error(PS_E_ARG, "ps_policy_loss: clip_low must be in [0, 1] and clip_high >= 0");
  if (!(q->kl_coef >= 0.0) || std::isinf(q->kl_coef)) return set_error(PS_E_ARG, "ps_policy_loss: kl_coef must be >= 0 and finite");
  if (!std::isfinite(q->scale)) return set_error(PS_E_ARG, "ps_policy_loss: scale must be finite");
  if (q->kl_coef > 0.0 && !q->ref_logp && r.rows) return set_error(PS_E_ARG, "ps_policy_loss: kl_coef without ref_logp");
  if (!workspace || workspace_bytes < kLossSpace || ((uintptr_t)workspace & 7)) return set_error(PS_E_ARG, "ps_policy_loss: workspace missing, unaligned or smaller than ps_policy_loss_workspace()");
  Launches run{(hipStream_t)stream};
  LossSpace w{(int64_t*)workspace, (double*)workspace + 1};
  Policy p{q->old_logp, q->advantage, q->ref_logp, 1.0 - q->clip_low, 1.0 + q->clip_high, q->kl_coef, q->scale, r.mask ? w.count : nullptr, q->mean};
  const int grid = r.rows ? row_grid(r.rows) : 0;
  if (r.mask) run(k_count, 1, 1024, r.mask, r.rows, w.count);
  if (grid)
    by_type(d->dtype, [&](auto* t) {
      typedef std::remove_pointer_t<decltype(t)> T;
      if (grad) run(k_rows<T, POLICY, true>, grid, kRowThreads, r, p, logp, (float2*)stat, coef, (T*)grad, w.part);
      else run(k_rows<T, POLICY, false>, grid, kRowThreads, r, p, logp, (float2*)stat, coef, (T*)nullptr, w.part);
      return 0;
    });
  run(k_policy_finish, 1, 256, p, r.rows, w.part, grid, loss, kl, clip_frac);
  return run.result("ps_policy_loss");
}

extern "C" int64_t ps_preference_loss_workspace(int64_t) { return 8 * (int64_t)kMaxGrid; }

extern "C" int ps_preference_loss(const ps_preference* q, float* loss, float* margin, float* coef, void* workspace, int64_t workspace_bytes, void* stream) {
  if (!q || q->pairs < 1 || q->better_steps < 0 || q->worse_steps < 0) return set_error(PS_E_ARG, "ps_preference_loss: pairs must be >= 1 and steps >= 0");
  if ((q->better_steps && !q->better) || (q->worse_steps && !q->worse) || !loss || !margin || !coef) return set_error(PS_E_ARG, "ps_preference_loss: NULL better, worse, loss, margin or coef");
  if (!std::isfinite(q->beta) || !(q->label_smoothing >= 0.0 && q->label_smoothing <= 1.0) || !std::isfinite(q->scale)) return set_error(PS_E_ARG, "ps_preference_loss: beta and scale must be finite, label_smoothing in [0, 1]");
  if (!workspace || workspace_bytes < ps_preference_loss_workspace(q->pairs) || ((uintptr_t)workspace & 7)) return set_error(PS_E_ARG, "ps_preference_loss: workspace missing, unaligned or smaller than ps_preference_loss_workspace()");
  Launches run{(hipStream_t)stream};
  const int grid = row_grid(q->pairs);
  const double scale = q->scale / (q->mean ? (double)q->pairs : 1.0);
  run(k_pairs, grid, 256, Side{q->better, q->better_ref, q->better_mask, q->better_steps}, Side{q->worse, q->worse_ref, q->worse_mask, q->worse_steps},
                                                 q->pairs, q->beta, q->label_smoothing, scale, margin, coef, (double*)workspace);
  run(k_pairs_finish, 1, 256, (const double*)workspace, grid, scale, loss);
  return run.result("ps_preference_loss");
}

extern "C" int ps_preference_grad(const ps_preference* q, const float* coef, const float* gain, float* better_grad, float* worse_grad, void* stream) {
  if (!q || q->pairs < 1 || q->better_steps < 0 || q->worse_steps < 0 || !coef || !gain) return set_error(PS_E_ARG, "ps_preference_grad: bad pairs, or NULL coef or gain");
  Launches run{(hipStream_t)stream};
  const int64_t nb = q->pairs * q->better_steps, nw = q->pairs * q->worse_steps;
  auto grid = [](int64_t n) { const int64_t b = (n + 255) / 256; return (int)(b < kMaxGrid ? b : kMaxGrid); };
  if (better_grad && nb) run(k_pairs_grad, grid(nb), 256, coef, gain, q->better_mask, q->pairs, q->better_steps, 1.0f, better_grad);
  if (worse_grad && nw) run(k_pairs_grad, grid(nw), 256, coef, gain, q->worse_mask, q->pairs, q->worse_steps, -1.0f, worse_grad);
  return run.result("ps_preference_grad");
}

namespace {
int64_t clip_blocks(int64_t n) { return (n + kClipChunk - 1) / kClipChunk; }
constexpr int64_t kClipPiece = 1LL << 31;     // elements of a table entry (a longer tensor takes several)
int check_clip(const char* what, int32_t n, void* const* ptr, const int64_t* numel, const int32_t* dtype) {
  if (n < 0 || (n && (!ptr || !numel || !dtype))) return set_error(PS_E_ARG, "%s: NULL table", what);
  for (int32_t i = 0; i < n; ++i)
    if (numel[i] < 0 || (numel[i] && !ptr[i]) || (dtype[i] != PS_F32 && dtype[i] != PS_BF16 && dtype[i] != PS_F16) || ((uintptr_t)ptr[i] & (dtype[i] == PS_F32 ? 3 : 1)))
      return set_error(PS_E_ARG, "%s: tensor %d has a negative size, a NULL or unaligned pointer or an unknown element type", what, (int)i);
  return PS_OK;
}
// fill one table after the other, each of one element type, and launch it
template <typename F> void clip_tables(int32_t n, void* const* ptr, const int64_t* numel, const int32_t* dtype, F launch) {
  ClipTable t;
  int64_t block0 = 0;
  for (int ty : {PS_F32, PS_BF16, PS_F16}) {
    const int64_t size = ty == PS_F32 ? 4 : 2;
    int blocks = 0;
    t.n = 0;
    for (int32_t i = 0; i <= n; ++i) {
      if (i < n && (dtype[i] != ty || !numel[i])) continue;
      for (int64_t a = 0; i == n || a < numel[i]; a += kClipPiece) {
        if (t.n && (i == n || t.n == kClipSlots || blocks > (1 << 21))) {
          t.block0 = (int)block0;
          launch(t, blocks, ty);
          block0 += blocks;
          blocks = 0;
          t.n = 0;
        }
        if (i == n) break;
        const int64_t len = numel[i] - a < kClipPiece ? numel[i] - a : kClipPiece;
        t.ptr[t.n] = (char*)ptr[i] + a * size;
        t.numel[t.n] = (uint32_t)len;
        t.first[t.n++] = blocks;
        blocks += (int)clip_blocks(len);
      }
    }
  }
}
}  // namespace

extern "C" int64_t ps_clip_grads_workspace(int32_t n, const int64_t* numel) {
  int64_t b = 0;
  for (int32_t i = 0; i < n; ++i) b += clip_blocks(numel[i] > 0 ? numel[i] : 0);
  return 8 * (b + 1);
}

extern "C" int ps_clip_grads(int32_t n, void* const* ptr, const int64_t* numel, const int32_t* dtype, double max_norm, double eps, float* norm,
                             void* workspace, int64_t workspace_bytes, void* stream) {
  if (int e = check_clip("ps_clip_grads", n, ptr, numel, dtype)) return e;
  if (!(max_norm >= 0.0) || !(eps >= 0.0) || std::isinf(eps)) return set_error(PS_E_ARG, "ps_clip_grads: max_norm must be >= 0, eps >= 0 and finite");
  if (!norm) return set_error(PS_E_ARG, "ps_clip_grads: NULL norm");
  const int64_t need = ps_clip_grads_workspace(n, numel);
  if (need > (1LL << 31)) return set_error(PS_E_ARG, "ps_clip_grads: more than 2^43 elements");
  if (!workspace || workspace_bytes < need || ((uintptr_t)workspace & 7)) return set_error(PS_E_ARG, "ps_clip_grads: workspace missing, unaligned or smaller than ps_clip_grads_workspace()");
  Launches run{(hipStream_t)stream};
  float* coef = (float*)workspace;
  double* part = (double*)workspace + 1;
  clip_tables(n, ptr, numel, dtype, [&](const ClipTable& t, int blocks, int ty) {
    by_type(ty, [&](auto* p) { run(k_clip_norm<std::remove_pointer_t<decltype(p)>>, blocks, 256, t, part); return 0; });
  });
  run(k_clip_finish, 1, 1024, part, need / 8 - 1, max_norm, eps, norm, coef);
  clip_tables(n, ptr, numel, dtype, [&](const ClipTable& t, int blocks, int ty) {
    by_type(ty, [&](auto* p) { run(k_clip_scale<std::remove_pointer_t<decltype(p)>>, blocks, 256, t, coef); return 0; });
  });
  return run.result("ps_clip_grads");
}
