// Operators of closed-loop fine-tuning: log-probability of a drawn choice, clipped policy loss with a KL term, pairwise preference loss,
// gradient clipping by the global norm (C ABI: include/prosim_hip.h, "Fine-tuning operators").  gfx950 only.
//
// All of them move bytes: ~10 operations per element against 2 - 8 B of HBM traffic, so what is designed for is one pass over the data.
// Statistics (sums of exponentials, log-probabilities, squares, losses) are held in 64 bits; only elements and stored results are narrower.
// No atomics: every sum has an order that depends on sizes, types and the alignment of addresses alone (a gradient list's on which tensors are neighbours
// as well), so a call repeats its bits.
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

// e^d for d <= 0.  fp32 elements take the library's expf (their results keep 24 bits); 16-bit elements v_exp_f32 on d * log2(e), the constant
// in two parts (in one, its error would move every term of a sum the same way), the small one first: behind the rounded product it is less than half a
// step and would be lost.  What is left is one rounding, |d| 2^-24 relative.
template <typename T> __device__ __forceinline__ float exp_of(float d) {
  return __builtin_amdgcn_exp2f(fmaf(d, 1.44269502e+0f, d * 1.92596299e-8f));
}
template <> __device__ __forceinline__ float exp_of<float>(float d) { return expf(d); }
// The same in long rows, element j of a 16-byte piece: the product with log2(e) is rounded once, by a constant whose error is 1.3e-8 below in seven elements
// and 6.9e-8 above in the eighth -- together 0.3e-8, so a sum over many carries none of it worth naming, and each element less than its rounding.
template <typename T> __device__ __forceinline__ float exp_of(float d, int j) {
  return sizeof(T) == 4 ? exp_of<T>(d) : __builtin_amdgcn_exp2f(d * (j == 0 ? 1.44269514e+0f : 1.44269502e+0f));
}

// s += N of them, each added in 64 bits: 32-bit partial sums lose as much as a result's own rounding where one element carries the row (log-probabilities of
// 8192 x 64 fp32: 4.3e-8 against 2.8e-8 rms in sums of four; 2048 x 131072 bf16: 3.5e-8 against 2.9e-8 even in pairs, which would save 2 % of its time, 7 % of 3001 x 50021 fp16).
template <typename T, int N, bool LONG> __device__ __forceinline__ void add_exp(double& s, const float* f, float base) {
#pragma unroll
  for (int j = 0; j < N; ++j) s += (double)(LONG ? exp_of<T>(f[j] - base, j) : exp_of<T>(f[j] - base));
}

// The few 64-bit functions a row needs at its end, to about 1e-11 relative -- far beyond what its sum of exponentials carries -- in a quarter of the
// library's instructions (a wave spends as long on the library's log, exp and expm1 as on 1500 elements) and without its 40 registers of constants.
// exp: a = n ln 2 + f, |f| <= 0.35, Taylor's series to f^10 / 10!.  NaN stays, overflow is inf, underflow 0.
__device__ __forceinline__ double exp64(double a) {
  a = a > 800.0 ? 800.0 : a;
  a = a < -800.0 ? -800.0 : a;
  const double n = rint(a * 1.4426950408889634);
  const double f = fma(n, -1.9082149292705877e-10, fma(n, -0.6931471803691238, a));      // ln 2 in two parts, the first with 21 zero bits behind
  double p = 1.0 / 3628800.0;
  p = fma(p, f, 1.0 / 362880.0);
  p = fma(p, f, 1.0 / 40320.0);
  p = fma(p, f, 1.0 / 5040.0);
  p = fma(p, f, 1.0 / 720.0);
  p = fma(p, f, 1.0 / 120.0);
  p = fma(p, f, 1.0 / 24.0);
  p = fma(p, f, 1.0 / 6.0);
  p = fma(p, f, 0.5);
  p = fma(p, f, 1.0);
  p = fma(p, f, 1.0);
  return ldexp(p, (int)n);
}
// ln s for a finite s >= 2^-100: y = the 32-bit logarithm, then one step with s e^-y = 1 + r, ln s = y + r - r^2 / 2 + r^3 / 3, |r| < 1e-5.
__device__ __forceinline__ double log64(double s) {
  const double y = (double)(__builtin_amdgcn_logf((float)s) * 0.693147180559945f);
  const double r = fma(s, exp64(-y), -1.0);
  return y + r * fma(r, fma(r, 1.0 / 3.0, -0.5), 1.0);
}

// ---- block reductions (fixed order) ----------------------------------------------------------------------------------------
// over groups of G neighbouring lanes (a power of two), every lane gets the result
template <int G = 64> __device__ __forceinline__ double wave_sum(double v) {
#pragma unroll
  for (int o = G / 2; o; o >>= 1) v += __shfl_xor(v, o);
  return v;
}
template <int G = 64> __device__ __forceinline__ float wave_max(float v) {
#pragma unroll
  for (int o = G / 2; o; o >>= 1) v = fmaxf(v, __shfl_xor(v, o));
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
// three at once (`s`: three doubles per wave)
template <int THREADS> __device__ __forceinline__ void block_sum3(double* v, double* s) {
  for (int q = 0; q < 3; ++q) v[q] = wave_sum(v[q]);
  __syncthreads();
  if ((threadIdx.x & 63) == 0)
    for (int q = 0; q < 3; ++q) s[(threadIdx.x >> 6) * 3 + q] = v[q];
  __syncthreads();
  for (int q = 0; q < 3; ++q) {
    v[q] = 0.0;
    for (int i = 0; i < THREADS / 64; ++i) v[q] += s[i * 3 + q];
  }
}
// sum of n numbers by one block, eight loads in flight per thread
template <int THREADS> __device__ __forceinline__ double long_sum(const double* part, int64_t n, int64_t stride) {
  double v = 0.0;
  for (int64_t b = threadIdx.x; b < n; b += 8 * THREADS) {
    double u[8];
#pragma unroll
    for (int q = 0; q < 8; ++q) u[q] = b + q * THREADS < n ? part[(b + q * THREADS) * stride] : 0.0;
#pragma unroll
    for (int q = 0; q < 8; ++q) v += u[q];
  }
  return v;
}

// ---- rows of decisions -----------------------------------------------------------------------------------------------------
struct Rows {
  const void* x;          // [rows][stride], the first k of a row are its logits
  int64_t rows, k, stride;
  const void* choice;     // int32 or int64 per row
  const uint8_t* mask;    // per row, or NULL
  int choice64;
};
// (no branch on the type: its arithmetic would wait for the load where it stands)
__device__ __forceinline__ int64_t choice_of(const Rows& r, int64_t i) {
  const int32_t* p = (const int32_t*)r.choice + (i << r.choice64);
  const int32_t low = p[0], high = p[r.choice64];
  return r.choice64 ? (int64_t)high << 32 | (uint32_t)low : (int64_t)low;
}

struct Policy {
  const float *old_logp, *advantage, *ref_logp;
  double lo, hi, beta, scale;     // clipping range [lo, hi] of the ratio
  const int64_t* count;           // valid rows (device), or NULL: all of them
  int mean;
};

// what one row contributes: filled by every thread that needs it from the row's statistics
struct RowLoss { double loss, kl, clip, d_logp; };
struct RowTerms { float old_logp, advantage, ref_logp; };      // (read with the row, long before they are needed)
__device__ __forceinline__ RowTerms terms_of(const Policy& p, int64_t i) { return RowTerms{p.old_logp[i], p.advantage[i], p.ref_logp ? p.ref_logp[i] : 0.0f}; }
__device__ __forceinline__ RowLoss row_loss(const Policy& p, const RowTerms& t, double logp) {
  RowLoss o;
  const double adv = t.advantage, r = exp64(logp - (double)t.old_logp);
  // (comparisons written so that a NaN ratio or advantage stays NaN: fmin / fmax would drop it)
  const double rc = r < p.lo ? p.lo : (r > p.hi ? p.hi : r);
  const double s1 = r * adv, s2 = rc * adv;
  const bool clipped = s2 < s1;
  o.loss = clipped ? -s2 : -s1;
  o.d_logp = clipped ? 0.0 : -s1;
  o.clip = clipped ? 1.0 : 0.0;
  o.kl = 0.0;
  if (p.ref_logp) {
    const double d = (double)t.ref_logp - logp, em1 = exp64(d) - 1.0;
    o.kl = em1 - d;
    if (p.beta != 0.0) {
      o.loss += p.beta * o.kl;
      o.d_logp -= p.beta * em1;
    }
  }
  return o;
}
constexpr int LOGP = 0, POLICY = 1;
constexpr int GRAD_NONE = 0, GRAD_KEPT = 1, GRAD_PAST = 2;      // no gradient; one that its reader may find in the caches; one larger than the caches, written past them
constexpr int kMaxGrid = 2048;        // row blocks of a launch (8 per CU); rows are dealt out in turn

// What a launch over rows reads and writes.
struct RowIo {
  Rows r;
  Policy p;
  float* logp;
  float2* stat;         // (maximum, 1 / sum) per row, or NULL
  float* coef;          // d loss / d logp per row, or NULL
  void* dx;             // gradient, dense, or NULL
  double* part;         // (loss, kl, clipped) per block
  float *loss, *kl, *clip_frac;
};

// 16 bytes of a row, kept packed in registers.  Rows of odd length start at any element: gfx950 loads and stores 16 bytes at element alignment.
template <typename T> struct Reg {
  static constexpr int N = 16 / sizeof(T);
  uint32_t w[4];
  typedef uint32_t Words __attribute__((ext_vector_type(4), aligned(1)));      // (element-aligned; the attribute takes no expression of T)
  __device__ __forceinline__ void load(const T* p) {
    const Words m = *(const Words*)p;
#pragma unroll
    for (int i = 0; i < 4; ++i) w[i] = m[i];
  }
  __device__ __forceinline__ void store(T* p) const {
    const Words m = {w[0], w[1], w[2], w[3]};
    *(Words*)p = m;
  }
  // the same past the caches, for what nobody reads again soon
  __device__ __forceinline__ void load_once(const T* p) {
    const Words m = __builtin_nontemporal_load((const Words*)p);
#pragma unroll
    for (int i = 0; i < 4; ++i) w[i] = m[i];
  }
  __device__ __forceinline__ void store_once(T* p) const {
    const Words m = {w[0], w[1], w[2], w[3]};
    __builtin_nontemporal_store(m, (Words*)p);
  }
  // the packed words are what lives from one use to the next: without this the compiler keeps the 32-bit elements of the first use (twice the
  // registers, 128 - 2000 B of scratch per lane in the widest kernels)
  __device__ __forceinline__ void forget() { asm volatile("" : "+v"(w[0]), "+v"(w[1]), "+v"(w[2]), "+v"(w[3])); }
  __device__ __forceinline__ float top(float m) const;      // max(m, the elements)
  __device__ __forceinline__ void get(float* f) const;
  __device__ __forceinline__ void set(const float* f);
};
template <> __device__ __forceinline__ void Reg<float>::get(float* f) const {
#pragma unroll
  for (int i = 0; i < 4; ++i) f[i] = __uint_as_float(w[i]);
}
template <> __device__ __forceinline__ void Reg<float>::set(const float* f) {
#pragma unroll
  for (int i = 0; i < 4; ++i) w[i] = __float_as_uint(f[i]);
}
template <> __device__ __forceinline__ void Reg<bf16>::get(float* f) const {
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    f[2 * i] = __uint_as_float(w[i] << 16);
    f[2 * i + 1] = __uint_as_float(w[i] & 0xffff0000u);
  }
}
template <typename T> __device__ __forceinline__ uint32_t pack2(float a, float b) {
  typedef T T2 __attribute__((ext_vector_type(2)));
  const T2 t = {from_f32<T>(a), from_f32<T>(b)};
  uint32_t u;
  __builtin_memcpy(&u, &t, 4);
  return u;
}
template <> __device__ __forceinline__ void Reg<bf16>::set(const float* f) {
#pragma unroll
  for (int i = 0; i < 4; ++i) w[i] = pack2<bf16>(f[2 * i], f[2 * i + 1]);
}
template <> __device__ __forceinline__ void Reg<f16>::get(float* f) const {
  typedef f16 h2 __attribute__((ext_vector_type(2)));
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    h2 h;
    __builtin_memcpy(&h, &w[i], 4);
    f[2 * i] = (float)h.x;
    f[2 * i + 1] = (float)h.y;
  }
}
template <> __device__ __forceinline__ void Reg<f16>::set(const float* f) {
#pragma unroll
  for (int i = 0; i < 4; ++i) w[i] = pack2<f16>(f[2 * i], f[2 * i + 1]);
}
// The running maximum: fp16 two elements at a time without unpacking them (6 operations a piece instead of 12; with one rounding of the exponent's product
// less this took 3001 x 50021 fp16 from 57 to 54 us: two blocks of 8 waves share a CU's registers there, and their arithmetic, about 50 cycles an element and
// SIMD, 16 of them the exponential, is not all hidden behind each other's loads).  A NaN may be taken or passed
// over; the row's sum has it either way.  A bf16 word must not stand for its upper element as it is: -inf with bits behind it is a signalling NaN, which
// v_max_f32 answers with a NaN; and packed integer maxima for both signs took 65 us instead of 63.
template <> __device__ __forceinline__ float Reg<float>::top(float m) const {
#pragma unroll
  for (int i = 0; i < 4; ++i) m = fmaxf(m, __uint_as_float(w[i]));
  return m;
}
template <> __device__ __forceinline__ float Reg<bf16>::top(float m) const {
#pragma unroll
  for (int i = 0; i < 4; ++i) m = fmaxf(fmaxf(m, __uint_as_float(w[i] << 16)), __uint_as_float(w[i] & 0xffff0000u));
  return m;
}
__device__ __forceinline__ uint32_t pk_max(uint32_t a, uint32_t b) {
  uint32_t m;
  asm("v_pk_max_f16 %0, %1, %2" : "=v"(m) : "v"(a), "v"(b));      // (the builtin quiets both operands first, three instructions for one)
  return m;
}
template <> __device__ __forceinline__ float Reg<f16>::top(float m) const {
  typedef f16 h2 __attribute__((ext_vector_type(2)));
  const uint32_t a = pk_max(pk_max(w[0], w[1]), pk_max(w[2], w[3]));
  h2 h;
  __builtin_memcpy(&h, &a, 4);
  return fmaxf(fmaxf(m, (float)h.x), (float)h.y);
}

// (maximum, sum of exponentials relative to it) of a part of a row.  A part of -inf alone keeps the maximum -inf and the sum 0.
struct Part { double s; float m; };
__device__ __forceinline__ float base_of(float m) { return m == -INFINITY ? 0.0f : m; }
// join the parts of a group of lanes (G a power of two); every lane gets the result
template <int G> __device__ __forceinline__ Part join_lanes(Part a) {
  const float m = wave_max<G>(a.m);
  const double s = a.s == 0.0 ? 0.0 : a.s * exp64((double)a.m - (double)m);      // (NaN sums stay NaN: NaN == 0 is false)
  return Part{wave_sum<G>(s), m};
}

__device__ __forceinline__ int nonzero_bytes(const Reg<uint8_t>& q) {
  int c = 0;
#pragma unroll
  for (int i = 0; i < 4; ++i)
#pragma unroll
    for (int b = 0; b < 32; b += 8) c += (q.w[i] >> b & 255u) != 0;
  return c;
}
// The valid rows the mean divides by, as scale / n; `count` is filled for the epilogue.  Called by the whole block.
template <int THREADS> __device__ __forceinline__ double weight_of(const RowIo& io, int64_t* count, double* sd) {
  const Policy& p = io.p;
  int64_t n = io.r.rows;
  if (io.r.mask) {
    if (p.count) {
      n = *p.count;
    } else {
      const uint8_t* mask = io.r.mask;
      int c = 0;
      const int64_t full = io.r.rows / 16;
      for (int64_t j = threadIdx.x; j < full; j += THREADS) {
        Reg<uint8_t> q;
        q.load(mask + j * 16);
        c += nonzero_bytes(q);
      }
      if (threadIdx.x < 16 && full * 16 + threadIdx.x < io.r.rows) c += mask[full * 16 + threadIdx.x] != 0;
      n = (int64_t)block_sum<THREADS>((double)c, sd);
    }
  }
  *count = n;
  return p.scale / (double)(p.mean && n > 0 ? n : 1);
}
// What a row's statistics make of it: log-probability, loss terms, the coefficient of its gradient.  Every lane of the row's group calls it.
struct RowEnd { float coef, inv; };
template <int MODE> __device__ __forceinline__ RowEnd end_row(const RowIo& io, int64_t i, const RowTerms& t, bool ok, float xc, Part a, double weight, bool writer, double* acc) {
  const double logp = ok ? ((double)xc - (double)a.m) - log64(a.s) : (double)NAN;
  RowEnd e;
  e.inv = ok ? 1.0f / (float)a.s : NAN;      // (a choice outside the row makes its gradient NaN too)
  e.coef = 0.0f;
  if (MODE == POLICY) {
    const RowLoss o = row_loss(io.p, t, logp);
    e.coef = (float)(o.d_logp * weight);
    if (writer) {
      acc[0] += o.loss;
      acc[1] += o.kl;
      acc[2] += o.clip;
    }
  }
  if (writer) {
    io.logp[i] = (float)logp;
    if (io.stat) io.stat[i] = make_float2(a.m, e.inv);
    if (MODE == POLICY && io.coef) io.coef[i] = e.coef;
  }
  return e;
}
__device__ __forceinline__ void masked_row(const RowIo& io, int64_t i) {
  io.logp[i] = 0.0f;
  if (io.stat) io.stat[i] = make_float2(0.0f, 0.0f);
  if (io.coef) io.coef[i] = 0.0f;
}
// the block's share of the sums -- or, where the launch is one block, the results themselves.  Where a block has one row, thread 0 has all of it (ONE).
template <int THREADS, bool ONE> __device__ __forceinline__ void end_block(const RowIo& io, int64_t block, double* v, int64_t count, double weight, double* sd) {
  if (!ONE) block_sum3<THREADS>(v, sd);
  if (threadIdx.x) return;
  if (gridDim.x > 1 || gridDim.y > 1) {
    for (int q = 0; q < 3; ++q) io.part[block * 3 + q] = v[q];
    return;
  }
  const double inv = 1.0 / (double)(count > 0 ? count : 1);
  *io.loss = (float)(v[0] * weight);
  *io.kl = (float)(v[1] * inv);
  *io.clip_frac = (float)(v[2] * inv);
}

// Short rows: G lanes hold a row, N elements each.
template <typename T, int G, int N, int MODE, int GRAD> __global__ void __launch_bounds__(256) k_rows_short(RowIo io) {
  __shared__ double sd[12];
  double acc[3] = {0.0, 0.0, 0.0}, weight = 1.0;
  int64_t count = 0;
  if (MODE == POLICY) weight = weight_of<256>(io, &count, sd);
  const Rows& r = io.r;
  const int lane = threadIdx.x & (G - 1), k = (int)r.k;
  for (int64_t i = (int64_t)blockIdx.x * (256 / G) + threadIdx.x / G; i < r.rows; i += (int64_t)gridDim.x * (256 / G)) {
    T* dx = GRAD ? (T*)io.dx + i * k : nullptr;
    if (r.mask && !r.mask[i]) {
      if (lane == 0) masked_row(io, i);
      if (GRAD)
#pragma unroll
        for (int q = 0; q < N; ++q)
          if (q * G + lane < k) dx[q * G + lane] = from_f32<T>(0.0f);
      continue;
    }
    const T* x = (const T*)r.x + i * r.stride;
    const int64_t c = choice_of(r, i);
    const bool ok = c >= 0 && c < k;
    const float xc = to_f32(x[ok ? c : 0]);
    const RowTerms terms = MODE == POLICY ? terms_of(io.p, i) : RowTerms{};
    float f[N];
    Part a{0.0, -INFINITY};
#pragma unroll
    for (int q = 0; q < N; ++q) {
      f[q] = q * G + lane < k ? to_f32(x[q * G + lane]) : -INFINITY;
      a.m = fmaxf(a.m, f[q]);
    }
    a.m = wave_max<G>(a.m);
    const float base = base_of(a.m);
#pragma unroll
    for (int q = 0; q < N; ++q) {
      f[q] = exp_of<T>(f[q] - base);
      a.s += (double)f[q];
    }
    a.s = wave_sum<G>(a.s);
    const RowEnd e = end_row<MODE>(io, i, terms, ok, xc, a, weight, lane == 0, acc);
    if (GRAD) {
      const float scale = -e.coef * e.inv;
#pragma unroll
      for (int q = 0; q < N; ++q)
        if (q * G + lane < k) dx[q * G + lane] = from_f32<T>(fmaf(f[q], scale, q * G + lane == c ? e.coef : 0.0f));
    }
  }
  if (MODE == POLICY) end_block<256, false>(io, blockIdx.x, acc, count, weight, sd);
}

// One 16-byte piece of a row's gradient, -coef e^(x - m) inv; the chosen element's share of coef is added behind it (chosen_element).  16-bit results
// take the factor into the exponent, |scale| e^d = 2^(d log2 e + log2 |scale|), and its sign afterwards: 6 instead of 8 operations an element beside the
// exponential, at most (|d| + |log2 scale|) 2^-23 relative, a few hundredths of their half step.
struct GradScale {
  float m, scale, log2_scale;
  uint32_t sign;
  __device__ __forceinline__ GradScale(float m_, float scale_) : m(m_), scale(scale_), log2_scale(__builtin_amdgcn_logf(fabsf(scale_))), sign(__float_as_uint(scale_) >> 31 ? 0x80008000u : 0u) {}
};
template <typename T> __device__ __forceinline__ void grad_piece(Reg<T>& v, const GradScale& s) {
  float f[Reg<T>::N];
  v.get(f);
  if (sizeof(T) == 4) {
#pragma unroll
    for (int i = 0; i < Reg<T>::N; ++i) f[i] = exp_of<T>(f[i] - s.m) * s.scale;
    v.set(f);
  } else {
#pragma unroll
    for (int i = 0; i < Reg<T>::N; ++i) f[i] = __builtin_amdgcn_exp2f(fmaf(f[i] - s.m, 1.44269502e+0f, s.log2_scale));
    v.set(f);
#pragma unroll
    for (int i = 0; i < 4; ++i) v.w[i] ^= s.sign;
  }
}
// How TPR threads share a stretch of `len` elements at p: whole 16-byte pieces from the first aligned address on, dealt out in turn, and the elements before
// and behind them (`edges` of them, a thread each).  Rows of odd length start anywhere; pieces at element alignment work on gfx950 too, but a wave's
// kilobyte then lies across nine cache lines instead of eight (3001 x 50021 fp16: 67 us, aligned 54 us).
template <typename T, int TPR> struct Shared {
  static constexpr int V = Reg<T>::N;
  static constexpr int ALIGN = TPR >= 128 ? 128 : TPR >= 16 ? TPR : sizeof(T) == 4 ? 16 : (int)sizeof(T);     // bytes; the edges have to fit the threads
  static_assert(ALIGN / (int)sizeof(T) + V - 2 <= TPR || ALIGN == (int)sizeof(T), "a thread per edge element");
  int head, pieces, edges;
  __device__ __forceinline__ Shared(const T* p, int64_t len) {
    const int lead = (int)(-(uintptr_t)p & (ALIGN - 1)) / (int)sizeof(T);
    head = lead < len ? lead : (int)len;
    pieces = (int)((len - head) / V);
    edges = (int)(len - (int64_t)pieces * V);
  }
  // column of thread t's edge element (t < edges)
  __device__ __forceinline__ int64_t edge(int t) const { return t < head ? t : (int64_t)pieces * V + t; }
  // the thread that writes column o
  __device__ __forceinline__ int owner(int64_t o) const {
    if (o < head) return (int)o;
    const int64_t q = (o - head) / V;
    return q < pieces ? (int)(q % TPR) : (int)(o - (int64_t)pieces * V);
  }
};
// The chosen element of a stretch (column o of it, outside for most stretches), written once more and whole by the thread that wrote its piece.
template <typename T, int TPR> __device__ __forceinline__ void chosen_element(T* dx, const Shared<T, TPR>& sh, int64_t len, int64_t o, int t, float xc, float m, float scale, float coef) {
  if (o >= 0 && o < len && t == sh.owner(o)) dx[o] = from_f32<T>(fmaf(exp_of<T>(xc - m), scale, coef));
}
template <typename T, int TPR> __device__ __forceinline__ void zero_row(T* dx, int64_t len, int t) {
  Reg<T> z;
  z.w[0] = z.w[1] = z.w[2] = z.w[3] = 0;
  const Shared<T, TPR> sh(dx, len);
  for (int q = t; q < sh.pieces; q += TPR) z.store(dx + sh.head + (int64_t)q * Reg<T>::N);
  if (t < sh.edges) dx[sh.edge(t)] = from_f32<T>(0.0f);
}

// Rows that fit the registers of TPR threads (8 .. 64 lanes of a wave, or that many waves of a block), NV 16-byte pieces per thread: one read of the
// row for its statistics and its gradient.  One row per group and no loop over rows: inside a loop the compiler would keep the 64-bit functions'
// constants in registers all the time.
template <typename T, int TPR, int NV, int MODE, int GRAD> __global__ void __launch_bounds__(TPR <= 64 ? 256 : TPR) k_rows_held(RowIo io) {
  constexpr int THREADS = TPR <= 64 ? 256 : TPR, WAVES = TPR <= 64 ? 1 : TPR / 64, LANES = TPR < 64 ? TPR : 64, V = Reg<T>::N;
  __shared__ double sd[3 * THREADS / 64];
  __shared__ Part joined[WAVES];
  const int64_t block = (int64_t)blockIdx.y * gridDim.x + blockIdx.x;
  if (block * (THREADS / TPR) >= io.r.rows) return;      // (the last line of a two-dimensional grid)
  double acc[3] = {0.0, 0.0, 0.0}, weight = 1.0;
  int64_t count = 0;
  if (MODE == POLICY) weight = weight_of<THREADS>(io, &count, sd);
  const Rows& r = io.r;
  const int t = threadIdx.x % TPR;
  // (where a wave has one row, its addresses live in scalar registers)
  const int64_t i = block * (THREADS / TPR) + (TPR < 64 ? (int)threadIdx.x / TPR : __builtin_amdgcn_readfirstlane(threadIdx.x / TPR));
  if (i < r.rows) {
    T* dx = GRAD ? (T*)io.dx + i * r.k : nullptr;
    const int64_t c = choice_of(r, i);        // (beside the mask's byte and before the row: the chosen logit's address waits for nothing else)
    if (r.mask && !r.mask[i]) {        // (the same for all of the row's threads)
      if (t == 0) masked_row(io, i);
      if (GRAD) zero_row<T, TPR>(dx, r.k, t);
    } else {
      const T* x = (const T*)r.x + i * r.stride;
      const Shared<T, TPR> sh(x, r.k);
      const int nv = sh.pieces;
      Reg<T> v[NV];
#pragma unroll
      for (int q = 0; q < NV; ++q)
        if (q * TPR + t < nv) v[q].load_once(x + sh.head + q * (TPR * V) + (uint32_t)(t * V));
      const T end = x[t < sh.edges ? sh.edge(t) : 0];      // (in every thread: converted where only some have one, it would wait for the whole row)
      const bool ok = c >= 0 && c < r.k;
      const float xc = to_f32(x[ok ? c : 0]);
      const RowTerms terms = MODE == POLICY ? terms_of(io.p, i) : RowTerms{};
      Part a{0.0, -INFINITY};
#pragma unroll
      for (int q = 0; q < NV; ++q)
        if (q * TPR + t < nv) a.m = v[q].top(a.m);
      const float last = t < sh.edges ? to_f32(end) : -INFINITY;
      a.m = wave_max<LANES>(fmaxf(a.m, last));
      const float base = base_of(a.m);
      a.s = (double)exp_of<T>(last - base);
#pragma unroll
      for (int q = 0; q < NV; ++q)
        if (q * TPR + t < nv) {
          float f[V];
          v[q].forget();
          v[q].get(f);
          add_exp<T, V, TPR >= 64>(a.s, f, base);
          __builtin_amdgcn_sched_barrier(0);
        }
      a.s = wave_sum<LANES>(a.s);
      if (WAVES > 1) {
        const int lane = threadIdx.x & 63;
        if (lane == 0) joined[threadIdx.x >> 6] = a;
        __syncthreads();
        a = joined[lane & (WAVES - 1)];
        a = join_lanes<WAVES>(a);
      }
      const RowEnd e = end_row<MODE>(io, i, terms, ok, xc, a, weight, t == 0, acc);
      if (GRAD) {
        const float scale = -e.coef * e.inv;
        const GradScale gs(a.m, scale);
#pragma unroll
        for (int q = 0; q < NV; ++q)
          if (q * TPR + t < nv) {
            v[q].forget();
            grad_piece<T>(v[q], gs);
            if (GRAD == GRAD_PAST) v[q].store_once(dx + sh.head + q * (TPR * V) + (uint32_t)(t * V));
            else v[q].store(dx + sh.head + q * (TPR * V) + (uint32_t)(t * V));
            __builtin_amdgcn_sched_barrier(0);
          }
        if (t < sh.edges) dx[sh.edge(t)] = from_f32<T>(exp_of<T>(last - a.m) * scale);
        chosen_element<T, TPR>(dx, sh, r.k, c, t, xc, a.m, scale, e.coef);
      }
    }
  }
  if (MODE == POLICY) end_block<THREADS, (TPR > 64)>(io, block, acc, count, weight, sd);
}

// (maximum, sum) of the elements [j0, j1) of a row by one block, in one pass, four pieces in flight per thread: every thread keeps its running maximum
// and rescales its sum when it grows.  THREADS a power of two of waves.
template <typename T, int THREADS> __device__ __forceinline__ Part stream_part(const T* x, int64_t j0, int64_t j1, Part* slots) {
  constexpr int V = Reg<T>::N, U = 4;
  Part a{0.0, -INFINITY};
  x += j0;
  const Shared<T, THREADS> sh(x, j1 - j0);
  const int n = sh.pieces;
  auto raise = [&](float m) {
    if (m > a.m) {
      if (a.s != 0.0) a.s *= (double)exp_of<T>(a.m - m);      // (nothing yet, or -inf alone: 0 stays 0)
      a.m = m;
    }
  };
  for (int q = threadIdx.x; q < n; q += U * THREADS) {
    Reg<T> v[U];
#pragma unroll
    for (int u = 0; u < U; ++u)
      if (q + u * THREADS < n) v[u].load_once(x + sh.head + (int64_t)(q + u * THREADS) * V);
    float m = -INFINITY;
#pragma unroll
    for (int u = 0; u < U; ++u)
      if (q + u * THREADS < n) m = v[u].top(m);
    raise(m);
    const float base = base_of(a.m);
#pragma unroll
    for (int u = 0; u < U; ++u)
      if (q + u * THREADS < n) {
        float f[V];
        v[u].forget();
        v[u].get(f);
        add_exp<T, V, true>(a.s, f, base);
      }
  }
  if ((int)threadIdx.x < sh.edges) {
    const float f = to_f32(x[sh.edge(threadIdx.x)]);
    raise(f);
    a.s += (double)exp_of<T>(f - base_of(a.m));
  }
  a = join_lanes<64>(a);
  __syncthreads();
  if ((threadIdx.x & 63) == 0) slots[threadIdx.x >> 6] = a;
  __syncthreads();
  a = slots[threadIdx.x & (THREADS / 64 - 1)];
  return join_lanes<THREADS / 64>(a);
}
template <typename T, int THREADS> __device__ __forceinline__ void stream_grad(const T* x, T* dx, int64_t j0, int64_t j1, float m, float scale, float coef, int64_t c, float xc) {
  x += j0;
  dx += j0;
  const Shared<T, THREADS> sh(x, j1 - j0);
  const GradScale gs(m, scale);
  for (int q = threadIdx.x; q < sh.pieces; q += THREADS) {
    Reg<T> v;
    v.load_once(x + sh.head + (int64_t)q * Reg<T>::N);
    grad_piece<T>(v, gs);
    v.store(dx + sh.head + (int64_t)q * Reg<T>::N);
  }
  if ((int)threadIdx.x < sh.edges) {
    const int64_t j = sh.edge(threadIdx.x);
    dx[j] = from_f32<T>(exp_of<T>(to_f32(x[j]) - m) * scale);
  }
  chosen_element<T, THREADS>(dx, sh, j1 - j0, c - j0, threadIdx.x, xc, m, scale, coef);
}

// Rows that no block holds, or few and long: `splits` blocks share a row (at most 64), `step` elements each.  First launch: the blocks' (maximum, sum) ...
template <typename T> __global__ void __launch_bounds__(256) k_split_part(Rows r, int splits, int64_t step, Part* out) {
  __shared__ Part slots[4];
  const int64_t b = (int64_t)blockIdx.y * gridDim.x + blockIdx.x, i = b / splits, j0 = (b - i * splits) * step;
  if (i >= r.rows || (r.mask && !r.mask[i])) return;
  const Part a = stream_part<T, 256>((const T*)r.x + i * r.stride, j0, min(j0 + step, r.k), slots);
  if (threadIdx.x == 0) out[b] = a;
}
// ... second launch: joined, the row's end -- by one block per row, or (GRAD) by every block for its own stretch of the gradient as well.
template <typename T, int MODE, int GRAD> __global__ void __launch_bounds__(256) k_split_end(RowIo io, int splits, int64_t step, const Part* parts) {
  __shared__ double sd[4];
  const Rows& r = io.r;
  const int per_row = GRAD ? splits : 1;
  const int64_t b = (int64_t)blockIdx.y * gridDim.x + blockIdx.x, i = b / per_row, j0 = (b - i * per_row) * step, j1 = min(j0 + step, r.k);
  if (i >= r.rows) return;
  double acc[3] = {0.0, 0.0, 0.0}, weight = 1.0;
  int64_t count = 0;
  if (MODE == POLICY) weight = weight_of<256>(io, &count, sd);
  const bool first = j0 == 0 && threadIdx.x == 0;
  T* dx = GRAD ? (T*)io.dx + i * r.k : nullptr;
  if (r.mask && !r.mask[i]) {
    if (first) masked_row(io, i);
    if (GRAD) zero_row<T, 256>(dx + j0, j1 - j0, threadIdx.x);
  } else {
    const T* x = (const T*)r.x + i * r.stride;
    const int64_t c = choice_of(r, i);
    const bool ok = c >= 0 && c < r.k;
    const float xc = to_f32(x[ok ? c : 0]);
    const RowTerms terms = MODE == POLICY ? terms_of(io.p, i) : RowTerms{};
    const int lane = threadIdx.x & 63;
    Part a{0.0, -INFINITY};
    if (lane < splits) a = parts[i * splits + lane];
    a = join_lanes<64>(a);
    const RowEnd e = end_row<MODE>(io, i, terms, ok, xc, a, weight, first, acc);
    if (GRAD) stream_grad<T, 256>(x, dx, j0, j1, a.m, -e.coef * e.inv, e.coef, c, xc);
  }
  if (MODE == POLICY && first)
    for (int q = 0; q < 3; ++q) io.part[i * 3 + q] = acc[q];
}

// dx = gain * coef (one-hot - p) from the stored statistics (m, 1 / s).  skip_one: dx already holds the result for gain 1.
// Short rows: G lanes per row, as in k_rows_short ...
template <typename T, int G> __global__ void __launch_bounds__(256) k_grad_short(Rows r, const float* coef_in, const float2* stat, const float* gain, int skip_one, T* grad) {
  const float g = gain ? *gain : 1.0f;
  if (skip_one && g == 1.0f) return;
  const int lane = threadIdx.x & (G - 1), k = (int)r.k;
  for (int64_t i = (int64_t)blockIdx.x * (256 / G) + threadIdx.x / G; i < r.rows; i += (int64_t)gridDim.x * (256 / G)) {
    const T* x = (const T*)r.x + i * r.stride;
    const float coef = r.mask && !r.mask[i] ? 0.0f : coef_in[i] * g;
    const float2 st = stat[i];
    const int64_t c = choice_of(r, i);
    const float scale = -coef * st.y;
#pragma unroll
    for (int q = 0; q < 4; ++q) {
      const int j = q * G + lane;
      if (j < k) grad[i * k + j] = from_f32<T>(coef == 0.0f ? 0.0f : fmaf(exp_of<T>(to_f32(x[j]) - st.x), scale, j == c ? coef : 0.0f));
    }
  }
}
// ... rows of up to 8 TPR pieces: TPR lanes per row, four pieces in flight ...
template <typename T, int TPR> __global__ void __launch_bounds__(256) k_grad_rows(Rows r, const float* coef_in, const float2* stat, const float* gain, int skip_one, T* grad) {
  const float g = gain ? *gain : 1.0f;
  if (skip_one && g == 1.0f) return;
  const int t = threadIdx.x % TPR;
  for (int64_t i = (int64_t)blockIdx.x * (256 / TPR) + threadIdx.x / TPR; i < r.rows; i += (int64_t)gridDim.x * (256 / TPR)) {
    const int64_t c = choice_of(r, i);
    const float2 st = stat[i];
    const float coef = r.mask && !r.mask[i] ? 0.0f : coef_in[i] * g;
    T* dx = grad + i * r.k;
    if (coef == 0.0f) {
      zero_row<T, TPR>(dx, r.k, t);
      continue;
    }
    const T* x = (const T*)r.x + i * r.stride;
    const Shared<T, TPR> sh(x, r.k);
    const float last = t < sh.edges ? to_f32(x[sh.edge(t)]) : 0.0f, xc = c >= 0 && c < r.k ? to_f32(x[c]) : 0.0f;
    const float scale = -coef * st.y;
    const GradScale gs(st.x, scale);
    for (int q0 = t; q0 < sh.pieces; q0 += 4 * TPR) {
      Reg<T> v[4];
#pragma unroll
      for (int u = 0; u < 4; ++u)
        if (q0 + u * TPR < sh.pieces) v[u].load_once(x + sh.head + (q0 + u * TPR) * Reg<T>::N);
#pragma unroll
      for (int u = 0; u < 4; ++u)
        if (q0 + u * TPR < sh.pieces) {
          grad_piece<T>(v[u], gs);
          v[u].store(dx + sh.head + (q0 + u * TPR) * Reg<T>::N);
        }
    }
    if (t < sh.edges) dx[sh.edge(t)] = from_f32<T>(exp_of<T>(last - st.x) * scale);
    chosen_element<T, TPR>(dx, sh, r.k, c, t, xc, st.x, scale, coef);
  }
}
// ... longer rows: stretches of kGradPieces pieces per thread, `splits` of them per row.  A block per stretch -- or, where the call most likely has nothing
// to do (skip_one), few blocks that would share them: 65536 blocks that only return take 10 us, 1024 take 2.
// 8192 x 32768 bf16: 8 KB per block 168 us (6.2 TB/s), 4 KB 190, 16 KB 180, 32 KB 195; a loop of single pieces over 16 KB 205.
constexpr int kGradPieces = 2;
template <typename T> constexpr int64_t grad_step() { return 256 * kGradPieces * Reg<T>::N; }
template <typename T> __global__ void __launch_bounds__(256) k_grad_long(Rows r, const float* coef_in, const float2* stat, const float* gain, int skip_one, int splits, T* grad) {
  const float g = gain ? *gain : 1.0f;
  if (skip_one && g == 1.0f) return;
  const int t = threadIdx.x;
  for (int64_t b = (int64_t)blockIdx.y * gridDim.x + blockIdx.x; b < r.rows * splits; b += (int64_t)gridDim.x * gridDim.y) {
    const int64_t i = b / splits, j0 = (b - i * splits) * grad_step<T>();
    const int64_t len = min(grad_step<T>(), r.k - j0), c = choice_of(r, i) - j0;
    const float2 st = stat[i];
    const float coef = r.mask && !r.mask[i] ? 0.0f : coef_in[i] * g;
    T* dx = grad + i * r.k + j0;
    if (coef == 0.0f) {
      zero_row<T, 256>(dx, len, t);
      continue;
    }
    const T* x = (const T*)r.x + i * r.stride + j0;
    const Shared<T, 256> sh(x, len);
    Reg<T> v[kGradPieces];
#pragma unroll
    for (int q = 0; q < kGradPieces; ++q)
      if (q * 256 + t < sh.pieces) v[q].load_once(x + sh.head + q * (256 * Reg<T>::N) + t * Reg<T>::N);
    const float last = t < sh.edges ? to_f32(x[sh.edge(t)]) : 0.0f, xc = c >= 0 && c < len ? to_f32(x[c]) : 0.0f;
    const float scale = -coef * st.y;
    const GradScale gs(st.x, scale);
#pragma unroll
    for (int q = 0; q < kGradPieces; ++q)
      if (q * 256 + t < sh.pieces) {
        grad_piece<T>(v[q], gs);
        v[q].store(dx + sh.head + q * (256 * Reg<T>::N) + t * Reg<T>::N);
      }
    if (t < sh.edges) dx[sh.edge(t)] = from_f32<T>(exp_of<T>(last - st.x) * scale);
    chosen_element<T, 256>(dx, sh, len, c, t, xc, st.x, scale, coef);
  }
}

__global__ void __launch_bounds__(1024) k_count(const uint8_t* mask, int64_t n, int64_t* out) {
  __shared__ double sd[16];
  int64_t c = 0;
  for (int64_t i = threadIdx.x; i < n / 16; i += 4 * 1024) {      // (four pieces in flight)
    Reg<uint8_t> q[4];
#pragma unroll
    for (int u = 0; u < 4; ++u) {
      q[u].w[0] = q[u].w[1] = q[u].w[2] = q[u].w[3] = 0;
      if (i + u * 1024 < n / 16) q[u].load(mask + (i + u * 1024) * 16);
    }
#pragma unroll
    for (int u = 0; u < 4; ++u) c += nonzero_bytes(q[u]);
  }
  const int64_t rest = n / 16 * 16 + threadIdx.x;
  if (threadIdx.x < 16 && rest < n) c += mask[rest] != 0;
  const double t = block_sum<1024>((double)c, sd);     // (counts below 2^53 are exact)
  if (threadIdx.x == 0) *out = (int64_t)t;
}

// loss, mean kl, clipped share from the blocks' partial sums
__global__ void __launch_bounds__(256) k_policy_finish(RowIo io, int64_t blocks) {
  __shared__ double sd[12];
  int64_t count;
  const double weight = weight_of<256>(io, &count, sd);
  double v[3];
  for (int q = 0; q < 3; ++q) v[q] = long_sum<256>(io.part + q, blocks, 3);
  end_block<256, false>(io, 0, v, count, weight, sd);
}

// ---- preference pairs ------------------------------------------------------------------------------------------------------
struct Side { const float *logp, *ref; const uint8_t* mask; int64_t steps; };
struct __attribute__((packed)) Bytes4 { uint32_t w; };
// sum of the log ratios of pair p's valid steps by TPP threads, pieces of four steps, four of them in flight; masked steps are read with their piece
// and dropped by selection
template <int TPP> __device__ __forceinline__ double side_sum(const Side& s, int64_t p, int t) {
  constexpr int U = TPP < 64 ? 1 : 4;
  const float *a = s.logp + p * s.steps, *r = s.ref ? s.ref + p * s.steps : nullptr;
  const uint8_t* m = s.mask ? s.mask + p * s.steps : nullptr;
  const int64_t n = s.steps / 4;
  double v = 0.0;
  for (int64_t q = t; q < n; q += U * TPP) {
    Reg<float> x[U], y[U];
    uint32_t keep[U];
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const int64_t o = q + u * TPP;
      keep[u] = o < n ? 0xffffffffu : 0u;
#pragma unroll
      for (int j = 0; j < 4; ++j) x[u].w[j] = y[u].w[j] = 0;
      if (o < n) {
        x[u].load(a + o * 4);
        if (r) y[u].load(r + o * 4);
        if (m) keep[u] = ((const Bytes4*)(m + o * 4))->w;
      }
    }
#pragma unroll
    for (int u = 0; u < U; ++u)
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const double d = (double)__uint_as_float(x[u].w[j]) - (double)__uint_as_float(y[u].w[j]);
        v += keep[u] >> 8 * j & 255u ? d : 0.0;
      }
  }
  const int64_t j = n * 4 + t;
  if (t < 4 && j < s.steps && (!m || m[j])) v += (double)a[j] - (r ? (double)r[j] : 0.0);
  return v;
}
struct PairIo {
  Side w, l;
  int64_t pairs;
  double beta, eps, scale;      // scale: 1 / pairs of the mean included
  float *margin, *coef, *loss;
  double* part;
};
// TPP threads per pair: 16 lanes or a wave where the sequences are short, a block where they are long.
template <int TPP> __global__ void __launch_bounds__(256) k_pairs(PairIo io) {
  __shared__ double sd[4];
  const int t = threadIdx.x % TPP;
  double loss = 0.0;
  for (int64_t p = (int64_t)blockIdx.x * (256 / TPP) + threadIdx.x / TPP; p < io.pairs; p += (int64_t)gridDim.x * (256 / TPP)) {
    double h = side_sum<TPP>(io.w, p, t) - side_sum<TPP>(io.l, p, t);
    h = TPP <= 64 ? wave_sum<TPP <= 64 ? TPP : 64>(h) : block_sum<256>(h, sd);
    if (t == 0) {
      const double z = io.beta * h, e = exp64(-fabs(z)), lp = log1p(e);
      const double neg = (z < 0.0 ? -z : 0.0) + lp, pos = (z > 0.0 ? z : 0.0) + lp;      // -ln sigmoid(z), -ln sigmoid(-z)
      const double small = e / (1.0 + e), big = 1.0 / (1.0 + e), up = z >= 0.0 ? big : small, down = z >= 0.0 ? small : big;   // sigmoid(z), sigmoid(-z)
      io.margin[p] = (float)z;
      io.coef[p] = (float)(io.scale * io.beta * (io.eps * up - (1.0 - io.eps) * down));
      loss += z != z ? z : (1.0 - io.eps) * neg + io.eps * pos;
    }
  }
  loss = block_sum<256>(loss, sd);
  if (threadIdx.x) return;
  if (gridDim.x > 1) io.part[blockIdx.x] = loss;
  else *io.loss = (float)(loss * io.scale);       // (a launch of one block has the whole sum)
}
__global__ void __launch_bounds__(256) k_pairs_finish(const double* part, int blocks, double scale, float* out) {
  __shared__ double sd[4];
  const double v = block_sum<256>(long_sum<256>(part, blocks, 1), sd);
  if (threadIdx.x == 0) *out = (float)(v * scale);
}
constexpr int64_t kPairPiece = 1024;      // steps a wave writes
struct GradSide { float* out; const uint8_t* mask; int64_t steps, pieces; float sign; };
// Waves over (pair, piece of its steps), the better side's before the worse side's.
__global__ void __launch_bounds__(256) k_pairs_grad(const float* coef, const float* gain, int64_t pairs, GradSide b, GradSide w) {
  const float g = *gain;
  const int lane = threadIdx.x & 63;
  const int64_t total = pairs * (b.pieces + w.pieces);
  for (int64_t u = (int64_t)blockIdx.x * 4 + threadIdx.x / 64; u < total; u += (int64_t)gridDim.x * 4) {
    const bool first = u < pairs * b.pieces;
    const GradSide& s = first ? b : w;
    const int64_t v = first ? u : u - pairs * b.pieces, p = v / s.pieces, j0 = (v - p * s.pieces) * kPairPiece, j1 = min(j0 + kPairPiece, s.steps);
    const float c = coef[p] * g * s.sign;
    float* out = s.out + p * s.steps;
    const uint8_t* m = s.mask ? s.mask + p * s.steps : nullptr;
#pragma unroll
    for (int q = 0; q < 4; ++q) {
      const int64_t j = j0 + (q * 64 + lane) * 4;
      if (j + 4 <= j1) {
        const uint32_t keep = m ? ((const Bytes4*)(m + j))->w : 0xffffffffu;
        Reg<float> x;
#pragma unroll
        for (int i = 0; i < 4; ++i) x.w[i] = keep >> 8 * i & 255u ? __float_as_uint(c) : 0u;
        x.store(out + j);
      } else {
        for (int64_t i = j; i < j1; ++i) out[i] = !m || m[i] ? c : 0.0f;
      }
    }
  }
}

// ---- gradient lists --------------------------------------------------------------------------------------------------------
constexpr int kClipSlots = 240;          // ranges of a launch: the table travels in the kernel's arguments (under 4 KB), no copy to wait for
constexpr int kClipPieces = 8;           // 16-byte pieces of a thread, all in flight at once: 32 KB per block
template <typename T> constexpr int64_t clip_chunk() { return 256 * kClipPieces * Reg<T>::N; }      // elements of a block
struct ClipTable {
  void* ptr[kClipSlots];
  uint32_t numel[kClipSlots];
  int32_t first[kClipSlots];             // first block of the range
  int n, blocks, block0;                 // block0: index of the launch's first block among the partial sums
};
// the elements block b has of its range: whole pieces from a cache line's start on, and, for the range's first block, those before it
template <typename T> struct ClipPart {
  T* g;               // first piece
  int n, head, rest;  // whole pieces; elements before (at most 127 bytes) and behind them
  __device__ __forceinline__ ClipPart(const ClipTable& t, int b) {
    int lo = 0, hi = t.n - 1;
    while (lo < hi) {
      const int mid = (lo + hi + 1) >> 1;
      if (t.first[mid] <= b) lo = mid; else hi = mid - 1;
    }
    T* p = (T*)t.ptr[lo];
    const int64_t numel = t.numel[lo];
    int64_t lead = (int64_t)(-(uintptr_t)p & 127) / (int64_t)sizeof(T);
    if (lead > numel) lead = numel;
    const int64_t a = lead + (int64_t)(b - t.first[lo]) * clip_chunk<T>(), left = numel - a;
    const int len = (int)(left < 0 ? 0 : left < clip_chunk<T>() ? left : clip_chunk<T>());
    g = p + a;
    n = len / Reg<T>::N;
    rest = len - n * Reg<T>::N;
    head = b == t.first[lo] ? (int)lead : 0;
  }
  __device__ __forceinline__ T* edge() const {      // this thread's element beside the pieces, or NULL
    const int t = threadIdx.x;
    return t < head ? g - head + t : t < head + rest ? g + n * Reg<T>::N + (t - head) : nullptr;
  }
};
// Sum of squares of a block's elements, in 64 bits from the square on (a 32-bit square overflows from 1.8e19 and vanishes below 3.7e-23).
template <typename T> __global__ void __launch_bounds__(256) k_clip_norm(ClipTable t, double* part) {
  constexpr int V = Reg<T>::N;
  __shared__ double sd[4];
  const ClipPart<T> part_of(t, blockIdx.x);
  const T* g = part_of.g;
  const int n = part_of.n;
  Reg<T> v[kClipPieces];
#pragma unroll
  for (int q = 0; q < kClipPieces; ++q) {
    v[q].w[0] = v[q].w[1] = v[q].w[2] = v[q].w[3] = 0;
    if (q * 256 + (int)threadIdx.x < n) v[q].load_once(g + q * (256 * V) + threadIdx.x * V);
  }
  double a = 0.0;
  if (const T* e = part_of.edge()) {
    const double d = (double)to_f32(*e);
    a = d * d;
  }
#pragma unroll
  for (int q = 0; q < kClipPieces; ++q) {
    float f[V];
    v[q].get(f);
#pragma unroll
    for (int j = 0; j < V; ++j) a = fma((double)f[j], (double)f[j], a);
  }
  a = block_sum<256>(a, sd);
  if (threadIdx.x == 0) part[t.block0 + blockIdx.x] = a;
}
__global__ void __launch_bounds__(1024) k_clip_finish(const double* part, int64_t blocks, double max_norm, double eps, float* norm, float* coef) {
  __shared__ double sd[16];
  const double v = block_sum<1024>(long_sum<1024>(part, blocks, 1), sd);
  if (threadIdx.x == 0) {
    const double n = sqrt(v), c = isinf(max_norm) ? 1.0 : max_norm / (n + eps);
    *norm = (float)n;
    *coef = c >= 1.0 ? 1.0f : (float)c;       // (a NaN norm makes NaN gradients)
  }
}
// The last block first: what the norm's pass read last is still in the 256 MB cache.
template <typename T> __global__ void __launch_bounds__(256) k_clip_scale(ClipTable t, const float* coef) {
  constexpr int V = Reg<T>::N;
  const float c = *coef;
  if (c == 1.0f) return;
  const ClipPart<T> part_of(t, t.blocks - 1 - blockIdx.x);
  T* g = part_of.g;
  const int n = part_of.n;
  Reg<T> v[kClipPieces];
#pragma unroll
  for (int q = 0; q < kClipPieces; ++q)
    if (q * 256 + (int)threadIdx.x < n) v[q].load_once(g + q * (256 * V) + threadIdx.x * V);
  if (T* e = part_of.edge()) *e = from_f32<T>(to_f32(*e) * c);
#pragma unroll
  for (int q = 0; q < kClipPieces; ++q)
    if (q * 256 + (int)threadIdx.x < n) {
      float f[V];
      v[q].get(f);
#pragma unroll
      for (int j = 0; j < V; ++j) f[j] *= c;
      v[q].set(f);
      v[q].store(g + q * (256 * V) + threadIdx.x * V);
    }
}

// ---- host side -------------------------------------------------------------------------------------------------------------
// The launches of one entry: the first error ends it and is the entry's result (hipLaunchKernel's own return value -- hipGetLastError would
// also report, and clear, what an earlier call of somebody else's left).
struct Launches {
  hipStream_t stream;
  hipError_t err = hipSuccess;
  template <typename... P, size_t... I> void go(void (*k)(P...), dim3 grid, int threads, std::tuple<P...> args, std::index_sequence<I...>) {
    void* ptr[] = {(void*)&std::get<I>(args)...};
    if (err == hipSuccess) err = hipLaunchKernel((const void*)k, grid, dim3(threads), ptr, 0, stream);
  }
  template <typename... P, typename... A> void operator()(void (*k)(P...), dim3 grid, int threads, A... a) {
    go(k, grid, threads, std::tuple<P...>(a...), std::index_sequence_for<P...>{});
  }
  int result(const char* what) const { return err == hipSuccess ? PS_OK : set_error(PS_E_HIP, "%s: %s", what, hipGetErrorString(err)); }
};
int block_grid(int64_t rows) { return (int)(rows < kMaxGrid ? rows : kMaxGrid); }

// more blocks than one dimension takes threads for: lines of 65536 (the kernels drop what the last line has too many)
dim3 grid2d(int64_t blocks) {
  const int64_t wide = 1 << 16;
  return dim3((unsigned)(blocks < wide ? blocks : wide), (unsigned)((blocks + wide - 1) / wide));
}

int check_rows(const ps_decisions* d, const char* what, Rows* r) {
  if (!d) return set_error(PS_E_ARG, "%s: no decisions", what);
  if (d->rows < 0 || d->choices < 1 || d->choices > (1LL << 31) - 1 || d->rows > (1LL << 31)) return set_error(PS_E_ARG, "%s: rows must be in [0, 2^31] and choices in [1, 2^31)", what);
  if (d->row_stride < d->choices && d->rows > 1) return set_error(PS_E_ARG, "%s: row_stride < choices", what);
  if (d->dtype != PS_F32 && d->dtype != PS_BF16 && d->dtype != PS_F16) return set_error(PS_E_ARG, "%s: unknown element type", what);
  if (d->choice_bits != 32 && d->choice_bits != 64) return set_error(PS_E_ARG, "%s: choice_bits must be 32 or 64", what);
  if (d->rows && (!d->logits || !d->choice)) return set_error(PS_E_ARG, "%s: NULL logits or choice", what);
  if (((uintptr_t)d->logits & (d->dtype == PS_F32 ? 3 : 1)) || ((uintptr_t)d->choice & (d->choice_bits / 8 - 1))) return set_error(PS_E_ARG, "%s: logits or choice are not aligned to their elements", what);
  *r = Rows{d->logits, d->rows, d->choices, d->row_stride, d->choice, d->mask, d->choice_bits == 64};
  return PS_OK;
}

template <typename F> int by_type(int dtype, F f) {
  return dtype == PS_F32 ? f((float*)nullptr) : dtype == PS_BF16 ? f((bf16*)nullptr) : f((f16*)nullptr);
}

// How rows are laid out over the chip: a rule on their number, length and type.
enum RowKind { SHORT, HELD, SPLIT, VERY_LONG };
struct RowPlan {
  RowKind kind;
  int64_t grid;         // blocks of the first launch
  int splits;
  int64_t step;
  int64_t parts(int64_t rows) const { return kind == SPLIT || kind == VERY_LONG ? rows : grid; }      // partial sums of the loss
};
constexpr int64_t kPastCaches = 256 << 20;      // bytes of the last-level cache
constexpr int kShort = 32;             // elements a row of k_rows_short may have
// lanes of a short row, four elements each: the fewest, because a wave pays the end of a row once for all the rows it has
// (10^6 rows of 6 fp32 with gradient: 8 lanes of one element 69 us, 2 of four 26; of 30 bf16, forward: 32 of one 140 us, 8 of four 41)
int short_lanes(int64_t k) { return k <= 4 ? 1 : k <= 8 ? 2 : k <= 16 ? 4 : 8; }
RowPlan plan_rows(int64_t rows, int64_t k, int size, int mode) {
  const int64_t bytes = k * size, pieces = k * size / 16;
  RowPlan p{SHORT, 1, 1, k};
  auto grid = [&](int64_t per_block, int64_t most) { const int64_t b = (rows + per_block - 1) / per_block; return b < most ? b : most; };
  auto split = [&](int64_t want) {
    p.splits = (int)(want < 1 ? 1 : want > 64 ? 64 : want);
    p.step = ((k + p.splits - 1) / p.splits + 63) / 64 * 64;
    p.splits = (int)((k + p.step - 1) / p.step);
    p.grid = rows * p.splits;
  };
  if (k <= kShort) {
    const int g = short_lanes(k);
    p.grid = rows <= 2 * 256 / g ? 1 : grid(256 / g, kMaxGrid);      // (two turns of one block cost less than the launch that joins blocks)
  } else if (pieces > 8192 && rows <= 64) {
    // Several blocks to a row cost a second launch and a second read; they pay where a block alone would be long at it and most of the chip idle.
    // bf16 policy loss with gradient, one block / split: 131072 elements 1 row 16.8 / 11.3 us, 32 rows 23.9 / 14.6, 64 rows 24.8 / 19.0, 128 rows
    // 27.6 / 32.2; 32768 elements 1 row 8.6 / 11.2, 64 rows 13.0 / 12.8, 128 rows 13.2 / 14.8.
    p.kind = SPLIT;
    split(512 / rows);
  } else if (pieces <= 512) {
    p.kind = HELD;
    p.grid = grid(pieces <= 64 ? 32 : pieces <= 128 ? 16 : pieces <= 256 ? 8 : 4, rows);
  } else if (pieces <= (mode == LOGP && rows > 128 ? 8192 : 16384)) {
    // (with no gradient in view parts of rows overlap better than a block of 16 waves per CU: 131072 bf16, one block / parts, 2048 rows 111 / 88 us, 300 rows
    // 25.7 / 21.5, 100 rows 12.0 / 13.9; shorter rows, 65536 bf16 x 4096: 85 / 90)
    p.kind = HELD;
    p.grid = rows;
  } else {
    p.kind = VERY_LONG;      // (300 x 250000 fp32 with gradient: 162 us; a block per row in two passes 222)
    split((bytes + 65535) / 65536);
  }
  return p;
}
template <typename T> void launch_grad(Launches& run, const Rows& r, const float* coef, const float2* stat, const float* gain, int skip, T* grad) {
  const int64_t pieces = r.k / Reg<T>::N;
  auto grid = [&](int lanes) { const int64_t b = (r.rows + 256 / lanes - 1) / (256 / lanes), most = skip ? 512 : 1 << 20; return (int)(b < most ? b : most); };
  if (r.k <= kShort) {
    const int g = short_lanes(r.k);
    run(g == 1 ? k_grad_short<T, 1> : g == 2 ? k_grad_short<T, 2> : g == 4 ? k_grad_short<T, 4> : k_grad_short<T, 8>, grid(g), 256, r, coef, stat, gain, skip, grad);
  } else if (pieces <= 256) {
    const int lanes = pieces <= 64 ? 8 : 32;
    run(lanes == 8 ? k_grad_rows<T, 8> : k_grad_rows<T, 32>, grid(lanes), 256, r, coef, stat, gain, skip, grad);
  } else {
    const int splits = (int)((r.k + grad_step<T>() - 1) / grad_step<T>());
    const int64_t all = r.rows * splits;
    run(k_grad_long<T>, grid2d(skip && all > 1024 ? 1024 : all), 256, r, coef, stat, gain, skip, splits, grad);
  }
}
template <typename T, int MODE, int GRAD> void launch_rows(Launches& run, const RowIo& io, const RowPlan& p, Part* parts) {
  const int64_t k = io.r.k, pieces = k / Reg<T>::N;
  const dim3 grid = grid2d(p.grid);
  constexpr int G1 = GRAD == GRAD_PAST ? GRAD_KEPT : GRAD;       // (the kernels that make no difference)
  if (p.kind == SHORT) {
    const int g = short_lanes(k);
    run(g == 1 ? k_rows_short<T, 1, 4, MODE, G1> : g == 2 ? k_rows_short<T, 2, 4, MODE, G1> : g == 4 ? k_rows_short<T, 4, 4, MODE, G1> : k_rows_short<T, 8, 4, MODE, G1>, grid, 256, io);
  } else if (p.kind == HELD) {
    // Threads per row by its pieces.  Few threads with many pieces each beat many with few: the end of a row (64-bit functions, reductions) costs
    // every wave of it the same (8192-element rows: 1 x 512 rows of 64 threads x 16 pieces 87 us, 2 x 8 89 us, 4 x 4 114 us), and rows that need not
    // wait for each other overlap one's reading with another's writing (65536-element rows with gradient: 8 waves x 16 pieces 192 us, 16 x 8 251 us).
    constexpr bool fwd = MODE == LOGP;       // (the policy loss takes the same kernel with and without its gradient: the same bits)
    if (pieces <= 16) run(k_rows_held<T, 8, 2, MODE, GRAD>, grid, 256, io);
    else if (pieces <= 32) run(k_rows_held<T, 8, 4, MODE, GRAD>, grid, 256, io);
    else if (pieces <= 64) run(k_rows_held<T, 8, 8, MODE, GRAD>, grid, 256, io);
    else if (pieces <= 128) run(k_rows_held<T, 16, 8, MODE, GRAD>, grid, 256, io);
    else if (pieces <= 256) run(k_rows_held<T, 32, 8, MODE, GRAD>, grid, 256, io);
    else if (pieces <= 512) run(k_rows_held<T, 64, 8, MODE, GRAD>, grid, 256, io);
    else if (pieces <= 1024) run(k_rows_held<T, 128, 8, MODE, GRAD>, grid, 128, io);
    else if (pieces <= 2048) run(k_rows_held<T, fwd ? 128 : 256, fwd ? 16 : 8, MODE, GRAD>, grid, fwd ? 128 : 256, io);
    else if (pieces <= 4096) run(k_rows_held<T, 256, 16, MODE, GRAD>, grid, 256, io);
    else if (pieces <= 8192) run(k_rows_held<T, 512, 16, MODE, GRAD>, grid, 512, io);
    else run(k_rows_held<T, 1024, 16, MODE, GRAD>, grid, 1024, io);
  } else {
    run(k_split_part<T>, grid, 256, io.r, p.splits, p.step, parts);
    if (p.kind == SPLIT) {
      run(k_split_end<T, MODE, G1>, GRAD ? grid : grid2d(io.r.rows), 256, io, p.splits, p.step, (const Part*)parts);
    } else {
      run(k_split_end<T, MODE, GRAD_NONE>, grid2d(io.r.rows), 256, io, p.splits, p.step, (const Part*)parts);
      if (GRAD) launch_grad<T>(run, io.r, io.coef, io.stat, nullptr, 0, (T*)io.dx);
    }
  }
}

// count | (loss, kl, clipped) per block | partial results of split rows | (maximum, 1 / sum) and coefficient of very long rows
int64_t row_space(const ps_decisions* d, int mode) {
  if (d->rows < 1 || d->choices < 1) return 8;
  const RowPlan p = plan_rows(d->rows, d->choices, d->dtype == PS_F32 ? 4 : 2, mode);
  return 8 + 24 * p.parts(d->rows) + (p.kind == SPLIT || p.kind == VERY_LONG ? 16 * p.grid : 0) + (p.kind == VERY_LONG ? 12 * d->rows : 0);
}
struct RowSpace {
  int64_t* count;
  double* part;
  Part* parts;
  float2* stat;
  float* coef;
  RowSpace(void* p, const RowPlan& plan, int64_t rows)
      : count((int64_t*)p), part((double*)p + 1), parts((Part*)(part + 3 * plan.parts(rows))), stat((float2*)(parts + (plan.kind == VERY_LONG ? plan.grid : 0))), coef((float*)(stat + rows)) {}
};
int check_space(const void* p, int64_t bytes, int64_t need, const char* what) {
  if (!p || bytes < need || ((uintptr_t)p & 7)) return set_error(PS_E_ARG, "%s: workspace missing, unaligned or smaller than %lld bytes", what, (long long)need);
  return PS_OK;
}
}  // namespace

extern "C" int64_t ps_choice_workspace(const ps_decisions* d) { 
  if (!d) return set_error(PS_E_ARG, "ps_choice_workspace: no decisions");
  const int64_t a = row_space(d, LOGP), b = row_space(d, POLICY);
  return a > b ? a : b;
}

extern "C" int ps_choice_logp(const ps_decisions* d, float* logp, float* stat, void* workspace, int64_t workspace_bytes, void* stream) {
  RowIo io{};
  if (int e = check_rows(d, "ps_choice_logp", &io.r)) return e;
  if (!io.r.rows) return PS_OK;
  if (!logp || ((uintptr_t)stat & 7)) return set_error(PS_E_ARG, "ps_choice_logp: NULL logp, or stat is not aligned");
  if (int e = check_space(workspace, workspace_bytes, row_space(d, LOGP), "ps_choice_logp")) return e;
  Launches run{(hipStream_t)stream};
  io.logp = logp;
  io.stat = (float2*)stat;
  by_type(d->dtype, [&](auto* t) {
    typedef std::remove_pointer_t<decltype(t)> T;
    const RowPlan p = plan_rows(io.r.rows, io.r.k, sizeof(T), LOGP);
    launch_rows<T, LOGP, GRAD_NONE>(run, io, p, RowSpace(workspace, p, io.r.rows).parts);
    return 0;
  });
  return run.result("ps_choice_logp");
}

extern "C" int ps_choice_grad(const ps_decisions* d, const float* coef, const float* stat, const float* gain, int32_t skip_if_one, void* grad, void* stream) {
  Rows r;
  if (int e = check_rows(d, "ps_choice_grad", &r)) return e;
  if (!r.rows) return PS_OK;
  if (!coef || !stat || !grad) return set_error(PS_E_ARG, "ps_choice_grad: NULL coef, stat or grad");
  if (((uintptr_t)grad & (d->dtype == PS_F32 ? 3 : 1)) || ((uintptr_t)stat & 7)) return set_error(PS_E_ARG, "ps_choice_grad: grad or stat is not aligned");
  Launches run{(hipStream_t)stream};
  by_type(d->dtype, [&](auto* t) {
    typedef std::remove_pointer_t<decltype(t)> T;
    launch_grad<T>(run, r, coef, (const float2*)stat, gain, skip_if_one, (T*)grad);
    return 0;
  });
  return run.result("ps_choice_grad");
}

extern "C" int ps_policy_loss(const ps_decisions* d, const ps_policy_terms* q, float* loss, float* kl, float* clip_frac, float* logp, float* stat,
                              float* coef, void* grad, void* workspace, int64_t workspace_bytes, void* stream) {
  RowIo io{};
  if (int e = check_rows(d, "ps_policy_loss", &io.r)) return e;
  const Rows& r = io.r;
  if (!q || !loss || !kl || !clip_frac || (r.rows && (!q->old_logp || !q->advantage || !logp))) return set_error(PS_E_ARG, "ps_policy_loss: NULL terms, loss, kl, clip_frac, old_logp, advantage or logp");
  if (!(q->clip_low >= 0.0 && q->clip_low <= 1.0) || !(q->clip_high >= 0.0)) return set_error(PS_E_ARG, "ps_policy_loss: clip_low must be in [0, 1] and clip_high >= 0");
  if (!(q->kl_coef >= 0.0) || std::isinf(q->kl_coef)) return set_error(PS_E_ARG, "ps_policy_loss: kl_coef must be >= 0 and finite");
  if (!std::isfinite(q->scale)) return set_error(PS_E_ARG, "ps_policy_loss: scale must be finite");
  if (q->kl_coef > 0.0 && !q->ref_logp && r.rows) return set_error(PS_E_ARG, "ps_policy_loss: kl_coef without ref_logp");
  if (((uintptr_t)grad & (d->dtype == PS_F32 ? 3 : 1)) || ((uintptr_t)stat & 7)) return set_error(PS_E_ARG, "ps_policy_loss: grad or stat is not aligned");
  if (int e = check_space(workspace, workspace_bytes, row_space(d, POLICY), "ps_policy_loss")) return e;
  Launches run{(hipStream_t)stream};
  const RowPlan p = r.rows ? plan_rows(r.rows, r.k, d->dtype == PS_F32 ? 4 : 2, POLICY) : RowPlan{SHORT, 0, 1, 0};
  const RowSpace w(workspace, p, r.rows);
  // the valid rows of a short mask are counted by every block for itself (1 - 2 us, all at once where the blocks are few), else by a launch (5 us)
  const bool counted = r.mask && (r.rows > 16384 || p.grid > 1024);
  io.p = Policy{q->old_logp, q->advantage, q->ref_logp, 1.0 - q->clip_low, 1.0 + q->clip_high, q->kl_coef, q->scale, counted ? w.count : nullptr, q->mean};
  io.logp = logp;
  io.stat = stat || p.kind != VERY_LONG || !grad ? (float2*)stat : w.stat;
  io.coef = coef || p.kind != VERY_LONG || !grad ? coef : w.coef;
  io.dx = grad;
  io.part = w.part;
  io.loss = loss;
  io.kl = kl;
  io.clip_frac = clip_frac;
  const bool past = r.rows * r.k * (d->dtype == PS_F32 ? 4 : 2) >= kPastCaches;
  if (counted) run(k_count, 1, 1024, r.mask, r.rows, w.count);
  if (r.rows)
    by_type(d->dtype, [&](auto* t) {
      typedef std::remove_pointer_t<decltype(t)> T;
      if (grad && past && p.kind == HELD) launch_rows<T, POLICY, GRAD_PAST>(run, io, p, w.parts);
      else if (grad) launch_rows<T, POLICY, GRAD_KEPT>(run, io, p, w.parts);
      else launch_rows<T, POLICY, GRAD_NONE>(run, io, p, w.parts);
      return 0;
    });
  if (p.grid != 1 || p.kind == SPLIT || p.kind == VERY_LONG) run(k_policy_finish, 1, 256, io, p.parts(r.rows));      // (a launch of one block has written the results itself)
  return run.result("ps_policy_loss");
}

extern "C" int64_t ps_preference_loss_workspace(int64_t) { return 8 * (int64_t)kMaxGrid; }

extern "C" int ps_preference_loss(const ps_preference* q, float* loss, float* margin, float* coef, void* workspace, int64_t workspace_bytes, void* stream) {
  if (!q || q->pairs < 1 || q->better_steps < 0 || q->worse_steps < 0) return set_error(PS_E_ARG, "ps_preference_loss: pairs must be >= 1 and steps >= 0");
  if ((q->better_steps && !q->better) || (q->worse_steps && !q->worse) || !loss || !margin || !coef) return set_error(PS_E_ARG, "ps_preference_loss: NULL better, worse, loss, margin or coef");
  if (!std::isfinite(q->beta) || !(q->label_smoothing >= 0.0 && q->label_smoothing <= 1.0) || !std::isfinite(q->scale)) return set_error(PS_E_ARG, "ps_preference_loss: beta and scale must be finite, label_smoothing in [0, 1]");
  if (int e = check_space(workspace, workspace_bytes, ps_preference_loss_workspace(q->pairs), "ps_preference_loss")) return e;
  Launches run{(hipStream_t)stream};
  const double scale = q->scale / (q->mean ? (double)q->pairs : 1.0);
  const PairIo io{Side{q->better, q->better_ref, q->better_mask, q->better_steps}, Side{q->worse, q->worse_ref, q->worse_mask, q->worse_steps}, q->pairs, q->beta, q->label_smoothing,
                  scale, margin, coef, loss, (double*)workspace};
  // 16 lanes per pair up to 64 steps of its longer side, a wave up to 512, a block beyond; pairs that fit one block need no second launch
  const int64_t steps = q->better_steps > q->worse_steps ? q->better_steps : q->worse_steps;
  const int per_block = steps <= 64 ? 16 : steps <= 512 ? 4 : 1;
  const int grid = block_grid((q->pairs + per_block - 1) / per_block);
  run(per_block == 16 ? k_pairs<16> : per_block == 4 ? k_pairs<64> : k_pairs<256>, grid, 256, io);
  if (grid > 1) run(k_pairs_finish, 1, 256, (const double*)workspace, grid, scale, loss);
  return run.result("ps_preference_loss");
}

extern "C" int ps_preference_grad(const ps_preference* q, const float* coef, const float* gain, float* better_grad, float* worse_grad, void* stream) {
  if (!q || q->pairs < 1 || q->better_steps < 0 || q->worse_steps < 0 || !coef || !gain) return set_error(PS_E_ARG, "ps_preference_grad: bad pairs, or NULL coef or gain");
  Launches run{(hipStream_t)stream};
  auto side = [&](float* out, const uint8_t* mask, int64_t steps, float sign) { return GradSide{out, mask, steps, out ? (steps + kPairPiece - 1) / kPairPiece : 0, sign}; };
  const GradSide b = side(better_grad, q->better_mask, q->better_steps, 1.0f), w = side(worse_grad, q->worse_mask, q->worse_steps, -1.0f);
  const int64_t units = q->pairs * (b.pieces + w.pieces);
  if (units) run(k_pairs_grad, block_grid((units + 3) / 4), 256, coef, gain, q->pairs, b, w);
  return run.result("ps_preference_grad");
}

namespace {
int64_t clip_blocks(int64_t n, int dtype) {
  const int64_t chunk = dtype == PS_F32 ? clip_chunk<float>() : clip_chunk<bf16>();
  return (n + chunk - 1) / chunk;
}
constexpr int64_t kClipPiece = 1LL << 31;     // elements of a table entry (a longer tensor takes several)
int check_clip(const char* what, int32_t n, void* const* ptr, const int64_t* numel, const int32_t* dtype) {
  if (n < 0 || (n && (!ptr || !numel || !dtype))) return set_error(PS_E_ARG, "%s: NULL table", what);
  for (int32_t i = 0; i < n; ++i)
    if (numel[i] < 0 || (numel[i] && !ptr[i]) || (dtype[i] != PS_F32 && dtype[i] != PS_BF16 && dtype[i] != PS_F16) || ((uintptr_t)ptr[i] & (dtype[i] == PS_F32 ? 3 : 1)))
      return set_error(PS_E_ARG, "%s: tensor %d has a negative size, a NULL or unaligned pointer or an unknown element type", what, (int)i);
  return PS_OK;
}
// fill one table after the other, each of one element type, and launch it; returns the blocks of all launches
template <typename F> int64_t clip_tables(int32_t n, void* const* ptr, const int64_t* numel, const int32_t* dtype, F launch) {
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
          t.blocks = blocks;
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
        blocks += (int)clip_blocks(len, ty);
      }
    }
  }
  return block0;
}
}  // namespace

extern "C" int64_t ps_clip_grads_workspace(int32_t n, const int64_t* numel, const int32_t* dtype) {
  if (n < 0 || (n && (!numel || !dtype))) return set_error(PS_E_ARG, "ps_clip_grads_workspace: NULL table");
  int64_t b = 0;
  for (int32_t i = 0; i < n; ++i) b += clip_blocks(numel[i] > 0 ? numel[i] : 0, dtype[i]);
  return 8 * (b + 1);
}

extern "C" int ps_clip_grads(int32_t n, void* const* ptr, const int64_t* numel, const int32_t* dtype, double max_norm, double eps, float* norm,
                             void* workspace, int64_t workspace_bytes, void* stream) {
  if (int e = check_clip("ps_clip_grads", n, ptr, numel, dtype)) return e;
  if (!(max_norm >= 0.0) || !(eps >= 0.0) || std::isinf(eps)) return set_error(PS_E_ARG, "ps_clip_grads: max_norm must be >= 0, eps >= 0 and finite");
  if (!norm) return set_error(PS_E_ARG, "ps_clip_grads: NULL norm");
  const int64_t need = ps_clip_grads_workspace(n, numel, dtype);
  if (need / 8 > (1LL << 30)) return set_error(PS_E_ARG, "ps_clip_grads: more than 2^43 elements");
  if (int e = check_space(workspace, workspace_bytes, need, "ps_clip_grads")) return e;
  Launches run{(hipStream_t)stream};
  float* coef = (float*)workspace;
  double* part = (double*)workspace + 1;
  const int64_t blocks = clip_tables(n, ptr, numel, dtype, [&](const ClipTable& t, int blocks, int ty) {
    by_type(ty, [&](auto* p) { run(k_clip_norm<std::remove_pointer_t<decltype(p)>>, blocks, 256, t, part); return 0; });
  });
  run(k_clip_finish, 1, 1024, part, blocks, max_norm, eps, norm, coef);
  clip_tables(n, ptr, numel, dtype, [&](const ClipTable& t, int blocks, int ty) {
    by_type(ty, [&](auto* p) { run(k_clip_scale<std::remove_pointer_t<decltype(p)>>, blocks, 256, t, coef); return 0; });
  });
  return run.result("ps_clip_grads");
}
