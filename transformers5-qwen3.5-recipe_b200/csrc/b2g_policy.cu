// Post-training losses on rows of logits: token log-probabilities with their gradient, the clipped policy loss with a KL
// term (loss and cotangent in one pass over the logits), and the preference loss on paired sequences.
//   lse = m/tau + log d,  m = max z,  d = sum exp((z - m)/tau),  logp = z_y/tau - lse,
//   dz = c (onehot - p)/tau,  p = exp(z/tau - lse)
// What bounds them is HBM: one read of the logits, and one write of the cotangent.  The scalars of a row are finished in 64
// bits, because a ratio exp(logp - old) next to a clipping border, e^d - d - 1 of nearly equal policies and the sum of a long
// sequence all lose what a 32-bit log-probability has already rounded away.
#include "b2g_common.cuh"

#include <cmath>

namespace b2g {
namespace policy {

constexpr float kLowest = -3.402823466e38f;
// ex2.approx falls short by 4.9e-8 of its value on average (measured over 4 Mi arguments in [-20, 0], 3.7e-8 to 5.9e-8 in
// the eight octiles of the fraction); a sum of many of them is that much too small.  That is an average of what lies well below the
// reference: by bins of the argument it is 5.0e-8 to 5.2e-8 from -32 to -2, 4.2e-8 to 5.4e-8 from -2 to -0.5, 1e-8 to 2e-8 from -0.5
// to 0, and above 0 ex2 is 3.4e-8 too LARGE.  So it overdoes rows that are carried by terms at or above the reference: 2.5e-8 in
// wide rows of normal logits of spread 2 (5e-8 at temperature 0.7), whose reference is the largest of a sample, and 4.9e-8 where
// all logits are equal.  Rows with a dominant token, whose terms lie below, are off by 5e-9.
constexpr double kEx2Shortfall = 4.9e-8;

template <typename T>
__device__ __forceinline__ float to_float(T v) {
  if constexpr (sizeof(T) == 2) return __bfloat162float(v);
  else return v;
}
template <typename T>
__device__ __forceinline__ T from_float(float v) {
  if constexpr (sizeof(T) == 2) return __float2bfloat16_rn(v);
  else return v;
}
__device__ __forceinline__ float ex2(float x) {
  float r;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(x));
  return r;
}

// exp((z - m) / tau).  16-bit logits: one ex2, its factor log2(e)/tau in two parts (a single fp32 factor is off by 1.3e-8,
// which times the spread of the logits would reach every log-probability with the same sign).  fp32 logits, whose gradient
// keeps 24 bits, take the full exponential, its factor 1/tau in two parts for the same reason (off by up to 6e-8, and the same
// in the sum and in the gradient, whose entries cancel over a row); they move twice the bytes per value, so it is as well hidden.
struct Scale { float hi, lo, inv, inv_lo; };
// Two floats in one 64-bit register pair: one instruction of the two-wide fp32 pipe each.
struct F2 { uint64_t v; };
__device__ __forceinline__ F2 f2(float lo, float hi) {
  F2 r;
  asm("mov.b64 %0, {%1, %2};" : "=l"(r.v) : "f"(lo), "f"(hi));
  return r;
}
__device__ __forceinline__ void split(F2 a, float& lo, float& hi) { asm("mov.b64 {%0, %1}, %2;" : "=f"(lo), "=f"(hi) : "l"(a.v)); }
__device__ __forceinline__ F2 operator+(F2 a, F2 b) {
  F2 r;
  asm("add.rn.f32x2 %0, %1, %2;" : "=l"(r.v) : "l"(a.v), "l"(b.v));
  return r;
}
__device__ __forceinline__ F2 operator*(F2 a, F2 b) {
  F2 r;
  asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(r.v) : "l"(a.v), "l"(b.v));
  return r;
}
__device__ __forceinline__ F2 fma2(F2 a, F2 b, F2 c) {
  F2 r;
  asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(r.v) : "l"(a.v), "l"(b.v), "l"(c.v));
  return r;
}

// A pair of exponentials.  kSum: for the sum, where the factor's second part counts; a 16-bit cotangent is good without it.
template <typename T, bool kSum>
__device__ __forceinline__ F2 exp_from(F2 z, F2 minus_m, const Scale& c) {
  const F2 x = z + minus_m;
  float lo, hi;
  if constexpr (sizeof(T) == 2) {
    const F2 h = f2(c.hi, c.hi);
    split(kSum ? fma2(x, h, x * f2(c.lo, c.lo)) : x * h, lo, hi);
    return f2(ex2(lo), ex2(hi));
  } else {
    split(fma2(x, f2(c.inv, c.inv), x * f2(c.inv_lo, c.inv_lo)), lo, hi);
    return f2(expf(lo), expf(hi));
  }
}
// The sum without ex2's shortfall.
template <typename T>
__device__ __forceinline__ double whole_sum(double d) { return sizeof(T) == 2 ? d * (1.0 + kEx2Shortfall) : d; }

// Sixteen bytes of logits as floats, and back.
template <typename T>
struct Vec {
  static constexpr int N = 16 / sizeof(T);
  uint32_t w[4];
  __device__ __forceinline__ float get(int i) const {
    if constexpr (sizeof(T) == 2) return (i & 1) ? dev::bf16_hi(w[i >> 1]) : dev::bf16_lo(w[i >> 1]);
    else return __uint_as_float(w[i]);
  }
  // pair i of the N / 2
  __device__ __forceinline__ F2 pair(int i) const {
    if constexpr (sizeof(T) == 2) return f2(dev::bf16_lo(w[i]), dev::bf16_hi(w[i]));
    else return f2(__uint_as_float(w[2 * i]), __uint_as_float(w[2 * i + 1]));
  }
  // Between two passes over registers: the compiler may not keep the unpacked floats of the first, at a register each.
  __device__ __forceinline__ void packed_again() {
#pragma unroll
    for (int i = 0; i < 4; ++i) asm volatile("" : "+r"(w[i]));
  }
  // -inf in place of value j
  __device__ __forceinline__ void take_out(int j) {
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      if (sizeof(T) == 4) w[i] = i == j ? 0xFF800000u : w[i];
      else w[i] = i != j >> 1 ? w[i] : (j & 1) ? (w[i] & 0xFFFFu) | 0xFF800000u : (w[i] & 0xFFFF0000u) | 0xFF80u;
    }
  }
  __device__ __forceinline__ void set_nothing() {   // -inf everywhere: the maximum and the sum do not see it
#pragma unroll
    for (int i = 0; i < 4; ++i) w[i] = sizeof(T) == 2 ? 0xFF80FF80u : 0xFF800000u;
  }
};

// Sum of exponentials of a vector, summed as a tree.
template <typename T>
__device__ __forceinline__ F2 exp_sum(const Vec<T>& x, F2 minus_m, const Scale& c) {
  constexpr int P = Vec<T>::N / 2;
  F2 e[P];
#pragma unroll
  for (int i = 0; i < P; ++i) e[i] = exp_from<T, true>(x.pair(i), minus_m, c);
#pragma unroll
  for (int s = P / 2; s > 0; s >>= 1)
#pragma unroll
    for (int i = 0; i < s; ++i) e[i] = e[i] + e[i + s];
  return e[0];
}
__device__ __forceinline__ float sum_of(F2 a) {
  float lo, hi;
  split(a, lo, hi);
  return lo + hi;
}

// factor * exponentials of a vector, in the logits' type.
template <typename T>
__device__ __forceinline__ Vec<T> scaled_exp(const Vec<T>& x, F2 minus_m, F2 factor, const Scale& c) {
  Vec<T> r;
#pragma unroll
  for (int i = 0; i < Vec<T>::N / 2; ++i) {
    float lo, hi;
    split(exp_from<T, false>(x.pair(i), minus_m, c) * factor, lo, hi);
    if constexpr (sizeof(T) == 2) {
      r.w[i] = dev::pack_bf16(lo, hi);
    } else {
      r.w[2 * i] = __float_as_uint(lo);
      r.w[2 * i + 1] = __float_as_uint(hi);
    }
  }
  return r;
}

template <typename T>
__device__ __forceinline__ Vec<T> scaled(const Vec<T>& e, F2 factor) {
  Vec<T> r;
#pragma unroll
  for (int i = 0; i < Vec<T>::N / 2; ++i) {
    float lo, hi;
    split(e.pair(i) * factor, lo, hi);
    r.w[2 * i] = __float_as_uint(lo);
    r.w[2 * i + 1] = __float_as_uint(hi);
  }
  return r;
}

// A row as 16-byte vectors of the memory it lies in: vector v holds the columns [v * N - shift, (v + 1) * N - shift), so the
// inner vectors are aligned whatever the row's own alignment is, and at most the first and the last one are partial.
template <typename T>
struct Row {
  static constexpr int N = Vec<T>::N;
  const T* x;
  int shift, nvec, first_full, full_end;
  int V;
  __device__ Row(const T* p, int64_t width) : x(p), shift((int)((reinterpret_cast<uintptr_t>(p) / sizeof(T)) % N)), V((int)width) {
    nvec = (int)((width + shift + N - 1) / N);
    first_full = shift ? 1 : 0;
    full_end = (int)((width + shift) / N);
  }
  __device__ __forceinline__ int64_t column(int v) const { return (int64_t)v * N - shift; }
  __device__ __forceinline__ bool full(int v) const { return v >= first_full && v < full_end; }
  __device__ __forceinline__ Vec<T> load(int v) const {
    Vec<T> r;
    if (full(v)) {
      const uint4 q = __ldcs(reinterpret_cast<const uint4*>(x + column(v)));
      r.w[0] = q.x; r.w[1] = q.y; r.w[2] = q.z; r.w[3] = q.w;
    } else {
      r.set_nothing();
#pragma unroll
      for (int i = 0; i < N; ++i) {
        const int64_t c = column(v) + i;
        if (c >= 0 && c < V) {
          if constexpr (sizeof(T) == 2) {
            const uint32_t b = __bfloat16_as_ushort(x[c]);
            r.w[i >> 1] = (i & 1) ? (r.w[i >> 1] & 0xFFFFu) | (b << 16) : (r.w[i >> 1] & 0xFFFF0000u) | b;
          } else {
            r.w[i] = __float_as_uint(x[c]);
          }
        }
      }
    }
    return r;
  }
  // Writes a vector to the same columns of `out`; `wide`: out is aligned as the row is.
  __device__ __forceinline__ void store(T* out, int v, const Vec<T>& g, bool wide) const {
    if (wide && full(v)) {
      __stcs(reinterpret_cast<uint4*>(out + column(v)), make_uint4(g.w[0], g.w[1], g.w[2], g.w[3]));
    } else {
#pragma unroll
      for (int i = 0; i < N; ++i) {
        const int64_t c = column(v) + i;
        if (c >= 0 && c < V) {
          if constexpr (sizeof(T) == 2) out[c] = __ushort_as_bfloat16((unsigned short)((i & 1) ? g.w[i >> 1] >> 16 : g.w[i >> 1] & 0xFFFFu));
          else out[c] = __uint_as_float(g.w[i]);
        }
      }
    }
  }
};
template <typename T>
__device__ __forceinline__ Vec<T> zeros() {
  Vec<T> z;
  z.w[0] = z.w[1] = z.w[2] = z.w[3] = 0u;
  return z;
}
template <typename T>
__device__ __forceinline__ bool same_alignment(const T* a, const T* b) {
  return ((reinterpret_cast<uintptr_t>(a) ^ reinterpret_cast<uintptr_t>(b)) & 15) == 0;
}

// What a launch computes for its rows, and where the row's scalars come from and go to.
struct RowArgs {
  const int64_t* target;
  int64_t V, ignore_index;
  float tau;
  double inv_tau;
  Scale c;
  int* status;
  // log-probabilities
  void* logp;          // fp32, or fp64 when logp64
  int logp64;
  float4* stats;       // what the backward pass of the log-probabilities reads: m, 1/sum of exp((z - m)/tau), 1 - p of the target; and lse for the caller
  // policy loss
  const float *advantage, *old_logp, *ref_logp, *weight;
  float clip_low, clip_high, kl_coef;
  float *loss, *kl;
};

__device__ __forceinline__ bool target_ok(int64_t y, const RowArgs& a, bool report) {
  if (y == a.ignore_index) return false;
  if (y >= 0 && y < a.V) return true;
  if (report && a.status) atomicCAS(a.status, 0, 902);
  return false;
}

// The scalars of a row that a policy loss reads.
struct Given { float weight, advantage, old_logp, ref_logp; };
__device__ __forceinline__ Given given(const RowArgs& a, int64_t row) {
  return Given{a.weight ? a.weight[row] : 1.f, a.advantage[row], a.old_logp ? a.old_logp[row] : 0.f, a.ref_logp ? a.ref_logp[row] : 0.f};
}

__device__ __forceinline__ void put_logp(const RowArgs& a, int64_t row, double logp, float4 stats) {
  if (a.logp64) static_cast<double*>(a.logp)[row] = logp;
  else static_cast<float*>(a.logp)[row] = (float)logp;
  a.stats[row] = stats;
}

// Loss, log-probability and KL estimate of a live row; returns d loss / d logp.
__device__ __forceinline__ float policy_scalars(const RowArgs& a, const Given& in, double logp, int64_t row, bool write) {
  const double adv = in.advantage, ratio = a.old_logp ? exp(logp - (double)in.old_logp) : (logp != logp ? logp : 1.0);
  const double clipped = fmin(fmax(ratio, 1.0 - (double)a.clip_low), 1.0 + (double)a.clip_high);
  const bool inside = ratio * adv <= clipped * adv || ratio != ratio || adv != adv;      // NaN goes on to the gradient
  double loss = inside ? -ratio * adv : -clipped * adv, slope = inside ? -ratio * adv : 0.0, kl = 0.0;
  if (a.ref_logp) {
    const double d = (double)in.ref_logp - logp, em = expm1(d);
    kl = em - d;
    loss += (double)a.kl_coef * kl;
    slope -= (double)a.kl_coef * em;
  }
  if (write) {
    a.loss[row] = (float)(in.weight * loss);
    static_cast<float*>(a.logp)[row] = (float)logp;
    a.kl[row] = (float)kl;
  }
  return (float)(in.weight * slope);
}

// What the exponentials of a row, or of a part of it, were taken against, and their sum WITHOUT the target's own term.  A
// reference starts at the type's lowest value, not at -inf, so that -inf logits (a masked vocabulary) meet a finite one:
// exp(-inf - lowest) = 0.
struct Stat { float m; double d; };

// The joint sum of `count` lanes (a power of two), in every one of them.
template <int kCount>
__device__ __forceinline__ Stat join_lanes(Stat s, double inv_tau) {
  float m = s.m;
#pragma unroll
  for (int o = kCount / 2; o > 0; o >>= 1) m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, o));
  if (s.d != 0.0 && s.m != m) s.d *= exp(((double)s.m - (double)m) * inv_tau);
#pragma unroll
  for (int o = kCount / 2; o > 0; o >>= 1) s.d += __shfl_xor_sync(0xffffffffu, s.d, o);
  return Stat{m, s.d};
}

// The scalars of a live row.  The target's own term is added in 64 bits: where it dominates, nothing of the small rest is lost to
// its rounding, and 1 - p is the rest's share without a cancellation.  Writes them (`write`) and, for the policy loss, returns the
// coefficient of the cotangent, what to multiply the exponentials by, their reference and the target's entry.
template <typename T, bool kPolicy>
__device__ __forceinline__ float4 conclude(const RowArgs& a, const Stat& t, float zy, const Given& in, int64_t r, bool write) {
  const double d = whole_sum<T>(t.d), above = ((double)zy - (double)t.m) * a.inv_tau, own = exp(above), all = own + d;
  const double logp = own > d ? -log1p(d / own) : above - log(all);
  const float per_sum = 1.f / (float)all, rest = (float)d * per_sum;
  if (!kPolicy) {
    if (write) put_logp(a, r, logp, make_float4(t.m, per_sum, rest, (float)((double)zy * a.inv_tau - logp)));
    return make_float4(0.f, 0.f, 0.f, 0.f);
  }
  const float coef = (float)(policy_scalars(a, in, logp, r, write) * a.inv_tau);
  return make_float4(coef, -coef * per_sum, t.m, coef * rest);
}

// A row that takes no part.
template <bool kPolicy>
__device__ __forceinline__ void conclude_nothing(const RowArgs& a, int64_t r) {
  if (kPolicy) {
    a.loss[r] = 0.f;
    a.kl[r] = 0.f;
    static_cast<float*>(a.logp)[r] = 0.f;
  } else {
    put_logp(a, r, 0.0, make_float4(0.f, 0.f, 0.f, 0.f));
  }
}

// ---- rows held on chip ----------------------------------------------------------------------------
// One CTA per row.  Every thread copies its vectors to shared memory (cp.async, no registers) and is the only one that reads
// them back, so no barrier stands between the copy and the three passes over it: maximum (while later groups of the copy are on
// their way), sum, cotangent.  The row crosses HBM once.
constexpr int kGroups = 4;

__device__ __forceinline__ void copy16(uint32_t dst, const void* src) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(dst), "l"(src) : "memory");
}
__device__ __forceinline__ void copy_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int kLeft>
__device__ __forceinline__ void copy_wait() { asm volatile("cp.async.wait_group %0;" ::"n"(kLeft) : "memory"); }

template <typename T>
__device__ __forceinline__ Vec<T> from_shared(uint32_t at) {
  const uint4 q = dev::lds128(at);
  Vec<T> x;
  x.w[0] = q.x; x.w[1] = q.y; x.w[2] = q.z; x.w[3] = q.w;
  return x;
}

template <typename T>
__device__ __forceinline__ float vec_max(const Vec<T>& x, float m) {
  if constexpr (sizeof(T) == 2) {
    __nv_bfloat162 h[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) h[i] = *reinterpret_cast<const __nv_bfloat162*>(&x.w[i]);
    const __nv_bfloat162 t = __hmax2(__hmax2(h[0], h[1]), __hmax2(h[2], h[3]));
    return fmaxf(m, fmaxf(__low2float(t), __high2float(t)));
  } else {
#pragma unroll
    for (int i = 0; i < 4; ++i) m = fmaxf(m, x.get(i));
    return m;
  }
}

constexpr int kHeldThreads = 128;

template <typename T, bool kPolicy>
__global__ void __launch_bounds__(kHeldThreads, 8) held_kernel(const T* logits, int64_t ld, RowArgs a, T* out, int64_t ld_out) {
  constexpr int kWarps = kHeldThreads / 32, kStep = kHeldThreads * 16;
  extern __shared__ __align__(16) uint8_t held[];
  __shared__ Stat warp_stat[kWarps];
  __shared__ float4 bcast;
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int64_t r = blockIdx.x, y = a.target[r];
  const Row<T> row(logits + r * ld, a.V);
  T* const o = kPolicy ? out + r * ld_out : nullptr;
  const bool wide = kPolicy && same_alignment(row.x, (const T*)o);
  bool live = target_ok(y, a, threadIdx.x == 0);
  Given in{1.f, 0.f, 0.f, 0.f};
  if (kPolicy) {
    in = given(a, r);
    live = live && in.weight != 0.f;
  }
  if (!live) {
    if (threadIdx.x == 0) conclude_nothing<kPolicy>(a, r);
    if (kPolicy)
      for (int v = threadIdx.x; v < row.nvec; v += kHeldThreads) row.store(o, v, zeros<T>(), wide);
    return;
  }

  // this thread's vectors: threadIdx.x + i * kHeldThreads, i < n, at mine + i * kStep
  const int n = row.nvec > (int)threadIdx.x ? (row.nvec - 1 - (int)threadIdx.x) / kHeldThreads + 1 : 0;
  const uint32_t mine = dev::smem_u32(held) + threadIdx.x * 16;
  const int group = (row.nvec + kHeldThreads * kGroups - 1) / (kHeldThreads * kGroups);
  const T* const base = row.x - row.shift;          // vector v lies at base + v * N
#pragma unroll
  for (int g = 0; g < kGroups; ++g) {
    const int stop = min(n, (g + 1) * group);
#pragma unroll 4
    for (int i = g * group; i < stop; ++i) {
      const int v = threadIdx.x + i * kHeldThreads;
      const uint32_t at = mine + i * kStep;
      if (row.full(v)) {
        copy16(at, base + (int64_t)v * Row<T>::N);
      } else {
        const Vec<T> x = row.load(v);
        dev::sts128(at, x.w[0], x.w[1], x.w[2], x.w[3]);
      }
    }
    copy_commit();
  }
  const float zy = to_float(row.x[y]);
  float m = fmaxf(kLowest, zy);
  auto max_of = [&](int g) {
    const int stop = min(n, (g + 1) * group);
#pragma unroll 4
    for (int i = g * group; i < stop; ++i) m = vec_max(from_shared<T>(mine + i * kStep), m);
  };
  copy_wait<3>(); max_of(0);
  copy_wait<2>(); max_of(1);
  copy_wait<1>(); max_of(2);
  copy_wait<0>(); max_of(3);
#pragma unroll
  for (int s = 16; s > 0; s >>= 1) m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, s));

  // the target's term is added in the end
  const int vy = (int)((y + row.shift) / Row<T>::N);
  const bool writer = vy % kHeldThreads == threadIdx.x;
  if (writer) {
    const uint32_t at = mine + vy / kHeldThreads * kStep;
    Vec<T> x = from_shared<T>(at);
    x.take_out((int)((y + row.shift) % Row<T>::N));
    dev::sts128(at, x.w[0], x.w[1], x.w[2], x.w[3]);
  }
  // Every warp sums against its own maximum, so no barrier comes first.  The terms of two vectors are summed in 32 bits,
  // everything above them in 64.
  const Scale c = a.c;
  double d = 0.0;
  {
    const F2 minus_m = f2(-m, -m);
    int i = 0;
#pragma unroll 2
    for (; i + 1 < n; i += 2)
      d += (double)sum_of(exp_sum(from_shared<T>(mine + i * kStep), minus_m, c) + exp_sum(from_shared<T>(mine + (i + 1) * kStep), minus_m, c));
    if (i < n) d += (double)sum_of(exp_sum(from_shared<T>(mine + i * kStep), minus_m, c));
  }
#pragma unroll
  for (int s = 16; s > 0; s >>= 1) d += __shfl_xor_sync(0xffffffffu, d, s);
  if (lane == 0) warp_stat[warp] = Stat{m, d};
  __syncthreads();
  if (warp == 0) {
    const Stat t = join_lanes<kWarps>(lane < kWarps ? warp_stat[lane] : Stat{kLowest, 0.0}, a.inv_tau);
    if (lane == 0) bcast = conclude<T, kPolicy>(a, t, zy, in, r, true);
  }
  if (!kPolicy) return;
  __syncthreads();
  const float4 b = bcast;
  if (b.x == 0.f) {                           // clipped: nothing of the row is wanted
    for (int i = 0; i < n; ++i) row.store(o, threadIdx.x + i * kHeldThreads, zeros<T>(), wide);
    return;
  }
  const F2 factor = f2(b.y, b.y), minus_m = f2(-b.z, -b.z);
  T* const to = o - row.shift;
#pragma unroll 2
  for (int i = 0; i < n; ++i) {
    const int v = threadIdx.x + i * kHeldThreads;
    const Vec<T> g = scaled_exp(from_shared<T>(mine + i * kStep), minus_m, factor, c);
    if (wide && row.full(v)) __stcs(reinterpret_cast<uint4*>(to + (int64_t)v * Row<T>::N), make_uint4(g.w[0], g.w[1], g.w[2], g.w[3]));
    else row.store(o, v, g, wide);
  }
  if (writer) o[y] = from_float<T>(b.w);      // its writer puts the target's entry right
}

// ---- short rows --------------------------------------------------------------------------------------
// One warp per row, kVecs vectors of it in every lane's registers: no barrier, and the scalars of the rows that share an SM
// overlap.
constexpr int kShortWarps = 4;
template <typename T, int kVecs, bool kPolicy>
__global__ void __launch_bounds__(kShortWarps * 32) short_kernel(const T* logits, int64_t ld, RowArgs a, T* out, int64_t ld_out, int64_t rows) {
  const int lane = threadIdx.x & 31;
  const int64_t r = (int64_t)blockIdx.x * kShortWarps + (threadIdx.x >> 5);
  if (r >= rows) return;
  const int64_t y = a.target[r];
  const Row<T> row(logits + r * ld, a.V);
  T* const o = kPolicy ? out + r * ld_out : nullptr;
  const bool wide = kPolicy && same_alignment(row.x, (const T*)o);
  bool live = target_ok(y, a, lane == 0);
  Given in{1.f, 0.f, 0.f, 0.f};
  if (kPolicy) {
    in = given(a, r);
    live = live && in.weight != 0.f;
  }
  if (!live) {
    if (lane == 0) conclude_nothing<kPolicy>(a, r);
    if (kPolicy)
      for (int v = lane; v < row.nvec; v += 32) row.store(o, v, zeros<T>(), wide);
    return;
  }
  Vec<T> x[kVecs];
  float m = kLowest;
#pragma unroll
  for (int i = 0; i < kVecs; ++i) {
    const int v = lane + i * 32;
    if (v < row.nvec) x[i] = row.load(v);
    else x[i].set_nothing();
  }
  const float zy = to_float(row.x[y]);
  const int vy = (int)((y + row.shift) / Vec<T>::N), jy = (int)((y + row.shift) % Vec<T>::N);
#pragma unroll
  for (int i = 0; i < kVecs; ++i) m = vec_max(x[i], m);
#pragma unroll
  for (int s = 16; s > 0; s >>= 1) m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, s));
  // the target's term is added in the end: -inf in its place, by masks made once (x is in registers, whose index must be static)
  Vec<T> keep, put = zeros<T>();
#pragma unroll
  for (int i = 0; i < 4; ++i) keep.w[i] = ~0u;
  put.take_out(jy);
  if (sizeof(T) == 2) {
#pragma unroll
    for (int i = 0; i < 4; ++i) keep.w[i] = put.w[i] >> 16 ? 0xFFFFu : put.w[i] ? 0xFFFF0000u : ~0u;
  } else {
#pragma unroll
    for (int i = 0; i < 4; ++i) keep.w[i] = put.w[i] ? 0u : ~0u;
  }
  double d = 0.0;
#pragma unroll
  for (int i = 0; i < kVecs; ++i) {
    if (lane + i * 32 == vy) {
#pragma unroll
      for (int k = 0; k < 4; ++k) x[i].w[k] = (x[i].w[k] & keep.w[k]) | put.w[k];
    }
    x[i].packed_again();
    d += (double)sum_of(exp_sum(x[i], f2(-m, -m), a.c));
  }
#pragma unroll
  for (int s = 16; s > 0; s >>= 1) d += __shfl_xor_sync(0xffffffffu, d, s);
  const float4 b = conclude<T, kPolicy>(a, Stat{m, d}, zy, in, r, lane == 0);
  if constexpr (kPolicy) {
#pragma unroll
    for (int i = 0; i < kVecs; ++i) {
      const int u = lane + i * 32;
      x[i].packed_again();
      if (u < row.nvec) row.store(o, u, b.x == 0.f ? zeros<T>() : scaled_exp(x[i], f2(-m, -m), f2(b.y, b.y), a.c), wide);
    }
    if (b.x != 0.f && vy % 32 == lane) o[y] = from_float<T>(b.w);      // its writer puts the target's entry right
  }
}

// ---- rows in a pipeline ------------------------------------------------------------------------------
// Clusters that stay and go from row to row, two CTAs on every SM (two whose phases differ keep memory and the special-function
// unit busier than one of twice the size: 1024 x 248320 bf16 in 218 against 233 us).  12 warps work, three on each scheduler, two
// more do everything that is latency (207 us; with 13 workers 211, with 8 209, with 16, at 56 registers a thread, 219).  For every row k:
//   the first of them reads 128 samples and the target's logit, and publishes their maximum as the row's reference: a sum of
//     exponentials needs no maximum, only a number near it, so the workers need no pass for one and their sums simply add up;
//   S(k): the workers' sums of exp((z - reference)/tau) over everything but the target, one number per warp.  A warp whose sum
//     says that a logit of its own lies far above the reference (more than 14 log2 units: the exponent would be rounded too
//     coarsely there, and overflow at 128) sums once more, against its own maximum;
//   the first warp adds them up and sends the CTA's share to the others of the cluster (asynchronous remote stores that count on
//     their barrier); the second adds the shares, finishes the row's scalars and lets the workers know;
//   G(k), the policy loss's cotangent, `lead` rows after S(k): the workers never wait for the exchange.
// Policy loss: a CTA holds `slots` slices of rows.  A warp's vectors are its own: it fetches them (one bulk copy per row, issued
// by one lane: as 16-byte copies of every lane they took the load-store unit as long as the arithmetic), reads them in S and in G,
// and fetches those of the row `slots` further on into the same place.  One copy per CTA and row, by a warp that waits until all
// are done with the slot, 240 against 219 us; a slice that passes twice, the second time from L2, 233 us.
//   Bound: two exponentials per logit at 16 per cycle and SM (126 us of the 207), then HBM (155 us); the two overlap only between
//   CTAs.  Replacing one exponential in four by a polynomial on the fp32 pipe was slower (231 us): the loops issue 12 instructions
//   per logit, and the polynomial adds six to every one that it replaces.
//   fp32 logits: an exponential has as many bits as its logit, takes its place in S, and G only scales it (2000 x 16000: 62 against
//   68 us).  A bf16 logit's place is too small for it: a cotangent that is rounded twice is not what the type can hold.
// Log-probabilities: nothing is wanted twice, so a slice passes through the slots in chunks of kTurns vectors a lane, which a warp
// of its own copies, 54 KB at a time (a bulk copy costs some 40 ns beside its bytes: with 4 KB copies by every warp 105 us in
// place of 89, 1024 x 248320 bf16 with a tenth of the rows left out).
//   Bound: HBM (70 us; the same kernel without its arithmetic takes 6 us less).
// All waits are bounded; a CTA whose wait ran out stops working, and all CTAs of a cluster leave together.
constexpr int kWorkerWarps = 12, kWorkers = kWorkerWarps * 32, kRing = 8, kMaxCluster = 10, kMaxLead = 3, kAhead = 7, kInfo = 16, kSamples = 4;
constexpr int kMaxSlots = 2;                                             // policy loss
constexpr int kStages = 2, kTurns = 9, kChunk = kWorkers * kTurns;       // log-probabilities

struct Share { float m, unused; double d; };       // what a CTA sends: its sum and what it is against (16 bytes: one store)

__device__ __forceinline__ bool wait_cluster(uint32_t bar, uint32_t parity, volatile int* abort_flag, int* status, int where) {
  for (uint32_t spin = 0; spin < B2G_SPIN_LIMIT; ++spin) {
    uint32_t ok;
    asm volatile(
        "{\n\t.reg .pred p;\n\t"
        "mbarrier.try_wait.parity.acquire.cluster.shared::cta.b64 p, [%1], %2;\n\t"
        "selp.u32 %0, 1, 0, p;\n\t}"
        : "=r"(ok)
        : "r"(bar), "r"(parity)
        : "memory");
    if (ok) return true;
    if ((spin & 255u) == 255u && *abort_flag) return false;
  }
  *abort_flag = 1;
  if (status) atomicCAS(status, 0, where);
  return false;
}
__device__ __forceinline__ void send_share(uint32_t to, uint32_t bar, const Share& s) {
  const uint64_t lo = __float_as_uint(s.m), hi = (uint64_t)__double_as_longlong(s.d);
  asm volatile("st.async.weak.shared::cluster.mbarrier::complete_tx::bytes.v2.b64 [%0], {%1, %2}, [%3];" ::"r"(to), "l"(lo), "l"(hi), "r"(bar)
               : "memory");
}
// The first and the last vector of a row, where they are partial: out of line, they are few.
template <typename T>
__device__ __noinline__ void fetch_edge(const T* x, int64_t V, int v, uint32_t at) {
  const Vec<T> w = Row<T>(x, V).load(v);
  dev::sts128(at, w.w[0], w.w[1], w.w[2], w.w[3]);
}
template <typename T>
__device__ __noinline__ void store_edge(const T* x, int64_t V, int v, T* out, Vec<T> w) { Row<T>(x, V).store(out, v, w, false); }

// A row's part of one warp: vectors [begin, end), of which those in [full_begin, full_end) are whole; lane l reads begin + l + 32 i,
// i < n.  Rows whose pitch is a multiple of 16 bytes all have the same one.
template <typename T>
struct Part {
  static constexpr int N = Vec<T>::N;
  int shift, full_begin, full_end, end, n;
  __device__ __forceinline__ Part(const T* x, uint32_t V, int begin, int limit, int lane) {
    shift = (int)((uint32_t)reinterpret_cast<uintptr_t>(x) & 15u) / (int)sizeof(T);
    const uint32_t width = V + shift;
    full_begin = max(begin, shift != 0 ? 1 : 0);
    end = min(limit, (int)((width + N - 1) / N));
    full_end = min(end, (int)(width / N));
    n = end > begin + lane ? (end - 1 - begin - lane) / 32 + 1 : 0;
  }
  __device__ __forceinline__ bool full(int v) const { return v >= full_begin && v < full_end; }
  // One lane: the whole vectors as one bulk copy that counts on `bar`, the partial ones by hand.  `at`: place of vector `begin`.
  __device__ __forceinline__ void fetch(const T* x, int begin, uint32_t at, uint32_t bar, int64_t V) const {
    const int whole = max(0, full_end - full_begin);
    for (int v = begin; v < min(full_begin, end); ++v) fetch_edge(x, V, v, at + (v - begin) * 16);
    for (int v = max(full_end, full_begin); v < end; ++v) fetch_edge(x, V, v, at + (v - begin) * 16);
    dev::mbar_arrive_expect_tx(bar, (uint32_t)whole * 16);
    if (whole)
      asm volatile("cp.async.bulk.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1], %2, [%3];" ::"r"(at + (full_begin - begin) * 16),
                   "l"(x - shift + (int64_t)full_begin * N), "r"(whole * 16), "r"(bar)
                   : "memory");
  }
  // index i of this lane's vector that holds column y, or -1
  __device__ __forceinline__ int owns(int y, int begin, int lane) const {
    const int v = (int)((uint32_t)(y + shift) / N), k = v - begin - lane;
    return k >= 0 && v < end && k % 32 == 0 ? k / 32 : -1;
  }
};

// What the workers need to know of a row: what to sum against, and its target, or -1 where it takes no part.
struct Info { float reference; int y; };

constexpr double kFarAbove = 16384.0;      // 2^14
// A lane's sum over its n vectors in shared memory, kStep bytes apart, and the warp's.  kKeep: 32-bit exponentials take the places
// of their logits.
template <typename T, int kStep, bool kKeep = false>
__device__ __forceinline__ double lane_sum_against(uint32_t place, int n, float ref, const Scale& c) {
  if constexpr (kKeep) {
    static_assert(sizeof(T) == 4, "an exponential needs as many bits as its logit has");
    F2 sum = f2(0.f, 0.f);
    float lo, hi;
#pragma unroll 2
    for (int i = 0; i < n; ++i) {
      const Vec<T> x = from_shared<T>(place + i * kStep);
      const F2 m = f2(-ref, -ref), e = exp_from<T, true>(x.pair(0), m, c), f = exp_from<T, true>(x.pair(1), m, c);
      sum = sum + (e + f);
      float w[4];
      split(e, w[0], w[1]);
      split(f, w[2], w[3]);
      dev::sts128(place + i * kStep, __float_as_uint(w[0]), __float_as_uint(w[1]), __float_as_uint(w[2]), __float_as_uint(w[3]));
    }
    split(sum, lo, hi);
    return (double)lo + (double)hi;
  }
  const F2 minus_ref = f2(-ref, -ref);
  F2 d = f2(0.f, 0.f);
  int i = 0;
#pragma unroll 4
  for (; i + 1 < n; i += 2)
    d = d + (exp_sum(from_shared<T>(place + i * kStep), minus_ref, c) + exp_sum(from_shared<T>(place + (i + 1) * kStep), minus_ref, c));
  if (i < n) d = d + exp_sum(from_shared<T>(place + i * kStep), minus_ref, c);
  float lo, hi;
  split(d, lo, hi);
  return (double)lo + (double)hi;
}
__device__ __forceinline__ double warp_total(double d) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) d += __shfl_xor_sync(0xffffffffu, d, o);
  return d;
}
template <typename T, int kStep, bool kKeep = false>
__device__ __forceinline__ double warp_sum_against(uint32_t place, int n, float ref, const Scale& c) {
  return warp_total(lane_sum_against<T, kStep, kKeep>(place, n, ref, c));
}
// The same against its own maximum; out of line, it is rare.
template <typename T, int kStep, bool kKeep = false>
__device__ __noinline__ Stat warp_sum_far(uint32_t place, int n, Scale c) {
  float m = kLowest;
  for (int i = 0; i < n; ++i) m = vec_max(from_shared<T>(place + i * kStep), m);
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, o));
  return Stat{m, warp_sum_against<T, kStep, kKeep>(place, n, m, c)};
}
// Logits that their exponentials have replaced, from memory once more: vectors v, v + 32, ... of a row.
template <typename T, int kStep>
__device__ __noinline__ void fetch_again(const T* x, int64_t V, int v, uint32_t place, int n) {
  const Row<T> row(x, V);
  for (int i = 0; i < n; ++i) {
    const Vec<T> w = row.load(v + i * 32);
    dev::sts128(place + i * kStep, w.w[0], w.w[1], w.w[2], w.w[3]);
  }
}

__device__ __forceinline__ Stat join_two(Stat a, Stat b, double inv_tau) {
  const float m = fmaxf(a.m, b.m);
  if (a.d != 0.0 && a.m != m) a.d *= exp(((double)a.m - (double)m) * inv_tau);
  if (b.d != 0.0 && b.m != m) b.d *= exp(((double)b.m - (double)m) * inv_tau);
  return Stat{m, a.d + b.d};
}
// -inf in place of value j of the vector at `at`
template <typename T>
__device__ __forceinline__ void hide(uint32_t at, int j) {
  if (sizeof(T) == 2) asm volatile("st.shared.u16 [%0], %1;" ::"r"(at + j * 2), "h"((unsigned short)0xFF80) : "memory");
  else asm volatile("st.shared.u32 [%0], %1;" ::"r"(at + j * 4), "r"(0xFF800000u) : "memory");
}
// A wait has run out: the copies that are still on their way have nowhere to go once the CTA has left.
__device__ __noinline__ void drain(uint32_t bar, uint32_t parity) {
  for (uint32_t spin = 0; spin < (1u << 16) && !dev::mbar_try_wait(bar, parity); ++spin) {}
}

template <bool kPolicy>
constexpr int kPipeThreads = kWorkers + (kPolicy ? 64 : 96);      // two CTAs of either fit an SM's registers: 72 and 64 a thread

template <typename T, bool kPolicy>
__global__ void __launch_bounds__(kPipeThreads<kPolicy>, 2) pipe_kernel(const T* logits, int64_t ld, RowArgs a, T* out, int64_t ld_out, int64_t rows,
                                                                int cluster, int slots, int lead, int per) {
  constexpr int N = Vec<T>::N, kStep = 32 * 16;
  constexpr bool kKeep = kPolicy && sizeof(T) == 4;      // G finds the exponentials of S in the logits' places
  extern __shared__ __align__(16) uint8_t space[];
  // policy loss: one per slot and warp, whose copies are its own; log-probabilities: one per slot, and every warp is done with it
  constexpr int kPlaces = kPolicy ? kMaxSlots : kStages, kOwners = kPolicy ? kWorkerWarps : 1;
  __shared__ uint64_t arrived[kPlaces][kOwners], emptied[kPlaces];
  __shared__ __align__(16) Share share[kRing][kMaxCluster];
  __shared__ Stat sums[kRing][kWorkerWarps];
  __shared__ __align__(8) Info info[kInfo];
  __shared__ float known[kInfo];                 // the target's logit
  __shared__ float4 bcast[kRing];
  __shared__ uint64_t referred[kInfo], summed[kRing], joined[kRing], ready[kRing];
  __shared__ int gave_up;
  const int rank = blockIdx.x % cluster, lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int64_t first = blockIdx.x / cluster, stride = gridDim.x / cluster;
  const int count = (int)((rows - first + stride - 1) / stride);       // rows of this cluster: first + k * stride
  if (threadIdx.x == 0) {
    gave_up = 0;
    for (int i = 0; i < kInfo; ++i) dev::mbar_init(dev::smem_u32(&referred[i]), 1);
    for (int i = 0; i < kPlaces * kOwners; ++i) dev::mbar_init(dev::smem_u32(&arrived[i / kOwners][i % kOwners]), 1);
    for (int i = 0; i < kPlaces; ++i) dev::mbar_init(dev::smem_u32(&emptied[i]), kWorkerWarps);
    for (int i = 0; i < kRing; ++i) {
      dev::mbar_init(dev::smem_u32(&summed[i]), kWorkerWarps);
      dev::mbar_init(dev::smem_u32(&joined[i]), 1);
      dev::mbar_init(dev::smem_u32(&ready[i]), 1);
    }
    dev::fence_barrier_init();
  }
  dev::cluster_sync_all();          // nobody sends to a barrier that is not there yet

  if (warp == kWorkerWarps) {       // references, and the CTA's share
    const int64_t apart = a.V / (32 * kSamples);
    float sample[kSamples], target_logit = 0.f;
    int y_ahead = -1;
    // the target and weight of the row after the one that is looked at, so that its logit's address is at hand in time
    int64_t target_next = a.target[first];
    float weight_next = kPolicy && a.weight ? a.weight[first] : 1.f;
    auto look_at = [&](int k) {     // issue the loads of row k's reference
      if (k >= count) return;
      const int64_t r = first + k * stride, y = target_next;
      const T* x = logits + r * ld;
#pragma unroll
      for (int i = 0; i < kSamples; ++i) sample[i] = to_float(x[(lane * kSamples + i) * apart]);
      const bool in_range = y >= 0 && y < a.V;
      target_logit = in_range ? to_float(x[y]) : -INFINITY;
      y_ahead = in_range && y != a.ignore_index && weight_next != 0.f ? (int)y : -1;
      if (k + 1 < count) {
        target_next = a.target[r + stride];
        if (kPolicy && a.weight) weight_next = a.weight[r + stride];
      }
    };
    auto refer = [&](int k) {
      if (k >= count) return;
      float m = fmaxf(kLowest, target_logit);
#pragma unroll
      for (int i = 0; i < kSamples; ++i) m = fmaxf(m, sample[i]);
#pragma unroll
      for (int o = 16; o > 0; o >>= 1) m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, o));
      if (lane == 0) {
        info[k % kInfo] = Info{m, y_ahead};
        known[k % kInfo] = target_logit;
        dev::mbar_arrive(dev::smem_u32(&referred[k % kInfo]));
      }
    };
    for (int k = 0; k < kAhead; ++k) {
      look_at(k);
      refer(k);
    }
    for (int k = 0; k < count; ++k) {
      const int p = k % kRing, parity = (k / kRing) & 1;
      look_at(k + kAhead);
      if (!dev::mbar_wait(dev::smem_u32(&summed[p]), parity, &gave_up, a.status, 501)) break;
      // of a row that takes no part nobody looks at it
      const Stat t = join_lanes<32>(lane < kWorkerWarps ? sums[p][lane] : Stat{kLowest, 0.0}, a.inv_tau);
      if (lane < cluster)
        send_share(dev::map_to_cta(dev::smem_u32(&share[p][rank]), lane), dev::map_to_cta(dev::smem_u32(&joined[p]), lane), Share{t.m, 0.f, t.d});
      refer(k + kAhead);
    }
  } else if (warp == kWorkerWarps + 1) {       // the row's scalars
    int64_t target_next = a.target[first];
    Given given_next{1.f, 0.f, 0.f, 0.f};
    if (kPolicy) given_next = given(a, first);
    for (int k = 0; k < count; ++k) {
      const int64_t r = first + k * stride, y = target_next;
      const Given in = given_next;
      if (k + 1 < count) {
        target_next = a.target[r + stride];
        if (kPolicy) given_next = given(a, r + stride);
      }
      const int p = k % kRing, parity = (k / kRing) & 1;
      const uint32_t bar = dev::smem_u32(&joined[p]);
      if (lane == 0) dev::mbar_arrive_expect_tx(bar, cluster * (uint32_t)sizeof(Share));
      const bool live = target_ok(y, a, rank == 0 && lane == 0) && in.weight != 0.f;
      if (!wait_cluster(bar, parity, &gave_up, a.status, 502)) break;
      if (live) {
        const Stat sum = join_lanes<32>(lane < cluster ? Stat{share[p][lane].m, share[p][lane].d} : Stat{kLowest, 0.0}, a.inv_tau);
        if (lane == 0) {
          const float4 b = conclude<T, kPolicy>(a, sum, known[k % kInfo], in, r, rank == 0);
          if (kPolicy) bcast[p] = b;
        }
      } else if (rank == 0 && lane == 0) {
        conclude_nothing<kPolicy>(a, r);
      }
      __syncwarp();
      if (lane == 0) dev::mbar_arrive(dev::smem_u32(&ready[p]));
    }
  } else if (!kPolicy && warp == kWorkerWarps + 2) {       // the copies
    const int begin = rank * per, limit = begin + per, chunks = (per + kChunk - 1) / kChunk;
    const T* x = logits + first * ld;
    uint32_t turn = 0u, slot = 0u;             // times round the slots, and slots filled in this one
    bool fine = true;
    for (int k = 0; k < count && fine; ++k, x += stride * ld) {
      // the first chunks are fetched before anybody knows whether their rows take part: a call of few rows is all latency
      bool live = true;
      if (turn) {
        fine = dev::mbar_wait(dev::smem_u32(&referred[k % kInfo]), (k / kInfo) & 1, &gave_up, a.status, 504);
        live = fine && info[k % kInfo].y >= 0;
      }
      for (int i = 0; i < chunks && fine; ++i) {
        if (turn) fine = dev::mbar_wait(dev::smem_u32(&emptied[slot]), (turn - 1u) & 1u, &gave_up, a.status, 505);
        if (!fine) break;
        if (lane == 0) {
          const uint32_t bar = dev::smem_u32(&arrived[slot][0]);
          const int from = begin + i * kChunk;
          dev::fence_proxy_async_smem();       // of partial vectors that stood in the slot
          if (live) Part<T>(x, (uint32_t)a.V, from, min(limit, from + kChunk), 0).fetch(x, from, dev::smem_u32(space) + slot * (kChunk * 16), bar, a.V);
          else dev::mbar_arrive(bar);
        }
        __syncwarp();
        if (++slot == kStages) { slot = 0u; ++turn; }
      }
    }
    if (gave_up)
      for (uint32_t i = 0; i < kStages; ++i)       // the last time round that filled slot i
        if (turn || i < slot) drain(dev::smem_u32(&arrived[i][0]), (i < slot ? turn : turn - 1u) & 1u);
  } else if constexpr (!kPolicy) {
    constexpr int kTurn = kWorkers * 16;
    const int begin = rank * per, limit = begin + per, mine = warp * 32 + lane;      // every kWorkers-th vector of a chunk from `mine` on
    const uint32_t base = dev::smem_u32(space) + mine * 16;
    const Scale c = a.c;
    const T* x = logits + first * ld;
    uint32_t slot = 0u, parity = 0u;
    bool fine = true;
    for (int k = 0; k < count && fine; ++k, x += stride * ld) {
      fine = dev::mbar_wait(dev::smem_u32(&referred[k % kInfo]), (k / kInfo) & 1, &gave_up, a.status, 504);
      if (!fine) break;
      const Info row = info[k % kInfo];
      const Part<T> part(x, (uint32_t)a.V, begin, limit, 0);
      const int owner = row.y >= 0 ? (int)((uint32_t)(row.y + part.shift) / N) : -1;      // the vector that holds the target
      double d = 0.0;
      Stat far{kLowest, 0.0};
      for (int from = begin; from < limit; from += kChunk) {
        fine = dev::mbar_wait(dev::smem_u32(&arrived[slot][0]), parity, &gave_up, a.status, 506);
        if (!fine) break;
        if (row.y >= 0) {
          const uint32_t place = base + slot * (kChunk * 16);
          const int at = owner - from - mine;           // the target's term is the scalar warp's
          if (at >= 0 && at < kChunk && at % kWorkers == 0 && owner < limit) hide<T>(place + at * 16, (row.y + part.shift) % N);
          const int left = part.end - from - mine, n = left > 0 ? min(kTurns, (left - 1) / kWorkers + 1) : 0;
          const double one = lane_sum_against<T, kTurn>(place, n, row.reference, c);
          if (__any_sync(0xffffffffu, !(one < kFarAbove))) far = join_two(far, warp_sum_far<T, kTurn>(place, n, c), a.inv_tau);
          else d += one;
          dev::fence_proxy_async_smem();                // the next copy into the slot comes after what has been done in it
        }
        __syncwarp();
        if (lane == 0) dev::mbar_arrive(dev::smem_u32(&emptied[slot]));
        if (++slot == kStages) { slot = 0u; parity ^= 1u; }
      }
      if (!fine) break;
      if (row.y >= 0) {
        Stat sum{row.reference, warp_total(d)};
        if (far.d != 0.0) sum = join_two(sum, far, a.inv_tau);
        if (lane == 0) sums[k % kRing][warp] = sum;
      }
      __syncwarp();
      if (lane == 0) dev::mbar_arrive(dev::smem_u32(&summed[k % kRing]));
      // the rings bound how far the workers run ahead
      const int j = k - kMaxLead;
      if (j >= 0) fine = dev::mbar_wait(dev::smem_u32(&ready[j % kRing]), (j / kRing) & 1, &gave_up, a.status, 503);
    }
  } else {
    // whole turns of 32 vectors, dealt out as evenly as they can be
    const int turns = (per + 31) / 32, from = warp * turns / kWorkerWarps * 32, to = (warp + 1) * turns / kWorkerWarps * 32;
    const int begin = rank * per + from, limit = rank * per + min(per, to), slot_bytes = per * 16;
    const uint32_t base = dev::smem_u32(space) + from * 16, V = (uint32_t)a.V;
    const Scale c = a.c;
    const bool steady = (ld * (int64_t)sizeof(T)) % 16 == 0;
    const T* const x0 = logits + first * ld;
    const int64_t pitch = stride * ld;
    Part<T> part(x0, V, begin, limit, lane);            // of the row at hand
    auto look_up = [&](int k) { return info[k % kInfo]; };
    auto wait_for = [&](int k) { return dev::mbar_wait(dev::smem_u32(&referred[k % kInfo]), (k / kInfo) & 1, &gave_up, a.status, 504); };
    uint32_t phase = 0u;            // bit i: parity of the next arrival in slot i
    float against[kMaxSlots] = {0.f, 0.f};       // what this warp's exponentials in a slot were taken against
    // the first rows are fetched before anybody knows whether they take part: a call of few rows is all latency
    for (int k = 0; k < min(slots, count); ++k) {
      const T* const x = x0 + k * pitch;
      if (!steady) part = Part<T>(x, V, begin, limit, lane);
      if (lane == 0) part.fetch(x, begin, base + k * slot_bytes, dev::smem_u32(&arrived[k][warp]), a.V);
      __syncwarp();
    }
    int s_slot = 0, g_slot = 0;
    for (int k = 0; k < count + lead; ++k) {
      const int j = k - lead, q = j + slots;      // G's row, and the row that takes the place freed in this turn
      int slot = s_slot;                          // the place at hand
      if (k < count) {
        const int p = k % kRing;
        if (k < slots && !wait_for(k)) break;
        const Info row = look_up(k);
        if (row.y >= 0 || k < slots) {
          if (!dev::mbar_wait(dev::smem_u32(&arrived[s_slot][warp]), phase >> s_slot & 1u, &gave_up, a.status, 506)) break;
          phase ^= 1u << s_slot;
          __syncwarp();                                 // partial vectors are lane 0's ordinary stores
        }
        if (row.y >= 0) {
          if (!steady) part = Part<T>(x0 + k * pitch, V, begin, limit, lane);
          const uint32_t place = base + s_slot * slot_bytes + lane * 16;
          const int mine = part.owns(row.y, begin, lane);
          auto hide_mine = [&] { if (mine >= 0) hide<T>(place + mine * kStep, (row.y + part.shift) % N); };
          hide_mine();                                  // the target's term is the scalar warp's
          Stat mine_sum{row.reference, warp_sum_against<T, kStep, kKeep>(place, part.n, row.reference, c)};
          if (!(mine_sum.d < kFarAbove)) {
            if (kKeep) {
              fetch_again<T, kStep>(x0 + k * pitch, a.V, begin + lane, place, part.n);
              hide_mine();
            }
            mine_sum = warp_sum_far<T, kStep, kKeep>(place, part.n, c);
          }
          if (lane == 0) sums[p][warp] = mine_sum;
          if (s_slot == 0) against[0] = mine_sum.m;
          else against[1] = mine_sum.m;
        }
        __syncwarp();
        if (lane == 0) dev::mbar_arrive(dev::smem_u32(&summed[p]));
        if (++s_slot == slots) s_slot = 0;
      }

      bool fill = false;
      if (q >= slots && q < count) {
        if (!wait_for(q)) break;
        fill = look_up(q).y >= 0;
      }
      if (j >= 0) {
        const int p = j % kRing;
        if (!dev::mbar_wait(dev::smem_u32(&ready[p]), (j / kRing) & 1, &gave_up, a.status, 503)) break;
        slot = g_slot;
        const int y = look_up(j).y;
        const float4 b = y >= 0 ? bcast[p] : make_float4(0.f, 0.f, 0.f, 0.f);
        const T* const x = x0 + j * pitch;
        T* const o = out + (first + j * stride) * ld_out;
        if (!steady) part = Part<T>(x, V, begin, limit, lane);
        const uint32_t place = base + g_slot * slot_bytes + lane * 16;
        T* const to = o - part.shift;
        const bool wide = same_alignment(x, (const T*)o);
        auto put = [&](int v, const Vec<T>& w) {
          if (wide && part.full(v)) __stcs(reinterpret_cast<uint4*>(to + (int64_t)v * N), make_uint4(w.w[0], w.w[1], w.w[2], w.w[3]));
          else store_edge(x, a.V, v, o, w);
        };
        if (b.x == 0.f) {                     // a clipped token, a row that takes no part: nothing of the logits is wanted
          for (int i = 0; i < part.n; ++i) put(begin + lane + i * 32, zeros<T>());
        } else {
          if constexpr (kKeep) {
            const float own = g_slot == 0 ? against[0] : against[1], f = own == b.z ? b.y : b.y * (float)exp(((double)own - (double)b.z) * a.inv_tau);
            const F2 factor = f2(f, f);
#pragma unroll 2
            for (int i = 0; i < part.n; ++i) put(begin + lane + i * 32, scaled(from_shared<T>(place + i * kStep), factor));
          } else {
            const F2 factor = f2(b.y, b.y), minus_ref = f2(-b.z, -b.z);
            if (wide && part.full_begin == begin && part.full_end == part.end) {
              uint4* const to16 = reinterpret_cast<uint4*>(to) + begin + lane;
#pragma unroll 4
              for (int i = 0; i < part.n; ++i) {
                const Vec<T> w = scaled_exp(from_shared<T>(place + i * kStep), minus_ref, factor, c);
                __stcs(to16 + i * 32, make_uint4(w.w[0], w.w[1], w.w[2], w.w[3]));
              }
            } else {
#pragma unroll 1
              for (int i = 0; i < part.n; ++i) put(begin + lane + i * 32, scaled_exp(from_shared<T>(place + i * kStep), minus_ref, factor, c));
            }
          }
          if (part.owns(y, begin, lane) >= 0) o[y] = from_float<T>(b.w);              // its writer puts the target's entry right
        }
        if (++g_slot == slots) g_slot = 0;
      }
      if (fill) {                               // into the place that this warp is done with
        const T* const x = x0 + q * pitch;
        if (!steady) part = Part<T>(x, V, begin, limit, lane);
        dev::fence_proxy_async_smem();
        __syncwarp();
        if (lane == 0) part.fetch(x, begin, base + slot * slot_bytes, dev::smem_u32(&arrived[slot][warp]), a.V);
        __syncwarp();
      }
    }
    if (gave_up)
      for (int i = 0; i < slots; ++i) drain(dev::smem_u32(&arrived[i][warp]), phase >> i & 1u);
  }
  dev::cluster_sync_all();          // no CTA's memory goes before what was sent to it has come
}

// ---- rows of any width ----------------------------------------------------------------------------
// Policy loss: one CTA per row that reads it three times (maximum, sum, cotangent), vocabularies wider than a cluster's shared
// memory holds.
template <typename T>
__global__ void __launch_bounds__(512) wide_kernel(const T* logits, int64_t ld, RowArgs a, T* out, int64_t ld_out) {
  constexpr int N = Vec<T>::N, kThreads = 512, kWarps = kThreads / 32;
  __shared__ Stat warp_stat[kWarps];
  __shared__ float4 bcast;
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int64_t r = blockIdx.x, y = a.target[r];
  const Row<T> row(logits + r * ld, a.V);
  T* const o = out + r * ld_out;
  const bool wide = same_alignment(row.x, (const T*)o);
  const Given in = given(a, r);
  if (!target_ok(y, a, threadIdx.x == 0) || in.weight == 0.f) {
    if (threadIdx.x == 0) conclude_nothing<true>(a, r);
    for (int v = threadIdx.x; v < row.nvec; v += kThreads) row.store(o, v, zeros<T>(), wide);
    return;
  }
  float m = kLowest;
  for (int v = threadIdx.x; v < row.nvec; v += kThreads) m = vec_max(row.load(v), m);
#pragma unroll
  for (int s = 16; s > 0; s >>= 1) m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, s));
  const Scale c = a.c;
  const float zy = to_float(row.x[y]);
  const int vy = (int)((y + row.shift) / N), jy = (int)((y + row.shift) % N);
  double d = 0.0;
  for (int v = threadIdx.x; v < row.nvec; v += kThreads) {
    Vec<T> x = row.load(v);
    if (v == vy) x.take_out(jy);                // the target's term is added in the end
    d += (double)sum_of(exp_sum(x, f2(-m, -m), c));
  }
#pragma unroll
  for (int s = 16; s > 0; s >>= 1) d += __shfl_xor_sync(0xffffffffu, d, s);
  if (lane == 0) warp_stat[warp] = Stat{m, d};
  __syncthreads();
  if (warp == 0) {
    const Stat t = join_lanes<kWarps>(lane < kWarps ? warp_stat[lane] : Stat{kLowest, 0.0}, a.inv_tau);
    if (lane == 0) bcast = conclude<T, true>(a, t, zy, in, r, true);
  }
  __syncthreads();
  const float4 b = bcast;
  const F2 factor = f2(b.y, b.y), minus_m = f2(-b.z, -b.z);
  for (int v = threadIdx.x; v < row.nvec; v += kThreads)
    row.store(o, v, b.x == 0.f ? zeros<T>() : scaled_exp(row.load(v), minus_m, factor, c), wide);
  if (b.x != 0.f && vy % kThreads == threadIdx.x) o[y] = from_float<T>(b.w);
}

// ---- gradient of the log-probabilities --------------------------------------------------------------
// dz = g (onehot - exp((z - m)/tau)/d)/tau: one pass without a reduction, kBwdVecs vectors per thread.
constexpr int kBwdVecs = 4;
template <typename T, int kBwdThreads>
__global__ void __launch_bounds__(kBwdThreads) logp_bwd_kernel(const T* logits, int64_t ld, RowArgs a, const void* __restrict__ grad_logp, T* out,
                                                               int64_t ld_out, int blocks) {
  constexpr int N = Vec<T>::N;
  const int64_t r = blockIdx.x / blocks, y = a.target[r];
  const int begin = (int)(blockIdx.x % blocks) * kBwdThreads * kBwdVecs;
  const Row<T> row(logits + r * ld, a.V);
  T* const o = out + r * ld_out;
  const bool wide = same_alignment(row.x, (const T*)o);
  const bool live = y != a.ignore_index && y >= 0 && y < a.V;
  float g = 0.f;
  if (live) g = (a.logp64 ? (float)static_cast<const double*>(grad_logp)[r] : static_cast<const float*>(grad_logp)[r]) / a.tau;
  if (g == 0.f) {
    for (int i = 0; i < kBwdVecs; ++i) {
      const int v = begin + i * kBwdThreads + threadIdx.x;
      if (v < row.nvec) row.store(o, v, zeros<T>(), wide);
    }
    return;
  }
  const float4 st = a.stats[r];
  const F2 factor = f2(-g * st.y, -g * st.y), minus_m = f2(-st.x, -st.x);
  Vec<T> x[kBwdVecs];
#pragma unroll
  for (int i = 0; i < kBwdVecs; ++i) {
    const int v = begin + i * kBwdThreads + threadIdx.x;
    if (v < row.nvec) x[i] = row.load(v);
    else x[i].set_nothing();
  }
#pragma unroll
  for (int i = 0; i < kBwdVecs; ++i) {
    const int v = begin + i * kBwdThreads + threadIdx.x;
    if (v < row.nvec) row.store(o, v, scaled_exp(x[i], minus_m, factor, a.c), wide);
  }
  const int at = (int)((y + row.shift) / N) - begin - (int)threadIdx.x;      // its writer puts the target's entry right
  if (at >= 0 && at < kBwdThreads * kBwdVecs && at % kBwdThreads == 0) o[y] = from_float<T>(g * st.z);
}

// ---- preference loss ------------------------------------------------------------------------------
// Latency, not bytes: a pair is a few thousand tokens.  A CTA of 1024 threads per pair, half of it on either sequence, and a
// cluster of up to eight where the sequences are long on average; kAtOnce loads of each array are under way per thread.
constexpr int kPairThreads = 1024, kHalf = kPairThreads / 2, kAtOnce = 4, kPairClusterMax = 8;

// The bounds of sequence s, brought into [0, N]; a bound that had to be moved is reported.
__device__ __forceinline__ void bounds(const int64_t* offsets, int64_t s, int64_t N, int64_t& begin, int64_t& end, int* status) {
  const int64_t b = offsets[s], e = offsets[s + 1];
  begin = b < 0 ? 0 : (b > N ? N : b);
  end = e < begin ? begin : (e > N ? N : e);
  if ((b != begin || e != end) && threadIdx.x % kHalf == 0 && status) atomicCAS(status, 0, 905);
}

__device__ __forceinline__ double log_sigmoid(double u) { return fmin(u, 0.0) - log1p(exp(-fabs(u))); }

template <typename L, typename R>
__global__ void __launch_bounds__(kPairThreads) pair_kernel(const L* __restrict__ logp, const R* __restrict__ ref,
                                                            const int64_t* __restrict__ target, const int64_t* __restrict__ offsets, int64_t N,
                                                            int64_t P, int64_t ignore_index, float beta, float smoothing, int squared, int average,
                                                            float* __restrict__ loss, float* __restrict__ chosen, float* __restrict__ rejected,
                                                            float* __restrict__ coef, int* status, int cluster) {
  constexpr int kHalfWarps = kHalf / 32;
  __shared__ double warp_sum[kPairThreads / 32];
  __shared__ int warp_count[kPairThreads / 32];
  __shared__ double2 part[kPairClusterMax][2];       // of the cluster's first CTA: every CTA's sum and count of either sequence
  const int rank = blockIdx.x % cluster, half = threadIdx.x / kHalf, thread = threadIdx.x % kHalf, lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int64_t p = blockIdx.x / cluster;
  // Another CTA's shared memory may be written only once that CTA has started: all arrive here, and wait before they send.  A CTA
  // with nothing to read comes to its store after two loads.
  dev::cluster_arrive();
  int64_t begin, end;
  bounds(offsets, p + half * P, N, begin, end, status);
  double s = 0.0;                                    // differences and sums in 64 bits
  int n = 0;
  const int64_t step = (int64_t)cluster * kHalf;
  for (int64_t i = begin + (int64_t)rank * kHalf + thread; i < end; i += step * kAtOnce) {
    int64_t y[kAtOnce];
    L l[kAtOnce];
    R f[kAtOnce];
#pragma unroll
    for (int u = 0; u < kAtOnce; ++u) {
      const int64_t at = i + u * step;
      const bool in = at < end;
      y[u] = in ? (target ? target[at] : ~ignore_index) : ignore_index;
      l[u] = in ? logp[at] : (L)0;
      f[u] = in && ref ? ref[at] : (R)0;
    }
#pragma unroll
    for (int u = 0; u < kAtOnce; ++u) {
      if (y[u] != ignore_index) {                    // what stands in ignored places is not looked at
        s += (double)l[u] - (double)f[u];
        ++n;
      }
    }
  }
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) {
    s += __shfl_xor_sync(0xffffffffu, s, o);
    n += __shfl_xor_sync(0xffffffffu, n, o);
  }
  if (lane == 0) { warp_sum[warp] = s; warp_count[warp] = n; }
  __syncthreads();
  dev::cluster_wait();
  if (threadIdx.x < 2) {                             // thread h: sequence h
    double sum = 0.0, count = 0.0;
    for (int i = 0; i < kHalfWarps; ++i) { sum += warp_sum[threadIdx.x * kHalfWarps + i]; count += (double)warp_count[threadIdx.x * kHalfWarps + i]; }
    const uint32_t to = dev::map_to_cta(dev::smem_u32(&part[rank][threadIdx.x]), 0);
    asm volatile("st.shared::cluster.v2.f64 [%0], {%1, %2};" ::"r"(to), "d"(sum), "d"(count) : "memory");
  }
  dev::cluster_sync_all();
  if (rank == 0 && threadIdx.x == 0) {
    double value[2], count[2];
    for (int h = 0; h < 2; ++h) {
      value[h] = count[h] = 0.0;
      for (int i = 0; i < cluster; ++i) { value[h] += part[i][h].x; count[h] += part[i][h].y; }
      count[h] = average ? fmax(count[h], 1.0) : 1.0;
      value[h] /= count[h];
    }
    const double b = beta, gap = value[0] - value[1], u = b * gap, e = smoothing;
    double l, slope;     // slope = d loss / d gap
    if (squared) {
      const double h = gap - 0.5 / b;
      l = h * h;
      slope = 2.0 * h;
    } else {
      l = -(1.0 - e) * log_sigmoid(u);
      if (e > 0.0) l -= e * log_sigmoid(-u);         // a rejected token that cannot occur makes it infinite; without smoothing it is no matter
      slope = b * (e / (1.0 + exp(-u)) - (1.0 - e) / (1.0 + exp(u)));
    }
    loss[p] = (float)l;
    chosen[p] = (float)(b * value[0]);
    rejected[p] = (float)(b * value[1]);
    coef[p] = (float)(slope / count[0]);
    coef[P + p] = (float)(-slope / count[1]);
  }
}

// grad_logp[i] = grad_loss[pair] * coef[sequence] for counted tokens of a sequence, 0 elsewhere.  A thread's first token finds its
// sequence by bisection, in a copy of the offsets on chip where they fit; its others follow from there.
constexpr int kPairBwdThreads = 256, kPairBwdTokens = 4, kOffsetsOnChip = 2049;
template <typename L>
__global__ void __launch_bounds__(kPairBwdThreads) pair_bwd_kernel(const float* __restrict__ grad_loss, const float* __restrict__ coef,
                                                                   const int64_t* __restrict__ target, const int64_t* __restrict__ offsets,
                                                                   L* __restrict__ grad_logp, int64_t N, int64_t P, int64_t ignore_index) {
  __shared__ int64_t on_chip[kOffsetsOnChip];
  const int64_t entries = 2 * P + 1;
  const bool copied = entries <= kOffsetsOnChip;
  if (copied) {
    for (int i = threadIdx.x; i < (int)entries; i += kPairBwdThreads) on_chip[i] = offsets[i];
    __syncthreads();
  }
  const int64_t tile = (int64_t)blockIdx.x * (kPairBwdThreads * kPairBwdTokens);
  int64_t y[kPairBwdTokens];
#pragma unroll
  for (int u = 0; u < kPairBwdTokens; ++u) {
    const int64_t i = tile + u * kPairBwdThreads + threadIdx.x;
    y[u] = i < N && target ? target[i] : ~ignore_index;
  }
  auto offset = [&](int64_t k) { return copied ? on_chip[k] : offsets[k]; };
  int64_t lo = 0;                          // the number of offsets <= i
#pragma unroll
  for (int u = 0; u < kPairBwdTokens; ++u) {
    const int64_t i = tile + u * kPairBwdThreads + threadIdx.x;
    if (i >= N) return;
    // most tiles lie within one sequence
    if (u == 0 || (lo < entries && offset(lo) <= i)) {
      int64_t hi = entries;
      while (lo < hi) {
        const int64_t mid = (lo + hi) >> 1;
        if (offset(mid) <= i) lo = mid + 1;
        else hi = mid;
      }
    }
    float g = 0.f;
    if (lo >= 1 && lo <= 2 * P && y[u] != ignore_index) {
      const int64_t s = lo - 1;
      g = grad_loss[s < P ? s : s - P] * coef[s];
    }
    grad_logp[i] = g;
  }
}

}  // namespace policy
}  // namespace b2g

using namespace b2g;

static int check_rows(const char* what, int dtype, int64_t rows, int64_t V, int64_t ld, float tau) {
  B2G_REQUIRE(dtype == 0 || dtype == 1, "%s: logits_dtype must be 0 (bf16) or 1 (fp32)", what);
  B2G_REQUIRE(rows >= 0 && rows < (1ll << 28) && V >= 1 && V < (1ll << 31) && (rows <= 1 || ld >= V), "%s: bad shape rows=%lld V=%lld ld=%lld", what,
              (long long)rows, (long long)V, (long long)ld);
  B2G_REQUIRE(tau >= 1e-20f && tau <= 1e20f, "%s: the temperature must lie in 1e-20..1e20", what);
  return 0;
}

static policy::RowArgs row_args(const int64_t* target, int64_t V, int64_t ignore_index, float tau, int* status) {
  policy::RowArgs a = {};
  a.target = target; a.V = V; a.ignore_index = ignore_index; a.tau = tau; a.status = status;
  a.inv_tau = 1.0 / tau;
  // the low parts are positive: -inf logits times both parts stay -inf
  auto in_two = [](double c, float& hi, float& lo) {
    hi = (float)c;
    if ((double)hi >= c) hi = nextafterf(hi, 0.f);
    lo = (float)(c - (double)hi);
  };
  in_two(1.4426950408889634 / tau, a.c.hi, a.c.lo);    // log2(e) / tau
  in_two(1.0 / tau, a.c.inv, a.c.inv_lo);
  return a;
}

// Which kernel, cluster and slices.
//   Rows of at most 16 vectors of 16 bytes a lane (bf16: 4081 logits): short_kernel, a warp per row (200,000 x 1000 bf16: log-
//     probabilities 123 us, 617 us with a CTA per row).
//   Rows of at most kSmallRow bytes: held_kernel with one CTA of 128 threads per row, many CTAs per SM (20,000 x 10,000 bf16: loss
//     183 us, 262 us in the pipeline, whose rows cost as much as 20 to 30 KB however short they are; 16,000: 161 and 188; 20,000:
//     186 and 189).
//   Else pipe_kernel with the cluster size whose clusters have the fewest bytes to go through one after the other,
//     rounds * (slice + kRoundBytes),  rounds = rows / clusters that the device holds at once (of 296 places 8-CTA clusters fill
//     264, 9-CTA clusters 270, 5-CTA clusters 280: the GPCs have 16 to 20 SMs), for the policy loss among those whose slices
//     leave room for two slots.  kRoundBytes stands for what a row costs however short its slices are (12 KB against 8: policy
//     loss without temperature, old or reference log-probabilities of 301 x 32003 fp32 21.0 and 23.3 us, of 301 x 32003 bf16 14.6 and
//     17.9, of 150 x 64000 bf16 13.6 and 14.8).
//   Policy loss of rows too wide for that: one slot; beyond it wide_kernel.
// Two CTAs share an SM's 228 KB: 1 KB each is the system's, and pipe_kernel's own arrays may take 5 KB beside the slices.
constexpr int64_t kSmallRow = 36 * 1024, kSliceLimit = 108 * 1024, kRoundBytes = 12 * 1024;
constexpr int64_t kStreamBytes = policy::kStages * policy::kChunk * 16;
static_assert(kStreamBytes <= kSliceLimit, "two CTAs share an SM");

template <typename T, bool kPolicy>
static cudaLaunchConfig_t pipe_config(int cluster, int64_t bytes, cudaLaunchAttribute* at) {
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3((unsigned)cluster);
  cfg.blockDim = dim3(policy::kPipeThreads<kPolicy>);
  cfg.dynamicSmemBytes = (size_t)bytes;
  at[0].id = cudaLaunchAttributeClusterDimension;
  at[0].val.clusterDim = {(unsigned)cluster, 1, 1};
  cfg.attrs = at;
  cfg.numAttrs = 1;
  return cfg;
}

// Clusters of pipe_kernel that the device holds at once, with all the shared memory that a CTA may take: asked once per size.
template <typename T, bool kPolicy>
static int resident_clusters(int cluster, int* out) {
  static std::atomic<int> known[64][policy::kMaxCluster + 1];
  int dev = 0;
  B2G_CUDA_OK(cudaGetDevice(&dev));
  B2G_REQUIRE(dev >= 0 && dev < 64, "device index %d out of range", dev);
  int n = known[dev][cluster].load(std::memory_order_relaxed);
  if (n == 0) {
    cudaLaunchAttribute at[1];
    const cudaLaunchConfig_t cfg = pipe_config<T, kPolicy>(cluster, kSliceLimit, at);
    B2G_CUDA_OK(cudaOccupancyMaxActiveClusters(&n, policy::pipe_kernel<T, kPolicy>, &cfg));
    n = n < 1 ? -1 : n;
    known[dev][cluster].store(n, std::memory_order_relaxed);
  }
  *out = n < 0 ? 0 : n;
  return 0;
}

template <typename T, bool kPolicy>
static int launch_pipe(const T* logits, int64_t ld, const policy::RowArgs& a, T* out, int64_t ld_out, int64_t rows, cudaStream_t s, bool* taken) {
  constexpr int N = 16 / sizeof(T);
  B2G_ONCE_PER_DEVICE(
      B2G_CUDA_OK(cudaFuncSetAttribute(policy::pipe_kernel<T, kPolicy>, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)kSliceLimit));
      B2G_CUDA_OK(cudaFuncSetAttribute(policy::pipe_kernel<T, kPolicy>, cudaFuncAttributeNonPortableClusterSizeAllowed, 1)));
  const int64_t need = (a.V + 2 * (N - 1)) / N;      // vectors of a row at its worst alignment
  int best = 0, best_resident = 0;
  for (int slots = policy::kMaxSlots; slots >= 1 && best == 0; --slots) {
    int64_t best_cost = 0;
    for (int c = 1; c <= policy::kMaxCluster; ++c) {
      const int64_t slice = (need + c - 1) / c * 16;
      if (kPolicy && slice * slots > kSliceLimit) continue;
      int resident = 0;
      if (int rc = resident_clusters<T, kPolicy>(c, &resident)) return rc;
      if (resident == 0) continue;
      const int64_t cost = (rows + resident - 1) / resident * (slice + kRoundBytes);
      if (best == 0 || cost < best_cost) { best = c; best_cost = cost; best_resident = resident; }
    }
  }
  *taken = best != 0;
  if (best == 0) return 0;
  const int64_t slice = (need + best - 1) / best * 16;
  const int slots = !kPolicy || kSliceLimit / slice < policy::kMaxSlots ? 1 : policy::kMaxSlots;
  const int lead = slots - 1;      // G trails S by a row where there is a second slot to wait in
  cudaLaunchAttribute at[1];
  cudaLaunchConfig_t cfg = pipe_config<T, kPolicy>(best, kPolicy ? slice * slots : kStreamBytes, at);
  cfg.gridDim = dim3((unsigned)((rows < best_resident ? rows : best_resident) * best));
  cfg.stream = s;
  B2G_CUDA_OK(cudaLaunchKernelEx(&cfg, policy::pipe_kernel<T, kPolicy>, logits, ld, a, out, ld_out, rows, best, slots, lead, (int)(slice / 16)));
  return 0;
}

template <typename T, bool kPolicy>
static int launch_held(const T* logits, int64_t ld, const policy::RowArgs& a, T* out, int64_t ld_out, int64_t rows, int64_t bytes, cudaStream_t s) {
  B2G_KERNEL_SMEM((policy::held_kernel<T, kPolicy>), kSmallRow);
  policy::held_kernel<T, kPolicy><<<(unsigned)rows, policy::kHeldThreads, (size_t)bytes, s>>>(logits, ld, a, out, ld_out);
  B2G_CUDA_OK(cudaGetLastError());
  return 0;
}

template <typename T, int kVecs, bool kPolicy>
static int launch_short(const T* logits, int64_t ld, const policy::RowArgs& a, T* out, int64_t ld_out, int64_t rows, cudaStream_t s) {
  policy::short_kernel<T, kVecs, kPolicy><<<(unsigned)((rows + policy::kShortWarps - 1) / policy::kShortWarps), policy::kShortWarps * 32, 0, s>>>(
      logits, ld, a, out, ld_out, rows);
  B2G_CUDA_OK(cudaGetLastError());
  return 0;
}

template <typename T, bool kPolicy>
static int launch_rows(const T* logits, int64_t ld, const policy::RowArgs& a, T* out, int64_t ld_out, int64_t rows, cudaStream_t s) {
  constexpr int N = 16 / sizeof(T);
  const int64_t need = (a.V + 2 * (N - 1)) / N, bytes = need * 16;
  if (need <= 32 * 4) return launch_short<T, 4, kPolicy>(logits, ld, a, out, ld_out, rows, s);
  if (need <= 32 * 8) return launch_short<T, 8, kPolicy>(logits, ld, a, out, ld_out, rows, s);
  if (need <= 32 * 16) return launch_short<T, 16, kPolicy>(logits, ld, a, out, ld_out, rows, s);
  if (bytes <= kSmallRow) return launch_held<T, kPolicy>(logits, ld, a, out, ld_out, rows, bytes, s);
  bool taken = false;
  if (int rc = launch_pipe<T, kPolicy>(logits, ld, a, out, ld_out, rows, s, &taken)) return rc;
  if (!taken) {
    if constexpr (kPolicy) {
      policy::wide_kernel<T><<<(unsigned)rows, 512, 0, s>>>(logits, ld, a, out, ld_out);
      B2G_CUDA_OK(cudaGetLastError());
    } else {
      B2G_REQUIRE(taken, "the device has no room for a CTA of %d threads", policy::kPipeThreads<kPolicy>);
    }
  }
  return 0;
}

// Blocks of 32, 128 or 256 threads, so that a short row does not leave most of one idle.
template <typename T, int kThreads>
static int launch_bwd_as(const T* logits, int64_t ld, const policy::RowArgs& a, const void* grad_logp, T* out, int64_t ld_out, int64_t rows,
                         int64_t need, cudaStream_t s) {
  const int64_t tile = kThreads * policy::kBwdVecs, blocks = (need + tile - 1) / tile;
  B2G_REQUIRE(rows * blocks < (1ll << 31), "token_logprobs_bwd: %lld rows of %lld logits are too many for one call", (long long)rows, (long long)a.V);
  policy::logp_bwd_kernel<T, kThreads><<<(unsigned)(rows * blocks), kThreads, 0, s>>>(logits, ld, a, grad_logp, out, ld_out, (int)blocks);
  B2G_CUDA_OK(cudaGetLastError());
  return 0;
}
template <typename T>
static int launch_bwd(const T* logits, int64_t ld, const policy::RowArgs& a, const void* grad_logp, T* out, int64_t ld_out, int64_t rows, cudaStream_t s) {
  constexpr int N = 16 / sizeof(T);
  const int64_t need = (a.V + 2 * (N - 1)) / N;
  if (need <= 32 * policy::kBwdVecs) return launch_bwd_as<T, 32>(logits, ld, a, grad_logp, out, ld_out, rows, need, s);
  if (need <= 128 * policy::kBwdVecs) return launch_bwd_as<T, 128>(logits, ld, a, grad_logp, out, ld_out, rows, need, s);
  return launch_bwd_as<T, 256>(logits, ld, a, grad_logp, out, ld_out, rows, need, s);
}

extern "C" int b2g_token_logprobs(const void* logits, int64_t ld, int logits_dtype, const int64_t* target, void* logp, int logp_dtype, float* stats,
                                  int64_t rows, int64_t V, float temperature, int64_t ignore_index, int* status, void* stream) {
  if (int rc = check_rows("token_logprobs", logits_dtype, rows, V, ld, temperature)) return rc;
  B2G_REQUIRE(logp_dtype == 0 || logp_dtype == 1, "token_logprobs: logp_dtype must be 0 (fp32) or 1 (fp64)");
  if (rows == 0) return 0;
  B2G_REQUIRE(logits && target && logp && stats, "token_logprobs: null pointer");
  B2G_REQUIRE(aligned16(stats), "token_logprobs: stats must be 16-byte aligned");
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  policy::RowArgs a = row_args(target, V, ignore_index, temperature, status);
  a.logp = logp; a.logp64 = logp_dtype; a.stats = reinterpret_cast<float4*>(stats);
  if (logits_dtype) return launch_rows<float, false>(static_cast<const float*>(logits), ld, a, nullptr, 0, rows, s);
  return launch_rows<__nv_bfloat16, false>(static_cast<const __nv_bfloat16*>(logits), ld, a, nullptr, 0, rows, s);
}

extern "C" int b2g_token_logprobs_bwd(const void* logits, int64_t ld, int logits_dtype, const int64_t* target, const float* stats,
                                      const void* grad_logp, int logp_dtype, void* grad_logits, int64_t ld_grad, int64_t rows, int64_t V,
                                      float temperature, int64_t ignore_index, void* stream) {
  if (int rc = check_rows("token_logprobs_bwd", logits_dtype, rows, V, ld < ld_grad ? ld : ld_grad, temperature)) return rc;
  B2G_REQUIRE(logp_dtype == 0 || logp_dtype == 1, "token_logprobs_bwd: logp_dtype must be 0 (fp32) or 1 (fp64)");
  if (rows == 0) return 0;
  B2G_REQUIRE(logits && target && stats && grad_logp && grad_logits, "token_logprobs_bwd: null pointer");
  B2G_REQUIRE(aligned16(stats), "token_logprobs_bwd: stats must be 16-byte aligned");
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  policy::RowArgs a = row_args(target, V, ignore_index, temperature, nullptr);
  a.logp64 = logp_dtype; a.stats = reinterpret_cast<float4*>(const_cast<float*>(stats));
  if (logits_dtype)
    return launch_bwd(static_cast<const float*>(logits), ld, a, grad_logp, static_cast<float*>(grad_logits), ld_grad, rows, s);
  return launch_bwd(static_cast<const __nv_bfloat16*>(logits), ld, a, grad_logp, static_cast<__nv_bfloat16*>(grad_logits), ld_grad, rows, s);
}

extern "C" int b2g_policy_loss(const void* logits, int64_t ld, int logits_dtype, const int64_t* target, const float* advantage,
                               const float* old_logp, const float* ref_logp, const float* weight, float clip_low, float clip_high, float kl_coef,
                               float temperature, float* loss, float* logp, float* kl, void* grad_logits, int64_t ld_grad, int64_t rows, int64_t V,
                               int64_t ignore_index, int* status, void* stream) {
  if (int rc = check_rows("policy_loss", logits_dtype, rows, V, ld < ld_grad ? ld : ld_grad, temperature)) return rc;
  B2G_REQUIRE(clip_low >= 0.f && clip_low <= 1.f && clip_high >= 0.f && clip_high <= 3.4e38f, "policy_loss: clip_low outside 0..1 or clip_high negative");
  B2G_REQUIRE(kl_coef >= 0.f && kl_coef <= 3.4e38f, "policy_loss: kl_coef must be finite and not negative");
  B2G_REQUIRE(kl_coef == 0.f || ref_logp, "policy_loss: a KL term needs the reference log-probabilities");
  if (rows == 0) return 0;
  B2G_REQUIRE(logits && target && advantage && loss && logp && kl && grad_logits, "policy_loss: null pointer");
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  policy::RowArgs a = row_args(target, V, ignore_index, temperature, status);
  a.logp = logp; a.advantage = advantage; a.old_logp = old_logp; a.ref_logp = ref_logp; a.weight = weight;
  a.clip_low = clip_low; a.clip_high = clip_high; a.kl_coef = kl_coef; a.loss = loss; a.kl = kl;
  if (logits_dtype)
    return launch_rows<float, true>(static_cast<const float*>(logits), ld, a, static_cast<float*>(grad_logits), ld_grad, rows, s);
  return launch_rows<__nv_bfloat16, true>(static_cast<const __nv_bfloat16*>(logits), ld, a, static_cast<__nv_bfloat16*>(grad_logits), ld_grad, rows, s);
}

extern "C" int b2g_preference_loss(const void* logp, int logp_dtype, const void* ref_logp, int ref_dtype, const int64_t* target, const int64_t* offsets, int64_t N,
                                   int64_t pairs, int64_t ignore_index, float beta, float label_smoothing, int loss_type, int average, float* loss,
                                   float* chosen, float* rejected, float* coef, int* status, void* stream) {
  B2G_REQUIRE(N >= 0 && pairs >= 0 && pairs < (1ll << 28), "preference_loss: bad shape N=%lld pairs=%lld", (long long)N, (long long)pairs);
  B2G_REQUIRE(logp_dtype == 0 || logp_dtype == 1, "preference_loss: logp_dtype must be 0 (fp32) or 1 (fp64)");
  B2G_REQUIRE(ref_dtype == 0 || ref_dtype == 1, "preference_loss: ref_dtype must be 0 (fp32) or 1 (fp64)");
  B2G_REQUIRE(beta > 0.f && beta <= 3.4e38f, "preference_loss: beta must be positive and finite");
  B2G_REQUIRE(label_smoothing >= 0.f && label_smoothing < 0.5f, "preference_loss: label_smoothing outside [0, 0.5)");
  B2G_REQUIRE(loss_type == 0 || loss_type == 1, "preference_loss: loss_type must be 0 (sigmoid) or 1 (squared)");
  B2G_REQUIRE(loss_type == 0 || label_smoothing == 0.f, "preference_loss: label smoothing belongs to the sigmoid loss");
  if (pairs == 0) return 0;
  B2G_REQUIRE((logp || N == 0) && offsets && loss && chosen && rejected && coef, "preference_loss: null pointer");
  // a CTA goes through 2048 tokens of either sequence in one turn of its loads
  int cluster = 1;
  while (cluster < policy::kPairClusterMax && N / (2 * pairs) > 2048 * cluster) cluster *= 2;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3((unsigned)(pairs * cluster));
  cfg.blockDim = dim3(policy::kPairThreads);
  cfg.stream = static_cast<cudaStream_t>(stream);
  cudaLaunchAttribute at[1];
  at[0].id = cudaLaunchAttributeClusterDimension;
  at[0].val.clusterDim = {(unsigned)cluster, 1, 1};
  cfg.attrs = at;
  cfg.numAttrs = 1;
#define B2G_PAIRS(L, R)                                                                                                                      \
  B2G_CUDA_OK(cudaLaunchKernelEx(&cfg, policy::pair_kernel<L, R>, static_cast<const L*>(logp), static_cast<const R*>(ref_logp), target, offsets, N, \
                                 pairs, ignore_index, beta, label_smoothing, loss_type, average, loss, chosen, rejected, coef, status, cluster))
  if (logp_dtype) {
    if (ref_dtype) B2G_PAIRS(double, double);
    else B2G_PAIRS(double, float);
  } else {
    if (ref_dtype) B2G_PAIRS(float, double);
    else B2G_PAIRS(float, float);
  }
#undef B2G_PAIRS
  return 0;
}

extern "C" int b2g_preference_loss_bwd(const float* grad_loss, const float* coef, const int64_t* target, const int64_t* offsets, void* grad_logp,
                                       int logp_dtype, int64_t N, int64_t pairs, int64_t ignore_index, void* stream) {
  B2G_REQUIRE(N >= 0 && N < (1ll << 38) && pairs >= 0 && pairs < (1ll << 30), "preference_loss_bwd: bad shape N=%lld pairs=%lld", (long long)N, (long long)pairs);
  B2G_REQUIRE(logp_dtype == 0 || logp_dtype == 1, "preference_loss_bwd: logp_dtype must be 0 (fp32) or 1 (fp64)");
  if (N == 0) return 0;
  B2G_REQUIRE((grad_loss && coef || pairs == 0) && offsets && grad_logp, "preference_loss_bwd: null pointer");
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  const int64_t tile = policy::kPairBwdThreads * policy::kPairBwdTokens;
  const unsigned blocks = (unsigned)((N + tile - 1) / tile);
  if (logp_dtype)
    policy::pair_bwd_kernel<<<blocks, policy::kPairBwdThreads, 0, s>>>(grad_loss, coef, target, offsets, static_cast<double*>(grad_logp), N, pairs, ignore_index);
  else
    policy::pair_bwd_kernel<<<blocks, policy::kPairBwdThreads, 0, s>>>(grad_loss, coef, target, offsets, static_cast<float*>(grad_logp), N, pairs, ignore_index);
  B2G_CUDA_OK(cudaGetLastError());
  return 0;
}
