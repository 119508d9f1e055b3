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
// the eight octiles of the fraction); a sum of many of them is that much too small.
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
// keeps 24 bits, take the full exponential; they move twice the bytes per value, so it is as well hidden.
struct Scale { float hi, lo, inv; };
template <typename T>
__device__ __forceinline__ float exp_from(float z, float m, const Scale& c) {
  const float x = z - m;
  if constexpr (sizeof(T) == 2) return ex2(fmaf(x, c.hi, x * c.lo));
  else return expf(x * c.inv);
}
// The sum without ex2's shortfall; the largest term is exp(0), which is exact.
template <typename T>
__device__ __forceinline__ double whole_sum(double d) { return sizeof(T) == 2 ? d + (d - 1.0) * kEx2Shortfall : d; }

// Sixteen bytes of logits as floats, and back.
template <typename T>
struct Vec {
  static constexpr int N = 16 / sizeof(T);
  uint32_t w[4];
  __device__ __forceinline__ float get(int i) const {
    if constexpr (sizeof(T) == 2) return (i & 1) ? dev::bf16_hi(w[i >> 1]) : dev::bf16_lo(w[i >> 1]);
    else return __uint_as_float(w[i]);
  }
  __device__ __forceinline__ void set_nothing() {   // -inf everywhere: the maximum and the sum do not see it
#pragma unroll
    for (int i = 0; i < 4; ++i) w[i] = sizeof(T) == 2 ? 0xFF80FF80u : 0xFF800000u;
  }
};

// A row as 16-byte vectors of the memory it lies in: vector v holds the columns [v * N - shift, (v + 1) * N - shift), so the
// inner vectors are aligned whatever the row's own alignment is, and at most the first and the last one are partial.
template <typename T>
struct Row {
  static constexpr int N = Vec<T>::N;
  const T* x;
  int shift, nvec;
  int64_t V;
  __device__ Row(const T* p, int64_t V_) : x(p), shift((int)((reinterpret_cast<uintptr_t>(p) / sizeof(T)) % N)), V(V_) {
    nvec = (int)((V + shift + N - 1) / N);
  }
  __device__ __forceinline__ int64_t column(int v) const { return (int64_t)v * N - shift; }
  __device__ __forceinline__ bool full(int v) const { return column(v) >= 0 && column(v) + N <= V; }
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
  // Writes g[0..N) to the same columns of `out`; `wide`: out is aligned as the row is.
  __device__ __forceinline__ void store(T* out, int v, const float (&g)[N], bool wide) const {
    if (wide && full(v)) {
      uint4 q;
      if constexpr (sizeof(T) == 2)
        q = make_uint4(dev::pack_bf16(g[0], g[1]), dev::pack_bf16(g[2], g[3]), dev::pack_bf16(g[4], g[5]), dev::pack_bf16(g[6], g[7]));
      else
        q = make_uint4(__float_as_uint(g[0]), __float_as_uint(g[1]), __float_as_uint(g[2]), __float_as_uint(g[3]));
      __stcs(reinterpret_cast<uint4*>(out + column(v)), q);
    } else {
#pragma unroll
      for (int i = 0; i < N; ++i) {
        const int64_t c = column(v) + i;
        if (c >= 0 && c < V) out[c] = from_float<T>(g[i]);
      }
    }
  }
};
template <typename T>
__device__ __forceinline__ bool same_alignment(const T* a, const T* b) {
  return ((reinterpret_cast<uintptr_t>(a) ^ reinterpret_cast<uintptr_t>(b)) & 15) == 0;
}

// What a launch computes for its rows, and where the row's scalars come from and go to.
struct RowArgs {
  const int64_t* target;
  int64_t V, ignore_index;
  float tau;
  Scale c;
  int* status;
  // log-probabilities
  void* logp;          // fp32, or fp64 when logp64
  int logp64;
  float4* stats;       // what the backward pass of the log-probabilities reads: m, 1/d, 1 - p of the target, lse
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

// What a row's maximum, sum and target logit say.  `rest` is 1 - p of the target, the entry of the cotangent that cancels when
// the target is nearly certain.  16-bit logits take it from the 64-bit log-probability; fp32 logits from z/tau, m/tau and lse
// rounded to 32 bits, as the elementary form of the gradient in that type does (off by half a step of lse).  A vocabulary
// masked throughout by the type's lowest value has an lse that holds no log d any more and stays with 64 bits.
struct Scalars { double lse, logp; float rest; };
template <typename T>
__device__ __forceinline__ Scalars row_scalars(float m, double d, float zy, float tau) {
  Scalars s;
  s.lse = (double)m / (double)tau + log(d);
  s.logp = ((double)zy - (double)m) / (double)tau - log(d);
  s.rest = sizeof(T) == 4 && fabs(s.lse) < 16384.0 ? 1.f - expf(zy / tau - (float)((double)(m / tau) + log(d))) : (float)-expm1(s.logp);
  return s;
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
  const bool inside = ratio * adv <= clipped * adv || ratio != ratio;
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

// A maximum and the sum of exponentials against it.  The maximum starts at the type's lowest value, not at -inf, so that -inf
// logits (a masked vocabulary) meet a finite maximum: exp(-inf - lowest) = 0.
struct Stat { float m; double d; };
__device__ __forceinline__ Stat join(const Stat& a, const Stat& b, float tau) {
  const float m = fmaxf(a.m, b.m);
  const double da = a.m == m ? a.d : a.d * exp(((double)a.m - m) / tau), db = b.m == m ? b.d : b.d * exp(((double)b.m - m) / tau);
  return Stat{m, da + db};
}

// ---- rows held on chip ----------------------------------------------------------------------------
// A cluster of 1, 2, 4 or 8 CTAs per row.  Every thread copies its vectors of the CTA's slice to shared memory (cp.async, no
// registers) and is the only one that reads them back, so no barrier stands between the copy and the three passes over it:
// maximum (while later groups of the copy are on their way), sum, cotangent.  Maximum and sum are joined over the cluster
// through distributed shared memory.  The row crosses HBM once.
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

template <typename T, int kThreads, bool kPolicy>
__global__ void __launch_bounds__(kThreads, 1536 / kThreads) held_kernel(const T* logits, int64_t ld, RowArgs a, T* out, int64_t ld_out,
                                                                         int cluster) {
  constexpr int N = Vec<T>::N, kWarps = kThreads / 32;
  extern __shared__ __align__(16) uint8_t slice[];
  __shared__ float warp_m[kWarps];
  __shared__ double warp_d[kWarps];
  __shared__ Stat slot[8];
  __shared__ float4 bcast;
  const int rank = blockIdx.x % cluster, lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int64_t r = blockIdx.x / cluster, y = a.target[r];
  const bool first = rank == 0 && threadIdx.x == 0;
  const Row<T> row(logits + r * ld, a.V);
  T* const o = kPolicy ? out + r * ld_out : nullptr;
  const bool wide = kPolicy && same_alignment(row.x, (const T*)o);
  const int per = (row.nvec + cluster - 1) / cluster, begin = rank * per, end = min(begin + per, row.nvec);

  bool live = target_ok(y, a, first);
  Given in{1.f, 0.f, 0.f, 0.f};
  if (kPolicy) {
    in = given(a, r);
    live = live && in.weight != 0.f;
  }
  if (!live) {      // the same for every CTA of the cluster
    if (first) {
      if (kPolicy) { a.loss[r] = 0.f; a.kl[r] = 0.f; static_cast<float*>(a.logp)[r] = 0.f; }
      else put_logp(a, r, 0.0, make_float4(0.f, 0.f, 0.f, 0.f));
    }
    if (kPolicy) {
      const float zero[N] = {};
      for (int v = begin + threadIdx.x; v < end; v += kThreads) row.store(o, v, zero, wide);
    }
    return;
  }

  // this thread's vectors: begin + threadIdx.x + i * kThreads, i < n, at mine + i * kThreads * 16
  const int v0 = begin + threadIdx.x, n = v0 < end ? (end - v0 + kThreads - 1) / kThreads : 0;
  const uint32_t mine = dev::smem_u32(slice) + threadIdx.x * 16;
  const int group = (per + kThreads * kGroups - 1) / (kThreads * kGroups);
#pragma unroll
  for (int g = 0; g < kGroups; ++g) {
    for (int i = g * group; i < min(n, (g + 1) * group); ++i) {
      const int v = v0 + i * kThreads;
      const uint32_t at = mine + i * (kThreads * 16);
      if (row.full(v)) {
        copy16(at, row.x + row.column(v));
      } else {
        const Vec<T> x = row.load(v);
        dev::sts128(at, x.w[0], x.w[1], x.w[2], x.w[3]);
      }
    }
    copy_commit();
  }
  const float zy = to_float(row.x[y]);      // before any CTA of the row can overwrite it

  float m = kLowest;
  auto max_of = [&](int g) {
#pragma unroll 4
    for (int i = g * group; i < min(n, (g + 1) * group); ++i) m = vec_max(from_shared<T>(mine + i * (kThreads * 16)), m);
  };
  copy_wait<3>(); max_of(0);
  copy_wait<2>(); max_of(1);
  copy_wait<1>(); max_of(2);
  copy_wait<0>(); max_of(3);
#pragma unroll
  for (int s = 16; s > 0; s >>= 1) m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, s));
  if (lane == 0) warp_m[warp] = m;
  __syncthreads();
#pragma unroll
  for (int i = 0; i < kWarps; ++i) m = fmaxf(m, warp_m[i]);

  // eight (four) terms are summed in 32 bits, everything above them in 64
  const Scale c = a.c;
  double d = 0.0;
#pragma unroll 2
  for (int i = 0; i < n; ++i) {
    const Vec<T> x = from_shared<T>(mine + i * (kThreads * 16));
    float e[N];
#pragma unroll
    for (int j = 0; j < N; ++j) e[j] = exp_from<T>(x.get(j), m, c);
#pragma unroll
    for (int s = N / 2; s > 0; s >>= 1)
#pragma unroll
      for (int j = 0; j < s; ++j) e[j] += e[j + s];
    d += (double)e[0];
  }
#pragma unroll
  for (int s = 16; s > 0; s >>= 1) d += __shfl_xor_sync(0xffffffffu, d, s);
  if (lane == 0) warp_d[warp] = d;
  __syncthreads();
  if (threadIdx.x < cluster) {              // thread k gives this CTA's share to CTA k
    d = 0.0;
    for (int i = 0; i < kWarps; ++i) d += warp_d[i];
    const uint32_t to = dev::map_to_cta(dev::smem_u32(&slot[rank]), threadIdx.x);
    asm volatile("st.shared::cluster.f32 [%0], %1;" ::"r"(to), "f"(m) : "memory");
    asm volatile("st.shared::cluster.f64 [%0], %1;" ::"r"(to + 8), "d"(d) : "memory");
  }
  dev::cluster_sync_all();
  if (threadIdx.x == 0) {
    Stat t = slot[0];
    for (int i = 1; i < cluster; ++i) t = join(t, slot[i], a.tau);
    t.d = whole_sum<T>(t.d);
    const Scalars v = row_scalars<T>(t.m, t.d, zy, a.tau);
    if (kPolicy) {
      const float coef = policy_scalars(a, in, v.logp, r, rank == 0) / a.tau;
      bcast = make_float4(coef, (float)(coef / t.d), t.m, coef * v.rest);
    } else if (rank == 0) {
      put_logp(a, r, v.logp, make_float4(t.m, (float)(1.0 / t.d), v.rest, (float)v.lse));
    }
  }
  if (!kPolicy) return;
  __syncthreads();
  const float coef = bcast.x, k = bcast.y, top = bcast.z, at_target = bcast.w;
  const int vy = (int)((y + row.shift) / N), jy = (int)((y + row.shift) % N);
#pragma unroll 2
  for (int i = 0; i < n; ++i) {
    const int v = v0 + i * kThreads;
    const Vec<T> x = from_shared<T>(mine + i * (kThreads * 16));
    float g[N];
#pragma unroll
    for (int j = 0; j < N; ++j) g[j] = coef == 0.f ? 0.f : -k * exp_from<T>(x.get(j), top, c);
    if (v == vy && coef != 0.f) {
#pragma unroll
      for (int j = 0; j < N; ++j)
        if (j == jy) g[j] = at_target;
    }
    row.store(o, v, g, wide);
  }
}

// ---- rows of any width ----------------------------------------------------------------------------
// One CTA per row that reads it twice (maximum, then sum) and, for the policy loss, a third time: vocabularies wider than a
// cluster's registers hold.
template <typename T, bool kPolicy>
__global__ void __launch_bounds__(512) wide_kernel(const T* logits, int64_t ld, RowArgs a, T* out, int64_t ld_out) {
  constexpr int N = Vec<T>::N, kThreads = 512, kWarps = kThreads / 32;
  __shared__ float warp_m[kWarps];
  __shared__ double warp_d[kWarps];
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
    if (threadIdx.x == 0) {
      if (kPolicy) { a.loss[r] = 0.f; a.kl[r] = 0.f; static_cast<float*>(a.logp)[r] = 0.f; }
      else put_logp(a, r, 0.0, make_float4(0.f, 0.f, 0.f, 0.f));
    }
    if (kPolicy) {
      const float zero[N] = {};
      for (int v = threadIdx.x; v < row.nvec; v += kThreads) row.store(o, v, zero, wide);
    }
    return;
  }
  float m = kLowest;
  for (int v = threadIdx.x; v < row.nvec; v += kThreads) {
    const Vec<T> x = row.load(v);
#pragma unroll
    for (int j = 0; j < N; ++j) m = fmaxf(m, x.get(j));
  }
#pragma unroll
  for (int s = 16; s > 0; s >>= 1) m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, s));
  if (lane == 0) warp_m[warp] = m;
  __syncthreads();
  for (int i = 0; i < kWarps; ++i) m = fmaxf(m, warp_m[i]);
  const Scale c = a.c;
  double d = 0.0;
  for (int v = threadIdx.x; v < row.nvec; v += kThreads) {
    const Vec<T> x = row.load(v);
    float e = 0.f;
#pragma unroll
    for (int j = 0; j < N; ++j) e += exp_from<T>(x.get(j), m, c);
    d += (double)e;
  }
#pragma unroll
  for (int s = 16; s > 0; s >>= 1) d += __shfl_xor_sync(0xffffffffu, d, s);
  if (lane == 0) warp_d[warp] = d;
  const float zy = to_float(row.x[y]);
  __syncthreads();
  if (threadIdx.x == 0) {
    d = 0.0;
    for (int i = 0; i < kWarps; ++i) d += warp_d[i];
    d = whole_sum<T>(d);
    const Scalars v = row_scalars<T>(m, d, zy, a.tau);
    if (kPolicy) {
      const float coef = policy_scalars(a, in, v.logp, r, true) / a.tau;
      bcast = make_float4(coef, (float)(coef / d), m, coef * v.rest);
    } else {
      put_logp(a, r, v.logp, make_float4(m, (float)(1.0 / d), v.rest, (float)v.lse));
    }
  }
  if (!kPolicy) return;
  __syncthreads();
  const float coef = bcast.x, k = bcast.y, at_target = bcast.w;
  const int vy = (int)((y + row.shift) / N), jy = (int)((y + row.shift) % N);
  for (int v = threadIdx.x; v < row.nvec; v += kThreads) {
    const Vec<T> x = row.load(v);
    float g[N];
#pragma unroll
    for (int j = 0; j < N; ++j) {
      g[j] = coef == 0.f ? 0.f : -k * exp_from<T>(x.get(j), m, c);
      if (v == vy && j == jy && coef != 0.f) g[j] = at_target;
    }
    row.store(o, v, g, wide);
  }
}

// ---- gradient of the log-probabilities --------------------------------------------------------------
// dz = g (onehot - exp((z - m)/tau)/d)/tau: one pass without a reduction, kBwdVecs vectors per thread.
constexpr int kBwdThreads = 256, kBwdVecs = 4;
template <typename T>
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
    const float zero[N] = {};
    for (int i = 0; i < kBwdVecs; ++i) {
      const int v = begin + i * kBwdThreads + threadIdx.x;
      if (v < row.nvec) row.store(o, v, zero, wide);
    }
    return;
  }
  const float4 st = a.stats[r];
  const float m = st.x, k = g * st.y, at_target = g * st.z;
  const Scale c = a.c;
  const int vy = (int)((y + row.shift) / N), jy = (int)((y + row.shift) % N);
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
    if (v < row.nvec) {
      float e[N];
#pragma unroll
      for (int j = 0; j < N; ++j) {
        e[j] = -k * exp_from<T>(x[i].get(j), m, c);
        if (v == vy && j == jy) e[j] = at_target;
      }
      row.store(o, v, e, wide);
    }
  }
}

// ---- preference loss ------------------------------------------------------------------------------
constexpr int kPairThreads = 256;

// Sums of 64 bits over one sequence's counted tokens.
template <typename L>
__device__ __forceinline__ void sequence_sum(const L* logp, const float* ref, const int64_t* target, int64_t begin, int64_t end,
                                             int64_t ignore_index, double& sum, double& count) {
  __shared__ double ps[kPairThreads / 32], pc[kPairThreads / 32];
  double s = 0.0;
  long long n = 0;
  for (int64_t i = begin + threadIdx.x; i < end; i += kPairThreads) {
    if (target && target[i] == ignore_index) continue;
    s += ref ? (double)logp[i] - (double)ref[i] : (double)logp[i];
    ++n;
  }
  double cnt = (double)n;
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) {
    s += __shfl_xor_sync(0xffffffffu, s, o);
    cnt += __shfl_xor_sync(0xffffffffu, cnt, o);
  }
  __syncthreads();
  if ((threadIdx.x & 31) == 0) { ps[threadIdx.x >> 5] = s; pc[threadIdx.x >> 5] = cnt; }
  __syncthreads();
  sum = count = 0.0;
  for (int i = 0; i < kPairThreads / 32; ++i) { sum += ps[i]; count += pc[i]; }
}

// The bounds of sequence s, brought into [0, N]; a bound that had to be moved is reported.
__device__ __forceinline__ void bounds(const int64_t* offsets, int64_t s, int64_t N, int64_t& begin, int64_t& end, int* status) {
  const int64_t b = offsets[s], e = offsets[s + 1];
  begin = b < 0 ? 0 : (b > N ? N : b);
  end = e < begin ? begin : (e > N ? N : e);
  if ((b != begin || e != end) && threadIdx.x == 0 && status) atomicCAS(status, 0, 905);
}

__device__ __forceinline__ double log_sigmoid(double u) { return fmin(u, 0.0) - log1p(exp(-fabs(u))); }

template <typename L>
__global__ void __launch_bounds__(kPairThreads) pair_kernel(const L* __restrict__ logp, const float* __restrict__ ref,
                                                            const int64_t* __restrict__ target, const int64_t* __restrict__ offsets, int64_t N,
                                                            int64_t P, int64_t ignore_index, float beta, float smoothing, int squared, int average,
                                                            float* __restrict__ loss, float* __restrict__ chosen, float* __restrict__ rejected,
                                                            float* __restrict__ coef, int* status) {
  const int64_t p = blockIdx.x;
  double sum[2], count[2];
  for (int h = 0; h < 2; ++h) {
    int64_t begin, end;
    bounds(offsets, p + h * P, N, begin, end, status);
    sequence_sum(logp, ref, target, begin, end, ignore_index, sum[h], count[h]);
    if (!average) count[h] = 1.0;
    count[h] = fmax(count[h], 1.0);
    sum[h] /= count[h];
  }
  if (threadIdx.x == 0) {
    const double b = beta, gap = sum[0] - sum[1], u = b * gap, e = smoothing;
    double l, slope;     // slope = d loss / d gap
    if (squared) {
      const double h = gap - 0.5 / b;
      l = h * h;
      slope = 2.0 * h;
    } else {
      l = -(1.0 - e) * log_sigmoid(u) - e * log_sigmoid(-u);
      slope = b * (e / (1.0 + exp(-u)) - (1.0 - e) / (1.0 + exp(u)));
    }
    loss[p] = (float)l;
    chosen[p] = (float)(b * sum[0]);
    rejected[p] = (float)(b * sum[1]);
    coef[p] = (float)(slope / count[0]);
    coef[P + p] = (float)(-slope / count[1]);
  }
}

// grad_logp[i] = grad_loss[pair] * coef[sequence] for counted tokens of a sequence, 0 elsewhere.  The sequence of a token is
// found by bisection in the offsets.
template <typename L>
__global__ void __launch_bounds__(256) pair_bwd_kernel(const float* __restrict__ grad_loss, const float* __restrict__ coef,
                                                       const int64_t* __restrict__ target, const int64_t* __restrict__ offsets,
                                                       L* __restrict__ grad_logp, int64_t N, int64_t P, int64_t ignore_index) {
  const int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x;
  if (i >= N) return;
  int64_t lo = 0, hi = 2 * P + 1;         // the number of offsets <= i
  while (lo < hi) {
    const int64_t mid = (lo + hi) >> 1;
    if (offsets[mid] <= i) lo = mid + 1;
    else hi = mid;
  }
  float g = 0.f;
  if (lo >= 1 && lo <= 2 * P && !(target && target[i] == ignore_index)) {
    const int64_t s = lo - 1;
    g = grad_loss[s < P ? s : s - P] * coef[s];
  }
  grad_logp[i] = g;
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
  const double c = 1.4426950408889634 / tau;    // log2(e) / tau
  a.c.hi = (float)c;
  if ((double)a.c.hi >= c) a.c.hi = nextafterf(a.c.hi, 0.f);   // the low part is positive: -inf logits times both parts stay -inf
  a.c.lo = (float)(c - (double)a.c.hi);
  a.c.inv = 1.f / tau;
  return a;
}

// Cluster size and threads of the held kernel.  The cluster is the smallest that leaves three CTAs' slices room on an SM, and
// larger while there are so few rows that SMs would be idle.  Slices of at most 16 KB use CTAs of 128 threads, whose
// reductions are shorter.  Rows beyond 8 CTAs' shared memory go to wide_kernel.
constexpr int64_t kSliceBytes = 72 * 1024, kSliceLimit = 224 * 1024;

template <typename T, int kThreads, bool kPolicy>
static int launch_held(const T* logits, int64_t ld, const policy::RowArgs& a, T* out, int64_t ld_out, int64_t rows, int cluster, int64_t bytes,
                       cudaStream_t s) {
  B2G_KERNEL_SMEM((policy::held_kernel<T, kThreads, kPolicy>), kSliceLimit);
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3((unsigned)(rows * cluster));
  cfg.blockDim = dim3(kThreads);
  cfg.dynamicSmemBytes = (size_t)bytes;
  cfg.stream = s;
  cudaLaunchAttribute at[1];
  at[0].id = cudaLaunchAttributeClusterDimension;
  at[0].val.clusterDim = {(unsigned)cluster, 1, 1};
  cfg.attrs = at;
  cfg.numAttrs = 1;
  B2G_CUDA_OK(cudaLaunchKernelEx(&cfg, policy::held_kernel<T, kThreads, kPolicy>, logits, ld, a, out, ld_out, cluster));
  return 0;
}

template <typename T, bool kPolicy>
static int launch_rows(const T* logits, int64_t ld, const policy::RowArgs& a, T* out, int64_t ld_out, int64_t rows, cudaStream_t s) {
  constexpr int N = 16 / sizeof(T);
  const int64_t need = (a.V + 2 * (N - 1)) / N;      // vectors of a row at its worst alignment
  auto slice = [&](int c) { return (need + c - 1) / c * 16; };
  int cluster = 1;
  while (cluster < 8 && slice(cluster) > kSliceBytes) cluster *= 2;
  while (cluster < 8 && rows * cluster < 2 * sm_count() && slice(cluster) > 8 * 1024) cluster *= 2;
  const int64_t bytes = slice(cluster);
  if (bytes > kSliceLimit) {
    policy::wide_kernel<T, kPolicy><<<(unsigned)rows, 512, 0, s>>>(logits, ld, a, out, ld_out);
    B2G_CUDA_OK(cudaGetLastError());
    return 0;
  }
  if (bytes <= 16 * 1024) return launch_held<T, 128, kPolicy>(logits, ld, a, out, ld_out, rows, cluster, bytes, s);
  return launch_held<T, 512, kPolicy>(logits, ld, a, out, ld_out, rows, cluster, bytes, s);
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
  const int n = logits_dtype ? 4 : 8, tile = policy::kBwdThreads * policy::kBwdVecs;
  const int64_t blocks = ((V + 2 * (n - 1)) / n + tile - 1) / tile;
  B2G_REQUIRE(rows * blocks < (1ll << 31), "token_logprobs_bwd: %lld rows of %lld logits are too many for one call", (long long)rows, (long long)V);
  if (logits_dtype)
    policy::logp_bwd_kernel<float><<<(unsigned)(rows * blocks), policy::kBwdThreads, 0, s>>>(
        static_cast<const float*>(logits), ld, a, grad_logp, static_cast<float*>(grad_logits), ld_grad, (int)blocks);
  else
    policy::logp_bwd_kernel<__nv_bfloat16><<<(unsigned)(rows * blocks), policy::kBwdThreads, 0, s>>>(
        static_cast<const __nv_bfloat16*>(logits), ld, a, grad_logp, static_cast<__nv_bfloat16*>(grad_logits), ld_grad, (int)blocks);
  B2G_CUDA_OK(cudaGetLastError());
  return 0;
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

extern "C" int b2g_preference_loss(const void* logp, int logp_dtype, const float* ref_logp, const int64_t* target, const int64_t* offsets, int64_t N,
                                   int64_t pairs, int64_t ignore_index, float beta, float label_smoothing, int loss_type, int average, float* loss,
                                   float* chosen, float* rejected, float* coef, int* status, void* stream) {
  B2G_REQUIRE(N >= 0 && pairs >= 0 && pairs < (1ll << 30), "preference_loss: bad shape N=%lld pairs=%lld", (long long)N, (long long)pairs);
  B2G_REQUIRE(logp_dtype == 0 || logp_dtype == 1, "preference_loss: logp_dtype must be 0 (fp32) or 1 (fp64)");
  B2G_REQUIRE(beta > 0.f && beta <= 3.4e38f, "preference_loss: beta must be positive and finite");
  B2G_REQUIRE(label_smoothing >= 0.f && label_smoothing < 0.5f, "preference_loss: label_smoothing outside [0, 0.5)");
  B2G_REQUIRE(loss_type == 0 || loss_type == 1, "preference_loss: loss_type must be 0 (sigmoid) or 1 (squared)");
  B2G_REQUIRE(loss_type == 0 || label_smoothing == 0.f, "preference_loss: label smoothing belongs to the sigmoid loss");
  if (pairs == 0) return 0;
  B2G_REQUIRE((logp || N == 0) && offsets && loss && chosen && rejected && coef, "preference_loss: null pointer");
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  if (logp_dtype)
    policy::pair_kernel<<<(unsigned)pairs, policy::kPairThreads, 0, s>>>(static_cast<const double*>(logp), ref_logp, target, offsets, N, pairs,
                                                                         ignore_index, beta, label_smoothing, loss_type, average, loss, chosen, rejected,
                                                                         coef, status);
  else
    policy::pair_kernel<<<(unsigned)pairs, policy::kPairThreads, 0, s>>>(static_cast<const float*>(logp), ref_logp, target, offsets, N, pairs,
                                                                         ignore_index, beta, label_smoothing, loss_type, average, loss, chosen, rejected,
                                                                         coef, status);
  B2G_CUDA_OK(cudaGetLastError());
  return 0;
}

extern "C" int b2g_preference_loss_bwd(const float* grad_loss, const float* coef, const int64_t* target, const int64_t* offsets, void* grad_logp,
                                       int logp_dtype, int64_t N, int64_t pairs, int64_t ignore_index, void* stream) {
  B2G_REQUIRE(N >= 0 && N < (1ll << 38) && pairs >= 0 && pairs < (1ll << 30), "preference_loss_bwd: bad shape N=%lld pairs=%lld", (long long)N, (long long)pairs);
  B2G_REQUIRE(logp_dtype == 0 || logp_dtype == 1, "preference_loss_bwd: logp_dtype must be 0 (fp32) or 1 (fp64)");
  if (N == 0) return 0;
  B2G_REQUIRE((grad_loss && coef || pairs == 0) && offsets && grad_logp, "preference_loss_bwd: null pointer");
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  const unsigned blocks = (unsigned)((N + 255) / 256);
  if (logp_dtype)
    policy::pair_bwd_kernel<<<blocks, 256, 0, s>>>(grad_loss, coef, target, offsets, static_cast<double*>(grad_logp), N, pairs, ignore_index);
  else
    policy::pair_bwd_kernel<<<blocks, 256, 0, s>>>(grad_loss, coef, target, offsets, static_cast<float*>(grad_logp), N, pairs, ignore_index);
  B2G_CUDA_OK(cudaGetLastError());
  return 0;
}
