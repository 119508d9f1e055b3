// Routing to experts: scores, balance bias, groups, top-k and renormalised weights, with the gradient of the logits.
//   s = softmax(l) | sigmoid(l) | sqrt(log(1 + e^l)),  c = s + b,  best M of G groups by the sum of their n best c,
//   best k of c in them,  w_j = alpha s_j / (sum_i s_i + 1e-20)  or  alpha s_j.
// Softmax weights that are renormalised are the softmax of the chosen logits (the common denominator cancels).
//
// One warp per token; lane i holds experts [i * kPer, (i + 1) * kPer), so the lowest lane of a tie holds the lowest expert.
// The order of c is its order in 64 bits (without a bias: the order of the logits), so the choice does not depend on how an
// exponential is rounded.  The work is done in 32 bits; where a choice lies closer to its neighbour among the chosen, or the last
// one to anything left out, than their 32-bit values can be wrong, and the two are not equal by construction (same logit, same
// bias), the warp ranks its candidates, or its groups, once more in 64 bits.  NaN among the logits (with groups: among the choices)
// send it over the whole token in 64 bits.
#include "b2g_common.cuh"

namespace b2g {
namespace experts {

constexpr int kWarps = 4;
constexpr int kMaxExperts = 512, kMaxTopK = 32, kMaxGroups = 32;
enum { kSoftmax = 0, kSigmoid = 1, kSqrtSoftplus = 2 };

// 64-bit key whose unsigned order is the order of the doubles; equal zeros compare equal, NaN is below every number, and 0
// (below every key) means "not to be chosen".
__device__ __forceinline__ unsigned long long key_of(double v) {
  if (v != v) return 1ull;
  const unsigned long long b = static_cast<unsigned long long>(__double_as_longlong(v + 0.0));
  return b ^ ((b >> 63) ? ~0ull : 0x8000000000000000ull);
}

__device__ __forceinline__ double score_of(double x, int fn) {
  if (fn == kSigmoid) return 1.0 / (1.0 + exp(-x));
  return sqrt(fmax(x, 0.0) + log1p(exp(-fabs(x))));
}

// Relative error 2^-20.8 at most: exponential, fast quotient and logarithm 2^-22 each, sum and root half a step.
__device__ __forceinline__ float score_of(float x, int fn) {
  const float n = expf(-fabsf(x));
  if (fn == kSigmoid) return __fdividef(x >= 0.f ? 1.f : n, 1.f + n);
  // far below 0 the logarithm is n to within n^2 / 2, and its root is exp(x / 2), which does not underflow where n does
  return x < -16.f ? expf(0.5f * x) : sqrtf(fmaxf(x, 0.f) + log1pf(n));
}

__device__ __forceinline__ unsigned long long warp_max(unsigned long long v) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) {
    const unsigned long long u = __shfl_xor_sync(0xffffffffu, v, o);
    v = u > v ? u : v;
  }
  return v;
}

template <typename T>
__device__ __forceinline__ float load_logit(const T* p, int64_t i) {
  if constexpr (sizeof(T) == 2) return __bfloat162float(p[i]);
  else return p[i];
}

// One token's scores in 64 bits: of a warp whose lanes hold its experts.
template <typename T, int kPer>
struct Exact {
  const T* row;
  const float* bias;
  int fn;
  double top, sum;
  __device__ Exact(const T* row_, const float* bias_, int fn_, int E) : row(row_), bias(bias_), fn(fn_), top(-INFINITY), sum(0.0) {
    if (fn != kSoftmax) return;
    const int first = (threadIdx.x & 31) * kPer, mine = max(0, min(kPer, E - first));
#pragma unroll 1
    for (int j = 0; j < mine; ++j) top = fmax(top, (double)load_logit(row, first + j));
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) top = fmax(top, __shfl_xor_sync(0xffffffffu, top, o));
#pragma unroll 1
    for (int j = 0; j < mine; ++j) sum += part((double)load_logit(row, first + j));
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
  }
  __device__ double part(double x) const { return top == -INFINITY && x == x ? 0.0 : exp(x - top); }
  __device__ double score(double x) const {
    if (fn != kSoftmax) return score_of(x, fn);
    const double e = part(x);
    return e == 0.0 ? 0.0 : e / sum;
  }
};

// The best M of G groups, as a bit mask, in 64 bits.  `value` holds 32 * kPer doubles of shared memory.
template <typename T, int kPer>
__device__ __noinline__ unsigned groups_in_64_bits(const T* row, const float* bias, int fn, int G, int M, int best, int E, double* value) {
  const Exact<T, kPer> exact(row, bias, fn, E);
  const int lane = threadIdx.x & 31, first = lane * kPer, mine = max(0, min(kPer, E - first)), per = E / G;
#pragma unroll 2
  for (int j = 0; j < mine; ++j) {
    const double v = exact.score((double)load_logit(row, first + j));
    value[first + j] = bias ? v + (double)bias[first + j] : v;
  }
  __syncwarp();
  unsigned long long worth = 0ull;
  if (lane < G) {
    double a = -INFINITY, b = -INFINITY;
    int at = lane % per;                       // lanes start apart, so that they meet few of one another's banks
#pragma unroll 2
    for (int i = 0; i < per; ++i) {
      const double v = value[lane * per + at];
      at = at + 1 == per ? 0 : at + 1;
      if (v > a || v != v) { b = a; a = v; }
      else if (v > b) b = v;
    }
    worth = key_of(best == 2 && per > 1 ? a + b : a);
  }
  unsigned kept = 0u;
#pragma unroll 1
  for (int r = 0; r < M; ++r) {
    const unsigned long long all = warp_max(worth);
    const int g = __ffs(__ballot_sync(0xffffffffu, worth == all)) - 1;
    kept |= 1u << g;
    if (lane == g) worth = 0ull;
  }
  __syncwarp();
  return kept;
}

// The whole route of one token in 64 bits, by one warp.  The choices live in `value` (32 * kPer doubles of shared memory) and
// everything else is computed again where it is needed: few registers, because the 32-bit pass would have to keep as many free.
template <typename T, int kPer>
__device__ __noinline__ void route_in_64_bits(const T* row, const float* bias, int fn, int G, int M, int best, int renorm, float alpha,
                                              float* weights, int64_t* indices, int E, int K, double* value) {
  const Exact<T, kPer> exact(row, bias, fn, E);
  const int lane = threadIdx.x & 31, first = lane * kPer, mine = max(0, min(kPer, E - first));
  uint32_t gone = 0u;       // bit j: expert first + j has been chosen, or its group dropped
  if (M < G) {
    const unsigned kept = groups_in_64_bits<T, kPer>(row, bias, fn, G, M, best, E, value);
    const int per = E / G;
    for (int j = 0; j < mine; ++j)
      if (!((kept >> ((first + j) / per)) & 1u)) gone |= 1u << j;
  }
#pragma unroll 1
  for (int j = 0; j < mine; ++j) {
    const double x = load_logit(row, first + j);
    value[first + j] = bias ? exact.score(x) + (double)bias[first + j] : x;
  }
  __syncwarp();
  int id = 0;         // lane r keeps the r-th choice
#pragma unroll 1
  for (int r = 0; r < K; ++r) {
    unsigned long long own = 0ull;
    int at = 0;
#pragma unroll 1
    for (int j = 0; j < mine; ++j) {
      const unsigned long long k = (gone >> j) & 1u ? 0ull : key_of(value[first + j]);
      if (k > own) { own = k; at = j; }
    }
    const unsigned long long all = warp_max(own);
    const int src = __ffs(__ballot_sync(0xffffffffu, own == all)) - 1;
    const int e = __shfl_sync(0xffffffffu, first + at, src);
    if (lane == src) gone |= 1u << at;
    if (lane == r) id = e;
  }
  const bool out = lane < K;
  const double raw = out ? (double)load_logit(row, id) : -INFINITY;
  double w = 0.0;
  if (renorm && fn == kSoftmax) {     // softmax of the chosen logits
    double m = raw;
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) m = fmax(m, __shfl_xor_sync(0xffffffffu, m, o));
    if (out) w = m == -INFINITY && raw == raw ? 0.0 : exp(raw - m);
  } else if (out) {
    w = exact.score(raw);
  }
  if (renorm) {
    double total = w;
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) total += __shfl_xor_sync(0xffffffffu, total, o);
    w = w / (total + 1e-20);
  }
  if (out) {
    weights[lane] = (float)(w * alpha);
    indices[lane] = id;
  }
}

// kPer consecutive values of a row; `wide`: 16-byte loads are aligned.
template <typename T, int kPer>
__device__ __forceinline__ void load_lane(const T* row, int first, int E, bool wide, float fill, float (&x)[kPer]) {
  constexpr int N = 16 / sizeof(T);
  if constexpr (kPer % N == 0) {
    if (wide && first + kPer <= E) {
#pragma unroll
      for (int i = 0; i < kPer; i += N) {
        const uint4 q = __ldg(reinterpret_cast<const uint4*>(row + first + i));
        const uint32_t w[4] = {q.x, q.y, q.z, q.w};
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          if constexpr (sizeof(T) == 2) { x[i + 2 * j] = dev::bf16_lo(w[j]); x[i + 2 * j + 1] = dev::bf16_hi(w[j]); }
          else x[i + j] = __uint_as_float(w[j]);
        }
      }
      return;
    }
  }
#pragma unroll
  for (int j = 0; j < kPer; ++j) x[j] = first + j < E ? load_logit(row, first + j) : fill;
}

__device__ __forceinline__ float warp_maxf(float v) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) v = fmaxf(v, __shfl_xor_sync(0xffffffffu, v, o));
  return v;
}
__device__ __forceinline__ float warp_sum(float v) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
  return v;
}

// The largest of 32 lanes' values; NaN (a lane without a value) loses against every number.
__device__ __forceinline__ float lanes_max(float v) {
  float r;
  asm volatile("redux.sync.max.f32 %0, %1, 0xffffffff;" : "=f"(r) : "f"(v));
  return r;
}

constexpr int kCandidates = 64;     // two per lane

// A candidate: the value it is chosen by, and its id.
struct Pick { float c; int id; };

template <int kPer>
struct WarpSpace {
  union {
    double value[32 * kPer];                 // the 64-bit pass
    float choice[32 * kPer];                 // groups that do not fall on lane borders
    Pick candidate[32 * kPer];
  };
  Pick sorted[kMaxTopK + 1];
  double exact[kCandidates];
};

// The best two of a group's choices.
struct Two { float a, b; };
__device__ __forceinline__ Two add_to(Two t, float v) { return Two{fmaxf(t.a, v), fmaxf(t.b, fminf(t.a, v))}; }
__device__ __forceinline__ Two merge(Two t, Two u) { return Two{fmaxf(t.a, u.a), fmaxf(fminf(t.a, u.a), fmaxf(t.b, u.b))}; }

// per = E / G; lane_shift: log2 of the lanes that hold a group where groups are whole powers of two of lanes, else -1 (the host
// divides once; eight divisions a lane cost more than the groups' arithmetic).
// kScored: the choice needs the scores (a bias, groups) or the weights need the whole row's (softmax that is not renormalised).
template <typename T, int kPer, bool kScored>
__global__ void __launch_bounds__(kWarps * 32) route_kernel(const T* __restrict__ logits, int64_t ld, const float* __restrict__ bias, int fn,
                                                            int G, int M, int best, int per, int lane_shift, int renorm, float alpha,
                                                            float* __restrict__ weights, int64_t* __restrict__ indices, int64_t tokens, int E,
                                                            int K) {
  __shared__ WarpSpace<kPer> space[kWarps];
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, first = lane * kPer;
  const int64_t t = (int64_t)blockIdx.x * kWarps + warp;
  if (t >= tokens) return;
  const T* row = logits + t * ld;
  WarpSpace<kPer>& ws = space[warp];
  const bool wide = (reinterpret_cast<uintptr_t>(row) & 15) == 0, grouped = kScored && M < G, biased = kScored && bias;
  // 32-bit scores are off by 2^-20.8 (softmax: 2^-17.5, the exponent being rounded at sizes up to 100): eps / 2; sums by half a step of
  // theirs, 2^-24, for which a quarter of kStep stands
  const float eps = fn == kSoftmax ? 1.52587890625e-5f : 1.9073486328125e-6f;
  constexpr float kStep = 2.384185791015625e-7f;

  // c[j]: what expert first + j is chosen by; NaN where there is none to choose
  float c[kPer], top = -INFINITY, denominator = 1.f, smax = 1.f;
  load_lane<T, kPer>(row, first, E, wide, kScored ? -INFINITY : NAN, c);
  const bool ragged = first + kPer > E;
  bool unsure = false;
  if constexpr (kScored) {
    float s[kPer];
    float sum = c[0];
    top = c[0];
#pragma unroll
    for (int j = 1; j < kPer; ++j) {
      sum += c[j];
      top = fmaxf(top, c[j]);
    }
    unsure = __any_sync(0xffffffffu, sum != sum);      // NaN among the logits (or infinities of both signs): left to the 64-bit pass
    top = lanes_max(top);
    if (fn == kSoftmax) {
      denominator = 0.f;
#pragma unroll
      for (int j = 0; j < kPer; ++j) {
        s[j] = top == -INFINITY || !(c[j] == c[j]) ? 0.f : expf(c[j] - top);
        denominator += s[j];
      }
      denominator = warp_sum(denominator);
      smax = 1.f / denominator;
#pragma unroll
      for (int j = 0; j < kPer; ++j) s[j] = s[j] == 0.f ? 0.f : s[j] * smax;
    } else {
#pragma unroll
      for (int j = 0; j < kPer; ++j) s[j] = score_of(c[j], fn);
      smax = score_of(top, fn);
    }
    if (biased) {
      float b[kPer];
      load_lane<float, kPer>(bias, first, E, (reinterpret_cast<uintptr_t>(bias) & 15) == 0, 0.f, b);
#pragma unroll
      for (int j = 0; j < kPer; ++j) s[j] = c[j] = s[j] + b[j];
    }
    if (grouped) {                                     // s: what the groups are compared by
      // A group's two best may cancel, so what rounding has cost them goes by the largest choice and not by their sum.
      float largest = smax;
      if (biased) {
        float all = 0.f;
#pragma unroll
        for (int j = 0; j < kPer; ++j) {
          all += fabsf(s[j]);
          largest = fmaxf(largest, fabsf(s[j]) < INFINITY ? fabsf(s[j]) : 0.f);
        }
        unsure = unsure || __any_sync(0xffffffffu, all != all);
        largest = lanes_max(largest);
      }
      Two two{-INFINITY, -INFINITY};
      int group = lane;
      if (lane_shift >= 0) {                           // its first lane speaks for a group
#pragma unroll
        for (int j = 0; j < kPer; ++j) two = add_to(two, s[j]);
        for (int o = 1; o < 1 << lane_shift; o *= 2) two = merge(two, Two{__shfl_xor_sync(0xffffffffu, two.a, o), __shfl_xor_sync(0xffffffffu, two.b, o)});
        group = (lane & ((1 << lane_shift) - 1)) == 0 ? lane >> lane_shift : G;
      } else {
#pragma unroll
        for (int j = 0; j < kPer; ++j) ws.choice[first + j] = s[j];
        __syncwarp();
        if (lane < G) {
          int at = lane % per;                         // lanes start apart, so that they meet few of one another's banks
          for (int i = 0; i < per; ++i) {
            two = add_to(two, ws.choice[lane * per + at]);
            at = at + 1 == per ? 0 : at + 1;
          }
        }
        __syncwarp();
      }
      float worth = group < G ? (best == 2 && per > 1 ? two.a + two.b : two.a) : NAN;
      unsigned kept = 0u;
      float last = 0.f;
      for (int r = 0; r <= M; ++r) {
        const float all = lanes_max(worth);
        if (r < M) {
          const int src = __ffs(__ballot_sync(0xffffffffu, worth == all)) - 1;
          kept |= 1u << __shfl_sync(0xffffffffu, group & 31, max(src, 0));
          last = all;
          if (lane == src) worth = NAN;
        } else {
          // two choices in either group, eps / 2 of a score and half a step of itself each, and half a step of their sum
          if (!(last - all > 2.f * eps * smax + 2.f * kStep * largest) && !unsure)
            kept = groups_in_64_bits<T, kPer>(row, bias, fn, G, M, best, E, ws.value);
        }
      }
      if (lane_shift >= 0) {
        const bool stays = kept >> (lane >> lane_shift) & 1u;
#pragma unroll
        for (int j = 0; j < kPer; ++j) c[j] = stays ? c[j] : NAN;
      } else {
        int g = first / per, left = (g + 1) * per - first;      // group, and how many of its experts are still to come
#pragma unroll
        for (int j = 0; j < kPer; ++j) {
          if (left == 0) { ++g; left = per; }
          --left;
          if (!(kept >> (g & 31) & 1u)) c[j] = NAN;
        }
      }
    }
    if (ragged) {
#pragma unroll
      for (int j = 0; j < kPer; ++j)
        if (first + j >= E) c[j] = NAN;
    }
  }

  // Candidates: everything not below the L-th largest lane maximum, L = the ranks that are looked at (with a bias, whether the
  // last choice is clear of the first one left out).  At least L of them, hardly ever more than 2 L, whatever the order is.
  const int ranks = K + (biased ? 1 : 0);
  float head = c[0], floor_value = -INFINITY;
#pragma unroll
  for (int j = 1; j < kPer; ++j) head = fmaxf(head, c[j]);
  if (ranks <= 32) {
    for (int r = 0; r < ranks; ++r) {
      floor_value = lanes_max(head);
      if (head == floor_value) head = NAN;
    }
    if (floor_value != floor_value) floor_value = -INFINITY;
    // so that nothing outside can belong among the first K even if the 32-bit choices are wrong
    if (biased) floor_value -= 2.f * eps * smax + kStep * 2.f * fabsf(floor_value);
  }
  int n = 0;
#pragma unroll
  for (int j = 0; j < kPer; ++j) {
    const bool in = c[j] >= floor_value;
    const unsigned mask = __ballot_sync(0xffffffffu, in);
    if (in) ws.candidate[n + __popc(mask & ((1u << lane) - 1u))] = Pick{c[j], first + j};
    n += __popc(mask);
  }
  unsure = unsure || n > kCandidates || n < K;         // few: there are NaN among the logits
  if (!unsure) {
    __syncwarp();
    {
      const Pick mine = lane < n ? ws.candidate[lane] : Pick{0.f, 0};
      int rank = 0;
#pragma unroll 4
      for (int q = 0; q < n; ++q) {
        const Pick o = ws.candidate[q];
        rank += o.c > mine.c || (o.c == mine.c && o.id < mine.id);
      }
      if (lane < n && rank < ranks) ws.sorted[rank] = mine;
    }
    if (n > 32) {
      const Pick mine = lane + 32 < n ? ws.candidate[lane + 32] : Pick{0.f, 0};
      int rank = 0;
#pragma unroll 4
      for (int q = 0; q < n; ++q) {
        const Pick o = ws.candidate[q];
        rank += o.c > mine.c || (o.c == mine.c && o.id < mine.id);
      }
      if (lane + 32 < n && rank < ranks) ws.sorted[rank] = mine;
    }
    __syncwarp();
    const bool out = lane < K;
    Pick p = out ? ws.sorted[lane] : Pick{0.f, 0};
    if (biased) {
      // What a 32-bit choice may be off by: a score is at most its choice less its bias, give or take a step.
      auto slack = [&](float choice, float b) { return 0.5f * eps * fabsf(choice - b) + kStep * (fabsf(choice) + fabsf(b)); };
      auto near = [&](const Pick& u, const Pick& v) {  // u.c >= v.c: is v before u in 64 bits, for all that is known?
        const float bu = bias[u.id], bv = bias[v.id];
        return !(u.c - v.c > slack(u.c, bu) + slack(v.c, bv)) && !(bu == bv && load_logit(row, u.id) == load_logit(row, v.id));
      };
      bool close = out && lane + 1 < K && near(p, ws.sorted[lane + 1]);
      // The border: anything that was left out, not only the first of it.  One of a large score under a large negative bias may be
      // off by more than the others, and one that equals the last choice by construction says nothing about those behind it.
      const Pick last = ws.sorted[K - 1];
      const float reach = eps * smax + 2.f * kStep * (smax + fabsf(last.c));
      for (int h = lane; h < n; h += 32) {
        const Pick o = ws.candidate[h];
        const bool left_out = o.c < last.c || (o.c == last.c && o.id > last.id);
        if (left_out && !(last.c - o.c > reach + 2.f * kStep * fabsf(o.c))) close = close || near(last, o);
      }
      if (__any_sync(0xffffffffu, close)) {            // the candidates once more, in 64 bits
        double all = 1.0;
        const bool nothing = top == -INFINITY;         // every score is 0
        if (fn == kSoftmax && !nothing) {
          float x[kPer];
          load_lane<T, kPer>(row, first, E, wide, -INFINITY, x);
          all = 0.0;
#pragma unroll
          for (int j = 0; j < kPer; ++j) all += exp((double)x[j] - (double)top);
#pragma unroll
          for (int o = 16; o > 0; o >>= 1) all += __shfl_xor_sync(0xffffffffu, all, o);
        }
        for (int h = lane; h < n; h += 32) {
          const int id = ws.candidate[h].id;
          const double x = load_logit(row, id);
          ws.exact[h] = (fn != kSoftmax ? score_of(x, fn) : nothing ? 0.0 : exp(x - (double)top) / all) + (double)bias[id];
        }
        __syncwarp();
        for (int h = lane; h < n; h += 32) {
          const double mine = ws.exact[h];
          const int id = ws.candidate[h].id;
          int rank = 0;
          for (int q = 0; q < n; ++q) rank += ws.exact[q] > mine || (ws.exact[q] == mine && ws.candidate[q].id < id);
          if (rank < K) ws.sorted[rank] = ws.candidate[h];
        }
        __syncwarp();
        if (out) p = ws.sorted[lane];
      }
    }
    const float x = biased || grouped ? load_logit(row, p.id) : p.c;
    float w = 0.f;
    if (fn == kSoftmax) {
      if (kScored) w = top == -INFINITY ? 0.f : expf(x - top) / denominator;
    } else {
      w = score_of(x, fn);
    }
    if (!out) w = 0.f;
    if (renorm) {
      if (fn == kSoftmax) {
        const float m = kScored ? warp_maxf(out ? x : -INFINITY) : __shfl_sync(0xffffffffu, x, 0);
        w = !out || m == -INFINITY ? 0.f : expf(x - m);
      }
      w = w / (warp_sum(w) + 1e-20f);
    }
    if (out) {
      weights[t * K + lane] = w * alpha;
      indices[t * K + lane] = p.id;
    }
  } else {
    __syncwarp();
    route_in_64_bits<T, kPer>(row, bias, fn, G, M, best, renorm, alpha, weights + t * K, indices + t * K, E, K, ws.value);
  }
}

// dl from dw.  With u_j = w_j / alpha and dot = sum_i g_i w_i:  renormalised ds_j s_j = u_j (alpha g_j - dot), else ds_j s_j = g_j w_j;
// the slopes of the score functions relative to the score are 1 - sigmoid (sigmoid), sigmoid / (2 softplus) (sqrtsoftplus) and
// 1 (softmax, whose common denominator cancels when renormalised and otherwise gives every expert - s_e * dot).
// The choices' own terms are in 64 bits, from the logits and not from the weights that fp32 has rounded, and each product is rounded
// before the difference: alpha g_j - dot cancels where one expert has nearly all the weight, and with a single choice it is 0 and
// has to come out as 0.  Softmax that is not renormalised needs the sum over the row for that; its 32-bit exponentials are added in
// 64 bits, so that the rest beside a dominant one keeps its digits.
// A warp takes kTokens tokens at once, 32 / kTokens lanes on the choices of each, and then writes their rows one after the other:
// with one token a warp spent most of its time waiting for three short loads (65536 x 256 bf16, top 8: 16 us, 13.5 us with four).
template <typename T, int kPer, int kTokens>
__global__ void __launch_bounds__(kWarps * 32) route_bwd_kernel(const T* __restrict__ logits, int64_t ld, const float* __restrict__ grad_w,
                                                                const int64_t* __restrict__ indices, int fn, int renorm, float alpha,
                                                                T* __restrict__ grad, int64_t tokens, int E, int K) {
  constexpr int N = 16 / sizeof(T), kLanes = 32 / kTokens, kNotChosen = 0x7FC0DEAD;      // a NaN that no arithmetic gives
  __shared__ __align__(16) float value[kWarps][kTokens][32 * kPer];
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, first = lane * kPer, mine = lane / kLanes, slot = lane % kLanes;
  const int64_t t0 = ((int64_t)blockIdx.x * kWarps + warp) * kTokens, t = t0 + mine;
  if (t0 >= tokens) return;
  const bool in = t < tokens && slot < K;
  const float g = in ? grad_w[t * K + slot] : 0.f;
  const int64_t e64 = in ? indices[t * K + slot] : -1;
  const bool ok = e64 >= 0 && e64 < E;
  const int e = ok ? (int)e64 : 0;
  const float raw = ok ? load_logit(logits + t * ld, e) : 0.f;
  const bool whole_row = fn == kSoftmax && !renorm;
#pragma unroll
  for (int u = 0; u < kTokens; ++u)
#pragma unroll
    for (int j = 0; j < kPer; ++j) value[warp][u][first + j] = whole_row ? __int_as_float(kNotChosen) : 0.f;
  const double g64 = g, raw64 = raw;
  double own = 0.0, part = 0.0, total = 1.0;         // a score, its weight, and what it was divided by
  if (!whole_row) {
    if (fn == kSoftmax) {                            // of the chosen logits
      float m = ok ? raw : -INFINITY;
#pragma unroll
      for (int o = kLanes / 2; o > 0; o >>= 1) m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, o));
      own = !ok || (m == -INFINITY && raw == raw) ? 0.0 : exp(raw64 - (double)m);
    } else {
      own = ok ? score_of(raw64, fn) : 0.0;
    }
    if (renorm) {
      total = own;
#pragma unroll
      for (int o = kLanes / 2; o > 0; o >>= 1) total += __shfl_xor_sync(0xffffffffu, total, o);
      total += 1e-20;
    }
    part = __dmul_rn((double)alpha, own) / total;
  }
  double dot = __dmul_rn(g64, part);
#pragma unroll
  for (int o = kLanes / 2; o > 0; o >>= 1) dot += __shfl_xor_sync(0xffffffffu, dot, o);
  double slope = __dmul_rn((double)alpha, g64);      // dL/ds
  if (renorm) slope = __dadd_rn(slope, -dot) / total;
  double d;
  if (fn == kSoftmax) {
    d = slope * own;                                 // the slope is divided by the sum of the choices
  } else {
    const double sig = 1.0 / (1.0 + exp(-raw64));
    if (fn == kSigmoid) d = slope * (sig * (1.0 / (1.0 + exp(raw64))));
    else d = raw64 < -600.0 ? slope * 0.5 * own : slope * (sig / (2.0 * own));      // far below 0 both are e^(x/2) / 2
  }
  __syncwarp();
  if (ok && !whole_row) value[warp][mine][e] = (float)d;
  __syncwarp();
#pragma unroll
  for (int u = 0; u < kTokens; ++u) {
    if (t0 + u >= tokens) return;
    float v[kPer];
    if (!whole_row) {
#pragma unroll
      for (int j = 0; j < kPer; ++j) v[j] = value[warp][u][first + j];
    } else {                                         // every expert has its share; the choices' entries go through shared memory
      const T* row = logits + (t0 + u) * ld;
      float x[kPer];
      load_lane<T, kPer>(row, first, E, (reinterpret_cast<uintptr_t>(row) & 15) == 0, -INFINITY, x);
      float top = x[0];
#pragma unroll
      for (int j = 1; j < kPer; ++j) top = fmaxf(top, x[j]);
      top = warp_maxf(top);
      double sum = 0.0;
#pragma unroll
      for (int j = 0; j < kPer; ++j) {
        x[j] = top == -INFINITY && x[j] == x[j] ? 0.f : expf(x[j] - top);
        sum += (double)x[j];
      }
#pragma unroll
      for (int o = 16; o > 0; o >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
      const bool chosen = ok && mine == u;
      const double s = !chosen || (top == -INFINITY && raw == raw) ? 0.0 : exp(raw64 - (double)top) / sum;
      double of_row = chosen ? __dmul_rn(__dmul_rn((double)alpha, g64), s) : 0.0;
#pragma unroll
      for (int o = 16; o > 0; o >>= 1) of_row += __shfl_xor_sync(0xffffffffu, of_row, o);
      const float each = (float)(of_row / sum);
      if (chosen) value[warp][u][e] = (float)(s * __dadd_rn(__dmul_rn((double)alpha, g64), -of_row));
      __syncwarp();
#pragma unroll
      for (int j = 0; j < kPer; ++j) {
        v[j] = value[warp][u][first + j];
        if (__float_as_int(v[j]) == kNotChosen) v[j] = x[j] == 0.f ? 0.f : -x[j] * each;
      }
    }
    T* out = grad + (t0 + u) * (int64_t)E;
    bool written = false;
    if constexpr (kPer % N == 0) {
      if (first + kPer <= E && (reinterpret_cast<uintptr_t>(out) & 15) == 0) {
        written = true;
#pragma unroll
        for (int i = 0; i < kPer; i += N) {
          uint4 q;
          if constexpr (sizeof(T) == 2)
            q = make_uint4(dev::pack_bf16(v[i], v[i + 1]), dev::pack_bf16(v[i + 2], v[i + 3]), dev::pack_bf16(v[i + 4], v[i + 5]),
                           dev::pack_bf16(v[i + 6], v[i + 7]));
          else
            q = make_uint4(__float_as_uint(v[i]), __float_as_uint(v[i + 1]), __float_as_uint(v[i + 2]), __float_as_uint(v[i + 3]));
          *reinterpret_cast<uint4*>(out + first + i) = q;
        }
      }
    }
    if (!written) {
#pragma unroll
      for (int j = 0; j < kPer; ++j) {
        if (first + j < E) {
          if constexpr (sizeof(T) == 2) out[first + j] = __float2bfloat16_rn(v[j]);
          else out[first + j] = v[j];
        }
      }
    }
  }
}

}  // namespace experts
}  // namespace b2g

using namespace b2g;

static int check_route(const char* what, const void* logits, int64_t ld, int dtype, int fn, float alpha, int64_t T, int E, int K) {
  B2G_REQUIRE(T >= 0 && T < (1ll << 31), "%s: bad token count %lld", what, (long long)T);
  B2G_REQUIRE(E >= 1 && E <= experts::kMaxExperts, "%s: %d experts outside 1..%d", what, E, experts::kMaxExperts);
  B2G_REQUIRE(K >= 1 && K <= E && K <= experts::kMaxTopK, "%s: top_k=%d outside 1..%d", what, K, E < experts::kMaxTopK ? E : experts::kMaxTopK);
  B2G_REQUIRE(dtype == 0 || dtype == 1, "%s: logits_dtype must be 0 (bf16) or 1 (fp32)", what);
  B2G_REQUIRE(fn >= 0 && fn <= 2, "%s: score_fn must be 0 (softmax), 1 (sigmoid) or 2 (sqrtsoftplus)", what);
  B2G_REQUIRE(alpha > 0.f && alpha <= 3.4e38f, "%s: the scaling factor must be positive and finite", what);
  B2G_REQUIRE(T <= 1 || ld >= E, "%s: row pitch %lld below %d experts", what, (long long)ld, E);
  B2G_REQUIRE(T == 0 || logits, "%s: null pointer", what);
  return 0;
}

// The narrowest instance whose 32 lanes hold E experts.
#define B2G_BY_EXPERTS(E, LAUNCH)      \
  do {                                 \
    if ((E) <= 32) { LAUNCH(1); }      \
    else if ((E) <= 64) { LAUNCH(2); } \
    else if ((E) <= 128) { LAUNCH(4); } \
    else if ((E) <= 256) { LAUNCH(8); } \
    else { LAUNCH(16); }               \
  } while (0)

extern "C" int b2g_route_experts(const void* logits, int64_t ld, int logits_dtype, const float* bias, int score_fn, int groups, int top_groups,
                                 int group_experts, int renormalize, float scaling, float* weights, int64_t* indices, int64_t T, int E,
                                 int top_k, void* stream) {
  if (int rc = check_route("route_experts", logits, ld, logits_dtype, score_fn, scaling, T, E, top_k)) return rc;
  B2G_REQUIRE(groups >= 1 && groups <= experts::kMaxGroups && E % groups == 0, "route_experts: %d groups do not split %d experts evenly (or exceed %d)",
              groups, E, experts::kMaxGroups);
  B2G_REQUIRE(top_groups >= 1 && top_groups <= groups, "route_experts: top_groups=%d outside 1..%d", top_groups, groups);
  B2G_REQUIRE(top_k <= top_groups * (E / groups), "route_experts: top_k=%d exceeds the %d experts of the kept groups", top_k,
              top_groups * (E / groups));
  B2G_REQUIRE(group_experts == 1 || group_experts == 2, "route_experts: group_experts must be 1 or 2");
  if (T == 0) return 0;
  B2G_REQUIRE(weights && indices, "route_experts: null pointer");
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  const int blocks = (int)((T + experts::kWarps - 1) / experts::kWarps);
  const bool scored = bias || top_groups < groups || (score_fn == experts::kSoftmax && !renormalize);
  const int per_group = E / groups;
  auto lane_shift = [&](int per_lane) {
    for (int shift = 0; shift <= 5; ++shift)
      if (per_group == per_lane << shift) return shift;
    return -1;
  };
#define B2G_ROUTE_AS(TYPE, PER, SCORED)                                                                                                \
  experts::route_kernel<TYPE, PER, SCORED><<<blocks, experts::kWarps * 32, 0, s>>>(static_cast<const TYPE*>(logits), ld, bias, score_fn, groups, \
      top_groups, group_experts, per_group, lane_shift(PER), renormalize, scaling, weights, indices, T, E, top_k)
#define B2G_ROUTE(PER)                                                   \
  do {                                                                   \
    if (logits_dtype) {                                                  \
      if (scored) B2G_ROUTE_AS(float, PER, true);                        \
      else B2G_ROUTE_AS(float, PER, false);                              \
    } else {                                                             \
      if (scored) B2G_ROUTE_AS(__nv_bfloat16, PER, true);                \
      else B2G_ROUTE_AS(__nv_bfloat16, PER, false);                      \
    }                                                                    \
  } while (0)
  B2G_BY_EXPERTS(E, B2G_ROUTE);
  B2G_CUDA_OK(cudaGetLastError());
  return 0;
}

extern "C" int b2g_route_experts_bwd(const void* logits, int64_t ld, int logits_dtype, const float* grad_weights, const float* weights,
                                     const int64_t* indices, int score_fn, int renormalize, float scaling, void* grad_logits, int64_t T, int E,
                                     int top_k, void* stream) {
  if (int rc = check_route("route_experts_bwd", logits, ld, logits_dtype, score_fn, scaling, T, E, top_k)) return rc;
  if (T == 0) return 0;
  B2G_REQUIRE(grad_weights && indices && grad_logits, "route_experts_bwd: null pointer");
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  // four tokens a warp where their choices fit its lanes and there are tokens for all SMs
  const int tokens = top_k <= 8 && T >= 8192 ? 4 : 1;
  const int blocks = (int)((T + experts::kWarps * tokens - 1) / (experts::kWarps * tokens));
#define B2G_ROUTE_BWD_AS(TYPE, PER, TOKENS)                                                                                                \
  experts::route_bwd_kernel<TYPE, PER, TOKENS><<<blocks, experts::kWarps * 32, 0, s>>>(static_cast<const TYPE*>(logits), ld, grad_weights, \
      indices, score_fn, renormalize, scaling, static_cast<TYPE*>(grad_logits), T, E, top_k)
#define B2G_ROUTE_BWD(PER)                                              \
  do {                                                                  \
    if (logits_dtype) {                                                 \
      if (tokens == 4) B2G_ROUTE_BWD_AS(float, PER, 4);                 \
      else B2G_ROUTE_BWD_AS(float, PER, 1);                             \
    } else {                                                            \
      if (tokens == 4) B2G_ROUTE_BWD_AS(__nv_bfloat16, PER, 4);         \
      else B2G_ROUTE_BWD_AS(__nv_bfloat16, PER, 1);                     \
    }                                                                   \
  } while (0)
  B2G_BY_EXPERTS(E, B2G_ROUTE_BWD);
  B2G_CUDA_OK(cudaGetLastError());
  return 0;
}
