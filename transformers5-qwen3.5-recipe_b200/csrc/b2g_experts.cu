// Routing to experts: scores, balance bias, groups, top-k and renormalised weights, with the gradient of the logits.
//   s = softmax(l) | sigmoid(l) | sqrt(log(1 + e^l)),  c = s + b,  best M of G groups by the sum of their n best c,
//   best k of c in them,  w_j = alpha s_j / (sum_i s_i + 1e-20)  or  alpha s_j.
// Softmax weights that are renormalised are the softmax of the chosen logits (the common denominator cancels).
// One warp per token; lane i holds experts [i * kPer, (i + 1) * kPer), so the lowest lane of a tie holds the lowest expert.
// The order of c is its order in 64 bits (without a bias: the order of the logits), so the choice does not depend on how an
// exponential is rounded.
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

template <typename T, int kPer>
__global__ void __launch_bounds__(kWarps * 32) route_kernel(const T* __restrict__ logits, int64_t ld, const float* __restrict__ bias, int fn,
                                                            int G, int M, int best, int renorm, float alpha, float* __restrict__ weights,
                                                            int64_t* __restrict__ indices, int64_t tokens, int E, int K) {
  __shared__ double value[kWarps][32 * kPer];
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int64_t t = (int64_t)blockIdx.x * kWarps + warp;
  if (t >= tokens) return;
  const T* row = logits + t * ld;
  double x[kPer], s[kPer];
  double top = -INFINITY;
#pragma unroll
  for (int j = 0; j < kPer; ++j) {
    const int e = lane * kPer + j;
    x[j] = e < E ? (double)load_logit(row, e) : -INFINITY;
    top = fmax(top, x[j]);
  }
  if (fn == kSoftmax) {
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) top = fmax(top, __shfl_xor_sync(0xffffffffu, top, o));
    double sum = 0.0;
#pragma unroll
    for (int j = 0; j < kPer; ++j) {
      s[j] = top == -INFINITY && x[j] == x[j] ? 0.0 : exp(x[j] - top);
      sum += s[j];
    }
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
#pragma unroll
    for (int j = 0; j < kPer; ++j) s[j] = s[j] == 0.0 ? 0.0 : s[j] / sum;
  } else {
#pragma unroll
    for (int j = 0; j < kPer; ++j) s[j] = score_of(x[j], fn);
  }
  unsigned long long key[kPer];
#pragma unroll
  for (int j = 0; j < kPer; ++j) {
    const int e = lane * kPer + j;
    key[j] = e < E ? key_of(bias ? s[j] + (double)bias[e] : x[j]) : 0ull;
  }
  if (M < G) {
    const int per = E / G;
#pragma unroll
    for (int j = 0; j < kPer; ++j) {
      const int e = lane * kPer + j;
      value[warp][e] = e < E ? (bias ? s[j] + (double)bias[e] : s[j]) : 0.0;
    }
    __syncwarp();
    unsigned long long mine = 0ull;
    if (lane < G) {
      double a = -INFINITY, b = -INFINITY;
      for (int i = 0; i < per; ++i) {
        const double v = value[warp][lane * per + i];
        if (v > a || v != v) { b = a; a = v; }
        else if (v > b) b = v;
      }
      mine = key_of(best == 2 && per > 1 ? a + b : a);
    }
    unsigned kept = 0u;
    for (int r = 0; r < M; ++r) {
      const unsigned long long all = warp_max(mine);
      const int g = __ffs(__ballot_sync(0xffffffffu, mine == all)) - 1;
      kept |= 1u << g;
      if (lane == g) mine = 0ull;
    }
#pragma unroll
    for (int j = 0; j < kPer; ++j) {
      const int e = lane * kPer + j;
      if (e < E && !((kept >> (e / per)) & 1u)) key[j] = 0ull;
    }
  }
  int id = 0;         // lane r keeps the r-th choice
  double picked = 0.0, raw = -INFINITY;
  for (int r = 0; r < K; ++r) {
    unsigned long long own = key[0];
    int at = 0;
#pragma unroll
    for (int j = 1; j < kPer; ++j)
      if (key[j] > own) { own = key[j]; at = j; }
    const unsigned long long all = warp_max(own);
    const int src = __ffs(__ballot_sync(0xffffffffu, own == all)) - 1;
    double sj = 0.0, xj = 0.0;
#pragma unroll
    for (int j = 0; j < kPer; ++j)
      if (j == at) { sj = s[j]; xj = x[j]; if (lane == src) key[j] = 0ull; }
    const int ej = __shfl_sync(0xffffffffu, lane * kPer + at, src);
    sj = __shfl_sync(0xffffffffu, sj, src);
    xj = __shfl_sync(0xffffffffu, xj, src);
    if (lane == r) { id = ej; picked = sj; raw = xj; }
  }
  const bool out = lane < K;
  double w = out ? picked : 0.0;
  if (renorm) {
    if (fn == kSoftmax) {     // softmax of the chosen logits
      double m = out ? raw : -INFINITY;
#pragma unroll
      for (int o = 16; o > 0; o >>= 1) m = fmax(m, __shfl_xor_sync(0xffffffffu, m, o));
      w = !out ? 0.0 : (m == -INFINITY && raw == raw ? 0.0 : exp(raw - m));
    }
    double sum = w;
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
    w = w / (sum + 1e-20);
  }
  if (out) {
    weights[t * K + lane] = (float)(w * alpha);
    indices[t * K + lane] = id;
  }
}

// dl from dw.  With u_j = w_j / alpha and dot = sum_i g_i w_i:  renormalised ds_j s_j = u_j (alpha g_j - dot), else ds_j s_j = g_j w_j;
// the slopes of the score functions relative to the score are 1 - sigmoid (sigmoid), sigmoid / (2 softplus) (sqrtsoftplus) and
// 1 (softmax, whose common denominator cancels when renormalised and otherwise gives every expert - s_e * dot).
template <typename T, int kPer>
__global__ void __launch_bounds__(kWarps * 32) route_bwd_kernel(const T* __restrict__ logits, int64_t ld, const float* __restrict__ grad_w,
                                                                const float* __restrict__ weights, const int64_t* __restrict__ indices, int fn,
                                                                int renorm, float alpha, T* __restrict__ grad, int64_t tokens, int E, int K) {
  __shared__ float value[kWarps][32 * kPer];
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int64_t t = (int64_t)blockIdx.x * kWarps + warp;
  if (t >= tokens) return;
  const T* row = logits + t * ld;
  const bool in = lane < K;
  const float g = in ? grad_w[t * K + lane] : 0.f, w = in ? weights[t * K + lane] : 0.f;
  const int64_t e64 = in ? indices[t * K + lane] : -1;
  const bool ok = e64 >= 0 && e64 < E;
  const int e = ok ? (int)e64 : 0;
  float dot = g * w;
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) dot += __shfl_xor_sync(0xffffffffu, dot, o);
  float d = renorm ? (w / alpha) * (alpha * g - dot) : g * w;
  if (ok && fn != kSoftmax) {
    const float x = load_logit(row, e);
    const float n = expf(-fabsf(x));
    const float sig = x >= 0.f ? 1.f / (1.f + n) : n / (1.f + n);
    if (fn == kSigmoid) d *= x >= 0.f ? n / (1.f + n) : 1.f / (1.f + n);
    else d *= x < -16.f ? 0.5f : sig / (2.f * (fmaxf(x, 0.f) + log1pf(n)));
  }
  for (int j = lane; j < E; j += 32) value[warp][j] = 0.f;
  __syncwarp();
  if (ok) value[warp][e] = d;
  __syncwarp();
  T* out = grad + t * (int64_t)E;
  float x[kPer], top = -INFINITY, sum = 0.f;
  const bool full = fn == kSoftmax && !renorm;
  if (full) {
#pragma unroll
    for (int j = 0; j < kPer; ++j) {
      const int i = j * 32 + lane;
      x[j] = i < E ? load_logit(row, i) : -INFINITY;
      top = fmaxf(top, x[j]);
    }
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, o));
#pragma unroll
    for (int j = 0; j < kPer; ++j) {
      x[j] = top == -INFINITY && x[j] == x[j] ? 0.f : expf(x[j] - top);
      sum += x[j];
    }
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
  }
#pragma unroll
  for (int j = 0; j < kPer; ++j) {
    const int i = j * 32 + lane;
    if (i < E) {
      float v = value[warp][i];
      if (full) v -= x[j] == 0.f ? 0.f : x[j] / sum * dot;
      if constexpr (sizeof(T) == 2) out[i] = __float2bfloat16_rn(v);
      else out[i] = v;
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
#define B2G_ROUTE(PER)                                                                                                                  \
  if (logits_dtype)                                                                                                                     \
    experts::route_kernel<float, PER><<<blocks, experts::kWarps * 32, 0, s>>>(static_cast<const float*>(logits), ld, bias, score_fn, groups, \
        top_groups, group_experts, renormalize, scaling, weights, indices, T, E, top_k);                                                \
  else                                                                                                                                  \
    experts::route_kernel<__nv_bfloat16, PER><<<blocks, experts::kWarps * 32, 0, s>>>(static_cast<const __nv_bfloat16*>(logits), ld, bias, \
        score_fn, groups, top_groups, group_experts, renormalize, scaling, weights, indices, T, E, top_k)
  B2G_BY_EXPERTS(E, B2G_ROUTE);
  B2G_CUDA_OK(cudaGetLastError());
  return 0;
}

extern "C" int b2g_route_experts_bwd(const void* logits, int64_t ld, int logits_dtype, const float* grad_weights, const float* weights,
                                     const int64_t* indices, int score_fn, int renormalize, float scaling, void* grad_logits, int64_t T, int E,
                                     int top_k, void* stream) {
  if (int rc = check_route("route_experts_bwd", logits, ld, logits_dtype, score_fn, scaling, T, E, top_k)) return rc;
  if (T == 0) return 0;
  B2G_REQUIRE(grad_weights && weights && indices && grad_logits, "route_experts_bwd: null pointer");
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  const int blocks = (int)((T + experts::kWarps - 1) / experts::kWarps);
#define B2G_ROUTE_BWD(PER)                                                                                                                 \
  if (logits_dtype)                                                                                                                        \
    experts::route_bwd_kernel<float, PER><<<blocks, experts::kWarps * 32, 0, s>>>(static_cast<const float*>(logits), ld, grad_weights, weights, \
        indices, score_fn, renormalize, scaling, static_cast<float*>(grad_logits), T, E, top_k);                                           \
  else                                                                                                                                     \
    experts::route_bwd_kernel<__nv_bfloat16, PER><<<blocks, experts::kWarps * 32, 0, s>>>(static_cast<const __nv_bfloat16*>(logits), ld,   \
        grad_weights, weights, indices, score_fn, renormalize, scaling, static_cast<__nv_bfloat16*>(grad_logits), T, E, top_k)
  B2G_BY_EXPERTS(E, B2G_ROUTE_BWD);
  B2G_CUDA_OK(cudaGetLastError());
  return 0;
}
