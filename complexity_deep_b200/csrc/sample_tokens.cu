// The next token of every row of logits, from a given uniform number u:
//
//   w_i = exp((x_i - max) / T);  top-k: x_i at least the k-th largest (ties stay);  top-p: in descending order, ties by the lowest
//   index, i stays where the mass ahead of it is at most p times the mass that top-k has left;  min-p: w_i >= min_p;
//   id = the first i, in the order of the vocabulary, with sum_{j <= i} w_j > u sum_j w_j over what stayed.
//
// The result is a whole number that hangs on where sums lie next to a border, so weights are 64-bit exponentials, held as multiples
// of 2^-44: sums of up to 2^18 of them are exact, and the same in any order.
//
// One block a row; the row is read again (from L2) by every pass. The k-th largest value and the last value of the nucleus are found
// digit by digit, by counts and by masses.
#include <cuda_bf16.h>
#include <cuda_runtime.h>
#include "elem.cuh"
#include "kernels.h"
#include "ptx.cuh"

namespace cdeep {

namespace {

constexpr int kThreads = 1024;
constexpr double kOne = 17592186044416.0;                 // 2^44
using u64 = unsigned long long;

// Order of logits as unsigned numbers; NaN below -inf.
__device__ __forceinline__ uint32_t key_of(float x) {
  const uint32_t u = __float_as_uint(x + 0.f);
  return x != x ? 0u : u & 0x80000000u ? ~u : u | 0x80000000u;
}
__device__ __forceinline__ float value_of(uint32_t k) { return __uint_as_float(k & 0x80000000u ? k & 0x7fffffffu : ~k); }
constexpr uint32_t kMinusInf = 0x007fffffu;

__device__ __forceinline__ u64 fraction(float f) {        // of 2^64, f clamped to [0, 1)
  return f > 0.f ? f < 1.f ? static_cast<u64>(static_cast<double>(f) * 18446744073709551616.0) : ~0ull : 0ull;
}

template <typename V>
__device__ __forceinline__ V block_sum(V v, V* s) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
  __syncthreads();
  if ((threadIdx.x & 31) == 0) s[threadIdx.x >> 5] = v;
  __syncthreads();
  v = 0;
  for (int w = 0; w < kThreads / 32; ++w) v += s[w];
  return v;
}
// Sum over the threads ahead of this one.
template <typename V>
__device__ __forceinline__ V block_before(V v, V* s) {
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  V in = v;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const V up = __shfl_up_sync(0xffffffffu, in, o);
    if (lane >= o) in += up;
  }
  __syncthreads();
  if (lane == 31) s[warp] = in;
  __syncthreads();
  V before = in - v;
  for (int w = 0; w < warp; ++w) before += s[w];
  return before;
}

template <typename T>
__global__ void __launch_bounds__(kThreads) sample_tokens_kernel(const T* logits, long long ld, int V, cd_sample p, long long* ids,
                                                                 float* probs) {
  __shared__ u64 s_hist[256], s_sum[32];
  __shared__ unsigned s_key;
  __shared__ u64 s_left;
  __shared__ int s_id;
  griddep_wait();
  griddep_launch_dependents();
  const int b = blockIdx.x, tid = threadIdx.x;
  const T* x = logits + b * ld;
  const float temperature = p.temperatures ? p.temperatures[b] : p.temperature;
  const float top_p = p.top_ps ? p.top_ps[b] : p.top_p;
  const double min_p = fmin(1.0, static_cast<double>(p.min_ps ? p.min_ps[b] : p.min_p));
  const int top_k = p.top_ks ? p.top_ks[b] : p.top_k;
  if (tid == 0) s_key = 0, s_id = V;
  __syncthreads();
  unsigned best = 0;
  for (int i = tid; i < V; i += kThreads) best = max(best, key_of(to_f32(x[i])));
  atomicMax(&s_key, best);
  __syncthreads();
  best = s_key;
  __syncthreads();
  if (best <= kMinusInf) {                                // nothing to draw from
    if (tid == 0) ids[b] = 0, probs[b] = 0.f;
    return;
  }
  if (!(temperature > 0.f)) {
    for (int i = tid; i < V; i += kThreads)
      if (key_of(to_f32(x[i])) == best) {
        atomicMin(&s_id, i);
        break;
      }
    __syncthreads();
    if (tid == 0) ids[b] = s_id, probs[b] = 1.f;
    return;
  }
  const double top = value_of(best), inv_t = 1.0 / static_cast<double>(temperature);
  auto weight = [&](unsigned k) -> double {
    if (k == best) return 1.0;
    return k <= kMinusInf ? 0.0 : exp((static_cast<double>(value_of(k)) - top) * inv_t);
  };
  auto fixed = [&](unsigned k) { return static_cast<u64>(weight(k) * kOne + 0.5); };

  // The lowest value of a digit-by-digit walk from the largest on: by counts (the `left`-th value), or by masses (the last value that
  // has at most `left` ahead of it). Returns it with what is left of `left` at it.
  auto walk = [&](unsigned from, bool masses, u64& left) -> unsigned {
    unsigned prefix = 0;
    for (int shift = 24; shift >= 0; shift -= 8) {
      __syncthreads();
      if (tid < 256) s_hist[tid] = 0;
      __syncthreads();
      for (int i = tid; i < V; i += kThreads) {
        const unsigned k = key_of(to_f32(x[i]));
        if (k >= from && (shift == 24 || (k >> (shift + 8)) == (prefix >> (shift + 8))))
          atomicAdd(&s_hist[k >> shift & 255], masses ? fixed(k) : 1ull);
      }
      __syncthreads();
      if (tid == 0) {
        // counts: the first digit at which `left` values are reached; masses: the last with at most `left` ahead of it
        int d = 255, last = -1;
        u64 ahead = 0, at = 0;
        for (; d >= 0; --d) {
          if (s_hist[d] == 0) continue;
          if (masses ? ahead > left : last >= 0 && ahead >= left) break;
          last = d;
          at = ahead;
          ahead += s_hist[d];
        }
        s_key = last;
        s_left = left - at;
      }
      __syncthreads();
      prefix |= s_key << shift;
      left = s_left;
    }
    return prefix;
  };

  unsigned from = kMinusInf + 1;
  if (top_k > 0 && top_k < V) {
    u64 left = top_k;
    from = max(from, walk(0, false, left));
  }
  unsigned border = from;                                 // equal values from here on are counted
  u64 ties = ~0ull;                                       // how many values equal to the border stay
  if (top_p < 1.f) {
    u64 sum = 0;
    for (int i = tid; i < V; i += kThreads) {
      const unsigned k = key_of(to_f32(x[i]));
      if (k >= from) sum += fixed(k);
    }
    u64 left = __umul64hi(fraction(top_p), block_sum(sum, s_sum));
    border = walk(from, true, left);
    const u64 w = fixed(border);
    if (w > 0) ties = left / w + 1;
  }

  // A run of neighbouring tokens per thread.
  const int run = (V + kThreads - 1) / kThreads, lo = min(V, tid * run), hi = min(V, lo + run);
  u64 count = 0;
  for (int i = lo; i < hi; ++i) count += key_of(to_f32(x[i])) == border;
  const u64 ties_before = block_before(count, s_sum);
  auto mass = [&](int i, u64& tie) -> u64 {
    const unsigned k = key_of(to_f32(x[i]));
    if (k < border || (k == border && tie++ >= ties)) return 0;
    const double w = weight(k);
    return w < min_p ? 0 : static_cast<u64>(w * kOne + 0.5);
  };
  u64 own = 0, tie = ties_before;
  for (int i = lo; i < hi; ++i) own += mass(i, tie);
  const u64 total = block_sum(own, s_sum), before = block_before(own, s_sum);
  const u64 target = __umul64hi(fraction(p.uniform[b]), total);
  if (before <= target && target < before + own) {
    u64 sum = before;
    tie = ties_before;
    for (int i = lo; i < hi; ++i) {
      const u64 m = mass(i, tie);
      sum += m;
      if (sum > target) {
        ids[b] = i;
        probs[b] = static_cast<float>(static_cast<double>(m) / static_cast<double>(total));
        break;
      }
    }
  }
}

}  // namespace

cudaError_t launch_sample_tokens(const void* logits, int fp32, long long ld, int B, int V, const cd_sample& p, int64_t* ids, float* probs,
                                 cudaStream_t stream) {
  long long* to = reinterpret_cast<long long*>(ids);
  if (fp32)
    return launch_kernel(sample_tokens_kernel<float>, dim3(B), dim3(kThreads), 0, stream, static_cast<const float*>(logits), ld, V, p, to,
                         probs);
  return launch_kernel(sample_tokens_kernel<bf16>, dim3(B), dim3(kThreads), 0, stream, static_cast<const bf16*>(logits), ld, V, p, to, probs);
}

}  // namespace cdeep
