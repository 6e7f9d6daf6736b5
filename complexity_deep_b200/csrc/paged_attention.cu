// Attention of one new token per sequence over a paged cache: the rows of a sequence lie in pages that a table names, and every
// sequence has a length of its own (read on the device).
//
//   s_{g,r} = scale q_g . k_r;  p = exp(s - max) / sum;  out_g = sum_r p_{g,r} v_r;  weights_r += sum_g p_{g,r}
//
// for the G query heads g of a KV head. One block a (sequence, KV head): its warps take the rows in turn, a lane D / 32 columns,
// each with a running maximum and sum, which meet in shared memory. Scores are kept for the accumulator, whose share of a row is
// known only when maximum and sum are.
//
// A step (kStep) brings the raw projections: the block normalises and rotates its heads first, writes key and value into the new
// row's place and takes that row with the others. The query stays in 32 bits.
#include <cfloat>
#include <cuda_bf16.h>
#include <cuda_runtime.h>
#include "checks.cuh"
#include "elem.cuh"
#include "kernels.h"
#include "ptx.cuh"

namespace cdeep {

namespace {

// warps of a block: their sums of kG heads share its 48 KB
__host__ __device__ constexpr int warps_of(int kG) { return kG > 8 ? 4 : 8; }

struct Args {
  cd_paged c;
  const bf16* q;
  long long q_stride;
  cd_paged_step st;
  float scale;
  int G, hq;
  bf16* out;
  float* scores;
  int* status;
};

__device__ __forceinline__ float warp_sum(float v) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
  return v;
}

// RMS norm (w or none) and rotation of a head; lane l holds columns l + 32 i.
template <int D>
__device__ __forceinline__ void norm_rotate(const bf16* x, const bf16* w, const float* cs, const float* sn, float eps, int lane,
                                            float (&y)[D / 32]) {
  constexpr int N = D / 32;
  float v[N], ss = 0.f;
#pragma unroll
  for (int i = 0; i < N; ++i) {
    v[i] = to_f32(x[lane + 32 * i]);
    ss += v[i] * v[i];
  }
  if (w) {
    const float r = rsqrtf(warp_sum(ss) / D + eps);
#pragma unroll
    for (int i = 0; i < N; ++i) v[i] *= r * to_f32(w[lane + 32 * i]);
  }
#pragma unroll
  for (int i = 0; i < N; ++i) {
    const float other = i < N / 2 ? -v[i + N / 2] : v[i - N / 2];
    y[i] = v[i] * cs[lane + 32 * i] + other * sn[lane + 32 * i];
  }
}

template <int D, int kG, bool kStep>
__global__ void __launch_bounds__(warps_of(kG) * 32) paged_attention_kernel(Args a) {
  constexpr int N = D / 32, kWarps = warps_of(kG);
  __shared__ float s_q[kG][D];
  __shared__ float s_m[kWarps][kG], s_l[kWarps][kG], s_acc[kWarps][kG][D];
  griddep_wait();
  griddep_launch_dependents();
  const int h = blockIdx.x, b = blockIdx.y, hkv = gridDim.x, G = a.G;
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int* table = a.c.table + b * a.c.table_stride;
  const int limit = a.c.width * a.c.page;
  int n = a.c.lengths[b];
  const int at = n;                                     // the new row, where there is one
  bool ok = n <= limit;
  if constexpr (kStep) {
    ok = n < limit;
    if (ok && n >= 0) {
      const int pos = a.st.positions[b], page = table[n / a.c.page];
      ok = pos >= 0 && pos < a.st.table_rows && page >= 0 && page < a.c.pages;
    }
    n = n < 0 ? 0 : n + 1;
  }
  if (!ok) {
    if (threadIdx.x == 0) atomicMax(a.status, kStatusBounds);
    n = 0;
  }
  bf16* out = a.out + (static_cast<long long>(b) * a.hq + h * G) * D;
  if (n <= 0) {
    for (int i = threadIdx.x; i < G * D; i += blockDim.x) out[i] = from_f32<bf16>(0.f);
    return;
  }
  const long long pair = static_cast<long long>(b) * hkv + h;
  const bf16* row = a.q + b * a.q_stride;
  bf16* kp = static_cast<bf16*>(a.c.k) + h * a.c.stride_h;
  bf16* vp = static_cast<bf16*>(a.c.v) + h * a.c.stride_h;
  if constexpr (kStep) {
    const int pos = a.st.positions[b];
    const float *cs = a.st.cos_t + static_cast<long long>(pos) * D, *sn = a.st.sin_t + static_cast<long long>(pos) * D;
    for (int g = warp; g <= G; g += kWarps) {
      float y[N];
      const bool key = g == G;
      norm_rotate<D>(row + static_cast<long long>(key ? a.hq + h : h * G + g) * D, static_cast<const bf16*>(key ? a.st.k_w : a.st.q_w),
                     cs, sn, a.st.eps, lane, y);
      if (!key) {
#pragma unroll
        for (int i = 0; i < N; ++i) s_q[g][lane + 32 * i] = y[i];
        continue;
      }
      const long long to = table[at / a.c.page] * a.c.stride_p + at % a.c.page * a.c.stride_t;
#pragma unroll
      for (int i = 0; i < N; ++i) {
        kp[to + lane + 32 * i] = from_f32<bf16>(y[i]);
        vp[to + lane + 32 * i] = row[static_cast<long long>(a.hq + hkv + h) * D + lane + 32 * i];
      }
      if (lane == 0 && a.st.row_positions) a.st.row_positions[pair * limit + at] = pos;
    }
  } else {
    for (int i = threadIdx.x; i < G * D; i += blockDim.x) s_q[i / D][i % D] = to_f32(row[static_cast<long long>(h) * G * D + i]);
  }
  __syncthreads();

  float m[kG], l[kG], acc[kG][N];
#pragma unroll
  for (int g = 0; g < kG; ++g) {
    m[g] = -FLT_MAX;
    l[g] = 0.f;
#pragma unroll
    for (int i = 0; i < N; ++i) acc[g][i] = 0.f;
  }
  float* scores = a.scores ? a.scores + pair * G * limit : nullptr;
  for (int r = warp; r < n; r += kWarps) {
    const int page = table[r / a.c.page];
    const bool have = page >= 0 && page < a.c.pages;
    if (!have && lane == 0) atomicMax(a.status, kStatusBounds);
    float kf[N], vf[N];
    const long long from = page * a.c.stride_p + r % a.c.page * a.c.stride_t;
#pragma unroll
    for (int i = 0; i < N; ++i) {
      kf[i] = have ? to_f32(kp[from + lane + 32 * i]) : 0.f;
      vf[i] = have ? to_f32(vp[from + lane + 32 * i]) : 0.f;
    }
#pragma unroll
    for (int g = 0; g < kG; ++g) {
      if (g < G) {
        float s = 0.f;
#pragma unroll
        for (int i = 0; i < N; ++i) s += s_q[g][lane + 32 * i] * kf[i];
        s = warp_sum(s) * a.scale;
        if (scores && lane == 0) scores[static_cast<long long>(g) * limit + r] = s;
        if (s > m[g]) {
          const float f = expf(m[g] - s);
          l[g] *= f;
#pragma unroll
          for (int i = 0; i < N; ++i) acc[g][i] *= f;
          m[g] = s;
        }
        const float p = expf(s - m[g]);
        l[g] += p;
#pragma unroll
        for (int i = 0; i < N; ++i) acc[g][i] += p * vf[i];
      }
    }
  }
#pragma unroll
  for (int g = 0; g < kG; ++g) {
    if (lane == 0) {
      s_m[warp][g] = m[g];
      s_l[warp][g] = l[g];
    }
#pragma unroll
    for (int i = 0; i < N; ++i) s_acc[warp][g][lane + 32 * i] = acc[g][i];
  }
  __syncthreads();
  auto whole = [&](int g, float& top, float& sum) {
    top = -FLT_MAX;
    sum = 0.f;
#pragma unroll
    for (int w = 0; w < kWarps; ++w) top = fmaxf(top, s_m[w][g]);
#pragma unroll
    for (int w = 0; w < kWarps; ++w) sum += s_l[w][g] * expf(s_m[w][g] - top);
  };
  for (int i = threadIdx.x; i < G * D; i += blockDim.x) {
    const int g = i / D, d = i - g * D;
    float top, sum, v = 0.f;
    whole(g, top, sum);
#pragma unroll
    for (int w = 0; w < kWarps; ++w) v += s_acc[w][g][d] * expf(s_m[w][g] - top);
    out[i] = from_f32<bf16>(v / sum);
  }
  if (scores) {
    float top[kG], inv[kG];
#pragma unroll
    for (int g = 0; g < kG; ++g) {
      whole(g, top[g], inv[g]);
      inv[g] = 1.f / inv[g];
    }
    float* weights = a.c.weights + pair * limit;
    for (int r = threadIdx.x; r < n; r += blockDim.x) {
      float share = kStep && r == at ? 0.f : weights[r];
      for (int g = 0; g < G; ++g) share += expf(scores[static_cast<long long>(g) * limit + r] - top[g]) * inv[g];
      weights[r] = share;
    }
  }
}

template <bool kStep>
cudaError_t launch_any(const Args& a, int B, int hkv, int D, cudaStream_t stream) {
  const dim3 grid(hkv, B);
#define CDEEP_PAGED(DD, GG) \
  if (D == DD && a.G <= GG) return launch_kernel(paged_attention_kernel<DD, GG, kStep>, grid, dim3(warps_of(GG) * 32), 0, stream, a);
  CDEEP_PAGED(64, 2) CDEEP_PAGED(64, 4) CDEEP_PAGED(64, 8) CDEEP_PAGED(64, 16)
  CDEEP_PAGED(128, 2) CDEEP_PAGED(128, 4) CDEEP_PAGED(128, 8) CDEEP_PAGED(128, 16)
#undef CDEEP_PAGED
  return cudaErrorInvalidValue;
}

}  // namespace

size_t paged_attention_workspace_bytes(int B, int hq, int, int, int page, int width, bool weights) {
  return weights ? sizeof(float) * B * hq * width * page : 0;
}

cudaError_t launch_paged_attention(const cd_paged& c, const cd_paged_step* step, const void* q, long long q_stride, float scale, int B,
                                   int hq, int hkv, int D, void* out, void* ws, int* status, cudaStream_t stream) {
  Args a;
  a.c = c;
  a.q = static_cast<const bf16*>(q);
  a.q_stride = q_stride;
  a.st = step ? *step : cd_paged_step{};
  a.scale = scale;
  a.G = hq / hkv;
  a.hq = hq;
  a.out = static_cast<bf16*>(out);
  a.scores = c.weights ? static_cast<float*>(ws) : nullptr;
  a.status = status;
  return step ? launch_any<true>(a, B, hkv, D, stream) : launch_any<false>(a, B, hkv, D, stream);
}

}  // namespace cdeep
