// Cuts a paged cache back to `keep` rows per (layer, sequence, KV head): the newest `recent` rows stay, then those of the largest
// accumulated attention weight, ties by the lowest row. Of the rows that stay, those behind row `keep` move into the places of those
// given up in front of it, in order, so nothing is read that has been written and only the moved rows are touched.
//
// One block a (layer, sequence, head). The keep-th largest key is found digit by digit (histograms of eight bits, keys read again
// from L2), then one walk in row order gives every row its fate and the movers and holes their ranks.
#include <cuda_bf16.h>
#include <cuda_runtime.h>
#include "checks.cuh"
#include "kernels.h"
#include "ptx.cuh"

namespace cdeep {

namespace {

constexpr int kThreads = 1024;

struct Args {
  cd_paged c;
  long long stride_l;
  cd_evict e;
  int B, hkv, D;
  int* lists;            // [pairs][2][most]: moved rows, holes
  int most;
  int* status;
};

// Order of rows as unsigned numbers: by weight, NaN above all weights, protected rows above everything.
__device__ __forceinline__ uint32_t key_of(float w, bool newest) {
  const uint32_t u = __float_as_uint(w + 0.f);
  const uint32_t k = w != w ? 0xfffffffeu : u & 0x80000000u ? ~u : u | 0x80000000u;
  return newest ? 0xffffffffu : k;
}

__global__ void __launch_bounds__(kThreads) evict_rows_kernel(Args a) {
  __shared__ unsigned s_hist[256];
  __shared__ int s_scan[3][kThreads / 32];
  __shared__ unsigned s_digit, s_left;
  griddep_wait();
  griddep_launch_dependents();
  const int h = blockIdx.x % a.hkv, b = blockIdx.x / a.hkv % a.B, layer = blockIdx.x / (a.hkv * a.B);
  const int rows = a.c.width * a.c.page, keep = a.e.keep;
  const int n = min(a.c.lengths[b], rows);
  const long long base = static_cast<long long>(blockIdx.x) * rows;
  const float* w = a.c.weights + base;
  const int* pos = a.e.row_positions + base;
  float* w_out = a.e.weights_out + base;
  int* pos_out = a.e.row_positions_out + base;
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const bool in_place = w_out == w;
  if (n <= keep) {
    if (!in_place)
      for (int i = tid; i < n; i += kThreads) w_out[i] = w[i], pos_out[i] = pos[i];
    return;
  }
  const long long oldest = static_cast<long long>(a.e.positions[b]) - a.e.recent;
  auto key = [&](int i) { return key_of(w[i], pos[i] >= oldest); };

  unsigned prefix = 0, left = keep;
  for (int shift = 24; shift >= 0; shift -= 8) {
    if (tid < 256) s_hist[tid] = 0;
    __syncthreads();
    for (int i = tid; i < n; i += kThreads) {
      const unsigned k = key(i);
      if (shift == 24 || (k >> (shift + 8)) == (prefix >> (shift + 8))) atomicAdd(&s_hist[k >> shift & 255], 1u);
    }
    __syncthreads();
    if (tid == 0) {
      int d = 255;
      while (d > 0 && s_hist[d] < left) left -= s_hist[d--];
      s_digit = d;
      s_left = left;
    }
    __syncthreads();
    prefix |= s_digit << shift;
    left = s_left;
  }

  // Rows in order, a tile at a time: counts of equal keys, holes and movers ahead of each.
  int* moved = a.lists + static_cast<long long>(blockIdx.x) * 2 * a.most;
  int* holes = moved + a.most;
  int seen[3] = {0, 0, 0};
  auto ranks = [&](bool flag, int which) {                // flags ahead of this thread's, all tiles
    const unsigned vote = __ballot_sync(0xffffffffu, flag);
    if (lane == 0) s_scan[which][warp] = __popc(vote);
    __syncthreads();
    int before = seen[which], total = 0;
    for (int x = 0; x < kThreads / 32; ++x) {
      const int c = s_scan[which][x];
      if (x < warp) before += c;
      total += c;
    }
    seen[which] += total;
    __syncthreads();
    return before + __popc(vote & ((1u << lane) - 1));
  };
  for (int t = 0; t < n; t += kThreads) {
    const int i = t + tid;
    const unsigned k = i < n ? key(i) : 0;
    const bool tie = i < n && k == prefix;
    const int tie_rank = ranks(tie, 0);
    const bool stays = i < n && (k > prefix || (tie && tie_rank < static_cast<int>(left)));
    const bool hole = i < keep && !stays, mover = i >= keep && stays;
    const int hole_rank = ranks(hole, 1), mover_rank = ranks(mover, 2);
    if (hole) holes[hole_rank] = i;
    if (mover) moved[mover_rank] = i;
    if (!in_place && i < keep && stays) w_out[i] = w[i], pos_out[i] = pos[i];
  }
  __syncthreads();
  const int moves = seen[2];
  const int* table = a.c.table + b * a.c.table_stride;
  for (int x = tid; x < moves; x += kThreads) {
    w_out[holes[x]] = w[moved[x]];
    pos_out[holes[x]] = pos[moved[x]];
  }
  const int pieces = a.D / 8;                             // 16 bytes each
  const long long at = layer * a.stride_l + h * a.c.stride_h;
  uint4* pools[2] = {reinterpret_cast<uint4*>(a.c.k), reinterpret_cast<uint4*>(a.c.v)};
  for (int x = tid; x < 2 * moves * pieces; x += kThreads) {
    const int row = x / (2 * pieces), piece = x % pieces, which = x / pieces % 2;
    const int src = moved[row], dst = holes[row], ps = table[src / a.c.page], pd = table[dst / a.c.page];
    if (ps < 0 || ps >= a.c.pages || pd < 0 || pd >= a.c.pages) {
      atomicMax(a.status, kStatusBounds);
      continue;
    }
    pools[which][(at + pd * a.c.stride_p + dst % a.c.page * a.c.stride_t) / 8 + piece] =
        pools[which][(at + ps * a.c.stride_p + src % a.c.page * a.c.stride_t) / 8 + piece];
  }
}

}  // namespace

int evict_most(int width, int page, int keep) {
  const long long rows = static_cast<long long>(width) * page;
  return rows <= keep ? 0 : static_cast<int>(rows - keep < keep ? rows - keep : keep);
}

size_t evict_rows_workspace_bytes(int layers, int B, int hkv, int page, int width, int keep) {
  return sizeof(int) * 2 * layers * B * hkv * evict_most(width, page, keep);
}

cudaError_t launch_evict_rows(const cd_paged& c, const cd_evict& e, int layers, long long stride_l, int B, int hkv, int D, void* ws,
                              int* status, cudaStream_t stream) {
  Args a;
  a.c = c;
  a.stride_l = stride_l;
  a.e = e;
  a.B = B;
  a.hkv = hkv;
  a.D = D;
  a.lists = static_cast<int*>(ws);
  a.most = evict_most(c.width, c.page, e.keep);
  a.status = status;
  return launch_kernel(evict_rows_kernel, dim3(layers * B * hkv), dim3(kThreads), 0, stream, a);
}

}  // namespace cdeep
