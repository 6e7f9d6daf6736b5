// Cuts a paged cache back to `keep` rows per (layer, sequence, KV head): the newest `recent` rows stay, then those of the largest
// accumulated attention weight, ties by the lowest row. Of the rows that stay, those behind row `keep` move into the places of those
// given up in front of it, in order, so nothing is read that has been written and only the moved rows are touched: 16 D bytes
// each (read and written, keys and values), beside 8 bytes of weight and position of every row.
//
// A block a (layer, sequence, head). Keys (the weights' order as unsigned numbers) are read once into shared memory. The keep-th
// largest is found by histograms of 11, 11 and 10 bits; of the first, sign, exponent and two bits, lognormal weights use some
// forty bins, which keeps warps from queueing at a few. Then warps walk their stretches of rows by ballots: ties, fates (a
// bit a row), and the ranks of holes and movers, whose lists take the keys' place.
//
// Few pairs of long caches take several blocks each, a cluster: each has a share of the rows, the histograms and the counts ahead of a
// share are added up over their shared memory, and the lists lie in the workspace, from which each moves a part. (Every block
// finding all fates by itself: 28 us for 32 pairs of 32 768 rows, four blocks each.)
#include <cuda_bf16.h>
#include <cuda_runtime.h>
#include "checks.cuh"
#include "kernels.h"
#include "ptx.cuh"

namespace cdeep {

namespace {

constexpr int kBins = 2048;
constexpr int kMostBlocks = 8;            // of a pair
constexpr int kHeldRows = 48 * 1024;      // of a block; beyond, keys are read again and lists lie in the workspace

struct Args {
  cd_paged c;
  long long stride_l;
  cd_evict e;
  int B, hkv, D;
  int shift;              // log2 of the page, or -1
  int blocks;             // of a pair
  int* lists;             // [pairs][rows + words]: of several blocks, or where keys are not held
  int rows, half, words;  // of a sequence at most; of a list at most; of the fates' bits
  int share;              // rows of a block at most
  int* status;
};

// Order of rows as unsigned numbers: by weight, NaN above all weights, protected rows above everything.
__device__ __forceinline__ uint32_t key_of(float w, bool newest) {
  const uint32_t u = __float_as_uint(w + 0.f);
  const uint32_t k = w != w ? 0xfffffffeu : u & 0x80000000u ? ~u : u | 0x80000000u;
  return newest ? 0xffffffffu : k;
}

// Sum over the warps ahead of this one, and over all, of a number that every lane of a warp has.
template <int kWarps>
__device__ __forceinline__ int warps_before(int v, int* s, int& all) {
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  __syncthreads();
  if (lane == 0) s[warp] = v;
  __syncthreads();
  const int x = lane < kWarps ? s[lane] : 0;
  all = __reduce_add_sync(0xffffffffu, x);
  return __reduce_add_sync(0xffffffffu, lane < warp ? x : 0);
}

__device__ __forceinline__ uint4 peer_load4(const void* p, int rank) {
  uint4 v;
  asm volatile("ld.shared::cluster.v4.u32 {%0, %1, %2, %3}, [%4];" : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w) : "r"(map_to_cta(smem_u32(p), rank)) : "memory");
  return v;
}
__device__ __forceinline__ unsigned long long peer_load2(const void* p, int rank) {
  unsigned long long v;
  asm volatile("ld.shared::cluster.u64 %0, [%1];" : "=l"(v) : "r"(map_to_cta(smem_u32(p), rank)) : "memory");
  return v;
}
__device__ __forceinline__ int peer_load(const int* p, int rank) {
  int v;
  asm volatile("ld.shared::cluster.u32 %0, [%1];" : "=r"(v) : "r"(map_to_cta(smem_u32(p), rank)) : "memory");
  return v;
}

template <int kThreads, bool kHeld>
__global__ void __launch_bounds__(kThreads, kThreads == 128 ? 7 : kThreads == 256 ? 4 : 1) evict_rows_kernel(const Args a) {
  constexpr int kWarps = kThreads / 32, kOwn = kBins / kThreads;
  static_assert(kOwn < 4 || kOwn % 8 == 0, "a thread's bins are read four at a time, also of the 1 024 of the last histogram");
  extern __shared__ __align__(16) unsigned s_dyn[];
  __shared__ int s_warps[kWarps], s_counts[3];            // counts: of equal rows, holes and movers of this block
  __shared__ unsigned s_digit, s_left, s_equal;
  griddep_wait();
  griddep_launch_dependents();
  const int blocks = a.blocks, pair = blockIdx.x / blocks, rank = blockIdx.x - pair * blocks;
  const bool several = blocks > 1;
  const int h = pair % a.hkv, b = pair / a.hkv % a.B, layer = pair / (a.hkv * a.B);
  const int keep = a.e.keep, n = a.c.lengths[b];
  const long long base = static_cast<long long>(pair) * a.rows;
  const float* w = a.c.weights + base;
  const int* pos = a.e.row_positions + base;
  float* w_out = a.e.weights_out + base;
  int* pos_out = a.e.row_positions_out + base;
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const bool in_place = w_out == w;
  if (n > a.rows) {                       // the same for all blocks of the pair, as below
    if (threadIdx.x == 0) atomicMax(a.status, kStatusBounds);
    return;
  }
  if (n <= keep) {
    if (!in_place)
      for (int i = rank * kThreads + tid; i < n; i += blocks * kThreads) w_out[i] = w[i], pos_out[i] = pos[i];
    return;
  }
  // this block's rows: whole words of fates
  const int share = ((n + blocks - 1) / blocks + 31) / 32 * 32, row0 = min(n, rank * share), rows = min(n, row0 + share) - row0;
  unsigned* hist = s_dyn;                 // of several blocks one a pass: others read it while the next is filled
  unsigned* keys = s_dyn + kBins * (several ? 3 : 1);
  int* own = a.lists + static_cast<long long>(pair) * (a.rows + a.words);
  int* lists = kHeld && !several ? reinterpret_cast<int*>(keys) : own;     // holes, then movers; they may take the keys' place
  unsigned* fates = kHeld ? keys + a.share : reinterpret_cast<unsigned*>(own + a.rows) + row0 / 32;
  const long long oldest = static_cast<long long>(a.e.positions[b]) - a.e.recent;
  auto key = [&](int i) -> unsigned {     // of the block's row i
    if constexpr (kHeld) return keys[i];
    return key_of(w[row0 + i], pos[row0 + i] >= oldest);
  };
  if constexpr (kHeld) {
    constexpr int kAhead = 8;
    for (int i0 = tid; i0 < rows; i0 += kAhead * kThreads) {
      float wi[kAhead];
      int pi[kAhead];
#pragma unroll
      for (int x = 0; x < kAhead; ++x) {
        const int i = i0 + x * kThreads;
        wi[x] = i < rows ? w[row0 + i] : 0.f;
        pi[x] = i < rows ? pos[row0 + i] : 0;
      }
#pragma unroll
      for (int x = 0; x < kAhead; ++x) {
        const int i = i0 + x * kThreads;
        if (i < rows) keys[i] = key_of(wi[x], pi[x] >= oldest);
      }
    }
  }

  // the keep-th largest key, and how many of those equal to it stay
  unsigned prefix = 0, left = keep;
#pragma unroll
  for (int pass = 0; pass < 3; ++pass) {
    const int shift = pass == 0 ? 21 : pass == 1 ? 10 : 0, bins = pass == 2 ? 1024 : 2048;
    if (several && pass > 0) hist += kBins;
    for (int i = tid; i < bins / 4; i += kThreads) reinterpret_cast<uint4*>(hist)[i] = make_uint4(0, 0, 0, 0);
    __syncthreads();
    for (int i = tid; i < rows; i += kThreads) {
      const unsigned k = key(i);
      if (pass == 0 || (k ^ prefix) >> (shift + (pass == 1 ? 11 : 10)) == 0) atomicAdd(&hist[k >> shift & (bins - 1)], 1u);
    }
    if (several) {
      cluster_sync_all();
    } else {
      __syncthreads();
    }
    // thread 0 has the largest bins; every thread neighbouring ones, read four (two) at a time
    const int own_bins = bins / kThreads, low = bins - (tid + 1) * own_bins;
    unsigned count[kOwn] = {}, sum = 0;                     // the largest first
#pragma unroll
    for (int r = 0; r < kMostBlocks; ++r) {
      if (r >= blocks) continue;
      if constexpr (kOwn < 4) {
        if (own_bins > 1) {
          const unsigned long long two = several ? peer_load2(hist + low, r) : *reinterpret_cast<const unsigned long long*>(hist + low);
          count[1] += static_cast<unsigned>(two);
          count[0] += static_cast<unsigned>(two >> 32);
        } else {
          count[0] += several ? peer_load(reinterpret_cast<const int*>(hist + low), r) : hist[low];
        }
      } else {
#pragma unroll
        for (int x = 0; x < kOwn; x += 4) {
          if (x >= own_bins) continue;
          const unsigned* at = hist + low + own_bins - 4 - x;
          const uint4 c = several ? peer_load4(at, r) : *reinterpret_cast<const uint4*>(at);
          count[x] += c.w;
          count[x + 1] += c.z;
          count[x + 2] += c.y;
          count[x + 3] += c.x;
        }
      }
    }
#pragma unroll
    for (int x = 0; x < kOwn; ++x) sum += count[x];
    unsigned upto = sum;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const unsigned up = __shfl_up_sync(0xffffffffu, upto, o);
      if (lane >= o) upto += up;
    }
    int all;
    unsigned before = warps_before<kWarps>(static_cast<int>(__shfl_sync(0xffffffffu, upto, 31)), s_warps, all) + upto - sum;
#pragma unroll
    for (int x = 0; x < kOwn; ++x) {
      if (before < left && left <= before + count[x]) {
        s_digit = low + own_bins - 1 - x;
        s_left = left - before;
        s_equal = count[x];
      }
      before += count[x];
    }
    __syncthreads();
    prefix |= s_digit << shift;
    left = s_left;
  }

  // fates, a bit a row: a warp has a stretch of whole words; where only some of the equal rows stay, their order counts
  const int words = (rows + 31) / 32, stretch = (words + kWarps - 1) / kWarps;
  const int from = min(words, warp * stretch), to = min(words, from + stretch);
  const unsigned below = (1u << lane) - 1;
  const bool some = s_equal != left;      // the same in all blocks
  // a count of this block as one of all: what the blocks ahead have
  auto blocks_ahead = [&](int which, int& all) {
    int ahead = 0;
    all = 0;
    for (int r = 0; r < blocks; ++r) {
      const int c = several ? peer_load(&s_counts[which], r) : s_counts[which];
      if (r < rank) ahead += c;
      all += c;
    }
    return ahead;
  };
  int tie = 0, all;
  if (some) {
    int ties = 0;
    for (int x = from; x < to; ++x) {
      const int i = x * 32 + lane;
      ties += __popc(__ballot_sync(0xffffffffu, i < rows && key(i) == prefix));
    }
    tie = warps_before<kWarps>(ties, s_warps, all);
    if (several) {
      if (tid == 0) s_counts[0] = all;
      cluster_sync_all();
      tie += blocks_ahead(0, all);
    }
  }
#pragma unroll 4
  for (int x = from; x < to; ++x) {
    const int i = x * 32 + lane;
    const unsigned k = i < rows ? key(i) : 0;
    bool stays = i < rows && k >= prefix;
    if (some) {
      const unsigned equal = __ballot_sync(0xffffffffu, i < rows && k == prefix);
      if (k == prefix && tie + __popc(equal & below) >= static_cast<int>(left)) stays = false;
      tie += __popc(equal);
    }
    const unsigned bits = __ballot_sync(0xffffffffu, stays);
    if (lane == 0) fates[x] = bits;
  }
  __syncthreads();                        // every key has been read
  if (!in_place) {                        // rows that stay where they are; those that do not are filled below
    constexpr int kAhead = 4;
    const int front = min(rows, keep - row0);
    for (int i0 = tid; i0 < front; i0 += kThreads * kAhead) {
      float wi[kAhead];
      int pi[kAhead];
#pragma unroll
      for (int x = 0; x < kAhead; ++x) {
        const int i = row0 + min(i0 + x * kThreads, front - 1);
        wi[x] = w[i];
        pi[x] = pos[i];
      }
#pragma unroll
      for (int x = 0; x < kAhead; ++x) {
        const int i = i0 + x * kThreads;
        if (i < front && (fates[i >> 5] >> (i & 31) & 1)) w_out[row0 + i] = wi[x], pos_out[row0 + i] = pi[x];
      }
    }
  }
  // holes and movers of a word: rows in front of row `keep` that go, rows behind that stay
  auto of_word = [&](int x, unsigned& hole, unsigned& mover) {
    const int ahead = keep - row0 - x * 32, last = rows - x * 32;
    const unsigned bits = x < words ? fates[x] : 0, front = ahead >= 32 ? ~0u : ahead <= 0 ? 0u : (1u << ahead) - 1;
    const unsigned there = last >= 32 ? ~0u : last <= 0 ? 0u : (1u << last) - 1;
    hole = ~bits & front & there;
    mover = bits & ~front;
  };
  int seen_holes = 0, moves = 0, total_moves = 0;
  if (several) {                          // how many the blocks ahead have
    int counts[2] = {0, 0};
    for (int x = tid; x < words; x += kThreads) {
      unsigned hole, mover;
      of_word(x, hole, mover);
      counts[0] += __popc(hole);
      counts[1] += __popc(mover);
    }
#pragma unroll
    for (int e = 0; e < 2; ++e) {
      warps_before<kWarps>(__reduce_add_sync(0xffffffffu, counts[e]), s_warps, all);
      if (tid == 0) s_counts[1 + e] = all;
    }
    cluster_sync_all();
    seen_holes = blocks_ahead(1, all);
    moves = blocks_ahead(2, total_moves);
  }
  // their lists in order, a thread a word
  for (int x0 = 0; x0 < words; x0 += kThreads) {
    unsigned hole, mover;
    of_word(x0 + tid, hole, mover);
    const int counts = __popc(hole) | __popc(mover) << 16;                 // of a warp at most 1 024 each
    int upto = counts;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const int up = __shfl_up_sync(0xffffffffu, upto, o);
      if (lane >= o) upto += up;
    }
    const int warp_counts = __shfl_sync(0xffffffffu, upto, 31);
    upto -= counts;
    int all_holes, all_movers;
    int to_hole = seen_holes + warps_before<kWarps>(warp_counts & 0xffff, s_warps, all_holes) + (upto & 0xffff);
    int to_mover = moves + warps_before<kWarps>(warp_counts >> 16, s_warps, all_movers) + (upto >> 16);
    const int row = row0 + (x0 + tid) * 32 - 1;
    for (; hole; hole &= hole - 1) lists[to_hole++] = row + __ffs(hole);
    for (; mover; mover &= mover - 1) lists[a.half + to_mover++] = row + __ffs(mover);
    seen_holes += all_holes;
    moves += all_movers;
  }
  if (several) {
    cluster_sync_all();                   // lists are whole, and every block has read its weights
    moves = total_moves;
  } else {
    __syncthreads();
  }

  // the rows, a warp several at a time: its lanes take 16 bytes each, of keys and then of values
  const int* table = a.c.table + b * a.c.table_stride;
  const long long at = layer * a.stride_l + h * a.c.stride_h;
  const int pieces = a.D / 8;
  auto place = [&](int row) -> long long {
    const int page = a.shift >= 0 ? row >> a.shift : row / a.c.page, within = row - page * a.c.page, id = table[page];
    if (id >= 0 && id < a.c.pages) return (at + id * a.c.stride_p + within * a.c.stride_t) / 8;
    atomicMax(a.status, kStatusBounds);
    return -1;
  };
  uint4* const k = static_cast<uint4*>(a.c.k);
  uint4* const v = static_cast<uint4*>(a.c.v);
  constexpr int kAhead = 4;
  for (int m0 = (rank * kWarps + warp) * kAhead; m0 < moves; m0 += blocks * kWarps * kAhead) {
    // lane x: row m0 + x
    const int m = m0 + (lane & (kAhead - 1));
    long long src = -1, dst = -1;
    if (m < moves) {
      const int s = lists[a.half + m], d = lists[m];
      src = place(s);
      dst = place(d);
      if (lane < kAhead) {
        w_out[d] = w[s];
        pos_out[d] = pos[s];
      }
    }
    if (src < 0 || dst < 0) src = dst = -1;
    for (int p0 = 0; p0 < 2 * pieces; p0 += 32) {
      const int p = p0 + lane;
      uint4* const pool = p < pieces ? k : v;
      const int x = p < pieces ? p : p - pieces;
      uint4 held[kAhead];
#pragma unroll
      for (int r = 0; r < kAhead; ++r) {
        const long long s = __shfl_sync(0xffffffffu, src, r);
        if (p < 2 * pieces && s >= 0) held[r] = pool[s + x];
      }
#pragma unroll
      for (int r = 0; r < kAhead; ++r) {
        const long long d = __shfl_sync(0xffffffffu, dst, r);
        if (p < 2 * pieces && d >= 0) pool[d + x] = held[r];
      }
    }
  }
}

template <int kThreads, bool kHeld>
cudaError_t launch_one(const Args& a, int pairs, cudaStream_t stream) {
  constexpr auto kKernel = evict_rows_kernel<kThreads, kHeld>;
  const int bytes = 4 * (kBins * (a.blocks > 1 ? 3 : 1) + (kHeld ? a.share + (a.share + 31) / 32 : 0));
  const cudaError_t e = allow_smem<kKernel>(bytes);
  if (e != cudaSuccess) return e;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(a.blocks * pairs);
  cfg.blockDim = dim3(kThreads);
  cfg.dynamicSmemBytes = bytes;
  cfg.stream = stream;
  cudaLaunchAttribute attr[2];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = pdl_enabled() ? 1 : 0;
  attr[1].id = cudaLaunchAttributeClusterDimension;
  attr[1].val.clusterDim.x = a.blocks;
  attr[1].val.clusterDim.y = attr[1].val.clusterDim.z = 1;
  cfg.attrs = attr;
  cfg.numAttrs = a.blocks > 1 ? 2 : 1;
  return cudaLaunchKernelEx(&cfg, kKernel, a);
}

// Blocks of a pair: more than one where there are SMs without, and 4 096 rows, or 512 that may move, for each, and all clusters run at
// the same time (of the blocks of 1 024 threads that are likely then, an SM has one). 16 pairs of 18 830 rows to 1 176 with eight blocks
// each, of which not all 16 run together, 51 us, with four 29; 34 of them 49 and 37.
int blocks_of(long long pairs, int rows, int keep) {
  const int most = rows - keep < keep ? rows - keep : keep;
  int blocks = 1;
  while (blocks < kMostBlocks && 2 * blocks * pairs <= current_sm_count() && (most >= 512 * blocks || rows >= 4096 * blocks)) blocks *= 2;
  while (blocks > 1 && pairs > clusters_side_by_side<evict_rows_kernel<1024, true>>(blocks, 1024, 32 * 1024)) blocks /= 2;
  return blocks;
}
int share_of(int rows, int blocks) { return ((rows + blocks - 1) / blocks + 31) / 32 * 32; }

}  // namespace

size_t evict_rows_workspace_bytes(int layers, int B, int hkv, int page, int width, int keep) {
  const long long all = static_cast<long long>(width) * page, pairs = static_cast<long long>(layers) * B * hkv;
  if (all <= keep) return 0;
  const int rows = static_cast<int>(all), blocks = blocks_of(pairs, rows, keep);
  return blocks == 1 && share_of(rows, 1) <= kHeldRows ? 0 : sizeof(int) * pairs * (all + (all + 31) / 32);
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
  a.shift = -1;
  for (int s = 0; s < 31; ++s)
    if (c.page == 1 << s) a.shift = s;
  const int pairs = layers * B * hkv;
  a.rows = c.width * c.page;
  a.half = a.rows / 2;                    // there are as many movers as holes
  a.words = (a.rows + 31) / 32;
  a.blocks = a.rows <= e.keep ? 1 : blocks_of(pairs, a.rows, e.keep);
  a.share = share_of(a.rows, a.blocks);
  a.lists = static_cast<int*>(ws);
  a.status = status;
  // One block an SM is large. More of them overlap one's search with another's moves: 256 threads, and 128 where even those are too
  // many; long shares stay with large blocks. us, cold L2, events included, threads x blocks a pair: 4 pairs of 2 048 rows to 1 024
  // 128x1 63, 256x1 38, 1024x1 25, 1024x4 23; 8 of 131 072 to 8 192 1024x1 258, 1024x8 55; 32 of 32 768 to 2 048 1024x1 64, 256x4 66,
  // 1024x4 37. With one block a pair, 128, 256 and 1 024 threads: 128 of 2 304 to 2 048 43, 29, 23; 160 of 3 000 to 2 048 100, 61, 55;
  // 192 of 1 100 to 1 024 23, 18, 29; 192 of 4 096 to 2 048 154, 90, 72; 256 of 2 304 49, 35, 37; 512 57, 47, 68; 512 of 3 300 144,
  // 106, 125; 512 of 8 192 to 4 096 366, 246, 254; 1 024 of 2 304 80, 82, 115; 768 of 1 100 33, 37, 70; 640 of 3 300 156, 160, 154; 640
  // of 4 096 197, 201, 182; 3 072 of 4 096 705, 698, 757; 6 144 of 2 304 395, 376, 637 (a table may have room for
  // more rows than there are, which smaller blocks mind less).
  const long long grid = static_cast<long long>(pairs) * a.blocks, sms = current_sm_count();
  if (grid > 4 * sms && a.share <= 2560) return launch_one<128, true>(a, pairs, stream);
  if (a.share <= (grid <= sms ? 511 : grid <= 4 * sms ? 4000 : 8192)) return launch_one<256, true>(a, pairs, stream);
  return a.share <= kHeldRows ? launch_one<1024, true>(a, pairs, stream) : launch_one<1024, false>(a, pairs, stream);
}

}  // namespace cdeep
