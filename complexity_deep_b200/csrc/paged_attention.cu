// Attention of one new token per sequence over a paged cache: the rows of a sequence lie in pages that a table names, and every
// sequence has a length of its own (read on the device).
//
//   s_{g,r} = scale q_g . k_r;  p = exp(s - max) / sum;  out_g = sum_r p_{g,r} v_r;  weights_r += sum_g p_{g,r}
//
// for the G query heads g of a KV head: every cached row is read once for all of them, so the read (4 D bytes a row and head) is
// the bound, and G only has to stay out of its way. Hence matrix instructions (m16n8k16): the query heads are the 16 rows of one
// operand. Keys and values are bf16; q (of a step) and p have 32 bits and enter as three bf16 numbers, which hold all 24 of their
// significant ones. Up to eight heads leave half of the rows free: the first two numbers share a product, the third takes one of its
// own, in the rows of the second. More heads take three. (Of a q that comes as bf16 the others are zero; the third is left out.) us on the device with two numbers and
// with three: step of 32 x 256 to 2 047 rows, 8 x 2 x 128, weights, 30.3 / 31.8, of 64 x 1 000 to 16 384 224 / 221, of 64 x 250 to 4 000,
// 4 x 16 x 128, 55.6 / 65; without a step the last 52.7 / 55.5, 2 x 32 768 rows of 8 x 2 x 128 49.2 / 49.8.
//
// Work is cut into tiles of 64 rows; all tiles of all (sequence, KV head) pairs stand in one line, of which every block takes an equal
// stretch, whatever the lengths are (a pair's beginning counts as a few tiles: pair_units). A stretch that covers a pair writes its output; a pair that is cut leaves a partial sum per
// block, which a second kernel adds in order (results do not depend on timing). A warp feeds tiles to the ring with TMA (a
// box per page, 128-byte swizzle), four warps take 16 rows of a tile each, with a running maximum and sum of their own.
//
// Short caches take a cluster of blocks a pair instead (kCluster), whose sums meet in shared memory: one launch, no workspace to meet
// in, and no line to find one's place in.
//
// The share of a row in its softmax is known only when the pair's maximum and sum are: where weights are asked for, scores are
// left in the workspace and the second kernel turns them into shares (clusters do so themselves, when their sums have met).
//
// A sixth warp prepares the next pair while the tiles of this one are taken: the query heads as operand fragments, of a step
// (kStep) normalised and rotated from the raw projections, and, where the block has the pair's last tile, the new key and value, which
// it writes into the cache and the warp that has the row puts into its copy of the tile. Doing this in the four warps, between
// pairs, cost 2 to 3 us a pair.
#include <cfloat>
#include <cuda.h>
#include <cuda_bf16.h>
#include <cuda_runtime.h>
#include "checks.cuh"
#include "kernels.h"
#include "mma.cuh"
#include "ptx.cuh"

namespace cdeep {

namespace {

constexpr int kTile = 64;                 // rows of a tile
constexpr int kWarps = 4;                 // that compute; one more feeds them, one prepares pairs
constexpr int kThreads = 32 * (kWarps + 2);
constexpr int kSlots = kWarps / 2;        // in which warps hand over their sums
constexpr float kLog2e = 1.4426950408889634f;
constexpr int kMostCluster = 8;           // blocks of a pair
constexpr int kClusterTiles = 16;         // tiles of a block, up to which pairs have clusters

__host__ __device__ constexpr int stage_bytes(int D) { return 2 * kTile * D * 2; }
// floats of a lane that a warp hands over: its columns of each head it holds
__host__ __device__ constexpr int lane_floats(int D, bool wide) { return D / 8 * (wide ? 4 : 2); }
__host__ __device__ constexpr int merge_bytes(int D, bool wide) { return kSlots * 32 * (lane_floats(D, wide) + 4) * 4; }
// operand fragments of a pair's query heads (the first two numbers), the new row's key and value, the fragments' third numbers
__host__ __device__ constexpr int query_bytes(int D, bool wide) { return D / 16 * 32 * (16 + 8) * (wide ? 2 : 1) + 2 * D * 2; }
// Two blocks an SM (113 KB each): one computes while the other starts a pair or ends one. 16 heads of 128 leave room for one.
__host__ __device__ constexpr int blocks_per_sm(int D, bool wide) { return wide && D == 128 ? 1 : 2; }
__host__ __device__ constexpr int stages_of(int D, bool wide) {
  // an SM's 228 KB, of which each block takes 1 KB for the system, up to 1 KB for the ring's alignment, 512 bytes outside of it
  return (233472 / blocks_per_sm(D, wide) - 1024 * 2 - 512 - merge_bytes(D, wide) - query_bytes(D, wide)) / stage_bytes(D);
}
__host__ __device__ constexpr int smem_bytes(int D, bool wide) {
  return 1024 + stages_of(D, wide) * stage_bytes(D) + merge_bytes(D, wide) + query_bytes(D, wide);
}

// What beginning a pair costs, in tiles: of the line, these come ahead of the pair's own. Without them a stretch of many short pairs holds
// all others up. us a step with 0 / 1 / 2 / 4 (two numbers of q and p; three add 1 to 7 us to all): 64 sequences of 32 to 2 047 rows, 8 x 2 x 128, 56 / 43 / 37 / 37, 16 of them empty 40 / 30 /
// 26 / 27, 32 of 256 to 2 047 with weights 31.9 / 30.8 / 30.8 / 31.5, 64 x 1 000 to 16 384 264 / 267 / 266 / 270; of 16 heads, 0 / 1 / 3 / 4 / 5:
// 55 of 1 197 and eight empty ones, 4 x 16 x 128, 133 / 84 / 62 / 62 / 63, 64 of 250 to 4 000 66 / 61 / 60 / 61 / 62.
__host__ __device__ constexpr int pair_units(bool wide) { return wide ? 3 : 2; }

// For the second kernel: a block's stretch and the pairs at its ends, all that it has to know before it can ask for anything.
struct End {
  int pair;
  int first, last;        // blocks that have tiles of it
  int second;             // whether the first of them had begun with another pair
};
struct __align__(16) Stretch {
  int blocks, begins, ends, pad;          // of the line; this block's tiles
  End end[2];
};

struct Args {
  cd_paged c;
  const bf16* q;
  long long q_stride;
  cd_paged_step st;
  float scale_log2;
  int B, hkv, G;
  int boxes, box_rows;    // pages of a tile, rows of a page that a tile takes
  bf16* out;
  int* status;
  int cluster;            // blocks of a pair, or 0: stretches of the line
  long long pair_tiles;   // that a pair has room for
  // workspace
  Stretch* stretches;     // [blocks of the grid]
  float* part;            // [blocks][2][G D + 2 G, to a multiple of four]: of the first pair of a block and of the last
  int4* tile_rows;        // [tiles] pair, first row, rows of the sequence; this and the next two where weights are asked for
  float2* top_sum;        // [B hkv][G] maximum and 1 / sum of pairs that are not cut
  float* scores;          // [tiles][G][64], times log2 e
};

// Floats of a part: the heads' columns, then their maxima and sums.
__host__ __device__ constexpr int part_floats(int G, int D) { return (G * (D + 2) + 3) / 4 * 4; }

// Equal stretches of a line of `units`: the first ones are one longer where it does not divide.
struct Line {
  unsigned each, longer;
  __device__ __forceinline__ Line(unsigned units, unsigned blocks) : each(units / blocks), longer(units % blocks) {}
  __device__ __forceinline__ int first(unsigned block) const { return block * each + min(block, longer); }
  __device__ __forceinline__ int block_of(unsigned unit) const {
    const unsigned head = longer * (each + 1);
    return unit < head ? unit / (each + 1) : longer + (unit - head) / each;
  }
};

// Rows of a sequence that this call attends to; -1 where table, length or position do not hold.
template <bool kStep>
__device__ __forceinline__ int rows_of(const Args& a, int b) {
  const int n = a.c.lengths[b], limit = a.c.width * a.c.page;
  if (n < 0) return 0;
  if constexpr (!kStep) return n <= limit ? n : -1;
  if (n >= limit) return -1;
  const int pos = a.st.positions[b], page = a.c.table[b * a.c.table_stride + n / a.c.page];
  return pos >= 0 && pos < a.st.table_rows && page >= 0 && page < a.c.pages ? n + 1 : -1;
}
__device__ __forceinline__ int tiles_of(int rows) { return rows > 0 ? (rows + kTile - 1) / kTile : 0; }

// A block's way along its stretch.
struct Walk {
  int b, h, t, rows;
  int left;               // units of the stretch from here on
};
template <bool kWide, bool kStep>
__device__ __forceinline__ void next_pair(const Args& a, Walk& w, int taken) {
  w.left -= taken + pair_units(kWide);
  w.t = 0;
  if (++w.h < a.hkv) return;
  w.h = 0;
  if (w.left <= 0) return;
  do w.rows = rows_of<kStep>(a, ++w.b);
  while (w.rows <= 0 && w.b + 1 < a.B);
}

__device__ __forceinline__ void tma_load_4d(uint32_t dst, const CUtensorMap* m, uint64_t* bar, int x, int row, int head, int page) {
  asm volatile(
      "cp.async.bulk.tensor.4d.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1, {%3, %4, %5, %6}], [%2];"
      :
      : "r"(dst), "l"(reinterpret_cast<uint64_t>(m)), "r"(smem_u32(bar)), "r"(x), "r"(row), "r"(head), "r"(page)
      : "memory");
}

__device__ __forceinline__ void warps_sync() { asm volatile("bar.sync 1, %0;" ::"n"(32 * kWarps) : "memory"); }

// Query heads as operand fragments: of every 16 columns, lane l holds columns 2 (l % 4) + {0, 1, 8, 9} of head l / 4 (and of head
// l / 4 + 8 where there are more than eight). A head's columns j and j + D / 2 are in the same lane.
template <int D, bool kStep>
__device__ __forceinline__ void load_head(const Args& a, const bf16* x, bool there, int pos, int lane, float (&v)[D / 16][4]) {
  constexpr int kAt = kStep ? D / 16 : 1;
  const int col = 2 * (lane & 3);
  uint32_t two[D / 16][2], norm[kAt][2];
  float2 cs[kAt][2], sn[kAt][2];
  // everything is asked for at once
#pragma unroll
  for (int k = 0; k < D / 16; ++k) {
#pragma unroll
    for (int e = 0; e < 2; ++e) {
      const int at = 16 * k + 8 * e + col;
      two[k][e] = there ? *reinterpret_cast<const uint32_t*>(x + at) : 0u;
      if constexpr (kStep) {
        cs[k][e] = *reinterpret_cast<const float2*>(a.st.cos_t + static_cast<long long>(pos) * D + at);
        sn[k][e] = *reinterpret_cast<const float2*>(a.st.sin_t + static_cast<long long>(pos) * D + at);
        norm[k][e] = a.st.q_w ? *reinterpret_cast<const uint32_t*>(static_cast<const bf16*>(a.st.q_w) + at) : 0u;
      }
    }
  }
  float ss = 0.f;
#pragma unroll
  for (int k = 0; k < D / 16; ++k) {
#pragma unroll
    for (int e = 0; e < 2; ++e) {
      v[k][2 * e] = bf_lo(two[k][e]);
      v[k][2 * e + 1] = bf_hi(two[k][e]);
      ss += v[k][2 * e] * v[k][2 * e] + v[k][2 * e + 1] * v[k][2 * e + 1];
    }
  }
  if constexpr (kStep) {
    ss += __shfl_xor_sync(0xffffffffu, ss, 1);
    ss += __shfl_xor_sync(0xffffffffu, ss, 2);
    if (a.st.q_w) {
      const float r = rsqrtf(ss / D + a.st.eps);
#pragma unroll
      for (int k = 0; k < D / 16; ++k) {
#pragma unroll
        for (int e = 0; e < 2; ++e) {
          v[k][2 * e] *= r * bf_lo(norm[k][e]);
          v[k][2 * e + 1] *= r * bf_hi(norm[k][e]);
        }
      }
    }
#pragma unroll
    for (int k = 0; k < D / 32; ++k) {
#pragma unroll
      for (int e = 0; e < 2; ++e) {
        const float2 c1 = cs[k][e], s1 = sn[k][e], c2 = cs[k + D / 32][e], s2 = sn[k + D / 32][e];
        float(&lo)[4] = v[k], (&hi)[4] = v[k + D / 32];
        const float x0 = lo[2 * e], x1 = lo[2 * e + 1], y0 = hi[2 * e], y1 = hi[2 * e + 1];
        lo[2 * e] = x0 * c1.x - y0 * s1.x;
        lo[2 * e + 1] = x1 * c1.y - y1 * s1.y;
        hi[2 * e] = y0 * c2.x + x0 * s2.x;
        hi[2 * e + 1] = y1 * c2.y + x1 * s2.y;
      }
    }
  }
}

// The new row's key, normalised and rotated, and value: lane l holds columns 32 i + l. What it takes is asked for first.
template <int D>
struct NewRow {
  static constexpr int N = D / 32;
  bf16 x[N], w[N], value[N];
  float cs[N], sn[N];
  __device__ __forceinline__ void load(const Args& a, const bf16* key, const bf16* val, int pos, int lane) {
#pragma unroll
    for (int i = 0; i < N; ++i) {
      x[i] = key[lane + 32 * i];
      value[i] = val[lane + 32 * i];
      w[i] = a.st.k_w ? static_cast<const bf16*>(a.st.k_w)[lane + 32 * i] : bf16();
      cs[i] = a.st.cos_t[static_cast<long long>(pos) * D + lane + 32 * i];
      sn[i] = a.st.sin_t[static_cast<long long>(pos) * D + lane + 32 * i];
    }
  }
  __device__ __forceinline__ void key(const Args& a, bf16 (&y)[N]) const {
    float v[N], ss = 0.f;
#pragma unroll
    for (int i = 0; i < N; ++i) {
      v[i] = to_f32(x[i]);
      ss += v[i] * v[i];
    }
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) ss += __shfl_xor_sync(0xffffffffu, ss, o);
    if (a.st.k_w) {
      const float r = rsqrtf(ss / D + a.st.eps);
#pragma unroll
      for (int i = 0; i < N; ++i) v[i] *= r * to_f32(w[i]);
    }
#pragma unroll
    for (int i = 0; i < N; ++i) {
      const float other = i < N / 2 ? -v[i + N / 2] : v[i - N / 2];
      y[i] = from_f32<bf16>(v[i] * cs[i] + other * sn[i]);
    }
  }
};

// Byte of column x of row r within a tile: halves of 64 columns, rows of 128 bytes, 16-byte pieces exchanged by the row (as TMA does).
__device__ __forceinline__ uint32_t place(int r, int x) { return (x >> 6) * (kTile * 128) + r * 128 + ((((x >> 3) & 7) ^ (r & 7)) << 4) + (x & 7) * 2; }

// Shares of the rows of tiles that this warp has scored, from the lanes that hold the scores: four rows of one or two heads each.
template <int kHeads, bool kStep>
__device__ __forceinline__ void add_weights(const Args& a, long long unit, int pair, int t0, int tiles, int rows, int warp, int lane,
                                            const float2* final) {
  const int g0 = lane >> 2, col = 16 * warp + 2 * (lane & 3);
  float2 f[kHeads];
#pragma unroll
  for (int i = 0; i < kHeads; ++i) f[i] = final[g0 + 8 * i];
  float* weights = a.c.weights + static_cast<long long>(pair) * a.c.width * a.c.page;
  constexpr int kAhead = 4;                               // tiles whose loads are under way
  for (int t1 = 0; t1 < tiles; t1 += kAhead) {
    float2 x[kAhead][kHeads][2], old[kAhead];
#pragma unroll
    for (int t = 0; t < kAhead; ++t) {
      const long long at = unit + min(t1 + t, tiles - 1);
      const int r = (t0 + t1 + t) * kTile + col + 8 * g0;             // of lanes that write: g0 = 0, 1
      old[t] = g0 < 2 && t1 + t < tiles && r < rows ? *reinterpret_cast<const float2*>(weights + r) : make_float2(0.f, 0.f);
#pragma unroll
      for (int i = 0; i < kHeads; ++i) {
        const float* s = a.scores + (at * a.G + min(g0 + 8 * i, a.G - 1)) * kTile + col;
        x[t][i][0] = *reinterpret_cast<const float2*>(s);
        x[t][i][1] = *reinterpret_cast<const float2*>(s + 8);
      }
    }
#pragma unroll
    for (int t = 0; t < kAhead; ++t) {
      float2 p[2] = {};
#pragma unroll
      for (int i = 0; i < kHeads; ++i) {
        const float inv = g0 + 8 * i < a.G ? f[i].y : 0.f;
#pragma unroll
        for (int e = 0; e < 2; ++e) {
          p[e].x += inv == 0.f ? 0.f : exp2f(x[t][i][e].x - f[i].x) * inv;
          p[e].y += inv == 0.f ? 0.f : exp2f(x[t][i][e].y - f[i].x) * inv;
        }
      }
#pragma unroll
      for (int e = 0; e < 2; ++e) {
#pragma unroll
        for (int o = 4; o < 32; o <<= 1) {
          p[e].x += __shfl_xor_sync(0xffffffffu, p[e].x, o);
          p[e].y += __shfl_xor_sync(0xffffffffu, p[e].y, o);
        }
      }
      const int r = (t0 + t1 + t) * kTile + col + 8 * g0;
      if (g0 < 2 && t1 + t < tiles && r < rows) {         // a new row's weight starts from 0
        const float2 own = g0 ? p[1] : p[0];
        weights[r] = (kStep && r == rows - 1 ? 0.f : old[t].x) + own.x;
        if (r + 1 < rows) weights[r + 1] = (kStep && r + 1 == rows - 1 ? 0.f : old[t].y) + own.y;
      }
    }
  }
}

template <int D, bool kWide, bool kStep, bool kCluster>
__global__ void __launch_bounds__(kThreads, blocks_per_sm(D, kWide))
paged_attention_kernel(const __grid_constant__ CUtensorMap k_map, const __grid_constant__ CUtensorMap v_map, const Args a) {
  constexpr int kStages = stages_of(D, kWide), kHalf = kTile * D * 2;
  constexpr int kHeads = kWide ? 2 : 1;                   // of a lane
  constexpr int kFloats = lane_floats(D, kWide), kPair = pair_units(kWide);
  // A product adds to its accumulator without rounding: what 24 bits do not hold is cut off, which over hundreds of tiles adds up to
  // 1e-5 of a sum. Hence, where it costs nothing, sums of 16 rows that are added outside of the products (of 524 288 outputs of 64
  // sequences of 1 000 to 16 384 rows, 8 x 2 x 128, 159 are rounded otherwise than in 64 bits, 924 without, 472 by sums in 32 bits in
  // another order; 267 us and 269). Not so in a step, which has a product more (32 x 256 to 2 047 rows 33.4 us and 31.5), for more than eight
  // heads (64 x 250 to 4 000, 4 x 16 x 128, 58 and 55), and in clusters, where a block has 16 tiles at most. There a tile is cut once or, of
  // more than eight heads, three times: the third numbers of up to eight go beside the second, whose sums are small.
  constexpr bool kRound = !kStep && !kWide && !kCluster;
  extern __shared__ unsigned char s_dyn[];
  __shared__ __align__(8) uint64_t s_full[kStages], s_empty[kStages], s_query, s_query_taken;
  __shared__ int2 s_scan[kThreads / 32];
  __shared__ int s_unit, s_at;
  __shared__ Walk s_start;
  __shared__ float2 s_final[16];                          // maximum and 1 / sum of a pair's heads
  __shared__ float2 s_sums[16];                           // of this block (clusters)
  __shared__ int s_abort;
  unsigned char* ring = s_dyn + ((1024 - (smem_u32(s_dyn) & 1023)) & 1023);
  float* s_merge = reinterpret_cast<float*>(ring + kStages * stage_bytes(D));
  uint4* s_heads = reinterpret_cast<uint4*>(ring + kStages * stage_bytes(D) + merge_bytes(D, kWide));
  bf16* s_new = reinterpret_cast<bf16*>(s_heads + D / 16 * 32 * (kWide ? 2 : 1));
  uint2* s_rest = reinterpret_cast<uint2*>(s_new + 2 * D);
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const int block = blockIdx.x;

  if (tid == 0) {
    for (int s = 0; s < kStages; ++s) {
      mbar_init(&s_full[s], 1);
      mbar_init(&s_empty[s], kWarps);
    }
    mbar_init(&s_query, 1);
    mbar_init(&s_query_taken, kWarps);
    fence_barrier_init();
    s_abort = 0;
    tma_prefetch_desc(&k_map);
    tma_prefetch_desc(&v_map);
  }
  griddep_wait();
  griddep_launch_dependents();

  long long unit = 0;                                     // tiles ahead of this one, of scores
  int units = 0, blocks = 0, place_in_line = 0;           // of the line; that have a stretch; of the current tile
  Walk w;
  if constexpr (kCluster) {
    const int pair = block / a.cluster, rank = block - pair * a.cluster, b = pair / a.hkv;
    const int rows = rows_of<kStep>(a, b), tiles = tiles_of(rows);
    if (rows <= 0) {                                      // all blocks of the pair
      if (rows < 0 && tid == 0) atomicMax(a.status, kStatusBounds);
      if (rank == 0 && tid < a.G * D / 8)
        for (int i = tid; i < a.G * D / 8; i += kThreads)
          reinterpret_cast<uint4*>(a.out + static_cast<long long>(pair) * a.G * D)[i] = make_uint4(0, 0, 0, 0);
      return;
    }
    const int t0 = rank * tiles / a.cluster;
    w = {b, pair - b * a.hkv, t0, rows, (rank + 1) * tiles / a.cluster - t0};
    unit = pair * a.pair_tiles + t0;
    __syncthreads();
  } else {
    // Tiles ahead of each sequence, and sequences that have any: every thread a run of sequences.
    const int run = (a.B + kThreads - 1) / kThreads, from = min(a.B, tid * run), to = min(a.B, from + run);
    int2 mine = {0, 0};
    for (int b = from; b < to; ++b) {
      const int rows = rows_of<kStep>(a, b);
      mine.x += tiles_of(rows);
      mine.y += rows > 0;
      if (rows < 0 && block == 0) atomicMax(a.status, kStatusBounds);
    }
    int2 before = mine, all = {0, 0};
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const int x = __shfl_up_sync(0xffffffffu, before.x, o), y = __shfl_up_sync(0xffffffffu, before.y, o);
      if (lane >= o) before.x += x, before.y += y;
    }
    if (lane == 31) s_scan[warp] = before;
    before.x -= mine.x;
    before.y -= mine.y;
    __syncthreads();
#pragma unroll
    for (int x = 0; x < kThreads / 32; ++x) {
      const int2 sum = s_scan[x];
      if (x < warp) before.x += sum.x, before.y += sum.y;
      all.x += sum.x, all.y += sum.y;
    }
    units = (all.x + kPair * all.y) * a.hkv;
    blocks = min(static_cast<int>(gridDim.x), all.x * a.hkv);
    if (block < blocks) {
      const Line line(units, blocks);
      const int u0 = line.first(block), u1 = line.first(block + 1), begin = (before.x + kPair * before.y) * a.hkv;
      if (u0 >= begin && u0 < begin + (mine.x + kPair * mine.y) * a.hkv) {
        int at = begin, tiles_ahead = before.x * a.hkv, b = from, rows = 0, tiles = 0;
        for (;; ++b) {
          rows = rows_of<kStep>(a, b);
          tiles = tiles_of(rows);
          const int here = tiles > 0 ? (tiles + kPair) * a.hkv : 0;
          if (u0 < at + here) break;
          at += here;
          tiles_ahead += tiles * a.hkv;
        }
        const int h = (u0 - at) / (tiles + kPair), t = max(0, u0 - at - h * (tiles + kPair) - kPair);
        at += h * (tiles + kPair) + kPair + t;
        s_start = {b, h, t, rows, u1 - at};
        s_unit = tiles_ahead + h * tiles + t;
        s_at = at;
      }
    }
    // sequences without rows: zeros
    for (int b = block; b < a.B; b += gridDim.x) {
      if (rows_of<kStep>(a, b) > 0) continue;
      for (int i = tid; i < a.hkv * a.G * D / 8; i += kThreads)
        reinterpret_cast<uint4*>(a.out + static_cast<long long>(b) * a.hkv * a.G * D)[i] = make_uint4(0, 0, 0, 0);
    }
    __syncthreads();
    if (tid == 0) a.stretches[block].blocks = blocks;
    if (block >= blocks) return;
    w = s_start;
    unit = s_unit;
    place_in_line = s_at;
    if (w.left <= 0) {                                    // a part of a pair's beginning only
      if (tid == 0) {
        const End none = {-1, block, block, 0};
        a.stretches[block].begins = a.stretches[block].ends = 0;
        a.stretches[block].end[0] = a.stretches[block].end[1] = none;
      }
      return;
    }
    if (tid == 0) a.stretches[block].begins = static_cast<int>(unit);
  }

  int stage = 0, phase = 0;
  auto advance = [&] {
    if (++stage == kStages) {
      stage = 0;
      phase ^= 1;
    }
  };
  if (warp == kWarps) {
    // ------------------------------------------------------------------ feeds the ring
    // A lane a box: the tile's page, the key or the value, the half of its columns.
    constexpr int kParts = D / 64 * 2;
    const int box = lane / kParts, part = lane % kParts;
    const bool value = part >= D / 64;
    const int x = part % (D / 64) * 64;
    while (w.left > 0) {
      const int tiles = tiles_of(w.rows), take = min(tiles - w.t, w.left);
      const int* table = a.c.table + w.b * a.c.table_stride;
      for (int t = w.t; t < w.t + take; ++t) {
        const int row = t * kTile + box * a.box_rows;
        const bool mine_box = box < a.boxes && row < w.rows;
        int page = 0;
        if (mine_box) {
          page = table[row / a.c.page];
          if (page < 0 || page >= a.c.pages) {           // the map has no such page: zeros arrive
            page = a.c.pages;
            atomicMax(a.status, kStatusBounds);
          }
        }
        if (!mbar_wait(&s_empty[stage], phase ^ 1, &s_abort)) atomicMax(a.status, kStatusWaitTimeout);
        const int count = min(a.boxes, (w.rows - t * kTile + a.box_rows - 1) / a.box_rows);
        if (lane == 0) mbar_arrive_expect_tx(&s_full[stage], count * kParts * a.box_rows * 128);
        __syncwarp();
        if (mine_box)
          tma_load_4d(smem_u32(ring + stage * stage_bytes(D)) + (value ? kHalf : 0) + (x / 64) * (kTile * 128) + box * a.box_rows * 128,
                      value ? &v_map : &k_map, &s_full[stage], x, row % a.c.page, w.h, page);
        advance();
      }
      next_pair<kWide, kStep>(a, w, take);
    }
    if (!kCluster) return;
  }
  if (warp == kWarps + 1) {
    // ------------------------------------------------------------------ prepares pairs
    for (int turn = 0; w.left > 0; turn ^= 1) {
      const int tiles = tiles_of(w.rows), take = min(tiles - w.t, w.left), g0 = lane >> 2;
      const bool last_tile = w.t + take == tiles;
      const bf16* q = a.q + w.b * a.q_stride;
      const int pos = kStep ? a.st.positions[w.b] : 0;
      NewRow<D> row;
      if (kStep && last_tile)
        row.load(a, q + static_cast<long long>(a.hkv * a.G + w.h) * D, q + static_cast<long long>(a.hkv * (a.G + 1) + w.h) * D, pos, lane);
      float v[kHeads][D / 16][4];
#pragma unroll
      for (int i = 0; i < kHeads; ++i)
        load_head<D, kStep>(a, q + static_cast<long long>(w.h * a.G + g0 + 8 * i) * D, g0 + 8 * i < a.G, pos, lane, v[i]);
      bf16 key[D / 32];
      if (kStep && last_tile) {
        row.key(a, key);
        const int at = w.rows - 1;
        const long long to = a.c.table[w.b * a.c.table_stride + at / a.c.page] * a.c.stride_p + w.h * a.c.stride_h + at % a.c.page * a.c.stride_t;
        // the tile's copy of this row may be of before or after: it is replaced
#pragma unroll
        for (int i = 0; i < D / 32; ++i) {
          static_cast<bf16*>(a.c.k)[to + lane + 32 * i] = key[i];
          static_cast<bf16*>(a.c.v)[to + lane + 32 * i] = row.value[i];
        }
        if (lane == 0 && a.st.row_positions)
          a.st.row_positions[(static_cast<long long>(w.b) * a.hkv + w.h) * a.c.width * a.c.page + at] = pos;
      }
      if (!mbar_wait(&s_query_taken, turn ^ 1, &s_abort)) atomicMax(a.status, kStatusWaitTimeout);
#pragma unroll
      for (int k = 0; k < D / 16; ++k) {
        uint32_t hi[kHeads][2], lo[kHeads][2], rest[kHeads][2];
#pragma unroll
        for (int i = 0; i < kHeads; ++i) {
          split_all(v[i][k][0], v[i][k][1], hi[i][0], lo[i][0], rest[i][0]);
          split_all(v[i][k][2], v[i][k][3], hi[i][1], lo[i][1], rest[i][1]);
        }
        if constexpr (kWide) {
          s_heads[2 * k * 32 + lane] = make_uint4(hi[0][0], hi[1][0], hi[0][1], hi[1][1]);
          s_heads[(2 * k + 1) * 32 + lane] = make_uint4(lo[0][0], lo[1][0], lo[0][1], lo[1][1]);
        } else {
          s_heads[k * 32 + lane] = make_uint4(hi[0][0], lo[0][0], hi[0][1], lo[0][1]);
        }
        if constexpr (kStep) {
#pragma unroll
          for (int i = 0; i < kHeads; ++i) s_rest[(kHeads * k + i) * 32 + lane] = make_uint2(rest[i][0], rest[i][1]);
        }
      }
      if (kStep && last_tile) {
#pragma unroll
        for (int i = 0; i < D / 32; ++i) {
          s_new[lane + 32 * i] = key[i];
          s_new[D + lane + 32 * i] = row.value[i];
        }
      }
      __syncwarp();
      if (lane == 0) mbar_arrive(&s_query);
      next_pair<kWide, kStep>(a, w, take);
    }
    if (!kCluster) return;
  }

  // ---------------------------------------------------------------------- computes
  const int g0 = lane >> 2, col = 2 * (lane & 3);
  const long long unit0 = unit;
  bool handed = false;                                    // the buffers of the warps' sums are in use
  bool first_pair = true;
  int query_phase = 0;
  while (warp < kWarps && (kCluster || w.left > 0)) {
    const int tiles = tiles_of(w.rows), take = min(tiles - w.t, w.left);
    const int pair = w.b * a.hkv + w.h;
    const bool last_tile = w.t + take == tiles && take > 0;
    uint32_t qh[D / 16][4], ql[kWide ? D / 16 : 1][4];
    const int new_row = w.rows - 1;
    const bool owner = kStep && last_tile && (new_row % kTile) / 16 == warp;   // of the new row: the warp whose rows include it
    bf16 nk[D / 32], nv[D / 32];
    if (take > 0) {
      if (!mbar_wait(&s_query, query_phase, &s_abort)) atomicMax(a.status, kStatusWaitTimeout);
      query_phase ^= 1;
#pragma unroll
      for (int k = 0; k < D / 16; ++k) {
        const uint4 hi = s_heads[k * (kWide ? 2 : 1) * 32 + lane];
        qh[k][0] = hi.x, qh[k][1] = hi.y, qh[k][2] = hi.z, qh[k][3] = hi.w;
        if constexpr (kWide) {
          const uint4 lo = s_heads[(2 * k + 1) * 32 + lane];
          ql[k][0] = lo.x, ql[k][1] = lo.y, ql[k][2] = lo.z, ql[k][3] = lo.w;
        }
      }
      if (owner) {
#pragma unroll
        for (int i = 0; i < D / 32; ++i) {
          nk[i] = s_new[lane + 32 * i];
          nv[i] = s_new[D + lane + 32 * i];
        }
      }
      __syncwarp();
      if (!kStep && lane == 0) mbar_arrive(&s_query_taken);  // the third numbers of a step are read with every tile
    }
    if (!kCluster && tid == 0) {
      const bool last_pair = w.left - take <= kPair;
      if (first_pair || last_pair) {
        const Line line(units, blocks);
        const int at = place_in_line - w.t, first = line.block_of(at);
        const End end = {pair, first, line.block_of(at + tiles - 1), line.first(first) < at - kPair ? 1 : 0};
        if (first_pair) a.stretches[block].end[0] = end;
        if (last_pair) a.stretches[block].end[1] = end, a.stretches[block].ends = static_cast<int>(unit) + take;
      }
      place_in_line += take + kPair;
    }

    float m[kHeads], l[kHeads], o[D / 8][kRound ? 2 : 4];
#pragma unroll
    for (int i = 0; i < kHeads; ++i) {
      m[i] = -FLT_MAX;
      l[i] = 0.f;
    }
#pragma unroll
    for (int j = 0; j < D / 8; ++j) {
#pragma unroll
      for (int e = 0; e < (kRound ? 2 : 4); ++e) o[j][e] = 0.f;
    }

    for (int t = w.t; t < w.t + take; ++t, ++unit) {
      if (!mbar_wait(&s_full[stage], phase, &s_abort)) atomicMax(a.status, kStatusWaitTimeout);
      const uint32_t ks = smem_u32(ring + stage * stage_bytes(D)), vs = ks + kHalf;
      const int r0 = 16 * warp, valid = w.rows - t * kTile - r0;   // of this warp's 16 rows
      if (!kCluster && a.scores && tid == 0) a.tile_rows[unit] = make_int4(pair, t * kTile, w.rows, 0);
      if (valid > 0) {
        if (kStep && owner && t == tiles - 1) {
#pragma unroll
          for (int i = 0; i < D / 32; ++i) {
            unsigned char* tile = ring + stage * stage_bytes(D);
            const uint32_t at = place(new_row % kTile, lane + 32 * i);
            *reinterpret_cast<bf16*>(tile + at) = nk[i];
            *reinterpret_cast<bf16*>(tile + kHalf + at) = nv[i];
          }
          __syncwarp();
          fence_proxy_async();                            // the next copy into this stage comes behind these writes
        }
        float s[2][4] = {};
        const int key = (lane >> 4) * 8 + (lane & 7), piece = (lane >> 3) & 1;
#pragma unroll
        for (int k = 0; k < D / 16; ++k) {
          uint32_t kb[4];
          ldsm4(kb, ks + place(r0 + key, 16 * k + 8 * piece));
          mma16816(s[0], qh[k], kb[0], kb[1]);
          mma16816(s[1], qh[k], kb[2], kb[3]);
          if constexpr (kWide) {
            mma16816(s[0], ql[k], kb[0], kb[1]);
            mma16816(s[1], ql[k], kb[2], kb[3]);
          }
          if constexpr (kStep) {
            const uint2 r = s_rest[kHeads * k * 32 + lane], r2 = kWide ? s_rest[(kHeads * k + 1) * 32 + lane] : make_uint2(0, 0);
            const uint32_t rest[4] = {kWide ? r.x : 0, kWide ? r2.x : r.x, kWide ? r.y : 0, kWide ? r2.y : r.y};
            mma16816(s[0], rest, kb[0], kb[1]);
            mma16816(s[1], rest, kb[2], kb[3]);
          }
        }
        // p of head i of this lane at keys col + {0, 1, 8, 9}
        uint32_t ph[4], pl[4], pr[4] = {};
#pragma unroll
        for (int i = 0; i < kHeads; ++i) {
          float x[4];
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            const float sum = kWide ? s[e >> 1][2 * i + (e & 1)] : s[e >> 1][e & 1] + s[e >> 1][2 + (e & 1)];
            x[e] = col + (e & 1) + (e >> 1) * 8 < valid ? sum * a.scale_log2 : -INFINITY;
          }
          if (a.scores && g0 + 8 * i < a.G) {
            float* to_scores = a.scores + (unit * a.G + g0 + 8 * i) * kTile + r0 + col;
            *reinterpret_cast<float2*>(to_scores) = make_float2(x[0], x[1]);
            *reinterpret_cast<float2*>(to_scores + 8) = make_float2(x[2], x[3]);
          }
          float top = fmaxf(fmaxf(x[0], x[1]), fmaxf(x[2], x[3]));
          top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 1));
          top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 2));
          if (top > m[i]) {                               // rare after the first tiles
            const float f = exp2f(m[i] - top);
            m[i] = top;
            l[i] *= f;
#pragma unroll
            for (int j = 0; j < D / 8; ++j) {
              o[j][2 * i] *= f;
              o[j][2 * i + 1] *= f;
              if constexpr (!kWide && !kRound) {
                o[j][2] *= f;
                o[j][3] *= f;
              }
            }
          }
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            x[e] = exp2f(x[e] - m[i]);
            l[i] += x[e];
          }
          uint32_t hi[2], lo[2];
          split_all(x[0], x[1], hi[0], lo[0], pr[kWide ? i : 1]);          // beside the second, whose sums are small
          split_all(x[2], x[3], hi[1], lo[1], pr[kWide ? 2 + i : 3]);
          if constexpr (kWide) {
            ph[i] = hi[0];
            ph[2 + i] = hi[1];
            pl[i] = lo[0];
            pl[2 + i] = lo[1];
          } else {
            ph[0] = hi[0];
            ph[1] = lo[0];
            ph[2] = hi[1];
            ph[3] = lo[1];
          }
        }
        // values behind the end may be anything: 0 times NaN is not 0
        uint32_t keep0 = 0xffffffffu, keep1 = 0xffffffffu;
        if (valid < 16) {
          keep0 = (col < valid ? 0x0000ffffu : 0u) | (col + 1 < valid ? 0xffff0000u : 0u);
          keep1 = (col + 8 < valid ? 0x0000ffffu : 0u) | (col + 9 < valid ? 0xffff0000u : 0u);
        }
        const int vkey = ((lane >> 3) & 1) * 8 + (lane & 7), vpiece = lane >> 4;
#pragma unroll
        for (int j = 0; j < D / 16; ++j) {
          uint32_t vb[4];
          ldsm4_t(vb, vs + place(r0 + vkey, 16 * j + 8 * vpiece));
          if (valid < 16) {
            vb[0] &= keep0;
            vb[1] &= keep1;
            vb[2] &= keep0;
            vb[3] &= keep1;
          }
          auto add = [&](float (&to)[4], uint32_t b0, uint32_t b1) {
            mma16816(to, pr, b0, b1);
            if constexpr (kWide) mma16816(to, pl, b0, b1);
            mma16816(to, ph, b0, b1);
          };
#pragma unroll
          for (int e = 0; e < 2; ++e) {
            if constexpr (kRound) {
              float sum[4] = {};
              add(sum, vb[2 * e], vb[2 * e + 1]);
              o[2 * j + e][0] += sum[0] + sum[2];
              o[2 * j + e][1] += sum[1] + sum[3];
            } else {
              add(o[2 * j + e], vb[2 * e], vb[2 * e + 1]);
            }
          }
        }
      }
      __syncwarp();
      if (lane == 0) mbar_arrive(&s_empty[stage]);
      advance();
    }
    if (kStep && take > 0 && lane == 0) mbar_arrive(&s_query_taken);

    // The four warps' sums meet in the first, lane by lane (all hold the same heads and columns).
    float f[kFloats];
#pragma unroll
    for (int j = 0; j < D / 8; ++j) {
      if constexpr (kWide || kRound) {
#pragma unroll
        for (int e = 0; e < 2 * kHeads; ++e) f[2 * kHeads * j + e] = o[j][e];
      } else {
        f[2 * j] = o[j][0] + o[j][2];
        f[2 * j + 1] = o[j][1] + o[j][3];
      }
    }
#pragma unroll
    for (int i = 0; i < kHeads; ++i) {
      l[i] += __shfl_xor_sync(0xffffffffu, l[i], 1);
      l[i] += __shfl_xor_sync(0xffffffffu, l[i], 2);
    }
    if (handed) warps_sync();                             // the last pair's have been read
    handed = true;
    auto hand_over = [&](int slot) {
      float4* to = reinterpret_cast<float4*>(s_merge + slot * 32 * (kFloats + 4));
#pragma unroll
      for (int x = 0; x < kFloats / 4; ++x) to[x * 32 + lane] = make_float4(f[4 * x], f[4 * x + 1], f[4 * x + 2], f[4 * x + 3]);
      to[kFloats / 4 * 32 + lane] = make_float4(m[0], l[0], m[kHeads - 1], l[kHeads - 1]);
    };
    auto take_over = [&](int slot) {
      const float4* s = reinterpret_cast<const float4*>(s_merge + slot * 32 * (kFloats + 4));
      const float4 ml = s[kFloats / 4 * 32 + lane];
      float own[kHeads], its[kHeads];
#pragma unroll
      for (int i = 0; i < kHeads; ++i) {
        const float om = i ? ml.z : ml.x, ol = i ? ml.w : ml.y, top = fmaxf(m[i], om);
        own[i] = exp2f(m[i] - top);
        its[i] = exp2f(om - top);
        l[i] = l[i] * own[i] + ol * its[i];
        m[i] = top;
      }
#pragma unroll
      for (int x = 0; x < kFloats / 4; ++x) {
        const float4 v = s[x * 32 + lane];
        // pairs of columns: of one head, or of the lane's two in turn
        f[4 * x] = f[4 * x] * own[0] + v.x * its[0];
        f[4 * x + 1] = f[4 * x + 1] * own[0] + v.y * its[0];
        f[4 * x + 2] = f[4 * x + 2] * own[kHeads - 1] + v.z * its[kHeads - 1];
        f[4 * x + 3] = f[4 * x + 3] * own[kHeads - 1] + v.w * its[kHeads - 1];
      }
    };
    if (warp >= kSlots) hand_over(warp - kSlots);
    warps_sync();
    if (warp < kSlots) take_over(warp);
    if (warp == 1) hand_over(1);
    warps_sync();
    if (warp == 0) {
      take_over(1);
      const bool whole = w.t == 0 && last_tile;
      if constexpr (kCluster) {
        // for the other blocks: the columns where the third warp's have been, and the heads' maxima and sums
        float4* to_others = reinterpret_cast<float4*>(s_merge);
#pragma unroll
        for (int x = 0; x < kFloats / 4; ++x) to_others[x * 32 + lane] = make_float4(f[4 * x], f[4 * x + 1], f[4 * x + 2], f[4 * x + 3]);
#pragma unroll
        for (int i = 0; i < kHeads; ++i)
          if ((lane & 3) == 0) s_sums[g0 + 8 * i] = make_float2(m[i], l[i]);
      } else {
#pragma unroll
        for (int i = 0; i < kHeads; ++i) {
          const int g = g0 + 8 * i;
          if (g >= a.G) continue;
          if (whole) {
            const float inv = 1.f / l[i];
            bf16* out = a.out + (static_cast<long long>(pair) * a.G + g) * D + col;
#pragma unroll
            for (int j = 0; j < D / 8; ++j)
              *reinterpret_cast<uint32_t*>(out + 8 * j) =
                  bf_pack(f[2 * kHeads * j + 2 * i] * inv, f[2 * kHeads * j + 2 * i + 1] * inv);
            if (a.scores && (lane & 3) == 0) a.top_sum[pair * a.G + g] = make_float2(m[i], inv);
          } else {
            float* part = a.part + (2LL * block + (first_pair ? 0 : 1)) * part_floats(a.G, D);
#pragma unroll
            for (int j = 0; j < D / 8; ++j)
              *reinterpret_cast<float2*>(part + g * D + 8 * j + col) =
                  make_float2(f[2 * kHeads * j + 2 * i], f[2 * kHeads * j + 2 * i + 1]);
            if ((lane & 3) == 0) {
              part[a.G * D + 2 * g] = m[i];
              part[a.G * D + 2 * g + 1] = l[i];
            }
          }
        }
      }
    }
    if constexpr (kCluster) break;
    first_pair = false;
    next_pair<kWide, kStep>(a, w, take);
  }
  if constexpr (kCluster) {
    // Every block adds the heads' maxima and sums, the first one the columns too: a warp a share of them.
    __syncwarp();
    cluster_sync_all();
    const int pair = block / a.cluster, rank = block - pair * a.cluster;
    if (tid < 16) {
      float top = -FLT_MAX, sum = 0.f;
      for (int c = 0; c < a.cluster; ++c) {
        const uint32_t at = map_to_cta(smem_u32(&s_sums[tid]), c);
        float2 ml;
        asm volatile("ld.shared::cluster.v2.f32 {%0, %1}, [%2];" : "=f"(ml.x), "=f"(ml.y) : "r"(at) : "memory");
        const float next = fmaxf(top, ml.x);
        sum = sum * exp2f(top - next) + ml.y * exp2f(ml.x - next);
        top = next;
      }
      s_final[tid] = make_float2(top, 1.f / sum);
    }
    __syncthreads();
    if (rank == 0 && warp < kWarps) {
#pragma unroll
      for (int x0 = 0; x0 < kFloats / 4; x0 += kWarps) {
        const int x = x0 + warp;                          // columns 16 x .. of a head, or 8 x .. of the lane's two
        if (x >= kFloats / 4) continue;
        float4 v = make_float4(0.f, 0.f, 0.f, 0.f);
        const int ga = g0, gb = kWide ? g0 + 8 : g0;
        const float2 fa = s_final[ga], fb = s_final[gb];
        for (int c = 0; c < a.cluster; ++c) {
          const float4 p = ld_shared_cluster_f4(map_to_cta(smem_u32(s_merge) + (x * 32 + lane) * 16, c));
          float ma, mb;
          asm volatile("ld.shared::cluster.f32 %0, [%1];" : "=f"(ma) : "r"(map_to_cta(smem_u32(&s_sums[ga]), c)) : "memory");
          asm volatile("ld.shared::cluster.f32 %0, [%1];" : "=f"(mb) : "r"(map_to_cta(smem_u32(&s_sums[gb]), c)) : "memory");
          const float ea = exp2f(ma - fa.x), eb = exp2f(mb - fb.x);
          v.x += p.x * ea;
          v.y += p.y * ea;
          v.z += p.z * eb;
          v.w += p.w * eb;
        }
        bf16* out = a.out + static_cast<long long>(pair) * a.G * D;
        const int first = kWide ? 8 * x : 16 * x, second = kWide ? 8 * x : 16 * x + 8;
        if (ga < a.G) *reinterpret_cast<uint32_t*>(out + ga * D + first + col) = bf_pack(v.x * fa.y, v.y * fa.y);
        if (gb < a.G) *reinterpret_cast<uint32_t*>(out + gb * D + second + col) = bf_pack(v.z * fb.y, v.w * fb.y);
      }
    }
    if (a.scores && warp < kWarps) add_weights<kHeads, kStep>(a, unit0, pair, w.t, w.left, w.rows, warp, lane, s_final);
    __syncwarp();
    cluster_sync_all();                                   // nobody leaves while its sums are being read
  }
}


constexpr int kMostBlocks = 2 * 160;
constexpr int kFinishThreads = 256;

// What a stretch has left: the maxima and sums of the pairs at its two ends where they are cut, half of the warps each; its share of the
// columns of the pair at its beginning (those behind a pair's first cut have a share each, neighbouring lanes some parts of a
// column each); then the weights of its tiles, a warp a tile. A chain of three loads, each for all that the one before has made known:
// 3 us, where asking for things as they came took 9 (32 sequences, 3 600 tiles). One block for all columns of a pair took long where few pairs
// are cut into many parts: 1 x 14 204 rows, 16 heads of 128, 124 us a call (24 now), 2 x 32 768, 8 x 2 x 128, 50.6 (48.6).
template <bool kStep>
__global__ void __launch_bounds__(kFinishThreads) paged_finish_kernel(const Args a, int D) {
  constexpr int kHalf = kFinishThreads / 2, kAhead = 4;
  __shared__ float s_scale[2][kMostBlocks * 16];          // of a part's head
  __shared__ float2 s_final[2][16];
  griddep_wait();
  griddep_launch_dependents();
  const int c = blockIdx.x, tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, G = a.G;
  const Stretch st = a.stretches[c];
  if (c >= st.blocks) return;
  // the first tile: scores of its first heads
  int u = st.begins + warp;
  const bool tile = a.scores && u < st.ends;
  const float* scores = a.scores + static_cast<long long>(u) * G * kTile + 2 * lane;
  int4 at = make_int4(-1, 0, 0, 0);
  float2 ahead[kAhead];
  if (tile) {
    at = a.tile_rows[u];
#pragma unroll
    for (int g = 0; g < kAhead; ++g) ahead[g] = *reinterpret_cast<const float2*>(scores + min(g, G - 1) * kTile);
  }
  const bool same = st.end[0].pair == st.end[1].pair;     // all warps for the one
  const int half = !same && tid >= kHalf;
  const End p = half ? st.end[1] : st.end[0];
  const bool cut = p.first < p.last;
  const int parts = p.last - p.first + 1, size = part_floats(G, D);
  auto part = [&](int x) { return a.part + (2LL * (p.first + x) + (x == 0 ? p.second : 0)) * size; };
  // columns: four a lane, `each` lanes of them; a lane's first parts are asked for here
  const End b = st.end[0];
  const int b_parts = b.last - b.first + 1;
  auto b_part = [&](int x) { return a.part + (2LL * (b.first + x) + (x == 0 ? b.second : 0)) * size; };
  int from = 0, to = 0, shift = 0;
  if (b.first < c) {
    const unsigned all = G * D / 4, share = (all + b_parts - 2) / static_cast<unsigned>(b_parts - 1);
    from = min(all, (c - b.first - 1) * share);
    to = min(all, from + share);
    while (shift < 5 && 1 << shift < b_parts && (to - from) << (shift + 1) <= kFinishThreads) ++shift;
  }
  const int each = 1 << shift, turn = tid & (each - 1);
  int i = from + (tid >> shift);
  float4 column[kAhead];
  if (i < to) {
#pragma unroll
    for (int x = 0; x < kAhead; ++x) column[x] = *reinterpret_cast<const float4*>(b_part(min(turn + x * each, b_parts - 1)) + 4 * i);
  }
  if (cut) {
    for (int g = (tid - half * kHalf) >> 5; g < G; g += (same ? kFinishThreads : kHalf) / 32) {
      float top = -FLT_MAX, sum = 0.f;
#pragma unroll 4
      for (int x = lane; x < parts; x += 32) {
        const float2 ml = *reinterpret_cast<const float2*>(part(x) + G * D + 2 * g);
        const float next = fmaxf(top, ml.x);
        sum = sum * exp2f(top - next) + ml.y * exp2f(ml.x - next);
        top = next;
        s_scale[half][x * G + g] = ml.x;
      }
      float most = top;
#pragma unroll
      for (int o = 16; o > 0; o >>= 1) most = fmaxf(most, __shfl_xor_sync(0xffffffffu, most, o));
      sum *= exp2f(top - most);
#pragma unroll
      for (int o = 16; o > 0; o >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
      if (lane == 0) s_final[half][g] = make_float2(most, 1.f / sum);
      for (int x = lane; x < parts; x += 32) s_scale[half][x * G + g] = exp2f(s_scale[half][x * G + g] - most);
    }
  }
  __syncthreads();
  for (int i0 = from; i0 < to; i0 += kFinishThreads >> shift, i += kFinishThreads >> shift) {     // the same for all lanes
    const bool has = i < to;
    const int g = has ? i >> (D == 64 ? 4 : 5) : 0;
    float4 v = make_float4(0.f, 0.f, 0.f, 0.f);
    auto add = [&](const float4& p4, float f) {
      v.x += p4.x * f;
      v.y += p4.y * f;
      v.z += p4.z * f;
      v.w += p4.w * f;
    };
    if (has) {
#pragma unroll
      for (int x = 0; x < kAhead; ++x) {
        const int at = turn + x * each;
        if (i0 > from) column[x] = *reinterpret_cast<const float4*>(b_part(min(at, b_parts - 1)) + 4 * i);
        if (at < b_parts) add(column[x], s_scale[0][at * G + g]);
      }
#pragma unroll 4
      for (int at = turn + (kAhead << shift); at < b_parts; at += each) add(*reinterpret_cast<const float4*>(b_part(at) + 4 * i), s_scale[0][at * G + g]);
    }
    for (int o = 1; o < each; o <<= 1) {
      v.x += __shfl_xor_sync(0xffffffffu, v.x, o);
      v.y += __shfl_xor_sync(0xffffffffu, v.y, o);
      v.z += __shfl_xor_sync(0xffffffffu, v.z, o);
      v.w += __shfl_xor_sync(0xffffffffu, v.w, o);
    }
    if (has && turn == 0) {
      const float inv = s_final[0][g].y;
      *reinterpret_cast<uint2*>(a.out + static_cast<long long>(b.pair) * G * D + 4 * i) =
          make_uint2(bf_pack(v.x * inv, v.y * inv), bf_pack(v.z * inv, v.w * inv));
    }
  }
  if (!tile) return;
  while (true) {
    const int row = at.y + 2 * lane, rows = at.z;
    float* w = a.c.weights + static_cast<long long>(at.x) * a.c.width * a.c.page + row;
    const float2 old = row < rows ? *reinterpret_cast<const float2*>(w) : make_float2(0.f, 0.f);
    const float2* final = a.top_sum + static_cast<long long>(at.x) * G;
    if (at.x == st.end[0].pair && st.end[0].first < st.end[0].last) {
      final = s_final[0];
    } else if (at.x == st.end[1].pair && st.end[1].first < st.end[1].last) {
      final = s_final[1];
    }
    // the next tile is asked for before this one's numbers are needed
    const bool more = u + kFinishThreads / 32 < st.ends;
    const float* next_scores = scores + kFinishThreads / 32 * G * kTile;
    int4 next_at = at;
    float2 next[kAhead];
    if (more) {
      next_at = a.tile_rows[u + kFinishThreads / 32];
#pragma unroll
      for (int g = 0; g < kAhead; ++g) next[g] = *reinterpret_cast<const float2*>(next_scores + min(g, G - 1) * kTile);
    }
    float s0 = 0.f, s1 = 0.f;
#pragma unroll
    for (int g = 0; g < kAhead; ++g) {
      if (g >= G) continue;
      const float2 f = final[g];
      s0 += exp2f(ahead[g].x - f.x) * f.y;
      s1 += exp2f(ahead[g].y - f.x) * f.y;
    }
#pragma unroll 4
    for (int g = kAhead; g < G; ++g) {
      const float2 s = *reinterpret_cast<const float2*>(scores + g * kTile), f = final[g];
      s0 += exp2f(s.x - f.x) * f.y;
      s1 += exp2f(s.y - f.x) * f.y;
    }
    // a new row's weight starts from 0
    if (row < rows) w[0] = (kStep && row == rows - 1 ? 0.f : old.x) + s0;
    if (row + 1 < rows) w[1] = (kStep && row + 1 == rows - 1 ? 0.f : old.y) + s1;
    if (!more) return;
    u += kFinishThreads / 32;
    scores = next_scores;
    at = next_at;
#pragma unroll
    for (int g = 0; g < kAhead; ++g) ahead[g] = next[g];
  }
}

// What a step needs of an SM is the same.
int clusters_of_pairs(int D, bool wide, int blocks) {
#define CDEEP_FIT(DD, WIDE)  \
  if (D == DD && wide == WIDE) return clusters_side_by_side<paged_attention_kernel<DD, WIDE, false, true>>(blocks, kThreads, smem_bytes(DD, WIDE));
  CDEEP_FIT(64, false) CDEEP_FIT(64, true) CDEEP_FIT(128, false) CDEEP_FIT(128, true)
#undef CDEEP_FIT
  return 1 << 30;
}

// Blocks of a pair where short caches take clusters, else 0: as many as give every block an SM to itself, twice as many where they
// would have more than eight tiles and two fit an SM; up to 16 tiles a block. us, cold L2, events included, line / clusters of 1 / 2 / 4 / 8,
// 8 heads of 2 x 128: 1 x 512 rows 15 / 16 / 13 / 12 / 12, 1 x 4 096 26 / 55 / 33 / 23 / 16, 4 x 1 024 20 / 21 / 16 / 14 / 16, 4 x 4 096
// 30 / 55 / 35 / 27 / 27, 8 x 512 18 / 16 / 14 / 16 / 23, 8 x 2 048 30 / 33 / 27 / 25 / 33, 16 x 1 024 30 / 25 / 25 / 31, 16 x 2 048
// 42 / 39 / 39 / 43, 32 x 256 22 / 19 / 24, 32 x 1 024 42 / 37 / 43, 64 x 128 22 / 23, 64 x 512 42 / 41; with weights, lengths between a
// half and all: 8 x 1 024 24 / 27 / 23 / 21 / 27, 32 x 1 024 40 / 39 / 45.
// Clusters that do not fit side by side (they lie within a part of the GPU, and 16 heads of 128 have an SM to a block) are halved: 16
// clusters of eight took two turns, 4 x 1 000 rows, 4 x 16 x 128, 20.3, of four 11.4.
int cluster_of(long long pairs, long long tiles, int D, bool wide) {
  const int fit = blocks_per_sm(D, wide);
  const long long sms = current_sm_count();
  int blocks = 1;
  while (blocks < kMostCluster && 2 * blocks * pairs <= sms && 2 * blocks <= tiles) blocks *= 2;
  if (blocks < kMostCluster && 2 * blocks * pairs <= fit * sms && tiles > kClusterTiles / 2 * blocks) blocks *= 2;
  while (blocks > 1 && pairs > clusters_of_pairs(D, wide, blocks)) blocks /= 2;
  return blocks * pairs <= fit * sms && (tiles + blocks - 1) / blocks <= kClusterTiles ? blocks : 0;
}

// Where things lie in the workspace.
struct Layout {
  int cluster;
  long long tiles;        // of a pair
  size_t part, tile_rows, top_sum, scores, bytes;
};
Layout layout(int B, int hkv, int G, int D, int page, int width, bool weights) {
  Layout l = {};
  l.cluster = cluster_of(static_cast<long long>(B) * hkv, (static_cast<long long>(width) * page + kTile - 1) / kTile, D, G > 8);
  auto take = [&](size_t n) {
    const size_t at = l.bytes;
    l.bytes += (n + 255) / 256 * 256;
    return at;
  };
  const long long rows = static_cast<long long>(width) * page, pairs = static_cast<long long>(B) * hkv;
  l.tiles = (rows + kTile - 1) / kTile;
  if (!l.cluster) {
    take(sizeof(Stretch) * kMostBlocks);
    l.part = take(sizeof(float) * kMostBlocks * 2 * part_floats(G, D));
    l.tile_rows = weights ? take(sizeof(int4) * l.tiles * pairs) : 0;
    l.top_sum = weights ? take(sizeof(float2) * pairs * G) : 0;
  }
  l.scores = weights ? take(sizeof(float) * l.tiles * pairs * G * kTile) : 0;
  return l;
}

template <int D, bool kWide, bool kStep>
cudaError_t launch_one(const CUtensorMap& k, const CUtensorMap& v, const Args& a, cudaStream_t stream) {
  const long long pairs = static_cast<long long>(a.B) * a.hkv;
  if (a.cluster) {
    constexpr auto kKernel = paged_attention_kernel<D, kWide, kStep, true>;
    const cudaError_t e = allow_smem<kKernel>(smem_bytes(D, kWide));
    if (e != cudaSuccess) return e;
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3(static_cast<unsigned>(pairs * a.cluster));
    cfg.blockDim = dim3(kThreads);
    cfg.dynamicSmemBytes = smem_bytes(D, kWide);
    cfg.stream = stream;
    cudaLaunchAttribute attr[2];
    attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[0].val.programmaticStreamSerializationAllowed = pdl_enabled() ? 1 : 0;
    attr[1].id = cudaLaunchAttributeClusterDimension;
    attr[1].val.clusterDim.x = a.cluster;
    attr[1].val.clusterDim.y = attr[1].val.clusterDim.z = 1;
    cfg.attrs = attr;
    cfg.numAttrs = 2;
    return cudaLaunchKernelEx(&cfg, kKernel, k, v, a);
  }
  constexpr auto kKernel = paged_attention_kernel<D, kWide, kStep, false>;
  cudaError_t e = allow_smem<kKernel>(smem_bytes(D, kWide));
  if (e != cudaSuccess) return e;
  const long long most = current_sm_count() * blocks_per_sm(D, kWide) < kMostBlocks ? current_sm_count() * blocks_per_sm(D, kWide) : kMostBlocks;
  const int blocks = static_cast<int>(pairs * a.pair_tiles < most ? pairs * a.pair_tiles : most);
  e = launch_kernel(kKernel, dim3(blocks), dim3(kThreads), smem_bytes(D, kWide), stream, k, v, a);
  if (e != cudaSuccess) return e;
  return launch_kernel(paged_finish_kernel<kStep>, dim3(blocks), dim3(kFinishThreads), 0, stream, a, D);
}

}  // namespace

size_t paged_attention_workspace_bytes(int B, int hq, int hkv, int D, int page, int width, bool weights) {
  return layout(B, hkv, hq / hkv, D, page, width, weights).bytes;
}

cudaError_t launch_paged_attention(const cd_paged& c, const cd_paged_step* step, const void* q, long long q_stride, float scale, int B,
                                   int hq, int hkv, int D, void* out, void* ws, int* status, cudaStream_t stream) {
  const Layout l = layout(B, hkv, hq / hkv, D, c.page, c.width, c.weights != nullptr);
  char* base = static_cast<char*>(ws);
  Args a;
  a.c = c;
  a.q = static_cast<const bf16*>(q);
  a.q_stride = q_stride;
  a.st = step ? *step : cd_paged_step{};
  a.scale_log2 = scale * kLog2e;
  a.B = B;
  a.hkv = hkv;
  a.G = hq / hkv;
  a.box_rows = c.page < kTile ? c.page : kTile;
  a.boxes = kTile / a.box_rows;
  a.out = static_cast<bf16*>(out);
  a.status = status;
  a.pair_tiles = l.tiles;
  a.cluster = l.cluster;
  a.stretches = reinterpret_cast<Stretch*>(base);
  a.part = reinterpret_cast<float*>(base + l.part);
  a.tile_rows = reinterpret_cast<int4*>(base + l.tile_rows);
  a.top_sum = reinterpret_cast<float2*>(base + l.top_sum);
  a.scores = c.weights ? reinterpret_cast<float*>(base + l.scores) : nullptr;
  CUtensorMap k, v;
  const int dims[4] = {D, c.page, hkv, c.pages};
  const long long strides[3] = {c.stride_t, c.stride_h, c.stride_p};
  if (!encode_map_4d(&k, c.k, dims, strides, a.box_rows) || !encode_map_4d(&v, c.v, dims, strides, a.box_rows))
    return cudaErrorInvalidValue;
#define CDEEP_PAGED(DD, WIDE)                                                                                     \
  if (D == DD && (a.G > 8) == WIDE)                                                                               \
    return step ? launch_one<DD, WIDE, true>(k, v, a, stream) : launch_one<DD, WIDE, false>(k, v, a, stream);
  CDEEP_PAGED(64, false) CDEEP_PAGED(64, true) CDEEP_PAGED(128, false) CDEEP_PAGED(128, true)
#undef CDEEP_PAGED
  return cudaErrorInvalidValue;
}

}  // namespace cdeep
