// The next token of every row of logits, from a given uniform number u:
//
//   w_i = exp((x_i - max) / T);  top-k: x_i at least the k-th largest (ties stay);  top-p: in descending order, ties by the lowest
//   index, i stays where the mass ahead of it is at most p times the mass that top-k has left;  min-p: w_i >= min_p;
//   id = the first i, in the order of the vocabulary, with sum_{j <= i} w_j > u sum_j w_j over what stayed.
//
// The result is a whole number that hangs on where sums lie next to a border, so weights are 64-bit exponentials, held as multiples
// of 2^-44: sums of up to 2^18 of them are exact, and the same in any order.
//
// A cluster of blocks a row, which is read once and stays in their shared memory. A warp has a stretch of neighbouring tokens, its
// lanes take 16 bytes of it in turn.
//
// A small top-k leaves a few dozen of 100 000 tokens. The k-th largest of any k or more values bounds the k-th largest of all from
// below; taken of the largest lane maxima of every warp, twice k of them, it is hardly less. What reaches the bound (little more than
// k tokens) goes into a list; order, masses and the draw are then a matter of comparing its entries pair by pair.
//
// Where everything counts (no top-k, a large one, many equal values), the border of the top-k or of the nucleus is looked for by
// histograms over equal steps of the value between the largest and the smallest one left: counts, or masses as three numbers of 15
// bits, then the bin of the border alone, by pairs where it holds few values and in finer steps where it does not.
#include <cuda_bf16.h>
#include <cuda_runtime.h>
#include "elem.cuh"
#include "kernels.h"
#include "ptx.cuh"

namespace cdeep {

namespace {

constexpr int kThreads = 1024, kWarps = kThreads / 32;
constexpr int kBins = 2048;
constexpr int kList = 512;                 // entries compared pair by pair
constexpr int kFew = 256;                  // the largest k that takes the bound
constexpr int kMostBlocks = 8;             // of a row: the largest cluster that every device takes
constexpr int kSliceBytes = 128 * 1024;    // of a row that a block holds at most: 2^18 numbers of 32 bits are eight
using u64 = unsigned long long;
constexpr u64 kOne = 1ull << 44;

// Order of logits as unsigned numbers; NaN below -inf.
__device__ __forceinline__ uint32_t key_of(float x) {
  const uint32_t u = __float_as_uint(x + 0.f);
  return x != x ? 0u : u & 0x80000000u ? ~u : u | 0x80000000u;
}
__device__ __forceinline__ float value_of(uint32_t k) { return __uint_as_float(k & 0x80000000u ? k & 0x7fffffffu : ~k); }
constexpr uint32_t kMinusInf = 0x007fffffu;
// One order of all tokens: by value, ties by the lowest index.
__device__ __forceinline__ u64 token(uint32_t key, int i) { return static_cast<u64>(key) << 32 | ~static_cast<uint32_t>(i); }

__device__ __forceinline__ u64 fraction(float f) {        // of 2^64, f clamped to [0, 1)
  return f > 0.f ? f < 1.f ? static_cast<u64>(static_cast<double>(f) * 18446744073709551616.0) : ~0ull : 0ull;
}

__device__ __forceinline__ uint32_t peer32(const void* p, int rank) {
  uint32_t v;
  asm volatile("ld.shared::cluster.u32 %0, [%1];" : "=r"(v) : "r"(map_to_cta(smem_u32(p), rank)) : "memory");
  return v;
}
__device__ __forceinline__ u64 peer64(const void* p, int rank) {
  u64 v;
  asm volatile("ld.shared::cluster.u64 %0, [%1];" : "=l"(v) : "r"(map_to_cta(smem_u32(p), rank)) : "memory");
  return v;
}

struct Shared {
  double powers[64];                       // 2^(j / 64 + 44)
  u64 sums[kWarps];
  u64 total;                               // of this block, for the others
  u64 list[kList];                         // tokens; of this block, then (in the first) of all
  u64 mass[kList], sorted[kList];
  u64 found, before;
  unsigned hist[3][kBins];
  unsigned tops[kThreads], all_tops[kThreads];
  unsigned high, low, tau, count, key;
  int bin;
};

template <typename T>
struct Row {
  static constexpr int kVec = 16 / sizeof(T);
  Shared* s;
  const uint4* data;                       // this block's share of the row
  int begin, stretch;                      // its first token, tokens of a warp
  int rank, blocks;
  uint32_t best;
  double top, rate;                        // rate: 64 log2 e / T

  __device__ __forceinline__ void sync() const {
    if (blocks > 1) {
      cluster_sync_all();
    } else {
      __syncthreads();
    }
  }
  // f(key, token index) for this thread's share; -inf and NaN are left out
  template <typename F>
  __device__ __forceinline__ void each(F f) const {
    const int lane = threadIdx.x & 31, from = (threadIdx.x >> 5) * stretch;
    for (int v = from + lane * kVec; v < from + stretch; v += 32 * kVec) vec(v, f);
  }
  template <typename F>
  __device__ __forceinline__ void vec(int v, F f) const {
    const uint4 q = data[v / kVec];
    const uint32_t w[4] = {q.x, q.y, q.z, q.w};
#pragma unroll
    for (int e = 0; e < kVec; ++e) {
      const float x = sizeof(T) == 4 ? __uint_as_float(w[e * sizeof(T) / 4]) : e & 1 ? bf_hi(w[e / 2 % 4]) : bf_lo(w[e / 2 % 4]);
      const uint32_t k = key_of(x);
      if (k > kMinusInf) f(k, begin + v + e);
    }
  }
  // exp((x - max) / T) as a multiple of 2^-44: 2^(n / 64) from the table, the rest by a Taylor polynomial (error 2^-44)
  __device__ __forceinline__ u64 mass(uint32_t key) const {
    if (key == best) return kOne;
    const double y = (static_cast<double>(value_of(key)) - top) * rate;
    if (!(y > -64.0 * 46)) return 0;
    const double t = y + 6755399441055744.0;              // 1.5 2^52: rounds to a whole number, in the low bits
    const int n = __double2loint(t);
    const double r = (y - (t - 6755399441055744.0)) * 0.010830424696249145;   // ln 2 / 64
    double p = fma(r, 1.0 / 24, 1.0 / 6);
    p = fma(r, p, 0.5);
    p = fma(r, p, 1.0);
    p = fma(r, p, 1.0) * s->powers[n & 63];
    p = __hiloint2double(__double2hiint(p) + ((n >> 6) << 20), __double2loint(p));
    return __double_as_longlong(p + 4503599627370496.0) & 0xfffffffffffffull;   // + 2^52: rounds, the number in the low bits
  }
};

__device__ __forceinline__ u64 warp_sum(u64 v) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
  return v;
}
__device__ __forceinline__ u64 warp_upto(u64 v) {
  const int lane = threadIdx.x & 31;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const u64 up = __shfl_up_sync(0xffffffffu, v, o);
    if (lane >= o) v += up;
  }
  return v;
}
// Sum over the threads ahead of this one; `sums` holds every warp's.
__device__ __forceinline__ u64 block_before(u64 v, u64* sums) {
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const u64 upto = warp_upto(v);
  __syncthreads();
  if (lane == 31) sums[warp] = upto;
  __syncthreads();
  const u64 ahead = warp_sum(lane < warp ? sums[lane] : 0);
  return ahead + upto - v;
}
__device__ __forceinline__ u64 all_sums(const u64* sums) { return warp_sum(sums[threadIdx.x & 31]); }

// Lists the tokens that `takes` holds for, in every block those of all blocks. Returns how many there are; more than kList are not
// kept.
template <typename T, typename F>
__device__ __forceinline__ unsigned collect(const Row<T>& r, F takes) {
  Shared& s = *r.s;
  __syncthreads();
  if (threadIdx.x == 0) s.count = 0;
  __syncthreads();
  r.each([&](uint32_t k, int i) {
    if (takes(k, i)) {
      const unsigned at = atomicAdd(&s.count, 1u);
      if (at < kList) s.list[at] = token(k, i);
    }
  });
  r.sync();
  if (r.blocks == 1) return s.count;
  unsigned all = 0;
  for (int b = 0; b < r.blocks; ++b) all += peer32(&s.count, b);
  if (all <= kList) {                      // every block has them all, in the same places
    u64 t = 0;
    if (threadIdx.x < all) {
      unsigned at = threadIdx.x;
      int b = 0;
      for (unsigned m; at >= (m = peer32(&s.count, b)); ++b) at -= m;
      t = peer64(&s.list[at], b);
    }
    r.sync();
    if (threadIdx.x < all) s.list[threadIdx.x] = t;
    __syncthreads();
  }
  return all;
}

// Sum over all blocks; s.before: that of the blocks ahead of this one, s.sums: those of its warps.
template <typename T>
__device__ __forceinline__ u64 row_sum(const Row<T>& r, u64 own) {
  Shared& s = *r.s;
  __syncthreads();
  const u64 w = warp_sum(own);
  if ((threadIdx.x & 31) == 0) s.sums[threadIdx.x >> 5] = w;
  __syncthreads();
  const u64 block = all_sums(s.sums);
  if (r.blocks == 1) {
    if (threadIdx.x == 0) s.before = 0;
    __syncthreads();
    return block;
  }
  if (threadIdx.x == 0) s.total = block;
  r.sync();
  u64 all = 0, before = 0;
  for (int b = 0; b < r.blocks; ++b) {
    const u64 t = peer64(&s.total, b);
    if (b < r.rank) before += t;
    all += t;
  }
  r.sync();
  if (threadIdx.x == 0) s.before = before;
  __syncthreads();
  return all;
}

// The r-th (from 0) of the tokens with this key, in the order of the vocabulary; all if there are no more than r.
template <typename T>
__device__ __forceinline__ int nth_equal(const Row<T>& r, uint32_t key, u64 nth) {
  Shared& s = *r.s;
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  if (threadIdx.x == 0) s.found = ~0ull;
  u64 own = 0;
  r.each([&](uint32_t k, int) { own += k == key; });
  row_sum(r, own);
  const u64 mine = s.sums[warp];
  u64 before = s.before + warp_sum(lane < warp ? s.sums[lane] : 0);
  if (before <= nth && nth < before + mine) {             // it lies in this warp's stretch
    for (int v0 = warp * r.stretch; v0 < (warp + 1) * r.stretch; v0 += 32 * Row<T>::kVec) {
      const int v = v0 + lane * Row<T>::kVec;
      u64 n = 0;
      if (v < (warp + 1) * r.stretch) r.vec(v, [&](uint32_t k, int) { n += k == key; });
      const u64 upto = warp_upto(n);
      u64 at = before + upto - n;
      if (n > 0 && at <= nth && nth < at + n)
        r.vec(v, [&](uint32_t k, int i) {
          if (k == key && at++ == nth) s.found = i;
        });
      before += __shfl_sync(0xffffffffu, upto, 31);
    }
  }
  r.sync();
  u64 found = s.found;
  for (int b = 0; b < r.blocks && r.blocks > 1; ++b) found = min(found, peer64(&s.found, b));
  r.sync();
  return found == ~0ull ? 0x7fffffff : static_cast<int>(found);
}

// The last token, in descending order through the keys from `high` down to `low` (both there), that has at most so much ahead of it:
// `left` tokens, or (kMass) that fraction of the mass of all. For counts only the key of the result means something.
template <bool kMass, typename T>
__device__ __forceinline__ u64 border(const Row<T>& r, uint32_t low, uint32_t high, u64 left) {
  Shared& s = *r.s;
  const int tid = threadIdx.x;
  bool first = true;
  while (low < high) {
    // equal steps of the value behind the largest, which has bin 0 to itself: every turn leaves it behind or ends with it
    const float most = value_of(high);
    const float steps = static_cast<float>((kBins - 1) / (static_cast<double>(most) - static_cast<double>(value_of(low))));
    auto bin_of = [&](uint32_t k) { return k == high ? 0 : 1 + min(kBins - 2, __float2int_rz((most - value_of(k)) * steps)); };
    for (int i = tid; i < (kMass ? 3 : 1) * kBins; i += kThreads) (&s.hist[0][0])[i] = 0;
    if (tid == 0) s.bin = -1, s.high = 0, s.low = 0xffffffffu;
    __syncthreads();
    r.each([&](uint32_t k, int) {
      if (k < low || k > high) return;
      const int b = bin_of(k);
      if constexpr (kMass) {
        const u64 m = r.mass(k);
        const unsigned m0 = m & 0x7fff, m1 = m >> 15 & 0x7fff, m2 = static_cast<unsigned>(m >> 30);
        if (m0) atomicAdd(&s.hist[0][b], m0);
        if (m1) atomicAdd(&s.hist[1][b], m1);
        if (m2) atomicAdd(&s.hist[2][b], m2);
      } else {
        atomicAdd(&s.hist[0][b], 1u);
      }
    });
    r.sync();
    u64 held[2];
#pragma unroll
    for (int x = 0; x < 2; ++x) {
      held[x] = 0;
      for (int b = 0; b < r.blocks; ++b) {
#pragma unroll
        for (int e = 0; e < (kMass ? 3 : 1); ++e) {
          const unsigned* at = &s.hist[e][2 * tid + x];
          held[x] += static_cast<u64>(r.blocks > 1 ? peer32(at, b) : *at) << 15 * e;
        }
      }
    }
    const u64 before = block_before(held[0] + held[1], s.sums);
    if (kMass && first) left = __umul64hi(left, all_sums(s.sums));
    first = false;
    const int last = held[1] > 0 && before + held[0] <= left ? 2 * tid + 1 : held[0] > 0 && before <= left ? 2 * tid : -1;
    if (last >= 0) atomicMax(&s.bin, last);
    __syncthreads();
    const int bin = s.bin;
    if (last == bin && last >= 0) s.before = before + (last & 1 ? held[0] : 0);
    __syncthreads();
    left -= s.before;
    unsigned hi = 0, lo = 0xffffffffu;
    const unsigned n = collect(r, [&](uint32_t k, int) {
      if (k < low || k > high || bin_of(k) != bin) return false;
      hi = max(hi, k);
      lo = min(lo, k);
      return true;
    });
    if (n <= kList) {
      const u64 mine = tid < n ? s.list[tid] : 0;
      if (tid < n && kMass) s.mass[tid] = r.mass(static_cast<uint32_t>(mine >> 32));
      if (tid == 0) s.found = ~0ull;
      __syncthreads();
      if (tid < n) {
        u64 ahead = 0;
        for (int j = 0; j < n; ++j)
          if (s.list[j] > mine) ahead += kMass ? s.mass[j] : 1;
        if (ahead <= left) atomicMin(&s.found, mine);
      }
      __syncthreads();
      const u64 found = s.found;
      __syncthreads();
      return found;
    }
    hi = __reduce_max_sync(0xffffffffu, hi);
    lo = __reduce_min_sync(0xffffffffu, lo);
    if ((tid & 31) == 0) {
      atomicMax(&s.high, hi);
      atomicMin(&s.low, lo);
    }
    r.sync();
    high = 0;
    low = 0xffffffffu;
    for (int b = 0; b < r.blocks; ++b) {
      high = max(high, r.blocks > 1 ? peer32(&s.high, b) : s.high);
      low = min(low, r.blocks > 1 ? peer32(&s.low, b) : s.low);
    }
    r.sync();
  }
  // equal values only
  if (!kMass) return token(high, 0);
  const u64 m = r.mass(high);
  if (first) {
    u64 own = 0;
    r.each([&](uint32_t k, int) { own += k == high; });
    left = __umul64hi(left, row_sum(r, own) * m);
  }
  return token(high, nth_equal(r, high, m > 0 ? left / m : ~0ull));
}

template <typename T>
__global__ void __launch_bounds__(kThreads) sample_tokens_kernel(const T* logits, long long ld, int V, int slice, int stretch, cd_sample p,
                                                                 long long* ids, float* probs) {
  constexpr int kVec = Row<T>::kVec;
  extern __shared__ uint4 s_dyn[];
  Shared& s = *reinterpret_cast<Shared*>(s_dyn);
  uint4* s_data = s_dyn + (sizeof(Shared) + 15) / 16;
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  if (tid < 64) s.powers[tid] = exp2(tid / 64.0 + 44.0);
  if (tid == 0) s.key = 0, s.low = 0xffffffffu, s.tau = 0;
  __syncthreads();
  griddep_wait();
  griddep_launch_dependents();
  Row<T> r;
  r.s = &s;
  r.data = s_data;
  r.blocks = gridDim.x;
  r.rank = blockIdx.x;
  r.begin = r.rank * slice;
  r.stretch = stretch;
  const int b = blockIdx.y, length = max(0, min(slice, V - r.begin));
  const T* x = logits + b * ld + r.begin;
  const float temperature = p.temperatures ? p.temperatures[b] : p.temperature;
  const float top_p = p.top_ps ? p.top_ps[b] : p.top_p;
  const float min_p = p.min_ps ? p.min_ps[b] : p.min_p;
  const int top_k = p.top_ks ? p.top_ks[b] : p.top_k;

  // the row's share into shared memory, NaN behind its end
  uint32_t high = 0, low = 0xffffffffu;
  const bool whole = (reinterpret_cast<uintptr_t>(x) & 15) == 0;
  for (int v = warp * stretch + lane * kVec; v < (warp + 1) * stretch; v += 32 * kVec) {
    uint4 q = make_uint4(0xffffffffu, 0xffffffffu, 0xffffffffu, 0xffffffffu);
    if (whole && v + kVec <= length) {
      q = *reinterpret_cast<const uint4*>(x + v);
    } else {
      T* e = reinterpret_cast<T*>(&q);
      for (int i = 0; i < kVec && v + i < length; ++i) e[i] = x[v + i];
    }
    s_data[v / kVec] = q;
    r.vec(v, [&](uint32_t k, int) {
      high = max(high, k);
      low = min(low, k);
    });
  }
  // the largest lane maxima of every warp
  const int warps = min(r.blocks * kWarps, (V + stretch - 1) / stretch);     // that have tokens
  const int draws = max(2, (2 * top_k + warps - 1) / warps);
  const bool few = top_k > 0 && top_k < V && top_k <= kFew && draws <= 32;
  if (few) {
    uint32_t m = high;
    for (int d = 0; d < draws; ++d) {
      const uint32_t largest = __reduce_max_sync(0xffffffffu, m);
      const unsigned has = __ballot_sync(0xffffffffu, m == largest);
      if (lane == __ffs(has) - 1) m = 0;
      if (lane == 0) s.tops[warp * draws + d] = largest;
    }
  }
  high = __reduce_max_sync(0xffffffffu, high);
  low = __reduce_min_sync(0xffffffffu, low);
  if (lane == 0) {
    atomicMax(&s.key, high);
    atomicMin(&s.low, low);
  }
  r.sync();
  uint32_t best = 0, least = 0xffffffffu;
  for (int c = 0; c < r.blocks; ++c) {
    best = max(best, r.blocks > 1 ? peer32(&s.key, c) : s.key);
    least = min(least, r.blocks > 1 ? peer32(&s.low, c) : s.low);
  }
  if (few) {                                              // the k-th largest of them
    const int each = min(kWarps, warps) * draws, n = warps * draws;
    if (tid < n) s.all_tops[tid] = r.blocks > 1 ? peer32(&s.tops[tid % each], tid / each) : s.tops[tid];
    __syncthreads();
    if (tid < n) {
      const uint32_t mine = s.all_tops[tid];
      int rank = 0;
      for (int j = 0; j < n; ++j) {
        const uint32_t t = s.all_tops[j];
        rank += t > mine || (t == mine && j < tid);
      }
      if (rank == top_k - 1) s.tau = mine;
    }
  }
  r.sync();
  const uint32_t tau = s.tau;
  r.best = best;
  r.top = value_of(best);
  r.rate = 92.332482616893656 / static_cast<double>(temperature);          // 64 log2 e

  if (best <= kMinusInf) {                                // nothing to draw from
    if (tid == 0 && r.rank == 0) ids[b] = 0, probs[b] = 0.f;
    return;
  }
  if (!(temperature > 0.f)) {
    const int first = nth_equal(r, best, 0);
    if (tid == 0 && r.rank == 0) ids[b] = first, probs[b] = 1.f;
    return;
  }
  const u64 least_mass = min_p >= 1.f ? kOne : min_p > 0.f ? static_cast<u64>(ceil(static_cast<double>(min_p) * kOne)) : 0;
  const u64 u = fraction(p.uniform[b]), share = fraction(top_p);
  uint32_t from = kMinusInf + 1;
  bool listed = false;
  unsigned n = 0;
  if (few) {
    n = collect(r, [&](uint32_t k, int) { return k >= tau; });
    listed = n <= kList;
  }
  if (listed) {
    // everything that top-k may keep is in every block's list
    if (r.rank == 0) {
      const u64 mine = tid < n ? s.list[tid] : 0;
      const uint32_t key = mine >> 32;
      int rank = 0, greater = 0;
      if (tid < n) {
        for (int j = 0; j < n; ++j) {
          const u64 t = s.list[j];
          rank += t > mine;
          greater += static_cast<uint32_t>(t >> 32) > key;
        }
        s.mass[tid] = greater < top_k ? r.mass(key) : 0;
        s.sorted[rank] = s.mass[tid];
      }
      __syncthreads();
      const u64 w = tid < n ? s.sorted[tid] : 0;
      const u64 ahead = block_before(w, s.sums), total = all_sums(s.sums);
      __syncthreads();
      if (tid < n) s.sorted[tid] = top_p < 1.f && ahead > __umul64hi(share, total) ? 0 : w < least_mass ? 0 : w;
      __syncthreads();
      const u64 kept = tid < n ? s.sorted[rank] : 0;
      __syncthreads();
      if (tid < n) s.mass[tid] = kept;
      block_before(kept, s.sums);
      const u64 left = all_sums(s.sums);
      __syncthreads();
      // a token's reach in the vocabulary's order
      if (kept > 0) {
        u64 before = 0;
        const uint32_t at = static_cast<uint32_t>(mine);                   // ~index
        for (int j = 0; j < n; ++j)
          if (static_cast<uint32_t>(s.list[j]) > at) before += s.mass[j];
        const u64 target = __umul64hi(u, left);
        if (before <= target && target < before + kept) {
          ids[b] = static_cast<int>(~at);
          probs[b] = static_cast<float>(static_cast<double>(kept) / static_cast<double>(left));
        }
      }
    }
    if (r.blocks > 1) r.sync();
    return;
  }
  if (top_k > 0 && top_k < V) from = max(from, static_cast<uint32_t>(border<false>(r, least, best, static_cast<u64>(top_k - 1)) >> 32));
  u64 last = token(from, 0x7fffffff);                     // the last token that stays
  if (top_p < 1.f) last = border<true>(r, max(from, least), best, share);
  auto held = [&](uint32_t k, int i) -> u64 {
    if (token(k, i) < last) return 0;
    const u64 w = r.mass(k);
    return w < least_mass ? 0 : w;
  };
  u64 own = 0;
  r.each([&](uint32_t k, int i) { own += held(k, i); });
  const u64 total = row_sum(r, own), target = __umul64hi(u, total);
  const u64 mine = s.sums[warp];
  u64 before = s.before + warp_sum(lane < warp ? s.sums[lane] : 0);
  if (before <= target && target < before + mine) {       // in this warp's stretch
    for (int v0 = warp * stretch; v0 < (warp + 1) * stretch; v0 += 32 * kVec) {
      const int v = v0 + lane * kVec;
      u64 w = 0;
      if (v < (warp + 1) * stretch) r.vec(v, [&](uint32_t k, int i) { w += held(k, i); });
      const u64 upto = warp_upto(w);
      u64 at = before + upto - w;
      if (w > 0 && at <= target && target < at + w)
        r.vec(v, [&](uint32_t k, int i) {
          const u64 e = held(k, i);
          if (e > 0 && at <= target && target < at + e) {
            ids[b] = i;
            probs[b] = static_cast<float>(static_cast<double>(e) / static_cast<double>(total));
          }
          at += e;
        });
      before += __shfl_sync(0xffffffffu, upto, 31);
    }
  }
}

int sm_count() {
  int device = 0, n = 0;
  if (cudaGetDevice(&device) != cudaSuccess || cudaDeviceGetAttribute(&n, cudaDevAttrMultiProcessorCount, device) != cudaSuccess) return 148;
  return n;
}

template <typename T>
cudaError_t launch_one(const void* logits, long long ld, int B, int V, const cd_sample& p, int64_t* ids, float* probs, cudaStream_t stream) {
  constexpr auto kKernel = sample_tokens_kernel<T>;
  constexpr int kVec = Row<T>::kVec;
  // as many blocks a row as its size asks for, and more while the device has SMs without one and a block has 4 096 tokens
  int blocks = 1;
  while (static_cast<long long>(V) * sizeof(T) > static_cast<long long>(blocks) * kSliceBytes) blocks *= 2;
  while (blocks < kMostBlocks && 2LL * blocks * B <= sm_count() && V / (2 * blocks) >= 4096) blocks *= 2;
  const int least = 32 * kVec;                            // of a warp: 16 bytes a lane
  int stretch = (V + blocks * kWarps - 1) / (blocks * kWarps);
  stretch = stretch < least ? least : (stretch + kVec - 1) / kVec * kVec;
  const int slice = stretch * kWarps, bytes = (sizeof(Shared) + 15) / 16 * 16 + slice * static_cast<int>(sizeof(T));
  cudaError_t e = allow_smem<kKernel>(bytes);
  if (e != cudaSuccess) return e;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(blocks, B);
  cfg.blockDim = dim3(kThreads);
  cfg.dynamicSmemBytes = bytes;
  cfg.stream = stream;
  cudaLaunchAttribute attr[2];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = pdl_enabled() ? 1 : 0;
  attr[1].id = cudaLaunchAttributeClusterDimension;
  attr[1].val.clusterDim.x = blocks;
  attr[1].val.clusterDim.y = attr[1].val.clusterDim.z = 1;
  cfg.attrs = attr;
  cfg.numAttrs = blocks > 1 ? 2 : 1;
  return cudaLaunchKernelEx(&cfg, kKernel, static_cast<const T*>(logits), ld, V, slice, stretch, p, reinterpret_cast<long long*>(ids), probs);
}

}  // namespace

cudaError_t launch_sample_tokens(const void* logits, int fp32, long long ld, int B, int V, const cd_sample& p, int64_t* ids, float* probs,
                                 cudaStream_t stream) {
  return fp32 ? launch_one<float>(logits, ld, B, V, p, ids, probs, stream) : launch_one<bf16>(logits, ld, B, V, p, ids, probs, stream);
}

}  // namespace cdeep
