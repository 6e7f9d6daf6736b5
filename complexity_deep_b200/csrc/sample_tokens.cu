// The next token of every row of logits, from a given uniform number u:
//
//   w_i = exp((x_i - max) / T);  top-k: x_i at least the k-th largest (ties stay);  top-p: in descending order, ties by the lowest
//   index, i stays where the mass ahead of it is at most p times the mass that top-k has left;  min-p: w_i >= min_p;
//   id = the first i, in the order of the vocabulary, with sum_{j <= i} w_j > u sum_j w_j over what stayed.
//
// The result is a whole number that hangs on where sums lie next to a border, so weights are good to 2^-30.6 of themselves and held as
// multiples of 2^-44: sums of up to 2^18 of them are exact, and the same in any order. Some thirty instructions on 32 bits give such a
// weight (Row::mass); in 64-bit arithmetic it took 2.6 times as long.
//
// A cluster of blocks a row, which is read once and stays in their shared memory. A warp has a stretch of neighbouring tokens, its
// lanes take 16 bytes of it in turn.
//
// A small top-k leaves a few dozen of 100 000 tokens. The k-th largest of any k or more values bounds the k-th largest of all from
// below; taken of the largest lane maxima of every warp, twice k of them, it is hardly less. What reaches the bound (little more than
// k tokens) goes into a list; order, masses and the draw are then a matter of comparing its entries pair by pair.
//
// Where everything counts (no top-k, a large one, many equal values), the border of the top-k or of the nucleus is looked for by
// histograms over equal steps of the value between the largest and the smallest one left: counts, or masses as their lower halves and
// the upper ones with what the lower carry. Then the bin of the border alone: in finer steps where it holds many values; otherwise as a
// list, of which every warp weighs what lies ahead of one, 32 at a time (294 values: 7 000 clocks; all pairs of them 10 700).
// The draw weighs what has stayed once more: picked from 32 tokens of a lane at a time, 18 000 clocks for 100 000 tokens of which a
// third stays, 24 000 with a weight for every token. The warp's stretch in which it ends is taken by the whole block: 2 200 clocks, 8 000
// for the warp alone.
#include <cuda_bf16.h>
#include <cuda_runtime.h>
#include "elem.cuh"
#include "kernels.h"
#include "ptx.cuh"

namespace cdeep {

namespace {

constexpr int kList = 512;                 // entries compared with one another
constexpr int kFew = 256;                  // the largest k that takes the bound
constexpr int kMany = 2048;                // tokens that a larger top-k leaves in a block, as a list
constexpr int kMostBlocks = 8;             // of a row: the largest cluster that every device takes
constexpr int kSliceBytes = 160 * 1024;    // of a row in a block, beside what Shared takes: 2^18 numbers of 32 bits are eight blocks
using u64 = unsigned long long;
constexpr u64 kOne = 1ull << 44;

// Order of logits as unsigned numbers, NaN below -inf, -0 as 0, +inf as the largest number; bf16 in the upper half.
template <typename T>
struct Key;
template <>
struct Key<float> {
  static constexpr uint32_t kMinusInf = 0x007fffffu;
  static __device__ __forceinline__ uint32_t of(uint32_t bits) {
    const uint32_t u = __float_as_uint(__uint_as_float(bits) + 0.f);
    const uint32_t k = u ^ (static_cast<uint32_t>(static_cast<int>(u) >> 31) | 0x80000000u);
    return (bits & 0x7fffffffu) > 0x7f800000u ? 0u : min(k, 0xff7fffffu);
  }
  static __device__ __forceinline__ float value(uint32_t k) {
    return __uint_as_float(k ^ (~static_cast<uint32_t>(static_cast<int>(k) >> 31) | 0x80000000u));
  }
  // the key of a number or of one just below it
  static __device__ __forceinline__ uint32_t near(float x) { return of(__float_as_uint(x)); }
  static __device__ __forceinline__ uint32_t most(uint32_t a, uint32_t b) { return max(a, b); }
  static __device__ __forceinline__ uint32_t largest(uint32_t m) { return m; }
  static __device__ __forceinline__ uint32_t unpack(const uint32_t (&w)[4], int e) { return w[e]; }
  static __device__ __forceinline__ uint32_t at(const uint4* data, int i) { return reinterpret_cast<const uint32_t*>(data)[i]; }
};
template <>
struct Key<bf16> {                         // two at a time
  static constexpr uint32_t kMinusInf = 0x007f0000u;
  static __device__ __forceinline__ uint32_t of(uint32_t bits) {
    const __nv_bfloat162 x = __hadd2(*reinterpret_cast<const __nv_bfloat162*>(&bits), __nv_bfloat162(from_f32<bf16>(0.f), from_f32<bf16>(0.f)));
    const uint32_t nan = __hneu2_mask(x, x), u = *reinterpret_cast<const uint32_t*>(&x);
    const uint32_t k = u ^ ((u >> 15 & 0x00010001u) * 0xffffu | 0x80008000u);
    return __vminu2(k & ~nan, 0xff7fff7fu);
  }
  static __device__ __forceinline__ float value(uint32_t k) {
    return __uint_as_float((k ^ (~static_cast<uint32_t>(static_cast<int>(k) >> 31) | 0x80000000u)) & 0xffff0000u);
  }
  static __device__ __forceinline__ uint32_t near(float x) { return Key<float>::of(__float_as_uint(x)) & 0xffff0000u; }
  static __device__ __forceinline__ uint32_t most(uint32_t a, uint32_t b) { return __vmaxu2(a, b); }
  static __device__ __forceinline__ uint32_t largest(uint32_t m) { return max(m & 0xffff0000u, m << 16); }
  static __device__ __forceinline__ uint32_t unpack(const uint32_t (&w)[4], int e) { return e & 1 ? w[e / 2] & 0xffff0000u : w[e / 2] << 16; }
  static __device__ __forceinline__ uint32_t at(const uint4* data, int i) { return static_cast<uint32_t>(reinterpret_cast<const uint16_t*>(data)[i]) << 16; }
};
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

template <int kThreads>
struct Shared {
  static constexpr int kWarps = kThreads / 32, kBins = 2 * kThreads;
  u64 list[kList + 2], mass[kList + 2];    // tokens; their masses
  u64 kept[kList + 2], many[kMany];
  unsigned all_tops[kThreads + 2];
  unsigned powers[256];                    // 2^(j / 256 + 31)
  u64 sums[kWarps];
  u64 total;                               // of this block, for the others
  u64 found, before;
  u64 open[kWarps];                        // tokens between the last known to stay and the first known to go
  bool stays[kWarps];
  unsigned hist[2][kBins];                 // masses: their lower halves, and the upper ones with what the lower carry
  unsigned tops[kThreads];
  unsigned high, low, tau, count, key;
  unsigned ends[2];                        // keys of a bin
  unsigned counts[kMostBlocks], opens;
  int bin;
};

static_assert((sizeof(Shared<1024>) + 15) / 16 * 16 + kSliceBytes + 32 * 16 <= 232448, "a block's share and what it is taken apart with");

template <typename T, int kThreads>
struct Row {
  static constexpr int kVec = 16 / sizeof(T);
  Shared<kThreads>* s;
  const uint4* data;                       // this block's share of the row
  int begin, stretch;                      // its first token, tokens of a warp
  int many = -1;
  int rank, blocks;
  uint32_t best;
  float top, rate, rate_low;               // 256 log2 e / T as two numbers

  __device__ __forceinline__ void sync() const {
    if (blocks > 1) {
      cluster_sync_all();
    } else {
      __syncthreads();
    }
  }
  // This thread's share of the tokens, in the order of the vocabulary: warps have stretches, lanes 16 bytes of it in turn, or one
  // entry of the list of tokens that top-k has left (many >= 0 of them in this block).
  __device__ __forceinline__ int width() const { return many < 0 ? kVec : 1; }
  __device__ __forceinline__ int from() const { return static_cast<int>(threadIdx.x >> 5) * stretch; }
  __device__ __forceinline__ int to() const { return many < 0 ? from() + stretch : min(many, from() + stretch); }
  // f(key, token index) for the tokens at place v; -inf and NaN are the keys up to kMinusInf
  template <typename F>
  __device__ __forceinline__ void at(int v, F f) const {
    if (many >= 0) {
      const u64 t = s->many[v];
      f(static_cast<uint32_t>(t >> 32), static_cast<int>(~static_cast<uint32_t>(t)));
      return;
    }
    const uint4 q = data[v / kVec];
    const uint32_t w[4] = {q.x, q.y, q.z, q.w};
#pragma unroll
    for (int e = 0; e < kVec; ++e) f(Key<T>::unpack(w, e), begin + v + e);
  }
  // f(key, token index) for the one token at place v
  template <typename F>
  __device__ __forceinline__ void one(int v, F f) const {
    if (many >= 0) {
      at(v, f);
    } else {
      f(Key<T>::at(data, v), begin + v);
    }
  }
  template <typename F>
  __device__ __forceinline__ void each(F f) const {
    const int w = width();
    for (int v = from() + static_cast<int>(threadIdx.x & 31) * w; v < to(); v += 32 * w) at(v, f);
  }
  // f(key, token index) for those of a key that takes(key) holds for, in any order: bits of 32 tokens of a lane first, so that a warp
  // turns as often as its lane of the most of them and not for every token that one lane takes.
  template <typename P, typename F>
  __device__ __forceinline__ void each_that(P takes, F f) const {
    if (many >= 0) {
      each([&](uint32_t k, int i) {
        if (takes(k)) f(k, i);
      });
      return;
    }
    for (int v0 = from() + static_cast<int>(threadIdx.x & 31) * kVec; v0 < to(); v0 += 32 * 32) {
      uint32_t bits = 0;
#pragma unroll
      for (int g = 0; g < 32; g += kVec) {
        const int v = v0 + 32 * g;
        if (v >= to()) break;
        const uint4 q = data[v / kVec];
        const uint32_t w[4] = {q.x, q.y, q.z, q.w};
#pragma unroll
        for (int e = 0; e < kVec; ++e)
          if (takes(Key<T>::unpack(w, e))) bits |= 1u << (g + e);
      }
      while (bits) {
        const int bit = 31 - __clz(bits), v = v0 + 32 * (bit & -kVec) + (bit & (kVec - 1));
        bits ^= 1u << bit;
        f(Key<T>::at(data, v), begin + v);
      }
    }
  }
  // f(places of the lanes' tokens) for the warp's steps: lanes beyond the end get a place that is not below to()
  template <typename F>
  __device__ __forceinline__ void steps(F f) const {
    const int w = width();
    for (int v = from(); v < to(); v += 32 * w) f(v + static_cast<int>(threadIdx.x & 31) * w);
  }
  // exp((x - max) / T) as a multiple of 2^-44, good to 2^-30.6 of itself (2^-32 each from the table and from the sum with q, the rest from
  // the polynomial; of 6 million logits 2^-30.69 at most, one in a thousand beyond 2^-31, 2^-37 on average; the upper half of the product
  // alone was off by up to 2^-29.4, always downwards): y = (x - max) 256 log2 e / T as a sum of two numbers, the whole part n of its
  // 256ths from the table, 2^(f / 256) = 1 + q of the rest by a polynomial, q in 2^-31ths. The largest has exactly 1. What lies below
  // 2^-45, -inf and NaN shift everything out. Whole-number instructions run at half the rate of the others here: what can be had from
  // products and sums is.
  __device__ __forceinline__ u64 mass(uint32_t key) const {
    const float x = Key<T>::value(key), d = x - top;
    float rest = 0.f;
    if constexpr (sizeof(T) == 4) {                       // what the difference has lost (of bf16 numbers: nothing that counts)
      const float back = d - x;
      rest = (x - (d - back)) - (top + back);
    }
    const float y = d * rate;
    const float low = fmaf(d, rate_low, fmaf(rest, rate, fmaf(d, rate, -y)));
    const float t = y + 12582912.f;                       // 1.5 2^23: rounds to a whole number, in the low bits
    const uint32_t n = __float_as_uint(t);                // 0x4b400000 + the whole part
    const float f = (y - (t - 12582912.f)) + low;
    const float q = f * fmaf(f, fmaf(f, 3.3083e-9f, 3.66556e-6f), 2.7076062e-3f);       // (ln 2 / 256)^i / i!
    const uint32_t one_q = __float_as_uint(q + 5.859375e-3f) + (0x80000000u - 0x3bc00000u);   // 1.5 2^-8; (1 + q) 2^31
    const u64 w = static_cast<u64>(s->powers[n & 255]) * one_q;                          // times 2^62
    const uint32_t w_hi = static_cast<uint32_t>(w >> 32), w_lo = static_cast<uint32_t>(w);
    const uint32_t shift = 18 + 0x4b4000u - (n >> 8);
    uint32_t hi, lo, far;
    asm("shr.u32 %0, %1, %2;" : "=r"(hi) : "r"(w_hi), "r"(shift));          // by 32 and more: 0
    asm("shr.u32 %0, %1, %2;" : "=r"(far) : "r"(w_hi), "r"(shift - 32));
    asm("shf.r.clamp.b32 %0, %1, %2, %3;" : "=r"(lo) : "r"(w_lo), "r"(w_hi), "r"(shift));
    return static_cast<u64>(hi) << 32 | (shift < 32 ? lo : far);
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
template <int kWarps>
__device__ __forceinline__ u64 all_sums(const u64 (&sums)[kWarps]) { return warp_sum((threadIdx.x & 31) < kWarps ? sums[threadIdx.x & 31] : 0); }

// Comparing n <= kThreads entries of a list with one another: a power of two of neighbouring lanes an entry, each of which takes every
// such pair of entries j and j + 1; the list goes on for one that does not count.
template <int kThreads>
struct Pairs {
  int n, parts, entry, part;
  __device__ __forceinline__ explicit Pairs(int entries) : n(entries), parts(1) {
    int shift = 0;
    while (shift < 3 && n << (shift + 1) <= kThreads) ++shift;
    parts = 1 << shift;
    entry = static_cast<int>(threadIdx.x) >> shift;
    part = static_cast<int>(threadIdx.x) & (parts - 1);
  }
  __device__ __forceinline__ bool has() const { return entry < n; }
  __device__ __forceinline__ bool first() const { return part == 0 && entry < n; }       // one thread of each entry
  template <typename F>
  __device__ __forceinline__ void each(F f) const {
    if (!has()) return;
#pragma unroll 2
    for (int j = 2 * part; j < n; j += 2 * parts) f(j);
  }
  // of an entry's lanes; all lanes of the block come here
  template <typename V>
  __device__ __forceinline__ V sum(V v) const {
    for (int o = 1; o < parts; o <<= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
    return v;
  }
};

// Lists the tokens that `takes` holds for, in every block those of all blocks. Returns how many there are; more than kList are not
// kept.
template <typename T, int kThreads, typename P, typename F>
__device__ __forceinline__ unsigned collect(const Row<T, kThreads>& r, P takes, F f) {
  Shared<kThreads>& s = *r.s;
  __syncthreads();
  if (threadIdx.x == 0) s.count = 0;
  __syncthreads();
  r.each_that(takes, [&](uint32_t k, int i) {
    const unsigned at = atomicAdd(&s.count, 1u);
    if (at < kList) s.list[at] = token(k, i);
    f(k);
  });
  r.sync();
  if (r.blocks == 1) return s.count;
  if (threadIdx.x < r.blocks) s.counts[threadIdx.x] = peer32(&s.count, threadIdx.x);
  __syncthreads();
  unsigned all = 0;
  for (int b = 0; b < r.blocks; ++b) all += s.counts[b];
  if (all <= kList) {                      // every block has them all, in the same places
    u64 t = 0;
    if (threadIdx.x < all) {
      unsigned at = threadIdx.x;
      int b = 0;
      for (; at >= s.counts[b]; ++b) at -= s.counts[b];
      t = peer64(&s.list[at], b);
    }
    r.sync();
    if (threadIdx.x < all) s.list[threadIdx.x] = t;
    __syncthreads();
  }
  return all;
}

// Sum over all blocks; s.before: that of the blocks ahead of this one, s.sums: those of its warps.
template <typename T, int kThreads>
__device__ __forceinline__ u64 row_sum(const Row<T, kThreads>& r, u64 own) {
  Shared<kThreads>& s = *r.s;
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
template <typename T, int kThreads>
__device__ __forceinline__ int nth_equal(const Row<T, kThreads>& r, uint32_t key, u64 nth) {
  Shared<kThreads>& s = *r.s;
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  if (threadIdx.x == 0) s.found = ~0ull;
  u64 own = 0;
  r.each([&](uint32_t k, int) { own += k == key; });
  row_sum(r, own);
  const u64 mine = s.sums[warp];
  u64 before = s.before + warp_sum(lane < warp ? s.sums[lane] : 0);
  if (before <= nth && nth < before + mine) {             // it lies in this warp's stretch
    r.steps([&](int v) {
      u64 n = 0;
      if (v < r.to()) r.at(v, [&](uint32_t k, int) { n += k == key; });
      const u64 upto = warp_upto(n);
      u64 at = before + upto - n;
      if (n > 0 && at <= nth && nth < at + n)
        r.at(v, [&](uint32_t k, int i) {
          if (k == key && at++ == nth) s.found = i;
        });
      before += __shfl_sync(0xffffffffu, upto, 31);
    });
  }
  r.sync();
  u64 found = s.found;
  for (int b = 0; b < r.blocks && r.blocks > 1; ++b) found = min(found, peer64(&s.found, b));
  r.sync();
  return found == ~0ull ? 0x7fffffff : static_cast<int>(found);
}

// The last number from a to b for which `holds`, which does so up to some number and not behind it; a where it never does. A warp.
template <typename F>
__device__ __forceinline__ uint32_t last_with(uint32_t a, uint32_t b, F holds, int lane) {
  while (a < b) {
    const uint32_t step = (b - a) / 32 + 1, at = a + min(lane * step, b - a);
    const unsigned yes = __ballot_sync(0xffffffffu, holds(at));
    const uint32_t first = a + (yes ? min((31 - __clz(yes)) * step, b - a) : 0);
    b = first + min(step - 1, b - first);
    if (!yes) b = a;
    a = first;
  }
  return a;
}

// The last token, in descending order through the keys from `high` down to `low`, that has at most so much ahead of it:
// `left` tokens, or (kMass) that fraction of the mass of all. For counts only the key of the result means something.
template <bool kMass, typename T, int kThreads>
__device__ __forceinline__ u64 border(const Row<T, kThreads>& r, uint32_t low, uint32_t high, u64 left) {
  constexpr int kBins = Shared<kThreads>::kBins, kWarps = kThreads / 32;
  Shared<kThreads>& s = *r.s;
  const int tid = threadIdx.x;
  bool first = true;
  while (low < high) {
    // equal steps of the value behind the largest, which has bin 0 to itself: every turn leaves it behind or ends with it
    const float most = Key<T>::value(high);
    const float steps = static_cast<float>((kBins - 2) / (static_cast<double>(most) - static_cast<double>(Key<T>::value(low))));
    // 2^23 + 1 and up: rounded to whole numbers, in the low bits (0 times an infinite number of steps: fminf takes the other)
    auto bin_of = [&](uint32_t k) {
      const float at = fminf((most - Key<T>::value(k)) * steps, kBins - 2.f) + 8388609.f;
      return k == high ? 0 : __float_as_int(at) & (kBins - 1);
    };
    for (int i = tid; i < (kMass ? 2 : 1) * kBins; i += kThreads) (&s.hist[0][0])[i] = 0;
    if (tid == 0) s.bin = -1, s.high = 0, s.low = 0xffffffffu;
    __syncthreads();
    r.each([&](uint32_t k, int) {
      const int b = bin_of(k);
      const u64 m = kMass ? r.mass(k) : 1;
      if (k - low > high - low) return;
      if constexpr (kMass) {
        const unsigned some = static_cast<unsigned>(m);
        const unsigned rest = static_cast<unsigned>(m >> 32) + (atomicAdd(&s.hist[0][b], some) > ~some);
        if (rest > 0) atomicAdd(&s.hist[1][b], rest);
      } else {
        atomicAdd(&s.hist[0][b], 1u);
      }
    });
    r.sync();
    u64 held[2] = {0, 0};
#pragma unroll
    for (int b = 0; b < kMostBlocks; ++b) {
      if (b < r.blocks) {
#pragma unroll
        for (int e = 0; e < (kMass ? 2 : 1); ++e) {
          const u64 two = peer64(&s.hist[e][2 * tid], b);
          held[0] += (two & 0xffffffffu) << 32 * e;
          held[1] += two >> 32 << 32 * e;
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
    // the bin as a range of keys: bins fall as keys rise, so its ends are the last keys above it and up to it
    if (tid < 64) {
      const int least = bin + (tid < 32);                 // warp 0: the last key of a larger bin; warp 1: of this or a larger one
      const uint32_t key = last_with(low, high, [&](uint32_t k) { return bin_of(k) >= least; }, tid & 31);
      if ((tid & 31) == 0) s.ends[tid >> 5] = tid >= 32 ? key : bin_of(low) >= least ? key + 1 : low;
    }
    __syncthreads();
    const uint32_t bottom = s.ends[0], span = s.ends[1] - bottom;
    unsigned hi = 0, lo = 0xffffffffu;
    const unsigned n = collect(r, [&](uint32_t k) { return k - bottom <= span; }, [&](uint32_t k) {
      hi = max(hi, k);
      lo = min(lo, k);
    });
    if (n <= kList) {
      // a warp weighs what lies ahead of one of them; those between the last known to stay and the first known to go are next
      const int lane = tid & 31, warp = tid >> 5;
      const u64 mine = tid < n ? s.list[tid] : 0;
      if (tid < n) s.mass[tid] = kMass ? r.mass(static_cast<uint32_t>(mine >> 32)) : 1;
      if (tid == 0) s.opens = 0;
      u64 found = ~0ull, gone = 0;
      while (true) {
        __syncthreads();
        const unsigned open = __ballot_sync(0xffffffffu, mine > gone && mine < found);
        if (open) {
          unsigned at = 0;
          if (lane == 0) at = atomicAdd(&s.opens, __popc(open));
          at = __shfl_sync(0xffffffffu, at, 0) + __popc(open & ((1u << lane) - 1));
          if ((open >> lane & 1) && at < kWarps) s.open[at] = mine;
        }
        __syncthreads();
        const int total = s.opens, all = min(kWarps, total);
        if (warp < all) {
          const u64 one = s.open[warp];
          u64 ahead = 0;
#pragma unroll 4
          for (int j = lane; j < n; j += 32) ahead += s.list[j] > one ? s.mass[j] : 0;
          ahead = warp_sum(ahead);
          if (lane == 0) s.stays[warp] = ahead <= left;
        }
        __syncthreads();
        if (tid == 0) s.opens = 0;
        const bool known = lane < all, stays = known && s.stays[lane];
        const u64 one = known ? s.open[lane] : 0;
        u64 least = stays ? one : found, most = known && !stays ? one : gone;
#pragma unroll
        for (int o = 16; o > 0; o >>= 1) {
          least = min(least, __shfl_xor_sync(0xffffffffu, least, o));
          most = max(most, __shfl_xor_sync(0xffffffffu, most, o));
        }
        found = least;
        gone = most;
        if (total <= kWarps) return found;
      }
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

// Where the block has few enough tokens from key `from` on, a list of them takes its share's place, in order.
template <typename T, int kThreads>
__device__ __forceinline__ void list_from(Row<T, kThreads>& r, uint32_t from) {
  Shared<kThreads>& s = *r.s;
  constexpr int kWarps = kThreads / 32;
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  int own = 0;
  r.each([&](uint32_t k, int) { own += k >= from; });
  own = __reduce_add_sync(0xffffffffu, own);
  __syncthreads();
  if (lane == 0) s.sums[warp] = own;
  __syncthreads();
  const int other = lane < kWarps ? static_cast<int>(s.sums[lane]) : 0;
  const int all = __reduce_add_sync(0xffffffffu, other);
  int before = __reduce_add_sync(0xffffffffu, lane < warp ? other : 0);
  if (all > kMany) return;
  r.steps([&](int v) {
    int n = 0;
    if (v < r.to()) r.at(v, [&](uint32_t k, int) { n += k >= from; });
    int upto = n;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const int up = __shfl_up_sync(0xffffffffu, upto, o);
      if (lane >= o) upto += up;
    }
    int at = before + upto - n;
    if (n > 0)
      r.at(v, [&](uint32_t k, int i) {
        if (k >= from) s.many[at++] = token(k, i);
      });
    before += __shfl_sync(0xffffffffu, upto, 31);
  });
  r.many = all;
  r.stretch = (all + kWarps - 1) / kWarps;
  __syncthreads();
}

template <typename T, int kThreads>
__global__ void __launch_bounds__(kThreads, 1024 / kThreads) sample_tokens_kernel(const T* logits, long long ld, int V, int blocks, int slice, int stretch, cd_sample p,
                                                                 long long* ids, float* probs) {
  constexpr int kVec = Row<T, kThreads>::kVec, kWarps = kThreads / 32;
  extern __shared__ uint4 s_dyn[];
  Shared<kThreads>& s = *reinterpret_cast<Shared<kThreads>*>(s_dyn);
  uint4* s_data = s_dyn + (sizeof(s) + 15) / 16;
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  if (tid < 256) s.powers[tid] = static_cast<unsigned>(exp2(tid / 256.0 + 31.0) + 0.5);
  if (tid == 0) s.key = 0, s.tau = 0, s.count = 0, s.low = 0xffffffffu;
  __syncthreads();
  griddep_wait();
  griddep_launch_dependents();
  Row<T, kThreads> r;
  r.s = &s;
  r.data = s_data;
  r.blocks = blocks;
  r.rank = blockIdx.x % blocks;
  r.begin = r.rank * slice;
  r.stretch = stretch;
  const int b = blockIdx.x / blocks, length = max(0, min(slice, V - r.begin));
  const T* x = logits + b * ld + r.begin;
  const float temperature = p.temperatures ? p.temperatures[b] : p.temperature;
  const float top_p = p.top_ps ? p.top_ps[b] : p.top_p;
  const float min_p = p.min_ps ? p.min_ps[b] : p.min_p;
  const int top_k = p.top_ks ? p.top_ks[b] : p.top_k;

  // the row's share into shared memory, NaN behind its end
  uint32_t high = 0;
  const bool whole = (reinterpret_cast<uintptr_t>(x) & 15) == 0;
  constexpr int kAhead = 4;                               // loads of a thread under way
  for (int v0 = warp * stretch + lane * kVec; v0 < (warp + 1) * stretch; v0 += kAhead * 32 * kVec) {
    uint4 q[kAhead];
#pragma unroll
    for (int a = 0; a < kAhead; ++a) {
      const int v = v0 + a * 32 * kVec;
      q[a] = make_uint4(0xffffffffu, 0xffffffffu, 0xffffffffu, 0xffffffffu);
      if (v >= (warp + 1) * stretch) continue;
      if (whole && v + kVec <= length) {
        q[a] = *reinterpret_cast<const uint4*>(x + v);
      } else {
        T e[kVec];
#pragma unroll
        for (int i = 0; i < kVec; ++i) e[i] = v + i < length ? x[v + i] : from_f32<T>(__int_as_float(0x7fffffff));
        q[a] = *reinterpret_cast<const uint4*>(e);
      }
    }
#pragma unroll
    for (int a = 0; a < kAhead; ++a) {
      const int v = v0 + a * 32 * kVec;
      if (v >= (warp + 1) * stretch) continue;
      const uint4 k = make_uint4(Key<T>::of(q[a].x), Key<T>::of(q[a].y), Key<T>::of(q[a].z), Key<T>::of(q[a].w));
      high = Key<T>::most(high, Key<T>::most(Key<T>::most(k.x, k.y), Key<T>::most(k.z, k.w)));
      s_data[v / kVec] = k;
    }
  }
  high = Key<T>::largest(high);
  // the largest lane maxima of every warp
  const int warps = min(r.blocks * kWarps, (V + stretch - 1) / stretch);     // that have tokens
  const int draws = (2 * top_k + warps - 1) / warps;
  const bool few = top_k > 0 && top_k < V && top_k <= kFew && draws <= 32 && warps * draws <= kThreads;
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
  if (lane == 0) atomicMax(&s.key, high);
  r.sync();
  uint32_t best = 0;
  for (int c = 0; c < r.blocks; ++c) best = max(best, r.blocks > 1 ? peer32(&s.key, c) : s.key);
  if (few) {                                              // the k-th largest of them
    const int each = min(kWarps, warps) * draws, n = warps * draws;
    if (tid < n) s.all_tops[tid] = r.blocks > 1 ? peer32(&s.tops[tid % each], tid / each) : s.tops[tid];
    if (tid == 0) s.all_tops[n] = 0;
    __syncthreads();
    const Pairs<kThreads> pairs(n);
    const uint32_t mine = pairs.has() ? s.all_tops[pairs.entry] : 0;
    int least = 0, above = 0;                             // at least as large, larger
    pairs.each([&](int j) {
      const uint2 t = *reinterpret_cast<const uint2*>(&s.all_tops[j]);
      least += (t.x >= mine) + (t.y >= mine);
      above += (t.x > mine) + (t.y > mine);
    });
    least = pairs.sum(least);
    above = pairs.sum(above);
    if (pairs.first() && mine > 0 && above < top_k && top_k <= least) s.tau = mine;
  }
  r.sync();
  const uint32_t reach = max(s.tau, Key<T>::kMinusInf + 1);
  r.best = best;
  r.top = Key<T>::value(best);
  const double rate = fmin(369.32993046757462 / static_cast<double>(temperature), 1e38);   // 256 log2 e, and finite: 0 times it is 0
  r.rate = static_cast<float>(rate);
  r.rate_low = static_cast<float>(rate - static_cast<double>(r.rate));

  if (best <= Key<T>::kMinusInf) {                                // nothing to draw from
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
  uint32_t from = Key<T>::kMinusInf + 1;
  bool listed = false;
  unsigned n = 0;
  if (few) {                                              // straight into the first block's list
    const uint32_t count = map_to_cta(smem_u32(&s.count), 0), list = map_to_cta(smem_u32(s.list), 0);
    r.each_that([&](uint32_t k) { return k >= reach; }, [&](uint32_t k, int i) {
      unsigned at;
      asm volatile("atom.shared::cluster.add.u32 %0, [%1], 1;" : "=r"(at) : "r"(count) : "memory");
      if (at < kList) asm volatile("st.shared::cluster.u64 [%0], %1;" ::"r"(list + 8 * at), "l"(token(k, i)) : "memory");
    });
    r.sync();
    n = r.rank == 0 ? s.count : peer32(&s.count, 0);
    listed = n <= kList;
    r.sync();
  }
  if (listed) {
    if (r.rank == 0) {
      const Pairs<kThreads> pairs(n);
      const u64 mine = pairs.has() ? s.list[pairs.entry] : 0;
      const uint32_t key = mine >> 32;
      if (tid == 0) s.list[n] = 0, s.mass[n] = 0, s.kept[n] = 0;           // behind everything
      __syncthreads();
      int greater = 0;
      pairs.each([&](int j) {
        const ulonglong2 t = *reinterpret_cast<const ulonglong2*>(&s.list[j]);
        greater += (static_cast<uint32_t>(t.x >> 32) > key) + (static_cast<uint32_t>(t.y >> 32) > key);
      });
      const u64 w = pairs.sum(greater) < top_k && pairs.has() ? r.mass(key) : 0;
      if (pairs.first()) s.mass[pairs.entry] = w;
      __syncthreads();
      u64 ahead = 0, total = 0;
      pairs.each([&](int j) {
        const ulonglong2 t = *reinterpret_cast<const ulonglong2*>(&s.list[j]), m = *reinterpret_cast<const ulonglong2*>(&s.mass[j]);
        ahead += (t.x > mine ? m.x : 0) + (t.y > mine ? m.y : 0);
        total += m.x + m.y;
      });
      ahead = pairs.sum(ahead);
      total = pairs.sum(total);
      const u64 kept = (top_p < 1.f && ahead > __umul64hi(share, total)) || w < least_mass ? 0 : w;
      if (pairs.first()) s.kept[pairs.entry] = kept;
      __syncthreads();
      // a token's reach in the vocabulary's order
      const uint32_t at = static_cast<uint32_t>(mine);      // ~index
      u64 before = 0, left = 0;
      pairs.each([&](int j) {
        const ulonglong2 t = *reinterpret_cast<const ulonglong2*>(&s.list[j]), m = *reinterpret_cast<const ulonglong2*>(&s.kept[j]);
        before += (static_cast<uint32_t>(t.x) > at ? m.x : 0) + (static_cast<uint32_t>(t.y) > at ? m.y : 0);
        left += m.x + m.y;
      });
      before = pairs.sum(before);
      left = pairs.sum(left);
      const u64 target = __umul64hi(u, left);
      if (pairs.first() && kept > 0 && before <= target && target < before + kept) {
        ids[b] = static_cast<int>(~at);
        probs[b] = static_cast<float>(static_cast<double>(kept) / static_cast<double>(left));
      }
    }
    return;
  }
  if (top_k > 0 && top_k < V) {
    uint32_t least = 0xffffffffu;                         // the smallest value that there is
    r.each([&](uint32_t k, int) { least = min(least, k > Key<T>::kMinusInf ? k : 0xffffffffu); });
    least = __reduce_min_sync(0xffffffffu, least);
    if (lane == 0) atomicMin(&s.low, least);
    r.sync();
    for (int c = 0; c < r.blocks; ++c) least = min(least, r.blocks > 1 ? peer32(&s.low, c) : s.low);
    r.sync();
    from = static_cast<uint32_t>(border<false>(r, least, best, static_cast<u64>(top_k - 1)) >> 32);
    list_from(r, from);
  }
  u64 last = token(from, 0x7fffffff);                     // the last token that stays
  // 45 octaves below the largest there are no masses left
  if (top_p < 1.f) last = border<true>(r, max(from, Key<T>::near(r.top - 32.f * temperature)), best, share);
  if (least_mass > 0) {                                   // min-p as a token: weights rise with the keys
    if (warp == 0) {
      const uint32_t key = last_with(from, best, [&](uint32_t k) { return r.mass(k) < least_mass; }, lane);
      if (lane == 0) s.key = r.mass(from) < least_mass ? key + 1 : from;
    }
    __syncthreads();
    last = max(last, token(s.key, 0x7fffffff));
  }
  const uint32_t last_key = last >> 32;
  const int last_equal = static_cast<int>(~static_cast<uint32_t>(last));
  auto held = [&](uint32_t k, int i) -> u64 {
    const u64 w = r.mass(k);
    return k > last_key || (k == last_key && i <= last_equal) ? w : 0;
  };
  u64 own = 0;
  r.each_that([&](uint32_t k) { return k >= last_key; }, [&](uint32_t k, int i) { own += held(k, i); });
  const u64 total = row_sum(r, own), target = __umul64hi(u, total);
  // the warp's stretch that it falls into, of which every thread of the block then takes a few neighbouring tokens
  const u64 of_warp = lane < kWarps ? s.sums[lane] : 0, upto = s.before + warp_upto(of_warp);
  const unsigned beyond = __ballot_sync(0xffffffffu, upto > target);
  if (s.before > target || beyond == 0) return;           // in another block
  const int pick = __ffs(beyond) - 1;
  const u64 ahead = __shfl_sync(0xffffffffu, upto - of_warp, pick);
  const int first = pick * r.stretch, places = (r.many < 0 ? first + r.stretch : min(r.many, first + r.stretch)) - first;
  const int each = (places + kThreads - 1) / kThreads;
  const int v0 = first + min(places, tid * each), v1 = first + min(places, (tid + 1) * each);
  u64 some = 0;
  for (int v = v0; v < v1; ++v) r.one(v, [&](uint32_t k, int i) { some += held(k, i); });
  u64 at = ahead + block_before(some, s.sums);
  if (at > target || target >= at + some) return;
  for (int v = v0; v < v1; ++v)
    r.one(v, [&](uint32_t k, int i) {
      const u64 e = held(k, i);
      if (at <= target && target < at + e) {
        ids[b] = i;
        probs[b] = static_cast<float>(static_cast<double>(e) / static_cast<double>(total));
      }
      at += e;
    });
}

template <typename T, int kThreads>
cudaError_t launch_blocks(int blocks, const T* logits, long long ld, int B, int V, const cd_sample& p, long long* ids, float* probs,
                          cudaStream_t stream) {
  constexpr auto kKernel = sample_tokens_kernel<T, kThreads>;
  constexpr int kVec = Row<T, kThreads>::kVec, kWarps = kThreads / 32;
  const int least = 32 * kVec;                            // of a warp: 16 bytes a lane
  int stretch = (V + blocks * kWarps - 1) / (blocks * kWarps);
  stretch = stretch < least ? least : (stretch + kVec - 1) / kVec * kVec;
  const int slice = stretch * kWarps, bytes = (sizeof(Shared<kThreads>) + 15) / 16 * 16 + slice * static_cast<int>(sizeof(T));
  const cudaError_t e = allow_smem<kKernel>(bytes);
  if (e != cudaSuccess) return e;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(static_cast<unsigned>(blocks) * B);
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
  return cudaLaunchKernelEx(&cfg, kKernel, logits, ld, V, blocks, slice, stretch, p, ids, probs);
}

// As many blocks a row as its size asks for, and more while there is an SM for each and 4 096 tokens; long shares take 1 024 threads.
// us, 1 / 2 / 4 / 8 blocks: of 512 threads 1 x 32 000 9.3 / 9.4 / 9.0 / 9.5, 32 x 100 000 - / 13.3 / 14.4 / 16.5, nucleus of 64 x 100 000
// - / 73 / 76 / 115, 256 x 32 000 in 32 bits with rules by row 51 / 48 / 67 / 124; of 1 024 threads 10.1 / 10.6 / 10.4 / 11.0,
// - / 14.3 / 12.4 / 32.7, - / 51 / 74 / 160, 46 / 68 / 111 / 259.
template <typename T>
cudaError_t launch_one(const void* logits, long long ld, int B, int V, const cd_sample& p, int64_t* ids, float* probs, cudaStream_t stream) {
  int blocks = 1;
  while (static_cast<long long>(V) * sizeof(T) > static_cast<long long>(blocks) * kSliceBytes) blocks *= 2;
  while (blocks < kMostBlocks && 2LL * blocks * B <= current_sm_count() && V / (2 * blocks) >= 4096) blocks *= 2;
  // 1 024 threads are an SM's: clusters of them that would have to wait for one another are halved, where halves have room for the row. us, 37 x 100 000
  // with a top-k of 50 19 -> 13, its nucleus 65 -> 44, nucleus of 18 x 250 000 116 -> 74.
  while (blocks > 1 && V / blocks > 16384 && B > clusters_side_by_side<sample_tokens_kernel<T, 1024>>(blocks, 1024, 1024) &&
         2 * static_cast<long long>(V) * sizeof(T) <= static_cast<long long>(blocks) * kSliceBytes)
    blocks /= 2;
  const T* x = static_cast<const T*>(logits);
  long long* to = reinterpret_cast<long long*>(ids);
  return V / blocks > 16384 ? launch_blocks<T, 1024>(blocks, x, ld, B, V, p, to, probs, stream)
                            : launch_blocks<T, 512>(blocks, x, ld, B, V, p, to, probs, stream);
}

}  // namespace

cudaError_t launch_sample_tokens(const void* logits, int fp32, long long ld, int B, int V, const cd_sample& p, int64_t* ids, float* probs,
                                 cudaStream_t stream) {
  return fp32 ? launch_one<float>(logits, ld, B, V, p, ids, probs, stream) : launch_one<bf16>(logits, ld, B, V, p, ids, probs, stream);
}

}  // namespace cdeep
