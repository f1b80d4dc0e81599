// Sampling from float32 logits [rows, vocab] with temperature, top-k, top-p and min-p and one given random number u in [0, 1) per row.
//
// z_v = logit_v / T. In falling order of z (ties in the order of the vocabulary): K1 the first k; K2 those of K1 whose mass (of exp(z - max)) before them is
// below top_p times K1's; K3 those of K2 with exp(z - max) >= min_p. The token is the first v of K3, in the order of the vocabulary, with
// sum_{K3, w <= v} exp(z_w - max) > u sum_{K3}. T = 0 takes the first of the largest logits. NaN counts as -inf; nothing in -inf's place is ever drawn; a row
// that is nothing else gives token 0. Several +inf share the row. A row whose u is not in [0, 1) (a negative one, NaN) is left as it was.
//
// Masses are integers: exp(z - max) in 64-bit floating point, times 2^bits, rounded to the nearest (bits: as many as leave room for the sum of the whole row, at most
// 45). Sums of integers do not depend on their order, so the same row gives the same token whatever adds it up, and borders fall where 64 bits put them: a
// mass is off by 2^-(bits + 1) of the likeliest token's at most (2^-46 up to 131,072 tokens, 2^-45 for 151,936, 2^-43 for 2^20), and tokens below that have none.
#include <cfloat>

#include <cooperative_groups.h>

#include "common.cuh"

namespace ms {

__device__ __forceinline__ float clean(float x) { return x == x ? x : -INFINITY; }
// a number's place in the order of floats, larger for larger (-inf: the least)
__device__ __forceinline__ uint32_t order_of(float x) {
  x += 0.f;  // -0 and 0 are one
  const uint32_t u = __float_as_uint(x);
  return (u & 0x80000000u) ? ~u : u | 0x80000000u;
}

typedef unsigned long long u64;
namespace cg = cooperative_groups;

// A token's place in a row: its logit's, then (of equals) the earlier one first. Larger is likelier, and no two are the same.
constexpr int INDEX_BITS = 20;
__device__ __forceinline__ u64 place_of(float x, int v) { return ((u64)order_of(x) << INDEX_BITS) | (u64)((1 << INDEX_BITS) - 1 - v); }
__device__ __forceinline__ int index_of(u64 place) { return (1 << INDEX_BITS) - 1 - (int)(place & ((1 << INDEX_BITS) - 1)); }
__device__ __forceinline__ float logit_of(u64 place) {
  const uint32_t key = (uint32_t)(place >> INDEX_BITS);
  return __uint_as_float((key & 0x80000000u) ? key & 0x7fffffffu : ~key);
}

// What makes a mass of a logit.
constexpr int STEPS = 64;  // of 2^x between two powers of two
struct Scale {
  float zmax;            // the row's largest logit
  float least;           // logits below round to no mass (-inf among them)
  double ref;            // zmax, or 0 where that is infinite (then it alone has a mass)
  double per;            // steps a unit of logit: STEPS log2(e) / T
  int bits;
  const double* powers;  // 2^(i / STEPS)
};
// exp(z - max) 2^bits, not rounded: a power of two, a step of the table, and the exponential series of what is left (half a step at most, so five terms are good to
// 2^-54). Rounding to whole numbers is adding a number whose last place is one. Eleven operations of 64 bits and no conversions but x's, where exp() behind a
// division takes several times that (masses were half of the kernel's time); no branches, so that several tokens' chains run beside each other.
__device__ __forceinline__ double weight_of(float x, const Scale& f) {
  constexpr double ROUND = 6755399441055744.0, L = 0.69314718055994530942 / STEPS;  // 1.5 * 2^52; ln 2 / STEPS
  const double d = x == f.zmax ? 0.0 : (double)fmaxf(x, f.least) - f.ref;
  const double shifted = fma(d, f.per, ROUND), r = fma(d, f.per, ROUND - shifted);
  const int n = __double2loint(shifted);  // steps: 0 or below
  double p = fma(r, L * L * L * L * L / 120, L * L * L * L / 24);
  p = fma(r, p, L * L * L / 6);
  p = fma(r, p, L * L / 2);
  p = fma(r, p, L);
  p = fma(r, p, 1.0);
  const double m = f.powers[n & (STEPS - 1)] * p;
  const double w = __hiloint2double(__double2hiint(m) + (((n >> 6) + f.bits) << 20), __double2loint(m));  // (2^-4 at the least: a normal number)
  return x >= f.least ? w : 0.0;
}
static_assert(STEPS == 1 << 6, "the step's index");
// the nearest whole number, below 2^51
__device__ __forceinline__ u64 to_mass(double w) {
  constexpr double ONES = 4503599627370496.0;  // 2^52
  return (u64)(__double_as_longlong(w + ONES) - __double_as_longlong(ONES));
}

// A row belongs to a cluster of CTAs, each of which keeps its stretch of the logits in shared memory. A filter's cut is a place, found by a histogram over the fall below the
// largest logit (BINS bins up to where masses end), then the places of the one bin that the cut falls into, sorted. top-k alone, or ahead of the
// other filters, leaves a short list, on which one CTA does all that is left. Everything that is added up is whole numbers.
constexpr int SF_THREADS = 512, SF_WARPS = SF_THREADS / 32, SF_CTAS = 16, BINS = 1024, LIST = 1024, LIMB = 15;

struct SfShared {
  u64 xchg[2][SF_CTAS][2];  // two numbers of every CTA of the cluster, two turns
  u64 red[SF_WARPS][2];
  u64 said[4];              // what one CTA tells all
  union {
    u64 list[LIST];               // (the first CTA's) places of one bin, or of all that is left
    uint32_t merged_count[BINS];  // counts of this CTA's share of the bins, over the cluster
  };
  union {
    u64 sums[LIST];
    u64 merged[BINS];  // their masses
  };
  uint32_t count[BINS], limb[3][BINS];
  double powers[STEPS];
  int listed;
};

struct Cluster {
  cg::cluster_group group;
  SfShared& sh;
  int rank, ctas, turn;

  // a and b added up (or the largest taken) over all threads of all CTAs; the same in every thread
  template <bool MAX>
  __device__ __forceinline__ void reduce(u64& a, u64& b) {
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    auto join = [](u64 x, u64 y) { return MAX ? (x > y ? x : y) : x + y; };
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) {
      a = join(a, __shfl_xor_sync(0xffffffffu, a, o));
      b = join(b, __shfl_xor_sync(0xffffffffu, b, o));
    }
    if (lane == 0) {
      sh.red[warp][0] = a;
      sh.red[warp][1] = b;
    }
    __syncthreads();
    if (warp == 0) {
      a = lane < SF_WARPS ? sh.red[lane][0] : 0;
      b = lane < SF_WARPS ? sh.red[lane][1] : 0;
#pragma unroll
      for (int o = 16; o > 0; o >>= 1) {
        a = join(a, __shfl_xor_sync(0xffffffffu, a, o));
        b = join(b, __shfl_xor_sync(0xffffffffu, b, o));
      }
      if (lane < ctas) {
        u64* to = group.map_shared_rank(&sh.xchg[turn][rank][0], lane);
        to[0] = a;
        to[1] = b;
      }
    }
    group.sync();
    a = sh.xchg[turn][0][0];
    b = sh.xchg[turn][0][1];
    for (int c = 1; c < ctas; ++c) {
      a = join(a, sh.xchg[turn][c][0]);
      b = join(b, sh.xchg[turn][c][1]);
    }
    turn ^= 1;
  }
  // `said` of the CTA that has something to say (its first thread, before), in all of them
  __device__ __forceinline__ void tell(const u64 (&what)[4]) {
    for (int c = 0; c < ctas; ++c) {
      u64* to = group.map_shared_rank(&sh.said[0], c);
#pragma unroll
      for (int i = 0; i < 4; ++i) to[i] = what[i];
    }
  }
};

// list[0 .. n) sorted, the largest first; n <= LIST. Up to a number a thread: partners of the same warp by shuffles, others through the list.
__device__ __forceinline__ void sort_list(u64* list, int n) {
  int size = 32;
  while (size < n) size <<= 1;
  const int tid = threadIdx.x;
  __syncthreads();
  if (size <= SF_THREADS) {
    u64 v = tid < n ? list[tid] : 0;
    if (size == 32 && tid >= 32) v = 0;
    for (int k = 2; k <= size; k <<= 1)
      for (int j = k >> 1; j > 0; j >>= 1) {
        u64 other;
        if (j >= 32) {
          if (tid < size) list[tid] = v;
          __syncthreads();
          other = tid < size ? list[tid ^ j] : 0;
          __syncthreads();
        } else {
          other = __shfl_xor_sync(0xffffffffu, v, j);
        }
        v = (((tid & k) == 0) == ((tid & j) == 0)) == (v > other) ? v : other;
      }
    if (tid < size) list[tid] = v;
    __syncthreads();
    return;
  }
  for (int i = n + tid; i < size; i += SF_THREADS) list[i] = 0;
  __syncthreads();
  for (int k = 2; k <= size; k <<= 1)
    for (int j = k >> 1; j > 0; j >>= 1) {
      const int p = tid;
      if (p < size / 2) {
        const int i = 2 * p - (p & (j - 1)), other = i + j;
        const u64 x = list[i], y = list[other];
        if (((i & k) == 0) ? x < y : x > y) {
          list[i] = y;
          list[other] = x;
        }
      }
      __syncthreads();
    }
}
// the sums up to and with each of the n numbers in `sums` (n <= 2 SF_THREADS); returns nothing, all threads call it
__device__ __forceinline__ void running_sums(u64* sums, int n, u64 (&red)[SF_WARPS][2]) {
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, i = 2 * threadIdx.x;
  u64 a = i < n ? sums[i] : 0, b = i + 1 < n ? sums[i + 1] : 0, s = a + b;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const u64 x = __shfl_up_sync(0xffffffffu, s, o);
    if (lane >= o) s += x;
  }
  __syncthreads();
  if (lane == 31) red[warp][0] = s;
  __syncthreads();
  u64 before = s - a - b;
  for (int w = 0; w < warp; ++w) before += red[w][0];
  if (i < n) sums[i] = before + a;
  if (i + 1 < n) sums[i + 1] = before + a + b;
  __syncthreads();
}

__global__ void __launch_bounds__(SF_THREADS)
sample_filtered_kernel(int* __restrict__ tokens, const float* __restrict__ logits, const float* __restrict__ temperature, const void* __restrict__ uniform,
                       const int* __restrict__ top_k, const float* __restrict__ top_p, const float* __restrict__ min_p, int vocab, int slice, int staged, int bits,
                       int uniform64) {
  extern __shared__ __align__(16) float sf_logits[];
  __shared__ SfShared sh;
  cg::cluster_group group = cg::this_cluster();
  Cluster cl{group, sh, (int)group.block_rank(), (int)group.num_blocks(), 0};
  pdl_prologue(tokens, logits, temperature, uniform, top_k, top_p, min_p);
  const int ctas = cl.ctas, rank = cl.rank, r = blockIdx.x / ctas, tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const double u = uniform64 ? reinterpret_cast<const double*>(uniform)[r] : (double)reinterpret_cast<const float*>(uniform)[r];
  if (!(u >= 0.0 && u < 1.0)) return;  // (the whole cluster)
  cluster_started_arrive();
  const float t = temperature[r];
  const int k = top_k ? top_k[r] : 0;
  const float p = top_p ? top_p[r] : 1.f, mp = min_p ? min_p[r] : 0.f;
  const double least = mp > 0.f ? fmin((double)mp, 1.0) * (double)(1ull << bits) : 0.0;
  const int begin = min(rank * slice, vocab), n = min(slice, vocab - begin);
  const float* xs = logits + (size_t)r * vocab + begin;

  // the largest logit and the least finite one (NaN is neither)
  float top = -INFINITY, low = INFINITY;
  auto meet = [&](float x) {
    top = fmaxf(top, x);
    low = fminf(low, x > -INFINITY ? x : INFINITY);
    return clean(x);
  };
  if (tid < STEPS) sh.powers[tid] = exp2((double)tid / STEPS);
  if (staged && (reinterpret_cast<uintptr_t>(xs) & 15) == 0) {
    constexpr int AHEAD = 5;
    for (int i0 = 4 * tid; i0 + 3 < n; i0 += 4 * SF_THREADS * AHEAD) {
      float4 x[AHEAD];
#pragma unroll
      for (int q = 0; q < AHEAD; ++q) {
        const int i = i0 + q * 4 * SF_THREADS;
        if (i + 3 < n) x[q] = behind_loadf4(xs + i);
      }
#pragma unroll
      for (int q = 0; q < AHEAD; ++q) {
        const int i = i0 + q * 4 * SF_THREADS;
        if (i + 3 < n) *reinterpret_cast<float4*>(sf_logits + i) = make_float4(meet(x[q].x), meet(x[q].y), meet(x[q].z), meet(x[q].w));
      }
    }
    for (int i = (n & ~3) + tid; i < n; i += SF_THREADS) sf_logits[i] = meet(xs[i]);
  } else {
    for (int i = tid; i < n; i += SF_THREADS) {
      const float x = meet(xs[i]);
      if (staged) sf_logits[i] = x;
    }
  }
  for (int i = tid; i < BINS; i += SF_THREADS) sh.count[i] = sh.limb[0][i] = sh.limb[1][i] = sh.limb[2][i] = 0;
  if (tid == 0) sh.listed = 0;
  u64 best = order_of(top), lowest = low < INFINITY ? (u64)~order_of(low) : 0;
  cluster_started_wait();
  cl.reduce<true>(best, lowest);
  const float zmax = logit_of(best << INDEX_BITS);
  const float* mine = staged ? sf_logits : xs;
  if (!(t > 0.f) || zmax == -INFINITY) {
    // the first of the largest (of nothing but -inf: 0)
    u64 first = 0, none = 0;
    if (zmax > -INFINITY)
      for (int i = tid; i < n; i += SF_THREADS)
        if (mine[i] == zmax) {
          first = (u64)(vocab - begin - i);
          break;
        }
    cl.reduce<true>(first, none);
    if (rank == 0 && tid == 0) tokens[r] = zmax == -INFINITY ? 0 : vocab - (int)first;
    return;
  }
  const double steps = STEPS * 1.4426950408889634074 / (double)t;
  // the least logit that is not below 2^-3 of a mass (rounded up, so that no logit from it on is either)
  const float from = zmax < INFINITY ? __double2float_ru((double)zmax - (double)(bits + 3) * STEPS / steps) : INFINITY;
  const Scale f{zmax, fmaxf(from, -FLT_MAX), zmax < INFINITY ? (double)zmax : 0.0, steps, bits, sh.powers};
  // Bins by the fall below the largest: up to the least finite logit, and no further than masses go (2^-46, the least there is, is 31.9 falls of T).
  const float floor_ = logit_of(((u64)~(uint32_t)lowest) << INDEX_BITS);
  const float width = fminf((float)BINS / fmaxf(fminf(zmax - floor_, 32.f * t), 1e-35f), 1e37f);
  auto bin_of = [&](float x) { return x == zmax ? 0 : (int)fminf((zmax - x) * width, (float)(BINS - 1)); };

  u64 cut = 0;  // kept: places from here on
  auto at = [&](int i) { return staged ? sf_logits[i] : clean(xs[i]); };
  auto counted = [&](float x, int v) { return x > -INFINITY && (cut == 0 || place_of(x, v) >= cut); };
  // f(i, x) of the CTA's tokens i of [from, to), `step` threads side by side, four of a thread's at a time
  auto each = [&](int from, int to, int step, auto f4) {
    for (int i0 = from; i0 < to; i0 += 4 * step) {
      float x[4];
      bool in[4];
#pragma unroll
      for (int q = 0; q < 4; ++q) {
        in[q] = i0 + q * step < to;
        x[q] = in[q] ? at(i0 + q * step) : -INFINITY;
      }
      f4(i0, x, in);
    }
  };
  // the places of the counted tokens of bins [low, high] in the first CTA's list
  auto gather = [&](int low, int high) {
    SfShared* first = group.map_shared_rank(&sh, 0);
    each(tid, n, SF_THREADS, [&](int i0, const float (&x)[4], const bool (&in)[4]) {
#pragma unroll
      for (int q = 0; q < 4; ++q) {
        const int bin = bin_of(x[q]), v = begin + i0 + q * SF_THREADS;
        if (bin < low || bin > high || !in[q] || !counted(x[q], v)) continue;
        const int slot = atomicAdd(&first->listed, 1);
        if (slot < LIST) first->list[slot] = place_of(x[q], v);
      }
    });
  };
  // Where the running sum over the bins, likeliest first, is `enough` for the first time: said[0] the bin, [1] the count and [2] the mass before it, [3] its count.
  auto crossing = [&](auto enough, bool masses) {
    const int per = BINS / ctas;
    u64 count = 0, mass = 0;
    // lanes side by side have a bin, and half of the cluster's CTAs each
    for (int i0 = 0; i0 < per; i0 += SF_THREADS / 2) {
      const int i = i0 + tid / 2;
      u64 c = 0, m = 0;
      if (i < per) {
        const int bin = rank * per + i;
#pragma unroll
        for (int q = 0; q < SF_CTAS / 2; ++q) {
          if (2 * q + (tid & 1) >= ctas) break;
          const SfShared* other = group.map_shared_rank(&sh, 2 * q + (tid & 1));
          c += other->count[bin];
          if (masses) m += (u64)other->limb[0][bin] + ((u64)other->limb[1][bin] << LIMB) + ((u64)other->limb[2][bin] << (2 * LIMB));
        }
      }
      count += c;
      mass += m;
      c += __shfl_xor_sync(0xffffffffu, c, 1);
      m += __shfl_xor_sync(0xffffffffu, m, 1);
      if (i < per && (tid & 1) == 0) {
        sh.merged_count[i] = (uint32_t)c;
        sh.merged[i] = m;
      }
    }
    const int turn = cl.turn;
    cl.reduce<false>(count, mass);  // (every CTA's sums are in xchg[turn]; the totals in count and mass)
    u64 cb = 0, mb = 0;
    for (int q = 0; q < rank; ++q) {
      cb += sh.xchg[turn][q][0];
      mb += sh.xchg[turn][q][1];
    }
    if (warp == 0 && !(rank > 0 && enough(cb, mb, count, mass)) && (enough(cb + sh.xchg[turn][rank][0], mb + sh.xchg[turn][rank][1], count, mass) || rank == ctas - 1)) {
      // this CTA's: lanes take runs of its bins
      const int each = per / 32;
      u64 c = 0, m = 0;
      for (int i = 0; i < each; ++i) {
        c += sh.merged_count[lane * each + i];
        m += sh.merged[lane * each + i];
      }
      u64 ci = c, mi = m;
#pragma unroll
      for (int o = 1; o < 32; o <<= 1) {
        const u64 x = __shfl_up_sync(0xffffffffu, ci, o), y = __shfl_up_sync(0xffffffffu, mi, o);
        if (lane >= o) {
          ci += x;
          mi += y;
        }
      }
      const unsigned hit = __ballot_sync(0xffffffffu, enough(cb + ci, mb + mi, count, mass));
      if (lane == (hit ? __ffs(hit) - 1 : 31)) {
        u64 c1 = cb + ci - c, m1 = mb + mi - m;
        int i = 0;
        for (; i + 1 < each; ++i) {
          const u64 c2 = c1 + sh.merged_count[lane * each + i], m2 = m1 + sh.merged[lane * each + i];
          if (enough(c2, m2, count, mass)) break;
          c1 = c2;
          m1 = m2;
        }
        const u64 what[4] = {(u64)(rank * per + lane * each + i), c1, m1, sh.merged_count[lane * each + i]};
        cl.tell(what);
      }
    }
    group.sync();
    return mass;
  };
  // The cut itself, the place at which `enough` comes true, within bin said[0]: by its places sorted in the first CTA; of more than those hold, by halving the range, a pass
  // and a meeting for each of some 40 bits (by top-p of 151,936 tokens, us, one row and 8: logits that are whole numbers 145 and 219; one token far below the rest, which makes the bins wide, 190 and 307; else 33 and 43).
  auto settle = [&](auto enough, u64 all_count, u64 all_mass) {
    const int bin = (int)sh.said[0];
    const u64 cb = sh.said[1], mb = sh.said[2], members = sh.said[3];
    if (members == 0) return;  // (fewer tokens than top-k would keep)
    if (members <= LIST) {
      gather(bin, bin);
      group.sync();
      if (rank == 0) {
        const int have = min(sh.listed, LIST);
        sort_list(sh.list, have);
        for (int i = tid; i < have; i += SF_THREADS) sh.sums[i] = to_mass(weight_of(logit_of(sh.list[i]), f));
        __syncthreads();
        running_sums(sh.sums, have, sh.red);
        for (int i = tid; i < have; i += SF_THREADS) {
          const bool now = enough(cb + i + 1, mb + sh.sums[i], all_count, all_mass);
          const bool then = i > 0 && enough(cb + i, mb + sh.sums[i - 1], all_count, all_mass);
          if ((now && !then) || (i == have - 1 && !now)) {
            const u64 what[4] = {sh.list[i], 0, 0, 0};
            cl.tell(what);
          }
        }
        __syncthreads();
        if (tid == 0) sh.listed = 0;
      }
      group.sync();
      cut = sh.said[0];
    } else {
      u64 hi = 0, lo = 0;  // the bin's largest place, and its smallest
      for (int i = tid; i < n; i += SF_THREADS) {
        const float x = at(i);
        if (bin_of(x) != bin || !counted(x, begin + i)) continue;
        const u64 place = place_of(x, begin + i);
        hi = place > hi ? place : hi;
        lo = ~place > lo ? ~place : lo;
      }
      cl.reduce<true>(hi, lo);
      lo = ~lo;
      while (lo < hi) {  // the largest place that is enough
        const u64 mid = lo + ((hi - lo + 1) >> 1);
        u64 count = 0, mass = 0;
        for (int i = tid; i < n; i += SF_THREADS) {
          const float x = at(i);
          const u64 place = place_of(x, begin + i);
          if (place < mid || bin_of(x) != bin || !counted(x, begin + i)) continue;
          ++count;
          mass += to_mass(weight_of(x, f));
        }
        cl.reduce<false>(count, mass);
        if (enough(cb + count, mb + mass, all_count, all_mass)) lo = mid; else hi = mid - 1;
      }
      cut = lo;
    }
  };
  auto histogram = [&](bool masses) {
    each(tid, n, SF_THREADS, [&](int i0, const float (&x)[4], const bool (&in)[4]) {
      u64 m[4];
#pragma unroll
      for (int q = 0; q < 4; ++q) m[q] = masses ? to_mass(weight_of(x[q], f)) : 0;
#pragma unroll
      for (int q = 0; q < 4; ++q) {
        if (!in[q] || !counted(x[q], begin + i0 + q * SF_THREADS)) continue;
        const int bin = bin_of(x[q]);
        atomicAdd(&sh.count[bin], 1u);
        if (masses) {
          atomicAdd(&sh.limb[0][bin], (uint32_t)m[q] & ((1u << LIMB) - 1));
          atomicAdd(&sh.limb[1][bin], (uint32_t)(m[q] >> LIMB) & ((1u << LIMB) - 1));
          atomicAdd(&sh.limb[2][bin], (uint32_t)(m[q] >> (2 * LIMB)));
        }
      }
    });
    group.sync();
  };

  if (k > 0 && k < vocab) {
    histogram(false);
    auto enough = [k](u64 count, u64, u64, u64) { return count >= (u64)k; };
    crossing(enough, false);
    const u64 listed = sh.said[1] + sh.said[3];
    if (listed <= LIST) {
      // all that top-k can leave is a short list: the first CTA finishes the row
      gather(0, (int)sh.said[0]);
      group.sync();
      if (rank) return;
      const int have = min(sh.listed, LIST), kept_k = min(have, k);
      sort_list(sh.list, have);
      for (int i = tid; i < kept_k; i += SF_THREADS) sh.sums[i] = to_mass(weight_of(logit_of(sh.list[i]), f));
      __syncthreads();
      running_sums(sh.sums, kept_k, sh.red);
      // what is kept is a run from the likeliest on
      const double target = p < 1.f ? fmax((double)p * (double)sh.sums[kept_k - 1], 0.5) : INFINITY;
      int kept = 0;
      for (int i = tid; i < kept_k; i += SF_THREADS)
        if ((i == 0 || (double)sh.sums[i - 1] < target) && weight_of(logit_of(sh.list[i]), f) >= least) ++kept;
      kept = __reduce_add_sync(0xffffffffu, kept);
      __syncthreads();
      if (lane == 0) sh.red[warp][0] = kept;
      __syncthreads();
      kept = 0;
      for (int w = 0; w < SF_WARPS; ++w) kept += (int)sh.red[w][0];
      const u64 all = sh.sums[kept - 1];
      u64 aim = (u64)(u * (double)all);
      if (aim >= all) aim = all - 1;
      // in the order of the vocabulary: places by what they have of the index, which falls with it
      u64 held[LIST / SF_THREADS];
#pragma unroll
      for (int q = 0; q < LIST / SF_THREADS; ++q) {
        const int i = tid + q * SF_THREADS;
        if (i < kept) held[q] = sh.list[i];
      }
      __syncthreads();
#pragma unroll
      for (int q = 0; q < LIST / SF_THREADS; ++q) {
        const int i = tid + q * SF_THREADS;
        if (i < kept) sh.list[i] = (held[q] << 44) | (held[q] >> INDEX_BITS);  // the index in front, its complement: earlier tokens are larger
      }
      __syncthreads();
      sort_list(sh.list, kept);
      for (int i = tid; i < kept; i += SF_THREADS) sh.sums[i] = to_mass(weight_of(logit_of((sh.list[i] & 0xffffffffull) << INDEX_BITS), f));
      __syncthreads();
      running_sums(sh.sums, kept, sh.red);
      for (int i = tid; i < kept; i += SF_THREADS)
        if (sh.sums[i] > aim && (i == 0 || sh.sums[i - 1] <= aim)) tokens[r] = (1 << INDEX_BITS) - 1 - (int)(sh.list[i] >> 44);
      return;
    }
    settle(enough, 0, 0);
    for (int i = tid; i < BINS; i += SF_THREADS) sh.count[i] = 0;
    __syncthreads();
  }
  if (p < 1.f) {
    histogram(true);
    const double part = (double)p;
    auto enough = [part](u64, u64 mass, u64, u64 all) { return (double)mass >= fmax(part * (double)all, 0.5); };
    const u64 all = crossing(enough, true);
    settle(enough, 0, all);
  }
  // the token whose mass takes the sum beyond u of all: a stretch of the CTA's tokens a warp
  const int per_warp = ((n + SF_WARPS - 1) / SF_WARPS + 31) / 32 * 32, wb = min(warp * per_warp, n), we = min(wb + per_warp, n);
  const float edge = cut ? logit_of(cut) : -INFINITY;  // the cut's logit
  auto mass_of = [&](float x, int i) -> u64 {
    const double w = weight_of(x, f);
    return w >= least && (x > edge || (x == edge && place_of(x, begin + i) >= cut)) ? to_mass(w) : 0;
  };
  u64 sum = 0, none = 0;
  each(wb + lane, we, 32, [&](int i0, const float (&x)[4], const bool (&in)[4]) {
    u64 m[4];
    // (a warp whose tokens are all below the cut has nothing to work out: all but a few of them where a row has a few likely tokens)
    if (!__any_sync(__activemask(), fmaxf(fmaxf(x[0], x[1]), fmaxf(x[2], x[3])) >= edge)) return;
#pragma unroll
    for (int q = 0; q < 4; ++q) m[q] = mass_of(x[q], i0 + 32 * q);
#pragma unroll
    for (int q = 0; q < 4; ++q) sum += in[q] ? m[q] : 0;
  });
  const int turn = cl.turn;
  cl.reduce<false>(sum, none);  // (a warp's sums are left in red)
  u64 aim = (u64)(u * (double)sum);
  if (aim >= sum) aim = sum - 1;
  u64 before = 0;
  for (int q = 0; q < rank; ++q) before += sh.xchg[turn][q][0];
  for (int w = 0; w < warp; ++w) before += sh.red[w][0];
  if (before <= aim && aim < before + sh.red[warp][0]) {
    for (int i0 = wb; i0 < we; i0 += 32) {
      u64 s = i0 + lane < we ? mass_of(at(i0 + lane), i0 + lane) : 0;
#pragma unroll
      for (int o = 1; o < 32; o <<= 1) {
        const u64 x = __shfl_up_sync(0xffffffffu, s, o);
        if (lane >= o) s += x;
      }
      const unsigned hit = __ballot_sync(0xffffffffu, before + s > aim);
      if (hit) {
        if (lane == 0) tokens[r] = begin + i0 + __ffs(hit) - 1;
        break;
      }
      before += __shfl_sync(0xffffffffu, s, 31);
    }
  }
}

}  // namespace ms

using namespace ms;

MS_DEFINE_LAST_ERROR(ms_filters_last_error)
MS_DEFINE_PDL_SWITCH(ms_filters_set_pdl)

// top_k, top_p, min_p: a number per row, or null. uniform: float64 (uniform64 = 1) or float32.
MS_EXPORT int ms_sample_filtered(int* tokens, const float* logits, const float* temperature, const void* uniform, const int* top_k, const float* top_p,
                                 const float* min_p, int rows, int vocab, int uniform64, cudaStream_t stream) {
  MS_CHECK_ARG(rows >= 0 && vocab > 0 && vocab <= (1 << INDEX_BITS), "sample_filtered: bad sizes rows=%d vocab=%d", rows, vocab);
  MS_CHECK_ARG(tokens && logits && temperature && uniform, "sample_filtered: null pointer");
  if (rows == 0) return 0;
  int bits = 62;  // a row's sum stays within 2^62
  while ((1ll << (62 - bits)) < vocab) --bits;
  if (bits > 3 * LIMB) bits = 3 * LIMB;
  // Sixteen CTAs a row while that leaves each an SM of its own, else eight (8 rows of 151,936 tokens by top-p alone 38.9 us, 55.7 with eight; one row by top-k 15.0 and 16.8).
  const int ctas = vocab < 16384 ? 1 : rows * SF_CTAS <= (sm_count() > 0 ? sm_count() : 148) ? SF_CTAS : SF_CTAS / 2, slice = ceil_div(ceil_div(vocab, ctas), 32) * 32;
  MS_CHECK_ARG((long long)rows * ctas <= 0x7fffffffLL, "sample_filtered: %d rows are too many for one launch", rows);
  const size_t smem = (size_t)slice * sizeof(float);
  const int staged = smem <= 160 * 1024;  // (longer rows are read again for each search)
  if (ctas == SF_CTAS) {
    static std::atomic<unsigned long long> wide{0};
    int dev = 0;
    MS_CHECK_CUDA(cudaGetDevice(&dev));
    if (dev >= KNOWN_DEVICES || !((wide.load(std::memory_order_relaxed) >> dev) & 1ull)) {
      MS_CHECK_CUDA(cudaFuncSetAttribute((const void*)sample_filtered_kernel, cudaFuncAttributeNonPortableClusterSizeAllowed, 1));
      if (dev < KNOWN_DEVICES) wide.fetch_or(1ull << dev, std::memory_order_relaxed);
    }
  }
  if (staged) {
    static std::atomic<unsigned long long> allowed{0};
    MS_CHECK_CUDA(allow_shared_memory((const void*)sample_filtered_kernel, 160 * 1024, allowed));
  }
  MS_LAUNCH_CLUSTERED(sample_filtered_kernel, rows * ctas, SF_THREADS, staged ? smem : 0, stream, ctas, tokens, logits, temperature, uniform, top_k, top_p, min_p,
                      vocab, slice, staged, bits, uniform64);
  return 0;
}
