// Sampling from float32 logits [rows, vocab] with temperature, top-k, top-p and min-p and one given random number u in [0, 1) per row.
//
// z_v = logit_v / T. In falling order of z (ties in the order of the vocabulary): K1 the first k; K2 those of K1 whose mass (of exp(z - max)) before them is
// below top_p times K1's; K3 those of K2 with exp(z - max) >= min_p. The token is the first v of K3, in the order of the vocabulary, with
// sum_{K3, w <= v} exp(z_w - max) > u sum_{K3}. T = 0 takes the first of the largest logits. NaN counts as -inf; nothing in -inf's place is ever drawn; a row
// that is nothing else gives token 0. Several +inf share the row. A row whose u is not in [0, 1) (a negative one, NaN) is left as it was.
//
// Masses are integers: exp(z - max) in 64-bit floating point, times 2^bits, rounded to the nearest (bits: as many as leave room for the sum of the whole row, at most
// 45). Sums of integers do not depend on their order, so the same row gives the same token whatever adds it up, and borders fall where 64 bits put them: a
// mass is off by 2^-46 of the likeliest token's at most, and tokens below that have none.
#include "common.cuh"

namespace ms {

__device__ __forceinline__ float clean(float x) { return x == x ? x : -INFINITY; }
// a number's place in the order of floats, larger for larger (-inf: the least)
__device__ __forceinline__ uint32_t order_of(float x) {
  x += 0.f;  // -0 and 0 are one
  const uint32_t u = __float_as_uint(x);
  return (u & 0x80000000u) ? ~u : u | 0x80000000u;
}

struct RowFilter {
  float zmax;      // the largest logit
  double t;
  double unit;     // 2^bits
  double min_p;
  uint32_t key;    // kept: places above `key`, and those at it up to index `last`
  int last;
};

// exp(z - max) of a logit, 0 .. 1
__device__ __forceinline__ double likeness(float x, const RowFilter& f) {
  if (x == f.zmax) return 1.0;
  if (x == -INFINITY) return 0.0;
  return exp(((double)x - (double)f.zmax) / f.t);
}
__device__ __forceinline__ unsigned long long mass_of(float x, const RowFilter& f) { return (unsigned long long)__double2ll_rn(likeness(x, f) * f.unit); }

constexpr int SF_THREADS = 1024;
struct Sums {
  unsigned long long mass;
  int count;
};
__device__ __forceinline__ Sums block_sums(Sums s, Sums* scratch) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) {
    s.mass += __shfl_xor_sync(0xffffffffu, s.mass, o);
    s.count += __shfl_xor_sync(0xffffffffu, s.count, o);
  }
  __syncthreads();
  if ((threadIdx.x & 31) == 0) scratch[threadIdx.x >> 5] = s;
  __syncthreads();
  Sums all{0, 0};
  for (int w = 0; w < SF_THREADS / 32; ++w) {
    all.mass += scratch[w].mass;
    all.count += scratch[w].count;
  }
  return all;
}

// A block per row; every search looks at the whole row again.
__global__ void __launch_bounds__(SF_THREADS)
sample_filtered_kernel(int* __restrict__ tokens, const float* __restrict__ logits, const float* __restrict__ temperature, const void* __restrict__ uniform,
                       const int* __restrict__ top_k, const float* __restrict__ top_p, const float* __restrict__ min_p, int vocab, int bits, int uniform64) {
  __shared__ Sums scratch[SF_THREADS / 32];
  __shared__ unsigned long long before_warp[SF_THREADS / 32 + 1];
  __shared__ int found;
  pdl_prologue(tokens, logits, temperature, uniform, top_k, top_p, min_p);
  const int r = blockIdx.x, lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const double u = uniform64 ? reinterpret_cast<const double*>(uniform)[r] : (double)reinterpret_cast<const float*>(uniform)[r];
  if (!(u >= 0.0 && u < 1.0)) return;
  const float* lg = logits + (size_t)r * vocab;
  const float t = temperature[r];
  RowFilter f;
  // the largest, by its place in the order
  uint32_t best = 0;
  for (int v = threadIdx.x; v < vocab; v += SF_THREADS) best = max(best, order_of(clean(lg[v])));
  best = __reduce_max_sync(0xffffffffu, best);
  __syncthreads();
  if (lane == 0) scratch[warp].count = (int)best;
  if (threadIdx.x == 0) found = 0x7fffffff;
  __syncthreads();
  for (int w = 0; w < SF_THREADS / 32; ++w) best = max(best, (uint32_t)scratch[w].count);
  __syncthreads();
  if (best <= order_of(-INFINITY) || !(t > 0.f)) {
    // nothing but -inf, or the likeliest token: the first at the largest
    for (int v = threadIdx.x; v < vocab; v += SF_THREADS)
      if (order_of(clean(lg[v])) == best) {
        atomicMin(&found, v);
        break;
      }
    __syncthreads();
    if (threadIdx.x == 0) tokens[r] = best <= order_of(-INFINITY) ? 0 : found;
    return;
  }
  f.zmax = __uint_as_float((best & 0x80000000u) ? best & 0x7fffffffu : ~best);
  f.t = (double)t;
  f.unit = (double)(1ull << bits);
  f.key = 0;
  f.last = 0x7fffffff;
  const float mp = min_p ? min_p[r] : 0.f;
  f.min_p = mp > 0.f ? fmin((double)mp, 1.0) : 0.0;
  auto kept_key = [&](uint32_t key, int v) { return key > f.key || (key == f.key && v <= f.last); };
  // The cut of a filter: the largest key at which `enough` holds of the (mass, count) of what is kept and at or above it; of the tokens at the key itself the first `ties(above)`.
  auto cut = [&](auto enough, auto ties) {
    uint32_t lo = 0, hi = best;  // enough(lo) holds
    while (lo < hi) {
      const uint32_t mid = lo + ((hi - lo + 1) >> 1);
      Sums s{0, 0};
      for (int v = threadIdx.x; v < vocab; v += SF_THREADS) {
        const float x = clean(lg[v]);
        const uint32_t key = order_of(x);
        if (key >= mid && kept_key(key, v)) {
          s.mass += mass_of(x, f);
          ++s.count;
        }
      }
      s = block_sums(s, scratch);
      if (enough(s)) lo = mid; else hi = mid - 1;
    }
    Sums above{0, 0};
    for (int v = threadIdx.x; v < vocab; v += SF_THREADS) {
      const float x = clean(lg[v]);
      const uint32_t key = order_of(x);
      if (key > lo && kept_key(key, v)) {
        above.mass += mass_of(x, f);
        ++above.count;
      }
    }
    above = block_sums(above, scratch);
    const float at = __uint_as_float((lo & 0x80000000u) ? lo & 0x7fffffffu : ~lo);
    const long long keep = ties(above, mass_of(at, f));
    // the index of the keep-th token at the key, by bisection over indices
    int first = 0, last = vocab - 1;
    while (first < last) {
      const int mid = (first + last) >> 1;
      Sums s{0, 0};
      for (int v = threadIdx.x; v <= mid; v += SF_THREADS)
        if (order_of(clean(lg[v])) == lo && kept_key(lo, v)) ++s.count;
      s = block_sums(s, scratch);
      if (s.count >= keep) last = mid; else first = mid + 1;
    }
    f.last = (f.key == lo) ? min(f.last, first) : first;
    f.key = lo;
  };
  const int k = top_k ? top_k[r] : 0;
  if (k > 0 && k < vocab) cut([&](const Sums& s) { return s.count >= k; }, [&](const Sums& above, unsigned long long) { return (long long)k - above.count; });
  const float p = top_p ? top_p[r] : 1.f;
  auto total = [&]() {
    Sums s{0, 0};
    for (int v = threadIdx.x; v < vocab; v += SF_THREADS) {
      const float x = clean(lg[v]);
      if (kept_key(order_of(x), v)) {
        const double like = likeness(x, f);
        if (like >= f.min_p) s.mass += (unsigned long long)__double2ll_rn(like * f.unit);
      }
    }
    return block_sums(s, scratch).mass;
  };
  if (p < 1.f) {
    const double held = f.min_p;
    f.min_p = 0.0;
    // kept while the mass before is below the target, the likeliest in any case
    const double target = fmax((double)p * (double)total(), 0.5);
    f.min_p = held;
    cut([&](const Sums& s) { return (double)s.mass >= target; },
        [&](const Sums& above, unsigned long long each) {
          const double n = ceil((target - (double)above.mass) / (double)each);
          return n < 2147483647.0 ? (long long)n : 2147483647ll;
        });
  }
  const unsigned long long all = total();
  unsigned long long target = (unsigned long long)(u * (double)all);
  if (target >= all) target = all - 1;
  // the token whose mass takes the sum beyond the target: a stretch of the row a warp
  const int per_warp = (vocab + SF_THREADS - 1) / SF_THREADS * 32, begin = min(vocab, warp * per_warp), end = min(vocab, begin + per_warp);
  auto kept_mass = [&](int v) -> unsigned long long {
    if (v >= end) return 0;
    const float x = clean(lg[v]);
    if (!kept_key(order_of(x), v)) return 0;
    const double like = likeness(x, f);
    return like >= f.min_p ? (unsigned long long)__double2ll_rn(like * f.unit) : 0;
  };
  unsigned long long mine = 0;
  for (int v = begin + lane; v < end; v += 32) mine += kept_mass(v);
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) mine += __shfl_xor_sync(0xffffffffu, mine, o);
  if (lane == 0) before_warp[warp + 1] = mine;
  __syncthreads();
  if (threadIdx.x == 0) {
    before_warp[0] = 0;
    for (int w = 0; w < SF_THREADS / 32; ++w) before_warp[w + 1] += before_warp[w];
  }
  __syncthreads();
  if (before_warp[warp] <= target && target < before_warp[warp + 1]) {
    unsigned long long before = before_warp[warp];
    for (int v0 = begin; v0 < end; v0 += 32) {
      unsigned long long sum = kept_mass(v0 + lane);
#pragma unroll
      for (int o = 1; o < 32; o <<= 1) {
        const unsigned long long other = __shfl_up_sync(0xffffffffu, sum, o);
        if (lane >= o) sum += other;
      }
      const unsigned hit = __ballot_sync(0xffffffffu, before + sum > target);
      if (hit) {
        if (lane == 0) tokens[r] = v0 + __ffs(hit) - 1;
        break;
      }
      before += __shfl_sync(0xffffffffu, sum, 31);
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
  MS_CHECK_ARG(rows >= 0 && vocab > 0, "sample_filtered: bad sizes rows=%d vocab=%d", rows, vocab);
  MS_CHECK_ARG(tokens && logits && temperature && uniform, "sample_filtered: null pointer");
  if (rows == 0) return 0;
  int bits = 62;  // a row's sum stays within 2^62
  while ((1ll << (62 - bits)) < vocab) --bits;
  if (bits > 45) bits = 45;
  MS_LAUNCH(sample_filtered_kernel, rows, SF_THREADS, 0, stream, tokens, logits, temperature, uniform, top_k, top_p, min_p, vocab, bits, uniform64);
  return 0;
}
