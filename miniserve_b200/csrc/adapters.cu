// Low-rank adapters of many requests at once beside a projection that all requests share:
//   y[t, n] = (W x_t)_n + c_s sum_j B_s[n, j] (A_s x_t)[p(n) r + j],   s = slot_of_row[row_of_token[t]],
// r numbers for each part p of the stacked output (q|k|v, gate|up), B's row n with the numbers of its part. A slot below 0: no adapter.
// The shared product is the package's own (ops.linear); here are v = c_s A_s x_t (float32, the scale inside) and what B makes of it.
//
// A slot outside the pool raises the status word (code 6), and the token counts as one without an adapter.
#include "common.cuh"

namespace ms {

constexpr int MAX_PARTS = 4;

// What the kernels know of a projection's adapters and of the step's tokens.
struct Adapters {
  const void* a;          // [slots, parts * rank, K], the model's type
  const void* b;          // [slots, N, rank]
  const float* scale;     // [slots]
  const int* slot_of_row;
  const int* row_of_token;
  int* status;
  int slots, rank, parts, ends[MAX_PARTS];  // ends[p]: the first column behind part p
};

__device__ __forceinline__ int adapter_of(const Adapters& ad, int t) {
  const int s = behind_load(ad.slot_of_row + behind_load(ad.row_of_token + t));
  if (s < ad.slots) return s < 0 ? -1 : s;
  atomicExch(ad.status, 6);
  return -1;
}
__device__ __forceinline__ int part_of(const Adapters& ad, int n) {
  int p = 0;
#pragma unroll
  for (int i = 0; i + 1 < MAX_PARTS; ++i)
    if (i + 1 < ad.parts && n >= ad.ends[i]) p = i + 1;
  return p;
}

template <typename T>
struct Wide;  // 16 bytes as float32
template <>
struct Wide<float> {
  static constexpr int N = 4;
  static __device__ __forceinline__ void get(const uint4& v, float (&f)[4]) {
    f[0] = __uint_as_float(v.x); f[1] = __uint_as_float(v.y); f[2] = __uint_as_float(v.z); f[3] = __uint_as_float(v.w);
  }
};
template <>
struct Wide<__nv_bfloat16> {
  static constexpr int N = 8;
  static __device__ __forceinline__ void get(const uint4& v, float (&f)[8]) { bf16x8_to_float(v, f); }
};

// v[t, j] = c_s sum_k A_s[j, k] x[t, k]. A block: one token, SHRINK_WARPS / split numbers; `split` warps share a number's k, their sums added in
// order. The order of a sum follows from K alone, so a token's numbers do not depend on the step around it.
constexpr int SHRINK_WARPS = 8;
template <typename T>
__global__ void __launch_bounds__(SHRINK_WARPS * 32)
adapter_shrink_kernel(float* __restrict__ v, const T* __restrict__ x, const Adapters ad, int K, int split) {
  constexpr int W = Wide<T>::N;
  __shared__ float sums[SHRINK_WARPS];
  pdl_prologue(v, x);
  const int t = blockIdx.x, warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int s = adapter_of(ad, t), numbers = ad.parts * ad.rank;
  if (s < 0) return;
  const int j = (int)blockIdx.y * (SHRINK_WARPS / split) + warp / split, piece = warp % split;
  const int chunks = K / W, each = (chunks + split - 1) / split, end = min(chunks, (piece + 1) * each);
  float sum = 0.f;
  if (j < numbers) {
    const uint4* row = reinterpret_cast<const uint4*>(reinterpret_cast<const T*>(ad.a) + ((size_t)s * numbers + j) * K);
    const uint4* xs = reinterpret_cast<const uint4*>(x + (size_t)t * K);
#pragma unroll 4
    for (int c = piece * each + lane; c < end; c += 32) {
      float fa[W], fx[W];
      Wide<T>::get(row[c], fa);
      Wide<T>::get(xs[c], fx);
#pragma unroll
      for (int i = 0; i < W; ++i) sum = fmaf(fa[i], fx[i], sum);
    }
  }
  sum = warp_sum(sum);
  if (lane == 0) sums[warp] = sum;
  __syncthreads();
  if (lane == 0 && piece == 0 && j < numbers) {
    float total = sums[warp];
    for (int i = 1; i < split; ++i) total += sums[warp + i];
    v[(size_t)t * numbers + j] = total * ad.scale[s];
  }
}

// y[t, n] += sum_j B_s[n, j] v[t, p(n) r + j], a thread a column. O: y's type.
template <typename T, typename O>
__global__ void __launch_bounds__(256)
adapter_expand_kernel(O* __restrict__ y, const float* __restrict__ v, const Adapters ad, int N) {
  constexpr int W = Wide<T>::N;
  extern __shared__ __align__(16) float vs[];
  pdl_prologue(y, v);
  const int t = blockIdx.y, s = adapter_of(ad, t), numbers = ad.parts * ad.rank;
  if (s < 0) return;
  for (int i = threadIdx.x; i < numbers; i += blockDim.x) vs[i] = v[(size_t)t * numbers + i];
  __syncthreads();
  const int n = blockIdx.x * 256 + threadIdx.x;
  if (n >= N) return;
  const float* mine = vs + part_of(ad, n) * ad.rank;
  const uint4* row = reinterpret_cast<const uint4*>(reinterpret_cast<const T*>(ad.b) + ((size_t)s * N + n) * ad.rank);
  float sum = 0.f;
  for (int c = 0; c < ad.rank / W; ++c) {
    float fb[W];
    Wide<T>::get(row[c], fb);
#pragma unroll
    for (int i = 0; i < W; ++i) sum = fmaf(fb[i], mine[c * W + i], sum);
  }
  O* at = y + (size_t)t * N + n;
  Elem<O>::store(at, Elem<O>::load(at) + sum);
}

}  // namespace ms

using namespace ms;

MS_DEFINE_LAST_ERROR(ms_adapters_last_error)
MS_DEFINE_PDL_SWITCH(ms_adapters_set_pdl)

static int check_adapters(const Adapters* ad, int T, int N, int K) {
  MS_CHECK_ARG(ad != nullptr && T >= 0 && N > 0 && K > 0 && ad->slots > 0 && ad->rank > 0 && ad->parts >= 1 && ad->parts <= MAX_PARTS,
               "adapters: bad sizes T=%d N=%d K=%d", T, N, K);
  MS_CHECK_ARG(ad->rank % 8 == 0 && K % 8 == 0, "adapters: rank=%d and K=%d must be multiples of 8", ad->rank, K);
  MS_CHECK_ARG((uintptr_t)ad->a % 16 == 0 && (uintptr_t)ad->b % 16 == 0, "adapters: the matrices must be 16-byte aligned");
  for (int p = 0; p < ad->parts; ++p)
    MS_CHECK_ARG(ad->ends[p] > (p ? ad->ends[p - 1] : 0) && (p + 1 < ad->parts ? ad->ends[p] < N : ad->ends[p] == N), "adapters: part %d ends at %d of %d", p,
                 ad->ends[p], N);
  MS_CHECK_ARG(ad->scale && ad->slot_of_row && ad->row_of_token && ad->status, "adapters: null pointer");
  return 0;
}

// v float32 [T, parts * rank]; rows of tokens without an adapter are left as they were.
MS_EXPORT int ms_adapter_shrink(float* v, const void* x, const Adapters* ad, int T, int N, int K, int dtype, cudaStream_t stream) {
  if (int rc = check_adapters(ad, T, N, K)) return rc;
  MS_CHECK_ARG((uintptr_t)x % 16 == 0, "adapters: x must be 16-byte aligned");
  if (T == 0) return 0;
  const int numbers = ad->parts * ad->rank;
  int split = 1;
  while (split < SHRINK_WARPS && K > 2048 * split) split *= 2;
  const dim3 grid(T, ceil_div(numbers, SHRINK_WARPS / split));
  if (dtype == MS_F32) MS_LAUNCH(adapter_shrink_kernel<float>, grid, SHRINK_WARPS * 32, 0, stream, v, (const float*)x, *ad, K, split);
  else MS_LAUNCH(adapter_shrink_kernel<__nv_bfloat16>, grid, SHRINK_WARPS * 32, 0, stream, v, (const __nv_bfloat16*)x, *ad, K, split);
  return 0;
}

// y [T, N] (out_dtype) += what B makes of v.
MS_EXPORT int ms_adapter_expand(void* y, const float* v, const Adapters* ad, int T, int N, int K, int dtype, int out_dtype, cudaStream_t stream) {
  if (int rc = check_adapters(ad, T, N, K)) return rc;
  MS_CHECK_ARG(T <= 65535, "adapters: %d tokens are too many for one launch", T);
  if (T == 0) return 0;
  const dim3 grid(ceil_div(N, 256), T);
  const size_t smem = (size_t)ad->parts * ad->rank * sizeof(float);
  if (dtype == MS_F32) MS_LAUNCH((adapter_expand_kernel<float, float>), grid, 256, smem, stream, (float*)y, v, *ad, N);
  else if (out_dtype == MS_F32) MS_LAUNCH((adapter_expand_kernel<__nv_bfloat16, float>), grid, 256, smem, stream, (float*)y, v, *ad, N);
  else MS_LAUNCH((adapter_expand_kernel<__nv_bfloat16, __nv_bfloat16>), grid, 256, smem, stream, (__nv_bfloat16*)y, v, *ad, N);
  return 0;
}
