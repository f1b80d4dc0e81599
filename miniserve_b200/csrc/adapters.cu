// Low-rank adapters of many requests at once beside a projection that all requests share:
//   y[t, n] = (W x_t)_n + c_s sum_j B_s[n, j] (A_s x_t)[p(n) r + j],   s = slot_of_row[row_of_token[t]],
// r numbers for each part p of the stacked output (q|k|v, gate|up), B's row n with the numbers of its part. A slot below 0: no adapter.
//
// Here are v = c_s A_s x_t (the scale inside) and, where the shared product does not take adapters into its own sums, what B makes of v added to a product in float32,
// so that an output is rounded once. Steps of many tokens have a plan: for each row tile of 256 tokens the adapters in it.
#include "adapters.cuh"

namespace ms {

// ---------------------------------------------------------------- the plan of a step of many tokens
// One CTA. A warp takes a row tile at a time and lists the adapters in it, the smallest slot first; tile_first is a running count over the tiles.
constexpr int PLAN_THREADS = 1024;
__global__ void __launch_bounds__(PLAN_THREADS)
adapter_plan_kernel(int* __restrict__ tile_first, int* __restrict__ block_slot, AdapterBlock* __restrict__ blocks, const Adapters ad, int T, int max_blocks) {
  pdl_prologue(tile_first, block_slot, blocks);
  constexpr int PER = ADAPTER_ROWS / 32, NONE = 0x7fffffff;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, tiles = (T + ADAPTER_ROWS - 1) / ADAPTER_ROWS;
  int slot[PER];
  // f(i, slot, left) for every adapter of the tile, i counting them; `left`: the slots of those still to come
  auto each = [&](int (&left)[PER], auto f) {
    for (int i = 0;; ++i) {
      int least = NONE;
#pragma unroll
      for (int q = 0; q < PER; ++q) least = min(least, left[q]);
      least = __reduce_min_sync(0xffffffffu, least);
      if (least == NONE) return i;
      f(i, least, left);
#pragma unroll
      for (int q = 0; q < PER; ++q)
        if (left[q] == least) left[q] = NONE;
    }
  };
  auto slots_of = [&](int tile) {
#pragma unroll
    for (int q = 0; q < PER; ++q) {
      const int t = tile * ADAPTER_ROWS + 32 * q + lane;
      const int s = t < T ? adapter_of(ad, t) : -1;
      slot[q] = s < 0 ? NONE : s;
    }
  };
  for (int tile = warp; tile < tiles; tile += PLAN_THREADS / 32) {
    slots_of(tile);
    const int n = each(slot, [](int, int, int (&)[PER]) {});
    if (lane == 0) tile_first[tile + 1] = n;
  }
  __syncthreads();
  if (warp == 0) {
    int before = 0;
    for (int tile0 = 0; tile0 < tiles; tile0 += 32) {
      const int tile = tile0 + lane;
      int n = tile < tiles ? tile_first[tile + 1] : 0;
#pragma unroll
      for (int o = 1; o < 32; o <<= 1) {
        const int x = __shfl_up_sync(0xffffffffu, n, o);
        if (lane >= o) n += x;
      }
      n += before;
      before = __shfl_sync(0xffffffffu, n, 31);
      if (tile < tiles) tile_first[tile + 1] = min(n, max_blocks);
    }
    if (lane == 0) {
      tile_first[0] = 0;
      if (before > max_blocks) atomicExch(ad.status, 6);  // (tokens that are not in the order of their requests)
    }
  }
  __syncthreads();
  for (int tile = warp; tile < tiles; tile += PLAN_THREADS / 32) {
    slots_of(tile);
    const int first = tile_first[tile], last = tile_first[tile + 1];
    each(slot, [&](int i, int s, int (&left)[PER]) {
      if (first + i >= last) return;
      unsigned mine = 0;
#pragma unroll
      for (int q = 0; q < PER; ++q) {
        const unsigned m = __ballot_sync(0xffffffffu, left[q] == s);
        if (lane == q) mine = m;
      }
      if (lane < PER) blocks[first + i].members[lane] = mine;
      if (lane == 0) {
        block_slot[first + i] = s;
        blocks[first + i].slot = s;
        blocks[first + i].tile = tile;
      }
    });
  }
}

// ---------------------------------------------------------------- v of a few tokens
// v[t, j] = c_s sum_k A_s[j, k] x[t, k]. A block: one token, SHRINK_WARPS / split numbers; `split` warps share a number's k, their sums added in
// order. The order of a sum follows from K alone, so a token's numbers do not depend on the step around it.
constexpr int SHRINK_WARPS = 8;
template <typename T>
__global__ void __launch_bounds__(SHRINK_WARPS * 32)
adapter_shrink_kernel(float* v, const T* x, const Adapters ad, int K, int split) {
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
#pragma unroll 8
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

// ---------------------------------------------------------------- what B makes of v, beside a product in float32
// out[t, n] = y[t, n] + sum_j B_s[n, j] v[t, p(n) r + j], or (GATED) silu of a gate column times its up column, a thread a column, TOKENS tokens a block (a block's
// rows of B stay in its multiprocessor's first cache from token to token). out may be y.
template <typename T, typename O, bool GATED, int TOKENS>
__global__ void __launch_bounds__(256)
adapter_expand_kernel(O* out, const float* y, const float* v, const Adapters ad, int N, int T_all) {
  extern __shared__ __align__(16) float vs[];  // [TOKENS][parts * rank]
  __shared__ int slot[TOKENS];
  pdl_prologue(out, y, v);
  const int numbers = ad.parts * ad.rank, cols = GATED ? N / 2 : N, n = blockIdx.x * 256 + threadIdx.x, t0 = blockIdx.y * TOKENS, count = min(TOKENS, T_all - t0);
  if ((int)threadIdx.x < count) slot[threadIdx.x] = adapter_of(ad, t0 + threadIdx.x);
  float gate[TOKENS], up[TOKENS];
  if (n < cols) {
#pragma unroll
    for (int t = 0; t < TOKENS; ++t) {
      gate[t] = t < count ? y[(size_t)(t0 + t) * N + n] : 0.f;
      up[t] = GATED && t < count ? y[(size_t)(t0 + t) * N + cols + n] : 0.f;
    }
  }
  __syncthreads();
  for (int i = threadIdx.x; i < count * numbers; i += 256)
    if (slot[i / numbers] >= 0) vs[i] = v[(size_t)t0 * numbers + i];
  __syncthreads();
  if (n >= cols) return;
  const T* b = reinterpret_cast<const T*>(ad.b);
  auto term = [&](int t, int c) { return adapter_dot(b + ((size_t)slot[t] * N + c) * ad.rank, vs + t * numbers + part_of(ad, c) * ad.rank, ad.rank); };
#pragma unroll
  for (int t = 0; t < TOKENS; ++t) {
    if (t >= count) break;
    float o = gate[t], u = up[t];
    if (slot[t] >= 0) {
      o += term(t, n);
      if (GATED) u += term(t, cols + n);
    }
    if (GATED) o = o / (1.0f + expf(-o)) * u;
    Elem<O>::store(out + (size_t)(t0 + t) * cols + n, o);
  }
}

}  // namespace ms

using namespace ms;

MS_DEFINE_LAST_ERROR(ms_adapters_last_error)
MS_DEFINE_PDL_SWITCH(ms_adapters_set_pdl)

static int check_adapters(const Adapters* ad, int T, int N, int K) {
  MS_CHECK_ARG(ad != nullptr && T >= 0 && N > 0 && adapters_ok(*ad, N, K), "adapters: bad sizes T=%d N=%d K=%d", T, N, K);
  return 0;
}

// The capture that the stream is part of (0: none): a plan that a graph holds is written by every replay.
MS_EXPORT unsigned long long ms_adapter_capture_id(cudaStream_t stream) {
  cudaStreamCaptureStatus state = cudaStreamCaptureStatusNone;
  unsigned long long id = 0;
  if (cudaStreamGetCaptureInfo(stream, &state, &id) != cudaSuccess) {
    cudaGetLastError();  // (the default stream while another one is captured)
    return 0;
  }
  return state == cudaStreamCaptureStatusActive ? id + 1 : 0;
}

// tile_first [tiles of 256 tokens + 1], block_slot [max_blocks], blocks AdapterBlock [max_blocks] (on 16 bytes). Of ad only the tokens' lists, slots and status are read.
MS_EXPORT int ms_adapter_plan(int* tile_first, int* block_slot, void* blocks, const Adapters* ad, int T, int max_blocks, cudaStream_t stream) {
  MS_CHECK_ARG(tile_first && block_slot && blocks && (uintptr_t)blocks % 16 == 0 && ad && ad->slot_of_row && ad->row_of_token && ad->status && T > 0 && max_blocks > 0,
               "adapters: bad plan of %d tokens, %d blocks", T, max_blocks);
  MS_LAUNCH(adapter_plan_kernel, 1, PLAN_THREADS, 0, stream, tile_first, block_slot, (AdapterBlock*)blocks, *ad, T, max_blocks);
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

template <typename T, typename O>
static int launch_expand(void* out, const float* y, const float* v, const Adapters* ad, int T_all, int N, int gated, cudaStream_t stream) {
  const int cols = gated ? N / 2 : N, numbers = ad->parts * ad->rank;
  // eight tokens a block where that leaves blocks enough
  const bool eight = T_all > 65535 || (long long)ceil_div(cols, 256) * T_all > 8 * 2 * 148;
  const dim3 grid(ceil_div(cols, 256), ceil_div(T_all, eight ? 8 : 1));
  const size_t smem = (size_t)numbers * (eight ? 8 : 1) * sizeof(float);
  if (gated && eight) MS_LAUNCH((adapter_expand_kernel<T, O, true, 8>), grid, 256, smem, stream, (O*)out, y, v, *ad, N, T_all);
  else if (gated) MS_LAUNCH((adapter_expand_kernel<T, O, true, 1>), grid, 256, smem, stream, (O*)out, y, v, *ad, N, T_all);
  else if (eight) MS_LAUNCH((adapter_expand_kernel<T, O, false, 8>), grid, 256, smem, stream, (O*)out, y, v, *ad, N, T_all);
  else MS_LAUNCH((adapter_expand_kernel<T, O, false, 1>), grid, 256, smem, stream, (O*)out, y, v, *ad, N, T_all);
  return 0;
}

// out [T, N] (out_dtype; y itself where that is float32) = y float32 [T, N] and what B makes of v; gated: out [T, N / 2] = silu of the first half of the columns times the other.
MS_EXPORT int ms_adapter_expand(void* out, const float* y, const float* v, const Adapters* ad, int T, int N, int K, int dtype, int out_dtype, int gated, cudaStream_t stream) {
  if (int rc = check_adapters(ad, T, N, K)) return rc;
  MS_CHECK_ARG(T <= 8 * 65535, "adapters: %d tokens are too many for one launch", T);
  MS_CHECK_ARG(!gated || N % 2 == 0, "adapters: %d gate and up columns", N);
  if (T == 0) return 0;
  if (dtype == MS_F32) return launch_expand<float, float>(out, y, v, ad, T, N, gated, stream);
  if (out_dtype == MS_F32) return launch_expand<__nv_bfloat16, float>(out, y, v, ad, T, N, gated, stream);
  return launch_expand<__nv_bfloat16, __nv_bfloat16>(out, y, v, ad, T, N, gated, stream);
}
