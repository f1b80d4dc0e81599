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
adapter_plan_kernel(int* __restrict__ tile_first, int* __restrict__ block_slot, int* __restrict__ block_tile, int* __restrict__ token_slot, const Adapters ad, int T,
                    int max_blocks) {
  pdl_prologue(tile_first, block_slot, block_tile, token_slot);
  constexpr int PER = ADAPTER_ROWS / 32, NONE = 0x7fffffff;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, tiles = (T + ADAPTER_ROWS - 1) / ADAPTER_ROWS;
  int slot[PER];
  // f(i, slot) for every adapter of the tile, i counting them
  auto each = [&](int (&left)[PER], auto f) {
    for (int i = 0;; ++i) {
      int least = NONE;
#pragma unroll
      for (int q = 0; q < PER; ++q) least = min(least, left[q]);
      least = __reduce_min_sync(0xffffffffu, least);
      if (least == NONE) return i;
      f(i, least);
#pragma unroll
      for (int q = 0; q < PER; ++q)
        if (left[q] == least) left[q] = NONE;
    }
  };
  for (int tile = warp; tile < tiles; tile += PLAN_THREADS / 32) {
#pragma unroll
    for (int q = 0; q < PER; ++q) {
      const int t = tile * ADAPTER_ROWS + 32 * q + lane;
      const int s = t < T ? adapter_of(ad, t) : -1;
      if (t < T) token_slot[t] = s;
      slot[q] = s < 0 ? NONE : s;
    }
    const int n = each(slot, [](int, int) {});
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
#pragma unroll
    for (int q = 0; q < PER; ++q) {
      const int t = tile * ADAPTER_ROWS + 32 * q + lane;
      const int s = t < T ? token_slot[t] : -1;
      slot[q] = s < 0 ? NONE : s;
    }
    const int first = tile_first[tile], last = tile_first[tile + 1];
    each(slot, [&](int i, int s) {
      if (lane == 0 && first + i < last) {
        block_slot[first + i] = s;
        block_tile[first + i] = tile;
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

// ---------------------------------------------------------------- v of many tokens, by the plan's blocks
// A block of threads takes 32 rows of a block of the plan and NT * 8 numbers. Its warps share out K and multiply straight from memory: a lane's 16 bytes of a row are
// 8 k of the instruction's order, the same for both operands, so any order of k does. Both operands lie in L2 (x was just written, A is a few hundred KB).
// COMPACT: float32 v [T, numbers] for tokens with an adapter; else bfloat16 V [blocks * 256, numbers], what the product's tensor cores take: v is rounded to 8 bits
// (2^-8 of an adapter's share of an output, where the output itself is rounded so).
constexpr int BLOCKS_WARPS = 8, BLOCKS_ROWS = 32;
__device__ __forceinline__ void mma_bf16_16816(float (&c)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1) {
  asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};\n"
               : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
               : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}
template <int NT, bool COMPACT>
__global__ void __launch_bounds__(BLOCKS_WARPS * 32)
adapter_shrink_blocks_kernel(void* __restrict__ v, const __nv_bfloat16* __restrict__ x, const Adapters ad, const int* __restrict__ tile_first,
                             const int* __restrict__ block_slot, const int* __restrict__ block_tile, const int* __restrict__ token_slot, int T, int K) {
  extern __shared__ __align__(16) float sb_sums[];  // [warps][32 rows][NT * 8]
  constexpr int N = NT * 8;
  pdl_prologue(v, x, tile_first, block_slot, block_tile, token_slot);
  const int b = blockIdx.y, tiles = (T + ADAPTER_ROWS - 1) / ADAPTER_ROWS;
  if (b >= tile_first[tiles]) return;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, g = lane >> 2, t4 = lane & 3;
  const int s = block_slot[b], row0 = blockIdx.x * BLOCKS_ROWS, tok0 = block_tile[b] * ADAPTER_ROWS + row0, numbers = ad.parts * ad.rank, j0 = blockIdx.z * N;
  const bool member = tok0 + lane < T && token_slot[tok0 + lane] == s;
  const unsigned members = __ballot_sync(0xffffffffu, member);
  if (members == 0) {
    if (!COMPACT)
      for (int i = threadIdx.x; i < BLOCKS_ROWS * N; i += blockDim.x) {
        const int j = j0 + i % N;
        if (j < numbers) reinterpret_cast<__nv_bfloat16*>(v)[((size_t)b * ADAPTER_ROWS + row0 + i / N) * numbers + j] = __float2bfloat16_rn(0.f);
      }
    return;
  }
  float acc[2][NT][4];
#pragma unroll
  for (int m = 0; m < 2; ++m)
#pragma unroll
    for (int n = 0; n < NT; ++n) acc[m][n][0] = acc[m][n][1] = acc[m][n][2] = acc[m][n][3] = 0.f;
  const int per = (K + BLOCKS_WARPS * 32 - 1) / (BLOCKS_WARPS * 32) * 32, k0 = warp * per, k1 = min(K, k0 + per);
  const __nv_bfloat16* xr[4];
  bool has[4];
#pragma unroll
  for (int m = 0; m < 4; ++m) {
    has[m] = (members >> (8 * m + g)) & 1;
    xr[m] = x + (size_t)(tok0 + (has[m] ? 8 * m + g : 0)) * K + 8 * t4;
  }
  const __nv_bfloat16* ar = reinterpret_cast<const __nv_bfloat16*>(ad.a) + ((size_t)s * numbers + j0 + g) * K + 8 * t4;
#pragma unroll 2
  for (int k = k0; k < k1; k += 32) {
    const bool in = k + 8 * t4 < k1;
    uint4 xv[4], av[NT];
    const uint4 zero = make_uint4(0u, 0u, 0u, 0u);
#pragma unroll
    for (int m = 0; m < 4; ++m) xv[m] = in && has[m] ? *reinterpret_cast<const uint4*>(xr[m] + k) : zero;
#pragma unroll
    for (int n = 0; n < NT; ++n) av[n] = in && j0 + 8 * n + g < numbers ? *reinterpret_cast<const uint4*>(ar + (size_t)(8 * n) * K + k) : zero;
#pragma unroll
    for (int n = 0; n < NT; ++n)
#pragma unroll
      for (int m = 0; m < 2; ++m) {
        mma_bf16_16816(acc[m][n], xv[2 * m].x, xv[2 * m + 1].x, xv[2 * m].y, xv[2 * m + 1].y, av[n].x, av[n].y);
        mma_bf16_16816(acc[m][n], xv[2 * m].z, xv[2 * m + 1].z, xv[2 * m].w, xv[2 * m + 1].w, av[n].z, av[n].w);
      }
  }
  float* mine = sb_sums + (size_t)warp * BLOCKS_ROWS * N;
#pragma unroll
  for (int m = 0; m < 2; ++m)
#pragma unroll
    for (int n = 0; n < NT; ++n) {
      *reinterpret_cast<float2*>(mine + (16 * m + g) * N + 8 * n + 2 * t4) = make_float2(acc[m][n][0], acc[m][n][1]);
      *reinterpret_cast<float2*>(mine + (16 * m + g + 8) * N + 8 * n + 2 * t4) = make_float2(acc[m][n][2], acc[m][n][3]);
    }
  __syncthreads();
  const float c = ad.scale[s];
  for (int i = threadIdx.x; i < BLOCKS_ROWS * N; i += blockDim.x) {
    const int row = i / N, j = j0 + i % N;
    float sum = 0.f;
#pragma unroll
    for (int w = 0; w < BLOCKS_WARPS; ++w) sum += sb_sums[(size_t)w * BLOCKS_ROWS * N + i];
    const bool is = (members >> row) & 1;
    if (j >= numbers) continue;
    if (COMPACT) {
      if (is) reinterpret_cast<float*>(v)[(size_t)(tok0 + row) * numbers + j] = sum * c;
    } else {
      reinterpret_cast<__nv_bfloat16*>(v)[((size_t)b * ADAPTER_ROWS + row0 + row) * numbers + j] = __float2bfloat16_rn(is ? sum * c : 0.f);
    }
  }
}

// ---------------------------------------------------------------- what B makes of v, beside a product in float32
// out[t, n] = y[t, n] + sum_j B_s[n, j] v[t, p(n) r + j], or (GATED) silu of a gate column times its up column, a thread a column, `tokens` tokens a block. out may be y.
template <typename T, typename O, bool GATED>
__global__ void __launch_bounds__(256)
adapter_expand_kernel(O* out, const float* y, const float* v, const Adapters ad, int N, int T_all, int tokens) {
  extern __shared__ __align__(16) float vs[];
  pdl_prologue(out, y, v);
  const int numbers = ad.parts * ad.rank, cols = GATED ? N / 2 : N, n = blockIdx.x * 256 + threadIdx.x;
  const T* b = reinterpret_cast<const T*>(ad.b);
  const int t0 = blockIdx.y * tokens, t1 = min(T_all, t0 + tokens);
  for (int t = t0; t < t1; ++t) {
    const int s = adapter_of(ad, t);
    __syncthreads();
    if (s >= 0)
      for (int i = threadIdx.x; i < numbers; i += blockDim.x) vs[i] = v[(size_t)t * numbers + i];
    __syncthreads();
    if (n >= cols) continue;
    auto column = [&](int c) {
      const float sum = y[(size_t)t * N + c];
      return s < 0 ? sum : sum + adapter_dot(b + ((size_t)s * N + c) * ad.rank, vs + part_of(ad, c) * ad.rank, ad.rank);
    };
    float o = column(n);
    if (GATED) {
      const float up = column(cols + n);
      o = o / (1.0f + expf(-o)) * up;
    }
    Elem<O>::store(out + (size_t)t * cols + n, o);
  }
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

// tile_first [tiles of 256 tokens + 1], block_slot and block_tile [max_blocks], token_slot [T]. Of ad only the tokens' lists, slots and status are read.
MS_EXPORT int ms_adapter_plan(int* tile_first, int* block_slot, int* block_tile, int* token_slot, const Adapters* ad, int T, int max_blocks, cudaStream_t stream) {
  MS_CHECK_ARG(tile_first && block_slot && block_tile && token_slot && ad && ad->slot_of_row && ad->row_of_token && ad->status && T > 0 && max_blocks > 0,
               "adapters: bad plan of %d tokens, %d blocks", T, max_blocks);
  MS_LAUNCH(adapter_plan_kernel, 1, PLAN_THREADS, 0, stream, tile_first, block_slot, block_tile, token_slot, *ad, T, max_blocks);
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

template <int NT, bool COMPACT>
static int launch_blocks(void* v, const void* x, const Adapters* ad, const int* tile_first, const int* block_slot, const int* block_tile, const int* token_slot, int T, int K,
                         int max_blocks, cudaStream_t stream) {
  constexpr size_t smem = (size_t)BLOCKS_WARPS * BLOCKS_ROWS * NT * 8 * sizeof(float);
  auto kernel = adapter_shrink_blocks_kernel<NT, COMPACT>;
  if (smem > 48 * 1024) {
    static std::atomic<unsigned long long> allowed{0};
    MS_CHECK_CUDA(allow_shared_memory((const void*)kernel, (int)smem, allowed));
  }
  const dim3 grid(ADAPTER_ROWS / BLOCKS_ROWS, max_blocks, ceil_div(ad->parts * ad->rank, NT * 8));
  MS_LAUNCH(kernel, grid, BLOCKS_WARPS * 32, smem, stream, v, (const __nv_bfloat16*)x, *ad, tile_first, block_slot, block_tile, token_slot, T, K);
  return 0;
}

// By a plan: compact = 0: v bfloat16 [max_blocks * 256, parts * rank]; 1: as ms_adapter_shrink's.
MS_EXPORT int ms_adapter_shrink_blocks(void* v, const void* x, const Adapters* ad, const int* tile_first, const int* block_slot, const int* block_tile,
                                       const int* token_slot, int T, int N, int K, int max_blocks, int compact, cudaStream_t stream) {
  if (int rc = check_adapters(ad, T, N, K)) return rc;
  MS_CHECK_ARG((uintptr_t)x % 16 == 0 && max_blocks > 0 && max_blocks <= 65535, "adapters: x must be 16-byte aligned, %d blocks", max_blocks);
  if (T == 0) return 0;
  const int numbers = ad->parts * ad->rank, nt = numbers <= 16 ? 2 : numbers <= 32 ? 4 : numbers <= 48 ? 6 : 8;
#define MS_BLOCKS(NT)                                                                                                                              \
  return compact ? launch_blocks<NT, true>(v, x, ad, tile_first, block_slot, block_tile, token_slot, T, K, max_blocks, stream)                     \
                 : launch_blocks<NT, false>(v, x, ad, tile_first, block_slot, block_tile, token_slot, T, K, max_blocks, stream)
  switch (nt) {
    case 2: MS_BLOCKS(2);
    case 4: MS_BLOCKS(4);
    case 6: MS_BLOCKS(6);
    default: MS_BLOCKS(8);
  }
#undef MS_BLOCKS
}

template <typename T, typename O>
static int launch_expand(void* out, const float* y, const float* v, const Adapters* ad, int T_all, int N, int gated, cudaStream_t stream) {
  const int tokens = T_all <= 64 ? 1 : 8;
  const dim3 grid(ceil_div(gated ? N / 2 : N, 256), ceil_div(T_all, tokens));
  const size_t smem = (size_t)ad->parts * ad->rank * sizeof(float);
  if (gated) MS_LAUNCH((adapter_expand_kernel<T, O, true>), grid, 256, smem, stream, (O*)out, y, v, *ad, N, T_all, tokens);
  else MS_LAUNCH((adapter_expand_kernel<T, O, false>), grid, 256, smem, stream, (O*)out, y, v, *ad, N, T_all, tokens);
  return 0;
}

// out [T, N] (out_dtype; y itself where that is float32) = y float32 [T, N] and what B makes of v; gated: out [T, N / 2] = silu of the first half of the columns times the other.
MS_EXPORT int ms_adapter_expand(void* out, const float* y, const float* v, const Adapters* ad, int T, int N, int K, int dtype, int out_dtype, int gated, cudaStream_t stream) {
  if (int rc = check_adapters(ad, T, N, K)) return rc;
  MS_CHECK_ARG(ceil_div(T, 8) <= 65535, "adapters: %d tokens are too many for one launch", T);
  MS_CHECK_ARG(!gated || N % 2 == 0, "adapters: %d gate and up columns", N);
  if (T == 0) return 0;
  if (dtype == MS_F32) return launch_expand<float, float>(out, y, v, ad, T, N, gated, stream);
  if (out_dtype == MS_F32) return launch_expand<__nv_bfloat16, float>(out, y, v, ad, T, N, gated, stream);
  return launch_expand<__nv_bfloat16, __nv_bfloat16>(out, y, v, ad, T, N, gated, stream);
}
