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
adapter_plan_kernel(int* __restrict__ tile_first, AdapterBlock* __restrict__ blocks, const Adapters ad, int T, int max_blocks) {
  pdl_prologue(tile_first, blocks);
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
        blocks[first + i].slot = s;
        blocks[first + i].tile = tile;
      }
    });
  }
}

// ---------------------------------------------------------------- v of a few tokens
// v[t, j] = c_s sum_k A_s[j, k] x[t, k]. A block: one token, SHRINK_WARPS / split sets of EACH numbers; `split` warps share their k, the sums added in
// order. The order of a sum follows from K alone, so a token's numbers do not depend on the step around it. Bound by the trips to memory of a block (where an adapter is, its
// rows, the sum): 64 tokens of 96 numbers, k 4,096 take 7.6 us with four numbers a warp, 16.3 with one; 8 tokens of 16 numbers 2.7.
constexpr int SHRINK_WARPS = 8, AHEAD_CHUNK = 16384;  // (bytes that a thread asks for at a time)
template <typename T, int EACH>
__global__ void __launch_bounds__(SHRINK_WARPS * 32, EACH == 1 ? 3 : 4)
adapter_shrink_kernel(float* v, const T* x, const Adapters ad, int tokens, int K, int split, const unsigned char* ahead, long long ahead_bytes) {
  constexpr int W = Wide<T>::N;
  __shared__ float sums[SHRINK_WARPS][EACH];
  // Blocks beyond the tokens' ask the weight of the product behind into L2 while the kernels before this one still run.
  if ((int)blockIdx.x >= tokens) {
    const long long first = (long long)(blockIdx.x - tokens) * gridDim.y + blockIdx.y, step = (long long)(gridDim.x - tokens) * gridDim.y;
    if (threadIdx.x == 0)
      for (long long at = first * AHEAD_CHUNK; at < ahead_bytes; at += step * AHEAD_CHUNK)
        asm volatile("cp.async.bulk.prefetch.L2.global [%0], %1;\n" ::"l"(ahead + at), "r"((uint32_t)(ahead_bytes - at < AHEAD_CHUNK ? ahead_bytes - at : AHEAD_CHUNK)) : "memory");
    return;
  }
  // The wait comes first: a product behind may start on what earlier kernels have left, before this one has ended.
  pdl_wait(v, x);
  pdl_launch_dependents();
  const int t = blockIdx.x, warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int s = adapter_of(ad, t), numbers = ad.parts * ad.rank;
  if (s < 0) return;
  const int j = ((int)blockIdx.y * (SHRINK_WARPS / split) + warp / split) * EACH, piece = warp % split;  // (numbers: a multiple of 8)
  const int chunks = K / W, each = (chunks + split - 1) / split, end = min(chunks, (piece + 1) * each);
  float sum[EACH] = {};
  if (j < numbers) {
    const uint4* row = reinterpret_cast<const uint4*>(reinterpret_cast<const T*>(ad.a) + ((size_t)s * numbers + j) * K);
    const uint4* xs = reinterpret_cast<const uint4*>(x + (size_t)t * K);
#pragma unroll (EACH == 1 ? 8 : 2)
    for (int c = piece * each + lane; c < end; c += 32) {
      float fa[W], fx[W];
      uint4 a[EACH];
#pragma unroll
      for (int q = 0; q < EACH; ++q) a[q] = row[(size_t)q * chunks + c];
      Wide<T>::get(xs[c], fx);
#pragma unroll
      for (int q = 0; q < EACH; ++q) {
        Wide<T>::get(a[q], fa);
#pragma unroll
        for (int i = 0; i < W; ++i) sum[q] = fmaf(fa[i], fx[i], sum[q]);
      }
    }
  }
#pragma unroll
  for (int q = 0; q < EACH; ++q) {
    sum[q] = warp_sum(sum[q]);
    if (lane == 0) sums[warp][q] = sum[q];
  }
  __syncthreads();
  if (lane < EACH && piece == 0 && j < numbers) {
    float total = sums[warp][lane];
    for (int i = 1; i < split; ++i) total += sums[warp + i][lane];
    v[(size_t)t * numbers + j + lane] = total * ad.scale[s];
  }
}

// ---------------------------------------------------------------- what B makes of v, beside a product in float32; float32 adapters
// out[t, n] = y[t, n] + sum_j B_s[n, j] v[t, p(n) r + j], or (GATED) silu of a gate column times its up column, a thread a column, TOKENS tokens a block (a block's
// rows of B stay in its multiprocessor's first cache from token to token). out may be y.
template <bool GATED, int TOKENS>
__global__ void __launch_bounds__(256)
adapter_expand_kernel(float* out, const float* y, const float* v, const Adapters ad, int N, int T_all) {
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
  const float* b = reinterpret_cast<const float*>(ad.b);
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
    out[(size_t)(t0 + t) * cols + n] = o;
  }
}

// The same for bfloat16 adapters on the tensor cores: up to 32 tokens a block, and 128 columns (GATED: 64 gate and their 64 up columns) at a time of every gridDim.x-th such
// tile; the product's numbers of the next one are asked for ahead. A warp has 32 columns, four of them (a set) all columns, and the sets share the tokens' adapters out.
// Bound by the trips for B and v of each group of eight tokens: us, tokens of one adapter / of 16, rank 16, 4,096 columns: 64 5.2 / 9.5, 512 9.7 / 19.2 (in 32 bits 5.4 / 9.7 and 9.8 / 19.7; one tile of columns a block, 512
// threads: 16.6 / 35.9); 2 x 12,288 columns, 64 10.9 / 20.0. Three blocks a multiprocessor spill registers: 8.5 / 17.3, 19.9 / 48.3.
constexpr int EXPAND_TOKENS = 32, EXPAND_COLS = 128, EXPAND_SETS = 2, EXPAND_THREADS = EXPAND_SETS * 128, EXPAND_RESIDENT = 2;
template <typename O, bool GATED>
__global__ void __launch_bounds__(EXPAND_THREADS, EXPAND_RESIDENT)
adapter_expand_mma_kernel(O* out, const float* y, const float* v, const Adapters ad, int N, int T_all) {
  __shared__ float sums[EXPAND_TOKENS][EXPAND_COLS];
  __shared__ TokenGroups<EXPAND_TOKENS> tokens;
  constexpr int ROWS = GATED ? EXPAND_COLS / 2 : EXPAND_COLS, EACH = EXPAND_TOKENS / EXPAND_SETS;
  pdl_prologue(out, y, v);
  const int e = threadIdx.x, warp = e >> 5, lane = e & 31, quad = warp & 3, cols = GATED ? N / 2 : N;
  const int t0 = blockIdx.y * EXPAND_TOKENS, M = min(EXPAND_TOKENS, T_all - t0), step = gridDim.x * ROWS;
  if (e < M) tokens.slot[e] = adapter_slot(ad, t0 + e);
  // the product's numbers: a thread's column of every EXPAND_SETS-th token
  const int c = e & (EXPAND_COLS - 1), row = GATED ? c & (ROWS - 1) : c, set = e / EXPAND_COLS;
  float held[EACH];
  auto load = [&](int n0) {
#pragma unroll
    for (int q = 0; q < EACH; ++q) {
      const int t = EXPAND_SETS * q + set;
      if (t < M && n0 + row < cols) held[q] = y[(size_t)(t0 + t) * N + (GATED && c >= ROWS ? cols : 0) + n0 + row];
    }
  };
  load(blockIdx.x * ROWS);
  group_tokens(tokens, M, e, [] { __syncthreads(); });
  for (int n0 = blockIdx.x * ROWS; n0 < cols; n0 += step) {
#pragma unroll
    for (int q = 0; q < EACH; ++q) sums[EXPAND_SETS * q + set][c] = held[q];
    load(n0 + step);
    __syncthreads();
    int n[4];
    bool has[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const int r = quad * 32 + 8 * i + (lane >> 2);
      has[i] = n0 + (GATED ? r & (ROWS - 1) : r) < cols;
      n[i] = GATED && r >= ROWS ? cols + n0 + r - ROWS : n0 + r;
    }
    warp_terms<sizeof(O) == 4 ? 3 : TERM_PIECES>(ad, v + (size_t)t0 * ad.parts * ad.rank, tokens, M, warp >> 2, EXPAND_SETS, n, has, [] {},
               [&](int tok, int i) { return &sums[tok][quad * 32 + (lane >> 2) + 8 * i]; });
    __syncthreads();
    constexpr int SIDE = EXPAND_THREADS / ROWS;  // tokens side by side
    const int col = e & (ROWS - 1);
    if (n0 + col < cols)
      for (int t = e / ROWS; t < M; t += SIDE) {
        float o = sums[t][col];
        if (GATED) o = o / (1.0f + expf(-o)) * sums[t][ROWS + col];
        Elem<O>::store(out + (size_t)(t0 + t) * cols + n0 + col, o);
      }
    __syncthreads();
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

// tile_first [tiles of 256 tokens + 1], blocks AdapterBlock [max_blocks] (on 16 bytes). Of ad only the tokens' lists, slots and status are read.
MS_EXPORT int ms_adapter_plan(int* tile_first, void* blocks, const Adapters* ad, int T, int max_blocks, cudaStream_t stream) {
  MS_CHECK_ARG(tile_first && blocks && (uintptr_t)blocks % 16 == 0 && ad && ad->slot_of_row && ad->row_of_token && ad->status && T > 0 && max_blocks > 0,
               "adapters: bad plan of %d tokens, %d blocks", T, max_blocks);
  MS_LAUNCH(adapter_plan_kernel, 1, PLAN_THREADS, 0, stream, tile_first, (AdapterBlock*)blocks, *ad, T, max_blocks);
  return 0;
}

template <typename T>
static int launch_shrink(float* v, const void* x, const Adapters& ad, int tokens, int K, int numbers, int split, const void* ahead, long long ahead_bytes, cudaStream_t stream) {
  // four numbers a warp, which then reads x once for them, where that leaves warps enough
  const int each = (long long)tokens * numbers * split > 3 * 8 * 148 ? 4 : 1;
  const int chunks = (int)((ahead_bytes + AHEAD_CHUNK - 1) / AHEAD_CHUNK), rows = ceil_div(numbers, SHRINK_WARPS / split * each);
  const dim3 grid(tokens + ceil_div(chunks < 148 ? chunks : 148, rows), rows);
  if (each == 4) MS_LAUNCH((adapter_shrink_kernel<T, 4>), grid, SHRINK_WARPS * 32, 0, stream, v, (const T*)x, ad, tokens, K, split, (const unsigned char*)ahead, ahead_bytes);
  else MS_LAUNCH((adapter_shrink_kernel<T, 1>), grid, SHRINK_WARPS * 32, 0, stream, v, (const T*)x, ad, tokens, K, split, (const unsigned char*)ahead, ahead_bytes);
  return 0;
}

// v float32 [T, parts * rank]; rows of tokens without an adapter are left as they were.
// ahead: ahead_bytes (a multiple of 16; 0: none) that the launch behind will read and that no kernel that may still run writes.
MS_EXPORT int ms_adapter_shrink(float* v, const void* x, const Adapters* ad, int T, int N, int K, int dtype, const void* ahead, long long ahead_bytes, cudaStream_t stream) {
  if (int rc = check_adapters(ad, T, N, K)) return rc;
  MS_CHECK_ARG((uintptr_t)x % 16 == 0 && (uintptr_t)ahead % 16 == 0, "adapters: x and the weight must be 16-byte aligned");
  MS_CHECK_ARG(ahead_bytes >= 0 && ahead_bytes % 16 == 0 && (ahead != nullptr || ahead_bytes == 0), "adapters: bad bytes ahead: %lld", ahead_bytes);
  if (T == 0) return 0;
  const int numbers = ad->parts * ad->rank;
  int split = 1;
  while (split < SHRINK_WARPS && K > 2048 * split) split *= 2;
  return dtype == MS_F32 ? launch_shrink<float>(v, x, *ad, T, K, numbers, split, ahead, ahead_bytes, stream)
                         : launch_shrink<__nv_bfloat16>(v, x, *ad, T, K, numbers, split, ahead, ahead_bytes, stream);
}

static int launch_expand(float* out, const float* y, const float* v, const Adapters* ad, int T_all, int N, int gated, cudaStream_t stream) {
  const int cols = gated ? N / 2 : N, numbers = ad->parts * ad->rank;
  // eight tokens a block where that leaves blocks enough
  const bool eight = T_all > 65535 || (long long)ceil_div(cols, 256) * T_all > 8 * 2 * 148;
  const dim3 grid(ceil_div(cols, 256), ceil_div(T_all, eight ? 8 : 1));
  const size_t smem = (size_t)numbers * (eight ? 8 : 1) * sizeof(float);
  if (gated && eight) MS_LAUNCH((adapter_expand_kernel<true, 8>), grid, 256, smem, stream, out, y, v, *ad, N, T_all);
  else if (gated) MS_LAUNCH((adapter_expand_kernel<true, 1>), grid, 256, smem, stream, out, y, v, *ad, N, T_all);
  else if (eight) MS_LAUNCH((adapter_expand_kernel<false, 8>), grid, 256, smem, stream, out, y, v, *ad, N, T_all);
  else MS_LAUNCH((adapter_expand_kernel<false, 1>), grid, 256, smem, stream, out, y, v, *ad, N, T_all);
  return 0;
}

template <typename O>
static int launch_expand_mma(void* out, const float* y, const float* v, const Adapters* ad, int T_all, int N, int gated, cudaStream_t stream) {
  // as many blocks as are resident at a time, where the tiles are more
  const int blocks = ceil_div(T_all, EXPAND_TOKENS), tiles = ceil_div(gated ? N / 2 : N, gated ? EXPAND_COLS / 2 : EXPAND_COLS);
  const int rounds = ceil_div(blocks * (long long)tiles, EXPAND_RESIDENT * 148);
  const dim3 grid(ceil_div(tiles, rounds), blocks);
  if (gated) MS_LAUNCH((adapter_expand_mma_kernel<O, true>), grid, EXPAND_THREADS, 0, stream, (O*)out, y, v, *ad, N, T_all);
  else MS_LAUNCH((adapter_expand_mma_kernel<O, false>), grid, EXPAND_THREADS, 0, stream, (O*)out, y, v, *ad, N, T_all);
  return 0;
}

// out [T, N] (out_dtype; y itself where that is float32) = y float32 [T, N] and what B makes of v; gated: out [T, N / 2] = silu of the first half of the columns times the other.
MS_EXPORT int ms_adapter_expand(void* out, const float* y, const float* v, const Adapters* ad, int T, int N, int K, int dtype, int out_dtype, int gated, cudaStream_t stream) {
  if (int rc = check_adapters(ad, T, N, K)) return rc;
  MS_CHECK_ARG(T <= 8 * 65535, "adapters: %d tokens are too many for one launch", T);
  MS_CHECK_ARG(!gated || N % 2 == 0, "adapters: %d gate and up columns", N);
  if (T == 0) return 0;
  if (dtype == MS_F32) return launch_expand((float*)out, y, v, ad, T, N, gated, stream);
  return out_dtype == MS_F32 ? launch_expand_mma<float>(out, y, v, ad, T, N, gated, stream) : launch_expand_mma<__nv_bfloat16>(out, y, v, ad, T, N, gated, stream);
}
