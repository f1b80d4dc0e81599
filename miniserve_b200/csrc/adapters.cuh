// Low-rank adapters of many requests at once beside a projection that all requests share: what the kernels of adapters.cu and the products that take
// adapters in their own sums (gemm_tc.cu, gemm_skinny.cu) know of them.
#pragma once

#include "common.cuh"

namespace ms {

constexpr int MAX_PARTS = 4;       // of a stacked projection
constexpr int ADAPTER_ROWS = 256;  // tokens of a row tile of the plan, rows of a block of V: the row tiles of the 2-CTA product

// The adapters of one projection, and the step's tokens.
struct Adapters {
  const void* a;          // [slots, parts * rank, K], the model's type
  const void* b;          // [slots, N, rank]
  const float* scale;     // [slots]
  const int* slot_of_row;
  const int* row_of_token;
  int* status;            // raised (6) by a slot that is not there
  int slots, rank, parts, ends[MAX_PARTS];  // ends[p]: the first column behind part p (of parts that there are not, N)
};

// An adapted product of many tokens: what launches before it have written for it (ms_adapter_plan, ms_gemm_tc_adapter_v). A block is the tokens of one row tile that have
// one adapter: 256 rows of V, zeros in those of other tokens.
struct AdaptedProduct {
  Adapters ad;
  const void* v;          // bfloat16 [max_blocks * 256, parts * rank]
  const int* tile_first;  // [row tiles + 1]
  const int* block_slot;  // [max_blocks]
  int max_blocks;
};

// What a block is: its adapter, its row tile, and which of the tile's tokens have it, a bit each.
struct AdapterBlock {
  int slot, tile, pad[2];
  unsigned members[ADAPTER_ROWS / 32];
};
static_assert(sizeof(AdapterBlock) == 48, "what the host allots");

// An adapted product of few tokens: v float32 [T, parts * rank]; rows of tokens without an adapter are not read. tickets null: an earlier launch made v (ms_adapter_shrink);
// else the product's own CTAs make it, and tickets are two zeros that no other launch has.
struct AdapterTerms {
  float* v;
  Adapters ad;
  int* tickets;
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
  for (int i = 0; i + 1 < MAX_PARTS; ++i) p += n >= ad.ends[i];
  return p;
}

// (host) Whether the sizes are ones that the kernels take.
inline bool adapters_ok(const Adapters& ad, int N, int K) {
  if (ad.slots < 1 || ad.rank < 8 || ad.rank % 8 || ad.parts < 1 || ad.parts > MAX_PARTS || K < 8 || K % 8) return false;
  if ((uintptr_t)ad.a % 16 || (uintptr_t)ad.b % 16 || !ad.scale || !ad.slot_of_row || !ad.row_of_token || !ad.status) return false;
  for (int p = 0; p < MAX_PARTS; ++p)
    if (p + 1 < ad.parts ? ad.ends[p] <= (p ? ad.ends[p - 1] : 0) || ad.ends[p] >= N : ad.ends[p] != N) return false;
  return true;
}

// 16 bytes as float32
template <typename T>
struct Wide;
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

// sum_j row[j] v[j], `rank` numbers (a multiple of 8; both on 16 bytes)
template <typename T>
__device__ __forceinline__ float adapter_dot(const T* row, const float* v, int rank) {
  constexpr int W = Wide<T>::N;
  float sum = 0.f;
  for (int c = 0; c < rank; c += W) {
    float f[W];
    Wide<T>::get(*reinterpret_cast<const uint4*>(row + c), f);
#pragma unroll
    for (int i = 0; i < W; i += 4) {
      const float4 x = *reinterpret_cast<const float4*>(v + c + i);
      sum = fmaf(f[i], x.x, sum);
      sum = fmaf(f[i + 1], x.y, sum);
      sum = fmaf(f[i + 2], x.z, sum);
      sum = fmaf(f[i + 3], x.w, sum);
    }
  }
  return sum;
}

}  // namespace ms
