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
  int* status;            // raised (6) by a slot or a row that is not there
  int rows, unused;       // of slot_of_row
  int slots, rank, parts, ends[MAX_PARTS];  // ends[p]: the first column behind part p (of parts that there are not, N)
};

// An adapted product of many tokens: what launches before it have written for it (ms_adapter_plan, ms_gemm_tc_adapter_v). A block is the tokens of one row tile that have
// one adapter: 256 rows of V, zeros in those of other tokens.
struct AdaptedProduct {
  Adapters ad;
  const void* v;          // bfloat16 [max_blocks * 256, parts * rank]
  const int* tile_first;  // [row tiles + 1]
  const void* blocks;     // AdapterBlock [max_blocks]
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
  const int row = behind_load(ad.row_of_token + t);
  if ((unsigned)row < (unsigned)ad.rows) {
    const int s = behind_load(ad.slot_of_row + row);
    if (s < ad.slots) return s < 0 ? -1 : s;
  }
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

// ---- terms of few tokens on the tensor cores: sum_j B_s[n, j] v[t, j], v as the sum of PIECES bfloat16 numbers: three hold all of its 24 bits, for outputs in
// 32 bits; two hold 16, for outputs that are rounded to 8. One (2^-8 of an adapter's share lost) / two, us: 64 tokens of 16 adapters of rank 32, 4096 -> 6144 24.2 / 24.3, 32 of 1024 -> 4096 10.3 / 10.4, 8 of
// 12288 -> 4096 21.0 / 21.0, 200 beside a product apart 50.8 / 51.1; one / three with outputs in 32 bits: 33.2 / 33.8, 14.2 / 14.6, 42.9 / 43.3, 50.7 / 51.4.
constexpr int NO_SLOT = 0x7fffffff, TERM_PIECES = 2;
__device__ __forceinline__ void mma_16816(float (&c)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1) {
  asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};\n"
               : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
               : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}
// Waits until other CTAs of the launch have counted up to `all`, for at most MS_WAIT_NS: false then. What they wrote before is visible behind it.
__device__ __forceinline__ bool tickets_reach(const int* counter, int all) {
  unsigned long long began = 0;
  for (unsigned polls = 1;; ++polls) {
    int done;
    asm volatile("ld.acquire.gpu.global.s32 %0, [%1];\n" : "=r"(done) : "l"(counter) : "memory");
    if (done >= all) return true;
    if (polls % 64) continue;
    unsigned long long now;
    asm volatile("mov.u64 %0, %%globaltimer;\n" : "=l"(now));
    if (began == 0) began = now;
    else if (now - began > MS_WAIT_NS) return false;
  }
}
__device__ __forceinline__ int adapter_slot(const Adapters& ad, int t) {
  const int s = adapter_of(ad, t);
  return s < 0 ? NO_SLOT : s;
}
// Tokens in the order of their slots, and the groups: runs of up to eight of one slot.
template <int MOST>
struct TokenGroups {
  int slot[MOST];
  int2 token[MOST];  // in order: the token, its slot
  int2 group[MOST];  // where the group begins among them, its slot
  int count;
  bool begins[MOST];
};
// From g.slot [M], written by the calling threads (e = 0 .., at least M of them); sync: their barrier.
template <int MOST, typename Sync>
__device__ __forceinline__ void group_tokens(TokenGroups<MOST>& g, int M, int e, Sync sync) {
  sync();
  if (e < M) {
    const int s = g.slot[e];
    int before = 0, same = 0;
    for (int j = 0; j < M; ++j) {
      before += g.slot[j] < s;
      same += g.slot[j] == s && j < e;
    }
    g.token[before + same] = make_int2(e, s);
    g.begins[before + same] = s != NO_SLOT && same % 8 == 0;
  }
  sync();
  if (e < M) {
    int at = 0, all = 0;
    for (int j = 0; j < M; ++j) {
      at += j < e && g.begins[j];
      all += g.begins[j];
    }
    if (g.begins[e]) g.group[at] = make_int2(e, g.token[e].y);
    if (e == 0) g.count = all;
  }
  sync();
}
// A warp's 32 rows of B (n[i] is this lane's row 8 i + lane / 4 of them, has[i] whether there is one) times the tokens of the groups first, first + step, ..: the terms are
// added to *cell(token, i) for the lane's rows. An instruction is 16 rows and the eight tokens of a group; a group and 32 of the rank's numbers are an item, the next one's asked
// for ahead of this one's instructions. ready: called before the first of v is read. v: float32 [.., parts * rank], by the tokens of g. One warp a scheduler has nothing to hide its
// trips to shared memory behind, so an item makes few: its tokens, then all of its cells at once.
template <int PIECES, int MOST, typename Ready, typename Cell>
__device__ __forceinline__ void warp_terms(const Adapters& ad, const float* v, const TokenGroups<MOST>& g, int M, int first, int step, const int (&n)[4], const bool (&has)[4],
                                           Ready ready, Cell cell) {
  const int lane = threadIdx.x & 31, col = lane >> 2, t4 = lane & 3, numbers = ad.parts * ad.rank, rows = ad.ends[MAX_PARTS - 1];
  int part[4], low = MAX_PARTS, high = -1;  // the parts that the rows belong to: one, but where two meet
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    part[i] = has[i] ? part_of(ad, n[i]) : -1;
    if (has[i]) {
      low = min(low, part[i]);
      high = max(high, part[i]);
    }
  }
  low = __reduce_min_sync(0xffffffffu, low);
  high = __reduce_max_sync(0xffffffffu, high);
  struct Item {
    int at, slot, c0;  // the group's first token in order, its slot, the first of 32 numbers of the rank
    uint32_t b[2][2][4];
    float2 v[2][2];
  };
  const __nv_bfloat16* b_all = reinterpret_cast<const __nv_bfloat16*>(ad.b);
  for (int p = low; p <= high; ++p) {
    int next = first, c_next = 0;  // the group and the numbers that are asked for next
    auto load_b = [&](Item& it) {
      const int2 where = g.group[next];
      it.at = where.x;
      it.slot = where.y;
      it.c0 = c_next;
      c_next += 32;
      if (c_next >= ad.rank) {
        c_next = 0;
        next += step;
      }
      const __nv_bfloat16* b = b_all + (size_t)it.slot * rows * ad.rank + it.c0 + 2 * t4;
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const uint32_t* row = reinterpret_cast<const uint32_t*>(b + (size_t)n[i] * ad.rank);
#pragma unroll
        for (int k = 0; k < 2; ++k)
#pragma unroll
          for (int h = 0; h < 2; ++h)
            it.b[k][i >> 1][2 * h + (i & 1)] = part[i] == p && it.c0 + 16 * k + 8 * h < ad.rank ? row[8 * k + 4 * h] : 0u;  // (the rank is a multiple of 8)
      }
    };
    auto load_v = [&](Item& it) {
      const int2 who = it.at + col < M ? g.token[it.at + col] : make_int2(0, NO_SLOT);
      const float2* row = reinterpret_cast<const float2*>(v + (size_t)who.x * numbers + p * ad.rank + it.c0 + 2 * t4);
#pragma unroll
      for (int k = 0; k < 2; ++k)
#pragma unroll
        for (int h = 0; h < 2; ++h) it.v[k][h] = who.y == it.slot && it.c0 + 16 * k + 8 * h < ad.rank ? __ldcg(row + 8 * k + 4 * h) : make_float2(0.f, 0.f);
    };
    auto multiply = [&](const Item& it) {
      int2 who[2];
      float* to[2][4];
      float sum[2][4];
#pragma unroll
      for (int q = 0; q < 2; ++q) who[q] = it.at + 2 * t4 + q < M ? g.token[it.at + 2 * t4 + q] : make_int2(0, NO_SLOT);
#pragma unroll
      for (int q = 0; q < 2; ++q)
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          to[q][i] = cell(who[q].x, i);
          sum[q][i] = *to[q][i];
        }
      float acc[2][4] = {};
#pragma unroll
      for (int k = 0; k < 2; ++k) {
        float2 left[2] = {it.v[k][0], it.v[k][1]};  // of v behind the pieces so far
#pragma unroll
        for (int piece = 0; piece < PIECES; ++piece) {
          uint32_t b[2];
#pragma unroll
          for (int h = 0; h < 2; ++h) {
            const __nv_bfloat162 now = __floats2bfloat162_rn(left[h].x, left[h].y);
            const float2 back = __bfloat1622float2(now);
            left[h].x = fabsf(back.x) < INFINITY ? left[h].x - back.x : 0.f;  // (infinity and NaN leave nothing)
            left[h].y = fabsf(back.y) < INFINITY ? left[h].y - back.y : 0.f;
            b[h] = *reinterpret_cast<const uint32_t*>(&now);
          }
#pragma unroll
          for (int m = 0; m < 2; ++m) mma_16816(acc[m], it.b[k][m][0], it.b[k][m][1], it.b[k][m][2], it.b[k][m][3], b[0], b[1]);
        }
      }
#pragma unroll
      for (int q = 0; q < 2; ++q)
        if (who[q].y == it.slot) {
#pragma unroll
          for (int i = 0; i < 4; ++i) *to[q][i] = sum[q][i] + acc[i >> 1][2 * (i & 1) + q];
        }
    };
    if (next >= g.count) return;
    Item a, b;
    load_b(a);
    if (p == low) ready();
    load_v(a);
    for (;;) {
      const bool more = next < g.count;
      if (more) {
        load_b(b);
        load_v(b);
      }
      multiply(a);
      if (!more) break;
      const bool again = next < g.count;
      if (again) {
        load_b(a);
        load_v(a);
      }
      multiply(b);
      if (!again) break;
    }
  }
}

}  // namespace ms
