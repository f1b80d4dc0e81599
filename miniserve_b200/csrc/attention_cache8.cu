// Attention over the paged cache in 8 bits (cache8.cuh), compiled for ONE head size (-DMS_HEAD_DIM=D, a multiple of 16 up to 256): keys
// split over warps and CTAs.
//
// Formula: softmax(scale q k^T + causal mask) v; query head h reads kv head h / (heads / kv_heads), the query at position p sees keys 0..p or
// the last `window` of them, a sink adds exp(0) to the denominator (miniserve/model/attention.py:60-67, 125-133).
//
// A CTA takes 16 query rows (consecutive tokens of a request times the query heads of one kv head) and a share of their keys; its four warps
// take 16-key slices in turn. Codes become float16 (exact: e4m3 has 4 significant bits) and both products run on mma.sync with float32 sums:
//   s_j = (q' . code_j) * qf * 2^ek_j,          q' = q * 2^sh in float16, with sh so that the row's largest |q'| lies in [2^14, 2^15): q's 8
//                                               significant bits are kept down to 2^-29 of the largest; qf = scale * log2(e) * 2^-sh
//   m = max_j (s_j + ev_j) - 14                 running, over scores and the values' exponents together
//   o = sum_j 2^(s_j + ev_j - m) code(v_j),     l = sum_j 2^(s_j - m)
// so a weight with its value's scale is at most 2^14, a float16 with 11 significant bits down to 2^-28 of the largest; l and o are float32.
#include "cache8.cuh"

#ifndef MS_HEAD_DIM
#error "compile with -DMS_HEAD_DIM=<head size>"
#endif

namespace ms {

constexpr int D = MS_HEAD_DIM;
static_assert(D % 16 == 0 && D >= 16 && D <= 256, "head size must be a multiple of 16 up to 256");
constexpr int CHUNKS = D / 16;                       // 16-byte chunks of a row of codes
constexpr int KSTEPS = D / 16, DTILES = D / 8;
constexpr int WIDE = D / 64, REST = (D % 64) / 16;   // k-steps of q k^T whose codes come four by four, and one by one
constexpr int VB = D % 128 == 0 ? 16 : (D % 64 == 0 ? 8 : 4), VBLOCKS = D / (8 * VB), VTAIL = D % 32 / 16;  // how a lane reads values: VB bytes a block
constexpr int QPAD = D + 8;                          // float16 row stride of q in shared memory
constexpr bool Q_IN_REGS = D <= 128;
constexpr float LOG2E = 1.4426950408889634f;
constexpr int SLICE = 16, WARPS = 4, THREADS = WARPS * 32, STAGES = 3, ROWS = 16;
constexpr int ROW_BYTES = D % 64 == 0 ? D : D + 16;
constexpr int STAGE_BYTES = 2 * SLICE * ROW_BYTES + 2 * SLICE;  // K codes, V codes, K exponents, V exponents
static_assert(STAGE_BYTES % 16 == 0, "");

__device__ __forceinline__ uint32_t smem_addr(const void* p) { return (uint32_t)__cvta_generic_to_shared(p); }
__device__ __forceinline__ void cp_async16(uint32_t dst, const void* src, bool valid) {
  const int n = valid ? 16 : 0;  // 0: zero-filled, nothing is read
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;\n" ::"r"(dst), "l"(src), "r"(n));
}
__device__ __forceinline__ void cp_async8(uint32_t dst, const void* src, bool valid) {
  const int n = valid ? 8 : 0;
  asm volatile("cp.async.ca.shared.global [%0], [%1], 8, %2;\n" ::"r"(dst), "l"(src), "r"(n));
}
__device__ __forceinline__ void cp_async_commit() { asm volatile("cp.async.commit_group;\n" ::); }
template <int N>
__device__ __forceinline__ void cp_async_wait() { asm volatile("cp.async.wait_group %0;\n" ::"n"(N)); }
__device__ __forceinline__ void mma_f16(float (&c)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
  asm volatile(
      "mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};\n"
      : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
      : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
__device__ __forceinline__ uint32_t pack_half2(float lo, float hi) {
  __half2 v = __floats2half2_rn(lo, hi);
  return *reinterpret_cast<uint32_t*>(&v);
}
__device__ __forceinline__ float quad_max(float v) {
  v = fmaxf(v, __shfl_xor_sync(0xffffffffu, v, 1));
  return fmaxf(v, __shfl_xor_sync(0xffffffffu, v, 2));
}
__device__ __forceinline__ float quad_sum(float v) {
  v += __shfl_xor_sync(0xffffffffu, v, 1);
  return v + __shfl_xor_sync(0xffffffffu, v, 2);
}
__device__ __forceinline__ uint32_t lds32(uint32_t at) {
  uint32_t v;
  asm volatile("ld.shared.u32 %0, [%1];\n" : "=r"(v) : "r"(at));
  return v;
}
__device__ __forceinline__ uint32_t lds16(uint32_t at) {
  uint16_t v;
  asm volatile("ld.shared.u16 %0, [%1];\n" : "=h"(v) : "r"(at));
  return v;
}
__device__ __forceinline__ uint32_t lds8(uint32_t at) {
  uint32_t v;
  asm volatile("ld.shared.u8 %0, [%1];\n" : "=r"(v) : "r"(at));
  return v;
}
template <int BYTES>
__device__ __forceinline__ void lds_words(uint32_t (&v)[BYTES / 4], uint32_t at) {
  if constexpr (BYTES == 16) asm volatile("ld.shared.v4.u32 {%0,%1,%2,%3}, [%4];\n" : "=r"(v[0]), "=r"(v[1]), "=r"(v[2]), "=r"(v[3]) : "r"(at));
  if constexpr (BYTES == 8) asm volatile("ld.shared.v2.u32 {%0,%1}, [%2];\n" : "=r"(v[0]), "=r"(v[1]) : "r"(at));
  if constexpr (BYTES == 4) v[0] = lds32(at);
}

// Where chunk `chunk` of row `row` of a slice lies. Head sizes of whole 128s and 64 swizzle their chunks so that neither the reads of keys (8 rows,
// 4 lanes a row) nor those of values (4 rows of every second, the lanes of a row side by side) meet in a bank.
__device__ __forceinline__ uint32_t chunk_at(int row, int chunk) {
  if (D % 128 == 0) return row * ROW_BYTES + ((chunk ^ (row & 7)) << 4);
  if (D == 64) return (row >> 1) * 128 + ((((row & 1) * 4 + chunk) ^ (2 * ((row >> 1) & 3))) << 4);
  return row * ROW_BYTES + (chunk << 4);
}
// The number of the head's channels that lane t of a quad takes in k-step `kk` of q k^T: 4 from here on. (The order of the channels is free: queries
// are read in the same one.)
__device__ __forceinline__ int channel_of(int kk, int t) {
  if (kk < WIDE * 4) {
    const int grp = kk >> 2, w = kk & 3;
    const int chunk = D % 128 == 0 ? (grp >> 1) * 8 + 2 * t + (grp & 1) : grp * 4 + t;
    return chunk * 16 + w * 4;
  }
  return kk * 16 + 4 * t;
}

struct Split8 {
  const int* cu_q;          // [rows + 1]
  const int* q_start;       // [rows]
  const int* page_indptr;   // [rows + 1]
  const int* page_indices;
  int* status;
  float* part_o;            // splits > 1: [item][split][16][D] and [item][split][16][2], an item a (row, tile, kv head)
  float* part_ml;
  int* counters;            // [items], zero before the first launch, left zero by every launch
  int rows, tiles;          // tiles of 16 query rows a request has at most
  int nq, nkv, window, sink, page_size, splits;
  float scale;
  int num_pages;
};

// One slice (16 keys from key0 on) on its way into a stage; keys outside [lo, hi), and those of pages that the table or the pool does not have, are zeros.
__device__ __forceinline__ void load_slice(uint32_t st, const uint8_t* k_codes, const uint8_t* k_exps, const uint8_t* v_codes, const uint8_t* v_exps,
                                           const int* pages, int entries, const Split8& p, int kvh, int page_shift, int key0, int lo, int hi, int lane) {
  // lanes 0 and 1: the pages of the slice's two halves of 8 keys
  long long base = -1;  // row of the pool that the half's first key lies in
  if (lane < 2) {
    const int key = key0 + 8 * lane;
    if (key + 8 > lo && key < hi) {
      const int entry = key >> page_shift, page = entry < entries ? pages[entry] : -1;
      if (page >= 0 && page < p.num_pages)
        base = (((long long)page * p.nkv + kvh) << page_shift) + (key & ((1 << page_shift) - 1));
      else
        atomicExch(p.status, 2);
    }
  }
  const long long base0 = __shfl_sync(0xffffffffu, base, 0), base1 = __shfl_sync(0xffffffffu, base, 1);
#pragma unroll
  for (int idx = lane; idx < SLICE * CHUNKS; idx += 32) {
    const int row = idx / CHUNKS, chunk = idx - row * CHUNKS;
    const long long b = row < 8 ? base0 : base1;
    const bool valid = b >= 0 && key0 + row >= lo && key0 + row < hi;
    const size_t off = valid ? (size_t)(b + (row & 7)) * D + chunk * 16 : 0;
    cp_async16(st + chunk_at(row, chunk), k_codes + off, valid);
    cp_async16(st + SLICE * ROW_BYTES + chunk_at(row, chunk), v_codes + off, valid);
  }
  if (lane < 4) {  // exponents, 8 at a time
    const long long b = (lane & 1) ? base1 : base0;
    const uint8_t* src = lane < 2 ? k_exps : v_exps;
    cp_async8(st + 2 * SLICE * ROW_BYTES + lane * 8, src + (b >= 0 ? b : 0), b >= 0);
  }
}

__global__ void __launch_bounds__(THREADS)
attn_cache8_split_kernel(__nv_bfloat16* __restrict__ out, const __nv_bfloat16* __restrict__ q, const uint8_t* __restrict__ k_codes,
                         const uint8_t* __restrict__ k_exps, const uint8_t* __restrict__ v_codes, const uint8_t* __restrict__ v_exps, const Split8 p) {
  const int *cu_q = p.cu_q, *q_start = p.q_start, *page_indptr = p.page_indptr, *page_indices = p.page_indices;
  pdl_prologue(q, k_codes, k_exps, v_codes, v_exps, cu_q, q_start, page_indptr, page_indices);
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, g = lane >> 2, t = lane & 3;
  const int kvh = blockIdx.y, group = p.nq / p.nkv;
  const int split = blockIdx.x % p.splits, place = blockIdx.x / p.splits, r = place / p.tiles, tile = place - r * p.tiles;
  const int tok0 = cu_q[r], rows_all = (cu_q[r + 1] - tok0) * group;
  const int row0 = tile * ROWS;
  if (row0 >= rows_all) return;
  const int rows_here = min(ROWS, rows_all - row0), start = q_start[r];
  const int q_first = start + row0 / group, q_last = start + (row0 + rows_here - 1) / group;
  const int lo = p.window > 0 ? max(0, q_first - p.window + 1) : 0, hi = q_last + 1;
  const int first_slice = lo / SLICE, end_slice = (hi + SLICE - 1) / SLICE;
  const int per_split = (end_slice - first_slice + p.splits - 1) / p.splits;
  const int s_begin = first_slice + split * per_split, s_end = min(end_slice, s_begin + per_split);
  const int page_shift = 31 - __clz(p.page_size);
  const int* pages = page_indices + page_indptr[r];
  const int entries = page_indptr[r + 1] - page_indptr[r];

  extern __shared__ __align__(128) unsigned char smem_raw[];
  __half* qs = reinterpret_cast<__half*>(smem_raw);
  __shared__ float q_factor[ROWS];
  const uint32_t pipe = smem_addr(smem_raw) + (ROWS * QPAD * 2 + 127) / 128 * 128 + warp * ((STAGES * STAGE_BYTES + 127) / 128 * 128);

  const int my_first = s_begin + warp, my_count = my_first < s_end ? (s_end - my_first + WARPS - 1) / WARPS : 0;
  auto issue = [&](int i) {
    if (i < my_count)
      load_slice(pipe + (i % STAGES) * STAGE_BYTES, k_codes, k_exps, v_codes, v_exps, pages, entries, p, kvh, page_shift, (my_first + i * WARPS) * SLICE, lo, hi, lane);
    cp_async_commit();
  };
#pragma unroll
  for (int i = 0; i < STAGES - 1; ++i) issue(i);

  // queries: four rows a warp, to float16 with the row's own power of two
  for (int i = warp; i < ROWS; i += WARPS) {
    float x[D / 32 + 1];
    float most = 0.f;
    const int row = row0 + i, tok = row / group;
    const __nv_bfloat16* src = q + ((size_t)(tok0 + tok) * p.nq + kvh * group + (row - tok * group)) * D;
#pragma unroll
    for (int c = 0; c < D / 32 + 1; ++c) {
      const int ch = c * 32 + lane;
      x[c] = i < rows_here && ch < D ? __bfloat162float(src[ch]) : 0.f;
      most = fmaxf(most, fabsf(x[c]));
    }
    most = warp_max(most);
    const int field = (__float_as_uint(most) >> 23) & 255;
    const int sh = most > 0.f && field < 255 ? min(max(14 + 127 - field, -113), 100) : 0;
    const float up = __uint_as_float((uint32_t)(127 + sh) << 23);
#pragma unroll
    for (int c = 0; c < D / 32 + 1; ++c) {
      const int ch = c * 32 + lane;
      if (ch < D) qs[i * QPAD + ch] = __float2half_rn(x[c] * up);
    }
    if (lane == 0) q_factor[i] = p.scale * LOG2E * __uint_as_float((uint32_t)(127 - sh) << 23);
  }
  __syncthreads();
  auto load_q = [&](uint32_t (&a)[4], int kk) {
    const int ch = channel_of(kk, t);
    const uint2 top = *reinterpret_cast<const uint2*>(qs + g * QPAD + ch), low = *reinterpret_cast<const uint2*>(qs + (g + 8) * QPAD + ch);
    a[0] = top.x; a[1] = low.x; a[2] = top.y; a[3] = low.y;
  };
  uint32_t qf[Q_IN_REGS ? KSTEPS : 1][4];
  if (Q_IN_REGS) {
#pragma unroll
    for (int kk = 0; kk < (Q_IN_REGS ? KSTEPS : 1); ++kk) load_q(qf[kk], kk);
  }
  const float row_factor[2] = {q_factor[g], q_factor[g + 8]};
  const int q_pos[2] = {start + (row0 + g) / group, start + (row0 + g + 8) / group};

  float o[DTILES][4];
#pragma unroll
  for (int i = 0; i < DTILES; ++i) o[i][0] = o[i][1] = o[i][2] = o[i][3] = 0.f;
  float m_run[2] = {-INFINITY, -INFINITY}, l_run[2] = {0.f, 0.f};

  for (int i = 0; i < my_count; ++i) {
    issue(i + STAGES - 1);
    cp_async_wait<STAGES - 1>();
    __syncwarp();
    const uint32_t st = pipe + (i % STAGES) * STAGE_BYTES, vt = st + SLICE * ROW_BYTES, et = st + 2 * SLICE * ROW_BYTES;
    const int key0 = (my_first + i * WARPS) * SLICE;
    float s[2][4] = {{0.f, 0.f, 0.f, 0.f}, {0.f, 0.f, 0.f, 0.f}};
#pragma unroll
    for (int grp = 0; grp < WIDE; ++grp) {
      uint32_t kw[2][4];
      const int chunk = channel_of(grp * 4, t) >> 4;
      lds_words<16>(kw[0], st + chunk_at(g, chunk));
      lds_words<16>(kw[1], st + chunk_at(g + 8, chunk));
#pragma unroll
      for (int w = 0; w < 4; ++w) {
        uint32_t a[4];
        if (Q_IN_REGS) {
          const int kk = grp * 4 + w;
          a[0] = qf[kk][0]; a[1] = qf[kk][1]; a[2] = qf[kk][2]; a[3] = qf[kk][3];
        } else {
          load_q(a, grp * 4 + w);
        }
#pragma unroll
        for (int n = 0; n < 2; ++n) mma_f16(s[n], a, c8_half2_lo(kw[n][w]), c8_half2_hi(kw[n][w]));
      }
    }
#pragma unroll
    for (int rest = 0; rest < REST; ++rest) {
      const int kk = WIDE * 4 + rest;
      uint32_t a[4];
      if (Q_IN_REGS) {
        const int at = Q_IN_REGS ? kk : 0;
        a[0] = qf[at][0]; a[1] = qf[at][1]; a[2] = qf[at][2]; a[3] = qf[at][3];
      } else {
        load_q(a, kk);
      }
#pragma unroll
      for (int n = 0; n < 2; ++n) {
        const uint32_t w = lds32(st + chunk_at(g + 8 * n, kk) + 4 * t);
        mma_f16(s[n], a, c8_half2_lo(w), c8_half2_hi(w));
      }
    }
    // mask, then the running softmax of rows g and g + 8
    float kf[4], ev[4];
#pragma unroll
    for (int n = 0; n < 2; ++n) {
      const uint32_t kb = lds16(et + n * 8 + 2 * t), vb = lds16(et + SLICE + n * 8 + 2 * t);
      kf[2 * n] = c8_factor(kb & 255);
      kf[2 * n + 1] = c8_factor(kb >> 8);
      ev[2 * n] = (vb & 255) == C8_NAN ? __uint_as_float(0x7FFFFFFFu) : (float)((int)(vb & 255) - 127);
      ev[2 * n + 1] = (vb >> 8) == C8_NAN ? __uint_as_float(0x7FFFFFFFu) : (float)((int)(vb >> 8) - 127);
    }
    bool ok[2][4];
    float m_new[2] = {m_run[0], m_run[1]};
#pragma unroll
    for (int n = 0; n < 2; ++n)
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        const int key = key0 + n * 8 + 2 * t + (e & 1), qp = q_pos[e >> 1];
        ok[n][e] = key <= qp && (p.window <= 0 || key > qp - p.window);
        s[n][e] = s[n][e] * row_factor[e >> 1] * kf[2 * n + (e & 1)];
        if (ok[n][e]) m_new[e >> 1] = fmaxf(m_new[e >> 1], s[n][e] + ev[2 * n + (e & 1)]);
      }
    float alpha[2], m_use[2], row_sum[2] = {0.f, 0.f};
#pragma unroll
    for (int j = 0; j < 2; ++j) {
      m_new[j] = quad_max(m_new[j]);
      m_use[j] = m_new[j] == -INFINITY ? 0.f : m_new[j] - 14.f;
      alpha[j] = m_run[j] == -INFINITY ? 0.f : exp2f(m_run[j] - m_new[j]);
      m_run[j] = m_new[j];
    }
    uint32_t a[4];
    float weight[2][4];
#pragma unroll
    for (int n = 0; n < 2; ++n)
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        const float x = s[n][e] - m_use[e >> 1];
        row_sum[e >> 1] += ok[n][e] ? exp2f(x) : 0.f;
        weight[n][e] = ok[n][e] ? exp2f(x + ev[2 * n + (e & 1)]) : 0.f;
      }
#pragma unroll
    for (int j = 0; j < 2; ++j) l_run[j] = l_run[j] * alpha[j] + row_sum[j];
    a[0] = pack_half2(weight[0][0], weight[0][1]);
    a[1] = pack_half2(weight[0][2], weight[0][3]);
    a[2] = pack_half2(weight[1][0], weight[1][1]);
    a[3] = pack_half2(weight[1][2], weight[1][3]);
    if (__any_sync(0xffffffffu, alpha[0] != 1.f || alpha[1] != 1.f)) {
#pragma unroll
      for (int dt = 0; dt < DTILES; ++dt) {
        o[dt][0] *= alpha[0]; o[dt][1] *= alpha[0]; o[dt][2] *= alpha[1]; o[dt][3] *= alpha[1];
      }
    }
    // values: lane group g's channels of the rows 2t, 2t + 1, 2t + 8, 2t + 9, paired along the keys byte by byte
#pragma unroll
    for (int blk = 0; blk < VBLOCKS; ++blk) {
      uint32_t vw[4][VB / 4];
      const int ch = blk * 8 * VB + g * VB;
#pragma unroll
      for (int j = 0; j < 4; ++j) lds_words<VB>(vw[j], vt + chunk_at(2 * t + (j & 1) + 8 * (j >> 1), ch >> 4) + (ch & 15));
#pragma unroll
      for (int w = 0; w < VB / 4; ++w) {
        const uint32_t b0 = __byte_perm(vw[0][w], vw[1][w], 0x5140), b1 = __byte_perm(vw[2][w], vw[3][w], 0x5140);
        const uint32_t c0 = __byte_perm(vw[0][w], vw[1][w], 0x7362), c1 = __byte_perm(vw[2][w], vw[3][w], 0x7362);
        const int dt = blk * VB + w * 4;
        mma_f16(o[dt], a, c8_half2_lo(b0), c8_half2_lo(b1));
        mma_f16(o[dt + 1], a, c8_half2_hi(b0), c8_half2_hi(b1));
        mma_f16(o[dt + 2], a, c8_half2_lo(c0), c8_half2_lo(c1));
        mma_f16(o[dt + 3], a, c8_half2_hi(c0), c8_half2_hi(c1));
      }
    }
    if (VTAIL) {
      const int ch = VBLOCKS * 8 * VB + 2 * g;
      uint32_t vw[4];
#pragma unroll
      for (int j = 0; j < 4; ++j) vw[j] = lds16(vt + chunk_at(2 * t + (j & 1) + 8 * (j >> 1), ch >> 4) + (ch & 15));
      const uint32_t b0 = __byte_perm(vw[0], vw[1], 0x5140), b1 = __byte_perm(vw[2], vw[3], 0x5140);
      mma_f16(o[DTILES - 2], a, c8_half2_lo(b0), c8_half2_lo(b1));
      mma_f16(o[DTILES - 1], a, c8_half2_hi(b0), c8_half2_hi(b1));
    }
    __syncwarp();
  }
  cp_async_wait<0>();
#pragma unroll
  for (int j = 0; j < 2; ++j) l_run[j] = quad_sum(l_run[j]);
  __syncthreads();  // the pipelines are drained: shared memory becomes the merge area [warps][16][D + 2]

  float* merge = reinterpret_cast<float*>(smem_raw);
#pragma unroll
  for (int j = 0; j < 2; ++j) {
    float* row = merge + ((size_t)warp * ROWS + g + 8 * j) * (D + 2);
#pragma unroll
    for (int dt = 0; dt < DTILES; ++dt)
#pragma unroll
      for (int c = 0; c < 2; ++c) {
        const int from = 2 * t + c;  // the lane group whose channels this column is
        const int ch = dt < VBLOCKS * VB ? (dt / VB) * 8 * VB + from * VB + dt % VB : VBLOCKS * 8 * VB + 2 * from + (dt - VBLOCKS * VB);
        row[ch] = o[dt][2 * j + c];
      }
    if (t == 0) {
      row[D] = m_run[j];
      row[D + 1] = l_run[j];
    }
  }
  __syncthreads();
  const size_t item = (size_t)place * p.nkv + kvh;
  auto store = [&](int row, int c, float acc, float l, float m) {
    if (p.sink) l += exp2f(14.f - m);  // (the sums are in units of 2^(m - 14))
    const int rho = row0 + row, tok = rho / group;
    out[((size_t)(tok0 + tok) * p.nq + kvh * group + (rho - tok * group)) * D + c] = __float2bfloat16_rn(l == 0.f ? 0.f : acc / l);
  };
  for (int idx = tid; idx < rows_here * D; idx += THREADS) {
    const int row = idx / D, c = idx - row * D;
    float m = -INFINITY;
#pragma unroll
    for (int w = 0; w < WARPS; ++w) m = fmaxf(m, merge[((size_t)w * ROWS + row) * (D + 2) + D]);
    float acc = 0.f, l = 0.f;
#pragma unroll
    for (int w = 0; w < WARPS; ++w) {
      const float* src = merge + ((size_t)w * ROWS + row) * (D + 2);
      const float wgt = src[D] == -INFINITY ? 0.f : exp2f(src[D] - m);
      acc += wgt * src[c];
      l += wgt * src[D + 1];
    }
    if (p.splits == 1) {
      store(row, c, acc, l, m);
    } else {
      const size_t at = (item * p.splits + split) * ROWS + row;
      p.part_o[at * D + c] = acc;
      if (c == 0) {
        p.part_ml[2 * at] = m;
        p.part_ml[2 * at + 1] = l;
      }
    }
  }
  if (p.splits == 1) return;
  // the split that finishes last adds them all up (a ticket; nobody waits)
  __shared__ int last_one;
  __threadfence();
  __syncthreads();
  if (tid == 0) {
    const int prev = atomicAdd(p.counters + item, 1);
    last_one = prev == p.splits - 1;
    if (last_one) p.counters[item] = 0;
  }
  __syncthreads();
  if (!last_one) return;
  __threadfence();
  for (int idx = tid; idx < rows_here * D; idx += THREADS) {
    const int row = idx / D, c = idx - row * D;
    float m = -INFINITY, acc = 0.f, l = 0.f;
    for (int sp = 0; sp < p.splits; ++sp) m = fmaxf(m, __ldcg(p.part_ml + 2 * ((item * p.splits + sp) * ROWS + row)));
    for (int sp = 0; sp < p.splits; ++sp) {
      const size_t at = (item * p.splits + sp) * ROWS + row;
      const float ms = __ldcg(p.part_ml + 2 * at), wgt = ms == -INFINITY ? 0.f : exp2f(ms - m);
      acc += wgt * __ldcg(p.part_o + at * D + c);
      l += wgt * __ldcg(p.part_ml + 2 * at + 1);
    }
    store(row, c, acc, l, m);
  }
}

}  // namespace ms

using namespace ms;

#define MS_CAT2(a, b) a##b
#define MS_CAT(a, b) MS_CAT2(a, b)
#define MS_ATTN8_FN(name) MS_CAT(MS_CAT(MS_CAT(ms_attn_cache8_d, MS_HEAD_DIM), _), name)

MS_DEFINE_LAST_ERROR(MS_ATTN8_FN(last_error))
MS_DEFINE_PDL_SWITCH(MS_ATTN8_FN(set_pdl))

static constexpr size_t split_smem() {
  const size_t pipe = (ROWS * QPAD * 2 + 127) / 128 * 128 + (size_t)WARPS * ((STAGES * STAGE_BYTES + 127) / 128 * 128);
  const size_t merge = (size_t)WARPS * ROWS * (D + 2) * 4;
  return pipe > merge ? pipe : merge;
}

// Rows [0, p->rows) of the geometry in p. Scratch and counters (splits > 1): see Split8.
MS_EXPORT int MS_ATTN8_FN(split)(const Split8* p, void* out, const void* q, const void* k_codes, const void* k_exps, const void* v_codes, const void* v_exps,
                                 cudaStream_t stream) {
  if (p->rows == 0) return 0;
  MS_CHECK_ARG(p->nq > 0 && p->nkv > 0 && p->nq % p->nkv == 0, "attention: %d query heads are not a multiple of %d kv heads", p->nq, p->nkv);
  MS_CHECK_ARG(p->page_size >= 8 && (p->page_size & (p->page_size - 1)) == 0, "attention: page_size=%d must be a power of two from 8 on for an 8-bit cache", p->page_size);
  MS_CHECK_ARG(p->rows > 0 && p->tiles > 0 && p->splits > 0 && (long long)p->rows * p->tiles * p->splits < (1LL << 31) && p->nkv <= 65535,
               "attention: %d rows of %d tiles, %d splits, %d kv heads are too many for one launch", p->rows, p->tiles, p->splits, p->nkv);
  MS_CHECK_ARG(p->splits == 1 || (p->part_o && p->part_ml && p->counters), "attention: splits need scratch memory");
  MS_CHECK_ARG((uintptr_t)q % 16 == 0 && (uintptr_t)k_codes % 16 == 0 && (uintptr_t)v_codes % 16 == 0 && (uintptr_t)k_exps % 8 == 0 && (uintptr_t)v_exps % 8 == 0,
               "attention: an 8-bit cache's tensors must be 16-byte aligned");
  static bool configured[64] = {};  // the attribute belongs to a device
  int dev = 0;
  MS_CHECK_CUDA(cudaGetDevice(&dev));
  MS_CHECK_ARG(dev >= 0 && dev < 64, "attention: device index %d is not supported", dev);
  if (!configured[dev]) {
    MS_CHECK_CUDA(cudaFuncSetAttribute(attn_cache8_split_kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)split_smem()));
    configured[dev] = true;
  }
  MS_LAUNCH(attn_cache8_split_kernel, dim3((unsigned)(p->rows * p->tiles * p->splits), p->nkv), THREADS, split_smem(), stream, (__nv_bfloat16*)out,
            (const __nv_bfloat16*)q, (const uint8_t*)k_codes, (const uint8_t*)k_exps, (const uint8_t*)v_codes, (const uint8_t*)v_exps, *p);
  return 0;
}
