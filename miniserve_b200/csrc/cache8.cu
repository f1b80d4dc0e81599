// Writing the 8-bit paged cache and reading it back (the format: cache8.cuh).
//
// The write is the step between the q|k|v product and attention: per-head RMSNorm of q and k, rotation of halves, queries out in
// bfloat16, keys (behind norm and rotation) and values quantised from float32 into their pages: one rounding, to the code.
// Formulas of the norm and the rotation: miniserve/model/qwen3.py:98-108, 118-123; the reference keeps its cache in the model's
// type (miniserve/cache/kv_pool.py:46-50).
#include "cache8.cuh"

namespace ms {

constexpr int C8_MAX_D = 256;

// A step's page tables: `rows` of them in page_indices [entries], entry 0 of row r at page_indptr[r]. Where a window gave pages back that place can lie ahead of the
// tables or inside another row's entries (csrc/host_core.cpp, the step packer), so that neighbouring places do not tell a row's length: what bounds it is the end of all.
struct Tables8 {
  const int *page_indptr, *page_indices;
  int rows, entries;
  // Where they end: asked for early, so that nothing waits for it behind the row and its beginning. (Of a page_indptr with room for more rows than there are the next row's
  // beginning still says so of whole tables.)
  __device__ __forceinline__ int end() const { return page_indptr[rows]; }
  // The page of position `pos` of request `row`; negative where the tables have none, or none that the pool has.
  __device__ __forceinline__ int page(int row, int pos, int end, int page_shift, int num_pages) const {
    if ((unsigned)row >= (unsigned)rows || pos < 0) return -1;
    const int at = page_indptr[row] + (pos >> page_shift), next = page_indptr[row + 1];
    const int page = at >= 0 && at < entries ? page_indices[at] : -1;  // (asked for before the end is known)
    return at < max(end, next) && page < num_pages ? page : -1;
  }
};

// A warp per (token, head).
__global__ void __launch_bounds__(256)
cache8_write_kernel(__nv_bfloat16* __restrict__ q_out, uint8_t* __restrict__ k_codes, uint8_t* __restrict__ k_exps, uint8_t* __restrict__ v_codes,
                    uint8_t* __restrict__ v_exps, const __nv_bfloat16* __restrict__ qkv, const __nv_bfloat16* __restrict__ q_norm_w,
                    const __nv_bfloat16* __restrict__ k_norm_w, const float* __restrict__ inv_freq, const float* __restrict__ cos_sin,
                    const int* __restrict__ positions, const int* __restrict__ row_of_token, Tables8 tables, int num_tokens, int nq, int nkv, int d, int rot, float eps, int page_shift, int num_pages,
                    int* __restrict__ status) {
  pdl_prologue(qkv, q_norm_w, k_norm_w, inv_freq, cos_sin, positions, row_of_token, tables.page_indptr, tables.page_indices);
  __shared__ float held[8][C8_MAX_D];
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, heads = nq + 2 * nkv;
  const long long item = (long long)blockIdx.x * 8 + warp;
  if (item >= (long long)num_tokens * heads) return;
  const int t = (int)(item / heads), h = (int)(item - (long long)t * heads);
  const __nv_bfloat16* src = qkv + ((size_t)t * heads + h) * d;
  const bool is_q = h < nq, is_v = h >= nq + nkv;
  const int pos = positions[t];
  float* x = held[warp];
  float ss = 0.f;
  for (int c = lane; c < d; c += 32) {
    x[c] = __bfloat162float(src[c]);
    ss += x[c] * x[c];
  }
  const __nv_bfloat16* nw = is_v ? nullptr : (is_q ? q_norm_w : k_norm_w);
  if (nw) {
    const float inv = 1.0f / sqrtf(warp_sum(ss) / (float)d + eps);
    for (int c = lane; c < d; c += 32) x[c] = (x[c] * inv) * __bfloat162float(nw[c]);
  }
  __syncwarp();
  if (!is_v && inv_freq) {
    const int half = rot >> 1;
    for (int j = lane; j < half; j += 32) {
      float sn, cs;
      if (cos_sin) {
        cs = cos_sin[(size_t)t * rot + j];
        sn = cos_sin[(size_t)t * rot + half + j];
      } else {
        sincosf((float)pos * inv_freq[j], &sn, &cs);
      }
      const float lo = x[j], hi = x[j + half];
      x[j] = lo * cs - hi * sn;
      x[j + half] = hi * cs + lo * sn;
    }
    __syncwarp();
  }
  if (is_q) {
    __nv_bfloat16* dst = q_out + ((size_t)t * nq + h) * d;
    for (int c = lane; c < d; c += 32) dst[c] = __float2bfloat16_rn(x[c]);
    return;
  }
  const int page = tables.page(row_of_token[t], pos, tables.end(), page_shift, num_pages);
  if (page < 0) {
    if (lane == 0) atomicExch(status, 2);
    return;
  }
  uint32_t amax = 0;
  for (int c = lane; c < d; c += 32) amax = max(amax, __float_as_uint(x[c]) & 0x7FFFFFFFu);
  const int b = c8_exponent(__reduce_max_sync(0xffffffffu, amax));
  const float inv = c8_inverse(b);
  const size_t at = ((size_t)page * nkv + (h - nq) % nkv) * ((size_t)1 << page_shift) + (pos & ((1 << page_shift) - 1));
  uint32_t* codes = reinterpret_cast<uint32_t*>((is_v ? v_codes : k_codes) + at * d);
  for (int c = lane; c < d / 4; c += 32)
    codes[c] = c8_keep(c8_codes4(x[4 * c] * inv, x[4 * c + 1] * inv, x[4 * c + 2] * inv, x[4 * c + 3] * inv), b);
  if (lane == 0) (is_v ? v_exps : k_exps)[at] = (uint8_t)b;
}

__device__ __forceinline__ void c8_float4(float (&f)[4], const uint2& v) {  // of bfloat16
  f[0] = __uint_as_float(v.x << 16);
  f[1] = __uint_as_float(v.x & 0xFFFF0000u);
  f[2] = __uint_as_float(v.y << 16);
  f[3] = __uint_as_float(v.y & 0xFFFF0000u);
}
__device__ __forceinline__ uint2 c8_bf16x4(const float (&f)[4]) {
  __nv_bfloat162 a = __floats2bfloat162_rn(f[0], f[1]), b = __floats2bfloat162_rn(f[2], f[3]);
  return make_uint2(*reinterpret_cast<uint32_t*>(&a), *reinterpret_cast<uint32_t*>(&b));
}

// Head sizes 64, 128 and 256 rotated whole or not at all: a block per token, D / 8 lanes per head. A lane holds 4 numbers of the head's first half and the 4 of the second that
// rotate with them; a head's lanes exchange a sum of squares and a maximum. What hangs on the token alone is fetched once a lane, and its first numbers before the
// page is looked up (three loads, one behind the other); a further trip's are asked for ahead of the work on the last. Bound by those chains, not by bytes: written and read back
// (cache8_read_kernel), 2,048 tokens of 48 heads take 17.8 us (56 MB: 8.5 us at the rate of a copy), 777 tokens of 40 heads of 64 6.4; without the loads ahead the first take 19.5, with
// five blocks a multiprocessor 17.2 and 7.1.
// TABLE: the angles' cosines and sines are given, or nothing is rotated (the form that makes them itself needs more registers).
template <int D, bool TABLE>
__global__ void __launch_bounds__(256, TABLE ? 4 : 1)
cache8_write_token_kernel(__nv_bfloat16* __restrict__ q_out, uint8_t* __restrict__ k_codes, uint8_t* __restrict__ k_exps, uint8_t* __restrict__ v_codes,
                          uint8_t* __restrict__ v_exps, const __nv_bfloat16* __restrict__ qkv, const __nv_bfloat16* __restrict__ q_norm_w,
                          const __nv_bfloat16* __restrict__ k_norm_w, const float* __restrict__ inv_freq, const float* __restrict__ cos_sin,
                          const int* __restrict__ positions, const int* __restrict__ row_of_token, Tables8 tables, int nq, int nkv, float eps, int page_shift, int num_pages, int* __restrict__ status) {
  pdl_prologue(qkv, q_norm_w, k_norm_w, inv_freq, cos_sin, positions, row_of_token, tables.page_indptr, tables.page_indices);
  constexpr int LPH = D / 8, HPW = 32 / LPH, HALF = D / 2, BATCH = 2;
  const int t = blockIdx.x, warp = threadIdx.x >> 5, lane = threadIdx.x & 31, sub = lane % LPH, slot = lane / LPH, j0 = sub * 4;
  const int heads = nq + 2 * nkv, stride = (int)(blockDim.x >> 5) * HPW;  // heads a pass
  const __nv_bfloat16* row_in = qkv + (size_t)t * heads * D + j0;
  uint2 lo_raw[BATCH], hi_raw[BATCH];
  auto fetch = [&](int base) {
#pragma unroll
    for (int b = 0; b < BATCH; ++b) {
      const __nv_bfloat16* src = row_in + (size_t)min(base + warp * HPW + slot + b * stride, heads - 1) * D;  // past the end: the last head again, unused
      lo_raw[b] = *reinterpret_cast<const uint2*>(src);
      hi_raw[b] = *reinterpret_cast<const uint2*>(src + HALF);
    }
  };
  const int pos = positions[t], request = row_of_token[t], tables_end = tables.end();
  fetch(0);
  const bool normed = q_norm_w != nullptr;
  uint2 wq_lo = make_uint2(0u, 0u), wq_hi = wq_lo, wk_lo = wq_lo, wk_hi = wq_lo;
  if (normed) {
    wq_lo = *reinterpret_cast<const uint2*>(q_norm_w + j0);
    wq_hi = *reinterpret_cast<const uint2*>(q_norm_w + HALF + j0);
    wk_lo = *reinterpret_cast<const uint2*>(k_norm_w + j0);
    wk_hi = *reinterpret_cast<const uint2*>(k_norm_w + HALF + j0);
  }
  float cs[4] = {1.f, 1.f, 1.f, 1.f}, sn[4] = {0.f, 0.f, 0.f, 0.f};
  if (inv_freq != nullptr) {
    if (TABLE) {
      const float4 c = *reinterpret_cast<const float4*>(cos_sin + (size_t)t * D + j0), s = *reinterpret_cast<const float4*>(cos_sin + (size_t)t * D + HALF + j0);
      cs[0] = c.x; cs[1] = c.y; cs[2] = c.z; cs[3] = c.w;
      sn[0] = s.x; sn[1] = s.y; sn[2] = s.z; sn[3] = s.w;
    } else {
#pragma unroll
      for (int i = 0; i < 4; ++i) sincosf((float)pos * inv_freq[j0 + i], &sn[i], &cs[i]);
    }
  }
  const int page = tables.page(request, pos, tables_end, page_shift, num_pages);
  if (page < 0 && threadIdx.x == 0) atomicExch(status, 2);
  const size_t at0 = ((size_t)max(page, 0) * nkv << page_shift) + (pos & ((1 << page_shift) - 1));
  for (int base = 0; base < heads; base += BATCH * stride) {  // the same trips for every lane: they exchange sums
    uint2 lo_now[BATCH], hi_now[BATCH];
#pragma unroll
    for (int b = 0; b < BATCH; ++b) {
      lo_now[b] = lo_raw[b];
      hi_now[b] = hi_raw[b];
    }
    if (base + BATCH * stride < heads) fetch(base + BATCH * stride);
#pragma unroll
    for (int b = 0; b < BATCH; ++b) {
      const int h = base + warp * HPW + slot + b * stride;
      const bool is_q = h < nq, is_v = h >= nq + nkv;
      float lo[4], hi[4];
      c8_float4(lo, lo_now[b]);
      c8_float4(hi, hi_now[b]);
      float ss = 0.f;
#pragma unroll
      for (int i = 0; i < 4; ++i) ss += lo[i] * lo[i] + hi[i] * hi[i];
#pragma unroll
      for (int off = LPH / 2; off > 0; off >>= 1) ss += __shfl_xor_sync(0xffffffffu, ss, off);
      if (!is_v) {
        float wl[4], wh[4];
        const float inv = normed ? 1.0f / sqrtf(ss * (1.f / D) + eps) : 1.f;
        c8_float4(wl, is_q ? wq_lo : wk_lo);
        c8_float4(wh, is_q ? wq_hi : wk_hi);
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const float l = normed ? (lo[i] * inv) * wl[i] : lo[i], u = normed ? (hi[i] * inv) * wh[i] : hi[i];
          lo[i] = l * cs[i] - u * sn[i];
          hi[i] = u * cs[i] + l * sn[i];
        }
      }
      uint32_t amax = 0;
      if (base + warp * HPW + b * stride + HPW > nq) {  // (some head of the warp's is to be quantised)
#pragma unroll
        for (int i = 0; i < 4; ++i) amax = max(amax, max(__float_as_uint(lo[i]) & 0x7FFFFFFFu, __float_as_uint(hi[i]) & 0x7FFFFFFFu));
#pragma unroll
        for (int off = LPH / 2; off > 0; off >>= 1) amax = max(amax, __shfl_xor_sync(0xffffffffu, amax, off));
      }
      if (h >= heads) continue;
      if (is_q) {
        __nv_bfloat16* dst = q_out + ((size_t)t * nq + h) * D + j0;
        *reinterpret_cast<uint2*>(dst) = c8_bf16x4(lo);
        *reinterpret_cast<uint2*>(dst + HALF) = c8_bf16x4(hi);
        continue;
      }
      if (page < 0) continue;
      const int e = c8_exponent(amax);
      const float inv = c8_inverse(e);
      const size_t at = at0 + ((size_t)(h - nq - (is_v ? nkv : 0)) << page_shift);
      uint8_t* dst = (is_v ? v_codes : k_codes) + at * D + j0;
      *reinterpret_cast<uint32_t*>(dst) = c8_keep(c8_codes4(lo[0] * inv, lo[1] * inv, lo[2] * inv, lo[3] * inv), e);
      *reinterpret_cast<uint32_t*>(dst + HALF) = c8_keep(c8_codes4(hi[0] * inv, hi[1] * inv, hi[2] * inv, hi[3] * inv), e);
      if (sub == 0) (is_v ? v_exps : k_exps)[at] = (uint8_t)e;
    }
  }
}

// 8 codes times a power of two
__device__ __forceinline__ void c8_numbers8(float (&f)[8], const uint2& raw, float factor) {
  const uint32_t words[2] = {raw.x, raw.y};
#pragma unroll
  for (int i = 0; i < 2; ++i) {
    const float2 lo = c8_float2(c8_half2_lo(words[i])), hi = c8_float2(c8_half2_hi(words[i]));
    f[4 * i] = lo.x * factor;
    f[4 * i + 1] = lo.y * factor;
    f[4 * i + 2] = hi.x * factor;
    f[4 * i + 3] = hi.y * factor;
  }
}
__device__ __forceinline__ void c8_store8(float* dst, const uint2& raw, float factor) {
  float f[8];
  c8_numbers8(f, raw, factor);
#pragma unroll
  for (int i = 0; i < 2; ++i) reinterpret_cast<float4*>(dst)[i] = make_float4(f[4 * i], f[4 * i + 1], f[4 * i + 2], f[4 * i + 3]);
}
__device__ __forceinline__ void c8_store8(__nv_bfloat16* dst, const uint2& raw, float factor) {
  float f[8];
  c8_numbers8(f, raw, factor);
  *reinterpret_cast<uint4*>(dst) = float_to_bf16x8(f);
}

// Eight numbers of K and V at a time: neighbours' loads (8 bytes) and stores (16 in bfloat16) lie side by side. A thread takes READ_EACH such pieces of a token, all asked for
// together, so that where the token lies is looked up once for them. Block (tokens, share of a token).
constexpr int READ_EACH = 4;
template <typename T>
__global__ void __launch_bounds__(256)
cache8_read_kernel(T* __restrict__ k_out, T* __restrict__ v_out, const uint8_t* __restrict__ k_codes, const uint8_t* __restrict__ k_exps,
                   const uint8_t* __restrict__ v_codes, const uint8_t* __restrict__ v_exps, const int* __restrict__ positions,
                   const int* __restrict__ row_of_token, Tables8 tables, int num_tokens, int nkv, int d, int page_shift, int num_pages, int* __restrict__ status) {
  pdl_prologue(k_codes, k_exps, v_codes, v_exps, positions, row_of_token, tables.page_indptr, tables.page_indices);
  const int eights = d >> 3, pieces = nkv * eights, threads = (pieces + READ_EACH - 1) / READ_EACH;  // of a token
  const int tokens = max(1, 256 / threads), mine = threadIdx.x / threads, t = blockIdx.x * tokens + (tokens > 1 ? mine : 0);
  const int first = tokens > 1 ? threadIdx.x - mine * threads : blockIdx.y * 256 + threadIdx.x;
  if (t >= num_tokens || first >= threads || (tokens > 1 && mine >= tokens)) return;
  const int pos = positions[t], request = row_of_token[t], page = tables.page(request, pos, tables.end(), page_shift, num_pages);
  if (page < 0) {
    if (first == 0) atomicExch(status, 2);
    return;
  }
  const size_t at0 = ((size_t)page * nkv << page_shift) + (pos & ((1 << page_shift) - 1));
  uint2 raw[READ_EACH][2];
  int b[READ_EACH][2];
#pragma unroll
  for (int i = 0; i < READ_EACH; ++i) {
    const int piece = min(first + i * threads, pieces - 1), h = div_small(piece, eights), c = piece - h * eights;  // (the last one again, unused)
    const size_t at = at0 + ((size_t)h << page_shift);
    raw[i][0] = *reinterpret_cast<const uint2*>(k_codes + at * d + c * 8);
    raw[i][1] = *reinterpret_cast<const uint2*>(v_codes + at * d + c * 8);
    b[i][0] = k_exps[at];
    b[i][1] = v_exps[at];
  }
#pragma unroll
  for (int i = 0; i < READ_EACH; ++i) {
    const int piece = first + i * threads;
    if (piece >= pieces) break;
#pragma unroll
    for (int w = 0; w < 2; ++w) c8_store8((w ? v_out : k_out) + ((size_t)t * pieces + piece) * 8, raw[i][w], c8_factor(b[i][w]));
  }
}

// The pages that rows [first, rows) of a step look at, as bfloat16 pages of their own, and the tables that say so: a row's pages from the first that its window reaches (page 0 without one)
// to the last that holds a token, counted through all rows, become pages 0, 1, ... of k_out and v_out; indptr_out[r] + entry is where entry `entry` of row r's table now lies in ids, and
// ids[i] = i, 0 behind the last. So what the products behind this look up lies in [0, gridDim.x) whatever the step's own table is like: its rows may begin ahead of the table or inside one
// another, where a window has given pages back. A page that the table or the pool does not have becomes zeros. Rows that look at more pages than the launch was made for (the host counted
// other lengths) raise the status word and look at some of these. What is done to a value vector that is not
// finite is done for the products that follow, which weigh what a query does not see by zero: its key becomes NaN (a score that is masked where it is not seen), the value itself
// zero. Block (page, share of it), READ_EACH pieces of 8 numbers of K and V a thread; every warp finds the page's row for itself, 32 rows a look.
__global__ void __launch_bounds__(256)
cache8_unpack_kernel(__nv_bfloat16* __restrict__ k_out, __nv_bfloat16* __restrict__ v_out, int* __restrict__ ids, int* __restrict__ indptr_out, const uint8_t* __restrict__ k_codes,
                     const uint8_t* __restrict__ k_exps, const uint8_t* __restrict__ v_codes, const uint8_t* __restrict__ v_exps, const int* __restrict__ cu_q,
                     const int* __restrict__ q_start, const int* __restrict__ page_indptr, const int* __restrict__ page_indices, int first, int rows, int all_rows, int nkv, int d,
                     int window, int page_shift, int num_pages, int num_entries, int num_ids, int* __restrict__ status) {
  pdl_prologue(k_codes, k_exps, v_codes, v_exps, cu_q, q_start, page_indptr, page_indices);
  const int out_page = blockIdx.x, page_size = 1 << page_shift, lane = threadIdx.x & 31;
  int a = -1, entry = out_page, left = 0, ahead = 0, table = 0, stop = 0;  // the row, which of its pages, how many there are behind it, the row's first, where its table lies and ends
  for (int r0 = first; r0 < rows; r0 += 32) {
    const int r = r0 + lane;
    int need = 0, passed = 0, at = 0, end = 0;
    if (r < rows) {
      const int from = q_start[r], tokens = cu_q[r + 1] - cu_q[r];
      passed = window > 0 ? max(0, from - window + 1) >> page_shift : 0;
      if (tokens > 0) need = max(0, ((from + tokens + page_size - 1) >> page_shift) - passed);
      at = page_indptr[r];
      end = min(page_indptr[window > 0 ? all_rows : r + 1], num_entries);  // (without a window a table is whole, and ends where the next begins)
    }
    int incl = need;
#pragma unroll
    for (int off = 1; off < 32; off <<= 1) {
      const int before = __shfl_up_sync(0xffffffffu, incl, off);
      if (lane >= off) incl += before;
    }
    const unsigned behind = __ballot_sync(0xffffffffu, incl > entry);
    if (behind) {
      const int src = __ffs(behind) - 1;
      a = r0 + src;
      left = __shfl_sync(0xffffffffu, incl, src) - entry - 1;
      entry -= __shfl_sync(0xffffffffu, incl - need, src);
      ahead = __shfl_sync(0xffffffffu, passed, src);
      table = __shfl_sync(0xffffffffu, at, src);
      stop = __shfl_sync(0xffffffffu, end, src);
      break;
    }
    entry -= __shfl_sync(0xffffffffu, incl, 31);
  }
  const bool leads = blockIdx.y == 0 && threadIdx.x == 0;
  if (leads) ids[out_page] = out_page;
  if (blockIdx.y == 0)
    for (int i = gridDim.x + blockIdx.x * 256 + threadIdx.x; i < num_ids; i += gridDim.x * 256) ids[i] = 0;
  if (a < 0) return;
  if (leads && entry == 0) indptr_out[a] = out_page - ahead;
  if (leads && blockIdx.x == gridDim.x - 1) {
    for (int r = a + 1; r < rows; ++r) {
      if (cu_q[r + 1] == cu_q[r]) continue;
      indptr_out[r] = window > 0 ? -(max(0, q_start[r] - window + 1) >> page_shift) : 0;
      left = 1;
    }
    if (left > 0) atomicExch(status, 2);
  }
  const int eights = d >> 3, pieces = nkv * page_size * eights, idx0 = blockIdx.y * (256 * READ_EACH) + threadIdx.x;
  if (idx0 >= pieces) return;
  const int f = table + ahead + entry;
  const int page = f >= 0 && f < stop ? page_indices[f] : -1;
  const bool there = (unsigned)page < (unsigned)num_pages;
  if (!there && threadIdx.x == 0) atomicExch(status, 2);
  const size_t from = (size_t)(there ? page : 0) * nkv * page_size, to = (size_t)out_page * pieces;
  uint2 raw[READ_EACH][2];
  int b8[READ_EACH][2];
#pragma unroll
  for (int i = 0; i < READ_EACH; ++i) {
    const int idx = min(idx0 + 256 * i, pieces - 1), row = div_small(idx, eights);  // (the last one again, unused)
    const size_t at = (from * eights + idx) * 8;
    raw[i][0] = *reinterpret_cast<const uint2*>(k_codes + at);
    raw[i][1] = *reinterpret_cast<const uint2*>(v_codes + at);
    b8[i][0] = k_exps[from + row];
    b8[i][1] = v_exps[from + row];
    if (!there) {
      raw[i][0] = raw[i][1] = make_uint2(0u, 0u);
      b8[i][0] = b8[i][1] = 0;
    }
  }
#pragma unroll
  for (int i = 0; i < READ_EACH; ++i) {
    const int idx = idx0 + 256 * i;
    if (idx >= pieces) break;
    const bool fine = b8[i][1] != C8_NAN;
    c8_store8(k_out + (to + idx) * 8, raw[i][0], c8_factor(fine ? b8[i][0] : C8_NAN));
    c8_store8(v_out + (to + idx) * 8, raw[i][1], fine ? c8_factor(b8[i][1]) : 0.f);
  }
}

}  // namespace ms

using namespace ms;

MS_DEFINE_LAST_ERROR(ms_cache8_last_error)
MS_DEFINE_PDL_SWITCH(ms_cache8_set_pdl)

static int c8_check(const char* what, int nkv, int d, int page_size, long long num_pages) {
  MS_CHECK_ARG(nkv > 0 && d >= 16 && d <= C8_MAX_D && d % 16 == 0, "%s: bad sizes nkv=%d d=%d (head sizes are multiples of 16 up to %d)", what, nkv, d, C8_MAX_D);
  MS_CHECK_ARG(page_size >= 8 && (page_size & (page_size - 1)) == 0, "%s: page_size=%d must be a power of two from 8 on", what, page_size);
  MS_CHECK_ARG(num_pages > 0 && num_pages < (1LL << 31), "%s: %lld pages", what, num_pages);
  return 0;
}

// The pools' device as the current one, for the length of a call.
struct OnDevice {
  int before = -1;
  explicit OnDevice(int device) {
    int now = 0;
    if (cudaGetDevice(&now) == cudaSuccess && now != device && cudaSetDevice(device) == cudaSuccess) before = now;
  }
  ~OnDevice() {
    if (before >= 0) cudaSetDevice(before);
  }
};

// Arguments come as one block: 24 of them one by one take the caller 1.7 us more, where a call takes 8.
struct Write8 {
  void *q_out, *k_codes, *k_exps, *v_codes, *v_exps;
  const void *qkv, *q_norm_w, *k_norm_w;
  const float *inv_freq, *cos_sin;
  const int *positions, *row_of_token, *page_indptr, *page_indices;
  int* status;
  cudaStream_t stream;
  long long num_pages;
  int device, rows, num_entries, num_tokens, nq, nkv, d, rot, page_size;  // rows of page_indptr, entries of page_indices
  float eps;
};
struct Read8 {
  void *k_out, *v_out;
  const void *k_codes, *k_exps, *v_codes, *v_exps;
  const int *positions, *row_of_token, *page_indptr, *page_indices;
  int* status;
  cudaStream_t stream;
  long long num_pages;
  int device, rows, num_entries, num_tokens, nkv, d, page_size, dtype;
};

static_assert(sizeof(Write8) == 176 && sizeof(Read8) == 136, "packed by the caller without gaps");

MS_EXPORT int ms_cache8_write(const Write8* args) {
  const auto [q_out, k_codes, k_exps, v_codes, v_exps, qkv, q_norm_w, k_norm_w, inv_freq, cos_sin, positions, row_of_token, page_indptr, page_indices, status, stream, num_pages, device,
              rows, num_entries, num_tokens, nq, nkv, d, rot, page_size, eps] = *args;
  if (num_tokens == 0) return 0;
  const OnDevice here(device);
  if (int rc = c8_check("cache8_write", nkv, d, page_size, num_pages)) return rc;
  MS_CHECK_ARG(nq >= 0 && num_tokens > 0 && rows >= 0, "cache8_write: nq=%d, %d tokens, %d rows", nq, num_tokens, rows);
  const Tables8 tables = {page_indptr, page_indices, rows, num_entries};
  MS_CHECK_ARG(rot >= 0 && rot <= d && rot % 2 == 0, "cache8_write: rotary_dim=%d must be even and at most the head size %d", rot, d);
  MS_CHECK_ARG((uintptr_t)k_codes % 16 == 0 && (uintptr_t)v_codes % 16 == 0, "cache8_write: pools must be 16-byte aligned");
  if ((d == 64 || d == 128 || d == 256) && (rot == d || rot == 0 || inv_freq == nullptr) && (q_norm_w != nullptr) == (k_norm_w != nullptr) && (uintptr_t)qkv % 8 == 0 &&
      (uintptr_t)q_out % 8 == 0 && (uintptr_t)q_norm_w % 8 == 0 && (uintptr_t)k_norm_w % 8 == 0 && (uintptr_t)cos_sin % 16 == 0) {
    const bool table = cos_sin != nullptr || rot == 0 || inv_freq == nullptr;
    auto kernel = d == 64    ? (table ? cache8_write_token_kernel<64, true> : cache8_write_token_kernel<64, false>)
                  : d == 128 ? (table ? cache8_write_token_kernel<128, true> : cache8_write_token_kernel<128, false>)
                             : (table ? cache8_write_token_kernel<256, true> : cache8_write_token_kernel<256, false>);
    // as many warps as bring all heads in equal trips of two a lane group, 8 at most: 48 heads of 128 in two trips of 6 warps 17.8 us, of 8 warps 19.9 (the sizes above)
    const int a_trip = 2 * (32 / (d / 8)), trips = ceil_div(nq + 2 * nkv, 8 * a_trip), warps = ceil_div(nq + 2 * nkv, a_trip * trips);
    MS_LAUNCH(kernel, num_tokens, 32 * warps, 0, stream, (__nv_bfloat16*)q_out, (uint8_t*)k_codes, (uint8_t*)k_exps, (uint8_t*)v_codes, (uint8_t*)v_exps,
              (const __nv_bfloat16*)qkv, (const __nv_bfloat16*)q_norm_w, (const __nv_bfloat16*)k_norm_w, rot ? inv_freq : (const float*)nullptr, cos_sin, positions,
              row_of_token, tables, nq, nkv, eps, c8_page_shift(page_size), (int)num_pages, status);
    return 0;
  }
  const long long items = (long long)num_tokens * (nq + 2 * nkv);
  MS_LAUNCH(cache8_write_kernel, (unsigned)((items + 7) / 8), 256, 0, stream, (__nv_bfloat16*)q_out, (uint8_t*)k_codes, (uint8_t*)k_exps, (uint8_t*)v_codes,
            (uint8_t*)v_exps, (const __nv_bfloat16*)qkv, (const __nv_bfloat16*)q_norm_w, (const __nv_bfloat16*)k_norm_w, rot ? inv_freq : (const float*)nullptr,
            cos_sin, positions, row_of_token, tables, num_tokens, nq, nkv, d, rot, eps, c8_page_shift(page_size), (int)num_pages, status);
  return 0;
}

MS_EXPORT int ms_cache8_read(const Read8* args) {
  const auto [k_out, v_out, k_codes, k_exps, v_codes, v_exps, positions, row_of_token, page_indptr, page_indices, status, stream, num_pages, device, rows, num_entries,
              num_tokens, nkv, d, page_size, dtype] = *args;
  if (num_tokens == 0) return 0;
  const OnDevice here(device);
  if (int rc = c8_check("cache8_read", nkv, d, page_size, num_pages)) return rc;
  MS_CHECK_ARG((uintptr_t)k_codes % 16 == 0 && (uintptr_t)v_codes % 16 == 0 && (uintptr_t)k_out % 16 == 0 && (uintptr_t)v_out % 16 == 0,
               "cache8_read: tensors must be 16-byte aligned");
  MS_CHECK_ARG(dtype == MS_F32 || dtype == MS_BF16, "cache8_read: dtype code %d", dtype);
  MS_CHECK_ARG(num_tokens > 0 && rows >= 0, "cache8_read: %d tokens, %d rows", num_tokens, rows);
  const Tables8 tables = {page_indptr, page_indices, rows, num_entries};
  const int threads = ceil_div(nkv * (d / 8), READ_EACH), tokens = threads < 256 ? 256 / threads : 1;
  const dim3 grid(ceil_div(num_tokens, tokens), ceil_div(threads, 256));
  MS_CHECK_ARG(grid.y <= 65535, "cache8_read: too many heads (%d)", nkv);
  if (dtype == MS_F32) {
    MS_LAUNCH(cache8_read_kernel<float>, grid, 256, 0, stream, (float*)k_out, (float*)v_out, (const uint8_t*)k_codes, (const uint8_t*)k_exps,
              (const uint8_t*)v_codes, (const uint8_t*)v_exps, positions, row_of_token, tables, num_tokens, nkv, d, c8_page_shift(page_size),
              (int)num_pages, status);
  } else {
    MS_LAUNCH(cache8_read_kernel<__nv_bfloat16>, grid, 256, 0, stream, (__nv_bfloat16*)k_out, (__nv_bfloat16*)v_out, (const uint8_t*)k_codes,
              (const uint8_t*)k_exps, (const uint8_t*)v_codes, (const uint8_t*)v_exps, positions, row_of_token, tables, num_tokens, nkv, d,
              c8_page_shift(page_size), (int)num_pages, status);
  }
  return 0;
}

// Which capture the stream is part of (never 0), 0: none.
MS_EXPORT unsigned long long ms_cache8_capture_id(cudaStream_t stream) {
  cudaStreamCaptureStatus state = cudaStreamCaptureStatusNone;
  unsigned long long id = 0;
  if (cudaStreamGetCaptureInfo(stream, &state, &id) != cudaSuccess) {
    cudaGetLastError();  // (the default stream while another one is captured)
    return 0;
  }
  return state == cudaStreamCaptureStatusActive ? id + 1 : 0;
}

// Rows [first, rows) of all_rows look at `entries` pages, which k_out and v_out [entries, nkv, page_size, d] hold; their tables are ids [num_ids] and, by row, indptr_out. page_indices has
// num_entries entries; ids that many more than pages, so that no row of lengths other than the host's leaves it.
MS_EXPORT int ms_cache8_unpack(void* k_out, void* v_out, int* ids, int* indptr_out, const void* k_codes, const void* k_exps, const void* v_codes, const void* v_exps, const int* cu_q,
                               const int* q_start, const int* page_indptr, const int* page_indices, int first, int rows, int all_rows, int entries, int nkv, int d, int window,
                               int page_size, long long num_pages, int num_entries, int num_ids, int* status, cudaStream_t stream) {
  if (entries == 0) return 0;
  if (int rc = c8_check("cache8_unpack", nkv, d, page_size, num_pages)) return rc;
  MS_CHECK_ARG(first >= 0 && rows > first && all_rows >= rows && entries > 0 && num_ids >= entries, "cache8_unpack: rows %d to %d of %d, %d entries, %d ids", first, rows, all_rows, entries,
               num_ids);
  MS_CHECK_ARG((uintptr_t)k_codes % 16 == 0 && (uintptr_t)v_codes % 16 == 0 && (uintptr_t)k_out % 16 == 0 && (uintptr_t)v_out % 16 == 0,
               "cache8_unpack: tensors must be 16-byte aligned");
  MS_CHECK_ARG((long long)nkv * page_size <= 1 << 20, "cache8_unpack: pages of %d tokens and %d heads are too large", page_size, nkv);
  const int blocks = ceil_div(nkv * page_size * (d / 8), 256 * READ_EACH);
  MS_CHECK_ARG(blocks <= 65535, "cache8_unpack: pages of %d tokens and %d heads are too large", page_size, nkv);
  MS_LAUNCH(cache8_unpack_kernel, dim3(entries, blocks), 256, 0, stream, (__nv_bfloat16*)k_out, (__nv_bfloat16*)v_out, ids, indptr_out, (const uint8_t*)k_codes, (const uint8_t*)k_exps,
            (const uint8_t*)v_codes, (const uint8_t*)v_exps, cu_q, q_start, page_indptr, page_indices, first, rows, all_rows, nkv, d, window, c8_page_shift(page_size),
            (int)num_pages, num_entries, num_ids, status);
  return 0;
}
