// Writing the 8-bit paged cache and reading it back (the format: cache8.cuh).
//
// The write is the step between the q|k|v product and attention: per-head RMSNorm of q and k, rotation of halves, queries out in
// bfloat16, keys (behind norm and rotation) and values quantised from float32 into their pages: one rounding, to the code.
// Formulas of the norm and the rotation: miniserve/model/qwen3.py:98-108, 118-123; the reference keeps its cache in the model's
// type (miniserve/cache/kv_pool.py:46-50).
#include "cache8.cuh"

namespace ms {

constexpr int C8_MAX_D = 256;

// The page of position `pos` of request `row`; -1 where the table has none, or none that the pool has.
__device__ __forceinline__ int c8_page(const int* page_indptr, const int* page_indices, int row, int pos, int page_shift, int num_pages) {
  const int first = page_indptr[row], n = page_indptr[row + 1] - first, entry = pos >> page_shift;
  if (entry < 0 || entry >= n) return -1;
  const int page = page_indices[first + entry];
  return page < num_pages ? page : -1;
}

// A warp per (token, head).
__global__ void __launch_bounds__(256)
cache8_write_kernel(__nv_bfloat16* __restrict__ q_out, uint8_t* __restrict__ k_codes, uint8_t* __restrict__ k_exps, uint8_t* __restrict__ v_codes,
                    uint8_t* __restrict__ v_exps, const __nv_bfloat16* __restrict__ qkv, const __nv_bfloat16* __restrict__ q_norm_w,
                    const __nv_bfloat16* __restrict__ k_norm_w, const float* __restrict__ inv_freq, const float* __restrict__ cos_sin,
                    const int* __restrict__ positions, const int* __restrict__ row_of_token, const int* __restrict__ page_indptr,
                    const int* __restrict__ page_indices, int num_tokens, int nq, int nkv, int d, int rot, float eps, int page_shift, int num_pages,
                    int* __restrict__ status) {
  pdl_prologue(qkv, q_norm_w, k_norm_w, inv_freq, cos_sin, positions, row_of_token, page_indptr, page_indices);
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
  const int page = c8_page(page_indptr, page_indices, row_of_token[t], pos, page_shift, num_pages);
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

// Head sizes 64, 128 and 256 rotated whole or not at all: a block per token, D / 16 lanes per head. A lane holds 8 numbers of the head's first half and the 8 of the second that
// rotate with them, in 16-byte loads and stores (8 of codes); a head's lanes exchange a sum of squares and a maximum. What hangs on the token alone is fetched once a lane,
// and its first numbers before the page is looked up (three loads, one behind the other).
template <int D>
__global__ void __launch_bounds__(256)
cache8_write_token_kernel(__nv_bfloat16* __restrict__ q_out, uint8_t* __restrict__ k_codes, uint8_t* __restrict__ k_exps, uint8_t* __restrict__ v_codes,
                          uint8_t* __restrict__ v_exps, const __nv_bfloat16* __restrict__ qkv, const __nv_bfloat16* __restrict__ q_norm_w,
                          const __nv_bfloat16* __restrict__ k_norm_w, const float* __restrict__ inv_freq, const float* __restrict__ cos_sin,
                          const int* __restrict__ positions, const int* __restrict__ row_of_token, const int* __restrict__ page_indptr,
                          const int* __restrict__ page_indices, int nq, int nkv, float eps, int page_shift, int num_pages, int* __restrict__ status) {
  pdl_prologue(qkv, q_norm_w, k_norm_w, inv_freq, cos_sin, positions, row_of_token, page_indptr, page_indices);
  constexpr int LPH = D / 16, HPW = 32 / LPH, HALF = D / 2, BATCH = 2;
  const int t = blockIdx.x, warp = threadIdx.x >> 5, lane = threadIdx.x & 31, sub = lane % LPH, slot = lane / LPH, j0 = sub * 8;
  const int heads = nq + 2 * nkv, stride = (int)(blockDim.x >> 5) * HPW;  // heads a pass
  const __nv_bfloat16* row_in = qkv + (size_t)t * heads * D;
  uint4 lo_raw[BATCH], hi_raw[BATCH];
  auto fetch = [&](int base) {
#pragma unroll
    for (int b = 0; b < BATCH; ++b) {
      const __nv_bfloat16* src = row_in + (size_t)min(base + warp * HPW + slot + b * stride, heads - 1) * D;  // past the end: the last head again, unused
      lo_raw[b] = *reinterpret_cast<const uint4*>(src + j0);
      hi_raw[b] = *reinterpret_cast<const uint4*>(src + HALF + j0);
    }
  };
  fetch(0);
  const int pos = positions[t], request = row_of_token[t];
  const bool normed = q_norm_w != nullptr;
  uint4 w_raw[2][2] = {};  // of q and k, both halves
  if (normed) {
    w_raw[0][0] = *reinterpret_cast<const uint4*>(q_norm_w + j0);
    w_raw[0][1] = *reinterpret_cast<const uint4*>(q_norm_w + HALF + j0);
    w_raw[1][0] = *reinterpret_cast<const uint4*>(k_norm_w + j0);
    w_raw[1][1] = *reinterpret_cast<const uint4*>(k_norm_w + HALF + j0);
  }
  float cs[8], sn[8];
  if (inv_freq == nullptr) {
#pragma unroll
    for (int i = 0; i < 8; ++i) { cs[i] = 1.f; sn[i] = 0.f; }
  } else if (cos_sin) {
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      const float4 c = reinterpret_cast<const float4*>(cos_sin + (size_t)t * D + j0)[i], s = reinterpret_cast<const float4*>(cos_sin + (size_t)t * D + HALF + j0)[i];
      cs[4 * i] = c.x; cs[4 * i + 1] = c.y; cs[4 * i + 2] = c.z; cs[4 * i + 3] = c.w;
      sn[4 * i] = s.x; sn[4 * i + 1] = s.y; sn[4 * i + 2] = s.z; sn[4 * i + 3] = s.w;
    }
  } else {
#pragma unroll
    for (int i = 0; i < 8; ++i) sincosf((float)pos * inv_freq[j0 + i], &sn[i], &cs[i]);
  }
  const int page = c8_page(page_indptr, page_indices, request, pos, page_shift, num_pages);
  if (page < 0 && threadIdx.x == 0) atomicExch(status, 2);
  const size_t at0 = ((size_t)max(page, 0) * nkv << page_shift) + (pos & ((1 << page_shift) - 1));
  for (int base = 0; base < heads; base += BATCH * stride) {  // the same trips for every lane: they exchange sums
    if (base > 0) fetch(base);
#pragma unroll
    for (int b = 0; b < BATCH; ++b) {
      const int h = base + warp * HPW + slot + b * stride;
      const bool is_q = h < nq, is_v = h >= nq + nkv;
      float lo[8], hi[8];
      bf16x8_to_float(lo_raw[b], lo);
      bf16x8_to_float(hi_raw[b], hi);
      float ss = 0.f;
#pragma unroll
      for (int i = 0; i < 8; ++i) ss += lo[i] * lo[i] + hi[i] * hi[i];
#pragma unroll
      for (int off = LPH / 2; off > 0; off >>= 1) ss += __shfl_xor_sync(0xffffffffu, ss, off);
      if (!is_v) {
        float wl[8], wh[8];
        const float inv = normed ? 1.0f / sqrtf(ss / (float)D + eps) : 1.f;
        bf16x8_to_float(w_raw[is_q ? 0 : 1][0], wl);
        bf16x8_to_float(w_raw[is_q ? 0 : 1][1], wh);
#pragma unroll
        for (int i = 0; i < 8; ++i) {
          const float l = normed ? (lo[i] * inv) * wl[i] : lo[i], u = normed ? (hi[i] * inv) * wh[i] : hi[i];
          lo[i] = l * cs[i] - u * sn[i];
          hi[i] = u * cs[i] + l * sn[i];
        }
      }
      uint32_t amax = 0;
#pragma unroll
      for (int i = 0; i < 8; ++i) amax = max(amax, max(__float_as_uint(lo[i]) & 0x7FFFFFFFu, __float_as_uint(hi[i]) & 0x7FFFFFFFu));
#pragma unroll
      for (int off = LPH / 2; off > 0; off >>= 1) amax = max(amax, __shfl_xor_sync(0xffffffffu, amax, off));
      if (h >= heads) continue;
      if (is_q) {
        __nv_bfloat16* dst = q_out + ((size_t)t * nq + h) * D;
        *reinterpret_cast<uint4*>(dst + j0) = float_to_bf16x8(lo);
        *reinterpret_cast<uint4*>(dst + HALF + j0) = float_to_bf16x8(hi);
        continue;
      }
      if (page < 0) continue;
      const int e = c8_exponent(amax);
      const float inv = c8_inverse(e);
      const size_t at = at0 + ((size_t)(h - nq - (is_v ? nkv : 0)) << page_shift);
      uint8_t* dst = (is_v ? v_codes : k_codes) + at * D;
      *reinterpret_cast<uint2*>(dst + j0) = make_uint2(c8_keep(c8_codes4(lo[0] * inv, lo[1] * inv, lo[2] * inv, lo[3] * inv), e),
                                                       c8_keep(c8_codes4(lo[4] * inv, lo[5] * inv, lo[6] * inv, lo[7] * inv), e));
      *reinterpret_cast<uint2*>(dst + HALF + j0) = make_uint2(c8_keep(c8_codes4(hi[0] * inv, hi[1] * inv, hi[2] * inv, hi[3] * inv), e),
                                                              c8_keep(c8_codes4(hi[4] * inv, hi[5] * inv, hi[6] * inv, hi[7] * inv), e));
      if (sub == 0) (is_v ? v_exps : k_exps)[at] = (uint8_t)e;
    }
  }
}

// 16 codes times a power of two
__device__ __forceinline__ void c8_numbers16(float (&f)[16], const uint4& raw, float factor) {
  const uint32_t words[4] = {raw.x, raw.y, raw.z, raw.w};
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const float2 lo = c8_float2(c8_half2_lo(words[i])), hi = c8_float2(c8_half2_hi(words[i]));
    f[4 * i] = lo.x * factor;
    f[4 * i + 1] = lo.y * factor;
    f[4 * i + 2] = hi.x * factor;
    f[4 * i + 3] = hi.y * factor;
  }
}
__device__ __forceinline__ void c8_store16(float* dst, const uint4& raw, float factor) {
  float f[16];
  c8_numbers16(f, raw, factor);
#pragma unroll
  for (int i = 0; i < 4; ++i) reinterpret_cast<float4*>(dst)[i] = make_float4(f[4 * i], f[4 * i + 1], f[4 * i + 2], f[4 * i + 3]);
}
__device__ __forceinline__ void c8_store16(__nv_bfloat16* dst, const uint4& raw, float factor) {
  float f[16];
  c8_numbers16(f, raw, factor);
#pragma unroll
  for (int i = 0; i < 2; ++i) {
    float part[8];
#pragma unroll
    for (int j = 0; j < 8; ++j) part[j] = f[8 * i + j];
    reinterpret_cast<uint4*>(dst)[i] = float_to_bf16x8(part);
  }
}

// A thread per 16 numbers of a (token, kv head): K and V.
template <typename T>
__global__ void __launch_bounds__(256)
cache8_read_kernel(T* __restrict__ k_out, T* __restrict__ v_out, const uint8_t* __restrict__ k_codes, const uint8_t* __restrict__ k_exps,
                   const uint8_t* __restrict__ v_codes, const uint8_t* __restrict__ v_exps, const int* __restrict__ positions,
                   const int* __restrict__ row_of_token, const int* __restrict__ page_indptr, const int* __restrict__ page_indices, int num_tokens,
                   int nkv, int d, int page_shift, int num_pages, int* __restrict__ status) {
  pdl_prologue(k_codes, k_exps, v_codes, v_exps, positions, row_of_token, page_indptr, page_indices);
  const int chunks = d >> 4;
  const long long idx = (long long)blockIdx.x * blockDim.x + threadIdx.x;
  if (idx >= (long long)num_tokens * nkv * chunks) return;
  const int c = (int)(idx % chunks);
  const long long item = idx / chunks;
  const int t = (int)(item / nkv), h = (int)(item - (long long)t * nkv), pos = positions[t];
  const int page = c8_page(page_indptr, page_indices, row_of_token[t], pos, page_shift, num_pages);
  if (page < 0) {
    if (c == 0 && h == 0) atomicExch(status, 2);
    return;
  }
  const size_t at = ((size_t)page * nkv + h) * ((size_t)1 << page_shift) + (pos & ((1 << page_shift) - 1));
  const uint4 raw[2] = {*reinterpret_cast<const uint4*>(k_codes + at * d + c * 16), *reinterpret_cast<const uint4*>(v_codes + at * d + c * 16)};
  const int b[2] = {k_exps[at], v_exps[at]};
#pragma unroll
  for (int w = 0; w < 2; ++w) c8_store16((w ? v_out : k_out) + (size_t)item * d + c * 16, raw[w], c8_factor(b[w]));
}

// The pages that rows [first, rows) of a step list, as bfloat16 pages of their own: entry f of the table becomes page f - indptr[first], and ids[f] says so. Entries that no query of their
// row looks at (ahead of a window) are left out. What is done to a value vector that is not finite is done for the products that follow, which weigh what a query does
// not see by zero: its key becomes NaN (a score that is masked where it is not seen), the value itself zero. Block (entry, share of its page): a thread per 16 numbers of a key
// and a value, 34 bytes in, 64 out.
__global__ void __launch_bounds__(256)
cache8_unpack_kernel(__nv_bfloat16* __restrict__ k_out, __nv_bfloat16* __restrict__ v_out, int* __restrict__ ids, const uint8_t* __restrict__ k_codes,
                     const uint8_t* __restrict__ k_exps, const uint8_t* __restrict__ v_codes, const uint8_t* __restrict__ v_exps, const int* __restrict__ cu_q,
                     const int* __restrict__ q_start, const int* __restrict__ page_indptr, const int* __restrict__ page_indices, int first, int rows, int nkv, int d, int window,
                     int page_shift, int num_pages, int num_ids, int* __restrict__ status) {
  pdl_prologue(k_codes, k_exps, v_codes, v_exps, cu_q, q_start, page_indptr, page_indices);
  const int out_page = blockIdx.x, f = page_indptr[first] + out_page, page_size = 1 << page_shift;
  if (blockIdx.y == 0) {
    if (threadIdx.x == 0 && f < num_ids) ids[f] = out_page;
    // (the products behind this trust the tables: rows whose table is too short are found here)
    if (out_page == 0)
      for (int r = first + threadIdx.x; r < rows; r += 256)
        if (((page_indptr[r + 1] - page_indptr[r]) << page_shift) < q_start[r] + cu_q[r + 1] - cu_q[r]) atomicExch(status, 2);
  }
  if (f >= page_indptr[rows]) return;
  const int chunks = d >> 4, idx = blockIdx.y * 256 + threadIdx.x;
  if (idx >= nkv * page_size * chunks) return;
  int a = first, b = rows;  // the row of the entry
  while (b - a > 1) {
    const int mid = (a + b) / 2;
    if (page_indptr[mid] <= f) a = mid;
    else b = mid;
  }
  const int key = (f - page_indptr[a]) << page_shift, start = q_start[a], hi = start + cu_q[a + 1] - cu_q[a], lo = window > 0 ? max(0, start - window + 1) : 0;
  if (key + page_size <= lo || key >= hi) return;
  const int page = page_indices[f];
  if ((unsigned)page >= (unsigned)num_pages) {
    atomicExch(status, 2);
    return;
  }
  const int row = idx / chunks;
  const size_t from = (size_t)page * nkv * page_size, at = (from * chunks + idx) * 16, to = ((size_t)out_page * nkv * page_size * chunks + idx) * 16;
  const uint4 raw[2] = {*reinterpret_cast<const uint4*>(k_codes + at), *reinterpret_cast<const uint4*>(v_codes + at)};
  const int eb = k_exps[from + row], vb = v_exps[from + row];
  const float factor[2] = {c8_factor(vb == C8_NAN ? C8_NAN : eb), vb == C8_NAN ? 0.f : c8_factor(vb)};
#pragma unroll
  for (int w = 0; w < 2; ++w) c8_store16((w ? v_out : k_out) + to, raw[w], factor[w]);
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

MS_EXPORT int ms_cache8_write(void* q_out, void* k_codes, void* k_exps, void* v_codes, void* v_exps, const void* qkv, const void* q_norm_w, const void* k_norm_w,
                              const float* inv_freq, const float* cos_sin, const int* positions, const int* row_of_token, const int* page_indptr,
                              const int* page_indices, int num_tokens, int nq, int nkv, int d, int rot, float eps, int page_size, long long num_pages,
                              int* status, cudaStream_t stream) {
  if (num_tokens == 0) return 0;
  if (int rc = c8_check("cache8_write", nkv, d, page_size, num_pages)) return rc;
  MS_CHECK_ARG(nq >= 0 && num_tokens > 0, "cache8_write: nq=%d, %d tokens", nq, num_tokens);
  MS_CHECK_ARG(rot >= 0 && rot <= d && rot % 2 == 0, "cache8_write: rotary_dim=%d must be even and at most the head size %d", rot, d);
  MS_CHECK_ARG((uintptr_t)k_codes % 16 == 0 && (uintptr_t)v_codes % 16 == 0, "cache8_write: pools must be 16-byte aligned");
  if ((d == 64 || d == 128 || d == 256) && (rot == d || rot == 0 || inv_freq == nullptr) && (q_norm_w != nullptr) == (k_norm_w != nullptr) && (uintptr_t)qkv % 16 == 0 &&
      (uintptr_t)q_out % 16 == 0 && (uintptr_t)q_norm_w % 16 == 0 && (uintptr_t)k_norm_w % 16 == 0 && (uintptr_t)cos_sin % 16 == 0) {
    auto kernel = d == 64 ? cache8_write_token_kernel<64> : (d == 128 ? cache8_write_token_kernel<128> : cache8_write_token_kernel<256>);
    const int a_pass = 32 / (d / 16), warps = ceil_div(nq + 2 * nkv, a_pass) < 8 ? ceil_div(nq + 2 * nkv, a_pass) : 8;  // heads a warp and pass
    MS_LAUNCH(kernel, num_tokens, 32 * warps, 0, stream, (__nv_bfloat16*)q_out, (uint8_t*)k_codes, (uint8_t*)k_exps, (uint8_t*)v_codes, (uint8_t*)v_exps,
              (const __nv_bfloat16*)qkv, (const __nv_bfloat16*)q_norm_w, (const __nv_bfloat16*)k_norm_w, rot ? inv_freq : (const float*)nullptr, cos_sin, positions,
              row_of_token, page_indptr, page_indices, nq, nkv, eps, c8_page_shift(page_size), (int)num_pages, status);
    return 0;
  }
  const long long items = (long long)num_tokens * (nq + 2 * nkv);
  MS_LAUNCH(cache8_write_kernel, (unsigned)((items + 7) / 8), 256, 0, stream, (__nv_bfloat16*)q_out, (uint8_t*)k_codes, (uint8_t*)k_exps, (uint8_t*)v_codes,
            (uint8_t*)v_exps, (const __nv_bfloat16*)qkv, (const __nv_bfloat16*)q_norm_w, (const __nv_bfloat16*)k_norm_w, rot ? inv_freq : (const float*)nullptr,
            cos_sin, positions, row_of_token, page_indptr, page_indices, num_tokens, nq, nkv, d, rot, eps, c8_page_shift(page_size), (int)num_pages, status);
  return 0;
}

MS_EXPORT int ms_cache8_read(void* k_out, void* v_out, const void* k_codes, const void* k_exps, const void* v_codes, const void* v_exps, const int* positions,
                             const int* row_of_token, const int* page_indptr, const int* page_indices, int num_tokens, int nkv, int d, int page_size,
                             long long num_pages, int* status, int dtype, cudaStream_t stream) {
  if (num_tokens == 0) return 0;
  if (int rc = c8_check("cache8_read", nkv, d, page_size, num_pages)) return rc;
  MS_CHECK_ARG((uintptr_t)k_codes % 16 == 0 && (uintptr_t)v_codes % 16 == 0 && (uintptr_t)k_out % 16 == 0 && (uintptr_t)v_out % 16 == 0,
               "cache8_read: tensors must be 16-byte aligned");
  MS_CHECK_ARG(dtype == MS_F32 || dtype == MS_BF16, "cache8_read: dtype code %d", dtype);
  const long long items = (long long)num_tokens * nkv * (d / 16);
  const unsigned grid = (unsigned)((items + 255) / 256);
  if (dtype == MS_F32) {
    MS_LAUNCH(cache8_read_kernel<float>, grid, 256, 0, stream, (float*)k_out, (float*)v_out, (const uint8_t*)k_codes, (const uint8_t*)k_exps,
              (const uint8_t*)v_codes, (const uint8_t*)v_exps, positions, row_of_token, page_indptr, page_indices, num_tokens, nkv, d, c8_page_shift(page_size),
              (int)num_pages, status);
  } else {
    MS_LAUNCH(cache8_read_kernel<__nv_bfloat16>, grid, 256, 0, stream, (__nv_bfloat16*)k_out, (__nv_bfloat16*)v_out, (const uint8_t*)k_codes,
              (const uint8_t*)k_exps, (const uint8_t*)v_codes, (const uint8_t*)v_exps, positions, row_of_token, page_indptr, page_indices, num_tokens, nkv, d,
              c8_page_shift(page_size), (int)num_pages, status);
  }
  return 0;
}

// Rows [first, rows) list `entries` pages, which k_out and v_out [entries, nkv, page_size, d] hold; ids has num_ids numbers.
MS_EXPORT int ms_cache8_unpack(void* k_out, void* v_out, int* ids, const void* k_codes, const void* k_exps, const void* v_codes, const void* v_exps, const int* cu_q,
                               const int* q_start, const int* page_indptr, const int* page_indices, int first, int rows, int entries, int nkv, int d, int window, int page_size,
                               long long num_pages, int num_ids, int* status, cudaStream_t stream) {
  if (entries == 0) return 0;
  if (int rc = c8_check("cache8_unpack", nkv, d, page_size, num_pages)) return rc;
  MS_CHECK_ARG(first >= 0 && rows > first && entries > 0, "cache8_unpack: rows %d to %d, %d entries", first, rows, entries);
  MS_CHECK_ARG((uintptr_t)k_codes % 16 == 0 && (uintptr_t)v_codes % 16 == 0 && (uintptr_t)k_out % 16 == 0 && (uintptr_t)v_out % 16 == 0,
               "cache8_unpack: tensors must be 16-byte aligned");
  const int blocks = ceil_div(nkv * page_size * (d / 16), 256);
  MS_CHECK_ARG(blocks <= 65535, "cache8_unpack: pages of %d tokens and %d heads are too large", page_size, nkv);
  MS_LAUNCH(cache8_unpack_kernel, dim3(entries, blocks), 256, 0, stream, (__nv_bfloat16*)k_out, (__nv_bfloat16*)v_out, ids, (const uint8_t*)k_codes, (const uint8_t*)k_exps,
            (const uint8_t*)v_codes, (const uint8_t*)v_exps, cu_q, q_start, page_indptr, page_indices, first, rows, nkv, d, window, c8_page_shift(page_size), (int)num_pages,
            num_ids, status);
  return 0;
}
