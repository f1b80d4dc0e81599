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

__device__ __forceinline__ void c8_store16(float* dst, const float (&f)[16]) {
#pragma unroll
  for (int i = 0; i < 4; ++i) reinterpret_cast<float4*>(dst)[i] = make_float4(f[4 * i], f[4 * i + 1], f[4 * i + 2], f[4 * i + 3]);
}
__device__ __forceinline__ void c8_store16(__nv_bfloat16* dst, const float (&f)[16]) {
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
#pragma unroll
  for (int w = 0; w < 2; ++w) {
    const uint4 raw = *reinterpret_cast<const uint4*>((w ? v_codes : k_codes) + at * d + c * 16);
    const float factor = c8_factor((w ? v_exps : k_exps)[at]);
    const uint32_t words[4] = {raw.x, raw.y, raw.z, raw.w};
    float f[16];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const float2 lo = c8_float2(c8_half2_lo(words[i])), hi = c8_float2(c8_half2_hi(words[i]));
      f[4 * i] = lo.x * factor;
      f[4 * i + 1] = lo.y * factor;
      f[4 * i + 2] = hi.x * factor;
      f[4 * i + 3] = hi.y * factor;
    }
    c8_store16((w ? v_out : k_out) + (size_t)item * d + c * 16, f);
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

MS_EXPORT int ms_cache8_write(void* q_out, void* k_codes, void* k_exps, void* v_codes, void* v_exps, const void* qkv, const void* q_norm_w, const void* k_norm_w,
                              const float* inv_freq, const float* cos_sin, const int* positions, const int* row_of_token, const int* page_indptr,
                              const int* page_indices, int num_tokens, int nq, int nkv, int d, int rot, float eps, int page_size, long long num_pages,
                              int* status, cudaStream_t stream) {
  if (num_tokens == 0) return 0;
  if (int rc = c8_check("cache8_write", nkv, d, page_size, num_pages)) return rc;
  MS_CHECK_ARG(nq >= 0 && num_tokens > 0, "cache8_write: nq=%d, %d tokens", nq, num_tokens);
  MS_CHECK_ARG(rot >= 0 && rot <= d && rot % 2 == 0, "cache8_write: rotary_dim=%d must be even and at most the head size %d", rot, d);
  MS_CHECK_ARG((uintptr_t)k_codes % 16 == 0 && (uintptr_t)v_codes % 16 == 0, "cache8_write: pools must be 16-byte aligned");
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
