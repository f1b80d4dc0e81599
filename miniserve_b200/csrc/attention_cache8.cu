// Attention over the paged cache in 8 bits (cache8.cuh), compiled for ONE head size (-DMS_HEAD_DIM=D, a multiple of 16 up to 256): keys
// split over warps and CTAs.
//
// Formula: softmax(scale q k^T + causal mask) v; query head h reads kv head h / (heads / kv_heads), the query at position p sees keys 0..p or
// the last `window` of them, a sink adds exp(0) to the denominator (miniserve/model/attention.py:60-67, 125-133).
//
// Both products run on mma.sync with float32 sums, keys (and the head's channels) along the instruction's 16 rows and query rows along its 8
// columns: S^T = K Q^T, O^T = V^T P^T, so the few query rows of a decode step fill it. Codes become float16 (exact: e4m3 has 4 significant bits):
//   s_j = (q' . code_j) * qf * 2^ek_j,          q' = q * 2^sh in float16, with sh so that the row's largest |q'| lies in [2^14, 2^15): q's 8
//                                               significant bits are kept down to 2^-29 of the largest; qf = scale * log2(e) * 2^-sh
//   m + c >= max_j (s_j + ev_j) - 8             of scores and the values' exponents together, in two parts: m a largest score, c the rest (scores may be so
//                                               large that an exponent is lost beside them); moves only when it is passed by more than 8
//   o = sum_j 2^(s_j - m - c + 6 + ev_j) code(v_j),      l = sum_j 2^(s_j - m - c + 6)
// so a weight with its value's scale is at most 2^14, a float16 with 11 significant bits down to 2^-20 of the largest; l and o are float32. Exponents ev below the
// writer's least, -60, count as that in c, and what is left of them scales the weight behind: so no value, however small, makes the weights without their scale leave float32.
//
// Work: up to 8, 16 or (head sizes up to 64) 24 query rows (consecutive tokens of a request times the query heads of a kv head) and a kv head are an item; all
// items' slices of 32 keys in a row are cut into equal runs, one a warp, whatever the requests' lengths (or few items get a CTA each: alone_most). Each warp has a
// ring of stages of its own, filled by 16-byte copies that run on from item to item. What a warp has of an item that other warps of its CTA share lies in shared
// memory until all are done, and the warps add the pieces up together, in the warps' order. Items cut by a CTA's end leave one piece a CTA in global memory for a
// second small kernel. The lengths are read on the device, so a captured launch serves every context.
//
// What bounds it: the codes' bytes for full batches (64 requests of 1,024 to 3,985 keys, 8 kv heads of 128: 61 us, 5.4 TB/s, 0.83 of a copy), then the fixed
// latencies of a slice's chain with two warps a scheduler; for few keys the three dependent trips to memory before the first slice (4 us) and the second kernel
// (one token behind 299 keys 7.5 us, 8 behind 2,048 14.3).
#include "cache8.cuh"

#ifndef MS_HEAD_DIM
#error "compile with -DMS_HEAD_DIM=<head size>"
#endif

namespace ms {

constexpr int D = MS_HEAD_DIM;
static_assert(D % 16 == 0 && D >= 16 && D <= 256, "head size must be a multiple of 16 up to 256");
constexpr int CHUNKS = D / 16;                       // 16-byte chunks of a row of codes
constexpr int KSTEPS = D / 16, MTILES = D / 16;    // of q k^T along the head, of v^T p^T down it
constexpr int WIDE = D / 64, REST = (D % 64) / 16;   // k-steps of q k^T whose codes come four by four, and one by one
constexpr int VB = D % 128 == 0 ? 16 : (D % 64 == 0 ? 8 : 4), VBLOCKS = D / (8 * VB), VTAIL = D % 32 / 16;  // how a lane reads values: VB bytes a block
constexpr float LOG2E = 1.4426950408889634f;
constexpr int MOST_NT = D <= 64 ? 3 : 2;              // tiles of 8 query rows of an item at most: what the registers hold
constexpr int SLICE = 32, ROWS = 8 * MOST_NT;         // keys of a slice; the most query rows of an item
constexpr int ROW_BYTES = D % 64 == 0 ? D : D + 16;
constexpr int CODE_BYTES = SLICE * ROW_BYTES, STAGE_BYTES = 2 * CODE_BYTES + 2 * SLICE;  // K codes, V codes, K exponents, V exponents
// Warps of a CTA and stages of a warp's ring: one stage is worked on, the others are on their way. Head size 128, 64 requests of 1,024 to 3,985 keys: 7 warps of 3 stages
// 65.0 us, 8 of 2 61.9, 8 of 3 66.1, 9 of 2 65.1; 12 of 3 with slices of 16 keys 65.0 where 8 of 2 with 32 take 60.7.
constexpr int warps_of(int) { return D > 128 ? 4 : 8; }
constexpr int stages_of(int) { return D > 64 ? 2 : 4; }
constexpr int PART = D + 4;                          // floats of a row's partial: o, m, l, c (and one that keeps rows on 16 bytes)
// Items that are no more than CTAs get one each, whole, where the longest's warps then have a third and one slice more than in equal runs of `each`, at most three: that is what
// cutting costs (pieces, and a second kernel). Measured, us whole / cut: one token, 8 kv heads of 128, behind 300 keys (2 slices a warp to 1) 7.4 / 8.1, behind 600 (3 to 1) 8.4 / 8.2;
// 8 tokens behind 500 (3 to 2) 9.0 / 10.0, 1,000 (5 to 2) 11.3 / 10.3, 1,500 (6 to 3) 14.0 / 11.7; 16 behind 2,048 (9 to 8) 17.8 / 19.7, 4,000 (16 to 14) 26.6 / 29.4; 16
// requests of 5 drafted tokens, 4 kv heads of 64, behind 1,500 to 2,415 keys (10 to 7) 22.9 / 25.8.
__host__ __device__ constexpr int alone_most(int each) { return each + (1 + each / 3 < 3 ? 1 + each / 3 : 3); }
// Slices that going on to an item counts for in the row of slices (its queries, its pages, what is kept of the last one): warps that do have so many fewer. Measured, us with
// 0 / 1 / 2 / 3 / 4: 8 single tokens, 8 kv heads of 128, at 2,048 keys 15.3 / 14.7 / 14.0 / 14.0 / 14.0; 64 at 200 to 515 keys 19.5 / 18.9 / 18.0 / 18.4 / 18.5, at 1,024 to 3,985
// 60.5 / 60.9 / 60.0 / 59.9 / 60.6; 4 requests of 5 drafted tokens, 4 kv heads of 64, around 1,600 keys 20.8 / 18.1 / 18.2 / 18.1 / 17.9.
constexpr int SWITCH = 2;
constexpr int MAX_UNITS = 256;                       // (request, tile) pairs of a launch

__device__ __forceinline__ uint32_t smem_addr(const void* p) { return (uint32_t)__cvta_generic_to_shared(p); }
__device__ __forceinline__ void cp_async16(uint32_t dst, const void* src) { asm volatile("cp.async.cg.shared.global.L2::256B [%0], [%1], 16;\n" ::"r"(dst), "l"(src)); }
__device__ __forceinline__ void cp_async8(uint32_t dst, const void* src) { asm volatile("cp.async.ca.shared.global [%0], [%1], 8;\n" ::"r"(dst), "l"(src)); }
__device__ __forceinline__ void cp_async_commit() { asm volatile("cp.async.commit_group;\n" ::: "memory"); }
template <int N>
__device__ __forceinline__ void cp_async_wait() { asm volatile("cp.async.wait_group %0;\n" ::"n"(N) : "memory"); }
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
// over the eight lanes of equal lane % 4
__device__ __forceinline__ float oct_max(float v) {
  v = fmaxf(v, __shfl_xor_sync(0xffffffffu, v, 4));
  v = fmaxf(v, __shfl_xor_sync(0xffffffffu, v, 8));
  return fmaxf(v, __shfl_xor_sync(0xffffffffu, v, 16));
}
__device__ __forceinline__ float oct_sum(float v) {
  v += __shfl_xor_sync(0xffffffffu, v, 4);
  v += __shfl_xor_sync(0xffffffffu, v, 8);
  return v + __shfl_xor_sync(0xffffffffu, v, 16);
}
__device__ __forceinline__ float ex2(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;\n" : "=f"(y) : "f"(x));
  return y;
}
// an 8 x 8 tile of float16 pairs, rows across lane groups, transposed
__device__ __forceinline__ uint32_t transposed(uint32_t v) {
  uint32_t r;
  asm volatile("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;\n" : "=r"(r) : "r"(v));
  return r;
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
__device__ __forceinline__ float4 lds_float4(uint32_t at) {
  float4 v;
  asm volatile("ld.shared.v4.f32 {%0,%1,%2,%3}, [%4];\n" : "=f"(v.x), "=f"(v.y), "=f"(v.z), "=f"(v.w) : "r"(at));
  return v;
}
template <int BYTES>
__device__ __forceinline__ void lds_words(uint32_t (&v)[BYTES / 4], uint32_t at) {
  if constexpr (BYTES == 16) asm volatile("ld.shared.v4.u32 {%0,%1,%2,%3}, [%4];\n" : "=r"(v[0]), "=r"(v[1]), "=r"(v[2]), "=r"(v[3]) : "r"(at));
  if constexpr (BYTES == 8) asm volatile("ld.shared.v2.u32 {%0,%1}, [%2];\n" : "=r"(v[0]), "=r"(v[1]) : "r"(at));
  if constexpr (BYTES == 4) v[0] = lds32(at);
}

// Where chunk `chunk` of row `row` of a slice lies: chunks are swizzled so that the reads of keys (8 rows, 4 lanes a row) do not meet in a bank, nor
// those of values (4 rows of every second, the lanes of a row side by side).
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
  const int* page_indptr;   // [all_rows + 1]
  const int* page_indices;  // [num_entries]
  int* status;
  float* part;              // [2 * ctas][ROWS][PART]: a CTA's partial of the item that began before it, and of the one that goes on behind it
  int4* cut;                // [ctas]: for the second kernel, of the cut item that begins in the CTA: its first query row (counted in tokens x heads of a kv head), rows, kv head, pieces; 0: none
  int rows, tile0, tiles;   // requests; tiles [tile0, tile0 + tiles) of query rows of each
  int nq, nkv, window, sink, page_size, ctas;
  float scale;
  int num_pages;
  int behind;               // the second kernel runs: an item may be cut. 0 only where kv heads x rows x tiles are no more than CTAs
  int all_rows, num_entries;  // page_indptr[all_rows] is where all rows' tables end
  int ahead;                // the tables above, and the keys and values of tokens before the step's, were in place before the step's first kernel: read ahead of the wait
};

// The keys that a tile of query rows sees: those that some row does [lo, hi), those that all do [seen_lo, seen_hi).
struct Span {
  int lo, hi, seen_lo, seen_hi, first_slice;
};
__device__ __forceinline__ Span span_of(const Split8& p, int start, int row0, int rows_here, int group) {
  const int first = start + div_small(row0, group), last = start + div_small(row0 + rows_here - 1, group);
  Span s;
  s.lo = p.window > 0 ? max(0, first - p.window + 1) : 0;
  s.hi = last + 1;
  s.seen_lo = p.window > 0 ? max(0, last - p.window + 1) : 0;
  s.seen_hi = first + 1;
  s.first_slice = s.lo / SLICE;
  return s;
}

constexpr float ABOVE = 6.f, SLACK = 8.f;  // weights are in units of 2^(m + c - ABOVE); m + c is passed by at most SLACK
constexpr float START = -1e30f, NOTHING = -3e38f;  // c before the first key (m is 0 then); m of a partial without one

// o, m and l of a row, added up: out = o / l (a sink's term in the denominator), zero where no key was seen
__device__ __forceinline__ float sink_term(int sink, float m, float c) { return sink ? exp2f((ABOVE - c) - m) : 0.f; }

// What a CTA knows of a (request, tile) pair.
struct Unit {
  int at;                    // slices of all kv heads before it
  int n, stride;             // its slices of one kv head; how far apart its kv heads lie in the row of slices (n, or more: see `alone`)
  int tok0, start, row0, rows_here;
  int table, table_end;      // of its request in page_indices
  Span keys;
};
// An item that several warps of a CTA share.
struct Joint {
  int unit, kvh, last_warp, whole, piece;  // piece: which of the CTA's two in global memory, where it is not whole
};

// NT: tiles of 8 query rows of an item
template <int NT>
__global__ void __launch_bounds__(warps_of(NT) * 32, 1)
attn_cache8_split_kernel(__nv_bfloat16* __restrict__ out, const __nv_bfloat16* __restrict__ q, const uint8_t* __restrict__ k_codes,
                         const uint8_t* __restrict__ k_exps, const uint8_t* __restrict__ v_codes, const uint8_t* __restrict__ v_exps, const Split8 p, int part_rows) {
  constexpr int TILE_ROWS = 8 * NT, WARPS = warps_of(NT), THREADS = WARPS * 32, STAGES = stages_of(NT);
  extern __shared__ __align__(128) unsigned char smem[];
  __shared__ Unit table[MAX_UNITS + 1];
  __shared__ int scan[3][WARPS];
  __shared__ Joint joint[WARPS];  // by the warp that its CTA's share begins in; last_warp 0: none
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, g = lane >> 2, t = lane & 3;
  const int *cu_q = p.cu_q, *q_start = p.q_start, *page_indptr = p.page_indptr, *page_indices = p.page_indices;
  if (tid < WARPS) joint[tid].last_warp = 0;
  pdl_launch_dependents();
  if (!p.ahead) pdl_wait(q, k_codes, k_exps, v_codes, v_exps, cu_q, q_start, page_indptr, page_indices);

  const int group = div_small(p.nq, p.nkv), units = p.rows * p.tiles;
  // ---- where every tile's slices begin: a scan over the tiles, in order
  int live, total;
  {
    const int each = (units + THREADS - 1) / THREADS, first = tid * each;
    int slices = 0, count = 0, longest = 0;
    Unit mine;
    auto unit_of = [&](int u) {
      const int r = div_small(u, p.tiles);
      // (without a window a table is whole, and ends where the next begins; with one that says nothing: the step packer in csrc/host_core.cpp)
      const int tok_end = cu_q[r + 1], table_end = page_indptr[p.window > 0 ? p.all_rows : r + 1];
      mine.tok0 = cu_q[r];
      mine.start = q_start[r];
      mine.table = page_indptr[r];
      mine.table_end = min(table_end, p.num_entries);
      mine.row0 = (p.tile0 + u - r * p.tiles) * TILE_ROWS;
      const int rows_all = (tok_end - mine.tok0) * group;
      mine.rows_here = min(min(TILE_ROWS, part_rows), rows_all - mine.row0);  // (no more than there is room for)
      mine.n = 0;
      if (mine.rows_here > 0) {
        mine.keys = span_of(p, mine.start, mine.row0, mine.rows_here, group);
        mine.n = max(1, (mine.keys.hi + SLICE - 1) / SLICE - mine.keys.first_slice);  // (rows that see nothing have a slice, all of it masked)
      }
    };
    for (int u = first; u < min(first + each, units); ++u) {
      unit_of(u);
      slices += mine.n > 0 ? mine.n + SWITCH : 0;
      count += mine.n > 0;
      longest = max(longest, mine.n);
    }
    longest = __reduce_max_sync(0xffffffffu, longest);
    int s_incl = slices, c_incl = count;
#pragma unroll
    for (int off = 1; off < 32; off <<= 1) {
      const int a = __shfl_up_sync(0xffffffffu, s_incl, off), b = __shfl_up_sync(0xffffffffu, c_incl, off);
      if (lane >= off) {
        s_incl += a;
        c_incl += b;
      }
    }
    if (lane == 31) {
      scan[0][warp] = s_incl;
      scan[1][warp] = c_incl;
      scan[2][warp] = longest;
    }
    __syncthreads();
    int s_at = s_incl - slices, c_at = c_incl - count;
    live = total = longest = 0;
#pragma unroll
    for (int w = 0; w < WARPS; ++w) {
      if (w < warp) {
        s_at += scan[0][w];
        c_at += scan[1][w];
      }
      total += scan[0][w];
      live += scan[1][w];
      longest = max(longest, scan[2][w]);
    }
    // Few items, none much longer than an equal share: a CTA each, whole, so that nothing is left to add up behind. (Without the second kernel always: there are
    // no more items than CTAs then, whatever the lengths have become since the host looked at them.)
    const int longest_each = (longest + WARPS - 1) / WARPS, equal_each = (total * p.nkv + p.ctas * WARPS - 1) / (p.ctas * WARPS);
    const int alone = !p.behind || (live * p.nkv <= p.ctas && longest_each <= alone_most(equal_each)) ? longest_each * WARPS : 0;
    if (alone) total = live * alone;
    for (int u = first; u < min(first + each, units); ++u) {
      if (each > 1) unit_of(u);
      if (mine.n == 0) continue;
      mine.stride = alone ? alone : mine.n + SWITCH;
      mine.at = (alone ? c_at * alone : s_at) * p.nkv;
      table[c_at++] = mine;
      s_at += mine.n + SWITCH;
    }
    total *= p.nkv;
    if (tid == 0) table[live].at = total;
    __syncthreads();
    if (alone) live |= 1 << 30;
  }
  const bool alone = live >> 30;
  live &= (1 << 30) - 1;
  // ---- this warp's run of slices, [begin, end), and its CTA's
  const int each = alone ? table[0].stride / WARPS : (total + p.ctas * WARPS - 1) / (p.ctas * WARPS);
  const int cta_begin = min((int)blockIdx.x * each * WARPS, total), cta_end = min(cta_begin + each * WARPS, total);
  const int begin = min(cta_begin + warp * each, cta_end), end = min(begin + each, cta_end);
  auto find = [&](int pos) {  // the last tile that begins at or before `pos`
    int a = 0, b = live;
    while (b - a > 1) {
      const int mid = (a + b) / 2;
      if (table[mid].at <= pos) a = mid;
      else b = mid;
    }
    return a;
  };
  const uint32_t ring = smem_addr(smem) + warp * STAGES * STAGE_BYTES;
  float* heads = reinterpret_cast<float*>(smem + WARPS * STAGES * STAGE_BYTES);  // [warps][part_rows][PART]: of items that began before the warp's run
  float* tail = reinterpret_cast<float*>(smem + warp * STAGES * STAGE_BYTES);    // of the one that goes on behind it: the ring is done with by then
  const int page_shift = 31 - __clz(p.page_size);

  // ---- what is asked for. Pages are looked up 32 at a time, a lane each, and the next 32 while these are used.
  int a_pos = begin, a_left = 0, a_unit = find(begin), a_kvh = 0, a_key = 0, a_lo = 0, a_hi = 0, a_old = 0, a_table = 0, a_table_end = 0;
  int window = 0, page_ahead = 0, page_row = 0;  // the first of the 32 table entries; the lane's page of the next ones; the pool's row at which its page of these begins
  const int first_unit = a_unit;
  auto page_of = [&](int entry) {
    const int key = entry << page_shift;
    if (key + p.page_size <= a_lo || key >= a_hi) return 0;  // (not needed: any page that is there)
    const int at = a_table + entry;
    return at >= 0 && at < a_table_end ? page_indices[at] : -1;
  };
  auto turn = [&]() {  // to the entries looked up last
    int page = page_ahead;
    if ((unsigned)page >= (unsigned)p.num_pages) {
      atomicExch(p.status, 2);
      page = 0;  // (what comes of it is not used)
    }
    page_row = (page * p.nkv + a_kvh) << page_shift;
    page_ahead = page_of(window + 32 + lane);
  };
  auto next_item = [&]() {  // the item that a_pos lies in, if there is one
    while (a_pos < end) {
      const Unit& u = table[a_unit];
      const int past = a_pos - u.at;
      a_kvh = div_small(past, u.stride);
      const int off = past - a_kvh * u.stride;
      if (a_kvh >= p.nkv) {
        ++a_unit;
      } else if (off >= u.n) {  // (behind a lone item's end)
        a_pos += u.stride - off;
      } else {
        a_lo = u.keys.lo;
        a_hi = u.keys.hi;
        a_old = u.start;
        a_key = (u.keys.first_slice + off) * SLICE;
        a_table = u.table;
        a_table_end = u.table_end;
        a_left = min(u.n - off, end - a_pos);
        window = a_key >> page_shift;
        page_ahead = page_of(window + lane);
        return;
      }
    }
  };
  bool turned = false;  // (the first look at an item's pages waits until the copies are made)
  auto fire = [&](uint32_t st) {  // the slice looked up last, into a stage; then the next one is looked up
    if (a_left > 0) {
      if (!turned) {
        turn();
        turned = true;
      } else if ((a_key >> page_shift) - window >= 32) {
        window += 32;
        turn();
      }
      const uint32_t kt = st, vt = st + CODE_BYTES, et = st + 2 * CODE_BYTES;
      int rows8[SLICE / 8];  // the pool's rows at which every eight keys begin
#pragma unroll
      for (int i = 0; i < SLICE / 8; ++i) {
        const int key = a_key + 8 * i;
        rows8[i] = __shfl_sync(0xffffffffu, page_row, (key >> page_shift) - window) + (key & (p.page_size - 1));
      }
      if (8 * CHUNKS % 32 == 0) {
#pragma unroll
        for (int i = 0; i < SLICE / 8; ++i) {
          const size_t at = (size_t)rows8[i] * D + lane * 16;
#pragma unroll
          for (int c = 0; c < 8 * CHUNKS / 32; ++c) {
            const int idx = c * 32 + lane, row = idx / CHUNKS, chunk = idx - row * CHUNKS;
            cp_async16(kt + chunk_at(8 * i + row, chunk), k_codes + at + c * 512);
            cp_async16(vt + chunk_at(8 * i + row, chunk), v_codes + at + c * 512);
          }
        }
      } else {
#pragma unroll
        for (int i = 0; i < SLICE / 8; ++i)
          for (int idx = lane; idx < 8 * CHUNKS; idx += 32) {
            const int row = idx / CHUNKS, chunk = idx - row * CHUNKS;
            cp_async16(kt + chunk_at(8 * i + row, chunk), k_codes + (size_t)rows8[i] * D + idx * 16);
            cp_async16(vt + chunk_at(8 * i + row, chunk), v_codes + (size_t)rows8[i] * D + idx * 16);
          }
      }
      const int mine = (lane & 2) ? ((lane & 1) ? rows8[3] : rows8[2]) : ((lane & 1) ? rows8[1] : rows8[0]);
      if (lane < 8) cp_async8(et + lane * 8, (lane < 4 ? k_exps : v_exps) + mine);  // exponents, 8 a lane: of K, then of V
      ++a_pos;
      a_key += SLICE;
      if (--a_left == 0) {
        next_item();
        turned = false;
      }
    }
    cp_async_commit();
  };
  next_item();
  int filled = 0;  // stages asked for
  if (p.ahead) {
    // slices of tokens before the step's; the others, and the queries, come from the kernels before this one
#pragma unroll 1
    for (; filled < STAGES && a_left > 0 && a_key + SLICE <= a_old; ++filled) fire(ring + filled * STAGE_BYTES);
    pdl_wait(q, k_codes, k_exps, v_codes, v_exps, cu_q, q_start, page_indptr, page_indices);
  }
  if (tid == 0 && p.behind) {
    int4 cut = make_int4(0, 0, 0, 0);
    if (cta_begin < cta_end && !alone) {
      const Unit& u = table[find(cta_end - 1)];
      const int kvh = div_small(cta_end - 1 - u.at, u.stride), at = u.at + kvh * u.stride;
      // the item that goes on behind the CTA's end, where it began in this CTA
      if (at >= cta_begin && at + u.n > cta_end) cut = make_int4(u.tok0 * group + u.row0, u.rows_here, kvh, (at + u.n - 1) / (each * WARPS) - (int)blockIdx.x + 1);
    }
    p.cut[blockIdx.x] = cut;
  }

  // ---- what is computed
  int unit = first_unit, kvh = 0, item_end = begin, item_begin = 0;
  int start = 0, row0 = 0, rows_here = 0, tok0 = 0, n = 0;
  Span it = {};
  uint32_t qf[NT][KSTEPS][2];
  float row_factor[NT][2];
  int q_pos[NT][2];
  float o[NT][MTILES][4], m_run[NT][2], c_run[NT][2], l_run[NT][2];
  uint32_t st = ring;

  for (int pos = begin; pos < end; ++pos) {
    if (pos >= item_end) {
      // ---- a new item: its queries, from memory straight into the fragments
      for (;; ++unit) {
        kvh = div_small(pos - table[unit].at, table[unit].stride);
        if (kvh < p.nkv) break;
      }
      {
        const Unit& u = table[unit];
        n = u.n;
        item_begin = u.at + kvh * u.stride;
        item_end = min(item_begin + n, end);
        if (pos >= item_begin + n) {  // (behind a lone item's end)
          pos = item_begin + u.stride - 1;
          item_end = 0;
          continue;
        }
        start = u.start;
        row0 = u.row0;
        rows_here = u.rows_here;
        tok0 = u.tok0;
        it = u.keys;
      }
      uint2 raw[NT][KSTEPS];
#pragma unroll
      for (int j = 0; j < NT; ++j) {
        const int i = g + 8 * j, row = row0 + i, tok = div_small(row, group);
        const __nv_bfloat16* src = q + ((size_t)(tok0 + tok) * p.nq + kvh * group + (row - tok * group)) * D;
#pragma unroll
        for (int kk = 0; kk < KSTEPS; ++kk) {
          raw[j][kk] = make_uint2(0u, 0u);
          if (i < rows_here) raw[j][kk] = *reinterpret_cast<const uint2*>(src + channel_of(kk, t));
        }
      }
      // (the first copies go out while the first queries are on their way)
#pragma unroll 1
      for (; filled < STAGES; ++filled) fire(ring + filled * STAGE_BYTES);
#pragma unroll
      for (int j = 0; j < NT; ++j) {
        uint32_t bits = 0;
#pragma unroll
        for (int kk = 0; kk < KSTEPS; ++kk) {
          const uint32_t x = raw[j][kk].x, y = raw[j][kk].y;
          bits = max(bits, max(max((x << 16) & 0x7FFFFFFFu, x & 0x7FFF0000u), max((y << 16) & 0x7FFFFFFFu, y & 0x7FFF0000u)));
        }
        bits = max(bits, __shfl_xor_sync(0xffffffffu, bits, 1));
        bits = max(bits, __shfl_xor_sync(0xffffffffu, bits, 2));
        // the row's power of two (a query that is not finite leaves its row NaN whatever it is multiplied by)
        const int field = (int)(bits >> 23), sh = field > 0 && field < 255 ? min(max(14 + 127 - field, -113), 100) : 0;
        const float up = __uint_as_float((uint32_t)(127 + sh) << 23), down = p.scale * LOG2E * __uint_as_float((uint32_t)(127 - sh) << 23);
#pragma unroll
        for (int c = 0; c < 2; ++c) {
          q_pos[j][c] = start + div_small(row0 + 8 * j + 2 * t + c, group);
          row_factor[j][c] = __shfl_sync(0xffffffffu, down, (2 * t + c) * 4);
        }
#pragma unroll
        for (int kk = 0; kk < KSTEPS; ++kk) {
          const uint32_t x = raw[j][kk].x, y = raw[j][kk].y;
          qf[j][kk][0] = pack_half2(__uint_as_float(x << 16) * up, __uint_as_float(x & 0xFFFF0000u) * up);
          qf[j][kk][1] = pack_half2(__uint_as_float(y << 16) * up, __uint_as_float(y & 0xFFFF0000u) * up);
        }
#pragma unroll
        for (int i = 0; i < MTILES; ++i) o[j][i][0] = o[j][i][1] = o[j][i][2] = o[j][i][3] = 0.f;
        m_run[j][0] = m_run[j][1] = 0.f;
        c_run[j][0] = c_run[j][1] = START;
        l_run[j][0] = l_run[j][1] = 0.f;
      }
    }
    // ---- a slice: its halves of 16 keys are two of the instruction's row tiles
    cp_async_wait<STAGES - 1>();
    __syncwarp();
    const uint32_t kt = st, vt = kt + CODE_BYTES, et = kt + 2 * CODE_BYTES;
    float s[2][NT][4];
    uint32_t vb[2][2];                       // the exponents' bytes of the values g, g + 8, g + 16, g + 24
    float vf[2][2], kfac[2][2];              // 2^ev, of the writer's least exponent at least, and 2^ek (255: infinity, which the codes of such a vector, all zero, make NaN)
#pragma unroll
    for (int h = 0; h < 2; ++h) {
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        kfac[h][i] = c8_power(lds8(et + 16 * h + 8 * i + g));
        vb[h][i] = lds8(et + SLICE + 16 * h + 8 * i + g);
        vf[h][i] = c8_power(max(vb[h][i], (uint32_t)C8_EXP_MIN));
      }
#pragma unroll
      for (int j = 0; j < NT; ++j) s[h][j][0] = s[h][j][1] = s[h][j][2] = s[h][j][3] = 0.f;
    }
#pragma unroll
    for (int grp = 0; grp < WIDE; ++grp) {
      uint32_t kw[2][2][4];
      const int chunk = channel_of(grp * 4, t) >> 4;
#pragma unroll
      for (int h = 0; h < 2; ++h)
#pragma unroll
        for (int i = 0; i < 2; ++i) lds_words<16>(kw[h][i], kt + chunk_at(16 * h + 8 * i + g, chunk));
#pragma unroll
      for (int w = 0; w < 4; ++w)
#pragma unroll
        for (int h = 0; h < 2; ++h) {
          const uint32_t kf[4] = {c8_half2_lo(kw[h][0][w]), c8_half2_lo(kw[h][1][w]), c8_half2_hi(kw[h][0][w]), c8_half2_hi(kw[h][1][w])};
#pragma unroll
          for (int j = 0; j < NT; ++j) mma_f16(s[h][j], kf, qf[j][grp * 4 + w][0], qf[j][grp * 4 + w][1]);
        }
    }
#pragma unroll
    for (int rest = 0; rest < REST; ++rest) {
      const int kk = WIDE * 4 + rest;
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        const uint32_t top = lds32(kt + chunk_at(16 * h + g, kk) + 4 * t), low = lds32(kt + chunk_at(16 * h + g + 8, kk) + 4 * t);
        const uint32_t kf[4] = {c8_half2_lo(top), c8_half2_lo(low), c8_half2_hi(top), c8_half2_hi(low)};
#pragma unroll
        for (int j = 0; j < NT; ++j) mma_f16(s[h][j], kf, qf[j][kk][0], qf[j][kk][1]);
      }
    }
    const int key0 = (it.first_slice + pos - item_begin) * SLICE;
    const bool edge = key0 < it.seen_lo || key0 + SLICE > it.seen_hi;  // some row does not see all of the slice
    if (edge && (key0 < it.lo || key0 + SLICE > it.hi)) {
      // values that must not be weighed, not even by zero (they may hold anything)
      for (int idx = lane; idx < SLICE * CHUNKS; idx += 32) {
        const int row = idx / CHUNKS, chunk = idx - row * CHUNKS;
        if (key0 + row < it.lo || key0 + row >= it.hi) asm volatile("st.shared.v4.b32 [%0], {%1, %1, %1, %1};\n" ::"r"(vt + chunk_at(row, chunk)), "r"(0) : "memory");
      }
      __syncwarp();
    }
    // scores in units of log2, relative to m, masked; weights 2^(s - m - c + ABOVE) times the values' 2^ev
    float x[2][NT][4], w[2][NT][4];
    auto weigh = [&]() {
      float most = 0.f;
#pragma unroll
      for (int j = 0; j < NT; ++j)
#pragma unroll
        for (int h = 0; h < 2; ++h)
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            x[h][j][e] = ex2(s[h][j][e] + (ABOVE - c_run[j][e & 1]));
            w[h][j][e] = x[h][j][e] * vf[h][e >> 1];
          }
      if (edge) {  // (a value that is NaN, or no value at all, reaches only who sees it)
#pragma unroll
        for (int j = 0; j < NT; ++j)
#pragma unroll
          for (int h = 0; h < 2; ++h)
#pragma unroll
            for (int e = 0; e < 4; ++e) w[h][j][e] = s[h][j][e] == -INFINITY ? 0.f : w[h][j][e];
      }
#pragma unroll
      for (int j = 0; j < NT; ++j)
#pragma unroll
        for (int h = 0; h < 2; ++h)
#pragma unroll
          for (int e = 0; e < 4; ++e) most = fmaxf(most, w[h][j][e]);
      return most;
    };
#pragma unroll
    for (int j = 0; j < NT; ++j)
#pragma unroll
      for (int h = 0; h < 2; ++h)
#pragma unroll
        for (int e = 0; e < 4; ++e) s[h][j][e] = fmaf(s[h][j][e], row_factor[j][e & 1] * kfac[h][e >> 1], -m_run[j][e & 1]);
    if (edge) {
#pragma unroll
      for (int j = 0; j < NT; ++j)
#pragma unroll
        for (int h = 0; h < 2; ++h)
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            const int key = key0 + 16 * h + g + 8 * (e >> 1), qp = q_pos[j][e & 1];
            if (key > qp || (p.window > 0 && key <= qp - p.window)) s[h][j][e] = -INFINITY;
          }
    }
    // m + c moves only where a weight passes 2^(ABOVE + SLACK); values of exponents below the writer's least come this way too
    const bool small = min(min(vb[0][0], vb[0][1]), min(vb[1][0], vb[1][1])) < (uint32_t)C8_EXP_MIN;
    if (__any_sync(0xffffffffu, weigh() > exp2f(ABOVE + SLACK) || small)) {
#pragma unroll
      for (int j = 0; j < NT; ++j)
#pragma unroll
        for (int c = 0; c < 2; ++c) {
          // the largest score, relative to the one before, then the largest score with its exponent, relative to that
          float up = oct_max(fmaxf(fmaxf(s[0][j][c], s[0][j][2 + c]), fmaxf(s[1][j][c], s[1][j][2 + c]))), c_new = -INFINITY;
          if (up == -INFINITY || (up < 0.f && c_run[j][c] > START)) up = 0.f;  // (the first key's score is taken whatever its sign)
#pragma unroll
          for (int h = 0; h < 2; ++h)
#pragma unroll
            for (int i = 0; i < 2; ++i) {
              s[h][j][2 * i + c] -= up;
              c_new = fmaxf(c_new, s[h][j][2 * i + c] + (float)(max((int)vb[h][i], C8_EXP_MIN) - 127));
            }
          c_new = fmaxf(c_run[j][c] - up, oct_max(c_new));
          const float alpha = ex2((c_run[j][c] - up) - c_new);
          m_run[j][c] += up;
          c_run[j][c] = c_new;
          l_run[j][c] *= alpha;
#pragma unroll
          for (int i = 0; i < MTILES; ++i) {
            o[j][i][c] *= alpha;
            o[j][i][2 + c] *= alpha;
          }
        }
      weigh();
#pragma unroll
      for (int h = 0; h < 2; ++h)
#pragma unroll
        for (int i = 0; i < 2; ++i) {
          const float rest = c8_power(127 - (uint32_t)max(C8_EXP_MIN - (int)vb[h][i], 0));
#pragma unroll
          for (int j = 0; j < NT; ++j) {
            w[h][j][2 * i] *= rest;
            w[h][j][2 * i + 1] *= rest;
          }
        }
    }
    uint32_t wf[2][NT][2];
#pragma unroll
    for (int j = 0; j < NT; ++j)
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        l_run[j][0] += x[h][j][0] + x[h][j][2];
        l_run[j][1] += x[h][j][1] + x[h][j][3];
        wf[h][j][0] = transposed(pack_half2(w[h][j][0], w[h][j][1]));
        wf[h][j][1] = transposed(pack_half2(w[h][j][2], w[h][j][3]));
      }
    // values: lane group g's channels of the rows 2t, 2t + 1, 2t + 8, 2t + 9, paired along the keys byte by byte
#pragma unroll
    for (int h = 0; h < 2; ++h) {
#pragma unroll
      for (int blk = 0; blk < VBLOCKS; ++blk) {
        uint32_t vw[4][VB / 4];
        const int ch = blk * 8 * VB + g * VB;
#pragma unroll
        for (int i = 0; i < 4; ++i) lds_words<VB>(vw[i], vt + chunk_at(16 * h + 2 * t + (i & 1) + 8 * (i >> 1), ch >> 4) + (ch & 15));
#pragma unroll
        for (int w = 0; w < VB / 4; ++w) {
          const uint32_t b0 = __byte_perm(vw[0][w], vw[1][w], 0x5140), b1 = __byte_perm(vw[2][w], vw[3][w], 0x5140);
          const uint32_t c0 = __byte_perm(vw[0][w], vw[1][w], 0x7362), c1 = __byte_perm(vw[2][w], vw[3][w], 0x7362);
          const uint32_t va[4] = {c8_half2_lo(b0), c8_half2_hi(b0), c8_half2_lo(b1), c8_half2_hi(b1)};
          const uint32_t vc[4] = {c8_half2_lo(c0), c8_half2_hi(c0), c8_half2_lo(c1), c8_half2_hi(c1)};
          const int mt = blk * (VB / 2) + w * 2;
#pragma unroll
          for (int j = 0; j < NT; ++j) {
            mma_f16(o[j][mt], va, wf[h][j][0], wf[h][j][1]);
            mma_f16(o[j][mt + 1], vc, wf[h][j][0], wf[h][j][1]);
          }
        }
      }
      if (VTAIL) {
        const int ch = VBLOCKS * 8 * VB + 2 * g;
        uint32_t vw[4];
#pragma unroll
        for (int i = 0; i < 4; ++i) vw[i] = lds16(vt + chunk_at(16 * h + 2 * t + (i & 1) + 8 * (i >> 1), ch >> 4) + (ch & 15));
        const uint32_t b0 = __byte_perm(vw[0], vw[1], 0x5140), b1 = __byte_perm(vw[2], vw[3], 0x5140);
        const uint32_t va[4] = {c8_half2_lo(b0), c8_half2_hi(b0), c8_half2_lo(b1), c8_half2_hi(b1)};
#pragma unroll
        for (int j = 0; j < NT; ++j) mma_f16(o[j][MTILES - 1], va, wf[h][j][0], wf[h][j][1]);
      }
    }
    __syncwarp();
    fire(st);
    st = st + STAGE_BYTES == ring + STAGES * STAGE_BYTES ? ring : st + STAGE_BYTES;

    if (pos + 1 < item_end) continue;
    // ---- this warp's last slice of the item
#pragma unroll
    for (int j = 0; j < NT; ++j)
#pragma unroll
      for (int c = 0; c < 2; ++c) {
        l_run[j][c] = oct_sum(l_run[j][c]);
        if (c_run[j][c] == START) m_run[j][c] = NOTHING;
      }
    const int seg_begin = max(item_begin, cta_begin), seg_end = min(item_begin + n, cta_end);  // the CTA's share of it
    const int first_warp = div_small(seg_begin - cta_begin, each), last_warp = div_small(seg_end - 1 - cta_begin, each);
    const bool whole = seg_begin == item_begin && seg_end == item_begin + n;
    float* piece = p.part + (size_t)(2 * blockIdx.x + (seg_begin == item_begin)) * ROWS * PART;  // (a cut item: began before this CTA, or goes on behind it)
    __nv_bfloat16* dst = out + ((size_t)tok0 * p.nq + kvh * group) * D;
    auto row_of = [&](int row) {  // where query row `row` of the item begins in the output
      const int rho = row0 + row, tok = div_small(rho, group);
      return dst + ((size_t)tok * p.nq + (rho - tok * group)) * D;
    };
    // the lane group's channels 2 i and 2 i + 1 of a block
    auto channel = [&](int i) { return i < VBLOCKS * (VB / 2) ? i / (VB / 2) * 8 * VB + g * VB + i % (VB / 2) * 2 : VBLOCKS * 8 * VB + 2 * g; };
    if (first_warp == last_warp && whole) {
      // nobody else has a share of it
#pragma unroll
      for (int j = 0; j < NT; ++j)
#pragma unroll
        for (int c = 0; c < 2; ++c) {
          if (8 * j + 2 * t + c >= rows_here) continue;
          const float den = l_run[j][c] + sink_term(p.sink, m_run[j][c], c_run[j][c]), inv = den == 0.f ? 0.f : 1.0f / den;
          __nv_bfloat16* row = row_of(8 * j + 2 * t + c);
#pragma unroll
          for (int i = 0; i < MTILES; ++i)
            *reinterpret_cast<__nv_bfloat162*>(row + channel(i)) = __floats2bfloat162_rn(o[j][i][c] * inv, o[j][i][2 + c] * inv);
        }
      continue;
    }
    // its piece: to global memory where it is the CTA's only one, else to shared memory
    const bool lone = first_warp == last_warp, is_tail = !lone && warp == first_warp;
    if (is_tail) cp_async_wait<0>();  // (the ring's last, empty groups)
    float* area = lone ? piece : (is_tail ? tail : heads + (size_t)warp * part_rows * PART);
#pragma unroll
    for (int j = 0; j < NT; ++j)
#pragma unroll
      for (int c = 0; c < 2; ++c) {
        if (8 * j + 2 * t + c >= rows_here) continue;
        float* row = area + (size_t)(8 * j + 2 * t + c) * PART;
#pragma unroll
        for (int i = 0; i < MTILES; ++i) *reinterpret_cast<float2*>(row + channel(i)) = make_float2(o[j][i][c], o[j][i][2 + c]);
        if (g == 0) *reinterpret_cast<float4*>(row + D) = make_float4(m_run[j][c], l_run[j][c], c_run[j][c], 0.f);
      }
    if (is_tail && lane == 0) joint[warp] = {unit, kvh, last_warp, whole, seg_begin == item_begin};
  }
  cp_async_wait<0>();
  __syncthreads();
  // ---- items that warps share: their rows one by one, a row a warp
  int task = 0;
  for (int first_warp = 0; first_warp < WARPS; ++first_warp) {
    const Joint item = joint[first_warp];
    if (item.last_warp == 0) continue;
    const Unit& u = table[item.unit];
    for (int row = 0; row < u.rows_here; ++row) {
      if (task++ % WARPS != warp) continue;
      // every lane has all pieces' numbers (no exchanges between lanes: their latency is what a row would take)
      float4 mlc[WARPS];
      uint32_t at[WARPS];
#pragma unroll
      for (int w = 0; w < WARPS; ++w) {
        at[w] = (w == first_warp ? smem_addr(smem) + first_warp * STAGES * STAGE_BYTES : smem_addr(heads) + w * part_rows * PART * 4) + row * PART * 4;
        mlc[w] = w >= first_warp && w <= item.last_warp ? lds_float4(at[w] + D * 4) : make_float4(NOTHING, 0.f, 0.f, 0.f);
      }
      float m = NOTHING, c_all = -INFINITY, l = 0.f, wgt[WARPS];
#pragma unroll
      for (int w = 0; w < WARPS; ++w) m = fmaxf(m, mlc[w].x);
#pragma unroll
      for (int w = 0; w < WARPS; ++w) {
        wgt[w] = w >= first_warp && w <= item.last_warp ? (mlc[w].x - m) + mlc[w].z : -INFINITY;
        c_all = fmaxf(c_all, wgt[w]);
      }
#pragma unroll
      for (int w = 0; w < WARPS; ++w) {
        wgt[w] = ex2(wgt[w] - c_all);
        l += wgt[w] * mlc[w].y;
      }
      const float den = l + sink_term(p.sink, m, c_all), inv = den == 0.f ? 0.f : 1.0f / den;
      const int rho = u.row0 + row, tok = div_small(rho, group);
      __nv_bfloat16* dst = out + ((size_t)(u.tok0 + tok) * p.nq + item.kvh * group + (rho - tok * group)) * D;
      float* piece = p.part + ((size_t)(2 * blockIdx.x + item.piece) * ROWS + row) * PART;
#pragma unroll
      for (int c0 = 0; c0 < D; c0 += 128) {
        const int c = min(c0 + 4 * lane, D - 4);
        float4 x[WARPS], acc = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
        for (int w = 0; w < WARPS; ++w) x[w] = w >= first_warp && w <= item.last_warp ? lds_float4(at[w] + c * 4) : make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
        for (int w = 0; w < WARPS; ++w) {
          acc.x += wgt[w] * x[w].x;
          acc.y += wgt[w] * x[w].y;
          acc.z += wgt[w] * x[w].z;
          acc.w += wgt[w] * x[w].w;
        }
        if (c0 + 4 * lane >= D) continue;
        if (item.whole) {
          uint2 pk;
          __nv_bfloat162 lo2 = __floats2bfloat162_rn(acc.x * inv, acc.y * inv), hi2 = __floats2bfloat162_rn(acc.z * inv, acc.w * inv);
          pk.x = *reinterpret_cast<uint32_t*>(&lo2);
          pk.y = *reinterpret_cast<uint32_t*>(&hi2);
          *reinterpret_cast<uint2*>(dst + c) = pk;
        } else {
          *reinterpret_cast<float4*>(piece + c) = acc;
        }
      }
      if (!item.whole && lane == 0) *reinterpret_cast<float4*>(piece + D) = make_float4(m, l, c_all, 0.f);
    }
  }
}

// The items that were cut: a CTA's second partial and its successors' first ones, added up in their order. Block (cta, row). Threads side by side take
// 4 channels each, shares of them every SHARES-th piece. Up to 4 pieces (requests of a batch): every lane has all their numbers, asked for together with the question how many
// there are (their places are there in any case). Up to 32 (one long request): a lane has a piece's, all that a thread adds up is asked for at once, and every warp makes the weights
// for itself: 50.9 us for the call behind 131,072 keys, 8 kv heads of 128, against 52.4 with a block's maxima and sums one behind the other, as beyond 32.
constexpr int MERGE_THREADS = 128;
__global__ void __launch_bounds__(MERGE_THREADS)
attn_cache8_merge_kernel(__nv_bfloat16* __restrict__ out, const Split8 p) {
  const int4* cuts = p.cut;
  const float* parts = p.part;
  pdl_prologue(cuts, parts);
  constexpr int COLS = D / 4, SHARES = MERGE_THREADS / COLS, EACH = (32 + SHARES - 1) / SHARES, EARLY = 4;
  const int cta = blockIdx.x, row = blockIdx.y, group = p.nq / p.nkv, tid = threadIdx.x, lane = tid & 31, col = tid % COLS, share = tid / COLS;
  auto at = [&](int i) { return parts + ((size_t)(2 * min(cta + i, p.ctas - 1) + (i == 0)) * ROWS + row) * PART; };
  const int4 cut = cuts[cta];
  float4 first[EARLY];
#pragma unroll
  for (int i = 0; i < EARLY; ++i) first[i] = *reinterpret_cast<const float4*>(at(i) + D);
  const float4 mine = *reinterpret_cast<const float4*>(at(share) + 4 * col);
  if (cut.w < 2 || row >= cut.y) return;
  __shared__ float4 sums[MERGE_THREADS];
  __shared__ float weight[MERGE_THREADS], red[MERGE_THREADS / 32];
  float m = NOTHING, c_all = -INFINITY, l = 0.f;
  float4 acc = make_float4(0.f, 0.f, 0.f, 0.f);
  auto add = [&](const float4& x, float w) {
    acc.x += w * x.x;
    acc.y += w * x.y;
    acc.z += w * x.z;
    acc.w += w * x.w;
  };
  // the largest m of all pieces, then the largest m + c, the weights and the sum of the weighed l
  if (cut.w <= EARLY) {
    float w[EARLY];
#pragma unroll
    for (int i = 0; i < EARLY; ++i) m = i < cut.w ? fmaxf(m, first[i].x) : m;
#pragma unroll
    for (int i = 0; i < EARLY; ++i) {
      w[i] = i < cut.w ? (first[i].x - m) + first[i].z : -INFINITY;
      c_all = fmaxf(c_all, w[i]);
    }
#pragma unroll
    for (int i = 0; i < EARLY; ++i) {
      w[i] = ex2(w[i] - c_all);
      if (i < cut.w) l += w[i] * first[i].y;
      if (i == share && i < cut.w) add(mine, w[i]);
    }
    if (share < SHARES)
      for (int i = share + SHARES; i < cut.w; i += SHARES) add(*reinterpret_cast<const float4*>(at(i) + 4 * col), ex2(((at(i)[D] - m) + at(i)[D + 2]) - c_all));
  } else if (cut.w <= 32) {
    const float4 head = *reinterpret_cast<const float4*>(at(lane) + D);
    float4 x[EACH];
#pragma unroll
    for (int i = 0; i < EACH; ++i) {
      x[i] = i == 0 ? mine : make_float4(0.f, 0.f, 0.f, 0.f);
      if (i > 0 && share + i * SHARES < cut.w) x[i] = *reinterpret_cast<const float4*>(at(share + i * SHARES) + 4 * col);
    }
    m = warp_max(lane < cut.w ? head.x : NOTHING);
    const float rel = lane < cut.w ? (head.x - m) + head.z : -INFINITY;
    c_all = warp_max(rel);
    const float w = ex2(rel - c_all);
    l = warp_sum(lane < cut.w ? w * head.y : 0.f);
#pragma unroll
    for (int i = 0; i < EACH; ++i) {
      const int piece = share + i * SHARES;
      const float wi = __shfl_sync(0xffffffffu, w, piece & 31);
      if (share < SHARES && piece < cut.w) add(x[i], wi);
    }
  } else {
    auto block_max = [&](float v) {
      v = warp_max(v);
      __syncthreads();
      if (tid % 32 == 0) red[tid / 32] = v;
      __syncthreads();
      return fmaxf(fmaxf(red[0], red[1]), fmaxf(red[2], red[3]));
    };
    for (int i = tid; i < cut.w; i += MERGE_THREADS) m = fmaxf(m, at(i)[D]);
    m = block_max(m);
    for (int i = tid; i < cut.w; i += MERGE_THREADS) c_all = fmaxf(c_all, (at(i)[D] - m) + at(i)[D + 2]);
    c_all = block_max(c_all);
    for (int first = 0; first < cut.w; first += MERGE_THREADS) {
      __syncthreads();
      if (first + tid < cut.w) {
        const float4 h = *reinterpret_cast<const float4*>(at(first + tid) + D);
        weight[tid] = ex2(((h.x - m) + h.z) - c_all);
        l += weight[tid] * h.y;
      }
      __syncthreads();
      if (share < SHARES) {
#pragma unroll 8
        for (int i = share; i < min(MERGE_THREADS, cut.w - first); i += SHARES) add(*reinterpret_cast<const float4*>(at(first + i) + 4 * col), weight[i]);
      }
    }
    l = warp_sum(l);
    __syncthreads();
    if (tid % 32 == 0) red[tid / 32] = l;
    __syncthreads();
    l = (red[0] + red[1]) + (red[2] + red[3]);
  }
  sums[tid] = acc;
  __syncthreads();
  if (share == 0) {
    for (int i = 1; i < min(SHARES, cut.w); ++i) {
      const float4 x = sums[i * COLS + col];
      acc.x += x.x;
      acc.y += x.y;
      acc.z += x.z;
      acc.w += x.w;
    }
    const int rho = cut.x + row, tok = div_small(rho, group);
    const float den = l + sink_term(p.sink, m, c_all), inv = den == 0.f ? 0.f : 1.0f / den;
    __nv_bfloat162 lo = __floats2bfloat162_rn(acc.x * inv, acc.y * inv), hi = __floats2bfloat162_rn(acc.z * inv, acc.w * inv);
    uint2 pk;
    pk.x = *reinterpret_cast<uint32_t*>(&lo);
    pk.y = *reinterpret_cast<uint32_t*>(&hi);
    *reinterpret_cast<uint2*>(out + ((size_t)tok * p.nq + (rho - tok * group) + (size_t)cut.z * group) * D + 4 * col) = pk;
  }
}

}  // namespace ms

using namespace ms;

#define MS_CAT2(a, b) a##b
#define MS_CAT(a, b) MS_CAT2(a, b)
#define MS_ATTN8_FN(name) MS_CAT(MS_CAT(MS_CAT(ms_attn_cache8_d, MS_HEAD_DIM), _), name)

MS_DEFINE_LAST_ERROR(MS_ATTN8_FN(last_error))
MS_DEFINE_PDL_SWITCH(MS_ATTN8_FN(set_pdl))

constexpr int SMEM_MOST = 227 * 1024 - 16 * 1024;  // (the table of tiles is static: 15 KB)

// Floats of partial results that a launch of `ctas` CTAs needs; the table of cut items (4 ints a CTA) lies behind them.
MS_EXPORT long long MS_ATTN8_FN(part_floats)(int ctas) { return 2LL * ctas * ROWS * PART; }
MS_EXPORT int MS_ATTN8_FN(max_units)() { return MAX_UNITS; }
MS_EXPORT int MS_ATTN8_FN(most_rows)() { return ROWS; }
MS_EXPORT int MS_ATTN8_FN(slice)() { return SLICE; }
MS_EXPORT int MS_ATTN8_FN(warps)(int tile_rows) { return warps_of(tile_rows / 8); }
MS_EXPORT int MS_ATTN8_FN(alone_most)(int each) { return alone_most(each); }
MS_EXPORT int MS_ATTN8_FN(switch_slices)() { return SWITCH; }

template <int NT>
static int launch_split(const Split8& p, int rows_tile, void* out, const void* q, const void* k_codes,
                        const void* k_exps, const void* v_codes, const void* v_exps, cudaStream_t stream) {
  static bool configured[64] = {};  // the attribute belongs to a device
  int dev = 0;
  MS_CHECK_CUDA(cudaGetDevice(&dev));
  MS_CHECK_ARG(dev >= 0 && dev < 64, "attention: device index %d is not supported", dev);
  if (!configured[dev]) {
    MS_CHECK_CUDA(cudaFuncSetAttribute(attn_cache8_split_kernel<NT>, cudaFuncAttributeMaxDynamicSharedMemorySize, SMEM_MOST));
    configured[dev] = true;
  }
  constexpr int ring = warps_of(NT) * stages_of(NT) * STAGE_BYTES;
  static_assert(ring + warps_of(NT) * 8 * NT * PART * 4 <= SMEM_MOST && 8 * NT * PART * 4 <= stages_of(NT) * STAGE_BYTES, "the rings and the pieces of shared items fit");
  MS_LAUNCH(attn_cache8_split_kernel<NT>, p.ctas, warps_of(NT) * 32, ring + warps_of(NT) * rows_tile * PART * 4, stream, (__nv_bfloat16*)out, (const __nv_bfloat16*)q,
            (const uint8_t*)k_codes, (const uint8_t*)k_exps, (const uint8_t*)v_codes, (const uint8_t*)v_exps, p, rows_tile);
  return 0;
}

// Rows [0, p->rows) of the geometry in p, in tiles of `tile_rows` (a multiple of 8) query rows, of which no request has more than `rows_most`.
MS_EXPORT int MS_ATTN8_FN(split)(const Split8* p, int tile_rows, int rows_most, void* out, const void* q, const void* k_codes, const void* k_exps, const void* v_codes,
                                 const void* v_exps, cudaStream_t stream) {
  if (p->rows == 0) return 0;
  MS_CHECK_ARG(p->nq > 0 && p->nkv > 0 && p->nq % p->nkv == 0, "attention: %d query heads are not a multiple of %d kv heads", p->nq, p->nkv);
  MS_CHECK_ARG(p->page_size >= 8 && (p->page_size & (p->page_size - 1)) == 0, "attention: page_size=%d must be a power of two from 8 on for an 8-bit cache", p->page_size);
  MS_CHECK_ARG(p->rows > 0 && p->tiles > 0 && (long long)p->rows * p->tiles <= MAX_UNITS, "attention: %d rows of %d tiles are too many for one launch", p->rows, p->tiles);
  MS_CHECK_ARG(p->ctas > 0 && p->part && p->cut && tile_rows > 0 && tile_rows <= ROWS && tile_rows % 8 == 0 && rows_most > 0, "attention: %d CTAs need scratch memory, tiles %d rows of %d",
               p->ctas, tile_rows, rows_most);
  MS_CHECK_ARG(p->behind || (long long)p->rows * p->tiles * p->nkv <= p->ctas, "attention: %d rows of %d tiles and %d kv heads are cut", p->rows, p->tiles, p->nkv);
  const long long pool_rows = (long long)p->num_pages * p->nkv * p->page_size;
  MS_CHECK_ARG(pool_rows > 0 && pool_rows < (1LL << 31), "attention: pools of %lld rows", pool_rows);
  MS_CHECK_ARG((uintptr_t)q % 8 == 0 && (uintptr_t)out % 8 == 0 && (uintptr_t)k_codes % 16 == 0 && (uintptr_t)v_codes % 16 == 0 && (uintptr_t)k_exps % 8 == 0 &&
                   (uintptr_t)v_exps % 8 == 0 && (uintptr_t)p->part % 16 == 0 && (uintptr_t)p->cut % 16 == 0,
               "attention: an 8-bit cache's tensors must be 16-byte aligned");
  const int rows_tile = rows_most < tile_rows ? rows_most : tile_rows;
  auto launch = tile_rows == 8 ? launch_split<1> : (tile_rows == 16 ? launch_split<2> : launch_split<MOST_NT>);
  if (int rc = launch(*p, rows_tile, out, q, k_codes, k_exps, v_codes, v_exps, stream)) return rc;
  if (p->behind) MS_LAUNCH(attn_cache8_merge_kernel, dim3(p->ctas, rows_tile), MERGE_THREADS, 0, stream, (__nv_bfloat16*)out, *p);
  return 0;
}
