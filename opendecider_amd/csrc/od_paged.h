// The pages of a K/V cache as the kernels over them see them: where a token's row lies, how its values are held, the checks of
// the arguments that every entry point makes.
#pragma once

#include <type_traits>

#include "od_common.h"

namespace {

// What a page's rows are: bf16 values; int8 ones with an fp32 scale a row; 4-bit ones with a bf16 scale per 32 of them.
// (kImage: int8 or 4-bit rows converted to fp16 ahead, as the tile kernels of the attention read them.)
enum { kBf16 = 0, kInt8 = 1, kImage = 2, kInt4 = 3 };

// The pages and the sequences in them, as every kernel here takes them.
struct Paged {
  void* k;
  void* v;
  float* ks;  // int8 rows' scales
  float* vs;
  uint16_t* k4;  // 4-bit rows' scales, D / 32 a row
  uint16_t* v4;
  const int32_t* table;
  const int32_t* start;  // [B + 1]; not used by page_read
  const int32_t* ctx;    // [B]
  int64_t ld_table, n_pages;
  int cols, shift, B, N, Hkv;  // page = 1 << shift
};

// First row (over all heads of the pool) of the page that holds position `pos` of sequence b for head h, plus the row
// in the page: the index of a token row of D values and of its scale. -1: no such page.
__device__ __forceinline__ int64_t row_of(const Paged& p, int b, int h, int64_t pos) {
  const int64_t col = pos >> p.shift;
  if (pos < 0 || col >= p.cols) return -1;
  const int pg = p.table[b * p.ld_table + col];
  if (pg < 0 || pg >= p.n_pages) return -1;
  return (((int64_t)pg * p.Hkv + h) << p.shift) + (pos & ((1 << p.shift) - 1));
}

// The last sequence that starts at or before packed row t, by all 64 lanes together (a 64-way search: one load per lane
// and level, one level up to 64 sequences, two up to 4096); 0 if there is none. t is wave-uniform. In bounds for any
// contents of start.
__device__ __forceinline__ int seq_search(const int32_t* start, int B, int t) {
  const int lane = threadIdx.x & 63;
  int lo = 0, n = B;
  while (n > 1) {
    const int step = (n + 63) >> 6, at = lane * step;
    const bool le = at < n && start[lo + at] <= t;
    const int cnt = __builtin_popcountll(__builtin_amdgcn_ballot_w64(le));
    if (cnt == 0) return 0;
    const int skip = (cnt - 1) * step;
    lo += skip;
    n = min(step, n - skip);
  }
  return lo;
}

// Row of the pools that packed row t writes for head h, its sequence found from b on (a sequence that starts at or before t);
// -1: a row of no sequence (a range outside the packed rows is none), or no page.
__device__ __forceinline__ int64_t row_to_write(const Paged& p, int b, int t, int h) {
  while (b < p.B && p.start[b + 1] <= t) ++b;
  if (b >= p.B) return -1;
  const int s0 = p.start[b];
  if (t < s0 || s0 < 0 || p.start[b + 1] > p.N) return -1;
  return row_of(p, b, h, (int64_t)max(p.ctx[b], 0) + (t - s0));
}

// -------------------------------------------------------------------------------------------------- rows of 4 bits
// Blocks of 32 values: (u - 8) d, u in 0 .. 15, d in bf16. m the value of the largest magnitude of the block (the first of
// several), d = m / -8 (exact), u = floor(x / d + 8.5) in 0 .. 15: m itself gets -8, the widest code. A block below 2^-100 has
// d = 0 and u = 8; one that holds an infinity or NaN has d = NaN. Eight values make a word, value 2 i at bit 4 i, 2 i + 1 at
// bit 16 + 4 i: masks then give pairs of neighbours in the halves of a register.
//
// x / d of bf16 numbers is n + 1/2 for an integer n, or at least 1 / 1020 away from it (their significands have 8 bits), so
// x (1 / d) + 8.5 + 2^-12, off by less than 2^-19, has the floor of the quotient plus 8.5.
constexpr uint32_t kQ4Least = 0x0d80u;  // 2^-100 in bf16

// The largest magnitude among 8 bf16 values (w: 4 words, `first` the place of the first in its block), as a number that also
// holds the place and the sign: the maximum of two is the one of larger magnitude, or of lower place.
__device__ __forceinline__ uint32_t q4_lead(const uint32_t (&w)[4], int first) {
  uint32_t m = 0;
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const uint32_t at = (uint32_t)(31 - first - 2 * i) << 1;
    m = max(m, (w[i] << 16 & 0x7fff0000u) | at | (w[i] >> 15 & 1u));
    m = max(m, (w[i] & 0x7fff0000u) | (at - 2) | (w[i] >> 31));
  }
  return m;
}
// The block's scale as bf16 bits, and 1 / d for its codes (0: a block of zeros, or of none).
__device__ __forceinline__ uint32_t q4_scale(uint32_t lead, float& inv) {
  const uint32_t size = lead >> 16;
  inv = 0.0f;
  if (size >= 0x7f80u) return 0x7fc0u;
  if (size < kQ4Least) return 0u;
  const uint32_t d = (size - 0x180u) | ((lead & 1u) ^ 1u) << 15;
  inv = __builtin_amdgcn_rcpf(__uint_as_float(d << 16));
  return d;
}
__device__ __forceinline__ uint32_t q4_word(const uint32_t (&w)[4], float inv) {
  uint32_t q = 0;
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const float lo = __builtin_fmaf(__uint_as_float(w[i] << 16), inv, 8.5f + 0x1p-12f);
    const float hi = __builtin_fmaf(__uint_as_float(w[i] & 0xffff0000u), inv, 8.5f + 0x1p-12f);
    // (the median gives 0 for NaN)
    q |= (uint32_t)__builtin_amdgcn_fmed3f(lo, 0.0f, 15.0f) << (4 * i);
    q |= (uint32_t)__builtin_amdgcn_fmed3f(hi, 0.0f, 15.0f) << (16 + 4 * i);
  }
  return q;
}
// Value i of a word's (0 as +0).
__device__ __forceinline__ float q4_value(uint32_t w, int i, float d) {
  return (float)((int)(w >> (4 * (i >> 1) + 16 * (i & 1)) & 15u) - 8) * d + 0.0f;
}

// -------------------------------------------------------------------------------------------------- host
// A launch has fewer than 2^32 threads: workgroups of 256.
constexpr int64_t kMaxGroups = (1 << 24) - 1;

bool aligned4(const void* p) { return (((uintptr_t)p) & 3u) == 0; }

// Checks of the pages that every entry point makes; fills P. format: OD_PAGE_*.
int paged_args(Paged& P, int format, const void* k_pages, const void* k_scale, const void* v_pages, const void* v_scale,
               int64_t n_pages, int64_t page, const int32_t* table, int64_t ld_table, int64_t cols,
               const int32_t* start, const int32_t* ctx, int64_t B, int64_t N, int64_t Hkv, int64_t D) {
  if (B < 0 || N < 0 || Hkv < 1 || n_pages < 0 || cols < 0 || ld_table < cols) return OD_ERR_SHAPE;
  if (D != 64 && D != 128 && D != 256) return OD_ERR_UNSUPPORTED;
  if (page < 16 || page > (1 << 20) || (page & (page - 1))) return OD_ERR_UNSUPPORTED;
  if (format != OD_PAGE_BF16 && format != OD_PAGE_INT8 && format != OD_PAGE_INT4) return OD_ERR_UNSUPPORTED;
  if (B > (1 << 24) || N > 0x3fffffff || cols > 0x3fffffff || Hkv > 65535 || n_pages > 0x7fffffff) return OD_ERR_SHAPE;
  if (cols * page > 0x7fffff00ll) return OD_ERR_SHAPE;
  if (!k_scale != !v_scale) return OD_ERR_NULL;
  if (n_pages > 0 && (!k_pages || !v_pages || (format != OD_PAGE_BF16 && !k_scale))) return OD_ERR_NULL;
  if (!od_aligned16(k_pages) || !od_aligned16(v_pages) || !aligned4(k_scale) || !aligned4(v_scale)) return OD_ERR_ALIGN;
  if (format == OD_PAGE_INT4 && (!od_aligned16(k_scale) || !od_aligned16(v_scale))) return OD_ERR_ALIGN;
  const bool q8 = format == OD_PAGE_INT8, q4 = format == OD_PAGE_INT4;
  P = Paged{const_cast<void*>(k_pages), const_cast<void*>(v_pages),
            q8 ? static_cast<float*>(const_cast<void*>(k_scale)) : nullptr,
            q8 ? static_cast<float*>(const_cast<void*>(v_scale)) : nullptr,
            q4 ? static_cast<uint16_t*>(const_cast<void*>(k_scale)) : nullptr,
            q4 ? static_cast<uint16_t*>(const_cast<void*>(v_scale)) : nullptr,
            table, start, ctx, ld_table, n_pages, (int)cols, __builtin_ctzll(page), (int)B, (int)N, (int)Hkv};
  return OD_OK;
}

template <class F>
void by_head_dim(int64_t D, F&& f) {
  if (D == 64) f(std::integral_constant<int, 64>{});
  else if (D == 128) f(std::integral_constant<int, 128>{});
  else f(std::integral_constant<int, 256>{});
}
template <class F>
void by_format(int format, F&& f) {
  if (format == OD_PAGE_BF16) f(std::integral_constant<int, kBf16>{});
  else if (format == OD_PAGE_INT8) f(std::integral_constant<int, kInt8>{});
  else f(std::integral_constant<int, kInt4>{});
}

}  // namespace
