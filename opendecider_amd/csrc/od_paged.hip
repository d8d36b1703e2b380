// A paged K/V cache, for gfx950: new tokens written into pages, sequences read back, attention over pages.
//
// Layout. A layer's K and V are two pools of n_pages pages; page p holds `page` (a power of two >= 16) token rows of every
// KV head, [n_pages, Hkv, page, D], int8 with one fp32 scale per row ([n_pages, Hkv, page]) or bf16. Position j of sequence
// b is row j % page of page table[b, j / page]. A (page, head) block is contiguous, so that an attention workgroup of one
// head reads whole runs of `page` rows. Batches are packed and ragged: sequence b's new tokens are the packed rows
// start[b] .. start[b + 1] - 1, at the positions ctx[b], ctx[b] + 1, ...
//
// Nothing on the device is trusted to stay in bounds: a table entry outside [0, n_pages), a position past the table's
// columns, a negative length and packed rows outside [0, N) are found by the kernels and skipped (no such key is seen, no
// such row written). The host needs no copy of start, ctx or table.
#include <type_traits>

#include "od_common.h"

namespace {

constexpr int kThreads = 256;
constexpr float kLog2e = 1.44269504088896341f;
constexpr float kLn2 = 0.693147180559945309f;

// The pages and the sequences in them, as every kernel here takes them.
struct Paged {
  void* k;
  void* v;
  float* ks;  // null: bf16 pages
  float* vs;
  const int32_t* table;
  const int32_t* start;  // [B + 1]; not used by page_read
  const int32_t* ctx;    // [B]
  int64_t ld_table, n_pages;
  int cols, shift, B, N, Hkv;  // page = 1 << shift
};

// First row (over all heads of the pool) of the page that holds position `pos` of sequence b for head h, plus the row in
// the page: the index of a token row of D values and of its scale. -1: no such page.
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

// ------------------------------------------------------------------------------------------------------- append
// Rows of D values, 16 per lane (two 16-byte loads), G = D / 16 lanes per row. A wave takes 64 / G consecutive items of
// the packed (token, K heads then V heads) order, so it reads whole runs of the projection's row. int8 pages take the
// bytes and the scale of the row quantizer (od_q8_words: absmax / 127, round half to even), bf16 pages the values.
// Bound by launch latency for a decode step and by memory for chunks: 2 bytes read and 1 written per value.
struct AppendArgs {
  Paged p;
  const uint16_t* k;
  const uint16_t* v;
  int64_t skt, skh, svt, svh;
};

template <int D, bool Q8>
__global__ __launch_bounds__(kThreads) void page_append_kernel(AppendArgs a) {
  constexpr int G = D / 16, RPW = 64 / G;
  const Paged& p = a.p;
  const int lane = threadIdx.x & 63, j = lane % G;
  const int64_t wave = (int64_t)blockIdx.x * (kThreads / 64) + (threadIdx.x >> 6);
  const int heads = 2 * p.Hkv;
  const int64_t items = (int64_t)p.N * heads, first = wave * RPW;
  if (first >= items) return;  // wave-uniform
  const int t0 = __builtin_amdgcn_readfirstlane((int)(first / heads));
  int b = seq_search(p.start, p.B, t0);
  const int64_t item = first + lane / G;
  const int t = (int)(item / heads), h = (int)(item % heads);
  // this lane's row may belong to a later token than the wave's first one
  while (b < p.B && p.start[b + 1] <= t) ++b;
  if (item >= items || b >= p.B) return;  // whole G-lane groups leave together
  const int s0 = p.start[b];
  if (t < s0) return;
  const bool isv = h >= p.Hkv;
  const int kh = isv ? h - p.Hkv : h;
  const int64_t row = row_of(p, b, kh, (int64_t)max(p.ctx[b], 0) + (t - s0));
  if (row < 0) return;
  const uint16_t* x = (isv ? a.v + t * a.svt + kh * a.svh : a.k + t * a.skt + kh * a.skh) + 16 * j;
  const uint4 lo = *reinterpret_cast<const uint4*>(x), hi = *reinterpret_cast<const uint4*>(x + 8);
  if constexpr (!Q8) {
    uint4* dst = reinterpret_cast<uint4*>(static_cast<uint16_t*>(isv ? p.v : p.k) + row * D + 16 * j);
    dst[0] = lo;
    dst[1] = hi;
  } else {
    const uint32_t w[8] = {lo.x, lo.y, lo.z, lo.w, hi.x, hi.y, hi.z, hi.w};
    float y[16];
    uint32_t am = 0;
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      am = od_absmax_bf16x2(am, w[i]);
      y[2 * i] = __uint_as_float(w[i] << 16);
      y[2 * i + 1] = __uint_as_float(w[i] & 0xffff0000u);
    }
    uint32_t bits = __float_as_uint(od_absmax_bf16x2_value(am));
#pragma unroll
    for (int o = G / 2; o > 0; o >>= 1) bits = max(bits, (uint32_t)__shfl_xor((int)bits, o, 64));
    const float scale = od_q8_scale(__uint_as_float(bits)), inv = 1.0f / scale;
    uint32_t q[4];
    od_q8_words<16>(y, scale, inv, q);
    *reinterpret_cast<uint4*>(static_cast<int8_t*>(isv ? p.v : p.k) + row * D + 16 * j) =
        make_uint4(q[0], q[1], q[2], q[3]);
    if (j == 0) (isv ? p.vs : p.ks)[row] = scale;
  }
}

// --------------------------------------------------------------------------------------------------------- read
// Dense (B, Hkv, T, D) K and V of every sequence's first ctx[b] tokens, zeros behind them: the values q * s (one fp32
// product, rounded once to bf16 where that is asked), bf16 rows as they are, or the int8 rows with their scales. A group
// of G = D / 16 lanes takes one token row of K and the same of V (16 values per lane). Bound by memory.
struct ReadArgs {
  Paged p;
  void* k;
  void* v;
  float* ks;  // int8 output only
  float* vs;
  int64_t rows;  // B * Hkv * T
  int T;
};
enum { kReadBf16 = 0, kReadF32 = 1, kReadI8 = 2 };

template <bool Q8, int OUT>
__device__ __forceinline__ void read_side(const void* pool, const float* scales, int64_t row, int D, int j, void* out,
                                          float* out_s, int64_t at) {
  float y[16];
  if constexpr (Q8) {
    uint4 q = make_uint4(0, 0, 0, 0);
    float s = 0.0f;
    if (row >= 0) {
      q = *reinterpret_cast<const uint4*>(static_cast<const int8_t*>(pool) + row * D + 16 * j);
      s = scales[row];
    }
    if constexpr (OUT == kReadI8) {
      *reinterpret_cast<uint4*>(static_cast<int8_t*>(out) + at * D + 16 * j) = q;
      if (j == 0) out_s[at] = s;
      return;
    }
    const uint32_t w[4] = {q.x, q.y, q.z, q.w};
#pragma unroll
    for (int i = 0; i < 16; ++i) y[i] = (float)(int8_t)(w[i / 4] >> (8 * (i % 4))) * s;
  } else {
    uint4 lo = make_uint4(0, 0, 0, 0), hi = lo;
    if (row >= 0) {
      const uint16_t* x = static_cast<const uint16_t*>(pool) + row * D + 16 * j;
      lo = *reinterpret_cast<const uint4*>(x);
      hi = *reinterpret_cast<const uint4*>(x + 8);
    }
    if constexpr (OUT == kReadBf16) {
      uint4* dst = reinterpret_cast<uint4*>(static_cast<uint16_t*>(out) + at * D + 16 * j);
      dst[0] = lo;
      dst[1] = hi;
      return;
    }
    const uint32_t w[8] = {lo.x, lo.y, lo.z, lo.w, hi.x, hi.y, hi.z, hi.w};
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      y[2 * i] = __uint_as_float(w[i] << 16);
      y[2 * i + 1] = __uint_as_float(w[i] & 0xffff0000u);
    }
  }
  if constexpr (OUT == kReadF32) {
    float4* dst = reinterpret_cast<float4*>(static_cast<float*>(out) + at * D + 16 * j);
#pragma unroll
    for (int i = 0; i < 4; ++i) dst[i] = make_float4(y[4 * i], y[4 * i + 1], y[4 * i + 2], y[4 * i + 3]);
  } else {
    uint32_t w[8];
#pragma unroll
    for (int i = 0; i < 8; ++i) w[i] = od_pack_bf16x2(y[2 * i], y[2 * i + 1]);
    uint4* dst = reinterpret_cast<uint4*>(static_cast<uint16_t*>(out) + at * D + 16 * j);
    dst[0] = make_uint4(w[0], w[1], w[2], w[3]);
    dst[1] = make_uint4(w[4], w[5], w[6], w[7]);
  }
}

template <int D, bool Q8, int OUT>
__global__ __launch_bounds__(kThreads) void page_read_kernel(ReadArgs a) {
  constexpr int G = D / 16;
  const int64_t at = (int64_t)blockIdx.x * (kThreads / G) + threadIdx.x / G;
  if (at >= a.rows) return;
  const int j = threadIdx.x % G;
  const int64_t bh = at / a.T;
  const int pos = (int)(at % a.T), b = (int)(bh / a.p.Hkv), h = (int)(bh % a.p.Hkv);
  const int64_t row = pos < a.p.ctx[b] ? row_of(a.p, b, h, pos) : -1;
  read_side<Q8, OUT>(a.p.k, a.p.ks, row, D, j, a.k, a.ks, at);
  read_side<Q8, OUT>(a.p.v, a.p.vs, row, D, j, a.v, a.vs, at);
}

// ---------------------------------------------------------------------------------------------------- attention
// New token i of sequence b (packed row n = start[b] + i) sees the cached positions 0 .. ctx[b] - 1 and the new tokens
// row_begin[n] .. i of its own sequence (row_begin null: from 0), bf16 as they come: o = sum_j p_j v_j / sum_j p_j with
// p_j = exp(scale q.k_j - max), lse = max + log sum p; a token that sees nothing has o = 0 and lse = -inf.
struct AttnArgs {
  Paged p;
  const uint16_t* q;
  const uint16_t* k;  // the new tokens' K and V; null: they see the cache only
  const uint16_t* v;
  const int32_t* row_begin;
  uint16_t* out;
  float* lse;
  int64_t sqt, sqh, skt, skh, svt, svh, sot, soh;
  int Hq, rep;
  float scale_log2;
};

// One wave per (packed row, query head), 64 keys at a time: a lane takes a key's whole score, then D / 64 columns of the
// output over the 64 probabilities.
template <int D, bool Q8>
__global__ __launch_bounds__(64) void paged_attn_rows_kernel(AttnArgs a) {
  constexpr int C = D / 64;
  __shared__ float sq[D];
  const Paged& p = a.p;
  const int n = blockIdx.x, head = blockIdx.y, g = head / a.rep, lane = threadIdx.x;
  int b = seq_search(p.start, p.B, n);
  if (p.start[b] > n || p.start[b + 1] <= n) return;
  const int i = n - p.start[b], s0 = p.start[b];
  const int64_t ctx = min((int64_t)max(p.ctx[b], 0), (int64_t)p.cols << p.shift);
  const int begin = a.row_begin ? max(a.row_begin[n], 0) : 0;
  for (int d = lane; d < D; d += 64) sq[d] = od_bf16_to_f32(a.q[n * a.sqt + head * a.sqh + d]);
  __syncthreads();
  float m = -INFINITY, l = 0.0f, o[C];
#pragma unroll
  for (int c = 0; c < C; ++c) o[c] = 0.0f;
  const int64_t total = ctx + (a.k ? i + 1 : 0);
  for (int64_t j0 = 0; j0 < total; j0 += 64) {
    const int64_t j = j0 + lane;
    const int64_t row = j < ctx ? row_of(p, b, g, j) : -1;
    const bool cached = row >= 0, own = j >= ctx && j < total && j - ctx >= begin;
    float y = -INFINITY;
    if (cached || own) {
      float s = 0.0f;
      if (cached && Q8) {
        const int8_t* kr = static_cast<const int8_t*>(p.k) + row * D;
        for (int d = 0; d < D; ++d) s = fmaf(sq[d], (float)kr[d], s);
        s *= p.ks[row];
      } else {
        const uint16_t* kr = cached ? static_cast<const uint16_t*>(p.k) + row * D : a.k + (s0 + j - ctx) * a.skt + g * a.skh;
        for (int d = 0; d < D; ++d) s = fmaf(sq[d], od_bf16_to_f32(kr[d]), s);
      }
      y = s * a.scale_log2;
    }
    const float mx = od_wave_max(y), m2 = fmaxf(m, mx), ms = m2 == -INFINITY ? 0.0f : m2;
    const float alpha = __builtin_amdgcn_exp2f(m - ms), pr = __builtin_amdgcn_exp2f(y - ms);
    l = l * alpha + od_wave_sum_dpp(pr);
    m = m2;
#pragma unroll
    for (int c = 0; c < C; ++c) o[c] *= alpha;
    for (int t = 0; t < 64; ++t) {
      const int64_t r = __shfl((long long)row, t, 64), jt = j0 + t;
      const float pt = __shfl(pr, t, 64);
      const int ok = __shfl((int)(cached || own), t, 64);
      if (!ok) continue;
#pragma unroll
      for (int c = 0; c < C; ++c) {
        const int d = c * 64 + lane;
        float vv;
        if (r >= 0 && Q8) vv = (float)static_cast<const int8_t*>(p.v)[r * D + d] * p.vs[r];
        else vv = od_bf16_to_f32(r >= 0 ? static_cast<const uint16_t*>(p.v)[r * D + d] : a.v[(s0 + jt - ctx) * a.svt + g * a.svh + d]);
        o[c] = fmaf(pt, vv, o[c]);
      }
    }
  }
  const float inv = l == 0.0f ? 0.0f : 1.0f / l;
#pragma unroll
  for (int c = 0; c < C; ++c) a.out[n * a.sot + head * a.soh + c * 64 + lane] = od_f32_to_bf16(l == 0.0f ? 0.0f : o[c] * inv);
  if (a.lse && lane == 0) a.lse[(int64_t)n * a.Hq + head] = (m + __log2f(l)) * kLn2;
}

bool aligned4(const void* p) { return (((uintptr_t)p) & 3u) == 0; }

// Checks of the pages that every entry point makes; fills P.
int paged_args(Paged& P, const void* k_pages, const float* k_scale, const void* v_pages, const float* v_scale, int64_t n_pages,
               int64_t page, const int32_t* table, int64_t ld_table, int64_t cols, const int32_t* start, const int32_t* ctx,
               int64_t B, int64_t N, int64_t Hkv, int64_t D) {
  if (B < 0 || N < 0 || Hkv < 1 || n_pages < 0 || cols < 0 || ld_table < cols) return OD_ERR_SHAPE;
  if (D != 64 && D != 128 && D != 256) return OD_ERR_UNSUPPORTED;
  if (page < 16 || page > (1 << 20) || (page & (page - 1))) return OD_ERR_UNSUPPORTED;
  if (B > (1 << 24) || N > 0x3fffffff || cols > 0x3fffffff || Hkv > 65535 || n_pages > 0x7fffffff) return OD_ERR_SHAPE;
  if (cols * page > 0x7fffff00ll) return OD_ERR_SHAPE;
  if (!k_scale != !v_scale) return OD_ERR_NULL;
  if (n_pages > 0 && (!k_pages || !v_pages)) return OD_ERR_NULL;
  if (!od_aligned16(k_pages) || !od_aligned16(v_pages) || !aligned4(k_scale) || !aligned4(v_scale)) return OD_ERR_ALIGN;
  P = Paged{const_cast<void*>(k_pages), const_cast<void*>(v_pages), const_cast<float*>(k_scale), const_cast<float*>(v_scale),
            table, start, ctx, ld_table, n_pages, (int)cols, __builtin_ctzll(page), (int)B, (int)N, (int)Hkv};
  return OD_OK;
}

template <class F>
void by_head_dim(int64_t D, F&& f) {
  if (D == 64) f(std::integral_constant<int, 64>{});
  else if (D == 128) f(std::integral_constant<int, 128>{});
  else f(std::integral_constant<int, 256>{});
}

}  // namespace

extern "C" int od_page_append(const uint16_t* k, int64_t skt, int64_t skh, const uint16_t* v, int64_t svt, int64_t svh,
                              void* k_pages, float* k_scale, void* v_pages, float* v_scale, int64_t n_pages, int64_t page,
                              const int32_t* table, int64_t ld_table, int64_t cols, const int32_t* start,
                              const int32_t* ctx_len, int64_t B, int64_t N, int64_t Hkv, int64_t D, od_stream_t stream) {
  AppendArgs a;
  if (const int rc = paged_args(a.p, k_pages, k_scale, v_pages, v_scale, n_pages, page, table, ld_table, cols, start, ctx_len,
                                B, N, Hkv, D))
    return rc;
  if (B == 0 || N == 0 || cols == 0 || n_pages == 0) return OD_OK;
  if (!k || !v || !table || !start || !ctx_len) return OD_ERR_NULL;
  const int64_t strides[] = {skt, skh, svt, svh};
  for (int64_t s : strides)
    if (s < 0 || s % 8) return OD_ERR_ALIGN;
  if (!od_aligned16(k) || !od_aligned16(v)) return OD_ERR_ALIGN;
  a.k = k;
  a.v = v;
  a.skt = skt;
  a.skh = skh;
  a.svt = svt;
  a.svh = svh;
  const int64_t per_block = (int64_t)(kThreads / 64) * (64 / (D / 16)), blocks = (N * 2 * Hkv + per_block - 1) / per_block;
  if (blocks > 0x7fffffff) return OD_ERR_SHAPE;
  by_head_dim(D, [&](auto DC) {
    constexpr int DD = decltype(DC)::value;
    const dim3 grid((unsigned)blocks);
    if (k_scale) page_append_kernel<DD, true><<<grid, dim3(kThreads), 0, (hipStream_t)stream>>>(a);
    else page_append_kernel<DD, false><<<grid, dim3(kThreads), 0, (hipStream_t)stream>>>(a);
  });
  return od_launch_status();
}

extern "C" int od_page_read(const void* k_pages, const float* k_scale, const void* v_pages, const float* v_scale,
                            int64_t n_pages, int64_t page, const int32_t* table, int64_t ld_table, int64_t cols,
                            const int32_t* length, int64_t B, int64_t T, int64_t Hkv, int64_t D, int form, void* k_out,
                            float* ks_out, void* v_out, float* vs_out, od_stream_t stream) {
  ReadArgs a;
  if (const int rc = paged_args(a.p, k_pages, k_scale, v_pages, v_scale, n_pages, page, table, ld_table, cols, nullptr, length,
                                B, 0, Hkv, D))
    return rc;
  if (T < 0 || T > 0x3fffffff) return OD_ERR_SHAPE;
  if (form != OD_READ_BF16 && form != OD_READ_FP32 && form != OD_READ_INT8) return OD_ERR_UNSUPPORTED;
  if (form == OD_READ_INT8 && !k_scale) return OD_ERR_UNSUPPORTED;
  if (B == 0 || T == 0) return OD_OK;
  if (!length || !k_out || !v_out || (cols > 0 && !table)) return OD_ERR_NULL;
  if (form == OD_READ_INT8 && (!ks_out || !vs_out)) return OD_ERR_NULL;
  if (!od_aligned16(k_out) || !od_aligned16(v_out) || !aligned4(ks_out) || !aligned4(vs_out)) return OD_ERR_ALIGN;
  a.k = k_out;
  a.v = v_out;
  a.ks = ks_out;
  a.vs = vs_out;
  a.T = (int)T;
  if (B * Hkv > (1ll << 40) / T) return OD_ERR_SHAPE;
  a.rows = B * Hkv * T;
  const int64_t per_block = kThreads / (D / 16), blocks = (a.rows + per_block - 1) / per_block;
  if (blocks > 0x7fffffff) return OD_ERR_SHAPE;
  by_head_dim(D, [&](auto DC) {
    constexpr int DD = decltype(DC)::value;
    const dim3 grid((unsigned)blocks), block(kThreads);
    hipStream_t st = (hipStream_t)stream;
    if (k_scale) {
      if (form == OD_READ_BF16) page_read_kernel<DD, true, kReadBf16><<<grid, block, 0, st>>>(a);
      else if (form == OD_READ_FP32) page_read_kernel<DD, true, kReadF32><<<grid, block, 0, st>>>(a);
      else page_read_kernel<DD, true, kReadI8><<<grid, block, 0, st>>>(a);
    } else {
      if (form == OD_READ_BF16) page_read_kernel<DD, false, kReadBf16><<<grid, block, 0, st>>>(a);
      else page_read_kernel<DD, false, kReadF32><<<grid, block, 0, st>>>(a);
    }
  });
  return od_launch_status();
}

extern "C" int od_paged_attn_ws(int64_t B, int64_t N, int64_t Hq, int64_t Hkv, int64_t D, int64_t max_new, int64_t max_ctx,
                                int64_t* ws_floats) {
  if (!ws_floats) return OD_ERR_NULL;
  if (B < 0 || N < 0 || Hq < 1 || Hkv < 1 || max_new < 0 || max_ctx < 0) return OD_ERR_SHAPE;
  if (Hq % Hkv || (D != 64 && D != 128 && D != 256)) return OD_ERR_UNSUPPORTED;
  *ws_floats = 0;
  return OD_OK;
}

extern "C" int od_paged_attn(const uint16_t* q, int64_t sqt, int64_t sqh, const uint16_t* k, int64_t skt, int64_t skh,
                             const uint16_t* v, int64_t svt, int64_t svh, const void* k_pages, const float* k_scale,
                             const void* v_pages, const float* v_scale, int64_t n_pages, int64_t page, const int32_t* table,
                             int64_t ld_table, int64_t cols, const int32_t* start, const int32_t* ctx_len,
                             const int32_t* row_begin, uint16_t* out, int64_t sot, int64_t soh, float* lse, int64_t B,
                             int64_t N, int64_t Hq, int64_t Hkv, int64_t D, int64_t max_new, int64_t max_ctx, float scale,
                             float* ws, int64_t ws_floats, od_stream_t stream) {
  AttnArgs a;
  if (const int rc = paged_args(a.p, k_pages, k_scale, v_pages, v_scale, n_pages, page, table, ld_table, cols, start, ctx_len,
                                B, N, Hkv, D))
    return rc;
  if (Hq < 1 || Hq > 65535 || max_new < 0 || max_ctx < 0) return OD_ERR_SHAPE;
  if (Hq % Hkv || !(scale > 0.0f) || !(scale < INFINITY)) return OD_ERR_UNSUPPORTED;
  if (B == 0 || N == 0) return OD_OK;
  if (!q || !out || !start || !ctx_len || !k != !v || (cols > 0 && !table)) return OD_ERR_NULL;
  const int64_t strides[] = {sqt, sqh, skt, skh, svt, svh, sot, soh};
  for (int64_t s : strides)
    if (s < 0 || s % 8) return OD_ERR_ALIGN;
  if (!od_aligned16(q) || !od_aligned16(k) || !od_aligned16(v) || !od_aligned16(out) || !aligned4(lse)) return OD_ERR_ALIGN;
  a.q = q;
  a.k = k;
  a.v = v;
  a.row_begin = row_begin;
  a.out = out;
  a.lse = lse;
  a.sqt = sqt;
  a.sqh = sqh;
  a.skt = skt;
  a.skh = skh;
  a.svt = svt;
  a.svh = svh;
  a.sot = sot;
  a.soh = soh;
  a.Hq = (int)Hq;
  a.rep = (int)(Hq / Hkv);
  a.scale_log2 = scale * kLog2e;
  by_head_dim(D, [&](auto DC) {
    constexpr int DD = decltype(DC)::value;
    const dim3 grid((unsigned)N, (unsigned)Hq);
    if (k_scale) paged_attn_rows_kernel<DD, true><<<grid, dim3(64), 0, (hipStream_t)stream>>>(a);
    else paged_attn_rows_kernel<DD, false><<<grid, dim3(64), 0, (hipStream_t)stream>>>(a);
  });
  return od_launch_status();
}
