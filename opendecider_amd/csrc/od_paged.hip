// A paged K/V cache, for gfx950: new tokens written into pages, sequences read back, attention over pages.
//
// Layout. A layer's K and V are two pools of n_pages pages; page p holds `page` (a power of two >= 16) token rows of
// every KV head, [n_pages, Hkv, page, D], int8 with one fp32 scale per row ([n_pages, Hkv, page]), bf16, or 4 bits a value with a
// bf16 scale per 32 ([n_pages, Hkv, page, D / 2] bytes and [n_pages, Hkv, page, D / 32]). Position j of sequence b is row
// j % page of page table[b, j / page]. A (page, head) block is contiguous, so that an attention
// workgroup of one head reads whole runs of `page` rows. Batches are packed and ragged: sequence b's new tokens are the
// packed rows start[b] .. start[b + 1] - 1, at the positions ctx[b], ctx[b] + 1, ...
//
// Nothing on the device is trusted to stay in bounds: a table entry outside [0, n_pages), a position past the table's
// columns, a negative length and packed rows outside [0, N) are found by the kernels and skipped (no such key is seen,
// no such row written). The host needs no copy of start, ctx or table.
#include "od_paged.h"

namespace {

typedef uint32_t v4u __attribute__((ext_vector_type(4)));

constexpr int kThreads = 256;
constexpr float kLog2e = 1.44269504088896341f;
constexpr float kLn2 = 0.693147180559945309f;

// ------------------------------------------------------------------------------------------------------- append
// Rows of D values, 16 per lane (two 16-byte loads), G = D / 16 lanes per row. A wave takes 64 / G consecutive items of
// the packed (token, K heads then V heads) order, so it reads whole runs of the projection's row. int8 pages take the
// bytes and the scale of the row quantizer (od_q8_words: absmax / 127, round half to even), bf16 pages the values.
// Bound by launch latency for a decode step (a token for each of 64 sequences 4.7 us) and by vector work and memory for
// chunks, 2 bytes read and 1 written per value (64 x 900 tokens of 8 heads of 128 55 us, 4.4 TB/s; bf16 pages 58, 5.6).
struct AppendArgs {
  Paged p;
  const uint16_t* k;
  const uint16_t* v;
  int64_t skt, skh, svt, svh;
};

template <int D, int P>
__global__ __launch_bounds__(kThreads) void page_append_kernel(AppendArgs a) {
  constexpr int G = D / 16, RPW = 64 / G;
  const Paged& p = a.p;
  const int lane = threadIdx.x & 63, j = lane % G;
  const int64_t wave = (int64_t)blockIdx.x * (kThreads / 64) + (threadIdx.x >> 6);
  const int heads = 2 * p.Hkv;
  const int64_t items = (int64_t)p.N * heads, first = wave * RPW, item = first + lane / G;
  if (first >= items) return;  // wave-uniform
  const int t0 = __builtin_amdgcn_readfirstlane((int)(first >> 31 ? first / heads : (uint32_t)first / (uint32_t)heads));
  const int b = seq_search(p.start, p.B, t0);
  if (item >= items) return;  // whole G-lane groups leave together
  const uint32_t from = (uint32_t)(item - (int64_t)t0 * heads);
  const int t = t0 + (int)(from / (uint32_t)heads), h = (int)(from % (uint32_t)heads);
  const bool isv = h >= p.Hkv;
  const int kh = isv ? h - p.Hkv : h;
  const int64_t row = row_to_write(p, b, t, kh);  // this lane's row may belong to a later token than the wave's first one
  if (row < 0) return;
  const uint16_t* x = (isv ? a.v + t * a.svt + kh * a.svh : a.k + t * a.skt + kh * a.skh) + 16 * j;
  const uint4 lo = *reinterpret_cast<const uint4*>(x), hi = *reinterpret_cast<const uint4*>(x + 8);
  if constexpr (P == kBf16) {
    uint4* dst = reinterpret_cast<uint4*>(static_cast<uint16_t*>(isv ? p.v : p.k) + row * D + 16 * j);
    dst[0] = lo;
    dst[1] = hi;
  } else if constexpr (P == kInt4) {
    const uint32_t w0[4] = {lo.x, lo.y, lo.z, lo.w}, w1[4] = {hi.x, hi.y, hi.z, hi.w};
    uint32_t lead = max(q4_lead(w0, 16 * (j & 1)), q4_lead(w1, 16 * (j & 1) + 8));
    lead = max(lead, (uint32_t)__shfl_xor((int)lead, 1, 64));  // two lanes a block
    float inv;
    const uint32_t d = q4_scale(lead, inv);
    *reinterpret_cast<uint2*>(static_cast<char*>(isv ? p.v : p.k) + row * (D / 2) + 8 * j) =
        make_uint2(q4_word(w0, inv), q4_word(w1, inv));
    if ((j & 1) == 0) (isv ? p.v4 : p.k4)[row * (D / 32) + j / 2] = (uint16_t)d;
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

// ---------------------------------------------------------------------------------------------------------- read
// Dense (B, Hkv, T, D) K and V of every sequence's first ctx[b] tokens, zeros behind them: the values q * s (one fp32
// product, rounded once to bf16 where that is asked), bf16 rows as they are, or the int8 rows with their scales. Bound
// by memory: 64 sequences of 8192 tokens, 8 heads of 128, 1.1 GB read and 2.1 GB written in 505 us, 5.7 TB/s. A lane
// takes the V values of a row of K, and of V, that make 16 bytes there, so that a wave's stores are whole lines (16
// values and two stores of bf16 a lane took 652 us), past the caches (one row a lane 547 without that, 4 rows a lane
// 564).
struct ReadArgs {
  Paged p;
  void* k;
  void* v;
  float* ks;  // int8 output only
  float* vs;
  int T, tiles;  // tiles: workgroups per (sequence, head)
};
enum { kReadBf16 = 0, kReadF32 = 1, kReadI8 = 2 };
constexpr int read_values(int out) { return out == kReadI8 ? 16 : out == kReadBf16 ? 8 : 4; }

template <int BYTES>
struct Chunk {
  uint32_t w[BYTES / 4];
};
template <int BYTES>
__device__ __forceinline__ Chunk<BYTES> read_chunk(const void* p) {
  Chunk<BYTES> c;
  if constexpr (BYTES == 4) {
    c.w[0] = *static_cast<const uint32_t*>(p);
  } else if constexpr (BYTES == 8) {
    const uint2 u = *static_cast<const uint2*>(p);
    c.w[0] = u.x, c.w[1] = u.y;
  } else {
    const uint4 u = *static_cast<const uint4*>(p);
    c.w[0] = u.x, c.w[1] = u.y, c.w[2] = u.z, c.w[3] = u.w;
  }
  return c;
}
template <int D, int P, int OUT>
__global__ __launch_bounds__(kThreads) void page_read_kernel(ReadArgs a) {
  constexpr bool Q8 = P == kInt8, Q4 = P == kInt4;
  constexpr int V = read_values(OUT), G = D / V, BYTES = Q4 ? 4 : V * (Q8 ? 1 : 2);
  const int bh = blockIdx.x / a.tiles, b = bh / a.p.Hkv, h = bh % a.p.Hkv;
  const int pos = (blockIdx.x % a.tiles) * (kThreads / G) + threadIdx.x / G, j = threadIdx.x % G;
  if (pos >= a.T) return;
  const int64_t row = pos < a.p.ctx[b] ? row_of(a.p, b, h, pos) : -1, at = (int64_t)bh * a.T + pos;
  Chunk<BYTES> x[2] = {};
  float s[2] = {};
  if (row >= 0) {
    // 4 bits: the word of 8 values that holds the lane's
    const int64_t from = Q4 ? row * (D / 2) + 4 * (j * V / 8) : (row * G + j) * BYTES;
    x[0] = read_chunk<BYTES>(static_cast<const char*>(a.p.k) + from);
    x[1] = read_chunk<BYTES>(static_cast<const char*>(a.p.v) + from);
    if constexpr (Q8) {
      s[0] = a.p.ks[row];
      s[1] = a.p.vs[row];
    } else if constexpr (Q4) {
      s[0] = od_bf16_to_f32(a.p.k4[row * (D / 32) + j * V / 32]);
      s[1] = od_bf16_to_f32(a.p.v4[row * (D / 32) + j * V / 32]);
    }
  }
#pragma unroll
  for (int side = 0; side < 2; ++side) {
    const Chunk<BYTES>& c = x[side];
    v4u o;
    if constexpr (OUT == kReadI8 || (OUT == kReadBf16 && P == kBf16)) {
      o = v4u{c.w[0], c.w[1], c.w[2], c.w[3]};
      if (OUT == kReadI8 && j == 0) (side ? a.vs : a.ks)[at] = s[side];
    } else {
      float y[V];
#pragma unroll
      for (int i = 0; i < V; ++i)
        y[i] = Q4 ? q4_value(V == 4 ? c.w[0] >> (8 * (j & 1)) : c.w[0], i, s[side])
             : Q8 ? (float)(int8_t)(c.w[i / 4] >> (8 * (i % 4))) * s[side]
                  : __uint_as_float(i % 2 ? c.w[i / 2] & 0xffff0000u : c.w[i / 2] << 16);
#pragma unroll
      for (int i = 0; i < 4; ++i)
        o[i] = OUT == kReadF32 ? __float_as_uint(y[i]) : od_pack_bf16x2(y[2 * i % V], y[(2 * i + 1) % V]);
    }
    __builtin_nontemporal_store(o, reinterpret_cast<v4u*>(static_cast<char*>(side ? a.v : a.k) + (at * G + j) * 16));
  }
}

// ---------------------------------------------------------------------------------------------------- attention
// New token i of sequence b (packed row n = start[b] + i) sees the cached positions 0 .. ctx[b] - 1 and the new tokens
// row_begin[n] .. i of its own sequence (row_begin null: from 0), bf16 as they come: o = sum_j p_j v_j / sum_j p_j with
// p_j = exp(scale q.k_j - max), lse = max + log sum p; a token that sees nothing has o = 0 and lse = -inf. An int8 row whose
// scale is not finite counts as NaN. A value that is infinite gives an infinite output where it is seen (NaN beside one of
// the other sign, and where a cached one's probability is 0 in fp32).
//
// A "slot" is a (new token, head of the KV group) pair: slot z of a sequence is token z / rep, head g rep + z % rep.
// Both kernels go over the keys once with a running maximum m and sum l in fp32 (log2 units). m moves only when a
// block's maximum lies more than 2^kSlack above it, so most blocks do not rescale the output: p <= 2^kSlack.
struct AttnArgs {
  Paged p;
  const uint16_t* q;
  const uint16_t* k;  // the new tokens' K and V; null: they see the cache only
  const uint16_t* v;
  const int32_t* row_begin;
  uint16_t* out;
  float* lse;
  float* part;  // splits: normalized outputs [nsplit, N, Hq, D], then their LSEs [nsplit, N, Hq] (log2 units)
  int64_t sqt, sqh, skt, skh, svt, svh, sot, soh;
  int Hq, rep;
  float scale_log2;
  int nsplit, chunk;  // split sp takes the key tiles sp chunk .. of a sequence, the last split all that are left
  int tiles;          // slot tiles of a sequence that the grid covers (the workgroups go on from there)
  int run;            // tiles that lie together on one XCD
  // the image of int8 pages, img_blocks blocks of every (sequence, KV head): 64 rows of K, then of V, fp16 in frames
  uint16_t* img;
  struct ImageBlock* img_heads;
  int* img_vexp;       // the frame of all of a (sequence, KV head)'s V
  int img_blocks;      // 0: no image
  bool rest;           // the kernel without the image, for the sequences that have none
};
// Of one block of the image: its keys that exist, the frame of its K, the largest of its V scales (as bits).
struct ImageBlock {
  uint64_t seen;
  int kexp;
  uint32_t v_bits;
};

typedef float v4f __attribute__((ext_vector_type(4)));
typedef float v16f __attribute__((ext_vector_type(16)));
typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));
typedef _Float16 f16x8 __attribute__((ext_vector_type(8)));
typedef _Float16 f16x2 __attribute__((ext_vector_type(2)));

constexpr float kSlack = 8.0f;

// One sequence as a workgroup sees it (all wave-uniform).
struct Seq {
  int s0, n;  // its new tokens are the packed rows s0 .. s0 + n - 1
  int ctx;    // its cached tokens, within the table
};
__device__ __forceinline__ Seq seq_of(const AttnArgs& a, int b) {
  Seq s;
  const int end = a.p.start[b + 1];
  s.s0 = a.p.start[b];
  s.n = s.s0 < 0 || end < s.s0 || end > a.p.N ? 0 : end - s.s0;  // 0: not a range of packed rows
  s.ctx = min(max(a.p.ctx[b], 0), a.p.cols << a.p.shift);
  return s;
}
// The splits of a sequence with `tiles` key tiles that hold any (split 0 holds the new tokens too).
__device__ __forceinline__ int splits_of(const AttnArgs& a, int tiles) {
  return max(1, min((tiles + a.chunk - 1) / a.chunk, a.nsplit));
}

__device__ __forceinline__ uint32_t fin_bf16x2(uint32_t w) {  // infinities and NaN -> 0
  uint32_t r = w;
  if ((w & 0x7f80u) == 0x7f80u) r &= 0xffff0000u;
  if ((w & 0x7f800000u) == 0x7f800000u) r &= 0xffffu;
  return r;
}
__device__ __forceinline__ v4u fin_bf16x8(v4u w) {
  return v4u{fin_bf16x2(w[0]), fin_bf16x2(w[1]), fin_bf16x2(w[2]), fin_bf16x2(w[3])};
}
// a bf16 that is infinite or NaN, as fp32; else 0
__device__ __forceinline__ float odd_bf16(uint32_t b) {
  return (b & 0x7f80u) == 0x7f80u ? __uint_as_float(b << 16) : 0.0f;
}
__device__ __forceinline__ bool any_inf_bf16x8(v4u w) {
  uint32_t m = 0;
#pragma unroll
  for (int i = 0; i < 4; ++i) m = od_absmax_bf16x2(m, w[i]);
  return (m & 0xffffu) >= 0x7f80u || (m >> 16) >= 0x7f80u;
}

// 4 int8 -> 4 exact bf16: |q| <= 128 has at most 8 significant bits, so the top half of the fp32 value is it
__device__ __forceinline__ void i8x4_to_bf16(uint32_t w, uint32_t& lo, uint32_t& hi) {
  const uint32_t f0 = __float_as_uint((float)(int8_t)(w & 0xffu)),
      f1 = __float_as_uint((float)(int8_t)((w >> 8) & 0xffu));
  const uint32_t f2 = __float_as_uint((float)(int8_t)((w >> 16) & 0xffu)),
      f3 = __float_as_uint((float)(int8_t)(w >> 24));
  lo = __builtin_amdgcn_perm(f1, f0, 0x07060302u);
  hi = __builtin_amdgcn_perm(f3, f2, 0x07060302u);
}

// exponent e with x < 2^e for the bits of a finite x > 0; 0 for 0
__device__ __forceinline__ int exp_above(uint32_t bits) { return bits ? (int)(bits >> 23) - 126 : 0; }

constexpr float kLift = 7.0f;  // probabilities are kept 2^kLift above their value

// The factor scale 2^e of a block's fp16 scores (of 2^36 at most), a number above 0 whatever the exponents: the scores of
// masked keys are -inf ahead of it, and 2^-126 makes any score as good as 0.
__device__ __forceinline__ float score_factor(float scale_log2, int e) {
  return __builtin_amdgcn_fmed3f(__builtin_ldexpf(scale_log2, e), 0x1p-126f, 0x1.fffffep127f);
}

// A word of 8 four-bit values times their scale, as fp16, in order. A value u at bits 6 to 9 of 16.0's fp16 is 16 + u, so a pair
// is one shift, one and-or and one fma with 24 s: u - 8 has 3 significant bits and s 8 (f16_scale), so that 24 s and the result
// are exact (12 instructions a word).
struct Q4Scale {
  f16x2 s, c;  // s and -24 s
};
__device__ __forceinline__ Q4Scale q4_pair(f16x2 s) {
  const f16x2 k = {(_Float16)-24.0f, (_Float16)-24.0f};
  return {s, s * k};
}
// 16 in both halves, from a vector register: the and-or takes one scalar operand, which is the mask.
__device__ __forceinline__ uint32_t q4_sixteen() {
  uint32_t b = 0x4c004c00u;
  asm("" : "+v"(b));
  return b;
}
// Pair i of a word's (bits 4 i of both halves), times its scale.
__device__ __forceinline__ uint32_t q4_pair_f16(uint32_t w, int i, const Q4Scale& q, uint32_t sixteen) {
  const uint32_t at = i == 0 ? w << 6 : i == 1 ? w << 2 : i == 2 ? w >> 2 : w >> 6;
  const f16x2 x = __builtin_bit_cast(f16x2, (at & 0x03c003c0u) | sixteen);
  return __builtin_bit_cast(uint32_t, __builtin_elementwise_fma(x, q.s, q.c));
}
__device__ __forceinline__ v4u q4x8_f16(uint32_t w, const Q4Scale& q, uint32_t sixteen) {
  return v4u{q4_pair_f16(w, 0, q, sixteen), q4_pair_f16(w, 1, q, sixteen), q4_pair_f16(w, 2, q, sixteen),
             q4_pair_f16(w, 3, q, sixteen)};
}
// A bf16 scale times 2^e in fp16, NaN where it is not finite (an infinite one would make scores of -inf, which are no keys);
// exact unless it falls below fp16's normal numbers.
__device__ __forceinline__ _Float16 f16_scale(uint32_t bits, int e) {
  const float s = (bits & 0x7f80u) == 0x7f80u ? NAN : __uint_as_float(bits << 16);
  return (_Float16)__builtin_ldexpf(s, e);
}
// The frame of 4-bit values whose largest scale has these bf16 bits: 2^E above it, and values below 8 times it, so that q 2^(7 -
// (E - 4)) is below 2^14, as for int8.
__device__ __forceinline__ int q4_frame(uint32_t bits) { return bits ? (int)(bits >> 7) - 126 - 4 : 0; }
// ------------------------------------------------------------------------------------------ few slots: streaming
// Up to 16 or 32 slots of a (sequence, KV head) in a workgroup: decode steps. 4 rep D FLOP per key against 2 D (+ 8)
// bytes of int8 K and V: bound by reading the pages (64 x 4096 tokens of 8 heads of 128 in 70 us, 5.4 TB/s). A wave holds
// 16 slots as the columns of V_MFMA_F32_16X16X32_BF16, or 32 as two of them, and takes 32-key tiles straight from memory
// into registers; the waves of a workgroup take every NW-th tile of the split's range and merge in LDS. Lane (j, g) =
// (lane % 16, lane / 16):
//  * scores S^T[kr] = K[kr] Q^T for the 16-key half tiles kr: the four lanes of a key read 64 contiguous bytes of it at
//    a time (s_dim: a permutation of the reduction index, the same on both sides; reading D / 4 contiguous values per
//    lane instead took 101 against 76 us for the loads of 16 x 8000 bf16 tokens); int8 values enter as exact bf16
//    integers and the score takes the fp32 factor ks_j. The result gives lane (j, g) slot j and keys 16 kr + 4 g + i;
//  * O^T[dt] += V^T[dt] P^T with output row r of d tile dt being d = (D / 16) r + dt and the keys in the order 4 g + i
//    (i < 4), 12 + 4 g + i: the B operand is the lane's own 8 probabilities, the A operand value dt of the D / 16
//    contiguous values it reads of each of those keys. P (times vs_j) enters as bf16 hi + lo parts, 16 significant
//    bits: the columns of the matrix instructions are mostly empty here, and it takes no frames (the low part of a
//    product below 2^-117 begins to be lost under bf16's range).
// Half tiles are reached through buffer descriptors of their own (a half tile never crosses a page), whose length ends
// at the last cached token: what lies behind reads as zeros. Two register sets: a tile's loads are all issued before
// the products of the tile ahead of it, unconditionally (past a wave's last tile with descriptors of no length, so that
// the waits are counted but nothing is read). Rows of 256 go in tiles of one half (R = 1): two sets of whole ones do
// not fit the registers (16 x 8000 tokens 62 us, 49 with halves); bf16 ones then still take a SIMD alone.
//
// 4-bit pages: all of it in fp16, since a value is exact there as (u - 8) d in a power-of-two frame (3 significant bits by 8): the
// slot's queries as fp16 in its frame (in LDS), K and V each in the frame of the largest scale that the wave has seen so far (O moves
// along with V's), probabilities kept 2^7 above their value as in the tile kernels. One product takes P then, no low part: fp16 is
// off by 2^-11 of a probability at most, an eighth of the output's own rounding, and the loop, which the conversions bound beside
// memory, is spared four packings and eight products a tile; l is summed from the unrounded ones.
// Four lanes of a key read all of it (D / 2 bytes), so a lane's K has one scale (two of heads of 256), loaded with it; V's scales
// come one or two a lane and go to the lanes that need them through the LDS crossbar. The new tokens come last, in bf16, where O
// leaves its frame.
constexpr int s_halves(int D, int P) { return D == 256 && P != kInt4 ? 1 : 2; }
template <int D, int P>
struct STile {
  static constexpr bool Q8 = P == kInt8;
  static constexpr int R = s_halves(D, P), KW = D / 4 * (Q8 ? 1 : 2) / 16;  // KW: 16-byte loads of a key's D / 4 values
  static constexpr int VB = D / 16 * (Q8 ? 1 : 2);                           // bytes of a key's D / 16 values: 4 to 32
  v4u k[R][KW];
  uint32_t v[4 * R][VB / 4];
  float ks, vs;  // lane l: the scales of key l % 32
  int len[R];    // keys of the half tiles (wave-uniform)
};
// The key of a half tile that is row r of the products: those of the four lane groups lie side by side, so that a load of V takes
// whole lines (a row of heads of 128 has half a line).
__device__ __forceinline__ constexpr int s_key4(int r) { return 4 * (r & 3) + (r >> 2); }
template <int D>
struct STile<D, kInt4> {
  static constexpr int R = 2, KC = D == 256 ? 2 : 1, KW = D / 32 / KC, VB = D == 256 ? 8 : 4;
  uint32_t k[R][KC][KW];  // chunk c: bytes (64 c +) D / 8 / KC g .. of key j, its words
  uint32_t v[4 * R][VB / 4];
  uint32_t ks[R][KC];  // the scales of those chunks
  uint32_t vs[R];      // lane l: scale l of the half tile's 16 D / 32 (heads of 64: l % 32; of 256: 2 l and 2 l + 1)
  int len[R];
};

// first of the 8 dims that lanes of group g hold in k-step ks
template <int D, int P>
__device__ __forceinline__ int s_dim(int g, int ks) {
  if constexpr (P == kInt4) return D == 256 ? 128 * (ks / 4) + 32 * g + 8 * (ks % 4) : D / 4 * g + 8 * ks;
  return P == kInt8 ? 64 * (ks / 2) + 16 * g + 8 * (ks & 1) : 32 * ks + 8 * g;
}

constexpr int kOnce = 2;  // non-temporal: each byte is read once
__device__ __forceinline__ __amdgpu_buffer_rsrc_t rsrc(const void* p, int bytes) {
  return __builtin_amdgcn_make_buffer_rsrc(const_cast<void*>(p), (short)0, bytes, 0x00020000);
}

// The pages of 64 / R tiles of a wave, one load: lane l has the page of half tile l % R of the wave's tile number l / R
// from here (`pos` of tile 0, `step` positions from tile to tile; -1: no key or no page).
template <int R>
__device__ __forceinline__ int s_pages(const Paged& p, int b, int pos, int step) {
  const int l = threadIdx.x & 63;
  const int64_t at = (int64_t)pos + (int64_t)(l / R) * step + 16 * (l % R), col = at >> p.shift;
  const int pg = col < p.cols ? p.table[b * p.ld_table + col] : -1;
  return pg < p.n_pages ? pg : -1;
}
// A tile's loads, its pages in place `nth` of `pages`. Lane l takes the scales of key l % 32, each 16 lanes their half
// tile's.
template <int D, int P>
__device__ __forceinline__ void s_load_rows(const AttnArgs& a, const Seq& s, int g, int kb, int pages, int nth,
                                       STile<D, P>& x) {
  using T = STile<D, P>;
  constexpr bool Q8 = T::Q8;
  constexpr int E = Q8 ? 1 : 2;
  const int lane = threadIdx.x & 63, j = lane & 15, gl = lane >> 4;
  int64_t row[T::R];
#pragma unroll
  for (int r = 0; r < T::R; ++r) {
    const int pos = kb + 16 * r, pg = __builtin_amdgcn_readlane(pages, nth * T::R + r);
    x.len[r] = pg < 0 || pos >= s.ctx ? 0 : min(16, s.ctx - pos);
    row[r] = (((int64_t)max(pg, 0) * a.p.Hkv + g) << a.p.shift) + (pos & ((1 << a.p.shift) - 1));
    const auto dk = rsrc(static_cast<const char*>(a.p.k) + row[r] * (D * E), x.len[r] * (D * E));
#pragma unroll
    for (int w = 0; w < T::KW; ++w)
      x.k[r][w] = __builtin_bit_cast(
          v4u, __builtin_amdgcn_raw_buffer_load_b128(dk, j * D * E + 64 * w + 16 * gl, 0, kOnce));
    const auto dv = rsrc(static_cast<const char*>(a.p.v) + row[r] * (D * E), x.len[r] * (D * E));
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const int at = (4 * gl + i) * D * E + j * T::VB;
      if constexpr (T::VB == 4) {
        x.v[4 * r + i][0] = __builtin_amdgcn_raw_buffer_load_b32(dv, at, 0, kOnce);
      } else if constexpr (T::VB == 8) {
        const auto u = __builtin_amdgcn_raw_buffer_load_b64(dv, at, 0, kOnce);
        x.v[4 * r + i][0] = u[0];
        x.v[4 * r + i][1] = u[1];
      } else {
#pragma unroll
        for (int w = 0; w < T::VB / 16; ++w) {
          const v4u u = __builtin_bit_cast(v4u, __builtin_amdgcn_raw_buffer_load_b128(dv, at + 16 * w, 0, kOnce));
#pragma unroll
          for (int c = 0; c < 4; ++c) x.v[4 * r + i][4 * w + c] = u[c];
        }
      }
    }
  }
  if constexpr (Q8) {
    // a lane's own row: one descriptor cannot reach both half tiles, so lanes without a key read the pool's first scale
    constexpr int kUpper = T::R - 1;  // tiles of one half: lanes 16 .. 31 take the same keys as 0 .. 15
    const int c = lane & 31;
    const bool in = (c & 15) < (c < 16 ? x.len[0] : x.len[kUpper]);
    const int64_t at = in ? (c < 16 ? row[0] : row[kUpper]) + (c & 15) : 0;
    const float k1 = a.p.ks[at], v1 = a.p.vs[at];
    x.ks = in ? k1 : 0.0f;
    x.vs = in ? v1 : 0.0f;
  }
}
template <int D, int P>
__device__ __forceinline__ void s_load(const AttnArgs& a, const Seq& s, int g, int kb, int pages, int nth, STile<D, P>& x) {
  if constexpr (P == kInt4) {
    using T = STile<D, P>;
    const int lane = threadIdx.x & 63, j = lane & 15, gl = lane >> 4;
#pragma unroll
    for (int r = 0; r < 2; ++r) {
      const int pos = kb + 16 * r, pg = __builtin_amdgcn_readlane(pages, nth * 2 + r);
      x.len[r] = pg < 0 || pos >= s.ctx ? 0 : min(16, s.ctx - pos);
      const int64_t row = (((int64_t)max(pg, 0) * a.p.Hkv + g) << a.p.shift) + (pos & ((1 << a.p.shift) - 1));
      const auto dk = rsrc(static_cast<const char*>(a.p.k) + row * (D / 2), x.len[r] * (D / 2));
      const auto dv = rsrc(static_cast<const char*>(a.p.v) + row * (D / 2), x.len[r] * (D / 2));
      const auto sk = rsrc(a.p.k4 + row * (D / 32), x.len[r] * (D / 16)), sv = rsrc(a.p.v4 + row * (D / 32), x.len[r] * (D / 16));
#pragma unroll
      for (int c = 0; c < T::KC; ++c) {
        const int at = s_key4(j) * (D / 2) + 64 * c + 4 * T::KW * gl;
        if constexpr (T::KW == 4) {
          const v4u u = __builtin_bit_cast(v4u, __builtin_amdgcn_raw_buffer_load_b128(dk, at, 0, kOnce));
#pragma unroll
          for (int w = 0; w < 4; ++w) x.k[r][c][w] = u[w];
        } else {
          const auto u = __builtin_amdgcn_raw_buffer_load_b64(dk, at, 0, kOnce);
          x.k[r][c][0] = u[0], x.k[r][c][1] = u[1];
        }
        x.ks[r][c] = (uint16_t)__builtin_amdgcn_raw_buffer_load_b16(sk, 2 * (s_key4(j) * (D / 32) + 4 * c + (D == 64 ? gl / 2 : gl)), 0, 0);
      }
#pragma unroll
      for (int i = 0; i < 4; ++i) {  // heads of 64: two lanes share a word
        const int at = s_key4(4 * gl + i) * (D / 2) + (D == 64 ? 4 * (j / 2) : T::VB * j);
        if constexpr (T::VB == 4) {
          x.v[4 * r + i][0] = __builtin_amdgcn_raw_buffer_load_b32(dv, at, 0, kOnce);
        } else {
          const auto u = __builtin_amdgcn_raw_buffer_load_b64(dv, at, 0, kOnce);
          x.v[4 * r + i][0] = u[0], x.v[4 * r + i][1] = u[1];
        }
      }
      if constexpr (D == 256) x.vs[r] = __builtin_amdgcn_raw_buffer_load_b32(sv, 4 * lane, 0, 0);
      else x.vs[r] = (uint16_t)__builtin_amdgcn_raw_buffer_load_b16(sv, 2 * (D == 64 ? lane & 31 : lane), 0, 0);
    }
  } else {
    s_load_rows<D, P>(a, s, g, kb, pages, nth, x);
  }
}
__device__ __forceinline__ v4f mfma16(v4u a, v4u b, v4f c) {
  return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8, a), __builtin_bit_cast(bf16x8, b), c, 0,
                                                 0, 0);
}

__device__ __forceinline__ v4f mfma16h(v4u a, v4u b, v4f c) {
  return __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(f16x8, a), __builtin_bit_cast(f16x8, b), c, 0, 0, 0);
}

// The slot state of a lane: column j's running max and its share of the sum, output rows 4 g + i of every d tile.
template <int D>
struct SAcc {
  float m, l;
  v4f o[D / 16];
};

// One tile's online softmax: y the lane's 8 scores (log2 units, -inf masked); p out, 2^s_lift above its value.
constexpr float s_lift(int P) { return P == kInt4 ? kLift : 0.0f; }
template <int P, int D>
__device__ __forceinline__ void s_probabilities(float (&y)[8], SAcc<D>& x, float (&p)[8]) {
  float mx = y[0];
#pragma unroll
  for (int i = 1; i < 8; ++i) mx = fmaxf(mx, y[i]);
  mx = fmaxf(mx, __shfl_xor(mx, 16, 64));
  mx = od_xor32_max(mx);
  const bool move = mx > x.m + kSlack;
  if (__builtin_amdgcn_ballot_w64(move) != 0) {
    const float c = move ? __builtin_amdgcn_exp2f(x.m - mx) : 1.0f;  // m = -inf: 0
#pragma unroll
    for (int dt = 0; dt < D / 16; ++dt)
#pragma unroll
      for (int i = 0; i < 4; ++i) x.o[dt][i] *= c;
    x.l *= c;
    if (move) x.m = mx;
  }
  const float ms = (x.m == -INFINITY ? 0.0f : x.m) - s_lift(P);
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    p[i] = __builtin_amdgcn_exp2f(y[i] - ms);
    x.l += p[i];
  }
}
// The same from scores in units of 1 / c (c > 0), into fp16.
template <int D>
__device__ __forceinline__ v4u s_half(const float (&y)[8], float c, SAcc<D>& x) {
  float mx = y[0];
#pragma unroll
  for (int i = 1; i < 8; ++i) mx = fmaxf(mx, y[i]);
  mx = fmaxf(mx, __shfl_xor(mx, 16, 64));
  mx = od_xor32_max(mx) * c;
  const bool move = mx > x.m + kSlack;
  if (__builtin_amdgcn_ballot_w64(move) != 0) {
    const float f = move ? __builtin_amdgcn_exp2f(x.m - mx) : 1.0f;  // m = -inf: 0
#pragma unroll
    for (auto& o : x.o) o *= f;
    x.l *= f;
    if (move) x.m = mx;
  }
  const float ms = (x.m == -INFINITY ? 0.0f : x.m) - kLift;
  v4u r;
#pragma unroll
  for (int e = 0; e < 4; ++e) {
    const float p0 = __builtin_amdgcn_exp2f(__builtin_fmaf(y[2 * e], c, -ms));
    const float p1 = __builtin_amdgcn_exp2f(__builtin_fmaf(y[2 * e + 1], c, -ms));
    x.l += p0;
    x.l += p1;
    const f16x2 w = {(_Float16)p0, (_Float16)p1};
    r[e] = __builtin_bit_cast(uint32_t, w);
  }
  return r;
}
// The same into bf16 hi and lo parts: f a factor on p for the P.V product only (the V scales).
template <int D, int P, bool F>
__device__ __forceinline__ void s_softmax(float (&y)[8], const float (&f)[8], SAcc<D>& x, v4u& hi, v4u& lo) {
  float p[8];
  s_probabilities<P>(y, x, p);
#pragma unroll
  for (int e = 0; e < 4; ++e) {
    const float u = F ? p[2 * e] * f[2 * e] : p[2 * e], w = F ? p[2 * e + 1] * f[2 * e + 1] : p[2 * e + 1];
    hi[e] = od_pack_bf16x2(u, w);
    lo[e] = od_pack_bf16x2(u - __uint_as_float(hi[e] << 16), w - __uint_as_float(hi[e] & 0xffff0000u));
  }
}

// value dt of each of the lane's 8 keys, as the bf16 A operand
template <int D, int P, int NK>
__device__ __forceinline__ v4u s_vfrag(const uint32_t (&v)[NK][STile<D, P>::VB / 4], int dt) {
  constexpr bool Q8 = P == kInt8;
  v4u r = v4u{0, 0, 0, 0};
#pragma unroll
  for (int e = 0; e < NK / 2; ++e) {
    if constexpr (Q8) {
      const uint32_t a = v[2 * e][dt / 4], b = v[2 * e + 1][dt / 4];
      const int sh = 8 * (dt % 4);
      r[e] = __builtin_amdgcn_perm(__float_as_uint((float)(int8_t)(b >> sh)),
          __float_as_uint((float)(int8_t)(a >> sh)), 0x07060302u);
    } else {
      r[e] = __builtin_amdgcn_perm(v[2 * e + 1][dt / 2], v[2 * e][dt / 2], dt % 2 ? 0x07060302u : 0x05040100u);
    }
  }
  return r;
}

// The maxima of both halves of a word over the wave.
template <int CTRL, int ROW_MASK>
__device__ __forceinline__ uint32_t s_max2_step(uint32_t x) {
  return od_absmax_bf16x2(x, (uint32_t)__builtin_amdgcn_update_dpp((int)x, (int)x, CTRL, ROW_MASK, 0xf, false));
}
__device__ __forceinline__ uint32_t s_wave_max2(uint32_t x) {
  x = s_max2_step<0xB1, 0xf>(x);   // quad_perm [1,0,3,2]
  x = s_max2_step<0x4E, 0xf>(x);   // quad_perm [2,3,0,1]
  x = s_max2_step<0x124, 0xf>(x);  // row_ror:4
  x = s_max2_step<0x128, 0xf>(x);  // row_ror:8
  x = s_max2_step<0x142, 0xa>(x);  // row_bcast:15 into rows 1 and 3
  x = s_max2_step<0x143, 0xc>(x);  // row_bcast:31 into rows 2 and 3
  return (uint32_t)__builtin_amdgcn_readlane((int)x, 63);
}

// In the frames of fp16, values are below 2^14 and no sum of them passes fp32. The new tokens' bf16 values are as they are, and
// probabilities of up to 2^(kLift + kSlack) beside values of 2^113 do pass it, though O / l is finite. Work whose O is not, once they
// were added, is done again with one factor of the products times 2^-64 (0 below 2^-63) and O in units of 2^64: no sum of finite values
// passes fp32 then. Only the outputs that were not finite are taken from it: what is small beside large or infinite values stays as it
// was. Rare: it costs a look at O.
constexpr int kLower = 64;
// Four outputs, or a split's, at their place; again: only those that are not finite there (the lane's own, written before).
__device__ __forceinline__ void put4(uint16_t* at, float4 y, bool again) {
  uint2 w = make_uint2(od_pack_bf16x2(y.x, y.y), od_pack_bf16x2(y.z, y.w));
  if (again) {
    const uint2 old = *reinterpret_cast<const uint2*>(at);
    auto pick = [](uint32_t o, uint32_t n) {
      const uint32_t keep = ((o & 0x7f80u) != 0x7f80u ? 0xffffu : 0u) | ((o & 0x7f800000u) != 0x7f800000u ? 0xffff0000u : 0u);
      return (o & keep) | (n & ~keep);
    };
    w = make_uint2(pick(old.x, w.x), pick(old.y, w.y));
  }
  *reinterpret_cast<uint2*>(at) = w;
}
__device__ __forceinline__ void put4(float* at, float4 y, bool again) {
  if (again) {
    const float4 old = *reinterpret_cast<const float4*>(at);
    auto pick = [](float o, float n) { return fabsf(o) < INFINITY ? o : n; };
    y = make_float4(pick(old.x, y.x), pick(old.y, y.y), pick(old.z, y.z), pick(old.w, y.w));
  }
  *reinterpret_cast<float4*>(at) = y;
}
__device__ __forceinline__ uint32_t lower_bf16x2(uint32_t w) {  // infinities and NaN as they are
  uint32_t r = w & 0x80008000u;
#pragma unroll
  for (int i = 0; i < 32; i += 16) {
    const int m = (int)(w >> i & 0x7fffu);
    r |= (uint32_t)(m >= 0x7f80 ? m : max(m - (kLower << 7), 0)) << i;
  }
  return r;
}

constexpr int kStreamWaves = 4;
// waves a SIMD's registers hold
constexpr int s_waves(int D, int P, int columns) {
  if (D * columns >= (P == kBf16 ? 256 : 512)) return 1;
  return P == kInt4 && D <= 128 && columns == 1 ? 3 : 2;
}

template <int D, int P, int CT, int WAVES = s_waves(D, P, CT)>
__global__ __launch_bounds__(kStreamWaves * 64, WAVES) void paged_stream_kernel(AttnArgs a) {
  constexpr bool Q8 = P == kInt8, Q4 = P == kInt4;
  using Tile = STile<D, P>;
  // QR: 16 slots' rows start in 16 distinct 16-byte bank groups
  constexpr int NW = kStreamWaves, KS = D / 32, R = s_halves(D, P), QR = D + 8;
  __shared__ __attribute__((aligned(16))) union {
    struct {
      uint16_t q[16 * CT * QR];
      uint16_t q16[Q4 ? 16 * CT * QR : 8];  // 4-bit pages: the queries as fp16 in their frames, whose exponents are qe
    };
    float o[NW][16][D + 4];
  } sm;
  __shared__ int qe[Q4 ? 16 * CT : 1], frames[NW], over;  // over: some O is not finite
  __shared__ float sml[NW][2][16];
  // a tile's per-key factors, from lane order to score order (one wave writes and reads)
  __shared__ float4 skf[Q8 ? NW : 1][2][8];
  const int sp = blockIdx.x, g = blockIdx.y % a.p.Hkv, b = blockIdx.z;
  constexpr int W = 16 * R, PT = 64 / R, SETS = 2;  // PT: tiles whose pages one load brings
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int j = lane & 15, qd = lane >> 4, c = lane & 31;
  // A short call is a chain of memory latencies: lengths and page numbers; queries, then the first tiles; the rest.
  const int t_lo = sp * a.chunk;
  const int pages0 = s_pages<R>(a.p, b, (t_lo + wave) * W, NW * W);
  const Seq s = seq_of(a, b);
  const int tiles = (s.ctx + W - 1) / W, nv = splits_of(a, tiles);
  if (s.n == 0 || sp >= nv) return;  // uniform over the workgroup
  const int t_hi = sp == a.nsplit - 1 ? tiles : min(tiles, t_lo + a.chunk);
  // 4-bit pages: what is not needed in the loop over the tiles is formed from the thread's number where it is, not kept in
  // registers over it (they spill else, and a kernel with scratch memory costs 64 tokens over 4096 each 57 us, 52 without).
  auto thread = [&] {
    int t = threadIdx.x;
    if constexpr (Q4) asm volatile("" : "+v"(t));
    return t;
  };
  // one round unless max_new was too small
  int lower = 0;  // the power of two that the new tokens' probabilities are lowered by
  const int z_lo = blockIdx.y / a.p.Hkv * 16 * CT;
  for (int z0 = z_lo; z0 < s.n * a.rep;) {
    constexpr int QN = 16 * CT * (D / 8), QC = QN / (NW * 64) ? QN / (NW * 64) : 1;
    uint4 qw[QC];
#pragma unroll
    for (int k = 0; k < QC; ++k) {
      const int i = k * NW * 64 + threadIdx.x, z = z0 + i / (D / 8), d0 = (i % (D / 8)) * 8;
      qw[k] = make_uint4(0, 0, 0, 0);
      if (i < QN && z < s.n * a.rep)
        qw[k] = *reinterpret_cast<const uint4*>(a.q + (int64_t)(s.s0 + z / a.rep) * a.sqt +
                                                (int64_t)(g * a.rep + z % a.rep) * a.sqh + d0);
    }
    int tt = t_lo + wave, nth = -1;
    int pages = !Q4 || (z0 == z_lo && lower == 0) ? pages0 : s_pages<R>(a.p, b, tt * W, NW * W);
    // the wave's next tile into x (past the last one: an empty one, without traffic)
    Tile tl[SETS];
    int asked = tt - NW;  // the tile last asked for
    auto next = [&](Tile& x) {
      const bool more = asked + NW < t_hi;
      if (more) {
        asked += NW;
        if (++nth == PT) {
          nth = 0;
          pages = s_pages<R>(a.p, b, asked * W, NW * W);
        }
      }
      s_load<D, P>(a, s, g, more ? asked * W : s.ctx, pages, nth, x);
      __builtin_amdgcn_sched_barrier(0);
    };
    if (tt < t_hi) {
#pragma unroll
      for (int i = 0; i < SETS - 1; ++i) next(tl[i]);
    }
    __syncthreads();  // an earlier round's readers are done
    if (Q4 && threadIdx.x == 0) over = 0;
#pragma unroll
    for (int k = 0; k < QC; ++k) {
      const int i = k * NW * 64 + threadIdx.x;
      if (i < QN) *reinterpret_cast<uint4*>(sm.q + (i / (D / 8)) * QR + (i % (D / 8)) * 8) = qw[k];
      if constexpr (Q4) {  // (D / 8 lanes a slot)
        uint32_t am = od_absmax_bf16x2(od_absmax_bf16x2(od_absmax_bf16x2(od_absmax_bf16x2(0, qw[k].x), qw[k].y), qw[k].z), qw[k].w);
        am = max(am & 0xffffu, am >> 16);
#pragma unroll
        for (int o = D / 16; o > 0; o >>= 1) am = max(am, (uint32_t)__shfl_xor((int)am, o, 64));
        const int e = am < 0x7f80u ? exp_above(am << 16) : 0;
        const uint32_t w[4] = {qw[k].x, qw[k].y, qw[k].z, qw[k].w};
        uint32_t h[4];
#pragma unroll
        for (int c2 = 0; c2 < 4; ++c2) {
          const f16x2 r = {(_Float16)__builtin_ldexpf(__uint_as_float(w[c2] << 16), 14 - e),
                           (_Float16)__builtin_ldexpf(__uint_as_float(w[c2] & 0xffff0000u), 14 - e)};
          h[c2] = __builtin_bit_cast(uint32_t, r);
        }
        const int i4 = k * NW * 64 + thread();
        if (i4 < QN) {
          *reinterpret_cast<uint4*>(sm.q16 + (i4 / (D / 8)) * QR + (i4 % (D / 8)) * 8) = make_uint4(h[0], h[1], h[2], h[3]);
          if (i4 % (D / 8) == 0) qe[i4 / (D / 8)] = e;
        }
      }
    }
    __syncthreads();
    auto qfrag = [&](int ct, int ks) {
      return __builtin_bit_cast(v4u, *reinterpret_cast<const uint4*>(sm.q + (16 * ct + j) * QR + s_dim<D, P>(qd, ks)));
    };
    int frame = 0;  // 4-bit pages: O is in units of 2^frame
    SAcc<D> acc[CT];
#pragma unroll
    for (auto& x : acc) {
      x.m = -INFINITY;
      x.l = 0.0f;
#pragma unroll
      for (int dt = 0; dt < D / 16; ++dt) x.o[dt] = v4f{0, 0, 0, 0};
    }

    // The new tokens, tiles of 16 bf16 keys (as many as the slots have tokens), in split 0: by the last waves, which
    // have the fewest tiles of pages, and first, while the pages are on their way (heads of 256: last, the registers do
    // not hold both).
    auto new_tokens = [&] {
      if (sp != 0 || !a.k) return;
      const int t0 = thread(), j = t0 & 15, qd = t0 >> 4 & 3, c = t0 & 31;
      if (Q4 && frame != lower) {
        const float f = __builtin_ldexpf(1.0f, frame - lower);
#pragma unroll
        for (auto& x : acc)
#pragma unroll
          for (auto& o : x.o)
#pragma unroll
            for (int i = 0; i < 4; ++i) o[i] *= f;
      }
      if constexpr (Q4) frame = lower;
      const int t_end = min((z0 + 16 * CT - 1) / a.rep, s.n - 1);  // last token of these slots
      int k_lo = 0;                                                // the first one that any of them sees
      if (a.row_begin) {
        k_lo = max(a.row_begin[s.s0 + min((z0 + c) / a.rep, t_end)], 0);  // c: the slots of both columns
#pragma unroll
        for (int o = 16; o > 0; o >>= 1) k_lo = min(k_lo, __shfl_xor(k_lo, o, 64));
        k_lo = __builtin_amdgcn_readfirstlane(min(k_lo, t_end + 1)) & ~15;
      }
#pragma unroll 1
      for (int k0 = k_lo + 16 * (NW - 1 - wave); k0 <= t_end; k0 += 16 * NW) {
        const int left = min(16, s.n - k0);
        const uint16_t* kp = a.k + (int64_t)(s.s0 + k0 + min(j, left - 1)) * a.skt + (int64_t)g * a.skh;
        v4u kr[KS];
#pragma unroll
        for (int ks = 0; ks < KS; ++ks)
          kr[ks] = __builtin_bit_cast(v4u, *reinterpret_cast<const uint4*>(kp + s_dim<D, P>(qd, ks)));
        uint32_t v[4][D / 32];
        bool odd = false;
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const uint16_t* vp =
              a.v + (int64_t)(s.s0 + k0 + min(4 * qd + i, left - 1)) * a.svt + (int64_t)g * a.svh + j * (D / 16);
#pragma unroll
          for (int w = 0; w < D / 64; ++w) {
            const uint2 u = *reinterpret_cast<const uint2*>(vp + 4 * w);
            v[i][2 * w] = u.x;
            v[i][2 * w + 1] = u.y;
          }
        }
        // infinities or NaN among the values: 0 times one must not reach a slot that does not see it, so the products
        // take 0 in their places, and the slots that see one get it added
#pragma unroll
        for (int i = 0; i < 4; ++i)
#pragma unroll
          for (int w = 0; w < D / 32; ++w) {
            const uint32_t f = fin_bf16x2(v[i][w]);
            odd |= f != v[i][w];
            v[i][w] = f;
          }
#pragma unroll
        for (int ct = 0; ct < CT; ++ct) {
          const int z = z0 + 16 * ct + j, tok = min(z / a.rep, s.n - 1);
          const int begin = a.row_begin ? max(a.row_begin[s.s0 + tok], 0) : 0;
          SAcc<D>& x = acc[ct];
          v4f sc = v4f{0, 0, 0, 0};
#pragma unroll
          for (int ks = 0; ks < KS; ++ks) sc = mfma16(kr[ks], qfrag(ct, ks), sc);
          float y[8], f[8];
#pragma unroll
          for (int i = 0; i < 8; ++i) {
            const int key = k0 + 4 * qd + i;
            y[i] = i < 4 && z < s.n * a.rep && key >= begin && key <= tok ? sc[i & 3] * a.scale_log2 : -INFINITY;
            f[i] = 1.0f;
          }
          v4u hi, lo;
          s_softmax<D, P, false>(y, f, x, hi, lo);
          if (Q4 && lower) {
#pragma unroll
            for (int e = 0; e < 2; ++e) hi[e] = lower_bf16x2(hi[e]), lo[e] = lower_bf16x2(lo[e]);
          }
          if (__builtin_amdgcn_ballot_w64(odd) != 0) {
#pragma unroll 1
            for (int key = k0; key < k0 + left; ++key) {
              if (z >= s.n * a.rep || key < begin || key > tok) continue;
              const uint16_t* vp = a.v + (int64_t)(s.s0 + key) * a.svt + (int64_t)g * a.svh + 4 * qd * (D / 16);
#pragma unroll
              for (int dt = 0; dt < D / 16; ++dt)
#pragma unroll
                for (int i = 0; i < 4; ++i) x.o[dt][i] += odd_bf16(vp[i * (D / 16) + dt]);
            }
          }
#pragma unroll
          for (int dt = 0; dt < D / 16; ++dt) {
            const v4u v8 = s_vfrag<D, kBf16, 4>(v, dt);
            x.o[dt] = mfma16(v8, hi, x.o[dt]);
            x.o[dt] = mfma16(v8, lo, x.o[dt]);
          }
        }
      }
    };
    constexpr bool first = D < 256 && !Q4;
    if constexpr (first) new_tokens();

    // one tile's scores, softmax and products
    // 4-bit pages: the largest scales within the frames, as bits (0 at first: no frame yet), K's frame
    uint32_t bound = 0;
    int kexp = 0;
    int qexp[CT];
    if constexpr (Q4) {
#pragma unroll
      for (int ct = 0; ct < CT; ++ct) qexp[ct] = qe[16 * ct + j];
    }
    auto products4 = [&](auto& tl, auto& acc) {
      using T = std::decay_t<decltype(tl)>;
      const uint32_t sixteen = q4_sixteen();
      // Scales past the frames (K's in the low halves of a word, V's in the high ones): rare, the frames then rise.
      uint32_t big = bound;
#pragma unroll
      for (int r = 0; r < 2; ++r) {
        big = od_absmax_bf16x2(big, tl.ks[r][0] | tl.vs[r] << 16);
        if constexpr (D == 256) big = od_absmax_bf16x2(big, tl.ks[r][1] | (tl.vs[r] & 0xffff0000u));
      }
      if (__builtin_amdgcn_ballot_w64(big != bound) != 0) {
        big = bound;
#pragma unroll
        for (int r = 0; r < 2; ++r) {  // the finite ones
          big = od_absmax_bf16x2(big, fin_bf16x2(tl.ks[r][0] | tl.vs[r] << 16));
          if constexpr (D == 256) big = od_absmax_bf16x2(big, fin_bf16x2(tl.ks[r][1] | (tl.vs[r] & 0xffff0000u)));
        }
        big = s_wave_max2(big) | 0x007f007fu;
        if ((big & 0xffffu) > (bound & 0xffffu)) kexp = q4_frame(big & 0xffffu);
        if (big >> 16 > bound >> 16) {
          const int to = q4_frame(big >> 16) - 7;
          if (bound >> 16) {
            const float f = __builtin_ldexpf(1.0f, frame - to);
#pragma unroll
            for (auto& x : acc)
#pragma unroll
              for (auto& o : x.o)
#pragma unroll
                for (int i = 0; i < 4; ++i) o[i] *= f;
          }
          frame = to;
        }
        bound = big;
      }
      v4f sc[CT][2];
#pragma unroll
      for (auto& c2 : sc) c2[0] = c2[1] = v4f{0, 0, 0, 0};
#pragma unroll
      for (int c4 = 0; c4 < T::KC; ++c4) {
        Q4Scale q[2];
#pragma unroll
        for (int r = 0; r < 2; ++r) {
          const _Float16 h = (_Float16)__builtin_ldexpf(__uint_as_float(tl.ks[r][c4] << 16), 7 - kexp);
          q[r] = q4_pair(f16x2{h, h});  // (an infinite scale makes NaN: inf - inf)
        }
#pragma unroll
        for (int w = 0; w < T::KW; ++w) {
          v4u qf[CT];
#pragma unroll
          for (int ct = 0; ct < CT; ++ct)
            qf[ct] = __builtin_bit_cast(v4u, *reinterpret_cast<const uint4*>(sm.q16 + (16 * ct + j) * QR +
                                                                            s_dim<D, P>(qd, 4 * c4 + w)));
#pragma unroll
          for (int r = 0; r < 2; ++r) {
            const v4u k8 = q4x8_f16(tl.k[r][c4][w], q[r], sixteen);
#pragma unroll
            for (int ct = 0; ct < CT; ++ct) sc[ct][r] = mfma16h(k8, qf[ct], sc[ct][r]);
          }
        }
      }
      v4u pb[CT];
#pragma unroll
      for (int ct = 0; ct < CT; ++ct) {
        float y[8];
#pragma unroll
        for (int i = 0; i < 8; ++i) y[i] = sc[ct][i >> 2][i & 3];
        if (__builtin_expect(tl.len[0] + tl.len[1] != 32, 0)) {
          // a branch: else the comparisons are made for every tile, and the keys' places kept over all of them
          const int q = thread() >> 4 & 3;
#pragma unroll
          for (int i = 0; i < 8; ++i)
            if (s_key4(4 * q + (i & 3)) >= tl.len[i >> 2]) y[i] = -INFINITY;
        }
        pb[ct] = s_half<D>(y, score_factor(a.scale_log2, qexp[ct] - 14 + kexp - 7), acc[ct]);
      }
      // V's scales of the lane's columns and of its 8 keys, in pairs of keys
      Q4Scale vq[4];
#pragma unroll
      for (int r = 0; r < 2; ++r) {
        const _Float16 h0 = (_Float16)__builtin_ldexpf(__uint_as_float(tl.vs[r] << 16), -frame);
        uint32_t mine = __builtin_bit_cast(uint16_t, h0);
        if constexpr (D == 256) {
          const _Float16 h1 = (_Float16)__builtin_ldexpf(__uint_as_float(tl.vs[r] & 0xffff0000u), -frame);
          mine |= (uint32_t)__builtin_bit_cast(uint16_t, h1) << 16;
        }
        uint32_t of[4];
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const int from = D == 64 ? 2 * s_key4(4 * qd + i) + (j >> 3) : 4 * s_key4(4 * qd + i) + (j >> 2);
          of[i] = (uint32_t)__builtin_amdgcn_ds_bpermute(4 * from, (int)mine);
        }
        const uint32_t sel = D == 256 && (j & 2) ? 0x07060302u : 0x05040100u;
#pragma unroll
        for (int i = 0; i < 2; ++i)
          vq[2 * r + i] = q4_pair(__builtin_bit_cast(f16x2, __builtin_amdgcn_perm(of[2 * i + 1], of[2 * i], sel)));
      }
      // columns dt: value dt of the lane's D / 16, from the words of two keys the even values and the odd ones side by side
      constexpr int WORDS = D == 256 ? 2 : 1, PER = D == 64 ? 2 : 4;  // value pairs of a word
#pragma unroll
      for (int w = 0; w < WORDS; ++w) {
        uint32_t even[4], odd[4];
#pragma unroll
        for (int k2 = 0; k2 < 4; ++k2) {
          uint32_t x0 = tl.v[2 * k2][w], x1 = tl.v[2 * k2 + 1][w];
          if constexpr (D == 64) x0 >>= 8 * (j & 1), x1 >>= 8 * (j & 1);
          even[k2] = __builtin_amdgcn_perm(x1, x0, 0x05040100u);
          odd[k2] = __builtin_amdgcn_perm(x1, x0, 0x07060302u);
        }
#pragma unroll
        for (int dt = 0; dt < 2 * PER; ++dt) {
          v4u v8;
#pragma unroll
          for (int k2 = 0; k2 < 4; ++k2) {
            v8[k2] = q4_pair_f16(dt & 1 ? odd[k2] : even[k2], dt / 2, vq[k2], sixteen);
          }
#pragma unroll
          for (int ct = 0; ct < CT; ++ct) acc[ct].o[8 * w + dt] = mfma16h(v8, pb[ct], acc[ct].o[8 * w + dt]);
        }
      }
    };
    auto products = [&](auto& tl) {
      if constexpr (Q8) {  // in-order LDS access within the wave; lanes c and c + 32 write the same value
        // (an infinite scale as NaN: a score of -inf would be no key)
        reinterpret_cast<float*>(skf[wave][0])[c] = tl.ks < INFINITY ? tl.ks * a.scale_log2 : NAN;
        reinterpret_cast<float*>(skf[wave][1])[c] = tl.vs;
      }
      v4f sc[CT][2];
#pragma unroll
      for (auto& c2 : sc) c2[0] = c2[1] = v4f{0, 0, 0, 0};
#pragma unroll
      for (int ks = 0; ks < KS; ++ks)
#pragma unroll
        for (int r = 0; r < R; ++r) {
          v4u k8;
          if constexpr (Q8) {
            uint32_t w[4];
            i8x4_to_bf16(tl.k[r][ks / 2][2 * (ks & 1)], w[0], w[1]);
            i8x4_to_bf16(tl.k[r][ks / 2][2 * (ks & 1) + 1], w[2], w[3]);
            k8 = v4u{w[0], w[1], w[2], w[3]};
          } else {
            k8 = tl.k[r][ks];
          }
#pragma unroll
          for (int ct = 0; ct < CT; ++ct) sc[ct][r] = mfma16(k8, qfrag(ct, ks), sc[ct][r]);
        }
      float kk[8], f[8];
#pragma unroll
      for (int r = 0; r < 2; ++r) {
        const float4 kf = Q8 ? skf[wave][0][4 * r + qd]
                             : make_float4(a.scale_log2, a.scale_log2, a.scale_log2, a.scale_log2);
        const float4 vf = Q8 ? skf[wave][1][4 * r + qd] : make_float4(1, 1, 1, 1);
        const float k4[4] = {kf.x, kf.y, kf.z, kf.w}, v4[4] = {vf.x, vf.y, vf.z, vf.w};
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          kk[4 * r + i] = k4[i];
          f[4 * r + i] = v4[i];
        }
      }
      int there = 0;
#pragma unroll
      for (int r = 0; r < R; ++r) there += tl.len[r];
      v4u hi[CT], lo[CT];
#pragma unroll
      for (int ct = 0; ct < CT; ++ct) {
        float y[8];
#pragma unroll
        for (int i = 0; i < 8; ++i) y[i] = i < 4 * R ? sc[ct][i >> 2][i & 3] * kk[i] : -INFINITY;
        if (there != 16 * R) {
#pragma unroll
          for (int i = 0; i < 4 * R; ++i)
            if (4 * qd + (i & 3) >= tl.len[i >> 2]) y[i] = -INFINITY;
        }
        s_softmax<D, P, Q8>(y, f, acc[ct], hi[ct], lo[ct]);
      }
      if constexpr (!Q8) {
        // The low part of a probability may be 0 or negative: infinities and NaN among the values are taken by the high
        // part alone, ahead of the products, which take 0 in their places.
        uint32_t m = 0;
#pragma unroll
        for (auto& key : tl.v)
#pragma unroll
          for (const uint32_t w : key) m = od_absmax_bf16x2(m, w);
        if (__builtin_amdgcn_ballot_w64((m & 0xffffu) >= 0x7f80u || (m >> 16) >= 0x7f80u) != 0) {
#pragma unroll
          for (int dt = 0; dt < D / 16; ++dt) {
            const v4u v8 = s_vfrag<D, P, 4 * R>(tl.v, dt), fin = fin_bf16x8(v8);
#pragma unroll
            for (int ct = 0; ct < CT; ++ct) acc[ct].o[dt] = mfma16(v8 ^ fin, hi[ct], acc[ct].o[dt]);
          }
#pragma unroll
          for (auto& key : tl.v)
#pragma unroll
            for (uint32_t& w : key) w = fin_bf16x2(w);
        }
      }
#pragma unroll
      for (int dt = 0; dt < D / 16; ++dt) {
        const v4u v8 = s_vfrag<D, P, 4 * R>(tl.v, dt);
#pragma unroll
        for (int ct = 0; ct < CT; ++ct) {
          acc[ct].o[dt] = mfma16(v8, hi[ct], acc[ct].o[dt]);
          acc[ct].o[dt] = mfma16(v8, lo[ct], acc[ct].o[dt]);
        }
      }
    };
    if (tt < t_hi) {
      for (bool more = true; more;) {
#pragma unroll
        for (int i = 0; i < SETS; ++i) {
          next(tl[(i + SETS - 1) % SETS]);
          if constexpr (Q4) products4(tl[i], acc);
          else products(tl[i]);
          tt += NW;
          if (!(more = tt < t_hi)) break;
        }
      }
    }

    if constexpr (!first) new_tokens();

    if (Q4 && sp == 0 && a.k && lower == 0) {
      v4f sum = v4f{0, 0, 0, 0};  // NaN where an O is past 2^124: the waves' sum is finite below it
#pragma unroll
      for (auto& x : acc)
#pragma unroll
        for (auto& o : x.o)
#pragma unroll
          for (int i = 0; i < 4; ++i) sum[i] = __builtin_fmaf(o[i] * 16.0f, 0.0f, sum[i]);
      if (sum[0] + sum[1] + sum[2] + sum[3] != 0.0f) over = 1;
    }
    // merge the waves, then the output or this split's normalized partial
    const int tid = thread(), j = tid & 15, qd = tid >> 4 & 3;
#pragma unroll
    for (int ct = 0; ct < CT; ++ct) {
      const SAcc<D>& x = acc[ct];
      float l = x.l + __shfl_xor(x.l, 16, 64);
      l = od_xor32_sum(l);
      __syncthreads();  // every wave is done with the queries, or the columns before
#pragma unroll
      for (int i = 0; i < 4; ++i)
#pragma unroll
        for (int d4 = 0; d4 < D / 64; ++d4)
          *reinterpret_cast<float4*>(&sm.o[wave][j][(4 * qd + i) * (D / 16) + 4 * d4]) =
              make_float4(x.o[4 * d4][i], x.o[4 * d4 + 1][i], x.o[4 * d4 + 2][i], x.o[4 * d4 + 3][i]);
      if (qd == 0) {
        sml[wave][0][j] = x.m;
        sml[wave][1][j] = l;
      }
      if (Q4 && (tid & 63) == 0) frames[wave] = frame;
      __syncthreads();
      for (int i = tid; i < 16 * (D / 4); i += NW * 64) {
        const int zz = i / (D / 4), d0 = (i % (D / 4)) * 4, z = z0 + 16 * ct + zz;
        if (z >= s.n * a.rep) continue;
        float M = -INFINITY;
#pragma unroll
        for (int w = 0; w < NW; ++w) M = fmaxf(M, sml[w][0][zz]);
        float L = 0.0f;
        float4 sum = make_float4(0, 0, 0, 0);
        int top = -(1 << 20);  // 4-bit pages: the highest frame of a wave that has seen a key
        if constexpr (Q4) {
#pragma unroll
          for (int w = 0; w < NW; ++w)
            if (sml[w][0][zz] != -INFINITY) top = max(top, frames[w]);
        }
#pragma unroll
        for (int w = 0; w < NW; ++w) {
          const float mw = sml[w][0][zz];
          float e = mw == -INFINITY ? 0.0f : __builtin_amdgcn_exp2f(mw - M);
          const float4 v = *reinterpret_cast<const float4*>(&sm.o[w][zz][d0]);
          L += e * sml[w][1][zz];
          if constexpr (Q4) e = mw == -INFINITY ? 0.0f : __builtin_ldexpf(e, frames[w] - top);
          sum.x += e * v.x;
          sum.y += e * v.y;
          sum.z += e * v.z;
          sum.w += e * v.w;
        }
        // a sum of 0: no key seen (o is 0 then); a wave with NaN scores has a NaN sum, which reaches L
        const float inv = L == 0.0f ? 0.0f : 1.0f / L, ls = M + __log2f(L) - s_lift(P);
        const int64_t n = s.s0 + z / a.rep, head = g * a.rep + z % a.rep;
        sum = make_float4(sum.x * inv, sum.y * inv, sum.z * inv, sum.w * inv);
        if constexpr (Q4) {
          if (top > -(1 << 20))
            sum = make_float4(__builtin_ldexpf(sum.x, top), __builtin_ldexpf(sum.y, top), __builtin_ldexpf(sum.z, top),
                              __builtin_ldexpf(sum.w, top));
        }
        if (nv == 1) {
          put4(a.out + n * a.sot + head * a.soh + d0, sum, lower != 0);
          if (a.lse && d0 == 0) a.lse[n * a.Hq + head] = ls * kLn2;
        } else {
          const int64_t slot = ((int64_t)sp * a.p.N + n) * a.Hq + head;
          put4(a.part + slot * D + d0, sum, lower != 0);
          if (d0 == 0) a.part[(int64_t)a.nsplit * a.p.N * a.Hq * D + slot] = ls;
        }
      }
    }
    lower = Q4 && lower == 0 && __builtin_amdgcn_readfirstlane(over) ? kLower : 0;
    if (lower == 0) z0 += a.tiles * 16 * CT;
  }
}

// The splits of a slot merged by log-sum-exp: 4 columns a thread, S groups of threads share a slot's splits, 4 of them
// in flight in each. One group where there are few splits (chunks: many slots), all of a workgroup where there are many
// (decode steps: few slots; 8 tokens over 32768, 8 splits, 7 us with one group, 4.5 with 8). `width`: keys per tile.
template <int D, int S>
__global__ __launch_bounds__(kThreads) void paged_combine_kernel(AttnArgs a, int width) {
  constexpr int C = D / 4, SL = kThreads / (C * S), AHEAD = 4;
  __shared__ float4 so[SL][S][C];
  __shared__ float sml[SL][S][2];
  const int c = threadIdx.x % C, grp = threadIdx.x / C % S, sl = threadIdx.x / (C * S);
  const int n = blockIdx.x, my = blockIdx.y * SL + sl, head = min(my, a.Hq - 1);  // every lane takes part in the search
  const int64_t slot = (int64_t)n * a.Hq + head, step = (int64_t)a.p.N * a.Hq;
  const float* ls = a.part + (int64_t)a.nsplit * step * D;
  const float* po = a.part + slot * D + 4 * c;
  // The first splits are asked for before their number is known: what no split has written is not used.
  float l4[AHEAD];
  float4 u4[AHEAD];
#pragma unroll
  for (int i = 0; i < AHEAD; ++i) {
    const int64_t sp = min(grp + i * S, a.nsplit - 1);
    l4[i] = ls[sp * step + slot];
    u4[i] = *reinterpret_cast<const float4*>(po + sp * step * D);
  }
  const int b = seq_search(a.p.start, a.p.B, n);
  const Seq s = seq_of(a, b);
  const int nv = splits_of(a, (s.ctx + width - 1) / width);
  if (n < s.s0 || n >= s.s0 + s.n || nv == 1) return;  // uniform over the workgroup
  float M = -INFINITY, L = 0.0f;
  float4 acc = make_float4(0, 0, 0, 0);
  // (parts in units of 2^8: the sum of as many as a call is split into, 128, is finite)
  auto part = [](float4 u) { return make_float4(u.x * 0x1p-8f, u.y * 0x1p-8f, u.z * 0x1p-8f, u.w * 0x1p-8f); };
  auto add = [&](float l, float w, float4 u) {  // w: the weight that comes with l
    const float m2 = fmaxf(M, l), ms = m2 == -INFINITY ? 0.0f : m2;  // a NaN l leaves M and makes the sums NaN
    const float r = __builtin_amdgcn_exp2f(M - ms), f = __builtin_amdgcn_exp2f(l - ms);
    L = L * r + w * f;
    acc = make_float4(acc.x * r + f * u.x, acc.y * r + f * u.y, acc.z * r + f * u.z, acc.w * r + f * u.w);
    M = m2;
  };
#pragma unroll
  for (int i = 0; i < AHEAD; ++i)
    if (grp + i * S < nv) add(l4[i], 1.0f, part(u4[i]));
#pragma unroll 4
  for (int sp = grp + AHEAD * S; sp < nv; sp += S)
    add(ls[sp * step + slot], 1.0f, part(*reinterpret_cast<const float4*>(po + sp * step * D)));
  if constexpr (S > 1) {
    so[sl][grp][c] = acc;
    if (c == 0) {
      sml[sl][grp][0] = M;
      sml[sl][grp][1] = L;
    }
    __syncthreads();
#pragma unroll
    for (int k = 1; k < S; ++k)
      if (grp == 0) add(sml[sl][k][0], sml[sl][k][1], so[sl][k][c]);
  }
  if (grp != 0 || my >= a.Hq) return;
  const float inv = L == 0.0f ? 0.0f : 0x1p8f / L;
  *reinterpret_cast<uint2*>(a.out + n * a.sot + head * a.soh + 4 * c) =
      make_uint2(od_pack_bf16x2(acc.x * inv, acc.y * inv), od_pack_bf16x2(acc.z * inv, acc.w * inv));
  if (a.lse && c == 0) a.lse[slot] = (M + __log2f(L)) * kLn2;
}

// ------------------------------------------------------------------------------------------------ many slots: tiles
// Chunks and option rows: bound by the matrix cores and the softmax's vector work (a chunk of 2048 over 32768 tokens,
// 32 heads of 128, 1130 to 1180 us by the card, 960 to 1000 TFLOP/s, 59 and 47% of the cycles). A workgroup of NW waves owns 32 slots per wave of
// one (sequence, KV head) and goes over 64-key blocks: first the cached ones, then the new tokens'. Scores are taken
// transposed, S^T = K Q^T on 32 x 32 x 16 matrix instructions (64 keys by the wave's 32 slots), so that a slot's
// softmax is lane-local but for one exchange, and the probabilities sit where O^T += V^T P^T wants them; V^T comes from
// row-major LDS by transposing reads. The kernel here is for heads of 64 and 128; heads of 256 have one of their own
// below, of the same parts.
//
// int8 blocks are converted once per workgroup on the way into LDS, or once for all of them ahead (the image, below),
// to fp16 in power-of-two frames: K' = fp16(q ks_j 2^(7 - E)) with 2^E above the block's largest scale, V' = fp16(q
// vs_j 2^(7 - F)) with 2^F above the largest so far (the accumulator moves along when F rises), queries as fp16 q 2^(14
// - e) with 2^e above the slot's largest (exact while they are normal). One rounding of 2^-11 at most for every cached
// value, far below the 2^-8 of their int8 grid, and the scores' factor 2^(e - 14 + E - 7) is one number per slot and
// block. Probabilities are fp16 there, kept 2^7 above what they are (2^15 at most under kSlack), so that one as small
// as 2^-31 of the largest still counts. bf16 pages and the new tokens go in as they are, with bf16 probabilities (2^-8
// each, as the output's own rounding).
//
// The next block's loads are in flight during a block's products; its conversion into the other LDS buffer comes first
// in the next step. Cached keys behind the last one, and pages that are none, enter as zeros with masked scores.
constexpr int kBK = 64;

// K rows in LDS: 16-byte chunks XORed so that 16 rows hit 16 bank groups
template <int D>
__device__ __forceinline__ int tk_off(int key, int chunk) {
  return key * D + ((chunk ^ (D == 64 ? ((key >> 1) & 7) : (key & 15))) << 3);
}
// V rows: 4 consecutive keys' chunks of a transposing read 64 bytes apart
template <int D>
__device__ __forceinline__ int tv_chunk(int key, int chunk) {
  return D == 64 ? chunk ^ ((key & 2) << 1) : chunk ^ ((key & 3) << 2);
}

__device__ __forceinline__ void dma_wait() { asm volatile("s_waitcnt vmcnt(0)" ::: "memory"); }
// A block's bf16 rows into LDS by DMA: instruction i of a wave fills the 1 KB at 1024 (i NW + wave) of K or V, so a
// lane owns a place there, (key, swizzled chunk), and copies the chunk that the swizzle puts into it. at(key): its row.
template <int D, int NW, typename KeyRow>
__device__ __forceinline__ void dma_rows(const uint16_t* lds, int wave, bool v, KeyRow&& row) {
  int lane = threadIdx.x & 63;
  // places are formed here each time, not kept in registers over the block loop
  if constexpr (D > 64) asm volatile("" : "+v"(lane));
#pragma unroll
  for (int i = 0; i < D / (8 * NW); ++i) {
    const int pe = (i * NW + wave) * 512 + 8 * lane, key = pe / D, slot = pe % D / 8;
    const int ch = v ? tv_chunk<D>(key, slot) : slot ^ (D == 64 ? ((key >> 1) & 7) : (key & 15));
    od_dma16(row(key) + 8 * ch, od_lds_addr(lds) + 1024 * (i * NW + wave));
  }
}

// A block's bf16 rows from the pages; lane l has the page of key l. An instruction's 1 KB is 512 / D keys, which never
// cross a page, so its address is one of the wave.
template <int D, int NW>
__device__ __forceinline__ void dma_pages(const uint16_t* lds, int wave, bool v, const Paged& p, int g, int blk,
    int pg) {
  int lane = threadIdx.x & 63;
  if constexpr (D > 64) asm volatile("" : "+v"(lane));
  const uint16_t* pool = static_cast<const uint16_t*>(v ? p.v : p.k);
#pragma unroll
  for (int i = 0; i < D / (8 * NW); ++i) {
    const int first = (i * NW + wave) * (512 / D), page = max(__builtin_amdgcn_readlane(pg, first), 0);
    const int64_t row = (((int64_t)page * p.Hkv + g) << p.shift) + ((blk * kBK + first) & ((1 << p.shift) - 1));
    const int key = lane / (D / 8), slot = lane % (D / 8);
    const int ch = v ? tv_chunk<D>(first + key, slot)
                     : slot ^ (D == 64 ? (((first + key) >> 1) & 7) : ((first + key) & 15));
    od_dma16_at(pool + row * D, 2 * (key * D + 8 * ch), od_lds_addr(lds) + 1024 * (i * NW + wave));
  }
}
// The same from a block of the image, which lies in memory as it does in LDS.
template <int D, int NW>
__device__ __forceinline__ void dma_block(const uint16_t* lds, int wave, const uint16_t* src) {
#pragma unroll
  for (int i = 0; i < D / (8 * NW); ++i)
    od_dma16_at(src + (i * NW + wave) * 512, 16 * (threadIdx.x & 63), od_lds_addr(lds) + 1024 * (i * NW + wave));
}

template <bool H>
__device__ __forceinline__ v16f mfma32(v4u a, v4u b, v16f c) {
  if constexpr (H)
    return __builtin_amdgcn_mfma_f32_32x32x16_f16(__builtin_bit_cast(f16x8, a), __builtin_bit_cast(f16x8, b), c, 0,
                                                  0, 0);
  else
    return __builtin_amdgcn_mfma_f32_32x32x16_bf16(__builtin_bit_cast(bf16x8, a), __builtin_bit_cast(bf16x8, b), c,
                                                   0, 0, 0);
}
__device__ __forceinline__ v16f zero16() { return v16f{0, 0, 0, 0, 0, 0, 0, 0, 0, 0, 0, 0, 0, 0, 0, 0}; }

// 16 int8 times f, each product rounded once to fp16: byte u = q + 128 becomes the fp16 1024 + u by its bits, and (1024
// + u) f - 1152 f is one fp32 fma per value (v_fma_mix). f has its last 4 bits clear (frame_scale), so that 1152 f is
// exact and the result is q f rounded once, 0 for q = 0.
__device__ __forceinline__ void i8x16_scaled(v4u w, float f, v4u& lo, v4u& hi) {
  const float c = -1152.0f * f;
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const uint32_t u = w[i] ^ 0x80808080u;
#pragma unroll
    for (int k = 0; k < 2; ++k) {
      const f16x2 h = __builtin_bit_cast(f16x2, __builtin_amdgcn_perm(0x64646464u, u, k ? 0x04030402u : 0x04010400u));
      const f16x2 r = {(_Float16)__builtin_fmaf((float)h.x, f, c), (_Float16)__builtin_fmaf((float)h.y, f, c)};
      (i < 2 ? lo : hi)[2 * (i & 1) + k] = __builtin_bit_cast(uint32_t, r);
    }
  }
}

// s 2^e with 20 significant bits: within 2^-20 of it
__device__ __forceinline__ float frame_scale(float s, int e) {
  return __uint_as_float(__float_as_uint(__builtin_ldexpf(s, e)) & ~15u);
}

// The largest magnitude of the finite ones of N packed pairs of bf16 scales, as bits.
template <int N>
__device__ __forceinline__ uint32_t q4_largest(const uint32_t (&w)[N]) {
  uint32_t m = 0;
#pragma unroll
  for (int i = 0; i < N; ++i) m = od_absmax_bf16x2(m, fin_bf16x2(w[i]));
  return max(m & 0xffffu, m >> 16);
}
// The D / 32 scales of a row.
template <int D>
__device__ __forceinline__ void q4_row_scales(const uint16_t* scales, int64_t row, uint32_t (&w)[D / 64]) {
  const uint16_t* at = scales + row * (D / 32);
  if constexpr (D == 64) {
    w[0] = *reinterpret_cast<const uint32_t*>(at);
  } else if constexpr (D == 128) {
    const uint2 u = *reinterpret_cast<const uint2*>(at);
    w[0] = u.x, w[1] = u.y;
  } else {
    const uint4 u = *reinterpret_cast<const uint4*>(at);
    w[0] = u.x, w[1] = u.y, w[2] = u.z, w[3] = u.w;
  }
}
// A block of 32 values (16 bytes, block c of key `key`) into the places of a tile's K or V.
template <int D>
__device__ __forceinline__ void q4_put(uint16_t* dst, bool v, int key, int c, const v4u& r, _Float16 s) {
  const Q4Scale q = q4_pair(f16x2{s, s});
  const uint32_t sixteen = q4_sixteen();
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const int ch = 4 * c + i, at = v ? key * D + (tv_chunk<D>(key, ch) << 3) : tk_off<D>(key, ch);
    *reinterpret_cast<uint4*>(dst + at) = __builtin_bit_cast(uint4, q4x8_f16(r[i], q, sixteen));
  }
}

template <int D, int NW>
struct alignas(16) TSmem {
  uint16_t k[2][kBK * D];
  uint16_t v[2][kBK * D];
  int lo[NW], hi[NW];
  int over;  // a slot's O is not finite
  int odd;  // infinities or NaN among the new values of a block that some slot sees only a part of
};

// Value tiles of 32 columns that a wave accumulates (D = 256: half of the columns).
constexpr int t_cols(int D) { return D == 256 ? 4 : D / 32; }
// One slot tile's constants per lane, and its state.
template <int D>
struct TSlot {
  int ok, tok, head, begin;  // the slot exists; its token and head; the first new token that it sees
  v4u q[D / 16];             // dims 16 ks + 8 h .. + 7
  int qe;                    // fp16 queries: their exponent
  float m, l;
  v16f o[t_cols(D)];
};

template <int D>
__device__ __forceinline__ void t_load_q(const AttnArgs& a, const Seq& s, TSlot<D>& t) {
  const int h = (threadIdx.x & 63) >> 5;
  const uint16_t* qp = a.q + (int64_t)(s.s0 + t.tok) * a.sqt + (int64_t)t.head * a.sqh + 8 * h;
#pragma unroll
  for (int ks = 0; ks < D / 16; ++ks)
    t.q[ks] = t.ok ? __builtin_bit_cast(v4u, *reinterpret_cast<const uint4*>(qp + 16 * ks)) : v4u{0, 0, 0, 0};
}
// the queries as fp16 in the slot's frame
template <int D>
__device__ __forceinline__ void t_q_to_f16(TSlot<D>& t) {
  uint32_t am = 0;
#pragma unroll
  for (int ks = 0; ks < D / 16; ++ks)
#pragma unroll
    for (int i = 0; i < 4; ++i) am = od_absmax_bf16x2(am, t.q[ks][i]);
  const float mx = od_xor32_max(od_absmax_bf16x2_value(am));
  t.qe = mx < INFINITY ? exp_above(__float_as_uint(mx)) : 0;
#pragma unroll
  for (int ks = 0; ks < D / 16; ++ks)
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const uint32_t w = t.q[ks][i];
      const f16x2 r = {(_Float16)__builtin_ldexpf(__uint_as_float(w << 16), 14 - t.qe),
                       (_Float16)__builtin_ldexpf(__uint_as_float(w & 0xffff0000u), 14 - t.qe)};
      t.q[ks][i] = __builtin_bit_cast(uint32_t, r);
    }
}

// S^T of one block.
template <int D, bool H>
__device__ __forceinline__ void t_scores(const uint16_t* kb, const TSlot<D>& t, v16f (&s)[2]) {
  const int lane = threadIdx.x & 63, h = lane >> 5, col = lane & 31;
  constexpr int NQ = D / 16 * 2, RA = 2;  // MFMA i: k-step i / 2, key tile i % 2; reads run RA ahead
  int place = tk_off<D>(col, h);
  asm volatile("" : "+v"(place));  // the places are formed here each time, not kept in registers
  s[0] = zero16();
  s[1] = zero16();
  v4u kf[RA + 1];
  auto rd = [&](int i) {
    const uint16_t* at = &kb[(place ^ (i / 2 << 4)) + (i % 2) * 32 * D];  // tk_off<D>(key, 2 (i / 2) + h)
    kf[i % (RA + 1)] = __builtin_bit_cast(v4u, *reinterpret_cast<const uint4*>(at));
  };
#pragma unroll
  for (int i = 0; i < RA; ++i) rd(i);
#pragma unroll
  for (int i = 0; i < NQ; ++i) {
    if (i + RA < NQ) rd(i + RA);
    s[i % 2] = mfma32<H>(kf[i % (RA + 1)], t.q[i / 2], s[i % 2]);
  }
  __builtin_amdgcn_sched_group_barrier(0x100, RA, 0);
#pragma unroll
  for (int i = 0; i < NQ; ++i) {
    if (i + RA < NQ) __builtin_amdgcn_sched_group_barrier(0x100, 1, 0);
    __builtin_amdgcn_sched_group_barrier(0x008, 1, 0);
  }
}

// The block's online softmax into P; c > 0: the scores' factor (log2 units), masked scores -inf.
template <int D, bool H>
__device__ __forceinline__ void t_softmax(v16f (&s)[2], float c, TSlot<D>& t, v4u (&pb)[4]) {
  float mx = -INFINITY;
#pragma unroll
  for (int kt = 0; kt < 2; ++kt)
#pragma unroll
    for (int r = 0; r < 16; ++r) mx = fmaxf(mx, s[kt][r]);
  mx = od_xor32_max(mx) * c;
  const bool move = mx > t.m + kSlack;
  if (__builtin_amdgcn_ballot_w64(move) != 0) {
    const float f = move ? __builtin_amdgcn_exp2f(t.m - mx) : 1.0f;  // m = -inf: 0
#pragma unroll
    for (auto& o : t.o)
#pragma unroll
      for (int r = 0; r < 16; ++r) o[r] *= f;
    t.l *= f;
    if (move) t.m = mx;
  }
  const float ms = (t.m == -INFINITY ? 0.0f : t.m) - kLift;
  float sum = 0.0f;
#pragma unroll
  for (int kt = 0; kt < 2; ++kt)
#pragma unroll
    for (int r = 0; r < 16; r += 2) {
      const float p0 = __builtin_amdgcn_exp2f(__builtin_fmaf(s[kt][r], c, -ms));
      const float p1 = __builtin_amdgcn_exp2f(__builtin_fmaf(s[kt][r + 1], c, -ms));
      sum += p0;
      sum += p1;
      if constexpr (H) {
        const f16x2 w = {(_Float16)p0, (_Float16)p1};
        pb[kt * 2 + (r >> 3)][(r & 7) >> 1] = __builtin_bit_cast(uint32_t, w);
      } else {
        pb[kt * 2 + (r >> 3)][(r & 7) >> 1] = od_pack_bf16x2(p0, p1);
      }
    }
  t.l += sum;  // this lane's share: keys of its half
}

// The A operand for value rows of d tile dt (vb: the lane's base there), keys 16 kk + 8 (i / 4) + 4 (lane / 32) + i %
// 4.
template <int D>
__device__ __forceinline__ v4u t_vfrag(const uint16_t* vblk, int vb, int kk) {
  typedef short v4s __attribute__((ext_vector_type(4)));
  typedef __attribute__((address_space(3))) v4s lds_v4s;
  uint16_t* base = const_cast<uint16_t*>(vblk) + vb + kk * 16 * D;
  const v4s lo = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_v4s*)base);
  const v4s hi = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_v4s*)(base + 8 * D));
  return __builtin_bit_cast(v4u, __builtin_shufflevector(lo, hi, 0, 1, 2, 3, 4, 5, 6, 7));
}

template <int D, bool H>
__device__ __forceinline__ void t_values(const uint16_t* vblk, const int (&vb)[t_cols(D)], const v4u (&pb)[4],
    TSlot<D>& t) {
  constexpr int DT = t_cols(D), NV = 4 * DT, RA = D == 256 ? 1 : 2;  // MFMA i: k-step i / DT, d tile i % DT
  v4u vf[RA + 1];
  auto rd = [&](int i) { vf[i % (RA + 1)] = t_vfrag<D>(vblk, vb[i % DT], i / DT); };
#pragma unroll
  for (int i = 0; i < RA; ++i) rd(i);
#pragma unroll
  for (int i = 0; i < NV; ++i) {
    if (i + RA < NV) rd(i + RA);
    t.o[i % DT] = mfma32<H>(vf[i % (RA + 1)], pb[i / DT], t.o[i % DT]);
  }
  __builtin_amdgcn_sched_group_barrier(0x100, RA * 2, 0);
#pragma unroll
  for (int i = 0; i < NV; ++i) {
    if (i + RA < NV) __builtin_amdgcn_sched_group_barrier(0x100, 2, 0);
    __builtin_amdgcn_sched_group_barrier(0x008, 1, 0);
  }
}
// Where a workgroup's work lies (sp < 0: nowhere). Workgroups are dealt round-robin over the 8 XCDs, each with an L2 of
// its own. A group is the slot tiles of one (sequence, KV head, split), which read the same keys; its tiles go to one
// XCD in runs of `run` (a whole group, or a part of it where there are few groups), and the runs are dealt round-robin,
// each turn of 8 shifted by 3 against the last (else the first of two sequences of 4 heads, or every first split, would
// stay with half of the XCDs): contiguous ranges of the groups gave each XCD the sequences of a ragged batch as they
// came (4 ragged chunks of 256-wide heads 618 us, so 446). A causal tile's work grows with its index: last first (both:
// 4 ragged first chunks of 2000, 199 us, 124). Of up to 64 sequences the longest come first, so that the last
// workgroups to run are short ones (option rows of 8 ragged requests 158 us, 140).
struct TilePlace {
  int b, g, sp, tile;
};
__device__ __forceinline__ TilePlace tile_place(const AttnArgs& a) {
  const int xcd = blockIdx.x & 7, loc = blockIdx.x >> 3, runs = (a.tiles + a.run - 1) / a.run, turn = loc / a.run;
  const int rid = turn * 8 + ((xcd + 3 * turn) & 7), pairs = a.p.B * a.p.Hkv, pair = rid / runs % pairs;
  TilePlace w;
  w.tile = a.tiles - 1 - (rid % runs * a.run + loc % a.run);
  w.sp = rid / runs / pairs;
  w.g = pair % a.p.Hkv;
  w.b = pair / a.p.Hkv;
  if (w.tile < 0 || w.sp >= a.nsplit) w.sp = -1;
  if (a.p.B > 1 && a.p.B <= 64) {  // the place among the sequences, longest first -> the sequence
    const int lane = threadIdx.x & 63;
    int64_t size = -1;
    if (lane < a.p.B) size = (int64_t)max(a.p.ctx[lane], 0) + a.p.start[lane + 1] - a.p.start[lane];
    const int key = (int)min(max(size, (int64_t)0), (int64_t)0x7fffffff);
    int ahead = 0;
    for (int i = 0; i < a.p.B; ++i) {
      const int other = __builtin_amdgcn_readlane(key, i);
      ahead += other > key || (other == key && i < lane);
    }
    w.b = __builtin_ctzll(__builtin_amdgcn_ballot_w64(lane < a.p.B && ahead == w.b));
  }
  return w;
}

// The new tokens that a slot tile sees: blocks lo .. hi - 1 of them. Of the wave's slots (w_) and the workgroup's (g_):
// the first and last token that any sees (w_lo, w_hi), and the span that all see whole, w_in .. w_tok.
struct NewSpan {
  int lo, hi, w_lo, w_hi, w_in, w_tok, g_in, g_tok;
  // a block that some slot of the workgroup sees only a part of
  __device__ __forceinline__ bool partial(int blk) const { return blk * kBK + kBK - 1 > g_tok || blk * kBK < g_in; }
};
template <int D>
__device__ __forceinline__ NewSpan new_span(const AttnArgs& a, const Seq& s, int tile, int spt, int zw, bool live,
                                            const TSlot<D>& t, int* lo, int* hi, int* odd, int nw, int wave) {
  const int lane = threadIdx.x & 63;
  NewSpan n;
  n.w_tok = min(zw / a.rep, s.n - 1);
  n.w_hi = min((zw + 31) / a.rep, s.n - 1);
  n.w_lo = n.w_in = 0;
  if (a.row_begin) {
    n.w_lo = t.ok ? t.begin : 0x7fffffff;
    n.w_in = t.begin;
#pragma unroll
    for (int o = 32; o > 0; o >>= 1) {
      n.w_lo = min(n.w_lo, __shfl_xor(n.w_lo, o, 64));
      n.w_in = max(n.w_in, __shfl_xor(n.w_in, o, 64));
    }
  }
  n.w_lo = __builtin_amdgcn_readfirstlane(n.w_lo);
  n.w_in = __builtin_amdgcn_readfirstlane(n.w_in);
  if (threadIdx.x == 0) *odd = 0;
  if (lane == 0) {
    lo[wave] = live ? n.w_lo : 0x7fffffff;
    hi[wave] = live ? n.w_in : 0;
  }
  __syncthreads();
  int g_lo = 0x7fffffff;
  n.g_in = 0;
  for (int i = 0; i < nw; ++i) {
    g_lo = min(g_lo, lo[i]);
    n.g_in = max(n.g_in, hi[i]);
  }
  n.g_tok = min(tile * spt / a.rep, s.n - 1);
  const int g_hi = min((tile * spt + spt - 1) / a.rep, s.n - 1);
  n.lo = min(g_lo, g_hi + 1) / kBK;
  n.hi = g_hi / kBK + 1;
  return n;
}
// A partly seen block's infinities and NaN become 0 (0 times one would reach the slots that do not see it) ...
template <int D, int NT>
__device__ __forceinline__ void make_finite(uint16_t* v, int* odd) {
  for (int c = threadIdx.x; c < kBK * (D / 8); c += NT) {
    uint4* at = reinterpret_cast<uint4*>(&v[8 * c]);
    const v4u x = __builtin_bit_cast(v4u, *at);
    if (any_inf_bf16x8(x)) {
      *at = __builtin_bit_cast(uint4, fin_bf16x8(x));
      *odd = 1;
    }
  }
}
// ... and the slots that see one get it added.
template <int D>
__device__ __forceinline__ void add_odd(const AttnArgs& a, const Seq& s, int g, int half, const NewSpan& n,
    TSlot<D>& t) {
  const int h = (threadIdx.x & 63) >> 5;
#pragma unroll 1
  for (int key = max(n.lo * kBK, t.begin); key <= t.tok; ++key) {
    if (!n.partial(key / kBK)) continue;
    const uint16_t* vp = a.v + (int64_t)(s.s0 + key) * a.svt + (int64_t)g * a.svh + half * 128 + 4 * h;
#pragma unroll
    for (int dt = 0; dt < t_cols(D); ++dt)
#pragma unroll
      for (int i = 0; i < 16; ++i) t.o[dt][i] += odd_bf16(vp[dt * 32 + 8 * (i >> 2) + (i & 3)]);
  }
}
// out = O / l, or the split's normalized partial (again: as put4); lane: slot col, value rows 32 dt + 8 (i / 4) + 4 h + i % 4
template <int D>
__device__ __forceinline__ void t_out(const AttnArgs& a, const Seq& s, const TSlot<D>& t, float l, int frame, int sp,
    int nv, int half, bool again) {
  if (!t.ok) return;
  const int h = (threadIdx.x & 63) >> 5;
  // 2^frame may be subnormal, so it comes last
  const float inv = l == 0.0f ? 0.0f : 1.0f / l, unit = __builtin_ldexpf(1.0f, frame), ls = t.m + __log2f(l) - kLift;
  const int64_t n = s.s0 + t.tok;
#pragma unroll
  for (int dt = 0; dt < t_cols(D); ++dt)
#pragma unroll
    for (int i4 = 0; i4 < 4; ++i4) {
      const int d0 = half * 128 + dt * 32 + 8 * i4 + 4 * h;
      const float4 y = make_float4(t.o[dt][4 * i4] * inv * unit, t.o[dt][4 * i4 + 1] * inv * unit,
          t.o[dt][4 * i4 + 2] * inv * unit, t.o[dt][4 * i4 + 3] * inv * unit);
      if (nv == 1)
        put4(a.out + n * a.sot + t.head * a.soh + d0, y, again);
      else
        put4(a.part + (((int64_t)sp * a.p.N + n) * a.Hq + t.head) * D + d0, y, again);
    }
  if (h == 0 && half == 0) {
    if (nv > 1) a.part[(int64_t)a.nsplit * a.p.N * a.Hq * D + ((int64_t)sp * a.p.N + n) * a.Hq + t.head] = ls;
    else if (a.lse) a.lse[n * a.Hq + t.head] = ls * kLn2;
  }
}

// A block's bf16 values times 2^-kLower. (A thread takes the chunks that it does in make_finite.)
template <int D, int NT>
__device__ __forceinline__ void t_lower(uint16_t* v) {
  for (int c = threadIdx.x; c < kBK * (D / 8); c += NT) {
    uint4* at = reinterpret_cast<uint4*>(&v[8 * c]);
    const uint4 x = *at;
    *at = make_uint4(lower_bf16x2(x.x), lower_bf16x2(x.y), lower_bf16x2(x.z), lower_bf16x2(x.w));
  }
}
// Whether an O is infinite or NaN, after bf16 values (kLower).
template <int D>
__device__ __forceinline__ bool t_over(const TSlot<D>& t) {
  v4f x = v4f{0, 0, 0, 0};
#pragma unroll
  for (int dt = 0; dt < t_cols(D); ++dt)
#pragma unroll
    for (int i = 0; i < 16; ++i) x[i & 3] = __builtin_fmaf(t.o[dt][i], 0.0f, x[i & 3]);
  return t.ok && x[0] + x[1] + x[2] + x[3] != 0.0f;
}

// Waves a SIMD: heads of 64 leave the registers for three, but for the conversion of int8 and 4-bit blocks.
constexpr int t_waves(int D, int src) { return D == 64 && (src == kBf16 || src == kImage) ? 3 : 2; }
template <int D, int SRC, int NW>
__global__ __launch_bounds__(NW * 64, t_waves(D, SRC)) void paged_tile_kernel(AttnArgs a) {
  // REG: blocks that are converted on their way, through registers
  constexpr bool Q4 = SRC == kInt4, REG = SRC == kInt8 || Q4, IMG = SRC == kImage, H16 = SRC != kBf16;
  constexpr int NT = NW * 64, SPT = 32 * NW, DT = D / 32;
  extern __shared__ __attribute__((aligned(16))) char smem_raw[];
  TSmem<D, NW>& sm = *reinterpret_cast<TSmem<D, NW>*>(smem_raw);
  const TilePlace at = tile_place(a);
  if (at.sp < 0) return;
  const int sp = at.sp, g = at.g, b = at.b;
  const Seq s = seq_of(a, b);
  const int nslots = s.n * a.rep, blocks = (s.ctx + kBK - 1) / kBK, nv = splits_of(a, blocks);
  if (sp >= nv || (IMG ? blocks > a.img_blocks : a.rest && blocks <= a.img_blocks)) return;
  const int b_lo = sp * a.chunk, b_hi = sp == a.nsplit - 1 ? blocks : min(blocks, b_lo + a.chunk);
  const int tid = threadIdx.x, lane = tid & 63, h = lane >> 5, col = lane & 31;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  int vb[DT];  // transposing-read bases
  {
    const int hh = lane >> 5, mh = (lane >> 4) & 1, e = (lane >> 2) & 3, c = lane & 3;
#pragma unroll
    for (int dt = 0; dt < DT; ++dt)
      vb[dt] = (4 * hh + e) * D + (tv_chunk<D>(e, 4 * dt + 2 * mh + (c >> 1)) << 3) + 4 * (c & 1);
  }

  int lower = 0;  // the power of two that bf16 values are lowered by
  for (int tile = at.tile; tile * SPT < nslots;) {
    __syncthreads();  // an earlier tile's readers are done
    if (tid == 0) sm.over = 0;
    TSlot<D> t;
    const int zw = tile * SPT + wave * 32, z = zw + col;
    const bool live = zw < nslots;  // the wave has slots
    t.ok = z < nslots;
    t.tok = t.ok ? z / a.rep : s.n - 1;
    t.head = g * a.rep + (t.ok ? z % a.rep : 0);
    t.begin = a.row_begin && t.ok ? max(a.row_begin[s.s0 + t.tok], 0) : 0;
    t.m = -INFINITY;
    t.l = 0.0f;
    t.qe = 0;
#pragma unroll
    for (auto& o : t.o) o = zero16();
    t_load_q<D>(a, s, t);
    int frame = H16 ? 0 : lower;  // O is in units of 2^frame

    // ---- the cached blocks b_lo .. b_hi - 1
    if (b_lo < b_hi) {
      if constexpr (H16) t_q_to_f16<D>(t);
      const int64_t first = ((int64_t)b * a.p.Hkv + g) * a.img_blocks;  // image: the sequence's first block
      if constexpr (IMG) frame = a.img_vexp[b * a.p.Hkv + g] - 7;
      // int8 and 4-bit blocks pass through registers, NC 16-byte chunks per thread, K's first; bf16 ones go by DMA
      constexpr int CPK = D / (Q4 ? 32 : 16), CH = kBK * CPK, NC = 2 * CH / NT;
      v4u r[REG ? NC : 1];
      uint32_t rs[Q4 ? NC : 1];         // 4 bits: the scales of the chunks
      uint32_t ks4 = 0, vs4 = 0;        // 4 bits, lane l: the largest scales of key l of the loaded block
      int pg = -1;             // lane l: the page of key l of the block whose loads come next
      float ks = 0, vs = 0;    // lane l: the scales of key l of the loaded block
      uint64_t there = 0;      // the loaded block's keys that exist
      const int in_page = (1 << a.p.shift) - 1;
      int first_lane = lane;  // (so that the first blocks' places are not kept in registers from tile to tile)
      if constexpr (REG) asm volatile("" : "+v"(first_lane));
      auto pages = [&](int blk, int l) {
        if constexpr (IMG) return;
        const int pos = blk * kBK + l;
        pg = pos < s.ctx ? a.p.table[b * a.p.ld_table + (pos >> a.p.shift)] : -1;
        if (pg >= a.p.n_pages) pg = -1;
      };
      int kexp_in = 0;  // image: the loaded block's frame
      auto load = [&](int blk, int buf) {
        if constexpr (IMG) {
          const uint16_t* src = a.img + (first + blk) * (2 * kBK * D);
          dma_block<D, NW>(sm.k[buf], wave, src);
          dma_block<D, NW>(sm.v[buf], wave, src + kBK * D);
          there = a.img_heads[first + blk].seen;
          kexp_in = a.img_heads[first + blk].kexp;
          return;
        }
        there = __builtin_amdgcn_ballot_w64(pg >= 0);
        const int page = max(pg, 0);  // a key that is not there is read from page 0 and left out later
        auto row = [&](int key) {
          return (((int64_t)__shfl(page, key, 64) * a.p.Hkv + g) << a.p.shift) + ((blk * kBK + key) & in_page);
        };
        if constexpr (REG) {
          const int64_t at = (((int64_t)page * a.p.Hkv + g) << a.p.shift) + ((blk * kBK + lane) & in_page);
          if constexpr (Q4) {
            uint32_t w[D / 64];
            q4_row_scales<D>(a.p.k4, at, w);
            ks4 = q4_largest(w);
            q4_row_scales<D>(a.p.v4, at, w);
            vs4 = q4_largest(w);
          } else {
            ks = a.p.ks[at];
            vs = a.p.vs[at];
          }
#pragma unroll
          for (int i = 0; i < NC; ++i) {
            const int cid = i * NT + tid, side = cid / CH, key = cid % CH / CPK, ch = cid % CPK;
            const char* pool = static_cast<const char*>(side ? a.p.v : a.p.k);
            const int64_t from = row(key);
            r[i] = __builtin_bit_cast(v4u, *reinterpret_cast<const uint4*>(pool + from * (16 * CPK) + 16 * ch));
            if constexpr (Q4) rs[i] = (side ? a.p.v4 : a.p.k4)[from * CPK + ch];
          }
        } else {
          dma_pages<D, NW>(sm.k[buf], wave, false, a.p, g, blk, pg);
          dma_pages<D, NW>(sm.v[buf], wave, true, a.p, g, blk, pg);
        }
      };
      int kexp = 0, vexp = 0;  // the stored block's frames
      bool vexp_set = false;
      uint64_t seen = 0;
      auto store = [&](int buf) {
        seen = there;
        if constexpr (IMG) {
          kexp = kexp_in;
        } else if constexpr (Q4) {
          const bool on = (there >> lane) & 1;
          kexp = q4_frame(od_wave_umax_dpp(on ? ks4 : 0u));
          const uint32_t vm = od_wave_umax_dpp(on ? vs4 : 0u);
          if (vm) vexp = vexp_set ? max(vexp, q4_frame(vm)) : q4_frame(vm);
          if (vm) vexp_set = true;
#pragma unroll
          for (int i = 0; i < NC; ++i) {
            const int cid = i * NT + tid, side = cid / CH, key = cid % CH / CPK, ch = cid % CPK;
            const _Float16 sc = f16_scale((there >> key) & 1 ? rs[i] : 0u, 7 - (side ? vexp : kexp));
            q4_put<D>(side ? sm.v[buf] : sm.k[buf], side, key, ch, r[i], sc);
          }
        } else if constexpr (REG) {
          // every wave takes the block's frames from the same 64 scales; keys that are none, and scales that are not
          // finite, leave them alone
          const bool on = (there >> lane) & 1;
          const uint32_t kb = on && ks < INFINITY && ks > 0 ? __float_as_uint(ks) : 0u,
              vb2 = on && vs < INFINITY && vs > 0 ? __float_as_uint(vs) : 0u;
          kexp = exp_above(od_wave_umax_dpp(kb));
          const uint32_t vm = od_wave_umax_dpp(vb2);
          if (vm) vexp = vexp_set ? max(vexp, exp_above(vm)) : exp_above(vm);
          if (vm) vexp_set = true;
          const float kf = on ? frame_scale(ks, 7 - kexp) : 0.0f, vf = on ? frame_scale(vs, 7 - vexp) : 0.0f;
#pragma unroll
          for (int i = 0; i < NC; ++i) {
            const int cid = i * NT + tid, side = cid / CH, key = cid % CH / CPK, ch = cid % CPK;
            uint16_t* dst = side ? sm.v[buf] : sm.k[buf];
            v4u lo, hi;
            i8x16_scaled(r[i], __shfl(side ? vf : kf, key, 64), lo, hi);
            const int o0 = side ? key * D + (tv_chunk<D>(key, 2 * ch) << 3) : tk_off<D>(key, 2 * ch);
            const int o1 = side ? key * D + (tv_chunk<D>(key, 2 * ch + 1) << 3) : tk_off<D>(key, 2 * ch + 1);
            *reinterpret_cast<uint4*>(dst + o0) = __builtin_bit_cast(uint4, lo);
            *reinterpret_cast<uint4*>(dst + o1) = __builtin_bit_cast(uint4, hi);
          }
        } else if (seen != ~0ull || lower) {  // values of keys that are not there: 0 (their scores are masked)
          dma_wait();
          __syncthreads();
          for (int c = tid; c < kBK * (D / 8); c += NT)
            if (!((seen >> (c / (D / 8))) & 1)) *reinterpret_cast<uint4*>(&sm.v[buf][8 * c]) = make_uint4(0, 0, 0, 0);
          if (lower) t_lower<D, NT>(sm.v[buf]);
        }
      };
      // One step: block blk's products; ahead of them, for int8 and 4 bits the conversion of block blk + 1 (in registers since the
      // last step) and the loads of blk + 2, for bf16 the copy of blk + 1.
      pages(b_lo, first_lane);
      load(b_lo, 0);
      pages(b_lo + 1, first_lane);
      if constexpr (!REG) dma_wait();
      store(0);
      if constexpr (REG) frame = vexp - 7;  // O is 0 still: no rescaling, by what may be no fp32 number
      if (REG && b_lo + 1 < b_hi) {
        load(b_lo + 1, 1);
        pages(b_lo + 2, first_lane);
      }
      __syncthreads();
      for (int blk = b_lo; blk < b_hi; ++blk) {
        const int cur = (blk - b_lo) & 1;
        const float c = H16 ? score_factor(a.scale_log2, t.qe - 14 + kexp - 7) : a.scale_log2;
        const int f_new = REG ? vexp - 7 : 0;
        const uint64_t mask = seen;
        if (blk + 1 < b_hi) {
          if constexpr (REG) {
            store(cur ^ 1);
            if (blk + 2 < b_hi) {
              load(blk + 2, cur);
              pages(blk + 3, lane);
            }
          } else {
            load(blk + 1, cur ^ 1);
            pages(blk + 2, lane);
          }
        }
        if (REG && f_new != frame) {  // the values' frame rose: uniform over the workgroup
          // (or is the first one, and may lie lower by any amount: O is 0 still, or NaN)
          const float f = __builtin_ldexpf(1.0f, min(frame - f_new, 0));
#pragma unroll
          for (auto& o : t.o)
#pragma unroll
            for (int i = 0; i < 16; ++i) o[i] *= f;
          frame = f_new;
        }
        if (live) {
          v16f sc[2];
          v4u pb[4];
          t_scores<D, H16>(sm.k[cur], t, sc);
          if (mask != ~0ull) {
            const uint64_t m4 = mask >> (4 * h);
#pragma unroll
            for (int kt = 0; kt < 2; ++kt)
#pragma unroll
              for (int i = 0; i < 16; ++i)
                if (!((m4 >> (kt * 32 + 8 * (i >> 2) + (i & 3))) & 1)) sc[kt][i] = -INFINITY;
          }
          t_softmax<D, H16>(sc, c, t, pb);
          t_values<D, H16>(sm.v[cur], vb, pb, t);
        }
        if (!REG && blk + 1 < b_hi) {
          dma_wait();
          store(cur ^ 1);
        }
        __syncthreads();
      }
    }

    // ---- the new tokens, in split 0
    if (sp == 0 && a.k) {
      if (H16 && b_lo < b_hi) {  // back to bf16 queries and values as they are
        t_load_q<D>(a, s, t);
        if (frame != lower) {
          const float f = __builtin_ldexpf(1.0f, frame - lower);
#pragma unroll
          for (auto& o : t.o)
#pragma unroll
            for (int i = 0; i < 16; ++i) o[i] *= f;
        }
      }
      frame = lower;
      const NewSpan n = new_span(a, s, tile, SPT, zw, live, t, sm.lo, sm.hi, &sm.odd, NW, wave);
      auto load = [&](int blk, int buf) {
        const uint16_t* kp = a.k + (int64_t)s.s0 * a.skt + (int64_t)g * a.skh;
        const uint16_t* vp = a.v + (int64_t)s.s0 * a.svt + (int64_t)g * a.svh;
        dma_rows<D, NW>(sm.k[buf], wave, false, [&](int key) { return kp + min(blk * kBK + key, s.n - 1) * a.skt; });
        dma_rows<D, NW>(sm.v[buf], wave, true, [&](int key) { return vp + min(blk * kBK + key, s.n - 1) * a.svt; });
      };
      auto finite = [&](int blk, int buf) {
        if (!n.partial(blk) && !lower) return;
        __syncthreads();  // every wave's part of the copy is there
        if (n.partial(blk)) make_finite<D, NT>(sm.v[buf], &sm.odd);
        if (lower) t_lower<D, NT>(sm.v[buf]);
      };
      if (n.lo < n.hi) {
        load(n.lo, 0);
        dma_wait();
        finite(n.lo, 0);
        __syncthreads();
        for (int blk = n.lo; blk < n.hi; ++blk) {
          const int cur = (blk - n.lo) & 1, j0 = blk * kBK;
          if (blk + 1 < n.hi) load(blk + 1, cur ^ 1);
          if (live && j0 <= n.w_hi && j0 + kBK > n.w_lo) {
            v16f sc[2];
            v4u pb[4];
            t_scores<D, false>(sm.k[cur], t, sc);
            if (j0 + kBK - 1 > n.w_tok || j0 < n.w_in) {
#pragma unroll
              for (int kt = 0; kt < 2; ++kt)
#pragma unroll
                for (int i = 0; i < 16; ++i) {
                  const int key = j0 + kt * 32 + 8 * (i >> 2) + 4 * h + (i & 3);
                  if (key > t.tok || key < t.begin) sc[kt][i] = -INFINITY;
                }
            }
            t_softmax<D, false>(sc, a.scale_log2, t, pb);
            t_values<D, false>(sm.v[cur], vb, pb, t);
          }
          if (blk + 1 < n.hi) {
            dma_wait();
            finite(blk + 1, cur ^ 1);
          }
          __syncthreads();
        }
        if (sm.odd && t.ok) add_odd<D>(a, s, g, 0, n, t);
      }
    }

    t_out<D>(a, s, t, od_xor32_sum(t.l), frame, sp, nv, 0, lower != 0);
    if (lower == 0 && (!H16 || (sp == 0 && a.k))) {
      if (t_over<D>(t)) sm.over = 1;
      __syncthreads();
      if (__builtin_amdgcn_readfirstlane(sm.over)) {
        lower = kLower;
        continue;
      }
    }
    lower = 0;
    tile += a.tiles;
  }
}

// ------------------------------------------------------------------------------------------ many slots, heads of 256
// 256 value columns of accumulators do not fit a wave's registers beside 256-wide queries, so two waves share 32 slots:
// each accumulates 128 of the columns. Each takes the scores of 32 of the block's 64 keys, and its half of the softmax,
// and they exchange the maximum and the probabilities through LDS (as the fragments that the products want); taking all
// the scores in both instead, 48 matrix instructions a block and wave for 32, cost a chunk of 2048 over 16000 bf16
// tokens 17% more, and 4 ragged first chunks of 2000 54%. Now: 661 us (860 TFLOP/s), over an image of int8 pages 652,
// 197 us. For that the waves meet twice a block. K runs a block ahead of V, so that both meetings also order the
// buffers:
//   scores(b) | maxima out, barrier | K(b + 2), V(b + 1) into the buffers of blocks that all are done with; softmax,
//   probabilities out, barrier | products(b), scores(b + 1) ...
struct alignas(16) WSmem {
  uint16_t k[2][kBK * 256];
  uint16_t v[2][kBK * 256];
  v4u p[4][4][64];     // [slot group][k-step][lane]
  float mx[2][4][32];  // [half][slot group][slot]
  int lo[8], hi[8];
  int over, odd;
};

template <int SRC>
__global__ __launch_bounds__(512, 2) void paged_wide_kernel(AttnArgs a) {
  // REG: blocks that are converted on their way, through registers
  constexpr bool Q4 = SRC == kInt4, REG = SRC == kInt8 || Q4, IMG = SRC == kImage, H16 = SRC != kBf16;
  constexpr int D = 256, NW = 8, NT = 512, SPT = 128, DT = 4;
  extern __shared__ __attribute__((aligned(16))) char smem_raw[];
  WSmem& sm = *reinterpret_cast<WSmem*>(smem_raw);
  const TilePlace at = tile_place(a);
  if (at.sp < 0) return;
  const int sp = at.sp, g = at.g, b = at.b;
  const Seq s = seq_of(a, b);
  const int nslots = s.n * a.rep, blocks = (s.ctx + kBK - 1) / kBK, nv = splits_of(a, blocks);
  if (sp >= nv || (IMG ? blocks > a.img_blocks : a.rest && blocks <= a.img_blocks)) return;
  const int b_lo = sp * a.chunk, b_hi = sp == a.nsplit - 1 ? blocks : min(blocks, b_lo + a.chunk);
  const int tid = threadIdx.x, lane = tid & 63, h = lane >> 5, col = lane & 31;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6), half = wave >> 2, grp = wave & 3;
  int vb[DT];  // transposing-read bases
#pragma unroll
  for (int dt = 0; dt < DT; ++dt) {
    const int hh = lane >> 5, mh = (lane >> 4) & 1, e = (lane >> 2) & 3, c = lane & 3;
    vb[dt] = (4 * hh + e) * D + (tv_chunk<D>(e, half * 16 + 4 * dt + 2 * mh + (c >> 1)) << 3) + 4 * (c & 1);
  }

  int lower = 0;  // the power of two that bf16 values are lowered by
  for (int tile = at.tile; tile * SPT < nslots;) {
    __syncthreads();  // an earlier tile's readers are done
    if (tid == 0) sm.over = 0;
    TSlot<D> t;
    const int zw = tile * SPT + grp * 32, z = zw + col;
    const bool live = zw < nslots;  // the wave has slots
    t.ok = z < nslots;
    t.tok = t.ok ? z / a.rep : s.n - 1;
    t.head = g * a.rep + (t.ok ? z % a.rep : 0);
    t.begin = a.row_begin && t.ok ? max(a.row_begin[s.s0 + t.tok], 0) : 0;
    t.m = -INFINITY;
    t.l = 0.0f;
    t.qe = 0;
#pragma unroll
    for (auto& o : t.o) o = zero16();
    t_load_q<D>(a, s, t);
    int frame = H16 ? 0 : lower;  // O is in units of 2^frame

    // this wave's half of a block's scores: keys 32 half + 8 (i / 4) + 4 h + i % 4
    auto scores = [&](auto H, const uint16_t* kb) {
      int place = tk_off<D>(half * 32 + col, h);
      asm volatile("" : "+v"(place));  // the places are formed here each time, not kept in registers
      v16f x = zero16();
      v4u kf[2];
      auto rd = [&](int i) {
        const uint16_t* at = &kb[place ^ (i << 4)];  // tk_off<D>(key, 2 i + h): chunks are 8 values, rows 256
        kf[i % 2] = __builtin_bit_cast(v4u, *reinterpret_cast<const uint4*>(at));
      };
      rd(0);
#pragma unroll
      for (int i = 0; i < D / 16; ++i) {
        if (i + 1 < D / 16) rd(i + 1);
        x = mfma32<decltype(H)::value>(kf[i % 2], t.q[i], x);
      }
      __builtin_amdgcn_sched_group_barrier(0x100, 1, 0);  // reads stay one ahead
#pragma unroll
      for (int i = 0; i < D / 16; ++i) {
        if (i + 1 < D / 16) __builtin_amdgcn_sched_group_barrier(0x100, 1, 0);
        __builtin_amdgcn_sched_group_barrier(0x008, 1, 0);
      }
      return x;
    };
    // maxima out; after the barrier: the common maximum decides, the probabilities go out
    auto put_max = [&](const v16f& x, float c) {
      float mx = -INFINITY;
#pragma unroll
      for (int r = 0; r < 16; ++r) mx = fmaxf(mx, x[r]);
      mx = od_xor32_max(mx) * c;
      if (h == 0) sm.mx[half][grp][col] = mx;
      return mx;
    };
    auto softmax = [&](auto H, const v16f& x, float c, float mine) {
      const float mx = fmaxf(mine, sm.mx[half ^ 1][grp][col]);
      const bool move = mx > t.m + kSlack;
      if (__builtin_amdgcn_ballot_w64(move) != 0) {
        const float f = move ? __builtin_amdgcn_exp2f(t.m - mx) : 1.0f;  // m = -inf: 0
#pragma unroll
        for (auto& o : t.o)
#pragma unroll
          for (int r = 0; r < 16; ++r) o[r] *= f;
        t.l *= f;
        if (move) t.m = mx;
      }
      const float ms = (t.m == -INFINITY ? 0.0f : t.m) - kLift;
      float sum = 0.0f;
      v4u mp[2];
#pragma unroll
      for (int r = 0; r < 16; r += 2) {
        const float p0 = __builtin_amdgcn_exp2f(__builtin_fmaf(x[r], c, -ms));
        const float p1 = __builtin_amdgcn_exp2f(__builtin_fmaf(x[r + 1], c, -ms));
        sum += p0;
        sum += p1;
        if constexpr (decltype(H)::value) {
          const f16x2 w = {(_Float16)p0, (_Float16)p1};
          mp[r >> 3][(r & 7) >> 1] = __builtin_bit_cast(uint32_t, w);
        } else {
          mp[r >> 3][(r & 7) >> 1] = od_pack_bf16x2(p0, p1);
        }
      }
      t.l += sum;  // this lane's share: its keys of this wave's half
      sm.p[grp][2 * half][lane] = mp[0];
      sm.p[grp][2 * half + 1][lane] = mp[1];
    };
    auto get_p = [&](v4u (&pb)[4]) {
#pragma unroll
      for (int k = 0; k < 4; ++k) pb[k] = sm.p[grp][k][lane];
    };
    auto rescale = [&](int f_new, int by) {  // uniform over the workgroup
      if (f_new == frame) return;
      const float f = __builtin_ldexpf(1.0f, by);
#pragma unroll
      for (auto& o : t.o)
#pragma unroll
        for (int i = 0; i < 16; ++i) o[i] *= f;
      frame = f_new;
    };
    using HT = std::integral_constant<bool, H16>;

    // ---- the cached blocks b_lo .. b_hi - 1
    if (b_lo < b_hi) {
      if constexpr (H16) t_q_to_f16<D>(t);
      const int64_t first = ((int64_t)b * a.p.Hkv + g) * a.img_blocks;  // image: the sequence's first block
      if constexpr (IMG) frame = a.img_vexp[b * a.p.Hkv + g] - 7;
      constexpr int CPK = D / (Q4 ? 32 : 16), NC = kBK * CPK / NT;  // 16-byte chunks per row; per thread and side
      const int in_page = (1 << a.p.shift) - 1;
      // lane l: the page of key l of a block, or -1
      auto pages = [&](int blk) {
        if constexpr (IMG) return -1;
        const int pos = blk * kBK + lane;
        const int pg = pos < s.ctx ? a.p.table[b * a.p.ld_table + (pos >> a.p.shift)] : -1;
        return pg < a.p.n_pages ? pg : -1;
      };
      auto row = [&](int blk, int pg, int key) {  // a key that is not there is read from page 0 and left out later
        return (((int64_t)max(__shfl(pg, key, 64), 0) * a.p.Hkv + g) << a.p.shift) + ((blk * kBK + key) & in_page);
      };
      // int8: a block's K or V into registers, and lane l the scale of key l
      // (the places below are formed each time: kept over the block loop they cost the kernel 60 spilled registers)
      auto load8 = [&](int blk, int pg, const void* pool, const float* scales, v4u (&r)[NC], float& sc) {
        int ti = tid;
        asm volatile("" : "+v"(ti));
        sc = scales[(((int64_t)max(pg, 0) * a.p.Hkv + g) << a.p.shift) + ((blk * kBK + lane) & in_page)];
#pragma unroll
        for (int i = 0; i < NC; ++i) {
          const int key = (i * NT + ti) / CPK, ch = (i * NT + ti) % CPK;
          const char* at = static_cast<const char*>(pool) + row(blk, pg, key) * D + 16 * ch;
          r[i] = __builtin_bit_cast(v4u, *reinterpret_cast<const uint4*>(at));
        }
      };
      auto scale_bits = [&](int pg, float sc) {  // the largest scale of the block's keys that is a number, as bits
        return od_wave_umax_dpp(pg >= 0 && sc < INFINITY && sc > 0 ? __float_as_uint(sc) : 0u);
      };
      auto put8 = [&](uint16_t* dst, bool v, const v4u (&r)[NC], float f) {
        int ti = tid;
        asm volatile("" : "+v"(ti));
#pragma unroll
        for (int i = 0; i < NC; ++i) {
          const int key = (i * NT + ti) / CPK, ch = (i * NT + ti) % CPK;
          v4u lo, hi;
          __builtin_amdgcn_sched_barrier(0);
          i8x16_scaled(r[i], __shfl(f, key, 64), lo, hi);
          const int o0 = v ? key * D + (tv_chunk<D>(key, 2 * ch) << 3) : tk_off<D>(key, 2 * ch);
          const int o1 = v ? key * D + (tv_chunk<D>(key, 2 * ch + 1) << 3) : tk_off<D>(key, 2 * ch + 1);
          *reinterpret_cast<uint4*>(dst + o0) = __builtin_bit_cast(uint4, lo);
          *reinterpret_cast<uint4*>(dst + o1) = __builtin_bit_cast(uint4, hi);
        }
      };
      // 4 bits: a block's K or V (one chunk a thread), the chunk's scale in the high half of sc and in the low one, lane l, the
      // largest of key l's
      auto load4 = [&](int blk, int pg, const void* pool, const uint16_t* scales, v4u (&r)[NC], uint32_t& sc) {
        const int key = tid / CPK, ch = tid % CPK;
        uint32_t w[D / 64];
        q4_row_scales<D>(scales, (((int64_t)max(pg, 0) * a.p.Hkv + g) << a.p.shift) + ((blk * kBK + lane) & in_page), w);
        const int64_t from = row(blk, pg, key);
        r[0] = __builtin_bit_cast(v4u, *reinterpret_cast<const uint4*>(static_cast<const char*>(pool) + from * (D / 2) + 16 * ch));
        sc = q4_largest(w) | (uint32_t)scales[from * CPK + ch] << 16;
      };
      auto largest4 = [&](int pg, uint32_t sc) { return od_wave_umax_dpp(pg >= 0 ? sc & 0xffffu : 0u); };
      auto put4 = [&](uint16_t* dst, bool v, const v4u (&r)[NC], uint32_t sc, int pg, int e) {
        const int key = tid / CPK;
        q4_put<D>(dst, v, key, tid % CPK, r[0], f16_scale(__shfl(pg, key, 64) >= 0 ? sc >> 16 : 0u, 7 - e));
      };
      v4u rk[REG ? NC : 1], rv[REG ? NC : 1];
      float ks = 0, vs = 0;
      uint32_t ks4 = 0, vs4 = 0;
      int ke0 = 0, ke1 = 0;  // the frames of the K blocks in the two buffers
      int vexp = 0;          // the frame of the last V block stored
      bool vexp_set = false;
      auto store_k = [&](int blk, int pg) {
        if constexpr (REG) {
          int e;
          if constexpr (Q4) {
            e = q4_frame(largest4(pg, ks4));
            put4(sm.k[blk & 1], false, rk, ks4, pg, e);
          } else {
            e = exp_above(scale_bits(pg, ks));
            put8(sm.k[blk & 1], false, rk, pg >= 0 ? frame_scale(ks, 7 - e) : 0.0f);
          }
          if (blk & 1) ke1 = e;
          else ke0 = e;
        }
      };
      auto store_v = [&](int blk, int pg) {
        if constexpr (REG) {
          const uint32_t bits = Q4 ? largest4(pg, vs4) : scale_bits(pg, vs);
          const int e = Q4 ? q4_frame(bits) : exp_above(bits);
          if (bits) vexp = vexp_set ? max(vexp, e) : e;
          if (bits) vexp_set = true;
          if constexpr (Q4) put4(sm.v[blk & 1], true, rv, vs4, pg, vexp);
          else put8(sm.v[blk & 1], true, rv, pg >= 0 ? frame_scale(vs, 7 - vexp) : 0.0f);
        }
      };
      auto load_k = [&](int blk, int pg) {
        if constexpr (Q4) load4(blk, pg, a.p.k, a.p.k4, rk, ks4);
        else if constexpr (REG) load8(blk, pg, a.p.k, a.p.ks, rk, ks);
        else if constexpr (IMG) dma_block<D, NW>(sm.k[blk & 1], wave, a.img + (first + blk) * (2 * kBK * D));
        else dma_pages<D, NW>(sm.k[blk & 1], wave, false, a.p, g, blk, pg);
      };
      auto load_v = [&](int blk, int pg) {
        if constexpr (Q4) load4(blk, pg, a.p.v, a.p.v4, rv, vs4);
        else if constexpr (REG) load8(blk, pg, a.p.v, a.p.vs, rv, vs);
        else if constexpr (IMG) dma_block<D, NW>(sm.v[blk & 1], wave, a.img + (first + blk) * (2 * kBK * D) + kBK * D);
        else dma_pages<D, NW>(sm.v[blk & 1], wave, true, a.p, g, blk, pg);
      };
      // pages of the blocks blk (the current one), blk + 1, blk + 2, blk + 3; past the last block: none
      int p0 = pages(b_lo), p1 = pages(b_lo + 1), p2 = pages(b_lo + 2), p3 = pages(b_lo + 3);
      load_k(b_lo, p0);
      load_v(b_lo, p0);
      if constexpr (REG) {
        v4u rn[NC];
        float sn = 0;
        uint32_t sn4 = 0;
        if constexpr (Q4) load4(b_lo + 1, p1, a.p.k, a.p.k4, rn, sn4);
        else load8(b_lo + 1, p1, a.p.k, a.p.ks, rn, sn);
        store_k(b_lo, p0);
        store_v(b_lo, p0);
#pragma unroll
        for (int i = 0; i < NC; ++i) rk[i] = rn[i];
        ks = sn;
        ks4 = sn4;
        store_k(b_lo + 1, p1);
        load_k(b_lo + 2, p2);
        load_v(b_lo + 1, p1);
      } else {
        if (!IMG || b_lo + 1 < b_hi) load_k(b_lo + 1, p1);
        dma_wait();
      }
      int f_cur = vexp - 7;
      if constexpr (REG) frame = f_cur;  // O is 0 still: no rescaling, by what may be no fp32 number
      __syncthreads();
      ImageBlock head = {};
      if constexpr (IMG) head = a.img_heads[first + b_lo];
      for (int blk = b_lo; blk < b_hi; ++blk) {
        const int kexp = IMG ? head.kexp : blk & 1 ? ke1 : ke0;
        const float c = H16 ? score_factor(a.scale_log2, t.qe - 14 + kexp - 7) : a.scale_log2;
        const uint64_t seen = IMG ? head.seen : __builtin_amdgcn_ballot_w64(p0 >= 0);
        if (IMG && blk + 1 < b_hi) head = a.img_heads[first + blk + 1];
        v16f x;
        float mine = -INFINITY;
        if (live) {
          x = scores(HT{}, sm.k[blk & 1]);
          if (seen != ~0ull) {
            const uint64_t m4 = seen >> (32 * half + 4 * h);
#pragma unroll
            for (int i = 0; i < 16; ++i)
              if (!((m4 >> (8 * (i >> 2) + (i & 3))) & 1)) x[i] = -INFINITY;
          }
          mine = put_max(x, c);
        }
        if constexpr (!REG) dma_wait();  // this wave's part of V(blk) and K(blk + 1)
        __syncthreads();
        if (!H16 && (seen != ~0ull || lower)) {  // values of keys that are not there: 0 (their scores are masked)
          for (int i = tid; i < kBK * (D / 8); i += NT)
            if (!((seen >> (i / (D / 8))) & 1))
              *reinterpret_cast<uint4*>(&sm.v[blk & 1][8 * i]) = make_uint4(0, 0, 0, 0);
          if (lower) t_lower<D, NT>(sm.v[blk & 1]);
        }
        const int f_now = f_cur;
        if constexpr (REG) {
          if (blk + 2 < b_hi) store_k(blk + 2, p2);
          if (blk + 1 < b_hi) store_v(blk + 1, p1);
          f_cur = vexp - 7;
          if (blk + 3 < b_hi) load_k(blk + 3, p3);
          if (blk + 2 < b_hi) load_v(blk + 2, p2);
        } else {
          if (blk + 2 < b_hi) load_k(blk + 2, p2);
          if (blk + 1 < b_hi) load_v(blk + 1, p1);
        }
        p0 = p1;
        p1 = p2;
        p2 = p3;
        p3 = pages(blk + 4);
        v4u pb[4];
        if (live) {
          // the values' frame rose (or is the first one, and may lie lower by any amount: O is 0 still, or NaN)
          if constexpr (REG) rescale(f_now, min(frame - f_now, 0));
          softmax(HT{}, x, c, mine);
        }
        __syncthreads();
        if (live) {
          get_p(pb);
          t_values<D, H16>(sm.v[blk & 1], vb, pb, t);
        }
      }
    }

    // ---- the new tokens, in split 0
    if (sp == 0 && a.k) {
      if (H16 && b_lo < b_hi) {  // back to bf16 queries and values as they are
        t_load_q<D>(a, s, t);
        rescale(lower, frame - lower);
      }
      frame = lower;
      const NewSpan n = new_span(a, s, tile, SPT, zw, live, t, sm.lo, sm.hi, &sm.odd, NW, wave);
      auto load_k = [&](int blk) {
        const uint16_t* kp = a.k + (int64_t)s.s0 * a.skt + (int64_t)g * a.skh;
        dma_rows<D, NW>(sm.k[blk & 1], wave, false,
                        [&](int key) { return kp + min(blk * kBK + key, s.n - 1) * a.skt; });
      };
      auto load_v = [&](int blk) {
        const uint16_t* vp = a.v + (int64_t)s.s0 * a.svt + (int64_t)g * a.svh;
        dma_rows<D, NW>(sm.v[blk & 1], wave, true, [&](int key) { return vp + min(blk * kBK + key, s.n - 1) * a.svt; });
      };
      if (n.lo < n.hi) {
        load_k(n.lo);
        load_v(n.lo);
        if (n.lo + 1 < n.hi) load_k(n.lo + 1);
        dma_wait();
        __syncthreads();
        for (int blk = n.lo; blk < n.hi; ++blk) {
          const int j0 = blk * kBK;
          const bool work = live && j0 <= n.w_hi && j0 + kBK > n.w_lo;
          v16f x;
          float mine = -INFINITY;
          if (work) {
            x = scores(std::false_type{}, sm.k[blk & 1]);
            if (j0 + kBK - 1 > n.w_tok || j0 < n.w_in) {
#pragma unroll
              for (int i = 0; i < 16; ++i) {
                const int key = j0 + half * 32 + 8 * (i >> 2) + 4 * h + (i & 3);
                if (key > t.tok || key < t.begin) x[i] = -INFINITY;
              }
            }
            mine = put_max(x, a.scale_log2);
          }
          dma_wait();
          __syncthreads();
          if (n.partial(blk)) make_finite<D, NT>(sm.v[blk & 1], &sm.odd);
          if (lower) t_lower<D, NT>(sm.v[blk & 1]);
          if (blk + 2 < n.hi) load_k(blk + 2);
          if (blk + 1 < n.hi) load_v(blk + 1);
          v4u pb[4];
          if (work) softmax(std::false_type{}, x, a.scale_log2, mine);
          __syncthreads();
          if (work) {
            get_p(pb);
            t_values<D, false>(sm.v[blk & 1], vb, pb, t);
          }
        }
        if (sm.odd && t.ok) add_odd<D>(a, s, g, half, n, t);
      }
    }

    // ---- the sum of both halves, then as above
    float l = od_xor32_sum(t.l);
    __syncthreads();  // the last block's maxima are read
    if (h == 0) sm.mx[half][grp][col] = l;
    __syncthreads();
    l += sm.mx[half ^ 1][grp][col];
    t_out<D>(a, s, t, l, frame, sp, nv, half, lower != 0);
    if (lower == 0 && (!H16 || (sp == 0 && a.k))) {
      if (t_over<D>(t)) sm.over = 1;
      __syncthreads();
      if (__builtin_amdgcn_readfirstlane(sm.over)) {
        lower = kLower;
        continue;
      }
    }
    lower = 0;
    tile += a.tiles;
  }
}

// ------------------------------------------------------------------------------------------ the image of int8 pages
// Where many slot tiles read the same int8 pages, converting them in each costs more than once for all: the two kernels
// here write the blocks that the tile kernels want, fp16 in frames and in the order of LDS, into the workspace. V's
// frame is that of its largest scale over the whole (sequence, KV head), K's that of the block. Sequences longer than
// img_blocks (the caller's bound was too low) have none; sequences without new tokens need none. A wave takes the frame
// of one block's V (5 us; of all of them in a workgroup per (sequence, KV head), 32768 tokens took 20). The
// image of 32768 tokens, 8 heads of 128, takes 35 to 47 us, 4.3 to 5.6 TB/s.
template <int D, int P>
__global__ __launch_bounds__(kThreads) void page_frame_kernel(AttnArgs a) {
  const int blk = blockIdx.x * (kThreads / 64) + (threadIdx.x >> 6), g = blockIdx.y, b = blockIdx.z;
  const Seq s = seq_of(a, b);
  const int blocks = (s.ctx + kBK - 1) / kBK, pos = blk * kBK + (threadIdx.x & 63);
  if (s.n == 0 || blk >= blocks || blocks > a.img_blocks) return;
  const int64_t row = pos < s.ctx ? row_of(a.p, b, g, pos) : -1;
  uint32_t bits = 0;
  if constexpr (P == kInt4) {
    uint32_t w[D / 64] = {};
    if (row >= 0) q4_row_scales<D>(a.p.v4, row, w);
    bits = q4_largest(w) << 16;
  } else {
    const float vs = row >= 0 ? a.p.vs[row] : 0.0f;
    bits = vs < INFINITY && vs > 0 ? __float_as_uint(vs) : 0u;
  }
  const uint32_t m = od_wave_umax_dpp(bits);
  if ((threadIdx.x & 63) == 0)
    a.img_heads[((int64_t)b * a.p.Hkv + g) * a.img_blocks + blk].v_bits = m;
}
template <int D, int P>
__global__ __launch_bounds__(kThreads) void page_image_kernel(AttnArgs a) {
  constexpr bool Q4 = P == kInt4;
  constexpr int CPK = D / (Q4 ? 32 : 16), CH = kBK * CPK, NC = 2 * CH / kThreads;
  const int blk = blockIdx.x, g = blockIdx.y, b = blockIdx.z, lane = threadIdx.x & 63;
  const Seq s = seq_of(a, b);
  const int blocks = (s.ctx + kBK - 1) / kBK;
  if (s.n == 0 || blk >= blocks || blocks > a.img_blocks) return;
  const int64_t at = ((int64_t)b * a.p.Hkv + g) * a.img_blocks + blk;
  const int pos = blk * kBK + lane;
  const int64_t mine = pos < s.ctx ? row_of(a.p, b, g, pos) : -1, row = max(mine, (int64_t)0);
  const bool on = mine >= 0;  // a key that is not there: the pool's first row, times 0
  float ks = 0, vs = 0;       // int8
  uint32_t k_bits;
  if constexpr (Q4) {
    uint32_t w[D / 64];
    q4_row_scales<D>(a.p.k4, row, w);
    k_bits = q4_largest(w);
  } else {
    ks = a.p.ks[row], vs = a.p.vs[row];
    k_bits = ks < INFINITY && ks > 0 ? __float_as_uint(ks) : 0u;
  }
  const uint64_t seen = __builtin_amdgcn_ballot_w64(on);
  const uint32_t km = od_wave_umax_dpp(on ? k_bits : 0u);
  const int kexp = Q4 ? q4_frame(km) : exp_above(km);
  // the largest of all blocks, by every wave
  uint32_t vm = 0;
#pragma unroll 4
  for (int i = lane; i < blocks; i += 64) vm = max(vm, a.img_heads[at - blk + i].v_bits);
  vm = od_wave_umax_dpp(vm);
  const int vexp = Q4 ? q4_frame(vm >> 16) : exp_above(vm);
  const float kf = on ? frame_scale(ks, 7 - kexp) : 0.0f, vf = on ? frame_scale(vs, 7 - vexp) : 0.0f;
  if (threadIdx.x == 0) {
    a.img_heads[at].seen = seen;
    a.img_heads[at].kexp = kexp;
    if (blk == 0) a.img_vexp[b * a.p.Hkv + g] = vexp;
  }
  v4u r[NC];
  uint32_t rs[NC];  // 4 bits: the chunks' scales
#pragma unroll
  for (int i = 0; i < NC; ++i) {
    const int cid = i * kThreads + threadIdx.x, side = cid / CH, key = cid % CH / CPK, ch = cid % CPK;
    const int64_t from = ((int64_t)__shfl((int)(row >> 32), key, 64) << 32) | (uint32_t)__shfl((int)row, key, 64);
    r[i] = __builtin_bit_cast(v4u, *reinterpret_cast<const uint4*>(static_cast<const char*>(side ? a.p.v : a.p.k) +
                                                                  from * (16 * CPK) + 16 * ch));
    if constexpr (Q4) rs[i] = (side ? a.p.v4 : a.p.k4)[from * CPK + ch];
  }
#pragma unroll
  for (int i = 0; i < NC; ++i) {
    const int cid = i * kThreads + threadIdx.x, side = cid / CH, key = cid % CH / CPK, ch = cid % CPK;
    uint16_t* dst = a.img + at * (2 * kBK * D) + side * (kBK * D);
    if constexpr (Q4) {
      q4_put<D>(dst, side, key, ch, r[i], f16_scale((seen >> key) & 1 ? rs[i] : 0u, 7 - (side ? vexp : kexp)));
    } else {
      v4u lo, hi;
      i8x16_scaled(r[i], __shfl(side ? vf : kf, key, 64), lo, hi);
      const int o0 = side ? key * D + (tv_chunk<D>(key, 2 * ch) << 3) : tk_off<D>(key, 2 * ch);
      const int o1 = side ? key * D + (tv_chunk<D>(key, 2 * ch + 1) << 3) : tk_off<D>(key, 2 * ch + 1);
      *reinterpret_cast<uint4*>(dst + o0) = __builtin_bit_cast(uint4, lo);
      *reinterpret_cast<uint4*>(dst + o1) = __builtin_bit_cast(uint4, hi);
    }
  }
}

// How a call is split. Sequences' lengths are on the device; the host knows bounds.
struct Plan {
  bool stream;
  int ct, waves;  // stream: columns of 16 slots, 1 or 2; waves a SIMD
  int nw, tiles, run, width, chunk, nsplit;
  int64_t img_blocks;  // of every (sequence, KV head); 0: no image
  // the workspace, in floats: partials, then the image's V frames, heads and blocks
  int64_t part, vexp, heads, img;
  int64_t floats() const { return part + vexp + heads + img; }
};
Plan plan_of(int64_t B, int64_t N, int64_t Hq, int64_t Hkv, int64_t D, int64_t max_new, int64_t max_ctx, int format) {
  const bool q8 = format == OD_PAGE_INT8, q4 = format == OD_PAGE_INT4;
  Plan p;
  // hints past any call's own size say nothing; below 2^30 no split begins past the positions an int holds
  max_new = max_new < N ? max_new : N;
  max_ctx = max_ctx < (1 << 30) ? max_ctx : 1 << 30;
  const int64_t rep = Hq / Hkv, slots = (max_new < 1 ? 1 : max_new) * rep, cus = od_cu_count();
  // Up to 32 slots stream: 8 tokens of 4 heads a group over 16 ragged x 4000 int8 tokens 37 us, 51 as tiles of 128
  // slots (bf16 42 and 45; over 1 x 4000 15 and 29, bf16 15 and 25). Up to 64, as two workgroups of 32, over int8 pages
  // of heads of 64 and 128, where half of a tile's waves would idle beside its conversions (16 tokens over 32 x 8000
  // 146 and 201 us, heads of 64 over 16 x 4000 35 and 44; but bf16 235 and 185, int8 heads of 256 140 and 139, 80 slots
  // 90 and 78). More of them where there is little work: a step of the tile kernel is a chain of some 2 us that needs
  // company on its CU, a streaming one has nothing to wait for but memory. The workgroups fit in at once and have no
  // more than 128 KB of K a CU to read, from the L2 mostly: 16 tokens over 1 x 4000 16 us, 30 as tiles; 256 over 1 x
  // 100 15 and 24; 32 over 2 x 4000 21 and 32; above it 32 over 1 x 32000 62 and 50, bf16 80 and 42, 120 of one head
  // over 1 x 8000 bf16 tokens 37 and 34.
  // 4-bit pages take int8's limit of slots and bf16's of bytes. Streaming and as tiles they take: heads of 128, 64 slots, 16 x 16
  // tokens over 4000 49 us and 59, 32 x 16 over 8000 135 and 191; 80 slots 72 and 61; 96, 8 x 24 over 2000 33 and 35; heads of 64, 64
  // slots, 16 x 16 over 4000 25 and 35, 80 slots 34 and 37; within the bytes 1 x 128 over 1000 22 and 35, 1 x 256 over 100 17 and 25;
  // past them 1 x 64 over 4000 26 and 35, 1 x 32 over 32000 48 and 43, 2 x 64 over 16000 78 and 67. Both limits are low for heads of
  // 256: 16 x 16 over 4000 55 and 86, 8 x 32 over 4000 55 and 69, 2 x 64 over 16000 86 and 93.
  const int64_t few = B * Hkv * ((slots + 31) / 32);
  const int64_t always = (q8 || q4) && D <= 128 && Hkv < (1 << 15) ? 64 : 32;  // (a grid has 65535 rows)
  p.stream = slots <= always || (slots <= 1024 && few <= 2 * cus && few * max_ctx * D * (q8 ? 1 : 2) <= (cus << 17));
  p.ct = slots <= 16 ? 1 : 2;
  // workgroups without splits for tiles of spt slots: every sequence's, but no more than the tokens make
  auto wgs_of = [&](int64_t spt) {
    const int64_t each = (slots + spt - 1) / spt * B, all = N * rep / spt + B;
    return (each < all ? each : all) * Hkv;
  };
  // Heads of 128 take 8 waves, which share a block (chunk of 2048 over 32768 1140 us, 4 waves 1193; bf16 1137 and
  // 1304), or 4 for few slots and for several sequences that leave CUs without work: the longest of them decides then,
  // and its workgroups run faster where they have a CU to themselves (2 ragged x 1024 over 8000 244 us with 8, 195 with
  // 4; bf16 271 and 244; 3 x 700 over 4000 142 and 123; but 2 x 2000 over 500, 432 of 8, 90 and 98). Heads of 64: 4
  // (bf16 chunks of 2048 over 16000 234 and 202).
  const bool wide8 = D == 128 && slots > 128 && (B == 1 || wgs_of(256) >= cus);
  p.nw = p.stream ? kStreamWaves : D == 256 || wide8 ? 8 : 4;
  p.width = p.stream ? 16 * s_halves((int)D, q4 ? kInt4 : q8 ? kInt8 : kBf16) : kBK;
  const int64_t spt = p.stream ? 16 * p.ct : D == 256 ? 128 : 32 * p.nw;
  const int64_t tiles = (slots + spt - 1) / spt, wgs = wgs_of(spt), keys = (max_ctx + p.width - 1) / p.width;
  p.tiles = (int)tiles;
  // how many run at once: two a CU, one where a wave or the shared memory needs it whole, three that stream 4-bit pages (8 ragged
  // states of up to 32768 tokens 60 us in 12 splits, 66 in 8; 16 x 16000 59 and 61; but 64 x 4096 55 and 53). Heads of 256 over
  // 4-bit pages: one, whose wave holds all it works on, where all of them are in at once (a token over 4 x 8000 19.8 us, 23.2 with
  // two; 64 x 700 19.6 and 24.9, 64 x 2000 39.4 and 47; but 128 x 1000 48.6 and 43.4, 256 x 300 49 and 37)
  p.waves = !p.stream ? 0 : q4 && D == 256 && p.ct == 1 && wgs <= cus ? 1 : s_waves((int)D, q4 ? kInt4 : q8 ? kInt8 : kBf16, p.ct);
  const int64_t fit = cus * (p.stream ? p.waves : p.nw == 8 ? 1 : 2);
  // key tiles that are worth a workgroup of their own (128 tokens over 1 x 1000: 37 us with 8 blocks at least, 35 with
  // 2)
  // (4-bit pages: 2 where the workgroups are few or the heads wide: a token over 1 x 1500, heads of 256 10.8 us, 14.7 with 8, heads
  // of 128 9.0 and 11.4, 4 x 3000 13.3 and 14.4; but 16 x 700 13.9 and 11.9)
  const int64_t least = !p.stream || (q4 && (D == 256 || 8 * wgs <= cus)) ? 2 : 8;
  int64_t most = keys / least < 128 ? keys / least : 128, n = 1;
  if (N > kMaxGroups) most = 1;  // no merge, which has a workgroup a token
  // two streams of that size take as long as one (a token over 500: 9.9 us, 10.1 whole), with a launch more for the
  // host, 4 us of it; not so heads of 256 over 4-bit pages (over 700 10.5 us, 17.4 whole; over 400 10.6 and 14.0)
  if (p.stream && keys / 8 < (q4 && D == 256 ? 2 : 3)) most = 1;
  if (p.stream) {
    n = fit / (wgs < 1 ? 1 : wgs);
    if (n > most) n = most;
    if (n < 1) n = 1;
  } else {
    // The n of least cost: rounds of workgroups times a workgroup's blocks and what it costs besides them, about 12
    // blocks (the queries, the first loads, the new tokens, the partials). x > 1 rounds count as x + 1/2, 1.6 at least:
    // a workgroup starts where another ends, and the last ones leave CUs idle. A chunk of 512 over 16000 takes 583 us
    // whole, 223 in 3, 192 in 4 (one round), 234 in 6 parts; 5 ragged bf16 600 over 2000 (592 workgroups) whole rounds
    // chose 2 parts, 108 us, and this takes 3, 91; 8 x 384 over 6000 272 and 251. Heads of 64: three workgroups a CU
    // where that takes 4 parts at most (ragged bf16 chunks of 700 over 3000 in 3 parts 44 us, in 2 50; 2048 over 16000
    // 187 and 204; but 4 x 256 over 6000 in 7 parts 66, in 5 53).
    int64_t best = 0;
    for (int64_t i = 1; i <= most || i == 1; ++i) {
      const int64_t at_once = D == 64 && tiles >= 4 && i <= 4 ? 3 * cus : fit;
      const int64_t x10 = 10 * wgs * i / at_once + 5, rounds10 = wgs * i <= at_once ? 10 : x10 < 16 ? 16 : x10;
      const int64_t cost = rounds10 * ((keys + i - 1) / i + 12);
      if (best == 0 || cost < best) {
        best = cost;
        n = i;
      }
    }
  }
  p.chunk = (int)((keys + n - 1) / n);
  if (p.chunk < 1) p.chunk = 1;
  p.nsplit = (int)((keys + p.chunk - 1) / p.chunk);
  if (p.nsplit < 1) p.nsplit = 1;
  // (Bounds far above a batch's own lengths could ask for more slot tiles than a launch holds: its workgroups go on to the
  // tiles behind the grid's.)
  const int64_t groups = B * Hkv * p.nsplit, room = kMaxGroups / 8 / groups;
  if (!p.stream && p.tiles > room) p.tiles = room < 1 ? 1 : (int)room;
  // runs of tiles: as many as give every XCD the same number, or a few each
  int parts = 1;
  while (parts < 8 && groups * parts % 8 && groups * parts < 64) parts *= 2;
  p.run = (p.tiles + parts - 1) / parts;
  p.part = p.nsplit > 1 ? (p.nsplit * N * Hq * (D + 1) + 3) / 4 * 4 : 0;
  // The image, up to 1 GB of it, where 4 slot tiles or more share a block and the conversions that it saves are worth
  // its launches: counted in values a slot they are wgs keys D / spt. Chunks of 2048 over 32768 1382 us, with it 1183;
  // 256-wide heads, 4 ragged 900 over 6000 402, 284; 1 x 256 over 6000 (3000 blocks in all) 82, 76; 8 x 64 (2 tiles)
  // 115, 121; heads of 128, 8 x 256 over 6000 (4 tiles) 217, 183, 8 x 128 (2 tiles) 150, 139, 4 x 1024 over 1000 (8000
  // blocks) 85, 87, 4 x 256 over 6000 (12000) 152, 115.
  // 4-bit pages take the same rule, without the image and with it: heads of 128, 2048 over 16384 660 us and 565, 4 x 1024 over 1000
  // 150 and 145, 4 x 256 over 6000 151 and 154; heads of 256, 4 x 900 over 6000 770 and 532, 256 over 6000 86 and 80, 8 x 64 121 and
  // 165; heads of 64, 2048 over 16000 298 and 192. Several sequences of few tiles of 128-wide heads would do better without: 8 x
  // 256 over 6000 240 and 279, 8 x 128 151 and 200, 4 x 256 over 2000 68 and 76; option rows, 8 x 512 over 2048, take as long.
  p.img_blocks = !p.stream && (q8 || q4) && tiles >= 4 && wgs * keys * D / spt > 5 << 10 ? keys : 0;
  if (p.img_blocks * B * Hkv > (1ll << 28) / (kBK * D)) p.img_blocks = 0;
  p.vexp = p.img_blocks ? (B * Hkv + 3) / 4 * 4 : 0;
  p.heads = p.img_blocks * B * Hkv * 4;
  p.img = p.img_blocks * B * Hkv * kBK * D;
  return p;
}

// slots of a KV head, so that an int holds them and a stride of tiles past them
constexpr int64_t kMaxSlots = 0x3fff0000;

// A launch with more than 64 KB of LDS, which a kernel has to be allowed once per device.
template <auto* Kernel>
int launch_big(const AttnArgs& a, unsigned groups, int threads, int bytes, hipStream_t st) {
  static std::atomic<uint64_t> allowed{0};
  int dev = 0;
  if (hipGetDevice(&dev) != hipSuccess || dev < 0 || dev >= 64) return OD_ERR_LAUNCH;
  if (!((allowed.load(std::memory_order_relaxed) >> dev) & 1)) {
    if (hipFuncSetAttribute(reinterpret_cast<const void*>(Kernel), hipFuncAttributeMaxDynamicSharedMemorySize,
        bytes) != hipSuccess)
      return OD_ERR_LAUNCH;
    allowed.fetch_or(1ull << dev, std::memory_order_relaxed);
  }
  Kernel<<<dim3(groups), dim3(threads), bytes, st>>>(a);
  return OD_OK;
}
template <int D, int SRC, int NW>
int launch_tiles(const AttnArgs& a, unsigned groups, hipStream_t st) {
  return launch_big<&paged_tile_kernel<D, SRC, NW>>(a, groups, NW * 64, (int)sizeof(TSmem<D, NW>), st);
}

}  // namespace

extern "C" int od_page_append_ex(const uint16_t* k, int64_t skt, int64_t skh, const uint16_t* v, int64_t svt, int64_t svh,
                                 int format, void* k_pages, void* k_scale, void* v_pages, void* v_scale, int64_t n_pages,
                                 int64_t page, const int32_t* table, int64_t ld_table, int64_t cols, const int32_t* start,
                                 const int32_t* ctx_len, int64_t B, int64_t N, int64_t Hkv, int64_t D,
                                 od_stream_t stream) {
  AppendArgs a;
  if (const int rc = paged_args(a.p, format, k_pages, k_scale, v_pages, v_scale, n_pages, page, table, ld_table,
                                cols, start, ctx_len, B, N, Hkv, D))
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
  const int64_t per_block = (int64_t)(kThreads / 64) * (64 / (D / 16));
  const int64_t blocks = (N * 2 * Hkv + per_block - 1) / per_block;
  if (blocks > kMaxGroups) return OD_ERR_SHAPE;
  by_head_dim(D, [&](auto DC) {
    constexpr int DD = decltype(DC)::value;
    const dim3 grid((unsigned)blocks);
    by_format(format, [&](auto PC) {
      page_append_kernel<DD, decltype(PC)::value><<<grid, dim3(kThreads), 0, (hipStream_t)stream>>>(a);
    });
  });
  return od_launch_status();
}

extern "C" int od_page_append(const uint16_t* k, int64_t skt, int64_t skh, const uint16_t* v, int64_t svt, int64_t svh,
                              void* k_pages, float* k_scale, void* v_pages, float* v_scale, int64_t n_pages,
                              int64_t page, const int32_t* table, int64_t ld_table, int64_t cols, const int32_t* start,
                              const int32_t* ctx_len, int64_t B, int64_t N, int64_t Hkv, int64_t D,
                              od_stream_t stream) {
  return od_page_append_ex(k, skt, skh, v, svt, svh, k_scale || v_scale ? OD_PAGE_INT8 : OD_PAGE_BF16, k_pages, k_scale,
                           v_pages, v_scale, n_pages, page, table, ld_table, cols, start, ctx_len, B, N, Hkv, D, stream);
}

extern "C" int od_page_read_ex(int format, const void* k_pages, const void* k_scale, const void* v_pages, const void* v_scale,
                               int64_t n_pages, int64_t page, const int32_t* table, int64_t ld_table, int64_t cols,
                               const int32_t* length, int64_t B, int64_t T, int64_t Hkv, int64_t D, int form, void* k_out,
                               float* ks_out, void* v_out, float* vs_out, od_stream_t stream) {
  ReadArgs a;
  if (const int rc = paged_args(a.p, format, k_pages, k_scale, v_pages, v_scale, n_pages, page, table, ld_table,
                                cols, nullptr, length, B, 0, Hkv, D))
    return rc;
  if (T < 0 || T > 0x3fffffff) return OD_ERR_SHAPE;
  if (form != OD_READ_BF16 && form != OD_READ_FP32 && form != OD_READ_INT8) return OD_ERR_UNSUPPORTED;
  if (form == OD_READ_INT8 && format != OD_PAGE_INT8) return OD_ERR_UNSUPPORTED;
  if (B == 0 || T == 0) return OD_OK;
  if (!length || !k_out || !v_out || (cols > 0 && !table)) return OD_ERR_NULL;
  if (form == OD_READ_INT8 && (!ks_out || !vs_out)) return OD_ERR_NULL;
  if (!od_aligned16(k_out) || !od_aligned16(v_out) || !aligned4(ks_out) || !aligned4(vs_out)) return OD_ERR_ALIGN;
  a.k = k_out;
  a.v = v_out;
  a.ks = ks_out;
  a.vs = vs_out;
  a.T = (int)T;
  const int64_t per_block = kThreads / (D / read_values(form)), tiles = (T + per_block - 1) / per_block;
  if (B * Hkv > kMaxGroups / tiles) return OD_ERR_SHAPE;
  a.tiles = (int)tiles;
  by_head_dim(D, [&](auto DC) {
    constexpr int DD = decltype(DC)::value;
    const dim3 grid((unsigned)(B * Hkv * tiles)), block(kThreads);
    hipStream_t st = (hipStream_t)stream;
    by_format(format, [&](auto PC) {
      constexpr int P = decltype(PC)::value;
      if (form == OD_READ_BF16) page_read_kernel<DD, P, kReadBf16><<<grid, block, 0, st>>>(a);
      else if (form == OD_READ_FP32) page_read_kernel<DD, P, kReadF32><<<grid, block, 0, st>>>(a);
      else if constexpr (P == kInt8) page_read_kernel<DD, P, kReadI8><<<grid, block, 0, st>>>(a);
    });
  });
  return od_launch_status();
}

extern "C" int od_page_read(const void* k_pages, const float* k_scale, const void* v_pages, const float* v_scale,
                            int64_t n_pages, int64_t page, const int32_t* table, int64_t ld_table, int64_t cols,
                            const int32_t* length, int64_t B, int64_t T, int64_t Hkv, int64_t D, int form, void* k_out,
                            float* ks_out, void* v_out, float* vs_out, od_stream_t stream) {
  return od_page_read_ex(k_scale || v_scale ? OD_PAGE_INT8 : OD_PAGE_BF16, k_pages, k_scale, v_pages, v_scale, n_pages, page,
                         table, ld_table, cols, length, B, T, Hkv, D, form, k_out, ks_out, v_out, vs_out, stream);
}

extern "C" int od_paged_attn_ws_ex(int64_t B, int64_t N, int64_t Hq, int64_t Hkv, int64_t D, int64_t max_new,
                                   int64_t max_ctx, int format, int64_t* ws_floats) {
  if (!ws_floats) return OD_ERR_NULL;
  if (B < 0 || N < 0 || Hq < 1 || Hkv < 1 || max_new < 0 || max_ctx < 0) return OD_ERR_SHAPE;
  if (Hq % Hkv || (D != 64 && D != 128 && D != 256)) return OD_ERR_UNSUPPORTED;
  if (format != OD_PAGE_BF16 && format != OD_PAGE_INT8 && format != OD_PAGE_INT4) return OD_ERR_UNSUPPORTED;
  if (B > 65535 || Hq > 65535 || N > kMaxSlots / (Hq / Hkv)) return OD_ERR_SHAPE;
  *ws_floats = B == 0 || N == 0 ? 0 : plan_of(B, N, Hq, Hkv, D, max_new, max_ctx, format).floats();
  return OD_OK;
}

extern "C" int od_paged_attn_ws_of(int64_t B, int64_t N, int64_t Hq, int64_t Hkv, int64_t D, int64_t max_new,
                                   int64_t max_ctx, int int8_pages, int64_t* ws_floats) {
  return od_paged_attn_ws_ex(B, N, Hq, Hkv, D, max_new, max_ctx, int8_pages ? OD_PAGE_INT8 : OD_PAGE_BF16, ws_floats);
}

extern "C" int od_paged_attn_ws(int64_t B, int64_t N, int64_t Hq, int64_t Hkv, int64_t D, int64_t max_new,
                                int64_t max_ctx, int64_t* ws_floats) {
  int64_t n8 = 0;
  if (const int rc = od_paged_attn_ws_of(B, N, Hq, Hkv, D, max_new, max_ctx, 1, &n8)) return rc;
  if (const int rc = od_paged_attn_ws_of(B, N, Hq, Hkv, D, max_new, max_ctx, 0, ws_floats)) return rc;
  if (n8 > *ws_floats) *ws_floats = n8;
  return OD_OK;
}

extern "C" int od_paged_attn_ex(const uint16_t* q, int64_t sqt, int64_t sqh, const uint16_t* k, int64_t skt, int64_t skh,
                                const uint16_t* v, int64_t svt, int64_t svh, int format, const void* k_pages,
                                const void* k_scale, const void* v_pages, const void* v_scale, int64_t n_pages, int64_t page,
                                const int32_t* table, int64_t ld_table, int64_t cols, const int32_t* start,
                                const int32_t* ctx_len, const int32_t* row_begin, uint16_t* out, int64_t sot, int64_t soh,
                                float* lse, int64_t B, int64_t N, int64_t Hq, int64_t Hkv, int64_t D, int64_t max_new,
                                int64_t max_ctx, float scale, float* ws, int64_t ws_floats, od_stream_t stream) {
  AttnArgs a;
  if (const int rc = paged_args(a.p, format, k_pages, k_scale, v_pages, v_scale, n_pages, page, table, ld_table,
                                cols, start, ctx_len, B, N, Hkv, D))
    return rc;
  if (Hq < 1 || Hq > 65535 || B > 65535 || max_new < 0 || max_ctx < 0) return OD_ERR_SHAPE;
  if (Hq >= Hkv && N > kMaxSlots / (Hq / Hkv)) return OD_ERR_SHAPE;
  if (Hq % Hkv || !(scale > 0.0f) || !(scale < INFINITY)) return OD_ERR_UNSUPPORTED;
  if (B == 0 || N == 0) return OD_OK;
  if (!q || !out || !start || !ctx_len || !k != !v || (cols > 0 && !table)) return OD_ERR_NULL;
  const int64_t strides[] = {sqt, sqh, skt, skh, svt, svh, sot, soh};
  for (int64_t s : strides)
    if (s < 0 || s % 8) return OD_ERR_ALIGN;
  if (!od_aligned16(q) || !od_aligned16(k) || !od_aligned16(v) || !od_aligned16(out) || !aligned4(lse))
    return OD_ERR_ALIGN;
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
  const Plan p = plan_of(B, N, Hq, Hkv, D, max_new, max_ctx, format);
  if (p.floats()) {
    if (!ws) return OD_ERR_NULL;
    if (ws_floats < p.floats()) return OD_ERR_SHAPE;
    if (!od_aligned16(ws)) return OD_ERR_ALIGN;
  }
  a.part = ws;
  a.img_vexp = reinterpret_cast<int*>(ws + p.part);
  a.img_heads = reinterpret_cast<ImageBlock*>(ws + p.part + p.vexp);
  a.img = reinterpret_cast<uint16_t*>(ws + p.part + p.vexp + p.heads);
  a.img_blocks = (int)p.img_blocks;
  a.rest = false;
  a.nsplit = p.nsplit;
  a.chunk = p.chunk;
  a.tiles = p.tiles;
  a.run = p.run;
  if (n_pages == 0) a.p.cols = 0;
  hipStream_t st = (hipStream_t)stream;
  // tiles: every run of every group, a multiple of 8 runs
  const int64_t runs = (p.tiles + p.run - 1) / p.run, groups = (p.nsplit * Hkv * B * runs + 7) / 8 * 8 * p.run;
  if (!p.stream && groups * p.nw > 4 * kMaxGroups) return OD_ERR_SHAPE;
  int rc = OD_OK;
  by_head_dim(D, [&](auto DC) {
    constexpr int DD = decltype(DC)::value;
    auto tiles = [&](auto SC) {
      constexpr int SRC = decltype(SC)::value;
      if constexpr (DD == 64) rc = launch_tiles<DD, SRC, 4>(a, (unsigned)groups, st);
      else if constexpr (DD == 256) rc = launch_big<&paged_wide_kernel<SRC>>(a, (unsigned)groups, 512,
          (int)sizeof(WSmem), st);
      else if (p.nw == 8) rc = launch_tiles<DD, SRC, 8>(a, (unsigned)groups, st);
      else rc = launch_tiles<DD, SRC, 4>(a, (unsigned)groups, st);
    };
    auto stream = [&](auto PC) {
      constexpr int P = decltype(PC)::value;
      const dim3 grid((unsigned)p.nsplit, (unsigned)(Hkv * p.tiles), (unsigned)B);
      if (p.ct == 1 && p.waves < s_waves(DD, P, 1)) {
        if constexpr (P == kInt4 && DD == 256) paged_stream_kernel<DD, P, 1, 1><<<grid, dim3(kStreamWaves * 64), 0, st>>>(a);
      } else if (p.ct == 1) paged_stream_kernel<DD, P, 1><<<grid, dim3(kStreamWaves * 64), 0, st>>>(a);
      else paged_stream_kernel<DD, P, 2><<<grid, dim3(kStreamWaves * 64), 0, st>>>(a);
    };
    if (p.stream) {
      by_format(format, stream);
    } else if (format == OD_PAGE_BF16) {
      tiles(std::integral_constant<int, kBf16>{});
    } else {
      by_format(format, [&](auto PC) {
        constexpr int P = decltype(PC)::value;
        if constexpr (P != kBf16) {
          if (p.img_blocks) {
            const dim3 grid((unsigned)p.img_blocks, (unsigned)Hkv, (unsigned)B);
            page_frame_kernel<DD, P><<<dim3((unsigned)((p.img_blocks + 3) / 4), grid.y, grid.z), dim3(kThreads), 0, st>>>(a);
            page_image_kernel<DD, P><<<grid, dim3(kThreads), 0, st>>>(a);
            tiles(std::integral_constant<int, kImage>{});
            a.rest = true;
          }
          // the sequences without an image, if there can be any
          if (rc == OD_OK && (p.img_blocks == 0 || p.img_blocks * kBK < ((int64_t)a.p.cols << a.p.shift))) tiles(PC);
        }
      });
    }
    if (rc == OD_OK && p.nsplit > 1) {
      // groups when a workgroup has one slot; slots when a slot has one group
      constexpr int S = 4 * kThreads / DD, SL = S;
      const dim3 one((unsigned)N, (unsigned)Hq), many((unsigned)N, (unsigned)((Hq + SL - 1) / SL)), block(kThreads);
      if (p.nsplit > 4) paged_combine_kernel<DD, S><<<one, block, 0, st>>>(a, p.width);
      else paged_combine_kernel<DD, 1><<<many, block, 0, st>>>(a, p.width);
    }
  });
  return rc == OD_OK ? od_launch_status() : rc;
}

extern "C" int od_paged_attn(const uint16_t* q, int64_t sqt, int64_t sqh, const uint16_t* k, int64_t skt, int64_t skh,
                             const uint16_t* v, int64_t svt, int64_t svh, const void* k_pages, const float* k_scale,
                             const void* v_pages, const float* v_scale, int64_t n_pages, int64_t page,
                             const int32_t* table, int64_t ld_table, int64_t cols, const int32_t* start,
                             const int32_t* ctx_len, const int32_t* row_begin, uint16_t* out, int64_t sot, int64_t soh,
                             float* lse, int64_t B, int64_t N, int64_t Hq, int64_t Hkv, int64_t D, int64_t max_new,
                             int64_t max_ctx, float scale, float* ws, int64_t ws_floats, od_stream_t stream) {
  return od_paged_attn_ex(q, sqt, sqh, k, skt, skh, v, svt, svh, k_scale || v_scale ? OD_PAGE_INT8 : OD_PAGE_BF16, k_pages,
                          k_scale, v_pages, v_scale, n_pages, page, table, ld_table, cols, start, ctx_len, row_begin, out, sot,
                          soh, lse, B, N, Hq, Hkv, D, max_new, max_ctx, scale, ws, ws_floats, stream);
}
