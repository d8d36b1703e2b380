// Linears with 4-bit weights, for gfx950: out[m, n] = bf16(sum_k x[m, k] W[n, k] (+ bias[n]) (+ residual[m, n])), x in bf16, W in
// blocks of 32 along a row, (u - 8) d with u in 0 .. 15 and one fp16 d a block (a block's 16 bytes: values 0 - 15 in the low
// halves, 16 - 31 in the high ones; src/opendecider/quant.py:206-246).
#include <type_traits>

#include "od_common.h"

namespace {

typedef uint32_t v4u __attribute__((ext_vector_type(4)));
typedef float v4f __attribute__((ext_vector_type(4)));
typedef float v16f __attribute__((ext_vector_type(16)));
typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));
typedef _Float16 f16x8 __attribute__((ext_vector_type(8)));
typedef _Float16 f16x2 __attribute__((ext_vector_type(2)));

struct Q4Args {
  const uint16_t* x;
  const uint8_t* qs;
  const uint16_t* d;
  const uint16_t* bias;      // [N] or null
  const uint16_t* residual;  // [M, N] or null
  uint16_t* out;
  int64_t ldx, ldq, ldd, ldr, ldo;
  int64_t M, N, K;
  // many rows: x in fp16 frames, the frames' exponents, the splits' sums
  uint16_t* x16;
  int* xexp;
  float* part;
  int64_t Kp;  // K in whole stages
  int tiles_m, tiles_n, nsplit, stages, bm;  // bm: the rows of a tile of x
  // few rows: the turns of steps whose x lies in LDS at a time; 2^20 / (4 rows of x), rounded up
  int held, per20;
};

__device__ __forceinline__ __amdgpu_buffer_rsrc_t rsrc(const void* p, int64_t bytes) {
  return __builtin_amdgcn_make_buffer_rsrc(const_cast<void*>(p), (short)0, (int)bytes, 0x00020000);
}

// ------------------------------------------------------------------------------------------------ few rows of x
// Bound by reading the weights. V_MFMA_F32_16X16X32_BF16 with 16 weight rows as the A operand and up to 16 rows of x as the B
// operand, 32 values a time, which is one block: the sums of a block, exact in their products, take the fp32 factor d afterwards,
// so no weight is rounded. A step of a wave is 4 blocks of 16 weight rows (64 contiguous bytes of each). Lane (j, g) = (lane % 16,
// lane / 16):
//  * reads block 4 s + g of weight row j, 16 bytes; four lane exchanges (a transposition over g) give it word g of each of the
//    four blocks: values 4 g .. 4 g + 3 and 16 + 4 g .. + 3 of the block;
//  * four bits u at the bottom of 128.0's bf16 are 128 + u: one shift and one and-or for two values. The 136 that it is above
//    u - 8 leaves by the C operand, -136 times the sum of x over the block, itself a product with a constant A. (A row of x that
//    holds an infinity or NaN so becomes NaN. The block's fp32 sums are of up to 143 |x| a value for the 8 |x| that are left: their
//    roundings are some seven bits more than of the plain sums, 2^-17 of |x| d a value, far below the output's 2^-8 unless x is
//    thousands of times larger where the weights are near 0 than elsewhere.)
//  * holds weight rows 4 g + i of column j of the result; d of row 4 g + i and block b is the one that lane 16 g + 4 i + b loaded.
// A workgroup's WR x WK waves take WR sets of RT row tiles, WK of them every WK-th step of one, and add up in LDS. x lies in LDS in
// the order of the B operand, as many steps of it as fit at a time, two buffers of it; the weights of the PD next steps are in
// registers or on their way meanwhile, whatever the workgroup waits for. One row of x, in a captured graph: 4096 x
// 4096 6.3 us (9.4 MB; an eager call takes the host 9.5), 24576 x 4096 19.9 us (2.8 TB/s), 151936 x 4096 88 us (4.0 TB/s); 24 rows over
// 24576 x 4096 27.4 us, where x, staged by every workgroup, is as much as the weights.
typedef uint32_t v2u __attribute__((ext_vector_type(2)));

__device__ __forceinline__ v4f mfma16(v4u a, v4u b, v4f c) {
  return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8, a), __builtin_bit_cast(bf16x8, b), c, 0, 0, 0);
}
// word w of block g in lane row g -> word g of block w
__device__ __forceinline__ void transpose4(v4u& w) {
  const auto a = __builtin_amdgcn_permlane32_swap(w[0], w[2], false, false), b = __builtin_amdgcn_permlane32_swap(w[1], w[3], false, false);
  const auto c = __builtin_amdgcn_permlane16_swap(a[0], b[0], false, false), e = __builtin_amdgcn_permlane16_swap(a[1], b[1], false, false);
  w = v4u{c[0], c[1], e[0], e[1]};
}
// 8 values as bf16 128 + u, in the order 0 2 16 18 1 3 17 19 (from 4 g); base: 128 in both halves, from a vector register (the
// and-or takes one scalar operand, which is the mask)
__device__ __forceinline__ v4u raised(uint32_t t, uint32_t base) {
  v4u r;
#pragma unroll
  for (int i = 0; i < 4; ++i) r[i] = ((t >> (4 * i)) & 0x000f000fu) | base;
  return r;
}
// x in that order
__device__ __forceinline__ v4u ordered(v2u a, v2u b) {
  return v4u{__builtin_amdgcn_perm(a[1], a[0], 0x05040100u), __builtin_amdgcn_perm(b[1], b[0], 0x05040100u),
             __builtin_amdgcn_perm(a[1], a[0], 0x07060302u), __builtin_amdgcn_perm(b[1], b[0], 0x07060302u)};
}
// lane N of each row of 16, in all of them
template <int N>
__device__ __forceinline__ float row_lane(float v) {
  return __int_as_float(__builtin_amdgcn_update_dpp(0, __float_as_int(v), 0x150 + N, 0xf, 0xf, true));
}

template <int RT>
struct Q4Step {
  v4u w[RT];
  uint32_t d[RT];
};

__device__ __forceinline__ void q4_store(const Q4Args& a, int64_t m, int64_t n, v4f y) {
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    if (n + i >= a.N) continue;
    if (a.bias) y[i] += od_bf16_to_f32(a.bias[n + i]);
    if (a.residual) y[i] += od_bf16_to_f32(a.residual[m * a.ldr + n + i]);
  }
  uint16_t* at = a.out + m * a.ldo + n;
  if (n + 3 < a.N && (reinterpret_cast<uintptr_t>(at) & 7u) == 0) {
    *reinterpret_cast<uint2*>(at) = make_uint2(od_pack_bf16x2(y[0], y[1]), od_pack_bf16x2(y[2], y[3]));
  } else {
#pragma unroll
    for (int i = 0; i < 4; ++i)
      if (n + i < a.N) at[i] = od_f32_to_bf16(y[i]);
  }
}

// A buffer of x in LDS holds up to 2048 units of 8 values. A unit's tokens lie 16 bytes apart, its rows (tokens | 1) times that: the
// four that a token writes, or reads, at once are in other banks.
constexpr int kXUnits = 2048, kXBytes = 16 * kXUnits / 16 * 17;

template <int RT, int CT, int WK, int WR, int PD>
__global__ __launch_bounds__(WK * WR * 64) void q4_rows_kernel(Q4Args a) {
  constexpr int NT = WK * WR * 64;
  extern __shared__ __attribute__((aligned(16))) char lds_x[];  // x: [step][block][g][token] 16 bytes; at the end the waves' sums
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), j = lane & 15, g = lane >> 4;
  const int wr = wave / WK, wk = wave % WK;
  const int64_t n0 = ((int64_t)blockIdx.x * WR + wr) * (16 * RT);
  const int rows = (int)max(min((int64_t)16 * RT, a.N - n0), (int64_t)0), toks = (int)a.M;
  const int blocks = (int)(a.K / 32), steps = (blocks + 3) / 4, turns = (steps + WK - 1) / WK;
  const auto none = rsrc(a.x, 0);
  const auto rw = rows ? rsrc(a.qs + n0 * a.ldq, (rows - 1) * a.ldq + a.K / 2) : none;
  const auto rd = rows ? rsrc(a.d + n0 * a.ldd, ((rows - 1) * a.ldd + blocks) * 2) : none;
  const int wo = (int)(j * a.ldq) + 16 * g, dofs = 2 * (int)((lane >> 2) * a.ldd + (lane & 3));
  auto load = [&](int turn, Q4Step<RT>& t) {  // past the last step: nothing is read
    const int s = turn * WK + wk;
    const bool in = s < steps;
#pragma unroll
    for (int r = 0; r < RT; ++r) {
      t.w[r] = __builtin_bit_cast(v4u, __builtin_amdgcn_raw_buffer_load_b128(in ? rw : none, wo + (int)(16 * r * a.ldq), 64 * s, 2));
      t.d[r] = (uint16_t)__builtin_amdgcn_raw_buffer_load_b16(in ? rd : none, dofs + (int)(32 * r * a.ldd), 8 * s, 0);
    }
    __builtin_amdgcn_sched_barrier(0);
  };
  Q4Step<RT> t[PD];
#pragma unroll
  for (int i = 0; i < PD; ++i) load(i, t[i]);

  // x in chunks of `held` turns, in units of 8 values of a row (block, token, g). The next chunk's units are in registers while one
  // is multiplied.
  constexpr int UX = kXUnits / NT;
  const int held = a.held, units = held * WK * 16 * toks, tp = toks | 1;
  const auto rx = rsrc(a.x, ((toks - 1) * a.ldx + a.K) * 2);
  int from[UX], to[UX], at_block[UX];  // a unit's offset in x in bytes, its place in LDS (below 0: none), its block of a chunk
#pragma unroll
  for (int i = 0; i < UX; ++i) {
    const int u = i * NT + threadIdx.x, blk = (int)((uint32_t)u * (uint32_t)a.per20 >> 20);  // u / (4 toks): u < 2^11, toks <= 2^5
    const int tok = u / 4 - blk * toks, ug = u & 3;
    from[i] = (int)(tok * a.ldx * 2) + 64 * blk + 8 * ug;
    to[i] = u < units ? 16 * ((4 * blk + ug) * tp + tok) : -1;
    at_block[i] = u < units ? blk : 1 << 30;
  }
  v2u xa[UX], xb[UX];
  auto fetch = [&](int chunk) {
#pragma unroll
    for (int i = 0; i < UX; ++i) {
      const int at = chunk * (held * WK * 4) + at_block[i] < blocks ? from[i] : (int)0x80000000;  // (past the end: zeros)
      xa[i] = __builtin_bit_cast(v2u, __builtin_amdgcn_raw_buffer_load_b64(rx, at, chunk * (held * WK * 256), 0));
      xb[i] = __builtin_bit_cast(v2u, __builtin_amdgcn_raw_buffer_load_b64(rx, at + 32, chunk * (held * WK * 256), 0));
    }
    __builtin_amdgcn_sched_barrier(0);
  };
  auto put = [&](int chunk) {
#pragma unroll
    for (int i = 0; i < UX; ++i)
      if (to[i] >= 0) *reinterpret_cast<v4u*>(lds_x + (chunk & 1) * kXBytes + to[i]) = ordered(xa[i], xb[i]);
  };
  v4f acc[RT][CT];
#pragma unroll
  for (auto& r : acc)
#pragma unroll
    for (auto& c : r) c = v4f{0, 0, 0, 0};
  const v4u down = {0xc308c308u, 0xc308c308u, 0xc308c308u, 0xc308c308u};  // -136
  int mine[CT];  // the lane's row of x (a row past the last one: the last, its result is left out)
#pragma unroll
  for (int c = 0; c < CT; ++c) mine[c] = 16 * (g * tp + min(16 * c + j, toks - 1));
  uint32_t base = 0x43004300u;
  asm("" : "+v"(base));
  auto compute = [&](int turn, int buf, int in_lds, Q4Step<RT>& t) {
    const int s = turn * WK + wk;
    float d[RT];
#pragma unroll
    for (int r = 0; r < RT; ++r) {
      transpose4(t.w[r]);
      // (past the row's last block lies the next row's first one)
      d[r] = 4 * s + (lane & 3) < blocks ? (float)__builtin_bit_cast(_Float16, (uint16_t)t.d[r]) : 0.0f;
    }
    const char* xs = lds_x + buf + (in_lds * WK + wk) * (256 * tp);
    auto block = [&](auto B) {
      constexpr int b = decltype(B)::value;
      v4u x[CT];
      v4f off[CT];
#pragma unroll
      for (int c = 0; c < CT; ++c) {
        x[c] = *reinterpret_cast<const v4u*>(xs + b * 64 * tp + mine[c]);
        off[c] = mfma16(down, x[c], v4f{0, 0, 0, 0});
      }
#pragma unroll
      for (int r = 0; r < RT; ++r) {
        const v4u w = raised(t.w[r][b], base);
        const float d0 = row_lane<b>(d[r]), d1 = row_lane<4 + b>(d[r]), d2 = row_lane<8 + b>(d[r]), d3 = row_lane<12 + b>(d[r]);
#pragma unroll
        for (int c = 0; c < CT; ++c) {
          const v4f p = mfma16(w, x[c], off[c]);
          acc[r][c][0] = __builtin_fmaf(d0, p[0], acc[r][c][0]);
          acc[r][c][1] = __builtin_fmaf(d1, p[1], acc[r][c][1]);
          acc[r][c][2] = __builtin_fmaf(d2, p[2], acc[r][c][2]);
          acc[r][c][3] = __builtin_fmaf(d3, p[3], acc[r][c][3]);
        }
      }
    };
    block(std::integral_constant<int, 0>{});
    block(std::integral_constant<int, 1>{});
    block(std::integral_constant<int, 2>{});
    block(std::integral_constant<int, 3>{});
  };
  int in_lds = held, chunk = -1;  // every wave of a workgroup takes the same turns
  fetch(0);
  for (int turn = 0; turn < turns; turn += PD) {
#pragma unroll
    for (int i = 0; i < PD; ++i) {
      if (turn + i >= turns) break;
      if (in_lds == held) {  // (the buffer's readers, of the chunk before the last, are past a barrier)
        ++chunk;
        put(chunk);
        __syncthreads();
        if (turn + i + held < turns) fetch(chunk + 1);
        in_lds = 0;
      }
      if ((turn + i) * WK + wk < steps) compute(turn + i, (chunk & 1) * kXBytes, in_lds, t[i]);
      ++in_lds;
      load(turn + i + PD, t[i]);
    }
  }
  constexpr int T = RT * CT;
  __syncthreads();
  float4* red = reinterpret_cast<float4*>(lds_x);
#pragma unroll
  for (int i = 0; i < T; ++i) {
    const v4f v = acc[i / CT][i % CT];
    red[(wave * T + i) * 64 + lane] = make_float4(v[0], v[1], v[2], v[3]);
  }
  __syncthreads();
  for (int i = threadIdx.x; i < WR * T * 64; i += NT) {
    const int tile = i / (T * 64), c = i / 64 % T, l = i & 63;
    v4f y = v4f{0, 0, 0, 0};
#pragma unroll
    for (int w = 0; w < WK; ++w) {
      const float4 v = red[((tile * WK + w) * T + c) * 64 + l];
      y += v4f{v.x, v.y, v.z, v.w};
    }
    const int64_t m = 16 * (c % CT) + (l & 15), n = (((int64_t)blockIdx.x * WR + tile) * RT + c / CT) * 16 + 4 * (l >> 4);
    if (m < a.M && n < a.N) q4_store(a, m, n, y);
  }
}

// ------------------------------------------------------------------------------------------------ many rows of x
// Matrix products of tiles. x goes to fp16 once, each row in a power-of-two frame (2^(14 - e), 2^e above its largest value: exact
// but for values below 2^-29 of it, which move by 2^-38 of it at most), zero-padded to whole stages, in tiles that lie in memory as
// they do in LDS, the values of a block in the order in which its weights come out of the conversion. Weights become (u - 8) d in
// fp16 in the registers that multiply them: one rounding, 2^-11 at most (so |W| up to 65504, fp16's range). A row of x that holds
// an infinity or NaN is NaN. (The pass over x reads a row twice, the second time past the L2 as well: 2000 x
// 12288 in 22 us, 96 MB read and 48 written.)
constexpr int kXThreads = 256, BK = 64, kStageBytes = 2 * BK;  // values, and bytes of a row of x, in a stage
__global__ __launch_bounds__(kXThreads) void q4_x_kernel(Q4Args a) {
  __shared__ uint32_t red[kXThreads / 64];
  const int64_t m = blockIdx.x;
  const uint16_t* row = a.x + m * a.ldx;
  const int words = (int)(a.K / 8);  // words of 8 values
  uint32_t am = 0;
  for (int i = threadIdx.x; i < words; i += kXThreads) {
    const uint4 u = *reinterpret_cast<const uint4*>(row + 8 * i);
    am = od_absmax_bf16x2(od_absmax_bf16x2(od_absmax_bf16x2(od_absmax_bf16x2(am, u.x), u.y), u.z), u.w);
  }
  am = od_wave_umax_dpp(max(am & 0xffffu, am >> 16));
  if ((threadIdx.x & 63) == 0) red[threadIdx.x >> 6] = am;
  __syncthreads();
#pragma unroll
  for (int w = 0; w < kXThreads / 64; ++w) am = max(am, red[w]);
  const bool odd = am >= 0x7f80u;
  const int e = am && !odd ? (int)(am >> 7) - 126 : 0;
  if (threadIdx.x == 0) a.xexp[m] = e;
  const int r = (int)(m % a.bm);
  char* at16 = reinterpret_cast<char*>(a.x16) + m / a.bm * a.bm * a.Kp * 2 + r * kStageBytes;
  // chunk c of a block: values 4 c, 4 c + 2, 16 + 4 c, 16 + 4 c + 2, 4 c + 1, 4 c + 3, 16 + 4 c + 1, 16 + 4 c + 3
  for (int i = threadIdx.x; i < a.Kp / 8; i += kXThreads) {
    uint4 o = make_uint4(0, 0, 0, 0);
    if (i < words) {
      const uint16_t* at = row + 32 * (i / 4) + 4 * (i % 4);
      const uint2 lo = *reinterpret_cast<const uint2*>(at), hi = *reinterpret_cast<const uint2*>(at + 16);
      auto pair = [&](uint32_t w0, uint32_t w1, bool high) {  // the low, or high, halves of two words
        const uint32_t p = high ? w0 & 0xffff0000u : w0 << 16, q = high ? w1 & 0xffff0000u : w1 << 16;
        const f16x2 r = {(_Float16)__builtin_ldexpf(__uint_as_float(p), 14 - e), (_Float16)__builtin_ldexpf(__uint_as_float(q), 14 - e)};
        return odd ? 0x7e007e00u : __builtin_bit_cast(uint32_t, r);
      };
      o = make_uint4(pair(lo.x, lo.y, false), pair(hi.x, hi.y, false), pair(lo.x, lo.y, true), pair(hi.x, hi.y, true));
    }
    *reinterpret_cast<uint4*>(at16 + (int64_t)(i / 8) * a.bm * kStageBytes + 16 * ((i % 8) ^ (r / 2 & 7))) = o;
  }
}

constexpr int kThreads = 256;

// Word I of 8 values (u - 8) d in fp16, each rounded once: u - 8 from 1024 + u, or 16 (u - 8) from 1024 + 16 u, times d or d / 16
// (raised: 1024 in both halves, from a vector register).
__device__ __forceinline__ uint32_t q4_f16(int i, uint32_t w, f16x2 d, uint32_t raised) {
  const f16x2 base = {(_Float16)-1032.0f, (_Float16)-1032.0f}, base16 = {(_Float16)-72.0f, (_Float16)-72.0f},
              sixteenth = {(_Float16)0.0625f, (_Float16)0.0625f};
  const uint32_t s = i < 2 ? w : w >> 8;
  const f16x2 u = __builtin_bit_cast(f16x2, (s & (i & 1 ? 0x00f000f0u : 0x000f000fu)) | raised);
  const f16x2 n = i & 1 ? __builtin_elementwise_fma(u, sixteenth, base16) : u + base;
  return __builtin_bit_cast(uint32_t, n * d);
}

// A tile of 32 MT rows of x by 256 weight rows, by 4 waves of 32 MT by 64. x goes through LDS, two stages of 64 values of it, by DMA,
// its 16-byte chunks swizzled by row / 2. The weights go straight into the registers of the lanes that multiply them: lane (r, h)
// of V_MFMA_F32_32X32X16_F16 takes block 2 s + h of weight row r, one 16-byte load, whose four words make the A operands of four
// instructions (word t of two blocks each; chunk t of x's two blocks is their B operand), so they cost no LDS traffic. They are
// asked for two stages ahead. 2000 rows over 4096 x 12288: 223 us (900 TF/s), 8000 over 24576 x 4096 1.66 ms (970 TF/s). What it
// waits for is memory, the 32 bytes of a row that a stage takes of a 128-byte line above all (with the loads of the weights
// and d on one line: 200 and 1.40 ms; with x's as well 178 us), and the products' own rate. (Asking for two stages' weights at
// once, so that the second finds its line in the cache, takes as long.)
constexpr int NT = 2, BN = 256;
template <int MT>
__global__ __launch_bounds__(kThreads, 1) void q4_tile_kernel(Q4Args p) {
  constexpr int BM = 32 * MT, kStage = BM * kStageBytes, LD = MT;  // LD: 1 KB copies of a wave a stage
  extern __shared__ __attribute__((aligned(16))) char lds[];
  // flat ids are dealt round-robin over the 8 XCDs; id = the XCD's contiguous range; row tiles fastest
  const int ntiles = p.tiles_m * p.tiles_n * p.nsplit;
  const int f = blockIdx.x, xcd = f & 7, local = f >> 3, per = ntiles >> 3, rem = ntiles & 7;
  const int id = xcd < rem ? xcd * (per + 1) + local : rem * (per + 1) + (xcd - rem) * per + local;
  const int tm = id % p.tiles_m, tn = id / p.tiles_m % p.tiles_n, sp = id / p.tiles_m / p.tiles_n;
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int64_t m0 = (int64_t)tm * BM, n0 = (int64_t)tn * BN + wave * (32 * NT);
  const int all = (int)(p.Kp / BK), k_lo = sp * p.stages, nk = min(p.stages, all - k_lo);
  const int col = lane & 31, h = lane >> 5, blocks = (int)(p.K / 32);

  // weights: rows past N read as zeros
  const int rows = (int)max(min((int64_t)32 * NT, p.N - n0), (int64_t)0);
  const auto none = rsrc(p.x16, 0);
  const auto rb = rows ? rsrc(p.qs + n0 * p.ldq, (rows - 1) * p.ldq + p.K / 2) : none;
  const auto rd = rows ? rsrc(p.d + n0 * p.ldd, ((rows - 1) * p.ldd + blocks) * 2) : none;
  const int b_vo = (int)(col * p.ldq) + 16 * h, d_vo = 2 * (int)(col * p.ldd + h);
  struct Raw {
    v4u w[NT];
    uint32_t d[NT];
  };
  auto load_w = [&](int j, int kt, Raw& r) {
    const int k = k_lo + kt;
    r.w[j] = __builtin_bit_cast(v4u, __builtin_amdgcn_raw_buffer_load_b128(kt < nk ? rb : none, b_vo + (int)(32 * j * p.ldq), 32 * k, 0));
    r.d[j] = (uint16_t)__builtin_amdgcn_raw_buffer_load_b16(kt < nk ? rd : none, d_vo + (int)(64 * j * p.ldd), 4 * k, 0);
  };
  auto load_w_all = [&](int kt, Raw& r) {
#pragma unroll
    for (int j = 0; j < NT; ++j) load_w(j, kt, r);
    __builtin_amdgcn_sched_barrier(0);
  };
  auto wait_w = [&](Raw& r) {
#pragma unroll
    for (int j = 0; j < NT; ++j) asm volatile("" : "+v"(r.w[j]), "+v"(r.d[j]));
  };
  // x: copy i of a wave is its i-th KB of every four; a stage of a tile lies in memory as it does in LDS
  const char* x_at = reinterpret_cast<const char*>(p.x16) + (int64_t)tm * BM * p.Kp * 2 + (int64_t)k_lo * kStage;
  auto copy_x = [&](int i, int kt, int to) {
    od_dma16_at(x_at + (int64_t)min(kt, nk - 1) * kStage + 1024 * (4 * i + wave), 16 * lane, od_lds_addr(lds) + to + 1024 * (4 * i + wave));
  };
  // chunk 4 h + t of row 32 i + col
  const int x_sw = (col >> 1) & 7;  // (32 i is a multiple of 16)
  auto frag_x = [&](int at, int t, int i) {
    return *reinterpret_cast<const v4u*>(lds + at + (col + 32 * i) * kStageBytes + (((4 * h + t) ^ x_sw) << 4));
  };
  uint32_t raised = 0x64006400u;
  asm("" : "+v"(raised));
  f16x2 d2[NT];
  auto scales = [&](int kt, const Raw& r) {  // (past the row's last block lies the next row's first one)
    const bool in = 2 * (k_lo + kt) + h < blocks;
#pragma unroll
    for (int j = 0; j < NT; ++j) {
      const _Float16 d = __builtin_bit_cast(_Float16, (uint16_t)(in ? r.d[j] : 0u));
      d2[j] = f16x2{d, d};
    }
  };
  v16f acc[NT][MT];
#pragma unroll
  for (auto& r : acc)
#pragma unroll
    for (auto& c : r) c = v16f{0, 0, 0, 0, 0, 0, 0, 0, 0, 0, 0, 0, 0, 0, 0, 0};

  // A stage is four steps of MT NT products; the next step's operands are made between them. Before the last step the next stage's
  // x has to be there and everyone done reading this one's: the one wait and barrier of a stage. (The compiler does not see the
  // copies: its own wait for raw weights counts the loads alone, so a stage's copies go before its loads.)
  Raw raw[3];
  v4u fx[2][MT], fw[2][NT];
  constexpr int kSlots = MT * NT, kWords = 4 * NT;
  auto step = [&](auto T, int at, const Raw& next, auto between) {  // products of step T; operands of step T + 1, x of it at `at`
    constexpr int t = decltype(T)::value, cur = t & 1, t1 = (t + 1) & 3;
#pragma unroll
    for (int s = 0; s < kSlots; ++s) {
      const int j = s / MT, i = s % MT;
      acc[j][i] = __builtin_amdgcn_mfma_f32_32x32x16_f16(__builtin_bit_cast(f16x8, fw[cur][j]),
                                                         __builtin_bit_cast(f16x8, fx[cur][i]), acc[j][i], 0, 0, 0);
      if (s < MT) fx[cur ^ 1][s] = frag_x(at, t1, s);
#pragma unroll
      for (int w = s * kWords / kSlots; w < (s + 1) * kWords / kSlots; ++w)
        fw[cur ^ 1][w / 4][w % 4] = q4_f16(w % 4, next.w[w / 4][t1], d2[w / 4], raised);
      between(s);
      __builtin_amdgcn_sched_barrier(0);
    }
  };
  auto nothing = [](int) {};
  int here = 0, there = kStage;
  auto stage = [&](int kt, Raw& r, Raw& r1) {
    step(std::integral_constant<int, 0>{}, here, r, nothing);
    step(std::integral_constant<int, 1>{}, here, r, nothing);
    step(std::integral_constant<int, 2>{}, here, r, nothing);
    asm volatile("s_waitcnt vmcnt(%0) lgkmcnt(0)\n\ts_barrier" ::"i"(2 * NT) : "memory");
    wait_w(r1);
    scales(kt + 1, r1);
    step(std::integral_constant<int, 3>{}, there, r1, [&](int s) {
#pragma unroll
      for (int c = s * (LD + NT) / kSlots; c < (s + 1) * (LD + NT) / kSlots; ++c) {
        if (c < LD) {
          copy_x(c, kt + 2, here);
        } else {
          load_w(c - LD, kt + 3, r);
        }
      }
    });
    const int o = here;
    here = there;
    there = o;
  };
#pragma unroll
  for (int i = 0; i < 2; ++i) {
#pragma unroll
    for (int c = 0; c < LD; ++c) copy_x(c, i, i * kStage);
    __builtin_amdgcn_sched_barrier(0);
    if (i == 0) load_w_all(0, raw[0]), load_w_all(1, raw[1]);
  }
  load_w_all(2, raw[2]);
  asm volatile("s_waitcnt vmcnt(%0)\n\ts_barrier" ::"i"(2 * NT) : "memory");
  wait_w(raw[0]);
  scales(0, raw[0]);
#pragma unroll
  for (int i = 0; i < MT; ++i) fx[0][i] = frag_x(0, 0, i);
#pragma unroll
  for (int w = 0; w < kWords; ++w) fw[0][w / 4][w % 4] = q4_f16(w % 4, raw[0].w[w / 4][0], d2[w / 4], raised);
  __builtin_amdgcn_sched_barrier(0);
  for (int kt = 0; kt < nk; kt += 3) {
    stage(kt, raw[0], raw[1]);
    if (kt + 1 < nk) stage(kt + 1, raw[1], raw[2]);
    if (kt + 2 < nk) stage(kt + 2, raw[2], raw[0]);
  }
  asm volatile("s_waitcnt vmcnt(0)" ::: "memory");  // (copies of a stage past the last one may be on their way)
  // lane: row lane % 32 of x, weight rows 8 (r / 4) + 4 (lane / 32) + r % 4 of the tile's 32
#pragma unroll
  for (int i = 0; i < MT; ++i) {
    const int64_t m = m0 + i * 32 + col;
    if (m >= p.M) continue;
    const int e = p.xexp[m];
    const float unit = __builtin_ldexpf(1.0f, e / 2 - 7), unit2 = __builtin_ldexpf(1.0f, e - e / 2 - 7);
#pragma unroll
    for (int j = 0; j < NT; ++j)
#pragma unroll
      for (int q = 0; q < 4; ++q) {
        const int64_t n = n0 + j * 32 + 8 * q + 4 * h;
        if (n >= p.N) continue;
        v4f y = v4f{acc[j][i][4 * q], acc[j][i][4 * q + 1], acc[j][i][4 * q + 2], acc[j][i][4 * q + 3]};
        y = y * unit * unit2;
        if (p.nsplit == 1) {
          q4_store(p, m, n, y);
        } else {  // rows of a multiple of 4 columns
          *reinterpret_cast<v4f*>(p.part + ((int64_t)sp * p.M + m) * ((p.N + 3) / 4 * 4) + n) = y;
        }
      }
  }
}

__global__ __launch_bounds__(256) void q4_sum_kernel(Q4Args p) {
  const int64_t N4 = (p.N + 3) / 4, i = (int64_t)blockIdx.x * 256 + threadIdx.x;
  if (i >= p.M * N4) return;
  const int64_t m = i / N4, n = 4 * (i % N4);
  v4f y = v4f{0, 0, 0, 0};
  for (int s = 0; s < p.nsplit; ++s) y += *reinterpret_cast<const v4f*>(p.part + ((int64_t)s * p.M + m) * (4 * N4) + n);
  q4_store(p, m, n, y);
}

// Up to 32 rows take the first kernel, above it the tiles: 24576 x 4096, 32 rows 29 against 45 us, 64 rows 46 (by 64 rows of x
// at a time) against 45; 4096 x 4096, 32 rows 15 against 20, 64 rows 44 against 23.
constexpr int64_t kFewRows = 32;

struct Q4Plan {
  int bm, nsplit, stages;
  int64_t Kp, tiles_m, tiles_n, xexp, x16, part;  // the workspace, in floats
  int64_t floats() const { return xexp + x16 + part; }
};
Q4Plan q4_plan(int64_t M, int64_t N, int64_t K) {
  Q4Plan q = {};
  if (M <= kFewRows) return q;
  q.Kp = (K + BK - 1) / BK * BK;
  q.bm = M <= 64 ? 64 : 128;
  q.tiles_m = (M + q.bm - 1) / q.bm;
  q.tiles_n = (N + BN - 1) / BN;
  // K is split for two workgroups a CU, of 8 stages at least: 2000 rows over 4096 x 12288 (256 tiles) 245 us in two parts, 266 in
  // one; 300 rows 74 in five, 125 in two, 228 in one
  const int64_t all = q.Kp / BK;
  int64_t n = 2 * od_cu_count() / (q.tiles_m * q.tiles_n);
  if (n > all / 8) n = all / 8;
  if (n < 1) n = 1;
  q.stages = (int)((all + n - 1) / n);
  q.nsplit = (int)((all + q.stages - 1) / q.stages);
  q.xexp = (M + 3) / 4 * 4;
  q.x16 = q.tiles_m * q.bm * q.Kp / 2;
  q.part = q.nsplit > 1 ? q.nsplit * M * ((N + 3) / 4 * 4) : 0;
  return q;
}

bool q4_sizes_ok(int64_t M, int64_t N, int64_t K) {
  return M >= 0 && N >= 1 && K >= 32 && K % 32 == 0 && M <= (1ll << 22) && N <= (1ll << 24) && K <= (1ll << 20);
}

// Dynamic LDS above 64 KB, which a kernel has to be allowed once per device.
int allow_lds(const void* kernel, int bytes, std::atomic<uint64_t>& allowed) {
  int dev = 0;
  if (hipGetDevice(&dev) != hipSuccess || dev < 0 || dev >= 64) return OD_ERR_LAUNCH;
  if (!((allowed.load(std::memory_order_relaxed) >> dev) & 1)) {
    if (hipFuncSetAttribute(kernel, hipFuncAttributeMaxDynamicSharedMemorySize, bytes) != hipSuccess) return OD_ERR_LAUNCH;
    allowed.fetch_or(1ull << dev, std::memory_order_relaxed);
  }
  return OD_OK;
}

template <int RT, int CT, int WK, int WR, int PD>
int launch_rows(Q4Args& a, hipStream_t st) {
  static std::atomic<uint64_t> allowed{0};
  static_assert(16 * CT * 16 * WK <= kXUnits, "a turn's x fits a buffer");
  const int64_t toks = a.M, turn = 256 * (toks | 1) * WK, turns = (a.K / 32 + 4 * WK - 1) / (4 * WK);  // M <= 16 CT
  int64_t held = kXUnits / (16 * toks * WK);
  if (held * turn > kXBytes) held = kXBytes / turn;
  if (held > turns) held = turns;
  constexpr int64_t sums = (int64_t)WK * WR * RT * CT * 1024;
  int64_t bytes = held < turns ? 2 * kXBytes : held * turn;
  if (bytes < sums) bytes = sums;
  if (bytes > 65536) {
    if (const int rc = allow_lds(reinterpret_cast<const void*>(q4_rows_kernel<RT, CT, WK, WR, PD>), 160 << 10, allowed)) return rc;
  }
  a.held = (int)held;
  a.per20 = (int)(((1 << 20) + 4 * toks - 1) / (4 * toks));
  const unsigned groups = (unsigned)((a.N + 16 * RT * WR - 1) / (16 * RT * WR));
  q4_rows_kernel<RT, CT, WK, WR, PD><<<dim3(groups), dim3(WK * WR * 64), (size_t)bytes, st>>>(a);
  return od_launch_status();
}

// The shapes of the first kernel (one row of x; 16 rows; us). Where the row tiles are few, a tile a workgroup: 4096 x 4096 6.3; 8.6
// (as eager calls 8.9; 9.5, two sets of two tiles 11.9; 15.3). Then two tiles a wave, which share x: 49152 x 4096 28.6; 37.2 (one tile a workgroup 38.8;
// 60.7, two 32.2; 44.5). With many of them and several rows of x, four sets, whose x is staged half as often: 98304 x 4096, 16 rows
// 65.9 against 70.4, 32 rows 79.1 against 87.3; at one row 58.9 against 55.2, and 32 rows over 49152 x 4096 51.8 against 47.7.
// Above 16 rows x is as much to stage as the weights are to read: eight sets of a tile where these are one workgroup for every CU
// (24 rows over 24576 x 4096 27.5 against 31.6, 32768 x 4096 27.7 and 32.0; but 12288 x 4096 26.7 and 20.7).
int launch_few(Q4Args& a, hipStream_t st) {
  const int64_t tiles = (a.N + 15) / 16, cus = od_cu_count();
  if (a.M <= 16) {
    if (tiles <= 2 * cus) return launch_rows<1, 1, 8, 1, 4>(a, st);
    return tiles <= 14 * cus || a.M <= 8 ? launch_rows<2, 1, 4, 2, 2>(a, st) : launch_rows<2, 1, 2, 4, 2>(a, st);
  }
  if (tiles <= 2 * cus) return launch_rows<1, 2, 4, 2, 4>(a, st);
  if (tiles > 4 * cus && tiles <= 8 * cus) return launch_rows<1, 2, 2, 8, 4>(a, st);
  return tiles <= 14 * cus ? launch_rows<2, 2, 4, 2, 2>(a, st) : launch_rows<2, 2, 2, 4, 2>(a, st);
}

template <int MT>
int launch_tiles(const Q4Args& a, unsigned groups, hipStream_t st) {
  static_assert(2 * 32 * MT * kStageBytes <= 65536, "two stages of x");
  q4_tile_kernel<MT><<<dim3(groups), dim3(kThreads), 2 * 32 * MT * kStageBytes, st>>>(a);
  return od_launch_status();
}

}  // namespace

extern "C" int od_q4_linear_ws(int64_t M, int64_t N, int64_t K, int64_t* ws_floats) {
  if (!ws_floats) return OD_ERR_NULL;
  if (!q4_sizes_ok(M, N, K)) return OD_ERR_SHAPE;
  *ws_floats = q4_plan(M, N, K).floats();
  return OD_OK;
}

extern "C" int od_q4_linear(const uint16_t* x, int64_t ldx, const uint8_t* qs, int64_t ldq, const uint16_t* d, int64_t ldd,
                            const uint16_t* bias, const uint16_t* residual, int64_t ldr, uint16_t* out, int64_t ldo, int64_t M,
                            int64_t N, int64_t K, float* ws, int64_t ws_floats, od_stream_t stream) {
  if (!q4_sizes_ok(M, N, K) || ldx < K || ldq < K / 2 || ldd < K / 32 || ldo < N || (residual && ldr < N)) return OD_ERR_SHAPE;
  // offsets within a tile's panels are 32-bit
  if (ldx > (1 << 21) || ldq > (1 << 22) || ldd > (1 << 21)) return OD_ERR_SHAPE;
  if (M == 0) return OD_OK;
  if (!x || !qs || !d || !out) return OD_ERR_NULL;
  if (!od_aligned16(x) || ldx % 8 || !od_aligned16(qs) || ldq % 16 || (((uintptr_t)d) & 1u) || (((uintptr_t)out) & 1u))
    return OD_ERR_ALIGN;
  const Q4Plan q = q4_plan(M, N, K);
  if (q.floats()) {
    if (!ws) return OD_ERR_NULL;
    if (ws_floats < q.floats()) return OD_ERR_SHAPE;
    if (!od_aligned16(ws)) return OD_ERR_ALIGN;
  }
  Q4Args a{x, qs, d, bias, residual, out, ldx, ldq, ldd, ldr, ldo, M, N, K};
  hipStream_t st = (hipStream_t)stream;
  if (M <= kFewRows) return launch_few(a, st);
  a.xexp = reinterpret_cast<int*>(ws);
  a.x16 = reinterpret_cast<uint16_t*>(ws + q.xexp);
  a.part = ws + q.xexp + q.x16;
  a.Kp = q.Kp;
  a.tiles_m = (int)q.tiles_m;
  a.tiles_n = (int)q.tiles_n;
  a.nsplit = q.nsplit;
  a.bm = q.bm;
  a.stages = q.stages;
  const int64_t groups = q.tiles_m * q.tiles_n * q.nsplit;
  if (groups > (1 << 23) || M * ((N + 3) / 4) > (1ll << 32) - 256) return OD_ERR_SHAPE;
  q4_x_kernel<<<dim3((unsigned)M), dim3(kXThreads), 0, st>>>(a);
  const int rc = q.bm == 128 ? launch_tiles<4>(a, (unsigned)groups, st) : launch_tiles<2>(a, (unsigned)groups, st);
  if (rc != OD_OK || q.nsplit == 1) return rc;
  q4_sum_kernel<<<dim3((unsigned)((M * ((N + 3) / 4) + 255) / 256)), dim3(256), 0, st>>>(a);
  return od_launch_status();
}
