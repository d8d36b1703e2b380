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
  int64_t Kp;  // K in whole stages: the row stride of x16
  int tiles_m, tiles_n, nsplit, stages;
};

__device__ __forceinline__ __amdgpu_buffer_rsrc_t rsrc(const void* p, int64_t bytes) {
  return __builtin_amdgcn_make_buffer_rsrc(const_cast<void*>(p), (short)0, (int)bytes, 0x00020000);
}

// ------------------------------------------------------------------------------------------------ few rows of x
// Bound by reading the weights. A workgroup's NW waves share 16 RT weight rows, each wave every NW-th step of 128 values (4
// blocks of every row, 64 contiguous bytes), and add up in LDS. V_MFMA_F32_16X16X32_BF16 with the weights as the A operand, 16
// rows, and up to 16 rows of x as the B operand, 32 values a time, which is one block: the sums of a block, exact in their
// products, take the fp32 factor d afterwards, so no weight is rounded. Lane (j, g) = (lane % 16, lane / 16):
//  * reads block 4 s + g of weight row j, 16 bytes; four lane exchanges (a transposition over g) give it word g of each of the
//    four blocks: values 4 g .. 4 g + 3 and 16 + 4 g .. + 3 of the block;
//  * four bits u at the bottom of 128.0's bf16 are 128 + u: one shift and one and-or for two values. The 136 that it is above
//    u - 8 leaves by the C operand, -136 times the sum of x over the block, itself a product with a constant A (shared by the RT
//    row tiles). (A row of x that holds an infinity or NaN so becomes NaN.)
//  * holds weight rows 4 g + i of column j of the result; d of row 4 g + i and block b is the one that lane 16 g + 4 i + b loaded.
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
// 8 values as bf16 128 + u, in the order 0 2 16 18 1 3 17 19 (from 4 g)
__device__ __forceinline__ v4u raised(uint32_t t) {
  v4u r;
#pragma unroll
  for (int i = 0; i < 4; ++i) r[i] = ((t >> (4 * i)) & 0x000f000fu) | 0x43004300u;
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

template <int RT, int CT>
struct Q4Step {
  v4u w[RT];
  uint32_t d[RT];
  v2u x[CT][4][2];
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

template <int RT, int CT, int NW>
__global__ __launch_bounds__(NW * 64) void q4_rows_kernel(Q4Args a) {
  __shared__ float4 red[NW][RT * CT][64];
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), j = lane & 15, g = lane >> 4;
  const int64_t n0 = (int64_t)blockIdx.x * (16 * RT), m0 = (int64_t)blockIdx.y * (16 * CT);
  const int rows = (int)min((int64_t)16 * RT, a.N - n0), toks = (int)min((int64_t)16 * CT, a.M - m0), blocks = (int)(a.K / 32);
  const auto rw = rsrc(a.qs + n0 * a.ldq, (rows - 1) * a.ldq + a.K / 2);
  const auto rd = rsrc(a.d + n0 * a.ldd, ((rows - 1) * a.ldd + blocks) * 2);
  const auto rx = rsrc(a.x + m0 * a.ldx, ((toks - 1) * a.ldx + a.K) * 2);
  const auto none = rsrc(a.x, 0);
  const int steps = (blocks + 3) / 4;
  const int wo = (int)(j * a.ldq) + 16 * g, dofs = 2 * (int)((lane >> 2) * a.ldd + (lane & 3)), xo = 2 * (int)(j * a.ldx + 4 * g);
  using Step = Q4Step<RT, CT>;
  auto load = [&](int s, Step& t) {  // past the last step: nothing is read
    const bool in = s < steps;
#pragma unroll
    for (int r = 0; r < RT; ++r) {
      t.w[r] = __builtin_bit_cast(v4u, __builtin_amdgcn_raw_buffer_load_b128(in ? rw : none, wo + (int)(16 * r * a.ldq), 64 * s, 2));
      t.d[r] = (uint16_t)__builtin_amdgcn_raw_buffer_load_b16(in ? rd : none, dofs + (int)(32 * r * a.ldd), 8 * s, 0);
    }
#pragma unroll
    for (int c = 0; c < CT; ++c)
#pragma unroll
      for (int b = 0; b < 4; ++b)
#pragma unroll
        for (int h = 0; h < 2; ++h)
          t.x[c][b][h] = __builtin_bit_cast(v2u, __builtin_amdgcn_raw_buffer_load_b64(
              4 * s + b < blocks ? rx : none, xo + (int)(32 * c * a.ldx) + 64 * b + 32 * h, 256 * s, 0));
    __builtin_amdgcn_sched_barrier(0);
  };
  v4f acc[RT][CT];
#pragma unroll
  for (auto& r : acc)
#pragma unroll
    for (auto& c : r) c = v4f{0, 0, 0, 0};
  const v4u down = {0xc308c308u, 0xc308c308u, 0xc308c308u, 0xc308c308u};  // -136
  auto compute = [&](int s, Step& t) {
    v4u xf[CT][4];
    v4f off[CT][4];
#pragma unroll
    for (int c = 0; c < CT; ++c)
#pragma unroll
      for (int b = 0; b < 4; ++b) {
        xf[c][b] = ordered(t.x[c][b][0], t.x[c][b][1]);
        off[c][b] = mfma16(down, xf[c][b], v4f{0, 0, 0, 0});
      }
#pragma unroll
    for (int r = 0; r < RT; ++r) {
      transpose4(t.w[r]);
      // (past the row's last block lies the next row's first one)
      const float d = 4 * s + (lane & 3) < blocks ? (float)__builtin_bit_cast(_Float16, (uint16_t)t.d[r]) : 0.0f;
      auto block = [&](auto B) {
        constexpr int b = decltype(B)::value;
        const v4u w = raised(t.w[r][b]);
        const float d0 = row_lane<b>(d), d1 = row_lane<4 + b>(d), d2 = row_lane<8 + b>(d), d3 = row_lane<12 + b>(d);
#pragma unroll
        for (int c = 0; c < CT; ++c) {
          const v4f p = mfma16(w, xf[c][b], off[c][b]);
          acc[r][c][0] = __builtin_fmaf(d0, p[0], acc[r][c][0]);
          acc[r][c][1] = __builtin_fmaf(d1, p[1], acc[r][c][1]);
          acc[r][c][2] = __builtin_fmaf(d2, p[2], acc[r][c][2]);
          acc[r][c][3] = __builtin_fmaf(d3, p[3], acc[r][c][3]);
        }
      };
      block(std::integral_constant<int, 0>{});
      block(std::integral_constant<int, 1>{});
      block(std::integral_constant<int, 2>{});
      block(std::integral_constant<int, 3>{});
    }
  };
  Step t[2];
  if (wave < steps) {
    load(wave, t[0]);
    for (int s = wave; s < steps; s += 2 * NW) {
      load(s + NW, t[1]);
      compute(s, t[0]);
      if (s + NW >= steps) break;
      load(s + 2 * NW, t[0]);
      compute(s + NW, t[1]);
    }
  }
#pragma unroll
  for (int r = 0; r < RT; ++r)
#pragma unroll
    for (int c = 0; c < CT; ++c) red[wave][r * CT + c][lane] = make_float4(acc[r][c][0], acc[r][c][1], acc[r][c][2], acc[r][c][3]);
  __syncthreads();
  for (int i = threadIdx.x; i < RT * CT * 64; i += NW * 64) {
    const int tile = i >> 6, l = i & 63;
    v4f y = v4f{0, 0, 0, 0};
#pragma unroll
    for (int w = 0; w < NW; ++w) {
      const float4 v = red[w][tile][l];
      y += v4f{v.x, v.y, v.z, v.w};
    }
    const int64_t m = m0 + tile % CT * 16 + (l & 15), n = n0 + tile / CT * 16 + 4 * (l >> 4);
    if (m < a.M && n < a.N) q4_store(a, m, n, y);
  }
}

// ------------------------------------------------------------------------------------------------ many rows of x
// Bound by the matrix cores. x goes to fp16 once, each row in a power-of-two frame (2^(14 - e), 2^e above its largest value: exact
// but for values below 2^-29 of it, which move by 2^-40 of it at most), zero-padded to whole stages, the values of a block in the
// order in which its weights come out of the conversion. Weights become (u - 8) d in fp16 on their way into LDS: one rounding,
// 2^-11 at most (so |W| up to 65504, fp16's range). A row of x that holds an infinity or NaN is NaN.
constexpr int kXThreads = 256;
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
    *reinterpret_cast<uint4*>(a.x16 + m * a.Kp + 8 * i) = o;
  }
}

constexpr int kThreads = 512;
constexpr int BN = 256, BK = 64, kRow = 2 * BK;  // weight rows of a tile, values and bytes of a stage
__device__ __forceinline__ int swz(int row, int chunk) { return row * kRow + ((chunk ^ ((row >> 1) & 7)) << 4); }
__device__ __forceinline__ void barrier_lds() { asm volatile("s_waitcnt lgkmcnt(0)\n\ts_barrier" ::: "memory"); }

// 8 values (u - 8) d in fp16, each rounded once: u - 8 from 1024 + u, or 16 (u - 8) from 1024 + 16 u, times d or d / 16
__device__ __forceinline__ v4u q4_f16(uint32_t w, f16x2 d) {
  const f16x2 base = {(_Float16)-1032.0f, (_Float16)-1032.0f}, base16 = {(_Float16)-72.0f, (_Float16)-72.0f},
              sixteenth = {(_Float16)0.0625f, (_Float16)0.0625f};
  v4u r;
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const uint32_t s = i < 2 ? w : w >> 8;
    const f16x2 u = __builtin_bit_cast(f16x2, (s & (i & 1 ? 0x00f000f0u : 0x000f000fu)) | 0x64006400u);
    const f16x2 n = i & 1 ? __builtin_elementwise_fma(u, sixteenth, base16) : u + base;
    r[i] = __builtin_bit_cast(uint32_t, n * d);
  }
  return r;
}

template <int BM>
__global__ __launch_bounds__(kThreads, 1) void q4_tile_kernel(Q4Args p) {
  constexpr int WM = BM / 64, WN = 8 / WM, TM = 2, TN = BN / WN / 32;  // waves, and their 32 x 32 tiles
  constexpr int kSlabA = BM * kRow, kStage = kSlabA + BN * kRow, LA = BM * (kRow / 16) / kThreads;
  extern __shared__ __attribute__((aligned(16))) int8_t smem[];
  // flat ids are dealt round-robin over the 8 XCDs; id = the XCD's contiguous range; row tiles fastest
  const int ntiles = p.tiles_m * p.tiles_n * p.nsplit;
  const int f = blockIdx.x, xcd = f & 7, local = f >> 3, per = ntiles >> 3, rem = ntiles & 7;
  const int id = xcd < rem ? xcd * (per + 1) + local : rem * (per + 1) + (xcd - rem) * per + local;
  const int tm = id % p.tiles_m, tn = id / p.tiles_m % p.tiles_n, sp = id / p.tiles_m / p.tiles_n;
  const int64_t m0 = (int64_t)tm * BM, n0 = (int64_t)tn * BN;
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6, wm = wave / WN, wn = wave % WN;
  const int all = (int)(p.Kp / BK), k_lo = sp * p.stages, nk = min(p.stages, all - k_lo);

  const int64_t rows_a = min((int64_t)BM, p.M - m0), rows_b = min((int64_t)BN, p.N - n0);
  const auto ra = rsrc(p.x16 + m0 * p.Kp + (int64_t)k_lo * BK, ((rows_a - 1) * p.Kp + (int64_t)nk * BK) * 2);
  const auto rb = rsrc(p.qs + n0 * p.ldq, (rows_b - 1) * p.ldq + p.K / 2);
  const auto rd = rsrc(p.d + n0 * p.ldd, ((rows_b - 1) * p.ldd + p.K / 32) * 2);
  const auto none = rsrc(p.x16, 0);
  const int a_row = tid / 8, a_chunk = tid % 8;
  const int a_vo = (int)(a_row * p.Kp * 2) + a_chunk * 16, a_step = (int)(p.Kp * 2 * 64), a_lo = swz(a_row, a_chunk);
  const int b_row = tid / 2, b_c = tid % 2;  // thread t: block t % 2 of the stage's two, weight row t / 2
  const int b_vo = (int)(b_row * p.ldq) + 16 * b_c, d_vo = 2 * (int)(b_row * p.ldd + b_c);
  const int blocks = (int)(p.K / 32);

  v4u ga[LA], gb;
  uint16_t gd = 0;
  int g_block = 0;
  auto gload_a = [&](int kt, int i) {
    ga[i] = __builtin_bit_cast(v4u, __builtin_amdgcn_raw_buffer_load_b128(kt < nk ? ra : none, a_vo, kt * kRow + i * a_step, 0));
  };
  auto gload_b = [&](int kt) {
    const int k = k_lo + kt;
    gb = __builtin_bit_cast(v4u, __builtin_amdgcn_raw_buffer_load_b128(kt < nk ? rb : none, b_vo, 32 * k, 0));
    gd = (uint16_t)__builtin_amdgcn_raw_buffer_load_b16(kt < nk ? rd : none, d_vo, 4 * k, 0);
    g_block = 2 * k + b_c;
  };
  auto swrite_a = [&](int buf, int i) { *reinterpret_cast<v4u*>(smem + buf * kStage + a_lo + i * 64 * kRow) = ga[i]; };
  auto swrite_b = [&](int buf) {
    int8_t* lb = smem + buf * kStage + kSlabA;
    const _Float16 d = __builtin_bit_cast(_Float16, g_block < blocks ? gd : (uint16_t)0);
    const f16x2 d2 = {d, d};
#pragma unroll
    for (int q = 0; q < 4; ++q) *reinterpret_cast<v4u*>(lb + swz(b_row, 4 * b_c + q)) = q4_f16(gb[q], d2);
  };
  auto frags = [&](int buf, int s, v4u (&fa)[TM], v4u (&fb)[TN]) {
    const int chunk = s * 2 + (lane >> 5);
    const int8_t* la = smem + buf * kStage;
    const int8_t* lb = la + kSlabA;
#pragma unroll
    for (int i = 0; i < TM; ++i) fa[i] = *reinterpret_cast<const v4u*>(la + swz(wm * 64 + i * 32 + (lane & 31), chunk));
#pragma unroll
    for (int j = 0; j < TN; ++j) fb[j] = *reinterpret_cast<const v4u*>(lb + swz(wn * (TN * 32) + j * 32 + (lane & 31), chunk));
  };
  v16f acc[TN][TM];
#pragma unroll
  for (auto& r : acc)
#pragma unroll
    for (auto& c : r) c = v16f{0, 0, 0, 0, 0, 0, 0, 0, 0, 0, 0, 0, 0, 0, 0, 0};
  // the weights as the A operand: a lane then holds 4 neighbouring columns of out
  constexpr int kMf = TM * TN;
  auto mma = [&](const v4u (&fa)[TM], const v4u (&fb)[TN], auto fill, auto OPS) {
    constexpr int kOps = decltype(OPS)::value;
#pragma unroll
    for (int x = 0; x < kMf; ++x) {
      acc[x / TM][x % TM] = __builtin_amdgcn_mfma_f32_32x32x16_f16(__builtin_bit_cast(f16x8, fb[x / TM]),
                                                                  __builtin_bit_cast(f16x8, fa[x % TM]), acc[x / TM][x % TM], 0, 0, 0);
#pragma unroll
      for (int o = 0; o < kOps; ++o)
        if (o * kMf / (kOps > 0 ? kOps : 1) == x) fill(o);
      __builtin_amdgcn_sched_barrier(0);
    }
  };
  auto nofill = [](int) {};
  using Zero = std::integral_constant<int, 0>;
  v4u f0a[TM], f0b[TN], f1a[TM], f1b[TN];
  auto load_all = [&](int kt) {
#pragma unroll
    for (int i = 0; i < LA; ++i) gload_a(kt, i);
    gload_b(kt);
  };
  load_all(0);
#pragma unroll
  for (int i = 0; i < LA; ++i) swrite_a(0, i);
  swrite_b(0);
  load_all(1);
  barrier_lds();
  frags(0, 0, f0a, f0b);
  constexpr int kOps0 = 2 * (LA + 1);
  for (int kt = 0; kt < nk; ++kt) {
    const int cur = kt & 1, nxt = cur ^ 1;
    frags(cur, 1, f1a, f1b);
    __builtin_amdgcn_sched_barrier(0);
    auto fill0 = [&](int o) {
      if (o < LA) swrite_a(nxt, o);
      else if (o == LA) swrite_b(nxt);
      else if (o < 2 * LA + 1) gload_a(kt + 2, o - LA - 1);
      else gload_b(kt + 2);
    };
    mma(f0a, f0b, fill0, std::integral_constant<int, kOps0>{});
    frags(cur, 2, f0a, f0b);
    __builtin_amdgcn_sched_barrier(0);
    mma(f1a, f1b, nofill, Zero{});
    frags(cur, 3, f1a, f1b);
    __builtin_amdgcn_sched_barrier(0);
    mma(f0a, f0b, nofill, Zero{});
    barrier_lds();
    frags(nxt, 0, f0a, f0b);
    __builtin_amdgcn_sched_barrier(0);
    mma(f1a, f1b, nofill, Zero{});
  }
  // lane: row lane % 32 of x, weight rows 8 (r / 4) + 4 (lane / 32) + r % 4 of the tile's 32
  const int col = lane & 31, h = lane >> 5;
#pragma unroll
  for (int i = 0; i < TM; ++i) {
    const int64_t m = m0 + wm * 64 + i * 32 + col;
    if (m >= p.M) continue;
    const float unit = __builtin_ldexpf(1.0f, p.xexp[m] / 2 - 7), unit2 = __builtin_ldexpf(1.0f, p.xexp[m] - p.xexp[m] / 2 - 7);
#pragma unroll
    for (int j = 0; j < TN; ++j)
#pragma unroll
      for (int q = 0; q < 4; ++q) {
        const int64_t n = n0 + wn * (TN * 32) + j * 32 + 8 * q + 4 * h;
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

constexpr int kFewRows = 32;

struct Q4Plan {
  int bm, nsplit, stages;
  int64_t Kp, tiles_m, tiles_n, xexp, x16, part;  // the workspace, in floats
  int64_t floats() const { return xexp + x16 + part; }
};
Q4Plan q4_plan(int64_t M, int64_t N, int64_t K) {
  Q4Plan q = {};
  if (M <= kFewRows) return q;
  const int64_t cus = od_cu_count();
  q.Kp = (K + BK - 1) / BK * BK;
  q.tiles_n = (N + BN - 1) / BN;
  q.bm = (M + 255) / 256 * q.tiles_n >= cus ? 256 : 128;
  q.tiles_m = (M + q.bm - 1) / q.bm;
  const int64_t all = q.Kp / BK, tiles = q.tiles_m * q.tiles_n;
  int64_t n = tiles >= cus ? 1 : cus / tiles;
  if (n > all / 8) n = all / 8;  // 8 stages at least
  if (n < 1) n = 1;
  q.stages = (int)((all + n - 1) / n);
  q.nsplit = (int)((all + q.stages - 1) / q.stages);
  q.xexp = (M + 3) / 4 * 4;
  q.x16 = M * q.Kp / 2;
  q.part = q.nsplit > 1 ? q.nsplit * M * ((N + 3) / 4 * 4) : 0;
  return q;
}

bool q4_sizes_ok(int64_t M, int64_t N, int64_t K) {
  return M >= 0 && N >= 1 && K >= 32 && K % 32 == 0 && M <= (1ll << 22) && N <= (1ll << 24) && K <= (1ll << 20);
}

template <int BM>
int launch_tile(const Q4Args& a, unsigned groups, hipStream_t st) {
  static std::atomic<uint64_t> allowed{0};
  constexpr int bytes = 2 * (BM + BN) * kRow;
  int dev = 0;
  if (hipGetDevice(&dev) != hipSuccess || dev < 0 || dev >= 64) return OD_ERR_LAUNCH;
  if (!((allowed.load(std::memory_order_relaxed) >> dev) & 1)) {
    if (hipFuncSetAttribute(reinterpret_cast<const void*>(q4_tile_kernel<BM>), hipFuncAttributeMaxDynamicSharedMemorySize, bytes) !=
        hipSuccess)
      return OD_ERR_LAUNCH;
    allowed.fetch_or(1ull << dev, std::memory_order_relaxed);
  }
  q4_tile_kernel<BM><<<dim3(groups), dim3(kThreads), bytes, st>>>(a);
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
  if (M <= kFewRows) {
    const unsigned gx = (unsigned)((N + 15) / 16), g2 = (unsigned)((N + 31) / 32);
    if (M <= 16) q4_rows_kernel<1, 1, 8><<<dim3(gx), dim3(512), 0, st>>>(a);
    else q4_rows_kernel<2, 2, 8><<<dim3(g2), dim3(512), 0, st>>>(a);
    return od_launch_status();
  }
  a.xexp = reinterpret_cast<int*>(ws);
  a.x16 = reinterpret_cast<uint16_t*>(ws + q.xexp);
  a.part = ws + q.xexp + q.x16;
  a.Kp = q.Kp;
  a.tiles_m = (int)q.tiles_m;
  a.tiles_n = (int)q.tiles_n;
  a.nsplit = q.nsplit;
  a.stages = q.stages;
  const int64_t groups = q.tiles_m * q.tiles_n * q.nsplit;
  if (groups > (1 << 23) || M * ((N + 3) / 4) > (1ll << 32) - 256) return OD_ERR_SHAPE;
  q4_x_kernel<<<dim3((unsigned)M), dim3(kXThreads), 0, st>>>(a);
  const int rc = q.bm == 256 ? launch_tile<256>(a, (unsigned)groups, st) : launch_tile<128>(a, (unsigned)groups, st);
  if (rc != OD_OK || q.nsplit == 1) return rc;
  q4_sum_kernel<<<dim3((unsigned)((M * ((N + 3) / 4) + 255) / 256)), dim3(256), 0, st>>>(a);
  return od_launch_status();
}
