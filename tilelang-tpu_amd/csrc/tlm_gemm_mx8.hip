// Products of 8-bit operands with power-of-two scales: C = A B^T, and SwiGLU of two of them with an 8-bit result.
//
// v_mfma_scale_f32_16x16x128_f8f6f4 multiplies each block of 32 k by 2^(ea + eb) as it adds it. Lane l holds row l % 16 of
// its operand and the 16-byte chunks q and q + 4 of its 128 k (q = l / 16), and the scale of k block q. The weights are the first
// operand, so that a lane's sums are neighbouring columns of one row of C.
#include "tlm_mx8.h"

#include <algorithm>

namespace {

using mx8::BLOCK;

struct Mat {  // codes [rows, K] and scales
  const uint8_t* codes;
  const uint8_t* scales;
};

struct Args {
  Mat a, b, b2;  // b2: the second weights of a gated product
  void* c;       // 16-bit rows, or codes
  uint8_t* c_scales;
  int64_t M, N;
  int K, kt;  // kt: k steps of 128
};

// Rows r0 + F i + f, f = 0 .. F - 1, of a matrix as F operands: row i of operand f. Rows behind the last are the last.
template <int F>
struct Rows {
  const uint8_t* p[F];
  const uint8_t* s;
  TLM_DEV Rows(const Mat& m, int64_t rows, int64_t r0, int K, int kt, int lane) {
    const int i = lane & 15, q = lane >> 4;
#pragma unroll
    for (int f = 0; f < F; ++f) p[f] = m.codes + min(r0 + F * i + f, rows - 1) * K + 16 * q;
    s = m.scales + mx8::scale_at(r0, 0, kt) + q * 64 + F * i;
  }
  // operands and scales (operand f's in byte f) of k step t; past K: codes 0, scale 1
  template <bool TAIL>
  TLM_DEV void load(int t, int K, int lane, i32x8 (&o)[F], uint32_t& sc) const {
    const int q = lane >> 4;
    const bool ok0 = !TAIL || t * 128 + 16 * q < K, ok1 = !TAIL || t * 128 + 64 + 16 * q < K;
#pragma unroll
    for (int f = 0; f < F; ++f) {
      u32x4 x = {}, y = {};
      if (ok0) x = *(const u32x4*)(p[f] + (int64_t)t * 128);
      if (ok1) y = *(const u32x4*)(p[f] + (int64_t)t * 128 + 64);
      o[f] = i32x8{(int)x[0], (int)x[1], (int)x[2], (int)x[3], (int)y[0], (int)y[1], (int)y[2], (int)y[3]};
    }
    const uint8_t* const at = s + (int64_t)t * 256;
    if constexpr (F == 1) sc = *at;
    else if constexpr (F == 2) sc = *(const uint16_t*)at;
    else sc = *(const uint32_t*)at;
    if (TAIL && t * 128 + 32 * q >= K) sc = 0x7f7f7f7fu;
  }
};

template <int SA, int SB>
TLM_DEV f32x4 mma(const i32x8& a, const i32x8& b, f32x4 c, uint32_t sa, uint32_t sb) {
  return __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(a, b, c, 0, 0, SA, (int)sa, SB, (int)sb);
}

using ldsop::unroll;

// up * silu(gate).
TLM_DEV float gated(float gate, float up) { return up * (gate * __builtin_amdgcn_rcpf(fast_exp(-gate) + 1.0f)); }

constexpr int D_WAVES = 8;

// OUT: TLM_F16, TLM_BF16: C = A B^T. TLM_F8E4M3: up * silu(gate) with its scales.
// A workgroup computes 16 MT rows and 16 NF columns (32 of the gated product: NF 2 of each matrix), its waves
// every 8th k step of them.
template <int MT, int NF, int OUT>
__global__ __launch_bounds__(64 * D_WAVES) void gemm_mx8_direct(Args a) {
  constexpr bool DUAL = OUT == TLM_F8E4M3;
  constexpr int W = DUAL ? 2 * NF : NF;
  __shared__ f32x4 red[D_WAVES][W * MT][64];
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const int64_t m0 = (int64_t)blockIdx.y * 16 * MT, n0 = (int64_t)blockIdx.x * 16 * NF;
  const Rows<MT> x(a.a, a.M, m0, a.K, a.kt, lane);
  const Rows<NF> w(a.b, a.N, n0, a.K, a.kt, lane), w2(DUAL ? a.b2 : a.b, a.N, n0, a.K, a.kt, lane);
  f32x4 acc[W][MT];
#pragma unroll
  for (int f = 0; f < W; ++f)
#pragma unroll
    for (int t = 0; t < MT; ++t) acc[f][t] = f32x4{};
  auto step = [&](int t, auto tail) {
    constexpr bool TAIL = decltype(tail)::value;
    i32x8 xo[MT], wo[NF], vo[NF];
    uint32_t xs, ws, vs = 0;
    x.template load<TAIL>(t, a.K, lane, xo, xs);
    w.template load<TAIL>(t, a.K, lane, wo, ws);
    if constexpr (DUAL) w2.template load<TAIL>(t, a.K, lane, vo, vs);
    unroll<0, W>([&](auto fc) {
      constexpr int f = decltype(fc)::value;
      unroll<0, MT>([&](auto tc) {
        constexpr int m = decltype(tc)::value;
        if constexpr (f < NF) acc[f][m] = mma<f, m>(wo[f], xo[m], acc[f][m], ws, xs);
        else acc[f][m] = mma<f - NF, m>(vo[f - NF], xo[m], acc[f][m], vs, xs);
      });
    });
  };
  const int full = a.K / 128;
  for (int t = wave; t < full; t += D_WAVES) step(t, std::false_type{});
  if (full < a.kt && full % D_WAVES == wave) step(full, std::true_type{});

#pragma unroll
  for (int f = 0; f < W; ++f)
#pragma unroll
    for (int t = 0; t < MT; ++t) red[wave][f * MT + t][lane] = acc[f][t];
  __syncthreads();
  // wave t finishes operand t of A: the lane's row is m0 + MT i + t, its columns n0 + NF (4 g + e) + f
  if (wave >= MT) return;
  const int i = lane & 15, g = lane >> 4;
  f32x4 sum[W];
#pragma unroll
  for (int f = 0; f < W; ++f) {
    sum[f] = red[0][f * MT + wave][lane];
#pragma unroll
    for (int v = 1; v < D_WAVES; ++v) sum[f] += red[v][f * MT + wave][lane];
  }
  const int64_t row = m0 + MT * i + wave, col = n0 + NF * 4 * g;
  float v[4 * NF];
#pragma unroll
  for (int e = 0; e < 4; ++e)
#pragma unroll
    for (int f = 0; f < NF; ++f) {
      if constexpr (DUAL) v[e * NF + f] = gated(sum[f][e], sum[NF + f][e]);
      else v[e * NF + f] = sum[f][e];
    }
  if constexpr (DUAL) {
    static_assert(NF == 2, "32 columns, a block");
    uint32_t m = 0;
#pragma unroll
    for (int j = 0; j < 8; ++j) m = max(m, mx8::abs_bits(v[j]));
    m = max(m, (uint32_t)__shfl_xor((int)m, 16));
    m = max(m, (uint32_t)__shfl_xor((int)m, 32));
    if (row >= a.M) return;
    const uint32_t byte = mx8::scale_byte(m);
    const float inv = mx8::inverse(byte);
    *(u32x2*)((uint8_t*)a.c + row * a.N + col) = u32x2{mx8::codes4(v[0], v[1], v[2], v[3], inv, byte < 255),
                                                       mx8::codes4(v[4], v[5], v[6], v[7], inv, byte < 255)};
    if (g == 0) a.c_scales[mx8::scale_at(row, (int)(n0 / BLOCK), (int)((a.N + 127) / 128))] = (uint8_t)byte;
  } else {
    if (row >= a.M) return;
    using H = h16<OUT == TLM_BF16>;
    uint16_t* const c = (uint16_t*)a.c + row * a.N + col;
#pragma unroll
    for (int j = 0; j < 4 * NF; ++j)
      if (col + j < a.N) c[j] = (uint16_t)H::from_f32(v[j]);
  }
}

// ---- whole prompts: 256 x 256 tiles

// The ping-pong schedule of gemm8_256x256 (tlm_gemm_fp8.hip): the two waves of a SIMD take turns, one reads its next operands from LDS
// while the other multiplies, and LDS-DMA is issued only beside the reads. Here W, the weights, is the operand a wave holds
// (128 rows: 8 operands) and X the one it reads as it multiplies (64 rows: 4).
//
// Slot 16 f + i of a 64-row group of an LDS stage holds row 4 i + f, so that operand f, read from 16 neighbouring slots, has the rows
// whose scales are byte f of the lanes' words: three words a k step, loaded a step ahead, are all the scales a wave needs. Of the
// sums, a lane then has 16 neighbouring columns of each of its rows: C is stored, or a block of 32 quantised with one exchange
// between two lanes, without a way through LDS.
constexpr int P_T = 512, P_M = 256, P_N = 256, P_ST = 256 * 128;  // P_ST: bytes of a stage of one operand
constexpr int P_W = 2, P_X = 3;                                   // stages of W and X
constexpr uint32_t OOB = 0x80000000u;                             // past every descriptor's end, also with 3 K more

TLM_DEV void wait_lgkm0() { __builtin_amdgcn_s_waitcnt(0xc07f); }
template <int N>
TLM_DEV void wait_lgkm() {
  __builtin_amdgcn_s_waitcnt(0xc07f | (N << 8));
}
template <int N>
TLM_DEV void wait_vm() {
  static_assert(N < 64, "vmcnt is 6 bits");
  __builtin_amdgcn_sched_barrier(0);
  __builtin_amdgcn_s_waitcnt(0x3f70 | (N & 15) | ((N >> 4) << 14));
  __builtin_amdgcn_sched_barrier(0);
}
TLM_DEV void barrier() {
  __builtin_amdgcn_sched_barrier(0);
  asm volatile("" ::: "memory");
  wait_lgkm0();
  __builtin_amdgcn_s_barrier();
  asm volatile("" ::: "memory");
  __builtin_amdgcn_sched_barrier(0);
}
TLM_DEV i32x8 cat8(u32x4 lo, u32x4 hi) {
  return i32x8{(int)lo[0], (int)lo[1], (int)lo[2], (int)lo[3], (int)hi[0], (int)hi[1], (int)hi[2], (int)hi[3]};
}
// 16 bytes per lane at base + off to dst and on; zeros from `end` on.
TLM_DEV void dma16(const uint8_t* base, int end, uint8_t* dst, uint32_t off) {
  const __amdgpu_buffer_rsrc_t rs = __builtin_amdgcn_make_buffer_rsrc((void*)base, (short)0, end, 0x00020000);
  __builtin_amdgcn_raw_ptr_buffer_load_lds(rs, (__attribute__((address_space(3))) void*)dst, 16, off, 0, 0, 0);
}

// XCD x (workgroup % 8) takes a contiguous range of tiles, row tiles in groups of four, so that its L2 serves both operands.
TLM_DEV void tile_of(int wg, int tiles_m, int tiles_n, int& tm, int& tn) {
  const int total = tiles_m * tiles_n, xcd = wg & 7;
  const int lin = xcd * (total >> 3) + min(xcd, total & 7) + (wg >> 3);
  const int per = 4 * tiles_n, first = lin / per * 4, gm = min(tiles_m - first, 4), r = lin % per;
  tm = first + r % gm;
  tn = r / gm;
}

// 16 neighbouring columns col .. of a row of C.
template <int OUT>
TLM_DEV void store16(uint16_t* c, const float (&v)[16], int64_t left, bool vec) {
  using H = h16<OUT == TLM_BF16>;
  if (vec && left >= 16) {
#pragma unroll
    for (int h = 0; h < 2; ++h)
      *(u32x4*)(c + 8 * h) = u32x4{H::pack(v[8 * h], v[8 * h + 1]), H::pack(v[8 * h + 2], v[8 * h + 3]),
                                   H::pack(v[8 * h + 4], v[8 * h + 5]), H::pack(v[8 * h + 6], v[8 * h + 7])};
    return;
  }
#pragma unroll
  for (int j = 0; j < 16; ++j)
    if (j < left) c[j] = (uint16_t)H::from_f32(v[j]);
}

TLM_DEV uint32_t xrow_max_bits(uint32_t m) {  // of lanes l and l ^ 16
  const auto r = __builtin_amdgcn_permlane16_swap(m, m, false, false);
  return max(r[0], r[1]);
}

template <int OUT>
__global__ __launch_bounds__(P_T, 1) void gemm_mx8_256(Args a) {
  constexpr bool DUAL = OUT == TLM_F8E4M3;
  constexpr int BN = DUAL ? P_N / 2 : P_N;  // columns of the result
  __shared__ __attribute__((aligned(1024))) uint8_t smem[(P_W + P_X) * P_ST];
  const int tid = threadIdx.x, lane = tid & 63;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int grp = wave >> 2, quarter = wave & 3;  // half of W, 64 rows of X
  const int M = (int)a.M, N = (int)a.N, K = a.K, KT = a.kt;
  int tm, tn;
  tile_of(blockIdx.x, (M + P_M - 1) / P_M, (N + BN - 1) / BN, tm, tn);
  const int m0 = tm * P_M, n0 = tn * BN;

  // ---- LDS-DMA: wave w of a group fills slots 64 w .. 64 w + 63 of its operand's stage, 8 a instruction
  const bool is_w = grp == 0;
  const bool second = DUAL && is_w && (quarter & 1);
  // rows of the wave's 64 slots start here (gated: gate and up groups of 64 alternate)
  const int r0 = is_w ? n0 + (DUAL ? 64 * (quarter >> 1) : 64 * quarter) : m0 + 64 * quarter;
  const int rows = is_w ? N : M;
  const uint8_t* const base = (is_w ? (second ? a.b2.codes : a.b.codes) : a.a.codes) + (int64_t)min(r0, rows) * K;
  // instruction j: slots 8 j + lane / 8, rows 32 (j % 2) + 4 (lane / 8) + j / 2; what is past the last row lies past the
  // descriptor's end
  const int left = max(0, min(64, rows - r0)) * K;
  int chunk[2];
  uint32_t off[2];
#pragma unroll
  for (int h = 0; h < 2; ++h) {
    chunk[h] = 16 * ((lane & 7) ^ (4 * h + (lane >> 4)));
    off[h] = (uint32_t)((32 * h + 4 * (lane >> 3)) * K + chunk[h]);
  }
  auto w_st = [&](int t) { return smem + (t & 1) * P_ST; };
  auto x_st = [&](int t) { return smem + P_W * P_ST + (t % P_X) * P_ST; };
  auto fill = [&](int t, uint8_t* st, int j) {
    const uint32_t o = chunk[j & 1] < K - t * 128 ? off[j & 1] : OOB;
    dma16(base + (int64_t)t * 128, max(0, left - t * 128), st + quarter * 8192 + j * 1024, o + (j >> 1) * K);
  };

  // ---- scales: words of the wave's two groups of W and its group of X; past the last row, another's
  auto words = [&](const uint8_t* s, int r, int n) {
    return s + (int64_t)(min(r, n - 1) >> 6) * KT * 256 + 4 * lane;
  };
  const uint8_t* const s0 = words(a.b.scales, n0 + (DUAL ? 64 : 128) * grp, N);
  const uint8_t* const s1 = DUAL ? words(a.b2.scales, n0 + 64 * grp, N) : words(a.b.scales, n0 + 128 * grp + 64, N);
  const uint8_t* const sx = words(a.a.scales, m0 + 64 * quarter, M);
  struct Scales {
    uint32_t w[2], x;
  };
  auto scales_of = [&](int t) {
    const int64_t o = (int64_t)t * 256;
    Scales s{{*(const uint32_t*)(s0 + o), *(const uint32_t*)(s1 + o)}, *(const uint32_t*)(sx + o)};
    return s;
  };
  auto mask_tail = [&](Scales& s, int t) {  // past K: codes 0, scale 1
    if (t * 128 + 32 * (lane >> 4) >= K) s = Scales{{0x7f7f7f7fu, 0x7f7f7f7fu}, 0x7f7f7f7fu};
  };

  // ---- operands
  const int q = lane >> 4;
  const int xr = ((lane & 15) >> 1) & 7;
  const uint32_t w_row = ldsop::lds_u32(smem) + (grp * 128 + (lane & 15)) * 128;
  const uint32_t x_row = ldsop::lds_u32(smem) + P_W * P_ST + (quarter * 64 + (lane & 15)) * 128;
  uint32_t ch[2];
#pragma unroll
  for (int p = 0; p < 2; ++p) ch[p] = 16 * ((4 * p + q) ^ xr);
  f32x4 acc[8][4];
#pragma unroll
  for (int f = 0; f < 8; ++f)
#pragma unroll
    for (int t = 0; t < 4; ++t) acc[f][t] = f32x4{};
  u32x4 wop[8][2], xop0[2];
  auto read_x = [&](int t, auto nc, u32x4 (&o)[2]) {
    constexpr int n = decltype(nc)::value;
    const uint32_t st = x_row + (t % P_X) * P_ST;
#pragma unroll
    for (int p = 0; p < 2; ++p) ldsop::ds_b128<n * 2048>(o[p], st + ch[p]);
  };
  // the wave's 8 operands of W and its first of X, a pair of DMA instructions after every four reads
  auto load_phase = [&](int t, int dma_t, uint8_t* dma_st) {
    const uint32_t st = w_row + (t & 1) * P_ST;
    unroll<0, 4>([&](auto qc) {
      constexpr int j = decltype(qc)::value;
#pragma unroll
      for (int p = 0; p < 2; ++p) {
        ldsop::ds_b128<2 * j * 2048>(wop[2 * j][p], st + ch[p]);
        ldsop::ds_b128<(2 * j + 1) * 2048>(wop[2 * j + 1][p], st + ch[p]);
      }
      if (dma_t >= 0) {
        fill(dma_t, dma_st, 2 * j);
        fill(dma_t, dma_st, 2 * j + 1);
      }
    });
    read_x(t, std::integral_constant<int, 0>{}, xop0);
    __builtin_amdgcn_sched_barrier(0);
    wait_lgkm0();
    __builtin_amdgcn_sched_barrier(0);
#pragma unroll
    for (int f = 0; f < 8; ++f)
#pragma unroll
      for (int p = 0; p < 2; ++p) ldsop::landed(wop[f][p]);
    ldsop::landed(xop0[0]);
    ldsop::landed(xop0[1]);
  };
  auto compute_phase = [&](int t, const Scales& s) {
    u32x4 x[3][2];  // ring: operand n in x[n % 3], read two ahead
    x[0][0] = xop0[0];
    x[0][1] = xop0[1];
    read_x(t, std::integral_constant<int, 1>{}, x[1]);
    unroll<0, 4>([&](auto nc) {
      constexpr int n = decltype(nc)::value;
      if constexpr (n + 2 < 4) read_x(t, std::integral_constant<int, n + 2>{}, x[(n + 2) % 3]);
      __builtin_amdgcn_sched_barrier(0);
      if constexpr (n + 2 < 4) wait_lgkm<4>();
      else if constexpr (n + 1 < 4) wait_lgkm<2>();
      else wait_lgkm<0>();
      __builtin_amdgcn_sched_barrier(0);
      ldsop::landed(x[n % 3][0]);
      ldsop::landed(x[n % 3][1]);
      unroll<0, 8>([&](auto fc) {
        constexpr int f = decltype(fc)::value;
        acc[f][n] = mma<f % 4, n>(cat8(wop[f][0], wop[f][1]), cat8(x[n % 3][0], x[n % 3][1]), acc[f][n], s.w[f / 4], s.x);
      });
    });
  };
  Scales cur = scales_of(0);
  if (KT == 1) mask_tail(cur, 0);
  // prologue: W of step 0 (group 0), X of steps 0 and 1 (group 1)
  if (grp == 0) {
#pragma unroll
    for (int j = 0; j < 8; ++j) fill(0, w_st(0), j);
  } else {
#pragma unroll
    for (int j = 0; j < 8; ++j) fill(0, x_st(0), j);
    if (1 < KT) {
#pragma unroll
      for (int j = 0; j < 8; ++j) fill(1, x_st(1), j);
    }
  }
  wait_vm<0>();
  barrier();
  if (grp == 0) {
    for (int t = 0; t < KT; ++t) {
      Scales nxt = scales_of(min(t + 1, KT - 1));
      load_phase(t, t + 1 < KT ? t + 1 : -1, w_st(t + 1));
      barrier();
      compute_phase(t, cur);
      wait_vm<0>();  // W of t + 1 and its scales
      cur = nxt;
      if (t + 2 == KT) mask_tail(cur, t + 1);
      barrier();
    }
    barrier();  // group 1 multiplies the last step
  } else {
    barrier();
    for (int t = 0; t < KT; ++t) {
      const bool more = t + 2 < KT;
      Scales nxt = scales_of(min(t + 1, KT - 1));
      load_phase(t, more ? t + 2 : -1, x_st(t + 2));
      // X of t + 1 (issued a load phase ago) and the scales, older than this phase's 8, have landed
      if (more) wait_vm<8>();
      else wait_vm<0>();
      barrier();
      compute_phase(t, cur);
      cur = nxt;
      if (t + 2 == KT) mask_tail(cur, t + 1);
      barrier();
    }
  }

  // ---- the lane's rows are m0 + 64 quarter + 4 i + t, its columns 16 g + 4 e + f of a group
  const int i = lane & 15, g = lane >> 4;
  if constexpr (DUAL) {
    const int col = n0 + 64 * grp + 16 * g;
    uint32_t byte[4];
    unroll<0, 4>([&](auto tc) {
      constexpr int t = decltype(tc)::value;
      const int row = m0 + 64 * quarter + 4 * i + t;
      float v[16];
      uint32_t m = 0;
#pragma unroll
      for (int e = 0; e < 4; ++e)
#pragma unroll
        for (int f = 0; f < 4; ++f) {
          v[4 * e + f] = gated(acc[f][t][e], acc[4 + f][t][e]);
          m = max(m, mx8::abs_bits(v[4 * e + f]));
        }
      byte[t] = mx8::scale_byte(xrow_max_bits(m));
      const float inv = mx8::inverse(byte[t]);
      u32x4 p;
#pragma unroll
      for (int e = 0; e < 4; ++e)
        p[e] = mx8::codes4(v[4 * e], v[4 * e + 1], v[4 * e + 2], v[4 * e + 3], inv, byte[t] < 255);
      if (row < M && col < N) *(u32x4*)((uint8_t*)a.c + (int64_t)row * N + col) = p;
    });
    if ((g & 1) == 0 && col < N) {
      const int row = m0 + 64 * quarter + 4 * i;
      uint8_t* const s = a.c_scales + mx8::scale_at(row, col / BLOCK, (N + 127) / 128);
      if (row + 4 <= M) *(uint32_t*)s = byte[0] | byte[1] << 8 | byte[2] << 16 | byte[3] << 24;
      else
        for (int t = 0; t < 3; ++t)
          if (row + t < M) s[t] = (uint8_t)byte[t];
    }
  } else {
    const bool vec = N % 8 == 0 && ((uintptr_t)a.c & 15) == 0;
    unroll<0, 4>([&](auto tc) {
      constexpr int t = decltype(tc)::value;
      const int row = m0 + 64 * quarter + 4 * i + t;
      if (row >= M) return;
      unroll<0, 2>([&](auto pc) {
        constexpr int p = decltype(pc)::value;
        const int col = n0 + 128 * grp + 64 * p + 16 * g;
        float v[16];
#pragma unroll
        for (int e = 0; e < 4; ++e)
#pragma unroll
          for (int f = 0; f < 4; ++f) v[4 * e + f] = acc[4 * p + f][t][e];
        store16<OUT>((uint16_t*)a.c + (int64_t)row * N + col, v, (int64_t)N - col, vec);
      });
    });
  }
}

template <int OUT>
int direct(const Args& a, hipStream_t s) {
  constexpr int NF = OUT == TLM_F8E4M3 ? 2 : 1;
  const int mt = a.M <= 16 ? 1 : a.M <= 32 ? 2 : 4;
  if (a.M > 256 && a.K > 0) {
    const int bn = OUT == TLM_F8E4M3 ? P_N / 2 : P_N;
    const int64_t tiles = ((a.M + P_M - 1) / P_M) * ((a.N + bn - 1) / bn);
    gemm_mx8_256<OUT><<<(unsigned)tiles, P_T, 0, s>>>(a);
    return TLM_OK;
  }
  const dim3 grid((unsigned)((a.N + 16 * NF - 1) / (16 * NF)), (unsigned)((a.M + 16 * mt - 1) / (16 * mt)));
  auto go = [&](auto kern) { kern<<<grid, 64 * D_WAVES, 0, s>>>(a); };
  if (mt == 1) go(gemm_mx8_direct<1, NF, OUT>);
  else if (mt == 2) go(gemm_mx8_direct<2, NF, OUT>);
  else go(gemm_mx8_direct<4, NF, OUT>);
  return TLM_OK;
}

int check_sizes(const char* fn, int64_t M, int64_t N, int64_t K) {
  if (M < 0 || N < 0 || K < 0 || M > INT32_MAX - 255 || N > INT32_MAX - 255 || M > 64 * 65535) {
    tlm_set_error("%s: bad sizes M=%lld N=%lld K=%lld", fn, (long long)M, (long long)N, (long long)K);
    return TLM_EINVAL;
  }
  return TLM_OK;
}

}  // namespace

extern "C" int tlm_gemm_mx8(const void* a, const void* a_scales, const void* b, const void* b_scales, void* c,
                            int64_t M, int64_t N, int64_t K, int out_dtype, void* stream) {
  if (int rc = check_sizes("tlm_gemm_mx8", M, N, K)) return rc;
  if (int rc = mx8::check("tlm_gemm_mx8", "A", a, a_scales, M, K)) return rc;
  if (int rc = mx8::check("tlm_gemm_mx8", "B", b, b_scales, N, K)) return rc;
  if (out_dtype != TLM_F16 && out_dtype != TLM_BF16) {
    tlm_set_error("tlm_gemm_mx8: out dtype %d unsupported (F16 or BF16)", out_dtype);
    return TLM_EUNSUPPORTED;
  }
  if (M == 0 || N == 0) return TLM_OK;
  if (!c) {
    tlm_set_error("tlm_gemm_mx8: null pointer argument");
    return TLM_EINVAL;
  }
  if (!tlm_aligned(c, 2)) {
    tlm_set_error("tlm_gemm_mx8: misaligned C");
    return TLM_EINVAL;
  }
  const Args g{{(const uint8_t*)a, (const uint8_t*)a_scales}, {(const uint8_t*)b, (const uint8_t*)b_scales}, {},
               c, nullptr, M, N, (int)K, (int)((K + 127) / 128)};
  hipStream_t s = (hipStream_t)stream;
  out_dtype == TLM_BF16 ? direct<TLM_BF16>(g, s) : direct<TLM_F16>(g, s);
  TLM_LAUNCH_CHECK("tlm_gemm_mx8");
  return TLM_OK;
}

extern "C" int tlm_gemm_mx8_swiglu(const void* a, const void* a_scales, const void* gate, const void* gate_scales,
                                   const void* up, const void* up_scales, void* codes, void* scales, int64_t M,
                                   int64_t N, int64_t K, void* stream) {
  if (int rc = check_sizes("tlm_gemm_mx8_swiglu", M, N, K)) return rc;
  if (int rc = mx8::check("tlm_gemm_mx8_swiglu", "A", a, a_scales, M, K)) return rc;
  if (int rc = mx8::check("tlm_gemm_mx8_swiglu", "B_gate", gate, gate_scales, N, K)) return rc;
  if (int rc = mx8::check("tlm_gemm_mx8_swiglu", "B_up", up, up_scales, N, K)) return rc;
  if (int rc = mx8::check("tlm_gemm_mx8_swiglu", "the result", codes, scales, M, N)) return rc;
  if (M == 0 || N == 0) return TLM_OK;
  const Args g{{(const uint8_t*)a, (const uint8_t*)a_scales},
               {(const uint8_t*)gate, (const uint8_t*)gate_scales},
               {(const uint8_t*)up, (const uint8_t*)up_scales},
               codes, (uint8_t*)scales, M, N, (int)K, (int)((K + 127) / 128)};
  direct<TLM_F8E4M3>(g, (hipStream_t)stream);
  TLM_LAUNCH_CHECK("tlm_gemm_mx8_swiglu");
  return TLM_OK;
}
