// Products of 8-bit operands with power-of-two scales: C = A B^T, and SwiGLU of two of them with an 8-bit result.
//
//   c[m][n] = sum over blocks b of 32 k:  2^(ea[m][b] + eb[n][b]) sum over the block of a[m][k] b[n][k]
//
// v_mfma_scale_f32_16x16x128_f8f6f4 multiplies each block of 32 k by 2^(ea + eb) as it adds it, at 35 cycles instead of the
// plain form's 32. Lane l holds row l % 16 of its operand and the 16-byte chunks q and q + 4 of its 128 k (q = l / 16), and the
// scale of k block q. The weights are the first operand, so that a lane's sums are neighbouring columns of one row of C. The
// sums are fp32, but before they are added the products of 8 neighbouring k are cut, towards zero, below 2^-13 of the largest
// 2^(exponent of a + exponent of b) among them (codes below the least normal one have its exponent): 4e-5 of a random result of
// K 4096, and at worst 7 2^-13 of the sum of the groups' largest. So no 32-bit C is offered, and gated products, whose 8-bit results
// would show it, are summed in fp32 by a form of the tiles that widens its operands (WIDE, below), as a caller may ask of both.
//
// Tiles of 16 to 256 rows, chosen by a model of their time (choose, below). Few rows wait for the stream of B, some hundreds for
// the operands' way from L2 to a CU, whole prompts for the matrix cores' power, where sums are of fp32 for the conversions of the
// operands as well. Measured in us, several cards: 16 x 4096 x 14336 11.3 with weights in the 256 MB cache, 15 to 17 from HBM; 500 x 4096
// x 4096 13.4 to 15; 4096^3 50 to 55 (2.5 to 2.7 PFLOP/s; the library's product without scales 51 to 52); gated 64 x 2048 x 7168 12
// (by the 8-bit instruction 11), gated 4096 x 11008 x 4096 700 to 790 (290).
#include "tlm_gemm_tile.h"
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
  int K, kt;   // kt: k steps of 128
  int64_t ld;  // columns of the whole result, of which a call may compute a part
};

template <int SA, int SB>
TLM_DEV f32x4 mma(const i32x8& a, const i32x8& b, f32x4 c, uint32_t sa, uint32_t sb) {
  return __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(a, b, c, 0, 0, SA, (int)sa, SB, (int)sb);
}

using ldsop::unroll;

// up * silu(gate).
TLM_DEV float gated(float gate, float up) { return up * (gate * __builtin_amdgcn_rcpf(fast_exp(-gate) + 1.0f)); }

// ---- whole prompts: 256 x 256 tiles

// Four waves, one per SIMD, of 128 x 128 each: their sums fill the accumulation registers, and LDS is read a third less than by
// eight waves of 128 x 64 that take turns (57.9 us at 4096^3, now 52 to 55). A wave multiplies without a pause: beside the
// products of a k step it reads the rest of the step's operands of X (the rows of A; a ring of four registers), all of the next
// step's of W, and issues the LDS-DMA of steps to come. A step takes 2,420 cycles, its 64 products alone 2,240; the clock is
// what power leaves, 1.5 to 1.7 GHz with data and 2.2 with zeros.
//
// Slot 16 f + i of a 64-row group of an LDS stage holds row 4 i + f, so that operand f, read from 16 neighbouring slots, has the
// rows whose scales are byte f of the lanes' words: four words a k step, loaded a step ahead, are all the scales a wave needs. Of
// the sums, a lane then has 16 neighbouring columns of each of its rows: C is stored, or a block of 32 quantised with one
// exchange between two lanes, without a way through LDS.
constexpr int P_T = 256, P_M = 256, P_N = 256, P_ST = 256 * 128;  // P_ST: bytes of a stage of one operand
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

// W neighbouring columns of a row of C (16; 4 or 8 of narrow tiles), the first `left` of them there. Rows of any width start on
// any element: the wide stores are such as need no alignment beyond an element's (4096 x 4091 x 4096 65 us, with 2-byte stores 95).
template <int OUT, int W>
TLM_DEV void store_cols(uint16_t* c, const float (&v)[W], int64_t left) {
  using H = h16<OUT == TLM_BF16>;
  constexpr int P = W < 8 ? W : 8;
  typedef uint32_t any __attribute__((ext_vector_type(P / 2), aligned(2)));
  if (left >= W) {
#pragma unroll
    for (int h = 0; h < W / P; ++h) {
      any x;
#pragma unroll
      for (int j = 0; j < P / 2; ++j) x[j] = H::pack(v[P * h + 2 * j], v[P * h + 2 * j + 1]);
      *(any*)(c + P * h) = x;
    }
    return;
  }
#pragma unroll
  for (int j = 0; j < W; ++j)
    if (j < left) c[j] = (uint16_t)H::from_f32(v[j]);
}

TLM_DEV uint32_t xrow_max_bits(uint32_t m) {  // of lanes l and l ^ 16
  const auto r = __builtin_amdgcn_permlane16_swap(m, m, false, false);
  return max(r[0], r[1]);
}

TLM_DEV uint32_t xhalf_max_bits(uint32_t m) {  // of lanes l and l ^ 32
  const auto r = __builtin_amdgcn_permlane32_swap(m, m, false, false);
  return max(r[0], r[1]);
}

// c += the product, in place in the accumulation registers: left to itself, the compiler lets 256 of them change places from step
// to step and spends 168 moves on that in two of them. It knows no matrix instruction here, so nothing else reads or writes c
// until settle(), operands come from waited LDS reads, and 64 of these lie between two on the same c.
template <int SA, int SB>
TLM_DEV void mma_in_place(f32x4& c, const i32x8& a, const i32x8& b, uint32_t sa, uint32_t sb) {
  asm volatile("v_mfma_scale_f32_16x16x128_f8f6f4 %0, %1, %2, %0, %3, %4 op_sel:[%5,%6,0] op_sel_hi:[%7,%8,0]"
               : "+a"(c)
               : "v"(a), "v"(b), "v"(sa), "v"(sb), "n"(SA & 1), "n"(SB & 1), "n"(SA >> 1), "n"(SB >> 1));
}
TLM_DEV void pin(f32x4& c) { asm volatile("" : "+a"(c)); }
// The last products' results can be read (18 wait states), the first ones' operands have been written.
TLM_DEV void settle() { asm volatile("s_nop 15\n\ts_nop 15" ::: "memory"); }

template <int OUT>
__global__ __launch_bounds__(P_T, 1) void gemm_mx8_256(Args a) {
  constexpr bool DUAL = OUT == TLM_F8E4M3;
  constexpr int BN = DUAL ? P_N / 2 : P_N;  // columns of the result
  __shared__ __attribute__((aligned(1024))) uint8_t smem[(P_W + P_X) * P_ST];
  const int tid = threadIdx.x, lane = tid & 63;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int wm = wave >> 1, wn = wave & 1;  // 128 rows of X, of W
  const int M = (int)a.M, N = (int)a.N, K = a.K, KT = a.kt;
  int tm, tn;
  tile_of(blockIdx.x, (M + P_M - 1) / P_M, (N + BN - 1) / BN, tm, tn);
  const int m0 = tm * P_M, n0 = tn * BN;

  // ---- LDS-DMA: wave w fills the 64 slots of group w of both stages (gated: gate and up groups alternate), 8 an instruction:
  // instruction j slots 8 j + lane / 8, rows 32 (j % 2) + 4 (lane / 8) + j / 2. What is past the last row or k, and every step from
  // KT on, lies past the descriptor's end and gives zeros.
  const int rw = n0 + (DUAL ? 64 * (wave >> 1) : 64 * wave), rx = m0 + 64 * wave;
  const uint8_t* const w_base = (DUAL && (wave & 1) ? a.b2.codes : a.b.codes) + (int64_t)min(rw, N) * K;
  const uint8_t* const x_base = a.a.codes + (int64_t)min(rx, M) * K;
  const int w_end = max(0, min(64, N - rw)) * K, x_end = max(0, min(64, M - rx)) * K;
  int chunk[2];
  uint32_t off[2];
#pragma unroll
  for (int h = 0; h < 2; ++h) {
    chunk[h] = 16 * ((lane & 7) ^ (4 * h + (lane >> 4)));
    off[h] = (uint32_t)((32 * h + 4 * (lane >> 3)) * K + chunk[h]);
  }
  auto fill = [&](const uint8_t* base, int end, int t, uint8_t* st, int j) __attribute__((always_inline)) {
    const uint32_t o = chunk[j & 1] < K - t * 128 ? off[j & 1] : OOB;
    dma16(base + (int64_t)t * 128, t < KT ? max(0, end - t * 128) : 0, st + wave * 8192 + j * 1024, o + (j >> 1) * K);
  };
  auto fill_w = [&](int t, int j) __attribute__((always_inline)) { fill(w_base, w_end, t, smem + (t & 1) * P_ST, j); };
  auto fill_x = [&](int t, int j) __attribute__((always_inline)) {
    fill(x_base, x_end, t, smem + (P_W + t % P_X) * P_ST, j);
  };

  // ---- scales: words of the wave's two groups of W and of X; past the last row, another's
  auto words = [&](const uint8_t* s, int r, int n) {
    return s + (int64_t)(min(r, n - 1) >> 6) * KT * 256 + 4 * lane;
  };
  const uint8_t* const sw0 = words(a.b.scales, n0 + (DUAL ? 64 : 128) * wn, N);
  const uint8_t* const sw1 = DUAL ? words(a.b2.scales, n0 + 64 * wn, N) : words(a.b.scales, n0 + 128 * wn + 64, N);
  const uint8_t* const sx0 = words(a.a.scales, m0 + 128 * wm, M);
  const uint8_t* const sx1 = words(a.a.scales, m0 + 128 * wm + 64, M);
  struct Scales {
    uint32_t w[2], x[2];
  };
  auto scales_of = [&](int t) __attribute__((always_inline)) {
    const int64_t o = (int64_t)t * 256;
    return Scales{{*(const uint32_t*)(sw0 + o), *(const uint32_t*)(sw1 + o)},
                  {*(const uint32_t*)(sx0 + o), *(const uint32_t*)(sx1 + o)}};
  };

  // ---- operands
  const uint32_t xr = ((lane & 15) >> 1) & 7;
  const uint32_t w_row = ldsop::lds_u32(smem) + (wn * 128 + (lane & 15)) * 128;
  const uint32_t x_row = ldsop::lds_u32(smem) + P_W * P_ST + (wm * 128 + (lane & 15)) * 128;
  uint32_t ch[2];
#pragma unroll
  for (int p = 0; p < 2; ++p) ch[p] = 16 * ((4 * p + (lane >> 4)) ^ xr);
  f32x4 acc[8][8];
#pragma unroll
  for (int f = 0; f < 8; ++f)
#pragma unroll
    for (int n = 0; n < 8; ++n) {
      acc[f][n] = f32x4{};
      pin(acc[f][n]);
    }
  u32x4 wa[8][2], wb[8][2], x[4][2];
  auto read_w = [&](uint32_t st, u32x4 (&o)[8][2], auto rc) __attribute__((always_inline)) {
    constexpr int r = decltype(rc)::value;
    ldsop::ds_b128<r / 2 * 2048>(o[r / 2][r % 2], w_row + st + ch[r % 2]);
  };
  auto read_x = [&](uint32_t st, auto rc) __attribute__((always_inline)) {  // half r % 2 of operand r / 2
    constexpr int r = decltype(rc)::value;
    ldsop::ds_b128<r / 2 * 2048>(x[r / 2 % 4][r % 2], x_row + st + ch[r % 2]);
  };

  // ---- k step t, W in `w`: eight products with each operand of X. Operand n + 2 is read beside those of operand n, W of step t + 1
  // beside the first five. Before operand 6 all waves meet: they have read what is left of step t and all of W of t + 1, and X of
  // t + 1 and W of t + 2 have landed. From there on the first two operands of X of t + 1 are read. Two LDS-DMA instructions go
  // with every operand (more at once would wait at issue, and the products with them): W of t + 3 with the last two and the next
  // step's first two, X of t + 2 with the four between, which the next meeting waits for.
  constexpr int W_READS[8] = {4, 3, 3, 3, 3, 0, 0, 0}, W_FIRST[8] = {0, 4, 7, 10, 13, 16, 16, 16};
  auto kstep = [&](int t, u32x4 (&w)[8][2], u32x4 (&next)[8][2], Scales& s) __attribute__((always_inline)) {
    if (t == KT - 1 && t * 128 + 32 * (lane >> 4) >= K)  // past K: codes 0, scale 1
      s = Scales{{0x7f7f7f7fu, 0x7f7f7f7fu}, {0x7f7f7f7fu, 0x7f7f7f7fu}};
    const uint32_t xs = (uint32_t)(t % P_X) * P_ST, xn = (uint32_t)((t + 1) % P_X) * P_ST;
    const uint32_t ws = (uint32_t)((t + 1) & 1) * P_ST;
    Scales ahead;
    unroll<0, 8>([&](auto nc) __attribute__((always_inline)) {
      constexpr int n = decltype(nc)::value;
      __builtin_amdgcn_sched_barrier(0);
      // operand n has landed; younger reads may be under way
      if constexpr (n < 6) wait_lgkm<(n > 1 ? W_READS[n - 2] : 0) + 2 + (n > 0 ? W_READS[n - 1] : 0)>();
      else if constexpr (n == 6) {
        wait_vm<8>();
        barrier();
      }
      __builtin_amdgcn_sched_barrier(0);
      ldsop::landed(x[n % 4][0]);
      ldsop::landed(x[n % 4][1]);
      if constexpr (n == 0) {
#pragma unroll
        for (int f = 0; f < 8; ++f)
#pragma unroll
          for (int p = 0; p < 2; ++p) ldsop::landed(w[f][p]);
        ahead = scales_of(min(t + 1, KT - 1));
        asm volatile("s_nop 1" : "+v"(s.w[0]), "+v"(s.w[1]), "+v"(s.x[0]), "+v"(s.x[1]));
      }
      unroll<0, 8>([&](auto fc) __attribute__((always_inline)) {
        constexpr int f = decltype(fc)::value;
        mma_in_place<f % 4, n % 4>(acc[f][n], cat8(w[f][0], w[f][1]), cat8(x[n % 4][0], x[n % 4][1]), s.w[f / 4], s.x[n / 4]);
        if constexpr (f < 2) {
          if constexpr (n < 6) read_x(xs, std::integral_constant<int, 2 * (n + 2) + f>{});
          else read_x(xn, std::integral_constant<int, 2 * (n - 6) + f>{});
        } else if constexpr (f < 6) {
          if constexpr (f - 2 < W_READS[n]) read_w(ws, next, std::integral_constant<int, W_FIRST[n] + f - 2>{});
        } else if constexpr (n < 2) {
          fill_w(t + 2, 4 + 2 * n + f - 6);
        } else if constexpr (n < 6) {
          fill_x(t + 2, 2 * (n - 2) + f - 6);
        } else {
          fill_w(t + 3, 2 * (n - 6) + f - 6);
        }
        __builtin_amdgcn_sched_barrier(0);
      });
    });
    s = ahead;
  };
  Scales s = {};
  if (KT > 0) s = scales_of(0);  // without k there are none
#pragma unroll
  for (int j = 0; j < 8; ++j) fill_w(0, j);
#pragma unroll
  for (int j = 0; j < 8; ++j) fill_x(0, j);
#pragma unroll
  for (int j = 0; j < 8; ++j) fill_w(1, j);
#pragma unroll
  for (int j = 0; j < 8; ++j) fill_x(1, j);
  wait_vm<8>();
  barrier();
  unroll<0, 16>([&](auto rc) __attribute__((always_inline)) { read_w(0, wa, rc); });
  wait_vm<8>();
  barrier();
#pragma unroll
  for (int j = 0; j < 4; ++j) fill_w(2, j);
  unroll<0, 4>([&](auto rc) __attribute__((always_inline)) { read_x(0, rc); });
  int t = 0;
  for (; t + 1 < KT; t += 2) {
    kstep(t, wa, wb, s);
    kstep(t + 1, wb, wa, s);
  }
  if (t < KT) kstep(t, wa, wb, s);
  wait_vm<0>();  // nothing is written to LDS that is no longer the workgroup's
  wait_lgkm0();
  settle();
#pragma unroll
  for (int f = 0; f < 8; ++f)
#pragma unroll
    for (int n = 0; n < 8; ++n) pin(acc[f][n]);

  // ---- the lane's rows are m0 + 128 wm + 64 (n / 4) + 4 i + n % 4, its columns 16 g + 4 e + f of a group
  const int i = lane & 15, g = lane >> 4;
  if constexpr (DUAL) {
    const int col = n0 + 64 * wn + 16 * g;
    unroll<0, 2>([&](auto hc) __attribute__((always_inline)) {
      constexpr int h = decltype(hc)::value;
      const int row0 = m0 + 128 * wm + 64 * h + 4 * i;
      uint32_t byte[4];
      unroll<0, 4>([&](auto tc) __attribute__((always_inline)) {
        constexpr int r = decltype(tc)::value, n = 4 * h + r;
        float v[16];
        uint32_t m = 0;
#pragma unroll
        for (int e = 0; e < 4; ++e)
#pragma unroll
          for (int f = 0; f < 4; ++f) {
            v[4 * e + f] = gated(acc[f][n][e], acc[4 + f][n][e]);
            m = max(m, mx8::abs_bits(v[4 * e + f]));
          }
        byte[r] = mx8::scale_byte(xrow_max_bits(m));
        const float inv = mx8::inverse(byte[r]);
        u32x4 p;
#pragma unroll
        for (int e = 0; e < 4; ++e)
          p[e] = mx8::codes4(v[4 * e], v[4 * e + 1], v[4 * e + 2], v[4 * e + 3], inv, byte[r] < 255);
        if (row0 + r < M && col < N) *(u32x4*)((uint8_t*)a.c + (row0 + r) * a.ld + col) = p;
      });
      if ((g & 1) == 0 && col < N) {
        uint8_t* const sc = a.c_scales + mx8::scale_at(row0, col / BLOCK, (int)((a.ld + 127) / 128));
        if (row0 + 4 <= M) {
          *(uint32_t*)sc = byte[0] | byte[1] << 8 | byte[2] << 16 | byte[3] << 24;
        } else {
#pragma unroll
          for (int r = 0; r < 3; ++r)
            if (row0 + r < M) sc[r] = (uint8_t)byte[r];
        }
      }
    });
  } else {
    unroll<0, 8>([&](auto nc) __attribute__((always_inline)) {
      constexpr int n = decltype(nc)::value;
      const int row = m0 + 128 * wm + 64 * (n / 4) + 4 * i + n % 4;
      if (row >= M) return;
      unroll<0, 2>([&](auto pc) __attribute__((always_inline)) {
        constexpr int p = decltype(pc)::value;
        const int col = n0 + 128 * wn + 64 * p + 16 * g;
        float v[16];
#pragma unroll
        for (int e = 0; e < 4; ++e)
#pragma unroll
          for (int f = 0; f < 4; ++f) v[4 * e + f] = acc[4 * p + f][n][e];
        store_cols<OUT>((uint16_t*)a.c + row * a.ld + col, v, (int64_t)N - col);
      });
    });
  }
}

// ---- between one decode step and whole prompts: smaller tiles, K split where they are fewer than the CUs

// What bounds it: the stream of B with few rows, with more the rate at which a CU takes operand tiles from L2 (40 to 48 B/clk).
// Four waves only fill the ring: an LDS-DMA instruction waits at issue while the CU has enough of them under way, and a wave
// that multiplies would wait with it (500 x 4096 x 4096 16.8 us, with waves of their own on the same card 13.7). NC others are
// BM / (16 FX) x BN / 64 wave tiles times KG k-groups. A stage of the NST-stage ring holds KG k steps, one for each k-group, and their scales;
// the operands of stage t are read from LDS while the products of stage t - 1 run. The k-groups' sums meet in LDS, those of the
// `ns` workgroups that share a tile's K in memory, where the last to arrive adds them in order: the result does not depend on
// the order of arrival.
//
// Narrow tiles, of 16 or 32 columns, give few rows' products a workgroup per CU without a split, with 512 neighbouring bytes
// of a row in a load: 16 x 4096 x 14336 11.6 instead of 13.1 (64 columns, two workgroups on a tile's K), 1 x 4096 x 11008 10.3
// instead of 12.2, 16 x 8192 x 14336 22.9 instead of 24.5; weights that the 256 MB cache no longer holds, 1 x 4096 x 4096 6.1
// instead of 8.2, 1 x 4096 x 11008 14.2 instead of 14.4, 16 x 4096 x 14336 17.2 where the best split takes 16.6 (another card: 6.1,
// 13.6, 15.0). Up to 7 stages are no faster there. A wave has NF = 1 or 2 operands of W, row NF i + f in slot 16 f + i.
//
// WIDE: the operands are widened to bf16, exactly, and multiplied by v_mfma_f32_16x16x32_bf16, whose sums are those of fp32. What
// the 8-bit instruction cuts off sends 1 in 2,500 of a random gated product's values to the other side of an 8-bit step (an fp16
// MLP ends 2e-3 from the formula instead of 2e-4), and is all there is where large products cancel. So gated products are summed
// this way unless their caller chooses otherwise. It costs half the matrix rate and a conversion of each operand in each wave:
// gated 64 x 2048 x 7168 12.0 us instead of 11.2, 500 x 11008 x 4096 94 instead of 49, 4096 x 11008 x 4096 703 instead of 290;
// conversions that take turns with the matrix instructions, and those all at the start of a step, take the same time. Elements of
// 2^128 and more count as infinite there.
template <int BM_, int BN_, int FX_, int KG_, int NST_, int OUT_, bool WIDE_ = false>
struct Tile {
  static constexpr int BM = BM_, BN = BN_, FX = FX_, KG = KG_, NST = NST_, OUT = OUT_;
  static constexpr bool WIDE = WIDE_;
  static constexpr bool DUAL = OUT == TLM_F8E4M3;
  static constexpr int BNC = DUAL ? BN / 2 : BN;       // columns of the result
  static constexpr int NF = BN < 64 ? BN / 16 : 4;      // operands of W per wave
  static constexpr int WM = BM / (16 * FX), WN = BN / (16 * NF);
  static constexpr int NC = WM * WN * KG, NP = 4;      // waves that multiply, waves that load
  static constexpr int BKB = 128 * KG;                 // bytes of k per stage
  static constexpr int SX = BM * BKB, SW = BN * BKB;
  static constexpr int GX = (BM + 63) / 64, GW = DUAL ? 2 * ((BNC + 63) / 64) : (BN + 63) / 64;  // 64-row groups of scales
  static constexpr int NX = SX / (NP * 1024), NW = SW / (NP * 1024);  // LDS-DMA instructions per wave: codes
  static constexpr int NSC = (GX + GW + NP - 1) / NP;                 // and scales, 1 KB per group: KG k steps and nothing
  static constexpr int PER = NX + NW + NSC;
  static constexpr int ST = SX + SW + NSC * NP * 1024;
  static constexpr int TO = FX > KG ? FX / KG : 1, FIN = FX > KG ? KG : FX;  // operands of X that a k-group finishes, k-groups that do
  static constexpr int RED = KG > 1 ? NC * NF * FX * 1024 : 0;
  static constexpr int SMEM = NST * ST > RED ? NST * ST : RED;
  static constexpr int THREADS = 64 * (NC + NP);
  static_assert((NC == 4 || NC == 8) && KG <= 4 && NX * NP * 1024 == SX && NW * NP * 1024 == SW && SMEM <= 160 * 1024, "layout");
};

template <int BKB>
TLM_DEV int swz(int slot) {  // 16 lanes that read one chunk of 16 neighbouring slots hit all banks
  return BKB == 128 ? (slot >> 1) & 7 : slot & 15;
}
template <int OFF>
TLM_DEV void ds_b32(uint32_t& r, uint32_t a) {
  asm volatile("ds_read_b32 %0, %1 offset:%2" : "=v"(r) : "v"(a), "i"(OFF) : "memory");
}
template <int OFF>
TLM_DEV void ds_u16(uint32_t& r, uint32_t a) {
  asm volatile("ds_read_u16 %0, %1 offset:%2" : "=v"(r) : "v"(a), "i"(OFF) : "memory");
}
template <int OFF>
TLM_DEV void ds_u8(uint32_t& r, uint32_t a) {
  asm volatile("ds_read_u8 %0, %1 offset:%2" : "=v"(r) : "v"(a), "i"(OFF) : "memory");
}
TLM_DEV void landed1(uint32_t& a) { asm volatile("" : "+v"(a)); }
TLM_DEV void plain_barrier() {
  __builtin_amdgcn_sched_barrier(0);
  asm volatile("" ::: "memory");
  __builtin_amdgcn_s_barrier();
  asm volatile("" ::: "memory");
  __builtin_amdgcn_sched_barrier(0);
}

// A lane's 32 codes as bf16, times the scales in byte B of s (one for each half).
template <int B>
TLM_DEV void widen(bf16x8 (&o)[4], const u32x4 (&x)[2], const uint32_t (&s)[2]) {
  typedef __bf16 b2 __attribute__((ext_vector_type(2)));
#pragma unroll
  for (int h = 0; h < 2; ++h) {
    const float scale = __uint_as_float((s[h] >> (8 * B) & 255u) << 23);
#pragma unroll
    for (int d = 0; d < 4; ++d) {
      const b2 lo = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(x[h][d], scale, false);
      const b2 hi = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(x[h][d], scale, true);
      const int j = 4 * (d & 1);
      o[2 * h + d / 2][j] = lo[0], o[2 * h + d / 2][j + 1] = lo[1];
      o[2 * h + d / 2][j + 2] = hi[0], o[2 * h + d / 2][j + 3] = hi[1];
    }
  }
}

template <typename T>
__global__ __launch_bounds__(T::THREADS, 1) void gemm_mx8_tile(Args a, int ns, float* __restrict__ part,
                                                               unsigned* __restrict__ arrivals) {
  constexpr int BKB = T::BKB, KG = T::KG, FX = T::FX, NST = T::NST;
  constexpr bool DUAL = T::DUAL;
  constexpr int NF = T::NF;
  __shared__ __attribute__((aligned(1024))) uint8_t smem[T::SMEM];
  const int tid = threadIdx.x, lane = tid & 63;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const bool multiplies = wave < T::NC;
  const int sp = wave / KG, kg = wave % KG;
  const int wm = sp / T::WN, wn = sp % T::WN;
  const int M = (int)a.M, N = (int)a.N, K = a.K;

  // XCD x takes a contiguous range of (split, column tile, row tile), row tiles fastest: they share a strip of B
  const int tiles_m = (M + T::BM - 1) / T::BM, tiles_n = (N + T::BNC - 1) / T::BNC;
  const int tiles = tiles_m * tiles_n, total = tiles * ns, xcd = blockIdx.x & 7;
  const int lin = xcd * (total >> 3) + min(xcd, total & 7) + (blockIdx.x >> 3);
  const int tile = lin % tiles, split = lin / tiles;
  const int m0 = tile % tiles_m * T::BM, n0 = tile / tiles_m * T::BNC;
  const int lo = (int)((int64_t)split * a.kt / ns), hi = (int)((int64_t)(split + 1) * a.kt / ns);  // k steps
  const int n = (hi - lo + KG - 1) / KG;          // stages
  const int kend = min(K, hi * 128) - lo * 128;  // bytes of k
  const int i = lane & 15, q = lane >> 4;
  f32x4 acc[NF][FX];

  // Stage t lives at t % NST. Before barrier t the loading waves wait for stage t; after it stage t - 1, whose operands every wave
  // has read by then, takes stage t + NST - 1.
  if (!multiplies) {
    const int pw = wave - T::NC;
    uint32_t off[T::NX + T::NW];  // a lane's offset from the stage's first k, and its k within the stage
    int kch[T::NX + T::NW];
#pragma unroll
    for (int j = 0; j < T::NX + T::NW; ++j) {
      constexpr int CPR = BKB / 16;
      const int slot = (T::NP * (j < T::NX ? j : j - T::NX) + pw) * (64 / CPR) + lane / CPR;
      const int c = (lane % CPR) ^ swz<BKB>(slot);
      int row;
      if (j < T::NX) row = slot / (16 * FX) * (16 * FX) + FX * (slot & 15) + (slot >> 4) % FX;
      else if (DUAL) row = (slot >> 6) * 32 + 2 * (slot & 15) + (slot >> 4 & 1);
      else row = (slot & ~63) + NF * (slot & 15) + (slot >> 4 & 3);
      off[j] = (uint32_t)(row * K + 16 * c);
      kch[j] = 16 * c;
    }
    const uint8_t* const x_base = a.a.codes + (int64_t)m0 * K + lo * 128;
    const uint8_t* const w_base = a.b.codes + (int64_t)n0 * K + lo * 128;
    const uint8_t* const v_base = (DUAL ? a.b2.codes : a.b.codes) + (int64_t)n0 * K + lo * 128;
    const int x_end = min(M - m0, T::BM) * K - lo * 128, w_end = min(N - n0, T::BNC) * K - lo * 128;
    // scales: X's groups, W's (gated: gate's, then up's); past the last row, another's
    const uint8_t* sc_base[T::NSC];
#pragma unroll
    for (int j = 0; j < T::NSC; ++j) {
      const int g = min(T::NP * j + pw, T::GX + T::GW - 1), h = g - T::GX;
      const Mat& m = h < 0 ? a.a : DUAL && h >= T::GW / 2 ? a.b2 : a.b;
      const int r = h < 0 ? min(m0 + 64 * g, M - 1) : min(n0 + 64 * (DUAL && h >= T::GW / 2 ? h - T::GW / 2 : h), N - 1);
      sc_base[j] = m.scales + (int64_t)(r >> 6) * a.kt * 256;
    }
    auto issue = [&](int t, int stage) __attribute__((always_inline)) {
      uint8_t* const st = smem + stage * T::ST;
      unroll<0, T::NX + T::NW>([&](auto jc) __attribute__((always_inline)) {
        constexpr int j = decltype(jc)::value;
        const uint32_t o = kch[j] < kend - t * BKB ? off[j] : OOB;
        if constexpr (j < T::NX) {
          dma16(x_base + t * BKB, max(0, x_end - t * BKB), st + (T::NP * j + pw) * 1024, o);
        } else {
          constexpr int u = j - T::NX;
          const bool second = DUAL && ((T::NP * u + pw) * (1024 / BKB) >> 5 & 1);
          dma16((second ? v_base : w_base) + t * BKB, max(0, w_end - t * BKB), st + T::SX + (T::NP * u + pw) * 1024, o);
        }
      });
#pragma unroll
      for (int j = 0; j < T::NSC; ++j)
        dma16(sc_base[j], a.kt * 256, st + T::SX + T::SW + (T::NP * j + pw) * 1024,
              lane < 16 * KG ? (uint32_t)((lo + t * KG) * 256 + 16 * lane) : OOB);
    };
#pragma unroll
    for (int t = 0; t < NST - 1; ++t)
      if (t < n) issue(t, t);
    int stage = NST - 1;
    for (int t = 0; t < n; ++t) {
      const int more = min(NST - 2, n - 1 - t);  // stages after t whose loads may stay in flight
      unroll<0, NST - 1>([&](auto ic) __attribute__((always_inline)) {
        constexpr int j = decltype(ic)::value;
        if (more == j) wait_vm<j * T::PER>();
      });
      plain_barrier();
      if (t + NST - 1 < n) issue(t + NST - 1, stage);
      stage = stage == NST - 1 ? 0 : stage + 1;
    }
  } else {
  // ---- operand reads (addresses within stage 0)
  const uint32_t b0 = ldsop::lds_u32(smem);
  uint32_t x_addr[2], w_addr[2];
#pragma unroll
  for (int p = 0; p < 2; ++p) {
    const int x = 16 * ((8 * kg + 4 * p + q) ^ swz<BKB>(i));
    x_addr[p] = b0 + (wm * 16 * FX + i) * BKB + x;
    w_addr[p] = b0 + T::SX + (wn * 16 * NF + i) * BKB + x;
  }
  const uint32_t sc0 = b0 + T::SX + T::SW + kg * 256;
  const int xrow = (m0 & 63) + wm * 16 * FX;  // the wave's rows within the first group
  // the lane's block of the k step: q; wide, where each half of an operand has a scale of its own, q / 2 and q / 2 + 2
  const int blk = T::WIDE ? q >> 1 : q;
  const uint32_t xs_addr = sc0 + (xrow >> 6) * 1024 + blk * 64 + (xrow & 63) + FX * i;
  const int wcol = (n0 & 63) + 32 * wn;  // gated: the wave's columns within the first group
  const uint32_t ws_addr = DUAL ? sc0 + (T::GX + (wcol >> 6)) * 1024 + blk * 64 + (wcol & 63) + 2 * i
                       : NF < 4 ? sc0 + T::GX * 1024 + blk * 64 + (n0 & 63) + NF * i
                                 : sc0 + (T::GX + wn) * 1024 + blk * 64 + 4 * i;
  constexpr int VS = T::GW / 2 * 1024;  // from gate's scales to up's
  constexpr int HALVES = T::WIDE ? 2 : 1;
  struct Ops {
    u32x4 x[FX][2], w[NF][2];
    uint32_t xs[HALVES], ws[HALVES], vs[HALVES];
  };
  constexpr int NR = 2 * FX + 2 * NF + 2;
  auto read1 = [&](Ops& o, uint32_t so, auto ic) __attribute__((always_inline)) {
    constexpr int r = decltype(ic)::value;
    if constexpr (r < 2 * NF) ldsop::ds_b128<r / 2 * 16 * BKB>(o.w[r / 2][r % 2], w_addr[r % 2] + so);
    else if constexpr (r < 2 * NF + 2 * FX)
      ldsop::ds_b128<(r - 2 * NF) / 2 * 16 * BKB>(o.x[(r - 2 * NF) / 2][r % 2], x_addr[r % 2] + so);
    else
      unroll<0, HALVES>([&](auto hc) __attribute__((always_inline)) {
        constexpr int h = decltype(hc)::value;
        if constexpr (r == 2 * NF + 2 * FX) {
          if constexpr (FX == 4) ds_b32<128 * h>(o.xs[h], xs_addr + so);
          else if constexpr (FX == 1) ds_u8<128 * h>(o.xs[h], xs_addr + so);
          else ds_u16<128 * h>(o.xs[h], xs_addr + so);
        } else if constexpr (DUAL) {
          ds_u16<128 * h>(o.ws[h], ws_addr + so);
          ds_u16<128 * h>(o.vs[h], ws_addr + VS + so);
        } else if constexpr (NF == 2) {
          ds_u16<128 * h>(o.ws[h], ws_addr + so);
        } else if constexpr (NF == 1) {
          ds_u8<128 * h>(o.ws[h], ws_addr + so);
        } else {
          ds_b32<128 * h>(o.ws[h], ws_addr + so);
        }
      });
  };
  auto ops_landed = [&](Ops& o, int t) __attribute__((always_inline)) {
    __builtin_amdgcn_sched_barrier(0);
    wait_lgkm0();
    __builtin_amdgcn_sched_barrier(0);
#pragma unroll
    for (int p = 0; p < 2; ++p) {
#pragma unroll
      for (int f = 0; f < FX; ++f) ldsop::landed(o.x[f][p]);
#pragma unroll
      for (int f = 0; f < NF; ++f) ldsop::landed(o.w[f][p]);
    }
#pragma unroll
    for (int h = 0; h < HALVES; ++h) {
      landed1(o.xs[h]);
      landed1(o.ws[h]);
      if constexpr (DUAL) landed1(o.vs[h]);
      // past the end: codes 0, scale 1
      if ((t * KG + kg) * 128 + 32 * (blk + 2 * h) >= kend) o.xs[h] = o.ws[h] = o.vs[h] = 0x7f7f7f7fu;
    }
  };
#pragma unroll
  for (int f = 0; f < NF; ++f)
#pragma unroll
    for (int t = 0; t < FX; ++t) acc[f][t] = f32x4{};
  constexpr int NM = NF * FX;
  struct Widened {
    bf16x8 x[T::WIDE ? FX : 1][4], w[4];
  } wide;
  auto mul1 = [&](const Ops& o, auto ic) __attribute__((always_inline)) {
    constexpr int m = decltype(ic)::value;
    if constexpr (T::WIDE) {
      constexpr int f = m / FX, t = m % FX;
      if constexpr (m == 0)
        unroll<0, FX>([&](auto uc) __attribute__((always_inline)) {
          constexpr int u = decltype(uc)::value;
          widen<u>(wide.x[u], o.x[u], o.xs);
        });
      if constexpr (t == 0) widen<DUAL ? f & 1 : f>(wide.w, o.w[f], DUAL && f >= 2 ? o.vs : o.ws);
#pragma unroll
      for (int g = 0; g < 4; ++g)
        acc[f][t] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(wide.w[g], wide.x[t][g], acc[f][t], 0, 0, 0);
    } else {
      constexpr int t = m / NF, f = m % NF;
      const i32x8 w = cat8(o.w[f][0], o.w[f][1]), x = cat8(o.x[t][0], o.x[t][1]);
      if constexpr (DUAL) acc[f][t] = mma<f & 1, t>(w, x, acc[f][t], f < 2 ? o.ws[0] : o.vs[0], o.xs[0]);
      else acc[f][t] = mma<f, t>(w, x, acc[f][t], o.ws[0], o.xs[0]);
    }
  };

  int stage = 0;
  auto step = [&](int t, Ops& cur, const Ops& prev) __attribute__((always_inline)) {
    plain_barrier();
    const uint32_t so = (uint32_t)(stage * T::ST);
    unroll<0, NM>([&](auto ic) __attribute__((always_inline)) {
      constexpr int m = decltype(ic)::value;
      constexpr int RS = NM > 4 ? NM * 3 / 4 : NM;  // the reads go out in the first 3/4
      unroll<(m < RS ? m * NR / RS : NR), (m + 1 < RS ? (m + 1) * NR / RS : NR)>(
          [&](auto rc) __attribute__((always_inline)) { read1(cur, so, rc); });
      mul1(prev, ic);
      __builtin_amdgcn_sched_barrier(0);
    });
    ops_landed(cur, t);
    stage = stage == NST - 1 ? 0 : stage + 1;
  };
  if (n > 0) {
    Ops x, y;
    plain_barrier();
    unroll<0, NR>([&](auto rc) __attribute__((always_inline)) { read1(x, 0, rc); });
    ops_landed(x, 0);
    stage = 1;
    int t = 1;
    for (; t + 1 < n; t += 2) {
      step(t, y, x);
      step(t + 1, x, y);
    }
    if (t < n) {
      step(t, y, x);
      x = y;  // a second copy of the last products would take registers from the loop, up to 15 of them to scratch memory
    }
    unroll<0, NM>([&](auto ic) __attribute__((always_inline)) { mul1(x, ic); });
  }
  }

  // ---- the k-groups' sums: k-group g finishes operands g TO .. g TO + TO - 1 of X
  const bool fin = multiplies && kg < T::FIN;
  f32x4 sum[T::TO][NF];
  if constexpr (KG > 1) {
    f32x4* const red = (f32x4*)smem;
    __syncthreads();  // every operand has been read
    unroll<0, FX>([&](auto tc) __attribute__((always_inline)) {
      constexpr int t = decltype(tc)::value;
      if (multiplies && kg != t / T::TO)
#pragma unroll
        for (int f = 0; f < NF; ++f) red[((wave * FX + t) * NF + f) * 64 + lane] = acc[f][t];
    });
    __syncthreads();
    unroll<0, FX>([&](auto tc) __attribute__((always_inline)) {
      constexpr int t = decltype(tc)::value;
      if (multiplies && kg == t / T::TO) {
#pragma unroll
        for (int f = 0; f < NF; ++f) {
          f32x4 s = {};
#pragma unroll
          for (int g = 0; g < KG; ++g)
            s += g == t / T::TO ? acc[f][t] : red[(((sp * KG + g) * FX + t) * NF + f) * 64 + lane];
          sum[t % T::TO][f] = s;
        }
      }
    });
  } else {
#pragma unroll
    for (int t = 0; t < FX; ++t)
#pragma unroll
      for (int f = 0; f < NF; ++f) sum[t][f] = acc[f][t];
  }

  // ---- split K: partial tiles go through memory by write-through stores and loads that miss every cache
  if (ns > 1) {
    __shared__ unsigned last;
    const int at = (((sp * T::FIN + kg) * T::TO * NF) * 64 + lane) * 16;
    if (fin) {
      float* const mine = part + ((int64_t)split * tiles + tile) * (T::BM * T::BN);
#pragma unroll
      for (int v = 0; v < NF * T::TO; ++v) st_cp<CP_SC01>(mine, at + v * 1024, __builtin_bit_cast(u32x4, sum[v / NF][v % NF]));
    }
    __builtin_amdgcn_s_waitcnt(0x3f70);  // vmcnt(0): the tile has been written
    __syncthreads();
    if (tid == 0) last = atomicAdd(&arrivals[tile], 1u) == (unsigned)(ns - 1);
    __syncthreads();
    if (!last) return;
    if (fin) {
      f32x4 all[T::TO][NF];
#pragma unroll
      for (int v = 0; v < NF * T::TO; ++v) all[v / NF][v % NF] = f32x4{};
      for (int s0 = 0; s0 < ns; s0 += 2) {  // two splits' tiles requested together
        f32x4 p[2][NF * T::TO];
#pragma unroll
        for (int u = 0; u < 2; ++u) {
          const float* const src = part + ((int64_t)min(s0 + u, ns - 1) * tiles + tile) * (T::BM * T::BN);
#pragma unroll
          for (int v = 0; v < NF * T::TO; ++v) p[u][v] = __builtin_bit_cast(f32x4, ld_cp<CP_SC01>(src, at + v * 1024));
        }
#pragma unroll
        for (int u = 0; u < 2; ++u)
          if (s0 + u < ns)
#pragma unroll
            for (int v = 0; v < NF * T::TO; ++v) all[v / NF][v % NF] += p[u][v];
      }
#pragma unroll
      for (int v = 0; v < NF * T::TO; ++v) sum[v / NF][v % NF] = all[v / NF][v % NF];
    }
    if (tid == 0) atomicExch(&arrivals[tile], 0u);
  }
  if (!fin) return;

  // ---- the lane's rows are m0 + 16 FX wm + FX i + t; its columns 16 q + 4 e + f (gated: 8 q + 2 e + f) of the wave's
  unroll<0, T::TO>([&](auto oc) __attribute__((always_inline)) {
    constexpr int o = decltype(oc)::value;
    const int row = m0 + 16 * FX * wm + FX * i + kg * T::TO + o;
    if constexpr (DUAL) {
      const int col = n0 + 32 * wn;
      float v[8];
      uint32_t m = 0;
#pragma unroll
      for (int e = 0; e < 4; ++e)
#pragma unroll
        for (int f = 0; f < 2; ++f) {
          v[2 * e + f] = gated(sum[o][f][e], sum[o][2 + f][e]);
          m = max(m, mx8::abs_bits(v[2 * e + f]));
        }
      m = xhalf_max_bits(xrow_max_bits(m));
      if (row < M && col < N) {
        const uint32_t byte = mx8::scale_byte(m);
        const float inv = mx8::inverse(byte);
        *(u32x2*)((uint8_t*)a.c + row * a.ld + col + 8 * q) =
            u32x2{mx8::codes4(v[0], v[1], v[2], v[3], inv, byte < 255), mx8::codes4(v[4], v[5], v[6], v[7], inv, byte < 255)};
        if (q == 0) a.c_scales[mx8::scale_at(row, col / BLOCK, (int)((a.ld + 127) / 128))] = (uint8_t)byte;
      }
    } else {
      const int col = n0 + 16 * NF * wn + 4 * NF * q;
      if (row < M) {
        float v[4 * NF];
#pragma unroll
        for (int e = 0; e < 4; ++e)
#pragma unroll
          for (int f = 0; f < NF; ++f) v[NF * e + f] = sum[o][f][e];
        store_cols<T::OUT>((uint16_t*)a.c + row * a.ld + col, v, (int64_t)N - col);
      }
    }
  });
}

// ---- choice of tile and split on the host
enum { T16 = 0, T32, T16W, T32W, T64, T128, T256, T16N, T32N, T32H, T_COUNT };  // the last three: not gated
struct Shape {
  int bm, bn, kg, threads;
};
constexpr Shape SHAPES[T_COUNT] = {{16, 64, 4, 512},  {32, 64, 4, 512},   {16, 128, 2, 512}, {32, 128, 2, 512},
                                   {64, 128, 2, 768}, {128, 128, 1, 512}, {256, 256, 1, 256}, {16, 16, 4, 512},
                                   {32, 16, 4, 512},  {32, 32, 4, 512}};
struct Plan {
  int tile, ns;
  double us;
};
// Columns of the result that a tile computes.
constexpr int cols_of(int t, bool dual) { return dual ? SHAPES[t].bn / 2 : SHAPES[t].bn; }
inline int64_t tiles_of(int t, bool dual, int64_t M, int64_t N) {
  return ((M + SHAPES[t].bm - 1) / SHAPES[t].bm) * ((N + cols_of(t, dual) - 1) / cols_of(t, dual));
}

// Whether a call multiplies widened operands: where sums of fp32 are asked for, and gated products of few rows, which wait for memory
// (16 x 4096 x 14336 25.2 instead of 24.7 us, 32 x 14336 x 4096 26.8 instead of 27.8, 32 x 4096 x 4096 9.7 instead of 9.0). It is the
// call's rows that count, so that its parts (Cut, below) are summed alike.
constexpr bool is_wide(bool dual, bool fp32_sums, int64_t M) { return fp32_sums || (dual && M <= 32); }

// The cheapest (tile, split) by a model of the time in us: a launch, the operands from memory, the rounds of 256 workgroups
// times their k steps (dearer the more CUs share L2) with a ramp for each after the first, and for a split the exchange. The coefficients are a
// fit to the times of all tiles and splits at 459 products of M 1-4096, N 100-22016, K 512-14336; by it, 1,231 other products of
// M 1-2048, N 32-20000, K 128-16352 take 0.7% longer than with the best of them on average, 36% at worst (without narrow tiles 17%
// longer). max_ns 1: no split.
inline double price(bool dual, bool wide, int t, int ns, int64_t M, int64_t N, int64_t K) {
  struct Cost {
    double a, b0, b1, r;  // launch; per k step alone; more per k step with every CU at work; a further round
  };
  // of 543 gated products of M 1-2600, which take 0.4% longer than with the best on average, 15% at worst; by it 1,082 products
  // that are not gated take 0.4% longer, 19% at worst
  static constexpr Cost WIDE_COST[T256] = {{3.810, 0.110, 0.011, 2.90}, {4.248, 0.131, 0.007, 3.45}, {3.813, 0.192, 0.019, 2.99},
                                           {4.182, 0.241, 0.023, 3.25}, {5.034, 0.391, 0.029, 4.13}, {5.583, 0.762, 0.007, 4.51}};
  static constexpr Cost COST[T_COUNT] = {{3.685, 0.082, 0.023, 2.64}, {3.984, 0.096, 0.024, 3.09}, {3.510, 0.152, 0.036, 2.65},
                                         {3.852, 0.166, 0.043, 3.03}, {4.715, 0.187, 0.096, 3.50}, {4.823, 0.252, 0.170, 3.86},
                                         {8.409, 0.832, 0.449, 8.24}, {3.049, 0.043, 0.000, 1.59}, {3.308, 0.052, 0.000, 1.93},
                                         {3.434, 0.066, 0.000, 2.47}};
  const Cost& c = wide && t < T256 ? WIDE_COST[t] : COST[t];  // 256 x 256 has no such form
  const Shape s = SHAPES[t];
  const int64_t wg = tiles_of(t, dual, M, N) * ns, kt = (K + 127) / 128;
  const int64_t steps = ((kt + ns - 1) / ns + s.kg - 1) / s.kg * s.kg;
  const double rounds = (double)((wg + 255) / 256);
  double us = c.a + (wide ? 0.103e-6 : 0.078e-6) * (double)((dual ? 2 * N : N) + M) * (double)K + c.r * (rounds - 1) +
              rounds * (double)steps * (c.b0 + c.b1 * (double)wg / rounds / 256.0);
  if (ns > 1) us += 0.78 + 0.36 * ns + 1.29 * s.bm * s.bn / 4096.0 * std::min(1.0, (double)wg / 256.0);
  return us;
}
inline Plan choose(bool dual, bool wide, int64_t M, int64_t N, int64_t K, int max_ns) {
  const int64_t kt = (K + 127) / 128;
  Plan best{T256, 1, 1e300};
  for (int t = 0; t < (wide ? T256 : dual ? T16N : T_COUNT); ++t) {
    const Shape s = SHAPES[t];
    const int64_t tiles = tiles_of(t, dual, M, N);
    for (int ns = 1; ns <= (t == T256 ? 1 : max_ns); ++ns) {
      const int64_t wg = tiles * ns;
      if (wg * s.threads > UINT32_MAX) break;  // a launch counts its threads in 32 bits
      if (ns > 1 && (tiles > TLM_SPLIT_TILES || kt < 2 * ns || (size_t)wg * s.bm * s.bn * 4 > tlm_split_bytes(false)))
        break;
      const double us = price(dual, wide, t, ns, M, N, K);
      if (us < best.us) best = Plan{t, ns, us};
    }
  }
  return best;
}

// 256 x 256 tiles in whole rounds of the CUs, the rest of the rows or columns by what is cheapest for it, where the model says that
// this saves 3%: a last round of a few tiles takes as long as a full one. (4096 x 4352 x 4096
// 79 instead of 91 us, 4400 x 4096 x 4096 68 instead of 90, 2000 x 9000 x 4096 71 instead of 96.) Not of products that widen
// their operands, which 256 x 256 tiles do not.
struct Cut {
  int64_t rows, cols;  // of the first part; 0: no cut
};
inline Cut cut_of(bool dual, bool wide, int64_t M, int64_t N, int64_t K, const Plan& whole) {
  Cut best{0, 0};
  if (wide) return best;
  const int64_t tm = (M + 255) / 256, bn = cols_of(T256, dual), tn = (N + bn - 1) / bn, full = tm * tn / 256 * 256;
  if (full == 0 || full == tm * tn) return best;
  double least = 0.97 * whole.us;
  auto consider = [&](int64_t rows, int64_t cols) {
    if (rows <= 0 || cols <= 0 || rows > M || cols > N) return;
    const double us = price(dual, false, T256, 1, rows, cols, K) +
                      (rows < M ? choose(dual, false, M - rows, N, K, 16) : choose(dual, false, M, N - cols, K, 16)).us;
    if (us < least) least = us, best = Cut{rows, cols};
  };
  consider(M, full / tm * bn);
  consider(full / tn * 256, N);
  return best;
}

template <int OUT>
void run_part(const Args& a, bool wide, Plan p, hipStream_t s) {
  constexpr bool DUAL = OUT == TLM_F8E4M3;
  float* part = nullptr;
  unsigned* arrivals = nullptr;
  if (p.ns > 1 && !gt::split_workspace(false, s, false, &part, &arrivals)) p = choose(DUAL, wide, a.M, a.N, a.K, 1);
  const unsigned wg = (unsigned)(tiles_of(p.tile, DUAL, a.M, a.N) * p.ns);
  auto go = [&](auto tile) {
    using T = decltype(tile);
    static_assert(T::THREADS == 512 || T::BM == 64, "SHAPES");
    gemm_mx8_tile<T><<<wg, T::THREADS, 0, s>>>(a, p.ns, part, arrivals);
  };
  auto ring = [&](auto w) {
    constexpr bool W = decltype(w)::value;
    switch (p.tile) {
      case T16: return go(Tile<16, 64, 1, 4, 3, OUT, W>{});
      case T32: return go(Tile<32, 64, 2, 4, 3, OUT, W>{});
      case T16W: return go(Tile<16, 128, 1, 2, 3, OUT, W>{});
      case T32W: return go(Tile<32, 128, 2, 2, 3, OUT, W>{});
      case T64: return go(Tile<64, 128, 2, 2, 3, OUT, W>{});
      default: return go(Tile<128, 128, 4, 1, 4, OUT, W>{});
    }
  };
  if (wide) return ring(std::true_type{});
  if constexpr (!DUAL) {
    if (p.tile == T16N) return go(Tile<16, 16, 1, 4, 4, OUT>{});
    if (p.tile == T32N) return go(Tile<32, 16, 2, 4, 4, OUT>{});
    if (p.tile == T32H) return go(Tile<32, 32, 2, 4, 4, OUT>{});
  }
  if (p.tile == T256) return (void)(gemm_mx8_256<OUT><<<wg, P_T, 0, s>>>(a));
  ring(std::false_type{});
}

template <int OUT>
void run(const Args& a, bool fp32_sums, hipStream_t s) {
  constexpr bool DUAL = OUT == TLM_F8E4M3;
  const bool wide = is_wide(DUAL, fp32_sums, a.M);
  const Plan p = choose(DUAL, wide, a.M, a.N, a.K, 16);
  const Cut cut = cut_of(DUAL, wide, a.M, a.N, a.K, p);
  if (cut.rows == 0) {
    run_part<OUT>(a, wide, p, s);
    return;
  }
  Args first = a, rest = a;
  first.M = cut.rows, first.N = cut.cols;
  auto skip = [&](Mat& m, int64_t rows) {
    m.codes += rows * a.K;
    m.scales += rows / 64 * a.kt * 256;
  };
  const int64_t out_kt = (a.ld + 127) / 128;
  if (cut.rows < a.M) {  // whole groups of 64 rows
    rest.M -= cut.rows;
    skip(rest.a, cut.rows);
    rest.c = (uint8_t*)a.c + cut.rows * a.ld * (DUAL ? 1 : 2);
    if (DUAL) rest.c_scales += cut.rows / 64 * out_kt * 256;
  } else {  // whole groups of 128 columns
    rest.N -= cut.cols;
    skip(rest.b, cut.cols);
    if (DUAL) skip(rest.b2, cut.cols);
    rest.c = (uint8_t*)a.c + cut.cols * (DUAL ? 1 : 2);
    if (DUAL) rest.c_scales += cut.cols / 128 * 256;
  }
  run_part<OUT>(first, false, Plan{T256, 1, 0}, s);
  run_part<OUT>(rest, false, choose(DUAL, false, rest.M, rest.N, a.K, 16), s);
}

int check_sizes(const char* fn, int64_t M, int64_t N, int64_t K, bool dual, bool fp32_sums) {
  if (M < 0 || N < 0 || K < 0 || M > INT32_MAX - 255 || N > INT32_MAX - 255 ||
      ((M + 255) / 256) * ((N + 127) / 128) > UINT32_MAX / 512) {
    tlm_set_error("%s: bad sizes M=%lld N=%lld K=%lld (2^23 tiles of 256 x 128 at most)", fn, (long long)M, (long long)N,
                  (long long)K);
    return TLM_EINVAL;
  }
  if (fp32_sums && tiles_of(T128, dual, M, N) > UINT32_MAX / SHAPES[T128].threads) {
    tlm_set_error("%s: M=%lld N=%lld has more than 2^23 tiles of 128 x %d, the largest that sum in fp32", fn, (long long)M,
                  (long long)N, cols_of(T128, dual));
    return TLM_EINVAL;
  }
  return TLM_OK;
}

int product(const char* fn, const void* a, const void* a_scales, const void* b, const void* b_scales, void* c, int64_t M,
            int64_t N, int64_t K, int out_dtype, bool fp32_sums, void* stream) {
  if (int rc = check_sizes(fn, M, N, K, false, fp32_sums)) return rc;
  if (int rc = mx8::check(fn, "A", a, a_scales, M, K)) return rc;
  if (int rc = mx8::check(fn, "B", b, b_scales, N, K)) return rc;
  if (out_dtype != TLM_F16 && out_dtype != TLM_BF16) {
    tlm_set_error("%s: out dtype %d unsupported (F16 or BF16)", fn, out_dtype);
    return TLM_EUNSUPPORTED;
  }
  if (M == 0 || N == 0) return TLM_OK;
  if (!c) {
    tlm_set_error("%s: null pointer argument", fn);
    return TLM_EINVAL;
  }
  if (!tlm_aligned(c, 2)) {
    tlm_set_error("%s: misaligned C", fn);
    return TLM_EINVAL;
  }
  const Args g{{(const uint8_t*)a, (const uint8_t*)a_scales}, {(const uint8_t*)b, (const uint8_t*)b_scales}, {},
               c, nullptr, M, N, (int)K, (int)((K + 127) / 128), N};
  hipStream_t s = (hipStream_t)stream;
  out_dtype == TLM_BF16 ? run<TLM_BF16>(g, fp32_sums, s) : run<TLM_F16>(g, fp32_sums, s);
  TLM_LAUNCH_CHECK(fn);
  return TLM_OK;
}

int gated_product(const char* fn, const void* a, const void* a_scales, const void* gate, const void* gate_scales, const void* up,
                  const void* up_scales, void* codes, void* scales, int64_t M, int64_t N, int64_t K, bool fp32_sums,
                  void* stream) {
  if (int rc = check_sizes(fn, M, N, K, true, fp32_sums)) return rc;
  if (int rc = mx8::check(fn, "A", a, a_scales, M, K)) return rc;
  if (int rc = mx8::check(fn, "B_gate", gate, gate_scales, N, K)) return rc;
  if (int rc = mx8::check(fn, "B_up", up, up_scales, N, K)) return rc;
  if (int rc = mx8::check(fn, "the result", codes, scales, M, N)) return rc;
  if (M == 0 || N == 0) return TLM_OK;
  const Args g{{(const uint8_t*)a, (const uint8_t*)a_scales},
               {(const uint8_t*)gate, (const uint8_t*)gate_scales},
               {(const uint8_t*)up, (const uint8_t*)up_scales},
               codes, (uint8_t*)scales, M, N, (int)K, (int)((K + 127) / 128), N};
  run<TLM_F8E4M3>(g, fp32_sums, (hipStream_t)stream);
  TLM_LAUNCH_CHECK(fn);
  return TLM_OK;
}

}  // namespace

extern "C" int tlm_gemm_mx8_plan(int64_t M, int64_t N, int64_t K, int gated, int split, int* rows, int* cols, int* ns,
                                 int64_t* first_rows, int64_t* first_cols) {
  if (M <= 0 || N <= 0 || K < 0 || K > mx8::MAX_K || !rows || !cols || !ns || !first_rows || !first_cols) {
    tlm_set_error("tlm_gemm_mx8_plan: bad sizes (K up to 2^22) or null pointer");
    return TLM_EINVAL;
  }
  const bool dual = gated & 1, fp32_sums = gated & 2;
  if (int rc = check_sizes("tlm_gemm_mx8_plan", M, N, K, dual, fp32_sums)) return rc;
  const bool wide = is_wide(dual, fp32_sums, M);
  const Plan p = choose(dual, wide, M, N, K, split ? 16 : 1);
  const Cut cut = cut_of(dual, wide, M, N, K, p);
  const Shape t = SHAPES[cut.rows ? T256 : p.tile];
  *rows = t.bm, *cols = t.bn, *ns = cut.rows ? 1 : p.ns;
  *first_rows = cut.rows ? cut.rows : M, *first_cols = cut.rows ? cut.cols : N;
  return TLM_OK;
}

extern "C" int tlm_gemm_mx8(const void* a, const void* a_scales, const void* b, const void* b_scales, void* c,
                            int64_t M, int64_t N, int64_t K, int out_dtype, void* stream) {
  return product("tlm_gemm_mx8", a, a_scales, b, b_scales, c, M, N, K, out_dtype, false, stream);
}

extern "C" int tlm_gemm_mx8_ex(const void* a, const void* a_scales, const void* b, const void* b_scales, void* c,
                               int64_t M, int64_t N, int64_t K, int out_dtype, int fp32_sums, void* stream) {
  return product("tlm_gemm_mx8_ex", a, a_scales, b, b_scales, c, M, N, K, out_dtype, fp32_sums != 0, stream);
}

extern "C" int tlm_gemm_mx8_swiglu(const void* a, const void* a_scales, const void* gate, const void* gate_scales,
                                   const void* up, const void* up_scales, void* codes, void* scales, int64_t M,
                                   int64_t N, int64_t K, void* stream) {
  return gated_product("tlm_gemm_mx8_swiglu", a, a_scales, gate, gate_scales, up, up_scales, codes, scales, M, N, K, true,
                       stream);
}

extern "C" int tlm_gemm_mx8_swiglu_ex(const void* a, const void* a_scales, const void* gate, const void* gate_scales,
                                      const void* up, const void* up_scales, void* codes, void* scales, int64_t M,
                                      int64_t N, int64_t K, int fp32_sums, void* stream) {
  return gated_product("tlm_gemm_mx8_swiglu_ex", a, a_scales, gate, gate_scales, up, up_scales, codes, scales, M, N, K,
                       fp32_sums != 0, stream);
}
