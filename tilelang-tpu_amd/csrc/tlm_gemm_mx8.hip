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

template <int OUT>
int direct(const Args& a, hipStream_t s) {
  constexpr int NF = OUT == TLM_F8E4M3 ? 2 : 1;
  const int mt = a.M <= 16 ? 1 : a.M <= 32 ? 2 : 4;
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
