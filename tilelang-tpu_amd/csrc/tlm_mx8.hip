// Rows become 8-bit operands: the plain quantiser, and the residual's addition with RMS norm.
//
//   r' = round(x + r),  y = r' w / sqrt(mean(r'^2) + eps);  of 32 values with M = max |v|: e the least with M <= 448 2^e,
//   codes v / 2^e rounded to e4m3.
//
// A thread holds 8 neighbouring values, so 4 lanes share a scale. add_rmsnorm keeps its row in registers between the
// sum of squares and the result: every operand is read once and every result written once.
//
// Bound: HBM, and below some hundred rows the launch. 8192 x 7168 bf16 rows with stream and 8-bit result: 413 MB in 77 us (5.4 TB/s; a
// copy moves 4.9 TB/s); 14336 x 4096 fp32 values quantised in 51 us (5.8 TB/s); 16 x 4096 normed in 3.5 us. The byte-wise
// writes of scales cost 4% of the large norm; four rows per workgroup, which write them four at a time, cost 7% more.
#include "tlm_mx8.h"

#include <algorithm>

namespace {

using mx8::BLOCK;

// IN: 0 fp16, 1 bf16, 2 fp32. Eight values at p.
template <int IN>
TLM_DEV void load8(const void* p, int64_t i, float (&v)[8]) {
  if constexpr (IN == 2) {
    const f32x4 a = *(const f32x4*)((const float*)p + i), b = *(const f32x4*)((const float*)p + i + 4);
#pragma unroll
    for (int j = 0; j < 4; ++j) v[j] = a[j], v[4 + j] = b[j];
  } else {
    using H = h16<IN == 1>;
    const u32x4 a = *(const u32x4*)((const uint16_t*)p + i);
#pragma unroll
    for (int j = 0; j < 4; ++j) v[2 * j] = H::lo(a[j]), v[2 * j + 1] = H::hi(a[j]);
  }
}
template <int OUT, bool NT = false>
TLM_DEV void store8(void* p, int64_t i, const float (&v)[8]) {
  auto put = [](void* at, u32x4 x) {
    if constexpr (NT) st_nt((u32x4*)at, x);
    else *(u32x4*)at = x;
  };
  if constexpr (OUT == 2) {
    put((float*)p + i, __builtin_bit_cast(u32x4, f32x4{v[0], v[1], v[2], v[3]}));
    put((float*)p + i + 4, __builtin_bit_cast(u32x4, f32x4{v[4], v[5], v[6], v[7]}));
  } else {
    using H = h16<OUT == 1>;
    put((uint16_t*)p + i, u32x4{H::pack(v[0], v[1]), H::pack(v[2], v[3]), H::pack(v[4], v[5]), H::pack(v[6], v[7])});
  }
}

// Codes and scale of the lane's 8 values, columns c .. c + 7 of a row; the 4 lanes of a block call it together.
TLM_DEV void put_mx8(const float (&v)[8], uint8_t* codes, uint8_t* scales, int64_t row, int c, int cols, int kt) {
  uint32_t m = 0;
#pragma unroll
  for (int j = 0; j < 8; ++j) m = max(m, mx8::abs_bits(v[j]));
  const uint32_t byte = mx8::scale_byte(mx8::quad_max(m));
  const float inv = mx8::inverse(byte);
  *(u32x2*)(codes + row * cols + c) = u32x2{mx8::codes4(v[0], v[1], v[2], v[3], inv, byte < 255),
                                            mx8::codes4(v[4], v[5], v[6], v[7], inv, byte < 255)};
  if ((c & (BLOCK - 1)) == 0) scales[mx8::scale_at(row, c / BLOCK, kt)] = (uint8_t)byte;
}

constexpr int Q_T = 256;

// Q_T / TX rows by TX pieces of 8 columns per workgroup.
template <int IN, int TX>
__global__ __launch_bounds__(Q_T) void mx8_quant_kernel(const void* x, int64_t stride, uint8_t* codes, uint8_t* scales,
                                                        int64_t rows, int cols, int kt) {
  constexpr int TY = Q_T / TX;
  const int tx = threadIdx.x % TX, ty = threadIdx.x / TX;
  for (int64_t row = (int64_t)blockIdx.y * TY + ty; row < rows; row += (int64_t)gridDim.y * TY)
    for (int c8 = blockIdx.x * TX + tx; c8 < cols / 8; c8 += gridDim.x * TX) {
      float v[8];
      load8<IN>(x, row * stride + 8 * c8, v);
      put_mx8(v, codes, scales, row, 8 * c8, cols, kt);
    }
}

struct Norm {
  const void *x, *residual, *w;
  void *residual_out, *y;
  uint8_t *codes, *scales;
  int64_t rows;
  int cols, kt;
  float inv_cols, eps;
};

constexpr int N_GRID = 1 << 20;  // rows along x: a launch counts its threads along a side in 32 bits

// A workgroup of T threads per row, V pieces of 8 columns per thread in registers.
template <bool BF16, bool R32, int T, int V>
__global__ __launch_bounds__(T) void add_rmsnorm_kernel(Norm a) {
  __shared__ float part[T / 64];
  constexpr int X = BF16, R = R32 ? 2 : X;
  const int64_t row = (int64_t)blockIdx.y * N_GRID + blockIdx.x, at = row * a.cols;
  if (row >= a.rows) return;
  float h[V][8];
  u32x4 w[V];  // asked for with the row, not after its sum
#pragma unroll
  for (int i = 0; i < V; ++i) {
    const int c = 8 * (i * T + (int)threadIdx.x);
#pragma unroll
    for (int j = 0; j < 8; ++j) h[i][j] = 0.f;
    if (c >= a.cols) continue;
    load8<X>(a.x, at + c, h[i]);
    if (a.w) w[i] = *(const u32x4*)((const uint16_t*)a.w + c);
    if (a.residual) {
      float r[8];
      load8<R>(a.residual, at + c, r);
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        h[i][j] += r[j];
        // the norm is that of the stream as later layers read it
        if constexpr (!R32) h[i][j] = h16<BF16>::to_f32(h16<BF16>::from_f32(h[i][j]));
      }
      store8<R, true>(a.residual_out, at + c, h[i]);
    }
  }
  auto squares = [&]() __attribute__((always_inline)) {  // the row's sum of them, the same bits in all its threads
    float ss = 0.f;
#pragma unroll
    for (int i = 0; i < V; ++i)
#pragma unroll
      for (int j = 0; j < 8; ++j) ss = fmaf(h[i][j], h[i][j], ss);
    ss = wave_sum(ss);
    if constexpr (T > 64) {
      if ((threadIdx.x & 63) == 0) part[threadIdx.x >> 6] = ss;
      __syncthreads();
      ss = 0.f;
#pragma unroll
      for (int i = 0; i < T / 64; ++i) ss += part[i];
    }
    return ss;
  };
  float m = squares() * a.inv_cols + a.eps;
  // Rows whose mean square is no normal number of fp32 are scaled by a power of two, eps with them: up from below 2^-126, all of which
  // the root would take for 0, or down from 2^128 on, where what falls below 2^-118 of the root loses bits.
  if (m < 0x1p-126f || m == INFINITY) {
    const float f = m < 1.f ? 0x1p96f : 0x1p-72f;
#pragma unroll
    for (int i = 0; i < V; ++i)
#pragma unroll
      for (int j = 0; j < 8; ++j) h[i][j] *= f;
    __syncthreads();  // `part` has been read
    m = squares() * a.inv_cols + a.eps * f * f;
  }
  // one Newton step makes r exact to its last place; of 16-bit streams h w is exact, so that the result is rounded once
  const float r0 = __frsqrt_rn(m);
  const float r = m < INFINITY && r0 < INFINITY ? fmaf(0.5f * r0, fmaf(-m * r0, r0, 1.f), r0) : r0;
#pragma unroll
  for (int i = 0; i < V; ++i) {
    const int c = 8 * (i * T + (int)threadIdx.x);
    if (c >= a.cols) continue;
    using H = h16<BF16>;
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      h[i][2 * j] = (a.w ? h[i][2 * j] * H::lo(w[i][j]) : h[i][2 * j]) * r;
      h[i][2 * j + 1] = (a.w ? h[i][2 * j + 1] * H::hi(w[i][j]) : h[i][2 * j + 1]) * r;
    }
    if (a.y) store8<X>(a.y, at + c, h[i]);
    if (a.codes) put_mx8(h[i], a.codes, a.scales, row, c, a.cols, a.kt);
  }
}

template <bool BF16, bool R32>
void norm_go(const Norm& a, hipStream_t s) {
  auto go = [&](auto t, auto v) {
    constexpr int T = decltype(t)::value, V = decltype(v)::value;
    const dim3 grid((unsigned)std::min<int64_t>(a.rows, N_GRID), (unsigned)((a.rows + N_GRID - 1) / N_GRID));
    add_rmsnorm_kernel<BF16, R32, T, V><<<grid, T, 0, s>>>(a);
  };
  using std::integral_constant;
  const int per = a.cols / 8;
  if (per <= 64) go(integral_constant<int, 64>{}, integral_constant<int, 1>{});
  else if (per <= 128) go(integral_constant<int, 128>{}, integral_constant<int, 1>{});
  else if (per <= 256) go(integral_constant<int, 256>{}, integral_constant<int, 1>{});
  else if (per <= 512) go(integral_constant<int, 512>{}, integral_constant<int, 1>{});
  // few rows: more threads on each (64 x 7168 4.6 instead of 5.1 us; 1000 x 8192 13.8 instead of 13.3)
  else if (per <= 1024 && a.rows < 512) go(integral_constant<int, 1024>{}, integral_constant<int, 1>{});
  else if (per <= 2048 && a.rows < 512) go(integral_constant<int, 1024>{}, integral_constant<int, 2>{});
  else if (per <= 1024) go(integral_constant<int, 512>{}, integral_constant<int, 2>{});
  else if (per <= 2048) go(integral_constant<int, 512>{}, integral_constant<int, 4>{});
  else go(integral_constant<int, 512>{}, integral_constant<int, 8>{});
}

constexpr int MAX_COLS = 512 * 8 * 8;

}  // namespace

extern "C" int tlm_mx8_quant(const void* x, int64_t x_stride, int x_dtype, void* codes, void* scales, int64_t rows,
                             int64_t cols, void* stream) {
  if (int rc = mx8::check("tlm_mx8_quant", "x", codes, scales, rows, cols)) return rc;
  if (x_dtype != TLM_F16 && x_dtype != TLM_BF16 && x_dtype != TLM_F32) {
    tlm_set_error("tlm_mx8_quant: dtype %d unsupported (F16, BF16 or F32)", x_dtype);
    return TLM_EUNSUPPORTED;
  }
  if (rows == 0 || cols == 0) return TLM_OK;
  if (!x) {
    tlm_set_error("tlm_mx8_quant: null pointer argument");
    return TLM_EINVAL;
  }
  if (x_stride < 0 || x_stride % 8 != 0 || !tlm_aligned(x, 16)) {
    tlm_set_error("tlm_mx8_quant: x must be 16-byte aligned with a row stride of a multiple of 8 elements");
    return TLM_EINVAL;
  }
  auto go = [&](auto kern, int tx) {
    const dim3 grid((unsigned)((cols / 8 + tx - 1) / tx), (unsigned)std::min<int64_t>((rows * tx + Q_T - 1) / Q_T, 65535));
    kern<<<grid, Q_T, 0, (hipStream_t)stream>>>(x, x_stride, (uint8_t*)codes, (uint8_t*)scales, rows, (int)cols,
                                                (int)((cols + 127) / 128));
  };
  // narrow rows share a workgroup
  auto by_width = [&](auto in) {
    constexpr int IN = decltype(in)::value;
    if (cols <= 512) go(mx8_quant_kernel<IN, 64>, 64);
    else if (cols <= 1024) go(mx8_quant_kernel<IN, 128>, 128);
    else go(mx8_quant_kernel<IN, 256>, 256);
  };
  if (x_dtype == TLM_F16) by_width(std::integral_constant<int, 0>{});
  else if (x_dtype == TLM_BF16) by_width(std::integral_constant<int, 1>{});
  else by_width(std::integral_constant<int, 2>{});
  TLM_LAUNCH_CHECK("tlm_mx8_quant");
  return TLM_OK;
}

extern "C" int tlm_add_rmsnorm(const void* x, const void* residual, const void* w, void* residual_out, void* y,
                               void* codes, void* scales, int64_t rows, int64_t cols, float eps, int x_dtype,
                               int residual_dtype, void* stream) {
  if (codes || scales) {
    if (int rc = mx8::check("tlm_add_rmsnorm", "the result", codes, scales, rows, cols)) return rc;
  }
  if (x_dtype != TLM_F16 && x_dtype != TLM_BF16) {
    tlm_set_error("tlm_add_rmsnorm: x dtype %d unsupported (F16 or BF16)", x_dtype);
    return TLM_EUNSUPPORTED;
  }
  if (residual && residual_dtype != x_dtype && residual_dtype != TLM_F32) {
    tlm_set_error("tlm_add_rmsnorm: the residual must have x's dtype or be F32");
    return TLM_EUNSUPPORTED;
  }
  if (rows < 0 || cols <= 0 || rows > INT32_MAX) {
    tlm_set_error("tlm_add_rmsnorm: bad sizes");
    return TLM_EINVAL;
  }
  if (cols % 8 != 0 || cols > MAX_COLS) {
    tlm_set_error("tlm_add_rmsnorm: columns must be a multiple of 8 up to %d", MAX_COLS);
    return TLM_EUNSUPPORTED;
  }
  if (!(eps >= 0.f)) {
    tlm_set_error("tlm_add_rmsnorm: eps must be >= 0");
    return TLM_EINVAL;
  }
  if (rows == 0) return TLM_OK;
  if (!x || (!codes != !scales) || (!residual != !residual_out) || (!y && !codes)) {
    tlm_set_error("tlm_add_rmsnorm: null pointer argument");
    return TLM_EINVAL;
  }
  for (const void* p : {x, residual, w, (const void*)residual_out, (const void*)y})
    if (!tlm_aligned(p, 16)) {
      tlm_set_error("tlm_add_rmsnorm: pointers must be 16-byte aligned");
      return TLM_EINVAL;
    }
  const Norm a{x, residual, w, residual_out, y, (uint8_t*)codes, (uint8_t*)scales, rows, (int)cols,
               (int)((cols + 127) / 128), 1.0f / (float)cols, eps};
  hipStream_t s = (hipStream_t)stream;
  const bool bf = x_dtype == TLM_BF16, r32 = residual && residual_dtype == TLM_F32;
  if (bf) r32 ? norm_go<true, true>(a, s) : norm_go<true, false>(a, s);
  else r32 ? norm_go<false, true>(a, s) : norm_go<false, false>(a, s);
  TLM_LAUNCH_CHECK("tlm_add_rmsnorm");
  return TLM_OK;
}
