// The 4-bit K/V cache: quantising rows as they are written, and reading them back.
//
// Format (OCP MX): 32 dims of a token and head share a power-of-two scale 2^e; an element is e2m1. With
// M = max |x| of the block, e is the least exponent with M <= 7 2^e: e2m1 reaches 6 and its widest step
// is 2, so values up to 7 are off by no more than any other. e follows from M's bits: M = 1.f 2^E gives
// e = E - 2, one more where 1.f > 1.75. M is the largest of the absolute bit patterns, which orders
// infinities behind every number and NaN behind those. v_cvt_scalef32_pk_fp4_* divides by the scale, rounds to
// nearest even, saturates and keeps the sign of zero (every 16-bit pattern compared with exact arithmetic); the reverse
// conversions are exact and pass a NaN scale on.
//
// Bound: HBM. A token and head moves 4 D bytes of 16-bit rows and 1.0625 D bytes of cache. 8 heads of 128: 63,997 tokens read
// back in 53 us (6.2 TB/s; with plain stores 70 us, one 8-dim chunk per thread with its own search and divisions 148 us);
// 13,312 tokens appended in 16.2 us (4.3 TB/s; one chunk per thread 30 us). A decode step's rows take 3.6 us,
// which is launch and three dependent loads.
#include "tlm_kv4.h"

#include <algorithm>

namespace {

using kv4::Cache;
constexpr int K4_T = 256;
constexpr int K4_GRID = 1 << 16;  // workgroups along the tokens at most; they go on from there

typedef __bf16 b2 __attribute__((ext_vector_type(2)));
typedef _Float16 h2 __attribute__((ext_vector_type(2)));
typedef float f2 __attribute__((ext_vector_type(2)));

template <int SEL>
TLM_DEV uint32_t to_fp4(uint32_t old, uint32_t w, float s, std::true_type) {
  return __builtin_amdgcn_cvt_scalef32_pk_fp4_bf16(old, __builtin_bit_cast(b2, w), s, SEL);
}
template <int SEL>
TLM_DEV uint32_t to_fp4(uint32_t old, uint32_t w, float s, std::false_type) {
  return __builtin_amdgcn_cvt_scalef32_pk_fp4_f16(old, __builtin_bit_cast(h2, w), s, SEL);
}

// Page and place of position p of sequence b; false outside the table or the pool.
TLM_DEV bool place(const Cache& c, int b, int64_t p, int64_t& pid, int& off) {
  if (p < 0 || p >= (int64_t)c.max_pages * c.page) return false;
  const int i = (int)p / c.page;
  off = (int)p - i * c.page;
  pid = c.table[(int64_t)b * c.max_pages + i];
  return pid >= 0 && pid < c.pages;
}

// A workgroup takes K4_T / (D / 8) tokens, 8 dims of a head per thread, and walks through its share of the 2 H_kv
// heads of K and V, U of them in flight: tokens next to each other make whole lines of codes, a head's D / 8 threads
// whole lines of rows.
constexpr int K4_U = 4;  // twice as many for long appends
struct Lane {
  int d8, tok;  // 8 dims, token of the workgroup
  bool live;
};
TLM_DEV Lane lane_of(int D) {
  const int per = D / 8, tok = (int)threadIdx.x / per;
  return Lane{(int)threadIdx.x - tok * per, tok, tok < K4_T / per};
}

template <bool BF16, int U>
__global__ __launch_bounds__(K4_T) void kv4_append_kernel(Cache c, const uint16_t* k, const uint16_t* v,
                                                          int64_t kb, int64_t kr, int64_t vb, int64_t vr,
                                                          const int32_t* start, const int32_t* count, int B,
                                                          int T, int heads) {
  const Lane t = lane_of(c.D);
  const int h0 = blockIdx.y * heads, h1 = min(2 * c.Hkv, h0 + heads);
  const int tokens = K4_T / (c.D / 8);
  for (int b = blockIdx.z; b < B; b += gridDim.z) {
    const int n = t.live ? min(count[b], T) : 0;
    for (int64_t j = (int64_t)blockIdx.x * tokens + t.tok; j < n; j += (int64_t)gridDim.x * tokens) {
      int64_t pid;
      int off;
      if (!place(c, b, start[b] + j, pid, off)) continue;
      const uint16_t* const ks = k + b * kb + j * kr + 8 * t.d8;
      const uint16_t* const vs = v + b * vb + j * vr + 8 * t.d8;
      uint8_t* const codes = c.codes + pid * c.codes_page + (int64_t)off * (c.D / 2) + 4 * t.d8;
      uint8_t* const scales = c.scales + pid * c.scales_page + (int64_t)(t.d8 / 4) * c.page + off;
      for (int h = h0; h < h1; h += U) {
        u32x4 x[U];
#pragma unroll
        for (int u = 0; u < U; ++u) {
          const int hu = min(h + u, h1 - 1);
          x[u] = ld_nt((const u32x4*)(hu < c.Hkv ? ks + (int64_t)hu * c.D : vs + (int64_t)(hu - c.Hkv) * c.D));
        }
#pragma unroll
        for (int u = 0; u < U; ++u) {
          if (h + u >= h1) break;
          uint32_t m = 0;
#pragma unroll
          for (int e = 0; e < 4; ++e) m = max(m, max(x[u][e] & 0x7fffu, (x[u][e] >> 16) & 0x7fffu));
          m = max(m, (uint32_t)__builtin_amdgcn_mov_dpp((int)m, 0xB1, 0xf, 0xf, false));  // lane ^ 1
          m = max(m, (uint32_t)__builtin_amdgcn_mov_dpp((int)m, 0x4E, 0xf, 0xf, false));  // lane ^ 2
          const uint32_t f = __float_as_uint(h16<BF16>::to_f32(m));
          int byte = (int)(f >> 23) - 2 + ((f & 0x7fffffu) > 0x600000u);
          byte = max(1, min(252, byte));
          uint32_t code = 0;
          if (f > 0x7f800000u) {
            byte = 255;  // NaN
          } else {
            const float s = kv4::scale_of(byte);
            const std::bool_constant<BF16> tag;
            code = to_fp4<0>(code, x[u][0], s, tag);
            code = to_fp4<1>(code, x[u][1], s, tag);
            code = to_fp4<2>(code, x[u][2], s, tag);
            code = to_fp4<3>(code, x[u][3], s, tag);
          }
          *(uint32_t*)(codes + (int64_t)(h + u) * c.page * (c.D / 2)) = code;
          if ((t.d8 & 3) == 0) scales[(int64_t)(h + u) * (c.D / kv4::BLOCK) * c.page] = (uint8_t)byte;
        }
      }
    }
  }
}

// OUT: 0 fp16, 1 bf16, 2 fp32.
template <int OUT>
TLM_DEV void put8(uint8_t* dst, uint32_t code, float s) {
  if constexpr (OUT == 1) {
    st_nt((u32x4*)dst, u32x4{__builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(code, s, 0)),
                             __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(code, s, 1)),
                             __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(code, s, 2)),
                             __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(code, s, 3))});
  } else {
    const f2 a[4] = {__builtin_amdgcn_cvt_scalef32_pk_f32_fp4(code, s, 0),
                     __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(code, s, 1),
                     __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(code, s, 2),
                     __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(code, s, 3)};
    if constexpr (OUT == 2) {
      const f32x4 x = {a[0][0], a[0][1], a[1][0], a[1][1]}, y = {a[2][0], a[2][1], a[3][0], a[3][1]};
      st_nt((u32x4*)dst, __builtin_bit_cast(u32x4, x));
      st_nt((u32x4*)dst + 1, __builtin_bit_cast(u32x4, y));
    } else {
      using H = h16<false>;
      st_nt((u32x4*)dst, u32x4{H::pack(a[0][0], a[0][1]), H::pack(a[1][0], a[1][1]), H::pack(a[2][0], a[2][1]),
                               H::pack(a[3][0], a[3][1])});
    }
  }
}

constexpr int K4_CU = 1024;  // sequence starts that are searched in LDS

template <int OUT>
__global__ __launch_bounds__(K4_T) void kv4_read_kernel(Cache c, const int32_t* start, const int32_t* cu,
                                                        uint8_t* k_out, uint8_t* v_out, int B, int64_t total,
                                                        int heads) {
  constexpr int ES = OUT == 2 ? 4 : 2;
  __shared__ int32_t cu_s[K4_CU];
  if (B < K4_CU) {
    for (int i = threadIdx.x; i <= B; i += K4_T) cu_s[i] = cu[i];
    __syncthreads();
  }
  const Lane t = lane_of(c.D);
  const int h0 = blockIdx.y * heads, h1 = min(2 * c.Hkv, h0 + heads);
  const int tokens = K4_T / (c.D / 8);
  for (int64_t r = (int64_t)blockIdx.x * tokens + t.tok; t.live && r < total; r += (int64_t)gridDim.x * tokens) {
    int lo = 0, hi = B + 1;  // cu[lo - 1] <= r < cu[hi]
    while (lo < hi) {
      const int mid = lo + ((hi - lo) >> 1);  // lo + hi passes 2^31 from 2^30 sequences on
      if ((B < K4_CU ? cu_s[mid] : cu[mid]) <= r) lo = mid + 1;
      else hi = mid;
    }
    const int b = lo - 1;
    if (b < 0 || b >= B) continue;  // a row of no sequence
    int64_t pid;
    int off;
    const bool ok = place(c, b, (start ? (int64_t)start[b] : 0) + (r - (B < K4_CU ? cu_s[b] : cu[b])), pid, off);
    if (!ok) pid = off = 0;
    const uint8_t* const codes = c.codes + pid * c.codes_page + (int64_t)off * (c.D / 2) + 4 * t.d8;
    const uint8_t* const scales = c.scales + pid * c.scales_page + (int64_t)(t.d8 / 4) * c.page + off;
    const int64_t row = (r * c.Hkv * c.D + 8 * t.d8) * ES;
    for (int h = h0; h < h1; h += K4_U) {
      uint32_t code[K4_U], byte[K4_U];
#pragma unroll
      for (int u = 0; u < K4_U; ++u) {
        const int hu = min(h + u, h1 - 1);
        code[u] = *(const uint32_t*)(codes + (int64_t)hu * c.page * (c.D / 2));
        byte[u] = scales[(int64_t)hu * (c.D / kv4::BLOCK) * c.page];
        if (!ok) code[u] = 0, byte[u] = 127;
      }
#pragma unroll
      for (int u = 0; u < K4_U; ++u) {
        const int hu = h + u;
        if (hu >= h1) break;
        put8<OUT>((hu < c.Hkv ? k_out + row + (int64_t)hu * c.D * ES : v_out + row + (int64_t)(hu - c.Hkv) * c.D * ES),
                  code[u], kv4::scale_of(byte[u]));
      }
    }
  }
}

// Heads (of 2 H_kv) per workgroup: all of them, or fewer where `wgs` workgroups would not fill the CUs.
inline int heads_per_wg(int64_t wgs, int64_t Hkv, int U) {
  int64_t heads = 2 * Hkv;
  while (heads > U && wgs * ((2 * Hkv + heads - 1) / heads) < 16384) heads = (heads + 1) / 2;
  return (int)heads;
}

}  // namespace

extern "C" int tlm_kv4_append(const void* k, const void* v, int64_t k_batch_stride, int64_t k_row_stride,
                              int64_t v_batch_stride, int64_t v_row_stride, int x_dtype,
                              const int32_t* start, const int32_t* count, const int32_t* block_table,
                              int64_t max_pages, int64_t page, void* codes, int64_t codes_page_stride,
                              void* scales, int64_t scales_page_stride, int64_t pages, int64_t B, int64_t T,
                              int64_t H_kv, int64_t D, void* stream) {
  Cache c{(uint8_t*)codes, (uint8_t*)scales, codes_page_stride, scales_page_stride, pages, block_table};
  if (int rc = kv4::check("tlm_kv4_append", c, max_pages, page, H_kv, D, B)) return rc;
  const bool any = B != 0 && T != 0;
  if (int rc = kv4::check_rows("tlm_kv4_append", "k", k, any, k_batch_stride, k_row_stride, x_dtype)) return rc;
  if (int rc = kv4::check_rows("tlm_kv4_append", "v", v, any, v_batch_stride, v_row_stride, x_dtype)) return rc;
  if (B != 0 && (!start || !count)) {
    tlm_set_error("tlm_kv4_append: null pointer argument");
    return TLM_EINVAL;
  }
  if (T < 0 || T > INT32_MAX) {
    tlm_set_error("tlm_kv4_append: bad sizes");
    return TLM_EINVAL;
  }
  if (!any) return TLM_OK;
  c.max_pages = (int)max_pages, c.page = (int)page, c.Hkv = (int)H_kv, c.D = (int)D;
  const int64_t per = K4_T / (D / 8), gx = std::min<int64_t>((T + per - 1) / per, K4_GRID);
  const int64_t gz = std::min<int64_t>(B, 65535);
  // eight heads in flight where that leaves 8 workgroups per CU (40,000 tokens of 8 heads of 128: 38.6 instead of 41.4 us), else
  // four (32 tokens: 3.7 instead of 4.6 us)
  const int U = gx * gz * ((2 * H_kv + 7) / 8) >= 2048 ? 2 * K4_U : K4_U;
  const int heads = heads_per_wg(gx * gz, H_kv, U);
  const dim3 grid((unsigned)gx, (unsigned)((2 * H_kv + heads - 1) / heads), (unsigned)gz);
  auto go = [&](auto kern) {
    kern<<<grid, K4_T, 0, (hipStream_t)stream>>>(c, (const uint16_t*)k, (const uint16_t*)v, k_batch_stride,
                                                 k_row_stride, v_batch_stride, v_row_stride, start, count,
                                                 (int)B, (int)T, heads);
  };
  const bool bf = x_dtype == TLM_BF16;
  if (U > K4_U) bf ? go(kv4_append_kernel<true, 2 * K4_U>) : go(kv4_append_kernel<false, 2 * K4_U>);
  else bf ? go(kv4_append_kernel<true, K4_U>) : go(kv4_append_kernel<false, K4_U>);
  TLM_LAUNCH_CHECK("tlm_kv4_append");
  return TLM_OK;
}

extern "C" int tlm_kv4_read(const void* codes, int64_t codes_page_stride, const void* scales,
                            int64_t scales_page_stride, int64_t pages, const int32_t* block_table,
                            int64_t max_pages, int64_t page, const int32_t* start,
                            const int32_t* cu_seqlens, void* k_out, void* v_out, int64_t B, int64_t total,
                            int64_t H_kv, int64_t D, int out_dtype, void* stream) {
  Cache c{(uint8_t*)codes, (uint8_t*)scales, codes_page_stride, scales_page_stride, pages, block_table};
  if (int rc = kv4::check("tlm_kv4_read", c, max_pages, page, H_kv, D, B)) return rc;
  if (!cu_seqlens || (total != 0 && (!k_out || !v_out))) {
    tlm_set_error("tlm_kv4_read: null pointer argument");
    return TLM_EINVAL;
  }
  if (out_dtype != TLM_BF16 && out_dtype != TLM_F16 && out_dtype != TLM_F32) {
    tlm_set_error("tlm_kv4_read: out dtype %d unsupported (BF16, F16 or F32)", out_dtype);
    return TLM_EUNSUPPORTED;
  }
  if (total < 0 || total > INT32_MAX) {
    tlm_set_error("tlm_kv4_read: bad sizes (total rows up to 2^31 - 1)");
    return TLM_EINVAL;
  }
  if (!tlm_aligned(k_out, 16) || !tlm_aligned(v_out, 16)) {
    tlm_set_error("tlm_kv4_read: k_out and v_out must be 16-byte aligned");
    return TLM_EINVAL;
  }
  if (B == 0 || total == 0) return TLM_OK;
  c.max_pages = (int)max_pages, c.page = (int)page, c.Hkv = (int)H_kv, c.D = (int)D;
  const int64_t per = K4_T / (D / 8), gx = std::min<int64_t>((total + per - 1) / per, K4_GRID);
  const int heads = heads_per_wg(gx, H_kv, K4_U);
  const dim3 grid((unsigned)gx, (unsigned)((2 * H_kv + heads - 1) / heads));
  auto go = [&](auto kern) {
    kern<<<grid, K4_T, 0, (hipStream_t)stream>>>(c, start, cu_seqlens, (uint8_t*)k_out, (uint8_t*)v_out,
                                                 (int)B, total, heads);
  };
  if (out_dtype == TLM_BF16) go(kv4_read_kernel<1>);
  else if (out_dtype == TLM_F16) go(kv4_read_kernel<0>);
  else go(kv4_read_kernel<2>);
  TLM_LAUNCH_CHECK("tlm_kv4_read");
  return TLM_OK;
}
