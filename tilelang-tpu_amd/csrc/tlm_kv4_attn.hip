// Grouped-query attention over the 4-bit K/V cache (tlm_kv4_attn).
//
// One wave per query row and head: 64 keys at a time, a lane per key for the scores, a running maximum and
// sum, and lanes over the dims for the weighted values.
#include "tlm_kv4.h"

namespace {

using kv4::Cache;
typedef float f2 __attribute__((ext_vector_type(2)));

struct Args {
  Cache c;
  const uint16_t* q;
  int64_t qb, qr;
  const int32_t* seqlens;
  const int32_t* count;
  uint16_t* o;
  float* lse;
  int B, T, H, causal;
  float scale2;  // sm_scale log2(e)
};

TLM_DEV float value(const Cache& c, int64_t pid, int w, int h, int off, int d) {
  const int64_t at = (int64_t)w * c.Hkv + h;
  const uint32_t code = c.codes[pid * c.codes_page + (at * c.page + off) * (c.D / 2) + d / 2];
  const uint32_t byte = c.scales[pid * c.scales_page + (at * (c.D / kv4::BLOCK) + d / kv4::BLOCK) * c.page + off];
  const f2 x = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(code, kv4::scale_of(byte), 0);
  return x[d & 1];
}

template <bool BF16>
__global__ __launch_bounds__(64) void kv4_attn_rows(Args a) {
  using H16 = h16<BF16>;
  __shared__ float qs[256], p[64];
  __shared__ int64_t where[64];
  const Cache& c = a.c;
  const int lane = threadIdx.x;
  const int h = blockIdx.x % a.H;
  const int64_t bj = blockIdx.x / a.H;
  const int b = (int)(bj / a.T), j = (int)(bj - (int64_t)b * a.T);
  const int n = a.count ? max(0, min(a.count[b], a.T)) : a.T;
  if (j >= n) return;
  const int L = max(0, min(a.seqlens[b], c.max_pages * c.page));
  const int keys = a.causal ? max(0, L - n + j + 1) : L;
  const int hk = h / (a.H / c.Hkv);
  const uint16_t* q = a.q + b * a.qb + j * a.qr + (int64_t)h * c.D;
  for (int d = lane; d < c.D; d += 64) qs[d] = H16::to_f32(q[d]);
  __syncthreads();
  float m = -INFINITY, l = 0.f, acc[4] = {0.f, 0.f, 0.f, 0.f};
  for (int t0 = 0; t0 < keys; t0 += 64) {
    const int t = t0 + lane;
    float s = -INFINITY;
    int64_t pid = -1;
    int off = 0;
    if (t < keys) {
      off = t % c.page;
      pid = c.table[(int64_t)b * c.max_pages + t / c.page];
      if (pid >= c.pages) pid = -1;
      s = 0.f;
      if (pid >= 0)
        for (int d = 0; d < c.D; ++d) s += qs[d] * value(c, pid, 0, hk, off, d);
      s *= a.scale2;
    }
    const bool bad = __any(s != s);
    const float top = bad ? NAN : fmaxf(m, wave_max(s));
    const float ref = top == -INFINITY ? 0.f : top;
    const float f = fast_exp2(m - ref), e = fast_exp2(s - ref);
    l = l * f + wave_sum(e);
    m = top;
    p[lane] = e;
    where[lane] = pid < 0 ? -1 : pid * c.page + off;
    __syncthreads();
    for (int i = 0; i < 4 && 64 * i + lane < c.D; ++i) {
      float x = acc[i] * f;
      for (int u = 0; u < min(64, keys - t0); ++u)
        if (where[u] >= 0) x += p[u] * value(c, where[u] / c.page, 1, hk, (int)(where[u] % c.page), 64 * i + lane);
      acc[i] = x;
    }
    __syncthreads();
  }
  const int64_t row = bj * a.H + h;
  const float inv = l == 0.f ? 0.f : 1.f / l;
  for (int i = 0; i < 4 && 64 * i + lane < c.D; ++i)
    a.o[row * c.D + 64 * i + lane] = (uint16_t)H16::from_f32(acc[i] * inv);
  if (a.lse && lane == 0) a.lse[row] = l == 0.f ? -INFINITY : m + __log2f(l);
}

}  // namespace

extern "C" size_t tlm_kv4_attn_workspace_bytes(int64_t B, int64_t T, int64_t H, int64_t H_kv, int64_t D) {
  return 0;
}

extern "C" int tlm_kv4_attn(const void* q, int64_t q_batch_stride, int64_t q_row_stride, const void* codes,
                            int64_t codes_page_stride, const void* scales, int64_t scales_page_stride,
                            int64_t pages, const int32_t* block_table, int64_t max_pages, int64_t page,
                            const int32_t* seqlens, const int32_t* count, void* o, float* lse, void* ws,
                            size_t ws_bytes, int64_t B, int64_t T, int64_t H, int64_t H_kv, int64_t D,
                            int causal, float sm_scale, int dtype, void* stream) {
  Cache c{(uint8_t*)codes, (uint8_t*)scales, codes_page_stride, scales_page_stride, pages, block_table};
  if (int rc = kv4::check("tlm_kv4_attn", c, max_pages, page, H_kv, D, B)) return rc;
  if (int rc = kv4::check_rows("tlm_kv4_attn", "q", q, q_batch_stride, q_row_stride, dtype)) return rc;
  if (!seqlens || !o) {
    tlm_set_error("tlm_kv4_attn: null pointer argument");
    return TLM_EINVAL;
  }
  if (T < 0 || H <= 0 || H % H_kv != 0) {
    tlm_set_error("tlm_kv4_attn: bad sizes (H must be a multiple of H_kv)");
    return TLM_EINVAL;
  }
  if (!tlm_aligned(o, 16) || !tlm_aligned(lse, 4)) {
    tlm_set_error("tlm_kv4_attn: o must be 16-byte and lse 4-byte aligned");
    return TLM_EINVAL;
  }
  if (B == 0 || T == 0) return TLM_OK;
  if (H > INT32_MAX / B || T > INT32_MAX / (B * H)) {
    tlm_set_error("tlm_kv4_attn: problem too large (2^31 query rows)");
    return TLM_EINVAL;
  }
  if (ws_bytes < tlm_kv4_attn_workspace_bytes(B, T, H, H_kv, D)) {
    tlm_set_error("tlm_kv4_attn: workspace too small");
    return TLM_EWORKSPACE;
  }
  c.max_pages = (int)max_pages, c.page = (int)page, c.Hkv = (int)H_kv, c.D = (int)D;
  const Args a{c, (const uint16_t*)q, q_batch_stride, q_row_stride, seqlens, count, (uint16_t*)o, lse,
               (int)B, (int)T, (int)H, causal, sm_scale * 1.4426950408889634f};
  const unsigned grid = (unsigned)(B * T * H);
  if (dtype == TLM_BF16) kv4_attn_rows<true><<<grid, 64, 0, (hipStream_t)stream>>>(a);
  else kv4_attn_rows<false><<<grid, 64, 0, (hipStream_t)stream>>>(a);
  TLM_LAUNCH_CHECK("tlm_kv4_attn");
  return TLM_OK;
}
