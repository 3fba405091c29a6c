// The 4-bit K/V cache (include/tlmi355x.h): its argument checks and the addressing its kernels share.
#pragma once

#include "tlm_common.h"

namespace kv4 {

constexpr int BLOCK = 32;  // dims per scale
constexpr int MAX_B = INT32_MAX - (1 << 16);  // a sequence's number plus a grid's depth stays in 32 bits

// The cache as the kernels get it. Offsets into the pools are 64-bit: a pool may pass 4 GB.
struct Cache {
  uint8_t* codes;
  uint8_t* scales;
  int64_t codes_page, scales_page;  // bytes from page to page
  int64_t pages;
  const int32_t* table;
  int max_pages, page, Hkv, D;
};

// Scale byte -> the fp32 whose exponent the gfx950 conversions take (255: a NaN scale, which they pass on).
TLM_DEV float scale_of(uint32_t byte) { return __uint_as_float(byte << 23); }

// Checks what the entry points share; 0 or a status with the message set.
inline int check(const char* fn, const Cache& c, int64_t max_pages, int64_t page, int64_t Hkv, int64_t D,
                 int64_t B) {
  if (!c.codes || !c.scales || (!c.table && B != 0)) {
    tlm_set_error("%s: null pointer argument", fn);
    return TLM_EINVAL;
  }
  if (c.pages <= 0 || max_pages <= 0 || page <= 0 || Hkv <= 0 || D <= 0 || B < 0) {
    tlm_set_error("%s: bad sizes", fn);
    return TLM_EINVAL;
  }
  if (D % BLOCK != 0 || D > 256 || page % 8 != 0) {
    tlm_set_error("%s: D must be a multiple of 32 up to 256 and page a multiple of 8", fn);
    return TLM_EUNSUPPORTED;
  }
  if (B > MAX_B) {
    tlm_set_error("%s: problem too large (%d sequences)", fn, MAX_B);
    return TLM_EINVAL;
  }
  if (page > (1 << 20) || Hkv > (1 << 16) || max_pages > (INT32_MAX - 4096) / page || B > INT32_MAX / max_pages) {
    tlm_set_error("%s: problem too large (2^31 positions per table row and entries per table)", fn);
    return TLM_EINVAL;
  }
  if (Hkv * page > INT32_MAX / D) {
    tlm_set_error("%s: problem too large (2^31 bytes of codes per page)", fn);
    return TLM_EINVAL;
  }
  if (c.codes_page % 16 != 0 || c.scales_page % 8 != 0 || c.codes_page < Hkv * page * D ||
      c.scales_page < 2 * Hkv * page * (D / BLOCK)) {
    tlm_set_error("%s: bad page stride", fn);
    return TLM_EINVAL;
  }
  if (!tlm_aligned(c.codes, 16) || !tlm_aligned(c.scales, 8)) {
    tlm_set_error("%s: codes must be 16-byte and scales 8-byte aligned", fn);
    return TLM_EINVAL;
  }
  return TLM_OK;
}

// Rows [B, T, heads, D] with heads and dims dense; without any, x may be null.
inline int check_rows(const char* fn, const char* name, const void* x, bool any, int64_t batch_stride,
                      int64_t row_stride, int dtype) {
  if (any && !x) {
    tlm_set_error("%s: null pointer argument", fn);
    return TLM_EINVAL;
  }
  if (dtype != TLM_BF16 && dtype != TLM_F16) {
    tlm_set_error("%s: %s dtype %d unsupported (BF16 or F16)", fn, name, dtype);
    return TLM_EUNSUPPORTED;
  }
  if (batch_stride < 0 || row_stride < 0) {
    tlm_set_error("%s: bad sizes", fn);
    return TLM_EINVAL;
  }
  if (batch_stride % 8 != 0 || row_stride % 8 != 0 || !tlm_aligned(x, 16)) {
    tlm_set_error("%s: %s must be 16-byte aligned with strides of multiples of 8 elements", fn, name);
    return TLM_EINVAL;
  }
  return TLM_OK;
}

}  // namespace kv4
