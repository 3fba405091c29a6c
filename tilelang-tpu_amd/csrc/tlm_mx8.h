// 8-bit operands with power-of-two scales (OCP MX e4m3, include/tlmi355x.h): what their kernels share.
//
// Codes are row-major; the scales of 64 rows and 128 k lie together, 64 bytes per 32 k: lane (i, q) = (l % 16, l / 16)
// of a 16x16x128 matrix instruction needs the scale of k block q for one row, so 64 rows' scales of a k step are one
// 256-byte load of a wave, and the 4 bytes of a lane serve four instructions, whose row i is row 4 i + f of the 64.
#pragma once

#include "tlm_common.h"

namespace mx8 {

constexpr int BLOCK = 32;       // values per scale
constexpr int MAX_K = 1 << 22;  // values per row

// Byte offset of the scale of row r, block b. kt: k steps of 128, ceil(K / 128).
TLM_DEV int64_t scale_at(int64_t r, int b, int kt) {
  return ((r >> 6) * kt + (b >> 2)) * 256 + (b & 3) * 64 + (r & 63);
}

// Largest magnitude of a block, as the bits of its absolute value (infinities behind every number, NaN behind those),
// -> scale byte: the least e with M <= 448 2^e = 1.75 2^(e + 8), -126 at least. 255: the block holds no number.
TLM_DEV uint32_t scale_byte(uint32_t m) {
  const int e = (int)(m >> 23) - 8 + ((m & 0x7fffffu) > 0x600000u);
  return m >= 0x7f800000u ? 255u : (uint32_t)max(e, 1);
}
// 2^-e of a scale byte below 255. Products with it are exact but where they fall below 2^-126, whose codes are 0.
TLM_DEV float inverse(uint32_t byte) { return __uint_as_float((254u - byte) << 23); }

// Four codes; magnitudes are at most 448, so nothing is out of the type's range. A block without a number gets zeros:
// its scale says what it is.
TLM_DEV uint32_t codes4(float a, float b, float c, float d, float inv, bool number) {
  int p = __builtin_amdgcn_cvt_pk_fp8_f32(a * inv, b * inv, 0, false);
  p = __builtin_amdgcn_cvt_pk_fp8_f32(c * inv, d * inv, p, true);
  return number ? (uint32_t)p : 0u;
}

TLM_DEV uint32_t abs_bits(float x) { return __float_as_uint(x) & 0x7fffffffu; }

// Largest of the four lanes of a quad.
TLM_DEV uint32_t quad_max(uint32_t m) {
  m = max(m, (uint32_t)__builtin_amdgcn_mov_dpp((int)m, 0xB1, 0xf, 0xf, false));  // lane ^ 1
  return max(m, (uint32_t)__builtin_amdgcn_mov_dpp((int)m, 0x4E, 0xf, 0xf, false));  // lane ^ 2
}

// Checks codes [rows, K] and their scales; 0 or a status with the message set.
inline int check(const char* fn, const char* name, const void* codes, const void* scales, int64_t rows, int64_t K) {
  if (rows < 0 || K < 0 || rows > INT32_MAX - 255 || K > MAX_K) {
    tlm_set_error("%s: bad sizes of %s (rows below 2^31 - 255, up to 2^22 columns)", fn, name);
    return TLM_EINVAL;
  }
  if (K % BLOCK != 0) {
    tlm_set_error("%s: columns of %s must be a multiple of 32", fn, name);
    return TLM_EUNSUPPORTED;
  }
  if (rows != 0 && K != 0 && (!codes || !scales)) {
    tlm_set_error("%s: null pointer argument", fn);
    return TLM_EINVAL;
  }
  if (!tlm_aligned(codes, 16) || !tlm_aligned(scales, 4)) {
    tlm_set_error("%s: codes of %s must be 16-byte and scales 4-byte aligned", fn, name);
    return TLM_EINVAL;
  }
  return TLM_OK;
}

}  // namespace mx8
