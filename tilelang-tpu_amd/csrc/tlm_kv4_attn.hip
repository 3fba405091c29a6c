// Grouped-query attention over the 4-bit K/V cache (tlm_kv4_attn): the newest tokens of each sequence attend to what is
// cached of it. No program of the reference does this.
//
// Per query row: s_t = sm_scale q k_t, o = sum_t 2^((s_t - m) log2 e) v_t / sum_t 2^((s_t - m) log2 e) in one pass over the keys,
// m a reference that follows the running maximum. A K/V head's rows are its new tokens times its query heads; a
// workgroup holds 16 or 32 of them (QT).
//
// What bounds it: one new token, the stream of codes: 64 sequences of 512 .. 8,192 tokens, 32 / 8 heads of 128 (bf16): 304 MB
// in 55 us, 5.6 TB/s; the same without the arithmetic 52 us. Few tokens, the chain launch, lengths, table, tile, exchange: 6.4 us
// for one sequence of 1,000, 2.8 for the join. Prompt chunks, instruction issue: chunks of 768 and 1,024 over 8,192 and
// 16,384 tokens 507 us (720 TFLOP/s); a 32-token tile of 32 rows issues 32 MFMAs (512 cycles), 64 conversions and 32
// permutations (420) and the softmax (340), which hide under each other little (one wave's MFMA and VALU work do not overlap
// at all).
//
//   * Partition: entry (sequence, row tile) costs its 128-token units plus KA_PIECE; the cost line of the batch is cut into
//     up to G equal ranges, one workgroup each per K/V head, found from the lengths by the workgroups themselves. A
//     range's part of an entry (a piece) is the output or, where the entry was cut, goes to the workspace, from where
//     kv4_attn_join merges it. Pieces priced at 1 unit: 5 % slower at 24 sequences of 1 .. 2,047 tokens, the same elsewhere.
//   * Its four waves take 32-token tiles in turn, each with its own reference, sums and O^T: no barrier until the piece
//     ends. Every wave has an LDS ring of 2 to 4 tiles that it fills by LDS-DMA (one instruction per 64 blocks of 32 dims, one for
//     all scales at D 128) with a per-lane order that makes every LDS read linear in the lane. Prefetch into registers, 13 loads
//     per tile: 85 us instead of 79 at that stage, and per-lane addresses where a page id is now scalar.
//   * S^T = K Q^T: a lane's 16 bytes of K are one block, so one scale; v_cvt_scalef32_pk_*_fp4 makes two operands of a byte,
//     scale included, exactly. The MFMA leaves a lane the scores of 8 tokens of one query, and just those 8 tokens' rows of V
//     are what O^T += V^T P^T wants of it: P never moves between lanes. V^T costs one permutation per pair of values.
//   * Types: bf16 queries meet K in bf16 and their weights, as fp16 numbers, V in fp16 (half a step of a weight is 2^-12 to
//     2^-11; the output's is 2^-9 to 2^-8). fp16 queries meet K in fp16, their weights V in bf16 in two terms, since one rounding
//     to fp16 would show in an fp16 output (1.4 times its error). Where a scale does not suit fp16, a V is NaN or a score far
//     out, the rest of the piece runs in bf16, weights and fp16 queries in two terms (64 sequences with a V of zeros, scale
//     byte 1, in every token: 80 us). Both forms in one loop would spill: with scratch memory in use the kernel above takes 68
//     instead of 55 us.
//   * The reference of a row moves when a score passes it by 2^KA_SLACK only, so O is rescaled a few times per row.
//   * Codes that only one row tile reads bypass the caches (74 -> 65 us); those of longer chunks are shared through the L2 of
//     the XCD that the K/V head's workgroups are on (8 heads).
//   * 64 rows per wave (one wave per SIMD): 680 instead of 555 us for the chunks. Four waves of 32 rows sharing each tile's
//     conversions through LDS, a barrier per tile: 550 instead of 528.
#include "tlm_kv4.h"

#include <algorithm>

namespace {

using kv4::Cache;
using ldsop::unroll;

constexpr int KA_W = 4;          // waves per workgroup
constexpr int KA_BN = 32;        // tokens per tile (one wave)
constexpr int KA_UNIT = KA_W * KA_BN;
constexpr int KA_PIECE = 2;      // cost of a piece beside its units, in units
constexpr int KA_LEAST = 3;      // of a range, where a CU has more than one
// Workgroups per CU, and stages of a ring in their share of the LDS.
constexpr int ka_per_cu(int D, int QT) { return QT == 1 ? (D <= 128 ? 3 : 2) : D <= 128 ? 2 : 1; }
template <int D, int QT>
constexpr int ka_stages() {
  const int n = (160 * 1024 / ka_per_cu(D, QT) - 1024) / (KA_W * (32 * D + 256 * ((D + 127) / 128)));
  return n < 4 ? n : 4;
}
// Weights are 2^(s - reference): 2^BIAS for the score that set the reference, which is kept until another passes
// that one by SLACK. At most 2^15, an fp16 number, and normal ones down to 2^-25 of the largest.
constexpr float KA_BIAS = 11.f, KA_SLACK = 4.f;
// From here on a reference is the score itself and the tile takes the slower form, which rounds products with the scale before
// it subtracts: the product inside an fma is exact, the reference was rounded, so a row's weights are off by a common factor of
// up to 2^(a step of fp32): 2^(1/4) below KA_FAR, but past fp16 from 2^25 on, and nothing or infinite farther out.
constexpr float KA_FAR = 0x1p22f;

struct alignas(16) KaCut {
  int b, rt, n;  // sequence (-1: nothing to join), row tile, new tokens
  int p0, p1;    // first and last range that hold units of it
};

struct KaArgs {
  Cache c;
  const uint16_t* q;
  int64_t qb, qr;
  const int32_t* seqlens;
  const int32_t* count;
  uint16_t* o;
  float* lse;
  KaCut* cuts;  // [G]: the entry that the cut before range r goes through, if it is the entry's first
  float* part;  // [2 G][Hkv][16 QT][D + 2]: rows, their references, their sums
  int B, T, H, group, causal, G;
  int few;            // ka_find64 will do, with 2^(few - 1) lanes per sequence
  int once;           // codes are read by one row tile only: past the caches
  uint32_t page_mul, group_mul;  // x / page = x page_mul >> page_shift, for x < 2^31; the same for group
  int page_shift, group_shift;
  float scale2;       // |sm_scale| log2(e)
  uint32_t q_sign;    // the sign of sm_scale on both halves of a word
};

// An entry of the cost line: 16 QT query rows of one sequence (rows run over its new tokens and, within one,
// over the heads of a K/V head).
struct KaEntry {
  int L, n;           // cached tokens, new ones
  int row0, rows;     // first row, rows
  int keys, keys_min; // keys that its last row sees, and its first
  int units;
};
TLM_DEV int ka_token_of(const KaArgs& a, int row) {  // row / group
  return (int)((uint64_t)(uint32_t)row * a.group_mul >> a.group_shift);
}
template <int MT>
TLM_DEV KaEntry ka_entry(const KaArgs& a, int L, int n, int rt) {
  KaEntry e;
  e.L = L, e.n = n;
  e.row0 = rt * MT;
  e.rows = min(MT, n * a.group - e.row0);
  if (a.causal) {
    e.keys = max(0, L - n + 1 + ka_token_of(a, e.row0 + e.rows - 1));
    e.keys_min = max(0, L - n + 1 + ka_token_of(a, e.row0));
  } else {
    e.keys = e.keys_min = L;
  }
  e.units = (e.keys + KA_UNIT - 1) / KA_UNIT;
  return e;
}
TLM_DEV int ka_len(const KaArgs& a, int b) { return max(0, min(a.seqlens[b], a.c.max_pages * a.c.page)); }
TLM_DEV int ka_new(const KaArgs& a, int b) { return a.count ? max(0, min(a.count[b], a.T)) : a.T; }
template <int MT>
TLM_DEV int ka_tiles(const KaArgs& a, int n) { return (n * a.group + MT - 1) / MT; }

// Ranges of the cost line: range r of g starts at floor(r total / g). With g <= 768 products of the rest are below 2^20, and
// (x + 1/2) / g is 1 / 1536 away from every integer, more than fp32 is off by (2^-21 of 768 at most).
struct KaCuts {
  int64_t quot;
  uint32_t rem, g;
  float inv;
  TLM_DEV KaCuts(int64_t total, int ranges) : g((uint32_t)ranges), inv(__builtin_amdgcn_rcpf((float)ranges)) {
    if (total >> 32) {
      quot = total / ranges;
      rem = (uint32_t)(total - quot * ranges);
    } else {
      const uint32_t q = (uint32_t)total / g;
      quot = q;
      rem = (uint32_t)total - q * g;
    }
  }
  TLM_DEV int64_t at(int r) const { return quot * r + (uint32_t)(((float)(rem * (uint32_t)r) + 0.5f) * inv); }
  TLM_DEV int range_of(int64_t x, int64_t total) const {  // the one that holds x: estimated, then exact
    int r = max(0, min((int)g - 1, (int)((float)x * (float)g / (float)total)));
    while (at(r) > x) --r;
    while (r + 1 < (int)g && at(r + 1) <= x) ++r;
    return r;
  }
};

// Ranges of a cost line: one workgroup per CU with anything, more where each gets KA_LEAST (two with a unit each on a CU take
// longer than one with both, and leave the join twice the pieces: 12 sequences of 1,000 .. 6,000, 2 heads of 256, 13.6 + 4.0 us
// instead of 15.8 + 5.0; 2 and 4 as the least 15.4 and 13.6).
template <int D, int QT>
TLM_DEV int ka_ranges(const KaArgs& a, int64_t total) {
  if (total >= KA_LEAST * a.G) return a.G;
  return min((int)total, max(max(1, a.G / ka_per_cu(D, QT)), (int)total / KA_LEAST));
}

// Position x of the cost line in units of an entry that starts at `before`: its KA_PIECE come first.
TLM_DEV int ka_unit_at(int64_t x, int64_t before, int units) {
  const int64_t u = x - before - KA_PIECE;
  return u < 0 ? 0 : u > units ? units : (int)u;
}

// The whole cost, and the entry that holds position `at` of it (at < 0: none); by a block of KA_W waves.
struct KaPoint {
  int64_t total, before;
  int b, rt, L, n;
};
template <int MT, typename F>
TLM_DEV KaPoint ka_find(const KaArgs& a, int64_t* sh, F&& want) {
  constexpr int NT = 64 * KA_W;
  const int tid = threadIdx.x;
  const int per = (a.B + NT - 1) / NT;
  const int b0 = min(a.B, tid * per), b1 = min(a.B, b0 + per);
  int64_t mine = 0;
  for (int b = b0; b < b1; ++b) {
    const int L = ka_len(a, b), n = ka_new(a, b), rts = ka_tiles<MT>(a, n);
    for (int rt = 0; rt < rts; ++rt) mine += ka_entry<MT>(a, L, n, rt).units + KA_PIECE;
  }
  int64_t x = mine;
#pragma unroll
  for (int o = 1; o < 64; o <<= 1) {
    const int64_t y = __shfl_up(x, o, 64);
    if ((tid & 63) >= o) x += y;
  }
  if ((tid & 63) == 63) sh[tid >> 6] = x;
  __syncthreads();
  KaPoint p{0, 0, 0, 0};
  int64_t pre = x - mine;
#pragma unroll
  for (int i = 0; i < KA_W; ++i) {
    const int64_t v = sh[i];
    if (i < tid >> 6) pre += v;
    p.total += v;
  }
  const int64_t at = want(p.total);
  if (at >= pre && at < pre + mine) {
    int64_t s = pre;
    int b = b0, rt = 0;
    for (; b < b1; ++b) {
      const int L = ka_len(a, b), n = ka_new(a, b), rts = ka_tiles<MT>(a, n);
      for (rt = 0; rt < rts; ++rt) {
        const int cost = ka_entry<MT>(a, L, n, rt).units + KA_PIECE;
        if (at < s + cost) break;
        s += cost;
      }
      if (rt < rts) break;
    }
    sh[KA_W] = s;
    sh[KA_W + 1] = b;
    sh[KA_W + 2] = rt;
  }
  __syncthreads();
  p.before = sh[KA_W];
  p.b = (int)sh[KA_W + 1];
  p.rt = (int)sh[KA_W + 2];
  p.L = at >= 0 ? ka_len(a, p.b) : 0;
  p.n = at >= 0 ? ka_new(a, p.b) : 0;
  return p;
}
// The same for up to 64 sequences by every wave for itself: no barrier, one trip to memory. A sequence has 2^(few - 1) lanes,
// as many as there are, each with a run of its row tiles (one prompt of 8,192 tokens has 1,024 of them).
template <int MT, typename F>
TLM_DEV KaPoint ka_find64(const KaArgs& a, F&& want) {
  const int lane = threadIdx.x & 63, sh = a.few - 1, seq = lane >> sh;
  int L = 0, n = 0, rt0 = 0, mine = 0;  // (the caller has made sure that all costs together fit)
  if (seq < a.B) {
    L = ka_len(a, seq), n = ka_new(a, seq);
    const int rts = ka_tiles<MT>(a, n), run = (rts + (1 << sh) - 1) >> sh;
    rt0 = min(rts, (lane & ((1 << sh) - 1)) * run);
    const int rt1 = min(rts, rt0 + run);
    for (int rt = rt0; rt < rt1; ++rt) mine += ka_entry<MT>(a, L, n, rt).units + KA_PIECE;
  }
  int x = mine;
#pragma unroll
  for (int o = 1; o < 64; o <<= 1) {
    const int y = __shfl_up(x, o, 64);
    if (lane >= o) x += y;
  }
  KaPoint p{};
  const int total = __builtin_amdgcn_readlane(x, 63);
  p.total = total;
  const int at = (int)want((int64_t)total);
  const uint64_t m = __ballot(at >= x - mine && at < x);
  if (m == 0) return p;
  const int from = __builtin_ctzll(m);
  p.b = from >> sh;
  p.L = __builtin_amdgcn_readlane(L, from);
  p.n = __builtin_amdgcn_readlane(n, from);
  p.rt = __builtin_amdgcn_readlane(rt0, from);
  int s = __builtin_amdgcn_readlane(x - mine, from);
  for (;; ++p.rt) {
    const int cost = ka_entry<MT>(a, p.L, p.n, p.rt).units + KA_PIECE;
    if (at < s + cost) break;
    s += cost;
  }
  p.before = s;
  return p;
}

// Dims in segments of 128, 64 and 32: W = 8, 4, 2 dims per lane of 16 and W / 2 words of K per lane.
template <int D>
struct Segs {
  static constexpr int N128 = D / 128, N = N128 + (D % 128) / 64 + (D % 64) / 32;
  static constexpr int w(int s) { return s < N128 ? 8 : (s == N128 && D % 128 >= 64) ? 4 : 2; }
  static constexpr int base(int s) {
    int b = 0;
    for (int i = 0; i < s; ++i) b += 16 * w(i);
    return b;
  }
};

__device__ const u32x4 ka_zeros[1] = {};  // codes and scales of tokens without a page

// A tile in a wave's ring of LDS, in 16-byte slots (32 dims of a token): K in the order that the lanes read it as MFMA
// operands, then V in token order of its operand, so that all reads are linear in the lane; then the scales,
// [K, V][D / 32][32 tokens].
template <int D>
struct Stage {
  static constexpr int CODES = 32 * D, NC = D / 32;           // bytes; LDS-DMA instructions of 64 slots
  static constexpr int NS = (D + 127) / 128, SCALES = 256 * NS;  // 64 words each
  static constexpr int BYTES = CODES + SCALES, PER = NC + NS;
};
// What a lane has of a tile: K of tokens jl and 16 + jl; V of tokens 4 g + (0 .. 3) and 16 + 4 g + (0 .. 3), so
// that a lane's scores are those of its V rows.
template <int D>
struct KaTile {
  uint32_t k[2][D / 32], v[8][Segs<D>::N];
  uint32_t ks[2][Segs<D>::N];
  u32x2 vs[Segs<D>::N];
};
TLM_DEV int ka_token(int g, int i) { return 16 * (i >> 2) + 4 * g + (i & 3); }  // of a lane's V row i

using ldsop::lds_u32;
template <int N>
TLM_DEV void vm_wait() {  // all but the last N vector loads and LDS-DMA instructions of this wave have landed
  static_assert(N >= 0 && N < 64, "vmcnt is 6 bits");
  __builtin_amdgcn_sched_barrier(0);
  __builtin_amdgcn_s_waitcnt(0x3f70 | (N & 15) | ((N >> 4) << 14));
  __builtin_amdgcn_sched_barrier(0);
}

// A segment's part of a tile for the lane, from its LDS addresses; waited for within the block. K with all scales first, V
// only when the scores are done (fewer registers).
template <int W, int KO, int KSO, int VSO>
TLM_DEV void ka_read_k(uint32_t (&k0)[W / 2], uint32_t (&k1)[W / 2], uint32_t& s0, uint32_t& s1, u32x2& vs, uint32_t ka,
                       uint32_t ksa, uint32_t vsa) {
  std::conditional_t<W == 8, u32x4, std::conditional_t<W == 4, u32x2, uint32_t>> a, b;
#define KA_READ_K(OP)                                                                                                 \
  asm volatile(OP " %0, %5 offset:%8\n\t" OP " %1, %5 offset:%9\n\tds_read_u8 %2, %6 offset:%10\n\t"                  \
                  "ds_read_u8 %3, %6 offset:%11\n\tds_read2_b32 %4, %7 offset0:0 offset1:4\n\ts_waitcnt lgkmcnt(0)"    \
               : "=&v"(a), "=&v"(b), "=&v"(s0), "=&v"(s1), "=&v"(vs)                                                  \
               : "v"(ka), "v"(ksa), "v"(vsa + VSO), "i"(KO), "i"(KO + 128 * W), "i"(KSO), "i"(KSO + 16)               \
               : "memory")
  if constexpr (W == 8) KA_READ_K("ds_read_b128");
  else if constexpr (W == 4) KA_READ_K("ds_read_b64");
  else KA_READ_K("ds_read_b32");
#undef KA_READ_K
  if constexpr (W == 2) {
    k0[0] = a, k1[0] = b;
  } else {
#pragma unroll
    for (int i = 0; i < W / 2; ++i) k0[i] = a[i], k1[i] = b[i];
  }
}
template <int W, int VO>
TLM_DEV void ka_read_v(uint32_t (&v)[8], uint32_t va) {
  if constexpr (W == 8) {
    u32x2 x[4];
    asm volatile(
        "ds_read2st64_b32 %0, %4 offset0:0 offset1:1\n\t"
        "ds_read2st64_b32 %1, %4 offset0:2 offset1:3\n\t"
        "ds_read2st64_b32 %2, %4 offset0:4 offset1:5\n\t"
        "ds_read2st64_b32 %3, %4 offset0:6 offset1:7\n\t"
        "s_waitcnt lgkmcnt(0)"
        : "=&v"(x[0]), "=&v"(x[1]), "=&v"(x[2]), "=&v"(x[3])
        : "v"(va + VO)
        : "memory");
#pragma unroll
    for (int i = 0; i < 8; ++i) v[i] = x[i >> 1][i & 1];
  } else {
#define KA_READ_V(OP)                                                                                                 \
  asm volatile(OP " %0, %8 offset:%9\n\t" OP " %1, %8 offset:%10\n\t" OP " %2, %8 offset:%11\n\t" OP                  \
                  " %3, %8 offset:%12\n\t" OP " %4, %8 offset:%13\n\t" OP " %5, %8 offset:%14\n\t" OP                 \
                  " %6, %8 offset:%15\n\t" OP " %7, %8 offset:%16\n\ts_waitcnt lgkmcnt(0)"                           \
               : "=&v"(v[0]), "=&v"(v[1]), "=&v"(v[2]), "=&v"(v[3]), "=&v"(v[4]), "=&v"(v[5]), "=&v"(v[6]),           \
                 "=&v"(v[7])                                                                                          \
               : "v"(va), "i"(VO), "i"(VO + 32 * W), "i"(VO + 64 * W), "i"(VO + 96 * W), "i"(VO + 128 * W),           \
                 "i"(VO + 160 * W), "i"(VO + 192 * W), "i"(VO + 224 * W)                                              \
               : "memory")
    if constexpr (W == 4) KA_READ_V("ds_read_u16");
    else KA_READ_V("ds_read_u8");
#undef KA_READ_V
  }
}

// Two codes of a word, times their scale, as 16-bit floats: exact in bf16; in fp16 for the scales that ka_not_f16 passes.
template <bool F16, int SEL>
TLM_DEV uint32_t ka_cvt(uint32_t w, float s) {
  if constexpr (F16)
    return __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_f16_fp4(w, s, SEL));
  else
    return __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(w, s, SEL));
}
template <bool F16>
TLM_DEV f32x4 ka_mma(u32x4 a, u32x4 b, f32x4 c) {
  if constexpr (F16)
    return __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(f16x8, a), __builtin_bit_cast(f16x8, b), c, 0, 0, 0);
  else
    return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8, a), __builtin_bit_cast(bf16x8, b), c, 0, 0,
                                                   0);
}
// Scale bytes 109 .. 140 (2^-18 .. 2^13): every code times them is an fp16 number, subnormal ones among them, which
// the matrix cores take. Zero where all bytes of w are such: plus 19 they are 128 .. 159, and a byte's carry comes from
// one that is out of range itself.
TLM_DEV uint32_t ka_not_f16(uint32_t w) { return ((w + 0x13131313u) ^ 0x80808080u) & 0xe0e0e0e0u; }
// Scale bytes 253 .. 255, which V takes as NaN: bit 7 of each such byte of w.
TLM_DEV uint32_t ka_nan(uint32_t w) { return ((w & 0x7f7f7f7fu) + 0x03030303u) & w & 0x80808080u; }

// x y, rounded by itself: no part of an fma.
TLM_DEV float ka_mul(float x, float y) {
#pragma clang fp contract(off)
  return x * y;
}

// Two floats -> their bf16 parts and the bf16 parts of what is left: 16 bits of each.
TLM_DEV void ka_split(float x, float y, uint32_t& hi, uint32_t& lo) {
  hi = h16<true>::pack(x, y);
  lo = h16<true>::pack(x - h16<true>::lo(hi), y - h16<true>::hi(hi));
}
TLM_DEV void ka_split_f16(u32x4 x, u32x4& hi, u32x4& lo) {  // fp16 words: exact; an infinity leaves nothing
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const float y0 = h16<false>::lo(x[i]), y1 = h16<false>::hi(x[i]);
    hi[i] = h16<true>::pack(y0, y1);
    const float z0 = h16<true>::lo(hi[i]), z1 = h16<true>::hi(hi[i]);
    lo[i] = h16<true>::pack(fabsf(z0) < INFINITY ? y0 - z0 : 0.f, fabsf(z1) < INFINITY ? y1 - z1 : 0.f);
  }
}

// A range's part of an entry, for one K/V head.
struct KaPiece {
  int b, h, t0, t1;  // tokens t0 .. t1 - 1
  KaEntry e;
  float* slot;  // where its rows go unless it is all of the entry
};
struct KaShared {
  float m[KA_W][16], l[KA_W][16];
};

// What a lane fetches with each LDS-DMA instruction of a tile, from where its part of the tile (32 / NP tokens) begins.
template <int D, int NP>
struct KaFetch {
  using S = Segs<D>;
  using St = Stage<D>;
  uint32_t off_c[St::NC], off_s[St::NS];
  int part_c[St::NC], part_s[St::NS];
  TLM_DEV KaFetch(const Cache& c, int lane) {
    constexpr int PT = KA_BN / NP, NK = D / 32;
#pragma unroll
    for (int j = 0; j < St::NC; ++j) {
      const bool is_v = 64 * j + lane >= D;
      const int p = 64 * j + lane - (is_v ? D : 0);
      int tok = 0, byte = 0;
      unroll<0, S::N>([&](auto s) {
        constexpr int W = S::w(s), B0 = S::base(s);
        const int x = p - B0;
        if (x < 0 || x >= 16 * W) return;
        if (is_v) {
          tok = ka_token(x / (W / 2) % 4, x / (2 * W));
          byte = B0 / 2 + 16 * (x % (W / 2));
        } else {
          tok = 16 * (x / (8 * W)) + x % 16;
          byte = B0 / 2 + 16 * (x / 16 % (W / 2));
        }
      });
      part_c[j] = tok / PT;
      off_c[j] = (uint32_t)((is_v ? c.Hkv * c.page * (D / 2) : 0) + tok % PT * (D / 2) + byte);
    }
#pragma unroll
    for (int j = 0; j < St::NS; ++j) {
      const int x = 64 * j + lane < D / 2 ? 64 * j + lane : 0;  // lanes past the scales fetch the first word again
      const int half = x / (8 * NK), blk = x / 8 % NK, tok = 4 * (x % 8);
      part_s[j] = tok / PT;
      off_s[j] = (uint32_t)((half * c.Hkv * NK + blk) * c.page + tok % PT);
    }
  }
};

// One piece. NP: pages that a tile may touch, 1 (page a multiple of 32), 2 (of 16) or 4.
template <int D, int QT, bool BF16, int NP>
TLM_DEV void ka_piece(const KaArgs& a, const KaPiece& pc, const KaFetch<D, NP>& fetch, uint8_t* smem, KaShared& sh) {
  using S = Segs<D>;
  using St = Stage<D>;
  constexpr int MT = 16 * QT, NK = D / 32, ND = D / 16, NST = ka_stages<D, QT>(), PT = KA_BN / NP;
  constexpr int SO = D + 4;  // floats of a row of the exchange
  static_assert(KA_W * NST * St::BYTES >= KA_W * 16 * SO * (int)sizeof(float), "the exchange lies in the rings");
  auto so = (float(*)[16][SO])smem;
  const Cache& c = a.c;
  const KaEntry& e = pc.e;
  const int tid = threadIdx.x, lane = tid & 63;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int g = lane >> 4, jl = lane & 15;
  const int b = pc.b, h = pc.h, L = e.L, n = e.n;
  const int64_t k_head = (int64_t)h * c.page * (D / 2), ks_head = (int64_t)h * c.page * NK;
  const uint32_t ring = lds_u32(smem) + wave * (NST * St::BYTES);
  const uint32_t k64 = 256 * (g >> 1) + 16 * jl + 8 * (g & 1), k32 = 16 * jl + 4 * g;

  const int tend = pc.t1;
  int t0 = pc.t0 + wave * KA_BN;
  f32x4 o[QT][ND];
  float ref[QT], thr[QT], l[QT];
#pragma unroll
  for (int t = 0; t < QT; ++t) {
    ref[t] = 0.f, thr[t] = -INFINITY, l[t] = 0.f;
#pragma unroll
    for (int i = 0; i < ND; ++i) o[t][i] = f32x4{0.f, 0.f, 0.f, 0.f};
  }

  // the table is only read here: as constant memory its uniform reads are scalar
  const auto* table = (const __attribute__((address_space(4))) int32_t*)(c.table + (int64_t)b * c.max_pages);
  auto page_of = [&](int tok) { return (int)((uint64_t)(uint32_t)tok * a.page_mul >> a.page_shift); };
  struct Pages {
    int id[NP];
  };
  auto look_up = [&](int tk) {  // -1 where the piece has no such tokens
    Pages p;
#pragma unroll
    for (int i = 0; i < NP; ++i) {
      p.id[i] = -1;
      if (tk + PT * i < tend) p.id[i] = table[page_of(tk + PT * i)];
    }
    return p;
  };
  int at_issue = 0, at_read = 0;  // byte offsets of stages
  auto issue = [&](int tk, const Pages& pg) {
    uint8_t* const dst = smem + wave * (NST * St::BYTES) + at_issue;
    at_issue = at_issue + St::BYTES == NST * St::BYTES ? 0 : at_issue + St::BYTES;
    auto lds = [&](int off) { return (__attribute__((address_space(3))) void*)(dst + off); };
    if constexpr (NP == 1) {
      const bool ok = pg.id[0] >= 0 && pg.id[0] < c.pages;  // otherwise a buffer of no bytes: zeros
      const int64_t p0 = ok ? pg.id[0] : 0, off = ok ? tk - page_of(tk) * c.page : 0;
      const __amdgpu_buffer_rsrc_t rc = __builtin_amdgcn_make_buffer_rsrc(
          (void*)(c.codes + p0 * c.codes_page + k_head + off * (D / 2)), (short)0, ok ? 0x7fffffff : 0, 0x00020000);
      const __amdgpu_buffer_rsrc_t rs = __builtin_amdgcn_make_buffer_rsrc(
          (void*)(c.scales + p0 * c.scales_page + ks_head + off), (short)0, ok ? 0x7fffffff : 0, 0x00020000);
      if (a.once) {
#pragma unroll
        for (int j = 0; j < St::NC; ++j)
          __builtin_amdgcn_raw_ptr_buffer_load_lds(rc, lds(1024 * j), 16, (int)fetch.off_c[j], 0, 0, CP_NT);
      } else {
#pragma unroll
        for (int j = 0; j < St::NC; ++j)
          __builtin_amdgcn_raw_ptr_buffer_load_lds(rc, lds(1024 * j), 16, (int)fetch.off_c[j], 0, 0, CP_PLAIN);
      }
#pragma unroll
      for (int j = 0; j < St::NS; ++j)
        __builtin_amdgcn_raw_ptr_buffer_load_lds(rs, lds(St::CODES + 256 * j), 4, (int)fetch.off_s[j], 0, 0, 0);
    } else {
      const uint8_t *bc[NP], *bs[NP];
      bool ok[NP], all = true;
#pragma unroll
      for (int i = 0; i < NP; ++i) {
        const int64_t p = pg.id[i];
        ok[i] = p >= 0 && p < c.pages;
        all = all && ok[i];
        const int64_t off = tk + PT * i - page_of(tk + PT * i) * c.page;
        bc[i] = c.codes + p * c.codes_page + k_head + off * (D / 2);
        bs[i] = c.scales + p * c.scales_page + ks_head + off;
      }
      auto from = [&](const uint8_t* const (&base)[NP], int i, uint32_t off, bool every) {
        const uint8_t* b = base[0];
        bool o = ok[0];
#pragma unroll
        for (int n = 1; n < NP; ++n) b = i == n ? base[n] : b, o = i == n ? ok[n] : o;
        b += off;
        if (!every) b = o ? b : (const uint8_t*)ka_zeros;
        return (const __attribute__((address_space(1))) void*)b;
      };
      auto get = [&](bool every) {
#pragma unroll
        for (int j = 0; j < St::NC; ++j)
          __builtin_amdgcn_global_load_lds(from(bc, fetch.part_c[j], fetch.off_c[j], every), lds(1024 * j), 16, 0, 0);
#pragma unroll
        for (int j = 0; j < St::NS; ++j)
          __builtin_amdgcn_global_load_lds(from(bs, fetch.part_s[j], fetch.off_s[j], every), lds(St::CODES + 256 * j), 4, 0, 0);
      };
      if (all) get(true);
      else get(false);
    }
  };
  auto read_k = [&](KaTile<D>& x) {  // and the scales
    const uint32_t st = ring + at_read;
    unroll<0, S::N>([&](auto s) {
      constexpr int W = S::w(s), B0 = S::base(s);
      uint32_t k0[W / 2], k1[W / 2];
      ka_read_k<W, 16 * B0, St::CODES + B0, St::CODES + D + B0>(
          k0, k1, x.ks[0][s], x.ks[1][s], x.vs[s], st + (W == 8 ? 16u * lane : W == 4 ? k64 : k32),
          st + jl + 32 * (4 * W * g / 32), st + 4 * g + 32 * (W * jl / 32));
#pragma unroll
      for (int i = 0; i < W / 2; ++i) x.k[0][B0 / 32 + i] = k0[i], x.k[1][B0 / 32 + i] = k1[i];
    });
  };
  auto read_v = [&](KaTile<D>& x) {  // and on to the next stage
    const uint32_t st = ring + at_read;
    at_read = at_read + St::BYTES == NST * St::BYTES ? 0 : at_read + St::BYTES;
    unroll<0, S::N>([&](auto s) {
      constexpr int W = S::w(s), B0 = S::base(s);
      uint32_t v[8];
      ka_read_v<W, 16 * (D + B0)>(v, st + W / 2 * lane);
#pragma unroll
      for (int i = 0; i < 8; ++i) x.v[i][s] = v[i];
    });
  };

  u32x4 q[QT][NK];  // columns jl of the 16-row tiles
  int lim[QT];      // keys that they see
  // S^T of the tile: rows are keys, columns queries
  auto scores = [&](const KaTile<D>& x, f32x4 (&sc)[QT][2], auto f16) {
    constexpr bool F16 = decltype(f16)::value;
    unroll<0, S::N>([&](auto s) {
      constexpr int W = S::w(s), B0 = S::base(s);
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        const float f = kv4::scale_of(x.ks[i][s]);
#pragma unroll
        for (int w = 0; w < W / 2; ++w) {
          const uint32_t kw = x.k[i][B0 / 32 + w];
          const u32x4 kf = {ka_cvt<F16, 0>(kw, f), ka_cvt<F16, 1>(kw, f), ka_cvt<F16, 2>(kw, f), ka_cvt<F16, 3>(kw, f)};
#pragma unroll
          for (int t = 0; t < QT; ++t) {
            if constexpr (BF16 || F16) {
              sc[t][i] = ka_mma<F16>(kf, q[t][B0 / 32 + w], sc[t][i]);
            } else {
              u32x4 qh, ql;
              ka_split_f16(q[t][B0 / 32 + w], qh, ql);
              sc[t][i] = ka_mma<false>(kf, ql, ka_mma<false>(kf, qh, sc[t][i]));
            }
          }
        }
      }
    });
  };
  // the column's reference moves when a score passes it by too much; whether one moved to KA_FAR or beyond
  auto weigh = [&](int t, float top) {
    bool far = false;
    if (__any(top > thr[t])) {
      top = xhalf_max(xrow_max(top));  // over the four lanes of the column
      const bool up = top > thr[t];
      const float next = fabsf(top) < KA_FAR ? top - KA_BIAS : top;
      far = __any(up && fabsf(top) >= KA_FAR && top < INFINITY);  // (with an infinity the row is NaN in either form)
      const float f = !up ? 1.f : thr[t] == -INFINITY ? 0.f : fast_exp2(ref[t] - next);
      ref[t] = up ? next : ref[t];
      thr[t] = up ? top + KA_SLACK : thr[t];
      l[t] *= f;
#pragma unroll
      for (int i = 0; i < ND; ++i) o[t][i] *= f;
    }
    return far;
  };
  // V^T operands of each 16 dims: row jl is a dim, the lane's eight tokens lie along
  auto values = [&](auto f16, auto&& word, auto&& scale, auto&& use) {
    constexpr bool F16 = decltype(f16)::value;
    unroll<0, S::N>([&](auto s) {
      constexpr int W = S::w(s), B0 = S::base(s);
      unroll<0, W / 2>([&](auto sel) {
        uint32_t cv[8];
#pragma unroll
        for (int i = 0; i < 8; ++i) cv[i] = ka_cvt<F16, sel>(word(i, s), scale(i, s));
        u32x4 even, other;
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          even[i] = __builtin_amdgcn_perm(cv[2 * i + 1], cv[2 * i], 0x05040100);
          other[i] = __builtin_amdgcn_perm(cv[2 * i + 1], cv[2 * i], 0x07060302);
        }
        use(B0 / 16 + 2 * sel, even);
        use(B0 / 16 + 2 * sel + 1, other);
      });
    });
  };

  // What a last tile has beyond the keys becomes zeros of scale 1.
  auto clear_scales = [&](KaTile<D>& x, int tk) {
    unroll<0, S::N>([&](auto s) {
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        const int at = 8 * (i & 3);
        x.vs[s][i >> 2] = tk + ka_token(g, i) < e.keys ? x.vs[s][i >> 2] : (x.vs[s][i >> 2] & ~(255u << at)) | 127u << at;
      }
#pragma unroll
      for (int i = 0; i < 2; ++i) x.ks[i][s] = tk + 16 * i + jl < e.keys ? x.ks[i][s] : 127u;
    });
  };
  auto clear_v = [&](KaTile<D>& x, int tk) {
    unroll<0, S::N>([&](auto s) {
#pragma unroll
      for (int i = 0; i < 8; ++i) x.v[i][s] = tk + ka_token(g, i) < e.keys ? x.v[i][s] : 0u;
    });
  };
  // Whether fp16 holds all V (bf16 queries) or K (fp16 queries) of the tile, and no V is NaN.
  auto suits = [&](const KaTile<D>& x) {
    uint32_t no = 0;
    unroll<0, S::N>([&](auto s) {
      no |= BF16 ? ka_not_f16(x.vs[s][0]) | ka_not_f16(x.vs[s][1])
                 : ((ka_not_f16(x.ks[0][s]) | ka_not_f16(x.ks[1][s])) & 255u) | ka_nan(x.vs[s][0]) | ka_nan(x.vs[s][1]);
    });
    return !__any(no != 0);
  };
  // A tile. ALL: every row sees all of it (FAST only). FAST (it suits): V (bf16 queries) or K (fp16) in fp16; else all in bf16, weights
  // and fp16 queries in two terms. False where a score is too far for the fast form: the tile is still to be done.
  auto compute = [&](KaTile<D>& x, int tk, auto all, auto form) {
    constexpr bool ALL = decltype(all)::value, FAST = decltype(form)::value, PV16 = BF16 && FAST;
    f32x4 sc[QT][2];
#pragma unroll
    for (int t = 0; t < QT; ++t) sc[t][0] = sc[t][1] = f32x4{0.f, 0.f, 0.f, 0.f};
    scores(x, sc, std::bool_constant<!BF16 && FAST>{});
    if constexpr (!ALL) {
#pragma unroll
      for (int t = 0; t < QT; ++t)
#pragma unroll
        for (int i = 0; i < 8; ++i)
          sc[t][i >> 2][i & 3] = tk + ka_token(g, i) < lim[t] ? sc[t][i >> 2][i & 3] : -INFINITY;
    }
    u32x4 ph[QT], pl[QT];
#pragma unroll
    for (int t = 0; t < QT; ++t) {
      float top = -INFINITY;
#pragma unroll
      for (int i = 0; i < 8; ++i) top = fmaxf(top, sc[t][i >> 2][i & 3]);
      const bool far = weigh(t, top * a.scale2);
      if (FAST && far) return false;
      float y[8];
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        const float x = sc[t][i >> 2][i & 3];
        y[i] = fast_exp2(FAST ? fmaf(x, a.scale2, -ref[t]) : ka_mul(x, a.scale2) - ref[t]);
      }
      l[t] += ((y[0] + y[1]) + (y[2] + y[3])) + ((y[4] + y[5]) + (y[6] + y[7]));
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        if constexpr (PV16) {
          ph[t][i] = h16<false>::pack(y[2 * i], y[2 * i + 1]);
        } else {
          uint32_t hw, lw;
          ka_split(y[2 * i], y[2 * i + 1], hw, lw);
          ph[t][i] = hw, pl[t][i] = lw;
        }
      }
    }
    read_v(x);
    if constexpr (!ALL) clear_v(x, tk);
    if constexpr (!FAST) {
      // NaN of V that a row does not see must not meet its weight of 0: such blocks become zeros, and the rows that see
      // one become NaN by their count of it
      u32x4 seen[QT];
      __builtin_amdgcn_sched_barrier(0);
#pragma unroll
      for (int t = 0; t < QT; ++t)
#pragma unroll
        for (int i = 0; i < 4; ++i)
          seen[t][i] = (tk + ka_token(g, 2 * i) < lim[t] ? 0x3f80u : 0u) |
                       (tk + ka_token(g, 2 * i + 1) < lim[t] ? 0x3f800000u : 0u);
      unroll<0, S::N>([&](auto s) {
        constexpr int W = S::w(s), B0 = S::base(s);
        u32x4 bad = {0, 0, 0, 0};
#pragma unroll
        for (int i = 0; i < 8; ++i) {
          const int at = 8 * (i & 3);
          const bool nan = (ka_nan(x.vs[s][i >> 2]) >> at & 128u) != 0;
          bad[i >> 1] |= !nan ? 0u : (i & 1) ? 0x3f800000u : 0x3f80u;
          x.v[i][s] = nan ? 0u : x.v[i][s];
          x.vs[s][i >> 2] = nan ? (x.vs[s][i >> 2] & ~(255u << at)) | 127u << at : x.vs[s][i >> 2];
        }
#pragma unroll
        for (int t = 0; t < QT; ++t) {
          const f32x4 count = ka_mma<false>(bad, seen[t], f32x4{0.f, 0.f, 0.f, 0.f});
#pragma unroll
          for (int d = 0; d < W; ++d)
#pragma unroll
            for (int i = 0; i < 4; ++i) o[t][B0 / 16 + d][i] = count[i] > 0.f ? NAN : o[t][B0 / 16 + d][i];
          __builtin_amdgcn_sched_barrier(0);
        }
      });
    }
    if constexpr (!FAST) __builtin_amdgcn_sched_barrier(0);
    values(std::bool_constant<PV16>{}, [&](int i, int s) { return x.v[i][s]; },
           [&](int i, int s) { return kv4::scale_of((x.vs[s][i >> 2] >> (8 * (i & 3))) & 255u); },
           [&](int d, u32x4 vf) {
#pragma unroll
             for (int t = 0; t < QT; ++t) {
               o[t][d] = ka_mma<PV16>(vf, ph[t], o[t][d]);
               if constexpr (!PV16) o[t][d] = ka_mma<false>(vf, pl[t], o[t][d]);
             }
             if constexpr (!FAST) __builtin_amdgcn_sched_barrier(0);  // fewer registers
           });
    return true;
  };

  if (t0 < tend) {
    Pages pg[NST];
#pragma unroll
    for (int i = 0; i < NST; ++i) pg[i] = look_up(t0 + i * KA_UNIT);
#pragma unroll
    for (int t = 0; t < QT; ++t) {
      const int i = 16 * t + jl;
      const int row = e.row0 + i, j = ka_token_of(a, row);
      const bool live = i < e.rows;
      lim[t] = live && a.causal ? max(0, L - n + 1 + j) : e.keys;
      const uint16_t* p = a.q + b * a.qb + j * a.qr + (int64_t)(h * a.group + row - j * a.group) * D;
      unroll<0, S::N>([&](auto s) {
        constexpr int W = S::w(s), B0 = S::base(s);
#pragma unroll
        for (int w = 0; w < W / 2; ++w)
          q[t][B0 / 32 + w] = live ? *(const u32x4*)(p + B0 + 4 * W * g + 8 * w) : u32x4{0, 0, 0, 0};
      });
    }
#pragma unroll
    for (int i = 0; i < NST - 1; ++i) issue(t0 + i * KA_UNIT, pg[i]);
    Pages ahead = pg[NST - 1];
    int ti = t0 + (NST - 1) * KA_UNIT;
#pragma unroll
    for (int t = 0; t < QT; ++t)
#pragma unroll
      for (int i = 0; i < NK; ++i)
#pragma unroll
        for (int w = 0; w < 4; ++w) q[t][i][w] ^= a.q_sign;

    auto next = [&] {  // the tile at t0 is in LDS, and one more on the way
      issue(ti, ahead);
      ti += KA_UNIT;
      ahead = look_up(ti);
      vm_wait<(NST - 1) * St::PER>();
    };
    // Loops of one form each (a choice within a loop costs registers): tiles that every row sees whole, the others, and
    // from the first tile on that does not suit or has a score too far
    const int whole_end = min(tend, e.keys_min);
    bool fast = true;
    for (; t0 + KA_BN <= whole_end; t0 += KA_UNIT) {
      next();
      KaTile<D> x;
      read_k(x);
      fast = suits(x) && compute(x, t0, std::true_type{}, std::true_type{});
      if (!fast) break;
    }
    if (fast)
      for (; t0 < tend; t0 += KA_UNIT) {
        next();
        KaTile<D> x;
        read_k(x);
        clear_scales(x, t0);
        fast = suits(x) && compute(x, t0, std::false_type{}, std::true_type{});
        if (!fast) break;
      }
    for (bool here = true; !fast && t0 < tend; t0 += KA_UNIT, here = false) {
      if (!here) next();
      KaTile<D> x;
      read_k(x);
      clear_scales(x, t0);
      compute(x, t0, std::false_type{}, std::false_type{});
    }
  }
  vm_wait<0>();  // nothing may land in the exchange
  __syncthreads();

  // the waves' rows meet: 16 at a time
#pragma unroll
  for (int t = 0; t < QT; ++t) {
    float sum = l[t];
    sum += __shfl_xor(sum, 16, 64);
    sum += __shfl_xor(sum, 32, 64);
    if (g == 0) {
      sh.m[wave][jl] = thr[t] == -INFINITY && sum == 0.f ? -INFINITY : ref[t];
      sh.l[wave][jl] = sum;
    }
    unroll<0, S::N>([&](auto s) {
      constexpr int W = S::w(s), B0 = S::base(s);
#pragma unroll
      for (int i = 0; i < 4; ++i)
#pragma unroll
        for (int d = 0; d < W; ++d) so[wave][jl][B0 + 4 * W * g + W * i + d] = o[t][B0 / 16 + d][i];
    });
    __syncthreads();
    for (int x = tid; x < 16 * (D / 4); x += 64 * KA_W) {
      const int row = x / (D / 4), d = 4 * (x - row * (D / 4));
      const int i = 16 * t + row;
      if (i >= e.rows) continue;
      float m = -INFINITY, sum2 = 0.f;
      f32x4 acc = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
      for (int w = 0; w < KA_W; ++w) m = fmaxf(m, sh.m[w][row]);
#pragma unroll
      for (int w = 0; w < KA_W; ++w) {
        if (sh.m[w][row] == -INFINITY) continue;
        const float f = fast_exp2(sh.m[w][row] - m);
        sum2 += f * sh.l[w][row];
        acc += f * *(const f32x4*)&so[w][row][d];
      }
      if (pc.slot == nullptr) {
        const int qrow = e.row0 + i, j = ka_token_of(a, qrow);
        const int64_t at_o = ((int64_t)b * a.T + j) * a.H + h * a.group + (qrow - j * a.group);
        const float inv = sum2 == 0.f ? 0.f : 1.f / sum2;
        *(u32x2*)(a.o + at_o * D + d) = u32x2{h16<BF16>::pack(acc[0] * inv, acc[1] * inv),
                                              h16<BF16>::pack(acc[2] * inv, acc[3] * inv)};
        if (a.lse && d == 0) a.lse[at_o] = sum2 == 0.f ? -INFINITY : m + __log2f(sum2);
      } else {
        *(f32x4*)(pc.slot + i * D + d) = acc;
        if (d == 0) {
          pc.slot[MT * D + i] = m;
          pc.slot[MT * D + MT + i] = sum2;
        }
      }
    }
    __syncthreads();
  }
}

template <int D, int QT, bool BF16, int NP>
__global__ __launch_bounds__(64 * KA_W, ka_per_cu(D, QT)) void kv4_attn_ranges(const KaArgs a) {
#if defined(__HIP_DEVICE_COMPILE__)
  constexpr int MT = 16 * QT;
  __shared__ __attribute__((aligned(1024))) uint8_t smem[KA_W * ka_stages<D, QT>() * Stage<D>::BYTES];
  __shared__ KaShared sh;
  __shared__ int64_t find[KA_W + 3];
  const int tid = threadIdx.x;
  const int h = blockIdx.x % a.c.Hkv, r = blockIdx.x / a.c.Hkv;

  int64_t lo = 0, hi = 0;
  auto want = [&](int64_t total) {
    const int ng = ka_ranges<D, QT>(a, total);
    if (r < ng) {
      const KaCuts cuts(total, ng);
      lo = cuts.at(r);
      hi = cuts.at(r + 1);
    }
    return r < ng ? lo : (int64_t)-1;
  };
  const KaPoint start = a.few ? ka_find64<MT>(a, want) : ka_find<MT>(a, find, want);
  if (h == 0 && tid == 0) {
    KaCut cut{-1, 0, 0, 0, 0};
    if (lo < hi && start.before < lo) {
      const int ng = ka_ranges<D, QT>(a, start.total);
      const KaCuts cuts(start.total, ng);
      if (cuts.at(r - 1) <= start.before) {
        const int units = ka_entry<MT>(a, start.L, start.n, start.rt).units;
        const int p0 = cuts.range_of(start.before + KA_PIECE, start.total);
        const int p1 = cuts.range_of(start.before + KA_PIECE + units - 1, start.total);
        if (units > 0 && p1 > p0) cut = KaCut{start.b, start.rt, start.n, p0, p1};
      }
    }
    a.cuts[r] = cut;
  }
  if (lo >= hi) return;  // whole workgroup

  const KaFetch<D, NP> fetch(a.c, tid & 63);
  int64_t before = start.before;
  int rt = start.rt;
  for (int b = start.b; b < a.B && before < hi; ++b, rt = 0) {
    const int L = b == start.b ? start.L : ka_len(a, b), n = b == start.b ? start.n : ka_new(a, b);
    const int rts = ka_tiles<MT>(a, n);
    for (; rt < rts && before < hi; ++rt) {
      KaPiece pc;
      pc.e = ka_entry<MT>(a, L, n, rt);
      const int64_t at = before;
      before += pc.e.units + KA_PIECE;
      const int u0 = ka_unit_at(lo, at, pc.e.units), u1 = ka_unit_at(hi, at, pc.e.units);
      if (u0 >= u1 && !(pc.e.units == 0 && lo <= at)) continue;
      pc.b = b, pc.h = h;
      pc.t0 = u0 * KA_UNIT, pc.t1 = min(pc.e.keys, u1 * KA_UNIT);
      pc.slot = nullptr;
      if (u0 > 0 || u1 < pc.e.units)
        pc.slot = a.part + ((int64_t)(u0 == 0 ? 2 * r + 1 : 2 * r) * a.c.Hkv + h) * (MT * (D + 2));
      ka_piece<D, QT, BF16, NP>(a, pc, fetch, smem, sh);
    }
  }
#endif
}

// Entries that lie in several ranges: one workgroup per entry's first cut, K/V head and 4 / WPR rows, WPR waves for
// a row. Lanes hold 4 dims each; a row's groups of D / 4 lanes share its pieces, four of them requested at once and merged
// against a running reference, then the groups' results meet in LDS: two trips to memory, the cut and the pieces.
template <int D, int QT, bool BF16, int WPR>
__global__ __launch_bounds__(256) void kv4_attn_join(const KaArgs a) {
  constexpr int MT = 16 * QT, LPG = D / 4, GPW = 64 / LPG, STEP = GPW * WPR;
  __shared__ f32x4 acc_s[4][64];
  __shared__ float top_s[4][GPW], sum_s[4][GPW];
  const int h = blockIdx.y, wave = threadIdx.x >> 6, lane = threadIdx.x & 63;
  const int i = blockIdx.z * (4 / WPR) + wave / WPR;  // row of the entry
  const KaCut cut = a.cuts[blockIdx.x + 1];
  if (cut.b < 0) return;
  const int row = cut.rt * MT + i;
  const int np = i < MT && row < cut.n * a.group ? cut.p1 - cut.p0 + 1 : 0;
  const int grp = lane / LPG, d = 4 * (lane - grp * LPG);
  float top = -INFINITY, sum = 0.f;
  f32x4 acc = {0.f, 0.f, 0.f, 0.f};
  for (int p = wave % WPR * GPW + grp; grp < GPW && p < np; p += 4 * STEP) {
    f32x4 o[4];
    float m[4], l[4];
#pragma unroll
    for (int u = 0; u < 4; ++u) {
      const int pu = min(p + u * STEP, np - 1);
      // the first piece lies at its range's end, the others at the start
      const float* s = a.part + ((int64_t)(2 * (cut.p0 + pu) + (pu == 0)) * a.c.Hkv + h) * (MT * (D + 2));
      o[u] = *(const f32x4*)(s + i * D + d);
      m[u] = s[MT * D + i];
      l[u] = s[MT * D + MT + i];
    }
    float next = top;
#pragma unroll
    for (int u = 0; u < 4; ++u) {
      if (p + u * STEP >= np) m[u] = -INFINITY;
      next = fmaxf(next, m[u]);
    }
    if (next == -INFINITY) continue;
    const float f = top == -INFINITY ? 0.f : fast_exp2(top - next);
    sum *= f;
    acc *= f;
#pragma unroll
    for (int u = 0; u < 4; ++u)
      if (m[u] != -INFINITY) {
        const float w = fast_exp2(m[u] - next);
        sum += w * l[u];
        acc += w * o[u];
      }
    top = next;
  }
  acc_s[wave][lane] = acc;
  if (grp < GPW && d == 0) top_s[wave][grp] = top, sum_s[wave][grp] = sum;
  __syncthreads();
  if (np == 0 || wave % WPR != 0 || lane >= LPG) return;
  top = -INFINITY, sum = 0.f;
  acc = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
  for (int w = 0; w < WPR; ++w)
#pragma unroll
    for (int u = 0; u < GPW; ++u) top = fmaxf(top, top_s[wave + w][u]);
#pragma unroll
  for (int w = 0; w < WPR; ++w)
#pragma unroll
    for (int u = 0; u < GPW; ++u) {
      if (top_s[wave + w][u] == -INFINITY) continue;
      const float f = fast_exp2(top_s[wave + w][u] - top);
      sum += f * sum_s[wave + w][u];
      acc += f * acc_s[wave + w][u * LPG + lane];
    }
  const int j = ka_token_of(a, row);
  const int64_t at_o = ((int64_t)cut.b * a.T + j) * a.H + h * a.group + (row - j * a.group);
  const float inv = sum == 0.f ? 0.f : 1.f / sum;
  *(u32x2*)(a.o + at_o * D + d) = u32x2{h16<BF16>::pack(acc[0] * inv, acc[1] * inv),
                                        h16<BF16>::pack(acc[2] * inv, acc[3] * inv)};
  if (a.lse && lane == 0) a.lse[at_o] = sum == 0.f ? -INFINITY : top + __log2f(sum);
}

constexpr int KA_CUS = 256;

struct KaPlan {
  int qt, G;
  size_t meta, part;  // bytes
};
KaPlan ka_plan(int64_t rows, int64_t Hkv, int64_t D) {
  KaPlan p;
  p.qt = rows <= 16 || D > 128 ? 1 : 2;
  const int per_cu = ka_per_cu((int)D, p.qt);
  p.G = (int)std::max<int64_t>(1, KA_CUS * per_cu / Hkv);
  p.meta = (size_t)p.G * sizeof(KaCut);
  p.part = (size_t)2 * p.G * Hkv * 16 * p.qt * (D + 2) * sizeof(float);
  return p;
}

template <int D, int QT, bool BF16>
void ka_launch(const KaArgs& a, hipStream_t st) {
  const dim3 grid((unsigned)(a.G * a.c.Hkv));
  if (a.c.page % 32 == 0) kv4_attn_ranges<D, QT, BF16, 1><<<grid, 64 * KA_W, 0, st>>>(a);
  else if (a.c.page % 16 == 0) kv4_attn_ranges<D, QT, BF16, 2><<<grid, 64 * KA_W, 0, st>>>(a);
  else kv4_attn_ranges<D, QT, BF16, 4><<<grid, 64 * KA_W, 0, st>>>(a);
  if (a.G == 1) return;
  // pieces per entry, on average: with many, four waves share a row
  const int rows = (int)std::min<int64_t>(16 * QT, (int64_t)a.T * a.group);
  const int64_t entries = (int64_t)a.B * (((int64_t)a.T * a.group + 16 * QT - 1) / (16 * QT));
  if (a.G >= 8 * entries)
    kv4_attn_join<D, QT, BF16, 4><<<dim3(a.G - 1, a.c.Hkv, rows), 256, 0, st>>>(a);
  else
    kv4_attn_join<D, QT, BF16, 1><<<dim3(a.G - 1, a.c.Hkv, (rows + 3) / 4), 256, 0, st>>>(a);
}
template <int D>
void ka_go(const KaArgs& a, int qt, bool bf, hipStream_t st) {
  if constexpr (D <= 128) {
    if (qt == 2) return bf ? ka_launch<D, 2, true>(a, st) : ka_launch<D, 2, false>(a, st);
  }
  bf ? ka_launch<D, 1, true>(a, st) : ka_launch<D, 1, false>(a, st);
}

}  // namespace

extern "C" size_t tlm_kv4_attn_workspace_bytes(int64_t B, int64_t T, int64_t H, int64_t H_kv, int64_t D) {
  if (B <= 0 || T <= 0 || H <= 0 || H_kv <= 0 || D <= 0 || H % H_kv != 0) return 0;
  // enough for fewer rows, too: a chunk and the decode steps after it may share a workspace
  size_t most = 0;
  for (int64_t rows = 1, all = T * (H / H_kv); rows <= std::min<int64_t>(all, 64); ++rows) {
    const KaPlan p = ka_plan(rows, H_kv, D);
    most = std::max(most, p.meta + p.part);
  }
  return most;
}

extern "C" int tlm_kv4_attn(const void* q, int64_t q_batch_stride, int64_t q_row_stride, const void* codes,
                            int64_t codes_page_stride, const void* scales, int64_t scales_page_stride,
                            int64_t pages, const int32_t* block_table, int64_t max_pages, int64_t page,
                            const int32_t* seqlens, const int32_t* count, void* o, float* lse, void* ws,
                            size_t ws_bytes, int64_t B, int64_t T, int64_t H, int64_t H_kv, int64_t D,
                            int causal, float sm_scale, int dtype, void* stream) {
  Cache c{(uint8_t*)codes, (uint8_t*)scales, codes_page_stride, scales_page_stride, pages, block_table};
  if (int rc = kv4::check("tlm_kv4_attn", c, max_pages, page, H_kv, D, B)) return rc;
  const bool any = B != 0 && T != 0;
  if (int rc = kv4::check_rows("tlm_kv4_attn", "q", q, any, q_batch_stride, q_row_stride, dtype)) return rc;
  if ((B != 0 && !seqlens) || (any && !o)) {
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
  if (!any) return TLM_OK;
  if (H > (INT32_MAX - 64) / B || T > (INT32_MAX - 64) / (B * H)) {
    tlm_set_error("tlm_kv4_attn: problem too large (2^31 query rows)");
    return TLM_EINVAL;
  }
  const KaPlan p = ka_plan(T * (H / H_kv), H_kv, D);
  if (!ws || ws_bytes < p.meta + p.part) {
    tlm_set_error("tlm_kv4_attn: workspace of %zu bytes, %zu needed", ws ? ws_bytes : (size_t)0, p.meta + p.part);
    return TLM_EWORKSPACE;
  }
  if (!tlm_aligned(ws, 16)) {
    tlm_set_error("tlm_kv4_attn: the workspace must be 16-byte aligned");
    return TLM_EINVAL;
  }
  c.max_pages = (int)max_pages, c.page = (int)page, c.Hkv = (int)H_kv, c.D = (int)D;
  const int64_t tiles = (T * (H / H_kv) + 16 * p.qt - 1) / (16 * p.qt);
  int few = 0;
  if (B <= 64 && tiles <= INT32_MAX / (B * (max_pages * page / KA_UNIT + 1 + KA_PIECE)))
    for (few = 1; B << few <= 64;) ++few;
  // (a scale of 0 becomes the least there is: masked scores are -inf, and -inf times 0 is no weight)
  const float scale2 = std::max(fabsf(sm_scale) * 1.4426950408889634f, 0x1p-149f);
  KaArgs a{c, (const uint16_t*)q, q_batch_stride, q_row_stride, seqlens, count, (uint16_t*)o, lse,
           (KaCut*)ws, (float*)((char*)ws + p.meta), (int)B, (int)T, (int)H, (int)(H / H_kv), causal != 0, p.G, few,
           T * (H / H_kv) <= 16 * p.qt, 0, 0, 0, 0, scale2, sm_scale < 0.f ? 0x80008000u : 0u};
  // with 2^(k-1) < d <= 2^k and m = floor(2^(31+k) / d) + 1: m d - 2^(31+k) <= 2^k, so that x m / 2^(31+k) is
  // less than 1 / d above x / d for x < 2^31; and m fits 32 bits
  auto reciprocal = [](int64_t d, uint32_t& mul, int& shift) {
    for (shift = 31; (1ll << (shift - 31)) < d;) ++shift;
    mul = (uint32_t)((1ull << shift) / (uint64_t)d + 1);
  };
  reciprocal(page, a.page_mul, a.page_shift);
  reciprocal(a.group, a.group_mul, a.group_shift);
  hipStream_t st = (hipStream_t)stream;
  const bool bf = dtype == TLM_BF16;
  switch (D) {
    case 32: ka_go<32>(a, p.qt, bf, st); break;
    case 64: ka_go<64>(a, p.qt, bf, st); break;
    case 96: ka_go<96>(a, p.qt, bf, st); break;
    case 128: ka_go<128>(a, p.qt, bf, st); break;
    case 160: ka_go<160>(a, p.qt, bf, st); break;
    case 192: ka_go<192>(a, p.qt, bf, st); break;
    case 224: ka_go<224>(a, p.qt, bf, st); break;
    default: ka_go<256>(a, p.qt, bf, st); break;
  }
  TLM_LAUNCH_CHECK("tlm_kv4_attn");
  return TLM_OK;
}
