// Grouped-query attention over the 4-bit K/V cache (tlm_kv4_attn).
#include "tlm_kv4.h"

#include <algorithm>

namespace {

using kv4::Cache;
using ldsop::unroll;

constexpr int KA_W = 4;          // waves per workgroup
constexpr int KA_BN = 32;        // tokens per tile (one wave)
constexpr int KA_UNIT = KA_W * KA_BN;
constexpr int KA_PIECE = 1;      // cost of a piece beside its units, in units
constexpr float KA_SLACK = 8.f;  // a reference is kept until a score passes it by this much (log2)

struct KaArgs {
  Cache c;
  const uint16_t* q;
  int64_t qb, qr;
  const int32_t* seqlens;
  const int32_t* count;
  uint16_t* o;
  float* lse;
  int64_t* meta;  // [G][4]: where range r starts: sequence, row tile, cost before the entry, all cost
  float* part;    // [2 G][Hkv][16 QT][D + 2]
  int B, T, H, group, causal, G, page_shift;
  float scale2;  // sm_scale log2(e)
};

// An entry of the cost line: 16 QT query rows of one sequence (rows run over its new tokens and, within one,
// over the heads of a K/V head).
struct KaEntry {
  int L, n;           // cached tokens, new ones
  int row0, rows;     // first row, rows
  int keys, keys_min; // keys that its last row sees, and its first
  int units;
};
template <int MT>
TLM_DEV KaEntry ka_entry(const KaArgs& a, int L, int n, int rt) {
  KaEntry e;
  e.L = L, e.n = n;
  e.row0 = rt * MT;
  e.rows = min(MT, n * a.group - e.row0);
  if (a.causal) {
    e.keys = max(0, L - n + 1 + (e.row0 + e.rows - 1) / a.group);
    e.keys_min = max(0, L - n + 1 + e.row0 / a.group);
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

TLM_DEV int64_t ka_cut(int64_t total, int g, int r) { return total / g * r + total % g * r / g; }

// Units of an entry at cost `before` that fall into range [lo, hi): none of its first KA_PIECE.
TLM_DEV int ka_unit_at(int64_t x, int64_t before, int units) {
  const int64_t u = x - before - KA_PIECE;
  return u < 0 ? 0 : u > units ? units : (int)u;
}

// The whole cost, and the entry that holds position `at` of it (at < 0: none); by a block of KA_W waves.
struct KaPoint {
  int64_t total, before;
  int b, rt;
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

__device__ const u32x4 ka_zeros[64] = {};  // codes and scales of tokens without a page

template <int D>
struct KaTile {
  uint32_t k[2][D / 32], v[8][Segs<D>::N];
  uint32_t ks[2][Segs<D>::N];
  u32x2 vs[Segs<D>::N];
};

template <int N>
TLM_DEV void ka_load(uint32_t* dst, const uint8_t* p) {  // N bytes
  if constexpr (N == 16) {
    const u32x4 x = *(const u32x4*)p;
    dst[0] = x[0], dst[1] = x[1], dst[2] = x[2], dst[3] = x[3];
  } else if constexpr (N == 8) {
    const u32x2 x = *(const u32x2*)p;
    dst[0] = x[0], dst[1] = x[1];
  } else if constexpr (N == 4) {
    dst[0] = *(const uint32_t*)p;
  } else if constexpr (N == 2) {
    dst[0] = *(const uint16_t*)p;
  } else {
    dst[0] = *p;
  }
}

template <int SEL>
TLM_DEV uint32_t ka_cvt(uint32_t w, float s) {
  return __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(w, s, SEL));
}
TLM_DEV f32x4 ka_mma(u32x4 a, u32x4 b, f32x4 c) {
  return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8, a), __builtin_bit_cast(bf16x8, b), c, 0,
                                                 0, 0);
}

// Two floats -> their bf16 parts and the bf16 parts of what is left: 16 bits of each.
TLM_DEV void ka_split(float x, float y, uint32_t& hi, uint32_t& lo) {
  hi = h16<true>::pack(x, y);
  lo = h16<true>::pack(x - h16<true>::lo(hi), y - h16<true>::hi(hi));
}

template <int D, int QT, bool BF16>
__global__ __launch_bounds__(64 * KA_W, (QT == 1 && D <= 128) ? 3 : QT == 1 ? 2 : 1) void kv4_attn_ranges(const KaArgs a) {
#if defined(__HIP_DEVICE_COMPILE__)
  using S = Segs<D>;
  constexpr int MT = 16 * QT, NK = D / 32, ND = D / 16, QN = BF16 ? 1 : 2;
  constexpr int SO = D + 4;  // floats of a row of the exchange
  __shared__ float so[KA_W][16][SO];
  __shared__ float sm[KA_W][16], sl[KA_W][16];
  __shared__ int64_t sh[KA_W + 3];
  const Cache& c = a.c;
  const int tid = threadIdx.x, lane = tid & 63;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int g = lane >> 4, jl = lane & 15;
  const int h = blockIdx.x % c.Hkv, r = blockIdx.x / c.Hkv;

  int64_t lo = 0, hi = 0;
  const KaPoint start = ka_find<MT>(a, sh, [&](int64_t total) {
    const int ng = (int)min((int64_t)a.G, total);
    if (r < ng) {
      lo = ka_cut(total, ng, r);
      hi = ka_cut(total, ng, r + 1);
    }
    return r < ng ? lo : (int64_t)-1;
  });
  if (h == 0 && tid == 0) {
    int64_t* m = a.meta + 4 * r;
    m[0] = lo < hi ? start.b : -1;
    m[1] = start.rt;
    m[2] = start.before;
    m[3] = start.total;
  }
  if (lo >= hi) return;  // whole workgroup

  const int64_t k_head = (int64_t)h * c.page * (D / 2), v_head = (int64_t)(c.Hkv + h) * c.page * (D / 2);
  const int64_t ks_head = (int64_t)h * c.page * NK, vs_head = (int64_t)(c.Hkv + h) * c.page * NK;
  const int kg = jl >> 2, kr = jl & 3;  // the lane's K rows: tokens 8 kg + kr and + 4; its V rows: 8 g .. + 7

  int64_t before = start.before;
  int rt = start.rt;
  for (int b = start.b; b < a.B && before < hi; ++b, rt = 0) {
    const int L = ka_len(a, b), n = ka_new(a, b), rts = ka_tiles<MT>(a, n);
    const int32_t* table = c.table + (int64_t)b * c.max_pages;
    for (; rt < rts && before < hi; ++rt) {
      const KaEntry e = ka_entry<MT>(a, L, n, rt);
      const int64_t at = before;
      before += e.units + KA_PIECE;
      const int u0 = ka_unit_at(lo, at, e.units), u1 = ka_unit_at(hi, at, e.units);
      if (u0 >= u1 && !(e.units == 0 && lo <= at)) continue;

      // Q: column jl of each 16-row tile, as (one or two terms of) bf16
      u32x4 q[QN][QT][NK];
      int lim[QT];
#pragma unroll
      for (int t = 0; t < QT; ++t) {
        const int i = 16 * t + jl;
        const int row = e.row0 + i, j = row / a.group;
        const bool live = i < e.rows;
        lim[t] = live && a.causal ? max(0, L - n + 1 + j) : e.keys;
        const uint16_t* p = a.q + b * a.qb + j * a.qr + (int64_t)(h * a.group + row - j * a.group) * D;
        unroll<0, S::N>([&](auto s) {
          constexpr int W = S::w(s), B0 = S::base(s);
#pragma unroll
          for (int w = 0; w < W / 2; ++w) {
            const u32x4 x = live ? *(const u32x4*)(p + B0 + 4 * W * g + 8 * w) : u32x4{0, 0, 0, 0};
            if constexpr (BF16) {
              q[0][t][B0 / 32 + w] = x;
            } else {
              u32x4 xh, xl;
#pragma unroll
              for (int i2 = 0; i2 < 4; ++i2) {
                const float y0 = h16<false>::lo(x[i2]), y1 = h16<false>::hi(x[i2]);
                const uint32_t hw = h16<true>::pack(y0, y1);
                const float z0 = h16<true>::lo(hw), z1 = h16<true>::hi(hw);
                xh[i2] = hw;  // an infinity has nothing left
                xl[i2] = h16<true>::pack(fabsf(z0) < INFINITY ? y0 - z0 : 0.f, fabsf(z1) < INFINITY ? y1 - z1 : 0.f);
              }
              q[0][t][B0 / 32 + w] = xh;
              q[QN - 1][t][B0 / 32 + w] = xl;
            }
          }
        });
      }
      f32x4 o[QT][ND];
      float ref[QT], thr[QT], l[QT];
#pragma unroll
      for (int t = 0; t < QT; ++t) {
        ref[t] = 0.f, thr[t] = -INFINITY, l[t] = 0.f;
#pragma unroll
        for (int i = 0; i < ND; ++i) o[t][i] = f32x4{0.f, 0.f, 0.f, 0.f};
      }

      const int tend = min(e.keys, u1 * KA_UNIT);  // tokens from here on are not this piece's
      int t0 = u0 * KA_UNIT + wave * KA_BN;
      auto page_of = [&](int tok) { return a.page_shift >= 0 ? tok >> a.page_shift : tok / c.page; };
      auto pid_of = [&](int tok) {  // -1 where the token has no page
        const int i = page_of(tok);
        int p = -1;
        if (tok < tend) p = table[i];
        return p;
      };
      int pk = pid_of(t0 + 8 * kg), pv = pid_of(t0 + 8 * g);
      auto load = [&](KaTile<D>& x, int tk) {
        const int tok_k = tk + 8 * kg, tok_v = tk + 8 * g;
        const int pk1 = pid_of(tok_k + KA_UNIT), pv1 = pid_of(tok_v + KA_UNIT);
        const bool ok_k = pk >= 0 && pk < c.pages, ok_v = pv >= 0 && pv < c.pages;
        const int off_k = tok_k - page_of(tok_k) * c.page + kr, off_v = tok_v - page_of(tok_v) * c.page;
        const uint8_t* z = (const uint8_t*)ka_zeros;
        const uint8_t* ka = ok_k ? c.codes + pk * c.codes_page + k_head + (int64_t)off_k * (D / 2) : z;
        const uint8_t* ksa = ok_k ? c.scales + pk * c.scales_page + ks_head + off_k : z;
        const uint8_t* va = ok_v ? c.codes + pv * c.codes_page + v_head + (int64_t)off_v * (D / 2) : z;
        const uint8_t* vsa = ok_v ? c.scales + pv * c.scales_page + vs_head + off_v : z;
        const int64_t kst = ok_k ? c.page : 0, vst = ok_v ? c.page : 0;
        unroll<0, S::N>([&](auto s) {
          constexpr int W = S::w(s), B0 = S::base(s);
#pragma unroll
          for (int i = 0; i < 2; ++i) {
            ka_load<2 * W>(&x.k[i][B0 / 32], ka + i * 4 * (D / 2) + B0 / 2 + 2 * W * g);
            x.ks[i][s] = ksa[(B0 / 32 + 4 * W * g / 32) * kst + 4 * i];
          }
        });
        unroll<0, S::N>([&](auto s) {
          constexpr int W = S::w(s), B0 = S::base(s);
#pragma unroll
          for (int i = 0; i < 8; ++i) ka_load<W / 2>(&x.v[i][s], va + i * (D / 2) + B0 / 2 + jl * W / 2);
          x.vs[s] = *(const u32x2*)(vsa + (B0 / 32 + W * jl / 32) * vst);
        });
        pk = pk1, pv = pv1;
      };

      auto compute = [&](KaTile<D>& x, int tk, auto edge) {
        constexpr bool EDGE = decltype(edge)::value;
        f32x4 sc[QT][2];
#pragma unroll
        for (int t = 0; t < QT; ++t) sc[t][0] = sc[t][1] = f32x4{0.f, 0.f, 0.f, 0.f};
        unroll<0, S::N>([&](auto s) {
          constexpr int W = S::w(s), B0 = S::base(s);
#pragma unroll
          for (int i = 0; i < 2; ++i) {
            const float f = kv4::scale_of(x.ks[i][s]);
#pragma unroll
            for (int w = 0; w < W / 2; ++w) {
              const uint32_t kw = x.k[i][B0 / 32 + w];
              const u32x4 kf = {ka_cvt<0>(kw, f), ka_cvt<1>(kw, f), ka_cvt<2>(kw, f), ka_cvt<3>(kw, f)};
#pragma unroll
              for (int t = 0; t < QT; ++t)
#pragma unroll
                for (int u = 0; u < QN; ++u) sc[t][i] = ka_mma(kf, q[u][t][B0 / 32 + w], sc[t][i]);
            }
          }
        });
        u32x4 ph[QT], pl[QT];
#pragma unroll
        for (int t = 0; t < QT; ++t) {
          float y[8], top = -INFINITY;
#pragma unroll
          for (int i = 0; i < 8; ++i) {
            y[i] = sc[t][i >> 2][i & 3] * a.scale2;
            if constexpr (EDGE) y[i] = tk + 8 * g + i < lim[t] ? y[i] : -INFINITY;
            top = fmaxf(top, y[i]);
          }
          if (__any(top > thr[t])) {
            top = xhalf_max(xrow_max(top));  // over the four lanes of the column
            const bool up = top > thr[t];
            const float f = !up ? 1.f : thr[t] == -INFINITY ? 0.f : fast_exp2(ref[t] - top);
            ref[t] = up ? top : ref[t];
            thr[t] = up ? top + KA_SLACK : thr[t];
            l[t] *= f;
#pragma unroll
            for (int i = 0; i < ND; ++i) o[t][i] *= f;
          }
#pragma unroll
          for (int i = 0; i < 8; ++i) y[i] = fast_exp2(y[i] - ref[t]);
          l[t] += ((y[0] + y[1]) + (y[2] + y[3])) + ((y[4] + y[5]) + (y[6] + y[7]));
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            uint32_t hw, lw;
            ka_split(y[2 * i], y[2 * i + 1], hw, lw);
            ph[t][i] = hw, pl[t][i] = lw;
          }
        }
        bool odd = false;  // some V that 0 times is not 0, in a tile that not every row sees all of
        if constexpr (EDGE) {
          unroll<0, S::N>([&](auto s) {
#pragma unroll
            for (int i = 0; i < 8; ++i) {
              const uint32_t byte = (x.vs[s][i >> 2] >> (8 * (i & 3))) & 255u;
              if (tk + 8 * g + i >= e.keys) {
                x.v[i][s] = 0;
                x.vs[s][i >> 2] &= ~(255u << (8 * (i & 3)));
              } else {
                odd |= byte > 252u;
              }
            }
          });
          odd = __any(odd);
        }
        auto values = [&](auto&& word, auto&& scale, auto&& use) {
          unroll<0, S::N>([&](auto s) {
            constexpr int W = S::w(s), B0 = S::base(s);
            unroll<0, W / 2>([&](auto sel) {
              uint32_t cv[8];
#pragma unroll
              for (int i = 0; i < 8; ++i) cv[i] = ka_cvt<sel>(word(i, s), scale(i, s));
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
        auto word = [&](int i, int s) { return x.v[i][s]; };
        auto scale = [&](int i, int s) { return kv4::scale_of((x.vs[s][i >> 2] >> (8 * (i & 3))) & 255u); };
        if (!EDGE || !odd) {
          values(word, scale, [&](int d, u32x4 vf) {
#pragma unroll
            for (int t = 0; t < QT; ++t) o[t][d] = ka_mma(vf, pl[t], ka_mma(vf, ph[t], o[t][d]));
          });
        } else {
          // row by row: what the row does not see is 0 before it meets the row's weight of 0
          for (int t = 0; t < QT; ++t)
            for (int col = 0; col < 16; ++col) {
              const int seen = __shfl(lim[t], col, 64);
              values([&](int i, int s) { return tk + 8 * g + i < seen ? x.v[i][s] : 0u; },
                     [&](int i, int s) { return tk + 8 * g + i < seen ? scale(i, s) : 1.f; },
                     [&](int d, u32x4 vf) {
#pragma unroll
                       for (int t2 = 0; t2 < QT; ++t2) {
                         if (t2 != t) continue;
                         const f32x4 y = ka_mma(vf, pl[t2], ka_mma(vf, ph[t2], o[t2][d]));
#pragma unroll
                         for (int i = 0; i < 4; ++i) o[t2][d][i] = jl == col ? y[i] : o[t2][d][i];
                       }
                     });
            }
        }
      };

      if (t0 < tend) {
        KaTile<D> x, y;
        load(x, t0);
        // both tiles of a step are seen whole by every row
        for (; t0 + KA_UNIT + KA_BN <= min(tend, e.keys_min); t0 += 2 * KA_UNIT) {
          load(y, t0 + KA_UNIT);
          compute(x, t0, std::false_type{});
          load(x, t0 + 2 * KA_UNIT);
          compute(y, t0 + KA_UNIT, std::false_type{});
        }
        for (; t0 < tend; t0 += KA_UNIT) {
          load(y, t0 + KA_UNIT);
          compute(x, t0, std::true_type{});
          x = y;
        }
      }

      // the waves' rows meet: 16 at a time
      const bool whole = u0 == 0 && u1 == e.units;
      float* slot = a.part + ((int64_t)(u0 == 0 ? 2 * r + 1 : 2 * r) * c.Hkv + h) * (MT * (D + 2));
#pragma unroll
      for (int t = 0; t < QT; ++t) {
        float sum = l[t];
        sum += __shfl_xor(sum, 16, 64);
        sum += __shfl_xor(sum, 32, 64);
        if (g == 0) {
          sm[wave][jl] = thr[t] == -INFINITY && sum == 0.f ? -INFINITY : ref[t];
          sl[wave][jl] = sum;
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
          for (int w = 0; w < KA_W; ++w) m = fmaxf(m, sm[w][row]);
#pragma unroll
          for (int w = 0; w < KA_W; ++w) {
            if (sm[w][row] == -INFINITY) continue;
            const float f = fast_exp2(sm[w][row] - m);
            sum2 += f * sl[w][row];
            acc += f * *(const f32x4*)&so[w][row][d];
          }
          if (whole) {
            const int qrow = e.row0 + i, j = qrow / a.group;
            const int64_t at_o = ((int64_t)b * a.T + j) * a.H + h * a.group + (qrow - j * a.group);
            const float inv = sum2 == 0.f ? 0.f : 1.f / sum2;
            *(u32x2*)(a.o + at_o * D + d) = u32x2{h16<BF16>::pack(acc[0] * inv, acc[1] * inv),
                                                  h16<BF16>::pack(acc[2] * inv, acc[3] * inv)};
            if (a.lse && d == 0) a.lse[at_o] = sum2 == 0.f ? -INFINITY : m + __log2f(sum2);
          } else {
            *(f32x4*)(slot + i * D + d) = acc;
            if (d == 0) {
              slot[MT * D + i] = m;
              slot[MT * D + MT + i] = sum2;
            }
          }
        }
        __syncthreads();
      }
    }
  }
#endif
}

// Entries that a cut between two ranges went through: one workgroup per cut, K/V head and 16 rows; the first cut of
// an entry does the work.
template <int D, int QT, bool BF16>
__global__ __launch_bounds__(256) void kv4_attn_join(const KaArgs a) {
  constexpr int MT = 16 * QT;
  const int h = blockIdx.y, t = blockIdx.z;
  const int r = blockIdx.x + 1;
  const int64_t* m = a.meta + 4 * r;
  const int b = (int)m[0], rt = (int)m[1];
  if (b < 0) return;
  const int64_t at = m[2], total = m[3];
  const int ng = (int)min((int64_t)a.G, total);
  if (ka_cut(total, ng, r) <= at || ka_cut(total, ng, r - 1) > at) return;
  const int L = ka_len(a, b), n = ka_new(a, b);
  const KaEntry e = ka_entry<MT>(a, L, n, rt);
  const int64_t end = at + e.units + KA_PIECE;
  for (int x = threadIdx.x; x < 16 * (D / 4); x += 256) {
    const int row = x / (D / 4), d = 4 * (x - row * (D / 4));
    const int i = 16 * t + row;
    if (i >= e.rows) continue;
    float top = -INFINITY, sum = 0.f;
    f32x4 acc = {0.f, 0.f, 0.f, 0.f};
    int pieces = 0;
    for (int p = r - 1; p < ng; ++p) {
      const int64_t lo = ka_cut(total, ng, p), hi = ka_cut(total, ng, p + 1);
      if (lo >= end) break;
      const int u0 = ka_unit_at(lo, at, e.units), u1 = ka_unit_at(hi, at, e.units);
      if (u0 >= u1) continue;
      if (u0 == 0 && u1 == e.units) {  // one range had it all
        pieces = 0;
        break;
      }
      ++pieces;
      const float* slot = a.part + ((int64_t)(u0 == 0 ? 2 * p + 1 : 2 * p) * a.c.Hkv + h) * (MT * (D + 2));
      const float pm = slot[MT * D + i], ps = slot[MT * D + MT + i];
      const f32x4 po = *(const f32x4*)(slot + i * D + d);
      if (pm == -INFINITY) continue;
      const float next = fmaxf(top, pm);
      const float f = top == -INFINITY ? 0.f : fast_exp2(top - next), fp = fast_exp2(pm - next);
      sum = sum * f + ps * fp;
      acc = acc * f + po * fp;
      top = next;
    }
    if (pieces == 0) return;
    const int qrow = e.row0 + i, j = qrow / a.group;
    const int64_t at_o = ((int64_t)b * a.T + j) * a.H + h * a.group + (qrow - j * a.group);
    const float inv = sum == 0.f ? 0.f : 1.f / sum;
    *(u32x2*)(a.o + at_o * D + d) = u32x2{h16<BF16>::pack(acc[0] * inv, acc[1] * inv),
                                          h16<BF16>::pack(acc[2] * inv, acc[3] * inv)};
    if (a.lse && d == 0) a.lse[at_o] = sum == 0.f ? -INFINITY : top + __log2f(sum);
  }
}

constexpr int KA_CUS = 256;

struct KaPlan {
  int qt, G;
  size_t meta, part;  // bytes
};
KaPlan ka_plan(int64_t rows, int64_t Hkv, int64_t D) {
  KaPlan p;
  p.qt = rows <= 16 ? 1 : 2;
  const int per_cu = p.qt == 1 ? (D <= 128 ? 3 : 2) : 1;
  p.G = (int)std::max<int64_t>(1, KA_CUS * per_cu / Hkv);
  p.meta = (size_t)p.G * 4 * sizeof(int64_t);
  p.part = (size_t)2 * p.G * Hkv * 16 * p.qt * (D + 2) * sizeof(float);
  return p;
}

template <int D, int QT, bool BF16>
void ka_launch(const KaArgs& a, hipStream_t st) {
  kv4_attn_ranges<D, QT, BF16><<<(unsigned)(a.G * a.c.Hkv), 64 * KA_W, 0, st>>>(a);
  if (a.G > 1)
    kv4_attn_join<D, QT, BF16><<<dim3((unsigned)(a.G - 1), (unsigned)a.c.Hkv, QT), 256, 0, st>>>(a);
}
template <int D>
void ka_go(const KaArgs& a, int qt, bool bf, hipStream_t st) {
  if (qt == 1)
    bf ? ka_launch<D, 1, true>(a, st) : ka_launch<D, 1, false>(a, st);
  else
    bf ? ka_launch<D, 2, true>(a, st) : ka_launch<D, 2, false>(a, st);
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
  KaArgs a{c, (const uint16_t*)q, q_batch_stride, q_row_stride, seqlens, count, (uint16_t*)o, lse,
           (int64_t*)ws, (float*)((char*)ws + p.meta), (int)B, (int)T, (int)H, (int)(H / H_kv), causal != 0, p.G,
           (page & (page - 1)) == 0 ? __builtin_ctzll((unsigned long long)page) : -1,
           sm_scale * 1.4426950408889634f};
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
