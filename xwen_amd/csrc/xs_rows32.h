// xs_rows32.h -- attention of 32 rows a wave over keys that lie in LDS.  Device
// code; private to the library.
//
// With v_mfma_f32_32x32x16 (lane = 32 g + x; A[m = x][k = 8 g + e], B[k = 8 g + e][n = x],
// C[m = 8 (r / 4) + 4 g + r % 4][n = x]):
//
//   S^T = K Q^T   a lane holds scores of one row (n = x), of 16 of every 32 keys
//   O^T = V^T P^T the contraction runs over the keys in the order in which the
//                 lane holds them (position 8 g + e of 16 is key 8 (e / 4) + 4 g +
//                 e % 4), so the weights go to B as they are; V's fragments come
//                 through transposing LDS reads, four keys of a column each
//
// The softmax is that of xs_attend.h: one pass, a running reference which is one
// of the row's own scores, products that start from it, moved only when the best
// has grown by 2^8.
#pragma once

#include "xs_attend.h"

namespace xst {

typedef float f32x16 __attribute__((ext_vector_type(16)));
typedef short s16x4 __attribute__((ext_vector_type(4)));

XS_DEV f32x16 mfma32(Bf16, u32x4 a, u32x4 b, f32x16 c) {
  return __builtin_amdgcn_mfma_f32_32x32x16_bf16(__builtin_bit_cast(bf16x8, a), __builtin_bit_cast(bf16x8, b), c, 0, 0, 0);
}
XS_DEV f32x16 mfma32(F16, u32x4 a, u32x4 b, f32x16 c) {
  return __builtin_amdgcn_mfma_f32_32x32x16_f16(__builtin_bit_cast(f16x8, a), __builtin_bit_cast(f16x8, b), c, 0, 0, 0);
}
XS_DEV f32x16 fill16(float v) { return (f32x16){v, v, v, v, v, v, v, v, v, v, v, v, v, v, v, v}; }

// Over the two lanes of a row.
XS_DEV float pair_max(float v) {
  const u32x2 a = __builtin_bit_cast(u32x2, __builtin_amdgcn_permlane32_swap(__float_as_uint(v), __float_as_uint(v), false, false));
  return fmaxf(__uint_as_float(a[0]), __uint_as_float(a[1]));
}
XS_DEV float pair_sum(float v) {
  const u32x2 a = __builtin_bit_cast(u32x2, __builtin_amdgcn_permlane32_swap(__float_as_uint(v), __float_as_uint(v), false, false));
  return __uint_as_float(a[0]) + __uint_as_float(a[1]);
}

constexpr int SK = 64;  // keys of a stage

// A stage in LDS: rows of CH 16-byte chunks.  Chunk c of a row lies at c ^ turn,
// so that rows read together meet all banks: 16 rows' chunk of K (16 bytes each),
// four rows' 64 bytes of V.
template <int DP>
struct Keys {
  static constexpr int CH = DP / 8, STAGE = SK * CH;
  XS_DEV static int turn_k(int row) { return CH % 16 == 0 ? row & 15 : CH % 8 == 0 ? row >> 1 & 7 : row >> 2 & 3; }
  XS_DEV static int turn_v(int row) { return CH % 16 == 0 ? (row & 3) << 2 : CH % 8 == 0 ? (row >> 1 & 1) << 2 : 0; }
};

// The lane's byte offsets within a stage: K's chunk 2 c + g of row x (of 32 u +
// x: 32 rows on), V's columns 32 d + 16 q4 + 4 (i % 4) of row 4 g + i / 4, with q4
// and i the lane's half and place of 32.  What a chunk's number turns is kept
// apart from the row's part, and its sums with constants are formed where they
// are used (kept instead, they fill the registers).
template <int DP>
struct Reads {
  using K = Keys<DP>;
  static constexpr int CH = K::CH;
  int krow, kturn, vrow, vturn;
  XS_DEV Reads() {
    const int lane = threadIdx.x & 63, x = lane & 31, g = lane >> 5, i = lane & 15, vr = 4 * g + (i >> 2);
    krow = x * CH * 16;
    kturn = 16 * (g ^ K::turn_k(x));
    vrow = vr * CH * 16 + 8 * (i & 1);
    vturn = 16 * ((2 * ((lane >> 4) & 1) + ((i & 3) >> 1)) ^ K::turn_v(vr));
  }
  XS_DEV u32x4 key(const u32x4* stage, int turn, int u, int c) const {
    int at;
    if constexpr (CH % 16 == 0) at = (turn ^ (32 * (c % 8))) + 256 * (c / 8);
    else if constexpr (CH % 8 == 0) at = turn ^ (32 * c);
    else at = (turn ^ (32 * (c % 2))) + 64 * (c / 2);
    return *(const u32x4*)((const char*)stage + krow + at + 32 * u * CH * 16);
  }
  // keys 32 u + 16 c .. + 16 of columns 32 d .. + 32
  XS_DEV u32x4 value(const u32x4* stage, int turn, int d, int u, int c) const {
    const char* p = (const char*)stage + vrow + (CH % 16 == 0 ? (turn ^ (64 * (d % 4))) + 256 * (d / 4) : CH % 8 == 0 ? turn ^ (64 * d) : turn + 64 * d);
    u32x2 v[2];
#pragma unroll
    for (int h = 0; h < 2; h++)
      v[h] = __builtin_bit_cast(u32x2, __builtin_amdgcn_ds_read_tr16_b64_v4i16(
                                           (__attribute__((address_space(3))) s16x4*)(p + (32 * u + 16 * c + 8 * h) * CH * 16)));
    return (u32x4){v[0][0], v[0][1], v[1][0], v[1][1]};
  }
};

// Which keys of a step the lane's row sees, counted from the lane's first: those
// up to a limit, or those of a bit mask (shifted by the lane's first).  again()
// is the same to the compiler's eyes new, so that it forms the comparisons anew
// where they are rarely needed instead of keeping 32 of them.
struct Upto {
  int lim;
  XS_DEV bool operator()(int i) const { return i <= lim; }
  XS_DEV Upto again() const {
    Upto y = *this;
    asm volatile("" : "+v"(y.lim));
    return y;
  }
};
struct Bits {
  uint32_t lo, hi;
  XS_DEV bool operator()(int i) const { return ((i < 32 ? lo : hi) >> (i & 31)) & 1u; }
  XS_DEV Bits again() const {
    Bits y = *this;
    asm volatile("" : "+v"(y.lo), "+v"(y.hi));
    return y;
  }
};

// Rows of inputs T; queries are NQ parts that add up (of type M, as keys and
// weights are for the products), weights NQ parts too.
template <typename M, int DP, int NQ>
struct Rows32 {
  static constexpr int KC = DP / 16, DT = DP / 32;
  u32x4 q[NQ][KC];
  f32x16 o[DT], base;  // base: minus the reference, which the products start from
  float most, l;       // the x above which the reference moves: NaN until the row's first score

  XS_DEV void init() {
    base = fill16(-0.0f);
#pragma unroll
    for (int d = 0; d < DT; d++) o[d] = fill16(0.0f);
    most = __builtin_nanf("");
    l = 0.0f;
  }
  XS_DEV float reference() const { return -base[0]; }

  // A step of U tiles of 32 keys, the first of the stages ks and vs (KN parts that add up):
  // on (Upto, Bits) is asked for key 32 u + 8 (r / 4) + r % 4 where `masked`.
  template <int U, int KN, typename On>
  XS_DEV void step(const Reads<DP>& at, const u32x4* const (&ks)[KN], const u32x4* const (&vs)[KN], float scale, bool masked, const On on) {
    constexpr float OFF = offset_of(M{});
    int kt = at.kturn, vt = at.vturn;
    asm volatile("" : "+v"(kt), "+v"(vt));
    f32x16 s[U];
#pragma unroll
    for (int u = 0; u < U; u++) s[u] = base;
#pragma unroll
    for (int m = 0; m < KN; m++)
#pragma unroll
      for (int c = 0; c < KC; c++)
#pragma unroll
        for (int u = 0; u < U; u++) {
          const u32x4 k = at.key(ks[m], kt, u, c);
#pragma unroll
          for (int n = 0; n < NQ; n++) s[u] = mfma32(M{}, k, q[n][c], s[u]);
        }
    float x[U][16], top;
    auto weigh = [&](bool from0, float ref, const On& on) {
#pragma unroll
      for (int u = 0; u < U; u++)
#pragma unroll
        for (int r = 0; r < 16; r++) {
          const float v = from0 ? s[u][r] - ref : s[u][r];
          x[u][r] = OFF == 0.0f ? v * scale : __builtin_fmaf(v, scale, OFF);
        }
      if (masked) {
#pragma unroll
        for (int u = 0; u < U; u++)
#pragma unroll
          for (int r = 0; r < 16; r++) x[u][r] = on(32 * u + 8 * (r / 4) + r % 4) ? x[u][r] : NEG_INF;
      }
      top = NEG_INF;
#pragma unroll
      for (int u = 0; u < U; u++)
#pragma unroll
        for (int r = 0; r < 16; r++) top = fmaxf(top, x[u][r]);
    };
    weigh(false, 0.0f, on);
    if (__any(!(top <= most))) [[unlikely]] {
      // the references of the rows that have grown move to their best scores
      const On rare = on.again();
      asm volatile("" : "+v"(kt));
#pragma unroll
      for (int u = 0; u < U; u++) {
        s[u] = fill16(0.0f);
#pragma unroll
        for (int m = 0; m < KN; m++)
#pragma unroll
          for (int c = 0; c < KC; c++) {
            const u32x4 k = at.key(ks[m], kt, u, c);
#pragma unroll
            for (int n = 0; n < NQ; n++) s[u] = mfma32(M{}, k, q[n][c], s[u]);
            __builtin_amdgcn_sched_barrier(0);  // (one chunk in registers at a time)
          }
      }
      const float sign = scale < 0.0f ? -1.0f : 1.0f, old = reference();
      const bool unset = most != most;
      // never below the old one (a product that starts elsewhere rounds elsewhere)
      float best = unset ? NEG_INF : old * sign;
#pragma unroll
      for (int u = 0; u < U; u++)
#pragma unroll
        for (int r = 0; r < 16; r++) {
          const float y = s[u][r] * sign;
          best = fmaxf(best, !masked || rare(32 * u + 8 * (r / 4) + r % 4) ? y : NEG_INF);
        }
      best = pair_max(best);
      float ref = old;
      if (best > NEG_INF) {
        ref = scale == 0.0f ? 0.0f : best * sign;
        const float keep = unset ? 0.0f : __builtin_amdgcn_exp2f((old - ref) * scale);
        base = fill16(-ref);
        most = LAZY + OFF;
        l *= keep;
#pragma unroll
        for (int d = 0; d < DT; d++) o[d] *= keep;
      }
      weigh(true, ref, rare.again());
    }
    u32x4 pf[NQ][U][2];
#pragma unroll
    for (int u = 0; u < U; u++)
#pragma unroll
      for (int c = 0; c < 2; c++) {
        float p[8];
#pragma unroll
        for (int e = 0; e < 8; e++) p[e] = __builtin_amdgcn_exp2f(x[u][8 * c + e]);
        l += ((p[0] + p[1]) + (p[2] + p[3])) + ((p[4] + p[5]) + (p[6] + p[7]));
#pragma unroll
        for (int e = 0; e < 4; e++) {
          pf[0][u][c][e] = pack2(M{}, p[2 * e], p[2 * e + 1]);
          if constexpr (NQ == 2)
            pf[1][u][c][e] = pack2(M{}, p[2 * e] - M::widen((uint16_t)pf[0][u][c][e]), p[2 * e + 1] - M::widen((uint16_t)(pf[0][u][c][e] >> 16)));
        }
      }
#pragma unroll
    for (int m = 0; m < KN; m++)
#pragma unroll
      for (int d = 0; d < DT; d++)
#pragma unroll
        for (int u = 0; u < U; u++)
#pragma unroll
          for (int c = 0; c < 2; c++) {
            const u32x4 v = at.value(vs[m], vt, d, u, c);
#pragma unroll
            for (int n = 0; n < NQ; n++) o[d] = mfma32(M{}, v, pf[n][u][c], o[d]);
          }
  }
};

}  // namespace xst
