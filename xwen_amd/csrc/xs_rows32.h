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
// of the row's own scores, products that start from it.  It moves when a lane's
// weights of a step add up to more than 2^8, which their sum, needed anyway, says
// without a maximum (a prompt of 16,384 tokens with one: 2,064 us, so 2,028).
// Fragments are asked for two products ahead of theirs, the first values before
// the exponentials, and those go before the other wave's products (2,013, so 1,900).
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
  XS_DEV explicit Reads(int lane) {
    const int x = lane & 31, g = lane >> 5, i = lane & 15, vr = 4 * g + (i >> 2);
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
// weights are for the products), weights NQ parts too.  A step may instead take
// q[0] alone, with keys of a type of their own (QN, QM).
template <typename M, int DP, int NQ>
struct Rows32 {
  static constexpr int KC = DP / 16, DT = DP / 32;
  u32x4 q[NQ][KC];
  f32x16 o[DT], base;  // base: minus the reference, which the products start from
  float most, l;       // the sum of a step's weights above which the reference moves: -1 until the row's first score

  XS_DEV void init() {
    base = fill16(-0.0f);
#pragma unroll
    for (int d = 0; d < DT; d++) o[d] = fill16(0.0f);
    most = -1.0f;
    l = 0.0f;
  }
  XS_DEV float reference() const { return -base[0]; }

  // A step of U tiles of 32 keys, the first of the stages ks and vs (VN parts that add up):
  // on (Upto, Bits) is asked for key 32 u + 8 (r / 4) + r % 4 where `masked`.
  template <int U, int VN, int QN = NQ, typename QM = M, typename On>
  XS_DEV void step(const Reads<DP>& at, const u32x4* ks, const u32x4* const (&vs)[VN], float scale, bool masked, const On on) {
    constexpr float OFF = offset_of(M{});
    int kt = at.kturn, vt = at.vturn;
    asm volatile("" : "+v"(kt), "+v"(vt));
    f32x16 s[U];
#pragma unroll
    for (int u = 0; u < U; u++) s[u] = base;
    // fragments AHEAD of their products, so that LDS answers beside the others'
    constexpr int AHEAD = 2;
    u32x4 k[AHEAD + 1][U];
#pragma unroll
    for (int i = 0; i < AHEAD; i++)
#pragma unroll
      for (int u = 0; u < U; u++) k[i][u] = at.key(ks, kt, u, i);
    __builtin_amdgcn_sched_barrier(0);
#pragma unroll
    for (int i = 0; i < KC; i++) {
      if (i + AHEAD < KC) {
#pragma unroll
        for (int u = 0; u < U; u++) k[(i + AHEAD) % (AHEAD + 1)][u] = at.key(ks, kt, u, i + AHEAD);
      }
#pragma unroll
      for (int u = 0; u < U; u++)
#pragma unroll
        for (int n = 0; n < QN; n++) s[u] = mfma32(QM{}, k[i % (AHEAD + 1)][u], q[n][i], s[u]);
      __builtin_amdgcn_sched_barrier(0);
    }
    u32x4 v[2][U][2];
    auto values = [&](int i) {
#pragma unroll
      for (int u = 0; u < U; u++)
#pragma unroll
        for (int c = 0; c < 2; c++) v[i & 1][u][c] = at.value(vs[i / DT], vt, i % DT, u, c);
    };
    values(0);
    __builtin_amdgcn_sched_barrier(0);
    // (the other wave of the SIMD, in its products, needs an issue only every 32 cycles)
    __builtin_amdgcn_s_setprio(1);
    float p[U][16], sum;
    auto weigh = [&](bool from0, float ref, const On& on) {
#pragma unroll
      for (int u = 0; u < U; u++)
#pragma unroll
        for (int r = 0; r < 16; r++) {
          const float v = from0 ? s[u][r] - ref : s[u][r];
          p[u][r] = OFF == 0.0f ? v * scale : __builtin_fmaf(v, scale, OFF);
        }
      if (masked) {
#pragma unroll
        for (int u = 0; u < U; u++)
#pragma unroll
          for (int r = 0; r < 16; r++) p[u][r] = on(32 * u + 8 * (r / 4) + r % 4) ? p[u][r] : NEG_INF;
      }
      sum = 0.0f;
#pragma unroll
      for (int u = 0; u < U; u++)
#pragma unroll
        for (int r = 0; r < 16; r += 4) {
#pragma unroll
          for (int e = 0; e < 4; e++) p[u][r + e] = __builtin_amdgcn_exp2f(p[u][r + e]);
          sum += (p[u][r] + p[u][r + 1]) + (p[u][r + 2] + p[u][r + 3]);
        }
    };
    weigh(false, 0.0f, on);
    if (__any(sum > most)) [[unlikely]] {  // (a NaN does not move it: the row is lost)
      // The references of the rows that have grown move to their best scores: all
      // rows', whose products are formed again from 0, or those that start there.
      const On rare = on.again();
      const float sign = scale < 0.0f ? -1.0f : 1.0f, old = reference();
      const bool unset = most < 0.0f, far = __any(sum > most && old != 0.0f);
      if (far) [[unlikely]] {
        asm volatile("" : "+v"(kt));
#pragma unroll
        for (int u = 0; u < U; u++) {
          s[u] = fill16(0.0f);
#pragma unroll
          for (int c = 0; c < KC; c++) {
            const u32x4 k = at.key(ks, kt, u, c);
#pragma unroll
            for (int n = 0; n < QN; n++) s[u] = mfma32(QM{}, k, q[n][c], s[u]);
            __builtin_amdgcn_sched_barrier(0);  // (one chunk in registers at a time)
          }
        }
      }
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
      float ref = far ? old : 0.0f;  // (of a row that does not move: what its s lacks)
      if ((far || old == 0.0f) && best > NEG_INF) {
        ref = scale == 0.0f ? 0.0f : best * sign;
        const float keep = unset ? 0.0f : __builtin_amdgcn_exp2f((old - ref) * scale);
        base = fill16(-ref);
        most = OFF == 0.0f ? 0x1p8f : 0x1p14f;  // (2^(8 + OFF))
        l *= keep;
#pragma unroll
        for (int d = 0; d < DT; d++) o[d] *= keep;
      }
      weigh(true, ref, rare.again());
    }
    l += sum;
    u32x4 pf[NQ][U][2];
#pragma unroll
    for (int u = 0; u < U; u++)
#pragma unroll
      for (int c = 0; c < 2; c++) {
#pragma unroll
        for (int e = 0; e < 4; e++) {
          const float y0 = p[u][8 * c + 2 * e], y1 = p[u][8 * c + 2 * e + 1];
          pf[0][u][c][e] = pack2(M{}, y0, y1);
          if constexpr (NQ == 2)
            pf[1][u][c][e] = pack2(M{}, y0 - M::widen((uint16_t)pf[0][u][c][e]), y1 - M::widen((uint16_t)(pf[0][u][c][e] >> 16)));
        }
      }
    __builtin_amdgcn_s_setprio(0);
    __builtin_amdgcn_sched_barrier(0);
#pragma unroll
    for (int i = 0; i < VN * DT; i++) {
      if (i + 1 < VN * DT) values(i + 1);
#pragma unroll
      for (int u = 0; u < U; u++)
#pragma unroll
        for (int c = 0; c < 2; c++)
#pragma unroll
          for (int n = 0; n < NQ; n++) o[i % DT] = mfma32(M{}, v[i & 1][u][c], pf[n][u][c], o[i % DT]);
      __builtin_amdgcn_sched_barrier(0);
    }
  }
};

}  // namespace xst
