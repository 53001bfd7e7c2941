// xs_attend.h -- what the attention kernels over a cache share: a tree's
// ancestors, the softmax of row tiles on the matrix cores, the stores, and the
// join of split results.  Device code; private to the library.
//
// Compiled with -ffp-contract=off; fused multiply-adds are written out.
#pragma once

#include <hip/hip_runtime.h>

#include <algorithm>
#include <type_traits>
#include <math.h>
#include <stdint.h>

#include "../../include/xsamp.h"

#define XS_DEV __device__ __forceinline__

namespace xst {

constexpr float LOG2E = 1.44269504088896340736f;
constexpr float LN2 = 0.69314718055994530942f;
constexpr float NEG_INF = -__builtin_huge_valf();

// Elements of the two types as f32.
struct Bf16 {
  XS_DEV static float widen(uint16_t u) { return __uint_as_float((uint32_t)u << 16); }
};
struct F16 {
  XS_DEV static float widen(uint16_t u) { return (float)__builtin_bit_cast(_Float16, u); }
};

// Inclusive prefix sums over a wave.
XS_DEV uint32_t wave_scan(uint32_t v) {
  // within rows of 16 lanes, then each row's last to the rows after it
#define XS_STEP(ctrl, rows) v += (uint32_t)__builtin_amdgcn_update_dpp(0, (int)v, ctrl, rows, 0xF, false)
  XS_STEP(0x111, 0xF);
  XS_STEP(0x112, 0xF);
  XS_STEP(0x114, 0xF);
  XS_STEP(0x118, 0xF);
  XS_STEP(0x142, 0xA);
  XS_STEP(0x143, 0xC);
#undef XS_STEP
  return v;
}

// The nodes a node sees: bit j of lane i's result is set when j is i or an
// ancestor of i; 0 where i's chain of parents does not end in -1 by way of
// ever lower nodes below n.  Each round doubles the distance a lane has gone
// up, so six rounds reach the root from any of 64 nodes.  One whole wave; p is
// the lane's parent (parent_of).
XS_DEV uint64_t ancestors(int p, int n) {
  const int lane = threadIdx.x & 63;
  int up = -2;  // -1: at the root; -2: the chain is broken
  if (lane < n) up = p == -1 ? -1 : (p >= 0 && p < lane ? p : -2);
  uint64_t seen = lane < n ? 1ull << lane : 0ull;
#pragma unroll
  for (int r = 0; r < 6; r++) {
    const int from = up < 0 ? lane : up;
    const uint64_t s = __shfl(seen, from);
    const int u = __shfl(up, from);
    if (up >= 0) {
      seen |= s;
      up = u;
    }
  }
  return up == -1 ? seen : 0ull;
}
XS_DEV int parent_of(const xs_tree_attend_args& a, int b) { return a.parent[b * a.nodes + min((int)threadIdx.x & 63, (int)a.nodes - 1)]; }

// ---------------------------------------------------------------------------
// Attention.
//
// The rows of one (sequence, kv head) are its nodes times the group of q heads
// that share the head: row r = node * group + q head.  A wave takes RT tiles of
// 16 rows and walks the keys in blocks of 32, with v_mfma_f32_16x16x32 (lane =
// 16 * g + x; A[m = x][k = 8 g + e], B[k = 8 g + e][n = x], C[m = 4 g + r][n = x]):
//
//   S^T = K Q^T   A is K (m a key, k the head's elements), B is Q, so a lane
//                 holds the scores of one row (n = x) with eight keys of the
//                 block, and a row's statistics are lane-local up to two swaps
//                 of lane groups;
//   O^T = V^T P^T the contraction runs over the keys, in the order in which the
//                 lane already holds them (position 8 g + e is key 4 g + e for
//                 e < 4 and key 16 + 4 g + e - 4 above), so the weights go
//                 from the scores' registers to B without crossing lanes, and
//                 a row's rescaling is lane-local too.  A lane loads 16 bytes of each of
//                 its eight keys' values, and byte permutes make the eight
//                 A fragments of them: fragment j is element 8 x + j of V.
//
// Softmax in one pass: weights exp2(x), x = (q.k - m) scale log2(e), with m a
// running reference, one of the row's own q.k, that follows the best of them
// only when that has grown by more than 2^8 since (a rescaling of every
// accumulator is otherwise left out; weights stay below 2^8, and the quotient
// by their sum is the same).  The products start from -m, which costs nothing
// and leaves no large term to cancel where every q.k is huge (a mask of the
// type's lowest value).  A block whose scores lie far above m would be lost in
// its rounding (masked keys before others): when the reference moves, the
// block's products are formed again from 0.  Nothing divides by the scale, and
// references are compared before they are scaled: equal scores have equal
// weights, and a q.k that is finite may overflow once it is scaled.  f16
// weights carry 2^6 more, so that the small ones of a long row stay above the
// type's subnormals.  Weights round to the inputs' type once; everything else
// is f32.

typedef float f32x2 __attribute__((ext_vector_type(2)));
typedef float f32x4 __attribute__((ext_vector_type(4)));
typedef uint32_t u32x2 __attribute__((ext_vector_type(2)));
typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));
typedef __bf16 bf16x2 __attribute__((ext_vector_type(2)));
typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));
typedef _Float16 f16x2 __attribute__((ext_vector_type(2)));
typedef _Float16 f16x8 __attribute__((ext_vector_type(8)));

constexpr int KB = 32;     // keys of a block
constexpr int NW = 4;      // waves of a workgroup
constexpr float LAZY = 8.0f;

XS_DEV f32x4 mfma(Bf16, u32x4 a, u32x4 b, f32x4 c) {
  return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8, a), __builtin_bit_cast(bf16x8, b), c, 0, 0, 0);
}
XS_DEV f32x4 mfma(F16, u32x4 a, u32x4 b, f32x4 c) {
  return __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(f16x8, a), __builtin_bit_cast(f16x8, b), c, 0, 0, 0);
}
// Two f32 rounded to the type (nearest even), the first in the low half.
XS_DEV uint32_t pack2(Bf16, float x, float y) { return __builtin_bit_cast(uint32_t, __builtin_convertvector((f32x2){x, y}, bf16x2)); }
XS_DEV uint32_t pack2(F16, float x, float y) { return __builtin_bit_cast(uint32_t, __builtin_convertvector((f32x2){x, y}, f16x2)); }
// The power of two that weights carry, and the least magnitude that is not finite.
XS_DEV constexpr float offset_of(Bf16) { return 0.0f; }
XS_DEV constexpr float offset_of(F16) { return 6.0f; }
XS_DEV constexpr uint32_t inf_of(Bf16) { return 0x7F80u; }
XS_DEV constexpr uint32_t inf_of(F16) { return 0x7C00u; }

// A value that is not finite reaches the rows that give it weight, which a product
// does not see to (0 times it is NaN).  Where a result is not finite, and its row's
// weights are numbers, the keys are walked again, three times: with 1 in the place
// of every value that is inf or NaN and 0 in the others', so that a result above 0
// says that such a value has weight; so for -inf or NaN; and with the finite values
// alone.  Two elements of V as a pass takes them:
enum { WALK = 0, ABOVE = 1, BELOW = 2, FINITE = 3 };
XS_DEV constexpr uint32_t one_of(Bf16) { return 0x3F80u; }
XS_DEV constexpr uint32_t one_of(F16) { return 0x3C00u; }
template <typename T>
XS_DEV uint32_t passed(T, uint32_t two, int pass) {
  uint32_t y = 0, inf = inf_of(T{}), one = one_of(T{});
  asm volatile("" : "+s"(inf), "+s"(one));  // (formed here, not kept in registers of the loops around)
#pragma unroll
  for (int i = 0; i < 32; i += 16) {
    const uint32_t v = (two >> i) & 0xFFFFu, size = v & 0x7FFFu;
    const bool odd = size >= inf, has = size > inf || (v >> 15) == (pass == BELOW ? 1u : 0u);
    y |= (pass == FINITE ? (odd ? 0u : v) : odd && has ? one : 0u) << i;
  }
  return y;
}
// y as marks say: inf where a value above has weight, -inf, or NaN where both have.
XS_DEV float marked(float y, uint32_t above, uint32_t below, int i) {
  uint32_t inf = 0x7F800000u;
  asm volatile("" : "+s"(inf));
  y += __uint_as_float(inf & (0u - ((above >> i) & 1u)));
  return y - __uint_as_float(inf & (0u - ((below >> i) & 1u)));
}

// Over the four lanes of a row (x, 16 + x, 32 + x, 48 + x).
XS_DEV float row_max(float v) {
  const u32x2 a = __builtin_bit_cast(u32x2, __builtin_amdgcn_permlane32_swap(__float_as_uint(v), __float_as_uint(v), false, false));
  v = fmaxf(__uint_as_float(a[0]), __uint_as_float(a[1]));
  const u32x2 b = __builtin_bit_cast(u32x2, __builtin_amdgcn_permlane16_swap(__float_as_uint(v), __float_as_uint(v), false, false));
  return fmaxf(__uint_as_float(b[0]), __uint_as_float(b[1]));
}
XS_DEV float row_sum(float v) {
  const u32x2 a = __builtin_bit_cast(u32x2, __builtin_amdgcn_permlane32_swap(__float_as_uint(v), __float_as_uint(v), false, false));
  v = __uint_as_float(a[0]) + __uint_as_float(a[1]);
  const u32x2 b = __builtin_bit_cast(u32x2, __builtin_amdgcn_permlane16_swap(__float_as_uint(v), __float_as_uint(v), false, false));
  return __uint_as_float(b[0]) + __uint_as_float(b[1]);
}

// The i-th of a unit's n workgroups takes this of its parts.  Workgroups go to
// the XCDs in turn: with n even, a part would be on the same XCDs for every
// unit, and the first XCDs would have the short sequences' few parts to
// themselves (32 sequences of 327 to 8,192 slots: 188 us, turned 151); with n
// odd the units turn by themselves.
XS_DEV int turned(int i, int unit, int n) { return n & 1 ? i : (int)((unsigned)(i + unit) % (unsigned)n); }

// How a call is cut: `groups` (sequence, kv head, split) of `tiles` row tiles
// each, a split taking `chunk` key blocks of its sequence.
struct Cut {
  int32_t G, tiles, nsplit, chunk, groups;
  float scale;          // times log2(e)
  float* part;          // [groups * tiles] partial results (nsplit > 1)
};

// A sequence's sizes, or its error.
struct Seq {
  int len, n;
  bool bad;
  XS_DEV Seq(const xs_tree_attend_args& a, int b) {
    const int64_t limit = a.max_len ? a.max_len : a.capacity;
    len = a.len[b];
    n = a.n_nodes ? a.n_nodes[b] : (int)a.nodes;
    bad = len < 0 || len > limit || n < 0 || n > a.nodes;
  }
  XS_DEV int blocks() const { return (len + KB - 1) / KB + (n + KB - 1) / KB; }
};

template <int DP, int RT>
struct Shape {
  static constexpr int KC = DP / 32;                 // 32-element chunks of a key
  static constexpr int VH = DP > 128 ? 2 : 1;        // halves of a value row
  static constexpr int VE = DP >= 128 ? 8 : 4;       // value elements a lane loads of a half
  static constexpr int NF = VH * VE;                 // A fragments of V^T
  static constexpr int STAT = RT * NF * 256;         // floats of a partial result: fragments,
  static constexpr int PART = STAT + RT * 32 + 4;    // then m and l of each row, and 16 bytes to spare: what contexts are sized by
  static constexpr int MARKS = (RT * NF + 7) / 8;    // words of a bit for each of a lane's elements
};

template <typename T, int DP, int RT>
struct Wave {
  using S = Shape<DP, RT>;
  u32x4 q[RT][S::KC];
  f32x4 o[RT][S::NF];
  // Minus the row's reference (of q.k), which the scores' products start from:
  // four times, as they take it, or once where registers are short (four times,
  // the wide kernel's loop reads one from scratch memory, behind the loads of the
  // next stage: 283 us for 225 where 8 sequences of 64 nodes see 8,192 slots of
  // head size 136).
  static constexpr bool ONCE = DP > 128;
  std::conditional_t<ONCE, float, f32x4> c[RT];
  float most[RT];  // the x above which the reference moves: NaN until the row's first score
  float l[RT];

  XS_DEV float minus(float v) const { return v; }
  XS_DEV float minus(const f32x4& v) const { return v[0]; }
  XS_DEV f32x4 start(int t) const {
    const float v = minus(c[t]);
    return (f32x4){v, v, v, v};
  }
  XS_DEV void refer(int t, float ref) {
    if constexpr (ONCE) c[t] = -ref;
    else c[t] = (f32x4){-ref, -ref, -ref, -ref};
  }

  XS_DEV void init() {
#pragma unroll
    for (int t = 0; t < RT; t++) {
      refer(t, -0.0f);
      most[t] = __builtin_nanf("");
      l[t] = 0.0f;
#pragma unroll
      for (int f = 0; f < S::NF; f++) o[t][f] = (f32x4){0.0f, 0.0f, 0.0f, 0.0f};
    }
  }

  // A tile's eight scores s (less the reference) times the scale; the largest.
  // `on` is the lane's mask of the block's keys.
  template <bool MASKED>
  XS_DEV float scaled(const f32x4 (&s)[2], float scale, uint32_t on, float (&x)[8]) {
    constexpr float OFF = offset_of(T{});
    const int g = (threadIdx.x & 63) >> 4;
#pragma unroll
    for (int e = 0; e < 8; e++) {
      x[e] = OFF == 0.0f ? s[e >> 2][e & 3] * scale : __builtin_fmaf(s[e >> 2][e & 3], scale, OFF);
      if (MASKED) x[e] = ((on >> (4 * g + (e & 3) + 16 * (e >> 2))) & 1u) ? x[e] : NEG_INF;
    }
    return fmaxf(fmaxf(fmaxf(x[0], x[1]), fmaxf(x[2], x[3])), fmaxf(fmaxf(x[4], x[5]), fmaxf(x[6], x[7])));
  }
  // Whether the lane's row has a score past its reference's reach, or its first
  // one (-inf too, which then changes nothing).
  XS_DEV bool passes(int t, float top) const { return !(top <= most[t]); }
  // Moves the references of the tile's rows to their best score (rare).  s: the
  // scores from 0, of all rows or of those whose reference is 0.
  template <bool MASKED>
  XS_DEV void rebase(int t, const f32x4 (&s)[2], bool all, float scale, uint32_t on, float (&x)[8]) {
    constexpr float OFF = offset_of(T{});
    const int g = (threadIdx.x & 63) >> 4;
    asm volatile("" : "+s"(scale));  // (nothing of it is kept from block to block)
    const float sign = scale < 0.0f ? -1.0f : 1.0f, old = -minus(c[t]);
    const bool unset = most[t] != most[t];
    // never below the old one (a product that starts elsewhere rounds elsewhere)
    float best = unset ? NEG_INF : old * sign;
#pragma unroll
    for (int e = 0; e < 8; e++) {
      const float y = s[e >> 2][e & 3] * sign;
      best = fmaxf(best, !MASKED || ((on >> (4 * g + (e & 3) + 16 * (e >> 2))) & 1u) ? y : NEG_INF);
    }
    best = row_max(best);
    if ((all || old == 0.0f) && best > NEG_INF) {
      const float ref = scale == 0.0f ? 0.0f : best * sign;
      const float keep = unset ? 0.0f : __builtin_amdgcn_exp2f((old - ref) * scale);
      refer(t, ref);
      most[t] = LAZY + OFF;
      l[t] *= keep;
#pragma unroll
      for (int f = 0; f < S::NF; f++) o[t][f] *= keep;
#pragma unroll
      for (int e = 0; e < 8; e++) {
        x[e] = (s[e >> 2][e & 3] - ref) * scale + OFF;
        if (MASKED) x[e] = ((on >> (4 * g + (e & 3) + 16 * (e >> 2))) & 1u) ? x[e] : NEG_INF;
      }
    }
  }
  // The weights, rounded, in B's order.
  XS_DEV u32x4 weights(int t, const float (&x)[8]) {
    float p[8];
#pragma unroll
    for (int e = 0; e < 8; e++) p[e] = __builtin_amdgcn_exp2f(x[e]);
    l[t] += ((p[0] + p[1]) + (p[2] + p[3])) + ((p[4] + p[5]) + (p[6] + p[7]));
    u32x4 b;
#pragma unroll
    for (int i = 0; i < 4; i++) b[i] = pack2(T{}, p[2 * i], p[2 * i + 1]);
    return b;
  }
  // The reference, so that the larger one is the better: l and o carry 2 to the
  // minus reference |scale|, and offset_of more.
  XS_DEV float reference(int t, float scale) const { return scale < 0.0f ? minus(c[t]) : -minus(c[t]); }
};

// After a wave's pass over its keys (passed): whether it was the last.  `mine`: what
// the lane's rows see of the tree, 0 where they count for nothing; marks: 2 MARKS
// words of the lane, 64 apart.
template <typename T, int DP, int RT>
XS_DEV bool finished(Wave<T, DP, RT>& w, int pass, const uint64_t (&mine)[RT], uint32_t* marks) {
  using S = Shape<DP, RT>;
  if (pass == WALK) {
    bool bad = false;
#pragma unroll
    for (int t = 0; t < RT; t++) {
      float z = 0.0f;
#pragma unroll
      for (int f = 0; f < S::NF; f++)
#pragma unroll
        for (int r = 0; r < 4; r++) z = __builtin_fmaf(w.o[t][f][r], 0.0f, z);
      bad |= row_sum(w.l[t]) > 0.0f && z != z && mine[t] != 0;
    }
    if (!__any(bad)) [[likely]] return true;
  } else {
#pragma unroll
    for (int i = 0; i < S::MARKS; i++) {
      auto element = [&](int j) -> f32x4& { return w.o[(8 * i + j / 4) / S::NF][(8 * i + j / 4) % S::NF]; };
      constexpr int LAST = 4 * RT * S::NF;
      if (pass == FINITE) {
        const uint32_t above = marks[64 * i], below = marks[64 * (S::MARKS + i)];
#pragma unroll
        for (int j = 0; j < 32 && 32 * i + j < LAST; j++) element(j)[j % 4] = marked(element(j)[j % 4], above, below, j);
      } else {
        uint32_t m = 0;
#pragma unroll
        for (int j = 31; j >= 0; j--)
          if (32 * i + j < LAST) m = m << 1 | (element(j)[j % 4] > 0.0f ? 1u : 0u);
        marks[64 * (pass == BELOW ? S::MARKS + i : i)] = m;
      }
    }
    if (pass == FINITE) return true;
  }
  w.init();
  return false;
}

// O^T += V^T P^T over a block: v holds 16 bytes of each of the lane's eight
// keys, pf the weights.
template <typename T, int DP, int RT>
XS_DEV void accumulate(Wave<T, DP, RT>& w, const uint32_t (&v)[8][Shape<DP, RT>::VH][Shape<DP, RT>::VE / 2], const u32x4 (&pf)[RT]) {
  using S = Shape<DP, RT>;
#pragma unroll
  for (int h = 0; h < S::VH; h++)
#pragma unroll
    for (int j = 0; j < S::VE; j++) {
      u32x4 a;
#pragma unroll
      for (int i = 0; i < 4; i++)
        a[i] = __builtin_amdgcn_perm(v[2 * i + 1][h][j / 2], v[2 * i][h][j / 2], (j & 1) ? 0x07060302u : 0x05040100u);
#pragma unroll
      for (int t = 0; t < RT; t++) w.o[t][h * S::VE + j] = mfma(T{}, a, pf[t], w.o[t][h * S::VE + j]);
    }
}

// One block of 32 keys from base pointers (elements of one kv head): `limit`
// keys of the source exist, `on` is the lane's mask of the block's keys for
// each row tile, `pass` what is made of the values (passed; masked blocks only).
template <typename T, int DP, int RT, bool EXACT, bool MASKED>
XS_DEV void block(Wave<T, DP, RT>& w, const uint16_t* kp, const uint16_t* vp, int64_t stride, int key0, int limit, int D, float scale,
                  const uint32_t* on, int pass) {
  using S = Shape<DP, RT>;
  const int lane = threadIdx.x & 63, x = lane & 15, g = lane >> 4;
  u32x4 k[2][S::KC];
  const u32x4 zero4 = {0, 0, 0, 0};
#pragma unroll
  for (int t = 0; t < 2; t++) {
    int key = key0 + 16 * t + x;
    if (MASKED) key = min(key, limit - 1);
    const uint16_t* p = kp + key * stride;
#pragma unroll
    for (int c = 0; c < S::KC; c++) {
      const int d = 32 * c + 8 * g;
      if (EXACT) k[t][c] = *(const u32x4*)(p + d);
      else k[t][c] = d < D ? *(const u32x4*)(p + d) : zero4;
    }
  }
  // the values of the lane's eight keys; elements past the head's are those of
  // its last 16 bytes (their products are never stored)
  uint32_t v[8][S::VH][S::VE / 2];
#pragma unroll
  for (int e = 0; e < 8; e++) {
    int key = key0 + 4 * g + (e & 3) + 16 * (e >> 2);
    if (MASKED) key = min(key, limit - 1);
    const uint16_t* p = vp + key * stride;
#pragma unroll
    for (int h = 0; h < S::VH; h++) {
      int d = 128 * h + S::VE * x;
      if (!EXACT) d = min(d, D - S::VE);
      if (S::VE == 8) {
        const u32x4 r = *(const u32x4*)(p + d);
#pragma unroll
        for (int i = 0; i < 4; i++) v[e][h][i] = r[i];
      } else {
        const u32x2 r = *(const u32x2*)(p + d);
#pragma unroll
        for (int i = 0; i < 2; i++) v[e][h][i] = r[i];
      }
    }
  }
  u32x4 pf[RT];
#pragma unroll
  for (int t = 0; t < RT; t++) {
    f32x4 s[2] = {w.start(t), w.start(t)};
#pragma unroll
    for (int c = 0; c < S::KC; c++) {
      s[0] = mfma(T{}, k[0][c], w.q[t][c], s[0]);
      s[1] = mfma(T{}, k[1][c], w.q[t][c], s[1]);
    }
    float xs[8];
    const float top = w.template scaled<MASKED>(s, scale, MASKED ? on[t] : 0u, xs);
    if (__any(w.passes(t, top))) [[unlikely]] {  // (its registers spill before those of the loop)
      const bool far = __any(w.passes(t, top) && w.minus(w.c[t]) != 0.0f);
      if (far) [[unlikely]] {
        s[0] = s[1] = (f32x4){0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
        for (int u = 0; u < 2; u++) {
          int at = lane;
          asm volatile("" : "+v"(at));  // (addressed and read again: kept instead, both would spill)
          int key = key0 + 16 * u + (at & 15);
          if (MASKED) key = min(key, limit - 1);
          const uint16_t* p = kp + key * stride + 8 * (at >> 4);
#pragma unroll
          for (int c = 0; c < S::KC; c++) {
            s[u] = mfma(T{}, EXACT || 32 * c + 8 * (at >> 4) < D ? *(const u32x4*)(p + 32 * c) : zero4, w.q[t][c], s[u]);
            __builtin_amdgcn_sched_barrier(0);  // (one chunk in registers at a time)
          }
        }
      }
      w.template rebase<MASKED>(t, s, far, scale, MASKED ? on[t] : 0u, xs);
    }
    pf[t] = w.weights(t, xs);
  }
  if (MASKED) {
    // Values of keys past the source count for nothing, whatever they hold.
#pragma unroll
    for (int e = 0; e < 8; e++)
#pragma unroll
      for (int h = 0; h < S::VH; h++)
#pragma unroll
        for (int i = 0; i < S::VE / 2; i++)
          if (key0 + 4 * g + (e & 3) + 16 * (e >> 2) >= limit) v[e][h][i] = 0;
    if (pass != WALK) [[unlikely]] {
#pragma unroll
      for (int e = 0; e < 8; e++)
#pragma unroll
        for (int h = 0; h < S::VH; h++)
#pragma unroll
          for (int i = 0; i < S::VE / 2; i++) {
            v[e][h][i] = passed(T{}, v[e][h][i], pass);
            __builtin_amdgcn_sched_barrier(0);
          }
    }
  }
  accumulate(w, v, pf);
}

// A mean is no larger than the largest value, but rounded weights over the sum
// of exact ones may pass it by half a step, which at f16's end would round to an
// infinity (bf16's end is f32's, where the sums overflow first).
XS_DEV float within(Bf16, float x) { return x; }
XS_DEV float within(F16, float x) { return fabsf(x) < -NEG_INF ? fminf(fmaxf(x, -65504.0f), 65504.0f) : x; }
// (Values of another type than the output's may have a mean past its end, and
// weights of more bits than half a step of it leave the rest where it is.)
template <typename T, typename W>
XS_DEV float ended(float x) {
  if constexpr (std::is_same_v<T, W>) return within(T{}, x);
  else return x;
}

// ln of a row's sum of weights, from its reference and l (weights of type W).
template <typename W>
XS_DEV float lse_of(const xs_tree_attend_args& a, float ref, float l) {
  return l == 0.0f ? NEG_INF : __builtin_fmaf(ref, fabsf(a.scale), LN2 * (__builtin_amdgcn_logf(l) - offset_of(W{})));
}

// A result times what its weights are brought to another reference by; nothing,
// whatever it is, where that is 0.
XS_DEV f32x4 times(f32x4 y, float f) { return f == 0.0f ? (f32x4){0.0f, 0.0f, 0.0f, 0.0f} : y * f; }

// Two fragments (2 pair and 2 pair + 1 of half h) of a row tile's result: the
// accumulators over l.  Lane (x, g) holds row x, elements 128 h + VE (4 g + r)
// + 2 pair of each r.
template <typename T, int DP, typename W = T>
XS_DEV void store_pair(const xs_tree_attend_args& a, int G, int b, int kh, int row, int R, int h, int pair, f32x4 o0, f32x4 o1, float ref, float l) {
  constexpr int VE = Shape<DP, 1>::VE;
  const int g = (threadIdx.x & 63) >> 4;
  const int node = min(row, R - 1) / G, head = kh * G + min(row, R - 1) % G;
  if (row >= R) return;
  const float inv = l == 0.0f ? 0.0f : 1.0f / l;
  uint16_t* out = (uint16_t*)a.out + b * a.out_seq_stride + node * a.out_node_stride + head * a.out_head_stride;
#pragma unroll
  for (int r = 0; r < 4; r++) {
    const int d = 128 * h + VE * (4 * g + r) + 2 * pair;
    if (d < a.head_dim) *(uint32_t*)(out + d) = pack2(T{}, ended<T, W>(o0[r] * inv), ended<T, W>(o1[r] * inv));
  }
  if (a.lse && h == 0 && pair == 0 && g == 0)
    a.lse[(b * a.nodes + node) * a.q_heads + head] = lse_of<W>(a, ref, l);
}

// All fragments of half h, VE elements of each r at a time (pairs of 4 bytes
// instead: 19 us of a workgroup's 58 where 32 sequences of 500 slots have 256 rows each).
template <typename T, int DP, int RT>
XS_DEV void store_half(const xs_tree_attend_args& a, int G, int b, int kh, int row, int R, int h, const f32x4 (&o)[Shape<DP, RT>::NF], float ref,
                       float l) {
  constexpr int VE = Shape<DP, 1>::VE;
  const int g = (threadIdx.x & 63) >> 4;
  if (row >= R) return;
  const int node = row / G, head = kh * G + row % G;
  const float inv = l == 0.0f ? 0.0f : 1.0f / l;
  uint16_t* out = (uint16_t*)a.out + b * a.out_seq_stride + node * a.out_node_stride + head * a.out_head_stride;
#pragma unroll
  for (int r = 0; r < 4; r++) {
    const int d = 128 * h + VE * (4 * g + r);
    uint32_t y[VE / 2];
#pragma unroll
    for (int i = 0; i < VE / 2; i++) y[i] = pack2(T{}, within(T{}, o[h * VE + 2 * i][r] * inv), within(T{}, o[h * VE + 2 * i + 1][r] * inv));
    if (d < a.head_dim) {
      if constexpr (VE == 8) *(u32x4*)(out + d) = (u32x4){y[0], y[1], y[2], y[3]};
      else *(u32x2*)(out + d) = (u32x2){y[0], y[1]};
    }
  }
  if (a.lse && h == 0 && g == 0) a.lse[(b * a.nodes + node) * a.q_heads + head] = lse_of<T>(a, ref, l);
}

// Joins the splits of 16 rows and one half of the head: each wave two
// fragments of one of SHARES shares of the splits, so that the loads of many
// splits are in flight at once (a wave that goes through 64 splits one after
// the other takes 100 us), while a few splits take one wave's loads (256 units of four
// tiles in four splits would start 65,536 waves otherwise).
constexpr int SPLITS = 256;     // the most splits of a sequence
constexpr int FEW = 8;          // splits that one share goes through
template <int DP>
constexpr int join_shares(bool few) { return few ? 1 : 16 / (Shape<DP, 1>::VE / 2); }
template <int DP>
constexpr int join_threads(bool few) { return 64 * (Shape<DP, 1>::VE / 2) * join_shares<DP>(few); }

template <typename T, int DP, int RT, bool FEWER>
__global__ __launch_bounds__(join_threads<DP>(FEWER)) void join_kernel(const xs_tree_attend_args a, const Cut cut) {
  using S = Shape<DP, RT>;
  constexpr int PAIRS = S::VE / 2, SHARES = join_shares<DP>(FEWER), WAVES = PAIRS * SHARES;
  constexpr int MOST = FEWER ? FEW : SPLITS, TURNS = (MOST + 4 * WAVES - 1) / (4 * WAVES);
  __shared__ float weight[TURNS * 4 * WAVES][16];
  __shared__ float stat[2][WAVES][16];
  __shared__ f32x4 sum[SHARES][S::VE][64];
  const int lane = threadIdx.x & 63, x = lane & 15, g = lane >> 4;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int h = blockIdx.x % S::VH, t = blockIdx.x / S::VH % RT, tile = blockIdx.x / (S::VH * RT) % cut.tiles;
  const int bh = blockIdx.x / (S::VH * RT * cut.tiles);
  const int kh = bh % (int)a.kv_heads, b = bh / (int)a.kv_heads;
  const Seq sq(a, b);
  const int R = sq.n * cut.G, row0 = (tile * RT + t) * 16;
  const int n = (sq.blocks() + cut.chunk - 1) / cut.chunk;
  if (sq.bad || row0 >= R || n <= 1) return;
  const float* part = cut.part + ((int64_t)bh * cut.nsplit * cut.tiles + tile) * S::PART;
  const int64_t step = (int64_t)cut.tiles * S::PART;
  // the first fragments, on their way while the weights are formed
  constexpr int AHEAD = FEWER ? FEW : 4;
  const int pair = wave % PAIRS, share = wave / PAIRS, f0 = h * S::VE + 2 * pair;
  f32x4 y[AHEAD][2];
#pragma unroll
  for (int i = 0; i < AHEAD; i++) {
    const f32x4* p = (const f32x4*)(part + min(share + SHARES * i, n - 1) * step) + (t * S::NF + f0) * 64 + lane;
    y[i][0] = p[0];
    y[i][1] = p[64];
  }
  // lane (x, g) of wave w takes splits 4 w + g, + 4 WAVES, ... of row x
  float m[TURNS], l[TURNS], top = NEG_INF, all = 0.0f;
#pragma unroll
  for (int i = 0; i < TURNS; i++) {
    const int s = 4 * (WAVES * i + wave) + g;
    const float* p = part + min(s, n - 1) * step + S::STAT + 32 * t + x;
    m[i] = s < n ? p[0] : NEG_INF;
    l[i] = p[16];
    top = fmaxf(top, m[i]);
  }
  top = row_max(top);
  if (g == 0) stat[0][wave][x] = top;
  __syncthreads();
#pragma unroll
  for (int j = 0; j < WAVES; j++) top = fmaxf(top, stat[0][j][x]);
#pragma unroll
  for (int i = 0; i < TURNS; i++) {
    const float f = m[i] == NEG_INF ? 0.0f : __builtin_amdgcn_exp2f((m[i] - top) * fabsf(cut.scale));
    if (m[i] != NEG_INF) all += l[i] * f;
    weight[4 * (WAVES * i + wave) + g][x] = f;
  }
  all = row_sum(all);
  if (g == 0) stat[1][wave][x] = all;
  __syncthreads();
  f32x4 o[2] = {{0.0f, 0.0f, 0.0f, 0.0f}, {0.0f, 0.0f, 0.0f, 0.0f}};
#pragma unroll
  for (int i = 0; i < AHEAD; i++) {
    if (share + SHARES * i >= n) break;
    const float f = weight[share + SHARES * i][x];
    o[0] += times(y[i][0], f);
    o[1] += times(y[i][1], f);
  }
#pragma unroll 8
  for (int s = share + SHARES * AHEAD; s < n; s += SHARES) {
    const f32x4* p = (const f32x4*)(part + s * step) + (t * S::NF + f0) * 64 + lane;
    const float f = weight[s][x];
    o[0] += times(p[0], f);
    o[1] += times(p[64], f);
  }
  all = 0.0f;
#pragma unroll
  for (int j = 0; j < WAVES; j++) all += stat[1][j][x];
  if constexpr (SHARES > 1) {
    sum[share][2 * pair][lane] = o[0];
    sum[share][2 * pair + 1][lane] = o[1];
    __syncthreads();
    if (share != 0) return;
#pragma unroll
    for (int j = 1; j < SHARES; j++) {
      o[0] += sum[j][2 * pair][lane];
      o[1] += sum[j][2 * pair + 1][lane];
    }
  }
  store_pair<T, DP>(a, cut.G, b, kh, row0 + x, R, h, pair, o[0], o[1], top, all);
}

}  // namespace xst
