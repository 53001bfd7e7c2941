// xs_tree.hip -- a tree of drafted tokens over a bounded cache (MI355X, gfx950):
// attention of the tree's nodes, the commit of the accepted path with the
// attention weight it gave, and the eviction of the slots with the least.
//
// Compiled with -ffp-contract=off; fused multiply-adds are written out.

#include <hip/hip_runtime.h>

#include <algorithm>
#include <type_traits>
#include <math.h>
#include <stdint.h>
#include <stdlib.h>

#include "../../include/xsamp.h"
#include "xs_device.h"
#include "xs_host.h"

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
typedef unsigned short u16x2 __attribute__((ext_vector_type(2)));
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
  static constexpr int ODD = STAT + RT * 32;         // then m and l of each row,
  static constexpr int PART = ODD + 4;               // then whether odd values are left out
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
  int odd;         // a node's values held a NaN or an infinity

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
    odd = 0;
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
// each row tile (masked blocks only).
template <typename T, int DP, int RT, bool EXACT, bool MASKED>
XS_DEV void block(Wave<T, DP, RT>& w, const uint16_t* kp, const uint16_t* vp, int64_t stride, int key0, int limit, int D, float scale,
                  const uint32_t* on, bool in_tree) {
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
    // A NaN or an infinity of a node would, through the product (0 times it),
    // reach the rows that do not see the node: it is taken out here, and
    // store_pair adds it to the rows that do.
    u16x2 top = {0, 0};
#pragma unroll
    for (int e = 0; e < 8; e++)
#pragma unroll
      for (int h = 0; h < S::VH; h++)
#pragma unroll
        for (int i = 0; i < S::VE / 2; i++) {
          if (key0 + 4 * g + (e & 3) + 16 * (e >> 2) >= limit) v[e][h][i] = 0;
          top = __builtin_elementwise_max(top, __builtin_bit_cast(u16x2, v[e][h][i] & 0x7FFF7FFFu));
        }
    if (in_tree && __any(max(top[0], top[1]) >= inf_of(T{}))) {
      w.odd = 1;
#pragma unroll
      for (int e = 0; e < 8; e++)
#pragma unroll
        for (int h = 0; h < S::VH; h++)
#pragma unroll
          for (int i = 0; i < S::VE / 2; i++) {
            if ((v[e][h][i] & 0x7FFFu) >= inf_of(T{})) v[e][h][i] &= 0xFFFF0000u;
            if (((v[e][h][i] >> 16) & 0x7FFFu) >= inf_of(T{})) v[e][h][i] &= 0xFFFFu;
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

// ln of a row's sum of weights, from its reference and l.
template <typename T>
XS_DEV float lse_of(const xs_tree_attend_args& a, float ref, float l) {
  return l == 0.0f ? NEG_INF : __builtin_fmaf(ref, fabsf(a.scale), LN2 * (__builtin_amdgcn_logf(l) - offset_of(T{})));
}

// Two fragments (2 pair and 2 pair + 1 of half h) of a row tile's result: the
// accumulators over l.  Lane (x, g) holds row x, elements 128 h + VE (4 g + r)
// + 2 pair of each r.
template <typename T, int DP>
XS_DEV void store_pair(const xs_tree_attend_args& a, int G, int b, int kh, int row, int R, int h, int pair, f32x4 o0, f32x4 o1, float ref, float l, int odd,
                       int n) {
  constexpr int VE = Shape<DP, 1>::VE;
  const int g = (threadIdx.x & 63) >> 4;
  const int node = min(row, R - 1) / G, head = kh * G + min(row, R - 1) % G;
  if (odd) {  // (rare) the NaNs and infinities among the values of the nodes that the row sees, but of an empty row's
    const uint64_t sees = __shfl(ancestors(parent_of(a, b), n), node);
    const uint16_t* v = (const uint16_t*)a.fresh.v + b * a.fresh.seq_stride + kh * a.fresh.head_stride;
#pragma unroll 1
    for (int j = 0; j < n; j++)
#pragma unroll
      for (int r = 0; r < 4; r++) {
        const int d = 128 * h + VE * (4 * g + r) + 2 * pair;
        const uint32_t two = *(const uint32_t*)(v + j * a.fresh.slot_stride + min(d, a.head_dim - 2));
        const uint16_t lo = (uint16_t)two, hi = (uint16_t)(two >> 16);
        if (((sees >> j) & 1ull) && l != 0.0f && (lo & 0x7FFFu) >= inf_of(T{})) o0[r] += T::widen(lo);
        if (((sees >> j) & 1ull) && l != 0.0f && (hi & 0x7FFFu) >= inf_of(T{})) o1[r] += T::widen(hi);
      }
  }
  if (row >= R) return;
  const float inv = l == 0.0f ? 0.0f : 1.0f / l;
  uint16_t* out = (uint16_t*)a.out + b * a.out_seq_stride + node * a.out_node_stride + head * a.out_head_stride;
#pragma unroll
  for (int r = 0; r < 4; r++) {
    const int d = 128 * h + VE * (4 * g + r) + 2 * pair;
    if (d < a.head_dim) *(uint32_t*)(out + d) = pack2(T{}, within(T{}, o0[r] * inv), within(T{}, o1[r] * inv));
  }
  if (a.lse && h == 0 && pair == 0 && g == 0)
    a.lse[(b * a.nodes + node) * a.q_heads + head] = lse_of<T>(a, ref, l);
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

// grid: groups of eight (sequence, kv head, split), each group's row tiles on
// one XCD (workgroup index mod 8), which then reads their keys once.
template <typename T, int DP, int RT, bool EXACT>
__global__ __launch_bounds__(64 * NW, DP * RT <= 64 ? 4 : DP * RT <= 128 ? 3 : DP * RT <= 256 ? 2 : 1) void attend_kernel(const xs_tree_attend_args a, const Cut cut) {
  using S = Shape<DP, RT>;
  __shared__ float stat[NW][RT][2][16];
  __shared__ f32x4 sum[NW][RT][S::NF][64];
  __shared__ int odds[NW];
  const int lane = threadIdx.x & 63, x = lane & 15, g = lane >> 4;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int tile = (blockIdx.x >> 3) % cut.tiles;
  const int group = ((blockIdx.x >> 3) / cut.tiles) * 8 + (blockIdx.x & 7);
  if (group >= cut.groups) return;
  const int bh = group / cut.nsplit, split = turned(group % cut.nsplit, bh, cut.nsplit);
  const int kh = bh % (int)a.kv_heads, b = bh / (int)a.kv_heads;
  // (the rows that the launch is sized for: their loads need not wait for the
  // sequence's own sizes)
  const int row0 = tile * RT * 16, parent = parent_of(a, b);
  Wave<T, DP, RT> w;
  w.init();
#pragma unroll
  for (int t = 0; t < RT; t++) {
    const int row = row0 + 16 * t + x;
    const bool in = row < (int)a.nodes * cut.G;
    const int node = in ? row / cut.G : 0, head = kh * cut.G + (in ? row % cut.G : 0);
    const uint16_t* p = (const uint16_t*)a.q + b * a.q_seq_stride + node * a.q_node_stride + head * a.q_head_stride;
#pragma unroll
    for (int c = 0; c < S::KC; c++) {
      const int d = 32 * c + 8 * g;
      w.q[t][c] = in && (EXACT || d < a.head_dim) ? *(const u32x4*)(p + d) : (u32x4){0, 0, 0, 0};
    }
  }
  const Seq sq(a, b);
  if (split == 0 && tile == 0 && kh == 0 && threadIdx.x == 0) a.seq_status[b] = sq.bad ? XS_ROW_BAD_PARAM : XS_ROW_OK;
  if (sq.bad) return;
  const int R = sq.n * cut.G;
  const int total = sq.blocks(), cached = (sq.len + KB - 1) / KB;
  const int first = split * cut.chunk, last = min(first + cut.chunk, total);
  if (row0 >= R || first >= total) return;

  const uint16_t* ck = (const uint16_t*)a.cache.k + b * a.cache.seq_stride + kh * a.cache.head_stride;
  const uint16_t* cv = (const uint16_t*)a.cache.v + b * a.cache.seq_stride + kh * a.cache.head_stride;
  int i = first + wave;
  // whole blocks of the cache
  for (; i < last && (i + 1) * KB <= sq.len; i += NW)
    block<T, DP, RT, EXACT, false>(w, ck, cv, a.cache.slot_stride, i * KB, sq.len, a.head_dim, cut.scale, nullptr, false);
  // its last one, and the tree's
  const uint64_t sees = ancestors(parent, sq.n);
  uint64_t mine[RT];  // what the lane's rows see of the tree
#pragma unroll
  for (int t = 0; t < RT; t++) {
    const int row = row0 + 16 * t + x;
    mine[t] = __shfl(sees, min(row / cut.G, 63));
    if (row >= R) mine[t] = 0;
  }
#pragma unroll 1
  for (; i < last; i += NW) {
    const bool in_tree = i >= cached;
    const int key0 = (in_tree ? i - cached : i) * KB, limit = in_tree ? sq.n : sq.len;
    const xs_kv& kv = in_tree ? a.fresh : a.cache;
    const int64_t at = b * kv.seq_stride + kh * kv.head_stride;
    uint32_t on[RT];
#pragma unroll
    for (int t = 0; t < RT; t++) on[t] = in_tree ? (uint32_t)(mine[t] >> key0) : (1u << (sq.len - key0)) - 1u;
    block<T, DP, RT, EXACT, true>(w, (const uint16_t*)kv.k + at, (const uint16_t*)kv.v + at, kv.slot_stride, key0, limit, a.head_dim,
                                  cut.scale, on, in_tree);
  }

  // the waves' sums, brought to one reference; rows that see nothing of the
  // tree see nothing of the cache either
  float ref[RT];
  if (lane == 0) odds[wave] = w.odd;
#pragma unroll
  for (int t = 0; t < RT; t++) {
    w.l[t] = row_sum(w.l[t]);
    if (mine[t] == 0) w.l[t] = 0.0f;
    ref[t] = w.l[t] == 0.0f ? NEG_INF : w.reference(t, cut.scale);
    if (g == 0) {
      stat[wave][t][0][x] = ref[t];
      stat[wave][t][1][x] = w.l[t];
    }
  }
  __syncthreads();
  const float mag = fabsf(cut.scale);
#pragma unroll
  for (int t = 0; t < RT; t++) {
    float top = NEG_INF;
#pragma unroll
    for (int j = 0; j < NW; j++) top = fmaxf(top, stat[j][t][0][x]);
    const float f = ref[t] == NEG_INF ? 0.0f : __builtin_amdgcn_exp2f((ref[t] - top) * mag);
#pragma unroll
    for (int k = 0; k < S::NF; k++) sum[wave][t][k][lane] = ref[t] == NEG_INF ? (f32x4){0.0f, 0.0f, 0.0f, 0.0f} : w.o[t][k] * f;
  }
  __syncthreads();
  // a wave takes every fourth pair of fragments
  constexpr int PAIRS = S::VE / 2;
  const bool whole = first == 0 && last == total;
  const int odd = odds[0] | odds[1] | odds[2] | odds[3];
  float* part = cut.part + (((int64_t)bh * cut.nsplit + split) * cut.tiles + tile) * S::PART;
#pragma unroll 1
  for (int u = wave; u < RT * S::VH * PAIRS; u += NW) {
    const int pair = u % PAIRS, h = u / PAIRS % S::VH, t = u / (PAIRS * S::VH), f0 = h * S::VE + 2 * pair;
    float top = NEG_INF, all = 0.0f;
#pragma unroll
    for (int j = 0; j < NW; j++) top = fmaxf(top, stat[j][t][0][x]);
    f32x4 o[2] = {{0.0f, 0.0f, 0.0f, 0.0f}, {0.0f, 0.0f, 0.0f, 0.0f}};
#pragma unroll
    for (int j = 0; j < NW; j++) {
      const float mj = stat[j][t][0][x];
      all += mj == NEG_INF ? 0.0f : stat[j][t][1][x] * __builtin_amdgcn_exp2f((mj - top) * mag);
      o[0] += sum[j][t][f0][lane];
      o[1] += sum[j][t][f0 + 1][lane];
    }
    if (whole) {
      store_pair<T, DP>(a, cut.G, b, kh, row0 + 16 * t + x, R, h, pair, o[0], o[1], top, all, odd, sq.n);
    } else {
      f32x4* p = (f32x4*)part + (t * S::NF + f0) * 64 + lane;
      p[0] = o[0];
      p[64] = o[1];
      if (h == 0 && pair == 0 && g == 0) {
        part[S::STAT + 32 * t + x] = top;
        part[S::STAT + 32 * t + 16 + x] = all;
        part[S::ODD] = odd ? 1.0f : 0.0f;
      }
    }
  }
}

// Many rows (more than one wave's): the four waves of a workgroup take RT row
// tiles each and share the keys, which come through LDS in stages of SK, three
// buffers deep: while one is read, the next is complete and the one after it
// on its way from memory in registers.  Per block of 32 keys a wave does RT * (2 DP/32 + DP/16)
// matrix instructions of 16 cycles and about as many cycles of vector work (8
// exponentials a tile of 16 cycles each, then scaling, maxima, sums, packing,
// the byte permutes), so the two are laid side by side: the next block's
// scores beside this block's exponentials, this block's products beside the next
// block's maxima.  Reading the keys from L2 in every wave instead, 64 bytes a
// cycle and CU, takes as long as the matrix instructions, and not beside them:
// 8 sequences of 64 nodes over 32,768 slots (256 rows of 8 kv heads) 520 us,
// so 354 to 366 (751 to 776 TFLOP/s, of the 1,291 of a large library product).
template <int DP>
struct Stage {
  static constexpr int SK = DP > 128 ? 32 : 64;
  static constexpr int CH = DP / 8;                    // 16-byte chunks of a row
  static constexpr int PER = SK * CH / (64 * NW);      // chunks a thread moves, of k and of v
  static constexpr int TURN = CH < 16 ? CH - 1 : 15;   // k's chunks are turned by the row, so that 16 rows' reads meet 16 banks
};

template <typename T, int DP, int RT, bool EXACT>
__global__ __launch_bounds__(64 * NW, 1) void attend_wide_kernel(const xs_tree_attend_args a, const Cut cut) {
  using S = Shape<DP, RT>;
  using G = Stage<DP>;
  __shared__ u32x4 lk[3][G::SK * G::CH];
  __shared__ u32x4 lv[3][G::SK * G::CH];
  const int lane = threadIdx.x & 63, x = lane & 15, g = lane >> 4;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int wgs = cut.tiles / NW;  // workgroups of a split: NW tiles each
  const int wg = (blockIdx.x >> 3) % wgs, tile = wg * NW + wave;
  const int group = ((blockIdx.x >> 3) / wgs) * 8 + (blockIdx.x & 7);
  if (group >= cut.groups) return;
  const int bh = group / cut.nsplit, split = turned(group % cut.nsplit, bh, cut.nsplit);
  const int kh = bh % (int)a.kv_heads, b = bh / (int)a.kv_heads;
  const int row0 = tile * RT * 16, parent = parent_of(a, b);
  const Seq sq(a, b);
  if (split == 0 && wg == 0 && kh == 0 && threadIdx.x == 0) a.seq_status[b] = sq.bad ? XS_ROW_BAD_PARAM : XS_ROW_OK;
  if (sq.bad) return;
  const int R = sq.n * cut.G;
  const int total = sq.blocks(), cached = (sq.len + KB - 1) / KB;
  const int first = split * cut.chunk, last = min(first + cut.chunk, total);
  if (wg * NW * RT * 16 >= R || first >= total) return;

  Wave<T, DP, RT> w;
  w.init();
#pragma unroll
  for (int t = 0; t < RT; t++) {
    const int row = row0 + 16 * t + x;
    const bool in = row < R;
    const int node = in ? row / cut.G : 0, head = kh * cut.G + (in ? row % cut.G : 0);
    const uint16_t* p = (const uint16_t*)a.q + b * a.q_seq_stride + node * a.q_node_stride + head * a.q_head_stride;
#pragma unroll
    for (int c = 0; c < S::KC; c++) {
      const int d = 32 * c + 8 * g;
      w.q[t][c] = in && (EXACT || d < a.head_dim) ? *(const u32x4*)(p + d) : (u32x4){0, 0, 0, 0};
    }
  }

  // whole stages of the cache
  constexpr int SB = G::SK / KB;
  const int stages = max(0, min(last, sq.len / KB) - first) / SB;
  const int64_t c0 = b * a.cache.seq_stride + kh * a.cache.head_stride;
  u32x4 rk[G::PER], rv[G::PER];
  auto fetch = [&](int s) {
#pragma unroll
    for (int i = 0; i < G::PER; i++) {
      const int q = i * 64 * NW + threadIdx.x, row = q / G::CH, ch = q % G::CH;
      const int64_t at = c0 + (int64_t)(first * KB + s * G::SK + row) * a.cache.slot_stride + ch * 8;
      const bool in = EXACT || ch * 8 < a.head_dim;
      rk[i] = in ? *(const u32x4*)((const uint16_t*)a.cache.k + at) : (u32x4){0, 0, 0, 0};
      rv[i] = in ? *(const u32x4*)((const uint16_t*)a.cache.v + at) : (u32x4){0, 0, 0, 0};
    }
  };
  auto put = [&](int s) {
#pragma unroll
    for (int i = 0; i < G::PER; i++) {
      const int q = i * 64 * NW + threadIdx.x, row = q / G::CH, ch = q % G::CH;
      lk[s % 3][row * G::CH + (ch ^ (row & G::TURN))] = rk[i];
      lv[s % 3][q] = rv[i];
    }
  };
  // 16 keys' chunk c of block j, counted in blocks from `first`
  auto key = [&](int j, int u, int c) {
    const int row = (j % SB) * KB + 16 * u + x;
    return lk[(j / SB) % 3][row * G::CH + ((4 * c + g) ^ (row & G::TURN))];
  };
  // the scores of block j
  auto scores = [&](int j, f32x4 (&s)[RT][2]) {
#pragma unroll
    for (int t = 0; t < RT; t++) s[t][0] = s[t][1] = w.start(t);
#pragma unroll
    for (int c = 0; c < S::KC; c++) {
      const u32x4 f[2] = {key(j, 0, c), key(j, 1, c)};
#pragma unroll
      for (int t = 0; t < RT; t++) {
        s[t][0] = mfma(T{}, f[0], w.q[t][c], s[t][0]);
        s[t][1] = mfma(T{}, f[1], w.q[t][c], s[t][1]);
      }
    }
  };
  if (stages > 0) {
    fetch(0);
    put(0);
    __syncthreads();
    if (stages > 1) fetch(1);
    float xs[RT][8];
    auto prepare = [&](const f32x4 (&s)[RT][2]) {
      float top[RT];
      bool move = false;
#pragma unroll
      for (int t = 0; t < RT; t++) {
        top[t] = w.template scaled<false>(s[t], cut.scale, 0u, xs[t]);
        move = move | w.passes(t, top[t]);
      }
      return move;
    };
    auto settle = [&](int j) {
#pragma unroll
      for (int t = 0; t < RT; t++) {
        f32x4 s[2] = {{0.0f, 0.0f, 0.0f, 0.0f}, {0.0f, 0.0f, 0.0f, 0.0f}};
#pragma unroll
        for (int c = 0; c < S::KC; c++) {
          s[0] = mfma(T{}, key(j, 0, c), w.q[t][c], s[0]);
          s[1] = mfma(T{}, key(j, 1, c), w.q[t][c], s[1]);
        }
        w.template rebase<false>(t, s, true, cut.scale, 0u, xs[t]);
        // (one tile in registers at a time: else the loop spills, 457 us for 365
        // where 8 sequences of 64 nodes see 32,768 slots)
        __builtin_amdgcn_sched_barrier(0);
      }
    };
    {
      f32x4 s[RT][2];
      scores(0, s);
      if (__any(prepare(s))) settle(0);
    }
    const int blocks = stages * SB;
#pragma unroll 1
    for (int st = 0; st < stages; st++) {
#pragma unroll
      for (int sub = 0; sub < SB; sub++) {
        const int j = st * SB + sub;
        if (sub == SB - 1 && st + 1 < stages) {
          put(st + 1);
          __syncthreads();
          if (st + 2 < stages) fetch(st + 2);
        }
        const bool more = j + 1 < blocks;
        f32x4 s[RT][2];
        u32x4 pf[RT];
        scores(more ? j + 1 : j, s);
#pragma unroll
        for (int t = 0; t < RT; t++) pf[t] = w.weights(t, xs[t]);
        uint32_t v[8][S::VH][S::VE / 2];
        const uint32_t* base = (const uint32_t*)lv[st % 3];
#pragma unroll
        for (int e = 0; e < 8; e++) {
          const int row = sub * KB + 4 * g + (e & 3) + 16 * (e >> 2);
#pragma unroll
          for (int h = 0; h < S::VH; h++)
#pragma unroll
            for (int i = 0; i < S::VE / 2; i++) v[e][h][i] = base[row * G::CH * 4 + 64 * h + S::VE / 2 * x + i];
        }
        accumulate(w, v, pf);
        const bool move = prepare(s);
        if (more && __any(move)) [[unlikely]] settle(j + 1);
      }
    }
  }

  // the rest: part of a stage, the last block of the cache, the tree
  const uint64_t sees = ancestors(parent, sq.n);
  uint64_t mine[RT];  // what the lane's rows see of the tree
#pragma unroll
  for (int t = 0; t < RT; t++) {
    const int row = row0 + 16 * t + x;
    mine[t] = __shfl(sees, min(row / cut.G, 63));
    if (row >= R) mine[t] = 0;
  }
  if (row0 >= R) return;
#pragma unroll 1
  for (int i = first + stages * SB; i < last; i++) {
    const bool in_tree = i >= cached;
    const int key0 = (in_tree ? i - cached : i) * KB, limit = in_tree ? sq.n : sq.len;
    const xs_kv& kv = in_tree ? a.fresh : a.cache;
    const int64_t at = b * kv.seq_stride + kh * kv.head_stride;
    uint32_t on[RT];
#pragma unroll
    for (int t = 0; t < RT; t++)
      on[t] = in_tree ? (uint32_t)(mine[t] >> key0) : sq.len - key0 >= KB ? ~0u : (1u << (sq.len - key0)) - 1u;
    block<T, DP, RT, EXACT, true>(w, (const uint16_t*)kv.k + at, (const uint16_t*)kv.v + at, kv.slot_stride, key0, limit, a.head_dim,
                                  cut.scale, on, in_tree);
  }
  constexpr int PAIRS = S::VE / 2;
  const bool whole = first == 0 && last == total;
  float* part = cut.part + (((int64_t)bh * cut.nsplit + split) * cut.tiles + tile) * S::PART;
#pragma unroll
  for (int t = 0; t < RT; t++) {
    float l = row_sum(w.l[t]);
    if (mine[t] == 0) l = 0.0f;
    const float ref = l == 0.0f ? NEG_INF : w.reference(t, cut.scale);
#pragma unroll
    for (int f = 0; f < S::NF; f++)
      if (l == 0.0f) w.o[t][f] = (f32x4){0.0f, 0.0f, 0.0f, 0.0f};
    if (whole && !w.odd) {
#pragma unroll
      for (int h = 0; h < S::VH; h++) store_half<T, DP, RT>(a, cut.G, b, kh, row0 + 16 * t + x, R, h, w.o[t], ref, l);
    } else if (whole) {
#pragma unroll
      for (int h = 0; h < S::VH; h++)
#pragma unroll
        for (int pair = 0; pair < PAIRS; pair++)
          store_pair<T, DP>(a, cut.G, b, kh, row0 + 16 * t + x, R, h, pair, w.o[t][h * S::VE + 2 * pair], w.o[t][h * S::VE + 2 * pair + 1], ref,
                            l, w.odd, sq.n);
    } else {
#pragma unroll
      for (int f = 0; f < S::NF; f++) ((f32x4*)part)[(t * S::NF + f) * 64 + lane] = w.o[t][f];
      if (g == 0) {
        part[S::STAT + 32 * t + x] = ref;
        part[S::STAT + 32 * t + 16 + x] = l;
        part[S::ODD] = w.odd ? 1.0f : 0.0f;
      }
    }
  }
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
  __shared__ int odd;
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
  if (threadIdx.x == 0) odd = 0;
  __syncthreads();
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
    if (p[S::ODD - S::STAT - 32 * t - x] != 0.0f) odd = 1;  // (any of them)
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
    o[0] += y[i][0] * f;
    o[1] += y[i][1] * f;
  }
#pragma unroll 8
  for (int s = share + SHARES * AHEAD; s < n; s += SHARES) {
    const f32x4* p = (const f32x4*)(part + s * step) + (t * S::NF + f0) * 64 + lane;
    const float f = weight[s][x];
    o[0] += p[0] * f;
    o[1] += p[64] * f;
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
  store_pair<T, DP>(a, cut.G, b, kh, row0 + x, R, h, pair, o[0], o[1], top, all, odd, sq.n);
}

// A sequence's path in lanes [0, m) of the calling wave, or its error.
XS_DEV int read_path(const xs_cache_commit_args& a, int b, int len, int64_t limit, int* node, int* m) {
  const int lane = threadIdx.x & 63;
  *m = a.n_path[b];
  *node = -1;
  if (len < 0 || len > limit || *m < 0 || *m > a.nodes) return XS_ROW_BAD_PARAM;
  if (lane < *m) *node = a.path[b * a.path_ld + lane];
  if (__ballot(lane < *m && (*node < 0 || *node >= a.nodes))) return XS_ROW_BAD_PARAM;
  return (int64_t)len + *m > a.capacity ? XS_ROW_CACHE_FULL : XS_ROW_OK;
}

// ---------------------------------------------------------------------------
// Commit.
//
// Weights: S = Q K^T with A = Q (m a row, path rank * group + q head) and B = K
// (n a key), so that a lane holds one key and its sum over the rows is a sum over
// registers and row tiles, and over lane groups once.  A wave keeps RT row tiles
// in registers and walks its share of the keys in blocks of 32; more rows than that take further passes
// over the share, which add to what the same lanes wrote.  Bound by the one
// read of the keys.  A head's first workgroup weighs the path's own keys (a
// row sees the ranks up to its own), with two waves, and appends the path with the others.

template <int DP, int RT>
struct Rows {
  u32x4 q[RT][DP / 32];
  float lse[RT][4];  // of rows 4 g + r
  uint32_t on;       // bit 4 t + r: the lane's row 4 g + r of tile t counts
};

// Rows row0 .. row0 + 16 RT of the path (R in all).
template <int DP, int RT, bool EXACT>
XS_DEV void load_rows(const xs_cache_commit_args& a, Rows<DP, RT>& w, int b, int kh, int G, int node, int row0, int R) {
  const int lane = threadIdx.x & 63, x = lane & 15, g = lane >> 4;
  w.on = 0;
#pragma unroll
  for (int t = 0; t < RT; t++) {
    if (row0 + 16 * t >= R) break;
    const int row = row0 + 16 * t + x;
    const int rank = min(row, R - 1) / G, head = kh * G + min(row, R - 1) % G;
    const int i = __shfl(node, rank);
    const uint16_t* p = (const uint16_t*)a.q + b * a.q_seq_stride + i * a.q_node_stride + head * a.q_head_stride;
#pragma unroll
    for (int c = 0; c < DP / 32; c++) {
      const int d = 32 * c + 8 * g;
      w.q[t][c] = EXACT || d < a.head_dim ? *(const u32x4*)(p + d) : (u32x4){0, 0, 0, 0};
    }
#pragma unroll
    for (int r = 0; r < 4; r++) {
      const int mine = row0 + 16 * t + 4 * g + r, m = min(mine, R - 1);
      const int k = __shfl(node, m / G);
      const float v = a.lse[(b * a.nodes + k) * a.q_heads + kh * G + m % G];
      if (mine < R && v != NEG_INF) w.on |= 1u << (4 * t + r);
      w.lse[t][r] = v;
    }
  }
}

// Two tiles of 16 keys.
template <int DP, bool EXACT>
XS_DEV void load_keys(const uint16_t* const (&kp)[2], int D, u32x4 (&k)[2][DP / 32]) {
  const int g = (threadIdx.x & 63) >> 4;
#pragma unroll
  for (int u = 0; u < 2; u++)
#pragma unroll
    for (int c = 0; c < DP / 32; c++) {
      const int d = 32 * c + 8 * g;
      k[u][c] = EXACT || d < D ? *(const u32x4*)(kp[u] + d) : (u32x4){0, 0, 0, 0};
    }
}

// The weight that the rows give to two tiles of keys, in every lane group.
// TAIL: keys are path ranks, seen from their own rank on.
template <typename T, int DP, int RT, bool TAIL>
XS_DEV void weigh(const Rows<DP, RT>& w, const u32x4 (&k)[2][DP / 32], float scale, int row0, int R, int G, int rank0, float (&sum)[2]) {
  const int lane = threadIdx.x & 63, x = lane & 15, g = lane >> 4;
  sum[0] = sum[1] = 0.0f;
#pragma unroll
  for (int t = 0; t < RT; t++) {
    if (row0 + 16 * t >= R) break;
    f32x4 s[2] = {{0.0f, 0.0f, 0.0f, 0.0f}, {0.0f, 0.0f, 0.0f, 0.0f}};
#pragma unroll
    for (int c = 0; c < DP / 32; c++) {
      s[0] = mfma(T{}, w.q[t][c], k[0][c], s[0]);
      s[1] = mfma(T{}, w.q[t][c], k[1][c], s[1]);
    }
#pragma unroll
    for (int r = 0; r < 4; r++)
#pragma unroll
      for (int u = 0; u < 2; u++) {
        // The difference of two large terms, rounded once; then to base 2.  No
        // slot of the cache weighs more than 1; where the two are huge, lse's
        // own rounding may leave more, and exp of that an infinity.  A row of
        // a path that is no chain may weigh a fresh key more: there only what
        // rounding leaves (some steps of lse, 2^-24 of it each) is cut.
        float y = __builtin_fmaf(s[u][r], scale, -w.lse[t][r]);
        if (y > 0.0f && (!TAIL || y <= fabsf(w.lse[t][r]) * 0x1p-20f)) y = 0.0f;
        const float p = __builtin_amdgcn_exp2f(y * LOG2E);
        bool on = (w.on >> (4 * t + r)) & 1u;
        if (TAIL) on = on && (row0 + 16 * t + 4 * g + r) / G >= rank0 + 16 * u + x;
        sum[u] += on ? p : 0.0f;
      }
  }
  sum[0] = row_sum(sum[0]);
  sum[1] = row_sum(sum[1]);
}

template <typename T, int DP, int RT, bool EXACT>
__global__ __launch_bounds__(64 * NW, DP * RT <= 256 ? 3 : 2) void commit_kernel(const xs_cache_commit_args a, int shares, int share) {
  const int lane = threadIdx.x & 63, x = lane & 15, g = lane >> 4;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int bh = blockIdx.x / shares, blk = turned(blockIdx.x % shares, bh, shares);
  const int kh = bh % (int)a.kv_heads, b = bh / (int)a.kv_heads;
  const bool tail = blk == 0;
  const int len = a.len[b], G = (int)(a.q_heads / a.kv_heads);
  if (!tail && (blk - 1) * NW * share * KB >= len) return;
  int node, m;
  const int st = read_path(a, b, len, a.max_len ? a.max_len : a.capacity, &node, &m);
  if (tail && kh == 0 && threadIdx.x == 0) {
    a.seq_status[b] = st;
    a.new_len[b] = st == XS_ROW_OK ? len + m : len;
    if (a.pos) a.new_next_pos[b] = a.next_pos[b] + (st == XS_ROW_OK ? m : 0);
  }
  if (st != XS_ROW_OK) return;
  const int64_t slots = (b * a.kv_heads + kh) * a.slot_ld;
  const int R = m * G;
  Rows<DP, RT> w;
  if (!tail) {
    const uint16_t* ck = (const uint16_t*)a.cache.k + b * a.cache.seq_stride + kh * a.cache.head_stride;
    const int end = min(blk * NW * share * KB, len);
    int row0 = 0;
    do {
      load_rows<DP, RT, EXACT>(a, w, b, kh, G, node, row0, R);
      const float* from = row0 == 0 ? a.mass : a.new_mass;
      auto load = [&](int key0, u32x4 (&k)[2][DP / 32], float& old) {
        const uint16_t* kp[2];
#pragma unroll
        for (int u = 0; u < 2; u++) kp[u] = ck + min(key0 + 16 * u + x, len - 1) * a.cache.slot_stride;
        load_keys<DP, EXACT>(kp, a.head_dim, k);
        const int slot = key0 + 16 * (g & 1) + x;
        old = g < 2 && slot < end ? from[slots + slot] : 0.0f;
      };
      int key0 = ((blk - 1) * NW * share + wave) * KB;
      u32x4 k[2][DP / 32];
      float old;
      if (key0 < end) load(key0, k, old);
      while (key0 < end) {
        const int next = key0 + NW * KB;
        float sum[2];
        weigh<T, DP, RT, false>(w, k, a.scale, row0, R, G, 0, sum);
        const int slot = key0 + 16 * (g & 1) + x;
        if (g < 2 && slot < end) a.new_mass[slots + slot] = old + ((g & 1) ? sum[1] : sum[0]);
        if (next < end) load(next, k, old);
        key0 = next;
      }
      row0 += 16 * RT;
    } while (row0 < R);
    return;
  }
  if (a.q && wave * KB < m) {  // (two waves for at most 64 ranks)
    const uint16_t* kp[2];
    const uint16_t* fk = (const uint16_t*)a.fresh.k + b * a.fresh.seq_stride + kh * a.fresh.head_stride;
#pragma unroll
    for (int u = 0; u < 2; u++) kp[u] = fk + __shfl(node, min(wave * KB + 16 * u + x, m - 1)) * a.fresh.slot_stride;
    u32x4 k[2][DP / 32];
    load_keys<DP, EXACT>(kp, a.head_dim, k);
    float all[2] = {0.0f, 0.0f};
    for (int row0 = 0; row0 < R; row0 += 16 * RT) {
      load_rows<DP, RT, EXACT>(a, w, b, kh, G, node, row0, R);
      float sum[2];
      weigh<T, DP, RT, true>(w, k, a.scale, row0, R, G, wave * KB, sum);
      all[0] += sum[0];
      all[1] += sum[1];
    }
    const int rank = wave * KB + 16 * (g & 1) + x;
    if (g < 2 && rank < m) a.new_mass[slots + len + rank] = (g & 1) ? all[1] : all[0];
  }
  if (a.pos && (int)threadIdx.x < m) a.pos[slots + len + threadIdx.x] = a.next_pos[b] + threadIdx.x;
  const int parts = a.head_dim / 8;
  const int64_t from = b * a.fresh.seq_stride + kh * a.fresh.head_stride, to = b * a.cache.seq_stride + kh * a.cache.head_stride;
  const int skip = a.q ? 128 : 0;  // (the weighing waves' threads)
  if ((int)threadIdx.x < skip) return;
  for (int j = threadIdx.x - skip; j - lane < m * parts; j += 64 * NW - skip) {  // (whole waves: the path is in their lanes)
    const int r = min(j / parts, m - 1), d = j % parts * 8;
    const int64_t f = from + __shfl(node, r) * a.fresh.slot_stride + d, s = to + (len + r) * a.cache.slot_stride + d;
    if (j >= m * parts) continue;
    *(u32x4*)((uint16_t*)a.cache.k + s) = *(const u32x4*)((const uint16_t*)a.fresh.k + f);
    *(u32x4*)((uint16_t*)a.cache.v + s) = *(const u32x4*)((const uint16_t*)a.fresh.v + f);
  }
}

// ---------------------------------------------------------------------------
// Eviction.
//
// One workgroup per (sequence, kv head) finds the `keep`-th of the slots'
// weights (weight_word) by counting digits of 11 bits from the top, each pass
// over the slots whose digits so far are the chosen ones, until a digit's
// slots are exactly those still needed, or few enough (LIST) to compare each
// with each; equal weights go on into their positions, and those into the slots.  Prefix
// counts pair the i-th free slot below `keep` with the i-th kept one past it.
// Only these move: `keep` of `keep` + a few slots moves a few rows, where
// keeping the slots in order would move nearly all.

constexpr int EB = 1024;         // threads
constexpr int EW = EB / 64;      // waves
constexpr int DIGIT = 11;

// A slot's place in the order of xs_cache_evict, larger first, in two words:
// the held slots above all others, then the weights (the bits of an f32 put in
// order; NaN below -inf), and among equal ones the lower position first.
XS_DEV uint32_t weight_word(float mass, bool held) {
  const uint32_t u = __float_as_uint(mass + 0.0f);  // (-0 as 0)
  const uint32_t w = mass != mass ? 0u : (u & 0x80000000u ? ~u : u | 0x80000000u);
  return held ? 0xFFFFFFFFu : w;
}
XS_DEV uint32_t position_word(int pos) { return ~((uint32_t)pos ^ 0x80000000u); }

struct EvictWork {
  uint64_t* kept;   // [heads, words] bitmap of the kept slots
  int32_t* free_;   // [heads, pairs] freed slots, ascending
  int32_t* filler;  // [heads, pairs] the slots that move there, ascending
  int32_t* moves;   // [heads]
  int64_t words, pairs;
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
XS_DEV uint64_t wave_scan(uint64_t v) {
  const int lane = threadIdx.x & 63;
#pragma unroll
  for (int o = 1; o < 64; o <<= 1) {
    const uint64_t y = __shfl_up(v, o);
    if (lane >= o) v += y;
  }
  return v;
}

// Exclusive prefix sums over the workgroup, and the total.  Two barriers.
template <typename U>
XS_DEV U block_scan(U v, U* lds, U* total) {
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const U run = wave_scan(v);
  if (lane == 63) lds[wave] = run;
  __syncthreads();
  U before = 0, all = 0;
#pragma unroll
  for (int i = 0; i < EW; i++) {
    const U y = lds[i];
    if (i < wave) before += y;
    all += y;
  }
  __syncthreads();
  *total = all;
  return before + run - v;
}

// Copies row `from` to row `to` of one kv head's k and v, 16 bytes a lane.
XS_DEV void move_part(const xs_cache_evict_args& a, int64_t head, int from, int to, int d) {
  const int64_t f = head + from * a.cache.slot_stride + d, t = head + to * a.cache.slot_stride + d;
  *(u32x4*)((uint16_t*)a.cache.k + t) = *(const u32x4*)((const uint16_t*)a.cache.k + f);
  *(u32x4*)((uint16_t*)a.cache.v + t) = *(const u32x4*)((const uint16_t*)a.cache.v + f);
}

constexpr int REP = 4;     // copies of the counts, by the lane: weights crowd into few digits
constexpr int LIST = 256;  // slots that are ranked by comparing each with each
constexpr int NEAR = 128;  // moves that a head's own workgroup makes; more are left to evict_rows_kernel

// A slot's place: weight word, position word, and the slot itself, the first
// two larger first.  Kept is what lies at or before the cutoff (whole: what
// lies before its weight word).
struct Cutoff {
  uint32_t weight, position;
  int slot;
  bool whole;
  XS_DEV bool keeps(uint32_t w, int s, const int32_t* pos) const {
    if (whole || w != weight) return w > weight;
    const uint32_t p = position_word(pos[s]);  // (few slots)
    return p != position ? p > position : s <= slot;
  }
};

struct SelectLds {
  uint32_t hist[REP << DIGIT];
  uint32_t scan[EW];
  uint64_t place[LIST];  // weight and position words
  int slot[LIST];
  int listed;
  int found[4];  // the digit, the slots still needed of it, whether that is all of it, how many it has
  Cutoff cutoff;
};

// The cutoff that keeps `need` of len slots (need < len).  each(f) calls
// f(slot, weight word) for every slot, whole waves at a time (slots past len
// among them).  bits, if not null: a bitmap over the slots, empty, where the
// slots that are kept beside those of the cutoff are set.
// again(f) does the same from memory, for the words after the weight's.
template <typename Each, typename Again>
XS_DEV Cutoff find_cutoff(SelectLds& lds, int len, int need, const int32_t* pos, uint32_t* bits, Each each, Again again) {
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
  u32x4* const own = (u32x4*)lds.hist + 2 * ((1 << (DIGIT - 1)) - 1 - tid);  // thread i: the i-th pair of digits from the top
  static_assert(REP == 4, "the copies of a count fill a vector");
  own[0] = own[1] = (u32x4){0, 0, 0, 0};
  if (tid == 0) lds.listed = 0;
  __syncthreads();
  // The words of a slot's place, from the weight's (L = 0) to the slot's (2).
  // The words before L are `known`, and of that one the bits from `shift` on
  // are `prefix`.
  uint32_t known[2] = {0, 0}, prefix = 0;
  int shift = 32;
  auto word = [&](auto L, int s, uint32_t k) {
    if constexpr (L == 0) return k;
    else if constexpr (L == 1) return position_word(pos[s]);
    else return ~(uint32_t)s;
  };
  auto among = [&](auto L, int s, uint32_t k) {
    if (s >= len || (L >= 1 && k != known[0])) return false;
    if constexpr (L == 2)
      if (position_word(pos[s]) != known[1]) return false;
    return shift == 32 || word(L, s, k) >> (shift & 31) == prefix;
  };
  auto over = [&](auto L, auto f) {
    if constexpr (L == 0) each(f);
    else again(f);
  };
  // Counts one word's digits until the cutoff is known, few slots are left, or
  // the word is at its end.
  enum { END, DONE, FEWER };
  auto settle = [&](auto L) {
    prefix = 0;
    for (shift = 32; shift > 0;) {
      const int bits = min(DIGIT, shift), next = shift - bits;
      over(L, [&](int s, uint32_t k) {
        const bool in = among(L, s, k);
        uint32_t digit = 0;
        if (L == 0 || in) digit = (word(L, s, k) >> next) & ((1u << bits) - 1u);
        // (a wave that holds one digit adds it at once: equal weights)
        const uint32_t first = __builtin_amdgcn_readfirstlane(digit);
        if (__ballot(digit != first) == 0) {
          const uint64_t who = __ballot(in);
          if (lane == 0) atomicAdd(&lds.hist[first * REP], (uint32_t)__popcll(who));
        } else if (in) {
          atomicAdd(&lds.hist[digit * REP + (lane & (REP - 1))], 1u);
        }
      });
      __syncthreads();
      const u32x4 h0 = own[0], h1 = own[1];
      own[0] = own[1] = (u32x4){0, 0, 0, 0};  // (for the next digit)
      const int c1 = (int)((h1[0] + h1[1]) + (h1[2] + h1[3])), c0 = (int)((h0[0] + h0[1]) + (h0[2] + h0[3]));
      const uint32_t run = wave_scan((uint32_t)(c1 + c0));
      if (lane == 63) lds.scan[wave] = run;
      __syncthreads();
      int before = (int)run - c1 - c0;
#pragma unroll
      for (int i = 0; i < EW; i++) before += i < wave ? (int)lds.scan[i] : 0;
      if (before < need && need <= before + c1 + c0) {
        const bool one = need <= before + c1;
        lds.found[0] = 2 * ((1 << (DIGIT - 1)) - 1 - tid) + (one ? 1 : 0);
        lds.found[1] = need - before - (one ? 0 : c1);
        lds.found[2] = lds.found[1] == (one ? c1 : c0);
        lds.found[3] = one ? c1 : c0;
      }
      __syncthreads();
      need = lds.found[1];
      prefix = shift == 32 ? (uint32_t)lds.found[0] : prefix << bits | (uint32_t)lds.found[0];
      shift = next;
      if (lds.found[2]) return DONE;
      if (lds.found[3] <= LIST) return FEWER;
    }
    return END;
  };
  auto list = [&](auto L) {
    over(L, [&](int s, uint32_t k) {
      if (!among(L, s, k)) return;
      const int i = atomicAdd(&lds.listed, 1);
      lds.place[i] = (uint64_t)k << 32;
      lds.slot[i] = s;
    });
    __syncthreads();
    if (tid < lds.listed) lds.place[tid] |= position_word(pos[lds.slot[tid]]);
  };
  const std::integral_constant<int, 0> W;
  const std::integral_constant<int, 1> P;
  const std::integral_constant<int, 2> S;
  // (all of a digit's slots kept: the cutoff lies just before its lowest word)
  int how = settle(W);
  if (how == DONE) return Cutoff{(prefix << shift) - 1, 0, 0, true};
  const bool mark = how == FEWER && bits != nullptr;
  const uint32_t above = prefix << shift | ((1u << shift) - 1u);  // (the listed weights' largest)
  if (how == FEWER) list(W);
  if (how == END) {
    known[0] = prefix;
    how = settle(P);
    if (how == DONE) return Cutoff{known[0], (prefix << shift) - 1, -1, false};
    if (how == FEWER) list(P);
  }
  if (how == END) {
    known[1] = prefix;
    how = settle(S);
    if (how == DONE) return Cutoff{known[0], known[1], (int)~(prefix << shift), false};
    list(S);
  }
  // few are left: each counts those before it
  static_assert(EB / LIST == 4, "the threads of a slot");
  __syncthreads();
  const int n = lds.listed, i = tid / (EB / LIST);  // (four threads a slot)
  if (i < n) {
    const uint64_t mine = lds.place[i];
    const int s = lds.slot[i];
    int before = 0;
#pragma unroll 8
    for (int j = tid % (EB / LIST); j < n; j += EB / LIST) {
      const uint64_t p = lds.place[j];
      const int o = lds.slot[j];
      before += (int)(p > mine) | ((int)(p == mine) & (int)(o < s));
    }
    before += __shfl_xor(before, 1);
    before += __shfl_xor(before, 2);
    if (tid % (EB / LIST) == 0) {
      if (before == need - 1) lds.cutoff = Cutoff{(uint32_t)(mine >> 32), (uint32_t)mine, s, false};
      if (mark && before < need) atomicOr(&bits[s >> 5], 1u << (s & 31));
    }
  }
  __syncthreads();
  return mark ? Cutoff{above, 0, 0, true} : lds.cutoff;
}

// A head's sizes, and the sequence's outputs; false where there is nothing to
// cut (the slots are then copied, if need be).
struct Head {
  int64_t bh;
  int b, kh, len, keep;
  const float* mass;
  const int32_t* pos;
  float* new_mass;
  int32_t* new_pos;
  int64_t next, sinks, recent;
  bool cut;
  XS_DEV Head(const xs_cache_evict_args& a, const EvictWork& w) {
    bh = blockIdx.x;
    b = (int)(bh / a.kv_heads);
    kh = (int)(bh % a.kv_heads);
    len = a.len[b];
    const int64_t limit = a.max_len ? a.max_len : a.capacity;
    const bool bad = len < 0 || len > limit;
    keep = (int)min((int64_t)len, a.keep);
    if (threadIdx.x == 0) {
      w.moves[bh] = 0;
      if (kh == 0) {
        a.seq_status[b] = bad ? XS_ROW_BAD_PARAM : XS_ROW_OK;
        a.new_len[b] = bad ? len : keep;
      }
    }
    mass = a.mass + bh * a.slot_ld;
    pos = a.pos + bh * a.slot_ld;
    new_mass = a.new_mass + bh * a.slot_ld;
    new_pos = a.new_pos + bh * a.slot_ld;
    next = a.next_pos[b];
    sinks = a.sinks;
    recent = a.recent;
    cut = !bad && len > keep;
    if (!bad && !cut) copy(keep);
  }
  XS_DEV void copy(int n) const {
    if (new_mass == mass) return;
    for (int s = threadIdx.x; s < n; s += EB) {
      new_mass[s] = mass[s];
      new_pos[s] = pos[s];
    }
  }
  XS_DEV bool held(int p) const { return p < sinks || p >= next - recent; }
};

// f(slot, weight word) for every slot, from memory.
template <typename F>
XS_DEV void each_slot(const Head& h, F f) {
  const int lane = threadIdx.x & 63;
#pragma unroll 4
  for (int s0 = threadIdx.x - lane; s0 < h.len; s0 += EB) {
    const int s = min(s0 + lane, h.len - 1);
    f(s0 + lane, weight_word(h.mass[s], h.held(h.pos[s])));
  }
}

// Slots in registers: V times four consecutive ones a thread (len <= 4 V EB;
// 16-byte aligned arrays of a slot_ld that is a multiple of 4).  apart: the rows of
// k and v are left to evict_rows_kernel; else there are at most NEAR moves,
// made here.  Bound by latency and by one CU's share: 128 heads of 4,128 slots
// cut to 4,096 take 12.8 us (26.6 when every pass read its slots again), 32
// heads of 1,311 to 32,768 cut to 2,048 take 28 us here (54) and 9 for the rows.
template <int V>
__global__ __launch_bounds__(EB) void evict_kernel(const xs_cache_evict_args a, const EvictWork w, int apart) {
  __shared__ SelectLds lds;
  __shared__ uint32_t base[V * EW];
  __shared__ uint32_t bits[V * EB / 8];
  __shared__ int near_free[NEAR], near_filler[NEAR];
  const int tid = threadIdx.x, lane = tid & 63;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const Head h(a, w);
  if (!h.cut) return;
  const int len = h.len, keep = h.keep;
  uint32_t word[V][4];
  {
    f32x4 m[V];
    u32x4 p[V];
#pragma unroll
    for (int e = 0; e < V; e++) {
      const int s = (e * EB + tid) * 4, at = s < len ? s : 0;
      m[e] = *(const f32x4*)(h.mass + at);
      p[e] = *(const u32x4*)(h.pos + at);
    }
#pragma unroll
    for (int e = 0; e < V; e++) {
      const int s = (e * EB + tid) * 4;
#pragma unroll
      for (int j = 0; j < 4; j++) word[e][j] = weight_word(m[e][j], h.held((int)p[e][j]));
      if (h.new_mass != h.mass && s < keep) {
        if (s + 4 <= keep) {
          *(f32x4*)(h.new_mass + s) = m[e];
          *(u32x4*)(h.new_pos + s) = p[e];
        } else {
#pragma unroll
          for (int j = 0; j < 3; j++)
            if (s + j < keep) {
              h.new_mass[s + j] = m[e][j];
              h.new_pos[s + j] = (int)p[e][j];
            }
        }
      }
    }
  }
  if (tid < V * EB / 8) bits[tid] = 0;  // (find_cutoff's barriers order it)
  const Cutoff c = find_cutoff(lds, len, keep, h.pos, bits, [&](auto f) {
#pragma unroll
    for (int e = 0; e < V; e++)
      if ((e * EB + wave * 64) * 4 < len)
#pragma unroll
        for (int j = 0; j < 4; j++) f((e * EB + tid) * 4 + j, word[e][j]);
  }, [&](auto f) { each_slot(h, f); });
  // bit 4 e + j: the slot is kept
  uint32_t kept = 0;
#pragma unroll
  for (int e = 0; e < V; e++) kept |= (bits[(e * EB + tid) >> 3] >> (4 * (tid & 7)) & 15u) << (4 * e);
#pragma unroll
  for (int e = 0; e < V; e++)
#pragma unroll
    for (int j = 0; j < 4; j++) {
      const int s = (e * EB + tid) * 4 + j;
      if (s < len && c.keeps(word[e][j], s, h.pos)) kept |= 1u << (4 * e + j);
    }
  // Freed slots below keep, then the kept ones past it, as many: in their
  // order, the flagged slots' two halves.
  int32_t* freed = apart ? w.free_ + h.bh * w.pairs : near_free;
  int32_t* filler = apart ? w.filler + h.bh * w.pairs : near_filler;
  auto flag = [&](int e, int j) { return ((kept >> (4 * e + j)) & 1u) != ((e * EB + tid) * 4 + j < keep ? 1u : 0u); };
#pragma unroll
  for (int e = 0; e < V; e++) {
    uint32_t n = 0;
#pragma unroll
    for (int j = 0; j < 4; j++) n += (uint32_t)__popcll(__ballot(flag(e, j)));
    if (lane == 0) base[e * EW + wave] = n;
  }
  __syncthreads();
  uint32_t total;
  const uint32_t mine = block_scan(tid < V * EW ? base[tid] : 0u, lds.scan, &total);
  if (tid < V * EW) base[tid] = mine;
  __syncthreads();
  const int moves = (int)total / 2;
#pragma unroll
  for (int e = 0; e < V; e++) {
    uint32_t n = base[e * EW + wave];
#pragma unroll
    for (int j = 0; j < 4; j++) {
      const uint64_t who = __ballot(flag(e, j));
      n = __builtin_amdgcn_mbcnt_hi((uint32_t)(who >> 32), __builtin_amdgcn_mbcnt_lo((uint32_t)who, n));
    }
#pragma unroll
    for (int j = 0; j < 4; j++)
      if (flag(e, j)) {
        const int s = (e * EB + tid) * 4 + j, i = (int)n++;
        if (s < keep) freed[i] = s;
        else filler[i - moves] = s;
      }
  }
  __syncthreads();
  if (tid == 0) w.moves[h.bh] = moves;
  for (int i = tid; i < moves; i += EB) {
    const int to = freed[i], from = filler[i];
    h.new_mass[to] = h.mass[from];
    h.new_pos[to] = h.pos[from];
  }
  if (apart) return;
  const int parts = a.head_dim / 8;
  const int64_t head = h.b * a.cache.seq_stride + h.kh * a.cache.head_stride;
  for (int j = tid; j < moves * parts; j += EB) move_part(a, head, near_filler[j / parts], near_free[j / parts], j % parts * 8);
}

// The same for any length and alignment: every pass reads the slots again, the
// kept ones go to a bitmap, and all rows are left to evict_rows_kernel.
__global__ __launch_bounds__(EB) void evict_long_kernel(const xs_cache_evict_args a, const EvictWork w) {
  __shared__ SelectLds lds;
  __shared__ uint64_t scan[EW];
  __shared__ uint64_t base[EB];
  const int tid = threadIdx.x, lane = tid & 63;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const Head h(a, w);
  if (!h.cut) return;
  const int len = h.len, keep = h.keep;
  h.copy(keep);
  auto each = [&](auto f) { each_slot(h, f); };
  const Cutoff c = find_cutoff(lds, len, keep, h.pos, nullptr, each, each);
  uint64_t* kept = w.kept + h.bh * w.words;
  const int words = (len + 63) / 64;
  each([&](int s, uint32_t k) {
    const uint64_t bit = __ballot(s < len && c.keeps(k, s, h.pos));
    if (lane == 0) kept[s / 64] = bit;
  });
  __syncthreads();
  // freed slots below keep and kept ones past it, by their ranks
  int32_t* freed = w.free_ + h.bh * w.pairs;
  int32_t* filler = w.filler + h.bh * w.pairs;
  uint64_t run = 0;  // low half: free slots so far, high: fillers
  auto split = [&](int i, uint64_t bits, uint64_t* f, uint64_t* m) {
    const int in = min(max(keep - i * 64, 0), 64);  // the word's slots below keep
    const uint64_t low = in == 64 ? ~0ull : (1ull << in) - 1ull;
    *f = ~bits & low;
    *m = bits & ~low;
  };
  for (int w0 = 0; w0 < words; w0 += EB) {
    const int i = w0 + tid;
    uint64_t f = 0, m = 0;
    if (i < words) split(i, kept[i], &f, &m);
    uint64_t total;
    base[tid] = run + block_scan((uint64_t)__popcll(f) | (uint64_t)__popcll(m) << 32, scan, &total);
    run += total;
    __syncthreads();
    for (int j = wave; j < EB && w0 + j < words; j += EW) {
      split(w0 + j, kept[w0 + j], &f, &m);
      const uint64_t below = (1ull << lane) - 1ull, at = base[j];
      const int slot = (w0 + j) * 64 + lane;
      if ((f >> lane) & 1ull) freed[(uint32_t)at + __popcll(f & below)] = slot;
      if ((m >> lane) & 1ull) filler[(uint32_t)(at >> 32) + __popcll(m & below)] = slot;
    }
    __syncthreads();
  }
  const int moves = (int)(run >> 32);
  if (tid == 0) w.moves[h.bh] = moves;
  for (int i = tid; i < moves; i += EB) {
    const int to = freed[i], from = filler[i];
    h.new_mass[to] = h.mass[from];
    h.new_pos[to] = h.pos[from];
  }
}

// The rows of a head's moves, ROWS of them a workgroup.
constexpr int ROWS = 64;
__global__ __launch_bounds__(256) void evict_rows_kernel(const xs_cache_evict_args a, const EvictWork w, int blocks) {
  const int64_t bh = blockIdx.x / blocks;
  const int first = (blockIdx.x % blocks) * ROWS, n = min(ROWS, w.moves[bh] - first);
  const int parts = a.head_dim / 8;
  const int64_t head = bh / a.kv_heads * a.cache.seq_stride + bh % a.kv_heads * a.cache.head_stride;
  for (int j = threadIdx.x; j < n * parts; j += 256) {
    const int64_t at = bh * w.pairs + first + j / parts;
    move_part(a, head, w.filler[at], w.free_[at], j % parts * 8);
  }
}

}  // namespace xst

// ---------------------------------------------------------------------------
// Host side: the cache context and its calls.

struct xs_cache_context {
  int device;
  hipStream_t stream;
  xs_cache_dims dims;
  xst::EvictWork evict;
  int n_cu;
  float* part;    // attention's partial results, one for each workgroup of a split call
  int64_t part_floats;
};

namespace {

// Workgroups of attend_kernel that a CU holds at once (by its registers; its
// launch bound asks for as many), by the head's size and the row tiles.
constexpr int64_t per_cu(int dp, int rt) { return dp * rt <= 64 ? 4 : dp * rt <= 128 ? 3 : dp * rt <= 256 ? 2 : 1; }
// How many times over a split call fills the device: once where all sequences
// end together (one of them: 8 heads over 131,072 slots 113 us, filled four
// times 145), more often where some end early (32 sequences of 327 to 8,192
// slots: 134 us, filled twice 151; but 32 of 8,192 take 222 instead of 214).
constexpr int64_t rounds(int64_t seqs) { return seqs > 1 ? 4 : 1; }

template <typename T, int DP, int RT, bool EXACT, bool WIDE>
int attend_run(xs_cache_context* c, const xs_tree_attend_args& a) {
  xst::Cut cut;
  cut.G = (int32_t)(a.q_heads / a.kv_heads);
  constexpr int WAVES = WIDE ? xst::NW : 1;  // of a workgroup, with rows of their own
  const int64_t wgs = (a.nodes * cut.G + 16 * RT * WAVES - 1) / (16 * RT * WAVES);
  cut.tiles = (int32_t)(wgs * WAVES);
  cut.scale = a.scale * xst::LOG2E;
  cut.part = c->part;
  const int64_t limit = a.max_len ? a.max_len : a.capacity;
  const int64_t blocks = (limit + xst::KB - 1) / xst::KB + (a.nodes + xst::KB - 1) / xst::KB;
  const int64_t units = a.seqs * a.kv_heads * wgs;
  // (rows of several waves: once, their partial results cost as much as 8 blocks each)
  const int64_t most = c->n_cu * (WIDE ? 1 : per_cu(DP, RT) * rounds(a.seqs));
  const int64_t nsplit = std::max<int64_t>(1, std::min<int64_t>(xst::SPLITS, most / units));
  cut.chunk = (int32_t)((blocks + nsplit - 1) / nsplit);
  // Two blocks a wave at least, and no split for its own sake: a join costs
  // 5 us (300 slots: 9.8 us whole, 15 split; 1,777 slots: 14.9 split, 15.8 in
  // halves).
  if (cut.chunk < 2 * xst::NW) cut.chunk = 2 * xst::NW;
  if (blocks <= 4 * xst::NW) cut.chunk = (int32_t)blocks;
  cut.nsplit = (int32_t)((blocks + cut.chunk - 1) / cut.chunk);
  const int64_t groups = a.seqs * a.kv_heads * cut.nsplit;
  const int64_t grid = (groups + 7) / 8 * 8 * wgs, join = a.seqs * a.kv_heads * cut.tiles * RT * xst::Shape<DP, RT>::VH;
  const int64_t joiners = xst::join_threads<DP>(cut.nsplit <= xst::FEW);
  if (!xs_host_launch_fits(grid, 64 * xst::NW) || (cut.nsplit > 1 && !xs_host_launch_fits(join, joiners))) return XS_ERR_CAPACITY;
  if (cut.nsplit > 1 && groups * cut.tiles * xst::Shape<DP, RT>::PART > c->part_floats) return XS_ERR_CAPACITY;  // (never: groups * tiles <= most)
  cut.groups = (int32_t)groups;
  if constexpr (WIDE)
    hipLaunchKernelGGL((xst::attend_wide_kernel<T, DP, RT, EXACT>), dim3((unsigned)grid), dim3(64 * xst::NW), 0, c->stream, a, cut);
  else
    hipLaunchKernelGGL((xst::attend_kernel<T, DP, RT, EXACT>), dim3((unsigned)grid), dim3(64 * xst::NW), 0, c->stream, a, cut);
  if (cut.nsplit > xst::FEW)
    hipLaunchKernelGGL((xst::join_kernel<T, DP, RT, false>), dim3((unsigned)join), dim3(xst::join_threads<DP>(false)), 0, c->stream, a, cut);
  else if (cut.nsplit > 1)
    hipLaunchKernelGGL((xst::join_kernel<T, DP, RT, true>), dim3((unsigned)join), dim3(xst::join_threads<DP>(true)), 0, c->stream, a, cut);
  return hipGetLastError() == hipSuccess ? XS_OK : XS_ERR_HIP;
}

// The partial results of the largest split call within `dims`: those that fill
// the device, by the shapes that attend_rows takes for so many rows a head.
int64_t attend_floats(const xs_cache_dims& dims, int n_cu) {
  const int64_t rows = dims.max_nodes * dims.q_heads;  // (of one kv head)
  if ((dims.capacity + xst::KB - 1) / xst::KB + (dims.max_nodes + xst::KB - 1) / xst::KB <= 4 * xst::NW) return 0;  // (none is split)
  int64_t most = 0;
  auto narrow = [&](int64_t per_cu, int64_t part) { most = std::max(most, n_cu * per_cu * rounds(dims.max_seqs) * part); };
  auto wide = [&](int64_t part) { most = std::max(most, n_cu * xst::NW * part); };
  narrow(per_cu(64, 1), xst::Shape<64, 1>::PART);
  if (rows > 16) narrow(per_cu(64, 2), xst::Shape<64, 2>::PART);
  if (rows > 32) narrow(per_cu(64, 4), xst::Shape<64, 4>::PART);
  if (rows > 64) wide(xst::Shape<64, 2>::PART);
  if (rows > 128) wide(xst::Shape<64, 4>::PART);
  if (dims.head_dim > 64) {
    narrow(per_cu(128, 1), xst::Shape<128, 1>::PART);
    if (rows > 16) narrow(per_cu(128, 2), xst::Shape<128, 2>::PART);
    if (rows > 32) narrow(per_cu(128, 4), xst::Shape<128, 4>::PART);
    if (rows > 64) wide(xst::Shape<128, 2>::PART);
    if (rows > 128) wide(xst::Shape<128, 4>::PART);
  }
  if (dims.head_dim > 128) {
    narrow(per_cu(256, 1), xst::Shape<256, 1>::PART);
    if (rows > 16) narrow(per_cu(256, 2), xst::Shape<256, 2>::PART);
    if (rows > 32) wide(xst::Shape<256, 2>::PART);
  }
  return most;
}

template <typename T, int DP, int RT, bool WIDE>
int attend_exact(xs_cache_context* c, const xs_tree_attend_args& a) {
  return a.head_dim == DP ? attend_run<T, DP, RT, true, WIDE>(c, a) : attend_run<T, DP, RT, false, WIDE>(c, a);
}

template <typename T, int DP>
int attend_rows(xs_cache_context* c, const xs_tree_attend_args& a) {
  const int64_t rows = a.nodes * (a.q_heads / a.kv_heads);
  if (rows <= 16) return attend_exact<T, DP, 1, false>(c, a);
  if (rows <= 32) return attend_exact<T, DP, 2, false>(c, a);
  if constexpr (DP <= 128) {
    // (128 rows as two row tiles of four waves: 261 us for 8 x 32 nodes over
    // 32,768 slots; as two workgroups of 64 rows each, reading the keys twice, 317)
    if (rows <= 64) return attend_exact<T, DP, 4, false>(c, a);
    if (rows <= 128) return attend_exact<T, DP, 2, true>(c, a);
    return attend_exact<T, DP, 4, true>(c, a);
  } else {
    return attend_exact<T, DP, 2, true>(c, a);
  }
}

template <typename T>
int attend_dim(xs_cache_context* c, const xs_tree_attend_args& a) {
  if (a.head_dim <= 64) return attend_rows<T, 64>(c, a);
  if (a.head_dim <= 128) return attend_rows<T, 128>(c, a);
  return attend_rows<T, 256>(c, a);
}

// Workgroups of commit_kernel that a CU holds at once, as its launch bound asks.
constexpr int64_t commit_per_cu(int dp, int rt) { return dp * rt <= 256 ? 3 : 2; }

template <typename T, int DP, int RT>
int commit_run(xs_cache_context* c, const xs_cache_commit_args& a) {
  const int64_t limit = a.max_len ? a.max_len : a.capacity;
  const int64_t blocks = (limit + xst::KB - 1) / xst::KB, heads = a.seqs * a.kv_heads;
  // Key blocks of a wave: the device filled once, or, where sequences may end
  // early, five times (64 sequences of 327 to 8,192 slots: 170 us with four,
  // 146 so), and at least RT, so that a wave reads twice as many keys as rows (2
  // sequences of 65,536 slots of 256, 8 nodes: 34 us with 4, 63 with 1).
  const int64_t waves = xst::NW * c->n_cu * commit_per_cu(DP, RT) * (a.seqs > 1 ? 5 : 1);
  const int64_t share = std::max<int64_t>(RT, (blocks * heads + waves - 1) / waves);
  const int64_t shares = (a.q ? (blocks + xst::NW * share - 1) / (xst::NW * share) : 0) + 1;
  if (!xs_host_launch_fits(heads * shares, 64 * xst::NW)) return XS_ERR_CAPACITY;
  const dim3 grid((unsigned)(heads * shares)), block(64 * xst::NW);
  if (a.head_dim == DP)
    hipLaunchKernelGGL((xst::commit_kernel<T, DP, RT, true>), grid, block, 0, c->stream, a, (int)shares, (int)share);
  else
    hipLaunchKernelGGL((xst::commit_kernel<T, DP, RT, false>), grid, block, 0, c->stream, a, (int)shares, (int)share);
  return hipGetLastError() == hipSuccess ? XS_OK : XS_ERR_HIP;
}

template <typename T, int DP>
int commit_rows(xs_cache_context* c, const xs_cache_commit_args& a) {
  const int64_t rows = a.nodes * (a.q_heads / a.kv_heads);
  if (rows <= 16) return commit_run<T, DP, 1>(c, a);
  return rows <= 32 ? commit_run<T, DP, 2>(c, a) : commit_run<T, DP, 4>(c, a);
}

template <typename T>
int commit_dim(xs_cache_context* c, const xs_cache_commit_args& a) {
  if (a.head_dim <= 64) return commit_rows<T, 64>(c, a);
  if (a.head_dim <= 128) return commit_rows<T, 128>(c, a);
  return commit_rows<T, 256>(c, a);
}

template <int V>
void evict_run(xs_cache_context* c, const xs_cache_evict_args& a, bool apart) {
  hipLaunchKernelGGL((xst::evict_kernel<V>), dim3((unsigned)(a.seqs * a.kv_heads)), dim3(xst::EB), 0, c->stream, a, c->evict, apart ? 1 : 0);
}

bool aligned16(const void* p) { return ((uintptr_t)p & 15u) == 0; }

using xs_host::OnDevice;

// The failure is the call's to report: left in the thread, it would fail the
// next launch that asks for the last error.
int create_failed() {
  (void)hipGetLastError();
  return XS_ERR_HIP;
}

}  // namespace

extern "C" {

int xs_cache_create(int device, const xs_cache_dims* dims, xs_cache_context** out) {
  if (!out) return XS_ERR_ARG;
  *out = nullptr;
  const int rc = xs_host_check_dims(dims);
  if (rc) return rc;
  const OnDevice on(device);
  if (!on.ok) return create_failed();
  xs_cache_context* c = (xs_cache_context*)calloc(1, sizeof(xs_cache_context));
  if (!c) return XS_ERR_HIP;
  c->device = device;
  c->dims = *dims;
  if (hipDeviceGetAttribute(&c->n_cu, hipDeviceAttributeMultiprocessorCount, device) != hipSuccess || c->n_cu < 1)
    c->n_cu = 256;
  c->part_floats = attend_floats(*dims, c->n_cu);
  const int64_t heads = dims->max_seqs * dims->kv_heads;
  c->evict.words = (dims->capacity + 63) / 64;
  c->evict.pairs = dims->capacity / 2 + 1;
  if (hipMalloc((void**)&c->part, c->part_floats * sizeof(float)) != hipSuccess ||
      hipMalloc((void**)&c->evict.kept, heads * c->evict.words * sizeof(uint64_t)) != hipSuccess ||
      hipMalloc((void**)&c->evict.free_, heads * c->evict.pairs * sizeof(int32_t)) != hipSuccess ||
      hipMalloc((void**)&c->evict.filler, heads * c->evict.pairs * sizeof(int32_t)) != hipSuccess ||
      hipMalloc((void**)&c->evict.moves, heads * sizeof(int32_t)) != hipSuccess) {
    xs_cache_destroy(c);
    return create_failed();
  }
  *out = c;
  return XS_OK;
}

int xs_cache_destroy(xs_cache_context* c) {
  if (!c) return XS_OK;
  const OnDevice on(c->device);
  if (c->stream) (void)hipStreamSynchronize(c->stream); else (void)hipDeviceSynchronize();
  if (c->part) (void)hipFree(c->part);
  if (c->evict.kept) (void)hipFree(c->evict.kept);
  if (c->evict.free_) (void)hipFree(c->evict.free_);
  if (c->evict.filler) (void)hipFree(c->evict.filler);
  if (c->evict.moves) (void)hipFree(c->evict.moves);
  free(c);
  return XS_OK;
}

int xs_cache_set_stream(xs_cache_context* c, void* s) {
  if (!c) return XS_ERR_ARG;
  c->stream = (hipStream_t)s;
  return XS_OK;
}

int xs_tree_attend(xs_cache_context* c, const xs_tree_attend_args* in) {
  const int rc = xs_host_check_attend(c ? &c->dims : nullptr, in);
  if (rc) return rc;
  if (in->seqs == 0) return XS_OK;
  const OnDevice on(c->device);
  if (!on.ok) return XS_ERR_HIP;
  if (in->dtype == XS_BF16) return attend_dim<xst::Bf16>(c, *in);
  return attend_dim<xst::F16>(c, *in);
}

int xs_cache_commit(xs_cache_context* c, const xs_cache_commit_args* in) {
  const int rc = xs_host_check_commit(c ? &c->dims : nullptr, in);
  if (rc) return rc;
  if (in->seqs == 0) return XS_OK;
  const OnDevice on(c->device);
  if (!on.ok) return XS_ERR_HIP;
  if (in->dtype == XS_BF16) return commit_dim<xst::Bf16>(c, *in);
  return commit_dim<xst::F16>(c, *in);
}

int xs_cache_evict(xs_cache_context* c, const xs_cache_evict_args* in) {
  const int rc = xs_host_check_evict(c ? &c->dims : nullptr, in);
  if (rc) return rc;
  if (in->seqs == 0) return XS_OK;
  const OnDevice on(c->device);
  if (!on.ok) return XS_ERR_HIP;
  const int64_t limit = in->max_len ? in->max_len : in->capacity;
  const int64_t heads = in->seqs * in->kv_heads;
  // moves of a head: at most the slots past keep, and the slots of keep
  const int64_t most = limit > in->keep ? std::min(in->keep, limit - in->keep) : 0;
  const bool fits = limit <= 32 * xst::EB && aligned16(in->mass) && aligned16(in->pos) && aligned16(in->new_mass) &&
                    aligned16(in->new_pos) && in->slot_ld % 4 == 0;
  const bool apart = most > xst::NEAR || (!fits && most > 0);
  const int64_t blocks = (most + xst::ROWS - 1) / xst::ROWS;
  if (!xs_host_launch_fits(heads, xst::EB) || (apart && !xs_host_launch_fits(heads * blocks, 256))) return XS_ERR_CAPACITY;
  if (!fits) hipLaunchKernelGGL(xst::evict_long_kernel, dim3((unsigned)heads), dim3(xst::EB), 0, c->stream, *in, c->evict);
  else if (limit <= 4 * xst::EB) evict_run<1>(c, *in, apart);
  else if (limit <= 8 * xst::EB) evict_run<2>(c, *in, apart);
  else evict_run<8>(c, *in, apart);
  if (apart)
    hipLaunchKernelGGL(xst::evict_rows_kernel, dim3((unsigned)(heads * blocks)), dim3(256), 0, c->stream, *in, c->evict, (int)blocks);
  return hipGetLastError() == hipSuccess ? XS_OK : XS_ERR_HIP;
}

}  // extern "C"
