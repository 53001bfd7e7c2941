// xs_prompt.hip -- a prompt's way to its attention (MI355X, gfx950): norms and
// positions of queries and keys, and causal attention of packed prompts.
//
// Compiled with -ffp-contract=off; fused multiply-adds are written out.

#include <hip/hip_runtime.h>

#include <algorithm>
#include <stdint.h>

#include "../../include/xsamp.h"
#include "xs_attend.h"
#include "xs_cache.h"
#include "xs_device.h"
#include "xs_host.h"
#include "xs_rows32.h"

namespace xsp {

using namespace xst;

// ---------------------------------------------------------------------------
// Norms and positions.
//
// A head of a token is LPH lanes (a power of two, head_dim / 16 at least) of 16
// elements each: two 16-byte pieces, which for halves are those of a rotated
// pair, so that no element crosses lanes.  A workgroup takes `passes` passes of
// RT / LPH heads in a row (tokens outermost, a token's q heads before its kv
// heads), a pass's pieces on their way while the last one is worked on; the
// angles of its tokens, and the weights, are in LDS.  Bound by the one read and
// write of the heads: 16,384 tokens of 40 heads of 128 (336 MB) in 80 to 86 us by card.
// All passes' pieces in registers at once take 204 of them, which leaves two
// waves a SIMD: 186 us.

constexpr int RT = 256;  // threads of a workgroup
constexpr int ROT_PASSES = 8;

template <typename T>
XS_DEV void widen8(u32x4 r, float (&x)[8]) {
#pragma unroll
  for (int i = 0; i < 4; i++) {
    x[2 * i] = T::widen((uint16_t)r[i]);
    x[2 * i + 1] = T::widen((uint16_t)(r[i] >> 16));
  }
}

template <typename T, int LPH>
__global__ __launch_bounds__(RT, 8) void rotate_kernel(const xs_qk_rotate_args a, int passes) {
  extern __shared__ float shared[];  // [q, k][head_dim] weights; [tokens of the workgroup][rot_dim / 2] cos, sin
  constexpr int PER = RT / LPH;      // heads of a pass
  const int heads = (int)(a.q_heads + a.kv_heads), D = a.head_dim, half = a.rot_dim / 2;
  const bool halves = a.pairs == XS_ROT_HALVES, norm = a.q_weight || a.k_weight;
  f32x2* turn = (f32x2*)(shared + 2 * D);
  const int p = threadIdx.x % LPH;
  const int64_t first = (int64_t)blockIdx.x * PER * passes, all = a.tokens * heads;
  const int64_t t0 = first / heads;

  // the lane's two pieces
  const int rc = halves ? half / 8 : 0, chunks = D / 8;
  const int c0 = p < rc ? p : 2 * p, c1 = p < rc ? p + rc : 2 * p + 1;
  const bool in0 = c0 < chunks, in1 = c1 < chunks;

  // the lane's head of the first pass; a pass on is `over` tokens and `by` heads
  int64_t at = first + threadIdx.x / LPH;
  int t = (int)(at - t0 * heads) / heads, h = (int)(at - t0 * heads) - t * heads;  // (t counted from t0)
  const int over = PER / heads, by = PER % heads;

  auto fetch = [&](u32x4 (&raw)[2]) {
    raw[0] = raw[1] = (u32x4){0, 0, 0, 0};
    if (at >= all) return;
    const uint16_t* x = h < a.q_heads ? (const uint16_t*)a.q + (t0 + t) * a.q_token_stride + h * a.q_head_stride
                                      : (const uint16_t*)a.k + (t0 + t) * a.k_token_stride + (h - a.q_heads) * a.k_head_stride;
    if (in0) raw[0] = *(const u32x4*)(x + 8 * c0);
    if (in1) raw[1] = *(const u32x4*)(x + 8 * c1);
  };
  u32x4 raw[2];
  fetch(raw);

  if (norm)
    for (int i = threadIdx.x; i < 2 * D; i += RT) {
      const float* w = i < D ? a.q_weight : a.k_weight;
      shared[i] = w ? w[i < D ? i : i - D] : 0.0f;
    }
  if (half > 0) {
    // The angle in turns, from f64 (a position of 2^31 times a frequency of 1
    // leaves 2^-23 of a turn); cos and sin of its fraction in f32.
    const int64_t last = min(first + (int64_t)PER * passes, all) - 1;
    const int tokens = (int)(last / heads - t0) + 1;
    for (int i = threadIdx.x; i < tokens * half; i += RT) {
      const double y = (double)a.pos[t0 + i / half] * (double)a.inv_freq[i % half] * 0.15915494309189533577;
      float sn, cn;
      sincospif((float)(2.0 * (y - rint(y))), &sn, &cn);
      turn[i] = (f32x2){cn, sn};
    }
  }
  __syncthreads();

#pragma unroll 1
  for (int i = 0; i < passes; i++) {
    const bool live = at < all, key = h >= a.q_heads;
    const int t1 = t, h1 = h;
    float x[2][8];
    widen8<T>(raw[0], x[0]);
    widen8<T>(raw[1], x[1]);
    at += PER;
    t += over;
    h += by;
    if (h >= heads) {
      h -= heads;
      t++;
    }
    if (i + 1 < passes) fetch(raw);
    if (norm) {
      auto squares = [&](float by) {
        float sum = 0.0f;
#pragma unroll
        for (int e = 0; e < 8; e++) {
          const float u = x[0][e] * by, v = x[1][e] * by;
          sum = __builtin_fmaf(v, v, __builtin_fmaf(u, u, sum));
        }
#pragma unroll
        for (int m = 1; m < LPH; m *= 2) sum += __shfl_xor(sum, m);
        return sum / (float)D;
      };
      const float mean = squares(1.0f) + a.eps;
      float inv = __builtin_amdgcn_rsqf(mean);  // (to a step or so)
      const bool tiny = mean < 0x1p-80f;
      if (__any(tiny || mean == -NEG_INF)) {  // (rare) squares past f32's range: those of elements 2^96 times as large, or as small
        const float by = tiny ? 0x1p96f : 0x1p-96f, far = __builtin_amdgcn_rsqf(squares(by) + a.eps * by * by);
        if (tiny || mean == -NEG_INF) {
#pragma unroll
          for (int j = 0; j < 2; j++)
#pragma unroll
            for (int e = 0; e < 8; e++) x[j][e] = tiny ? x[j][e] * by * far : x[j][e] * far * by;
          inv = 1.0f;
        }
      }
      const float* w = shared + (key ? D : 0);
#pragma unroll
      for (int e = 0; e < 8; e++) {
        if (in0) x[0][e] = x[0][e] * inv * w[8 * c0 + e];
        if (in1) x[1][e] = x[1][e] * inv * w[8 * c1 + e];
      }
    }
    const f32x2* cs = turn + t1 * half;
    if (halves) {
      if (live && p < rc) {
#pragma unroll
        for (int e = 0; e < 8; e++) {
          const f32x2 z = cs[8 * p + e];
          const float u = x[0][e], v = x[1][e];
          x[0][e] = __builtin_fmaf(u, z[0], -(v * z[1]));
          x[1][e] = __builtin_fmaf(v, z[0], u * z[1]);
        }
      }
    } else {
#pragma unroll
      for (int j = 0; j < 2; j++)
        if (live && 8 * (2 * p + j) < a.rot_dim) {
#pragma unroll
          for (int e = 0; e < 8; e += 2) {
            const f32x2 z = cs[4 * (2 * p + j) + e / 2];
            const float u = x[j][e], v = x[j][e + 1];
            x[j][e] = __builtin_fmaf(u, z[0], -(v * z[1]));
            x[j][e + 1] = __builtin_fmaf(v, z[0], u * z[1]);
          }
        }
    }
    if (!live) break;
    uint16_t* y = key ? (uint16_t*)a.k_out + (t0 + t1) * a.k_out_token_stride + (h1 - a.q_heads) * a.k_out_head_stride
                      : (uint16_t*)a.q_out + (t0 + t1) * a.q_out_token_stride + h1 * a.q_out_head_stride;
    u32x4 r;
    if (in0) {
#pragma unroll
      for (int j = 0; j < 4; j++) r[j] = pack2(T{}, x[0][2 * j], x[0][2 * j + 1]);
      *(u32x4*)(y + 8 * c0) = r;
    }
    if (in1) {
#pragma unroll
      for (int j = 0; j < 4; j++) r[j] = pack2(T{}, x[1][2 * j], x[1][2 * j + 1]);
      *(u32x4*)(y + 8 * c1) = r;
    }
  }
}

// ---------------------------------------------------------------------------
// Causal attention of packed prompts.
//
// The rows of one (sequence, kv head) are its tokens times the group of q heads
// that share the head: row r = token * group + q head.  A workgroup takes 128 / WK
// rows, 32 a wave (xs_rows32.h; WK waves share them, each with its half of a stage's
// keys, and add up at the end), and walks the keys up to its last row's token in
// stages of 64, through two LDS buffers that loads fill while the other is read.
// Results that are not finite are walked for again (xs_attend.h, passed).
//
// Bound by the matrix cores and the vector units beside them: a stage of a wave at
// head size 128 is 32 products of 32 cycles and some 900 cycles of vector work
// (32 exponentials of 16, then scaling, sums, packing), which two waves a SIMD lay
// side by side: the products run 62 to 64 % of the time at the clock that the power
// leaves (1.8 GHz).  A prompt of 16,384 tokens, 32 q and 8 kv heads of 128: 1,870
// to 2,080 us by card (1,176 to 1,057 TFLOP/s; a large library product reaches 1,334
// to 1,366); 16 prompts of 164 to 4,096: 944 to 1,054 us (977 to 875 TFLOP/s).
// With NaN among the values, walked for again, 4.9 times as long.  One wave's
// exponentials laid by hand beside its own next products, scores of two stages in
// registers, spills: 2,346 us.

// The sequence and the row tile of a workgroup: tiles of the device's valid
// sequences, those with the most keys first, sequences of more than 64 in order.
struct Place {
  int b, tile;  // b < 0: none
  int first, n;
};

template <int ROWS>
XS_DEV Place place(const xs_prompt_attend_args& a, int G, uint32_t want, bool report) {
  const int lane = threadIdx.x & 63;
  Place p = {-1, 0, 0, 0};
  int high = 0;        // the largest entry of start so far
  uint32_t before = 0; // tiles of earlier sequences (2^30 rows at most)
  auto last = [](uint32_t v) { return (uint32_t)__builtin_amdgcn_readlane((int)wave_scan(v), 63); };
  for (int64_t b0 = 0; b0 < a.seqs; b0 += 64) {
    const int64_t b = b0 + lane;
    const bool in = b < a.seqs;
    const int s = in ? a.start[b] : INT32_MIN, e = in ? a.start[b + 1] : 0;
    int top = s;  // inclusive prefix maximum
    const int prev = __shfl_up(s, 1);
    if (__any(in && lane > 0 && prev > s)) {  // (rare)
#pragma unroll
      for (int m = 1; m < 64; m *= 2) {
        const int y = __shfl_up(top, m);
        if (lane >= m) top = max(top, y);
      }
    }
    top = max(top, high);
    const bool good = in && s >= top && e >= s && e <= a.tokens;
    if (report && in) a.seq_status[b] = good ? XS_ROW_OK : XS_ROW_BAD_PARAM;
    if (b0 + 64 < a.seqs) high = __builtin_amdgcn_readlane(top, 63);
    if (p.b >= 0) continue;  // (found; the rest is only reported)
    const uint32_t tiles = good ? (uint32_t)(((int64_t)(e - s) * G + ROWS - 1) / ROWS) : 0u;
    int who = -1, tile = 0;
    if (a.seqs <= 64) {
      // above(L): tiles at a level past L, the level of a tile its place in its sequence
      auto above = [&](uint32_t L) { return last(tiles > L ? tiles - L : 0u); };
      const uint32_t total = above(0);
      if (a.seqs == 1) {
        tile = (int)total - 1 - (int)want;
        if (tile >= 0) who = 0;
      } else if (total > want) {
        uint32_t lo = 0, hi = total;  // the largest L with above(L) > want
        while (hi - lo > 1) {
          const uint32_t mid = (lo + hi) / 2;
          if (above(mid) > want) lo = mid;
          else hi = mid;
        }
        uint64_t have = __ballot(tiles > lo);
        for (uint32_t i = above(lo + 1); i < want; i++) have &= have - 1;
        who = __ffsll((unsigned long long)have) - 1;
        tile = (int)lo;
      }
    } else {
      const uint32_t upto = wave_scan(tiles) + before;
      const uint64_t past = __ballot(upto > want);
      before = (uint32_t)__builtin_amdgcn_readlane((int)upto, 63);
      if (past) {
        who = __ffsll((unsigned long long)past) - 1;
        tile = __builtin_amdgcn_readlane((int)upto, who) - 1 - (int)want;  // the last of a sequence first
      }
    }
    if (who >= 0) {
      p.b = (int)b0 + who;
      p.tile = tile;
      p.first = __builtin_amdgcn_readlane(s, who);
      p.n = __builtin_amdgcn_readlane(e, who) - p.first;
      if (!report) return p;
    }
  }
  return p;
}

// 16 bytes a lane from global memory to LDS (lane i's at to + 16 i), in flight
// until vmcnt says otherwise.  In assembly, so that the compiler, which cannot
// tell the buffers apart, does not wait for it before every read of LDS; what
// reads the bytes waits first (arrived).
XS_DEV void load_lds(const uint16_t* base, uint32_t bytes, u32x4* to) {
  const uint32_t lds = (uint32_t)(uintptr_t)(__attribute__((address_space(3))) void*)to;
  asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %1, %2" ::"s"(lds), "v"(bytes), "s"(base) : "memory", "m0");
}
XS_DEV void arrived() { asm volatile("s_waitcnt vmcnt(0)" ::: "memory"); }

template <typename T, int DP, int WK, bool EXACT>
__global__ __launch_bounds__(64 * NW, DP <= 128 ? 2 : 1) void prompt_kernel(const xs_prompt_attend_args a, float scale) {
  using K = Keys<DP>;
  constexpr int KC = DP / 16, DT = DP / 32, ROWS = 32 * NW / WK, CH = K::CH, STAGE = K::STAGE;
  constexpr int PER = STAGE / (64 * NW);             // of a thread
  static_assert(STAGE % (64 * NW) == 0, "a stage is whole chunks of every thread");
  __shared__ u32x4 lds[2][2][STAGE];                  // [buffer][k, v]
  __shared__ uint16_t marks[2][DT][64 * NW];          // [above, below] a lane's elements that an infinity reaches
  __shared__ int odds;                                // a result is not finite
  const int lane = threadIdx.x & 63, x = lane & 31, g = lane >> 5;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), wr = wave / WK, wk = wave % WK;
  const int G = (int)(a.q_heads / a.kv_heads);
  const int kh = (int)(blockIdx.x % (unsigned)a.kv_heads);
  const Place at = place<ROWS>(a, G, blockIdx.x / (unsigned)a.kv_heads, blockIdx.x == 0 && wave == 0);
  const int b = __builtin_amdgcn_readfirstlane(at.b);
  if (b < 0) return;
  const int n = __builtin_amdgcn_readfirstlane(at.n), t0 = __builtin_amdgcn_readfirstlane(at.first);
  const int R = n * G;
  const int row0 = __builtin_amdgcn_readfirstlane(at.tile) * ROWS, wrow = row0 + 32 * wr;
  const int row = wrow + x, token = min(row, R - 1) / G, head = kh * G + min(row, R - 1) % G;
  const int low = min(wrow, R - 1) / G, top_token = min(wrow + 31, R - 1) / G;  // of the wave's rows
  const int end = min(row0 + ROWS - 1, R - 1) / G + 1;                         // keys that it needs
  const int stages = (end + SK - 1) / SK;
  const bool live = wrow < R;

  // A stage's chunks, each by the lane whose place in LDS it takes.  Chunks past
  // the head's end are zero from the start.
  const uint16_t* kp = (const uint16_t*)a.k + (int64_t)t0 * a.kv_token_stride + kh * a.kv_head_stride;
  const uint16_t* vp = (const uint16_t*)a.v + (int64_t)t0 * a.kv_token_stride + kh * a.kv_head_stride;
  auto clear = [&] {
    if (EXACT) return;
#pragma unroll
    for (int i = 0; i < 4 * PER; i++) (&lds[0][0][0])[i * 64 * NW + threadIdx.x] = (u32x4){0, 0, 0, 0};
    __syncthreads();
  };
  auto fetch = [&](int s) {
    const int64_t o = (int64_t)s * SK * a.kv_token_stride;
    const int last = n - 1 - s * SK;
    const uint32_t stride = 2 * (uint32_t)a.kv_token_stride;
#pragma unroll
    for (int i = 0; i < PER; i++) {
      const int u = i * 64 * NW + threadIdx.x, r = u / CH, ck = u % CH ^ K::turn_k(r), cv = u % CH ^ K::turn_v(r);
      const uint32_t rows = (uint32_t)min(r, last) * stride;
      u32x4* to = &lds[s & 1][0][i * 64 * NW + 64 * wave];
      if (EXACT || 8 * ck < a.head_dim) load_lds(kp + o, rows + 16u * ck, to);
      if (EXACT || 8 * cv < a.head_dim) load_lds(vp + o, rows + 16u * cv, to + STAGE);
    }
  };

  clear();
  fetch(0);
  const Reads<DP> reads(lane);
  if (threadIdx.x == 0) odds = 0;

  Rows32<T, DP, 1> w;
  {
    const uint16_t* p = (const uint16_t*)a.q + (int64_t)(t0 + token) * a.q_token_stride + head * a.q_head_stride;
#pragma unroll
    for (int c = 0; c < KC; c++) {
      const int d = 16 * c + 8 * g;
      w.q[0][c] = row < R && (EXACT || d < a.head_dim) ? *(const u32x4*)(p + d) : (u32x4){0, 0, 0, 0};
    }
  }
  __builtin_amdgcn_s_waitcnt(0x0F70);  // vmcnt(0): the rows' loads too, which the loop would wait for at every stage
  float l, ref;
  f32x16(&o)[DT] = w.o;
#pragma unroll 1
  for (int pass = WALK;; pass++) {
    w.init();
    for (int s = 0; s < stages; s++) {
      arrived();
      __syncthreads();
      if (s + 1 < stages) fetch(s + 1);
      if (pass != WALK) [[unlikely]] {
#pragma unroll
        for (int i = 0; i < PER; i++) {
          u32x4 v = lds[s & 1][1][i * 64 * NW + threadIdx.x];
#pragma unroll
          for (int j = 0; j < 4; j++) v[j] = passed(T{}, v[j], pass);
          lds[s & 1][1][i * 64 * NW + threadIdx.x] = v;
        }
        __syncthreads();
      }
      if (live && s * SK <= top_token) {
        const bool masked = s * SK + SK - 1 > low;
        if constexpr (WK == 1 && DP <= 128) {
          w.template step<2, 1>(reads, lds[s & 1][0], {lds[s & 1][1]}, scale, masked, Upto{token - s * SK - 4 * g});
        } else {
          // a tile of 32 keys at a time: a wave's own, or what the registers hold
#pragma unroll
          for (int i = 0; i < 2 / WK; i++) {
            const int u = WK == 1 ? i : wk;
            w.template step<1, 1>(reads, lds[s & 1][0] + 32 * u * CH, {lds[s & 1][1] + 32 * u * CH}, scale, masked, Upto{token - s * SK - 32 * u - 4 * g});
          }
        }
      }
    }

    l = pair_sum(w.l), ref = l == 0.0f ? NEG_INF : scale < 0.0f ? -w.reference() : w.reference();
    if constexpr (WK == 2) {  // the two waves of the rows add up
      __syncthreads();        // (the last stage's readers)
      f32x16* sum = (f32x16*)&lds[0][0][0] + wr * DT * 64;
      float* stat = (float*)&lds[1][0][0] + wr * 128;
      if (wk == 1) {
#pragma unroll
        for (int d = 0; d < DT; d++) sum[d * 64 + lane] = o[d];
        stat[lane] = ref;
        stat[64 + lane] = l;
      }
      __syncthreads();
      if (wk == 0) {
        const float ref1 = stat[lane], l1 = stat[64 + lane], top = fmaxf(ref, ref1), mag = fabsf(scale);
        // (a half without weights may hold what its masked products left)
        const float f0 = ref == NEG_INF ? 0.0f : __builtin_amdgcn_exp2f((ref - top) * mag), f1 = ref1 == NEG_INF ? 0.0f : __builtin_amdgcn_exp2f((ref1 - top) * mag);
        l = (ref == NEG_INF ? 0.0f : l * f0) + (ref1 == NEG_INF ? 0.0f : l1 * f1);
#pragma unroll
        for (int d = 0; d < DT; d++) {
          const f32x16 y = sum[d * 64 + lane];
#pragma unroll
          for (int i = 0; i < 16; i++) o[d][i] = (ref == NEG_INF ? 0.0f : o[d][i] * f0) + (ref1 == NEG_INF ? 0.0f : y[i] * f1);
        }
        ref = top;
      }
    }
    if (pass == WALK) {
      float z = 0.0f;
#pragma unroll
      for (int d = 0; d < DT; d++)
#pragma unroll
        for (int i = 0; i < 16; i++) z = __builtin_fmaf(o[d][i], 0.0f, z);
      if (wk == 0 && row < R && l > 0.0f && z != z) odds = 1;
      __syncthreads();
      if (!__builtin_amdgcn_readfirstlane(odds)) [[likely]] break;
    } else if (pass == FINITE) {
#pragma unroll
      for (int d = 0; d < DT; d++)
#pragma unroll
        for (int i = 0; i < 16; i++) o[d][i] = marked(o[d][i], marks[0][d][threadIdx.x], marks[1][d][threadIdx.x], i);
      break;
    } else {
#pragma unroll
      for (int d = 0; d < DT; d++) {
        uint32_t m = 0;
#pragma unroll
        for (int i = 15; i >= 0; i--) m = m << 1 | (o[d][i] > 0.0f ? 1u : 0u);
        marks[pass - ABOVE][d][threadIdx.x] = (uint16_t)m;
      }
      __syncthreads();  // (the stages' readers)
    }
    clear();
    fetch(0);
  }
  if (wk == 1 || row >= R) return;
  if (l == 0.0f) {  // every score -inf
#pragma unroll
    for (int d = 0; d < DT; d++) o[d] = fill16(0.0f);
  }
  const float inv = l == 0.0f ? 0.0f : 1.0f / l;
  uint16_t* out = (uint16_t*)a.out + (int64_t)(t0 + token) * a.out_token_stride + head * a.out_head_stride;
#pragma unroll
  for (int d = 0; d < DT; d++)
#pragma unroll
    for (int r = 0; r < 16; r += 4) {
      const int e = 32 * d + 2 * r + 4 * g;
      if (e < a.head_dim)
        *(u32x2*)(out + e) = (u32x2){pack2(T{}, within(T{}, o[d][r] * inv), within(T{}, o[d][r + 1] * inv)),
                                     pack2(T{}, within(T{}, o[d][r + 2] * inv), within(T{}, o[d][r + 3] * inv))};
    }
  if (a.lse && g == 0)
    a.lse[(int64_t)(t0 + token) * a.q_heads + head] =
        l == 0.0f ? NEG_INF : __builtin_fmaf(ref, fabsf(a.scale), LN2 * (__builtin_amdgcn_logf(l) - offset_of(T{})));
}

// No token: only the sequences' statuses.
__global__ __launch_bounds__(64) void prompt_status_kernel(const xs_prompt_attend_args a) { place<64>(a, 1, UINT32_MAX, true); }

}  // namespace xsp

// ---------------------------------------------------------------------------
// Host side.

namespace {

using xs_host::OnDevice;

template <typename T, int LPH>
int rotate_lanes(xs_cache_context* c, const xs_qk_rotate_args& a) {
  const int64_t heads = a.q_heads + a.kv_heads, all = a.tokens * heads;
  constexpr int64_t per = xsp::RT / LPH;
  // as many passes as leave every CU eight workgroups, of 16 tokens at most (their
  // angles fill LDS)
  const int64_t want = std::min(all / (per * 8 * c->n_cu), 16 * heads / per);
  const int passes = (int)std::max<int64_t>(1, std::min<int64_t>(xsp::ROT_PASSES, want));
  const int64_t span = per * passes, grid = (all + span - 1) / span;
  if (!xs_host_launch_fits(grid, xsp::RT)) return XS_ERR_CAPACITY;
  const int64_t tokens = std::min(a.tokens, (span + heads - 1) / heads + 1);
  const size_t lds = 8 * (size_t)(a.head_dim + tokens * (a.rot_dim / 2));
  hipLaunchKernelGGL((xsp::rotate_kernel<T, LPH>), dim3((unsigned)grid), dim3(xsp::RT), lds, c->stream, a, passes);
  return hipGetLastError() == hipSuccess ? XS_OK : XS_ERR_HIP;
}

template <typename T>
int rotate_dim(xs_cache_context* c, const xs_qk_rotate_args& a) {
  if (a.head_dim <= 16) return rotate_lanes<T, 1>(c, a);
  if (a.head_dim <= 32) return rotate_lanes<T, 2>(c, a);
  if (a.head_dim <= 64) return rotate_lanes<T, 4>(c, a);
  if (a.head_dim <= 128) return rotate_lanes<T, 8>(c, a);
  return rotate_lanes<T, 16>(c, a);
}

template <typename T, int DP, int WK, bool EXACT>
int prompt_run(xs_cache_context* c, const xs_prompt_attend_args& a) {
  const int64_t rows = a.tokens * (a.q_heads / a.kv_heads), tile = 32 * xst::NW / WK;
  // no more tiles than this, whatever the sequences' lengths: each leaves less than one
  const int64_t grid = (rows / tile + std::min(a.seqs, a.tokens)) * a.kv_heads;
  if (!xs_host_launch_fits(grid, 64 * xst::NW)) return XS_ERR_CAPACITY;
  hipLaunchKernelGGL((xsp::prompt_kernel<T, DP, WK, EXACT>), dim3((unsigned)grid), dim3(64 * xst::NW), 0, c->stream, a, a.scale * xst::LOG2E);
  return hipGetLastError() == hipSuccess ? XS_OK : XS_ERR_HIP;
}

// Rows of 128 a workgroup, or of 64 where those do not fill the device (1,024
// tokens 29 and 23 us, 2,048 tokens 55 and 59; heads of 256, one workgroup a CU,
// gain nothing by it: 100 tokens 17 and 20).
template <typename T, int DP, bool EXACT>
int prompt_rows(xs_cache_context* c, const xs_prompt_attend_args& a) {
  if constexpr (DP <= 128) {
    if (a.tokens * a.q_heads < c->n_cu * 2 * 128) return prompt_run<T, DP, 2, EXACT>(c, a);
  }
  return prompt_run<T, DP, 1, EXACT>(c, a);
}

template <typename T, int DP>
int prompt_exact(xs_cache_context* c, const xs_prompt_attend_args& a) {
  return a.head_dim == DP ? prompt_rows<T, DP, true>(c, a) : prompt_rows<T, DP, false>(c, a);
}

template <typename T>
int prompt_dim(xs_cache_context* c, const xs_prompt_attend_args& a) {
  if (a.head_dim <= 64) return prompt_exact<T, 64>(c, a);
  if (a.head_dim <= 96) return prompt_exact<T, 96>(c, a);
  if (a.head_dim <= 128) return prompt_exact<T, 128>(c, a);
  return prompt_exact<T, 256>(c, a);
}

}  // namespace

extern "C" {

int xs_qk_rotate(xs_cache_context* c, const xs_qk_rotate_args* in) {
  const int rc = c ? xs_host_check_rotate(in) : XS_ERR_ARG;
  if (rc) return rc;
  if (in->tokens == 0 || in->q_heads + in->kv_heads == 0) return XS_OK;
  const OnDevice on(c->device);
  if (!on.ok) return XS_ERR_HIP;
  xs_qk_rotate_args a = *in;  // (whether there is a norm is for the sides that have heads to say)
  if (a.q_heads == 0) a.q_weight = nullptr;
  if (a.kv_heads == 0) a.k_weight = nullptr;
  if (a.dtype == XS_BF16) return rotate_dim<xst::Bf16>(c, a);
  return rotate_dim<xst::F16>(c, a);
}

int xs_prompt_attend(xs_cache_context* c, const xs_prompt_attend_args* in) {
  const int rc = c ? xs_host_check_prompt(in) : XS_ERR_ARG;
  if (rc) return rc;
  if (in->seqs == 0) return XS_OK;
  const OnDevice on(c->device);
  if (!on.ok) return XS_ERR_HIP;
  if (in->tokens == 0) {
    hipLaunchKernelGGL(xsp::prompt_status_kernel, dim3(1), dim3(64), 0, c->stream, *in);
    return hipGetLastError() == hipSuccess ? XS_OK : XS_ERR_HIP;
  }
  if (in->dtype == XS_BF16) return prompt_dim<xst::Bf16>(c, *in);
  return prompt_dim<xst::F16>(c, *in);
}

}  // extern "C"
