// xs_cache8.hip -- a cache of keys and values held in 8 bits (MI355X, gfx950):
// rows appended to it, and a tree's attention over it.
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

namespace xs8 {

using namespace xst;

constexpr int EXP_MIN = -100;  // the least exponent of a scale: 448 * 2^-100 is 0 to any use

// 2^e as f32, for the exponents that occur (a byte of another range gives some
// power of two, not a fault).
XS_DEV float pow2(int e) { return __uint_as_float((uint32_t)min(max(e + 127, 1), 254) << 23); }

// ---------------------------------------------------------------------------
// Append.
//
// One workgroup a block of 32 slots of one head, keys and values.  A thread takes
// 16 elements of up to two rows of each; the largest finite magnitude is a
// maximum over bit patterns.  The block's e is the least with amax <= 448 * 2^e:
// with amax = m * 2^x, m in [1/2, 1), that is x - 9, and one more where m > 7/8
// (448 is 7/8 of 2^9).  A power of two loses nothing where the element type is
// itself a float, but for the lowest of its subnormals, and makes both the
// products and a later change of the scale exact.  Bound by reading the rows and
// writing the bytes: 4 prompts of 328 to 8,192 rows of 8 heads of 128 (112 MB) in
// 25 us; a step's 5 rows for each of 16 sequences 4.5 us, latency.

constexpr int AB = 256;  // threads

XS_DEV int exponent_of(float amax) {
  if (amax == 0.0f) return EXP_MIN;
  const int e = __builtin_amdgcn_frexp_expf(amax) - 9 + (__builtin_amdgcn_frexp_mantf(amax) > 0.875f ? 1 : 0);
  return max(e, EXP_MIN);
}

// Four values to bytes.
XS_DEV uint32_t bytes4(float a, float b, float c, float d) {
  int r = __builtin_amdgcn_cvt_pk_fp8_f32(a, b, 0, false);
  return (uint32_t)__builtin_amdgcn_cvt_pk_fp8_f32(c, d, r, true);
}

template <typename T>
__global__ __launch_bounds__(AB) void append_kernel(const xs_cache_append8_args a, int blocks) {
  __shared__ uint32_t tops[2][AB / 64];
  __shared__ int bads;
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
  const int blk = (int)(blockIdx.x % (unsigned)blocks);
  const int64_t bh = blockIdx.x / (unsigned)blocks;
  const int kh = (int)(bh % a.kv_heads), b = (int)(bh / a.kv_heads);
  const int len = a.len[b];
  const int64_t fresh_rows = a.start ? a.tokens : a.rows;
  int64_t row0 = 0, n = a.rows;
  bool bad = len < 0 || len > a.capacity;
  if (a.start) {
    row0 = a.start[b];
    n = a.start[b + 1] - row0;
    bad |= row0 < 0 || row0 + n > fresh_rows;
  } else if (a.n_path) {
    n = a.n_path[b];
  }
  bad |= n < 0 || n > a.rows;
  if (!bad && a.path) {
    if (tid == 0) bads = 0;
    __syncthreads();
    for (int64_t i = tid; i < n; i += AB) {
      const int p = a.path[b * a.path_ld + i];
      if (p < 0 || p >= fresh_rows) bads = 1;
    }
    __syncthreads();
    bad = bads;
  }
  const int status = bad ? XS_ROW_BAD_PARAM : len + n > a.capacity ? XS_ROW_CACHE_FULL : XS_ROW_OK;
  if (kh == 0 && blk == 0 && tid == 0) {
    a.seq_status[b] = status;
    a.new_len[b] = status == XS_ROW_OK ? len + (int)n : len;
  }
  if (status != XS_ROW_OK) return;
  const int64_t slot0 = (int64_t)(len / XS_CACHE8_BLOCK + blk) * XS_CACHE8_BLOCK;  // of the block
  if (slot0 >= len + n) return;
  const int lo = (int)max(len - slot0, (int64_t)0), hi = (int)min(len + n - slot0, (int64_t)XS_CACHE8_BLOCK);  // its new rows
  const int64_t eat = bh * a.cache.exp_ld + slot0 / XS_CACHE8_BLOCK;
  const int old[2] = {lo > 0 ? a.cache.k_exp[eat] - 127 : EXP_MIN, lo > 0 ? a.cache.v_exp[eat] - 127 : EXP_MIN};

  const int parts = a.head_dim / 16;
  u32x4 raw[2][2][2];  // [keys, values][piece][16 bytes]
  uint32_t top[2] = {0, 0};
#pragma unroll
  for (int j = 0; j < 2; j++) {
    const int u = j * AB + tid, r = u / parts, d = u % parts * 16;
    if (r < lo || r >= hi) continue;
    const int64_t i = slot0 + r - len;
    const int64_t from = a.path ? a.path[b * a.path_ld + i] : row0 + i;
    const int64_t at = (a.start ? 0 : b * a.fresh.seq_stride) + from * a.fresh.slot_stride + kh * a.fresh.head_stride + d;
#pragma unroll
    for (int w = 0; w < 2; w++) {
      const u32x4* p = (const u32x4*)((const uint16_t*)(w ? a.fresh.v : a.fresh.k) + at);
      raw[w][j][0] = p[0];
      raw[w][j][1] = p[1];
    }
  }
#pragma unroll
  for (int j = 0; j < 2; j++) {
    const int r = (j * AB + tid) / parts;
    if (r < lo || r >= hi) continue;
#pragma unroll
    for (int w = 0; w < 2; w++)
#pragma unroll
      for (int h = 0; h < 2; h++)
#pragma unroll
        for (int e = 0; e < 4; e++) {
          const uint32_t x = raw[w][j][h][e] & 0x7FFFu, y = (raw[w][j][h][e] >> 16) & 0x7FFFu;
          top[w] = max(top[w], max(x < inf_of(T{}) ? x : 0u, y < inf_of(T{}) ? y : 0u));
        }
  }
#pragma unroll
  for (int w = 0; w < 2; w++) {
#pragma unroll
    for (int m = 1; m < 64; m *= 2) top[w] = max(top[w], (uint32_t)__shfl_xor((int)top[w], m));
    if (lane == 0) tops[w][wave] = top[w];
  }
  __syncthreads();
#pragma unroll
  for (int w = 0; w < 2; w++) {
#pragma unroll
    for (int i = 0; i < AB / 64; i++) top[w] = max(top[w], tops[w][i]);
    const int e = max(exponent_of(T::widen((uint16_t)top[w])), old[w]);
    const float inv = pow2(-e), shrink = pow2(old[w] - e);
    uint8_t* cache = (w ? a.cache.v : a.cache.k) + b * a.cache.seq_stride + kh * a.cache.head_stride;
#pragma unroll
    for (int j = 0; j < 2; j++) {
      const int u = j * AB + tid, r = u / parts, d = u % parts * 16;
      u32x4* to = (u32x4*)(cache + (slot0 + r) * a.cache.slot_stride + d);
      if (r >= lo && r < hi) {
        u32x4 y;
#pragma unroll
        for (int i = 0; i < 4; i++) {
          const uint32_t p = raw[w][j][i / 2][2 * (i % 2)], q = raw[w][j][i / 2][2 * (i % 2) + 1];
          y[i] = bytes4(T::widen((uint16_t)p) * inv, T::widen((uint16_t)(p >> 16)) * inv, T::widen((uint16_t)q) * inv,
                        T::widen((uint16_t)(q >> 16)) * inv);
        }
        *to = y;
      } else if (r < lo && e > old[w]) {  // slots that the block held, at its new scale
        u32x4 y = *to;
#pragma unroll
        for (int i = 0; i < 4; i++) {
          const f32x2 p = __builtin_amdgcn_cvt_pk_f32_fp8((int)y[i], false), q = __builtin_amdgcn_cvt_pk_f32_fp8((int)y[i], true);
          y[i] = bytes4(p[0] * shrink, p[1] * shrink, q[0] * shrink, q[1] * shrink);
        }
        *to = y;
      }
    }
    if (tid == 0) (w ? a.cache.v_exp : a.cache.k_exp)[eat] = (uint8_t)(e + 127);
  }
}

// ---------------------------------------------------------------------------
// Attention.
//
// That of xs_attend.h with keys and values as bf16, which holds byte * 2^e
// exactly: a block of 32 keys is one block of the cache, its scales two uniform
// exponents, applied by the conversion itself.  f16 queries and fresh values, and
// the weights of f16 calls are sums of two bf16 (a float of 11 bits is one
// exactly, a weight to 16 bits), each part a product of its own.  The tree's own
// scores are products of f16 as they stand: parts of an infinity times parts of a
// query would not add up to it (0 times -inf, or -inf and +inf).
// A lane loads 16 bytes of a key: elements 64 c + 16 g + 8 h .. + 8 are chunk
// 2 c + h of the products, for queries and fresh keys too.  Bound by the one read
// of the cache up to 16 rows a head: decoding 32 sequences of 327 to 8,192 slots, 8
// kv heads of 128 (302 MB), 77 to 80 us by card, of which the join of the splits takes
// 5; without starts and ends the keys come at 5.2 to 5.9 TB/s.

struct E4m3 {};  // (weights carry no power of two)
XS_DEV constexpr float offset_of(E4m3) { return 0.0f; }

template <typename T> struct Parts { static constexpr int N = 1; };
template <> struct Parts<F16> { static constexpr int N = 2; };

// Eight elements of the type as bf16: themselves, or a sum of two.
XS_DEV void split8(Bf16, u32x4 r, u32x4 (&y)[1]) { y[0] = r; }
XS_DEV void split8(F16, u32x4 r, u32x4 (&y)[2]) {
#pragma unroll
  for (int i = 0; i < 4; i++) {
    const float a = F16::widen((uint16_t)r[i]), b = F16::widen((uint16_t)(r[i] >> 16));
    y[0][i] = pack2(Bf16{}, a, b);
    const float c = Bf16::widen((uint16_t)y[0][i]), d = Bf16::widen((uint16_t)(y[0][i] >> 16));
    // (what is not finite is all in the first)
    y[1][i] = pack2(Bf16{}, fabsf(a) < -NEG_INF ? a - c : 0.0f, fabsf(b) < -NEG_INF ? b - d : 0.0f);
  }
}

XS_DEV uint32_t wide2(uint32_t r, float scale, bool high) {
  return __builtin_bit_cast(uint32_t, high ? __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(r, scale, true)
                                           : __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(r, scale, false));
}

template <typename T, int DP, int RT>
struct Tile {
  using S = Shape<DP, RT>;
  static constexpr int N = Parts<T>::N;
  Wave<Bf16, DP, RT> w;                 // (its q is not used)
  u32x4 q[N][RT][S::KC];
};

// The weights of a row tile from its scores, as parts.
template <typename T, int DP, int RT>
XS_DEV void weights8(Tile<T, DP, RT>& z, int t, const float (&x)[8], u32x4 (&pf)[Parts<T>::N][RT]) {
  if constexpr (Parts<T>::N == 1) {
    pf[0][t] = z.w.weights(t, x);
  } else {
    float p[8];
#pragma unroll
    for (int e = 0; e < 8; e++) p[e] = __builtin_amdgcn_exp2f(x[e]);
    z.w.l[t] += ((p[0] + p[1]) + (p[2] + p[3])) + ((p[4] + p[5]) + (p[6] + p[7]));
#pragma unroll
    for (int i = 0; i < 4; i++) {
      pf[0][t][i] = pack2(Bf16{}, p[2 * i], p[2 * i + 1]);
      pf[1][t][i] = pack2(Bf16{}, p[2 * i] - Bf16::widen((uint16_t)pf[0][t][i]), p[2 * i + 1] - Bf16::widen((uint16_t)(pf[0][t][i] >> 16)));
    }
  }
}

// The weights of 32 keys, from products of type M with the first QN parts of the
// queries: keys(u, c) is chunk c of 16 of them, again(u, c) the same formed anew
// where references move.
template <typename T, int DP, int RT, bool MASKED, typename M, int QN, typename Keys, typename Again>
XS_DEV void softmax8(Tile<T, DP, RT>& z, float scale, const uint32_t* on, u32x4 (&pf)[Parts<T>::N][RT], Keys keys, Again again) {
  using S = Shape<DP, RT>;
  f32x4 s[RT][2];
#pragma unroll
  for (int t = 0; t < RT; t++) s[t][0] = s[t][1] = z.w.start(t);
#pragma unroll
  for (int c = 0; c < S::KC; c++)
#pragma unroll
    for (int u = 0; u < 2; u++) {
      const u32x4 k = keys(u, c);
#pragma unroll
      for (int t = 0; t < RT; t++)
#pragma unroll
        for (int n = 0; n < QN; n++) s[t][u] = mfma(M{}, k, z.q[n][t][c], s[t][u]);
    }
#pragma unroll
  for (int t = 0; t < RT; t++) {
    float x[8];
    const float top = z.w.template scaled<MASKED>(s[t], scale, MASKED ? on[t] : 0u, x);
    if (__any(z.w.passes(t, top))) [[unlikely]] {
      const bool far = __any(z.w.passes(t, top) && z.w.minus(z.w.c[t]) != 0.0f);
      if (far) [[unlikely]] {
        s[t][0] = s[t][1] = (f32x4){0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
        for (int c = 0; c < S::KC; c++)
#pragma unroll
          for (int u = 0; u < 2; u++) {
            const u32x4 k = again(u, c);
#pragma unroll
            for (int n = 0; n < QN; n++) s[t][u] = mfma(M{}, k, z.q[n][t][c], s[t][u]);
            __builtin_amdgcn_sched_barrier(0);  // (one chunk in registers at a time)
          }
      }
      z.w.template rebase<MASKED>(t, s[t], far, scale, MASKED ? on[t] : 0u, x);
    }
    weights8<T, DP, RT>(z, t, x, pf);
  }
}

// A block of the cache as it lies there, and the bytes of its exponents.
template <int DP>
struct Raw {
  using S = Shape<DP, 1>;
  u32x4 k[2][S::KC / 2];
  uint32_t v[8][S::VH][S::VE / 4];
  uint32_t ke, ve;
};

// Load block i; of the last, `limit` slots are in use.  Rows' bases are uniform,
// so that a lane keeps two 32-bit offsets for all of them (made new to the
// compiler's eyes, else it keeps sixteen sums of 64 bits).
template <int DP, bool EXACT, bool MASKED>
XS_DEV void load_keys8(Raw<DP>& r, const xs_kv8& c8, int64_t at, int64_t eat, int i, int limit, int D) {
  using S = Shape<DP, 1>;
  const int lane = threadIdx.x & 63, x = lane & 15, g = lane >> 4;
  const uint32_t stride = (uint32_t)c8.slot_stride;
  uint32_t ko = x * stride + 16 * g;
  asm volatile("" : "+v"(ko));
  const uint8_t* kp = c8.k + (at + (int64_t)i * KB * c8.slot_stride);
  r.ke = c8.k_exp[eat + i];
#pragma unroll
  for (int u = 0; u < 2; u++)
#pragma unroll
    for (int c = 0; c < S::KC / 2; c++) {
      const uint32_t off = MASKED ? min(16 * u + x, limit - 1) * stride + 16 * g : ko;
      const uint8_t* p = (kp + (MASKED ? 0 : (int64_t)(16 * u) * stride) + 64 * c) + off;
      r.k[u][c] = EXACT || 64 * c + 16 * g < D ? *(const u32x4*)p : (u32x4){0, 0, 0, 0};
    }
}
template <int DP, bool EXACT, bool MASKED>
XS_DEV void load_values8(Raw<DP>& r, const xs_kv8& c8, int64_t at, int64_t eat, int i, int limit, int D) {
  using S = Shape<DP, 1>;
  const int lane = threadIdx.x & 63, x = lane & 15, g = lane >> 4;
  const uint32_t stride = (uint32_t)c8.slot_stride;
  uint32_t vo = 4 * g * stride + S::VE * x;
  asm volatile("" : "+v"(vo));
  const uint8_t* vp = c8.v + (at + (int64_t)i * KB * c8.slot_stride);
  r.ve = c8.v_exp[eat + i];
#pragma unroll
  for (int e = 0; e < 8; e++) {
    const int slot = 4 * g + (e & 3) + 16 * (e >> 2);
#pragma unroll
    for (int h = 0; h < S::VH; h++) {
      const int d = EXACT ? 128 * h + S::VE * x : min(128 * h + S::VE * x, D - S::VE);  // (products of elements past the head's are never stored)
      const uint8_t* p;
      if constexpr (MASKED) p = vp + (uint32_t)(min(slot, limit - 1) * stride + d);
      else if constexpr (EXACT) p = (vp + (int64_t)((e & 3) + 16 * (e >> 2)) * stride + 128 * h) + vo;
      else p = vp + (int64_t)((e & 3) + 16 * (e >> 2)) * stride + (uint32_t)(4 * g * stride + d);
      if constexpr (S::VE == 8) {
        const u32x2 y = *(const u32x2*)p;
        r.v[e][h][0] = y[0];
        r.v[e][h][1] = y[1];
      } else {
        r.v[e][h][0] = *(const uint32_t*)p;
      }
      if (MASKED && slot >= limit) {
#pragma unroll
        for (int w = 0; w < S::VE / 4; w++) r.v[e][h][w] = 0;  // count for nothing, whatever they hold
      }
    }
  }
}

// The weights of a block of the cache.
template <typename T, int DP, int RT, bool MASKED>
XS_DEV void cache_weights(Tile<T, DP, RT>& z, const Raw<DP>& r, float scale, const uint32_t* on, u32x4 (&pf)[Parts<T>::N][RT]) {
  const float kscale = pow2((int)r.ke - 127);
  auto widen = [](uint32_t a, uint32_t b, float s) { return (u32x4){wide2(a, s, false), wide2(a, s, true), wide2(b, s, false), wide2(b, s, true)}; };
  softmax8<T, DP, RT, MASKED, Bf16, Parts<T>::N>(
      z, scale, on, pf, [&](int u, int c) { return widen(r.k[u][c / 2][2 * (c % 2)], r.k[u][c / 2][2 * (c % 2) + 1], kscale); },
      [&](int u, int c) {
        uint32_t a = r.k[u][c / 2][2 * (c % 2)], b = r.k[u][c / 2][2 * (c % 2) + 1];
        asm volatile("" : "+v"(a), "+v"(b));  // (not the first products' operands, kept)
        return widen(a, b, kscale);
      });
}

// Its second product, of values as `pass` takes them (xs_attend.h, passed).
template <typename T, int DP, int RT>
XS_DEV void cache_product(Tile<T, DP, RT>& z, const Raw<DP>& r, const u32x4 (&pf)[Parts<T>::N][RT], int pass) {
  using S = Shape<DP, RT>;
  const float vscale = pow2((int)r.ve - 127);
#pragma unroll
  for (int h = 0; h < S::VH; h++)
#pragma unroll
    for (int j = 0; j < S::VE; j += 2) {  // two fragments: element j and j + 1 of the lane's eight keys
      uint32_t y[8];
#pragma unroll
      for (int e = 0; e < 8; e++) y[e] = wide2(r.v[e][h][j / 4], vscale, j / 2 % 2);
      if (pass != WALK) {
#pragma unroll
        for (int e = 0; e < 8; e++) y[e] = passed(Bf16{}, y[e], pass);
      }
      u32x4 a[2];
#pragma unroll
      for (int i = 0; i < 4; i++) {
        a[0][i] = __builtin_amdgcn_perm(y[2 * i + 1], y[2 * i], 0x05040100u);
        a[1][i] = __builtin_amdgcn_perm(y[2 * i + 1], y[2 * i], 0x07060302u);
      }
#pragma unroll
      for (int w = 0; w < 2; w++)
#pragma unroll
        for (int t = 0; t < RT; t++)
#pragma unroll
          for (int n = 0; n < Parts<T>::N; n++) z.w.o[t][h * S::VE + j + w] = mfma(Bf16{}, a[w], pf[n][t], z.w.o[t][h * S::VE + j + w]);
    }
}

// A block of the tree's own keys, in the inputs' type, as the queries are here
// (z.q[0]).
template <typename T, int DP, int RT, bool EXACT>
XS_DEV void tree_block(Tile<T, DP, RT>& z, const uint16_t* kp, const uint16_t* vp, int64_t stride, int key0, int limit, int D, float scale,
                       const uint32_t* on, int pass) {
  using S = Shape<DP, RT>;
  constexpr int N = Parts<T>::N;
  const int lane = threadIdx.x & 63, x = lane & 15, g = lane >> 4;
  u32x4 pf[N][RT];
  auto keys = [&](int u, int c) {
    const int key = min(key0 + 16 * u + x, limit - 1), d = 64 * (c / 2) + 16 * g + 8 * (c % 2);
    return EXACT || d < D ? *(const u32x4*)(kp + key * stride + d) : (u32x4){0, 0, 0, 0};
  };
  softmax8<T, DP, RT, true, T, 1>(z, scale, on, pf, keys, keys);
  __builtin_amdgcn_sched_barrier(0);  // (the values' registers not beside the keys')
  uint32_t v[N][8][S::VH][S::VE / 2];
#pragma unroll
  for (int e = 0; e < 8; e++) {
    const int slot = key0 + 4 * g + (e & 3) + 16 * (e >> 2), key = min(slot, limit - 1);
#pragma unroll
    for (int h = 0; h < S::VH; h++) {
      int d = 128 * h + S::VE * x;
      if (!EXACT) d = min(d, D - S::VE);
      u32x4 r = {0, 0, 0, 0};
      if constexpr (S::VE == 8) {
        r = *(const u32x4*)(vp + key * stride + d);
      } else {
        const u32x2 y = *(const u32x2*)(vp + key * stride + d);
        r[0] = y[0];
        r[1] = y[1];
      }
#pragma unroll
      for (int i = 0; i < S::VE / 2; i++) {
        if (slot >= limit) r[i] = 0;
        if (pass != WALK) r[i] = passed(T{}, r[i], pass);
      }
      u32x4 y[N];
      split8(T{}, r, y);
#pragma unroll
      for (int n = 0; n < N; n++)
#pragma unroll
        for (int i = 0; i < S::VE / 2; i++) v[n][e][h][i] = y[n][i];
    }
  }
#pragma unroll
  for (int m = 0; m < N; m++)
#pragma unroll
    for (int n = 0; n < N; n++) accumulate(z.w, v[m], pf[n]);
}

// How a call is cut.  The keys are counted in units (blocks of 32, stages of 64),
// and a sequence of u units is split in u / share of them, rounded up.  The share
// is one for all sequences, so that long and short ones' workgroups end together:
// the smallest that leaves no more splits than `room` for each head and row tile:
// as many as the device holds at once, so that no workgroup starts when the others
// end (as many splits for every sequence instead, 32 of 327 to 8,192 slots: 87 us for
// 81), but no more than a join takes of one sequence (SPLITS: of one kv head of 128,
// single rows then fill a third of the device) or than the context has partial
// results for.  The lengths are on the device, so every workgroup finds the share and
// its place among the sequences itself.
struct Cut8 {
  int32_t G, tiles, units, room;  // units: (sequence, split) that the launch has; room 0: nothing is split
  float scale;
  float* part;                    // [units, kv heads, tiles] partial results
  int32_t* plan;                  // [seqs] first unit << 16 and splits, for the join
};
struct Place8 {
  int b, split, share, n;  // b < 0: none; n: splits of the sequence
  int len, nodes;          // of the sequence; nodes < 0: bad
};

// UNIT keys a unit, shares of LEAST units at least, sequences of up to WHOLE of
// them in one piece.
template <int UNIT>
XS_DEV int units_of(const Seq& sq) { return sq.bad ? 0 : (sq.len + UNIT - 1) / UNIT + (sq.n + UNIT - 1) / UNIT; }

template <int UNIT, int LEAST, int WHOLE>
XS_DEV Place8 place8(const xs_tree_attend_args& a, const Cut8& cut, int want) {
  const int lane = threadIdx.x & 63, seqs = (int)a.seqs;
  if (cut.room == 0) {
    if (want >= seqs) return {-1, 0, 1, 1, 0, 0};
    const Seq sq(a, want);
    return {want, 0, 1, 1, sq.len, sq.bad ? -1 : sq.n};
  }
  uint32_t u = 0;  // of the lane's sequence (of the last 64)
  int len = 0, nodes = -1;
  auto load = [&](int b0) {
    u = 0;
    if (b0 + lane >= seqs) return;
    const Seq sq(a, b0 + lane);
    u = (uint32_t)units_of<UNIT>(sq);
    len = sq.len;
    nodes = sq.bad ? -1 : sq.n;
  };
  auto last = [](uint32_t v) { return (uint32_t)__builtin_amdgcn_readlane((int)wave_scan(v), 63); };
  auto splits = [&](int b0, uint32_t share) { return b0 + lane >= seqs ? 0u : u <= WHOLE ? 1u : (u + share - 1) / share; };
  uint32_t all = 0;  // (at most 256 sequences of 2^23 units and some)
  for (int b0 = 0; b0 < seqs; b0 += 64) {
    load(b0);
    all += last(u);
  }
  const uint32_t room = (uint32_t)cut.room;
  uint32_t share = max((uint32_t)LEAST, (all + room - 1) / room);
  if (room > (uint32_t)seqs) {
    uint32_t high = max(share, (all + room - seqs - 1) / (room - seqs));  // (a share too many for each sequence fits)
    while (share < high) {
      const uint32_t mid = (share + high) / 2;
      uint32_t sum = 0;
      for (int b0 = 0; b0 < seqs; b0 += 64) {
        if (seqs > 64) load(b0);
        sum += last(splits(b0, mid));
      }
      if (sum <= room) high = mid;
      else share = mid + 1;
    }
  }
  uint32_t before = 0;
  for (int b0 = 0; b0 < seqs; b0 += 64) {
    if (seqs > 64) load(b0);
    const uint32_t n = splits(b0, share), upto = wave_scan(n) + before;
    const uint64_t hit = __ballot(b0 + lane < seqs && upto > (uint32_t)want);
    before = (uint32_t)__builtin_amdgcn_readlane((int)upto, 63);
    if (!hit) continue;
    const int who = __ffsll((unsigned long long)hit) - 1, parts = __builtin_amdgcn_readlane((int)n, who);
    const int first = __builtin_amdgcn_readlane((int)upto, who) - parts;
    return {b0 + who, want - first, (int)share, parts, __builtin_amdgcn_readlane(len, who), __builtin_amdgcn_readlane(nodes, who)};
  }
  return {-1, 0, 1, 1, 0, 0};
}

// Workgroup i's part: groups of eight (kv head, sequence, split), each group's row
// tiles on one XCD (workgroup index mod 8), which then reads their keys once.  A
// head's units one after the other: with a unit's heads side by side, where a
// slot's heads lie side by side too, every XCD reads one head's 128 bytes of every
// 1,024, and 32 sequences of 4,608 slots take 84 us for 74.
XS_DEV void deal(const Cut8& cut, int* tile, int* kh, int* unit) {
  const int i = blockIdx.x >> 3, group = i / cut.tiles * 8 + (blockIdx.x & 7);
  *tile = i % cut.tiles;
  *unit = group % cut.units;
  *kh = group / cut.units;
}

// Up to 16 RT rows a workgroup, whose waves split the keys and add up through
// LDS.
template <typename T, int DP, int RT, bool EXACT>
__global__ __launch_bounds__(64 * NW, DP * RT <= 64 ? 4 : DP * RT <= 128 ? 3 : DP * RT <= 256 ? 2 : 1) void attend8_kernel(
    const xs_tree_attend_args a, const xs_kv8 c8, const Cut8 cut) {
  using S = Shape<DP, RT>;
  __shared__ float stat[NW][RT][2][16];
  __shared__ f32x4 sum[NW][RT][S::NF][64];
  const int lane = threadIdx.x & 63, x = lane & 15, g = lane >> 4;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  int tile, kh, unit;
  deal(cut, &tile, &kh, &unit);
  if (kh >= (int)a.kv_heads) return;
  const Place8 pl = place8<KB, 2 * NW, 4 * NW>(a, cut, unit);
  const int b = __builtin_amdgcn_readfirstlane(pl.b), split = __builtin_amdgcn_readfirstlane(pl.split);
  const int splits = __builtin_amdgcn_readfirstlane(pl.n);
  if (b < 0) return;
  const int share = __builtin_amdgcn_readfirstlane(pl.share), bh = b * (int)a.kv_heads + kh;
  const int len = __builtin_amdgcn_readfirstlane(pl.len), n = __builtin_amdgcn_readfirstlane(pl.nodes);
  if (split == 0 && tile == 0 && kh == 0 && threadIdx.x == 0) {
    a.seq_status[b] = n < 0 ? XS_ROW_BAD_PARAM : XS_ROW_OK;
    if (cut.room) cut.plan[b] = unit << 16 | splits;
  }
  const int R = n * cut.G, row0 = tile * RT * 16;
  const int cached = (len + KB - 1) / KB, total = cached + (n + KB - 1) / KB;
  const int first = split * share, last = splits == 1 ? total : min(first + share, total);  // (one split: share says nothing)
  if (row0 >= R || first >= total) return;  // (nodes below 0 too)

  // the first keys and values leave before the queries
  const int64_t at = b * c8.seq_stride + kh * c8.head_stride, eat = (int64_t)bh * c8.exp_ld;
  int i = first + wave;
  const int end = min(last, len / KB);
  Raw<DP> r;
  if (i < end) {
    load_keys8<DP, EXACT, false>(r, c8, at, eat, i, KB, a.head_dim);
    load_values8<DP, EXACT, false>(r, c8, at, eat, i, KB, a.head_dim);
  }
  const int parent = parent_of(a, b);
  Tile<T, DP, RT> z;
  z.w.init();
  auto query = [&](int row) {
    const int r = min(row, R - 1);  // (rows past the last are not stored)
    return (const uint16_t*)a.q + b * a.q_seq_stride + r / cut.G * a.q_node_stride + (kh * cut.G + r % cut.G) * a.q_head_stride + 16 * g;
  };
  auto chunk = [&](const uint16_t* p, int c) {
    const int d = 64 * (c / 2) + 8 * (c % 2);
    return EXACT || d + 16 * g < a.head_dim ? *(const u32x4*)(p + d) : (u32x4){0, 0, 0, 0};
  };
  auto queries = [&]() __attribute__((always_inline)) {
#pragma unroll
    for (int t = 0; t < RT; t++) {
      const uint16_t* p = query(row0 + 16 * t + x);
#pragma unroll
      for (int c = 0; c < S::KC; c++) {
        u32x4 y[Tile<T, DP, RT>::N];
        split8(T{}, chunk(p, c), y);
#pragma unroll
        for (int m = 0; m < Tile<T, DP, RT>::N; m++) z.q[m][t][c] = y[m];
      }
    }
  };
  queries();

  // whole blocks of the cache: a block's registers take the next one's keys once
  // its scores are formed, and the next one's values after its second product (a
  // wave's last one again after it: a branch round the loads would have the
  // products wait for all of them)
#pragma unroll 1
  for (; i < end; i += NW) {
    u32x4 pf[Parts<T>::N][RT];
    cache_weights<T, DP, RT, false>(z, r, cut.scale, nullptr, pf);
    const int next = min(i + NW, end - 1);
    __builtin_amdgcn_sched_barrier(0);  // (the loads leave here, not where the last ones have come)
    load_keys8<DP, EXACT, false>(r, c8, at, eat, next, KB, a.head_dim);
    __builtin_amdgcn_sched_barrier(0);
    cache_product<T, DP, RT>(z, r, pf, WALK);
    __builtin_amdgcn_sched_barrier(0);
    load_values8<DP, EXACT, false>(r, c8, at, eat, next, KB, a.head_dim);
    __builtin_amdgcn_sched_barrier(0);
  }
  // its last one, and the tree's
  const uint64_t sees = ancestors(parent, n);
  uint64_t mine[RT];  // what the lane's rows see of the tree
#pragma unroll
  for (int t = 0; t < RT; t++) {
    const int row = row0 + 16 * t + x;
    mine[t] = __shfl(sees, min(row / cut.G, 63));
    if (row >= R) mine[t] = 0;
  }
  auto rest = [&](int i, auto pass) __attribute__((always_inline)) {
#pragma unroll 1
    for (; i < min(last, cached); i += NW) {
      const int limit = len - i * KB;
      uint32_t on[RT];
#pragma unroll
      for (int t = 0; t < RT; t++) on[t] = limit >= KB ? ~0u : (1u << limit) - 1u;
      load_keys8<DP, EXACT, true>(r, c8, at, eat, i, limit, a.head_dim);
      u32x4 pf[Parts<T>::N][RT];
      load_values8<DP, EXACT, true>(r, c8, at, eat, i, limit, a.head_dim);
      __builtin_amdgcn_sched_barrier(0);
      cache_weights<T, DP, RT, true>(z, r, cut.scale, on, pf);
      __builtin_amdgcn_sched_barrier(0);
      cache_product<T, DP, RT>(z, r, pf, pass);
    }
    if (Parts<T>::N == 2 && i < last) {  // (whole queries, read again rather than kept)
#pragma unroll
      for (int t = 0; t < RT; t++) {
        int row = row0 + 16 * t + x;
        asm volatile("" : "+v"(row));
        const uint16_t* p = query(row);
#pragma unroll
        for (int c = 0; c < S::KC; c++) z.q[0][t][c] = chunk(p, c);
      }
    }
#pragma unroll 1
    for (; i < last; i += NW) {
      const int key0 = (i - cached) * KB;
      uint32_t on[RT];
#pragma unroll
      for (int t = 0; t < RT; t++) on[t] = (uint32_t)(mine[t] >> key0);
      const int64_t f = b * a.fresh.seq_stride + kh * a.fresh.head_stride;
      tree_block<T, DP, RT, EXACT>(z, (const uint16_t*)a.fresh.k + f, (const uint16_t*)a.fresh.v + f, a.fresh.slot_stride, key0, n, a.head_dim,
                                   cut.scale, on, pass);
    }
  };
  rest(i, std::integral_constant<int, WALK>{});
  uint32_t* marked = (uint32_t*)&sum[wave] + lane;
  if (!finished(z.w, WALK, mine, marked)) [[unlikely]] {
    int pass = ABOVE;
#pragma unroll 1
    do {
      if constexpr (Parts<T>::N == 2) queries();
      rest(first + wave, pass);
    } while (!finished(z.w, pass++, mine, marked));
  }

  // the waves' sums, brought to one reference; rows that see nothing of the
  // tree see nothing of the cache either
  float ref[RT];
#pragma unroll
  for (int t = 0; t < RT; t++) {
    z.w.l[t] = row_sum(z.w.l[t]);
    if (mine[t] == 0) z.w.l[t] = 0.0f;
    ref[t] = z.w.l[t] == 0.0f ? NEG_INF : z.w.reference(t, cut.scale);
    if (g == 0) {
      stat[wave][t][0][x] = ref[t];
      stat[wave][t][1][x] = z.w.l[t];
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
    for (int k = 0; k < S::NF; k++) sum[wave][t][k][lane] = times(z.w.o[t][k], f);
  }
  __syncthreads();
  // a wave takes every fourth pair of fragments
  constexpr int PAIRS = S::VE / 2;
  const bool whole = first == 0 && last == total;
  float* part = cut.part + (((int64_t)unit * a.kv_heads + kh) * cut.tiles + tile) * S::PART;
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
      store_pair<T, DP, E4m3>(a, cut.G, b, kh, row0 + 16 * t + x, R, h, pair, o[0], o[1], top, all);
    } else {
      f32x4* p = (f32x4*)part + (t * S::NF + f0) * 64 + lane;
      p[0] = o[0];
      p[64] = o[1];
      if (h == 0 && pair == 0 && g == 0) {
        part[S::STAT + 32 * t + x] = top;
        part[S::STAT + 32 * t + 16 + x] = all;
      }
    }
  }
}

// Joins the splits of 16 rows and one half of the head: a pair of fragments a
// wave, over one of SHARES shares of the splits.
template <int DP, int SHARES>
constexpr int join8_threads() { return 64 * (Shape<DP, 1>::VE / 2) * SHARES; }

template <typename T, int DP, int SHARES>
__global__ __launch_bounds__((join8_threads<DP, SHARES>())) void join8_kernel(const xs_tree_attend_args a, const Cut8 cut) {
  using S = Shape<DP, 1>;
  constexpr int PAIRS = S::VE / 2, WAVES = PAIRS * SHARES;
  __shared__ float weight[SPLITS][16];
  __shared__ float stat[2][4 * WAVES][16];
  __shared__ f32x4 sum[SHARES][S::VE][64];
  const int lane = threadIdx.x & 63, x = lane & 15, g = lane >> 4;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), pair = wave % PAIRS, share = wave / PAIRS;
  const int h = blockIdx.x % S::VH, tile = blockIdx.x / S::VH % cut.tiles, bh = blockIdx.x / (S::VH * cut.tiles);
  const int kh = bh % (int)a.kv_heads, b = bh / (int)a.kv_heads;
  const int plan = __builtin_amdgcn_readfirstlane(cut.plan[b]), n = plan & 0xFFFF;
  const Seq sq(a, b);
  const int nodes = __builtin_amdgcn_readfirstlane(sq.bad ? -1 : sq.n), R = nodes * cut.G, row0 = 16 * tile;
  if (row0 >= R || n <= 1) return;
  const float* part = cut.part + (((int64_t)(plan >> 16) * a.kv_heads + kh) * cut.tiles + tile) * S::PART;
  const int64_t step = a.kv_heads * cut.tiles * S::PART;
  // the first fragments, on their way while the weights are formed
  constexpr int AHEAD = 4;
  const int f0 = h * S::VE + 2 * pair;
  f32x4 y[AHEAD][2];
#pragma unroll
  for (int i = 0; i < AHEAD; i++) {
    const f32x4* p = (const f32x4*)(part + min(share + SHARES * i, n - 1) * step) + f0 * 64 + lane;
    y[i][0] = p[0];
    y[i][1] = p[64];
  }
  // a quarter of a wave takes a split's rows
  float top = NEG_INF, all = 0.0f;
  for (int s = 4 * wave + g; s < n; s += 4 * WAVES) {
    const float* p = part + s * step;
    top = fmaxf(top, p[S::STAT + x]);
  }
  stat[0][4 * wave + g][x] = top;
  __syncthreads();
#pragma unroll 8
  for (int j = 0; j < 4 * WAVES; j++) top = fmaxf(top, stat[0][j][x]);
  for (int s = 4 * wave + g; s < n; s += 4 * WAVES) {
    const float* p = part + s * step + S::STAT + x;
    const float m = p[0], y = m == NEG_INF ? 0.0f : __builtin_amdgcn_exp2f((m - top) * fabsf(cut.scale));
    if (m != NEG_INF) all += p[16] * y;
    weight[s][x] = y;
  }
  stat[1][4 * wave + g][x] = all;
  __syncthreads();
  f32x4 o[2] = {{0.0f, 0.0f, 0.0f, 0.0f}, {0.0f, 0.0f, 0.0f, 0.0f}};
#pragma unroll
  for (int i = 0; i < AHEAD; i++) {
    if (share + SHARES * i >= n) break;
    const float f = weight[share + SHARES * i][x];
    o[0] += times(y[i][0], f);
    o[1] += times(y[i][1], f);
  }
#pragma unroll 4
  for (int s = share + SHARES * AHEAD; s < n; s += SHARES) {
    const f32x4* p = (const f32x4*)(part + s * step) + f0 * 64 + lane;
    const float f = weight[s][x];
    o[0] += times(p[0], f);
    o[1] += times(p[64], f);
  }
  sum[share][2 * pair][lane] = o[0];
  sum[share][2 * pair + 1][lane] = o[1];
  __syncthreads();
  if (share != 0) return;
  all = 0.0f;
#pragma unroll 8
  for (int j = 0; j < 4 * WAVES; j++) all += stat[1][j][x];
#pragma unroll
  for (int j = 1; j < SHARES; j++) {
    o[0] += sum[j][2 * pair][lane];
    o[1] += sum[j][2 * pair + 1][lane];
  }
  store_pair<T, DP, E4m3>(a, cut.G, b, kh, row0 + x, R, h, pair, o[0], o[1], top, all);
}

// More rows than that: 32 a wave (xs_rows32.h), of keys that the workgroup's
// threads turn into bf16 on their way to LDS, in stages of 64 through two
// buffers: while one is read, the next is written from registers and the one
// after it on its way from memory.  WK waves share 32 rows, each with its half of
// a stage's keys, and add up at the end; 32 W / WK rows a workgroup of W waves.  Bound
// by the products and the vector work beside them (xs_rows32.h), the widening among
// it, which eight waves share where rows fill them (four, two workgroups a CU: 181
// us for 170): 8 x 64 nodes of 32 q and 8 kv heads of 128 over 16,384 slots 160 to
// 187 us by card (856 to 733 TFLOP/s), of which the join takes 12.  By memory where
// rows are few: 16 nodes over 131,072 slots 72 to 88 us (3.7 to 3.1 TB/s).  The
// 16-row kernel with four row tiles instead takes 721 and 216 us: its waves widen
// every key for 64 rows each.
template <int DP, int WK, int W>
struct Shape32 {
  static constexpr int ROWS = 32 * W / WK, WR = W / WK;
  static constexpr int DT = DP / 32, NF = 4 * DT;    // fragments of four elements a lane
  static constexpr int STAT = WR * NF * 256;         // floats of a partial result: fragments,
  static constexpr int PART = STAT + 2 * ROWS;       // then m and l of each row
};

// Stages of a sequence: the cache's, and the tree's one.
constexpr int STAGES_LEAST = 4, STAGES_WHOLE = 8;

// Fragment f (elements e .. e + 4 of row `row`, e = 8 f + 4 g) of the result.
template <typename T>
XS_DEV void store_four(const xs_tree_attend_args& a, int G, int b, int kh, int row, int R, int f, f32x4 o, float ref, float l) {
  const int g = (threadIdx.x & 63) >> 5, e = 8 * f + 4 * g;
  const int node = min(row, R - 1) / G, head = kh * G + min(row, R - 1) % G;
  if (row >= R) return;
  const float inv = l == 0.0f ? 0.0f : 1.0f / l;
  uint16_t* out = (uint16_t*)a.out + b * a.out_seq_stride + node * a.out_node_stride + head * a.out_head_stride;
  if (e < a.head_dim) *(u32x2*)(out + e) = (u32x2){pack2(T{}, o[0] * inv, o[1] * inv), pack2(T{}, o[2] * inv, o[3] * inv)};
  if (a.lse && f == 0 && g == 0) a.lse[(b * a.nodes + node) * a.q_heads + head] = lse_of<E4m3>(a, ref, l);
}

template <typename T, int DP, int WK, int W, bool EXACT>
__global__ __launch_bounds__(64 * W, DP <= 128 ? 2 : 1) void attend8_wide_kernel(const xs_tree_attend_args a, const xs_kv8 c8, const Cut8 cut) {
  using S = Shape32<DP, WK, W>;
  using K = Keys<DP>;
  constexpr int N = Parts<T>::N, CH = K::CH, KC = DP / 16, DT = DP / 32, TH = 64 * W;
  constexpr int PER = SK * (DP / 16) / TH;  // 16-byte pieces of the cache that a thread moves, of k and of v
  static_assert(SK * (DP / 16) % TH == 0, "a stage is whole pieces of every thread");
  __shared__ u32x4 lk[2][K::STAGE];
  __shared__ u32x4 lv[2][K::STAGE];
  __shared__ uint16_t marks[2][DT][TH];  // [above, below] a lane's elements that an infinity reaches
  __shared__ int odds;                   // a result is not finite
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), wr = wave / WK, wk = wave % WK;
  int tile, kh, unit;
  deal(cut, &tile, &kh, &unit);
  if (kh >= (int)a.kv_heads) return;
  const Place8 pl = place8<SK, STAGES_LEAST, STAGES_WHOLE>(a, cut, unit);
  const int b = __builtin_amdgcn_readfirstlane(pl.b), split = __builtin_amdgcn_readfirstlane(pl.split);
  const int splits = __builtin_amdgcn_readfirstlane(pl.n);
  if (b < 0) return;
  const int share = __builtin_amdgcn_readfirstlane(pl.share), bh = b * (int)a.kv_heads + kh;
  const int len = __builtin_amdgcn_readfirstlane(pl.len), n = __builtin_amdgcn_readfirstlane(pl.nodes);
  if (split == 0 && tile == 0 && kh == 0 && threadIdx.x == 0) {
    a.seq_status[b] = n < 0 ? XS_ROW_BAD_PARAM : XS_ROW_OK;
    if (cut.room) cut.plan[b] = unit << 16 | splits;
  }
  const int R = n * cut.G;
  const int cached = (len + SK - 1) / SK, total = cached + (n > 0 ? 1 : 0), first = split * share, last = splits == 1 ? total : min(first + share, total);
  if (tile * S::ROWS >= R || first >= total) return;  // (nodes below 0 too)

  // whole and part stages of the cache
  const int end = min(last, cached);
  const int64_t at = b * c8.seq_stride + kh * c8.head_stride, eat = (int64_t)bh * c8.exp_ld;
  const uint32_t stride = (uint32_t)c8.slot_stride;
  Rows32<Bf16, DP, N> w;
  float l, ref;
  int row;
  if (threadIdx.x == 0) odds = 0;
#pragma unroll 1
  for (int pass = WALK;; pass++) {
    int tid = threadIdx.x;
    asm volatile("" : "+v"(tid));  // (nothing of a lane's is kept from pass to pass)
    const int lane = tid & 63, x = lane & 31, g = lane >> 5;
    row = tile * S::ROWS + 32 * wr + x;
    const int parent = parent_of(a, b);
    auto query = [&](int r) {
      const int node = min(r, R - 1) / cut.G, head = kh * cut.G + min(r, R - 1) % cut.G;
      return (const uint16_t*)a.q + b * a.q_seq_stride + node * a.q_node_stride + head * a.q_head_stride;
    };
    auto chunk = [&](const uint16_t* p, int c) {
      const int d = 16 * c + 8 * g;
      return row < R && (EXACT || d < a.head_dim) ? *(const u32x4*)(p + d) : (u32x4){0, 0, 0, 0};
    };
    {
      const uint16_t* p = query(row);
#pragma unroll
      for (int c = 0; c < KC; c++) w.q[0][c] = chunk(p, c);
      if constexpr (N == 2) {
#pragma unroll
        for (int c = 0; c < KC; c++) {
          __builtin_amdgcn_sched_barrier(0);  // (one chunk's comparisons at a time)
          u32x4 y[N];
          split8(T{}, w.q[0][c], y);
          w.q[0][c] = y[0];
          w.q[1][c] = y[1];
        }
      }
    }
    const uint64_t seen = ancestors(parent, n);
    const uint64_t mine = __shfl(seen, min(row / cut.G, 63)) & (row < R ? ~0ull : 0ull);  // what the lane's row sees of the tree
    const Reads<DP> reads(lane);

    u32x4 rk[PER], rv[PER];
    uint32_t ex;  // a stage's exponents: of the keys' two blocks, then of the values', by lane & 3
    auto fetch = [&](int s) {
      const int64_t base = at + (int64_t)s * SK * c8.slot_stride;
      const int most = len - 1 - s * SK;
      ex = ((lane & 2) ? c8.v_exp : c8.k_exp)[eat + min(s * (SK / KB) + (lane & 1), (len - 1) / KB)];
#pragma unroll
      for (int j = 0; j < PER; j++) {
        const int p = j * TH + tid, r = min(p / (DP / 16), most), c = p % (DP / 16);
        const uint32_t off = (uint32_t)r * stride + 16 * c;
        const bool in = EXACT || 16 * c < a.head_dim;
        rk[j] = in ? *(const u32x4*)(c8.k + base + off) : (u32x4){0, 0, 0, 0};
        rv[j] = in ? *(const u32x4*)(c8.v + base + off) : (u32x4){0, 0, 0, 0};
      }
    };
    auto put = [&](int s) {
      const int most = len - 1 - s * SK;
#pragma unroll
      for (int j = 0; j < PER; j++) {
        const int p = j * TH + tid, r = p / (DP / 16), c = p % (DP / 16);
        // (a wave's pieces j lie in one block)
        const int block = PER > 1 ? j * (TH / (DP / 16)) / KB : __builtin_amdgcn_readfirstlane(r / KB);
        const float ks = pow2(__builtin_amdgcn_readlane((int)ex, block) - 127), vs = pow2(__builtin_amdgcn_readlane((int)ex, 2 + block) - 127);
        const u32x4 y = r <= most ? rv[j] : (u32x4){0, 0, 0, 0};  // (past the length: nothing, whatever it holds)
#pragma unroll
        for (int h = 0; h < 2; h++) {
          u32x4 k, v;
#pragma unroll
          for (int i = 0; i < 4; i++) {
            k[i] = wide2(rk[j][2 * h + i / 2], ks, i % 2);
            v[i] = wide2(y[2 * h + i / 2], vs, i % 2);
          }
          lk[s & 1][r * CH + ((2 * c + h) ^ K::turn_k(r))] = k;
          lv[s & 1][r * CH + ((2 * c + h) ^ K::turn_v(r))] = v;
        }
      }
      if (pass != WALK) [[unlikely]] {  // (the thread's own pieces)
#pragma unroll 1
        for (int i = 0; i < 2 * PER; i++) {
          const int p = i / 2 * TH + tid, r = p / (DP / 16);
          u32x4* v = &lv[s & 1][r * CH + ((2 * (p % (DP / 16)) + i % 2) ^ K::turn_v(r))];
#pragma unroll
          for (int e = 0; e < 4; e++) (*v)[e] = passed(Bf16{}, (*v)[e], pass);
        }
      }
    };
    auto step = [&](const u32x4* ks, const u32x4* vs, bool masked, uint64_t on) {
      // (f16: a tile at a time, which the registers hold beside two parts of each row)
      constexpr int U = N == 1 && WK == 1 ? 2 : 1, STEPS = 2 / (U * WK);
#pragma unroll
      for (int i = 0; i < STEPS; i++) {
        const int u = WK == 1 ? i : wk;
        const uint64_t bits = on >> (32 * u + 4 * g);
        w.template step<U, 1>(reads, ks + 32 * u * CH, {vs + 32 * u * CH}, cut.scale, masked, Bits{(uint32_t)bits, (uint32_t)(bits >> 32)});
      }
    };

    w.init();
    if (first < end) {
      fetch(first);
      put(first);
      if (first + 1 < end) fetch(first + 1);
    }
#pragma unroll 1
    for (int s = first; s < end; s++) {
      __syncthreads();
      if constexpr (N == 2) asm volatile("" : "+v"(tid));  // (its addresses, formed anew, need no registers)
      if (s + 1 < end) put(s + 1);
      if (s + 2 < end) fetch(s + 2);
      const int limit = len - s * SK;
      step(lk[s & 1], lv[s & 1], limit < SK, limit < SK ? (1ull << limit) - 1ull : ~0ull);
    }
    // the tree: keys and queries as they are, parts of the values in a buffer each
    if (last == total) {
      __syncthreads();
      const int64_t f = b * a.fresh.seq_stride + kh * a.fresh.head_stride;
#pragma unroll 1
      for (int p = tid; p < K::STAGE; p += TH) {
        const int r = p / CH, c = p % CH;
        u32x4 k = {0, 0, 0, 0}, v = {0, 0, 0, 0};
        if (r < n && (EXACT || 8 * c < a.head_dim)) {
          k = *(const u32x4*)((const uint16_t*)a.fresh.k + f + r * a.fresh.slot_stride + 8 * c);
          v = *(const u32x4*)((const uint16_t*)a.fresh.v + f + r * a.fresh.slot_stride + 8 * c);
        }
        if (pass != WALK) [[unlikely]] {
#pragma unroll
          for (int i = 0; i < 4; i++) v[i] = passed(T{}, v[i], pass);
        }
        lk[0][r * CH + (c ^ K::turn_k(r))] = k;
        u32x4 vs[N];
        split8(T{}, v, vs);
#pragma unroll
        for (int m = 0; m < N; m++) lv[m][r * CH + (c ^ K::turn_v(r))] = vs[m];
      }
      __syncthreads();
      if constexpr (N == 2) {
        int again = row;
        asm volatile("" : "+v"(again));  // (whole queries, read again rather than kept)
        const uint16_t* p = query(again);
#pragma unroll
        for (int c = 0; c < KC; c++) w.q[0][c] = chunk(p, c);
      }
#pragma unroll 1
      for (int i = 0; i < 2 / WK; i++) {
        const int u = WK == 1 ? i : wk;
        const uint64_t bits = mine >> (32 * u + 4 * g);
        const Bits on = {(uint32_t)bits, (uint32_t)(bits >> 32)};
        if (32 * u >= n) continue;
        if constexpr (N == 1) w.template step<1, 1>(reads, lk[0] + 32 * u * CH, {lv[0] + 32 * u * CH}, cut.scale, true, on);
        else w.template step<1, 2, 1, F16>(reads, lk[0] + 32 * u * CH, {lv[0] + 32 * u * CH, lv[1] + 32 * u * CH}, cut.scale, true, on);
      }
    }

    // rows that see nothing of the tree see nothing of the cache either
    l = mine == 0 ? 0.0f : pair_sum(w.l);
    ref = l == 0.0f ? NEG_INF : cut.scale < 0.0f ? -w.reference() : w.reference();
    if (l == 0.0f) {
#pragma unroll
      for (int d = 0; d < DT; d++) w.o[d] = fill16(0.0f);
    }
    if constexpr (WK == 2) {
      __syncthreads();  // (the stages' last readers)
      f32x4* sum = (f32x4*)&lk[0][0] + wr * S::NF * 64;
      float* stat = (float*)&lv[0][0] + wr * 64;
      if (wk == 1) {
#pragma unroll
        for (int f = 0; f < S::NF; f++) {
          const f32x16 o = w.o[f / 4];
          sum[f * 64 + lane] = (f32x4){o[4 * (f % 4)], o[4 * (f % 4) + 1], o[4 * (f % 4) + 2], o[4 * (f % 4) + 3]};
        }
        if (g == 0) {
          stat[x] = ref;
          stat[32 + x] = l;
        }
      }
      __syncthreads();
      if (wk == 0) {
        const float ref1 = stat[x], l1 = stat[32 + x], top = fmaxf(ref, ref1), mag = fabsf(cut.scale);
        const float f0 = ref == NEG_INF ? 0.0f : __builtin_amdgcn_exp2f((ref - top) * mag);
        const float f1 = ref1 == NEG_INF ? 0.0f : __builtin_amdgcn_exp2f((ref1 - top) * mag);
        l = (ref == NEG_INF ? 0.0f : l * f0) + (ref1 == NEG_INF ? 0.0f : l1 * f1);
        ref = top;
#pragma unroll
        for (int f = 0; f < S::NF; f++) {
          const f32x4 y = sum[f * 64 + lane];
#pragma unroll
          for (int i = 0; i < 4; i++) w.o[f / 4][4 * (f % 4) + i] = __builtin_fmaf(w.o[f / 4][4 * (f % 4) + i], f0, y[i] * f1);
        }
      }
    }
    if (pass == WALK) {
      float z = 0.0f;
#pragma unroll
      for (int d = 0; d < DT; d++)
#pragma unroll
        for (int i = 0; i < 16; i++) z = __builtin_fmaf(w.o[d][i], 0.0f, z);
      if (wk == 0 && row < R && l > 0.0f && z != z) odds = 1;
      __syncthreads();
      if (!__builtin_amdgcn_readfirstlane(odds)) [[likely]] break;
    } else if (pass == FINITE) {
#pragma unroll
      for (int d = 0; d < DT; d++)
#pragma unroll
        for (int i = 0; i < 16; i++) w.o[d][i] = marked(w.o[d][i], marks[0][d][tid], marks[1][d][tid], i);
      break;
    } else {
#pragma unroll
      for (int d = 0; d < DT; d++) {
        uint32_t m = 0;
#pragma unroll
        for (int i = 15; i >= 0; i--) m = m << 1 | (w.o[d][i] > 0.0f ? 1u : 0u);
        marks[pass - ABOVE][d][tid] = (uint16_t)m;
      }
      __syncthreads();  // (the stages' readers)
    }
  }
  if (wk == 1) return;
  const int lane = threadIdx.x & 63, x = lane & 31, g = lane >> 5;
  const bool whole = first == 0 && last == total;
  float* part = cut.part + (((int64_t)unit * a.kv_heads + kh) * cut.tiles + tile) * S::PART;
#pragma unroll
  for (int f = 0; f < S::NF; f++) {
    const f32x16 o = w.o[f / 4];
    const f32x4 y = {o[4 * (f % 4)], o[4 * (f % 4) + 1], o[4 * (f % 4) + 2], o[4 * (f % 4) + 3]};
    if (whole) store_four<T>(a, cut.G, b, kh, row, R, f, y, ref, l);
    else ((f32x4*)part)[(wr * S::NF + f) * 64 + lane] = y;
  }
  if (!whole && g == 0) {
    part[S::STAT + 32 * wr + x] = ref;
    part[S::STAT + S::ROWS + 32 * wr + x] = l;
  }
}

// Joins the splits of 32 rows, four fragments a workgroup: each wave one of them
// over one of SHARES shares of the splits.
template <typename T, int DP, int WK, int W, int SHARES>
__global__ __launch_bounds__(256 * SHARES) void join32_kernel(const xs_tree_attend_args a, const Cut8 cut) {
  using S = Shape32<DP, WK, W>;
  constexpr int WAVES = 4 * SHARES;
  __shared__ float weight[SPLITS][32];
  __shared__ float stat[2][2 * WAVES][32];
  __shared__ f32x4 sum[SHARES][4][64];
  const int lane = threadIdx.x & 63, x = lane & 31, g = lane >> 5;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), share = wave / 4;
  const int f = blockIdx.x % S::DT * 4 + wave % 4, wr = blockIdx.x / S::DT % S::WR, tile = blockIdx.x / (S::DT * S::WR) % cut.tiles;
  const int bh = blockIdx.x / (S::DT * S::WR * cut.tiles), kh = bh % (int)a.kv_heads, b = bh / (int)a.kv_heads;
  const int plan = __builtin_amdgcn_readfirstlane(cut.plan[b]), n = plan & 0xFFFF;
  const Seq sq(a, b);
  const int nodes = __builtin_amdgcn_readfirstlane(sq.bad ? -1 : sq.n), R = nodes * cut.G, row = tile * S::ROWS + 32 * wr + x;
  if (tile * S::ROWS + 32 * wr >= R || n <= 1) return;
  const float* part = cut.part + (((int64_t)(plan >> 16) * a.kv_heads + kh) * cut.tiles + tile) * S::PART;
  const int64_t step = a.kv_heads * cut.tiles * S::PART;
  // the first fragments, on their way while the weights are formed
  constexpr int AHEAD = SHARES > 1 ? 16 : 4;
  f32x4 y[AHEAD];
#pragma unroll
  for (int i = 0; i < AHEAD; i++) y[i] = ((const f32x4*)(part + min(share + SHARES * i, n - 1) * step))[(wr * S::NF + f) * 64 + lane];
  // half a wave takes a split's rows
  float top = NEG_INF, all = 0.0f;
  for (int s = 2 * wave + g; s < n; s += 2 * WAVES) {
    const float* p = part + s * step;
    top = fmaxf(top, p[S::STAT + 32 * wr + x]);
  }
  stat[0][2 * wave + g][x] = top;
  __syncthreads();
#pragma unroll 8
  for (int j = 0; j < 2 * WAVES; j++) top = fmaxf(top, stat[0][j][x]);
  for (int s = 2 * wave + g; s < n; s += 2 * WAVES) {
    const float* p = part + s * step + S::STAT + 32 * wr + x;
    const float m = p[0], y = m == NEG_INF ? 0.0f : __builtin_amdgcn_exp2f((m - top) * fabsf(cut.scale));
    if (m != NEG_INF) all += p[S::ROWS] * y;
    weight[s][x] = y;
  }
  stat[1][2 * wave + g][x] = all;
  __syncthreads();
  f32x4 o = {0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
  for (int i = 0; i < AHEAD; i++) {
    if (share + SHARES * i >= n) break;
    o += times(y[i], weight[share + SHARES * i][x]);
  }
#pragma unroll 8
  for (int s = share + SHARES * AHEAD; s < n; s += SHARES) o += times(((const f32x4*)(part + s * step))[(wr * S::NF + f) * 64 + lane], weight[s][x]);
  sum[share][wave % 4][lane] = o;
  __syncthreads();
  if (share != 0) return;
  all = 0.0f;
#pragma unroll 8
  for (int j = 0; j < 2 * WAVES; j++) all += stat[1][j][x];
#pragma unroll
  for (int j = 1; j < SHARES; j++) o += sum[j][wave % 4][lane];
  store_four<T>(a, cut.G, b, kh, row, R, f, o, top, all);
}

}  // namespace xs8

// ---------------------------------------------------------------------------
// Host side.

namespace {

using xs_host::OnDevice;
using xs_host::per_cu;

// The launch's units and room, for shares of up to `slots` workgroups with
// partial results of `part` floats; false: too many for one launch.
bool cut8(xs_cache_context* c, const xs_tree_attend_args& a, int rows, int64_t slots, int64_t part, int64_t unit, int64_t least, int64_t whole,
          xs8::Cut8* cut, int64_t* grid) {
  cut->G = (int32_t)(a.q_heads / a.kv_heads);
  cut->tiles = (int32_t)((a.nodes * cut->G + rows - 1) / rows);
  cut->scale = a.scale * xst::LOG2E;
  cut->part = c->part;
  cut->plan = c->evict.moves;  // (of max_seqs entries and more; an eviction fills it anew)
  const int64_t limit = a.max_len ? a.max_len : a.capacity, units = (limit + unit - 1) / unit + (a.nodes + unit - 1) / unit;
  const int64_t heads = a.kv_heads * cut->tiles;
  const int64_t places = c->part_floats / (heads * part);
  int64_t room = std::min<int64_t>(std::min(slots / heads, places), xst::SPLITS);
  // one round of the device, or, of more sequences than that, more by a share each
  const bool fits = room > a.seqs || places >= room + a.seqs;
  if (units <= whole || a.seqs > 256 || room < 2 || !fits) room = 0;
  cut->room = (int32_t)room;
  cut->units = (int32_t)(!room ? a.seqs : std::min(room > a.seqs ? room : room + a.seqs, a.seqs * ((units + least - 1) / least)));
  *grid = ((int64_t)cut->units * a.kv_heads + 7) / 8 * 8 * cut->tiles;
  return xs_host_launch_fits(*grid, 128 * xst::NW);
}

// Shares of the splits that a join goes through side by side: several where a
// sequence has many (an average of more than eight).
bool many8(const xs8::Cut8& cut, const xs_tree_attend_args& a) { return cut.room > 8 * a.seqs; }

template <typename T, int DP, bool EXACT>
int attend8_run(xs_cache_context* c, const xs_tree_attend_args& a, const xs_kv8& c8) {
  xs8::Cut8 cut;
  int64_t grid;
  if (!cut8(c, a, 16, c->n_cu * per_cu(DP, 1), xst::Shape<DP, 1>::PART, xst::KB, 2 * xst::NW, 4 * xst::NW, &cut, &grid)) return XS_ERR_CAPACITY;
  const int64_t join = a.seqs * a.kv_heads * cut.tiles * xst::Shape<DP, 1>::VH;
  if (cut.room && !xs_host_launch_fits(join, xs8::join8_threads<DP, 4>())) return XS_ERR_CAPACITY;
  hipLaunchKernelGGL((xs8::attend8_kernel<T, DP, 1, EXACT>), dim3((unsigned)grid), dim3(64 * xst::NW), 0, c->stream, a, c8, cut);
  if (cut.room && many8(cut, a))
    hipLaunchKernelGGL((xs8::join8_kernel<T, DP, 4>), dim3((unsigned)join), dim3(xs8::join8_threads<DP, 4>()), 0, c->stream, a, cut);
  else if (cut.room)
    hipLaunchKernelGGL((xs8::join8_kernel<T, DP, 1>), dim3((unsigned)join), dim3(xs8::join8_threads<DP, 1>()), 0, c->stream, a, cut);
  return hipGetLastError() == hipSuccess ? XS_OK : XS_ERR_HIP;
}

template <typename T, int DP, int WK, int W, bool EXACT>
int attend8_wide_run(xs_cache_context* c, const xs_tree_attend_args& a, const xs_kv8& c8) {
  using S = xs8::Shape32<DP, WK, W>;
  xs8::Cut8 cut;
  int64_t grid;
  // (as many workgroups as a CU's LDS holds)
  if (!cut8(c, a, S::ROWS, c->n_cu * (DP <= 128 && W == xst::NW ? 2 : 1), S::PART, xst::SK, xs8::STAGES_LEAST, xs8::STAGES_WHOLE, &cut, &grid)) return XS_ERR_CAPACITY;
  const int64_t join = a.seqs * a.kv_heads * cut.tiles * S::WR * S::DT;
  if (cut.room && !xs_host_launch_fits(join, 1024)) return XS_ERR_CAPACITY;
  hipLaunchKernelGGL((xs8::attend8_wide_kernel<T, DP, WK, W, EXACT>), dim3((unsigned)grid), dim3(64 * W), 0, c->stream, a, c8, cut);
  if (cut.room && many8(cut, a)) hipLaunchKernelGGL((xs8::join32_kernel<T, DP, WK, W, 4>), dim3((unsigned)join), dim3(1024), 0, c->stream, a, cut);
  else if (cut.room) hipLaunchKernelGGL((xs8::join32_kernel<T, DP, WK, W, 1>), dim3((unsigned)join), dim3(256), 0, c->stream, a, cut);
  return hipGetLastError() == hipSuccess ? XS_OK : XS_ERR_HIP;
}

template <typename T, int DP, bool EXACT>
int attend8_rows(xs_cache_context* c, const xs_tree_attend_args& a, const xs_kv8& c8) {
  const int64_t rows = a.nodes * (a.q_heads / a.kv_heads);
  if (rows <= 16) return attend8_run<T, DP, EXACT>(c, a, c8);
  if (rows <= 64) return attend8_wide_run<T, DP, 2, xst::NW, EXACT>(c, a, c8);
  if constexpr (DP == 128) {  // (heads of 64 have half a piece a thread, heads of 256 registers for one wave a SIMD)
    if ((rows + 127) / 128 % 2 == 0) return attend8_wide_run<T, DP, 1, 2 * xst::NW, EXACT>(c, a, c8);
  }
  return attend8_wide_run<T, DP, 1, xst::NW, EXACT>(c, a, c8);
}

template <typename T, int DP>
int attend8_exact(xs_cache_context* c, const xs_tree_attend_args& a, const xs_kv8& c8) {
  return a.head_dim == DP ? attend8_rows<T, DP, true>(c, a, c8) : attend8_rows<T, DP, false>(c, a, c8);
}

template <typename T>
int attend8_dim(xs_cache_context* c, const xs_tree_attend_args& a, const xs_kv8& c8) {
  if (a.head_dim <= 64) return attend8_exact<T, 64>(c, a, c8);
  if (a.head_dim <= 128) return attend8_exact<T, 128>(c, a, c8);
  return attend8_exact<T, 256>(c, a, c8);
}

}  // namespace

extern "C" {

int xs_cache_append8(xs_cache_context* c, const xs_cache_append8_args* in) {
  const int rc = xs_host_check_append8(c ? &c->dims : nullptr, in);
  if (rc) return rc;
  if (in->seqs == 0) return XS_OK;
  const OnDevice on(c->device);
  if (!on.ok) return XS_ERR_HIP;
  // blocks that `rows` rows can touch, the first of them partly in use
  const int64_t rows = std::min(in->rows, in->capacity), blocks = (rows + XS_CACHE8_BLOCK - 1) / XS_CACHE8_BLOCK + 1;
  const int64_t grid = in->seqs * in->kv_heads * blocks;
  if (!xs_host_launch_fits(grid, xs8::AB)) return XS_ERR_CAPACITY;
  if (in->dtype == XS_BF16)
    hipLaunchKernelGGL((xs8::append_kernel<xst::Bf16>), dim3((unsigned)grid), dim3(xs8::AB), 0, c->stream, *in, (int)blocks);
  else
    hipLaunchKernelGGL((xs8::append_kernel<xst::F16>), dim3((unsigned)grid), dim3(xs8::AB), 0, c->stream, *in, (int)blocks);
  return hipGetLastError() == hipSuccess ? XS_OK : XS_ERR_HIP;
}

int xs_tree_attend8(xs_cache_context* c, const xs_tree_attend8_args* in) {
  const int rc = xs_host_check_attend8(c ? &c->dims : nullptr, in);
  if (rc) return rc;
  if (in->seqs == 0) return XS_OK;
  const OnDevice on(c->device);
  if (!on.ok) return XS_ERR_HIP;
  // all but the cache as the kernels of xs_attend.h take it
  xs_tree_attend_args a = {};
  a.dtype = in->dtype, a.head_dim = in->head_dim, a.seqs = in->seqs, a.nodes = in->nodes, a.q_heads = in->q_heads, a.kv_heads = in->kv_heads;
  a.q = in->q, a.q_seq_stride = in->q_seq_stride, a.q_node_stride = in->q_node_stride, a.q_head_stride = in->q_head_stride;
  a.capacity = in->capacity, a.max_len = in->max_len, a.len = in->len, a.fresh = in->fresh;
  a.parent = in->parent, a.n_nodes = in->n_nodes, a.scale = in->scale;
  a.out = in->out, a.out_seq_stride = in->out_seq_stride, a.out_node_stride = in->out_node_stride, a.out_head_stride = in->out_head_stride;
  a.lse = in->lse, a.seq_status = in->seq_status;
  if (in->dtype == XS_BF16) return attend8_dim<xst::Bf16>(c, a, in->cache);
  return attend8_dim<xst::F16>(c, a, in->cache);
}

}  // extern "C"
