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
// writing the bytes.

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
// exponents, applied by the conversion itself.  f16 queries, fresh keys and
// values, and the weights of f16 calls are sums of two bf16 (a float of 11 bits
// is one exactly, a weight to 16 bits), each part a product of its own.
// A lane loads 16 bytes of a key: elements 64 c + 16 g + 8 h .. + 8 are chunk
// 2 c + h of the products, for queries and fresh keys too.

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

// The scores of 32 keys (parts kn of each), from the reference or from 0.
template <typename T, int DP, int RT, int KN>
XS_DEV void scores(const Tile<T, DP, RT>& z, int t, const u32x4 (&k)[KN][2][Shape<DP, RT>::KC], f32x4 start, f32x4 (&s)[2]) {
  s[0] = s[1] = start;
#pragma unroll
  for (int m = 0; m < KN; m++)
#pragma unroll
    for (int n = 0; n < Tile<T, DP, RT>::N; n++)
#pragma unroll
      for (int c = 0; c < Shape<DP, RT>::KC; c++) {
        s[0] = mfma(Bf16{}, k[m][0][c], z.q[n][t][c], s[0]);
        s[1] = mfma(Bf16{}, k[m][1][c], z.q[n][t][c], s[1]);
      }
}

// The softmax and the second product of a block, keys and values as parts.
template <typename T, int DP, int RT, bool MASKED, int KN>
XS_DEV void block8(Tile<T, DP, RT>& z, const u32x4 (&k)[KN][2][Shape<DP, RT>::KC], const uint32_t (&v)[KN][8][Shape<DP, RT>::VH][Shape<DP, RT>::VE / 2],
                   float scale, const uint32_t* on) {
  constexpr int N = Tile<T, DP, RT>::N;
  u32x4 pf[N][RT];
#pragma unroll
  for (int t = 0; t < RT; t++) {
    f32x4 s[2];
    scores<T, DP, RT, KN>(z, t, k, z.w.start(t), s);
    float x[8];
    const float top = z.w.template scaled<MASKED>(s, scale, MASKED ? on[t] : 0u, x);
    if (__any(z.w.passes(t, top))) [[unlikely]] {
      const bool far = __any(z.w.passes(t, top) && z.w.minus(z.w.c[t]) != 0.0f);
      if (far) [[unlikely]] scores<T, DP, RT, KN>(z, t, k, (f32x4){0.0f, 0.0f, 0.0f, 0.0f}, s);
      z.w.template rebase<MASKED>(t, s, far, scale, MASKED ? on[t] : 0u, x);
    }
    if constexpr (N == 1) {
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
#pragma unroll
  for (int m = 0; m < KN; m++)
#pragma unroll
    for (int n = 0; n < N; n++) accumulate(z.w, v[m], pf[n]);
}

// A block of the cache: 32 slots, `limit` of them in use.
template <typename T, int DP, int RT, bool EXACT, bool MASKED>
XS_DEV void cache_block(Tile<T, DP, RT>& z, const uint8_t* kp, const uint8_t* vp, int64_t stride, int ke, int ve, int limit, int D, float scale,
                        const uint32_t* on) {
  using S = Shape<DP, RT>;
  const int lane = threadIdx.x & 63, x = lane & 15, g = lane >> 4;
  const float kscale = pow2(ke - 127), vscale = pow2(ve - 127);
  u32x4 k8[2][S::KC / 2];
#pragma unroll
  for (int t = 0; t < 2; t++) {
    const int key = MASKED ? min(16 * t + x, limit - 1) : 16 * t + x;
#pragma unroll
    for (int c = 0; c < S::KC / 2; c++) {
      const int d = 64 * c + 16 * g;
      k8[t][c] = EXACT || d < D ? *(const u32x4*)(kp + key * stride + d) : (u32x4){0, 0, 0, 0};
    }
  }
  uint32_t v8[8][S::VH][S::VE / 4];
#pragma unroll
  for (int e = 0; e < 8; e++) {
    const int slot = 4 * g + (e & 3) + 16 * (e >> 2), key = MASKED ? min(slot, limit - 1) : slot;
#pragma unroll
    for (int h = 0; h < S::VH; h++) {
      int d = 128 * h + S::VE * x;
      if (!EXACT) d = min(d, D - S::VE);  // (products of elements past the head's are never stored)
      const uint8_t* p = vp + key * stride + d;
      if constexpr (S::VE == 8) {
        const u32x2 r = *(const u32x2*)p;
        v8[e][h][0] = r[0];
        v8[e][h][1] = r[1];
      } else {
        v8[e][h][0] = *(const uint32_t*)p;
      }
      if (MASKED && slot >= limit) {
#pragma unroll
        for (int i = 0; i < S::VE / 4; i++) v8[e][h][i] = 0;  // count for nothing, whatever they hold
      }
    }
  }
  u32x4 k[1][2][S::KC];
#pragma unroll
  for (int t = 0; t < 2; t++)
#pragma unroll
    for (int c = 0; c < S::KC; c++)
#pragma unroll
      for (int i = 0; i < 4; i++) k[0][t][c][i] = wide2(k8[t][c / 2][2 * (c % 2) + i / 2], kscale, i % 2);
  uint32_t v[1][8][S::VH][S::VE / 2];
#pragma unroll
  for (int e = 0; e < 8; e++)
#pragma unroll
    for (int h = 0; h < S::VH; h++)
#pragma unroll
      for (int i = 0; i < S::VE / 2; i++) v[0][e][h][i] = wide2(v8[e][h][i / 2], vscale, i % 2);
  block8<T, DP, RT, MASKED, 1>(z, k, v, scale, on);
}

// A block of the tree's own keys, in the inputs' type.
template <typename T, int DP, int RT, bool EXACT>
XS_DEV void tree_block(Tile<T, DP, RT>& z, const uint16_t* kp, const uint16_t* vp, int64_t stride, int key0, int limit, int D, float scale,
                       const uint32_t* on) {
  using S = Shape<DP, RT>;
  constexpr int N = Tile<T, DP, RT>::N;
  const int lane = threadIdx.x & 63, x = lane & 15, g = lane >> 4;
  u32x4 k[N][2][S::KC];
#pragma unroll
  for (int t = 0; t < 2; t++) {
    const int key = min(key0 + 16 * t + x, limit - 1);
#pragma unroll
    for (int c = 0; c < S::KC; c++) {
      const int d = 64 * (c / 2) + 16 * g + 8 * (c % 2);
      u32x4 y[N];
      split8(T{}, EXACT || d < D ? *(const u32x4*)(kp + key * stride + d) : (u32x4){0, 0, 0, 0}, y);
#pragma unroll
      for (int n = 0; n < N; n++) k[n][t][c] = y[n];
    }
  }
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
      // What is not finite would, through the product, reach the rows that do not
      // see the node: taken out here, added by store_pair to the rows that do.
#pragma unroll
      for (int i = 0; i < S::VE / 2; i++) {
        if (slot >= limit) r[i] = 0;
        if ((r[i] & 0x7FFFu) >= inf_of(T{})) r[i] &= 0xFFFF0000u, z.w.odd = 1;
        if (((r[i] >> 16) & 0x7FFFu) >= inf_of(T{})) r[i] &= 0xFFFFu, z.w.odd = 1;
      }
      u32x4 y[N];
      split8(T{}, r, y);
#pragma unroll
      for (int n = 0; n < N; n++)
#pragma unroll
        for (int i = 0; i < S::VE / 2; i++) v[n][e][h][i] = y[n][i];
    }
  }
  z.w.odd = __any(z.w.odd);
  block8<T, DP, RT, true, N>(z, k, v, scale, on);
}

// Up to 16 RT rows a workgroup, whose waves split the keys and add up through
// LDS; grid as in attend_kernel.
template <typename T, int DP, int RT, bool EXACT>
__global__ __launch_bounds__(64 * NW, DP * RT <= 64 ? 4 : DP * RT <= 128 ? 3 : DP * RT <= 256 ? 2 : 1) void attend8_kernel(
    const xs_tree_attend_args a, const xs_kv8 c8, const Cut cut) {
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
  const int row0 = tile * RT * 16, parent = parent_of(a, b);
  Tile<T, DP, RT> z;
  z.w.init();
#pragma unroll
  for (int t = 0; t < RT; t++) {
    const int row = row0 + 16 * t + x;
    const bool in = row < (int)a.nodes * cut.G;
    const int node = in ? row / cut.G : 0, head = kh * cut.G + (in ? row % cut.G : 0);
    const uint16_t* p = (const uint16_t*)a.q + b * a.q_seq_stride + node * a.q_node_stride + head * a.q_head_stride;
#pragma unroll
    for (int c = 0; c < S::KC; c++) {
      const int d = 64 * (c / 2) + 16 * g + 8 * (c % 2);
      u32x4 y[Tile<T, DP, RT>::N];
      split8(T{}, in && (EXACT || d < a.head_dim) ? *(const u32x4*)(p + d) : (u32x4){0, 0, 0, 0}, y);
#pragma unroll
      for (int n = 0; n < Tile<T, DP, RT>::N; n++) z.q[n][t][c] = y[n];
    }
  }
  const Seq sq(a, b);
  if (split == 0 && tile == 0 && kh == 0 && threadIdx.x == 0) a.seq_status[b] = sq.bad ? XS_ROW_BAD_PARAM : XS_ROW_OK;
  if (sq.bad) return;
  const int R = sq.n * cut.G;
  const int total = sq.blocks(), cached = (sq.len + KB - 1) / KB;
  const int first = split * cut.chunk, last = min(first + cut.chunk, total);
  if (row0 >= R || first >= total) return;

  const int64_t at = b * c8.seq_stride + kh * c8.head_stride, eat = (int64_t)bh * c8.exp_ld;
  const uint64_t sees = ancestors(parent, sq.n);
  uint64_t mine[RT];  // what the lane's rows see of the tree
#pragma unroll
  for (int t = 0; t < RT; t++) {
    const int row = row0 + 16 * t + x;
    mine[t] = __shfl(sees, min(row / cut.G, 63));
    if (row >= R) mine[t] = 0;
  }
  int i = first + wave;
  for (; i < last && (i + 1) * KB <= sq.len; i += NW)
    cache_block<T, DP, RT, EXACT, false>(z, c8.k + at + (int64_t)i * KB * c8.slot_stride, c8.v + at + (int64_t)i * KB * c8.slot_stride,
                                         c8.slot_stride, c8.k_exp[eat + i], c8.v_exp[eat + i], KB, a.head_dim, cut.scale, nullptr);
#pragma unroll 1
  for (; i < last; i += NW) {
    uint32_t on[RT];
    if (i < cached) {
      const int limit = sq.len - i * KB;
#pragma unroll
      for (int t = 0; t < RT; t++) on[t] = limit >= KB ? ~0u : (1u << limit) - 1u;
      cache_block<T, DP, RT, EXACT, true>(z, c8.k + at + (int64_t)i * KB * c8.slot_stride, c8.v + at + (int64_t)i * KB * c8.slot_stride,
                                          c8.slot_stride, c8.k_exp[eat + i], c8.v_exp[eat + i], limit, a.head_dim, cut.scale, on);
    } else {
      const int key0 = (i - cached) * KB;
#pragma unroll
      for (int t = 0; t < RT; t++) on[t] = (uint32_t)(mine[t] >> key0);
      const int64_t f = b * a.fresh.seq_stride + kh * a.fresh.head_stride;
      tree_block<T, DP, RT, EXACT>(z, (const uint16_t*)a.fresh.k + f, (const uint16_t*)a.fresh.v + f, a.fresh.slot_stride, key0, sq.n,
                                   a.head_dim, cut.scale, on);
    }
  }

  // the waves' sums, brought to one reference; rows that see nothing of the
  // tree see nothing of the cache either
  float ref[RT];
  if (lane == 0) odds[wave] = z.w.odd;
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
    for (int k = 0; k < S::NF; k++) sum[wave][t][k][lane] = ref[t] == NEG_INF ? (f32x4){0.0f, 0.0f, 0.0f, 0.0f} : z.w.o[t][k] * f;
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
      store_pair<T, DP, E4m3>(a, cut.G, b, kh, row0 + 16 * t + x, R, h, pair, o[0], o[1], top, all, odd, sq.n);
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

}  // namespace xs8

// ---------------------------------------------------------------------------
// Host side.

namespace {

using xs_host::OnDevice;
using xs_host::per_cu;
using xs_host::rounds;

template <typename T, int DP, int RT, bool EXACT>
int attend8_run(xs_cache_context* c, const xs_tree_attend_args& a, const xs_kv8& c8) {
  xst::Cut cut;
  cut.G = (int32_t)(a.q_heads / a.kv_heads);
  cut.tiles = (int32_t)((a.nodes * cut.G + 16 * RT - 1) / (16 * RT));
  cut.scale = a.scale * xst::LOG2E;
  cut.part = c->part;
  const int64_t limit = a.max_len ? a.max_len : a.capacity;
  const int64_t blocks = (limit + xst::KB - 1) / xst::KB + (a.nodes + xst::KB - 1) / xst::KB;
  const int64_t units = a.seqs * a.kv_heads * cut.tiles;
  const int64_t most = c->n_cu * per_cu(DP, RT) * rounds(a.seqs);
  const int64_t nsplit = std::max<int64_t>(1, std::min<int64_t>(xst::SPLITS, most / units));
  cut.chunk = (int32_t)((blocks + nsplit - 1) / nsplit);
  if (cut.chunk < 2 * xst::NW) cut.chunk = 2 * xst::NW;
  if (blocks <= 4 * xst::NW) cut.chunk = (int32_t)blocks;
  cut.nsplit = (int32_t)((blocks + cut.chunk - 1) / cut.chunk);
  const int64_t groups = a.seqs * a.kv_heads * cut.nsplit;
  const int64_t grid = (groups + 7) / 8 * 8 * cut.tiles, join = a.seqs * a.kv_heads * cut.tiles * RT * xst::Shape<DP, RT>::VH;
  const int64_t joiners = xst::join_threads<DP>(cut.nsplit <= xst::FEW);
  if (!xs_host_launch_fits(grid, 64 * xst::NW) || (cut.nsplit > 1 && !xs_host_launch_fits(join, joiners))) return XS_ERR_CAPACITY;
  if (cut.nsplit > 1 && groups * cut.tiles * xst::Shape<DP, RT>::PART > c->part_floats) return XS_ERR_CAPACITY;  // (never: groups * tiles <= most)
  cut.groups = (int32_t)groups;
  hipLaunchKernelGGL((xs8::attend8_kernel<T, DP, RT, EXACT>), dim3((unsigned)grid), dim3(64 * xst::NW), 0, c->stream, a, c8, cut);
  if (cut.nsplit > xst::FEW)
    hipLaunchKernelGGL((xst::join_kernel<T, DP, RT, false, xs8::E4m3>), dim3((unsigned)join), dim3(xst::join_threads<DP>(false)), 0, c->stream, a, cut);
  else if (cut.nsplit > 1)
    hipLaunchKernelGGL((xst::join_kernel<T, DP, RT, true, xs8::E4m3>), dim3((unsigned)join), dim3(xst::join_threads<DP>(true)), 0, c->stream, a, cut);
  return hipGetLastError() == hipSuccess ? XS_OK : XS_ERR_HIP;
}

template <typename T, int DP, int RT>
int attend8_exact(xs_cache_context* c, const xs_tree_attend_args& a, const xs_kv8& c8) {
  return a.head_dim == DP ? attend8_run<T, DP, RT, true>(c, a, c8) : attend8_run<T, DP, RT, false>(c, a, c8);
}

template <typename T, int DP>
int attend8_rows(xs_cache_context* c, const xs_tree_attend_args& a, const xs_kv8& c8) {
  const int64_t rows = a.nodes * (a.q_heads / a.kv_heads);
  if (rows <= 16) return attend8_exact<T, DP, 1>(c, a, c8);
  if constexpr (DP <= 128) {
    if (rows > 32) return attend8_exact<T, DP, 4>(c, a, c8);
  }
  return attend8_exact<T, DP, 2>(c, a, c8);
}

template <typename T>
int attend8_dim(xs_cache_context* c, const xs_tree_attend_args& a, const xs_kv8& c8) {
  if (a.head_dim <= 64) return attend8_rows<T, 64>(c, a, c8);
  if (a.head_dim <= 128) return attend8_rows<T, 128>(c, a, c8);
  return attend8_rows<T, 256>(c, a, c8);
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
