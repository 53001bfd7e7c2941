// xs_tree.hip -- a tree of drafted tokens over a bounded cache (MI355X, gfx950):
// attention of the tree's nodes, the commit of the accepted path with the
// attention weight it gave, and the eviction of the slots with the least.
//
// Compiled with -ffp-contract=off; fused multiply-adds are written out.

#include <hip/hip_runtime.h>

#include <algorithm>
#include <stdint.h>
#include <stdlib.h>

#include "../../include/xsamp.h"
#include "xs_attend.h"
#include "xs_cache.h"
#include "xs_device.h"
#include "xs_host.h"

namespace xst {

// grid: groups of eight (sequence, kv head, split), each group's row tiles on
// one XCD (workgroup index mod 8), which then reads their keys once.
template <typename T, int DP, int RT, bool EXACT>
__global__ __launch_bounds__(64 * NW, DP * RT <= 64 ? 4 : DP * RT <= 128 ? 3 : DP * RT <= 256 ? 2 : 1) void attend_kernel(const xs_tree_attend_args a, const Cut cut) {
  using S = Shape<DP, RT>;
  __shared__ float stat[NW][RT][2][16];
  __shared__ f32x4 sum[NW][RT][S::NF][64];
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
    block<T, DP, RT, EXACT, false>(w, ck, cv, a.cache.slot_stride, i * KB, sq.len, a.head_dim, cut.scale, nullptr, WALK);
  // its last one, and the tree's
  const uint64_t sees = ancestors(parent, sq.n);
  uint64_t mine[RT];  // what the lane's rows see of the tree
#pragma unroll
  for (int t = 0; t < RT; t++) {
    const int row = row0 + 16 * t + x;
    mine[t] = __shfl(sees, min(row / cut.G, 63));
    if (row >= R) mine[t] = 0;
  }
  auto rest = [&](int i, auto pass) __attribute__((always_inline)) {
#pragma unroll 1
    for (; i < last; i += NW) {
      const bool in_tree = i >= cached;
      const int key0 = (in_tree ? i - cached : i) * KB, limit = in_tree ? sq.n : sq.len;
      const xs_kv& kv = in_tree ? a.fresh : a.cache;
      const int64_t at = b * kv.seq_stride + kh * kv.head_stride;
      uint32_t on[RT];
#pragma unroll
      for (int t = 0; t < RT; t++)
        on[t] = in_tree ? (uint32_t)(mine[t] >> key0) : sq.len - key0 >= KB ? ~0u : (1u << (sq.len - key0)) - 1u;
      block<T, DP, RT, EXACT, true>(w, (const uint16_t*)kv.k + at, (const uint16_t*)kv.v + at, kv.slot_stride, key0, limit, a.head_dim,
                                    cut.scale, on, pass);
    }
  };
  rest(i, std::integral_constant<int, WALK>{});
  uint32_t* marked = (uint32_t*)&sum[wave] + lane;
  if (!finished(w, WALK, mine, marked)) [[unlikely]] {
    int pass = ABOVE;
#pragma unroll 1
    do rest(first + wave, pass);
    while (!finished(w, pass++, mine, marked));
  }

  // the waves' sums, brought to one reference; rows that see nothing of the
  // tree see nothing of the cache either
  float ref[RT];
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
    for (int k = 0; k < S::NF; k++) sum[wave][t][k][lane] = times(w.o[t][k], f);
  }
  __syncthreads();
  // a wave takes every fourth pair of fragments
  constexpr int PAIRS = S::VE / 2;
  const bool whole = first == 0 && last == total;
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
      store_pair<T, DP>(a, cut.G, b, kh, row0 + 16 * t + x, R, h, pair, o[0], o[1], top, all);
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
  __shared__ uint32_t marks[NW][2 * S::MARKS][64];
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
  auto rest = [&](int i, auto pass) __attribute__((always_inline)) {
#pragma unroll 1
    for (; i < last; i++) {
      const bool in_tree = i >= cached;
      const int key0 = (in_tree ? i - cached : i) * KB, limit = in_tree ? sq.n : sq.len;
      const xs_kv& kv = in_tree ? a.fresh : a.cache;
      const int64_t at = b * kv.seq_stride + kh * kv.head_stride;
      uint32_t on[RT];
#pragma unroll
      for (int t = 0; t < RT; t++)
        on[t] = in_tree ? (uint32_t)(mine[t] >> key0) : sq.len - key0 >= KB ? ~0u : (1u << (sq.len - key0)) - 1u;
      block<T, DP, RT, EXACT, true>(w, (const uint16_t*)kv.k + at, (const uint16_t*)kv.v + at, kv.slot_stride, key0, limit, a.head_dim,
                                    cut.scale, on, pass);
    }
  };
  rest(first + stages * SB, std::integral_constant<int, WALK>{});
  uint32_t* marked = &marks[wave][0][lane];
  if (!finished(w, WALK, mine, marked)) [[unlikely]] {
    int pass = ABOVE;
#pragma unroll 1
    do rest(first, pass);
    while (!finished(w, pass++, mine, marked));
  }
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
    if (whole) {
#pragma unroll
      for (int h = 0; h < S::VH; h++) store_half<T, DP, RT>(a, cut.G, b, kh, row0 + 16 * t + x, R, h, w.o[t], ref, l);
    } else {
#pragma unroll
      for (int f = 0; f < S::NF; f++) ((f32x4*)part)[(t * S::NF + f) * 64 + lane] = w.o[t][f];
      if (g == 0) {
        part[S::STAT + 32 * t + x] = ref;
        part[S::STAT + 32 * t + 16 + x] = l;
      }
    }
  }
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

namespace {

using xs_host::per_cu;
using xs_host::rounds;

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
