// xs_tree.hip -- a tree of drafted tokens over a bounded cache (MI355X, gfx950):
// attention of the tree's nodes, the commit of the accepted path with the
// attention weight it gave, and the eviction of the slots with the least.
//
// Compiled with -ffp-contract=off; fused multiply-adds are written out.

#include <hip/hip_runtime.h>

#include <math.h>
#include <stdint.h>
#include <stdlib.h>
#include <string.h>

#include "../../include/xsamp.h"
#include "xs_host.h"

#define XS_DEV __device__ __forceinline__

namespace xst {

constexpr float LOG2E = 1.44269504088896340736f;
constexpr float LN2 = 0.69314718055994530942f;
constexpr float NEG_INF = -__builtin_huge_valf();

// Elements of the two types as f32.
struct Bf16 {
  XS_DEV static float widen(uint16_t u) { return __uint_as_float((uint32_t)u << 16); }
  // round to nearest even; NaN stays NaN
  XS_DEV static uint16_t narrow(float f) {
    const uint32_t u = __float_as_uint(f);
    if (f != f) return (uint16_t)((u >> 16) | 0x40u);
    return (uint16_t)((u + 0x7FFFu + ((u >> 16) & 1u)) >> 16);
  }
};
struct F16 {
  XS_DEV static float widen(uint16_t u) { return (float)__builtin_bit_cast(_Float16, u); }
  XS_DEV static uint16_t narrow(float f) { return __builtin_bit_cast(uint16_t, (_Float16)f); }
};

// The nodes a node sees: bit j of lane i's result is set when j is i or an
// ancestor of i; 0 where i's chain of parents does not end in -1 by way of
// ever lower nodes below n.  Each round doubles the distance a lane has gone
// up, so six rounds reach the root from any of 64 nodes.  One whole wave.
XS_DEV uint64_t ancestors(const int32_t* parent, int n) {
  const int lane = threadIdx.x & 63;
  int up = -2;  // -1: at the root; -2: the chain is broken
  if (lane < n) {
    const int p = parent[lane];
    up = p == -1 ? -1 : (p >= 0 && p < lane ? p : -2);
  }
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

// One wave per (sequence, node, q head): the keys in blocks of 64, a lane's
// key each for the scores, a lane's elements of the head each for the values.
template <typename T>
__global__ __launch_bounds__(64) void attend_kernel(const xs_tree_attend_args a) {
  __shared__ float qs[256];
  const int lane = threadIdx.x, D = a.head_dim;
  const int h = blockIdx.x % a.q_heads, i = (blockIdx.x / a.q_heads) % a.nodes, b = blockIdx.x / (a.q_heads * a.nodes);
  const int64_t limit = a.max_len ? a.max_len : a.capacity;
  const int len = a.len[b], n = a.n_nodes ? a.n_nodes[b] : (int)a.nodes;
  const bool bad = len < 0 || len > limit || n < 0 || n > a.nodes;
  if (h == 0 && i == 0 && lane == 0) a.seq_status[b] = bad ? XS_ROW_BAD_PARAM : XS_ROW_OK;
  if (bad || i >= n) return;
  const int kh = h / (int)(a.q_heads / a.kv_heads);
  const uint16_t* q = (const uint16_t*)a.q + b * a.q_seq_stride + i * a.q_node_stride + h * a.q_head_stride;
  for (int d = lane; d < 256; d += 64) qs[d] = d < D ? T::widen(q[d]) : 0.0f;
  __syncthreads();
  const uint64_t seen = __shfl(ancestors(a.parent + b * a.nodes, n), i);
  float m = NEG_INF, l = 0.0f, acc[4] = {0.0f, 0.0f, 0.0f, 0.0f};
  const int total = seen ? len + n : 0;
  for (int s0 = 0; s0 < total; s0 += 64) {
    const int s = s0 + lane;
    const bool on = s < len || (s < total && ((seen >> (s - len)) & 1ull));
    float x = NEG_INF;
    if (on) {
      const uint16_t* k = s < len ? (const uint16_t*)a.cache.k + b * a.cache.seq_stride + s * a.cache.slot_stride + kh * a.cache.head_stride
                                  : (const uint16_t*)a.fresh.k + b * a.fresh.seq_stride + (s - len) * a.fresh.slot_stride + kh * a.fresh.head_stride;
      float dot = 0.0f;
      for (int d = 0; d < D; d++) dot = __builtin_fmaf(qs[d], T::widen(k[d]), dot);
      x = dot * a.scale;
    }
    float top = x;
    for (int o = 32; o; o >>= 1) top = fmaxf(top, __shfl_xor(top, o));
    const float mn = fmaxf(m, top);
    const float shift = mn == NEG_INF ? 0.0f : mn;
    const float keep = expf(m - shift);
    const float p = on ? expf(x - shift) : 0.0f;
    m = mn;
    float sum = p;
    for (int o = 32; o; o >>= 1) sum += __shfl_xor(sum, o);
    l = l * keep + sum;
    for (int e = 0; e < 4; e++) acc[e] *= keep;
    const uint64_t live = __ballot(on);
    for (int j = 0; j < 64; j++) {
      if (!((live >> j) & 1ull)) continue;
      const int t = s0 + j;
      const float w = __shfl(p, j);
      const uint16_t* v = t < len ? (const uint16_t*)a.cache.v + b * a.cache.seq_stride + t * a.cache.slot_stride + kh * a.cache.head_stride
                                  : (const uint16_t*)a.fresh.v + b * a.fresh.seq_stride + (t - len) * a.fresh.slot_stride + kh * a.fresh.head_stride;
      for (int e = 0; e < 4; e++)
        if (lane + 64 * e < D) acc[e] = __builtin_fmaf(w, T::widen(v[lane + 64 * e]), acc[e]);
    }
  }
  uint16_t* out = (uint16_t*)a.out + b * a.out_seq_stride + i * a.out_node_stride + h * a.out_head_stride;
  for (int e = 0; e < 4; e++)
    if (lane + 64 * e < D) out[lane + 64 * e] = T::narrow(l == 0.0f ? 0.0f : acc[e] / l);
  if (a.lse && lane == 0) a.lse[(b * a.nodes + i) * a.q_heads + h] = l == 0.0f ? NEG_INF : m + logf(l);
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

// One wave per (sequence, kv head, block of 64 slots), a lane a slot; the last
// block of a head appends the path instead.
template <typename T>
__global__ __launch_bounds__(64) void commit_kernel(const xs_cache_commit_args a, int blocks) {
  const int lane = threadIdx.x, D = a.head_dim;
  const int blk = blockIdx.x % blocks, kh = (blockIdx.x / blocks) % a.kv_heads, b = blockIdx.x / (blocks * a.kv_heads);
  const int64_t limit = a.max_len ? a.max_len : a.capacity;
  const int len = a.len[b], G = (int)(a.q_heads / a.kv_heads);
  int node, m;
  const int st = read_path(a, b, len, limit, &node, &m);
  const bool tail = blk == blocks - 1;
  if (tail && kh == 0 && lane == 0) {
    a.seq_status[b] = st;
    a.new_len[b] = st == XS_ROW_OK ? len + m : len;
    if (a.pos) a.new_next_pos[b] = a.next_pos[b] + (st == XS_ROW_OK ? m : 0);
  }
  if (st != XS_ROW_OK) return;
  const int64_t slots = (b * a.kv_heads + kh) * a.slot_ld;
  const int s = tail ? lane : blk * 64 + lane;
  if (a.q && s < (tail ? m : len)) {
    const uint16_t* k = tail ? (const uint16_t*)a.fresh.k + b * a.fresh.seq_stride + node * a.fresh.slot_stride + kh * a.fresh.head_stride
                             : (const uint16_t*)a.cache.k + b * a.cache.seq_stride + s * a.cache.slot_stride + kh * a.cache.head_stride;
    float sum = 0.0f;
    for (int r = tail ? s : 0; r < m; r++) {
      const int64_t i = a.path[b * a.path_ld + r];
      for (int g = 0; g < G; g++) {
        const int h = kh * G + g;
        const uint16_t* q = (const uint16_t*)a.q + b * a.q_seq_stride + i * a.q_node_stride + h * a.q_head_stride;
        const float lse = a.lse[(b * a.nodes + i) * a.q_heads + h];
        float dot = 0.0f;
        for (int d = 0; d < D; d++) dot = __builtin_fmaf(T::widen(q[d]), T::widen(k[d]), dot);
        if (lse != NEG_INF) sum += expf(dot * a.scale - lse);
      }
    }
    if (tail) a.new_mass[slots + len + s] = sum;
    else a.new_mass[slots + s] = a.mass[slots + s] + sum;
  }
  if (!tail) return;
  if (a.pos && lane < m) a.pos[slots + len + lane] = a.next_pos[b] + lane;
  for (int r = 0; r < m; r++) {
    const int64_t i = __builtin_amdgcn_readlane(node, r);
    const int64_t from = b * a.fresh.seq_stride + i * a.fresh.slot_stride + kh * a.fresh.head_stride;
    const int64_t to = b * a.cache.seq_stride + (len + r) * a.cache.slot_stride + kh * a.cache.head_stride;
    for (int d = lane; d < D; d += 64) {
      ((uint16_t*)a.cache.k)[to + d] = ((const uint16_t*)a.fresh.k)[from + d];
      ((uint16_t*)a.cache.v)[to + d] = ((const uint16_t*)a.fresh.v)[from + d];
    }
  }
}

// A slot's place in the order of xs_cache_evict, larger first: the held slots
// above all others, then the weights (the bits of an f32 put in order; NaN
// below -inf), ties to the lower position.
XS_DEV uint64_t rank_key(float mass, int pos, bool held) {
  const uint32_t u = __float_as_uint(mass + 0.0f);  // (-0 as 0)
  const uint32_t w = mass != mass ? 0u : (u & 0x80000000u ? ~u : u | 0x80000000u);
  return ((uint64_t)(held ? 0xFFFFFFFFu : w) << 32) | (uint32_t)~((uint32_t)pos ^ 0x80000000u);
}

// kept[slot] by counting the slots before it.
__global__ __launch_bounds__(256) void evict_rank_kernel(const xs_cache_evict_args a, uint8_t* kept, int blocks) {
  const int blk = blockIdx.x % blocks;
  const int64_t bh = blockIdx.x / blocks;
  const int b = (int)(bh / a.kv_heads);
  const int64_t limit = a.max_len ? a.max_len : a.capacity;
  const int len = a.len[b];
  const int s = blk * 256 + threadIdx.x;
  if (len < 0 || len > limit || len <= a.keep || s >= len) return;
  const float* mass = a.mass + bh * a.slot_ld;
  const int32_t* pos = a.pos + bh * a.slot_ld;
  const int64_t next = a.next_pos[b];
  auto key = [&](int t) { return rank_key(mass[t], pos[t], pos[t] < a.sinks || pos[t] >= next - a.recent); };
  const uint64_t mine = key(s);
  int before = 0;
  for (int t = 0; t < len; t++) {
    const uint64_t k = key(t);
    before += k > mine || (k == mine && t < s);
  }
  kept[bh * a.capacity + s] = before < a.keep;
}

// One wave per (sequence, kv head): pairs each free slot with its filler.
__global__ __launch_bounds__(64) void evict_move_kernel(const xs_cache_evict_args a, const uint8_t* kept) {
  const int64_t bh = blockIdx.x;
  const int b = (int)(bh / a.kv_heads), kh = (int)(bh % a.kv_heads), lane = threadIdx.x;
  const int64_t limit = a.max_len ? a.max_len : a.capacity;
  const int len = a.len[b];
  const bool bad = len < 0 || len > limit;
  const int keep = (int)min((int64_t)len, a.keep);
  if (kh == 0 && lane == 0) {
    a.seq_status[b] = bad ? XS_ROW_BAD_PARAM : XS_ROW_OK;
    a.new_len[b] = bad ? len : keep;
  }
  if (bad) return;
  const int64_t slots = bh * a.slot_ld;
  if (a.new_mass != a.mass)
    for (int s = lane; s < keep; s += 64) {
      a.new_mass[slots + s] = a.mass[slots + s];
      a.new_pos[slots + s] = a.pos[slots + s];
    }
  if (len <= keep) return;
  __syncthreads();
  const uint8_t* mine = kept + bh * a.capacity;
  int filler = keep;
  for (int s = 0; s < keep; s++) {
    if (mine[s]) continue;
    while (!mine[filler]) filler++;
    if (lane == 0) {
      a.new_mass[slots + s] = a.mass[slots + filler];
      a.new_pos[slots + s] = a.pos[slots + filler];
    }
    const int64_t row = b * a.cache.seq_stride + kh * a.cache.head_stride;
    for (int d = lane; d < a.head_dim; d += 64) {
      ((uint16_t*)a.cache.k)[row + s * a.cache.slot_stride + d] = ((const uint16_t*)a.cache.k)[row + filler * a.cache.slot_stride + d];
      ((uint16_t*)a.cache.v)[row + s * a.cache.slot_stride + d] = ((const uint16_t*)a.cache.v)[row + filler * a.cache.slot_stride + d];
    }
    filler++;
  }
}

}  // namespace xst

// ---------------------------------------------------------------------------
// Host side: the cache context and its calls.

struct xs_cache_context {
  int device;
  hipStream_t stream;
  xs_cache_dims dims;
  uint8_t* kept;  // [max_seqs, kv_heads, capacity]
};

extern "C" {

int xs_cache_create(int device, const xs_cache_dims* dims, xs_cache_context** out) {
  if (!out) return XS_ERR_ARG;
  *out = nullptr;
  const int rc = xs_host_check_dims(dims);
  if (rc) return rc;
  if (hipSetDevice(device) != hipSuccess) return XS_ERR_HIP;
  xs_cache_context* c = (xs_cache_context*)calloc(1, sizeof(xs_cache_context));
  if (!c) return XS_ERR_HIP;
  c->device = device;
  c->dims = *dims;
  if (hipMalloc((void**)&c->kept, dims->max_seqs * dims->kv_heads * dims->capacity) != hipSuccess) {
    xs_cache_destroy(c);
    return XS_ERR_HIP;
  }
  *out = c;
  return XS_OK;
}

int xs_cache_destroy(xs_cache_context* c) {
  if (!c) return XS_OK;
  (void)hipSetDevice(c->device);
  if (c->stream) (void)hipStreamSynchronize(c->stream); else (void)hipDeviceSynchronize();
  if (c->kept) (void)hipFree(c->kept);
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
  if (hipSetDevice(c->device) != hipSuccess) return XS_ERR_HIP;
  const int64_t grid = in->seqs * in->nodes * in->q_heads;
  if (grid > 0x7FFFFFFF) return XS_ERR_CAPACITY;
  if (in->dtype == XS_BF16) hipLaunchKernelGGL(xst::attend_kernel<xst::Bf16>, dim3((unsigned)grid), dim3(64), 0, c->stream, *in);
  else hipLaunchKernelGGL(xst::attend_kernel<xst::F16>, dim3((unsigned)grid), dim3(64), 0, c->stream, *in);
  return hipGetLastError() == hipSuccess ? XS_OK : XS_ERR_HIP;
}

int xs_cache_commit(xs_cache_context* c, const xs_cache_commit_args* in) {
  const int rc = xs_host_check_commit(c ? &c->dims : nullptr, in);
  if (rc) return rc;
  if (in->seqs == 0) return XS_OK;
  if (hipSetDevice(c->device) != hipSuccess) return XS_ERR_HIP;
  const int64_t limit = in->max_len ? in->max_len : in->capacity;
  const int64_t blocks = in->q ? (limit + 63) / 64 + 1 : 1;
  const int64_t grid = in->seqs * in->kv_heads * blocks;
  if (grid > 0x7FFFFFFF) return XS_ERR_CAPACITY;
  if (in->dtype == XS_BF16) hipLaunchKernelGGL(xst::commit_kernel<xst::Bf16>, dim3((unsigned)grid), dim3(64), 0, c->stream, *in, (int)blocks);
  else hipLaunchKernelGGL(xst::commit_kernel<xst::F16>, dim3((unsigned)grid), dim3(64), 0, c->stream, *in, (int)blocks);
  return hipGetLastError() == hipSuccess ? XS_OK : XS_ERR_HIP;
}

int xs_cache_evict(xs_cache_context* c, const xs_cache_evict_args* in) {
  const int rc = xs_host_check_evict(c ? &c->dims : nullptr, in);
  if (rc) return rc;
  if (in->seqs == 0) return XS_OK;
  if (hipSetDevice(c->device) != hipSuccess) return XS_ERR_HIP;
  const int64_t limit = in->max_len ? in->max_len : in->capacity;
  const int64_t blocks = (limit + 255) / 256, grid = in->seqs * in->kv_heads * blocks;
  if (grid > 0x7FFFFFFF) return XS_ERR_CAPACITY;
  if (limit > in->keep)
    hipLaunchKernelGGL(xst::evict_rank_kernel, dim3((unsigned)grid), dim3(256), 0, c->stream, *in, c->kept, (int)blocks);
  hipLaunchKernelGGL(xst::evict_move_kernel, dim3((unsigned)(in->seqs * in->kv_heads)), dim3(64), 0, c->stream, *in, c->kept);
  return hipGetLastError() == hipSuccess ? XS_OK : XS_ERR_HIP;
}

}  // extern "C"
