// xs_host.cpp -- the host-only part of the C ABI: the argument checks of the
// device entry points, and the host entry points xs_select_option
// (select_option, batch.rs:1545-1588) and xs_keep_confident (keep_confident,
// generate.rs:3898-3905).  Plain C++: libxsamp.so links it, and oracle/Makefile
// builds it alone under AddressSanitizer and UBSan (target asan).
#include "xs_host.h"

#include <math.h>
#include <string.h>

#include <algorithm>
#include <cmath>
#include <utility>
#include <vector>

namespace {

bool aligned16(const void* p) { return ((uintptr_t)p & 15u) == 0; }

// The checks every device call shares: pointers, sizes, alignment, capacity.
int check_common(const xs_host_limits* lim, const float* logits, int64_t rows, int64_t ld,
                 int64_t width, int64_t enc, const void* params, const float* uniforms,
                 const uint32_t* allowed, int64_t allowed_words, int64_t allowed_ld) {
  if (!lim || !logits || !params || !uniforms) return XS_ERR_ARG;
  if (rows < 0 || enc < 1 || ld < 1) return XS_ERR_ARG;
  if (rows > lim->max_rows || enc > lim->vocab) return XS_ERR_CAPACITY;
  if (ld % 4 != 0 || !aligned16(logits)) return XS_ERR_ARG;
  if (width > ld) return XS_ERR_ARG;
  if (enc > ld && width >= enc) return XS_ERR_ARG;
  if (allowed && (allowed_ld < allowed_words || allowed_words < 0)) return XS_ERR_ARG;
  if (xs_host::chunks_for(enc) > lim->max_chunks) return XS_ERR_CAPACITY;
  return XS_OK;
}

// The last element of [n0, n1, n2, head_dim] by these strides lies within a
// 64-bit offset (of elements of 8 bytes at most).
bool spans_fit(int64_t n0, int64_t s0, int64_t n1, int64_t s1, int64_t n2, int64_t s2) {
  int64_t a, b, c, d;
  if (__builtin_mul_overflow(n0, s0, &a) || __builtin_mul_overflow(n1, s1, &b) || __builtin_mul_overflow(n2, s2, &c))
    return false;
  return !__builtin_add_overflow(a, b, &d) && !__builtin_add_overflow(d, c, &d) && d < (INT64_MAX >> 4);
}

// Strides of rows of head_dim elements that 16-byte loads reach.  Rows that
// the call writes may not overlap: taken from the smallest stride up, each
// passes over all that the smaller ones span (an input may repeat its rows,
// stride 0).
bool strides_ok(int64_t n0, int64_t s0, int64_t n1, int64_t s1, int64_t n2, int64_t s2, int64_t head_dim, bool written) {
  if (s0 < 0 || s1 < 0 || s2 < 0 || s0 % 8 || s1 % 8 || s2 % 8) return false;
  if (!spans_fit(n0, s0, n1, s1, n2, s2)) return false;
  if (!written) return true;
  std::pair<int64_t, int64_t> d[3] = {{s0, n0}, {s1, n1}, {s2, n2}};
  std::sort(d, d + 3);
  int64_t extent = head_dim;
  for (const auto& [s, n] : d) {
    if (n <= 1) continue;
    if (s < extent) return false;
    extent += s * (n - 1);
  }
  return true;
}

bool kv_ok(const xs_kv& kv, int64_t seqs, int64_t slots, int64_t kv_heads, int64_t head_dim, bool written) {
  return kv.k && kv.v && aligned16(kv.k) && aligned16(kv.v) &&
         strides_ok(seqs, kv.seq_stride, slots, kv.slot_stride, kv_heads, kv.head_stride, head_dim, written);
}

// The same in bytes, of which 16 are a load; and the exponents.
bool kv8_ok(const xs_kv8& kv, int64_t seqs, int64_t slots, int64_t kv_heads, int64_t head_dim, bool written) {
  return kv.k && kv.v && kv.k_exp && kv.v_exp && aligned16(kv.k) && aligned16(kv.v) && kv.seq_stride % 16 == 0 &&
         kv.slot_stride % 16 == 0 && kv.head_stride % 16 == 0 && kv.exp_ld >= (slots + XS_CACHE8_BLOCK - 1) / XS_CACHE8_BLOCK &&
         kv.exp_ld <= (INT64_MAX >> 4) / kv_heads / (seqs > 0 ? seqs : 1) &&
         strides_ok(seqs, kv.seq_stride, slots, kv.slot_stride, kv_heads, kv.head_stride, head_dim, written);
}

// Two per-sequence arrays share no entry.
bool apart(const int32_t* p, const int32_t* q, int64_t seqs) {
  const uintptr_t x = (uintptr_t)p, y = (uintptr_t)q, n = (uintptr_t)seqs * sizeof(int32_t);
  return x + n <= y || y + n <= x;
}

// Per-slot arrays [seqs, kv_heads, slot_ld] lie within a 64-bit offset.
bool slots_fit(int64_t seqs, int64_t kv_heads, int64_t slot_ld) {
  return slot_ld <= (INT64_MAX >> 4) / kv_heads / (seqs > 0 ? seqs : 1);
}

// The sizes every cache call shares, against what its context holds.
int check_sizes(const xs_cache_dims* dims, int32_t dtype, int64_t head_dim, int64_t seqs, int64_t kv_heads,
                int64_t capacity, int64_t max_len) {
  if (dtype != XS_BF16 && dtype != XS_F16) return XS_ERR_ARG;
  if (head_dim < 8 || head_dim > 256 || head_dim % 8) return XS_ERR_ARG;
  if (seqs < 0 || kv_heads < 1 || capacity < 1 || max_len < 0 || max_len > capacity) return XS_ERR_ARG;
  if (seqs > dims->max_seqs || kv_heads > dims->kv_heads || head_dim > dims->head_dim || capacity > dims->capacity)
    return XS_ERR_CAPACITY;
  return XS_OK;
}

int check_queries(const xs_cache_dims* dims, int64_t nodes, int64_t q_heads, int64_t kv_heads) {
  if (nodes < 1 || nodes > XS_TREE_MAX || q_heads < 1 || q_heads % kv_heads) return XS_ERR_ARG;
  return nodes > dims->max_nodes || q_heads > dims->q_heads ? XS_ERR_CAPACITY : XS_OK;
}

}  // namespace

extern "C" {

bool xs_host_wants_lse(const xs_sample_args* in) {
  return in->row_max || in->row_lse || in->top_id || in->top_logprob || in->top_logprob64 ||
         in->score_ids || in->class_masks || in->probs;
}

bool xs_host_wants_scores(const xs_sample_args* in) {
  return in->score_ids || in->class_masks || in->probs;
}

int xs_host_check_sample(const xs_host_limits* lim, const xs_sample_args* in) {
  if (!lim || !in || !in->token || !in->status) return XS_ERR_ARG;
  const int rc = check_common(lim, in->logits, in->rows, in->ld, in->width, in->enc, in->params,
                              in->uniforms, in->allowed, in->allowed_words, in->allowed_ld);
  if (rc) return rc;
  if ((in->cand_id || in->cand_w) && in->cand_ld < 1) return XS_ERR_ARG;
  if (in->k_max < 0) return XS_ERR_ARG;
  if (in->n_top < 0 || in->n_top > XS_TOP_MAX) return XS_ERR_ARG;
  if ((in->top_id || in->top_logprob || in->top_logprob64) && in->top_ld < in->n_top) return XS_ERR_ARG;
  // the scoring reads (generate.rs:1871-1899)
  if (in->score_logprob && !in->score_ids) return XS_ERR_ARG;
  if (in->score_ids && (!in->score_logprob || in->n_score < 0 || in->n_score > XS_SCORE_MAX ||
                        in->score_ld < in->n_score))
    return XS_ERR_ARG;
  if ((in->class_masks != nullptr) != (in->class_mass != nullptr)) return XS_ERR_ARG;
  if (in->class_masks && (in->n_class < 0 || in->n_class > XS_CLASS_MAX || in->class_ld < (in->enc + 31) / 32))
    return XS_ERR_ARG;
  if (in->probs && in->probs_ld < in->enc) return XS_ERR_ARG;
  if (in->row_order) {  // a permutation of 0..rows-1 (a longer one is checked, then not applied)
    uint64_t small[XS_ORDER_MAX / 64] = {};
    std::vector<uint64_t> large;
    uint64_t* seen = small;
    if (in->rows > XS_ORDER_MAX) {
      large.assign((size_t)((in->rows + 63) / 64), 0ull);
      seen = large.data();
    }
    for (int64_t i = 0; i < in->rows; i++) {
      const int32_t r = in->row_order[i];
      if (r < 0 || r >= in->rows || ((seen[r >> 6] >> (r & 63)) & 1u)) return XS_ERR_ARG;
      seen[r >> 6] |= 1ull << (r & 63);
    }
  }
  return XS_OK;
}

int xs_host_check_verify(const xs_host_limits* lim, const xs_verify_args* in) {
  if (!lim || !in || !in->row_token || !in->row_status || !in->accepted || !in->committed ||
      !in->n_committed || !in->seq_status)
    return XS_ERR_ARG;
  if (in->seqs < 0 || in->span < 1 || in->n_eog < 0 || in->k_max < 0) return XS_ERR_ARG;
  if (in->n_eog > 0 && !in->eog) return XS_ERR_ARG;
  if (in->span > 1 && !in->drafts) return XS_ERR_ARG;
  if (in->seqs > INT64_MAX / in->span) return XS_ERR_CAPACITY;
  return check_common(lim, in->logits, in->seqs * in->span, in->ld, in->width, in->enc, in->params,
                      in->uniforms, in->allowed, in->allowed_words, in->allowed_ld);
}

int xs_host_check_verify_tree(const xs_host_limits* lim, const xs_verify_tree_args* in) {
  if (!lim || !in) return XS_ERR_ARG;
  if (in->seqs < 0 || in->nodes < 1 || in->nodes > XS_TREE_MAX || in->n_eog < 0 || in->k_max < 0) return XS_ERR_ARG;
  if (in->seqs == 0) return XS_OK;
  if (!in->row_token || !in->row_status || !in->accepted || !in->path || !in->committed || !in->n_committed ||
      !in->seq_status || !in->tokens || !in->parent)
    return XS_ERR_ARG;
  if (in->n_eog > 0 && !in->eog) return XS_ERR_ARG;
  if (in->seqs > INT64_MAX / in->nodes) return XS_ERR_CAPACITY;
  return check_common(lim, in->logits, in->seqs * in->nodes, in->ld, in->width, in->enc, in->params,
                      in->uniforms, in->allowed, in->allowed_words, in->allowed_ld);
}

int xs_host_check_dims(const xs_cache_dims* d) {
  if (!d || d->max_seqs < 1 || d->max_nodes < 1 || d->max_nodes > XS_TREE_MAX || d->q_heads < 1 || d->kv_heads < 1 ||
      d->head_dim < 8 || d->head_dim > 256 || d->capacity < 1)
    return XS_ERR_ARG;
  // slots and rows are counted in 32 bits
  if (d->max_seqs > 65536 || d->q_heads > 4096 || d->kv_heads > d->q_heads || d->capacity > (1 << 28)) return XS_ERR_CAPACITY;
  return XS_OK;
}

int xs_host_check_attend(const xs_cache_dims* dims, const xs_tree_attend_args* in) {
  if (!dims || !in) return XS_ERR_ARG;
  int rc = check_sizes(dims, in->dtype, in->head_dim, in->seqs, in->kv_heads, in->capacity, in->max_len);
  if (rc == XS_OK) rc = check_queries(dims, in->nodes, in->q_heads, in->kv_heads);
  if (rc != XS_OK || in->seqs == 0) return rc;
  if (!in->len || !in->parent || !in->seq_status || !in->q || !in->out || in->q == in->out) return XS_ERR_ARG;
  if (!aligned16(in->q) || !aligned16(in->out) ||
      !kv_ok(in->cache, in->seqs, in->capacity, in->kv_heads, in->head_dim, false) ||
      !kv_ok(in->fresh, in->seqs, in->nodes, in->kv_heads, in->head_dim, false) ||
      !strides_ok(in->seqs, in->q_seq_stride, in->nodes, in->q_node_stride, in->q_heads, in->q_head_stride, in->head_dim, false) ||
      !strides_ok(in->seqs, in->out_seq_stride, in->nodes, in->out_node_stride, in->q_heads, in->out_head_stride, in->head_dim, true))
    return XS_ERR_ARG;
  return XS_OK;
}

int xs_host_check_commit(const xs_cache_dims* dims, const xs_cache_commit_args* in) {
  if (!dims || !in) return XS_ERR_ARG;
  int rc = check_sizes(dims, in->dtype, in->head_dim, in->seqs, in->kv_heads, in->capacity, in->max_len);
  if (rc == XS_OK) rc = check_queries(dims, in->nodes, in->q_heads, in->kv_heads);
  if (rc != XS_OK || in->seqs == 0) return rc;
  if (!in->len || !in->path || !in->n_path || !in->new_len || !in->seq_status || !apart(in->len, in->new_len, in->seqs)) return XS_ERR_ARG;
  if (in->path_ld < in->nodes || in->slot_ld < in->capacity) return XS_ERR_ARG;
  if (!slots_fit(in->seqs, in->kv_heads, in->slot_ld) || in->path_ld > INT32_MAX) return XS_ERR_ARG;
  const int positions = (in->next_pos != nullptr) + (in->pos != nullptr) + (in->new_next_pos != nullptr);
  if ((positions != 0 && positions != 3) || (positions == 3 && !apart(in->next_pos, in->new_next_pos, in->seqs))) return XS_ERR_ARG;
  const int weights = (in->q != nullptr) + (in->lse != nullptr) + (in->mass != nullptr) + (in->new_mass != nullptr);
  if (weights != 0 && weights != 4) return XS_ERR_ARG;
  if (!kv_ok(in->cache, in->seqs, in->capacity, in->kv_heads, in->head_dim, true) ||
      !kv_ok(in->fresh, in->seqs, in->nodes, in->kv_heads, in->head_dim, false))
    return XS_ERR_ARG;
  if (weights && (!aligned16(in->q) || !strides_ok(in->seqs, in->q_seq_stride, in->nodes, in->q_node_stride, in->q_heads,
                                                   in->q_head_stride, in->head_dim, false)))
    return XS_ERR_ARG;
  return XS_OK;
}

int xs_host_check_evict(const xs_cache_dims* dims, const xs_cache_evict_args* in) {
  if (!dims || !in) return XS_ERR_ARG;
  const int rc = check_sizes(dims, in->dtype, in->head_dim, in->seqs, in->kv_heads, in->capacity, in->max_len);
  if (rc != XS_OK || in->seqs == 0) return rc;
  if (!in->len || !in->mass || !in->new_mass || !in->pos || !in->new_pos || !in->next_pos || !in->new_len ||
      !in->seq_status || !apart(in->len, in->new_len, in->seqs))
    return XS_ERR_ARG;
  if ((in->new_mass == in->mass) != (in->new_pos == in->pos)) return XS_ERR_ARG;
  if (in->keep < 1 || in->sinks < 0 || in->recent < 0 || in->sinks > in->keep || in->recent > in->keep - in->sinks)
    return XS_ERR_ARG;
  if (in->slot_ld < in->capacity || !slots_fit(in->seqs, in->kv_heads, in->slot_ld)) return XS_ERR_ARG;
  return kv_ok(in->cache, in->seqs, in->capacity, in->kv_heads, in->head_dim, true) ? XS_OK : XS_ERR_ARG;
}

int xs_host_check_rotate(const xs_qk_rotate_args* in) {
  if (!in) return XS_ERR_ARG;
  const int64_t d = in->head_dim, r = in->rot_dim;
  if (in->dtype != XS_BF16 && in->dtype != XS_F16) return XS_ERR_ARG;
  if (d < 8 || d > 256 || d % 8 || in->tokens < 0 || in->q_heads < 0 || in->kv_heads < 0) return XS_ERR_ARG;
  if (in->pairs != XS_ROT_HALVES && in->pairs != XS_ROT_NEIGHBOURS) return XS_ERR_ARG;
  if (r < 0 || r > d || r % (in->pairs == XS_ROT_HALVES ? 16 : 8)) return XS_ERR_ARG;
  if (!(in->eps >= 0.0f)) return XS_ERR_ARG;
  // heads are counted in 32 bits
  if (in->q_heads > 65536 || in->kv_heads > 65536) return XS_ERR_CAPACITY;
  if (in->tokens == 0 || in->q_heads + in->kv_heads == 0) return XS_OK;
  if (r > 0 && (!in->inv_freq || !in->pos)) return XS_ERR_ARG;
  if (in->q_heads && in->kv_heads && !in->q_weight != !in->k_weight) return XS_ERR_ARG;
  auto side = [&](int64_t heads, const void* x, int64_t ts, int64_t hs, const float* w, void* y, int64_t yts, int64_t yhs) {
    if (heads == 0) return true;
    return x && y && aligned16(x) && aligned16(y) && aligned16(w) && strides_ok(in->tokens, ts, heads, hs, 1, 0, d, false) &&
           strides_ok(in->tokens, yts, heads, yhs, 1, 0, d, true) && (x != y || ((in->tokens == 1 || ts == yts) && (heads == 1 || hs == yhs)));
  };
  if (!side(in->q_heads, in->q, in->q_token_stride, in->q_head_stride, in->q_weight, in->q_out, in->q_out_token_stride, in->q_out_head_stride) ||
      !side(in->kv_heads, in->k, in->k_token_stride, in->k_head_stride, in->k_weight, in->k_out, in->k_out_token_stride, in->k_out_head_stride))
    return XS_ERR_ARG;
  if (in->q_heads && in->kv_heads && (in->q_out == in->k_out || in->q_out == in->k || in->k_out == in->q)) return XS_ERR_ARG;
  return XS_OK;
}

int xs_host_check_prompt(const xs_prompt_attend_args* in) {
  if (!in) return XS_ERR_ARG;
  if (in->dtype != XS_BF16 && in->dtype != XS_F16) return XS_ERR_ARG;
  if (in->head_dim < 8 || in->head_dim > 256 || in->head_dim % 8) return XS_ERR_ARG;
  if (in->seqs < 0 || in->tokens < 0 || in->q_heads < 1 || in->kv_heads < 1 || in->q_heads % in->kv_heads) return XS_ERR_ARG;
  // a sequence's rows (tokens and q heads of one kv head) are counted in 32 bits
  if (in->seqs > 65536 || in->q_heads > 4096 || in->tokens > (1 << 30) / (in->q_heads / in->kv_heads)) return XS_ERR_CAPACITY;
  // and so are the elements that 64 tokens of k span
  if (in->kv_token_stride > (1 << 24)) return XS_ERR_CAPACITY;
  if (in->seqs == 0) return XS_OK;
  if (!in->start || !in->seq_status) return XS_ERR_ARG;
  if (in->tokens == 0) return XS_OK;
  if (!in->q || !in->k || !in->v || !in->out || in->out == in->q || in->out == in->k || in->out == in->v) return XS_ERR_ARG;
  if (!aligned16(in->q) || !aligned16(in->k) || !aligned16(in->v) || !aligned16(in->out) ||
      !strides_ok(in->tokens, in->q_token_stride, in->q_heads, in->q_head_stride, 1, 0, in->head_dim, false) ||
      !strides_ok(in->tokens, in->kv_token_stride, in->kv_heads, in->kv_head_stride, 1, 0, in->head_dim, false) ||
      !strides_ok(in->tokens, in->out_token_stride, in->q_heads, in->out_head_stride, 1, 0, in->head_dim, true))
    return XS_ERR_ARG;
  return XS_OK;
}

int xs_host_check_append8(const xs_cache_dims* dims, const xs_cache_append8_args* in) {
  if (!dims || !in) return XS_ERR_ARG;
  const int rc = check_sizes(dims, in->dtype, in->head_dim, in->seqs, in->kv_heads, in->capacity, 0);
  if (rc != XS_OK) return rc;
  if (in->head_dim % 16 || in->rows < 0 || in->tokens < 0) return XS_ERR_ARG;
  if (in->rows > INT32_MAX || in->tokens > INT32_MAX || in->path_ld > INT32_MAX) return XS_ERR_CAPACITY;
  if (in->seqs == 0) return XS_OK;
  if (!in->len || !in->new_len || !in->seq_status || !apart(in->len, in->new_len, in->seqs)) return XS_ERR_ARG;
  if (in->start && (in->path || in->n_path)) return XS_ERR_ARG;
  if (in->path && in->path_ld < in->rows) return XS_ERR_ARG;
  if (!kv8_ok(in->cache, in->seqs, in->capacity, in->kv_heads, in->head_dim, true)) return XS_ERR_ARG;
  const int64_t source = in->start ? in->tokens : in->rows;
  if (in->rows == 0 || source == 0) return XS_OK;  // (no row to read)
  xs_kv fresh = in->fresh;
  if (in->start) fresh.seq_stride = 0;
  return kv_ok(fresh, in->seqs, source, in->kv_heads, in->head_dim, false) ? XS_OK : XS_ERR_ARG;
}

int xs_host_check_attend8(const xs_cache_dims* dims, const xs_tree_attend8_args* in) {
  if (!dims || !in) return XS_ERR_ARG;
  int rc = check_sizes(dims, in->dtype, in->head_dim, in->seqs, in->kv_heads, in->capacity, in->max_len);
  if (rc == XS_OK) rc = check_queries(dims, in->nodes, in->q_heads, in->kv_heads);
  if (rc == XS_OK && in->head_dim % 16) return XS_ERR_ARG;
  if (rc != XS_OK || in->seqs == 0) return rc;
  // the bytes that 64 slots span are counted in 32 bits
  if (in->cache.slot_stride > (1 << 25)) return XS_ERR_CAPACITY;
  if (!in->len || !in->parent || !in->seq_status || !in->q || !in->out || in->q == in->out) return XS_ERR_ARG;
  if (!aligned16(in->q) || !aligned16(in->out) ||
      !kv8_ok(in->cache, in->seqs, in->capacity, in->kv_heads, in->head_dim, false) ||
      !kv_ok(in->fresh, in->seqs, in->nodes, in->kv_heads, in->head_dim, false) ||
      !strides_ok(in->seqs, in->q_seq_stride, in->nodes, in->q_node_stride, in->q_heads, in->q_head_stride, in->head_dim, false) ||
      !strides_ok(in->seqs, in->out_seq_stride, in->nodes, in->out_node_stride, in->q_heads, in->out_head_stride, in->head_dim, true))
    return XS_ERR_ARG;
  return XS_OK;
}

bool xs_host_launch_fits(int64_t workgroups, int64_t threads) {
  return workgroups <= INT32_MAX && workgroups * threads <= (int64_t)UINT32_MAX;
}

int xs_host_check_argmax(const xs_host_limits* lim, const xs_argmax_args* in) {
  if (!lim || !in || !in->logits || !in->ids || !in->probs) return XS_ERR_ARG;
  if (in->rows < 0 || in->width < 1 || in->ld < in->width) return XS_ERR_ARG;
  if (in->rows > lim->max_rows || in->width > lim->vocab) return XS_ERR_CAPACITY;
  if (in->ld % 4 != 0 || !aligned16(in->logits)) return XS_ERR_ARG;
  if (xs_host::chunks_for(in->width) > lim->max_chunks) return XS_ERR_CAPACITY;
  return XS_OK;
}

int32_t xs_select_option(const double* scores, int64_t n, double temperature, int64_t top_k,
                         double top_p, double u, int64_t* index) {
  if (!scores || !index || n < 1) return XS_ERR_ARG;
  if (temperature <= 0.0 || top_k <= 1) {  // argmax_index: the first maximal score
    double best = -INFINITY;
    int64_t at = 0;
    for (int64_t i = 0; i < n; i++)
      if (scores[i] > best) {
        best = scores[i];
        at = i;
      }
    *index = at;
    return XS_ROW_OK;
  }
  // renormalize at the temperature: f64 softmax (the f64::max fold skips NaN)
  std::vector<double> p((size_t)n);
  double mx = -INFINITY;
  for (int64_t i = 0; i < n; i++) {
    p[i] = scores[i] / temperature;
    if (p[i] > mx) mx = p[i];
  }
  double total = -0.0;
  for (double& v : p) {
    v = std::exp(v - mx);
    total += v;
  }
  for (double& v : p) v = v / total;
  // rank by probability (f64::total_cmp, descending), ties to the lower index
  auto key = [](double d) {
    uint64_t b;
    memcpy(&b, &d, 8);
    return (b >> 63) ? ~b : (b | 0x8000000000000000ull);
  };
  std::vector<int64_t> order((size_t)n);
  for (int64_t i = 0; i < n; i++) order[i] = i;
  std::stable_sort(order.begin(), order.end(), [&](int64_t x, int64_t y) { return key(p[x]) > key(p[y]); });
  const int64_t kept_k = std::min(top_k, n);
  // the nucleus over the survivors' own mass; the crossing option stays
  int64_t keep = kept_k;
  if (!(top_p >= 1.0)) {
    double mass = -0.0;
    for (int64_t i = 0; i < kept_k; i++) mass += p[order[i]];
    if (!(mass <= 0.0)) {
      double run = 0.0;
      for (int64_t i = 0; i < kept_k; i++) {
        run += p[order[i]] / mass;
        if (run >= top_p) {
          keep = i + 1;
          break;
        }
      }
    }
  }
  // WeightedIndex<f64> (rand 0.9): cumulative weights before each later
  // weight, the draw x = u * total, the count of cumulative weights <= x
  double acc = p[order[0]];
  if (!(acc >= 0.0)) return XS_ROW_ZERO_WEIGHT;
  std::vector<double> cum;
  for (int64_t i = 1; i < keep; i++) {
    const double w = p[order[i]];
    if (!(w >= 0.0)) return XS_ROW_ZERO_WEIGHT;
    cum.push_back(acc);
    acc += w;
  }
  if (acc == 0.0 || !std::isfinite(acc)) return XS_ROW_ZERO_WEIGHT;
  const double x = u * acc + 0.0;
  const int64_t c = std::upper_bound(cum.begin(), cum.end(), x) - cum.begin();
  *index = order[c];
  return XS_ROW_OK;
}

int64_t xs_keep_confident(const float* probs, int64_t n, float p_min) {
  int64_t kept = 0;
  while (kept < n && probs[kept] >= p_min) kept++;
  return kept;
}

}  // extern "C"
