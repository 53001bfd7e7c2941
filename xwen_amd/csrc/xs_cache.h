// xs_cache.h -- the cache context and the rules by which its calls fill the
// device.  Private to the library.
#pragma once

#include <hip/hip_runtime.h>
#include <stdint.h>

#include "../../include/xsamp.h"

namespace xst {
struct EvictWork {
  uint64_t* kept;   // [heads, words] bitmap of the kept slots
  int32_t* free_;   // [heads, pairs] freed slots, ascending
  int32_t* filler;  // [heads, pairs] the slots that move there, ascending
  int32_t* moves;   // [heads]
  int64_t words, pairs;
};
}  // namespace xst

struct xs_cache_context {
  int device;
  hipStream_t stream;
  xs_cache_dims dims;
  xst::EvictWork evict;
  int n_cu;
  float* part;    // attention's partial results, one for each workgroup of a split call
  int64_t part_floats;
};

namespace xs_host {

// Workgroups of attend_kernel that a CU holds at once (by its registers; its
// launch bound asks for as many), by the head's size and the row tiles.
constexpr int64_t per_cu(int dp, int rt) { return dp * rt <= 64 ? 4 : dp * rt <= 128 ? 3 : dp * rt <= 256 ? 2 : 1; }
// How many times over a split call fills the device: once where all sequences
// end together (one of them: 8 heads over 131,072 slots 113 us, filled four
// times 145), more often where some end early (32 sequences of 327 to 8,192
// slots: 134 us, filled twice 151; but 32 of 8,192 take 222 instead of 214).
constexpr int64_t rounds(int64_t seqs) { return seqs > 1 ? 4 : 1; }

}  // namespace xs_host
