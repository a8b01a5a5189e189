// Between the library's own sources (not exported).
#pragma once

#include <stdint.h>

#include "../../include/pagedbatch_b200.h"

namespace pb {

// Group keys that pb_sample_ws leaves in its workspace: for every row, the key of the largest value of
// each 128 bytes (8 vectors of 16), `groups` of them, rows `stride` keys apart (a multiple of 4).
struct GroupKeys {
  const uint32_t* keys;
  int32_t stride, groups;
};

// The group keys of a pb_sample_ws call with these arguments, or keys = nullptr where it takes its
// other launch, which leaves none.
GroupKeys sample_ws_keys(const void* logits, int dtype, int64_t n_rows, int64_t vocab, int64_t row_stride,
                         const void* workspace, int64_t ws_bytes);

// pb_sample_ws's launches for a batch whose group keys sample_ws_keys names, each waiting for the whole of the one
// before. (pb_sample_ws lets them overlap, and where no row is greedy or small top-k none of them waits: the
// last one may end before the keys are written.)
int sample_ws_in_turn(const void* logits, int dtype, int64_t n_rows, int64_t vocab, int64_t row_stride,
                      const pb_row_params* params, int64_t* out_token, pb_row_info* info, void* workspace, void* stream);

// The cluster kernel over the rows whose status in `info` is PB_ROW_FALLBACK (vocab < 2^24, valid
// arguments): their tokens and records are written, the other rows' are left as they are.
int sample_fallback_rows(const void* logits, int dtype, int64_t n_rows, int64_t vocab, int64_t row_stride,
                         const pb_row_params* params, int64_t* out_token, pb_row_info* info, void* stream);

}  // namespace pb
