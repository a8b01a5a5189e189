// Between the library's own sources (not exported).
#pragma once

#include <stdint.h>

namespace pb {

// Group keys that pb_sample_ws leaves in its workspace: for every row, the key of the largest value of
// each `elems` consecutive elements (128 bytes), `groups` of them, rows `stride` keys apart (a multiple
// of 4).
struct GroupKeys {
  const uint32_t* keys;
  int32_t stride, groups, elems;
};

// The group keys of a pb_sample_ws call with these arguments, or keys = nullptr where it takes its
// other launch, which leaves none.
GroupKeys sample_ws_keys(const void* logits, int dtype, int64_t n_rows, int64_t vocab, int64_t row_stride,
                         const void* workspace, int64_t ws_bytes);

}  // namespace pb
