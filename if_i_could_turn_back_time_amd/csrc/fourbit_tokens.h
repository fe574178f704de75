// Places by token, for the embedding's gradient and for the head's.
#pragma once
#include <hip/hip_runtime.h>

#include <cstdint>

#include "fourbit.h"

// Sorting.  Not part of the library's ABI.
namespace fb_gpu {
// Workspace of sort_tokens.
__attribute__((visibility("hidden"))) size_t sort_bytes(int64_t rows, int32_t vocab);
// key, place: the tokens in [0, vocab) in ascending order, equal ones by their place, then the others
// (key vocab); clears bytes of `zeros` (16-byte aligned, contiguous) beside it.  Returns an fb_status.
__attribute__((visibility("hidden"))) int sort_tokens(const int64_t* token, int64_t rows, int32_t vocab,
                                                      unsigned* key, unsigned* place, void* zeros,
                                                      int64_t bytes, void* ws, hipStream_t hs);
}  // namespace fb_gpu
