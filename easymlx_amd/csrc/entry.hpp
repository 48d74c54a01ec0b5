// What the C entry points of every translation unit share (emx_attn.hip holds it): the last error
// of the calling thread, and the checks that all attention calls have in common.
#pragma once

#include <stdint.h>

namespace emx {

// Sets emx_last_error() and returns `code`.
int entry_fail(int code, const char* message);
// EMX_OK, or EMX_ERR_HIP where the launch just made failed.
int entry_check_launch(const char* what);
int entry_check_attention(const void* q, int num_tokens, int hq, int d, int hkv, int nb, int bs, const int32_t* bt,
                          int S, int max_blocks, const int32_t* kv_lens, const int32_t* qsl, int decode,
                          const void* out);

}  // namespace emx
