// Packed attention of short sequences: a few lanes a row instead of matrix tiles (packed_short.hip).
#pragma once

#include "bf_common.h"

namespace bf {

// Whether a call's sequences are short enough (p->longest, 0: unknown).
bool packed_is_short(const bf_packed_attn* p);

// bf_packed_attn_fwd / _bwd of such a call; arguments checked by the caller.
int packed_short_fwd(const bf_packed_attn* p, const void* q, const void* k, const void* v, void* out, float* lse,
                     hipStream_t st);
int packed_short_bwd(const bf_packed_attn* p, const void* q, const void* k, const void* v, const void* out, const float* lse,
                     const void* dout, void* dq, void* dk, void* dv, float* delta, hipStream_t st);

}  // namespace bf
