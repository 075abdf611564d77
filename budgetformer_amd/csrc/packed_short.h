// Packed attention of short sequences: a few lanes a row instead of matrix tiles (packed_short.hip).
#pragma once

#include "bf_common.h"

namespace bf {

// Whether a call's sequences are short enough (p->longest, 0: unknown), and with a bias (or NULL) its table.
bool packed_is_short(const bf_packed_attn* p, const bf_packed_bias* bias);

// bf_packed_attn_fwd / _bwd of such a call, with a bias or not (NULL); arguments checked by the caller. bias_part: the sums of the
// scores' gradients by bucket, packed_short_parts(p) parts of [heads_q, buckets].
int64_t packed_short_parts(const bf_packed_attn* p);
int packed_short_fwd(const bf_packed_attn* p, const bf_packed_bias* bias, const void* q, const void* k, const void* v, void* out,
                     float* lse, hipStream_t st);
int packed_short_bwd(const bf_packed_attn* p, const bf_packed_bias* bias, const void* q, const void* k, const void* v, const void* out,
                     const float* lse, const void* dout, void* dq, void* dk, void* dv, float* delta, float* bias_part, hipStream_t st);

}  // namespace bf
