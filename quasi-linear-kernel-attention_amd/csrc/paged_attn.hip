// Attention of new tokens over a cache in pages, bf16 (fp32: paged_attn_f32.hip; two files, which compile at the same
// time).
#include "paged_attn.h"

namespace qlka {

int pg_attend_bf16(int held, const PgParams& p, hipStream_t st) { return pg_attend_type<__bf16>(held, p, st); }

}  // namespace qlka
