// Attention of new tokens over a cache in pages, fp32.
#include "paged_attn.h"

namespace qlka {

int pg_attend_f32(int held, const PgParams& p, hipStream_t st) { return pg_attend_type<float>(held, p, st); }

}  // namespace qlka
