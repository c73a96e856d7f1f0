// Attention over pages (paged_attention.hpp): F32 queries, F32 keys and values.
#include "paged_attention.hpp"

namespace da {
DA_PAGED_TYPES(F32, F32)
}  // namespace da
