// Attention over pages (paged_attention.hpp): F16 queries, E4M3 keys and values.
#include "paged_attention.hpp"

namespace da {
DA_PAGED_TYPES(F16, E4M3)
}  // namespace da
