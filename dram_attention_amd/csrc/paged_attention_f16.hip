// Attention over pages (paged_attention.hpp): F16 queries, F16 keys and values.
#include "paged_attention.hpp"

namespace da {
DA_PAGED_TYPES(F16, F16)
}  // namespace da
