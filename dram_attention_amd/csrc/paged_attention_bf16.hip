// Attention over pages (paged_attention.hpp): BF16 queries, BF16 keys and values.
#include "paged_attention.hpp"

namespace da {
DA_PAGED_TYPES(BF16, BF16)
}  // namespace da
