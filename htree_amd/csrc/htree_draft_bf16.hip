// Attention over a paged cache: __bf16 queries, keys and values.
#include "htree_draft.h"

namespace htree {
HTREE_DRAFT_TYPE(__bf16)
}  // namespace htree
