// Attention over a paged cache: _Float16 queries, keys and values.
#include "htree_draft.h"

namespace htree {
HTREE_DRAFT_TYPE(_Float16)
}  // namespace htree
