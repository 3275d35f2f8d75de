// Attention over a paged cache: float queries, keys and values.
#include "htree_draft.h"

namespace htree {
HTREE_DRAFT_TYPE(float)
}  // namespace htree
