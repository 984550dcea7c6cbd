// SPDX-License-Identifier: MIT
// FLASH_ATTN_EXT over a Q8_0 K and a Q4_0 V: the kernels of mx_fa_q.h.
#include "mx_fa_q.h"

namespace mx {
FQ_TYPES(Q8_0, Q4_0)
}  // namespace mx
