// Attention over packed documents, f16 operands (packed_attention.h; one element type per file: they compile in parallel).
#include "packed_attention.h"

namespace ldot {
template int attn_launch<_Float16>(const AttnParams&, bool, int, int64_t, int64_t, hipStream_t);
}
