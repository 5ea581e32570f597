// Attention over packed documents, f32 operands (packed_attention.h; one element type per file: they compile in parallel).
#include "packed_attention.h"

namespace ldot {
template int attn_launch<float>(const AttnParams&, bool, int, int64_t, int64_t, hipStream_t);
}
