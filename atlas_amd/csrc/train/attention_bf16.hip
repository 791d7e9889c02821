// attention.h for BF16 elements
#include "attention.h"

namespace atlas_train {
template int attention_forward_t<BF16>(const AttnP&, int, int, void*, hipStream_t);
template int attention_backward_t<BF16>(const AttnP&, int, int, void*, hipStream_t);
template size_t attention_bytes<BF16>(const AttnP&, int, int, bool);
}
