// attention.h for F32 elements
#include "attention.h"

namespace atlas_train {
template int attention_forward_t<F32>(const AttnP&, int, int, void*, hipStream_t);
template int attention_backward_t<F32>(const AttnP&, int, int, void*, hipStream_t);
template size_t attention_bytes<F32>(const AttnP&, int, int, bool);
}
