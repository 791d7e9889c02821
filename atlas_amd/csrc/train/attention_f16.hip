// attention.h for F16 elements
#include "attention.h"

namespace atlas_train {
template int attention_forward_t<F16>(const AttnP&, int, int, void*, hipStream_t);
template int attention_backward_t<F16>(const AttnP&, int, int, void*, hipStream_t);
template size_t attention_bytes<F16>(const AttnP&, int, int, bool);
}
