// attention.h for F16 elements
#include "attention.h"

namespace atlas_train {
template int attention_forward_t<F16>(const AttnP&, int, hipStream_t);
template int attention_backward_t<F16>(const AttnP&, int, int, hipStream_t);
}
