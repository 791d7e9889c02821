// gemm.h for F16 elements
#include "gemm.h"

namespace atlas_train {
template int gemm_t<F16>(GemmP, bool, bool, hipStream_t);
template int gemm_splits<F16>(const GemmP&, bool, bool);
}
