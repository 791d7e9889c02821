// gemm.h for F32 elements
#include "gemm.h"

namespace atlas_train {
template int gemm_t<F32>(GemmP, bool, bool, hipStream_t);
template int gemm_splits<F32>(const GemmP&, bool, bool);
}
