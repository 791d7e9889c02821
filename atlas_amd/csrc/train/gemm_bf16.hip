// gemm.h for BF16 elements
#include "gemm.h"

namespace atlas_train {
template int gemm_t<BF16>(GemmP, bool, bool, hipStream_t);
template int gemm_splits<BF16>(const GemmP&, bool, bool);
}
