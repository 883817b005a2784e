// Every dense GEMM kernel in the GEMM_ROW_INT8 scaling mode for activation rows with zero points (see gemm_dispatch.h).
#include "gemm_dispatch.h"

namespace sglamd {
template int dispatch_out_zero_point<GEMM_ROW_INT8>(const GemmArgs&, int, hipStream_t, void*, int64_t);
template int dispatch_quantising_zero_point<GEMM_ROW_INT8>(const GemmArgs&, int, hipStream_t, bool);
}  // namespace sglamd
