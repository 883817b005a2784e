// Residual addition and RMSNorm with 8-bit rows and a scale per row (row_out.h has the arithmetic).
#include "row_out_kernels.h"

using namespace sglamd;

template <typename T>
static int rms_to(const RowOutArgs& a, int weight_dtype, int q_kind, RowPieces pieces, hipStream_t st) {
  if (weight_dtype == SGLAMD_F32) return launch_row_out_to<T, F32, ROW_RMS>(a, q_kind, pieces, st);
  return launch_row_out_to<T, T, ROW_RMS>(a, q_kind, pieces, st);
}

extern "C" int sglamd_fused_rms_row_quant(const void* x, int64_t x_row_stride, const void* res, int64_t res_row_stride, const void* weight,
                                          float eps, const float* fixed_scale, int64_t rows, int64_t hidden, void* output_q, float* output_s,
                                          int32_t* output_zp, void* y, void* res_out, int dtype, int weight_dtype, int q_dtype, void* stream) {
  const char* op = "fused_rms_row_quant";
  RowOutArgs a = {};
  a.x = x, a.x_stride = x_row_stride, a.res = res, a.res_stride = res_row_stride, a.res_out = res_out, a.w = weight, a.eps = eps;
  a.y = y, a.q = (uint8_t*)output_q, a.s = output_s, a.zp = output_zp, a.fixed = fixed_scale, a.hidden = hidden, a.rows = rows;
  const int rc = check_row_out(op, a, hidden, q_dtype);
  if (rc) return rc;
  SGLAMD_REQUIRE(weight, SGLAMD_EINVAL, "%s: null weight", op);
  SGLAMD_REQUIRE(dtype == SGLAMD_BF16 || dtype == SGLAMD_F16, SGLAMD_EINVAL, "%s: activations must be Half or BFloat16", op);
  SGLAMD_REQUIRE(weight_dtype == SGLAMD_F32 || weight_dtype == dtype, SGLAMD_EINVAL, "%s: the weight must be Float or of the activations' type", op);
  SGLAMD_REQUIRE(!res == !res_out, SGLAMD_EINVAL, "%s: a residual and its updated form go together", op);
  SGLAMD_REQUIRE(!res || (res_row_stride >= 0 && (res_row_stride >= hidden || res_row_stride == 0)), SGLAMD_EINVAL,
                 "%s: residual row stride %lld is smaller than the row", op, (long long)res_row_stride);
  if (rows == 0) return SGLAMD_OK;
  const DeviceScope scope;
  const int kind = row_out_kind(a, q_dtype);
  return dtype == SGLAMD_BF16 ? rms_to<BF16>(a, weight_dtype, kind, row_out_pieces(a), (hipStream_t)stream)
                              : rms_to<F16>(a, weight_dtype, kind, row_out_pieces(a), (hipStream_t)stream);
}
