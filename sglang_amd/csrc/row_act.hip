// SiLU(gate) * up with 8-bit rows and a scale per row, int8 rows with zero points (row_out.h has the arithmetic), and the
// sums over the weight rows that a product of such rows needs.
#include "row_out_kernels.h"

namespace sglamd {

// Sums over the rows of an int8 matrix [n, k], a wave per row: 16 bytes a lane and four dot products with ones, or byte by byte.
__global__ __launch_bounds__(256) void int8_row_sums_kernel(const int8_t* __restrict__ b, int64_t ldb, int64_t n, int64_t k, bool pieces,
                                                            int32_t* __restrict__ sums) {
  const int64_t row = (int64_t)blockIdx.x * 4 + (threadIdx.x >> 6);
  if (row >= n) return;
  const int lane = threadIdx.x & 63;
  const int8_t* src = b + row * ldb;
  int sum = 0;
  if (pieces) {
    for (int64_t i = lane; i < (k >> 4); i += 64) {
      const v4i w = *((const v4i*)src + i);
#pragma unroll
      for (int j = 0; j < 4; j++) sum = __builtin_amdgcn_sdot4(w[j], 0x01010101, sum, false);
    }
  } else {
    for (int64_t i = lane; i < k; i += 64) sum += src[i];
  }
#pragma unroll
  for (int off = 32; off >= 1; off >>= 1) sum += __shfl_xor(sum, off, 64);
  if (lane == 0) sums[row] = sum;
}

}  // namespace sglamd

using namespace sglamd;

extern "C" int sglamd_silu_mul_row_quant(const void* x, int64_t x_row_stride, const float* fixed_scale, int64_t rows, int64_t hidden,
                                         void* output_q, float* output_s, int32_t* output_zp, int dtype, int q_dtype, void* stream) {
  const char* op = "silu_mul_row_quant";
  RowOutArgs a = {};
  a.x = x, a.x_stride = x_row_stride, a.q = (uint8_t*)output_q, a.s = output_s, a.zp = output_zp, a.fixed = fixed_scale;
  a.hidden = hidden, a.rows = rows;
  const int rc = check_row_out(op, a, 2 * hidden, q_dtype);
  if (rc) return rc;
  SGLAMD_REQUIRE(dtype == SGLAMD_BF16 || dtype == SGLAMD_F16, SGLAMD_EINVAL, "%s: activations must be Half or BFloat16", op);
  if (rows == 0) return SGLAMD_OK;
  const DeviceScope scope;
  const int kind = row_out_kind(a, q_dtype);
  return dtype == SGLAMD_BF16 ? launch_row_out_to<BF16, F32, ROW_SILU>(a, kind, row_out_pieces(a), (hipStream_t)stream)
                              : launch_row_out_to<F16, F32, ROW_SILU>(a, kind, row_out_pieces(a), (hipStream_t)stream);
}

extern "C" int sglamd_per_token_quant_int8_asym(const void* x, int64_t x_row_stride, int dtype, int64_t rows, int64_t hidden, int8_t* output_q,
                                                float* output_s, int32_t* output_zp, void* stream) {
  const char* op = "per_token_quant_int8_asym";
  RowOutArgs a = {};
  a.x = x, a.x_stride = x_row_stride, a.q = (uint8_t*)output_q, a.s = output_s, a.zp = output_zp, a.hidden = hidden, a.rows = rows;
  const int rc = check_row_out(op, a, hidden, SGLAMD_I8);
  if (rc) return rc;
  SGLAMD_REQUIRE(output_zp, SGLAMD_EINVAL, "%s: null pointer", op);
  SGLAMD_REQUIRE(dtype == SGLAMD_F32 || dtype == SGLAMD_BF16 || dtype == SGLAMD_F16, SGLAMD_EINVAL,
                 "%s: input dtype must be F32, F16 or BF16", op);
  if (rows == 0) return SGLAMD_OK;
  const DeviceScope scope;
  hipStream_t st = (hipStream_t)stream;
  if (dtype == SGLAMD_BF16) launch_row_out<BF16, F32, ROW_PLAIN, ROW_TO_ASYM>(a, row_out_pieces(a), st);
  else if (dtype == SGLAMD_F16) launch_row_out<F16, F32, ROW_PLAIN, ROW_TO_ASYM>(a, row_out_pieces(a), st);
  else launch_row_out<F32, F32, ROW_PLAIN, ROW_TO_ASYM>(a, ROW_VALUES, st);
  return check_launch(op);
}

extern "C" int sglamd_int8_weight_sums(const void* b, int64_t ldb, int64_t N, int64_t K, int32_t* sums, void* stream) {
  const char* op = "int8_weight_sums";
  SGLAMD_REQUIRE(b && sums, SGLAMD_EINVAL, "%s: null pointer", op);
  SGLAMD_REQUIRE(N >= 0 && N < (1ll << 26) && K > 0 && K < (1ll << 24), SGLAMD_EINVAL, "%s: bad sizes N=%lld K=%lld", op, (long long)N,
                 (long long)K);  // (a launch holds fewer than 2^32 lanes; sums of fewer than 2^24 codes stay inside 32 bits)
  SGLAMD_REQUIRE(ldb >= K, SGLAMD_EINVAL, "%s: leading dimension smaller than the row", op);
  if (N == 0) return SGLAMD_OK;
  const bool pieces = K % 16 == 0 && ldb % 16 == 0 && aligned_to(b, 16);
  hipLaunchKernelGGL(int8_row_sums_kernel, dim3((unsigned)ceil_div(N, 4)), dim3(256), 0, (hipStream_t)stream, (const int8_t*)b, ldb, N, K,
                     pieces, sums);
  return check_launch(op);
}
