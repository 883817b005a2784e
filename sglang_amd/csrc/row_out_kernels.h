// The kernels of row_out.h, instantiated by row_norm.hip (RMSNorm) and row_act.hip (SiLU * up, plain rows).
#pragma once
#include "row_out.h"

namespace sglamd {

// Eight values of a lane's piece `i` (0: a row of zeros past its end).
template <typename T>
__device__ __forceinline__ void unpack8(const v4i& raw, float* out) {
  u16 b[8];
  __builtin_memcpy(b, &raw, 16);
#pragma unroll
  for (int j = 0; j < 8; j++) out[j] = T::to_f32(b[j]);
}
template <typename T>
__device__ __forceinline__ v4i pack8(const float* v) {
  return v4i{(int)T::pack2(v[0], v[1]), (int)T::pack2(v[2], v[3]), (int)T::pack2(v[4], v[5]), (int)T::pack2(v[6], v[7])};
}
// exp by the hardware's exp2 and a reciprocal of 1 ulp each: relative error of some 2^-23 * (2 + |gate|), the second part only
// on gates so negative that the value is lost beside the row's largest
__device__ __forceinline__ float silu_mul(float gate, float up) {
  const float t = __builtin_amdgcn_exp2f(gate * -1.44269504088896340736f);
  return gate * __builtin_amdgcn_rcpf(1.0f + t) * up;
}

// A piece of a row in one instruction, wherever it starts (global memory takes any alignment).
template <typename V, bool RAGGED, typename E>
__device__ __forceinline__ V load_piece(const E* p) {
  if constexpr (!RAGGED) return *(const V*)p;
  V v;
  __builtin_memcpy(&v, p, sizeof(V));
  return v;
}
template <bool RAGGED, typename V, typename E>
__device__ __forceinline__ void store_piece(E* p, const V& v) {
  if constexpr (RAGGED) __builtin_memcpy(p, &v, sizeof(V));
  else *(V*)p = v;
}

// A row's lanes: TEAM = 64, one wave (no barrier), or 0, the workgroup.  Each holds NV pieces of 8 values.  RAGGED: rows of any
// alignment and any length from 8; the last piece is the row's last 8 values, of which those that the piece before it has too
// are written twice and counted once.
template <typename T, typename WT, int SRC, int QK, int NV, int TEAM, bool RAGGED>
__device__ __forceinline__ void row_out_body(const RowOutArgs& a, const int64_t row, uint32_t* red) {
  const int nt = TEAM ? TEAM : (int)blockDim.x, tid = TEAM ? (int)threadIdx.x & 63 : (int)threadIdx.x;
  const int hidden = (int)a.hidden, nvec = row < a.rows ? (RAGGED ? (hidden + 7) >> 3 : hidden >> 3) : 0;
  auto start = [&](int i) { return RAGGED ? min(i * 8, hidden - 8) : i * 8; };
  const u16* x = (const u16*)a.x + row * a.x_stride;
  const v4i zero = {0, 0, 0, 0};

  // every load of the row is requested before the first is used
  v4i raw[NV], second[SRC == ROW_PLAIN ? 1 : NV], wraw[SRC == ROW_RMS ? NV : 1][sizeof(typename WT::storage) == 4 ? 2 : 1];
#pragma unroll
  for (int k = 0; k < NV; k++) {
    const int i = tid + k * nt;
    const bool live = i < nvec;
    raw[k] = live ? load_piece<v4i, RAGGED>(x + start(i)) : zero;
    if constexpr (SRC == ROW_SILU) second[k] = live ? load_piece<v4i, RAGGED>(x + hidden + start(i)) : zero;
    if constexpr (SRC == ROW_RMS) {
      second[k] = live && a.res ? load_piece<v4i, RAGGED>((const u16*)a.res + row * a.res_stride + start(i)) : zero;
      if constexpr (sizeof(typename WT::storage) == 4) {
        wraw[k][0] = live ? load_piece<v4i, RAGGED>((const float*)a.w + start(i)) : zero;
        wraw[k][1] = live ? load_piece<v4i, RAGGED>((const float*)a.w + start(i) + 4) : zero;
      } else {
        wraw[k][0] = live ? load_piece<v4i, RAGGED>((const u16*)a.w + start(i)) : zero;
      }
    }
  }

  float u[NV][8];
  RowStats t = {0.f, 0u, 0u};
  float poison = 0.f;
#pragma unroll
  for (int k = 0; k < NV; k++) {
    unpack8<T>(raw[k], u[k]);
    if constexpr (SRC == ROW_SILU) {
      float up[8];
      unpack8<T>(second[k], up);
#pragma unroll
      for (int j = 0; j < 8; j++) u[k][j] = silu_mul(u[k][j], up[j]);
    }
    if constexpr (SRC == ROW_RMS) {
      if (a.res) {
        float r[8];
        unpack8<T>(second[k], r);
#pragma unroll
        for (int j = 0; j < 8; j++) u[k][j] += r[j];
        const int i = tid + k * nt;
        if (i < nvec) store_piece<RAGGED>((u16*)a.res_out + row * a.hidden + start(i), pack8<T>(u[k]));
      }
      float w[8];
      if constexpr (sizeof(typename WT::storage) == 4) {
        __builtin_memcpy(w, wraw[k], 32);
      } else {
        unpack8<WT>(wraw[k][0], w);
      }
#pragma unroll
      for (int j = 0; j < 8; j++) {
        const int i = tid + k * nt;
        if (!RAGGED || start(i) + j >= i * 8) t.ss = fmaf(u[k][j], u[k][j], t.ss);
        u[k][j] *= w[j];
      }
    }
#pragma unroll
    for (int j = 0; j < 8; j++) {
      row_stats_add<SRC, QK>(t, u[k][j]);
      if (QK == ROW_TO_ASYM) poison = fmaf(u[k][j], 0.f, poison);
    }
  }
  if (QK == ROW_TO_ASYM) row_stats_poison(t, poison);
  t = TEAM ? row_stats_wave<SRC, QK>(t) : row_stats_block<SRC, QK>(t, red);
  const RowScale o = row_scale<SRC, QK>(a, t);
  if (row >= a.rows) return;
  if (tid == 0) {
    a.s[row] = o.scale;
    if (QK == ROW_TO_ASYM) a.zp[row] = (int32_t)o.zp;
  }
  uint8_t* q = a.q + row * a.hidden;
#pragma unroll
  for (int k = 0; k < NV; k++) {
    const int i = tid + k * nt;
    if (i >= nvec) break;
    store_piece<RAGGED>(q + start(i), v2i{(int)row_codes4<QK>(u[k], o), (int)row_codes4<QK>(u[k] + 4, o)});
    if (SRC == ROW_RMS && a.y) {
      float y[8];
#pragma unroll
      for (int j = 0; j < 8; j++) y[j] = u[k][j] * o.r;
      store_piece<RAGGED>((u16*)a.y + row * a.hidden + start(i), pack8<T>(y));
    }
  }
}

// A launch holds fewer than 2^32 lanes in each dimension: workgroups beyond 2^20 go into the second one.
constexpr int ROW_OUT_GRID_BITS = 20;
__device__ __forceinline__ int64_t row_out_block() { return ((int64_t)blockIdx.y << ROW_OUT_GRID_BITS) + blockIdx.x; }
static inline dim3 row_out_grid(int64_t blocks) {
  const int64_t most = 1ll << ROW_OUT_GRID_BITS;
  return dim3((unsigned)(blocks < most ? blocks : most), (unsigned)ceil_div(blocks, most));
}

template <typename T, typename WT, int SRC, int QK, int NT, int NV, bool RAGGED>
__global__ __launch_bounds__(NT) void row_out_kernel(RowOutArgs a) {
  __shared__ uint32_t red[48];
  row_out_body<T, WT, SRC, QK, NV, 0, RAGGED>(a, row_out_block(), red);
}
// Short rows, a wave each.
template <typename T, typename WT, int SRC, int QK, int NV, bool RAGGED>
__global__ __launch_bounds__(256) void row_out_team_kernel(RowOutArgs a) {
  row_out_body<T, WT, SRC, QK, NV, 64, RAGGED>(a, row_out_block() * 4 + (threadIdx.x >> 6), nullptr);
}

// Rows below 8 values and beyond 32768, 32-bit rows: a workgroup per row, values one by one, the row read twice (the second time
// from L2).
template <typename T, typename WT, int SRC, int QK>
__global__ __launch_bounds__(256) void row_out_any_kernel(RowOutArgs a) {
  typedef typename T::storage S;
  __shared__ uint32_t red[48];
  const int64_t row = row_out_block();
  if (row >= a.rows) return;
  const S* x = (const S*)a.x + row * a.x_stride;
  const S* res = a.res ? (const S*)a.res + row * a.res_stride : nullptr;
  auto sum_at = [&](int64_t i) -> float { return T::to_f32(x[i]) + (res ? T::to_f32(res[i]) : 0.f); };
  auto value_at = [&](int64_t i) -> float {
    if constexpr (SRC == ROW_RMS) return sum_at(i) * WT::to_f32(((const typename WT::storage*)a.w)[i]);
    else if constexpr (SRC == ROW_SILU) return silu_mul(T::to_f32(x[i]), T::to_f32(x[a.hidden + i]));
    else return T::to_f32(x[i]);
  };
  RowStats t = {0.f, 0u, 0u};
  float poison = 0.f;
  for (int64_t i = threadIdx.x; i < a.hidden; i += 256) {
    if constexpr (SRC == ROW_RMS) {
      const float v = sum_at(i);
      t.ss = fmaf(v, v, t.ss);
      if (res) ((S*)a.res_out)[row * a.hidden + i] = T::from_f32(v);
    }
    const float u = value_at(i);
    row_stats_add<SRC, QK>(t, u);
    if (QK == ROW_TO_ASYM) poison = fmaf(u, 0.f, poison);
  }
  if (QK == ROW_TO_ASYM) row_stats_poison(t, poison);
  t = row_stats_block<SRC, QK>(t, red);
  const RowScale o = row_scale<SRC, QK>(a, t);
  if (threadIdx.x == 0) {
    a.s[row] = o.scale;
    if (QK == ROW_TO_ASYM) a.zp[row] = (int32_t)o.zp;
  }
  for (int64_t i = threadIdx.x; i < a.hidden; i += 256) {
    float v[4] = {value_at(i), 0.f, 0.f, 0.f};
    a.q[row * a.hidden + i] = (uint8_t)row_codes4<QK>(v, o);
    if (SRC == ROW_RMS && a.y) ((S*)a.y)[row * a.hidden + i] = T::from_f32(v[0] * o.r);
  }
}

constexpr int64_t ROW_OUT_MAX_HIDDEN = 512 * 8 * 8;  // the longest row that 512 or 1024 lanes keep in registers

// Bound by memory with many rows (a copy's rate from some thousand rows of 4096 values: 4096 x 8192 with a residual 45 us, 5.2 TB/s;
// SiLU of 4096 x [7168 | 7168] 29.5, 5.0), by one row's latency with few (one row of 7168 3.0 us, 2 of them a launch; SiLU of 28672
// values 5.9, the exponentials and reciprocals of a row on one CU).  Lanes x pieces per row: enough lanes that a row is short, few
// enough registers that a CU holds several rows.  Best | next best, us, asymmetric codes (norm: e4m3), data from HBM:
//   a wave of 1 or 2 pieces  norm 16384 x 512 14.6 | 21.2 (256 x 1), SiLU 10.9 | 24.0; SiLU 16384 x 1024 17.6 | 28.7; norm 300 x 1024 3.5 against 3.1
//   a wave of 4, plain rows  16384 x 2048 20.9 | 24.6 (256 x 1)
//   256 x 1                  norm 16384 x 2048 43.9 | 48.4 (512 x 1), SiLU 32.7 | 34.6 (a wave of 4)
//   512 x 1 (norm), 256 x 2  norm 1000 x 4096 8.7 | 9.3, SiLU 4096 x 4096 18.0 | 19.3, plain 16384 x 4096 38.4 | 48.1
//   512 x 2, 256 x 4 (plain) norm 1000 x 8192 14.2 | 15.3 (256 x 4), SiLU 4096 x 7168 29.5 | 30.8 (256 x 4), plain 19.0 | 20.6 (512 x 2)
//   1024 x 2                 norm 4096 x 14336 77 | 78 (512 x 4), SiLU 54.6 | 56.7, plain 33.9 | 34.1
//   512 x 8                  SiLU 3001 x 18432 53.8 | 55.0 (1024 x 4), 2000 x 28672 54.4 | 56.6
//   1024 x 4                 norm 4096 x 18432 114.9 | 118.5 (512 x 8), SiLU to symmetric codes, which keep fewer registers, 72.8 | 76.0
template <typename T, typename WT, int SRC, int QK, bool RAGGED>
static void launch_row_pieces(const RowOutArgs& a, hipStream_t st) {
  if constexpr (sizeof(typename T::storage) == 2) {
    const dim3 grid = row_out_grid(a.rows);
    const int64_t nvec = (a.hidden + 7) >> 3;
    const bool many = a.rows >= 2 * (int64_t)device_cus();
    constexpr bool RMS = SRC == ROW_RMS, PLAIN = SRC == ROW_PLAIN;
#define SGLAMD_ROW_TEAM(NV) hipLaunchKernelGGL((row_out_team_kernel<T, WT, SRC, QK, NV, RAGGED>), row_out_grid(ceil_div(a.rows, 4)), dim3(256), 0, st, a)
#define SGLAMD_ROW_OUT(NT, NV) hipLaunchKernelGGL((row_out_kernel<T, WT, SRC, QK, NT, NV, RAGGED>), grid, dim3(NT), 0, st, a)
    if (nvec <= 64) SGLAMD_ROW_TEAM(1);
    else if (nvec <= 128 && (many || !RMS)) SGLAMD_ROW_TEAM(2);
    else if (PLAIN && many && nvec <= 256) SGLAMD_ROW_TEAM(PLAIN ? 4 : 2);
    else if (nvec <= 256) SGLAMD_ROW_OUT(256, 1);
    else if (nvec <= 512) SGLAMD_ROW_OUT((RMS ? 512 : 256), (RMS ? 1 : 2));
    else if (nvec <= 1024) SGLAMD_ROW_OUT((PLAIN ? 256 : 512), (PLAIN ? 4 : 2));
    else if (nvec <= 2048) SGLAMD_ROW_OUT(1024, 2);
    else SGLAMD_ROW_OUT((!RMS && QK == ROW_TO_ASYM ? 512 : 1024), (!RMS && QK == ROW_TO_ASYM ? 8 : 4));
#undef SGLAMD_ROW_OUT
#undef SGLAMD_ROW_TEAM
  }
}
// How the rows can be taken: in pieces of 8 values, 16 bytes in and 8 out, that stay in registers, each of them aligned or not, or
// value by value.  Aligned | unaligned, us: norm 4096 x 8192 39.8 | 43.8, SiLU 30.4 | 33.9, norm of one row of 7168 3.2 | 4.0.  Unaligned |
// value by value: norm 4096 x 4095 22.4 | 58.9, SiLU 892 x 10542 13.3 | 41.9, norm of one row of 7169 3.3 | 18.9.
enum RowPieces { ROW_VALUES, ROW_PIECES_ANYWHERE, ROW_PIECES };
template <typename T, typename WT, int SRC, int QK>
static void launch_row_out(const RowOutArgs& a, RowPieces pieces, hipStream_t st) {
  if (pieces == ROW_PIECES) launch_row_pieces<T, WT, SRC, QK, false>(a, st);
  else if (pieces == ROW_PIECES_ANYWHERE) launch_row_pieces<T, WT, SRC, QK, true>(a, st);
  else hipLaunchKernelGGL((row_out_any_kernel<T, WT, SRC, QK>), row_out_grid(a.rows), dim3(256), 0, st, a);
}
template <typename T, typename WT, int SRC>
static int launch_row_out_to(const RowOutArgs& a, int q_kind, RowPieces pieces, hipStream_t st) {
  if (q_kind == ROW_TO_FP8) launch_row_out<T, WT, SRC, ROW_TO_FP8>(a, pieces, st);
  else if (q_kind == ROW_TO_INT8) launch_row_out<T, WT, SRC, ROW_TO_INT8>(a, pieces, st);
  else launch_row_out<T, WT, SRC, ROW_TO_ASYM>(a, pieces, st);
  return check_launch("row_out");
}

// What every entry point asks of its rows and outputs.
static inline int check_row_out(const char* op, const RowOutArgs& a, int64_t width, int q_dtype) {
  SGLAMD_REQUIRE(a.x && a.q && a.s, SGLAMD_EINVAL, "%s: null pointer", op);
  SGLAMD_REQUIRE(a.rows >= 0 && a.rows < (1ll << 31) && a.hidden > 0 && a.hidden < (1ll << 31), SGLAMD_EINVAL,
                 "%s: bad sizes (%lld rows of %lld)", op, (long long)a.rows, (long long)a.hidden);
  SGLAMD_REQUIRE(a.x_stride >= 0 && (a.x_stride >= width || a.x_stride == 0), SGLAMD_EINVAL,
                 "%s: row stride %lld is smaller than the row (%lld)", op, (long long)a.x_stride, (long long)width);
  SGLAMD_REQUIRE(q_dtype == SGLAMD_FP8_E4M3 || q_dtype == SGLAMD_I8, SGLAMD_EINVAL, "%s: the codes must be FP8_E4M3 or I8", op);
  SGLAMD_REQUIRE(!a.zp || q_dtype == SGLAMD_I8, SGLAMD_EINVAL, "%s: zero points go with I8 codes", op);
  SGLAMD_REQUIRE(!a.fixed || q_dtype == SGLAMD_FP8_E4M3, SGLAMD_ENOTSUP, "%s: a given scale goes with FP8_E4M3 codes", op);
  return SGLAMD_OK;
}
static inline int row_out_kind(const RowOutArgs& a, int q_dtype) {
  return q_dtype == SGLAMD_FP8_E4M3 ? ROW_TO_FP8 : a.zp ? ROW_TO_ASYM : ROW_TO_INT8;
}
static inline bool aligned_to(const void* p, uintptr_t bytes) { return ((uintptr_t)p & (bytes - 1)) == 0; }
static inline RowPieces row_out_pieces(const RowOutArgs& a) {
  if (a.hidden < 8 || a.hidden > ROW_OUT_MAX_HIDDEN) return ROW_VALUES;
  const bool aligned = a.hidden % 8 == 0 && a.x_stride % 8 == 0 && aligned_to(a.x, 16) && aligned_to(a.q, 8) &&
                       (!a.res || (a.res_stride % 8 == 0 && aligned_to(a.res, 16) && aligned_to(a.res_out, 16))) && (!a.w || aligned_to(a.w, 16)) &&
                       (!a.y || aligned_to(a.y, 16));
  return aligned ? ROW_PIECES : ROW_PIECES_ANYWHERE;
}

}  // namespace sglamd
