// The expert layer of a few tokens whose rows are in 8 bits already, in two launches.
//
//   h = xs[t] * s13[e] * (x[t] . w13[e]) (+ b13[e]);  a = silu(h_gate) * h_up in fp32            first launch
//   a in 8 bits per (token, expert) pair;  out[t] = factor * sum over the token's pairs, in their order, of
//   weight * (as * s2[e] * (a . w2[e]) (+ b2[e]))                                                 second launch
//
// Bound by reading the chosen experts' weights once.  With one to some tokens an expert meets a handful of rows, and its
// product is that many dot products: they are formed by the vector unit (v_dot4_i32_i8; e4m3 as pairs of halves, which hold
// every e4m3 number, in v_dot2_f32_f16), at a few instructions per weight byte where the memory delivers ten bytes per
// clock to a CU.  So nothing is staged: LPR lanes read LPR * 16 contiguous bytes of a weight row, the weights go straight
// from memory into the registers of the lanes that multiply them, and LPR lanes add up at the end of a row.
//   * Pairs that name the same expert are one group: its weights are read once for up to R rows.  Groups are found from the
//     ids by ballots, by every wave for itself, so there is no sorting launch and nothing to clear.
//   * First launch: a wave owns 64 / LPR columns of one group, gate row and up row side by side, and writes a.
//   * Second launch: a workgroup owns 2 * 64 / LPR output columns and ALL pairs, a group to a wave in turn.  A wave quantises
//     the rows of its group itself, while its first weights are on their way; the pairs' results meet in LDS and are summed
//     in the pairs' order, so the sum over a token's experts needs neither atomics nor a launch.
#include "row_out.h"

namespace sglamd {

struct FewArgs {
  const uint8_t* x;   // [M, H] codes
  const float* xs;    // [M]
  const uint8_t* w;   // first: [E, 2 * I, H], second: [E, H, I]
  const float* s;     // first: [E, 2 * I], second: [E, H]
  const void* b;      // optional, like s, in the output's type
  const float* weights;  // [M, topk]
  const void* ids;       // [M, topk]
  int ids_i64;
  float* act;  // [M * topk, I]
  void* out;   // [M, H]
  float factor;
  int M, H, I, E, topk;
};

constexpr int FEW_MAX_PAIRS = 64;  // one lane each
constexpr int FEW_MAX_INTER = 16384;

typedef _Float16 h2 __attribute__((ext_vector_type(2)));

__device__ __forceinline__ v4i load_once(const uint8_t* p) { return __builtin_nontemporal_load((const v4i*)p); }

// acc[0][r] += w0 . x[r], acc[1][r] += w1 . x[r] over 16 codes.
template <bool INT8, int R, typename A>
__device__ __forceinline__ void dot16(const v4i& w0, const v4i& w1, const v4i (&x)[R], A (&acc)[2][R]) {
#pragma unroll
  for (int d = 0; d < 4; d++) {
    if constexpr (INT8) {
#pragma unroll
      for (int r = 0; r < R; r++) {
        acc[0][r] = __builtin_amdgcn_sdot4(w0[d], x[r][d], acc[0][r], false);
        acc[1][r] = __builtin_amdgcn_sdot4(w1[d], x[r][d], acc[1][r], false);
      }
    } else {
      const h2 a0 = __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(w0[d], 1.0f, false), a1 = __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(w0[d], 1.0f, true);
      const h2 b0 = __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(w1[d], 1.0f, false), b1 = __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(w1[d], 1.0f, true);
#pragma unroll
      for (int r = 0; r < R; r++) {
        const h2 x0 = __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(x[r][d], 1.0f, false), x1 = __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(x[r][d], 1.0f, true);
        acc[0][r] = __builtin_amdgcn_fdot2(a1, x1, __builtin_amdgcn_fdot2(a0, x0, acc[0][r], false), false);
        acc[1][r] = __builtin_amdgcn_fdot2(b1, x1, __builtin_amdgcn_fdot2(b0, x0, acc[1][r], false), false);
      }
    }
  }
}

// A batch of S steps of LPR * 16 bytes of two weight rows, per lane.
template <int S>
struct FewBatch {
  v4i w0[S], w1[S];
};
template <int S, int LPR>
__device__ __forceinline__ FewBatch<S> few_load(const uint8_t* w0, const uint8_t* w1, int step) {
  FewBatch<S> b;
#pragma unroll
  for (int s = 0; s < S; s++) {
    b.w0[s] = load_once(w0 + (int64_t)(step + s) * (LPR * 16));
    b.w1[s] = load_once(w1 + (int64_t)(step + s) * (LPR * 16));
  }
  return b;
}

// acc over a whole row of K codes.  w0, w1: the lane's piece of the first step; fetch(step, r): its piece of row r; `first`: the
// first batch where there is one (K / (LPR * 16) >= S).
template <bool INT8, int R, int LPR, int S, typename A, typename F>
__device__ __forceinline__ void few_dot(const uint8_t* w0, const uint8_t* w1, int K, int sub, const FewBatch<S>& first, F fetch, A (&acc)[2][R]) {
  const int full = K / (LPR * 16);
  int i = 0;
  FewBatch<S> cur = first;
  for (; i + S <= full; i += S) {
    FewBatch<S> next = cur;
    if (i + 2 * S <= full) next = few_load<S, LPR>(w0, w1, i + S);
    v4i x[S][R];
#pragma unroll
    for (int s = 0; s < S; s++)
#pragma unroll
      for (int r = 0; r < R; r++) x[s][r] = fetch(i + s, r);
#pragma unroll
    for (int s = 0; s < S; s++) dot16<INT8, R>(cur.w0[s], cur.w1[s], x[s], acc);
    cur = next;
  }
  // single steps, the last of them with lanes past the end of the row
  for (; i * (LPR * 16) < K; i++) {
    const bool live = i * (LPR * 16) + sub * 16 < K;
    v4i x[R], a = {0, 0, 0, 0}, b = {0, 0, 0, 0};
#pragma unroll
    for (int r = 0; r < R; r++) x[r] = v4i{0, 0, 0, 0};
    if (live) {
      a = load_once(w0 + (int64_t)i * (LPR * 16));
      b = load_once(w1 + (int64_t)i * (LPR * 16));
#pragma unroll
      for (int r = 0; r < R; r++) x[r] = fetch(i, r);
    }
    dot16<INT8, R>(a, b, x, acc);
  }
}

// Sum over each aligned group of LPR lanes, in all of them.
template <int LPR, typename A>
__device__ __forceinline__ A lanes_sum(A v) {
  auto add = [&](auto other) { v += other; };
  if constexpr (sizeof(A) == sizeof(float) && std::is_same<A, float>::value) {
    add(dpp_f<0xB1>(v));
    add(dpp_f<0x4E>(v));
    add(dpp_f<0x141>(v));
    if constexpr (LPR >= 16) add(dpp_f<0x140>(v));
  } else {
    add((A)dpp_u<0xB1>((uint32_t)v));
    add((A)dpp_u<0x4E>((uint32_t)v));
    add((A)dpp_u<0x141>((uint32_t)v));
    if constexpr (LPR >= 16) add((A)dpp_u<0x140>((uint32_t)v));
  }
  if constexpr (LPR >= 32) add(__shfl_xor(v, 16, 64));
  return v;
}

// The ids as the lanes hold them: lane p has the expert of pair p, -1 where there is no pair or it names an expert that lives
// elsewhere.
__device__ __forceinline__ int few_expert(const FewArgs& a, int pair) {
  if (pair >= a.M * a.topk) return -1;
  const int64_t id = a.ids_i64 ? ((const int64_t*)a.ids)[pair] : ((const int32_t*)a.ids)[pair];
  return id >= 0 && id < a.E ? (int)id : -1;
}
// Calls body(group, expert, members) for the groups in the order of their first pairs.
template <typename F>
__device__ __forceinline__ void few_groups(const FewArgs& a, F body) {
  const int mine = few_expert(a, threadIdx.x & 63);
  unsigned long long rest = __ballot(mine >= 0);
  for (int group = 0; rest; group++) {
    const int expert = __builtin_amdgcn_readlane(mine, __builtin_ctzll(rest));
    const unsigned long long members = __ballot(mine == expert);
    rest &= ~members;
    if (!body(group, expert, members)) return;
  }
}
// The next R members; pairs[] beyond their number repeat the first.
template <int R>
__device__ __forceinline__ int few_take(unsigned long long& members, int (&pairs)[R]) {
  int n = 0;
#pragma unroll
  for (int r = 0; r < R; r++) {
    pairs[r] = members ? (int)__builtin_ctzll(members) : pairs[0];
    n += members != 0;
    members &= members - 1;
  }
  return n;
}
template <int R>
__device__ __forceinline__ float few_pick(const float (&v)[R], int r) {
  float o = v[0];
#pragma unroll
  for (int j = 1; j < R; j++) o = r == j ? v[j] : o;
  return o;
}

template <bool INT8, typename OT, int R, int LPR, int S>
__device__ __forceinline__ void few_up_rows(const FewArgs& a, int expert, unsigned long long& members, int col, int sub) {
  typedef typename std::conditional<INT8, int, float>::type acc_t;
  const int n = min(col, a.I - 1);
  const int64_t gate_row = (int64_t)expert * 2 * a.I + n, up_row = gate_row + a.I;
  const uint8_t* w0 = a.w + gate_row * a.H + sub * 16;
  const uint8_t* w1 = a.w + up_row * a.H + sub * 16;
  FewBatch<S> first = {};
  if (a.H / (LPR * 16) >= S) first = few_load<S, LPR>(w0, w1, 0);
  int pairs[R];
  const int count = few_take<R>(members, pairs);
  const uint8_t* x[R];
#pragma unroll
  for (int r = 0; r < R; r++) x[r] = a.x + (int64_t)(pairs[r] / a.topk) * a.H + sub * 16;
  const float sg = a.s[gate_row], su = a.s[up_row];
  float bg = 0.f, bu = 0.f;
  if (a.b) {
    bg = OT::to_f32(((const typename OT::storage*)a.b)[gate_row]);
    bu = OT::to_f32(((const typename OT::storage*)a.b)[up_row]);
  }
  acc_t acc[2][R] = {};
  few_dot<INT8, R, LPR, S>(w0, w1, a.H, sub, first, [&](int step, int r) { return *(const v4i*)(x[r] + (int64_t)step * (LPR * 16)); }, acc);
  float v[R];
#pragma unroll
  for (int r = 0; r < R; r++) {
    const float xs = a.xs[pairs[r] / a.topk];
    const float g = (float)lanes_sum<LPR>(acc[0][r]) * (xs * sg) + bg, u = (float)lanes_sum<LPR>(acc[1][r]) * (xs * su) + bu;
    v[r] = g / (1.0f + expf(-g)) * u;
  }
#pragma unroll
  for (int r = 0; r < R; r++)
    if (sub == r && r < count && col < a.I) a.act[(int64_t)pairs[r] * a.I + col] = v[r];
}

// grid: column tiles of 4 waves x pairs (the groups are at most as many).
template <bool INT8, typename OT, int RMAX, int LPR>
__global__ __launch_bounds__(256) void few_up_kernel(FewArgs a) {
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int col = ((int)blockIdx.x * 4 + wave) * (64 / LPR) + lane / LPR;
  few_groups(a, [&](int group, int expert, unsigned long long members) {
    if (group != (int)blockIdx.y) return true;
    while (members) {
      if (RMAX == 1 || (members & (members - 1)) == 0) few_up_rows<INT8, OT, 1, LPR, 4>(a, expert, members, col, lane % LPR);
      else few_up_rows<INT8, OT, RMAX, LPR, 2>(a, expert, members, col, lane % LPR);
    }
    return false;
  });
}

// Row `pair` of a, quantised into LDS; returns its scale.  Up to 2048 values stay in registers between the maximum and the
// codes, longer rows are read again.
template <bool INT8>
__device__ __forceinline__ float few_quantise(const FewArgs& a, int pair, uint8_t* dst, int lane) {
  constexpr int KEEP = 8;
  const v4f* src = (const v4f*)(a.act + (int64_t)pair * a.I);
  const int chunks = a.I >> 2;
  v4f v[KEEP];
  uint32_t top = 0;
  auto take = [&](const v4f& c) {
#pragma unroll
    for (int j = 0; j < 4; j++) top = umax(top, __float_as_uint(c[j]) & 0x7fffffffu);
  };
#pragma unroll
  for (int k = 0; k < KEEP; k++) v[k] = lane + k * 64 < chunks ? src[lane + k * 64] : v4f{0.f, 0.f, 0.f, 0.f};
#pragma unroll
  for (int k = 0; k < KEEP; k++) take(v[k]);
  for (int c = lane + KEEP * 64; c < chunks; c += 64) take(src[c]);
  const float amax0 = __uint_as_float(wave_umax(top));
  float scale, mul;
  if constexpr (INT8) {
    const float amax = amax0 > 1e-10f || amax0 != amax0 ? amax0 : 1e-10f;
    scale = amax / 127.0f;
    mul = 127.0f / amax;
  } else {
    scale = amax0 / 448.0f;
    mul = scale == 0.f ? 0.f : 1.0f / scale;
  }
  const RowScale o = {scale, mul, 0.f, 1.f};
  auto put = [&](int c, const v4f& q) {
    const float f[4] = {q[0], q[1], q[2], q[3]};
    *(uint32_t*)(dst + 4 * c) = row_codes4<INT8 ? ROW_TO_INT8 : ROW_TO_FP8>(f, o);
  };
#pragma unroll
  for (int k = 0; k < KEEP; k++)
    if (lane + k * 64 < chunks) put(lane + k * 64, v[k]);
  for (int c = lane + KEEP * 64; c < chunks; c += 64) put(c, src[c]);
  return scale;
}

template <bool INT8, typename OT, int R, int LPR, int S>
__device__ __forceinline__ void few_down_rows(const FewArgs& a, int expert, unsigned long long& members, int n0, int sub, int lane, uint8_t* codes,
                                              float* part) {
  typedef typename std::conditional<INT8, int, float>::type acc_t;
  constexpr int COLS = 64 / LPR;
  const int na = min(n0, a.H - 1), nb = min(n0 + COLS, a.H - 1);
  const int64_t ra = (int64_t)expert * a.H + na, rb = (int64_t)expert * a.H + nb;
  const uint8_t* w0 = a.w + ra * a.I + sub * 16;
  const uint8_t* w1 = a.w + rb * a.I + sub * 16;
  FewBatch<S> first = {};
  if (a.I / (LPR * 16) >= S) first = few_load<S, LPR>(w0, w1, 0);
  int pairs[R];
  const int count = few_take<R>(members, pairs);
  float scale[R];
#pragma unroll
  for (int r = 0; r < R; r++) scale[r] = r < count ? few_quantise<INT8>(a, pairs[r], codes + r * a.I, lane) : 0.f;
  // (the rows are this wave's own: its LDS instructions run in order)
  asm volatile("s_waitcnt lgkmcnt(0)" : : : "memory");
  const float sa = a.s[ra], sb = a.s[rb];
  float ba = 0.f, bb = 0.f;
  if (a.b) {
    ba = OT::to_f32(((const typename OT::storage*)a.b)[ra]);
    bb = OT::to_f32(((const typename OT::storage*)a.b)[rb]);
  }
  const uint8_t* x = codes + sub * 16;
  acc_t acc[2][R] = {};
  few_dot<INT8, R, LPR, S>(w0, w1, a.I, sub, first,
                           [&](int step, int r) { return *(const v4i*)(x + (r < count ? r : 0) * a.I + step * (LPR * 16)); }, acc);
  float va[R], vb[R];
#pragma unroll
  for (int r = 0; r < R; r++) {
    const float wt = a.weights[pairs[r]];
    va[r] = ((float)lanes_sum<LPR>(acc[0][r]) * (scale[r] * sa) + ba) * wt;
    vb[r] = ((float)lanes_sum<LPR>(acc[1][r]) * (scale[r] * sb) + bb) * wt;
  }
#pragma unroll
  for (int r = 0; r < R; r++)
    if (sub == r && r < count) {
      part[pairs[r] * (2 * COLS) + lane / LPR] = va[r];
      part[pairs[r] * (2 * COLS) + COLS + lane / LPR] = vb[r];
    }
  asm volatile("" : : : "memory");  // the next rows overwrite the codes behind these reads
}

// grid: tiles of 2 * 64 / LPR output columns.  LDS: RMAX rows of I codes for each wave.
template <bool INT8, typename OT, int RMAX, int LPR>
__global__ __launch_bounds__(512) void few_down_kernel(FewArgs a) {
  typedef typename OT::storage OS;
  constexpr int COLS = 64 / LPR;
  extern __shared__ __attribute__((aligned(16))) uint8_t smem[];
  __shared__ float part[FEW_MAX_PAIRS * 2 * COLS];
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), waves = (int)blockDim.x >> 6;
  uint8_t* codes = smem + wave * RMAX * a.I;
  const int tile0 = (int)blockIdx.x * 2 * COLS;
  few_groups(a, [&](int group, int expert, unsigned long long members) {
    if (group % waves != wave) return true;
    while (members) {
      if (RMAX == 1 || (members & (members - 1)) == 0) few_down_rows<INT8, OT, 1, LPR, 4>(a, expert, members, tile0 + lane / LPR, lane % LPR, lane, codes, part);
      else few_down_rows<INT8, OT, RMAX, LPR, 2>(a, expert, members, tile0 + lane / LPR, lane % LPR, lane, codes, part);
    }
    return true;
  });
  __syncthreads();
  for (int i = threadIdx.x; i < a.M * 2 * COLS; i += blockDim.x) {
    const int t = i / (2 * COLS), c = i % (2 * COLS);
    if (tile0 + c >= a.H) continue;
    float sum = 0.f;
    for (int k = 0; k < a.topk; k++) {
      const int pair = t * a.topk + k;
      if (few_expert(a, pair) >= 0) sum += part[pair * (2 * COLS) + c];
    }
    ((OS*)a.out)[(int64_t)t * a.H + tile0 + c] = OT::from_f32(sum * a.factor);
  }
}

// Lanes per weight row: the fewest (8, the most work for a wave) that still give every CU `want` waves.
static int few_lanes(int64_t rows_of_groups, int rows_at_8, int want) {
  for (int lpr = 8; lpr < 32; lpr *= 2)
    if (rows_of_groups * lpr >= (int64_t)want * device_cus() * rows_at_8 * 8) return lpr;
  return 32;
}

template <bool INT8, typename OT, int RMAX, int LPR>
static int few_start_up(const FewArgs& a, hipStream_t st) {
  const dim3 grid((unsigned)ceil_div(a.I, 4 * (64 / LPR)), (unsigned)(a.M * a.topk));
  hipLaunchKernelGGL((few_up_kernel<INT8, OT, RMAX, LPR>), grid, dim3(256), 0, st, a);
  return check_launch("few_up");
}
template <bool INT8, typename OT, int RMAX, int LPR>
static int few_start_down(const FewArgs& a, int waves, hipStream_t st) {
  auto kern = few_down_kernel<INT8, OT, RMAX, LPR>;
  const int smem = waves * RMAX * a.I;
  if (smem > 60 * 1024) {
    static SmemAttrOnce attr;
    const hipError_t e = raise_dynamic_smem(attr, (const void*)kern, smem);
    if (e != hipSuccess) return fail(SGLAMD_EHIP, "hipFuncSetAttribute: %s", hipGetErrorString(e));
  }
  hipLaunchKernelGGL(kern, dim3((unsigned)ceil_div(a.H, 2 * (64 / LPR))), dim3(64 * waves), smem, st, a);
  return check_launch("few_down");
}

template <bool INT8, typename OT>
static int few_layer(const FewArgs& up, const FewArgs& down, hipStream_t st) {
  const int pairs = up.M * up.topk;
  const int waves = pairs < 8 ? pairs : 8;
  // Rows that one pass over an expert's weights may serve: as many as there are tokens, as LDS holds of them.
  int rmax = up.M == 1 ? 1 : up.M == 2 ? 2 : 4;
  while (rmax > 1 && waves * rmax * up.I > 64 * 1024) rmax /= 2;
  const int lpr1 = few_lanes((int64_t)up.I * pairs, 8, 12), lpr2 = few_lanes((int64_t)up.H * pairs, 16, 12);
#define SGLAMD_FEW(START, R, LPR, ...) (LPR == 8 ? START<INT8, OT, R, 8>(__VA_ARGS__) : LPR == 16 ? START<INT8, OT, R, 16>(__VA_ARGS__) : START<INT8, OT, R, 32>(__VA_ARGS__))
  const int rc = rmax == 1   ? SGLAMD_FEW(few_start_up, 1, lpr1, up, st)
                 : rmax == 2 ? SGLAMD_FEW(few_start_up, 2, lpr1, up, st)
                             : SGLAMD_FEW(few_start_up, 4, lpr1, up, st);
  if (rc) return rc;
  return rmax == 1   ? SGLAMD_FEW(few_start_down, 1, lpr2, down, waves, st)
         : rmax == 2 ? SGLAMD_FEW(few_start_down, 2, lpr2, down, waves, st)
                     : SGLAMD_FEW(few_start_down, 4, lpr2, down, waves, st);
#undef SGLAMD_FEW
}

}  // namespace sglamd

using namespace sglamd;

extern "C" int64_t sglamd_fused_experts_few_tokens_workspace(int64_t M, int64_t I, int topk) {
  return M > 0 && I > 0 && topk > 0 && M <= FEW_MAX_PAIRS && topk <= FEW_MAX_PAIRS && I <= FEW_MAX_INTER ? M * topk * I * 4 : 0;
}

extern "C" int sglamd_fused_experts_few_tokens(const void* x, const float* x_scale, int q_dtype, int64_t M, int64_t H, int64_t I, int E, int topk,
                                               const void* w13, const float* w13_scale, const void* b13, const void* w2,
                                               const float* w2_scale, const void* b2, const float* topk_weights, const void* topk_ids,
                                               int ids_dtype, void* out, int out_dtype, float routed_scaling_factor, void* workspace,
                                               int64_t workspace_bytes, void* stream) {
  const char* op = "fused_experts_few_tokens";
  SGLAMD_REQUIRE(x && x_scale && w13 && w13_scale && w2 && w2_scale && topk_weights && topk_ids && out && workspace, SGLAMD_EINVAL,
                 "%s: null pointer", op);
  SGLAMD_REQUIRE(q_dtype == SGLAMD_FP8_E4M3 || q_dtype == SGLAMD_I8, SGLAMD_EINVAL, "%s: the rows must be FP8_E4M3 or I8", op);
  SGLAMD_REQUIRE(out_dtype == SGLAMD_BF16 || out_dtype == SGLAMD_F16, SGLAMD_EINVAL, "%s: the output must be Half or BFloat16", op);
  SGLAMD_REQUIRE(ids_dtype == SGLAMD_I32 || ids_dtype == SGLAMD_I64, SGLAMD_EINVAL, "%s: topk_ids must be int32 or int64", op);
  SGLAMD_REQUIRE(M > 0 && E > 0 && topk > 0, SGLAMD_EINVAL, "%s: bad M/E/topk", op);
  SGLAMD_REQUIRE(M <= FEW_MAX_PAIRS && topk <= FEW_MAX_PAIRS && M * topk <= FEW_MAX_PAIRS, SGLAMD_ENOTSUP,
                 "%s: %lld tokens of %d experts are more than %d pairs", op, (long long)M, topk, FEW_MAX_PAIRS);
  SGLAMD_REQUIRE(H > 0 && I > 0 && H % 16 == 0 && I % 16 == 0, SGLAMD_EINVAL,
                 "%s: hidden (%lld) and intermediate (%lld) sizes must be multiples of 16", op, (long long)H, (long long)I);
  SGLAMD_REQUIRE(H < (1ll << 24) && I <= FEW_MAX_INTER, SGLAMD_ENOTSUP, "%s: sizes %lld and %lld are beyond %d and %d", op, (long long)H,
                 (long long)I, (1 << 24) - 1, FEW_MAX_INTER);
  // (sums of 2^31 / 128^2 int8 products stay inside 32 bits)
  SGLAMD_REQUIRE(q_dtype != SGLAMD_I8 || H <= 131071, SGLAMD_ENOTSUP, "%s: int8 rows of %lld are beyond 131071", op, (long long)H);
  SGLAMD_REQUIRE((((uintptr_t)x | (uintptr_t)w13 | (uintptr_t)w2 | (uintptr_t)workspace) & 15) == 0, SGLAMD_EINVAL,
                 "%s: rows, weights and workspace must be 16-byte aligned", op);
  SGLAMD_REQUIRE(workspace_bytes >= M * topk * I * 4, SGLAMD_EINVAL, "%s: workspace too small", op);
  const DeviceScope scope;
  FewArgs a = {};
  a.x = (const uint8_t*)x, a.xs = x_scale, a.w = (const uint8_t*)w13, a.s = w13_scale, a.b = b13, a.weights = topk_weights;
  a.ids = topk_ids, a.ids_i64 = ids_dtype == SGLAMD_I64, a.act = (float*)workspace, a.out = out, a.factor = routed_scaling_factor;
  a.M = (int)M, a.H = (int)H, a.I = (int)I, a.E = E, a.topk = topk;
  FewArgs d = a;
  d.w = (const uint8_t*)w2, d.s = w2_scale, d.b = b2;
  hipStream_t st = (hipStream_t)stream;
  if (q_dtype == SGLAMD_I8) return out_dtype == SGLAMD_BF16 ? few_layer<true, BF16>(a, d, st) : few_layer<true, F16>(a, d, st);
  return out_dtype == SGLAMD_BF16 ? few_layer<false, BF16>(a, d, st) : few_layer<false, F16>(a, d, st);
}
