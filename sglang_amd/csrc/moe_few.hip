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
//   * Pairs that name the same expert are one group: its weights are read once for up to RMAX rows.  Groups are found from the
//     ids by ballots, by every wave for itself, so there is no sorting launch and nothing to clear.
//   * First launch: a wave owns 64 / LPR columns of one group, gate row and up row side by side, and writes a.
//   * Second launch: a workgroup owns 2 * 64 / LPR output columns and ALL pairs, a group to a wave in turn.  A wave quantises
//     the rows of its group itself, in front of which it has requested its first weights; the pairs' results meet in LDS and
//     are summed in the pairs' order, so the sum over a token's experts needs neither atomics nor a launch.
//
// Measured (medians of traced launches, us; in brackets a bare read of the weights' bytes): 6 of 64 int8 experts of 4096 x 1536, one token,
// 14.1 + 10.3 (16.4); 8 of 128 e4m3 experts of 2048 x 768, three tokens, 14.6 + 11.5 (15.5); 8 of 256 of 7168 x 2048, one token 36.9 + 22.8
// (51), four 130 + 79 (195).  Large layers run at the rate of a read; small ones wait for two launches, and in each for a chain of ids, rows
// and first weights, some 4 us a launch.  Intermediate sizes beyond 2048 are far from it: the rows of a pass below, in few_layer, and too few
// waves in the second launch (8 int8 experts of 4096 x 14336, both launches and the quantiser, a read in brackets: two pairs of one token 101
// (51), eight tokens of two 603 (205)).
// Tried: the second launch's rows quantised by the workgroup together, behind a barrier (four tokens of the large layer 80 -> 89: all
// waves quantise at once and all stream at once); sixteen waves to all its workgroups (registers spill, or fewer are left for the loads:
// four tokens of the large layer 205 -> 214, both launches); a wave's next group requested under the results of the one before
// (80 -> 97 where it spills, 78 -> 80 elsewhere); the first launch's rows from L1 instead of LDS (their loads return behind the weights
// that were requested before them: 4096 x 1408, four tokens, 20.6 against 13.3).
#include <algorithm>

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
constexpr int FEW_MAX_HIDDEN = 32768, FEW_MAX_INTER = 16384;  // a row in LDS, eight of them
constexpr int FEW_DOWN_WAVES = 8;      // of the second launch, twice as many on up to FEW_SHORT_INTER values
constexpr int FEW_SHORT_INTER = 1024;
constexpr int FEW_LDS = 64 * 1024;  // what several rows for a pass may take, two workgroups to a CU

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

// A batch of S steps of LPR * 16 bytes of two weight rows, per lane.  The loads of a batch are straight-line code, and the next
// batch is requested without a condition: at a join of two paths the compiler could not tell how many loads are newer than the
// ones it waits for, and would wait for all (a conditional request cost a tenth of a layer of 64 experts of 4096 x 1536).
// Steps of a batch: two; four where several rows share a pass in a large layer (7168 x 2048, four tokens, 137 + 83 -> 133 + 80; one token of
// 4096 x 1536 with four 16.4 instead of 15.2).
constexpr int few_batch(int rmax, int lpr) { return rmax > 1 && lpr == 8 ? 4 : 2; }
template <int S>
struct FewBatch {
  v4i w0[S], w1[S];
};
template <int S, int LPR>
__device__ __forceinline__ void few_load(FewBatch<S>& b, const uint8_t* w0, const uint8_t* w1, int step) {
#pragma unroll
  for (int s = 0; s < S; s++) {
    b.w0[s] = load_once(w0 + (step + s) * (LPR * 16));
    b.w1[s] = load_once(w1 + (step + s) * (LPR * 16));
  }
}
// The batch that ends a row of K codes: pieces past its end are fetched from its last one and replaced by zeros.  (Behind zero
// weights the rows' codes are fetched from there too: only a row that holds a NaN multiplies one by a zero.)
template <int LPR>
__device__ __forceinline__ int few_piece(int step, int K, int sub) { return min(step * (LPR * 16), K - 16 - sub * 16); }
template <int S, int LPR>
__device__ __forceinline__ void few_load_last(FewBatch<S>& b, const uint8_t* w0, const uint8_t* w1, int step, int K, int sub) {
#pragma unroll
  for (int s = 0; s < S; s++) {
    const int at = few_piece<LPR>(step + s, K, sub);
    b.w0[s] = load_once(w0 + at);
    b.w1[s] = load_once(w1 + at);
  }
}
template <int S, int LPR>
__device__ __forceinline__ void few_load_first(FewBatch<S>& b, const uint8_t* w0, const uint8_t* w1, int K, int sub) {
  if (S * (LPR * 16) <= K) few_load<S, LPR>(b, w0, w1, 0);
  else few_load_last<S, LPR>(b, w0, w1, 0, K, sub);
}

// acc over a whole row of K codes.  w0, w1: the lane's piece of the first step, `cur` the first batch; fetch(offset, r): the lane's
// piece of row r, `offset` bytes behind that of its first step.
template <bool INT8, int R, int LPR, int S, typename A, typename F>
__device__ __forceinline__ void few_dot(const uint8_t* w0, const uint8_t* w1, int K, int sub, FewBatch<S>& cur, F fetch, A (&acc)[2][R]) {
  const int full = K / (LPR * 16), steps = (K + LPR * 16 - 1) / (LPR * 16);
  auto consume = [&](const FewBatch<S>& b, int i) {
#pragma unroll
    for (int s = 0; s < S; s++) {
      v4i x[R];
#pragma unroll
      for (int r = 0; r < R; r++) x[r] = fetch((i + s) * (LPR * 16), r);
      dot16<INT8, R>(b.w0[s], b.w1[s], x, acc);
    }
  };
  auto consume_last = [&](const FewBatch<S>& b, int i) {
#pragma unroll
    for (int s = 0; s < S; s++)
      if (i + s < steps) {
        const v4i zero = {0, 0, 0, 0};
        const bool live = (i + s) * (LPR * 16) + sub * 16 < K;
        v4i x[R];
#pragma unroll
        for (int r = 0; r < R; r++) x[r] = fetch(few_piece<LPR>(i + s, K, sub), r);
        dot16<INT8, R>(live ? b.w0[s] : zero, live ? b.w1[s] : zero, x, acc);
        }
  };
  FewBatch<S> next;
  int i = 0;
  if (S <= full) {
    for (; i + 2 * S <= full; i += S) {
      few_load<S, LPR>(next, w0, w1, i + S);
      consume(cur, i);
      cur = next;
    }
    few_load_last<S, LPR>(next, w0, w1, min(i + S, steps - 1), K, sub);  // (where nothing is left, the last step again)
    consume(cur, i);
    cur = next;
    i += S;
  }
  if (i < steps) consume_last(cur, i);
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
// The rows of a group that are still to be multiplied (0: none).
struct FewGroup {
  int expert;
  unsigned long long members;
};
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
// grid: column tiles of 4 waves x pairs (the groups are at most as many).  LDS: RMAX rows of H codes.
template <bool INT8, typename OT, int RMAX, int LPR>
__global__ __launch_bounds__(256) void few_up_kernel(FewArgs a) {
  typedef typename std::conditional<INT8, int, float>::type acc_t;
  constexpr int S = few_batch(RMAX, LPR);
  extern __shared__ __attribute__((aligned(16))) uint8_t rows[];
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), sub = lane % LPR;
  const int col = ((int)blockIdx.x * 4 + wave) * (64 / LPR) + lane / LPR;
  FewGroup g = {0, 0};
  few_groups(a, [&](int group, int expert, unsigned long long members) {
    if (group == (int)blockIdx.y) g = {expert, members};
    return group != (int)blockIdx.y;
  });
  if (!g.members) return;  // (the same for the whole workgroup)
  const int64_t gate_row = (int64_t)g.expert * 2 * a.I + min(col, a.I - 1), up_row = gate_row + a.I;
  const uint8_t *w0 = a.w + gate_row * a.H + sub * 16, *w1 = a.w + up_row * a.H + sub * 16;
  const float sg = a.s[gate_row], su = a.s[up_row];
  float bg = 0.f, bu = 0.f;
  if (a.b) {
    bg = OT::to_f32(((const typename OT::storage*)a.b)[gate_row]);
    bu = OT::to_f32(((const typename OT::storage*)a.b)[up_row]);
  }
  for (;;) {
    FewBatch<S> batch;
    few_load_first<S, LPR>(batch, w0, w1, a.H, sub);
    int pairs[RMAX];
    const int count = few_take<RMAX>(g.members, pairs);
    const int chunks = a.H >> 4;
#pragma unroll
    for (int r = 0; r < RMAX; r++) {
      if (r >= count) break;
      const v4i* src = (const v4i*)(a.x + (int64_t)(pairs[r] / a.topk) * a.H);
      for (int c = threadIdx.x; c < chunks; c += 256) *(v4i*)(rows + r * a.H + c * 16) = src[c];
    }
    __syncthreads();
    acc_t acc[2][RMAX] = {};
    auto fetch = [&](int at, int r) { return *(const v4i*)(rows + (r < count ? r : 0) * a.H + sub * 16 + at); };
    if (RMAX > 1 && count > 1) {
      few_dot<INT8, RMAX, LPR, S>(w0, w1, a.H, sub, batch, fetch, acc);
    } else {
      acc_t one[2][1] = {};
      few_dot<INT8, 1, LPR, S>(w0, w1, a.H, sub, batch, fetch, one);
      acc[0][0] = one[0][0], acc[1][0] = one[1][0];
    }
#pragma unroll
    for (int r = 0; r < RMAX; r++) {
      if (r >= count) break;
      const float xs = a.xs[pairs[r] / a.topk];
      const float gate = (float)lanes_sum<LPR>(acc[0][r]) * (xs * sg) + bg, up = (float)lanes_sum<LPR>(acc[1][r]) * (xs * su) + bu;
      if (sub == r && col < a.I) a.act[(int64_t)pairs[r] * a.I + col] = gate / (1.0f + expf(-gate)) * up;
    }
    if (!g.members) return;
    __syncthreads();  // the next rows take the place of these
  }
}

// Row `pair` of a, quantised into LDS; returns its scale.  Up to KEEP * 256 values stay in registers between the maximum and the
// codes, longer rows are read again.
template <int KEEP>
__device__ __forceinline__ void few_act_load(const FewArgs& a, int pair, int lane, v4f (&v)[KEEP]) {
  const v4f* src = (const v4f*)(a.act + (int64_t)pair * a.I);
#pragma unroll
  for (int k = 0; k < KEEP; k++) v[k] = src[min(lane + k * 64, (a.I >> 2) - 1)];  // (repeats change no maximum)
}
template <bool INT8, int KEEP>
__device__ __forceinline__ float few_quantise(const FewArgs& a, int pair, uint8_t* dst, int lane, const v4f (&v)[KEEP]) {
  const v4f* src = (const v4f*)(a.act + (int64_t)pair * a.I);
  const int chunks = a.I >> 2;
  uint32_t top = 0;
  auto take = [&](const v4f& c) {
#pragma unroll
    for (int j = 0; j < 4; j++) top = umax(top, __float_as_uint(c[j]) & 0x7fffffffu);
  };
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
    mul = fp8_row_multiplier(1.0f, scale);
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

// grid: tiles of 2 * 64 / LPR output columns, a group to a wave in turn.  LDS: RMAX rows of I codes for each wave.
template <bool INT8, typename OT, int RMAX, int LPR, int KEEP, int NT>
__global__ __launch_bounds__(NT) void few_down_kernel(FewArgs a) {
  typedef typename OT::storage OS;
  typedef typename std::conditional<INT8, int, float>::type acc_t;
  constexpr int COLS = 64 / LPR, S = few_batch(RMAX, LPR);
  extern __shared__ __attribute__((aligned(16))) uint8_t smem[];
  __shared__ float part[FEW_MAX_PAIRS * 2 * COLS];
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), waves = (int)blockDim.x >> 6;
  const int sub = lane % LPR, tile0 = (int)blockIdx.x * 2 * COLS;
  const int na = min(tile0 + lane / LPR, a.H - 1), nb = min(tile0 + COLS + lane / LPR, a.H - 1);
  uint8_t* codes = smem + wave * RMAX * a.I;
  const int mine = few_expert(a, lane);
  unsigned long long rest = __ballot(mine >= 0);
  int turn = wave;
  auto next = [&](const FewGroup& g) -> FewGroup {
    if (g.members) return g;  // more rows of this group than one pass serves
    while (rest) {
      const int expert = __builtin_amdgcn_readlane(mine, __builtin_ctzll(rest));
      const unsigned long long members = __ballot(mine == expert);
      rest &= ~members;
      if (turn-- == 0) {
        turn = waves - 1;
        return {expert, members};
      }
    }
    return {0, 0};
  };
  // A group's first row, then its first weights: loads return in the order of their requests.
  v4f row[KEEP];
  FewBatch<S> batch;
  const uint8_t *w0, *w1;
  auto request = [&](const FewGroup& g) {
    few_act_load(a, __builtin_ctzll(g.members), lane, row);
    w0 = a.w + ((int64_t)g.expert * a.H + na) * a.I + sub * 16;
    w1 = a.w + ((int64_t)g.expert * a.H + nb) * a.I + sub * 16;
    few_load_first<S, LPR>(batch, w0, w1, a.I, sub);
  };
  FewGroup g = next({0, 0});
  if (g.members) request(g);
  while (g.members) {
    int pairs[RMAX];
    const int count = few_take<RMAX>(g.members, pairs);
    float scale[RMAX];
#pragma unroll
    for (int r = 0; r < RMAX; r++) {
      scale[r] = 0.f;
      if (r >= count) continue;
      if (r > 0) few_act_load(a, pairs[r], lane, row);
      scale[r] = few_quantise<INT8, KEEP>(a, pairs[r], codes + r * a.I, lane, row);
    }
    // (the rows are this wave's own: its LDS instructions run in order)
    asm volatile("s_waitcnt lgkmcnt(0)" : : : "memory");
    const int64_t ra = (int64_t)g.expert * a.H + na, rb = (int64_t)g.expert * a.H + nb;
    const float sa = a.s[ra], sb = a.s[rb];
    float ba = 0.f, bb = 0.f;
    if (a.b) {
      ba = OT::to_f32(((const OS*)a.b)[ra]);
      bb = OT::to_f32(((const OS*)a.b)[rb]);
    }
    acc_t acc[2][RMAX] = {};
    auto fetch = [&](int at, int r) { return *(const v4i*)(codes + (r < count ? r : 0) * a.I + sub * 16 + at); };
    if (RMAX > 1 && count > 1) {
      few_dot<INT8, RMAX, LPR, S>(w0, w1, a.I, sub, batch, fetch, acc);
    } else {
      acc_t one[2][1] = {};
      few_dot<INT8, 1, LPR, S>(w0, w1, a.I, sub, batch, fetch, one);
      acc[0][0] = one[0][0], acc[1][0] = one[1][0];
    }
    asm volatile("" : : : "memory");  // the next rows overwrite the codes behind these reads
#pragma unroll
    for (int r = 0; r < RMAX; r++) {
      if (r >= count) break;
      const float wt = a.weights[pairs[r]];
      const float va = ((float)lanes_sum<LPR>(acc[0][r]) * (scale[r] * sa) + ba) * wt, vb = ((float)lanes_sum<LPR>(acc[1][r]) * (scale[r] * sb) + bb) * wt;
      if (sub == r) {
        part[pairs[r] * (2 * COLS) + lane / LPR] = va;
        part[pairs[r] * (2 * COLS) + COLS + lane / LPR] = vb;
      }
    }
    g = next(g);
    if (g.members) request(g);
  }
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

template <bool INT8, typename OT, int RMAX, int LPR>
static int few_start_up(const FewArgs& a, hipStream_t st) {
  const dim3 grid((unsigned)ceil_div(a.I, 4 * (64 / LPR)), (unsigned)(a.M * a.topk));
  auto kern = few_up_kernel<INT8, OT, RMAX, LPR>;
  const int smem = std::min(RMAX, a.M * a.topk) * a.H;
  if (smem > 56 * 1024) {
    static SmemAttrOnce attr;
    const hipError_t e = raise_dynamic_smem(attr, (const void*)kern, smem);
    if (e != hipSuccess) return fail(SGLAMD_EHIP, "hipFuncSetAttribute: %s", hipGetErrorString(e));
  }
  hipLaunchKernelGGL(kern, grid, dim3(256), smem, st, a);
  return check_launch("few_up");
}
template <bool INT8, typename OT, int RMAX, int LPR, int WAVES>
static int few_start_down_waves(const FewArgs& a, hipStream_t st) {
  auto kern = few_down_kernel<INT8, OT, RMAX, LPR, WAVES == FEW_DOWN_WAVES ? 8 : FEW_SHORT_INTER / 256, 64 * WAVES>;
  const int waves = std::min(a.M * a.topk, WAVES), smem = waves * RMAX * a.I;
  if (smem > 56 * 1024) {
    static SmemAttrOnce attr;
    const hipError_t e = raise_dynamic_smem(attr, (const void*)kern, smem);
    if (e != hipSuccess) return fail(SGLAMD_EHIP, "hipFuncSetAttribute: %s", hipGetErrorString(e));
  }
  hipLaunchKernelGGL(kern, dim3((unsigned)ceil_div(a.H, 2 * (64 / LPR))), dim3(64 * waves), smem, st, a);
  return check_launch("few_down");
}

// Eight waves; sixteen of at most two rows a pass where the pairs take more than one turn on rows so short that the registers of
// sixteen suffice, and the chain of a turn counts, not its bytes (8 | 16 waves, both launches: 8 of 128 experts of 2048 x 768, three tokens
// 30.0 | 26.2 us, eight 63.6 | 53.9; 6 of 64 of 2048 x 1024, four 33.0 | 30.6; 8 of 64 of 1024 x 512, eight 32.9 | 27.6; where eight lanes
// read a row they spill: 8 of 64 of 4096 x 1024, three 57.5 | 66.8, of one row a pass 58.8).
template <bool INT8, typename OT, int RMAX, int LPR>
static int few_start_down(const FewArgs& a, hipStream_t st) {
  if constexpr (LPR > 8)
    if (a.M * a.topk > FEW_DOWN_WAVES && a.I <= FEW_SHORT_INTER) return few_start_down_waves<INT8, OT, RMAX == 1 ? 1 : 2, LPR, 2 * FEW_DOWN_WAVES>(a, st);
  return few_start_down_waves<INT8, OT, RMAX, LPR, FEW_DOWN_WAVES>(a, st);
}

template <bool INT8, typename OT>
static int few_layer(const FewArgs& up, const FewArgs& down, hipStream_t st) {
  const int pairs = up.M * up.topk, cus = device_cus();
  // Rows that one pass over an expert's weights serves, in both launches: as many as there are tokens, as LDS holds of them (with eight pairs
  // and more four up to I = 2048, two up to 4096, else one).
  int rmax = up.M == 1 ? 1 : up.M == 2 ? 2 : 4;
  while (rmax > 1 && (std::min(pairs, FEW_DOWN_WAVES) * rmax * up.I > FEW_LDS || rmax * up.H > FEW_LDS)) rmax /= 2;
  // Lanes per weight row.  First launch: eight, where that gives a CU six waves, else 32 (8 | 32 lanes: 7168 x 2048, one token, eight waves
  // a CU, 37.6 | 38.5 us; 2048 x 768, three tokens, nine, 15.0 | 16.7; 4096 x 1536, one token, 4.5, 16.5 | 14.9; 2048 x 768, one token,
  // three, 8.5 | 6.8).  Second: the fewest of 8, 16 and 32 whose column tiles reach every CU (8 | 16: 4096 columns, 256 tiles of 8,
  // 10.2 | 12.0; 2048 columns, 128 tiles of 8, 17.4 | 13.9; 8 | 16 | 32: 1024 columns 9.2 | 8.2 | 7.8).
  const bool wide = (int64_t)pairs * up.I >= 6 * 8 * (int64_t)cus;
  const int lpr = up.H >= 16 * cus ? 8 : up.H >= 8 * cus ? 16 : 32;
#define SGLAMD_FEW_UP(R) (wide ? few_start_up<INT8, OT, R, 8>(up, st) : few_start_up<INT8, OT, R, 32>(up, st))
#define SGLAMD_FEW_DOWN(R) \
  (lpr == 8 ? few_start_down<INT8, OT, R, 8>(down, st) : lpr == 16 ? few_start_down<INT8, OT, R, 16>(down, st) : few_start_down<INT8, OT, R, 32>(down, st))
  const int rc = rmax == 1 ? SGLAMD_FEW_UP(1) : rmax == 2 ? SGLAMD_FEW_UP(2) : SGLAMD_FEW_UP(4);
  if (rc) return rc;
  return rmax == 1 ? SGLAMD_FEW_DOWN(1) : rmax == 2 ? SGLAMD_FEW_DOWN(2) : SGLAMD_FEW_DOWN(4);
#undef SGLAMD_FEW_UP
#undef SGLAMD_FEW_DOWN
}

}  // namespace sglamd

using namespace sglamd;

extern "C" int64_t sglamd_fused_experts_few_tokens_workspace(int64_t M, int64_t I, int topk) {
  const bool taken = M > 0 && I > 0 && topk > 0 && M <= FEW_MAX_PAIRS && topk <= FEW_MAX_PAIRS && M * topk <= FEW_MAX_PAIRS && I <= FEW_MAX_INTER;
  return taken ? M * topk * I * 4 : 0;
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
  SGLAMD_REQUIRE(H <= FEW_MAX_HIDDEN && I <= FEW_MAX_INTER, SGLAMD_ENOTSUP, "%s: sizes %lld and %lld are beyond %d and %d", op, (long long)H,
                 (long long)I, FEW_MAX_HIDDEN, FEW_MAX_INTER);
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
