// Heads of queries, keys and values between a projection and its attention: RMSNorm of each head, rotary positions, rows of a
// paged cache in 16 or 8 bits, and such rows back in 16 bits.
//
//   norm    y = x * r * w,  r = 1 / sqrt(mean(x^2) + eps) over one head
//   rotate  pair i of a token on position p: (a, b) -> (a c - b s, b c + a s), c = table[p][i], s = table[p][i + pairs]
//   codes   those of row_out.h: e4m3 with scale = max|y| / 448 or as given, int8 with scale = max(max|y|, 1e-10) / 127
//
// Everything between the load of a head and its stores is in fp32 and rounded once, to the type of the row that is written.
//
// All of it is bound by HBM at prompt sizes (some ten operations per value, each value read once and written once) and by the launch
// at decode sizes, so one launch does everything that a layer needs between its projection and its attention.  Measured
// against a copy of as many bytes (5.05 TB/s): 8191 tokens of 64 + 2 x 8 heads of 128, rotated, into e4m3 rows 5.4 TB/s; 4096 tokens
// of 128 rotary parts, 128 bytes in each 384, 4.5 (a copy of such pieces 4.6); gathered int8 rows 5.0; heads with a norm 4.5 to 4.7,
// alternating axes 4.2.  Written are exactly the outputs' bytes, read 1.01 to 1.07 of the inputs' (counters).
// What decided it, in this order: pieces in words (a piece of eight 16-bit values that may not be there was held in
// eight registers), one head per lane group in at most 64 registers (four heads: 4.9 TB/s instead of 5.4), loads without
// conditions (a condition between two loads makes the first wait for both), and the kernel's arguments touched at the start.
#include <utility>

#include "row_out.h"

namespace sglamd {

enum { HEADS_TO_NONE = 0, HEADS_TO_16 = 1, HEADS_TO_FP8 = 2, HEADS_TO_INT8 = 3 };

struct HeadPart {
  const u16* x;
  int64_t x_token, x_head;
  const void* w;  // RMSNorm weight, or null
  u16* out;       // 16-bit rows, or null
  int64_t out_token, out_head;
  uint8_t* cache;  // rows of the slots, or null; strides in bytes
  int64_t cache_page, cache_slot, cache_head;
  const float* given;  // scale, one or one per head
  float* scales;       // scales that are found here, one per row or per 128 values of it
  int64_t given_head, scales_page, scales_slot, scales_head, scales_group;
  float eps, inv_dim;
  uint32_t groups;  // lane groups of this part: tokens * per_token
  FastDiv per_token_div;
  int per_token, heads, units, rot_units;
  int lanes_log2, kind, w_is_f32, grouped;  // grouped: a scale per 128 values
};

constexpr int MAX_PARTS = 3;

struct HeadArgs {
  HeadPart part[MAX_PARTS];
  uint32_t first_block[MAX_PARTS];  // of each part; behind the last block for parts that are not there
  // rotation
  const void* table;
  int64_t table_stride, table_rows, axis_stride, position_stride;
  const void* positions;
  int pairs, table_is_f32, positions_are_i64, axes;
  uint32_t axis_bits[2][16];  // the axis of each pair, its low and its high bit
  // slots
  const void* slots;
  int64_t slot_stride, num_slots;
  int slots_are_i64, page_size;
  FastDiv page_div;
};

// Every line of the kernel's arguments into the scalar cache, in one round trip: they lie in memory that the caches below do not
// hold, and line after line, each where its fields are first used, a workgroup waits about a microsecond for each.
__device__ __forceinline__ int touched(uint32_t word) {
  asm volatile("" ::"s"(word));
  return 0;
}
template <typename ARGS, int... I>
__device__ __forceinline__ void touch_lines(const ARGS& a, std::integer_sequence<int, I...>) {
  const uint32_t w[] = {((const uint32_t*)&a)[16 * I]...};
  const int done[] = {touched(w[I])...};
  (void)done;
}
template <typename ARGS>
__device__ __forceinline__ void touch_arguments(const ARGS& a) {
  touch_lines(a, std::make_integer_sequence<int, (sizeof(ARGS) + 63) / 64>());
}

// V 16-bit values as loaded: words, so that a piece that may not be there is held in words too.
template <int V>
struct Piece {
  typedef uint32_t type __attribute__((ext_vector_type(V / 2)));
};
template <>
struct Piece<1> {
  typedef uint32_t type;
};
template <int V>
__device__ __forceinline__ typename Piece<V>::type load_values(const u16* p) {  // (global memory takes any alignment)
  if constexpr (V == 1) {
    return *p;
  } else {
    typename Piece<V>::type v;
    __builtin_memcpy(&v, p, sizeof(v));
    return v;
  }
}
template <typename T, int V>
__device__ __forceinline__ void to_floats(const typename Piece<V>::type& p, float* f) {
  if constexpr (V == 1) {
    f[0] = T::to_f32((u16)p);
  } else {
#pragma unroll
    for (int i = 0; i < V / 2; i++) f[2 * i] = T::to_f32((u16)p[i]), f[2 * i + 1] = T::to_f32((u16)(p[i] >> 16));
  }
}
// The last product of a value is rounded to fp32 before its conversion: one instruction makes both for halves and rounds once, and
// the compiler takes it for some values of a row and not for others, so that a row's last bits would depend on the instance.
template <typename T>
__device__ __forceinline__ float in_fp32(float f) {
  if constexpr (T::tag == SGLAMD_F16) asm("" : "+v"(f));
  return f;
}
template <typename T, int V>
__device__ __forceinline__ void store_values(u16* p, const float* f) {
  if constexpr (V == 1) {
    *p = T::from_f32(in_fp32<T>(f[0]));
  } else {
    uint32_t w[V / 2];
#pragma unroll
    for (int i = 0; i < V / 2; i++) w[i] = T::pack2(in_fp32<T>(f[2 * i]), in_fp32<T>(f[2 * i + 1]));
    __builtin_memcpy(p, w, 2 * V);
  }
}
template <int QK, int V>
__device__ __forceinline__ void store_codes(uint8_t* p, const float* f, const RowScale& o) {
  if constexpr (V == 1) {
    const float v[4] = {f[0], 0.f, 0.f, 0.f};
    *p = (uint8_t)row_codes4<QK>(v, o);
  } else {
    uint32_t w[V / 4];
#pragma unroll
    for (int i = 0; i < V / 4; i++) w[i] = row_codes4<QK>(f + 4 * i, o);
    __builtin_memcpy(p, w, V);
  }
}
// N cosines or sines at a byte offset into the table: 32 bits, beside its address in scalar registers.
template <typename T, int N>
__device__ __forceinline__ void load_table(const HeadArgs& a, uint32_t at, float* f) {
  const char* p = (const char*)a.table + at;
  if (a.table_is_f32) __builtin_memcpy(f, p, 4 * N);
  else to_floats<T, N>(load_values<N>((const u16*)p), f);
}
// Weights as fp32, ones where there are none; those of 16 bits have been loaded already.
template <typename T, int V>
__device__ __forceinline__ void weights(const HeadPart& p, int at, const typename Piece<V>::type& raw, float* w) {
  if (p.w_is_f32) {
    __builtin_memcpy(w, (const char*)p.w + (uint32_t)(4 * at), 4 * V);
  } else {
    to_floats<T, V>(raw, w);
#pragma unroll
    for (int i = 0; i < V; i++) w[i] = p.w ? w[i] : 1.f;
  }
}
// An index in two words, without a branch on its type: what is loaded behind it can be waited for by itself.
struct Index {
  int lo, hi;
  __device__ __forceinline__ int64_t value(int is_i64) const { return (int64_t)(uint32_t)lo | (int64_t)(is_i64 ? hi : lo >> 31) << 32; }
};
__device__ __forceinline__ Index load_index(const void* base, int64_t at, int is_i64) {
  const int* p = (const int*)base + (is_i64 ? 2 * at : at);
  return {p[0], p[is_i64 ? 1 : 0]};
}

// The values are computed here and not later, and what is loaded below is not loaded above.
template <int V>
__device__ __forceinline__ void pin(float* f) {
#pragma unroll
  for (int i = 0; i < V; i++) asm volatile("" : "+v"(f[i])::"memory");
}

// Sum and maximum over aligned groups of 2^log lanes, in all of them; `log` is the same in the whole wave.
__device__ __forceinline__ float group_sum(float v, int log) {
  if (log >= 1) v += dpp_f<0xB1>(v);   // quad_perm [1, 0, 3, 2]
  if (log >= 2) v += dpp_f<0x4E>(v);   // quad_perm [2, 3, 0, 1]
  if (log >= 3) v += dpp_f<0x141>(v);  // row_half_mirror
  if (log >= 4) v += dpp_f<0x140>(v);  // row_mirror
  if (log >= 5) v += __shfl_xor(v, 16, 64);
  if (log >= 6) v += __shfl_xor(v, 32, 64);
  return v;
}
__device__ __forceinline__ uint32_t group_umax(uint32_t v, int log) {
  if (log >= 1) v = umax(v, dpp_u<0xB1>(v));
  if (log >= 2) v = umax(v, dpp_u<0x4E>(v));
  if (log >= 3) v = umax(v, dpp_u<0x141>(v));
  if (log >= 4) v = umax(v, dpp_u<0x140>(v));
  if (log >= 5) v = umax(v, (uint32_t)__shfl_xor((int)v, 16, 64));
  if (log >= 6) v = umax(v, (uint32_t)__shfl_xor((int)v, 32, 64));
  return v;
}

// Which axes the N pairs from `first` on turn by: the low and the high bits of their numbers.
struct AxisBits {
  uint32_t lo, hi;
};
template <int N>
__device__ __forceinline__ AxisBits axes_of_pairs(const HeadArgs& a, int first) {
  constexpr uint32_t ALL = (1u << N) - 1;
  AxisBits b = {0, 0};
  // (word by word, in scalar registers: vector loads of kernel arguments cross to the host's memory)
  for (int w = 0; w * 32 < a.pairs; w++) {
    const uint32_t lo = __builtin_amdgcn_readfirstlane(a.axis_bits[0][w]), hi = __builtin_amdgcn_readfirstlane(a.axis_bits[1][w]);
    b.lo = first >> 5 == w ? lo : b.lo;
    b.hi = first >> 5 == w ? hi : b.hi;
  }
  return {b.lo >> (first & 31) & ALL, b.hi >> (first & 31) & ALL};
}
// (values and not an array: the choice of an address would put it into memory)
template <typename E>
__device__ __forceinline__ E of_axis(const AxisBits& b, int i, E v0, E v1, E v2, E v3) {
  const E low = b.lo >> i & 1 ? v1 : v0, high = b.lo >> i & 1 ? v3 : v2;
  return b.hi >> i & 1 ? high : low;
}

// Cosines and sines of the N pairs from `first` on, `rows` (byte offsets into the table) and `inside` for each axis.  A position
// outside of the table gives NaN, and reads the table's first row.
template <typename T, int N, bool AXES>
__device__ __forceinline__ void load_turn(const HeadArgs& a, const uint32_t (&rows)[AXES ? 4 : 1], const bool (&inside)[AXES ? 4 : 1],
                                          const AxisBits& axes, int first, float* c, float* s) {
  const int item = a.table_is_f32 ? 4 : 2;
  const uint32_t pair = (uint32_t)(first * item), sines = (uint32_t)(a.pairs * item);
  if constexpr (!AXES) {
    load_table<T, N>(a, rows[0] + pair, c);
    load_table<T, N>(a, rows[0] + pair + sines, s);
    if (__any(!inside[0])) {
#pragma unroll
      for (int i = 0; i < N; i++) c[i] = inside[0] ? c[i] : NAN, s[i] = inside[0] ? s[i] : NAN;
    }
  } else {
    constexpr uint32_t ALL = (1u << N) - 1;
    // (a text token has the same position on every axis; axes in blocks change once in a while)
    const bool same = rows[0] == rows[1] && rows[0] == rows[2] && rows[0] == rows[3];
    if (same || ((axes.lo == 0 || axes.lo == ALL) && (axes.hi == 0 || axes.hi == ALL))) {
      const uint32_t at = of_axis(axes, 0, rows[0], rows[1], rows[2], rows[3]) + pair;
      load_table<T, N>(a, at, c);
      load_table<T, N>(a, at + sines, s);
    } else if (a.table_is_f32) {
#pragma unroll
      for (int i = 0; i < N; i++) {
        const uint32_t at = of_axis(axes, i, rows[0], rows[1], rows[2], rows[3]) + pair + 4 * i;
        c[i] = *(const float*)((const char*)a.table + at);
        s[i] = *(const float*)((const char*)a.table + (uint32_t)(at + sines));
      }
    } else {
#pragma unroll
      for (int i = 0; i < N; i++) {
        const uint32_t at = of_axis(axes, i, rows[0], rows[1], rows[2], rows[3]) + pair + 2 * i;
        c[i] = T::to_f32(*(const u16*)((const char*)a.table + at));
        s[i] = T::to_f32(*(const u16*)((const char*)a.table + (uint32_t)(at + sines)));
      }
    }
    if (__any(!(inside[0] && inside[1] && inside[2] && inside[3]))) {
#pragma unroll
      for (int i = 0; i < N; i++) {
        const bool ok = of_axis(axes, i, inside[0], inside[1], inside[2], inside[3]);
        c[i] = ok ? c[i] : NAN, s[i] = ok ? s[i] : NAN;
      }
    }
  }
}

// f0 and f1: the V values of a unit's two pieces.
template <int V, bool ADJACENT>
__device__ __forceinline__ void turn(float* f0, float* f1, const float* c, const float* s) {
  if constexpr (!ADJACENT || V == 1) {
#pragma unroll
    for (int i = 0; i < V; i++) {
      const float x = f0[i], y = f1[i];
      f0[i] = fmaf(x, c[i], -(y * s[i]));
      f1[i] = fmaf(y, c[i], x * s[i]);
    }
  } else {
#pragma unroll
    for (int i = 0; i < V; i++) {
      float* f = i < V / 2 ? f0 + 2 * i : f1 + 2 * i - V;
      const float x = f[0], y = f[1];
      f[0] = fmaf(x, c[i], -(y * s[i]));
      f[1] = fmaf(y, c[i], x * s[i]);
    }
  }
}

template <int QK>
__device__ __forceinline__ RowScale found_scale(uint32_t hi_bits) {
  RowScale o = {};
  const float hi = __uint_as_float(hi_bits);
  if constexpr (QK == ROW_TO_FP8) {
    o.scale = hi / 448.0f;
    o.mul = fp8_row_multiplier(1.0f, o.scale);
  } else {
    const float amax = hi > 1e-10f || hi != hi ? hi : 1e-10f;
    o.scale = amax / 127.0f;
    o.mul = 127.0f / amax;
  }
  return o;
}

// A head belongs to 2^lanes_log2 lanes, each with K units of two pieces of V values.  The pieces of a unit lie half a stretch apart, a
// stretch being the rotated part, the part behind it, or 128 values with a scale of their own: so both values of a pair are in
// one lane, half to half or side by side, and neighbouring lanes load and store neighbouring pieces.  A lane group takes up to
// HEADS heads of one token, loads them all before it waits for the first and uses the table's row and the weights for all of them.
template <typename T, int V, int K, int HEADS, bool ADJACENT, bool AXES, bool NORM>
__global__ __launch_bounds__(256, V == 8 && HEADS == 1 ? 8 : 1) void head_rows_kernel(const HeadArgs a) {
  constexpr bool PAIRS_IN_PIECES = ADJACENT && V > 1;
  constexpr int GROUP_UNITS = 64 / V, GROUP_LOG2 = V == 8 ? 3 : V == 4 ? 4 : 6;
  touch_arguments(a);
  const uint32_t block = blockIdx.x;
  const int index = (block >= a.first_block[1]) + (block >= a.first_block[2]);
  const HeadPart& p = a.part[index];
  const int lanes_log2 = p.lanes_log2;
  const uint32_t group = ((block - a.first_block[index]) << (8 - lanes_log2)) + (threadIdx.x >> lanes_log2);
  if (group >= p.groups) return;
  const int per_token = p.per_token, units = p.units, rot_units = p.rot_units, kind = p.kind, heads = p.heads;
  const uint32_t token = p.per_token_div.divide(group);
  const int first_head = (int)(group - token * (uint32_t)per_token), lane = threadIdx.x & ((1 << lanes_log2) - 1);

  // where a lane's pieces lie in a head
  int at0[K], at1[K];
  bool rotated[K], real[K];
#pragma unroll
  for (int j = 0; j < K; j++) {
    const int wanted = lane + (j << lanes_log2), u = min(wanted, units - 1);
    real[j] = wanted < units;
    rotated[j] = u < rot_units;
    if (ADJACENT && V == 1 && rotated[j]) {
      at0[j] = 2 * u;
      at1[j] = at0[j] + 1;
    } else if (p.grouped) {
      at0[j] = ((u >> GROUP_LOG2) << 7) + (u & (GROUP_UNITS - 1)) * V;
      at1[j] = at0[j] + 64;
    } else {
      at0[j] = (rotated[j] ? u : u + rot_units) * V;
      at1[j] = at0[j] + (rotated[j] ? rot_units : units - rot_units) * V;
    }
  }

  // Positions first: the table's rows hang on them.  Then the heads, all at once and without a condition (lanes and heads that are
  // none read the last one), so that neither waits for the other.
  AxisBits axes0[K] = {}, axes1[K] = {};
  Index pos[AXES ? 4 : 1] = {}, slot_index = {};
  if (rot_units) {
#pragma unroll
    for (int k = 0; k < (AXES ? 4 : 1); k++)
      pos[k] = load_index(a.positions, (AXES ? min(k, a.axes - 1) * a.axis_stride : 0) + (int64_t)token * a.position_stride, a.positions_are_i64);
    if constexpr (AXES) {
#pragma unroll
      for (int j = 0; j < K; j++) {
        if (!rotated[j]) continue;
        if (PAIRS_IN_PIECES) axes0[j] = axes_of_pairs<V / 2 + (V == 1)>(a, at0[j] / 2), axes1[j] = axes_of_pairs<V / 2 + (V == 1)>(a, at1[j] / 2);
        else axes0[j] = axes_of_pairs<V>(a, ADJACENT ? at0[j] / 2 : at0[j]);
      }
    }
  }
  if (kind != HEADS_TO_NONE) slot_index = load_index(a.slots, (int64_t)token * a.slot_stride, a.slots_are_i64);

  typename Piece<V>::type raw0[HEADS][K], raw1[HEADS][K];
  const u16* x = p.x + (int64_t)token * p.x_token + first_head * p.x_head;
  const int64_t x_step = per_token * p.x_head;
#pragma unroll
  for (int h = 0; h < HEADS; h++) {
#pragma unroll
    for (int j = 0; j < K; j++) {
      raw0[h][j] = load_values<V>(x + at0[j]);
      raw1[h][j] = load_values<V>(x + at1[j]);
    }
    x += first_head + (h + 1) * per_token < heads ? x_step : 0;
  }

  float c[K][V], s[K][V];
  if (rot_units) {
    uint32_t table_row[AXES ? 4 : 1];
    bool inside[AXES ? 4 : 1];
#pragma unroll
    for (int k = 0; k < (AXES ? 4 : 1); k++) {
      const int64_t v = pos[k].value(a.positions_are_i64);
      inside[k] = (uint64_t)v < (uint64_t)a.table_rows;
      table_row[k] = inside[k] ? (uint32_t)v * (uint32_t)(a.table_stride * (a.table_is_f32 ? 4 : 2)) : 0;
    }
#pragma unroll
    for (int j = 0; j < K; j++) {
      if (!rotated[j]) continue;
      if constexpr (PAIRS_IN_PIECES) {
        load_turn<T, V / 2, AXES>(a, table_row, inside, axes0[j], at0[j] / 2, c[j], s[j]);
        load_turn<T, V / 2, AXES>(a, table_row, inside, axes1[j], at1[j] / 2, c[j] + V / 2, s[j] + V / 2);
      } else {
        load_turn<T, V, AXES>(a, table_row, inside, axes0[j], ADJACENT ? at0[j] / 2 : at0[j], c[j], s[j]);
      }
    }
  }
  typename Piece<V>::type raw_w0[K] = {}, raw_w1[K] = {};
  if (NORM && p.w && !p.w_is_f32) {
#pragma unroll
    for (int j = 0; j < K; j++) {
      raw_w0[j] = load_values<V>((const u16*)((const char*)p.w + (uint32_t)(2 * at0[j])));
      raw_w1[j] = load_values<V>((const u16*)((const char*)p.w + (uint32_t)(2 * at1[j])));
    }
  }
  uint32_t slot = ~0u;
  if (kind != HEADS_TO_NONE) {
    const int64_t wide = slot_index.value(a.slots_are_i64);
    slot = (uint64_t)wide < (uint64_t)a.num_slots ? (uint32_t)wide : ~0u;  // (a negative slot is padding)
  }

#pragma unroll
  for (int h = 0; h < HEADS; h++) {
    const int head = first_head + h * per_token;
    if (head >= heads) return;
    if (HEADS > 1) __builtin_amdgcn_sched_barrier(0);  // (heads side by side would not fit the registers)
    float f0[K][V], f1[K][V];
#pragma unroll
    for (int j = 0; j < K; j++) {
      to_floats<T, V>(raw0[h][j], f0[j]);
      to_floats<T, V>(raw1[h][j], f1[j]);
    }
    if constexpr (NORM) {
      float r = 1.f;
      if (p.w) {
        float sum = 0.f;
#pragma unroll
        for (int j = 0; j < K; j++)
#pragma unroll
          for (int i = 0; i < V; i++) {
            const float x0 = K == 1 || real[j] ? f0[j][i] : 0.f, x1 = K == 1 || real[j] ? f1[j][i] : 0.f;
            sum = fmaf(x0, x0, fmaf(x1, x1, sum));
          }
        if (K == 1 && !real[0]) sum = 0.f;
        sum = group_sum(sum, lanes_log2);
        // (a sum beyond fp32 would give zeros)
        r = sum < INFINITY ? rsqrtf(fmaf(sum, p.inv_dim, p.eps)) : NAN;
      }
      // heads of a part without a weight are multiplied by ones: no second copy of the registers
#pragma unroll
      for (int j = 0; j < K; j++) {
        float w[V];
        weights<T, V>(p, at0[j], raw_w0[j], w);
#pragma unroll
        for (int i = 0; i < V; i++) f0[j][i] = f0[j][i] * r * w[i];
        pin<V>(f0[j]);
        weights<T, V>(p, at1[j], raw_w1[j], w);
#pragma unroll
        for (int i = 0; i < V; i++) f1[j][i] = f1[j][i] * r * w[i];
        pin<V>(f1[j]);
      }
    }
#pragma unroll
    for (int j = 0; j < K; j++)
      if (rotated[j]) turn<V, ADJACENT>(f0[j], f1[j], c[j], s[j]);

    if (p.out) {
      u16* const out = p.out + (int64_t)token * p.out_token + head * p.out_head;
#pragma unroll
      for (int j = 0; j < K; j++)
        if (real[j]) {
          store_values<T, V>(out + at0[j], f0[j]);
          store_values<T, V>(out + at1[j], f1[j]);
        }
    }
    if (kind == HEADS_TO_NONE || slot == ~0u) continue;
    const uint32_t page = a.page_div.divide(slot), in_page = slot - page * (uint32_t)a.page_size;
    uint8_t* const row = p.cache + page * p.cache_page + in_page * p.cache_slot + head * p.cache_head;
    if (kind == HEADS_TO_16) {
#pragma unroll
      for (int j = 0; j < K; j++)
        if (real[j]) {
          store_values<T, V>((u16*)row + at0[j], f0[j]);
          store_values<T, V>((u16*)row + at1[j], f1[j]);
        }
      continue;
    }
    uint32_t hi[K];
    if (!p.given) {
      uint32_t whole = 0;
#pragma unroll
      for (int j = 0; j < K; j++) {
        hi[j] = 0;
#pragma unroll
        for (int i = 0; i < V; i++) {
          hi[j] = umax(hi[j], __float_as_uint(f0[j][i]) & 0x7fffffffu);
          hi[j] = umax(hi[j], __float_as_uint(f1[j][i]) & 0x7fffffffu);
        }
        if (!real[j]) hi[j] = 0;
        whole = umax(whole, hi[j]);
      }
      if (!p.grouped) whole = group_umax(whole, lanes_log2);
#pragma unroll
      for (int j = 0; j < K; j++) hi[j] = p.grouped ? group_umax(hi[j], GROUP_LOG2) : whole;
    }
#pragma unroll
    for (int j = 0; j < K; j++) {
      if (!real[j]) continue;
      RowScale o = {};
      if (p.given) {
        o.mul = fp8_row_multiplier(1.0f, p.given[head * p.given_head]);
      } else {
        o = kind == HEADS_TO_FP8 ? found_scale<ROW_TO_FP8>(hi[j]) : found_scale<ROW_TO_INT8>(hi[j]);
        const int u = lane + (j << lanes_log2), n = p.grouped ? u >> GROUP_LOG2 : 0;
        if (u == n << GROUP_LOG2)
          p.scales[page * p.scales_page + in_page * p.scales_slot + head * p.scales_head + n * p.scales_group] = o.scale;
      }
      if (kind == HEADS_TO_FP8) {
        store_codes<ROW_TO_FP8, V>(row + at0[j], f0[j], o);
        store_codes<ROW_TO_FP8, V>(row + at1[j], f1[j], o);
      } else {
        store_codes<ROW_TO_INT8, V>(row + at0[j], f0[j], o);
        store_codes<ROW_TO_INT8, V>(row + at1[j], f1[j], o);
      }
    }
  }
}

// ---------------------------------------------------------------------------------------
// rows of a paged cache back in 16 bits
// ---------------------------------------------------------------------------------------
struct GatherPart {
  const uint8_t* cache;  // strides in bytes
  int64_t cache_page, cache_slot, cache_head;
  const float* given;
  const float* scales;
  int64_t given_head, scales_page, scales_slot, scales_head, scales_group;
  u16* out;
  int64_t out_row, out_head;
  uint32_t first_block, units;  // units of V values: rows * heads * per_head
  FastDiv per_row_div, per_head_div;
  int per_row, per_head;
  int kind, group_units_log2;  // units per scale of a row, 31: the whole row
};
struct GatherArgs {
  GatherPart part[2];
  int parts, slots_are_i64, page_size;
  const void* slots;
  int64_t slot_stride, num_slots;
  FastDiv page_div;
};

template <int V>
struct Bytes {
  uint8_t v[V];
};

// A lane takes UNITS units of V values, 256 units apart.  The slots of all of them are asked for first, then the rows without a
// condition (where there is no slot, those of slot 0): two round trips, whatever UNITS.  Pieces of eight values, not sixteen: stores
// of 16 bytes beside each other (65000 int8 rows of 2 x 8 x 128: 80 us, a copy of as much 80; sixteen 95).
template <typename T, int V, int UNITS>
__global__ __launch_bounds__(256) void gather_rows_kernel(const GatherArgs a) {
  touch_arguments(a);
  const int index = a.parts > 1 && blockIdx.x >= a.part[1].first_block;
  const GatherPart& p = a.part[index];
  const uint32_t base = (blockIdx.x - p.first_block) * (256 * UNITS) + threadIdx.x;
  uint32_t row[UNITS], head[UNITS], unit[UNITS];
  Index slot_index[UNITS];
#pragma unroll
  for (int k = 0; k < UNITS; k++) {
    const uint32_t i = min(base + 256 * k, p.units - 1);  // (lanes and units that are none read the last one)
    row[k] = p.per_row_div.divide(i);
    const uint32_t in_row = i - row[k] * (uint32_t)p.per_row;
    head[k] = p.per_head_div.divide(in_row);
    unit[k] = in_row - head[k] * (uint32_t)p.per_head;
    slot_index[k] = load_index(a.slots, (int64_t)row[k] * a.slot_stride, a.slots_are_i64);
  }
  Bytes<V> codes[UNITS] = {};
  typename Piece<V>::type values[UNITS];
  float scale[UNITS] = {};
  bool inside[UNITS];
#pragma unroll
  for (int k = 0; k < UNITS; k++) {
    const int64_t wide = slot_index[k].value(a.slots_are_i64);
    inside[k] = (uint64_t)wide < (uint64_t)a.num_slots;
    const uint32_t slot = inside[k] ? (uint32_t)wide : 0;
    const uint32_t page = a.page_div.divide(slot), in_page = slot - page * (uint32_t)a.page_size;
    const uint8_t* src = p.cache + page * p.cache_page + in_page * p.cache_slot + head[k] * p.cache_head;
    values[k] = 0;
    if (a.num_slots == 0) continue;
    if (p.kind == HEADS_TO_16) {
      values[k] = load_values<V>((const u16*)src + unit[k] * V);
    } else {
      __builtin_memcpy(&codes[k], src + unit[k] * V, V);
      scale[k] = p.given ? p.given[head[k] * p.given_head]
                         : p.scales[page * p.scales_page + in_page * p.scales_slot + head[k] * p.scales_head +
                                    (unit[k] >> p.group_units_log2) * p.scales_group];
    }
  }
#pragma unroll
  for (int k = 0; k < UNITS; k++) {
    if (base + 256 * k >= p.units) return;
    u16* out = p.out + (int64_t)row[k] * p.out_row + head[k] * p.out_head + unit[k] * V;
    if (p.kind == HEADS_TO_16 || !inside[k]) {
      if (!inside[k]) values[k] = 0;
      __builtin_memcpy(out, &values[k], 2 * V);  // (one value: the low half)
      continue;
    }
    float f[V];
    if (p.kind == HEADS_TO_FP8) {
      if constexpr (V == 1) {
        f[0] = __builtin_amdgcn_cvt_f32_fp8(codes[k].v[0], 0) * scale[k];
      } else {
        typedef float v2f __attribute__((ext_vector_type(2)));
        uint32_t w[V / 4];
        __builtin_memcpy(w, &codes[k], V);
#pragma unroll
        for (int i = 0; i < V / 4; i++) {
          const v2f lo = __builtin_amdgcn_cvt_pk_f32_fp8(w[i], false), hi = __builtin_amdgcn_cvt_pk_f32_fp8(w[i], true);
          f[4 * i] = lo[0] * scale[k], f[4 * i + 1] = lo[1] * scale[k];
          f[4 * i + 2] = hi[0] * scale[k], f[4 * i + 3] = hi[1] * scale[k];
        }
      }
    } else {
#pragma unroll
      for (int i = 0; i < V; i++) f[i] = (float)(int8_t)codes[k].v[i] * scale[k];
    }
    store_values<T, V>(out, f);
  }
}

}  // namespace sglamd

using namespace sglamd;

static int check_slots(const char* op, const sglamd_slots* s) {
  SGLAMD_REQUIRE(s && s->slots, SGLAMD_EINVAL, "%s: a cache needs slots", op);
  SGLAMD_REQUIRE(s->slots_dtype == SGLAMD_I32 || s->slots_dtype == SGLAMD_I64, SGLAMD_EINVAL, "%s: slots must be I32 or I64", op);
  SGLAMD_REQUIRE(s->page_size > 0 && s->pages >= 0 && s->page_size < (1ll << 31) && s->pages < (1ll << 31) && s->page_size * s->pages < (1ll << 31),
                 SGLAMD_EINVAL, "%s: %lld pages of %lld slots: fewer than 2^31 slots are served", op, (long long)s->pages, (long long)s->page_size);
  return SGLAMD_OK;
}

static int cache_kind(const char* op, int cache_dtype, int dtype, const void* given, const void* scales, int* kind) {
  if (cache_dtype == dtype) {
    SGLAMD_REQUIRE(!given && !scales, SGLAMD_EINVAL, "%s: a 16-bit cache has no scales", op);
    *kind = HEADS_TO_16;
    return SGLAMD_OK;
  }
  SGLAMD_REQUIRE(cache_dtype == SGLAMD_FP8_E4M3 || cache_dtype == SGLAMD_I8, SGLAMD_EINVAL,
                 "%s: a cache is of the activations' type, Float8_e4m3fn or Char", op);
  SGLAMD_REQUIRE(!given != !scales, SGLAMD_EINVAL, "%s: an 8-bit cache has either one given scale or scales of its rows", op);
  *kind = cache_dtype == SGLAMD_FP8_E4M3 ? HEADS_TO_FP8 : HEADS_TO_INT8;
  return SGLAMD_OK;
}

static int log2_up(int64_t n) {
  int log = 0;
  while ((1ll << log) < n) log++;
  return log;
}

template <typename T, int V, int K, int HEADS, bool AXES, bool NORM>
static void launch_heads(const HeadArgs& a, unsigned blocks, bool adjacent, hipStream_t st) {
  if (adjacent) hipLaunchKernelGGL((head_rows_kernel<T, V, K, HEADS, true, AXES, NORM>), dim3(blocks), dim3(256), 0, st, a);
  else hipLaunchKernelGGL((head_rows_kernel<T, V, K, HEADS, false, AXES, NORM>), dim3(blocks), dim3(256), 0, st, a);
}
template <typename T, int HEADS, bool AXES>
static void launch_heads_of_8(const HeadArgs& a, unsigned blocks, bool adjacent, bool norm, hipStream_t st) {
  if (norm) launch_heads<T, 8, 1, HEADS, AXES, true>(a, blocks, adjacent, st);
  else launch_heads<T, 8, 1, HEADS, AXES, false>(a, blocks, adjacent, st);
}

// How many heads of a token a lane group takes where it has to find its cosines pair by pair.
constexpr int HEADS_MANY = 2;
// ... and where its pieces are of four values.
constexpr int HEADS_OF_FOURS = 4;

extern "C" int sglamd_head_rows(const sglamd_heads* parts, int num_parts, int64_t tokens, int dtype, const sglamd_rotation* rotation,
                                const sglamd_slots* slots, void* stream) {
  const char* op = "head_rows";
  SGLAMD_REQUIRE(parts && num_parts > 0 && num_parts <= MAX_PARTS, SGLAMD_EINVAL, "%s: one to %d tensors of heads", op, MAX_PARTS);
  SGLAMD_REQUIRE(dtype == SGLAMD_BF16 || dtype == SGLAMD_F16, SGLAMD_EINVAL, "%s: heads must be Half or BFloat16", op);
  SGLAMD_REQUIRE(tokens >= 0 && tokens < (1ll << 31), SGLAMD_EINVAL, "%s: bad token count %lld", op, (long long)tokens);
  HeadArgs a = {};
  int64_t width = 0;  // of the rotated part
  bool norm = false;
  for (int i = 0; i < num_parts; i++) {
    norm = norm || parts[i].weight;
    if (parts[i].rotate) {
      SGLAMD_REQUIRE(rotation, SGLAMD_EINVAL, "%s: a rotation without its table", op);
      width = rotation->width;
    }
  }
  if (width || rotation) {
    const sglamd_rotation& r = *rotation;
    width = r.width;
    SGLAMD_REQUIRE(r.cos_sin && r.positions, SGLAMD_EINVAL, "%s: null table or positions", op);
    SGLAMD_REQUIRE(r.table_dtype == SGLAMD_F32 || r.table_dtype == dtype, SGLAMD_EINVAL, "%s: the table must be Float or of the heads' type", op);
    SGLAMD_REQUIRE(r.positions_dtype == SGLAMD_I32 || r.positions_dtype == SGLAMD_I64, SGLAMD_EINVAL, "%s: positions must be I32 or I64", op);
    SGLAMD_REQUIRE(r.width > 0 && r.width % 2 == 0 && r.width <= 1024, SGLAMD_EINVAL, "%s: a rotated width of %lld: even, 2 to 1024", op,
                   (long long)r.width);
    const int64_t stride = r.table_rows > 1 ? r.table_stride : 0;
    SGLAMD_REQUIRE(r.table_rows > 0 && r.table_rows < (1ll << 31) && stride >= 0 && stride < (1ll << 31) &&
                       (r.table_rows - 1) * stride + r.width <= (1ll << (r.table_dtype == SGLAMD_F32 ? 29 : 30)),
                   SGLAMD_EINVAL, "%s: a table of %lld positions: one to 2 GiB are served", op, (long long)r.table_rows);
    SGLAMD_REQUIRE(r.axes >= 1 && r.axes <= 4, SGLAMD_EINVAL, "%s: one to four position axes", op);
    a.table = r.cos_sin, a.table_stride = stride, a.table_rows = r.table_rows, a.table_is_f32 = r.table_dtype == SGLAMD_F32;
    a.positions = r.positions, a.positions_are_i64 = r.positions_dtype == SGLAMD_I64;
    a.axis_stride = r.axis_stride, a.position_stride = r.position_stride;
    a.pairs = (int)(r.width / 2), a.axes = r.axes;
    if (r.axes > 1) {
      int64_t sum = 0, past[4];  // past[k]: behind the last pair of axis k
      for (int k = 0; k < r.axes; k++) {
        SGLAMD_REQUIRE(r.sections[k] >= 0, SGLAMD_EINVAL, "%s: a section is negative", op);
        sum += r.sections[k];
        past[k] = r.alternating ? (int64_t)r.axes * r.sections[k] : sum;
        // (the pairs that the rule leaves to axis 0 beyond its own turns have to be as many as its section says)
        SGLAMD_REQUIRE(!r.alternating || k == 0 || r.sections[k] == 0 || k + (int64_t)r.axes * (r.sections[k] - 1) < a.pairs, SGLAMD_EINVAL,
                       "%s: alternating sections: axis %d has no %d turns in %d pairs", op, k, (int)r.sections[k], a.pairs);
      }
      SGLAMD_REQUIRE(sum == a.pairs, SGLAMD_EINVAL, "%s: sections of %lld pairs for a rotated width of %lld", op, (long long)sum, (long long)r.width);
      for (int i = 0; i < a.pairs; i++) {
        int k = 0;
        if (r.alternating) k = i < past[i % r.axes] ? i % r.axes : 0;
        else while (i >= past[k]) k++;
        a.axis_bits[0][i / 32] |= (uint32_t)(k & 1) << (i % 32);
        a.axis_bits[1][i / 32] |= (uint32_t)(k >> 1) << (i % 32);
      }
    }
  }
  if (slots) {
    const int rc = check_slots(op, slots);
    if (rc) return rc;
    a.slots = slots->slots, a.slot_stride = slots->slot_stride, a.slots_are_i64 = slots->slots_dtype == SGLAMD_I64;
    a.num_slots = slots->page_size * slots->pages, a.page_size = (int)slots->page_size, a.page_div = FastDiv::of((uint32_t)slots->page_size);
  }

  // values per piece: 8, or what divides every head and its rotated part
  int v = 8;
  for (int i = 0; i < num_parts; i++) {
    const sglamd_heads& h = parts[i];
    SGLAMD_REQUIRE(h.heads >= 0 && h.heads < (1 << 20) && h.dim > 0 && h.dim <= 1024 && h.dim % 2 == 0, SGLAMD_EINVAL,
                   "%s: %lld heads of %lld values: even sizes up to 1024 are served", op, (long long)h.heads, (long long)h.dim);
    SGLAMD_REQUIRE(!h.rotate || width <= h.dim, SGLAMD_EINVAL, "%s: a rotated width of %lld in heads of %lld", op, (long long)width, (long long)h.dim);
    while (v > 1 && (h.dim % (2 * v) || (h.rotate && width % (2 * v)))) v /= 2;
  }
  if (v == 2) v = 1;
  for (int i = 0; i < num_parts; i++)
    if (v == 4 && parts[i].dim > 512) v = 1;
  const int k = v == 1 ? 8 : 1;

  // One head per lane group: 57 to 64 registers, eight waves a SIMD, and the most loads in flight (8191 tokens of 64 + 2 x 8 heads
  // of 128 into e4m3 rows: 59.9 us, two heads 62.3, four 66.1).  With several axes a lane may need sixteen loads for its pairs, which
  // two heads share from 1024 lanes a CU on, half of what it holds.  One | two | four heads, us in a graph, tokens x heads of 128:
  //   alternating     256 x 32  4.1 | 4.4 | 5.3    768 x 32  6.8 | 6.3 | 6.2    1024 x 32  8.5 | 7.3 | 7.2    2901 x 32  15.9 | 13.1 | 12.2
  //   with a norm     256 x 32  4.6 | 5.2 | 6.8    768 x 32  7.4 | 7.3 | 7.7    1024 x 32  9.1 | 8.2 | 8.7    4096 x 72  42.1 | 36.7 | 36.5
  //   blocks of axes  256 x 32  3.4 | 3.8 | 4.4   1024 x 32  5.6 | 5.8 | 6.2    2901 x 32  10.5 | 10.3 | 10.3   4096 x 72  34.5 | 33.2 | 35.5
  // Two for both kinds of sections, one rule: four would be 7 to 9 % faster for 2901 tokens of 32 heads and more where axes alternate,
  // and is no faster for 72 heads; one up to 5 % faster for blocks of axes at 1024 to 2901 tokens of 32.
  int64_t lanes = 0;
  for (int i = 0; i < num_parts; i++) lanes += tokens * parts[i].heads << log2_up(ceil_div(parts[i].dim, 2 * v * k));
  // Pieces of four: the lanes' addresses are most of the work, four heads share them (4096 tokens of 72 heads of 72, normalised:
  // 27.2 us, two heads 30.6, eight 30.7, one 38.7; 500 of 80 heads of 72 into e4m3 rows: four 7.6, two 6.1, one 7.2).
  const DeviceScope scope;
  const int64_t cus = device_cus();
  const int many = v == 4 && lanes >= cus * 4096 ? HEADS_OF_FOURS : v == 8 && a.axes > 1 && lanes >= cus * 1024 ? HEADS_MANY : 1;

  uint64_t blocks = 0;
  for (int i = 0; i < num_parts; i++) {
    const sglamd_heads& h = parts[i];
    HeadPart& p = a.part[i];
    SGLAMD_REQUIRE(h.x || tokens == 0 || h.heads == 0, SGLAMD_EINVAL, "%s: null heads", op);
    SGLAMD_REQUIRE(h.out || h.cache, SGLAMD_EINVAL, "%s: heads that go nowhere", op);
    SGLAMD_REQUIRE(h.x_token >= 0 && h.x_head >= 0, SGLAMD_EINVAL, "%s: negative strides", op);
    SGLAMD_REQUIRE(!h.weight || h.weight_dtype == SGLAMD_F32 || h.weight_dtype == dtype, SGLAMD_EINVAL,
                   "%s: a norm weight must be Float or of the heads' type", op);
    SGLAMD_REQUIRE(!h.weight || (h.eps >= 0.f && h.eps < INFINITY), SGLAMD_EINVAL, "%s: epsilon must be finite and not negative", op);
    p.x = (const u16*)h.x, p.x_token = h.x_token, p.x_head = h.x_head;
    p.w = h.weight, p.w_is_f32 = h.weight && h.weight_dtype == SGLAMD_F32, p.eps = h.eps, p.inv_dim = 1.0f / (float)h.dim;
    p.out = (u16*)h.out, p.out_token = h.out_token, p.out_head = h.out_head;
    p.heads = (int)h.heads, p.units = (int)(h.dim / (2 * v)), p.rot_units = h.rotate ? (int)(width / (2 * v)) : 0;
    p.lanes_log2 = log2_up(ceil_div(p.units, k));
    if (h.cache) {
      SGLAMD_REQUIRE(slots, SGLAMD_EINVAL, "%s: a cache needs slots", op);
      const int rc = cache_kind(op, h.cache_dtype, dtype, h.given_scale, h.scales, &p.kind);
      if (rc) return rc;
      SGLAMD_REQUIRE(p.kind != HEADS_TO_INT8 || h.scales, SGLAMD_EINVAL, "%s: Char rows have scales of their own", op);
      const int64_t bytes = p.kind == HEADS_TO_16 ? 2 : 1;
      p.cache = (uint8_t*)h.cache, p.cache_page = h.cache_page * bytes, p.cache_slot = h.cache_slot * bytes, p.cache_head = h.cache_head * bytes;
      p.given = h.given_scale, p.given_head = h.given_head, p.scales = h.scales;
      p.scales_page = h.scales_page, p.scales_slot = h.scales_slot, p.scales_head = h.scales_head, p.scales_group = h.scales_group;
      if (h.scales && h.scale_group != h.dim) {
        SGLAMD_REQUIRE(h.scale_group == 128 && h.dim % 128 == 0 && !h.rotate, SGLAMD_EINVAL,
                       "%s: a scale per row, or per 128 values of rows that are not rotated and a multiple of 128 long", op);
        p.grouped = 1;
        if (k > 1) p.lanes_log2 = 6;  // a round of the wave's lanes is one scale
      }
    }
    p.per_token = (int)ceil_div(h.heads, many);
    const uint64_t groups = (uint64_t)tokens * (uint64_t)p.per_token;
    SGLAMD_REQUIRE(groups << p.lanes_log2 < (1ull << 31), SGLAMD_EINVAL, "%s: %lld tokens of %lld heads are too many for one launch", op,
                   (long long)tokens, (long long)h.heads);
    p.groups = (uint32_t)groups, p.per_token_div = FastDiv::of((uint32_t)(p.per_token ? p.per_token : 1));
    a.first_block[i] = (uint32_t)blocks;
    blocks += ((groups << p.lanes_log2) + 255) / 256;
  }
  for (int i = num_parts; i < MAX_PARTS; i++) a.first_block[i] = ~0u;
  if (blocks == 0) return SGLAMD_OK;
  SGLAMD_REQUIRE(blocks < (1ull << 24), SGLAMD_EINVAL, "%s: %lld tokens are too many for one launch", op, (long long)tokens);
  const bool adjacent = rotation && rotation->interleaved;
  hipStream_t st = (hipStream_t)stream;
#define SGLAMD_HEADS(T)                                                                       \
  do {                                                                                        \
    if (v == 8 && many > 1) launch_heads_of_8<T, HEADS_MANY, true>(a, (unsigned)blocks, adjacent, norm, st); \
    else if (v == 8 && a.axes > 1) launch_heads_of_8<T, 1, true>(a, (unsigned)blocks, adjacent, norm, st);   \
    else if (v == 8) launch_heads_of_8<T, 1, false>(a, (unsigned)blocks, adjacent, norm, st);                \
    else if (v == 4 && many > 1) launch_heads<T, 4, 1, HEADS_OF_FOURS, true, true>(a, (unsigned)blocks, adjacent, st); \
    else if (v == 4) launch_heads<T, 4, 1, 1, true, true>(a, (unsigned)blocks, adjacent, st);                    \
    else launch_heads<T, 1, 8, 1, true, true>(a, (unsigned)blocks, adjacent, st);             \
  } while (0)
  if (dtype == SGLAMD_BF16) SGLAMD_HEADS(BF16);
  else SGLAMD_HEADS(F16);
#undef SGLAMD_HEADS
  return check_launch(op);
}

template <typename T, int V>
static void launch_gather(const GatherArgs& a, unsigned blocks, int per_lane, hipStream_t st) {
  if (per_lane == 4) hipLaunchKernelGGL((gather_rows_kernel<T, V, 4>), dim3(blocks), dim3(256), 0, st, a);
  else hipLaunchKernelGGL((gather_rows_kernel<T, V, 1>), dim3(blocks), dim3(256), 0, st, a);
}

extern "C" int sglamd_gather_head_rows(const sglamd_gather* parts, int num_parts, int64_t rows, int dtype, const sglamd_slots* slots, void* stream) {
  const char* op = "gather_head_rows";
  SGLAMD_REQUIRE(parts && (num_parts == 1 || num_parts == 2), SGLAMD_EINVAL, "%s: one or two caches", op);
  SGLAMD_REQUIRE(dtype == SGLAMD_BF16 || dtype == SGLAMD_F16, SGLAMD_EINVAL, "%s: rows come back as Half or BFloat16", op);
  SGLAMD_REQUIRE(rows >= 0 && rows < (1ll << 31), SGLAMD_EINVAL, "%s: bad row count %lld", op, (long long)rows);
  if (rows == 0) return SGLAMD_OK;
  int rc = check_slots(op, slots);
  if (rc) return rc;
  GatherArgs a = {};
  a.parts = num_parts, a.slots = slots->slots, a.slot_stride = slots->slot_stride, a.slots_are_i64 = slots->slots_dtype == SGLAMD_I64;
  a.num_slots = slots->page_size * slots->pages, a.page_size = (int)slots->page_size, a.page_div = FastDiv::of((uint32_t)slots->page_size);
  int v = 8;
  for (int i = 0; i < num_parts; i++) {
    const sglamd_gather& g = parts[i];
    SGLAMD_REQUIRE(g.heads >= 0 && g.heads < (1 << 20) && g.dim > 0 && g.dim <= 1024, SGLAMD_EINVAL, "%s: %lld heads of %lld values: up to 1024", op,
                   (long long)g.heads, (long long)g.dim);
    while (v > 1 && g.dim % v) v /= 2;
  }
  if (v == 2) v = 1;
  // Four units a lane once one each fills the chip several times over (int8 rows of 2 x 8 x 128, one | four: 500 of them 2.6 | 4.0 us,
  // 10000 13.5 | 13.7, 20000 30.6 | 28.4, 65000 92.9 | 80.6).
  const DeviceScope scope;
  int64_t all = 0;
  for (int i = 0; i < num_parts; i++) all += rows * parts[i].heads * (parts[i].dim / v);
  const int per_lane = all > (int64_t)device_cus() * 16384 ? 4 : 1;
  uint64_t blocks = 0;
  for (int i = 0; i < num_parts; i++) {
    const sglamd_gather& g = parts[i];
    GatherPart& p = a.part[i];
    SGLAMD_REQUIRE(g.cache && g.out, SGLAMD_EINVAL, "%s: null cache or output", op);
    rc = cache_kind(op, g.cache_dtype, dtype, g.given_scale, g.scales, &p.kind);
    if (rc) return rc;
    SGLAMD_REQUIRE(p.kind != HEADS_TO_INT8 || g.scales, SGLAMD_EINVAL, "%s: Char rows have scales of their own", op);
    SGLAMD_REQUIRE(!g.scales || g.scale_group == g.dim || (g.scale_group == 128 && g.dim % 128 == 0), SGLAMD_EINVAL,
                   "%s: a scale per row, or per 128 values", op);
    const int64_t bytes = p.kind == HEADS_TO_16 ? 2 : 1;
    p.cache = (const uint8_t*)g.cache, p.cache_page = g.cache_page * bytes, p.cache_slot = g.cache_slot * bytes, p.cache_head = g.cache_head * bytes;
    p.given = g.given_scale, p.given_head = g.given_head, p.scales = g.scales;
    p.scales_page = g.scales_page, p.scales_slot = g.scales_slot, p.scales_head = g.scales_head, p.scales_group = g.scales_group;
    p.group_units_log2 = g.scales && g.scale_group != g.dim ? log2_up(128 / v) : 31;
    p.out = (u16*)g.out, p.out_row = g.out_row, p.out_head = g.out_head;
    p.per_head = (int)(g.dim / v), p.per_row = p.per_head * (int)g.heads;
    const uint64_t units = (uint64_t)rows * (uint64_t)p.per_row;
    SGLAMD_REQUIRE((uint64_t)g.heads * (uint64_t)p.per_head < (1ull << 31) && units < (1ull << 31) - 1024, SGLAMD_EINVAL,
                   "%s: %lld rows are too many for one launch", op, (long long)rows);
    p.units = (uint32_t)units, p.per_row_div = FastDiv::of((uint32_t)(p.per_row ? p.per_row : 1)), p.per_head_div = FastDiv::of((uint32_t)p.per_head);
    p.first_block = (uint32_t)blocks;
    blocks += (units + 256 * per_lane - 1) / (256 * per_lane);
  }
  if (blocks == 0) return SGLAMD_OK;
  hipStream_t st = (hipStream_t)stream;
#define SGLAMD_GATHER(T)                                                       \
  do {                                                                         \
    if (v == 8) launch_gather<T, 8>(a, (unsigned)blocks, per_lane, st);        \
    else if (v == 4) launch_gather<T, 4>(a, (unsigned)blocks, per_lane, st);   \
    else launch_gather<T, 1>(a, (unsigned)blocks, per_lane, st);               \
  } while (0)
  if (dtype == SGLAMD_BF16) SGLAMD_GATHER(BF16);
  else SGLAMD_GATHER(F16);
#undef SGLAMD_GATHER
  return check_launch(op);
}
