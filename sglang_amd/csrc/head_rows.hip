// Heads of queries, keys and values between a projection and its attention: RMSNorm of each head, rotary positions, rows of a
// paged cache in 16 or 8 bits, and such rows back in 16 bits.
//
//   norm    y = x * r * w,  r = 1 / sqrt(mean(x^2) + eps) over one head
//   rotate  pair i of a token on position p: (a, b) -> (a c - b s, b c + a s), c = table[p][i], s = table[p][i + pairs]
//   codes   those of row_out.h: e4m3 with scale = max|y| / 448 or as given, int8 with scale = max(max|y|, 1e-10) / 127
//
// Everything between the load of a head and its stores is in fp32 and rounded once, to the type of the row that is written.
//
// All of it is bound by HBM at prompt sizes (a few operations per value, each value read once and written once) and by the
// launch at decode sizes, so the aim is one launch for everything that a layer does between its projection and its attention.
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
  float* scales;       // scales that are found here, one per `scale_units` units of a row
  int64_t given_head, scales_page, scales_slot, scales_head, scales_group;
  float eps, inv_dim;
  uint32_t first_block, groups;  // lane groups of this part: tokens * per_token
  FastDiv per_token_div;
  int per_token, heads, units, rot_units;
  int lanes_log2, scale_lanes_log2, scale_units;
  int kind, w_is_f32;
};

constexpr int MAX_PARTS = 4;

struct HeadArgs {
  HeadPart part[MAX_PARTS];
  int parts;
  // rotation
  const void* table;
  int64_t table_stride, table_rows, axis_stride, position_stride;
  const void* positions;
  int pairs, table_is_f32, positions_are_i64, axes, alternating;
  int section[4], axis_inv;  // blocks: where axes 1, 2 and 3 begin; alternating: pairs of each axis, 65536 / axes rounded up
  // slots
  const void* slots;
  int64_t slot_stride, num_slots;
  int slots_are_i64, page_size;
  FastDiv page_div;
};

template <int V>
struct Piece {
  u16 v[V];
};
template <int V, typename E>
__device__ __forceinline__ Piece<V> load_values(const E* p) {  // (global memory takes any alignment)
  Piece<V> v;
  __builtin_memcpy(&v, p, sizeof(v));
  return v;
}
template <typename T, int V>
__device__ __forceinline__ void to_floats(const Piece<V>& p, float* f) {
#pragma unroll
  for (int i = 0; i < V; i++) f[i] = T::to_f32(p.v[i]);
}
template <typename T, int V>
__device__ __forceinline__ void store_values(u16* p, const float* f) {
  if constexpr (V == 1) {
    *p = T::from_f32(f[0]);
  } else {
    uint32_t w[V / 2];
#pragma unroll
    for (int i = 0; i < V / 2; i++) w[i] = T::pack2(f[2 * i], f[2 * i + 1]);
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
// V values of fp32 or of the 16-bit type, as fp32.
template <typename T, int V>
__device__ __forceinline__ void load_mixed(const void* base, int64_t at, bool f32, float* f) {
  if (f32) __builtin_memcpy(f, (const float*)base + at, 4 * V);
  else to_floats<T>(load_values<V>((const u16*)base + at), f);
}
__device__ __forceinline__ int64_t load_index(const void* base, int64_t at, int is_i64) {
  return is_i64 ? ((const int64_t*)base)[at] : (int64_t)((const int32_t*)base)[at];
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

__device__ __forceinline__ int axis_of_pair(const HeadArgs& a, int i) {
  if (a.alternating) {
    const int m = i - ((i * a.axis_inv) >> 16) * a.axes;  // i mod axes
    const int n = m == 0 ? a.section[0] : m == 1 ? a.section[1] : m == 2 ? a.section[2] : a.section[3];
    return i < a.axes * n ? m : 0;
  }
  return (i >= a.section[1]) + (i >= a.section[2]) + (i >= a.section[3]);
}

// Cosines and sines of pairs [first, first + V) of a token.  A position outside of the table gives NaN: nothing is read there.
template <typename T, int V>
__device__ __forceinline__ void load_turn(const HeadArgs& a, const int64_t (&pos)[4], int first, float* c, float* s) {
  int ax = 0;
  bool mixed = false;
  if (a.axes > 1) {
    ax = axis_of_pair(a, first);
    if (V > 1) {
      const bool same = pos[0] == pos[1] && (a.axes < 3 || pos[0] == pos[2]) && (a.axes < 4 || pos[0] == pos[3]);
      mixed = !same && (a.alternating || axis_of_pair(a, first + V - 1) != ax);
    }
  }
  const int64_t p = ax == 0 ? pos[0] : ax == 1 ? pos[1] : ax == 2 ? pos[2] : pos[3];
  if (!mixed) {
    if ((uint64_t)p < (uint64_t)a.table_rows) {
      load_mixed<T, V>(a.table, p * a.table_stride + first, a.table_is_f32, c);
      load_mixed<T, V>(a.table, p * a.table_stride + first + a.pairs, a.table_is_f32, s);
    } else {
#pragma unroll
      for (int i = 0; i < V; i++) c[i] = s[i] = NAN;
    }
    return;
  }
  if constexpr (V > 1) {  // one row after the other, each pair keeps its own axis's values
#pragma unroll
    for (int i = 0; i < V; i++) c[i] = s[i] = NAN;
#pragma unroll
    for (int k = 0; k < 4; k++) {
      if (k < a.axes && (uint64_t)pos[k] < (uint64_t)a.table_rows) {
        float ck[V], sk[V];
        load_mixed<T, V>(a.table, pos[k] * a.table_stride + first, a.table_is_f32, ck);
        load_mixed<T, V>(a.table, pos[k] * a.table_stride + first + a.pairs, a.table_is_f32, sk);
#pragma unroll
        for (int i = 0; i < V; i++) {
          const bool mine = axis_of_pair(a, first + i) == k;
          c[i] = mine ? ck[i] : c[i];
          s[i] = mine ? sk[i] : s[i];
        }
      }
    }
  }
}

// (f0, f1) are pieces V pairs apart, or 2 V consecutive values.
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

// A head belongs to 2^lanes_log2 lanes, each with K units of 2 V values: V pairs of the rotated part (both halves of them, so
// that a rotation needs no other lane), or 2 V consecutive values.  A lane group takes up to HEADS heads of one token, loads them
// all before it waits for the first and uses the table's row and the weights for all of them.
template <typename T, int V, int K, int HEADS, bool ADJACENT>
__global__ __launch_bounds__(256) void head_rows_kernel(const HeadArgs a) {
  int index = 0;
  while (index + 1 < a.parts && blockIdx.x >= a.part[index + 1].first_block) index++;
  const HeadPart& p = a.part[index];
  const uint32_t group = ((blockIdx.x - p.first_block) << (8 - p.lanes_log2)) + (threadIdx.x >> p.lanes_log2);
  if (group >= p.groups) return;
  const uint32_t token = p.per_token_div.divide(group);
  const int first_head = (int)(group - token * (uint32_t)p.per_token), lane = threadIdx.x & ((1 << p.lanes_log2) - 1);

  int64_t pos[4] = {0, 0, 0, 0}, slot = -1;
  if (p.rot_units) {
#pragma unroll
    for (int k = 0; k < 4; k++)
      if (k < a.axes) pos[k] = load_index(a.positions, k * a.axis_stride + (int64_t)token * a.position_stride, a.positions_are_i64);
  }
  if (p.kind != HEADS_TO_NONE) slot = load_index(a.slots, (int64_t)token * a.slot_stride, a.slots_are_i64);

  // where a lane's pieces lie in a head
  int at0[K], at1[K];
  bool rotated[K], real[K];
#pragma unroll
  for (int j = 0; j < K; j++) {
    const int u = lane + (j << p.lanes_log2);
    real[j] = u < p.units;
    rotated[j] = u < p.rot_units;
    const bool halves = !ADJACENT && rotated[j];
    at0[j] = halves ? u * V : 2 * u * V;
    at1[j] = at0[j] + (halves ? a.pairs : V);
  }

  Piece<V> raw0[HEADS][K], raw1[HEADS][K];
  const u16* x = p.x + (int64_t)token * p.x_token;
#pragma unroll
  for (int h = 0; h < HEADS; h++) {
    const int head = first_head + h * p.per_token;
#pragma unroll
    for (int j = 0; j < K; j++) {
      raw0[h][j] = {}, raw1[h][j] = {};
      if (head < p.heads && real[j]) {
        raw0[h][j] = load_values<V>(x + head * p.x_head + at0[j]);
        raw1[h][j] = load_values<V>(x + head * p.x_head + at1[j]);
      }
    }
  }
  float c[K][V], s[K][V], w0[K][V], w1[K][V];
#pragma unroll
  for (int j = 0; j < K; j++) {
#pragma unroll
    for (int i = 0; i < V; i++) w0[j][i] = w1[j][i] = 1.f;
    if (rotated[j]) load_turn<T, V>(a, pos, (lane + (j << p.lanes_log2)) * V, c[j], s[j]);
    if (p.w && real[j]) {
      load_mixed<T, V>(p.w, at0[j], p.w_is_f32, w0[j]);
      load_mixed<T, V>(p.w, at1[j], p.w_is_f32, w1[j]);
    }
  }

  const bool kept = (uint64_t)slot < (uint64_t)a.num_slots;  // (a negative slot is padding)
  uint32_t page = 0, in_page = 0;
  if (kept) {
    page = a.page_div.divide((uint32_t)slot);
    in_page = (uint32_t)slot - page * (uint32_t)a.page_size;
  }

#pragma unroll
  for (int h = 0; h < HEADS; h++) {
    const int head = first_head + h * p.per_token;
    if (head >= p.heads) return;
    float f0[K][V], f1[K][V];
#pragma unroll
    for (int j = 0; j < K; j++) {
      to_floats<T>(raw0[h][j], f0[j]);
      to_floats<T>(raw1[h][j], f1[j]);
    }
    if (p.w) {
      float sum = 0.f;
#pragma unroll
      for (int j = 0; j < K; j++)
#pragma unroll
        for (int i = 0; i < V; i++) sum = fmaf(f0[j][i], f0[j][i], fmaf(f1[j][i], f1[j][i], sum));
      sum = group_sum(sum, p.lanes_log2);
      // (a sum beyond fp32 would give zeros)
      const float r = sum < INFINITY ? rsqrtf(fmaf(sum, p.inv_dim, p.eps)) : NAN;
#pragma unroll
      for (int j = 0; j < K; j++)
#pragma unroll
        for (int i = 0; i < V; i++) {
          f0[j][i] = f0[j][i] * r * w0[j][i];
          f1[j][i] = f1[j][i] * r * w1[j][i];
        }
    }
#pragma unroll
    for (int j = 0; j < K; j++)
      if (rotated[j]) turn<V, ADJACENT>(f0[j], f1[j], c[j], s[j]);

    if (p.out) {
      u16* out = p.out + (int64_t)token * p.out_token + head * p.out_head;
#pragma unroll
      for (int j = 0; j < K; j++)
        if (real[j]) {
          store_values<T, V>(out + at0[j], f0[j]);
          store_values<T, V>(out + at1[j], f1[j]);
        }
    }
    if (p.kind == HEADS_TO_NONE || !kept) continue;
    uint8_t* row = p.cache + page * p.cache_page + in_page * p.cache_slot + head * p.cache_head;
    if (p.kind == HEADS_TO_16) {
#pragma unroll
      for (int j = 0; j < K; j++)
        if (real[j]) {
          store_values<T, V>((u16*)row + at0[j], f0[j]);
          store_values<T, V>((u16*)row + at1[j], f1[j]);
        }
      continue;
    }
    // one scale per row, or per 128 values of it
    uint32_t hi[K], whole = 0;
    RowScale given = {};
    if (p.given) {
      given.mul = fp8_row_multiplier(1.0f, p.given[head * p.given_head]);
    } else {
#pragma unroll
      for (int j = 0; j < K; j++) {
        hi[j] = 0;
#pragma unroll
        for (int i = 0; i < V; i++) {
          hi[j] = umax(hi[j], __float_as_uint(f0[j][i]) & 0x7fffffffu);
          hi[j] = umax(hi[j], __float_as_uint(f1[j][i]) & 0x7fffffffu);
        }
        if (!real[j]) hi[j] = 0;  // (a row of NaN: its idle lanes' zeros are NaN too)
        whole = umax(whole, hi[j]);
      }
      if (K == 1 || p.scale_units == p.units) {
        whole = group_umax(whole, p.scale_lanes_log2);
#pragma unroll
        for (int j = 0; j < K; j++) hi[j] = whole;
      } else {
#pragma unroll
        for (int j = 0; j < K; j++) hi[j] = group_umax(hi[j], p.scale_lanes_log2);
      }
    }
#pragma unroll
    for (int j = 0; j < K; j++) {
      if (!real[j]) continue;
      RowScale o = given;
      if (!p.given) {
        o = p.kind == HEADS_TO_FP8 ? found_scale<ROW_TO_FP8>(hi[j]) : found_scale<ROW_TO_INT8>(hi[j]);
        const int u = lane + (j << p.lanes_log2);
        const int n = p.scale_units == p.units ? 0 : u >> p.scale_lanes_log2;
        if (u == n * p.scale_units)
          p.scales[page * p.scales_page + in_page * p.scales_slot + head * p.scales_head + n * p.scales_group] = o.scale;
      }
      if (p.kind == HEADS_TO_FP8) {
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

constexpr int GATHER_UNITS = 4;  // a lane's units: their loads are in flight together

template <int V>
struct Bytes {
  uint8_t v[V];
};

template <typename T, int V>
__global__ __launch_bounds__(256) void gather_rows_kernel(const GatherArgs a) {
  const int index = a.parts > 1 && blockIdx.x >= a.part[1].first_block;
  const GatherPart& p = a.part[index];
  const uint32_t base = (blockIdx.x - p.first_block) * (256 * GATHER_UNITS) + threadIdx.x;
  uint32_t row[GATHER_UNITS], head[GATHER_UNITS], unit[GATHER_UNITS];
  int64_t slot[GATHER_UNITS];
#pragma unroll
  for (int k = 0; k < GATHER_UNITS; k++) {
    const uint32_t i = base + 256 * k;
    row[k] = p.per_row_div.divide(i);
    const uint32_t in_row = i - row[k] * (uint32_t)p.per_row;
    head[k] = p.per_head_div.divide(in_row);
    unit[k] = in_row - head[k] * (uint32_t)p.per_head;
    slot[k] = i < p.units ? load_index(a.slots, (int64_t)row[k] * a.slot_stride, a.slots_are_i64) : -1;
  }
  Bytes<V> codes[GATHER_UNITS];
  Piece<V> values[GATHER_UNITS];
  float scale[GATHER_UNITS];
#pragma unroll
  for (int k = 0; k < GATHER_UNITS; k++) {
    codes[k] = {}, values[k] = {}, scale[k] = 0.f;
    if ((uint64_t)slot[k] < (uint64_t)a.num_slots) {
      const uint32_t page = a.page_div.divide((uint32_t)slot[k]), in_page = (uint32_t)slot[k] - page * (uint32_t)a.page_size;
      const uint8_t* src = p.cache + page * p.cache_page + in_page * p.cache_slot + head[k] * p.cache_head;
      if (p.kind == HEADS_TO_16) {
        values[k] = load_values<V>((const u16*)src + unit[k] * V);
      } else {
        __builtin_memcpy(&codes[k], src + unit[k] * V, V);
        scale[k] = p.given ? p.given[head[k] * p.given_head]
                           : p.scales[page * p.scales_page + in_page * p.scales_slot + head[k] * p.scales_head +
                                      (unit[k] >> p.group_units_log2) * p.scales_group];
      }
    }
  }
#pragma unroll
  for (int k = 0; k < GATHER_UNITS; k++) {
    if (base + 256 * k >= p.units) return;
    u16* out = p.out + (int64_t)row[k] * p.out_row + head[k] * p.out_head + unit[k] * V;
    if (p.kind == HEADS_TO_16) {
      __builtin_memcpy(out, &values[k], 2 * V);
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
    // (a slot that is none gives zeros, also where a given scale is not finite)
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

template <typename T, int V, int K, int HEADS>
static void launch_heads(const HeadArgs& a, unsigned blocks, bool adjacent, hipStream_t st) {
  if (adjacent) hipLaunchKernelGGL((head_rows_kernel<T, V, K, HEADS, true>), dim3(blocks), dim3(256), 0, st, a);
  else hipLaunchKernelGGL((head_rows_kernel<T, V, K, HEADS, false>), dim3(blocks), dim3(256), 0, st, a);
}

// How many heads of a token a lane group takes.
constexpr int HEADS_MANY = 4;

extern "C" int sglamd_head_rows(const sglamd_heads* parts, int num_parts, int64_t tokens, int dtype, const sglamd_rotation* rotation,
                                const sglamd_slots* slots, void* stream) {
  const char* op = "head_rows";
  SGLAMD_REQUIRE(parts && num_parts > 0 && num_parts <= MAX_PARTS, SGLAMD_EINVAL, "%s: one to %d tensors of heads", op, MAX_PARTS);
  SGLAMD_REQUIRE(dtype == SGLAMD_BF16 || dtype == SGLAMD_F16, SGLAMD_EINVAL, "%s: heads must be Half or BFloat16", op);
  SGLAMD_REQUIRE(tokens >= 0 && tokens < (1ll << 31), SGLAMD_EINVAL, "%s: bad token count %lld", op, (long long)tokens);
  HeadArgs a = {};
  a.parts = num_parts;
  int64_t width = 0;  // of the rotated part
  for (int i = 0; i < num_parts; i++)
    if (parts[i].rotate) {
      SGLAMD_REQUIRE(rotation, SGLAMD_EINVAL, "%s: a rotation without its table", op);
      width = rotation->width;
    }
  if (width || rotation) {
    const sglamd_rotation& r = *rotation;
    width = r.width;
    SGLAMD_REQUIRE(r.cos_sin && r.positions, SGLAMD_EINVAL, "%s: null table or positions", op);
    SGLAMD_REQUIRE(r.table_dtype == SGLAMD_F32 || r.table_dtype == dtype, SGLAMD_EINVAL, "%s: the table must be Float or of the heads' type", op);
    SGLAMD_REQUIRE(r.positions_dtype == SGLAMD_I32 || r.positions_dtype == SGLAMD_I64, SGLAMD_EINVAL, "%s: positions must be I32 or I64", op);
    SGLAMD_REQUIRE(r.width > 0 && r.width % 2 == 0 && r.width <= 1024, SGLAMD_EINVAL, "%s: a rotated width of %lld: even, 2 to 1024", op,
                   (long long)r.width);
    SGLAMD_REQUIRE(r.table_rows >= 0 && r.table_rows < (1ll << 40) && (r.table_rows <= 1 || r.table_stride >= 0), SGLAMD_EINVAL,
                   "%s: bad table rows or stride", op);
    SGLAMD_REQUIRE(r.axes >= 1 && r.axes <= 4, SGLAMD_EINVAL, "%s: one to four position axes", op);
    a.table = r.cos_sin, a.table_stride = r.table_stride, a.table_rows = r.table_rows, a.table_is_f32 = r.table_dtype == SGLAMD_F32;
    a.positions = r.positions, a.positions_are_i64 = r.positions_dtype == SGLAMD_I64;
    a.axis_stride = r.axis_stride, a.position_stride = r.position_stride;
    a.pairs = (int)(r.width / 2), a.axes = r.axes, a.alternating = r.alternating && r.axes > 1;
    if (r.axes > 1) {
      int64_t sum = 0;
      for (int k = 0; k < r.axes; k++) {
        SGLAMD_REQUIRE(r.sections[k] >= 0, SGLAMD_EINVAL, "%s: a section is negative", op);
        sum += r.sections[k];
      }
      SGLAMD_REQUIRE(sum == a.pairs, SGLAMD_EINVAL, "%s: sections of %lld pairs for a rotated width of %lld", op, (long long)sum, (long long)r.width);
      if (a.alternating) {
        a.axis_inv = (65536 + r.axes - 1) / r.axes;
        for (int k = 0; k < 4; k++) a.section[k] = k < r.axes ? r.sections[k] : 0;
        // the pairs that the rule gives to axis 0 beyond its own turns have to be as many as its section says
        for (int k = 1; k < r.axes; k++)
          SGLAMD_REQUIRE(r.sections[k] == 0 || k + (int64_t)r.axes * (r.sections[k] - 1) < a.pairs, SGLAMD_EINVAL,
                         "%s: alternating sections: axis %d has no %d turns in %d pairs", op, k, (int)r.sections[k], a.pairs);
      } else {
        int at = 0;
        for (int k = 0; k < 4; k++) {  // where axis k begins (axes that are not there: behind the last pair)
          a.section[k] = k < r.axes ? at : a.pairs;
          if (k < r.axes) at += r.sections[k];
        }
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

  // one head per lane group until the heads of a launch fill the chip
  int64_t lanes = 0;
  for (int i = 0; i < num_parts; i++) lanes += tokens * parts[i].heads << log2_up(ceil_div(parts[i].dim, 2 * v * k));
  const int many = v == 8 && lanes >= (int64_t)device_cus() * 2048 * 4 ? HEADS_MANY : 1;

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
    p.w = h.weight, p.w_is_f32 = h.weight_dtype == SGLAMD_F32, p.eps = h.eps, p.inv_dim = 1.0f / (float)h.dim;
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
      p.scale_units = p.units, p.scale_lanes_log2 = p.lanes_log2;
      if (h.scales && h.scale_group != h.dim) {
        SGLAMD_REQUIRE(h.scale_group == 128 && h.dim % 128 == 0 && !h.rotate, SGLAMD_EINVAL,
                       "%s: a scale per row, or per 128 values of rows that are not rotated and a multiple of 128 long", op);
        p.scale_units = 64 / v, p.scale_lanes_log2 = log2_up(p.scale_units);
        if (k > 1) p.lanes_log2 = 6;  // a round of the wave's lanes is one scale
      }
    }
    p.per_token = (int)ceil_div(h.heads, many);
    const uint64_t groups = (uint64_t)tokens * (uint64_t)p.per_token;
    SGLAMD_REQUIRE(groups << p.lanes_log2 < (1ull << 31), SGLAMD_EINVAL, "%s: %lld tokens of %lld heads are too many for one launch", op,
                   (long long)tokens, (long long)h.heads);
    p.groups = (uint32_t)groups, p.per_token_div = FastDiv::of((uint32_t)(p.per_token ? p.per_token : 1));
    p.first_block = (uint32_t)blocks;
    blocks += ((groups << p.lanes_log2) + 255) / 256;
  }
  if (blocks == 0) return SGLAMD_OK;
  SGLAMD_REQUIRE(blocks < (1ull << 24), SGLAMD_EINVAL, "%s: %lld tokens are too many for one launch", op, (long long)tokens);
  const bool adjacent = rotation && rotation->interleaved;
  hipStream_t st = (hipStream_t)stream;
  const DeviceScope scope;
#define SGLAMD_HEADS(T)                                                                       \
  do {                                                                                        \
    if (v == 8 && many > 1) launch_heads<T, 8, 1, HEADS_MANY>(a, (unsigned)blocks, adjacent, st); \
    else if (v == 8) launch_heads<T, 8, 1, 1>(a, (unsigned)blocks, adjacent, st);             \
    else if (v == 4) launch_heads<T, 4, 1, 1>(a, (unsigned)blocks, adjacent, st);             \
    else launch_heads<T, 1, 8, 1>(a, (unsigned)blocks, adjacent, st);                         \
  } while (0)
  if (dtype == SGLAMD_BF16) SGLAMD_HEADS(BF16);
  else SGLAMD_HEADS(F16);
#undef SGLAMD_HEADS
  return check_launch(op);
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
  int v = 16;
  for (int i = 0; i < num_parts; i++) {
    const sglamd_gather& g = parts[i];
    SGLAMD_REQUIRE(g.heads >= 0 && g.heads < (1 << 20) && g.dim > 0 && g.dim <= 1024, SGLAMD_EINVAL, "%s: %lld heads of %lld values: up to 1024", op,
                   (long long)g.heads, (long long)g.dim);
    while (v > 1 && g.dim % v) v /= 2;
  }
  if (v < 8) v = v == 4 ? 4 : 1;
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
    SGLAMD_REQUIRE((uint64_t)g.heads * (uint64_t)p.per_head < (1ull << 31) && units < (1ull << 31) - 256 * GATHER_UNITS, SGLAMD_EINVAL,
                   "%s: %lld rows are too many for one launch", op, (long long)rows);
    p.units = (uint32_t)units, p.per_row_div = FastDiv::of((uint32_t)(p.per_row ? p.per_row : 1)), p.per_head_div = FastDiv::of((uint32_t)p.per_head);
    p.first_block = (uint32_t)blocks;
    blocks += (units + 256 * GATHER_UNITS - 1) / (256 * GATHER_UNITS);
  }
  if (blocks == 0) return SGLAMD_OK;
  hipStream_t st = (hipStream_t)stream;
#define SGLAMD_GATHER(T)                                                                                                       \
  do {                                                                                                                         \
    if (v == 16) hipLaunchKernelGGL((gather_rows_kernel<T, 16>), dim3((unsigned)blocks), dim3(256), 0, st, a);                 \
    else if (v == 8) hipLaunchKernelGGL((gather_rows_kernel<T, 8>), dim3((unsigned)blocks), dim3(256), 0, st, a);              \
    else if (v == 4) hipLaunchKernelGGL((gather_rows_kernel<T, 4>), dim3((unsigned)blocks), dim3(256), 0, st, a);              \
    else hipLaunchKernelGGL((gather_rows_kernel<T, 1>), dim3((unsigned)blocks), dim3(256), 0, st, a);                          \
  } while (0)
  if (dtype == SGLAMD_BF16) SGLAMD_GATHER(BF16);
  else SGLAMD_GATHER(F16);
#undef SGLAMD_GATHER
  return check_launch(op);
}
