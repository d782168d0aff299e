// elem.h -- activations of the row kernels (layer norm, distillation):
// fp32, bf16 or fp16 in memory, fp32 in registers.
#pragma once
#include "common.h"

namespace concord {

struct BF16 {
  uint16_t bits;
};

CONCORD_DEV float to_f32(float v) { return v; }
CONCORD_DEV float to_f32(_Float16 v) { return (float)v; }
CONCORD_DEV float to_f32(BF16 v) { return bf16_to_f32(v.bits); }
template <class T>
CONCORD_DEV T from_f32(float v);
template <>
CONCORD_DEV float from_f32<float>(float v) { return v; }
template <>
CONCORD_DEV _Float16 from_f32<_Float16>(float v) { return (_Float16)v; }
template <>
CONCORD_DEV BF16 from_f32<BF16>(float v) { return BF16{(uint16_t)pack_bf16x2(v, 0.0f)}; }

// VEC elements that one load or store moves (16 bytes, or one element)
template <class T, int VEC>
struct alignas(sizeof(T) * VEC) Chunk {
  T v[VEC];
};

// a store of a result that this kernel does not read again: past the caches,
// which keep the operands (layer norm in bf16, 16384 x 384: forward 9.5 -> 7.5 us;
// 32768 x 4096: backward 160 -> 149 us, forward 96 either way)
template <class V>
CONCORD_DEV void store_stream(V* p, const V& v) {
  if constexpr (sizeof(V) == 16) {
    typedef int32_t i32x4 __attribute__((ext_vector_type(4)));
    __builtin_nontemporal_store(__builtin_bit_cast(i32x4, v), (i32x4*)p);
  } else {
    *p = v;
  }
}

// the value of element i of a vector of any of the three types
CONCORD_DEV float load_any(const void* p, int dtype, int64_t i) {
  if (dtype == CONCORD_F32) return ((const float*)p)[i];
  if (dtype == CONCORD_BF16) return bf16_to_f32(((const uint16_t*)p)[i]);
  return (float)((const _Float16*)p)[i];
}
CONCORD_DEV void store_any(void* p, int dtype, int64_t i, float v) {
  if (dtype == CONCORD_F32) ((float*)p)[i] = v;
  else if (dtype == CONCORD_BF16) ((BF16*)p)[i] = from_f32<BF16>(v);
  else ((_Float16*)p)[i] = (_Float16)v;
}

// Sum over the wave's 64 lanes, to every lane (a scalar), in a fixed order:
// prefix sums within each 16-lane row (row_shr 1, 2, 4, 8), lane 15 of a row
// into the next (row_bcast:15), lane 31 into the upper rows (row_bcast:31);
// wave_max has the steps one by one.  Lanes without a source add 0.
CONCORD_DEV float wave_sum(float v) {
#define CONCORD_DPP_ADD(ctrl) \
  v = __fadd_rn(v, __int_as_float(__builtin_amdgcn_update_dpp(0, __float_as_int(v), ctrl, 0xF, 0xF, true)))
  CONCORD_DPP_ADD(0x111);
  CONCORD_DPP_ADD(0x112);
  CONCORD_DPP_ADD(0x114);
  CONCORD_DPP_ADD(0x118);
  CONCORD_DPP_ADD(0x142);
  CONCORD_DPP_ADD(0x143);
#undef CONCORD_DPP_ADD
  return lane_value(v, 63);
}

// Sum over each group of 16 lanes, to each of them: lanes 1, 2 apart, then the
// mirrored half and the mirrored other half.
CONCORD_DEV float row16_sum(float v) {
#define CONCORD_DPP_ADD(ctrl) \
  v = __fadd_rn(v, __int_as_float(__builtin_amdgcn_update_dpp(0, __float_as_int(v), ctrl, 0xF, 0xF, true)))
  CONCORD_DPP_ADD(0xB1);    // quad_perm 1, 0, 3, 2
  CONCORD_DPP_ADD(0x4E);    // quad_perm 2, 3, 0, 1
  CONCORD_DPP_ADD(0x141);   // row_half_mirror
  CONCORD_DPP_ADD(0x140);   // row_mirror
#undef CONCORD_DPP_ADD
  return v;
}

// Maximum over the wave's 64 lanes, to every lane.  Lanes without a source
// keep their own value (old = v).
CONCORD_DEV float wave_max_f32(float v) {
#define CONCORD_DPP_MAX(ctrl)                                                                             \
  v = fmaxf(v, __int_as_float(__builtin_amdgcn_update_dpp(__float_as_int(v), __float_as_int(v), ctrl, 0xF, \
                                                          0xF, false)))
  CONCORD_DPP_MAX(0x111);
  CONCORD_DPP_MAX(0x112);
  CONCORD_DPP_MAX(0x114);
  CONCORD_DPP_MAX(0x118);
  CONCORD_DPP_MAX(0x142);
  CONCORD_DPP_MAX(0x143);
#undef CONCORD_DPP_MAX
  return lane_value(v, 63);
}

}  // namespace concord
