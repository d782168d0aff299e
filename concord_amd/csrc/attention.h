// attention.h -- what the attention kernels share: where a workgroup's tile
// lies in the sequences, operand tiles in LDS and their MFMA fragments.
//
// A product runs on v_mfma_f32_32x32x16_bf16.  Its A operand has 32 rows, B
// has 32 columns, both 16 deep: lane l holds row (column) l & 31 and the depth
// indices 8 (l >> 5) .. + 7; of the 32 x 32 result it holds column l & 31 and
// the rows 8 (r >> 2) + 4 (l >> 5) + (r & 3), r = 0 .. 15.  The depth order is
// free as long as both operands agree, so a result feeds the next product as
// its B operand without any exchange between lanes: registers 8 t .. 8 t + 7
// of a result are the depth indices 16 t + {0 .. 3, 8 .. 11} + 4 (l >> 5), and
// the A operand is read in that order (Tile::cols).
#pragma once
#include <type_traits>
#include <utility>

#include "common.h"

namespace concord {

typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));
typedef float f32x16 __attribute__((ext_vector_type(16)));
typedef int32_t i32x4 __attribute__((ext_vector_type(4)));
typedef short i16x4 __attribute__((ext_vector_type(4)));
typedef __attribute__((address_space(3))) char lds_char;
typedef __attribute__((address_space(3))) i32x4 lds_i32x4;
typedef __attribute__((address_space(3))) i16x4 lds_i16x4;
typedef __attribute__((address_space(3))) float lds_float;

constexpr float kLog2e = 1.4426950408889634f;

CONCORD_DEV f32x16 mfma(bf16x8 a, bf16x8 b, f32x16 c) {
  return __builtin_amdgcn_mfma_f32_32x32x16_bf16(a, b, c, 0, 0, 0);
}
CONCORD_DEV f32x16 zero16() {
  f32x16 z;
#pragma unroll
  for (int i = 0; i < 16; ++i) z[i] = 0.0f;
  return z;
}
// registers 8 t .. 8 t + 7 of a result, rounded to bf16: a B operand
CONCORD_DEV bf16x8 round8(const f32x16& v, int t) {
  i32x4 w;
#pragma unroll
  for (int i = 0; i < 4; ++i) w[i] = (int32_t)pack_bf16x2(v[8 * t + 2 * i], v[8 * t + 2 * i + 1]);
  return __builtin_bit_cast(bf16x8, w);
}

// the other half wave's value of the same column (lane l ^ 32), as a pair
// {lower half's, upper half's}
struct Halves {
  float lo, hi;
};
CONCORD_DEV Halves halves(float v) {
  const auto r = __builtin_amdgcn_permlane32_swap(__float_as_uint(v), __float_as_uint(v), false, false);
  return Halves{__uint_as_float(r[0]), __uint_as_float(r[1])};
}

// f(0), f(1), ... f(N - 1) with compile-time arguments
template <class F, int... I>
CONCORD_DEV void static_for_impl(F&& f, std::integer_sequence<int, I...>) {
  (f(std::integral_constant<int, I>()), ...);
}
template <int N, class F>
CONCORD_DEV void static_for(F&& f) {
  static_for_impl(f, std::make_integer_sequence<int, N>());
}
#define CONCORD_INLINE_LAMBDA __attribute__((always_inline))

// ---- LDS and barriers --------------------------------------------------------
CONCORD_DEV uint32_t lds_addr(const void* p) {
  typedef __attribute__((address_space(3))) const void* lds_ptr;
  return (uint32_t)__builtin_amdgcn_readfirstlane((int)(uint32_t)(uintptr_t)(lds_ptr)p);
}
CONCORD_DEV const lds_char* lds_at(uint32_t a) { return (const lds_char*)(uintptr_t)0 + a; }

// s_waitcnt immediate: at most n vector memory operations outstanding
constexpr int vmcnt_imm(int n) { return (n & 0xF) | (0x7 << 4) | (0xF << 8) | (((n >> 4) & 3) << 14); }

// a workgroup barrier that orders LDS alone (the DMAs are waited for by hand)
CONCORD_DEV void lds_barrier() {
  __builtin_amdgcn_fence(__ATOMIC_RELEASE, "workgroup", "local");
  __builtin_amdgcn_s_barrier();
  __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "workgroup", "local");
}

// One LDS-DMA load of 16 bytes per lane, to LDS bytes lds + 16 lane; zeros for
// a lane at or past num_records.  Inline assembly, so that the compiler does
// not wait for it before every LDS read (s_nop: M0 needs a wait state between
// its write and the DMA).
CONCORD_DEV void dma16(i32x4 rsrc, uint32_t voff, uint32_t lds) {
  asm volatile("s_mov_b32 m0, %2\n\ts_nop 0\n\tbuffer_load_dwordx4 %0, %1, 0 offen lds"
               :
               : "v"(voff), "s"(rsrc), "s"(lds)
               : "memory", "m0");
}

// the same with 4 bytes per lane
CONCORD_DEV void dma4(i32x4 rsrc, uint32_t voff, uint32_t lds) {
  asm volatile("s_mov_b32 m0, %2\n\ts_nop 0\n\tbuffer_load_dword %0, %1, 0 offen lds"
               :
               : "v"(voff), "s"(rsrc), "s"(__builtin_amdgcn_readfirstlane((int)lds))
               : "memory", "m0");
}

// a lane offset past every buffer's num_records (at most 2^31)
constexpr uint32_t kOOB = 0x80000000u;

// raw buffer over rows [0, rows) of `ld2` bytes each, `row_bytes` of a row
// readable: everything at or past the last row's end reads as zero
CONCORD_DEV i32x4 rows_rsrc(const uint16_t* p, int rows, uint32_t ld2, uint32_t row_bytes) {
  const uint64_t a = (uint64_t)(uintptr_t)p;
  const uint32_t n = rows > 0 ? (uint32_t)(rows - 1) * ld2 + row_bytes : 0u;
  return i32x4{__builtin_amdgcn_readfirstlane((int32_t)(uint32_t)a),
               __builtin_amdgcn_readfirstlane((int32_t)(uint32_t)((a >> 32) & 0xFFFF)),
               __builtin_amdgcn_readfirstlane((int32_t)n), 0x00020000};
}
CONCORD_DEV __amdgpu_buffer_rsrc_t rows_buffer(const uint16_t* p, int rows, uint32_t ld2, uint32_t row_bytes) {
  const uint32_t n = rows > 0 ? (uint32_t)(rows - 1) * ld2 + row_bytes : 0u;
  return __builtin_amdgcn_make_buffer_rsrc(const_cast<uint16_t*>(p), (short)0, (int)n, 0x00020000);
}

// ---- operand tiles -------------------------------------------------------------
// Head dimensions up to 16 NK, padded with zeros to it.
template <int NK_>
struct Dim {
  static constexpr int NK = NK_;               // depth steps of a product over the head dimension
  static constexpr int ND = (NK + 1) / 2;      // 32-wide blocks of it
  static constexpr int PITCH = NK > 4 ? 256 : 128;   // LDS bytes of a row
};

// A tile of ROWS rows of a token-major operand (row: one token's head, up to
// PITCH bytes) in LDS, loaded by DMA and read as an A operand in both
// directions:
//   rows(i, k): 32 of its rows by 16 of the head dimension (row fragment)
//   cols(t, d): 32 of the head dimension by 16 of its rows (transposed)
// A DMA instruction fills a group of GROUP rows, 1 KB, in which the 16-byte
// chunk c of row r lies in slot c ^ swz(r); PAD bytes follow each group.  LDS
// has 64 banks.  A row fragment's 16-byte reads go in phases of 16 lanes, four
// times four rows that start at rows 0, 12, 20, 24 (and 4, 8, 16, 28) of the
// 32; a transposed read's 8-byte reads go 4 rows by 64 bytes at a time.  The
// four rows differ in the slot's bits 2 and up (with 128-byte rows in bit 2
// and the row's parity), the four groups of rows in its bits 0 and 1, by the
// padding and swz: neither read has bank conflicts (a swizzle for 16 rows in a
// row cost half as much again in LDS time with 128-byte rows).  swz leaves the
// slot's bit 1 alone, so two depth steps share an address register (Frags).
template <class DIM, int ROWS, int WAVES>
struct Tile {
  static constexpr int PITCH = DIM::PITCH, GROUP = 1024 / PITCH, GBYTES = 1024 + (PITCH == 256 ? 16 : 32);
  static constexpr int BYTES = ROWS / GROUP * GBYTES, SLOTS = PITCH / 16;
  static constexpr int PER = ROWS / GROUP / WAVES;   // DMA instructions of a wave
  static_assert(PER * GROUP * WAVES == ROWS, "rows split evenly over the waves");
  static CONCORD_DEV int swz(int r) { return PITCH == 256 ? (r & 3) << 2 : ((r & 2) << 1) | ((r & 4) >> 2); }
  // the address of row r (a multiple of GROUP) in the tile
  static constexpr uint32_t at(int r) { return (uint32_t)(r / GROUP * GBYTES); }
  uint32_t voff;
  uint32_t ld2, row_bytes;
  // ld: elements between rows; D: head dimension
  CONCORD_DEV void init(int64_t ld, int D, int lane) {
    ld2 = (uint32_t)(ld * 2);
    row_bytes = (uint32_t)D * 2;
    const int r = lane / SLOTS, c = (lane % SLOTS) ^ swz(r);
    voff = c * 8 < D ? (uint32_t)r * ld2 + (uint32_t)c * 16 : kOOB;
  }
  // rows [0, left) at p (the others read as zeros) into the tile at LDS address `lds`
  CONCORD_DEV void load(const uint16_t* p, int left, uint32_t lds, int wave) const {
    const int first = wave * PER * GROUP, n = left - first;
    const i32x4 rs = rows_rsrc(p + (int64_t)first * (ld2 / 2), n < PER * GROUP ? n : PER * GROUP, ld2, row_bytes);
#pragma unroll
    for (int q = 0; q < PER; ++q)
      dma16(rs, voff + (uint32_t)(q * GROUP) * ld2,
            (uint32_t)__builtin_amdgcn_readfirstlane((int)(lds + (uint32_t)((wave * PER + q) * GBYTES))));
  }
};

// (an opaque value: the constants added to an address stay in the instructions'
// offsets, where the compiler would otherwise keep a register for each sum)
CONCORD_DEV void pin(uint32_t& v) { asm volatile("" : "+v"(v)); }

// A lane's addresses in the tiles from LDS address `base` on; a tile's place,
// blocks of rows and depth steps are constants added to them.
template <class DIM>
struct Frags {
  typedef Tile<DIM, 64, 4> T;
  static constexpr int NR = (DIM::NK + 1) / 2;
  uint32_t row[NR];          // rows(): by pair of steps
  uint32_t col[DIM::ND];     // cols(): by 32-wide block
  CONCORD_DEV void init(uint32_t base, int lane) {
    const int r = lane & 31, h = lane >> 5;
    const uint32_t r0 = base + T::at(r & ~(T::GROUP - 1)) + (uint32_t)((r & (T::GROUP - 1)) * DIM::PITCH);
#pragma unroll
    for (int j = 0; j < NR; ++j)
      row[j] = r0 + (uint32_t)(((4 * j + h) ^ T::swz(r)) << 4), pin(row[j]);
    const int cr = 4 * h + ((lane >> 2) & 3), chunk = 2 * ((lane >> 4) & 1) + ((lane & 3) >> 1);
    const uint32_t c0 = base + T::at(cr & ~(T::GROUP - 1)) + (uint32_t)((cr & (T::GROUP - 1)) * DIM::PITCH);
#pragma unroll
    for (int d = 0; d < DIM::ND; ++d)
      col[d] = c0 + (uint32_t)((((4 * d + chunk) ^ T::swz(cr)) << 4) + ((lane & 1) << 3)), pin(col[d]);
  }
  // to the tiles `bytes` further on
  CONCORD_DEV void move(int32_t bytes) {
#pragma unroll
    for (int j = 0; j < NR; ++j) row[j] += (uint32_t)bytes;
#pragma unroll
    for (int d = 0; d < DIM::ND; ++d) col[d] += (uint32_t)bytes;
  }
  // rows 32 i .. 32 i + 31, head dimension 16 k .. 16 k + 15
  CONCORD_DEV bf16x8 rows(uint32_t tile, int i, int k) const {
    const uint32_t o = tile + T::at(32 * i) + (uint32_t)((k & 1) * 32);
    return __builtin_bit_cast(bf16x8, *(const lds_i32x4*)(lds_at(row[k >> 1]) + o));
  }
  // head dimension 32 d .. 32 d + 31, rows 16 t .. 16 t + 15 in the order of
  // a result's registers
  CONCORD_DEV bf16x8 cols(uint32_t tile, int d, int t) const {
    const i16x4 lo = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_i16x4*)(lds_at(col[d]) + tile + T::at(16 * t)));
    const i16x4 hi = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_i16x4*)(lds_at(col[d]) + tile + T::at(16 * t + 8)));
    return __builtin_bit_cast(bf16x8, __builtin_shufflevector(lo, hi, 0, 1, 2, 3, 4, 5, 6, 7));
  }
};

// A B operand that stays in registers: 32 rows of a token-major operand (the
// product's columns), all of the head dimension.
template <class DIM>
struct Fixed {
  bf16x8 f[DIM::NK];
  // rows [0, left) at p; the others and dimensions past D read as zeros
  CONCORD_DEV void load(const uint16_t* p, int left, int64_t ld, int D, int lane) {
    const uint32_t ld2 = (uint32_t)(ld * 2);
    const auto rs = rows_buffer(p, left < 32 ? left : 32, ld2, (uint32_t)D * 2);
    const int r = lane & 31, h = lane >> 5;
#pragma unroll
    for (int k = 0; k < DIM::NK; ++k) {
      const int c = 2 * k + h;
      const uint32_t off = c * 8 < D && r < left ? (uint32_t)r * ld2 + (uint32_t)c * 16 : kOOB;
      f[k] = __builtin_bit_cast(bf16x8, __builtin_amdgcn_raw_buffer_load_b128(rs, off, 0, 0));
    }
  }
};

// sum over the head dimension of the lane's row of out and of b, half of
// it in each half wave: out is the row in bf16 and its left-over bytes
template <class DIM>
CONCORD_DEV float row_dot(const Fixed<DIM>& out, const int8_t* low, int left, int64_t low_ld, int D, const Fixed<DIM>& b,
                          int lane) {
  const int r = lane & 31, h = lane >> 5;
  float s = 0.0f;
#pragma unroll
  for (int k = 0; k < DIM::NK; ++k) {
    const int c = (2 * k + h) * 8;
    uint2 w = make_uint2(0, 0);
    if (r < left && c < D) w = *(const uint2*)(low + (int64_t)r * low_ld + c);
    const i32x4 hi = __builtin_bit_cast(i32x4, out.f[k]);
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      const uint32_t bits = e & 1 ? (uint32_t)hi[e >> 1] & 0xFFFF0000u : (uint32_t)hi[e >> 1] << 16;
      const int32_t byte = __builtin_amdgcn_sbfe((int32_t)(e < 4 ? w.x : w.y), 8 * (e & 3), 8);
      s = __builtin_fmaf(__uint_as_float(bits + (uint32_t)(byte * 256)), (float)b.f[k][e], s);
    }
  }
  const Halves both = halves(s);
  return both.lo + both.hi;
}

// Store a transposed result block (rows: head dimension 32 d .., columns: the
// tokens of p's rows) times the columns' factor, as bf16.  The half waves
// exchange registers so that each lane stores 16 bytes of its token.  low, if
// given, takes what the rounding left over (concord_attn_args.out_low).
CONCORD_DEV int32_t left_over(float x, uint32_t bf16) {
  const int32_t r = (int32_t)(__float_as_uint(x) - (bf16 << 16)) >> 8;   // -128 .. 128
  return min(r, 127) & 255;
}
CONCORD_DEV void store_block(uint16_t* p, int64_t ld, int left, int D, int d, const f32x16& v, float factor, int lane,
                             int8_t* low = nullptr, int64_t low_ld = 0) {
  const int r = lane & 31, h = lane >> 5;
  if (r >= left) return;
  uint16_t* q = p + (int64_t)r * ld;
#pragma unroll
  for (int g = 0; g < 4; g += 2) {
    uint32_t a[2], b[2], la = 0, lb = 0;
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      const float x0 = v[4 * g + 2 * i] * factor, x1 = v[4 * g + 2 * i + 1] * factor;
      const float y0 = v[4 * g + 4 + 2 * i] * factor, y1 = v[4 * g + 5 + 2 * i] * factor;
      a[i] = pack_bf16x2(x0, x1);
      b[i] = pack_bf16x2(y0, y1);
      la |= (uint32_t)(left_over(x0, a[i] & 0xFFFF) | left_over(x1, a[i] >> 16) << 8) << (16 * i);
      lb |= (uint32_t)(left_over(y0, b[i] & 0xFFFF) | left_over(y1, b[i] >> 16) << 8) << (16 * i);
      // lower half: its own and the upper half's part of group g; upper half:
      // both parts of group g + 1
      const auto s = __builtin_amdgcn_permlane32_swap(a[i], b[i], false, false);
      a[i] = s[0];
      b[i] = s[1];
    }
    const int c = 32 * d + 8 * (g + h);
    if (c < D) *(i32x4*)(q + c) = i32x4{(int32_t)a[0], (int32_t)a[1], (int32_t)b[0], (int32_t)b[1]};
    if (low) {
      const auto s = __builtin_amdgcn_permlane32_swap(la, lb, false, false);
      if (c < D) *(uint2*)(low + (int64_t)r * low_ld + c) = make_uint2(s[0], s[1]);
    }
  }
}

// a lane's values of a transposed result (ND blocks), unrounded, to its token's
// row of D floats
template <int ND>
CONCORD_DEV void store_sums(float* row, const f32x16 (&v)[ND], int D, int lane) {
#pragma unroll
  for (int d = 0; d < ND; ++d)
#pragma unroll
    for (int g = 0; g < 4; ++g) {
      const int c = 32 * d + 8 * g;
      if (c < D)
        *(float4*)(row + c + 4 * (lane >> 5)) =
            make_float4(v[d][4 * g], v[d][4 * g + 1], v[d][4 * g + 2], v[d][4 * g + 3]);
    }
}

// ---- sequences -------------------------------------------------------------------
struct AttnSeqs {
  const int32_t *starts, *k_starts;   // NULL: B sequences of equal length
  int64_t TQ, TK;
  int32_t B;
  int32_t per;    // equal lengths: tiles per sequence; else slots of the packed tokens
};

// a tile's sequence: its queries and keys, and the tile's first row among the
// tiled side's (`first` < 0: nothing to do)
struct AttnPlace {
  int64_t q0, k0;    // first token
  int32_t lq, lk;
  int32_t first;
};

// Tiles of TM rows over packed tokens of unknown lengths, without a count from
// the host: with the boundaries e[0] = 0 <= e[1] <= .. (the tokens before the
// first and after the last sequence are sequences too, without keys), sequence
// i owns the slots from e[i] / TM + i on; that gives it at least as many as its
// rows fill, and T / TM + B + 2 in all.  A wave looks 64 boundaries up at a
// time.  Boundaries are clamped to [0, T], so no table reaches past a tensor.
CONCORD_DEV int32_t boundary(const int32_t* s, int B, int64_t T, int i) {
  if (i <= 0) return 0;
  if (i > B + 1) return (int32_t)T;
  const int32_t v = s[i - 1];
  return v < 0 ? 0 : (int64_t)v > T ? (int32_t)T : v;
}
template <int TM, bool KEYS>
CONCORD_DEV AttnPlace attn_place(const AttnSeqs& s, int slot) {
  AttnPlace p;
  if (!s.starts) {
    const int b = slot / s.per;
    p.lq = (int32_t)(s.TQ / s.B);
    p.lk = (int32_t)(s.TK / s.B);
    p.q0 = (int64_t)b * p.lq;
    p.k0 = (int64_t)b * p.lk;
    p.first = (slot - b * s.per) * TM;
    return p;
  }
  const int32_t* tab = KEYS ? s.k_starts : s.starts;
  const int64_t T = KEYS ? s.TK : s.TQ;
  const int lane = threadIdx.x & 63;
  int lo = 0, n = s.B + 2;
  while (n > 1) {
    const int step = (n + 63) / 64;
    const int i = lo + lane * step;
    const bool below = lane * step < n && boundary(tab, s.B, T, i) / TM + i <= slot;
    const int c = __popcll(__builtin_amdgcn_ballot_w64(below));
    const int at = c > 0 ? (c - 1) * step : 0;
    lo += at;
    n = min(n - at, step);
  }
  lo = __builtin_amdgcn_readfirstlane(lo);
  const int32_t e0 = boundary(tab, s.B, T, lo), e1 = boundary(tab, s.B, T, lo + 1);
  p.first = (slot - e0 / TM - lo) * TM;
  // (slots count over e0 / TM of all the tokens: the first tile starts at e0)
  if (p.first < 0 || p.first >= e1 - e0) p.first = -1;
  const bool outside = lo == 0 || lo == s.B + 1;
  const int32_t q0 = boundary(s.starts, s.B, s.TQ, lo), q1 = boundary(s.starts, s.B, s.TQ, lo + 1);
  const int32_t k0 = boundary(s.k_starts, s.B, s.TK, lo), k1 = boundary(s.k_starts, s.B, s.TK, lo + 1);
  p.q0 = q0;
  p.k0 = k0;
  p.lq = outside && KEYS ? 0 : max(q1 - q0, 0);
  p.lk = outside && !KEYS ? 0 : max(k1 - k0, 0);
  return p;
}

// workgroup w -> (slot, query head) or (slot, key head): XCD x takes a
// contiguous range of key-head-major order, so that the tiles of a key head
// share an L2; the last slots first, which under a causal mask have the most
// to do
__host__ __device__ inline int attn_xcd(int w, int total) {
  const int xcd = w % 8, slot = w / 8;
  const int q = total / 8, rem = total % 8;
  return xcd * q + (xcd < rem ? xcd : rem) + slot;
}

// ---- host ------------------------------------------------------------------------
// strides: of a token at least D (a repeated row is no tensor of its own) and
// below 2^24, so that a tile's lane offsets fit 31 bits; multiples of 8, with
// the base on 16 bytes, so that every chunk is one load
inline bool attn_operand(const void* p, int64_t t, int64_t h, int64_t T, int D) {
  return T == 0 || (p && ((uintptr_t)p & 15) == 0 && t % 8 == 0 && h % 8 == 0 && t >= D && t < (1 << 24) && h >= 0);
}

// what the arithmetic on the sizes alone rests on
inline int attn_sizes(const char* what, const concord_attn_args& a) {
  CONCORD_CHECK(a.TQ >= 0 && a.TK >= 0 && a.TQ < (1LL << 31) - 256 && a.TK < (1LL << 31) - 256 && a.B >= 0 &&
                    a.B < (1LL << 24),
                "%s: bad size", what);
  CONCORD_CHECK(a.D >= 8 && a.D <= 128 && a.D % 8 == 0, "%s: the head dimension must be a multiple of 8 up to 128",
                what);
  CONCORD_CHECK(a.H >= 1 && a.HK >= 1 && a.H % a.HK == 0 && a.H < (1 << 16), "%s: H must be a multiple of HK", what);
  CONCORD_CHECK(a.B > 0 || a.starts || (a.TQ == 0 && a.TK == 0), "%s: no sequence", what);
  if (!a.starts) {
    CONCORD_CHECK(!a.k_starts, "%s: k_starts without starts", what);
    CONCORD_CHECK(a.B == 0 || (a.TQ % a.B == 0 && a.TK % a.B == 0), "%s: unequal sequences need starts", what);
  } else {
    CONCORD_CHECK(a.k_starts || a.TQ == a.TK, "%s: k_starts needed where TK differs from TQ", what);
  }
  return CONCORD_OK;
}

inline int attn_check(const char* what, const concord_attn_args& a) {
  if (const int rc = attn_sizes(what, a)) return rc;
  CONCORD_CHECK(a.scale > 0.0f && a.scale < INFINITY, "%s: the scale must be positive", what);
  CONCORD_CHECK(attn_operand(a.q, a.q_t, a.q_h, a.TQ, a.D) && attn_operand(a.out, a.o_t, a.o_h, a.TQ, a.D) &&
                    attn_operand(a.k, a.k_t, a.k_h, a.TK, a.D) && attn_operand(a.v, a.v_t, a.v_h, a.TK, a.D),
                "%s: NULL, misaligned or badly strided argument", what);
  return CONCORD_OK;
}

// tiles of TM rows of T tokens: per sequence (equal lengths) and in all
inline int64_t attn_slots(AttnSeqs& s, int64_t T, int TM) {
  if (s.starts) {
    s.per = 0;
    return T / TM + s.B + 2;
  }
  s.per = (int32_t)cdiv(T / s.B, TM);
  return (int64_t)s.per * s.B;
}

inline AttnSeqs attn_seqs(const concord_attn_args& a) {
  AttnSeqs s{};
  s.starts = a.starts;
  s.k_starts = a.k_starts ? a.k_starts : a.starts;
  s.TQ = a.TQ, s.TK = a.TK, s.B = (int32_t)a.B;
  return s;
}

template <class F>
inline void attn_by_dim(int D, F&& f) {
  if (D <= 32) f(std::integral_constant<int, 2>());
  else if (D <= 64) f(std::integral_constant<int, 4>());
  else if (D <= 96) f(std::integral_constant<int, 6>());
  else f(std::integral_constant<int, 8>());
}

// Shares the keys of a tile of 128 queries are split into (forward and dq; `flops`
// per query-key pair and dimension): where the tiles alone leave CUs idle, as
// many as fill the chip with two (four with heads up to 64) workgroups a CU, of
// four steps of 64 keys at least, while the shares' sums (8 bytes an element)
// stay below a sixth of the launch's time as above (dkv_splits).  One query of
// 32768 keys, 32 / 8 heads of 128: 483 us in one share, 56 + 12 us in 16.
inline int key_splits(const concord_attn_args& g, double flops) {
  if (g.TQ < 1 || g.TK < 1) return 1;
  AttnSeqs s = attn_seqs(g);
  const double wgs = (double)attn_slots(s, g.TQ, 128) * g.H, room = g.D <= 64 ? 1024.0 : 512.0;
  const double keys = (double)g.TK / (double)std::max<int64_t>(g.B, 1);
  const double time = flops * g.TQ * keys * g.H * g.D / 1e15 * std::max(1.0, room / wgs);
  const double share = 8.0 * g.TQ * g.H * g.D / 5e12;
  const double n = std::min(std::min(room / wgs, keys / 256.0), time / 6.0 / share);
  return n < 2.0 ? 1 : n < 64.0 ? (int)n : 64;
}

}  // namespace concord
