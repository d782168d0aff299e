// act8.hip -- activations kept in 8 bits from the forward to the backward: the
// form itself (pack, unpack), and gelu and its gated form, whose forward writes
// the input's 8-bit form beside the result and whose backward reads nothing else
// of the forward.
//
//   gelu:   y = x Phi(x) (or its tanh form);   dx = dy f'(z)
//   gated:  y = a f(g), a and g the halves of a row;   da = dy f(gz), dg = dy az f'(gz)
// z, az, gz: the values that the codes stand for.
//
// Bound by memory.  A thread takes 8 adjacent values; the four threads of a quad
// hold a block of the 8-bit form, so its largest magnitude is two lane exchanges
// away.  Rows that begin on no 16-byte boundary (odd widths) are read and written
// with the same wide accesses at the alignment of one element, which this GPU
// takes; a row's last 1 to 7 values go one by one.
#include "act8.h"

namespace concord {

struct Act8Args {
  const void* x;        // forward, pack
  int64_t ldx;
  const void* dy;       // backward
  int64_t lddy;
  void* out;            // y, dx or the unpacked values
  int64_t ldo;
  uint8_t* codes;       // [rows][C], or [rows][2 C]
  uint8_t* exps;        // [rows][nb], or [rows][2][nb]
  int64_t rows, C;      // C: columns of the result
  uint32_t nb;          // blocks of C columns
};

template <class T, bool ALIGNED>
struct alignas(ALIGNED ? sizeof(T) * 8 < 16 ? sizeof(T) * 8 : 16 : sizeof(T)) Eight {
  T v[8];
};

template <class T, bool ALIGNED>
CONCORD_DEV void load8(float (&v)[8], const T* p, int64_t n) {
  typedef Eight<T, ALIGNED> E;
  E r = {};
  if (n >= 8) {
    r = *(const E*)p;
  } else if (!ALIGNED) {
#pragma unroll
    for (int i = 0; i < 7; ++i)
      if (i < n) r.v[i] = p[i];
  }
#pragma unroll
  for (int i = 0; i < 8; ++i) v[i] = to_f32(r.v[i]);
}
template <class T, bool ALIGNED>
CONCORD_DEV void store8(T* p, int64_t n, const float (&v)[8]) {
  typedef Eight<T, ALIGNED> E;
  E r;
#pragma unroll
  for (int i = 0; i < 8; ++i) r.v[i] = from_f32<T>(v[i]);
  if (n >= 8) {
    *(E*)p = r;
  } else if (!ALIGNED) {
#pragma unroll
    for (int i = 0; i < 7; ++i)
      if (i < n) p[i] = r.v[i];
  }
}
template <bool ALIGNED>
CONCORD_DEV void store_codes(uint8_t* p, int64_t n, uint32_t lo, uint32_t hi) {
  typedef Eight<uint8_t, ALIGNED> E;
  if (n >= 8) {
    *(E*)p = __builtin_bit_cast(E, (uint64_t)hi << 32 | lo);
  } else if (!ALIGNED) {
#pragma unroll
    for (int i = 0; i < 7; ++i)
      if (i < n) p[i] = (uint8_t)((i < 4 ? lo : hi) >> (8 * (i & 3)));
  }
}
template <bool ALIGNED>
CONCORD_DEV void load_codes(const uint8_t* p, int64_t n, uint32_t& lo, uint32_t& hi) {
  typedef Eight<uint8_t, ALIGNED> E;
  lo = hi = 0;
  if (n >= 8) {
    const uint64_t w = __builtin_bit_cast(uint64_t, *(const E*)p);
    lo = (uint32_t)w, hi = (uint32_t)(w >> 32);
  } else if (!ALIGNED) {
#pragma unroll
    for (int i = 0; i < 7; ++i)
      if (i < n) (i < 4 ? lo : hi) |= (uint32_t)p[i] << (8 * (i & 3));
  }
}

// the thread's place: eight columns from c of a row
struct Place8 {
  int64_t row, c, n;   // n: columns that the row still has (0 or less: none)
  uint32_t block;
};
template <class T>
CONCORD_DEV Place8 place8(const Act8Args& a, uint32_t id) {
  Place8 p;
  const uint32_t per = a.nb * 4, row = id / per, in = id - row * per;
  p.row = row;
  p.c = (int64_t)in * 8;
  p.n = a.C - p.c;
  p.block = in >> 2;
  return p;
}

// encode the thread's eight values; the quad's first thread writes the exponent
template <bool ALIGNED>
CONCORD_DEV void keep8(const float (&v)[8], const Place8& p, uint8_t* codes, uint8_t* exps) {
  uint32_t top = 0;
#pragma unroll
  for (int i = 0; i < 8; ++i) top = max(top, abs_bits(v[i]));
  top = max(top, (uint32_t)__builtin_amdgcn_update_dpp(0, (int)top, 0xB1, 0xF, 0xF, true));   // quad_perm 1, 0, 3, 2
  top = max(top, (uint32_t)__builtin_amdgcn_update_dpp(0, (int)top, 0x4E, 0xF, 0xF, true));   // quad_perm 2, 3, 0, 1
  const uint32_t e8 = exponent8(top);
  const float inv = inverse_step8(e8);
  store_codes<ALIGNED>(codes + p.c, p.n, codes8(v, inv, e8 == kBad8), codes8(v + 4, inv, e8 == kBad8));
  if ((threadIdx.x & 3) == 0) exps[p.block] = (uint8_t)e8;
}
template <class T, bool ALIGNED>
CONCORD_DEV void kept8(float (&v)[8], const Place8& p, const uint8_t* codes, const uint8_t* exps) {
  uint32_t lo, hi;
  load_codes<ALIGNED>(codes + p.c, p.n, lo, hi);
  const uint32_t e8 = exps[p.block];
  const float step = step8(e8);
  const bool large = e8 >= Largest<T>::e8;
#pragma unroll
  for (int i = 0; i < 8; ++i) v[i] = value8<T>(__builtin_amdgcn_sbfe((int)(i < 4 ? lo : hi), 8 * (i & 3), 8), step, large);
}

template <class T, bool ALIGNED>
__global__ __launch_bounds__(256) void pack8_kernel(Act8Args a, uint32_t count) {
  const uint32_t id = blockIdx.x * 256 + threadIdx.x;
  if (id >= count) return;
  const Place8 p = place8<T>(a, id);
  float v[8];
  load8<T, ALIGNED>(v, (const T*)a.x + p.row * a.ldx + p.c, p.n);
  keep8<ALIGNED>(v, p, a.codes + p.row * a.C, a.exps + p.row * a.nb);
}

template <class T, bool ALIGNED>
__global__ __launch_bounds__(256) void unpack8_kernel(Act8Args a, uint32_t count) {
  const uint32_t id = blockIdx.x * 256 + threadIdx.x;
  if (id >= count) return;
  const Place8 p = place8<T>(a, id);
  float v[8];
  kept8<T, ALIGNED>(v, p, a.codes + p.row * a.C, a.exps + p.row * a.nb);
  store8<T, ALIGNED>((T*)a.out + p.row * a.ldo + p.c, p.n, v);
}

template <class T, class F, bool GATED, bool ALIGNED>
__global__ __launch_bounds__(256) void gelu8_fwd_kernel(Act8Args a, uint32_t count) {
  const uint32_t id = blockIdx.x * 256 + threadIdx.x;
  if (id >= count) return;
  const Place8 p = place8<T>(a, id);
  const T* x = (const T*)a.x + p.row * a.ldx + p.c;
  float v[8], y[8];
  if (GATED) {
    float g[8];
    load8<T, ALIGNED>(v, x, p.n);
    load8<T, ALIGNED>(g, x + a.C, p.n);
#pragma unroll
    for (int i = 0; i < 8; ++i) y[i] = v[i] * F::value(g[i]);
    if (a.codes) {
      uint8_t *codes = a.codes + p.row * 2 * a.C, *exps = a.exps + p.row * 2 * a.nb;
      keep8<ALIGNED>(v, p, codes, exps);
      keep8<ALIGNED>(g, p, codes + a.C, exps + a.nb);
    }
  } else {
    load8<T, ALIGNED>(v, x, p.n);
#pragma unroll
    for (int i = 0; i < 8; ++i) y[i] = F::value(v[i]);
    if (a.codes) keep8<ALIGNED>(v, p, a.codes + p.row * a.C, a.exps + p.row * a.nb);
  }
  store8<T, ALIGNED>((T*)a.out + p.row * a.ldo + p.c, p.n, y);
}

template <class T, class F, bool GATED, bool ALIGNED>
__global__ __launch_bounds__(256) void gelu8_bwd_kernel(Act8Args a, uint32_t count) {
  const uint32_t id = blockIdx.x * 256 + threadIdx.x;
  if (id >= count) return;
  const Place8 p = place8<T>(a, id);
  float dy[8], z[8];
  load8<T, ALIGNED>(dy, (const T*)a.dy + p.row * a.lddy + p.c, p.n);
  T* out = (T*)a.out + p.row * a.ldo + p.c;
  if (GATED) {
    const uint8_t *codes = a.codes + p.row * 2 * a.C, *exps = a.exps + p.row * 2 * a.nb;
    float g[8];
    kept8<T, ALIGNED>(z, p, codes, exps);
    kept8<T, ALIGNED>(g, p, codes + a.C, exps + a.nb);
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      float v, d;
      F::both(g[i], v, d);
      g[i] = dy[i] * z[i] * d;
      z[i] = dy[i] * v;
    }
    store8<T, ALIGNED>(out, p.n, z);
    store8<T, ALIGNED>(out + a.C, p.n, g);
  } else {
    kept8<T, ALIGNED>(z, p, a.codes + p.row * a.C, a.exps + p.row * a.nb);
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      float v, d;
      F::both(z[i], v, d);
      z[i] = dy[i] * d;
    }
    store8<T, ALIGNED>(out, p.n, z);
  }
}

// ---- host -------------------------------------------------------------------
enum Act8Pass { kPack8, kUnpack8, kFwd8, kBwd8 };

// eight-value places, those behind a row's end included; -1: too many for a launch
static int64_t act8_count(int64_t rows, int64_t C) {
  const int64_t nb = cdiv(C, kBlock8);
  return rows > ((1LL << 32) - 256) / 4 / nb ? -1 : rows * nb * 4;
}

template <class T, class F, bool GATED, bool ALIGNED>
static void act8_launch(Act8Pass pass, const Act8Args& a, uint32_t count, hipStream_t st) {
  const dim3 grid((unsigned)cdiv(count, 256)), th(256);
  if (pass == kPack8) hipLaunchKernelGGL((pack8_kernel<T, ALIGNED>), grid, th, 0, st, a, count);
  else if (pass == kUnpack8) hipLaunchKernelGGL((unpack8_kernel<T, ALIGNED>), grid, th, 0, st, a, count);
  else if (pass == kFwd8) hipLaunchKernelGGL((gelu8_fwd_kernel<T, F, GATED, ALIGNED>), grid, th, 0, st, a, count);
  else hipLaunchKernelGGL((gelu8_bwd_kernel<T, F, GATED, ALIGNED>), grid, th, 0, st, a, count);
}

static bool act8_on16(const void* p, int64_t ld, size_t es) { return ((uintptr_t)p & 15) == 0 && ld * es % 16 == 0; }

template <class T, class F, bool GATED>
static void act8_rows(Act8Pass pass, const Act8Args& a, uint32_t count, hipStream_t st) {
  const size_t es = sizeof(T);
  const bool aligned = a.C % 8 == 0 && (!a.x || act8_on16(a.x, a.ldx, es)) && (!a.dy || act8_on16(a.dy, a.lddy, es)) &&
                       (!a.out || act8_on16(a.out, a.ldo, es)) && ((uintptr_t)a.codes & 7) == 0;
  if (aligned) act8_launch<T, F, GATED, true>(pass, a, count, st);
  else act8_launch<T, F, GATED, false>(pass, a, count, st);
}
template <class T>
static void act8_form(Act8Pass pass, const Act8Args& a, uint32_t count, bool tanh, bool gated, hipStream_t st) {
  if (gated) {
    if (tanh) act8_rows<T, GeluTanh, true>(pass, a, count, st);
    else act8_rows<T, Gelu, true>(pass, a, count, st);
  } else {
    if (tanh) act8_rows<T, GeluTanh, false>(pass, a, count, st);
    else act8_rows<T, Gelu, false>(pass, a, count, st);
  }
}
static void act8_run(Act8Pass pass, int dtype, Act8Args a, bool tanh, bool gated, hipStream_t st) {
  // rows one after another in whole blocks are one long row
  if (!gated && a.C % kBlock8 == 0 && (!a.x || a.ldx == a.C) && (!a.dy || a.lddy == a.C) && (!a.out || a.ldo == a.C)) {
    a.C *= a.rows;
    a.rows = 1;
    a.ldx = a.lddy = a.ldo = a.C;
  }
  a.nb = (uint32_t)cdiv(a.C, kBlock8);
  const uint32_t count = (uint32_t)act8_count(a.rows, a.C);
  if (dtype == CONCORD_F32) act8_form<float>(pass, a, count, tanh, gated, st);
  else if (dtype == CONCORD_BF16) act8_form<BF16>(pass, a, count, tanh, gated, st);
  else act8_form<_Float16>(pass, a, count, tanh, gated, st);
}

static int act8_check(const char* name, int dtype, int64_t rows, int64_t C) {
  CONCORD_CHECK(rows >= 0 && C >= 1 && rows < (1LL << 40) && C < (1LL << 40), "%s: bad size", name);
  CONCORD_CHECK(dtype == CONCORD_F32 || dtype == CONCORD_BF16 || dtype == CONCORD_F16, "%s: bad type", name);
  CONCORD_CHECK(act8_count(rows, C) >= 0, "%s: too many values for a launch", name);
  return CONCORD_OK;
}

}  // namespace concord

using namespace concord;

extern "C" int concord_pack8(const void* x, int64_t ld_x, int dtype, int64_t rows, int64_t C, int8_t* codes,
                             uint8_t* exponents, void* stream) {
  if (const int rc = act8_check("concord_pack8", dtype, rows, C)) return rc;
  CONCORD_CHECK(ld_x >= C, "concord_pack8: leading dimension < C");
  if (rows == 0) return CONCORD_OK;
  CONCORD_CHECK(x && codes && exponents, "concord_pack8: NULL argument");
  Act8Args a{};
  a.x = x, a.ldx = ld_x, a.codes = (uint8_t*)codes, a.exps = exponents, a.rows = rows, a.C = C;
  act8_run(kPack8, dtype, a, false, false, (hipStream_t)stream);
  return launch_status("pack8");
}

extern "C" int concord_unpack8(const int8_t* codes, const uint8_t* exponents, int64_t rows, int64_t C, void* x, int64_t ld_x,
                               int dtype, void* stream) {
  if (const int rc = act8_check("concord_unpack8", dtype, rows, C)) return rc;
  CONCORD_CHECK(ld_x >= C, "concord_unpack8: leading dimension < C");
  if (rows == 0) return CONCORD_OK;
  CONCORD_CHECK(x && codes && exponents, "concord_unpack8: NULL argument");
  Act8Args a{};
  a.out = x, a.ldo = ld_x, a.codes = (uint8_t*)codes, a.exps = (uint8_t*)exponents, a.rows = rows, a.C = C;
  act8_run(kUnpack8, dtype, a, false, false, (hipStream_t)stream);
  return launch_status("unpack8");
}

extern "C" int concord_gelu8_fwd(const void* x, int64_t ld_x, int dtype, int64_t rows, int64_t C, int gated, int tanh_form,
                                 void* y, int64_t ld_y, int8_t* codes, uint8_t* exponents, void* stream) {
  if (const int rc = act8_check("concord_gelu8_fwd", dtype, rows, C)) return rc;
  CONCORD_CHECK(ld_x >= (gated ? 2 * C : C) && ld_y >= C, "concord_gelu8_fwd: leading dimension < C");
  CONCORD_CHECK(!codes == !exponents, "concord_gelu8_fwd: codes without exponents");
  if (rows == 0) return CONCORD_OK;
  CONCORD_CHECK(x && y, "concord_gelu8_fwd: NULL argument");
  Act8Args a{};
  a.x = x, a.ldx = ld_x, a.out = y, a.ldo = ld_y, a.codes = (uint8_t*)codes, a.exps = exponents, a.rows = rows, a.C = C;
  act8_run(kFwd8, dtype, a, tanh_form != 0, gated != 0, (hipStream_t)stream);
  return launch_status("gelu8_fwd");
}

extern "C" int concord_gelu8_bwd(const void* dy, int64_t ld_dy, const int8_t* codes, const uint8_t* exponents, int dtype,
                                 int64_t rows, int64_t C, int gated, int tanh_form, void* dx, int64_t ld_dx, void* stream) {
  if (const int rc = act8_check("concord_gelu8_bwd", dtype, rows, C)) return rc;
  CONCORD_CHECK(ld_dx >= (gated ? 2 * C : C) && ld_dy >= C, "concord_gelu8_bwd: leading dimension < C");
  if (rows == 0) return CONCORD_OK;
  CONCORD_CHECK(dy && codes && exponents && dx, "concord_gelu8_bwd: NULL argument");
  Act8Args a{};
  a.dy = dy, a.lddy = ld_dy, a.out = dx, a.ldo = ld_dx, a.codes = (uint8_t*)codes, a.exps = (uint8_t*)exponents;
  a.rows = rows, a.C = C;
  act8_run(kBwd8, dtype, a, tanh_form != 0, gated != 0, (hipStream_t)stream);
  return launch_status("gelu8_bwd");
}
