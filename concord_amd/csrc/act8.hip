// act8.hip -- activations kept in 8 bits from the forward to the backward: the
// form itself (pack, unpack), and gelu and its gated form, whose forward writes
// the input's 8-bit form beside the result and whose backward reads nothing else
// of the forward.
//
//   gelu:   y = x Phi(x) (or its tanh form);   dx = dy f'(z)
//   gated:  y = a f(g), a and g the halves of a row;   da = dy f(gz), dg = dy az f'(gz)
// z, az, gz: the values that the codes stand for.
//
// Bound by memory and instructions alike.  A thread takes 16 bytes of adjacent values at
// a time; four adjacent threads (fp32: eight) hold a block of the 8-bit form, so its
// largest magnitude is two or three lane exchanges away.  Rows that begin on no 16-byte boundary (odd widths) are read and written
// with the same wide accesses at the alignment of one element, which this GPU
// takes; what is left at a row's end goes one by one.
//
// Kernel times, bf16: gelu of 16384 x 1536 23 us forward and 25 backward (127 MB each, 5.4
// and 5.1 TB/s; a 1 GiB copy moves 5.1), the gated form of 8192 x 2560 27 and 29
// (169 MB), pack and unpack of 2048 x 5120 6.3 and 5.8 (31 MB, latencies included).  Odd
// rows, 4099 x 2051 fp16: 12.1 and 13.5 (3.3 TB/s).  fp32, the same sizes: 34 and 38 (227
// MB), gated 48 and 46 (295 MB), odd rows 17.6 and 18 (76 MB, 4.3 TB/s), the tanh form as
// fast: bound by memory, the longer polynomial does not show.  Results go past the caches:
// the gated backward 37 -> 30 us, unpacking 6.6 -> 5.2.
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

// N adjacent elements, on 16 bytes (or their own size) or wherever an element may begin
template <class T, int N, bool ALIGNED>
struct alignas(ALIGNED ? (sizeof(T) * N < 16 ? sizeof(T) * N : 16) : sizeof(T)) Run {
  T v[N];
};

// a result that this kernel does not read again: past the caches, where it lies on its size
template <bool ALIGNED, class V>
CONCORD_DEV void store_wide(void* p, const V& v) {
  if constexpr (!ALIGNED) {
    *(V*)p = v;
  } else if constexpr (sizeof(V) == 4) {
    __builtin_nontemporal_store(__builtin_bit_cast(uint32_t, v), (uint32_t*)p);
  } else if constexpr (sizeof(V) == 8) {
    __builtin_nontemporal_store(__builtin_bit_cast(uint64_t, v), (uint64_t*)p);
  } else {
    store_stream((V*)p, v);
  }
}

// Values that a thread takes at a time: 16 bytes of them, so that a wave's accesses
// leave no gaps (fp32: 4, unpacking 4099 x 1283 took 9.7 us by 8, by 4 it takes 8.0)
template <class T>
constexpr int kWide = 16 / (int)sizeof(T);

// V values of a row as they lie in memory, zeros past its end
template <class T, bool ALIGNED>
struct Values {
  static constexpr int V = kWide<T>;
  typedef Run<T, V, ALIGNED> All;
  All r;
  CONCORD_DEV void load(const T* p, int n) {
    if constexpr (ALIGNED) {   // (all of them or none: p is readable either way)
      r = *(const All*)p;
      if (n < V) r = All{};
      return;
    }
    r = All{};
    if (n >= V) {
      r = *(const All*)p;
    } else {
#pragma unroll
      for (int i = 0; i < V - 1; ++i)
        if (i < n) r.v[i] = p[i];
    }
  }
  CONCORD_DEV void get(float (&v)[V]) const {
#pragma unroll
    for (int i = 0; i < V; ++i) v[i] = to_f32(r.v[i]);
  }
  // bits of the largest magnitude as an fp32 number (above infinity's where there is a NaN)
  CONCORD_DEV uint32_t top() const {
    struct Words {
      uint32_t w[4];
    };
    const Words w = __builtin_bit_cast(Words, r);
    if constexpr (sizeof(T) == 4) {
      return max(max(w.w[0] & 0x7FFFFFFFu, w.w[1] & 0x7FFFFFFFu), max(w.w[2] & 0x7FFFFFFFu, w.w[3] & 0x7FFFFFFFu));
    } else {
      // two values a word: 16-bit numbers without their signs are in order as integers
      typedef uint16_t u16x2 __attribute__((ext_vector_type(2)));
      u16x2 m = {0, 0};
#pragma unroll
      for (int i = 0; i < 4; ++i) m = __builtin_elementwise_max(m, __builtin_bit_cast(u16x2, w.w[i] & 0x7FFF7FFFu));
      return __float_as_uint(to_f32(__builtin_bit_cast(T, max(m.x, m.y))));
    }
  }
  CONCORD_DEV void store(T* p, int n, const float (&v)[V]) {
#pragma unroll
    for (int i = 0; i < V; ++i) r.v[i] = from_f32<T>(v[i]);
    if (n >= V) {
      store_wide<ALIGNED>(p, r);
    } else if (!ALIGNED) {
#pragma unroll
      for (int i = 0; i < V - 1; ++i)
        if (i < n) p[i] = r.v[i];
    }
  }
};

// their codes
template <class T, bool ALIGNED>
struct Codes {
  static constexpr int V = kWide<T>;
  typedef Run<uint8_t, V, ALIGNED> All;
  struct Words {
    uint32_t w[V / 4];
  } c;
  CONCORD_DEV void load(const uint8_t* p, int n) {
    if constexpr (ALIGNED) {
      c = __builtin_bit_cast(Words, *(const All*)p);
      return;
    }
    c = {};
    if (n >= V) {
      c = __builtin_bit_cast(Words, *(const All*)p);
    } else {
#pragma unroll
      for (int i = 0; i < V - 1; ++i)
        if (i < n) c.w[i >> 2] |= (uint32_t)p[i] << (8 * (i & 3));
    }
  }
  CONCORD_DEV void store(uint8_t* p, int n) const {
    if (n >= V) {
      store_wide<ALIGNED>(p, __builtin_bit_cast(All, c));
    } else if (!ALIGNED) {
#pragma unroll
      for (int i = 0; i < V - 1; ++i)
        if (i < n) p[i] = (uint8_t)(c.w[i >> 2] >> (8 * (i & 3)));
    }
  }
};

// A thread's place: V columns from c of a row.  It loads from `at`, which is c or, behind the
// row's end, the row's beginning: no load of aligned rows waits behind a branch, which the
// compiler would not move it over.
struct Place {
  int64_t row, c, at;
  int n;            // columns that the row still has, V for more (0 or less: none)
  uint32_t block;
};
template <int V>
CONCORD_DEV Place place(const Act8Args& a, uint32_t id) {
  constexpr uint32_t EACH = kBlock8 / V;   // threads of a block
  Place p;
  const uint32_t per = a.nb * EACH, row = a.rows == 1 ? 0 : id / per, in = id - row * per;
  p.row = row;
  p.c = (int64_t)in * V;
  p.n = (int)min(a.C - p.c, (int64_t)V);
  p.at = p.n > 0 ? p.c : 0;
  p.block = in / EACH;
  return p;
}

// A block of 256 threads takes K * 256 places, a thread every 256th of them: what a wave
// loads or stores at once lies side by side, and its loads are all out before it waits for
// the first.  f(place) for each place there is.
template <int K, int V, class F>
CONCORD_DEV void each_place(const Act8Args& a, uint32_t count, F&& f) {
#pragma unroll
  for (int k = 0; k < K; ++k) {
    const uint32_t id = (blockIdx.x * K + k) * 256 + threadIdx.x;
    if (id < count) f(k, place<V>(a, id));
  }
}

// one place where its loads are many already (a gated row's two halves) or its rows do
// not begin on 16 bytes
constexpr int places(bool gated, bool aligned) { return gated || !aligned ? 1 : 2; }

// encode the thread's values; the first thread of a block's four or eight writes the exponent
template <class T, bool ALIGNED>
CONCORD_DEV void keep8(const Values<T, ALIGNED>& x, const float (&v)[kWide<T>], const Place& p, uint8_t* codes,
                       uint8_t* exps) {
  constexpr int V = kWide<T>, EACH = kBlock8 / V;
  uint32_t top = x.top();
  top = max(top, (uint32_t)__builtin_amdgcn_update_dpp(0, (int)top, 0xB1, 0xF, 0xF, true));   // quad_perm 1, 0, 3, 2
  top = max(top, (uint32_t)__builtin_amdgcn_update_dpp(0, (int)top, 0x4E, 0xF, 0xF, true));   // quad_perm 2, 3, 0, 1
  if (EACH == 8) top = max(top, (uint32_t)__builtin_amdgcn_update_dpp(0, (int)top, 0x141, 0xF, 0xF, true));   // row_half_mirror
  const uint32_t e8 = exponent8(top);
  const float inv = inverse_step8(e8);
  Codes<T, ALIGNED> c;
#pragma unroll
  for (int i = 0; i < V / 4; ++i) c.c.w[i] = e8 == kBad8 ? 0 : codes8(v + 4 * i, inv);
  c.store(codes + p.c, p.n);
  if ((threadIdx.x & (EACH - 1)) == 0) exps[p.block] = (uint8_t)e8;
}
template <class T, bool ALIGNED>
CONCORD_DEV void kept8(float (&v)[kWide<T>], const Codes<T, ALIGNED>& c, uint32_t e8) {
#pragma unroll
  for (int i = 0; i < kWide<T> / 4; ++i) values8<T>(v + 4 * i, c.c.w[i], e8);
}

template <class T, bool ALIGNED>
__global__ __launch_bounds__(256) void pack8_kernel(Act8Args a, uint32_t count) {
  constexpr int V = kWide<T>, K = places(false, ALIGNED);
  Values<T, ALIGNED> x[K];
  each_place<K, V>(a, count, [&](int k, const Place& p) { x[k].load((const T*)a.x + p.row * a.ldx + p.at, p.n); });
  each_place<K, V>(a, count, [&](int k, const Place& p) {
    float v[V];
    x[k].get(v);
    keep8(x[k], v, p, a.codes + p.row * a.C, a.exps + p.row * a.nb);
  });
}

template <class T, bool ALIGNED>
__global__ __launch_bounds__(256) void unpack8_kernel(Act8Args a, uint32_t count) {
  constexpr int V = kWide<T>, K = places(false, ALIGNED);
  Codes<T, ALIGNED> c[K];
  uint32_t e8[K];
  each_place<K, V>(a, count, [&](int k, const Place& p) {
    c[k].load(a.codes + p.row * a.C + p.at, p.n);
    e8[k] = a.exps[p.row * a.nb + p.block];
  });
  each_place<K, V>(a, count, [&](int k, const Place& p) {
    float v[V];
    kept8(v, c[k], e8[k]);
    Values<T, ALIGNED> x;
    x.store((T*)a.out + p.row * a.ldo + p.c, p.n, v);
  });
}

template <class T, class F, bool GATED, bool ALIGNED>
__global__ __launch_bounds__(256) void gelu8_fwd_kernel(Act8Args a, uint32_t count) {
  constexpr int V = kWide<T>, K = places(GATED, ALIGNED);
  Values<T, ALIGNED> x[K], g[K];
  each_place<K, V>(a, count, [&](int k, const Place& p) {
    const T* at = (const T*)a.x + p.row * a.ldx + p.at;
    x[k].load(at, p.n);
    if (GATED) g[k].load(at + a.C, p.n);
  });
  each_place<K, V>(a, count, [&](int k, const Place& p) {
    float v[V], w[V], y[V];
    x[k].get(v);
    const int wide = GATED ? 2 : 1;
    uint8_t *codes = a.codes + p.row * wide * a.C, *exps = a.exps + p.row * wide * a.nb;
    if (a.codes) keep8(x[k], v, p, codes, exps);
    if (GATED) {
      g[k].get(w);
      if (a.codes) keep8(g[k], w, p, codes + a.C, exps + a.nb);
    }
#pragma unroll
    for (int i = 0; i < V; ++i) y[i] = GATED ? v[i] * F::value(w[i]) : F::value(v[i]);
    x[k].store((T*)a.out + p.row * a.ldo + p.c, p.n, y);
  });
}

template <class T, class F, bool GATED, bool ALIGNED>
__global__ __launch_bounds__(256) void gelu8_bwd_kernel(Act8Args a, uint32_t count) {
  constexpr int V = kWide<T>, K = places(GATED, ALIGNED);
  Values<T, ALIGNED> r[K];
  Codes<T, ALIGNED> c[K], cg[K];
  uint32_t e8[K], eg[K];
  each_place<K, V>(a, count, [&](int k, const Place& p) {
    const int wide = GATED ? 2 : 1;
    const uint8_t *codes = a.codes + p.row * wide * a.C + p.at, *exps = a.exps + p.row * wide * a.nb + p.block;
    r[k].load((const T*)a.dy + p.row * a.lddy + p.at, p.n);
    c[k].load(codes, p.n);
    e8[k] = exps[0];
    if (GATED) {
      cg[k].load(codes + a.C, p.n);
      eg[k] = exps[a.nb];
    }
  });
  each_place<K, V>(a, count, [&](int k, const Place& p) {
    float dy[V], z[V];
    T* out = (T*)a.out + p.row * a.ldo + p.c;
    r[k].get(dy);
    kept8(z, c[k], e8[k]);
    if (GATED) {
      float g[V];
      kept8(g, cg[k], eg[k]);
#pragma unroll
      for (int i = 0; i < V; ++i) {
        float v, d;
        F::both(g[i], v, d);
        g[i] = dy[i] * d * z[i];   // (|d| < 1.13: only the whole product can overflow)
        z[i] = dy[i] * v;
      }
      r[k].store(out, p.n, z);
      r[k].store(out + a.C, p.n, g);
    } else {
#pragma unroll
      for (int i = 0; i < V; ++i) z[i] = dy[i] * F::slope(z[i]);
      r[k].store(out, p.n, z);
    }
  });
}

// ---- host -------------------------------------------------------------------
enum Act8Pass { kPack8, kUnpack8, kFwd8, kBwd8 };

// threads' places, those behind a row's end included; -1: too many for a launch
static int64_t act8_count(int dtype, int64_t rows, int64_t C) {
  const int64_t nb = cdiv(C, kBlock8), each = dtype == CONCORD_F32 ? 8 : 4;
  return rows > ((1LL << 32) - 4096) / each / nb ? -1 : rows * nb * each;
}

template <class T, class F, bool GATED, bool ALIGNED>
static void act8_launch(Act8Pass pass, const Act8Args& a, uint32_t count, hipStream_t st) {
  const dim3 grid((unsigned)cdiv(count, 256 * places(GATED, ALIGNED))), th(256);
  if (pass == kPack8) hipLaunchKernelGGL((pack8_kernel<T, ALIGNED>), grid, th, 0, st, a, count);
  else if (pass == kUnpack8) hipLaunchKernelGGL((unpack8_kernel<T, ALIGNED>), grid, th, 0, st, a, count);
  else if (pass == kFwd8) hipLaunchKernelGGL((gelu8_fwd_kernel<T, F, GATED, ALIGNED>), grid, th, 0, st, a, count);
  else hipLaunchKernelGGL((gelu8_bwd_kernel<T, F, GATED, ALIGNED>), grid, th, 0, st, a, count);
}

static bool act8_on16(const void* p, int64_t ld, size_t es) { return ((uintptr_t)p & 15) == 0 && ld * es % 16 == 0; }

template <class T, class F, bool GATED>
static void act8_rows(Act8Pass pass, const Act8Args& a, uint32_t count, hipStream_t st) {
  const size_t es = sizeof(T);
  const bool aligned = a.C % kWide<T> == 0 && (!a.x || act8_on16(a.x, a.ldx, es)) && (!a.dy || act8_on16(a.dy, a.lddy, es)) &&
                       (!a.out || act8_on16(a.out, a.ldo, es)) && ((uintptr_t)a.codes & (kWide<T> - 1)) == 0;
  if (aligned) act8_launch<T, F, GATED, true>(pass, a, count, st);
  else act8_launch<T, F, GATED, false>(pass, a, count, st);
}
template <class T>
static void act8_form(Act8Pass pass, const Act8Args& a, uint32_t count, bool tanh, bool gated, hipStream_t st) {
  constexpr bool FINE = sizeof(T) == 4;
  if (gated) {
    if (tanh) act8_rows<T, GeluTanh<FINE>, true>(pass, a, count, st);
    else act8_rows<T, Gelu<FINE>, true>(pass, a, count, st);
  } else {
    if (tanh) act8_rows<T, GeluTanh<FINE>, false>(pass, a, count, st);
    else act8_rows<T, Gelu<FINE>, false>(pass, a, count, st);
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
  const uint32_t count = (uint32_t)act8_count(dtype, a.rows, a.C);
  if (dtype == CONCORD_F32) act8_form<float>(pass, a, count, tanh, gated, st);
  else if (dtype == CONCORD_BF16) act8_form<BF16>(pass, a, count, tanh, gated, st);
  else act8_form<_Float16>(pass, a, count, tanh, gated, st);
}

static int act8_check(const char* name, int dtype, int64_t rows, int64_t C) {
  CONCORD_CHECK(rows >= 0 && C >= 1 && rows < (1LL << 40) && C < (1LL << 40), "%s: bad size", name);
  CONCORD_CHECK(dtype == CONCORD_F32 || dtype == CONCORD_BF16 || dtype == CONCORD_F16, "%s: bad type", name);
  CONCORD_CHECK(act8_count(dtype, rows, C) >= 0, "%s: too many values for a launch", name);
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
