"""The 8-bit form's arithmetic (csrc/act8.h), compiled for the host and compared with
exact arithmetic over every code and exponent byte."""
import ctypes
import os
import shutil
import subprocess

import numpy as np
import pytest

HERE = os.path.dirname(os.path.abspath(__file__))
ACT8 = os.path.join(os.path.dirname(HERE), "concord_amd", "csrc", "act8.h")

# what act8.h takes from elem.h and from the compiler's GPU target
ELEM = """
#pragma once
#include <math.h>
#include <stdint.h>
#include <string.h>
#include <algorithm>
using std::max;
#define CONCORD_DEV inline
#define _Float16 HostHalf   // (a name for the type alone: the values are fp32 here)
struct HostHalf {};
namespace concord {
struct BF16 {};
}
inline float __uint_as_float(uint32_t u) { float f; memcpy(&f, &u, 4); return f; }
inline uint32_t __float_as_uint(float f) { uint32_t u; memcpy(&u, &f, 4); return u; }
inline int sbfe_host(uint32_t w, int at, int bits) { return (int)(w << (32 - at - bits)) >> (32 - bits); }
inline uint32_t perm_host(uint32_t a, uint32_t b, uint32_t sel) {
  const uint64_t both = (uint64_t)a << 32 | b;
  uint32_t r = 0;
  for (int i = 0; i < 4; ++i) {
    const uint32_t s = sel >> (8 * i) & 0xFF;
    r |= (s == 0x0C ? 0u : (uint32_t)(both >> (8 * s)) & 0xFF) << (8 * i);
  }
  return r;
}
#define __builtin_amdgcn_sbfe sbfe_host
#define __builtin_amdgcn_perm perm_host
#define __builtin_amdgcn_exp2f exp2f
#define __builtin_amdgcn_rcpf(x) (1.0f / (x))
"""


@pytest.fixture(scope="module")
def act8(tmp_path_factory):
    from concord_amd import build as B
    d = str(tmp_path_factory.mktemp("act8_host"))
    shutil.copy(ACT8, d)
    with open(os.path.join(d, "elem.h"), "w") as f:
        f.write(ELEM)
    out = os.path.join(d, "act8_host.so")
    r = subprocess.run([B.CXX, "-O1", "-std=c++17", "-ffp-contract=off", "-fPIC", "-shared", "-w", "-I" + d, "-o", out,
                        os.path.join(HERE, "act8_host.cpp")], capture_output=True, text=True)
    assert r.returncode == 0, r.stderr[-4000:]
    lib = ctypes.CDLL(out)
    lib.decode8.argtypes = [ctypes.c_int, ctypes.c_uint32, ctypes.c_void_p, ctypes.c_void_p]
    lib.encode8.argtypes = [ctypes.c_void_p, ctypes.c_float, ctypes.c_void_p]
    lib.encode8.restype = ctypes.c_uint32
    return lib


MOST = [np.finfo(np.float32).max, 255.0 * 2.0 ** 120, 65504.0]   # fp32, bf16, fp16


@pytest.mark.parametrize("kind", [0, 1, 2])
def test_every_code_of_every_exponent(act8, kind):
    """code 2^(byte - 127), limited to the type's largest number: exact, so no tolerance"""
    codes = np.arange(-128, 128).astype(np.int8)
    got = np.empty(256, np.float32)
    for e8 in range(1, 250):
        act8.decode8(kind, e8, codes.ctypes.data, got.ctypes.data)
        want = np.clip(codes.astype(np.float64) * 2.0 ** (e8 - 127), -MOST[kind], MOST[kind])
        assert np.array_equal(got.astype(np.float64), want), (e8, got[got != want][:4], want[got != want][:4])
    act8.decode8(kind, 255, codes.ctypes.data, got.ctypes.data)
    assert np.isnan(got[codes == 0]).all()   # (a block of byte 255 has codes 0)


@pytest.mark.parametrize("top", [2.0 ** 127, 2e38, 127 * 2.0 ** 121, 127.5 * 2.0 ** 121, 2.0 ** 126, 127 * 2.0 ** 120,
                                 1.0, 127 / 64, 127.5 / 64, 2.0 ** -120, 2.0 ** -126, 2.0 ** -140])
def test_there_and_back(act8, top):
    """off by half a step at most, the small values of a large block among them"""
    top = float(np.float32(top))
    x = np.array([top, -top / 3, top / 200, 0.0], np.float32)
    word = np.zeros(1, np.uint32)
    e8 = act8.encode8(x.ctypes.data, top, word.ctypes.data)
    step = 2.0 ** (e8 - 127)
    assert 1 <= e8 <= 249 and top <= 127 * step and (e8 == 1 or top > 127 * step / 2)
    words, got = np.full(64, word[0], np.uint32), np.empty(256, np.float32)
    act8.decode8(0, e8, words.ctypes.data, got.ctypes.data)
    assert (np.abs(got[:4].astype(np.float64) - x) <= step / 2).all()
