// act8_host.cpp -- the 8-bit form of csrc/act8.h on the host: a copy of that header is
// compiled beside the elem.h that elem_host() of test_act8_host.py writes, whose
// stand-ins for the GPU's builtins do the same arithmetic.
#include "act8.h"

using namespace concord;

template <class T>
static void decode(uint32_t e8, const uint32_t* words, float* out) {
  for (int i = 0; i < 64; ++i) values8<T>(out + 4 * i, words[i], e8);
}

// the 256 codes (64 words of four) as values of type 0 (fp32), 1 (bf16) or 2 (fp16)
extern "C" void decode8(int type, uint32_t e8, const uint32_t* words, float* out) {
  if (type == 0) decode<float>(e8, words, out);
  else if (type == 1) decode<BF16>(e8, words, out);
  else decode<_Float16>(e8, words, out);
}

// four values to codes; returns the exponent byte for a largest magnitude of `top`
extern "C" uint32_t encode8(const float* x, float top, uint32_t* word) {
  const uint32_t e8 = exponent8(__float_as_uint(top));
  *word = e8 == kBad8 ? 0 : codes8(x, inverse_step8(e8));
  return e8;
}
