// The paged cache of 4 bits: what its store and its attention share.
//
// A head's vector of a token is lo + step * code, codes 0 to 15, lo and step bfloat16, one pair for the D elements:
//   lo = bf16(min), step = bf16((max - lo) / 15), code = clamp(rint((x - lo) / step), 0, 15), 0 where step is not positive.
// A vector with anything not finite (or whose range is beyond float32) is held as lo = NaN, step = 0: all of it reads NaN.
//
// Of every page and head, 4 <= page_size, a multiple of 4:
//   keys    [offset, D / 2] bytes: element 2 i in the low half of byte i, 2 i + 1 in the high one;
//   values  by fours of tokens [offset / 4, 16, D / 32, 4]: byte (c, w, j) is token j's elements 32 w + c (low) and 32 w + 16 + c;
//   steps   [offset, 4] bfloat16: the key's lo and step, the value's.
// A lane of the attention reads D / 8 neighbouring bytes for 16 keys either way: of the keys the quarter of one key's elements
// that its operand takes, of the values all 16-wide tiles of one element for four keys, so that neither operand crosses lanes.
#pragma once
#include "common.h"

struct PageMagic {  // division of numbers below 2^31 by the page size, or the like, without dividing
  unsigned size, by;
};
inline PageMagic page_magic(int size) {
  return {(unsigned)size, size == 1 ? ~0u : (unsigned)(((1ull << 32) + size - 1) / size)};
}
__device__ __forceinline__ void page_of(PageMagic m, int key, int& page, int& offset) {
  unsigned q = __umulhi((unsigned)key, m.by);  // one too many at most; by 1, one too few at most
  int r = key - (int)(q * m.size);
  if (r < 0) r += m.size, --q;
  if (r >= (int)m.size) r -= m.size, ++q;
  page = (int)q, offset = r;
}
