// The bytes from the first to the last of a [rows][stride] block of `width` elements, to refuse calls whose output lies over an input.
#pragma once
#include <stdint.h>

namespace hps {

struct Span {
  uint64_t lo = 0, hi = 0;   // hi 0: nothing
  Span(const void* p, uint64_t rows, uint64_t stride, uint64_t width, uint64_t bytes) {
    if (!p || rows == 0 || width == 0) return;
    lo = (uint64_t)(uintptr_t)p;
    const unsigned __int128 end = lo + ((unsigned __int128)(rows - 1) * stride + width) * bytes;
    hi = end > UINT64_MAX ? UINT64_MAX : (uint64_t)end;
  }
  bool meets(const Span& o) const { return hi != 0 && o.hi != 0 && lo < o.hi && o.lo < hi; }
};

}  // namespace hps
