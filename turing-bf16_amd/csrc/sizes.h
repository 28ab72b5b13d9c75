// Sizes in units and rounded up; plain C++.
#pragma once
#include <stddef.h>
#include <stdint.h>

namespace tbf16 {

inline int64_t cdiv(int64_t a, int64_t b) { return (a + b - 1) / b; }
inline size_t align_up(size_t v, size_t a) { return (v + a - 1) / a * a; }

}  // namespace tbf16
