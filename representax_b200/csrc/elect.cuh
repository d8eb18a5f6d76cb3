// Warp-uniform issue of tensor-core instructions.
#pragma once
#include <stdint.h>

namespace rx {

// One lane of a converged warp, the same one each time. Code that a whole warp runs with only the
// tensor-core instructions under this predicate keeps their operands in uniform registers; under
// `lane == 0` around the whole loop every operand is moved there again for each instruction.
__device__ __forceinline__ bool elect_one() {
  uint32_t p;
  asm volatile("{\n\t.reg .pred q;\n\telect.sync _|q, 0xffffffff;\n\tselp.b32 %0, 1, 0, q;\n\t}" : "=r"(p));
  return p != 0;
}

}  // namespace rx
