// Host build of the tape's exponent rule (tape.cuh).
#include <cuda_runtime.h>

#include "../../ullis_b200/csrc/tape.cuh"

extern "C" void tape_exponent_bytes(const uint32_t* amax_bits, uint8_t* out, size_t n) {
    for (size_t i = 0; i < n; ++i) out[i] = (uint8_t)ullis::tape::exponent_byte(amax_bits[i]);
}
