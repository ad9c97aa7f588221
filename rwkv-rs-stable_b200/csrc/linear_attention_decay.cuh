// The factor by which the kernels of linear attention scale a state again and again: a power of the decay, which is hardly ever an fp32 number.
#pragma once

#include <cuda_runtime.h>

#include <cmath>
#include <cstdint>

namespace rwkv7 {

// The rounded power, taken 256 times over a long memory, would be off 256 times the same way (by up to 3e-8 of a state, and as expf gives it by more:
// 1.6e-5 after 256 chunks).  So it is rounded now down, now up, each as often as the power lies near it: the product of any number of factors in a row
// is off by one step of one factor.
// (The part that rounding took could be multiplied as well, at an instruction more for each two elements, and as 0 x inf or inf - inf it would make
// an infinite element NaN.)  Nothing is carried from factor to factor but their number, so that it may stand in shared memory.
struct SteadyPower {
    float down, up;      // the power's neighbours
    uint32_t up_part;    // how much of the way from one to the other it lies on, in 2^-32

    SteadyPower() = default;
    __device__ __forceinline__ explicit SteadyPower(double power) {
        down = __double2float_rd(power);
        up = __double2float_ru(power);
        up_part = 0;
        if (up == INFINITY) down = INFINITY;   // (nothing to choose from)
        else if (up > down) up_part = __float2uint_rz((float)(power - (double)down) / (up - down) * 4294967296.f);
    }
    // The k-th factor: of k the first k up_part + 1/2, rounded down, are `up`.
    __device__ __forceinline__ float factor(uint32_t k) const {
        const uint32_t before = 0x80000000u + k * up_part;
        return before + up_part < before ? up : down;   // (carried)
    }
};

}  // namespace rwkv7
