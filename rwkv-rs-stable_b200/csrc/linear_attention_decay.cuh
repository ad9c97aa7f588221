// The factor by which the kernels of linear attention scale a state again and again: a power of the decay, which is hardly ever an fp32 number.
#pragma once

#include <cuda_runtime.h>

#include <cmath>

namespace rwkv7 {

// The rounded power, taken 256 times over a long memory, would be off 256 times the same way (1.6e-5 of a state, 3e-8 a chunk).  So it is rounded
// now down, now up, each as often as the power lies near it: the product of any number of factors in a row is off by one step of one factor.
// (The part that rounding took could be multiplied as well, at an instruction more for each two elements, and as 0 x inf or inf - inf it would make
// an infinite element NaN.)
class SteadyPower {
   public:
    SteadyPower() = default;
    __device__ __forceinline__ explicit SteadyPower(double power) {
        down_ = __double2float_rd(power);
        up_ = __double2float_ru(power);
        if (up_ == INFINITY) down_ = INFINITY;   // (nothing to choose from)
        else if (up_ > down_) up_part_ = (float)(power - (double)down_) / (up_ - down_);
    }
    __device__ __forceinline__ float next() {
        at_ += up_part_;
        if (at_ < 1.f) return down_;
        at_ -= 1.f;
        return up_;
    }

   private:
    float down_, up_, up_part_ = 0.f, at_ = 0.5f;
};

}  // namespace rwkv7
