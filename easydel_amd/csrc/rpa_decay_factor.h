// Linear attention with a decay per head: the factor that a chain of whole chunks applies to its state.  Plain arithmetic, for the
// kernels and for any host compiler.
#pragma once

#ifdef __HIP__
#define RPA_DECAY_FN __host__ __device__ inline
#else
#define RPA_DECAY_FN inline
#endif

namespace rpa {

// A chunk multiplies the state by l^C = hi + lo.  Each factor is rounded so that the product of all of them so far stays within a
// rounding of the true power (`off`: how far it is, relatively), however long the chain.
struct DecayFactor {
  float hi, lo, per, off;
  RPA_DECAY_FN void init(float hi_, float lo_) {
    hi = hi_; lo = lo_;
    // A subnormal power stays as it is: its reciprocal may be infinite, and what such a factor leaves of a state is below the
    // rounding of the tokens behind it.
    per = hi >= 0x1p-126f ? 1.f / hi : 0.f;
    off = 0.f;
  }
  RPA_DECAY_FN float next() {
    const float l = hi + (lo - hi * off);
    off += ((l - hi) - lo) * per;
    return l;
  }
};

}  // namespace rpa
