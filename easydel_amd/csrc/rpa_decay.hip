// Linear attention with one decay per KV head: the launch of the recurrent form alone, for calls of few tokens or of rows too far
// apart for the chunked form, whose launch takes the short sequences along otherwise.
#include "rpa_decay_steps.h"

namespace rpa {

namespace {

template <int DT, int CG, int NR>
__global__ __launch_bounds__(256) void decay_recurrent_kernel(DecayParams p) {
  __shared__ StepLds<256, CG> lds;
  if ((int)blockIdx.y >= p.S) {
    clear_padded_rows<DT>(p, (blockIdx.y - p.S) * gridDim.x + blockIdx.x, (gridDim.y - p.S) * gridDim.x);
    return;
  }
  const int slices = (p.Dv + 4 * CG - 1) / (4 * CG), h = blockIdx.x / slices;
  decay_steps<DT, 256, CG, NR>(p, blockIdx.y, h, (blockIdx.x - h * slices) * 4 * CG, lds);
}

// A workgroup takes 32 columns of a state: few states want many workgroups (8 states of 32 heads of 128 x 128: 7.8 us; 8.5 us with 128
// columns each).
template <int DT>
int launch_rows(hipStream_t stream, const DecayParams& p) {
  constexpr int CG = 8, RG = 256 / CG;
  const int slices = (p.Dv + 4 * CG - 1) / (4 * CG);
  const int wide = p.Hkv * slices;
  const dim3 grid(wide, p.S + (256 + wide - 1) / wide), block(256);  // the last rows of workgroups clear padded rows
  const int need = (p.Dk + RG - 1) / RG;
  if (need <= 64 / RG) hipLaunchKernelGGL((decay_recurrent_kernel<DT, CG, 64 / RG>), grid, block, 0, stream, p);
  else if (need <= 128 / RG) hipLaunchKernelGGL((decay_recurrent_kernel<DT, CG, 128 / RG>), grid, block, 0, stream, p);
  else hipLaunchKernelGGL((decay_recurrent_kernel<DT, CG, 256 / RG>), grid, block, 0, stream, p);
  return (int)hipGetLastError();
}

}  // namespace

int launch_decay_recurrent(hipStream_t stream, const DecayParams& p) {
  switch (p.dtype) {
    case RPA_F32: return launch_rows<RPA_F32>(stream, p);
    case RPA_BF16: return launch_rows<RPA_BF16>(stream, p);
    case RPA_F16: return launch_rows<RPA_F16>(stream, p);
    default: return (int)hipErrorInvalidValue;
  }
}

}  // namespace rpa
