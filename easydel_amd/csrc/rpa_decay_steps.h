// Linear attention with one decay per KV head, recurrent form: the work of one workgroup.
//     S <- l S + k_t v_t^T,   o_t = scale * q_t S.
// For few tokens the state is the traffic: 4 Dk Dv bytes read and as many written per head and sequence against 2 (Dk + Dv)
// elements of q, k, v, o per token, so it is bound by HBM.  A workgroup owns 4 CG columns of one head's state in registers: thread
// (r, c) holds rows r, r + RG, ... of four columns, read in 16-byte loads that are all in flight before the first is used.
#pragma once
#include "rpa_decay.h"

namespace rpa {

// A state is next wanted a whole model's worth of traffic later: past the caches, reads and writes stream faster (256 states of 64
// heads of 128 x 128: 393 -> 374 us).
__device__ __forceinline__ float4 load_once(const float* at) {
  typedef float f4 __attribute__((ext_vector_type(4)));
  const f4 x = __builtin_nontemporal_load((const f4*)at);
  return make_float4(x[0], x[1], x[2], x[3]);
}
__device__ __forceinline__ void store_once(float* at, const float4& v) {
  typedef float f4 __attribute__((ext_vector_type(4)));
  const f4 x = {v.x, v.y, v.z, v.w};
  __builtin_nontemporal_store(x, (f4*)at);
}

// Zeros in the output rows of tokens that belong to no sequence, shared out over `blocks` workgroups.
template <int DT>
__device__ __forceinline__ void clear_padded_rows(const DecayParams& p, int block, int blocks) {
  const int n = decay_live_rows(p), lo = n > 0 ? min(max(p.qsl[0], 0), p.T) : p.T, hi = n > 0 ? min(max(p.qsl[n], lo), p.T) : p.T;
  const int64_t row = (int64_t)p.Hq * p.Dv * ElemBytes<DT>::v / 8;  // 8 bytes at a time: rows are multiples of four elements
  for (int r = block; r < lo + (p.T - hi); r += blocks) {
    uint2* at = (uint2*)p.out + (int64_t)(r < lo ? r : hi + (r - lo)) * row;
    for (int64_t k = threadIdx.x; k < row; k += blockDim.x) at[k] = make_uint2(0u, 0u);
  }
}

template <int NT, int CG>
struct StepLds {
  float k[256], q[256], v[4 * CG];  // 256 keys at most
  float4 part[NT / 64][CG];
};

// Sequence i's tokens, if they are at most p.rows, for columns c0 .. of KV head h; NT threads, CG groups of four columns, NR
// rows a thread.
template <int DT, int NT, int CG, int NR>
__device__ __forceinline__ void decay_steps(const DecayParams& p, int i, int h, int c0, StepLds<NT, CG>& lds) {
  constexpr int RG = NT / CG;
  float *sk = lds.k, *sq = lds.q, *sv = lds.v;
  auto& part = lds.part;
  const int tid = threadIdx.x, cg = tid % CG, rg = tid / CG;
  const DecaySeq s = decay_seq(p, i);
  if (s.q_len <= 0 || s.q_len > p.rows) return;
  const int col = c0 + 4 * cg;
  const bool in_cols = col < p.Dv;
  const int64_t head = (int64_t)p.Dk * p.Dv, at = (int64_t)h * head + col;
  float4 S[NR];
#pragma unroll
  for (int j = 0; j < NR; ++j) {
    const int r = rg + j * RG;
    S[j] = make_float4(0.f, 0.f, 0.f, 0.f);
    if (s.in >= 0 && in_cols && r < p.Dk) S[j] = load_once(p.state + (int64_t)s.in * p.Hkv * head + at + (int64_t)r * p.Dv);
  }
  const float2 l = decay_power(p.log_decay[h], 1);
  for (int n = 0; n < s.q_len; ++n) {
    const int64_t t = s.q0 + n;
    for (int d = tid; d < p.Dk; d += NT) sk[d] = load_elem<DT>(p.k, t * p.k_stride + h * p.Dk + d);
    for (int d = tid; d < 4 * CG; d += NT) sv[d] = c0 + d < p.Dv ? load_elem<DT>(p.v, t * p.v_stride + h * p.Dv + c0 + d) : 0.f;
    for (int g = 0; g < p.group; ++g) {
      const int hq = h * p.group + g;
      for (int d = tid; d < p.Dk; d += NT) sq[d] = load_elem<DT>(p.q, t * p.q_stride + hq * p.Dk + d);
      __syncthreads();
      if (g == 0) {
        const float4 v = *(const float4*)&sv[4 * cg];
#pragma unroll
        for (int j = 0; j < NR; ++j) {
          const int r = rg + j * RG;
          const float k = r < p.Dk ? sk[r] : 0.f;
          S[j].x = fmaf(S[j].x, l.y, fmaf(S[j].x, l.x, k * v.x));
          S[j].y = fmaf(S[j].y, l.y, fmaf(S[j].y, l.x, k * v.y));
          S[j].z = fmaf(S[j].z, l.y, fmaf(S[j].z, l.x, k * v.z));
          S[j].w = fmaf(S[j].w, l.y, fmaf(S[j].w, l.x, k * v.w));
        }
      }
      float4 o = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
      for (int j = 0; j < NR; ++j) {
        const int r = rg + j * RG;
        const float q = r < p.Dk ? sq[r] : 0.f;
        o.x = fmaf(q, S[j].x, o.x); o.y = fmaf(q, S[j].y, o.y); o.z = fmaf(q, S[j].z, o.z); o.w = fmaf(q, S[j].w, o.w);
      }
#pragma unroll
      for (int m = 32; m >= CG; m >>= 1) {
        o.x += __shfl_xor(o.x, m); o.y += __shfl_xor(o.y, m); o.z += __shfl_xor(o.z, m); o.w += __shfl_xor(o.w, m);
      }
      if ((tid & 63) < CG) part[tid >> 6][cg] = o;
      __syncthreads();
      if (tid < 4 * CG && c0 + tid < p.Dv) {
        const float* f = (const float*)part;
        float r = (f[tid] + f[4 * CG + tid]) + (f[8 * CG + tid] + f[12 * CG + tid]);
        if constexpr (NT == 512) r += (f[16 * CG + tid] + f[20 * CG + tid]) + (f[24 * CG + tid] + f[28 * CG + tid]);
        store_out<DT>(p.out, (t * p.Hq + hq) * p.Dv + c0 + tid, r * p.scale);
      }
    }
  }
  if (s.out < 0 || !in_cols) return;
#pragma unroll
  for (int j = 0; j < NR; ++j) {
    const int r = rg + j * RG;
    if (r < p.Dk) store_once(p.state + (int64_t)s.out * p.Hkv * head + at + (int64_t)r * p.Dv, S[j]);
  }
}

}  // namespace rpa
