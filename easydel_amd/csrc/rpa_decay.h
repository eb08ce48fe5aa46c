// Linear attention with a decay per head: parameters and launchers.
#pragma once
#include "rpa_common.h"

namespace rpa {

struct DecayParams {
  const void* q;  // rows of Hq heads of Dk, q_stride elements apart; k (Hkv heads of Dk) and v (Hkv heads of Dv) likewise
  const void* k;
  const void* v;
  const float* log_decay;  // [Hkv]
  float* state;            // [num_slots][Hkv][Dk][Dv]
  const int32_t* slot_in;   // [S]
  const int32_t* slot_out;  // [S]
  const int32_t* context_lens;  // [S] or null
  const int32_t* qsl;
  const int32_t* num_seqs;
  void* out;  // [T][Hq][Dv]
  int T, S, num_slots, Hq, Hkv, group, Dk, Dv;
  int64_t q_stride, k_stride, v_stride;  // elements
  int dtype;
  float scale;
  int rows;          // sequences of at most this many tokens take the recurrent form, the others the chunked one (rows >= T: none)
  // chunked form
  int vec;           // q, k and v rows allow 16-byte loads
  int seg_len;       // tokens of a segment
  int whole_len;     // sequences of up to this many tokens (>= seg_len) are one segment
  int slots;         // scratch slots: floor(T / seg_len) + 1, 0 where no sequence can be cut
  int first_ids;     // numbers that first segments may have ...
  int first_by_seq;  // ... which are their sequences' (1) or floor(qsl[i] / (kDecayRows + 1)) (0)
  int chunk_blocks;  // workgroups of the chunked form, ahead of those of the recurrent one in the same launch
  int direct;        // the bf16 kernel serves the call (the float32 one otherwise): the order of a scratch state's keys
  int key_tiles;     // tiles of 16 keys the kernels compute with (4, 8 or 16)
  int scratch_vecs;  // 16-byte vectors of a scratch state: columns and keys padded to what the kernels compute with
  void* scratch;     // [2 * slots][Hkv][scratch_vecs]
};

constexpr int kDecayRows = 16;
constexpr int kDecayWhole = 256;  // sequences of up to this many tokens are never cut (the Python layer asks for no scratch below it either)

struct DecaySeq {
  int q0, q_len;
  int in, out;  // slots, -1: a zero state / not written
};

__device__ __forceinline__ int decay_live_rows(const DecayParams& p) { return min(p.num_seqs[0], p.S); }

// Sequence i's tokens (never past T) and slots; q_len 0 where there is nothing to do.
__device__ __forceinline__ DecaySeq decay_seq(const DecayParams& p, int i) {
  DecaySeq s = {0, 0, -1, -1};
  if (i >= decay_live_rows(p)) return s;
  const int q0 = p.qsl[i], n = p.qsl[i + 1] - q0;
  if (n <= 0 || q0 < 0) return s;
  s.q0 = q0;
  s.q_len = min(n, p.T - q0);
  const bool fresh = p.context_lens != nullptr && p.context_lens[i] <= n;
  const int a = p.slot_in[i], b = p.slot_out[i];
  s.in = (fresh || a < 0 || a >= p.num_slots) ? -1 : a;
  s.out = (b < 0 || b >= p.num_slots) ? -1 : b;
  return s;
}

// exp(g n): -inf (nothing kept) times 0 would be NaN, so g is held at a value whose exponential is 0.  decay_power gives it as an
// unevaluated sum of two floats: a factor that a long prompt applies hundreds of times must not carry its own rounding along.
__device__ __forceinline__ double decay_exact(float g, int n) { return exp((double)(g < -1e30f ? -1e30f : g) * (double)n); }
// ... in float32, off by |g n| 2^-24 at most where that counts: for a factor applied once.
__device__ __forceinline__ float decay_float(float g, int n) { return expf((g < -1e30f ? -1e30f : g) * (float)n); }
__device__ __forceinline__ float2 decay_power(float g, int n) {
  const double e = decay_exact(g, n);
  const float hi = (float)e;
  return make_float2(hi, __builtin_isfinite(hi) ? (float)(e - (double)hi) : 0.f);
}

int launch_decay_chunk(hipStream_t stream, const DecayParams& p);
int launch_decay_recurrent(hipStream_t stream, const DecayParams& p);

}  // namespace rpa
