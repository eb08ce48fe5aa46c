// Linear attention with one decay per KV head, chunked form, for sequences of more than a few tokens.
//
// Within a chunk of C tokens from a state S0, with l = exp(g) and n, m = 0 .. C-1 inside the chunk:
//     o_n = scale * ( l^(n+1) q_n S0  +  sum_{m <= n} l^(n-m) (q_n . k_m) v_m )
//     S1  = l^C S0 + sum_m l^(C-1-m) k_m v_m^T
// No exponent is negative, so nothing overflows that the token-by-token recurrence would not.
//
// A sequence is a chain of chunks, which leaves only heads x sequences to work on side by side.  So a long sequence is cut
// into segments of seg_len tokens: (1) every segment but a sequence's last sums up what it adds to a zero state, (2) a scan
// turns these into the state ahead of each segment, (3) every segment runs its chunks from there.  (1) and (2) are only
// launched where the bounds allow a sequence of more than one segment.  The first segments are numbered by sequence or by
// floor(qsl[i] / (kDecayRows + 1)), the others by floor(qsl[i] / seg_len) + j - 1: both are distinct without a plan, since such
// a sequence is longer than the divisor.
#include "rpa_decay.h"
#include "rpa_mfma.h"

namespace rpa {

namespace {

typedef float f32x16 __attribute__((ext_vector_type(16)));

struct Segment {
  int j, t0, n;      // segment of its sequence, first token, tokens
  int in, out;       // slots of the sequence
  int base;          // scratch slot behind its first segment
  int segments;
  bool last;
};

// The segment that scratch slot `slot` lies behind (AHEAD: the one that starts from it).
template <bool AHEAD>
__device__ __forceinline__ bool find_by_slot(const DecayParams& p, int slot, Segment& g) {
  const int n_live = decay_live_rows(p);
  const int64_t t = (int64_t)slot * p.seg_len + p.seg_len - 1;
  if (n_live <= 0 || t < p.qsl[0]) return false;
  // sequences behind one of several segments start at its last segment or later: the last to start up to t owns the slot
  const int i = find_seq_wave(p.qsl, n_live, (int)min(t, (int64_t)INT32_MAX));
  const DecaySeq s = decay_seq(p, i);
  if (s.q_len <= kDecayRows) return false;
  const int segments = g.segments = (s.q_len + p.seg_len - 1) / p.seg_len;
  g.base = s.q0 / p.seg_len;
  g.j = slot - g.base + (AHEAD ? 1 : 0);
  if (g.j >= segments - (AHEAD ? 0 : 1)) return false;
  g.t0 = s.q0 + g.j * p.seg_len;
  g.n = min(s.q_len - g.j * p.seg_len, p.seg_len);
  g.in = s.in; g.out = s.out;
  g.last = g.j == segments - 1;
  return true;
}

// Segment of workgroup row `id`: ids below p.first_ids are first segments, the others start from a scratch state.
__device__ __forceinline__ bool find_segment(const DecayParams& p, int id, Segment& g) {
  if (id >= p.first_ids) return find_by_slot<true>(p, id - p.first_ids, g);
  const int n_live = decay_live_rows(p);
  if (n_live <= 0) return false;
  int i = id;
  if (!p.first_by_seq) {
    const int64_t t = (int64_t)id * (kDecayRows + 1) + kDecayRows;
    if (t < p.qsl[0]) return false;
    i = find_seq_wave(p.qsl, n_live, (int)min(t, (int64_t)INT32_MAX));
    if (p.qsl[i] / (kDecayRows + 1) != id) return false;
  }
  const DecaySeq s = decay_seq(p, i);
  if (s.q_len <= kDecayRows) return false;
  g.j = 0;
  g.t0 = s.q0;
  g.n = min(s.q_len, p.seg_len);
  g.in = s.in; g.out = s.out;
  g.base = s.q0 / p.seg_len;
  g.segments = (s.q_len + p.seg_len - 1) / p.seg_len;
  g.last = g.segments == 1;
  return true;
}

__device__ __forceinline__ float* scratch_state(const DecayParams& p, int slot, int h) {
  return p.scratch + ((int64_t)slot * p.Hkv + h) * p.Dk * p.Dv;
}

// Where a segment's state comes from (null: zeros).  A sequence of several segments may write the slot it started from while
// its first segment has yet to run, so the scan keeps the state it starts from, in a second set of scratch slots.
__device__ __forceinline__ const float* state_ahead(const DecayParams& p, const Segment& g, int h) {
  if (g.j > 0) return scratch_state(p, g.base + g.j - 1, h);
  if (!g.last) return scratch_state(p, p.slots + g.base, h);
  return g.in < 0 ? nullptr : p.state + ((int64_t)g.in * p.Hkv + h) * p.Dk * p.Dv;
}

// Scratch slots hold what each segment adds to a zero state; afterwards slot base + j holds the state behind segment j.
__global__ __launch_bounds__(256) void decay_scan_kernel(DecayParams p) {
  Segment g;
  if (!find_by_slot<false>(p, blockIdx.z, g) || g.j != 0) return;
  const int h = blockIdx.y, e = (blockIdx.x * 256 + threadIdx.x) * 4;
  if (e >= p.Dk * p.Dv) return;
  float4 r = make_float4(0.f, 0.f, 0.f, 0.f);
  if (g.in >= 0) r = *(const float4*)(p.state + ((int64_t)g.in * p.Hkv + h) * p.Dk * p.Dv + e);
  *(float4*)(scratch_state(p, p.slots + g.base, h) + e) = r;
  const float2 l = decay_power(p.log_decay[h], p.seg_len);
  for (int slot = g.base; slot < g.base + g.segments - 1; ++slot) {
    float4* at = (float4*)(scratch_state(p, slot, h) + e);
    const float4 a = *at;
    r.x = fmaf(r.x, l.y, fmaf(r.x, l.x, a.x)); r.y = fmaf(r.y, l.y, fmaf(r.y, l.x, a.y));
    r.z = fmaf(r.z, l.y, fmaf(r.z, l.x, a.z)); r.w = fmaf(r.w, l.y, fmaf(r.w, l.x, a.w));
    *at = r;
  }
}

// ---- bfloat16: matrix instructions on bf16 operands ---------------------------------------------------------
// Chunks of 32 tokens.  Wave w owns 32 columns of the state and of the output: its part of S stays in accumulators for the whole
// segment, as 32 x 32 tiles whose lane half h and register r hold key 32 d + 16 (r / 8) + 8 h + r % 8.  In that order eight
// registers, rounded to bf16, are one operand of the product with the queries as they lie in memory; the order comes for free,
// since the rows of K^T can be read in any order of four.
//   scores   S^T = K Q^T, three of the four 16 x 16 tiles, shared out over the waves, through LDS as bf16
//   output   O^T = S0^T Q^T, columns scaled by l^(n+1) in float32, then + V^T P^T
//   state    l^n S + K^T (l^(n-1-m) V): the decayed values are float32, so they enter as the sum of three bf16 numbers
//            (24 bits); the state keeps float32 accuracy.
// Rounded to bf16 are the scores and, for the product with the queries only, the state: what they add to an output is rounded
// to bf16 as well.  The tiles of the next chunk are on their way into LDS (direct loads, two buffers) while this one is worked on;
// registers hold no tile in flight, so two workgroups share a CU and fill each other's waits.

constexpr int kChunk = 32;
constexpr int kStrip = 80;  // bytes of a row of 32 bf16 values in LDS, spread over the banks

// 16-byte chunks of a row of WIDTH elements are stored XOR-ed with this key: eight consecutive rows read at one chunk, and four
// rows read at a pair of chunks by the transposing loads, fall on distinct banks.
template <int WIDTH>
__device__ __forceinline__ int tile_key(int row) {
  if constexpr (WIDTH >= 128) return (row & 7) << 1;
  else return ((row >> 1) & 3) << 1;
}

typedef __attribute__((address_space(3))) const char lds_char;
__device__ __forceinline__ uint32_t lds_address(const char* p) { return (uint32_t)(uintptr_t)(lds_char*)p; }

template <int WIDTH>
__device__ __forceinline__ u32x4 row_operand(const char* tile, int row, int chunk) {
  return *(const u32x4*)(tile + row * WIDTH * 2 + ((chunk ^ tile_key<WIDTH>(row)) << 4));
}

// Four rows from `row` on of sixteen columns, one column a lane (of each group of sixteen): the lane supplies the address of row
// row + (lane & 15) / 4 and of the four columns `mine` on that lanes 4 (lane & 3) .. + 3 are to hold.
template <int WIDTH>
__device__ __forceinline__ u32x2 column_operand(const char* tile, int row, int mine) {
  const int r = row + ((threadIdx.x & 15) >> 2);
  const char* a = tile + r * WIDTH * 2 + (((mine >> 3) ^ tile_key<WIDTH>(r)) << 4) + ((mine & 7) << 1);
  return __builtin_bit_cast(u32x2, __builtin_amdgcn_ds_read_tr16_b64_v4i16((__attribute__((address_space(3))) s16x4*)(uintptr_t)lds_address(a)));
}

__device__ __forceinline__ f32x16 mfma_bf16(u32x4 a, u32x4 b, f32x16 c) {
  return __builtin_amdgcn_mfma_f32_32x32x16_bf16(__builtin_bit_cast(bf16x8, a), __builtin_bit_cast(bf16x8, b), c, 0, 0, 0);
}

__device__ __forceinline__ float low_half(uint32_t w) { return __uint_as_float(w << 16); }
__device__ __forceinline__ float high_half(uint32_t w) { return __uint_as_float(w & 0xffff0000u); }

__device__ uint4 decay_zeros;  // 16 bytes of zeros: the source of what a tile holds beyond its rows and columns

// A tile of kChunk rows of WIDTH elements on its way into LDS: rows 0 .. n-1 of `cols` elements exist, `stride` elements apart, the
// others become zeros.  VEC: direct loads of 16 bytes a lane, 1 KiB an instruction, complete when this wave's vector-memory
// counter says so; a whole tile takes its lanes' offsets from registers and its base from scalars.  Otherwise rows at any
// address, element by element, complete at the next barrier.
template <int WIDTH, int NT, bool VEC>
struct TileLoad {
  static constexpr int PER_ROW = WIDTH / 8, N = kChunk * PER_ROW / NT;
  static_assert(N >= 1, "at least one piece a thread");
  uint32_t at[VEC ? N : 1];
  int64_t stride;
  int cols;
  // wave w's instruction k fills bytes [(w N + k) 1024, + 1024) of the tile
  static __device__ __forceinline__ int piece(int k) { return ((threadIdx.x >> 6) * N + k) * 64 + (threadIdx.x & 63); }
  static __device__ __forceinline__ int column(int k) { return ((piece(k) % PER_ROW) ^ tile_key<WIDTH>(piece(k) / PER_ROW)) * 8; }
  __device__ __forceinline__ void init(int64_t stride_, int cols_) {
    stride = stride_; cols = cols_;
    if constexpr (VEC) {
#pragma unroll
      for (int k = 0; k < N; ++k) at[k] = ((uint32_t)(piece(k) / PER_ROW) * (uint32_t)stride + column(k)) * 2;  // 32 rows span less than 2^31 bytes
    }
  }
  __device__ __forceinline__ void start(char* tile, const uint16_t* src, int n) const {
    if constexpr (VEC) {
      const uint32_t to = __builtin_amdgcn_readfirstlane(lds_address(tile) + (threadIdx.x >> 6) * N * 1024);
      if (n >= kChunk && cols >= WIDTH) {
#pragma unroll
        for (int k = 0; k < N; ++k) dma16(to + k * 1024, at[k], src);
      } else {
#pragma unroll
        for (int k = 0; k < N; ++k) {
          const int row = piece(k) / PER_ROW, c = column(k);
          const void* from = row < n && c < cols ? (const void*)(src + row * stride + c) : (const void*)&decay_zeros;
          asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %1, off" ::"s"(to + k * 1024), "v"(from) : "memory");
        }
      }
    } else {
#pragma unroll
      for (int k = 0; k < N; ++k) {
        const int row = piece(k) / PER_ROW, c = column(k);
        uint64_t lo = 0, hi = 0;
        if (row < n) {
          const uint16_t* from = src + row * stride + c;
#pragma unroll 1
          for (int x = min(cols - c, 8) - 1; x >= 0; --x) {
            hi = (hi << 16) | (lo >> 48);
            lo = (lo << 16) | from[x];
          }
        }
        *(u32x4*)(tile + piece(k) * 16) = u32x4{(uint32_t)lo, (uint32_t)(lo >> 32), (uint32_t)hi, (uint32_t)(hi >> 32)};
      }
    }
  }
};

// Eight decayed values as three bf16 operands whose sum is the float32 value.
__device__ __forceinline__ void split3(u32x4 v, const float4& w0, const float4& w1, u32x4& hi, u32x4& mid, u32x4& lo) {
  const float w[8] = {w0.x, w0.y, w0.z, w0.w, w1.x, w1.y, w1.z, w1.w};
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    float a = low_half(v[i]) * w[2 * i], b = high_half(v[i]) * w[2 * i + 1];
    hi[i] = pack_bf16(a, b);
    a -= low_half(hi[i]); b -= high_half(hi[i]);
    mid[i] = pack_bf16(a, b);
    a -= low_half(mid[i]); b -= high_half(mid[i]);
    lo[i] = pack_bf16(a, b);
  }
}

__device__ __forceinline__ uint32_t finite_halves(uint32_t w) {
  if ((w & 0x7f80u) == 0x7f80u) w &= 0xffff0000u;
  if ((w & 0x7f800000u) == 0x7f800000u) w &= 0xffffu;
  return w;
}

template <int DK, int NW, bool OUT, bool VEC>
__global__ __launch_bounds__(64 * NW, DK <= 128 ? 2 : 1) void decay_chunk_bf16_kernel(DecayParams p) {
  constexpr int NT = 64 * NW, DV = 32 * NW, ND = DK / 32;
  constexpr int KB = kChunk * DK * 2, VB = kChunk * DV * 2;
  __shared__ __align__(1024) char sK[2][KB];
  __shared__ __align__(1024) char sV[2][VB];
  __shared__ __align__(1024) char sQ[OUT ? 2 : 1][OUT ? KB : 16];
  __shared__ __align__(16) char sP[OUT ? kChunk * kStrip : 16];
  __shared__ __align__(16) char sO[OUT ? NW * kChunk * kStrip : 16];
  __shared__ __align__(16) float pw[kChunk + 4];  // l^0 .. l^C
  __shared__ __align__(16) float left[kChunk];    // l^(n-1-m) for the n tokens m of a chunk, 0 behind them

  const int slices = (p.Dv + DV - 1) / DV, heads = p.Hkv * slices;
  const int id = blockIdx.x / heads, hs = blockIdx.x - id * heads, h = hs / slices, c0 = (hs - h * slices) * DV;
  Segment g;
  if (OUT ? !find_segment(p, id, g) : !find_by_slot<false>(p, id, g)) return;
  const int tid = threadIdx.x, lane = tid & 63, w = tid >> 6, half = lane >> 5, l31 = lane & 31;
  const int chunks = (g.n + kChunk - 1) / kChunk;
  const uint16_t* q = (const uint16_t*)p.q + (int64_t)g.t0 * p.q_stride + (int64_t)h * p.group * p.Dk;
  const uint16_t* k = (const uint16_t*)p.k + (int64_t)g.t0 * p.k_stride + (int64_t)h * p.Dk;
  const uint16_t* v = (const uint16_t*)p.v + (int64_t)g.t0 * p.v_stride + (int64_t)h * p.Dv + c0;
  const int vcols = min(p.Dv - c0, DV), groups = OUT ? p.group : 1;
  TileLoad<DK, NT, VEC> lq, lk;
  TileLoad<DV, NT, VEC> lv;
  lk.init(p.k_stride, p.Dk);
  lv.init(p.v_stride, vcols);
  const int64_t first = OUT ? 0 : (int64_t)(chunks - 1) * kChunk;
  lk.start(sK[0], k + first * p.k_stride, g.n);
  lv.start(sV[0], v + first * p.v_stride, g.n);
  if constexpr (OUT) {
    lq.init(p.q_stride, p.Dk);
    lq.start(sQ[0], q, g.n);
  }

  const float rate = p.log_decay[h];
  if (tid <= kChunk) pw[tid] = decay_power(rate, tid).x;
  if (tid >= 64 && tid < 64 + kChunk) left[tid - 64] = decay_power(rate, kChunk - 1 - (tid - 64)).x;
  if constexpr (OUT) {
    if (tid < 64) *(u32x4*)(sP + (tid & 15) * kStrip + 32 + (tid >> 4 & 1) * 16) = u32x4{0u, 0u, 0u, 0u};  // the tile of masked scores alone
  }

  const int col = c0 + 32 * w + l31;
  const bool mine = col < p.Dv;
  f32x16 S[ND];
  const float* from = OUT ? state_ahead(p, g, h) : nullptr;
#pragma unroll
  for (int d = 0; d < ND; ++d) S[d] = f32x16{};
  if (from != nullptr) {
    const float* at = from + (mine ? col : 0);
#pragma unroll
    for (int d = 0; d < ND; ++d)
#pragma unroll
      for (int r = 0; r < 16; ++r) {
        const int key = 32 * d + 16 * (r >> 3) + 8 * half + (r & 7);
        const float x = at[min(key, p.Dk - 1) * p.Dv];  // unconditional loads, all in flight at once
        S[d][r] = mine && key < p.Dk ? x : 0.f;
      }
  }

  // The state is multiplied by l^C once a chunk: each factor is rounded so that the product of all of them so far stays within a
  // rounding of the true power (`off`: how far it is, relatively), however long the segment.
  const double full_power = decay_exact(rate, kChunk);
  const double tail_power = decay_exact(rate, g.n - (chunks - 1) * kChunk);
  const double per = full_power > 0.0 ? 1.0 / full_power : 0.0;
  double off = 0.0, over = 1.0;

  // this lane's share of the transposing loads
  const int vcol = 32 * w + 16 * ((lane >> 4) & 1) + 4 * (lane & 3);
  const int kcol = 16 * ((lane >> 4) & 1) + 4 * (((lane & 1) << 1) | ((lane >> 1) & 1));

  for (int c = 0; c < chunks; ++c) {
    const int n = OUT ? min(g.n - c * kChunk, kChunk) : kChunk;
    const char *tK = sK[c & 1], *tV = sV[c & 1];
    u32x4 vop[2];
    for (int gq = 0; gq < groups; ++gq) {
      const int step = c * groups + gq;
      // this step's tiles have arrived (so have the output rows of the step before), and the other buffers have been read
      if constexpr (VEC) wait_loads<0>();
      __syncthreads();
      const bool on = gq == groups - 1;  // the next step is another chunk's
      const int cn = c + (on ? 1 : 0);
      if (cn < chunks) {
        const int64_t ahead = (int64_t)(OUT ? cn : chunks - 1 - cn) * kChunk;
        if constexpr (OUT) lq.start(sQ[(step + 1) & 1], q + ahead * p.q_stride + (on ? 0 : (gq + 1) * p.Dk), g.n - cn * kChunk);
        if (on) {
          lk.start(sK[cn & 1], k + ahead * p.k_stride, OUT ? g.n - cn * kChunk : kChunk);
          lv.start(sV[cn & 1], v + ahead * p.v_stride, OUT ? g.n - cn * kChunk : kChunk);
        }
      }
      if (n < kChunk && gq == 0 && tid < kChunk) left[tid] = tid < n ? pw[n - 1 - tid] : 0.f;  // the last chunk alone
      if constexpr (OUT) {
        const char* tQ = sQ[step & 1];
        // scores, decayed and masked: tile (keys 16 a.., queries 16 b..) of S^T
        const int i16 = lane & 15, g4 = lane >> 4;
#pragma unroll
        for (int tile = 0; tile < 3; ++tile) {
          if (tile % NW != w) continue;
          const int a = tile == 1 ? 1 : 0, b = tile == 0 ? 0 : 1;
          f32x4 acc = {};
#pragma unroll
          for (int ks = 0; ks < DK / 32; ++ks)
            acc = HalfOf<RPA_BF16>::mfma32(row_operand<DK>(tK, 16 * a + i16, 4 * ks + g4), row_operand<DK>(tQ, 16 * b + i16, 4 * ks + g4), acc);
          const int t = 16 * b + i16, s0 = 16 * a + 4 * g4;
          float f[4];
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            const int gap = t - s0 - e;
            f[e] = gap >= 0 ? acc[e] * pw[max(gap, 0)] : 0.f;  // chosen, not multiplied: masked scores may be infinite
          }
          *(u32x2*)(sP + t * kStrip + s0 * 2) = u32x2{pack_bf16(f[0], f[1]), pack_bf16(f[2], f[3])};
        }
        __syncthreads();
        // O^T of this wave's columns: lane = token, registers = columns 8 (r / 4) + 4 half + r % 4
        f32x16 o = {};
#pragma unroll
        for (int d = 0; d < ND; ++d)
#pragma unroll
          for (int x = 0; x < 2; ++x) {
            const u32x4 s = {pack_bf16(S[d][8 * x], S[d][8 * x + 1]), pack_bf16(S[d][8 * x + 2], S[d][8 * x + 3]),
                             pack_bf16(S[d][8 * x + 4], S[d][8 * x + 5]), pack_bf16(S[d][8 * x + 6], S[d][8 * x + 7])};
            o = mfma_bf16(s, row_operand<DK>(tQ, l31, 4 * d + 2 * x + half), o);
          }
        const float ahead_of = pw[l31 + 1];
#pragma unroll
        for (int r = 0; r < 16; ++r) o[r] *= ahead_of;
        // A value that is not finite would meet the zeros of the masked scores as well, and 0 x Inf is NaN: such values stay out of
        // the product, and the rows that see one become NaN by hand.
        uint32_t full = 0;
#pragma unroll
        for (int ks = 0; ks < 2; ++ks) {
          const u32x2 x = column_operand<DV>(tV, 16 * ks + 8 * half, vcol), y = column_operand<DV>(tV, 16 * ks + 8 * half + 4, vcol);
          vop[ks] = u32x4{x[0], x[1], y[0], y[1]};
#pragma unroll
          for (int e = 0; e < 4; ++e) full |= (vop[ks][e] & 0x7f807f80u) + 0x00800080u;  // bit 15 or 31: an exponent of all ones
        }
        const bool odd = __any((full & 0x80008000u) != 0);
#pragma unroll
        for (int ks = 0; ks < 2; ++ks) {
          u32x4 vo = vop[ks];
          if (odd) {
#pragma unroll
            for (int e = 0; e < 4; ++e) vo[e] = finite_halves(vo[e]);
          }
          o = mfma_bf16(vo, *(const u32x4*)(sP + l31 * kStrip + (2 * ks + half) * 16), o);
        }
        if (odd) {
          const int at = 32 * w + l31;
          int bad = 0;
          for (; bad < n; ++bad) {
            const uint16_t bits = *(const uint16_t*)(tV + bad * DV * 2 + (((at >> 3) ^ tile_key<DV>(bad)) << 4) + ((at & 7) << 1));
            if ((bits & 0x7f80) == 0x7f80) break;
          }
#pragma unroll
          for (int r = 0; r < 16; ++r) {
            const int first = __shfl(bad, 8 * (r >> 2) + 4 * half + (r & 3));
            o[r] = l31 >= first ? __builtin_nanf("") : o[r];
          }
        }
        // through this wave's own strip of LDS (whose accesses stay in order) to whole rows of 32 columns
        char* strip = sO + w * kChunk * kStrip;
#pragma unroll
        for (int r4 = 0; r4 < 4; ++r4)
          *(u32x2*)(strip + l31 * kStrip + 16 * r4 + 8 * half) = u32x2{pack_bf16(o[4 * r4] * p.scale, o[4 * r4 + 1] * p.scale),
                                                                       pack_bf16(o[4 * r4 + 2] * p.scale, o[4 * r4 + 3] * p.scale)};
        __builtin_amdgcn_wave_barrier();
        char* out = (char*)p.out + (((int64_t)(g.t0 + c * kChunk) * p.Hq + h * p.group + gq) * p.Dv + c0 + 32 * w) * 2;
        const int piece = lane & 3, cols = p.Dv - c0 - 32 * w - 8 * piece;  // columns of the piece that exist
        for (int row = lane >> 2; row < n; row += 16) {
          const u32x4 v8 = *(const u32x4*)(strip + row * kStrip + 16 * piece);
          char* to = out + (int64_t)row * p.Hq * p.Dv * 2 + 16 * piece;
          if (cols >= 8 && (p.Dv & 7) == 0) *(u32x4*)to = v8;
          else if (cols >= 4) { *(u32x2*)to = u32x2{v8[0], v8[1]}; if (cols >= 8) *(u32x2*)(to + 8) = u32x2{v8[2], v8[3]}; }
        }
        __builtin_amdgcn_wave_barrier();
      }
    }
    if (OUT && c == chunks - 1 && (!g.last || g.out < 0)) break;  // nobody reads the state behind this chunk
    // OUT: the state is decayed over the chunk.  Otherwise it starts from zero, the chunks come last to first (all are whole) and
    // their tokens enter with their decay to the end of the segment, which leaves the state alone.
    const float behind = (float)over;
    over *= full_power;
    if constexpr (OUT) {
      const double exact = n < kChunk ? tail_power : full_power;
      const float l = (float)(exact * (1.0 - off));
      off += ((double)l - exact) * per;
#pragma unroll
      for (int d = 0; d < ND; ++d)
#pragma unroll
        for (int r = 0; r < 16; ++r) S[d][r] *= l;
    }
#pragma unroll
    for (int ks = 0; ks < 2; ++ks) {
      const int m = 16 * ks + 8 * half;
      if constexpr (!OUT) {
        const u32x2 x = column_operand<DV>(tV, m, vcol), y = column_operand<DV>(tV, m + 4, vcol);
        vop[ks] = u32x4{x[0], x[1], y[0], y[1]};
      }
      u32x4 hi, mid, lo;
      float4 w0 = *(const float4*)&left[m], w1 = *(const float4*)&left[m + 4];
      if constexpr (!OUT) {
        w0.x *= behind; w0.y *= behind; w0.z *= behind; w0.w *= behind;
        w1.x *= behind; w1.y *= behind; w1.z *= behind; w1.w *= behind;
      }
      split3(vop[ks], w0, w1, hi, mid, lo);
#pragma unroll
      for (int d = 0; d < ND; ++d) {
        const u32x2 u = column_operand<DK>(tK, m, 32 * d + kcol), z = column_operand<DK>(tK, m + 4, 32 * d + kcol);
        const u32x4 kt = {u[0], u[1], z[0], z[1]};
        S[d] = mfma_bf16(kt, lo, S[d]);
        S[d] = mfma_bf16(kt, mid, S[d]);
        S[d] = mfma_bf16(kt, hi, S[d]);
      }
    }
  }
  if (OUT && (!g.last || g.out < 0)) return;
  float* to = OUT ? p.state + ((int64_t)g.out * p.Hkv + h) * p.Dk * p.Dv : scratch_state(p, g.base + g.j, h);
  int back = 8 * half;
  asm volatile("" : "+v"(back));  // the addresses and masks are not those of the beginning, kept through the loop
  if (!mine) return;
  float* at = to + back * p.Dv + col;
#pragma unroll
  for (int d = 0; d < ND; ++d)
#pragma unroll
    for (int r = 0; r < 16; ++r) {
      const int key = 32 * d + 16 * (r >> 3) + (r & 7);
      if (key + back < p.Dk) at[key * p.Dv] = S[d][r];
    }
}

template <int DK, int NW, bool VEC>
void launch_bf16(hipStream_t stream, const DecayParams& p) {
  const int slices = (p.Dv + 32 * NW - 1) / (32 * NW), heads = p.Hkv * slices;
  if (p.slots > 0) {
    hipLaunchKernelGGL((decay_chunk_bf16_kernel<DK, NW, false, VEC>), dim3(p.slots * heads), dim3(64 * NW), 0, stream, p);
    hipLaunchKernelGGL(decay_scan_kernel, dim3((p.Dk * p.Dv / 4 + 255) / 256, p.Hkv, p.slots), dim3(256), 0, stream, p);
  }
  hipLaunchKernelGGL((decay_chunk_bf16_kernel<DK, NW, true, VEC>), dim3((p.first_ids + p.slots) * heads), dim3(64 * NW), 0, stream, p);
}

template <int DK>
void launch_bf16_cols(hipStream_t stream, const DecayParams& p) {
  if (!p.vec) launch_bf16<DK, 4, false>(stream, p);
  else if (p.Dv <= 64) launch_bf16<DK, 2, true>(stream, p);
  else launch_bf16<DK, 4, true>(stream, p);
}

}  // namespace

bool decay_chunk_supported(const DecayParams& p) { return p.dtype == RPA_BF16; }

int launch_decay_chunk(hipStream_t stream, const DecayParams& p) {
  if (p.Dk <= 64) launch_bf16_cols<64>(stream, p);
  else if (p.Dk <= 128) launch_bf16_cols<128>(stream, p);
  else launch_bf16_cols<256>(stream, p);
  return (int)hipGetLastError();
}

}  // namespace rpa
