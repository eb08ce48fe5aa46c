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
#include "rpa_decay_factor.h"
#include "rpa_decay_steps.h"
#include "rpa_mfma.h"

namespace rpa {

namespace {

constexpr int kClearBlocks = 64;

struct Segment {
  int j, t0, n;      // segment of its sequence, first token, tokens
  int in, out;       // slots of the sequence
  int base;          // scratch slot behind its first segment
  int segments;
  bool last;
};

// Sequences of up to whole_len tokens are not cut.
__device__ __forceinline__ int segments_of(const DecayParams& p, int q_len) {
  return q_len <= p.whole_len ? 1 : (q_len + p.seg_len - 1) / p.seg_len;
}

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
  const int segments = g.segments = segments_of(p, s.q_len);
  g.base = s.q0 / p.seg_len;
  g.j = slot - g.base + (AHEAD ? 1 : 0);
  if (segments == 1 || g.j >= segments - (AHEAD ? 0 : 1)) return false;
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
  g.segments = segments_of(p, s.q_len);
  g.last = g.segments == 1;
  g.n = g.last ? s.q_len : p.seg_len;
  g.in = s.in; g.out = s.out;
  g.base = s.q0 / p.seg_len;
  return true;
}

// A scratch state lies as the lanes of the chunk kernels hold it, 16 bytes a lane and tile of 16 keys: [16-column group][tile][lane].
__device__ __forceinline__ f32x4* scratch_state(const DecayParams& p, int slot, int h) {
  return (f32x4*)p.scratch + ((int64_t)slot * p.Hkv + h) * p.scratch_vecs;
}

// Workgroups behind the chunked form's own take the sequences of few tokens, then the padded rows: the chains of chunks leave HBM
// room that the states of decode rows use.  (48 decode rows beside six prompts of 650 to 2000 tokens, 64 heads of 128 x 128: 222 us;
// a launch of its own for the decode rows 190 + 65 us.  256 decode rows alone: 358 to 370 us, 5.8 to 6.0 TB/s, against 385 + 6 us.)
template <int DT, int DK, int NW>
__device__ __forceinline__ void beside_chunks(const DecayParams& p, int id, int heads, int slices, char* lds) {
  if (id >= p.S * heads) {
    clear_padded_rows<DT>(p, id - p.S * heads, kClearBlocks);
    return;
  }
  const int i = id / heads, hs = id - i * heads, h = hs / slices;
  decay_steps<DT, 64 * NW, 4 * NW, DK / 16>(p, i, h, (hs - h * slices) * 16 * NW, *(StepLds<64 * NW, 4 * NW>*)lds);
}

// The first of the four keys that a lane group holds of tile d: in the order in which the bf16 kernel reads the queries, or as they
// come (the float32 kernel).
__device__ __forceinline__ int first_key(int direct, int d, int g4) { return direct ? 32 * (d >> 1) + 8 * g4 + 4 * (d & 1) : 16 * d + 4 * g4; }

// Scratch slots hold what each segment adds to a zero state; afterwards slot base + j holds the state behind segment j.  A sequence
// of several segments may write the slot of the pool it started from while its first segment has yet to run, so the state it
// starts from is kept too, in a second set of scratch slots.
__global__ __launch_bounds__(256) void decay_scan_kernel(DecayParams p) {
  constexpr int VECS = 2, AHEAD = 4;  // vectors a thread; slots read ahead: the chain is in the sums alone
  Segment g;
  if (!find_by_slot<false>(p, blockIdx.z, g) || g.j != 0) return;
  const int h = blockIdx.y, e0 = blockIdx.x * 256 * VECS + threadIdx.x;
  f32x4 r[VECS];
#pragma unroll
  for (int v = 0; v < VECS; ++v) {
    const int e = e0 + v * 256, lane = e & 63, d = (e >> 6) % p.key_tiles, col = 16 * ((e >> 6) / p.key_tiles) + (lane & 15);
    const int key = first_key(p.direct, d, lane >> 4);
    r[v] = f32x4{};
    if (g.in >= 0 && col < p.Dv) {
      const float* from = p.state + ((int64_t)g.in * p.Hkv + h) * p.Dk * p.Dv + col;
#pragma unroll
      for (int j = 0; j < 4; ++j) r[v][j] = key + j < p.Dk ? from[(key + j) * p.Dv] : 0.f;
    }
    scratch_state(p, p.slots + g.base, h)[e] = r[v];
  }
  const float2 l = decay_power(p.log_decay[h], p.seg_len);
  const int end = g.base + g.segments - 1;
  for (int slot = g.base; slot < end; slot += AHEAD) {
    f32x4 a[AHEAD][VECS];
#pragma unroll
    for (int u = 0; u < AHEAD; ++u)
#pragma unroll
      for (int v = 0; v < VECS; ++v) a[u][v] = scratch_state(p, min(slot + u, end - 1), h)[e0 + v * 256];
#pragma unroll
    for (int u = 0; u < AHEAD; ++u) {
      if (slot + u >= end) break;
#pragma unroll
      for (int v = 0; v < VECS; ++v) {
#pragma unroll
        for (int j = 0; j < 4; ++j) r[v][j] = fmaf(r[v][j], l.y, fmaf(r[v][j], l.x, a[u][v][j]));
        scratch_state(p, slot + u, h)[e0 + v * 256] = r[v];
      }
    }
  }
}

// The state that a segment starts from, as the lanes of one column group hold it.
template <int ND, bool DIRECT>
__device__ __forceinline__ void load_state(const DecayParams& p, const Segment& g, int h, int group, int lane, f32x4 (&S)[ND]) {
  if (g.j > 0 || !g.last) {
    const f32x4* at = scratch_state(p, g.j > 0 ? g.base + g.j - 1 : p.slots + g.base, h) + (int64_t)group * ND * 64 + lane;
#pragma unroll
    for (int d = 0; d < ND; ++d) S[d] = at[d * 64];
    return;
  }
#pragma unroll
  for (int d = 0; d < ND; ++d) S[d] = f32x4{};
  if (g.in < 0) return;
  const int col = 16 * group + (lane & 15);
  const float* at = p.state + ((int64_t)g.in * p.Hkv + h) * p.Dk * p.Dv + min(col, p.Dv - 1);
#pragma unroll
  for (int d = 0; d < ND; ++d)
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const int key = first_key(DIRECT, d, lane >> 4) + j;
      const float f = at[min(key, p.Dk - 1) * p.Dv];  // unconditional loads, all in flight at once
      S[d][j] = col < p.Dv && key < p.Dk ? f : 0.f;
    }
}

// The state behind a segment: into the pool (OUT, where it is a sequence's last), or what the segment added into its scratch slot.
template <int ND, bool DIRECT, bool OUT>
__device__ __forceinline__ void store_state(const DecayParams& p, const Segment& g, int h, int group, int lane, const f32x4 (&S)[ND]) {
  if constexpr (!OUT) {
    f32x4* at = scratch_state(p, g.base + g.j, h) + (int64_t)group * ND * 64 + lane;
#pragma unroll
    for (int d = 0; d < ND; ++d) at[d * 64] = S[d];
  } else {
    const int col = 16 * group + (lane & 15);
    if (col >= p.Dv) return;
    float* at = p.state + ((int64_t)g.out * p.Hkv + h) * p.Dk * p.Dv + col;
#pragma unroll
    for (int d = 0; d < ND; ++d)
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const int key = first_key(DIRECT, d, lane >> 4) + j;
        if (key < p.Dk) at[key * p.Dv] = S[d][j];
      }
  }
}

// ---- bfloat16: matrix instructions on bf16 operands ---------------------------------------------------------
// Chunks of 32 tokens, 16 x 16 tiles (32 k-values an instruction).  Wave w owns 16 columns of the state and of the output: its part
// of S stays in accumulators for the whole segment.  Lane (i, g) = (lane & 15, lane / 16) holds column i; register j of tile d
// holds key 32 (d / 2) + 8 g + 4 (d & 1) + j, so that two tiles, rounded to bf16, are one operand of the product with the queries
// as they lie in memory.  The order comes for free: the rows of K^T can be read in any order of four.
//   scores   S^T = K Q^T, three of the four tiles, one a wave, through LDS as bf16
//   output   O^T = S0^T Q^T, columns scaled by l^(n+1) in float32, then + V^T P^T
//   state    l^n S + K^T (l^(n-1-m) V): the decayed values are float32, so they enter as the sum of three bf16 numbers
//            (24 bits); the state keeps float32 accuracy.
// Rounded to bf16 are the scores and, for the product with the queries only, the state: what they add to an output is rounded
// to bf16 as well.  The tiles of the next chunk are on their way into LDS (direct loads, two buffers) while this one is worked on.
// What a chunk costs is mostly the latency of its chain (tiles, scores, barrier, products, store); sixteen waves a CU with 16
// columns each hide it better than eight with 32 (152 against 127 us below).
// Measured: one prompt of 16384 tokens, 32 heads of 128 x 128: sums 70 us (268 MB, 3.8 TB/s), scan 14 us, outputs 126 to 146 us (537 MB,
// 3.7 to 4.3 TB/s).  In a round of two workgroups a CU (9400 cycles) the matrix units work for 2300 cycles, LDS for
// 2300, the vector units for 3900, one after the other more than side by side.

constexpr int kChunk = 32;
constexpr int kScoreRow = 80;  // bytes of a row of 32 bf16 scores in LDS, spread over the banks

// 16-byte chunks of a row of WIDTH elements are stored XOR-ed with this key.  LDS serves a 16-byte read in groups of sixteen lanes that
// take rows 0-3 and 12-15 from one lane group and rows 4-11 from its neighbour, whose chunk differs in the lowest bit: with the
// last two bits of the key counting down over the quads of rows, all sixteen fall on distinct banks (counting up, pairs
// collide: 30 % more LDS cycles, the segments of five prompts of 1200 tokens of 16 heads 162 instead of 158 us a call).  The transposing reads of a pair of chunks find theirs distinct as well; those of four
// chunks (the keys) read one half of each and meet the same banks twice whatever the key.
template <int WIDTH>
__device__ __forceinline__ int tile_key(int row) {
  const int down = -(row >> 2) & 3;
  if constexpr (WIDTH >= 128) return ((row & 3) << 2) | down;
  else return (((row >> 1) & 1) << 2) | down;  // (128-byte rows: their lowest bit chooses half of the banks)
}

typedef __attribute__((address_space(3))) const char lds_char;
__device__ __forceinline__ uint32_t lds_address(const char* p) { return (uint32_t)(uintptr_t)(lds_char*)p; }

__device__ __forceinline__ u32x4 lds_read(uint32_t at) { return *(__attribute__((address_space(3))) const u32x4*)(uintptr_t)at; }
__device__ __forceinline__ u32x2 lds_read_columns(uint32_t at) {
  return __builtin_bit_cast(u32x2, __builtin_amdgcn_ds_read_tr16_b64_v4i16((__attribute__((address_space(3))) s16x4*)(uintptr_t)at));
}

// Where a lane reads a tile of rows of WIDTH elements.  Chunk 4 s + c of a row lies at the lane's address for chunk c with bits 6 and
// up XOR-ed with s (tiles start at multiples of 1 KiB): one register a pattern.
template <int WIDTH>
struct TileRows {  // row i (of sixteen, more a constant further on), eight elements from 32 s + 8 g on
  uint32_t at;
  __device__ __forceinline__ void init(int i16, int g4) { at = i16 * WIDTH * 2 + ((g4 ^ tile_key<WIDTH>(i16)) << 4); }
  __device__ __forceinline__ u32x4 read(uint32_t tile, int s) const { return lds_read((tile + at) ^ (s << 6)); }
};
template <int WIDTH>
struct TileColumns {  // rows 8 g .. 8 g + 7 of the columns that the transposing reads hand out, four of them from this lane's address on
  uint32_t at[2];  // the first four rows' and the last four rows'
  // `column`: a multiple of 4 of this lane's own
  __device__ __forceinline__ void init(int g4, int lane, int column) {
#pragma unroll
    for (int y = 0; y < 2; ++y) {
      const int row = 8 * g4 + ((lane & 15) >> 2) + 4 * y;
      at[y] = row * WIDTH * 2 + (((column >> 3) ^ tile_key<WIDTH>(row)) << 4) + ((column & 7) << 1);
    }
  }
  __device__ __forceinline__ u32x4 read(uint32_t tile) const {
    const u32x2 x = lds_read_columns(tile + at[0]), y = lds_read_columns(tile + at[1]);
    return u32x4{x[0], x[1], y[0], y[1]};
  }
};
template <int WIDTH>
struct TileKeys {  // the same rows of columns 32 s + 8 (lane & 3) + 4 odd
  uint32_t at[2];
  __device__ __forceinline__ void init(int g4, int lane) {
#pragma unroll
    for (int y = 0; y < 2; ++y) {
      const int row = 8 * g4 + ((lane & 15) >> 2) + 4 * y;
      at[y] = row * WIDTH * 2 + (((lane & 3) ^ tile_key<WIDTH>(row)) << 4);
    }
  }
  __device__ __forceinline__ u32x4 read(uint32_t tile, int s, int odd) const {
    const u32x2 x = lds_read_columns(((tile + at[0]) ^ (s << 6)) + 8 * odd), y = lds_read_columns(((tile + at[1]) ^ (s << 6)) + 8 * odd);
    return u32x4{x[0], x[1], y[0], y[1]};
  }
};

__device__ __forceinline__ f32x4 mfma_bf16(u32x4 a, u32x4 b, f32x4 c) { return HalfOf<RPA_BF16>::mfma32(a, b, c); }

__device__ __forceinline__ float low_half(uint32_t w) { return __uint_as_float(w << 16); }
__device__ __forceinline__ float high_half(uint32_t w) { return __uint_as_float(w & 0xffff0000u); }

__device__ uint4 decay_zeros;  // 16 bytes of zeros: the source of what a tile holds beyond its rows and columns

// A value that the compiler cannot know to be the same in every turn of a loop: what rare paths derive from it is worked out there and
// not held in registers (or spilled, behind loads that would then be waited for) by all turns.
__device__ __forceinline__ int opaque(int v) {
  asm volatile("" : "+v"(v));
  return v;
}

// A tile of kChunk rows of WIDTH elements on its way into LDS: rows 0 .. n-1 of `cols` elements exist, `stride` elements apart, the
// others become zeros.  Direct loads of 16 bytes a lane, 1 KiB an instruction, complete when this wave's vector-memory counter
// says so; a whole tile takes its lanes' offsets from registers and its base from scalars.
template <int WIDTH, int NT>
struct TileLoad {
  static constexpr int PER_ROW = WIDTH / 8, PIECES = kChunk * PER_ROW, N = PIECES >= NT ? PIECES / NT : 1;  // fewer pieces than threads: the first waves'
  uint32_t at[N];
  int64_t stride;
  int cols;
  // wave w's instruction k fills bytes [(w N + k) 1024, + 1024) of the tile
  static __device__ __forceinline__ int row_of(int thread, int k) { return (((thread >> 6) * N + k) * 64 + (thread & 63)) / PER_ROW; }
  static __device__ __forceinline__ int column_of(int thread, int k) { return (((thread & 63) % PER_ROW) ^ tile_key<WIDTH>(row_of(thread, k))) * 8; }
  __device__ __forceinline__ void init(int64_t stride_, int cols_) {
    stride = stride_; cols = cols_;
#pragma unroll
    for (int k = 0; k < N; ++k) at[k] = ((uint32_t)row_of(threadIdx.x, k) * (uint32_t)stride + column_of(threadIdx.x, k)) * 2;  // 32 rows span less than 2^31 bytes
  }
  __device__ __forceinline__ void start(char* tile, const uint16_t* src, int n) const {
    if (PIECES < NT && (int)threadIdx.x >= PIECES) return;
    const uint32_t to = __builtin_amdgcn_readfirstlane(lds_address(tile) + (threadIdx.x >> 6) * N * 1024);
    if (n >= kChunk && cols >= WIDTH) {
#pragma unroll
      for (int k = 0; k < N; ++k) dma16(to + k * 1024, at[k], src);
    } else {
      const int thread = opaque(threadIdx.x);
#pragma unroll
      for (int k = 0; k < N; ++k) {
        const int row = row_of(thread, k), c = column_of(thread, k);
        const void* from = row < n && c < cols ? (const void*)(src + row * stride + c) : (const void*)&decay_zeros;
        asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %1, off" ::"s"(to + k * 1024), "v"(from) : "memory");
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

template <int DK, int NW, bool OUT>
__global__ __launch_bounds__(64 * NW, DK <= 128 ? 4 : 2) void decay_chunk_bf16_kernel(DecayParams p) {
  constexpr int NT = 64 * NW, DV = 16 * NW, ND = DK / 16;
  constexpr int KB = kChunk * DK * 2, VB = kChunk * DV * 2;
  __shared__ __align__(1024) char sK[2][KB];
  __shared__ __align__(1024) char sV[2][VB];
  __shared__ __align__(1024) char sQ[OUT ? 2 : 1][OUT ? KB : 16];
  __shared__ __align__(16) char sP[OUT ? kChunk * kScoreRow : 16];
  __shared__ __align__(16) float pw[kChunk + 4];  // l^0 .. l^C
  __shared__ __align__(16) float left[kChunk];    // l^(n-1-m) for the n tokens m of a chunk, 0 behind them

  const int slices = (p.Dv + DV - 1) / DV, heads = p.Hkv * slices;
  const int id = blockIdx.x / heads, hs = blockIdx.x - id * heads, h = hs / slices, c0 = (hs - h * slices) * DV;
  if constexpr (OUT) {
    static_assert(sizeof(sK) >= sizeof(StepLds<NT, 4 * NW>), "the short sequences' work uses the tiles' memory");
    if ((int)blockIdx.x >= p.chunk_blocks) {
      beside_chunks<RPA_BF16, DK, NW>(p, blockIdx.x - p.chunk_blocks, heads, slices, (char*)sK);
      return;
    }
  }
  Segment g;
  if (OUT ? !find_segment(p, id, g) : !find_by_slot<false>(p, id, g)) return;
  const int tid = threadIdx.x, lane = tid & 63, w = tid >> 6, i16 = lane & 15, g4 = lane >> 4;
  const int chunks = (g.n + kChunk - 1) / kChunk;
  const uint16_t* q = (const uint16_t*)p.q + (int64_t)g.t0 * p.q_stride + (int64_t)h * p.group * p.Dk;
  const uint16_t* k = (const uint16_t*)p.k + (int64_t)g.t0 * p.k_stride + (int64_t)h * p.Dk;
  const uint16_t* v = (const uint16_t*)p.v + (int64_t)g.t0 * p.v_stride + (int64_t)h * p.Dv + c0;
  const int vcols = min(p.Dv - c0, DV), groups = OUT ? p.group : 1;
  TileLoad<DK, NT> lq, lk;
  TileLoad<DV, NT> lv;
  lk.init(p.k_stride, p.Dk);
  lv.init(p.v_stride, vcols);
  const int64_t first = OUT ? 0 : (int64_t)(chunks - 1) * kChunk;
  lk.start(sK[0], k + first * p.k_stride, g.n);
  lv.start(sV[0], v + first * p.v_stride, g.n);
  if constexpr (OUT) {
    lq.init(p.q_stride, p.Dk);
    lq.start(sQ[0], q, g.n);
  }

  f32x4 S[ND];
#pragma unroll
  for (int d = 0; d < ND; ++d) S[d] = f32x4{};
  if constexpr (OUT) load_state<ND, true>(p, g, h, c0 / 16 + w, lane, S);
  const float rate = p.log_decay[h];
  const float2 full = decay_power(rate, kChunk);
  DecayFactor factor;
  factor.init(full.x, full.y);
  double over = 1.0;
  if (tid <= kChunk) pw[tid] = decay_float(rate, tid);
  if (tid >= 64 && tid < 64 + kChunk) left[tid - 64] = decay_float(rate, kChunk - 1 - (tid - 64));
  if constexpr (OUT) {
    if (tid >= 128 && tid < 160) *(u32x4*)(sP + (tid & 15) * kScoreRow + 32 + (tid >> 4 & 1) * 16) = u32x4{0u, 0u, 0u, 0u};  // the tile of masked scores alone
  }

  TileRows<DK> rows;
  TileKeys<DK> keys;
  TileColumns<DV> columns;
  rows.init(i16, g4);
  keys.init(g4, lane);
  columns.init(g4, lane, 16 * w + 4 * (lane & 3));
  const uint32_t aK = lds_address(sK[0]), aV = lds_address(sV[0]), aQ = lds_address(sQ[0]), aP = lds_address(sP);
  const bool whole = OUT && c0 + 16 * w + 16 <= p.Dv;
  for (int c = 0; c < chunks; ++c) {
    const int n = OUT ? min(g.n - c * kChunk, kChunk) : kChunk;
    const uint32_t tK = aK + (c & 1) * KB, tV = aV + (c & 1) * VB;
    u32x4 vop;  // tokens 8 g .. 8 g + 7 of column i
    for (int gq = 0; gq < groups; ++gq) {
      const int step = c * groups + gq;
      // this step's tiles have arrived, and the other buffers have been read.  Behind the tiles' loads this wave issued the two
      // stores of the step before, which need not be waited for, if it holds 16 columns (`whole`) and that step's chunk was full:
      // the chunks before this one are, and this one is if it has kChunk tokens.  In a part of a chunk a wave without rows to write
      // issues fewer stores, and a wait for two outstanding operations would let the tile itself be one of them.
      if (whole && step > 0 && (gq == 0 || n == kChunk)) wait_loads<2>();
      else wait_loads<0>();
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
      vop = columns.read(tV);
      if constexpr (OUT) {
        const uint32_t tQ = aQ + (step & 1) * KB;
        // scores, decayed and masked: tile (keys 16 a.., queries 16 b..) of S^T
        if (w < 3) {
          const int a = w == 1 ? 1 : 0, b = w == 0 ? 0 : 1;
          f32x4 acc = {};
#pragma unroll
          for (int ks = 0; ks < DK / 32; ++ks)
            acc = mfma_bf16(rows.read(tK + a * 16 * DK * 2, ks), rows.read(tQ + b * 16 * DK * 2, ks), acc);
          const int own = opaque(lane), t = 16 * b + (own & 15), s0 = 16 * a + 4 * (own >> 4);
          float f[4];
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            const int gap = t - s0 - e;
            f[e] = gap >= 0 ? acc[e] * pw[max(gap, 0)] : 0.f;  // chosen, not multiplied: masked scores may be infinite
          }
          *(u32x2*)(sP + t * kScoreRow + s0 * 2) = u32x2{pack_bf16(f[0], f[1]), pack_bf16(f[2], f[3])};
        }
        // O^T of this wave's columns: lane i = token, registers = columns 4 g + j; its product with the state needs no scores
        f32x4 o[2] = {};
#pragma unroll
        for (int s = 0; s < ND / 2; ++s) {
          const u32x4 st = {pack_bf16(S[2 * s][0], S[2 * s][1]), pack_bf16(S[2 * s][2], S[2 * s][3]),
                            pack_bf16(S[2 * s + 1][0], S[2 * s + 1][1]), pack_bf16(S[2 * s + 1][2], S[2 * s + 1][3])};
#pragma unroll
          for (int tt = 0; tt < 2; ++tt) o[tt] = mfma_bf16(st, rows.read(tQ + tt * 16 * DK * 2, s), o[tt]);
        }
#pragma unroll
        for (int tt = 0; tt < 2; ++tt) o[tt] *= pw[16 * tt + i16 + 1];
        // A value that is not finite would meet the zeros of the masked scores as well, and 0 x Inf is NaN: such values stay out of
        // the product, and the rows that see one become NaN by hand.
        uint32_t ones = 0;
#pragma unroll
        for (int e = 0; e < 4; ++e) ones |= (vop[e] & 0x7f807f80u) + 0x00800080u;  // bit 15 or 31: an exponent of all ones
        const bool odd = __any((ones & 0x80008000u) != 0);
        u32x4 vo = vop;
        if (odd) {
#pragma unroll
          for (int e = 0; e < 4; ++e) vo[e] = finite_halves(vo[e]);
        }
        __syncthreads();
#pragma unroll
        for (int tt = 0; tt < 2; ++tt) o[tt] = mfma_bf16(vo, lds_read(aP + (16 * tt + i16) * kScoreRow + g4 * 16), o[tt]);
        if (odd) {
          const int at = 16 * w + (opaque(lane) & 15);
          int bad = 0;
          for (; bad < n; ++bad) {
            const uint16_t bits = *(const uint16_t*)(sV[c & 1] + bad * DV * 2 + (((at >> 3) ^ tile_key<DV>(bad)) << 4) + ((at & 7) << 1));
            if ((bits & 0x7f80) == 0x7f80) break;
          }
#pragma unroll
          for (int j = 0; j < 4; ++j) {
            const int first_bad = __shfl(bad, 4 * g4 + j);
#pragma unroll
            for (int tt = 0; tt < 2; ++tt) o[tt][j] = 16 * tt + i16 >= first_bad ? __builtin_nanf("") : o[tt][j];
          }
        }
        // four columns a lane, 32 bytes of a row a wave
        char* out = (char*)p.out + (((int64_t)(g.t0 + c * kChunk) * p.Hq + h * p.group + gq) * p.Dv + c0 + 16 * w) * 2;
        const uint32_t at = (uint32_t)(i16 * p.Hq * p.Dv + 4 * g4) * 2, half = (uint32_t)(16 * p.Hq * p.Dv) * 2;
        const u32x2 lo = {pack_bf16(o[0][0] * p.scale, o[0][1] * p.scale), pack_bf16(o[0][2] * p.scale, o[0][3] * p.scale)};
        const u32x2 hi = {pack_bf16(o[1][0] * p.scale, o[1][1] * p.scale), pack_bf16(o[1][2] * p.scale, o[1][3] * p.scale)};
        if (whole && n == kChunk) {
          *(u32x2*)(out + at) = lo;
          *(u32x2*)(out + half + at) = hi;
        } else if (c0 + 16 * w + 4 * g4 < p.Dv) {
          if (i16 < n) *(u32x2*)(out + at) = lo;
          if (i16 + 16 < n) *(u32x2*)(out + half + at) = hi;
        }
      }
    }
    if (OUT && c == chunks - 1 && (!g.last || g.out < 0)) break;  // nobody reads the state behind this chunk
    // OUT: the state is decayed over the chunk.  Otherwise it starts from zero, the chunks come last to first (all are whole) and
    // their tokens enter with their decay to the end of the segment, which leaves the state alone.
    float behind = 1.f;
    if constexpr (OUT) {
      const float l = n < kChunk ? pw[n] : factor.next();
#pragma unroll
      for (int d = 0; d < ND; ++d) S[d] *= l;
    } else {
      behind = (float)over;
      over *= (double)full.x + (double)full.y;
    }
    float4 w0 = *(const float4*)&left[8 * g4], w1 = *(const float4*)&left[8 * g4 + 4];
    if constexpr (!OUT) {
      w0.x *= behind; w0.y *= behind; w0.z *= behind; w0.w *= behind;
      w1.x *= behind; w1.y *= behind; w1.z *= behind; w1.w *= behind;
    }
    u32x4 hi, mid, lo;
    split3(vop, w0, w1, hi, mid, lo);
#pragma unroll
    for (int d = 0; d < ND; ++d) {
      const u32x4 kt = keys.read(tK, d >> 1, d & 1);
      S[d] = mfma_bf16(kt, lo, S[d]);
      S[d] = mfma_bf16(kt, mid, S[d]);
      S[d] = mfma_bf16(kt, hi, S[d]);
    }
  }
  if (OUT && (!g.last || g.out < 0)) return;
  store_state<ND, true, OUT>(p, g, h, c0 / 16 + w, opaque(lane), S);  // (addresses of its own, not those of the beginning kept through the loop)
}

// ---- float32 and half, and bf16 rows that are not aligned: matrix instructions on float32 operands --------------------------
// The same chunks, tiles and owners with 16 x 16 x 4 float32 instructions (a sixteenth of the bf16 rate), elements widened to
// float32 on their way into LDS.  Nothing is rounded on the way, and any row the checks allow can be read; the tiles of the next
// chunk wait in registers (six pieces of four elements a thread at 128 keys).  Lane (i, g), register j of tile d of the state: key
// 16 d + 4 g + j of column i.  Measured: four float32 prompts of 450 to 1100 tokens, 16 + 8 heads of 64 x 96: sums 12.6 us, scan 7.6 us,
// outputs 34 us: chains of four chunks of two query heads, 8000 cycles of matrix instructions in each at the two waves that
// share a SIMD.
constexpr int kWidePad = 4;  // floats behind a row of LDS: rows start four banks apart

template <int DT>
__device__ __forceinline__ float4 load_four(const void* src, int64_t at, bool vec) {
  float f[4];
  if constexpr (DT == RPA_F32) {
    if (vec) return *(const float4*)((const float*)src + at);
  } else if (vec) {
    const u32x2 w = *(const u32x2*)((const uint16_t*)src + at);
    if constexpr (DT == RPA_BF16) {
      return make_float4(low_half(w[0]), high_half(w[0]), low_half(w[1]), high_half(w[1]));
    } else {
      typedef _Float16 f16x4 __attribute__((ext_vector_type(4)));
      const f16x4 x = __builtin_bit_cast(f16x4, w);
      return make_float4((float)x[0], (float)x[1], (float)x[2], (float)x[3]);
    }
  }
#pragma unroll
  for (int e = 0; e < 4; ++e) f[e] = load_elem<DT>(src, at + e);
  return make_float4(f[0], f[1], f[2], f[3]);
}

template <int DT, int WIDTH, int NT>
struct WideTile {
  static constexpr int PER_ROW = WIDTH / 4, N = kChunk * PER_ROW / NT, PITCH = WIDTH + kWidePad;
  float4 r[N];
  __device__ __forceinline__ void load(const void* src, int64_t at, int64_t stride, int n, int cols, bool vec) {
#pragma unroll
    for (int k = 0; k < N; ++k) {
      const int idx = threadIdx.x + k * NT, row = idx / PER_ROW, c = (idx % PER_ROW) * 4;
      const bool in = row < n && c < cols;
      const float4 x = load_four<DT>(src, at + (in ? row * stride + c : 0), vec);  // unconditional: all in flight at once
      r[k] = in ? x : make_float4(0.f, 0.f, 0.f, 0.f);
    }
  }
  __device__ __forceinline__ void store(float* tile) const {
#pragma unroll
    for (int k = 0; k < N; ++k) {
      const int idx = threadIdx.x + k * NT, row = idx / PER_ROW, c = (idx % PER_ROW) * 4;
      *(float4*)(tile + row * PITCH + c) = r[k];
    }
  }
};

__device__ __forceinline__ f32x4 mfma_f32(float a, float b, f32x4 c) { return __builtin_amdgcn_mfma_f32_16x16x4f32(a, b, c, 0, 0, 0); }

template <int DT, int DK, int NW, bool OUT>
__global__ __launch_bounds__(64 * NW) void decay_chunk_wide_kernel(DecayParams p) {
  constexpr int NT = 64 * NW, DV = 16 * NW, ND = DK / 16;
  constexpr int KP = DK + kWidePad, VP = DV + kWidePad, PP = kChunk + kWidePad;
  __shared__ __align__(16) float sQ[OUT ? kChunk * KP : 4];
  __shared__ __align__(16) float sK[kChunk * KP];
  __shared__ __align__(16) float sV[kChunk * VP];
  __shared__ __align__(16) float sP[OUT ? kChunk * PP : 4];
  __shared__ __align__(16) float pw[kChunk + 4];
  __shared__ __align__(16) float left[kChunk];

  const int slices = (p.Dv + DV - 1) / DV, heads = p.Hkv * slices;
  const int id = blockIdx.x / heads, hs = blockIdx.x - id * heads, h = hs / slices, c0 = (hs - h * slices) * DV;
  if constexpr (OUT) {
    static_assert(sizeof(sK) >= sizeof(StepLds<NT, 4 * NW>), "the short sequences' work uses the tiles' memory");
    if ((int)blockIdx.x >= p.chunk_blocks) {
      beside_chunks<DT, DK, NW>(p, blockIdx.x - p.chunk_blocks, heads, slices, (char*)sK);
      return;
    }
  }
  Segment g;
  if (OUT ? !find_segment(p, id, g) : !find_by_slot<false>(p, id, g)) return;
  const int tid = threadIdx.x, lane = tid & 63, w = tid >> 6, i16 = lane & 15, g4 = lane >> 4;
  const int chunks = (g.n + kChunk - 1) / kChunk;
  const int vcols = min(p.Dv - c0, DV), groups = OUT ? p.group : 1;
  const int64_t q0 = (int64_t)g.t0 * p.q_stride + (int64_t)h * p.group * p.Dk, k0 = (int64_t)g.t0 * p.k_stride + (int64_t)h * p.Dk,
                v0 = (int64_t)g.t0 * p.v_stride + (int64_t)h * p.Dv + c0;
  WideTile<DT, DK, NT> nq, nk;
  WideTile<DT, DV, NT> nv;
  const int64_t first = OUT ? 0 : (int64_t)(chunks - 1) * kChunk;  // states alone: last chunk first
  if constexpr (OUT) nq.load(p.q, q0, p.q_stride, g.n, p.Dk, p.vec);
  nk.load(p.k, k0 + first * p.k_stride, p.k_stride, g.n, p.Dk, p.vec);
  nv.load(p.v, v0 + first * p.v_stride, p.v_stride, g.n, vcols, p.vec);

  f32x4 S[ND];
#pragma unroll
  for (int d = 0; d < ND; ++d) S[d] = f32x4{};
  if constexpr (OUT) load_state<ND, false>(p, g, h, c0 / 16 + w, lane, S);
  const float rate = p.log_decay[h];
  const float2 full = decay_power(rate, kChunk);
  DecayFactor factor;
  factor.init(full.x, full.y);
  double over = 1.0;
  if (tid <= kChunk) pw[tid] = decay_float(rate, tid);
  if (tid >= 64 && tid < 64 + kChunk) left[tid - 64] = decay_float(rate, kChunk - 1 - (tid - 64));
  if constexpr (OUT) {
    if (tid >= 128 && tid < 192) *(float4*)(sP + (tid & 15) * PP + 16 + ((tid >> 4) & 3) * 4) = make_float4(0.f, 0.f, 0.f, 0.f);
  }

  for (int c = 0; c < chunks; ++c) {
    const int n = OUT ? min(g.n - c * kChunk, kChunk) : kChunk;
    float vv[2][4];  // tokens 16 b + 4 g + e of column i
    for (int gq = 0; gq < groups; ++gq) {
      __syncthreads();  // the tiles of the step before have been read
      if constexpr (OUT) nq.store(sQ);
      if (gq == 0) {
        nk.store(sK);
        nv.store(sV);
        if (n < kChunk && tid < kChunk) left[tid] = tid < n ? pw[n - 1 - tid] : 0.f;
      }
      __syncthreads();
      const bool on = gq == groups - 1;
      const int cn = c + (on ? 1 : 0);
      if (cn < chunks) {
        const int64_t ahead = (int64_t)(OUT ? cn : chunks - 1 - cn) * kChunk;
        const int rows = OUT ? g.n - cn * kChunk : kChunk;
        if constexpr (OUT) nq.load(p.q, q0 + ahead * p.q_stride + (on ? 0 : (gq + 1) * p.Dk), p.q_stride, rows, p.Dk, p.vec);
        if (on) {
          nk.load(p.k, k0 + ahead * p.k_stride, p.k_stride, rows, p.Dk, p.vec);
          nv.load(p.v, v0 + ahead * p.v_stride, p.v_stride, rows, vcols, p.vec);
        }
      }
#pragma unroll
      for (int b = 0; b < 2; ++b)
#pragma unroll
        for (int e = 0; e < 4; ++e) vv[b][e] = sV[(16 * b + 4 * g4 + e) * VP + 16 * w + i16];
      if constexpr (OUT) {
        if (w < 3) {  // scores: tile (keys 16 a.., queries 16 b..) of S^T
          const int a = w == 1 ? 1 : 0, b = w == 0 ? 0 : 1;
          f32x4 acc = {};
#pragma unroll
          for (int d = 0; d < ND; ++d) {
            const float4 x = *(const float4*)&sK[(16 * a + i16) * KP + 16 * d + 4 * g4], y = *(const float4*)&sQ[(16 * b + i16) * KP + 16 * d + 4 * g4];
            acc = mfma_f32(x.x, y.x, acc); acc = mfma_f32(x.y, y.y, acc); acc = mfma_f32(x.z, y.z, acc); acc = mfma_f32(x.w, y.w, acc);
          }
          const int t = 16 * b + i16, s0 = 16 * a + 4 * g4;
          float f[4];
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            const int gap = t - s0 - e;
            f[e] = gap >= 0 ? acc[e] * pw[max(gap, 0)] : 0.f;
          }
          *(float4*)&sP[t * PP + s0] = make_float4(f[0], f[1], f[2], f[3]);
        }
        f32x4 o[2] = {};
#pragma unroll
        for (int d = 0; d < ND; ++d)
#pragma unroll
          for (int tt = 0; tt < 2; ++tt) {
            const float4 y = *(const float4*)&sQ[(16 * tt + i16) * KP + 16 * d + 4 * g4];
            o[tt] = mfma_f32(S[d][0], y.x, o[tt]); o[tt] = mfma_f32(S[d][1], y.y, o[tt]);
            o[tt] = mfma_f32(S[d][2], y.z, o[tt]); o[tt] = mfma_f32(S[d][3], y.w, o[tt]);
          }
#pragma unroll
        for (int tt = 0; tt < 2; ++tt) o[tt] *= pw[16 * tt + i16 + 1];
        bool fine = true;
#pragma unroll
        for (int b = 0; b < 2; ++b)
#pragma unroll
          for (int e = 0; e < 4; ++e) fine = fine && __builtin_isfinite(vv[b][e]);
        const bool odd = __any(!fine);  // as in the bf16 kernel: kept out of the product, NaN by hand
        __syncthreads();
#pragma unroll
        for (int b = 0; b < 2; ++b)
#pragma unroll
          for (int tt = b; tt < 2; ++tt) {
            const float4 y = *(const float4*)&sP[(16 * tt + i16) * PP + 16 * b + 4 * g4];
            const float s4[4] = {y.x, y.y, y.z, y.w};
#pragma unroll
            for (int e = 0; e < 4; ++e) o[tt] = mfma_f32(odd && !__builtin_isfinite(vv[b][e]) ? 0.f : vv[b][e], s4[e], o[tt]);
          }
        if (odd) {
          int bad = 0;
          for (; bad < n; ++bad)
            if (!__builtin_isfinite(sV[bad * VP + 16 * w + i16])) break;
#pragma unroll
          for (int j = 0; j < 4; ++j) {
            const int first_bad = __shfl(bad, 4 * g4 + j);
#pragma unroll
            for (int tt = 0; tt < 2; ++tt) o[tt][j] = 16 * tt + i16 >= first_bad ? __builtin_nanf("") : o[tt][j];
          }
        }
        const int at = c0 + 16 * w + 4 * g4;
#pragma unroll
        for (int tt = 0; tt < 2; ++tt) {
          const int t = 16 * tt + i16;
          if (t >= n || at >= p.Dv) continue;
          const int64_t to = ((int64_t)(g.t0 + c * kChunk + t) * p.Hq + h * p.group + gq) * p.Dv + at;
          const f32x4 x = o[tt] * p.scale;
          if constexpr (DT == RPA_F32) *(f32x4*)((float*)p.out + to) = x;
          else *(u32x2*)((uint16_t*)p.out + to) = u32x2{Half16<DT>::pack(x[0], x[1]), Half16<DT>::pack(x[2], x[3])};
        }
      }
    }
    if (OUT && c == chunks - 1 && (!g.last || g.out < 0)) break;  // nobody reads the state behind this chunk
    float behind = 1.f;
    if constexpr (OUT) {
      const float l = n < kChunk ? pw[n] : factor.next();
#pragma unroll
      for (int d = 0; d < ND; ++d) S[d] *= l;
    } else {
      behind = (float)over;
      over *= (double)full.x + (double)full.y;
    }
#pragma unroll
    for (int b = 0; b < 2; ++b) {
      const float4 lf = *(const float4*)&left[16 * b + 4 * g4];
      const float l4[4] = {lf.x, lf.y, lf.z, lf.w};
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        const float x = vv[b][e] * (l4[e] * behind);
#pragma unroll
        for (int d = 0; d < ND; ++d) S[d] = mfma_f32(sK[(16 * b + 4 * g4 + e) * KP + 16 * d + i16], x, S[d]);
      }
    }
  }
  if (OUT && (!g.last || g.out < 0)) return;
  store_state<ND, false, OUT>(p, g, h, c0 / 16 + w, opaque(lane), S);
}

// Rows of 16-byte aligned bf16 take the bf16 kernel, everything else the float32 one; eight waves (128 columns) a workgroup, four
// where the values have at most 64.
template <int DT, int DK, int NW, bool DIRECT>
void launch_tiles(hipStream_t stream, DecayParams p) {
  const int slices = (p.Dv + 16 * NW - 1) / (16 * NW), heads = p.Hkv * slices;
  p.chunk_blocks = (p.first_ids + p.slots) * heads;
  const dim3 block(64 * NW), sums(p.slots * heads), outs(p.chunk_blocks + p.S * heads + kClearBlocks);
  if (p.slots > 0) {
    if constexpr (DIRECT) hipLaunchKernelGGL((decay_chunk_bf16_kernel<DK, NW, false>), sums, block, 0, stream, p);
    else hipLaunchKernelGGL((decay_chunk_wide_kernel<DT, DK, NW, false>), sums, block, 0, stream, p);
    hipLaunchKernelGGL(decay_scan_kernel, dim3(p.scratch_vecs / 512, p.Hkv, p.slots), dim3(256), 0, stream, p);
  }
  if constexpr (DIRECT) hipLaunchKernelGGL((decay_chunk_bf16_kernel<DK, NW, true>), outs, block, 0, stream, p);
  else hipLaunchKernelGGL((decay_chunk_wide_kernel<DT, DK, NW, true>), outs, block, 0, stream, p);
}

template <int DT, int DK, bool DIRECT>
void launch_columns(hipStream_t stream, const DecayParams& p) {
  if (p.Dv <= 64) launch_tiles<DT, DK, 4, DIRECT>(stream, p);
  else launch_tiles<DT, DK, 8, DIRECT>(stream, p);
}

template <int DT, bool DIRECT>
void launch_keys(hipStream_t stream, const DecayParams& p) {
  if (p.Dk <= 64) launch_columns<DT, 64, DIRECT>(stream, p);
  else if (p.Dk <= 128) launch_columns<DT, 128, DIRECT>(stream, p);
  else launch_columns<DT, 256, DIRECT>(stream, p);
}

}  // namespace

int launch_decay_chunk(hipStream_t stream, const DecayParams& p) {
  if (p.dtype == RPA_BF16 && p.vec) launch_keys<RPA_BF16, true>(stream, p);
  else if (p.dtype == RPA_BF16) launch_keys<RPA_BF16, false>(stream, p);
  else if (p.dtype == RPA_F16) launch_keys<RPA_F16, false>(stream, p);
  else launch_keys<RPA_F32, false>(stream, p);
  return (int)hipGetLastError();
}

}  // namespace rpa
