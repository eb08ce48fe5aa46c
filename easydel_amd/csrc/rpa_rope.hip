// Append with rotation: queries turned into their output, keys turned into the pages, values copied into the pages.
//
// A pair (a, b) of a head and the cosine c and sine s of its angle at the token's position become
//     a' = a c - b s,    b' = b c + a s.
// Every element is read once and written once, with a few operations in between: the work is bound by HBM for prompt
// chunks and by the chain of dependent loads (sequence search -> context length -> table row and page id -> data) for
// decode rows.  A workgroup owns one token, so the chain is walked once per token and by all tokens at once; its
// threads share out the token's heads in pieces of 2 * VEC elements, the most that aligned 16-byte accesses carry.
// Measured (bf16, 32 + 8 heads of 128): one token 4.0 us, 256 decode rows 5.8 us (the chain), prompt chunks of 8192 tokens 37 us =
// 5.5 TB/s, where a large copy reaches 5.1; latent pages, 128 heads of 64 beside rows of 512: 256 rows 7.7 us, 4096 tokens 27 us =
// 5.4 TB/s.
#include "rpa_rope.h"

namespace rpa {

namespace {

template <int BYTES> struct Raw;
template <> struct Raw<16> { typedef uint4 t; };
template <> struct Raw<8> { typedef uint2 t; };
template <> struct Raw<4> { typedef uint32_t t; };
template <> struct Raw<2> { typedef uint16_t t; };
template <> struct Raw<1> { typedef uint8_t t; };

template <int DT>
__device__ __forceinline__ float bits_to_float(const unsigned char* b) {
  if constexpr (DT == RPA_F32) return *(const float*)b;
  else if constexpr (DT == RPA_BF16) return bf16_bits_to_float(*(const uint16_t*)b);
  else return (float)*(const _Float16*)b;
}

// The bare cast into an fp8 cache: round to nearest even, what rounds beyond 448 becomes NaN (464 is the tie, which rounds
// to the even 448).
__device__ __forceinline__ uint8_t fp8_cast(float x) {
  const float c = __builtin_fminf(__builtin_fmaxf(x, -448.f), 448.f);
  const int w = __builtin_amdgcn_cvt_pk_fp8_f32(c, c, 0, false);
  const bool in = __builtin_fabsf(x) <= 464.f;  // false for NaN
  return in ? (uint8_t)(w & 0xff) : (uint8_t)(0x7f | ((__float_as_uint(x) >> 24) & 0x80));
}

template <int DT>
__device__ __forceinline__ void float_to_bits(unsigned char* b, float f) {
  if constexpr (DT == RPA_F32) *(float*)b = f;
  else if constexpr (DT == RPA_BF16) *(uint16_t*)b = float_to_bf16_bits(f);
  else if constexpr (DT == RPA_F16) *(_Float16*)b = (_Float16)f;
  else *b = fp8_cast(f);
}

// N elements from / to memory aligned to the whole group.
template <int DT, int N>
__device__ __forceinline__ void load_group(const char* p, float* f) {
  constexpr int E = ElemBytes<DT>::v;
  typedef typename Raw<N * E>::t R;
  const R r = *(const R*)p;
  unsigned char b[N * E];
  __builtin_memcpy(b, &r, N * E);
#pragma unroll
  for (int i = 0; i < N; ++i) f[i] = bits_to_float<DT>(b + i * E);
}

template <int DT, int N>
__device__ __forceinline__ void store_group(char* p, const float* f) {
  constexpr int E = ElemBytes<DT>::v;
  typedef typename Raw<N * E>::t R;
  unsigned char b[N * E];
#pragma unroll
  for (int i = 0; i < N; ++i) float_to_bits<DT>(b + i * E, f[i]);
  R r;
  __builtin_memcpy(&r, b, N * E);
  *(R*)p = r;
}

template <int N>
__device__ __forceinline__ void load_floats(const float* p, float* f) {
  if constexpr (N >= 4) {
#pragma unroll
    for (int i = 0; i < N; i += 4) {
      const float4 v = *(const float4*)(p + i);
      f[i] = v.x; f[i + 1] = v.y; f[i + 2] = v.z; f[i + 3] = v.w;
    }
  } else {
#pragma unroll
    for (int i = 0; i < N; ++i) f[i] = p[i];
  }
}

// Piece `piece` of a head row: its two groups of VEC elements, starting at elements d0 and d1, turned if the piece lies in
// the turning part.  Products and sums are rounded one by one (no contraction into fused multiply-adds), so that the
// result is the same here, in the quantising write, and in any other float32 evaluation of the two formulas.
template <int SRC, int VEC>
__device__ __forceinline__ void load_piece(const char* head, const float* angles, int half, int neox, int piece, bool key,
                                           float* f, int& d0, int& d1) {
#pragma clang fp contract(off)
  constexpr int E = ElemBytes<SRC>::v;
  const bool turn = key && piece * VEC < half;
  const bool split = turn && neox;
  d0 = split ? piece * VEC : piece * 2 * VEC;
  d1 = split ? d0 + half : d0 + VEC;
  load_group<SRC, VEC>(head + (int64_t)d0 * E, f);
  load_group<SRC, VEC>(head + (int64_t)d1 * E, f + VEC);
  if (!turn) return;
  float c[VEC], s[VEC];
  load_floats<VEC>(angles + piece * VEC, c);
  load_floats<VEC>(angles + half + piece * VEC, s);
#pragma unroll
  for (int i = 0; i < VEC; ++i) {
    const float a = neox ? f[i] : f[2 * i], b = neox ? f[VEC + i] : f[2 * i + 1];
    const float ac = a * c[i], bs = b * s[i], bc = b * c[i], as = a * s[i];
    const float x = ac - bs, y = bc + as;
    if (neox) { f[i] = x; f[VEC + i] = y; } else { f[2 * i] = x; f[2 * i + 1] = y; }
  }
}

__device__ __forceinline__ int rope_live(const RopeParams& p) { return p.num_seqs ? min(p.num_seqs[0], p.S) : p.S; }

__device__ __forceinline__ const float* angle_row(const RopeParams& p, int t, int pos) {
  int row = p.positions ? p.positions[t] : pos;
  row = min(max(row, 0), p.table_rows - 1);
  return p.cos_sin + (int64_t)row * p.rope;
}

// Where token t's rows go: its cache position and the byte offset of its row in the pages, -1 if it is not written.
struct Place {
  int pos;
  int64_t row;
};
__device__ __forceinline__ Place place_of(const RopeParams& p, int n_live, int t) {
  const int i = find_seq_wave(p.qsl, n_live, t);
  Place w;
  w.pos = p.context_lens[i] - (p.qsl[i + 1] - p.qsl[i]) + (t - p.qsl[i]);
  w.row = -1;
  if (w.pos < 0) return w;
  const int j = w.pos / p.page_size;
  if (j >= p.M) return w;
  const int page = p.block_tables[(int64_t)i * p.M + j];
  if (page < 0 || page >= p.P) return w;
  w.row = (int64_t)page * p.page_stride + (int64_t)(w.pos - j * p.page_size) * p.token_stride;
  return w;
}

// The token's query heads, by the whole workgroup; rows of padded tokens become zeros.
template <int SRC, int VEC>
__device__ __forceinline__ void turn_queries(const RopeParams& p, int t, const float* angles, bool live, int tid, int nthreads) {
  constexpr int E = ElemBytes<SRC>::v;
  if (!live && p.q_in_place) return;
  const int per = p.D / (2 * VEC), half = p.rope >> 1;
  const char* src = (const char*)p.q + (int64_t)t * p.q_stride * E;
  char* dst = (char*)p.q_out + (int64_t)t * p.Hq * p.D * E;
  for (int k = tid; k < p.Hq * per; k += nthreads) {
    const int h = k / per, piece = k - h * per;
    const int64_t at = (int64_t)h * p.D * E;
    float f[2 * VEC];
    int d0 = piece * 2 * VEC, d1 = d0 + VEC;
    if (live) {
      load_piece<SRC, VEC>(src + at, angles, half, p.neox, piece, true, f, d0, d1);
    } else {
#pragma unroll
      for (int i = 0; i < 2 * VEC; ++i) f[i] = 0.f;
    }
    store_group<SRC, VEC>(dst + at + d0 * E, f);
    store_group<SRC, VEC>(dst + at + d1 * E, f + VEC);
  }
}

// ---- plain pages ------------------------------------------------------------------------------------------
template <int SRC, int KV, int VEC>
__global__ __launch_bounds__(256) void rope_append_kernel(RopeParams p) {
  constexpr int E = ElemBytes<SRC>::v, EK = ElemBytes<KV>::v;
  const int t = blockIdx.x, tid = threadIdx.x;
  const int n_live = rope_live(p);
  const bool live = n_live > 0 && t >= p.qsl[0] && t < p.qsl[n_live];
  if (!live) {
    turn_queries<SRC, VEC>(p, t, nullptr, false, tid, 256);
    return;
  }
  const Place w = place_of(p, n_live, t);
  const float* angles = angle_row(p, t, w.pos);
  turn_queries<SRC, VEC>(p, t, angles, true, tid, 256);
  if (w.row < 0) return;
  const int per = p.Dp / (2 * VEC), half = p.rope >> 1;  // pieces of a stored row, its padding included
  for (int k = tid; k < 2 * p.Hkv * per; k += 256) {
    const int c = k / per, piece = k - c * per;
    const bool key = c < p.Hkv;
    const int h = key ? c : c - p.Hkv;
    const char* src = (key ? (const char*)p.k + (int64_t)t * p.k_stride * E : (const char*)p.v + (int64_t)t * p.v_stride * E) + (int64_t)h * p.D * E;
    char* dst = (key ? p.k_pages : p.v_pages) + w.row + h * p.head_stride;
    int d0 = piece * 2 * VEC, d1 = d0 + VEC;
    if (SRC == KV && d0 < p.D && !(key && piece * VEC < half)) {  // nothing to compute: the bits themselves
      typedef typename Raw<VEC * E>::t R;
      *(R*)(dst + d0 * E) = *(const R*)(src + d0 * E);
      *(R*)(dst + d1 * E) = *(const R*)(src + d1 * E);
      continue;
    }
    float f[2 * VEC];
    if (d0 < p.D) {
      load_piece<SRC, VEC>(src, angles, half, p.neox, piece, key, f, d0, d1);
    } else {
#pragma unroll
      for (int i = 0; i < 2 * VEC; ++i) f[i] = 0.f;
    }
    store_group<KV, VEC>(dst + d0 * EK, f);
    store_group<KV, VEC>(dst + d1 * EK, f + VEC);
  }
}

// ---- scaled 8-bit pages -----------------------------------------------------------------------------------
// quant and decode of the quantising scatter (rpa_scatter.hip), one value at a time.
template <int KVT>
__device__ __forceinline__ uint32_t quant1(float a) {
  if constexpr (KVT == RPA_FP8_E4M3) {
    a = fminf(fmaxf(a, -448.f), 448.f);
    return (uint32_t)__builtin_amdgcn_cvt_pk_fp8_f32(a, a, 0, false) & 0xff;
  } else {
    return (uint32_t)(int)rintf(fminf(fmaxf(a, -127.f), 127.f)) & 0xff;
  }
}
template <int KVT>
__device__ __forceinline__ float decode1(uint8_t c) {
  if constexpr (KVT == RPA_FP8_E4M3) return fp8_e4m3_to_float(c);
  else return (float)(int8_t)c;
}

template <int KVT, int VEC>
__device__ __forceinline__ void store_codes(unsigned char* dst, const float* f, float scale) {
  if constexpr (VEC == 4) {
    uint32_t w = 0;
#pragma unroll
    for (int i = 0; i < 4; ++i) w |= quant1<KVT>(f[i] / scale) << (8 * i);
    *(uint32_t*)dst = w;
  } else {
#pragma unroll
    for (int i = 0; i < VEC; ++i) dst[i] = (unsigned char)quant1<KVT>(f[i] / scale);
  }
}

// Largest i in [0, n) with qsl[i] / page_size + 2 i <= id, by the whole wavefront (find_seq_wave's search over another
// strictly increasing sequence).
__device__ __forceinline__ int find_run_wave(const int32_t* qsl, int n, int page_size, int id) {
  const int lane = threadIdx.x & 63;
  int lo = 0, hi = n;
  while (hi - lo > 1) {
    const int stride = (hi - lo + 63) >> 6;
    const int idx = lo + lane * stride;
    const bool le = idx < hi && qsl[idx] / page_size + 2 * idx <= id;
    const int last = __popcll(__ballot(le)) - 1;
    lo += last * stride;
    hi = min(lo + stride, hi);
  }
  return lo;
}

// A run is the new tokens one sequence writes to one page.  Runs are numbered without a plan: a sequence of n tokens from
// qsl[i] on touches at most (n - 1) / page_size + 2 pages, and floor(qsl[i] / page_size) + 2 i leaves room for as many
// ahead of the next sequence's first number.  One workgroup codes one run of one combined head by the rule of the quantising
// scatter: amax over the (turned) values, the new scale, old codes again if it grew, new codes.  Its threads hold the turned
// values between the maximum and the codes (64 tokens of 128 elements: four pieces of eight a thread); of longer runs the
// pieces behind those are read and turned again, from the caches.  (64 decode rows and 2048 prompt
// tokens of 40 + 8 heads into fp8 pages: 26 us, of which the queries alone take 10 and the runs alone 18; a chain of nine dependent
// loads bounds a run.  A wave a run, with everything turned twice, took 37 us; all of a thread's pieces loaded ahead of the first
// one's use 29 us, with 113 registers instead of 88.)
constexpr int kHold = 4;

template <int SRC, int KVT, int VEC>
__device__ __forceinline__ void append_run(const RopeParams& p, int n_live, int run, int c, float* most) {
  constexpr int E = ElemBytes<SRC>::v;
  const int tid = threadIdx.x;
  const int i = find_run_wave(p.qsl, n_live, p.page_size, run);
  const int q0 = p.qsl[i], q_len = p.qsl[i + 1] - q0;
  const int ctx = p.context_lens[i];
  if (q_len <= 0 || q0 < 0) return;
  const int pos0 = max(ctx - q_len, 0);                        // first position written
  const int j = pos0 / p.page_size + (run - (q0 / p.page_size + 2 * i));
  const int64_t begin = (int64_t)j * p.page_size;              // first position of the page
  if (j < 0 || j >= p.M || begin >= ctx) return;
  const int page = p.block_tables[(int64_t)i * p.M + j];
  if (page < 0 || page >= p.P) return;
  const int pos = max(pos0, (int)begin);
  const int first = pos - (int)begin;
  const int t0 = q0 + pos - (ctx - q_len);                     // the run's first token
  const int n = min(min(ctx, (int)begin + p.page_size) - pos, p.T - t0);
  if (n <= 0) return;
  const bool key = !(c & 1);
  const int h = c >> 1, half = p.rope >> 1, per = p.D / (2 * VEC), pieces = n * per;
  const int64_t stride = key ? p.k_stride : p.v_stride;
  const char* src = (const char*)(key ? p.k : p.v) + ((int64_t)t0 * stride + (int64_t)h * p.D) * E;
  unsigned char* dst = (unsigned char*)p.k_pages + (int64_t)page * p.page_stride + (int64_t)c * p.Dp;
  const int64_t dst_row = p.token_stride;
  const int64_t si = (int64_t)page * p.C + c;
  const float old_scale = first == 0 ? 0.f : p.scales[si];
  float held[kHold][2 * VEC];

  float amax = 0.f;
#pragma unroll
  for (int u = 0; u < kHold; ++u) {
    const int k = tid + u * 256;
    if (k < pieces) {
      const int r = k / per, piece = k - r * per;
      int d0, d1;
      load_piece<SRC, VEC>(src + r * stride * E, angle_row(p, t0 + r, pos + r), half, p.neox, piece, key, held[u], d0, d1);
#pragma unroll
      for (int e = 0; e < 2 * VEC; ++e) amax = fmaxf(amax, fabsf(held[u][e]));
    }
  }
  for (int k = tid + kHold * 256; k < pieces; k += 256) {
    const int r = k / per, piece = k - r * per;
    float f[2 * VEC];
    int d0, d1;
    load_piece<SRC, VEC>(src + r * stride * E, angle_row(p, t0 + r, pos + r), half, p.neox, piece, key, f, d0, d1);
#pragma unroll
    for (int e = 0; e < 2 * VEC; ++e) amax = fmaxf(amax, fabsf(f[e]));
  }
#pragma unroll
  for (int o = 32; o > 0; o >>= 1) amax = fmaxf(amax, __shfl_xor(amax, o));
  if ((tid & 63) == 0) most[tid >> 6] = amax;
  __syncthreads();
  amax = fmaxf(fmaxf(most[0], most[1]), fmaxf(most[2], most[3]));
  constexpr float unit = KVT == RPA_FP8_E4M3 ? 1.f / 448.f : 1.f / 127.f;
  float new_scale = fmaxf(old_scale, amax * unit);
  if (new_scale == 0.f) new_scale = 1.f;

  if (new_scale > old_scale && first > 0) {
    const int words = p.D >> 2;  // head rows are multiples of four codes
    for (int k = tid; k < first * words; k += 256) {
      const int r = k / words, d = (k - r * words) * 4;
      uint32_t* at = (uint32_t*)(dst + r * dst_row + d);
      const uint32_t was = *at;
      uint32_t w = 0;
#pragma unroll
      for (int e = 0; e < 4; ++e) w |= quant1<KVT>((decode1<KVT>((was >> (8 * e)) & 0xff) * old_scale) / new_scale) << (8 * e);
      *at = w;
    }
  }
  const bool split_rows = key && p.neox;
#pragma unroll
  for (int u = 0; u < kHold; ++u) {
    const int k = tid + u * 256;
    if (k < pieces) {
      const int r = k / per, piece = k - r * per;
      const bool split = split_rows && piece * VEC < half;
      const int d0 = split ? piece * VEC : piece * 2 * VEC, d1 = split ? d0 + half : d0 + VEC;
      unsigned char* row = dst + (first + r) * dst_row;
      store_codes<KVT, VEC>(row + d0, held[u], new_scale);
      store_codes<KVT, VEC>(row + d1, held[u] + VEC, new_scale);
    }
  }
  for (int k = tid + kHold * 256; k < pieces; k += 256) {
    const int r = k / per, piece = k - r * per;
    float f[2 * VEC];
    int d0, d1;
    load_piece<SRC, VEC>(src + r * stride * E, angle_row(p, t0 + r, pos + r), half, p.neox, piece, key, f, d0, d1);
    unsigned char* row = dst + (first + r) * dst_row;
    store_codes<KVT, VEC>(row + d0, f, new_scale);
    store_codes<KVT, VEC>(row + d1, f + VEC, new_scale);
  }
  const int pad = (p.Dp - p.D) >> 2;
  for (int k = tid; k < n * pad; k += 256) {
    const int r = k / pad, d = (k - r * pad) * 4;
    *(uint32_t*)(dst + (first + r) * dst_row + p.D + d) = 0u;
  }
  if (tid == 0) p.scales[si] = new_scale;  // every wave has read the old one: it lies ahead of the barrier
}

template <int SRC, int KVT, int VEC>
__global__ __launch_bounds__(256) void rope_append_quant_kernel(RopeParams p, int run_blocks) {
  __shared__ float most[4];
  const int n_live = rope_live(p);
  if ((int)blockIdx.x < run_blocks) {
    if (n_live <= 0) return;
    const int run = blockIdx.x / (2 * p.Hkv), c = blockIdx.x - run * 2 * p.Hkv;
    if (run < p.qsl[0] / p.page_size) return;  // ahead of the first sequence's numbers
    append_run<SRC, KVT, VEC>(p, n_live, run, c, most);
    return;
  }
  const int t = blockIdx.x - run_blocks;
  const bool live = n_live > 0 && t >= p.qsl[0] && t < p.qsl[n_live];
  const float* angles = live ? angle_row(p, t, p.positions ? 0 : place_of(p, n_live, t).pos) : nullptr;
  turn_queries<SRC, VEC>(p, t, angles, live, threadIdx.x, 256);
}

// ---- latent pages -----------------------------------------------------------------------------------------
template <int SRC, int KV, int VEC>
__global__ __launch_bounds__(256) void rope_latent_kernel(RopeParams p) {
  constexpr int E = ElemBytes<SRC>::v, EK = ElemBytes<KV>::v;
  const int t = blockIdx.x, tid = threadIdx.x;
  const int n_live = rope_live(p);
  const bool live = n_live > 0 && t >= p.qsl[0] && t < p.qsl[n_live];
  if (!live) {
    turn_queries<SRC, VEC>(p, t, nullptr, false, tid, 256);
    return;
  }
  const Place w = place_of(p, n_live, t);
  const float* angles = angle_row(p, t, w.pos);
  turn_queries<SRC, VEC>(p, t, angles, true, tid, 256);
  if (w.row < 0) return;
  char* row = p.k_pages + w.row;
  // the latent part and the padding as 4-byte words (lkv and rope are multiples of 8, row_elems of 4), the rope key turned
  const int words = p.row_elems * EK / 4, latent_words = p.lkv * EK / 4;
  const int rope0 = p.rope_off * EK / 4, rope1 = rope0 + p.rope * EK / 4;
  const uint32_t* src = (const uint32_t*)((const char*)p.latent + (int64_t)t * p.lkv * EK);
  for (int k = tid; k < words; k += 256) {
    if (k >= rope0 && k < rope1) continue;
    ((uint32_t*)row)[k] = k < latent_words ? src[k] : 0u;
  }
  const int per = p.rope / (2 * VEC), half = p.rope >> 1;
  const char* pe = (const char*)p.k + (int64_t)t * p.k_stride * E;
  for (int piece = tid; piece < per; piece += 256) {
    float f[2 * VEC];
    int d0, d1;
    load_piece<SRC, VEC>(pe, angles, half, p.neox, piece, true, f, d0, d1);
    store_group<KV, VEC>(row + (p.rope_off + d0) * EK, f);
    store_group<KV, VEC>(row + (p.rope_off + d1) * EK, f + VEC);
  }
}

bool fits(const void* ptr, int64_t bytes) { return ptr == nullptr || ((uintptr_t)ptr % bytes) == 0; }

// Elements per aligned group: the most that divide the turning part, the head rows and every stride and address, up to 16
// bytes of the source type.  (Groups of one element read and write two bytes at a time; they serve the odd shapes.)
template <bool LATENT>
int group_of(const RopeParams& p, int most) {
  const int e = elem_bytes(p.src_dtype), ek = elem_bytes(p.kv_dtype);
  for (int v = most; v > 1; v >>= 1) {
    if (v == 2) continue;
    bool ok = p.rope % (2 * v) == 0 && p.D % (2 * v) == 0 && fits(p.q, v * e) && fits(p.k, v * e) && fits(p.q_out, v * e) &&
              fits(p.cos_sin, 16) && p.q_stride % v == 0 && p.k_stride % v == 0 && fits(p.k_pages, v * ek) && p.token_stride % (v * ek) == 0 &&
              p.page_stride % (v * ek) == 0;
    if (!LATENT) ok = ok && p.Dp % (2 * v) == 0 && p.v_stride % v == 0 && fits(p.v, v * e) && fits(p.v_pages, v * ek) && p.head_stride % (v * ek) == 0;
    if (ok) return v;
  }
  return 1;
}

}  // namespace

namespace {

// Groups of 8 where source and pages are both narrower than float32 (32 bytes of float32 would be two accesses), of 4, or of 1.
template <int SRC, int KV, bool LATENT>
int launch_pages(hipStream_t stream, const RopeParams& p) {
  constexpr int MOST = SRC == RPA_F32 || KV == RPA_F32 ? 4 : 8;
  const int v = group_of<LATENT>(p, MOST);
  const dim3 grid(p.T), block(256);
#define RPA_ROPE(VEC)                                                                                        \
  do {                                                                                                       \
    if constexpr (LATENT) hipLaunchKernelGGL((rope_latent_kernel<SRC, KV, VEC>), grid, block, 0, stream, p); \
    else hipLaunchKernelGGL((rope_append_kernel<SRC, KV, VEC>), grid, block, 0, stream, p);                  \
  } while (0)
  if (v == 8) {
    if constexpr (MOST == 8) RPA_ROPE(8);
  } else if (v == 4) {
    RPA_ROPE(4);
  } else {
    RPA_ROPE(1);
  }
#undef RPA_ROPE
  return (int)hipGetLastError();
}

template <int SRC, bool LATENT>
int launch_src(hipStream_t stream, const RopeParams& p) {
  switch (p.kv_dtype) {
    case RPA_F32: return launch_pages<SRC, RPA_F32, LATENT>(stream, p);
    case RPA_BF16: return launch_pages<SRC, RPA_BF16, LATENT>(stream, p);
    case RPA_F16: return launch_pages<SRC, RPA_F16, LATENT>(stream, p);
    case RPA_FP8_E4M3: return launch_pages<SRC, RPA_FP8_E4M3, LATENT>(stream, p);
    default: return (int)hipErrorInvalidValue;
  }
}

template <bool LATENT>
int launch_plain(hipStream_t stream, const RopeParams& p) {
  switch (p.src_dtype) {
    case RPA_F32: return launch_src<RPA_F32, LATENT>(stream, p);
    case RPA_BF16: return launch_src<RPA_BF16, LATENT>(stream, p);
    case RPA_F16: return launch_src<RPA_F16, LATENT>(stream, p);
    default: return (int)hipErrorInvalidValue;
  }
}

template <int SRC, int KVT>
int launch_quant(hipStream_t stream, const RopeParams& p) {
  const int64_t run_blocks = ((int64_t)p.T / p.page_size + 2 * (int64_t)p.S) * 2 * p.Hkv;  // (run, combined head) pairs
  if (run_blocks + p.T > 0x7fffffff) return (int)hipErrorInvalidValue;
  const dim3 grid((unsigned)(run_blocks + p.T)), block(256);
  if (group_of<false>(p, 4) == 4) hipLaunchKernelGGL((rope_append_quant_kernel<SRC, KVT, 4>), grid, block, 0, stream, p, (int)run_blocks);
  else hipLaunchKernelGGL((rope_append_quant_kernel<SRC, KVT, 1>), grid, block, 0, stream, p, (int)run_blocks);
  return (int)hipGetLastError();
}

}  // namespace

int launch_rope_append(hipStream_t stream, const RopeParams& p) { return launch_plain<false>(stream, p); }

int launch_rope_latent(hipStream_t stream, const RopeParams& p) { return launch_plain<true>(stream, p); }

int launch_rope_append_quant(hipStream_t stream, const RopeParams& p) {
  const bool fp8 = p.kv_dtype == RPA_FP8_E4M3;
  switch (p.src_dtype) {
    case RPA_F32: return fp8 ? launch_quant<RPA_F32, RPA_FP8_E4M3>(stream, p) : launch_quant<RPA_F32, RPA_INT8>(stream, p);
    case RPA_BF16: return fp8 ? launch_quant<RPA_BF16, RPA_FP8_E4M3>(stream, p) : launch_quant<RPA_BF16, RPA_INT8>(stream, p);
    case RPA_F16: return fp8 ? launch_quant<RPA_F16, RPA_FP8_E4M3>(stream, p) : launch_quant<RPA_F16, RPA_INT8>(stream, p);
    default: return (int)hipErrorInvalidValue;
  }
}

}  // namespace rpa
