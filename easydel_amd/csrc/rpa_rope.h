// Append with rotation: parameters and launchers.
#pragma once
#include "rpa_common.h"

namespace rpa {

struct RopeParams {
  const void* q;  // rows of Hq heads, q_stride elements apart; k, v likewise (Hkv heads)
  const void* k;
  const void* v;
  void* q_out;           // [T][Hq][D]
  char* k_pages;         // K of KV head h of a token: k_pages + page*page_stride + token*token_stride + h*head_stride
  char* v_pages;         // V likewise
  float* scales;         // [P][C] or null (then the pages hold plain values)
  const float* cos_sin;  // [table_rows][rope]: cosines, then sines
  const int32_t* positions;  // [T] table rows, or null: cache positions
  const int32_t* context_lens;
  const int32_t* block_tables;
  const int32_t* qsl;
  const int32_t* num_seqs;  // or null: all S rows are live
  int T, S, M, P, page_size, Hq, Hkv, D, Dp, C, rope, table_rows, neox;
  int q_in_place;  // q_out is q: padded rows stay as they are
  int64_t q_stride, k_stride, v_stride;                // elements
  int64_t head_stride, token_stride, page_stride;      // bytes
  int src_dtype, kv_dtype;
  // latent pages: the rope key of a token goes to rope_off of its row, keys_values [T][lkv] to its start
  const void* latent;
  int lkv, rope_off, row_elems;
};

int launch_rope_append(hipStream_t stream, const RopeParams& p);
int launch_rope_append_quant(hipStream_t stream, const RopeParams& p);
int launch_rope_latent(hipStream_t stream, const RopeParams& p);

}  // namespace rpa
