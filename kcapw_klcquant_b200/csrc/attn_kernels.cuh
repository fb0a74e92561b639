// Launch parameters and internal entry points of the attention kernels.
#pragma once

#include <cuda.h>

#include "klc_common.cuh"

namespace klc {
namespace attn {

// tensor-core kernel (attn_tc.cu): prompts, and the shared prefix of decode rows
struct TcParams {
  const int32_t* cu_q;  // [batch + 1] first query row of each sequence (or group of rows)
  const int32_t* cu_k;  // prompts: [batch + 1] first key row
  int batch;
  int64_t total_q, total_k;
  int heads, kv_heads, group, tpt;  // query and key heads; query heads per key head; tokens per row tile
  float scale_log2;       // scale * log2(e)
  int window;
  const float* sinks;
  void* out;
  int64_t out_ts, out_hs;
  float* lse;
  DeviceStatus* status;
  const void* v;       // values, for elements that are not finite: token and head stride (prompts), page stride (v_ts, prefix)
  int64_t v_ts, v_hs;
  // prefix of decode rows
  const int32_t* prefix_lens;  // [batch]
  const int32_t* lens;         // [total_q]
  const int32_t* block_table;
  int64_t table_stride, pages;
  int page_size;
  int splits;       // shares the prefix's keys are cut into
  float* part_o;    // [splits][total_q][heads][D]
  float2* part_ml;  // [splits][total_q][heads]
};

// decode kernel and join (attn_decode.cu)
struct DecodeParams {
  const void* q;
  int64_t q_ts, q_hs;
  const int32_t* block_table;
  int64_t table_stride, pages;
  int table_width, page_size;
  const int32_t* lens;
  int batch;
  const int32_t* group_starts;
  const int32_t* prefix_lens;
  int groups;
  int heads, kv_heads, group, row_tiles;
  float scale_log2;
  int window;
  const float* sinks;
  void* out;
  int64_t out_ts, out_hs;
  float* lse;
  DeviceStatus* status;
  // workspace
  int* cum;             // [batch + 1] the split's units before each sequence
  float2* part_ml;      // [2 * ctas][16] shares of cut items
  float* part_o;        // [2 * ctas][16][D]
  float2* prefix_ml;    // [splits + 1][batch][heads]: the prefix's shares, and uncut items behind a prefix
  float* prefix_o;      // [splits + 1][batch][heads][D]
  int splits;
  bool after_prefix;    // launched to overlap the prefix kernel
};

int launch_prefix(const klc_attn_dims& dims, const DecodeParams& d, const void* q, const void* k_pages, const void* v_pages,
                  int64_t page_stride, cudaStream_t stream);

int check_rows(const char* who, const char* what, const void* base, int64_t tokens, int64_t ts, int64_t hs, int heads, int d);

// K or V pool [pages][kv_heads][page_size][D] (page stride in elements), box of box_rows x 64
int pool_map(CUtensorMap* m, int dtype, int head_dim, const void* base, int64_t pages, int kv_heads, int page_size,
             int64_t page_stride, int box_rows);

}  // namespace attn
}  // namespace klc
