// Rotary embedding of queries and keys and the write of keys and values into
// the cache's pages, in one pass.
//
//   (x1, x2) -> (x1 c - x2 s, x2 c + x1 s),  c = cos[pos], s = sin[pos]
//
// x1, x2 the halves of a head's row; fp32, rounded once.  The angles come as
// fp32 tables [max_pos, D / 2] (a position of 10^5 times a frequency needs
// more than fp32 before the cosine is taken, so the caller makes them in
// fp64, once).  Bytes bound it: q, k, v are read once, q and the pages written
// once.  A thread rotates eight pairs (two 16-byte loads and stores) or copies eight values; a block finds the
// places of its tokens once.  9 prompts (9,000 tokens) of 64 / 8 heads of 64: 33 us, 5.2 TB/s.
#include <algorithm>

#include "attn_common.cuh"
#include "attn_kernels.cuh"

namespace klc {
namespace attn {
namespace {

constexpr int kThreads = 256;
constexpr int kMaxTokens = 8;  // tokens a block

struct RopeParams {
  const void *q, *k, *v;
  int64_t q_ts, q_hs, k_ts, k_hs, v_ts, v_hs;
  const float *cos, *sin;
  int64_t max_pos;
  const int32_t *pos, *rows;
  int64_t tokens;
  int heads, kv_heads;
  void *q_out, *k_out;
  int64_t qo_ts, qo_hs, ko_ts, ko_hs;
  void *k_pages, *v_pages;
  int64_t pages, page_stride;
  int page_size;
  const int32_t* table;
  int64_t table_rows, table_width, table_stride;
  DeviceStatus* status;
};

template <typename T>
__device__ __forceinline__ void rotate8(const uint4& a, const uint4& b, const float* c, const float* s, uint4* oa, uint4* ob) {
  const uint32_t av[4] = {a.x, a.y, a.z, a.w}, bv[4] = {b.x, b.y, b.z, b.w};
  uint32_t ra[4], rb[4];
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const float2 x = Elem<T>::unpack(av[i]), y = Elem<T>::unpack(bv[i]);
    ra[i] = Elem<T>::pack(x.x * c[2 * i] - y.x * s[2 * i], x.y * c[2 * i + 1] - y.y * s[2 * i + 1]);
    rb[i] = Elem<T>::pack(y.x * c[2 * i] + x.x * s[2 * i], y.y * c[2 * i + 1] + x.y * s[2 * i + 1]);
  }
  *oa = make_uint4(ra[0], ra[1], ra[2], ra[3]);
  *ob = make_uint4(rb[0], rb[1], rb[2], rb[3]);
}

template <typename T, int D>
__global__ void __launch_bounds__(kThreads) rope_append_kernel(const RopeParams p, int block_tokens) {
  constexpr int kPairs = D / 16, kVals = D / 8;  // threads a head's rotation / copy takes
  __shared__ int64_t slot_s[kMaxTokens];         // of the token's first key head in the pools; -1: no place, -2: write nothing
  __shared__ int pos_s[kMaxTokens];
  pdl_trigger();
  pdl_wait();
  const int64_t t0 = int64_t(blockIdx.x) * block_tokens;
  const int n = int(min(int64_t(block_tokens), p.tokens - t0));
  if (threadIdx.x < n) {
    const int64_t t = t0 + threadIdx.x;
    const int row = p.rows[t], pos = p.pos[t];
    int64_t slot = -2;  // row -1 is padding
    if (row != -1) {
      if (row < 0 || row >= p.table_rows || pos < 0 || pos >= p.max_pos || pos / p.page_size >= p.table_width) {
        record_fault(p.status, KLC_ERR_DEVICE_FAULT, 540, int(t));
      } else {
        const int page = p.table[int64_t(row) * p.table_stride + pos / p.page_size];
        slot = -1;
        if (page < 0 || page >= p.pages) record_fault(p.status, KLC_ERR_DEVICE_FAULT, 541, page);
        else slot = int64_t(page) * p.page_stride + int64_t(pos % p.page_size) * D;
      }
    }
    slot_s[threadIdx.x] = slot;
    pos_s[threadIdx.x] = pos;
  }
  __syncthreads();
  const int rot = (p.heads + p.kv_heads) * kPairs, per_token = rot + p.kv_heads * kVals;
  const int64_t head_pitch = int64_t(p.page_size) * D;
#pragma unroll 2
  for (int i = threadIdx.x; i < n * per_token; i += kThreads) {
    const int j = i / per_token, u = i - j * per_token;
    const int64_t slot = slot_s[j], t = t0 + j;
    const bool is_q = u < p.heads * kPairs;
    if (slot == -2 || (slot == -1 && !is_q)) continue;
    if (u < rot) {
      const int head = u / kPairs, part = u - head * kPairs;  // eight pairs from column 8 * part
      const int kh = head - p.heads;
      const T* src = (is_q ? reinterpret_cast<const T*>(p.q) + t * p.q_ts + int64_t(head) * p.q_hs
                           : reinterpret_cast<const T*>(p.k) + t * p.k_ts + int64_t(kh) * p.k_hs) +
                     part * 8;
      const uint4 a = *reinterpret_cast<const uint4*>(src), b = *reinterpret_cast<const uint4*>(src + D / 2);
      float c[8], s[8];
      const int64_t ang = int64_t(pos_s[j]) * (D / 2) + part * 8;
#pragma unroll
      for (int e = 0; e < 8; e += 4) {
        *reinterpret_cast<float4*>(c + e) = *reinterpret_cast<const float4*>(p.cos + ang + e);
        *reinterpret_cast<float4*>(s + e) = *reinterpret_cast<const float4*>(p.sin + ang + e);
      }
      uint4 oa, ob;
      rotate8<T>(a, b, c, s, &oa, &ob);
      if (is_q) {
        T* dst = reinterpret_cast<T*>(p.q_out) + t * p.qo_ts + int64_t(head) * p.qo_hs + part * 8;
        *reinterpret_cast<uint4*>(dst) = oa;
        *reinterpret_cast<uint4*>(dst + D / 2) = ob;
      } else {
        T* dst = reinterpret_cast<T*>(p.k_pages) + slot + kh * head_pitch + part * 8;
        *reinterpret_cast<uint4*>(dst) = oa;
        *reinterpret_cast<uint4*>(dst + D / 2) = ob;
        if (p.k_out != nullptr) {
          T* ko = reinterpret_cast<T*>(p.k_out) + t * p.ko_ts + int64_t(kh) * p.ko_hs + part * 8;
          *reinterpret_cast<uint4*>(ko) = oa;
          *reinterpret_cast<uint4*>(ko + D / 2) = ob;
        }
      }
    } else {
      const int w = u - rot, kh = w / kVals, part = w - kh * kVals;
      const T* src = reinterpret_cast<const T*>(p.v) + t * p.v_ts + int64_t(kh) * p.v_hs + part * 8;
      *reinterpret_cast<uint4*>(reinterpret_cast<T*>(p.v_pages) + slot + kh * head_pitch + part * 8) =
          *reinterpret_cast<const uint4*>(src);
    }
  }
}

template <typename T, int D>
int launch(const RopeParams& p, cudaStream_t s) {
  // enough blocks to fill the SMs eight times over, up to kMaxTokens tokens each
  const int64_t bt = std::max<int64_t>(1, std::min<int64_t>(kMaxTokens, p.tokens / (int64_t(sm_count()) * 8)));
  const int64_t blocks = (p.tokens + bt - 1) / bt;
  KLC_CHECK_ARG(blocks < (int64_t(1) << 31), "klc_rope_append: too many tokens for one call");
  KLC_CUDA(launch_chain(rope_append_kernel<T, D>, dim3(unsigned(blocks)), dim3(kThreads), 0, s, 0, p, int(bt)));
  KLC_LAUNCH_CHECK("rope_append");
  return KLC_OK;
}

}  // namespace
}  // namespace attn
}  // namespace klc

extern "C" int klc_rope_append(const klc_attn_dims* dims, const void* q, int64_t q_token_stride, int64_t q_head_stride,
                               const void* k, int64_t k_token_stride, int64_t k_head_stride, const void* v,
                               int64_t v_token_stride, int64_t v_head_stride, const float* cos, const float* sin,
                               int64_t max_pos, const int32_t* positions, const int32_t* rows, int64_t tokens, void* q_out,
                               int64_t qo_token_stride, int64_t qo_head_stride, void* k_out, int64_t ko_token_stride,
                               int64_t ko_head_stride, void* k_pages, void* v_pages, int64_t pages, int page_size,
                               int64_t page_stride, const int32_t* block_table, int64_t table_rows, int64_t table_width,
                               int64_t table_stride, void* status, void* stream) {
  using namespace klc;
  using namespace klc::attn;
  const char* who = "klc_rope_append";
  KLC_CHECK_ARG(dims != nullptr, "klc_rope_append: null dims");
  int st = check_heads(who, dims->dtype, dims->heads, dims->kv_heads, dims->head_dim);
  if (st != KLC_OK) return st;
  KLC_CHECK_ARG(tokens >= 0 && max_pos >= 0, "klc_rope_append: negative size");
  KLC_CHECK_ARG(page_size_ok(page_size), "klc_rope_append: page_size must be 16, 32, 64 or 128");
  KLC_CHECK_ARG(pages >= 1 && pages < (1 << 30), "klc_rope_append: pages must be between 1 and 2^30");
  KLC_CHECK_ARG(table_rows >= 0 && table_width >= 0 && table_width < (int64_t(1) << 31) && table_stride >= table_width, "klc_rope_append: bad block table size or stride");
  if (tokens == 0) return KLC_OK;
  const int d = dims->head_dim;
  KLC_CHECK_ARG(tokens < (int64_t(1) << 31), "klc_rope_append: too many tokens for one call");
  KLC_CHECK_ARG(positions != nullptr && rows != nullptr && cos != nullptr && sin != nullptr, "klc_rope_append: null pointer");
  KLC_CHECK_ARG(block_table != nullptr && k_pages != nullptr && v_pages != nullptr, "klc_rope_append: null cache");
  KLC_CHECK_ARG(aligned16(cos) && aligned16(sin) && aligned16(k_pages) && aligned16(v_pages),
                "klc_rope_append: the tables and pools must be 16-byte aligned");
  KLC_CHECK_ARG(page_stride % 8 == 0 && page_stride >= int64_t(dims->kv_heads) * page_size * d && page_stride < (int64_t(1) << 38),
                "klc_rope_append: page_stride must be a multiple of 8 and hold a page");
  if ((st = check_rows(who, "q", q, tokens, q_token_stride, q_head_stride, dims->heads, d)) != KLC_OK) return st;
  if ((st = check_rows(who, "k", k, tokens, k_token_stride, k_head_stride, dims->kv_heads, d)) != KLC_OK) return st;
  if ((st = check_rows(who, "v", v, tokens, v_token_stride, v_head_stride, dims->kv_heads, d)) != KLC_OK) return st;
  if ((st = check_rows(who, "q_out", q_out, tokens, qo_token_stride, qo_head_stride, dims->heads, d)) != KLC_OK) return st;
  if (k_out != nullptr &&
      (st = check_rows(who, "k_out", k_out, tokens, ko_token_stride, ko_head_stride, dims->kv_heads, d)) != KLC_OK)
    return st;
  RopeParams p{q, k, v, q_token_stride, q_head_stride, k_token_stride, k_head_stride, v_token_stride, v_head_stride, cos, sin,
               max_pos, positions, rows, tokens, dims->heads, dims->kv_heads, q_out, k_out, qo_token_stride, qo_head_stride,
               ko_token_stride, ko_head_stride, k_pages, v_pages, pages, page_stride, page_size, block_table, table_rows,
               table_width, table_stride, reinterpret_cast<DeviceStatus*>(status)};
  cudaStream_t s = as_stream(stream);
  if (dims->dtype == KLC_BF16) return d == 64 ? launch<__nv_bfloat16, 64>(p, s) : launch<__nv_bfloat16, 128>(p, s);
  return d == 64 ? launch<__half, 64>(p, s) : launch<__half, 128>(p, s);
}
