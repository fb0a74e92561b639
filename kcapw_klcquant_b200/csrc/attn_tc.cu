// Attention on the tensor cores (tcgen05, TMEM accumulators): whole prompts,
// and the prefix that a group of single-token rows shares.
//
//   s_ij = scale q_i . k_j,  p_ij = exp(s_ij - m_i),  o_i = sum_j p_ij v_j / l_i,  l_i = sum_j p_ij + exp(sink - m_i)
//
// over the keys j a row sees: j <= pos_i, and j > pos_i - window with a window.
//
// One CTA takes one key head of one sequence and two row tiles.  A row tile
// is `tpt` tokens x G query heads (G = heads per key head, tpt = 128 / G):
// all heads that read the same keys share the tile's loads, and short
// sequences fill tiles that 128 tokens of one head would not.  Keys come in
// tiles of 128.  Warps:
//   0-3, 4-7  softmax of row tile 0 / 1, one row per thread (TMEM lane = row)
//   8         MMA issuer (one thread); zeroes value rows past the keys' end
//   9         TMA producer (queries once, then a ring of key and value tiles)
// Per key tile and row tile: S = Q K^T into TMEM (128 fp32 columns), the
// softmax thread reads its row, writes P as 16-bit pairs over S, and O += P V
// reads P from TMEM.  The tensor pipe works on one row tile while the other is
// in its softmax.  Row statistics are fp32.  O is rescaled only when a row's
// maximum has grown by more than 2^8 since the last rescale: until then P is at most
// 2^8, far inside both types' range, and its relative rounding (2^-9 / 2^-12,
// the price of a 16-bit P operand) does not depend on the reference maximum.
#include <algorithm>

#include "attn_common.cuh"
#include "attn_kernels.cuh"
#include "tc_common.cuh"

namespace klc {
namespace attn {

using namespace tc;

namespace {

constexpr int kRows = 128;     // rows of a row tile (TMEM lanes)
constexpr int kKeys = 128;     // keys of a key tile
constexpr int kThreads = 320;  // 8 softmax warps, MMA warp, TMA warp
constexpr int kWarpMma = 8, kWarpTma = 9;
constexpr uint32_t kTmemCols = 512;
constexpr float kRescaleLog2 = 8.f;

__device__ __forceinline__ void tmem_ld32(uint32_t taddr, float* v) {
  uint32_t* r = reinterpret_cast<uint32_t*>(v);
  asm volatile(
      "tcgen05.ld.sync.aligned.32x32b.x32.b32 {%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15, "
      "%16, %17, %18, %19, %20, %21, %22, %23, %24, %25, %26, %27, %28, %29, %30, %31}, [%32];"
      : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]), "=r"(r[8]), "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15]), "=r"(r[16]), "=r"(r[17]), "=r"(r[18]), "=r"(r[19]), "=r"(r[20]), "=r"(r[21]), "=r"(r[22]), "=r"(r[23]), "=r"(r[24]), "=r"(r[25]), "=r"(r[26]), "=r"(r[27]), "=r"(r[28]), "=r"(r[29]), "=r"(r[30]), "=r"(r[31])
      : "r"(taddr)
      : "memory");
}

// waits for the loads into v; the operands keep their uses behind the wait
__device__ __forceinline__ void tmem_wait_ld32(float* v) {
  uint32_t* r = reinterpret_cast<uint32_t*>(v);
  asm volatile("tcgen05.wait::ld.sync.aligned;"
               : "+r"(r[0]), "+r"(r[1]), "+r"(r[2]), "+r"(r[3]), "+r"(r[4]), "+r"(r[5]), "+r"(r[6]), "+r"(r[7]), "+r"(r[8]), "+r"(r[9]), "+r"(r[10]), "+r"(r[11]), "+r"(r[12]), "+r"(r[13]), "+r"(r[14]), "+r"(r[15]), "+r"(r[16]), "+r"(r[17]), "+r"(r[18]), "+r"(r[19]), "+r"(r[20]), "+r"(r[21]), "+r"(r[22]), "+r"(r[23]), "+r"(r[24]), "+r"(r[25]), "+r"(r[26]), "+r"(r[27]), "+r"(r[28]), "+r"(r[29]), "+r"(r[30]), "+r"(r[31])
               :
               : "memory");
}

__device__ __forceinline__ void tmem_st16(uint32_t taddr, const uint32_t* r) {
  asm volatile(
      "tcgen05.st.sync.aligned.32x32b.x16.b32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15, %16};" ::"r"(
          taddr),
      "r"(r[0]), "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7]), "r"(r[8]), "r"(r[9]), "r"(r[10]),
      "r"(r[11]), "r"(r[12]), "r"(r[13]), "r"(r[14]), "r"(r[15])
      : "memory");
}

__device__ __forceinline__ void tmem_st32(uint32_t taddr, const uint32_t* r) {
  asm volatile(
      "tcgen05.st.sync.aligned.32x32b.x32.b32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15, %16, "
      "%17, %18, %19, %20, %21, %22, %23, %24, %25, %26, %27, %28, %29, %30, %31, %32};" ::"r"(taddr), "r"(r[0]), "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7]), "r"(r[8]), "r"(r[9]), "r"(r[10]), "r"(r[11]), "r"(r[12]), "r"(r[13]), "r"(r[14]), "r"(r[15]), "r"(r[16]), "r"(r[17]), "r"(r[18]), "r"(r[19]), "r"(r[20]), "r"(r[21]), "r"(r[22]), "r"(r[23]), "r"(r[24]), "r"(r[25]), "r"(r[26]), "r"(r[27]), "r"(r[28]), "r"(r[29]), "r"(r[30]), "r"(r[31])
      : "memory");
}

// D[tmem] (+)= A[tmem or smem] * B[smem]
__device__ __forceinline__ void mma_ss(uint32_t d, uint64_t a, uint64_t b, uint32_t idesc, uint32_t acc) {
  asm volatile(
      "{\n\t.reg .pred p;\n\tsetp.ne.u32 p, %4, 0;\n\t"
      "tcgen05.mma.cta_group::1.kind::f16 [%0], %1, %2, %3, p;\n\t}" ::"r"(d),
      "l"(a), "l"(b), "r"(idesc), "r"(acc)
      : "memory");
}
__device__ __forceinline__ void mma_ts(uint32_t d, uint32_t a, uint64_t b, uint32_t idesc, uint32_t acc) {
  asm volatile(
      "{\n\t.reg .pred p;\n\tsetp.ne.u32 p, %4, 0;\n\t"
      "tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], %2, %3, p;\n\t}" ::"r"(d),
      "r"(a), "l"(b), "r"(idesc), "r"(acc)
      : "memory");
}

// fp32 accumulator, both operands of one 16-bit format, A K-major; B K-major or (bit 16) MN-major
template <typename T>
__device__ __forceinline__ constexpr uint32_t f16_idesc(int m, int n, bool b_mn_major) {
  return (1u << 4) | (Elem<T>::kMmaFormat << 7) | (Elem<T>::kMmaFormat << 10) | (b_mn_major ? 1u << 16 : 0u) |
         (uint32_t(n >> 3) << 17) | (uint32_t(m >> 4) << 24);
}

// MN-major operand, 128-byte swizzle: rows of 64 contiguous MN elements, one row per K; eight-row
// groups 1024 bytes apart along K (SBO), the next 64 MN elements `mn_stride` bytes on (LBO).
__device__ __forceinline__ uint64_t sw128_mn_desc(uint32_t saddr, uint32_t mn_stride) {
  return uint64_t((saddr & 0x3FFFFu) >> 4) | (uint64_t(mn_stride >> 4) << 16) | (uint64_t(1024 >> 4) << 32) |
         (uint64_t(1) << 46) | (uint64_t(2) << 61);
}

template <int D>
struct Cfg {
  static constexpr int kChunks = D / 64;                    // 128-byte columns of a head's row
  static constexpr int kTile = kKeys * D * 2;               // bytes of a query, key or value tile
  static constexpr int kStages = D == 64 ? 10 : 5;          // ring of key and value tiles: 160 KB
  static constexpr int OFF_Q = 0;                           // two row tiles
  static constexpr int OFF_KV = 2 * kTile;
  static constexpr int OFF_BAR = OFF_KV + kStages * kTile;
  static constexpr int kBars = 1 + 2 * kStages + 2 + 2 + 2 + 1;
  static constexpr int OFF_MISC = OFF_BAR + kBars * 8;
  static constexpr int kSmem = OFF_MISC + 64 + 1024;        // + alignment of the swizzled tiles
};

struct Item {
  int q0, qn;  // the sequence's first query row and its number of query rows (tokens)
  int k0, kn;  // first key row and number of keys
  int tok0;    // first token of the CTA's two row tiles
  int lo, hi;  // key tiles [lo, hi)
};

// ---------------------------------------------------------------------------
// PREFIX = false: packed prompts.  PREFIX = true: single-token rows over the pages of their group's prefix, keys split over
// gridDim.z; shares (m, l, o) go to the workspace and are joined by the decode combine.
// ---------------------------------------------------------------------------
template <typename T, int D, bool PREFIX>
__global__ void __launch_bounds__(kThreads, 1)
attn_tc_kernel(const __grid_constant__ CUtensorMap map_q, const __grid_constant__ CUtensorMap map_k,
               const __grid_constant__ CUtensorMap map_v, const TcParams p) {
  using C = Cfg<D>;
  extern __shared__ unsigned char smem_raw[];
  unsigned char* smem = reinterpret_cast<unsigned char*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  const int kvh = blockIdx.y;
  const int G = p.group, tpt = p.tpt;

  const uint32_t bar0 = smem_u32(smem + C::OFF_BAR);
  const uint32_t q_full = bar0;
  auto kv_full = [&](int s) { return bar0 + 8u * (1 + s); };
  auto kv_empty = [&](int s) { return bar0 + 8u * (1 + C::kStages + s); };
  auto s_full = [&](int t) { return bar0 + 8u * (1 + 2 * C::kStages + t); };
  auto p_full = [&](int t) { return bar0 + 8u * (3 + 2 * C::kStages + t); };
  auto o_full = [&](int t) { return bar0 + 8u * (5 + 2 * C::kStages + t); };
  const uint32_t mma_done = bar0 + 8u * (7 + 2 * C::kStages);
  uint32_t* tmem_holder = reinterpret_cast<uint32_t*>(smem + C::OFF_MISC);
  volatile int* abort_flag = reinterpret_cast<volatile int*>(smem + C::OFF_MISC + 4);
  Item* item_s = reinterpret_cast<Item*>(smem + C::OFF_MISC + 8);
  const Ctl ctl{abort_flag, p.status};

  if (PREFIX) pdl_trigger();  // the decode kernel may run beside this one

  // ---- which sequence (group) and rows: warp 0 walks the sequences' numbers of row-tile pairs
  if (warp == 0) {
    const int n_seq = p.batch;
    int base = 0;
    Item it{0, 0, 0, 0, -1, 0, 0};
    for (int s0 = 0; s0 < n_seq; s0 += 32) {
      const int s = s0 + lane;
      int qb = 0, qn = 0, kb = 0, kn = 0;
      if (s < n_seq) {
        qb = p.cu_q[s];
        qn = p.cu_q[s + 1] - qb;
        if (PREFIX) {
          kn = p.prefix_lens[s];
        } else {
          kb = p.cu_k[s];
          kn = p.cu_k[s + 1] - kb;
        }
        // offsets that do not describe rows of the tensors: report, and leave the sequence out
        bool bad = qb < 0 || qn < 0 || int64_t(qb) + qn > p.total_q || kb < 0 || kn < 0 || int64_t(kb) + kn > p.total_k;
        if (PREFIX) bad = bad || kn % p.page_size != 0;
        if (bad) {
          record_fault(p.status, KLC_ERR_DEVICE_FAULT, PREFIX ? 520 : 500, s);
          qn = kn = 0;
        }
        if (PREFIX && kn == 0) qn = 0;
      }
      const int pairs = (qn + 2 * tpt - 1) / (2 * tpt);
      int incl = pairs;
#pragma unroll
      for (int o = 1; o < 32; o <<= 1) {
        const int v = __shfl_up_sync(0xffffffffu, incl, o);
        if (lane >= o) incl += v;
      }
      const int excl = base + incl - pairs;
      const bool mine = int(blockIdx.x) >= excl && int(blockIdx.x) < excl + pairs;
      const unsigned hit = __ballot_sync(0xffffffffu, mine);
      if (hit != 0) {
        // a sequence's last rows see the most keys: its tiles run in descending order
        if (mine) it = Item{qb, qn, kb, kn, (pairs - 1 - (int(blockIdx.x) - excl)) * 2 * tpt, 0x7fffffff, 0};
        const int src = __ffs(hit) - 1;
        it.q0 = __shfl_sync(0xffffffffu, it.q0, src);
        it.qn = __shfl_sync(0xffffffffu, it.qn, src);
        it.k0 = __shfl_sync(0xffffffffu, it.k0, src);
        it.kn = __shfl_sync(0xffffffffu, it.kn, src);
        it.tok0 = __shfl_sync(0xffffffffu, it.tok0, src);
        it.lo = 0x7fffffff;
        it.hi = 0;
        break;
      }
      base += __shfl_sync(0xffffffffu, incl, 31);
    }
    if (lane == 0) *item_s = it;
  }
  if (tid == 32 * kWarpTma) {
    mbar_init(q_full, 1);
    for (int s = 0; s < C::kStages; ++s) {
      mbar_init(kv_full(s), 1);
      mbar_init(kv_empty(s), 1);
    }
    for (int t = 0; t < 2; ++t) {
      mbar_init(s_full(t), 1);
      mbar_init(p_full(t), kRows);
      mbar_init(o_full(t), 1);
    }
    mbar_init(mma_done, 1);
    *abort_flag = 0;
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
  }
  __syncthreads();
  if (item_s->tok0 < 0) return;  // past the last pair
  if (warp == kWarpMma) {
    asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(tmem_holder)),
                 "r"(kTmemCols));
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;");
  }

  // ---- each softmax thread's row: token, head, and the keys [jlo, jhi] it sees
  const int t = warp >> 2;  // row tile of a softmax warp
  const int r = tid & (kRows - 1);
  const int tok_in = r / G, g = r - tok_in * G;
  const int tok = item_s->tok0 + t * tpt + tok_in;
  const bool row_ok = warp < 8 && r < tpt * G && tok < item_s->qn;
  int jlo = 0x7fffffff, jhi = -1;
  if (row_ok) {
    const int pos = PREFIX ? p.lens[item_s->q0 + tok] - 1 : item_s->kn - item_s->qn + tok;
    jhi = PREFIX ? min(pos, item_s->kn - 1) : pos;
    jlo = p.window > 0 ? max(0, pos - p.window + 1) : 0;
    if (jlo > jhi) jlo = 0x7fffffff, jhi = -1;
  }
  if (warp < 8) {
    const int wlo = __reduce_min_sync(0xffffffffu, jlo), whi = __reduce_max_sync(0xffffffffu, jhi);
    if (lane == 0) {
      atomicMin(&item_s->lo, wlo);
      atomicMax(&item_s->hi, whi + 1);
    }
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = *tmem_holder;
  const Item it = *item_s;
  int tile_lo = it.hi > 0 ? it.lo / kKeys : 0, tile_hi = it.hi > 0 ? (it.hi + kKeys - 1) / kKeys : 0;
  if (PREFIX) {  // this CTA's share of the keys
    const int n_all = tile_hi - tile_lo, z = blockIdx.z, nz = gridDim.z;
    const int a = tile_lo + int(int64_t(n_all) * z / nz), b = tile_lo + int(int64_t(n_all) * (z + 1) / nz);
    tile_lo = a;
    tile_hi = b;
  }
  const int n = tile_hi - tile_lo;

  if (warp == kWarpTma) {
    // ---------------------------------------------------------------- loads
    if (lane == 0 && n > 0) {
      mbar_arrive_expect_tx(q_full, 2u * C::kChunks * uint32_t(tpt * G) * 128u);
      for (int tt = 0; tt < 2; ++tt)
        for (int c = 0; c < C::kChunks; ++c)
          tma_load_3d(smem_u32(smem + C::OFF_Q + tt * C::kTile + c * (kRows * 128)), &map_q, c * 64, kvh * G,
                      it.q0 + it.tok0 + tt * tpt, q_full);
      uint32_t issued = 0;
      bool ok = true;
      for (int i = 0; i < n && ok; ++i) {
        const int key = (tile_lo + i) * kKeys;
        for (int kv = 0; kv < 2; ++kv, ++issued) {
          const int s = issued % C::kStages;
          if (!(ok = wait_bar(kv_empty(s), ((issued / C::kStages) & 1) ^ 1, ctl, 501))) break;
          const uint32_t dst = smem_u32(smem + C::OFF_KV + s * C::kTile);
          const CUtensorMap* map = kv ? &map_v : &map_k;
          mbar_arrive_expect_tx(kv_full(s), uint32_t(C::kTile));
          if (!PREFIX) {
            for (int c = 0; c < C::kChunks; ++c)
              tma_load_3d(dst + c * (kKeys * 128), map, c * 64, kvh, it.k0 + key, kv_full(s));
          } else {
            // pages past the prefix, and ids that are no page of the pool, read as zeros (coordinate past the end)
            for (int j = 0; j < kKeys; j += p.page_size) {
              int page = int(p.pages);
              if (key + j < it.kn) {
                page = p.block_table[int64_t(it.q0) * p.table_stride + (key + j) / p.page_size];
                if (page < 0 || page >= p.pages) {
                  record_fault(p.status, KLC_ERR_DEVICE_FAULT, 521, page);
                  page = int(p.pages);
                }
              }
              for (int c = 0; c < C::kChunks; ++c)
                tma_load_4d(dst + c * (kKeys * 128) + j * 128, map, c * 64, 0, kvh, page, kv_full(s));
            }
          }
        }
      }
      if (!ok) {
        drain_wait(q_full, 0);
        drain_ring(kv_full(0), C::kStages, issued);
      }
    }
  } else if (warp == kWarpMma) {
    // ---------------------------------------------------------------- MMA
    constexpr uint32_t idesc_qk = f16_idesc<T>(kRows, kKeys, false);
    constexpr uint32_t idesc_pv = f16_idesc<T>(kRows, D, true);
    bool ok = true;
    auto stage_ptr = [&](int s) { return smem + C::OFF_KV + s * C::kTile; };
    auto wait_all = [&](uint32_t bar, uint32_t parity, int site) {
      const bool w = wait_bar(bar, parity, ctl, site);
      return __all_sync(0xffffffffu, w) != 0;
    };
    auto qk = [&](int tt, int s) {  // S_tt = Q_tt K^T
      const uint64_t a = sw128_desc(smem_u32(smem + C::OFF_Q + tt * C::kTile)), b = sw128_desc(smem_u32(stage_ptr(s)));
#pragma unroll
      for (int kk = 0; kk < D / 16; ++kk) {
        const uint64_t off = uint64_t((kk >> 2) * (kRows * 128) + (kk & 3) * 32) >> 4;
        mma_ss(tmem + uint32_t(tt * kKeys), a + off, b + off, idesc_qk, kk > 0);
      }
      tc_commit(s_full(tt));
    };
    auto pv = [&](int tt, int s, bool first) {  // O_tt += P_tt V
      const uint64_t b = sw128_mn_desc(smem_u32(stage_ptr(s)), kKeys * 128);
#pragma unroll
      for (int kk = 0; kk < kKeys / 16; ++kk)
        mma_ts(tmem + uint32_t(2 * kKeys + tt * D), tmem + uint32_t(tt * kKeys + kk * 8), b + (uint64_t(kk * 16 * 128) >> 4),
               idesc_pv, !(first && kk == 0));
    };
    if (n > 0) {
      ok = wait_all(q_full, 0, 502) && wait_all(kv_full(0), 0, 503);
      tc_fence_after();
      if (ok && lane == 0) {
        qk(0, 0);
        qk(1, 0);
        tc_commit(kv_empty(0));
      }
      for (int i = 0; i < n && ok; ++i) {
        const int iv = 2 * i + 1, sv = iv % C::kStages, ik = 2 * i + 2, sk = ik % C::kStages;
        const bool more = i + 1 < n;
        if (!(ok = wait_all(kv_full(sv), (iv / C::kStages) & 1, 504))) break;
        if (!PREFIX) {
          // value rows past the sequence's last key belong to someone else: 0 * anything finite or not must be 0
          const int valid = it.kn - (tile_lo + i) * kKeys;
          if (valid < kKeys) {
            for (int j = valid * 8 + lane; j < kKeys * 8; j += 32)
#pragma unroll
              for (int c = 0; c < C::kChunks; ++c)
                *reinterpret_cast<uint4*>(stage_ptr(sv) + c * (kKeys * 128) + j * 16) = make_uint4(0, 0, 0, 0);
            fence_proxy_async();
            __syncwarp();
          }
        }
        for (int tt = 0; tt < 2 && ok; ++tt) {
          if (!(ok = wait_all(p_full(tt), i & 1, 505 + tt))) break;
          tc_fence_after();
          if (lane == 0) {
            pv(tt, sv, i == 0);
            if (tt == 1) tc_commit(kv_empty(sv));
            if (!more) tc_commit(o_full(tt));
          }
          if (more) {
            if (tt == 0 && !(ok = wait_all(kv_full(sk), (ik / C::kStages) & 1, 507))) break;
            tc_fence_after();
            if (lane == 0) {
              qk(tt, sk);
              if (tt == 1) tc_commit(kv_empty(sk));
            }
          }
          __syncwarp();
        }
      }
      if (!ok && lane == 0) {  // aborting: no MMA may still be in flight when TMEM is freed
        tc_commit(mma_done);
        drain_wait(mma_done, 0);
      }
      __syncwarp();
    }
  } else {
    // ---------------------------------------------------------------- softmax
    const uint32_t lane_base = uint32_t((warp & 3) * 32) << 16;
    const uint32_t s_col = tmem + lane_base + uint32_t(t * kKeys);
    const uint32_t o_col = tmem + lane_base + uint32_t(2 * kKeys + t * D);
    float m = -INFINITY, l = 0.f;  // m: reference maximum (log2 units) of the stored P and O
    bool ok = true;
    for (int i = 0; i < n; ++i) {
      ok = wait_bar(s_full(t), i & 1, ctl, 508);
      if (!(ok = __all_sync(0xffffffffu, ok))) break;
      tc_fence_after();
      // The row is read twice, 32 columns at a time: for its maximum, then for the exponentials
      // (TMEM reads are cheap next to keeping 128 scores in registers).
      const int kb = (tile_lo + i) * kKeys;
      const bool masked = __any_sync(0xffffffffu, kb < jlo || kb + kKeys - 1 > jhi);
      const int ja = jlo - kb, jb = jhi - kb;
      auto load_scores = [&](int c, float* s) {
        tmem_ld32(s_col + uint32_t(32 * c), s);
        tmem_wait_ld32(s);
        if (masked) {
#pragma unroll
          for (int j = 0; j < 32; ++j) s[j] = (32 * c + j >= ja && 32 * c + j <= jb) ? s[j] : -INFINITY;
        }
      };
      float mx = -INFINITY;
#pragma unroll
      for (int c = 0; c < 4; ++c) {
        float s[32];
        load_scores(c, s);
#pragma unroll
        for (int j = 0; j < 32; ++j) mx = fmaxf(mx, s[j]);
      }
      const float m_new = fmaxf(m, mx * p.scale_log2);
      const bool grow = m_new > m + kRescaleLog2 || (m == -INFINITY && m_new > m);
      if (__any_sync(0xffffffffu, grow)) {
        const float f = grow ? (m == -INFINITY ? 0.f : exp2_approx(m - m_new)) : 1.f;
        if (grow) {
          m = m_new;
          l *= f;
        }
        if (i > 0) {  // S of this tile is issued behind the previous P V: O is complete
#pragma unroll
          for (int c = 0; c < D / 32; ++c) {
            float o[32];
            tmem_ld32(o_col + uint32_t(32 * c), o);
            tmem_wait_ld32(o);
#pragma unroll
            for (int j = 0; j < 32; ++j) o[j] *= f;
            tmem_st32(o_col + uint32_t(32 * c), reinterpret_cast<const uint32_t*>(o));
          }
        }
      }
      const float mref = m == -INFINITY ? 0.f : m;
      float sum[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
      for (int c = 0; c < 4; ++c) {
        float s[32];
        uint32_t pk[16];
        load_scores(c, s);
#pragma unroll
        for (int j = 0; j < 32; j += 2) {
          const float e0 = exp2_approx(fmaf(s[j], p.scale_log2, -mref));
          const float e1 = exp2_approx(fmaf(s[j + 1], p.scale_log2, -mref));
          sum[j & 2] += e0;
          sum[(j & 2) + 1] += e1;
          pk[j / 2] = Elem<T>::pack(e0, e1);
        }
        tmem_st16(s_col + uint32_t(16 * c), pk);  // over columns whose scores have been read
      }
      l += (sum[0] + sum[1]) + (sum[2] + sum[3]);
      tmem_wait_st();
      tc_fence_before();
      mbar_arrive(p_full(t));
    }
    // ---- epilogue: the row's output
    if (ok && n > 0) {
      ok = wait_bar(o_full(t), 0, ctl, 509);
      ok = __all_sync(0xffffffffu, ok);
      tc_fence_after();
    }
    if (ok) {
      const int64_t row = int64_t(it.q0) + tok;
      const int head = kvh * G + g;
      if (PREFIX) {
        const int64_t slot = (int64_t(blockIdx.z) * p.total_q + row) * p.heads + head;
        if (row_ok) p.part_ml[slot] = make_float2(m, l);
        if (n > 0) {
#pragma unroll
          for (int c = 0; c < D / 32; ++c) {
            float o[32];
            tmem_ld32(o_col + uint32_t(32 * c), o);
            tmem_wait_ld32(o);
            if (row_ok) {
              float4* dst = reinterpret_cast<float4*>(p.part_o + slot * D + 32 * c);
#pragma unroll
              for (int j = 0; j < 8; ++j) dst[j] = make_float4(o[4 * j], o[4 * j + 1], o[4 * j + 2], o[4 * j + 3]);
            }
          }
        }
      } else {
        const bool has_sink = p.sinks != nullptr;
        float inv = 0.f, lse = 0.f;
        if (row_ok) {
          finish_row(m, l, has_sink, has_sink ? p.sinks[head] * kLog2e : 0.f, &inv, &lse);
          if (p.lse != nullptr) p.lse[row * p.heads + head] = lse;
        }
        uint4* dst = reinterpret_cast<uint4*>(reinterpret_cast<T*>(p.out) + row * p.out_ts + int64_t(head) * p.out_hs);
#pragma unroll
        for (int c = 0; c < D / 32; ++c) {
          float o[32];
          if (n > 0) {
            tmem_ld32(o_col + uint32_t(32 * c), o);
            tmem_wait_ld32(o);
          } else {
#pragma unroll
            for (int j = 0; j < 32; ++j) o[j] = 0.f;
          }
          if (row_ok) {
#pragma unroll
            for (int j = 0; j < 4; ++j) {
              uint4 w;
              w.x = Elem<T>::pack(o[8 * j] * inv, o[8 * j + 1] * inv);
              w.y = Elem<T>::pack(o[8 * j + 2] * inv, o[8 * j + 3] * inv);
              w.z = Elem<T>::pack(o[8 * j + 4] * inv, o[8 * j + 5] * inv);
              w.w = Elem<T>::pack(o[8 * j + 6] * inv, o[8 * j + 7] * inv);
              dst[c * 4 + j] = w;
            }
          }
        }
      }
    }
  }

  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  if (warp == kWarpMma)
    asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(kTmemCols));
}

template <typename T, int D, bool PREFIX>
int launch(const CUtensorMap& mq, const CUtensorMap& mk, const CUtensorMap& mv, const TcParams& p, dim3 grid, cudaStream_t s) {
  auto kernel = attn_tc_kernel<T, D, PREFIX>;
  KLC_CUDA(cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, Cfg<D>::kSmem));
  kernel<<<grid, kThreads, Cfg<D>::kSmem, s>>>(mq, mk, mv, p);
  KLC_LAUNCH_CHECK(PREFIX ? "attn_prefix" : "attn_prompt");
  return KLC_OK;
}

template <bool PREFIX>
int launch_typed(int dtype, int head_dim, const CUtensorMap& mq, const CUtensorMap& mk, const CUtensorMap& mv,
                 const TcParams& p, dim3 grid, cudaStream_t s) {
  if (dtype == KLC_BF16)
    return head_dim == 64 ? launch<__nv_bfloat16, 64, PREFIX>(mq, mk, mv, p, grid, s)
                          : launch<__nv_bfloat16, 128, PREFIX>(mq, mk, mv, p, grid, s);
  return head_dim == 64 ? launch<__half, 64, PREFIX>(mq, mk, mv, p, grid, s) : launch<__half, 128, PREFIX>(mq, mk, mv, p, grid, s);
}

CUtensorMapDataType map_type(int dtype) {
  return dtype == KLC_BF16 ? CU_TENSOR_MAP_DATA_TYPE_BFLOAT16 : CU_TENSOR_MAP_DATA_TYPE_FLOAT16;
}

// rows [tokens][heads][D] with token / head strides in elements; box of `box_heads` x `box_tokens`
int rows_map(CUtensorMap* m, int dtype, int head_dim, const void* base, int64_t tokens, int heads, int64_t ts, int64_t hs,
             int box_heads, int box_tokens) {
  const uint64_t dims[3] = {uint64_t(head_dim), uint64_t(heads), uint64_t(tokens)};
  const uint64_t strides[2] = {uint64_t(hs) * 2, uint64_t(ts) * 2};
  const uint32_t box[3] = {64, uint32_t(box_heads), uint32_t(box_tokens)};
  return make_map(m, map_type(dtype), 3, base, dims, strides, box, CU_TENSOR_MAP_SWIZZLE_128B);
}

}  // namespace

int check_rows(const char* who, const char* what, const void* base, int64_t tokens, int64_t ts, int64_t hs, int heads, int d) {
  const std::string w = std::string(who) + ": " + what;
  KLC_CHECK_ARG(base != nullptr, w + " is null");
  KLC_CHECK_ARG(aligned16(base), w + " must be 16-byte aligned");
  KLC_CHECK_ARG(ts % 8 == 0 && hs % 8 == 0, w + " strides must be multiples of 8 elements");
  KLC_CHECK_ARG((heads == 1 || hs >= d) && (tokens <= 1 || ts >= d), w + " strides must be at least head_dim");
  KLC_CHECK_ARG(ts < (int64_t(1) << 38) && hs < (int64_t(1) << 38), w + " strides are too large");
  return KLC_OK;
}

int pool_map(CUtensorMap* m, int dtype, int head_dim, const void* base, int64_t pages, int kv_heads, int page_size,
             int64_t page_stride, int box_rows) {
  const uint64_t dims[4] = {uint64_t(head_dim), uint64_t(page_size), uint64_t(kv_heads), uint64_t(pages)};
  const uint64_t strides[3] = {uint64_t(head_dim) * 2, uint64_t(page_size) * head_dim * 2, uint64_t(page_stride) * 2};
  const uint32_t box[4] = {64, uint32_t(box_rows), 1, 1};
  return make_map(m, map_type(dtype), 4, base, dims, strides, box, CU_TENSOR_MAP_SWIZZLE_128B);
}

int launch_prefix(const klc_attn_dims& dims, const DecodeParams& d, const void* q, const void* k_pages, const void* v_pages,
                  int64_t page_stride, cudaStream_t stream) {
  TcParams p{};
  p.cu_q = d.group_starts;
  p.batch = d.groups;
  p.total_q = d.batch;
  p.total_k = int64_t(d.table_width) * d.page_size;
  p.heads = d.heads;
  p.group = d.group;
  p.tpt = kRows / d.group;
  p.scale_log2 = d.scale_log2;
  p.window = d.window;
  p.status = d.status;
  p.prefix_lens = d.prefix_lens;
  p.lens = d.lens;
  p.block_table = d.block_table;
  p.table_stride = d.table_stride;
  p.pages = d.pages;
  p.page_size = d.page_size;
  p.part_o = d.prefix_o;
  p.part_ml = d.prefix_ml;
  CUtensorMap mq, mk, mv;
  int st = rows_map(&mq, dims.dtype, dims.head_dim, q, d.batch, d.heads, d.q_ts, d.q_hs, d.group, p.tpt);
  if (st == KLC_OK) st = pool_map(&mk, dims.dtype, dims.head_dim, k_pages, d.pages, d.kv_heads, d.page_size, page_stride, d.page_size);
  if (st == KLC_OK) st = pool_map(&mv, dims.dtype, dims.head_dim, v_pages, d.pages, d.kv_heads, d.page_size, page_stride, d.page_size);
  if (st != KLC_OK) return st;
  const int tok = 2 * p.tpt;
  const int pairs = d.groups == 1 ? (d.batch + tok - 1) / tok : std::min(d.batch, d.batch / tok + d.groups);
  return launch_typed<true>(dims.dtype, dims.head_dim, mq, mk, mv, p,
                            dim3(unsigned(pairs), unsigned(d.kv_heads), unsigned(d.splits)), stream);
}

}  // namespace attn
}  // namespace klc

extern "C" int klc_attn_prompt(const klc_attn_dims* dims, const void* q, int64_t q_tokens, int64_t q_token_stride,
                               int64_t q_head_stride, const void* k, int64_t k_token_stride, int64_t k_head_stride,
                               const void* v, int64_t v_token_stride, int64_t v_head_stride, int64_t k_tokens,
                               const int32_t* cu_q, const int32_t* cu_k, int64_t batch, const float* sinks, void* out,
                               int64_t out_token_stride, int64_t out_head_stride, float* lse, void* status, void* stream) {
  using namespace klc;
  using namespace klc::attn;
  const char* who = "klc_attn_prompt";
  KLC_CHECK_ARG(dims != nullptr, "klc_attn_prompt: null dims");
  int st = check_heads(who, dims->dtype, dims->heads, dims->kv_heads, dims->head_dim);
  if (st == KLC_OK) st = check_scale(who, dims->scale);
  if (st != KLC_OK) return st;
  KLC_CHECK_ARG(dims->window >= 0, "klc_attn_prompt: negative window");
  KLC_CHECK_ARG(q_tokens >= 0 && k_tokens >= 0 && batch >= 0, "klc_attn_prompt: negative size");
  KLC_CHECK_ARG(q_tokens < (1 << 30) && k_tokens < (1 << 30) && batch < (1 << 24), "klc_attn_prompt: sizes are too large");
  if (q_tokens == 0 || batch == 0) return KLC_OK;
  KLC_CHECK_ARG(cu_q != nullptr && cu_k != nullptr, "klc_attn_prompt: null sequence offsets");
  const int d = dims->head_dim;
  if ((st = check_rows(who, "q", q, q_tokens, q_token_stride, q_head_stride, dims->heads, d)) != KLC_OK) return st;
  if ((st = check_rows(who, "out", out, q_tokens, out_token_stride, out_head_stride, dims->heads, d)) != KLC_OK) return st;
  if (k_tokens > 0) {
    if ((st = check_rows(who, "k", k, k_tokens, k_token_stride, k_head_stride, dims->kv_heads, d)) != KLC_OK) return st;
    if ((st = check_rows(who, "v", v, k_tokens, v_token_stride, v_head_stride, dims->kv_heads, d)) != KLC_OK) return st;
  } else {  // no keys at all: every row is empty; the maps still need a tensor
    k = v = q;
    k_token_stride = v_token_stride = q_token_stride;
    k_head_stride = v_head_stride = q_head_stride;
  }
  const int G = dims->heads / dims->kv_heads;
  TcParams p{};
  p.cu_q = cu_q;
  p.cu_k = cu_k;
  p.batch = int(batch);
  p.total_q = q_tokens;
  p.total_k = k_tokens;
  p.heads = dims->heads;
  p.group = G;
  p.tpt = kRows / G;
  p.scale_log2 = dims->scale * kLog2e;
  p.window = dims->window;
  p.sinks = sinks;
  p.out = out;
  p.out_ts = out_token_stride;
  p.out_hs = out_head_stride;
  p.lse = lse;
  p.status = reinterpret_cast<DeviceStatus*>(status);
  CUtensorMap mq, mk, mv;
  if ((st = rows_map(&mq, dims->dtype, d, q, q_tokens, dims->heads, q_token_stride, q_head_stride, G, p.tpt)) != KLC_OK) return st;
  const int64_t kt = std::max<int64_t>(k_tokens, 1);
  if ((st = rows_map(&mk, dims->dtype, d, k, kt, dims->kv_heads, k_token_stride, k_head_stride, 1, kKeys)) != KLC_OK) return st;
  if ((st = rows_map(&mv, dims->dtype, d, v, kt, dims->kv_heads, v_token_stride, v_head_stride, 1, kKeys)) != KLC_OK) return st;
  // pairs of row tiles: sum over sequences of ceil(len / (2 tpt)), at most this
  const int64_t gx = q_tokens / (2 * p.tpt) + std::min<int64_t>(batch, q_tokens);
  return launch_typed<false>(dims->dtype, d, mq, mk, mv, p, dim3(unsigned(gx), unsigned(dims->kv_heads)), as_stream(stream));
}
